// Causal attention over expanded latent keys and values
// (nvb_latent_prefill_fwd). No counterpart in the reference, whose models have
// one head size for keys and values.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale (q_i . k_j + q'_i . r_j))
//
// over the keys j that query i sees; k and v are a head's (128 values each), r
// is the rotated part (64) that all heads share. Work item: two adjacent tiles A
// and B of 128 queries of one (sequence, head), or one where a launch has fewer
// pairs than SMs. Per tile of 128 keys and x in {A, B}:
//
//   S_x = Q_x K_j^T   tcgen05.mma M=128 N=128 K=192 (two pieces of k, one of r)
//   P_x = exp2(S_x * scale * log2 e - m), a warpgroup, a thread a row; written
//         back over S_x in TMEM as packed BF16
//   O_x += P_x V_j    tcgen05.mma M=128 N=128 K=128, P from TMEM
//
// The two tiles' chains run out of phase, as in prefill.cu. Shared memory: Q of
// both tiles (96 KB) and a ring of eight 16 KB pieces (128 keys x 64 values) in
// the order of their use, K_j (three) and V_j (two): V_j+1 takes the places that
// K_j leaves, K_j+2 those of V_j.
//
// What bounds it: the tensor core takes 2,560 cycles for a step of both tiles
// and 128 keys, the exponentials 1,800 of the MUFU unit; the chain of softmax,
// product and next scores makes it 3,900 to 4,700 (S has one buffer a tile: O and
// S of both fill TMEM). Measured (B200, calls back to back for seconds, where the
// power cap holds the SM clock between 1.58 and 1.71 GHz for 1.97; in brackets the
// best of a few calls; TFLOP/s of the pairs that are seen): 4 prompts of 8192 tokens, 16
// heads 1.35 ms, 1,010 TFLOP/s (1.17 ms, 1,170); 4 x ~506 queries behind 4000 to
// 8000 keys, 32 heads 288 us, 800 (250 us, 920); 32 prompts of 64 to 2048 303 us,
// 610 (256 us, 720; a ragged end of a tile and the masked half of the diagonal are
// 18 % of the work, an item's start and end ~8,000 cycles of ~32,000); one of 300
// 11.6 us. Tried and no faster: tile B started half a step behind tile A, the next
// item looked up early.
//
// Roles (16 warps, one CTA an SM):
//   warp 0      claims items: a CTA that has begun takes over the indices of CTAs
//               that have not (cluster launch control), so nothing is kept in
//               memory between launches; publishes them in a two-slot ring and
//               loads Q, K and V by TMA
//   warp 1      TMEM; one thread issues the S MMAs
//   warp 2      one thread issues the PV MMAs
//   warp 3      mends V: rows behind the sequence are zeroed, and so is what is
//               not finite in keys that not all queries see (their probability
//               of 0 would not cancel it); the epilogue adds it where it is seen
//   warps 4-7   softmax of tile A, warps 8-11 of tile B
//   warps 12-15 epilogue: O / l in BF16
// Every wait is bounded; a timeout records an error code, and the CTA waits for
// its copies and MMAs, frees TMEM and exits.
#include "latent_common.cuh"

namespace nvb {

namespace latent_prefill_detail {

using namespace latent_common;

constexpr int kRows = 128, kKeys = 128;
constexpr int kPiece = 128 * 128;            // 128 rows x 64 BF16, 128-byte swizzled
constexpr int kQPieces = 3, kKPieces = 3, kTilePieces = 5;
constexpr int kSlots = 8;
constexpr int kThreads = 512;
constexpr int kTmemCols = 512;
constexpr int kSCol = 0, kOCol = 256;        // S/P of tile x at kSCol + 128 x, O at kOCol + 128 x
// Registers after set-up: the softmax warpgroups hold a row's 128 scores.
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 200, kOtherRegs = 56;
static_assert(2 * 128 * kSoftmaxRegs + 2 * 128 * kOtherRegs == kThreads * kLaunchRegs, "register split");

// Empty: one a place. Landed and mended tiles alternate between two barriers: K of tile g + 2, and V behind it, takes
// places that V of tile g leaves, so all that waits for tile g's has passed. [2] else: per query tile, or alternating.
enum Bar {
  kEmpty = 0, kKFull = kEmpty + kSlots, kVFull = kKFull + 2, kVReady = kVFull + 2, kQFull = kVReady + 2,
  kQFree = kQFull + 2, kSFull = kQFree + 2, kPFull = kSFull + 2, kPVDone = kPFull + 2, kODone = kPVDone + 2,
  kOFree = kODone + 2, kStatsFull = kOFree + 2,
  kStatsFree = kStatsFull + 2, kItemFull = kStatsFree + 2, kItemEmpty = kItemFull + 2, kClaim = kItemEmpty + 2,
  kSDrain, kPVDrain, kNumBars
};
// S issuer, PV issuer, mender (one arrival each), 8 softmax and 4 epilogue warps.
constexpr int kItemReaders = 15;

struct Item {
  int b, h, q_begin, k_begin, keys, prefix;
  int q0[2];       // first query of tile A / B within the sequence
  int qx[2];       // queries in the tile (0: the tile is past the sequence)
  int n[2];        // KV tiles the tile visits
  int full[2];     // leading KV tiles every row of the tile sees whole
};
constexpr int kMaxOrdered = 256;             // sequences that a launch puts in order
constexpr int kTmemSlotOff = kNumBars * 8;
constexpr int kBadOff = kTmemSlotOff + 4;    // int [4]: whether item i % 4 had V values that were taken out
constexpr int kClaimOff = (kBadOff + 16 + 15) & ~15;        // 16 bytes: the answer to a claim
constexpr int kItemOff = kClaimOff + 16;                    // Item [2]
constexpr int kStatsOff = (kItemOff + 2 * int(sizeof(Item)) + 15) & ~15;  // float [2][128]: 1 / l
constexpr int kOrderOff = kStatsOff + 2 * kRows * 4;        // uint16 [kMaxOrdered]: sequences, the longest first
constexpr int kHeadBytes = 3 * 1024;
static_assert(kOrderOff + kMaxOrdered * 2 <= kHeadBytes && 2 * kRows >= kMaxOrdered, "head layout");
constexpr int kQOff = kHeadBytes;
constexpr int kRingOff = kQOff + 2 * kQPieces * kPiece;
constexpr int kSmemBytes = kRingOff + kSlots * kPiece;
static_assert(kSmemBytes <= 232448, "per-CTA shared memory limit");

// PV of 64 dims: B MN-major, N = 64.
constexpr uint32_t kIdescPVHalf =
    (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24) | ((64u >> 3) << 17) | (1u << 16);

// ------------------------------------------------------------------- items
struct Sizes {
  int q_begin, n, q_len, k_begin, keys;  // q_len: the queries that are worked on
};
__device__ __forceinline__ Sizes sizes(const LatentPrefillParams& p, int b) {
  Sizes s;
  s.q_begin = min(max(p.cu_q[b], 0), p.total_q);
  s.n = min(max(p.cu_q[b + 1], s.q_begin), p.total_q) - s.q_begin;
  s.q_len = min(s.n, p.max_q);
  const int begin = p.cu_k[b], end = p.cu_k[b + 1];
  const bool valid = begin >= 0 && end >= begin && end <= p.total_k;
  s.k_begin = valid ? begin : 0;
  s.keys = valid ? end - begin : 0;
  return s;
}

// Items in the order of their claims: by sequence (the longest first, up to kMaxOrdered sequences), its last queries
// first, heads next to one another. Tiles are paired from the sequence's end, so that one without a partner, whose steps
// take as long as a pair's, is the one with the fewest keys. A warp looks at 32 sequences at a time.
struct Cursor {
  int r0 = -32, base = 0;        // first of the 32, items before them
  int b = -1, items = 0, upto = 0;  // this lane's sequence, its items, items up to and with it among the 32
};
__device__ __forceinline__ void cursor_load(const LatentPrefillParams& p, const uint16_t* order, Cursor& c, int lane) {
  const int r = c.r0 + lane;
  c.b = r < p.batch ? (order ? int(order[r]) : r) : -1;
  c.items = 0;
  if (c.b >= 0) c.items = (sizes(p, c.b).q_len + p.item_rows - 1) / p.item_rows * p.heads;
  c.upto = c.items;
#pragma unroll
  for (int off = 1; off < 32; off *= 2) {
    const int o = __shfl_up_sync(0xffffffffu, c.upto, off);
    if (lane >= off) c.upto += o;
  }
}
// Item v, or b = -1 where there is none.
__device__ __forceinline__ Item find_item(const LatentPrefillParams& p, const uint16_t* order, Cursor& c, int v,
                                          int lane) {
  Item it;
  it.b = -1;
  if (c.r0 < 0 || v < c.base) {
    c.r0 = c.base = 0;
    cursor_load(p, order, c, lane);
  }
  for (;;) {
    const int all = __shfl_sync(0xffffffffu, c.upto, 31);
    if (v < c.base + all) break;
    if (c.r0 + 32 >= p.batch) return it;
    c.base += all;
    c.r0 += 32;
    cursor_load(p, order, c, lane);
  }
  const int l = __ffs(__ballot_sync(0xffffffffu, c.base + c.upto > v)) - 1;
  const int b = __shfl_sync(0xffffffffu, c.b, l), items = __shfl_sync(0xffffffffu, c.items, l);
  const int within = v - c.base - (__shfl_sync(0xffffffffu, c.upto, l) - items);
  const int row = within / p.heads;
  const Sizes s = sizes(p, b);
  it.b = b;
  it.h = within - row * p.heads;
  it.q_begin = s.q_begin;
  it.k_begin = s.k_begin;
  it.keys = s.keys;
  it.prefix = s.keys - s.n;
  const int pair = p.item_rows / kRows, first = (s.q_len + kRows - 1) / kRows - pair * (row + 1);  // tile; -1: tile 0 alone
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    it.q0[x] = (max(first, 0) + x) * kRows;
    it.qx[x] = x < pair + min(first, 0) ? min(kRows, s.q_len - it.q0[x]) : 0;
    const int end = it.qx[x] ? max(0, min(s.keys, it.prefix + it.q0[x] + it.qx[x])) : 0;
    it.n[x] = (end + kKeys - 1) / kKeys;
    it.full[x] = max(0, min(s.keys, it.prefix + it.q0[x] + 1)) / kKeys;
  }
  return it;
}

// Item i of this CTA from the ring. Returns false at the end marker (b < 0) or if the wait gave up.
__device__ __forceinline__ bool take_item(uint64_t* bars, const Item* ring, int i, bool warp_level, Item& it) {
  const int slot = i & 1;
  const uint32_t par = (i >> 1) & 1;
  if (warp_level ? !wait_warp(&bars[kItemFull + slot], par) : !wait(&bars[kItemFull + slot], par)) return false;
  it = ring[slot];
  if (warp_level) __syncwarp();
  if (!warp_level || (threadIdx.x & 31) == 0) mbar_arrive(&bars[kItemEmpty + slot]);
  return it.b >= 0;
}

// 2^x of a pair on the FMA pipe (x <= 128): x = n + f with n the nearest integer (by the rounding of 1.5 * 2^23 + x),
// a polynomial of degree 4 for 2^f that is 1 at 0 (this file's fit, relative error below 2.9e-6), n added to its
// exponent. From x = -127 down that gives 0 exactly, so that a masked key (-inf) has no part in the result whatever
// finite value it has: 2^-125, as where inputs are clamped before the exponent reaches its end, is 7 with a value of
// 3e38. Between -127 and -126 it is off by 2^-127 at most (below the normal numbers).
__device__ __forceinline__ void exp2_to_zero_pair(float& a, float& b) {
  const float xa = fmaxf(a, -127.0f), xb = fmaxf(b, -127.0f);
  float ta, tb, na, nb, fa, fb, pa, pb;
  add2(ta, tb, xa, xb, 12582912.0f, 12582912.0f);
  add2(na, nb, ta, tb, -12582912.0f, -12582912.0f);
  fma2(fa, fb, na, nb, -1.0f, -1.0f, xa, xb);
  fma2(pa, pb, 0.009582852944731712f, 0.009582852944731712f, fa, fb, 0.055906426161527634f, 0.055906426161527634f);
  fma2(pa, pb, pa, pb, fa, fb, 0.24024099111557007f, 0.24024099111557007f);
  fma2(pa, pb, pa, pb, fa, fb, 0.6931241750717163f, 0.6931241750717163f);
  fma2(pa, pb, pa, pb, fa, fb, 1.0f, 1.0f);
  a = __int_as_float(__float_as_int(ta) * 8388608 + __float_as_int(pa));
  b = __int_as_float(__float_as_int(tb) * 8388608 + __float_as_int(pb));
}

// exp2(s * sl2 + nm) for keys [C0, C0 + 32) of a row -> 16 packed BF16 pairs; row-sum partials accumulate in `sum`.
// One pair in eight runs on the FMA pipe. BF16 is V's type: half a step of each probability; the sum keeps FP32.
template <int C0>
__device__ __forceinline__ void exp32(const float (&s)[128], float sl2, float nm, uint32_t (&pk)[16],
                                      float (&sum)[8]) {
#pragma unroll
  for (int c = C0; c < C0 + 32; c += 2) {
    float e0 = s[c], e1 = s[c + 1];
    fma2(e0, e1, e0, e1, sl2, sl2, nm, nm);
    if ((c & 15) == 14) {
      exp2_to_zero_pair(e0, e1);
    } else {
      e0 = fast_exp2(e0);
      e1 = fast_exp2(e1);
    }
    const int k = (c >> 1) & 3;
    add2(sum[2 * k], sum[2 * k + 1], sum[2 * k], sum[2 * k + 1], e0, e1);
    pk[(c - C0) >> 1] = pack_bf16x2(e0, e1);
  }
}

// The largest of three, NaN where one is.
__device__ __forceinline__ float max3n(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

__device__ __forceinline__ void softmax_role(const LatentPrefillParams& p, uint64_t* bars, const Item* ring,
                                             float* stats, uint32_t tmem, int warp, int lane) {
  const int x = (warp - 4) >> 2, quad = warp & 3;
  const int r = quad * 32 + lane;  // TMEM lane: query of the tile
  const uint32_t lane_base = tmem + (uint32_t(quad * 32) << 16);
  const uint32_t scol = lane_base + kSCol + x * kKeys, ocol = lane_base + kOCol + x * kKeys;
  const float sl2 = p.scale * kLog2e;
  int t = 0, ix = 0;  // tiles and items of this query tile
  bool alive = true;
  Item it;
  for (int i = 0; alive && take_item(bars, ring, i, true, it); ++i) {
    const int n = x ? it.n[1] : it.n[0], qx = x ? it.qx[1] : it.qx[0], q0 = x ? it.q0[1] : it.q0[0];
    const int full = x ? it.full[1] : it.full[0];
    if (n == 0) continue;
    // queries behind the last one see what that sees; their results are dropped
    const int limit = min(it.prefix + q0 + min(r, qx - 1), it.keys - 1);
    float m_used = -INFINITY, l = 0.0f;
    for (int j = 0; j < n; ++j, ++t) {
      if (!wait_warp(&bars[kSFull + x], t & 1)) {
        alive = false;
        break;
      }
      tc_fence_after();
      float s[128];
      {
        uint32_t a0[32], a1[32], a2[32], a3[32];
        tmem_ld32(scol, a0);
        tmem_ld32(scol + 32, a1);
        tmem_ld32(scol + 64, a2);
        tmem_ld32(scol + 96, a3);
        tmem_ld_wait();
        reg_fence(a0);
        reg_fence(a1);
        reg_fence(a2);
        reg_fence(a3);
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          s[c] = __uint_as_float(a0[c]);
          s[32 + c] = __uint_as_float(a1[c]);
          s[64 + c] = __uint_as_float(a2[c]);
          s[96 + c] = __uint_as_float(a3[c]);
        }
      }
      if (j >= full) {
        const int lim = limit - j * kKeys;
#pragma unroll
        for (int c = 0; c < 128; ++c)
          if (c > lim) s[c] = -INFINITY;
      }
      float mx[8];
#pragma unroll
      for (int i8 = 0; i8 < 8; ++i8) mx[i8] = s[i8];
#pragma unroll
      for (int c = 8; c < 120; c += 16)
#pragma unroll
        for (int i8 = 0; i8 < 8; ++i8) mx[i8] = max3n(mx[i8], s[c + i8], s[c + 8 + i8]);
#pragma unroll
      for (int i8 = 0; i8 < 8; ++i8) mx[i8] = max3n(mx[i8], s[120 + i8], s[120 + i8]);
      const float m_tile =
          max3n(max3n(mx[0], mx[1], mx[2]), max3n(mx[3], mx[4], mx[5]), max3n(mx[6], mx[7], mx[7])) * sl2;
      float alpha = 1.0f;
      if (m_tile > m_used + kRescaleLog2) {
        alpha = fast_exp2(m_used - m_tile);  // 0 with the first key
        m_used = m_tile;
      }
      if (j >= 1 && __any_sync(0xffffffffu, alpha != 1.0f)) {
        // PV_x of the tile before completed before S_x of this one was issued; the wait orders its writes of O here.
        if (!wait_warp(&bars[kPVDone + x], (t - 1) & 1)) {
          alive = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int h = 0; h < 4; ++h) {
          uint32_t o[32];
          tmem_ld32(ocol + h * 32, o);
          tmem_ld_wait();
          reg_fence(o);
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
          tmem_st32(ocol + h * 32, o);
        }
      }
      const float nm = m_used == -INFINITY ? 0.0f : -m_used;
      float sum[8];
#pragma unroll
      for (int i8 = 0; i8 < 8; ++i8) sum[i8] = 0.0f;
      {
        // keys [32 g, +32) -> packed columns [16 g, +16) of S_x
        uint32_t pk[16];
        exp32<0>(s, sl2, nm, pk, sum);
        tmem_st16(scol, pk);
        exp32<32>(s, sl2, nm, pk, sum);
        tmem_st16(scol + 16, pk);
        exp32<64>(s, sl2, nm, pk, sum);
        tmem_st16(scol + 32, pk);
        exp32<96>(s, sl2, nm, pk, sum);
        tmem_st16(scol + 48, pk);
      }
      l = l * alpha + (((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7])));
      if (!(m_tile < INFINITY)) l = NAN;  // the exponentials of the FMA pipe do not carry NaN
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kPFull + x]);
    }
    if (!alive) break;
    if (ix > 0 && !wait_warp(&bars[kStatsFree + x], (ix - 1) & 1)) break;
    // no key seen: the sum is 0; a row of NaN scores has a NaN sum
    stats[x * kRows + r] = l == 0.0f ? 0.0f : 1.0f / l;
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars[kStatsFull + x]);
    if (p.lse && r < qx)
      p.lse[(long long)(it.q_begin + q0 + r) * p.heads + it.h] =
          l == 0.0f ? -INFINITY : ((m_used == -INFINITY ? 0.0f : m_used) + fast_log2(l)) * kLn2;
    ++ix;
  }
}

__global__ void __launch_bounds__(kThreads, 1)
    latent_prefill_kernel(const LatentPrefillParams p, const __grid_constant__ CUtensorMap qmap,
                          const __grid_constant__ CUtensorMap kvmap, const __grid_constant__ CUtensorMap rmap) {
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t sbase = smem_addr(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kTmemSlotOff);
  volatile int* bad = reinterpret_cast<volatile int*>(smem + kBadOff);
  Item* ring = reinterpret_cast<Item*>(smem + kItemOff);
  float* stats = reinterpret_cast<float*>(smem + kStatsOff);
  uint16_t* order = reinterpret_cast<uint16_t*>(smem + kOrderOff);

  // Set-up that needs no input runs beside the end of the kernel before this one.
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) mbar_init(&bars[kEmpty + s], 1);
    for (int s = 0; s < 2; ++s) {
      for (int bar : {kKFull, kVFull, kVReady, kQFull, kQFree, kSFull, kPVDone, kODone, kItemFull})
        mbar_init(&bars[bar + s], 1);
      for (int bar : {kPFull, kOFree, kStatsFull, kStatsFree}) mbar_init(&bars[bar + s], 4);
      mbar_init(&bars[kItemEmpty + s], kItemReaders);
    }
    mbar_init(&bars[kClaim], 1);
    mbar_init(&bars[kSDrain], 1);
    mbar_init(&bars[kPVDrain], 1);
    fence_barrier_init();
    for (int i = 0; i < 4; ++i) bad[i] = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // that kernel has completed, its writes are visible
  // The sequences in falling order of their keys, so that the last claims are small items; equal ones by index.
  const bool ordered = p.batch <= kMaxOrdered;
  if (ordered) {
    int* keys = reinterpret_cast<int*>(stats);
    const int b = threadIdx.x;
    int mine = 0;
    if (b < p.batch) {
      const Sizes s = sizes(p, b);
      mine = s.q_len ? s.keys : -1;
      keys[b] = mine;
    }
    __syncthreads();
    if (b < p.batch) {
      int rank = 0;
      for (int o = 0; o < p.batch; ++o) rank += keys[o] > mine || (keys[o] == mine && o < b);
      order[rank] = uint16_t(b);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const bool aligned = (sbase & 1023u) == 0;
  if (!aligned && threadIdx.x == 0) record_error(kErrPrefillAlign);

  if (!aligned) {
  } else if (warp >= 4 && warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    softmax_role(p, bars, ring, stats, tmem, warp, lane);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 0) {
      // ------------------------------------------- claims and producer
      const bool leader = elect_one();
      if (leader) {
        tma_prefetch_desc(&qmap);
        tma_prefetch_desc(&kvmap);
        tma_prefetch_desc(&rmap);
      }
      Cursor cursor;
      int v = blockIdx.x, i = 0, claims = 0, issued = 0, gk = 0, gv = 0, ixq[2] = {0, 0};
      bool alive = true;
      // the next piece of the ring, once the MMAs that read its place have; `pieces` where a tile's first
      auto load = [&](const CUtensorMap* map, int xc, int head, int row, int bar, int pieces) {
        const int slot = issued % kSlots;
        if (issued >= kSlots) alive = alive && wait_warp(&bars[kEmpty + slot], ((issued / kSlots) + 1) & 1);
        if (!alive) return;
        if (leader) {
          if (pieces) expect_bytes(sbase + bar * 8, uint32_t(pieces) * kPiece);
          tma_load_3d_at(sbase + kRingOff + slot * kPiece, map, sbase + bar * 8, xc, head, row);
        }
        ++issued;
      };
      for (bool more = true; alive && more;) {
        if (leader) {  // the next index, while this item is loaded
          expect_bytes(sbase + kClaim * 8, 16);
          asm volatile(
              "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                  sbase + kClaimOff),
              "r"(sbase + kClaim * 8)
              : "memory");
        }
        const Item it = find_item(p, ordered ? order : nullptr, cursor, v, lane);
        if (it.b >= 0) {
          if (i >= 2) alive = wait_warp(&bars[kItemEmpty + (i & 1)], ((i >> 1) + 1) & 1);
          if (alive && lane == 0) {
            bad[i & 3] = 0;
            ring[i & 1] = it;
            mbar_arrive(&bars[kItemFull + (i & 1)]);
          }
          __syncwarp();
          ++i;
          const int nt = max(it.n[0], it.n[1]);
          auto load_k = [&](int j) {
            const int row = it.k_begin + j * kKeys;
            const int bar = kKFull + (gk & 1);
            load(&kvmap, 0, it.h, row, bar, kKPieces);
            load(&kvmap, 64, it.h, row, bar, 0);
            load(&rmap, 0, 0, row, bar, 0);
            ++gk;
          };
          // The item's first K tile goes out before its Q, whose place is free later.
          if (nt) load_k(0);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (it.n[x] == 0) continue;
            // free once the last S of its tile before has read it
            if (ixq[x] >= 1) alive = alive && wait_warp(&bars[kQFree + x], (ixq[x] - 1) & 1);
            if (!alive) break;
            if (leader) {
              const uint32_t full = sbase + (kQFull + x) * 8;
              expect_bytes(full, kQPieces * kPiece);
#pragma unroll
              for (int c = 0; c < kQPieces; ++c)
                tma_load_3d_at(sbase + kQOff + (x * kQPieces + c) * kPiece, &qmap, full, c * 64, it.h,
                               it.q_begin + it.q0[x]);
            }
            ++ixq[x];
          }
          for (int j = 0; j < nt && alive; ++j) {
            const int row = it.k_begin + j * kKeys;
            const int bar = kVFull + (gv & 1);
            load(&kvmap, 128, it.h, row, bar, kTilePieces - kKPieces);
            load(&kvmap, 192, it.h, row, bar, 0);
            ++gv;
            if (j + 1 < nt) load_k(j + 1);
          }
        }
        if (!wait_warp(&bars[kClaim], claims & 1)) break;
        ++claims;
        uint32_t taken, next;
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\tld.shared.b128 r, [%2];\n\t"
            "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
            "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
            : "=r"(taken), "=r"(next)
            : "r"(sbase + kClaimOff)
            : "memory");
        fence_proxy_async_smem();  // read before the next answer is written
        __syncwarp();
        more = taken != 0;
        v = int(next);
      }
      // the end marker
      if (alive && i >= 2) alive = wait_warp(&bars[kItemEmpty + (i & 1)], ((i >> 1) + 1) & 1);
      if (alive && lane == 0) {
        ring[i & 1].b = -1;
        mbar_arrive(&bars[kItemFull + (i & 1)]);
      }
      // Every copy has landed before the CTA may exit (on the normal path its readers have waited for it).
      for (int g = max(0, gk - 2); g < gk; ++g) wait_warp(&bars[kKFull + (g & 1)], (g >> 1) & 1);
      for (int g = max(0, gv - 2); g < gv; ++g) wait_warp(&bars[kVFull + (g & 1)], (g >> 1) & 1);
      for (int x = 0; x < 2; ++x)
        if (ixq[x] > 0) wait_warp(&bars[kQFull + x], (ixq[x] - 1) & 1);
    } else if (warp == 1) {
      // --------------------------------------------------- S MMA issuer
      if (elect_one()) {
        const uint64_t qd = sw128_desc(sbase + kQOff, 16, 1024), kd = sw128_desc(sbase + kRingOff, 16, 1024);
        const uint32_t q_lo = uint32_t(qd), q_hi = uint32_t(qd >> 32), k_lo = uint32_t(kd), k_hi = uint32_t(kd >> 32);
        int g = 0, tx[2] = {0, 0}, ixq[2] = {0, 0};
        bool alive = true;
        Item it;
        for (int i = 0; alive && take_item(bars, ring, i, false, it); ++i) {
          const int nt = max(it.n[0], it.n[1]);
          for (int j = 0; j < nt && alive; ++j, ++g) {
            uint32_t kb[kKPieces];
#pragma unroll
            for (int c = 0; c < kKPieces; ++c) kb[c] = k_lo + uint32_t((kTilePieces * g + c) % kSlots) * (kPiece >> 4);
            alive = wait(&bars[kKFull + (g & 1)], (g >> 1) & 1);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              if (j >= it.n[x]) continue;
              if (j == 0) alive = alive && wait(&bars[kQFull + x], ixq[x] & 1);
              // single-buffered: P of the tile's step before, in the same columns, has been read
              if (tx[x] >= 1) alive = alive && wait(&bars[kPVDone + x], (tx[x] - 1) & 1);
              if (!alive) break;
              tc_fence_after();
              const uint32_t qa = q_lo + uint32_t(x * kQPieces) * (kPiece >> 4), sd = tmem + kSCol + x * kKeys;
#pragma unroll
              for (int c = 0; c < kKPieces; ++c)
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                  umma_ss(sd, qa + uint32_t((c * kPiece + kk * 32) >> 4), q_hi, kb[c] + uint32_t(kk * 2), k_hi, kIdescS,
                          (c | kk) ? 1u : 0u);
              umma_commit(&bars[kSFull + x]);
              if (j == it.n[x] - 1) {
                umma_commit(&bars[kQFree + x]);
                ++ixq[x];
              }
              ++tx[x];
            }
            if (!alive) break;
#pragma unroll
            for (int c = 0; c < kKPieces; ++c) umma_commit(&bars[kEmpty + (kTilePieces * g + c) % kSlots]);
          }
        }
        // every MMA of this thread completes before TMEM is freed
        umma_commit(&bars[kSDrain]);
        wait(&bars[kSDrain], 0);
      }
    } else if (warp == 2) {
      // -------------------------------------------------- PV MMA issuer
      if (elect_one()) {
        // V: the two pieces of a tile are neighbours in the ring or its last and first
        const uint64_t vd = sw128_desc(sbase + kRingOff, kPiece, 1024);
        const uint32_t v_lo = uint32_t(vd), v_hi = uint32_t(vd >> 32);
        int g = 0, tx[2] = {0, 0}, ixo[2] = {0, 0};
        bool alive = true;
        Item it;
        for (int i = 0; alive && take_item(bars, ring, i, false, it); ++i) {
          const int nt = max(it.n[0], it.n[1]);
          for (int j = 0; j < nt && alive; ++j, ++g) {
            const int k = kTilePieces * g + kKPieces;
            const uint32_t v0 = v_lo + uint32_t(k % kSlots) * (kPiece >> 4),
                           v1 = v_lo + uint32_t((k + 1) % kSlots) * (kPiece >> 4);
            alive = wait(&bars[kVReady + (g & 1)], (g >> 1) & 1);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              if (j >= it.n[x]) continue;
              // the epilogue has read the tile's O before
              if (j == 0 && ixo[x] > 0) alive = alive && wait(&bars[kOFree + x], (ixo[x] - 1) & 1);
              alive = alive && wait(&bars[kPFull + x], tx[x] & 1);
              if (!alive) break;
              tc_fence_after();
              const uint32_t pa = tmem + kSCol + x * kKeys, od = tmem + kOCol + x * kKeys;
              const uint32_t fresh = j == 0 ? 0u : 1u;
              // 16 keys: 8 packed columns of P, 2048 bytes of V rows
              if (v1 > v0) {
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                  umma_ts(od, pa + kk * 8, v0 + kk * 128, v_hi, kIdescPV, kk ? 1u : fresh);
              } else {  // the ring's last and first piece: 64 dims each
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                  umma_ts(od, pa + kk * 8, v0 + kk * 128, v_hi, kIdescPVHalf, kk ? 1u : fresh);
#pragma unroll
                for (int kk = 0; kk < 8; ++kk)
                  umma_ts(od + 64, pa + kk * 8, v1 + kk * 128, v_hi, kIdescPVHalf, kk ? 1u : fresh);
              }
              umma_commit(&bars[kPVDone + x]);
              if (j == it.n[x] - 1) {
                umma_commit(&bars[kODone + x]);
                ++ixo[x];
              }
              ++tx[x];
            }
            if (!alive) break;
            umma_commit(&bars[kEmpty + k % kSlots]);
            umma_commit(&bars[kEmpty + (k + 1) % kSlots]);
          }
        }
        umma_commit(&bars[kPVDrain]);
        wait(&bars[kPVDrain], 0);
      }
    } else if (warp == 3) {
      // --------------------------------------------------------- mender
      int g = 0;
      bool alive = true;
      Item it;
      for (int i = 0; alive && take_item(bars, ring, i, true, it); ++i) {
        const int nt = max(it.n[0], it.n[1]);
        for (int j = 0; j < nt; ++j, ++g) {
          const int k = kTilePieces * g + kKPieces, key0 = j * kKeys;
          alive = alive && wait_warp(&bars[kVFull + (g & 1)], (g >> 1) & 1);
          if (!alive) break;
          const int real = min(kKeys, it.keys - key0);  // keys of the sequence
          // 16-byte piece i of the tile's rows, 16 a row
          auto piece = [&](int e) {
            return reinterpret_cast<uint4*>(smem + kRingOff + ((k + ((e >> 3) & 1)) % kSlots) * kPiece + (e >> 4) * 128 +
                                            (e & 7) * 16);
          };
          for (int e = 16 * real + lane; e < 16 * kKeys; e += 32) *piece(e) = make_uint4(0, 0, 0, 0);
          // the first key that a query which visits the tile does not see
          const int unseen = it.prefix + 1 + (j < it.n[0] ? it.q0[0] : it.q0[1]);
          const int from = 16 * max(0, min(unseen - key0, real)) + lane;
          // Looked for first: x * 0 adds NaN to a sum where x is not finite. The tile's PV waits for this (a test and a
          // branch a piece took 8,000 cycles for a whole tile, of an item's ~20,000).
          __nv_bfloat162 sum[4];
          const __nv_bfloat162 zero = __floats2bfloat162_rn(0.0f, 0.0f);
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[c] = zero;
#pragma unroll 4
          for (int e = from; e < 16 * real; e += 32) {
            const uint4 w = *piece(e);
            sum[0] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.x), zero, sum[0]);
            sum[1] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.y), zero, sum[1]);
            sum[2] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.z), zero, sum[2]);
            sum[3] = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w.w), zero, sum[3]);
          }
          const __nv_bfloat162 any = __hadd2(__hadd2(sum[0], sum[1]), __hadd2(sum[2], sum[3]));
          if (__hisnan(__low2bfloat16(any)) || __hisnan(__high2bfloat16(any))) {
            bad[i & 3] = 1;
            for (int e = from; e < 16 * real; e += 32) {
              const uint4 w = *piece(e);
              *piece(e) = make_uint4(finite_part(w.x), finite_part(w.y), finite_part(w.z), finite_part(w.w));
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars[kVReady + (g & 1)]);
        }
      }
    } else {
      // ------------------------------------------------------- epilogue
      const int quad = warp & 3, r = quad * 32 + lane;
      const uint32_t lane_base = tmem + (uint32_t(quad * 32) << 16);
      int ixo[2] = {0, 0};
      bool alive = true;
      Item it;
      for (int i = 0; alive && take_item(bars, ring, i, true, it); ++i) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (it.qx[x] == 0 || !alive) continue;
          const bool valid = r < it.qx[x];
          const long long row = (long long)(it.q_begin + it.q0[x] + r) * p.heads + it.h;
          __nv_bfloat16* dst = p.out + row * 128;
          if (it.n[x] == 0) {  // no query of the tile sees a key
            if (valid) {
              for (int d = 0; d < 128; d += 8) *reinterpret_cast<uint4*>(dst + d) = make_uint4(0, 0, 0, 0);
              if (p.lse) p.lse[row] = -INFINITY;
            }
            continue;
          }
          alive = alive && wait_warp(&bars[kStatsFull + x], ixo[x] & 1);
          const float inv = stats[x * kRows + r];
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars[kStatsFree + x]);
          alive = alive && wait_warp(&bars[kODone + x], ixo[x] & 1);
          if (!alive) break;
          tc_fence_after();
          const bool mend = bad[i & 3] != 0;
#pragma unroll 1
          for (int h = 0; h < 8; ++h) {
            uint32_t o[16];
            tmem_ld16(lane_base + kOCol + x * kKeys + h * 16, o);
            tmem_ld_wait();
            reg_fence(o);
            if (h == 7) {  // O_x is read
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&bars[kOFree + x]);
            }
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * inv);
            if (mend && valid) {
              // what the mender took out of the keys that this query sees
              const int limit = min(it.prefix + it.q0[x] + r, it.keys - 1);
              for (int key = max(0, it.prefix + it.q0[0] + 1); key <= limit; ++key) {
                const __nv_bfloat16* v = p.kv + ((long long)(it.k_begin + key) * p.heads + it.h) * 256 + 128 + h * 16;
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                  const float f = __bfloat162float(v[c]);
                  if (!isfinite(f)) o[c] = __float_as_uint(__uint_as_float(o[c]) + f);
                }
              }
            }
            __syncwarp();  // the queries' loops are of different lengths, the next TMEM load is the warp's
            if (valid) {
#pragma unroll
              for (int c = 0; c < 16; c += 8) {
                uint4 w;
                w.x = pack_bf16x2(__uint_as_float(o[c]), __uint_as_float(o[c + 1]));
                w.y = pack_bf16x2(__uint_as_float(o[c + 2]), __uint_as_float(o[c + 3]));
                w.z = pack_bf16x2(__uint_as_float(o[c + 4]), __uint_as_float(o[c + 5]));
                w.w = pack_bf16x2(__uint_as_float(o[c + 6]), __uint_as_float(o[c + 7]));
                *reinterpret_cast<uint4*>(dst + h * 16 + c) = w;
              }
            }
          }
          ++ixo[x];
        }
      }
    }
  }  // register split

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

}  // namespace latent_prefill_detail

cudaError_t launch_latent_prefill(LatentPrefillParams p, cudaStream_t stream) {
  using namespace latent_prefill_detail;
  CUtensorMap qmap, kvmap, rmap;
  {
    const uint32_t box[3] = {64, 1, 128};
    const uint64_t heads = uint64_t(p.heads);
    const uint64_t q_dims[3] = {192, heads, uint64_t(p.total_q)}, q_strides[2] = {384, heads * 384};
    const uint64_t kv_dims[3] = {256, heads, uint64_t(p.total_k)}, kv_strides[2] = {512, heads * 512};
    const uint64_t r_dims[3] = {64, 1, uint64_t(p.total_k)}, r_strides[2] = {128, uint64_t(p.rope_stride) * 2};
    if (make_map_3d(p.q, q_dims, q_strides, box, CU_TENSOR_MAP_SWIZZLE_128B, &qmap)) return cudaErrorInvalidValue;
    if (make_map_3d(p.kv, kv_dims, kv_strides, box, CU_TENSOR_MAP_SWIZZLE_128B, &kvmap)) return cudaErrorInvalidValue;
    if (make_map_3d(p.k_rope, r_dims, r_strides, box, CU_TENSOR_MAP_SWIZZLE_128B, &rmap)) return cudaErrorInvalidValue;
  }
  static unsigned configured[kContextSlots] = {};
  cudaError_t e = once_per_context(configured, [] {
    cudaError_t r =
        cudaFuncSetAttribute(latent_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (r != cudaSuccess) return r;
    // The register split assumes exactly kLaunchRegs a thread at launch; with fewer, setmaxnreg.inc would wait for ever.
    cudaFuncAttributes fa{};
    r = cudaFuncGetAttributes(&fa, latent_prefill_kernel);
    if (r != cudaSuccess) return r;
    return fa.numRegs == kLaunchRegs ? cudaSuccess : cudaErrorInvalidKernelImage;
  });
  if (e != cudaSuccess) return e;
  // At most this many items have queries; pairs of query tiles where they fill the SMs.
  auto items = [&](long long rows) {
    const long long by_rows = p.total_q / rows + p.batch, by_batch = (p.max_q + rows - 1) / rows * p.batch;
    return (by_rows < by_batch ? by_rows : by_batch) * p.heads;
  };
  p.item_rows = items(2 * kRows) < sm_count() ? kRows : 2 * kRows;
  const long long grid = items(p.item_rows);
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, latent_prefill_kernel, p, qmap, kvmap, rmap);
}

}  // namespace nvb

extern "C" {

int nvb_latent_prefill_fwd(void* stream, const void* q, const void* kv, const void* k_rope, long long rope_stride,
                           void* out, const int* cu_q, const int* cu_k, int batch, int total_q, int total_k,
                           int max_q, int q_heads, float scale, float* lse) {
  g_last_error[0] = 0;
  if (!q || !kv || !k_rope || !out || !cu_q || !cu_k || batch < 1 || batch > 65535 || total_q < 1 || total_k < 1 ||
      max_q < 1 || q_heads < 1 || q_heads > 256)
    return fail("invalid latent prefill attention arguments");
  if ((long long)total_q * q_heads > INT_MAX) return fail("total_q * q_heads must fit in int32");
  if (rope_stride < 64 || rope_stride > INT_MAX || rope_stride % 8)
    return fail("rows of k_rope need 64 values, their stride a multiple of 8 elements");
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail("scale must be positive and finite");
  if (!aligned16(q) || !aligned16(kv) || !aligned16(k_rope) || !aligned16(out))
    return fail("q, kv, k_rope and out must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(cu_q) | reinterpret_cast<uintptr_t>(cu_k) | reinterpret_cast<uintptr_t>(lse)) & 3)
    return fail("cu_q, cu_k and lse must be 4-byte aligned");
  const long long rows = (long long)total_q * q_heads;
  const nvb::Stretch stretches[] = {{"out", out, rows * 256},
                                    {"lse", lse, rows * 4},
                                    {"q", q, rows * 384},
                                    {"kv", kv, (long long)total_k * q_heads * 512},
                                    {"k_rope", k_rope, ((total_k - 1) * rope_stride + 64) * 2},
                                    {"cu_q", cu_q, (batch + 1) * 4LL},
                                    {"cu_k", cu_k, (batch + 1) * 4LL}};
  if (int rc = nvb::check_apart(stretches, 2)) return rc;
  nvb::LatentPrefillParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.kv = static_cast<const __nv_bfloat16*>(kv);
  p.k_rope = static_cast<const __nv_bfloat16*>(k_rope);
  p.rope_stride = rope_stride;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.lse = lse;
  p.batch = batch;
  p.total_q = total_q;
  p.total_k = total_k;
  p.max_q = max_q;
  p.heads = q_heads;
  p.scale = scale;
  return cuda_status(nvb::launch_latent_prefill(p, static_cast<cudaStream_t>(stream)),
                     "latent prefill attention launch");
}

}  // extern "C"
