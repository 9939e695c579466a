// Attention of a tree of drafted tokens over the paged K/V cache
// (nvb_paged_tree_fwd). No counterpart in the reference, which decodes one
// token per sequence and step.
//
// Query row i of a sequence is node i of its tree. The sequence's last n keys
// (n: its nodes) belong to the tree itself, the keys before them (the
// context) are visible to every node:
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(q_i k_j / sqrt(128)) over
//   j < ctx and over j = ctx + t where bit t of mask[i] is set.
//
// Tensor-core kernel: a CTA takes 128 rows of one (sequence, kv head) and one
// range of its keys. Rows pack the GQA group, row r = (node r / G, head
// r % G), so every K/V tile serves all nodes and heads of the group. Per tile
// of 64 keys
//
//   S = Q K^T   tcgen05.mma M=128 N=64 K=128, Q and K from shared memory
//   P = exp2(S * scale * log2 e - m), one thread a row, written back over S
//   O += P V    tcgen05.mma M=128 N=128 K=64, P from TMEM, V from shared memory
//
// What bounds it: HBM for trees of up to 128 rows, each K/V byte read once. A
// tile is 32 KB of K and V, 740 ns of an SM's share of HBM bandwidth (~1,350
// cycles); its MMAs take ~640 cycles (S reads 48 KB of operands, at 128 bytes
// a cycle) and its 128 x 64 exponentials 512 of the MUFU unit. S has two
// buffers, so S_j+1 is computed while the rows work on S_j, and two CTAs share
// an SM (256 TMEM columns each: S/P twice 64, O 128).
//
// Roles: warp 0 loads K and V tiles by TMA into one ring in the order of their
// use (K0 K1 V0 K2 V1 ...), warp 1 owns TMEM and issues the MMAs, warps 2-5
// hold the rows (a warp whose 32 rows are all past the last node only waits).
//
// Split keys: the CTAs of a cluster take equal ranges of a sequence's tiles.
// At the end each leaves its rows of O, their maxima and sums in its shared
// memory, and each joins every C-th row from all of them (distributed shared
// memory), so a launch of up to 8 splits writes no partials and needs no
// second kernel. More splits (few sequences, long contexts) are several
// clusters a sequence, whose joined rows go through lse_accum / out_accum.
//
// Measured (32 query and 8 KV heads, B200, copy rate 6.57 TB/s): 37 sequences
// of 8192 keys with 32 nodes each 190 us (6.56 TB/s); 64 of ~4050 keys with 32
// nodes 168 us (6.34 TB/s, launch included); 4 of ~32700 keys in 8 splits
// 91 us (5.86 TB/s: a launch has 256 CTAs, 40 of the 296 places stay empty); 1
// of 400 keys 8.6 us, where the launch, two round trips to memory and the join
// are the time.
//
// Keys that a node does not see get probability 0; their V rows must not hold
// infinities or NaN, as 0 times those is not 0. V rows of keys that nobody
// sees (behind the sequence, bad pages) are zeroed in shared memory. A tree
// key may be seen by some rows and not by others: its non-finite elements are
// zeroed too, and added at the end to the rows that see the key.
#include "prefill_common.cuh"

namespace nvb {

namespace tree_detail {

using namespace prefill_common;

constexpr int kRows = 128;              // rows of a CTA (TMEM lanes)
constexpr int kKeys = 64;               // keys of a tile
constexpr int kHalf = kKeys * 128;      // 64 rows x 64 BF16 (one swizzled half)
constexpr int kTileBytes = 2 * kHalf;   // K or V tile 64 x 128 BF16
constexpr int kQHalf = kRows * 128;     // Q: 128 rows x 64 BF16, twice
constexpr int kSlots = 5;               // ring slots shared by K and V tiles
constexpr int kThreads = 192;
constexpr int kMaxOrdered = 64;         // sequences that a launch puts in order
constexpr int kOrderedKeys = 2048;      // keys of a range from which on it does
constexpr int kMaxCluster = 8;          // CTAs that join through shared memory
constexpr int kTmemCols = 256;
constexpr int kOCol = 128;              // S/P buffers at 0 and 64
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kRescaleLog2 = 8.0f;    // the maximum in use moves when it grew by 2^8 (P <= 2^8)

// kSFull, kPFull: one per S buffer. A warp may be a tile ahead of another one,
// so the arrivals of two tiles in a row must not meet in one barrier.
enum Bar { kFull = 0, kEmpty = kFull + kSlots, kSFull = kEmpty + kSlots, kPFull = kSFull + 2,
           kPVDone = kPFull + 2, kODone, kDrain, kNumBars };
constexpr int kTmemSlotOff = kNumBars * 8;
constexpr int kFlagOff = kTmemSlotOff + 4;
constexpr int kLensOff = (kFlagOff + 4 + 15) & ~15;  // int [kMaxOrdered]: lengths, while the sequences are put in order
constexpr int kOutRow = 272;      // bytes of a row of the output in the ring
constexpr int kSumRow = 132 * 4;  // bytes of a row of O in the ring at the join: 4 banks apart from the next
constexpr int kHeadBytes = 1024;  // tiles start at the next 1 KB boundary
constexpr int kStatsOff = kHeadBytes;  // float2 [128] where Q was: a row's maximum in use and sum, for the join
constexpr int kFactorOff = kStatsOff + kRows * 8;  // float [rows of a CTA][cluster]
static_assert(kFactorOff + kRows * kMaxCluster * 4 <= kHeadBytes + 2 * kQHalf, "the join's tables fit where Q was");
static_assert(kLensOff + kMaxOrdered * 4 <= kHeadBytes, "barrier block must fit below the first 1 KB boundary");
static_assert(kRows * kSumRow <= kSlots * kTileBytes && kOutRow <= kSumRow, "the ring holds the rows of O at the join");
constexpr int kRingOff = kHeadBytes + 2 * kQHalf;
constexpr int kSmemBytes = kRingOff + kSlots * kTileBytes;  // two CTAs an SM: at most 113 KB each

// Place of tile j's K and V (of n tiles) in the order of the loads.
__device__ __forceinline__ int k_place(int j) { return j == 0 ? 0 : 2 * j - 1; }
__device__ __forceinline__ int v_place(int j, int n) { return j == n - 1 ? 2 * n - 1 : 2 * j + 2; }

// kind::f16, FP32 accumulate, BF16 A and B, M = 128, A K-major (Q) or from TMEM (P).
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 4) << 24);
constexpr uint32_t kIdescS = kIdesc | ((uint32_t(kKeys) >> 3) << 17);       // B K-major (keys)
constexpr uint32_t kIdescPV = kIdesc | ((128u >> 3) << 17) | (1u << 16);    // B MN-major (dims contiguous)

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
// Every thread of every CTA of the cluster; orders their shared memory accesses.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
  return mbar_wait(bar, parity, kErrTreeWait);
}
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait(bar, parity));
}

// Bits [t, t + 64) of a row's mask; bits outside it are 0.
__device__ __forceinline__ unsigned long long mask_window(const unsigned long long* row, int words, int t) {
  const int w = t >> 6, s = t & 63;  // t < 0 rounds down
  const unsigned long long lo = w >= 0 && w < words ? row[w] : 0ull;
  if (s == 0) return lo;
  const unsigned long long hi = w + 1 >= 0 && w + 1 < words ? row[w + 1] : 0ull;
  return (lo >> s) | (hi << (64 - s));
}

// Whether a pair of BF16 holds an infinity or NaN: an exponent of all ones carries into the sign's place.
__device__ __forceinline__ uint32_t nonfinite(uint32_t w) {
  return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}

__device__ __forceinline__ uint32_t finite_part(uint32_t w) {  // such halves as 0
  return w & ~(((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u));
}

__global__ void __launch_bounds__(kThreads, 2)
    tree_kernel(const TreeParams p, const FastDiv fd_group, const FastDiv fd_bs, const int row_tiles,
                const __nv_bfloat16* __restrict__ vcache, const __grid_constant__ CUtensorMap kmap,
                const __grid_constant__ CUtensorMap vmap) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_raw);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_raw + kTmemSlotOff);
  int* bad_v = reinterpret_cast<int*>(smem_raw + kFlagOff);
  const uint32_t raw_addr = smem_addr(smem_raw), sbase = raw_addr + kHeadBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // Splits are neighbours (a cluster's CTAs among them), then the row tiles, which read the same K and V.
  int cta = blockIdx.x;
  const int split = cta % p.num_splits;
  cta /= p.num_splits;
  const int tile = cta % row_tiles;
  cta /= row_tiles;
  const int kvhead = cta % p.kvh;
  int b = cta / p.kvh;
  const int group = p.qh / p.kvh;

  // Set-up that needs no input runs beside the end of the kernel before this one.
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(&bars[kFull + s], 1);
      mbar_init(&bars[kEmpty + s], 1);
    }
    for (int s = 0; s < 2; ++s) mbar_init(&bars[kSFull + s], 1);
    mbar_init(&bars[kPVDone], 1);
    mbar_init(&bars[kODone], 1);
    mbar_init(&bars[kDrain], 1);
    *bad_v = 0;
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // That kernel has completed, its writes are visible.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (p.by_length) {  // the b-th longest sequence (see launch_tree); equal lengths in their order
    const int t = threadIdx.x, len = t < p.batch ? p.kv_lens[t] : INT_MIN;  // after the last: behind all
    int* lens = reinterpret_cast<int*>(smem_raw + kLensOff);
    if (t < kMaxOrdered) lens[t] = len;
    __syncthreads();
    if (t < p.batch) {
      int place = 0;
      for (int u = 0; u < p.batch; u += 4) {
        const int4 o = *reinterpret_cast<const int4*>(lens + u);
        place += (o.x > len || (o.x == len && u < t)) + (o.y > len || (o.y == len && u + 1 < t)) +
                 (o.z > len || (o.z == len && u + 2 < t)) + (o.w > len || (o.w == len && u + 3 < t));
      }
      if (place == b) *bad_v = t;
    }
    __syncthreads();
    b = *bad_v;
    __syncthreads();
    if (t == 0) *bad_v = 0;
  }
  const int begin = p.cu_q[b], next = p.cu_q[b + 1], len = p.kv_lens[b];
  const int n = min(next, p.total_q) - begin, ctx = len - n;
  const int row0 = tile * kRows, rows = begin < 0 ? 0 : min(n, p.max_q) * group - row0;  // none for all of a cluster
  const bool valid = len >= n && len >= 0 && (long long)len <= (long long)p.table_stride * p.block_size;
  const int tiles_total = valid ? (len + kKeys - 1) / kKeys : 0;
  const int per_split = (tiles_total + p.num_splits - 1) / p.num_splits;
  const int t0 = split * per_split, ntiles = rows > 0 ? max(0, min(t0 + per_split, tiles_total) - t0) : 0;
  const int* table = p.block_table + (long long)b * p.table_stride;

  // This thread's row (warps 2-5): its TMEM lane, node and output place.
  const int r = (warp & 3) * 32 + lane;
  const bool row_ok = warp >= 2 && r < rows;
  const int node = fd_group.div(row_ok ? row0 + r : 0);
  const bool work = ntiles > 0 && (sbase & 1023u) == 0;
  if (ntiles > 0 && !work && threadIdx.x == 0) record_error(kErrPrefillAlign);

  const int active = (min(rows, kRows) + 31) / 32;  // warps with rows
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) mbar_init(&bars[kPFull + s], max(active, 1));
    fence_barrier_init();
  }
  // Load `place` of the ring (K or V of 64 keys from key0 on); a bad page's slot stays as it is, its keys are masked.
  auto load_tile = [&](int place, const CUtensorMap* map, int page, int logical, int key0) {
    const int slot = place % kSlots;
    if (!page_ok(page, p.num_blocks)) {
      mbar_arrive(&bars[kFull + slot]);
      return;
    }
    unsigned char* dst = smem_raw + kRingOff + slot * kTileBytes;
    const int trow = page * p.block_size + (key0 - logical * p.block_size);
    mbar_arrive_expect_tx(&bars[kFull + slot], kTileBytes);
    tma_load_3d(dst, map, &bars[kFull + slot], 0, kvhead, trow);
    tma_load_3d(dst + kHalf, map, &bars[kFull + slot], 64, kvhead, trow);
  };
  int page0 = -1;
  if (work && threadIdx.x == 0) {
    // The first K tile is on its way while the rows load Q (0.5 us of a CTA's start: 32 sequences of 128 to 1024 keys
    // 23.6 -> 22.7 us, 190 of 512 91 -> 87).
    const int logical = fd_bs.div(t0 * kKeys);
    page0 = table[logical];
    load_tile(0, &kmap, page0, logical, t0 * kKeys);
  }
  if (work && row_ok) {
    // this row of Q, K-major and 128-byte swizzled (rows past the last node stay as they are: their lanes' results
    // are dropped)
    const int head = kvhead * group + (row0 + r - node * group);
    const __nv_bfloat16* q = p.q + ((long long)(begin + node) * p.qh + head) * 128;
    uint4 w[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) w[c] = *reinterpret_cast<const uint4*>(q + c * 8);
#pragma unroll
    for (int c = 0; c < 16; ++c)
      *reinterpret_cast<uint4*>(smem_raw + kHeadBytes + (c >> 3) * kQHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
          w[c];
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The next kernel may be scheduled now: a CTA of it that takes TMEM and waits for this grid finds that all of this
  // grid's CTAs have theirs.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  float2* stats = reinterpret_cast<float2*>(smem_raw + kStatsOff);
  if (!work) {
    if (threadIdx.x < kRows) stats[threadIdx.x] = make_float2(-INFINITY, 0.0f);
  } else if (warp == 0) {
    // ---------------------------------------------------------- producer
    if (lane == 0) {
      tma_prefetch_desc(&kmap);
      tma_prefetch_desc(&vmap);
      const int final = fd_bs.div((t0 + ntiles - 1) * kKeys);
      int issued = 1, page = page0, last = fd_bs.div(t0 * kKeys);
      int ahead = last < final ? table[last + 1] : -1;  // the next page, loaded a page ahead
      int behind = page;                                // the one before: K runs a tile ahead of V
      for (int i = 1; i < 2 * ntiles; ++i) {
        const bool is_v = (i & 1) == 0 || i == 2 * ntiles - 1;
        const int j = i == 2 * ntiles - 1 ? ntiles - 1 : (is_v ? i / 2 - 1 : (i + 1) / 2);
        const int key0 = (t0 + j) * kKeys, logical = fd_bs.div(key0), slot = i % kSlots;
        if (logical > last) {
          behind = page;
          page = ahead;
          last = logical;
          ahead = logical < final ? table[logical + 1] : -1;
        }
        // released by the MMA that read the slot's last load: S of a K tile, PV of a V tile
        if (i >= kSlots && !wait(&bars[kEmpty + slot], ((i / kSlots) + 1) & 1)) break;
        load_tile(i, is_v ? &vmap : &kmap, logical == last ? page : behind, logical, key0);
        issued = i + 1;
      }
      // Every copy has landed before the CTA may exit (on the normal path its readers have waited for it).
      for (int i = max(0, issued - kSlots); i < issued; ++i)
        if (!wait(&bars[kFull + i % kSlots], (i / kSlots) & 1)) break;
    }
  } else if (warp == 1) {
    // -------------------------------------------------------- MMA issuer
    if (lane == 0) {
      const uint32_t ring = raw_addr + kRingOff;
      const uint64_t qd = sw128_desc(sbase, 16, 1024), kd = sw128_desc(ring, 16, 1024),
                     vd = sw128_desc(ring, kHalf, 1024);
      const uint32_t q_lo = uint32_t(qd), q_hi = uint32_t(qd >> 32), k_lo = uint32_t(kd), k_hi = uint32_t(kd >> 32),
                     v_lo = uint32_t(vd), v_hi = uint32_t(vd >> 32);
      bool alive = true;
      for (int j = -1; j < ntiles && alive; ++j) {
        if (j + 1 < ntiles) {  // S_j+1, beside the rows' work on S_j
          const int ki = k_place(j + 1), ks = ki % kSlots, buf = (j + 1) & 1;
          alive = wait(&bars[kFull + ks], (ki / kSlots) & 1);
          // its buffer held P_j-1: PV_j-1 must have read it
          if (alive && j >= 1) alive = wait(&bars[kPVDone], (j - 1) & 1);
          if (!alive) break;
          tc_fence_after();
          const uint32_t kb = k_lo + uint32_t(ks * (kTileBytes >> 4));
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            umma_ss(tmem + buf * kKeys, q_lo + uint32_t(((kk >> 2) * kQHalf + (kk & 3) * 32) >> 4), q_hi,
                    kb + uint32_t(((kk >> 2) * kHalf + (kk & 3) * 32) >> 4), k_hi, kIdescS, kk > 0 ? 1u : 0u);
          umma_commit(&bars[kSFull + buf]);
          umma_commit(&bars[kEmpty + ks]);
        }
        if (j < 0) continue;
        const int vi = v_place(j, ntiles), vs = vi % kSlots, buf = j & 1;
        alive = wait(&bars[kPFull + buf], (j >> 1) & 1) && wait(&bars[kFull + vs], (vi / kSlots) & 1);
        if (!alive) break;
        tc_fence_after();
        const uint32_t vb = v_lo + uint32_t(vs * (kTileBytes >> 4));
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)  // 16 keys: 8 packed columns of P, 2048 bytes of V rows
          umma_ts(tmem + kOCol, tmem + buf * kKeys + kk * 8, vb + kk * 128, v_hi, kIdescPV,
                  (j > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&bars[kPVDone]);
        umma_commit(&bars[kEmpty + vs]);
      }
      if (alive) umma_commit(&bars[kODone]);
      // every MMA completes before TMEM is freed
      umma_commit(&bars[kDrain]);
      wait(&bars[kDrain], 0);
    }
  } else if ((warp & 3) < active) {
    // ------------------------------------------------------------ softmax
    const int part = warp & 3;  // place among the warps with rows
    const uint32_t lane_base = tmem + (uint32_t(part * 32) << 16);
    const unsigned long long* mask = p.mask + (long long)(begin + node) * p.mask_words;
    const float sl2 = p.scale_log2;
    float m_used = -INFINITY, l = 0.0f;
    bool alive = true;
    // The next tile's page is loaded a tile ahead: with the shared memory taken by the tiles little is left for L1,
    // so the load goes to L2 (several hundred cycles, as long as the exponentials).
    int page = table[fd_bs.div(t0 * kKeys)];
    for (int j = 0; j < ntiles; ++j) {
      const int key0 = (t0 + j) * kKeys;
      const bool ok = page_ok(page, p.num_blocks);
      if (j + 1 < ntiles) page = table[fd_bs.div(key0 + kKeys)];
      const bool plain = ok && key0 + kKeys <= ctx;  // every row sees every key
      const int real = ok ? min(kKeys, len - key0) : 0;  // keys of the sequence
      unsigned long long seen = ~0ull;
      if (!plain) {
        const int t = key0 - ctx;
        seen = mask_window(mask, p.mask_words, t);
        if (t < 0) seen |= t > -64 ? ~0ull >> (64 + t) : ~0ull;  // context keys
        seen &= real > 0 ? ~0ull >> (64 - real) : 0ull;
      }
      if (!wait_warp(&bars[kSFull + (j & 1)], (j >> 1) & 1)) {
        alive = false;
        break;
      }
      tc_fence_after();
      const uint32_t scol = lane_base + (j & 1) * kKeys;
      float s[64];
      {
        uint32_t a0[32], a1[32];
        tmem_ld32(scol, a0);
        tmem_ld32(scol + 32, a1);
        tmem_ld_wait();
        reg_fence(a0);
        reg_fence(a1);
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          s[c] = __uint_as_float(a0[c]);
          s[32 + c] = __uint_as_float(a1[c]);
        }
      }
      if (!plain) {
        const uint32_t lo = uint32_t(seen), hi = uint32_t(seen >> 32);
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          if (!(lo >> c & 1u)) s[c] = -INFINITY;
          if (!(hi >> c & 1u)) s[32 + c] = -INFINITY;
        }
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c < 60; c += 8)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = max3(mx[i], s[c + i], s[c + 4 + i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) mx[i] = fmaxf(mx[i], s[60 + i]);
      const float m_tile = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sl2;
      // The maximum in use moves only when the row's grew by more than 2^8 (or with its first key): O is seldom
      // rescaled, and P <= 2^8 divides out at the end.
      const bool grew = m_tile > m_used + kRescaleLog2;
      const float alpha = grew ? fast_exp2(m_used - m_tile) : 1.0f;  // 0 with the first key
      m_used = grew ? m_tile : m_used;
      const float nm = m_used == -INFINITY ? 0.0f : -m_used;
      float sum[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] = 0.0f;
      uint32_t pk[32];
#pragma unroll
      for (int c = 0; c < 64; c += 2) {
        fma2(s[c], s[c + 1], s[c], s[c + 1], sl2, sl2, nm, nm);
        s[c] = fast_exp2(s[c]);
        s[c + 1] = fast_exp2(s[c + 1]);
        const int k = (c >> 1) & 3;
        add2(sum[2 * k], sum[2 * k + 1], sum[2 * k], sum[2 * k + 1], s[c], s[c + 1]);
        // BF16 for the tensor core (V's type): half a step of each probability. The sum keeps their FP32 values.
        pk[c >> 1] = pack_bf16x2(s[c], s[c + 1]);
      }
      tmem_st32(scol, pk);
      l = l * alpha + (((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7])));
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
        // PV_j-1 must be done with O (PV_j waits for this P; PV_j-2 completed before S_j was issued)
        if (!wait_warp(&bars[kPVDone], (j - 1) & 1)) {
          alive = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t o[32];
          tmem_ld32(lane_base + kOCol + 32 * h, o);
          tmem_ld_wait();
          reg_fence(o);
#pragma unroll
          for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
          tmem_st32(lane_base + kOCol + 32 * h, o);
        }
      }
      if (!plain) {
        // V rows of the tile that may not meet a probability of 0
        const int vi = v_place(j, ntiles), vs = vi % kSlots;
        if (!wait_warp(&bars[kFull + vs], (vi / kSlots) & 1)) {
          alive = false;
          break;
        }
        // 16-byte piece i of the tile's rows: the halves of a row are kHalf apart
        unsigned char* vt = smem_raw + kRingOff + vs * kTileBytes;
        auto piece = [&](int i) {
          return reinterpret_cast<uint4*>(vt + ((i >> 3) & 1) * kHalf + (i >> 4) * 128 + (i & 7) * 16);
        };
        for (int i = 16 * real + part * 32 + lane; i < 16 * kKeys; i += 32 * active) *piece(i) = make_uint4(0, 0, 0, 0);
        for (int i = 16 * max(0, ctx - key0) + part * 32 + lane; i < 16 * real; i += 32 * active) {
          const uint4 w = *piece(i);
          if (nonfinite(w.x) | nonfinite(w.y) | nonfinite(w.z) | nonfinite(w.w)) {
            *piece(i) = make_uint4(finite_part(w.x), finite_part(w.y), finite_part(w.z), finite_part(w.w));
            *bad_v = 1;
          }
        }
        fence_proxy_async_smem();
      }
      __syncwarp();  // the lanes of the loops above meet again before the warp-wide TMEM instructions
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kPFull + (j & 1)]);
    }
    // A barrier of its own: behind the last P, kPVDone may pass two phases before a slow warp looks at it.
    alive = alive && wait_warp(&bars[kODone], 0);
    tc_fence_after();
    const bool whole = p.num_splits == 1;  // no other range: this warp writes its rows itself
    const float inv = !whole ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);  // NaN stays NaN
    if (!whole) stats[r] = alive ? make_float2(m_used, l) : make_float2(-INFINITY, 0.0f);
    const bool mend = *reinterpret_cast<volatile int*>(bad_v) != 0;
    for (int h = 0; h < 4 && alive; ++h) {
      uint32_t o[32];
      tmem_ld32(lane_base + kOCol + 32 * h, o);
      tmem_ld_wait();
      reg_fence(o);
      float f[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) f[c] = __uint_as_float(o[c]) * inv;
      if (mend && row_ok) {  // what the tree keys' V rows held beside numbers
        for (int t = max(0, t0 * kKeys - ctx); t < min(n, (t0 + ntiles) * kKeys - ctx); ++t) {
          if (!(mask_window(mask, p.mask_words, t) & 1)) continue;
          const int vpage = table[fd_bs.div(ctx + t)];
          if (!page_ok(vpage, p.num_blocks)) continue;
          const __nv_bfloat16* row =
              vcache + (((long long)vpage * p.block_size + (ctx + t - fd_bs.div(ctx + t) * p.block_size)) * p.kvh +
                        kvhead) * 128 + 32 * h;
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            const float x = __bfloat162float(row[c]);
            if (!isfinite(x)) f[c] += x;
          }
        }
      }
      __syncwarp();  // the rows' loops are of different lengths, the next TMEM load is the warp's
      // into the ring, whose copies have all landed and been read
      if (whole) {
        uint4* dst = reinterpret_cast<uint4*>(smem_raw + kRingOff + r * kOutRow + h * 64);
#pragma unroll
        for (int c = 0; c < 32; c += 8)
          dst[c / 8] = make_uint4(pack_bf16x2(f[c], f[c + 1]), pack_bf16x2(f[c + 2], f[c + 3]),
                                  pack_bf16x2(f[c + 4], f[c + 5]), pack_bf16x2(f[c + 6], f[c + 7]));
      } else {
        float4* dst = reinterpret_cast<float4*>(smem_raw + kRingOff + r * kSumRow + h * 128);
#pragma unroll
        for (int c = 0; c < 32; c += 4) dst[c / 4] = make_float4(f[c], f[c + 1], f[c + 2], f[c + 3]);
      }
    }
    if (whole) {
      // 16 lanes a row, so that every store is of whole lines
      __syncwarp();
      for (int i = 0; i < 32; i += 2) {
        const int row = part * 32 + i + (lane >> 4);
        if (row >= min(rows, kRows)) break;
        const int at = fd_group.div(row0 + row);
        const long long item = (long long)(begin + at) * p.qh + kvhead * group + (row0 + row - at * group);
        const uint4 w = alive ? *reinterpret_cast<const uint4*>(smem_raw + kRingOff + row * kOutRow + (lane & 15) * 16)
                              : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(p.out + item * 128 + (lane & 15) * 8) = w;
      }
      __syncwarp();
      if (row_ok && p.lse) {
        const int head = kvhead * group + (row0 + r - node * group);
        p.lse[(long long)(begin + node) * p.qh + head] =
            !alive || l == 0.0f ? -INFINITY : (m_used + fast_log2(l)) * kLn2;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
  if (rows <= 0) return;
  if (p.num_splits == 1) {
    if (!work && row_ok) {  // no keys
      const int head = kvhead * group + (row0 + r - node * group);
      const long long item = (long long)(begin + node) * p.qh + head;
      for (int d = 0; d < 128; d += 8) *reinterpret_cast<uint4*>(p.out + item * 128 + d) = make_uint4(0, 0, 0, 0);
      if (p.lse) p.lse[item] = -INFINITY;
    }
    return;
  }

  // ---------------------------------------------------------------- join
  // Every C-th row from the cluster's C CTAs: sum_s 2^(m_s - max) O_s over the
  // same sum of their row sums. A thread works out a row's C factors, then
  // each takes four dimensions of a row.
  cluster_sync();
  const int size = int(cluster_size()), rank = int(cluster_rank());
  const int mine = (min(rows, kRows) - rank + size - 1) / size;  // rows of this CTA
  float* factor = reinterpret_cast<float*>(smem_raw + kFactorOff);
  if (int(threadIdx.x) < mine) {
    const int row = rank + size * threadIdx.x;
    float m[kMaxCluster], sum[kMaxCluster], mx = -INFINITY, total = 0.0f;
#pragma unroll
    for (int s = 0; s < kMaxCluster; ++s) {
      m[s] = -INFINITY;
      sum[s] = 0.0f;
      if (s < size)
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                     : "=f"(m[s]), "=f"(sum[s])
                     : "r"(peer_addr(raw_addr + kStatsOff + row * 8, s)));
    }
#pragma unroll
    for (int s = 0; s < kMaxCluster; ++s) mx = fmaxf(mx, sum[s] == 0.0f ? -INFINITY : m[s]);
#pragma unroll
    for (int s = 0; s < kMaxCluster; ++s) {
      // a range without a seen key has no part; one whose scores are all NaN has no maximum, its sum is NaN
      m[s] = sum[s] == 0.0f ? 0.0f : (m[s] == -INFINITY ? NAN : fast_exp2(m[s] - mx));
      total += m[s] * sum[s];
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
    for (int s = 0; s < kMaxCluster; ++s) factor[threadIdx.x * kMaxCluster + s] = m[s] == 0.0f ? 0.0f : m[s] * inv;
    const float lse = total == 0.0f ? -INFINITY : (mx + fast_log2(total)) * kLn2;
    const int at = fd_group.div(row0 + row);
    const long long item = (long long)(begin + at) * p.qh + kvhead * group + (row0 + row - at * group);
    if (p.num_splits > size)
      p.lse_accum[(long long)(split / size) * p.total_q * p.qh + item] = lse;
    else if (p.lse)
      p.lse[item] = lse;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * mine; i += kThreads) {
    const int k = i >> 5, row = rank + size * k;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f), v[kMaxCluster];
    float f[kMaxCluster];
#pragma unroll
    for (int s = 0; s < kMaxCluster; ++s) {
      f[s] = s < size ? factor[k * kMaxCluster + s] : 0.0f;
      if (f[s] != 0.0f)  // NaN too
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[s].x), "=f"(v[s].y), "=f"(v[s].z), "=f"(v[s].w)
                     : "r"(peer_addr(raw_addr + kRingOff + row * kSumRow + lane * 16, s)));
    }
#pragma unroll
    for (int s = 0; s < kMaxCluster; ++s) {
      if (f[s] == 0.0f) continue;
      acc.x = fmaf(f[s], v[s].x, acc.x);
      acc.y = fmaf(f[s], v[s].y, acc.y);
      acc.z = fmaf(f[s], v[s].z, acc.z);
      acc.w = fmaf(f[s], v[s].w, acc.w);
    }
    const int at = fd_group.div(row0 + row);
    const long long item = (long long)(begin + at) * p.qh + kvhead * group + (row0 + row - at * group);
    if (p.num_splits > size)
      *reinterpret_cast<float4*>(p.out_accum + ((long long)(split / size) * p.total_q * p.qh + item) * 128 +
                                 lane * 4) = acc;
    else
      *reinterpret_cast<uint2*>(p.out + item * 128 + lane * 4) =
          make_uint2(pack_bf16x2(acc.x, acc.y), pack_bf16x2(acc.z, acc.w));
  }
  cluster_sync();  // nobody leaves while its shared memory is read
}

// Joins the clusters' parts of each (node, head), a warp an item and a lane four
// dimensions. The LSEs and rows of eight parts are loaded together and the
// running maximum moves with them, so that an item costs one round trip to L2
// for eight parts: what bounds it is the latency of that.
constexpr int kCombineWarps = 4;
constexpr int kCombineBatch = 8;

__global__ void __launch_bounds__(kCombineWarps * 32) tree_combine_kernel(const TreeParams p, const int parts) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * kCombineWarps + (threadIdx.x >> 5);
  const long long stride = (long long)p.total_q * p.qh;
  if (item >= stride) return;
  // rows before the first sequence and behind the last have no partials and keep what they hold
  const bool live = item >= (long long)p.cu_q[0] * p.qh && item < (long long)p.cu_q[p.batch] * p.qh;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float total = 0.0f, mx = -INFINITY;
  for (int s0 = 0; s0 < parts; s0 += kCombineBatch) {
    float ls[kCombineBatch];
    float4 v[kCombineBatch];
#pragma unroll
    for (int u = 0; u < kCombineBatch; ++u) {
      ls[u] = -INFINITY;
      if (s0 + u < parts) {
        ls[u] = p.lse_accum[(s0 + u) * stride + item];
        v[u] = *reinterpret_cast<const float4*>(p.out_accum + ((s0 + u) * stride + item) * 128 + lane * 4);
      }
    }
    float m = mx;
#pragma unroll
    for (int u = 0; u < kCombineBatch; ++u) m = fmaxf(m, ls[u]);
    const float a = mx == m ? 1.0f : __expf(mx - m);  // 0 with the first split that saw a key
    mx = m;
    total *= a;
    acc.x *= a;
    acc.y *= a;
    acc.z *= a;
    acc.w *= a;
#pragma unroll
    for (int u = 0; u < kCombineBatch; ++u) {
      if (ls[u] == -INFINITY) continue;  // saw no key: its row was not written
      // a NaN score's split: the maximum passes over it, its row is NaN throughout
      const float w = isnan(ls[u]) ? NAN : __expf(ls[u] - mx);
      total += w;
      acc.x = fmaf(w, v[u].x, acc.x);
      acc.y = fmaf(w, v[u].y, acc.y);
      acc.z = fmaf(w, v[u].z, acc.z);
      acc.w = fmaf(w, v[u].w, acc.w);
    }
  }
  if (!live) return;
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  uint2 packed;
  packed.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  packed.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(p.out + item * 128 + lane * 4) = packed;
  if (lane == 0 && p.lse) p.lse[item] = total == 0.0f ? -INFINITY : mx + __logf(total);
}

// CTAs that join their ranges on chip: the largest cluster whose size divides the splits.
int tree_cluster(int num_splits) {
  int cluster = 1;
  for (int c = 2; c <= kMaxCluster; ++c)
    if (num_splits % c == 0) cluster = c;
  return cluster;
}
}  // namespace tree_detail

static int sm_count() {
  static int counts[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  int& n = counts[dev & 63];
  if (!n && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) n = 0;
  return n;
}

cudaError_t launch_tree(TreeParams p, const void* k, const void* v, int max_k, cudaStream_t stream) {
  using namespace tree_detail;
  CUtensorMap kmap, vmap;
  {
    const uint64_t dims[3] = {128, uint64_t(p.kvh), uint64_t(p.num_blocks) * uint64_t(p.block_size)};
    const uint64_t strides[2] = {256, uint64_t(p.kvh) * 256};
    const uint32_t box[3] = {64, 1, uint32_t(kKeys)};
    if (make_map_3d(k, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, &kmap)) return cudaErrorInvalidValue;
    if (make_map_3d(v, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, &vmap)) return cudaErrorInvalidValue;
  }
  static unsigned configured[kContextSlots] = {};
  cudaError_t e = once_per_context(configured, [] {
    cudaError_t r = cudaFuncSetAttribute(tree_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (r != cudaSuccess) return r;
    return cudaFuncSetAttribute(tree_kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                cudaSharedmemCarveoutMaxShared);
  });
  if (e != cudaSuccess) return e;
  const int group = p.qh / p.kvh;
  const int row_tiles = (p.max_q * group + kRows - 1) / kRows;
  const long long grid = (long long)p.batch * p.kvh * p.num_splits * row_tiles;
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  const int cluster = tree_cluster(p.num_splits);
  // Ragged batches: the longest sequences' CTAs start first and the short ones fill in behind and beside them (64
  // sequences of 16 to 8192 keys 237 -> 194 us; 16 of 500 to 8192 with 192 rows and two splits 127 -> 106). Only where
  // CTAs share an SM or wait for one, for ranges that outlast the ordering (~1 us a CTA: 190 sequences of 512 keys
  // 86 -> 99 us with it), and for at most 64 sequences (150 of 16 to 4096 keys, four CTAs one behind the other: 208 -> 216).
  p.by_length = grid > sm_count() && p.batch > 1 && p.batch <= kMaxOrdered && max_k >= p.num_splits * kOrderedKeys;
  // Programmatic dependents: launched while the kernel before them ends; they wait for it before any global access.
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, tree_kernel, p, FastDiv::make(group), FastDiv::make(p.block_size), row_tiles,
                         static_cast<const __nv_bfloat16*>(v), kmap, vmap);
  if (e != cudaSuccess || p.num_splits == cluster) return e;
  const long long items = (long long)p.total_q * p.qh;
  cfg.gridDim = dim3(unsigned((items + kCombineWarps - 1) / kCombineWarps));
  cfg.blockDim = dim3(kCombineWarps * 32);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, tree_combine_kernel, p, p.num_splits / cluster);
}

}  // namespace nvb

extern "C" {

int nvb_tree_parts(int num_splits) {
  return num_splits < 1 || num_splits > 128 ? 0 : num_splits / nvb::tree_detail::tree_cluster(num_splits);
}

int nvb_tree_num_splits(int batch, int max_q, int q_heads, int kv_heads, int max_k, int num_sms) {
  if (batch <= 0 || max_q <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || max_k <= 0 ||
      num_sms <= 0 || num_sms > 1024)
    return 0;
  const long long tiles = ((long long)max_q * (q_heads / kv_heads) + 127) / 128;  // row tiles of a kv head
  const long long work = (long long)batch * kv_heads * tiles;
  const long long fit = 2LL * num_sms / work;  // CTAs that fit at once, two an SM, for each unit of work
  // Powers of two join on chip in clusters of 8 at most. A range of less than two tiles costs more to join than to read.
  int splits = 1;
  while (2 * splits <= fit && splits < 128 && 2LL * splits * 128 <= max_k) splits *= 2;
  // The lengths of a batch are not known here. Long ranges are cut further, to 2560 keys and eight CTAs an SM at most,
  // so that a batch of different lengths does not wait for its longest (32 query and 8 KV heads: 10, 20, 32, 48 and 64
  // sequences of 500 to 32768, 32768, 8192, 8192 and 16384 keys 164 -> 66, 280 -> 89, 71 -> 49, 102 -> 78 and
  // 188 -> 114 us). Where all are of one length that costs 6 to 14 % (32 of 8192: 168 -> 177 us, 20: 135 -> 154), and
  // more the shorter the ranges (24 of 2048, two ranges: 44 -> 58).
  while (2 * splits * work <= 8LL * num_sms && 2 * splits <= nvb::tree_detail::kMaxCluster &&
         2LL * splits * 2560 <= max_k)
    splits *= 2;
  return splits;
}

int nvb_paged_tree_fwd(void* stream, const void* q, const void* k, const void* v, void* out, const int* cu_q,
                       const int* kv_lens, const int* block_table, const uint64_t* tree_mask, int mask_words,
                       int batch, int total_q, int max_q, int max_k, int q_heads, int kv_heads, int block_size,
                       int table_stride, int num_splits, float* lse, float* lse_accum, float* out_accum,
                       int num_blocks) {
  g_last_error[0] = 0;
  if (!q || !k || !v || !out || !cu_q || !kv_lens || !block_table || !tree_mask || batch <= 0 || batch > 65535 ||
      total_q < 1 || max_q < 1 || max_k < 1 || q_heads <= 0 || q_heads > 256 || kv_heads <= 0 ||
      q_heads % kv_heads || block_size <= 0 || block_size % 256 || table_stride <= 0 ||
      (long long)max_k > (long long)block_size * table_stride || (long long)block_size * table_stride > INT_MAX ||
      (long long)total_q * q_heads > INT_MAX || num_splits < 1 || num_splits > 128 ||
      (nvb_tree_parts(num_splits) > 1 && (!lse_accum || !out_accum)))
    return fail("invalid paged tree attention BF16 hdim128 arguments");
  if (mask_words < 1 || mask_words > 16 || max_q > 64 * mask_words)
    return fail("tree_mask needs a bit for each of max_q nodes in 1 to 16 words (max_q %d, %d words)", max_q,
                mask_words);
  if (num_blocks <= 0 || (long long)num_blocks * block_size > INT_MAX)
    return fail("num_blocks must be positive and num_blocks * block_size must fit in int32");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || (out_accum && !aligned16(out_accum)) ||
      (reinterpret_cast<uintptr_t>(tree_mask) & 7))
    return fail("q, k, v, out and out_accum must be 16-byte aligned, tree_mask 8-byte aligned");
  if ((reinterpret_cast<uintptr_t>(cu_q) | reinterpret_cast<uintptr_t>(kv_lens) |
       reinterpret_cast<uintptr_t>(block_table) | reinterpret_cast<uintptr_t>(lse) |
       reinterpret_cast<uintptr_t>(lse_accum)) & 3)
    return fail("cu_q, kv_lens, block_table, lse and lse_accum must be 4-byte aligned");
  TreeParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.cu_q = cu_q;
  p.kv_lens = kv_lens;
  p.block_table = block_table;
  p.mask = reinterpret_cast<const unsigned long long*>(tree_mask);
  p.lse = lse;
  p.lse_accum = lse_accum;
  p.out_accum = out_accum;
  p.batch = batch;
  p.total_q = total_q;
  p.max_q = max_q;
  p.qh = q_heads;
  p.kvh = kv_heads;
  p.block_size = block_size;
  p.table_stride = table_stride;
  p.num_blocks = num_blocks;
  p.num_splits = num_splits;
  p.mask_words = mask_words;
  p.scale_log2 = kScaleLog2;
  return cuda_status(launch_tree(p, k, v, max_k, static_cast<cudaStream_t>(stream)), "tree attention launch");
}

}  // extern "C"
