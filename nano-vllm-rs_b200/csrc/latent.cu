// Absorbed attention over the paged latent cache (nvb_paged_latent_fwd). No
// counterpart in the reference, whose models keep keys and values a head.
//
//   o_i = sum_j p_ij c_j[:512] / sum_j p_ij,  p_ij = exp(scale q_i . c_j)
//
// over the cache rows c_j (576 values) that query i sees. All heads share the
// rows, so (query, head) pairs are plain rows of one matrix: a CTA takes 64 of
// them and one range of a sequence's keys, 64 keys a tile:
//
//   S = Q C^T      tcgen05.mma M=64 N=64 K=576, both from shared memory
//   P = exp2(S * scale * log2 e - m), BF16, to shared memory
//   O^T += C^T P^T tcgen05.mma M=128 (dims) N=rows K=64 (keys), four times
//
// The second product is transposed because O with rows as TMEM lanes takes 512
// columns, all there are, whatever the rows; with dims as lanes it takes 4 x 64,
// and the scores have room beside it. A tile is loaded once and serves as K
// (K-major) and as V (MN-major) where it lies.
//
// What bounds it: HBM up to 64 rows a sequence. A tile is 73,728 bytes, 1.66 us
// of an SM's share of the copy rate (~3,150 cycles at 1.9 GHz); its products
// read 245 KB of operands from shared memory, ~1,920 cycles at 128 bytes a
// cycle. Q stays (72 KB), two tiles are in flight or in use (144 KB), so one
// CTA fills an SM.
//
// Work: all CTAs run at once and share out the tiles of the whole batch evenly,
// a CTA taking a run of them in the order of the sequences. Where a run's end
// cuts a sequence, both CTAs write their part (O^T, maxima, sums) to the
// scratch, at most two parts a CTA, and a second kernel joins them in the order
// of the parts. The plan is worked out by each CTA from the lengths on the
// device, so a captured call follows them.
//
// Roles (8 warps): warp 0 loads Q and the tiles by TMA, warp 1 issues the S
// products, warp 2 the PV products, warps 4-7 hold 16 rows each (softmax, and 32
// of each 128 dims at the end). Every wait is bounded; a timeout records an error
// code, and the CTA waits for its copies and MMAs, frees TMEM and exits.
//
// Measured (B200, copy rate 6.55 TB/s, calls back to back in a graph for seconds;
// in brackets the best of a few calls, before the power cap takes SM clock from
// 1.97 to ~1.73 GHz): 64 sequences of ~4050 keys, 64 heads 78 us (68), 3.9 TB/s
// over both kernels (4.5), a tile of the first 2,800 to 3,300 cycles once both
// stages are in use, the rate of HBM; 16 heads 65 us (61); 4 of ~32400 and 32
// heads 41; one of 500 keys 11. With several row tiles a sequence the chain
// load -> S -> softmax -> PV of two stages is the time, ~2,500 cycles a tile (128
// heads, 8 x 32000 keys: 110 us, 650 TFLOP/s; 99, 720). Tried and no faster:
// eight softmax warps, two loading threads, four more warps for the output, the
// parts joined by the last CTA to arrive (its fences and loads in a row take 6 us
// and more).
#include "latent_common.cuh"

namespace nvb {

namespace latent_detail {

using namespace latent_common;

constexpr int kLatent = 512, kWidth = 576;
// Keys up to this size (half of this GPU's L2 of 126 MB) are in L2 when another row tile reads them, whenever that is.
// Two row tiles a sequence, 8 and 40 sequences, apart and side by side: 64 MB of keys 40.5, 44.9 and 40.3, 44.7 us; 96 MB
// 49.7, 54.5 and 48.8, 53.1; 384 MB 140, 142 and 122, 130. Three, 8 sequences: 64 MB 47.0 both, 96 MB 62.0 and 60.9, 384
// MB 207 and 170. (Below it now the one, now the other is ahead, by up to 8 %, in two of 48 sizes by 11.)
constexpr int kHeldBytes = 64 << 20;
constexpr int kRows = 64;                       // rows of a CTA
constexpr int kKeys = 64;                       // keys of a tile
constexpr int kChunk = kKeys * 128;             // 64 keys (or rows) x 64 BF16, one swizzled piece
constexpr int kChunks = kWidth / 64;            // pieces of a tile: the rotated part first, then the latents
constexpr int kTileBytes = kChunks * kChunk;
constexpr int kUnits = 5;                       // a tile's barriers: the rotated piece, four pairs of latent ones
constexpr int kThreads = 256;
constexpr int kTmemCols = 512;
constexpr int kOCol = 128;                      // S at 0 and 64, O^T at 128 + 64 p

// kSFull, kSFree: one per S buffer. The rows may be a tile ahead of the S issuer's look at kSFree, so the arrivals of two
// tiles in a row must not meet in one barrier.
enum Bar { kFull = 0, kEmpty = kFull + 2 * kUnits, kSFull = kEmpty + 2 * kUnits, kSFree = kSFull + 2,
           kPFull = kSFree + 2, kPVDone, kQFree, kOFree, kSDrain, kPVDrain, kNumBars };
constexpr int kTmemSlotOff = kNumBars * 8;
constexpr int kPlanOff = (kTmemSlotOff + 4 + 15) & ~15;   // Plan
constexpr int kScanOff = kPlanOff + 64;                   // long long [8] and int [8] of the warps' sums
constexpr int kAlphaOff = kScanOff + 128;                 // float [64]: factors of O's columns
constexpr int kHeadBytes = 1024;
static_assert(kAlphaOff + kRows * 4 <= kHeadBytes, "head layout");
constexpr int kQOff = kHeadBytes;
constexpr int kRingOff = kQOff + kChunks * kChunk;
constexpr int kPOff = kRingOff + 2 * kTileBytes;
constexpr int kSmemBytes = kPOff + kRows * kKeys * 2;
static_assert(kSmemBytes <= 232448, "per-CTA shared memory limit");

// Scratch of a CTA: two parts (O^T as [p][row / 4][dim][row % 4], then {maximum, sum} of each row) and what the
// second kernel is to join for it.
constexpr int kPartFloats = kRows * kLatent + 2 * kRows;
constexpr int kCtaFloats = 2 * kPartFloats + 16;
struct Join {
  int first_row, rows, parts, stride;  // of the output; part 0 is this CTA's second, the others every stride-th CTA's first
};

// kind::f16, FP32 accumulate, BF16 A and B.
constexpr uint32_t kIdesc = (1u << 4) | (1u << 7) | (1u << 10);
constexpr uint32_t kIdescS = kIdesc | ((uint32_t(kRows) >> 4) << 24) | ((uint32_t(kKeys) >> 3) << 17);
constexpr uint32_t kIdescPV = kIdesc | ((128u >> 4) << 24) | (1u << 15);  // A MN-major (dims contiguous), N by the rows

// 16 lanes x 64 columns: thread t has rows t / 4 (r[4 i], r[4 i + 1]) and t / 4 + 8 (r[4 i + 2], r[4 i + 3]) at
// columns 8 i + 2 (t % 4) and the next.
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : NVB_R8(0), NVB_R8(8), NVB_R8(16), NVB_R8(24)
      : "r"(taddr));
}

// Whether any of the 128 threads of the softmax warps says yes; all of them meet here.
__device__ __forceinline__ bool any_of_four_warps(bool yes) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(uint32_t(yes))
      : "memory");
  return r != 0;
}

// ---------------------------------------------------------------- plan
// A round is `share` row tiles of a sequence, each a member's of the group of
// `share` CTAs that reads the round's keys together.
//
// The batch is cut as a whole: every round has a unit for its start and one for
// each tile, and group i takes units [i * per, (i + 1) * per). (Equal ranges of
// each sequence, a CTA having one, were no faster where they fit: 64 sequences of
// ~4050 keys and 64 heads on 128 of the SMs 73.5 us, by runs 74.6; 16 heads 67.5
// and 64; all before the keys left L2 first.)
struct Sequence {
  int begin, n, len, tiles, row_tiles;
};
__device__ __forceinline__ Sequence sequence(const LatentParams& p, int b) {
  Sequence q;
  q.begin = min(max(p.cu_q[b], 0), p.total_q);
  q.n = min(max(p.cu_q[b + 1], q.begin), p.total_q) - q.begin;
  q.len = p.kv_lens[b];
  const bool valid = q.len > 0 && (long long)q.len <= (long long)p.table_stride * p.block_size;
  q.tiles = valid ? (q.len + kKeys - 1) / kKeys : 0;
  q.row_tiles = (q.n * p.heads + kRows - 1) / kRows;
  return q;
}
struct Plan {
  long long first;  // the unit that sequence b starts at
  long long u0, u1, per;
  int b, share;
  bool streams;  // L2 is to drop the keys first
};
static_assert(sizeof(Plan) <= 64, "plan's place");

struct Segment {
  int b, begin, n, len;
  int row0;     // of the sequence's rows
  int rows;     // at most 64
  int t0, t1;   // tiles; t0 = t1: write zeros
  bool whole;
  int parts;    // of the rows, where this is the first of several
};
// The segments of a CTA, in order; every role walks them by itself.
struct Walk {
  long long at;  // first unit of round `round` of sequence b
  int b, round;
  __device__ __forceinline__ explicit Walk(const Plan& plan) : at(plan.first), b(plan.b), round(0) {}
  __device__ __forceinline__ bool next(const LatentParams& p, const Plan& plan, int member, Segment& s) {
    while (b < p.batch && at < plan.u1) {
      const Sequence q = sequence(p, b);
      const int rounds = (q.row_tiles + plan.share - 1) / plan.share;
      while (round < rounds && at < plan.u1) {
        const long long start = at;
        const int tile = round * plan.share + member;
        at += q.tiles + 1;
        ++round;
        if (at <= plan.u0 || tile >= q.row_tiles) continue;
        const long long t0 = max(plan.u0 - start - 1, 0ll), t1 = min(plan.u1 - start - 1, (long long)q.tiles);
        if (q.tiles ? t1 <= t0 : start < plan.u0) continue;
        if (t0 == 0 && t1 < q.tiles) s.parts = 1 + int((q.tiles - t1 + plan.per - 1) / plan.per);
        s.b = b;
        s.begin = q.begin;
        s.n = q.n;
        s.len = q.len;
        s.row0 = tile * kRows;
        s.rows = min(kRows, q.n * p.heads - s.row0);
        s.t0 = q.tiles ? int(t0) : 0;
        s.t1 = q.tiles ? int(t1) : 0;
        s.whole = s.t0 == 0 && s.t1 == q.tiles;
        return true;
      }
      if (round < rounds) break;
      ++b;
      round = 0;
    }
    return false;
  }
};

template <class T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}

// CTAs that read a round's keys together. Row tiles of one sequence then share them in L2 whatever the batch; that costs
// CTAs where sequences have fewer row tiles than others, so it is for batches whose keys L2 does not hold (kHeldBytes).
__device__ __forceinline__ int plan_share(const LatentParams& p, long long tiles, int row_tiles, int ctas) {
  if (tiles <= p.l2_tiles || row_tiles <= 1) return 1;
  const int most = min(4, ctas), rounds = (row_tiles + most - 1) / most;
  return (row_tiles + rounds - 1) / rounds;
}
__device__ __forceinline__ long long units_of(const Sequence& q, int share) {
  return (long long)((q.row_tiles + share - 1) / share) * (q.tiles + 1);
}
__device__ __forceinline__ void plan_runs(const LatentParams& p, Plan& plan, long long total, int share, int row_tiles,
                                          int ctas) {
  const int groups = ctas / share, group = blockIdx.x / share;
  const long long each = total <= 0x7fffffff ? (unsigned(total) + groups - 1) / unsigned(groups)
                                             : (total + groups - 1) / groups;
  plan.per = max(each, (long long)p.min_units);
  plan.u0 = group < groups ? min(group * plan.per, total) : total;
  plan.u1 = min(plan.u0 + plan.per, total);
  plan.share = share;
  // Keys that one CTA reads, or two at about the same time, leave L2 first, and the parts in the scratch stay there for
  // the join: 64 sequences of ~4050 keys 74.9 -> 67.7 us, 32 of ~1000 20.8 -> 19.5, one of 32000 (16 heads) 23.8 -> 22.2.
  // By size, 8 sequences of one row tile without and with: 4 MB of keys 14.7 and 14.6 us, 16 MB 29.5 and 29.1, 96 MB 49.5
  // and 48.3, 384 MB 95.3 and 91.2; pairs of row tiles, 96 MB 50.0 and 48.8, 384 MB 126 and 122. (From a quarter of
  // l2_tiles on: below, one of 2000 keys had 11.0 and 11.2.) Three or four readers of sequences of one size gain 2 % (8 of
  // three row tiles, 192 MB: 96.1 and 94.4), of mixed sizes they drift apart and read keys again: 16 of 500 to 8000 keys,
  // 2 to 6 queries of 32 heads, 55.1 us without and 56.6 with it. So not for these.
  plan.streams = (row_tiles <= 1 || share == 2) && total > p.l2_tiles / 4;
  plan.b = p.batch;  // unless a sequence has unit u0
  plan.first = total;
}
template <class T>
__device__ __forceinline__ T warp_scan(T v, int lane) {
#pragma unroll
  for (int off = 1; off < 32; off *= 2) {
    const T o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  return v;
}

// Up to 32 x kPlanEach sequences of usual sizes: every warp works the plan out for itself, in 32 bits. This stands before
// a CTA's first load, so it has few steps that wait for one another, and few instructions to fetch for 32 sequences
// (a batch of 32: 0.4 us less than with four a lane).
// False where the sizes are too large for it.
constexpr int kPlanMost = 4;
template <int kPlanEach>
__device__ __forceinline__ bool make_plan_warp(const LatentParams& p, int ctas, Plan& plan) {
  const int lane = threadIdx.x & 31, b0 = lane * kPlanEach;
  int tiles[kPlanEach], rounds[kPlanEach];
  bool large = false;  // sizes that 32 bits might not sum
  int all = 0, most = 0;
#pragma unroll
  for (int i = 0; i < kPlanEach; ++i) {
    tiles[i] = rounds[i] = 0;
    if (b0 + i < p.batch) {
      const Sequence q = sequence(p, b0 + i);
      rounds[i] = q.row_tiles;
      tiles[i] = q.row_tiles ? q.tiles : 0;
      large |= q.row_tiles > 128 || q.tiles > 65535;
      all += min(tiles[i], 65535);
      most = max(most, q.row_tiles);
    }
  }
  if (__any_sync(0xffffffffu, large)) return false;
  all = __reduce_add_sync(0xffffffffu, all);
  most = __reduce_max_sync(0xffffffffu, most);
  const int share = plan_share(p, all, most, ctas);
  if (share > 1) {
#pragma unroll
    for (int i = 0; i < kPlanEach; ++i) rounds[i] = (rounds[i] + share - 1) / share;
  }
  int units = 0;
#pragma unroll
  for (int i = 0; i < kPlanEach; ++i) units += rounds[i] * (tiles[i] + 1);
  const int upto = warp_scan(units, lane);
  plan_runs(p, plan, __shfl_sync(0xffffffffu, upto, 31), share, most, ctas);
  const int u0 = int(plan.u0);
  const unsigned has = __ballot_sync(0xffffffffu, units && upto - units <= u0 && u0 < upto);
  if (has) {
    int at = upto - units, b = b0;
#pragma unroll
    for (int i = 0; i + 1 < kPlanEach; ++i)
      if (b == b0 + i && u0 >= at + rounds[i] * (tiles[i] + 1)) {
        at += rounds[i] * (tiles[i] + 1);
        ++b;
      }
    plan.b = __shfl_sync(0xffffffffu, b, __ffs(has) - 1);
    plan.first = __shfl_sync(0xffffffffu, at, __ffs(has) - 1);
  }
  return true;
}

// Any number of sequences: all threads together; the plan is in shared memory when it returns.
__device__ __forceinline__ void make_plan(const LatentParams& p, unsigned char* smem, int ctas) {
  constexpr int kWarps = kThreads / 32;
  Plan* plan = reinterpret_cast<Plan*>(smem + kPlanOff);
  long long* sums = reinterpret_cast<long long*>(smem + kScanOff);
  int* most = reinterpret_cast<int*>(smem + kScanOff + kWarps * 8);
  static_assert(kWarps * 12 <= 128, "the warps' sums");
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int each = (p.batch + kThreads - 1) / kThreads;
  const int b0 = min(t * each, p.batch), b1 = min(b0 + each, p.batch);
  long long tiles = 0;
  int rt = 0;
  for (int b = b0; b < b1; ++b) {
    const Sequence q = sequence(p, b);
    if (!q.row_tiles) continue;
    tiles += q.tiles;
    rt = max(rt, q.row_tiles);
  }
  tiles = warp_sum(tiles);
  rt = __reduce_max_sync(0xffffffffu, rt);
  if (lane == 0) {
    sums[warp] = tiles;
    most[warp] = rt;
  }
  __syncthreads();
  tiles = 0;
  rt = 0;
  for (int w = 0; w < kWarps; ++w) {
    tiles += sums[w];
    rt = max(rt, most[w]);
  }
  const int share = plan_share(p, tiles, rt, ctas);
  long long units = 0;
  for (int b = b0; b < b1; ++b) units += units_of(sequence(p, b), share);
  long long upto = warp_scan(units, lane);  // with this thread's
  __syncthreads();
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  long long total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) upto += sums[w];
    total += sums[w];
  }
  Plan mine;
  plan_runs(p, mine, total, share, rt, ctas);
  if (t == 0) *plan = mine;
  __syncthreads();
  if (units && upto - units <= mine.u0 && mine.u0 < upto) {
    long long at = upto - units;
    for (int b = b0; b < b1; ++b) {
      const long long here = units_of(sequence(p, b), share);
      if (mine.u0 < at + here) {
        plan->b = b;
        plan->first = at;
        break;
      }
      at += here;
    }
  }
  __syncthreads();
}

// NaN where a row of O sees a key whose value there is not finite and was taken out of the tile. The key's score is then
// an infinity or NaN: the row's sums are NaN, or its probability is 0 and the product 0 * inf, as in a tile that all rows
// see whole. One warp's lanes, a dim of each 128 a lane (`cache` begins at it); keys [first, end), those that only some
// rows see. A call, seldom made: in line its code lies between the loops and costs every segment 0.2 us of fetches.
__device__ __noinline__ void put_back(const __nv_bfloat16* cache, const int* table, int first, int end, int ctx, int row0,
                                      int rows, int num_blocks, int block_size, int heads, uint32_t taddr) {
#pragma unroll 1
  for (int d = 0; d < 4; ++d)
#pragma unroll 1
    for (int c = 0; c < rows; c += 16) {
      uint32_t o[16];
      tmem_ld16(taddr + 64 * d + c, o);
      tmem_ld_wait();
      reg_fence(o);
#pragma unroll 1
      for (int key = first; key < end; ++key) {
        const int logical = key / block_size, page = table[logical];
        if (!page_ok(page, num_blocks)) continue;
        const long long row = (long long)page * block_size + (key - logical * block_size);
        if (isfinite(__bfloat162float(cache[row * kWidth + d * 128]))) continue;
        const int from = (key - ctx) * heads - row0;  // the first row that sees it
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c + i >= from) o[i] = 0x7fffffffu;
      }
      __syncwarp();
      tmem_st16(taddr + 64 * d + c, o);
    }
  tmem_st_wait();
}

__global__ void __launch_bounds__(kThreads, 1)
    latent_kernel(const LatentParams p, const FastDiv fd_heads, const FastDiv fd_bs,
                  const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap cmap) {
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kTmemSlotOff);
  const uint32_t sbase = smem_addr(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // Set-up that needs no input runs beside the end of the kernel before this one.
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2 * kUnits; ++s) {
      mbar_init(&bars[kFull + s], 1);
      mbar_init(&bars[kEmpty + s], 1);
    }
    mbar_init(&bars[kSFull], 1);
    mbar_init(&bars[kSFull + 1], 1);
    mbar_init(&bars[kSFree], 4);
    mbar_init(&bars[kSFree + 1], 4);
    mbar_init(&bars[kPFull], 4);
    mbar_init(&bars[kPVDone], 1);
    mbar_init(&bars[kQFree], 1);
    mbar_init(&bars[kOFree], 4);
    mbar_init(&bars[kSDrain], 1);
    mbar_init(&bars[kPVDrain], 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // that kernel has completed, its writes are visible
  Plan plan;
  const bool by_warp = p.batch <= 32 ? make_plan_warp<1>(p, gridDim.x, plan)  // the same in all warps
                                     : p.batch <= 32 * kPlanMost && make_plan_warp<kPlanMost>(p, gridDim.x, plan);
  if (!by_warp) make_plan(p, smem, gridDim.x);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (!by_warp) plan = *reinterpret_cast<const Plan*>(smem + kPlanOff);
  const int member = int(blockIdx.x % unsigned(plan.share));
  float* const part = p.scratch + (long long)blockIdx.x * kCtaFloats;
  const bool aligned = (sbase & 1023u) == 0;
  if (!aligned && threadIdx.x == 0) record_error(kErrPrefillAlign);

  Walk walk(plan);
  Segment s;
  if (!aligned) {
    // nothing to join: the second kernel goes by this whatever happened here
    if (threadIdx.x == 128) *reinterpret_cast<Join*>(part + 2 * kPartFloats) = Join{0, 0, 0, 0};
  } else if (warp == 0) {
    // ---------------------------------------------------------- producer
    if (elect_one()) {
      tma_prefetch_desc(&qmap);
      tma_prefetch_desc(&cmap);
      const uint64_t first_out = policy_evict_first();
      int g = 0, seg = 0;
      bool alive = true;
      while (alive && walk.next(p, plan, member, s)) {
        if (s.t0 == s.t1) continue;
        const int* table = p.block_table + (long long)s.b * p.table_stride;
        const int q_row = s.begin * p.heads + s.row0;
        // the last S of the segment before this one has read Q
        if (seg > 0) alive = wait(&bars[kQFree], (seg - 1) & 1);
        int page = alive ? table[fd_bs.div(s.t0 * kKeys)] : -1;
        for (int t = s.t0; t < s.t1 && alive; ++t, ++g) {
          const int key0 = t * kKeys, logical = fd_bs.div(key0), stage = g & 1;
          const bool ok = page_ok(page, p.num_blocks), with_q = t == s.t0;
          const int row = ok ? page * p.block_size + (key0 - logical * p.block_size) : 0;
          const uint32_t tile = sbase + kRingOff + stage * kTileBytes, full0 = sbase + (kFull + stage * kUnits) * 8;
#pragma unroll
          for (int u = 0; u < kUnits; ++u) {
            if (g >= 2) alive = alive && wait(&bars[kEmpty + stage * kUnits + u], ((g >> 1) + 1) & 1);
            if (!alive) break;
            constexpr int kPieces[kUnits] = {1, 2, 2, 2, 2};
            const int c0 = u == 0 ? 0 : 2 * u - 1;
            const uint32_t full = full0 + u * 8;
            expect_bytes(full, uint32_t(kPieces[u]) * kChunk * ((ok ? 1 : 0) + (with_q ? 1 : 0)));
            if (with_q) {
#pragma unroll
              for (int c = c0; c < c0 + kPieces[u]; ++c)
                tma_load_3d_at(sbase + kQOff + c * kChunk, &qmap, full, c == 0 ? kLatent : (c - 1) * 64, 0, q_row);
            }
            if (ok) {  // a bad page's keys are masked, whatever the tile holds
#pragma unroll
              for (int c = c0; c < c0 + kPieces[u]; ++c) {
                const int x = c == 0 ? kLatent : (c - 1) * 64;
                if (plan.streams)
                  tma_load_3d_at(tile + c * kChunk, &cmap, full, x, 0, row, first_out);
                else
                  tma_load_3d_at(tile + c * kChunk, &cmap, full, x, 0, row);
              }
            }
          }
          if (!alive) break;
          if (t + 1 < s.t1) {
            const int next = fd_bs.div(key0 + kKeys);
            if (next != logical) page = table[next];
          }
        }
        ++seg;
      }
      // Every copy has landed before the CTA may exit (on the normal path its readers have waited for it).
      for (int i = max(0, g - 2); i < g; ++i)
        for (int u = 0; u < kUnits; ++u)
          if (!wait(&bars[kFull + (i & 1) * kUnits + u], (i >> 1) & 1)) break;
    }
  } else if (warp == 1) {
    // ------------------------------------------------------ S MMA issuer
    if (elect_one()) {
      const uint64_t qd = sw128_desc(sbase + kQOff, 16, 1024), kd = sw128_desc(sbase + kRingOff, 16, 1024);
      const uint32_t q_lo = uint32_t(qd), q_hi = uint32_t(qd >> 32), k_lo = uint32_t(kd), k_hi = uint32_t(kd >> 32);
      int g = 0;
      bool alive = true;
      while (alive && walk.next(p, plan, member, s)) {
        for (int t = s.t0; t < s.t1 && alive; ++t, ++g) {
          const int stage = g & 1;
          const uint32_t kb = k_lo + uint32_t(stage * (kTileBytes >> 4)), sd = tmem + stage * kKeys;
          // the scores of the tile before the last have been read
          if (g >= 2) alive = wait(&bars[kSFree + stage], ((g >> 1) + 1) & 1);
#pragma unroll
          for (int u = 0; u < kUnits; ++u) {  // as the pieces land
            alive = alive && wait(&bars[kFull + stage * kUnits + u], (g >> 1) & 1);
            if (!alive) break;
            tc_fence_after();
#pragma unroll
            for (int c = u == 0 ? 0 : 2 * u - 1; c <= 2 * u; ++c)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) {
                const uint32_t off = uint32_t(c * kChunk + kk * 32) >> 4;
                umma_ss(sd, q_lo + off, q_hi, kb + off, k_hi, kIdescS, (c | kk) ? 1u : 0u);
              }
          }
          if (!alive) break;
          umma_commit(&bars[kSFull + stage]);
          umma_commit(&bars[kEmpty + stage * kUnits]);
          if (t + 1 == s.t1) umma_commit(&bars[kQFree]);
        }
      }
      // every MMA of this thread completes before TMEM is freed
      umma_commit(&bars[kSDrain]);
      wait(&bars[kSDrain], 0);
    }
  } else if (warp == 2) {
    // ----------------------------------------------------- PV MMA issuer
    // A thread of its own: S of the next tile runs beside the rows' work on this one, but a tile that has not landed yet
    // does not hold up the product that frees the place for the one after it.
    if (elect_one()) {
      const uint64_t vd = sw128_desc(sbase + kRingOff + kChunk, kChunk, 1024), pd = sw128_desc(sbase + kPOff, 16, 1024);
      const uint32_t v_lo = uint32_t(vd), v_hi = uint32_t(vd >> 32), p_lo = uint32_t(pd), p_hi = uint32_t(pd >> 32);
      int g = 0, seg = 0;
      bool alive = true;
      while (alive && walk.next(p, plan, member, s)) {
        if (s.t0 == s.t1) continue;
        const uint32_t idesc = kIdescPV | (uint32_t((s.rows + 15) / 16 * 2) << 17);
        // the output of the segment before this one has been read
        if (seg > 0) alive = wait(&bars[kOFree], (seg - 1) & 1);
        for (int t = s.t0; t < s.t1 && alive; ++t, ++g) {
          alive = wait(&bars[kPFull], g & 1);
          if (!alive) break;
          tc_fence_after();
          const int stage = g & 1;
          const uint32_t vb = v_lo + uint32_t(stage * (kTileBytes >> 4));
#pragma unroll
          for (int d = 0; d < 4; ++d) {  // 128 dims: two pieces
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // 16 keys: 2048 bytes of a piece's rows, 32 bytes of P's
              umma_ss(tmem + kOCol + 64 * d, vb + uint32_t((2 * d * kChunk + kk * 2048) >> 4), v_hi,
                      p_lo + uint32_t(kk * 2), p_hi, idesc, (t > s.t0 || kk) ? 1u : 0u);
            umma_commit(&bars[kEmpty + stage * kUnits + 1 + d]);
          }
          umma_commit(&bars[kPVDone]);
        }
        ++seg;
      }
      umma_commit(&bars[kPVDrain]);
      wait(&bars[kPVDrain], 0);
    }
  } else if (warp >= 4) {
    // ------------------------------------------- softmax, then the output
    const int quad = warp & 3;
    const uint32_t lane_base = tmem + (uint32_t(quad * 32) << 16);
    const int ra = quad * 16 + (lane >> 2), rb = ra + 8;  // this thread's rows, shared by four lanes
    float* alphas = reinterpret_cast<float*>(smem + kAlphaOff);
    const float sl2 = p.scale * kLog2e;
    int g = 0;
    // A warp whose wait gave up goes on without waiting, so that the four warps still meet at their named barriers.
    bool alive = true;
    Join join{0, 0, 0, 0};
    while (walk.next(p, plan, member, s)) {
      const long long first = (long long)s.begin * p.heads + s.row0;  // of the output's rows
      if (s.t0 == s.t1) {  // no keys
        for (int i = threadIdx.x - 128; i < s.rows * (kLatent / 8); i += 128)
          *reinterpret_cast<uint4*>(p.out + first * kLatent + i * 8) = make_uint4(0, 0, 0, 0);
        if (p.lse && threadIdx.x - 128 < s.rows) p.lse[first + threadIdx.x - 128] = -INFINITY;
        continue;
      }
      const int* table = p.block_table + (long long)s.b * p.table_stride;
      const int ctx = s.len - s.n;  // query i sees keys up to ctx + i
      const int seen = ctx + fd_heads.div(s.row0) + 1;  // keys that every row sees
      // rows behind the last one see what that sees; their results are dropped
      const int lim_a = ctx + fd_heads.div(s.row0 + min(ra, s.rows - 1)),
                lim_b = ctx + fd_heads.div(s.row0 + min(rb, s.rows - 1));
      float ma = -INFINITY, mb = -INFINITY, la = 0.0f, lb = 0.0f;
      bool taken = false;  // values that are not finite, out of keys that only some rows see
      int page = table[fd_bs.div(s.t0 * kKeys)];
      for (int t = s.t0; t < s.t1; ++t, ++g) {
        const int key0 = t * kKeys;
        const bool ok = page_ok(page, p.num_blocks);
        if (t + 1 < s.t1) page = table[fd_bs.div(key0 + kKeys)];  // a tile ahead: the load goes to L2
        const int real = ok ? min(kKeys, s.len - key0) : 0;  // keys of the sequence
        const bool plain = real == kKeys && key0 + kKeys <= seen;
        alive = alive && wait_warp(&bars[kSFull + (g & 1)], (g >> 1) & 1);
        tc_fence_after();
        uint32_t raw[32];
        tmem_ld_rows(lane_base + (g & 1) * kKeys, raw);
        tmem_ld_wait();
        reg_fence(raw);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[kSFree + (g & 1)]);
        float x[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(raw[i]);
        if (!plain) {
          const int a = min(lim_a - key0, real - 1) - 2 * (lane & 3), b = min(lim_b - key0, real - 1) - 2 * (lane & 3);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (8 * i > a) x[4 * i] = -INFINITY;
            if (8 * i + 1 > a) x[4 * i + 1] = -INFINITY;
            if (8 * i > b) x[4 * i + 2] = -INFINITY;
            if (8 * i + 1 > b) x[4 * i + 3] = -INFINITY;
          }
        }
        float ta = fmaxf(x[0], x[1]), tb = fmaxf(x[2], x[3]);
#pragma unroll
        for (int i = 1; i < 8; ++i) {
          ta = max3(ta, x[4 * i], x[4 * i + 1]);
          tb = max3(tb, x[4 * i + 2], x[4 * i + 3]);
        }
#pragma unroll
        for (int off = 1; off < 4; off *= 2) {
          ta = fmaxf(ta, __shfl_xor_sync(0xffffffffu, ta, off));
          tb = fmaxf(tb, __shfl_xor_sync(0xffffffffu, tb, off));
        }
        ta *= sl2;
        tb *= sl2;
        // The maximum in use moves only when the row's grew by more than 2^8 (or with its first key): O is seldom
        // rescaled, and P <= 2^8 divides out at the end.
        const bool grew_a = ta > ma + kRescaleLog2, grew_b = tb > mb + kRescaleLog2;
        const float fa = grew_a ? fast_exp2(ma - ta) : 1.0f, fb = grew_b ? fast_exp2(mb - tb) : 1.0f;
        ma = grew_a ? ta : ma;
        mb = grew_b ? tb : mb;
        const bool rescale = any_of_four_warps(t > s.t0 && (grew_a || grew_b));
        const float na = ma == -INFINITY ? 0.0f : -ma, nb = mb == -INFINITY ? 0.0f : -mb;
        float sa0 = 0.0f, sa1 = 0.0f, sb0 = 0.0f, sb1 = 0.0f;
        uint32_t pa[8], pb[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          fma2(x[4 * i], x[4 * i + 1], x[4 * i], x[4 * i + 1], sl2, sl2, na, na);
          fma2(x[4 * i + 2], x[4 * i + 3], x[4 * i + 2], x[4 * i + 3], sl2, sl2, nb, nb);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * i + e] = fast_exp2(x[4 * i + e]);
          add2(sa0, sa1, sa0, sa1, x[4 * i], x[4 * i + 1]);
          add2(sb0, sb1, sb0, sb1, x[4 * i + 2], x[4 * i + 3]);
          // BF16 for the tensor core (the values' type): half a step of each probability. The sum keeps FP32.
          pa[i] = pack_bf16x2(x[4 * i], x[4 * i + 1]);
          pb[i] = pack_bf16x2(x[4 * i + 2], x[4 * i + 3]);
        }
        la = la * fa + (sa0 + sa1);
        lb = lb * fb + (sb0 + sb1);
        if (rescale && (lane & 3) == 0) {
          alphas[ra] = fa;
          alphas[rb] = fb;
        }
        // the product before this one has read P and is done with O
        if (g > 0) alive = alive && wait_warp(&bars[kPVDone], (g - 1) & 1);
        unsigned char* prow = smem + kPOff + ra * 128 + (lane & 3) * 4;  // swizzled: 16-byte piece i of row r at i ^ (r % 8)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          *reinterpret_cast<uint32_t*>(prow + ((i ^ (ra & 7)) << 4)) = pa[i];
          *reinterpret_cast<uint32_t*>(prow + 1024 + ((i ^ (ra & 7)) << 4)) = pb[i];
        }
        if (rescale) {
          named_barrier(2, 128);  // the factors are there
          tc_fence_after();
#pragma unroll 1
          for (int d = 0; d < 4; ++d)
#pragma unroll 1
            for (int c = 0; c < s.rows; c += 16) {
              uint32_t o[16];
              tmem_ld16(lane_base + kOCol + 64 * d + c, o);
              tmem_ld_wait();
              reg_fence(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alphas[c + i]);
              tmem_st16(lane_base + kOCol + 64 * d + c, o);
            }
          tmem_st_wait();
        }
        if (!plain) {
          // Rows of the tile that may not meet a probability of 0: S has read them as keys, now they are values.
          unsigned char* v = smem + kRingOff + (g & 1) * kTileBytes + kChunk;
          const int me = threadIdx.x - 128;
          // 16-byte piece i of the tile's rows, 64 a row
          auto piece = [&](int i) {
            return reinterpret_cast<uint4*>(v + ((i >> 3) & 7) * kChunk + (i >> 6) * 128 + (i & 7) * 16);
          };
          for (int i = 64 * real + me; i < 64 * kKeys; i += 128) *piece(i) = make_uint4(0, 0, 0, 0);
          // What is not finite in a key that only some rows see counts for those at the end (put_back).
          for (int i = 64 * min(real, max(0, seen - key0)) + me; i < 64 * real; i += 128) {
            const uint4 w = *piece(i);
            if (nonfinite(w.x) | nonfinite(w.y) | nonfinite(w.z) | nonfinite(w.w)) {
              *piece(i) = make_uint4(finite_part(w.x), finite_part(w.y), finite_part(w.z), finite_part(w.w));
              taken = true;
            }
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[kPFull]);
      }
#pragma unroll
      for (int off = 1; off < 4; off *= 2) {
        la += __shfl_xor_sync(0xffffffffu, la, off);
        lb += __shfl_xor_sync(0xffffffffu, lb, off);
      }
      float* const mine = part + (s.t0 > 0 ? 0 : 1) * kPartFloats;
      const bool mend = any_of_four_warps(taken);  // (and nobody rescales any more)
      if ((lane & 3) == 0) {
        if (s.whole) {
          alphas[ra] = la == 0.0f ? 0.0f : 1.0f / la;  // NaN stays NaN
          alphas[rb] = lb == 0.0f ? 0.0f : 1.0f / lb;
          if (p.lse && ra < s.rows) p.lse[first + ra] = la == 0.0f ? -INFINITY : (ma + fast_log2(la)) * kLn2;
          if (p.lse && rb < s.rows) p.lse[first + rb] = lb == 0.0f ? -INFINITY : (mb + fast_log2(lb)) * kLn2;
        } else {
          float2* stats = reinterpret_cast<float2*>(mine + kRows * kLatent);
          stats[ra] = make_float2(ma, la);
          stats[rb] = make_float2(mb, lb);
        }
      }
      named_barrier(2, 128);
      alive = alive && wait_warp(&bars[kPVDone], (g - 1) & 1);
      tc_fence_after();
      const int dim = quad * 32 + lane;
      if (mend) {
        const int end = min(ctx + fd_heads.div(s.row0 + s.rows - 1) + 1, min(s.len, s.t1 * kKeys));
        put_back(p.cache + dim, table, max(max(seen, 0), s.t0 * kKeys), end, ctx, s.row0, s.rows, p.num_blocks, p.block_size,
                 p.heads, lane_base + kOCol);
      }
      // Loops kept as loops: a segment runs them once, and straight code would be fetched for it.
#pragma unroll 1
      for (int d = 0; d < 4; ++d)
#pragma unroll 1
        for (int c = 0; c < s.rows; c += 16) {
          uint32_t o[16];
          tmem_ld16(lane_base + kOCol + 64 * d + c, o);
          tmem_ld_wait();
          reg_fence(o);
          if (s.whole) {
            // Rows c + i and c + i + 1 of this dim; of the neighbour's the other one, so that a store has two dims of a row.
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const float u = __uint_as_float(o[i]) * alphas[c + i], v = __uint_as_float(o[i + 1]) * alphas[c + i + 1];
              const bool odd = lane & 1;
              const float other = __shfl_xor_sync(0xffffffffu, odd ? u : v, 1);
              const int row = c + i + (odd ? 1 : 0);
              if (row < s.rows)
                *reinterpret_cast<uint32_t*>(p.out + (first + row) * kLatent + d * 128 + (dim & ~1)) =
                    odd ? pack_bf16x2(other, v) : pack_bf16x2(u, other);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; i += 4)
              *reinterpret_cast<uint4*>(mine + ((d * 16 + (c + i) / 4) * 128 + dim) * 4) =
                  make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars[kOFree]);
      if (!s.whole && s.t0 == 0) {
        join = Join{int(first), s.rows, s.parts, plan.share};
      }
    }
    if (threadIdx.x == 128) *reinterpret_cast<Join*>(part + 2 * kPartFloats) = alive ? join : Join{0, 0, 0, 0};
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// Joins the parts of cut rows: sum over the parts s of 2^(m_s - max) O_s over
// the same sum of their row sums, in an order that goes by the parts alone.
// Every warp reads what the first kernel's CTAs left to join, and the CTAs take
// the pieces in turn. Of few parts a piece is 16 rows (of more than two: eight):
// a thread has one dim of them all. Of many it is four rows of 32 dims, and
// sixteen groups of 32 threads share the parts out. A warp a row works out the
// parts' factors while the first values are on their way. What bounds it is
// round trips to L2, so a piece has as many values in flight as the registers
// hold.
constexpr int kJoinThreads = 512, kJoinWarps = kJoinThreads / 32;
constexpr int kFewParts = 16, kManyDims = 32;
constexpr int kItemsEach = 5, kMaxCtas = 32 * kItemsEach;
__device__ __forceinline__ int piece_rows(int parts) { return parts <= 2 ? 16 : (parts <= kFewParts ? 8 : 4); }

// (A row without a seen key in a part has zeros there: probabilities of 0 and values that are finite.)
__device__ __forceinline__ void add_part(float4& a, const float4& f, const float4& v) {
  a.x = fmaf(f.x, v.x, a.x);
  a.y = fmaf(f.y, v.y, a.y);
  a.z = fmaf(f.z, v.z, a.z);
  a.w = fmaf(f.w, v.w, a.w);
}

// Few parts, kQuads x 4 rows from row0 on, kBatch parts in flight.
template <int kQuads, int kBatch, class Part, class Factors>
__device__ __forceinline__ void join_few(const LatentParams& p, const Join& j, int row0, const float4* factor4, Part part,
                                         Factors factors) {
  const int t = threadIdx.x, d = t >> 7, dim = t & 127;
  const int place = ((d * 16 + row0 / 4) * 128 + dim) * 4;
  float4 acc[kQuads], v[kBatch][kQuads];
  auto load = [&](int s0) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
#pragma unroll
      for (int r = 0; r < kQuads; ++r)
        v[k][r] = s0 + k < j.parts && row0 + 4 * r < j.rows
                      ? *reinterpret_cast<const float4*>(part(s0 + k) + place + r * 512)
                      : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  load(0);
  factors(4 * kQuads);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kQuads; ++r) acc[r] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < j.parts; s0 += kBatch) {
    if (s0) load(s0);
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (s0 + k < j.parts)
#pragma unroll
        for (int r = 0; r < kQuads; ++r) add_part(acc[r], factor4[(s0 + k) * kQuads + r], v[k][r]);
  }
#pragma unroll
  for (int r = 0; r < kQuads; ++r) {
    const float a[4] = {acc[r].x, acc[r].y, acc[r].z, acc[r].w};
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      // two rows of this dim; of the neighbour's the other one, so that a store has two dims of a row
      const bool odd = dim & 1;
      const float other = __shfl_xor_sync(0xffffffffu, odd ? a[i] : a[i + 1], 1);
      const int row = row0 + 4 * r + i + (odd ? 1 : 0);
      if (row < j.rows)
        *reinterpret_cast<uint32_t*>(p.out + ((long long)j.first_row + row) * kLatent + d * 128 + (dim & ~1)) =
            odd ? pack_bf16x2(other, a[i + 1]) : pack_bf16x2(a[i], other);
    }
  }
}

__global__ void __launch_bounds__(kJoinThreads, 2) latent_join_kernel(const LatentParams p, const int ctas) {
  __shared__ float4 factor4[kMaxCtas];  // [part][row of the piece]
  __shared__ float4 sums[kJoinWarps][kManyDims];
  __shared__ Join items[kMaxCtas];
  static_assert(2 * 16 <= 4 * kMaxCtas && kFewParts * 8 <= 4 * kMaxCtas && kJoinWarps >= 16, "factors: a warp a row");
  float* const factor = reinterpret_cast<float*>(factor4);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  static_assert(kMaxCtas <= kJoinThreads, "a thread an item");
  if (t < ctas) items[t] = *reinterpret_cast<const Join*>(p.scratch + (long long)t * kCtaFloats + 2 * kPartFloats);
  __syncthreads();
  int ends[kItemsEach], pieces = 0;  // of items lane, lane + 32, ...: pieces up to and with each
#pragma unroll
  for (int i = 0; i < kItemsEach; ++i) {
    int mine = 0;
    if (i * 32 + lane < ctas) {
      const Join j = items[i * 32 + lane];
      const int rows = piece_rows(j.parts);
      mine = (j.rows + rows - 1) / rows * (j.parts > kFewParts ? kLatent / kManyDims : 1);
    }
    ends[i] = pieces + warp_scan(mine, lane);
    pieces = __shfl_sync(0xffffffffu, ends[i], 31);
  }
  for (int piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
    int at = 0, before = 0;  // the item that has it: the number of those that end before it; and their pieces
#pragma unroll
    for (int i = 0; i < kItemsEach; ++i) {
      const int n = __popc(__ballot_sync(0xffffffffu, ends[i] <= piece));
      const int end = __shfl_sync(0xffffffffu, ends[i], n ? n - 1 : 0);
      if (n) {
        at = i * 32 + n;
        before = end;
      }
    }
    const Join j = items[at];
    const int within = piece - before;
    const bool few = j.parts <= kFewParts;
    const int row0 = few ? within * piece_rows(j.parts) : within / (kLatent / kManyDims) * 4;
    const float* const scratch = p.scratch + (long long)at * kCtaFloats;
    const long long step = (long long)j.stride * kCtaFloats;
    auto part = [&](int s) { return scratch + s * step + (s == 0 ? kPartFloats : 0); };
    auto factors = [&](int rows) {  // of `rows` rows, a warp each
      if (warp >= rows) return;
      auto stats = [&](int s) { return reinterpret_cast<const float2*>(part(s) + kRows * kLatent)[row0 + warp]; };
      const float2 own = lane < j.parts ? stats(lane) : make_float2(0.f, 0.f);
      float mx = own.y != 0.0f ? own.x : -INFINITY, total = 0.0f;  // a part that saw no key has no maximum
      for (int s = lane + 32; s < j.parts; s += 32) {
        const float2 ml = stats(s);
        if (ml.y != 0.0f) mx = fmaxf(mx, ml.x);
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      for (int s = lane; s < j.parts; s += 32) {
        const float2 ml = s == lane ? own : stats(s);
        // one whose scores are all NaN has none either, its sum is NaN
        const float f = ml.y == 0.0f ? 0.0f : (ml.x == -INFINITY ? NAN : fast_exp2(ml.x - mx));
        factor[s * rows + warp] = f;
        total += f * ml.y;  // NaN of a part that otherwise weighs nothing stays; the sums are not infinite
      }
      total = warp_sum(total);
      const float inv = total == 0.0f ? 0.0f : 1.0f / total;
      for (int s = lane; s < j.parts; s += 32) {
        float& f = factor[s * rows + warp];
        f = f == 0.0f ? 0.0f : f * inv;
      }
      if (lane == 0 && p.lse && row0 + warp < j.rows && (few || within % (kLatent / kManyDims) == 0))
        p.lse[j.first_row + row0 + warp] = total == 0.0f ? -INFINITY : (mx + fast_log2(total)) * kLn2;
    };
    if (j.parts <= 2) {
      join_few<4, 2>(p, j, row0, factor4, part, factors);
    } else if (few) {
      join_few<2, 4>(p, j, row0, factor4, part, factors);
    } else {
      const int dim0 = within % (kLatent / kManyDims) * kManyDims;  // of the 512
      const int place = (((dim0 >> 7) * 16 + row0 / 4) * 128 + (dim0 & 127) + lane) * 4;
      constexpr int kBatch = 8;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f), v[kBatch];
      auto load = [&](int s0) {
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const int s = s0 + k * kJoinWarps;
          v[k] = s < j.parts ? *reinterpret_cast<const float4*>(part(s) + place) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
      };
      load(warp);
      factors(4);
      __syncthreads();
      for (int s0 = warp; s0 < j.parts; s0 += kBatch * kJoinWarps) {
        if (s0 != warp) load(s0);
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
          if (s0 + k * kJoinWarps < j.parts) add_part(acc, factor4[s0 + k * kJoinWarps], v[k]);
      }
      sums[warp][lane] = acc;
      __syncthreads();
      if (t < 4 * kManyDims) {  // a row of a dim each
        const int row = t >> 5;
        float a = 0.0f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) a += reinterpret_cast<const float*>(&sums[w][lane])[row];
        const float other = __shfl_xor_sync(0xffffffffu, a, 1);
        if (!(lane & 1) && row0 + row < j.rows)
          *reinterpret_cast<uint32_t*>(p.out + ((long long)j.first_row + row0 + row) * kLatent + dim0 + lane) =
              pack_bf16x2(a, other);
      }
    }
    __syncthreads();
  }
}

}  // namespace latent_detail

cudaError_t launch_latent(LatentParams p, int ctas, cudaStream_t stream) {
  using namespace latent_detail;
  CUtensorMap qmap, cmap;
  {
    const uint64_t strides[2] = {kWidth * 2, kWidth * 2};
    const uint32_t box[3] = {64, 1, uint32_t(kKeys)};
    const uint64_t q_dims[3] = {kWidth, 1, uint64_t(p.total_q) * uint64_t(p.heads)};
    const uint64_t c_dims[3] = {kWidth, 1, uint64_t(p.num_blocks) * uint64_t(p.block_size)};
    if (make_map_3d(p.q, q_dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, &qmap)) return cudaErrorInvalidValue;
    if (make_map_3d(p.cache, c_dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, &cmap)) return cudaErrorInvalidValue;
  }
  static unsigned configured[kContextSlots] = {};
  cudaError_t e = once_per_context(configured, [] {
    cudaError_t r = cudaFuncSetAttribute(latent_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (r != cudaSuccess) return r;
    // as the first kernel has it, so that an SM need not change between them
    return cudaFuncSetAttribute(latent_join_kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                cudaSharedmemCarveoutMaxShared);
  });
  if (e != cudaSuccess) return e;
  // Runs of two units at least (one chat of 500 keys 12.5 us, with four 13.6; 2000 keys of 8 heads 12.4 and 15.2), and no
  // more CTAs than that makes of the longest sequences that the table and max_q have room for.
  p.min_units = 2;
  p.l2_tiles = kHeldBytes / kTileBytes;
  const long long rounds = ((long long)p.max_q * p.heads + kRows - 1) / kRows;
  const long long units = rounds * ((long long)p.table_stride * p.block_size / kKeys + 1);  // of one sequence, below 2^59
  if (units < (long long)ctas * p.min_units) {
    const long long runs = (units * p.batch + p.min_units - 1) / p.min_units;
    if (runs < ctas) ctas = int(runs);
  }
  // Programmatic dependents: launched while the kernel before them ends; they wait for it before any global access.
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, latent_kernel, p, FastDiv::make(p.heads), FastDiv::make(p.block_size), qmap, cmap);
  if (e != cudaSuccess || ctas == 1) return e;
  cfg.gridDim = dim3(unsigned(2 * ctas));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, latent_join_kernel, p, ctas);
}

}  // namespace nvb

extern "C" {

long long nvb_latent_scratch_floats(int num_sms) {
  return num_sms < 1 || num_sms > 1024 ? 0 : (long long)num_sms * nvb::latent_detail::kCtaFloats;
}

int nvb_paged_latent_fwd(void* stream, const void* q, const void* cache, void* out, const int* cu_q,
                         const int* kv_lens, const int* block_table, int batch, int total_q, int max_q, int q_heads,
                         int block_size, int table_stride, int num_blocks, float scale, float* lse, float* scratch,
                         long long scratch_floats) {
  g_last_error[0] = 0;
  if (!q || !cache || !out || !cu_q || !kv_lens || !block_table || batch < 1 || batch > 65535 || total_q < 1 ||
      max_q < 1 || q_heads < 1 || q_heads > 256 || block_size < 1 || table_stride < 1)
    return fail("invalid latent attention arguments");
  if (!scratch || scratch_floats < nvb_latent_scratch_floats(1) || scratch_floats > (1LL << 40))
    return fail("scratch must hold nvb_latent_scratch_floats(1) elements at least, 2^40 at most");
  if (block_size % 64) return fail("block_size must be a multiple of 64 (got %d)", block_size);
  if ((long long)block_size * table_stride > INT_MAX || (long long)total_q * q_heads > INT_MAX)
    return fail("block_size * table_stride and total_q * q_heads must fit in int32");
  if (num_blocks < 1 || (long long)num_blocks * block_size > INT_MAX)
    return fail("num_blocks must be positive and num_blocks * block_size must fit in int32");
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail("scale must be positive and finite");
  if (!aligned16(q) || !aligned16(cache) || !aligned16(out) || !aligned16(scratch))
    return fail("q, cache, out and scratch must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(cu_q) | reinterpret_cast<uintptr_t>(kv_lens) |
       reinterpret_cast<uintptr_t>(block_table) | reinterpret_cast<uintptr_t>(lse)) & 3)
    return fail("cu_q, kv_lens, block_table and lse must be 4-byte aligned");
  const long long rows = (long long)total_q * q_heads;
  const nvb::Stretch stretches[] = {{"out", out, rows * 1024},
                                    {"lse", lse, rows * 4},
                                    {"scratch", scratch, scratch_floats * 4},
                                    {"q", q, rows * 1152},
                                    {"cache", cache, (long long)num_blocks * block_size * 1152},
                                    {"cu_q", cu_q, (batch + 1) * 4LL},
                                    {"kv_lens", kv_lens, batch * 4LL},
                                    {"block_table", block_table, (long long)batch * table_stride * 4}};
  if (int rc = nvb::check_apart(stretches, 3)) return rc;
  const int sms = nvb::sm_count();
  if (sms < 1) return fail("the current device has no SM count");
  const long long fit = scratch_floats / nvb_latent_scratch_floats(1);
  nvb::LatentParams p{};
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.cache = static_cast<const __nv_bfloat16*>(cache);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.cu_q = cu_q;
  p.kv_lens = kv_lens;
  p.block_table = block_table;
  p.lse = lse;
  p.scratch = scratch;
  p.batch = batch;
  p.total_q = total_q;
  p.max_q = max_q;
  p.heads = q_heads;
  p.block_size = block_size;
  p.table_stride = table_stride;
  p.num_blocks = num_blocks;
  p.scale = scale;
  const int most = sms < nvb::latent_detail::kMaxCtas ? sms : nvb::latent_detail::kMaxCtas;
  return cuda_status(nvb::launch_latent(p, int(fit < most ? fit : most), static_cast<cudaStream_t>(stream)),
                     "latent attention launch");
}

}  // extern "C"
