// Verification of drafted tokens against the target's probabilities
// (nvbe_layer_verify). No counterpart in the reference, which decodes one
// token per sequence and step.
//
// A sequence's rows are the nodes of its tree, parents first; row 0 is the
// last committed token. With P = softmax(target / T) and Q = softmax(draft /
// T) of a node, its children (tokens t, in row order) are tested in turn:
//
//   a = min(1, P(t) / Q(t)); the child with u < a is accepted, else
//   P <- max(P - Q, 0) / sum max(P - Q, 0)   (P stays where the sum is 0)
//   Q <- Q without t, renormalised
//
// which is speculative sampling with drafts drawn without replacement: the
// accepted child, or the token drawn from the P that is left when all are
// rejected, is distributed as the target's P. Without draft probabilities Q
// is 1 at the child's token. T = 0 accepts the argmax's child.
//
// Four kernels. verify_stats_kernel reads the rows of nodes that have children
// once, cut over CTAs, for their maxima and sums. What bounds it is HBM; one
// exponential per logit takes 3/4 of the MUFU rate that goes with it.
// verify_tests_kernel, a warp a node, joins a node's parts and tests its first
// child, as if the node had been reached, so that all nodes run at once. Nodes
// whose first child is rejected with a sibling behind it go on a list, and
// verify_residuals_kernel works through that: a cluster of up to 8 CTAs a node,
// one more pass over its rows (from L2 where they fit) for each further
// sibling. As many clusters as fit the GPU take the list in turn. (One kernel with a
// cluster for every node, doing all of this, took 88 us for 64 trees of 8 nodes,
// the three take 38 + 4 + 24 us: most of a node's cluster's time went on its
// start, its joins and its tests, with nothing to read.)
//
// verify_sample_kernel follows the accepted children from the root and draws
// the next token from the last node's row, cut over CTAs. A token's score is
// log P(v) plus Gumbel noise of u(v); the noise takes a SplitMix64 and two
// logarithms, ~100 instructions in all, for 152 thousand tokens a sequence. A
// token can only beat a score L if 1 - u < P(v) e^-L (as -log u >= 1 - u), so
// the hash alone sorts out nearly all tokens once L is known. The best score of
// a CTA's first 2048 tokens, of weight Z, is below log Z - 5/2 five times in
// a million (exp(-e^2.5)): with that L the ~12 tokens that are left are scored;
// if none reached L all of them are. Their best is the L of the CTA's other
// tokens. What bounds it is the issue rate: ~35 instructions a token. The CTAs'
// best meet in a 64-bit maximum (score, then the lowest token), which no
// order of arrival changes.
//
// Measured (B200; 64 trees of 8 nodes, vocabulary 151,936, draft logits): 38 +
// 4 + 24 + 31 us, 95 together, for the 188 MB that have to be read (29 us).
// The sums take 160 MB of them at 4.2 TB/s, with 1.5 waves of CTAs and 59 % of
// the issue slots; the draw uses 61 % of those. One tree of 5 nodes takes 16.6
// us: four kernels, each a chain of reads that wait for one another.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "model_internal.cuh"
#include "sample_math.cuh"

namespace nvbm {

namespace {

using namespace sample_math;

constexpr int kThreads = 256;        // of a stats and a tests CTA
constexpr int kListThreads = 256;    // of a residuals CTA
constexpr int kSampleThreads = 256;  // of a sample CTA, 8 tokens a thread and chunk
constexpr int kMaxList = 256;        // tokens of the first chunk that may reach its bound
constexpr int kMaxParts = 32;        // CTAs that read a node's rows
constexpr int kMaxCluster = 8;       // CTAs of a node on the list
constexpr int kMaxNodes = 1024;      // of one tree (verify_max_nodes)
constexpr float kLog2e = 1.4426950408889634f;
// A part's sum in its unit (verify_stats_kernel) stays below this. The join takes every part to the highest unit: a
// part whose factor is flushed to 0 there (units more than 126 binary orders apart) is less than 2^-36 of the total
// then, which is 1 at least and at most kMaxParts times this. Exponents of up to 90 are off by 4e-6 at most by the
// rounding of their product. Lower bounds cost more second passes: 64 trees of 8 nodes (151,936 logits of spread 2.5)
// take 114 us at T = 0.1 and 217 at 0.05, with 2^60 118 and 227, with no bound (and wrong sums) 111 and 208; from
// T = 0.2 on all take the same.
constexpr float kMaxUnit = 0x1p90f;

// What the first two kernels leave per row. For a node with children: its
// statistics, accepted child and count of rejected children; for a child that
// was rejected: the level that its rejection adds.
struct VerifyRow {
  float m_p, z_p, m_q;   // a logit at most kMaxUnit below the highest, and the sum of exp((l - m) / T)
  float over_q, over_p;  // child: its level (Levels)
  int winner;            // node: accepted child's place in its sequence, or -1
  int rejected;          // node: children rejected; its complement where they are not regular (Levels)
  int unused;
};

// The best of a sequence's parts; zeroed by the first kernel.
struct VerifyBest {
  unsigned long long key;  // ordered score, then inverted token; 0: none
  unsigned done;           // slices that have added theirs
  unsigned unused;
};

struct VerifyParams {
  const __nv_bfloat16* logits;
  const __nv_bfloat16* draft;  // or null
  const int* tokens;
  const int* parents;
  const float* uniforms;
  const uint64_t* seeds;
  const float* temps;
  const int* cu_q;
  int* out_tokens;  // [batch, max_q]
  int* path;        // [batch, max_q]
  int* counts;      // [batch]
  float* accept;    // [rows]
  VerifyRow* ws;    // [rows]
  VerifyBest* best;  // [batch]
  float4* part;      // [rows, kMaxParts]: (m_p, z_p, m_q, z_q), or the best logit and its token at T = 0
  int4* list;        // [1 + rows]: (count, -), then (sequence, node, first row, nodes) of those with residuals
  int rows, max_q, vocab, parts;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Pairs of FP32 in one instruction (the ALU's f32x2 forms).
__device__ __forceinline__ float2 add2(const float2& a, const float2& b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(const float2& a, const float2& b) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(const float2& a, const float2& b, const float2& c) {
  float2 d;
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "mov.b64 rc, {%6, %7};\n\tfma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// exp((l - m) / T) with c = log2(e) / T. The difference of two BF16 is exact
// in FP32 (or as good), so the argument's error is relative. NaN logits have
// no probability; an infinite one takes all of it.
__device__ __forceinline__ float weight(float l, float m, float c) {
  if (!(l == l)) return 0.0f;
  if (m == INFINITY) return l == INFINITY ? 1.0f : 0.0f;
  return m == -INFINITY ? 0.0f : ex2((l - m) * c);
}

// log2(e) / T, never 0: logits of -inf have no probability at any temperature (0 times them is NaN)
__device__ __forceinline__ float inv_temperature(float t) { return fminf(fmaxf(kLog2e / t, 1.2e-38f), 1e38f); }

// ------------------------------------------------------------- rows of logits
// A row starts at any element (odd vocabularies), so it is read in the aligned
// 16-byte groups that cover it: group g holds elements [8 g - shift, + 8).
// Elements outside the row read as -inf.
struct Row {
  const __nv_bfloat16* p;
  int shift, groups, vocab;
  __device__ __forceinline__ Row(const __nv_bfloat16* row, int vocab_)
      : p(row), shift(int(reinterpret_cast<uintptr_t>(row) >> 1) & 7), groups((vocab_ + shift + 7) >> 3),
        vocab(vocab_) {}
};

__device__ __forceinline__ uint4 load8(const __nv_bfloat16* row, int at, int vocab) {
  if (at >= 0 && at + 8 <= vocab && (reinterpret_cast<uintptr_t>(row + at) & 15) == 0)
    return __ldg(reinterpret_cast<const uint4*>(row + at));
  uint64_t lo = 0, hi = 0;  // the last element first
#pragma unroll 1
  for (int e = at + 7; e >= at; --e) {
    hi = (hi << 16) | (lo >> 48);
    lo = (lo << 16) | (e >= 0 && e < vocab ? __bfloat16_as_ushort(row[e]) : 0xff80u);
  }
  return make_uint4(uint32_t(lo), uint32_t(lo >> 32), uint32_t(hi), uint32_t(hi >> 32));
}

// Calls f(at, p's group, q's group) for a thread's groups in [g0, g1) (elements
// from `at` on). kBatch groups' loads are issued before any is worked on; groups
// that cross an end of the row, and all where q is aligned otherwise than p,
// are read element by element.
template <int kBatch, class F>
__device__ __forceinline__ void each_group(const Row& p, const __nv_bfloat16* q, int g0, int g1, int threads, F&& f) {
  const bool even = q == nullptr || ((reinterpret_cast<uintptr_t>(q) ^ reinterpret_cast<uintptr_t>(p.p)) & 15) == 0;
  const int lo = even ? max(g0, p.shift ? 1 : 0) : g1, hi = even ? min(g1, (p.vocab + p.shift) >> 3) : g1;
  const uint4* vp = reinterpret_cast<const uint4*>(p.p - p.shift);
  const uint4* vq = reinterpret_cast<const uint4*>(q ? q - p.shift : p.p - p.shift);
  for (int g = lo + int(threadIdx.x); g < hi; g += kBatch * threads) {
    uint4 a[kBatch], b[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (g + u * threads < hi) {
        a[u] = __ldg(vp + g + u * threads);
        if (q) b[u] = __ldg(vq + g + u * threads);
      }
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (g + u * threads < hi) f(8 * (g + u * threads) - p.shift, a[u], b[u]);
  }
  for (int g = g0 + int(threadIdx.x); g < g1; g += threads) {
    if (g >= lo && g < hi) {
      g += max(0, (hi - 1 - g) / threads) * threads;  // past the groups above
      continue;
    }
    const int at = 8 * g - p.shift;
    uint4 b = make_uint4(0u, 0u, 0u, 0u);
    if (q) b = load8(q, at, p.vocab);
    f(at, load8(p.p, at, p.vocab), b);
  }
}

__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// The largest of eight logits, NaN left out (NaN where all are).
__device__ __forceinline__ float max8(const uint4& v) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

// Whether one of eight logits is NaN: magnitudes above infinity's.
__device__ __forceinline__ bool has_nan(const uint4& v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  bool found = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) found |= (w[i] & 0x7fffu) > 0x7f80u || (w[i] & 0x7fff0000u) > 0x7f800000u;
  return found;
}

// (l - m) c of eight logits.
__device__ __forceinline__ void exponents8(const uint4& v, float m, float c, float2 (&x)[4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = mul2(add2(make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)),
                     make_float2(-m, -m)),
                make_float2(c, c));
}

// Weights of eight logits without NaN and with a finite maximum.
__device__ __forceinline__ void weights8(const uint4& v, float m, float c, float2 (&w)[4]) {
  exponents8(v, m, c, w);
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = make_float2(ex2(w[e].x), ex2(w[e].y));
}

// Running maximum and sum of exp((l - m) / T). NaN and infinite logits make
// the sum NaN (the caller then adds it up anew with weight()).
struct Online {
  float m = -INFINITY, z = 0.0f;
  __device__ __forceinline__ void add(const uint4& v, float c) {
    const float gm = max8(v);
    if (gm > m) {
      z = m == -INFINITY ? z : z * ex2((m - gm) * c);
      m = gm;
    }
    if (!(m > -INFINITY)) {  // nothing but -inf so far, or NaN, which max8 leaves out
      if (has_nan(v)) z = NAN;
      return;
    }
    float2 w[4];
    exponents8(v, m, c, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = make_float2(ex2(w[i].x), ex2(w[i].y));
    const float2 t = add2(add2(w[0], w[1]), add2(w[2], w[3]));
    z += t.x + t.y;
  }
};

// ----------------------------------------------------------------- joins
// op(v, lanes) joins groups of `lanes` neighbouring lanes.
__device__ __forceinline__ float lanes_max(float v, int lanes) {
  for (int off = lanes / 2; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  for (int off = lanes / 2; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  return v;
}
struct SumOp {  // two sums
  __device__ __forceinline__ float4 operator()(const float4& v, int lanes) const {
    return make_float4(lanes_sum(v.x, lanes), lanes_sum(v.y, lanes), 0.f, 0.f);
  }
};
struct MaxOp {  // two maxima, x and z
  __device__ __forceinline__ float4 operator()(const float4& v, int lanes) const {
    return make_float4(lanes_max(v.x, lanes), 0.f, lanes_max(v.z, lanes), 0.f);
  }
};
struct BestOp {  // (score, index bits)
  __device__ __forceinline__ float4 operator()(const float4& v, int lanes) const {
    float score = v.x;
    int index = __float_as_int(v.y);
    for (int off = lanes / 2; off > 0; off >>= 1) {
      const float s = __shfl_xor_sync(0xffffffffu, score, off);
      const int i = __shfl_xor_sync(0xffffffffu, index, off);
      if (better(s, i, score, index)) {
        score = s;
        index = i;
      }
    }
    return make_float4(score, __int_as_float(index), 0.f, 0.f);
  }
};
struct OnlineOp {  // (m_p, z_p, m_q, z_q)
  float c;
  // a part without a finite maximum has sum 0, or NaN to pass on
  __device__ __forceinline__ float scaled(float z, float m, float top) const {
    return m == top || m == -INFINITY ? z : z * ex2((m - top) * c);
  }
  __device__ __forceinline__ float4 operator()(const float4& v, int lanes) const {
    const float mp = lanes_max(v.x, lanes), mq = lanes_max(v.z, lanes);
    return make_float4(mp, lanes_sum(scaled(v.y, v.x, mp), lanes), mq, lanes_sum(scaled(v.w, v.z, mq), lanes));
  }
};

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
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void peer_store(const float4* p, uint32_t rank, const float4& v) {
  const uint32_t addr = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "f"(v.x), "f"(v.y), "f"(v.z),
               "f"(v.w)
               : "memory");
}

// Joins what the threads of a cluster (or of a CTA, size 1) hold; all get the
// same result. CTAs leave their parts in each other's shared memory, so nobody
// has to stay behind for a reader. Two sets of buffers: a CTA may be one
// exchange ahead of another, not two.
template <int kT>
struct Exchange {
  float4 warp[2][kT / 32];
  float4 cta[2][kMaxCluster];
};
template <int kT, class Op>
__device__ __forceinline__ float4 exchange(float4 v, const float4& none, Exchange<kT>& x, int& turn, uint32_t size,
                                           uint32_t rank, Op op) {
  constexpr int kWarps = kT / 32;
  static_assert((kWarps & (kWarps - 1)) == 0 && kWarps <= 32, "the warps' parts join in one warp's lanes");
  const int t = turn++ & 1, lane = threadIdx.x & 31;
  v = op(v, 32);
  if (lane == 0) x.warp[t][threadIdx.x >> 5] = v;
  __syncthreads();
  v = op(x.warp[t][lane & (kWarps - 1)], kWarps);
  if (size == 1) return v;
  if (threadIdx.x < size) peer_store(&x.cta[t][rank], threadIdx.x, v);
  cluster_sync();
  return op((lane & (kMaxCluster - 1)) < int(size) ? x.cta[t][lane & (kMaxCluster - 1)] : none, kMaxCluster);
}

// A node's children that were rejected, in order: what P has become. `regular`:
// every rejection left something, and where there are draft probabilities
// P(t) < Q(t) held for its token, so that t has nothing left and a Q(t) that
// goes on being subtracted changes nothing.
struct Levels {
  const int* token;      // [n]
  const float* over_q;   // [n]: 1 / Q's remaining sum, 0 where nothing is left of Q
  const float* over_p;   // [n]: 1 / sum max(P - Q, 0); 0: P stayed
  bool has_q, regular;
};

// P of eight tokens from `at` on after the first `n` rejections, in place, for
// regular levels: x holds P's weights over their sum, wq Q's weights.
__device__ __forceinline__ void remaining8(float2 (&x)[4], const float2 (&wq)[4], int at, const Levels& lv, int n) {
  for (int i = 0; i < n; ++i) {
    const float over_p = lv.over_p[i];
    if (lv.has_q) {
      const float less = -lv.over_q[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 d = fma2(make_float2(less, less), wq[e], x[e]);
        x[e] = mul2(make_float2(fmaxf(d.x, 0.0f), fmaxf(d.y, 0.0f)), make_float2(over_p, over_p));
      }
    } else {
      const int gone = lv.token[i] - at;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[e] = make_float2(2 * e == gone ? 0.0f : x[e].x * over_p, 2 * e + 1 == gone ? 0.0f : x[e].y * over_p);
    }
  }
}

// The same of one token, for any levels.
__device__ __forceinline__ float remaining(float x, float wq, int v, const Levels& lv, int n) {
  for (int i = 0; i < n; ++i) {
    if (lv.over_p[i] == 0.0f) continue;
    if (lv.has_q) {
      bool gone = false;
      for (int j = 0; j < i; ++j) gone |= lv.token[j] == v;
      x = fmaxf(x - (gone ? 0.0f : wq * lv.over_q[i]), 0.0f);
    } else if (lv.token[i] == v) {
      x = 0.0f;
    }
    x *= lv.over_p[i];
  }
  return x;
}

// CTA (part, node, sequence): the part's maximum and sum of the node's rows.
__global__ void __launch_bounds__(kThreads, 6) verify_stats_kernel(const VerifyParams p) {
  __shared__ Exchange<kThreads> s_x;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.z, node = blockIdx.y, part = blockIdx.x;
  const int begin = p.cu_q[b], next = p.cu_q[b + 1];
  const float temperature = p.temps[b];
  const int n = min(min(next, p.rows) - begin, p.max_q);
  if (node == 0 && part == 0 && threadIdx.x == 0) p.best[b] = VerifyBest{0ull, 0u, 0u};
  if (b == 0 && node == 0 && part == 0 && threadIdx.x == 0) p.list[0] = make_int4(0, 0, 0, 0);
  if (begin < 0 || node >= n) return;
  bool mine = false;
  for (int i = node + 1 + int(threadIdx.x); i < n; i += kThreads) mine |= p.parents[begin + i] == node;
  const bool inner = __syncthreads_or(mine);
  const int row = begin + node;
  if (!inner && part == 0 && threadIdx.x == 0) {
    p.ws[row].winner = -1;
    p.ws[row].rejected = 0;
  }
  if (!inner) return;
  const Row lp(p.logits + (long long)row * p.vocab, p.vocab);
  const __nv_bfloat16* lq = p.draft ? p.draft + (long long)row * p.vocab : nullptr;
  const int per = (lp.groups + p.parts - 1) / p.parts, g0 = part * per, g1 = min(g0 + per, lp.groups);
  int turn = 0;
  float4 all;
  if (!(temperature > 0.0f)) {
    float best = -INFINITY;
    int best_index = kNone;
    each_group<4>(lp, nullptr, g0, g1, kThreads, [&](int at, const uint4& v, const uint4&) {
      if (max8(v) >= best || best_index == kNone) {  // a row's first tokens may come last
        float f[8];
        unpack8(v, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int t = at + i;
          if (t >= 0 && t < p.vocab && better(f[i], t, best, best_index)) {
            best = f[i];
            best_index = t;
          }
        }
      }
    });
    all = exchange(make_float4(best, __int_as_float(best_index), 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f), s_x, turn, 1,
                   0, BestOp());
  } else {
    // Any finite logit near the maximum serves as the unit that sums are taken in: the highest of the part's first
    // groups. Where the sum shows it to be far below the maximum (or is not finite) the maxima are followed.
    const float c = inv_temperature(temperature);
    const float4 none = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
    float4 unit = none;
    if (g0 + int(threadIdx.x) < g1) {
      const int at = 8 * (g0 + int(threadIdx.x)) - lp.shift;
      unit.x = max8(load8(lp.p, at, p.vocab));
      if (lq) unit.z = max8(load8(lq, at, p.vocab));
    }
    unit = exchange(unit, none, s_x, turn, 1, 0, MaxOp());
    float2 z_p = make_float2(0.f, 0.f), z_q = z_p;
    auto sum = [&](const uint4& v, float m) {
      float2 w[4];
      weights8(v, m, c, w);
      return add2(add2(w[0], w[1]), add2(w[2], w[3]));
    };
    if (lq)
      each_group<2>(lp, lq, g0, g1, kThreads, [&](int, const uint4& vp, const uint4& vq) {
        z_p = add2(z_p, sum(vp, unit.x));
        z_q = add2(z_q, sum(vq, unit.z));
      });
    else
      each_group<4>(lp, nullptr, g0, g1, kThreads,
                    [&](int, const uint4& vp, const uint4&) { z_p = add2(z_p, sum(vp, unit.x)); });
    all = exchange(make_float4(z_p.x + z_p.y, z_q.x + z_q.y, 0.f, 0.f), none, s_x, turn, 1, 0, SumOp());
    all = make_float4(unit.x, all.x, unit.z, all.y);
    if (!(all.y < kMaxUnit) || !(all.w < kMaxUnit)) {
      Online op, oq;
      each_group<1>(lp, lq, g0, g1, kThreads, [&](int, const uint4& vp, const uint4& vq) {
        op.add(vp, c);
        if (lq) oq.add(vq, c);
      });
      all = exchange(make_float4(op.m, op.z, oq.m, oq.z), none, s_x, turn, 1, 0, OnlineOp{c});
    }
  }
  if (threadIdx.x == 0) p.part[(long long)row * kMaxParts + part] = all;
}

// A node's statistics, joined from its parts by the lanes of a warp.
__device__ __forceinline__ float4 join_parts(const VerifyParams& p, int row, float c) {
  const int lane = threadIdx.x & 31;
  return OnlineOp{c}(lane < p.parts ? p.part[(long long)row * kMaxParts + lane]
                                    : make_float4(-INFINITY, 0.f, -INFINITY, 0.f), 32);
}
// Whether a node's sums have to be taken anew: NaN or infinite logits, or none but -inf (the maxima are right).
__device__ __forceinline__ bool unsafe_sums(const float4& s, bool has_q) {
  return !(s.y == s.y) || !(s.w == s.w) || s.x == INFINITY || s.z == INFINITY || s.x == -INFINITY ||
         (has_q && s.z == -INFINITY);
}
// a = min(1, P(t) / Q(t)). Below 2^-126 a probability is 0: weights are flushed there in a unit that may lie below the
// highest logit, so what is left of smaller ones goes by the unit.
__device__ __forceinline__ float acceptance(float pt, float qt) {
  constexpr float kLeast = 0x1p-126f;
  return !(pt >= kLeast) ? 0.0f : (qt >= kLeast ? fminf(pt / qt, 1.0f) : 1.0f);
}

// A warp a node: the test of its first child, and at T = 0 of all.
__global__ void __launch_bounds__(kThreads) verify_tests_kernel(const VerifyParams p, int batch) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long at = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, b = int(at / p.max_q), node = int(at % p.max_q);
  if (b >= batch) return;
  const int begin = p.cu_q[b], next = p.cu_q[b + 1];
  const float temperature = p.temps[b];
  const int n = min(min(next, p.rows) - begin, p.max_q);
  if (begin < 0 || node >= n) return;
  const int row = begin + node;
  VerifyRow* ws = p.ws + begin;
  if (lane == 0) {  // a node that is no node's child is tested by nobody
    const int parent = p.parents[row];
    if (node == 0 || parent < 0 || parent >= node) p.accept[row] = 0.0f;
  }
  int kids = 0, first = -1;
  for (int base = node + 1; base < n; base += 32) {
    const int i = base + lane;
    const unsigned hits = __ballot_sync(0xffffffffu, i < n && p.parents[begin + i] == node);
    if (first < 0 && hits) first = base + __ffs(hits) - 1;
    kids += __popc(hits);
  }
  if (kids == 0) return;
  int winner = -1;
  if (!(temperature > 0.0f)) {
    const float4 top = BestOp()(lane < p.parts ? p.part[(long long)row * kMaxParts + lane]
                                               : make_float4(-INFINITY, __int_as_float(kNone), 0.f, 0.f), 32);
    const int best = __float_as_int(top.y) == kNone ? 0 : __float_as_int(top.y);
    for (int base = node + 1; base < n; base += 32) {
      const int i = base + lane;
      const bool child = i < n && p.parents[begin + i] == node;
      const unsigned hits = __ballot_sync(0xffffffffu, child && p.tokens[begin + i] == best);
      const int taken = winner < 0 && hits ? base + __ffs(hits) - 1 : -1;
      if (taken >= 0) winner = taken;
      if (child) p.accept[begin + i] = i == taken ? 1.0f : 0.0f;
    }
    if (lane == 0) {
      ws[node].winner = winner;
      ws[node].rejected = 0;
    }
    return;
  }
  const float c = inv_temperature(temperature);
  const int t = p.tokens[begin + first];
  const bool inside = t >= 0 && t < p.vocab;
  const float lp = inside ? __bfloat162float(p.logits[(long long)row * p.vocab + t]) : -INFINITY;
  const float lq = inside && p.draft ? __bfloat162float(p.draft[(long long)row * p.vocab + t]) : -INFINITY;
  const float u = p.uniforms[begin + first];
  const float4 stats = join_parts(p, row, c);
  const bool safe = unsafe_sums(stats, p.draft != nullptr);
  const float over_q = stats.w > 0.0f ? 1.0f / stats.w : 0.0f;
  const float a = acceptance(weight(lp, stats.x, c) * (1.0f / stats.y),
                             p.draft ? weight(lq, stats.z, c) * over_q : 1.0f);
  if (safe || (!(u < a) && kids > 1)) {
    if (lane == 0) {
      const int place = atomicAdd(&p.list[0].x, 1);
      if (place < p.rows) {
        p.list[1 + place] = make_int4(b, node, begin, n);
      } else {  // sequences that overlap: more nodes than rows
        ws[node].winner = -1;
        ws[node].rejected = 0;
      }
    }
    return;
  }
  if (u < a) {
    winner = first;
    for (int i = first + 1 + lane; i < n; i += 32)
      if (p.parents[begin + i] == node) p.accept[begin + i] = 0.0f;
  }
  if (lane == 0) {
    p.accept[begin + first] = a;
    ws[first].over_q = over_q;
    ws[first].over_p = 1.0f;  // no sibling needs the sum; the draw does without
    VerifyRow& r = ws[node];
    r.m_p = stats.x;
    r.z_p = stats.y;
    r.m_q = stats.z;
    r.winner = winner;
    // a uniform of 1 or more rejects anything: then it is not regular
    r.rejected = winner >= 0 ? 0 : (a < 1.0f || !p.draft ? 1 : ~1);
  }
}

// Clusters take the list's nodes in turn: all their children's tests.
__global__ void __launch_bounds__(kListThreads, 2) verify_residuals_kernel(const VerifyParams p) {
  __shared__ Exchange<kListThreads> s_x;
  __shared__ int s_child[kMaxNodes], s_token[kMaxNodes];
  __shared__ float s_lp[kMaxNodes], s_lq[kMaxNodes], s_u[kMaxNodes];  // children's logits and uniforms
  __shared__ float s_over_q[kMaxNodes], s_over_p[kMaxNodes];
  __shared__ int s_tested[2];  // of two children in a row: 1 accepted, 0 rejected, -1 rejected irregularly
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const uint32_t size = cluster_size(), rank = cluster_rank();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int count = min(p.list[0].x, p.rows), step = int(gridDim.x / size);
  const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
  int turn = 0;
  if (size > 1) cluster_sync();  // all have started
  for (int at = int(blockIdx.x / size); at < count; at += step) {
    const int4 entry = p.list[1 + at];
    const int b = entry.x, node = entry.y, begin = entry.z, n = entry.w, row = begin + node;
    VerifyRow* ws = p.ws + begin;
    const Row lp(p.logits + (long long)row * p.vocab, p.vocab);
    const __nv_bfloat16* lq = p.draft ? p.draft + (long long)row * p.vocab : nullptr;
    // every warp counts the children, the first one collects them
    int kids = 0;
    for (int base = node + 1; base < n; base += 32) {
      const int i = base + lane;
      const bool child = i < n && p.parents[begin + i] == node;
      const unsigned hits = __ballot_sync(0xffffffffu, child);
      if (child && warp == 0) {
        const int k = kids + __popc(hits & ((1u << lane) - 1u)), t = p.tokens[begin + i];
        const bool inside = t >= 0 && t < p.vocab;
        s_child[k] = i;
        s_token[k] = t;
        s_u[k] = p.uniforms[begin + i];
        s_lp[k] = inside ? __bfloat162float(lp.p[t]) : -INFINITY;
        s_lq[k] = inside && lq ? __bfloat162float(lq[t]) : -INFINITY;
      }
      kids += __popc(hits);
    }
    const float c = inv_temperature(p.temps[b]);
    const float4 stats = join_parts(p, row, c);
    const float m_p = stats.x, m_q = stats.z;
    float z_p = stats.y, z_q = stats.w;
    const int per = (lp.groups + int(size) - 1) / int(size), g0 = int(rank) * per, g1 = min(g0 + per, lp.groups);
    const int v0 = max(8 * g0 - lp.shift, 0), v1 = min(8 * g1 - lp.shift, p.vocab);
    const bool safe = unsafe_sums(stats, lq != nullptr);
    if (safe) {
      float2 z = make_float2(0.f, 0.f);
      for (int v = v0 + int(threadIdx.x); v < v1; v += kListThreads) {
        z.x += weight(__bfloat162float(lp.p[v]), m_p, c);
        if (lq) z.y += weight(__bfloat162float(lq[v]), m_q, c);
      }
      const float4 all = exchange(make_float4(z.x, z.y, 0.f, 0.f), none, s_x, turn, size, rank, SumOp());
      z_p = all.x;
      z_q = all.y;
    }
    const float over_z = z_p > 0.0f ? 1.0f / z_p : 0.0f;
    Levels lv{s_token, s_over_q, s_over_p, lq != nullptr, true};
    int winner = -1, rejected = 0;
    float mass = z_q;
    for (int i = 0; i < kids; ++i) {
      const bool end = i + 1 == kids;
      if (warp == 0) {  // the child's probability
        __syncwarp();
        const int t = s_token[i];
        const float wq = lq ? weight(s_lq[i], m_q, c) : 0.0f;
        const float pt = remaining(weight(s_lp[i], m_p, c) * over_z, wq, t, lv, i);
        const float over_q = mass > 0.0f ? 1.0f / mass : 0.0f;
        bool gone = false;
        for (int j = 0; j < i; ++j) gone |= s_token[j] == t;
        const float a = acceptance(pt, lq ? (gone ? 0.0f : wq * over_q) : 1.0f);
        const bool taken = s_u[i] < a;
        if (lane == 0) {
          s_over_q[i] = over_q;
          s_over_p[i] = 1.0f;  // what the pass below adds up is its inverse
          s_tested[i & 1] = taken ? 1 : (a < 1.0f || !lq ? 0 : -1);  // a uniform of 1 or more rejects anything
          if (rank == 0) p.accept[begin + s_child[i]] = a;
        }
      }
      __syncthreads();
      const int tested = s_tested[i & 1];
      if (tested > 0) {
        winner = s_child[i];
        if (rank == 0)
          for (int j = i + 1 + int(threadIdx.x); j < kids; j += kListThreads) p.accept[begin + s_child[j]] = 0.0f;
        break;
      }
      rejected = i + 1;
      lv.regular = lv.regular && tested == 0;
      const float over_q = s_over_q[i];
      float over_p = 1.0f;  // where no sibling needs the sum; the draw does without
      if (!end) {
        // what is left of P, and Q's sum without the rejected tokens (added up anew: a difference would cancel where
        // the tokens had most)
        float left = 0.0f, rest = 0.0f;
        if (lv.regular && !safe) {
          each_group<4>(lp, lq, g0, g1, kListThreads, [&](int from, const uint4& vp, const uint4& vq) {
            float2 x[4], w[4];
            weights8(vp, m_p, c, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = mul2(x[e], make_float2(over_z, over_z));
            if (lq) {
              weights8(vq, m_q, c, w);
              uint32_t gone = 0;
              for (int j = 0; j <= i; ++j) {
                const unsigned e = unsigned(s_token[j] - from);
                if (e < 8u) gone |= 1u << e;
              }
              if (gone) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  rest += (gone >> (2 * e) & 1u ? 0.0f : w[e].x) + (gone >> (2 * e + 1) & 1u ? 0.0f : w[e].y);
              } else {
                const float2 t = add2(add2(w[0], w[1]), add2(w[2], w[3]));
                rest += t.x + t.y;
              }
            }
            remaining8(x, w, from, lv, i + 1);
            const float2 t = add2(add2(x[0], x[1]), add2(x[2], x[3]));
            left += t.x + t.y;
          });
        } else {
          for (int v = v0 + int(threadIdx.x); v < v1; v += kListThreads) {
            const float wv = lq ? weight(__bfloat162float(lq[v]), m_q, c) : 0.0f;
            bool gone = false;
            for (int j = 0; j <= i; ++j) gone |= s_token[j] == v;
            rest += gone ? 0.0f : wv;
            left += remaining(weight(__bfloat162float(lp.p[v]), m_p, c) * over_z, wv, v, lv, i + 1);
          }
        }
        const float4 all = exchange(make_float4(left, rest, 0.f, 0.f), none, s_x, turn, size, rank, SumOp());
        over_p = all.x > 0.0f ? 1.0f / all.x : 0.0f;
        lv.regular = lv.regular && over_p > 0.0f;
        mass = all.y;
      }
      if (threadIdx.x == 0) {
        s_over_p[i] = over_p;
        if (rank == 0) {
          ws[s_child[i]].over_q = over_q;
          ws[s_child[i]].over_p = over_p;
        }
      }
      __syncthreads();
    }
    if (rank == 0 && threadIdx.x == 0) {
      VerifyRow& r = ws[node];
      r.m_p = m_p;
      r.z_p = z_p;
      r.m_q = m_q;
      r.winner = winner;
      r.rejected = lv.regular && !safe ? rejected : ~rejected;
    }
    __syncthreads();  // the lists above are free for the next node
  }
}

// ---------------------------------------------------------------- next token
// Scores as an integer that orders like them (-0 as 0), then the lowest token first.
__device__ __forceinline__ unsigned long long sort_key(float score, int token) {
  if (!(score == score)) return 0ull;  // NaN is never it
  const uint32_t u = __float_as_uint(__fadd_rn(score, 0.0f)), o = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (static_cast<unsigned long long>(o) << 32) | (0xffffffffu - uint32_t(token));
}
__device__ __forceinline__ float key_score(unsigned long long key) {
  const uint32_t o = uint32_t(key >> 32);
  return key ? __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o) : -INFINITY;
}
__device__ __forceinline__ unsigned long long max_key(unsigned long long a, unsigned long long b) {
  return a > b ? a : b;
}

// Joins over a sample CTA's warps; every thread gets the result.
constexpr int kSampleWarps = kSampleThreads / 32;
static_assert((kSampleWarps & (kSampleWarps - 1)) == 0, "the warps' parts join in one warp's lanes");

__device__ __forceinline__ float sample_sum(float v, float* s) {
  v = lanes_sum(v, 32);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  return lanes_sum(s[threadIdx.x & (kSampleWarps - 1)], kSampleWarps);
}
__device__ __forceinline__ float sample_max(float v, float* s) {
  v = lanes_max(v, 32);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  return lanes_max(s[threadIdx.x & (kSampleWarps - 1)], kSampleWarps);
}
__device__ __forceinline__ unsigned long long lanes_key(unsigned long long v, int lanes) {
  for (int off = lanes / 2; off > 0; off >>= 1) v = max_key(v, __shfl_xor_sync(0xffffffffu, v, off));
  return v;
}
__device__ __forceinline__ unsigned long long sample_key(unsigned long long v, unsigned long long* s) {
  v = lanes_key(v, 32);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  return lanes_key(s[threadIdx.x & (kSampleWarps - 1)], kSampleWarps);
}

// The exact score: the sampler's of a logit where nothing was rejected, else
// of a probability. Few tokens come here, so it is not inlined.
__device__ __noinline__ float exact_score(float x, float temperature, uint64_t seed, int v, bool logit) {
  if (logit) return gumbel_score(x, temperature, seed, v);
  return x > 0.0f ? logf(x) - gumbel_log(seed, v) : NAN;
}

// CTA (part, sequence): the accepted path, and the best of the part's tokens.
__global__ void __launch_bounds__(kSampleThreads, 4) verify_sample_kernel(const VerifyParams p) {
  __shared__ float s_red[kSampleWarps];
  __shared__ unsigned long long s_key[kSampleWarps];
  __shared__ int s_winner[kMaxNodes], s_path[kMaxNodes], s_token[kMaxNodes];
  __shared__ float s_over_q[kMaxNodes], s_over_p[kMaxNodes];
  __shared__ int s_list[kMaxList];        // tokens that may reach the bound
  __shared__ float2 s_list_x[kMaxList];   // their logits and probabilities
  __shared__ int s_count, s_is_last, s_listed;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int b = blockIdx.y, begin = p.cu_q[b], next = p.cu_q[b + 1];
  const float temperature = p.temps[b];
  const int n = min(min(next, p.rows) - begin, p.max_q);
  int* tokens = p.out_tokens + (long long)b * p.max_q;
  int* path = p.path + (long long)b * p.max_q;
  if (begin < 0 || n <= 0) {
    if (blockIdx.x == 0) {
      for (int i = threadIdx.x; i < p.max_q; i += kSampleThreads) tokens[i] = path[i] = -1;
      if (threadIdx.x == 0) p.counts[b] = 0;
    }
    return;
  }
  const VerifyRow* ws = p.ws + begin;
  for (int i = threadIdx.x; i < n; i += kSampleThreads) s_winner[i] = ws[i].winner;
  if (threadIdx.x == 0) s_listed = 0;
  __syncthreads();
  if (threadIdx.x == 0) {
    int at = 0, count = 1;
    s_path[0] = 0;
    while (s_winner[at] > at && s_winner[at] < n) {  // n: sequences that overlap write each other's
      at = s_winner[at];
      s_path[count++] = at;
    }
    s_count = count;
  }
  __syncthreads();
  const int count = s_count, last = s_path[count - 1], row = begin + last;
  const Row lp(p.logits + (long long)row * p.vocab, p.vocab);
  const __nv_bfloat16* lq = p.draft ? p.draft + (long long)row * p.vocab : nullptr;
  const uint64_t seed = p.seeds[row];
  const int stored = ws[last].rejected;
  const int rejected = stored < 0 ? ~stored : stored;  // see VerifyRow
  const float m_p = ws[last].m_p, z_p = ws[last].z_p, m_q = ws[last].m_q;  // of nodes with children
  // this CTA's chunks of kSampleThreads groups
  const int chunks = (lp.groups + kSampleThreads - 1) / kSampleThreads;
  int chunk = blockIdx.x;
  auto load = [&](int k, uint4& vp, uint4& vq) {
    const int g = k * kSampleThreads + int(threadIdx.x), at = 8 * g - lp.shift;
    vp = vq = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
    if (g < lp.groups) {
      vp = load8(lp.p, at, p.vocab);
      if (lq && rejected) vq = load8(lq, at, p.vocab);
    }
  };
  uint4 vp, vq;
  load(chunk, vp, vq);
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < p.max_q; i += kSampleThreads) {
      path[i] = i < count ? s_path[i] : -1;
      if (i + 1 != count) tokens[i] = i + 1 < count ? p.tokens[begin + s_path[i + 1]] : -1;
    }
    if (threadIdx.x == 0) p.counts[b] = count;
  }
  if (rejected) {
    if (threadIdx.x < 32) {  // the rejected children's levels
      int kids = 0;
      for (int base = last + 1; base < n && kids < rejected; base += 32) {
        const int i = base + threadIdx.x;
        const bool mine = i < n && p.parents[begin + i] == last;
        const unsigned hits = __ballot_sync(0xffffffffu, mine);
        const int k = kids + __popc(hits & ((1u << threadIdx.x) - 1u));
        if (mine && k < rejected) {
          s_token[k] = p.tokens[begin + i];
          s_over_q[k] = ws[i].over_q;
          s_over_p[k] = ws[i].over_p;
        }
        kids += __popc(hits);
      }
    }
    __syncthreads();
  }
  const Levels lv{s_token, s_over_q, s_over_p, lq != nullptr, stored >= 0};
  const float c = inv_temperature(temperature), over_z = z_p > 0.0f ? 1.0f / z_p : 0.0f;
  auto score = [&](float l, float prob, int v, int levels) {
    return exact_score(levels == 0 ? l : prob, temperature, seed, v, levels == 0);
  };
  unsigned long long best = 0ull;
  if (!(temperature > 0.0f)) {
    float f[8];
    for (; chunk < chunks; chunk += gridDim.x) {
      const int at = 8 * (chunk * kSampleThreads + int(threadIdx.x)) - lp.shift;
      const uint4 v = vp;
      if (chunk + int(gridDim.x) < chunks) load(chunk + gridDim.x, vp, vq);
      unpack8(v, f);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at + e >= 0 && at + e < p.vocab) best = max_key(best, sort_key(f[e], at + e));
    }
    best = sample_key(best, s_key);
  } else {
    // P where something was rejected; else weights relative to the first chunk's maximum
    float top = 0.0f;
    float2 x[4];
    auto probabilities = [&](const uint4& a, const uint4& q, int at) {
      weights8(a, rejected ? m_p : top, c, x);
      if (rejected) {
        float2 w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = mul2(x[e], make_float2(over_z, over_z));
        if (lq) weights8(q, m_q, c, w);
        remaining8(x, w, at, lv, rejected);
      }
    };
    auto pick = [&](int e) { return e & 1 ? x[e >> 1].y : x[e >> 1].x; };  // of a constant e
    // Every token of a chunk, for what the bounds do not cover (NaN and infinite logits, irregular levels).
    auto score_all = [&](int k) {
      const int from = 8 * k * kSampleThreads - lp.shift, to = min(from + 8 * kSampleThreads, p.vocab);
      for (int v = from + int(threadIdx.x); v < to; v += kSampleThreads) {
        if (v < 0) continue;
        const float l = __bfloat162float(lp.p[v]);
        float pr = 0.0f;
        if (rejected)
          pr = remaining(weight(l, m_p, c) * over_z, lq ? weight(__bfloat162float(lq[v]), m_q, c) : 0.0f, v, lv,
                         rejected);
        best = max_key(best, sort_key(score(l, pr, v, rejected), v));
      }
    };
    int at = 8 * (chunk * kSampleThreads + int(threadIdx.x)) - lp.shift;
    if (rejected == 0) top = sample_max(max8(vp), s_red);
    probabilities(vp, vq, at);
    const float2 t = add2(add2(x[0], x[1]), add2(x[2], x[3]));
    const float z = sample_sum(t.x + t.y, s_red);
    const float base = rejected == 0 ? __fdividef(top, temperature) : 0.0f;  // log of the weights' unit
    // false with NaN too
    const bool bounded = lv.regular && z > 0.0f && z < INFINITY && top > -INFINITY && top < INFINITY;
    float least = base + logf(z) - 2.5f;  // a score; with 1/1000 for the roundings of the scores
    least += 1e-3f * (1.0f + fabsf(least));
    // 1 - u < x scale, 1 - u being the inverted hash's 23 bits and a half step: the bits as the mantissa of a number
    // in [1, 2). NaN may.
    auto may = [&](uint64_t hash, float prob, float scale) {
      const uint32_t k = uint32_t(hash >> 41) ^ 0x7fffffu;
      return !(__uint_as_float(0x3f800000u | k) > fmaf(prob, scale, 1.0f));
    };
    if (bounded) {
      const float first = __fdividef(12.2f, z);  // e^2.5 and a little
      uint64_t t = uint64_t(int64_t(at)) * 0xd2b74407b1ce6e93ULL;
#pragma unroll
      for (int e = 0; e < 8; ++e, t += 0xd2b74407b1ce6e93ULL)
        if (may(splitmix64(seed ^ t), pick(e), first) && at + e >= 0 && at + e < p.vocab) {
          const int i = atomicAdd(&s_listed, 1);
          if (i < kMaxList) {
            const uint32_t word = e < 2 ? vp.x : e < 4 ? vp.y : e < 6 ? vp.z : vp.w;
            s_list[i] = at + e;
            s_list_x[i] = make_float2(__uint_as_float(e & 1 ? word & 0xffff0000u : word << 16), pick(e));
          }
        }
      __syncthreads();
      for (int i = threadIdx.x; i < min(s_listed, kMaxList); i += kSampleThreads)
        best = max_key(best, sort_key(score(s_list_x[i].x, s_list_x[i].y, s_list[i], rejected), s_list[i]));
    }
    best = sample_key(best, s_key);
    if (!bounded || s_listed > kMaxList || !(key_score(best) >= least)) {
      score_all(chunk);
      best = sample_key(best, s_key);
    }
    // The other chunks: a token is scored where it may beat the best so far.
    if (chunk + int(gridDim.x) < chunks) load(chunk + gridDim.x, vp, vq);
    while ((chunk += gridDim.x) < chunks) {
      const float l = key_score(best);
      if (!lv.regular || !(l > -INFINITY && l < INFINITY)) {
        score_all(chunk);
        continue;
      }
      at = 8 * (chunk * kSampleThreads + int(threadIdx.x)) - lp.shift;
      const uint4 v = vp;
      probabilities(vp, vq, at);
      if (chunk + int(gridDim.x) < chunks) load(chunk + gridDim.x, vp, vq);
      // e^-(best - base) and a little; no less than e^-80, as weights go up to the largest float and their product with
      // a scale that is flushed, or of a few bits, bounds nothing (a larger one only has more tokens scored)
      const float scale = __expf(fmaxf(base - l + 2e-3f * (1.0f + fabsf(l)), -80.0f));
      uint64_t t = uint64_t(int64_t(at)) * 0xd2b74407b1ce6e93ULL;
      uint32_t hits = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e, t += 0xd2b74407b1ce6e93ULL)
        hits |= may(splitmix64(seed ^ t), pick(e), scale) ? 1u << e : 0u;
      while (hits) {
        const int e = __ffs(hits) - 1;
        hits &= hits - 1;
        if (at + e < 0 || at + e >= p.vocab) continue;
        const uint32_t word = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
        float pr = pick(0);
#pragma unroll
        for (int i = 1; i < 8; ++i) pr = e == i ? pick(i) : pr;
        best = max_key(best, sort_key(score(__uint_as_float(e & 1 ? word & 0xffff0000u : word << 16), pr, at + e,
                                            rejected),
                                      at + e));
      }
    }
    best = sample_key(best, s_key);
  }
  // join the parts; the last one writes the token
  if (threadIdx.x == 0) {
    if (best) atomicMax(&p.best[b].key, best);
    __threadfence();
    s_is_last = atomicAdd(&p.best[b].done, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!s_is_last) return;
  __threadfence();
  unsigned long long key = atomicMax(&p.best[b].key, 0ull);
  // The last rejection left nothing of P: it stays what it was before it. (The sums behind the others were not 0.)
  for (int levels = rejected - 1; key == 0ull && levels >= 0; --levels) {
    best = 0ull;
    for (int v = threadIdx.x; v < p.vocab; v += kSampleThreads) {
      const float l = __bfloat162float(lp.p[v]);
      float pr = 0.0f;
      if (levels)
        pr = remaining(weight(l, m_p, c) * over_z, lq ? weight(__bfloat162float(lq[v]), m_q, c) : 0.0f, v, lv, levels);
      best = max_key(best, sort_key(score(l, pr, v, levels), v));
    }
    key = sample_key(best, s_key);
  }
  if (threadIdx.x == 0) tokens[count - 1] = key ? int(0xffffffffu - uint32_t(key)) : 0;
}

}  // namespace

int verify_max_nodes() { return kMaxNodes; }

size_t verify_workspace(int rows, int batch) {
  return size_t(rows) * (kMaxParts * sizeof(float4) + sizeof(VerifyRow)) + size_t(batch) * sizeof(VerifyBest) +
         (size_t(rows) + 1) * sizeof(int4);
}

cudaError_t launch_verify(cudaStream_t s, const void* logits, const void* draft, const int* tokens,
                          const int* parents, const float* uniforms, const uint64_t* seeds, const float* temps,
                          const int* cu_q, int* out_tokens, int* path, int* counts, float* accept, int rows, int batch,
                          int max_q, int vocab, void* ws, int sms) {
  float4* const part = static_cast<float4*>(ws);
  VerifyRow* const row = reinterpret_cast<VerifyRow*>(part + size_t(rows) * kMaxParts);
  VerifyBest* const best = reinterpret_cast<VerifyBest*>(row + rows);
  VerifyParams p{static_cast<const __nv_bfloat16*>(logits), static_cast<const __nv_bfloat16*>(draft), tokens, parents,
                 uniforms, seeds, temps, cu_q, out_tokens, path, counts, accept, row, best, part,
                 reinterpret_cast<int4*>(best + batch), rows, max_q, vocab, 1};
  // CTAs that read a node's rows: 32 thousand logits each where that fills the GPU several times over (39 us for 360
  // inner nodes of 151,936 tokens, 41 us with 16 thousand), else 4 thousand.
  const long long coarse = (vocab + 32767) / 32768;
  p.parts = int(rows * coarse >= 8LL * sms ? coarse : (vocab + 4095) / 4096);
  if (p.parts > kMaxParts) p.parts = kMaxParts;
  // Programmatic dependents: launched while the kernel before them ends; they wait for it before any global access.
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(p.parts), unsigned(max_q), unsigned(batch));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, verify_stats_kernel, p);
  if (e != cudaSuccess) return e;
  const long long nodes = (long long)max_q * batch;
  cfg.gridDim = dim3(unsigned((nodes + kThreads / 32 - 1) / (kThreads / 32)));
  e = cudaLaunchKernelEx(&cfg, verify_tests_kernel, p, batch);
  if (e != cudaSuccess) return e;
  // Clusters for the list: CTAs of 4 thousand logits or more, two an SM, so that one's tests and joins run beside the
  // other's passes (64 trees, the whole call 95 us; 512 threads with one CTA an SM and clusters of 4 98, of 8 101;
  // two of 256 in clusters of 4 104, of 2 127), a few SMs left for the clusters' placing.
  int cluster = 1;
  while (cluster < kMaxCluster && vocab >= 2 * cluster * 4096) cluster *= 2;
  long long clusters = 2LL * sms * 7 / 8 / cluster;
  clusters = clusters < 1 ? 1 : (clusters > rows ? rows : clusters);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(unsigned(clusters * cluster));
  cfg.blockDim = dim3(kListThreads);
  cfg.numAttrs = 2;
  e = cudaLaunchKernelEx(&cfg, verify_residuals_kernel, p);
  if (e != cudaSuccess) return e;
  cfg.numAttrs = 1;
  // Parts of a sequence: as many as fit the GPU at once (four CTAs an SM), at most one for each chunk. A CTA's
  // start (the path, the levels, the first bound) costs about as much as two chunks.
  const int chunks = ((vocab + 14) / 8 + kSampleThreads - 1) / kSampleThreads;
  int parts = int(4LL * sms / batch);
  parts = parts < 1 ? 1 : (parts > chunks ? chunks : parts);
  cfg.gridDim = dim3(unsigned(parts), unsigned(batch));
  cfg.blockDim = dim3(kSampleThreads);
  return cudaLaunchKernelEx(&cfg, verify_sample_kernel, p);
}

}  // namespace nvbm
