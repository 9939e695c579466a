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
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "model_internal.cuh"
#include "sample_math.cuh"

namespace nvbm {

namespace {

using namespace sample_math;

constexpr int kThreads = 512;
constexpr int kMaxNodes = 1024;  // of one tree (verify_max_nodes)
constexpr float kLog2e = 1.4426950408889634f;

// What the first kernel leaves per row. For a node with children: its
// statistics, accepted child and count of rejected children; for a child that
// was rejected: the levels that its rejection adds.
struct VerifyRow {
  float m_p, z_p, m_q, z_q;  // max logit and sum of exp((l - max) / T)
  float mass_q;              // child: Q's remaining sum (of its z_q) when it was tested
  float left;                // child: sum max(P - Q, 0) at its rejection, <= 0: P stayed
  int winner;                // node: accepted child's row in its sequence, or -1
  int rejected;              // node: children rejected
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
  int rows, max_q, vocab;
};

// exp((l - m) / T) with c = log2(e) / T. NaN logits have no probability; an
// infinite one takes all of it.
__device__ __forceinline__ float weight(float l, float m, float c) {
  if (!(l == l)) return 0.0f;
  if (m == INFINITY) return l == INFINITY ? 1.0f : 0.0f;
  return m == -INFINITY ? 0.0f : exp2f((l - m) * c);
}

__device__ __forceinline__ float inv_temperature(float t) { return fminf(kLog2e / t, 1e38f); }

__device__ __forceinline__ float block_sum(float v, float* s) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int w = 0; w < kThreads / 32; ++w) v += s[w];
  return v;
}

__device__ __forceinline__ float block_max(float v, float* s) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, off));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = -INFINITY;
  for (int w = 0; w < kThreads / 32; ++w) v = fmaxf(v, s[w]);
  return v;
}

__device__ __forceinline__ void block_best(float& score, int& index, float* s, int* si) {
  warp_best(score, index);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    s[threadIdx.x >> 5] = score;
    si[threadIdx.x >> 5] = index;
  }
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w)
    if (better(s[w], si[w], score, index)) {
      score = s[w];
      index = si[w];
    }
}

// A node's children that were rejected, in order: what P has become.
struct Levels {
  int n;                   // rejected children
  const int* token;        // [n]
  const float* mass_q;     // [n]
  const float* left;       // [n]
};

// P(v) after the first `n` rejections, from P's weight over its sum (p) and
// Q's weight (q, 1 over z_q not applied).
__device__ __forceinline__ float remaining(float p, float wq, int v, bool has_q, const Levels& lv, int n) {
  for (int i = 0; i < n; ++i) {
    if (!(lv.left[i] > 0.0f)) continue;
    if (has_q) {
      bool gone = false;
      for (int j = 0; j < i; ++j) gone |= lv.token[j] == v;
      const float q = gone || !(lv.mass_q[i] > 0.0f) ? 0.0f : wq / lv.mass_q[i];
      p = fmaxf(p - q, 0.0f);
    } else if (lv.token[i] == v) {
      p = 0.0f;
    }
    p /= lv.left[i];
  }
  return p;
}

// One CTA per node: its statistics, and its children's tests.
__global__ void __launch_bounds__(kThreads) verify_nodes_kernel(const VerifyParams p) {
  __shared__ float s_red[kThreads / 32];
  __shared__ int s_idx[kThreads / 32];
  __shared__ int s_child[kMaxNodes], s_token[kMaxNodes];
  __shared__ float s_mass[kMaxNodes], s_left[kMaxNodes];
  __shared__ int s_kids;
  const int b = blockIdx.y, node = blockIdx.x;
  const int begin = p.cu_q[b], n = min(min(p.cu_q[b + 1], p.rows) - begin, p.max_q);
  if (begin < 0 || node >= n) return;
  VerifyRow* ws = p.ws + begin;
  const int row = begin + node;
  if (threadIdx.x < 32) {
    int kids = 0;
    for (int base = node + 1; base < n; base += 32) {
      const int i = base + threadIdx.x;
      const bool mine = i < n && p.parents[begin + i] == node;
      const unsigned hits = __ballot_sync(0xffffffffu, mine);
      if (mine) {
        const int at = kids + __popc(hits & ((1u << threadIdx.x) - 1u));
        s_child[at] = i;
        s_token[at] = p.tokens[begin + i];
      }
      kids += __popc(hits);
    }
    if (threadIdx.x == 0) s_kids = kids;
  }
  __syncthreads();
  const int kids = s_kids;
  const __nv_bfloat16* lp = p.logits + (long long)row * p.vocab;
  const __nv_bfloat16* lq = p.draft ? p.draft + (long long)row * p.vocab : nullptr;
  const float temperature = p.temps[b];
  if (threadIdx.x == 0) {  // a node that is no node's child is tested by nobody
    const int parent = p.parents[row];
    if (node == 0 || parent < 0 || parent >= node) p.accept[row] = 0.0f;
  }
  if (kids == 0 || !(temperature > 0.0f)) {
    float best = -INFINITY;
    int best_index = kNone;
    if (kids)
      for (int v = threadIdx.x; v < p.vocab; v += kThreads) {
        const float l = __bfloat162float(lp[v]);
        if (better(l, v, best, best_index)) {
          best = l;
          best_index = v;
        }
      }
    block_best(best, best_index, s_red, s_idx);
    if (best_index == kNone) best_index = 0;
    if (threadIdx.x == 0) {
      int winner = -1;
      for (int i = 0; i < kids; ++i) {
        const bool taken = winner < 0 && s_token[i] == best_index;
        p.accept[begin + s_child[i]] = taken ? 1.0f : 0.0f;
        if (taken) winner = s_child[i];
      }
      ws[node].winner = winner;
      ws[node].rejected = 0;
    }
    return;
  }
  const float c = inv_temperature(temperature);
  float m_p = -INFINITY, m_q = -INFINITY;
  for (int v = threadIdx.x; v < p.vocab; v += kThreads) {
    m_p = fmaxf(m_p, __bfloat162float(lp[v]));
    if (lq) m_q = fmaxf(m_q, __bfloat162float(lq[v]));
  }
  m_p = block_max(m_p, s_red);
  m_q = block_max(m_q, s_red);
  float z_p = 0.0f, z_q = 0.0f;
  for (int v = threadIdx.x; v < p.vocab; v += kThreads) {
    z_p += weight(__bfloat162float(lp[v]), m_p, c);
    if (lq) z_q += weight(__bfloat162float(lq[v]), m_q, c);
  }
  z_p = block_sum(z_p, s_red);
  z_q = block_sum(z_q, s_red);
  const Levels lv{0, s_token, s_mass, s_left};
  int winner = -1, rejected = 0;
  float mass = z_q;
  for (int i = 0; i < kids; ++i) {
    // every thread works out the child's probability
    const int t = s_token[i];
    float a = 0.0f;
    if (t >= 0 && t < p.vocab && z_p > 0.0f) {
      const float wq = lq ? weight(__bfloat162float(lq[t]), m_q, c) : 0.0f;
      const float pt = remaining(weight(__bfloat162float(lp[t]), m_p, c) / z_p, wq, t, lq != nullptr, lv, i);
      float qt = 1.0f;
      if (lq) {
        bool gone = false;
        for (int j = 0; j < i; ++j) gone |= s_token[j] == t;
        qt = gone || !(mass > 0.0f) ? 0.0f : wq / mass;
      }
      a = !(pt > 0.0f) ? 0.0f : (qt > 0.0f ? fminf(pt / qt, 1.0f) : 1.0f);
    }
    const bool taken = p.uniforms[begin + s_child[i]] < a;
    if (threadIdx.x == 0) p.accept[begin + s_child[i]] = a;
    if (taken) {
      winner = s_child[i];
      for (int j = i + 1 + threadIdx.x; j < kids; j += kThreads) p.accept[begin + s_child[j]] = 0.0f;
      break;
    }
    // rejected: what is left of P, and Q's sum without the rejected tokens
    // (added up anew: a difference would cancel where the tokens had most)
    if (threadIdx.x == 0) {
      s_mass[i] = mass;
      s_left[i] = 1.0f;  // its sum is what the pass below adds up
    }
    __syncthreads();
    float left = 0.0f, rest = 0.0f;
    for (int v = threadIdx.x; v < p.vocab; v += kThreads) {
      const float wq = lq ? weight(__bfloat162float(lq[v]), m_q, c) : 0.0f;
      left += remaining(weight(__bfloat162float(lp[v]), m_p, c) / z_p, wq, v, lq != nullptr, lv, i + 1);
      bool gone = false;
      for (int j = 0; j <= i; ++j) gone |= s_token[j] == v;
      rest += gone ? 0.0f : wq;
    }
    left = z_p > 0.0f ? block_sum(left, s_red) : 0.0f;
    mass = block_sum(rest, s_red);
    if (threadIdx.x == 0) {
      s_left[i] = left;
      VerifyRow& r = ws[s_child[i]];
      r.mass_q = s_mass[i];
      r.left = left;
    }
    __syncthreads();
    rejected = i + 1;
  }
  if (threadIdx.x == 0) {
    VerifyRow& r = ws[node];
    r.m_p = m_p;
    r.z_p = z_p;
    r.m_q = m_q;
    r.z_q = z_q;
    r.winner = winner;
    r.rejected = rejected;
  }
}

// One CTA per sequence: the accepted path, and the token behind it.
__global__ void __launch_bounds__(kThreads) verify_sample_kernel(const VerifyParams p) {
  __shared__ float s_red[kThreads / 32];
  __shared__ int s_idx[kThreads / 32];
  __shared__ int s_winner[kMaxNodes], s_token[kMaxNodes];
  __shared__ float s_mass[kMaxNodes], s_left[kMaxNodes];
  __shared__ int s_last, s_count;
  const int b = blockIdx.x, begin = p.cu_q[b], n = min(min(p.cu_q[b + 1], p.rows) - begin, p.max_q);
  int* tokens = p.out_tokens + (long long)b * p.max_q;
  int* path = p.path + (long long)b * p.max_q;
  if (begin < 0 || n <= 0) {
    for (int i = threadIdx.x; i < p.max_q; i += kThreads) tokens[i] = path[i] = -1;
    if (threadIdx.x == 0) p.counts[b] = 0;
    return;
  }
  const VerifyRow* ws = p.ws + begin;
  for (int i = threadIdx.x; i < n; i += kThreads) s_winner[i] = ws[i].winner;
  __syncthreads();
  if (threadIdx.x == 0) {
    int at = 0, count = 1;
    path[0] = 0;
    while (s_winner[at] > at) {
      at = s_winner[at];
      path[count] = at;
      tokens[count - 1] = p.tokens[begin + at];
      ++count;
    }
    s_last = at;
    s_count = count;
    p.counts[b] = count;
  }
  __syncthreads();
  const int last = s_last, count = s_count, row = begin + last;
  for (int i = count + threadIdx.x; i < p.max_q; i += kThreads) tokens[i] = path[i] = -1;
  const __nv_bfloat16* lp = p.logits + (long long)row * p.vocab;
  const __nv_bfloat16* lq = p.draft ? p.draft + (long long)row * p.vocab : nullptr;
  const float temperature = p.temps[b];
  const int rejected = ws[last].rejected;
  if (threadIdx.x < 32) {  // the rejected children's levels
    int kids = 0;
    for (int base = last + 1; base < n && kids < rejected; base += 32) {
      const int i = base + threadIdx.x;
      const bool mine = i < n && p.parents[begin + i] == last;
      const unsigned hits = __ballot_sync(0xffffffffu, mine);
      const int at = kids + __popc(hits & ((1u << threadIdx.x) - 1u));
      if (mine && at < rejected) {
        s_token[at] = p.tokens[begin + i];
        s_mass[at] = ws[i].mass_q;
        s_left[at] = ws[i].left;
      }
      kids += __popc(hits);
    }
  }
  __syncthreads();
  const Levels lv{rejected, s_token, s_mass, s_left};
  const float m_p = ws[last].m_p, z_p = ws[last].z_p, m_q = ws[last].m_q;
  const float c = inv_temperature(temperature);
  const uint64_t seed = p.seeds[row];
  float best = -INFINITY;
  int best_index = kNone;
  for (int v = threadIdx.x; v < p.vocab; v += kThreads) {
    const float l = __bfloat162float(lp[v]);
    float score;
    if (rejected == 0) {
      score = gumbel_score(l, temperature, seed, v);
    } else {
      const float wq = lq ? weight(__bfloat162float(lq[v]), m_q, c) : 0.0f;
      const float left = remaining(weight(l, m_p, c) / z_p, wq, v, lq != nullptr, lv, rejected);
      if (!(left > 0.0f)) continue;
      score = logf(left) - gumbel_log(seed, v);
    }
    if (better(score, v, best, best_index)) {
      best = score;
      best_index = v;
    }
  }
  block_best(best, best_index, s_red, s_idx);
  if (threadIdx.x == 0) tokens[count - 1] = best_index == kNone ? 0 : best_index;
}

}  // namespace

int verify_max_nodes() { return kMaxNodes; }

size_t verify_workspace(int rows) { return size_t(rows) * sizeof(VerifyRow); }

cudaError_t launch_verify(cudaStream_t s, const void* logits, const void* draft, const int* tokens,
                          const int* parents, const float* uniforms, const uint64_t* seeds, const float* temps,
                          const int* cu_q, int* out_tokens, int* path, int* counts, float* accept, int rows, int batch,
                          int max_q, int vocab, void* ws) {
  VerifyParams p{static_cast<const __nv_bfloat16*>(logits), static_cast<const __nv_bfloat16*>(draft), tokens,
                 parents, uniforms, seeds, temps, cu_q, out_tokens, path, counts, accept,
                 static_cast<VerifyRow*>(ws), rows, max_q, vocab};
  verify_nodes_kernel<<<dim3(max_q, batch), kThreads, 0, s>>>(p);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  verify_sample_kernel<<<batch, kThreads, 0, s>>>(p);
  return cudaGetLastError();
}

}  // namespace nvbm
