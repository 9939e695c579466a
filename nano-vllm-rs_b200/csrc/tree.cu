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
#include "internal.cuh"

namespace nvb {

namespace tree_detail {

constexpr float kLn2 = 0.693147180559945309f;
constexpr int kWarps = 8;

// One warp per (node, query head): a lane holds four dimensions.
__global__ void __launch_bounds__(kWarps * 32)
    tree_kernel(const TreeParams p, const __nv_bfloat16* __restrict__ kc, const __nv_bfloat16* __restrict__ vc) {
  const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = blockIdx.x * kWarps + warp;
  const int begin = p.cu_q[b], n = min(p.cu_q[b + 1], p.total_q) - begin;
  const int node = item / p.qh, head = item - node * p.qh;
  if (begin < 0 || node >= min(n, p.max_q)) return;
  const int len = p.kv_lens[b], ctx = len - n;
  const bool valid = ctx >= 0 && (long long)len <= (long long)p.table_stride * p.block_size;
  const long long row = begin + node;
  const uint2 qw = *reinterpret_cast<const uint2*>(p.q + (row * p.qh + head) * 128 + lane * 4);
  const float q0 = bf16lo(qw.x), q1 = bf16hi(qw.x), q2 = bf16lo(qw.y), q3 = bf16hi(qw.y);
  const int* table = p.block_table + (long long)b * p.table_stride;
  float m = -INFINITY, l = 0.0f, a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
  for (int key = 0; valid && key < len; ++key) {
    const int page = table[key / p.block_size];
    if (page < 0 || page >= p.num_blocks) continue;
    const int t = key - ctx;
    if (t >= 0 && (t >= 64 * p.mask_words || !((p.mask[row * p.mask_words + (t >> 6)] >> (t & 63)) & 1))) continue;
    const long long at =
        (((long long)page * p.block_size + key % p.block_size) * p.kvh + head / (p.qh / p.kvh)) * 128 + lane * 4;
    const uint2 kw = *reinterpret_cast<const uint2*>(kc + at), vw = *reinterpret_cast<const uint2*>(vc + at);
    float s = q0 * bf16lo(kw.x) + q1 * bf16hi(kw.x) + q2 * bf16lo(kw.y) + q3 * bf16hi(kw.y);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    s *= p.scale_log2;
    const float mn = fmaxf(m, s);
    const float alpha = m == -INFINITY ? 0.0f : exp2f(m - mn), w = exp2f(s - mn);
    m = mn;
    l = l * alpha + w;
    a0 = a0 * alpha + w * bf16lo(vw.x);
    a1 = a1 * alpha + w * bf16hi(vw.x);
    a2 = a2 * alpha + w * bf16lo(vw.y);
    a3 = a3 * alpha + w * bf16hi(vw.y);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint2 o;
  o.x = pack_bf16x2(a0 * inv, a1 * inv);
  o.y = pack_bf16x2(a2 * inv, a3 * inv);
  *reinterpret_cast<uint2*>(p.out + (row * p.qh + head) * 128 + lane * 4) = o;
  if (lane == 0 && p.lse) p.lse[row * p.qh + head] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

}  // namespace tree_detail

cudaError_t launch_tree(const TreeParams& p, const void* k, const void* v, cudaStream_t stream) {
  using namespace tree_detail;
  const dim3 grid(unsigned((p.max_q * p.qh + kWarps - 1) / kWarps), unsigned(p.batch));
  tree_kernel<<<grid, kWarps * 32, 0, stream>>>(p, static_cast<const __nv_bfloat16*>(k),
                                                static_cast<const __nv_bfloat16*>(v));
  return cudaGetLastError();
}

}  // namespace nvb

extern "C" {

int nvb_tree_num_splits(int batch, int max_q, int q_heads, int kv_heads, int max_k, int num_sms) {
  if (batch <= 0 || max_q <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || max_k <= 0 ||
      num_sms <= 0 || num_sms > 1024)
    return 0;
  return 1;
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
      (num_splits > 1 && (!lse_accum || !out_accum)))
    return fail("invalid paged tree attention BF16 hdim128 arguments");
  if (mask_words < 1 || mask_words > 16 || max_q > 64 * mask_words)
    return fail("tree_mask needs a bit for each of max_q nodes in 1 to 16 words (max_q %d, %d words)", max_q,
                mask_words);
  if (num_blocks <= 0 || (long long)num_blocks * block_size > INT_MAX)
    return fail("num_blocks must be positive and num_blocks * block_size must fit in int32");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || (out_accum && !aligned16(out_accum)) ||
      (reinterpret_cast<uintptr_t>(tree_mask) & 7))
    return fail("q, k, v, out and out_accum must be 16-byte aligned, tree_mask 8-byte aligned");
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
  return cuda_status(launch_tree(p, k, v, static_cast<cudaStream_t>(stream)), "tree attention launch");
}

}  // extern "C"
