// Causal attention over expanded latent keys and values (nvb_latent_prefill_fwd):
// the simple form, a warp for each (query, head).
#include "internal.cuh"

namespace nvb {

namespace latent_prefill_detail {

__global__ void __launch_bounds__(256) latent_prefill_kernel(const LatentPrefillParams p) {
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= (long long)p.total_q * p.heads) return;
  const int row = int(item / p.heads), head = int(item % p.heads);
  int lo = 0, hi = p.batch;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.cu_q[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  if (lo >= p.batch || p.cu_q[lo] > row || row - p.cu_q[lo] >= p.max_q) return;
  const int n = p.cu_q[lo + 1] - p.cu_q[lo], begin = p.cu_k[lo], end = p.cu_k[lo + 1];
  const bool valid = begin >= 0 && end <= p.total_k;
  const int seen = valid ? end - begin - n + (row - p.cu_q[lo]) + 1 : 0;
  float q[6], acc[4], m = -INFINITY, l = 0.0f;
  for (int i = 0; i < 6; ++i) q[i] = __bfloat162float(p.q[item * 192 + lane + 32 * i]) * p.scale;
  for (int i = 0; i < 4; ++i) acc[i] = 0.0f;
  for (int t = 0; t < seen; ++t) {
    const __nv_bfloat16* kv = p.kv + ((long long)(begin + t) * p.heads + head) * 256;
    const __nv_bfloat16* r = p.k_rope + (long long)(begin + t) * p.rope_stride;
    float s = 0.0f;
    for (int i = 0; i < 4; ++i) s = fmaf(q[i], __bfloat162float(kv[lane + 32 * i]), s);
    for (int i = 0; i < 2; ++i) s = fmaf(q[4 + i], __bfloat162float(r[lane + 32 * i]), s);
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    const float mx = fmaxf(m, s), nm = mx == -INFINITY ? 0.0f : mx;
    const float a = m == mx ? 1.0f : expf(m - nm), w = expf(s - nm);
    m = mx;
    l = l * a + w;
    for (int i = 0; i < 4; ++i) acc[i] = acc[i] * a + w * __bfloat162float(kv[128 + lane + 32 * i]);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  for (int i = 0; i < 4; ++i) p.out[item * 128 + lane + 32 * i] = __float2bfloat16_rn(acc[i] * inv);
  if (lane == 0 && p.lse) p.lse[item] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace latent_prefill_detail

cudaError_t launch_latent_prefill(const LatentPrefillParams& p, cudaStream_t stream) {
  const long long items = (long long)p.total_q * p.heads;
  latent_prefill_detail::latent_prefill_kernel<<<unsigned((items + 7) / 8), 256, 0, stream>>>(p);
  return cudaGetLastError();
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
