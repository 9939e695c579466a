// Absorbed attention over the paged latent cache (nvb_paged_latent_fwd): the
// simple form, a warp for each (query, head).
#include "internal.cuh"

namespace nvb {

namespace latent_detail {

constexpr int kLatent = 512, kWidth = 576;

__global__ void __launch_bounds__(256) latent_kernel(const LatentParams p) {
  const long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= (long long)p.total_q * p.heads) return;
  const int row = int(item / p.heads);
  int lo = 0, hi = p.batch;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (p.cu_q[mid] <= row) lo = mid;
    else hi = mid - 1;
  }
  if (lo >= p.batch || p.cu_q[lo] > row) return;
  const int n = p.cu_q[lo + 1] - p.cu_q[lo], len = p.kv_lens[lo];
  const bool valid = len >= 0 && (long long)len <= (long long)p.table_stride * p.block_size;
  const int seen = valid ? len - n + (row - p.cu_q[lo]) + 1 : 0;
  float q[18], acc[16], m = -INFINITY, l = 0.0f;
  for (int i = 0; i < 18; ++i) q[i] = __bfloat162float(p.q[item * kWidth + lane + 32 * i]) * p.scale;
  for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
  for (int t = 0; t < seen; ++t) {
    const int page = p.block_table[(long long)lo * p.table_stride + t / p.block_size];
    if (page < 0 || page >= p.num_blocks) continue;
    const __nv_bfloat16* k = p.cache + ((long long)page * p.block_size + t % p.block_size) * kWidth;
    float x[18], s = 0.0f;
    for (int i = 0; i < 18; ++i) {
      x[i] = __bfloat162float(k[lane + 32 * i]);
      s = fmaf(q[i], x[i], s);
    }
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    const float mx = fmaxf(m, s), nm = mx == -INFINITY ? 0.0f : mx;
    const float a = m == mx ? 1.0f : expf(m - nm), w = expf(s - nm);
    m = mx;
    l = l * a + w;
    for (int i = 0; i < 16; ++i) acc[i] = acc[i] * a + w * x[i];
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  for (int i = 0; i < 16; ++i) p.out[item * kLatent + lane + 32 * i] = __float2bfloat16_rn(acc[i] * inv);
  if (lane == 0 && p.lse) p.lse[item] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace latent_detail

cudaError_t launch_latent(const LatentParams& p, cudaStream_t stream) {
  const long long items = (long long)p.total_q * p.heads;
  latent_detail::latent_kernel<<<unsigned((items + 7) / 8), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace nvb

extern "C" {

long long nvb_latent_scratch_floats(int num_sms) { return num_sms < 1 || num_sms > 1024 ? 0 : 1024LL * num_sms; }

int nvb_paged_latent_fwd(void* stream, const void* q, const void* cache, void* out, const int* cu_q,
                         const int* kv_lens, const int* block_table, int batch, int total_q, int max_q, int q_heads,
                         int block_size, int table_stride, int num_blocks, float scale, float* lse, float* scratch,
                         long long scratch_floats) {
  g_last_error[0] = 0;
  if (!q || !cache || !out || !cu_q || !kv_lens || !block_table || !scratch || scratch_floats < nvb_latent_scratch_floats(1) || batch < 1 || batch > 65535 ||
      total_q < 1 || max_q < 1 || q_heads < 1 || q_heads > 256 || block_size < 1 || table_stride < 1)
    return fail("invalid latent attention arguments");
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
  return cuda_status(nvb::launch_latent(p, static_cast<cudaStream_t>(stream)), "latent attention launch");
}

}  // extern "C"
