// Copies within the paged K/V cache, over every layer in one launch:
// pages of forked sequences (nvb_cache_copy_pages) and the accepted path of a
// verified draft tree (nvb_cache_compact_paths). No counterpart in the
// reference, whose sequences never share a page they still write.
//
// Both move bytes only: the bound is HBM bandwidth (each row read once and
// written once), or the latency of one load and one store for small calls.
//
// Measured (B200, 56 caches of 8 heads of 128, copy rate 6.57 TB/s): 16 whole
// pages, 940 MB, 145 us (6.48 TB/s); the paths of 64 trees of 8 to 32 nodes, 117
// MB, 22 us (5.3 TB/s: a CTA reads counts, path and table before it moves 16 KB);
// one tree 2.7 us. With 4, 2 and 1 KV heads the same 64 trees take 16.0, 10.5 and
// 9.7 us, for 8.9, 4.5 and 2.2 at the copy rate: a thread is a column of the row,
// and a row of one head has 16 for a CTA's 128 threads.
#include "internal.cuh"

namespace nvb {

namespace cache_ops_detail {

// The layers' cache pointers travel as a kernel parameter, so a launch needs
// no device array and a CUDA graph keeps them by value.
struct LayerPtrs {
  void* p[2 * kCacheLayers];  // K then V of each layer
};

constexpr int kThreads = 256;
constexpr int kUnroll = 8;  // vectors a thread loads before it stores any

// Vec: 16 bytes where rows and caches allow it, else one 2-byte element.
template <class Vec>
__global__ void __launch_bounds__(kThreads)
    copy_pages_kernel(const __grid_constant__ LayerPtrs ptrs, const int* __restrict__ src,
                      const int* __restrict__ dst, const int* __restrict__ rows, int chunks, int row_vecs,
                      int block_size, int num_blocks) {
  const int chunk = blockIdx.x % chunks, pair = blockIdx.x / chunks;
  const int from = src[pair], to = dst[pair];
  if (from < 0 || from >= num_blocks || to < 0 || to >= num_blocks || from == to) return;
  const int n = rows ? min(max(rows[pair], 0), block_size) : block_size;
  const long long page_vecs = (long long)block_size * row_vecs, end = (long long)n * row_vecs;
  Vec* base = static_cast<Vec*>(ptrs.p[blockIdx.y]);
  const Vec* s = base + from * page_vecs;
  Vec* d = base + to * page_vecs;
  const long long i0 = (long long)chunk * (kThreads * kUnroll) + threadIdx.x;
  Vec v[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    if (i0 + u * kThreads < end) v[u] = s[i0 + u * kThreads];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u)
    if (i0 + u * kThreads < end) d[i0 + u * kThreads] = v[u];
}

constexpr int kMoveThreads = 128;

// Row ctx + path[d] moves to row ctx + d for the accepted nodes d = 1 ..
// counts - 1 of a sequence. A thread owns one column (vector) of the row and
// takes the moves in order, kUnroll at a time. That is enough for moves whose
// source is another one's target: the path grows strictly, so path[d] >= d,
// and a row that move d overwrites (ctx + d) is no later move's source
// (path[d'] >= d' > d). Batches of 4, 12 and 16 rows take 22.8, 22.7 and 24.5 us
// where 8 take 22.1; several caches a CTA, which share the path's reads, 24 to 55.
template <class Vec>
__global__ void __launch_bounds__(kMoveThreads)
    compact_paths_kernel(const __grid_constant__ LayerPtrs ptrs, const int* __restrict__ cu_q,
                         const int* __restrict__ kv_lens, const int* __restrict__ tables,
                         const int* __restrict__ path, const int* __restrict__ counts, int* __restrict__ new_lens,
                         int path_stride, int row_vecs, int block_size, int table_stride, int num_blocks,
                         bool write_lens) {
  __shared__ int s_src[kMoveThreads], s_dst[kMoveThreads];
  const int b = blockIdx.y, n = cu_q[b + 1] - cu_q[b], ctx = kv_lens[b] - n;
  const int count = min(max(counts[b], 0), path_stride);
  if (write_lens && blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) new_lens[b] = ctx + count;
  const int* table = tables + (long long)b * table_stride;
  Vec* base = static_cast<Vec*>(ptrs.p[blockIdx.x]);
  const int col = blockIdx.z * kMoveThreads + threadIdx.x;
  // slot of a position, or -1 (a page outside the cache moves nothing)
  auto slot = [&](long long pos) -> int {
    if (pos < 0 || pos >= (long long)table_stride * block_size) return -1;
    const int page = table[pos / block_size];
    return page >= 0 && page < num_blocks ? page * block_size + int(pos % block_size) : -1;
  };
  for (int d0 = 1; d0 < count; d0 += kMoveThreads) {
    const int m = min(kMoveThreads, count - d0);
    if (int(threadIdx.x) < m) {
      const int d = d0 + threadIdx.x, node = path[(long long)b * path_stride + d];
      const bool moves = node > d && node < n;  // a node already in place stays
      const int from = moves ? slot((long long)ctx + node) : -1, to = moves ? slot((long long)ctx + d) : -1;
      s_src[threadIdx.x] = to < 0 ? -1 : from;
      s_dst[threadIdx.x] = to;
    }
    __syncthreads();
    if (col < row_vecs) {
      for (int e = 0; e < m; e += kUnroll) {
        Vec v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (e + u < m && s_src[e + u] >= 0) v[u] = base[(long long)s_src[e + u] * row_vecs + col];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (e + u < m && s_src[e + u] >= 0) base[(long long)s_dst[e + u] * row_vecs + col] = v[u];
      }
    }
    __syncthreads();
  }
}

}  // namespace cache_ops_detail

cudaError_t launch_copy_pages(cudaStream_t stream, void* const* k, void* const* v, int layers, bool vec16,
                              const int* src, const int* dst, const int* rows, int pairs, int row_bytes,
                              int block_size, int num_blocks) {
  using namespace cache_ops_detail;
  const int row_vecs = row_bytes / (vec16 ? 16 : 2);
  const long long chunks = ((long long)block_size * row_vecs + kThreads * kUnroll - 1) / (kThreads * kUnroll);
  if (chunks * pairs > 0x7fffffffLL) return cudaErrorInvalidValue;
  LayerPtrs ptrs;
  for (int l = 0; l < layers; ++l) {
    ptrs.p[2 * l] = k[l];
    ptrs.p[2 * l + 1] = v[l];
  }
  const dim3 grid(unsigned(chunks * pairs), unsigned(2 * layers));
  if (vec16)
    copy_pages_kernel<uint4><<<grid, kThreads, 0, stream>>>(ptrs, src, dst, rows, int(chunks), row_vecs, block_size,
                                                            num_blocks);
  else
    copy_pages_kernel<unsigned short><<<grid, kThreads, 0, stream>>>(ptrs, src, dst, rows, int(chunks), row_vecs,
                                                                     block_size, num_blocks);
  return cudaGetLastError();
}

cudaError_t launch_compact_paths(cudaStream_t stream, void* const* k, void* const* v, int layers, bool vec16,
                                 const int* cu_q, const int* kv_lens, const int* tables, const int* path,
                                 const int* counts, int* new_lens, int batch, int path_stride, int row_bytes,
                                 int block_size, int table_stride, int num_blocks, bool write_lens) {
  using namespace cache_ops_detail;
  const int row_vecs = row_bytes / (vec16 ? 16 : 2);
  const int cols = (row_vecs + kMoveThreads - 1) / kMoveThreads;
  if (cols > 65535) return cudaErrorInvalidValue;
  LayerPtrs ptrs;
  for (int l = 0; l < layers; ++l) {
    ptrs.p[2 * l] = k[l];
    ptrs.p[2 * l + 1] = v[l];
  }
  const dim3 grid(unsigned(2 * layers), unsigned(batch), unsigned(cols));
  if (vec16)
    compact_paths_kernel<uint4><<<grid, kMoveThreads, 0, stream>>>(ptrs, cu_q, kv_lens, tables, path, counts,
                                                                   new_lens, path_stride, row_vecs, block_size,
                                                                   table_stride, num_blocks, write_lens);
  else
    compact_paths_kernel<unsigned short><<<grid, kMoveThreads, 0, stream>>>(ptrs, cu_q, kv_lens, tables, path,
                                                                            counts, new_lens, path_stride, row_vecs,
                                                                            block_size, table_stride, num_blocks,
                                                                            write_lens);
  return cudaGetLastError();
}

}  // namespace nvb

extern "C" {

// Checks shared by the two entry points; 0, or -1 with the message set.
static int cache_args(void* const* k_layers, void* const* v_layers, int layers, int kv_heads, int head_dim,
                      int block_size, int num_blocks, bool* vec16) {
  if (!k_layers || !v_layers || layers < 1 || layers > 1024 || kv_heads < 1 || head_dim < 1 || block_size < 1 ||
      num_blocks < 1)
    return fail("invalid cache arguments");
  if ((long long)num_blocks * block_size > INT_MAX) return fail("num_blocks * block_size must fit in int32");
  if ((long long)kv_heads * head_dim > (1 << 20)) return fail("kv_heads * head_dim must be at most 2^20");
  *vec16 = (long long)kv_heads * head_dim * 2 % 16 == 0;
  for (int l = 0; l < layers; ++l) {
    if (!k_layers[l] || !v_layers[l]) return fail("layer %d has no cache", l);
    if (k_layers[l] == v_layers[l]) return fail("layer %d has one cache for K and V", l);
    if ((reinterpret_cast<uintptr_t>(k_layers[l]) | reinterpret_cast<uintptr_t>(v_layers[l])) & 1)
      return fail("caches must be 2-byte aligned");
    *vec16 = *vec16 && aligned16(k_layers[l]) && aligned16(v_layers[l]);
  }
  return 0;
}

int nvb_cache_copy_pages(void* stream, void* const* k_layers, void* const* v_layers, int layers,
                         const int* src_pages, const int* dst_pages, const int* rows, int pairs, int kv_heads,
                         int head_dim, int block_size, int num_blocks) {
  g_last_error[0] = 0;
  bool vec16 = false;
  if (int rc = cache_args(k_layers, v_layers, layers, kv_heads, head_dim, block_size, num_blocks, &vec16)) return rc;
  if (pairs < 0 || pairs > num_blocks) return fail("pairs must be in [0, num_blocks]");
  if (pairs == 0) return 0;
  if (!src_pages || !dst_pages) return fail("src_pages and dst_pages are required");
  if ((reinterpret_cast<uintptr_t>(src_pages) | reinterpret_cast<uintptr_t>(dst_pages) |
       reinterpret_cast<uintptr_t>(rows)) & 3)
    return fail("src_pages, dst_pages and rows must be 4-byte aligned");
  for (int l = 0; l < layers; l += kCacheLayers) {
    const int n = layers - l < kCacheLayers ? layers - l : kCacheLayers;
    if (int rc = cuda_status(launch_copy_pages(static_cast<cudaStream_t>(stream), k_layers + l, v_layers + l, n,
                                               vec16, src_pages, dst_pages, rows, pairs, kv_heads * head_dim * 2,
                                               block_size, num_blocks),
                             "page copy launch"))
      return rc;
  }
  return 0;
}

int nvb_cache_compact_paths(void* stream, void* const* k_layers, void* const* v_layers, int layers,
                            const int* cu_q, const int* kv_lens, const int* block_table, const int* path,
                            const int* counts, int* new_kv_lens, int batch, int path_stride, int kv_heads,
                            int head_dim, int block_size, int table_stride, int num_blocks) {
  g_last_error[0] = 0;
  bool vec16 = false;
  if (int rc = cache_args(k_layers, v_layers, layers, kv_heads, head_dim, block_size, num_blocks, &vec16)) return rc;
  if (!cu_q || !kv_lens || !block_table || !path || !counts || !new_kv_lens || batch < 1 || batch > 65535 ||
      path_stride < 1 || table_stride < 1)
    return fail("invalid path compaction arguments");
  if (new_kv_lens == kv_lens) return fail("new_kv_lens must not be kv_lens");
  if ((reinterpret_cast<uintptr_t>(cu_q) | reinterpret_cast<uintptr_t>(kv_lens) |
       reinterpret_cast<uintptr_t>(block_table) | reinterpret_cast<uintptr_t>(path) |
       reinterpret_cast<uintptr_t>(counts) | reinterpret_cast<uintptr_t>(new_kv_lens)) & 3)
    return fail("cu_q, kv_lens, block_table, path, counts and new_kv_lens must be 4-byte aligned");
  for (int l = 0; l < layers; l += kCacheLayers) {
    const int n = layers - l < kCacheLayers ? layers - l : kCacheLayers;
    if (int rc = cuda_status(launch_compact_paths(static_cast<cudaStream_t>(stream), k_layers + l, v_layers + l, n,
                                                  vec16, cu_q, kv_lens, block_table, path, counts, new_kv_lens,
                                                  batch, path_stride, kv_heads * head_dim * 2, block_size,
                                                  table_stride, num_blocks, l == 0),
                             "path compaction launch"))
      return rc;
  }
  return 0;
}

}  // extern "C"
