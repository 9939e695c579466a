// Writing and reading the latent cache: nvb_latent_store, nvb_latent_gather.
// No counterpart in the reference, whose models keep keys and values a head.
//
// A row of the cache is 576 BF16 (1152 bytes): 512 normalised latent values c
// and 64 rotated key values r that all heads share,
//
//   c = x * w / sqrt(mean(x^2) + eps)          over the first 512 of a kv row
//   r = R(pos) x                               over its last 64
//
// where R turns pair i by the table's angle of (pos, i): elements (i, i + 32)
// or, interleaved, (2 i, 2 i + 1). The queries' rotary parts are turned by the
// same launch. Everything is FP32 and rounded to BF16 once.
//
// Both kernels move each byte once; what bounds them is HBM, and for a decode
// step's few rows the launch and one round trip to memory.
#include "latent_common.cuh"

namespace nvb {

namespace latent_cache_detail {

constexpr int kLatent = 512, kRope = 64, kWidth = kLatent + kRope;
constexpr int kWarps = 4;
constexpr int kHeadsPerWarp = 16;  // of the queries: four lanes a head, 16 values a lane of two heads

// 16 values of a 64-value rotary part: `lo` and `hi` hold its 8-value pieces c and c + 4 (c: the lane's place among
// the head's four) or, interleaved, 2 c and 2 c + 1. Both forms take pairs 8 c .. 8 c + 7 of the table.
__device__ __forceinline__ void rotate16(uint4& lo, uint4& hi, const float (&cs)[8], const float (&sn)[8],
                                         bool interleaved) {
  float a[8], b[8];
  unpack8(lo, a);
  unpack8(hi, b);
  uint32_t w[8];
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_bf16x2(a[2 * i] * cs[i] - a[2 * i + 1] * sn[i], a[2 * i + 1] * cs[i] + a[2 * i] * sn[i]);
      w[4 + i] =
          pack_bf16x2(b[2 * i] * cs[4 + i] - b[2 * i + 1] * sn[4 + i], b[2 * i + 1] * cs[4 + i] + b[2 * i] * sn[4 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = pack_bf16x2(a[2 * i] * cs[2 * i] - b[2 * i] * sn[2 * i],
                         a[2 * i + 1] * cs[2 * i + 1] - b[2 * i + 1] * sn[2 * i + 1]);
      w[4 + i] = pack_bf16x2(b[2 * i] * cs[2 * i] + a[2 * i] * sn[2 * i],
                             b[2 * i + 1] * cs[2 * i + 1] + a[2 * i + 1] * sn[2 * i + 1]);
    }
  }
  lo = make_uint4(w[0], w[1], w[2], w[3]);
  hi = make_uint4(w[4], w[5], w[6], w[7]);
}

struct StoreParams {
  const __nv_bfloat16* kv;      // [rows] x kv_stride, or null
  const __nv_bfloat16* weight;  // [512]
  const int* positions;         // [rows]
  const int* slots;             // [rows]
  __nv_bfloat16* cache;
  const __nv_bfloat16* q;       // [rows, heads] by strides, 64 values each, or null
  __nv_bfloat16* q_out;
  const float* table;           // [max_positions, 64]: cos | sin
  long long kv_stride, q_row, q_head, o_row, o_head, num_slots;
  int rows, heads, units, max_positions, interleaved;  // units: warps a row
  float eps;
};

// A warp takes one row's kv, or the rotary parts of 16 of its query heads. All that does not wait for the position is
// loaded before it (8191 rows of 32 heads: 18.4 us, 4.8 TB/s; eight heads a warp, loaded behind the table, and CTAs of
// eight warps 24.9). It reads what it needs once, in whole sectors; the loads of 40 % of an SM's warps (64 registers, and
// the launch's start and end) do not fill HBM for so short a time.
__global__ void __launch_bounds__(kWarps * 32) store_kernel(const StoreParams p, const FastDiv fd_units) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the next kernel may set itself up beside this one
  const int lane = threadIdx.x & 31;
  const long long at = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (at >= (long long)p.rows * p.units) return;
  const int row = fd_units.div(int(at)), unit = int(at) - row * p.units;
  const bool is_kv = p.kv && unit == 0;
  const int c = lane & 3;  // this lane's pairs of the table: 8 c to 8 c + 7
  const int lo_at = p.interleaved ? 16 * c : 8 * c, hi_at = p.interleaved ? 16 * c + 8 : 32 + 8 * c;

  float cs[8], sn[8];
  auto load_angles = [&] {  // positions outside the table turn by nothing
    const int position = p.positions[row];
    const bool known = position >= 0 && position < p.max_positions;
    const float4* t = reinterpret_cast<const float4*>(p.table + (long long)(known ? position : 0) * kRope + 8 * c);
    const float4 c0 = t[0], c1 = t[1], s0 = t[8], s1 = t[9];
    cs[0] = c0.x, cs[1] = c0.y, cs[2] = c0.z, cs[3] = c0.w, cs[4] = c1.x, cs[5] = c1.y, cs[6] = c1.z, cs[7] = c1.w;
    sn[0] = s0.x, sn[1] = s0.y, sn[2] = s0.z, sn[3] = s0.w, sn[4] = s1.x, sn[5] = s1.y, sn[6] = s1.z, sn[7] = s1.w;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      cs[i] = known ? cs[i] : 1.0f;
      sn[i] = known ? sn[i] : 0.0f;
    }
  };

  if (!is_kv) {
    const int head = (unit - (p.kv ? 1 : 0)) * kHeadsPerWarp + (lane >> 2);
    uint4 lo[2], hi[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      lo[k] = hi[k] = make_uint4(0, 0, 0, 0);
      if (head + 8 * k < p.heads) {
        const __nv_bfloat16* src = p.q + row * p.q_row + (head + 8 * k) * p.q_head;
        lo[k] = *reinterpret_cast<const uint4*>(src + lo_at);
        hi[k] = *reinterpret_cast<const uint4*>(src + hi_at);
      }
    }
    load_angles();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (head + 8 * k >= p.heads) break;
      rotate16(lo[k], hi[k], cs, sn, p.interleaved);
      __nv_bfloat16* dst = p.q_out + row * p.o_row + (head + 8 * k) * p.o_head;
      *reinterpret_cast<uint4*>(dst + lo_at) = lo[k];
      *reinterpret_cast<uint4*>(dst + hi_at) = hi[k];
    }
    return;
  }

  const __nv_bfloat16* src = p.kv + row * p.kv_stride;
  uint4 x[2], w[2], lo = make_uint4(0, 0, 0, 0), hi = lo;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    x[i] = *reinterpret_cast<const uint4*>(src + (i * 32 + lane) * 8);
    w[i] = *reinterpret_cast<const uint4*>(p.weight + (i * 32 + lane) * 8);
  }
  const int slot = p.slots[row];
  if (lane < 4) {
    lo = *reinterpret_cast<const uint4*>(src + kLatent + lo_at);
    hi = *reinterpret_cast<const uint4*>(src + kLatent + hi_at);
    load_angles();
  }
  if (slot < 0 || slot >= p.num_slots) return;  // the whole warp's
  __nv_bfloat16* dst = p.cache + (long long)slot * kWidth;
  float f[2][8], eps = p.eps;
#pragma unroll
  for (int i = 0; i < 2; ++i) unpack8(x[i], f[i]);
  auto sum_squares = [&] {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(f[i][e], f[i][e], sum);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    return sum;
  };
  float sum = sum_squares();
  // Values from 2^59 on: their squares' sum has no FP32, that of 2^-70 of them has.
  if (__any_sync(0xffffffffu, isinf(sum / kLatent + eps))) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] *= 0x1p-70f;
    eps = eps * 0x1p-70f * 0x1p-70f;
    sum = sum_squares();
  }
  const float inv = rsqrtf(sum / kLatent + eps);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float g[8];
    unpack8(w[i], g);
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = pack_bf16x2(f[i][2 * e] * inv * g[2 * e], f[i][2 * e + 1] * inv * g[2 * e + 1]);
    *reinterpret_cast<uint4*>(dst + (i * 32 + lane) * 8) = make_uint4(o[0], o[1], o[2], o[3]);
  }
  if (lane < 4) {
    rotate16(lo, hi, cs, sn, p.interleaved);
    *reinterpret_cast<uint4*>(dst + kLatent + lo_at) = lo;
    *reinterpret_cast<uint4*>(dst + kLatent + hi_at) = hi;
  }
}

struct GatherParams {
  const __nv_bfloat16* cache;
  const int* block_table;  // [batch, table_stride]
  const int* cu_k;         // [batch + 1]
  __nv_bfloat16* latent;
  __nv_bfloat16* rope;
  long long latent_stride, rope_stride;
  int batch, total_k, block_size, table_stride, num_blocks;
};

// A warp takes four rows: each of four lanes finds one row's place in the
// cache, then all 32 move their 16-byte pieces (72 a row), all loads before the
// stores (153,692 keys, 354 MB: 56.4 us, 96 % of the copy rate; one prefix of
// 1000 2.5; with eight rows a warp 0.7 more).
constexpr int kGatherRows = 4;
constexpr int kPieces = kWidth / 8;

__global__ void __launch_bounds__(kWarps * 32) gather_kernel(const GatherParams p, const FastDiv fd_bs) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the next kernel may set itself up beside this one
  const int lane = threadIdx.x & 31;
  const long long first = ((long long)blockIdx.x * kWarps + (threadIdx.x >> 5)) * kGatherRows;
  if (first >= p.total_k) return;
  // where lane i < 4 finds row first + i: its row of the cache, -1 for one of a bad page (zeros), -2 for none to write
  int place = -2;
  if (lane < kGatherRows && first + lane < p.total_k) {
    const int row = int(first) + lane;
    int lo = 0, hi = p.batch;  // the last sequence that begins at or before the row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.cu_k[mid] <= row) lo = mid;
      else hi = mid - 1;
    }
    if (lo < p.batch && p.cu_k[lo] <= row) {
      const long long key = (long long)row - p.cu_k[lo];  // past 32 bits behind an offset far below 0
      const int logical = key <= INT_MAX ? fd_bs.div(int(key)) : p.table_stride;
      const int page = logical < p.table_stride ? p.block_table[(long long)lo * p.table_stride + logical] : -1;
      place = page >= 0 && page < p.num_blocks ? page * p.block_size + (int(key) - logical * p.block_size) : -1;
    }
  }
  constexpr int kEach = kGatherRows * kPieces / 32;
  uint4 v[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int piece = i * 32 + lane, r = piece / kPieces;
    const int from = __shfl_sync(0xffffffffu, place, r);
    v[i] = make_uint4(0, 0, 0, 0);
    if (from >= 0)
      v[i] = *reinterpret_cast<const uint4*>(p.cache + (long long)from * kWidth + (piece - r * kPieces) * 8);
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int piece = i * 32 + lane, r = piece / kPieces, at = (piece - r * kPieces) * 8;
    if (__shfl_sync(0xffffffffu, place, r) == -2) continue;
    __nv_bfloat16* dst = at < kLatent ? p.latent + (first + r) * p.latent_stride + at
                                      : p.rope + (first + r) * p.rope_stride + (at - kLatent);
    *reinterpret_cast<uint4*>(dst) = v[i];
  }
}

// Launched while the kernel before it on the stream ends; it waits for that before any global access.
template <class K, class... A>
cudaError_t launch_dependent(K kernel, long long grid, cudaStream_t stream, const A&... args) {
  if (grid > 0x7fffffffLL) return cudaErrorInvalidValue;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Whether [rows, heads] pieces of 64 values at these strides keep apart from one another.
bool apart(long long rows, long long heads, long long row_stride, long long head_stride) {
  if (row_stride < 0 || head_stride < 0) return false;
  const bool by_row = (heads == 1 || head_stride >= kRope) && (rows == 1 || row_stride >= (heads - 1) * head_stride + kRope);
  const bool by_head = (rows == 1 || row_stride >= kRope) && (heads == 1 || head_stride >= (rows - 1) * row_stride + kRope);
  return by_row || by_head;
}

// Whether x and y, of `x_len` and `y_len` elements a row, lie beside one another in rows that are `stride` long.
bool beside(const void* x, long long x_len, const void* y, long long y_len, long long stride) {
  const long long gap = (static_cast<const char*>(y) - static_cast<const char*>(x)) / 2;
  return (gap >= x_len && gap + y_len <= stride) || (-gap >= y_len && x_len - gap <= stride);
}

}  // namespace latent_cache_detail
}  // namespace nvb

extern "C" {

int nvb_latent_store(void* stream, const void* kv, long long kv_stride, const void* weight, const int* positions,
                     const int* slots, void* cache, const void* q, long long q_row_stride, long long q_head_stride,
                     void* q_out, long long out_row_stride, long long out_head_stride, int rows, int q_heads,
                     int interleaved, int block_size, int num_blocks, float eps, const float* rope_table,
                     int max_positions) {
  using namespace nvb::latent_cache_detail;
  g_last_error[0] = 0;
  if ((!kv && !q) || !positions || !rope_table || rows < 1 || max_positions < 1 ||
      (kv && (!weight || !slots || !cache)) || (q && (!q_out || q_heads < 1)))
    return fail("invalid latent store arguments");
  if (kv && (block_size < 1 || num_blocks < 1 || (long long)block_size * num_blocks > INT_MAX))
    return fail("block_size and num_blocks must be positive and their product fit in int32");
  if (kv && (!(eps > 0.0f) || !std::isfinite(eps))) return fail("eps must be positive and finite");
  if (q && q_heads > 1024) return fail("q_heads must be at most 1024 (got %d)", q_heads);
  const long long limit = INT_MAX;  // of strides: their products with rows and heads stay in 64 bits
  if ((kv && (kv_stride < kWidth || kv_stride > limit)) ||
      (q && (q_row_stride < 0 || q_row_stride > limit || q_head_stride < 0 || q_head_stride > limit ||
             out_row_stride > limit || out_head_stride > limit ||
             !apart(rows, q_heads, out_row_stride, out_head_stride))))
    return fail("kv rows must hold 576 values, and the rows and heads of q_out must not overlap");
  if ((kv && kv_stride % 8) || (q && (q_row_stride % 8 || q_head_stride % 8 || out_row_stride % 8 || out_head_stride % 8)))
    return fail("strides must be multiples of 8 elements");
  if ((kv && (!aligned16(kv) || !aligned16(weight) || !aligned16(cache))) || (q && (!aligned16(q) || !aligned16(q_out))) ||
      !aligned16(rope_table))
    return fail("kv, weight, cache, q, q_out and rope_table must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(positions) | reinterpret_cast<uintptr_t>(slots)) & 3)
    return fail("positions and slots must be 4-byte aligned");
  // the last value of a part of 64 at these strides, and one
  const auto parts = [&](long long row_stride, long long head_stride) {
    return ((rows - 1) * row_stride + (q_heads - 1) * head_stride + kRope) * 2;
  };
  const bool in_place = q && q_out == q && q_row_stride == out_row_stride && q_head_stride == out_head_stride;
  const nvb::Stretch stretches[] = {
      {"cache", kv ? cache : nullptr, kv ? (long long)block_size * num_blocks * kWidth * 2 : 0},
      {"q_out", q ? q_out : nullptr, q ? parts(out_row_stride, out_head_stride) : 0},
      {"q", in_place ? nullptr : q, q ? parts(q_row_stride, q_head_stride) : 0},
      {"kv", kv, kv ? ((rows - 1) * kv_stride + kWidth) * 2 : 0},
      {"weight", kv ? weight : nullptr, kLatent * 2},
      {"positions", positions, rows * 4LL},
      {"slots", kv ? slots : nullptr, rows * 4LL},
      {"rope_table", rope_table, (long long)max_positions * kRope * 4}};
  // the queries and kv may be slices of the same rows, those of one projection
  const bool same_rows = kv && q && kv_stride == out_row_stride &&
                         beside(kv, kWidth, q_out, (q_heads - 1) * out_head_stride + kRope, kv_stride);
  for (int i = 0; i < 2; ++i)
    for (int j = i + 1; j < 8; ++j)
      if (!(i == 1 && j == 3 && same_rows) && nvb::overlap(stretches[i], stretches[j]))
        return fail("%s overlaps %s", stretches[i].name, stretches[j].name);
  StoreParams p{};
  p.kv = static_cast<const __nv_bfloat16*>(kv);
  p.weight = static_cast<const __nv_bfloat16*>(weight);
  p.positions = positions;
  p.slots = slots;
  p.cache = static_cast<__nv_bfloat16*>(cache);
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_out = static_cast<__nv_bfloat16*>(q_out);
  p.table = rope_table;
  p.kv_stride = kv_stride;
  p.q_row = q_row_stride;
  p.q_head = q_head_stride;
  p.o_row = out_row_stride;
  p.o_head = out_head_stride;
  p.num_slots = kv ? (long long)block_size * num_blocks : 0;
  p.rows = rows;
  p.heads = q ? q_heads : 0;
  p.units = (kv ? 1 : 0) + (p.heads + kHeadsPerWarp - 1) / kHeadsPerWarp;
  p.max_positions = max_positions;
  p.interleaved = interleaved != 0;
  p.eps = eps;
  if ((long long)rows * p.units > INT_MAX) return fail("too many rows and heads for one call");
  return cuda_status(launch_dependent(store_kernel, ((long long)rows * p.units + kWarps - 1) / kWarps,
                                      static_cast<cudaStream_t>(stream), p, nvb::FastDiv::make(p.units)),
                     "latent store launch");
}

int nvb_latent_gather(void* stream, const void* cache, const int* block_table, const int* cu_k, void* latent,
                      long long latent_stride, void* rope, long long rope_stride, int batch, int total_k,
                      int block_size, int table_stride, int num_blocks) {
  using namespace nvb::latent_cache_detail;
  g_last_error[0] = 0;
  if (!cache || !block_table || !cu_k || !latent || !rope || batch < 1 || batch > 65535 || total_k < 1 ||
      block_size < 1 || table_stride < 1)
    return fail("invalid latent gather arguments");
  if (num_blocks < 1 || (long long)num_blocks * block_size > INT_MAX)
    return fail("num_blocks must be positive and num_blocks * block_size must fit in int32");
  const long long limit = INT_MAX;
  if (latent_stride < kLatent || latent_stride > limit || latent_stride % 8 || rope_stride < kRope ||
      rope_stride > limit || rope_stride % 8)
    return fail("rows of latent and rope need 512 and 64 values, their strides multiples of 8 elements");
  if (!aligned16(cache) || !aligned16(latent) || !aligned16(rope))
    return fail("cache, latent and rope must be 16-byte aligned");
  if ((reinterpret_cast<uintptr_t>(block_table) | reinterpret_cast<uintptr_t>(cu_k)) & 3)
    return fail("block_table and cu_k must be 4-byte aligned");
  // latent and rope may be slices of the same rows, beside one another in each
  const bool same_rows = latent_stride == rope_stride && beside(latent, kLatent, rope, kRope, rope_stride);
  const nvb::Stretch sources[] = {{"latent", latent, ((total_k - 1) * latent_stride + kLatent) * 2},
                                  {"rope", rope, ((total_k - 1) * rope_stride + kRope) * 2},
                                  {"cache", cache, (long long)num_blocks * block_size * kWidth * 2},
                                  {"block_table", block_table, (long long)batch * table_stride * 4},
                                  {"cu_k", cu_k, (batch + 1) * 4LL}};
  for (int i = 0; i < 2; ++i)
    for (int j = i + 1; j < 5; ++j)
      if (!(j == 1 && same_rows) && nvb::overlap(sources[i], sources[j]))
        return fail("%s overlaps %s", sources[i].name, sources[j].name);
  GatherParams p{};
  p.cache = static_cast<const __nv_bfloat16*>(cache);
  p.block_table = block_table;
  p.cu_k = cu_k;
  p.latent = static_cast<__nv_bfloat16*>(latent);
  p.rope = static_cast<__nv_bfloat16*>(rope);
  p.latent_stride = latent_stride;
  p.rope_stride = rope_stride;
  p.batch = batch;
  p.total_k = total_k;
  p.block_size = block_size;
  p.table_stride = table_stride;
  p.num_blocks = num_blocks;
  const long long warps = ((long long)total_k + kGatherRows - 1) / kGatherRows;
  return cuda_status(launch_dependent(gather_kernel, (warps + kWarps - 1) / kWarps, static_cast<cudaStream_t>(stream),
                                      p, nvb::FastDiv::make(block_size)),
                     "latent gather launch");
}

}  // extern "C"
