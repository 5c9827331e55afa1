// Paged KV append: quantize-on-write of fp16 K/V into the int8 and K8V3 layouts.
//
// One wave64 handles one (token, kv-head) row: it reads D fp16 K and V values,
// rotates K with a fixed-order fp32 Walsh-Hadamard transform, quantizes, and
// scatters the bytes to storage row (block*Hkv + h)*bs + offset.  Lane l holds
// elements l, l+64, l+128, ... so that every global access of the wave is one
// contiguous span.
#include "s8kv_append_rows.h"
#include "s8kv_host.h"

namespace s8kv {

constexpr int kAppendWaves = 4;  // waves per workgroup

struct AppendArgs {
  const _Float16* k;
  const _Float16* v;
  int64_t num_tokens;
  int num_kv_heads;
  int64_t k_stride_t, k_stride_h, v_stride_t, v_stride_h;
  const int32_t* slot_mapping;
  void* k_cache;
  void* k_scale;
  void* v_cache;   // int8 V (int8 layout) or int32 packed V (k8v3)
  void* v_scale;   // fp32 V scale (int8) or fp32 V norms (k8v3)
  const float* v_codebook;
  uint32_t kc_bytes, ks_bytes, vc_bytes, vs_bytes;
  int big;  // a tensor past 4 GiB: the <.., BIG> kernels store through 64-bit pointers
  int64_t num_blocks;
  int block_size_log2;
  float rot_norm;  // float32(1/sqrt(D))
};

template <int D, bool K8V3, bool BIG>
__global__ __launch_bounds__(64 * kAppendWaves) void append_kernel(AppendArgs a) {
  constexpr int E = RowLayout<D>::E;
  const int lane = threadIdx.x & 63;
  const int64_t row_id = (int64_t)blockIdx.x * kAppendWaves + (threadIdx.x >> 6);
  const int64_t total = a.num_tokens * a.num_kv_heads;
  if (row_id >= total) return;
  const int64_t t = row_id / a.num_kv_heads;
  const int h = (int)(row_id - t * a.num_kv_heads);
  const int32_t slot = a.slot_mapping[t];
  if (slot < 0) return;
  const int bs = 1 << a.block_size_log2;
  const uint32_t blk = (uint32_t)slot >> a.block_size_log2;
  if ((int64_t)blk >= a.num_blocks) return;  // slot outside the pool
  const uint32_t off = (uint32_t)slot & (uint32_t)(bs - 1);
  const uint32_t row = ((blk * (uint32_t)a.num_kv_heads + (uint32_t)h) << a.block_size_log2) + off;

  // both rows' loads in flight together
  float x[E], y[E];
  load_row_f16<D>(a.k + t * a.k_stride_t + h * a.k_stride_h, x, lane);
  load_row_f16<D>(a.v + t * a.v_stride_t + h * a.v_stride_h, y, lane);

  // ---- K: rotate (fp32 FWHT, one multiply, RNE to fp16) then RTN ----
  fwht_row<D>(x, lane);
#pragma unroll
  for (int j = 0; j < E; ++j) x[j] = (float)(_Float16)materialize(x[j] * a.rot_norm);
  rtn_store_row<D>(x, lane, row_out<BIG>(a.k_cache, a.kc_bytes, (uint64_t)row * D),
                   row_out<BIG>(a.k_scale, a.ks_bytes, (uint64_t)row * 4u));

  // ---- V ----
  if constexpr (!K8V3) {
    rtn_store_row<D>(y, lane, row_out<BIG>(a.v_cache, a.vc_bytes, (uint64_t)row * D),
                     row_out<BIG>(a.v_scale, a.vs_bytes, (uint64_t)row * 4u));
  } else {
    static_assert(D == 128 || D == 256, "K8V3 needs head_dim 128 or 256");
    constexpr int NB = D / 128;   // Lloyd-Max blocks per row (lloyd_block = 128)
    constexpr int WORDS = D / 32 * 3;
    float cb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) cb[i] = a.v_codebook[i];
    uint32_t w;
    float nv;
    lloydmax3_encode_row<D>(y, cb, lane, w, nv);
    if (lane < WORDS) row_out<BIG>(a.v_cache, a.vc_bytes, (uint64_t)row * (WORDS * 4)).st32(lane * 4u, w);
    if (lane < NB)
      row_out<BIG>(a.v_scale, a.vs_bytes, (uint64_t)row * (NB * 4)).st32(lane * 4u, __builtin_bit_cast(uint32_t, nv));
  }
}

// Append with several rows per wave (RowsLayout); the bytes equal the
// one-row-per-wave kernel's.  Needs 16-byte aligned K and V rows.
//
// Row groups (kAppendWaves waves of RPW rows) per workgroup: the K8V3 kernel
// derives the codebook's thresholds once per workgroup and reuses them.
template <bool K8V3>
constexpr int kRowsIters = K8V3 ? 4 : 1;

template <int D, bool K8V3, bool BIG>
__global__ __launch_bounds__(64 * kAppendWaves) void append_rows_kernel(AppendArgs a) {
  using L = RowsLayout<D>;
  constexpr int RPW = L::RPW;
  const int lane = threadIdx.x & 63;
  const int li = L::part(lane);
  const RowsHadamard<D> hadamard(li, a.rot_norm);

  float cb[8], thr[8];
  bool search = false;
  if constexpr (K8V3) {
    __shared__ float thr_lds[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) cb[i] = a.v_codebook[i];
    search = lloyd3_search_ok(cb);  // uniform over the workgroup
    if (search) {
      if (threadIdx.x < 7) thr_lds[threadIdx.x + 1] = lloyd3_threshold(a.v_codebook[threadIdx.x], a.v_codebook[threadIdx.x + 1]);
      __syncthreads();
#pragma unroll
      for (int j = 1; j < 8; ++j) thr[j] = thr_lds[j];
    }
    thr[0] = 0.0f;
  }

  const int64_t total = a.num_tokens * a.num_kv_heads;
#pragma unroll 1
  for (int it = 0; it < kRowsIters<K8V3>; ++it) {
    const int64_t row_id =
        (((int64_t)blockIdx.x * kRowsIters<K8V3> + it) * kAppendWaves + (threadIdx.x >> 6)) * RPW + L::row(lane);
    bool live = row_id < total;
    int64_t t = 0;
    int h = 0;
    uint32_t row = 0;
    if (live) {
      t = row_id / a.num_kv_heads;
      h = (int)(row_id - t * a.num_kv_heads);
      const int32_t slot = a.slot_mapping[t];
      const uint32_t blk = (uint32_t)slot >> a.block_size_log2;
      live = slot >= 0 && (int64_t)blk < a.num_blocks;  // negative slots and slots outside the pool are skipped
      row = ((blk * (uint32_t)a.num_kv_heads + (uint32_t)h) << a.block_size_log2) +
            ((uint32_t)slot & ((1u << a.block_size_log2) - 1u));
    }
    // both row parts' loads in flight together
    float x[16], y[16];
    {
      half8_t k0{}, k1{}, v0{}, v1{};
      if (live) {
        const _Float16* kp = a.k + t * a.k_stride_t + h * a.k_stride_h + li * 16;
        const _Float16* vp = a.v + t * a.v_stride_t + h * a.v_stride_h + li * 16;
        k0 = *reinterpret_cast<const half8_t*>(kp);
        k1 = *reinterpret_cast<const half8_t*>(kp + 8);
        v0 = *reinterpret_cast<const half8_t*>(vp);
        v1 = *reinterpret_cast<const half8_t*>(vp + 8);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = (float)k0[i];
        x[8 + i] = (float)k1[i];
        y[i] = (float)v0[i];
        y[8 + i] = (float)v1[i];
      }
    }

    // ---- K: rotate, then RTN ----
    hadamard(x);
    rows_rtn_store<D>(x, live, li, row_out<BIG>(a.k_cache, a.kc_bytes, (uint64_t)row * D),
                      row_out<BIG>(a.k_scale, a.ks_bytes, (uint64_t)row * 4u));

    // ---- V: RTN, or 3-bit Lloyd-Max ----
    if constexpr (!K8V3) {
      rows_rtn_store<D>(y, live, li, row_out<BIG>(a.v_cache, a.vc_bytes, (uint64_t)row * D),
                        row_out<BIG>(a.v_scale, a.vs_bytes, (uint64_t)row * 4u));
    } else {
      static_assert(D == 128 || D == 256, "K8V3 needs head_dim 128 or 256");
      rows_lloydmax3_store<D>(y, live, li, search, cb, thr,
                              row_out<BIG>(a.v_cache, a.vc_bytes, (uint64_t)row * (D / 32 * 3 * 4)),
                              row_out<BIG>(a.v_scale, a.vs_bytes, (uint64_t)row * (D / 128 * 4)));
    }
  }
}

template <bool K8V3, bool BIG>
static int launch_append_impl(const AppendArgs& a, int head_dim, hipStream_t stream) {
  const int64_t rows = a.num_tokens * a.num_kv_heads;
  if (rows == 0) return S8KV_OK;
  const bool rows16 = ((uintptr_t)a.k % 16 == 0) && ((uintptr_t)a.v % 16 == 0) && a.k_stride_t % 8 == 0 &&
                      a.k_stride_h % 8 == 0 && a.v_stride_t % 8 == 0 && a.v_stride_h % 8 == 0;
  if (rows16) {  // several rows per wave
    const int rows_per_wg = kAppendWaves * 64 / (head_dim / 16) * kRowsIters<K8V3>;
    const int64_t grid = (rows + rows_per_wg - 1) / rows_per_wg;
    S8KV_REQUIRE(grid < (int64_t(1) << 31), S8KV_ERR_INVALID, "append: too many rows (%lld)", (long long)rows);
    dim3 g((unsigned)grid), b(64 * kAppendWaves);
    switch (head_dim) {
      case 32:
        if constexpr (!K8V3) { hipLaunchKernelGGL((append_rows_kernel<32, false, BIG>), g, b, 0, stream, a); break; }
        return S8KV_ERR_UNSUPPORTED;
      case 64:
        if constexpr (!K8V3) { hipLaunchKernelGGL((append_rows_kernel<64, false, BIG>), g, b, 0, stream, a); break; }
        return S8KV_ERR_UNSUPPORTED;
      case 128: hipLaunchKernelGGL((append_rows_kernel<128, K8V3, BIG>), g, b, 0, stream, a); break;
      case 256: hipLaunchKernelGGL((append_rows_kernel<256, K8V3, BIG>), g, b, 0, stream, a); break;
      default: return S8KV_ERR_UNSUPPORTED;
    }
    return check_launch(K8V3 ? "s8kv_append_k8v3" : "s8kv_append_int8");
  }
  const int64_t grid = (rows + kAppendWaves - 1) / kAppendWaves;
  S8KV_REQUIRE(grid < (int64_t(1) << 31), S8KV_ERR_INVALID, "append: too many rows (%lld)", (long long)rows);
  dim3 g((unsigned)grid), b(64 * kAppendWaves);
  switch (head_dim) {
    case 32:
      if constexpr (!K8V3) { hipLaunchKernelGGL((append_kernel<32, false, BIG>), g, b, 0, stream, a); break; }
      return S8KV_ERR_UNSUPPORTED;
    case 64:
      if constexpr (!K8V3) { hipLaunchKernelGGL((append_kernel<64, false, BIG>), g, b, 0, stream, a); break; }
      return S8KV_ERR_UNSUPPORTED;
    case 128: hipLaunchKernelGGL((append_kernel<128, K8V3, BIG>), g, b, 0, stream, a); break;
    case 256: hipLaunchKernelGGL((append_kernel<256, K8V3, BIG>), g, b, 0, stream, a); break;
    default: return S8KV_ERR_UNSUPPORTED;
  }
  return check_launch(K8V3 ? "s8kv_append_k8v3" : "s8kv_append_int8");
}

template <bool K8V3>
static int launch_append(const AppendArgs& a, int head_dim, hipStream_t stream) {
  return a.big ? launch_append_impl<K8V3, true>(a, head_dim, stream) : launch_append_impl<K8V3, false>(a, head_dim, stream);
}

static int common_append_checks(const void* k, const void* v, int64_t num_tokens, int num_kv_heads, int head_dim,
                                const int32_t* slot_mapping, int64_t num_blocks, int block_size) {
  S8KV_REQUIRE(num_tokens >= 0, S8KV_ERR_INVALID, "append: num_tokens < 0");
  S8KV_REQUIRE(num_kv_heads > 0, S8KV_ERR_INVALID, "append: num_kv_heads must be > 0");
  S8KV_REQUIRE(head_dim_ok(head_dim), S8KV_ERR_UNSUPPORTED, "append: head_dim %d not in {32,64,128,256}", head_dim);
  S8KV_REQUIRE(is_pow2(block_size) && block_size >= 4, S8KV_ERR_UNSUPPORTED,
               "append: block_size %d must be a power of two >= 4", block_size);
  S8KV_REQUIRE(num_blocks > 0, S8KV_ERR_INVALID, "append: num_blocks must be > 0");
  S8KV_REQUIRE(num_tokens == 0 || (k && v && slot_mapping), S8KV_ERR_INVALID, "append: null input pointer");
  return S8KV_OK;
}

}  // namespace s8kv

using namespace s8kv;

extern "C" int s8kv_append_int8(const void* k, const void* v, int64_t num_tokens, int num_kv_heads, int head_dim,
                                int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
                                const int32_t* slot_mapping, int8_t* k_cache, float* k_scale, int8_t* v_cache,
                                float* v_scale, int64_t num_blocks, int block_size, void* stream) {
  int rc = common_append_checks(k, v, num_tokens, num_kv_heads, head_dim, slot_mapping, num_blocks, block_size);
  if (rc) return rc;
  const int64_t rows = num_blocks * num_kv_heads * block_size;
  S8KV_REQUIRE(fits_u32(rows), S8KV_ERR_UNSUPPORTED, "append: more than 2^32 cache rows per layer");
  S8KV_REQUIRE(k_cache && k_scale && v_cache && v_scale, S8KV_ERR_INVALID, "append: null cache pointer");
  AppendArgs a{};
  a.k = (const _Float16*)k;
  a.v = (const _Float16*)v;
  a.num_tokens = num_tokens;
  a.num_kv_heads = num_kv_heads;
  a.k_stride_t = k_stride_t; a.k_stride_h = k_stride_h;
  a.v_stride_t = v_stride_t; a.v_stride_h = v_stride_h;
  a.slot_mapping = slot_mapping;
  a.k_cache = k_cache; a.k_scale = k_scale; a.v_cache = v_cache; a.v_scale = v_scale;
  a.big = !fits_u32(rows * head_dim);
  a.kc_bytes = cap_u32((uint64_t)(rows * head_dim));
  a.vc_bytes = cap_u32((uint64_t)(rows * head_dim));
  a.ks_bytes = cap_u32((uint64_t)(rows * 4));
  a.vs_bytes = cap_u32((uint64_t)(rows * 4));
  a.num_blocks = num_blocks;
  a.block_size_log2 = log2i(block_size);
  a.rot_norm = (float)(1.0 / __builtin_sqrt((double)head_dim));
  return launch_append<false>(a, head_dim, (hipStream_t)stream);
}

extern "C" int s8kv_append_k8v3(const void* k, const void* v, int64_t num_tokens, int num_kv_heads, int head_dim,
                                int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
                                const int32_t* slot_mapping, int8_t* k_cache, float* k_scale, int32_t* v_packed,
                                float* v_norm, const float* v_codebook, int lloyd_block, int64_t num_blocks,
                                int block_size, void* stream) {
  int rc = common_append_checks(k, v, num_tokens, num_kv_heads, head_dim, slot_mapping, num_blocks, block_size);
  if (rc) return rc;
  S8KV_REQUIRE(head_dim == 128 || head_dim == 256, S8KV_ERR_UNSUPPORTED,
               "append_k8v3: head_dim %d not in {128, 256}", head_dim);
  S8KV_REQUIRE(lloyd_block == 128, S8KV_ERR_UNSUPPORTED, "append_k8v3: lloyd_block %d != 128", lloyd_block);
  S8KV_REQUIRE(k_cache && k_scale && v_packed && v_norm && v_codebook, S8KV_ERR_INVALID,
               "append_k8v3: null cache pointer");
  const int64_t rows = num_blocks * num_kv_heads * block_size;
  S8KV_REQUIRE(fits_u32(rows), S8KV_ERR_UNSUPPORTED, "append_k8v3: more than 2^32 cache rows per layer");
  AppendArgs a{};
  a.k = (const _Float16*)k;
  a.v = (const _Float16*)v;
  a.num_tokens = num_tokens;
  a.num_kv_heads = num_kv_heads;
  a.k_stride_t = k_stride_t; a.k_stride_h = k_stride_h;
  a.v_stride_t = v_stride_t; a.v_stride_h = v_stride_h;
  a.slot_mapping = slot_mapping;
  a.k_cache = k_cache; a.k_scale = k_scale; a.v_cache = v_packed; a.v_scale = v_norm;
  a.v_codebook = v_codebook;
  a.big = !fits_u32(rows * head_dim);
  a.kc_bytes = cap_u32((uint64_t)(rows * head_dim));
  a.ks_bytes = cap_u32((uint64_t)(rows * 4));
  a.vc_bytes = cap_u32((uint64_t)(rows * (head_dim / 32 * 3) * 4));
  a.vs_bytes = cap_u32((uint64_t)(rows * (head_dim / 128) * 4));
  a.num_blocks = num_blocks;
  a.block_size_log2 = log2i(block_size);
  a.rot_norm = (float)(1.0 / __builtin_sqrt((double)head_dim));
  return launch_append<true>(a, head_dim, (hipStream_t)stream);
}
