// Causal linear attention with one decay per head.  Head h of sequence b keeps
// a D x D state S in fp32 (rows: key dims, columns: value dims); per token
//   S <- lambda_h S + k_t v_t^T,   o_t = scale q_t^T S,   lambda_h = exp(log_decay_h).
// States live in a pool [slots][heads][D][D]; state_slots names each
// sequence's slot.  A slot outside the pool makes its sequence a padding row:
// zeros out, nothing read or written.
#include "s8kv_device.h"
#include "s8kv_host.h"

namespace s8kv {
namespace linear {

typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

struct Args {
  const void *q, *k, *v;  // [tokens][heads][D], unit stride on D, element strides
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;
  void* out;
  int64_t o_t, o_h;
  int64_t tokens;
  int batch, heads, group;  // query heads, and of them those that share a key head
  const float* log_decay;   // [heads]
  float* state;
  int64_t state_slot, num_slots;  // elements between slots
  const int32_t* slots;   // [batch], NULL: sequence b has slot b
  const uint8_t* reset;   // [batch], NULL: none; non-zero starts from an empty state
  const int32_t* cu;      // [batch + 1], NULL: one token a sequence
  float scale;
};

template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  if constexpr (DT == 0) return (float)static_cast<const _Float16*>(p)[i];
  else return __builtin_bit_cast(float, (uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
}
template <int DT>
__device__ __forceinline__ void store1(void* p, int64_t i, float x) {
  if constexpr (DT == 0) static_cast<_Float16*>(p)[i] = (_Float16)x;
  else static_cast<__bf16*>(p)[i] = (__bf16)x;
}

// Tokens [first, last) of sequence b, clamped to the tensors.
__device__ __forceinline__ void extent(const Args& a, int b, int64_t& first, int64_t& last) {
  first = b;
  last = b + 1;
  if (a.cu) {
    first = min(max((int64_t)a.cu[b], (int64_t)0), a.tokens);
    last = min(max((int64_t)a.cu[b + 1], first), a.tokens);
  }
}

// exp(x) as an fp32 pair hi + lo: a decay is applied thousands of times in a
// row, and the rounding of a single fp32 factor would add up instead of
// cancelling (2^-25 a step, the same way each time).
struct Factor {
  float hi, lo;
  __device__ __forceinline__ explicit Factor(double x) {
    const double e = exp(x);
    hi = (float)e;
    lo = (float)(e - (double)hi);
  }
  __device__ __forceinline__ float operator()(float s) const { return __builtin_fmaf(s, hi, s * lo); }
};

// The recurrence, one workgroup per (sequence, head, CT value dims).  Threads
// hold four columns of every RG-th row of the state in registers.
template <int D, int DT, int CT>
__global__ __launch_bounds__(256) void recurrent_kernel(Args a) {
  constexpr int TX = CT / 4, RG = 256 / TX, RPT = D / RG, TILES = D / CT;
  static_assert(RPT >= 1 && TX <= 64, "tile");
  __shared__ float qs[D], ks[D];
  __shared__ float4_t part[4][TX];
  const int tile = blockIdx.x % TILES;
  const int h = blockIdx.x / TILES % a.heads;
  const int b = blockIdx.x / TILES / a.heads;
  const int tid = threadIdx.x, tx = tid % TX, rg = tid / TX;
  const int col = tile * CT + 4 * tx;

  int64_t first, last;
  extent(a, b, first, last);
  const int slot = a.slots ? a.slots[b] : b;
  const bool live = slot >= 0 && slot < a.num_slots;
  const bool fresh = live && a.reset && a.reset[b];
  if (!live) {
    for (int64_t t = first; t < last; ++t)
      for (int c = tid; c < CT; c += 256) store1<DT>(a.out, t * a.o_t + h * a.o_h + tile * CT + c, 0.0f);
  } else if (first < last || fresh) {
    float* st = a.state + slot * a.state_slot + (int64_t)h * D * D + col;
    const int hk = h / a.group;
    float4_t s[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
      s[i] = fresh ? float4_t{0, 0, 0, 0} : *reinterpret_cast<const float4_t*>(st + (int64_t)(rg + RG * i) * D);
    const Factor lambda((double)a.log_decay[h]);
    for (int64_t t = first; t < last; ++t) {
      __syncthreads();
      for (int d = tid; d < D; d += 256) {
        qs[d] = load1<DT>(a.q, t * a.q_t + h * a.q_h + d) * a.scale;
        ks[d] = load1<DT>(a.k, t * a.k_t + hk * a.k_h + d);
      }
      float4_t v;
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = load1<DT>(a.v, t * a.v_t + hk * a.v_h + col + c);
      __syncthreads();
      float4_t o = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < RPT; ++i) {
        const float k = ks[rg + RG * i], q = qs[rg + RG * i];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[i][c] = __builtin_fmaf(k, v[c], lambda(s[i][c]));
          o[c] = __builtin_fmaf(q, s[i][c], o[c]);
        }
      }
#pragma unroll
      for (int m = TX; m < 64; m <<= 1) {
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] += shfl_xor_f(o[c], m);
      }
      if ((tid & 63) < TX) part[tid >> 6][tx] = o;
      __syncthreads();
      if (tid < CT) {
        const int x = tid / 4, c = tid % 4;
        const float r = (part[0][x][c] + part[1][x][c]) + (part[2][x][c] + part[3][x][c]);
        store1<DT>(a.out, t * a.o_t + h * a.o_h + tile * CT + tid, r);
      }
    }
#pragma unroll
    for (int i = 0; i < RPT; ++i) *reinterpret_cast<float4_t*>(st + (int64_t)(rg + RG * i) * D) = s[i];
  }
  if (a.cu) {  // rows behind the last sequence: zeros, shared out over the sequences' workgroups
    const int64_t end = min(max((int64_t)a.cu[a.batch], (int64_t)0), a.tokens);
    for (int64_t t = end + b; t < a.tokens; t += a.batch)
      for (int c = tid; c < CT; c += 256) store1<DT>(a.out, t * a.o_t + h * a.o_h + tile * CT + c, 0.0f);
  }
}

template <int D, int DT, int CT>
static int launch_recurrent(const Args& a, const char* what, hipStream_t stream) {
  const int64_t grid = (int64_t)a.batch * a.heads * (D / CT);
  S8KV_REQUIRE(grid < (int64_t(1) << 31), S8KV_ERR_INVALID, "%s: too many (sequence, head) pairs", what);
  hipLaunchKernelGGL((recurrent_kernel<D, DT, CT>), dim3((unsigned)grid), dim3(256), 0, stream, a);
  return check_launch(what);
}

template <int DT>
static int launch(const Args& a, int head_dim, const char* what, hipStream_t stream) {
  switch (head_dim) {
    case 32: return launch_recurrent<32, DT, 32>(a, what, stream);
    case 64: return launch_recurrent<64, DT, 64>(a, what, stream);
    case 128: return launch_recurrent<128, DT, 128>(a, what, stream);
    case 256: return launch_recurrent<256, DT, 64>(a, what, stream);
  }
  return S8KV_ERR_UNSUPPORTED;
}

static int fill(Args& a, const char* what, const void* q, int64_t q_t, int64_t q_h, const void* k, int64_t k_t,
                int64_t k_h, const void* v, int64_t v_t, int64_t v_h, int64_t tokens, int num_q_heads,
                int num_kv_heads, int head_dim, int dtype, const float* log_decay, float* state, int64_t state_slot,
                int64_t num_slots, const int32_t* slots, const uint8_t* reset, int batch, float scale, void* out,
                int64_t o_t, int64_t o_h) {
  S8KV_REQUIRE(batch >= 0 && tokens >= 0, S8KV_ERR_INVALID, "%s: %d sequences, %lld tokens", what, batch,
               (long long)tokens);
  S8KV_REQUIRE(num_q_heads > 0 && num_kv_heads > 0 && num_q_heads % num_kv_heads == 0, S8KV_ERR_INVALID,
               "%s: %d q heads are not a multiple of %d kv heads", what, num_q_heads, num_kv_heads);
  S8KV_REQUIRE(head_dim_ok(head_dim), S8KV_ERR_UNSUPPORTED, "%s: head_dim %d not in {32,64,128,256}", what, head_dim);
  S8KV_REQUIRE(dtype == 0 || dtype == 1, S8KV_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  S8KV_REQUIRE(num_slots >= 0 && state_slot >= (int64_t)num_q_heads * head_dim * head_dim, S8KV_ERR_INVALID,
               "%s: state slots of %lld elements do not hold %d heads of %d x %d", what, (long long)state_slot,
               num_q_heads, head_dim, head_dim);
  S8KV_REQUIRE(batch == 0 || tokens == 0 || (q && k && v && log_decay && out), S8KV_ERR_INVALID, "%s: null pointer", what);
  S8KV_REQUIRE(num_slots == 0 || state, S8KV_ERR_INVALID, "%s: null state", what);
  S8KV_REQUIRE((uintptr_t)state % 16 == 0 && state_slot % 4 == 0, S8KV_ERR_INVALID,
               "%s: state slots must be 16-byte aligned", what);
  a = Args{q, k, v, q_t, q_h, k_t, k_h, v_t, v_h, out, o_t, o_h, tokens, batch, num_q_heads,
           num_q_heads / num_kv_heads, log_decay, state, state_slot, num_slots, slots, reset, nullptr, scale};
  return S8KV_OK;
}

}  // namespace linear
}  // namespace s8kv

using namespace s8kv;

extern "C" int s8kv_linear_attn_varlen(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
                                       int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                                       int64_t v_stride_h, int64_t num_tokens, int num_q_heads, int num_kv_heads,
                                       int head_dim, int dtype, const float* log_decay, float* state,
                                       int64_t state_stride_slot, int64_t num_slots, const int32_t* state_slots,
                                       const uint8_t* reset, const int32_t* cu_seqlens, int batch, int max_seqlen,
                                       float scale, void* out, int64_t out_stride_t, int64_t out_stride_h,
                                       void* workspace, int64_t workspace_bytes, void* stream) {
  linear::Args a{};
  const char* what = "s8kv_linear_attn_varlen";
  if (int rc = linear::fill(a, what, q, q_stride_t, q_stride_h, k, k_stride_t, k_stride_h, v, v_stride_t, v_stride_h,
                            num_tokens, num_q_heads, num_kv_heads, head_dim, dtype, log_decay, state,
                            state_stride_slot, num_slots, state_slots, reset, batch, scale, out, out_stride_t,
                            out_stride_h))
    return rc;
  S8KV_REQUIRE(batch == 0 || cu_seqlens, S8KV_ERR_INVALID, "%s: null pointer", what);
  S8KV_REQUIRE(max_seqlen >= 0, S8KV_ERR_INVALID, "%s: max_seqlen < 0", what);
  (void)workspace;
  (void)workspace_bytes;
  a.cu = cu_seqlens;
  if (batch == 0 || (num_tokens == 0 && !reset)) return S8KV_OK;
  return dtype == 0 ? linear::launch<0>(a, head_dim, what, (hipStream_t)stream)
                    : linear::launch<1>(a, head_dim, what, (hipStream_t)stream);
}

extern "C" int64_t s8kv_linear_attn_workspace_size(int batch, int num_q_heads, int head_dim, int max_seqlen) {
  (void)batch; (void)num_q_heads; (void)head_dim; (void)max_seqlen;
  return 0;
}

extern "C" int s8kv_linear_attn_decode(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* k,
                                       int64_t k_stride_b, int64_t k_stride_h, const void* v, int64_t v_stride_b,
                                       int64_t v_stride_h, int batch, int num_q_heads, int num_kv_heads, int head_dim,
                                       int dtype, const float* log_decay, float* state, int64_t state_stride_slot,
                                       int64_t num_slots, const int32_t* state_slots, const uint8_t* reset,
                                       float scale, void* out, int64_t out_stride_b, int64_t out_stride_h,
                                       void* stream) {
  linear::Args a{};
  const char* what = "s8kv_linear_attn_decode";
  if (int rc = linear::fill(a, what, q, q_stride_b, q_stride_h, k, k_stride_b, k_stride_h, v, v_stride_b, v_stride_h,
                            batch, num_q_heads, num_kv_heads, head_dim, dtype, log_decay, state, state_stride_slot,
                            num_slots, state_slots, reset, batch, scale, out, out_stride_b, out_stride_h))
    return rc;
  if (batch == 0) return S8KV_OK;
  return dtype == 0 ? linear::launch<0>(a, head_dim, what, (hipStream_t)stream)
                    : linear::launch<1>(a, head_dim, what, (hipStream_t)stream);
}
