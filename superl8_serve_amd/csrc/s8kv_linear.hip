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
  // the chunked form: segments a sequence may have, their tokens, their states
  int num_seg, seg_len;
  float* parts;  // [batch][heads][num_seg][D][D]
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

// ---------------------------------------------------------------------------
// The chunked form, on the matrix cores
// ---------------------------------------------------------------------------
// Tokens i, j of a chunk of n (row i' = C - n + i of C: short chunks are
// padded in front, so that every power of lambda below is the same in all):
//   o_i = scale (sum_{j <= i} lambda^{i-j} (q_i . k_j) v_j + lambda^{i+1} q_i^T S),
//   S <- lambda^n S + sum_j lambda^{n-1-j} k_j v_j^T.
// A workgroup walks a sequence's (or a segment's) chunks for one head, its
// D / 32 waves side by side over the value dims: a wave keeps its 32 columns
// of S in fp32 accumulators, where they are the first operand of q^T S as
// they stand (the accumulators' key dims come in groups of four, and q is
// read in the same order).  The chunk's q, k, v go through LDS once; the next
// chunk's loads are in flight meanwhile.  The C x C scores are made by up to
// three waves, one 32 x 32 tile on or below the diagonal each, and shared
// through LDS.  C is 64; 32 at head_dim 256, whose columns of S take 128
// registers a lane.
//
// Operands of the 16-bit MFMAs that are fp32 values -- the decayed scores, S,
// and the decayed v of the update -- go in as two halves, hi + lo (fp16
// within 2^-22, bf16 within 2^-18 of the value), so that the state keeps fp32
// grade and the output's only visible rounding is its last one; q, k and v
// themselves are exact.  fp16 halves only reach from 2^-24 to 65504: scores,
// state and values are scaled by powers of two that bring a bound of their
// size to 2^15 (the scores: from the chunk's largest |q| and |k|; S: its
// largest value; v and with it S as it is kept: the largest |v|, changed only
// when a chunk's leaves [2^4, 2^15]).
//
// A masked score is zero, but zero times an infinite or NaN v of a later
// token is not: a chunk with a non-finite value is redone token by token.
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

template <int D>
constexpr int kChunk = D == 256 ? 32 : 64;

template <int DT>
__device__ __forceinline__ float16_t mfma(u32x4_t a, u32x4_t b, float16_t c) {
  if constexpr (DT == 0)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {  // round to nearest even
  if constexpr (DT == 0) return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{a, b}, half2_t));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(float2_t{a, b}, bf16x2_t));
}
template <int DT>
__device__ __forceinline__ float first(uint32_t w) {
  if constexpr (DT == 0) return (float)__builtin_bit_cast(half2_t, w)[0];
  else return __builtin_bit_cast(float, w << 16);
}
template <int DT>
__device__ __forceinline__ float second(uint32_t w) {
  if constexpr (DT == 0) return (float)__builtin_bit_cast(half2_t, w)[1];
  else return __builtin_bit_cast(float, w & 0xFFFF0000u);
}
template <int DT>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack2<DT>(a, b);
  lo = pack2<DT>(a - first<DT>(hi), b - second<DT>(hi));
}
__device__ __forceinline__ uint32_t pk_max(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
// Both halves' maxima over the wave (a maximum does not mind meeting a lane twice).
__device__ __forceinline__ uint32_t wave_pk_max(uint32_t m) {
  m = pk_max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, false));   // lane ^ 1
  m = pk_max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, false));   // lane ^ 2
  m = pk_max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x141, 0xF, 0xF, false));  // mirrored in 8
  m = pk_max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x140, 0xF, 0xF, false));  // mirrored in 16
  const auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  m = pk_max((uint32_t)a[0], (uint32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  return pk_max((uint32_t)b[0], (uint32_t)b[1]);
}
// The magnitude that 16 bits stand for (sign cleared), the largest finite one for inf and NaN.
template <int DT>
__device__ __forceinline__ float magnitude(uint32_t bits) {
  if constexpr (DT == 0) return (float)__builtin_bit_cast(_Float16, (uint16_t)min(bits, 0x7BFFu));
  else return __builtin_bit_cast(float, min(bits, 0x7F7Fu) << 16);
}
// e such that values up to `bound` times 2^-e are below 2^top.
__device__ __forceinline__ int excess(float bound, int top) {
  return min(100, max(-100, (int)((__builtin_bit_cast(uint32_t, bound) >> 23) & 0xFFu) - 126 - top));
}
__device__ __forceinline__ float times_pow2(float x, int e) { return __builtin_amdgcn_ldexpf(x, e); }

// Segments of a sequence of `len` tokens: seg_len tokens each, the last one takes the rest.
__device__ __forceinline__ int segments(const Args& a, int64_t len) {
  const int64_t n = (len + a.seg_len - 1) / a.seg_len;
  return (int)min(max(n, (int64_t)1), (int64_t)a.num_seg);
}

// OUT: outputs (from the segments' start states, where a sequence has
// several) and the final state.  Else a segment's own contribution to the
// state, from zero, for scan_kernel.
template <int D, int DT, bool OUT>
__global__ __launch_bounds__(2 * D, 2) void chunk_kernel(Args a) {
  constexpr int NW = D / 32, NT = 64 * NW, KT = D / 32;
  constexpr int C = kChunk<D>, IT = C / 32, T = C / 16;  // its 32-token tiles and 16-token steps
  constexpr int QP = 2 * D + 16, KP = 2 * D + 32, PP = 2 * C + 16;  // row pitches that spread a read's rows over the banks
  constexpr int KO = OUT ? C * QP : 0, VO = KO + C * KP, PO = VO + C * KP, MO = PO + (OUT ? 2 * C * PP : 0);
  constexpr int LO = MO + (8 * NW + 15) / 16 * 16;  // lambda^0 .. lambda^C, then lambda^(C - 1) .. lambda^0
  constexpr int LR = LO + 4 * (C + 4);
  __shared__ __attribute__((aligned(16))) char lds[LR + 4 * C];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5, li = lane & 15;

  const int h = blockIdx.x % a.heads;
  const int seg = blockIdx.x / a.heads % a.num_seg;
  const int b = blockIdx.x / a.heads / a.num_seg;
  int64_t first_t, last_t;
  extent(a, b, first_t, last_t);
  const int slot = a.slots ? a.slots[b] : b;
  const bool live = slot >= 0 && slot < a.num_slots;
  const int nseg = segments(a, last_t - first_t);
  char* const out = static_cast<char*>(a.out);
  if (OUT && seg == 0 && a.cu) {  // rows behind the last sequence: zeros, shared out over the sequences' workgroups
    const int64_t end = min(max((int64_t)a.cu[a.batch], (int64_t)0), a.tokens);
    for (int64_t t = end + b; t < a.tokens; t += a.batch)
      for (int c = tid; c < D; c += NT) store1<DT>(a.out, t * a.o_t + h * a.o_h + c, 0.0f);
  }
  if (seg >= nseg || (!OUT && seg == nseg - 1)) return;
  int64_t pos = first_t + seg * (int64_t)a.seg_len;
  const int64_t end = seg == nseg - 1 ? last_t : pos + a.seg_len;
  if (!live) {
    if constexpr (OUT)
      for (int64_t t = pos; t < end; ++t)
        for (int c = tid; c < D; c += NT) store1<DT>(a.out, t * a.o_t + h * a.o_h + c, 0.0f);
    return;
  }
  const bool fresh = a.reset && a.reset[b];
  if (pos >= end && !fresh) return;
  const int hk = h / a.group;

  // ---- the state's columns 32 wv + l32: register r of tile mt is key dim 32 mt + 8 (r / 4) + 4 g + r % 4 ----
  float* const pool = a.state + slot * a.state_slot + (int64_t)h * D * D;
  float* const parts = a.parts + ((int64_t)b * a.heads + h) * a.num_seg * D * D;
  float16_t S[KT];
  {
    const float* src = nseg > 1 ? parts + (int64_t)seg * D * D : pool;
    const bool zero = !OUT || (nseg == 1 && fresh);
#pragma unroll
    for (int mt = 0; mt < KT; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        S[mt][r] = zero ? 0.0f : src[(32 * mt + 8 * (r / 4) + 4 * g + r % 4) * D + 32 * wv + l32];
  }

  // ---- powers of lambda ----
  const double gd = (double)a.log_decay[h];
  const float g2 = fmaxf((float)(gd * 1.4426950408889634), -1e5f);  // (-inf: 0 x inf would be NaN)
  float* const pw = reinterpret_cast<float*>(lds + LO);
  for (int n = tid; n <= C; n += NT) {
    const float x = exp2f(g2 * (float)n);
    pw[n] = x;
    if (n < C) reinterpret_cast<float*>(lds + LR)[C - 1 - n] = x;
  }
  int factor_len = C;
  Factor lambda_n(gd * C);

  // ---- chunk loads: 16 bytes of every 16th row a thread and tensor ----
  const int lc = tid % (D / 8), lr = tid / (D / 8);
  u32x4_t rq[T], rk[T], rv[T];
  auto load = [&](int64_t from, int len) {
    const int pad = C - len;
#pragma unroll
    for (int i = 0; i < T; ++i) {
      const int row = lr + 16 * i;
      rq[i] = rk[i] = rv[i] = u32x4_t{0, 0, 0, 0};
      if (row >= pad) {
        const int64_t t = from + row - pad;
        if constexpr (OUT) rq[i] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.q) + t * a.q_t + h * a.q_h + 8 * lc);
        rk[i] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.k) + t * a.k_t + hk * a.k_h + 8 * lc);
        rv[i] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(a.v) + t * a.v_t + hk * a.v_h + 8 * lc);
      }
    }
  };
  // operands: 8 consecutive values of a row (rows l32 of the tile), and of a column by transposed reads
  auto row8 = [&](int base, int pitch, int row, int col) {
    return *reinterpret_cast<const u32x4_t*>(lds + base + row * pitch + 2 * col);
  };
  auto col8 = [&](int base, int t, int col) {  // rows 16 t + 8 g .. + 7 of column col + l32
    const char* p = lds + base + (16 * t + 8 * g + (li >> 2)) * KP + 2 * (col + 16 * ((lane >> 4) & 1) + 4 * (li & 3));
    const u32x2_t x = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((S8KV_LDS i16x4_t*)(p)));
    const u32x2_t y = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((S8KV_LDS i16x4_t*)(p + 4 * KP)));
    return u32x4_t{x.x, x.y, y.x, y.y};
  };

  int sv = 0;  // S is kept times 2^-sv, which brings v's largest value near 2^10 (fp16)
  bool first_chunk = true;
  int64_t single_until = pos;
  int len = (int)min((int64_t)C, end - pos);
  if (pos < end) load(pos, len);
  while (pos < end) {
    // ---- stage ----
    uint32_t mq = 0, mk = 0, mv = 0;
#pragma unroll
    for (int i = 0; i < T; ++i) {
      const int row = lr + 16 * i;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if constexpr (OUT && DT == 0) {
          mq = pk_max(mq, rq[i][w] & 0x7FFF7FFFu);
          mk = pk_max(mk, rk[i][w] & 0x7FFF7FFFu);
        }
        if constexpr (OUT || DT == 0) mv = pk_max(mv, rv[i][w] & 0x7FFF7FFFu);
      }
      if constexpr (OUT) *reinterpret_cast<u32x4_t*>(lds + row * QP + 16 * lc) = rq[i];
      *reinterpret_cast<u32x4_t*>(lds + KO + row * KP + 16 * lc) = rk[i];
      *reinterpret_cast<u32x4_t*>(lds + VO + row * KP + 16 * lc) = rv[i];
    }
    if constexpr (OUT || DT == 0) {
      const uint32_t a0 = wave_pk_max((pk_max(mq, mq >> 16) & 0xFFFFu) | pk_max(mk, mk >> 16) << 16);
      const uint32_t a1 = wave_pk_max(pk_max(mv, mv >> 16));
      if (lane == 0) *reinterpret_cast<u32x2_t*>(lds + MO + 8 * wv) = u32x2_t{a0, a1};
    }
    __syncthreads();
    float qkmax = 0.0f;
    if constexpr (OUT || DT == 0) {
      uint32_t m0 = 0, m1 = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const u32x2_t m = *reinterpret_cast<const u32x2_t*>(lds + MO + 8 * w);
        m0 = pk_max(m0, m.x);
        m1 = pk_max(m1, m.y);
      }
      m0 = __builtin_amdgcn_readfirstlane((int)m0);
      m1 = __builtin_amdgcn_readfirstlane((int)m1) & 0xFFFF;
      constexpr uint32_t kInf = DT == 0 ? 0x7C00u : 0x7F80u;
      if (OUT && len > 1 && ((m0 & 0xFFFFu) >= kInf || (m0 >> 16) >= kInf || m1 >= kInf)) {
        single_until = pos + len;
        len = 1;
        __syncthreads();
        load(pos, 1);
        continue;
      }
      if constexpr (DT == 0) {
        qkmax = magnitude<0>(m0 & 0xFFFFu) * magnitude<0>(m0 >> 16);
        const float vmax = magnitude<0>(m1);
        if (first_chunk || (vmax > 0.0f && (times_pow2(vmax, -sv) < 16.0f || times_pow2(vmax, -sv) >= 32768.0f))) {
          const int now = excess(vmax, 10);
#pragma unroll
          for (int mt = 0; mt < KT; ++mt)
#pragma unroll
            for (int r = 0; r < 16; ++r) S[mt][r] = times_pow2(S[mt][r], sv - now);
          sv = now;
          first_chunk = false;
        }
      }
    }
    const int64_t next = pos + len;
    const int next_len = next < single_until ? 1 : (int)min((int64_t)C, end - next);
    if (next < end) load(next, next_len);
    if (len != factor_len) {
      factor_len = len;
      lambda_n = Factor(gd * len);
    }

    u32x4_t vf[T];  // the wave's columns of v, 8 tokens a lane
    if constexpr (OUT) {
      const int e = DT == 0 ? excess(qkmax * (float)D, 15) : 0;
      // ---- scores: rows j (key tokens), columns i; kept as P[i][j], hi and lo ----
      auto tile = [&](int it, int jt) {
        float16_t acc = {};
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
          acc = mfma<DT>(row8(KO, KP, 32 * jt + l32, 16 * ks + 8 * g), row8(0, QP, 32 * it + l32, 16 * ks + 8 * g), acc);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float p[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int ago = 32 * (it - jt) + l32 - (8 * q + 4 * g + c);
            p[c] = (DT == 0 ? times_pow2(acc[4 * q + c], -e) : acc[4 * q + c]) * pw[max(0, ago)];
            if (it == jt && ago < 0) p[c] = 0.0f;
          }
          uint32_t h0, h1, l0, l1;
          split2<DT>(p[0], p[1], h0, l0);
          split2<DT>(p[2], p[3], h1, l1);
          char* at = lds + PO + (32 * it + l32) * PP + 2 * (32 * jt + 8 * q + 4 * g);
          *reinterpret_cast<u32x2_t*>(at) = u32x2_t{h0, h1};
          *reinterpret_cast<u32x2_t*>(at + C * PP) = u32x2_t{l0, l1};
        }
      };
      if (wv == 0) tile(0, 0);
      if constexpr (IT == 2) {
        if (wv == (NW < 4 ? 0 : 1)) tile(1, 1);
        if (wv == (NW == 1 ? 0 : (NW == 2 ? 1 : 2))) tile(1, 0);
      }
      // ---- o^T = S^T q^T (rows: value dims, columns: tokens), then the tokens' decay ----
      float16_t O[IT] = {};
      int es = 0;
      if constexpr (DT == 0) {
        auto largest = [&](bool finite) {
          float m = 0.0f;
#pragma unroll
          for (int mt = 0; mt < KT; ++mt)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float x = fabsf(S[mt][r]);
              m = fmaxf(m, finite && !(x < __builtin_inff()) ? 0.0f : x);
            }
          m = fmaxf(m, xor_partner<1>(m));
          m = fmaxf(m, xor_partner<2>(m));
          m = fmaxf(m, xor_partner<4>(m));
          m = fmaxf(m, xor_partner<8>(m));
          return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, max_x32(max_x16(m)))));
        };
        float m = largest(false);
        if (m == __builtin_inff()) m = largest(true);
        es = excess(m, 15);
      }
#pragma unroll
      for (int mt = 0; mt < KT; ++mt) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          u32x4_t hi, lo;
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            uint32_t x, y;
            float s0 = S[mt][8 * s + 2 * p], s1 = S[mt][8 * s + 2 * p + 1];
            if constexpr (DT == 0) {
              s0 = times_pow2(s0, -es);
              s1 = times_pow2(s1, -es);
            }
            split2<DT>(s0, s1, x, y);
            hi[p] = x;
            lo[p] = y;
          }
#pragma unroll
          for (int it = 0; it < IT; ++it) {
            const char* qp = lds + (32 * it + l32) * QP + 2 * (32 * mt + 16 * s + 4 * g);
            const u32x2_t q0 = *reinterpret_cast<const u32x2_t*>(qp), q1 = *reinterpret_cast<const u32x2_t*>(qp + 16);
            const u32x4_t qf = {q0.x, q0.y, q1.x, q1.y};
            O[it] = mfma<DT>(hi, qf, O[it]);
            O[it] = mfma<DT>(lo, qf, O[it]);
          }
        }
      }
#pragma unroll
      for (int it = 0; it < IT; ++it) O[it] *= times_pow2(pw[max(0, 32 * it + l32 + 1 - (C - len))], es + sv - e);
      __syncthreads();
      // ---- + v^T P^T ----
#pragma unroll
      for (int t = 0; t < T; ++t) {
        vf[t] = col8(VO, t, 32 * wv);
#pragma unroll
        for (int it = 0; it < IT; ++it) {
          if (16 * t >= 32 * (it + 1)) continue;
          O[it] = mfma<DT>(vf[t], row8(PO, PP, 32 * it + l32, 16 * t + 8 * g), O[it]);
          O[it] = mfma<DT>(vf[t], row8(PO + C * PP, PP, 32 * it + l32, 16 * t + 8 * g), O[it]);
        }
      }
      const float up = times_pow2(a.scale, e);
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int row = 32 * it + l32 - (C - len);
        if (row >= 0) {
          char* p = out + 2 * ((pos + row) * a.o_t + h * a.o_h + 32 * wv + 4 * g);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<u32x2_t*>(p + 16 * q) = u32x2_t{pack2<DT>(O[it][4 * q] * up, O[it][4 * q + 1] * up),
                                                              pack2<DT>(O[it][4 * q + 2] * up, O[it][4 * q + 3] * up)};
        }
      }
    } else {
#pragma unroll
      for (int t = 0; t < T; ++t) vf[t] = col8(VO, t, 32 * wv);
    }
    // ---- S <- lambda^n S + k^T (decayed v) ----
#pragma unroll
    for (int mt = 0; mt < KT; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[mt][r] = lambda_n(S[mt][r]);
#pragma unroll
    for (int t = 0; t < T; ++t) {
      u32x4_t hi, lo;
      const float4_t* w = reinterpret_cast<const float4_t*>(lds + LR + 4 * (16 * t + 8 * g));
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        uint32_t x, y;
        split2<DT>(times_pow2(first<DT>(vf[t][p]), -sv) * w[p / 2][2 * p % 4],
                   times_pow2(second<DT>(vf[t][p]), -sv) * w[p / 2][2 * p % 4 + 1], x, y);
        hi[p] = x;
        lo[p] = y;
      }
#pragma unroll
      for (int mt = 0; mt < KT; ++mt) {
        const u32x4_t kf = col8(KO, t, 32 * mt);
        S[mt] = mfma<DT>(kf, hi, S[mt]);
        S[mt] = mfma<DT>(kf, lo, S[mt]);
      }
    }
    pos = next;
    len = next_len;
    __syncthreads();
  }
  if (OUT && seg < nseg - 1) return;
  float* dst = OUT ? pool : parts + (int64_t)(seg + 1) * D * D;
#pragma unroll
  for (int mt = 0; mt < KT; ++mt)
#pragma unroll
    for (int r = 0; r < 16; ++r) dst[(32 * mt + 8 * (r / 4) + 4 * g + r % 4) * D + 32 * wv + l32] = DT == 0 ? times_pow2(S[mt][r], sv) : S[mt][r];
}

// The segments' start states, in place over their contributions: part 0 takes
// the sequence's state, part s lambda^seg_len x part s - 1 + its own.
template <int D>
__global__ __launch_bounds__(256) void scan_kernel(Args a) {
  constexpr int TILES = D * D / 1024;
  const int tile = blockIdx.x % TILES;
  const int h = blockIdx.x / TILES % a.heads;
  const int b = blockIdx.x / TILES / a.heads;
  int64_t first_t, last_t;
  extent(a, b, first_t, last_t);
  const int slot = a.slots ? a.slots[b] : b;
  const int nseg = segments(a, last_t - first_t);
  if (nseg == 1 || slot < 0 || slot >= a.num_slots) return;
  const int64_t at = 1024 * tile + 4 * threadIdx.x;
  float* p = a.parts + ((int64_t)b * a.heads + h) * a.num_seg * D * D + at;
  const Factor lambda((double)a.log_decay[h] * a.seg_len);
  float4_t s = {0, 0, 0, 0};
  if (!(a.reset && a.reset[b])) s = *reinterpret_cast<const float4_t*>(a.state + slot * a.state_slot + (int64_t)h * D * D + at);
  *reinterpret_cast<float4_t*>(p) = s;
  for (int i = 1; i < nseg; ++i) {
    p += D * D;
    const float4_t x = *reinterpret_cast<const float4_t*>(p);
#pragma unroll
    for (int c = 0; c < 4; ++c) s[c] = lambda(s[c]) + x[c];
    *reinterpret_cast<float4_t*>(p) = s;
  }
}

template <int D, int DT>
static int launch_chunks(Args& a, const char* what, hipStream_t stream) {
  const int64_t pairs = (int64_t)a.batch * a.heads, grid = pairs * a.num_seg;
  S8KV_REQUIRE(grid < (int64_t(1) << 31) && pairs * (D * D / 1024) < (int64_t(1) << 31), S8KV_ERR_INVALID,
               "%s: too many (sequence, head) pairs", what);
  if (a.num_seg > 1) {
    hipLaunchKernelGGL((chunk_kernel<D, DT, false>), dim3((unsigned)grid), dim3(2 * D), 0, stream, a);
    hipLaunchKernelGGL((scan_kernel<D>), dim3((unsigned)(pairs * (D * D / 1024))), dim3(256), 0, stream, a);
  }
  hipLaunchKernelGGL((chunk_kernel<D, DT, true>), dim3((unsigned)grid), dim3(2 * D), 0, stream, a);
  return check_launch(what);
}

// Segments a sequence of max_seqlen tokens is split into (1: not split).
static int plan_segments(int batch, int heads, int head_dim, int max_seqlen) {
  const int64_t pairs = (int64_t)batch * heads, want = 2 * device_cus();
  if (pairs == 0 || pairs >= want / 2) return 1;
  int64_t n = want / pairs;
  const int64_t most = max_seqlen / 512;
  n = n < most ? n : most;
  return n < 1 ? 1 : (int)n;
}
static int64_t parts_bytes(int batch, int heads, int head_dim, int num_seg) {
  return num_seg <= 1 ? 0 : (int64_t)batch * heads * num_seg * head_dim * head_dim * 4;
}

template <int DT>
static int launch_varlen(Args& a, int head_dim, const char* what, hipStream_t stream) {
  auto rows = [](const void* p, int64_t t, int64_t h) { return (uintptr_t)p % 16 == 0 && t % 8 == 0 && h % 8 == 0; };
  if (!(rows(a.q, a.q_t, a.q_h) && rows(a.k, a.k_t, a.k_h) && rows(a.v, a.v_t, a.v_h) && rows(a.out, a.o_t, a.o_h)))
    return launch<DT>(a, head_dim, what, stream);
  switch (head_dim) {
    case 32: return launch_chunks<32, DT>(a, what, stream);
    case 64: return launch_chunks<64, DT>(a, what, stream);
    case 128: return launch_chunks<128, DT>(a, what, stream);
    case 256: return launch_chunks<256, DT>(a, what, stream);
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
           num_q_heads / num_kv_heads, log_decay, state, state_slot, num_slots, slots, reset, nullptr, scale, 1, 1 << 30, nullptr};
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
  a.cu = cu_seqlens;
  if (batch == 0 || (num_tokens == 0 && !reset)) return S8KV_OK;
  const int num_seg = linear::plan_segments(batch, num_q_heads, head_dim, max_seqlen);
  if (num_seg > 1 && workspace && (uintptr_t)workspace % 16 == 0 &&
      workspace_bytes >= linear::parts_bytes(batch, num_q_heads, head_dim, num_seg)) {
    a.num_seg = num_seg;
    a.seg_len = (max_seqlen / num_seg + 64) / 64 * 64;
    a.parts = static_cast<float*>(workspace);
  }
  return dtype == 0 ? linear::launch_varlen<0>(a, head_dim, what, (hipStream_t)stream)
                    : linear::launch_varlen<1>(a, head_dim, what, (hipStream_t)stream);
}

extern "C" int64_t s8kv_linear_attn_workspace_size(int batch, int num_q_heads, int head_dim, int max_seqlen) {
  if (batch <= 0 || num_q_heads <= 0 || head_dim <= 0 || max_seqlen <= 0) return 0;
  return linear::parts_bytes(batch, num_q_heads, head_dim,
                             linear::plan_segments(batch, num_q_heads, head_dim, max_seqlen));
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
