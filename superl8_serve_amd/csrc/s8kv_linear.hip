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
  int tokens, batch, heads, group;  // query heads, and of them those that share a key head
  const float* log_decay;   // [heads]
  float* state;
  int64_t state_slot, num_slots;  // elements between slots
  const int32_t* slots;   // [batch], NULL: sequence b has slot b
  const uint8_t* reset;   // [batch], NULL: none; non-zero starts from an empty state
  const int32_t* cu;      // [batch + 1], NULL: one token a sequence
  float scale;
  // the chunked form: segments a sequence may have, their tokens, their states
  int num_seg, seg_len;
  float* parts;  // [entries][heads][D][D], part_of
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

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// Tokens [first, last) of sequence b, clamped to the tensors (cu_seqlens holds 32-bit counts).
__device__ __forceinline__ void extent(const Args& a, int b, int& first, int& last) {
  first = b;
  last = b + 1;
  if (a.cu) {
    first = min(max(uniform(a.cu[b]), 0), a.tokens);
    last = min(max(uniform(a.cu[b + 1]), first), a.tokens);
  }
}
// Rows outside all sequences are zeros, shared out over the sequences' workgroups.
template <int DT>
__device__ __forceinline__ void zero_outside(const Args& a, int b, int h, int from, int cols) {
  const int before = min(max(uniform(a.cu[0]), 0), a.tokens), behind = max(before, min(max(uniform(a.cu[a.batch]), 0), a.tokens));
  for (int64_t i = b; i < a.tokens - behind + before; i += a.batch) {
    const int64_t t = i < before ? i : i - before + behind;
    for (int c = threadIdx.x; c < cols; c += blockDim.x) store1<DT>(a.out, t * a.o_t + h * a.o_h + from + c, 0.0f);
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
// hold four columns of every RG-th row of the state in registers, read once
// and written once; the columns of a row need no exchange, o is summed over the
// row groups.  Bound by the state's bytes: one token, 64 sequences x 32 heads of
// 128 39.6 us (268 MB, 6.8 TB/s: part of them stay in the memory-side cache), 64
// heads' worth of 256 203 us; one sequence x 32 heads 3.5 us, an empty launch's time.
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

  int first, last;
  extent(a, b, first, last);
  const int slot = uniform(a.slots ? a.slots[b] : b);
  const bool live = slot >= 0 && slot < a.num_slots;
  const bool fresh = live && a.reset && uniform(a.reset[b]);
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
  if (a.cu) zero_outside<DT>(a, b, h, tile * CT, CT);
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
  // fewer (sequence, head) pairs than CUs: 32 columns a workgroup, four or eight times the workgroups (one sequence x
  // 32 heads of 128: 3.5 us, 4.7 with whole heads; with more pairs whole heads read q and k once instead of four times)
  const bool few = (int64_t)a.batch * a.heads < device_cus();
  switch (head_dim) {
    case 32: return launch_recurrent<32, DT, 32>(a, what, stream);
    case 64: return launch_recurrent<64, DT, 64>(a, what, stream);
    case 128:
      if (few) return launch_recurrent<128, DT, 32>(a, what, stream);
      return launch_recurrent<128, DT, 128>(a, what, stream);
    case 256:
      if (few) return launch_recurrent<256, DT, 32>(a, what, stream);
      return launch_recurrent<256, DT, 64>(a, what, stream);
  }
  return S8KV_ERR_UNSUPPORTED;
}

// ---------------------------------------------------------------------------
// The chunked form, on the matrix cores
// ---------------------------------------------------------------------------
// Tokens i, j of a chunk of n <= C (row i' = C - n + i: short chunks are
// padded in front, so that every power of lambda below is the same in all):
//   o_i = scale (sum_{j <= i} lambda^{i-j} (q_i . k_j) v_j + lambda^{i+1} q_i^T S),
//   S <- lambda^n S + sum_j lambda^{n-1-j} k_j v_j^T.
// A workgroup walks a sequence's (or a segment's) chunks for one head, its
// D / 32 waves side by side over the value dims: a wave keeps its 32 columns
// of S in fp32 accumulators, where they are the first operand of S^T q^T as
// they stand (the accumulators' key dims come in groups of four, and LDS holds
// q's dims in that order).  The chunk's q, k, v go through LDS once; the next
// chunk's loads are in flight meanwhile.  The C x C scores are made by up to
// three waves, one 32 x 32 tile on or below the diagonal each, and exchanged
// through LDS.  C is 64; 32 at head_dim 256, whose columns of S take 128
// registers a lane, at head_dim 32, whose single wave makes the scores alone,
// and for short sequences.
//
// Operands of the 16-bit MFMAs that are fp32 values -- the decayed scores, S,
// and the decayed v of the update -- go in as two halves, hi + lo (fp16
// within 2^-22, bf16 within 2^-18 of the value; the update's bf16 v in three,
// 2^-26), so that the state keeps fp32 grade and the output's only visible
// rounding is its last one; q, k and v themselves are exact.  fp16 halves only reach from 2^-24 to 65504: scores,
// state and values are scaled by powers of two that bring their largest value
// below 2^15 (the scores': of a row of a tile; S's: of a wave's columns; v's,
// and with it the scale that S is kept at: of the chunk, changed only when a
// chunk's leaves [2^9, 2^15]).  What is 2^19 times smaller than its largest
// neighbour there starts to lose bits: the halves end at 2^-25.  (States stay
// below 2^64: their scale goes up by 2^37 under the least v, their products
// with q by 2^32 where a row's scores are zero.)
//
// What bounds it (32 heads of 128, 1.05 M (token, head) pairs): the output pass
// takes 254 us, 4.2 TB/s of q, k, v and out with the matrix cores 38 % busy, and
// 221 us when every row comes from the L2: memory and the vector instructions
// (820 a wave and chunk, most of them splits into halves) weigh the same; of 256,
// with chunks half as long, the instructions alone take 780 us of 850.
// 16-column waves (twice the waves, half the splits each): 10 % slower.
//
// A masked score is zero, but zero times an infinite or NaN v of a later
// token is not: a chunk whose v is not finite is redone token by token.
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

typedef float float16_t __attribute__((ext_vector_type(16)));

template <int D>
constexpr int kChunk = D == 64 || D == 128 ? 64 : 32;

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
// a fa, b fb as 16-bit pairs hi + lo; lo takes the exact remainder.  (fp16:
// v_fma_mixlo / mixhi would make each half in one instruction, but their
// partial writes cost wait states: the whole chunk 5.0 us instead of 5.2 this
// way, head_dim 128 with one workgroup a CU.  bf16: a dot product with (-1, 0)
// instead of the unpacking and the subtraction was 3 % slower.)
// PACKED: a and b come out of packed halves; fp16's multiply-add takes them there.
template <int DT, bool PACKED = false>
__device__ __forceinline__ void split2(float a, float fa, float b, float fb, uint32_t& hi, uint32_t& lo) {
  if constexpr (DT == 0 && PACKED) hi = pack2<DT>(__builtin_fmaf(a, fa, 0.0f), __builtin_fmaf(b, fb, 0.0f));
  else hi = pack2<DT>(a * fa, b * fb);
  asm("" : "+v"(hi));  // (the remainder reads hi as it was packed)
  lo = pack2<DT>(__builtin_fmaf(a, fa, -first<DT>(hi)), __builtin_fmaf(b, fb, -second<DT>(hi)));
}
// The same in three: what a bf16 pair leaves (2^-18) would be the state's error.
__device__ __forceinline__ void split3(float a, float fa, float b, float fb, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = pack2<1>(a * fa, b * fb);
  asm("" : "+v"(hi));
  const float ra = __builtin_fmaf(a, fa, -first<1>(hi)), rb = __builtin_fmaf(b, fb, -second<1>(hi));
  mid = pack2<1>(ra, rb);
  asm("" : "+v"(mid));
  lo = pack2<1>(ra - first<1>(mid), rb - second<1>(mid));
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
// The magnitude that fp16 bits stand for (sign cleared), the largest finite one for inf and NaN.
__device__ __forceinline__ float magnitude(uint32_t bits) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)min(bits, 0x7BFFu));
}
// e such that values up to `bound` times 2^-e are below 2^15, at least `least`.
__device__ __forceinline__ int excess(float bound, int least) {
  return min(100, max(least, (int)((__builtin_bit_cast(uint32_t, bound) >> 23) & 0xFFu) - 141));
}
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }  // |e| <= 100

// Segments of a sequence of `len` tokens: seg_len tokens each, the last one takes the rest.
__device__ __forceinline__ int segments(const Args& a, int len) {
  return min(max((int)(((unsigned)len + a.seg_len - 1) / (unsigned)a.seg_len), 1), a.num_seg);
}

// The entry of a sequence's first segment in `parts`: its segments take at
// most one more than its tokens fill, so sequences one behind the other get
// entries of their own, tokens / seg_len + batch altogether.
__device__ __forceinline__ int64_t part_of(const Args& a, int b, int first) { return first / a.seg_len + b; }

// OUT: outputs (from the segments' start states, where a sequence has
// several) and the final state.  Else a segment's own contribution to the
// state, from zero, for scan_kernel; of all its tokens, also those whose decay
// rounds to zero, since an infinite or NaN one has to arrive (leaving them out
// saved 3 % at 16,384 tokens, 32 heads of 128).
template <int D, int DT, bool OUT, int C = kChunk<D>>
__global__ __launch_bounds__(2 * D, 2) void chunk_kernel(Args a) {
  constexpr int NW = D / 32, NT = 64 * NW, KT = D / 32;
  constexpr int IT = C / 32, T = C / 16;  // its 32-token tiles and 16-token steps
  constexpr int QP = 2 * D + 16, KP = 2 * D + 32, PP = 2 * C + 16;  // row pitches that spread a read's rows over the banks
  constexpr int PH = C * PP;  // bytes of the scores' hi halves (and of lo)
  constexpr int KO = OUT ? C * QP : 0, VO = KO + C * KP, PO = VO + C * KP, EO = PO + (OUT ? 2 * PH : 0);
  constexpr int MO = EO + (OUT ? 4 * 32 * 4 : 0);  // (EO: the score rows' exponents by tile; MO: the waves' largest |v|)
  constexpr int LO = MO + (4 * NW + 15) / 16 * 16 + 128;  // 32 ones, lambda^0 .. lambda^C, then 2^-sv lambda^(C - 1) .. lambda^0
  constexpr int LR = LO + 4 * (C + 4);
  __shared__ __attribute__((aligned(16))) char lds[LR + 4 * C];
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, g = lane >> 5, li = lane & 15;

  const int h = blockIdx.x % a.heads;
  const int seg = blockIdx.x / a.heads % a.num_seg;
  const int b = blockIdx.x / a.heads / a.num_seg;
  int first_t, last_t;
  extent(a, b, first_t, last_t);
  const int slot = uniform(a.slots ? a.slots[b] : b);
  const bool live = slot >= 0 && slot < a.num_slots;
  const int nseg = segments(a, last_t - first_t);
  if (OUT && seg == 0) zero_outside<DT>(a, b, h, 0, D);
  if (seg >= nseg || (!OUT && seg == nseg - 1)) return;
  int pos = first_t + seg * a.seg_len;
  const int end = seg == nseg - 1 ? last_t : pos + a.seg_len;
  if (!live) {
    if constexpr (OUT)
      for (int64_t t = pos; t < end; ++t)
        for (int c = tid; c < D; c += NT) store1<DT>(a.out, t * a.o_t + h * a.o_h + c, 0.0f);
    return;
  }
  const bool fresh = a.reset && uniform(a.reset[b]);
  if (pos >= end && !fresh) return;
  const int hk = h / a.group;

  // ---- chunk loads through descriptors of the chunk's rows: the padding in front reads as zeros ----
  const int lc = tid % (D / 8), lr = tid / (D / 8);
  const uint32_t qs = 2 * (uint32_t)a.q_t, ks = 2 * (uint32_t)a.k_t, vs = 2 * (uint32_t)a.v_t, os = 2 * (uint32_t)a.o_t;  // row strides in bytes
  const uint32_t q_off = lr * qs + 16 * lc, k_off = lr * ks + 16 * lc, v_off = lr * vs + 16 * lc;
  u32x4_t rq[T], rk[T], rv[T];
  rsrc_t q_rows, k_rows, v_rows;
  auto aim = [&](int from, int len) {
    q_rows = make_rsrc(static_cast<const uint16_t*>(a.q) + (int64_t)from * a.q_t + h * a.q_h, (len - 1) * qs + 2 * D);
    k_rows = make_rsrc(static_cast<const uint16_t*>(a.k) + (int64_t)from * a.k_t + hk * a.k_h, (len - 1) * ks + 2 * D);
    v_rows = make_rsrc(static_cast<const uint16_t*>(a.v) + (int64_t)from * a.v_t + hk * a.v_h, (len - 1) * vs + 2 * D);
  };
  auto load_part = [&](int i, int len) {
    const uint32_t row = 16u * i - (uint32_t)(C - len);  // (a row before the first wraps to an offset past the end)
    rk[i] = bload128(k_rows, k_off + row * ks);
    rv[i] = bload128(v_rows, v_off + row * vs);
    if constexpr (OUT) rq[i] = bload128(q_rows, q_off + row * qs);
  };
  auto load = [&](int from, int len) {
    aim(from, len);
#pragma unroll
    for (int i = 0; i < T; ++i) load_part(i, len);
  };
  int single_until = pos;
  int len = min(C, end - pos);
  if (pos < end) load(pos, len);

  // ---- the state's columns 32 wv + l32: register r of tile mt is key dim 32 mt + 8 (r / 4) + 4 g + r % 4 ----
  const int64_t s_at = 4 * g * D + 32 * wv + l32;
  float* const pool = a.state + slot * a.state_slot + (int64_t)h * D * D + s_at;
  float* const parts = a.parts + ((part_of(a, b, first_t) + seg) * a.heads + h) * D * D + s_at;
  float16_t S[KT];
  if (!OUT || (nseg == 1 && fresh)) {
#pragma unroll
    for (int mt = 0; mt < KT; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[mt][r] = 0.0f;
  } else {
    const float* src = nseg > 1 ? parts : pool;
#pragma unroll
    for (int mt = 0; mt < KT; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) S[mt][r] = src[(32 * mt + 8 * (r / 4) + r % 4) * D];
  }

  // ---- powers of lambda ----
  float* const pw = reinterpret_cast<float*>(lds + LO);
  float* const left = reinterpret_cast<float*>(lds + LR);
  const double gd = (double)a.log_decay[h];
  if (tid < 32) pw[tid - 32] = 1.0f;  // (what masked scores meet)
  for (int n = tid; n <= C; n += NT) {
    const float x = (float)exp(n ? gd * n : 0.0);
    pw[n] = x;
    if (n < C) left[C - 1 - n] = x;
  }
  // lambda^C is applied as its fp32 value, whose rounding is made good 16 applications at a time
  const Factor lambda_c(gd * C);
  const float drift = lambda_c.hi > 0.0f ? 16.0f * lambda_c.lo / lambda_c.hi : 0.0f;
  int applied = 0;

  // operands: 8 values of a row (row l32 of the tile) and of a column (by
  // transposed reads).  q rows hold their dims in the order of S's
  // accumulators: of 16 dims 0-3, 8-11, 4-7, 12-15, so lane group g's eight are
  // 4 g .. + 3 and 8 + 4 g .. + 3; k's are read to match.
  auto q8 = [&](int it, int s) { return *reinterpret_cast<const u32x4_t*>(lds + (32 * it + l32) * QP + 32 * s + 16 * g); };
  auto k8 = [&](int jt, int s) {
    const char* p = lds + KO + (32 * jt + l32) * KP + 32 * s + 8 * g;
    const u32x2_t x = *reinterpret_cast<const u32x2_t*>(p), y = *reinterpret_cast<const u32x2_t*>(p + 16);
    return u32x4_t{x.x, x.y, y.x, y.y};
  };
  auto p8 = [&](int lo, int it, int t) {
    return *reinterpret_cast<const u32x4_t*>(lds + PO + lo * PH + (32 * it + l32) * PP + 32 * t + 16 * g);
  };
  auto col8 = [&](int base, int t, int col) {  // rows 16 t + 8 g .. + 7 of column col + l32
    const char* p = lds + base + (16 * t + 8 * g + (li >> 2)) * KP + 2 * (col + 16 * ((lane >> 4) & 1) + 4 * (li & 3));
    const u32x2_t x = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((S8KV_LDS i16x4_t*)(p)));
    const u32x2_t y = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((S8KV_LDS i16x4_t*)(p + 4 * KP)));
    return u32x4_t{x.x, x.y, y.x, y.y};
  };

  int sv = 0;  // S is kept times 2^-sv, which brings v's largest value near 2^13 (fp16)
  // the wave's score tile: (0, 0), (1, 1) and (1, 0) by wave; waves without one make one that is not read
  constexpr bool TURNS = IT == 2;  // (a chunk of one tile: its scores are the first wave's, ahead of the others' work)
  const int my_at = NW == 2 ? 2 * wv : (wv < 3 ? wv : 3);
  const int my_it = my_at == 1 || my_at == 2, my_jt = my_at == 1 || my_at == 3;
  // (vmcnt 0: with the state's loads still counted as outstanding at the loop's head, the compiler waits for the
  // loop's own loads where it overwrites registers that held the state's)
  __builtin_amdgcn_s_waitcnt(0x0F70);
  // A bound of the wave's finite |S|: the largest at first, then decayed and
  // raised by what each chunk can have added.
  auto largest = [&]() {
    uint32_t m = 0;
#pragma unroll
    for (int mt = 0; mt < KT; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float v = S[mt][r];  // (a copy: bit_cast of a vector's element reads element 0)
        const uint32_t x = __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu;
        m = max(m, x < 0x7F800000u ? x : 0u);
      }
    auto wider = [&](float y) { m = max(m, __builtin_bit_cast(uint32_t, y)); };
    auto f = [&]() { return __builtin_bit_cast(float, m); };
    wider(xor_partner<1>(f()));
    wider(xor_partner<2>(f()));
    wider(xor_partner<4>(f()));
    wider(xor_partner<8>(f()));
    const auto x = __builtin_amdgcn_permlane16_swap(m, m, false, false);
    m = max((uint32_t)x[0], (uint32_t)x[1]);
    const auto y = __builtin_amdgcn_permlane32_swap(m, m, false, false);
    return __builtin_bit_cast(float, uniform((int)max((uint32_t)y[0], (uint32_t)y[1])));
  };
  float s_bound = 0.0f;
  if constexpr (OUT && DT == 0) s_bound = largest();
  while (pos < end) {
    // ---- stage ----
    uint32_t mv = 0, mk = 0;
#pragma unroll
    for (int i = 0; i < T; ++i) {
      const int row = lr + 16 * i;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if constexpr (OUT || DT == 0) mv = pk_max(mv, rv[i][w] & 0x7FFF7FFFu);
        if constexpr (OUT && DT == 0) mk = pk_max(mk, rk[i][w] & 0x7FFF7FFFu);
      }
      if constexpr (OUT) {
        char* q = lds + row * QP + 32 * (lc / 2) + 8 * (lc % 2);
        *reinterpret_cast<u32x2_t*>(q) = u32x2_t{rq[i][0], rq[i][1]};
        *reinterpret_cast<u32x2_t*>(q + 16) = u32x2_t{rq[i][2], rq[i][3]};
      }
      *reinterpret_cast<u32x4_t*>(lds + KO + row * KP + 16 * lc) = rk[i];
      *reinterpret_cast<u32x4_t*>(lds + VO + row * KP + 16 * lc) = rv[i];
    }
    if constexpr (OUT || DT == 0) {
      mv = wave_pk_max((pk_max(mv, mv >> 16) & 0xFFFFu) | pk_max(mk, mk << 16) & 0xFFFF0000u);
      if (lane == 0) *reinterpret_cast<uint32_t*>(lds + MO + 4 * wv) = mv;
    }
    __syncthreads();
    float kv_max = 0.0f;  // what the chunk can add to a value of S
    if constexpr (OUT || DT == 0) {
      uint32_t m = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) m = pk_max(m, *reinterpret_cast<const uint32_t*>(lds + MO + 4 * w));
      m = (uint32_t)uniform((int)m);
      if constexpr (OUT && DT == 0) kv_max = (float)C * magnitude(m >> 16) * magnitude(m & 0xFFFFu);
      m &= 0xFFFFu;
      if (OUT && len > 1 && m >= (DT == 0 ? 0x7C00u : 0x7F80u)) {
        single_until = pos + len;
        len = 1;
        __syncthreads();
        load(pos, 1);
        __builtin_amdgcn_s_waitcnt(0x0F70);  // (as before the loop)
        continue;
      }
      if constexpr (DT == 0) {
        const float vmax = magnitude(m), now_v = vmax * pow2(-sv);
        if (vmax > 0.0f && (now_v < 512.0f || now_v >= 32768.0f)) {
          const int now = excess(vmax, -100) + 1;
#pragma unroll
          for (int mt = 0; mt < KT; ++mt) S[mt] = S[mt] * pow2(sv) * pow2(-now);
          s_bound = s_bound * pow2(sv) * pow2(-now);
          sv = now;
          for (int n = tid; n < C; n += NT) left[n] = pw[C - 1 - n] * pow2(-sv);
          __syncthreads();
        }
      }
    }
    const int next = pos + len;
    const int next_len = next < single_until ? 1 : min(C, end - next);
    const bool more = next < end;
    aim(more ? next : pos, more ? next_len : len);

    u32x4_t vf[T];  // the wave's columns of v, 8 tokens a lane
    float16_t O[IT] = {}, P = {};
    const int es = DT == 0 ? excess(s_bound, -100) : 0;
    const float lambda_n = pw[len];
    float down = 1.0f;
    // A tile of the scores (rows j: key tokens, columns i), done in three
    // parts: its MFMAs; the mask and the rows' exponents; P[i][j] of four
    // times eight key tokens, hi and lo.
    auto masked = [&](float16_t& acc, int diag, int at) {
      const int lim = diag ? l32 : C;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (lim < 8 * (r / 4) + 4 * g + r % 4) acc[r] = 0.0f;
      if constexpr (DT == 0) {
        uint32_t m = 0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float x = acc[r];
          m = max(m, __builtin_bit_cast(uint32_t, x) & 0x7FFFFFFFu);
        }
        const auto x = __builtin_amdgcn_permlane32_swap(m, m, false, false);
        // (products of fp16 values are 2^-48 or more; a row of zeros must not drive its exponent further)
        const int e = excess(__builtin_bit_cast(float, max((uint32_t)x[0], (uint32_t)x[1])), -32);
        down = pow2(-e);
        reinterpret_cast<int*>(lds + EO)[32 * at + l32] = e;
      }
    };
    auto exchanged = [&](const float16_t& acc, int it, int jt, int q) {
      const float* d = pw + 32 * (it - jt) + l32 - 4 * g - 8 * q;
      uint32_t h0, h1, l0, l1;
      split2<DT>(acc[4 * q], d[0] * down, acc[4 * q + 1], d[-1] * down, h0, l0);
      split2<DT>(acc[4 * q + 2], d[-2] * down, acc[4 * q + 3], d[-3] * down, h1, l1);
      char* to = lds + PO + (32 * it + l32) * PP + 2 * (32 * jt + 8 * q + 4 * g);
      *reinterpret_cast<u32x2_t*>(to) = u32x2_t{h0, h1};
      *reinterpret_cast<u32x2_t*>(to + PH) = u32x2_t{l0, l1};
    };
    if constexpr (OUT) {
      if constexpr (!TURNS || NW < 3) {  // the tile that no wave has a turn for below
        auto tile = [&](int it, int jt, int at) {
          float16_t acc = {};
#pragma unroll
          for (int s = 0; s < D / 16; ++s) acc = mfma<DT>(k8(jt, s), q8(it, s), acc);
          masked(acc, it == jt, at);
#pragma unroll
          for (int q = 0; q < 4; ++q) exchanged(acc, it, jt, q);
        };
        if (wv == 0) tile(TURNS, TURNS, TURNS);
      }
      // ---- o^T = S^T q^T (rows: value dims, columns: tokens), and the wave's score tile ----
      const float s_down = pow2(-es);
      u32x4_t qf[2][IT], hi[2], lo[2];
      auto halves = [&](int s) {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          uint32_t x, y;
          split2<DT>(S[s / 2][8 * (s % 2) + 2 * p], s_down, S[s / 2][8 * (s % 2) + 2 * p + 1], s_down, x, y);
          hi[s % 2][p] = x;
          lo[s % 2][p] = y;
        }
      };
      // one step's reads and halves ahead, and S's decay behind, in the shadow of the step's MFMAs
      u32x4_t kp[2];
#pragma unroll
      for (int it = 0; it < IT; ++it) qf[0][it] = q8(it, 0);
      if constexpr (TURNS) kp[0] = k8(my_jt, 0);
      halves(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < 2 * KT; ++s) {
        u32x4_t qp = qf[s % 2][0];
        if constexpr (IT == 2) {
#pragma unroll
          for (int w = 0; w < 4; ++w) qp[w] = my_it ? qf[s % 2][1][w] : qf[s % 2][0][w];
        }
        if (s + 1 < 2 * KT) {
#pragma unroll
          for (int it = 0; it < IT; ++it) qf[(s + 1) % 2][it] = q8(it, s + 1);
          if constexpr (TURNS) kp[(s + 1) % 2] = k8(my_jt, s + 1);
          halves(s + 1);
        } else {
#pragma unroll
          for (int t = 0; t < T; ++t) vf[t] = col8(VO, t, 32 * wv);
        }
        if (s % 2) S[s / 2] *= lambda_n;
#pragma unroll
        for (int it = 0; it < IT; ++it) O[it] = mfma<DT>(hi[s % 2], qf[s % 2][it], O[it]);
#pragma unroll
        for (int it = 0; it < IT; ++it) O[it] = mfma<DT>(lo[s % 2], qf[s % 2][it], O[it]);
        if constexpr (TURNS) P = mfma<DT>(kp[s % 2], qp, P);
        if (s + 1 < 2 * KT) __builtin_amdgcn_sched_group_barrier(0x100, TURNS ? IT + 2 : IT, 0);
        else __builtin_amdgcn_sched_group_barrier(0x100, 2 * T, 0);
#pragma unroll
        for (int n = 0; n < 2 * IT + TURNS; ++n) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, IT == 2 ? 9 : 14, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int mt = 0; mt < KT; ++mt) S[mt] *= lambda_n;
#pragma unroll
      for (int t = 0; t < T; ++t) vf[t] = col8(VO, t, 32 * wv);
    }
    // ---- S <- lambda^n S (done) + k^T (decayed v), the tile's exchange, and the next chunk's loads ----
    if (++applied == 16) {
      applied = 0;
#pragma unroll
      for (int mt = 0; mt < KT; ++mt)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[mt][r] = __builtin_fmaf(S[mt][r], drift, S[mt][r]);
    }
    constexpr int KB = KT < 2 ? KT : 2, KN = KT / KB, N = T * KN;  // key tiles a batch of reads, batches a step, batches
    constexpr int VN = DT == 0 ? 2 : 3;
    u32x4_t kf[2][KB], vp[VN][2];
    auto decayed = [&](int t) {
      const float4_t* w = reinterpret_cast<const float4_t*>(left + 16 * t + 8 * g);
      const float4_t w0 = w[0], w1 = w[1];
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float v0 = first<DT>(vf[t][p]), v1 = second<DT>(vf[t][p]);
        const float f0 = p < 2 ? w0[2 * p] : w1[2 * p - 4], f1 = p < 2 ? w0[2 * p + 1] : w1[2 * p - 3];
        uint32_t x, y;
        if constexpr (DT == 0) {
          split2<DT, true>(v0, f0, v1, f1, x, y);
        } else {
          uint32_t z;
          split3(v0, f0, v1, f1, x, y, z);
          vp[2][t % 2][p] = z;
        }
        vp[0][t % 2][p] = x;
        vp[1][t % 2][p] = y;
      }
    };
#pragma unroll
    for (int m = 0; m < KB; ++m) kf[0][m] = col8(KO, 0, 32 * m);
    decayed(0);
    if constexpr (OUT && TURNS) masked(P, my_it == my_jt, my_at);
    __builtin_amdgcn_sched_barrier(0);
    // (without a next chunk the descriptors are the present one's: the loads come to nothing, but their number is known)
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int t = n / KN, m0 = n % KN * KB;
#pragma unroll
      for (int i = 0; i < T; ++i)
        if (i * N / T == n) load_part(i, next_len);
      if (n + 1 < N) {
#pragma unroll
        for (int m = 0; m < KB; ++m) kf[(n + 1) % 2][m] = col8(KO, (n + 1) / KN, 32 * ((n + 1) % KN * KB + m));
        if ((n + 1) % KN == 0) decayed(t + 1);
      }
      if constexpr (OUT && TURNS) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q * N / 4 == n) exchanged(P, my_it, my_jt, q);
      }
#pragma unroll
      for (int i = 0; i < VN; ++i)
#pragma unroll
        for (int m = 0; m < KB; ++m) S[m0 + m] = mfma<DT>(kf[n % 2][m], vp[i][t % 2], S[m0 + m]);
      __builtin_amdgcn_sched_group_barrier(0x100, 2 * KB + 4, 0);
#pragma unroll
      for (int m = 0; m < VN * KB; ++m) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (OUT) {
      __syncthreads();
      // ---- times the tokens' decay, + v^T P^T ----
      const rsrc_t out_rows = make_rsrc(static_cast<uint16_t*>(a.out) + (int64_t)pos * a.o_t + h * a.o_h, (len - 1) * os + 2 * D);
      int e[IT], e1 = 0;  // the scores' exponents: of a row's first tile, and of its diagonal tile behind it
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        e[it] = 0;
        if constexpr (DT == 0) {
          const int* ex = reinterpret_cast<const int*>(lds + EO) + l32;
          e[it] = ex[it == 0 ? 0 : 64];
          if (it == 1) e1 = ex[32];
        }
        O[it] *= __builtin_amdgcn_ldexpf(pw[max(0, 32 * it + l32 + 1 - (C - len))], es + sv - e[it]);
      }
#pragma unroll
      for (int t = 0; t < T; ++t) {
        if (DT == 0 && t == 2) {
          O[IT - 1] *= __builtin_amdgcn_ldexpf(1.0f, e[IT - 1] - e1);
          e[IT - 1] = e1;
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
          for (int it = t / 2; it < IT; ++it) O[it] = mfma<DT>(vf[t], p8(half, it, t), O[it]);
      }
      if constexpr (DT == 0) {
        // (every 16 chunks the largest itself: the bound only grows in between, and what it has too much of costs bits)
        s_bound = applied ? s_bound * lambda_n + kv_max * pow2(-sv) : largest();
      }
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const float up = __builtin_amdgcn_ldexpf(a.scale, e[it]);
        // a lane pair (l, l + 32) holds value dims 8 q + 0 .. 3 and 4 .. 7 of a token; it trades two q's halves for 16-byte stores
        const uint32_t o = (uint32_t)(32 * it + l32 - (C - len)) * os + 2 * (32 * wv + 8 * g);  // (padding: past the end)
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          const auto x = __builtin_amdgcn_permlane32_swap(pack2<DT>(O[it][4 * q] * up, O[it][4 * q + 1] * up),
                                                          pack2<DT>(O[it][4 * q + 4] * up, O[it][4 * q + 5] * up), false, false);
          const auto y = __builtin_amdgcn_permlane32_swap(pack2<DT>(O[it][4 * q + 2] * up, O[it][4 * q + 3] * up),
                                                          pack2<DT>(O[it][4 * q + 6] * up, O[it][4 * q + 7] * up), false, false);
          bstore128(u32x4_t{(uint32_t)x[0], (uint32_t)y[0], (uint32_t)x[1], (uint32_t)y[1]}, out_rows, o + 16 * q);
        }
      }
    }
    pos = next;
    len = next_len;
    __syncthreads();
  }
  if (OUT && seg < nseg - 1) return;
  float* dst = OUT ? pool : parts + (int64_t)a.heads * D * D;  // (the next segment's start)
#pragma unroll
  for (int mt = 0; mt < KT; ++mt)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      dst[(32 * mt + 8 * (r / 4) + r % 4) * D] = DT == 0 ? __builtin_amdgcn_ldexpf(S[mt][r], sv) : S[mt][r];
}

// The segments' start states, in place over their contributions: part 0 takes
// the sequence's state, part s lambda^seg_len x part s - 1 + its own.  A thread
// takes four values of all of them (16 segments x 32 heads of 128: 12 us, 67 MB).
template <int D>
__global__ __launch_bounds__(256) void scan_kernel(Args a) {
  constexpr int TILES = D * D / 1024;
  const int tile = blockIdx.x % TILES;
  const int h = blockIdx.x / TILES % a.heads;
  const int b = blockIdx.x / TILES / a.heads;
  int first_t, last_t;
  extent(a, b, first_t, last_t);
  const int slot = uniform(a.slots ? a.slots[b] : b);
  const int nseg = segments(a, last_t - first_t);
  if (nseg == 1 || slot < 0 || slot >= a.num_slots) return;
  const int64_t at = 1024 * tile + 4 * threadIdx.x;
  float* p = a.parts + (part_of(a, b, first_t) * a.heads + h) * D * D + at;
  const Factor lambda((double)a.log_decay[h] * a.seg_len);
  float4_t s = {0, 0, 0, 0};
  if (!(a.reset && a.reset[b])) s = *reinterpret_cast<const float4_t*>(a.state + slot * a.state_slot + (int64_t)h * D * D + at);
  *reinterpret_cast<float4_t*>(p) = s;
  for (int i = 1; i < nseg; ++i) {
    p += (int64_t)a.heads * D * D;
    const float4_t x = *reinterpret_cast<const float4_t*>(p);
#pragma unroll
    for (int c = 0; c < 4; ++c) s[c] = lambda(s[c]) + x[c];
    *reinterpret_cast<float4_t*>(p) = s;
  }
}

template <int D, int DT>
static int launch_chunks(Args& a, int max_seqlen, const char* what, hipStream_t stream) {
  const int64_t pairs = (int64_t)a.batch * a.heads, grid = pairs * a.num_seg;
  S8KV_REQUIRE(grid < (int64_t(1) << 31) && pairs * (D * D / 1024) < (int64_t(1) << 31), S8KV_ERR_INVALID,
               "%s: too many (sequence, head) pairs", what);
  if (a.num_seg > 1) {
    hipLaunchKernelGGL((chunk_kernel<D, DT, false>), dim3((unsigned)grid), dim3(2 * D), 0, stream, a);
    hipLaunchKernelGGL((scan_kernel<D>), dim3((unsigned)(pairs * (D * D / 1024))), dim3(256), 0, stream, a);
  }
  // chunks of 32 for sequences that fill no more (32 sequences x 32 heads of 64, 16 tokens: 10.1 us, 17.3 with 64; of 128
  // 29.2 / 30.6); of 64 also for short ones in numbers, since more of their workgroups fit a CU's LDS (64 sequences x 32
  // heads: 40 tokens 26.1 / 32.3, 130 tokens 42.2 / 58.3, 250 tokens 85.0 / 84.6; four sequences of 100 12.2 / 11.3)
  if (kChunk<D> > 32 && (max_seqlen <= 32 || (D == 64 && max_seqlen <= 192 && pairs >= 2 * device_cus())))
    hipLaunchKernelGGL((chunk_kernel<D, DT, true, 32>), dim3((unsigned)grid), dim3(2 * D), 0, stream, a);
  else
    hipLaunchKernelGGL((chunk_kernel<D, DT, true>), dim3((unsigned)grid), dim3(2 * D), 0, stream, a);
  return check_launch(what);
}

// Tokens of the segments that long sequences are split into (0: no split).
// A CU works off one (sequence, head) alone at nearly the rate of two side by
// side, so a batch is even enough while its longest sequence is no longer than
// the tokens a CU has to do altogether; else segments of half of those, two a
// CU.  Splitting reads k and v of all but the last segments a second time.
// Where a CU has few tokens to do, a segment's chain of chunks and the scan over
// the segments' D x D states share the time, so segments grow with the root of
// length x D; past 256 tokens the chain weighs more.  (One sequence, us, with
// 128 / 256 tokens a segment and unsplit: 512 tokens x 32 heads of 128 30.2 / 35.5 /
// 34.1, of 64 21.6 / 29.0 / 31.0; 2,048 tokens of 128 51.5 / 45.5 / 119; with
// several sequences the CUs are full at more: 2 x 1,024 of 128, 192 tokens a
// segment 50.6, 256 44.4.  Less than two and a half segments do not pay: 300
// tokens of 128 26.1 split, 23.7 not; 384 26.9 / 27.3, of 64 20.2 / 24.3.)
static int segment_tokens(int64_t tokens, int heads, int head_dim, int max_seqlen) {
  if (max_seqlen > tokens) max_seqlen = (int)tokens;  // (a graph's bucket, say)
  const int64_t share = tokens * heads * head_dim / (128 * (int64_t)device_cus());
  int64_t least = 128;
  while (least < 256 && (3 * least < 4 * share || 4 * least * least < (int64_t)max_seqlen * head_dim)) least += 64;
  if (max_seqlen <= share + share / 5 || 2 * (int64_t)max_seqlen <= 5 * least) return 0;
  const int64_t seg = share / 2 > least ? share / 2 : least;
  const int64_t n = (max_seqlen + seg - 1) / seg;
  return (int)((max_seqlen + n - 1) / n + 63) / 64 * 64;
}
template <int DT>
static int launch_varlen(Args& a, int head_dim, int max_seqlen, const char* what, hipStream_t stream) {
  // (a chunk's rows have 32-bit offsets, one bit of them for the rows that are not there: rows that share bytes with
  // the next, broadcast tokens say, would find themselves there)
  auto rows = [head_dim](const void* p, int64_t t, int64_t h) {
    return (uintptr_t)p % 16 == 0 && t % 8 == 0 && h % 8 == 0 && t >= head_dim && t < (1 << 24);
  };
  if (!(rows(a.q, a.q_t, a.q_h) && rows(a.k, a.k_t, a.k_h) && rows(a.v, a.v_t, a.v_h) && rows(a.out, a.o_t, a.o_h)))
    return launch<DT>(a, head_dim, what, stream);
  // a few tokens: the recurrence reads and writes the state at once (recurrence / chunk, 32 sequences x 32 heads of 128:
  // 5 tokens 26.8 / 27.8 us, 8 tokens 31.6 / 28.1; one sequence 6.3 / 7.9, 8.2 / 7.9; of 64: 5 tokens 10.1 / 10.0, 8
  // tokens 12.8 / 10.1; of 256: 5 tokens 105 / 106, 8 tokens 120 / 106; of 32: 4 tokens 7.1 / 6.2, one sequence 4.8 / 5.2)
  if (max_seqlen <= (head_dim == 32 ? 3 : 5)) return launch<DT>(a, head_dim, what, stream);
  switch (head_dim) {
    case 32: return launch_chunks<32, DT>(a, max_seqlen, what, stream);
    case 64: return launch_chunks<64, DT>(a, max_seqlen, what, stream);
    case 128: return launch_chunks<128, DT>(a, max_seqlen, what, stream);
    case 256: return launch_chunks<256, DT>(a, max_seqlen, what, stream);
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
  S8KV_REQUIRE(tokens < (int64_t(1) << 31), S8KV_ERR_INVALID, "%s: %lld tokens are past 32 bits", what, (long long)tokens);
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
  a = Args{q, k, v, q_t, q_h, k_t, k_h, v_t, v_h, out, o_t, o_h, (int)tokens, batch, num_q_heads,
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
  const int seg = linear::segment_tokens(num_tokens, num_q_heads, head_dim, max_seqlen);
  if (seg && workspace && (uintptr_t)workspace % 16 == 0 &&
      workspace_bytes >= s8kv_linear_attn_workspace_size(batch, num_q_heads, head_dim, num_tokens, max_seqlen)) {
    const int longest = max_seqlen < num_tokens ? max_seqlen : (int)num_tokens;
    a.num_seg = (longest + seg - 1) / seg;
    a.seg_len = seg;
    a.parts = static_cast<float*>(workspace);
  }
  return dtype == 0 ? linear::launch_varlen<0>(a, head_dim, max_seqlen, what, (hipStream_t)stream)
                    : linear::launch_varlen<1>(a, head_dim, max_seqlen, what, (hipStream_t)stream);
}

extern "C" int64_t s8kv_linear_attn_workspace_size(int batch, int num_q_heads, int head_dim, int64_t num_tokens,
                                                   int max_seqlen) {
  if (batch <= 0 || num_q_heads <= 0 || head_dim <= 0 || num_tokens <= 0 || max_seqlen <= 0) return 0;
  const int seg = linear::segment_tokens(num_tokens, num_q_heads, head_dim, max_seqlen);
  return seg ? (num_tokens / seg + batch) * num_q_heads * head_dim * head_dim * 4 : 0;
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
