// Rotary positions of q and k, alone or on the way into the paged cache.
//
// A head of D values holds R / 2 pairs (R <= D, the other dims pass through):
// (x_p, x_{p + R/2}) with half-split pairing, (x_2p, x_{2p+1}) with adjacent
// pairing.  Pair p belongs to one position axis a(p) and turns by the angle of
// that axis's position: c = table[pos_a][p], s = table[pos_a][R/2 + p],
//   (x1, x2) -> (x1 c - x2 s, x2 c + x1 s),
// two fp32 products and one fp32 add per value, each rounded by itself (no
// contraction, so that the bytes do not hang on the compiler's choice).  With
// a norm weight the head is first scaled to x r w, r = 1 / sqrt(mean(x^2) +
// eps), in fp32 with the squares added by a pairwise tree.  The result is
// rounded once, to the output's type; K rounds to fp16 and then goes the
// append's way (Hadamard, fp16, RTN int8), so the cache holds the bytes that
// the rotation followed by the append would store.
#include "s8kv_append_rows.h"
#include "s8kv_host.h"

#pragma clang fp contract(off)

namespace s8kv {
namespace rope {

constexpr int kWaves = 4;  // waves per workgroup

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

// element types: 0 fp16, 1 bf16, 2 fp32
template <int DT>
constexpr int kBytes = DT == 2 ? 4 : 2;

__device__ __forceinline__ float pin(float x) {  // keeps the product's rounding apart from what follows
  asm("" : "+v"(x));
  return x;
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
  if (dtype == 0) return (float)static_cast<const _Float16*>(p)[i];
  if (dtype == 1) return __builtin_bit_cast(float, (uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
  return static_cast<const float*>(p)[i];
}

struct Rows {  // [tokens][heads][D], unit stride on D; strides in elements
  char* p;
  int64_t st, sh;
  int heads;
  const void* norm;  // [D] weight, or NULL
};

struct Args {
  Rows q, k, v;
  char *q_out, *k_out;  // k_out may be NULL in the writing modes
  int64_t qo_t, qo_h, ko_t, ko_h;
  int64_t tokens;
  const int32_t* pos;  // [axes][tokens]
  int64_t pos_stride;
  int axes;
  uint64_t axis_map[4];  // two bits per pair
  const float* table;    // [max_pos][R]: cos of the R/2 pairs, then sin
  int64_t max_pos;
  int rot;
  int adjacent;
  int pairs_log2;  // lanes a token's pairs take: the power of two from R / 2 on, 64 at most
  int partner;  // half pairing: parts between a pair's values (1, 2, 4, 8), 0: both on one lane
  int norm_dtype;
  float eps, inv_d;
  int hpi_log2;      // heads per iteration of a wave
  int iters, per_wave;  // iterations over q, k and v heads; of them, a wave's
  // writing modes
  const int32_t* slot_mapping;
  char *k_cache, *v_cache;
  float *k_scale, *v_scale;
  const float* v_codebook;
  int64_t num_blocks;
  int block_size_log2;
  float rot_norm;
};

// The lane's 16 values of a row (or, fast path, four 16-byte words of it).
template <int DT>
struct Raw {
  u32x4_t w[DT == 2 ? 4 : 2];
};
template <int DT>
__device__ __forceinline__ Raw<DT> load_raw(const char* p) {
  Raw<DT> r;
#pragma unroll
  for (int i = 0; i < (DT == 2 ? 4 : 2); ++i) r.w[i] = reinterpret_cast<const u32x4_t*>(p)[i];
  return r;
}
template <int DT>
__device__ __forceinline__ void expand(const Raw<DT>& r, float (&x)[16]) {
  if constexpr (DT == 0) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const half8_t h = __builtin_bit_cast(half8_t, r.w[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[8 * j + i] = (float)h[i];
    }
  } else if constexpr (DT == 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t u = r.w[j / 4][j % 4];
      x[2 * j] = __builtin_bit_cast(float, u << 16);
      x[2 * j + 1] = __builtin_bit_cast(float, u & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = __builtin_bit_cast(float, (uint32_t)r.w[j / 4][j % 4]);
  }
}
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
// Stores the lane's 16 values at p.  16-bit types: lanes l and l ^ 1 (parts
// 2 g and 2 g + 1) trade halves first, so that each of the two stores writes
// whole 32-byte pieces (own halves in two stores made twice the write requests).
template <int DT>
__device__ __forceinline__ void store_part(char* p, const float (&x)[16], int lane) {
  if constexpr (DT == 2) {
    u32x4_t* o = reinterpret_cast<u32x4_t*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = u32x4_t{__builtin_bit_cast(uint32_t, x[4 * j]), __builtin_bit_cast(uint32_t, x[4 * j + 1]),
                     __builtin_bit_cast(uint32_t, x[4 * j + 2]), __builtin_bit_cast(uint32_t, x[4 * j + 3])};
  } else {
    u32x4_t w[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2_t v = {x[2 * i], x[2 * i + 1]};
      if constexpr (DT == 0) w[i / 4][i % 4] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, half2_t));
      else w[i / 4][i % 4] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
    }
    const bool odd = lane & 1;
    u32x4_t first, second;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t own0 = w[0][i], own1 = w[1][i];
      const uint32_t got = (uint32_t)__builtin_amdgcn_mov_dpp((int)(odd ? own0 : own1), 0xB1, 0xF, 0xF, false);  // lane ^ 1
      first[i] = odd ? got : own0;
      second[i] = odd ? own1 : got;
    }
    p -= odd ? 16 : 0;  // (an odd part begins 32 bytes on: its second 16 bytes of the pair's first 32)
    *reinterpret_cast<u32x4_t*>(p) = first;
    *reinterpret_cast<u32x4_t*>(p + 32) = second;
  }
}

// The table row of pair p's axis: the address of (cos, pair 0), or NULL for a
// position outside the table (its pairs become NaN; nothing is read).
__device__ __forceinline__ const float* table_row(const Args& a, int pos) {
  return pos >= 0 && (int64_t)pos < a.max_pos ? a.table + (int64_t)pos * a.rot : nullptr;
}
__device__ __forceinline__ int axis_of(const Args& a, int pair) {
  const uint64_t m = pair < 64 ? (pair < 32 ? a.axis_map[0] : a.axis_map[1]) : (pair < 96 ? a.axis_map[2] : a.axis_map[3]);
  return (int)(m >> (2 * (pair & 31))) & 3;
}
__device__ __forceinline__ int position(const Args& a, int axis, int64_t t) { return a.pos[axis * a.pos_stride + t]; }

// The cosines and sines of a wave's tokens, through the wave's part of LDS:
// each pair's two table values are read once a token, whatever the axes, and
// then by every lane that holds one of the pair's values (read straight from
// the table, 16 + 16 values a lane, the gathers of three axes took a third of
// the kernel's time).  Per token: c of the R/2 pairs, -s, s.
template <int D>
constexpr int kAngleFloats = 3 * (D / 2) * RowsLayout<D>::RPW;  // of a wave (at most RPW tokens)
template <int D>
struct Angles {
  float c[16], s[16];  // s: -s for a pair's first value, +s for its second
  bool turns;          // false: the lane's dims are past R
  static __device__ __forceinline__ void gather(const Args& a, int64_t t0, int tokens, int lane, float* lds) {
    const int half = a.rot >> 1;
    constexpr int U = 4;  // tokens whose two dependent loads are in flight together
    const int at = lane >> a.pairs_log2, first = lane & ((1 << a.pairs_log2) - 1), step = 64 >> a.pairs_log2;
    for (int pair = first; pair < half; pair += 64) {  // (more than 64 pairs: the whole wave on one token)
      const int axis = a.axes == 1 ? 0 : axis_of(a, pair);
      for (int k = at; k < tokens; k += U * step) {
        const float* row[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t t = t0 + k + u * step;
          row[u] = k + u * step < tokens && t < a.tokens ? table_row(a, position(a, axis, t)) : nullptr;
        }
        float c[U], s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          c[u] = s[u] = __builtin_nanf("");
          if (row[u]) {
            c[u] = row[u][pair];
            s[u] = row[u][half + pair];
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (k + u * step >= tokens) break;
          float* o = lds + (k + u * step) * 3 * half + pair;
          o[0] = c[u];
          o[half] = -s[u];
          o[2 * half] = s[u];
        }
      }
    }
    // (the wave's LDS instructions run in order; the fence keeps the compiler's order)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // the lane's values; `lds`: its token's
  __device__ __forceinline__ void take(const Args& a, const float* lds, int li) {
    const int half = a.rot >> 1;
    turns = 16 * li < a.rot;
    if (!turns) return;
    if (a.adjacent) {
      const float4_t* cp = reinterpret_cast<const float4_t*>(lds + 8 * li);
      const float4_t* np = reinterpret_cast<const float4_t*>(lds + half + 8 * li);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4_t cv = cp[j], nv = np[j];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          c[8 * j + 2 * i] = c[8 * j + 2 * i + 1] = cv[i];
          s[8 * j + 2 * i] = nv[i];
          s[8 * j + 2 * i + 1] = -nv[i];
        }
      }
    } else if (a.partner) {
      const int p0 = 16 * (li & (a.partner - 1));
      const float4_t* cp = reinterpret_cast<const float4_t*>(lds + p0);
      const float4_t* sp = reinterpret_cast<const float4_t*>(lds + ((li & a.partner) ? 2 * half : half) + p0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float4_t cv = cp[j], sv = sp[j];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          c[4 * j + i] = cv[i];
          s[4 * j + i] = sv[i];
        }
      }
    } else {  // R = 16: pairs (i, i + 8) of part 0
      const float4_t* cp = reinterpret_cast<const float4_t*>(lds);
      const float4_t* np = reinterpret_cast<const float4_t*>(lds + half);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4_t cv = cp[j], nv = np[j];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          c[4 * j + i] = c[8 + 4 * j + i] = cv[i];
          s[4 * j + i] = nv[i];
          s[8 + 4 * j + i] = -nv[i];
        }
      }
    }
  }
  __device__ __forceinline__ void turn(const Args& a, float (&x)[16]) const {
    float y[16];
    if (a.adjacent) {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = x[i ^ 1];
    } else if (a.partner == 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = xor_partner<1>(x[i]);
    } else if (a.partner == 2) {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = xor_partner<2>(x[i]);
    } else if (a.partner == 4) {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = xor_partner<RowsLayout<D>::LANE4>(x[i]);
    } else if (a.partner == 8) {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = xor_partner<8>(x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = x[i ^ 8];
    }
    if (a.rot == D) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = x[i] * c[i] + y[i] * s[i];
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float r = x[i] * c[i] + y[i] * s[i];
        x[i] = turns ? r : x[i];
      }
    }
  }
};

// x -> x r w: the squares add up by a pairwise tree over neighbouring dims
// (in-lane, then across the row's lanes), mean, + eps, correctly rounded
// square root and reciprocal.
template <int D>
__device__ __forceinline__ void normalise(const Args& a, const float* w, float (&x)[16]) {
  constexpr int LPR = RowsLayout<D>::LPR;
  float s[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = x[i] * x[i];
#pragma unroll
  for (int h = 1; h < 16; h <<= 1) {
#pragma unroll
    for (int i = 0; i < 16; i += 2 * h) s[i] = s[i] + s[i + h];
  }
  float t = s[0];
  if constexpr (LPR > 1) t = t + xor_partner<1>(t);
  if constexpr (LPR > 2) t = t + xor_partner<2>(t);
  if constexpr (LPR > 4) t = t + xor_partner<RowsLayout<D>::LANE4>(t);
  if constexpr (LPR > 8) t = t + xor_partner<8>(t);
  const float r = 1.0f / __builtin_sqrtf(t * a.inv_d + a.eps);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float4_t wv = reinterpret_cast<const float4_t*>(w)[j];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[4 * j + i] = x[4 * j + i] * r * wv[i];
  }
}

// A token's cache row of KV head h, or false: a negative slot or one outside
// the pool writes nothing.
__device__ __forceinline__ bool cache_row(const Args& a, int64_t t, int h, uint64_t& row) {
  const int32_t slot = a.slot_mapping[t];
  const uint32_t blk = (uint32_t)slot >> a.block_size_log2;
  row = (((uint64_t)blk * (uint32_t)a.k.heads + (uint32_t)h) << a.block_size_log2) +
        ((uint32_t)slot & ((1u << a.block_size_log2) - 1u));
  return slot >= 0 && (int64_t)blk < a.num_blocks;
}

// modes: 0 q and k out, 1 int8 cache, 2 K8V3 cache.  A wave takes the heads of
// its token (or tokens, where there are fewer heads than rows a wave) in
// iterations of RPW rows, q's first, then k's, then v's, with the next two
// iterations' rows in flight: its lanes' angles are fetched once.  Waves that
// share a token take its iterations in turn, so that each has rows of all three
// kinds (a 3-bit V row takes several times a q row's instructions: 2 % of the
// 20.0 us that 4,099 tokens of 28 + 4 heads take).
// What bounds it is memory, and its latency where the tokens are few: 7,001
// tokens of 32 + 8 bf16 heads of 128 with three axes 27 us (147 MB: 5.4 TB/s,
// partly from the memory-side cache); 12,289 of 16 + 4 fp16 heads of 256, a
// quarter rotated, 43 us (255 MB); with the int8 write, 16,384 tokens of 32 + 8
// normalised heads, 83 us (379 MB, 4.6 TB/s); one token 4 us, of which an empty
// launch takes 3.6.
template <int D, int DT, int MODE>
__global__ __launch_bounds__(64 * kWaves) void rope_rows_kernel(Args a) {
  using L = RowsLayout<D>;
  __shared__ __attribute__((aligned(16))) float lds[kWaves][kAngleFloats<D>];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int li = L::part(lane);
  const int chunks = (a.iters + a.per_wave - 1) / a.per_wave;
  const int64_t wave = (int64_t)blockIdx.x * kWaves + wv;
  const int64_t group = wave / chunks;
  const int it0 = (int)(wave - group * chunks), it1 = a.iters;  // every chunks-th iteration: q, k and v rows for each
  const int hpi = 1 << a.hpi_log2, tokens = L::RPW >> a.hpi_log2;
  const int64_t t = group * tokens + (L::row(lane) >> a.hpi_log2);
  const int sub = L::row(lane) & (hpi - 1);
  const bool here = t < a.tokens;
  const int nq = (a.q.heads + hpi - 1) >> a.hpi_log2, nk = (a.k.heads + hpi - 1) >> a.hpi_log2;

  // the norm weights in fp32, once a workgroup
  __shared__ __attribute__((aligned(16))) float norms[2][D];
  if (a.q.norm || a.k.norm) {
    for (int i = threadIdx.x; i < 2 * D; i += 64 * kWaves) {
      const void* w = i < D ? a.q.norm : a.k.norm;
      if (w) norms[i / D][i % D] = load_any(w, i % D, a.norm_dtype);
    }
    __syncthreads();
  }

  const RowsHadamard<D> hadamard(li, a.rot_norm);
  float cb[8];
  bool search = false;
  if constexpr (MODE == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) cb[i] = a.v_codebook[i];
    search = lloyd3_search_ok(cb);
  }
  auto kind_of = [&](int it) { return it < nq ? 0 : (it < nq + nk ? 1 : 2); };
  auto first_head = [&](int it, int kind) { return (it - (kind == 0 ? 0 : (kind == 1 ? nq : nq + nk))) << a.hpi_log2; };
  const char* const rows[3] = {a.q.p + (t * a.q.st + sub * a.q.sh + 16 * li) * kBytes<DT>,
                               a.k.p + (t * a.k.st + sub * a.k.sh + 16 * li) * kBytes<DT>,
                               MODE ? a.v.p + (t * a.v.st + sub * a.v.sh + 16 * li) * kBytes<DT> : nullptr};
  auto fetch = [&](int it) {
    const int kind = kind_of(it), h = first_head(it, kind);
    const int64_t sh = kind == 0 ? a.q.sh : (kind == 1 ? a.k.sh : a.v.sh);
    const int heads = kind == 0 ? a.q.heads : (kind == 1 ? a.k.heads : a.v.heads);
    const char* p = kind == 0 ? rows[0] : (kind == 1 ? rows[1] : rows[2]);
    Raw<DT> raw{};
    if (here && h + sub < heads) raw = load_raw<DT>(p + h * sh * kBytes<DT>);
    return raw;
  };
  Raw<DT> next{}, after{};  // the rows of the next iteration, and of the one after it
  if (it0 < it1) next = fetch(it0);
  if (it0 + chunks < it1) after = fetch(it0 + chunks);
  Angles<D> angles;
  if (it0 < nq + nk) {
    Angles<D>::gather(a, group * tokens, tokens, lane, lds[wv]);
    if (here) angles.take(a, lds[wv] + (L::row(lane) >> a.hpi_log2) * 3 * (a.rot >> 1), li);
  }

#pragma unroll 1
  for (int it = it0; it < it1; it += chunks) {
    const int kind = kind_of(it), h = first_head(it, kind) + sub;
    const bool live = here && h < (kind == 0 ? a.q.heads : a.k.heads);
    float x[16];
    expand<DT>(next, x);
    next = after;
    if (it + 2 * chunks < it1) after = fetch(it + 2 * chunks);
    if (kind < 2) {
      if (kind == 0 ? a.q.norm : a.k.norm) normalise<D>(a, norms[kind] + 16 * li, x);
      angles.turn(a, x);
      char* out = kind == 0 ? a.q_out : a.k_out;
      if (live && out) {
        const int64_t off = kind == 0 ? t * a.qo_t + h * a.qo_h : t * a.ko_t + h * a.ko_h;
        constexpr int OT = MODE ? 0 : DT;  // the writing modes hand q and k on in fp16
        store_part<OT>(out + (off + 16 * li) * kBytes<OT>, x, lane);
      }
    }
    if constexpr (MODE > 0) {
      if (kind == 0) continue;
      uint64_t row = 0;
      const bool write = live && cache_row(a, t, h, row);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = (float)(_Float16)pin(x[i]);
      if (kind == 1) {
        hadamard(x);
        rows_rtn_store<D>(x, write, li, PtrOut{a.k_cache + row * D}, PtrOut{reinterpret_cast<char*>(a.k_scale + row)});
      } else if constexpr (MODE == 1) {
        rows_rtn_store<D>(x, write, li, PtrOut{a.v_cache + row * D}, PtrOut{reinterpret_cast<char*>(a.v_scale + row)});
      } else {
        rows_lloydmax3_store<D, false>(x, write, li, search, cb, cb, PtrOut{a.v_cache + row * (D / 32 * 3 * 4)},
                                       PtrOut{reinterpret_cast<char*>(a.v_scale + row * (D / 128))});
      }
    }
  }
}

// Any alignment, any even R: one wave per row, lane l holds dims l, l + 64, ..
// and reads its pairs' other values itself.  The arithmetic and its order are
// the kernel's above.
template <int D, int DT, int MODE>
__global__ __launch_bounds__(64 * kWaves) void rope_kernel(Args a) {
  constexpr int E = RowLayout<D>::E;
  constexpr int OT = MODE ? 0 : DT;
  const int lane = threadIdx.x & 63;
  const bool active = lane < RowLayout<D>::ACTIVE;
  const int heads = a.q.heads + a.k.heads + a.v.heads;
  const int64_t id = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (id >= a.tokens * heads) return;
  const int64_t t = id / heads;
  int h = (int)(id - t * heads);
  const int kind = h < a.q.heads ? 0 : (h < a.q.heads + a.k.heads ? 1 : 2);
  const Rows& rows = kind == 0 ? a.q : (kind == 1 ? a.k : a.v);
  h -= kind == 0 ? 0 : (kind == 1 ? a.q.heads : a.q.heads + a.k.heads);
  const char* src = rows.p + (t * rows.st + h * rows.sh) * kBytes<DT>;
  float x[E];
#pragma unroll
  for (int j = 0; j < E; ++j) x[j] = active ? load_any(src, lane + 64 * j, DT) : 0.0f;
  if (kind < 2) {
    const int half = a.rot >> 1;
    float y[E], c[E], s[E];
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int d = lane + 64 * j;
      y[j] = 0.0f;
      c[j] = s[j] = __builtin_nanf("");
      if (active && d < a.rot) {
        const int pair = a.adjacent ? d >> 1 : (d < half ? d : d - half);
        const bool second = a.adjacent ? d & 1 : d >= half;
        y[j] = load_any(src, a.adjacent ? d ^ 1 : (second ? d - half : d + half), DT);
        const float* row = table_row(a, position(a, a.axes == 1 ? 0 : axis_of(a, pair), t));
        if (row) {
          c[j] = row[pair];
          s[j] = second ? row[half + pair] : -row[half + pair];
        }
      }
    }
    if (rows.norm) {
      float sq[E];
#pragma unroll
      for (int j = 0; j < E; ++j) {
        sq[j] = x[j] * x[j];
#pragma unroll
        for (int m = 1; m <= 32; m <<= 1) {
          if (m < D) sq[j] = sq[j] + shfl_xor_f(sq[j], m);
        }
      }
#pragma unroll
      for (int w = 1; w < E; w <<= 1) {
#pragma unroll
        for (int j = 0; j < E; j += 2 * w) sq[j] = sq[j] + sq[j + w];
      }
      const float r = 1.0f / __builtin_sqrtf(sq[0] * a.inv_d + a.eps);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int d = lane + 64 * j;
        if (active) {
          x[j] = x[j] * r * load_any(rows.norm, d, a.norm_dtype);
          if (d < a.rot)
            y[j] = y[j] * r * load_any(rows.norm, a.adjacent ? d ^ 1 : (d < half ? d + half : d - half), a.norm_dtype);
        }
      }
    }
    char* out = kind == 0 ? a.q_out : a.k_out;
    const int64_t off = kind == 0 ? t * a.qo_t + h * a.qo_h : t * a.ko_t + h * a.ko_h;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int d = lane + 64 * j;
      const float r = x[j] * c[j] + y[j] * s[j];
      x[j] = d < a.rot ? r : x[j];
      if (active && out) {
        if constexpr (OT == 0) reinterpret_cast<_Float16*>(out)[off + d] = (_Float16)pin(x[j]);
        else if constexpr (OT == 1) reinterpret_cast<__bf16*>(out)[off + d] = (__bf16)pin(x[j]);
        else reinterpret_cast<float*>(out)[off + d] = x[j];
      }
    }
  }
  if constexpr (MODE > 0) {
    uint64_t row = 0;
    if (kind == 0 || !cache_row(a, t, h, row)) return;
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = (float)(_Float16)pin(x[j]);
    if (kind == 1) {
      fwht_row<D>(x, lane);
#pragma unroll
      for (int j = 0; j < E; ++j) x[j] = (float)(_Float16)materialize(x[j] * a.rot_norm);
      rtn_store_row<D>(x, lane, PtrOut{a.k_cache + row * D}, PtrOut{reinterpret_cast<char*>(a.k_scale + row)});
    } else if constexpr (MODE == 1) {
      rtn_store_row<D>(x, lane, PtrOut{a.v_cache + row * D}, PtrOut{reinterpret_cast<char*>(a.v_scale + row)});
    } else {
      constexpr int NB = D / 128, WORDS = D / 32 * 3;
      float cb[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) cb[i] = a.v_codebook[i];
      uint32_t w;
      float nv;
      lloydmax3_encode_row<D>(x, cb, lane, w, nv);
      if (lane < WORDS) PtrOut{a.v_cache + row * (WORDS * 4)}.st32(lane * 4u, w);
      if (lane < NB) PtrOut{reinterpret_cast<char*>(a.v_scale + row * NB)}.st32(lane * 4u, __builtin_bit_cast(uint32_t, nv));
    }
  }
}

static bool aligned(const void* p, int64_t st, int64_t sh, int bytes) {
  return (uintptr_t)p % 16 == 0 && st * bytes % 16 == 0 && sh * bytes % 16 == 0;
}

template <int D, int DT, int MODE>
static int launch(Args& a, const char* what, hipStream_t stream) {
  const int bytes = kBytes<DT>, obytes = MODE ? 2 : bytes;
  const int apart = a.rot / 32;  // half pairing: parts between a pair's values
  const bool rows = aligned(a.q.p, a.q.st, a.q.sh, bytes) && aligned(a.k.p, a.k.st, a.k.sh, bytes) &&
                    aligned(a.v.p, a.v.st, a.v.sh, bytes) && aligned(a.q_out, a.qo_t, a.qo_h, obytes) &&
                    aligned(a.k_out, a.ko_t, a.ko_h, obytes) && (uintptr_t)a.table % 16 == 0 && a.rot % 16 == 0 &&
                    (a.adjacent || a.rot == 16 || (a.rot % 32 == 0 && is_pow2(apart)));
  if (rows) {
    constexpr int RPW = RowsLayout<D>::RPW;
    a.partner = a.adjacent || a.rot == 16 ? 0 : apart;
    a.pairs_log2 = log2i(a.rot / 2 < 64 ? a.rot / 2 : 64);
    int fewest = a.q.heads;
    if (a.k.heads && a.k.heads < fewest) fewest = a.k.heads;
    a.hpi_log2 = 0;
    while ((2 << a.hpi_log2) <= RPW && (2 << a.hpi_log2) <= fewest) ++a.hpi_log2;
    const int hpi = 1 << a.hpi_log2, tokens = RPW >> a.hpi_log2;
    a.iters = (a.q.heads + hpi - 1) / hpi + (a.k.heads + hpi - 1) / hpi + (a.v.heads + hpi - 1) / hpi;
    const int64_t groups = (a.tokens + tokens - 1) / tokens;
    // as many waves as the GPU holds (16 a CU, 12 with the 3-bit search's registers), no more: a wave's start, the chain
    // from the positions to the angles, takes as long as several iterations, and waves that wait for a place cost more
    // than longer ones (4,099 tokens of 28 + 4 heads into K8V3 24.9 us with 1.5 times as many, 21.6 with 1.3, 20.0 so;
    // 1,000 of 32 + 8 int8 10.3 / 8.6 / 8.6, 3,000 19.4 / 19.3 / 16.9)
    const int64_t want = (int64_t)device_cus() * (MODE == 2 ? 12 : 16);
    const int parts = (int)(want < groups ? 1 : (want / groups > a.iters ? a.iters : want / groups));
    a.per_wave = (a.iters + parts - 1) / parts;
    const int64_t waves = groups * ((a.iters + a.per_wave - 1) / a.per_wave);
    const int64_t grid = (waves + kWaves - 1) / kWaves;
    S8KV_REQUIRE(grid < (int64_t(1) << 31), S8KV_ERR_INVALID, "%s: too many tokens (%lld)", what, (long long)a.tokens);
    hipLaunchKernelGGL((rope_rows_kernel<D, DT, MODE>), dim3((unsigned)grid), dim3(64 * kWaves), 0, stream, a);
  } else {
    const int64_t n = a.tokens * (a.q.heads + a.k.heads + a.v.heads);
    const int64_t grid = (n + kWaves - 1) / kWaves;
    S8KV_REQUIRE(grid < (int64_t(1) << 31), S8KV_ERR_INVALID, "%s: too many rows (%lld)", what, (long long)n);
    hipLaunchKernelGGL((rope_kernel<D, DT, MODE>), dim3((unsigned)grid), dim3(64 * kWaves), 0, stream, a);
  }
  return check_launch(what);
}

template <int D, int MODE>
static int launch_dtype(Args& a, int dtype, const char* what, hipStream_t stream) {
  if (dtype == 0) return launch<D, 0, MODE>(a, what, stream);
  if (dtype == 1) return launch<D, 1, MODE>(a, what, stream);
  if constexpr (MODE == 0) return launch<D, 2, MODE>(a, what, stream);
  return S8KV_ERR_UNSUPPORTED;
}

template <int MODE>
static int launch_dim(Args& a, int head_dim, int dtype, const char* what, hipStream_t stream) {
  switch (head_dim) {
    case 32:
      if constexpr (MODE < 2) return launch_dtype<32, MODE>(a, dtype, what, stream);
      break;
    case 64:
      if constexpr (MODE < 2) return launch_dtype<64, MODE>(a, dtype, what, stream);
      break;
    case 128: return launch_dtype<128, MODE>(a, dtype, what, stream);
    case 256: return launch_dtype<256, MODE>(a, dtype, what, stream);
  }
  return S8KV_ERR_UNSUPPORTED;
}

// What the rotation alone and the writing forms share.
static int fill(Args& a, const char* what, const void* q, int num_q_heads, int64_t q_st, int64_t q_sh, const void* k,
                int num_kv_heads, int64_t k_st, int64_t k_sh, int64_t num_tokens, int head_dim, int dtype,
                const int32_t* positions, int num_axes, int64_t pos_axis_stride, const uint64_t* axis_map,
                const float* cos_sin, int64_t max_positions, int rot_dim, int pairing, const void* q_norm,
                const void* k_norm, int norm_dtype, float eps, void* q_out, int64_t qo_st, int64_t qo_sh, void* k_out,
                int64_t ko_st, int64_t ko_sh) {
  S8KV_REQUIRE(num_tokens >= 0 && num_q_heads > 0 && num_kv_heads >= 0, S8KV_ERR_INVALID,
               "%s: %lld tokens, %d q heads, %d kv heads", what, (long long)num_tokens, num_q_heads, num_kv_heads);
  S8KV_REQUIRE(head_dim_ok(head_dim), S8KV_ERR_UNSUPPORTED, "%s: head_dim %d not in {32,64,128,256}", what, head_dim);
  S8KV_REQUIRE(dtype >= 0 && dtype <= 2 && norm_dtype >= 0 && norm_dtype <= 2, S8KV_ERR_INVALID, "%s: unknown dtype", what);
  S8KV_REQUIRE(rot_dim > 0 && rot_dim % 2 == 0 && rot_dim <= head_dim, S8KV_ERR_INVALID,
               "%s: rot_dim %d must be even and in [2, head_dim %d]", what, rot_dim, head_dim);
  S8KV_REQUIRE(pairing == 0 || pairing == 1, S8KV_ERR_INVALID, "%s: pairing %d not in {0, 1}", what, pairing);
  S8KV_REQUIRE(num_axes >= 1 && num_axes <= 4 && (num_axes == 1 || axis_map), S8KV_ERR_INVALID,
               "%s: %d position axes (1 to 4, with an axis map for more than one)", what, num_axes);
  if (num_axes > 1)
    for (int p = 0; p < rot_dim / 2; ++p)
      S8KV_REQUIRE((int)((axis_map[p / 32] >> (2 * (p % 32))) & 3) < num_axes, S8KV_ERR_INVALID,
                   "%s: pair %d is on an axis past %d", what, p, num_axes);
  S8KV_REQUIRE(max_positions > 0, S8KV_ERR_INVALID, "%s: an empty cos / sin table", what);
  S8KV_REQUIRE(num_tokens == 0 || (q && q_out && positions && cos_sin && (num_kv_heads == 0 || k)), S8KV_ERR_INVALID,
               "%s: null pointer", what);
  a.q = Rows{(char*)q, q_st, q_sh, num_q_heads, q_norm};
  a.k = Rows{(char*)k, k_st, k_sh, num_kv_heads, k_norm};
  a.q_out = (char*)q_out;
  a.k_out = (char*)k_out;
  a.qo_t = qo_st; a.qo_h = qo_sh;
  a.ko_t = ko_st; a.ko_h = ko_sh;
  a.tokens = num_tokens;
  a.pos = positions;
  a.pos_stride = pos_axis_stride;
  a.axes = num_axes;
  if (num_axes > 1)
    for (int i = 0; i < 4; ++i) a.axis_map[i] = axis_map[i];
  a.table = cos_sin;
  a.max_pos = max_positions;
  a.rot = rot_dim;
  a.adjacent = pairing;
  a.norm_dtype = norm_dtype;
  a.eps = eps;
  a.inv_d = 1.0f / (float)head_dim;
  a.rot_norm = (float)(1.0 / __builtin_sqrt((double)head_dim));
  return S8KV_OK;
}

static int fill_cache(Args& a, const char* what, const void* v, int64_t v_st, int64_t v_sh, const int32_t* slot_mapping,
                      void* k_cache, float* k_scale, void* v_cache, float* v_scale, int64_t num_blocks,
                      int block_size) {
  S8KV_REQUIRE(a.k.heads > 0, S8KV_ERR_INVALID, "%s: num_kv_heads must be > 0", what);
  S8KV_REQUIRE(is_pow2(block_size) && block_size >= 4, S8KV_ERR_UNSUPPORTED,
               "%s: block_size %d must be a power of two >= 4", what, block_size);
  S8KV_REQUIRE(num_blocks > 0, S8KV_ERR_INVALID, "%s: num_blocks must be > 0", what);
  S8KV_REQUIRE(fits_u32(num_blocks * a.k.heads * block_size), S8KV_ERR_UNSUPPORTED,
               "%s: more than 2^32 cache rows per layer", what);
  S8KV_REQUIRE(a.tokens == 0 || (v && slot_mapping), S8KV_ERR_INVALID, "%s: null pointer", what);
  S8KV_REQUIRE(k_cache && k_scale && v_cache && v_scale, S8KV_ERR_INVALID, "%s: null cache pointer", what);
  a.v = Rows{(char*)v, v_st, v_sh, a.k.heads, nullptr};
  a.slot_mapping = slot_mapping;
  a.k_cache = (char*)k_cache;
  a.v_cache = (char*)v_cache;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.num_blocks = num_blocks;
  a.block_size_log2 = log2i(block_size);
  return S8KV_OK;
}

}  // namespace rope
}  // namespace s8kv

using namespace s8kv;

extern "C" int s8kv_rope(const void* q, int num_q_heads, int64_t q_stride_t, int64_t q_stride_h, const void* k,
                         int num_kv_heads, int64_t k_stride_t, int64_t k_stride_h, int64_t num_tokens, int head_dim,
                         int dtype, const int32_t* positions, int num_axes, int64_t pos_axis_stride,
                         const uint64_t* axis_map, const float* cos_sin, int64_t max_positions, int rot_dim,
                         int pairing, const void* q_norm, const void* k_norm, int norm_dtype, float eps, void* q_out,
                         int64_t q_out_stride_t, int64_t q_out_stride_h, void* k_out, int64_t k_out_stride_t,
                         int64_t k_out_stride_h, void* stream) {
  rope::Args a{};
  const char* what = "s8kv_rope";
  if (int rc = rope::fill(a, what, q, num_q_heads, q_stride_t, q_stride_h, k, num_kv_heads, k_stride_t, k_stride_h,
                          num_tokens, head_dim, dtype, positions, num_axes, pos_axis_stride, axis_map, cos_sin,
                          max_positions, rot_dim, pairing, q_norm, k_norm, norm_dtype, eps, q_out, q_out_stride_t,
                          q_out_stride_h, k_out, k_out_stride_t, k_out_stride_h))
    return rc;
  S8KV_REQUIRE(num_tokens == 0 || num_kv_heads == 0 || k_out, S8KV_ERR_INVALID, "%s: null pointer", what);
  if (num_tokens == 0) return S8KV_OK;
  return rope::launch_dim<0>(a, head_dim, dtype, what, (hipStream_t)stream);
}

extern "C" int s8kv_append_rope_int8(
    const void* q, int num_q_heads, int64_t q_stride_t, int64_t q_stride_h, const void* k, const void* v,
    int num_kv_heads, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
    int64_t num_tokens, int head_dim, int dtype, const int32_t* positions, int num_axes, int64_t pos_axis_stride,
    const uint64_t* axis_map, const float* cos_sin, int64_t max_positions, int rot_dim, int pairing,
    const void* q_norm, const void* k_norm, int norm_dtype, float eps, void* q_out, int64_t q_out_stride_t,
    int64_t q_out_stride_h, void* k_out, int64_t k_out_stride_t, int64_t k_out_stride_h, const int32_t* slot_mapping,
    int8_t* k_cache, float* k_scale, int8_t* v_cache, float* v_scale, int64_t num_blocks, int block_size,
    void* stream) {
  rope::Args a{};
  const char* what = "s8kv_append_rope_int8";
  S8KV_REQUIRE(dtype == 0 || dtype == 1, S8KV_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  if (int rc = rope::fill(a, what, q, num_q_heads, q_stride_t, q_stride_h, k, num_kv_heads, k_stride_t, k_stride_h,
                          num_tokens, head_dim, dtype, positions, num_axes, pos_axis_stride, axis_map, cos_sin,
                          max_positions, rot_dim, pairing, q_norm, k_norm, norm_dtype, eps, q_out, q_out_stride_t,
                          q_out_stride_h, k_out, k_out_stride_t, k_out_stride_h))
    return rc;
  if (int rc = rope::fill_cache(a, what, v, v_stride_t, v_stride_h, slot_mapping, k_cache, k_scale, v_cache, v_scale,
                                num_blocks, block_size))
    return rc;
  if (num_tokens == 0) return S8KV_OK;
  return rope::launch_dim<1>(a, head_dim, dtype, what, (hipStream_t)stream);
}

extern "C" int s8kv_append_rope_k8v3(
    const void* q, int num_q_heads, int64_t q_stride_t, int64_t q_stride_h, const void* k, const void* v,
    int num_kv_heads, int64_t k_stride_t, int64_t k_stride_h, int64_t v_stride_t, int64_t v_stride_h,
    int64_t num_tokens, int head_dim, int dtype, const int32_t* positions, int num_axes, int64_t pos_axis_stride,
    const uint64_t* axis_map, const float* cos_sin, int64_t max_positions, int rot_dim, int pairing,
    const void* q_norm, const void* k_norm, int norm_dtype, float eps, void* q_out, int64_t q_out_stride_t,
    int64_t q_out_stride_h, void* k_out, int64_t k_out_stride_t, int64_t k_out_stride_h, const int32_t* slot_mapping,
    int8_t* k_cache, float* k_scale, int32_t* v_packed, float* v_norm, const float* v_codebook, int lloyd_block,
    int64_t num_blocks, int block_size, void* stream) {
  rope::Args a{};
  const char* what = "s8kv_append_rope_k8v3";
  S8KV_REQUIRE(dtype == 0 || dtype == 1, S8KV_ERR_INVALID, "%s: dtype must be fp16 or bf16", what);
  if (int rc = rope::fill(a, what, q, num_q_heads, q_stride_t, q_stride_h, k, num_kv_heads, k_stride_t, k_stride_h,
                          num_tokens, head_dim, dtype, positions, num_axes, pos_axis_stride, axis_map, cos_sin,
                          max_positions, rot_dim, pairing, q_norm, k_norm, norm_dtype, eps, q_out, q_out_stride_t,
                          q_out_stride_h, k_out, k_out_stride_t, k_out_stride_h))
    return rc;
  S8KV_REQUIRE(head_dim == 128 || head_dim == 256, S8KV_ERR_UNSUPPORTED, "%s: head_dim %d not in {128, 256}", what,
               head_dim);
  S8KV_REQUIRE(lloyd_block == 128, S8KV_ERR_UNSUPPORTED, "%s: lloyd_block %d != 128", what, lloyd_block);
  S8KV_REQUIRE(v_codebook, S8KV_ERR_INVALID, "%s: null cache pointer", what);
  if (int rc = rope::fill_cache(a, what, v, v_stride_t, v_stride_h, slot_mapping, k_cache, k_scale, v_packed, v_norm,
                                num_blocks, block_size))
    return rc;
  a.v_codebook = v_codebook;
  if (num_tokens == 0) return S8KV_OK;
  return rope::launch_dim<2>(a, head_dim, dtype, what, (hipStream_t)stream);
}
