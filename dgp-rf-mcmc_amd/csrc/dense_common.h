// dense_common.h — what the kernels of the dense operators share (dense.hip, dense_gemm_impl.h):
// element types, the activations and their slopes, the dropout mask of the counter-based generator,
// and the epilogue arguments.
//
//   z = x W + b        y = r + s m a(z)        dropout:  y = r + s m x
//
// Sums, the bias, the activation, the mask's scale and the residual are in 32 bits; a value is
// rounded to the tensors' type once, where it is stored.
#pragma once
#include <type_traits>

#include "dgprf_internal.h"

namespace dense {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32v4_t __attribute__((ext_vector_type(4)));

template <class T>
struct Vec {
  typedef T v8 __attribute__((ext_vector_type(8)));
  // 16 bytes at any element (unaligned accesses are on for this platform's processes): rows of an odd
  // length are read and written as fast as others, where element by element a 16-bit access costs its
  // wave some hundred clocks (1777 x 1008 x 2049 in bf16 with a residual: 43 us, 19 with n = 2048)
  typedef T any4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  typedef T any8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

inline int elem_size(int dtype) { return dtype == DGPRF_F32 ? 4 : 2; }

// ---------------------------------------------------------------- activations
// Normal distribution function by its tail P(Z < -a), a = |z|: the negative side keeps its relative
// precision (no 1 - erf cancellation).  Both forms are own least-squares fits, reweighted towards the
// smallest maximal relative error.
//  * fp32: e^{-a^2 / 2} Q(a), Q(a) = erfcx(a / sqrt 2) / 2 = t (c0 + c1 t + ... + c8 t^8), t = 1 / (1 + 0.35 a),
//    a in [0, 14]: 3.2e-8 (4e-7 as evaluated in 32 bits, without gauss()'s own error).
//  * 16-bit types (whose rounding is 2^-12 and more): 2^{p(a)}, p of degree 7 fitted to log2 of the tail
//    for a in [0, 6.5]: 8.3e-6 as evaluated, falling to 0 beyond; two instructions in three of the other.
// e^x: v_exp_f32 is 2^x to 1 ulp; the product's rounding is an absolute error of the exponent, so the relative
// one grows with it, 1.5 2^-24 |x| (1.8e-6 at silu's z = -20; gauss() has 2.5 2^-24 z^2 / 2)
__device__ __forceinline__ float exp_of(float x) {
  return __builtin_amdgcn_exp2f(x * 1.4426950408889634f);
}
__device__ __forceinline__ float gauss(float z) {  // e^{-z^2 / 2}
  return __builtin_amdgcn_exp2f(z * z * -0.7213475204444817f);
}
template <class T>
__device__ __forceinline__ float tail_of(float a) {
  if constexpr (sizeof(T) == 4) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.35f, a, 1.f));
    float p = -0.02914646826684475f;
    p = fmaf(p, t, 0.14397425949573517f);
    p = fmaf(p, t, -0.2557194232940674f);
    p = fmaf(p, t, 0.1591798961162567f);
    p = fmaf(p, t, -0.023113638162612915f);
    p = fmaf(p, t, 0.10550954192876816f);
    p = fmaf(p, t, 0.11983250081539154f);
    p = fmaf(p, t, 0.13986191153526306f);
    p = fmaf(p, t, 0.13962140679359436f);
    return p * t * gauss(a);
  } else {
    float p = -1.7577908693056088e-06f;
    p = fmaf(p, a, 5.993694139760919e-05f);
    p = fmaf(p, a, -0.0009163665818050504f);
    p = fmaf(p, a, 0.008447404019534588f);
    p = fmaf(p, a, -0.05382455512881279f);
    p = fmaf(p, a, -0.45861563086509705f);
    p = fmaf(p, a, -1.1511802673339844f);
    return __builtin_amdgcn_exp2f(fmaf(p, a, -1.0000038146972656f));
  }
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + exp_of(-z)); }
// sqrt(2 / pi) (z + 0.044715 z^3), twice: tanh u = 2 sigmoid(2 u) - 1, so 0.5 z (1 + tanh u) = z sigmoid(2 u)
__device__ __forceinline__ float tanh_arg2(float z) {
  return 1.5957691216057308f * z * fmaf(0.044715f, z * z, 1.f);
}

template <class T, int ACT>
__device__ __forceinline__ float act_of(float z) {
  if constexpr (ACT == DGPRF_ACT_RELU) return z < 0.f ? 0.f : z;  // a NaN stays one
  if constexpr (ACT == DGPRF_ACT_GELU) {
    const float tail = tail_of<T>(fabsf(z));
    return z * (z < 0.f ? tail : 1.f - tail);
  }
  if constexpr (ACT == DGPRF_ACT_GELU_TANH) return z * sigmoid(tanh_arg2(z));
  if constexpr (ACT == DGPRF_ACT_SILU) return z * sigmoid(z);
  return z;
}

// a'(z), of what saved_of() kept.  z is clamped in the products that vanish for large |z|, so an infinite z has the limit
// (0 or 1) and not inf * 0.
template <class T, int ACT>
__device__ __forceinline__ float slope_of(float z) {
  const float zc = __builtin_amdgcn_fmed3f(z, -60.f, 60.f);
  if constexpr (ACT == DGPRF_ACT_RELU) return z;  // as saved
  if constexpr (ACT == DGPRF_ACT_GELU) {
    const float tail = tail_of<T>(fabsf(z));
    return fmaf(zc * 0.3989422804014327f, gauss(z), z < 0.f ? tail : 1.f - tail);
  }
  if constexpr (ACT == DGPRF_ACT_GELU_TANH) {
    // g = sigmoid(2u): g + z g (1 - g) 2u'
    const float g = sigmoid(tanh_arg2(z));
    return fmaf(zc * g * (1.f - g), 1.5957691216057308f * fmaf(3.f * 0.044715f, zc * zc, 1.f), g);
  }
  if constexpr (ACT == DGPRF_ACT_SILU) {
    const float g = sigmoid(z);
    return fmaf(zc * g, 1.f - g, g);
  }
  return 1.f;
}

// f(act) with the activation as a compile-time constant
template <class F>
__device__ __forceinline__ void with_act(int act, F f) {
  switch (act) {
    case DGPRF_ACT_RELU: f(std::integral_constant<int, DGPRF_ACT_RELU>()); break;
    case DGPRF_ACT_GELU: f(std::integral_constant<int, DGPRF_ACT_GELU>()); break;
    case DGPRF_ACT_GELU_TANH: f(std::integral_constant<int, DGPRF_ACT_GELU_TANH>()); break;
    case DGPRF_ACT_SILU: f(std::integral_constant<int, DGPRF_ACT_SILU>()); break;
    default: f(std::integral_constant<int, DGPRF_ACT_NONE>()); break;
  }
}

// What the backward pass needs of z, as it is stored.  Rounding z costs the slope less than the
// rounding of dz itself costs (z a''(z) is below 0.4); relu's slope is stored instead, because a
// small z could round to the other side of its jump (1 for a NaN, which relu passes on).
template <int ACT>
__device__ __forceinline__ float saved_of(float z) {
  if constexpr (ACT == DGPRF_ACT_RELU) return z <= 0.f ? 0.f : 1.f;
  return z;
}

// ---------------------------------------------------------------- dropout mask
// Eight elements of a row share one Philox4x32-10 call, 16 bits each: p is a multiple of 1 / 65536,
// and one call costs about what the loads and stores of eight 16-bit elements cost at full
// bandwidth (32 bits for each would make the generator the bound).  The counter is the group's
// number, so the mask does not depend on how a kernel is tiled and backward makes it again.
struct DropDev {
  uint32_t thr;  // an element is kept when its 16 bits >= thr; 0: no dropout, 65536: drops all
  float scale;   // 65536 / (65536 - thr); 0 when everything is dropped (with thr = 0: of all elements)
  uint32_t k0, k1;
  uint64_t sub;
  const int64_t* step;  // device counter added to sub, or null
};

__device__ __forceinline__ uint64_t drop_sub(const DropDev& d) {
  return d.sub + (d.step ? (uint64_t)*d.step : 0ull);
}
// philox4x32_10 of dgprf_device.h with the three-input exclusive or of gfx950: a fifth fewer instructions
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);
#else
  return a ^ b ^ c;
#endif
}
__device__ __forceinline__ u32x4 philox_words(u32x4 c, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c.x, p1 = (uint64_t)0xCD9E8D57u * c.z;
    c = u32x4{xor3((uint32_t)(p1 >> 32), c.y, k0), (uint32_t)p1, xor3((uint32_t)(p0 >> 32), c.w, k1), (uint32_t)p0};
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return c;
}
__device__ __forceinline__ u32x4 drop_words(const DropDev& d, uint64_t sub, uint64_t q) {
  u32x4 c;
  c.x = (uint32_t)q;
  c.y = (uint32_t)sub;
  c.z = (uint32_t)(sub >> 32);
  c.w = ((uint32_t)DGPRF_RNG_DROPOUT << 24) | ((uint32_t)(q >> 32) & 0x00FFFFFFu);
  return philox_words(c, d.k0, d.k1);
}
// keep or drop elements 2 i and 2 i + 1 by word i
__device__ __forceinline__ float drop_lo(float v, uint32_t word, const DropDev& d) {
  return (word & 0xFFFFu) >= d.thr ? v * d.scale : 0.f;
}
__device__ __forceinline__ float drop_hi(float v, uint32_t word, const DropDev& d) {
  return (word >> 16) >= d.thr ? v * d.scale : 0.f;
}

// ---------------------------------------------------------------- epilogue
struct EpiDev {
  const void* bias;  // [n] or null
  const void* res;   // [m][ldr] or null
  void* y;           // [m][ldy]
  void* aux;         // [m][ldaux] saved z (relu: slope) or null; 16-byte aligned rows
  int64_t ldr, ldy, ldaux;
  int32_t n, act;
  int32_t groups;    // ceil(n / 8)
  DropDev drop;
};

// columns col .. col + 3 of a row of n, element by element
template <class T>
__device__ __forceinline__ f4 load4_edge(const T* row, int col, int n) {
  f4 v = f4zero();
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (col + c < n) v[c] = (float)row[col + c];
  return v;
}
template <class T>
__device__ __forceinline__ void store4_edge(T* row, int col, int n, f4 v) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (col + c < n) row[col + c] = (T)v[c];
}

// ---------------------------------------------------------------- eight columns of a row
// row and group of the q-th of rows x groups (a 64-bit division takes some hundred instructions)
__device__ __forceinline__ int64_t row_of(int64_t q, int groups) {
  return q >> 32 ? q / groups : (int64_t)((uint32_t)q / (uint32_t)groups);
}
struct F8 {
  f4 lo, hi;
};
template <class T>
__device__ __forceinline__ F8 load8_whole(const T* p) {
  F8 v;
  if constexpr (sizeof(T) == 4) {
    v.lo = *reinterpret_cast<const typename Vec<T>::any4*>(p);
    v.hi = *reinterpret_cast<const typename Vec<T>::any4*>(p + 4);
  } else {
    const typename Vec<T>::any8 x = *reinterpret_cast<const typename Vec<T>::any8*>(p);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      v.lo[c] = (float)x[c];
      v.hi[c] = (float)x[c + 4];
    }
  }
  return v;
}
template <class T>
__device__ __forceinline__ void store8_whole(T* p, const F8& v) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<typename Vec<T>::any4*>(p) = v.lo;
    *reinterpret_cast<typename Vec<T>::any4*>(p + 4) = v.hi;
  } else {
    typename Vec<T>::any8 x;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      x[c] = (T)v.lo[c];
      x[c + 4] = (T)v.hi[c];
    }
    *reinterpret_cast<typename Vec<T>::any8*>(p) = x;
  }
}
// columns col .. col + 7 of a row of n
template <class T>
__device__ __forceinline__ F8 load8(const T* row, int col, int n) {
  if (col + 8 <= n) return load8_whole(row + col);
  F8 v;
  v.lo = load4_edge(row, col, n);
  v.hi = load4_edge(row, col + 4, n);
  return v;
}
template <class T>
__device__ __forceinline__ void store8(T* row, int col, int n, const F8& v) {
  if (col + 8 <= n) {
    store8_whole(row + col, v);
  } else {
    store4_edge(row, col, n, v.lo);
    store4_edge(row, col + 4, n, v.hi);
  }
}
__device__ __forceinline__ F8 drop8(F8 v, const u32x4& w, const DropDev& d) {
  v.lo[0] = drop_lo(v.lo[0], w.x, d);
  v.lo[1] = drop_hi(v.lo[1], w.x, d);
  v.lo[2] = drop_lo(v.lo[2], w.y, d);
  v.lo[3] = drop_hi(v.lo[3], w.y, d);
  v.hi[0] = drop_lo(v.hi[0], w.z, d);
  v.hi[1] = drop_hi(v.hi[1], w.z, d);
  v.hi[2] = drop_lo(v.hi[2], w.w, d);
  v.hi[3] = drop_hi(v.hi[3], w.w, d);
  return v;
}

// s m a(v + b) of eight columns of a row; stores what backward needs of v + b
template <class T, int ACT>
__device__ __forceinline__ F8 value_of(const EpiDev& e, int64_t row, int col, uint64_t sub, F8 v, const F8& b) {
  v.lo += b.lo;
  v.hi += b.hi;
  if constexpr (ACT != DGPRF_ACT_NONE) {
    if (e.aux) {
      F8 z;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        z.lo[c] = saved_of<ACT>(v.lo[c]);
        z.hi[c] = saved_of<ACT>(v.hi[c]);
      }
      store8_whole((T*)e.aux + row * e.ldaux + col, z);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      v.lo[c] = act_of<T, ACT>(v.lo[c]);
      v.hi[c] = act_of<T, ACT>(v.hi[c]);
    }
  }
  if (e.drop.thr) {
    v = drop8(v, drop_words(e.drop, sub, (uint64_t)row * (uint32_t)e.groups + (uint32_t)(col >> 3)), e.drop);
  } else if (ACT == DGPRF_ACT_NONE && e.drop.scale != 1.f) {  // the products of a backward pass
    v.lo *= e.drop.scale;
    v.hi *= e.drop.scale;
  }
  return v;
}

// ---------------------------------------------------------------- tiled product
// C[i][j] = sum_k A(i, k) B(k, j).  "K-contiguous" operands have k innermost in memory (A[i][k],
// B[j][k]), "K-strided" ones their row or column index (A[k][i], B[k][j]).
struct GemmArgs {
  const void *A, *B;
  int64_t lda, ldb;
  int32_t I, J;
  int32_t Ia, Ja;  // K-strided operands: columns that may be read (I, J rounded up where padded)
  int32_t Ka, Kb;  // K extent of A and B (they differ by A's zero padding)
  int32_t n_mt, n_nt, splits, stages, stages_split;
  float* part;     // split-K partials [splits][I][ldp], or null
  int64_t ldp;
};

enum { LAYOUT_NN = 0, LAYOUT_NT = 1, LAYOUT_TN = 2 };  // forward, dx, dW
// G: two groups of waves; those before TILE_128 are for 16-bit types
enum { TILE_256 = 0, TILE_256N, TILE_256G, TILE_128G, TILE_128, TILE_64, TILE_32, TILES };
struct TileShape {
  int bm, bn, kb, threads;  // rows, columns, bytes of K of a stage, threads at most
};
constexpr TileShape kTiles[TILES] = {{256, 256, 128, 256}, {256, 128, 64, 256}, {256, 128, 128, 512}, {128, 128, 128, 512},
                                     {128, 128, 64, 256},  {64, 64, 128, 512}, {32, 128, 128, 256}};

// one instantiation per element type (dense_<type>.hip): layout, tile, and epilogue (part == null:
// the linear epilogue e; otherwise partial sums)
hipError_t launch_gemm_bf16(int layout, int tile, const GemmArgs& a, const EpiDev& e, hipStream_t s);
hipError_t launch_gemm_f16(int layout, int tile, const GemmArgs& a, const EpiDev& e, hipStream_t s);
hipError_t launch_gemm_f32(int layout, int tile, const GemmArgs& a, const EpiDev& e, hipStream_t s);

}  // namespace dense
