// dense_gemm_impl.h — the tiled matrix product of the dense operators, one template for the three
// products of a layer: forward z = x W (A[i][k], B[k][j]), dx = dz W^T (A[i][k], B[j][k]) and
// dW = x^T dz (A[k][i], B[k][j]); x, W and dz stay in their row-major layouts.
//
// A workgroup computes a BM x BN tile; a stage is 128 bytes of K (64 16-bit or 32 fp32 elements).
// Both operands' stages go from memory to LDS without passing registers (16-byte buffer loads with
// the LDS destination), double-buffered: stage t + 1 is in flight while stage t is multiplied, one
// barrier per stage.  The LDS image of a load is linear in the lane, so bank conflicts are avoided
// by permuting which 16 bytes of the source each lane fetches (XOR on the 16-byte index).
//  * K-contiguous operand: rows of 128 bytes, slot = chunk ^ (row & 7); a lane's MFMA fragment is
//    one ds_read_b128.
//  * K-strided operand: rows of one k.  16-bit fragments come from two ds_read_b64_tr_b16 (a 16-lane
//    group reads a 4 k x 16 column block and gets it transposed); fp32 fragments from four b32 reads.
// The MFMA's first operand is the B fragment, so D holds C transposed: a lane has four consecutive
// columns of one row, which the epilogue loads and stores as vectors.
//
// Edges: rows / columns past I, J fetch the last row again or zeros, and are not stored; K past the
// end fetches zeros (offsets past the buffer descriptor's range read 0 without an access).
#pragma once
#include <type_traits>

#include "dense_common.h"

namespace dense {

typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr uint32_t kOob = DGPRF_OOB;

__device__ __forceinline__ rsrc_t rsrc_of(const void* p, int64_t bytes) {
  const int n = bytes > 0x7FFFFFF0ll ? 0x7FFFFFF0 : bytes < 0 ? 0 : (int)bytes;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, n, 0x00020000);
}

// XOR of the 16-byte index within row k of a K-strided stage, C columns wide
template <class T, int C>
__device__ __forceinline__ int swz_strided(int k) {
  if constexpr (sizeof(T) == 4) return C >= 64 ? 4 * ((k >> 2) & 3) : 4 * ((k >> 2) & 1);
  else if constexpr (C >= 128) return 2 * ((k & 3) | (((k >> 3) & 1) << 2));
  else if constexpr (C == 64) return 2 * (((k >> 1) & 1) | (((k >> 3) & 1) << 1));
  else return 2 * ((k >> 3) & 1);
}

// One operand's stages: R rows (KC) or columns of the tile, NT threads
template <class T, bool KC, int R, int NT>
struct Stage {
  static constexpr int CE = 16 / (int)sizeof(T);   // elements of a 16-byte chunk
  static constexpr int BK = 128 / (int)sizeof(T);  // K of a stage
  static constexpr int LOADS = R * 8 / NT;
  static constexpr int BYTES = R * 128;
  static constexpr int CPR = R / CE;               // chunks of a K-strided row
  static_assert(LOADS >= 1 && R * 8 % NT == 0, "tile too small for the workgroup");
  uint32_t off[LOADS];
  const char* base;
  int64_t step;   // bytes between stages
  int64_t range;  // K-strided: bytes from base to the operand's end; KC: of the tile's rows
  int k_end, kk;  // KC: K, and this lane's first chunk's element offset

  // rows r0 .. of `rows` (KC), or columns r0 .. of `cols` readable ones
  __device__ __forceinline__ void init(const void* p, int64_t ld, int r0, int rows, int cols, int K,
                                       int tid) {
    if constexpr (KC) {
      base = (const char*)p + (int64_t)r0 * ld * sizeof(T);
      step = 128;
      const int last = rows - 1 - r0;
      range = ((int64_t)min(last, R - 1) * ld + K) * sizeof(T);
      k_end = K;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int q = tid + NT * j, r = q >> 3, c = (q & 7) ^ (r & 7);
        off[j] = (uint32_t)(min(r, last) * (int)ld + c * CE) * (uint32_t)sizeof(T);
      }
      kk = ((tid & 7) ^ ((tid >> 3) & 7)) * CE;  // the same for every j: NT / 8 is a multiple of 8
    } else {
      base = (const char*)p + (int64_t)r0 * sizeof(T);
      step = (int64_t)BK * ld * sizeof(T);
      range = ((int64_t)(K - 1) * ld + (cols - r0)) * sizeof(T);
      k_end = 0;
      kk = 0;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int q = tid + NT * j, k = q / CPR, c = (q % CPR) ^ swz_strided<T, R>(k);
        off[j] = r0 + c * CE < cols ? (uint32_t)(k * (int)ld + c * CE) * (uint32_t)sizeof(T) : kOob;
      }
    }
  }
  // stage t to LDS at `to` (wave-uniform: the wave's first 16-byte slot)
  __device__ __forceinline__ void load(int t, char* to) const {
    const int64_t at = (int64_t)t * step;
    const rsrc_t r = rsrc_of(base + at, range - at);
    if (KC && (t + 1) * BK > k_end) {
      const bool in = t * BK + kk < k_end;
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(to + j * NT * 16), 16,
                                                 in ? off[j] : kOob, 0, 0, 0);
    } else {
#pragma unroll
      for (int j = 0; j < LOADS; ++j)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(to + j * NT * 16), 16, off[j], 0, 0,
                                                 0);
    }
  }
};

// A fragment: 16 bytes; 16-bit: k = 8 g + e of 32, fp32: k = 4 g + e of 16 (g = lane >> 4), row or
// column lane & 15.  NF fragments 16 apart, starting at w0 of the tile's R.
template <class T, bool KC, int R, int NF>
struct Frags {
  typedef typename std::conditional<sizeof(T) == 4, f4, typename Vec<T>::v8>::type frag;
  uint32_t at[KC ? 2 : NF];
  __device__ __forceinline__ void init(int w0, int lane) {
    const int g = lane >> 4, i = lane & 15;
    if constexpr (KC) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) at[ks] = (w0 + i) * 128 + (((ks * 4 + g) ^ (i & 7)) * 16);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int c = (w0 + 16 * f) / 4, k = 4 * g;
        at[f] = k * R * 4 + ((c + (i >> 2)) ^ swz_strided<T, R>(k)) * 16 + (i & 3) * 4;
      }
    } else {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int c = (w0 + 16 * f) / 8, k = 8 * g + (i >> 2);
        at[f] = k * R * 2 + ((c + ((i & 3) >> 1)) ^ swz_strided<T, R>(k)) * 16 + (i & 1) * 8;
      }
    }
  }
  __device__ __forceinline__ frag read(const char* lds, int ks, int f) const {
    if constexpr (KC) {
      return *reinterpret_cast<const frag*>(lds + at[ks] + f * 2048);
    } else if constexpr (sizeof(T) == 4) {
      frag v;
#pragma unroll
      for (int s = 0; s < 4; ++s)
        v[s] = *reinterpret_cast<const float*>(lds + at[f] + (ks * 16 + s) * R * 4);
      return v;
    } else {
      const char* p = lds + at[f] + ks * 32 * R * 2;
      union {
        s16x4 h[2];
        frag v;
      } u;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * R * 2));
      return u.v;
    }
  }
};

template <class T, class F>
__device__ __forceinline__ f4 mma(F b, F a, f4 c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = mfma16(b[s], a[s], c);
    return c;
  } else if constexpr (std::is_same<T, bf16_t>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a, c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(b, a, c, 0, 0, 0);
  }
}

// vmcnt(0), leaving the other counters alone
#define DENSE_WAIT_LOADS() __builtin_amdgcn_s_waitcnt(0x0F70)

template <class T, bool AKC, bool BKC, int BM, int BN, int WM, int WN, bool PART>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64) void k_dense(const GemmArgs a,
                                                                    const EpiDev e) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass needs the stub alone
  constexpr int NT = BM / WM * (BN / WN) * 64, MI = WM / 16, NI = WN / 16;
  typedef Stage<T, AKC, BM, NT> SA;
  typedef Stage<T, BKC, BN, NT> SB;
  typedef Frags<T, AKC, BM, MI> FA;
  typedef Frags<T, BKC, BN, NI> FB;
  static_assert(NI % 2 == 0, "the epilogue shares a generator call between two column blocks");
  extern __shared__ __attribute__((aligned(1024))) char smem[];

  // XCD-contiguous order (workgroup b runs on XCD b % 8), and within it column sweeps of 8 row
  // tiles, so the workgroups of an XCD's L2 share rows of A and columns of B
  int split, mt, nt;
  {
    const int G = gridDim.x, b = blockIdx.x, x = b & 7, q = G >> 3, r = G & 7;
    int L = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (b >> 3);
    const int tiles = a.n_mt * a.n_nt;
    split = L / tiles;
    L -= split * tiles;
    const int per = 8 * a.n_nt, g = L / per, rows = min(8, a.n_mt - 8 * g);
    L -= g * per;
    mt = 8 * g + L % rows;
    nt = L / rows;
  }
  const int i0 = mt * BM, j0 = nt * BN;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = wave / (BN / WN) * WM, wj = wave % (BN / WN) * WN;

  SA sa;
  SB sb;
  sa.init(a.A, a.lda, i0, a.I, a.Ia, a.Ka, tid);
  sb.init(a.B, a.ldb, j0, a.J, a.Ja, a.Kb, tid);
  FA fa;
  FB fb;
  fa.init(wi, lane);
  fb.init(wj, lane);

  f4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f4zero();

  const int t0 = split * a.stages_split, t1 = min(a.stages, t0 + a.stages_split);
  char* const lds_a = smem;
  char* const lds_b = smem + 2 * SA::BYTES;
  auto issue = [&](int t, int buf) {
    sa.load(t, lds_a + buf * SA::BYTES + wave * 1024);
    sb.load(t, lds_b + buf * SB::BYTES + wave * 1024);
  };
  auto multiply = [&](int buf) {
    const char* la = lds_a + buf * SA::BYTES;
    const char* lb = lds_b + buf * SB::BYTES;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      typename FB::frag bv[NI];
#pragma unroll
      for (int j = 0; j < NI; ++j) bv[j] = fb.read(lb, ks, j);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const typename FA::frag av = fa.read(la, ks, i);
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = mma<T>(bv[j], av, acc[i][j]);
      }
    }
  };
  auto arrive = [&]() {  // this wave's loads have landed, then everyone's
    DENSE_WAIT_LOADS();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  if (t0 < t1) issue(t0, 0);
  for (int t = t0; t < t1; t += 2) {
    arrive();
    if (t + 1 < t1) issue(t + 1, 1);
    multiply(0);
    if (t + 1 < t1) {
      arrive();
      if (t + 2 < t1) issue(t + 2, 0);
      multiply(1);
    }
  }

  const int g = lane >> 4, r0 = i0 + wi + (lane & 15), c0 = j0 + wj + 4 * g;
  if constexpr (PART) {
    float* const out = a.part + (int64_t)split * a.I * a.ldp;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int row = r0 + 16 * i;
      if (row >= a.I) continue;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int col = c0 + 16 * j;
        if (col < a.J) store4(out + (int64_t)row * a.ldp + col, acc[i][j]);  // ldp % 4 == 0
      }
    }
    return;
  }

  const int n = e.n;
  if (e.bias) {
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const f4 b = load4_edge((const T*)e.bias, c0 + 16 * j, n, false);
#pragma unroll
      for (int i = 0; i < MI; ++i) acc[i][j] += b;
    }
  }
  if (e.aux || e.act != DGPRF_ACT_NONE) {
    with_act(e.act, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int row = r0 + 16 * i;
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const int col = c0 + 16 * j;
          if (e.aux && row < a.I && col < n) {
            f4 z = acc[i][j];
#pragma unroll
            for (int c = 0; c < 4; ++c) z[c] = saved_of<ACT>(z[c]);
            store4((T*)e.aux + (int64_t)row * e.ldaux + col, z);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[i][j][c] = act_of<T, ACT>(acc[i][j][c]);
        }
      }
    });
  }
  const uint64_t sub = e.drop.thr ? drop_sub(e.drop) : 0;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int row = r0 + 16 * i;
    if (e.drop.thr) {
      // lanes g and g ^ 1 hold the halves of the same eight columns: in each pair of column blocks
      // the even one makes the words of the first block, the odd one of the second, then they swap
#pragma unroll
      for (int j = 0; j < NI; j += 2) {
        const int col = c0 + 16 * (j + (g & 1));
        const u32x4 w = drop_words(e.drop, sub, (uint64_t)row * (uint32_t)e.groups + (uint32_t)(col >> 3));
        const auto p = __builtin_amdgcn_permlane16_swap(w.x, w.z, false, false);
        const auto q = __builtin_amdgcn_permlane16_swap(w.y, w.w, false, false);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f4& v = acc[i][j + h];
          v[0] = drop_lo(v[0], p[h], e.drop);
          v[1] = drop_hi(v[1], p[h], e.drop);
          v[2] = drop_lo(v[2], q[h], e.drop);
          v[3] = drop_hi(v[3], q[h], e.drop);
        }
      }
    }
    if (row >= a.I) continue;
    const T* res = (const T*)e.res + (int64_t)row * e.ldr;
    T* y = (T*)e.y + (int64_t)row * e.ldy;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int col = c0 + 16 * j;
      if (col >= n) continue;
      f4 v = acc[i][j];
      if (e.res) v += load4_edge(res, col, n, e.vec_r);
      store4_edge(y, col, n, e.vec_y, v);
    }
  }
#endif
}

template <class T, bool AKC, bool BKC, int BM, int BN, int WM, int WN>
hipError_t launch_tile(GemmArgs a, const EpiDev& e, hipStream_t s) {
  constexpr int NT = BM / WM * (BN / WN) * 64;
  const size_t lds = 2 * (BM + BN) * 128;
  const dim3 grid((unsigned)(a.n_mt * a.n_nt * a.splits));
  if (a.part) {
    const auto fn = &k_dense<T, AKC, BKC, BM, BN, WM, WN, true>;
    dgprf::set_lds_limit((const void*)fn, lds);
    hipLaunchKernelGGL(fn, grid, dim3(NT), lds, s, a, e);
  } else {
    const auto fn = &k_dense<T, AKC, BKC, BM, BN, WM, WN, false>;
    dgprf::set_lds_limit((const void*)fn, lds);
    hipLaunchKernelGGL(fn, grid, dim3(NT), lds, s, a, e);
  }
  return hipGetLastError();
}

template <class T, bool AKC, bool BKC>
hipError_t launch_layout(int tile, const GemmArgs& a, const EpiDev& e, hipStream_t s) {
  if (tile == TILE_256) return launch_tile<T, AKC, BKC, 256, 256, 128, 64>(a, e, s);
  if (tile == TILE_128) return launch_tile<T, AKC, BKC, 128, 128, 64, 64>(a, e, s);
  return launch_tile<T, AKC, BKC, 32, 128, 32, 32>(a, e, s);
}

template <class T>
hipError_t launch_gemm(int layout, int tile, const GemmArgs& a, const EpiDev& e, hipStream_t s) {
  if (layout == LAYOUT_NN) return launch_layout<T, true, false>(tile, a, e, s);
  if (layout == LAYOUT_NT) return launch_layout<T, true, true>(tile, a, e, s);
  return launch_layout<T, false, false>(tile, a, e, s);
}

}  // namespace dense
