// dense_gemm_impl.h — the tiled matrix product of the dense operators, one template for the three
// products of a layer: forward z = x W (A[i][k], B[k][j]), dx = dz W^T (A[i][k], B[j][k]) and
// dW = x^T dz (A[k][i], B[k][j]); x, W and dz stay in their row-major layouts.
//
// A workgroup of four waves, or two groups of four, computes a BM x BN tile; a stage is KB bytes of K (64 or 128; 64 bytes
// are 32 16-bit or 16 fp32 elements, one step of the matrix instructions).  Both operands' stages go
// from memory to LDS without passing registers (16-byte buffer loads with the LDS destination) into
// ST buffers, one barrier per stage.  The LDS image of a load is linear in the lane, so bank conflicts
// are avoided by permuting which 16 bytes of the source each lane fetches (XOR on the 16-byte index).
//  * K-contiguous operand: rows of KB bytes, the slots permuted so that eight neighbouring rows' equal
//    chunks fall on all banks; a lane's MFMA fragment is one ds_read_b128.
//  * K-strided operand: rows of one k.  16-bit fragments come from two ds_read_b64_tr_b16 (a 16-lane
//    group reads a 4 k x 16 column block and gets it transposed); fp32 fragments from four b32 reads.
// The MFMA's first operand is the B fragment, so D holds C transposed: a lane has four consecutive
// columns of one row, which the epilogue loads and stores as vectors.
//
// Edges: rows / columns past I, J fetch the last row again or zeros, and are not stored; K past the
// end fetches zeros (offsets past the buffer descriptor's range read 0 without an access).
//
// Tiles (launch_layout), and what bounds them:
//  * 256 x 256, 16-bit: a wave's 128 x 128 sub-tile takes a register file of accumulators and the fewest
//    bytes from LDS (reads and the loads' writes 75 % of the matrix instructions' time; 128 x 64 a wave
//    would be at 112 %).  One workgroup a CU, 128-byte rows of K (whole cache lines: 4096^3 in bf16 97 us,
//    103 with 64-byte rows).  4096 x 8192 x 4096 in bf16: 183 us, 1.5 PFLOP/s, where a large library
//    product of the type reaches 1.26; bound by the matrix instructions at the clock that they allow.
//  * 256 x 128 (16-bit) and 128 x 128: two workgroups a CU, one's epilogue beside the other's product;
//    bound by LDS.
//  * The same with two groups of four waves (16-bit), one for each step of a stage: where a CU gets one
//    workgroup, a second wave on each SIMD runs while the first waits, for the same bytes from LDS (eight
//    smaller sub-tiles would take more).  At the end each group takes the other's sums of half of the
//    rows and finishes those.  4096 x 2048 over K = 8192 in bf16: 109 us with 256 x 128, 126 with one group;
//    2048 x 2048 x 2048: 20.9 with 128 x 128, 22.8.
//  * 64 x 64: for results of few tiles.  fp32 takes two groups (1024 x 2048 x 1024: 40 us, 43 with one);
//    16-bit steps are too short for that (1024 x 2048 x 2048 in bf16: 19 us, 16 with one).
//  * 32 x 128: for few rows; bound by the memory's rate (24 x 8192 x 2048 in fp16: 6.8 us, 4.9 TB/s).
#pragma once

#include <algorithm>
#include <atomic>

#include "dense_common.h"

namespace dense {

typedef __attribute__((address_space(3))) void lds_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr uint32_t kOob = DGPRF_OOB;

// Raw buffer descriptor (base, 0 | range in bytes | data format), in scalar registers.
typedef uint32_t desc_t __attribute__((ext_vector_type(4)));
// 16 bytes a lane from the descriptor's `off` (zeros past its range) to LDS at `to` + 16 lane.  Written
// as an instruction because the compiler, which cannot tell the buffers apart, would wait for every
// load in flight before each transposing LDS read; it has no destination register, and the waits are
// the loop's own (wait_loads).  M0 takes a wait state before the load reads it.
__device__ __forceinline__ void load_to_lds(desc_t d, uint32_t off, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(to), "v"(off), "s"(d)
               : "memory", "m0");
}

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// XOR of the 16-byte index within row k of a K-strided stage, C columns wide
template <class T, int C>
__device__ __forceinline__ int swz_strided(int k) {
  if constexpr (sizeof(T) == 4) return C >= 64 ? 4 * ((k >> 2) & 3) : 4 * ((k >> 2) & 1);
  else if constexpr (C >= 128) return 2 * ((k & 3) | (((k >> 3) & 1) << 2));
  else if constexpr (C == 64) return 2 * (((k >> 1) & 1) | (((k >> 3) & 1) << 1));
  else return 2 * ((k >> 3) & 1);
}

// slot permutation of a K-contiguous row
template <int KB>
__device__ __forceinline__ int swz_row(int r) {
  return KB == 64 ? (r >> 1) & 3 : r & 7;
}

// One operand's stages: R rows (KC) or columns of the tile, NT threads
template <class T, bool KC, int R, int KB, int NT>
struct Stage {
  static constexpr int CE = 16 / (int)sizeof(T);   // elements of a 16-byte chunk
  static constexpr int BK = KB / (int)sizeof(T);   // K of a stage
  static constexpr int CPK = KB / 16;              // chunks of a K-contiguous row
  static constexpr int CPR = R / CE;               // chunks of a K-strided row
  static constexpr int LOADS = R * CPK / NT;
  static constexpr int BYTES = R * KB;
  static_assert(LOADS >= 1 && R * CPK % NT == 0, "tile too small for the workgroup");
  static_assert(NT / CPK % 8 == 0, "a lane's chunk must be the same in each of its loads");
  uint32_t off[LOADS];
  desc_t desc;         // of the stage being loaded
  uint32_t step_lo, step_hi;  // bytes between stages
  uint32_t full, tail;  // bytes that a stage, and the last one with data, may reach over
  int last, k_last;    // its number; KC: K in it
  int kk;              // KC: element offset of this lane's chunk

  // rows r0 .. of `rows` (KC), or columns r0 .. of `cols` readable ones; stages t0 .. t1 - 1 of K
  __device__ __forceinline__ void init(const void* p, int64_t ld, int r0, int rows, int cols, int K, int t0,
                                       int t1, int tid) {
    const char* base = (const char*)p;
    const int end = (K + BK - 1) / BK - 1;
    int64_t f, t, step;
    k_last = K - end * BK;
    if constexpr (KC) {
      base += (int64_t)r0 * ld * sizeof(T);
      step = KB;
      const int lr = min(rows - 1 - r0, R - 1);
      f = (int64_t)lr * ld + BK;
      t = (int64_t)lr * ld + k_last;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int q = tid + NT * j, r = q / CPK, c = (q % CPK) ^ swz_row<KB>(r);
        off[j] = (uint32_t)(min(r, lr) * (int)ld + c * CE) * (uint32_t)sizeof(T);
      }
      kk = ((tid % CPK) ^ swz_row<KB>(tid / CPK)) * CE;
    } else {
      base += (int64_t)r0 * sizeof(T);
      step = (int64_t)BK * ld * sizeof(T);
      f = (int64_t)(BK - 1) * ld + (cols - r0);
      t = (int64_t)(k_last - 1) * ld + (cols - r0);
      kk = 0;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) {
        const int q = tid + NT * j, k = q / CPR, c = (q % CPR) ^ swz_strided<T, R>(k);
        off[j] = r0 + c * CE < cols ? (uint32_t)(k * (int)ld + c * CE) * (uint32_t)sizeof(T) : kOob;
      }
    }
    if (t1 - 1 < end) {  // this part of K ends before
      t = f;
      k_last = BK;
    }
    // wave-uniform all, and kept in scalar registers, where next() and the loads need them
    full = uniform((uint32_t)f * (uint32_t)sizeof(T));  // below 2^31 by the limits on widths
    tail = uniform((uint32_t)t * (uint32_t)sizeof(T));
    last = uniform(min(t1 - 1, end));
    k_last = uniform(k_last);
    step_lo = uniform((uint32_t)step);
    step_hi = uniform((uint32_t)(step >> 32));
    const uint64_t at = (uint64_t)base + (uint64_t)((t0 - 1) * step);  // next() goes to t0
    desc[0] = uniform((uint32_t)at);
    desc[1] = uniform((uint32_t)(at >> 32));
    desc[2] = 0;
    desc[3] = 0x00020000u;
  }
  // To stage t, the one after the last time's.  Its loads (load) go to `to` (wave-uniform: the wave's
  // first 16-byte slot); past the last stage, and of K past the end, they bring zeros, without an
  // access.  A few scalar instructions: they run between matrix instructions.
  __device__ __forceinline__ void next(int t) {
    const uint64_t at = ((uint64_t)desc[1] << 32 | desc[0]) + ((uint64_t)step_hi << 32 | step_lo);
    desc[0] = (uint32_t)at;
    desc[1] = (uint32_t)(at >> 32);
    desc[2] = t < last ? full : t == last ? tail : 0u;
    if (KC && t == last && k_last < BK) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) off[j] = kk < k_last ? off[j] : kOob;
    }
  }
  __device__ __forceinline__ void load(int j, uint32_t to) const { load_to_lds(desc, off[j], to + j * NT * 16); }
};

// A fragment: 16 bytes; 16-bit: k = 8 g + e of 32, fp32: k = 4 g + e of 16 (g = lane >> 4), row or
// column lane & 15.  NF fragments 16 apart, starting at w0 of the tile's R.
template <class T, bool KC, int R, int KB, int NF>
struct Frags {
  typedef typename std::conditional<sizeof(T) == 4, f4, typename Vec<T>::v8>::type frag;
  static constexpr int KS = KB / 64;  // steps of a stage
  uint32_t at[KC ? KS : NF];
  // ks0: the step that read() calls 0
  __device__ __forceinline__ void init(int w0, int lane, int ks0) {
    const int g = lane >> 4, i = lane & 15;
    if constexpr (KC) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) at[ks] = (w0 + i) * KB + ((((ks + ks0) * 4 + g) ^ swz_row<KB>(i)) * 16);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int c = (w0 + 16 * f) / 4, k = 16 * ks0 + 4 * g;
        at[f] = k * R * 4 + ((c + (i >> 2)) ^ swz_strided<T, R>(k)) * 16 + (i & 3) * 4;
      }
    } else {
#pragma unroll
      for (int f = 0; f < NF; ++f) {
        const int c = (w0 + 16 * f) / 8, k = 32 * ks0 + 8 * g + (i >> 2);
        at[f] = k * R * 2 + ((c + ((i & 3) >> 1)) ^ swz_strided<T, R>(k)) * 16 + (i & 1) * 8;
      }
    }
  }
  __device__ __forceinline__ frag read(const char* lds, int ks, int f) const {
    if constexpr (KC) {
      return *reinterpret_cast<const frag*>(lds + at[ks] + f * 16 * KB);
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

// part p of a step (fp32: of four, k = 4 g + p)
template <class T, class F>
__device__ __forceinline__ f4 mma(F b, F a, f4 c, int p) {
  if constexpr (sizeof(T) == 4) {
    return mfma16(b[p], a[p], c);
  } else if constexpr (std::is_same<T, bf16_t>::value) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, a, c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(b, a, c, 0, 0, 0);
  }
}

// LDS reads of a fragment
template <class T, bool KC>
constexpr int reads() {
  return KC ? 1 : sizeof(T) == 4 ? 4 : 2;
}

// The same into accumulation registers: with 64 accumulators (256 registers) the compiler moves them
// between the two register files in the loop; as an operand of this instruction one stays where it is.
// Its result is next read by the same instruction 64 of them later, or after settle().
template <class T, class F>
__device__ __forceinline__ void mma_acc(F b, F a, f4& c) {
  if constexpr (std::is_same<T, bf16_t>::value)
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(b), "v"(a));
  else
    asm volatile("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(b), "v"(a));
}
// ... and a load to LDS behind it, which it gives M0's wait state
template <class T, class F>
__device__ __forceinline__ void mma_acc_load(F b, F a, f4& c, desc_t d, uint32_t off, uint32_t to, uint32_t more) {
  if constexpr (std::is_same<T, bf16_t>::value)
    asm volatile("s_add_u32 m0, %5, %6\n\tv_mfma_f32_16x16x32_bf16 %0, %1, %2, %0\n\t"
                 "buffer_load_dwordx4 %3, %4, 0 offen lds"
                 : "+a"(c)
                 : "v"(b), "v"(a), "v"(off), "s"(d), "s"(to), "s"(more)
                 : "memory", "m0", "scc");
  else
    asm volatile("s_add_u32 m0, %5, %6\n\tv_mfma_f32_16x16x32_f16 %0, %1, %2, %0\n\t"
                 "buffer_load_dwordx4 %3, %4, 0 offen lds"
                 : "+a"(c)
                 : "v"(b), "v"(a), "v"(off), "s"(d), "s"(to), "s"(more)
                 : "memory", "m0", "scc");
}
// the last matrix instructions' results are readable (16 passes at most are in flight)
template <int MI, int NI>
__device__ __forceinline__ void settle(f4 (&acc)[MI][NI]) {
  asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) asm volatile("" : "+a"(acc[i][j]));
}

// LDS that a wave's rows take on their way out, CR at a time (a wave of two groups finishes half of its
// sub-tile's); the pitch spreads the rows of a write over the banks
template <int WM, int WN, int KG>
struct Turned {
  static constexpr int ROWS = WM / KG, CR = ROWS < 64 ? ROWS : 64, PITCH = WN + 4, BYTES = CR * PITCH * 4;
};
// the wave's LDS accesses before are done before those after
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// all LDS reads done and at most N loads outstanding
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | ((N >> 4) << 14));
}

template <class T, bool AKC, bool BKC, int BM, int BN, int WM, int WN, int KB, int ST, int OCC, int KG, bool PART>
__global__ __launch_bounds__(256 * KG, OCC) void k_dense(const GemmArgs a, const EpiDev e) {
#if defined(__HIP_DEVICE_COMPILE__)  // the host pass needs the stub alone
  constexpr int NT = 256 * KG, MI = WM / 16, NI = WN / 16;
  static_assert(BM / WM * (BN / WN) == 4, "four waves of a group");
  static_assert(KG == 1 || (KG == 2 && KB == 128), "a group of waves for each step of a stage");
  constexpr bool BIG = MI * NI == 64;  // accumulators fill a register file
  static_assert(!BIG || (MI == 8 && NI == 8 && sizeof(T) == 2 && BM == 256), "turn()'s groups");
  typedef Stage<T, AKC, BM, KB, NT> SA;
  typedef Stage<T, BKC, BN, KB, NT> SB;
  typedef Frags<T, AKC, BM, KB, MI> FA;
  typedef Frags<T, BKC, BN, KB, NI> FB;
  extern __shared__ __attribute__((aligned(1024))) char smem[];

  // XCD-contiguous order (workgroup b runs on XCD b % 8), and within it column sweeps of 4 row
  // tiles, so the workgroups of an XCD's L2 share rows of A and columns of B (8192 x 2048 x 8448 in
  // bf16: 255 us with sweeps of 4, 259 of 8, 269 of 16)
  int split, mt, nt;
  {
    const int G = gridDim.x, b = blockIdx.x, x = b & 7, q = G >> 3, r = G & 7;
    int L = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (b >> 3);
    const int tiles = a.n_mt * a.n_nt;
    split = L / tiles;
    L -= split * tiles;
    const int per = 4 * a.n_nt, g = L / per, rows = min(4, a.n_mt - 4 * g);
    L -= g * per;
    mt = 4 * g + L % rows;
    nt = L / rows;
  }
  const int i0 = mt * BM, j0 = nt * BN;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wpos = wave % 4, group = wave / 4;
  const int wi = wpos / (BN / WN) * WM, wj = wpos % (BN / WN) * WN;

  SA sa;
  SB sb;
  const int t0 = split * a.stages_split, t1 = min(a.stages, t0 + a.stages_split);
  sa.init(a.A, a.lda, i0, a.I, a.Ia, a.Ka, t0, t1, tid);
  sb.init(a.B, a.ldb, j0, a.J, a.Ja, a.Kb, t0, t1, tid);
  // the epilogue's columns of this lane, and their bias, which is on its way during the product
  const int lc = (lane % (WN / 8)) * 8, col = j0 + wj + lc;
  F8 b{f4zero(), f4zero()};
  if (!PART && e.bias && col < e.n) b = load8((const T*)e.bias, col, e.n);
  FA fa;
  FB fb;
  fa.init(wi, lane, group);
  fb.init(wj, lane, group);

  f4 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f4zero();

  // Steps run one ahead in registers: while step s is multiplied, the fragments of step s + 1 are read
  // from LDS into the other set.  A new stage's fragments are read after a barrier that says that its
  // loads have landed; the same barrier says that everyone has read the stage before it, whose buffer
  // then takes the stage ST later.  Stages past the end load zeros, so every stage has the same loads.
  constexpr int BUF = SA::BYTES + SB::BYTES, LOADS = SA::LOADS + SB::LOADS, KS = KB / 64 / KG;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)smem + wave * 1024;
  typename FA::frag av[2][MI];
  typename FB::frag bv[2][NI];
  auto barrier = []() {
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  auto read_one = [&](int f, int set, int at, int ks) {  // fragment f of a step: B's, then A's
    if (f < NI) bv[set][f] = fb.read(smem + at + SA::BYTES, ks, f);
    else av[set][f - NI] = fa.read(smem + at, ks, f - NI);
  };
  // One step: its matrix instructions with everything else between them, a little after each.  A wave
  // issues in order, and a matrix instruction of 16 cycles hides about three others behind it: in a
  // burst after several of them, the same instructions stand in the way of the next (4096^3 in bf16:
  // 114 us with groups of four).  Reads take the first three quarters, so that the last of them have
  // time to land before the next step.  next_at, next_ks: where the other set's fragments are;
  // new_stage: also load the stage ST later (t + ST) to buffer old.
  constexpr int PARTS = sizeof(T) == 4 ? 4 : 1, M = MI * NI * PARTS, F = MI + NI, MR = M * 3 / 4;
  auto run = [&](int set, bool reading, int next_at, int next_ks, bool new_stage, int t, int old) __attribute__((always_inline)) {
    int f = 0, l = 0;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      const int p = m / (MI * NI), i = m % (MI * NI) / NI, j = m % NI;  // p: part of the step
      bool load = new_stage && l < LOADS && m >= (2 * l + 1) * M / LOADS / 2;
      if constexpr (BIG) {
        if (load && l < SA::LOADS)
          mma_acc_load<T>(bv[set][j], av[set][i], acc[i][j], sa.desc, sa.off[l], lds0 + l * NT * 16, old);
        else if (load)
          mma_acc_load<T>(bv[set][j], av[set][i], acc[i][j], sb.desc, sb.off[l - SA::LOADS],
                          lds0 + SA::BYTES + (l - SA::LOADS) * NT * 16, old);
        else
          mma_acc<T>(bv[set][j], av[set][i], acc[i][j]);
      } else {
        acc[i][j] = mma<T>(bv[set][j], av[set][i], acc[i][j], p);
      }
      if (!BIG || !load)
        while (reading && f < F && m >= f * MR / F) read_one(f++, set ^ 1, next_at, next_ks);
      while (load) {
        if (!BIG && l < SA::LOADS) sa.load(l, lds0 + old);
        else if (!BIG) sb.load(l - SA::LOADS, lds0 + old + SA::BYTES);
        ++l;
        if (l == SA::LOADS) sa.next(t + ST + 1);
        if (l == LOADS) sb.next(t + ST + 1);
        load = !BIG && l < LOADS && m >= (2 * l + 1) * M / LOADS / 2;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  int cur = 0;  // buffer of stage t
  // multiplies the last step of stage t (set) while the first of stage t + 1 is read into the other
  auto turn = [&](int t, int set) __attribute__((always_inline)) {
    wait_loads<(ST - 2) * LOADS>();
    barrier();
    const int old = cur;
    cur = cur == (ST - 1) * BUF ? 0 : cur + BUF;
    run(set, true, cur, 0, true, t, old);
  };
#pragma unroll
  for (int i = 0; i < ST; ++i) {
    sa.next(t0 + i);
    sb.next(t0 + i);
#pragma unroll
    for (int k = 0; k < SA::LOADS; ++k) sa.load(k, lds0 + i * BUF);
#pragma unroll
    for (int k = 0; k < SB::LOADS; ++k) sb.load(k, lds0 + i * BUF + SA::BYTES);
  }
  sa.next(t0 + ST);
  sb.next(t0 + ST);
  wait_loads<(ST - 1) * LOADS>();
  barrier();
#pragma unroll
  for (int f = 0; f < F; ++f) read_one(f, 0, 0, 0);
  if constexpr (KS == 1) {
    int t = t0;
    for (; t + 1 < t1; t += 2) {
      turn(t, 0);
      turn(t + 1, 1);
    }
    if (t < t1) {
      wait_loads<0>();
      run(0, false, 0, 0, false, t, 0);
    }
  } else {
    for (int t = t0; t < t1; ++t) {
      run(0, true, cur, 1, false, t, 0);
      turn(t, 1);
    }
  }
  wait_loads<0>();
  if constexpr (BIG) settle(acc);
  // Two groups: each takes the other's sums of the half of the rows that it finishes.
  constexpr int MF = MI / KG;
  f4 half[MF][NI];
  f4 (&fin)[MF][NI] = KG == 1 ? reinterpret_cast<f4 (&)[MF][NI]>(acc) : half;
  if constexpr (KG > 1) {
    f4* const give = reinterpret_cast<f4*>(smem) + wave * (MF * NI * 64) + lane;
    const f4* const take = reinterpret_cast<f4*>(smem) + (wave ^ 4) * (MF * NI * 64) + lane;
    auto put = [&](auto from) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) give[(i * NI + j) * 64] = acc[decltype(from)::value + i][j];
    };
    auto sum = [&](auto from) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) half[i][j] = acc[decltype(from)::value + i][j] + take[(i * NI + j) * 64];
    };
    typedef std::integral_constant<int, 0> First;
    typedef std::integral_constant<int, MF> Second;
    __syncthreads();
    if (group == 0) put(Second());
    else put(First());
    __syncthreads();
    if (group == 0) sum(First());
    else sum(Second());
  }
  const int wr = i0 + wi + group * (WM / KG);  // the first row that this wave finishes

  const int g = lane >> 4;
  if constexpr (PART) {
    const int r0 = wr + (lane & 15), c0 = j0 + wj + 4 * g;
    float* const out = a.part + (int64_t)split * a.I * a.ldp;
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int row = r0 + 16 * i, col = c0 + 16 * j;
        if (row < a.I && col < a.ldp) *reinterpret_cast<f4*>(out + (int64_t)row * a.ldp + col) = fin[i][j];
      }
  } else {
    // The wave's sub-tile goes through its own part of LDS, CR rows at a time, so that a lane gets eight
    // columns of a row (one generator call, one 16-byte access) and neighbouring lanes the row's next
    // ones: rows of 16 lanes' accesses instead of pieces of 32 bytes, and a loop instead of a body for
    // every accumulator.  U row groups at a time have their residual loads in flight together.
    typedef Turned<WM, WN, KG> TU;
    constexpr int CR = TU::CR, PITCH = TU::PITCH, LPR = WN / 8, RPI = 64 / LPR, IT = CR / RPI;
    constexpr int U = BIG ? 4 : IT < 2 ? 1 : 2;
    __syncthreads();  // the LDS of the stages, and of the sums, is free
    float* const mine = reinterpret_cast<float*>(smem + wave * TU::BYTES);
    const uint64_t sub = e.drop.thr ? drop_sub(e.drop) : 0;
    const int lr = lane / LPR;
    auto out = [&](auto chunk) __attribute__((always_inline)) {
      constexpr int CH = decltype(chunk)::value;
#pragma unroll
      for (int i = 0; i < CR / 16; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
          *reinterpret_cast<f4*>(&mine[(16 * i + (lane & 15)) * PITCH + 16 * j + 4 * g]) = fin[CH * (CR / 16) + i][j];
      wave_sync();
      if (col < e.n) {
#pragma unroll 1
        for (int it = 0; it < IT; it += U) {
          F8 res[U], v[U];
          const int r = it * RPI + lr, row = wr + CH * CR + r;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (e.res && row + u * RPI < a.I) res[u] = load8((const T*)e.res + (int64_t)(row + u * RPI) * e.ldr, col, e.n);
            const float* p = &mine[(r + u * RPI) * PITCH + lc];
            v[u].lo = *reinterpret_cast<const f4*>(p);
            v[u].hi = *reinterpret_cast<const f4*>(p + 4);
          }
          with_act(e.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (row + u * RPI < a.I)
                v[u] = value_of<T, decltype(act)::value>(e, row + u * RPI, col, sub, v[u], b);
          });
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (row + u * RPI >= a.I) continue;
            if (e.res) {
              v[u].lo += res[u].lo;
              v[u].hi += res[u].hi;
            }
            store8((T*)e.y + (int64_t)(row + u * RPI) * e.ldy, col, e.n, v[u]);
          }
        }
      }
      wave_sync();
    };
    out(std::integral_constant<int, 0>());
    if constexpr (TU::ROWS / CR == 2) out(std::integral_constant<int, 1>());
    static_assert(TU::ROWS / CR <= 2, "chunks of a wave's rows");
  }
#endif
}

// Dynamic LDS above 64 KiB is asked for once per kernel and device (the call costs a launch's time).
inline void allow_lds(const void* fn, size_t bytes, std::atomic<uint64_t>& done) {
  if (bytes <= 65536) return;
  int dev = 0;
  (void)hipGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return;
  dgprf::set_lds_limit(fn, bytes);
  done.fetch_or(bit, std::memory_order_relaxed);
}

template <class T, bool AKC, bool BKC, int BM, int BN, int WM, int WN, int KB, int ST, int OCC, int KG = 1>
hipError_t launch_tile(const GemmArgs& a, const EpiDev& e, hipStream_t s) {
  constexpr int SUMS = KG > 1 ? BM * BN * 4 : 0;  // of two groups
  constexpr size_t lds = std::max({ST * (BM + BN) * KB, SUMS, 4 * KG * Turned<WM, WN, KG>::BYTES});
  static_assert(lds <= 160 * 1024, "LDS of a CU");
  const dim3 grid((unsigned)(a.n_mt * a.n_nt * a.splits));
  if (a.part) {
    const auto fn = &k_dense<T, AKC, BKC, BM, BN, WM, WN, KB, ST, OCC, KG, true>;
    static std::atomic<uint64_t> done;
    allow_lds((const void*)fn, lds, done);
    hipLaunchKernelGGL(fn, grid, dim3(256 * KG), lds, s, a, e);
  } else {
    const auto fn = &k_dense<T, AKC, BKC, BM, BN, WM, WN, KB, ST, OCC, KG, false>;
    static std::atomic<uint64_t> done;
    allow_lds((const void*)fn, lds, done);
    hipLaunchKernelGGL(fn, grid, dim3(256 * KG), lds, s, a, e);
  }
  return hipGetLastError();
}

template <class T, bool AKC, bool BKC>
hipError_t launch_layout(int tile, const GemmArgs& a, const EpiDev& e, hipStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (tile == TILE_256) return launch_tile<T, AKC, BKC, 256, 256, 128, 128, 128, 2, 1>(a, e, s);
    if (tile == TILE_256N) return launch_tile<T, AKC, BKC, 256, 128, 128, 64, 64, 3, 2>(a, e, s);
    if (tile == TILE_256G) return launch_tile<T, AKC, BKC, 256, 128, 128, 64, 128, 3, 2, 2>(a, e, s);
    if (tile == TILE_128G) return launch_tile<T, AKC, BKC, 128, 128, 64, 64, 128, 3, 2, 2>(a, e, s);
  }
  if (tile == TILE_128) return launch_tile<T, AKC, BKC, 128, 128, 64, 64, 64, 4, 2>(a, e, s);
  if (tile == TILE_64) return launch_tile<T, AKC, BKC, 64, 64, 32, 32, 128, 3, 3, sizeof(T) == 4 ? 2 : 1>(a, e, s);
  return launch_tile<T, AKC, BKC, 32, 128, 32, 32, 128, 4, 2>(a, e, s);
}

template <class T>
hipError_t launch_gemm(int layout, int tile, const GemmArgs& a, const EpiDev& e, hipStream_t s) {
  if (layout == LAYOUT_NN) return launch_layout<T, true, false>(tile, a, e, s);
  if (layout == LAYOUT_NT) return launch_layout<T, true, true>(tile, a, e, s);
  return launch_layout<T, false, false>(tile, a, e, s);
}

}  // namespace dense
