// dense.hip — the dense operators' entry points (dgprf_linear_forward / _backward, dgprf_dropout),
// the rules that choose their kernels, and the kernels around the tiled product (dense_gemm_impl.h).
#include <algorithm>
#include <cmath>

#include "dense_common.h"

using namespace dense;

namespace {

inline int64_t up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
inline int64_t cdiv(int64_t x, int64_t m) { return (x + m - 1) / m; }

// A launch has fewer than 2^32 threads in a dimension; element-wise kernels of more workgroups than
// kGridX have rows of them.
constexpr int kGridX = 1 << 22;
inline dim3 grid_of(int64_t blocks) {
  return dim3((unsigned)std::min<int64_t>(blocks, kGridX), (unsigned)cdiv(blocks, kGridX));
}
__device__ __forceinline__ int64_t block_of() { return (int64_t)blockIdx.y * kGridX + blockIdx.x; }

// ---------------------------------------------------------------- packing
// Rows of `cols` elements at any stride and alignment to rows of a multiple of eight, zero-padded: the
// tiled product reads 16 bytes at a time.  Two matrices a launch, so that a product with two odd operands
// pays one.
struct PackDev {
  const void* in;
  void* out;  // null: no matrix
  int64_t ld;
  int32_t rows, cols;
  __host__ __device__ int per() const { return (cols + 7) >> 3; }
  __host__ __device__ int64_t blocks() const { return out ? ((int64_t)rows * per() + 255) / 256 : 0; }
};
template <class T>
__device__ __forceinline__ void pack_block(const PackDev& a, const PackDev& b, int64_t at) {
  const int64_t na = a.blocks();
  const bool first = at < na;
  const PackDev p = first ? a : b;
  const int per = p.per();
  const int64_t q = (first ? at : at - na) * 256 + threadIdx.x;
  if (q >= (int64_t)p.rows * per) return;
  const int64_t row = row_of(q, per);
  const int col = (int)(q - row * per) * 8;
  const F8 v = load8((const T*)p.in + row * p.ld, col, p.cols);
  store8_whole((T*)p.out + row * (per * 8) + col, v);
}
template <class T>
__global__ __launch_bounds__(256) void k_pack(const PackDev a, const PackDev b) {
  pack_block<T>(a, b, block_of());
}

// ---------------------------------------------------------------- joining the parts of K
// Sums the parts and applies the epilogue.  A workgroup takes 64 groups of eight columns of a row;
// wave w adds parts w, w + 4, ... (four loads in flight: with few rows the time is the latency of a
// thread's chain of loads), then the four sums are added in order, so a result does not depend on
// which part was ready first.
template <class T>
__global__ __launch_bounds__(256) void k_join(const float* __restrict__ part, int64_t ldp, int parts,
                                              int64_t rows, const EpiDev e) {
  __shared__ __attribute__((aligned(16))) f4 sums[3][2][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t q = (int64_t)blockIdx.x * 64 + lane;
  const bool live = q < rows * e.groups;
  const int64_t row = live ? row_of(q, e.groups) : 0;
  const int col = live ? (int)(q - row * e.groups) * 8 : 0, n = e.n;
  const int64_t stride = rows * ldp;
  F8 v{f4zero(), f4zero()}, b{f4zero(), f4zero()}, r{f4zero(), f4zero()};
  if (live) {
    if (wave == 0) {  // on their way with the parts
      if (e.bias) b = load8((const T*)e.bias, col, n);
      if (e.res) r = load8((const T*)e.res + row * e.ldr, col, n);
    }
    const float* p = part + row * ldp + col;  // ldp % 8 == 0
#pragma unroll 4
    for (int s = wave; s < parts; s += 4) {
      v.lo += *reinterpret_cast<const f4*>(p + s * stride);
      v.hi += *reinterpret_cast<const f4*>(p + s * stride + 4);
    }
  }
  if (wave) {
    sums[wave - 1][0][lane] = v.lo;
    sums[wave - 1][1][lane] = v.hi;
  }
  __syncthreads();
  if (wave || !live) return;
#pragma unroll
  for (int w = 0; w < 3; ++w) {
    v.lo += sums[w][0][lane];
    v.hi += sums[w][1][lane];
  }
  const uint64_t sub = e.drop.thr ? drop_sub(e.drop) : 0;
  with_act(e.act, [&](auto act) { v = value_of<T, decltype(act)::value>(e, row, col, sub, v, b); });
  if (e.res) {
    v.lo += r.lo;
    v.hi += r.hi;
  }
  store8((T*)e.y + row * e.ldy, col, n, v);
}

// ---------------------------------------------------------------- few rows
// z = x W for one row, or two of a long K: W is read once, at memory speed, by many workgroups, and each
// product is a plain multiply-add (from three rows on the tiled product is faster: 4 x 2048 x 8192 in bf16
// 13.2 us, 15.3 this way; 2 x 4096 x 4096 12.9 and 11.4).  A
// workgroup takes 16 lanes' width of columns and up to 1024 k; its 16 k-lanes (4 of a wave, 4 waves)
// take groups of four k each, whose x values are one LDS read, and their sums are added in a fixed
// order.  Parts of K are joined by k_join.
template <class T>
struct Piece {  // 16 bytes of a row
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};
// the first `there` elements of a piece, zeros behind them
template <class T>
__device__ __forceinline__ typename Piece<T>::vec load_piece(const T* p, int there) {
  constexpr int CE = 16 / (int)sizeof(T);
  if (there >= CE) return *reinterpret_cast<const typename Piece<T>::vec*>(p);
  typename Piece<T>::vec v;
#pragma unroll
  for (int c = 0; c < CE; ++c) v[c] = c < there ? p[c] : (T)0.f;
  return v;
}
constexpr int kRowsK = 1024;
template <class T, int MR>
__global__ __launch_bounds__(256) void k_rows(const T* __restrict__ x, int64_t ldx,
                                              const T* __restrict__ w, int64_t ldw, int M, int K, int N,
                                              int k_part, float* __restrict__ part, int64_t ldp) {
  constexpr int CE = 16 / (int)sizeof(T), STRIP = 16 * CE;
  typedef typename Piece<T>::vec vec;
  __shared__ __attribute__((aligned(16))) float xs[MR * kRowsK];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int k0 = blockIdx.y * k_part, kn = min(k_part, K - k0), kp = (kn + 3) & ~3;
  const int col = blockIdx.x * STRIP + (lane & 15) * CE;
  for (int i = tid; i < MR * kp; i += 256) {
    const int m = i / kp, k = i - m * kp;
    xs[m * kRowsK + k] = m < M && k < kn ? (float)x[m * ldx + k0 + k] : 0.f;
  }
  __syncthreads();
  float acc[MR][CE];
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int c = 0; c < CE; ++c) acc[m][c] = 0.f;
  if (col < N) {
    const T* wp = w + (int64_t)k0 * ldw + col;
#pragma unroll 2
    for (int k = (wave * 4 + (lane >> 4)) * 4; k < kn; k += 64) {
      vec v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = k + r < kn ? load_piece<T>(wp + (int64_t)(k + r) * ldw, N - col) : (vec)(T)0.f;
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const f4 xv = *reinterpret_cast<const f4*>(&xs[m * kRowsK + k]);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int c = 0; c < CE; ++c) acc[m][c] = fmaf(xv[r], (float)v[r][c], acc[m][c]);
      }
    }
  }
  __syncthreads();
  // the four k-lanes of a wave, then the four waves
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int c = 0; c < CE; ++c) {
      float s = acc[m][c];
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      if (lane < 16) xs[(wave * MR + m) * STRIP + lane * CE + c] = s;
    }
  __syncthreads();
  float* out = part + (int64_t)blockIdx.y * M * ldp;
  for (int i = tid; i < MR * STRIP; i += 256) {
    const int m = i / STRIP, c = i - m * STRIP, j = blockIdx.x * STRIP + c;
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) s += xs[(v * MR + m) * STRIP + c];
    if (m < M && j < N) out[m * ldp + j] = s;
  }
}

// One row in one launch, for K up to kStripK: a workgroup of 16 waves takes 64 bytes of each row of W and
// all of K, so its sums are complete and it applies the epilogue itself.  A second launch costs a row about
// as much as the product (2048 x 4096 in bf16: 8.0 us this way, 11.7 with parts of K and k_join), but 64
// bytes of a row at a time do not reach the memory's rate (8192 x 2048: 19 and 10.8 us): K is at most what
// a thread has on its way at once, and W at most 8 MiB (2048 x 8192, not in a cache: 13.4 and 11.7 us).
// Neighbouring strips go to one XCD, whose L2 their rows' lines share.
constexpr int kStripAhead = 8, kStripK = 256 * kStripAhead;
constexpr int64_t kStripBytes = 8 << 20;
template <class T>
__global__ __launch_bounds__(1024) void k_strip(const T* __restrict__ x, const T* __restrict__ w, int64_t ldw,
                                                int K, const EpiDev e) {
  constexpr int LPR = 4, CE = 16 / (int)sizeof(T), STRIP = LPR * CE, KL = 1024 / LPR;
  typedef typename Piece<T>::vec vec;
  __shared__ float xs[kStripK];
  __shared__ __attribute__((aligned(16))) float part[16][STRIP];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, kl = tid / LPR;
  int strip;
  {
    const int G = gridDim.x, b = blockIdx.x, xcd = b & 7, q = G >> 3, r = G & 7;
    strip = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (b >> 3);
  }
  const int col = strip * STRIP + (tid % LPR) * CE;
  vec v[kStripAhead];  // on the way while x is
#pragma unroll
  for (int u = 0; u < kStripAhead; ++u) {
    const int k = kl + u * KL;
    v[u] = k < K && col < e.n ? load_piece<T>(w + (int64_t)k * ldw + col, e.n - col) : (vec)(T)0.f;
  }
  const int c0 = strip * STRIP + tid * 8;
  const bool out = tid < STRIP / 8 && c0 < e.n;  // this thread has eight columns of the result
  F8 z{f4zero(), f4zero()}, b{f4zero(), f4zero()}, r{f4zero(), f4zero()};
  if (out && e.bias) b = load8((const T*)e.bias, c0, e.n);
  if (out && e.res) r = load8((const T*)e.res, c0, e.n);
  for (int k = tid; k < K; k += 1024) xs[k] = (float)x[k];
  __syncthreads();
  float acc[CE];
#pragma unroll
  for (int c = 0; c < CE; ++c) acc[c] = 0.f;
#pragma unroll
  for (int u = 0; u < kStripAhead; ++u) {
    const int k = kl + u * KL;
    if (k < K) {
#pragma unroll
      for (int c = 0; c < CE; ++c) acc[c] = fmaf(xs[k], (float)v[u][c], acc[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < CE; ++c) {
    float s = acc[c];
#pragma unroll
    for (int d = LPR; d < 64; d *= 2) s += __shfl_xor(s, d);
    if (lane < LPR) part[wave][lane * CE + c] = s;
  }
  __syncthreads();
  if (!out) return;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const f4* p = reinterpret_cast<const f4*>(&part[i][tid * 8]);
    z.lo += p[0];
    z.hi += p[1];
  }
  const uint64_t sub = e.drop.thr ? drop_sub(e.drop) : 0;
  with_act(e.act, [&](auto act) { z = value_of<T, decltype(act)::value>(e, 0, c0, sub, z, b); });
  if (e.res) {
    z.lo += r.lo;
    z.hi += r.hi;
  }
  store8((T*)e.y, c0, e.n, z);
}

// ---------------------------------------------------------------- dz and its column sums
// dz / s = m dy a'(z) (rounded to the tensors' type, as the matrix instructions take it; its sums for
// db are of the unrounded values), one thread for eight columns and `rows_part` rows; dz is null
// where it would equal dy.  s is applied to the products and to db in 32 bits, because in fp16 s dy
// overflows where their results need not (p = 0.75: from dy = 16376 on).  Workgroups behind those pack the products' other operands, which saves odd
// sizes a launch (dx of 700 x 700 over 3500 in bf16: 28.9 us, 34.7 with two).
struct DzDev {
  const void* dy;
  const void* aux;
  void* dz;
  float* part;  // [parts][ldz] or null
  int64_t lddy, ldaux, ldz;
  int64_t M;
  int32_t N, groups, act, rows_part;
  int32_t strips, parts;  // of 64 groups, and of rows
  DropDev drop;
};
template <class T>
__global__ __launch_bounds__(256) void k_dz(const DzDev d, const PackDev a, const PackDev b) {
  __shared__ __attribute__((aligned(16))) float sums[4][64 * 8];
  const int64_t at = block_of();
  if (at >= (int64_t)d.strips * d.parts) return pack_block<T>(a, b, at - (int64_t)d.strips * d.parts);
  const int part = (int)at / d.strips, strip = (int)at - part * d.strips;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int gi = strip * 64 + lane, col = gi * 8;
  const int64_t m0 = (int64_t)part * d.rows_part, m1 = min(d.M, m0 + d.rows_part);
  const uint64_t sub = d.drop.thr ? drop_sub(d.drop) : 0;
  F8 acc;
  acc.lo = f4zero();
  acc.hi = f4zero();
  if (gi < d.groups) {
    with_act(d.act, [&](auto act) {
      constexpr int ACT = decltype(act)::value;
      constexpr int U = sizeof(T) == 4 ? 2 : 4;  // rows whose loads are in flight together
      for (int64_t m = m0 + wave; m < m1; m += 4 * U) {
        F8 g[U], z[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (m + 4 * u >= m1) continue;
          g[u] = load8((const T*)d.dy + (m + 4 * u) * d.lddy, col, d.N);
          if constexpr (ACT != DGPRF_ACT_NONE) z[u] = load8_whole((const T*)d.aux + (m + 4 * u) * d.ldaux + col);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (m + 4 * u >= m1) continue;
          F8 v = g[u];
          if constexpr (ACT != DGPRF_ACT_NONE) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              v.lo[c] *= slope_of<T, ACT>(z[u].lo[c]);
              v.hi[c] *= slope_of<T, ACT>(z[u].hi[c]);
            }
          }
          // last, so that a dropped element is 0 whatever its gradient and slope
          if (d.drop.thr)
            v = drop8(v, drop_words(d.drop, sub, (uint64_t)(m + 4 * u) * (uint32_t)d.groups + (uint32_t)gi), d.drop);
          // zeros past N: the tiled product multiplies the padding
          if (d.dz) {
            if (col + 8 > d.N) {
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                if (col + c >= d.N) v.lo[c] = 0.f;
                if (col + 4 + c >= d.N) v.hi[c] = 0.f;
              }
            }
            store8_whole((T*)d.dz + (m + 4 * u) * d.ldz + col, v);
          }
          acc.lo += v.lo;
          acc.hi += v.hi;
        }
      }
    });
  }
  if (!d.part) return;
  *reinterpret_cast<f4*>(&sums[wave][lane * 8]) = acc.lo;
  *reinterpret_cast<f4*>(&sums[wave][lane * 8 + 4]) = acc.hi;
  __syncthreads();
  for (int i = threadIdx.x; i < 512; i += 256) {
    const int c = strip * 512 + i;
    if (c < d.ldz) d.part[(int64_t)part * d.ldz + c] = sums[0][i] + sums[1][i] + sums[2][i] + sums[3][i];
  }
}

// db[c] = s times the sum of the parts: 32 columns of a workgroup, 32 threads each, in a fixed order
template <class T>
__global__ __launch_bounds__(1024) void k_db(const float* __restrict__ part, int64_t ldp, int parts, int N,
                                             float s_drop, T* __restrict__ db) {
  __shared__ float sums[32][33];
  const int cl = threadIdx.x & 31, r = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  float s = 0.f;
  if (c < N) {
#pragma unroll 8
    for (int p = r; p < parts; p += 32) s += part[p * ldp + c];
  }
  sums[r][cl] = s;
  __syncthreads();
  for (int h = 16; h > 0; h >>= 1) {
    if (r < h) sums[r][cl] += sums[r + h][cl];
    __syncthreads();
  }
  if (r == 0 && c < N) db[c] = (T)(s_drop * sums[0][cl]);
}

// ---------------------------------------------------------------- dropout
// FLAT: rows without gaps whose length is a multiple of 8: the group's number is its place
template <class T, bool FLAT>
__global__ __launch_bounds__(256) void k_dropout(const T* __restrict__ x, int64_t ldx,
                                                 const T* __restrict__ res, int64_t ldr,
                                                 T* __restrict__ y, int64_t total, int groups, int n,
                                                 const DropDev d) {
  const int64_t q = block_of() * 256 + threadIdx.x;
  if (q >= total) return;
  const uint64_t sub = drop_sub(d);
  if constexpr (FLAT) {
    F8 v = load8_whole(x + 8 * q);
    if (d.thr) v = drop8(v, drop_words(d, sub, (uint64_t)q), d);
    if (res) {
      const F8 r = load8_whole(res + 8 * q);
      v.lo += r.lo;
      v.hi += r.hi;
    }
    store8_whole(y + 8 * q, v);
  } else {
    const int64_t row = row_of(q, groups);
    const int col = (int)(q - row * groups) * 8;
    F8 v = load8(x + row * ldx, col, n);
    if (d.thr) v = drop8(v, drop_words(d, sub, (uint64_t)q), d);
    if (res) {
      const F8 r = load8(res + row * ldr, col, n);
      v.lo += r.lo;
      v.hi += r.hi;
    }
    store8(y + row * (int64_t)n, col, n, v);
  }
}

// ---------------------------------------------------------------- choices
// rows of 16-byte pieces: what the tiled product's loads to LDS read in place
bool in_place(const void* p, int64_t ld, int64_t cols, int es) {
  return (uintptr_t)p % 16 == 0 && ld * es % 16 == 0 && cols * es % 16 == 0;
}

struct Shape {
  int tile, n_mt, n_nt, splits, stages, stages_split;
};
constexpr int64_t kMaxWidth = 1 << 20;  // a tile's rows stay within a buffer descriptor's range
constexpr int64_t kMaxM = ((int64_t)1 << 31) - 512;  // row numbers up to a tile's end, and of stages, fit 32 bits
constexpr int64_t kMaxRow = ((int64_t)1 << 31) - 8;  // the end of a row's last group fits 32 bits

// Tile and parts of K for an I x J result: the pair with the least estimated time.  A CU that gets c
// workgroups takes  fixed + c (out + rate K / parts)  microseconds (K in units of 1024); joining P
// parts costs a launch and P I J 8 bytes of traffic at 5.5 TB/s.  The three numbers of a tile come from
// runs with one to four workgroups per CU at K = 512 .. 8192 (2048 x 2048 x 2048 in bf16: 47 us with
// 256 x 256 tiles, 32 with 256 x 128, 23 with 128 x 128, 30 with 64 x 64; 64 x 4096 x 4096: 12.4 with
// 32 x 128 and four parts, 19 with one).  Tiles with two groups of waves are for launches of at most one
// workgroup a CU: nothing runs beside a workgroup's last rows (256 x 128, 4096 x 2048 over K = 8192: 109 us,
// 126 with one group; 8192 x 8192 over 1024: 164 and 131).
struct TileCost {
  float fixed, out, rate;
};
constexpr TileCost kCost16[TILES] = {{3.f, 12.f, 22.5f}, {9.f, 1.f, 14.4f}, {6.f, 0.f, 13.f},  {7.6f, 0.f, 7.f},
                                     {5.f, 0.5f, 9.2f},  {4.5f, 0.5f, 3.3f}, {4.f, 0.5f, 3.4f}};
// fp32: 65 us of 4096 multiply-adds a clock; the 256-wide tiles' accumulators and fragments do not fit
constexpr TileCost kCost32[TILES] = {{}, {}, {}, {}, {5.f, 1.f, 59.f}, {5.f, 0.5f, 17.f}, {5.f, 0.5f, 17.5f}};

Shape shape_of(int64_t I, int64_t J, int64_t K, int es, int layout) {
  Shape best{};
  float least = INFINITY;
  for (int tile = es == 4 ? TILE_128 : TILE_256; tile < TILES; ++tile) {
    const TileShape ts = kTiles[tile];
    TileCost tc = es == 4 ? kCost32[tile] : kCost16[tile];
    // both operands read as whole fragments (1777 x 1008 over 2048: 15.6 us, 19.1 with 32 x 128)
    if (es == 2 && tile == TILE_64 && layout == LAYOUT_NT) tc.rate *= 0.9f;
    const int64_t mt = cdiv(I, ts.bm), nt = cdiv(J, ts.bn), stages = cdiv(K * es, ts.kb);
    // threads of a launch (check_dims leaves room for the 128 x 128 tile)
    if (mt * nt * ts.threads >= (int64_t)1 << 32) continue;
    for (int64_t want = 1; want <= 32; want *= 2) {
      if (want > 1 && (stages < 4 * want || mt * nt > 1024)) break;
      const int64_t per = cdiv(stages, want), parts = cdiv(stages, per);
      if ((tile == TILE_256G || tile == TILE_128G) && mt * nt * parts > 256) break;
      const float k = (float)per * ts.kb / es / 1024.f, rounds = (float)cdiv(mt * nt * parts, 256);
      float t = tc.fixed + rounds * (tc.out + tc.rate * k);
      if (parts > 1) t += 4.f + (float)parts * I * J * 8.f / 5.5e6f;
      if (t < least) {
        least = t;
        best = Shape{tile, (int)mt, (int)nt, (int)parts, (int)stages, (int)per};
      }
    }
  }
  return best;
}
int64_t part_bytes(const Shape& s, int64_t I, int64_t J) {
  return s.splits > 1 ? up((int64_t)s.splits * I * up(J, 8) * 4, 256) : 0;
}

// parts of K for the few-row kernel: enough workgroups to keep the memory busy
void rows_shape(int64_t N, int64_t K, int es, int* k_part, int* parts) {
  const int64_t strips = cdiv(N, 256 / es);
  int64_t p = std::max<int64_t>(cdiv(K, kRowsK), std::min<int64_t>(cdiv(1024, strips), cdiv(K, 64)));
  *k_part = (int)up(cdiv(K, p), 4);
  *parts = (int)cdiv(K, *k_part);
}

struct Scratch {  // a bump allocator over the caller's scratch; base null: only counts
  char* base;
  int64_t used = 0;
  void* take(int64_t bytes) {
    void* p = base ? base + used : nullptr;
    used += up(bytes, 256);
    return p;
  }
};

DropDev drop_dev(int32_t thr, uint64_t seed, uint64_t sub, const int64_t* step) {
  DropDev d;
  d.thr = (uint32_t)thr;
  d.scale = thr < 65536 ? 65536.f / (float)(65536 - thr) : 0.f;
  d.k0 = (uint32_t)seed;
  d.k1 = (uint32_t)(seed >> 32);
  d.sub = sub;
  d.step = step;
  return d;
}

hipError_t gemm(int dtype, int layout, const Shape& s, const GemmArgs& a, const EpiDev& e, hipStream_t st) {
  if (dtype == DGPRF_BF16) return launch_gemm_bf16(layout, s.tile, a, e, st);
  if (dtype == DGPRF_F16) return launch_gemm_f16(layout, s.tile, a, e, st);
  return launch_gemm_f32(layout, s.tile, a, e, st);
}

// f((T*)nullptr) for the element type
template <class F>
hipError_t with_type(int dtype, F f) {
  if (dtype == DGPRF_BF16) return f((bf16_t*)nullptr);
  if (dtype == DGPRF_F16) return f((f16_t*)nullptr);
  return f((float*)nullptr);
}
#define DENSE_T(p) typename std::remove_pointer<decltype(p)>::type

hipError_t pack(int dtype, const PackDev& a, const PackDev& b, hipStream_t s) {
  const int64_t blocks = a.blocks() + b.blocks();
  if (!blocks) return hipSuccess;
  return with_type(dtype, [&](auto* t) {
    hipLaunchKernelGGL((k_pack<DENSE_T(t)>), grid_of(blocks), dim3(256), 0, s, a, b);
    return hipGetLastError();
  });
}
// An operand [rows][cols] as the product reads it: in place, or a packed copy in scratch (p).  ld and
// width become those of what is read.
const void* operand(const void* m, int64_t* ld, int64_t rows, int64_t cols, int64_t* width, int es, Scratch& sc,
                    PackDev* p) {
  *p = PackDev{};
  *width = cols;
  if (in_place(m, *ld, cols, es)) return m;
  *p = PackDev{m, sc.take(rows * up(cols, 8) * es), *ld, (int)rows, (int)cols};
  *ld = *width = up(cols, 8);
  return p->out;
}

hipError_t join(int dtype, const float* part, int64_t ldp, int parts, int64_t rows, const EpiDev& e,
                hipStream_t s) {
  return with_type(dtype, [&](auto* t) {
    typedef DENSE_T(t) T;
    hipLaunchKernelGGL((k_join<T>), dim3((unsigned)cdiv(rows * e.groups, 64)), dim3(256), 0, s, part, ldp,
                       parts, rows, e);
    return hipGetLastError();
  });
}

template <class T, int MR>
hipError_t rows_launch(const dgprf_linear_t& a, int k_part, int parts, float* part, int64_t ldp,
                       hipStream_t s) {
  const dim3 grid((unsigned)cdiv(a.n, 256 / (int)sizeof(T)), (unsigned)parts);
  hipLaunchKernelGGL((k_rows<T, MR>), grid, dim3(256), 0, s, (const T*)a.x, a.ldx, (const T*)a.w, a.ldw, (int)a.m,
                     (int)a.k, (int)a.n, k_part, part, ldp);
  return hipGetLastError();
}

// One product of the layer: [I][J] over K into scratch parts or straight through the epilogue.
hipError_t product(int dtype, int layout, const void* A, int64_t lda, const void* B, int64_t ldb, int64_t I,
                   int64_t J, int64_t Ia, int64_t Ja, int64_t Ka, int64_t Kb, const EpiDev& e, Scratch& sc,
                   hipStream_t st, bool run) {
  const int es = elem_size(dtype);
  const Shape s = shape_of(I, J, std::max(Ka, Kb), es, layout);
  float* part = (float*)sc.take(part_bytes(s, I, J));
  if (!run) return hipSuccess;
  GemmArgs a;
  a.A = A;
  a.B = B;
  a.lda = lda;
  a.ldb = ldb;
  a.I = (int)I;
  a.J = (int)J;
  a.Ia = (int)Ia;
  a.Ja = (int)Ja;
  a.Ka = (int)Ka;
  a.Kb = (int)Kb;
  a.n_mt = s.n_mt;
  a.n_nt = s.n_nt;
  a.splits = s.splits;
  a.stages = s.stages;
  a.stages_split = s.stages_split;
  a.part = s.splits > 1 ? part : nullptr;
  a.ldp = up(J, 8);
  hipError_t err = gemm(dtype, layout, s, a, e, st);
  if (err == hipSuccess && a.part) err = join(dtype, part, a.ldp, s.splits, I, e, st);
  return err;
}

// y = s times the product
EpiDev epi_plain(void* y, int64_t n, float s) {
  EpiDev e{};
  e.y = y;
  e.ldy = n;
  e.n = (int)n;
  e.groups = (int)cdiv(n, 8);
  e.drop.scale = s;
  return e;
}

int check_drop(int32_t thr) { return thr < 0 || thr > 65536 ? DGPRF_E_ARG : DGPRF_OK; }

int check_dims(int32_t dtype, int32_t act, int64_t m, int64_t k, int64_t n, int64_t ldx, int64_t ldw) {
  if (dtype != DGPRF_F32 && dtype != DGPRF_F16 && dtype != DGPRF_BF16) return DGPRF_E_ARG;
  if (act < DGPRF_ACT_NONE || act > DGPRF_ACT_SILU) return DGPRF_E_ARG;
  if (m < 0 || k < 1 || n < 1 || ldx < k || ldw < n) return DGPRF_E_SHAPE;
  if (m > kMaxM || k > kMaxWidth || n > kMaxWidth || ldx > kMaxWidth || ldw > kMaxWidth)
    return DGPRF_E_SHAPE;
  // 128 x 128 tiles of a launch: 2^38 elements
  const int64_t w = std::max(k, n), most = (int64_t)1 << 24;
  if (cdiv(m, 128) * cdiv(w, 128) >= most || cdiv(k, 128) * cdiv(n, 128) >= most) return DGPRF_E_SHAPE;
  return DGPRF_OK;
}

// The forward pass; run = false only counts its scratch.
hipError_t forward(const dgprf_linear_t& a, Scratch& sc, hipStream_t st, bool run) {
  const int es = elem_size(a.dtype);
  const int64_t m = a.m, k = a.k, n = a.n;
  EpiDev e = epi_plain(a.y, n, 1.f);
  e.bias = a.bias;
  e.res = a.res;
  e.aux = a.act != DGPRF_ACT_NONE ? a.aux : nullptr;
  e.ldr = a.ldr;
  e.ldaux = up(n, 8);
  e.act = a.act;
  e.drop = drop_dev(a.drop_thr, a.seed, a.sub, a.step);
  if (m == 1 && k <= kStripK && k * n * es <= kStripBytes) {
    if (!run) return hipSuccess;
    return with_type(a.dtype, [&](auto* t) {
      typedef DENSE_T(t) T;
      hipLaunchKernelGGL((k_strip<T>), dim3((unsigned)cdiv(n, 64 / (int)sizeof(T))), dim3(1024), 0, st,
                         (const T*)a.x, (const T*)a.w, a.ldw, (int)k, e);
      return hipGetLastError();
    });
  }
  if (m == 1 || (m == 2 && k > kStripK)) {
    int k_part, parts;
    rows_shape(n, k, es, &k_part, &parts);
    const int64_t ldp = up(n, 8);
    float* part = (float*)sc.take((int64_t)parts * m * ldp * 4);
    if (!run) return hipSuccess;
    hipError_t err = with_type(a.dtype, [&](auto* t) {
      typedef DENSE_T(t) T;
      if (m == 1) return rows_launch<T, 1>(a, k_part, parts, part, ldp, st);
      return rows_launch<T, 2>(a, k_part, parts, part, ldp, st);
    });
    return err == hipSuccess ? join(a.dtype, part, ldp, parts, m, e, st) : err;
  }
  int64_t ldx = a.ldx, ldw = a.ldw, ka, nb;
  PackDev px, pw;
  const void* x = operand(a.x, &ldx, m, k, &ka, es, sc, &px);
  const void* w = operand(a.w, &ldw, k, n, &nb, es, sc, &pw);
  if (run)
    if (hipError_t err = pack(a.dtype, px, pw, st)) return err;
  return product(a.dtype, LAYOUT_NN, x, ldx, w, ldw, m, n, 0, nb, ka, k, e, sc, st, run);
}

hipError_t backward(const dgprf_linear_grad_t& a, Scratch& sc, hipStream_t st, bool run) {
  const int es = elem_size(a.dtype);
  const int64_t m = a.m, k = a.k, n = a.n;
  hipError_t err = hipSuccess;
  const DropDev drop = drop_dev(a.drop_thr, a.seed, a.sub, a.step);
  // dz / s, unless it is dy and dy can be read in place
  const bool products = a.dx || a.dw;
  // (rows that share memory are copied apart: their product's K range has no end to check against)
  const bool same = a.act == DGPRF_ACT_NONE && a.drop_thr == 0 && a.lddy >= n && in_place(a.dy, a.lddy, n, es);
  const void* dz = a.dy;
  int64_t lddz = a.lddy, na = n;
  if (products && !same) {
    lddz = na = up(n, 8);
    dz = sc.take(m * lddz * es);
  }
  int64_t ldx = a.ldx, ldw = a.ldw, ka = k, nb = n;
  PackDev px{}, pw{};
  const void* w = a.dx ? operand(a.w, &ldw, k, n, &nb, es, sc, &pw) : nullptr;
  const void* x = a.dw ? operand(a.x, &ldx, m, k, &ka, es, sc, &px) : nullptr;
  if ((products && !same) || a.db) {
    DzDev d{};
    d.dy = a.dy;
    d.aux = a.aux;
    d.dz = products && !same ? const_cast<void*>(dz) : nullptr;
    d.lddy = a.lddy;
    d.ldaux = d.ldz = up(n, 8);
    d.M = m;
    d.N = (int)n;
    d.groups = (int)cdiv(n, 8);
    d.act = a.act;
    d.drop = drop;
    d.drop.scale = 1.f;
    d.strips = (int)cdiv(d.groups, 64);
    // workgroups enough to fill the chip, down to a row for each wave
    const int64_t want = std::max<int64_t>(1, std::min<int64_t>(cdiv(1024, d.strips), cdiv(m, 4)));
    d.rows_part = (int)up(cdiv(m, want), 4);
    d.parts = (int)cdiv(m, d.rows_part);
    if (a.db) d.part = (float*)sc.take(d.parts * d.ldz * 4);
    if (run) {
      err = with_type(a.dtype, [&](auto* t) {
        typedef DENSE_T(t) T;
        hipLaunchKernelGGL((k_dz<T>), grid_of((int64_t)d.strips * d.parts + pw.blocks() + px.blocks()), dim3(256), 0, st,
                           d, pw, px);
        hipError_t er = hipGetLastError();
        if (er == hipSuccess && a.db) {
          hipLaunchKernelGGL((k_db<T>), dim3((unsigned)cdiv(n, 32)), dim3(1024), 0, st, d.part, d.ldz, d.parts,
                             (int)n, drop.scale, (T*)a.db);
          er = hipGetLastError();
        }
        return er;
      });
      if (err != hipSuccess) return err;
    }
  } else if (run && (err = pack(a.dtype, pw, px, st)) != hipSuccess) {
    return err;
  }
  if (a.dx) {  // [m][k] = s (dz / s) [m][n] (W [k][n])^T
    err = product(a.dtype, LAYOUT_NT, dz, lddz, w, ldw, m, k, 0, 0, na, nb, epi_plain(a.dx, k, drop.scale), sc, st, run);
    if (err != hipSuccess) return err;
  }
  if (a.dw)  // [k][n] = s (x [m][k])^T (dz / s) [m][n]
    err = product(a.dtype, LAYOUT_TN, x, ldx, dz, lddz, k, n, ka, na, m, m, epi_plain(a.dw, n, drop.scale), sc, st, run);
  return err;
}

// zeros without a memset node (a captured graph replays a fill kernel)
__global__ __launch_bounds__(256) void k_zero(uint16_t* p, int64_t n) {
  const int64_t i = block_of() * 256 + threadIdx.x;
  if (i < n) p[i] = 0;
}
hipError_t zero(void* p, int64_t bytes, hipStream_t s) {
  hipLaunchKernelGGL(k_zero, grid_of(cdiv(bytes / 2, 256)), dim3(256), 0, s, (uint16_t*)p, bytes / 2);
  return hipGetLastError();
}

int hip_rc(hipError_t e) { return e == hipSuccess ? DGPRF_OK : DGPRF_E_HIP; }

int check_forward(const dgprf_linear_t* a) {
  if (!a) return DGPRF_E_ARG;
  int rc = check_dims(a->dtype, a->act, a->m, a->k, a->n, a->ldx, a->ldw);
  if (!rc) rc = check_drop(a->drop_thr);
  if (!rc && a->res && (a->ldr < 0 || (a->ldr > 0 && a->ldr < a->n))) rc = DGPRF_E_SHAPE;
  return rc;
}
int check_backward(const dgprf_linear_grad_t* a) {
  if (!a) return DGPRF_E_ARG;
  int rc = check_dims(a->dtype, a->act, a->m, a->k, a->n, a->ldx, a->ldw);
  if (!rc) rc = check_drop(a->drop_thr);
  if (!rc && (a->lddy < 0 || (a->lddy > 0 && a->lddy < a->n) || a->lddy > kMaxWidth)) rc = DGPRF_E_SHAPE;
  return rc;
}

}  // namespace

extern "C" {

int dgprf_linear_scratch(const dgprf_linear_t* a, int64_t* bytes_out) {
  int rc = check_forward(a);
  if (rc) return rc;
  if (!bytes_out) return DGPRF_E_ARG;
  Scratch sc{nullptr};
  if (a->m > 0) (void)forward(*a, sc, nullptr, false);
  *bytes_out = sc.used;
  return DGPRF_OK;
}

int dgprf_linear_forward(const dgprf_linear_t* a, void* scratch, int64_t scratch_bytes, void* stream) {
  int64_t need = 0;
  int rc = dgprf_linear_scratch(a, &need);
  if (rc) return rc;
  if (a->m == 0) return DGPRF_OK;
  if (!a->x || !a->w || !a->y) return DGPRF_E_ARG;
  if (need > 0 && (!scratch || scratch_bytes < need || (uintptr_t)scratch % 16)) return DGPRF_E_ARG;
  if (a->aux && (uintptr_t)a->aux % 16) return DGPRF_E_ARG;
  Scratch sc{(char*)scratch};
  return hip_rc(forward(*a, sc, reinterpret_cast<hipStream_t>(stream), true));
}

int dgprf_linear_grad_scratch(const dgprf_linear_grad_t* a, int64_t* bytes_out) {
  int rc = check_backward(a);
  if (rc) return rc;
  if (!bytes_out) return DGPRF_E_ARG;
  Scratch sc{nullptr};
  if (a->m > 0) (void)backward(*a, sc, nullptr, false);
  *bytes_out = sc.used;
  return DGPRF_OK;
}

int dgprf_linear_backward(const dgprf_linear_grad_t* a, void* scratch, int64_t scratch_bytes, void* stream) {
  int64_t need = 0;
  int rc = dgprf_linear_grad_scratch(a, &need);
  if (rc) return rc;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (a->m == 0) {  // sums over no rows
    const int es = elem_size(a->dtype);
    hipError_t e = hipSuccess;
    if (a->dw) e = zero(a->dw, a->k * a->n * es, s);
    if (e == hipSuccess && a->db) e = zero(a->db, a->n * es, s);
    return hip_rc(e);
  }
  if (!a->dy || (a->dx && !a->w) || (a->dw && !a->x)) return DGPRF_E_ARG;
  if (a->act != DGPRF_ACT_NONE && !a->aux) return DGPRF_E_ARG;
  if (a->aux && (uintptr_t)a->aux % 16) return DGPRF_E_ARG;
  if (need > 0 && (!scratch || scratch_bytes < need || (uintptr_t)scratch % 16)) return DGPRF_E_ARG;
  Scratch sc{(char*)scratch};
  return hip_rc(backward(*a, sc, s, true));
}

int dgprf_dropout(int32_t dtype, const void* x, int64_t rows, int64_t n, int64_t ldx, const void* res,
                  int64_t ldr, int32_t drop_thr, uint64_t seed, uint64_t sub, const int64_t* step, void* y,
                  void* stream) {
  if (dtype != DGPRF_F32 && dtype != DGPRF_F16 && dtype != DGPRF_BF16) return DGPRF_E_ARG;
  if (check_drop(drop_thr)) return DGPRF_E_ARG;
  if (rows < 0 || n < 0 || n > kMaxRow || (rows > 1 && ldx != 0 && ldx < n) || ldx < 0) return DGPRF_E_SHAPE;
  if (res && (ldr < 0 || (rows > 1 && ldr != 0 && ldr < n))) return DGPRF_E_SHAPE;
  if (rows == 0 || n == 0) return DGPRF_OK;
  if (!x || !y) return DGPRF_E_ARG;
  const int64_t groups = cdiv(n, 8);
  if (rows > ((int64_t)1 << 39) / groups) return DGPRF_E_SHAPE;
  const int64_t total = rows * groups;
  const bool flat = n % 8 == 0 && (rows == 1 || (ldx == n && (!res || ldr == n)));
  const DropDev d = drop_dev(drop_thr, seed, sub, step);
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  return hip_rc(with_type(dtype, [&](auto* t) {
    typedef DENSE_T(t) T;
    const dim3 grid = grid_of(cdiv(total, 256));
    if (flat)
      hipLaunchKernelGGL((k_dropout<T, true>), grid, dim3(256), 0, s, (const T*)x, ldx, (const T*)res, ldr, (T*)y,
                         total, (int)groups, (int)n, d);
    else
      hipLaunchKernelGGL((k_dropout<T, false>), grid, dim3(256), 0, s, (const T*)x, ldx, (const T*)res, ldr, (T*)y,
                         total, (int)groups, (int)n, d);
    return hipGetLastError();
  }));
}

}  // extern "C"
