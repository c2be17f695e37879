// Layer norm over the last axis, forward and backward.
//
//   mean = sum x / C,  rstd = 1 / sqrt(sum (x - mean)^2 / C + eps),  xh = (x - mean) rstd,  y = xh w + b
//   gw = dy w,  dx = rstd (gw - sum gw / C - xh sum(gw xh) / C),  dw = sum_rows dy xh,  db = sum_rows dy
//
// All of it is bound by memory: the forward reads x and writes y, the backward reads x and dy and writes dx.  A thread
// owns the same few columns of all rows its block visits, so that the weights and the sums for dw and db stay in
// registers; TPR threads share a row, and every thread has several rows in flight, which is what hides the latency of
// memory between the two sums that a row needs before it can be written.  The variance is taken about the mean and not
// as a difference of squares, statistics and sums are float32, y and dx are rounded once.  The blocks' sums for dw and db
// go to a scratch buffer and a second kernel adds them in a fixed order, so that a result never depends on the order of
// atomics.
//
// 294912 rows of 1024 (bf16): forward 211 us, 5.7 TB/s, and backward 330 us, 5.5 TB/s, 87 and 84 % of a copy's rate; 100352
// rows of 128: 10.8 us and 17.8 us, which is the latency of the few rows each thread has; 64 rows: 2.4 us and 4.0 us.
#include <math.h>

#include <atomic>
#include <type_traits>

#include "f32x2.cuh"
#include "launch.cuh"

namespace nb {
namespace {

// `VB` bytes of `T` as loaded by one instruction.
template <int VB> struct Raw;
template <> struct Raw<16> { typedef uint4 type; };
template <> struct Raw<4> { typedef uint32_t type; };
template <> struct Raw<2> { typedef uint16_t type; };

template <typename T, int VB>
__device__ __forceinline__ void unpack(const typename Raw<VB>::type& raw, float* out) {
  const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
  for (int i = 0; i < VB / (int)sizeof(T); ++i) out[i] = to_f<T>(e[i]);
}
template <typename T, int VB>
__device__ __forceinline__ typename Raw<VB>::type pack(const float* in) {
  typename Raw<VB>::type raw;
  T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (int i = 0; i < VB / (int)sizeof(T); ++i) e[i] = from_f<T>(in[i]);
  return raw;
}

// N consecutive weights from column `col` (a multiple of N) as float32; the weights are T or float32.
template <typename T, int N>
__device__ __forceinline__ void load_weights(const void* w, bool f32, int col, float* out) {
  if (f32) {
    const float* p = static_cast<const float*>(w) + col;
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const float4 v = __ldg(reinterpret_cast<const float4*>(p) + i);
        out[4 * i] = v.x; out[4 * i + 1] = v.y; out[4 * i + 2] = v.z; out[4 * i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = __ldg(p + i);
    }
  } else {
    constexpr int VB = N * (int)sizeof(T);
    unpack<T, VB>(__ldg(reinterpret_cast<const typename Raw<VB>::type*>(static_cast<const T*>(w) + col)), out);
  }
}

// A thread's share of the weights, `none` where there are none.
template <typename T, int VE, int TPR, int NV>
__device__ __forceinline__ void weight_row(const void* w, bool f32, int lane, int C, float none, f32x2 (&out)[NV * VE / 2]) {
  float f[NV * VE];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * TPR + lane) * VE;
#pragma unroll
    for (int j = 0; j < VE; ++j) f[i * VE + j] = none;
    if (col < C && w != nullptr) load_weights<T, VE>(w, f32, col, f + i * VE);
  }
#pragma unroll
  for (int j = 0; j < NV * VE / 2; ++j) out[j] = pair(f[2 * j], f[2 * j + 1]);
}

struct NormArgs {
  const void* x;
  const void* weight;   // may be null
  const void* bias;     // may be null
  void* y;
  float* mean;          // may be null (both)
  float* rstd;
  // backward
  const void* dy;
  void* dx;             // may be null
  float* part;          // [blocks, 2, C]; null when neither dweight nor dbias is wanted
  uint32_t rows;
  int C;
  // row r of x starts at (r / inner) * outer_stride + (r % inner) * inner_stride elements
  uint32_t inner;
  long long outer_stride, inner_stride;
  float eps, inv_c;
  int w_f32;
};

__device__ __forceinline__ long long row_start(const NormArgs& a, uint32_t r) {
  if (a.inner == 1) return (long long)r * a.outer_stride;
  const uint32_t o = r / a.inner;
  return (long long)o * a.outer_stride + (long long)(r - o * a.inner) * a.inner_stride;
}

// Sums over the TPR threads of a row, for R rows at once; every thread gets them.  Rows wider than a warp meet in `buf`
// [R][warps]: two buffers used in turn make one barrier per sum enough.
template <int TPR, int R, int WARPS>
__device__ __forceinline__ void row_sums(float (&v)[R], float (*buf)[WARPS]) {
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < R; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (TPR > 32) {
    constexpr int N = TPR / 32;
    const int warp = threadIdx.x >> 5, first = warp / N * N;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int k = 0; k < R; ++k) buf[k][warp] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < R; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) v[k] += buf[k][first + i];
    }
  }
}

// The NV vectors of a row that a thread owns: columns (i * TPR + lane) * VE, zeros past the end and for rows that are not
// there.
template <typename T, int VB, int TPR, int NV>
__device__ __forceinline__ void load_row(const T* row, int lane, int C, bool live, typename Raw<VB>::type (&raw)[NV]) {
  typedef typename Raw<VB>::type R;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * TPR + lane) * (VB / (int)sizeof(T));
    raw[i] = live && col < C ? __ldg(reinterpret_cast<const R*>(row + col)) : R{};
  }
}

// Pair j of a thread's share of a row with zeros for columns past the end.
template <int VE, int TPR>
__device__ __forceinline__ f32x2 there(f32x2 v, int j, int lane, int C) {
  float lo, hi;
  unpair(v, lo, hi);
  return pair((2 * j / VE * TPR + lane) * VE < C ? lo : 0.f, ((2 * j + 1) / VE * TPR + lane) * VE < C ? hi : 0.f);
}

// The same as E / 2 pairs of float32.
template <typename T, int VB, int NV>
__device__ __forceinline__ void unpack_row(const typename Raw<VB>::type (&raw)[NV], f32x2 (&out)[NV * VB / (int)sizeof(T) / 2]) {
  constexpr int VE = VB / (int)sizeof(T);
  float f[NV * VE];
#pragma unroll
  for (int i = 0; i < NV; ++i) unpack<T, VB>(raw[i], f + i * VE);
#pragma unroll
  for (int j = 0; j < NV * VE / 2; ++j) out[j] = pair(f[2 * j], f[2 * j + 1]);
}
template <typename T, int VB, int TPR, int NV>
__device__ __forceinline__ void store_row(T* row, int lane, int C, const f32x2 (&v)[NV * VB / (int)sizeof(T) / 2]) {
  constexpr int VE = VB / (int)sizeof(T);
  float f[NV * VE];
#pragma unroll
  for (int j = 0; j < NV * VE / 2; ++j) unpair(v[j], f[2 * j], f[2 * j + 1]);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (i * TPR + lane) * VE;
    if (col < C) *reinterpret_cast<typename Raw<VB>::type*>(row + col) = pack<T, VB>(f + i * VE);
  }
}

// TPR threads per row, NV accesses of VB bytes per thread and row, R rows in flight.
template <typename T, int VB, int TPR, int NV, int R>
__global__ void __launch_bounds__(TPR > 64 ? TPR : 128)
layer_norm_fwd(const NormArgs a) {
  constexpr int VE = VB / (int)sizeof(T), E = NV * VE, BLOCK = TPR > 64 ? TPR : 128, GROUPS = BLOCK / TPR;
  __shared__ float buf[2][R][BLOCK / 32];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const bool full = ((NV - 1) * TPR + lane) * VE < a.C;      // all of the thread's columns are there
  f32x2 w[E / 2], b[E / 2];
  weight_row<T, VE, TPR, NV>(a.weight, a.w_f32, lane, a.C, 1.f, w);
  weight_row<T, VE, TPR, NV>(a.bias, a.w_f32, lane, a.C, 0.f, b);
  typename Raw<VB>::type raw[R][NV], next[R][NV];
  auto load = [&](uint32_t base) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const uint32_t r = base + k * GROUPS + group;
      load_row<T, VB, TPR, NV>(static_cast<const T*>(a.x) + (r < a.rows ? row_start(a, r) : 0), lane, a.C, r < a.rows, next[k]);
    }
  };
  const uint32_t step = gridDim.x * (GROUPS * R);
  load(blockIdx.x * (GROUPS * R));
  for (uint32_t base = blockIdx.x * (GROUPS * R); base < a.rows; base += step) {
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int i = 0; i < NV; ++i) raw[k][i] = next[k][i];
    if (base + step < a.rows) load(base + step);             // on their way while these rows are worked on
    float s[R];
    f32x2 f[R][E / 2];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      unpack_row<T, VB, NV>(raw[k], f[k]);
      f32x2 t = f[k][0];
#pragma unroll
      for (int j = 1; j < E / 2; ++j) t = add2(t, f[k][j]);
      s[k] = sum2(t);
    }
    row_sums<TPR, R, BLOCK / 32>(s, buf[0]);
    float mean[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      mean[k] = s[k] * a.inv_c;
      const f32x2 minus = pair(-mean[k], -mean[k]);
      f32x2 t = 0ull;
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        f[k][j] = add2(f[k][j], minus);
        if (!full) f[k][j] = there<VE, TPR>(f[k][j], j, lane, a.C);    // columns past the end stay out of the variance
        t = fma2(f[k][j], f[k][j], t);
      }
      s[k] = sum2(t);
    }
    row_sums<TPR, R, BLOCK / 32>(s, buf[1]);
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const uint32_t r = base + k * GROUPS + group;
      const float rstd = 1.f / sqrtf(s[k] * a.inv_c + a.eps);
      if (r < a.rows) {
        const f32x2 scale = pair(rstd, rstd);
#pragma unroll
        for (int j = 0; j < E / 2; ++j) f[k][j] = fma2(mul2(f[k][j], scale), w[j], b[j]);
        store_row<T, VB, TPR, NV>(static_cast<T*>(a.y) + (long long)r * a.C, lane, a.C, f[k]);
        if (a.mean != nullptr && lane == 0) {
          a.mean[r] = mean[k];
          a.rstd[r] = rstd;
        }
      }
    }
  }
}

// Threads of a block of the backward: several rows side by side while that fits 256.
constexpr int bwd_block(int tpr) { return tpr > 256 ? tpr : 256 / tpr * tpr; }

// dx of the rows and this block's sums of dw and db.
template <typename T, int VB, int TPR, int NV, int R>
__global__ void __launch_bounds__(bwd_block(TPR))
layer_norm_bwd(const NormArgs a) {
  constexpr int VE = VB / (int)sizeof(T), E = NV * VE, BLOCK = bwd_block(TPR), GROUPS = BLOCK / TPR, WARPS = BLOCK / 32;
  __shared__ float buf[2][2 * R][WARPS];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the joining kernel may be set up meanwhile
  f32x2 w[E / 2], dw[E / 2], db[E / 2];
  weight_row<T, VE, TPR, NV>(a.weight, a.w_f32, lane, a.C, 1.f, w);
#pragma unroll
  for (int j = 0; j < E / 2; ++j) dw[j] = db[j] = 0ull;
  typename Raw<VB>::type rx[R][NV], rg[R][NV], nx[R][NV], ng[R][NV];
  float mean[R], rstd[R], nmean[R], nrstd[R];
  auto load = [&](uint32_t base) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
      const uint32_t r = base + k * GROUPS + group;
      const bool live = r < a.rows;
      load_row<T, VB, TPR, NV>(static_cast<const T*>(a.x) + (live ? row_start(a, r) : 0), lane, a.C, live, nx[k]);
      load_row<T, VB, TPR, NV>(static_cast<const T*>(a.dy) + (live ? (long long)r * a.C : 0), lane, a.C, live, ng[k]);
      nmean[k] = live ? a.mean[r] : 0.f;
      nrstd[k] = live ? a.rstd[r] : 0.f;
    }
  };
  int flip = 0;
  const uint32_t step = gridDim.x * (GROUPS * R);
  load(blockIdx.x * (GROUPS * R));
  for (uint32_t base = blockIdx.x * (GROUPS * R); base < a.rows; base += step, flip ^= 1) {
#pragma unroll
    for (int k = 0; k < R; ++k) {
#pragma unroll
      for (int i = 0; i < NV; ++i) { rx[k][i] = nx[k][i]; rg[k][i] = ng[k][i]; }
      mean[k] = nmean[k];
      rstd[k] = nrstd[k];
    }
    if (base + step < a.rows) load(base + step);             // on their way while these rows are worked on
    float s[2 * R];
    // columns past the end hold zeros in x and dy; dy = 0 keeps them out of all four sums
#pragma unroll
    for (int k = 0; k < R; ++k) {
      f32x2 f[E / 2], g[E / 2], s0 = 0ull, s1 = 0ull;
      unpack_row<T, VB, NV>(rx[k], f);
      unpack_row<T, VB, NV>(rg[k], g);
      const f32x2 minus = pair(-mean[k], -mean[k]), scale = pair(rstd[k], rstd[k]);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        const f32x2 xh = mul2(add2(f[j], minus), scale), gw = mul2(g[j], w[j]);
        dw[j] = fma2(g[j], xh, dw[j]);
        db[j] = add2(db[j], g[j]);
        s0 = add2(s0, gw);
        s1 = fma2(gw, xh, s1);
      }
      s[2 * k] = sum2(s0);
      s[2 * k + 1] = sum2(s1);
    }
    if (a.dx != nullptr) {
      row_sums<TPR, 2 * R, WARPS>(s, buf[flip]);
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const uint32_t r = base + k * GROUPS + group;
        if (r < a.rows) {
          const float c1 = -s[2 * k] * a.inv_c, c2 = -s[2 * k + 1] * a.inv_c;
          const f32x2 minus = pair(-mean[k], -mean[k]), scale = pair(rstd[k], rstd[k]), p1 = pair(c1, c1), p2 = pair(c2, c2);
          f32x2 f[E / 2], g[E / 2];
          unpack_row<T, VB, NV>(rx[k], f);
          unpack_row<T, VB, NV>(rg[k], g);
#pragma unroll
          for (int j = 0; j < E / 2; ++j)
            f[j] = mul2(scale, fma2(mul2(add2(f[j], minus), scale), p2, fma2(g[j], w[j], p1)));
          store_row<T, VB, TPR, NV>(static_cast<T*>(a.dx) + (long long)r * a.C, lane, a.C, f);
        }
      }
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + (size_t)blockIdx.x * 2 * a.C;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        float lo, hi;
        unpair(which == 0 ? dw[j] : db[j], lo, hi);
        const int c0 = (2 * j / VE * TPR + lane) * VE + 2 * j % VE, c1 = ((2 * j + 1) / VE * TPR + lane) * VE + (2 * j + 1) % VE;
        if (c0 < a.C) part[which * a.C + c0] = lo;
        if (c1 < a.C) part[which * a.C + c1] = hi;
      }
  } else {
    // the rows side by side in a warp, then the groups of warps, in a fixed order
    constexpr int ROWS = TPR < 32 ? WARPS : GROUPS;
    __shared__ float acc[ROWS][TPR * E];
    const int at = TPR < 32 ? threadIdx.x >> 5 : group;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      float v[E];
#pragma unroll
      for (int j = 0; j < E / 2; ++j) unpair(which == 0 ? dw[j] : db[j], v[2 * j], v[2 * j + 1]);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        float t = v[j];
#pragma unroll
        for (int o = 16; o >= TPR; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (TPR >= 32 || (threadIdx.x & 31) < TPR) acc[at][((j / VE) * TPR + lane) * VE + j % VE] = t;
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.C; c += BLOCK) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < ROWS; ++i) t += acc[i][c];
        part[which * a.C + c] = t;
      }
      __syncthreads();
    }
  }
}

// Sum over a block of 512 threads.
__device__ __forceinline__ float block_sum(float v, float (*buf)[16]) {
  float one[1] = {v};
  row_sums<512, 1, 16>(one, buf);
  return one[0];
}

// Rows too wide for registers: a block walks the row once per pass; the second and third pass find it in the L2.
template <typename T>
__global__ void __launch_bounds__(512) layer_norm_fwd_wide(const NormArgs a) {
  __shared__ float buf[2][1][16];
  for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row_start(a, r);
    float s = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 512) s += to_f<T>(x[c]);
    const float mean = block_sum(s, buf[0]) * a.inv_c;
    float q = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 512) {
      const float d = to_f<T>(x[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(block_sum(q, buf[1]) * a.inv_c + a.eps);
    T* y = static_cast<T*>(a.y) + (long long)r * a.C;
    for (int c = threadIdx.x; c < a.C; c += 512) {
      float f = (to_f<T>(x[c]) - mean) * rstd, t;
      if (a.weight != nullptr) { load_weights<T, 1>(a.weight, a.w_f32, c, &t); f *= t; }
      if (a.bias != nullptr) { load_weights<T, 1>(a.bias, a.w_f32, c, &t); f += t; }
      y[c] = from_f<T>(f);
    }
    if (a.mean != nullptr && threadIdx.x == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(512) layer_norm_bwd_wide(const NormArgs a) {
  __shared__ float buf[2][2][16];
  int flip = 0;
  for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x, flip ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row_start(a, r);
    const T* dy = static_cast<const T*>(a.dy) + (long long)r * a.C;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < a.C; c += 512) {
      float gw = to_f<T>(dy[c]), t;
      if (a.weight != nullptr) { load_weights<T, 1>(a.weight, a.w_f32, c, &t); gw *= t; }
      s[0] += gw;
      s[1] = fmaf(gw, (to_f<T>(x[c]) - mean) * rstd, s[1]);
    }
    row_sums<512, 2, 16>(s, buf[flip]);
    const float c1 = s[0] * a.inv_c, c2 = s[1] * a.inv_c;
    T* dx = static_cast<T*>(a.dx) + (long long)r * a.C;
    for (int c = threadIdx.x; c < a.C; c += 512) {
      float gw = to_f<T>(dy[c]), t;
      if (a.weight != nullptr) { load_weights<T, 1>(a.weight, a.w_f32, c, &t); gw *= t; }
      dx[c] = from_f<T>(rstd * (gw - c1 - (to_f<T>(x[c]) - mean) * rstd * c2));
    }
  }
}

// Sums of dw and db over a slice of the rows (blockIdx.y) for 256 columns (blockIdx.x).
template <typename T>
__global__ void __launch_bounds__(256) layer_norm_sums_wide(const NormArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  float dw = 0.f, db = 0.f;
  for (uint32_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
    const float g = to_f<T>(static_cast<const T*>(a.dy)[(long long)r * a.C + c]);
    const float x = to_f<T>(static_cast<const T*>(a.x)[row_start(a, r) + c]);
    dw = fmaf(g, (x - a.mean[r]) * a.rstd[r], dw);
    db += g;
  }
  float* part = a.part + (size_t)blockIdx.y * 2 * a.C;
  part[c] = dw;
  part[a.C + c] = db;
}

// Adds the blocks' sums: 32 columns per block, 32 slices of the partial rows, slices joined in a fixed order.
template <typename W>
__global__ void __launch_bounds__(1024)
layer_norm_join(const float* __restrict__ part, int n, int C, W* __restrict__ dweight, W* __restrict__ dbias) {
  asm volatile("griddepcontrol.wait;" ::: "memory");      // for the end of the kernel that writes the sums
  __shared__ float s[32][33];
  const int half = blockIdx.y, c = blockIdx.x * 32 + threadIdx.x;
  W* out = half == 0 ? dweight : dbias;
  if (out == nullptr) return;
  float t = 0.f;
  if (c < C) {
#pragma unroll 8
    for (int i = threadIdx.y; i < n; i += 32) t += part[((size_t)i * 2 + half) * C + c];
  }
  s[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  if (threadIdx.y == 0 && c < C) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) t += s[i][threadIdx.x];
    out[c] = from_f<W>(t);
  }
}

constexpr int kSMs = 148;
constexpr int kMostSums = kSMs * 4;      // blocks of a backward, and so the partial sums it writes

// Widest access that the row length, the row starts and the tensors' alignment allow; 0 when elements are not aligned.
int access_bytes(const NormArgs& a, int size) {
  uintptr_t all = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.dy | (uintptr_t)a.dx | (uintptr_t)a.weight |
                  (uintptr_t)a.bias | (uintptr_t)((long long)a.C * size) | (uintptr_t)(a.outer_stride * size) |
                  (uintptr_t)(a.inner_stride * size);
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : all % size == 0 ? 2 : 0;
}

// Blocks of a kernel that an SM holds, asked once.
template <typename Kernel>
int resident(Kernel kernel, int block, std::atomic<int>& cached) {
  int n = cached.load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, block, 0) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      n = 1;
    }
    cached.store(n, std::memory_order_relaxed);
  }
  return n;
}

// Two rows in flight on top of the two that are being fetched, one where 1024 threads share a row and leave each 64
// registers: 3000 rows of 8192 (fp16) backward 56.6 us, and 319 us with two.  Below that two gain: 294912 rows of 1024
// (bf16) forward 211 us and backward 330 us, with one 223 us and 340 us; 8192 rows of 4096 57.5 us backward, 72.8 us.
template <typename T, int VB, int TPR>
void launch_fwd(const NormArgs& a, cudaStream_t s) {
  constexpr int BLOCK = TPR > 64 ? TPR : 128, NV = 8 * (int)sizeof(T) / VB, R = TPR > 512 ? 1 : 2, ROWS = BLOCK / TPR * R;
  static std::atomic<int> cached{0};
  const uint32_t blocks = (a.rows + ROWS - 1) / ROWS, most = kSMs * resident(layer_norm_fwd<T, VB, TPR, NV, R>, BLOCK, cached);
  NB_LAUNCH("layer_norm_fwd", s, layer_norm_fwd<T, VB, TPR, NV, R><<<blocks < most ? blocks : most, BLOCK, 0, s>>>(a));
}

template <typename T, int VB, int TPR>
int launch_bwd(const NormArgs& a, cudaStream_t s) {
  constexpr int BLOCK = bwd_block(TPR), NV = 8 * (int)sizeof(T) / VB, R = TPR > 512 ? 1 : 2, ROWS = BLOCK / TPR * R;
  static std::atomic<int> cached{0};
  const int fit = resident(layer_norm_bwd<T, VB, TPR, NV, R>, BLOCK, cached);
  // at most four blocks per SM, as each leaves sums of its own for dw and db, which have to be added up
  const uint32_t blocks = (a.rows + ROWS - 1) / ROWS, most = kSMs * (fit < 4 ? fit : 4);
  const int n = (int)(blocks < most ? blocks : most);
  NB_LAUNCH("layer_norm_bwd", s, layer_norm_bwd<T, VB, TPR, NV, R><<<n, BLOCK, 0, s>>>(a));
  return n;
}

// A row takes the fewest threads whose eight columns each cover it: a thread without columns costs as much as one with
// them.  With 16-byte accesses and variants for every fourth power of two only, rows of 512 took 34.5 us and 53.1 us
// instead of 20.5 us and 35.2 us (50000 rows, bf16, forward and backward), rows of 32 17.7 us and 27.7 us instead of
// 10.3 us and 18.7 us; with element accesses rows of 333 took 39.3 us and 54.5 us instead of 20.9 us and 30.8 us (40000
// rows, bf16).  Beyond 2560 columns a step of two has to do.
template <typename T, int VB, typename Launch>
int by_width(const NormArgs& a, Launch&& launch) {
#define NB_WIDTH(limit, threads) if (a.C <= limit) return launch(std::integral_constant<int, threads>())
  if constexpr (VB == 16) {
    NB_WIDTH(32, 4);
    NB_WIDTH(64, 8);
    NB_WIDTH(128, 16);
    NB_WIDTH(256, 32);
    NB_WIDTH(512, 64);
    NB_WIDTH(768, 96);
    NB_WIDTH(1024, 128);
    NB_WIDTH(1536, 192);
    NB_WIDTH(2560, 320);
  }
  NB_WIDTH(64, 8);
  if constexpr (VB < 16) NB_WIDTH(128, 16);
  NB_WIDTH(256, 32);
  if constexpr (VB < 16) NB_WIDTH(512, 64);
  NB_WIDTH(1024, 128);
  if constexpr (VB < 16) NB_WIDTH(2048, 256);
  NB_WIDTH(4096, 512);
  NB_WIDTH(8192, 1024);
#undef NB_WIDTH
  return 0;
}

template <typename T, int VB>
int fwd_by_width(const NormArgs& a, cudaStream_t s) {
  return by_width<T, VB>(a, [&](auto tpr) {
    launch_fwd<T, VB, decltype(tpr)::value>(a, s);
    return 1;
  });
}
template <typename T, int VB>
int bwd_by_width(const NormArgs& a, cudaStream_t s) {
  return by_width<T, VB>(a, [&](auto tpr) { return launch_bwd<T, VB, decltype(tpr)::value>(a, s); });
}

// Partial rows of the widths that take the wide kernels.
constexpr int kWideSlices = 64;

template <typename T>
int fwd(const NormArgs& a, cudaStream_t s) {
  int done;
  const int vb = access_bytes(a, sizeof(T));
  if (vb == 0) return set_error(NATTEN_B200_EINVAL, "layer_norm_forward: tensor pointers must be aligned to their elements");
  if (vb == 16) done = fwd_by_width<T, 16>(a, s);
  else if (vb == 4 || sizeof(T) == 4) done = fwd_by_width<T, 4>(a, s);
  else done = fwd_by_width<T, sizeof(T) == 4 ? 4 : 2>(a, s);
  if (!done) {
    const int blocks = a.rows < kSMs * 4u ? (int)a.rows : kSMs * 4;
    NB_LAUNCH("layer_norm_fwd", s, layer_norm_fwd_wide<T><<<blocks, 512, 0, s>>>(a));
  }
  return check_launch("layer norm forward");
}

template <typename T>
int bwd(const NormArgs& a, void* dweight, void* dbias, cudaStream_t s) {
  int n;
  const int vb = access_bytes(a, sizeof(T));
  if (vb == 0) return set_error(NATTEN_B200_EINVAL, "layer_norm_backward: tensor pointers must be aligned to their elements");
  if (vb == 16) n = bwd_by_width<T, 16>(a, s);
  else if (vb == 4 || sizeof(T) == 4) n = bwd_by_width<T, 4>(a, s);
  else n = bwd_by_width<T, sizeof(T) == 4 ? 4 : 2>(a, s);
  if (n == 0) {
    if (a.dx != nullptr) {
      const int blocks = a.rows < kSMs * 4u ? (int)a.rows : kSMs * 4;
      NB_LAUNCH("layer_norm_bwd", s, layer_norm_bwd_wide<T><<<blocks, 512, 0, s>>>(a));
    }
    if (a.part != nullptr) {
      n = a.rows < (uint32_t)kWideSlices ? (int)a.rows : kWideSlices;
      NB_LAUNCH("layer_norm_sums", s, layer_norm_sums_wide<T><<<dim3((a.C + 255) / 256, n), 256, 0, s>>>(a));
    }
  }
  if (int rc = check_launch("layer norm backward")) return rc;
  if (a.part == nullptr) return NATTEN_B200_OK;
  const dim3 grid((a.C + 31) / 32, 2), block(32, 32);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = s;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  const float* part = a.part;
  if (a.w_f32) NB_LAUNCH("layer_norm_join", s, (void)cudaLaunchKernelEx(&cfg, layer_norm_join<float>, part, n, a.C, (float*)dweight, (float*)dbias));
  else NB_LAUNCH("layer_norm_join", s, (void)cudaLaunchKernelEx(&cfg, layer_norm_join<T>, part, n, a.C, (T*)dweight, (T*)dbias));
  return check_launch("layer norm sums");
}

// Whether a pointer (null included) may be read as elements of `size` bytes.
bool aligned_to(const void* p, int size) { return (uintptr_t)p % size == 0; }

int check_rows(const char* what, int32_t dtype, int32_t wdtype, const natten_b200_rows* rows, NormArgs* a) {
  if (rows == nullptr) return set_error(NATTEN_B200_EINVAL, "%s: rows is null", what);
  if (dtype < NATTEN_B200_F32 || dtype > NATTEN_B200_BF16) return set_error(NATTEN_B200_EINVAL, "%s: unsupported dtype %d", what, dtype);
  if (wdtype != dtype && wdtype != NATTEN_B200_F32)
    return set_error(NATTEN_B200_EINVAL, "%s: weights must have the tensor's dtype or be float32", what);
  if (rows->channels < 1) return set_error(NATTEN_B200_EINVAL, "%s: channels must be positive", what);
  if (rows->rows < 0 || rows->rows > 0x7fffffffLL) return set_error(NATTEN_B200_EINVAL, "%s: rows must be in [0, 2^31)", what);
  if (rows->reserved != 0) return set_error(NATTEN_B200_EINVAL, "%s: reserved must be zero", what);
  if (rows->inner < 1 || rows->inner > 0x7fffffffLL) return set_error(NATTEN_B200_EINVAL, "%s: inner must be in [1, 2^31)", what);
  a->rows = (uint32_t)rows->rows;
  a->C = rows->channels;
  a->inner = (uint32_t)rows->inner;
  a->outer_stride = rows->outer_stride;
  a->inner_stride = rows->inner_stride;
  a->inv_c = 1.f / (float)rows->channels;
  a->w_f32 = wdtype == NATTEN_B200_F32;
  return NATTEN_B200_OK;
}

}  // namespace
}  // namespace nb

using namespace nb;

extern "C" {

int natten_b200_layer_norm_forward(int32_t dtype, int32_t weight_dtype, const natten_b200_rows* rows, const void* x,
                                   const void* weight, const void* bias, float eps, void* y, float* mean, float* rstd,
                                   void* stream) {
  NormArgs a{};
  if (int rc = check_rows("layer_norm_forward", dtype, weight_dtype, rows, &a)) return rc;
  if (!(eps >= 0.f)) return set_error(NATTEN_B200_EINVAL, "layer_norm_forward: eps must not be negative");
  if (a.rows == 0) return NATTEN_B200_OK;
  if (x == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr))
    return set_error(NATTEN_B200_EINVAL, "layer_norm_forward: null tensor");
  const int ws = a.w_f32 ? 4 : 2;
  if (!aligned_to(weight, ws) || !aligned_to(bias, ws) || !aligned_to(mean, 4) || !aligned_to(rstd, 4))
    return set_error(NATTEN_B200_EINVAL, "layer_norm_forward: weights and statistics must be aligned to their elements");
  a.x = x; a.weight = weight; a.bias = bias; a.eps = eps; a.y = y; a.mean = mean; a.rstd = rstd;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == NATTEN_B200_F32) return fwd<float>(a, s);
  return dtype == NATTEN_B200_F16 ? fwd<__half>(a, s) : fwd<__nv_bfloat16>(a, s);
}

size_t natten_b200_layer_norm_backward_scratch_bytes(int64_t rows, int32_t channels) {
  if (rows < 1 || channels < 1) return 0;
  const int64_t most = kMostSums;        // and no more blocks than rows
  return (size_t)(rows < most ? rows : most) * 2 * (size_t)channels * sizeof(float);
}

int natten_b200_layer_norm_backward(int32_t dtype, int32_t weight_dtype, const natten_b200_rows* rows, const void* x,
                                    const void* weight, const float* mean, const float* rstd, const void* dy, void* dx,
                                    void* dweight, void* dbias, void* scratch, size_t scratch_bytes, void* stream) {
  NormArgs a{};
  if (int rc = check_rows("layer_norm_backward", dtype, weight_dtype, rows, &a)) return rc;
  cudaStream_t s = (cudaStream_t)stream;
  if (a.rows == 0) {
    const size_t bytes = (size_t)a.C * (a.w_f32 ? 4 : 2);
    for (void* p : {dweight, dbias})
      if (p != nullptr && cudaMemsetAsync(p, 0, bytes, s) != cudaSuccess)
        return set_error(NATTEN_B200_ELAUNCH, "layer_norm_backward: %s", cudaGetErrorString(cudaGetLastError()));
    return NATTEN_B200_OK;
  }
  if (x == nullptr || mean == nullptr || rstd == nullptr || dy == nullptr)
    return set_error(NATTEN_B200_EINVAL, "layer_norm_backward: null tensor");
  const bool sums = dweight != nullptr || dbias != nullptr;
  if (dx == nullptr && !sums) return NATTEN_B200_OK;
  const size_t need = natten_b200_layer_norm_backward_scratch_bytes(rows->rows, rows->channels);
  if (sums && (scratch == nullptr || scratch_bytes < need || ((uintptr_t)scratch & 3) != 0))
    return set_error(NATTEN_B200_ERESOURCE, "layer_norm_backward: scratch has %zu bytes, needs %zu (4-byte aligned)",
                     scratch == nullptr ? (size_t)0 : scratch_bytes, need);
  const int ws = a.w_f32 ? 4 : 2;
  if (!aligned_to(weight, ws) || !aligned_to(dweight, ws) || !aligned_to(dbias, ws) || !aligned_to(mean, 4) || !aligned_to(rstd, 4))
    return set_error(NATTEN_B200_EINVAL, "layer_norm_backward: weights and statistics must be aligned to their elements");
  a.x = x; a.weight = weight; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dy = dy; a.dx = dx; a.part = sums ? static_cast<float*>(scratch) : nullptr;
  if (dtype == NATTEN_B200_F32) return bwd<float>(a, dweight, dbias, s);
  return dtype == NATTEN_B200_F16 ? bwd<__half>(a, dweight, dbias, s) : bwd<__nv_bfloat16>(a, dweight, dbias, s);
}

}  // extern "C"
