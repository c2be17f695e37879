// Layer norm over the last axis, forward and backward.
//
//   mean = sum x / C,  rstd = 1 / sqrt(sum (x - mean)^2 / C + eps),  xh = (x - mean) rstd,  y = xh w + b
//   gw = dy w,  dx = rstd (gw - sum gw / C - xh sum(gw xh) / C),  dw = sum_rows dy xh,  db = sum_rows dy
//
// All of it is bound by memory: the forward reads x and writes y, the backward reads x and dy and writes dx.  A row
// stays in the registers of the threads that own it (one load per element, the variance is taken about the mean and
// not as a difference of squares), statistics and sums are float32, y and dx are rounded once.  The rows of dw and db
// are summed by every thread for the columns it owns over all rows its block visits; the blocks' sums go to a scratch
// buffer and a second kernel adds them in a fixed order, so that a result never depends on the order of atomics.
#include <math.h>

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

// Sum over the TPR threads of a row; every one of them gets it.  Rows wider than a warp are a whole block, `buf` has
// a slot per warp, and two alternating buffers make one barrier per sum enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* buf) {
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) buf[warp] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) v += buf[i];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float2 v, float2* buf) {
  constexpr int W = TPR < 32 ? TPR : 32;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) buf[warp] = v;
    __syncthreads();
    v = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) { v.x += buf[i].x; v.y += buf[i].y; }
  }
  return v;
}

// TPR threads per row, NV accesses of VB bytes per thread.
template <typename T, int VB, int TPR, int NV>
__global__ void __launch_bounds__(TPR > 128 ? TPR : 128)
layer_norm_fwd(const NormArgs a) {
  constexpr int VE = VB / (int)sizeof(T), RPB = TPR > 128 ? 1 : 128 / TPR;
  typedef typename Raw<VB>::type R;
  __shared__ float buf[2][TPR / 32 + 1];
  const int lane = threadIdx.x % TPR;
  const uint32_t groups = (a.rows + RPB - 1) / RPB;
  for (uint32_t gr = blockIdx.x; gr < groups; gr += gridDim.x) {
    const uint32_t r = gr * RPB + threadIdx.x / TPR;
    const bool live = r < a.rows;
    const T* x = static_cast<const T*>(a.x) + (live ? row_start(a, r) : 0);
    R raw[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + lane) * VE;
      if (live && col < a.C) raw[i] = __ldg(reinterpret_cast<const R*>(x + col));
      else raw[i] = R{};
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[VE];
      unpack<T, VB>(raw[i], f);
#pragma unroll
      for (int j = 0; j < VE; ++j) s += f[j];
    }
    const float mean = row_sum<TPR>(s, buf[0]) * a.inv_c;
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if ((i * TPR + lane) * VE < a.C) {
        float f[VE];
        unpack<T, VB>(raw[i], f);
#pragma unroll
        for (int j = 0; j < VE; ++j) q = fmaf(f[j] - mean, f[j] - mean, q);
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(q, buf[1]) * a.inv_c + a.eps);
    if (live) {
      T* y = static_cast<T*>(a.y) + (long long)r * a.C;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * TPR + lane) * VE;
        if (col < a.C) {
          float f[VE], w[VE], b[VE];
          unpack<T, VB>(raw[i], f);
          if (a.weight != nullptr) load_weights<T, VE>(a.weight, a.w_f32, col, w);
          if (a.bias != nullptr) load_weights<T, VE>(a.bias, a.w_f32, col, b);
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            f[j] = (f[j] - mean) * rstd;
            if (a.weight != nullptr) f[j] *= w[j];
            if (a.bias != nullptr) f[j] += b[j];
          }
          *reinterpret_cast<R*>(y + col) = pack<T, VB>(f);
        }
      }
      if (a.mean != nullptr && lane == 0) {
        a.mean[r] = mean;
        a.rstd[r] = rstd;
      }
    }
  }
}

// dx of the rows and this block's sums of dw and db.  Rows wider than a warp are a whole block; otherwise a block of
// 256 threads holds 256 / TPR rows at a time.
template <typename T, int VB, int TPR, int NV>
__global__ void __launch_bounds__(TPR > 256 ? TPR : (TPR > 32 ? TPR : 256))
layer_norm_bwd(const NormArgs a) {
  constexpr int VE = VB / (int)sizeof(T), BLOCK = TPR > 32 ? TPR : 256, RPB = BLOCK / TPR, E = NV * VE;
  typedef typename Raw<VB>::type R;
  __shared__ float2 buf[2][TPR / 32 + 1];
  const int lane = threadIdx.x % TPR;
  const uint32_t groups = (a.rows + RPB - 1) / RPB;
  float dw[E], db[E];
#pragma unroll
  for (int j = 0; j < E; ++j) dw[j] = db[j] = 0.f;
  int flip = 0;
  for (uint32_t gr = blockIdx.x; gr < groups; gr += gridDim.x, flip ^= 1) {
    const uint32_t r = gr * RPB + threadIdx.x / TPR;
    const bool live = r < a.rows;
    const T* x = static_cast<const T*>(a.x) + (live ? row_start(a, r) : 0);
    const T* dy = static_cast<const T*>(a.dy) + (live ? (long long)r * a.C : 0);
    R rx[NV], rg[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + lane) * VE;
      if (live && col < a.C) {
        rx[i] = __ldg(reinterpret_cast<const R*>(x + col));
        rg[i] = __ldg(reinterpret_cast<const R*>(dy + col));
      } else {
        rx[i] = R{};
        rg[i] = R{};
      }
    }
    const float mean = live ? a.mean[r] : 0.f, rstd = live ? a.rstd[r] : 0.f;
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + lane) * VE;
      if (live && col < a.C) {
        float f[VE], g[VE], w[VE];
        unpack<T, VB>(rx[i], f);
        unpack<T, VB>(rg[i], g);
        if (a.weight != nullptr) load_weights<T, VE>(a.weight, a.w_f32, col, w);
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float xh = (f[j] - mean) * rstd;
          dw[i * VE + j] = fmaf(g[j], xh, dw[i * VE + j]);
          db[i * VE + j] += g[j];
          const float gw = a.weight != nullptr ? g[j] * w[j] : g[j];
          s.x += gw;
          s.y = fmaf(gw, xh, s.y);
        }
      }
    }
    if (a.dx != nullptr) {
      s = row_sum2<TPR>(s, buf[flip]);
      s.x *= a.inv_c;
      s.y *= a.inv_c;
      T* dx = static_cast<T*>(a.dx) + (long long)r * a.C;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int col = (i * TPR + lane) * VE;
        if (live && col < a.C) {
          float f[VE], g[VE], w[VE];
          unpack<T, VB>(rx[i], f);
          unpack<T, VB>(rg[i], g);
          if (a.weight != nullptr) load_weights<T, VE>(a.weight, a.w_f32, col, w);
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            const float xh = (f[j] - mean) * rstd;
            const float gw = a.weight != nullptr ? g[j] * w[j] : g[j];
            f[j] = rstd * (gw - s.x - xh * s.y);
          }
          *reinterpret_cast<R*>(dx + col) = pack<T, VB>(f);
        }
      }
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + (size_t)blockIdx.x * 2 * a.C;
  if constexpr (TPR > 32) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int col = (i * TPR + lane) * VE;
      if (col < a.C) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          part[col + j] = dw[i * VE + j];
          part[a.C + col + j] = db[i * VE + j];
        }
      }
    }
  } else {
    // the rows side by side in a warp, then the block's warps, in a fixed order
    constexpr int WARPS = BLOCK / 32;
    __shared__ float acc[WARPS][TPR * E];
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float* v = half == 0 ? dw : db;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        float t = v[j];
#pragma unroll
        for (int o = 16; o >= TPR; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if ((threadIdx.x & 31) < TPR) acc[warp][((j / VE) * TPR + lane) * VE + j % VE] = t;
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.C; c += BLOCK) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) t += acc[i][c];
        part[half * a.C + c] = t;
      }
      __syncthreads();
    }
  }
}

// Rows too wide for registers: a block walks the row once per pass; the second and third pass find it in the L2.
template <typename T>
__global__ void __launch_bounds__(512) layer_norm_fwd_wide(const NormArgs a) {
  __shared__ float buf[2][512 / 32 + 1];
  for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row_start(a, r);
    float s = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 512) s += to_f<T>(x[c]);
    const float mean = row_sum<512>(s, buf[0]) * a.inv_c;
    float q = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 512) {
      const float d = to_f<T>(x[c]) - mean;
      q = fmaf(d, d, q);
    }
    const float rstd = 1.f / sqrtf(row_sum<512>(q, buf[1]) * a.inv_c + a.eps);
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
  __shared__ float2 buf[2][512 / 32 + 1];
  int flip = 0;
  for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x, flip ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row_start(a, r);
    const T* dy = static_cast<const T*>(a.dy) + (long long)r * a.C;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float2 s = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < a.C; c += 512) {
      float gw = to_f<T>(dy[c]), t;
      if (a.weight != nullptr) { load_weights<T, 1>(a.weight, a.w_f32, c, &t); gw *= t; }
      s.x += gw;
      s.y = fmaf(gw, (to_f<T>(x[c]) - mean) * rstd, s.y);
    }
    s = row_sum2<512>(s, buf[flip]);
    s.x *= a.inv_c;
    s.y *= a.inv_c;
    T* dx = static_cast<T*>(a.dx) + (long long)r * a.C;
    for (int c = threadIdx.x; c < a.C; c += 512) {
      float gw = to_f<T>(dy[c]), t;
      if (a.weight != nullptr) { load_weights<T, 1>(a.weight, a.w_f32, c, &t); gw *= t; }
      dx[c] = from_f<T>(rstd * (gw - s.x - (to_f<T>(x[c]) - mean) * rstd * s.y));
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

// Blocks of the backward, and so the partial sums it writes.
int bwd_blocks(uint32_t rows, int rows_per_block, int per_sm) {
  const uint32_t groups = (rows + rows_per_block - 1) / rows_per_block;
  const uint32_t most = kSMs * per_sm;
  return (int)(groups < most ? groups : most);
}

// Widest access that the row length, the row starts and the tensors' alignment allow.
int access_bytes(const NormArgs& a, int size) {
  uintptr_t all = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.dy | (uintptr_t)a.dx | (uintptr_t)a.weight |
                  (uintptr_t)a.bias | (uintptr_t)((long long)a.C * size) | (uintptr_t)(a.outer_stride * size) |
                  (uintptr_t)(a.inner_stride * size);
  return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : all % size == 0 ? 2 : 0;
}

template <typename T, int VB, int TPR, int E>
void launch_fwd(const NormArgs& a, cudaStream_t s) {
  constexpr int BLOCK = TPR > 128 ? TPR : 128, NV = E * (int)sizeof(T) / VB;
  const uint32_t groups = (a.rows + BLOCK / TPR - 1) / (BLOCK / TPR);
  const uint32_t most = kSMs * (2048 / BLOCK);
  NB_LAUNCH("layer_norm_fwd", s, layer_norm_fwd<T, VB, TPR, NV><<<groups < most ? groups : most, BLOCK, 0, s>>>(a));
}

template <typename T, int VB>
bool fwd_by_width(const NormArgs& a, cudaStream_t s) {
  if (a.C <= 32) launch_fwd<T, VB, 4, 8>(a, s);
  else if (a.C <= 64) launch_fwd<T, VB, 8, 8>(a, s);
  else if (a.C <= 128) launch_fwd<T, VB, 16, 8>(a, s);
  else if (a.C <= 256) launch_fwd<T, VB, 32, 8>(a, s);
  else if (a.C <= 512) launch_fwd<T, VB, 32, 16>(a, s);
  else if (a.C <= 1024) launch_fwd<T, VB, 32, 32>(a, s);
  else if (a.C <= 4096) launch_fwd<T, VB, 128, 32>(a, s);
  else if (a.C <= 16384) launch_fwd<T, VB, 512, 32>(a, s);
  else return false;
  return true;
}

template <typename T, int VB, int TPR, int E>
int launch_bwd(const NormArgs& a, cudaStream_t s) {
  constexpr int BLOCK = TPR > 32 ? TPR : 256, NV = E * (int)sizeof(T) / VB;
  const int blocks = bwd_blocks(a.rows, BLOCK / TPR, 1024 / BLOCK);
  NB_LAUNCH("layer_norm_bwd", s, layer_norm_bwd<T, VB, TPR, NV><<<blocks, BLOCK, 0, s>>>(a));
  return blocks;
}

template <typename T, int VB>
int bwd_by_width(const NormArgs& a, cudaStream_t s) {
  if (a.C <= 32) return launch_bwd<T, VB, 4, 8>(a, s);
  if (a.C <= 64) return launch_bwd<T, VB, 8, 8>(a, s);
  if (a.C <= 128) return launch_bwd<T, VB, 16, 8>(a, s);
  if (a.C <= 256) return launch_bwd<T, VB, 32, 8>(a, s);
  if (a.C <= 512) return launch_bwd<T, VB, 32, 16>(a, s);
  if (a.C <= 1024) return launch_bwd<T, VB, 128, 8>(a, s);
  if (a.C <= 2048) return launch_bwd<T, VB, 128, 16>(a, s);
  if (a.C <= 8192) return launch_bwd<T, VB, 512, 16>(a, s);
  return 0;
}

// Partial rows of the widths that take the wide kernels.
constexpr int kWideSlices = 64;

template <typename T>
int fwd(const NormArgs& a, cudaStream_t s) {
  bool done;
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
  if (a.w_f32) NB_LAUNCH("layer_norm_join", s, layer_norm_join<float><<<grid, block, 0, s>>>(a.part, n, a.C, (float*)dweight, (float*)dbias));
  else NB_LAUNCH("layer_norm_join", s, layer_norm_join<T><<<grid, block, 0, s>>>(a.part, n, a.C, (T*)dweight, (T*)dbias));
  return check_launch("layer norm sums");
}

int check_rows(const char* what, int32_t dtype, int32_t wdtype, const natten_b200_rows* rows, NormArgs* a) {
  if (rows == nullptr) return set_error(NATTEN_B200_EINVAL, "%s: rows is null", what);
  if (dtype < NATTEN_B200_F32 || dtype > NATTEN_B200_BF16) return set_error(NATTEN_B200_EINVAL, "%s: unsupported dtype %d", what, dtype);
  if (wdtype != dtype && wdtype != NATTEN_B200_F32)
    return set_error(NATTEN_B200_EINVAL, "%s: weights must have the tensor's dtype or be float32", what);
  if (rows->channels < 1) return set_error(NATTEN_B200_EINVAL, "%s: channels must be positive", what);
  if (rows->rows < 0 || rows->rows > 0x7fffffffLL) return set_error(NATTEN_B200_EINVAL, "%s: rows must be in [0, 2^31)", what);
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
  a.x = x; a.weight = weight; a.bias = bias; a.eps = eps; a.y = y; a.mean = mean; a.rstd = rstd;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == NATTEN_B200_F32) return fwd<float>(a, s);
  return dtype == NATTEN_B200_F16 ? fwd<__half>(a, s) : fwd<__nv_bfloat16>(a, s);
}

size_t natten_b200_layer_norm_backward_scratch_bytes(int64_t rows, int32_t channels) {
  if (rows < 1 || channels < 1) return 0;
  // no more blocks than rows, and no more than a launch of the narrowest blocks has
  const int64_t most = kSMs * 8;
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
  a.x = x; a.weight = weight; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
  a.dy = dy; a.dx = dx; a.part = sums ? static_cast<float*>(scratch) : nullptr;
  if (dtype == NATTEN_B200_F32) return bwd<float>(a, dweight, dbias, s);
  return dtype == NATTEN_B200_F16 ? bwd<__half>(a, dweight, dbias, s) : bwd<__nv_bfloat16>(a, dweight, dbias, s);
}

}  // extern "C"
