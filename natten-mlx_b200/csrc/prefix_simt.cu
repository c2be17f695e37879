// Attention to a shared prefix on the CUDA cores (float32, and the head sizes that the tensor-core kernel does not
// take), the kernel that joins the parts of a split prefix, and the entry point of both families.
//
//   out = softmax(scale q k^T) v,  lse = log sum exp(scale q k^T)
//
// One pass over the keys with a running maximum and sum per row.  A block holds BM rows of one key/value head and walks
// its part of the prefix in tiles of BN keys: S = q k^T by register tiles of up to 4x8 out of shared memory, the
// probabilities through shared memory, O += P v in registers.  With many rows the float32 units bound it, with few the
// reading of k and v, which then is spread over all SMs by splitting the prefix.
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "prefix.cuh"

namespace nb {
namespace {

constexpr int kSMs = 148;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 2^x within two units of the last place.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Floats of a row in shared memory: an odd number of 16 bytes, so that 8 rows at one column are in different banks.
__host__ __device__ constexpr int row_floats(int D) { return (((D + 3) >> 2) | 1) << 2; }

// Four elements of a row from column c as float32; zeros past D and for rows that do not exist.
template <typename T>
__device__ __forceinline__ float4 load4(const T* row, int c, int D, bool vec, bool live) {
  float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
  if (!live) return r;
  if (vec && c + 4 <= D) {
    if constexpr (sizeof(T) == 4) {
      r = *reinterpret_cast<const float4*>(row + c);
    } else {
      const uint2 raw = *reinterpret_cast<const uint2*>(row + c);
      const T* e = reinterpret_cast<const T*>(&raw);
      r = make_float4(to_f<T>(e[0]), to_f<T>(e[1]), to_f<T>(e[2]), to_f<T>(e[3]));
    }
  } else {
    if (c < D) r.x = to_f<T>(row[c]);
    if (c + 1 < D) r.y = to_f<T>(row[c + 1]);
    if (c + 2 < D) r.z = to_f<T>(row[c + 2]);
    if (c + 3 < D) r.w = to_f<T>(row[c + 3]);
  }
  return r;
}

// A warp holds 4 RM rows and all BN keys of a tile, 8 threads to a row: RM x BN / 8 scores per thread, and RM rows of
// four columns out of each 32 (NH of them).  With 8 threads to a row two quarters of a warp ask for the same 128 bytes
// of keys or values, which costs half the passes through shared memory of 16 threads to a row, and the reads of shared
// memory bound this kernel next to the float32 units.  Measured, 2048 rows of 8 heads of 64 over 4096 keys, float32:
// 537 us, 32 TFLOP/s; 16 threads to a row and 64 rows to a block 659 us.  For head dims to 64 two blocks share an SM
// (128 registers): 585 us against 607 us for one block that fetches the next tile under the present one.
template <typename T, int W, int RM, int BN, int NH>
__global__ void __launch_bounds__(W * 32, (W == 8 && NH <= 2 ? 2 : 1)) prefix_simt(const PrefixArgs a, bool vec) {
  constexpr int BM = W * RM * 4, CN = BN / 8, LP = BN + 8, kThreads = W * 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // the joining kernel may be set up meanwhile
  extern __shared__ float smem[];
  const int Dp = (a.D + 3) & ~3, LD = row_floats(a.D);
  float* qs = smem;                    // [BM][LD]
  float* ks = qs + BM * LD;            // [BN][LD]
  float* vs = ks + BN * LD;            // [BN][Dp]
  float* ps = vs + BN * Dp;            // [BM][LP]
  const int tx = threadIdx.x & 7, ty = (threadIdx.x >> 5) * (RM * 4) + (threadIdx.x >> 3 & 3);
  const int hk = blockIdx.y;
  const uint32_t G = (uint32_t)a.G, rows = (uint32_t)a.tokens * G, row0 = blockIdx.x * (uint32_t)BM;     // below 2^31 + BM
  const int tiles = (a.prefix + BN - 1) / BN;
  const int t0 = (int)((long long)tiles * blockIdx.z / a.splits), t1 = (int)((long long)tiles * (blockIdx.z + 1) / a.splits);

  for (int i = threadIdx.x; i < BM * (Dp / 4); i += kThreads) {
    const int r = i / (Dp / 4), c = (i - r * (Dp / 4)) * 4;
    const uint32_t rr = row0 + r;
    const bool live = rr < rows;
    const uint32_t tok = live ? rr / G : 0, h = hk * G + (live ? rr - tok * G : 0);
    *reinterpret_cast<float4*>(qs + r * LD + c) =
        load4<T>(static_cast<const T*>(a.q) + (long long)tok * a.q_token + (long long)h * a.q_head, c, a.D, vec, live);
  }
  float m[RM], l[RM];                  // l: of this thread's keys; added up at the end
  float4 o[RM][NH];
  int lim[RM];
  int least = INT_MAX, own = 0;        // of the rows of this thread: no row sees less, none more
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
    const uint32_t rr = row0 + ty + 4 * i;
    lim[i] = rr < rows ? prefix_limit(a, rr / G) : 0;
    if (rr < rows) least = min(least, lim[i]);
    own = max(own, lim[i]);
#pragma unroll
    for (int h = 0; h < NH; ++h) o[i][h] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const float sc = a.scale * kLog2e;
  for (int t = t0; t < t1; ++t) {
    const int key0 = t * BN;
    if (!__syncthreads_or(own > key0)) break;       // also: the last tile's reads are over
    constexpr int Q4 = 8 * NH, N4 = BN * Q4 / kThreads;      // float4 of a row, and of a tile for each thread
    float4 nk[N4], nv[N4];                                   // all loads before the first store
#pragma unroll
    for (int i = 0; i < N4; ++i) {
      const int at = threadIdx.x + i * kThreads, r = at / Q4, c = at % Q4 * 4;
      const long long key = (long long)key0 + r;
      const bool live = key < a.prefix && c < a.D;
      nk[i] = load4<T>(static_cast<const T*>(a.k) + (live ? key * a.k_token : 0) + (long long)hk * a.k_head, c, a.D, vec, live);
      nv[i] = load4<T>(static_cast<const T*>(a.v) + (live ? key * a.v_token : 0) + (long long)hk * a.v_head, c, a.D, vec, live);
    }
#pragma unroll
    for (int i = 0; i < N4; ++i) {
      const int at = threadIdx.x + i * kThreads, r = at / Q4, c = at % Q4 * 4;
      if (c < Dp) {
        *reinterpret_cast<float4*>(ks + r * LD + c) = nk[i];
        *reinterpret_cast<float4*>(vs + r * Dp + c) = nv[i];
      }
    }
    __syncthreads();
    float s[RM][CN];
#pragma unroll
    for (int i = 0; i < RM; ++i)
#pragma unroll
      for (int j = 0; j < CN; ++j) s[i][j] = 0.f;
#pragma unroll 2
    for (int d = 0; d < Dp; d += 4) {
      float4 qv[RM];
#pragma unroll
      for (int i = 0; i < RM; ++i) qv[i] = *reinterpret_cast<const float4*>(qs + (ty + 4 * i) * LD + d);
#pragma unroll
      for (int j = 0; j < CN; ++j) {
        const float4 kv = *reinterpret_cast<const float4*>(ks + (tx + 8 * j) * LD + d);
#pragma unroll
        for (int i = 0; i < RM; ++i)
          s[i][j] = fmaf(qv[i].x, kv.x, fmaf(qv[i].y, kv.y, fmaf(qv[i].z, kv.z, fmaf(qv[i].w, kv.w, s[i][j]))));
      }
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < CN; ++j) {
        s[i][j] = key0 + tx + 8 * j < lim[i] ? s[i][j] * sc : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
#pragma unroll
      for (int w = 4; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn;
      const float alpha = ex2(m[i] - base);
      m[i] = mn;
      l[i] *= alpha;
#pragma unroll
      for (int j = 0; j < CN; ++j) {
        const float p = ex2(s[i][j] - base);
        l[i] += p;
        ps[(ty + 4 * i) * LP + tx + 8 * j] = p;
      }
#pragma unroll
      for (int h = 0; h < NH; ++h) { o[i][h].x *= alpha; o[i][h].y *= alpha; o[i][h].z *= alpha; o[i][h].w *= alpha; }
    }
    __syncwarp();                        // the threads of a row are in one warp
    // Values past a row's end stay out of its sum, whatever they hold: they are looked at one by one from the first
    // group of four that one of the thread's rows sees a part of.
    const int whole = a.lens == nullptr ? BN : max(0, min(BN, (least - key0) & ~3)), end = min(BN, own - key0);
#pragma unroll 1
    for (int kk = 0; kk < whole; kk += 4) {
      float4 pv[RM];
#pragma unroll
      for (int i = 0; i < RM; ++i) pv[i] = *reinterpret_cast<const float4*>(ps + (ty + 4 * i) * LP + kk);
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const int c = tx * 4 + 32 * h;
        if (c < Dp) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const float4 vv = *reinterpret_cast<const float4*>(vs + (kk + x) * Dp + c);
#pragma unroll
            for (int i = 0; i < RM; ++i) {
              const float p = x == 0 ? pv[i].x : x == 1 ? pv[i].y : x == 2 ? pv[i].z : pv[i].w;
              o[i][h].x = fmaf(p, vv.x, o[i][h].x);
              o[i][h].y = fmaf(p, vv.y, o[i][h].y);
              o[i][h].z = fmaf(p, vv.z, o[i][h].z);
              o[i][h].w = fmaf(p, vv.w, o[i][h].w);
            }
          }
        }
      }
    }
#pragma unroll 1
    for (int kk = whole; kk < end; ++kk)
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const int c = tx * 4 + 32 * h;
        if (c < Dp) {
          const float4 vv = *reinterpret_cast<const float4*>(vs + kk * Dp + c);
#pragma unroll
          for (int i = 0; i < RM; ++i)
            if (key0 + kk < lim[i]) {
              const float p = ps[(ty + 4 * i) * LP + kk];
              o[i][h].x = fmaf(p, vv.x, o[i][h].x);
              o[i][h].y = fmaf(p, vv.y, o[i][h].y);
              o[i][h].z = fmaf(p, vv.z, o[i][h].z);
              o[i][h].w = fmaf(p, vv.w, o[i][h].w);
            }
        }
      }
  }
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int w = 4; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const uint32_t rr = row0 + ty + 4 * i;
    if (rr >= rows) continue;
    const uint32_t tok = rr / G;
    const long long at = (long long)tok * a.Hq + hk * G + (rr - tok * G);
    const float inv = l[i] > 0.f ? 1.f / l[i] : (l[i] == 0.f ? 0.f : l[i]);     // a NaN sum stays one
    float lse = l[i] == 0.f ? -INFINITY : (m[i] + log2f(l[i])) * kLn2;
    float wa = 1.f, wb = 0.f;
    const bool last = a.splits == 1;
    const bool win = last && a.window_lse != nullptr;
    if (win) lse = join_weights(lse, a.window_lse[at], wa, wb);
    const T* wo = static_cast<const T*>(a.window_out) + at * a.D;
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const float f[4] = {o[i][h].x, o[i][h].y, o[i][h].z, o[i][h].w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int c = tx * 4 + 32 * h + x;
        if (c < a.D) {
          float v = f[x] * inv;
          if (win) v = (wa != 0.f ? v * wa : 0.f) + (wb != 0.f ? to_f<T>(wo[c]) * wb : 0.f);
          if (last) static_cast<T*>(a.out)[at * a.D + c] = from_f<T>(v);
          else a.part_out[((long long)blockIdx.z * a.tokens * a.Hq + at) * a.D + c] = v;
        }
      }
    }
    if (tx == 0) {
      if (!last) a.part_lse[(long long)blockIdx.z * a.tokens * a.Hq + at] = lse;
      else if (a.lse != nullptr) a.lse[at] = lse;
    }
  }
}

// Joins the parts of a row and the window's result: 4 columns per lane, and where a row leaves lanes over they take other
// parts; WARPS warps share a row's parts.  The order of the sums is fixed.  The kernel starts while the one that writes
// the parts still runs, and waits for its end.
constexpr int kMostParts = 256, kFewParts = 8;     // fewer than kFewParts: a warp per row

template <typename T, int WARPS>
__global__ void __launch_bounds__(128) prefix_join(const PrefixArgs a, int lanes) {
  __shared__ float weight[4 / WARPS][WARPS == 1 ? kFewParts : kMostParts];
  __shared__ float4 sums[WARPS][64];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, of = warp % WARPS, slot = warp / WARPS;
  const long long part = (long long)blockIdx.x * (4 / WARPS) + slot, rows = a.part_rows;
  const long long at = part < rows ? prefix_part_row(a, part) : -1;      // one row for all warps that meet below
  if (at < 0) return;
  const float lw = a.window_lse != nullptr ? a.window_lse[at] : -INFINITY;
  float m = lw;
  for (int i = lane; i < a.splits; i += 32) m = fmaxf(m, a.part_lse[i * rows + part]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float base = m == -INFINITY ? 0.f : m;
  float total = 0.f;
  for (int i = lane; i < a.splits; i += 32) {
    const float e = expf(a.part_lse[i * rows + part] - base);
    weight[slot][i] = e;                                   // the warps of a row write the same
    total += e;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const float ww = a.window_lse != nullptr ? expf(lw - base) : 0.f;
  total += ww;
  const float inv = total == 0.f ? 0.f : 1.f / total;
  __syncwarp();
  const int groups = 32 / lanes * WARPS, group = of * (32 / lanes) + lane / lanes;
  const int cols = (a.D + 3) / 4;
  const bool vec = a.D % 4 == 0;
  for (int first = 0; first < cols; first += lanes) {      // once, twice for head dims above 128
    const int c4 = first + lane % lanes;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c4 < cols) {
#pragma unroll 8
      for (int i = group; i < a.splits; i += groups) {
        const float e = weight[slot][i];                   // 0 for a part without keys, which left zeros
        const float* p = a.part_out + (i * rows + part) * a.D + c4 * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (vec) {
          v = __ldg(reinterpret_cast<const float4*>(p));
        } else {
          v.x = p[0];
          if (c4 * 4 + 1 < a.D) v.y = p[1];
          if (c4 * 4 + 2 < a.D) v.z = p[2];
          if (c4 * 4 + 3 < a.D) v.w = p[3];
        }
        s.x = fmaf(e, v.x, s.x); s.y = fmaf(e, v.y, s.y); s.z = fmaf(e, v.z, s.z); s.w = fmaf(e, v.w, s.w);
      }
    }
    for (int o = 16; o >= lanes; o >>= 1) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, o); s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
      s.z += __shfl_xor_sync(0xffffffffu, s.z, o); s.w += __shfl_xor_sync(0xffffffffu, s.w, o);
    }
    if (WARPS > 1) {
      if (lane < lanes) sums[of][c4] = s;
    } else if (lane < lanes && c4 < cols) {
      const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (c4 * 4 + x < a.D) {
          float o = v[x] * inv;
          if (ww != 0.f) o = fmaf(ww * inv, to_f<T>(static_cast<const T*>(a.window_out)[at * a.D + c4 * 4 + x]), o);
          static_cast<T*>(a.out)[at * a.D + c4 * 4 + x] = from_f<T>(o);
        }
    }
  }
  if (WARPS > 1) {
    __syncthreads();
    const float* s = reinterpret_cast<const float*>(sums);
    for (int d = threadIdx.x; d < a.D; d += 128) {
      float o = 0.f;
#pragma unroll
      for (int i = 0; i < WARPS; ++i) o += s[i * 256 + d];
      o *= inv;
      if (ww != 0.f) o = fmaf(ww * inv, to_f<T>(static_cast<const T*>(a.window_out)[at * a.D + d]), o);
      static_cast<T*>(a.out)[at * a.D + d] = from_f<T>(o);
    }
  }
  if (of == 0 && lane == 0 && a.lse != nullptr) a.lse[at] = m == -INFINITY ? m : m + logf(total);
}

bool simt_small(const PrefixArgs& a) { return a.tokens * a.G <= 16; }
int simt_bm(const PrefixArgs& a) { return simt_small(a) ? 16 : a.D <= 128 ? 128 : 64; }
int simt_bn(const PrefixArgs& a) { return a.D <= 64 ? 64 : 32; }

template <typename T, int W, int RM, int BN, int NH>
int launch(const PrefixArgs& a, cudaStream_t s) {
  constexpr int BM = W * RM * 4;
  const int Dp = (a.D + 3) & ~3, LD = row_floats(a.D);
  const size_t smem = (size_t)(BM * LD + BN * LD + BN * Dp + BM * (BN + 8)) * sizeof(float);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(prefix_simt<T, W, RM, BN, NH>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) {
      (void)cudaGetLastError();
      return set_error(NATTEN_B200_ELAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    }
  }
  const long long rows = a.tokens * a.G;
  const dim3 grid((unsigned)((rows + BM - 1) / BM), a.Hkv, a.splits);
  // four elements at a time when every row starts on such a boundary
  const uintptr_t all = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v |
                        (uintptr_t)((a.q_token | a.q_head | a.k_token | a.k_head | a.v_token | a.v_head) * (long long)sizeof(T));
  const bool vec = all % (4 * sizeof(T)) == 0;
  NB_LAUNCH("prefix_simt", s, prefix_simt<T, W, RM, BN, NH><<<grid, W * 32, smem, s>>>(a, vec));
  return check_launch("prefix attention");
}

template <typename T>
int run(const PrefixArgs& a, cudaStream_t s) {
  const bool small = simt_small(a);
  if (a.D <= 32) return small ? launch<T, 4, 1, 64, 1>(a, s) : launch<T, 8, 4, 64, 1>(a, s);
  if (a.D <= 64) return small ? launch<T, 4, 1, 64, 2>(a, s) : launch<T, 8, 4, 64, 2>(a, s);
  if (a.D <= 128) return small ? launch<T, 4, 1, 32, 4>(a, s) : launch<T, 8, 4, 32, 4>(a, s);
  return small ? launch<T, 4, 1, 32, 8>(a, s) : launch<T, 8, 2, 32, 8>(a, s);
}

template <typename T>
int join(const PrefixArgs& a, cudaStream_t s) {
  int lanes = 1;                         // of a row: a power of two
  while (lanes < 32 && lanes * 4 < a.D) lanes *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(128);
  cfg.stream = s;
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  // Four warps share a row's parts when each gets two or more: 37 parts of 512 rows x 128 11 us between events instead of
  // 21 us.  With fewer parts a warp has a row: two parts of 16384 rows x 64 16 us instead of 40 us.  (Events add 8 us.)
  if (a.splits >= kFewParts) {
    cfg.gridDim = dim3((unsigned)a.part_rows);
    NB_LAUNCH("prefix_join", s, (void)cudaLaunchKernelEx(&cfg, prefix_join<T, 4>, a, lanes));
  } else {
    cfg.gridDim = dim3((unsigned)((a.part_rows + 3) / 4));
    NB_LAUNCH("prefix_join", s, (void)cudaLaunchKernelEx(&cfg, prefix_join<T, 1>, a, lanes));
  }
  return check_launch("prefix attention, joining the parts");
}

}  // namespace

// Parts of the prefix: enough blocks for two on every SM, none shorter than two tiles (1989 rows of two heads over 256
// keys: 19.0 us; with four tiles, which is one part, 25.8 us).
int prefix_simt_splits(const PrefixArgs& a) {
  const int bm = simt_bm(a), bn = simt_bn(a);
  const long long blocks = ((a.tokens * a.G + bm - 1) / bm) * a.Hkv;
  const long long want = blocks >= kSMs * 2 ? 1 : std::min<long long>(kSMs * 2 / blocks, kMostParts), most = (a.prefix + 2 * bn - 1) / (2 * bn);
  const long long n = want < most ? want : most;
  return n < 1 ? 1 : (int)n;
}

int run_prefix_simt(const PrefixArgs& a, int dtype, cudaStream_t s) {
  if (dtype == NATTEN_B200_F32) return run<float>(a, s);
  return dtype == NATTEN_B200_F16 ? run<__half>(a, s) : run<__nv_bfloat16>(a, s);
}

namespace {

int make_args(const natten_b200_prefix_geom* g, PrefixArgs* a) {
  if (g == nullptr) return set_error(NATTEN_B200_EINVAL, "prefix: geometry is null");
  if (g->dtype < NATTEN_B200_F32 || g->dtype > NATTEN_B200_BF16) return set_error(NATTEN_B200_EINVAL, "prefix: unsupported dtype %d", g->dtype);
  if (g->heads_q < 1 || g->heads_kv < 1 || g->head_dim < 1) return set_error(NATTEN_B200_EINVAL, "prefix: heads and head_dim must be positive");
  if (g->head_dim > 256) return set_error(NATTEN_B200_EINVAL, "prefix: head_dim must be at most 256, got %d", g->head_dim);
  if (g->heads_q % g->heads_kv != 0)
    return set_error(NATTEN_B200_EINVAL, "prefix: heads_q (%d) must be divisible by heads_kv (%d)", g->heads_q, g->heads_kv);
  if (g->heads_kv > 65535) return set_error(NATTEN_B200_EINVAL, "prefix: at most 65535 key/value heads");
  if (g->batch < 0 || g->tokens < 0 || g->prefix < 0) return set_error(NATTEN_B200_EINVAL, "prefix: sizes must not be negative");
  if (g->batch > 0x7fffffffLL || g->tokens > 0x7fffffffLL || g->batch * g->tokens > 0x7fffffffLL / g->heads_q)
    return set_error(NATTEN_B200_EINVAL, "prefix: more than 2^31 rows");
  if (g->prefix > 0x7fffffffLL - 1024) return set_error(NATTEN_B200_EINVAL, "prefix: more than 2^31 tokens");
  if (!(g->scale > 0.f) || isinf(g->scale)) return set_error(NATTEN_B200_EINVAL, "prefix: scale must be positive and finite");
  a->Hq = g->heads_q; a->Hkv = g->heads_kv; a->G = g->heads_q / g->heads_kv; a->D = g->head_dim;
  a->tokens = g->batch * g->tokens;
  a->per_sample = (uint32_t)(g->tokens > 0 ? g->tokens : 1);
  a->prefix = (int)g->prefix;
  a->scale = g->scale;
  a->lens = g->lens;
  // a stride over an axis of length one is never taken: the dense one keeps the checks on strides simple
  a->q_head = a->Hq > 1 ? g->q_head_stride : a->D;
  a->q_token = a->tokens > 1 ? g->q_token_stride : (long long)a->Hq * a->D;
  a->k_head = a->Hkv > 1 ? g->k_head_stride : a->D;
  a->k_token = a->prefix > 1 ? g->k_token_stride : (long long)a->Hkv * a->D;
  a->v_head = a->Hkv > 1 ? g->v_head_stride : a->D;
  a->v_token = a->prefix > 1 ? g->v_token_stride : (long long)a->Hkv * a->D;
  a->splits = 1;
  return NATTEN_B200_OK;
}

// The family that serves the call and the parts it cuts the prefix into.
int choose(const natten_b200_prefix_geom* g, PrefixArgs* a, bool* tc) {
  const char* why = prefix_sm100_unsupported(*a, g->dtype);
  *tc = g->path != NATTEN_B200_PATH_SIMT && why == nullptr;
  if (g->path == NATTEN_B200_PATH_TCGEN05 && !*tc)
    return set_error(NATTEN_B200_EINVAL, "prefix: shape not supported by the tcgen05 kernels: %s", why);
  if (*tc) prefix_sm100_plan(a);
  else a->splits = prefix_simt_splits(*a);
  a->part_rows = a->splits <= 1 ? 0 : a->cut > 0 ? a->cut * 256 : a->tokens * a->Hq;
  return NATTEN_B200_OK;
}

size_t scratch_bytes_of(const PrefixArgs& a) {
  return a.splits <= 1 ? 0 : (size_t)a.splits * (size_t)a.part_rows * ((size_t)a.D + 1) * sizeof(float);
}

}  // namespace
}  // namespace nb

using namespace nb;

extern "C" {

size_t natten_b200_prefix_scratch_bytes(const natten_b200_prefix_geom* g) {
  PrefixArgs a{};
  bool tc;
  if (make_args(g, &a) || a.tokens == 0 || choose(g, &a, &tc)) return 0;
  return scratch_bytes_of(a);
}

int natten_b200_prefix_forward(const natten_b200_prefix_geom* g, const void* q, const void* k, const void* v,
                               const void* window_out, const float* window_lse, void* out, float* lse, void* scratch,
                               size_t scratch_bytes, void* stream) {
  PrefixArgs a{};
  if (int rc = make_args(g, &a)) return rc;
  if (a.tokens == 0) return NATTEN_B200_OK;
  if (q == nullptr || out == nullptr || (a.prefix > 0 && (k == nullptr || v == nullptr)))
    return set_error(NATTEN_B200_EINVAL, "prefix: null tensor");
  if ((window_out == nullptr) != (window_lse == nullptr))
    return set_error(NATTEN_B200_EINVAL, "prefix: window_out and window_lse must both be given or both be null");
  if (((uintptr_t)scratch & 31) != 0) return set_error(NATTEN_B200_EINVAL, "prefix: scratch must be 32-byte aligned");
  for (const void* p : {q, k, v, (const void*)window_out, (const void*)out})
    if (((uintptr_t)p & 15) != 0) return set_error(NATTEN_B200_EINVAL, "prefix: tensor pointers must be 16-byte aligned");
  if ((((uintptr_t)window_lse | (uintptr_t)lse | (uintptr_t)g->lens) & 3) != 0)
    return set_error(NATTEN_B200_EINVAL, "prefix: lens, lse and window_lse must be aligned to their elements");
  bool tc;
  if (int rc = choose(g, &a, &tc)) return rc;
  const size_t need = scratch_bytes_of(a);
  if (need > 0 && (scratch == nullptr || scratch_bytes < need))
    return set_error(NATTEN_B200_ERESOURCE, "prefix: scratch has %zu bytes, needs %zu", scratch == nullptr ? (size_t)0 : scratch_bytes, need);
  a.q = q; a.k = k; a.v = v; a.window_out = window_out; a.window_lse = window_lse; a.out = out; a.lse = lse;
  a.part_out = static_cast<float*>(scratch);
  a.part_lse = a.part_out == nullptr ? nullptr : a.part_out + (size_t)a.splits * a.part_rows * a.D;
  cudaStream_t s = (cudaStream_t)stream;
  set_last_path(tc ? "tcgen05" : "simt");
  if (int rc = tc ? run_prefix_sm100(a, g->dtype, s) : run_prefix_simt(a, g->dtype, s)) return rc;
  if (a.splits == 1) return NATTEN_B200_OK;
  if (g->dtype == NATTEN_B200_F32) return join<float>(a, s);
  return g->dtype == NATTEN_B200_F16 ? join<__half>(a, s) : join<__nv_bfloat16>(a, s);
}

}  // extern "C"
