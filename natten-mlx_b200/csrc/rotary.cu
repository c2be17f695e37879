// Rotary positions over one to three axes (sequence, image, video) for the queries and keys of one attention call.
//
// Pair p of a head belongs to an axis and turns by pos[axis] * f[p]:  (a, b) -> (a cos - b sin, a sin + b cos).  The
// pairs are neighbouring channels (interleaved) or the two halves of the rotated channels; channels past the rotated
// width pass through.  The gradient is the turn by the opposite angle, so the backward is the same kernel.
//
// Bound by memory: q and k are read once and written once.  No table of cosines is read: a block takes a run of tokens,
// computes the cosines and sines of their pairs once into shared memory, and all heads of q and k use them.  The
// angle is exact for any 32-bit position: f is held as a fraction of a turn in 64-bit fixed point, so that the integer
// product pos * f wraps around at whole turns by itself, and only the fraction that is left becomes a float.
#include <math.h>

#include "launch.cuh"

namespace nb {
namespace {

constexpr int kMaxPairs = 256;
constexpr int kTable = 1024;     // (token, pair) entries of a block's table: 8 KB
constexpr int kThreads = 256;
constexpr int kSMs = 148;

// Division of n < 2^31 by an invariant d >= 1 (Granlund and Montgomery, 1994): n * m >> (31 + s) with
// m = ceil(2^(31 + s) / d), 2^s >= d.
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div), s(0) {
    while ((1ull << s) < div) ++s;
    m = (uint32_t)(((1ull << (31 + s)) + div - 1) / div);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * m) >> (31 + s)); }
};

struct RotaryArgs {
  const void *q, *k;
  void *yq, *yk;
  long long q_token, q_head, k_token, k_head;   // strides in elements
  const void* positions;
  long long origin[3];
  uint32_t tokens, per_sample;
  int heads_q, heads_k, D, rank, axes;
  int kind, pos64, pos_batch, inverse;
  int pairs, axis_end[3];                       // pairs of axis a end at axis_end[a]
  int tile;                                     // tokens of a block's run
  FastDiv by_sample, by_ext[3], by_pairs, by_token, by_head;
  uint32_t units_token, units_head;             // work units of a token and of a head
  uint64_t phase[kMaxPairs];
};

enum { POS_GRID = 0, POS_OFFSET = 1, POS_GIVEN = 2 };
enum { MODE_PAIRS = 0, MODE_VEC_INTERLEAVED = 1, MODE_VEC_HALVES = 2, MODE_PAIRS_HALVES = 3 };

__device__ __forceinline__ long long position(const RotaryArgs& a, uint32_t token, int axis) {
  const uint32_t b = a.by_sample.div(token);
  const uint32_t n = token - b * a.per_sample;
  if (a.kind == POS_GIVEN) {
    const long long at = (long long)(a.pos_batch ? token : n) * a.axes + axis;
    return a.pos64 ? static_cast<const long long*>(a.positions)[at] : (long long)static_cast<const int*>(a.positions)[at];
  }
  // row-major coordinates: the last axis runs fastest
  uint32_t rest = n, idx = 0;
  for (int i = a.rank - 1; i >= axis; --i) {
    const uint32_t up = a.by_ext[i].div(rest);
    idx = rest - up * a.by_ext[i].d;
    rest = up;
  }
  long long p = a.origin[axis] + idx;
  if (a.kind == POS_OFFSET) {
    const long long at = (long long)b * a.rank + axis;
    p += a.pos64 ? static_cast<const long long*>(a.positions)[at] : (long long)static_cast<const int*>(a.positions)[at];
  }
  return p;
}

template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int VE = 16 / (int)sizeof(T);
  constexpr bool HALVES = MODE == MODE_PAIRS_HALVES;
  __shared__ uint64_t phase[kMaxPairs];
  __shared__ float2 table[kTable];
  for (int i = threadIdx.x; i < a.pairs; i += kThreads) phase[i] = a.phase[i];
  __syncthreads();
  const int half = a.pairs;                    // rotated channels: 2 * pairs
  const uint32_t runs = (a.tokens + a.tile - 1) / a.tile;
  for (uint32_t run = blockIdx.x; run < runs; run += gridDim.x) {
    const uint32_t first = run * a.tile;
    const uint32_t n = min((uint32_t)a.tile, a.tokens - first);
    for (uint32_t e = threadIdx.x; e < n * a.pairs; e += kThreads) {
      const uint32_t t = a.by_pairs.div(e);
      const int p = (int)(e - t * a.pairs);
      const int axis = p < a.axis_end[0] ? 0 : p < a.axis_end[1] ? 1 : 2;
      // the top half of the fraction, read as signed: half turns in [-1, 1) after scaling
      const int frac = (int)(((uint64_t)position(a, first + t, axis) * phase[p]) >> 32);
      float sn, cs;
      sincospif((float)frac * 4.656612873077393e-10f, &sn, &cs);
      table[e] = make_float2(cs, a.inverse ? -sn : sn);
    }
    __syncthreads();
    for (uint32_t u = threadIdx.x; u < n * a.units_token; u += kThreads) {
      const uint32_t t = a.by_token.div(u), in_token = u - t * a.units_token;
      const uint32_t hh = a.by_head.div(in_token);
      const int v = (int)(in_token - hh * a.units_head);
      const bool is_q = hh < (uint32_t)a.heads_q;
      const int h = is_q ? hh : hh - a.heads_q;
      const uint32_t token = first + t;
      const T* src = is_q ? static_cast<const T*>(a.q) + (long long)token * a.q_token + (long long)h * a.q_head
                          : static_cast<const T*>(a.k) + (long long)token * a.k_token + (long long)h * a.k_head;
      T* dst = is_q ? static_cast<T*>(a.yq) + ((long long)token * a.heads_q + h) * a.D
                    : static_cast<T*>(a.yk) + ((long long)token * a.heads_k + h) * a.D;
      const float2* cs = table + t * a.pairs;
      if constexpr (MODE == MODE_VEC_INTERLEAVED) {
        float f[VE];
        load16<T>(src + v * VE, f);
#pragma unroll
        for (int j = 0; j < VE / 2; ++j) {
          const int p = v * (VE / 2) + j;
          if (p < a.pairs) {
            const float2 c = cs[p];
            const float x = f[2 * j], y = f[2 * j + 1];
            f[2 * j] = x * c.x - y * c.y;
            f[2 * j + 1] = x * c.y + y * c.x;
          }
        }
        store16<T>(dst + v * VE, f);
      } else if constexpr (MODE == MODE_VEC_HALVES) {
        const int rot = half / VE;
        float f[VE], g[VE];
        if (v < rot) {
          load16<T>(src + v * VE, f);
          load16<T>(src + half + v * VE, g);
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            const float2 c = cs[v * VE + j];
            const float x = f[j], y = g[j];
            f[j] = x * c.x - y * c.y;
            g[j] = x * c.y + y * c.x;
          }
          store16<T>(dst + v * VE, f);
          store16<T>(dst + half + v * VE, g);
        } else {
          const int c = 2 * half + (v - rot) * VE;
          *reinterpret_cast<uint4*>(dst + c) = *reinterpret_cast<const uint4*>(src + c);
        }
      } else {
        if (v < half) {
          const int i0 = HALVES ? v : 2 * v, i1 = HALVES ? v + half : 2 * v + 1;
          const float2 c = cs[v];
          const float x = to_f<T>(src[i0]), y = to_f<T>(src[i1]);
          dst[i0] = from_f<T>(x * c.x - y * c.y);
          dst[i1] = from_f<T>(x * c.y + y * c.x);
        } else {
          dst[v + half] = src[v + half];
        }
      }
    }
    __syncthreads();
  }
}

template <typename T>
int launch(RotaryArgs& a, int mode, int units_head, cudaStream_t s) {
  a.units_head = units_head;
  a.units_token = units_head * (a.heads_q + a.heads_k);
  a.by_head = FastDiv(a.units_head);
  a.by_token = FastDiv(a.units_token);
  a.by_pairs = FastDiv(a.pairs);
  // as many tokens as the table holds, but no fewer than four runs for each SM while there are so many tokens
  const uint32_t spread = (a.tokens + kSMs * 4 - 1) / (kSMs * 4);
  a.tile = (int)(spread < (uint32_t)(kTable / a.pairs) ? spread : (uint32_t)(kTable / a.pairs));
  const uint32_t runs = (a.tokens + a.tile - 1) / a.tile, most = kSMs * 8;
  const int grid = (int)(runs < most ? runs : most);
  switch (mode) {
    case MODE_VEC_INTERLEAVED: NB_LAUNCH("rotary", s, rotary_kernel<T, MODE_VEC_INTERLEAVED><<<grid, kThreads, 0, s>>>(a)); break;
    case MODE_VEC_HALVES: NB_LAUNCH("rotary", s, rotary_kernel<T, MODE_VEC_HALVES><<<grid, kThreads, 0, s>>>(a)); break;
    case MODE_PAIRS_HALVES: NB_LAUNCH("rotary", s, rotary_kernel<T, MODE_PAIRS_HALVES><<<grid, kThreads, 0, s>>>(a)); break;
    default: NB_LAUNCH("rotary", s, rotary_kernel<T, MODE_PAIRS><<<grid, kThreads, 0, s>>>(a)); break;
  }
  return check_launch("rotary");
}

}  // namespace
}  // namespace nb

using namespace nb;

extern "C" int natten_b200_rotary(const natten_b200_rotary_geom* g, const void* q, const void* k, void* yq, void* yk,
                                  int32_t inverse, void* stream) {
  if (g == nullptr) return set_error(NATTEN_B200_EINVAL, "rotary: geometry is null");
  if (g->dtype < NATTEN_B200_F32 || g->dtype > NATTEN_B200_BF16) return set_error(NATTEN_B200_EINVAL, "rotary: unsupported dtype %d", g->dtype);
  if (g->rank < 1 || g->rank > 3) return set_error(NATTEN_B200_EINVAL, "rotary: rank must be 1, 2 or 3, got %d", g->rank);
  if (g->n_axes < 1 || g->n_axes > 3) return set_error(NATTEN_B200_EINVAL, "rotary: there must be 1, 2 or 3 axes, got %d", g->n_axes);
  if (g->position_kind < POS_GRID || g->position_kind > POS_GIVEN) return set_error(NATTEN_B200_EINVAL, "rotary: unknown position kind %d", g->position_kind);
  if (g->position_kind != POS_GIVEN && g->n_axes != g->rank)
    return set_error(NATTEN_B200_EINVAL, "rotary: positions from the grid need one axis per spatial dimension, got %d for rank %d", g->n_axes, g->rank);
  if (g->position_kind != POS_GRID && g->positions == nullptr) return set_error(NATTEN_B200_EINVAL, "rotary: positions is null");
  if (g->position_bits != 32 && g->position_bits != 64) return set_error(NATTEN_B200_EINVAL, "rotary: positions must have 32 or 64 bits");
  if (g->heads_q < 1 || g->heads_k < 1 || g->head_dim < 1) return set_error(NATTEN_B200_EINVAL, "rotary: heads and head_dim must be positive");
  if (g->heads_q > 65536 || g->heads_k > 65536 || g->head_dim > 65536) return set_error(NATTEN_B200_EINVAL, "rotary: heads or head_dim too large");
  if (g->phases == nullptr) return set_error(NATTEN_B200_EINVAL, "rotary: phases is null");
  RotaryArgs a{};
  long long n = 1;
  for (int i = 0; i < g->rank; ++i) {
    if (g->extent[i] < 0) return set_error(NATTEN_B200_EINVAL, "rotary: extents must not be negative");
    n *= g->extent[i];
    if (n > 0x7fffffffLL) break;
  }
  if (g->batch < 0 || n > 0x7fffffffLL || (long long)g->batch * n > 0x7fffffffLL)
    return set_error(NATTEN_B200_EINVAL, "rotary: more than 2^31 tokens");
  a.axes = g->n_axes;
  for (int i = 0; i < 3; ++i) {
    if (i < g->n_axes) {
      if (g->axis_dims[i] < 0 || g->axis_dims[i] % 2 != 0) return set_error(NATTEN_B200_EINVAL, "rotary: axis_dims must be even and not negative");
      if (g->axis_dims[i] > 2 * kMaxPairs) return set_error(NATTEN_B200_EINVAL, "rotary: at most %d rotated channels", 2 * kMaxPairs);
      a.pairs += g->axis_dims[i] / 2;
    }
    a.axis_end[i] = a.pairs;
    a.origin[i] = g->origin[i];
  }
  if (a.pairs < 1 || a.pairs > kMaxPairs) return set_error(NATTEN_B200_EINVAL, "rotary: the rotated channels must be in [2, %d]", 2 * kMaxPairs);
  if (2 * a.pairs > g->head_dim) return set_error(NATTEN_B200_EINVAL, "rotary: axis_dims sum to %d, head_dim is %d", 2 * a.pairs, g->head_dim);
  if (g->batch * n == 0) return NATTEN_B200_OK;
  if (q == nullptr || k == nullptr || yq == nullptr || yk == nullptr) return set_error(NATTEN_B200_EINVAL, "rotary: null tensor");
  const int size = g->dtype == NATTEN_B200_F32 ? 4 : 2;
  const uintptr_t ptrs = (uintptr_t)q | (uintptr_t)k | (uintptr_t)yq | (uintptr_t)yk;
  if (ptrs % size != 0) return set_error(NATTEN_B200_EINVAL, "rotary: tensor pointers must be aligned to their elements");
  a.q = q; a.k = k; a.yq = yq; a.yk = yk;
  a.q_token = g->q_token_stride; a.q_head = g->q_head_stride; a.k_token = g->k_token_stride; a.k_head = g->k_head_stride;
  a.positions = g->positions;
  a.tokens = (uint32_t)(g->batch * n);
  a.per_sample = (uint32_t)n;
  a.heads_q = g->heads_q; a.heads_k = g->heads_k; a.D = g->head_dim; a.rank = g->rank;
  a.kind = g->position_kind; a.pos64 = g->position_bits == 64; a.pos_batch = g->position_batch != 0; a.inverse = inverse != 0;
  a.by_sample = FastDiv(a.per_sample);
  for (int i = 0; i < g->rank; ++i) a.by_ext[i] = FastDiv((uint32_t)g->extent[i]);
  for (int i = 0; i < a.pairs; ++i) a.phase[i] = g->phases[i];
  // 16-byte accesses when every head starts on such a boundary and no vector straddles the two halves
  const int ve = 16 / size;
  const uintptr_t steps = (uintptr_t)((a.q_token | a.q_head | a.k_token | a.k_head) * size) | (uintptr_t)(a.D * size);
  const bool aligned = (ptrs | steps) % 16 == 0;
  int mode, units;
  if (g->interleaved) {
    mode = aligned ? MODE_VEC_INTERLEAVED : MODE_PAIRS;
    units = aligned ? a.D / ve : a.pairs + (a.D - 2 * a.pairs);
  } else {
    const bool vec = aligned && a.pairs % ve == 0;
    mode = vec ? MODE_VEC_HALVES : MODE_PAIRS_HALVES;
    units = vec ? a.pairs / ve + (a.D - 2 * a.pairs) / ve : a.pairs + (a.D - 2 * a.pairs);
  }
  if ((long long)units * (a.heads_q + a.heads_k) * kTable > 0x7fffffffLL) return set_error(NATTEN_B200_EINVAL, "rotary: heads times head_dim too large");
  cudaStream_t s = (cudaStream_t)stream;
  if (g->dtype == NATTEN_B200_F32) return launch<float>(a, mode, units, s);
  return g->dtype == NATTEN_B200_F16 ? launch<__half>(a, mode, units, s) : launch<__nv_bfloat16>(a, mode, units, s);
}
