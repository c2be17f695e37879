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
//
// Small heads are bound by instructions before they are bound by memory: 100352 tokens of 8 heads of 32 (bf16) took 7000
// thread instructions a token and 32 us while every 16 bytes worked out their own address and every pair its position
// and an exact sincospif; 22 us now (15.7 us of memory at 6.5 TB/s).  589824 tokens of 32 heads of 64: 750 us, 98 % of
// the copy rate.  Four units in flight per thread where a unit is one access, two where it is two (32 registers of data
// either way): one in flight costs 15 % at these heads of 64.  Blocks for four per SM: eight leave the last round of
// runs half empty at 100352 tokens (24.5 us).
#include <math.h>

#include <algorithm>

#include "launch.cuh"

namespace nb {
namespace {

constexpr int kMaxPairs = 256;
constexpr int kTable = 1024;     // (token, pair) entries of a block's table: 8 KB
constexpr int kRun = 256;        // most tokens of a run
constexpr int kThreads = 256;    // most threads of a block
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
  FastDiv by_sample, by_ext[3], by_pairs, by_lanes, by_head;
  int units_token, units_head;                  // work units (16 bytes, two halves, or a pair) of a token and of a head
  int passes, lanes, step;                      // threads for a token, passes over its units, tokens at a time
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

// Cosine and sine of a number of half turns in [-1, 1).  For 16-bit types the fast instructions: their error, below
// 2^-20, is far less than the rounding of the result (2^-12 and 2^-9 of it).
template <typename T>
__device__ __forceinline__ float2 cos_sin(float half_turns) {
  float2 r;
  if constexpr (sizeof(T) == 4) sincospif(half_turns, &r.y, &r.x);
  else __sincosf(half_turns * 3.14159265358979f, &r.y, &r.x);
  return r;
}

// A thread keeps its place in a token (head and channels) for a whole pass over the run and goes from token to token, so
// that no address costs a division; it reads U tokens' channels before it works on the first, and the first ones before
// the run's table is there.
template <typename T, int MODE, int U>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  constexpr int VE = 16 / (int)sizeof(T);
  constexpr bool VEC = MODE == MODE_VEC_INTERLEAVED || MODE == MODE_VEC_HALVES, HALVES = MODE == MODE_VEC_HALVES || MODE == MODE_PAIRS_HALVES;
  __shared__ long long pos[kRun * 3];
  __shared__ float2 table[kTable];
  const int pairs = a.pairs, tid = threadIdx.x, threads = blockDim.x;          // 2 * pairs channels are rotated
  const uint32_t runs = (a.tokens + a.tile - 1) / a.tile;
  // the table: pairs next to each other, `step` tokens at a time
  const int step = max(threads / pairs, 1), t_first = pairs <= threads ? (int)a.by_pairs.div(tid) : 0, p_first = tid - t_first * pairs;
  auto axis_of = [&](int p) { return p < a.axis_end[0] ? 0 : p < a.axis_end[1] ? 1 : 2; };
  auto entry = [&](long long at, uint64_t phase) {
    // the top half of the fraction, read as signed: half turns in [-1, 1) after scaling
    float2 c = cos_sin<T>((float)(int)(((uint64_t)at * phase) >> 32) * 4.656612873077393e-10f);
    if (a.inverse) c.y = -c.y;
    return c;
  };
  const uint64_t own_phase = p_first < pairs ? a.phase[p_first] : 0;
  for (uint32_t run = blockIdx.x; run < runs; run += gridDim.x) {
    const uint32_t first = run * a.tile;
    const int n = (int)min((uint32_t)a.tile, a.tokens - first);
    for (int pass = 0; pass < a.passes; ++pass) {
      const int t_own = pass == 0 ? (int)a.by_lanes.div(tid) : 0, lane = tid - t_own * a.lanes, in_token = pass * a.lanes + lane;
      const bool idle = t_own >= a.step || lane >= a.lanes || in_token >= a.units_token;
      const int hh = (int)a.by_head.div(in_token), v = in_token - hh * a.units_head;
      const bool is_q = hh < a.heads_q;
      const int h = is_q ? hh : hh - a.heads_q;
      const long long token = (long long)first + t_own, in = is_q ? a.q_token : a.k_token, out = (long long)(is_q ? a.heads_q : a.heads_k) * a.D;
      const T* src = static_cast<const T*>(is_q ? a.q : a.k) + token * in + h * (is_q ? a.q_head : a.k_head);
      T* dst = static_cast<T*>(is_q ? a.yq : a.yk) + token * out + (long long)h * a.D;
      // channels of the unit: [c0, c0 + VE) and, for two halves, [c1, c1 + VE); without vectors two channels
      const int rot = MODE == MODE_VEC_HALVES ? pairs / VE : MODE == MODE_VEC_INTERLEAVED ? a.units_head : pairs;
      const bool turns = v < rot;
      const int c0 = VEC ? (MODE == MODE_VEC_HALVES && !turns ? 2 * pairs + (v - rot) * VE : v * VE) : !turns ? v + pairs : HALVES ? v : 2 * v;
      const int c1 = HALVES ? c0 + pairs : c0 + 1;
      src += c0;
      dst += c0;
      const int end = idle ? 0 : n;
      const long long in_step = in * a.step, out_step = out * a.step;
      int t = t_own;
      do {                                                 // at least once: the table is made inside
        uint4 raw[U][2];
        T one[U][2];
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (t + i * a.step < end) {
            const T* x = src + i * in_step;
            if constexpr (VEC) {
              raw[i][0] = *reinterpret_cast<const uint4*>(x);
              if (HALVES && turns) raw[i][1] = *reinterpret_cast<const uint4*>(x + pairs);
            } else {
              one[i][0] = x[0];
              if (turns) one[i][1] = x[c1 - c0];
            }
          }
        if (pass == 0 && t == t_own) {
          if (n * pairs <= threads) {                      // an entry for each thread: it finds its position by itself
            if (t_first < n) table[tid] = entry(position(a, first + t_first, axis_of(p_first)), own_phase);
          } else {
            for (int i = tid; i < n * a.axes; i += threads) {
              const int tt = i / a.axes;
              pos[i] = position(a, first + tt, i - tt * a.axes);
            }
            __syncthreads();
            for (int p = p_first; p < pairs; p += threads) {
              const int axis = axis_of(p);
              const uint64_t phase = p == p_first ? own_phase : a.phase[p];
              if (t_first < step)
                for (int tt = t_first; tt < n; tt += step) table[tt * pairs + p] = entry(pos[tt * a.axes + axis], phase);
            }
          }
          __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < U; ++i)
          if (t + i * a.step < end) {
            const float2* cs = table + (t + i * a.step) * pairs;
            T* y = dst + i * out_step;
            if constexpr (MODE == MODE_VEC_INTERLEAVED) {
              float f[VE];
              load16<T>(reinterpret_cast<const T*>(&raw[i][0]), f);
#pragma unroll
              for (int j = 0; j < VE / 2; ++j) {
                const int p = v * (VE / 2) + j;
                if (p < pairs) {
                  const float2 c = cs[p];
                  const float x0 = f[2 * j], x1 = f[2 * j + 1];
                  f[2 * j] = x0 * c.x - x1 * c.y;
                  f[2 * j + 1] = x0 * c.y + x1 * c.x;
                }
              }
              store16<T>(y, f);
            } else if constexpr (MODE == MODE_VEC_HALVES) {
              if (turns) {
                float f[VE], g[VE];
                load16<T>(reinterpret_cast<const T*>(&raw[i][0]), f);
                load16<T>(reinterpret_cast<const T*>(&raw[i][1]), g);
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                  const float2 c = cs[v * VE + j];
                  const float x0 = f[j], x1 = g[j];
                  f[j] = x0 * c.x - x1 * c.y;
                  g[j] = x0 * c.y + x1 * c.x;
                }
                store16<T>(y, f);
                store16<T>(y + pairs, g);
              } else {
                *reinterpret_cast<uint4*>(y) = raw[i][0];
              }
            } else if (turns) {
              const float2 c = cs[v];
              const float x0 = to_f<T>(one[i][0]), x1 = to_f<T>(one[i][1]);
              y[0] = from_f<T>(x0 * c.x - x1 * c.y);
              y[c1 - c0] = from_f<T>(x0 * c.y + x1 * c.x);
            } else {
              y[0] = one[i][0];
            }
          }
        src += U * in_step;
        dst += U * out_step;
        t += U * a.step;
      } while (t < end);
    }
    __syncthreads();
  }
}

template <typename T>
int launch(RotaryArgs& a, int mode, int units_head, cudaStream_t s) {
  a.units_head = units_head;
  a.units_token = units_head * (a.heads_q + a.heads_k);
  // the lanes of a token, in as many passes as it needs, and as many tokens at a time as the block has room for
  a.passes = (a.units_token + kThreads - 1) / kThreads;
  a.lanes = (a.units_token + a.passes - 1) / a.passes;
  a.step = a.passes > 1 ? 1 : kThreads / a.lanes;
  const int threads = (a.lanes * a.step + 31) / 32 * 32;
  a.by_pairs = FastDiv(a.pairs);
  a.by_lanes = FastDiv(a.lanes);
  a.by_head = FastDiv(a.units_head);
  // as many tokens as the table holds, but runs for all blocks while there are so many tokens, and as many for each
  const uint32_t room = std::min(kTable / a.pairs, kRun), most = kSMs * 4, rounds = (uint32_t)((a.tokens + (uint64_t)most * room - 1) / ((uint64_t)most * room));
  a.tile = (int)((a.tokens + (uint64_t)most * rounds - 1) / ((uint64_t)most * rounds));
  const uint32_t runs = (a.tokens + a.tile - 1) / a.tile;
  const int grid = (int)(runs < most ? runs : most);
  switch (mode) {
    case MODE_VEC_INTERLEAVED: NB_LAUNCH("rotary", s, rotary_kernel<T, MODE_VEC_INTERLEAVED, 4><<<grid, threads, 0, s>>>(a)); break;
    case MODE_VEC_HALVES: NB_LAUNCH("rotary", s, rotary_kernel<T, MODE_VEC_HALVES, 2><<<grid, threads, 0, s>>>(a)); break;
    case MODE_PAIRS_HALVES: NB_LAUNCH("rotary", s, rotary_kernel<T, MODE_PAIRS_HALVES, 4><<<grid, threads, 0, s>>>(a)); break;
    default: NB_LAUNCH("rotary", s, rotary_kernel<T, MODE_PAIRS, 4><<<grid, threads, 0, s>>>(a)); break;
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
  if (g->position_kind != POS_GRID && (uintptr_t)g->positions % (g->position_bits / 8) != 0)
    return set_error(NATTEN_B200_EINVAL, "rotary: positions must be aligned to their elements");
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
