// Attention to a shared prefix on the tensor cores (bf16, fp16).
//
// The queries of one key/value head, over all samples, positions and heads of its group, are the rows of one product,
// so the prefix is read once for the batch.  A block owns two tiles of up to 128 rows and a range of 128-key chunks:
//   TMA warp       Q tiles once, then K and V chunks into a ring of shared-memory slots (zero fill past the ends)
//   MMA warp       S = Q K^T into tensor memory, O += P V with P from tensor memory (over S) and V MN-major
//   8 softmax warps   one thread per row (four warps per tile): the chunk's maximum, P = 2^(scale S - m) rounded to the
//                  tensors' type, the row's sum in float32; O stays in tensor memory for the whole range
// While one tile's softmax runs the tensor core works for the other tile.  The reference maximum m of a row follows the
// true one lazily: O and the sum are rescaled only when a chunk exceeds m by 2^8, so that P stays finite in either type.
#include <cuda.h>
#include <math.h>

#include <type_traits>

#include "fna_sm100.cuh"
#include "prefix.cuh"
#include "sm100_ptx.cuh"

namespace nb {
namespace {

using namespace sm100;

constexpr int kSMs = 148;
constexpr int kRows = 128;               // rows of a tile = lanes of tensor memory
constexpr int kKeys = 128;               // keys of a chunk
constexpr int kThreads = 320;
constexpr int kBlk = kRows * 128;        // bytes of 128 rows x 64 channels, one 128-byte swizzled row each
constexpr int kMaxSlots = 8;
constexpr float kLazy = 8.f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr uint32_t kOCol = 256;          // tensor memory: S / P of tile t at column t * 128, O at 256 + t * 128

struct alignas(64) PrefixMaps {
  CUtensorMap q, k, v;
};

struct PrefixTc {
  PrefixArgs a;
  int tile_tokens;                       // query tokens of a tile: 128 / G
  long long tiles;                       // row tiles of a key/value head
  int pairs;                             // blocks of two tiles
  int slots;                             // ring slots of one K or V chunk
  int chunks;
  float scale_log2;
  int* status;
};

enum { B_Q = 0, B_FULL = 1, B_EMPTY = B_FULL + kMaxSlots, B_S = B_EMPTY + kMaxSlots, B_P = B_S + 2, B_PV = B_P + 2, B_DRAIN = B_PV + 2, B_COUNT };

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <bool BF16>
__device__ __forceinline__ float2 unpack_pair(uint32_t v) {
  if constexpr (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
        "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// Sum over the keys [key0, key1) of one row, computed by a whole warp from global memory: for rows of a chunk in which
// their keys end and whose result came out non-finite, because a value past the row's end (which another sample sees)
// is not finite and met a zero probability in the matrix product.  m is the row's base-2 reference.  acc[i] gets column
// i * 32 + lane.
template <bool BF16>
__device__ __noinline__ void row_alone(const PrefixArgs& a, long long token, int h, int hk, int key0, int key1, float m,
                                       float scale_log2, float (&acc)[4]) {
  typedef typename std::conditional<BF16, __nv_bfloat16, __half>::type T;
  const int lane = threadIdx.x & 31;
  const T* q = static_cast<const T*>(a.q) + token * a.q_token + (long long)h * a.q_head;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = 0.f;
  for (int first = key0; first < key1; first += 32) {
    const int key = first + lane;
    float p = 0.f;
    if (key < key1) {
      const T* k = static_cast<const T*>(a.k) + (long long)key * a.k_token + (long long)hk * a.k_head;
      float s = 0.f;
      for (int d = 0; d < a.D; ++d) s = fmaf(to_f<T>(q[d]), to_f<T>(k[d]), s);
      p = to_f<T>(from_f<T>(ex2(fmaf(s, scale_log2, -m))));
    }
    const int n = min(32, key1 - first);
    for (int j = 0; j < n; ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j);
      const T* v = static_cast<const T*>(a.v) + (long long)(first + j) * a.v_token + (long long)hk * a.v_head;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i * 32 + lane < a.D) acc[i] = fmaf(pj, to_f<T>(v[i * 32 + lane]), acc[i]);
    }
  }
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
prefix_sm100(const __grid_constant__ PrefixTc p, const __grid_constant__ PrefixMaps maps) {
  constexpr int NB = DP / 64;                               // 64-channel blocks of a row
  constexpr uint32_t kTileBytes = NB * kBlk;                // a Q tile, a K chunk, a V chunk
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* ring = smem + 2 * kTileBytes;
  __shared__ uint64_t bars[B_COUNT];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word, limit_word;
  volatile int* abort_flag = &abort_word;

  const PrefixArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };

  // work item: row tiles run fastest, so that blocks that run together read the same keys
  uint32_t w = blockIdx.x;
  const int pair = (int)(w % (uint32_t)p.pairs); w /= (uint32_t)p.pairs;
  const int split = (int)(w % (uint32_t)a.splits); w /= (uint32_t)a.splits;
  const int hk = (int)w;
  const int c0 = (int)((long long)p.chunks * split / a.splits);
  int c1 = (int)((long long)p.chunks * (split + 1) / a.splits);
  const int nt = (long long)pair * 2 + 1 < p.tiles ? 2 : 1;

  if (tid == 0) {
    mbar_init(bar(B_Q), 1);
    for (int i = 0; i < kMaxSlots; ++i) { mbar_init(bar(B_FULL + i), 1); mbar_init(bar(B_EMPTY + i), 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(bar(B_S + i), 1); mbar_init(bar(B_P + i), 4); mbar_init(bar(B_PV + i), 1); }
    mbar_init(bar(B_DRAIN), 1);
    abort_word = 0;
    limit_word = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (warp == 9) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  // this thread's row (softmax warps)
  const int tile = warp >> 2;                               // 0 or 1; 2 for the other warps
  const int r = tid & 127;
  long long token = 0;
  int head = 0, limit = 0;
  bool alive = false;
  if (warp < 8) {
    const int tl = r / a.G;
    token = ((long long)pair * 2 + tile) * p.tile_tokens + tl;
    alive = tl < p.tile_tokens && token < a.tokens;
    head = hk * a.G + (r - tl * a.G);
    limit = alive ? prefix_limit(a, token) : 0;
    if (a.lens != nullptr) {
      const int most = __reduce_max_sync(0xffffffffu, limit);
      if (lane == 0) atomicMax(&limit_word, most);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  if (a.lens != nullptr) c1 = min(c1, (limit_word + kKeys - 1) / kKeys);      // keys that no row of the block sees
  const int n = max(c1 - c0, 0);

  if (warp == 8) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0 && n > 0) {
      bool ok = true;
      mbar_arrive_expect_tx(bar(B_Q), (uint32_t)(nt * NB * 128 * a.G * p.tile_tokens));
      for (int t = 0; t < nt; ++t)
        for (int b = 0; b < NB; ++b)
          tma_load_3d(smem_u32(smem + t * kTileBytes + b * kBlk), &maps.q, bar(B_Q), b * 64, hk * a.G,
                      (int)(((long long)pair * 2 + t) * p.tile_tokens));
      uint32_t st = 0, par = 1u;
      for (int i = 0; i < 2 * n; ++i) {                     // K and V of a chunk in turn
        ok = mbar_wait(bar(B_EMPTY + st), par, abort_flag);
        if (!ok) break;
        mbar_arrive_expect_tx(bar(B_FULL + st), kTileBytes);
        const CUtensorMap* m = (i & 1) ? &maps.v : &maps.k;
        for (int b = 0; b < NB; ++b)
          tma_load_3d(smem_u32(ring + st * kTileBytes + b * kBlk), m, bar(B_FULL + st), b * 64, hk, (c0 + (i >> 1)) * kKeys);
        if (++st == (uint32_t)p.slots) { st = 0; par ^= 1u; }
      }
      if (!ok) {                                            // copies in flight land before the block gives its memory back
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {}
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    // ------------------------------------------------------------------ MMA issuer
    if (lane == 0 && n > 0) {
      const uint32_t fmt = BF16 ? 1 : 0;
      const uint32_t idesc_qk = instr_desc(kRows, kKeys, fmt, 0, 0), idesc_pv = instr_desc(kRows, DP, fmt, 0, 1);
      const uint64_t kdesc0 = smem_desc(0, 16, 1024, 2), vdesc0 = smem_desc(0, kBlk, 1024, 2);
      const uint32_t q_lo = smem_u32(smem) >> 4, ring_lo = smem_u32(ring) >> 4;
      uint32_t st = 0, par = 0;
      auto next = [&]() { if (++st == (uint32_t)p.slots) { st = 0; par ^= 1u; } };
      auto qk = [&](int t, uint32_t slot) {
        const uint64_t ad = kdesc0 + q_lo + (uint32_t)t * (kTileBytes >> 4), bd = kdesc0 + ring_lo + slot * (kTileBytes >> 4);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            mma_ss(tmem + t * 128, ad + b * (kBlk >> 4) + 2 * ks, bd + b * (kBlk >> 4) + 2 * ks, idesc_qk, b + ks > 0 ? 1u : 0u);
        mma_commit(bar(B_S + t));
      };
      bool ok = mbar_wait(bar(B_Q), 0, abort_flag) && mbar_wait(bar(B_FULL + st), par, abort_flag);
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < nt; ++t) qk(t, st);
        mma_commit(bar(B_EMPTY + st));
        next();
      }
      for (int j = 0; j < n && ok; ++j) {
        const uint32_t v_st = st, v_par = par;
        next();
        const uint32_t k_st = st, k_par = par;
        const bool more = j + 1 < n;
        if (more) next();
        for (int t = 0; t < nt && ok; ++t) {
          if (t == 0) ok = mbar_wait(bar(B_FULL + v_st), v_par, abort_flag);
          ok = ok && mbar_wait_hot(bar(B_P + t), (uint32_t)j & 1u, abort_flag);
          if (!ok) break;
          tc_fence_after();
          uint64_t bd = vdesc0 + ring_lo + v_st * (kTileBytes >> 4);
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)            // 16 keys: next 16 rows of V, next 8 columns of packed P
            mma_ts(tmem + kOCol + t * 128, tmem + t * 128 + kk * 8, bd + kk * 128, idesc_pv, j + kk > 0 ? 1u : 0u);
          mma_commit(bar(B_PV + t));
          if (t == nt - 1) mma_commit(bar(B_EMPTY + v_st));
          if (more) {
            if (t == 0) ok = mbar_wait(bar(B_FULL + k_st), k_par, abort_flag);
            if (!ok) break;
            tc_fence_after();
            qk(t, k_st);                                     // executes after P V, which has read P from the same columns
            if (t == nt - 1) mma_commit(bar(B_EMPTY + k_st));
          }
        }
      }
      // every MMA is finished before tensor memory is given back
      mma_commit(bar(B_DRAIN));
      for (uint32_t i = 0; i < kSpinLimit; ++i)
        if (mbar_try_wait(bar(B_DRAIN), 0)) break;
    }
    __syncwarp();
  } else if (tile < nt) {
    // ------------------------------------------------------------------ softmax and epilogue
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + tile * 128, o_addr = tmem + lanes + kOCol + tile * 128;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = mbar_wait(bar(B_S + tile), (uint32_t)j & 1u, abort_flag);
      if (!ok) break;
      tc_fence_after();
      uint32_t s[128];
#pragma unroll
      for (int g = 0; g < 4; ++g) tmem_ld32(s_addr + g * 32, s + g * 32);
      tmem_wait_ld();
      const int left = limit - (c0 + j) * kKeys;             // keys of the chunk that the row sees
      if (__any_sync(0xffffffffu, alive && left < kKeys)) {
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i] = i < left ? s[i] : 0xff800000u;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 128; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(s[i]));
      const float mc = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
      const bool first = m == -INFINITY;
      const bool bump = alive && !first && mc > m + kLazy;
      if (__any_sync(0xffffffffu, bump)) {
        // O is being accumulated by the P V of the chunk before: wait for it, then scale
        ok = mbar_wait(bar(B_PV + tile), (uint32_t)(j - 1) & 1u, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const float alpha = bump ? ex2(m - mc) : 1.f;
#pragma unroll 1
        for (int g = 0; g < DP / 16; ++g) {
          uint32_t f[16];
          tmem_ld16(o_addr + g * 16, f);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = __float_as_uint(__uint_as_float(f[i]) * alpha);
          tmem_st16(o_addr + g * 16, f);
        }
        tmem_wait_st();
        l *= alpha;
        if (bump) m = mc;
      }
      if (first) m = mc;
      const float base = m == -INFINITY ? 0.f : m;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e0 = ex2(fmaf(__uint_as_float(s[g * 32 + 2 * i]), p.scale_log2, -base));
          const float e1 = ex2(fmaf(__uint_as_float(s[g * 32 + 2 * i + 1]), p.scale_log2, -base));
          sum[i & 3] += e0 + e1;
          pk[i] = pack_pair<BF16>(e0, e1);
        }
        tmem_st16(s_addr + g * 16, pk);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_P + tile));
    }
    if (ok && n > 0) ok = mbar_wait(bar(B_PV + tile), (uint32_t)(n - 1) & 1u, abort_flag);
    if (ok) {
      tc_fence_after();
      const bool last = a.splits == 1;
      const long long at = token * a.Hq + head;
      float lse = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
      float wa = 1.f, wb = 0.f;
      const bool win = last && a.window_lse != nullptr;
      if (win && alive) lse = join_weights(lse, a.window_lse[at], wa, wb);
      const float co = l == 0.f ? 0.f : wa / l;              // a NaN sum stays one
      bool odd = false;
#pragma unroll 1
      for (int g = 0; g < DP / 16; ++g) {
        uint32_t f[16];
        if (n > 0) {
          tmem_ld16(o_addr + g * 16, f);
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float v = co != 0.f && n > 0 ? __uint_as_float(f[i]) * co : 0.f;
          odd = odd || (co != 0.f && !isfinite(v) && g * 16 + i < a.D);
          f[i] = __float_as_uint(v);
        }
        if (alive) {
#pragma unroll
          for (int h8 = 0; h8 < 2; ++h8) {
            const int c = g * 16 + h8 * 8;
            if (c >= a.D) break;                             // head dims are multiples of 8
            if (last) {
              if (win && wb != 0.f) {
                const uint4 raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.window_out) + at * a.D + c));
                const uint32_t rw[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 o = unpack_pair<BF16>(rw[i]);
                  f[h8 * 8 + 2 * i] = __float_as_uint(fmaf(wb, o.x, __uint_as_float(f[h8 * 8 + 2 * i])));
                  f[h8 * 8 + 2 * i + 1] = __float_as_uint(fmaf(wb, o.y, __uint_as_float(f[h8 * 8 + 2 * i + 1])));
                }
              }
              uint32_t pk[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                pk[i] = pack_pair<BF16>(__uint_as_float(f[h8 * 8 + 2 * i]), __uint_as_float(f[h8 * 8 + 2 * i + 1]));
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at * a.D + c) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            } else {
              float* dst = a.part_out + ((long long)split * a.tokens * a.Hq + at) * a.D + c;
              *reinterpret_cast<uint4*>(dst) = make_uint4(f[h8 * 8], f[h8 * 8 + 1], f[h8 * 8 + 2], f[h8 * 8 + 3]);
              *reinterpret_cast<uint4*>(dst + 4) = make_uint4(f[h8 * 8 + 4], f[h8 * 8 + 5], f[h8 * 8 + 6], f[h8 * 8 + 7]);
            }
          }
        }
      }
      if (alive) {
        if (!last) a.part_lse[(long long)split * a.tokens * a.Hq + at] = lse;
        else if (a.lse != nullptr) a.lse[at] = lse;
      }
      // rows whose keys end inside the block's range and that met a non-finite value past their end
      uint32_t again = __ballot_sync(0xffffffffu, a.lens != nullptr && alive && odd && limit < c1 * kKeys);
      typedef typename std::conditional<BF16, __nv_bfloat16, __half>::type T;
      while (again != 0) {
        const int who = __ffs(again) - 1;
        again &= again - 1;
        const long long tok = __shfl_sync(0xffffffffu, token, who);
        const int h = __shfl_sync(0xffffffffu, head, who), lim = __shfl_sync(0xffffffffu, limit, who);
        const float mm = __shfl_sync(0xffffffffu, m, who), cc = __shfl_sync(0xffffffffu, co, who), bb = __shfl_sync(0xffffffffu, wb, who);
        float acc[4];
        row_alone<BF16>(a, tok, h, hk, c0 * kKeys, lim, mm, p.scale_log2, acc);
        const long long row = tok * a.Hq + h;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = i * 32 + lane;
          if (c < a.D) {
            float v = acc[i] * cc;
            if (last) {
              if (win && bb != 0.f) v = fmaf(bb, to_f<T>(static_cast<const T*>(a.window_out)[row * a.D + c]), v);
              static_cast<T*>(a.out)[row * a.D + c] = from_f<T>(v);
            } else {
              a.part_out[((long long)split * a.tokens * a.Hq + row) * a.D + c] = v;
            }
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (tid == 0 && *abort_flag && p.status != nullptr) atomicExch(p.status, 1);
}

// [tokens, heads, D] with any token and head stride: box of 64 channels x `heads` x `rows`.
int encode_rows(CUtensorMap* map, const void* base, int dtype, int D, int heads, long long tokens, long long head_stride,
                long long token_stride, int box_heads, int box_rows) {
  const auto enc = reinterpret_cast<CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill)>(sm100_encode_tiled());
  if (enc == nullptr) return set_error(NATTEN_B200_ENODEVICE, "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows}, step[3] = {1, 1, 1};
  const CUresult r = enc(map, dtype == NATTEN_B200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(NATTEN_B200_ELAUNCH, "cuTensorMapEncodeTiled failed with code %d", (int)r);
  return NATTEN_B200_OK;
}

template <int DP, bool BF16>
int launch(const PrefixTc& p, const PrefixMaps& maps, cudaStream_t s) {
  const size_t tile = (size_t)(DP / 64) * kBlk, smem = 1024 + 2 * tile + (size_t)p.slots * tile;
  const cudaError_t e = cudaFuncSetAttribute(prefix_sm100<DP, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return set_error(NATTEN_B200_ELAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  }
  const long long grid = (long long)p.pairs * p.a.splits * p.a.Hkv;
  NB_LAUNCH("prefix_sm100", s, prefix_sm100<DP, BF16><<<(unsigned)grid, kThreads, smem, s>>>(p, maps));
  return check_launch("prefix attention (tensor cores)");
}

long long row_tiles(const PrefixArgs& a) {
  const int tt = kRows / a.G;
  return (a.tokens + tt - 1) / tt;
}

}  // namespace

const char* prefix_sm100_unsupported(const PrefixArgs& a, int dtype) {
  if (dtype == NATTEN_B200_F32) return "float32";
  if (a.D % 8 != 0 || a.D > 128) return "head_dim is not a multiple of 8 up to 128";
  if (a.G > kRows) return "more than 128 query heads for one key/value head";
  if (a.prefix < 1) return "the prefix is empty";
  // tensor maps: strides are positive multiples of 16 bytes below 2^40
  for (long long st : {a.q_token, a.q_head, a.k_token, a.k_head, a.v_token, a.v_head})
    if (st < 8 || st % 8 != 0 || st >= (1ll << 38)) return "a stride is not a positive multiple of 16 bytes";
  if ((row_tiles(a) + 1) / 2 * a.Hkv > 0x7fffffLL) return "too many row tiles";
  return nullptr;
}

// Parts of the prefix.  A block takes about one unit of time per chunk of 128 keys and about three to start and finish;
// the blocks run in waves of one per SM, and joining parts costs another launch.
int prefix_sm100_splits(const PrefixArgs& a) {
  const long long items = (row_tiles(a) + 1) / 2 * a.Hkv, chunks = (a.prefix + kKeys - 1) / kKeys;
  long long best = 1;
  double best_cost = 1e300;
  for (long long n = 1; n <= chunks && n <= 256 && (n == 1 || items * n <= 2 * kSMs); ++n) {
    const double waves = (double)((items * n + kSMs - 1) / kSMs);
    const double cost = waves * ((double)((chunks + n - 1) / n) + 3.0) + (n > 1 ? 3.0 + 0.02 * (double)n : 0.0);
    if (cost < best_cost) { best_cost = cost; best = n; }
  }
  return (int)best;
}

int run_prefix_sm100(const PrefixArgs& a, int dtype, cudaStream_t s) {
  PrefixTc p{};
  p.a = a;
  p.tile_tokens = kRows / a.G;
  p.tiles = row_tiles(a);
  p.pairs = (int)((p.tiles + 1) / 2);
  p.chunks = (a.prefix + kKeys - 1) / kKeys;
  p.slots = a.D <= 64 ? 8 : 5;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.status = sm100_status_word();
  if (p.status == nullptr) return set_error(NATTEN_B200_ENODEVICE, "tensor-core kernels need an sm_100 device");
  PrefixMaps maps;
  if (int rc = encode_rows(&maps.q, a.q, dtype, a.D, a.Hq, a.tokens, a.q_head, a.q_token, a.G, p.tile_tokens)) return rc;
  if (int rc = encode_rows(&maps.k, a.k, dtype, a.D, a.Hkv, a.prefix, a.k_head, a.k_token, 1, kKeys)) return rc;
  if (int rc = encode_rows(&maps.v, a.v, dtype, a.D, a.Hkv, a.prefix, a.v_head, a.v_token, 1, kKeys)) return rc;
  const bool bf = dtype == NATTEN_B200_BF16;
  if (a.D <= 64) return bf ? launch<64, true>(p, maps, s) : launch<64, false>(p, maps, s);
  return bf ? launch<128, true>(p, maps, s) : launch<128, false>(p, maps, s);
}

}  // namespace nb
