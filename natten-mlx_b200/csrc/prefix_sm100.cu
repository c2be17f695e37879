// Attention to a shared prefix on the tensor cores (bf16, fp16).
//
// The queries of one key/value head, over all samples, positions and heads of its group, are the rows of one product,
// so the prefix is read once for the batch.  A block owns two tiles of up to 128 rows and a range of the prefix in chunks
// of 96 keys (head dims to 64) or 128:
//   TMA warp       Q tiles once, then K and V chunks into a ring of shared-memory slots (zero fill past the ends)
//   MMA warp       S = Q K^T into tensor memory, O += P V with P from tensor memory (over S) and V MN-major
//   softmax warps  a thread per row, or two (head dims to 64) that share the chunk's keys: the row's maximum, P =
//                  2^(scale S - m) rounded to the tensors' type, which the tensor core needs, the sum in float32; O stays
//                  in tensor memory throughout
// While one tile's softmax runs the tensor core works for the other tile.  A block that has one tile only lets its two
// halves take every other chunk for it.  The reference maximum m of a row follows the true one lazily: O and the sum are
// rescaled only when a chunk exceeds m by 2^8, so that P stays finite in either type.
//
// What bounds it, and what was measured (bf16, 4096 keys):
// - Heads of 128, 16384 rows of 8 heads: 255 us, 1078 TFLOP/s, 66 % of the rate of a large library matrix product.  The
//   tensor core is the bound, kept waiting at the ends of a block and by the one thread that issues its products.
// - Heads of 64, 16384 rows of 16 heads: 391 us, 703 TFLOP/s, 43 %.  The products alone would take 234 us (P V of
//   64 columns fills half of what the unit does at 128), the exponentials alone 239 us (16 per SM and clock), and the two
//   overlap in part only: a chunk is 96 keys so that two buffers of S for each tile fit tensor memory, and Q K^T of the
//   next chunk runs under this one's softmax.  Slower were: one buffer and 192 keys, two blocks per SM with chunks of 64
//   keys, three tiles of one buffer each (406 us; the tiles wait for the same two units in turn, whichever their number),
//   S read twice instead of kept, a second warp that issues products, a part of the exponentials as polynomials, and the
//   two tiles taking turns at the exponentials by a barrier (436 us), and exponentials beside the maximum, with the
//   reference so far, that are repeated where it does not hold (464 us: P can be handed over only after the check).
//   Without the exponentials it would take 294 us, without the exchange of maxima between a row's two threads 366 us.
// - Two threads per row: heads of 64 391 us, one 409 us; heads of 128 268 us, one 255 us (with 128 keys of S in its
//   registers a thread has no room for a second buffer's, and the pair's exchange of maxima costs more than it gives).
// - Few rows: 128 rows of 4 heads of 128 over 65536 keys (fp16) 40 us, of which the 134 MB of keys and values need 21 us;
//   the first S is there after 5 us, the parts' results and their joining take 7 us.
#include <cuda.h>
#include <math.h>

#include <type_traits>

#include "f32x2.cuh"
#include "fna_sm100.cuh"
#include "prefix.cuh"
#include "sm100_ptx.cuh"

namespace nb {
namespace {

using namespace sm100;

constexpr int kSMs = 148;
constexpr int kRows = 128;               // rows of a tile = lanes of tensor memory
constexpr int kSteps = 8;               // barriers of the ring, by step
// For heads padded to DP channels: keys of a chunk, buffers of S / P for a tile, threads per row and keys of each, and the
// threads of a block (the softmax warps of two tiles, a warp that loads, a warp that issues the products).
template <int DP> struct Shape {
  static constexpr int kKeys = DP == 64 ? 96 : 128, kBufs = DP == 64 ? 2 : 1, kSplit = DP == 64 ? 2 : 1, kEach = kKeys / kSplit;
  static constexpr int kSoftmax = 256 * kSplit, kThreads = kSoftmax + 64;
  static constexpr uint32_t kOCol = 2 * kBufs * kKeys;       // tensor memory: S / P of the tiles, then their O
  static_assert(kOCol + 2 * DP <= 512, "tensor memory");
};
constexpr float kLazy = 8.f;
constexpr float kLn2 = 0.6931471805599453f;

struct alignas(64) PrefixMaps {
  CUtensorMap q, k, v;
};

struct PrefixTc {
  PrefixArgs a;
  int tile_tokens;                       // query tokens of a tile: 128 / G
  long long tiles;                       // row tiles of a key/value head
  int pairs;                             // blocks of two tiles
  int whole, cut;                        // work items that are one block's, and items that are cut into parts
  int q_tiles;                           // Q tiles in shared memory: 1 when no block has two
  int slots;                             // ring slots of one K or V chunk
  int chunks;
  float scale_log2;
  int* status;
};

struct Results {
  float sums[2][2][kRows], refs[2][kRows];                  // by stream and part of the keys; by stream
};

enum { B_Q = 0, B_FULL = 1, B_EMPTY = B_FULL + kSteps, B_S = B_EMPTY + kSteps, B_P = B_S + 4, B_PV = B_P + 4, B_COUNT = B_PV + 4 };

template <int kBufs> struct Shared {
  float peak[kBufs][2][2][kRows];                           // a chunk's maximum by buffer, stream, half of the keys and row
  uint64_t bars[B_COUNT];
  uint32_t tmem_slot;
  int abort_word, limit_word;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Largest of three; NaN if one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
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

__device__ __forceinline__ void store32(float* p, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
               "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// For the many warps that wait for a product: each try suspends the warp for a short while, so that waiting takes few issue
// slots from the warps that compute.
__device__ __forceinline__ bool wait_softly(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
#pragma unroll 1
  for (uint32_t it = 0; it < kPollLimit; ++it) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred P1;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 P1, [%1], %2, %3;\n\t"
        "selp.b32 %0, 1, 0, P1;\n\t}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(20u)
        : "memory");
    if (ok) return true;
  }
  return mbar_wait(bar, parity, abort_flag);
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
__global__ void __launch_bounds__(Shape<DP>::kThreads, 1)
prefix_sm100(const __grid_constant__ PrefixTc p, const __grid_constant__ PrefixMaps maps) {
  constexpr int NB = DP / 64;                               // 64-channel blocks of a row
  typedef Shape<DP> Sh;
  constexpr int kKeys = Sh::kKeys, kSplit = Sh::kSplit, kEach = Sh::kEach, kBufs = Sh::kBufs, kWarps = Sh::kSoftmax / 32;
  constexpr uint32_t kOCol = Sh::kOCol;
  constexpr uint32_t kQBlk = kRows * 128, kBlk = kKeys * 128;      // bytes of 64 channels of a Q tile and of a chunk
  constexpr uint32_t kQBytes = NB * kQBlk, kTileBytes = NB * kBlk; // a Q tile; a K or V chunk
  // The tiles come first: they need 1024-byte alignment, which the start of a block's shared memory has, and with a
  // 128-channel ring of five slots there is no room to round it up.
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* ring = smem + p.q_tiles * kQBytes;
  Shared<kBufs>& sh = *reinterpret_cast<Shared<kBufs>*>(ring + p.slots * kTileBytes);
  Results& res = *reinterpret_cast<Results*>(smem);         // over Q, once every product is done
  volatile int* abort_flag = &sh.abort_word;

  const PrefixArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t bar0 = smem_u32(sh.bars);
  auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };

  // Work items are (row tile pair, key/value head), pairs running fastest so that blocks that run together read the
  // same keys.  The first p.whole of them are a block's each, the others are cut into a.splits ranges of chunks.
  const bool whole = blockIdx.x < (uint32_t)p.whole;
  const uint32_t x = whole ? blockIdx.x : blockIdx.x - p.whole;
  const int split = whole ? 0 : (int)(x % (uint32_t)a.splits), parts = whole ? 1 : a.splits;
  const uint32_t item = whole ? x : p.whole + x / (uint32_t)a.splits;
  const int hk = (int)(item / (uint32_t)p.pairs), pair_id = (int)(item - (uint32_t)hk * p.pairs);
  const int c0 = (int)((long long)p.chunks * split / parts);
  int c1 = (int)((long long)p.chunks * (split + 1) / parts);
  // two streams of products: two tiles, each over all chunks, or (twin) one tile of which either stream takes every
  // other chunk
  const bool twin = (long long)pair_id * 2 + 1 >= p.tiles;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the joining kernel may be set up meanwhile
  // The loading warp sets the barriers up and goes on to load at once; the others meet when tensor memory is there.
  if (warp == kWarps) {
    if (lane == 0) {
      mbar_init(bar(B_Q), 1);
      for (int i = 0; i < kSteps; ++i) { mbar_init(bar(B_FULL + i), 1); mbar_init(bar(B_EMPTY + i), 1); }
      for (int i = 0; i < 4; ++i) { mbar_init(bar(B_S + i), 1); mbar_init(bar(B_P + i), 4 * kSplit); mbar_init(bar(B_PV + i), 1); }
      sh.abort_word = (smem_u32(smem) & 1023u) != 0 ? 1 : 0;  // every wait then gives up, and the status says so
      sh.limit_word = 0;
      mbar_fence_init();
      tma_prefetch_desc(&maps.q);
      tma_prefetch_desc(&maps.k);
      tma_prefetch_desc(&maps.v);
    }
    __syncwarp();
  } else if (warp == kWarps + 1) {
    tmem_alloc(smem_u32(&sh.tmem_slot), 512);
    tmem_relinquish();
  }
  // softmax threads: stream, half of the chunk's keys, row
  const int stream = (warp / (4 * kSplit)) & 1, keys = kSplit == 1 ? 0 : (warp >> 2) & 1, r = tid & 127;
  long long token = 0;
  int head = 0, limit = 0;
  bool alive = false;
  if (warp < kWarps) {
    const int tl = r / a.G;
    token = ((long long)pair_id * 2 + (twin ? 0 : stream)) * p.tile_tokens + tl;
    alive = tl < p.tile_tokens && token < a.tokens;
    head = hk * a.G + (r - tl * a.G);
    limit = alive ? prefix_limit(a, token) : 0;
  }
  tc_fence_before();
  if (a.lens != nullptr) {                                  // keys that no row of the block sees are left out
    __syncthreads();
    const int most = __reduce_max_sync(0xffffffffu, limit);
    if (warp < kWarps && lane == 0) atomicMax(&sh.limit_word, most);
    __syncthreads();
    c1 = min(c1, (sh.limit_word + kKeys - 1) / kKeys);
  } else if (warp == kWarps) {
    __threadfence_block();
    asm volatile("bar.arrive 10, %0;" ::"n"(Sh::kThreads) : "memory");
  } else {
    asm volatile("bar.sync 10, %0;" ::"n"(Sh::kThreads) : "memory");
  }
  tc_fence_after();
  const uint32_t tmem = warp == kWarps ? 0u : sh.tmem_slot;
  const int n = max(c1 - c0, 0);
  // A stream has kBufs buffers of S / P, so Q K^T of its next chunks can run before P V of the present one.  Step s
  // issues P V of chunk s and then Q K^T of chunk s + ahead, into the buffer that has become free; the steps before 0 are
  // Q K^T alone.  V(s) and K(s + ahead) share a pair of barriers: full for both, and empty when Q K^T of chunk s + ahead is
  // done, which runs last.
  const int ahead = twin ? 2 * kBufs : kBufs;

  if (warp == kWarps) {
    // ------------------------------------------------------------------ TMA producer
    if (n > 0 && elect_one()) {
      bool ok = true;
      mbar_arrive_expect_tx(bar(B_Q), (uint32_t)((twin ? 1 : 2) * NB * 128 * a.G * p.tile_tokens));
      for (int t = 0; t < (twin ? 1 : 2); ++t)
        for (int b = 0; b < NB; ++b)
          tma_load_3d(smem_u32(smem + t * kQBytes + b * kQBlk), &maps.q, bar(B_Q), b * 64, hk * a.G,
                      (int)(((long long)pair_id * 2 + t) * p.tile_tokens));
      // The q-th chunk to be loaded goes to slot q % slots.  It is free when the chunk q - slots has been used: in the
      // step that chunk belongs to.
      int q = 0, slot = 0, freed = -ahead;                  // steps before `freed` are known to be over
      auto load = [&](const CUtensorMap* m, int c, int s) {
        const int old = q - p.slots;
        const int t = old < 0 ? -ahead - 1 : old < ahead ? old - ahead : (old - ahead) >> 1;
        for (; ok && freed <= t; ++freed)
          ok = mbar_wait(bar(B_EMPTY + ((freed + ahead) & (kSteps - 1))), (uint32_t)((freed + ahead) / kSteps) & 1u, abort_flag);
        if (!ok) return;
        for (int b = 0; b < NB; ++b)
          tma_load_3d(smem_u32(ring + slot * kTileBytes + b * kBlk), m, bar(B_FULL + ((s + ahead) & (kSteps - 1))), b * 64, hk,
                      (c0 + c) * kKeys);
        ++q;
        if (++slot == p.slots) slot = 0;
      };
      for (int s = -ahead; s < n && ok; ++s) {
        const bool v = s >= 0, k = s + ahead < n;
        // a barrier's phase of kSteps steps ago is over before its next one begins
        for (; ok && freed <= s - kSteps; ++freed)
          ok = mbar_wait(bar(B_EMPTY + ((freed + ahead) & (kSteps - 1))), (uint32_t)((freed + ahead) / kSteps) & 1u, abort_flag);
        if (!ok) break;
        if (!v && !k) continue;
        mbar_arrive_expect_tx(bar(B_FULL + ((s + ahead) & (kSteps - 1))), (v ? kTileBytes : 0u) + (k ? kTileBytes : 0u));
        if (v) load(&maps.v, s, s);
        if (ok && k) load(&maps.k, s + ahead, s);
      }
      if (!ok) {                                            // copies in flight land before the block gives its memory back
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {}
      }
    }
    __syncwarp();
  } else if (warp > kWarps) {
    // ------------------------------------------------------------------ MMA issuer
    if (n > 0 && elect_one()) {
      const int fmt = BF16 ? 1 : 0;
      const uint32_t idesc_qk = instr_desc(kRows, kKeys, fmt, 0, 0), idesc_pv = instr_desc(kRows, DP, fmt, 0, 1);
      const uint64_t kdesc0 = smem_desc(0, 16, 1024, 2) + (smem_u32(ring) >> 4), vdesc0 = smem_desc(0, kBlk, 1024, 2) + (smem_u32(ring) >> 4);
      const uint64_t qdesc0 = smem_desc(0, 16, 1024, 2) + (smem_u32(smem) >> 4);
      // One thread does all of this between two products, so its bookkeeping is kept to increments: a ready wait costs it
      // about 90 cycles and every dependent instruction four or five, against 64 for a product.
      constexpr uint32_t kTile16 = kTileBytes >> 4;
      const uint32_t ring16 = (uint32_t)p.slots * kTile16;
      uint32_t at = 0, full = 0, full_par = 0;
      auto take = [&]() {
        const uint32_t here = at;
        at += kTile16;
        if (at == ring16) at = 0;
        return here;
      };
      auto loaded = [&]() {
        const bool there = wait_softly(bar(B_FULL + full), full_par, abort_flag);
        if (++full == kSteps) { full = 0; full_par ^= 1u; }
        return there;
      };
      auto qk = [&](int e, int buf, uint32_t k_at) {
        const uint64_t ad = qdesc0 + (twin ? 0u : (uint32_t)e * (kQBytes >> 4)), bd = kdesc0 + k_at;
        const uint32_t to = tmem + (e * kBufs + buf) * kKeys;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int ks = 0; ks < 4; ++ks)
            mma_ss(to, ad + b * (kQBlk >> 4) + 2 * ks, bd + b * (kBlk >> 4) + 2 * ks, idesc_qk, b + ks > 0 ? 1u : 0u);
        mma_commit(bar(B_S + e * kBufs + buf));
      };
      auto pv = [&](int e, int buf, uint32_t v_at, bool first) {
        const uint32_t from = tmem + (e * kBufs + buf) * kKeys;
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)              // 16 keys: next 16 rows of V, next 8 columns of packed P
          mma_ts(tmem + kOCol + e * DP, from + (kk / (kEach / 16)) * kEach + (kk % (kEach / 16)) * 8, vdesc0 + v_at + kk * 128,
                 idesc_pv, first && kk == 0 ? 0u : 1u);
      };
      bool ok = wait_softly(bar(B_Q), 0, abort_flag);
      for (int c = 0; c < min(ahead, n) && ok; ++c) {
        ok = loaded();
        if (!ok) break;
        tc_fence_after();
        const uint32_t k_at = take();
        if (twin) {
          qk(c & 1, (c >> 1) & (kBufs - 1), k_at);
        } else {
          qk(0, c & (kBufs - 1), k_at);
          qk(1, c & (kBufs - 1), k_at);
        }
      }
      full = ahead;                                          // the step of chunk 0, also where there were fewer chunks
      uint32_t buf = 0, p_par = 0;
      for (int s = 0; s < n && ok; ++s) {
        ok = loaded();
        if (!ok) break;
        const bool more = s + ahead < n;
        const uint32_t v_at = take(), k_at = more ? take() : 0u;
        const int e0 = twin ? s & 1 : 0, e1 = twin ? s & 1 : 1;        // the chunk's stream, or both
#pragma unroll 1
        for (int e = e0; e <= e1; ++e) {
          ok = wait_softly(bar(B_P + e * kBufs + buf), p_par, abort_flag);
          if (!ok) break;
          tc_fence_after();
          pv(e, buf, v_at, twin ? s < 2 : s == 0);
          if (more) qk(e, buf, k_at);                        // executes after P V, which has read P from the same columns
          else mma_commit(bar(B_PV + e * kBufs + buf));      // no Q K^T follows to tell that this P V is done
        }
        if (!twin || (s & 1)) {                              // next chunk of the stream: other buffer, or next phase
          if (kBufs == 1 || buf == 1) p_par ^= 1u;
          buf = kBufs == 1 ? 0u : buf ^ 1u;
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------ softmax and epilogue
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_base = tmem + lanes + stream * kBufs * kKeys + keys * kEach, o_addr = tmem + lanes + kOCol + stream * DP;
    const int mine = twin ? (n - stream + 1) / 2 : n;        // chunks of this stream
    const int pair_bar = 1 + stream * 4 + (warp & 3);        // named barrier of the two warps that share 32 rows
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    const bool tells = (twin || stream == 1) && keys == 0 && (warp & 3) == 0 && lane == 0;
    int left = limit - (c0 + (twin ? stream : 0)) * kKeys - keys * kEach;       // keys of this half that the row sees
    uint32_t buf = 0, par = 0;
    for (int j = 0; j < mine; ++j, left -= twin ? 2 * kKeys : kKeys) {
      ok = __all_sync(0xffffffffu, wait_softly(bar(B_S + stream * kBufs + buf), par, abort_flag));
      // the chunk's keys have been used, and with them the step that held them
      if (tells) mbar_arrive(bar(B_EMPTY + ((twin ? 2 * j + stream : j) & (kSteps - 1))));
      if (!ok) {
        // the warp beside may have passed and wait there
        if (kSplit == 2) asm volatile("bar.arrive %0, 64;" ::"r"(pair_bar) : "memory");
        break;
      }
      tc_fence_after();
      const uint32_t s_addr = s_base + buf * kKeys;
      uint32_t s[kEach];
#pragma unroll
      for (int g = 0; g < kEach / 32; ++g) tmem_ld32(s_addr + g * 32, s + g * 32);
      if constexpr (kEach % 32 != 0) tmem_ld16(s_addr + kEach - 16, *reinterpret_cast<uint32_t(*)[16]>(s + kEach - 16));
      tmem_wait_ld();
      if (__any_sync(0xffffffffu, alive && left < kEach)) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) s[i] = i < left ? s[i] : 0xff800000u;
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < kEach / 2; ++i) mx[i & 3] = max3(mx[i & 3], __uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
      const float own = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
      float mc = own * p.scale_log2;
      if constexpr (kSplit == 2) {
        // the other warp has read what stood here: it has handed over P since, or met this warp at the barrier once more
        sh.peak[buf][stream][keys][r] = own;
        asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
        mc = max3(own, sh.peak[buf][stream][keys ^ 1][r], own) * p.scale_log2;
      }
      // a NaN counts as too far ahead, and ends in the row's result
      const bool first = m == -INFINITY, bump = alive && !first && !(mc <= m + kLazy);
      if (__any_sync(0xffffffffu, bump)) {
        // O has to be complete up to the chunk before.  With one buffer it is, as S of this chunk was issued after that
        // P V; with two it is when S of the next chunk is there, or, at the end, when the P V says so itself.
        if (kBufs == 2) {
          const uint32_t other = stream * kBufs + (buf ^ 1u);          // of the chunk before and the next one
          ok = j + 1 < mine ? mbar_wait(bar(B_S + other), buf == 1 ? par ^ 1u : par, abort_flag)
                            : mbar_wait(bar(B_PV + other), 0, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_after();
        }
        const float alpha = bump ? ex2(m - mc) : 1.f;
#pragma unroll 1
        for (int g = 0; ok && g < DP / 16 / kSplit; ++g) {       // each of the row's threads scales half of O
          uint32_t f[16];
          tmem_ld16(o_addr + keys * (DP / 2) + g * 16, f);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) f[i] = __float_as_uint(__uint_as_float(f[i]) * alpha);
          tmem_st16(o_addr + keys * (DP / 2) + g * 16, f);
        }
        l *= alpha;
        if (bump) m = mc;
      }
      if (first) m = mc;
      const float base = m == -INFINITY ? 0.f : m;
      const f32x2 scale2 = pair(p.scale_log2, p.scale_log2), shift = pair(-base, -base);
      f32x2 sum = pair(0.f, 0.f);
      uint32_t pk[kEach / 2];
#pragma unroll
      for (int i = 0; i < kEach / 2; ++i) {
        const f32x2 x = fma2(pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale2, shift);
        float e0, e1;
        unpair(x, e0, e1);
        e0 = ex2(e0);
        e1 = ex2(e1);
        sum = add2(sum, pair(e0, e1));
        pk[i] = pack_pair<BF16>(e0, e1);
        if (i % 16 == 15) tmem_st16(s_addr + (i - 15), *reinterpret_cast<uint32_t(*)[16]>(pk + (i - 15)));
        if (i % 16 == 7 && i + 1 == kEach / 2) tmem_st8(s_addr + (i - 7), *reinterpret_cast<uint32_t(*)[8]>(pk + (i - 7)));
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_P + stream * kBufs + buf));
      if (kBufs == 1 || buf == 1) par ^= 1u;
      buf = kBufs == 1 ? 0u : buf ^ 1u;
      float s0, s1;
      unpair(sum, s0, s1);
      l += s0 + s1;
    }
    if (!(m < INFINITY)) l = __int_as_float(0x7fffffff);     // a NaN or an infinity among the logits
    // the last P V of both streams: nothing reads Q any more, and a twin's O is in two places
    for (int e = 0; e < 2; ++e) {
      const int of = twin ? (n - e + 1) / 2 : n;
      if (of > 0) ok = mbar_wait(bar(B_PV + e * kBufs + (of - 1) % kBufs), 0, abort_flag) && ok;
    }
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    res.sums[stream][keys][r] = l;
    if (keys == 0) res.refs[stream][r] = m;
    asm volatile("bar.sync 9, %0;" ::"n"(Sh::kSoftmax) : "memory");
    // the row's result: of its stream, or of both streams joined
    const int st0 = twin ? 0 : stream;
    float f0 = 1.f, f1 = 0.f;
    l = res.sums[st0][0][r] + (kSplit == 2 ? res.sums[st0][1][r] : 0.f);
    m = res.refs[st0][r];
    if (twin && n > 1) {
      const float m1 = res.refs[1][r], l1 = res.sums[1][0][r] + (kSplit == 2 ? res.sums[1][1][r] : 0.f);
      const float top = fmaxf(m, m1), base = top == -INFINITY ? 0.f : top;
      f0 = ex2(m - base);
      f1 = ex2(m1 - base);
      l = (f0 != 0.f ? l * f0 : 0.f) + (f1 != 0.f ? l1 * f1 : 0.f);
      m = top;
    }
    if (ok) {
      typedef typename std::conditional<BF16, __nv_bfloat16, __half>::type T;
      const long long at = token * a.Hq + head;
      // a part's row in the buffers that the parts are joined from
      const long long prow = ((long long)split * p.cut + (item - p.whole)) * (2 * kRows) + (twin ? 0 : stream * kRows) + r;
      float lse = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
      float wa = 1.f, wb = 0.f;
      const bool win = whole && a.window_lse != nullptr;
      if (win && alive) lse = join_weights(lse, a.window_lse[at], wa, wb);
      const float co = l == 0.f ? 0.f : wa / l;              // a NaN sum stays one
      const float co0 = f0 != 0.f ? co * f0 : 0.f, co1 = f1 != 0.f ? co * f1 : 0.f;
      const bool o_none = !(co0 != 0.f) || n == 0, both = twin && n > 1;      // O of a row without keys may hold anything
      // this thread's columns of the row
      const int width = DP / kSplit / (twin ? 2 : 1), first_col = (twin ? stream * kSplit + keys : keys) * width;
      const uint32_t o0 = tmem + lanes + kOCol + st0 * DP;
      float check = 0.f;                                     // becomes NaN with any value that is not finite
#pragma unroll 1
      for (int col = first_col; col < first_col + width; col += 16) {
        uint32_t f[16], f2[16];
        tmem_ld16(o0 + col, f);
        if (both) tmem_ld16(o0 + DP + col, f2);
        tmem_wait_ld();
        if (!alive || col >= a.D) continue;                  // head dims are multiples of 8
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = o_none ? 0.f : __uint_as_float(f[i]) * co0;
        if (both && co1 != 0.f) {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = fmaf(__uint_as_float(f2[i]), co1, v[i]);
        }
        const int cols = min(16, a.D - col);
        if (a.lens != nullptr) {
#pragma unroll
          for (int i = 0; i < 16; ++i) check += i < cols ? v[i] - v[i] : 0.f;
        }
#pragma unroll
        for (int h8 = 0; h8 < 2; ++h8) {
          if (h8 * 8 >= cols) break;
          const float* u = v + h8 * 8;
          const int c = col + h8 * 8;
          if (!whole) {
            // a whole 32-byte sector at once
            store32(a.part_out + prow * a.D + c, u);
            continue;
          }
          float o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = u[i];
          if (win && wb != 0.f) {
            const uint4 raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.window_out) + at * a.D + c));
            const uint32_t rw[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 ow = unpack_pair<BF16>(rw[i]);
              o[2 * i] = fmaf(wb, ow.x, o[2 * i]);
              o[2 * i + 1] = fmaf(wb, ow.y, o[2 * i + 1]);
            }
          }
          uint32_t pk[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) pk[i] = pack_pair<BF16>(o[2 * i], o[2 * i + 1]);
          *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at * a.D + c) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
      }
      if (alive && first_col == 0) {
        if (!whole) a.part_lse[prow] = lse;
        else if (a.lse != nullptr) a.lse[at] = lse;
      }
      // rows whose keys end inside the block's range and that met a non-finite value past their end
      uint32_t again = __ballot_sync(0xffffffffu, a.lens != nullptr && alive && check != 0.f && limit < c1 * kKeys);
      while (again != 0) {
        const int who = __ffs(again) - 1;
        again &= again - 1;
        const long long tok = __shfl_sync(0xffffffffu, token, who), pr = __shfl_sync(0xffffffffu, prow, who);
        const int h = __shfl_sync(0xffffffffu, head, who), lim = __shfl_sync(0xffffffffu, limit, who);
        const float mm = __shfl_sync(0xffffffffu, m, who), cc = __shfl_sync(0xffffffffu, co, who), bb = __shfl_sync(0xffffffffu, wb, who);
        float acc[4];
        row_alone<BF16>(a, tok, h, hk, c0 * kKeys, lim, mm, p.scale_log2, acc);
        const long long row = tok * a.Hq + h;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = i * 32 + lane;
          if (c >= first_col && c < first_col + width && c < a.D) {
            float v = acc[i] * cc;
            if (whole) {
              if (win && bb != 0.f) v = fmaf(bb, to_f<T>(static_cast<const T*>(a.window_out)[row * a.D + c]), v);
              static_cast<T*>(a.out)[row * a.D + c] = from_f<T>(v);
            } else {
              a.part_out[pr * a.D + c] = v;
            }
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kWarps + 1) {
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
  const size_t smem = (size_t)DP * 2 * (p.q_tiles * kRows + p.slots * Shape<DP>::kKeys) + sizeof(Shared<Shape<DP>::kBufs>);
  const cudaError_t e = cudaFuncSetAttribute(prefix_sm100<DP, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return set_error(NATTEN_B200_ELAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  }
  const long long grid = p.whole + (long long)p.cut * p.a.splits;
  NB_LAUNCH("prefix_sm100", s, prefix_sm100<DP, BF16><<<(unsigned)grid, Shape<DP>::kThreads, smem, s>>>(p, maps));
  return check_launch("prefix attention (tensor cores)");
}

int chunk_keys(const PrefixArgs& a) { return a.D <= 64 ? Shape<64>::kKeys : Shape<128>::kKeys; }
int chunks_of(const PrefixArgs& a) { return (a.prefix + chunk_keys(a) - 1) / chunk_keys(a); }

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

// How the work items are spread over the SMs.  They run in waves of one block per slot; of the items that do not fill the
// last wave, or of all when there are few, each is cut into parts, whose results a second kernel joins.  In units of a
// chunk's time a block costs its chunks and about four to start and finish, the joining about three.
void prefix_sm100_plan(PrefixArgs* a) {
  const long long slots = kSMs;
  const long long items = (row_tiles(*a) + 1) / 2 * a->Hkv, chunks = chunks_of(*a), waves = items / slots;
  double best = 1e300;
  for (long long back = 0; back <= 1 && back <= waves; ++back) {
    const long long whole = (waves - back) * slots, rest = items - whole;
    for (long long n = 1; n <= chunks && n <= 256 && (n == 1 || rest * n <= 2 * slots); ++n) {
      const double cost = (double)(waves - back) * (double)(chunks + 4) + (double)((rest * n + slots - 1) / slots) * (double)((chunks + n - 1) / n + 4) +
                          (n > 1 && rest > 0 ? 3.0 : 0.0);
      if (cost < best) {
        best = cost;
        a->splits = rest > 0 ? (int)n : 1;
        a->cut = n > 1 ? rest : 0;
      }
    }
  }
}

int run_prefix_sm100(const PrefixArgs& a, int dtype, cudaStream_t s) {
  PrefixTc p{};
  p.a = a;
  p.tile_tokens = kRows / a.G;
  p.tiles = row_tiles(a);
  p.pairs = (int)((p.tiles + 1) / 2);
  p.chunks = chunks_of(a);
  p.cut = (int)a.cut;
  p.whole = p.pairs * a.Hkv - p.cut;
  p.q_tiles = p.tiles > 1 ? 2 : 1;
  p.slots = a.D <= 64 ? 14 : 7 - p.q_tiles;   // what fits beside Q
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.status = sm100_status_word();
  if (p.status == nullptr) return set_error(NATTEN_B200_ENODEVICE, "tensor-core kernels need an sm_100 device");
  PrefixMaps maps;
  if (int rc = encode_rows(&maps.q, a.q, dtype, a.D, a.Hq, a.tokens, a.q_head, a.q_token, a.G, p.tile_tokens)) return rc;
  if (int rc = encode_rows(&maps.k, a.k, dtype, a.D, a.Hkv, a.prefix, a.k_head, a.k_token, 1, chunk_keys(a))) return rc;
  if (int rc = encode_rows(&maps.v, a.v, dtype, a.D, a.Hkv, a.prefix, a.v_head, a.v_token, 1, chunk_keys(a))) return rc;
  const bool bf = dtype == NATTEN_B200_BF16;
  if (a.D <= 64) return bf ? launch<64, true>(p, maps, s) : launch<64, false>(p, maps, s);
  return bf ? launch<128, true>(p, maps, s) : launch<128, false>(p, maps, s);
}

}  // namespace nb
