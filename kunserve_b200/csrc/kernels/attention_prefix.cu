// Tile kernel of cached attention (attention_cached.cu): units of up to 128
// query rows, the queries of many requests behind one shared prefix (or a
// long chunk of one request), on the sm_100a tensor cores.
//
// A CTA takes (unit, KV head) pairs in turn: the unit's rows against blocks
// of 128 keys, S = Q K^T and O += P V by tcgen05.mma with S, P and O in TMEM.
//
//   warps 0-7  softmax: two threads a row (TMEM lane r), 64 of the block's
//              scores each in registers; the probabilities go as 16-bit
//              pairs to TMEM, from where O += P V reads them
//   warps 8, 9 TMA producers of K and of V: one box per page and 64-dim half,
//              a lane per box, its page looked up a block ahead
//   warp 10    issues QK (and owns TMEM), warp 11 issues PV: a thread that issues
//              one product waits for most of it, which would hold the other up
//
// The grid is persistent and every role counts blocks over the CTA's units,
// so the loads of a unit's first blocks run beside the end of the one before.
// S and P have two buffers each (with O all 512 TMEM columns, one CTA an SM):
// QK(i + 1) and PV(i - 1) run while block i's softmax does, which is what
// bounds an iteration.  Blocks of 128 keys and not 64: the tensor core reads
// Q from shared memory once per block, which at N = 64 takes longer than the
// products.  Probabilities are taken against a row's reference, at most a
// range above which they are taken again and O rescaled (the sum and O share
// the reference, whatever it is): struct Range.
//
// A block of 128 rows and keys takes about 1950 clk: 1024 of exponentials (16
// a clk), the rest waits around them; the products take 1400 beside that.
// 128 requests, 8 rows each per KV head, behind four prefixes of 16384: 73-85
// us for 70 GFLOP and 268 MB.
//
// P is rounded once to the element type on its way to O += P V; sums, maxima
// and O are fp32.  Its remainder would take a second product with V: some 2100
// clk of products a block, above what bounds it now.  Outputs are so off by 0.0023 (bf16) and 0.00029 (fp16) of
// their norm against 64 bits, where their own rounding makes 0.0017 and
// 0.00021, which is all that the row kernel is off by.
//
// The keys a unit covers end inside a page or a block: boxes past the end
// are not loaded, the tail rows of V are zeroed (a stale NaN times a zero
// probability would be NaN), scores past a row's limit are set to -inf.
// All mbarrier waits are bounded (common.cuh).
#include "../common.cuh"
#include "cache_elem.cuh"
#include "cache_ops.h"
#include <cudaTypedefs.h>
#include <algorithm>

namespace kus {
namespace gemm_impl {
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();
}
namespace cpt {

constexpr int kRows = kTileUnitRows;
constexpr int kKeys = kTileKeys;
constexpr int kSoftmax = 256;            // softmax threads: two a row
constexpr int kThreads = kSoftmax + 128;
constexpr uint32_t kCols = 512;          // S0, S1 [0, 256), P0, P1 [256, 384), O [384, 384 + HD)
constexpr uint32_t kColP = 256;
constexpr uint32_t kColO = 384;

// Probabilities P = 2^(s - m) of 16 bits, by element type: m is set kUp below
// a row's max, and again once a P would exceed 2^kMost.  bf16 has fp32's
// exponents: m is the max, and P up to 2^8 leaves it be.  fp16's end at
// 2^-24: P of up to 2^15 let a weight of 2^-36 of the row's largest still
// count (many light keys hold what a long context's output shows), and a max
// may grow 2^4 times before m follows.
template <typename T>
struct Range {
  static constexpr float kUp = 0.f, kMost = 8.f;
};
template <>
struct Range<__half> {
  static constexpr float kUp = 11.f, kMost = 15.f;
};

template <int HD>
struct Cfg {
  static constexpr int kHalves = HD / 64;
  static constexpr int kQHalf = kRows * 128;            // 64 dims of Q (16 KB)
  static constexpr int kHalf = kKeys * 128;             // 64 dims of a K or V block (16 KB)
  static constexpr int kTile = kHalves * kHalf;
  static constexpr int kKStages = HD == 128 ? 3 : 5, kVStages = HD == 128 ? 2 : 4;
  static constexpr int kKOff = kHalves * kQHalf;
  static constexpr int kVOff = kKOff + kKStages * kTile;
  static constexpr int kBarOff = kVOff + kVStages * kTile;
  static constexpr int kMaxOff = kBarOff + 256;         // fp32 [2 halves][rows]
  static constexpr int kSmem = kMaxOff + 2 * kRows * 4 + 1024;
  static_assert(kSmem > 114 * 1024 && kSmem <= 200 * 1024, "one CTA an SM, and room for a warp of the row kernel");
};

template <int HD>
struct Bars {
  uint64_t q_full;
  uint64_t k_full[Cfg<HD>::kKStages], k_empty[Cfg<HD>::kKStages];
  uint64_t v_full[Cfg<HD>::kVStages], v_empty[Cfg<HD>::kVStages];
  uint64_t s_full[2], s_empty[2], p_full[2], pv_done[2];
  uint64_t drained[2];   // all products of the issuers of QK, PV
  uint32_t tmem;
};
static_assert(sizeof(Bars<64>) <= 256 && sizeof(Bars<128>) <= 256, "they lie before the maxima");

KUS_DEVICE void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// 32 lanes x 16 columns.  Loads are not waited for; tmem_wait_ld waits for
// all of this thread's, and r, loaded before, cannot be used above it.
constexpr int kChunk = 16;
KUS_DEVICE void tmem_ld(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
KUS_DEVICE void tmem_wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
KUS_DEVICE void tmem_st(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
KUS_DEVICE void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Two fp32 lanes in one instruction, and the largest of three.
KUS_DEVICE float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)),
        "l"(reinterpret_cast<const unsigned long long&>(c)));
  return reinterpret_cast<float2&>(d);
}
KUS_DEVICE float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(d)
      : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
  return reinterpret_cast<float2&>(d);
}
KUS_DEVICE float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Whether `pred` holds in any of the `n` threads of named barrier `id`.
KUS_DEVICE bool barrier_any(int id, int n, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.u32 p, %3, 0;\nbarrier.cta.red.or.pred q, %1, %2, p;\nselp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"(id), "r"(n), "r"((uint32_t)pred)
      : "memory");
  return r != 0;
}

// D(tmem) (+)= A(tmem) * B(smem desc): A's rows are TMEM lanes, a column
// holds two 16-bit elements.
KUS_DEVICE void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Descriptor of V as MN-major operand: 64 dims (128 B) a row, keys 128 B
// apart, groups of 8 keys 1024 B, the next 64 dims `half` bytes on.
KUS_DEVICE uint64_t v_desc(uint32_t addr, uint32_t half) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)((half >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

template <typename T>
KUS_HOST_DEVICE constexpr uint32_t idesc(int N, bool b_mn) {
  const uint32_t f = std::is_same<T, __half>::value ? 0u : 1u;
  return (1u << 4) | (f << 7) | (f << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(kRows >> 4) << 24);
}

// What a unit record says (cache_ops.h), for one KV head.
struct Unit {
  int kh, tok0, ntok, ng, g0, key_lo, key_hi, lim0, page0, part0, nb;
};
KUS_DEVICE Unit unit_at(const CachedAttn& a, int item) {
  // heads vary fastest: CTAs of one unit read the same cache rows together
  const int u = item / a.g.kvh;
  const int4 u0 = __ldg(reinterpret_cast<const int4*>(a.tile_units) + 2 * u);
  const int4 u1 = __ldg(reinterpret_cast<const int4*>(a.tile_units) + 2 * u + 1);
  Unit r;
  r.kh = item - u * a.g.kvh;
  r.tok0 = u0.x;
  r.ntok = u0.y & 255;
  r.ng = (u0.y >> 8) & 255;
  r.g0 = u0.y >> 16;
  r.key_lo = u0.z;
  r.key_hi = u0.w;
  r.lim0 = u1.x;
  r.page0 = u1.y;
  r.part0 = u1.z;
  r.nb = (r.key_hi - r.key_lo + kKeys - 1) / kKeys;
  return r;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) tile_kernel(const __grid_constant__ CUtensorMap map, CachedAttn a,
                                                           int box, float scale_log2) {
  using Cf = Cfg<HD>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  Bars<HD>* bars = reinterpret_cast<Bars<HD>*>(smem + Cf::kBarOff);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int G = a.nq / a.g.kvh, n_items = a.n_tile_units * a.g.kvh;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, kSoftmax);
    for (int s = 0; s < Cf::kKStages; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
    }
    for (int s = 0; s < Cf::kVStages; ++s) {
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->s_full[b], 1);
      mbar_init(&bars->s_empty[b], kSoftmax);
      mbar_init(&bars->p_full[b], kSoftmax);
      mbar_init(&bars->pv_done[b], 1);
      mbar_init(&bars->drained[b], 1);
    }
    fence_barrier_init();
  }
  if (warp == 10) tmem_alloc(&bars->tmem, kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  pdl_wait();
  pdl_trigger();

  if (warp == 8 || warp == 9) {
    // ----------------------------------------------------------- producers
    const bool is_v = warp == 9;
    const int stages = is_v ? Cf::kVStages : Cf::kKStages;
    uint64_t* full = is_v ? bars->v_full : bars->k_full;
    uint64_t* empty = is_v ? bars->v_empty : bars->k_empty;
    const uint32_t region = sbase + (is_v ? Cf::kVOff : Cf::kKOff);
    if (lane == 0) prefetch_tmap(&map);
    int s = 0, loaded = 0;
    uint32_t ph = 1;
    bool ok = true;
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Unit un = unit_at(a, item);
      const int* table = a.pages + un.page0;
      // tensor map row of this lane's box of block i (-1: past the keys)
      auto row_of = [&](int i) {
        const int key = un.key_lo + i * kKeys + lane * box;
        if (lane * box >= kKeys || key >= un.key_hi) return -1;
        return kv_slot(a.g, __ldg(table + kv_page_col(a.g, key)), a.layer) * 2 * a.g.block_size +
               (is_v ? a.g.block_size : 0) + kv_page_slot(a.g, key);
      };
      int row = row_of(0);
      for (int i = 0; i < un.nb; ++i) {
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ph, kErrWaitEmpty));
        if (!ok) break;
        const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, row >= 0));
        if (lane == 0) mbar_arrive_expect_tx(&full[s], boxes * box * HD * 2);
        __syncwarp();
        if (row >= 0) {
          const uint32_t dst = region + s * Cf::kTile + lane * box * 128;
#pragma unroll
          for (int h = 0; h < Cf::kHalves; ++h) tma_load_3d(dst + h * Cf::kHalf, &map, &full[s], 64 * h, un.kh, row);
        }
        row = row_of(i + 1);
        ++loaded;
        if (++s == stages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    // every load has landed before the CTA may leave
    for (int i = max(0, loaded - stages); i < loaded; ++i)
      mbar_wait<true>(&full[i % stages], (uint32_t)(i / stages) & 1u, kErrWaitFull);
    __syncwarp();
  } else if (warp == 10) {
    // ------------------------------------------------------- S = Q K^T
    if (lane == 0) {
      constexpr uint32_t id_qk = idesc<T>(kKeys, false);
      bool ok = true;
      int s = 0, g = 0;   // stage, blocks so far
      uint32_t ph = 0, q_ph = 0;
      for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x, q_ph ^= 1) {
        const int nb = unit_at(a, item).nb;
        ok = mbar_wait(&bars->q_full, q_ph, kErrWaitFull);
        for (int i = 0; i < nb && ok; ++i, ++g) {
          const int b = g & 1;
          ok = mbar_wait(&bars->k_full[s], ph, kErrWaitFull);
          // the scores of block g - 2 are read, and its probabilities: S(g)
          // full tells the softmax that both buffers are free
          const uint32_t before = (uint32_t)((g >> 1) - 1) & 1u;
          if (g >= 2)
            ok = ok && mbar_wait(&bars->s_empty[b], before, kErrWaitTmemEmpty) &&
                 mbar_wait(&bars->pv_done[b], before, kErrWaitTmemEmpty);
          if (!ok) break;
          tc_fence_after();
          const uint64_t qd = umma_desc_sw128(sbase), kd = umma_desc_sw128(sbase + Cf::kKOff + s * Cf::kTile);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            umma_f16(tmem + b * kKeys, qd + (uint64_t)(((kk >> 2) * Cf::kQHalf >> 4) + 2 * (kk & 3)),
                     kd + (uint64_t)(((kk >> 2) * Cf::kHalf >> 4) + 2 * (kk & 3)), id_qk, kk > 0 ? 1u : 0u);
          umma_commit(&bars->s_full[b]);
          umma_commit(&bars->k_empty[s]);
          if (++s == Cf::kKStages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      // shared memory and TMEM stay until every product is done, whatever
      // wait ran out (here or in the softmax)
      umma_commit(&bars->drained[0]);
      mbar_wait<true>(&bars->drained[0], 0, kErrWaitTmemFull);
    }
    __syncwarp();
  } else if (warp == 11) {
    // ------------------------------------------------------- O += P V
    constexpr uint32_t id_pv = idesc<T>(HD, true);
    bool ok = true;
    int s = 0, g = 0;
    uint32_t ph = 0;
    for (int item = blockIdx.x; item < n_items && ok; item += gridDim.x) {
      const Unit un = unit_at(a, item);
      for (int i = 0; i < un.nb; ++i, ++g) {
        const int b = g & 1;
        ok = mbar_wait(&bars->v_full[s], ph, kErrWaitFull);
        const int have = un.key_hi - (un.key_lo + i * kKeys);
        if (have < kKeys) {
          // rows past the keys: the loaded boxes' stale slots and what was not loaded
          uint8_t* vt = smem + Cf::kVOff + s * Cf::kTile;
          for (int c = lane; c < (kKeys - have) * 8; c += 32)
#pragma unroll
            for (int h = 0; h < Cf::kHalves; ++h)
              *reinterpret_cast<uint4*>(vt + h * Cf::kHalf + have * 128 + c * 16) = make_uint4(0, 0, 0, 0);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->p_full[b], (uint32_t)(g >> 1) & 1u, kErrWaitFull));
        if (!ok) break;
        if (lane == 0) {
          tc_fence_after();
          const uint64_t vd = v_desc(sbase + Cf::kVOff + s * Cf::kTile, Cf::kHalf);
#pragma unroll
          for (int kk = 0; kk < kKeys / 16; ++kk)
            umma_f16_ta(tmem + kColO, tmem + kColP + b * (kKeys / 2) + kk * 8, vd + (uint64_t)(kk * 16 * 128 >> 4),
                        id_pv, (i > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&bars->pv_done[b]);
          umma_commit(&bars->v_empty[s]);
        }
        __syncwarp();
        if (++s == Cf::kVStages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    if (lane == 0) {
      umma_commit(&bars->drained[1]);
      mbar_wait<true>(&bars->drained[1], 0, kErrWaitTmemFull);
    }
    __syncwarp();
  } else {
    // --------------------------------------------------- Q, softmax, output
    const int half = warp >> 2, r = threadIdx.x & (kRows - 1);   // TMEM lane of warp w: 32 (w % 4) + lane
    const uint32_t tl = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_o = tl + kColO + half * (HD / 2);
    float* maxima = reinterpret_cast<float*>(smem + Cf::kMaxOff);
    bool ok = true;
    int g = 0;   // blocks so far
    for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
      const Unit un = unit_at(a, item);
      const int rows = un.ntok * un.ng;
      const bool valid = r < rows;
      const int j = valid ? r / un.ng : 0, gi = valid ? r - j * un.ng : 0;
      {
        // every product with the Q before is done: its last scores were read
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (un.tok0 + j) * a.qt +
                                                          (long long)(un.kh * G + un.g0 + gi) * a.qh);
        constexpr int kEach = HD / 16;   // 16-byte chunks of a thread
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          const int c = half * kEach + e;
          const uint4 v = valid ? src[c] : make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(smem + (c >> 3) * Cf::kQHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&bars->q_full);
      }
      const int end = min(un.key_hi, un.lim0 + j);       // keys this row sees
      const int end_min = min(un.key_hi, un.lim0);       // and every row sees
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < un.nb; ++i, ++g) {
        const int b = g & 1;
        const uint32_t t_s = tl + b * kKeys + half * 64, t_p = tl + kColP + b * (kKeys / 2) + half * 32;
        ok = ok && mbar_wait(&bars->s_full[b], (uint32_t)(g >> 1) & 1u, kErrWaitTmemFull);
        __syncwarp();
        tc_fence_after();
        const int key0 = un.key_lo + i * kKeys;
        uint32_t v[64];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld(t_s + kChunk * c, v + kChunk * c);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_wait_ld(v + kChunk * c);
        tc_fence_before();
        mbar_arrive(&bars->s_empty[b]);
        if (key0 + kKeys > end_min) {
          const int left = end - key0 - half * 64;   // of this thread's keys, those its row sees
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (e >= left) v[e] = 0xff800000u;   // -inf
        }
        // Probabilities against the reference so far, the block's own max beside
        // them: it is only seldom needed, and the exponentials bound this loop.
        uint32_t pk[32];
        float sum;
        float mx[2] = {-INFINITY, -INFINITY};
        auto probabilities = [&](float ref) {
          const float2 scale2 = make_float2(scale_log2, scale_log2), ref2 = make_float2(-ref, -ref);
          float2 acc[2] = {};
#pragma unroll
          for (int e = 0; e < 64; e += 2) {
            const float2 x = fma2(make_float2(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), scale2, ref2);
            const float2 p = make_float2(ex2(x.x), ex2(x.y));
            acc[(e / 2) & 1] = add2(acc[(e / 2) & 1], p);
            pk[e / 2] = pack2<T>(p.x, p.y);
          }
          sum = (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
        };
        probabilities(m == -INFINITY ? 0.f : m);
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          mx[0] = max3(mx[0], __uint_as_float(v[e]), __uint_as_float(v[e + 1]));
          mx[1] = max3(mx[1], __uint_as_float(v[e + 2]), __uint_as_float(v[e + 3]));
        }
        const float top = fmaxf(mx[0], mx[1]) * scale_log2;
        if (barrier_any(1 + (warp & 3), 64, top > m + Range<T>::kMost)) {
          // some row of this pair of warps outgrew its reference
          float* mine = maxima + r;
          mine[half * kRows] = top;
          named_barrier(1 + (warp & 3), 64);
          const float both = fmaxf(top, mine[(half ^ 1) * kRows]);
          const bool grow = both > m + Range<T>::kMost;
          const float mn = grow ? both - Range<T>::kUp : m;
          const float alpha = grow ? ex2(m - mn) : 1.f;
          probabilities(mn == -INFINITY ? 0.f : mn);   // no key seen yet: zeros
          if (i > 0) {
            // PV of the block before is done: O is stable
            ok = ok && mbar_wait(&bars->pv_done[b ^ 1], (uint32_t)((g - 1) >> 1) & 1u, kErrWaitTmemFull);
            __syncwarp();
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 2 / kChunk; ++c) {
              uint32_t o[kChunk];
              tmem_ld(t_o + kChunk * c, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int e = 0; e < kChunk; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st(t_o + kChunk * c, o);
            }
          }
          l *= alpha;
          m = mn;
        }
        tmem_st(t_p, pk);
        tmem_st(t_p + kChunk, pk + kChunk);
        l += sum;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&bars->p_full[b]);
      }
      // the halves' sums (m is the same in both)
      named_barrier(1 + (warp & 3), 64);
      float* mine = maxima + r;
      mine[half * kRows] = l;
      named_barrier(1 + (warp & 3), 64);
      l += mine[(half ^ 1) * kRows];
      ok = ok && mbar_wait(&bars->pv_done[(g - 1) & 1], (uint32_t)((g - 1) >> 1) & 1u, kErrWaitTmemFull);
      __syncwarp();
      tc_fence_after();
      const long long prow = un.part0 + (long long)un.kh * rows + r;
      float* dst = a.part_o + prow * HD + half * (HD / 2);
#pragma unroll
      for (int c = 0; c < HD / 2 / kChunk; ++c) {
        uint32_t o[kChunk];
        tmem_ld(t_o + kChunk * c, o);
        tmem_wait_ld(o);
        if (valid)
#pragma unroll
          for (int e = 0; e < kChunk; e += 4)
            *reinterpret_cast<uint4*>(dst + kChunk * c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      }
      if (valid && half == 0) a.part_ml[prow] = make_float2(m, l);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 10) tmem_dealloc(tmem, kCols);
}

template <typename T, int HD>
void launch(const CachedAttn& a, const CUtensorMap& map, int box, cudaStream_t s) {
  ensure_smem_attr(reinterpret_cast<const void*>(tile_kernel<T, HD>), Cfg<HD>::kSmem);
  int dev = 0, sms = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const unsigned grid = (unsigned)std::min<long long>(sms, (long long)a.n_tile_units * a.g.kvh);
  launch_k(tile_kernel<T, HD>, dim3(grid), dim3(kThreads), Cfg<HD>::kSmem, s, map, a, box,
           a.scale * 1.4426950408889634f);
}

}  // namespace cpt

int cache_tile_box(const KVGeom& g) {
  int box = 64;
  while (g.block_size % box) box /= 2;
  return box;
}

bool make_cache_tile_map(CUtensorMap* map, const KVGeom& g, long long bytes, int type) {
  auto fn = gemm_impl::get_encode_fn();
  const long long row_bytes = 2LL * g.kvh * g.hd, rows = bytes / row_bytes;
  const int box = cache_tile_box(g);
  // boxes below 8 rows would split a swizzle atom
  if (!fn || (g.hd != 64 && g.hd != 128) || box < 8 || rows >= (1LL << 31)) return false;
  cuuint64_t dims[3] = {(cuuint64_t)g.hd, (cuuint64_t)g.kvh, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)g.hd * 2, (cuuint64_t)row_bytes};
  cuuint32_t boxes[3] = {64, 1, (cuuint32_t)box};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, type == kTypeBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, g.base,
            dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

void cached_attention_tiles(const CachedAttn& a, const CUtensorMap& map, int type, cudaStream_t s) {
  const int box = cache_tile_box(a.g);
  if (type == kTypeBF16) {
    a.hd == 128 ? cpt::launch<__nv_bfloat16, 128>(a, map, box, s) : cpt::launch<__nv_bfloat16, 64>(a, map, box, s);
  } else {
    a.hd == 128 ? cpt::launch<__half, 128>(a, map, box, s) : cpt::launch<__half, 64>(a, map, box, s);
  }
}

}  // namespace kus
