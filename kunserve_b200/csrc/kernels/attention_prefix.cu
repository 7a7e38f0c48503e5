// Tile kernel of cached attention (attention_cached.cu): units of up to 128
// query rows, the queries of many requests behind one shared prefix (or a
// long chunk of one request), on the sm_100a tensor cores.
//
// One CTA takes one (unit, KV head): its rows against blocks of 64 keys,
// S = Q K^T and O += P V by tcgen05.mma with S, P and O in TMEM.
//
//   warps 0-3  softmax: thread r holds row r (TMEM lane r), a block's 64
//              scores in registers; P goes back to TMEM as 16-bit pairs over
//              the scores it came from, from where O += P V reads it
//   warp 4     TMA producer: K and V blocks, one box per page and 64-dim half
//   warp 5     MMA issuer and TMEM owner; QK(i + 1) is issued before PV(i),
//              so a block's scores are ready when the previous block's
//              probabilities are written
//
// Two S buffers; QK(i + 2) waits for PV(i), which reads its P from the same
// columns.  O is rescaled only when a row's max grew by more than 2^8 (the
// sum and O share the stale max).
// Two CTAs an SM (about 100 KB of shared memory, 256 TMEM columns each): one
// CTA's softmax runs beside the other's products.
//
// The keys a unit covers end inside a page or a block: boxes past the end
// are not loaded, the tail rows of V are zeroed (a stale NaN times a zero
// probability would be NaN), scores past a row's limit are set to -inf.
// All mbarrier waits are bounded (common.cuh).
#include "../common.cuh"
#include "cache_elem.cuh"
#include "cache_ops.h"
#include <cudaTypedefs.h>

namespace kus {
namespace gemm_impl {
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();
}
namespace cpt {

constexpr int kRows = kTileUnitRows;
constexpr int kKeys = 64;
constexpr int kThreads = 192;
constexpr uint32_t kCols = 256;          // S0 [0, 64), S1 [64, 128), O [128, 128 + HD)
constexpr uint32_t kColO = 128;
constexpr float kRescaleLog2 = 8.0f;

template <int HD>
struct Cfg {
  static constexpr int kHalves = HD / 64;
  static constexpr int kQHalf = kRows * 128;            // 64 dims of Q (16 KB)
  static constexpr int kHalf = kKeys * 128;             // 64 dims of a K or V block (8 KB)
  static constexpr int kTile = kHalves * kHalf;
  static constexpr int kStages = HD == 128 ? 2 : 4;
  static constexpr int kKOff = kHalves * kQHalf;
  static constexpr int kVOff = kKOff + kStages * kTile;
  static constexpr int kBarOff = kVOff + kStages * kTile;
  static constexpr int kSmem = kBarOff + 256 + 1024;    // at least a third of an SM: TMEM holds two CTAs
  static_assert(kSmem > 76 * 1024 && kSmem <= 113 * 1024, "two CTAs an SM");
};

template <int HD>
struct Bars {
  uint64_t q_full;
  uint64_t k_full[Cfg<HD>::kStages], k_empty[Cfg<HD>::kStages];
  uint64_t v_full[Cfg<HD>::kStages], v_empty[Cfg<HD>::kStages];
  uint64_t s_full[2];
  uint64_t p_full, pv_done;
  uint32_t tmem;
};

KUS_DEVICE void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// 32 lanes x 32 columns, not waited for.
KUS_DEVICE void tmem_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
KUS_DEVICE void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
KUS_DEVICE void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
KUS_DEVICE void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 2) tile_kernel(const __grid_constant__ CUtensorMap map, CachedAttn a,
                                                           int box, float scale_log2) {
  using Cf = Cfg<HD>;
  constexpr int kStages = Cf::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  Bars<HD>* bars = reinterpret_cast<Bars<HD>*>(smem + Cf::kBarOff);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int kvh = a.g.kvh, G = a.nq / kvh;
  // heads vary fastest: the CTAs of one unit read the same cache rows together
  const int unit = blockIdx.x / kvh, kh = blockIdx.x - unit * kvh;
  const int4 u0 = __ldg(reinterpret_cast<const int4*>(a.tile_units) + 2 * unit);
  const int4 u1 = __ldg(reinterpret_cast<const int4*>(a.tile_units) + 2 * unit + 1);
  const int tok0 = u0.x, ntok = u0.y & 255, ng = (u0.y >> 8) & 255, g0 = u0.y >> 16;
  const int key_lo = u0.z, key_hi = u0.w, lim0 = u1.x;
  const int rows = ntok * ng;
  const int nb = (key_hi - key_lo + kKeys - 1) / kKeys;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, kRows);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->k_empty[s], 1);
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->v_empty[s], 1);
    }
    mbar_init(&bars->s_full[0], 1);
    mbar_init(&bars->s_full[1], 1);
    mbar_init(&bars->p_full, kRows);
    mbar_init(&bars->pv_done, 1);
    fence_barrier_init();
  }
  if (warp == 5) tmem_alloc(&bars->tmem, kCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  pdl_wait();
  pdl_trigger();

  if (warp == 4) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      prefetch_tmap(&map);
      const int* table = a.pages + u1.y;
      const int per_slot = 2 * a.g.block_size;   // K rows, then V rows of one (page, layer)
      bool ok = true;
      for (int i = 0; i < nb && ok; ++i) {
        const int s = i % kStages;
        const uint32_t ph = (uint32_t)(i / kStages) & 1u;
        const int key0 = key_lo + i * kKeys;
        const int boxes = (min(kKeys, key_hi - key0) + box - 1) / box;
        const uint32_t bytes = (uint32_t)boxes * box * HD * 2;
        ok = mbar_wait(&bars->k_empty[s], ph ^ 1u, kErrWaitEmpty);
        if (!ok) break;
        mbar_arrive_expect_tx(&bars->k_full[s], bytes);
        const uint32_t kd = sbase + Cf::kKOff + s * Cf::kTile, vd = sbase + Cf::kVOff + s * Cf::kTile;
        auto row_of = [&](int j) {
          const int key = key0 + j * box;
          return kv_slot(a.g, __ldg(table + kv_page_col(a.g, key)), a.layer) * per_slot + kv_page_slot(a.g, key);
        };
        for (int j = 0; j < boxes; ++j) {
          const int row = row_of(j);
#pragma unroll
          for (int h = 0; h < Cf::kHalves; ++h)
            tma_load_3d(kd + h * Cf::kHalf + j * box * 128, &map, &bars->k_full[s], 64 * h, kh, row);
        }
        ok = mbar_wait(&bars->v_empty[s], ph ^ 1u, kErrWaitEmpty);
        if (!ok) break;
        mbar_arrive_expect_tx(&bars->v_full[s], bytes);
        for (int j = 0; j < boxes; ++j) {
          const int row = row_of(j) + a.g.block_size;
#pragma unroll
          for (int h = 0; h < Cf::kHalves; ++h)
            tma_load_3d(vd + h * Cf::kHalf + j * box * 128, &map, &bars->v_full[s], 64 * h, kh, row);
        }
      }
      // every load has landed before the CTA may leave
      for (int i = max(0, nb - kStages); i < nb; ++i) {
        mbar_wait(&bars->k_full[i % kStages], (uint32_t)(i / kStages) & 1u, kErrWaitFull);
        mbar_wait(&bars->v_full[i % kStages], (uint32_t)(i / kStages) & 1u, kErrWaitFull);
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    // ---------------------------------------------------------- MMA issuer
    constexpr uint32_t id_qk = idesc<T>(kKeys, false), id_pv = idesc<T>(HD, true);
    bool ok = __all_sync(0xffffffffu, mbar_wait(&bars->q_full, 0, kErrWaitFull));
    auto qk = [&](int i) {
      const int s = i % kStages;
      // PV(i - 2) has read its probabilities from the columns S(i) goes to
      if (i >= 2) ok = ok && mbar_wait(&bars->pv_done, (uint32_t)i & 1u, kErrWaitTmemEmpty);
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->k_full[s], (uint32_t)(i / kStages) & 1u, kErrWaitFull));
      tc_fence_after();
      if (ok && lane == 0) {
        const uint32_t qb = sbase, kb = sbase + Cf::kKOff + s * Cf::kTile;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          umma_f16(tmem + (i & 1) * kKeys, umma_desc_sw128(qb + (kk >> 2) * Cf::kQHalf) + (uint64_t)(2 * (kk & 3)),
                   umma_desc_sw128(kb + (kk >> 2) * Cf::kHalf) + (uint64_t)(2 * (kk & 3)), id_qk, kk > 0 ? 1u : 0u);
        umma_commit(&bars->s_full[i & 1]);
        umma_commit(&bars->k_empty[s]);
      }
      __syncwarp();
    };
    if (ok) qk(0);
    for (int i = 0; i < nb && ok; ++i) {
      if (i + 1 < nb) qk(i + 1);
      const int s = i % kStages;
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->v_full[s], (uint32_t)(i / kStages) & 1u, kErrWaitFull));
      const int have = key_hi - (key_lo + i * kKeys);
      if (ok && have < kKeys) {
        // rows past the keys: the loaded boxes' stale slots and what was not loaded
        uint8_t* vt = smem + Cf::kVOff + s * Cf::kTile;
        for (int c = lane; c < (kKeys - have) * 8; c += 32)
#pragma unroll
          for (int h = 0; h < Cf::kHalves; ++h)
            *reinterpret_cast<uint4*>(vt + h * Cf::kHalf + have * 128 + c * 16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
      }
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->p_full, (uint32_t)i & 1u, kErrWaitFull));
      tc_fence_after();
      if (ok && lane == 0) {
        const uint32_t vb = sbase + Cf::kVOff + s * Cf::kTile;
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          umma_f16_ta(tmem + kColO, tmem + (i & 1) * kKeys + kk * 8, v_desc(vb + kk * 16 * 128, Cf::kHalf), id_pv,
                      (i > 0 || kk > 0) ? 1u : 0u);
        umma_commit(&bars->pv_done);
        umma_commit(&bars->v_empty[s]);
      }
      __syncwarp();
    }
  } else {
    // --------------------------------------------------- Q, softmax, output
    const int r = threadIdx.x;
    const bool valid = r < rows;
    const int j = valid ? r / ng : 0, gi = valid ? r - j * ng : 0;
    {
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.q) + (tok0 + j) * a.qt +
                                                        (long long)(kh * G + g0 + gi) * a.qh);
#pragma unroll
      for (int h = 0; h < Cf::kHalves; ++h)
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint4 v = valid ? __ldg(src + h * 8 + c) : make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(smem + h * Cf::kQHalf + r * 128 + ((c ^ (r & 7)) << 4)) = v;
        }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&bars->q_full);
    }
    const int end = min(key_hi, lim0 + j);       // keys this row sees
    const int end_min = min(key_hi, lim0);       // and every row sees
    const uint32_t tl = tmem + ((uint32_t)(warp * 32) << 16);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; i < nb; ++i) {
      ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->s_full[i & 1], (uint32_t)(i >> 1) & 1u, kErrWaitTmemFull));
      tc_fence_after();
      const uint32_t ts = tl + (i & 1) * kKeys;
      uint32_t sv[64];
      tmem_ld32(ts, sv);
      tmem_ld32(ts + 32, sv + 32);
      tmem_wait_ld();
      const int key0 = key_lo + i * kKeys;
      if (key0 + kKeys > end_min) {
#pragma unroll
        for (int e = 0; e < 64; ++e)
          if (key0 + e >= end) sv[e] = 0xff800000u;   // -inf
      }
      float mx[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) mx[e] = __uint_as_float(sv[e]);
#pragma unroll
      for (int e = 4; e < 64; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(sv[e]));
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale_log2;
      const bool grow = top > m + kRescaleLog2;
      const float mn = grow ? top : m;
      const float alpha = grow ? ex2(m - mn) : 1.f;
      const float ref = mn == -INFINITY ? 0.f : mn;   // no key seen yet
      uint32_t pk[32];
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 64; e += 2) {
        const float p0 = ex2(fmaf(__uint_as_float(sv[e]), scale_log2, -ref));
        const float p1 = ex2(fmaf(__uint_as_float(sv[e + 1]), scale_log2, -ref));
        sum[0] += p0;
        sum[1] += p1;
        pk[e / 2] = pack2<T>(p0, p1);
      }
      tmem_st32(ts, pk);
      if (i > 0) {
        // PV(i - 1) is done: O is stable
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->pv_done, (uint32_t)(i - 1) & 1u, kErrWaitTmemFull));
        tc_fence_after();
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(tl + kColO + 32 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(tl + kColO + 32 * c, o);
          }
        }
      }
      tmem_wait_st();
      l = l * alpha + sum[0] + sum[1];
      m = mn;
      tc_fence_before();
      mbar_arrive(&bars->p_full);
    }
    ok = __all_sync(0xffffffffu, ok && mbar_wait(&bars->pv_done, (uint32_t)(nb - 1) & 1u, kErrWaitTmemFull));
    tc_fence_after();
    const long long prow = u1.z + (long long)kh * rows + r;
    float* dst = a.part_o + prow * HD;
#pragma unroll 1
    for (int c = 0; c < HD / 32; ++c) {
      uint32_t o[32];
      tmem_ld32(tl + kColO + 32 * c, o);
      tmem_wait_ld();
      if (valid)
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *reinterpret_cast<uint4*>(dst + 32 * c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
    }
    if (valid) a.part_ml[prow] = make_float2(m, l);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) tmem_dealloc(tmem, kCols);
}

template <typename T, int HD>
void launch(const CachedAttn& a, const CUtensorMap& map, int box, cudaStream_t s) {
  ensure_smem_attr(reinterpret_cast<const void*>(tile_kernel<T, HD>), Cfg<HD>::kSmem);
  launch_k(tile_kernel<T, HD>, dim3((unsigned)a.n_tile_units * a.g.kvh), dim3(kThreads), Cfg<HD>::kSmem, s, map, a, box,
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
