// Matrix product of 8-bit tokens with 8-bit weights on tcgen05 (kind::i8):
//   y[t, n] = (sum_k q[t, k] w[n, k]) s[t] v[n] + b[n]
// with exact int32 sums in TMEM, scaled in fp32 and rounded once.
//
// The weights are the MMA's M side whatever the number of tokens, the tokens
// its N side (a tile of 16 to 256): a decode step pads its few tokens to 16
// and no further.  A k-block is 128 bytes of K, 32 a product.  The weights
// lie in blocks of 128 channels x 128 bytes, so that a stage is one
// contiguous read of 16 KB.
//
// What bounds it.  Few tokens: the weights' bytes; 64 x 5120 x 27648 takes
// 24.4 us of the 22.2 that its bytes take at the copy bandwidth.  K is then
// split over the CTAs of a cluster until they fill the GPU, and their parts
// go through distributed shared memory: integers add up in any order, so no
// workspace, counter or second kernel is needed (64 x 5120 x 5120: 7.9 us in
// three parts, 9.0 whole where the next products start on the SMs left idle,
// 14 alone).  Many tokens: the tensor cores, and for them what an
// SM can load: a tile of 128 x 256 needs 96 bytes a clock at the int8 rate,
// one of 256 x 256 on a pair of CTAs (cta_group::2), each loading half of
// either side, 64.  8192 x 4096 x 28672: 789 us in single CTAs where pairs took
// 684, and 564 on a cool GPU with the pipe active for 94 % of the cycles, at
// 1.5 GHz under the power limit (3.4 PFLOP/s; 645 us, 3.0, when it runs on).
//
// Results: one warp a scheduler could not scale, convert and store a tile
// while the next one was multiplied (10 us against 9).  Two groups of four
// warps take every other 16 tokens, read TMEM as MMA fragments, and stmatrix
// turns channels into rows of 16 bytes.  The same product took 884 us with
// direct 2-byte stores and 805 with one group that went through shared memory
// by 2-byte stores, where this took 684.
#include <algorithm>
#include <cmath>
#include <mutex>
#include <utility>

#include "../common.cuh"
#include "cache_elem.cuh"
#include "int8_ops.h"

namespace kus {
namespace i8gemm {

constexpr int kThreads = 320;          // producer, issuer, two groups of four epilogue warps
constexpr int kBK = kInt8Block;        // bytes of K per stage
constexpr int kWBytes = kInt8Block * kBK;

constexpr int kMostStages = 8;
constexpr int kBarriers = 2 * kMostStages + 6;
// Shared memory of a CTA: alone on its SM, or one of two.
constexpr int kSmemAlone = 232448, kSmemHalf = 115712;
constexpr int kSmemSm = 233472, kSmemKept = 1024;      // of an SM, and what the driver keeps of it for each CTA
constexpr int kTmemSm = 512;                           // columns of an SM

// Results go through shared memory, so that whole lines are written: each
// group of epilogue warps has two buffers of 16 tokens x 128 channels, the
// tokens 272 bytes apart in 16 bits (stmatrix writes eight of them at once).
constexpr int kChunk = 16;
KUS_HOST_DEVICE constexpr int token_bytes(int element) { return kInt8Block * element + (element == 2 ? 16 : 0); }
KUS_HOST_DEVICE constexpr int out_bytes(int element) { return 4 * kChunk * token_bytes(element); }

KUS_HOST_DEVICE int x_rows(const Int8Plan& p) { return p.pair ? p.width / 2 : p.width; }   // tokens a CTA loads
KUS_HOST_DEVICE int stage_bytes(const Int8Plan& p) { return kWBytes + x_rows(p) * kBK; }
// Beside the stages: of whole units the results' buffers and two tiles' token
// scales, of split ones the parts of the sums that this CTA adds up (or over
// the stages).
KUS_HOST_DEVICE int side_bytes(const Int8Plan& p, int element) {
  if (p.splits == 1) return out_bytes(element) + 2 * p.width * 4;
  return p.apart ? (p.width + p.splits - 1) / p.splits * p.splits * kInt8Block * 4 : 0;
}
int smem_bytes(const Int8Plan& p, int element) {
  return p.stages * stage_bytes(p) + side_bytes(p, element) + kBarriers * 8 + 16 + 1024;
}
// What a CTA asks for, so that each wait for TMEM ends: it has no limit, and two
// clusters that each held a part of what the other waits for would never end.
//  - A CTA's share of an SM's shared memory is no less than its share of the
//    TMEM: whatever meets on an SM, of products of several streams too, fits.
//  - What fits may still find the columns cut up (they are given out on multiples
//    of their number, 256 behind 32 start at 256, and a pair's are the same on
//    both SMs).  CTAs that wait for others of their cluster while they hold TMEM
//    (pairs, and splits whose parts lie over the stages) therefore have their
//    SM's to themselves, or half of it: the other half is one more such CTA's, or
//    that of CTAs that wait for none.  Those, whole products and splits with
//    their parts beside the stages, free theirs as soon as they are done.
// (The framework's other clusters with TMEM, pairs of the bf16 product, leave
// room for no CTA here.)
constexpr int kSmemLeast = 2 * (kWBytes + 16 * kBK);                     // less than any CTA has
constexpr int kSmemLone = kSmemSm - kSmemKept - kSmemLeast - kSmemKept;  // beside it none has room
int least_smem(int tmem_columns) { return (tmem_columns * kSmemSm + kTmemSm - 1) / kTmemSm - kSmemKept; }

// D(tmem, s32) (+)= A(smem, s8) * B(smem, s8)^T; of a pair: A rows 128 and
// up and the second half of B's rows are the other CTA's (umma_f16_pair).
template <bool PAIR>
KUS_DEVICE void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  if (PAIR)
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Arrive on `bar` (PAIR: of both CTAs of the pair whose even rank is `lead`)
// once the products issued so far have ended.
template <bool PAIR>
KUS_DEVICE void commit(uint64_t* bar, uint32_t lead) {
  if (PAIR)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)(3u << lead))
        : "memory");
  else
    umma_commit(bar);
}

// Instruction descriptor: kind::i8, A and B signed and K-major, D s32, M x N.
KUS_DEVICE uint32_t idesc_s8(int M, int N) {
  return (2u << 4)                        // D format s32
         | (1u << 7)                      // A signed
         | (1u << 10)                     // B signed
         | ((uint32_t)(N >> 3) << 17)     // N / 8
         | ((uint32_t)(M >> 4) << 24);    // M / 16
}

KUS_DEVICE void tmem_ld16(uint32_t taddr, int (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// The halves of cluster_sync.
KUS_DEVICE void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
KUS_DEVICE void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// As if `bytes` of a copy had landed.
KUS_DEVICE void mbar_complete_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

KUS_DEVICE void st_cluster(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

template <typename O>
KUS_DEVICE O out_of(float x) { return Elem<O>::from_f(x); }
template <>
KUS_DEVICE float out_of<float>(float x) { return x; }
template <typename O>
KUS_DEVICE float float_of(O x) { return Elem<O>::to_f(x); }
template <>
KUS_DEVICE float float_of<float>(float x) { return x; }

// 16 lanes (channels) x 16 columns (tokens) of TMEM as the fragments of two
// 16 x 8 products: v[4 g + 2 s + i] is lane t / 4 + 8 s, column 8 g + 2 (t % 4) + i.
KUS_DEVICE void tmem_ld_frag(uint32_t taddr, int (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr));
}
KUS_DEVICE void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Four 8 x 8 matrices of 16 bits, each written with its columns as rows of 16
// bytes; lane 8 i + j gives the address of row j of matrix i.
KUS_DEVICE void stmatrix4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b),
               "r"(c), "r"(d)
               : "memory");
}

// Results of 16 tokens x the warp's 32 channels, from TMEM to a buffer of
// tokens x 128 channels.
template <typename O>
KUS_DEVICE void stage_chunk(uint32_t taddr, const float* xs, const float (&ws)[4], const float (&b)[4], uint8_t* to,
                            int quarter, int lane) {
  if constexpr (sizeof(O) == 2) {
    int v[2][8];
    tmem_ld_frag(taddr, v[0]);
    tmem_ld_frag(taddr + (16u << 16), v[1]);
    float2 x[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) x[g] = *reinterpret_cast<const float2*>(xs + 8 * g + 2 * (lane % 4));
    tmem_ld_wait();
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      uint32_t m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {      // channels 8 i .. of the warp's 32
        const int* w = &v[i / 2][4 * g + 2 * (i % 2)];
        m[i] = pack2<O>(fmaf((float)w[0] * x[g].x, ws[i], b[i]), fmaf((float)w[1] * x[g].y, ws[i], b[i]));
      }
      const int token = 8 * g + lane % 8, channel = quarter * 32 + lane / 8 * 8;
      stmatrix4_trans(smem_u32(to + token * token_bytes(2) + channel * 2), m[0], m[1], m[2], m[3]);
    }
  } else {
    int v[16];
    tmem_ld16(taddr, v);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      reinterpret_cast<float*>(to + i * token_bytes(4))[quarter * 32 + lane] = fmaf((float)v[i] * xs[i], ws[0], b[0]);
  }
}

// Where results go.
template <typename O>
struct Results {
  O* out;
  long long ldc;
  int N;
  bool aligned;      // whole vectors of 16 bytes

  KUS_DEVICE explicit Results(const Int8Gemm& a)
      : out(reinterpret_cast<O*>(a.out)),
        ldc(a.ldc),
        N(a.N),
        aligned((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.ldc * sizeof(O))) % 16 == 0) {}

  // `tokens` rows of 128 channels, `stride` bytes apart, by 128 threads.
  KUS_DEVICE void write(const uint8_t* from, int stride, int t0, int tokens, int n0, int thread) const {
    constexpr int kVec = 16 / sizeof(O), kPerRow = kInt8Block / kVec, kRows = 128 / kPerRow;
    if (aligned && n0 + kInt8Block <= N) {
      const int r = thread / kPerRow, e = thread % kPerRow * kVec;
      O* dst = out + (t0 + r) * ldc + n0 + e;
      from += r * stride + e * sizeof(O);
#pragma unroll
      for (int t = 0; t < kChunk; t += kRows) {
        if (t + r < tokens) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(from);
        dst += kRows * ldc;
        from += kRows * stride;
      }
    } else if (n0 + thread < N) {
      for (int t = 0; t < tokens; ++t)
        out[(t0 + t) * ldc + n0 + thread] = reinterpret_cast<const O*>(from + t * stride)[thread];
    }
  }
};

// Unit u of a plan: channel tile, token tile.  Token tiles run fastest within
// groups of `group`, so that a group's tokens stay in L2 while the weights
// stream past them once.
struct Unit {
  int n, t;
};
KUS_DEVICE Unit unit_at(const Int8Plan& p, int u) {
  const int per = p.group * p.channel_tiles;
  const int g = u / per, r = u - g * per;
  const int wide = min(p.group, p.token_tiles - g * p.group);
  Unit x;
  x.n = r / wide;
  x.t = g * p.group + r - x.n * wide;
  return x;
}

// PAIR: clusters of pairs of CTAs; a unit is 256 channels, CTA rank r of the
// pair stages channels 128 r.. and half of the tile's tokens, the even CTA
// issues cta_group::2 products over both, and each CTA holds and writes its
// own 128 channels.  SPLIT: the p.splits CTAs (pairs) of a cluster share one
// unit's K; else each walks whole units.
template <typename O, bool PAIR, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 2)
    gemm_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, Int8Gemm a,
                Int8Plan p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stages = p.stages, stage_size = stage_bytes(p);
  uint8_t* side = smem + stages * stage_size;
  uint8_t* staged = side;
  float* scales = reinterpret_cast<float*>(staged + out_bytes(sizeof(O)));
  uint64_t* full = reinterpret_cast<uint64_t*>(side + side_bytes(p, sizeof(O)));
  uint64_t* empty = full + kMostStages;
  uint64_t* tfull = empty + kMostStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* drained = tempty + 2;
  uint64_t* told = drained + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(told + 1);
  int* other_fills = reinterpret_cast<int*>(tmem_holder + 1);      // of a pair's leader: the other CTA's

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int blocks = (a.K + kBK - 1) / kBK;
  const int units = p.channel_tiles * p.token_tiles;
  constexpr int kCtas = PAIR ? 2 : 1;                    // of a unit (of a part of its K)
  const uint32_t rank = PAIR || SPLIT ? cluster_rank() : 0u;
  const int half = PAIR ? (int)(rank & 1) : 0;           // which of the pair
  const uint32_t lead = PAIR ? rank & ~1u : rank;
  const bool leads = rank == lead;
  const int part = SPLIT ? (int)rank / kCtas : 0;
  const int each = SPLIT ? (blocks + p.splits - 1) / p.splits : blocks;
  const int kb0 = part * each, kb1 = min(blocks, kb0 + each);
  const int first = (int)blockIdx.x / (SPLIT ? kCtas * p.splits : kCtas);
  const int step = SPLIT ? units : (int)gridDim.x / kCtas;

  const uint32_t lead_full = PAIR ? mapa_shared(smem_u32(full), lead) : 0u;
  auto load_w = [&](int st, const Unit& at, int kb) {
    uint8_t* to = smem + st * stage_size;
    const int row = ((at.n * kCtas + half) * blocks + kb) * kInt8Block;
    if (leads) mbar_arrive_expect_tx(&full[st], (uint32_t)stage_size * kCtas);    // both CTAs' bytes
    if (PAIR)
      tma_load_2d_pair(to, &tmW, lead_full + 8u * st, 0, row);
    else
      tma_load_2d(to, &tmW, &full[st], 0, row);
  };
  // The first stages' weights are on their way while this kernel sets up and
  // the one before ends: none but pack_kernel writes weights, and a copy
  // behind it keeps whatever follows from starting early.
  const Unit start = unit_at(p, first);
  const int early = first < units ? min(stages, kb1 - kb0) : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 2 * kCtas);      // each group of epilogue warps
    }
    mbar_init(drained, 1);
    mbar_init(told, 1);
    fence_barrier_init();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // the copies find the barriers ready
    if (!PAIR)
      for (int j = 0; j < early; ++j) load_w(j, start, kb0 + j);
  }
  // A pair's barriers are ready before the other CTA arrives on them; the
  // other CTAs of a split only have to run before they are given their parts
  // (and do, whatever keeps them waiting for TMEM).
  if (PAIR && warp == 1) tmem_alloc_pair(tmem_holder, p.tmem_columns);
  tc_fence_before();
  if (PAIR)
    cluster_sync();
  else if (SPLIT)
    cluster_arrive();
  if (!PAIR) {
    if (warp == 1) tmem_alloc(tmem_holder, p.tmem_columns);
    tc_fence_before();
    __syncthreads();
  }
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  if (warp != 0) {
    pdl_wait();
    pdl_trigger();
  }

  // SPLIT: this CTA's share of the unit's tokens, and what an epilogue warp
  // multiplies their sums with, loaded while they are computed
  bool summed = false;      // this warp's part of the sums is in TMEM
  const int t0_split = start.t * p.width, tokens_split = min(p.width, a.M - t0_split);
  const int share = (tokens_split + p.splits - 1) / p.splits, mine = t0_split + part * share;
  const int shared_tokens = min(share, tokens_split - part * share);
  const int n_split = (start.n * kCtas + half) * kInt8Block + lane * 4;
  float ws_split[4] = {0.f, 0.f, 0.f, 0.f}, b_split[4] = {0.f, 0.f, 0.f, 0.f}, xs_split = 0.f;
  if (SPLIT && warp >= 2) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (n_split + i >= a.N) continue;
      ws_split[i] = a.w_scales[n_split + i];
      if (a.bias) b_split[i] = float_of<O>(reinterpret_cast<const O*>(a.bias)[n_split + i]);
    }
    if (warp - 2 < shared_tokens) xs_split = a.x_scales[mine + warp - 2];
  }
  if (warp == 0) {
    if (elect_one_sync()) {
      auto load_x = [&](int st, const Unit& at, int kb) {
        uint8_t* to = smem + st * stage_size + kWBytes;
        const int row = at.t * p.width + half * x_rows(p);
        if (PAIR)
          tma_load_2d_pair(to, &tmX, lead_full + 8u * st, kb * kBK, row);
        else
          tma_load_2d(to, &tmX, &full[st], kb * kBK, row);
      };
      prefetch_tmap(&tmX);
      if (PAIR)
        for (int j = 0; j < early; ++j) load_w(j, start, kb0 + j);
      pdl_wait();
      pdl_trigger();
      for (int j = 0; j < early; ++j) load_x(j, start, kb0 + j);
      int fills = early, st = early == stages ? 0 : early;
      uint32_t phase = early == stages ? 1u : 0u;
      bool ok = true;
      int kb = kb0 + early;
      for (int u = first; ok && u < units; u += step) {
        const Unit at = unit_at(p, u);
        for (; kb < kb1; ++kb) {
          if (!mbar_wait(&empty[st], phase ^ 1, kErrWaitEmpty)) {
            ok = false;
            break;
          }
          load_w(st, at, kb);
          load_x(st, at, kb);
          ++fills;
          if (++st == stages) {
            st = 0;
            phase ^= 1;
          }
        }
        kb = kb0;
      }
      // Every copy has landed before the CTA ends (a pair's, before the leader
      // meets the other CTA at the end).  Where waits ran out, one CTA of a pair
      // may have filled stages that the other did not: the leader then expects
      // or makes up for one CTA's bytes.  Neither is ahead by more than the
      // stages, since a stage is free again once both have filled it.
      if (leads) {
        int other = fills;
        if (PAIR && mbar_wait_cluster<true>(told, 0, kErrWaitFull)) other = *other_fills;
        const int filled = max(fills, other);
        for (int f = max(0, filled - stages); f < filled; ++f) {
          if (PAIR && f >= fills) mbar_arrive_expect_tx(&full[f % stages], (uint32_t)stage_size);
          if (PAIR && f >= other) mbar_complete_tx(&full[f % stages], (uint32_t)stage_size);
          mbar_wait<true>(&full[f % stages], (f / stages) & 1, kErrWaitFull);
        }
      } else {
        st_cluster(mapa_shared(smem_u32(other_fills), lead), fills);
        mbar_arrive_remote(mapa_shared(smem_u32(told), lead));
      }
    }
  } else if (warp == 1) {
    if (leads && elect_one_sync()) {
      const uint32_t idesc = idesc_s8(kInt8Block * kCtas, p.width);
      int st = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int u = first; ok && u < units; u += step) {
        const bool freed = PAIR ? mbar_wait_cluster(&tempty[acc], acc_phase ^ 1, kErrWaitTmemEmpty)
                                : mbar_wait(&tempty[acc], acc_phase ^ 1, kErrWaitTmemEmpty);
        if (!freed) break;
        tc_fence_after();
        const uint32_t d = tmem_base + acc * p.width;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&full[st], phase, kErrWaitFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t dw = umma_desc_sw128(smem_u32(smem + st * stage_size));
          const uint64_t dx = umma_desc_sw128(smem_u32(smem + st * stage_size + kWBytes));
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k)
            umma_i8<PAIR>(d, dw + (uint64_t)(2 * k), dx + (uint64_t)(2 * k), idesc, (kb > kb0 || k > 0) ? 1u : 0u);
          commit<PAIR>(&empty[st], lead);
          if (++st == stages) {
            st = 0;
            phase ^= 1;
          }
        }
        commit<PAIR>(&tfull[acc], lead);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      // every product has ended before the CTA does
      commit<PAIR>(drained, lead);
      mbar_wait<true>(drained, 0, kErrWaitTmemFull);
    } else if (!leads && elect_one_sync()) {
      mbar_wait<true>(drained, 0, kErrWaitTmemFull);
    }
  } else {
    const int quarter = warp & 3, group = (warp - 2) / 4;
    const int row = quarter * 32 + lane;     // channel within the CTA's 128
    const int gt = (threadIdx.x - 64) % 128;
    const uint32_t lead_tempty = PAIR ? mapa_shared(smem_u32(tempty), lead) : 0u;
    const Results<O> results(a);
    int acc = 0, buffer = 0;
    uint32_t acc_phase = 0;
    for (int u = first; u < units; u += step) {
      const Unit at = unit_at(p, u);
      const int t0 = at.t * p.width, tokens = min(p.width, a.M - t0);
      const int n0 = (at.n * kCtas + half) * kInt8Block;
      float* xs = scales + acc * p.width;
      float ws[4], b[4];
      if (!SPLIT) {
        // this unit's token scales; the other accumulator's may still be read
        for (int i = threadIdx.x - 64; i < p.width; i += 256) xs[i] = i < tokens ? a.x_scales[t0 + i] : 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // of 16-bit results a thread has the channels lane / 4 + 8 i of its warp's 32, of 32-bit ones channel `lane`
          const int n = n0 + (sizeof(O) == 2 ? quarter * 32 + 8 * i + lane / 4 : row);
          ws[i] = n < a.N ? a.w_scales[n] : 0.f;
          b[i] = a.bias && n < a.N ? float_of<O>(reinterpret_cast<const O*>(a.bias)[n]) : 0.f;
          if (sizeof(O) == 4) break;
        }
        named_barrier(2, 256);
      }
      const bool ok = __all_sync(0xffffffffu, mbar_wait(&tfull[acc], acc_phase, kErrWaitTmemFull));
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * p.width);
      if (!SPLIT) {
#pragma unroll 1
        for (int c = group * kChunk; c < tokens; c += 2 * kChunk) {
          uint8_t* to = staged + (group * 2 + buffer) * kChunk * token_bytes(sizeof(O));
          buffer ^= 1;
          if (ok) stage_chunk<O>(taddr + c, xs + c, ws, b, to, quarter, lane);
          named_barrier(3 + group, 128);      // the group's other buffer has been read by now
          if (ok) results.write(to, token_bytes(sizeof(O)), t0 + c, min(kChunk, tokens - c), n0, gt);
        }
        tc_fence_before();
        named_barrier(3 + group, 128);
        if (gt == 0) PAIR ? mbar_arrive_remote(lead_tempty + 8u * acc) : mbar_arrive(&tempty[acc]);
      } else {
        summed = ok;
      }
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  }
  if (!SPLIT) {
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();      // the pair is done with both TMEMs and barriers
    if (warp == 1) PAIR ? tmem_dealloc_pair(tmem_base, p.tmem_columns) : tmem_dealloc(tmem_base, p.tmem_columns);
    return;
  }

  // The CTAs that hold parts of the same sums share the tile's tokens: each
  // gives the others their tokens' parts, [part][token][128] in the owner's
  // memory, and adds up all parts of its own (integers: any order gives the
  // same).  Over the stages where there is no room beside them, once every CTA
  // has used them up.
  const Results<O> results(a);
  const int most = (p.width + p.splits - 1) / p.splits;
  uint8_t* parts = p.apart ? side : smem;
  if (!PAIR) cluster_wait();
  if (!p.apart) cluster_sync();
  if (summed) {
    const int quarter = warp & 3;
    const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const uint32_t to = smem_u32(parts) + (uint32_t)((part * most * kInt8Block + quarter * 32 + lane) * 4);
#pragma unroll 1
    for (int c = (warp - 2) / 4 * 16; c < tokens_split; c += 32) {
      int v[16];
      tmem_ld16(taddr + c, v);
      int owner = c / share, at = c - owner * share;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (c + i < tokens_split) st_cluster(mapa_shared(to + at * (kInt8Block * 4), owner * kCtas + half), v[i]);
        if (++at == share) {
          at = 0;
          ++owner;
        }
      }
    }
  }
  tc_fence_before();
  // all parts are where they belong; a pair is done with both TMEMs, other CTAs
  // free theirs ahead of the wait
  if (PAIR) {
    cluster_sync();
    if (warp == 1) tmem_dealloc_pair(tmem_base, p.tmem_columns);
  } else {
    cluster_arrive();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, p.tmem_columns);
    cluster_wait();
  }
  if (warp < 2) return;
  for (int c = warp - 2; c < shared_tokens; c += 8) {
    const float xs = c < 8 ? xs_split : a.x_scales[mine + c];
    int s[4] = {0, 0, 0, 0};
    for (int r = 0; r < p.splits; ++r) {
      const int4 v = *reinterpret_cast<const int4*>(parts + ((r * most + c) * kInt8Block + lane * 4) * 4);
      s[0] += v.x;
      s[1] += v.y;
      s[2] += v.z;
      s[3] += v.w;
    }
    O* dst = results.out + (mine + c) * results.ldc + n_split;
    alignas(16) O y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = out_of<O>(fmaf((float)s[i] * xs, ws_split[i], b_split[i]));
    if (results.aligned && n_split + 4 <= a.N) {
      if constexpr (sizeof(O) == 2)
        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
      else
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(y);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n_split + i < a.N) dst[i] = y[i];
    }
  }
}

// 16 bytes of a packed block a thread.
__global__ void __launch_bounds__(256) pack_kernel(const int8_t* w, long long stride, int N, int K, int blocks,
                                                   int8_t* packed, long long vectors, bool on16) {
  pdl_wait();
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < vectors; i += (long long)gridDim.x * 256) {
    const long long block = i / (kInt8Block * kBK / 16);
    const int in = (int)(i % (kInt8Block * kBK / 16));
    const long long n = block / blocks * kInt8Block + in / (kBK / 16);
    const long long k = block % blocks * kBK + in % (kBK / 16) * 16;
    union {
      int8_t b[16];
      uint4 v;
    } x;
    if (n < N && k + 16 <= K && on16) {
      x.v = *reinterpret_cast<const uint4*>(w + n * stride + k);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x.b[e] = n < N && k + e < K ? w[n * stride + k + e] : (int8_t)0;
    }
    reinterpret_cast<uint4*>(packed)[i] = x.v;
  }
}

// Rows that start anywhere, to rows on 16 bytes (their ends up to the next 16
// bytes are never multiplied): 16 bytes a thread, inside a row from the two
// aligned vectors that hold them.
__global__ void __launch_bounds__(256) align_kernel(const int8_t* q, long long stride, int M, int K, int8_t* out) {
  pdl_wait();
  pdl_trigger();
  const int per = (K + 15) / 16;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < (long long)M * per; i += (long long)gridDim.x * 256) {
    const long long t = i / per;
    const int k = (int)(i - t * per) * 16;
    const int8_t* from = q + t * stride + k;
    union {
      int8_t b[16];
      uint4 v;
    } x;
    if (k >= 16 && k + 32 <= K) {
      const int by = (int)(reinterpret_cast<uintptr_t>(from) & 15);
      const uint4* p = reinterpret_cast<const uint4*>(from - by);
      x.v = by ? i8rows::shifted(p[0], p[1], by) : p[0];
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x.b[e] = k + e < K ? from[e] : (int8_t)0;
    }
    reinterpret_cast<uint4*>(out)[i] = x.v;
  }
}

bool byte_map(CUtensorMap* map, const void* base, long long rows, int cols, long long stride, int box_rows) {
  auto fn = gemm_impl::get_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)stride};
  cuuint32_t box[2] = {(cuuint32_t)kBK, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename O, bool PAIR, bool SPLIT>
void launch(const Int8Gemm& a, const Int8Plan& p, const CUtensorMap& w, const CUtensorMap& x, cudaStream_t s) {
  const auto kernel = gemm_kernel<O, PAIR, SPLIT>;
  ensure_smem_attr(reinterpret_cast<const void*>(kernel), kSmemAlone);
  launch_kc(kernel, dim3(p.grid), dim3(kThreads), p.smem, s, (PAIR ? 2 : 1) * p.splits, w, x, a, p);
}

template <typename O>
void launch_as(const Int8Gemm& a, const Int8Plan& p, const CUtensorMap& w, const CUtensorMap& x, cudaStream_t s) {
  if (p.pair)
    p.splits > 1 ? launch<O, true, true>(a, p, w, x, s) : launch<O, true, false>(a, p, w, x, s);
  else
    p.splits > 1 ? launch<O, false, true>(a, p, w, x, s) : launch<O, false, false>(a, p, w, x, s);
}

}  // namespace i8gemm

void int8_pack(const int8_t* w, long long stride, int N, int K, int8_t* packed, cudaStream_t s) {
  const int blocks = (int)int8_blocks(K);
  const long long vectors = int8_blocks(N) * blocks * (kInt8Block * kInt8Block / 16);
  const bool on16 = reinterpret_cast<uintptr_t>(w) % 16 == 0 && stride % 16 == 0;
  const long long grid = (vectors + 255) / 256;
  i8gemm::pack_kernel<<<(unsigned)(grid < 148 * 64 ? grid : 148 * 64), 256, 0, s>>>(w, stride, N, K, blocks, packed,
                                                                                 vectors, on16);
}

void int8_align(const int8_t* q, long long stride, int M, int K, int8_t* out, cudaStream_t s) {
  LaunchBehind behind;
  const long long grid = ((long long)M * ((K + 15) / 16) + 255) / 256;
  launch_k(i8gemm::align_kernel, dim3((unsigned)std::min<long long>(grid, 148 * 32)), dim3(256), 0, s, q, stride, M, K,
           out);
}

Int8Slots int8_slots() {
  using namespace i8gemm;
  constexpr int kMaxDev = 64;
  static std::mutex mu;
  static Int8Slots known[kMaxDev];
  static bool done[kMaxDev] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  if (dev >= 0 && dev < kMaxDev && done[dev]) return known[dev];
  Int8Slots s{};
  const auto kernel = gemm_kernel<float, true, true>;
  ensure_smem_attr(reinterpret_cast<const void*>(kernel), kSmemAlone);
  for (int c = 1; c <= 8; ++c) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c);
    cfg.blockDim = dim3(i8gemm::kThreads);
    cfg.dynamicSmemBytes = kSmemAlone;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = c;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 1;
    }
    s.clusters[c] = n;
  }
  if (dev >= 0 && dev < kMaxDev) {
    known[dev] = s;
    done[dev] = true;
  }
  return s;
}

namespace i8gemm {

// What a cut is expected to take, in us (less what every cut takes).  Of its
// products, stage by stage: the loads (92 bytes a clock of a CTA alone on its
// SM, 52 of each of two), 2 clocks a token and a clock for 600 bytes (what they
// take of the power: of tiles with as many rounds the widest wins under the
// power limit, 8192 x 14336 x 4096 in tiles of 256 346 us, of 224 361), at
// least 300 clocks (150) of latency; of the results 17 ns a token and tile to
// write; of the bytes that HBM moves.  Each hides some of the others: their
// root of squares.  The last tile is written when nothing is left to hide it, a
// round takes 0.67 us to fill the stages, adding up parts of K 0.7 us and 14 ns
// a token.  The numbers were fitted to 1251 cuts of 95 products (1 to 12000
// tokens, 64 to 45000 channels, K 64 to 16384) queued one behind the other:
// times are off by 14 % on average, and the cut that is cheapest by this takes
// 2.7 % longer than the best (up to a quarter for a few products of 4 to 6 us).
double cost(const Int8Plan& p, int M, int N, int K, int element, const Int8Slots& slots) {
  const int ctas = p.pair ? 2 : 1, blocks = (int)int8_blocks(K), units = p.token_tiles * p.channel_tiles;
  const int each = (blocks + p.splits - 1) / p.splits;
  // times that one CTA after another runs on an SM; two at once share it
  const int waves = p.splits > 1 ? 1 : (units + slots.clusters[ctas] - 1) / slots.clusters[ctas];
  const int rounds = p.splits > 1 && !p.alone ? 2 : waves;
  const double stage = std::max({stage_bytes(p) / (p.alone ? 92.0 : 52.0), 2.0 * p.width + stage_bytes(p) / 600.0,
                                 p.alone ? 300.0 : 150.0});
  const double write = 0.017 * p.width;
  const double products = rounds * each * stage / 1.9e3, writes = p.splits > 1 ? 0 : rounds * write;
  const double moved = ((double)N * K + (double)M * K + (double)M * N * element) / 8.5e6;
  double t = std::sqrt(products * products + writes * writes + moved * moved) + write;
  t += 0.67 * (p.alone ? waves : (waves + 1) / 2);
  if (p.splits > 1) t += 0.73 + 0.014 * p.width * (p.splits - 1) / p.splits;
  return t;
}

}  // namespace i8gemm

// The cheapest of: single CTAs (up to 400 tokens; from there pairs, which load
// half the tokens each, took less in every case) or pairs, tiles of 16 to 256
// tokens, K whole or split over a cluster's CTAs, one CTA an SM or two.
// Clusters of a split all run at once: a second wave would double the time
// (40 tiles of 5120 x 5120: 8.7 us split over 6, 13.7 over 7).  Two CTAs an SM
// only where one each would leave some out: they are placed two by two even
// where SMs stay idle (306 x 13824 x 5120 in 120 CTAs: 44 us, alone 27).
Int8Plan int8_plan(int M, int N, int K, int element, const Int8Slots& slots) {
  using namespace i8gemm;
  const int blocks = (int)int8_blocks(K);
  Int8Plan best{};
  double least = 0;
  for (int pair = M > 400; pair < 2; ++pair) {
    const int ctas = pair ? 2 : 1, step = 16 * ctas;
    int last = 0;
    for (int tile = step; tile <= 256; tile += tile < 32 ? 16 : 32) {
      Int8Plan p{};
      p.pair = pair;
      p.token_tiles = (int)(((long long)M + tile - 1) / tile);
      if (p.token_tiles > 64 && tile < 256) continue;
      p.width = (int)(((long long)M + p.token_tiles - 1) / p.token_tiles + step - 1) / step * step;
      if (p.width == last) continue;
      last = p.width;
      p.token_tiles = (int)(((long long)M + p.width - 1) / p.width);
      p.channel_tiles = (int)((int8_blocks(N) + ctas - 1) / ctas);
      const int units = p.token_tiles * p.channel_tiles;
      for (int splits = 1; splits * ctas <= 8 && splits <= blocks; ++splits) {
        const int each = (blocks + splits - 1) / splits, clusters = slots.clusters[splits * ctas];
        if ((splits - 1) * each >= blocks) continue;      // the last would have nothing
        if (splits > 1 && units > 2 * clusters) break;
        p.splits = splits;
        for (int alone = 0; alone < 2; ++alone) {
          if (alone ? splits > 1 && units > clusters : p.width > 128 || units <= clusters) continue;
          p.alone = alone;
          const double t = cost(p, M, N, K, element, slots);
          if (best.width == 0 || t < least) {
            best = p;
            least = t;
          }
        }
      }
    }
  }
  Int8Plan& p = best;
  const int ctas = p.pair ? 2 : 1, units = p.token_tiles * p.channel_tiles;
  const int most = (p.alone ? 1 : 2) * slots.clusters[ctas];
  p.grid = ctas * (p.splits > 1 ? units * p.splits : std::min(units, most));
  p.tmem_columns = 32;
  while (p.tmem_columns < 2 * p.width) p.tmem_columns *= 2;
  p.apart = p.splits > 1 && p.width <= (p.alone ? 64 : 32);
  p.stages = kMostStages;
  while (smem_bytes(p, element) > (p.alone ? kSmemAlone : kSmemHalf)) --p.stages;
  const bool waits = p.pair || (p.splits > 1 && !p.apart);      // for others, while it holds TMEM
  if (waits && !p.alone) p.tmem_columns = kTmemSm / 2;
  const int asked = std::max(least_smem(p.tmem_columns), waits && p.alone ? kSmemLone : 0);
  // What a CTA fills once needs no more room than that, and what it asks for
  // anyway: more of the next kernel fits beside it.
  if (p.splits > 1 ? p.apart : units <= most) {
    int stages = std::min(p.stages, std::max(2, (blocks + p.splits - 1) / p.splits));
    std::swap(stages, p.stages);
    while (p.stages < stages && smem_bytes(p, element) < asked) ++p.stages;
  }
  p.smem = std::max(smem_bytes(p, element), asked);
  // the tokens of a group: at most 32 MB
  p.group = (int)std::max(1ll, std::min<long long>(p.token_tiles, (32ll << 20) / ((long long)p.width * K)));
  return p;
}

bool int8_weight_map(CUtensorMap* map, const int8_t* packed, int N, int K) {
  const long long rows = int8_blocks(N) * int8_blocks(K) * kInt8Block;
  // (an odd pair asks for the block behind the last: zeros)
  return rows + int8_blocks(K) * kInt8Block < (1ll << 31) &&
         i8gemm::byte_map(map, packed, rows, kInt8Block, kInt8Block, kInt8Block);
}

bool int8_token_map(CUtensorMap* map, const int8_t* x, long long stride, int M, int K, const Int8Plan& p) {
  return i8gemm::byte_map(map, x, M, K, stride, i8gemm::x_rows(p));
}

void int8_gemm(const Int8Gemm& a, const Int8Plan& p, const CUtensorMap& weights, const CUtensorMap& tokens,
               cudaStream_t s) {
  if (a.M == 0) return;
  LaunchBehind behind;
  if (a.type == kInt8TypeBF16) return i8gemm::launch_as<__nv_bfloat16>(a, p, weights, tokens, s);
  if (a.type == kInt8TypeFP16) return i8gemm::launch_as<__half>(a, p, weights, tokens, s);
  return i8gemm::launch_as<float>(a, p, weights, tokens, s);
}

}  // namespace kus
