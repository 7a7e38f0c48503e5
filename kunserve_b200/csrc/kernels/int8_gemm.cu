// Matrix product of 8-bit tokens with 8-bit weights on tcgen05 (kind::i8):
//   y[t, n] = (sum_k q[t, k] w[n, k]) s[t] v[n] + b[n]
// with exact int32 sums in TMEM.
//
// The weights are the MMA's M side (128 channels a tile) whatever the number
// of tokens, the tokens its N side (a tile of 16 to 256): a decode step pads
// its few tokens to 16 and no further.  A k-block is 128 bytes of K, 32 a
// product.
#include "../common.cuh"
#include "cache_elem.cuh"
#include "int8_ops.h"

namespace kus {
namespace i8gemm {

constexpr int kThreads = 192;          // producer, issuer, four epilogue warps
constexpr int kBK = kInt8Block;        // bytes of K per stage
constexpr int kWBytes = kInt8Block * kBK;

// CAP: most tokens of a tile.  64: two CTAs an SM.
template <int CAP>
struct Cfg {
  static constexpr int kXBytes = CAP * kBK;
  static constexpr int kStageBytes = kWBytes + kXBytes;
  static constexpr int kStages = 4;
  static constexpr int kTmemCols = 2 * CAP;             // two accumulators
  static constexpr int kScaleBytes = 2 * CAP * 4;
  static constexpr int kSmemBytes = kStages * kStageBytes + kScaleBytes + 1024 + 256;
  static constexpr int kPerSm = CAP <= 64 ? 2 : 1;
};

// D(tmem, s32) (+)= A(smem, s8) * B(smem, s8)^T
KUS_DEVICE void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}"
      ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
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

KUS_DEVICE int4 ld_cluster(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <typename O>
KUS_DEVICE O out_of(float x) { return Elem<O>::from_f(x); }
template <>
KUS_DEVICE float out_of<float>(float x) { return x; }
template <typename O>
KUS_DEVICE float float_of(O x) { return Elem<O>::to_f(x); }
template <>
KUS_DEVICE float float_of<float>(float x) { return x; }

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

template <int CAP, typename O, bool SPLIT>
__global__ void __launch_bounds__(kThreads, Cfg<CAP>::kPerSm)
    gemm_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, Int8Gemm a,
                Int8Plan p) {
  using C = Cfg<CAP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_w = smem;
  uint8_t* smem_x = smem + C::kStages * kWBytes;
  float* scales = reinterpret_cast<float*>(smem + C::kStages * C::kStageBytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + 2 * CAP);
  uint64_t* empty = full + C::kStages;
  uint64_t* tfull = empty + C::kStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* drained = tempty + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drained + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int blocks = (a.K + kBK - 1) / kBK;
  const int units = p.channel_tiles * p.token_tiles;
  // SPLIT: a cluster per unit, CTA `rank` takes a range of its K; else each
  // CTA walks whole units
  const int rank = SPLIT ? (int)cluster_rank() : 0;
  const int each = SPLIT ? (blocks + p.splits - 1) / p.splits : blocks;
  const int kb0 = rank * each, kb1 = min(blocks, kb0 + each);
  const int first = SPLIT ? (int)blockIdx.x / p.splits : (int)blockIdx.x;
  const int step = SPLIT ? units : (int)gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 128);
    }
    mbar_init(drained, 1);
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(tmem_holder, C::kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  pdl_wait();
  pdl_trigger();

  if (warp == 0) {
    if (elect_one_sync()) {
      prefetch_tmap(&tmW);
      prefetch_tmap(&tmX);
      const uint32_t bytes = kWBytes + p.width * kBK;
      int fills = 0;
      bool ok = true;
      for (int u = first; ok && u < units; u += step) {
        const Unit at = unit_at(p, u);
        for (int kb = kb0; kb < kb1; ++kb, ++fills) {
          const int st = fills % C::kStages;
          if (!mbar_wait(&empty[st], ((fills / C::kStages) & 1) ^ 1, kErrWaitEmpty)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&full[st], bytes);
          tma_load_2d(smem_w + st * kWBytes, &tmW, &full[st], 0, (at.n * blocks + kb) * kInt8Block);
          tma_load_2d(smem_x + st * C::kXBytes, &tmX, &full[st], kb * kBK, at.t * p.width);
        }
      }
      // every copy has landed before the CTA ends
      for (int f = max(0, fills - C::kStages); f < fills; ++f)
        mbar_wait<true>(&full[f % C::kStages], (f / C::kStages) & 1, kErrWaitFull);
    }
  } else if (warp == 1) {
    if (elect_one_sync()) {
      const uint32_t idesc = idesc_s8(kInt8Block, p.width);
      int used = 0, acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int u = first; ok && u < units; u += step) {
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1, kErrWaitTmemEmpty)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + acc * CAP;
        for (int kb = kb0; kb < kb1; ++kb, ++used) {
          const int st = used % C::kStages;
          if (!mbar_wait(&full[st], (used / C::kStages) & 1, kErrWaitFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t dw = umma_desc_sw128(smem_u32(smem_w + st * kWBytes));
          const uint64_t dx = umma_desc_sw128(smem_u32(smem_x + st * C::kXBytes));
#pragma unroll
          for (int k = 0; k < kBK / 32; ++k)
            umma_i8(d, dw + (uint64_t)(2 * k), dx + (uint64_t)(2 * k), idesc, (kb > kb0 || k > 0) ? 1u : 0u);
          umma_commit(&empty[st]);
        }
        umma_commit(&tfull[acc]);
        if (++acc == 2) {
          acc = 0;
          acc_phase ^= 1;
        }
      }
      // every product has ended before the CTA does
      umma_commit(drained);
      mbar_wait<true>(drained, 0, kErrWaitTmemFull);
    }
  } else {
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;     // channel within the tile
    const int et = threadIdx.x - 64;
    O* out = reinterpret_cast<O*>(a.out);
    const O* bias = reinterpret_cast<const O*>(a.bias);
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int u = first; u < units; u += step) {
      const Unit at = unit_at(p, u);
      const int t0 = at.t * p.width, tokens = min(p.width, a.M - t0);
      const int n = at.n * kInt8Block + row;
      if (!SPLIT) {
        // this unit's token scales; the other half may still be read
        for (int i = et; i < p.width; i += 128) scales[acc * CAP + i] = i < tokens ? a.x_scales[t0 + i] : 0.f;
        named_barrier(2, 128);
      }
      const bool ok = __all_sync(0xffffffffu, mbar_wait(&tfull[acc], acc_phase, kErrWaitTmemFull));
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(acc * CAP);
      if (!SPLIT) {
        const float ws = n < a.N ? a.w_scales[n] : 0.f;
        const float b = bias && n < a.N ? float_of<O>(bias[n]) : 0.f;
        if (ok) {
#pragma unroll 1
          for (int c = 0; c < tokens; c += 16) {
            int v[16];
            tmem_ld16(taddr + c, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float y = fmaf((float)v[i] * scales[acc * CAP + c + i], ws, b);
              if (c + i < tokens && n < a.N) out[(long long)(t0 + c + i) * a.ldc + n] = out_of<O>(y);
            }
          }
        }
        tc_fence_before();
        mbar_arrive(&tempty[acc]);
      } else if (ok) {
        // this CTA's part of the sums, over the stages: all of them are used up
        int* part = reinterpret_cast<int*>(smem);
#pragma unroll 1
        for (int c = 0; c < tokens; c += 16) {
          int v[16];
          tmem_ld16(taddr + c, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) part[(c + i) * kInt8Block + row] = v[i];
        }
      }
      if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, C::kTmemCols);
  if (SPLIT) {
    // the cluster's CTAs share the tile's tokens: each adds up all parts of
    // its own (integers: any order gives the same)
    cluster_sync();
    const Unit at = unit_at(p, first);
    const int t0 = at.t * p.width, tokens = min(p.width, a.M - t0);
    const int share = (tokens + p.splits - 1) / p.splits;
    const int n = at.n * kInt8Block + lane * 4;
    const uint32_t part = smem_u32(smem);
    O* out = reinterpret_cast<O*>(a.out);
    const O* bias = reinterpret_cast<const O*>(a.bias);
    float ws[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ws[i] = n + i < a.N ? a.w_scales[n + i] : 0.f;
      b[i] = bias && n + i < a.N ? float_of<O>(bias[n + i]) : 0.f;
    }
    for (int c = rank * share + warp; c < min(tokens, (rank + 1) * share); c += kThreads / 32) {
      const float xs = a.x_scales[t0 + c];
      const uint32_t at_c = part + (uint32_t)(c * kInt8Block + lane * 4) * 4;
      int s[4] = {0, 0, 0, 0};
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (r < p.splits) {
          const int4 v = ld_cluster(mapa_shared(at_c, r));
          s[0] += v.x;
          s[1] += v.y;
          s[2] += v.z;
          s[3] += v.w;
        }
      }
      O* dst = out + (long long)(t0 + c) * a.ldc + n;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) dst[i] = out_of<O>(fmaf((float)s[i] * xs, ws[i], b[i]));
    }
    cluster_sync();    // no CTA ends while others read its part
  }
}

// 16 bytes of a packed block a thread.
__global__ void __launch_bounds__(256) pack_kernel(const int8_t* w, long long stride, int N, int K, int blocks,
                                                   int8_t* packed, long long vectors, bool on16) {
  // the next kernel may read weights ahead of its wait: this one never lets
  // it start early
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

template <int CAP, typename O>
void launch(const Int8Gemm& a, const Int8Plan& p, const CUtensorMap& w, const CUtensorMap& x, cudaStream_t s) {
  using C = Cfg<CAP>;
  if (p.splits > 1) {
    ensure_smem_attr(reinterpret_cast<const void*>(gemm_kernel<CAP, O, true>), C::kSmemBytes);
    launch_kc(gemm_kernel<CAP, O, true>, dim3(p.grid), dim3(kThreads), C::kSmemBytes, s, p.splits, w, x, a, p);
  } else {
    ensure_smem_attr(reinterpret_cast<const void*>(gemm_kernel<CAP, O, false>), C::kSmemBytes);
    launch_k(gemm_kernel<CAP, O, false>, dim3(p.grid), dim3(kThreads), C::kSmemBytes, s, w, x, a, p);
  }
}

template <typename O>
void launch_cap(const Int8Gemm& a, const Int8Plan& p, const CUtensorMap& w, const CUtensorMap& x, cudaStream_t s) {
  if (p.width <= 64)
    launch<64, O>(a, p, w, x, s);
  else
    launch<256, O>(a, p, w, x, s);
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

Int8Plan int8_plan(int M, int N, int K, int sms) {
  Int8Plan p{};
  const int blocks = (int)int8_blocks(K);
  p.token_tiles = (M + 255) / 256;
  p.width = ((M + p.token_tiles - 1) / p.token_tiles + 15) / 16 * 16;
  p.token_tiles = (M + p.width - 1) / p.width;
  p.channel_tiles = (int)int8_blocks(N);
  const long long units = (long long)p.token_tiles * p.channel_tiles;
  const int slots = sms * (p.width <= 64 ? 2 : 1);
  p.splits = 1;
  if (units < slots) {
    p.splits = (int)(slots / units);
    if (p.splits > 8) p.splits = 8;
    if (p.splits > blocks) p.splits = blocks;
    const int each = (blocks + p.splits - 1) / p.splits;
    p.splits = (blocks + each - 1) / each;
  }
  // the tokens of a group: at most 32 MB
  const long long tile = (long long)p.width * K;
  const long long group = (32ll << 20) / tile;
  p.group = (int)(group < 1 ? 1 : group > p.token_tiles ? p.token_tiles : group);
  p.grid = p.splits > 1 ? (int)units * p.splits : (int)(units < slots ? units : slots);
  return p;
}

bool int8_weight_map(CUtensorMap* map, const int8_t* packed, int N, int K) {
  const long long rows = int8_blocks(N) * int8_blocks(K) * kInt8Block;
  return rows < (1ll << 31) && i8gemm::byte_map(map, packed, rows, kInt8Block, kInt8Block, kInt8Block);
}

bool int8_token_map(CUtensorMap* map, const int8_t* x, long long stride, int M, int K, int width) {
  return i8gemm::byte_map(map, x, M, K, stride, width);
}

void int8_gemm(const Int8Gemm& a, const Int8Plan& p, const CUtensorMap& weights, const CUtensorMap& tokens,
               cudaStream_t s) {
  if (a.M == 0) return;
  LaunchBehind behind;
  if (a.type == kInt8TypeBF16) return i8gemm::launch_cap<__nv_bfloat16>(a, p, weights, tokens, s);
  if (a.type == kInt8TypeFP16) return i8gemm::launch_cap<__half>(a, p, weights, tokens, s);
  return i8gemm::launch_cap<float>(a, p, weights, tokens, s);
}

}  // namespace kus
