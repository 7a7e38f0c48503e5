// Attention over planned work units: the parts of a batch whose requests
// share prefixes, and single-token attention that keeps every key's weight.
//
//   out = softmax(scale q K^T) V over a query's keys, computed in parts: for
//   a range R of keys, m = max s, l = sum exp(s - m), O = sum exp(s - m) v;
//   parts join as M = max m, out = sum exp(m - M) O / sum exp(m - M) l.
//
// The keys of a shared prefix form ranges whose rows are the queries of all
// the requests behind it, so each key is read once for up to 16 (row kernel)
// or 128 rows (tile kernel, attention_prefix.cu).  A row without any key
// gives zeros.  All statistics and partial sums are fp32.
//
// Row kernel: one warp per (unit, KV head), no barriers beyond the warp.
// Stages of 32 keys (K and V rows, 16-byte cp.async, ends filled with zeros)
// run through a ring in shared memory; S = Q K^T and O += P V are m16n8k16
// tensor products with the unit's rows as M, so a key costs the same HBM
// bytes for 1 to 16 rows: bound by HBM (30 requests of 300-2300 tokens, 40
// heads: 812 MB in 130 us, 6.2 TB/s).  Six warps an SM hold 32 KB each; with
// few stages a warp's own latency counts: 3500 clk to its first stage, 2900 a
// stage, of which 1400 issue the next loads (TMA boxes instead gained nothing
// here, three stages neither: fewer warps then fit).
#include "../common.cuh"
#include "cache_elem.cuh"
#include "cache_ops.h"

namespace kus {
namespace cat {

constexpr int kKeys = kStageKeys;
constexpr float kLog2e = 1.4426950408889634f;

template <int HD>
struct RowCfg {
  static constexpr int kTile = kKeys * HD * 2;        // K or V of a stage
  static constexpr int kStage = 2 * kTile;
  static constexpr int kStages = HD == 128 ? 2 : 4;   // 32 KB a warp
  static constexpr int kSmem = kStages * kStage;
};

KUS_DEVICE void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
KUS_DEVICE void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
KUS_DEVICE void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
KUS_DEVICE void ldsm4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
KUS_DEVICE void ldsm4_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr)
               : "memory");
}
template <typename T>
KUS_DEVICE void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
KUS_DEVICE void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
KUS_DEVICE void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte offset of 16-byte chunk `ch` of tile row `r` (rows of HD elements,
// chunks exchanged within groups of 8 so that ldmatrix meets no bank twice).
template <int HD>
KUS_DEVICE uint32_t swz(int r, int ch) {
  return (uint32_t)(r * HD * 2 + (((ch & ~7) | ((ch ^ r) & 7)) << 4));
}

// Rounded part and remainder of two values as packed 16-bit pairs: hi + lo
// carries about 16 bits of P, so the product with V loses nothing that shows
// in a 16-bit output.  The second product is free where HBM is the bound.
// In fp16 the probabilities are taken 2^15 times too large (P <= 2^15, the
// sum with it): its exponents end at 2^-24, and many light keys together may
// hold weight that a long context's output shows.  What is below 2^-40 of the
// row's largest still vanishes.
template <typename T>
constexpr float kUpLog2 = std::is_same<T, __half>::value ? 15.f : 0.f;
template <typename T>
KUS_DEVICE void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack2<T>(a, b);
  const float2 r = Elem<T>::to_f2(*reinterpret_cast<typename Elem<T>::V2*>(&hi));
  lo = pack2<T>(a - r.x, b - r.y);
}

// `second`: launched behind the tile kernel of the same call, whose results it
// does not need: it starts beside it, and its first block only ends after it,
// so that the join (which waits for this kernel) finds both done.  (A block
// that waits keeps its place on the SM: the others leave it to the next.)
template <typename T, int HD, bool SCORES>
__global__ void __launch_bounds__(32) rows_kernel(CachedAttn a, float scale_log2, bool second) {
  using Cf = RowCfg<HD>;
  constexpr int kStages = Cf::kStages;
  constexpr int kCh = HD / 8;              // 16-byte chunks of a row
  constexpr int kRowsPer = 32 / kCh;       // rows that one load of the warp covers
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x;
  const int kvh = a.g.kvh, G = a.nq / kvh;
  if (!second) pdl_wait();
  pdl_trigger();
  const int u = blockIdx.x / kvh, kh = blockIdx.x - u * kvh;   // heads fastest: neighbours read the same cache rows
  const int4 u0 = __ldg(reinterpret_cast<const int4*>(a.row_units) + 2 * u);
  const int4 u1 = __ldg(reinterpret_cast<const int4*>(a.row_units) + 2 * u + 1);
  const int tok0 = u0.x, ntok = u0.y & 255, ng = (u0.y >> 8) & 255, g0 = u0.y >> 16;
  const int key_lo = u0.z, key_hi = u0.w, lim0 = u1.x;
  const int* table = a.pages + u1.y;
  const int rows = ntok * ng;
  const uint32_t ring = smem_u32(smem);
  const int nst = (key_hi - key_lo + kKeys - 1) / kKeys;
  const long long layer_elems = a.g.layer_stride / (int)sizeof(T);

  // keys: lane l looks up stage key l's page one stage ahead
  auto page_of = [&](int i) {
    const int key = key_lo + i * kKeys + lane;
    return key < key_hi ? __ldg(table + kv_page_col(a.g, key)) : -1;
  };
  int page = page_of(0);
  auto load = [&](int i) {
    long long off = -1;
    if (page >= 0) {
      const int key = key_lo + i * kKeys + lane;
      off = kv_slot(a.g, page, a.layer) * layer_elems + ((long long)kv_page_slot(a.g, key) * kvh + kh) * HD;
    }
    page = page_of(i + 1);
    const uint32_t dst = ring + (i % kStages) * Cf::kStage;
    const T* base = reinterpret_cast<const T*>(a.g.base);
#pragma unroll
    for (int p = 0; p < kKeys / kRowsPer; ++p) {
      const int r = p * kRowsPer + lane / kCh, ch = lane % kCh;
      const long long o = __shfl_sync(0xffffffffu, off, r);
      // rows past the range read nothing and become zeros: stale cache
      // contents (NaN included) never meet a zero weight
      const int bytes = o >= 0 ? 16 : 0;
      const T* src = base + (o >= 0 ? o + ch * 8 : 0);
      cp_async16(dst + swz<HD>(r, ch), src, bytes);
      cp_async16(dst + Cf::kTile + swz<HD>(r, ch), src + (o >= 0 ? layer_elems / 2 : 0), bytes);
    }
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (i < nst) load(i);
    cp_commit();
  }

  // A fragments: rows lane / 4 and lane / 4 + 8 of the unit (zeros past its rows)
  const int r_lo = lane >> 2;
  uint32_t qf[HD / 16][4];
  int lim[2];
#pragma unroll
  for (int hi = 0; hi < 2; ++hi) {
    const int r = r_lo + 8 * hi;
    const int j = r < rows ? r / ng : 0, gi = r < rows ? r - j * ng : 0;
    lim[hi] = lim0 + j;
    const T* qr = reinterpret_cast<const T*>(a.q) + (tok0 + j) * a.qt + (long long)(kh * G + g0 + gi) * a.qh +
                  2 * (lane & 3);
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) {
      qf[ks][hi] = r < rows ? *reinterpret_cast<const uint32_t*>(qr + ks * 16) : 0u;
      qf[ks][2 + hi] = r < rows ? *reinterpret_cast<const uint32_t*>(qr + ks * 16 + 8) : 0u;
    }
  }
  float o[HD / 8][4];
#pragma unroll
  for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};   // m: the max so far, less kUpLog2
  float* srow = nullptr;
  long long spitch = 0;
  if (SCORES) {
    // scores of the request: nq rows of its keys rounded up to a stage
    spitch = (lim0 + kKeys - 1) / kKeys * kKeys;
    srow = a.scores + (long long)u1.w * a.nq + (kh * G + g0) * spitch;
  }

  for (int i = 0; i < nst; ++i) {
    if (i + kStages - 1 < nst) load(i + kStages - 1);
    cp_commit();
    cp_wait<kStages - 1>();
    __syncwarp();
    const uint32_t kt = ring + (i % kStages) * Cf::kStage, vt = kt + Cf::kTile;
    constexpr int kNT = kKeys / 8;
    float s[kNT][4] = {};
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
      for (int kb = 0; kb < kKeys / 16; ++kb) {
        uint32_t b0, b1, b2, b3;
        ldsm4(kt + swz<HD>(kb * 16 + ((lane >> 4) << 3) + (lane & 7), ks * 2 + ((lane >> 3) & 1)), b0, b1, b2, b3);
        mma<T>(s[2 * kb], qf[ks], b0, b1);
        mma<T>(s[2 * kb + 1], qf[ks], b2, b3);
      }
    const int key = key_lo + i * kKeys + 2 * (lane & 3);
    uint32_t ph[kKeys / 16][4], pl[kKeys / 16][4];
    float alpha[2];
#pragma unroll
    for (int hi = 0; hi < 2; ++hi) {
      const int end = min(key_hi, lim[hi]);
      float mx = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float& x = s[nt][2 * hi + e];
          x = key + nt * 8 + e < end ? x * scale_log2 : -INFINITY;
          mx = fmaxf(mx, x);
        }
      if (SCORES && r_lo + 8 * hi < rows) {
        float* dst = srow + (r_lo + 8 * hi) * spitch + key;
#pragma unroll
        for (int nt = 0; nt < kNT; ++nt)
          *reinterpret_cast<float2*>(dst + nt * 8) = make_float2(s[nt][2 * hi], s[nt][2 * hi + 1]);
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mn = fmaxf(m[hi], mx - kUpLog2<T>);
      const float ref = mn == -INFINITY ? 0.f : mn;   // no key seen yet
      alpha[hi] = ex2(m[hi] - ref);
      m[hi] = mn;
      float sum = 0.f;
#pragma unroll
      for (int nt = 0; nt < kNT; ++nt) {
        const float p0 = ex2(s[nt][2 * hi] - ref), p1 = ex2(s[nt][2 * hi + 1] - ref);
        sum += p0 + p1;
        split2<T>(p0, p1, ph[nt / 2][2 * (nt & 1) + hi], pl[nt / 2][2 * (nt & 1) + hi]);
      }
      l[hi] = l[hi] * alpha[hi] + sum;
    }
    if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {   // some row's max grew
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) {
        o[d][0] *= alpha[0];
        o[d][1] *= alpha[0];
        o[d][2] *= alpha[1];
        o[d][3] *= alpha[1];
      }
    }
#pragma unroll
    for (int d = 0; d < HD / 16; ++d)
#pragma unroll
      for (int kb = 0; kb < kKeys / 16; ++kb) {
        uint32_t b0, b1, b2, b3;
        ldsm4_t(vt + swz<HD>(kb * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), d * 2 + (lane >> 4)), b0, b1, b2, b3);
        mma<T>(o[2 * d], ph[kb], b0, b1);
        mma<T>(o[2 * d + 1], ph[kb], b2, b3);
        mma<T>(o[2 * d], pl[kb], b0, b1);
        mma<T>(o[2 * d + 1], pl[kb], b2, b3);
      }
    __syncwarp();   // the slot is refilled in the next iteration
  }
  cp_wait<0>();

#pragma unroll
  for (int hi = 0; hi < 2; ++hi) {
    float sum = l[hi];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    const int r = r_lo + 8 * hi;
    if (r >= rows) continue;
    const long long prow = u1.z + (long long)kh * rows + r;
    float* dst = a.part_o + prow * HD + 2 * (lane & 3);
#pragma unroll
    for (int d = 0; d < HD / 8; ++d)
      *reinterpret_cast<float2*>(dst + d * 8) = make_float2(o[d][2 * hi], o[d][2 * hi + 1]);
    if ((lane & 3) == 0) a.part_ml[prow] = make_float2(m[hi], sum);
  }
  if (second && blockIdx.x == 0) pdl_wait();
}

// ------------------------------------------------------------------ joins
// (M, L) of two parts: the larger max, the sums brought to it.  The maxima
// skip NaN scores; the sums hold them, and keep what they hold here: a row
// with a NaN score has no softmax, its output is NaN.
KUS_DEVICE float2 join2(float2 a, float2 b) {
  const float m = fmaxf(a.x, b.x);
  if (m == -INFINITY) return make_float2(m, a.y + b.y);   // zeros or NaN
  return make_float2(m, a.y * ex2(a.x - m) + b.y * ex2(b.x - m));
}
KUS_DEVICE float2 warp_join(float2 s) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1)
    s = join2(s, make_float2(__shfl_xor_sync(0xffffffffu, s.x, off), __shfl_xor_sync(0xffffffffu, s.y, off)));
  return s;
}

// 1 / L; zero for a row without keys.
KUS_DEVICE float inverse_sum(float l) { return l == 0.f ? 0.f : 1.f / l; }
// What scores are taken against: M, or zero where all of them are -inf.
KUS_DEVICE float score_ref(float m) { return m == -INFINITY ? 0.f : m; }

// Partial row of list entry p for a KV head and a head of its group.
KUS_DEVICE long long part_row(int2 p, int kh, int g) { return p.x + (long long)kh * p.y + g; }

// The keys [key0, key1) of one (request, KV head): their weights
// exp(s - M) / L, summed over the group's heads, are added to the cache's;
// sh_m, sh_l: the heads' M and 1 / L.  A thread takes four neighbouring keys.
KUS_DEVICE void add_weights(const CachedAttn& a, const int* c, int kh, const float* sh_m, const float* sh_l) {
  const int G = a.nq / a.g.kvh, bs = a.g.block_size;
  const int key1 = c[2], first_page = c[3], len = c[4], col = c[5];
  const long long pitch = (len + kKeys - 1) / kKeys * kKeys;
  const int key = c[1] + 4 * threadIdx.x;
  if (key >= key1) return;
  // the rows of scores run on to a multiple of kKeys
  const float* src = a.scores + (long long)col * a.nq + kh * G * pitch + key;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int g = 0; g < G; ++g) {
    const float4 s = __ldcg(reinterpret_cast<const float4*>(src + g * pitch));
    const float m = sh_m[g], inv = sh_l[g];
    x.x += ex2(s.x - m) * inv;
    x.y += ex2(s.y - m) * inv;
    x.z += ex2(s.z - m) * inv;
    x.w += ex2(s.w - m) * inv;
  }
  auto at = [&](int k) {
    const int page = __ldg(a.pages + first_page + kv_page_col(a.g, k));
    return a.weights + ((long long)page * a.g.kvh + kh) * bs + kv_page_slot(a.g, k);
  };
  if (bs % 4 == 0 && key + 4 <= key1 && reinterpret_cast<uintptr_t>(a.weights) % 16 == 0) {
    float4* w = reinterpret_cast<float4*>(at(key));
    float4 v = *w;
    v.x += x.x;
    v.y += x.y;
    v.z += x.z;
    v.w += x.w;
    *w = v;
  } else {
    const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (key + i < key1) *at(key + i) += xs[i];
  }
}

constexpr int kJoinThreads = 128;
static_assert(4 * kJoinThreads == kChunkKeys, "add_weights takes a chunk, four keys a thread");

// Blocks [0, joins): W warps per (token, head) row join its parts, 4 / W rows
// a block; with a.stats the row's M and 1 / L are kept.  Blocks after them
// (weighted plans of few parts): one (chunk of keys, KV head) each, with the
// statistics joined again.  Each weight has one writer: no atomics.
// What the plan says is read before the wait on the kernels that wrote the
// parts.
template <typename T, int HD, int W>
__global__ void __launch_bounds__(32 * (W > 4 ? W : 4), W > 4 ? 4 : 8) join_kernel(CachedAttn a, unsigned joins) {
  constexpr int kPer = HD / 32;           // dims a lane holds
  constexpr int kRows = W > 4 ? 1 : 4 / W;
  __shared__ float sh_o[W > 1 ? W : 1][HD];
  __shared__ float2 sh_ml[W > 1 ? W : 1];
  __shared__ float sh_m[128], sh_l[128];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int kvh = a.g.kvh, G = a.nq / kvh;
  if (blockIdx.x < joins) {
    const long long row = (long long)blockIdx.x * kRows + warp / W;
    const bool have = row < (long long)a.T * a.nq;
    const int t = have ? (int)(row / a.nq) : 0, h = have ? (int)(row - (long long)t * a.nq) : 0;
    const int kh = h / G, g = h - kh * G;
    const int list = t * a.head_chunks + g / kRowUnitRows;
    const int e0 = __ldg(a.merge_off + list), e1 = have ? __ldg(a.merge_off + list + 1) : e0;
    const int first = e0 + 32 * (warp % W);
    int2 p = first + lane < e1 ? __ldg(a.merge + first + lane) : make_int2(0, 0);
    pdl_wait();
    pdl_trigger();
    float2 st = make_float2(-INFINITY, 0.f);
    float acc[kPer] = {};
    for (int b = first; b < e1; b += 32 * W) {
      if (b != first && b + lane < e1) p = __ldg(a.merge + b + lane);
      const long long prow = part_row(p, kh, g);
      float2 ml = make_float2(-INFINITY, 0.f);
      if (b + lane < e1) ml = __ldcg(a.part_ml + prow);
      const float2 sn = join2(st, warp_join(ml));
      const float w = ml.x == -INFINITY ? 0.f : ex2(ml.x - sn.x);
      const float keep = st.x == -INFINITY ? 0.f : ex2(st.x - sn.x);
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] *= keep;
      st = sn;
      const int n = min(32, e1 - b);
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, i);
        const long long ri = __shfl_sync(0xffffffffu, prow, i);
        const float* src = a.part_o + ri * HD + lane * kPer;
        // a part without keys has weight 0, whatever its sums hold
        if (kPer == 4) {
          const float4 v = __ldcg(reinterpret_cast<const float4*>(src));
          acc[0] += wi != 0.f ? wi * v.x : 0.f;
          acc[1] += wi != 0.f ? wi * v.y : 0.f;
          acc[kPer - 2] += wi != 0.f ? wi * v.z : 0.f;
          acc[kPer - 1] += wi != 0.f ? wi * v.w : 0.f;
        } else {
          const float2 v = __ldcg(reinterpret_cast<const float2*>(src));
          acc[0] += wi != 0.f ? wi * v.x : 0.f;
          acc[1] += wi != 0.f ? wi * v.y : 0.f;
        }
      }
    }
    if (W > 1) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) sh_o[warp][lane * kPer + i] = acc[i];
      if (lane == 0) sh_ml[warp] = st;
      __syncthreads();
      if (warp % W) return;
      float2 all = st;
      for (int j = 1; j < W; ++j) all = join2(all, sh_ml[j]);
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
      for (int j = 0; j < W; ++j) {
        const float w = sh_ml[j].x == -INFINITY ? 0.f : ex2(sh_ml[j].x - all.x);
#pragma unroll
        for (int i = 0; i < kPer; ++i) acc[i] += w * sh_o[j][lane * kPer + i];
      }
      st = all;
    }
    if (!have) return;
    const float inv = inverse_sum(st.y);
    T* dst = reinterpret_cast<T*>(a.out) + t * a.ot + h * a.oh + lane * kPer;
#pragma unroll
    for (int i = 0; i < kPer; i += 2)
      *reinterpret_cast<uint32_t*>(dst + i) = pack2<T>(acc[i] * inv, acc[i + 1] * inv);
    if (a.stats && lane == 0) a.stats[row] = make_float2(st.x, inv);
    return;
  }
  const unsigned w = blockIdx.x - joins;
  const int* c = a.chunks + (size_t)kChunkInts * (w / kvh);
  const int kh = w % kvh, t = __ldg(c);
  if (warp < 4)
    for (int g = warp; g < G; g += 4) {
      const int list = t * a.head_chunks + g / kRowUnitRows;
      const int e0 = __ldg(a.merge_off + list), e1 = __ldg(a.merge_off + list + 1);
      float2 st = make_float2(-INFINITY, 0.f);
      for (int e = e0 + lane; e < e1; e += 32) {
        const int2 p = __ldg(a.merge + e);
        if (e == e0 + lane && g == warp) pdl_wait();
        st = join2(st, __ldcg(a.part_ml + part_row(p, kh, g)));
      }
      st = warp_join(st);
      if (lane == 0) {
        sh_m[g] = score_ref(st.x);
        sh_l[g] = inverse_sum(st.y);
      }
    }
  pdl_wait();
  __syncthreads();
  if (threadIdx.x < kJoinThreads) add_weights(a, c, kh, sh_m, sh_l);
}

// Weights of plans with many parts: a block per (chunk of keys, KV head),
// with the statistics that join_kernel kept.
__global__ void __launch_bounds__(kJoinThreads, 8) weights_kernel(CachedAttn a) {
  __shared__ float sh_m[128], sh_l[128];
  const int kvh = a.g.kvh, G = a.nq / kvh;
  const int* c = a.chunks + (size_t)kChunkInts * (blockIdx.x / kvh);
  const int kh = blockIdx.x % kvh, t = __ldg(c);
  pdl_wait();
  if (threadIdx.x < G) {
    const float2 st = __ldcg(a.stats + (long long)t * a.nq + kh * G + threadIdx.x);
    sh_m[threadIdx.x] = score_ref(st.x);
    sh_l[threadIdx.x] = st.y;
  }
  __syncthreads();
  add_weights(a, c, kh, sh_m, sh_l);
}

template <typename T, int HD, bool SCORES>
void launch_rows(const CachedAttn& a, bool second, cudaStream_t s) {
  constexpr int smem = RowCfg<HD>::kSmem;
  ensure_smem_attr(reinterpret_cast<const void*>(rows_kernel<T, HD, SCORES>), smem);
  launch_k(rows_kernel<T, HD, SCORES>, dim3((unsigned)a.n_row_units * a.g.kvh), dim3(32), smem, s, a,
           a.scale * kLog2e, second);
}

template <typename T, int HD>
void launch(const CachedAttn& a, const CUtensorMap* map, int type, cudaStream_t s) {
  const bool tiles = a.n_tile_units > 0;
  if (tiles) cached_attention_tiles(a, *map, type, s);
  if (a.n_row_units > 0) a.scores ? launch_rows<T, HD, true>(a, tiles, s) : launch_rows<T, HD, false>(a, tiles, s);
  const long long rows = (long long)a.T * a.nq;
  // up to 32 parts fill one warp's lanes; rows of more take eight warps (their
  // statistics are then kept for the weights: joining them again for every
  // chunk of keys took longer than a launch)
  const bool wide = a.most_parts > 32;
  const unsigned joins = (unsigned)(wide ? rows : (rows + 3) / 4);
  const unsigned chunks = a.scores ? (unsigned)a.n_chunks * a.g.kvh : 0u;
  if (!wide) {
    CachedAttn b = a;
    b.stats = nullptr;
    launch_k(join_kernel<T, HD, 1>, dim3(joins + chunks), dim3(kJoinThreads), 0, s, b, joins);
  } else {
    launch_k(join_kernel<T, HD, 8>, dim3(joins), dim3(256), 0, s, a, joins);
    if (chunks) launch_k(weights_kernel, dim3(chunks), dim3(kJoinThreads), 0, s, a);
  }
}

}  // namespace cat

void cached_attention(const CachedAttn& a, const CUtensorMap* map, int type, cudaStream_t s) {
  if (a.T <= 0) return;
  const LaunchBehind behind;
  if (type == kTypeBF16) {
    a.hd == 128 ? cat::launch<__nv_bfloat16, 128>(a, map, type, s) : cat::launch<__nv_bfloat16, 64>(a, map, type, s);
  } else {
    a.hd == 128 ? cat::launch<__half, 128>(a, map, type, s) : cat::launch<__half, 64>(a, map, type, s);
  }
}

}  // namespace kus
