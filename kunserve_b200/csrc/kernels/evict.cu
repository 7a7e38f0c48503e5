// Eviction from a paged cache by accumulated attention weight.
//
// Of a request's n cached tokens each KV head keeps c = min(keep, n): the
// protected ones (position below `sinks`, or above newest - recent) before
// all others, then by weight, the lowest slot first among equals; NaN ranks
// last.  Kept tokens in slots >= c move into the evicted slots < c, in slot
// order, so that the first c slots hold what is kept: no more rows move than
// must, no destination is another move's source, and the order of keys does
// not matter to attention.
#include "../common.cuh"
#include "cache_ops.h"

namespace kus {
namespace evict {

constexpr int kBins = 2048;       // radix digits of 11, 11 and 10 bits
constexpr int kPasses = 3;

// Rank of a token as an unsigned number, larger kept first.
KUS_DEVICE uint32_t rank_key(float w, int pos, int sinks, int newest, int recent) {
  if (pos < sinks || (long long)pos > (long long)newest - recent) return 0xFFFFFFFFu;
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.f);   // -0 counts as 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

KUS_DEVICE uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// A cluster takes one (request, KV head) row, each CTA a slice of its slots.
// The boundary key is found by three radix passes over the row (histograms
// joined through distributed shared memory); the slots are then classified
// and ranked with ballots, each warp walking a contiguous piece.  With
// CACHED the slice's keys stay in shared memory; else they are read again.
template <int NT, bool CACHED>
__global__ void __launch_bounds__(NT) select_kernel(EvictSelect a, int ctas, int slice) {
  constexpr int kW = NT / 32;
  constexpr int kPer = kBins / NT;
  extern __shared__ uint32_t dyn[];
  uint32_t* hist = dyn;                        // [kPasses][kBins]
  uint32_t* keys = dyn + kPasses * kBins;      // [slice] (CACHED)
  __shared__ uint32_t warp_sum_s[kW], warp_sum2_s[kW];
  __shared__ uint32_t pick[2];
  __shared__ uint32_t share[4];                // ties, holes, movers of this CTA
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.x / ctas;
  const int rank = blockIdx.x - row * ctas;
  const int req = row / a.g.kvh, kh = row - req * a.g.kvh;
  const int4 rq = __ldg(reinterpret_cast<const int4*>(a.reqs) + req);
  const int n = rq.x;
  int2* moves = a.moves + (long long)row * a.cap;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (n <= a.keep) {   // the same for the whole cluster
    for (int i = rank * NT + tid; i < a.cap; i += ctas * NT) moves[i] = make_int2(-1, -1);
    if (rank == 0 && tid == 0) a.counts[row] = 0;
    return;
  }
  const int* table = a.pages + rq.y;
  const int lo = min(n, rank * slice), hi = min(n, lo + slice);
  auto read_key = [&](int i) {
    const int page = __ldg(table + kv_page_col(a.g, i));
    const long long at = ((long long)page * a.g.kvh + kh) * a.g.block_size + kv_page_slot(a.g, i);
    return rank_key(__ldg(a.weights + at), __ldg(a.slot_positions + at), a.sinks, rq.z, a.recent);
  };
  auto key_of = [&](int i) { return CACHED ? keys[i - lo] : read_key(i); };

  for (int i = tid; i < kPasses * kBins; i += NT) hist[i] = 0;
  if (CACHED) {
#pragma unroll 4
    for (int i = lo + tid; i < hi; i += NT) keys[i - lo] = read_key(i);
  }
  __syncthreads();

  // boundary key: the keep-th largest; `need` of its equals are kept
  uint32_t prefix = 0, mask = 0, need = (uint32_t)a.keep, equal = 0;
#pragma unroll 1
  for (int p = 0; p < kPasses; ++p) {
    const int shift = p == 0 ? 21 : p == 1 ? 10 : 0;
    const uint32_t digits = p == 2 ? 1023u : 2047u;
    uint32_t* h = hist + p * kBins;
    for (int i = lo + tid; i < hi; i += NT) {
      const uint32_t k = key_of(i);
      if ((k & mask) == prefix) atomicAdd(&h[(k >> shift) & digits], 1u);
    }
    if (ctas > 1) cluster_sync(); else __syncthreads();
    // bins from the largest digit down, kPer a thread
    uint32_t c[kPer], sum = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int bin = kBins - 1 - (tid * kPer + j);
      c[j] = 0;
      if (ctas > 1) {
        const uint32_t addr = smem_u32(h + bin);
        for (int r = 0; r < ctas; ++r) c[j] += ld_cluster(mapa_shared(addr, r));
      } else {
        c[j] = h[bin];
      }
      sum += c[j];
    }
    uint32_t incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    if (lane == 31) warp_sum_s[warp] = incl;
    __syncthreads();
    uint32_t before = incl - sum;
    for (int w = 0; w < warp; ++w) before += warp_sum_s[w];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (before < need && need <= before + c[j]) {
        pick[0] = (uint32_t)(kBins - 1 - (tid * kPer + j));
        pick[1] = need - before;
        share[3] = c[j];
      }
      before += c[j];
    }
    __syncthreads();
    prefix |= pick[0] << shift;
    mask |= digits << shift;
    need = pick[1];
    equal = share[3];
  }

  // each warp's contiguous piece of the slice
  const int piece = ((hi - lo + kW - 1) / kW + 31) / 32 * 32;
  const int w_lo = min(hi, lo + warp * piece), w_hi = min(hi, w_lo + piece);
  const uint32_t below = (1u << lane) - 1u;
  // sum over the warps (and CTAs) before this one
  auto scan = [&](uint32_t v, uint32_t* sums, int which) {
    if (lane == 0) sums[warp] = v;
    __syncthreads();
    uint32_t before = 0, total = 0;
    for (int w = 0; w < kW; ++w) {
      if (w == warp) before = total;
      total += sums[w];
    }
    if (tid == 0) share[which] = total;
    return before;
  };
  auto before_cta = [&](int which) {
    uint32_t v = 0;
    const uint32_t addr = smem_u32(share + which);
    for (int r = 0; r < rank; ++r) v += ld_cluster(mapa_shared(addr, r));
    return v;
  };
  uint32_t tie_at = 0;   // equals before this warp's piece
  if (equal > need) {
    uint32_t ties = 0;
    for (int i = w_lo; i < w_hi; i += 32) {
      const bool in = i + lane < w_hi;
      ties += __popc(__ballot_sync(0xffffffffu, in && key_of(i + lane) == prefix));
    }
    tie_at = scan(ties, warp_sum_s, 0);
    if (ctas > 1) {
      cluster_sync();
      tie_at += before_cta(0);
    }
  }
  // the kept slots of [i, i + 32) as a lane mask; advances `at` past their equals
  auto kept_mask = [&](int i, uint32_t& at) {
    const bool in = i + lane < w_hi;
    const uint32_t k = in ? key_of(i + lane) : 0u;
    const uint32_t eq = __ballot_sync(0xffffffffu, in && k == prefix);
    const bool kept = in && (k > prefix || (k == prefix && at + __popc(eq & below) < need));
    at += __popc(eq);
    return __ballot_sync(0xffffffffu, kept);
  };
  // holes: evicted slots below keep; movers: kept slots from keep on
  auto lanes_below = [&](int i, int end) -> uint32_t {   // lanes whose slot i + lane is below `end`
    return end <= i ? 0u : end - i >= 32 ? 0xffffffffu : (1u << (end - i)) - 1u;
  };
  uint32_t holes = 0, movers = 0, at = tie_at;
  for (int i = w_lo; i < w_hi; i += 32) {
    const uint32_t kept = kept_mask(i, at), low = lanes_below(i, a.keep), in = lanes_below(i, w_hi);
    holes += __popc(~kept & low & in);
    movers += __popc(kept & ~low);
  }
  __syncthreads();   // warp_sum_s is free again
  uint32_t hole_at = scan(holes, warp_sum_s, 1);
  uint32_t mover_at = scan(movers, warp_sum2_s, 2);
  uint32_t total = 0;
  if (ctas > 1) {
    cluster_sync();
    hole_at += before_cta(1);
    mover_at += before_cta(2);
    const uint32_t addr = smem_u32(share + 1);
    for (int r = 0; r < ctas; ++r) total += ld_cluster(mapa_shared(addr, r));
  } else {
    __syncthreads();
    total = share[1];
  }
  at = tie_at;
  for (int i = w_lo; i < w_hi; i += 32) {
    const uint32_t kept = kept_mask(i, at), low = lanes_below(i, a.keep), in = lanes_below(i, w_hi);
    const uint32_t hm = ~kept & low & in, mm = kept & ~low;
    if (hm >> lane & 1u) moves[hole_at + __popc(hm & below)].x = i + lane;
    if (mm >> lane & 1u) moves[mover_at + __popc(mm & below)].y = i + lane;
    hole_at += __popc(hm);
    mover_at += __popc(mm);
  }
  for (int i = (int)total + rank * NT + tid; i < a.cap; i += ctas * NT) moves[i] = make_int2(-1, -1);
  if (rank == 0 && tid == 0) a.counts[row] = (int)total;
  if (ctas > 1) cluster_sync();   // no CTA leaves while another reads its shared memory
}

template <int NT>
void launch_select(const EvictSelect& a, int ctas, int slice, cudaStream_t s) {
  constexpr int kHist = kPasses * kBins * 4;
  constexpr int kMost = 200 * 1024;
  const unsigned grid = (unsigned)a.n_reqs * a.g.kvh * ctas;
  const bool cached = kHist + slice * 4 <= kMost;
  if (cached) {
    const int smem = kHist + slice * 4;
    ensure_smem_attr(reinterpret_cast<const void*>(select_kernel<NT, true>), kMost);
    launch_kc(select_kernel<NT, true>, dim3(grid), dim3(NT), smem, s, ctas, a, ctas, slice);
  } else {
    launch_kc(select_kernel<NT, false>, dim3(grid), dim3(NT), kHist, s, ctas, a, ctas, slice);
  }
}

// A warp moves kMoves rows: their K and V as 16-byte vectors, all loads in
// flight before the first store, then their weights and positions.
constexpr int kMoves = 4;
constexpr int kCompactWarps = 8;

__global__ void __launch_bounds__(kCompactWarps * 32) compact_kernel(CacheCompact a, int per_row) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % 32;
  const long long w = (long long)blockIdx.x * kCompactWarps + threadIdx.x / 32;
  const int row = (int)(w / per_row), first = (int)(w - (long long)row * per_row) * kMoves;
  if (row >= a.n_reqs * a.g.kvh) return;
  const int n = min(a.counts[row], a.cap);
  if (first >= n) return;
  const int req = row / a.g.kvh, kh = row - req * a.g.kvh;
  const int4 rq = __ldg(reinterpret_cast<const int4*>(a.reqs) + req);
  const int* table = a.pages + rq.y;
  // lane m < kMoves: move first + m
  long long to = -1, from = 0;     // bytes of the K rows in the pool
  const long long v_off = a.g.layer_stride / 2;
  if (lane < kMoves && first + lane < n) {
    const int2 mv = a.moves[(long long)row * a.cap + first + lane];
    if (mv.x < 0 || mv.y < 0 || mv.x >= rq.x || mv.y >= rq.x) {
      set_error(kErrBounds, mv.x < 0 || mv.x >= rq.x ? mv.x : mv.y);
    } else {
      const int pd = __ldg(table + kv_page_col(a.g, mv.x)), ps = __ldg(table + kv_page_col(a.g, mv.y));
      const int sd = kv_page_slot(a.g, mv.x), ss = kv_page_slot(a.g, mv.y);
      to = kv_offset(a.g, pd, a.layer, false) + ((long long)sd * a.g.kvh + kh) * a.g.hd * 2;
      from = kv_offset(a.g, ps, a.layer, false) + ((long long)ss * a.g.kvh + kh) * a.g.hd * 2;
      const long long id = ((long long)pd * a.g.kvh + kh) * a.g.block_size + sd;
      const long long is = ((long long)ps * a.g.kvh + kh) * a.g.block_size + ss;
      if (a.weights) a.weights[id] = a.weights[is];
      if (a.slot_positions) a.slot_positions[id] = a.slot_positions[is];
    }
  }
  const int chunks = a.g.hd / 8, vecs = 2 * chunks * kMoves;   // 16-byte vectors of the moves
  constexpr int kBatch = 4;
  for (int v0 = 0; v0 < vecs; v0 += 32 * kBatch) {
    uint4 val[kBatch];
    long long dst[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int v = v0 + b * 32 + lane;
      const int m = v / (2 * chunks), c = v - m * 2 * chunks;
      const long long t = __shfl_sync(0xffffffffu, to, m < kMoves ? m : 0);
      const long long f = __shfl_sync(0xffffffffu, from, m < kMoves ? m : 0);
      const long long off = c < chunks ? c * 16 : v_off + (c - chunks) * 16;
      dst[b] = m < kMoves && t >= 0 ? t + off : -1;
      if (dst[b] >= 0) val[b] = *reinterpret_cast<const uint4*>(a.g.base + f + off);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (dst[b] >= 0) *reinterpret_cast<uint4*>(a.g.base + dst[b]) = val[b];
  }
}

}  // namespace evict

void evict_select(const EvictSelect& a, cudaStream_t s) {
  const int rows = a.n_reqs * a.g.kvh;
  if (rows <= 0) return;
  // Few long rows: several CTAs share one, down to 2048 slots each, while
  // the grid stays within two CTAs an SM.
  int ctas = 1;
  while (ctas < 8 && rows * ctas * 2 <= 2 * 148 && a.most_tokens > 2048 * ctas) ctas *= 2;
  const int slice = ((a.most_tokens + ctas - 1) / ctas + 31) / 32 * 32;
  if (slice <= 4096)
    evict::launch_select<256>(a, ctas, slice, s);
  else
    evict::launch_select<1024>(a, ctas, slice, s);
}

void cache_compact(const CacheCompact& a, cudaStream_t s) {
  const int rows = a.n_reqs * a.g.kvh;
  if (rows <= 0 || a.cap <= 0) return;
  const int per_row = (a.cap + evict::kMoves - 1) / evict::kMoves;
  const long long warps = (long long)rows * per_row;
  launch_k(evict::compact_kernel, dim3((unsigned)((warps + evict::kCompactWarps - 1) / evict::kCompactWarps)),
           dim3(evict::kCompactWarps * 32), 0, s, a, per_row);
}

}  // namespace kus
