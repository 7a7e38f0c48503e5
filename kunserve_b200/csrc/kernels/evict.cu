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
#include "cache_elem.cuh"
#include "cache_ops.h"

namespace kus {
namespace evict {

// Rank of a token as an unsigned number, larger kept first.
KUS_DEVICE uint32_t rank_key(float w, int pos, int sinks, int newest, int recent) {
  if (pos < sinks || (long long)pos > (long long)newest - recent) return 0xFFFFFFFFu;
  if (w != w) return 0u;
  const uint32_t b = __float_as_uint(w + 0.f);   // -0 counts as 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

KUS_DEVICE uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
// Sum of the word at `addr` over the first n CTAs of the cluster: all loads
// are issued before the first is used.
constexpr int kMostCtas = 8;
KUS_DEVICE uint32_t sum_cluster(uint32_t addr, int n) {
  uint32_t v[kMostCtas], sum = 0;
#pragma unroll
  for (int r = 0; r < kMostCtas; ++r) v[r] = r < n ? ld_cluster(mapa_shared(addr, r)) : 0u;
#pragma unroll
  for (int r = 0; r < kMostCtas; ++r) sum += v[r];
  return sum;
}

// Index of slot `i` of a page list's token among weights and positions.
KUS_DEVICE long long side_at(const KVGeom& g, int page, int kh, int i) {
  return ((long long)page * g.kvh + kh) * g.block_size + kv_page_slot(g, i);
}

// Sum of v over the warps before this one, and over all; `sums` holds a value
// a warp, and is free again after the next block barrier.
template <int NT>
KUS_DEVICE uint2 scan_warps(uint32_t v, uint32_t* sums) {
  constexpr int kW = NT / 32;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (lane == 0) sums[warp] = v;
  __syncthreads();
  const uint32_t mine = lane < kW ? sums[lane] : 0u;
  uint32_t incl = mine;
#pragma unroll
  for (int off = 1; off < kW; off <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += u;
  }
  return make_uint2(__shfl_sync(0xffffffffu, incl - mine, warp), __shfl_sync(0xffffffffu, incl, kW - 1));
}

// A cluster takes one (request, KV head) row, each CTA a slice of its slots.
// The boundary key (the keep-th largest) is found digit by digit from the
// top: a histogram of the digit over the keys that share the digits so far,
// joined over the cluster through distributed shared memory.  It ends as soon
// as all keys of the boundary's bin are kept, which for weights that differ
// is mostly after three of the four digits.  The slots
// are then classified and ranked with ballots, each warp walking a contiguous
// piece.  With CACHED the slice's keys stay in shared memory; else they are
// read again.  Bound by the latency of these steps: the keys are read once.
template <int NT, int BITS, bool CACHED>
__global__ void __launch_bounds__(NT) select_kernel(EvictSelect a, int ctas, int slice) {
  constexpr int kBins = 1 << BITS, kPasses = (31 + BITS) / BITS;
  constexpr int kPer = kBins / NT;
  static_assert(kPer >= 1, "a bin a thread at least");
  extern __shared__ uint32_t dyn[];
  uint32_t* hist = dyn;                        // [kPasses][kBins]
  uint32_t* keys = dyn + kPasses * kBins;      // [slice] (CACHED)
  __shared__ uint32_t sums[4][32];
  __shared__ uint32_t pick[kPasses][3];        // digit, kept of its keys, its keys
  __shared__ uint32_t share[3];                // ties, holes, movers of this CTA
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
    const long long at = side_at(a.g, __ldg(table + kv_page_col(a.g, i)), kh, i);
    return rank_key(a.weights[at], a.slot_positions[at], a.sinks, rq.z, a.recent);
  };
  auto key_of = [&](int i) { return CACHED ? keys[i - lo] : read_key(i); };

  for (int i = tid; i < kPasses * kBins; i += NT) hist[i] = 0;
  if (CACHED) {
    // kBatch keys a thread: their page lookups, then their loads, all in flight
    constexpr int kBatch = 6;
    for (int i0 = lo + tid; i0 < hi; i0 += kBatch * NT) {
      int page[kBatch], pos[kBatch];
      float w[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) page[b] = i0 + b * NT < hi ? __ldg(table + kv_page_col(a.g, i0 + b * NT)) : -1;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const long long at = side_at(a.g, max(page[b], 0), kh, i0 + b * NT);
        w[b] = page[b] >= 0 ? a.weights[at] : 0.f;
        pos[b] = page[b] >= 0 ? a.slot_positions[at] : 0;
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (page[b] >= 0) keys[i0 + b * NT - lo] = rank_key(w[b], pos[b], a.sinks, rq.z, a.recent);
    }
  }
  __syncthreads();

  // kept: keys whose digits so far are above `prefix`, and `need` of the
  // `equal` keys that match it
  uint32_t prefix = 0, mask = 0, need = (uint32_t)a.keep, equal = 0;
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    constexpr uint32_t kLast = (1u << (32 - BITS * (kPasses - 1))) - 1u;
    const int shift = p + 1 < kPasses ? 32 - BITS * (p + 1) : 0;
    const uint32_t digits = p + 1 < kPasses ? kBins - 1u : kLast;
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
      c[j] = ctas > 1 ? sum_cluster(smem_u32(h + bin), ctas) : h[bin];
      sum += c[j];
    }
    uint32_t incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    uint32_t before = incl - sum + scan_warps<NT>(__shfl_sync(0xffffffffu, incl, 31), sums[p & 1]).x;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (before < need && need <= before + c[j]) {
        pick[p][0] = (uint32_t)(kBins - 1 - (tid * kPer + j));
        pick[p][1] = need - before;
        pick[p][2] = c[j];
      }
      before += c[j];
    }
    __syncthreads();
    prefix |= pick[p][0] << shift;
    mask |= digits << shift;
    need = pick[p][1];
    equal = pick[p][2];
    if (need == equal) break;
  }

  // each warp's contiguous piece of the slice
  constexpr int kW = NT / 32;
  const int piece = ((hi - lo + kW - 1) / kW + 31) / 32 * 32;
  const int w_lo = min(hi, lo + warp * piece), w_hi = min(hi, w_lo + piece);
  const uint32_t below = (1u << lane) - 1u;
  auto before_cta = [&](int which) { return sum_cluster(smem_u32(share + which), rank); };
  uint32_t tie_at = 0;   // equals before this warp's piece
  const bool ties = need < equal;
  if (ties) {
    uint32_t t = 0;
    for (int i = w_lo; i < w_hi; i += 32) {
      const bool in = i + lane < w_hi;
      t += __popc(__ballot_sync(0xffffffffu, in && key_of(i + lane) == prefix));
    }
    const uint2 sc = scan_warps<NT>(t, sums[2]);
    tie_at = sc.x;
    if (ctas > 1) {
      if (tid == 0) share[0] = sc.y;
      cluster_sync();
      tie_at += before_cta(0);
    }
  }
  // the kept slots of [i, i + 32) as a lane mask; advances `at` past their equals
  auto kept_mask = [&](int i, uint32_t& at) {
    const bool in = i + lane < w_hi;
    const uint32_t k = in ? key_of(i + lane) & mask : 0u;
    bool kept = in && k >= prefix;
    if (ties) {
      const uint32_t eq = __ballot_sync(0xffffffffu, in && k == prefix);
      if (k == prefix) kept = kept && at + __popc(eq & below) < need;
      at += __popc(eq);
    }
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
  const uint2 hs = scan_warps<NT>(holes, sums[3]);
  __syncthreads();   // sums[3] is free again
  const uint2 ms = scan_warps<NT>(movers, sums[3]);
  uint32_t hole_at = hs.x, mover_at = ms.x, total = hs.y;
  if (ctas > 1) {
    if (tid == 0) {
      share[1] = hs.y;
      share[2] = ms.y;
    }
    cluster_sync();
    hole_at += before_cta(1);
    mover_at += before_cta(2);
    total = sum_cluster(smem_u32(share + 1), ctas);
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

constexpr int kMostSmem = 200 * 1024;
template <int NT, int BITS, bool CACHED>
void launch_select(const EvictSelect& a, int ctas, int slice, cudaStream_t s) {
  constexpr int kHist = (31 + BITS) / BITS * (1 << BITS) * 4;
  const int smem = kHist + (CACHED ? slice * 4 : 0);
  if (CACHED) ensure_smem_attr(reinterpret_cast<const void*>(select_kernel<NT, BITS, CACHED>), kMostSmem);
  launch_kc(select_kernel<NT, BITS, CACHED>, dim3((unsigned)a.n_reqs * a.g.kvh * ctas), dim3(NT), smem, s, ctas, a,
            ctas, slice);
}

// A warp moves kMoves tokens of a row: K and V as 16-byte vectors, weights and
// positions, all loads in flight before the first store.  Bound by the latency
// of index, page and row loads in turn, so by the warps an SM holds: all
// 64, at 32 registers a thread: 166,000 moves of 1 KB read and written in 33-36 us.
constexpr int kMoves = 4;
constexpr int kCompactWarps = 8;

// CH: 16-byte vectors of a row (0: any).
template <int CH>
__global__ void __launch_bounds__(kCompactWarps * 32, CH ? 8 : 4) compact_kernel(CacheCompact a, int per_row) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x % 32;
  const long long w = (long long)blockIdx.x * kCompactWarps + threadIdx.x / 32;
  const int row = (int)(w / per_row), first = (int)(w - (long long)row * per_row) * kMoves;
  if (row >= a.n_reqs * a.g.kvh) return;
  const int req = row / a.g.kvh, kh = row - req * a.g.kvh;
  // lane m < kMoves: move first + m
  const int n = min(a.counts[row], a.cap);
  int2 mv = make_int2(-1, -1);
  if (lane < kMoves && first + lane < a.cap) mv = a.moves[(long long)row * a.cap + first + lane];
  const int4 rq = __ldg(reinterpret_cast<const int4*>(a.reqs) + req);
  if (first >= n) return;
  const int* table = a.pages + rq.y;
  int to = -1, from = 0;           // K rows of this head's tokens, in rows of hd elements
  long long side = -1;             // the token's new place among weights and positions
  float weight = 0.f;
  int position = 0;
  if (lane < kMoves && first + lane < n) {
    if (mv.x < 0 || mv.y < 0 || mv.x >= rq.x || mv.y >= rq.x) {
      set_error(kErrBounds, mv.x < 0 || mv.x >= rq.x ? mv.x : mv.y);
    } else {
      const int pd = __ldg(table + kv_page_col(a.g, mv.x)), ps = __ldg(table + kv_page_col(a.g, mv.y));
      const int sd = kv_page_slot(a.g, mv.x), ss = kv_page_slot(a.g, mv.y);
      to = (kv_slot(a.g, pd, a.layer) * 2 * a.g.block_size + sd) * a.g.kvh + kh;
      from = (kv_slot(a.g, ps, a.layer) * 2 * a.g.block_size + ss) * a.g.kvh + kh;
      side = ((long long)pd * a.g.kvh + kh) * a.g.block_size + sd;
      const long long old = ((long long)ps * a.g.kvh + kh) * a.g.block_size + ss;
      if (a.weights) weight = a.weights[old];
      if (a.slot_positions) position = a.slot_positions[old];
    }
  }
  const int chunks = CH ? CH : a.g.hd / 8, vecs = 2 * chunks * kMoves;   // 16-byte vectors of the moves
  const int v_rows = a.g.block_size * a.g.kvh;                 // from a K row to its V row
  auto at = [&](int row, int c) {
    const int v = c >= chunks;
    return reinterpret_cast<uint4*>(a.g.base) + (long long)(row + (v ? v_rows : 0)) * chunks + (v ? c - chunks : c);
  };
  constexpr int kBatch = 4;
  for (int v0 = lane; v0 < vecs + lane; v0 += 32 * kBatch) {
    uint4 val[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int m = (v0 + b * 32) / (2 * chunks), c = v0 + b * 32 - m * 2 * chunks;
      const int f = __shfl_sync(0xffffffffu, from, m % kMoves), t = __shfl_sync(0xffffffffu, to, m % kMoves);
      if (m < kMoves && t >= 0) val[b] = *at(f, c);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int m = (v0 + b * 32) / (2 * chunks), c = v0 + b * 32 - m * 2 * chunks;
      const int t = __shfl_sync(0xffffffffu, to, m % kMoves);
      if (m < kMoves && t >= 0) *at(t, c) = val[b];
    }
  }
  if (side >= 0) {
    if (a.weights) a.weights[side] = weight;
    if (a.slot_positions) a.slot_positions[side] = position;
  }
}

}  // namespace evict

void evict_select(const EvictSelect& a, cudaStream_t s) {
  const int rows = a.n_reqs * a.g.kvh;
  if (rows <= 0) return;
  const LaunchBehind behind;
  // Few long rows: several CTAs share one, down to 2048 slots each, while the
  // grid stays within eight CTAs an SM.  Small blocks pay less for each of the
  // search's barriers (8 rows of 6001-20000 slots and 8 heads: 21 us, blocks of
  // 512 25 us, of 1024 29 us); from 4096 slots a CTA on the keys per thread
  // count for more (8 heads of 65000: 512 threads 21 us, 256 28 us).
  int ctas = 1;
  while (ctas < evict::kMostCtas && rows * ctas * 2 <= 8 * 148 && a.most_tokens > 2048 * ctas) ctas *= 2;
  const int slice = ((a.most_tokens + ctas - 1) / ctas + 31) / 32 * 32;
  if (slice <= 4096)
    evict::launch_select<256, 8, true>(a, ctas, slice, s);
  else if (slice <= (evict::kMostSmem - 8 * 1024) / 4)   // beside four histograms of 512 bins
    evict::launch_select<512, 9, true>(a, ctas, slice, s);
  else
    evict::launch_select<512, 9, false>(a, ctas, slice, s);
}

void cache_compact(const CacheCompact& a, cudaStream_t s) {
  const int rows = a.n_reqs * a.g.kvh;
  if (rows <= 0 || a.cap <= 0) return;
  const LaunchBehind behind;
  const int per_row = (a.cap + evict::kMoves - 1) / evict::kMoves;
  const long long warps = (long long)rows * per_row;
  const dim3 grid((unsigned)((warps + evict::kCompactWarps - 1) / evict::kCompactWarps));
  const dim3 block(evict::kCompactWarps * 32);
  if (a.g.hd == 128)
    launch_k(evict::compact_kernel<16>, grid, block, 0, s, a, per_row);
  else if (a.g.hd == 64)
    launch_k(evict::compact_kernel<8>, grid, block, 0, s, a, per_row);
  else
    launch_k(evict::compact_kernel<0>, grid, block, 0, s, a, per_row);
}

}  // namespace kus
