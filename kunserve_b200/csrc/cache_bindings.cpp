// Python bindings of the long-context cache operators (cache_ops.h): the
// handle of a paged cache, the plan of a batch, and one function per operator.
// Arguments are checked here; kunserve_b200/ops documents them.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>
#include <cmath>

#include "kernels/cache_ops.h"

namespace py = pybind11;
using namespace kus;

namespace {

// Text of an error message's parts.  Numbers are formatted with to_string:
// streaming them needs the locale tables of one C++ runtime, and the
// extension may be linked with another than the libraries it is loaded into.
std::string text(const char* s) { return s; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(torch::ScalarType t) { return c10::toString(t); }
std::string text(const torch::Device& d) { return d.str(); }
std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
template <typename... A>
std::string say(const A&... a) {
  std::string s;
  ((s += text(a)), ...);
  return s;
}
#define KUS_CHECK(cond, ...) TORCH_CHECK(cond, say(__VA_ARGS__))

int elem_type(const torch::Tensor& t, const char* what) {
  KUS_CHECK(t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat16, what,
              " must be bfloat16 or float16, got ", t.scalar_type());
  return t.scalar_type() == torch::kBFloat16 ? kTypeBF16 : kTypeFP16;
}

// A paged pool of one instance, addressed with the page ids of its fusion size.
struct PagedKV {
  torch::Tensor pool;
  KVGeom g{};
  int type;
  CUtensorMap map;
  bool tiles;   // the tile kernel can read this pool (map is valid)

  PagedKV(torch::Tensor p, int64_t P, int64_t N, int64_t Ls, int64_t L, int64_t block_size, int64_t kvh, int64_t hd)
      : pool(std::move(p)) {
    KUS_CHECK(pool.is_cuda() && pool.is_contiguous(), "pool must be a contiguous CUDA tensor");
    type = elem_type(pool, "pool");
    KUS_CHECK(P > 0 && N > 0 && Ls > 0 && block_size > 0 && kvh > 0, "sizes must be positive");
    KUS_CHECK(L == N * Ls, "layers must be a multiple of the fusion size");
    KUS_CHECK(hd > 0 && hd % 8 == 0, "head_dim must be a multiple of 8, got ", hd);
    KUS_CHECK(reinterpret_cast<uintptr_t>(pool.data_ptr()) % 16 == 0, "pool must start on 16 bytes");
    g.base = reinterpret_cast<char*>(pool.data_ptr());
    g.layer_stride = 4LL * block_size * kvh * hd;
    g.page_stride = g.layer_stride * L;
    const int64_t bytes = pool.numel() * 2;
    KUS_CHECK(bytes >= P * g.page_stride, "pool holds ", bytes, " bytes, its layout needs ", P * g.page_stride);
    KUS_CHECK(bytes / g.layer_stride < (1LL << 31) && N * P < (1LL << 31), "pool has too many pages");
    g.P = (int)P;
    g.N = (int)N;
    g.Ls = (int)Ls;
    g.block_size = (int)block_size;
    g.kvh = (int)kvh;
    g.hd = (int)hd;
    finish_geom(g, bytes - P * g.page_stride);
    c10::cuda::CUDAGuard guard(pool.device());
    tiles = make_cache_tile_map(&map, g, bytes, type);
  }

  int checked_layer(int64_t layer) const {
    KUS_CHECK(layer >= 0 && layer < g.Ls, "layer ", layer, " of ", g.Ls);
    return (int)layer;
  }
  // Per-slot values next to the cache: [pages, kv heads, block_size].
  void check_side(const torch::Tensor& t, torch::ScalarType type, const char* what) const {
    KUS_CHECK(t.device() == pool.device() && t.scalar_type() == type && t.is_contiguous() && t.dim() == 3 &&
                    t.size(0) == g.pages_total && t.size(1) == g.kvh && t.size(2) == g.block_size,
                what, " must be a contiguous ", type, " tensor [", g.pages_total, ", ", g.kvh, ", ", g.block_size,
                "] on ", pool.device(), ", got ", t.scalar_type(), " ", t.sizes());
  }
};

// The work units of one batch, one int32 blob on the device (cache_ops.h has
// their layout; kunserve_b200/ops/plans.py builds and checks them).
struct CachePlan {
  torch::Tensor blob;
  c10::cuda::CUDAStream made_on;
  int T, nq, kvh, block_size, hd, max_page;
  int n_row_units, n_tile_units, head_chunks, most_parts, n_chunks, n_reqs, most_tokens;
  int64_t o_row, o_tile, o_pages, o_off, o_merge, o_chunks, o_reqs;
  int64_t part_rows, score_cols;

  CachePlan(const torch::Tensor& ints, const PagedKV& kv, const std::map<std::string, int64_t>& d)
      : made_on(c10::cuda::getCurrentCUDAStream(kv.pool.get_device())) {
    c10::cuda::CUDAGuard guard(kv.pool.device());
    KUS_CHECK(ints.scalar_type() == torch::kInt32 && ints.dim() == 1 && !ints.is_cuda(), "plan: int32 ints");
    blob = ints.to(kv.pool.device());
    auto at = [&](const char* k) {
      auto it = d.find(k);
      KUS_CHECK(it != d.end(), "plan: no ", k);
      return it->second;
    };
    auto i32 = [&](const char* k) {
      const int64_t v = at(k);
      KUS_CHECK(v >= 0 && v < (1LL << 31), "plan: ", k, " is ", v);
      return (int)v;
    };
    T = i32("tokens");
    nq = i32("num_q_heads");
    kvh = kv.g.kvh;
    block_size = kv.g.block_size;
    hd = kv.g.hd;
    max_page = (int)at("max_page");
    KUS_CHECK(max_page < kv.g.pages_total, "plan: page ", max_page, " of ", kv.g.pages_total);
    n_row_units = i32("row_units");
    n_tile_units = i32("tile_units");
    head_chunks = i32("head_chunks");
    most_parts = i32("most_parts");
    n_chunks = i32("chunks");
    n_reqs = i32("requests");
    most_tokens = i32("most_tokens");
    o_row = at("at_row_units");
    o_tile = at("at_tile_units");
    o_pages = at("at_pages");
    o_off = at("at_merge_off");
    o_merge = at("at_merge");
    o_chunks = at("at_chunks");
    o_reqs = at("at_requests");
    part_rows = i32("part_rows");
    score_cols = i32("score_cols");
    KUS_CHECK((int64_t)n_row_units * kvh < (1LL << 31) - 4 && (int64_t)n_tile_units * kvh < (1LL << 31) &&
                    (int64_t)T * nq + (int64_t)n_chunks * kvh < (1LL << 31) - 4 &&
                    (int64_t)n_reqs * kvh * 8 < (1LL << 31),
                "plan: too many units for one launch");
  }

  const int* ints(int64_t at) const { return blob.data_ptr<int>() + at; }
  // The plan fits this cache, and outlives the work queued on the current stream.
  void use(const PagedKV& kv) const {
    KUS_CHECK(n_tile_units == 0 || kv.tiles, "the plan was made for a cache of another shape");
    KUS_CHECK(kv.g.kvh == kvh && kv.g.block_size == block_size && kv.g.hd == hd && max_page < kv.g.pages_total &&
                    kv.pool.device() == blob.device(),
                "the plan was made for a cache of another shape");
    const auto st = at::cuda::getCurrentCUDAStream(blob.get_device());
    if (st != made_on) blob.record_stream(st);
  }
};

torch::Tensor empty(at::IntArrayRef sizes, torch::ScalarType type, const torch::Device& device) {
  return torch::Tensor(at::detail::empty_cuda(sizes, type, device, {}));
}

void check_index(const torch::Tensor& t, int64_t n, const torch::Tensor& like, const char* what) {
  KUS_CHECK(t.device() == like.device() && t.scalar_type() == torch::kInt32 && t.is_contiguous() && t.numel() == n,
              what, " must be a contiguous int32 tensor of ", n, " on ", like.device());
}

// x or out of an operator: [T, heads, hd], elements of a head contiguous.
void check_heads(const torch::Tensor& t, int64_t T, int64_t heads, int64_t hd, const torch::Tensor& like,
                 const char* what) {
  KUS_CHECK(t.device() == like.device() && t.scalar_type() == like.scalar_type() && t.dim() == 3 &&
                  t.size(0) == T && t.size(1) == heads && t.size(2) == hd && (hd == 1 || t.stride(2) == 1),
              what, " must be a ", like.scalar_type(), " tensor [", T, ", ", heads, ", ", hd, "] on ", like.device(),
              " with contiguous heads, got ", t.scalar_type(), " ", t.sizes(), " strides ", t.strides());
}

// Every head of a 16-bit [T, heads, hd] tensor starts on 16 bytes.
bool heads_on_16(const torch::Tensor& t) {
  return (t.size(0) <= 1 || t.stride(0) % 8 == 0) && (t.size(1) <= 1 || t.stride(1) % 8 == 0) &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// The frequencies of a model's rotary positions (kunserve_b200/ops/rotary.py).
struct RotaryTable {
  torch::Tensor steps;
  c10::cuda::CUDAStream made_on;
  float scale;
  int hd, rot;
  bool interleaved;

  RotaryTable(torch::Tensor s, double scale_, int64_t hd_, bool interleaved_)
      : steps(std::move(s)),
        made_on(c10::cuda::getCurrentCUDAStream(steps.is_cuda() ? steps.get_device() : -1)),
        scale((float)scale_),
        hd((int)hd_),
        rot(0),
        interleaved(interleaved_) {
    KUS_CHECK(steps.is_cuda() && steps.scalar_type() == torch::kInt64 && steps.is_contiguous() && steps.dim() == 1,
              "rotary steps must be a contiguous int64 CUDA tensor");
    const int64_t r = 2 * steps.numel();
    KUS_CHECK(r > 0 && r <= hd_ && r <= 4096, "rotary_dim ", r, " of head_dim ", hd_);
    rot = (int)r;
  }
  // The frequencies outlive the work queued on `st`.
  void use(const c10::cuda::CUDAStream& st) const {
    if (st != made_on) steps.record_stream(st);
  }
};

RotaryArgs rotary_args(const RotaryTable* table, const torch::Tensor& x, const torch::Tensor& positions,
                       const torch::Tensor& out, bool inverse, const c10::cuda::CUDAStream& st) {
  KUS_CHECK(table && table->steps.device() == x.device(), "the rotary frequencies must be on ", x.device());
  const int64_t hd = x.size(2);
  KUS_CHECK(hd == table->hd, "head_dim ", hd, ", the rotary frequencies have ", (int64_t)table->hd);
  check_index(positions, x.size(0), x, "positions");
  table->use(st);
  KUS_CHECK(x.size(0) < (1LL << 31) && x.size(1) * hd < (1 << 23), "too many tokens or heads");
  RotaryArgs a{};
  a.x = x.data_ptr();
  a.xt = x.stride(0);
  a.xh = x.stride(1);
  a.out = out.data_ptr();
  a.ot = out.stride(0);
  a.oh = out.stride(1);
  a.positions = positions.data_ptr<int>();
  a.steps = reinterpret_cast<const unsigned long long*>(table->steps.data_ptr<int64_t>());
  a.scale = table->scale;
  a.sign = inverse ? -1.f : 1.f;
  a.T = (int)x.size(0);
  a.nq = (int)x.size(1);
  a.hd = (int)hd;
  a.rot = table->rot;
  a.interleaved = table->interleaved;
  return a;
}

// None: a gradient is asked for, the caller goes through autograd.
c10::optional<torch::Tensor> rotary_apply_op(const torch::Tensor& x, const torch::Tensor& positions,
                                             const RotaryTable* table, const c10::optional<torch::Tensor>& out,
                                             bool inverse) {
  KUS_CHECK(x.is_cuda() && x.dim() == 3, "x must be a CUDA tensor [T, heads, head_dim]");
  if ((x.requires_grad() || (out.has_value() && out->requires_grad())) && at::GradMode::is_enabled()) {
    TORCH_CHECK_VALUE(!out.has_value(), "results written to out= carry no gradient, but an argument requires one");
    return c10::nullopt;
  }
  const int type = elem_type(x, "x");
  c10::cuda::CUDAGuard guard(x.device());
  check_heads(x, x.size(0), x.size(1), x.size(2), x, "x");
  torch::Tensor o = out.has_value() ? *out : empty(x.sizes(), x.scalar_type(), x.device());
  check_heads(o, x.size(0), x.size(1), x.size(2), x, "out");
  const auto st = at::cuda::getCurrentCUDAStream();
  rotary(rotary_args(table, x, positions, o, inverse, st), type, st);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return o;
}

void rotary_append_op(const torch::Tensor& qkv, const torch::Tensor& positions, const torch::Tensor& pages,
                      const torch::Tensor& slots, const RotaryTable* table, const PagedKV& kv, int64_t layer,
                      const c10::optional<torch::Tensor>& out, const c10::optional<torch::Tensor>& weights,
                      const c10::optional<torch::Tensor>& slot_positions) {
  const KVGeom& g = kv.g;
  c10::cuda::CUDAGuard guard(kv.pool.device());
  KUS_CHECK(qkv.dim() == 3 && qkv.size(1) >= 2 * g.kvh, "qkv must be [T, q heads + 2 * ", (int64_t)g.kvh, ", ",
            (int64_t)g.hd, "]");
  const int64_t T = qkv.size(0), nq = qkv.size(1) - 2 * g.kvh;
  check_heads(qkv, T, nq + 2 * g.kvh, g.hd, kv.pool, "qkv");
  // without `out` the queries turn in place: they lie first in qkv
  if (out.has_value()) check_heads(*out, T, nq, g.hd, kv.pool, "out");
  const auto st = at::cuda::getCurrentCUDAStream();
  RotaryArgs a = rotary_args(table, qkv, positions, out.has_value() ? *out : qkv, false, st);
  check_index(pages, T, qkv, "pages");
  check_index(slots, T, qkv, "slots");
  KUS_CHECK(weights.has_value() == slot_positions.has_value(), "weights and slot_positions come together");
  a.nq = (int)nq;
  a.nkv = g.kvh;
  a.pages = pages.data_ptr<int>();
  a.slots = slots.data_ptr<int>();
  a.g = g;
  a.layer = kv.checked_layer(layer);
  if (weights.has_value()) {
    kv.check_side(*weights, torch::kFloat32, "weights");
    kv.check_side(*slot_positions, torch::kInt32, "slot_positions");
    a.weights = weights->data_ptr<float>();
    a.slot_positions = slot_positions->data_ptr<int>();
  }
  rotary(a, kv.type, st);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

torch::Tensor cached_attention_op(const torch::Tensor& q, const PagedKV& kv, int64_t layer, const CachePlan& plan,
                                  c10::optional<double> scale_arg, const c10::optional<torch::Tensor>& out,
                                  const c10::optional<torch::Tensor>& weights) {
  const double scale = scale_arg.has_value() ? *scale_arg : 1.0 / std::sqrt((double)kv.g.hd);
  plan.use(kv);
  c10::cuda::CUDAGuard guard(kv.pool.device());
  CachedAttn a{};
  a.g = kv.g;
  KUS_CHECK(a.g.hd == 64 || a.g.hd == 128, "attention takes head_dim 64 or 128, the cache has ", a.g.hd);
  KUS_CHECK(scale > 0 && std::isfinite(scale), "scale must be positive");
  check_heads(q, plan.T, plan.nq, a.g.hd, kv.pool, "q");
  KUS_CHECK(heads_on_16(q), "q's heads must start on 16 bytes");
  torch::Tensor o = out.has_value() ? *out
                                    : empty({plan.T, plan.nq, a.g.hd}, kv.pool.scalar_type(), kv.pool.device());
  check_heads(o, plan.T, plan.nq, a.g.hd, kv.pool, "out");
  KUS_CHECK(heads_on_16(o), "out's heads must start on 16 bytes");
  a.layer = kv.checked_layer(layer);
  a.q = q.data_ptr();
  a.qt = q.stride(0);
  a.qh = q.stride(1);
  a.out = o.data_ptr();
  a.ot = o.stride(0);
  a.oh = o.stride(1);
  a.T = plan.T;
  a.nq = plan.nq;
  a.hd = a.g.hd;
  a.scale = (float)scale;
  a.pages = plan.ints(plan.o_pages);
  a.row_units = plan.ints(plan.o_row);
  a.n_row_units = plan.n_row_units;
  a.tile_units = plan.ints(plan.o_tile);
  a.n_tile_units = plan.n_tile_units;
  a.merge_off = plan.ints(plan.o_off);
  a.merge = reinterpret_cast<const int2*>(plan.ints(plan.o_merge));
  a.head_chunks = plan.head_chunks;
  a.most_parts = plan.most_parts;
  // scratch of this call, in fp32: partial sums, (weighted) scores, partial
  // (max, sum) and the rows' statistics; all but the last are read in vectors
  const bool weighted = weights.has_value();
  const int64_t n_o = plan.part_rows * a.g.hd, n_s = weighted ? plan.score_cols * plan.nq : 0,
                n_st = weighted ? 2LL * plan.T * plan.nq : 0;
  const c10::DataPtr scratch =
      c10::cuda::CUDACachingAllocator::get()->allocate(4 * (n_o + n_s + 2 * plan.part_rows + n_st));
  a.part_o = static_cast<float*>(scratch.get());
  a.part_ml = reinterpret_cast<float2*>(a.part_o + n_o + n_s);
  if (weighted) {
    KUS_CHECK(plan.n_reqs > 0 || plan.T == 0, "weights need a decode plan");
    kv.check_side(*weights, torch::kFloat32, "weights");
    a.scores = a.part_o + n_o;
    a.stats = a.part_ml + plan.part_rows;
    a.weights = weights->data_ptr<float>();
    a.chunks = plan.ints(plan.o_chunks);
    a.n_chunks = plan.n_chunks;
  }
  cached_attention(a, &kv.map, kv.type, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return o;
}

std::tuple<torch::Tensor, torch::Tensor> select_evictions_op(const torch::Tensor& weights,
                                                             const torch::Tensor& slot_positions, const PagedKV& kv,
                                                             const CachePlan& plan, int64_t keep, int64_t sinks,
                                                             int64_t recent, int64_t cap) {
  plan.use(kv);
  c10::cuda::CUDAGuard guard(kv.pool.device());
  KUS_CHECK(plan.n_reqs > 0 || plan.T == 0, "eviction needs a decode plan");
  KUS_CHECK(keep > 0 && keep < (1LL << 31) && cap >= 0 && cap <= keep, "keep must be positive, got ", keep);
  KUS_CHECK(sinks >= 0 && recent >= 0 && sinks <= keep && recent <= keep - sinks, "sinks (", sinks, ") and recent (", recent,
              ") must fit in keep (", keep, ")");
  kv.check_side(weights, torch::kFloat32, "weights");
  kv.check_side(slot_positions, torch::kInt32, "slot_positions");
  torch::Tensor moves = empty({plan.n_reqs, kv.g.kvh, cap, 2}, torch::kInt32, kv.pool.device());
  torch::Tensor counts = empty({plan.n_reqs, kv.g.kvh}, torch::kInt32, kv.pool.device());
  EvictSelect a{};
  a.weights = weights.data_ptr<float>();
  a.slot_positions = slot_positions.data_ptr<int>();
  a.g = kv.g;
  a.pages = plan.ints(plan.o_pages);
  a.reqs = plan.ints(plan.o_reqs);
  a.n_reqs = plan.n_reqs;
  a.most_tokens = plan.most_tokens;
  a.keep = (int)keep;
  a.sinks = (int)sinks;
  a.recent = (int)recent;
  a.cap = (int)cap;
  a.moves = reinterpret_cast<int2*>(moves.data_ptr<int>());
  a.counts = counts.data_ptr<int>();
  evict_select(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {moves, counts};
}

void compact_cache_op(const PagedKV& kv, int64_t layer, const CachePlan& plan, const torch::Tensor& moves,
                      const torch::Tensor& counts, const c10::optional<torch::Tensor>& weights,
                      const c10::optional<torch::Tensor>& slot_positions) {
  plan.use(kv);
  c10::cuda::CUDAGuard guard(kv.pool.device());
  CacheCompact a{};
  a.g = kv.g;
  KUS_CHECK(kv.pool.numel() / kv.g.hd < (1LL << 31), "the pool has too many rows of head_dim ", kv.g.hd);
  a.layer = kv.checked_layer(layer);
  KUS_CHECK(moves.device() == kv.pool.device() && moves.scalar_type() == torch::kInt32 && moves.is_contiguous() &&
                  moves.dim() == 4 && moves.size(0) == plan.n_reqs && moves.size(1) == a.g.kvh && moves.size(3) == 2,
              "moves must be a contiguous int32 tensor [", plan.n_reqs, ", ", a.g.kvh, ", most, 2], got ",
              moves.sizes());
  check_index(counts, (int64_t)plan.n_reqs * a.g.kvh, kv.pool, "counts");
  KUS_CHECK((int64_t)plan.n_reqs * a.g.kvh * (moves.size(2) / 32 + 1) < (1LL << 31), "too many moves for one launch");
  a.pages = plan.ints(plan.o_pages);
  a.reqs = plan.ints(plan.o_reqs);
  a.n_reqs = plan.n_reqs;
  a.cap = (int)moves.size(2);
  a.moves = reinterpret_cast<const int2*>(moves.data_ptr<int>());
  a.counts = counts.data_ptr<int>();
  if (weights.has_value()) {
    kv.check_side(*weights, torch::kFloat32, "weights");
    a.weights = weights->data_ptr<float>();
  }
  if (slot_positions.has_value()) {
    kv.check_side(*slot_positions, torch::kInt32, "slot_positions");
    a.slot_positions = slot_positions->data_ptr<int>();
  }
  cache_compact(a, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace

void bind_cache_ops(py::module& m) {
  py::class_<PagedKV>(m, "PagedKV")
      .def(py::init<torch::Tensor, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t>())
      .def_property_readonly("pages_total", [](const PagedKV& k) { return k.g.pages_total; })
      .def_property_readonly("block_size", [](const PagedKV& k) { return k.g.block_size; })
      .def_property_readonly("num_kv_heads", [](const PagedKV& k) { return k.g.kvh; })
      .def_property_readonly("head_dim", [](const PagedKV& k) { return k.g.hd; })
      .def_property_readonly("tiles", [](const PagedKV& k) { return k.tiles; })
      .def_property_readonly("pool", [](const PagedKV& k) { return k.pool; });
  py::class_<CachePlan>(m, "CachePlan")
      .def(py::init<const torch::Tensor&, const PagedKV&, const std::map<std::string, int64_t>&>());
  py::class_<RotaryTable>(m, "RotaryTable").def(py::init<torch::Tensor, double, int64_t, bool>());
  m.def("rotary_apply", &rotary_apply_op);
  m.def("rotary_append_scaled", &rotary_append_op);
  m.def("cached_attention", &cached_attention_op);
  m.def("select_evictions", &select_evictions_op);
  m.def("compact_cache", &compact_cache_op);
  // what ops/plans.py lays plans out by
  py::dict c;
  c["UNIT_INTS"] = kUnitInts;
  c["ROW_UNIT_ROWS"] = kRowUnitRows;
  c["TILE_UNIT_ROWS"] = kTileUnitRows;
  c["STAGE_KEYS"] = kStageKeys;
  c["TILE_KEYS"] = kTileKeys;
  c["CHUNK_KEYS"] = kChunkKeys;
  c["NO_LIMIT"] = kNoLimit;
  m.attr("PLAN_CONSTANTS") = c;
}
