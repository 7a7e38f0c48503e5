// Rows written as 8-bit integers with one scale each, and back.
//
//   quantize  y = x
//   norm      h = x + r,  y = h / sqrt(mean h^2 + eps) * w;  h is kept too
//   silu      y = g / (1 + e^-g) * u
//   scale = max|y| / 127,  q = the integer nearest to 127 y / max|y|
//
// The norm's factor is common to a row, so max|y| = rstd max|h w| and
// q = rint(127 h w / max|h w|): sum h^2 and max|h w| come from one reduction
// over registers, and each element is read once and written once.
//
// Bound by HBM and, nearly as much, by instructions: 8192 rows of 5120 in
// bf16 take 24 us to quantise (126 MB, 13 instructions an element, most of the
// issue slots), 48 to add and norm (294 MB at 0.93 of the copy bandwidth), 34
// with SiLU (210 MB), 21 back (126 MB).  So integers come out of the adder
// (Quotient), inputs of a quantisation stay as they are until they are
// written, and a thread has 16 to 32 elements to share the reduction's cost.
// All loads of a row are issued ahead of its arithmetic; a persistent block
// that prefetched its next rows into shared memory was no faster.
#include <algorithm>
#include <type_traits>

#include "../common.cuh"
#include "cache_elem.cuh"
#include "int8_ops.h"

namespace kus {
namespace i8rows {

// max that keeps a NaN
KUS_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Pairs of floats in one instruction each.
struct Pair {
  unsigned long long v;
  KUS_DEVICE Pair(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  KUS_DEVICE explicit Pair(float a) : Pair(a, a) {}
  KUS_DEVICE float2 get() const {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
  }
};
KUS_DEVICE Pair operator*(Pair a, const Pair& b) {
  asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
KUS_DEVICE Pair operator+(Pair a, const Pair& b) {
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a.v) : "l"(b.v));
  return a;
}
KUS_DEVICE Pair fma(Pair a, const Pair& b, const Pair& c) {
  asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(a.v) : "l"(b.v), "l"(c.v));
  return a;
}

// g / (1 + e^-g) * u of two gates above -kWide.  e^-g = 2^n e^d: n is -g log2 e
// as the exponential takes it, d what that leaves out, without which y would be
// off by 1.2 |g| units more.  Of bf16, n is exact with log2 e in 16 bits, d the
// rest's product, up to 3.2e-4, and 1 + d is e^d to its square; of fp16, n is
// rounded, and d has the product's rounding and log2 e's.  y is off by at most
// 11 * 2^-24 of itself: 2^n by 4 (two units), d's square, the product with 1 + d
// and the sum by 1 each, the reciprocal by 2, two products by 1 each.  (Beyond
// 2e38 n is an infinity and e^-g zero.)  Over all gates of both types the scale
// of a row is off by 4.8 at most.  8192 rows of 14336 take 104 us with this
// (bf16; 100 in fp16), 103 (108) with e^-g of a rounded n alone.
constexpr float kWide = 64.f;
template <typename T>
KUS_DEVICE void silu_pair(float& g0, float& g1, float u0, float u1) {
  const Pair g(g0, g1);
  Pair n = g, d = g;
  if constexpr (std::is_same<T, __half>::value) {
    constexpr float kLog2e = 0x1.715476p+0f, kRest = 0x1.4ae0bep-26f, kLn2 = 0x1.62e430p-1f;
    n = g * Pair(-kLog2e);
    d = fma(g, Pair(kRest), fma(g, Pair(kLog2e), n)) * Pair(-kLn2);
  } else {
    constexpr float kLog2e = 0x1.7154p+0f, kRestLn2 = 0x1.480fb6p-18f;
    n = g * Pair(-kLog2e);
    d = g * Pair(-kRestLn2);
  }
  const float2 m = n.get();
  const Pair e(ex2(m.x), ex2(m.y));
  float2 r = (fma(e, d, e) + Pair(1.f)).get();
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r.x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r.y));
  const float2 y = (g * Pair(r.x, r.y) * Pair(u0, u1)).get();
  g0 = y.x;
  g1 = y.y;
}
// y of a gate that silu_pair does not know: below -kWide e^-g may leave the range
// where y does not.  Of one exponential as a square: off by 11 * 2^-24 of itself
// too (4 for each, three products).
KUS_DEVICE float silu_wide(float g, float u) {
  const float h = expf(0.5f * g);
  return (g * h) * (u * h);
}

// The largest of non-negative floats, NaN above all: their bits' order.
KUS_DEVICE float warp_top(float v) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

KUS_DEVICE float top_of(const float (&f)[8]) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max_nan(m, fabsf(f[e]));
  return m;
}

// 8 neighbours of a row as they lie in memory.
template <typename T>
struct Raw8 {
  using V2 = typename Elem<T>::V2;
  uint4 u;
  KUS_DEVICE void load(const T* p, bool there) {
    u = there ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
  }
  KUS_DEVICE void values(float (&f)[8]) const { unpack8<T>(u, f); }
  // largest magnitude, NaN above all
  KUS_DEVICE float top() const {
    const V2* v = reinterpret_cast<const V2*>(&u);
    const V2 m = __hmax2_nan(__hmax2_nan(__habs2(v[0]), __habs2(v[1])), __hmax2_nan(__habs2(v[2]), __habs2(v[3])));
    const float2 f = Elem<T>::to_f2(m);
    return max_nan(f.x, f.y);
  }
};
template <>
struct Raw8<float> {
  float4 a, b;
  KUS_DEVICE void load(const float* p, bool there) {
    a = there ? reinterpret_cast<const float4*>(p)[0] : make_float4(0, 0, 0, 0);
    b = there ? reinterpret_cast<const float4*>(p)[1] : make_float4(0, 0, 0, 0);
  }
  KUS_DEVICE void values(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  }
  KUS_DEVICE float top() const {
    float f[8];
    values(f);
    return top_of(f);
  }
};

template <typename T>
KUS_DEVICE float to_float(T x) { return Elem<T>::to_f(x); }
template <>
KUS_DEVICE float to_float<float>(float x) { return x; }
template <typename T>
KUS_DEVICE T from_float(float x) { return Elem<T>::from_f(x); }
template <>
KUS_DEVICE float from_float<float>(float x) { return x; }

// 16 bytes from byte `by` (below 16) of 32.
KUS_DEVICE uint4 shifted(const uint4& a, const uint4& b, int by) {
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (by & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (by & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  const int bits = (by & 3) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                    __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// 8 neighbours from column c of a 16-bit row that starts anywhere: inside the
// row from the two aligned vectors that hold them (both lie in the row), at
// its ends one by one.
template <typename T>
KUS_DEVICE uint4 load_anywhere(const T* row, int c, int K) {
  if (c >= 8 && c + 16 <= K) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + c);
    const int by = (int)(at & 15);
    const uint4* p = reinterpret_cast<const uint4*>(at - by);
    const uint4 a = p[0];
    return by ? shifted(a, p[1], by) : a;
  }
  uint32_t w[4] = {0, 0, 0, 0};
  for (int e = 0; e < 8; ++e)
    if (c + e < K) w[e / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(row)[c + e] << (16 * (e & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The same for writing, by a whole warp whose lanes hold neighbouring groups
// of 8: a lane writes the aligned vector that its group and the next lane's
// share; what is left at the warp's and the row's ends goes one by one.
template <typename T>
KUS_DEVICE void store_anywhere(T* row, int c, int K, const uint4& v) {
  T* p = row + c;
  const int by = (int)(reinterpret_cast<uintptr_t>(p) & 15), head = by ? 8 - by / 2 : 8;    // elements before the vector
  const uint4 next = make_uint4(__shfl_down_sync(0xffffffffu, v.x, 1), __shfl_down_sync(0xffffffffu, v.y, 1),
                                __shfl_down_sync(0xffffffffu, v.z, 1), __shfl_down_sync(0xffffffffu, v.w, 1));
  const int lane = threadIdx.x % 32;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  auto one_by_one = [&](int from, int to) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e >= from && e < to && c + e < K)
        reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
  };
  if (by == 0) {
    if (c + 8 <= K)
      *reinterpret_cast<uint4*>(p) = v;
    else
      one_by_one(0, 8);
    return;
  }
  if (lane == 0 || c + head > K) one_by_one(0, head);
  if (lane < 31 && c + head + 8 <= K)
    *reinterpret_cast<uint4*>(p + head) = shifted(v, next, 16 - by);
  else
    one_by_one(head, 8);
}

// First column of vector j of a thread.  Rows that start elsewhere than on 16
// bytes are read element by element, but each by the same thread: the order
// of the norm's sum, and so its bits, do not depend on strides.
KUS_DEVICE int column(int j, int lane, int lanes) { return (j * lanes + lane) * 8; }

template <typename T, int OP>
struct Row {
  const T* x;
  const T* other;
  const T* weight;
  T* total;
  int K;

  KUS_DEVICE Row(const Int8Rows& a, long long t)
      : x(reinterpret_cast<const T*>(a.x) + t * a.xs),
        other(a.other ? reinterpret_cast<const T*>(a.other) + t * a.os : nullptr),
        weight(reinterpret_cast<const T*>(a.weight)),
        total(a.total ? reinterpret_cast<T*>(a.total) + t * a.ts : nullptr),
        K(a.K) {}

  // y of 8 columns (the norm's without its common factor) from their inputs,
  // y holding x; `sum` gains h^2.
  KUS_DEVICE static void combine(float (&y)[8], const float (&w)[8], float& sum) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sum = fmaf(y[e], y[e], sum);
      y[e] *= w[e];
    }
  }
  // `least` gains the gates' least, negated; with one below -kWide y stays undone.
  // (The branch for each group also keeps a group's arithmetic ahead of later
  // groups' loads: 8192 x 14336 takes 5 us less than without.)
  KUS_DEVICE static void gate(float (&y)[8], const float (&o)[8], float& least) {
#pragma unroll
    for (int e = 0; e < 8; ++e) least = fmaxf(least, -y[e]);
    if (least > kWide) return;
#pragma unroll
    for (int e = 0; e < 8; e += 2) silu_pair<T>(y[e], y[e + 1], o[e], o[e + 1]);
  }
  // Any gates, each by its own formula.
  KUS_DEVICE static void gate_any(float (&y)[8], const float (&o)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float g0 = y[e], g1 = y[e + 1];
      silu_pair<T>(y[e], y[e + 1], o[e], o[e + 1]);
      if (g0 < -kWide) y[e] = silu_wide(g0, o[e]);
      if (g1 < -kWide) y[e + 1] = silu_wide(g1, o[e + 1]);
    }
  }

  // Element by element; `keep`: write x + residual.
  KUS_DEVICE void values(int c0, bool keep, float (&y)[8], float& sum) const {
    float o[8], w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = c0 + e;
      y[e] = o[e] = w[e] = 0.f;
      if (c >= K) continue;
      y[e] = to_float<T>(x[c]);
      if (OP == kRowsSilu || (OP == kRowsNorm && other)) o[e] = to_float<T>(other[c]);
      if (OP == kRowsNorm) w[e] = to_float<T>(weight[c]);
      if (OP == kRowsNorm && other) {
        y[e] += o[e];
        if (keep) total[c] = from_float<T>(y[e]);
      }
    }
    if (OP == kRowsNorm) combine(y, w, sum);
    if (OP == kRowsSilu) gate_any(y, o);
  }
};

// The integers nearest to 127 v / top, two's complement, in the low bytes:
// adding 1.5 * 2^23 rounds to a whole number and leaves it in the low bits (a
// conversion runs at a quarter of the rate).  127 / top is held in two floats,
// its rounding and what that left out, so that v times it is off by half a
// step and 2^-47 of itself: where 127 v / top is a float, a half say, the
// product is that float, and halves of quantised inputs go to even.  Computed
// values have roundings of their own; they take the first float alone.
struct Quotient {
  float high, low, small;
  KUS_DEVICE Quotient(float top, bool sound) {
    // 127 / top and its rest stay in range
    small = top > 1e30f ? 0x1p-30f : top < 1e-30f ? 0x1p60f : 1.f;
    const float over = sound && top > 0.f ? top * small : 1.f;
    high = 127.f / over;
    low = fmaf(-high, over, 127.f) / over;
  }
  KUS_DEVICE uint32_t near(float v) const { return __float_as_uint(fmaf(v, high, 12582912.f)); }
  KUS_DEVICE uint32_t nearest(float v) const { return __float_as_uint(fmaf(v, high, v * low) + 12582912.f); }
};

// Of squares the sum, of SiLU's gates the largest magnitude, and of values the
// largest: over the warp, and over the block through `part` (32 entries, not written
// again before every thread has read them).
KUS_DEVICE void reduce_warp(int op, float& sum, float& top) {
  if (op == kRowsNorm) sum = warp_sum(sum);
  if (op == kRowsSilu) sum = warp_top(sum);
  top = warp_top(top);
}
KUS_DEVICE void reduce_block(int op, float& sum, float& top, float2* part) {
  const int l = threadIdx.x % 32;
  if (l == 0) part[threadIdx.x / 32] = make_float2(sum, top);
  __syncthreads();
  const float2 p = l < blockDim.x / 32 ? part[l] : make_float2(0.f, 0.f);
  sum = p.x;
  top = p.y;
  reduce_warp(op, sum, top);
}

// The largest scale whose 127-fold is finite: the float nearest to the largest
// float / 127 is one above.
constexpr float kMostScale = 0x810203p98f;

// A row's scale, and its integers.  A row without finite values has scale NaN.
template <int OP>
struct Writer {
  int8_t* q;
  int K;
  bool sound;
  Quotient quotient;

  KUS_DEVICE static float factor(const Int8Rows& a, float sum) {
    return OP == kRowsNorm ? rsqrtf(sum / (float)a.K + a.eps) : 1.f;
  }
  // Whether the row's values are finite.  Of a norm the factor counts, at most
  // 2.7e22 (of the least eps): its cost is met by rows beyond 1e16 alone.
  KUS_DEVICE static bool finite(const Int8Rows& a, float sum, float top) {
    if (OP == kRowsNorm && top > 1e16f) return sum < INFINITY && top * factor(a, sum) < INFINITY;
    return top < INFINITY && (OP != kRowsNorm || sum < INFINITY);
  }
  KUS_DEVICE Writer(const Int8Rows& a, long long t, float sum, float top, bool first)
      : q(a.q + t * a.qs), K(a.K), sound(finite(a, sum, top)), quotient(top, sound) {
    if (first) a.scales[t] = sound ? fminf(top / 127.f * factor(a, sum), kMostScale) : NAN;
  }
  KUS_DEVICE void integers(const float (&v)[8], uint32_t (&r)[8]) const {
    if (quotient.small != 1.f) {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = quotient.nearest(v[e] * quotient.small);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = OP == kRowsQuantize ? quotient.nearest(v[e]) : quotient.near(v[e]);
    }
  }
  // 8 columns from c, a multiple of 8 (rows of q start on 16 bytes).
  KUS_DEVICE void write(int c, const float (&v)[8]) const {
    if (c >= K) return;
    uint32_t r[8];
    integers(v, r);
    uint2 u;
    u.x = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
    u.y = __byte_perm(__byte_perm(r[4], r[5], 0x0040), __byte_perm(r[6], r[7], 0x0040), 0x5410);
    if (!sound) u = make_uint2(0, 0);
    if (c + 8 <= K) {
      *reinterpret_cast<uint2*>(q + c) = u;
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (c + e < K) q[c + e] = (int8_t)((e < 4 ? u.x : u.y) >> (8 * (e % 4)));
    }
  }
};

// A row in registers: HELD vectors of 8 a thread, the inputs of a quantisation
// as they came, else y.
// ANYWHERE: rows that start on any element (16 bits).
template <typename T, int OP, int HELD, bool ANYWHERE>
struct Held {
  Raw8<T> raw[OP == kRowsQuantize ? HELD : 1];
  float y[OP == kRowsQuantize ? 1 : HELD][8];

  KUS_DEVICE static void load(Raw8<T>& r, const T* row, int c, int K) {
    if constexpr (ANYWHERE)
      r.u = load_anywhere(row, c, K);
    else
      r.load(row + c, c < K);
  }
  KUS_DEVICE void read(const Row<T, OP>& row, int lane, int lanes, float& sum, float& top) {
    constexpr int kOther = OP == kRowsQuantize ? 1 : HELD;
    Raw8<T> x[HELD], o[kOther];
    const bool two = OP == kRowsSilu || (OP == kRowsNorm && row.other);
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      const int c = column(j, lane, lanes);
      load(x[j], row.x, c, row.K);
      if (OP != kRowsQuantize && two) load(o[j % kOther], row.other, c, row.K);
    }
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      if constexpr (OP == kRowsQuantize) {
        raw[j] = x[j];
        top = max_nan(top, x[j].top());
      } else {
        float f[8];
        x[j].values(y[j]);
        if (two) o[j].values(f);
        if constexpr (OP == kRowsNorm) {
          if (two) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[j][e] += f[e];
            const int c = column(j, lane, lanes);
            if constexpr (ANYWHERE)
              store_anywhere(row.total, c, row.K, pack8<T>(y[j]));
            else if (c < row.K)
              *reinterpret_cast<uint4*>(row.total + c) = pack8<T>(y[j]);
          }
          Raw8<T> w;
          load(w, row.weight, column(j, lane, lanes), row.K);
          w.values(f);
          Row<T, OP>::combine(y[j], f, sum);
        } else {
          Row<T, OP>::gate(y[j], f, sum);
        }
        top = max_nan(top, top_of(y[j]));
      }
    }
  }
  KUS_DEVICE void write(const Writer<OP>& writer, int lane, int lanes) const {
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      float v[8];
      if constexpr (OP == kRowsQuantize) {
        raw[j].values(v);
        writer.write(column(j, lane, lanes), v);
      } else {
        writer.write(column(j, lane, lanes), y[j]);
      }
    }
  }
};

// SiLU of a row with any gates, read twice: 8192 rows of 14336 with one gate of
// -90 each take 236 us.  (Done where such a gate is met, it took the registers
// of rows under way.)
template <typename T, bool ONE_WARP, bool ANYWHERE>
KUS_DEVICE void row_of_any_gates(const Int8Rows& a, long long t, int lane, int lanes, float2* part) {
  const Row<T, kRowsSilu> row(a, t);
  auto group = [&](int c, float (&y)[8]) {
    Raw8<T> x, o;
    float f[8];
    Held<T, kRowsSilu, 1, ANYWHERE>::load(x, row.x, c, a.K);
    Held<T, kRowsSilu, 1, ANYWHERE>::load(o, row.other, c, a.K);
    x.values(y);
    o.values(f);
    row.gate_any(y, f);
  };
  float none = 0.f, top = 0.f, y[8];
#pragma unroll 1
  for (int c = lane * 8; c < a.K; c += lanes * 8) {
    group(c, y);
    top = max_nan(top, top_of(y));
  }
  reduce_warp(kRowsSilu, none, top);
  if (!ONE_WARP) {
    __syncthreads();
    reduce_block(kRowsSilu, none, top, part);
  }
  const Writer<kRowsSilu> writer(a, t, 0.f, top, lane == 0);
#pragma unroll 1
  for (int c = lane * 8; c < a.K; c += lanes * 8) {
    group(c, y);
    writer.write(c, y);
  }
}

// One row a warp (ONE_WARP; eight of them a block) or a block.
template <typename T, int OP, bool ONE_WARP, int HELD, bool ANYWHERE>
KUS_DEVICE void one_row(const Int8Rows& a) {
  __shared__ float2 part[32];
  pdl_wait();
  pdl_trigger();
  const int lanes = ONE_WARP ? 32 : blockDim.x, lane = ONE_WARP ? threadIdx.x % 32 : threadIdx.x;
  const long long t = ONE_WARP ? (long long)blockIdx.x * 8 + threadIdx.x / 32 : blockIdx.x;
  if (ONE_WARP && t >= a.T) return;
  float sum = 0.f, top = 0.f;
  Held<T, OP, HELD, ANYWHERE> held;
  held.read(Row<T, OP>(a, t), lane, lanes, sum, top);
  reduce_warp(OP, sum, top);
  if (!ONE_WARP) reduce_block(OP, sum, top, part);
  if (OP == kRowsSilu && sum > kWide)      // gates that silu_pair does not know
    return row_of_any_gates<T, ONE_WARP, ANYWHERE>(a, t, lane, lanes, part);
  held.write(Writer<OP>(a, t, sum, top, lane == 0), lane, lanes);
}
template <typename T, int OP, bool ONE_WARP, int HELD, bool ANYWHERE>
__global__ void __launch_bounds__(ONE_WARP ? 256 : 1024) rows_kernel(Int8Rows a) {
  one_row<T, OP, ONE_WARP, HELD, ANYWHERE>(a);
}
// A quantisation in 16 bits: in 40 registers a thread more rows are under way
// (8192 x 14336: 64 us, 79 in the 45 that it would take).
template <typename T, bool ONE_WARP, int HELD, bool ANYWHERE>
__global__ void __maxnreg__(40) quantize_kernel(Int8Rows a) {
  one_row<T, kRowsQuantize, ONE_WARP, HELD, ANYWHERE>(a);
}
// SiLU of long rows, in 56: where that is a block more on an SM than the 60 that
// it would take (8192 x 11008 in fp16: 80 us, 93 in 60; 8192 x 14336 in bf16,
// two blocks either way: 105 and 103).
template <typename T, bool ANYWHERE>
__global__ void __maxnreg__(56) silu_kernel(Int8Rows a) {
  one_row<T, kRowsSilu, false, 4, ANYWHERE>(a);
}

// Any row, read twice and element by element, a row a block: what is too long
// for registers, and fp32 that does not start on 16 bytes.
template <typename T, int OP>
__global__ void __launch_bounds__(1024) any_rows_kernel(Int8Rows a) {
  __shared__ float2 part[32];
  pdl_wait();
  pdl_trigger();
  const long long t = blockIdx.x;
  const Row<T, OP> row(a, t);
  float sum = 0.f, top = 0.f, y[8];
  for (int c = threadIdx.x * 8; c < a.K; c += blockDim.x * 8) {
    row.values(c, false, y, sum);
    top = max_nan(top, top_of(y));
  }
  reduce_warp(OP, sum, top);
  reduce_block(OP, sum, top, part);
  const Writer<OP> writer(a, t, sum, top, threadIdx.x == 0);
  // the sum x + residual is written in the second pass: it may lie over either of them
  for (int c = threadIdx.x * 8; c < a.K; c += blockDim.x * 8) {
    float unused = 0.f;
    row.values(c, true, y, unused);
    writer.write(c, y);
  }
}

template <typename T, int OP, bool ONE_WARP, int HELD>
void launch(const Int8Rows& a, bool vec, cudaStream_t s) {
  const int threads = ONE_WARP ? 256 : ((a.K + 8 * HELD - 1) / (8 * HELD) + 31) / 32 * 32;
  const dim3 grid((unsigned)(ONE_WARP ? (a.T + 7) / 8 : a.T));
  if constexpr (std::is_same<T, float>::value) {
    launch_k(rows_kernel<T, OP, ONE_WARP, HELD, false>, grid, dim3(threads), 0, s, a);
  } else if constexpr (OP == kRowsQuantize) {
    launch_k(vec ? quantize_kernel<T, ONE_WARP, HELD, false> : quantize_kernel<T, ONE_WARP, HELD, true>, grid,
             dim3(threads), 0, s, a);
  } else {
    if constexpr (OP == kRowsSilu && HELD == 4) {
      // warps that an SM's registers hold, 64 and 56 a thread
      const int warps = threads / 32;
      if (36 / warps > 32 / warps)
        return launch_k(vec ? silu_kernel<T, false> : silu_kernel<T, true>, grid, dim3(threads), 0, s, a);
    }
    launch_k(vec ? rows_kernel<T, OP, ONE_WARP, HELD, false> : rows_kernel<T, OP, ONE_WARP, HELD, true>, grid,
             dim3(threads), 0, s, a);
  }
}

bool on16(const void* p, long long stride, int bytes, int rows) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows <= 1 || stride * bytes % 16 == 0);
}

template <typename T, int OP>
void launch_op(const Int8Rows& a, cudaStream_t s) {
  const int el = sizeof(T);
  const bool vec = a.K % 8 == 0 && on16(a.x, a.xs, el, a.T) && (!a.other || on16(a.other, a.os, el, a.T)) &&
                   (!a.weight || on16(a.weight, 0, el, 1)) && (!a.total || on16(a.total, a.ts, el, a.T));
  const int n = (a.K + 7) / 8;
  if (n > 4096 || (!vec && std::is_same<T, float>::value)) {
    const int threads = std::min(1024, ((n + 3) / 4 + 31) / 32 * 32);
    launch_k(any_rows_kernel<T, OP>, dim3((unsigned)a.T), dim3(threads), 0, s, a);
    return;
  }
  // Vectors a thread: 8192 rows of 5120, us, 1 / 2 / 4: quantise - / 25.6 /
  // 24.6, norm 52.0 / 46.6 / 46.8, silu 41.2 / 43.3 / 33.9; 2048 rows of 4096:
  // 6.5 / 5.7 / 5.9, 12.1 / 11.5 / 12.5, 9.5 / 9.9 / 8.9.
  if (n <= 32) return launch<T, OP, true, 1>(a, vec, s);
  if (n <= 64) return launch<T, OP, true, 2>(a, vec, s);
  if (n <= (OP == kRowsNorm ? 1024 : 256)) return launch<T, OP, false, 2>(a, vec, s);
  return launch<T, OP, false, 4>(a, vec, s);
}

// The float of byte i of u, whose bytes are integers with their top bit
// turned over: 2^23 + 128 + q, less 2^23 + 128.  (A conversion runs at a
// quarter of the rate.)
KUS_DEVICE float value(uint32_t u, int i) { return __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + i)) - 8388736.f; }

// The 8 values of two words of integers.
KUS_DEVICE void values8(uint2 u, float s, float (&f)[8]) {
  u.x ^= 0x80808080u;
  u.y ^= 0x80808080u;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = value(e < 4 ? u.x : u.y, e % 4) * s;
}

// A row a block.  VEC: whole vectors, four groups of 8 elements a thread and
// step, a block's width apart: a warp's store is one piece (each of two that
// write 16 neighbours a thread fills half of the sectors that it touches), and
// four loads are on their way at once.  8192 rows of 14336, us: one group 75,
// two 62, four 54 (352 MB at the copy bandwidth), 16 neighbours 60.
constexpr int kGroups = 4;
template <typename T, bool VEC>
__global__ void __launch_bounds__(512) values_kernel(Int8Values a) {
  pdl_wait();
  pdl_trigger();
  const long long t = blockIdx.x;
  const int8_t* q = a.q + t * a.qs;
  T* out = reinterpret_cast<T*>(a.out) + t * a.os;
  const float s = a.scales[t];
  const int at = blockIdx.y * blockDim.x + threadIdx.x, step = gridDim.y * blockDim.x;
  if (VEC) {
    for (int c0 = at * 8; c0 < a.K; c0 += kGroups * step * 8) {
      uint2 u[kGroups];
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int c = c0 + g * step * 8;
        u[g] = c < a.K ? *reinterpret_cast<const uint2*>(q + c) : make_uint2(0, 0);
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const int c = c0 + g * step * 8;
        if (c >= a.K) continue;
        float f[8];
        values8(u[g], s, f);
        if constexpr (std::is_same<T, float>::value) {
          reinterpret_cast<float4*>(out + c)[0] = make_float4(f[0], f[1], f[2], f[3]);
          reinterpret_cast<float4*>(out + c)[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
          *reinterpret_cast<uint4*>(out + c) = pack8<T>(f);
        }
      }
    }
  } else if constexpr (std::is_same<T, float>::value) {
    for (int c = at; c < a.K; c += step) out[c] = (float)q[c] * s;
  } else {
    // 8 elements a thread, integers and results on any byte and element; whole warps
    for (int c = at * 8; c - (int)(threadIdx.x % 32) * 8 < a.K; c += step * 8) {
      uint2 u = make_uint2(0, 0);
      if (c + 8 <= a.K && (reinterpret_cast<uintptr_t>(q + c) & 7) == 0) {
        u = *reinterpret_cast<const uint2*>(q + c);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < a.K) (e < 4 ? u.x : u.y) |= (uint32_t)(uint8_t)q[c + e] << (8 * (e % 4));
      }
      float f[8];
      values8(u, s, f);
      store_anywhere(out, c, a.K, pack8<T>(f));
    }
  }
}

template <typename T>
void launch_values(const Int8Values& a, cudaStream_t s) {
  const bool vec = a.K % 8 == 0 && on16(a.out, a.os, sizeof(T), a.T) &&
                   reinterpret_cast<uintptr_t>(a.q) % 8 == 0 && (a.T <= 1 || a.qs % 8 == 0);
  const int items = vec ? (a.K / 8 + kGroups - 1) / kGroups : std::is_same<T, float>::value ? a.K : (a.K + 7) / 8;
  const int y = (items + 511) / 512, threads = ((items + y - 1) / y + 31) / 32 * 32;
  const dim3 grid((unsigned)a.T, (unsigned)(y < 64 ? y : 64));
  if (vec)
    launch_k(values_kernel<T, true>, grid, dim3(threads), 0, s, a);
  else
    launch_k(values_kernel<T, false>, grid, dim3(threads), 0, s, a);
}

}  // namespace i8rows

void int8_rows(const Int8Rows& a, cudaStream_t s) {
  using namespace i8rows;
  if (a.T == 0) return;
  LaunchBehind behind;
  switch (a.op) {
    case kRowsNorm:
      if (a.type == kInt8TypeBF16) return launch_op<__nv_bfloat16, kRowsNorm>(a, s);
      return launch_op<__half, kRowsNorm>(a, s);
    case kRowsSilu:
      if (a.type == kInt8TypeBF16) return launch_op<__nv_bfloat16, kRowsSilu>(a, s);
      return launch_op<__half, kRowsSilu>(a, s);
    default:
      if (a.type == kInt8TypeBF16) return launch_op<__nv_bfloat16, kRowsQuantize>(a, s);
      if (a.type == kInt8TypeFP16) return launch_op<__half, kRowsQuantize>(a, s);
      return launch_op<float, kRowsQuantize>(a, s);
  }
}

void int8_values(const Int8Values& a, cudaStream_t s) {
  using namespace i8rows;
  if (a.T == 0) return;
  LaunchBehind behind;
  if (a.type == kInt8TypeBF16) return launch_values<__nv_bfloat16>(a, s);
  if (a.type == kInt8TypeFP16) return launch_values<__half>(a, s);
  return launch_values<float>(a, s);
}

}  // namespace kus
