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

// 1 / x to one step
KUS_DEVICE float rcp(float x) {
  float r;
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// 8 elements from 16-byte vectors
template <typename T>
KUS_DEVICE void load8(const T* p, float (&f)[8]) {
  unpack8<T>(*reinterpret_cast<const uint4*>(p), f);
}
template <>
KUS_DEVICE void load8<float>(const float* p, float (&f)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
  f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
template <typename T>
KUS_DEVICE float to_float(T x) { return Elem<T>::to_f(x); }
template <>
KUS_DEVICE float to_float<float>(float x) { return x; }
template <typename T>
KUS_DEVICE T from_float(float x) { return Elem<T>::from_f(x); }
template <>
KUS_DEVICE float from_float<float>(float x) { return x; }

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

  // The row's values (the norm's without its common factor) of 8 columns;
  // `sum` gains h^2.  `keep`: write x + residual.
  template <bool VEC>
  KUS_DEVICE void values(int j, int lane, int lanes, bool keep, float (&y)[8], float& sum) const {
    float o[8], w[8];
    if (VEC) {
      const int c = column(j, lane, lanes);
      if (c >= K) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = 0.f;
        return;
      }
      load8<T>(x + c, y);
      if (OP == kRowsSilu || (OP == kRowsNorm && other)) load8<T>(other + c, o);
      if (OP == kRowsNorm) load8<T>(weight + c, w);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = column(j, lane, lanes) + e;
        y[e] = o[e] = w[e] = 0.f;
        if (c >= K) continue;
        y[e] = to_float<T>(x[c]);
        if (OP == kRowsSilu || (OP == kRowsNorm && other)) o[e] = to_float<T>(other[c]);
        if (OP == kRowsNorm) w[e] = to_float<T>(weight[c]);
      }
    }
    if (OP == kRowsNorm) {
      if (other) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] += o[e];
        if (keep) {
          if constexpr (!std::is_same<T, float>::value) {
            if (VEC) {
              *reinterpret_cast<uint4*>(total + column(j, lane, lanes)) = pack8<T>(y);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int c = column(j, lane, lanes) + e;
                if (c < K) total[c] = from_float<T>(y[e]);
              }
            }
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum = fmaf(y[e], y[e], sum);
        y[e] *= w[e];
      }
    }
    if (OP == kRowsSilu) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = y[e] * rcp(1.f + expf(-y[e])) * o[e];
    }
  }
};

// The integers nearest to 127 v / top, two's complement, in the low bytes.
// The quotient is that of a product with 1 / top, put right by its remainder
// once (Markstein 1990): where 127 v / top is a float, a half say, the result
// is that float, and halves go to even.  Adding 1.5 * 2^23 rounds to a whole
// number and leaves it in the low bits; a conversion runs at a quarter of the
// rate.
struct Quotient {
  float times, over, inverse;
  KUS_DEVICE Quotient(float top, bool sound) {
    const float small = top > 1e36f ? 0x1p-10f : top < 1e-30f ? 0x1p60f : 1.f;   // 127 v and 1 / top stay in range
    over = sound && top > 0.f ? top * small : 1.f;
    times = sound ? 127.f * small : 0.f;
    inverse = 1.f / over;
  }
  KUS_DEVICE uint32_t operator()(float v) const {
    const float t = v * times, r = t * inverse;
    return __float_as_uint(fmaf(fmaf(-r, over, t), inverse, r) + 12582912.f);
  }
};

// One row a warp (WARPS == 1; eight warps a block) or a block.  HELD: vectors
// of 8 a thread keeps between the two passes over its row; 0: the row is read
// again.
template <typename T, int OP, bool ONE_WARP, int HELD, bool VEC>
__global__ void __launch_bounds__(ONE_WARP ? 256 : 1024) rows_kernel(Int8Rows a) {
  __shared__ float2 part[32];
  pdl_wait();
  pdl_trigger();
  const int lanes = ONE_WARP ? 32 : blockDim.x;
  const int lane = ONE_WARP ? threadIdx.x % 32 : threadIdx.x;
  const long long t = ONE_WARP ? (long long)blockIdx.x * 8 + threadIdx.x / 32 : blockIdx.x;
  if (ONE_WARP && t >= a.T) return;
  const Row<T, OP> row(a, t);
  const int vectors = HELD > 0 ? HELD : (a.K + 8 * lanes - 1) / (8 * lanes);

  float y[HELD > 0 ? HELD : 1][8];
  float sum = 0.f, top = 0.f;
  if (HELD > 0) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) row.template values<VEC>(j, lane, lanes, true, y[j], sum);
#pragma unroll
    for (int j = 0; j < HELD; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max_nan(top, fabsf(y[j][e]));
  } else {
    for (int j = 0; j < vectors; ++j) {
      row.template values<VEC>(j, lane, lanes, false, y[0], sum);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max_nan(top, fabsf(y[0][e]));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (OP == kRowsNorm) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (!ONE_WARP) {
    const int warps = blockDim.x / 32, l = threadIdx.x % 32;
    if (l == 0) part[threadIdx.x / 32] = make_float2(sum, top);
    __syncthreads();
    const float2 p = l < warps ? part[l] : make_float2(0.f, 0.f);
    sum = p.x;
    top = p.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (OP == kRowsNorm) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
  }

  // scale and the integers' factor; a row without finite values has scale NaN
  float factor = 1.f;
  bool sound = top < INFINITY;
  if (OP == kRowsNorm) {
    factor = rsqrtf(sum / (float)a.K + a.eps);
    sound = sound && sum < INFINITY;
  }
  if (lane == 0) a.scales[t] = sound ? top / 127.f * factor : NAN;
  const Quotient quotient(top, sound);
  int8_t* q = a.q + t * a.qs;
  auto write = [&](int j, const float (&v)[8]) {
    uint32_t r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = sound ? quotient(v[e]) : 0;
    const int c = column(j, lane, lanes);
    if (VEC) {
      uint2 u;
      u.x = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
      u.y = __byte_perm(__byte_perm(r[4], r[5], 0x0040), __byte_perm(r[6], r[7], 0x0040), 0x5410);
      if (c < a.K) *reinterpret_cast<uint2*>(q + c) = u;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < a.K) q[c + e] = (int8_t)r[e];
    }
  };
  if (HELD > 0) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) write(j, y[j]);
  } else {
    // the sum x + residual is written in the second pass: it may lie over either of them
    for (int j = 0; j < vectors; ++j) {
      float unused = 0.f;
      row.template values<VEC>(j, lane, lanes, true, y[0], unused);
      write(j, y[0]);
    }
  }
}

template <typename T, int OP, bool ONE_WARP, int HELD>
void launch(const Int8Rows& a, bool vec, cudaStream_t s) {
  const int vectors = (a.K + 7) / 8;
  const int each = HELD > 0 ? HELD : 4;
  int threads = ONE_WARP ? 256 : ((vectors + each - 1) / each + 31) / 32 * 32;
  if (threads > 1024) threads = 1024;
  const dim3 grid((unsigned)(ONE_WARP ? (a.T + 7) / 8 : a.T));
  if (vec)
    launch_k(rows_kernel<T, OP, ONE_WARP, HELD, true>, grid, dim3(threads), 0, s, a);
  else
    launch_k(rows_kernel<T, OP, ONE_WARP, HELD, false>, grid, dim3(threads), 0, s, a);
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
  if (n <= 32) return launch<T, OP, true, 1>(a, vec, s);
  if (n <= 64) return launch<T, OP, true, 2>(a, vec, s);
  if (n <= 256) return launch<T, OP, false, 1>(a, vec, s);
  if (n <= 1024) return launch<T, OP, false, 2>(a, vec, s);
  if (n <= 4096) return launch<T, OP, false, 4>(a, vec, s);
  return launch<T, OP, false, 0>(a, vec, s);
}

// The float of byte i of u, whose bytes are integers with their top bit
// turned over: 2^23 + 128 + q, less 2^23 + 128.  (A conversion runs at a
// quarter of the rate.)
KUS_DEVICE float value(uint32_t u, int i) { return __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + i)) - 8388736.f; }

// A row a block; VEC: 16 elements a thread and step.
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
    for (int c = at * 16; c < a.K; c += step * 16) {
      const uint4 u = *reinterpret_cast<const uint4*>(q + c);
      const uint32_t w[4] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u, u.z ^ 0x80808080u, u.w ^ 0x80808080u};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = value(w[2 * h + e / 4], e % 4) * s;
        if constexpr (std::is_same<T, float>::value) {
          reinterpret_cast<float4*>(out + c + 8 * h)[0] = make_float4(f[0], f[1], f[2], f[3]);
          reinterpret_cast<float4*>(out + c + 8 * h)[1] = make_float4(f[4], f[5], f[6], f[7]);
        } else {
          *reinterpret_cast<uint4*>(out + c + 8 * h) = pack8<T>(f);
        }
      }
    }
  } else {
    for (int c = at; c < a.K; c += step) out[c] = from_float<T>((float)q[c] * s);
  }
}

template <typename T>
void launch_values(const Int8Values& a, cudaStream_t s) {
  const bool vec = a.K % 16 == 0 && on16(a.out, a.os, sizeof(T), a.T) && on16(a.q, a.qs, 1, a.T);
  const int items = vec ? a.K / 16 : a.K;
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
