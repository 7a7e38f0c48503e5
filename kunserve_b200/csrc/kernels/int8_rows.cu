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
      for (int e = 0; e < 8; ++e) y[e] = y[e] / (1.f + expf(-y[e])) * o[e];
    }
  }
};

// One row a group of LANES threads.  HELD: vectors of 8 a thread keeps
// between the two passes over its row; 0: the row is read again.
template <typename T, int OP, int LANES, int HELD, bool VEC>
__global__ void __launch_bounds__(LANES < 256 ? 256 : LANES) rows_kernel(Int8Rows a) {
  constexpr int kThreads = LANES < 256 ? 256 : LANES;
  constexpr int kRows = kThreads / LANES, kWarps = LANES / 32;
  __shared__ float2 part[kThreads / 32];
  pdl_wait();
  pdl_trigger();
  const int group = threadIdx.x / LANES, lane = threadIdx.x % LANES;
  const long long t = (long long)blockIdx.x * kRows + group;
  if (kRows > 1 && t >= a.T) return;      // whole groups leave; those of several warps are their block's only one
  const Row<T, OP> row(a, t);
  const int vectors = (a.K + 8 * LANES - 1) / (8 * LANES);

  float y[HELD > 0 ? HELD : 1][8];
  float sum = 0.f, top = 0.f;
  if (HELD > 0) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) row.template values<VEC>(j, lane, LANES, true, y[j], sum);
#pragma unroll
    for (int j = 0; j < HELD; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max_nan(top, fabsf(y[j][e]));
  } else {
    for (int j = 0; j < vectors; ++j) {
      row.template values<VEC>(j, lane, LANES, false, y[0], sum);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max_nan(top, fabsf(y[0][e]));
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (OP == kRowsNorm) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if (kWarps > 1) {
    const int w0 = group * kWarps;
    if (lane % 32 == 0) part[threadIdx.x / 32] = make_float2(sum, top);
    if (kRows > 1)
      named_barrier(1 + group, LANES);
    else
      __syncthreads();
    sum = 0.f;
    top = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float2 p = part[w0 + w];
      if (OP == kRowsNorm) sum += p.x;
      top = max_nan(top, p.y);
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
  const float small = top > 1e36f ? 0x1p-10f : 1.f;     // keeps 127 y in range
  const float times = sound ? 127.f * small : 0.f, over = sound && top > 0.f ? top * small : 1.f;
  int8_t* q = a.q + t * a.qs;
  auto write = [&](int j, const float (&v)[8]) {
    int r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = sound ? __float2int_rn(v[e] * times / over) : 0;
    if (VEC) {
      const int c = column(j, lane, LANES);
      uint2 u;
      u.x = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
      u.y = __byte_perm(__byte_perm(r[4], r[5], 0x0040), __byte_perm(r[6], r[7], 0x0040), 0x5410);
      if (c < a.K) *reinterpret_cast<uint2*>(q + c) = u;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = column(j, lane, LANES) + e;
        if (c < a.K) q[c] = (int8_t)r[e];
      }
    }
  };
  if (HELD > 0) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) write(j, y[j]);
  } else {
    // the sum x + residual is written in the second pass: it may lie over either of them
    for (int j = 0; j < vectors; ++j) {
      float unused = 0.f;
      row.template values<VEC>(j, lane, LANES, true, y[0], unused);
      write(j, y[0]);
    }
  }
}

template <typename T, int OP, int LANES, int HELD>
void launch(const Int8Rows& a, bool vec, cudaStream_t s) {
  constexpr int kThreads = LANES < 256 ? 256 : LANES;
  const dim3 grid((unsigned)((a.T + kThreads / LANES - 1) / (kThreads / LANES)));
  if (vec)
    launch_k(rows_kernel<T, OP, LANES, HELD, true>, grid, dim3(kThreads), 0, s, a);
  else
    launch_k(rows_kernel<T, OP, LANES, HELD, false>, grid, dim3(kThreads), 0, s, a);
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
  if (n <= 32) return launch<T, OP, 32, 1>(a, vec, s);
  if (n <= 64) return launch<T, OP, 32, 2>(a, vec, s);
  if (n <= 128) return launch<T, OP, 64, 2>(a, vec, s);
  if (n <= 256) return launch<T, OP, 128, 2>(a, vec, s);
  if (n <= 512) return launch<T, OP, 256, 2>(a, vec, s);
  if (n <= 768) return launch<T, OP, 256, 3>(a, vec, s);
  if (n <= 1024) return launch<T, OP, 512, 2>(a, vec, s);
  if (n <= 2048) return launch<T, OP, 512, 4>(a, vec, s);
  if (n <= 4096) return launch<T, OP, 1024, 4>(a, vec, s);
  return launch<T, OP, 1024, 0>(a, vec, s);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) values_kernel(Int8Values a) {
  pdl_wait();
  pdl_trigger();
  const long long t = blockIdx.x;
  const int8_t* q = a.q + t * a.qs;
  T* out = reinterpret_cast<T*>(a.out) + t * a.os;
  const float s = a.scales[t];
  if (VEC) {
    for (int c = (blockIdx.y * 256 + threadIdx.x) * 8; c < a.K; c += gridDim.y * 256 * 8) {
      const uint2 u = *reinterpret_cast<const uint2*>(q + c);
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (float)(int8_t)((e < 4 ? u.x : u.y) >> (8 * (e % 4))) * s;
      if constexpr (std::is_same<T, float>::value) {
        reinterpret_cast<float4*>(out + c)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(out + c)[1] = make_float4(f[4], f[5], f[6], f[7]);
      } else {
        *reinterpret_cast<uint4*>(out + c) = pack8<T>(f);
      }
    }
  } else {
    for (int c = blockIdx.y * 256 + threadIdx.x; c < a.K; c += gridDim.y * 256) out[c] = from_float<T>((float)q[c] * s);
  }
}

template <typename T>
void launch_values(const Int8Values& a, cudaStream_t s) {
  const bool vec = a.K % 8 == 0 && on16(a.out, a.os, sizeof(T), a.T) &&
                   reinterpret_cast<uintptr_t>(a.q) % 8 == 0 && (a.T <= 1 || a.qs % 8 == 0);
  const int per = vec ? 8 * 256 : 256;
  const int y = (a.K + per - 1) / per;
  const dim3 grid((unsigned)a.T, (unsigned)(y < 64 ? y : 64));
  if (vec)
    launch_k(values_kernel<T, true>, grid, dim3(256), 0, s, a);
  else
    launch_k(values_kernel<T, false>, grid, dim3(256), 0, s, a);
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
