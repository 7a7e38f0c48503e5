// Element helpers of the cache operators: bf16 and fp16 alike.
#pragma once
#include "../common.cuh"
#include <cuda_fp16.h>

namespace kus {

// 16-bit element types of the cache operators.
template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  using V2 = __nv_bfloat162;
  KUS_DEVICE static float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
  KUS_DEVICE static __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
  KUS_DEVICE static float2 to_f2(V2 x) { return __bfloat1622float2(x); }
  KUS_DEVICE static V2 from_f2(float a, float b) { return __floats2bfloat162_rn(a, b); }
};
template <>
struct Elem<__half> {
  using V2 = __half2;
  KUS_DEVICE static float to_f(__half x) { return __half2float(x); }
  KUS_DEVICE static __half from_f(float x) { return __float2half_rn(x); }
  KUS_DEVICE static float2 to_f2(V2 x) { return __half22float2(x); }
  KUS_DEVICE static V2 from_f2(float a, float b) { return __floats2half2_rn(a, b); }
};

template <typename T>
KUS_DEVICE void unpack8(const uint4& u, float (&f)[8]) {
  const typename Elem<T>::V2* h = reinterpret_cast<const typename Elem<T>::V2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = Elem<T>::to_f2(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <typename T>
KUS_DEVICE uint32_t pack2(float a, float b) {
  typename Elem<T>::V2 v = Elem<T>::from_f2(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <typename T>
KUS_DEVICE uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

// 2^x in one instruction (results below the normal range are zeros).
KUS_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// While one lives, this thread's launches carry programmatic serialization:
// a grid is set up while the one before it ends.  Every kernel of the cache
// operators waits for the one before (pdl_wait) ahead of its first access to
// what others write; only plans, which no kernel writes, are read earlier.
// They alone may be read with __ldg: it takes memory for read-only while the
// grid lives, and the grid before may still be writing when this one starts.
struct LaunchBehind {
  const bool was = pdl_flag();
  LaunchBehind() { pdl_flag() = true; }
  ~LaunchBehind() { pdl_flag() = was; }
};

}  // namespace kus
