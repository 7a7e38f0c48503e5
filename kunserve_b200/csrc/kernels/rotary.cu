// Rotary positions, fused with the append to the paged cache.
//
// Pair i of a head turns by the angle position * f_i:
//   (a, b) -> m (a cos - b sin, b cos + a sin)
// with (a, b) = dims (i, i + rot/2) of the half layout or (2i, 2i + 1) of the
// interleaved one, for the first `rot` dims of a head; the rest pass through.
// f_i is given in turns (f_i / 2 pi) as a 64-bit fraction, so position * f_i
// modulo one turn is a 64-bit integer product: exact for every 32-bit
// position, where position * f_i in fp32 is off by 2^-8 rad at 10^5.  sinpi
// and cospi then take the remaining fraction in half turns.
//
// Bound by HBM: each element is read once and written once.  A block takes
// one token (its cos and sin computed once, into shared memory, for all
// heads, while the first items' loads are under way); a thread turns 16
// elements of a head as two 16-byte vectors.  Full SMs (32 registers a thread)
// move more than several items in flight a thread: 16384 tokens of 64 + 8
// heads of 128, 672 MB, take 104-111 us in a steady run (102 in the first
// 100 ms); with three items at 62 registers 117 where these took 102.
#include "../common.cuh"
#include "cache_elem.cuh"
#include "cache_ops.h"

namespace kus {

namespace rot {

constexpr int kThreads = 256;   // at most; a block has what its items divide into

// VEC: 16-byte vectors (bases and strides of 16 bytes, hd and rot multiples
// of 16); otherwise single elements, one pair or one unrotated element a
// thread.
template <typename T, bool INTER, bool VEC>
__global__ void __launch_bounds__(kThreads, 8) rotary_kernel(RotaryArgs a) {
  extern __shared__ float2 cs[];   // (cos, sin) of the token's rot / 2 pairs
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x;
  const int half = a.rot / 2;
  const int heads = a.nq + 2 * a.nkv;
  const T* xrow = reinterpret_cast<const T*>(a.x) + t * a.xt;
  T* orow = reinterpret_cast<T*>(a.out) + t * a.ot;
  const int threads = blockDim.x, first = blockIdx.y * threads + threadIdx.x, step = gridDim.y * threads;

  // vector items: j-th 16 elements of head h, as two vectors at dims d0, d1:
  // the pairs (i, i + rot/2) where the half layout turns, else neighbours
  const int per = a.hd / 16, items = heads * per, turned = a.rot / 16;
  struct Item {
    int h, d0, d1;
    bool turn;
  };
  auto item_at = [&](int u) {
    Item it;
    it.h = u / per;
    const int j = u - it.h * per;
    it.turn = it.h < a.nq + a.nkv && j < turned;
    it.d0 = (!INTER && it.turn) ? 8 * j : 16 * j;
    it.d1 = (!INTER && it.turn) ? it.d0 + half : it.d0 + 8;
    return it;
  };
  uint4 v0, v1;
  auto load = [&](int u) {
    const Item it = item_at(u);
    const T* src = xrow + it.h * a.xh;
    v0 = *reinterpret_cast<const uint4*>(src + it.d0);
    v1 = *reinterpret_cast<const uint4*>(src + it.d1);
  };
  // the first item's loads run beside the angles
  if (VEC && first < items) load(first);

  const long long pos = a.positions[t];
  for (int i = threadIdx.x; i < half; i += threads) {
    const unsigned long long turn = (unsigned long long)pos * a.steps[i];
    float s, c;
    sincospif((float)(long long)turn * 0x1p-63f, &s, &c);
    cs[i] = make_float2(c * a.scale, s * a.scale * a.sign);
  }
  T* krow = nullptr;   // the token's cache row, KV head 0
  T* vrow = nullptr;
  if (a.nkv) {
    // a bad row would corrupt the cache: recorded, its keys and values dropped
    const int page = a.pages[t], slot = a.slots[t];
    if (page < 0 || page >= a.g.pages_total || slot < 0 || slot >= a.g.block_size) {
      if (threadIdx.x == 0 && blockIdx.y == 0) set_error(kErrBounds, page);
    } else {
      const long long off = (long long)slot * a.g.kvh * a.g.hd * (int)sizeof(T);
      krow = reinterpret_cast<T*>(a.g.base + kv_offset(a.g, page, a.layer, false) + off);
      vrow = reinterpret_cast<T*>(a.g.base + kv_offset(a.g, page, a.layer, true) + off);
      if (a.weights && blockIdx.y == 0)
        for (int h = threadIdx.x; h < a.nkv; h += threads) {
          const long long i = ((long long)page * a.nkv + h) * a.g.block_size + slot;
          a.weights[i] = 0.f;
          a.slot_positions[i] = (int)pos;
        }
    }
  }
  __syncthreads();
  // head h's destination; null: not written
  auto dest = [&](int h) -> T* {
    if (h < a.nq) return orow + h * a.oh;
    if (!krow) return nullptr;
    return h < a.nq + a.nkv ? krow + (long long)(h - a.nq) * a.hd : vrow + (long long)(h - a.nq - a.nkv) * a.hd;
  };
  if (VEC) {
    for (int u = first; u < items; u += step) {
      if (u != first) load(u);
      const Item it = item_at(u);
      T* dst = dest(it.h);
      if (!dst) continue;
      if (it.turn) {
        float x0[8], x1[8];
        unpack8<T>(v0, x0);
        unpack8<T>(v1, x1);
        if (INTER) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float2 p = cs[it.d0 / 2 + e / 2], r = cs[it.d1 / 2 + e / 2];
            const float a0 = x0[e], a1 = x1[e];
            x0[e] = a0 * p.x - x0[e + 1] * p.y;
            x0[e + 1] = x0[e + 1] * p.x + a0 * p.y;
            x1[e] = a1 * r.x - x1[e + 1] * r.y;
            x1[e + 1] = x1[e + 1] * r.x + a1 * r.y;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float2 p = cs[it.d0 + e];
            const float a0 = x0[e];
            x0[e] = a0 * p.x - x1[e] * p.y;
            x1[e] = x1[e] * p.x + a0 * p.y;
          }
        }
        v0 = pack8<T>(x0);
        v1 = pack8<T>(x1);
      }
      *reinterpret_cast<uint4*>(dst + it.d0) = v0;
      *reinterpret_cast<uint4*>(dst + it.d1) = v1;
    }
  } else {
    const int pairs = half + (a.hd - a.rot);
    for (int u = first; u < heads * a.hd; u += step) {
      const int h = u / a.hd, j = u - h * a.hd;
      T* dst = dest(h);
      if (!dst) continue;
      const T* src = xrow + h * a.xh;
      if (h >= a.nq + a.nkv) {
        dst[j] = src[j];
      } else if (j < half) {
        const int d0 = INTER ? 2 * j : j, d1 = INTER ? 2 * j + 1 : j + half;
        const float x0 = Elem<T>::to_f(src[d0]), x1 = Elem<T>::to_f(src[d1]);
        const float2 p = cs[j];
        dst[d0] = Elem<T>::from_f(x0 * p.x - x1 * p.y);
        dst[d1] = Elem<T>::from_f(x1 * p.x + x0 * p.y);
      } else if (j < pairs) {
        dst[j + half] = src[j + half];
      }
    }
  }
}

template <typename T, bool INTER>
void launch(const RotaryArgs& a, cudaStream_t s) {
  auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool vec = al(a.x) && al(a.out) && (a.nkv == 0 || al(a.g.base)) && a.xt % 8 == 0 && a.xh % 8 == 0 &&
                   a.ot % 8 == 0 && a.oh % 8 == 0 && a.hd % 16 == 0 && a.rot % 16 == 0;
  const int items = (a.nq + 2 * a.nkv) * (vec ? a.hd / 16 : a.hd);
  // few tokens: several blocks a token, each with the heads' share, so that
  // one token's heads are all in flight at once
  const int rounds = (items + kThreads - 1) / kThreads;
  const int split = a.T >= 2 * 148 ? 1 : rounds;
  const int threads = ((items + rounds - 1) / rounds + 31) / 32 * 32;   // no round is half empty
  const dim3 grid(a.T, split);
  const size_t smem = (size_t)a.rot / 2 * sizeof(float2);
  if (vec)
    launch_k(rotary_kernel<T, INTER, true>, grid, dim3(threads), smem, s, a);
  else
    launch_k(rotary_kernel<T, INTER, false>, grid, dim3(threads), smem, s, a);
}

}  // namespace rot

void rotary(const RotaryArgs& a, int type, cudaStream_t s) {
  if (a.T <= 0 || a.nq + a.nkv == 0) return;
  const LaunchBehind behind;
  if (type == kTypeBF16) {
    a.interleaved ? rot::launch<__nv_bfloat16, true>(a, s) : rot::launch<__nv_bfloat16, false>(a, s);
  } else {
    a.interleaved ? rot::launch<__half, true>(a, s) : rot::launch<__half, false>(a, s);
  }
}

}  // namespace kus
