// Host interface of the 8-bit operators: rows written as 8-bit integers with
// one scale each (quantisation, RMSNorm with the residual's addition,
// SiLU * up), and the matrix product of such rows with 8-bit weights.
#pragma once
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace kus {

enum : int { kInt8TypeBF16 = 0, kInt8TypeFP16 = 1, kInt8TypeFP32 = 2 };
enum Int8RowsOp : int { kRowsQuantize = 0, kRowsNorm = 1, kRowsSilu = 2 };

// ------------------------------------------------------- rows to 8 bits
struct Int8Rows {
  int op;
  int type;                  // of x, other, weight and total (fp32: quantize only)
  const void* x;             // [T, K], row stride xs elements; gate of kRowsSilu
  const void* other;         // residual of kRowsNorm (may be null), up of kRowsSilu
  const void* weight;        // [K] of kRowsNorm
  void* total;               // x + residual; null without a residual
  long long xs, os, ts;      // row strides of x, other and total
  float eps;
  int8_t* q;                 // [T, K], row stride qs (a multiple of 16 bytes, 16-byte base)
  long long qs;
  float* scales;             // [T]
  int T, K;
};
void int8_rows(const Int8Rows& a, cudaStream_t s);

struct Int8Values {
  const int8_t* q;           // [T, K], row stride qs
  long long qs;
  const float* scales;       // [T]
  void* out;                 // [T, K], row stride os
  long long os;
  int type;
  int T, K;
};
void int8_values(const Int8Values& a, cudaStream_t s);

// -------------------------------------------------------- matrix product
// Weights are kept in blocks of 128 channels x 128 bytes along K, one 16 KB
// block after the other along K, then along N, padded with zeros: a block is
// one contiguous read.
constexpr int kInt8Block = 128;
constexpr int kInt8MaxK = 131071;   // 2^31 / (128 * 128) terms fit an int32 sum
inline long long int8_blocks(long long n) { return (n + kInt8Block - 1) / kInt8Block; }

// A product reads its first weights ahead of its wait for the kernel before it,
// which alone makes that one's writes visible: behind int8_pack the caller
// queues something that never lets another start early, a copy say.
void int8_pack(const int8_t* w, long long stride, int N, int K, int8_t* packed, cudaStream_t s);

// Tokens whose rows start anywhere, in rows of K rounded up to 16 bytes.
void int8_align(const int8_t* q, long long stride, int M, int K, int8_t* out, cudaStream_t s);

struct Int8Gemm {
  int M, N, K;
  const float* x_scales;     // [M]
  const float* w_scales;     // [N]
  const void* bias;          // [N] of out's type, or null
  void* out;                 // [M, N], row stride ldc elements
  long long ldc;
  int type;
};
// How the kernel cuts a product.
struct Int8Plan {
  int pair;                  // pairs of CTAs share 256 channels; else a CTA has 128
  int width;                 // tokens of a tile (a multiple of 16, of a pair 32)
  int token_tiles, channel_tiles;
  int splits;                // CTAs (pairs) of a cluster that share a tile's K
  int alone;                 // one CTA an SM; else two
  int apart;                 // the parts of a split lie beside the stages, else over them
  int group;                 // token tiles walked before the next channel tile
  int grid;                  // CTAs
  int stages, tmem_columns;
  int smem;                  // bytes of dynamic shared memory a CTA asks for
};
// Clusters of 1 to 8 CTAs that the device holds at once, with one CTA an SM.
struct Int8Slots {
  int clusters[9];
};
Int8Slots int8_slots();
// `element`: bytes of a result.
Int8Plan int8_plan(int M, int N, int K, int element, const Int8Slots& slots);
// Tensor maps of the packed weights (made once) and of the tokens (each call;
// base and row stride are multiples of 16 bytes).
bool int8_weight_map(CUtensorMap* map, const int8_t* packed, int N, int K);
bool int8_token_map(CUtensorMap* map, const int8_t* x, long long stride, int M, int K, const Int8Plan& p);
void int8_gemm(const Int8Gemm& a, const Int8Plan& p, const CUtensorMap& weights, const CUtensorMap& tokens,
               cudaStream_t s);

}  // namespace kus
