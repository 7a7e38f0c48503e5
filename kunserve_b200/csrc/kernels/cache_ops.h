// Host interface of the long-context cache operators: rotary append, attention
// over planned work units (shared prefixes, weighted decode), eviction.
//
// Every operator works on 16-bit elements (bf16 or fp16) of one layer of a
// paged pool described by a KVGeom.
#pragma once
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>
#include "kernels.h"

namespace kus {

enum : int { kTypeBF16 = 0, kTypeFP16 = 1 };

// ------------------------------------------------------------------ rotary
struct RotaryArgs {
  const void* x;                 // [T, heads, hd]: heads = nq (rotated to out) + 2 * nkv (keys, values)
  long long xt, xh;              // element strides of a token and of a head
  void* out;                     // [T, nq, hd]; may be x
  long long ot, oh;
  const int* positions;          // [T]
  const unsigned long long* steps;   // [rot / 2] turns per position, 64-bit fractions
  float scale;                   // factor on cos and sin
  float sign;                    // +1, or -1 to rotate back
  int T, nq, nkv, hd, rot;
  bool interleaved;
  // append (nkv > 0): cache row of each token, and optionally the slot's
  // weight (cleared) and position (recorded), both [pages, nkv, block_size]
  const int* pages;
  const int* slots;
  KVGeom g;
  int layer;
  float* weights;
  int* slot_positions;
};
void rotary(const RotaryArgs& a, int type, cudaStream_t s);

// ------------------------------------------- attention over planned units
// A unit is a set of query rows (tokens x query heads of one KV head's
// group) and a range of the keys behind one page list; the same units run
// for every KV head.  Row r of a unit is token tok0 + r / ng, group head
// g0 + r % ng.  Ints of a unit:
//   0 tok0   1 ntok | ng << 8 | g0 << 16   2 first key   3 end of the keys
//   4 keys that token tok0 sees (token tok0 + j: j more)   5 first page
//   6 first partial row (of KV head 0; head kh: + kh * ntok * ng)
//   7 first column of the request's scores (weighted plans), else 0
constexpr int kUnitInts = 8;
constexpr int kRowUnitRows = 16;     // most rows of a unit of the row kernel
constexpr int kTileUnitRows = 128;   // most rows of a unit of the tile kernel
constexpr int kStageKeys = 32;       // keys per stage of the row kernel; ranges and rows of scores are multiples
constexpr int kTileKeys = 128;       // keys per block of the tile kernel; its ranges start on multiples
constexpr int kNoLimit = 1 << 30;    // unit int 4 of keys without a causal limit
// Ints of a weight chunk: token row, first key, end, first page, keys of the request, first score column.
constexpr int kChunkInts = 6;
constexpr int kChunkKeys = 512;      // keys of a chunk, at most

struct CachedAttn {
  const void* q;                 // [T, nq, hd]
  long long qt, qh;
  void* out;                     // [T, nq, hd]
  long long ot, oh;
  KVGeom g;
  int layer;
  int T, nq, hd;
  float scale;
  const int* pages;              // page lists of the units
  const int* row_units;          // [n_row_units, kUnitInts]
  int n_row_units;
  const int* tile_units;         // [n_tile_units, kUnitInts]
  int n_tile_units;
  // partial rows of each (token, chunk of 16 group heads): entries
  // [merge_off[i], merge_off[i + 1]) of (row of group head 0 at KV head 0, rows per KV head)
  const int* merge_off;
  const int2* merge;
  int head_chunks;
  int most_parts;                // longest of those lists
  float* part_o;                 // [partial rows, hd]
  float2* part_ml;               // [partial rows] reference of the sums (log2 units, near the max), sum
  // weighted plans: scores [request][nq][keys rounded up to kStageKeys] fp32, the
  // weights [pages, kvh, block_size] that each key's attention is added to
  float* scores;
  float2* stats;                 // [T, nq] (reference, 1 / sum) of weighted plans
  float* weights;
  const int* chunks;             // [n_chunks, kChunkInts]
  int n_chunks;
};
// The call: the tile kernel over the tile units, the row kernel over the row
// units, the join of their parts.  `map`: of make_cache_tile_map, needed with
// tile units only.
void cached_attention(const CachedAttn& a, const CUtensorMap* map, int type, cudaStream_t s);
void cached_attention_tiles(const CachedAttn& a, const CUtensorMap& map, int type, cudaStream_t s);
// Keys per TMA box of the tile kernel (a power of two that divides the page)
// and the tensor map of a pool of `bytes`; false where the tile kernel cannot
// read the pool: pages that are no multiple of 8 slots, other head sizes.
int cache_tile_box(const KVGeom& g);
bool make_cache_tile_map(CUtensorMap* map, const KVGeom& g, long long bytes, int type);

// ---------------------------------------------------------------- eviction
// Ints of a request: tokens, first page, newest position, 0.
constexpr int kRequestInts = 4;

struct EvictSelect {
  const float* weights;          // [pages, kvh, block_size]
  const int* slot_positions;     // [pages, kvh, block_size]
  KVGeom g;
  const int* pages;
  const int* reqs;               // [n_reqs, kRequestInts]
  int n_reqs, most_tokens;       // longest request
  int keep, sinks, recent, cap;
  int2* moves;                   // [n_reqs, kvh, cap] (to, from), -1 past the count
  int* counts;                   // [n_reqs, kvh]
};
void evict_select(const EvictSelect& a, cudaStream_t s);

struct CacheCompact {
  KVGeom g;
  int layer;
  const int* pages;
  const int* reqs;
  int n_reqs, cap;
  const int2* moves;
  const int* counts;
  float* weights;                // may be null
  int* slot_positions;           // may be null
};
void cache_compact(const CacheCompact& a, cudaStream_t s);

}  // namespace kus
