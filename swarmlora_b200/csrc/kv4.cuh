// The paged key/value cache held in 4 bits: block layout and host tables.
//
// A block holds 16 consecutive tokens of one kv head (K and V) in 18 * D bytes;
// a cache is [pages][page / 16][hkv][18 * D] bytes. Groups of 64 dimensions of
// one token share a scale s and a minimum m (bf16 each): value = s * code + m,
// code in 0..15, so a value costs 4.5 bits.
//
//   bytes [0, 8D)     K codes: word (t * 4 + (d / 8) % 4) * W + d / 32, nibble d % 8
//   bytes [8D, 9D)    K pairs: (s, m) of token t, group g at 4 * (t * D / 64 + g)
//   bytes [9D, 17D)   V codes: word ((t / 8) * 32 + (d / 4) % 8 * 4 + (t % 8) / 2) * W + d / 32,
//                     16-bit half t % 2, nibble d % 4
//   bytes [17D, 18D)  V pairs, as K's
// with W = D / 32 words (of 8 codes) per entry. The order is the one in which the
// attention's matrix fragments want the codes: lane (g, c) of a warp reads
// the K codes of tokens g and g + 8 (dimensions 32 j + 8 c ..) and the V codes of
// tokens 2c, 2c + 1, 2c + 8, 2c + 9 (dimensions 32 u + 4 g ..) as single aligned vectors, and
// a word's nibbles become pairs of bf16 by one shift and one logic operation.
// Every code of a token lies in whole 16-bit pieces, so tokens of one block
// are written without reading their neighbours.
#pragma once

#include <cstdint>

#include "worker_ops.h"

namespace swl {
namespace kv4 {

constexpr int kBlockTok = 16;
constexpr int kGroup = 64;

__host__ __device__ constexpr int block_bytes(int d) { return 18 * d; }
__host__ __device__ constexpr int k_pair_off(int d) { return 8 * d; }
__host__ __device__ constexpr int v_code_off(int d) { return 9 * d; }
__host__ __device__ constexpr int v_pair_off(int d) { return 17 * d; }

// Byte offset of the word holding dimensions d..d+7 (d % 8 == 0) of token t's K.
template <int D>
__device__ __forceinline__ int k_word(int t, int d) {
  return 4 * ((t * 4 + (d >> 3 & 3)) * (D / 32) + (d >> 5));
}
// Byte offset of the 16-bit piece holding dimensions d..d+3 (d % 4 == 0) of token t's V.
template <int D>
__device__ __forceinline__ int v_piece(int t, int d) {
  return v_code_off(D) + 4 * (((t >> 3) * 32 + (d >> 2 & 7) * 4 + (t >> 1 & 3)) * (D / 32) + (d >> 5)) + 2 * (t & 1);
}

// What a launch over slots reads: slot i's block table (page ids), cache and cached
// length. The entries of the slot's table and the pages of its cache bound every access.
// Packed slots go by base and step and share both bounds: an entry of a table in the parameter space is
// a cache miss of its own, several of them one behind the other at the start of every CTA.
// (A struct a slot in place of the arrays: append of 6499 rows and gather 47.0 us for 45.7.)
struct Cache {
  int packed;                    // 1: table0, cache0, len0, table_len0, pages0; 0: the tables
  int rows_each;                 // new rows of every slot where all have as many, else 0
  const int* table0;
  int64_t table_step;
  uint8_t* cache0;
  const int* len0;
  int table_len0;
  uint32_t pages0;
  int page_shift;                // log2(page / 16)
  int hkv;
  const int* block_table[kMaxSlots];
  uint8_t* cache[kMaxSlots];
  const int* seqlen[kMaxSlots];  // device int: tokens cached before this step
  int table_len[kMaxSlots];
  uint32_t pages[kMaxSlots];     // at most 2^31: a negative page id, taken as unsigned, lies outside
};

__device__ __forceinline__ const int* len_of(const Cache& c, int s) { return c.packed ? c.len0 + s : c.seqlen[s]; }
// First row of slot s.
__device__ __forceinline__ int row_of(const Cache& c, const RowSegments& seg, int s) {
  return c.rows_each ? s * c.rows_each : seg.row_start[s];
}

// The block of tile `tile` (tokens 16 tile ..) of head h, or nullptr where the
// table has no such entry or names no page of the cache.
// kEither: the cache may be a packed one (the appending and gathering kernels always get tables:
// the choice costs them registers that they are short of).
template <int D, bool kEither = false>
__device__ __forceinline__ uint8_t* block_of(const Cache& c, int s, int64_t tile, int h) {
  const int64_t pi = tile >> c.page_shift;
  const bool packed = kEither && c.packed;
  if (tile < 0 || pi >= (packed ? c.table_len0 : c.table_len[s])) return nullptr;
  const uint32_t page = (packed ? c.table0 + s * c.table_step : c.block_table[s])[pi];
  if (page >= (packed ? c.pages0 : c.pages[s])) return nullptr;
  const int64_t sub = tile & ((int64_t{1} << c.page_shift) - 1);
  return (packed ? c.cache0 : c.cache[s]) +
         (((static_cast<int64_t>(page) << c.page_shift) + sub) * c.hkv + h) * block_bytes(D);
}

// The slots of a call as its caller gives them: tables of pointers, or packed (base and step).
struct Slots {
  const void* const* block_tables = nullptr;
  void* const* caches = nullptr;
  const void* const* seqlens = nullptr;
  const int* table_lens = nullptr;     // entries of each block table (nullptr: all have table_len)
  const int64_t* num_pages = nullptr;  // pages of each cache (nullptr: all have num_pages)
  bool packed = false;
  const int* table0 = nullptr;
  int64_t table_step = 0;
  void* cache0 = nullptr;
  const int* len0 = nullptr;
};
// Checks and fills the parts every entry point shares. lens: whether the call reads context
// lengths; keep: whether packed slots stay so (else they become tables).
int fill_cache(Cache* c, const char* what, int nseg, const int* rows, const Slots& s, bool lens, bool keep, int table_len,
               int64_t num_pages, int hkv, int head_dim, int page);
// Row counts to row starts; the total is bounded so that row indices stay in 31 bits.
int fill_rows(RowSegments* s, const char* what, int nseg, const int* rows);
// The attention kernel's bounded-wait status on the current device; synchronous.
int read_and_clear_error(unsigned int* code);

}  // namespace kv4
}  // namespace swl
