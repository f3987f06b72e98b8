// Appending to the 4-bit paged cache and reading it back.
//
//  * kv4_append  rotates q and k of the new rows (NeoX pairs (i, i + D/2)),
//                writes rotated q (and k, for a prompt that attends to itself before
//                its cache is read), quantises k and v and writes their codes.
//  * kv4_gather  dequantises a range of each slot's tokens to packed bf16 rows.
//
// Rounding: the cos/sin table is bf16, so the four products of a rotated pair
// are exact in 32 bits and each result is rounded once (to fp32), then q_rot and k_rot
// once more to bf16; k is quantised from the fp32 result. Scale and minimum are rounded to bf16
// and the codes taken against the rounded pair: a value is off by at most half a step or, where
// the rounded ends leave it below code 0 or above code 15, by at most 2^-8 of the group's
// minimum and 2^-8 of its range. (A group of numbers far from zero pays for its bf16 minimum: between
// 100.3 and 100.4 that is 100.5, and every code is 0.) Division is IEEE: a
// quotient half way between two codes goes to the even one.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.h"
#include "kv4.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace swl {
namespace kv4 {

namespace {

struct AppendTable {
  RowSegments seg;
  int tile_start[kMaxSlots + 1];  // launch tiles: a slot's rows touch at most ceil((rows + 15) / 16) blocks
  const __nv_bfloat16* qkv[kMaxSlots];
  Cache c;
};
struct AppendParams {
  int hq;
  int64_t qkv_stride;
  const __nv_bfloat16* cos_sin;  // [max_pos, D]: cos (D/2) | sin (D/2)
  int max_pos;
  __nv_bfloat16* q_rot;          // [total_rows, hq * D]
  __nv_bfloat16* k_rot;          // [total_rows, hkv * D] or nullptr
  int heads_per_cta;
};

__device__ __forceinline__ int find_slot(const int* start, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint4 u;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  return u;
}
// NaN in a group makes its minimum and maximum NaN, and so the whole group.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// (s, m) of a group as stored: s in the low half, m in the high half.
__device__ __forceinline__ uint32_t group_pair(float lo, float hi) {
  const __nv_bfloat16 m = __float2bfloat16_rn(lo), s = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
  return static_cast<uint32_t>(__bfloat16_as_ushort(s)) | static_cast<uint32_t>(__bfloat16_as_ushort(m)) << 16;
}
__device__ __forceinline__ float pair_scale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float pair_min(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// The codes of 8 numbers: (x - m) / s rounded as IEEE division rounds it, then to
// the nearest integer, ties to even, within 0 .. 15. In the range where nothing under- or
// overflows the quotient comes from the rounded reciprocal r of s by Markstein's correction:
// q = a r, then q + r (a - q s). Here it gives the IEEE quotient, although q may be two ulp off,
// because s has 8 significant bits: a - q s is exact (10 bits), what the correction lacks is 2^-23
// ulp, and a / s lies at least 2^-9 ulp from the middle between two fp32 numbers (a middle
// times s, of 25 and up to 8 bits, is never a, and a multiple of the same unit). Elsewhere
// from a division. NaN (a group without a finite scale) ends as code 0.
__device__ __forceinline__ uint32_t codes8(const float (&x)[8], uint32_t pair) {
  const float s = pair_scale(pair), m = pair_min(pair);
  float q[8];
  if (s >= 0x1p-60f && s <= 0x1p60f) {
    const float r = __frcp_rn(s);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = __fsub_rn(x[e], m), q0 = __fmul_rn(a, r);
      q[e] = __fmaf_rn(r, __fmaf_rn(-q0, s, a), q0);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = s > 0.f ? __fdiv_rn(__fsub_rn(x[e], m), s) : 0.f;
  }
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e)  // adding 1.5 * 2^23 rounds and leaves the code in the low bits
    w |= (__float_as_uint(__fadd_rn(fminf(fmaxf(q[e], 0.f), 15.f), 12582912.f)) & 15u) << (4 * e);
  return w;
}

// CTA = (one block's 16 positions of a slot, heads_per_cta heads of q | k | v).
// TPH = D / 16 threads share a head: each holds 8 dimensions of the lower half
// and the 8 they are rotated with, which are one code word of K each; a warp
// holds 32 / TPH tokens, so the reductions over a group stay inside it. Memory bounds
// it (rows in, rotated rows and codes out): 6499 rows of 32 + 2 * 8 heads of 128 in 36.6 us,
// 154 MB at 4.2 TB/s; four CTAs an SM rather than three 39.2 -> 36.6.
template <int D>
__global__ void __launch_bounds__(256, 4) kv4_append_kernel(const __grid_constant__ AppendTable tab,
                                                         const AppendParams p) {
  constexpr int TPH = D / 16, TPW = 32 / TPH, TG = kBlockTok / TPW, HW = 8 / TG;  // HW heads side by side
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int s = find_slot(tab.tile_start, tab.seg.nseg, blockIdx.x);
  const int rows = tab.seg.row_start[s + 1] - tab.seg.row_start[s];
  const int64_t pos0 = *tab.c.seqlen[s];
  const int64_t tile = (pos0 >> 4) + (static_cast<int>(blockIdx.x) - tab.tile_start[s]);
  const int t = (warp % TG) * TPW + lane / TPH;  // token of the block
  const int64_t pos = tile * kBlockTok + t;
  const int64_t local = pos - pos0;
  const bool live = local >= 0 && local < rows;
  if (!__any_sync(0xffffffffu, live)) return;
  const int k = lane % TPH;
  const bool known = live && pos >= 0 && pos < p.max_pos;  // positions without an angle: zeros, nothing cached
  const int64_t gr = tab.seg.row_start[s] + local;
  float cs[8], sn[8];
  {
    uint4 a = make_uint4(0, 0, 0, 0), b = a;
    if (known) {
      const __nv_bfloat16* row = p.cos_sin + pos * D;
      a = *reinterpret_cast<const uint4*>(row + 8 * k);
      b = *reinterpret_cast<const uint4*>(row + D / 2 + 8 * k);
    }
    unpack8(a, cs);
    unpack8(b, sn);
  }
  const __nv_bfloat16* src = tab.qkv[s] + local * p.qkv_stride;
  const int hkv = tab.c.hkv;
  const int h0 = blockIdx.y * p.heads_per_cta, h1 = min(h0 + p.heads_per_cta, p.hq + 2 * hkv);
  uint4 u = make_uint4(0, 0, 0, 0), w = u;
  auto load = [&](int h) {
    if (known && h < h1) {
      u = *reinterpret_cast<const uint4*>(src + static_cast<int64_t>(h) * D + 8 * k);
      w = *reinterpret_cast<const uint4*>(src + static_cast<int64_t>(h) * D + D / 2 + 8 * k);
    }
  };
  load(h0 + warp / TG);
  for (int h = h0 + warp / TG; h < h1; h += HW) {
    float a[8], b[8];
    unpack8(u, a);
    unpack8(w, b);
    load(h + HW);  // the next head's rows are on their way while this one's are in work
    const bool is_v = h >= p.hq + hkv;
    if (!is_v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = a[e], y = b[e];
        a[e] = x * cs[e] - y * sn[e];
        b[e] = y * cs[e] + x * sn[e];
      }
      __nv_bfloat16* dst = h < p.hq ? p.q_rot + (gr * p.hq + h) * D
                                    : (p.k_rot ? p.k_rot + (gr * hkv + (h - p.hq)) * D : nullptr);
      if (live && dst) {
        *reinterpret_cast<uint4*>(dst + 8 * k) = pack8(a);
        *reinterpret_cast<uint4*>(dst + D / 2 + 8 * k) = pack8(b);
      }
      if (h < p.hq) continue;
    }
    // group minima and maxima: D = 128 has a group per half, D = 64 one over both
    float lo[2] = {a[0], b[0]}, hi[2] = {a[0], b[0]};
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      lo[0] = min_nan(lo[0], a[e]);
      hi[0] = max_nan(hi[0], a[e]);
      lo[1] = min_nan(lo[1], b[e]);
      hi[1] = max_nan(hi[1], b[e]);
    }
    if (D == 64) {
      lo[0] = lo[1] = min_nan(lo[0], lo[1]);
      hi[0] = hi[1] = max_nan(hi[0], hi[1]);
    }
#pragma unroll
    for (int o = 1; o < TPH; o <<= 1)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lo[i] = min_nan(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], o));
        hi[i] = max_nan(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], o));
      }
    const uint32_t pr[2] = {group_pair(lo[0], hi[0]), group_pair(lo[1], hi[1])};
    const uint32_t wa = codes8(a, pr[0]), wb = codes8(b, pr[1]);
    uint8_t* const blk = known ? block_of<D>(tab.c, s, tile, is_v ? h - p.hq - hkv : h - p.hq) : nullptr;
    if (!is_v) {
      if (blk) {
        *reinterpret_cast<uint32_t*>(blk + k_word<D>(t, 8 * k)) = wa;
        *reinterpret_cast<uint32_t*>(blk + k_word<D>(t, D / 2 + 8 * k)) = wb;
      }
    } else {
      // a V word holds 4 dimensions of two tokens: the even token's thread writes
      // the first 4 of its 8 dimensions for both, the odd token's the second 4;
      // a token whose neighbour is not written keeps to its own 16-bit pieces
      const bool odd = t & 1;
      const bool both = __shfl_xor_sync(0xffffffffu, static_cast<int>(blk != nullptr), TPH) && blk;
      const uint32_t ra = __shfl_xor_sync(0xffffffffu, odd ? wa & 0xffffu : wa >> 16, TPH);
      const uint32_t rb = __shfl_xor_sync(0xffffffffu, odd ? wb & 0xffffu : wb >> 16, TPH);
      if (both) {
        const int d4 = 8 * k + (odd ? 4 : 0);
        *reinterpret_cast<uint32_t*>(blk + v_piece<D>(t & ~1, d4)) = odd ? ra | (wa & 0xffff0000u) : (wa & 0xffffu) | ra << 16;
        *reinterpret_cast<uint32_t*>(blk + v_piece<D>(t & ~1, D / 2 + d4)) =
            odd ? rb | (wb & 0xffff0000u) : (wb & 0xffffu) | rb << 16;
      } else if (blk) {
        *reinterpret_cast<uint16_t*>(blk + v_piece<D>(t, 8 * k)) = static_cast<uint16_t>(wa);
        *reinterpret_cast<uint16_t*>(blk + v_piece<D>(t, 8 * k + 4)) = static_cast<uint16_t>(wa >> 16);
        *reinterpret_cast<uint16_t*>(blk + v_piece<D>(t, D / 2 + 8 * k)) = static_cast<uint16_t>(wb);
        *reinterpret_cast<uint16_t*>(blk + v_piece<D>(t, D / 2 + 8 * k + 4)) = static_cast<uint16_t>(wb >> 16);
      }
    }
    if (blk && k < D / kGroup)
      *reinterpret_cast<uint32_t*>(blk + (is_v ? v_pair_off(D) : k_pair_off(D)) + 4 * (t * (D / kGroup) + k)) = pr[k];
  }
}

struct GatherTable {
  RowSegments seg;                 // output rows of slot i
  int tile_start[kMaxSlots + 1];   // blocks that slot i's range touches
  int start[kMaxSlots];            // first token of slot i's range
  Cache c;
};

// CTA = one block of a slot and two kv heads: a thread turns 8 dimensions of one
// token and head at a time, 16 bytes out. 6499 tokens of 8 heads of 128: 7.4 us (all
// heads of a block in one CTA 10.0).
constexpr int kGatherHeads = 2;
template <int D>
__global__ void __launch_bounds__(256) kv4_gather_kernel(const __grid_constant__ GatherTable tab,
                                                         __nv_bfloat16* __restrict__ k_out,
                                                         __nv_bfloat16* __restrict__ v_out) {
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int s = find_slot(tab.tile_start, tab.seg.nseg, blockIdx.x);
  const int64_t tile = (tab.start[s] >> 4) + (static_cast<int>(blockIdx.x) - tab.tile_start[s]);
  const int rows = tab.seg.row_start[s + 1] - tab.seg.row_start[s];
  const int hkv = tab.c.hkv;
  constexpr int C = D / 8;
  const uint8_t* base = block_of<D>(tab.c, s, tile, 0);
#pragma unroll
  for (int i0 = 0; i0 < kBlockTok * kGatherHeads * C; i0 += 256) {
    const int i = i0 + threadIdx.x;
    const int t = i / (kGatherHeads * C), h = blockIdx.y * kGatherHeads + i / C % kGatherHeads, d = i % C * 8;
    const int64_t local = tile * kBlockTok + t - tab.start[s];
    if (local < 0 || local >= rows || h >= hkv) continue;
    float kv[8], vv[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) kv[e] = vv[e] = 0.f;  // a page that is not there: zeros
    if (base) {
      const uint8_t* blk = base + static_cast<int64_t>(h) * block_bytes(D);
      const int po = 4 * (t * (D / kGroup) + d / kGroup);
      const uint32_t kp = *reinterpret_cast<const uint32_t*>(blk + k_pair_off(D) + po);
      const uint32_t vp = *reinterpret_cast<const uint32_t*>(blk + v_pair_off(D) + po);
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(blk + k_word<D>(t, d));
      const uint32_t vw = *reinterpret_cast<const uint16_t*>(blk + v_piece<D>(t, d)) |
                          static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(blk + v_piece<D>(t, d + 4))) << 16;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        kv[e] = pair_scale(kp) * static_cast<float>(kw >> (4 * e) & 15u) + pair_min(kp);
        vv[e] = pair_scale(vp) * static_cast<float>(vw >> (4 * e) & 15u) + pair_min(vp);
      }
    }
    const int64_t o = ((tab.seg.row_start[s] + local) * hkv + h) * D + d;
    *reinterpret_cast<uint4*>(k_out + o) = pack8(kv);
    *reinterpret_cast<uint4*>(v_out + o) = pack8(vv);
  }
}

}  // namespace

int fill_rows(RowSegments* s, const char* what, int nseg, const int* rows) {
  if (nseg < 0 || nseg > kMaxSlots) return set_error(SWL_ERR_ARG, "%s: segment count %d outside 0..%d", what, nseg, kMaxSlots);
  if (nseg > 0 && !rows) return set_error(SWL_ERR_ARG, "%s: null row counts", what);
  int64_t acc = 0;
  s->nseg = nseg;
  for (int i = 0; i < nseg; ++i) {
    if (rows[i] < 0) return set_error(SWL_ERR_ARG, "%s: negative row count", what);
    s->row_start[i] = static_cast<int>(acc);
    acc += rows[i];
    if (acc > (int64_t{1} << 30)) return set_error(SWL_ERR_ARG, "%s: more than 2^30 rows", what);
  }
  s->row_start[nseg] = s->total_rows = static_cast<int>(acc);
  return SWL_OK;
}

int fill_cache(Cache* c, const char* what, int nseg, const int* rows, const Slots& s, bool lens, bool keep, int table_len,
               int64_t num_pages, int hkv, int head_dim, int page) {
  if (head_dim != 64 && head_dim != 128) return set_error(SWL_ERR_ARG, "%s: head_dim must be 64 or 128", what);
  if (hkv < 1 || hkv > 1024) return set_error(SWL_ERR_ARG, "%s: kv heads outside 1..1024", what);
  if (page < kBlockTok || page > 1024 || (page & (page - 1)))
    return set_error(SWL_ERR_ARG, "%s: page must be 16, 32, 64, .. 1024 tokens", what);
  // a slot without rows in this call is not looked at: it may have no table, cache or rows at all
  const bool any = std::any_of(rows, rows + nseg, [](int r) { return r > 0; });
  const auto empty = [&] { return set_error(SWL_ERR_ARG, "%s: empty block table or cache", what); };
  if (any && ((!s.table_lens && table_len < 1) || (!s.num_pages && num_pages < 1))) return empty();
  const auto bounded = [](int64_t pages) { return static_cast<uint32_t>(std::min(pages, int64_t{1} << 31)); };
  c->table_len0 = table_len;
  c->pages0 = bounded(num_pages);
  c->hkv = hkv;
  c->page_shift = 0;
  while ((kBlockTok << c->page_shift) < page) ++c->page_shift;
  c->rows_each = nseg > 0 ? rows[0] : 0;
  for (int i = 1; i < nseg; ++i)
    if (rows[i] != rows[0]) c->rows_each = 0;
  c->packed = s.packed && keep;
  c->table0 = s.table0;
  c->table_step = s.table_step;
  c->cache0 = static_cast<uint8_t*>(s.cache0);
  c->len0 = s.len0;
  if (!any) return SWL_OK;
  if (s.packed ? !s.table0 || !s.cache0 || (lens && !s.len0) : !s.block_tables || !s.caches || (lens && !s.seqlens))
    return set_error(SWL_ERR_ARG, "%s: null block tables, caches or context lengths", what);
  uintptr_t align = reinterpret_cast<uintptr_t>(s.cache0);
  for (int i = 0; i < nseg && !c->packed; ++i) {
    const int entries = s.table_lens ? s.table_lens[i] : table_len;
    const int64_t pages = s.num_pages ? s.num_pages[i] : num_pages;
    c->table_len[i] = entries;
    c->pages[i] = bounded(pages);
    if (rows[i] == 0) continue;
    if (entries < 1 || pages < 1) return empty();
    c->block_table[i] = s.packed ? s.table0 + i * s.table_step : static_cast<const int*>(s.block_tables[i]);
    c->cache[i] = static_cast<uint8_t*>(s.packed ? s.cache0 : s.caches[i]);
    c->seqlen[i] = !lens ? nullptr : s.packed ? s.len0 + i : static_cast<const int*>(s.seqlens[i]);
    if (!c->block_table[i] || !c->cache[i] || (lens && !c->seqlen[i]))
      return set_error(SWL_ERR_ARG, "%s: null per-slot pointer", what);
    align |= reinterpret_cast<uintptr_t>(c->cache[i]);
  }
  if (align & 15) return set_error(SWL_ERR_ARG, "%s: caches must be 16-byte aligned", what);
  return SWL_OK;
}

namespace {

// swl_kv4_append: qkv0 for packed rows, else a pointer per slot.
int append(int nseg, const int* rows, const void* qkv0, const void* const* qkv, int64_t qkv_stride, const Slots& slots,
           int table_len, int64_t num_pages, int hq, int hkv, int head_dim, int page, const void* cos_sin, int max_pos,
           void* q_rot, void* k_rot, void* stream) {
  AppendTable t;
  SWL_TRY(fill_rows(&t.seg, "kv4_append", nseg, rows));
  SWL_TRY(fill_cache(&t.c, "kv4_append", nseg, rows, slots, true, false, table_len, num_pages, hkv, head_dim, page));
  if (hq < 1 || hq > 4096) return set_error(SWL_ERR_ARG, "kv4_append: query heads outside 1..4096");
  if (qkv_stride < static_cast<int64_t>(hq + 2 * hkv) * head_dim || qkv_stride % 8)
    return set_error(SWL_ERR_ARG, "kv4_append: row stride must hold all heads and be a multiple of 8");
  if (t.seg.total_rows == 0) return SWL_OK;
  if (max_pos < 1 || !cos_sin || !q_rot) return set_error(SWL_ERR_ARG, "kv4_append: null or empty cos/sin table, or null q_rot");
  uintptr_t align = reinterpret_cast<uintptr_t>(cos_sin) | reinterpret_cast<uintptr_t>(q_rot) |
                    reinterpret_cast<uintptr_t>(k_rot) | reinterpret_cast<uintptr_t>(qkv0);
  if (!qkv && !qkv0) return set_error(SWL_ERR_ARG, "kv4_append: null rows");
  int64_t tiles = 0;
  for (int i = 0; i < nseg; ++i) {
    t.qkv[i] = qkv0 ? static_cast<const __nv_bfloat16*>(qkv0) + t.seg.row_start[i] * qkv_stride
                    : static_cast<const __nv_bfloat16*>(qkv[i]);
    t.tile_start[i] = static_cast<int>(tiles);
    if (rows[i] == 0) continue;
    if (!t.qkv[i]) return set_error(SWL_ERR_ARG, "kv4_append: null per-slot pointer");
    align |= reinterpret_cast<uintptr_t>(t.qkv[i]);
    tiles += (rows[i] + 30) / 16;
  }
  t.tile_start[nseg] = static_cast<int>(tiles);
  if (align & 15) return set_error(SWL_ERR_ARG, "kv4_append: rows, cos/sin table and outputs must be 16-byte aligned");
  AppendParams p;
  p.hq = hq;
  p.qkv_stride = qkv_stride;
  p.cos_sin = static_cast<const __nv_bfloat16*>(cos_sin);
  p.max_pos = max_pos;
  p.q_rot = static_cast<__nv_bfloat16*>(q_rot);
  p.k_rot = static_cast<__nv_bfloat16*>(k_rot);
  // One pass of heads a CTA while there are few CTAs (28 single tokens: 12.3 -> 5.7 us), four
  // passes, each loading ahead of the last, when there are many.
  const int side = head_dim == 128 ? 2 : 4, heads = hq + 2 * hkv;
  p.heads_per_cta = tiles * ((heads + side - 1) / side) <= 148 * 8 ? side : 4 * side;
  const dim3 grid(static_cast<unsigned>(tiles), (heads + p.heads_per_cta - 1) / p.heads_per_cta);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  SWL_CUDA_TRY(head_dim == 128 ? launch_kernel(kv4_append_kernel<128>, grid, dim3(256), 0, st, 1, t, p)
                               : launch_kernel(kv4_append_kernel<64>, grid, dim3(256), 0, st, 1, t, p));
  return SWL_OK;
}

int gather(int nseg, const int* starts, const int* lens, const Slots& slots, int table_len, int64_t num_pages, int hkv,
           int head_dim, int page, void* k_out, void* v_out, void* stream) {
  GatherTable t;
  SWL_TRY(fill_rows(&t.seg, "kv4_gather", nseg, lens));
  SWL_TRY(fill_cache(&t.c, "kv4_gather", nseg, lens, slots, false, false, table_len, num_pages, hkv, head_dim, page));
  if (t.seg.total_rows == 0) return SWL_OK;
  if (!starts) return set_error(SWL_ERR_ARG, "kv4_gather: null starts");
  if (!k_out || !v_out || ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15))
    return set_error(SWL_ERR_ARG, "kv4_gather: outputs must be 16-byte aligned");
  int64_t tiles = 0;
  for (int i = 0; i < nseg; ++i) {
    const int64_t end = static_cast<int64_t>(starts[i]) + lens[i];
    if (starts[i] < 0 || end > static_cast<int64_t>(t.c.table_len[i]) * page)
      return set_error(SWL_ERR_ARG, "kv4_gather: tokens %d..%lld of slot %d lie outside its block table", starts[i],
                       static_cast<long long>(end), i);
    t.start[i] = starts[i];
    t.tile_start[i] = static_cast<int>(tiles);
    if (lens[i]) tiles += (end - 1) / 16 - starts[i] / 16 + 1;
  }
  t.tile_start[nseg] = static_cast<int>(tiles);
  const dim3 grid(static_cast<unsigned>(tiles), (hkv + kGatherHeads - 1) / kGatherHeads);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  __nv_bfloat16 *ko = static_cast<__nv_bfloat16*>(k_out), *vo = static_cast<__nv_bfloat16*>(v_out);
  SWL_CUDA_TRY(head_dim == 128 ? launch_kernel(kv4_gather_kernel<128>, grid, dim3(256), 0, st, 1, t, ko, vo)
                               : launch_kernel(kv4_gather_kernel<64>, grid, dim3(256), 0, st, 1, t, ko, vo));
  return SWL_OK;
}

}  // namespace
}  // namespace kv4
}  // namespace swl

using namespace swl;

SWL_EXPORT int64_t swl_kv4_block_bytes(int head_dim) {
  return head_dim == 64 || head_dim == 128 ? kv4::block_bytes(head_dim) : 0;
}

SWL_EXPORT int swl_kv4_append(int nseg, const int* rows, const void* const* qkv, int64_t qkv_stride,
                              const void* const* block_tables, int table_len, void* const* caches,
                              int64_t num_pages, const void* const* seqlens, int hq, int hkv, int head_dim,
                              int page, const void* cos_sin, int max_pos, void* q_rot, void* k_rot,
                              void* stream) {
  kv4::Slots s;
  s.block_tables = block_tables;
  s.caches = caches;
  s.seqlens = seqlens;
  return kv4::append(nseg, rows, nullptr, qkv, qkv_stride, s, table_len, num_pages, hq, hkv, head_dim, page, cos_sin, max_pos,
                     q_rot, k_rot, stream);
}

SWL_EXPORT int swl_kv4_append_each(int nseg, const int* rows, const void* const* qkv, int64_t qkv_stride,
                                   const void* const* block_tables, const int* table_lens, void* const* caches,
                                   const int64_t* num_pages, const void* const* seqlens, int hq, int hkv, int head_dim,
                                   int page, const void* cos_sin, int max_pos, void* q_rot, void* k_rot, void* stream) {
  if (nseg > 0 && (!table_lens || !num_pages)) return set_error(SWL_ERR_ARG, "kv4_append: null table lengths or page counts");
  kv4::Slots s;
  s.block_tables = block_tables;
  s.caches = caches;
  s.seqlens = seqlens;
  s.table_lens = table_lens;
  s.num_pages = num_pages;
  return kv4::append(nseg, rows, nullptr, qkv, qkv_stride, s, 1, 1, hq, hkv, head_dim, page, cos_sin, max_pos, q_rot, k_rot,
                     stream);
}

SWL_EXPORT int swl_kv4_append_packed(int nseg, const int* rows, const void* qkv, int64_t qkv_stride, const int* block_tables,
                                     int64_t table_stride, int table_len, void* cache, int64_t num_pages, const int* seqlens,
                                     int hq, int hkv, int head_dim, int page, const void* cos_sin, int max_pos, void* q_rot,
                                     void* k_rot, void* stream) {
  kv4::Slots s;
  s.packed = true;
  s.table0 = block_tables;
  s.table_step = table_stride;
  s.cache0 = cache;
  s.len0 = seqlens;
  return kv4::append(nseg, rows, qkv, nullptr, qkv_stride, s, table_len, num_pages, hq, hkv, head_dim, page, cos_sin, max_pos,
                     q_rot, k_rot, stream);
}

SWL_EXPORT int swl_kv4_gather(int nseg, const int* starts, const int* lens, const void* const* block_tables,
                              int table_len, const void* const* caches, int64_t num_pages, int hkv,
                              int head_dim, int page, void* k_out, void* v_out, void* stream) {
  kv4::Slots s;
  s.block_tables = block_tables;
  s.caches = const_cast<void* const*>(caches);
  return kv4::gather(nseg, starts, lens, s, table_len, num_pages, hkv, head_dim, page, k_out, v_out, stream);
}

SWL_EXPORT int swl_kv4_gather_each(int nseg, const int* starts, const int* lens, const void* const* block_tables,
                                   const int* table_lens, const void* const* caches, const int64_t* num_pages, int hkv,
                                   int head_dim, int page, void* k_out, void* v_out, void* stream) {
  if (nseg > 0 && (!table_lens || !num_pages)) return set_error(SWL_ERR_ARG, "kv4_gather: null table lengths or page counts");
  kv4::Slots s;
  s.block_tables = block_tables;
  s.caches = const_cast<void* const*>(caches);
  s.table_lens = table_lens;
  s.num_pages = num_pages;
  return kv4::gather(nseg, starts, lens, s, 1, 1, hkv, head_dim, page, k_out, v_out, stream);
}

SWL_EXPORT int swl_kv4_gather_packed(int nseg, const int* starts, const int* lens, const int* block_tables,
                                     int64_t table_stride, int table_len, const void* cache, int64_t num_pages, int hkv,
                                     int head_dim, int page, void* k_out, void* v_out, void* stream) {
  kv4::Slots s;
  s.packed = true;
  s.table0 = block_tables;
  s.table_step = table_stride;
  s.cache0 = const_cast<void*>(cache);
  return kv4::gather(nseg, starts, lens, s, table_len, num_pages, hkv, head_dim, page, k_out, v_out, stream);
}
