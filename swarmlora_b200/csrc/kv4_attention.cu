// Causal GQA attention of each slot's newest rows over its paged 4-bit cache.
//
// The work is the cache's bytes: 18 D per 16 tokens and kv head, read once. One
// block (16 tokens of one kv head) is one contiguous piece, which a warp fetches with a single
// bulk copy into its own ring and turns into matrix fragments without any
// value being scaled on its own: a nibble v becomes the bf16 number 128 + v by
// one logic operation on two nibbles (0x4300 | v), and scales and minima are
// applied where they are cheap.
//
//   scores   q.k = sum over groups  s (sum q v) + m (sum q)
//            per token and query column, after the product, whose accumulator starts at
//            -128 sum q (known per piece) and so ends as sum q v.
//   values   o = sum over tokens  p s (128 + v) + p m - 128 p s
//            p s is rounded to bf16 as the second operand; the product with a
//            row of ones gives the sum of the same rounded numbers, so the 128 cancels
//            exactly but for fp32's sums. p m is summed in fp32.
//
// Tokens are the M dimension of the score product and dimensions that of the value
// product; the columns are the slot's new rows times the query heads of the kv
// head (8 NT of them a pass). The weights go from one layout to the other as fp16,
// times 2^7, through a transposing register move: they are at most 2^8 by the lazy
// reference, so that each is off by 2^-11 of itself or, below 2^-21, by 2^-32 (unscaled, a
// long flat tail behind one large score would fall below fp16's smallest number, 2^-24, and be lost:
// the sum of the weights keeps it). The reference maximum moves only when a score passes it
// by 2^8, so the common step needs one vote instead of a reduction.
//
// Work is shared out on the device, which alone knows the context lengths: with
// short contexts a CTA takes whole (slot, kv head) pairs; otherwise every CTA takes an equal
// contiguous range of all blocks, a pair cut by a range boundary leaves partial
// records (at most two a CTA) and a second launch joins them.
//
// What bounds it: integer logic, which runs at half rate. Turning a block's codes into operands
// is 112 of the 200 or so logic operations it takes, a fifth of the time; without any
// arithmetic the copies alone take 73 us where the whole takes 103 (16 slots of 16k-32k
// tokens, 8 kv heads of 128: 435 MB, 4.2 TB/s; 28 slots of 256-768 tokens 12.8 us). Four
// warps with 168 registers, three CTAs an SM: 113 us before blocks shared their scores, against
// 119 with 16 warps of 128 registers and 124 with 8 of 255. Measured and left out: fp8 operands for
// the score product (208 us, the warp-level product is slow in that type), two-byte fixed-point
// queries (111 against 113), shifts by multiplication (134).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "kv4.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace swl {
namespace kv4 {

namespace {

__device__ unsigned int g_kv4_error_word = 0;
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr unsigned kErrBlock = 111;
constexpr float kRescaleLog2 = 8.f;
// The weights are taken 2^7 times as large until they have been fp16: 2^8 * 2^7 is half of its range. (Left
// so for the sums as well, drafts take 55.5 us for 56.0, but values would overflow 2^7 sooner.)
constexpr float kHalfUp = 7.f, kHalfDown = 1.f / 128.f;
constexpr int kWarps = 4, kManyWarps = 6;  // of a CTA; the larger where whole pairs leave SMs half empty

struct AttnTable4 {
  RowSegments seg;
  int passes_each;               // column passes of every slot where all have as many rows
  __nv_bfloat16* out0;           // packed rows, or nullptr
  __nv_bfloat16* out[kMaxSlots];
  Cache c;
};
struct AttnParams4 {
  int hq, group;           // query heads, query heads per kv head
  int64_t out_stride;
  float scale_log2, inv_scale;
  int max_len;
  const __nv_bfloat16* q;  // [total_rows, hq * D]
  int whole;               // 1: CTAs take whole pairs; 0: equal ranges
  int pairs;               // (slot, kv head, pass)es in all
  float* part;             // equal ranges: O [record][column][D], then (m, l) [record][column][2]
};

template <int D, int NT, int NW>
struct Cfg4 {
  static constexpr int W = D / 32, NG = D / kGroup, kBlock = block_bytes(D);
  static constexpr int kStages = (NT == 1 ? 2 : 3) * (128 / D);  // of two blocks
  static constexpr int kCols = 8 * NT;
  static constexpr int kLd = D + 4;  // floats between columns of the merge buffer: no bank twice in a quarter warp
  static constexpr int kRing = NW * kStages * 2 * kBlock;
  static constexpr int kMerge = NW * 8 * kLd * 4;
  static constexpr int kSmem = kRing + kMerge;
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Two fp32 products in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_c(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                           uint32_t b1, float c0, float c1) {  // C: (c0, c1) in both halves of the rows
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
// Two nibbles (bits 0-3 of each half) as bf16 128 + v.
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
  uint32_t r;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(r) : "r"(w));  // (w & mask) | 128.0 twice
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <int N>
__device__ __forceinline__ void lds(const uint8_t* p, uint32_t* r) {
  if constexpr (N == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    r[0] = u.x; r[1] = u.y; r[2] = u.z; r[3] = u.w;
  } else if constexpr (N == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    r[0] = u.x; r[1] = u.y;
  } else {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
__device__ __forceinline__ float scale_of(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float min_of(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// The division of the work, the same in every CTA and in the joining launch.
struct Shares {
  int blocks[kMaxSlots];          // cache blocks of each slot's context
  int passes[kMaxSlots];          // column passes
  int64_t unit[kMaxSlots + 1];    // blocks x kv heads x passes ahead of slot i
  int pair[kMaxSlots + 1];        // kv heads x passes ahead of slot i
  int64_t per_cta;
};
// A piece: blocks [b0, b1) of one (slot, kv head, pass).
struct Piece {
  int slot, head, pass, b0, b1, blocks;
};

// Cache blocks of a slot's context with its new rows.
__device__ __forceinline__ int blocks_of(const AttnTable4& tab, const AttnParams4& p, int s, int rows) {
  const int64_t len = min(static_cast<int64_t>(*len_of(tab.c, s)) + rows, static_cast<int64_t>(p.max_len));
  return static_cast<int>((max(len, int64_t{1}) + kBlockTok - 1) / kBlockTok);
}

template <int D, int NT>
__device__ __forceinline__ void share_out(const AttnTable4& tab, const AttnParams4& p, Shares* sh, int ctas) {
  if (threadIdx.x < 32) {
    int64_t u = 0;
    int pr = 0;
    for (int s0 = 0; s0 < tab.seg.nseg; s0 += 32) {
      const int s = s0 + threadIdx.x;
      int nb = 0, np = 0;
      if (s < tab.seg.nseg) {
        const int rows = row_of(tab.c, tab.seg, s + 1) - row_of(tab.c, tab.seg, s);
        if (rows > 0) {
          nb = blocks_of(tab, p, s, rows);
          np = (rows * p.group + 8 * NT - 1) / (8 * NT) * tab.c.hkv;
        }
        sh->blocks[s] = nb;
        sh->passes[s] = np / tab.c.hkv;
      }
      int64_t a = static_cast<int64_t>(nb) * np;
      int b = np;
      const int64_t a0 = a;
      const int b0 = b;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, a, o);
        const int y = __shfl_up_sync(0xffffffffu, b, o);
        if (static_cast<int>(threadIdx.x) >= o) {
          a += x;
          b += y;
        }
      }
      if (s < tab.seg.nseg) {
        sh->unit[s] = u + a - a0;
        sh->pair[s] = pr + b - b0;
      }
      u += __shfl_sync(0xffffffffu, a, 31);
      pr += __shfl_sync(0xffffffffu, b, 31);
    }
    if (threadIdx.x == 0) {
      sh->unit[tab.seg.nseg] = u;
      sh->pair[tab.seg.nseg] = pr;
      sh->per_cta = max((u + ctas - 1) / ctas, int64_t{2 * kWarps});
    }
  }
  __syncthreads();
}

__device__ __forceinline__ int find_pair(const Shares& sh, int n, int pair) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (sh.pair[mid] <= pair) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Walks the pieces of this CTA.
struct Walk {
  int64_t u, end;  // equal ranges: next unit; whole pairs: next pair
  __device__ __forceinline__ Walk(const Shares& sh, const AttnTable4& tab, const AttnParams4& p) {
    if (p.whole) {
      u = blockIdx.x;
      end = p.pairs;
    } else {
      u = min(blockIdx.x * sh.per_cta, sh.unit[tab.seg.nseg]);
      end = min(u + sh.per_cta, sh.unit[tab.seg.nseg]);
    }
  }
  __device__ __forceinline__ bool next(const Shares& sh, const AttnTable4& tab, const AttnParams4& p, Piece* x) {
    if (u >= end) return false;
    const int n = tab.seg.nseg;
    if (p.whole) {
      int i = static_cast<int>(u), passes;
      if (tab.c.rows_each) {  // nothing to look up
        passes = tab.passes_each;
        x->slot = i / (passes * tab.c.hkv);
        i -= x->slot * passes * tab.c.hkv;
        x->blocks = blocks_of(tab, p, x->slot, tab.c.rows_each);
      } else {
        x->slot = find_pair(sh, n, i);
        i -= sh.pair[x->slot];
        passes = sh.passes[x->slot];
        x->blocks = sh.blocks[x->slot];
      }
      x->head = i / passes;
      x->pass = i % passes;
      x->b0 = 0;
      x->b1 = x->blocks;
      u += gridDim.x;
      return true;
    }
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (sh.unit[mid] <= u) lo = mid;
      else hi = mid - 1;
    }
    const int64_t r = u - sh.unit[lo];
    const int nb = sh.blocks[lo], i = static_cast<int>(r / nb);
    x->slot = lo;
    x->head = i / sh.passes[lo];
    x->pass = i % sh.passes[lo];
    x->blocks = nb;
    x->b0 = static_cast<int>(r - static_cast<int64_t>(i) * nb);
    x->b1 = static_cast<int>(min(static_cast<int64_t>(nb), x->b0 + (end - u)));
    u += x->b1 - x->b0;
    return true;
  }
};

// kDual (columns up to 4, NT = 1): columns 4 .. 7 repeat the queries of 0 .. 3; the first
// four go with the first block of a pair and the other four with its second, so that
// scores, exponentials and weights of two blocks are computed at once (columns
// that would otherwise be empty). The two sets keep their own references and meet at the merge.
template <int D, int NT, bool kDual, int NW>
__global__ void __launch_bounds__(NW * 32, NT == 1 && NW == kWarps ? 3 : 2)
    kv4_attention_kernel(const __grid_constant__ AttnTable4 tab, const __grid_constant__ AttnParams4 p) {
  using C = Cfg4<D, NT, NW>;
  constexpr int W = C::W, NG = C::NG, ST = C::kStages;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ Shares sh;
  __shared__ __align__(8) uint64_t bars[NW][ST];
  __shared__ float ml_sm[NW][8][2], corr_sm[NW][8][NG];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, c = lane & 3;
  uint8_t* const ring = dyn + warp * ST * 2 * C::kBlock;
  float* const merge = reinterpret_cast<float*>(dyn + C::kRing);
  if (lane == 0) {
    for (int i = 0; i < ST; ++i) ptx::mbar_init(&bars[warp][i], 1);
    ptx::fence_mbar_init();
  }
  __syncwarp();  // a warp's barriers are its own
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  if (!p.whole || !tab.c.rows_each) share_out<D, NT>(tab, p, &sh, gridDim.x);

  // A piece's queries are asked for before anything else of it: column g's dimensions 8 c .. of each 32.
  uint4 uq[NT][W];
  auto load_q = [&](const Piece& x) {
    const int row0 = row_of(tab.c, tab.seg, x.slot), ncols = (row_of(tab.c, tab.seg, x.slot + 1) - row0) * p.group;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = x.pass * C::kCols + (kDual ? g & 3 : nt * 8 + g);
      const __nv_bfloat16* src =
          p.q + (static_cast<int64_t>(row0 + col / p.group) * p.hq + x.head * p.group + col % p.group) * D;
#pragma unroll
      for (int j = 0; j < W; ++j)
        uq[nt][j] = col < ncols ? *reinterpret_cast<const uint4*>(src + 32 * j + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  Walk cw(sh, tab, p);
  Piece x;
  constexpr bool kAhead = NT == 1;  // two tiles of columns have no registers to spare for it
  bool have = cw.next(sh, tab, p, &x);
  if (have && kAhead) load_q(x);

  // ---- loads: this warp's pairs of blocks in the order in which it will use them ----
  Walk lw(sh, tab, p);
  Piece lp;
  bool more = lw.next(sh, tab, p, &lp);
  int lb = more ? lp.b0 + 2 * warp : 0;   // next block of the load piece that is not in the batch
  const uint8_t *addr0 = nullptr, *addr1 = nullptr;  // lane i: the batch's i-th pair (nullptr: no such block), which it fetches
  int batch = 0, taken = 0, issued = 0;
  uint32_t ok0 = 0, ok1 = 0, ring_ok = 0;  // a bit per batch entry; two bits per stage: the blocks exist
  auto issue = [&]() {
    while (more && taken == batch) {      // the next up to 32 pairs of this warp
      const int left = lp.b1 > lb ? (lp.b1 - lb + 2 * NW - 1) / (2 * NW) : 0;
      if (left == 0) {
        more = lw.next(sh, tab, p, &lp);
        lb = lp.b0 + 2 * warp;
        continue;
      }
      batch = min(left, 32);
      taken = 0;
      const int b = lb + lane * 2 * NW;
      addr0 = lane < batch ? block_of<D, true>(tab.c, lp.slot, b, lp.head) : nullptr;
      addr1 = lane < batch && b + 1 < lp.b1 ? block_of<D, true>(tab.c, lp.slot, b + 1, lp.head) : nullptr;
      ok0 = __ballot_sync(0xffffffffu, addr0 != nullptr);
      ok1 = __ballot_sync(0xffffffffu, addr1 != nullptr);
      lb += batch * 2 * NW;
    }
    if (!more) return;
    const int st = issued % ST;
    ring_ok = (ring_ok & ~(3u << 2 * st)) | ((ok0 >> taken & 1u) | (ok1 >> taken & 1u) << 1) << 2 * st;
    if (lane == taken) {
      uint64_t* const bar = &bars[warp][st];
      ptx::mbar_arrive_expect_tx(bar, (addr0 ? C::kBlock : 0) + (addr1 ? C::kBlock : 0));
      if (addr0) ptx::bulk_load(ring + st * 2 * C::kBlock, addr0, C::kBlock, bar);
      if (addr1) ptx::bulk_load(ring + (st * 2 + 1) * C::kBlock, addr1, C::kBlock, bar);
    }
    ++taken;
    ++issued;
  };
#pragma unroll 1
  for (int i = 0; i < ST - 1; ++i) issue();

  int used = 0;
  uint64_t limit = kWaitNs;  // after a wait that gave up the others give up soon
  while (have) {
    if (!kAhead) load_q(x);
    const int row0 = row_of(tab.c, tab.seg, x.slot), rows = row_of(tab.c, tab.seg, x.slot + 1) - row0;
    const int ncols = rows * p.group, col0 = x.pass * C::kCols;
    const int64_t len0 = *len_of(tab.c, x.slot);
    // ---- this piece's query columns: B fragments, sums per group, visible lengths ----
    uint32_t qb[NT][2 * W][2];
    float qs[NT][NG][2], qo[NT][NG][2];  // sum q, and -128 sum q
    int seen[NT][2], seen_g[NT];  // tokens that columns 2c, 2c + 1 and column g see
    auto sees = [&](int col) {
      const int64_t n = min(len0 + col / p.group + 1, static_cast<int64_t>(p.max_len));
      return col < ncols ? static_cast<int>(max(n, int64_t{0})) : 0;
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = col0 + (kDual ? g & 3 : nt * 8 + g);
      float part[NG];
#pragma unroll
      for (int i = 0; i < NG; ++i) part[i] = 0.f;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const uint4 u = uq[nt][j];
        qb[nt][2 * j][0] = __byte_perm(u.x, u.z, 0x5410);
        qb[nt][2 * j][1] = __byte_perm(u.x, u.z, 0x7632);
        qb[nt][2 * j + 1][0] = __byte_perm(u.y, u.w, 0x5410);
        qb[nt][2 * j + 1][1] = __byte_perm(u.y, u.w, 0x7632);
        const uint32_t w4[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          part[j / 2] += __uint_as_float(w4[e] << 16) + __uint_as_float(w4[e] & 0xffff0000u);
      }
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        part[i] += __shfl_xor_sync(0xffffffffu, part[i], 1);
        part[i] += __shfl_xor_sync(0xffffffffu, part[i], 2);
        qs[nt][i][0] = __shfl_sync(0xffffffffu, part[i], 8 * c);
        qs[nt][i][1] = __shfl_sync(0xffffffffu, part[i], 8 * c + 4);
        qo[nt][i][0] = -128.f * qs[nt][i][0];
        qo[nt][i][1] = -128.f * qs[nt][i][1];
      }
      const int c2 = kDual ? 2 * c & 3 : nt * 8 + 2 * c;
      seen[nt][0] = sees(col0 + c2);
      seen[nt][1] = sees(col0 + c2 + 1);
      seen_g[nt] = sees(col);
    }
    // from this block on some column does not see all of two blocks (the pass's first column belongs to its first row)
    const int edge_from = sees(col0) / kBlockTok - 1;
    // m: reference (scaled, base 2), nm: 7 - m, bar_: the raw score that moves it, l: sum of the weights times 2^7
    float o[NT][2 * W][4], ps[NT][NG][4], corr[NT][NG], m[NT][2], nm[NT][2], bar_[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        ps[nt][i][0] = ps[nt][i][1] = ps[nt][i][2] = ps[nt][i][3] = 0.f;
        corr[nt][i] = 0.f;
      }
      m[nt][0] = m[nt][1] = bar_[nt][0] = bar_[nt][1] = -INFINITY;
      nm[nt][0] = nm[nt][1] = 0.f;
      l[nt][0] = l[nt][1] = 0.f;
    }
    // Sums q v of N blocks (from blk on) and each group: tokens g, g + 8 and columns 2c, 2c + 1. The
    // chains of dependent products (a group of a block each) take turns.
    auto product = [&](const uint8_t* blk, auto& acc) {
      constexpr int N = sizeof(acc) / sizeof(acc[0]);
      uint32_t kw[N][2][W];
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) lds<W>(blk + i * C::kBlock + (h * 32 + lane) * W * 4, kw[i][h]);
#pragma unroll
      for (int step = 0; step < 4; ++step)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int gr = 0; gr < NG; ++gr) {
            const int j = 2 * gr + step / 2, e = step & 1;
            const uint32_t a0 = codes2(kw[i][0][j] >> (8 * e)), a1 = codes2(kw[i][1][j] >> (8 * e));
            const uint32_t a2 = codes2(kw[i][0][j] >> (8 * e + 4)), a3 = codes2(kw[i][1][j] >> (8 * e + 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (step == 0)  // the accumulator starts at -128 sum q
                mma16816_c(acc[i][nt][gr], a0, a1, a2, a3, qb[nt][2 * j][0], qb[nt][2 * j][1], qo[nt][gr][0], qo[nt][gr][1]);
              else
                mma16816(acc[i][nt][gr], a0, a1, a2, a3, qb[nt][2 * j + e][0], qb[nt][2 * j + e][1]);
            }
          }
    };
    // Their raw scores. edge: some column does not see all of the tokens (from tok0 on); a block
    // that is not there is seen by none.
    auto scores = [&](const uint8_t* blk, int tok0, bool there, const float (&acc)[NT][NG][4], float (&sc)[NT][4], auto edge_) {
      constexpr bool edge = decltype(edge_)::value;
      uint32_t kp[2][NG];
#pragma unroll
      for (int h = 0; h < 2; ++h) lds<NG>(blk + k_pair_off(D) + (h * 8 + g) * NG * 4, kp[h]);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float v = fmaf(min_of(kp[h][0]), qs[nt][0][k], scale_of(kp[h][0]) * acc[nt][0][2 * h + k]);
#pragma unroll
            for (int i = 1; i < NG; ++i)
              v = fmaf(min_of(kp[h][i]), qs[nt][i][k], fmaf(scale_of(kp[h][i]), acc[nt][i][2 * h + k], v));
            if (edge && (!there || tok0 + g + 8 * h >= seen[nt][k])) v = -INFINITY;
            sc[nt][2 * h + k] = v;
          }
    };
    // Moves the references to the largest of n scores a thread, and what is summed with them.
    auto rescale = [&](const float (&sc)[2][NT][4], int n) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float mx = fmaxf(sc[0][nt][k], sc[0][nt][2 + k]);
            if (n > 1) mx = fmaxf(mx, fmaxf(sc[1][nt][k], sc[1][nt][2 + k]));
#pragma unroll
            for (int q = 4; q < 32; q <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, q));
            const float mn = fmaxf(m[nt][k], mx * p.scale_log2);
            f[k] = m[nt][k] == mn ? 1.f : ex2(m[nt][k] - mn);
            m[nt][k] = mn;
            nm[nt][k] = mn == -INFINITY ? 0.f : kHalfUp - mn;  // nothing seen yet: every weight is zero
            const float bar = (mn + kRescaleLog2) * p.inv_scale;
            bar_[nt][k] = fmaf(-0x1p-21f, fabsf(bar), bar);  // rounded down: no weight passes 2^8, whatever the scores' size
            l[nt][k] *= f[k];
          }
#pragma unroll
          for (int i = 0; i < 2 * W; ++i) {
            o[nt][i][0] *= f[0];
            o[nt][i][1] *= f[1];
            o[nt][i][2] *= f[0];
            o[nt][i][3] *= f[1];
          }
          const float fe = __shfl_sync(0xffffffffu, f[0], g >> 1), fo = __shfl_sync(0xffffffffu, f[1], g >> 1);
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            ps[nt][i][0] *= f[0];
            ps[nt][i][1] *= f[1];
            corr[nt][i] *= (g & 1) ? fo : fe;
          }
        }
    };
    // The weights p s of one block's scores as the second operand of the value product: column g,
    // tokens 2c, 2c + 1 (+ 8 h). blk, tok0, there: the block of this lane's column g.
    auto weights = [&](const uint8_t* blk, int tok0, bool there, const float (&sc)[NT][4], uint32_t (&pb)[NT][NG][2],
                       auto edge_) {
      constexpr bool edge = decltype(edge_)::value;
      uint32_t vp[2][2 * NG];
#pragma unroll
      for (int h = 0; h < 2; ++h) lds<2 * NG>(blk + v_pair_off(D) + (h * 8 + 2 * c) * NG * 4, vp[h]);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float pe = ex2(fmaf(sc[nt][2 * h], p.scale_log2, nm[nt][0]));
          const float po = ex2(fmaf(sc[nt][2 * h + 1], p.scale_log2, nm[nt][1]));
          l[nt][0] += pe;
          l[nt][1] += po;
          const __half2 hp = __floats2half2_rn(pe, po);
          const uint32_t tr = transpose8x8(*reinterpret_cast<const uint32_t*>(&hp));
          // column g, tokens 2c, 2c + 1 (+ 8 h)
          const float2 w = mul2(__half22float2(*reinterpret_cast<const __half2*>(&tr)), make_float2(kHalfDown, kHalfDown));
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            uint32_t w0 = vp[h][i], w1 = vp[h][NG + i];
            if (edge) {  // a hidden token's pair may be anything, a NaN too: its weight of 0 does not meet it
              if (!there || tok0 + 8 * h + 2 * c >= seen_g[nt]) w0 = 0u;
              if (!there || tok0 + 8 * h + 2 * c + 1 >= seen_g[nt]) w1 = 0u;
            }
            pb[nt][i][h] = pack_bf16x2(w.x * scale_of(w0), w.y * scale_of(w1));
            corr[nt][i] = fmaf(w.x, min_of(w0), fmaf(w.y, min_of(w1), corr[nt][i]));
          }
        }
#pragma unroll
        for (int i = 0; i < NG; ++i)
          mma16816(ps[nt][i], 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, pb[nt][i][0], pb[nt][i][1]);
      }
    };
    // Adds one block's values with these weights.
    auto values = [&](const uint8_t* blk, const uint32_t (&pb)[NT][NG][2]) {
      uint32_t vw[2][W];
#pragma unroll
      for (int h = 0; h < 2; ++h) lds<W>(blk + v_code_off(D) + (h * 32 + lane) * W * 4, vw[h]);
#pragma unroll
      for (int u = 0; u < W; ++u)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t a0 = codes2(vw[0][u] >> (8 * e)), a1 = codes2(vw[0][u] >> (8 * e + 4));
          const uint32_t a2 = codes2(vw[1][u] >> (8 * e)), a3 = codes2(vw[1][u] >> (8 * e + 4));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][2 * u + e], a0, a1, a2, a3, pb[nt][u / 2][0], pb[nt][u / 2][1]);
        }
    };
    // Two blocks: their scores first, one vote on the references, then their values.
    auto two = [&](const uint8_t* blk, int tok0, uint32_t there, auto edge) {
      float sc[2][NT][4];
      bool grow = false;
      if constexpr (kDual) {
        float acc[2][NT][NG][4];
        product(blk, acc);
        const int mine = c >> 1, mine_g = g >> 2;  // the block of columns 2c, 2c + 1, and of column g
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (mine) acc[0][0][i][k] = acc[1][0][i][k];
        scores(blk + mine * C::kBlock, tok0 + mine * kBlockTok, there >> mine & 1u, acc[0], sc[0], edge);
#pragma unroll
        for (int k = 0; k < 4; ++k) grow |= sc[0][0][k] > bar_[0][k & 1];
        if (__any_sync(0xffffffffu, grow)) rescale(sc, 1);
        uint32_t pb[NT][NG][2];
        weights(blk + mine_g * C::kBlock, tok0 + mine_g * kBlockTok, there >> mine_g & 1u, sc[0], pb, edge);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t only[NT][NG][2];  // this block's columns
#pragma unroll
          for (int i = 0; i < NG; ++i) {
            only[0][i][0] = mine_g == j ? pb[0][i][0] : 0u;
            only[0][i][1] = mine_g == j ? pb[0][i][1] : 0u;
          }
          values(blk + j * C::kBlock, only);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (there >> i & 1u) {
            float acc[1][NT][NG][4];
            product(blk + i * C::kBlock, acc);
            scores(blk + i * C::kBlock, tok0 + i * kBlockTok, true, acc[0], sc[i], edge);
          } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sc[i][nt][0] = sc[i][nt][1] = sc[i][nt][2] = sc[i][nt][3] = -INFINITY;
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) grow |= sc[i][nt][k] > bar_[nt][k & 1];
        }
        if (__any_sync(0xffffffffu, grow)) rescale(sc, 2);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (there >> i & 1u) {
            uint32_t pb[NT][NG][2];
            weights(blk + i * C::kBlock, tok0 + i * kBlockTok, true, sc[i], pb, edge);
            values(blk + i * C::kBlock, pb);
          }
      }
    };
#pragma unroll 1
    for (int b = x.b0 + 2 * warp; b < x.b1; b += 2 * NW) {
      const int st = used % ST;
      const uint8_t* const blk = ring + st * 2 * C::kBlock;
      const uint32_t there = ring_ok >> 2 * st & 3u;
      if (!ptx::mbar_wait(&bars[warp][st], (used / ST) & 1, &g_kv4_error_word, kErrBlock, limit)) limit = 1000000;
      ++used;
      issue();  // into the stage that the previous pair left
      // some column ends here, or a block is missing
      if (b >= edge_from || there != 3u) two(blk, b * kBlockTok, there, std::true_type{});
      else two(blk, b * kBlockTok, there, std::false_type{});
      __syncwarp();  // every lane has read the stage before it is filled again
    }
    // ---- the warps' results joined ----
    const bool full = x.b0 == 0 && x.b1 == x.blocks;
    const int rec = 2 * blockIdx.x + (p.whole || static_cast<int64_t>(blockIdx.x) * sh.per_cta ==
                                                     cw.u - (x.b1 - x.b0) ? 0 : 1);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (col0 + nt * 8 >= ncols) break;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float s = l[nt][k];
#pragma unroll
        for (int q = 4; q < 32; q <<= 1) s += __shfl_xor_sync(0xffffffffu, s, q);
        if (g == 0) {
          ml_sm[warp][2 * c + k][0] = m[nt][k];
          ml_sm[warp][2 * c + k][1] = s * kHalfDown;
        }
        float* dst = merge + (warp * 8 + 2 * c + k) * C::kLd + 4 * g;
#pragma unroll
        for (int u = 0; u < W; ++u) {
          const float z = 128.f * ps[nt][u / 2][k];
          *reinterpret_cast<float4*>(dst + 32 * u) = make_float4(o[nt][2 * u][k] - z, o[nt][2 * u][2 + k] - z,
                                                                 o[nt][2 * u + 1][k] - z, o[nt][2 * u + 1][2 + k] - z);
        }
      }
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        float s = corr[nt][i];
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        if (c == 0) corr_sm[warp][g][i] = s;
      }
      __syncthreads();
      constexpr int kMerged = kDual ? 4 : 8;  // columns of the pass, and sets of results for each
      constexpr int kSets = kDual ? 2 * NW : NW;
      for (int at = threadIdx.x; at < kMerged * (D / 4); at += NW * 32) {
        const int mc = at / (D / 4), d4 = at % (D / 4) * 4;  // column, dimensions
        const int col = col0 + nt * 8 + mc;
        if (col >= ncols) continue;
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < kSets; ++e) top = fmaxf(top, ml_sm[e % NW][mc + e / NW * 4][0]);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < kSets; ++e) {
          const int w = e % NW, mw_c = mc + e / NW * 4;
          const float mw = ml_sm[w][mw_c][0], lw_ = ml_sm[w][mw_c][1];
          // no reference: nothing seen (no sum), or nothing but NaN, which stays
          const float f = mw == -INFINITY ? (lw_ == 0.f ? 0.f : 1.f) : ex2(mw - top);
          if (f == 0.f) continue;
          const float4 v = *reinterpret_cast<const float4*>(merge + (w * 8 + mw_c) * C::kLd + d4);
          const float z = corr_sm[w][mw_c][d4 / kGroup];
          sum += f * lw_;
          a.x += f * (v.x + z);
          a.y += f * (v.y + z);
          a.z += f * (v.z + z);
          a.w += f * (v.w + z);
        }
        if (full) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          uint2 w2;
          w2.x = pack_bf16x2(a.x * inv, a.y * inv);
          w2.y = pack_bf16x2(a.z * inv, a.w * inv);
          __nv_bfloat16* const out = tab.out0 ? tab.out0 + row0 * p.out_stride : tab.out[x.slot];
          *reinterpret_cast<uint2*>(out + static_cast<int64_t>(col / p.group) * p.out_stride +
                                    (x.head * p.group + col % p.group) * D + d4) = w2;
        } else {
          const int64_t r = static_cast<int64_t>(rec) * C::kCols + nt * 8 + mc;
          *reinterpret_cast<float4*>(p.part + r * D + d4) = a;
          if (d4 == 0) {
            float* ml = p.part + static_cast<int64_t>(2 * gridDim.x) * C::kCols * D + r * 2;
            ml[0] = top;
            ml[1] = sum;
          }
        }
      }
      __syncthreads();
    }
    have = cw.next(sh, tab, p, &x);
    if (have && kAhead) load_q(x);
  }
}

// Joins the partial records of one (slot, kv head, pass).
template <int D, int NT>
__global__ void __launch_bounds__(kWarps * 32)
    kv4_join_kernel(const __grid_constant__ AttnTable4 tab, const __grid_constant__ AttnParams4 p, int ctas) {
  using C = Cfg4<D, NT, kWarps>;
  __shared__ Shares sh;
  // the context lengths were complete before the attention launch, which started this one only then
  share_out<D, NT>(tab, p, &sh, ctas);
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int pair = blockIdx.x, n = tab.seg.nseg;
  if (pair >= sh.pair[n]) return;
  const int s = find_pair(sh, n, pair), i = pair - sh.pair[s];
  const int64_t u0 = sh.unit[s] + static_cast<int64_t>(i) * sh.blocks[s], u1 = u0 + sh.blocks[s];
  const int c0 = static_cast<int>(u0 / sh.per_cta), c1 = static_cast<int>((u1 - 1) / sh.per_cta);
  if (c0 == c1) return;  // written whole
  const int head = i / sh.passes[s], pass = i % sh.passes[s];
  const int row0 = row_of(tab.c, tab.seg, s), ncols = (row_of(tab.c, tab.seg, s + 1) - row0) * p.group;
  __nv_bfloat16* const out = tab.out0 ? tab.out0 + row0 * p.out_stride : tab.out[s];
  const float* mls = p.part + static_cast<int64_t>(2 * ctas) * C::kCols * D;
  for (int k = threadIdx.x; k < C::kCols * (D / 4); k += blockDim.x) {
    const int mc = k / (D / 4), d4 = k % (D / 4) * 4, col = pass * C::kCols + mc;
    if (col >= ncols) continue;
    auto record = [&](int cta) {
      return (2 * static_cast<int64_t>(cta) + (cta == c0 && u0 != c0 * sh.per_cta ? 1 : 0)) * C::kCols + mc;
    };
    // a pair may lie in a dozen records: their loads are in flight together
    float top = -INFINITY;
#pragma unroll 4
    for (int cta = c0; cta <= c1; ++cta) top = fmaxf(top, mls[record(cta) * 2]);
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int cta = c0; cta <= c1; ++cta) {
      const int64_t r = record(cta);
      const float2 mlw = *reinterpret_cast<const float2*>(mls + 2 * r);
      const float4 v = *reinterpret_cast<const float4*>(p.part + r * D + d4);
      const float f = mlw.x == -INFINITY ? (mlw.y == 0.f ? 0.f : 1.f) : ex2(mlw.x - top);
      const bool none = f == 0.f;  // what it holds has no say, an infinity neither
      sum += none ? 0.f : f * mlw.y;
      a.x += none ? 0.f : f * v.x;
      a.y += none ? 0.f : f * v.y;
      a.z += none ? 0.f : f * v.z;
      a.w += none ? 0.f : f * v.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint2 w2;
    w2.x = pack_bf16x2(a.x * inv, a.y * inv);
    w2.y = pack_bf16x2(a.z * inv, a.w * inv);
    *reinterpret_cast<uint2*>(out + static_cast<int64_t>(col / p.group) * p.out_stride +
                              (head * p.group + col % p.group) * D + d4) = w2;
  }
}

struct Plan4 {
  int nt, ctas, whole, warps;
  bool dual;
  int64_t pairs;
};

int sm_count4() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
}

Plan4 make_plan4(int nseg, const int* rows, int hq, int hkv, int max_len) {
  Plan4 pl;
  const int group = hq / hkv;
  int most = 0;
  for (int i = 0; i < nseg; ++i) most = std::max(most, rows[i]);
  pl.nt = static_cast<int64_t>(most) * group > 8 ? 2 : 1;
  pl.dual = static_cast<int64_t>(most) * group <= 4;
  pl.pairs = 0;
  for (int i = 0; i < nseg; ++i) pl.pairs += (static_cast<int64_t>(rows[i]) * group + 8 * pl.nt - 1) / (8 * pl.nt) * hkv;
  const int64_t blocks = (static_cast<int64_t>(max_len) + kBlockTok - 1) / kBlockTok;
  const int64_t sms = sm_count4();
  const int64_t slots = sms * (pl.nt == 1 ? 3 : 2);  // CTAs at a time
  // Whole pairs need no join (4 us and more), equal ranges keep every SM busy. Measured, whole
  // against cut, one row a slot, 32 query and 8 kv heads of 128 (six warps): 4 slots of up to 1000
  // tokens 11.0 and 15.2 us, 3000 22.5 and 18.7; 28 slots 1000 14.3 and 21.2, 3000 30.7 and 30.0, 8000 69
  // and 52. Two column tiles (28 slots of 4 rows): 4000 55 and 61, 8000 102 and 85. More pairs
  // than CTAs at a time (28 slots of 5 rows): 1000 37 and 50, 2000 58 and 60, 4000 104 and 85.
  pl.whole = blocks <= (pl.pairs > slots ? 136 : pl.nt == 1 ? 176 : 320) ? 1 : 0;
  pl.ctas = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>(slots, pl.whole ? pl.pairs : (pl.pairs * blocks + 2 * kWarps - 1) / (2 * kWarps))));
  // Whole pairs that fill two CTAs an SM at most have registers for six warps each: 28 slots of
  // 256 to 768 tokens 14.5 -> 12.8 us, of up to 1000 16.4 -> 14.4.
  pl.warps = pl.whole && pl.nt == 1 && blocks > 2 * kWarps && pl.pairs <= 2 * sms ? kManyWarps : kWarps;
  return pl;
}

template <int D, int NT, bool kDual, int NW>
int launch_kv4(const AttnTable4& t, const AttnParams4& p, const Plan4& pl, cudaStream_t st) {
  int dev = 0;
  SWL_CUDA_TRY(cudaGetDevice(&dev));
  static std::atomic<uint64_t> done{0};  // devices whose kernel has its shared memory limit raised
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    SWL_CUDA_TRY(cudaFuncSetAttribute(kv4_attention_kernel<D, NT, kDual, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      Cfg4<D, NT, NW>::kSmem));
    done.fetch_or(bit);
  }
  SWL_CUDA_TRY(launch_kernel(kv4_attention_kernel<D, NT, kDual, NW>, dim3(pl.ctas), dim3(NW * 32), Cfg4<D, NT, NW>::kSmem, st, 1,
                             t, p));
  if (!pl.whole)
    SWL_CUDA_TRY(launch_kernel(kv4_join_kernel<D, NT>, dim3(static_cast<unsigned>(pl.pairs)), dim3(kWarps * 32), 0, st, 1, t, p,
                               pl.ctas));
  return SWL_OK;
}

template <int D>
int launch_kv4_of(const AttnTable4& t, const AttnParams4& p, const Plan4& pl, cudaStream_t st) {
  if (pl.nt == 2) return launch_kv4<D, 2, false, kWarps>(t, p, pl, st);
  if (pl.warps == kManyWarps)
    return pl.dual ? launch_kv4<D, 1, true, kManyWarps>(t, p, pl, st) : launch_kv4<D, 1, false, kManyWarps>(t, p, pl, st);
  return pl.dual ? launch_kv4<D, 1, true, kWarps>(t, p, pl, st) : launch_kv4<D, 1, false, kWarps>(t, p, pl, st);
}

}  // namespace

int read_and_clear_error(unsigned int* code) {
  const unsigned int zero = 0;
  SWL_CUDA_TRY(cudaMemcpyFromSymbol(code, g_kv4_error_word, sizeof(zero)));
  if (*code) SWL_CUDA_TRY(cudaMemcpyToSymbol(g_kv4_error_word, &zero, sizeof(zero)));
  return SWL_OK;
}

}  // namespace kv4
}  // namespace swl

using namespace swl;

SWL_EXPORT int64_t swl_kv4_part_floats(int nseg, const int* rows, int hq, int hkv, int head_dim, int max_len) {
  RowSegments seg;
  if (kv4::fill_rows(&seg, "attention_kv4", nseg, rows) != SWL_OK || hkv < 1 || hq < 1 || hq % hkv || max_len < 1) return 0;
  if (head_dim != 64 && head_dim != 128) return 0;
  const kv4::Plan4 pl = kv4::make_plan4(nseg, rows, hq, hkv, max_len);
  return pl.whole ? 0 : static_cast<int64_t>(2 * pl.ctas) * 8 * pl.nt * (head_dim + 2);
}

namespace {

// swl_paged_attention_kv4: out0 for packed rows, else a pointer per slot.
int attention(int nseg, const int* rows, const kv4::Slots& slots, int table_len, int64_t num_pages, void* out0,
              void* const* out, int64_t out_stride, int hq, int hkv, int head_dim, int page, float scale, int max_len,
              const void* q_rot, float* part, void* stream) {
  kv4::AttnTable4 t;
  SWL_TRY(kv4::fill_rows(&t.seg, "attention_kv4", nseg, rows));
  SWL_TRY(kv4::fill_cache(&t.c, "attention_kv4", nseg, rows, slots, true, true, table_len, num_pages, hkv, head_dim, page));
  if (hq < 1 || hq > 4096 || hq % hkv) return set_error(SWL_ERR_ARG, "attention_kv4: query heads must be a multiple of kv heads");
  if (!(scale > 0.f) || !std::isfinite(scale)) return set_error(SWL_ERR_ARG, "attention_kv4: scale must be positive and finite");
  if (max_len < 1) return set_error(SWL_ERR_ARG, "attention_kv4: max_len must be positive");
  if (out_stride < static_cast<int64_t>(hq) * head_dim || out_stride % 8)
    return set_error(SWL_ERR_ARG, "attention_kv4: output stride must hold all heads and be a multiple of 8");
  if (t.seg.total_rows == 0) return SWL_OK;
  if (!q_rot || (reinterpret_cast<uintptr_t>(q_rot) & 15)) return set_error(SWL_ERR_ARG, "attention_kv4: q must be 16-byte aligned");
  if (!out && !out0) return set_error(SWL_ERR_ARG, "attention_kv4: null outputs");
  t.out0 = static_cast<__nv_bfloat16*>(out0);
  bool good = (reinterpret_cast<uintptr_t>(out0) & 15) == 0;
  for (int i = 0; i < nseg && !out0; ++i) {
    t.out[i] = static_cast<__nv_bfloat16*>(out[i]);
    good = good && (rows[i] == 0 || (t.out[i] && (reinterpret_cast<uintptr_t>(t.out[i]) & 15) == 0));
  }
  if (!good) return set_error(SWL_ERR_ARG, "attention_kv4: outputs must be 16-byte aligned");
  if (static_cast<int64_t>(t.seg.total_rows) * hq > (1 << 30)) return set_error(SWL_ERR_ARG, "attention_kv4: too many rows");
  const kv4::Plan4 pl = kv4::make_plan4(nseg, rows, hq, hkv, max_len);
  if (!pl.whole && (!part || (reinterpret_cast<uintptr_t>(part) & 15)))
    return set_error(SWL_ERR_ARG, "attention_kv4: missing or unaligned scratch");
  kv4::AttnParams4 p;
  p.hq = hq;
  p.group = hq / hkv;
  p.out_stride = out_stride;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.inv_scale = 1.f / p.scale_log2;
  p.max_len = max_len;
  p.q = static_cast<const __nv_bfloat16*>(q_rot);
  p.whole = pl.whole;
  p.pairs = static_cast<int>(pl.pairs);
  p.part = part;
  t.passes_each = (t.c.rows_each * p.group + 8 * pl.nt - 1) / (8 * pl.nt);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return head_dim == 128 ? kv4::launch_kv4_of<128>(t, p, pl, st) : kv4::launch_kv4_of<64>(t, p, pl, st);
}

}  // namespace

SWL_EXPORT int swl_paged_attention_kv4(int nseg, const int* rows, const void* const* block_tables, int table_len,
                                       const void* const* caches, int64_t num_pages, const void* const* seqlens,
                                       void* const* out, int64_t out_stride, int hq, int hkv, int head_dim, int page,
                                       float scale, int max_len, const void* q_rot, float* part, void* stream) {
  kv4::Slots s;
  s.block_tables = block_tables;
  s.caches = const_cast<void* const*>(caches);
  s.seqlens = seqlens;
  return attention(nseg, rows, s, table_len, num_pages, nullptr, out, out_stride, hq, hkv, head_dim, page, scale, max_len,
                   q_rot, part, stream);
}

SWL_EXPORT int swl_paged_attention_kv4_each(int nseg, const int* rows, const void* const* block_tables, const int* table_lens,
                                            const void* const* caches, const int64_t* num_pages, const void* const* seqlens,
                                            void* const* out, int64_t out_stride, int hq, int hkv, int head_dim, int page,
                                            float scale, int max_len, const void* q_rot, float* part, void* stream) {
  if (nseg > 0 && (!table_lens || !num_pages)) return set_error(SWL_ERR_ARG, "attention_kv4: null table lengths or page counts");
  kv4::Slots s;
  s.block_tables = block_tables;
  s.caches = const_cast<void* const*>(caches);
  s.seqlens = seqlens;
  s.table_lens = table_lens;
  s.num_pages = num_pages;
  return attention(nseg, rows, s, 1, 1, nullptr, out, out_stride, hq, hkv, head_dim, page, scale, max_len, q_rot, part, stream);
}

SWL_EXPORT int swl_paged_attention_kv4_packed(int nseg, const int* rows, const int* block_tables, int64_t table_stride,
                                              int table_len, const void* cache, int64_t num_pages, const int* seqlens,
                                              void* out, int64_t out_stride, int hq, int hkv, int head_dim, int page,
                                              float scale, int max_len, const void* q_rot, float* part, void* stream) {
  kv4::Slots s;
  s.packed = true;
  s.table0 = block_tables;
  s.table_step = table_stride;
  s.cache0 = const_cast<void*>(cache);
  s.len0 = seqlens;
  return attention(nseg, rows, s, table_len, num_pages, out, nullptr, out_stride, hq, hkv, head_dim, page, scale, max_len,
                   q_rot, part, stream);
}
