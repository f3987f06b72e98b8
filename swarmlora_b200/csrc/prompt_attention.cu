// Causal GQA attention over packed sequences of different lengths.
//
//   O_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^(c q_i.k_j - m_i),  c = scale * log2(e),
// over the keys j <= i + k_len - q_len, with a running reference m_i that any
// value near the running maximum serves for.
//
// A CTA takes one kv head and two tiles of query rows. The G query heads that share
// the kv head are packed with the tokens into the 128 rows of a tile (row =
// token * G + head), so K and V are read once for all of them and a short chunk still fills
// the tile. Per 128 keys, S = Q K^T goes to tensor memory, four warps (one row
// a thread) turn it into P in place, and O += P V is accumulated in tensor memory with P as the
// matrix operand from there: scores never leave the SM's tensor memory and
// registers. The two tiles alternate, so the tensor cores work on one while
// the warps of the other compute exponentials.
//
//   warps 0-3, 4-7   softmax of tile 0 and tile 1, and their epilogue
//   warp 8           TMA: Q once, K and V tiles through a ring; also looks over the V tiles
//                    of the masked range (below)
//   warp 9           issues every MMA (one lane); owns the tensor memory
//
// O is rescaled only when a row's maximum passes its reference by more than
// 2^8 (then by the softmax warps themselves, which have just seen the MMA
// that wrote O complete): weights up to 256 keep their relative precision in bf16 and
// their sum in fp32. P is rounded to bf16 for the product; the sum of the weights is taken
// before that, in fp32.
//
// Masked keys: a score is dropped by its index, whatever it holds. A weight of
// zero would still turn a NaN or infinity of V into NaN, so the V tiles in which some
// row's range ends are scanned before their product: non-finite values are set to
// zero there and, if any belongs to the sequence, added back in the epilogue to
// the rows that do see them.
#include <cuda_bf16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>

#include "common.h"
#include "kv4.cuh"
#include "launch.h"
#include "ptx.cuh"
#include "slot_round.h"

namespace swl {

namespace {

__device__ unsigned int g_prompt_error_word = 0;
constexpr uint64_t kWaitNs = 2000000000ull;
enum : unsigned { kErrSoftmax = 101, kErrMma = 102, kErrTma = 103 };

constexpr int kTile = 128;           // query rows of a tile, keys of a step
constexpr float kRescaleLog2 = 8.f;  // a row's weights may pass its reference by 2^8

struct PromptTable {
  int nseq;
  int q_start[kMaxSlots], q_len[kMaxSlots], k_start[kMaxSlots], k_len[kMaxSlots];
  int item_start[kMaxSlots + 1];  // query blocks (two tiles) of each sequence, longest sequence first
};
struct PromptParams {
  __nv_bfloat16* out;
  const __nv_bfloat16* v;
  int64_t out_stride, v_stride;
  int hq, hkv, group, tokens;  // query heads per kv head, tokens per tile
  float scale_log2;
  int splits;                  // CTAs that share a block's keys
  float* part;                 // splits > 1: O [row][head][split][D], then (m, l) pairs
  int64_t part_rows;           // rows * heads * splits
};

template <int D>
struct Cfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kSlots = D == 128 ? 4 : 6;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kSmem = (2 + kSlots) * kTileBytes + 1024;
  static constexpr uint32_t kS = 0, kO = 2 * kTile, kCols = 512;  // tensor memory columns
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// What the CTA of blockIdx.x works on.
struct Item {
  int seq, head, split;
  int t0[2], nt[2];   // first token and token count of each tile (0: no rows)
  int first[2];       // keys the first row of a tile sees (may be negative)
  int kb, ke[2];      // key tiles [kb, ke) of each tile
  int clean;          // key tiles from here on hold keys that some row does not see
};

__device__ __forceinline__ Item find_item(const PromptTable& t, const PromptParams& p) {
  Item it;
  int i = blockIdx.x;
  it.split = i % p.splits;
  i /= p.splits;
  it.head = i % p.hkv;
  i /= p.hkv;
  int lo = 0, hi = t.nseq - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.item_start[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  it.seq = lo;
  // the last block of a sequence has the most keys: it goes first
  const int block = t.item_start[lo + 1] - 1 - i;
  const int ql = t.q_len[lo], kl = t.k_len[lo];
  int n[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    it.t0[x] = (2 * block + x) * p.tokens;
    it.nt[x] = max(0, min(p.tokens, ql - it.t0[x]));
    it.first[x] = it.t0[x] + kl - ql + 1;
    const int last = min(kl, it.first[x] + it.nt[x] - 1);
    n[x] = it.nt[x] > 0 ? (max(0, last) + kTile - 1) / kTile : 0;
  }
  const int all = max(n[0], n[1]);
  it.kb = static_cast<int>(static_cast<int64_t>(all) * it.split / p.splits);
  const int ke = static_cast<int>(static_cast<int64_t>(all) * (it.split + 1) / p.splits);
#pragma unroll
  for (int x = 0; x < 2; ++x) it.ke[x] = max(it.kb, min(n[x], ke));
  it.clean = max(0, it.first[0]) / kTile;
  return it;
}

template <int D>
__global__ void __launch_bounds__(320, 1)
    prompt_attention_kernel(const __grid_constant__ PromptTable tab, const __grid_constant__ PromptParams p,
                            const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                            const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<D>;
  extern __shared__ uint8_t dyn_raw[];
  uint8_t* const dyn = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const q_sm = dyn;
  uint8_t* const ring = dyn + 2 * C::kTileBytes;
  __shared__ __align__(8) uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  __shared__ __align__(8) uint64_t full[C::kSlots], empty[C::kSlots], seen[4], drained;
  __shared__ uint32_t tmem_base;
  __shared__ int bad;  // a non-finite value of this sequence was taken out of a V tile
  unsigned int* const err = &g_prompt_error_word;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&q_full[i], 1);
      ptx::mbar_init(&s_full[i], 1);
      ptx::mbar_init(&p_full[i], 128);
      ptx::mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < C::kSlots; ++i) {
      ptx::mbar_init(&full[i], 1);
      ptx::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 4; ++i) ptx::mbar_init(&seen[i], 1);
    ptx::mbar_init(&drained, 1);
    bad = 0;
    ptx::fence_mbar_init();
  }
  if (warp == 9) ptx::tmem_alloc(&tmem_base, C::kCols);
  if (warp == 8 && lane == 0) {
    ptx::prefetch_tmap(&qmap);
    ptx::prefetch_tmap(&kmap);
    ptx::prefetch_tmap(&vmap);
  }
  const Item it = find_item(tab, p);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tmem_base;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();

  const int nk = max(it.ke[0], it.ke[1]) - it.kb;  // key tiles of this CTA
  if (warp == 8) {
    const int k_row0 = tab.k_start[it.seq];
    if (lane == 0 && nk > 0) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (it.ke[x] <= it.kb) continue;
        ptx::mbar_arrive_expect_tx(&q_full[x], p.tokens * p.group * D * 2);
        for (int h = 0; h < C::kHalves; ++h)
          ptx::tma_load_3d(ptx::smem_addr(q_sm + x * C::kTileBytes + h * kTile * 128), &qmap, &q_full[x], h * 64,
                           it.head * p.group, tab.q_start[it.seq] + it.t0[x]);
      }
    }
    const int klen = tab.k_len[it.seq];
    // Takes non-finite values out of V tile j (of this CTA) and announces it.
    auto look_over = [&](int j) {
      const int n = 2 * j + 1, s = n % C::kSlots;
      if (!ptx::mbar_wait(&full[s], (n / C::kSlots) & 1, err, kErrTma, kWaitNs)) return false;
      uint4* const v = reinterpret_cast<uint4*>(ring + s * C::kTileBytes);
      const __nv_bfloat162 zero = __float2bfloat162_rn(0.f);
      for (int i = lane; i < C::kTileBytes / 16; i += 32) {
        uint4 u = v[i];
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
        __nv_bfloat162 a = zero;
#pragma unroll
        for (int e = 0; e < 4; ++e) a = __hfma2(h[e], zero, a);  // 0 unless a factor is NaN or infinite
        if (__low2float(a) != 0.f || __high2float(a) != 0.f || __hisnan(a.x) || __hisnan(a.y)) {
          __nv_bfloat16* b = reinterpret_cast<__nv_bfloat16*>(&u);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (!isfinite(__bfloat162float(b[e]))) b[e] = __float2bfloat16_rn(0.f);
          v[i] = u;
          if ((it.kb + j) * kTile + (i / 8) % kTile < klen) bad = 1;
        }
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&seen[(it.kb + j - max(it.kb, it.clean)) & 3]);
      return true;
    };
    bool ok = true;
    int issued = 0;
    for (int j = 0; j < nk && ok; ++j) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int n = 2 * j + kv, s = n % C::kSlots;
        if (lane == 0 && ok) {
          ok = n < C::kSlots || ptx::mbar_wait(&empty[s], ((n / C::kSlots) & 1) ^ 1, err, kErrTma, kWaitNs);
          if (ok) {
            ptx::mbar_arrive_expect_tx(&full[s], C::kTileBytes);
            for (int h = 0; h < C::kHalves; ++h)
              ptx::tma_load_3d(ptx::smem_addr(ring + s * C::kTileBytes + h * kTile * 128), kv ? &vmap : &kmap, &full[s],
                               h * 64, it.head, k_row0 + (it.kb + j) * kTile);
            ++issued;
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, static_cast<int>(ok), 0);
      if (ok && j > 0 && it.kb + j - 1 >= it.clean) ok = look_over(j - 1);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (ok && nk > 0 && it.kb + nk - 1 >= it.clean) ok = look_over(nk - 1);
    if (!ok && lane == 0) {
      // a wait gave up: the copies that were issued land before the CTA ends
      for (int n = max(0, issued - C::kSlots); n < issued; ++n)
        ptx::mbar_wait(&full[n % C::kSlots], (n / C::kSlots) & 1, err, kErrTma, kWaitNs);
      for (int x = 0; x < 2; ++x)
        if (it.ke[x] > it.kb) ptx::mbar_wait(&q_full[x], 0, err, kErrTma, kWaitNs);
    }
  } else if (warp == 9) {
    if (lane == 0) {
      constexpr uint32_t idesc_s = ptx::idesc_bf16_f32(kTile, kTile);
      constexpr uint32_t idesc_o = ptx::idesc_bf16_f32(kTile, D) | ptx::kIdescBMnMajor;
      const int n[2] = {it.ke[0] - it.kb, it.ke[1] - it.kb};
      bool ok = true;
      auto scores = [&](int x, int j) {  // S_x = Q_x K_j^T
        const uint32_t q = ptx::smem_addr(q_sm + x * C::kTileBytes);
        const uint32_t k = ptx::smem_addr(ring + (2 * j) % C::kSlots * C::kTileBytes);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t o = (kk >> 2) * kTile * 128 + (kk & 3) * 32;
          ptx::mma_bf16_ss(tmem + C::kS + x * kTile, ptx::sw128_kmajor_desc(q + o), ptx::sw128_kmajor_desc(k + o),
                           idesc_s, kk > 0 ? 1u : 0u);
        }
        ptx::tc_commit(&s_full[x]);
      };
      auto wait_full = [&](int i) {
        return ptx::mbar_wait(&full[i % C::kSlots], (i / C::kSlots) & 1, err, kErrMma, kWaitNs);
      };
      if (nk > 0) {
        ok = wait_full(0);
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (ok && n[x] > 0) {
            ok = ptx::mbar_wait(&q_full[x], 0, err, kErrMma, kWaitNs);
            if (ok) {
              ptx::tc_fence_after();
              scores(x, 0);
            }
          }
        ptx::tc_commit(&empty[0]);
      }
      for (int j = 0; j < nk && ok; ++j) {
        const int vs = (2 * j + 1) % C::kSlots;
        ok = wait_full(2 * j + 1);
        const int looked = it.kb + j - max(it.kb, it.clean);
        if (ok && looked >= 0) ok = ptx::mbar_wait(&seen[looked & 3], (looked >> 2) & 1, err, kErrMma, kWaitNs);
        if (ok && j + 1 < nk) ok = wait_full(2 * j + 2);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (!ok || j >= n[x]) continue;
          ok = ptx::mbar_wait(&p_full[x], j & 1, err, kErrMma, kWaitNs);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint32_t v = ptx::smem_addr(ring + vs * C::kTileBytes);
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk)
            ptx::mma_bf16_ts(tmem + C::kO + x * D, tmem + C::kS + x * kTile + kk * 8,
                             ptx::sw128_mnmajor_desc(v + kk * 16 * 128, kTile * 128), idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
          if (j + 1 == n[x]) ptx::tc_commit(&o_full[x]);
          if (j + 1 < n[x]) scores(x, j + 1);
        }
        if (ok) {
          ptx::tc_commit(&empty[vs]);
          if (j + 1 < nk) ptx::tc_commit(&empty[(2 * j + 2) % C::kSlots]);
        }
      }
      if (!ok) {  // a wait gave up: what was issued finishes before the tensor memory is freed
        ptx::tc_commit(&drained);
        ptx::mbar_wait(&drained, 0, err, kErrMma, kWaitNs);
      }
    }
    __syncwarp();
  } else {
    const int x = warp >> 2;                 // tile
    const int r = (warp & 3) * 32 + lane;    // row of the tile = lane of the tensor memory
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + C::kS + x * kTile, to = tmem + lanes + C::kO + x * D;
    const int n = it.ke[x] - it.kb, token = r / p.group;
    const bool real = token < it.nt[x];
    const int klen = tab.k_len[it.seq];
    const int sees = real ? max(0, min(klen, it.first[x] + token)) : 0;  // keys 0 .. sees - 1
    const int whole = max(0, it.first[x]) / kTile;  // tiles before this one need no mask
    float m = -INFINITY, l = 0.f;  // reference (scaled, base 2) and sum of weights
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      ok = ptx::mbar_wait(&s_full[x], j & 1, err, kErrSoftmax, kWaitNs);
      if (!ok) break;
      ptx::tc_fence_after();
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32b_x32(ts + c * 32, s[c]);
#pragma unroll
      for (int c = 0; c < 4; ++c) ptx::tmem_wait_regs(s[c]);
      if (it.kb + j >= whole) {
        const int lim = sees - (it.kb + j) * kTile;
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (c * 32 + i >= lim) s[c][i] = 0xff800000u;
      }
      float mx[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx[c] = __uint_as_float(s[c][0]);
#pragma unroll
        for (int i = 1; i < 32; ++i) mx[c] = fmaxf(mx[c], __uint_as_float(s[c][i]));
      }
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
      if (__any_sync(0xffffffffu, top > m + kRescaleLog2)) {
        const float mn = fmaxf(m, top);
        const float f = m == mn ? 1.f : ex2(m - mn);
        m = mn;
        l *= f;
        if (j > 0) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            ptx::tmem_ld_32x32b_x32(to + c * 32, o);
            ptx::tmem_wait_regs(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            ptx::tmem_st_32x32b_x32(to + c * 32, o);
          }
        }
      }
      const float mm = m == -INFINITY ? 0.f : m;  // nothing seen yet: every weight is zero
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int cc = 2 * c + i / 16, ii = i % 16 * 2;
          const float a = ex2(fmaf(__uint_as_float(s[cc][ii]), p.scale_log2, -mm));
          const float b = ex2(fmaf(__uint_as_float(s[cc][ii + 1]), p.scale_log2, -mm));
          sum[(i & 1) * 2] += a;
          sum[(i & 1) * 2 + 1] += b;
          w[i] = pack_bf16x2(a, b);
        }
        ptx::tmem_st_32x32b_x32(ts + c * 32, w);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      ptx::mbar_arrive(&p_full[x]);
    }
    // ---- epilogue: this thread's row
    if (n > 0 && ok) {
      ok = ptx::mbar_wait(&o_full[x], 0, err, kErrSoftmax, kWaitNs);
      ptx::tc_fence_after();
    }
    const int64_t grow = tab.q_start[it.seq] + it.t0[x] + token;
    const int head = it.head * p.group + r % p.group;
    const bool fix = ok && n > 0 && *reinterpret_cast<volatile int*>(&bad);
    const float inv = p.splits > 1 ? 1.f : (l == 0.f ? 0.f : 1.f / l);
    const int64_t rec = (grow * p.hq + head) * p.splits + it.split;
    if (real && p.splits > 1) {
      float* ml = p.part + p.part_rows * D + rec * 2;
      ml[0] = n > 0 ? m : -INFINITY;
      ml[1] = l;
    }
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t o[32];
      if (n > 0) {
        ptx::tmem_ld_32x32b_x32(to + c * 32, o);
        ptx::tmem_wait_regs(o);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = 0u;
      }
      if (!real || !ok) continue;
      if (fix) {
        // non-finite values of V that this row does see
        for (int key = max(it.kb, it.clean) * kTile; key < min(sees, it.ke[x] * kTile); ++key) {
          const __nv_bfloat16* vr = p.v + (tab.k_start[it.seq] + static_cast<int64_t>(key)) * p.v_stride + it.head * D + c * 32;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float f = __bfloat162float(vr[i]);
            if (!isfinite(f)) o[i] = __float_as_uint(__uint_as_float(o[i]) + f);
          }
        }
      }
      if (p.splits > 1) {
        float4* dst = reinterpret_cast<float4*>(p.part + rec * D + c * 32);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          dst[i] = make_float4(__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]),
                               __uint_as_float(o[4 * i + 3]));
      } else {
        uint4* dst = reinterpret_cast<uint4*>(p.out + grow * p.out_stride + head * D + c * 32);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = pack_bf16x2(__uint_as_float(o[8 * i + 2 * e]) * inv, __uint_as_float(o[8 * i + 2 * e + 1]) * inv);
          dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    ptx::tc_fence_before();
  }
  __syncthreads();
  if (warp == 9) {
    ptx::tmem_relinquish();
    ptx::tmem_dealloc(tmem, C::kCols);
  }
}

// Merges the splits of one (row, head).
template <int D>
__global__ void __launch_bounds__(D) prompt_combine_kernel(const __grid_constant__ PromptParams p) {
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int64_t row = blockIdx.x;
  const int head = blockIdx.y, d = threadIdx.x;
  const int64_t rec = (row * p.hq + head) * p.splits;
  const float* ml = p.part + p.part_rows * D + rec * 2;
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[2 * s]);
  float l = 0.f, o = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const float ms = ml[2 * s], f = ms == -INFINITY ? 0.f : ex2(ms - m);
    // a split whose weights were NaN keeps its NaN although its reference says nothing
    l += ms == -INFINITY && ml[2 * s + 1] == 0.f ? 0.f : (ms == -INFINITY ? ml[2 * s + 1] : f * ml[2 * s + 1]);
    if (ms != -INFINITY || ml[2 * s + 1] != 0.f) o += (ms == -INFINITY ? 1.f : f) * p.part[(rec + s) * D + d];
  }
  p.out[row * p.out_stride + head * D + d] = __float2bfloat16_rn(l == 0.f ? 0.f : o / l);
}

struct Plan {
  PromptTable t;
  int items, splits;
  int64_t total_q, total_k;
};

int make_plan(Plan* pl, int nseg, const int* q_lens, const int* k_lens, int hq, int hkv, int head_dim) {
  RowSegments q, k;
  SWL_TRY(kv4::fill_rows(&q, "prompt_attention", nseg, q_lens));
  SWL_TRY(kv4::fill_rows(&k, "prompt_attention", nseg, k_lens));
  if (head_dim != 64 && head_dim != 128) return set_error(SWL_ERR_ARG, "prompt_attention: head_dim must be 64 or 128");
  if (hkv < 1 || hq < 1 || hq % hkv || hq / hkv > 128 || hq > 4096)
    return set_error(SWL_ERR_ARG, "prompt_attention: query heads must be a multiple of kv heads, at most 128 each");
  pl->total_q = q.total_rows;
  pl->total_k = k.total_rows;
  const int tokens = kTile / (hq / hkv);
  int order[kMaxSlots], n = 0;
  for (int i = 0; i < nseg; ++i)
    if (q_lens[i] > 0) order[n++] = i;
  std::stable_sort(order, order + n, [&](int a, int b) { return k_lens[a] > k_lens[b]; });
  PromptTable& t = pl->t;
  t.nseq = n;
  int64_t items = 0;
  int most = 0;  // key tiles of the longest block
  for (int i = 0; i < n; ++i) {
    const int s = order[i];
    t.q_start[i] = q.row_start[s];
    t.q_len[i] = q_lens[s];
    t.k_start[i] = k.row_start[s];
    t.k_len[i] = k_lens[s];
    t.item_start[i] = static_cast<int>(items);
    items += (q_lens[s] + 2 * tokens - 1) / (2 * tokens);
    most = std::max(most, (k_lens[s] + kTile - 1) / kTile);
  }
  t.item_start[n] = static_cast<int>(items);
  if (items * hkv > (int64_t{1} << 30)) return set_error(SWL_ERR_ARG, "prompt_attention: too many query blocks");
  pl->items = static_cast<int>(items);
  pl->splits = 1;
  return SWL_OK;
}

template <int D>
int launch_prompt(const Plan& pl, const PromptParams& p, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm,
                  cudaStream_t st) {
  int dev = 0;
  SWL_CUDA_TRY(cudaGetDevice(&dev));
  static std::atomic<uint64_t> done{0};  // devices whose kernel has its shared memory limit raised
  const uint64_t bit = uint64_t{1} << (dev & 63);
  if (!(done.load(std::memory_order_relaxed) & bit)) {
    SWL_CUDA_TRY(cudaFuncSetAttribute(prompt_attention_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem));
    done.fetch_or(bit);
  }
  SWL_CUDA_TRY(launch_kernel(prompt_attention_kernel<D>, dim3(static_cast<unsigned>(pl.items) * p.hkv * p.splits), dim3(320),
                             Cfg<D>::kSmem, st, 1, pl.t, p, qm, km, vm));
  if (p.splits > 1)
    SWL_CUDA_TRY(launch_kernel(prompt_combine_kernel<D>, dim3(static_cast<unsigned>(pl.total_q), p.hq), dim3(D), 0, st, 1, p));
  return SWL_OK;
}

}  // namespace
}  // namespace swl

using namespace swl;

SWL_EXPORT int64_t swl_prompt_attention_part_floats(int nseg, const int* q_lens, const int* k_lens, int hq, int hkv,
                                                    int head_dim) {
  Plan pl;
  if (make_plan(&pl, nseg, q_lens, k_lens, hq, hkv, head_dim) != SWL_OK || pl.splits == 1) return 0;
  return pl.total_q * hq * pl.splits * (head_dim + 2);
}

SWL_EXPORT int swl_prompt_attention(int nseg, const int* q_lens, const int* k_lens, const void* q, int64_t q_stride,
                                    const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* out,
                                    int64_t out_stride, int hq, int hkv, int head_dim, float scale, float* part,
                                    void* stream) {
  Plan pl;
  SWL_TRY(make_plan(&pl, nseg, q_lens, k_lens, hq, hkv, head_dim));
  if (!(scale > 0.f) || !std::isfinite(scale)) return set_error(SWL_ERR_ARG, "prompt_attention: scale must be positive and finite");
  const int64_t qw = static_cast<int64_t>(hq) * head_dim, kw = static_cast<int64_t>(hkv) * head_dim;
  if (q_stride < qw || out_stride < qw || k_stride < kw || v_stride < kw)
    return set_error(SWL_ERR_ARG, "prompt_attention: row strides must hold all heads");
  if ((q_stride | out_stride | k_stride | v_stride) % 8 || (q_stride | out_stride | k_stride | v_stride) >> 36)
    return set_error(SWL_ERR_ARG, "prompt_attention: row strides must be multiples of 8 below 2^36");
  if (pl.total_q == 0) return SWL_OK;
  if (!q || !out || (pl.total_k > 0 && (!k || !v))) return set_error(SWL_ERR_ARG, "prompt_attention: null tensor");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out)) & 15)
    return set_error(SWL_ERR_ARG, "prompt_attention: tensors must be 16-byte aligned");
  if (pl.splits > 1 && (!part || (reinterpret_cast<uintptr_t>(part) & 15)))
    return set_error(SWL_ERR_ARG, "prompt_attention: missing or unaligned scratch");
  PromptParams p;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.out_stride = out_stride;
  p.v_stride = v_stride;
  p.hq = hq;
  p.hkv = hkv;
  p.group = hq / hkv;
  p.tokens = kTile / p.group;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.splits = pl.splits;
  p.part = part;
  p.part_rows = pl.total_q * hq * pl.splits;
  // without any key the maps of K and V are never used: they describe q's row instead
  const bool keys = pl.total_k > 0;
  CUtensorMap qm, km, vm;
  SWL_TRY(encode_heads_tmap(&qm, q, pl.total_q, hq, head_dim, q_stride, p.group, p.tokens));
  SWL_TRY(encode_heads_tmap(&km, keys ? k : q, keys ? pl.total_k : 1, keys ? hkv : 1, head_dim, keys ? k_stride : head_dim, 1, kTile));
  SWL_TRY(encode_heads_tmap(&vm, keys ? v : q, keys ? pl.total_k : 1, keys ? hkv : 1, head_dim, keys ? v_stride : head_dim, 1, kTile));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return head_dim == 128 ? launch_prompt<128>(pl, p, qm, km, vm, st) : launch_prompt<64>(pl, p, qm, km, vm, st);
}

SWL_EXPORT int swl_attention_device_error(unsigned int* code) {
  if (!code) return set_error(SWL_ERR_ARG, "null code pointer");
  const unsigned int zero = 0;
  SWL_CUDA_TRY(cudaMemcpyFromSymbol(code, g_prompt_error_word, sizeof(zero)));
  if (*code) SWL_CUDA_TRY(cudaMemcpyToSymbol(g_prompt_error_word, &zero, sizeof(zero)));
  unsigned int other = 0;
  SWL_TRY(kv4::read_and_clear_error(&other));
  if (!*code) *code = other;
  return SWL_OK;
}
