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
//   warps 0-3, 4-7   softmax of row tile 0 and 1, and their epilogue
//   warp 8           TMA: Q, and K and V tiles through a ring
//   warps 9, 10      issue the products of row tile 0 and 1 (one lane); 9 owns the tensor memory
//   warp 11          looks over the V tiles of the masked range (below)
//
// A CTA stays and takes one item after the other, the next of the list whenever it is
// free: the copies and score products of the next item run while the rows of the last
// one are written. Against a list dealt out beforehand by length, sixteen prompts of 17 to
// 2048 tokens went from 248 to 218 us in bursts (250 in a loop) and five of up to 2000 with heads of 64 from 38 to 32 (a row
// tile's 128 keys take 2.1 us, what is fixed in an item 3 to 4, so shares counted in keys are uneven).
//
// One prompt of 8191 tokens, 32 query and 8 kv heads of 128: 442 us in a burst at 1965 MHz
// (1.24 PFLOP/s), 498 to 518 in a loop, where the power cap holds the clock at 1620 (1.06 to
// 1.10; the comparisons below are of loops). At full clock what bounds it is the chain of one row
// tile (product, 128 exponentials a thread, product: 2.1 us, of which its products take 0.55),
// two of which are in flight: tensor memory has no room for a third. Without the two issuing
// warps' turns it is 607 us, with the turn handed over before the score product 574, half way
// through it 519, two steps before its end 500. Two threads a row for the exponentials: 597 us.
// One in 2 to 8 of them as a polynomial, in an earlier build: 589 to 637 for 531.
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

constexpr int kThreads = 384;        // three warpgroups; the last has its registers moved to the others
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
  int items;                   // blocks x kv heads x splits
  int splits;                  // items that share a block's keys
  float* part;                 // splits > 1: O [row][head][split][D], then (m, l) pairs
  int64_t part_rows;           // rows * heads * splits
};

template <int D>
struct Cfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kStages = D == 128 ? 2 : 4;  // tiles of K, and of V
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kOutBytes = 8 * 32 * 64;     // epilogue: 32 rows x 64 B for each softmax warp
  static constexpr int kSmem = (2 + 2 * kStages) * kTileBytes + kOutBytes + 1024;
  static constexpr uint32_t kS = 0, kO = 2 * kTile, kCols = 512;  // tensor memory columns
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(r)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// One unit of a CTA's work: a block of queries of one sequence and kv head, over a range of its keys.
struct ItemTile {
  int t0, nt;  // first token and token count (0: no rows)
  int first;   // keys the first row sees (may be negative)
  int n;       // key tiles
};
struct __align__(16) Item {
  ItemTile tile[2];
  int head, split;
  int kb, nk;           // first key tile, key tiles
  int clean;            // key tiles of the item from this one on hold keys that some row does not see
  int q_row, k_row;     // first rows of the sequence
  int k_len;
};

__device__ __forceinline__ Item find_item(const PromptTable& t, const PromptParams& p, int i) {
  Item it;
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
  // the last block of a sequence has the most keys: it goes first
  const int block = t.item_start[lo + 1] - 1 - i;
  const int ql = t.q_len[lo], kl = t.k_len[lo];
  it.q_row = t.q_start[lo];
  it.k_row = t.k_start[lo];
  it.k_len = kl;
  int n[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    ItemTile& tl = it.tile[x];
    tl.t0 = (2 * block + x) * p.tokens;
    tl.nt = max(0, min(p.tokens, ql - tl.t0));
    tl.first = tl.t0 + kl - ql + 1;
    const int last = min(kl, tl.first + tl.nt - 1);
    n[x] = tl.nt > 0 ? (max(0, last) + kTile - 1) / kTile : 0;
  }
  const int all = max(n[0], n[1]);
  it.kb = static_cast<int>(static_cast<int64_t>(all) * it.split / p.splits);
  const int ke = static_cast<int>(static_cast<int64_t>(all) * (it.split + 1) / p.splits);
#pragma unroll
  for (int x = 0; x < 2; ++x) it.tile[x].n = max(0, min(n[x], ke) - it.kb);
  it.nk = max(it.tile[0].n, it.tile[1].n);
  it.clean = max(0, max(0, it.tile[0].first) / kTile - it.kb);
  return it;
}

// The items of a CTA: its own block's, then those of blocks that it cancels before they
// start, so that whoever is done first takes the next item of the list. The copying lane asks
// and works the item out, a ring hands it to the other roles.
constexpr int kItems = 4, kReaders = 11;  // the scanning and 2 issuing warps, 8 softmax warps
struct Items {
  Item item[kItems];
  uint4 answer;
  uint64_t answered, full[kItems], empty[kItems];
};
struct ItemReader {
  uint32_t k = 0;  // items so far
  // The next item, or null (none left, or a wait gave up: then *ok is false). kWarp: called by
  // a whole warp together, else by one lane. It is there until release().
  template <bool kWarp>
  __device__ __forceinline__ const Item* next(Items& a, unsigned int* err, unsigned int code, bool* ok) {
    *ok = ptx::mbar_wait(&a.full[k % kItems], (k / kItems) & 1, err, code, kWaitNs);
    if (kWarp) *ok = __all_sync(0xffffffffu, *ok);
    const Item* const it = &a.item[k % kItems];
    return *ok && it->nk >= 0 ? it : nullptr;
  }
  template <bool kWarp>
  __device__ __forceinline__ void release(Items& a) {
    if (kWarp) __syncwarp();
    if (!kWarp || (threadIdx.x & 31) == 0) ptx::mbar_arrive(&a.empty[k % kItems]);
    ++k;
  }
};
struct ItemWriter {
  uint32_t k = 0, asked = 0, taken = 0;  // items written, requests, answers read
  __device__ __forceinline__ bool put(Items& a, const Item& it, unsigned int* err, unsigned int code) {
    if (k >= kItems && !ptx::mbar_wait(&a.empty[k % kItems], (k / kItems - 1) & 1, err, code, kWaitNs)) return false;
    a.item[k % kItems] = it;
    ptx::mbar_arrive(&a.full[k++ % kItems]);
    return true;
  }
  __device__ __forceinline__ void ask(Items& a) {
    ptx::mbar_arrive_expect_tx(&a.answered, 16);
    ptx::try_cancel_block(&a.answer, &a.answered);
    ++asked;
  }
  // The number of the item that was asked for, -1: none left.
  __device__ __forceinline__ bool answer(Items& a, int* i, unsigned int* err, unsigned int code) {
    if (!ptx::mbar_wait(&a.answered, taken & 1, err, code, kWaitNs)) return false;
    ++taken;
    *i = ptx::cancelled_block(&a.answer);
    ptx::fence_proxy_async_smem();  // read before the next answer is written
    return true;
  }
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_attention_kernel(const __grid_constant__ PromptTable table, const __grid_constant__ PromptParams p,
                            const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                            const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<D>;
  constexpr int ST = C::kStages;
  extern __shared__ uint8_t dyn_raw[];
  uint8_t* const dyn = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(dyn_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const q_sm = dyn;
  uint8_t* const k_ring = dyn + 2 * C::kTileBytes;
  uint8_t* const v_ring = k_ring + ST * C::kTileBytes;
  uint8_t* const out_sm = v_ring + ST * C::kTileBytes;
  // Who completes each barrier: *_full the copy or product that fills, *_empty who has used it.
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], s_full[2], p_half[2], p_full[2], o_full[2], o_empty[2];
  __shared__ __align__(8) uint64_t k_full[ST], k_empty[ST], v_full[ST], v_empty[ST], turn[2], drained[2];
  // as many as V tiles: with fewer, the scan could run two phases ahead of an issuing warp's wait
  __shared__ __align__(8) uint64_t seen[ST];
  __shared__ uint32_t tmem_base;
  // [n & 7] == n + 1: a non-finite value of its sequence was taken out of a V tile of the
  // CTA's n-th item with keys (copies run at most 4 items ahead of the rows, so n's are done when n + 8 comes)
  __shared__ int bad[8];
  // the launch's table: reading it from the parameter space costs a miss an entry, for every item anew
  __shared__ PromptTable tab;
  __shared__ Items items;
  unsigned int* const err = &g_prompt_error_word;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&q_full[i], 1);
      ptx::mbar_init(&q_empty[i], 1);
      ptx::mbar_init(&s_full[i], 1);
      ptx::mbar_init(&p_half[i], 4);
      ptx::mbar_init(&p_full[i], 4);
      ptx::mbar_init(&o_full[i], 1);
      ptx::mbar_init(&o_empty[i], 4);
      ptx::mbar_init(&turn[i], 1);
      ptx::mbar_init(&drained[i], 1);
    }
    for (int i = 0; i < ST; ++i) {
      ptx::mbar_init(&k_full[i], 1);
      ptx::mbar_init(&k_empty[i], 2);
      ptx::mbar_init(&v_full[i], 1);
      ptx::mbar_init(&v_empty[i], 3);
      ptx::mbar_init(&seen[i], 1);
    }
    for (int i = 0; i < 8; ++i) bad[i] = 0;
    ptx::mbar_init(&items.answered, 1);
    for (int i = 0; i < kItems; ++i) {
      ptx::mbar_init(&items.full[i], 1);
      ptx::mbar_init(&items.empty[i], kReaders);
    }
    ptx::fence_mbar_init();
  }
  for (int i = threadIdx.x; i < table.nseq; i += kThreads) {
    tab.q_start[i] = table.q_start[i];
    tab.q_len[i] = table.q_len[i];
    tab.k_start[i] = table.k_start[i];
    tab.k_len[i] = table.k_len[i];
    tab.item_start[i + 1] = table.item_start[i + 1];
  }
  if (threadIdx.x == 0) {
    tab.nseq = table.nseq;
    tab.item_start[0] = 0;
  }
  if (warp == 9) ptx::tmem_alloc(&tmem_base, C::kCols);
  if (warp == 8 && lane == 0) {
    ptx::prefetch_tmap(&qmap);
    ptx::prefetch_tmap(&kmap);
    ptx::prefetch_tmap(&vmap);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = tmem_base;
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();

  // registers at launch: 384 x 168 = 64512; 256 x 208 + 128 x 80 = 63488
  if (warp >= 8) {
    ptx::reg_dec<80>();
    ItemReader work;
    uint32_t tiles = 0;  // key tiles of the items so far: ring position
    bool ok = true;
    if (warp == 8) {
      // ---- copies
      if (lane == 0) {
        uint32_t qn[2] = {0, 0}, issued = 0;  // copies of each row tile, and of K and V tiles
        ItemWriter list;
        int i = blockIdx.x;
        do {
          const Item it = find_item(tab, p, i);
          ok = list.put(items, it, err, kErrTma);
          // the rows of Q come from memory: they are on their way while the last item's tiles are used
          if (ok && list.k > 1)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              if (it.tile[x].n > 0)
                for (int h = 0; h < C::kHalves; ++h)
                  ptx::tma_prefetch_3d(&qmap, h * 64, it.head * p.group, it.q_row + it.tile[x].t0);
          auto load_q = [&](int x) {
            if (!ok || it.tile[x].n == 0) return;
            ok = qn[x] == 0 || ptx::mbar_wait(&q_empty[x], (qn[x] - 1) & 1, err, kErrTma, kWaitNs);
            if (!ok) return;
            ++qn[x];
            ptx::mbar_arrive_expect_tx(&q_full[x], p.tokens * p.group * D * 2);
            for (int h = 0; h < C::kHalves; ++h)
              ptx::tma_load_3d(ptx::smem_addr(q_sm + x * C::kTileBytes + h * kTile * 128), &qmap, &q_full[x], h * 64,
                               it.head * p.group, it.q_row + it.tile[x].t0);
          };
          // Q of row tile 0, K, Q of row tile 1, V: tile 0 starts on the item while tile 1 is at the last one
          load_q(0);
          const int row0 = it.k_row + it.kb * kTile;
          for (int j = 0; j < it.nk && ok; ++j, ++tiles) {
            const int s = tiles % ST;
            const uint32_t ph = ((tiles / ST) & 1) ^ 1;
            // (a CTA that asked for the next item earlier could be left with two while another has none)
            if (j + 1 == it.nk) list.ask(items);
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
              if (j == 0 && kv == 1) load_q(1);
              uint64_t* const bar = kv ? &v_full[s] : &k_full[s];
              ok = ok && (tiles < ST || ptx::mbar_wait(kv ? &v_empty[s] : &k_empty[s], ph, err, kErrTma, kWaitNs));
              if (!ok) break;
              ptx::mbar_arrive_expect_tx(bar, C::kTileBytes);
              const uint32_t dst = ptx::smem_addr((kv ? v_ring : k_ring) + s * C::kTileBytes);
              for (int h = 0; h < C::kHalves; ++h)
                ptx::tma_load_3d(dst + h * kTile * 128, kv ? &vmap : &kmap, bar, h * 64, it.head, row0 + j * kTile);
              ++issued;
            }
          }
          if (ok && it.nk == 0) list.ask(items);
          ok = ok && list.answer(items, &i, err, kErrTma);
        } while (ok && i >= 0);
        if (ok) {
          Item end;
          end.nk = -1;
          ok = list.put(items, end, err, kErrTma);
        }
        if (!ok) {  // a wait gave up: the copies that were issued land before the CTA ends
          for (uint32_t n = issued > 2 * ST ? issued - 2 * ST : 0; n < issued; ++n)
            ptx::mbar_wait((n & 1) ? &v_full[n / 2 % ST] : &k_full[n / 2 % ST], (n / 2 / ST) & 1, err, kErrTma, kWaitNs);
          for (int x = 0; x < 2; ++x)
            if (qn[x]) ptx::mbar_wait(&q_full[x], (qn[x] - 1) & 1, err, kErrTma, kWaitNs);
          if (list.asked > list.taken) ptx::mbar_wait(&items.answered, list.taken & 1, err, kErrTma, kWaitNs);
        }
      }
    } else if (warp == 11) {
      // ---- takes non-finite values out of the V tiles that some row sees only in part
      uint32_t looked = 0;
      int busy = 0;
      while (const Item* const it = work.next<true>(items, err, kErrTma, &ok)) {
        const int nk = it->nk, clean = it->clean, kb = it->kb, klen = it->k_len;
        work.release<true>(items);
        if (nk == 0) continue;
        for (int j = 0; j < nk && ok; ++j, ++tiles) {
          // every tile's barrier is waited for and released, so that it never runs two phases ahead
          ok = __all_sync(0xffffffffu, ptx::mbar_wait(&v_full[tiles % ST], (tiles / ST) & 1, err, kErrTma, kWaitNs));
          if (ok && j < clean && lane == 0) ptx::mbar_arrive(&v_empty[tiles % ST]);
          if (!ok || j < clean) continue;
          uint4* const v = reinterpret_cast<uint4*>(v_ring + (tiles % ST) * C::kTileBytes);
          const __nv_bfloat162 zero = __float2bfloat162_rn(0.f);
#pragma unroll 1
          for (int b = lane; b < C::kTileBytes / 16; b += 32 * 8) {
            uint4 u[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) u[q] = v[b + 32 * q];
            __nv_bfloat162 a[8];  // sums of 0 x: NaN where an x is not finite
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u[q]);
              a[q] = __hfma2(h[3], zero, __hfma2(h[2], zero, __hfma2(h[1], zero, __hmul2(h[0], zero))));
            }
#pragma unroll
            for (int w = 4; w; w >>= 1)
#pragma unroll
              for (int q = 0; q < w; ++q) a[q] = __hadd2(a[q], a[q + w]);
            if (!(__low2float(a[0]) == 0.f && __high2float(a[0]) == 0.f)) {
#pragma unroll 1
              for (int q = 0; q < 8; ++q) {
                __nv_bfloat16* w = reinterpret_cast<__nv_bfloat16*>(v + b + 32 * q);
#pragma unroll 1
                for (int e = 0; e < 8; ++e)
                  if (!isfinite(__bfloat162float(w[e]))) {
                    w[e] = __float2bfloat16_rn(0.f);
                    if ((kb + j) * kTile + (b + 32 * q) / 8 % kTile < klen) bad[busy & 7] = busy + 1;
                  }
              }
            }
          }
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            ptx::mbar_arrive(&seen[looked % ST]);
            ptx::mbar_arrive(&v_empty[tiles % ST]);
          }
          ++looked;
        }
        if (!ok) break;
        ++busy;
      }
    } else if (lane == 0) {
      // ---- products of row tile x: each tile has its own issuing warp, so that one's waits
      // pass while the other's products run
      const int x = warp - 9;
      constexpr uint32_t idesc_s = ptx::idesc_bf16_f32(kTile, kTile);
      constexpr uint32_t idesc_o = ptx::idesc_bf16_f32(kTile, D) | ptx::kIdescBMnMajor;
      const uint32_t ts = tmem + C::kS + x * kTile, to = tmem + C::kO + x * D;
      const uint64_t qd = ptx::sw128_kmajor_desc(ptx::smem_addr(q_sm + x * C::kTileBytes));
      const uint64_t kd = ptx::sw128_kmajor_desc(ptx::smem_addr(k_ring));
      const uint64_t vd = ptx::sw128_mnmajor_desc(ptx::smem_addr(v_ring), kTile * 128);
      uint32_t qn = 0, pn = 0, looked = 0;  // items and key tiles of this row tile; V tiles looked over
      // S = Q K^T; the other warp's turn (hand) comes two products before the end, so that its
      // wake-up passes while they run
      auto scores = [&](uint32_t tile, bool hand) {
        const uint64_t k = kd + (tile % ST) * (C::kTileBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          if (kk == D / 16 - 2 && hand) ptx::mbar_arrive(&turn[x ^ 1]);
          const uint32_t o = ((kk >> 2) * kTile * 128 + (kk & 3) * 32) >> 4;
          ptx::mma_bf16_ss(ts, qd + o, k + o, idesc_s, kk > 0 ? 1u : 0u);
        }
        ptx::tc_commit(&s_full[x]);
        ptx::tc_commit(&k_empty[tile % ST]);
      };
      while (const Item* const it = work.next<false>(items, err, kErrMma, &ok)) {
        const int n = it->tile[x].n, nk = it->nk, clean = it->clean;
        work.release<false>(items);
        if (nk == 0) continue;
        ok = ptx::mbar_wait(&k_full[tiles % ST], (tiles / ST) & 1, err, kErrMma, kWaitNs);
        if (ok && n > 0) {
          ok = ptx::mbar_wait(&q_full[x], qn & 1, err, kErrMma, kWaitNs);
          if (!ok) break;
          ptx::tc_fence_after();
          scores(tiles, false);
          if (n == 1) ptx::tc_commit(&q_empty[x]);
        } else if (ok) {
          ptx::mbar_arrive(&k_empty[tiles % ST]);
        }
        for (int j = 0; j < nk && ok; ++j, ++tiles) {
          const int s = tiles % ST;
          // everything this step needs is waited for, used or not, so that no barrier is ever two phases ahead
          ok = ptx::mbar_wait(&v_full[s], (tiles / ST) & 1, err, kErrMma, kWaitNs);
          if (ok && j >= clean) {
            ok = ptx::mbar_wait(&seen[looked % ST], (looked / ST) & 1, err, kErrMma, kWaitNs);
            ++looked;
          }
          if (ok && j + 1 < nk)
            ok = ptx::mbar_wait(&k_full[(tiles + 1) % ST], ((tiles + 1) / ST) & 1, err, kErrMma, kWaitNs);
          if (ok && j < n) {
            if (j == 0 && qn > 0) ok = ptx::mbar_wait(&o_empty[x], (qn - 1) & 1, err, kErrMma, kWaitNs);
            ok = ok && ptx::mbar_wait(&p_half[x], pn & 1, err, kErrMma, kWaitNs);
          }
          // the two warps issue a step in turn: 0, 1, 0, 1, ..., so the row tiles stay half a step apart
          // (in step, both would wait for their exponentials at once and leave the tensor cores idle)
          const bool both = ok && j < n && ptx::mbar_test(&p_full[x], pn & 1);
          if (ok && (x == 1 || tiles > 0)) ok = ptx::mbar_wait(&turn[x], (x == 1 ? tiles : tiles - 1) & 1, err, kErrMma, kWaitNs);
          if (!ok) break;
          if (j < n) {
            const uint64_t v = vd + s * (C::kTileBytes >> 4);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              if (half && !both) ok = ptx::mbar_wait(&p_full[x], pn & 1, err, kErrMma, kWaitNs);
              if (!ok) break;
              if (!half || !both) ptx::tc_fence_after();
#pragma unroll
              for (int kk = half * 4; kk < half * 4 + 4; ++kk)
                ptx::mma_bf16_ts(to, ts + kk * 8, v + kk * (16 * 128 >> 4), idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
            }
            if (!ok) break;
            ++pn;
            // the score product follows at once; what only frees memory is announced after it
            if (j + 1 == n) {
              ptx::tc_commit(&o_full[x]);
            } else {
              scores(tiles + 1, true);
              if (j + 2 == n) ptx::tc_commit(&q_empty[x]);
            }
            ptx::tc_commit(&v_empty[s]);
          } else {
            ptx::mbar_arrive(&v_empty[s]);
          }
          if (j + 1 >= n && j + 1 < nk) ptx::mbar_arrive(&k_empty[(tiles + 1) % ST]);
          if (j + 1 >= n) ptx::mbar_arrive(&turn[x ^ 1]);
        }
        if (!ok) break;
        if (n > 0) ++qn;
      }
      if (!ok) {  // a wait gave up: what was issued finishes before the tensor memory is freed
        ptx::tc_commit(&drained[x]);
        ptx::mbar_wait(&drained[x], 0, err, kErrMma, kWaitNs);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax and epilogue: a thread has one row
    ptx::reg_inc<208>();
    const int x = warp >> 2;                 // row tile
    const int r = (warp & 3) * 32 + lane;    // row of the tile = lane of the tensor memory
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + C::kS + x * kTile, to = tmem + lanes + C::kO + x * D;
    const int token = r / p.group, head_in = r % p.group;
    uint8_t* const stage = out_sm + warp * 32 * 64;
    // the rows that this thread writes 16 bytes of a pass: 8 q + lane / 4 of its warp
    int w_token[4];
    int64_t w_off[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int row = (warp & 3) * 32 + 8 * q + (lane >> 2);
      w_token[q] = row / p.group;
      w_off[q] = w_token[q] * p.out_stride + row % p.group * D + (lane & 3) * 8;
    }
    ItemReader work;
    int busy = 0;
    uint32_t sn = 0, on = 0;  // key tiles and items of this row tile so far
    bool ok = true;
    while (const Item* const next = work.next<true>(items, err, kErrSoftmax, &ok)) {
      const Item& it = *next;
      const ItemTile tl = it.tile[x];
      const int n = tl.n, kb = it.kb;
      const bool real = token < tl.nt;
      const int sees = real ? max(0, min(it.k_len, tl.first + token)) : 0;  // keys 0 .. sees - 1
      const int whole = max(0, tl.first) / kTile - kb;  // tiles before this one need no mask
      float m = -INFINITY, l = 0.f;  // reference (scaled, base 2) and sum of weights
      for (int j = 0; j < n; ++j, ++sn) {
        // (the warp's lanes go on or give up together)
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&s_full[x], sn & 1, err, kErrSoftmax, kWaitNs));
        if (!ok) break;
        ptx::tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32b_x32(ts + c * 32, s[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) ptx::tmem_wait_regs(s[c]);
        if (j >= whole) {
          const int lim = sees - (kb + j) * kTile;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (__any_sync(0xffffffffu, lim < c * 32 + 32)) {  // columns 32 c .. that some row does not see
              const int n_c = lim - c * 32;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (e >= n_c) s[c][e] = 0xff800000u;
            }
        }
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) mx[c] = fmaxf(__uint_as_float(s[c][0]), __uint_as_float(s[c][1]));
#pragma unroll
        for (int e = 2; e < 32; e += 2)
#pragma unroll
          for (int c = 0; c < 4; ++c) mx[c] = max3(mx[c], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
        // (rows behind the tile's last one hold anything: they have no say in when the others rescale)
        const float top = real ? fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * p.scale_log2 : -INFINITY;
        if (__any_sync(0xffffffffu, top > m + kRescaleLog2)) {
          const float mn = fmaxf(m, top);
          const float f = m == mn ? 1.f : ex2(m - mn);
          m = mn;
          l *= f;
          if (j > 0) {  // the product that wrote O is complete: S of this tile came after it
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              ptx::tmem_ld_32x32b_x32(to + c * 32, o);
              ptx::tmem_wait_regs(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              ptx::tmem_st_32x32b_x32(to + c * 32, o);
            }
          }
        }
        const float mm = m == -INFINITY ? 0.f : -m;  // nothing seen yet: every weight is zero
        const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), m2 = make_float2(mm, mm);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[32];
#pragma unroll
          for (int q = 0; q < 32; ++q) {
            const int cc = 2 * c + q / 16, ii = q % 16 * 2;
            float2 e = fma2(make_float2(__uint_as_float(s[cc][ii]), __uint_as_float(s[cc][ii + 1])), scale2, m2);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            sum[q & 1] = add2(sum[q & 1], e);
            w[q] = pack_bf16x2(e.x, e.y);
          }
          ptx::tmem_st_32x32b_x32(ts + c * 32, w);
          // the product of the first half of the keys starts while the second half is in work
          ptx::tmem_wait_st();
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(c == 0 ? &p_half[x] : &p_full[x]);
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      if (!ok) break;
      uint32_t o[D / 32][32];
      bool fix = false;
      if (n > 0) {
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&o_full[x], on & 1, err, kErrSoftmax, kWaitNs));
        if (!ok) break;
        ++on;
        ptx::tc_fence_after();
#pragma unroll
        for (int c = 0; c < D / 32; ++c) ptx::tmem_ld_32x32b_x32(to + c * 32, o[c]);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) ptx::tmem_wait_regs(o[c]);
        fix = *reinterpret_cast<volatile int*>(&bad[busy & 7]) == busy + 1;
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(&o_empty[x]);
      } else {
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int e = 0; e < 32; ++e) o[c][e] = 0u;
      }
      if (it.nk > 0) ++busy;
      const int64_t grow = static_cast<int64_t>(it.q_row) + tl.t0 + token;
      const int head = it.head * p.group + head_in;
      if (fix && real) {
        // non-finite values of V that this row does see
        for (int key = (kb + it.clean) * kTile; key < min(sees, (kb + n) * kTile); ++key) {
          const __nv_bfloat16* vr = p.v + (it.k_row + static_cast<int64_t>(key)) * p.v_stride + it.head * D;
#pragma unroll
          for (int c = 0; c < D / 32; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float f = __bfloat162float(vr[c * 32 + e]);
              if (!isfinite(f)) o[c][e] = __float_as_uint(__uint_as_float(o[c][e]) + f);
            }
        }
      }
      if (p.splits > 1 && real) {
        const int64_t rec = (grow * p.hq + head) * p.splits + it.split;
        float* ml = p.part + p.part_rows * D + rec * 2;
        ml[0] = n > 0 ? m : -INFINITY;
        ml[1] = l;
        float4* dst = reinterpret_cast<float4*>(p.part + rec * D);
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[c * 8 + e] = make_float4(__uint_as_float(o[c][4 * e]), __uint_as_float(o[c][4 * e + 1]),
                                         __uint_as_float(o[c][4 * e + 2]), __uint_as_float(o[c][4 * e + 3]));
      } else if (p.splits == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        // through shared memory, 32 dimensions a pass: a row straight from its thread would
        // touch 32 lines with every store (4096 line accesses an item, now 1024)
        __nv_bfloat16* const dst =
            p.out + (static_cast<int64_t>(it.q_row) + tl.t0) * p.out_stride + it.head * p.group * D;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              w[q] = pack_bf16x2(__uint_as_float(o[c][8 * e + 2 * q]) * inv, __uint_as_float(o[c][8 * e + 2 * q + 1]) * inv);
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((e ^ (lane >> 1 & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int row = 8 * q + (lane >> 2);
            const uint4 w = *reinterpret_cast<const uint4*>(stage + row * 64 + (((lane & 3) ^ (row >> 1 & 3)) << 4));
            if (w_token[q] < tl.nt) *reinterpret_cast<uint4*>(dst + w_off[q] + c * 32) = w;
          }
          __syncwarp();
        }
      }
      work.release<true>(items);
    }
    ptx::tc_fence_before();
  }
  __syncthreads();
  if (warp == 9) {
    ptx::tmem_relinquish();
    ptx::tmem_dealloc(tmem, C::kCols);
  }
}

// Merges the splits: D / 4 threads for each (row, head).
template <int D>
__global__ void __launch_bounds__(128) prompt_combine_kernel(const __grid_constant__ PromptParams p, int64_t rows) {
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x) / (D / 4);  // (row, head)
  const int d4 = threadIdx.x % (D / 4) * 4;
  if (at >= rows * p.hq) return;
  const int64_t rec = at * p.splits;
  const float* ml = p.part + p.part_rows * D + rec * 2;
  float m = -INFINITY;  // (the splits' loads are in flight together)
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[2 * s]);
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    // no reference: nothing seen (no sum), or nothing but NaN, which stays
    const float ms = ml[2 * s], ls = ml[2 * s + 1], f = ms == -INFINITY ? (ls == 0.f ? 0.f : 1.f) : ex2(ms - m);
    const float4 v = *reinterpret_cast<const float4*>(p.part + (rec + s) * D + d4);
    const bool none = f == 0.f;  // what it holds has no say, an infinity neither
    l += none ? 0.f : f * ls;
    o.x += none ? 0.f : f * v.x;
    o.y += none ? 0.f : f * v.y;
    o.z += none ? 0.f : f * v.z;
    o.w += none ? 0.f : f * v.w;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint2 w;
  w.x = pack_bf16x2(o.x * inv, o.y * inv);
  w.y = pack_bf16x2(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(p.out + at / p.hq * p.out_stride + at % p.hq * D + d4) = w;
}

int sm_count_prompt() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n > 0 ? n : 148;
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
  // Few blocks with many keys: the keys are split over the idle SMs and joined by a second
  // launch. Measured: a key tile takes 1.6 us where one row tile is at work alone, as in such blocks
  // (2.1 with two, heads of 128), the second launch 3 us and its partial results, written and read once, pass at 3 TB/s. One row behind 8000 keys 99.6 -> 20.7 us, behind
  // 1000 16.4 -> 10.2; 8 chunks of 16 rows behind 768 keys would go from 16.4 to 18.0.
  const int64_t ctas = std::max<int64_t>(1, items * hkv);
  const int64_t limit = std::min<int64_t>(sm_count_prompt() / ctas, most);
  double best = 1.6 * most;
  pl->splits = 1;
  for (int64_t s = 2; s <= limit; ++s) {
    const double us = 1.6 * ((most + s - 1) / s) + 3.0 + 8.0 * pl->total_q * hq * s * head_dim / 3.0e6;
    if (us < best) {
      best = us;
      pl->splits = static_cast<int>(s);
    }
  }
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
  SWL_CUDA_TRY(launch_kernel(prompt_attention_kernel<D>, dim3(p.items), dim3(kThreads),
                             Cfg<D>::kSmem, st, 1, pl.t, p, qm, km, vm));
  if (p.splits > 1)
    SWL_CUDA_TRY(launch_kernel(prompt_combine_kernel<D>, dim3(static_cast<unsigned>((pl.total_q * p.hq * (D / 4) + 127) / 128)),
                               dim3(128), 0, st, 1, p, pl.total_q));
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
  p.items = pl.items * hkv * pl.splits;
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
