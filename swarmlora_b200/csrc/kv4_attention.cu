// Causal GQA attention of each slot's newest rows over its paged 4-bit cache.
#include <cuda_bf16.h>

#include <cmath>

#include "common.h"
#include "kv4.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace swl {
namespace kv4 {

namespace {

struct AttnTable4 {
  RowSegments seg;
  __nv_bfloat16* out[kMaxSlots];
  Cache c;
};
struct AttnParams4 {
  int hq;
  int64_t out_stride;
  float scale;
  const __nv_bfloat16* q;  // [total_rows, hq * D]
};

// CTA = one (row, query head); a thread takes a key of each chunk of D tokens for the
// scores, then a dimension for the values.
template <int D>
__global__ void __launch_bounds__(D) kv4_attention_kernel(const __grid_constant__ AttnTable4 tab, const AttnParams4 p) {
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int gr = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  int s = 0;
  while (tab.seg.row_start[s + 1] <= gr) ++s;
  const int local = gr - tab.seg.row_start[s], hk = h / (p.hq / tab.c.hkv);
  const int64_t len = static_cast<int64_t>(*tab.c.seqlen[s]) + local + 1;
  __shared__ float q[D], pr[D], red[D / 32];
  q[tid] = __bfloat162float(p.q[(static_cast<int64_t>(gr) * p.hq + h) * D + tid]) * p.scale;
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int64_t t0 = 0; t0 < len; t0 += D) {
    __syncthreads();
    const int64_t pos = t0 + tid;
    const uint8_t* blk = pos < len ? block_of<D>(tab.c, s, pos >> 4, hk) : nullptr;
    float sc = -INFINITY;
    if (blk) {
      const int t = static_cast<int>(pos & 15);
      sc = 0.f;
      for (int d = 0; d < D; d += 8) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(blk + k_word<D>(t, d));
        const uint32_t pp = *reinterpret_cast<const uint32_t*>(blk + k_pair_off(D) + 4 * (t * (D / kGroup) + d / kGroup));
        for (int e = 0; e < 8; ++e)
          sc += q[d + e] * (__uint_as_float(pp << 16) * static_cast<float>(w >> (4 * e) & 15u) + __uint_as_float(pp & 0xffff0000u));
      }
    }
    float mx = sc;
    for (int x = 16; x; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    float mn = m;
    for (int w = 0; w < D / 32; ++w) mn = fmaxf(mn, red[w]);
    pr[tid] = sc == -INFINITY ? 0.f : expf(sc - mn);
    __syncthreads();
    const float corr = mn == -INFINITY ? 1.f : expf(m - mn);
    l *= corr;
    o *= corr;
    m = mn;
    const int n = static_cast<int>(min(static_cast<int64_t>(D), len - t0));
    for (int i = 0; i < n; ++i) {
      const uint8_t* b = block_of<D>(tab.c, s, (t0 + i) >> 4, hk);
      if (!b) continue;
      const int t = static_cast<int>((t0 + i) & 15);
      const uint32_t pp = *reinterpret_cast<const uint32_t*>(b + v_pair_off(D) + 4 * (t * (D / kGroup) + tid / kGroup));
      const uint32_t code = *reinterpret_cast<const uint16_t*>(b + v_piece<D>(t, tid & ~3)) >> (4 * (tid & 3)) & 15u;
      l += pr[i];
      o += pr[i] * (__uint_as_float(pp << 16) * static_cast<float>(code) + __uint_as_float(pp & 0xffff0000u));
    }
  }
  tab.out[s][static_cast<int64_t>(local) * p.out_stride + h * D + tid] = __float2bfloat16_rn(l == 0.f ? 0.f : o / l);
}

}  // namespace
}  // namespace kv4
}  // namespace swl

using namespace swl;

SWL_EXPORT int64_t swl_kv4_part_floats(int nseg, const int* rows, int hq, int hkv, int head_dim, int max_len) {
  (void)nseg; (void)rows; (void)hq; (void)hkv; (void)head_dim; (void)max_len;
  return 0;
}

SWL_EXPORT int swl_paged_attention_kv4(int nseg, const int* rows, const void* const* block_tables, int table_len,
                                       const void* const* caches, int64_t num_pages, const void* const* seqlens,
                                       void* const* out, int64_t out_stride, int hq, int hkv, int head_dim, int page,
                                       float scale, int max_len, const void* q_rot, float* part, void* stream) {
  kv4::AttnTable4 t;
  SWL_TRY(kv4::fill_rows(&t.seg, "attention_kv4", nseg, rows));
  if (!seqlens && nseg > 0) return set_error(SWL_ERR_ARG, "attention_kv4: null context lengths");
  SWL_TRY(kv4::fill_cache(&t.c, "attention_kv4", nseg, block_tables, table_len, const_cast<void* const*>(caches), num_pages,
                          seqlens, hkv, head_dim, page));
  if (hq < 1 || hq > 4096 || hq % hkv) return set_error(SWL_ERR_ARG, "attention_kv4: query heads must be a multiple of kv heads");
  if (!(scale > 0.f) || !std::isfinite(scale)) return set_error(SWL_ERR_ARG, "attention_kv4: scale must be positive and finite");
  if (max_len < 1) return set_error(SWL_ERR_ARG, "attention_kv4: max_len must be positive");
  if (!q_rot || (reinterpret_cast<uintptr_t>(q_rot) & 15)) return set_error(SWL_ERR_ARG, "attention_kv4: q must be 16-byte aligned");
  if (out_stride < static_cast<int64_t>(hq) * head_dim || out_stride % 8)
    return set_error(SWL_ERR_ARG, "attention_kv4: output stride must hold all heads and be a multiple of 8");
  if (nseg > 0 && !out) return set_error(SWL_ERR_ARG, "attention_kv4: null outputs");
  for (int i = 0; i < nseg; ++i) {
    t.out[i] = static_cast<__nv_bfloat16*>(out[i]);
    if (!t.out[i] || (reinterpret_cast<uintptr_t>(t.out[i]) & 15))
      return set_error(SWL_ERR_ARG, "attention_kv4: outputs must be 16-byte aligned");
  }
  (void)part;
  if (t.seg.total_rows == 0) return SWL_OK;
  kv4::AttnParams4 p;
  p.hq = hq;
  p.out_stride = out_stride;
  p.scale = scale;
  p.q = static_cast<const __nv_bfloat16*>(q_rot);
  const dim3 grid(t.seg.total_rows, hq);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  SWL_CUDA_TRY(head_dim == 128 ? launch_kernel(kv4::kv4_attention_kernel<128>, grid, dim3(128), 0, st, 1, t, p)
                               : launch_kernel(kv4::kv4_attention_kernel<64>, grid, dim3(64), 0, st, 1, t, p));
  return SWL_OK;
}
