// Causal GQA attention over packed sequences of different lengths.
#include <cuda_bf16.h>

#include <cmath>

#include "common.h"
#include "kv4.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace swl {

namespace {

struct PromptTable {
  RowSegments q, k;  // packed rows of the queries and of the keys
};
struct PromptParams {
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* out;
  int64_t q_stride, k_stride, v_stride, out_stride;
  int hq, hkv;
  float scale;
};

// CTA = one (row, query head); a thread takes a key of each chunk of D for the scores,
// then a dimension for the values.
template <int D>
__global__ void __launch_bounds__(D) prompt_attention_kernel(const __grid_constant__ PromptTable tab, const PromptParams p) {
  ptx::grid_dep_wait();
  ptx::grid_dep_launch();
  const int64_t gr = blockIdx.x;
  const int h = blockIdx.y, hk = h / (p.hq / p.hkv), tid = threadIdx.x;
  int s = 0;
  while (tab.q.row_start[s + 1] <= gr) ++s;
  const int ql = tab.q.row_start[s + 1] - tab.q.row_start[s], kl = tab.k.row_start[s + 1] - tab.k.row_start[s];
  const int len = static_cast<int>(gr - tab.q.row_start[s]) + kl - ql + 1;  // keys this row sees
  __shared__ float q[D], pr[D], red[D / 32];
  q[tid] = __bfloat162float(p.q[gr * p.q_stride + h * D + tid]) * p.scale;
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int t0 = 0; t0 < len; t0 += D) {
    __syncthreads();
    float sc = -INFINITY;
    if (t0 + tid < len) {
      const __nv_bfloat16* k = p.k + (tab.k.row_start[s] + t0 + tid) * p.k_stride + hk * D;
      sc = 0.f;
      for (int d = 0; d < D; ++d) sc = fmaf(q[d], __bfloat162float(k[d]), sc);
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
    for (int i = 0; i < min(D, len - t0); ++i) {
      l += pr[i];
      o = fmaf(pr[i], __bfloat162float(p.v[(tab.k.row_start[s] + t0 + i) * p.v_stride + hk * D + tid]), o);
    }
  }
  p.out[gr * p.out_stride + h * D + tid] = __float2bfloat16_rn(len > 0 ? o / l : 0.f);
}

}  // namespace
}  // namespace swl

using namespace swl;

SWL_EXPORT int64_t swl_prompt_attention_part_floats(int nseg, const int* q_lens, const int* k_lens, int hq, int hkv,
                                                    int head_dim) {
  (void)nseg; (void)q_lens; (void)k_lens; (void)hq; (void)hkv; (void)head_dim;
  return 0;
}

SWL_EXPORT int swl_prompt_attention(int nseg, const int* q_lens, const int* k_lens, const void* q, int64_t q_stride,
                                    const void* k, int64_t k_stride, const void* v, int64_t v_stride, void* out,
                                    int64_t out_stride, int hq, int hkv, int head_dim, float scale, float* part,
                                    void* stream) {
  PromptTable t;
  SWL_TRY(kv4::fill_rows(&t.q, "prompt_attention", nseg, q_lens));
  SWL_TRY(kv4::fill_rows(&t.k, "prompt_attention", nseg, k_lens));
  if (head_dim != 64 && head_dim != 128) return set_error(SWL_ERR_ARG, "prompt_attention: head_dim must be 64 or 128");
  if (hkv < 1 || hq < 1 || hq % hkv || hq / hkv > 128 || hq > 4096)
    return set_error(SWL_ERR_ARG, "prompt_attention: query heads must be a multiple of kv heads, at most 128 each");
  if (!(scale > 0.f) || !std::isfinite(scale)) return set_error(SWL_ERR_ARG, "prompt_attention: scale must be positive and finite");
  const int64_t qw = static_cast<int64_t>(hq) * head_dim, kw = static_cast<int64_t>(hkv) * head_dim;
  if (q_stride < qw || out_stride < qw || k_stride < kw || v_stride < kw)
    return set_error(SWL_ERR_ARG, "prompt_attention: row strides must hold all heads");
  if ((q_stride | out_stride | k_stride | v_stride) % 8 || (q_stride | out_stride | k_stride | v_stride) >> 36)
    return set_error(SWL_ERR_ARG, "prompt_attention: row strides must be multiples of 8 below 2^36");
  if (t.q.total_rows == 0) return SWL_OK;
  if (!q || !out || (t.k.total_rows > 0 && (!k || !v))) return set_error(SWL_ERR_ARG, "prompt_attention: null tensor");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out)) & 15)
    return set_error(SWL_ERR_ARG, "prompt_attention: tensors must be 16-byte aligned");
  (void)part;
  PromptParams p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.v = static_cast<const __nv_bfloat16*>(v);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.out_stride = out_stride;
  p.hq = hq;
  p.hkv = hkv;
  p.scale = scale;
  const dim3 grid(t.q.total_rows, hq);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  SWL_CUDA_TRY(head_dim == 128 ? launch_kernel(prompt_attention_kernel<128>, grid, dim3(128), 0, st, 1, t, p)
                               : launch_kernel(prompt_attention_kernel<64>, grid, dim3(64), 0, st, 1, t, p));
  return SWL_OK;
}
