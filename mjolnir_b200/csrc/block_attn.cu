// Attention of ragged query chunks over the block-scaled cache.
//
// One warp per (query token, query head): lanes hold the head row, keys are
// taken in turn with a running maximum and sum.
#include "block_cache.cuh"

namespace mj {

template <typename T, int D>
__global__ void __launch_bounds__(128) block_attn_kernel(mj_block_attn_args a, int lg) {
  constexpr int E = D / 32;
  const int64_t w = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int64_t t = w / a.h_q;
  const int hq = (int)(w % a.h_q), h = hq / (a.h_q / a.h_k);
  if (t >= a.num_tokens || t >= a.q_start[a.num_seqs]) return;
  int lo = 0, hi = a.num_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.q_start[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  const int n = a.q_start[lo + 1] - a.q_start[lo], L = a.seq_lens[lo];
  const int keys = a.causal ? L - n + (int)(t - a.q_start[lo]) + 1 : L;
  const T* qp = static_cast<const T*>(a.q) + t * a.q_stride_tok + hq * a.q_stride_head + lane * E;
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) q[i] = (float)qp[i] * a.softmax_scale, o[i] = 0.f;
  for (int j = 0; j < keys; ++j) {
    const int col = j / a.page_size, r = j % a.page_size;
    const int page = col < a.block_table_cols ? a.block_table[lo * a.block_table_stride + col] : -1;
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0) flag(a.status, MJ_DEV_BAD_PAGE);
      continue;
    }
    const unsigned char* kp = static_cast<const unsigned char*>(a.k_cache) + page * a.k_stride_page + r * a.k_stride_row + h * a.k_stride_head + lane * E;
    const unsigned char* vp = static_cast<const unsigned char*>(a.v_cache) + page * a.v_stride_page + r * a.v_stride_row + h * a.v_stride_head + lane * E;
    const float ks = block_scale(*(static_cast<const unsigned char*>(a.k_scales) + page * a.ks_stride_page + (r >> lg) * a.ks_stride_block + h * a.ks_stride_head));
    const float vs = block_scale(*(static_cast<const unsigned char*>(a.v_scales) + page * a.vs_stride_page + (r >> lg) * a.vs_stride_block + h * a.vs_stride_head));
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) s = fmaf(q[i], e4m3_value(kp[i]), s);
    s = warp_allsum(s) * ks;
    const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.f : __expf(m - mn), p = __expf(s - mn);
    l = l * c + p;
    m = mn;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = fmaf(p * vs, e4m3_value(vp[i]), o[i] * c);
  }
  T* op = static_cast<T*>(a.o) + t * a.o_stride_tok + hq * a.o_stride_head + lane * E;
#pragma unroll
  for (int i = 0; i < E; ++i) op[i] = (T)(l == 0.f ? 0.f : o[i] / l);  // a NaN sum stays NaN
  if (a.lse && lane == 0) a.lse[t * a.h_q + hq] = l == 0.f ? -INFINITY : m + logf(l);
}

cudaError_t launch_block_attention(const mj_block_attn_args& a, cudaStream_t stream) {
  const int lg = block_log2(a.kv_format);
  const dim3 grid((unsigned)((a.num_tokens * a.h_q + 3) / 4));
  if (a.dtype == MJ_DT_FP16) {
    if (a.head_size == 256) block_attn_kernel<__half, 256><<<grid, 128, 0, stream>>>(a, lg);
    else block_attn_kernel<__half, 128><<<grid, 128, 0, stream>>>(a, lg);
  } else {
    if (a.head_size == 256) block_attn_kernel<__nv_bfloat16, 256><<<grid, 128, 0, stream>>>(a, lg);
    else block_attn_kernel<__nv_bfloat16, 128><<<grid, 128, 0, stream>>>(a, lg);
  }
  return cudaGetLastError();
}

}  // namespace mj
