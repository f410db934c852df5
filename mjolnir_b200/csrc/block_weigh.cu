// The attention weight that each cached token receives in a step, added up per
// KV head: w[s][h][j] += sum over the rows (query, head of the group) that see
// key j of exp(scale q . k_j - lse).
#include <math.h>

#include "block_cache.cuh"

namespace mj {

// One warp per key: the row of K in registers, then every query row that sees it.
template <typename T, int D>
__global__ void __launch_bounds__(256) block_weigh_kernel(const __grid_constant__ mj_block_weigh_args a, int lg, int blocks) {
  griddep_wait();
  constexpr int E = D / 32;  // elements of a lane
  const int lane = threadIdx.x & 31;
  const int x = blockIdx.x % blocks, sh = blockIdx.x / blocks, h = sh % a.h_k, seq = sh / a.h_k;
  const int q0 = a.offsets[seq], q1 = a.offsets[seq + 1], L = a.seq_lens[seq], n = q1 - q0;
  if (q0 < 0 || n < 0 || q1 > a.num_rows || L < 0 || L > a.weights_cols || L > (int64_t)a.block_table_cols * a.page_size) {
    if (threadIdx.x == 0) flag(a.status, MJ_DEV_BAD_LENGTH);
    return;
  }
  const int h_r = a.h_q / a.h_k, first = a.window ? max(n - a.window, 0) : 0;
  float* w = a.weights + seq * a.w_stride_seq + h * a.w_stride_head;
  for (int j = x * 8 + (threadIdx.x >> 5); j < L; j += blocks * 8) {
    const int page = a.block_table[seq * a.block_table_stride + j / a.page_size], r = j % a.page_size;
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0) flag(a.status, MJ_DEV_BAD_PAGE);
      continue;
    }
    const unsigned char* row = static_cast<const unsigned char*>(a.k_cache) + page * a.k_stride_page + r * a.k_stride_row + h * a.k_stride_head;
    const float f = block_scale(static_cast<const unsigned char*>(a.k_scales)[page * a.ks_stride_page + (r >> lg) * a.ks_stride_block + h * a.ks_stride_head]);
    float k[E];
#pragma unroll
    for (int i = 0; i < E; ++i) k[i] = e4m3_value(row[lane * E + i]) * f;
    float sum = 0.f;
    for (int t = max(first, j - (L - n)); t < n; ++t)
      for (int g = 0; g < h_r; ++g) {
        const int hq = h * h_r + g;
        const T* q = static_cast<const T*>(a.q) + (int64_t)(q0 + t) * a.q_stride_tok + hq * a.q_stride_head + lane * E;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) s = fmaf((float)q[i], k[i], s);
        s = warp_allsum(s);
        const float z = a.lse[(int64_t)(q0 + t) * a.h_q + hq];
        if (z != -INFINITY) sum += expf(s * a.softmax_scale - z);
      }
    if (lane == 0) w[j] = (j >= L - n ? 0.f : w[j]) + sum;
  }
}

template <typename T>
static cudaError_t weigh_t(const mj_block_weigh_args& a, cudaStream_t stream) {
  const int blocks = 64;
  const dim3 grid((unsigned)(a.num_seqs * a.h_k * blocks));
  auto kern = a.head_size == 256 ? block_weigh_kernel<T, 256> : block_weigh_kernel<T, 128>;
  return launch_kernel(kern, grid, dim3(256), 0, stream, a, block_log2(a.kv_format), blocks);
}

cudaError_t launch_block_weigh(const mj_block_weigh_args& a, cudaStream_t stream) {
  return a.dtype == MJ_DT_FP16 ? weigh_t<__half>(a, stream) : weigh_t<__nv_bfloat16>(a, stream);
}

}  // namespace mj
