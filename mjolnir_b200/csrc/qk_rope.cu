// RMS norm of Q and K per head with the position rotation, in one pass.
//
// y = x * rsqrt(mean(x^2) + eps) * w, then for each pair (a, b) of the first
// rot_dim elements (a cos - b sin, b cos + a sin); fp32 throughout, one
// rounding at the store.
//
// A team of threads (a power of two, head_size / 16 rounded up) owns one head
// row; a thread owns two chunks of 8 elements. For the half-split pairing
// (i, i + rot_dim / 2) those are the same chunk of both halves, so every
// rotation is inside one thread and the row's sum of squares is the only
// exchange.
#include <type_traits>

#include "common.cuh"

namespace mj {

template <typename T>
struct Chunk;  // 8 elements
template <>
struct Chunk<float> {
  static __device__ __forceinline__ void load(const float* p, float* v, bool vec) {
    if (vec) {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p[i];
    }
  }
  static __device__ __forceinline__ void store(float* p, const float* v, bool vec) {
    if (vec) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = v[i];
    }
  }
};
template <typename T>
struct Half8 {
  static __device__ __forceinline__ float up(T x) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) return __half2float(x);
    else return __bfloat162float(x);
  }
  static __device__ __forceinline__ T down(float x) {
    if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
  }
  static __device__ __forceinline__ void load(const T* p, float* v, bool vec) {
    if (vec) {
      const uint4 raw = *reinterpret_cast<const uint4*>(p);
      const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = up(e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = up(p[i]);
    }
  }
  static __device__ __forceinline__ void store(T* p, const float* v, bool vec) {
    if (vec) {
      uint4 raw;
      T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = down(v[i]);
      *reinterpret_cast<uint4*>(p) = raw;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = down(v[i]);
    }
  }
};
template <>
struct Chunk<__half> : Half8<__half> {};
template <>
struct Chunk<__nv_bfloat16> : Half8<__nv_bfloat16> {};

__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
  const float x = a * c - b * s;
  b = b * c + a * s;
  a = x;
}

// vec: every row and table address is 16-byte aligned (host-checked)
template <typename T>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(mj_qk_norm_rope_args a, int team_log2, bool vec) {
  griddep_wait();
  const int team = 1 << team_log2;
  const int64_t row = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> team_log2;
  const int j = threadIdx.x & (team - 1);
  const int heads = a.h_q + a.h_k;
  const int64_t t = row / heads;
  int h = (int)(row - t * heads);
  const bool live = t < a.num_tokens;
  const int nc = a.head_size >> 3, r2 = a.rot_dim >> 4;  // chunks of a row, rotating chunk pairs
  const bool is_k = h >= a.h_q;
  if (is_k) h -= a.h_q;
  const bool mine = live && 2 * j < nc;
  const int ca = a.interleaved || j >= r2 ? 2 * j : j, cb = a.interleaved || j >= r2 ? 2 * j + 1 : j + r2;
  float x[8], y[8];
  if (mine) {
    const T* p = static_cast<const T*>(is_k ? a.k : a.q) + t * (is_k ? a.k_stride_tok : a.q_stride_tok) +
                 h * (is_k ? a.k_stride_head : a.q_stride_head);
    Chunk<T>::load(p + 8 * ca, x, vec);
    Chunk<T>::load(p + 8 * cb, y, vec);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
  }
  // summed for every row: teams of one warp may differ in having a weight
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], fmaf(y[i], y[i], ss));
  for (int o = team >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const void* w = is_k ? a.k_weight : a.q_weight;
  if (w && mine) {
    const float r = rsqrtf(ss / (float)a.head_size + a.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] *= r * load_elem(w, 8 * ca + i, a.weight_dtype);
      y[i] *= r * load_elem(w, 8 * cb + i, a.weight_dtype);
    }
  }
  if (!mine) return;
  if (r2) {
    const int64_t pos = a.positions[t];
    if (pos < 0 || pos >= a.num_positions) {
      if (j == 0) flag(a.status, MJ_DEV_BAD_POSITION);
      return;
    }
    const int64_t cs = pos * a.cos_sin_stride;
    const int half = a.rot_dim >> 1;
    if (a.interleaved) {
      if (ca * 8 < a.rot_dim) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          rotate(x[2 * i], x[2 * i + 1], load_elem(a.cos_sin, cs + 4 * ca + i, a.cos_sin_dtype),
                 load_elem(a.cos_sin, cs + half + 4 * ca + i, a.cos_sin_dtype));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          rotate(y[2 * i], y[2 * i + 1], load_elem(a.cos_sin, cs + 4 * cb + i, a.cos_sin_dtype),
                 load_elem(a.cos_sin, cs + half + 4 * cb + i, a.cos_sin_dtype));
      }
    } else if (j < r2) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        rotate(x[i], y[i], load_elem(a.cos_sin, cs + 8 * j + i, a.cos_sin_dtype),
               load_elem(a.cos_sin, cs + half + 8 * j + i, a.cos_sin_dtype));
    }
  }
  T* o = static_cast<T*>(is_k ? a.k_out : a.q_out) + t * (is_k ? a.ko_stride_tok : a.qo_stride_tok) +
         h * (is_k ? a.ko_stride_head : a.qo_stride_head);
  Chunk<T>::store(o + 8 * ca, x, vec);
  Chunk<T>::store(o + 8 * cb, y, vec);
}

cudaError_t launch_qk_norm_rope(const mj_qk_norm_rope_args& a, bool vec, cudaStream_t stream) {
  int team_log2 = 0;
  while ((16 << team_log2) < a.head_size) ++team_log2;
  const int64_t threads = a.num_tokens * (a.h_q + a.h_k) << team_log2;
  const dim3 grid((unsigned)((threads + 255) / 256));
  if (a.dtype == MJ_DT_FP32) return launch_kernel(qk_norm_rope_kernel<float>, grid, dim3(256), 0, stream, a, team_log2, vec);
  if (a.dtype == MJ_DT_FP16) return launch_kernel(qk_norm_rope_kernel<__half>, grid, dim3(256), 0, stream, a, team_log2, vec);
  return launch_kernel(qk_norm_rope_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, a, team_log2, vec);
}

}  // namespace mj
