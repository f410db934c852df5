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
#include "block_cache.cuh"

namespace mj {

using namespace sm100;

// 8 elements of a row; vec: its address is 16-byte aligned
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const float* v, bool vec) {
  if (vec) {
    store8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = (T)v[i];
  }
}
// 8 elements of a table of any of the three types: as they are in memory, so
// that several are on their way before one is used, then as floats
struct RawTable {
  uint4 v[2];
  __device__ __forceinline__ void load(const void* p, int64_t i, int dt, bool vec) {
    const char* q = static_cast<const char*>(p) + i * (dt == MJ_DT_FP32 ? 4 : 2);
    if (vec) {
      v[0] = reinterpret_cast<const uint4*>(q)[0];
      if (dt == MJ_DT_FP32) v[1] = reinterpret_cast<const uint4*>(q)[1];
    } else if (dt == MJ_DT_FP32) {
#pragma unroll
      for (int k = 0; k < 8; ++k) reinterpret_cast<uint32_t*>(v)[k] = reinterpret_cast<const uint32_t*>(q)[k];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) reinterpret_cast<uint16_t*>(v)[k] = reinterpret_cast<const uint16_t*>(q)[k];
    }
  }
  __device__ __forceinline__ void get(int dt, float* x) const {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      x[k] = dt == MJ_DT_BF16   ? (float)reinterpret_cast<const __nv_bfloat16*>(v)[k]
             : dt == MJ_DT_FP16 ? (float)reinterpret_cast<const __half*>(v)[k]
                                : reinterpret_cast<const float*>(v)[k];
  }
};

__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
  const float x = a * c - b * s;
  b = b * c + a * s;
  a = x;
}

// What bounds it: memory latency. A warp's rows, position, weights and cosines
// are four groups of loads, of which only the cosines wait for another
// (the position); five CTAs of 128 threads an SM keep 20 warps of them in
// flight (4: 39.9 us for 8192 tokens x 40 heads of 128, 5: 35.5, 4.8 TB/s, with
// one or two registers of the 16-bit variants spilled; 6, with more: 46). In fp32
// the same call is bound by memory, 55 us, 6.2 TB/s. A ring of cp.async stages in persistent CTAs took 62.
// A team takes HG heads of one token's Q, or of its K: the cosines, sines and
// weights of its two chunks stay in registers for all of them, and the heads'
// loads are in flight together.
// VEC: every row, weight and table address is 16-byte aligned (host-checked)
// TL: log2 of a team's threads
template <typename T, int HG, bool VEC, int TL>
__global__ void __launch_bounds__(128, sizeof(T) == 4 ? 3 : 5) qk_norm_rope_kernel(mj_qk_norm_rope_args a, float inv_d) {
  griddep_wait();
  constexpr int team = 1 << TL;
  const int64_t unit = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> TL;
  const int j = threadIdx.x & (team - 1);
  const int qg = (a.h_q + HG - 1) / HG, groups = qg + (a.h_k + HG - 1) / HG;
  const int64_t t = unit >> 32 ? unit / groups : (uint32_t)unit / (uint32_t)groups;  // a 64-bit division is a long routine
  int g = (int)(unit - t * groups);
  const int nc = a.head_size >> 3, r2 = a.rot_dim >> 4;  // chunks of a row, rotating chunk pairs
  const bool is_k = g >= qg;
  if (is_k) g -= qg;
  const int h0 = g * HG, heads = min(HG, (is_k ? a.h_k : a.h_q) - h0);
  const bool mine = t < a.num_tokens && 2 * j < nc;
  const int ca = a.interleaved || j >= r2 ? 2 * j : j, cb = a.interleaved || j >= r2 ? 2 * j + 1 : j + r2;
  const bool turns = mine && r2 && (a.interleaved ? 16 * j < a.rot_dim : j < r2);
  const int64_t pos = mine && r2 ? a.positions[t] : 0;
  const int64_t st = is_k ? a.k_stride_tok : a.q_stride_tok, sh = is_k ? a.k_stride_head : a.q_stride_head;
  const T* in = static_cast<const T*>(is_k ? a.k : a.q) + t * st + h0 * sh;
  // a missing head's or thread's chunks repeat ones that are there, and are not stored
  Raw8<T> rx[HG], ry[HG];
  if (t < a.num_tokens) {
    const int at = 2 * j < nc ? 1 : 0;
#pragma unroll
    for (int h = 0; h < HG; ++h) {
      const T* row = in + (h < heads ? h : 0) * sh;
      rx[h].load(row + 8 * ca * at, VEC);
      ry[h].load(row + 8 * cb * at, VEC);
    }
  }
  auto f = [](float2* p) { return reinterpret_cast<float*>(p); };
  const void* w = is_k ? a.k_weight : a.q_weight;
  float2 wx[4], wy[4], c[4], s[4];  // packed pairs: half the instructions
  RawTable raw[2], turn[2];
  if (mine && w) {
    raw[0].load(w, 8 * ca, a.weight_dtype, VEC);
    raw[1].load(w, 8 * cb, a.weight_dtype, VEC);
  }
  const bool bad = mine && r2 && (pos < 0 || pos >= a.num_positions);
  if (bad && j == 0) flag(a.status, MJ_DEV_BAD_POSITION);  // (looked at once the rows are on their way)
  if (turns && !bad) {  // a pair of chunks turns by 8 angles in either pairing
    turn[0].load(a.cos_sin, pos * a.cos_sin_stride + 8 * j, a.cos_sin_dtype, VEC);
    turn[1].load(a.cos_sin, pos * a.cos_sin_stride + (a.rot_dim >> 1) + 8 * j, a.cos_sin_dtype, VEC);
  }
  raw[0].get(a.weight_dtype, f(wx));
  raw[1].get(a.weight_dtype, f(wy));
  turn[0].get(a.cos_sin_dtype, f(c));
  turn[1].get(a.cos_sin_dtype, f(s));
  T* out = static_cast<T*>(is_k ? a.k_out : a.q_out) + t * (is_k ? a.ko_stride_tok : a.qo_stride_tok);
  const int64_t oh = is_k ? a.ko_stride_head : a.qo_stride_head;
#pragma unroll
  for (int h = 0; h < HG; ++h) {
    // summed for every row: teams of one warp may differ in having a weight
    float2 x[4], y[4], sq = make_float2(0.f, 0.f);
    rx[h].get(f(x));
    ry[h].get(f(y));
    if (mine) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sq = ffma2(x[i], x[i], ffma2(y[i], y[i], sq));
    }
    float ss = sq.x + sq.y;
#pragma unroll
    for (int o = team >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!mine || bad || h >= heads) continue;
    if (w) {
      const float r = rsqrtf(fmaf(ss, inv_d, a.eps));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = fmul2(x[i], fmul2(make_float2(r, r), wx[i]));
        y[i] = fmul2(y[i], fmul2(make_float2(r, r), wy[i]));
      }
    }
    if (turns) {
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          rotate(x[i].x, x[i].y, f(c)[i], f(s)[i]);
          rotate(y[i].x, y[i].y, f(c)[4 + i], f(s)[4 + i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 t = ffma2(x[i], c[i], fmul2(y[i], make_float2(-s[i].x, -s[i].y)));
          y[i] = ffma2(y[i], c[i], fmul2(x[i], s[i]));
          x[i] = t;
        }
      }
    }
    store_chunk(out + (h0 + h) * oh + 8 * ca, f(x), VEC);
    store_chunk(out + (h0 + h) * oh + 8 * cb, f(y), VEC);
  }
}

// Heads of a thread: four in large calls (8192 tokens x 40 heads 35 us; with two
// 43, with five 39; 6553 tokens 29, with one 37), one in small ones, to fill the
// GPU. The edge in 16 bits, one head and four, 40 heads of 128: 2^17 threads 3.2 and 3.6 us, 2^18
// 5.2 and 4.6, 2^18.9 9.7 and 8.5; in fp32 2^18.5 11.6 and 12.4, 2^20 26.4 and
// 25.7. Q's and K's heads go to fours each for itself, and the places of a four
// that no head takes cost as much as heads: at 2^20 threads 1 + 1 heads 19.9 us
// with one and 31.1 with four, 4 + 1 20.0 and 21.1, 6 + 2 19.8 and 20.5, 8 + 1
// 20.2 and 19.2. So four where there are at most 4 / 3 places a head.
constexpr int kHeads = 4;
template <typename T, int TL>
static cudaError_t launch_t(const mj_qk_norm_rope_args& a, bool vec, cudaStream_t stream) {
  if constexpr (TL < 5) {
    if (a.head_size > 16 << TL) return launch_t<T, TL + 1>(a, vec, stream);
  }
  const int64_t cs = a.cos_sin_dtype == MJ_DT_FP32 ? 4 : 2;
  vec = vec && (uintptr_t)a.q_weight % 16 == 0 && (uintptr_t)a.k_weight % 16 == 0 && (uintptr_t)a.cos_sin % 16 == 0 &&
        a.cos_sin_stride * cs % 16 == 0;
  auto grid = [&](int hg) {
    const int64_t units = a.num_tokens * ((a.h_q + hg - 1) / hg + (a.h_k + hg - 1) / hg);
    return dim3((unsigned)(((units << TL) + 127) / 128));
  };
  const float inv_d = 1.f / (float)a.head_size;
  if (!vec) return launch_kernel(qk_norm_rope_kernel<T, 1, false, TL>, grid(1), dim3(128), 0, stream, a, inv_d);
  const int64_t heads = (int64_t)a.h_q + a.h_k, places = kHeads * (((int64_t)a.h_q + kHeads - 1) / kHeads + ((int64_t)a.h_k + kHeads - 1) / kHeads);
  if ((a.num_tokens * heads << TL) >= (int64_t)1 << (sizeof(T) == 4 ? 19 : 18) && 3 * places <= 4 * heads)
    return launch_kernel(qk_norm_rope_kernel<T, kHeads, true, TL>, grid(kHeads), dim3(128), 0, stream, a, inv_d);
  return launch_kernel(qk_norm_rope_kernel<T, 1, true, TL>, grid(1), dim3(128), 0, stream, a, inv_d);
}

cudaError_t launch_qk_norm_rope(const mj_qk_norm_rope_args& a, bool vec, cudaStream_t stream) {
  if (a.dtype == MJ_DT_FP32) return launch_t<float, 0>(a, vec, stream);
  if (a.dtype == MJ_DT_FP16) return launch_t<__half, 0>(a, vec, stream);
  return launch_t<__nv_bfloat16, 0>(a, vec, stream);
}

}  // namespace mj
