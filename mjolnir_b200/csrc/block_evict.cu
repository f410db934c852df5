// Tokens of least weight dropped from a block-scaled cache, the others moved
// together in the sequence's own pages.
//
// A cluster of CTAs takes one (sequence, KV head).
// 1. The m-th largest weight (m = budget - recent) by radix selection: weights
//    as unsigned keys of the same order, three passes over 11, 11 and 10 of
//    their bits, each a histogram of the keys that agree so far.
// 2. The kept tokens in order: those above that key, the first of those equal
//    to it, the recent ones. A CTA takes a contiguous part of the tokens; what
//    the parts before it keep is summed over the cluster.
// 3. The rows move. Position i receives token kept[i] >= i, so a step that
//    reads all its tokens before it writes, and steps in ascending order, work
//    in place: rows from i on are not read by the steps before. A step is 128
//    positions a CTA, whole blocks of scales; the cluster's barrier lies
//    between its reads and its writes, and the next step's reads (of rows that
//    this one's writes are below) are on their way meanwhile.
#include <cooperative_groups.h>
#include <math.h>

#include "block_cache.cuh"

namespace mj {

namespace cg = cooperative_groups;
using namespace sm100;

namespace ev {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int STEP = 128;    // positions of a CTA's step
constexpr int BINS = 2048;   // of a radix pass

__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Weights in their order as unsigned keys; -0 is 0, NaN above all.
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 0xFFFFFFFFu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int D>
struct Smem {
  unsigned char rows[2][STEP][2 * D];  // a step's K | V rows
  float w[2][STEP];
  unsigned char e[2][2][STEP];         // [buffer][side]: their exponent bytes
  int hist[BINS];
  int e_new[2][STEP / 16];             // [side][block]
  int scan[WARPS + 1];
  int pick[2];                         // a radix pass's bin, and how many are above it
  int parts[2];                        // this CTA's tokens above the threshold, and equal to it
  int bad;
};

// Inclusive sums over the block; `total` of all of them.
__device__ __forceinline__ int block_scan(int v, int* scan, int& total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  __syncthreads();  // scan's last readers are done
  if (lane == 31) scan[wid] = v;
  __syncthreads();
  int below = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    const int x = scan[i];
    below += i < wid ? x : 0;
    total += x;
  }
  return v + below;
}

template <int D>
__global__ void __launch_bounds__(THREADS) block_evict_kernel(const __grid_constant__ mj_block_evict_args a, int lg) {
  extern __shared__ __align__(16) unsigned char raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>(raw);
  auto cluster = cg::this_cluster();
  const int CL = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int job = blockIdx.x / CL, h = job % a.h_k, seq = job / a.h_k;
  const int t = threadIdx.x, lane = t & 31, wid = t >> 5;
  griddep_wait();
  const int L = a.seq_lens[seq], budget = a.budget;
  int32_t* kept = a.kept + ((int64_t)seq * a.h_k + h) * budget;
  const bool cut = L > budget;
  const int64_t G = 1 << lg;
  // pages that hold a token, looked at before anything is written; the same
  // answer in every CTA and for every head
  const int32_t* table = a.block_table + seq * a.block_table_stride;
  bool bad = L < 0 || L > a.weights_cols || L > (int64_t)a.block_table_cols * a.page_size;
  if (bad && t == 0 && rank == 0) flag(a.status, MJ_DEV_BAD_LENGTH);
  if (!bad && cut) {
    const int pages = (int)((L + (int64_t)a.page_size - 1) / a.page_size);
    int missing = 0;
    for (int i = t; i < pages; i += THREADS) missing |= (unsigned)table[i] >= (uint64_t)a.num_pages;
    bad = __syncthreads_or(missing);
    if (bad && t == 0 && rank == 0) flag(a.status, MJ_DEV_BAD_PAGE);
  }
  if (h == 0 && rank == 0 && t == 0) a.new_lens[seq] = bad ? L : min(L, budget);
  if (bad || !cut) {  // the whole cluster
    for (int i = rank * THREADS + t; i < budget; i += CL * THREADS) kept[i] = !bad && i < L ? i : -1;
    return;
  }
  if (budget == 0) return;
  float* w = a.weights + seq * a.w_stride_seq + h * a.w_stride_head;

  // ---- 1. the threshold
  const int M = L - a.recent, m = budget - a.recent;  // 0 <= m < M
  const int part = (M + CL - 1) / CL, t0 = min(rank * part, M), t1 = min(t0 + part, M);
  uint32_t prefix = 0;  // the threshold's bits so far
  int above = 0;        // keys that are larger than any with these bits
  if (m > 0) {
    int shift = 32;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10;
      const uint32_t known = pass ? ~0u << shift : 0u;
      shift -= bits;
      for (int i = t; i < BINS; i += THREADS) sm.hist[i] = 0;
      __syncthreads();
      for (int i = t0 + t; i < t1; i += THREADS) {
        const uint32_t k = key_of(w[i]);
        if ((k & known) == prefix) atomicAdd(&sm.hist[(k >> shift) & ((1u << bits) - 1u)], 1);
      }
      cluster.sync();
      // four bins a thread, from the largest down
      int c[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = 0;
        for (int r = 0; r < CL; ++r) c[i] += cluster.map_shared_rank(sm.hist, r)[BINS - 1 - (4 * t + i)];
        sum += c[i];
      }
      int total;
      int before = block_scan(sum, sm.scan, total) - sum + above;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < m && before + c[i] >= m) {
          sm.pick[0] = BINS - 1 - (4 * t + i);
          sm.pick[1] = before;
        }
        before += c[i];
      }
      cluster.sync();  // histograms are read, the pick is written
      prefix |= (uint32_t)sm.pick[0] << shift;
      above = sm.pick[1];
      __syncthreads();
    }
  }
  const int ties = m - above;  // tokens of exactly the threshold's key to keep

  // ---- 2. the kept tokens, in order
  if (m > 0) {
    int gt = 0, eq = 0;
    for (int i = t0 + t; i < t1; i += THREADS) {
      const uint32_t k = key_of(w[i]);
      gt += k > prefix;
      eq += k == prefix;
    }
    int n_gt, n_eq;
    block_scan(gt, sm.scan, n_gt);
    block_scan(eq, sm.scan, n_eq);
    if (t == 0) {
      sm.parts[0] = n_gt;
      sm.parts[1] = n_eq;
    }
    cluster.sync();
    int base_gt = 0, base_eq = 0;
    for (int r = 0; r < rank; ++r) {
      base_gt += cluster.map_shared_rank(sm.parts, r)[0];
      base_eq += cluster.map_shared_rank(sm.parts, r)[1];
    }
    for (int i0 = t0; i0 < t1; i0 += THREADS) {
      const int i = i0 + t;
      const uint32_t k = i < t1 ? key_of(w[i]) : 0u;
      const int is_gt = i < t1 && k > prefix, is_eq = i < t1 && k == prefix;
      int s_gt, s_eq;
      const int up_gt = block_scan(is_gt, sm.scan, s_gt) + base_gt, up_eq = block_scan(is_eq, sm.scan, s_eq) + base_eq;
      if (is_gt || (is_eq && up_eq <= ties)) kept[up_gt + min(up_eq, ties) - 1] = i;
      base_gt += s_gt;
      base_eq += s_eq;
    }
  }
  for (int i = rank * THREADS + t; i < a.recent; i += CL * THREADS) kept[m + i] = M + i;
  cluster.sync();

  // ---- 3. the rows move
  constexpr int CPR = 2 * D / 16;  // 16-byte chunks of a K | V row
  const int steps = (budget + STEP * CL - 1) / (STEP * CL);
  auto fetch = [&](int step) {
    const int p0 = (step * CL + rank) * STEP, b = step & 1, count = min(max(budget - p0, 0), STEP);
    for (int c = t; c < count * CPR; c += THREADS) {
      const int i = c / CPR, u = c % CPR, src = kept[p0 + i], row = src % a.page_size, side = u >= CPR / 2;
      const int page = table[src / a.page_size];
      const unsigned char* from = side ? static_cast<const unsigned char*>(a.v_cache) + page * a.v_stride_page + row * a.v_stride_row + h * a.v_stride_head
                                       : static_cast<const unsigned char*>(a.k_cache) + page * a.k_stride_page + row * a.k_stride_row + h * a.k_stride_head;
      cp_async16(&sm.rows[b][i][u * 16], from + (u % (CPR / 2)) * 16);
      if (u % (CPR / 2) == 0)
        sm.e[b][side][i] = side ? static_cast<const unsigned char*>(a.v_scales)[page * a.vs_stride_page + (row >> lg) * a.vs_stride_block + h * a.vs_stride_head]
                                : static_cast<const unsigned char*>(a.k_scales)[page * a.ks_stride_page + (row >> lg) * a.ks_stride_block + h * a.ks_stride_head];
      if (u == 0) sm.w[b][i] = w[src];
    }
    cp_async_commit();
  };
  fetch(0);
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    const int p0 = (step * CL + rank) * STEP, b = step & 1, count = min(max(budget - p0, 0), STEP);
    if (step + 1 < steps) fetch(step + 1);
    else cp_async_commit();
    cp_async_wait<1>();
    __syncthreads();
    // a block's exponent: the largest finite magnitude of its rows times their scales, by a warp per (side, block)
    const int blocks = (int)((count + G - 1) >> lg);
    for (int x = wid; x < 2 * blocks; x += WARPS) {
      const int side = x / blocks, blk = x % blocks, r1 = min((blk + 1) << lg, count);
      float amax = 0.f;
      for (int c = lane; c < (r1 - (blk << lg)) * (D / 16); c += 32) {
        const int i = (blk << lg) + c / (D / 16);
        const uint4 q = *reinterpret_cast<const uint4*>(&sm.rows[b][i][side * D + (c % (D / 16)) * 16]);
        const uint32_t v[4] = {q.x, q.y, q.z, q.w};
        uint32_t most = 0;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const uint32_t mag = v[k >> 2] >> (8 * (k & 3)) & 0x7Fu;
          most = mag == 0x7Fu ? most : max(most, mag);
        }
        amax = fmaxf(amax, e4m3x2_to_f2((uint16_t)most).x * block_scale(sm.e[b][side][i]));
      }
      amax = warp_allmax(amax);
      if (lane == 0) sm.e_new[side][blk] = block_exponent(amax);
    }
    cluster.sync();  // every CTA of the cluster has read this step's tokens
    for (int c = t; c < count * CPR; c += THREADS) {
      const int i = c / CPR, u = c % CPR, pos = p0 + i, row = pos % a.page_size, side = u >= CPR / 2;
      const int page = table[pos / a.page_size], e = sm.e_new[side][i >> lg];
      const float f = __uint_as_float((uint32_t)(127 + block_e(sm.e[b][side][i]) - e) << 23);
      uint4 q = *reinterpret_cast<const uint4*>(&sm.rows[b][i][u * 16]);
      q = make_uint4(scale4(q.x, f), scale4(q.y, f), scale4(q.z, f), scale4(q.w, f));
      unsigned char* to = side ? static_cast<unsigned char*>(a.v_cache) + page * a.v_stride_page + row * a.v_stride_row + h * a.v_stride_head
                               : static_cast<unsigned char*>(a.k_cache) + page * a.k_stride_page + row * a.k_stride_row + h * a.k_stride_head;
      *reinterpret_cast<uint4*>(to + (u % (CPR / 2)) * 16) = q;
      if (u % (CPR / 2) == 0 && (i & (G - 1)) == 0) {
        if (side) static_cast<unsigned char*>(a.v_scales)[page * a.vs_stride_page + (row >> lg) * a.vs_stride_block + h * a.vs_stride_head] = (unsigned char)e;
        else static_cast<unsigned char*>(a.k_scales)[page * a.ks_stride_page + (row >> lg) * a.ks_stride_block + h * a.ks_stride_head] = (unsigned char)e;
      }
      if (u == 0) w[pos] = sm.w[b][i];
    }
    __syncthreads();  // this step's buffers are free
  }
  cluster.sync();  // (no CTA leaves while another reads its shared memory)
}

template <int D>
static cudaError_t launch_t(const mj_block_evict_args& a, cudaStream_t stream) {
  auto kern = block_evict_kernel<D>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Smem<D>));
  if (e != cudaSuccess) return e;
  int cl = 1;
  while (cl < 8 && a.num_seqs * a.h_k * cl < 296 && cl * STEP < a.budget) cl *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.num_seqs * a.h_k * cl));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = sizeof(Smem<D>);
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cl;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, a, block_log2(a.kv_format));
}

}  // namespace ev

cudaError_t launch_block_evict(const mj_block_evict_args& a, cudaStream_t stream) {
  return a.head_size == 256 ? ev::launch_t<256>(a, stream) : ev::launch_t<128>(a, stream);
}

}  // namespace mj
