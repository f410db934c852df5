// Tokens of least weight dropped from a block-scaled cache, the others moved
// together in the sequence's own pages.
//
// A cluster of CTAs takes one (sequence, KV head).
// 1. The m-th largest weight (m = budget - recent) by radix selection: weights
//    as unsigned keys of the same order, three passes over 11, 11 and 10 of
//    their bits, each a histogram of the keys that agree so far. Every CTA adds
//    up the cluster's histograms for itself, in vectors.
// 2. The kept tokens in order: those above that key, the first of those equal
//    to it, the recent ones. A CTA takes a contiguous part of the tokens, a warp
//    a contiguous part of that; what the parts before it keep is summed over the
//    block, then over the cluster.
// 3. The rows move. Position i receives token kept[i] >= i, so a step that
//    reads all its tokens before it writes, and steps in ascending order, work
//    in place: rows from i on are not read by the steps before. A step is 128
//    positions a CTA, whole blocks of scales; the cluster's barrier lies
//    between its reads and its writes, and the next step's reads (of rows that
//    this one's writes are below) are on their way into registers meanwhile.
//
// What bounds it: latency. Every pass of the selection and every step of the move
// waits for memory or for the cluster, and there are few of either a CTA. 4
// sequences of 1.1K tokens cut to 1K, 8 KV heads of 128: 13.4 us, 8.7 MB; 16 of 8K
// cut to 2K: 48.3 us, 2.9 TB/s of what has to move; one of 60K cut to 8K 42.5 us.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "block_cache.cuh"

namespace mj {

std::mutex& tc_init_mutex();

namespace cg = cooperative_groups;
using namespace sm100;

namespace ev {

constexpr int STEP = 128;   // positions of a CTA's step
constexpr int AHEAD = 8;    // steps whose positions are looked up together
constexpr int BINS = 2048;  // of a radix pass
constexpr int KEYS = 8192;  // tokens whose keys fit a CTA's shared memory

// Weights in their order as unsigned keys; -0 is 0, NaN above all.
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 0xFFFFFFFFu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int D>
struct Cfg {
  static constexpr int THREADS = D == 256 ? 1024 : 512, WARPS = THREADS / 32;  // a thread has four 16-byte chunks of a step
  struct Smem {
    // of the positions looked up, by side: the rows that they come from and go to
    const unsigned char* src[2][AHEAD * STEP];
    unsigned char* dst[2][AHEAD * STEP];
    unsigned char* scale[2][AHEAD * STEP / 16];  // destinations' exponent bytes, by 16 positions
    float w[AHEAD * STEP];
    unsigned char e[2][AHEAD * STEP];            // exponent bytes of the sources
    uint32_t f[2][STEP];                         // a step's two factors of a row, as f16
    int hist[3][BINS];                           // of the passes
    uint32_t key[KEYS];
    int amax[3][2][STEP / 16];                   // [step % 3][side][block]: largest magnitude of its rows, as bits
    int scan[WARPS];
    int pick[2];                                 // a pass's bin, and how many are above it
    int parts[2];                                // this CTA's tokens above the threshold, and equal to it
  };
};

// Sums over the warps before this one of a value that is the same in a warp's
// lanes; `total` over all.
template <int WARPS>
__device__ __forceinline__ int warps_before(int v, int* scan, int& total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  __syncthreads();  // scan's last readers are done
  if (lane == 0) scan[wid] = v;
  __syncthreads();
  int x = lane < WARPS ? scan[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  total = __shfl_sync(0xffffffffu, x, 31);
  const int below = __shfl_sync(0xffffffffu, x, wid ? wid - 1 : 0);
  return wid ? below : 0;
}

// the largest magnitude of 16 codes, NaN left out
__device__ __forceinline__ float max_abs16(uint4 c) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  __half2 m[2];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t h = e4m3x2_to_h2((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
    const __half2 x = __habs2(*reinterpret_cast<const __half2*>(&h));
    m[i & 1] = i < 2 ? x : __hmax2(m[i & 1], x);
  }
  m[0] = __hmax2(m[0], m[1]);
  return fmaxf(fmaxf((float)m[0].x, (float)m[0].y), 0.f);
}

// 4 codes times two powers of two, as codes, in f16: there a product below 2^-21
// may round, but is 0 as a code all the same
__device__ __forceinline__ uint32_t shift4(uint32_t codes, __half2 f, __half2 g) {
  uint32_t out[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t h = e4m3x2_to_h2((uint16_t)(codes >> (16 * i)));
    const __half2 x = __hmul2(__hmul2(*reinterpret_cast<const __half2*>(&h), f), g);
    uint16_t c;
    asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(c) : "r"(*reinterpret_cast<const uint32_t*>(&x)));
    out[i] = c;
  }
  return out[0] | out[1] << 16;
}
// The cluster's barrier between a step's reads and its writes, in two halves: what
// the CTAs read before they arrive they have read before one that waited writes.
// Only a release orders reads before it; it waits for the writes of the step before
// too (16 x 8K cut to 2K 48.3 us; with a relaxed arrival, whose order nothing
// promises, 45.9).
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Keeps the computation of x >= 0 before what follows: a store that never happens.
__device__ __forceinline__ void settle(float x, int* smem) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.f32 p, %0, 0f00000000;\n\t@p st.shared.u32 [%1], 0;\n\t}" ::"f"(x), "r"(smem_addr(smem)) : "memory");
}

// 2^k for -24 <= k <= 15
__device__ __forceinline__ uint32_t h_exp2(int k) { return k < -14 ? 1u << (k + 24) : (uint32_t)(15 + k) << 10; }

// SHARE: CTAs of a cluster share a job
template <int D, bool SHARE>
__global__ void __launch_bounds__(Cfg<D>::THREADS, D == 256 ? 1 : 2)
    block_evict_kernel(const __grid_constant__ mj_block_evict_args a, int lg, uint64_t per_page) {
  constexpr int THREADS = Cfg<D>::THREADS, WARPS = Cfg<D>::WARPS;
  extern __shared__ __align__(16) unsigned char raw[];
  auto& sm = *reinterpret_cast<typename Cfg<D>::Smem*>(raw);
  auto cluster = cg::this_cluster();
  const int CL = SHARE ? (int)cluster.num_blocks() : 1, rank = SHARE ? (int)cluster.block_rank() : 0;
  const int job = blockIdx.x / CL, h = job % a.h_k, seq = job / a.h_k;
  const int t = threadIdx.x, lane = t & 31, wid = t >> 5;
  griddep_wait();
  const int L = a.seq_lens[seq], budget = a.budget;
  int32_t* kept = a.kept + ((int64_t)seq * a.h_k + h) * budget;
  const bool cut = L > budget;
  // pages that hold a token, looked at before anything is written; the same
  // answer in every CTA and for every head
  const int32_t* table = a.block_table + seq * a.block_table_stride;
  bool bad = L < 0 || L > a.weights_cols || L > (int64_t)a.block_table_cols * a.page_size;
  if (bad && t == 0 && rank == 0) flag(a.status, MJ_DEV_BAD_LENGTH);
  if (!bad && cut) {
    const int pages = (int)quotient(L - 1, per_page) + 1;
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
  // Few enough tokens, and every CTA looks through all of them: that costs less
  // than exchanging histograms (4 sequences of 1.1K tokens 14.7 us, with the
  // exchange 26.9; 16 of 8K 49.5 and 49.8).
  const bool alone = M <= KEYS;
  const int part = alone ? M : (M + CL - 1) / CL, t0 = alone ? 0 : min(rank * part, M), n = min(part, M - t0);
  const bool held = part <= KEYS;  // keys are made once
  auto key_at = [&](int i) { return held ? sm.key[i] : key_of(w[t0 + i]); };
  uint32_t prefix = 0;  // the threshold's bits so far
  int above = 0;        // keys that are larger than any with these bits
  if (m > 0) {
    for (int i = t; i < 3 * BINS / 4; i += THREADS) reinterpret_cast<int4*>(sm.hist[0])[i] = make_int4(0, 0, 0, 0);
    if (held)
#pragma unroll 8
      for (int i = t; i < n; i += THREADS) sm.key[i] = key_of(w[t0 + i]);
    __syncthreads();
    int shift = 32;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10;
      const uint32_t known = pass ? ~0u << shift : 0u;
      shift -= bits;
      int* hist = sm.hist[pass];
#pragma unroll 4
      for (int i = t; i < n; i += THREADS) {
        const uint32_t k = key_at(i);
        if ((k & known) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1u)], 1);
      }
      if (alone) __syncthreads();
      else cluster.sync();
      // four bins a thread, from the largest down; all CTAs' on their way together
      int c[4] = {0, 0, 0, 0};
      if (t < BINS / 4 && alone) {
        const int4 v = reinterpret_cast<const int4*>(hist)[BINS / 4 - 1 - t];
        c[0] = v.w, c[1] = v.z, c[2] = v.y, c[3] = v.x;
      } else if (t < BINS / 4) {
        int4 v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          v[r] = r < CL ? reinterpret_cast<const int4*>(cluster.map_shared_rank(hist, r))[BINS / 4 - 1 - t] : make_int4(0, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 8; ++r) c[0] += v[r].w, c[1] += v[r].z, c[2] += v[r].y, c[3] += v[r].x;
      }
      int total, sum = c[0] + c[1] + c[2] + c[3], before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += x;
      }
      before += warps_before<WARPS>(__shfl_sync(0xffffffffu, before, 31), sm.scan, total) - sum + above;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (before < m && before + c[i] >= m) {
          sm.pick[0] = BINS - 1 - (4 * t + i);
          sm.pick[1] = before;
        }
        before += c[i];
      }
      __syncthreads();
      prefix |= (uint32_t)sm.pick[0] << shift;
      above = sm.pick[1];
    }
  }
  const int ties = m - above;  // tokens of exactly the threshold's key to keep

  // ---- 2. the kept tokens, in order (by one that knows all: those of its own steps)
  auto mine_to_write = [&](int p) { return !alone || (p / STEP & (CL - 1)) == rank; };
  if (m > 0) {
    // a warp has consecutive tokens, [begin, end) of the part
    const int chunk = ((n + WARPS - 1) / WARPS + 31) & ~31, begin = min(wid * chunk, n), end = min(begin + chunk, n);
    int gt = 0, eq = 0;
#pragma unroll 2
    for (int i0 = begin; i0 < end; i0 += 32) {
      const uint32_t k = i0 + lane < end ? key_at(i0 + lane) : 0u;
      gt += __popc(__ballot_sync(0xffffffffu, i0 + lane < end && k > prefix));
      eq += __popc(__ballot_sync(0xffffffffu, i0 + lane < end && k == prefix));
    }
    int n_gt, n_eq;
    gt = warps_before<WARPS>(gt, sm.scan, n_gt);
    eq = warps_before<WARPS>(eq, sm.scan, n_eq);
    if (!alone) {
      if (t == 0) {
        sm.parts[0] = n_gt;
        sm.parts[1] = n_eq;
      }
      cluster.sync();
      for (int r = 0; r < rank; ++r) {
        gt += cluster.map_shared_rank(sm.parts, r)[0];
        eq += cluster.map_shared_rank(sm.parts, r)[1];
      }
    }
#pragma unroll 2
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const uint32_t k = i < end ? key_at(i) : 0u, below = (1u << lane) - 1u;
      const bool is_gt = i < end && k > prefix, is_eq = i < end && k == prefix;
      const uint32_t all_gt = __ballot_sync(0xffffffffu, is_gt), all_eq = __ballot_sync(0xffffffffu, is_eq);
      const int my_eq = eq + __popc(all_eq & below), p = gt + __popc(all_gt & below) + min(my_eq, ties);
      if ((is_gt || (is_eq && my_eq < ties)) && mine_to_write(p)) kept[p] = t0 + i;
      gt += __popc(all_gt);
      eq += __popc(all_eq);
    }
  }
  if (alone) {
    for (int i = t; i < a.recent; i += THREADS)
      if (mine_to_write(m + i)) kept[m + i] = M + i;
    __syncthreads();
  } else {
    for (int i = rank * THREADS + t; i < a.recent; i += CL * THREADS) kept[m + i] = M + i;
    cluster.sync();
  }

  // ---- 3. the rows move
  constexpr int SIDE = D / 16, CPR = 2 * SIDE;  // 16-byte chunks of a K or V row, of both
  static_assert(STEP * CPR == 4 * THREADS, "four chunks a thread");
  const int steps = (budget + STEP * CL - 1) / (STEP * CL);
  const int u = t % CPR, side = u / SIDE;  // this thread's chunk of its four rows t / CPR, + 32, + 64, + 96
  auto first_of = [&](int step) { return (step * CL + rank) * STEP; };
  // positions of the steps from `step` on: where they come from and go to, the
  // sources' exponents and weights
  auto look_up = [&](int step) {
    constexpr int N = AHEAD * STEP / THREADS;
    int p[N], src[N];
    bool in[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int x = t + i * THREADS;
      p[i] = first_of(step + x / STEP) + x % STEP;
      in[i] = step + x / STEP < steps && p[i] < budget;
      src[i] = in[i] ? kept[p[i]] : 0;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!in[i]) continue;
      const int x = t + i * THREADS, sc = (int)quotient(src[i], per_page), dc = (int)quotient(p[i], per_page);
      const int64_t s_page = table[sc], s_row = src[i] - sc * a.page_size, d_page = table[dc], d_row = p[i] - dc * a.page_size;
      sm.w[x] = w[src[i]];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int64_t sp = y ? a.v_stride_page : a.k_stride_page, sr = y ? a.v_stride_row : a.k_stride_row;
        const int64_t ssp = y ? a.vs_stride_page : a.ks_stride_page, ssb = y ? a.vs_stride_block : a.ks_stride_block;
        unsigned char* cache = static_cast<unsigned char*>(y ? a.v_cache : a.k_cache) + h * (y ? a.v_stride_head : a.k_stride_head);
        unsigned char* scales = static_cast<unsigned char*>(y ? a.v_scales : a.k_scales) + h * (y ? a.vs_stride_head : a.ks_stride_head);
        sm.src[y][x] = cache + s_page * sp + s_row * sr;
        sm.dst[y][x] = cache + d_page * sp + d_row * sr;
        sm.e[y][x] = scales[s_page * ssp + (s_row >> lg) * ssb];
        if (x % 16 == 0) sm.scale[y][x / 16] = scales + d_page * ssp + (d_row >> lg) * ssb;
      }
    }
  };
  uint4 now[4], next[4];
  auto fetch = [&](int step, uint4* v) {
    const int count = budget - first_of(step);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = t / CPR + x * (STEP / 4), at = step % AHEAD * STEP + i;
      v[x] = make_uint4(0, 0, 0, 0);
      if (step < steps && i < count) v[x] = *reinterpret_cast<const uint4*>(sm.src[side][at] + u % SIDE * 16);
    }
  };
  if (t < 3 * 2 * (STEP / 16)) sm.amax[0][0][t] = 0;
#pragma unroll 1
  for (int step = 0; step < steps; ++step) {
    if (step % AHEAD == 0) {  // (the last step has ended behind a barrier)
      look_up(step);
      __syncthreads();
      fetch(step, now);
    }
    if ((step + 1) % AHEAD) fetch(step + 1, next);
    const int count = budget - first_of(step);
    float most[4];  // of the chunks
#pragma unroll
    for (int x = 0; x < 4; ++x) most[x] = max_abs16(now[x]);
    settle((most[0] + most[1]) + (most[2] + most[3]), sm.pick);  // (behind the barrier's halves they cost 16 x 8K 2 us)
    if (SHARE) cluster_arrive();
#pragma unroll
    for (int x = 0; x < 4; ++x) {  // of the rows, then the blocks
      const int i = t / CPR + x * (STEP / 4), at = step % AHEAD * STEP + i;
#pragma unroll
      for (int o = SIDE / 2; o > 0; o >>= 1) most[x] = fmaxf(most[x], __shfl_xor_sync(0xffffffffu, most[x], o));
      if (u % SIDE == 0 && i < count) atomicMax(&sm.amax[step % 3][side][i >> lg], __float_as_int(most[x] * block_scale(sm.e[side][at])));
    }
    __syncthreads();
    if (t < 2 * (STEP / 16)) sm.amax[(step + 2) % 3][0][t] = 0;  // (read last before that barrier, and next behind another)
    if (SHARE) cluster_wait();  // every CTA of the cluster has read this step's tokens
    if (t < 2 * STEP && t % STEP < count) {  // a row's side each: its block's exponent, and its codes' way there
      const int i = t % STEP, y = t / STEP, at = step % AHEAD * STEP + i;
      const int e = block_exponent(__int_as_float(sm.amax[step % 3][y][i >> lg]));
      // from -24 down every code becomes 0; above 15 (then all are tiny) in two steps
      const int k = max(block_e(sm.e[y][at]) - e, -24);
      sm.f[y][i] = h_exp2(min(k, 15)) | h_exp2(min(max(k - 15, 0), 15)) << 16;
      if ((i & ((1 << lg) - 1)) == 0) *sm.scale[y][at / 16] = (unsigned char)e;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = t / CPR + x * (STEP / 4), at = step % AHEAD * STEP + i;
      if (i < count) {
        const uint32_t fg = sm.f[side][i];
        const __half2 f = __half2half2(__ushort_as_half((unsigned short)fg)), g = __half2half2(__ushort_as_half((unsigned short)(fg >> 16)));
        *reinterpret_cast<uint4*>(sm.dst[side][at] + u % SIDE * 16) =
            make_uint4(shift4(now[x].x, f, g), shift4(now[x].y, f, g), shift4(now[x].z, f, g), shift4(now[x].w, f, g));
      }
      now[x] = next[x];
    }
    if (t < STEP && t < count) w[first_of(step) + t] = sm.w[step % AHEAD * STEP + t];
    if ((step + 1) % AHEAD == 0) __syncthreads();  // the looked-up positions are done with
  }
  cluster.sync();  // (no CTA leaves while another reads its shared memory)
}

constexpr int kMaxDevices = 64;

template <int D>
static cudaError_t launch_t(const mj_block_evict_args& a, cudaStream_t stream) {
  constexpr int smem = (int)sizeof(typename Cfg<D>::Smem);
  static std::atomic<int> ready[kMaxDevices];  // CTAs that the device holds at once, once the kernel is prepared on it
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  int room = ready[dev].load(std::memory_order_acquire);
  if (!room) {
    std::lock_guard<std::mutex> lock(tc_init_mutex());
    int sms = 0, per_sm = 0;
    if ((e = cudaFuncSetAttribute(block_evict_kernel<D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
    if ((e = cudaFuncSetAttribute(block_evict_kernel<D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, block_evict_kernel<D, true>, Cfg<D>::THREADS, smem)) != cudaSuccess) return e;
    room = std::max(1, sms * per_sm);
    ready[dev].store(room, std::memory_order_release);
  }
  // CTAs of a cluster: as many as fill the GPU once and find work, in steps of the
  // rows that stay or segments of the weights. One sequence of 60K tokens, 8 KV
  // heads, 8K staying: 306 us with one CTA, 85 with four, 41 with eight; 16 of 8K, 2K
  // staying: 55 with one, 49 with two. Beside another on its SM a CTA looks through
  // the weights at half the speed, so there it is to save more than one step (4
  // sequences of 1.1K, 1K staying, 13.8 us with eight CTAs, 13.1 with four; of 30K
  // tokens 34 and 24).
  const int64_t jobs = (int64_t)a.num_seqs * a.h_k;
  const int one_each = room / (D == 256 ? 1 : 2);
  int cl = 1;
  while (cl < 8 && 2 * cl * jobs <= room && ((2 * cl * jobs <= one_each ? cl : 2 * cl) * STEP < a.budget || (int64_t)cl * KEYS < a.weights_cols)) cl *= 2;
  auto kern = cl > 1 ? block_evict_kernel<D, true> : block_evict_kernel<D, false>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(jobs * cl));
  cfg.blockDim = dim3(Cfg<D>::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cl;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, a, block_log2(a.kv_format), reciprocal(a.page_size));
}

}  // namespace ev

cudaError_t launch_block_evict(const mj_block_evict_args& a, cudaStream_t stream) {
  return a.head_size == 256 ? ev::launch_t<256>(a, stream) : ev::launch_t<128>(a, stream);
}

}  // namespace mj
