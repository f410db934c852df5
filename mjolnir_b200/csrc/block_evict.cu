// Tokens of least weight dropped from a block-scaled cache, the others moved
// together in the sequence's own pages.
//
// A cluster of CTAs takes one (sequence, KV head).
// 1. The m-th largest weight (m = budget - recent) by radix selection: weights
//    as unsigned keys of the same order, three passes over 11, 11 and 10 of
//    their bits, each a histogram of the keys that agree so far. Every CTA adds
//    up the cluster's histograms for itself, in vectors.
// 2. The kept tokens in order: those above that key, the first of those equal
//    to it, the recent ones. A CTA takes a contiguous part of the tokens, a
//    thread a contiguous part of that; what the parts before it keep is summed
//    over the block, then over the cluster.
// 3. The rows move. Position i receives token kept[i] >= i, so a step that
//    reads all its tokens before it writes, and steps in ascending order, work
//    in place: rows from i on are not read by the steps before. A step is 128
//    positions a CTA, whole blocks of scales; the cluster's barrier lies
//    between its reads and its writes, and the next step's reads (of rows that
//    this one's writes are below) are on their way into registers meanwhile.
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
constexpr int PER = 8;      // tokens of a thread in a segment of the selection

// Weights in their order as unsigned keys; -0 is 0, NaN above all.
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);
  if (w != w) return 0xFFFFFFFFu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A position's source and destination: page and row of each
struct Move {
  int src_page, src_row, dst_page, dst_row;
};

template <int D>
struct Cfg {
  static constexpr int THREADS = D == 256 ? 1024 : 512, WARPS = THREADS / 32;  // a thread has four 16-byte chunks of a step
  struct Smem {
    Move moves[AHEAD * STEP];
    float w[AHEAD * STEP];
    unsigned char e[2][AHEAD * STEP];  // [side]: exponent bytes of the sources
    int hist[3][BINS];                 // of the passes
    int amax[3][2][STEP / 16];         // [step % 3][side][block]: largest magnitude of its rows, as bits
    int scan[WARPS + 1];
    int pick[2];                       // a pass's bin, and how many are above it
    int parts[2];                      // this CTA's tokens above the threshold, and equal to it
  };
};

// Inclusive sums over the block; `total` of all of them.
template <int WARPS>
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
  int x = lane < WARPS ? scan[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  total = __shfl_sync(0xffffffffu, x, 31);
  const int below = __shfl_sync(0xffffffffu, x, wid ? wid - 1 : 0);
  return v + (wid ? below : 0);
}

// the largest magnitude code of 16, NaN left out
__device__ __forceinline__ uint32_t max_code(uint4 c) {
  drop_nan_codes(c);
  uint32_t m = __vmaxu4(__vmaxu4(c.x & 0x7F7F7F7Fu, c.y & 0x7F7F7F7Fu), __vmaxu4(c.z & 0x7F7F7F7Fu, c.w & 0x7F7F7F7Fu));
  m = __vmaxu4(m, m >> 16);
  return max(m & 0xFFu, m >> 8 & 0xFFu);
}

template <int D>
__global__ void __launch_bounds__(Cfg<D>::THREADS, D == 256 ? 1 : 2)
    block_evict_kernel(const __grid_constant__ mj_block_evict_args a, int lg, uint64_t per_page) {
  constexpr int THREADS = Cfg<D>::THREADS, WARPS = Cfg<D>::WARPS, SEG = PER * THREADS;
  extern __shared__ __align__(16) unsigned char raw[];
  auto& sm = *reinterpret_cast<typename Cfg<D>::Smem*>(raw);
  auto cluster = cg::this_cluster();
  const int CL = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int job = blockIdx.x / CL, h = job % a.h_k, seq = job / a.h_k;
  const int t = threadIdx.x;
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
  const int part = (M + CL - 1) / CL, t0 = min(rank * part, M), t1 = min(t0 + part, M);
  // this thread's tokens of the segment that begins at s0; of a part of one
  // segment they stay in registers for all passes
  uint32_t key[PER];
  const int per = min((part + THREADS - 1) / THREADS, PER), seg = per * THREADS;
  auto load_keys = [&](int s0) {
#pragma unroll
    for (int x = 0; x < PER; ++x) {
      const int i = s0 + t * per + x;
      key[x] = x < per && i < t1 ? key_of(w[i]) : 0u;
    }
  };
  // tokens of them that are there
  auto count_of = [&](int s0) { return min(max(t1 - s0 - t * per, 0), per); };
  uint32_t prefix = 0;  // the threshold's bits so far
  int above = 0;        // keys that are larger than any with these bits
  if (m > 0) {
    for (int i = t; i < 3 * BINS; i += THREADS) sm.hist[0][i] = 0;
    load_keys(t0);
    __syncthreads();
    int shift = 32;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int bits = pass < 2 ? 11 : 10;
      const uint32_t known = pass ? ~0u << shift : 0u;
      shift -= bits;
      int* hist = sm.hist[pass];
      for (int s0 = t0; s0 < t1; s0 += seg) {
        if (part > seg) load_keys(s0);
        const int n = count_of(s0);
#pragma unroll
        for (int x = 0; x < PER; ++x)
          if (x < n && (key[x] & known) == prefix) atomicAdd(&hist[(key[x] >> shift) & ((1u << bits) - 1u)], 1);
      }
      cluster.sync();
      // four bins a thread, from the largest down; all CTAs' on their way together
      int c[4] = {0, 0, 0, 0};
      if (t < BINS / 4) {
        int4 v[8];
#pragma unroll
        for (int r = 0; r < 8; ++r)
          v[r] = r < CL ? reinterpret_cast<const int4*>(cluster.map_shared_rank(hist, r))[BINS / 4 - 1 - t] : make_int4(0, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 8; ++r) c[0] += v[r].w, c[1] += v[r].z, c[2] += v[r].y, c[3] += v[r].x;
      }
      int total;
      const int sum = c[0] + c[1] + c[2] + c[3];
      int before = block_scan<WARPS>(sum, sm.scan, total) - sum + above;
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

  // ---- 2. the kept tokens, in order
  if (m > 0) {
    auto tally = [&](int s0) {  // above the threshold in the low half, equal to it in the high half
      const int n = count_of(s0);
      int v = 0;
#pragma unroll
      for (int x = 0; x < PER; ++x) v += x < n ? (key[x] > prefix) + ((key[x] == prefix) << 16) : 0;
      return v;
    };
    int n_gt = 0, n_eq = 0, mine = 0, incl = 0;
    for (int s0 = t0; s0 < t1; s0 += seg) {
      if (part > seg) load_keys(s0);
      int total;
      mine = tally(s0);
      incl = block_scan<WARPS>(mine, sm.scan, total);
      n_gt += total & 0xFFFF;
      n_eq += total >> 16;
    }
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
    for (int s0 = t0; s0 < t1; s0 += seg) {
      if (part > seg) {
        int total;
        load_keys(s0);
        mine = tally(s0);
        incl = block_scan<WARPS>(mine, sm.scan, total);
        n_gt = total & 0xFFFF;
        n_eq = total >> 16;
      }
      const int n = count_of(s0);
      int gt = base_gt + (incl & 0xFFFF) - (mine & 0xFFFF), eq = base_eq + (incl >> 16) - (mine >> 16);
#pragma unroll
      for (int x = 0; x < PER; ++x) {
        if (x >= n) break;
        if (key[x] > prefix || (key[x] == prefix && eq < ties)) kept[gt + min(eq, ties)] = s0 + t * per + x;
        gt += key[x] > prefix;
        eq += key[x] == prefix;
      }
      base_gt += n_gt;
      base_eq += n_eq;
    }
  }
  for (int i = rank * THREADS + t; i < a.recent; i += CL * THREADS) kept[m + i] = M + i;
  cluster.sync();

  // ---- 3. the rows move
  constexpr int SIDE = D / 16, CPR = 2 * SIDE;  // 16-byte chunks of a K or V row, of both
  static_assert(STEP * CPR == 4 * THREADS, "four chunks a thread");
  const int steps = (budget + STEP * CL - 1) / (STEP * CL);
  const int u = t % CPR, side = u / SIDE;  // this thread's chunk of its four rows t / CPR, + 32, + 64, + 96
  const int64_t sp = side ? a.v_stride_page : a.k_stride_page, sr = side ? a.v_stride_row : a.k_stride_row;
  const int64_t ssp = side ? a.vs_stride_page : a.ks_stride_page, ssb = side ? a.vs_stride_block : a.ks_stride_block;
  unsigned char* cache = static_cast<unsigned char*>(side ? a.v_cache : a.k_cache) + h * (side ? a.v_stride_head : a.k_stride_head) + u % SIDE * 16;
  unsigned char* scales = static_cast<unsigned char*>(side ? a.v_scales : a.k_scales) + h * (side ? a.vs_stride_head : a.ks_stride_head);
  auto first_of = [&](int step) { return (step * CL + rank) * STEP; };
  // positions of the steps from `step` on: where they come from and go to, the
  // sources' exponents and weights
  auto look_up = [&](int step) {
    for (int x = t; x < AHEAD * STEP; x += THREADS) {
      const int p = first_of(step + x / STEP) + x % STEP;
      if (step + x / STEP >= steps || p >= budget) break;
      const int src = kept[p], sc = (int)quotient(src, per_page), dc = (int)quotient(p, per_page);
      const Move v = {table[sc], src - sc * a.page_size, table[dc], p - dc * a.page_size};
      sm.moves[x] = v;
      sm.w[x] = w[src];
      const int b = v.src_row >> lg;
      sm.e[0][x] = static_cast<const unsigned char*>(a.k_scales)[v.src_page * a.ks_stride_page + b * a.ks_stride_block + h * a.ks_stride_head];
      sm.e[1][x] = static_cast<const unsigned char*>(a.v_scales)[v.src_page * a.vs_stride_page + b * a.vs_stride_block + h * a.vs_stride_head];
    }
  };
  uint4 now[4], next[4];
  auto fetch = [&](int step, uint4* v) {
    const int count = budget - first_of(step);
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = t / CPR + x * (STEP / 4), at = step % AHEAD * STEP + i;
      v[x] = make_uint4(0, 0, 0, 0);
      if (step < steps && i < count) v[x] = *reinterpret_cast<const uint4*>(cache + sm.moves[at].src_page * sp + sm.moves[at].src_row * sr);
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
    const int p0 = first_of(step), count = budget - p0;
#pragma unroll
    for (int x = 0; x < 4; ++x) {  // the largest magnitudes of the step's blocks: by rows, then blocks
      const int i = t / CPR + x * (STEP / 4), at = step % AHEAD * STEP + i;
      uint32_t most = max_code(now[x]);
#pragma unroll
      for (int o = SIDE / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (u % SIDE == 0 && i < count) atomicMax(&sm.amax[step % 3][side][i >> lg], __float_as_int(e4m3x2_to_f2((uint16_t)most).x * block_scale(sm.e[side][at])));
    }
    cluster.sync();  // every CTA of the cluster has read this step's tokens
    if (t < 2 * (STEP / 16)) sm.amax[(step + 2) % 3][0][t] = 0;  // (read last before that barrier, and next behind another)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int i = t / CPR + x * (STEP / 4), at = step % AHEAD * STEP + i;
      if (i < count) {
        const Move v = sm.moves[at];
        const int e = block_exponent(__int_as_float(sm.amax[step % 3][side][i >> lg]));
        const float f = __uint_as_float((uint32_t)(127 + block_e(sm.e[side][at]) - e) << 23);
        *reinterpret_cast<uint4*>(cache + v.dst_page * sp + v.dst_row * sr) =
            make_uint4(scale4(now[x].x, f), scale4(now[x].y, f), scale4(now[x].z, f), scale4(now[x].w, f));
        if (u % SIDE == 0 && (i & ((1 << lg) - 1)) == 0) scales[v.dst_page * ssp + (v.dst_row >> lg) * ssb] = (unsigned char)e;
      }
      now[x] = next[x];
    }
    if (t < STEP && t < count) w[p0 + t] = sm.w[step % AHEAD * STEP + t];
    if ((step + 1) % AHEAD == 0) __syncthreads();  // the looked-up positions are done with
  }
  cluster.sync();  // (no CTA leaves while another reads its shared memory)
}

constexpr int kMaxDevices = 64;

template <int D>
static cudaError_t launch_t(const mj_block_evict_args& a, cudaStream_t stream) {
  auto kern = block_evict_kernel<D>;
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
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, Cfg<D>::THREADS, smem)) != cudaSuccess) return e;
    room = std::max(1, sms * per_sm);
    ready[dev].store(room, std::memory_order_release);
  }
  // CTAs of a cluster: as many as fill the GPU once and find work, in steps of the
  // rows that stay or segments of the weights
  const int64_t jobs = (int64_t)a.num_seqs * a.h_k;
  int cl = 1;
  while (cl < 8 && 2 * cl * jobs <= room && (cl * STEP < a.budget || (int64_t)cl * PER * Cfg<D>::THREADS < a.weights_cols)) cl *= 2;
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
