// The attention weight that each cached token receives in a step, added up per
// KV head, on the 5th-generation tensor cores (sm_100a):
// w[s][h][j] += sum over the rows (query, head of the group) that see key j of
// exp(scale q . k_j - lse).
//
// The scores are computed with the keys in the rows of the product, S^T = K Q^T:
// a lane of TMEM is a key, so a thread adds up its own key's weights in
// registers, no two threads meet, and the order of every sum is fixed: one thread
// writes an entry, once a call. A job is (sequence, KV head, tile of 128 keys): its
// K tile stays, the query rows that see it stream past in tiles of N. The block
// scales, one a key, go into the exponent with the softmax scale.
//
// Two kernels, by the rows that see a tile. Where they are many, both operands are
// 16 bits wide: Q enters as it is, by TMA, and K's e4m3 codes are converted, exactly,
// once for all rows. Where they are few, K enters as stored and Q in three e4m3
// terms: then reading K is all there is to do, and converting it cost more than
// reading it.
//
// What bounds them. Many: the exponentials, one an (row, key) pair, 16 a clock and
// SM. A prompt of 8192 tokens, 32 / 8 heads of 128, takes 333 us at 1965 MHz and 345
// to 360 at the clocks that its power leaves (275 GFLOP at 0.77 to 0.83 PFLOP/s);
// its exponentials alone are 240 us, the product 170. An eighth of them in
// arithmetic took 309 us at full clock but 346 under the power limit, and windows
// 7 % longer: not kept. Few: HBM. 32 single tokens behind 8K, 32 / 8 heads of 128 (192 MB),
// 37 us, 5.1 TB/s; head size 256, 16 behind 8K, 23 us, 4.1 TB/s; four behind 1000
// tokens 6.9 us, which is one job's latency.
//
// Jobs need no plan: one warp of each CTA walks the sequences' lengths on the
// device, so a captured graph replays for whatever they hold. Persistent CTAs
// take the jobs in rounds, every other round in reverse: a prompt's first keys
// are seen by all its rows, its last by few. Where there are too few jobs, the CTAs
// of a cluster share the rows of one and its first CTA adds up their sums, in order.
//
// Warp roles: 0 K (page walk, TMA, block scales), 1 Q (TMA; of few rows their
// terms), 2 MMA, 3 the jobs; then, of many rows, a warpgroup that converts K's
// codes, and those that take the S tiles in turn and add up. Every mbarrier wait
// is bounded; on a timeout the CTA flags MJ_DEV_TIMEOUT, all roles stop, copies and
// MMAs in flight complete and TMEM is freed.
#include <limits.h>
#include <math.h>

#include <atomic>
#include <mutex>
#include <type_traits>

#include <cuda.h>

#include "block_cache.cuh"

namespace mj {

std::mutex& tc_init_mutex();
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn tensor_map_encoder();

namespace bw {

using namespace sm100;

constexpr uint64_t kWaitNs = 500000000ull;  // per wait; a tile takes microseconds
constexpr float kLog2e = 1.4426950408889634f;
constexpr int KEYS = 128;

// What a role needs to know of a job. The K warp adds the scales.
struct Job {
  int seq, h, kt, nk, L, n, q0;  // seq < 0: no more; nk tiles of keys from kt on
  int t0[4], tiles[4];           // of each: the first query that counts and sees one of them, tiles of rows from it on
  int one;                       // they have one tile of rows, the same
  int parts;                     // CTAs of a cluster that share the job: of its tiles of rows, CTA r has r, r + parts, ... (`tiles`
                                 // counts each CTA's; those of some may lie behind the last row)
  float scale[4 * (KEYS / 16)];
};

// What the roles of a CTA share: its jobs and its waits.
template <int JOBS_>
struct Cta {
  static constexpr int JOBS = JOBS_;
  static_assert(JOBS >= 3, "the K warp looks two jobs ahead");
  const mj_block_weigh_args& a;
  Job* jobs;
  uint64_t *j_full, *j_empty;
  volatile int* abort_flag;
  int* never_abort;
  int lane;
  __device__ __forceinline__ bool wait(uint64_t* bar, int phase) const {
    if (mbar_wait(bar, (uint32_t)phase & 1u, abort_flag, kWaitNs)) return true;
    if (!*abort_flag) {
      *abort_flag = 1;
      flag(a.status, MJ_DEV_TIMEOUT);
    }
    return false;
  }
  // whole warps: every lane leaves with its warp
  __device__ __forceinline__ bool wait_warp(uint64_t* bar, int phase) const { return __all_sync(0xffffffffu, wait(bar, phase)) != 0; }
  // job i of this CTA, once it is there; false at the end
  __device__ __forceinline__ bool next_job(int i) const { return wait_warp(&j_full[i % JOBS], i / JOBS) && jobs[i % JOBS].seq >= 0; }
  __device__ __forceinline__ void done_job(int i) const {
    __syncwarp();
    if (lane == 0) mbar_arrive(&j_empty[i % JOBS]);
  }
  // copies in flight land: the last `stages` of `count`
  __device__ __forceinline__ void drain(uint64_t* full, int stages, int count) const {
    for (int x = max(count - stages, 0); x < count; ++x) mbar_wait(&full[x % stages], (x / stages) & 1, never_abort, kWaitNs);
  }
};

// The sequences that a launch takes: those with lo to hi queries that count. Of
// two launches the second begins while the first runs, which let it once all that
// both read was there; it waits for the first before it ends, for whatever follows
// waits for the second alone. No two sequences share a weight.
struct Take {
  int lo, hi;
  bool both;
};

// A sequence that the call complains of: n queries from q0 on, L tokens.
__device__ __forceinline__ bool out_of_range(const mj_block_weigh_args& a, int q0, int n, int L) {
  const int64_t room = (int64_t)a.block_table_cols * a.page_size;
  return (q0 < 0) | (n < 0) | (q0 + (int64_t)n > a.num_rows) | (L < 0) | (L > a.weights_cols) | (L > room) | (L > INT_MAX - 8 * KEYS);
}

// Of two launches, one that has none leaves before it takes anything; the first
// stays where there is something to complain of.
__device__ __forceinline__ bool has_any(const mj_block_weigh_args& a, Take take, bool first) {
  int any = 0;
  for (int s = threadIdx.x; s < a.num_seqs; s += blockDim.x) {
    const int q0 = a.offsets[s], n = a.offsets[s + 1] - q0, L = first ? a.seq_lens[s] : 0, m = a.window && a.window < n ? a.window : n;
    any |= (m >= take.lo && m <= take.hi) | (first && out_of_range(a, q0, n, L));  // (the loads wait once)
  }
  return __syncthreads_or(any) != 0;
}

// The warp that finds the CTA's jobs: up to TILES tiles of keys of one KV head.
// 32 sequences at a time, lane i has the key tiles of sequence s0 + i. The CTAs of
// a cluster take their own jobs, or share one where there are too few.
template <int TILES, bool SHARE, class C>
__device__ __forceinline__ void find_jobs(const C& cta, Take take, int tb, int ht, int cluster) {
  const mj_block_weigh_args& a = cta.a;
  const int lane = cta.lane;
  int L = 0, n = 0, q0 = 0;
  auto tiles_of = [&](int s, bool complain) {
    if (s >= a.num_seqs) return 0;
    q0 = a.offsets[s];
    n = a.offsets[s + 1] - q0;
    L = a.seq_lens[s];
    if (out_of_range(a, q0, n, L)) {
      if (complain) flag(a.status, MJ_DEV_BAD_LENGTH);
      return 0;
    }
    const int m = a.window && a.window < n ? a.window : n;
    return m >= take.lo && m <= take.hi ? (L + KEYS - 1) / KEYS : 0;
  };
  // Tiles a job: as many as leave every CTA two jobs (each costs its lookups'
  // latency; a few jobs more than CTAs leave some of them idle). 32 single tokens
  // behind 8K: 59 us with one tile a job, 37 with four; four behind 1000 tokens 6.6
  // and 8.2.
  int per = 1;
  if (TILES > 1) {
    int64_t tiles = 0;
    for (int s = lane; s - lane < a.num_seqs && tiles * a.h_k < 2ll * TILES * gridDim.x; s += 32) {
      int x = tiles_of(s, false);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
      tiles += x;
    }
    while (per < TILES && tiles * a.h_k >= 4ll * per * gridDim.x) per *= 2;
  }
  int parts = 1;
  if (SHARE) {
    // What takes longer, in tiles of rows: a job as many and 3 more for its keys, a
    // shared one its share and 5 more. Jobs before the step's first tokens have all
    // its rows, the others ever fewer; a lane adds up those of one worker.
    int jobs = 0, full = 0, rows = 0;
    for (int s = lane; s - lane < a.num_seqs && jobs < 1 << 20; s += 32) {
      const int x = tiles_of(s, false);
      if (x) {
        jobs += min(x, 1 << 20);
        full += min(max(L - n, 0) / KEYS, 1 << 20);
        rows = max(rows, (min(n, a.window ? a.window : n) + tb - 1) / tb * ht);
      }
    }
    jobs = __reduce_add_sync(0xffffffffu, min(jobs, 1 << 20));
    full = __reduce_add_sync(0xffffffffu, min(full, 1 << 20));
    rows = __reduce_max_sync(0xffffffffu, rows);
    if ((int64_t)jobs * a.h_k <= 3 * (int)gridDim.x) {  // (more even out by themselves)
      jobs *= a.h_k;
      full *= a.h_k;
      const float fall = jobs > full ? 1.f / (float)(jobs - full) : 0.f;
      auto time_of = [&](int share, float more) {
        const int w = (int)gridDim.x / share, at = lane * (w - 1) / 31;
        float sum = 0.f;
        for (int r = 0; r * w < jobs; ++r) {
          const int job = r * w + (r & 1 ? w - 1 - at : at);
          if (job < jobs) sum += more + ceilf((float)rows * (job < full ? 1.f : 1.f - (float)(job - full) * fall) / (float)share);
        }
        return __reduce_max_sync(0xffffffffu, (uint32_t)sum);
      };
      if (time_of(cluster, 5.f) < time_of(1, 3.f)) parts = cluster;
    }
  }
  const int workers = (int)gridDim.x / parts, me = (int)blockIdx.x / parts;
  int s0 = -32, i = 0;
  int64_t base = 0, total = 0, before = 0, count = 0;
  for (int64_t round = 0;; ++round, ++i) {
    const int64_t p = round * workers + (round & 1 ? workers - 1 - me : me);
    bool more = true;
    while (p >= base + total) {
      base += total;
      s0 += 32;
      if (s0 >= a.num_seqs) {
        more = false;
        break;
      }
      count = (int64_t)((tiles_of(s0 + lane, true) + per - 1) / per) * a.h_k;
      before = count;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += x;
      }
      total = __shfl_sync(0xffffffffu, before, 31);
      before -= count;
    }
    if (!cta.wait_warp(&cta.j_empty[i % C::JOBS], i / C::JOBS + 1)) return;
    Job& j = cta.jobs[i % C::JOBS];
    if (!more) {
      if (lane == 0) {
        j.seq = -1;
        mbar_arrive(&cta.j_full[i % C::JOBS]);
      }
      return;
    }
    const int64_t at = p - base - before;
    if (at >= 0 && at < count) {  // one lane: groups of key tiles, and the heads of each, in turn
      const int64_t group = at >> 32 ? at / a.h_k : (uint32_t)at / (uint32_t)a.h_k;  // a 64-bit division is a long routine
      j.seq = s0 + lane;
      j.h = (int)(at - group * a.h_k);
      j.kt = (int)group * per;
      j.nk = min(per, (L + KEYS - 1) / KEYS - j.kt);
      j.L = L;
      j.n = n;
      j.q0 = q0;
      for (int x = 0; x < j.nk; ++x) {
        j.t0[x] = max(a.window ? max(n - a.window, 0) : 0, (j.kt + x) * KEYS - (L - n));
        const int tiles = (n - j.t0[x] + tb - 1) / tb * ht;
        j.tiles[x] = parts > 1 ? (tiles + parts - 1) / parts : tiles;
      }
      j.parts = parts;
      j.one = j.tiles[0] == 1 && j.t0[j.nk - 1] == j.t0[0];  // (t0 grows with x)
      mbar_arrive(&cta.j_full[i % C::JOBS]);
    }
    __syncwarp();
  }
}

// The warp that fetches K, tile by tile into a ring of RS stages, and its block
// scales into the jobs. Lane i looks up the page of the job's 16-token group i two
// jobs ahead and reads its exponent one job ahead (a use at once would wait for
// memory).
template <int D, int RS, class C>
__device__ __forceinline__ void fetch_keys(const C& cta, int lg, const CUtensorMap& tmk, unsigned char* raw, uint64_t* r_full, uint64_t* r_empty) {
  constexpr int kNone = INT_MIN, JOBS = C::JOBS;
  const mj_block_weigh_args& a = cta.a;
  const int lane = cta.lane;
  const uint64_t policy = l2_policy_evict_normal();
  const int ps = a.page_size, lps = 31 - __clz(ps), groups = max(ps / 16, 1), pages = KEYS / ps;
  auto entry_of = [&](const Job& j) {
    const int pos = j.kt * KEYS + lane * 16;
    return lane < j.nk * (KEYS / 16) && pos < j.L ? __ldg(a.block_table + j.seq * a.block_table_stride + (pos >> lps)) : kNone;
  };
  auto exponent_of = [&](const Job& j, int page) -> unsigned char {
    if (page < 0) return 127;
    const int row = (j.kt * KEYS + lane * 16) & (ps - 1);
    return __ldg(static_cast<const unsigned char*>(a.k_scales) + page * a.ks_stride_page + (row >> lg) * a.ks_stride_block + j.h * a.ks_stride_head);
  };
  auto page_of = [&](int e) {  // -1: no such token, or a bad entry
    if ((unsigned)e < (uint64_t)a.num_pages) return e;
    if (e != kNone) flag(a.status, MJ_DEV_BAD_PAGE);
    return -1;
  };
  bool here = cta.next_job(0), ahead = here && cta.next_job(1), ok = true;
  int e0 = here ? entry_of(cta.jobs[0]) : kNone, e1 = ahead ? entry_of(cta.jobs[1 % JOBS]) : kNone;
  int page = page_of(e0);
  unsigned char ex = here ? exponent_of(cta.jobs[0], page) : 127;
  int i = 0, u = 0;
  for (; ok && here; ++i) {
    Job& j = cta.jobs[i % JOBS];
    const int nk = j.nk, h = j.h;
    j.scale[lane] = block_scale(ex);
    const int page1 = page_of(e1);
    const unsigned char ex1 = ahead ? exponent_of(cta.jobs[(i + 1) % JOBS], page1) : 127;
    const bool ahead2 = ahead && cta.next_job(i + 2);
    e1 = ahead2 ? entry_of(cta.jobs[(i + 2) % JOBS]) : kNone;
    __syncwarp();  // the scales are written before lane 0 arrives
    for (int x = 0; x < nk; ++x, ++u) {
      ok = cta.wait_warp(&r_empty[u % RS], u / RS + 1);
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&r_full[u % RS], KEYS * D);
      __syncwarp();
      const int pg = __shfl_sync(0xffffffffu, page, (x * (KEYS / 16) + lane * groups) & 31);
      if (lane < pages) {
#pragma unroll
        for (int dh = 0; dh < D / 128; ++dh)  // an absent page is read out of range: zeros
          tma_load_5d(raw + (u % RS) * (KEYS * D) + dh * (KEYS * 128) + lane * ps * 128, &tmk, &r_full[u % RS], 0, dh, 0, h,
                      pg < 0 ? (int)a.num_pages : pg, policy);
      }
    }
    if (!ok) break;
    cta.done_job(i);
    page = page1;
    ex = ex1;
    here = ahead;
    ahead = ahead2;
  }
  cta.drain(r_full, RS, u);
}

// byte offset of 16-byte unit u of row r in a [rows][128 bytes] swizzled block
__device__ __forceinline__ uint32_t unit_offset(uint32_t r, uint32_t u) { return r * 128 + ((u ^ (r & 7)) << 4); }

// A key's weight, which one thread writes: a token of the step begins at 0. The
// others are added to where they are, in L2: a load would be waited for, some
// 2000 cycles a tile.
__device__ __forceinline__ void put(float* w, float sum, bool begins) {
  if (begins) *w = sum;
  else atomicAdd(w, sum);
}

// ---- what CTAs of a cluster say to one another
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// `p` of CTA `rank`'s shared memory
__device__ __forceinline__ uint32_t at_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void store_there(uint32_t at, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }
__device__ __forceinline__ void arrive_there(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// For a phase that another CTA's threads complete; bounded as mbar_wait.
__device__ __forceinline__ bool wait_others(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const uint64_t t0 = globaltimer();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_addr(bar)), "r"(parity), "r"(20000u)
        : "memory");
    if (ok) return true;
    if (*abort_flag || globaltimer() - t0 > kWaitNs) return false;
  }
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ------------------------------------------------------------- many rows a tile
template <typename T, int D, int N>
struct Cfg {
  static constexpr int RAW = KEYS * D, K16 = 2 * RAW, QST = N * D * 2;  // a tile's codes; as 16 bits; a tile of Q rows
  // Warpgroups that add up: the exponentials bound it, and two or four warps on a
  // scheduler must hide one another's latency (8192 tokens, 32 / 8 heads: 376 us
  // with two warpgroups, 341 with four).
  static constexpr int WGS = 4, THREADS = 128 * (2 + WGS);
  // stages of K codes, of K in 16 bits, of Q
  static constexpr int RS = D == 256 ? 1 : 2, KS = D == 256 ? 1 : 2, QS = D == 256 ? 2 : 3;
  static constexpr int SB = 4;  // S buffers in TMEM; a warpgroup that adds up has three of its columns' lse
  // The tensor cores cut off what a step's sum has below fp32's last place. Over
  // the 16 steps of fp16 products at head size 256 weights came out 6.6e-7 too
  // small (1.2e-6 from 64 bits, plain fp32 arithmetic 3.7e-7), so there each half of
  // the head dim has a sum of its own.
  static constexpr bool SPLIT = std::is_same<T, __half>::value && D == 256;
  static constexpr int SN = SPLIT ? 2 * N : N;
  static_assert(SB * SN <= 512, "S buffers");
  static constexpr int JOBS = 16;  // (K is fetched for jobs that far ahead: 8 sequences of 6K, 64 rows 57 us with 4, 42 with 16)
  static constexpr int PARTS = 8;  // CTAs of a cluster, at most; each but the first has a buffer in that one for each warpgroup's sums
  static constexpr int PAIRS = WGS * (WGS - 1);  // of a warpgroup that writes weights and one that adds its part
  static constexpr int K_OFF = 0, R_OFF = K_OFF + KS * K16, Q_OFF = R_OFF + RS * RAW, Z_OFF = Q_OFF + QS * QST;
  static constexpr int RED_OFF = Z_OFF + 3 * WGS * N * 4, X_OFF = RED_OFF + PAIRS * KEYS * 4;
  static constexpr int JOB_OFF = X_OFF + (PARTS - 1) * WGS * KEYS * 4, BAR_OFF = JOB_OFF + JOBS * (int)sizeof(Job);
  static constexpr int NBARS = 2 * (RS + KS + QS + SB + JOBS + PAIRS) + WGS + 1 + PARTS * WGS;
  static constexpr int MISC_OFF = BAR_OFF + NBARS * 8;
  static constexpr int SMEM = MISC_OFF + 16;
  static_assert(SMEM <= 232448, "shared memory of a CTA");
  // a buffer is always waited for by the same warpgroup, whose waits are in order:
  // another's could take an older phase of the same parity for its own
  static_assert(SB % WGS == 0, "buffers of a warpgroup");
};

// 16 codes -> 16 values of T (exact)
template <typename T>
__device__ __forceinline__ void widen16(uint4 c, uint32_t* o) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (std::is_same<T, __half>::value) {
      o[2 * k] = e4m3x2_to_h2((uint16_t)w[k]);
      o[2 * k + 1] = e4m3x2_to_h2((uint16_t)(w[k] >> 16));
    } else {
      const float2 a = e4m3x2_to_f2((uint16_t)w[k]), b = e4m3x2_to_f2((uint16_t)(w[k] >> 16));
      const __nv_bfloat162 x = __floats2bfloat162_rn(a.x, a.y), y = __floats2bfloat162_rn(b.x, b.y);
      o[2 * k] = *reinterpret_cast<const uint32_t*>(&x);
      o[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&y);
    }
  }
}

// SHARE: for clusters
template <typename T, int D, int N, bool SHARE>
__global__ void __launch_bounds__(Cfg<T, D, N>::THREADS, 1)
    block_weigh_kernel(const __grid_constant__ mj_block_weigh_args a, Take take, int cluster, int lg, int hb, int tb, int ht,
                       const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmq) {
  using C = Cfg<T, D, N>;
  constexpr int RS = C::RS, KS = C::KS, QS = C::QS, SB = C::SB, JOBS = C::JOBS, WGS = C::WGS;
  extern __shared__ __align__(1024) unsigned char sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::BAR_OFF);
  uint64_t *r_full = bars, *r_empty = r_full + RS, *k_full = r_empty + RS, *k_empty = k_full + KS, *q_full = k_empty + KS,
           *q_empty = q_full + QS, *s_full = q_empty + QS, *s_empty = s_full + SB, *j_full = s_empty + SB, *j_empty = j_full + JOBS,
           *red_full = j_empty + JOBS, *red_empty = red_full + C::PAIRS, *z_full = red_empty + C::PAIRS, *drain = z_full + WGS,
           *x_full = drain + 1, *x_empty = x_full + (C::PARTS - 1) * WGS;
  Job* jobs = reinterpret_cast<Job*>(sm + C::JOB_OFF);
  float* red = reinterpret_cast<float*>(sm + C::RED_OFF);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + C::MISC_OFF + 4);
  int& never_abort = *reinterpret_cast<int*>(sm + C::MISC_OFF + 8);
  if (reinterpret_cast<uintptr_t>(sm) & 1023) {  // uniform: nothing taken yet
    if (threadIdx.x == 0) flag(a.status, MJ_DEV_BAD_SPLIT);
    return;
  }
  griddep_wait();
  if (take.both) {
    griddep_launch_dependents();
    if (!has_any(a, take, true)) return;  // (every CTA of a cluster)
  }
  if (threadIdx.x == 0) {
    auto init = [](uint64_t* b, int n, int count) {
      for (int i = 0; i < n; ++i) mbar_init(b + i, count);
    };
    init(r_full, RS, 1);
    init(r_empty, RS, 128);
    init(k_full, KS, 128);
    init(k_empty, KS, 1);
    init(q_full, QS, 1);
    init(q_empty, QS, 1);
    init(s_full, SB, 2);  // the product, and its issuer (who saw the job's scales)
    init(s_empty, SB, 128);
    init(j_full, JOBS, 1);
    init(j_empty, JOBS, 3 + 4 * (1 + WGS));  // the K, Q and MMA warps, those that convert, those that add up
    init(red_full, C::PAIRS, 128);
    init(red_empty, C::PAIRS, 128);
    init(z_full, WGS, 128);
    init(x_full, (C::PARTS - 1) * WGS, 128);
    init(x_empty, WGS, 128);
    mbar_init(drain, 1);
    *abort_flag = 0;
    never_abort = 0;
    fence_mbar_init();
  }
  // rows of a Q stage that no box fills stay zero
  for (int i = threadIdx.x; i < QS * C::QST / 16; i += C::THREADS) reinterpret_cast<uint4*>(sm + C::Q_OFF)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmq);
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  if (SHARE) cluster_sync();  // (nobody arrives at a barrier that is not there yet)
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t rank = SHARE ? cluster_rank() : 0;
  const Cta<JOBS> cta{a, jobs, j_full, j_empty, abort_flag, &never_abort, lane};
  auto wait_warp = [&](uint64_t* bar, int phase) { return cta.wait_warp(bar, phase); };
  auto next_job = [&](int i) { return cta.next_job(i); };
  auto done_job = [&](int i) { cta.done_job(i); };

  if (warp == 3) {
    find_jobs<1, SHARE>(cta, take, tb, ht, cluster);
  } else if (warp == 0) {
    fetch_keys<D, RS>(cta, lg, tmk, sm + C::R_OFF, r_full, r_empty);
  } else if (warp == 1) {
    // ------------------------------------------------------------------------- Q
    // Column c of a tile is (token c / hb, head c % hb of the tile's).
    const uint64_t policy = l2_policy_evict_normal();
    int it = 0;
    bool ok = true;
    for (int i = 0; ok && next_job(i); ++i) {
      const Job& j = jobs[i % JOBS];
      const int h = j.h, q0 = j.q0 + j.t0[0], tiles = j.tiles[0], parts = SHARE ? j.parts : 1;
      for (int tile = 0, at = parts > 1 ? rank : 0; tile < tiles; ++tile, at += parts, ++it) {
        const int s = it % QS, tok = (ht == 1 ? at : at / ht) * tb, head = ht == 1 ? 0 : at % ht * hb;  // (rows behind the last tensor row: zeros)
        ok = wait_warp(&q_empty[s], it / QS + 1);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&q_full[s], (D / 64) * 128 * hb * tb);
        __syncwarp();
        if (lane < D / 64) tma_load_4d(sm + C::Q_OFF + s * C::QST + lane * (N * 128), &tmq, &q_full[s], lane * 64, head, h, q0 + tok, policy);
      }
      if (ok) done_job(i);
    }
    cta.drain(q_full, QS, it);
  } else if (warp == 2) {
    // ---------------------------------------------------------------------- MMA
    constexpr uint32_t idesc = std::is_same<T, __half>::value ? idesc_f16(0, 0, N) : idesc_bf16(0, 0, N);
    const bool lead = elect_one();
    int it = 0;
    bool ok = true;
    auto ready = [&]() { return wait_warp(&q_full[it % QS], it / QS) && wait_warp(&s_empty[it % SB], it / SB + 1); };  // tile `it`
    for (int i = 0; ok && next_job(i); ++i) {
      const int tiles = jobs[i % JOBS].tiles[0];
      ok = wait_warp(&k_full[i % KS], i / KS) && ready();
      const uint64_t k = smem_desc_sw128(smem_addr(sm + C::K_OFF + (i % KS) * C::K16), 16, 1024);
      for (int tile = 0; ok && tile < tiles; ++tile) {
        const int b = it % SB, s = it % QS;
        tc_fence_after();
        const uint64_t q = smem_desc_sw128(smem_addr(sm + C::Q_OFF + s * C::QST), 16, 1024);
        auto steps = [&](auto half) {  // 16 head-dim elements a step
          constexpr int H = decltype(half)::value;
          if (lead) {
#pragma unroll
            for (int y = H * (D / 32); y < (H + 1) * (D / 32); ++y)
              mma_f16(tmem + b * C::SN + (C::SPLIT ? H * N : 0), k + y / 4 * (KEYS * 8) + y % 4 * 2, q + y / 4 * (N * 8) + y % 4 * 2, idesc,
                      y > (C::SPLIT ? H * (D / 32) : 0));
          }
        };
        steps(std::integral_constant<int, 0>());
        ++it;  // the waits for the next tile pass while these products run
        if (tile + 1 < tiles) ok = ready();
        steps(std::integral_constant<int, 1>());
        if (lead) {
          mma_commit(&s_full[b]);
          mbar_arrive(&s_full[b]);
          mma_commit(&q_empty[s]);
          if (tile + 1 == tiles) mma_commit(&k_empty[i % KS]);
        }
        __syncwarp();
      }
      if (ok) done_job(i);
    }
    if (lead) mma_commit(drain);  // all issued MMAs complete before TMEM is released
    mbar_wait(drain, 0, &never_abort, kWaitNs);
  } else if (warp < 8) {
    // ------------------------------------------------------------ codes -> 16 bits
    // Thread ct takes 16-code chunk 4 blk + quad of rows r0, r0 + STEP, ...: eight
    // neighbouring threads are four chunks of a 64-element block in rows r and
    // r ^ 5, so that both their staged reads and their stores cover all banks.
    const int ct = threadIdx.x & 127;
    constexpr int BLOCKS = D / 64, STEP = 32 / BLOCKS, NC = KEYS / STEP, BATCH = 4;
    const int quad = ct & 3, blk = (ct >> 3) % BLOCKS, pr = (ct >> 3) / BLOCKS;
    const int r0 = ((pr & 3) ^ ((ct >> 2) & 1 ? 5 : 0)) + (pr & ~3) * 2;
    for (int i = 0; next_job(i); ++i) {
      if (!wait_warp(&r_full[i % RS], i / RS) || !wait_warp(&k_empty[i % KS], i / KS + 1)) break;
      const unsigned char* raw = sm + C::R_OFF + (i % RS) * C::RAW + (blk >> 1) * (KEYS * 128);
      unsigned char* out = sm + C::K_OFF + (i % KS) * C::K16 + blk * (KEYS * 128);
#pragma unroll 1
      for (int x0 = 0; x0 < NC; x0 += BATCH) {
        uint4 d[BATCH];
#pragma unroll
        for (int x = 0; x < BATCH; ++x) d[x] = *reinterpret_cast<const uint4*>(raw + unit_offset(r0 + (x0 + x) * STEP, 4 * (blk & 1) + quad));
#pragma unroll
        for (int x = 0; x < BATCH; ++x) {
          uint32_t o[8];
          widen16<T>(d[x], o);
          *reinterpret_cast<uint4*>(out + unit_offset(r0 + (x0 + x) * STEP, 2 * quad)) = make_uint4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<uint4*>(out + unit_offset(r0 + (x0 + x) * STEP, 2 * quad + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
      // the stage is free once every value read from it went through the stores above
      mbar_arrive(&r_empty[i % RS]);
      fence_proxy_async_smem();
      mbar_arrive(&k_full[i % KS]);
      done_job(i);
    }
  } else {
    // ------------------------------------------------------------------ the sums
    const int wg = (warp - 8) >> 2, t = threadIdx.x & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const int h_r = a.h_q / a.h_k;
    // The lse of this warpgroup's tiles, by buffer: a tile's are stored while the
    // one before is added up, which warps that lag behind may still be at the
    // start of; so three.
    float* const zbuf = reinterpret_cast<float*>(sm + C::Z_OFF) + wg * (3 * N);
    int z_stored = 0, z_seen = 0;
    // this thread's column: its lse in tile `tile` of the queries from t0 on
    const int z_tok = t < hb * tb ? t / hb : INT_MAX / 2, z_head = t % hb;
    int parts = 1, part0 = 0;  // of the job: its CTAs, and this one's place
    auto tok_of = [&](int t0, int tile) { return t0 + (ht == 1 ? tile * parts + part0 : (tile * parts + part0) / ht) * tb; };
    auto load_lse = [&](const Job& j, int t0, int tile) {
      const int tok = tok_of(t0, tile), head = ht == 1 ? z_head : (tile * parts + part0) % ht * hb + z_head;
      return z_tok < j.n - tok && head < h_r ? __ldg(a.lse + (int64_t)(j.q0 + tok + z_tok) * a.h_q + j.h * h_r + head) : -INFINITY;
    };
    auto store_lse = [&](float z) {
      if (t < N) zbuf[z_stored % 3 * N + t] = z == -INFINITY ? -INFINITY : -z * kLog2e;  // a row without keys adds nothing
      mbar_arrive(&z_full[wg]);
      ++z_stored;
    };
    // This key's weights of the tile in S buffer b, columns [c_lo, c_hi) of it where
    // PART: the next columns are on their way from TMEM while these are added up.
    auto add_up = [&](auto part, int b, float c2, int c_lo, int c_hi) {
      constexpr bool PART = decltype(part)::value;
      const float4* zs = reinterpret_cast<const float4*>(zbuf + (z_seen + 2) % 3 * N);
      const uint32_t s_addr = tmem + b * C::SN + lane_base;
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)}, v[2][8], more[C::SPLIT ? 8 : 1];
      tmem_ld16(s_addr, reinterpret_cast<float*>(v[0]));
#pragma unroll
      for (int c = 0; c < N; c += 16) {
        float2* const now = v[c / 16 & 1];
        if (C::SPLIT) tmem_ld16(s_addr + N + c, reinterpret_cast<float*>(more));
        tmem_wait_ld();
        if (C::SPLIT)
#pragma unroll
          for (int x = 0; x < 8; ++x) now[x] = fadd2(now[x], more[C::SPLIT ? x : 0]);
        if (c + 16 < N) tmem_ld16(s_addr + c + 16, reinterpret_cast<float*>(v[c / 16 + 1 & 1]));
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (PART && c + 4 * x >= c_hi) break;  // uniform
          const float4 z = zs[c / 4 + x];
          float2 e[2] = {ffma2(now[2 * x], make_float2(c2, c2), make_float2(z.x, z.y)),
                         ffma2(now[2 * x + 1], make_float2(c2, c2), make_float2(z.z, z.w))};
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            if (PART) {
              const int c0 = c + 4 * x + 2 * y;
              e[y].x = c0 >= c_lo && c0 < c_hi ? e[y].x : -INFINITY;
              e[y].y = c0 + 1 >= c_lo && c0 + 1 < c_hi ? e[y].y : -INFINITY;
            }
            sum[y] = fadd2(sum[y], make_float2(exp2_approx(e[y].x), exp2_approx(e[y].y)));
          }
        }
      }
      return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
    };
    int it = 0, gave[WGS] = {}, took[WGS] = {};  // tiles; parts given at each place, and taken from it
    int x_jobs = 0;                              // shared jobs whose sums came together in this warpgroup
    bool ok = true;
    for (int i = 0; ok && next_job(i); ++i) {
      const Job& j = jobs[i % JOBS];
      const int ahead = j.L - j.n, n = j.n, L = j.L, key = j.kt * KEYS + t, t0 = j.t0[0], tiles = j.tiles[0];
      if (SHARE) {
        parts = j.parts;
        part0 = parts > 1 ? rank : 0;
      }
      // The warpgroups take the tiles in turn; this one has the job's tiles
      // place, place + WGS, ... The first place writes the weights.
      const int place = (wg - it) & (WGS - 1), it0 = it;
      it += tiles;
      if (place >= tiles) {
        done_job(i);
        continue;
      }
      float* w = a.weights + j.seq * a.w_stride_seq + j.h * a.w_stride_head + key;
      float z = 0.f;
      store_lse(load_lse(j, t0, place));
      if (place + WGS < tiles) z = load_lse(j, t0, place + WGS);
      float sum = 0.f, low = 0.f, c2 = 0.f;  // the sum, and what its rounding lost
#pragma unroll 1
      for (int tile = place; tile < tiles; tile += WGS) {
        ok = wait_warp(&z_full[wg], z_seen++);
        if (tile + WGS < tiles) {  // the lse of this warpgroup's next tile, and the load of the one's behind it
          store_lse(z);
          if (tile + 2 * WGS < tiles) z = load_lse(j, t0, tile + 2 * WGS);
        }
        const int b = (it0 + tile) % SB;
        ok = ok && wait_warp(&s_full[b], (it0 + tile) / SB);
        if (!ok) break;
        tc_fence_after();
        if (tile == place) c2 = a.softmax_scale * kLog2e * j.scale[t >> 4];
        // columns of queries that are there and see the key
        const int tok = tok_of(t0, tile), c_lo = max(key - ahead - tok, 0) * hb, c_hi = min(n - tok, tb) * hb;
        const bool part = tok + tb > n || key - t + KEYS - 1 > ahead + tok;  // uniform
        const float p = (part ? add_up(std::true_type(), b, c2, c_lo, c_hi) : add_up(std::false_type(), b, c2, 0, 0)) + low, next = sum + p;
        tc_fence_before();
        mbar_arrive(&s_empty[b]);
        low = p - (next - sum);
        sum = next;
      }
      if (!ok) break;
      // the other places' parts, in their order; every pair of warpgroups has a buffer
#pragma unroll
      for (int y = 1; y < WGS; ++y) {
        if (tiles <= y || (place != 0 && place != y)) continue;
        const int pair = (place == 0 ? wg : (wg - y) & (WGS - 1)) * (WGS - 1) + y - 1;
        if (place == y) {
          ok = ok && wait_warp(&red_empty[pair], gave[y] + 1);
          if (!ok) break;
          red[pair * KEYS + t] = sum;
          mbar_arrive(&red_full[pair]);
          ++gave[y];
        } else {
          ok = ok && wait_warp(&red_full[pair], took[y]);
          if (!ok) break;
          sum += red[pair * KEYS + t];
          mbar_arrive(&red_empty[pair]);
          ++took[y];
        }
      }
      if (!ok) break;
      if (SHARE && place == 0 && parts > 1) {
        // The other CTAs' sums, in their order. All have as many tiles, so it is the
        // same warpgroup's everywhere, and each has a buffer and barriers of its own.
        auto wait_x = [&](uint64_t* bar, int phase) {
          const bool there = wait_others(bar, (uint32_t)phase & 1u, abort_flag);
          if (!there && !*abort_flag) {
            *abort_flag = 1;
            flag(a.status, MJ_DEV_TIMEOUT);
          }
          return __all_sync(0xffffffffu, there) != 0;
        };
        float* const xbuf = reinterpret_cast<float*>(sm + C::X_OFF);
        if (rank) {
          const int b = ((int)rank - 1) * WGS + wg;
          ok = wait_x(&x_empty[wg], x_jobs + 1);
          if (!ok) break;
          store_there(at_rank(xbuf + b * KEYS + t, 0), sum);
          arrive_there(at_rank(&x_full[b], 0));
        } else {
          for (int r = 1; r < parts; ++r) {
            const int b = (r - 1) * WGS + wg;
            ok = wait_x(&x_full[b], x_jobs);
            if (!ok) break;
            sum += xbuf[b * KEYS + t];
            arrive_there(at_rank(&x_empty[wg], r));
          }
          if (!ok) break;
        }
        ++x_jobs;
      }
      if (place == 0 && (!SHARE || part0 == 0) && key < L) put(w, sum, key >= ahead);
      done_job(i);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (SHARE) cluster_sync();  // no CTA leaves while another may write to its shared memory
}

// -------------------------------------------------------------- few rows a tile
// Where a step's sequences have a few rows each, K is read for little arithmetic,
// and converting it would cost more than multiplying it. So K enters the product
// as stored, and Q, once a job, as three e4m3 terms of its row scaled by a power
// of two to [128, 256): x = hi + mid / 16 + lo / 256, in steps of 2^-17 at least. So
// bf16 elements (8 bits) are exact down to 2^-17 of the row's largest, fp16 ones (11)
// down to 2^-14, and what is below is off by 2^-25 of the largest at most. The terms
// are columns of their own, joined in fp32. Several CTAs an SM: their roles wait
// more than they work. (With K converted to 16 bits, two CTAs an SM, 32 x 8K
// single tokens of 32 / 8 heads took 58 us, with one 71.)
template <int D>
struct Few {
  static constexpr int R = 16, N = 3 * R;  // rows of a tile; its columns: hi, mid, lo of each
  static constexpr int RAW = KEYS * D, QST = N * D;
  static constexpr int CTAS = D == 128 ? 3 : 2, THREADS = 256;
  static constexpr int RS = D == 128 ? 3 : 2, QS = 2, SB = 2, JOBS = 8, TMEM_COLS = 128;
  static constexpr int R_OFF = 0, Q_OFF = R_OFF + RS * RAW, F_OFF = Q_OFF + QS * QST;  // F: a row's factor and its lse
  static constexpr int JOB_OFF = F_OFF + QS * R * 8, BAR_OFF = JOB_OFF + JOBS * (int)sizeof(Job);
  static constexpr int NBARS = 2 * (RS + QS + SB + JOBS) + 1;
  static constexpr int MISC_OFF = BAR_OFF + NBARS * 8;
  static constexpr int SMEM = MISC_OFF + 16;
  static_assert(SMEM + 1024 <= 233472 / CTAS, "shared memory of a CTA");  // (1 KB of each is the system's)
  static_assert(SB * N <= TMEM_COLS && CTAS * TMEM_COLS <= 512, "S buffers");
};

template <typename T, int D>
__global__ void __launch_bounds__(Few<D>::THREADS, Few<D>::CTAS)
    block_weigh_few_kernel(const __grid_constant__ mj_block_weigh_args a, Take take, int lg, int tb, const __grid_constant__ CUtensorMap tmk) {
  using C = Few<D>;
  constexpr int RS = C::RS, QS = C::QS, SB = C::SB, JOBS = C::JOBS, N = C::N, R = C::R;
  extern __shared__ __align__(1024) unsigned char sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::BAR_OFF);
  uint64_t *r_full = bars, *r_empty = r_full + RS, *q_full = r_empty + RS, *q_empty = q_full + QS, *s_full = q_empty + QS, *s_empty = s_full + SB,
           *j_full = s_empty + SB, *j_empty = j_full + JOBS, *drain = j_empty + JOBS;
  Job* jobs = reinterpret_cast<Job*>(sm + C::JOB_OFF);
  float2* rows = reinterpret_cast<float2*>(sm + C::F_OFF);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + C::MISC_OFF + 4);
  int& never_abort = *reinterpret_cast<int*>(sm + C::MISC_OFF + 8);
  if (reinterpret_cast<uintptr_t>(sm) & 1023) {  // uniform: nothing taken yet
    if (threadIdx.x == 0) flag(a.status, MJ_DEV_BAD_SPLIT);
    griddep_wait();
    return;
  }
  if (!take.both) {
    griddep_wait();
  } else if (!has_any(a, take, false)) {
    griddep_wait();
    return;
  }
  if (threadIdx.x == 0) {
    auto init = [](uint64_t* b, int n, int count) {
      for (int i = 0; i < n; ++i) mbar_init(b + i, count);
    };
    init(r_full, RS, 1);
    init(r_empty, RS, 1);
    init(q_full, QS, 1);
    init(q_empty, QS, 1 + 128);  // its products, and those that read its factors
    init(s_full, SB, 2);         // the product, and its issuer (who saw the job's scales and the rows' factors)
    init(s_empty, SB, 128);
    init(j_full, JOBS, 1);
    init(j_empty, JOBS, 3 + 4);  // the K, Q and MMA warps, those that add up
    mbar_init(drain, 1);
    *abort_flag = 0;
    never_abort = 0;
    fence_mbar_init();
  }
  // rows of a Q stage that no tile has had: nothing reads their columns
  for (int i = threadIdx.x; i < QS * C::QST / 16; i += C::THREADS) reinterpret_cast<uint4*>(sm + C::Q_OFF)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  if (warp == 0 && lane == 0) prefetch_tmap(&tmk);
  if (warp == 2) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Cta<JOBS> cta{a, jobs, j_full, j_empty, abort_flag, &never_abort, lane};
  const int h_r = a.h_q / a.h_k;

  if (warp == 3) {
    find_jobs<4, false>(cta, take, tb, 1, 1);
  } else if (warp == 0) {
    fetch_keys<D, RS>(cta, lg, tmk, sm + C::R_OFF, r_full, r_empty);
  } else if (warp == 1) {
    // ------------------------------------------------------------------------- Q
    // Row r of a tile is (token r / h_r, head r % h_r of the group). D / 8 lanes read
    // a row; a pass is the rows that a warp reads at once.
    constexpr int LPR = D / 8, RPP = 32 / LPR, PASSES = R / RPP;
    const int c = lane % LPR, row_of_lane = lane / LPR;
    int iq = 0;
    bool ok = true;
    for (int i = 0; ok && cta.next_job(i); ++i) {
      const Job& j = jobs[i % JOBS];
      const int nk = j.one ? 1 : j.nk, n = j.n, q0 = j.q0, h0 = j.h * h_r;
#pragma unroll 1
      for (int x = 0; ok && x < nk; ++x)
#pragma unroll 1
        for (int tok = j.t0[x]; tok < n; tok += tb, ++iq) {
          const int count = h_r * min(tb, n - tok), s = iq % QS;
          uint4 raw[PASSES];
          float z[PASSES];
#pragma unroll
          for (int p = 0; p < PASSES; ++p) {
            const int r = p * RPP + row_of_lane;
            if (r < count) {
              const int64_t t = q0 + tok + r / h_r, hq = h0 + r % h_r;
              raw[p] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + t * a.q_stride_tok + hq * a.q_stride_head + 8 * c);
              z[p] = __ldg(a.lse + t * a.h_q + hq);
            }
          }
          ok = cta.wait_warp(&q_empty[s], iq / QS + 1);
          if (!ok) break;
          unsigned char* qs = sm + C::Q_OFF + s * C::QST + (c >> 4) * (N * 128);
#pragma unroll
          for (int p = 0; p < PASSES; ++p) {
            if (p * RPP >= count) break;  // uniform
            const int r = p * RPP + row_of_lane;
            const T* e = reinterpret_cast<const T*>(&raw[p]);
            float v[8], amax = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              v[k] = r < count ? (float)e[k] : 0.f;
              amax = fmaxf(amax, fabsf(v[k]));  // NaN elements do not count
            }
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            // 2^k with amax 2^k in [128, 256), inside fp32's normal range; a row
            // with an infinity becomes NaN
            const int k2 = amax > 0.f ? min(max(134 - (int)(__float_as_uint(amax) >> 23), -126), 126) : 0;
            const float up = amax == INFINITY ? __int_as_float(0x7FFFFFFF) : __uint_as_float((uint32_t)(127 + k2) << 23);
            if (r < count) {
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] *= up;
#pragma unroll
              for (int term = 0; term < 3; ++term) {  // each the rounded rest of those before, times 16
                uint16_t code[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  code[k] = f2_to_e4m3x2(v[2 * k], v[2 * k + 1]);
                  const float2 f = e4m3x2_to_f2(code[k]);
                  v[2 * k] = (v[2 * k] - f.x) * 16.f;
                  v[2 * k + 1] = (v[2 * k + 1] - f.y) * 16.f;
                }
                *reinterpret_cast<uint2*>(qs + unit_offset(term * R + r, (c & 15) >> 1) + (c & 1) * 8) =
                    make_uint2(code[0] | ((uint32_t)code[1] << 16), code[2] | ((uint32_t)code[3] << 16));
              }
              if (c == 0)  // a row without keys adds nothing
                rows[s * R + r] = make_float2(a.softmax_scale * kLog2e * __uint_as_float((uint32_t)(127 - k2) << 23), z[p] == -INFINITY ? -INFINITY : -z[p] * kLog2e);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&q_full[s]);
        }
      if (ok) cta.done_job(i);
    }
  } else if (warp == 2) {
    // ---------------------------------------------------------------------- MMA
    constexpr uint32_t idesc = idesc_f8f6f4(0, 0, 0, 0, N);
    const bool lead = elect_one();
    int it = 0, u = 0, iq = 0;  // S tiles, K tiles, Q tiles
    bool ok = true;
    for (int i = 0; ok && cta.next_job(i); ++i) {
      const Job& j = jobs[i % JOBS];
      const int nk = j.nk;
      const bool one = j.one;
#pragma unroll 1
      for (int x = 0; ok && x < nk; ++x, ++u) {
        const int tiles = j.tiles[x];
        ok = cta.wait_warp(&r_full[u % RS], u / RS);
        const uint64_t k = smem_desc_sw128(smem_addr(sm + C::R_OFF + (u % RS) * C::RAW), 16, 1024);
#pragma unroll 1
        for (int tile = 0; ok && tile < tiles; ++tile, ++it) {
          const int b = it % SB, s = iq % QS;
          const bool last_q = !one || x + 1 == nk;  // use of the Q tile
          ok = ((one && x > 0) || cta.wait_warp(&q_full[s], iq / QS)) && cta.wait_warp(&s_empty[b], it / SB + 1);
          if (!ok) break;
          tc_fence_after();
          const uint64_t q = smem_desc_sw128(smem_addr(sm + C::Q_OFF + s * C::QST), 16, 1024);
          if (lead) {
#pragma unroll
            for (int y = 0; y < D / 32; ++y)  // 32 head-dim elements a step
              mma_f8f6f4(tmem + b * N, k + y / 4 * (KEYS * 8) + y % 4 * 2, q + y / 4 * (N * 8) + y % 4 * 2, idesc, y > 0);
            mma_commit(&s_full[b]);
            mbar_arrive(&s_full[b]);
            if (last_q) mma_commit(&q_empty[s]);
            if (tile + 1 == tiles) mma_commit(&r_empty[u % RS]);
          }
          __syncwarp();
          iq += last_q;
        }
      }
      if (ok) cta.done_job(i);
    }
    if (lead) mma_commit(drain);  // all issued MMAs complete before TMEM is released
    mbar_wait(drain, 0, &never_abort, kWaitNs);
  } else if (warp >= 4) {
    // ------------------------------------------------------------------ the sums
    const int t = threadIdx.x & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    int it = 0, iq = 0;
    bool ok = true;
    for (int i = 0; ok && cta.next_job(i); ++i) {
      const Job& j = jobs[i % JOBS];
      const int ahead = j.L - j.n, n = j.n, nk = j.nk, L = j.L;
      const bool one = j.one;
      float* w = a.weights + j.seq * a.w_stride_seq + j.h * a.w_stride_head + j.kt * KEYS + t;
#pragma unroll 1
      for (int x = 0; ok && x < nk; ++x, w += KEYS) {
        const int key = (j.kt + x) * KEYS + t, tiles = j.tiles[x];
        float sum = 0.f, low = 0.f;  // the sum, and what its rounding lost
        int tok = j.t0[x];
#pragma unroll 1
        for (int tile = 0; tile < tiles; ++tile, tok += tb, ++it) {
          const int b = it % SB, s = iq % QS;
          ok = cta.wait_warp(&s_full[b], it / SB);
          if (!ok) break;
          tc_fence_after();
          const float scale = j.scale[x * (KEYS / 16) + (t >> 4)];
          // rows of queries that are there and see the key
          const int r_lo = max(key - ahead - tok, 0) * h_r, r_hi = min(n - tok, tb) * h_r;
          float p = 0.f;
#pragma unroll
          for (int r0 = 0; r0 < R; r0 += 8) {
            if (r0 >= r_hi) break;  // uniform
            float hi[8], mid[8], lo[8];
            const uint32_t at = tmem + b * N + r0 + lane_base;
            tmem_ld8(at, hi);
            tmem_ld8(at + R, mid);
            tmem_ld8(at + 2 * R, lo);
            tmem_wait_ld();
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              const float2 f = rows[s * R + r0 + r];
              const float score = fmaf(fmaf(lo[r], 0.0625f, mid[r]), 0.0625f, hi[r]), e = exp2_approx(fmaf(score, scale * f.x, f.y));
              p += r0 + r >= r_lo && r0 + r < r_hi ? e : 0.f;
            }
          }
          const bool last_q = !one || x + 1 == nk;
          tc_fence_before();
          mbar_arrive(&s_empty[b]);
          if (last_q) mbar_arrive(&q_empty[s]);
          iq += last_q;
          p += low;
          const float next = sum + p;
          low = p - (next - sum);
          sum = next;
        }
        if (ok && key < L) put(w, sum, key >= ahead);
      }
      if (ok) cta.done_job(i);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
  if (take.both) griddep_wait();
}

constexpr int kMaxDevices = 64;

// How many CTAs of a kernel the current device holds at once, in clusters
// (prepared on first use).
template <class Kernel>
static cudaError_t prepare(Kernel kern, int threads, int smem, int ctas, int cluster, std::atomic<int>* ready, int* grid) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  *grid = ready[dev].load(std::memory_order_acquire);
  if (!*grid) {
    std::lock_guard<std::mutex> lock(tc_init_mutex());
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(grid, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    *grid *= ctas;
    if (cluster > 1) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3((unsigned)cluster);
      cfg.blockDim = dim3((unsigned)threads);
      cfg.dynamicSmemBytes = (size_t)smem;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = (unsigned)cluster;
      at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      int clusters = 0;
      if ((e = cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg)) != cudaSuccess) return e;
      *grid = clusters > 1 ? clusters * cluster : cluster;
    }
    ready[dev].store(*grid, std::memory_order_release);
  }
  return cudaSuccess;
}

// codes as (128 codes, 128-code halves of a row, page rows, KV heads, pages), boxes of one page's rows
static bool key_map(CUtensorMap* m, const mj_block_weigh_args& a) {
  auto fn = tensor_map_encoder();
  if (!fn) return false;
  cuuint64_t dims[5] = {128, (cuuint64_t)(a.head_size / 128), (cuuint64_t)a.page_size, (cuuint64_t)a.h_k, (cuuint64_t)a.num_pages};
  // a dimension of extent 1 never moves its coordinate: any legal stride
  cuuint64_t strides[4] = {128, (cuuint64_t)(a.k_stride_row ? a.k_stride_row : 16), (cuuint64_t)(a.k_stride_head ? a.k_stride_head : 16),
                           (cuuint64_t)(a.k_stride_page ? a.k_stride_page : 16)};
  cuuint32_t box[5] = {128, 1, (cuuint32_t)a.page_size, 1, 1}, estr[5] = {1, 1, 1, 1, 1};
  // 128 bytes at a time into L2: behind a row's 128 of K lie V's, which nobody reads
  // (32 x 8K single tokens: 53 us with 256)
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(a.k_cache), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, int N>
static cudaError_t launch_t(const mj_block_weigh_args& a, Take take, cudaStream_t stream) {
  using C = Cfg<T, D, N>;
  // CTAs of a cluster, which share a job's rows where there are too few jobs (4096
  // tokens of 24 / 4 heads of 256 144 us, without 257; 2000 behind 2000 of 6 / 1 heads
  // 28 and 73). One where the rows are few tiles, for looking costs (500 tokens behind
  // 7000, 8 / 2 heads, 22.6 and 19.9 us), or where they are enough for two jobs an SM,
  // as far as the tensor's rows tell (16 prompts of 512, 32 / 8 heads, 68 us, in
  // clusters 72; 500 tokens in a buffer of 8192 rows 20.3, in clusters 14.7). Two
  // otherwise, which fill all SMs. Four or eight, which on 148 SMs leave 16 and 28
  // out, where the weights are too short for more jobs than there are such clusters
  // (33 and 15; weights wider than their sequences take two): 600 tokens of 6 heads,
  // 15 jobs 28.8, 21.2, 17.2 and 15.8 us with one, two, four and eight, 24 jobs 28.8,
  // 21.1, 17.2 and 22.5, 36 jobs 29.5, 21.3, 23.3 and 29.3, 80 jobs, where none share,
  // 29.5 and 31 to 32.
  const int64_t most = a.window && a.window < a.num_rows ? a.window : a.num_rows, tiles = (most * (a.h_q / a.h_k) + N - 1) / N;
  const int64_t row_jobs = (a.num_rows + KEYS - 1) / KEYS * a.h_k, most_jobs = (a.weights_cols + KEYS - 1) / KEYS * a.num_seqs * a.h_k;
  auto kern = block_weigh_kernel<T, D, N, false>;
  static std::atomic<int> ready[4][kMaxDevices];
  int grid = 0, level = 0;  // log2 of a cluster's CTAs
  cudaError_t e = prepare(kern, C::THREADS, C::SMEM, 1, 1, ready[0], &grid);
  if (e != cudaSuccess) return e;
  if (tiles >= 8 && row_jobs < 2 * grid) {
    static_assert(1 << 3 <= C::PARTS, "buffers of a cluster's sums");
    kern = block_weigh_kernel<T, D, N, true>;
    for (level = 3;; --level) {
      if ((e = prepare(kern, C::THREADS, C::SMEM, 1, 1 << level, ready[level], &grid)) != cudaSuccess) return e;
      if (level == 1 || most_jobs <= grid >> level) break;
    }
  }
  const int cluster = 1 << level;
  CUtensorMap mk, mq;
  if (!key_map(&mk, a)) return cudaErrorInvalidValue;
  // a tile of Q rows: tb tokens of hb heads of a group, or, of a larger group, N heads of one token
  const int h_r = a.h_q / a.h_k, hb = h_r < N ? h_r : N, tb = N / hb, ht = (h_r + hb - 1) / hb;
  {  // rows as (elements, heads of a group, groups, tokens)
    const cuuint64_t head = a.h_q > 1 ? a.q_stride_head * 2 : 16, tok = a.num_rows > 1 ? a.q_stride_tok * 2 : 16;
    cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)h_r, (cuuint64_t)a.h_k, (cuuint64_t)a.num_rows}, strides[3] = {head, head * h_r, tok};
    cuuint32_t box[4] = {64, (cuuint32_t)hb, 1, (cuuint32_t)tb}, estr[4] = {1, 1, 1, 1};
    if (tensor_map_encoder()(&mq, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                             const_cast<void*>(a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, a, take, cluster, block_log2(a.kv_format), hb, tb, ht, mk, mq);
}

template <typename T, int D>
static cudaError_t launch_few(const mj_block_weigh_args& a, Take take, cudaStream_t stream) {
  using C = Few<D>;
  auto kern = block_weigh_few_kernel<T, D>;
  static std::atomic<int> ready[kMaxDevices];
  int grid = 0;
  const cudaError_t e = prepare(kern, C::THREADS, C::SMEM, C::CTAS, 1, ready, &grid);
  if (e != cudaSuccess) return e;
  CUtensorMap mk;
  if (!key_map(&mk, a)) return cudaErrorInvalidValue;
  return launch_kernel(kern, dim3((unsigned)grid), dim3(C::THREADS), C::SMEM, stream, a, take, block_log2(a.kv_format), C::R / (a.h_q / a.h_k), mk);
}

template <typename T>
static cudaError_t launch_d(const mj_block_weigh_args& a, cudaStream_t stream) {
  // The kernel for few rows takes the sequences whose rows are one tile of its 16:
  // of more it would make Q's terms again for every tile of keys (8 sequences of
  // 6K, 16 rows 24 us, 32 rows 65 and with the other kernel 51, 64 rows 120 and
  // 57). The lengths are the device's, so where there may be both, both are
  // launched: 64 single tokens of 8K beside a chunk of 512 take 155 us, with the
  // kernel for many rows alone 435; beside a chunk of 190 131, with the one for few
  // alone 717. (A launch that finds nothing costs 2 us: windows no longer than the
  // tile need none: 4 of each of 8 x 300 tokens behind 6K 24 us, with it 28.) With no
  // more tokens than sequences all are taken to be single ones.
  const int64_t most = a.window ? (int64_t)a.num_seqs * a.window : a.num_rows, tokens = a.num_rows < most ? a.num_rows : most;
  const int h_r = a.h_q / a.h_k, fit = 16 / h_r;
  const bool few = fit && (a.num_seqs > 1 || tokens <= fit),
             many = !few || (tokens > a.num_seqs && tokens > fit && !(a.window && a.window <= fit));
  if (many) {
    constexpr int N256 = std::is_same<T, __half>::value ? 64 : 96;  // (fp16's two sums of 96 do not fit TMEM)
    const Take take = {few ? fit + 1 : 1, INT_MAX, few};
    const cudaError_t e = a.head_size == 256 ? launch_t<T, 256, N256>(a, take, stream) : launch_t<T, 128, 128>(a, take, stream);
    if (e != cudaSuccess || !few) return e;
  }
  const Take take = {1, many ? fit : INT_MAX, many};
  return a.head_size == 256 ? launch_few<T, 256>(a, take, stream) : launch_few<T, 128>(a, take, stream);
}

}  // namespace bw

cudaError_t launch_block_weigh(const mj_block_weigh_args& a, cudaStream_t stream) {
  return a.dtype == MJ_DT_FP16 ? bw::launch_d<__half>(a, stream) : bw::launch_d<__nv_bfloat16>(a, stream);
}

}  // namespace mj
