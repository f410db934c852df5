// The attention weight that each cached token receives in a step, added up per
// KV head, on the 5th-generation tensor cores (sm_100a):
// w[s][h][j] += sum over the rows (query, head of the group) that see key j of
// exp(scale q . k_j - lse).
//
// The scores are computed with the keys in the rows of the product, S^T = K Q^T:
// a lane of TMEM is a key, so a thread adds up its own key's weights in
// registers, no two threads meet, and the order of every sum is fixed. A job is
// (sequence, KV head, tile of 128 keys): its K tile stays, the query rows that
// see it stream past in tiles of N.
//
// Both operands are 16 bits wide. Q enters as it is, by TMA; K's e4m3 codes are
// exact in either type, so the products are exact, and the block scales, one a
// key, go into the exponent with the softmax scale. (fp8 products would need Q
// in three e4m3 terms to leave an fp32 sum its precision.)
//
// Jobs need no plan: one warp of each CTA walks the sequences' lengths on the
// device, so a captured graph replays for whatever they hold. Persistent CTAs
// take the jobs in rounds, every other round in reverse: a prompt's first keys
// are seen by all its rows, its last by few.
//
// Warp roles: 0 K (page walk, TMA, block scales; where few rows see a tile, four
// warps of their own behind the others), 1 Q (TMA), 2 MMA, 3 the jobs; then
// warpgroups that convert K's codes, in turn, and warpgroups that take the S tiles
// in turn and add up. Every mbarrier wait is bounded; on a timeout the CTA flags
// MJ_DEV_TIMEOUT, all roles stop, copies and MMAs in flight complete and TMEM is
// freed.
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

// Tiles of keys of a job, at most: where few rows see them, a job's lookups and
// its descriptor serve several.
template <int N>
constexpr int kTiles = N >= 64 ? 1 : 4;

// What a role needs to know of a job. The K warp adds the scales.
struct Job {
  int seq, h, kt, nk, L, n, q0;  // seq < 0: no more; nk tiles of keys from kt on
  int t0[4], tiles[4];           // of each: the first query that counts and sees one of them, tiles of rows from it on
  int one;                       // they have one tile of rows, the same
  float scale[4 * (KEYS / 16)];
};

template <typename T, int D, int N>
struct Cfg {
  static constexpr int RAW = KEYS * D, K16 = 2 * RAW, QST = N * D * 2;  // a tile's codes; as 16 bits; a tile of Q rows
  static constexpr bool WIDE = N >= 64;
  // CTAs of an SM: a CTA's roles wait for one another more than they work where few
  // rows see a tile, so two (at head size 256 their shared memory allows one).
  static constexpr int CTAS = !WIDE && D == 128 ? 2 : 1;
  // Warpgroups that convert K's codes, and that add up. Many rows: the
  // exponentials bound it, and two or four warps on a scheduler must hide one
  // another's latency (8192 tokens, 32 / 8 heads: 376 us with two warpgroups, 341
  // with four). Few rows: every tile of keys is converted for one product.
  static constexpr int CWGS = WIDE || CTAS == 2 ? 1 : 2, WGS = WIDE ? 4 : CTAS == 2 ? 1 : 2;
  // Warps that fetch K. A lane's copies are issued one after another, over 100
  // cycles each; with pages of 16 a tile has eight.
  static constexpr int KWARPS = WIDE || CTAS == 2 ? 1 : 4, K0 = KWARPS == 1 ? 0 : 4 * (1 + CWGS + WGS), THREADS = 128 * (1 + CWGS + WGS) + (KWARPS == 1 ? 0 : 128);
  // stages of K codes, of K in 16 bits, of Q
  static constexpr int RS = WIDE && D == 256 ? 1 : 2, KS = WIDE && D == 256 ? 1 : 2, QS = D == 256 || !WIDE ? 2 : 3;
  static constexpr int SB = 4;  // S buffers in TMEM; a warpgroup that adds up has three of its columns' lse
  static constexpr int TMEM_COLS = CTAS == 2 ? 64 : 512;
  static_assert(SB * N <= TMEM_COLS, "S buffers");
  static constexpr int JOBS = WIDE ? 4 : 8;
  static constexpr int PAIRS = WGS * (WGS - 1);  // of a warpgroup that writes weights and one that adds its part
  static constexpr int K_OFF = 0, R_OFF = K_OFF + KS * K16, Q_OFF = R_OFF + RS * RAW, Z_OFF = Q_OFF + QS * QST;
  static constexpr int RED_OFF = Z_OFF + 3 * WGS * N * 4, JOB_OFF = RED_OFF + PAIRS * KEYS * 4, BAR_OFF = JOB_OFF + JOBS * (int)sizeof(Job);
  static constexpr int NBARS = 2 * (RS + KS + QS + SB + JOBS + PAIRS) + WGS + 1;
  static constexpr int MISC_OFF = BAR_OFF + NBARS * 8;
  static constexpr int SMEM = MISC_OFF + 16;
  static_assert(SMEM + 1024 <= 233472 / CTAS, "shared memory of a CTA");  // (1 KB of each is the system's)
  static_assert(JOBS >= 3, "the K warp looks two jobs ahead");
  // a buffer is always waited for by the same warpgroup, whose waits are in order:
  // another's could take an older phase of the same parity for its own
  static_assert(RS % CWGS == 0 && KS % CWGS == 0 && SB % WGS == 0, "buffers of a warpgroup");
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

// byte offset of 16-byte unit u of row r in a [rows][128 bytes] swizzled block
__device__ __forceinline__ uint32_t unit_offset(uint32_t r, uint32_t u) { return r * 128 + ((u ^ (r & 7)) << 4); }

template <typename T, int D, int N>
__global__ void __launch_bounds__(Cfg<T, D, N>::THREADS, Cfg<T, D, N>::CTAS)
    block_weigh_kernel(const __grid_constant__ mj_block_weigh_args a, int lg, int hb, int tb, int ht,
                       const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmq) {
  using C = Cfg<T, D, N>;
  constexpr int RS = C::RS, KS = C::KS, QS = C::QS, SB = C::SB, JOBS = C::JOBS, CWGS = C::CWGS, WGS = C::WGS;
  extern __shared__ __align__(1024) unsigned char sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::BAR_OFF);
  uint64_t *r_full = bars, *r_empty = r_full + RS, *k_full = r_empty + RS, *k_empty = k_full + KS, *q_full = k_empty + KS,
           *q_empty = q_full + QS, *s_full = q_empty + QS, *s_empty = s_full + SB, *j_full = s_empty + SB, *j_empty = j_full + JOBS,
           *red_full = j_empty + JOBS, *red_empty = red_full + C::PAIRS, *z_full = red_empty + C::PAIRS, *drain = z_full + WGS;
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
    init(j_empty, JOBS, 2 + C::KWARPS + 4 * (CWGS + WGS));  // the Q, MMA and K warps, those that convert, those that add up
    init(red_full, C::PAIRS, 128);
    init(red_empty, C::PAIRS, 128);
    init(z_full, WGS, 128);
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
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto wait = [&](uint64_t* bar, int phase) {
    if (mbar_wait(bar, (uint32_t)phase & 1u, abort_flag, kWaitNs)) return true;
    if (!*abort_flag) {
      *abort_flag = 1;
      flag(a.status, MJ_DEV_TIMEOUT);
    }
    return false;
  };
  // whole warps: every lane leaves with its warp
  auto wait_warp = [&](uint64_t* bar, int phase) { return __all_sync(0xffffffffu, wait(bar, phase)) != 0; };
  // job i of this CTA, once it is there; false at the end
  auto next_job = [&](int i) { return wait_warp(&j_full[i % JOBS], i / JOBS) && jobs[i % JOBS].seq >= 0; };
  auto done_job = [&](int i) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&j_empty[i % JOBS]);
  };

  if (warp == 3) {
    // ------------------------------------------------------------------ the jobs
    // 32 sequences at a time: lane i has the key tiles of sequence s0 + i
    int L = 0, n = 0, q0 = 0;
    auto tiles_of = [&](int s, bool complain) {
      if (s >= a.num_seqs) return 0;
      q0 = a.offsets[s];
      n = a.offsets[s + 1] - q0;
      L = a.seq_lens[s];
      if (q0 < 0 || n < 0 || q0 + (int64_t)n > a.num_rows || L < 0 || L > a.weights_cols ||
          L > (int64_t)a.block_table_cols * a.page_size || L > INT_MAX - 8 * KEYS) {
        if (complain) flag(a.status, MJ_DEV_BAD_LENGTH);
        return 0;
      }
      return n ? (L + KEYS - 1) / KEYS : 0;
    };
    // Tiles a job: as many as leave every CTA two jobs (each costs its lookups'
    // latency; a few jobs more than CTAs leave some of them idle).
    int per = 1;
    if (kTiles<N> > 1) {
      int64_t tiles = 0;
      for (int s = lane; s - lane < a.num_seqs && tiles * a.h_k < 2ll * kTiles<N> * gridDim.x; s += 32) {
        int x = tiles_of(s, false);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        tiles += x;
      }
      while (per < kTiles<N> && tiles * a.h_k >= 4ll * per * gridDim.x) per *= 2;
    }
    int s0 = -32, i = 0;
    int64_t base = 0, total = 0, before = 0, count = 0;
    bool ok = true;
    for (int64_t round = 0; ok; ++round, ++i) {
      const int64_t p = round * gridDim.x + (round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
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
      ok = wait_warp(&j_empty[i % JOBS], i / JOBS + 1);
      if (!ok) break;
      Job& j = jobs[i % JOBS];
      if (!more) {
        if (lane == 0) {
          j.seq = -1;
          mbar_arrive(&j_full[i % JOBS]);
        }
        break;
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
          j.tiles[x] = (n - j.t0[x] + tb - 1) / tb * ht;
        }
        j.one = j.tiles[0] == 1 && j.t0[j.nk - 1] == j.t0[0];  // (t0 grows with x)
        mbar_arrive(&j_full[i % JOBS]);
      }
      __syncwarp();
    }
  } else if (warp >= C::K0 && warp < C::K0 + C::KWARPS) {
    // -------------------------------------------------------- K: codes and scales
    // Every K warp looks up all pages and copies its share of each tile's.
    // Lane i looks up the page of the job's 16-token group i two jobs ahead and
    // reads its exponent one job ahead (a use at once would wait for memory).
    constexpr int kNone = INT_MIN;
    const uint64_t policy = l2_policy_evict_normal();
    const int kw = warp - C::K0;
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
    bool here = next_job(0), ahead = here && next_job(1), ok = true;
    int e0 = here ? entry_of(jobs[0]) : kNone, e1 = ahead ? entry_of(jobs[1 % JOBS]) : kNone;
    int page = page_of(e0);
    unsigned char ex = here ? exponent_of(jobs[0], page) : 127;
    int i = 0, u = 0;
    for (; ok && here; ++i) {
      Job& j = jobs[i % JOBS];
      const int nk = j.nk, h = j.h;
      if (kw == 0) j.scale[lane] = block_scale(ex);
      const int page1 = page_of(e1);
      const unsigned char ex1 = ahead ? exponent_of(jobs[(i + 1) % JOBS], page1) : 127;
      const bool ahead2 = ahead && next_job(i + 2);
      e1 = ahead2 ? entry_of(jobs[(i + 2) % JOBS]) : kNone;
      __syncwarp();  // the scales are written before lane 0 arrives
      for (int x = 0; x < nk; ++x, ++u) {
        ok = wait_warp(&r_empty[u % RS], u / RS + 1);
        if (!ok) break;
        if (kw == 0 && lane == 0) mbar_arrive_expect_tx(&r_full[u % RS], C::RAW);  // (whichever comes first, this or another warp's copies)
        __syncwarp();
        const int pg = __shfl_sync(0xffffffffu, page, (x * (KEYS / 16) + lane * groups) & 31);
        if (lane < pages && lane % C::KWARPS == kw) {
#pragma unroll
          for (int dh = 0; dh < D / 128; ++dh)  // an absent page is read out of range: zeros
            tma_load_5d(sm + C::R_OFF + (u % RS) * C::RAW + dh * (KEYS * 128) + lane * ps * 128, &tmk, &r_full[u % RS], 0, dh, 0, h,
                        pg < 0 ? (int)a.num_pages : pg, policy);
        }
      }
      if (!ok) break;
      done_job(i);
      page = page1;
      ex = ex1;
      here = ahead;
      ahead = ahead2;
    }
    for (int x = max(u - RS, 0); x < u; ++x) mbar_wait(&r_full[x % RS], (x / RS) & 1, &never_abort, kWaitNs);  // copies in flight land
  } else if (warp == 1) {
    // ------------------------------------------------------------------------- Q
    // Column c of a tile is (token c / hb, head c % hb of the tile's).
    const int h_r = a.h_q / a.h_k;
    const uint64_t policy = l2_policy_evict_normal();
    int it = 0;
    bool ok = true;
    for (int i = 0; ok && next_job(i); ++i) {
      const Job& j = jobs[i % JOBS];
      const int nk = j.one ? 1 : j.nk, h = j.h, n = j.n, q0 = j.q0;
      for (int x = 0; ok && x < nk; ++x)
        for (int tok = j.t0[x], head = 0; tok < n; ++it) {
          const int s = it % QS;
          ok = wait_warp(&q_empty[s], it / QS + 1);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&q_full[s], (D / 64) * 128 * hb * tb);
          __syncwarp();
          if (lane < D / 64) tma_load_4d(sm + C::Q_OFF + s * C::QST + lane * (N * 128), &tmq, &q_full[s], lane * 64, head, h, q0 + tok, policy);
          head += hb;
          if (head >= h_r) {
            head = 0;
            tok += tb;
          }
        }
      if (ok) done_job(i);
    }
    for (int y = max(it - QS, 0); y < it; ++y) mbar_wait(&q_full[y % QS], (y / QS) & 1, &never_abort, kWaitNs);
  } else if (warp == 2) {
    // ---------------------------------------------------------------------- MMA
    constexpr uint32_t idesc = std::is_same<T, __half>::value ? idesc_f16(0, 0, N) : idesc_bf16(0, 0, N);
    const bool lead = elect_one();
    int it = 0, u = 0, iq = 0;  // S tiles, K tiles, Q tiles
    bool ok = true;
    for (int i = 0; ok && next_job(i); ++i) {
      const Job& j = jobs[i % JOBS];
      const int nk = j.nk;
      const bool one = j.one;
      int x = 0, tile = 0, tiles = j.tiles[0];
      // everything that the tile at hand needs
      auto ready = [&]() {
        return (tile > 0 || wait_warp(&k_full[u % KS], u / KS)) && ((one && x > 0) || wait_warp(&q_full[iq % QS], iq / QS)) &&
               wait_warp(&s_empty[it % SB], it / SB + 1);
      };
      ok = ready();
      while (ok && x < nk) {
        const int b = it % SB, s = iq % QS, ku = u % KS;
        const bool last_k = tile + 1 == tiles, last_q = !one || x + 1 == nk;  // uses of the K tile, of the Q tile
        tc_fence_after();
        const uint64_t k = smem_desc_sw128(smem_addr(sm + C::K_OFF + ku * C::K16), 16, 1024);
        const uint64_t q = smem_desc_sw128(smem_addr(sm + C::Q_OFF + s * C::QST), 16, 1024);
        auto steps = [&](auto half) {  // 16 head-dim elements a step
          constexpr int H = decltype(half)::value;
          if (lead) {
#pragma unroll
            for (int y = H * (D / 32); y < (H + 1) * (D / 32); ++y)
              mma_f16(tmem + b * N, k + y / 4 * (KEYS * 8) + y % 4 * 2, q + y / 4 * (N * 8) + y % 4 * 2, idesc, y > 0);
          }
        };
        steps(std::integral_constant<int, 0>());
        // The waits for the keys' next tile pass while these products run. Not those
        // for other keys: this tile's K buffer would be free only after they are there.
        ++it;
        iq += last_q;
        ++tile;
        if (last_k) {
          tile = 0;
          ++u;
          if (++x < nk) tiles = j.tiles[x];
        }
        if (!last_k) ok = ready();
        steps(std::integral_constant<int, 1>());
        if (lead) {
          mma_commit(&s_full[b]);
          mbar_arrive(&s_full[b]);
          if (last_q) mma_commit(&q_empty[s]);
          if (last_k) mma_commit(&k_empty[ku]);
        }
        __syncwarp();
        if (last_k && x < nk) ok = ready();
      }
      if (ok) done_job(i);
    }
    if (lead) mma_commit(drain);  // all issued MMAs complete before TMEM is released
    mbar_wait(drain, 0, &never_abort, kWaitNs);
  } else if (warp == 0) {
    // (K has warps of its own)
  } else if (warp < 4 + 4 * CWGS) {
    // ------------------------------------------------------------ codes -> 16 bits
    // Thread ct takes 16-code chunk 4 blk + quad of rows r0, r0 + STEP, ...: eight
    // neighbouring threads are four chunks of a 64-element block in rows r and
    // r ^ 5, so that both their staged reads and their stores cover all banks.
    const int ct = threadIdx.x & 127, cwg = (warp - 4) >> 2;
    constexpr int BLOCKS = D / 64, STEP = 32 / BLOCKS, NC = KEYS / STEP, BATCH = 4;
    const int quad = ct & 3, blk = (ct >> 3) % BLOCKS, pr = (ct >> 3) / BLOCKS;
    const int r0 = ((pr & 3) ^ ((ct >> 2) & 1 ? 5 : 0)) + (pr & ~3) * 2;
    int u = 0;
    bool ok = true;
    auto convert = [&]() {
      if (!wait_warp(&r_full[u % RS], u / RS) || !wait_warp(&k_empty[u % KS], u / KS + 1)) return false;
      const unsigned char* raw = sm + C::R_OFF + (u % RS) * C::RAW + (blk >> 1) * (KEYS * 128);
      unsigned char* out = sm + C::K_OFF + (u % KS) * C::K16 + blk * (KEYS * 128);
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
      mbar_arrive(&r_empty[u % RS]);
      fence_proxy_async_smem();
      mbar_arrive(&k_full[u % KS]);
      return true;
    };
    for (int i = 0; ok && next_job(i); ++i) {
      const int nk = jobs[i % JOBS].nk;
#pragma unroll 1
      for (int x = 0; ok && x < nk; ++x, ++u)
        if (CWGS == 1 || u % CWGS == cwg) ok = convert();
      if (ok) done_job(i);
    }
  } else {
    // ------------------------------------------------------------------ the sums
    const int wg = (warp - 4 - 4 * CWGS) >> 2, t = threadIdx.x & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const int h_r = a.h_q / a.h_k;
    // The lse of this warpgroup's tiles, by buffer: a tile's are stored while the
    // one before is added up, which warps that lag behind may still be at the
    // start of; so three.
    float* const zbuf = reinterpret_cast<float*>(sm + C::Z_OFF) + wg * (3 * N);
    int z_stored = 0, z_seen = 0;
    // this thread's column: its lse in tile `tile` of the queries from t0 on
    const int z_tok = t < hb * tb ? t / hb : INT_MAX / 2, z_head = t % hb;
    auto tok_of = [&](int t0, int tile) { return t0 + (ht == 1 ? tile : tile / ht) * tb; };
    auto load_lse = [&](const Job& j, int t0, int tile) {
      const int tok = tok_of(t0, tile), head = ht == 1 ? z_head : tile % ht * hb + z_head;
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
      const uint32_t s_addr = tmem + b * N + lane_base;
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)}, v[2][8];
      tmem_ld16(s_addr, reinterpret_cast<float*>(v[0]));
#pragma unroll
      for (int c = 0; c < N; c += 16) {
        float2* const now = v[c / 16 & 1];
        tmem_wait_ld();
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
    bool ok = true;
    for (int i = 0; ok && next_job(i); ++i) {
      const Job& j = jobs[i % JOBS];
      const int ahead = j.L - j.n, n = j.n, nk = j.nk, L = j.L;
      int z_at = -1;  // the first query of the tile whose lse this warpgroup has, where it is its keys' only one
#pragma unroll 1
      for (int x = 0; x < nk; ++x) {
        const int key = (j.kt + x) * KEYS + t, t0 = j.t0[x], tiles = j.tiles[x];
        // The warpgroups take the tiles in turn; this one has the unit's tiles
        // place, place + WGS, ... The first place writes the weights.
        const int place = (wg - it) & (WGS - 1), it0 = it;
        it += tiles;
        if (place >= tiles) continue;
        float* w = a.weights + j.seq * a.w_stride_seq + j.h * a.w_stride_head + key;
        float old = 0.f;
        if (place == 0 && key < min(L, ahead)) old = *w;
        const bool again = tiles == 1 && z_at == t0;
        z_at = tiles == 1 ? t0 : -1;
        float z = 0.f;
        if (!again) {
          store_lse(load_lse(j, t0, place));
          if (place + WGS < tiles) z = load_lse(j, t0, place + WGS);
        }
        float sum = 0.f, low = 0.f, c2 = 0.f;  // the sum, and what its rounding lost
#pragma unroll 1
        for (int tile = place; tile < tiles; tile += WGS) {
          if (!again) ok = wait_warp(&z_full[wg], z_seen++);
          if (tile + WGS < tiles) {  // the lse of this warpgroup's next tile, and the load of the one's behind it
            store_lse(z);
            if (tile + 2 * WGS < tiles) z = load_lse(j, t0, tile + 2 * WGS);
          }
          const int b = (it0 + tile) % SB;
          ok = ok && wait_warp(&s_full[b], (it0 + tile) / SB);
          if (!ok) break;
          tc_fence_after();
          if (tile == place) c2 = a.softmax_scale * kLog2e * j.scale[x * (KEYS / 16) + (t >> 4)];
          // columns of queries that are there and see the key
          const int tok = tok_of(t0, tile), c_lo = max(key - ahead - tok, 0) * hb, c_hi = min(n - tok, tb) * hb;
          const bool part = N == 16 || tok + tb > n || key - t + KEYS - 1 > ahead + tok;  // uniform; few columns: always
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
        if (place == 0 && key < L) *w = old + sum;
      }
      if (ok) done_job(i);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

constexpr int kMaxDevices = 64;

template <typename T, int D, int N>
static cudaError_t launch_t(const mj_block_weigh_args& a, cudaStream_t stream) {
  using C = Cfg<T, D, N>;
  auto kern = block_weigh_kernel<T, D, N>;
  static std::atomic<int> ready[kMaxDevices];  // CTAs that the device holds at once, once the kernel is prepared on it
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  int ctas = ready[dev].load(std::memory_order_acquire);
  if (!ctas) {
    std::lock_guard<std::mutex> lock(tc_init_mutex());
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(&ctas, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    ctas *= C::CTAS;
    ready[dev].store(ctas, std::memory_order_release);
  }
  auto fn = tensor_map_encoder();
  if (!fn) return cudaErrorNotSupported;
  CUtensorMap mk, mq;
  {  // codes as (128 codes, 128-code halves of a row, page rows, KV heads, pages), boxes of one page's rows
    cuuint64_t dims[5] = {128, (cuuint64_t)(D / 128), (cuuint64_t)a.page_size, (cuuint64_t)a.h_k, (cuuint64_t)a.num_pages};
    // a dimension of extent 1 never moves its coordinate: any legal stride
    cuuint64_t strides[4] = {128, (cuuint64_t)(a.k_stride_row ? a.k_stride_row : 16), (cuuint64_t)(a.k_stride_head ? a.k_stride_head : 16),
                             (cuuint64_t)(a.k_stride_page ? a.k_stride_page : 16)};
    cuuint32_t box[5] = {128, 1, (cuuint32_t)a.page_size, 1, 1}, estr[5] = {1, 1, 1, 1, 1};
    if (fn(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(a.k_cache), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  }
  // a tile of Q rows: tb tokens of hb heads of a group, or, of a larger group, N heads of one token
  const int h_r = a.h_q / a.h_k, hb = h_r < N ? h_r : N, tb = N / hb, ht = (h_r + hb - 1) / hb;
  {  // rows as (elements, heads of a group, groups, tokens)
    const cuuint64_t head = a.h_q > 1 ? a.q_stride_head * 2 : 16, tok = a.num_rows > 1 ? a.q_stride_tok * 2 : 16;
    cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)h_r, (cuuint64_t)a.h_k, (cuuint64_t)a.num_rows}, strides[3] = {head, head * h_r, tok};
    cuuint32_t box[4] = {64, (cuuint32_t)hb, 1, (cuuint32_t)tb}, estr[4] = {1, 1, 1, 1};
    if (fn(&mq, std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(a.q),
           dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return cudaErrorInvalidValue;
  }
  return launch_kernel(kern, dim3((unsigned)ctas), dim3(C::THREADS), C::SMEM, stream, a, block_log2(a.kv_format), hb, tb, ht, mk, mq);
}

template <typename T>
static cudaError_t launch_d(const mj_block_weigh_args& a, cudaStream_t stream) {
  // rows of a sequence and KV head that count, on average
  const int64_t all = a.num_rows * (a.h_q / a.h_k), most = a.window ? (int64_t)a.num_seqs * a.window * (a.h_q / a.h_k) : all;
  const bool few = (all < most ? all : most) <= (int64_t)32 * a.num_seqs;
  if (a.head_size == 256) return few ? launch_t<T, 256, 16>(a, stream) : launch_t<T, 256, 96>(a, stream);
  return few ? launch_t<T, 128, 16>(a, stream) : launch_t<T, 128, 128>(a, stream);
}

}  // namespace bw

cudaError_t launch_block_weigh(const mj_block_weigh_args& a, cudaStream_t stream) {
  return a.dtype == MJ_DT_FP16 ? bw::launch_d<__half>(a, stream) : bw::launch_d<__nv_bfloat16>(a, stream);
}

}  // namespace mj
