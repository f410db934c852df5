// Attention of ragged query chunks over the block-scaled cache on the
// 5th-generation tensor cores (sm_100a).
//
// A CTA takes one work item of one KV head: NT tiles of 128 rows -- a row is
// (query token, head of the KV head's group), so a group shares every key read
// -- and a range of key tiles of BN tokens. Warp roles:
//   producer warps       one for K, one for V and the tile's block scales: page-
//                        table walk, one TMA box per page
//   converter warpgroup  staged V codes e4m3 -> f16 (exact) into the MN-major
//                        operand tiles
//   MMA warps            one per row tile: S = Q K^T (kind::f8f6f4, K as
//                        stored) of the next key tile, then O += P V of this
//                        one (kind::f16, P from TMEM, over the columns of its
//                        S). A wait costs its warp 100 to 200 cycles even when
//                        it finds the phase complete: one issuing warp for both
//                        row tiles left the tensor cores idle
//   softmax warpgroups   one per row tile, a thread = a row: S to registers,
//                        online softmax in base 2, P back to TMEM as f16
// S is double-buffered in TMEM (64 keys a tile, two buffers and O of both row
// tiles fill its 512 columns): the next tile's product runs beside this one's
// softmax, so a softmax warpgroup finds its next scores waiting (8192 tokens of
// 32 / 8 heads of 128: 641 us with 128 keys a tile and one buffer, 614 so).
//
// What bounds it: the softmax warps. Such a prompt takes 535 to 605 us in a graph
// (its 550 GFLOP at 0.91 to 1.03 PFLOP/s, by the clock that a run's power leaves:
// 582 us at a median of 1845 MHz, 1965 without a load), five chunks of 1.5K
// tokens behind 6K 495 to 555, a prompt of 4K at head size 256 and 24 / 4 heads
// 260 (0.79 PFLOP/s). The figures below for variants are medians of runs among
// one another; differences under 3 % are within that spread. A tile of 64 keys costs
// 1,312 cycles of tensor work and 1,024 of exponentials on the special-function
// unit, hence the polynomial for a quarter of them (587 -> 572 us; for half,
// 630); two softmax warps on a scheduler hide little of each other's latency,
// and four with half a row each did no better (586 to 601).
//
// Q enters as TERMS e4m3 terms of its row scaled by a power of two to [128,
// 256): hi + mid holds bf16's 8 bits, a third term f16's 11; what is lost is
// below 2^-17 of the row's largest element. Two terms at fp8's rate cost what
// one f16 product would, and K needs no conversion.
// Scales: score_ij = c 2^ek_j (q_i . kcode_j), and V's scale is folded into the
// exponent: z_ij = score_ij + ev_j (base 2), P' = 2^(z - m), O = sum P' vcode /
// sum P' 2^-ev. The running maximum m is thus over what enters O, so a large V
// scale cannot push the other rows' P out of f16's range. m moves lazily, when
// a z exceeds it by 15: moving it means waiting for the last product and
// rescaling O in TMEM, two thousand cycles of a tile's softmax, and a warp pays
// for each of its 32 rows (a threshold of 8 did so on most tiles of random
// scores).
// P' enters the product as f16 (an exact product would take two), the row sum in
// fp32: 11 bits down to 2^-14 of the maximum, steps of 2^-24 of it below. With
// bf16 outputs their own rounding hides that; fp16 outputs are 2.5e-4 to 3e-4 from 64
// bits where fp32 arithmetic leaves 2.1e-4. The maximum counts V's scales: an
// element that one block holds zeros in loses bits of a block whose V scale is
// more than 2^14 below that one's, and all of them beyond 2^25.
//
// Every mbarrier wait is bounded; on a timeout the CTA flags MJ_DEV_TIMEOUT,
// all roles stop, the copies and MMAs in flight complete and TMEM is freed.
#include <limits.h>
#include <math.h>

#include <atomic>
#include <mutex>

#include <cuda.h>

#include "block_cache.cuh"

namespace mj {

std::mutex& tc_init_mutex();
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn tensor_map_encoder();

namespace ba {

using namespace sm100;

constexpr uint64_t kWaitNs = 500000000ull;  // per wait; a tile takes microseconds
constexpr int kPolyOf4 = 1;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRaise = 15.f;  // the running maximum moves when a P' would pass 2^15 (f16's end is 2^16)

template <typename T, int D>
struct Cfg {
  static constexpr int NT = D == 256 ? 1 : 2;
  static constexpr int BN = MJ_BLOCK_KEYS;
  static constexpr int ROWS = NT * 128;
  static_assert(ROWS == MJ_BLOCK_ROWS(D), "the plan's rows");
  static constexpr int TERMS = std::is_same<T, __half>::value ? 3 : 2;
  static constexpr int THREADS = 256 + 128 * NT;
  // stages of K, of staged V codes and of V as f16
  static constexpr int KST = D == 128 ? 4 : TERMS == 2 ? 3 : 2, RST = D == 128 ? 3 : TERMS == 2 ? 2 : 1, VST = D == 128 ? 3 : 2;
  static constexpr int QTERM = 128 * D, QTILE = TERMS * QTERM;  // one row tile's e4m3 term; all its terms
  static constexpr int RAW = BN * D, VTILE = 2 * RAW;           // a tile's codes; V as f16
  static constexpr int K_OFF = NT * QTILE, R_OFF = K_OFF + KST * RAW, V_OFF = R_OFF + RST * RAW, SC_OFF = V_OFF + VST * VTILE;
  static constexpr int SC_SLOTS = 8, SC_BYTES = SC_SLOTS * (BN / 16) * 16;  // a tile's float4 per 16 tokens
  static constexpr int BAR_OFF = SC_OFF + SC_BYTES;
  static constexpr int NBARS = 14 + 2 * KST + 2 * RST + 2 * VST;
  static constexpr int MISC_OFF = BAR_OFF + NBARS * 8;
  static constexpr int SMEM = MISC_OFF + 16;
  // a slot is written again once K's stage is free, S of KST tiles before: then
  // the softmax of two tiles before that one is over
  static_assert(SC_SLOTS >= KST + 2, "scale slots");
  static_assert(SMEM <= 232448, "shared memory of a CTA");
  static constexpr int TMEM_COLS = 512;
  static constexpr int O_COL = 256;
};

// byte offset of 16-byte unit u of row r in a [rows][128 bytes] swizzled block
__device__ __forceinline__ uint32_t unit_offset(uint32_t r, uint32_t u) { return r * 128 + ((u ^ (r & 7)) << 4); }

// 8 values -> TERMS rows of e4m3 codes, each the rounded rest of those before
// (exact differences; NaN stays NaN in the first)
template <int TERMS>
__device__ __forceinline__ void split_terms(float2* v, uint2* out) {
#pragma unroll
  for (int k = 0; k < TERMS; ++k) {
    uint16_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = f2_to_e4m3x2(v[i].x, v[i].y);
      const float2 f = e4m3x2_to_f2(c[i]);
      v[i] = fadd2(v[i], make_float2(-f.x, -f.y));
    }
    out[k] = make_uint2(c[0] | ((uint32_t)c[1] << 16), c[2] | ((uint32_t)c[3] << 16));
  }
}

// 2^x of two values, x <= 15, without the special-function unit: x = n + f with
// |f| <= 1/2 (adding 1.5 * 2^23 rounds to n, in the low bits), 2^f by the
// degree-4 polynomial through the Chebyshev nodes of [-1/2, 1/2] (relative
// error 4e-6, under P's 2^-11), n into the exponent field. Below 2^-125 it
// gives 2^-125, which is 0 in f16.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  const float2 magic = make_float2(12582912.f, 12582912.f), down = make_float2(-12582912.f, -12582912.f);
  x = make_float2(fmaxf(x.x, -125.f), fmaxf(x.y, -125.f));
  const float2 t = fadd2(x, magic), n = fadd2(t, down), f = fadd2(x, make_float2(-n.x, -n.y));
  auto c = [](float v) { return make_float2(v, v); };
  float2 p = ffma2(f, c(0.009666369f), c(0.055921976f));
  p = ffma2(p, f, c(0.240223490f));
  p = ffma2(p, f, c(0.693121045f));
  p = ffma2(p, f, c(1.000000000f));
  return make_float2(__int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                     __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
}

// the largest of three; NaN if one is
__device__ __forceinline__ float nan_max3(float x, float y, float z) {
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(x), "f"(y), "f"(z));
  return m;
}

// two packed 16-bit values
__device__ __forceinline__ float2 up2(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 up2(__half2 v) { return __half22float2(v); }
template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  typedef __half2 type;
};
template <>
struct Pair<__nv_bfloat16> {
  typedef __nv_bfloat162 type;
};

template <typename T, int D>
__global__ void __launch_bounds__(Cfg<T, D>::THREADS, 1)
    block_attn_kernel(const __grid_constant__ mj_block_attn_args a, int lg, const __grid_constant__ CUtensorMap tmk,
                      const __grid_constant__ CUtensorMap tmv) {
  using C = Cfg<T, D>;
  constexpr int NT = C::NT, BN = C::BN, KST = C::KST, RST = C::RST, VST = C::VST;
  extern __shared__ __align__(1024) unsigned char sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::BAR_OFF);
  // s_full, p_full and o_full: [row tile][key tile & 1]
  uint64_t *s_full = bars, *p_full = bars + 4, *o_full = bars + 8, *q_full = bars + 12, *drain = bars + 13,
           *k_full = bars + 14, *k_empty = k_full + KST, *r_full = k_empty + KST, *r_empty = r_full + RST,
           *v_full = r_empty + RST, *v_empty = v_full + VST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + C::MISC_OFF + 4);
  int& never_abort = *reinterpret_cast<int*>(sm + C::MISC_OFF + 8);
  volatile int* nan_v = reinterpret_cast<volatile int*>(sm + C::MISC_OFF + 12);
  if (reinterpret_cast<uintptr_t>(sm) & 1023) {  // uniform: nothing taken yet
    if (threadIdx.x == 0) flag(a.status, MJ_DEV_BAD_SPLIT);
    return;
  }
  griddep_wait();
  const int4* item = reinterpret_cast<const int4*>(a.work) + 2 * (blockIdx.x / a.h_k);
  const int h = blockIdx.x % a.h_k;
  const int4 it0 = item[0];
  if (it0.x < 0 || it0.x >= a.num_seqs) {
    if (threadIdx.x == 0) flag(a.status, MJ_DEV_BAD_SPLIT);
    return;
  }
  const int seq = it0.x, row0 = it0.y, tb = it0.z, slot = item[1].x;
  const int h_r = a.h_q / a.h_k;
  const int q0 = a.q_start[seq], n_tok = a.q_start[seq + 1] - q0, L = a.seq_lens[seq];
  const int n_rows = n_tok * h_r;
  if (row0 < 0 || row0 >= n_rows || q0 < 0 || n_tok < 0 || q0 + (int64_t)n_tok > a.num_tokens || slot >= a.num_slots ||
      tb < 0 || it0.w > INT_MAX / BN - 2) {
    if (threadIdx.x == 0) flag(a.status, MJ_DEV_BAD_SPLIT);  // uniform: nothing taken yet
    return;
  }
  const int n = max(it0.w - tb, 0);  // key tiles
  const int na = NT == 1 || row0 + 128 < n_rows ? NT : 1;  // row tiles with rows in them

  if (threadIdx.x == 0) {
    for (int i = 0; i < KST; ++i) {
      mbar_init(&k_full[i], 2);  // K's copies, and the tile's scales
      mbar_init(&k_empty[i], na);
    }
    for (int i = 0; i < RST; ++i) {
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], 128);
    }
    for (int i = 0; i < VST; ++i) {
      mbar_init(&v_full[i], 128);
      mbar_init(&v_empty[i], na);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 2);  // the product, and its issuer (who saw the tile's scales)
      mbar_init(&p_full[i], 128);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(q_full, 128 * na);
    mbar_init(drain, na);
    *abort_flag = 0;
    never_abort = 0;
    *nan_v = 0;
    fence_mbar_init();
  }
  if (warp == 1 && lane == 0) {
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // all 512 columns, so the base is column 0, and TMEM addresses are constants
  if (*tmem_slot != 0) {  // uniform, and cannot happen
    if (threadIdx.x == 0) flag(a.status, MJ_DEV_BAD_SPLIT);
    if (warp == 0) tmem_dealloc(*tmem_slot, C::TMEM_COLS);
    return;
  }
  auto give_up = [&]() {
    *abort_flag = 1;
    flag(a.status, MJ_DEV_TIMEOUT);
  };
  auto wait = [&](uint64_t* bar, int phase) {
    if (mbar_wait(bar, (uint32_t)phase & 1u, abort_flag, kWaitNs)) return true;
    if (!*abort_flag) give_up();
    return false;
  };
  // S of row tile w for key tile j, with P over its first half; the index and
  // phase of that pair's barriers
  auto s_col = [&](int w, int j) { return (uint32_t)(w * 128 + (j & 1) * BN); };
  auto at = [&](int w, int j) { return 2 * w + (j & 1); };

  // The first key tile that some row of the item sees only part of. From there
  // on NaN codes of V reach the product as zeros (P = 0 times NaN would be NaN
  // in the rows that do not see them), and if there was one, the epilogue makes
  // those elements NaN in the rows that do.
  const int item_lim = a.causal ? L - n_tok + row0 / h_r : L - 1;
  const int j_part = max(item_lim + 1 - tb * BN, 0) / BN;

  // Page-table walk. An entry is loaded before it is needed and checked then:
  // checking it at once would wait a memory round trip.
  constexpr int kNone = INT_MIN;  // past the sequence or the item
  const int base = tb * BN, pmask = a.page_size - 1;
  auto entry_of = [&](int pos) -> int {
    if (pos >= L || pos >= base + n * BN) return kNone;
    const int c = pos >> (31 - __clz(a.page_size));
    return c < a.block_table_cols ? __ldg(a.block_table + seq * a.block_table_stride + c) : -1;
  };
  auto page_of = [&](int e) -> int {  // -1: no such token, or a bad entry
    if ((unsigned)e < (unsigned)a.num_pages) return e;
    if (e != kNone) flag(a.status, MJ_DEV_BAD_PAGE);
    return -1;
  };

  // Producer loop over one operand's ring: `before`, wait for the stage, then a
  // TMA box per page. Lane i < pages holds the table entry of the tile's page i
  // (a page may be larger than a tile: then the only box is a part of one).
  auto produce = [&](const CUtensorMap& map, int off, int stages, uint64_t* full, uint64_t* empty, auto before) {
    const uint64_t policy = l2_policy_evict_normal();  // other row blocks read the same keys
    const int ps = a.page_size, pages = max(BN / ps, 1), rows = min(ps, BN);
    auto entries = [&](int j) { return lane < pages ? entry_of(base + j * BN + lane * ps) : kNone; };
    int next = n > 0 ? entries(0) : kNone, j = 0;
    bool ok = true;
    for (; j < n; ++j) {
      // an absent page is read out of range: the TMA fills zeros
      const int page = page_of(next), where = page < 0 ? (int)a.num_pages : page;
      const int row = ps > BN ? (base + j * BN) & pmask : 0, s = j % stages;
      next = entries(j + 1);
      ok = before(j) && __all_sync(0xffffffffu, wait(&empty[s], j / stages + 1));
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(&full[s], C::RAW);
      __syncwarp();
      if (lane < pages) {
#pragma unroll
        for (int dh = 0; dh < D / 128; ++dh)
          tma_load_5d(sm + off + s * C::RAW + dh * (BN * 128) + lane * rows * 128, &map, &full[s], 0, dh, row, h, where, policy);
      }
    }
    if (!ok)  // copies in flight land before the CTA exits
      for (int i = max(j - stages, 0); i < j; ++i) mbar_wait(&full[i % stages], (i / stages) & 1, &never_abort, kWaitNs);
  };

  if (warp < 4) {
    const int w = warp >> 1;
    if (!(warp & 1) && w < na) {
      // --------------------------------------------------- MMAs of row tile w
      // (the whole warp runs the loop, one lane issues: see elect_one)
      const bool lead = elect_one();
      const uint64_t q = smem_desc_sw128(smem_addr(sm + w * C::QTILE), 16, 1024);
      auto scores = [&](int j) -> bool {  // every term of Q against the same K; 32 head-dim elements a step
        constexpr uint32_t idesc = idesc_f8f6f4(0, 0, 0, 0, BN);
        bool ok = wait(&k_full[j % KST], j / KST);
        // S goes over the P of tile j - 2, and MMAs of two kinds are not ordered
        // with each other: that product has to be complete
        if (j > 1) ok = ok && wait(&o_full[at(w, j)], (j - 2) >> 1);
        if (!__all_sync(0xffffffffu, ok)) return false;
        tc_fence_after();
        const uint64_t k = smem_desc_sw128(smem_addr(sm + C::K_OFF + (j % KST) * C::RAW), 16, 1024);
        if (lead) {
#pragma unroll
          for (int i = 0; i < C::TERMS * (D / 32); ++i) {
            const int term = i / (D / 32), dh = i % (D / 32) / 4, x = i % 4;
            mma_f8f6f4(s_col(w, j), q + term * (C::QTERM / 16) + dh * (128 * 8) + x * 2, k + dh * (BN * 8) + x * 2, idesc, i > 0);
          }
          mma_commit(&s_full[at(w, j)]);
          mbar_arrive(&s_full[at(w, j)]);
          mma_commit(&k_empty[j % KST]);
        }
        return true;
      };
      bool ok = n > 0 && __all_sync(0xffffffffu, wait(q_full, 0)) && scores(0);
      for (int j = 0; ok && j < n; ++j) {
        if (j + 1 < n) ok = scores(j + 1);
        ok = ok && wait(&v_full[j % VST], j / VST) && wait(&p_full[at(w, j)], j >> 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const uint64_t v = smem_desc_sw128(smem_addr(sm + C::V_OFF + (j % VST) * C::VTILE), BN * 128, 1024);
        if (lead) {  // 16 tokens a step: two 8-row atoms of V, 8 columns of P
          constexpr uint32_t idesc = idesc_f16(0, 1, D);
#pragma unroll
          for (int i = 0; i < BN / 16; ++i)
            mma_f16_ts(C::O_COL + w * 128, s_col(w, j) + i * 8, v + i * 128, idesc, j > 0 || i > 0);
          mma_commit(&o_full[at(w, j)]);
          mma_commit(&v_empty[j % VST]);
        }
      }
      if (lead) mma_commit(drain);  // all issued MMAs complete before TMEM is released
      mbar_wait(drain, 0, &never_abort, kWaitNs);
    } else if (warp == 1) {
      // ------------------------------------------------------------ producer: K
      produce(tmk, C::K_OFF, KST, k_full, k_empty, [](int) { return true; });
    } else if (warp == 3) {
      // -------------------------------------------------- producer: V and scales
      // Block scales of the tile's 16-token groups: lane i < BN / 16 looks the
      // page up two tiles ahead and reads the two exponents one tile ahead
      // (into registers that nothing combines before their tile: a use of them
      // would wait the memory round trip). They go with K's stage.
      auto group_entry = [&](int j) { return lane < BN / 16 ? entry_of(base + j * BN + lane * 16) : kNone; };
      unsigned char next_k = 127, next_v = 127;
      auto exponents = [&](int j, int p) {
        next_k = next_v = 127;
        if (p < 0) return;
        const int b = ((base + j * BN + lane * 16) & pmask) >> lg;
        next_k = __ldg(static_cast<const unsigned char*>(a.k_scales) + p * a.ks_stride_page + b * a.ks_stride_block + h * a.ks_stride_head);
        next_v = __ldg(static_cast<const unsigned char*>(a.v_scales) + p * a.vs_stride_page + b * a.vs_stride_block + h * a.vs_stride_head);
      };
      int sc_entry = kNone;
      if (n > 0) {
        const int e0 = group_entry(0);
        sc_entry = group_entry(1);
        exponents(0, page_of(e0));
      }
      produce(tmv, C::R_OFF, RST, r_full, r_empty, [&](int j) {
        if (!__all_sync(0xffffffffu, wait(&k_empty[j % KST], j / KST + 1))) return false;
        if (lane < BN / 16) {
          const int e = block_e(next_v);
          reinterpret_cast<float4*>(sm + C::SC_OFF)[(j % C::SC_SLOTS) * (BN / 16) + lane] =
              make_float4(block_scale(next_k), (float)(e - 127), __uint_as_float((uint32_t)(254 - e) << 23), 0.f);
        }
        __syncwarp();  // the scales are written before lane 0 arrives
        if (lane == 0) mbar_arrive(&k_full[j % KST]);
        exponents(j + 1, page_of(sc_entry));
        sc_entry = group_entry(j + 2);
        return true;
      });
    }
    __syncwarp();
  } else if (warp < 8) {
    // ------------------------------------------------------- converter warpgroup
    const int ct = threadIdx.x - 128;
    // Thread ct takes 16-code chunk 4 blk + quad of rows r0, r0 + STEP, ...:
    // eight neighbouring threads are four chunks of a 64-element block in rows
    // r and r ^ 5, so that both their staged reads (swizzled 16-byte chunks of
    // 16 codes) and their stores (of 8 f16) cover all banks.
    constexpr int BLOCKS = D / 64, STEP = 32 / BLOCKS, NC = BN / STEP;
    const int quad = ct & 3, blk = (ct >> 3) % BLOCKS, pr = (ct >> 3) / BLOCKS;
    const int r0 = ((pr & 3) ^ ((ct >> 2) & 1 ? 5 : 0)) + (pr & ~3) * 2;
    auto convert = [&](int j) -> bool {
      const int rows = L - (base + j * BN);  // from there on zeros: unwritten rows may hold NaN codes
      if (!wait(&r_full[j % RST], j / RST)) return false;
      const unsigned char* raw = sm + C::R_OFF + (j % RST) * C::RAW + (blk >> 1) * (BN * 128);
      uint4 d[NC];
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int r = r0 + i * STEP;
        d[i] = *reinterpret_cast<const uint4*>(raw + unit_offset(r, 4 * (blk & 1) + quad));
        if (r >= rows) d[i] = make_uint4(0, 0, 0, 0);
      }
      if (j >= j_part) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < NC; ++i) any |= drop_nan_codes(d[i]);
        if (any) *nan_v = 1;  // before this tile's arrival on v_full
      }
      if (!wait(&v_empty[j % VST], j / VST + 1)) return false;
      unsigned char* out = sm + C::V_OFF + (j % VST) * C::VTILE + blk * (BN * 128);
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const uint32_t w[4] = {d[i].x, d[i].y, d[i].z, d[i].w};
        uint32_t o[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[2 * k] = e4m3x2_to_h2((uint16_t)w[k]);
          o[2 * k + 1] = e4m3x2_to_h2((uint16_t)(w[k] >> 16));
        }
        *reinterpret_cast<uint4*>(out + unit_offset(r0 + i * STEP, 2 * quad)) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(out + unit_offset(r0 + i * STEP, 2 * quad + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
      }
      // the staging tile is free once every value read from it went through the
      // stores above: arriving before them let the compiler move reads behind it
      mbar_arrive(&r_empty[j % RST]);
      fence_proxy_async_smem();
      mbar_arrive(&v_full[j % VST]);
      return true;
    };
    for (int j = 0; j < n; ++j)
      if (!convert(j)) break;
  } else {
    // ------------------------------------------------------- softmax warpgroups
    const int w = (warp - 8) >> 2, t = threadIdx.x & 127;
    if (w < na) {
      const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
      const int R = row0 + w * 128 + t;
      const bool live = R < n_rows;
      const int tok = min(R, n_rows - 1) / h_r, hq = h * h_r + min(R, n_rows - 1) % h_r;
      const int lim = !live ? -1 : a.causal ? L - n_tok + tok : L - 1;  // the last key this row sees
      // the first row of the warp sees the fewest keys
      const int warp_lim = __shfl_sync(0xffffffffu, lim, 0);
      // ---- Q: the warp's rows in TERMS e4m3 terms into the K-major tiles. D / 8
      // lanes read a row, eight reads of each lane in flight; the row's owner
      // hands its address round and gets its power of two back.
      float c2 = a.softmax_scale * kLog2e;
      {
        typedef typename Pair<T>::type T2;
        constexpr int LPR = D / 8, RPI = 32 / LPR, BATCH = 8;  // lanes of a row, rows of a pass, passes in flight
        const int c = lane % LPR, wr = (warp & 3) * 32;
        const int64_t q_off = (int64_t)(q0 + tok) * a.q_stride_tok + hq * a.q_stride_head;
        unsigned char* qs = sm + w * C::QTILE;
        int mine = 0;  // the power of two of this thread's row
#pragma unroll 1
        for (int i0 = 0; i0 < 32 / RPI; i0 += BATCH) {
          uint4 raw[BATCH];
#pragma unroll
          for (int i = 0; i < BATCH; ++i)
            raw[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) +
                                                     __shfl_sync(0xffffffffu, q_off, (i0 + i) * RPI + lane / LPR) + 8 * c);
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            const int lr = wr + (i0 + i) * RPI + lane / LPR;  // row of the tile
            const T2* e = reinterpret_cast<const T2*>(&raw[i]);
            const float2 m2 = up2(__hmax2(__hmax2(__habs2(e[0]), __habs2(e[1])), __hmax2(__habs2(e[2]), __habs2(e[3]))));
            float amax = fmaxf(m2.x, m2.y);  // NaN elements do not count
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            // 2^k with amax 2^k in [128, 256), inside fp32's normal range; a row
            // with an infinity has no finite output and becomes NaN
            const int k = amax > 0.f ? min(max(134 - (int)(__float_as_uint(amax) >> 23), -126), 126) : 0;
            const float up = amax == INFINITY ? __int_as_float(0x7FFFFFFF) : __uint_as_float((uint32_t)(127 + k) << 23);
            float2 v[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) v[x] = fmul2(up2(e[x]), make_float2(up, up));
            uint2 terms[C::TERMS];
            split_terms<C::TERMS>(v, terms);
#pragma unroll
            for (int x = 0; x < C::TERMS; ++x)
              *reinterpret_cast<uint2*>(qs + x * C::QTERM + (c >> 4) * (128 * 128) + unit_offset(lr, (c >> 1) & 7) + (c & 1) * 8) = terms[x];
            const int got = __shfl_sync(0xffffffffu, k, (lane % RPI) * LPR);  // row i * RPI + lane % RPI
            if (lane / RPI == i0 + i) mine = got;
          }
        }
        c2 *= __uint_as_float((uint32_t)(127 - mine) << 23);
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      }
      // nm: minus the running maximum; a row that sees no key of the first tile
      // sees none at all (keys are a prefix) and keeps P = 0. l: the row sum.
      float nm = 0.f, l = 0.f;
      bool ok = true;
      const uint32_t o_addr = C::O_COL + w * 128 + lane_base;
      for (int j = 0; j < n; ++j) {
        ok = wait(&s_full[at(w, j)], j >> 1);
        // every thread leaves the loop with its warp: the TMEM loads are collective
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t s_addr = s_col(w, j) + lane_base;
        float2 s[BN / 2];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) tmem_ld32(s_addr + 32 * c, reinterpret_cast<float*>(s) + 32 * c);
        tmem_wait_ld();
        const float4* sc = reinterpret_cast<const float4*>(sm + C::SC_OFF) + (j % C::SC_SLOTS) * (BN / 16);
#pragma unroll
        for (int g = 0; g < BN / 16; ++g) {
          const float4 f = sc[g];
          const float2 m2 = make_float2(c2 * f.x, c2 * f.x), b2 = make_float2(f.y + nm, f.y + nm);
#pragma unroll
          for (int i = 0; i < 8; ++i) s[8 * g + i] = ffma2(s[8 * g + i], m2, b2);
        }
        const int j0 = (tb + j) * BN;
        if (j0 + BN - 1 > warp_lim) {  // some row of the warp sees only some of these keys
#pragma unroll
          for (int i = 0; i < BN / 2; ++i) {
            if (j0 + 2 * i > lim) s[i].x = -INFINITY;
            if (j0 + 2 * i + 1 > lim) s[i].y = -INFINITY;
          }
        }
        float mx4[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) mx4[i] = s[i].x;
#pragma unroll
        for (int i = 4; i < BN / 2; ++i) mx4[i & 3] = nan_max3(mx4[i & 3], s[i].x, s[i - 4].y);
#pragma unroll
        for (int i = 0; i < 4; ++i) mx4[i] = nan_max3(mx4[i], s[BN / 2 - 4 + i].y, mx4[0]);
        float mx = nan_max3(mx4[1], mx4[2], mx4[3]);
        if (__any_sync(0xffffffffu, j == 0 || !(mx <= kRaise))) {
          if (isnan(mx)) l = mx;  // a NaN score: so is the row (exp2_poly would lose it)
          const float up = (j == 0 ? mx > -INFINITY : mx > kRaise) ? -mx : 0.f;  // added to nm
          nm += up;
#pragma unroll
          for (int i = 0; i < BN / 2; ++i) s[i] = fadd2(s[i], make_float2(up, up));
          if (j > 0) {  // O and l follow, once the last product has landed
            const float f = exp2_approx(up);
            l *= f;
            ok = __all_sync(0xffffffffu, wait(&o_full[at(w, j - 1)], (j - 1) >> 1));
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              float o[16];
              tmem_ld16(o_addr + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= f;
              tmem_st16(o_addr + c, reinterpret_cast<const uint32_t*>(o));
            }
          }
        }
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) {  // 32 keys: 16 columns of P
          uint32_t p[16];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 d = s[16 * c + 8 * g + i];
              const float2 e = i % 4 < kPolyOf4 ? exp2_poly(d) : make_float2(exp2_approx(d.x), exp2_approx(d.y));
              sum = fadd2(sum, e);
              p[8 * g + i] = f2_to_h2(e.x, e.y);
            }
            l = fmaf(sum.x + sum.y, sc[2 * c + g].z, l);
          }
          tmem_st16(s_addr + 16 * c, p);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[at(w, j)]);
      }
      // ---- epilogue: O / l of this row
      // Staging below goes over the Q tile, whose rows other warps write too. The
      // last product is behind all of them; without a key tile there is none.
      if (n == 0) ok = wait(q_full, 0);
      if (ok && n > 0) ok = wait(&o_full[at(w, n - 1)], (n - 1) >> 1);
      if (ok && n > 0) ok = wait(&v_full[(n - 1) % VST], (n - 1) / VST);  // long complete: orders the read of nan_v
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      if (ok) {
        const bool nans = *nan_v != 0;
        if (lim < base) l = 0.f;  // no key in this item (exp2_poly's zero is 2^-125)
        const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN sum stays NaN
        const int64_t part = ((int64_t)slot * a.h_k + h) * C::ROWS + w * 128 + t;
        const int64_t o_off = (int64_t)(q0 + tok) * a.o_stride_tok + hq * a.o_stride_head;
        // final rows go through shared memory (this warp's part of the Q tile,
        // which no MMA reads any more), so that D / 8 lanes write a row
        constexpr int LPR = D / 8, RPI = 32 / LPR;
        unsigned char* stage = sm + w * C::QTILE + (warp & 3) * (32 * D * 2);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float v[32];
          if (n > 0) {
            tmem_ld32(o_addr + c, v);
            tmem_wait_ld();
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = l == 0.f ? 0.f : v[i] * inv;
          if (nans)  // rare
#pragma unroll 1
            for (int key = base + j_part * BN; key <= min(lim, base + n * BN - 1); ++key) {
              const int pg = page_of(entry_of(key));
              if (pg < 0) continue;
              const uint32_t* code = reinterpret_cast<const uint32_t*>(static_cast<const unsigned char*>(a.v_cache) + pg * a.v_stride_page +
                                                                       (key & pmask) * a.v_stride_row + h * a.v_stride_head + c);
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (nan_codes(__ldg(code + i / 4)) >> (8 * (i % 4)) & 0x80u) v[i] = __int_as_float(0x7FFFFFFF);
            }
          if (slot < 0) {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              store8(reinterpret_cast<T*>(stage + lane * (D * 2) + ((((c + i) >> 3) ^ (lane & 7)) << 4)), v + i);
          } else if (live) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) store8(a.o_part + part * D + c + i, v + i);
          }
          __syncwarp();  // the TMEM load is a whole-warp operation
        }
        if (slot < 0) {
          const int rows_here = min(max(n_rows - (row0 + w * 128 + (warp & 3) * 32), 0), 32);
#pragma unroll 4
          for (int i = 0; i < 32 / RPI; ++i) {
            const int r = i * RPI + lane / LPR;
            const int64_t at_row = __shfl_sync(0xffffffffu, o_off, r);
            const uint4 x = *reinterpret_cast<const uint4*>(stage + r * (D * 2) + (((lane % LPR) ^ (r & 7)) << 4));
            if (r < rows_here) *reinterpret_cast<uint4*>(static_cast<T*>(a.o) + at_row + 8 * (lane % LPR)) = x;
          }
        }
        if (live) {
          const float lse = l == 0.f ? -INFINITY : (log2f(l) - nm) * kLn2;
          if (slot >= 0) a.lse_part[part] = lse;
          else if (a.lse) a.lse[(int64_t)(q0 + tok) * a.h_q + hq] = lse;
        }
      }
      tc_fence_before();
    }
  }
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(0, C::TMEM_COLS);
  }
}

// Joins the partials of one row: weights e^(lse - max), a warp per row.
template <typename T, int D>
__global__ void __launch_bounds__(256) block_merge_kernel(const __grid_constant__ mj_block_attn_args a) {
  griddep_wait();
  constexpr int ROWS = MJ_BLOCK_ROWS(D), E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t wi = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) >> 5;
  const int r = (int)(wi % ROWS), h = (int)(wi / ROWS % a.h_k);
  const int64_t m = wi / ROWS / a.h_k;
  if (m >= a.num_merges) return;
  const int4 e = reinterpret_cast<const int4*>(a.merges)[m];
  if (e.w <= 0) return;
  if (e.x < 0 || e.x >= a.num_seqs || e.y < 0 || e.z < 0 || e.w > a.num_slots - e.z) {  // uniform in the warp
    if (lane == 0) flag(a.status, MJ_DEV_BAD_SPLIT);
    return;
  }
  const int h_r = a.h_q / a.h_k, q0 = a.q_start[e.x], n_tok = a.q_start[e.x + 1] - q0;
  if (q0 < 0 || n_tok < 0 || q0 + (int64_t)n_tok > a.num_tokens) {
    if (lane == 0) flag(a.status, MJ_DEV_BAD_SPLIT);
    return;
  }
  if (r >= n_tok * h_r - e.y) return;
  const int64_t step = (int64_t)a.h_k * ROWS, first = ((int64_t)e.z * a.h_k + h) * ROWS + r;
  float mx = -INFINITY;
  for (int s = 0; s < e.w; ++s) mx = nan_max(mx, a.lse_part[first + s * step]);  // a NaN partial makes its row NaN
  float o[E], l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  if (mx != -INFINITY) {
    for (int s = 0; s < e.w; ++s) {
      const float w = __expf(a.lse_part[first + s * step] - mx);
      l += w;
      const float4* p = reinterpret_cast<const float4*>(a.o_part + (first + s * step) * D) + lane;
#pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        const float4 v = p[32 * i];
        o[4 * i] = fmaf(w, v.x, o[4 * i]);
        o[4 * i + 1] = fmaf(w, v.y, o[4 * i + 1]);
        o[4 * i + 2] = fmaf(w, v.z, o[4 * i + 2]);
        o[4 * i + 3] = fmaf(w, v.w, o[4 * i + 3]);
      }
    }
  }
  const int R = e.y + r, hq = h * h_r + R % h_r;
  const int64_t tok = q0 + R / h_r;
  T* out = static_cast<T*>(a.o) + tok * a.o_stride_tok + hq * a.o_stride_head;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < E; ++i) out[128 * (i / 4) + 4 * lane + i % 4] = (T)(o[i] * inv);
  if (a.lse && lane == 0) a.lse[tok * a.h_q + hq] = l == 0.f ? -INFINITY : mx + logf(l);
}

constexpr int kMaxDevices = 64;

// One operand's codes as (128 codes, 128-code halves of a row, page rows, KV
// heads, pages), boxes of one page's rows (or a tile's, where a page is larger).
static bool make_map(CUtensorMap* m, const void* base, int64_t s_page, int64_t s_row, int64_t s_head,
                     const mj_block_attn_args& a) {
  auto fn = tensor_map_encoder();
  if (!fn) return false;
  // a dimension of extent 1 never moves its coordinate: any legal stride
  const cuuint64_t sr = s_row ? s_row : 16, sh = s_head ? s_head : 16, sp = s_page ? s_page : 16;
  const int keys = MJ_BLOCK_KEYS, rows = a.page_size < keys ? a.page_size : keys;
  cuuint64_t dims[5] = {128, (cuuint64_t)(a.head_size / 128), (cuuint64_t)a.page_size, (cuuint64_t)a.h_k, (cuuint64_t)a.num_pages};
  cuuint64_t strides[4] = {128, sr, sh, sp};
  cuuint32_t box[5] = {128, 1, (cuuint32_t)rows, 1, 1}, estr[5] = {1, 1, 1, 1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
static cudaError_t launch_t(const mj_block_attn_args& a, cudaStream_t stream) {
  using C = Cfg<T, D>;
  auto kern = block_attn_kernel<T, D>;
  static std::atomic<int> ready[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!ready[dev].load(std::memory_order_acquire)) {
    std::lock_guard<std::mutex> lock(tc_init_mutex());
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) != cudaSuccess) return e;
    ready[dev].store(1, std::memory_order_release);
  }
  if (a.num_work) {
    CUtensorMap mk, mv;
    if (!make_map(&mk, a.k_cache, a.k_stride_page, a.k_stride_row, a.k_stride_head, a) ||
        !make_map(&mv, a.v_cache, a.v_stride_page, a.v_stride_row, a.v_stride_head, a))
      return cudaErrorInvalidValue;
    e = launch_kernel(kern, dim3((unsigned)(a.num_work * a.h_k)), dim3(C::THREADS), C::SMEM, stream, a, block_log2(a.kv_format), mk, mv);
    if (e != cudaSuccess) return e;
  }
  if (a.num_merges) {
    const int64_t warps = (int64_t)a.num_merges * a.h_k * C::ROWS;
    return launch_kernel(block_merge_kernel<T, D>, dim3((unsigned)((warps + 7) / 8)), dim3(256), 0, stream, a);
  }
  return cudaSuccess;
}

}  // namespace ba

cudaError_t launch_block_attention(const mj_block_attn_args& a, cudaStream_t stream) {
  if (a.dtype == MJ_DT_FP16)
    return a.head_size == 256 ? ba::launch_t<__half, 256>(a, stream) : ba::launch_t<__half, 128>(a, stream);
  return a.head_size == 256 ? ba::launch_t<__nv_bfloat16, 256>(a, stream) : ba::launch_t<__nv_bfloat16, 128>(a, stream);
}

}  // namespace mj
