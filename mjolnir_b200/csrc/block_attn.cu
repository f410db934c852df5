// Attention of ragged query chunks over the block-scaled cache on the
// 5th-generation tensor cores (sm_100a).
//
// A CTA takes one work item of one KV head: NT tiles of 128 rows -- a row is
// (query token, head of the KV head's group), so a group shares every key read
// -- and a range of key tiles of BN tokens. Warp roles:
//   converter warpgroup  page-table walk, 16-byte code loads one operand ahead
//                        in registers, e4m3 -> f16 (exact), 128-byte swizzled
//                        K (K-major) and V (MN-major) tiles in two-stage rings;
//                        also the tile's block scales
//   MMA thread           S = Q K^T (both from shared memory), O += P V (P from
//                        TMEM, over the columns of the S it came from)
//   NT softmax warpgroups  thread = row: S to registers, online softmax in base
//                        2, P back to TMEM as f16
// With NT = 2 the tiles take turns: while one is in its softmax the tensor
// cores run the other's products. With NT = 1 (head_size 256, whose O takes
// half of TMEM) S is double-buffered and the next tile's product runs instead.
//
// Scales: score_ij = c 2^ek_j (q_i . kcode_j), and V's scale is folded into the
// exponent: z_ij = score_ij + ev_j (base 2), P' = 2^(z - m), O = sum P' vcode /
// sum P' 2^-ev. The running maximum m is thus over what enters O, so a large V
// scale cannot push the other rows' P out of f16's range. m moves lazily, when
// a z exceeds it by 2^8; P' keeps 2^6 of headroom above m so that f16 holds
// values down to 2^-31 of the maximum.
// Q enters as f16: exact for f16; a bf16 row is scaled by a power of two that
// puts its largest element into [2^14, 2^15), so elements down to 2^-31 of it
// are exact.
//
// Every mbarrier wait is bounded; on a timeout the CTA flags MJ_DEV_TIMEOUT,
// all roles stop, the MMAs in flight complete and TMEM is freed.
#include <limits.h>
#include <math.h>

#include <atomic>
#include <mutex>

#include "block_cache.cuh"

namespace mj {

std::mutex& tc_init_mutex();

namespace ba {

using namespace sm100;

constexpr uint64_t kWaitNs = 500000000ull;  // per wait; a tile takes microseconds
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kHeadroom = 6.f;            // P' of the running maximum is 2^6
constexpr float kRaise = kHeadroom + 8.f;   // raise it when a P' would pass 2^14

template <int D>
struct Cfg {
  static constexpr int NT = D == 256 ? 1 : 2;
  static constexpr int BN = MJ_BLOCK_KEYS(D);
  static constexpr int ROWS = NT * 128;
  static_assert(ROWS == MJ_BLOCK_ROWS(D), "the plan's rows");
  static constexpr int THREADS = 256 + 128 * NT;
  static constexpr int QTILE = 128 * D * 2, KTILE = BN * D * 2;
  static constexpr int K_OFF = NT * QTILE, V_OFF = K_OFF + 2 * KTILE, SC_OFF = V_OFF + 2 * KTILE;
  static constexpr int SC_BYTES = 4 * (BN / 16) * 16;  // four tiles' float4 per 16 tokens
  static constexpr int BAR_OFF = SC_OFF + SC_BYTES;
  static constexpr int NBARS = 8 + 4 + 2 + 2 + 4 + 2;
  static constexpr int MISC_OFF = BAR_OFF + NBARS * 8;
  static constexpr int SMEM = MISC_OFF + 64;
  static constexpr int TMEM_COLS = 512;
  static constexpr int O_COL = 256;
  // 512 threads share 65536 registers: the MMA warpgroup gives most of its up
  static constexpr int REG_MMA = NT == 2 ? 40 : 0, REG_CVT = NT == 2 ? 96 : 0, REG_SM = NT == 2 ? 184 : 0;
  static constexpr int REG_POOL = 128 * REG_MMA + 128 * REG_CVT + 128 * NT * REG_SM;
};

// byte offset of 16-byte unit u of row r in a [rows][64 f16] swizzled block
__device__ __forceinline__ uint32_t unit_offset(uint32_t r, uint32_t u) { return r * 128 + ((u ^ (r & 7)) << 4); }

template <typename T, int D>
__global__ void __launch_bounds__(Cfg<D>::THREADS, 1) block_attn_kernel(const __grid_constant__ mj_block_attn_args a, int lg) {
  using C = Cfg<D>;
  constexpr int NT = C::NT, BN = C::BN;
  extern __shared__ __align__(1024) unsigned char sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + C::BAR_OFF);
  uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6, *sc_full = bars + 8,
           *s_full = bars + 12, *p_full = bars + 14, *o_full = bars + 16, *q_full = bars + 20, *drain = bars + 21;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + C::MISC_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sm + C::MISC_OFF + 4);
  int& never_abort = *reinterpret_cast<int*>(sm + C::MISC_OFF + 8);
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
  if (row0 < 0 || row0 >= n_rows || q0 < 0 || q0 + (int64_t)n_tok > a.num_tokens || slot >= a.num_slots) {
    if (threadIdx.x == 0) flag(a.status, MJ_DEV_BAD_SPLIT);  // uniform: nothing taken yet
    return;
  }
  const int n = max(it0.w - tb, 0);  // key tiles
  const int na = NT == 1 || row0 + 128 < n_rows ? NT : 1;  // row tiles with rows in them

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 128);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 128);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 128);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&sc_full[i], 1);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(q_full, 128 * na);
    mbar_init(drain, 1);
    *abort_flag = 0;
    never_abort = 0;
    fence_mbar_init();
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
  // S of row tile w for key tile j (P over its first columns), and its barriers
  auto s_col = [&](int w, int j) { return (uint32_t)(NT == 2 ? w * 128 : (j & 1) * BN); };
  auto s_bar = [&](int w, int j) { return NT == 2 ? w : j & 1; };
  auto s_phase = [&](int j) { return NT == 2 ? j : j >> 1; };

  if (warp < 4) {
    if constexpr (C::REG_MMA > 0) setmaxnreg_dec<C::REG_MMA>();
    if (warp == 0) {
      // ------------------------------------------------------------ MMA issuer
      // (the whole warp runs the loop, one lane issues: see elect_one)
      const bool lead = elect_one();
      auto qk = [&](int w, int j) {  // 16 head-dim elements a step, 64 a swizzled block
        constexpr uint32_t idesc = idesc_f16(0, 0, BN);
        const uint64_t q = smem_desc_sw128(smem_addr(sm + w * C::QTILE), 16, 1024),
                       k = smem_desc_sw128(smem_addr(sm + C::K_OFF + (j & 1) * C::KTILE), 16, 1024);
        if (lead) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            mma_f16_ss(s_col(w, j), q + (i >> 2) * (128 * 8) + (i & 3) * 2, k + (i >> 2) * (BN * 8) + (i & 3) * 2, idesc, i > 0);
          mma_commit(&s_full[s_bar(w, j)]);
        }
      };
      auto pv = [&](int w, int j) {  // 16 tokens a step: two 8-row atoms of V, 8 columns of P
        constexpr uint32_t idesc = idesc_f16(0, 1, D);
        const uint64_t v = smem_desc_sw128(smem_addr(sm + C::V_OFF + (j & 1) * C::KTILE), BN * 128, 1024);
        if (lead) {
#pragma unroll
          for (int i = 0; i < BN / 16; ++i)
            mma_f16_ts(C::O_COL + w * 128, s_col(w, j) + i * 8, v + i * 128, idesc, j > 0 || i > 0);
          mma_commit(&o_full[2 * w + (j & 1)]);
        }
      };
      auto commit = [&](uint64_t* bar) {
        if (lead) mma_commit(bar);
      };
      bool ok = n > 0 && wait(q_full, 0) && wait(&k_full[0], 0);
      ok = __all_sync(0xffffffffu, ok);
      if (ok) {
        tc_fence_after();
        for (int w = 0; w < na; ++w) qk(w, 0);
        commit(&k_empty[0]);
      }
      for (int j = 0; ok && j < n; ++j) {
        const bool more = j + 1 < n;
        if (more) ok = __all_sync(0xffffffffu, wait(&k_full[(j + 1) & 1], (j + 1) >> 1));
        if (NT == 1 && ok && more) {
          tc_fence_after();
          qk(0, j + 1);
          commit(&k_empty[(j + 1) & 1]);
        }
        ok = ok && __all_sync(0xffffffffu, wait(&v_full[j & 1], j >> 1));
        for (int w = 0; ok && w < na; ++w) {
          ok = __all_sync(0xffffffffu, wait(&p_full[s_bar(w, j)], s_phase(j)));
          if (!ok) break;
          tc_fence_after();
          pv(w, j);
          if (w == na - 1) commit(&v_empty[j & 1]);
          if (NT == 2 && more) qk(w, j + 1);  // over S and P of tile j: behind its product, in issue order
        }
        if (NT == 2 && ok && more) commit(&k_empty[(j + 1) & 1]);
      }
      commit(drain);  // all issued MMAs complete before TMEM is released
      mbar_wait(drain, 0, &never_abort, kWaitNs);
    }
    __syncwarp();
  } else if (warp < 8) {
    // ------------------------------------------------------- converter warpgroup
    if constexpr (C::REG_CVT > 0) setmaxnreg_dec<C::REG_CVT>();
    const int ct = threadIdx.x - 128;
    constexpr int CPR = D / 16, STEP = 128 / CPR, NC = BN / STEP;  // 16-code chunks of a row; rows of a pass; passes
    const int col = ct % CPR, r0 = ct / CPR, base = tb * BN;
    const int32_t* table = a.block_table + seq * a.block_table_stride;
    const int ps_log2 = 31 - __clz(a.page_size), pmask = a.page_size - 1;
    const unsigned char* kbase = static_cast<const unsigned char*>(a.k_cache) + h * a.k_stride_head + col * 16;
    const unsigned char* vbase = static_cast<const unsigned char*>(a.v_cache) + h * a.v_stride_head + col * 16;
    // The table entry of token `pos` is loaded an operand before it is checked:
    // checking it at once would wait a memory round trip for every row.
    constexpr int kNone = INT_MIN;  // past the sequence
    const int last = base + n * BN;  // tokens from here on are not this item's
    auto entry_of = [&](int pos) -> int {
      if (pos >= L || pos >= last) return kNone;
      const int c = pos >> ps_log2;
      return c < a.block_table_cols ? __ldg(table + c) : -1;
    };
    auto page_of = [&](int e) -> int {  // -1: no such token, or a bad entry
      if ((unsigned)e < (unsigned)a.num_pages) return e;
      if (e != kNone) flag(a.status, MJ_DEV_BAD_PAGE);
      return -1;
    };
    // block scales of the tile's 16-token groups: thread ct < BN / 16 looks the
    // page up two tiles ahead and reads the two exponents one tile ahead
    constexpr uint32_t kOne = 127u | (127u << 8);
    const bool scaler = ct < BN / 16;
    auto exponents = [&](int pos, int p) -> uint32_t {
      if (p < 0) return kOne;
      const int b = (pos & pmask) >> lg;
      return __ldg(static_cast<const unsigned char*>(a.k_scales) + p * a.ks_stride_page + b * a.ks_stride_block + h * a.ks_stride_head) |
             ((uint32_t)__ldg(static_cast<const unsigned char*>(a.v_scales) + p * a.vs_stride_page + b * a.vs_stride_block + h * a.vs_stride_head) << 8);
    };
    uint4 data[NC];
    int page[NC];
    const uint4 zero = make_uint4(0, 0, 0, 0);
    auto load_k = [&](int pos, int p) { return p < 0 ? zero : __ldg(reinterpret_cast<const uint4*>(kbase + p * a.k_stride_page + (pos & pmask) * a.k_stride_row)); };
    auto load_v = [&](int pos, int p) { return p < 0 ? zero : __ldg(reinterpret_cast<const uint4*>(vbase + p * a.v_stride_page + (pos & pmask) * a.v_stride_row)); };
    // 16 codes -> two 16-byte units of f16; the threads of odd 64-column blocks
    // store their odd unit first, so that 8 threads of a row cover all banks
    const uint32_t block_at = (uint32_t)(col >> 2) * (BN * 128), unit = (uint32_t)(col & 3) * 2, odd = (uint32_t)(col >> 2) & 1;
    auto store = [&](unsigned char* buf, int r, uint4 d) {
      const uint32_t w[4] = {d.x, d.y, d.z, d.w};
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[2 * i] = e4m3x2_to_h2((uint16_t)w[i]);
        o[2 * i + 1] = e4m3x2_to_h2((uint16_t)(w[i] >> 16));
      }
      const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
      *reinterpret_cast<uint4*>(buf + block_at + unit_offset(r, unit + odd)) = odd ? hi : lo;
      *reinterpret_cast<uint4*>(buf + block_at + unit_offset(r, unit + 1 - odd)) = odd ? lo : hi;
    };
    int sc_entry = kNone;
    uint32_t sc_next = kOne;
    if (scaler) {
      const int e0 = entry_of(base + ct * 16);
      sc_entry = entry_of(base + BN + ct * 16);
      sc_next = exponents(base + ct * 16, page_of(e0));
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) page[i] = entry_of(base + r0 + i * STEP);
#pragma unroll
    for (int i = 0; i < NC; ++i) page[i] = page_of(page[i]);
#pragma unroll
    for (int i = 0; i < NC; ++i) data[i] = load_k(base + r0 + i * STEP, page[i]);
    for (int j = 0; j < n; ++j) {
      const int t0 = base + j * BN;
      if (scaler) {
        const int e = block_e((unsigned char)(sc_next >> 8));
        reinterpret_cast<float4*>(sm + C::SC_OFF)[(j & 3) * (BN / 16) + ct] =
            make_float4(block_scale((unsigned char)sc_next), (float)(e - 127), __uint_as_float((uint32_t)(254 - e) << 23), 0.f);
        sc_next = exponents(t0 + BN + ct * 16, page_of(sc_entry));
        sc_entry = entry_of(t0 + 2 * BN + ct * 16);
      }
      if (ct < 32) {
        __syncwarp();
        if (ct == 0) mbar_arrive(&sc_full[j & 3]);
      }
      if (!wait(&k_empty[j & 1], (j >> 1) + 1)) break;
      unsigned char* kb = sm + C::K_OFF + (j & 1) * C::KTILE;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int r = r0 + i * STEP;
        store(kb, r, data[i]);
        data[i] = load_v(t0 + r, page[i]);
        page[i] = entry_of(t0 + BN + r);
      }
      fence_proxy_async_smem();
      mbar_arrive(&k_full[j & 1]);
      if (!wait(&v_empty[j & 1], (j >> 1) + 1)) break;
      unsigned char* vb = sm + C::V_OFF + (j & 1) * C::KTILE;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        const int r = r0 + i * STEP;
        store(vb, r, data[i]);
        page[i] = page_of(page[i]);
        data[i] = load_k(t0 + BN + r, page[i]);
      }
      fence_proxy_async_smem();
      mbar_arrive(&v_full[j & 1]);
    }
  } else {
    if constexpr (C::REG_SM > 0) setmaxnreg_inc<C::REG_SM>();
    // ------------------------------------------------------- softmax warpgroups
    const int w = NT == 1 ? 0 : (warp - 8) >> 2;
    const int t = (threadIdx.x - 256) & 127;
    if (w < na) {
      const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
      const int R = row0 + w * 128 + t;
      const bool live = R < n_rows;
      const int tok = min(R, n_rows - 1) / h_r, hq = h * h_r + min(R, n_rows - 1) % h_r;
      const int lim = !live ? -1 : a.causal ? L - n_tok + tok : L - 1;  // the last key this row sees
      // the first row of the warp sees the fewest keys
      const int warp_lim = __shfl_sync(0xffffffffu, lim, 0);
      // ---- Q: this row as f16 into the K-major tile (dead rows are zeros)
      float c2 = a.softmax_scale * kLog2e;
      {
        const T* q = static_cast<const T*>(a.q) + (int64_t)(q0 + tok) * a.q_stride_tok + hq * a.q_stride_head;
        unsigned char* qs = sm + w * C::QTILE;
        float up = 1.f;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          float amax = 0.f;
          for (int c = 0; c < D / 8; ++c) {
            float v[8];
            load8(q + 8 * c, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
          }
          // 2^k with amax 2^k in [2^14, 2^15), inside fp32's normal range
          const int ex = (int)(__float_as_uint(amax) >> 23);
          if (ex > 0 && ex < 255) {
            const int k = min(max(141 - ex, -126), 126);
            up = __uint_as_float((uint32_t)(127 + k) << 23);
            c2 *= __uint_as_float((uint32_t)(127 - k) << 23);
          }
        }
        for (int c = 0; c < D / 8; ++c) {
          float v[8];
          load8(q + 8 * c, v);
          uint32_t o[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = live ? f2_to_h2(v[2 * i] * up, v[2 * i + 1] * up) : 0u;
          *reinterpret_cast<uint4*>(qs + (c >> 3) * (128 * 128) + unit_offset(t, c & 7)) = make_uint4(o[0], o[1], o[2], o[3]);
        }
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      }
      // nm: kHeadroom minus the running maximum; a row that sees no key of the
      // first tile sees none at all (keys are a prefix) and keeps P = 0
      float nm = 0.f, l = 0.f;
      bool ok = true;
      const uint32_t o_addr = C::O_COL + w * 128 + lane_base;
      for (int j = 0; j < n; ++j) {
        ok = wait(&sc_full[j & 3], j >> 2) && wait(&s_full[s_bar(w, j)], s_phase(j));
        // every thread leaves the loop with its warp: the collectives below
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
        const float4* sc = reinterpret_cast<const float4*>(sm + C::SC_OFF) + (j & 3) * (BN / 16);
#pragma unroll
        for (int g = 0; g < BN / 16; ++g) {
          const float4 f = sc[g];
          const float2 m2 = make_float2(c2 * f.x, c2 * f.x), b2 = make_float2(f.y + nm, f.y + nm);
#pragma unroll
          for (int i = 0; i < 8; ++i) s[8 * g + i] = ffma2(s[8 * g + i], m2, b2);
        }
        const int j0 = (tb + j) * BN;
        if (j0 + BN - 1 > warp_lim) {  // some row of the warp sees part of this tile
#pragma unroll
          for (int i = 0; i < BN / 2; ++i) {
            if (j0 + 2 * i > lim) s[i].x = -INFINITY;
            if (j0 + 2 * i + 1 > lim) s[i].y = -INFINITY;
          }
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < BN / 2; ++i) mx = fmaxf(mx, fmaxf(s[i].x, s[i].y));
        if (__any_sync(0xffffffffu, j == 0 || mx > kRaise)) {
          const float up = (j == 0 ? mx > -INFINITY : mx > kRaise) ? kHeadroom - mx : 0.f;  // added to nm
          nm += up;
#pragma unroll
          for (int i = 0; i < BN / 2; ++i) s[i] = fadd2(s[i], make_float2(up, up));
          if (j > 0) {  // O and l follow, once the last product has landed
            const float f = exp2_approx(up);
            l *= f;
            ok = wait(&o_full[2 * w + ((j - 1) & 1)], (j - 1) >> 1);
            if (!__all_sync(0xffffffffu, ok)) {
              ok = false;
              break;
            }
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
              const float2 e = make_float2(exp2_approx(d.x), exp2_approx(d.y));
              sum = fadd2(sum, e);
              p[8 * g + i] = f2_to_h2(e.x, e.y);
            }
            l = fmaf(sum.x + sum.y, sc[2 * c + g].z, l);
          }
          tmem_st16(s_addr + 16 * c, p);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[s_bar(w, j)]);
      }
      // ---- epilogue: O / l of this row
      if (ok && n > 0) {
        ok = wait(&o_full[2 * w + ((n - 1) & 1)], (n - 1) >> 1);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
      }
      if (ok) {
        const float inv = l == 0.f ? 0.f : 1.f / l;  // a NaN sum stays NaN
        const float lse = l == 0.f ? -INFINITY : (log2f(l) - nm) * kLn2;
        const int64_t part = ((int64_t)slot * a.h_k + h) * C::ROWS + w * 128 + t;
        T* o = static_cast<T*>(a.o) + (int64_t)(q0 + tok) * a.o_stride_tok + hq * a.o_stride_head;
#pragma unroll 1
        for (int c = 0; c < D; c += 16) {
          float v[16];
          if (n > 0) {
            tmem_ld16(o_addr + c, v);
            tmem_wait_ld();
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = l == 0.f ? 0.f : v[i] * inv;
          if (live && slot < 0) {
            store8(o + c, v);
            store8(o + c + 8, v + 8);
          } else if (live) {
#pragma unroll
            for (int i = 0; i < 16; i += 8) store8(a.o_part + part * D + c + i, v + i);
          }
          __syncwarp();  // the TMEM load is a whole-warp operation
        }
        if (live) {
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
  const int h_r = a.h_q / a.h_k, q0 = a.q_start[e.x], R = e.y + r;
  if (R >= (a.q_start[e.x + 1] - q0) * h_r || e.w <= 0) return;
  const int64_t step = (int64_t)a.h_k * ROWS, first = ((int64_t)e.z * a.h_k + h) * ROWS + r;
  float mx = -INFINITY;
  for (int s = 0; s < e.w; ++s) mx = fmaxf(mx, a.lse_part[first + s * step]);
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
  const int hq = h * h_r + R % h_r;
  const int64_t tok = q0 + R / h_r;
  T* out = static_cast<T*>(a.o) + tok * a.o_stride_tok + hq * a.o_stride_head;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < E; ++i) out[128 * (i / 4) + 4 * lane + i % 4] = (T)(o[i] * inv);
  if (a.lse && lane == 0) a.lse[tok * a.h_q + hq] = l == 0.f ? -INFINITY : mx + logf(l);
}

constexpr int kMaxDevices = 64;

template <typename T, int D>
static cudaError_t launch_t(const mj_block_attn_args& a, cudaStream_t stream) {
  using C = Cfg<D>;
  auto kern = block_attn_kernel<T, D>;
  static std::atomic<int> ready[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  if (!ready[dev].load(std::memory_order_acquire)) {
    std::lock_guard<std::mutex> lock(tc_init_mutex());
    cudaFuncAttributes fa;
    if ((e = cudaFuncGetAttributes(&fa, kern)) != cudaSuccess) return e;
    // the register split must fit the launch allocation, or the softmax
    // warpgroups would wait for registers that never come
    if (C::REG_POOL > fa.numRegs * C::THREADS) return cudaErrorNotSupported;
    if ((e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM)) != cudaSuccess) return e;
    ready[dev].store(1, std::memory_order_release);
  }
  if (a.num_work) {
    e = launch_kernel(kern, dim3((unsigned)(a.num_work * a.h_k)), dim3(C::THREADS), C::SMEM, stream, a, block_log2(a.kv_format));
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
