// The block-scaled cache: quantising write and read-back.
//
// A block is G consecutive tokens of a page for one KV head; its e4m3 codes
// share the scale 2^(e - 127). Powers of two keep x / scale, and the codes'
// move to a larger scale, exact in fp32 (only a code that becomes subnormal
// rounds), so a block filled token by token holds what one write of all its
// tokens would. e4m3 is a floating type: the shared exponent costs no
// precision until a value is 2^14 below its block's largest.
#include <limits.h>
#include <math.h>

#include <type_traits>

#include "block_cache.cuh"

namespace mj {

// The largest magnitude of a lane's chunks, NaN left out. 16-bit values are
// compared in pairs: two instructions a pair.
template <int NB>
__device__ __forceinline__ float max_abs(const Raw8<float> (&v)[NB]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    float x[8];
    v[i].get(x);
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(x[k]));
  }
  return m;
}
template <typename T, int NB>
__device__ __forceinline__ float max_abs(const Raw8<T> (&v)[NB]) {
  typedef typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type T2;
  T2 m[2];
#pragma unroll
  for (int i = 0; i < NB; ++i) {
    const T2* e = reinterpret_cast<const T2*>(v[i].v);
    const T2 x = __hmax2(__habs2(e[0]), __habs2(e[1])), y = __hmax2(__habs2(e[2]), __habs2(e[3]));
    m[0] = i ? __hmax2(m[0], x) : x;
    m[1] = i ? __hmax2(m[1], y) : y;
  }
  m[0] = __hmax2(m[0], m[1]);
  return fmaxf(fmaxf((float)m[0].x, (float)m[0].y), 0.f);
}

// Skipped tokens are passed 256 at a time, their loads in flight together (a
// token, or 32, a memory round trip: 8K of them before the first kept one 632 us,
// behind the last 77; so 15 and 23). True if any of the 256 from u on is kept,
// or the first or the last token of all where the 256 pass that end.
__device__ __forceinline__ bool any_kept(const int64_t* slots, int64_t u, int64_t num_tokens, int lane) {
  int sign = -1;  // the high words hold the sign
#pragma unroll
  for (int i = 0; i < 8; ++i) sign &= reinterpret_cast<const int*>(slots + min(max(u + 32 * i + lane, (int64_t)0), num_tokens - 1))[1];
  return __any_sync(0xffffffffu, sign >= 0);
}

// One warp per (tile of tokens, KV head, side). A lane per token finds the
// tokens that begin a block's run in slot_mapping; the warp then takes those
// blocks in turn: the run's largest magnitude, the scale, the codes, and (only
// where an open block's scale grew) the rows already there.
// What bounds it: memory latency (slots, then the rows, then the codes) beside
// two passes of arithmetic over the rows: 13K tokens of 8 heads 21.5 us, 3.6 TB/s
// (from fp32 28.2 us, 4.1 TB/s).
// NB: chunks of a lane in flight (16 read a run of 32 rows at once; 8 leave a small
// call's warps more room: 13K tokens 28.6 us with 8, 25.7 with 16, a step of 128
// rows 4.8 and 6.3, before the magnitudes were compared in pairs; now 21.5 and 4.1)
template <typename T, int D, int NB>
__global__ void __launch_bounds__(128) block_write_kernel(mj_cache_write_args a, int lg, int tile, uint64_t per_page) {
  griddep_wait();
  constexpr int CPR = D / 8;  // 8-element chunks of a row
  __shared__ int members_all[4][128];
  const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* members = members_all[wid];  // the run's tokens, as (offset from its first) << 7 | row of the block
  const int64_t tiles = (a.num_tokens + tile - 1) / tile;
  const int64_t w = blockIdx.x * (int64_t)4 + wid;
  if (w >= tiles * a.h_k * 2) return;  // whole warps
  const int side = (int)(w & 1);
  const uint32_t at = (uint32_t)(w >> 1);  // below 2^32: the grid's blocks are counted in 31 bits
  const int h = (int)(at % (uint32_t)a.h_k);
  const int64_t t0 = (int64_t)(at / (uint32_t)a.h_k) * tile;
  const int64_t* slots = a.slot_mapping;
  const T* src = static_cast<const T*>(side ? a.value : a.key) + h * (side ? a.value_stride_head : a.key_stride_head);
  const int64_t st = side ? a.value_stride_tok : a.key_stride_tok;
  unsigned char* cache = static_cast<unsigned char*>(side ? a.v_cache : a.k_cache) + h * (side ? a.v_stride_head : a.k_stride_head);
  const int64_t sp = side ? a.v_stride_page : a.k_stride_page, sr = side ? a.v_stride_row : a.k_stride_row;
  unsigned char* scales = static_cast<unsigned char*>(side ? a.v_scales : a.k_scales) + h * (side ? a.vs_stride_head : a.ks_stride_head);
  const int64_t ssp = side ? a.vs_stride_page : a.ks_stride_page, ssb = side ? a.vs_stride_row : a.ks_stride_row;
  const int G = 1 << lg;

  // lane i < tile: does token t0 + i begin its block's run? The kept token before
  // it is in the tile, but for the tile's first one, whose `far` one is looked
  // for 32 tokens at a time (lane 0 the nearest; the first 32 come with the tile).
  const int64_t t = t0 + lane;
  int64_t far = t0 > lane ? slots[t0 - 1 - lane] : -1;
  const int64_t mine = lane < tile && t < a.num_tokens ? slots[t] : -1;
  const uint32_t kept = __ballot_sync(0xffffffffu, mine >= 0);
  if (!kept) return;  // whole warps
  uint32_t found = __ballot_sync(0xffffffffu, far >= 0);
  for (int64_t u = t0 - 32; !found && u > 0; u -= 32) {
    while (u > 0 && !any_kept(slots, u - 256, a.num_tokens, lane)) u -= 256;
    far = u > lane ? slots[u - 1 - lane] : -1;
    found = __ballot_sync(0xffffffffu, far >= 0);
  }
  far = __shfl_sync(0xffffffffu, far, found ? __ffs(found) - 1 : 0);
  const uint32_t below = kept & ((1u << lane) - 1u);
  const int64_t near = __shfl_sync(0xffffffffu, mine, below ? 31 - __clz(below) : 0);
  const bool first = mine >= 0 && (mine >> lg) != ((below ? near : far) >> lg);
  for (uint32_t todo = __ballot_sync(0xffffffffu, first); todo; todo &= todo - 1) {
    const int64_t tb = t0 + __ffs(todo) - 1;
    const int64_t block = slots[tb] >> lg;
    const int64_t page = quotient(block, per_page);
    const int sub = (int)(block - page * (a.page_size >> lg));
    if (page >= a.num_pages) {
      if (lane == 0) flag(a.status, MJ_DEV_BAD_PAGE);
      continue;
    }
    const int64_t at_scale = page * ssp + sub * ssb;
    const unsigned char old_byte = scales[at_scale];  // (on its way while the run is read)
    // the run: its tokens in order, and which rows of the block they fill
    int count = 0;
    uint32_t rows[4] = {0, 0, 0, 0};
    for (int64_t u0 = tb; u0 < a.num_tokens; u0 += 32) {
      const int64_t u = u0 + lane;
      const int64_t s = u < a.num_tokens ? slots[u] : -1;
      const bool same = s >= 0 && (s >> lg) == block;
      const uint32_t stop = __ballot_sync(0xffffffffu, s >= 0 && !same);
      const uint32_t before = stop ? (stop & -stop) - 1u : 0xffffffffu;  // lanes before the next block's token
      const uint32_t in = __ballot_sync(0xffffffffu, same) & before;
      const bool take = (in >> lane) & 1u;
      const int at = count + __popc(in & ((1u << lane) - 1u));
      const int r = (int)(s & (G - 1));
      if (take && at < G) members[at] = (int)(u - tb) << 7 | r;
#pragma unroll
      for (int k = 0; k < 4; ++k) rows[k] |= __reduce_or_sync(0xffffffffu, take && (r >> 5) == k ? 1u << (r & 31) : 0u);
      count += __popc(in);
      if (stop || count >= G) break;
      if (!in)
        while (u0 + 32 < a.num_tokens && !any_kept(slots, u0 + 32, a.num_tokens, lane)) u0 += 256;
    }
    if (count > G) count = G;
    __syncwarp();
    // The run's chunks in batches of NB a lane, whose loads are in flight
    // together; a run of one batch stays in registers, a longer one is read
    // again (from L2) for its codes.
    const int total = count * CPR;
    Raw8<T> v[NB];
    auto fetch = [&](int c0) {
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int c = min(c0 + 32 * i, total - 1);  // lanes past the end repeat the last chunk
        v[i].load(src + (tb + (members[c / CPR] >> 7)) * st + (c % CPR) * 8, true);
      }
    };
    float amax = 0.f;
    for (int c0 = lane; c0 - lane < total; c0 += 32 * NB) {
      fetch(c0);
      float most = max_abs(v);
      if (most == INFINITY) {  // finite values only
        most = 0.f;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
          float x[8];
          v[i].get(x);
#pragma unroll
          for (int k = 0; k < 8; ++k) most = fabsf(x[k]) < INFINITY ? fmaxf(most, fabsf(x[k])) : most;
        }
      }
      amax = fmaxf(amax, most);
    }
    amax = warp_allmax(amax);
    int e = block_exponent(amax);
    unsigned char* base = cache + page * sp + (int64_t)(sub << lg) * sr;
    if (!(rows[0] & 1u)) {  // not opened by this call
      const int old = block_e(old_byte);
      if (e > old) {  // the rows already there follow
        const float f = __uint_as_float((uint32_t)(127 + old - e) << 23);
#pragma unroll 4
        for (int c = lane; c < G * CPR; c += 32) {
          const int r = c / CPR;
          if ((rows[r >> 5] >> (r & 31)) & 1u) continue;
          uint2* q = reinterpret_cast<uint2*>(base + r * sr + (c % CPR) * 8);
          const uint2 codes = *q;
          *q = make_uint2(scale4(codes.x, f), scale4(codes.y, f));
        }
      } else {
        e = old;
      }
    }
    __syncwarp();  // every lane has its copy of the old byte
    if (lane == 0) scales[at_scale] = (unsigned char)e;
    const float inv = __uint_as_float((uint32_t)(254 - e) << 23);  // 2^(127 - e)
    for (int c0 = lane; c0 - lane < total; c0 += 32 * NB) {
      if (total > 32 * NB) fetch(c0);
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int c = c0 + 32 * i;
        float x[8];
        v[i].get(x);
        if (c < total) *reinterpret_cast<uint2*>(base + (members[c / CPR] & 127) * sr + (c % CPR) * 8) = quantize8(x, inv);
      }
    }
    __syncwarp();  // members is rewritten for the next block
  }
}

template <typename T>
static cudaError_t write_t(const mj_cache_write_args& a, int lg, cudaStream_t stream) {
  // A warp looks through `tile` tokens for the runs that begin there. A prompt's
  // tokens begin one run in 16 or more, a decode step's one each: small calls
  // take single tokens, so that a step's rows are not written one after another
  // (128 rows of 8 heads: 22 us with 16). The slots do not tell the host which it
  // is; 2,048 warps favour the step. A limit of 1,024, 2,048 and 4,096 warps: a
  // step of 128 rows 4.7, 4.0 and 4.0 us, of 512 12.4, 9.4 and 9.9; a prompt of
  // 1000 tokens 5.9, 6.8 and 8.3, of 2000 5.8, 7.7 and 9.2, of 4000 7.5, 7.5, 11.1.
  int tile = 16;
  while (tile > 1 && (a.num_tokens + tile - 1) / tile * a.h_k * 2 < 2048) tile >>= 1;
  const int64_t warps = (a.num_tokens + tile - 1) / tile * a.h_k * 2;
  const dim3 grid((unsigned)((warps + 3) / 4));
  constexpr int NB = 16 / sizeof(T);
  auto kern = a.head_size == 256 ? tile < 16 ? block_write_kernel<T, 256, NB> : block_write_kernel<T, 256, 2 * NB>
              : tile < 16        ? block_write_kernel<T, 128, NB>
                                 : block_write_kernel<T, 128, 2 * NB>;
  return launch_kernel(kern, grid, dim3(128), 0, stream, a, lg, tile, reciprocal(a.page_size >> lg));
}

cudaError_t launch_block_write(const mj_cache_write_args& a, cudaStream_t stream) {
  const int lg = block_log2(a.kv_format);
  if (a.src_dtype == MJ_DT_FP32) return write_t<float>(a, lg, stream);
  if (a.src_dtype == MJ_DT_FP16) return write_t<__half>(a, lg, stream);
  return write_t<__nv_bfloat16>(a, lg, stream);
}

// One warp per (output row, group of up to 8 KV heads): the row's sequence and
// page are looked up once, then each pass moves 512 codes (K and V of two heads
// at head_size 128), four passes in flight. Bound by memory: 66K tokens of 8
// heads take 67 us, 5.9 TB/s (to fp32 114 us, 6.4 TB/s), at four CTAs an SM (at the three that the
// registers gave by themselves 74, at six 73 with spills; two passes in flight 73).
template <typename T, int D>
__global__ void __launch_bounds__(256, 4) block_read_kernel(mj_block_read_args a, int lg, bool wide, uint64_t per_page) {
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x * (int64_t)8 + (threadIdx.x >> 5);
  if (row >= a.num_rows) return;  // whole warps
  const int end = a.offsets[a.num_seqs];
  // The last sequence whose rows begin at or before this one: 32 of the offsets
  // at a time, each lane's start with it (one memory round trip up to 32 sequences).
  int lo = 0, len = a.num_seqs;
  int64_t pos;
  for (;;) {
    const int step = (len + 31) / 32, i = lane * step;
    const bool in = i < len;
    const int off = in ? a.offsets[lo + i] : INT_MAX, begin = in ? a.starts[lo + i] : 0;
    const uint32_t at = __ballot_sync(0xffffffffu, off <= row);
    const int k = at ? 31 - __clz(at) : 0;
    lo += k * step;
    pos = row - __shfl_sync(0xffffffffu, off, k) + __shfl_sync(0xffffffffu, begin, k);
    if (step == 1) break;
    len = min(step, len - k * step);
  }
  if (row >= end) return;
  const int64_t col = quotient(pos, per_page);
  const int r = (int)(pos - col * a.page_size);
  int page = -1;
  if (pos >= 0 && col < a.block_table_cols) page = a.block_table[lo * a.block_table_stride + col];
  if (page < 0 || page >= a.num_pages) {
    if (lane == 0) flag(a.status, MJ_DEV_BAD_PAGE);
    return;
  }
  const int h0 = blockIdx.y * 8, h1 = min(h0 + 8, a.h_k);
  constexpr int CPR = D / 16, NB = 4;
  const unsigned char* kc = static_cast<const unsigned char*>(a.k_cache) + page * a.k_stride_page + r * a.k_stride_row;
  const unsigned char* vc = static_cast<const unsigned char*>(a.v_cache) + page * a.v_stride_page + r * a.v_stride_row;
  const unsigned char* ks = static_cast<const unsigned char*>(a.k_scales) + page * a.ks_stride_page + (r >> lg) * a.ks_stride_block;
  const unsigned char* vs = static_cast<const unsigned char*>(a.v_scales) + page * a.vs_stride_page + (r >> lg) * a.vs_stride_block;
  T* ko = static_cast<T*>(a.k_out) + row * a.ko_stride_tok;
  T* vo = static_cast<T*>(a.v_out) + row * a.vo_stride_tok;
  const int total = (h1 - h0) * 2 * CPR;
  for (int c0 = lane; c0 < total; c0 += 32 * NB) {
    uint4 codes[NB];
    unsigned char e[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {  // every load of the batch in flight
      const int c = min(c0 + 32 * i, total - 1), h = h0 + c / (2 * CPR), side = (c / CPR) & 1;
      codes[i] = *reinterpret_cast<const uint4*>((side ? vc + h * a.v_stride_head : kc + h * a.k_stride_head) + (c % CPR) * 16);
      e[i] = *(side ? vs + h * a.vs_stride_head : ks + h * a.ks_stride_head);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int c = c0 + 32 * i, h = h0 + c / (2 * CPR), side = (c / CPR) & 1;
      if (c >= total) break;
      T* out = (side ? vo + h * a.vo_stride_head : ko + h * a.ko_stride_head) + (c % CPR) * 16;
      const float f = block_scale(e[i]);
      float v[16];
      dequantize8(make_uint2(codes[i].x, codes[i].y), f, v);
      dequantize8(make_uint2(codes[i].z, codes[i].w), f, v + 8);
      if (wide) {
        uint4 raw[sizeof(T)];
        store8(reinterpret_cast<T*>(raw), v);
        store8(reinterpret_cast<T*>(raw) + 8, v + 8);
#pragma unroll
        for (int x = 0; x < (int)sizeof(T); x += 2) store32(reinterpret_cast<uint4*>(out) + x, raw[x], raw[x + 1]);
      } else {
        store8(out, v);
        store8(out + 8, v + 8);
      }
    }
  }
}

template <typename T>
static cudaError_t read_t(const mj_block_read_args& a, int lg, cudaStream_t stream) {
  const dim3 grid((unsigned)((a.num_rows + 7) / 8), (unsigned)((a.h_k + 7) / 8));
  const uint64_t rec = reciprocal(a.page_size);
  const bool wide = ((uintptr_t)a.k_out | (uintptr_t)a.v_out | ((a.ko_stride_tok | a.ko_stride_head | a.vo_stride_tok | a.vo_stride_head) * sizeof(T))) % 32 == 0;
  if (a.head_size == 256) return launch_kernel(block_read_kernel<T, 256>, grid, dim3(256), 0, stream, a, lg, wide, rec);
  return launch_kernel(block_read_kernel<T, 128>, grid, dim3(256), 0, stream, a, lg, wide, rec);
}

cudaError_t launch_block_read(const mj_block_read_args& a, cudaStream_t stream) {
  const int lg = block_log2(a.kv_format);
  if (a.out_dtype == MJ_DT_FP32) return read_t<float>(a, lg, stream);
  if (a.out_dtype == MJ_DT_FP16) return read_t<__half>(a, lg, stream);
  return read_t<__nv_bfloat16>(a, lg, stream);
}

}  // namespace mj
