// C ABI of libmjolnir_b200: argument validation, error reporting, dispatch.
// Every entry point returns an int status and never aborts; the message of
// the last failure of the calling thread is available from mj_last_error().
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>

#include "block_cache.cuh"
#include "common.cuh"

namespace mj {
cudaError_t launch_cache_write(const mj_cache_write_args& a, cudaStream_t stream);
cudaError_t launch_decode_simt(const mj_decode_args& a, cudaStream_t stream);
cudaError_t launch_combine(const mj_decode_args& a, cudaStream_t stream);
cudaError_t launch_decode_tc(const mj_decode_args& a, cudaStream_t stream, bool* handled, bool dry);
const char* tc_ineligible(const mj_decode_args& a);
cudaError_t launch_expand_pages(const mj_expand_args& a, cudaStream_t stream);
cudaError_t launch_qk_norm_rope(const mj_qk_norm_rope_args& a, const mj_rope_axes* axes, bool vec, cudaStream_t stream);
cudaError_t launch_block_write(const mj_cache_write_args& a, cudaStream_t stream);
cudaError_t launch_block_read(const mj_block_read_args& a, cudaStream_t stream);
cudaError_t launch_block_attention(const mj_block_attn_args& a, cudaStream_t stream);
cudaError_t launch_block_join(const mj_block_join_args& a, cudaStream_t stream);
cudaError_t launch_block_weigh(const mj_block_weigh_args& a, cudaStream_t stream);
cudaError_t launch_block_evict(const mj_block_evict_args& a, cudaStream_t stream);
}  // namespace mj

static thread_local char g_err[512] = "";

static int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

static int cuda_status(cudaError_t e, const char* what) {
  if (e == cudaSuccess) {
    g_err[0] = 0;
    return MJ_OK;
  }
  return fail(MJ_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

static bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p % a) == 0; }

namespace mj {
// Lets other translation units of the library report through mj_last_error().
int set_last_error(int code, const char* msg) { return fail(code, "%s", msg); }

bool pdl_enabled() {
  static const bool on = [] {
    const char* v = getenv("MJOLNIR_PDL");
    return !(v && v[0] == '0' && v[1] == 0);
  }();
  return on;
}
}  // namespace mj

extern "C" {

const char* mj_last_error(void) { return g_err; }

int mj_abi_version(void) { return MJ_ABI_VERSION; }

int mj_row_bytes(int head_size, int kv_format) {
  if (head_size <= 0 || head_size % 16) return -1;
  if (kv_format == MJ_KV_FP8_E4M3 || mj::is_block_format(kv_format)) return head_size;
  if (kv_format == MJ_KV_E2M3 || kv_format == MJ_KV_E3M2) return head_size * 3 / 4;
  if (kv_format == MJ_KV_E2M1 || kv_format == MJ_KV_NVFP4) return head_size / 2;
  return -1;
}

// nvfp4 scale tensors: present, and (for the tensor-core kernel's 8-byte
// copies) with 8-byte aligned rows when `align8`.
static const char* nvfp4_scales_problem(const void* ks, const void* vs, const int64_t* strides, bool align8) {
  if (!ks || !vs) return "nvfp4 needs k_scales and v_scales";
  if (align8) {
    if (!aligned(ks, 8) || !aligned(vs, 8)) return "nvfp4 scale rows must be 8-byte aligned";
    for (int i = 0; i < 6; ++i)
      if (strides[i] % 8) return "nvfp4 scale strides must be multiples of 8 bytes";
  }
  return nullptr;
}

int mj_cache_write(const mj_cache_write_args* args, void* stream) {
  if (!args) return fail(MJ_ERR_INVALID, "mj_cache_write: null args");
  const mj_cache_write_args& a = *args;
  if (a.num_tokens < 0 || a.h_k <= 0) return fail(MJ_ERR_INVALID, "mj_cache_write: num_tokens %lld h_k %d", (long long)a.num_tokens, a.h_k);
  if (a.num_tokens == 0) {
    g_err[0] = 0;
    return MJ_OK;
  }
  const int rb = mj_row_bytes(a.head_size, a.kv_format);
  if (rb < 0 || mj::is_block_format(a.kv_format))
    return fail(MJ_ERR_UNSUPPORTED, "mj_cache_write: head_size %d / kv_format %d%s", a.head_size, a.kv_format,
                rb < 0 ? "" : " (block-scaled formats: mj_block_write)");
  if (a.src_dtype < MJ_DT_BF16 || a.src_dtype > MJ_DT_FP32) return fail(MJ_ERR_INVALID, "mj_cache_write: src_dtype %d", a.src_dtype);
  if (!a.key || !a.value || !a.k_cache || !a.v_cache || !a.slot_mapping || !a.k_scale || !a.v_scale)
    return fail(MJ_ERR_INVALID, "mj_cache_write: null pointer argument");
  if (a.page_size <= 0 || a.num_pages <= 0) return fail(MJ_ERR_INVALID, "mj_cache_write: page_size %d num_pages %lld", a.page_size, (long long)a.num_pages);
  for (int m : {a.k_scale_mode, a.v_scale_mode})
    if (m != MJ_SCALE_TENSOR && m != MJ_SCALE_HEAD && m != MJ_SCALE_CHANNEL)
      return fail(MJ_ERR_INVALID, "mj_cache_write: scale mode %d", m);
  if (a.num_tokens * a.h_k > (int64_t)INT32_MAX / 32) return fail(MJ_ERR_UNSUPPORTED, "mj_cache_write: too many rows");
  if (a.kv_format == MJ_KV_NVFP4) {
    if (a.head_size % 128) return fail(MJ_ERR_UNSUPPORTED, "mj_cache_write: nvfp4 head_size %d (a multiple of 128)", a.head_size);
    if (a.k_scale_mode == MJ_SCALE_CHANNEL || a.v_scale_mode == MJ_SCALE_CHANNEL)
      return fail(MJ_ERR_INVALID, "mj_cache_write: the nvfp4 global scale is per tensor or per KV head");
    const int64_t st[6] = {a.ks_stride_page, a.ks_stride_row, a.ks_stride_head, a.vs_stride_page, a.vs_stride_row, a.vs_stride_head};
    if (const char* why = nvfp4_scales_problem(a.k_scales, a.v_scales, st, false))
      return fail(MJ_ERR_INVALID, "mj_cache_write: %s", why);
  }
  return cuda_status(mj::launch_cache_write(a, (cudaStream_t)stream), "mj_cache_write launch");
}

static int validate_decode(const mj_decode_args& a, const char* who) {
  if (a.num_seqs < 0 || a.q_len < 1 || a.h_k <= 0 || a.h_q <= 0 || a.h_q % a.h_k)
    return fail(MJ_ERR_INVALID, "%s: num_seqs %d q_len %d h_q %d h_k %d", who, a.num_seqs, a.q_len, a.h_q, a.h_k);
  if (a.head_size != 128 && a.head_size != 256)
    return fail(MJ_ERR_UNSUPPORTED, "%s: head_size %d (128 or 256)", who, a.head_size);
  if (a.kv_format < MJ_KV_FP8_E4M3 || a.kv_format > MJ_KV_FP8_B128)
    return fail(MJ_ERR_INVALID, "%s: kv_format %d", who, a.kv_format);
  if (mj::is_block_format(a.kv_format) && (!a.k_scales || !a.v_scales || a.kernel == MJ_KERNEL_SIMT || mj::tc_ineligible(a)))
    return fail(MJ_ERR_UNSUPPORTED, "%s: block-scaled formats need k_scales and v_scales and run the tensor-core kernel only (%s)",
                who, a.kernel == MJ_KERNEL_SIMT ? "kernel" : mj::tc_ineligible(a) ? mj::tc_ineligible(a) : "scales");
  if (a.kv_format == MJ_KV_NVFP4) {
    const int64_t st[6] = {a.ks_stride_page, a.ks_stride_row, a.ks_stride_head, a.vs_stride_page, a.vs_stride_row, a.vs_stride_head};
    if (const char* why = nvfp4_scales_problem(a.k_scales, a.v_scales, st, false))
      return fail(MJ_ERR_INVALID, "%s: %s", who, why);
  }
  const int n_q = a.q_len * (a.h_q / a.h_k);
  if (n_q > 64) return fail(MJ_ERR_UNSUPPORTED, "%s: q_len * h_q / h_k = %d > 64 rows per KV head", who, n_q);
  if (a.q_dtype < MJ_DT_BF16 || a.q_dtype > MJ_DT_FP32 || a.o_dtype < MJ_DT_BF16 || a.o_dtype > MJ_DT_FP32)
    return fail(MJ_ERR_INVALID, "%s: q_dtype %d o_dtype %d", who, a.q_dtype, a.o_dtype);
  if (!a.q || !a.o || !a.k_cache || !a.v_cache || !a.block_table || !a.seq_lens || !a.work || !a.n_splits)
    return fail(MJ_ERR_INVALID, "%s: null pointer argument", who);
  if (a.page_size <= 0 || a.num_pages <= 0 || a.num_work < 0 || a.max_splits < 1)
    return fail(MJ_ERR_INVALID, "%s: page_size %d num_pages %lld num_work %d max_splits %d", who, a.page_size,
                (long long)a.num_pages, a.num_work, a.max_splits);
  const int64_t st[6] = {a.k_stride_page, a.k_stride_row, a.k_stride_head, a.v_stride_page, a.v_stride_row, a.v_stride_head};
  for (int i = 0; i < 6; ++i)
    if (st[i] < 0 || st[i] % 16) return fail(MJ_ERR_UNSUPPORTED, "%s: KV byte strides must be 16-byte multiples", who);
  if (!aligned(a.k_cache, 16) || !aligned(a.v_cache, 16)) return fail(MJ_ERR_UNSUPPORTED, "%s: KV views must be 16-byte aligned", who);
  if (!aligned(a.work, 16)) return fail(MJ_ERR_INVALID, "%s: work list must be 16-byte aligned", who);
  for (int m : {a.k_descale_mode, a.v_descale_mode})
    if (m != MJ_SCALE_TENSOR && m != MJ_SCALE_HEAD && m != MJ_SCALE_SEQ_HEAD)
      return fail(MJ_ERR_INVALID, "%s: descale mode %d", who, m);
  if (a.o_part && (!a.lse_part || a.part_seqs < a.num_seqs))
    return fail(MJ_ERR_INVALID, "%s: partial buffers need lse_part and part_seqs >= num_seqs", who);
  if (a.kernel < MJ_KERNEL_AUTO || a.kernel > MJ_KERNEL_TC) return fail(MJ_ERR_INVALID, "%s: kernel %d", who, a.kernel);
  if (a.kernel == MJ_KERNEL_TC && mj::tc_ineligible(a))
    return fail(MJ_ERR_UNSUPPORTED, "%s: the tensor-core kernel cannot run these arguments (%s)", who, mj::tc_ineligible(a));
  return MJ_OK;
}

int mj_decode_kernel(const mj_decode_args* args) {
  if (!args) return -fail(MJ_ERR_INVALID, "mj_decode_kernel: null args");
  int rc = validate_decode(*args, "mj_decode_kernel");
  if (rc) return -rc;
  if (args->kernel == MJ_KERNEL_SIMT || mj::tc_ineligible(*args)) return MJ_KERNEL_SIMT;
  // prepare the variant mj_decode would launch, without launching it
  bool handled = false;
  const cudaError_t e = mj::launch_decode_tc(*args, nullptr, &handled, true);
  if (e != cudaSuccess) return -cuda_status(e, "mj_decode_kernel (tensor-core variant)");
  return handled ? MJ_KERNEL_TC : MJ_KERNEL_SIMT;
}

int mj_decode(const mj_decode_args* args, void* stream) {
  if (!args) return fail(MJ_ERR_INVALID, "mj_decode: null args");
  const mj_decode_args& a = *args;
  int rc = validate_decode(a, "mj_decode");
  if (rc) return rc;
  if (a.num_seqs == 0 || a.num_work == 0) {
    g_err[0] = 0;
    return MJ_OK;
  }
  cudaStream_t s = (cudaStream_t)stream;
  bool handled = false;
  cudaError_t e = cudaSuccess;
  if (a.kernel != MJ_KERNEL_SIMT) {
    e = mj::launch_decode_tc(a, s, &handled, false);
    if (e != cudaSuccess) return cuda_status(e, "mj_decode launch (tensor-core kernel)");
  }
  if (!handled && mj::is_block_format(a.kv_format))
    return fail(MJ_ERR_UNSUPPORTED, "mj_decode: no tensor-core variant fits this build for the block-scaled formats");
  if (!handled) {
    e = mj::launch_decode_simt(a, s);
    if (e != cudaSuccess) return cuda_status(e, "mj_decode launch");
  }
  // the one-warpgroup tensor-core variants (every head_dim-256 one) merge in
  // the kernel when given counters
  const bool merged = handled && a.merge_counters && (a.q_len * (a.h_q / a.h_k) <= 16 || a.head_size == 256) &&
                      a.max_splits <= 16;
  if (a.with_combine && !merged) {
    if (!a.o_part) return fail(MJ_ERR_INVALID, "mj_decode: with_combine needs partial buffers");
    return cuda_status(mj::launch_combine(a, s), "mj_combine launch");
  }
  g_err[0] = 0;
  return MJ_OK;
}

int mj_combine(const mj_decode_args* args, void* stream) {
  if (!args) return fail(MJ_ERR_INVALID, "mj_combine: null args");
  const mj_decode_args& a = *args;
  int rc = validate_decode(a, "mj_combine");
  if (rc) return rc;
  if (!a.o_part) return fail(MJ_ERR_INVALID, "mj_combine: null partial buffers");
  if (a.num_seqs == 0) {
    g_err[0] = 0;
    return MJ_OK;
  }
  return cuda_status(mj::launch_combine(a, (cudaStream_t)stream), "mj_combine launch");
}

int mj_expand_pages(const mj_expand_args* args, void* stream) {
  if (!args) return fail(MJ_ERR_INVALID, "mj_expand_pages: null args");
  const mj_expand_args& a = *args;
  if (a.num_out_pages < 0 || a.h_k <= 0 || a.page_size <= 0 || a.num_pages <= 0)
    return fail(MJ_ERR_INVALID, "mj_expand_pages: num_out_pages %lld h_k %d page_size %d num_pages %lld",
                (long long)a.num_out_pages, a.h_k, a.page_size, (long long)a.num_pages);
  if (a.head_size <= 0 || a.head_size % 16)
    return fail(MJ_ERR_UNSUPPORTED, "mj_expand_pages: head_size %d (a multiple of 16)", a.head_size);
  if (a.kv_format < MJ_KV_E2M3 || a.kv_format > MJ_KV_NVFP4)
    return fail(MJ_ERR_INVALID, "mj_expand_pages: kv_format %d (a narrow format)", a.kv_format);
  if (a.kv_format == MJ_KV_NVFP4) {
    const int64_t st[6] = {a.ks_stride_page, a.ks_stride_row, a.ks_stride_head, a.vs_stride_page, a.vs_stride_row, a.vs_stride_head};
    if (const char* why = nvfp4_scales_problem(a.k_scales, a.v_scales, st, false))
      return fail(MJ_ERR_INVALID, "mj_expand_pages: %s", why);
  }
  if (a.num_out_pages == 0) {
    g_err[0] = 0;
    return MJ_OK;
  }
  if (!a.k_cache || !a.v_cache || !a.k_out || !a.v_out || !a.src_pages)
    return fail(MJ_ERR_INVALID, "mj_expand_pages: null pointer argument");
  for (int m : {a.k_ratio_mode, a.v_ratio_mode})
    if (m != MJ_SCALE_TENSOR && m != MJ_SCALE_HEAD && m != MJ_SCALE_CHANNEL)
      return fail(MJ_ERR_INVALID, "mj_expand_pages: ratio mode %d", m);
  const int64_t in_strides[6] = {a.k_stride_page, a.k_stride_row, a.k_stride_head,
                                 a.v_stride_page, a.v_stride_row, a.v_stride_head};
  const int64_t out_strides[6] = {a.ko_stride_page, a.ko_stride_row, a.ko_stride_head,
                                  a.vo_stride_page, a.vo_stride_row, a.vo_stride_head};
  bool ok = aligned(a.k_cache, 4) && aligned(a.v_cache, 4) && aligned(a.k_out, 16) && aligned(a.v_out, 16);
  for (int i = 0; i < 6; ++i) ok = ok && in_strides[i] % 4 == 0 && out_strides[i] % 16 == 0;
  if (!ok) return fail(MJ_ERR_UNSUPPORTED, "mj_expand_pages: packed rows must be 4-byte and output rows 16-byte aligned");
  if (a.num_out_pages * a.page_size * a.h_k > (int64_t)INT32_MAX)
    return fail(MJ_ERR_UNSUPPORTED, "mj_expand_pages: too many rows");
  return cuda_status(mj::launch_expand_pages(a, (cudaStream_t)stream), "mj_expand_pages launch");
}

// Shape, layout and scale tensors of a block-scaled cache (nullptr = valid):
// st = the six cache strides, ss the six scale strides, in bytes.
static const char* block_cache_problem(int head_size, int kv_format, int page_size, int h_k, int64_t num_pages,
                                       const void* k, const void* v, const int64_t* st, const void* ks, const void* vs,
                                       const int64_t* ss, uintptr_t align) {
  if (!mj::is_block_format(kv_format)) return "kv_format is not block-scaled (MJ_KV_FP8_B16 .. _B128)";
  if (head_size != 128 && head_size != 256) return "head_size must be 128 or 256";
  if (page_size <= 0 || page_size % (1 << mj::block_log2(kv_format))) return "a block must divide the page";
  if (page_size > (1 << 20)) return "page_size";
  if (h_k <= 0 || num_pages <= 0 || num_pages > INT32_MAX) return "h_k / num_pages";
  if (!k || !v || !ks || !vs) return "null cache or scale pointer";
  for (int i = 0; i < 6; ++i)
    if (st[i] < 0 || st[i] % (int64_t)align || ss[i] < 0) return "cache strides must be multiples of the row alignment";
  if (!aligned(k, align) || !aligned(v, align)) return "cache rows must be aligned";
  return nullptr;
}

// True where a stride of 0 lets pages, rows (blocks) or heads share their bytes.
// In the codes the tensor maps cannot hold that, and a write would race with itself.
static bool shared_bytes(const int64_t* strides, int64_t pages, int64_t rows, int64_t heads) {
  const int64_t n[3] = {pages, rows, heads};
  for (int i = 0; i < 6; ++i)
    if (n[i % 3] > 1 && !strides[i]) return true;
  return false;
}

static int norm_rope(const mj_qk_norm_rope_args* args, const mj_rope_axes* axes, void* stream) {
  if (!args) return fail(MJ_ERR_INVALID, "mj_qk_norm_rope: null args");
  const mj_qk_norm_rope_args& a = *args;
  if (a.num_tokens < 0 || a.h_q < 0 || a.h_k < 0)
    return fail(MJ_ERR_INVALID, "mj_qk_norm_rope: num_tokens %lld h_q %d h_k %d", (long long)a.num_tokens, a.h_q, a.h_k);
  if (a.head_size <= 0 || a.head_size % 16 || a.head_size > 512)
    return fail(MJ_ERR_UNSUPPORTED, "mj_qk_norm_rope: head_size %d (a multiple of 16, at most 512)", a.head_size);
  if (a.rot_dim < 0 || a.rot_dim % 16 || a.rot_dim > a.head_size)
    return fail(MJ_ERR_UNSUPPORTED, "mj_qk_norm_rope: rot_dim %d (a multiple of 16, at most head_size)", a.rot_dim);
  for (int dt : {a.dtype, a.cos_sin_dtype, a.weight_dtype})
    if (dt < MJ_DT_BF16 || dt > MJ_DT_FP32) return fail(MJ_ERR_INVALID, "mj_qk_norm_rope: dtype %d", dt);
  if (axes) {
    if (axes->num_axes < 1 || axes->num_axes > MJ_ROPE_AXES)
      return fail(MJ_ERR_UNSUPPORTED, "mj_qk_norm_rope_axes: %d axes (1 to %d)", axes->num_axes, MJ_ROPE_AXES);
    for (int i = 0; i < a.rot_dim / 2; ++i)
      if (axes->axis[i] >= axes->num_axes)
        return fail(MJ_ERR_INVALID, "mj_qk_norm_rope_axes: angle %d on axis %d of %d", i, axes->axis[i], axes->num_axes);
  }
  if (axes && a.num_positions > INT32_MAX) return fail(MJ_ERR_UNSUPPORTED, "mj_qk_norm_rope_axes: too many positions");
  if (a.num_tokens == 0 || a.h_q + a.h_k == 0) {
    g_err[0] = 0;
    return MJ_OK;
  }
  if ((a.h_q && (!a.q || !a.q_out)) || (a.h_k && (!a.k || !a.k_out)))
    return fail(MJ_ERR_INVALID, "mj_qk_norm_rope: null q / k pointer");
  if (a.rot_dim && (!a.positions || !a.cos_sin || a.num_positions <= 0))
    return fail(MJ_ERR_INVALID, "mj_qk_norm_rope: rotation needs positions and the cos / sin table");
  if (!(a.eps >= 0.f)) return fail(MJ_ERR_INVALID, "mj_qk_norm_rope: eps %g", (double)a.eps);
  if (a.num_tokens >= 1 << 30 || a.num_tokens * (a.h_q + a.h_k) > (int64_t)1 << 33) return fail(MJ_ERR_UNSUPPORTED, "mj_qk_norm_rope: too many rows");
  // 16-byte accesses where every row allows them
  const int64_t es = a.dtype == MJ_DT_FP32 ? 4 : 2;
  bool vec = true;
  if (a.h_q) {
    vec = vec && aligned(a.q, 16) && aligned(a.q_out, 16);
    for (int64_t s : {a.q_stride_tok, a.q_stride_head, a.qo_stride_tok, a.qo_stride_head}) vec = vec && (s * es) % 16 == 0;
  }
  if (a.h_k) {
    vec = vec && aligned(a.k, 16) && aligned(a.k_out, 16);
    for (int64_t s : {a.k_stride_tok, a.k_stride_head, a.ko_stride_tok, a.ko_stride_head}) vec = vec && (s * es) % 16 == 0;
  }
  return cuda_status(mj::launch_qk_norm_rope(a, axes, vec, (cudaStream_t)stream), "mj_qk_norm_rope launch");
}

int mj_qk_norm_rope(const mj_qk_norm_rope_args* args, void* stream) { return norm_rope(args, nullptr, stream); }

int mj_qk_norm_rope_axes(const mj_qk_norm_rope_args* args, const mj_rope_axes* axes, void* stream) {
  if (!axes) return fail(MJ_ERR_INVALID, "mj_qk_norm_rope_axes: null axes");
  return norm_rope(args, axes, stream);
}

int mj_block_write(const mj_cache_write_args* args, void* stream) {
  if (!args) return fail(MJ_ERR_INVALID, "mj_block_write: null args");
  const mj_cache_write_args& a = *args;
  if (a.num_tokens < 0) return fail(MJ_ERR_INVALID, "mj_block_write: num_tokens %lld", (long long)a.num_tokens);
  const int64_t st[6] = {a.k_stride_page, a.k_stride_row, a.k_stride_head, a.v_stride_page, a.v_stride_row, a.v_stride_head};
  const int64_t ss[6] = {a.ks_stride_page, a.ks_stride_row, a.ks_stride_head, a.vs_stride_page, a.vs_stride_row, a.vs_stride_head};
  if (const char* why = block_cache_problem(a.head_size, a.kv_format, a.page_size, a.h_k, a.num_pages, a.k_cache, a.v_cache,
                                            st, a.k_scales, a.v_scales, ss, 8))
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_write: %s (head_size %d, kv_format %d, page_size %d; 8-byte aligned rows)", why,
                a.head_size, a.kv_format, a.page_size);
  if (a.src_dtype < MJ_DT_BF16 || a.src_dtype > MJ_DT_FP32) return fail(MJ_ERR_INVALID, "mj_block_write: src_dtype %d", a.src_dtype);
  if (a.num_tokens == 0) {
    g_err[0] = 0;
    return MJ_OK;
  }
  if (!a.key || !a.value || !a.slot_mapping) return fail(MJ_ERR_INVALID, "mj_block_write: null pointer argument");
  const int64_t es = a.src_dtype == MJ_DT_FP32 ? 4 : 2;
  bool ok = aligned(a.key, 16) && aligned(a.value, 16);
  for (int64_t s : {a.key_stride_tok, a.key_stride_head, a.value_stride_tok, a.value_stride_head}) ok = ok && (s * es) % 16 == 0;
  if (!ok) return fail(MJ_ERR_UNSUPPORTED, "mj_block_write: key / value rows must be 16-byte aligned");
  if (a.num_tokens >= 1 << 24 || a.h_k > 1024) return fail(MJ_ERR_UNSUPPORTED, "mj_block_write: too many rows");
  if (shared_bytes(st, a.num_pages, a.page_size, a.h_k) ||
      shared_bytes(ss, a.num_pages, a.page_size >> mj::block_log2(a.kv_format), a.h_k))
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_write: a cache or scale stride of 0");
  return cuda_status(mj::launch_block_write(a, (cudaStream_t)stream), "mj_block_write launch");
}

int mj_block_read(const mj_block_read_args* args, void* stream) {
  if (!args) return fail(MJ_ERR_INVALID, "mj_block_read: null args");
  const mj_block_read_args& a = *args;
  if (a.num_seqs < 0 || a.num_rows < 0) return fail(MJ_ERR_INVALID, "mj_block_read: num_seqs %d num_rows %lld", a.num_seqs, (long long)a.num_rows);
  const int64_t st[6] = {a.k_stride_page, a.k_stride_row, a.k_stride_head, a.v_stride_page, a.v_stride_row, a.v_stride_head};
  const int64_t ss[6] = {a.ks_stride_page, a.ks_stride_block, a.ks_stride_head, a.vs_stride_page, a.vs_stride_block, a.vs_stride_head};
  if (const char* why = block_cache_problem(a.head_size, a.kv_format, a.page_size, a.h_k, a.num_pages, a.k_cache, a.v_cache,
                                            st, a.k_scales, a.v_scales, ss, 16))
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_read: %s (head_size %d, kv_format %d, page_size %d; 16-byte aligned rows)", why,
                a.head_size, a.kv_format, a.page_size);
  if (a.out_dtype < MJ_DT_BF16 || a.out_dtype > MJ_DT_FP32) return fail(MJ_ERR_INVALID, "mj_block_read: out_dtype %d", a.out_dtype);
  if (a.num_seqs == 0 || a.num_rows == 0) {
    g_err[0] = 0;
    return MJ_OK;
  }
  if (!a.block_table || a.block_table_cols <= 0 || !a.starts || !a.offsets || !a.k_out || !a.v_out)
    return fail(MJ_ERR_INVALID, "mj_block_read: null pointer argument");
  const int64_t es = a.out_dtype == MJ_DT_FP32 ? 4 : 2;
  bool ok = aligned(a.k_out, 16) && aligned(a.v_out, 16);
  for (int64_t s : {a.ko_stride_tok, a.ko_stride_head, a.vo_stride_tok, a.vo_stride_head}) ok = ok && (s * es) % 16 == 0;
  if (!ok) return fail(MJ_ERR_UNSUPPORTED, "mj_block_read: output rows must be 16-byte aligned");
  if (a.num_rows > INT32_MAX || a.num_rows * a.h_k > (int64_t)1 << 34) return fail(MJ_ERR_UNSUPPORTED, "mj_block_read: too many rows");
  return cuda_status(mj::launch_block_read(a, (cudaStream_t)stream), "mj_block_read launch");
}

int mj_block_attention(const mj_block_attn_args* args, void* stream) {
  if (!args) return fail(MJ_ERR_INVALID, "mj_block_attention: null args");
  const mj_block_attn_args& a = *args;
  if (a.num_seqs < 0 || a.num_tokens < 0 || a.h_k <= 0 || a.h_q <= 0 || a.h_q % a.h_k)
    return fail(MJ_ERR_INVALID, "mj_block_attention: num_seqs %d num_tokens %lld h_q %d h_k %d", a.num_seqs,
                (long long)a.num_tokens, a.h_q, a.h_k);
  const int64_t st[6] = {a.k_stride_page, a.k_stride_row, a.k_stride_head, a.v_stride_page, a.v_stride_row, a.v_stride_head};
  const int64_t ss[6] = {a.ks_stride_page, a.ks_stride_block, a.ks_stride_head, a.vs_stride_page, a.vs_stride_block, a.vs_stride_head};
  if (const char* why = block_cache_problem(a.head_size, a.kv_format, a.page_size, a.h_k, a.num_pages, a.k_cache, a.v_cache,
                                            st, a.k_scales, a.v_scales, ss, 16))
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_attention: %s (head_size %d, kv_format %d, page_size %d; 16-byte aligned rows)",
                why, a.head_size, a.kv_format, a.page_size);
  if (a.page_size != 16 && a.page_size != 32 && a.page_size != 64 && a.page_size != 128)
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_attention: page_size %d (16, 32, 64 or 128)", a.page_size);
  if (a.dtype != MJ_DT_BF16 && a.dtype != MJ_DT_FP16)
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_attention: dtype %d (bf16 or fp16)", a.dtype);
  if (a.num_seqs == 0 || a.num_tokens == 0) {
    g_err[0] = 0;
    return MJ_OK;
  }
  if (!a.q || !a.o || !a.block_table || a.block_table_cols <= 0 || !a.seq_lens || !a.q_start)
    return fail(MJ_ERR_INVALID, "mj_block_attention: null pointer argument");
  bool ok = aligned(a.q, 16) && aligned(a.o, 16);
  for (int64_t s : {a.q_stride_tok, a.q_stride_head, a.o_stride_tok, a.o_stride_head}) ok = ok && s % 8 == 0;
  if (!ok) return fail(MJ_ERR_UNSUPPORTED, "mj_block_attention: q / o rows must be 16-byte aligned");
  if (a.num_tokens * a.h_q > (int64_t)INT32_MAX) return fail(MJ_ERR_UNSUPPORTED, "mj_block_attention: too many rows");
  if (a.num_work < 0 || a.num_merges < 0 || a.num_slots < 0 || (a.num_work && (!a.work || !aligned(a.work, 16))) ||
      (a.num_merges && (!a.merges || !aligned(a.merges, 16))) || (a.num_slots && (!a.o_part || !a.lse_part || !aligned(a.o_part, 16))))
    return fail(MJ_ERR_INVALID, "mj_block_attention: plan or partial buffers");
  if ((int64_t)a.num_work * a.h_k > (int64_t)INT32_MAX) return fail(MJ_ERR_UNSUPPORTED, "mj_block_attention: too many work items");
  if (shared_bytes(st, a.num_pages, a.page_size, a.h_k)) return fail(MJ_ERR_UNSUPPORTED, "mj_block_attention: a cache stride of 0");
  return cuda_status(mj::launch_block_attention(a, (cudaStream_t)stream), "mj_block_attention launch");
}

int mj_block_join(const mj_block_join_args* args, void* stream) {
  if (!args) return fail(MJ_ERR_INVALID, "mj_block_join: null args");
  const mj_block_join_args& a = *args;
  if (a.num_seqs < 0 || a.num_tokens < 0 || a.h_k <= 0 || a.h_q <= 0 || a.h_q % a.h_k || a.num_joins < 0 || a.num_rows < 0 ||
      a.num_slots < 0 || a.max_splits < 0 || a.part_seqs < 0)
    return fail(MJ_ERR_INVALID, "mj_block_join: num_seqs %d num_tokens %lld h_q %d h_k %d num_joins %d num_rows %d", a.num_seqs,
                (long long)a.num_tokens, a.h_q, a.h_k, a.num_joins, a.num_rows);
  if (a.head_size != 128 && a.head_size != 256) return fail(MJ_ERR_UNSUPPORTED, "mj_block_join: head_size %d (128 or 256)", a.head_size);
  if (a.dtype != MJ_DT_BF16 && a.dtype != MJ_DT_FP16)
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_join: dtype %d (bf16 or fp16)", a.dtype);
  if (a.num_seqs == 0 || a.num_tokens == 0 || a.num_joins == 0 || a.num_rows == 0) {
    g_err[0] = 0;
    return MJ_OK;
  }
  if (!a.o || !a.joins || !aligned(a.joins, 16) || (a.num_slots && (!a.o_part || !a.lse_part || !aligned(a.o_part, 16))) ||
      (a.d_part && (!a.d_lse_part || !aligned(a.d_part, 16))))
    return fail(MJ_ERR_INVALID, "mj_block_join: plan or partial buffers");
  if (!aligned(a.o, 16) || a.o_stride_tok % 8 || a.o_stride_head % 8)
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_join: o rows must be 16-byte aligned");
  if ((int64_t)a.num_rows * a.h_k > (int64_t)INT32_MAX) return fail(MJ_ERR_UNSUPPORTED, "mj_block_join: too many rows");
  return cuda_status(mj::launch_block_join(a, (cudaStream_t)stream), "mj_block_join launch");
}

// Whether rows of `cols` elements of an (n0, n1) array share some, whose dims lie one outside the other.
static bool rows_overlap(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t cols) {
  if (n0 > 1 && n1 > 1) {
    const bool swap = s0 < s1;
    const int64_t outer = swap ? s1 : s0, inner = swap ? s0 : s1, n = swap ? n0 : n1;
    return inner < cols || outer < (__int128)inner * (n - 1) + cols;
  }
  return (n0 > 1 && s0 < cols) || (n1 > 1 && s1 < cols);
}

int mj_block_weigh(const mj_block_weigh_args* args, void* stream) {
  if (!args) return fail(MJ_ERR_INVALID, "mj_block_weigh: null args");
  const mj_block_weigh_args& a = *args;
  if (a.num_seqs < 0 || a.num_rows < 0 || a.h_k <= 0 || a.h_q <= 0 || a.h_q % a.h_k || a.window < 0)
    return fail(MJ_ERR_INVALID, "mj_block_weigh: num_seqs %d num_rows %lld h_q %d h_k %d window %d", a.num_seqs,
                (long long)a.num_rows, a.h_q, a.h_k, a.window);
  const int64_t st[6] = {a.k_stride_page, a.k_stride_row, a.k_stride_head, a.k_stride_page, a.k_stride_row, a.k_stride_head};
  const int64_t ss[6] = {a.ks_stride_page, a.ks_stride_block, a.ks_stride_head, a.ks_stride_page, a.ks_stride_block, a.ks_stride_head};
  if (const char* why = block_cache_problem(a.head_size, a.kv_format, a.page_size, a.h_k, a.num_pages, a.k_cache, a.k_cache,
                                            st, a.k_scales, a.k_scales, ss, 16))
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_weigh: %s (head_size %d, kv_format %d, page_size %d; 16-byte aligned rows)", why,
                a.head_size, a.kv_format, a.page_size);
  if (a.page_size != 16 && a.page_size != 32 && a.page_size != 64 && a.page_size != 128)
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_weigh: page_size %d (16, 32, 64 or 128)", a.page_size);
  if (a.dtype != MJ_DT_BF16 && a.dtype != MJ_DT_FP16)
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_weigh: dtype %d (bf16 or fp16)", a.dtype);
  if (a.num_seqs == 0 || a.num_rows == 0) {
    g_err[0] = 0;
    return MJ_OK;
  }
  if (!a.q || !a.lse || !a.block_table || a.block_table_cols <= 0 || !a.offsets || !a.seq_lens || !a.weights)
    return fail(MJ_ERR_INVALID, "mj_block_weigh: null pointer argument");
  if (a.weights_cols < 0 || a.w_stride_seq < 0 || a.w_stride_head < 0)
    return fail(MJ_ERR_INVALID, "mj_block_weigh: weights of %lld columns", (long long)a.weights_cols);
  if (rows_overlap(a.num_seqs, a.w_stride_seq, a.h_k, a.w_stride_head, a.weights_cols))
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_weigh: a weights stride by which rows share elements");
  if (!aligned(a.q, 16) || a.q_stride_tok % 8 || a.q_stride_head % 8 || a.q_stride_tok < 0 || a.q_stride_head < 0)
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_weigh: q rows must be 16-byte aligned");
  if ((a.num_rows > 1 && !a.q_stride_tok) || (a.h_q > 1 && !a.q_stride_head))
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_weigh: a q stride of 0");
  if (a.num_rows * a.h_q > (int64_t)INT32_MAX || a.num_seqs > 1 << 20) return fail(MJ_ERR_UNSUPPORTED, "mj_block_weigh: too many rows");
  if (shared_bytes(st, a.num_pages, a.page_size, a.h_k)) return fail(MJ_ERR_UNSUPPORTED, "mj_block_weigh: a cache stride of 0");
  return cuda_status(mj::launch_block_weigh(a, (cudaStream_t)stream), "mj_block_weigh launch");
}

int mj_block_evict(const mj_block_evict_args* args, void* stream) {
  if (!args) return fail(MJ_ERR_INVALID, "mj_block_evict: null args");
  const mj_block_evict_args& a = *args;
  if (a.num_seqs < 0 || a.budget < 0 || a.recent < 0 || a.recent > a.budget)
    return fail(MJ_ERR_INVALID, "mj_block_evict: num_seqs %d budget %d recent %d", a.num_seqs, a.budget, a.recent);
  const int64_t st[6] = {a.k_stride_page, a.k_stride_row, a.k_stride_head, a.v_stride_page, a.v_stride_row, a.v_stride_head};
  const int64_t ss[6] = {a.ks_stride_page, a.ks_stride_block, a.ks_stride_head, a.vs_stride_page, a.vs_stride_block, a.vs_stride_head};
  if (const char* why = block_cache_problem(a.head_size, a.kv_format, a.page_size, a.h_k, a.num_pages, a.k_cache, a.v_cache,
                                            st, a.k_scales, a.v_scales, ss, 16))
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_evict: %s (head_size %d, kv_format %d, page_size %d; 16-byte aligned rows)", why,
                a.head_size, a.kv_format, a.page_size);
  if (a.num_seqs == 0) {
    g_err[0] = 0;
    return MJ_OK;
  }
  if (!a.block_table || a.block_table_cols <= 0 || !a.seq_lens || !a.weights || !a.new_lens || (a.budget && !a.kept))
    return fail(MJ_ERR_INVALID, "mj_block_evict: null pointer argument");
  if (a.weights_cols < 0 || a.weights_cols > INT32_MAX - 65536 || a.w_stride_seq < 0 || a.w_stride_head < 0)
    return fail(MJ_ERR_INVALID, "mj_block_evict: weights of %lld columns", (long long)a.weights_cols);
  if (rows_overlap(a.num_seqs, a.w_stride_seq, a.h_k, a.w_stride_head, a.weights_cols))
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_evict: a weights stride by which rows share elements");
  if (a.new_lens < a.seq_lens + a.num_seqs && a.seq_lens < a.new_lens + a.num_seqs)
    return fail(MJ_ERR_INVALID, "mj_block_evict: new_lens overlaps seq_lens, which every KV head reads");
  if ((int64_t)a.num_seqs * a.h_k > 1 << 24 || a.budget > 1 << 24) return fail(MJ_ERR_UNSUPPORTED, "mj_block_evict: too many rows");
  if (shared_bytes(st, a.num_pages, a.page_size, a.h_k) ||
      shared_bytes(ss, a.num_pages, a.page_size >> mj::block_log2(a.kv_format), a.h_k))
    return fail(MJ_ERR_UNSUPPORTED, "mj_block_evict: a cache or scale stride of 0");
  return cuda_status(mj::launch_block_evict(a, (cudaStream_t)stream), "mj_block_evict launch");
}

}  // extern "C"
