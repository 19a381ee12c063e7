// C-ABI entry points of the paged-cache serving operators (declared in
// include/enl_attn.h): argument validation and kernel launches. Shares the
// helpers of enl_abi.cu (one translation unit).

namespace enl {
namespace {

int check_dtype(const char* fn, const char* name, int32_t dtype) {
  if (dtype != ENL_DTYPE_BF16 && dtype != ENL_DTYPE_FP32)
    return fail(ENL_ERR_INVALID, "%s: %s=%d", fn, name, dtype);
  return ENL_OK;
}

int check_heads(const char* fn, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim) {
  if (num_heads < 1 || num_kv_heads < 1 || num_heads % num_kv_heads != 0)
    return fail(ENL_ERR_INVALID, "%s: num_kv_heads=%d must divide num_heads=%d", fn, num_kv_heads,
                num_heads);
  if (head_dim < 8 || head_dim > 128 || head_dim % 8 != 0)
    return fail(ENL_ERR_UNSUPPORTED, "%s: head_dim=%d (supported: multiples of 8 up to 128)", fn,
                head_dim);
  return ENL_OK;
}

int elem_bytes(int32_t dtype) { return dtype == ENL_DTYPE_FP32 ? 4 : 2; }

// A strided (batch, seq, heads, head_dim) operand.
int check_operand(const char* fn, const char* name, const void* ptr, int64_t sb, int64_t ss,
                  int64_t sh, int32_t dtype) {
  if (!ptr) return fail(ENL_ERR_INVALID, "%s: %s must be non-NULL", fn, name);
  if (!aligned16(ptr)) return fail(ENL_ERR_INVALID, "%s: %s must be 16-byte aligned", fn, name);
  return check_strides_16B(name, sb, ss, sh, elem_bytes(dtype));
}

int check_pool(const char* fn, const void* k, const void* v, int64_t sp, int64_t sh, int64_t ss,
               int32_t num_pages, int32_t page_size, const int32_t* table, int64_t table_stride,
               int32_t max_pages, int32_t dtype) {
  if (!k || !v || !table)
    return fail(ENL_ERR_INVALID, "%s: k_pages, v_pages and block_table must be non-NULL", fn);
  if (!aligned16(k) || !aligned16(v))
    return fail(ENL_ERR_INVALID, "%s: k_pages and v_pages must be 16-byte aligned", fn);
  if (int st = check_strides_16B("page", sp, ss, sh, elem_bytes(dtype))) return st;
  if (num_pages < 1 || page_size < 1 || max_pages < 1 || table_stride < 0 ||
      (long long)max_pages * page_size > 0x7fffffffll)
    return fail(ENL_ERR_INVALID,
                "%s: num_pages=%d page_size=%d max_pages=%d table_stride_b=%lld out of range "
                "(max_pages * page_size must stay below 2^31)",
                fn, num_pages, page_size, max_pages, (long long)table_stride);
  return ENL_OK;
}

// (token, head) pairs are numbered with 32 bits, those that fill up a last block too.
int check_units(const char* fn, int32_t batch, int32_t seq, int32_t num_heads) {
  if ((long long)batch * seq * num_heads > 0x7fffffffll - 256)
    return fail(ENL_ERR_UNSUPPORTED, "%s: batch * seq * num_heads = %lld exceeds 2^31 - 257", fn,
                (long long)batch * seq * num_heads);
  return ENL_OK;
}

// The norm weights and rotation tables that forward and backward share.
int check_norm_rope(const char* fn, const float* wq, const float* wk, const float* cos_t,
                    const float* sin_t, int64_t rows) {
  if ((wq == nullptr) != (wk == nullptr))
    return fail(ENL_ERR_INVALID, "%s: q_weight and k_weight come in pairs", fn);
  if ((cos_t == nullptr) != (sin_t == nullptr))
    return fail(ENL_ERR_INVALID, "%s: rope_cos and rope_sin come in pairs", fn);
  if (cos_t && rows < 1)
    return fail(ENL_ERR_INVALID, "%s: rope_rows=%lld must be >= 1", fn, (long long)rows);
  if ((wq && (!aligned16(wq) || !aligned16(wk))) || (cos_t && (!aligned16(cos_t) || !aligned16(sin_t))))
    return fail(ENL_ERR_INVALID, "%s: weights and tables must be 16-byte aligned", fn);
  return ENL_OK;
}

}  // namespace
}  // namespace enl

extern "C" {

int enl_qk_norm_rope(const enl_qk_norm_rope_args* a, void* stream) {
  const char* fn = "enl_qk_norm_rope";
  if (!a) return fail(ENL_ERR_INVALID, "%s: args is NULL", fn);
  if (a->batch < 0 || a->seq < 0)
    return fail(ENL_ERR_INVALID, "%s: batch=%d seq=%d must be >= 0", fn, a->batch, a->seq);
  int st;
  if ((st = check_heads(fn, a->num_heads, a->num_kv_heads, a->head_dim))) return st;
  if ((st = check_dtype(fn, "in_dtype", a->in_dtype))) return st;
  if ((st = check_dtype(fn, "out_dtype", a->out_dtype))) return st;
  if ((st = check_norm_rope(fn, a->q_weight, a->k_weight, a->rope_cos, a->rope_sin, a->rope_rows)))
    return st;
  const bool paged = a->k_pages || a->v_pages;
  if (!paged && !a->q_weight && !a->rope_cos)
    return fail(ENL_ERR_INVALID, "%s: needs norm weights, rotation tables or both", fn);
  if (!paged && a->n_new) return fail(ENL_ERR_INVALID, "%s: n_new needs k_pages", fn);
  if (a->batch == 0 || a->seq == 0) return ENL_OK;
  if ((st = check_units(fn, a->batch, a->seq, a->num_heads))) return st;
  if ((st = check_operand(fn, "q", a->q, a->q_stride_b, a->q_stride_s, a->q_stride_h, a->in_dtype)))
    return st;
  if ((st = check_operand(fn, "k", a->k, a->k_stride_b, a->k_stride_s, a->k_stride_h, a->in_dtype)))
    return st;
  if ((st = check_operand(fn, "q_out", a->q_out, a->qo_stride_b, a->qo_stride_s, a->qo_stride_h,
                          a->out_dtype)))
    return st;
  if (paged) {
    if ((st = check_operand(fn, "v", a->v, a->v_stride_b, a->v_stride_s, a->v_stride_h,
                            a->in_dtype)))
      return st;
    if ((st = check_pool(fn, a->k_pages, a->v_pages, a->page_stride_p, a->page_stride_h,
                         a->page_stride_s, a->num_pages, a->page_size, a->block_table,
                         a->table_stride_b, a->max_pages, a->out_dtype)))
      return st;
    if (!a->start) return fail(ENL_ERR_INVALID, "%s: start must be non-NULL with k_pages", fn);
    if (a->in_dtype != a->out_dtype)
      return fail(ENL_ERR_INVALID, "%s: in_dtype and out_dtype must be equal with k_pages", fn);
    if (a->pos0 != 0)
      return fail(ENL_ERR_INVALID, "%s: pos0 must be 0 with k_pages (positions are slots)", fn);
  } else if ((st = check_operand(fn, "k_out", a->k_out, a->ko_stride_b, a->ko_stride_s,
                                 a->ko_stride_h, a->out_dtype))) {
    return st;
  }
  QkRopeParams p{};
  p.B = a->batch, p.S = a->seq, p.H = a->num_heads, p.Hkv = a->num_kv_heads, p.D = a->head_dim;
  p.x[0] = a->q, p.x_sb[0] = a->q_stride_b, p.x_ss[0] = a->q_stride_s, p.x_sh[0] = a->q_stride_h;
  p.x[1] = a->k, p.x_sb[1] = a->k_stride_b, p.x_ss[1] = a->k_stride_s, p.x_sh[1] = a->k_stride_h;
  p.x[2] = a->v, p.x_sb[2] = a->v_stride_b, p.x_ss[2] = a->v_stride_s, p.x_sh[2] = a->v_stride_h;
  p.y[0] = a->q_out, p.y_sb[0] = a->qo_stride_b, p.y_ss[0] = a->qo_stride_s,
  p.y_sh[0] = a->qo_stride_h;
  p.y[1] = a->k_out, p.y_sb[1] = a->ko_stride_b, p.y_ss[1] = a->ko_stride_s,
  p.y_sh[1] = a->ko_stride_h;
  p.in_fp32 = a->in_dtype == ENL_DTYPE_FP32;
  p.out_fp32 = a->out_dtype == ENL_DTYPE_FP32;
  p.w[0] = a->q_weight, p.w[1] = a->k_weight;
  p.eps = a->eps;
  p.cos_t = a->rope_cos, p.sin_t = a->rope_sin;
  p.rows = a->rope_rows, p.pos0 = a->pos0, p.start = a->start;
  if (paged) {
    p.pages[0] = a->k_pages, p.pages[1] = a->v_pages;
    p.p_sp = a->page_stride_p, p.p_sh = a->page_stride_h, p.p_ss = a->page_stride_s;
    p.n_pages = a->num_pages, p.page_size = a->page_size;
    p.table = a->block_table, p.t_sb = a->table_stride_b, p.max_pages = a->max_pages;
    p.n_new = a->n_new;
  }
  cudaError_t e = launch_qk_norm_rope(p, reinterpret_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "enl_qk_norm_rope launch");
  return ENL_OK;
}

size_t enl_qk_norm_rope_backward_workspace_bytes(const enl_qk_norm_rope_backward_args* a) {
  if (!a || !a->q_weight || a->batch < 1 || a->seq < 1 || a->num_heads < 1 ||
      a->num_kv_heads < 1 || a->head_dim < 8 || a->head_dim > 128)
    return 0;
  int sms = 0;
  if (sm_count(&sms)) return 0;
  return (size_t)qk_rope_bwd_blocks(a->batch, a->seq, a->num_heads, a->num_kv_heads, a->head_dim,
                                    sms) * a->head_dim * sizeof(float);
}

int enl_qk_norm_rope_backward(const enl_qk_norm_rope_backward_args* a, void* stream) {
  const char* fn = "enl_qk_norm_rope_backward";
  if (!a) return fail(ENL_ERR_INVALID, "%s: args is NULL", fn);
  if (a->batch < 1 || a->seq < 1)
    return fail(ENL_ERR_INVALID, "%s: batch=%d seq=%d must be >= 1", fn, a->batch, a->seq);
  int st;
  if ((st = check_heads(fn, a->num_heads, a->num_kv_heads, a->head_dim))) return st;
  if ((st = check_dtype(fn, "in_dtype", a->in_dtype))) return st;
  if ((st = check_dtype(fn, "grad_dtype", a->grad_dtype))) return st;
  if ((st = check_dtype(fn, "out_dtype", a->out_dtype))) return st;
  if ((st = check_norm_rope(fn, a->q_weight, a->k_weight, a->rope_cos, a->rope_sin, a->rope_rows)))
    return st;
  if (!a->q_weight && !a->rope_cos)
    return fail(ENL_ERR_INVALID, "%s: needs norm weights, rotation tables or both", fn);
  if ((st = check_units(fn, a->batch, a->seq, a->num_heads))) return st;
  if ((st = check_operand(fn, "dq_out", a->dq_out, a->dqo_stride_b, a->dqo_stride_s,
                          a->dqo_stride_h, a->grad_dtype)))
    return st;
  if ((st = check_operand(fn, "dk_out", a->dk_out, a->dko_stride_b, a->dko_stride_s,
                          a->dko_stride_h, a->grad_dtype)))
    return st;
  if ((st = check_operand(fn, "dq", a->dq, a->dq_stride_b, a->dq_stride_s, a->dq_stride_h,
                          a->out_dtype)))
    return st;
  if ((st = check_operand(fn, "dk", a->dk, a->dk_stride_b, a->dk_stride_s, a->dk_stride_h,
                          a->out_dtype)))
    return st;
  int sms = 0;
  if ((st = sm_count(&sms))) return st;
  const int blocks =
      qk_rope_bwd_blocks(a->batch, a->seq, a->num_heads, a->num_kv_heads, a->head_dim, sms);
  if (a->q_weight) {
    if ((st = check_operand(fn, "q", a->q, a->q_stride_b, a->q_stride_s, a->q_stride_h,
                            a->in_dtype)))
      return st;
    if ((st = check_operand(fn, "k", a->k, a->k_stride_b, a->k_stride_s, a->k_stride_h,
                            a->in_dtype)))
      return st;
    if (!a->dq_weight || !a->dk_weight)
      return fail(ENL_ERR_INVALID, "%s: dq_weight and dk_weight must be non-NULL with norm weights",
                  fn);
    const size_t need = (size_t)blocks * a->head_dim * sizeof(float);
    if (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace))
      return fail(ENL_ERR_INVALID, "%s: needs a 16-byte aligned workspace of %zu bytes (got %zu)",
                  fn, need, a->workspace ? a->workspace_bytes : (size_t)0);
  }
  QkRopeBwdParams p{};
  p.B = a->batch, p.S = a->seq, p.H = a->num_heads, p.Hkv = a->num_kv_heads, p.D = a->head_dim;
  p.dy[0] = a->dq_out, p.dy_sb[0] = a->dqo_stride_b, p.dy_ss[0] = a->dqo_stride_s,
  p.dy_sh[0] = a->dqo_stride_h;
  p.dy[1] = a->dk_out, p.dy_sb[1] = a->dko_stride_b, p.dy_ss[1] = a->dko_stride_s,
  p.dy_sh[1] = a->dko_stride_h;
  p.x[0] = a->q, p.x_sb[0] = a->q_stride_b, p.x_ss[0] = a->q_stride_s, p.x_sh[0] = a->q_stride_h;
  p.x[1] = a->k, p.x_sb[1] = a->k_stride_b, p.x_ss[1] = a->k_stride_s, p.x_sh[1] = a->k_stride_h;
  p.dx[0] = a->dq, p.dx_sb[0] = a->dq_stride_b, p.dx_ss[0] = a->dq_stride_s,
  p.dx_sh[0] = a->dq_stride_h;
  p.dx[1] = a->dk, p.dx_sb[1] = a->dk_stride_b, p.dx_ss[1] = a->dk_stride_s,
  p.dx_sh[1] = a->dk_stride_h;
  p.dw[0] = a->dq_weight, p.dw[1] = a->dk_weight;
  p.in_fp32 = a->in_dtype == ENL_DTYPE_FP32;
  p.grad_fp32 = a->grad_dtype == ENL_DTYPE_FP32;
  p.out_fp32 = a->out_dtype == ENL_DTYPE_FP32;
  p.w[0] = a->q_weight, p.w[1] = a->k_weight;
  p.eps = a->eps;
  p.cos_t = a->rope_cos, p.sin_t = a->rope_sin;
  p.rows = a->rope_rows, p.pos0 = a->pos0, p.start = a->start;
  p.partial = reinterpret_cast<float*>(a->workspace);
  p.n_blocks = blocks;
  cudaError_t e = launch_qk_norm_rope_backward(p, reinterpret_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "enl_qk_norm_rope_backward launch");
  return ENL_OK;
}

size_t enl_paged_decode_workspace_bytes(const enl_paged_decode_args* a) {
  if (!a || a->batch < 1 || a->num_heads < 1 || a->num_kv_heads < 1 || a->head_dim < 1) return 0;
  int sms = 0;
  if (sm_count(&sms)) return 0;
  return paged_decode_workspace(a->batch, a->num_heads, a->num_kv_heads, a->head_dim, sms);
}

int enl_attn_decode_paged(const enl_paged_decode_args* a, void* stream) {
  const char* fn = "enl_attn_decode_paged";
  if (!a) return fail(ENL_ERR_INVALID, "%s: args is NULL", fn);
  if (a->batch < 0) return fail(ENL_ERR_INVALID, "%s: batch=%d must be >= 0", fn, a->batch);
  int st;
  if ((st = check_heads(fn, a->num_heads, a->num_kv_heads, a->head_dim))) return st;
  if ((st = check_dtype(fn, "in_dtype", a->in_dtype))) return st;
  if ((st = check_dtype(fn, "out_dtype", a->out_dtype))) return st;
  if (a->sinks < 0) return fail(ENL_ERR_INVALID, "%s: sinks=%d must be >= 0", fn, a->sinks);
  if (a->batch == 0) return ENL_OK;
  if (!a->seq_lens) return fail(ENL_ERR_INVALID, "%s: seq_lens must be non-NULL", fn);
  if ((st = check_operand(fn, "q", a->q, a->q_stride_b, 0, a->q_stride_h, a->in_dtype))) return st;
  if ((st = check_operand(fn, "o", a->o, a->o_stride_b, 0, a->o_stride_h, a->out_dtype))) return st;
  if ((st = check_pool(fn, a->k_pages, a->v_pages, a->page_stride_p, a->page_stride_h,
                       a->page_stride_s, a->num_pages, a->page_size, a->block_table,
                       a->table_stride_b, a->max_pages, a->in_dtype)))
    return st;
  if (a->batch > 65535)
    return fail(ENL_ERR_UNSUPPORTED, "%s: batch=%d exceeds 65535", fn, a->batch);
  PagedDecodeParams p{};
  if ((st = sm_count(&p.n_sms))) return st;
  const size_t need =
      paged_decode_workspace(a->batch, a->num_heads, a->num_kv_heads, a->head_dim, p.n_sms);
  if (!a->workspace || a->workspace_bytes < need ||
      (reinterpret_cast<uintptr_t>(a->workspace) & 255u) != 0)
    return fail(ENL_ERR_INVALID, "%s: needs a 256-byte aligned workspace of %zu bytes (got %zu)",
                fn, need, a->workspace ? a->workspace_bytes : (size_t)0);
  p.q = a->q, p.q_sb = a->q_stride_b, p.q_sh = a->q_stride_h;
  p.k = a->k_pages, p.v = a->v_pages;
  p.p_sp = a->page_stride_p, p.p_sh = a->page_stride_h, p.p_ss = a->page_stride_s;
  p.n_pages = a->num_pages, p.page_size = a->page_size;
  p.table = a->block_table, p.t_sb = a->table_stride_b, p.max_pages = a->max_pages;
  p.lens = a->seq_lens;
  p.o = a->o, p.o_sb = a->o_stride_b, p.o_sh = a->o_stride_h;
  p.lse = a->lse;
  p.B = a->batch, p.H = a->num_heads, p.Hkv = a->num_kv_heads, p.D = a->head_dim;
  p.window = a->window < 0 ? -1 : a->window;
  p.sinks = a->window < 0 ? 0 : a->sinks;
  p.alibi = a->alibi_slopes;
  p.scale = a->scale;
  p.in_fp32 = a->in_dtype == ENL_DTYPE_FP32;
  p.out_fp32 = a->out_dtype == ENL_DTYPE_FP32;
  p.workspace = a->workspace;
  cudaError_t e = launch_paged_decode(p, reinterpret_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "enl_attn_decode_paged launch");
  return ENL_OK;
}

int enl_sample_tokens(const enl_sample_args* a, void* stream) {
  const char* fn = "enl_sample_tokens";
  if (!a) return fail(ENL_ERR_INVALID, "%s: args is NULL", fn);
  if (a->batch < 0) return fail(ENL_ERR_INVALID, "%s: batch=%d must be >= 0", fn, a->batch);
  if (a->vocab < 1 || a->vocab > (1 << 22))
    return fail(ENL_ERR_UNSUPPORTED, "%s: vocab=%d (supported: 1 to 2^22)", fn, a->vocab);
  if (int st = check_dtype(fn, "dtype", a->dtype)) return st;
  if (a->batch == 0) return ENL_OK;
  if (!a->logits || !a->u || !a->tokens)
    return fail(ENL_ERR_INVALID, "%s: logits, u and tokens must be non-NULL", fn);
  if (a->batch > 1 && a->stride_b < a->vocab)
    return fail(ENL_ERR_INVALID, "%s: stride_b=%lld is less than vocab=%d", fn,
                (long long)a->stride_b, a->vocab);
  if ((reinterpret_cast<uintptr_t>(a->logits) & (elem_bytes(a->dtype) - 1)) != 0)
    return fail(ENL_ERR_INVALID, "%s: logits are not aligned to their elements", fn);
  SampleParams p{};
  p.logits = a->logits, p.stride = a->stride_b, p.fp32 = a->dtype == ENL_DTYPE_FP32;
  p.B = a->batch, p.V = a->vocab, p.u = a->u;
  p.temperature = a->temperature, p.top_k = a->top_k, p.top_p = a->top_p, p.min_p = a->min_p;
  p.temperature_all = a->temperature_all, p.top_k_all = a->top_k_all;
  p.top_p_all = a->top_p_all, p.min_p_all = a->min_p_all;
  p.tokens = reinterpret_cast<long long*>(a->tokens);
  if (int st = sm_count(&p.n_sms)) return st;
  cudaError_t e = launch_sample(p, reinterpret_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(e, "enl_sample_tokens launch");
  return ENL_OK;
}

}  // extern "C"
