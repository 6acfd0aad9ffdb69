// apx_step.cu — C entry points of the steps between the projections: argument checks, then the
// launchers of apx_step.h.
#include <cstdint>

#include "apx_kv4.cuh"
#include "apx_step.h"

namespace {

bool aligned(const void *p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Queues a launch on the context's device, whichever is current: kernels go to the current one, and
// a default stream says nothing of it.
template <typename Launch>
int on_device(const apx_ctx *ctx, Launch launch) {
  const int dev = apx::context_device(ctx);
  int now = -1;
  if (cudaGetDevice(&now) != cudaSuccess || (now != dev && cudaSetDevice(dev) != cudaSuccess))
    return APX_ERR_CUDA;
  const cudaError_t e = launch();
  if (now != dev) cudaSetDevice(now);
  return e == cudaSuccess ? APX_OK : APX_ERR_CUDA;
}

// The cache's geometry: APX_OK, or why it is not served.
int check_cache(const apx_kv4_cache *c) {
  if (!c || c->n_kv_heads <= 0) return APX_ERR_INVALID_ARGUMENT;
  if (!apx_kv4_page_bytes(c->head_dim, c->page_tokens)) return APX_ERR_LAYOUT_MISMATCH;
  if (c->n_pages > (size_t)INT32_MAX || c->n_kv_heads > 65535) return APX_ERR_TOO_LARGE;
  if (!c->d_pages || !aligned(c->d_pages, 16)) return APX_ERR_INVALID_ARGUMENT;
  return APX_OK;
}

int check_batch(const apx_seq_batch *b) {
  if (!b || b->n_seqs < 0 || b->max_pages < 0 || b->max_q < 0) return APX_ERR_INVALID_ARGUMENT;
  if (b->n_tokens > (size_t)INT32_MAX || b->n_seqs > 65535) return APX_ERR_TOO_LARGE;
  if (b->n_tokens == 0 || b->n_seqs == 0)
    return b->n_tokens == 0 ? APX_OK : APX_ERR_INVALID_ARGUMENT;
  if (!b->d_cu || !b->d_kv_len || (b->max_pages && !b->d_table) || b->max_q < 1 ||
      (size_t)b->max_q > b->n_tokens)
    return APX_ERR_INVALID_ARGUMENT;
  return APX_OK;
}

}  // namespace

extern "C" {

size_t apx_kv4_page_bytes(int head_dim, int page_tokens) {
  if (head_dim != 64 && head_dim != 128) return 0;
  if (page_tokens != 16 && page_tokens != 32 && page_tokens != 64 && page_tokens != 128) return 0;
  return (size_t)(page_tokens / apx::kKvTile) * apx::kv4_tile_bytes(head_dim);
}

int apx_add_rms_norm_quant_async(apx_ctx *ctx, const apx_norm_args *a, void *stream) {
  if (!ctx || !a) return APX_ERR_INVALID_ARGUMENT;
  if (a->n > (size_t)INT32_MAX - 256 || a->k > (size_t)INT32_MAX) return APX_ERR_TOO_LARGE;
  if (a->k == 0) return APX_OK;
  const bool any = a->d_codes || a->d_exps || a->d_descs;
  if (a->n == 0 || !a->d_x || a->ldx < a->n || (a->d_add && a->ld_add < a->n) ||
      (a->d_resid && a->ld_resid < a->n) || (a->d_y && a->ldy < a->n) ||
      (a->d_deq && (a->ld_deq < a->n || (a->deq_type != APX_DTYPE_F32 &&
                                         a->deq_type != APX_DTYPE_BF16))) ||
      (any && !(a->d_codes && a->d_exps && a->d_descs)) || !aligned(a->d_codes, 4) ||
      !aligned(a->d_descs, 16) || !(a->eps >= 0.0f))
    return APX_ERR_INVALID_ARGUMENT;
  const int sms = apx::context_sms(ctx);
  return on_device(
      ctx, [&] { return apx::launch_add_rms_norm_quant(*a, sms, (cudaStream_t)stream); });
}

int apx_rope_table_async(apx_ctx *ctx, const apx_rope_freqs *f, size_t n_pos, float *d_table,
                         void *stream) {
  if (!ctx || !f || f->rot_dim < 0 || f->rot_dim % 2 || !(f->base > 1.0) ||
      f->scaling < APX_ROPE_PLAIN || f->scaling > APX_ROPE_RAMP ||
      (f->scaling != APX_ROPE_PLAIN && !(f->factor > 0.0)) ||
      (f->scaling >= APX_ROPE_BANDS &&
       !(f->low > 0.0 && f->high > f->low && f->original > 0.0)))
    return APX_ERR_INVALID_ARGUMENT;
  if (n_pos > (size_t)INT32_MAX || f->rot_dim > 4096) return APX_ERR_TOO_LARGE;
  if (n_pos == 0 || f->rot_dim == 0) return APX_OK;
  if (!d_table || !aligned(d_table, 8)) return APX_ERR_INVALID_ARGUMENT;
  return on_device(
      ctx, [&] { return apx::launch_rope_table(*f, n_pos, d_table, (cudaStream_t)stream); });
}

int apx_rope_kv4_append_async(apx_ctx *ctx, const apx_rope_args *a, const apx_kv4_cache *c,
                              const apx_seq_batch *b, void *stream) {
  if (!ctx || !a) return APX_ERR_INVALID_ARGUMENT;
  int rc = check_cache(c);
  if (rc == APX_OK) rc = check_batch(b);
  if (rc != APX_OK) return rc;
  if (a->rot_dim < 0 || a->rot_dim % 8 || a->rot_dim > c->head_dim)
    return APX_ERR_LAYOUT_MISMATCH;
  if (a->layout != APX_ROPE_HALF && a->layout != APX_ROPE_INTERLEAVED)
    return APX_ERR_INVALID_ARGUMENT;
  if (a->n_heads < 0 || a->n_heads > 65535) return APX_ERR_INVALID_ARGUMENT;
  if (b->n_tokens == 0) return APX_OK;
  const size_t kv = (size_t)c->n_kv_heads * c->head_dim, nq = (size_t)a->n_heads * c->head_dim;
  if (!a->d_k || !a->d_v || a->ldk < kv || a->ldv < kv || a->ldk % 4 || a->ldv % 4 ||
      !aligned(a->d_k, 16) || !aligned(a->d_v, 16) || (a->d_q != nullptr) != (a->d_q_out != nullptr) ||
      a->n_pos > (size_t)INT32_MAX || (a->rot_dim && (!a->d_table || !aligned(a->d_table, 16))) ||
      !aligned(a->d_k_deq, 8) || !aligned(a->d_v_deq, 8))
    return APX_ERR_INVALID_ARGUMENT;
  if (a->d_q &&
      (a->n_heads == 0 || a->ldq < nq || a->ldq_out < nq || a->ldq % 4 || a->ldq_out % 4 ||
       !aligned(a->d_q, 16) || !aligned(a->d_q_out, 16) || a->q_type < APX_DTYPE_F32 ||
       a->q_type > APX_DTYPE_BF16))
    return APX_ERR_INVALID_ARGUMENT;
  if (a->d_q && a->d_q_out == a->d_q &&
      (a->q_type != APX_DTYPE_F32 || (a->ldq_out != a->ldq && b->n_tokens > 1)))
    return APX_ERR_INVALID_ARGUMENT;  // another token's values would be written over
  return on_device(
      ctx, [&] { return apx::launch_rope_kv4_append(*a, *c, *b, (cudaStream_t)stream); });
}

int apx_attn_kv4_async(apx_ctx *ctx, const apx_attn_args *a, const apx_kv4_cache *c,
                       const apx_seq_batch *b, void *stream) {
  if (!ctx || !a) return APX_ERR_INVALID_ARGUMENT;
  int rc = check_cache(c);
  if (rc == APX_OK) rc = check_batch(b);
  if (rc != APX_OK) return rc;
  if (a->n_heads <= 0 || a->n_heads > 65535 || a->type < APX_DTYPE_F32 ||
      a->type > APX_DTYPE_BF16 || a->window < 0 || a->sinks < 0 ||
      !(a->scale >= -3e38f && a->scale <= 3e38f))
    return APX_ERR_INVALID_ARGUMENT;
  if (a->n_heads % c->n_kv_heads) return APX_ERR_LAYOUT_MISMATCH;
  if (b->n_tokens == 0) return APX_OK;
  const size_t nq = (size_t)a->n_heads * c->head_dim, el = a->type == APX_DTYPE_F32 ? 4 : 2;
  if (!a->d_q || !a->d_out || a->ldq < nq || a->ldo < nq || a->ldq * el % 16 ||
      a->ldo * el % 16 || !aligned(a->d_q, 16) || !aligned(a->d_out, 16))
    return APX_ERR_INVALID_ARGUMENT;
  void *work = apx::context_attn_work(ctx);
  const int sms = apx::context_sms(ctx);
  return on_device(
      ctx, [&] { return apx::launch_attn_kv4(*a, *c, *b, work, sms, (cudaStream_t)stream); });
}

int apx_sample_async(apx_ctx *ctx, const apx_sample_args *a, void *stream) {
  if (!ctx || !a) return APX_ERR_INVALID_ARGUMENT;
  if (a->vocab > APX_SAMPLE_MAX_VOCAB || a->rows > 65535) return APX_ERR_TOO_LARGE;
  if (a->rows == 0) return APX_OK;
  if (!a->d_logits || !a->d_u || !a->d_token || a->vocab == 0 || a->ld < a->vocab)
    return APX_ERR_INVALID_ARGUMENT;
  const int sms = apx::context_sms(ctx);
  return on_device(ctx, [&] { return apx::launch_sample(*a, sms, (cudaStream_t)stream); });
}

}  // extern "C"
