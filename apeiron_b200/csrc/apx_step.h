// apx_step.h — launchers of the steps between the projections (norm, positions and KV append,
// attention, sampler), called by their C entry points in apx_step.cu after validation.
#pragma once

#include <cuda_runtime.h>

#include "../../include/apeiron_cuda.h"

namespace apx {

// apx_norm.cu
cudaError_t launch_add_rms_norm_quant(const apx_norm_args &a, int sms, cudaStream_t stream);

// apx_rope.cu
cudaError_t launch_rope_table(const apx_rope_freqs &f, size_t n_pos, float *table,
                              cudaStream_t stream);
cudaError_t launch_rope_kv4_append(const apx_rope_args &a, const apx_kv4_cache &c,
                                   const apx_seq_batch &b, cudaStream_t stream);

// apx_attn.cu.  work: attn_work_bytes(sms) bytes, zero before the first call that uses them.
size_t attn_work_bytes(int sms);
cudaError_t launch_attn_kv4(const apx_attn_args &a, const apx_kv4_cache &c,
                            const apx_seq_batch &b, void *work, int sms, cudaStream_t stream);

// apx_runtime.cu: the context's attention workspace (attn_work_bytes, zeroed when the context was
// opened), its SM count and its device.
void *context_attn_work(apx_ctx *ctx);
int context_sms(const apx_ctx *ctx);
int context_device(const apx_ctx *ctx);

// apx_sample.cu
cudaError_t launch_sample(const apx_sample_args &a, int sms, cudaStream_t stream);

}  // namespace apx
