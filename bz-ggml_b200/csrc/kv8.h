// The 8-bit paged key/value cache: what the C entry points (include/bzb_ext.h) hand to its kernels.
#pragma once

#include <cuda_runtime.h>

#include "../../include/bzb_ext.h"

namespace bzb {

// Each checks its arguments (std::runtime_error names the one that is wrong) and enqueues on `s`,
// on the current device; nothing is allocated and nothing is waited for.
void kv8_append(const bzb_kv8_cache & c, const bzb_kv8_batch & b, const bzb_kv8_rows * q, const bzb_kv8_rows & k,
                const bzb_kv8_rows & v, const bzb_kv8_rows * q_out, const float * q_norm, const float * k_norm, float eps,
                const float * rope, int rope_len, cudaStream_t s);
void kv8_read(const bzb_kv8_cache & c, const bzb_kv8_batch & b, const bzb_kv8_rows & k_out, const bzb_kv8_rows & v_out,
              cudaStream_t s);
long long kv8_attention_workspace(const bzb_kv8_cache & c, const bzb_kv8_batch & b, int n_head, int causal, int window);
void kv8_attention(const bzb_kv8_cache & c, const bzb_kv8_batch & b, const bzb_kv8_rows & q, const bzb_kv8_rows & out,
                   float * lse, float scale, int causal, int window, void * workspace, long long workspace_bytes,
                   cudaStream_t s);

// the many-row kernel's poll limit in the calls that follow (tests; negative: the default)
void kv8_debug_polls(long long polls);

}  // namespace bzb
