// ggq_steps.h -- launchers of the operators around a layer's matmuls in a step
// over new tokens (ggq_norm.hip, ggq_sample.hip, ggq_delta.hip, ggq_kv_chunk.hip).
// All are asynchronous on `s`; shapes are validated by the caller (ggq_api.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ggq.h"
#include "ggq_attn.h"

namespace ggq {

hipError_t launch_norm(const ggq_norm_params& p, hipStream_t s);

// Sampling; ws holds sample_ws_bytes(...) bytes.
size_t sample_ws_bytes(const ggq_sample_params& p);
hipError_t launch_sample(const ggq_sample_params& p, void* ws, hipStream_t s);

// Gated delta rule.  Row by row without a workspace, in parts of 16 rows with
// delta_ws_bytes(...) bytes (0: row by row is the better choice).  `scale` is
// what q is multiplied by.
size_t delta_ws_bytes(const ggq_delta_rule_params& p);
hipError_t launch_delta(const ggq_delta_rule_params& p, void* ws, hipStream_t s);

// Attention of several rows a sequence over its quantized cache.  scale in powers of two.
struct KvChunkArgs {
    ggq_kv_cache c;
    ggq_kv_seqs q;
    const int32_t* row_off;  // null: one row a sequence
    int n_rows;
    const float* Q;
    int64_t ldq;
    int n_head;
    float scale;
    int window;
    float* out;
    int64_t ldo;
};
struct KvChunkPlan {
    int tiles;              // column tiles of a wavefront; 0: by planes of operands, as prompts
    AttnPromptPlan planes;
    int splits;
    size_t ws_bytes;
};
KvChunkPlan kv_chunk_plan(const KvChunkArgs& a, bool workspace);
hipError_t launch_kv_chunk(const KvChunkArgs& a, const KvChunkPlan& pl, void* ws, hipStream_t s);
// (ggq_attn_prompt.hip)
AttnPromptPlan attn_kv_planes_plan(const KvChunkArgs& a);
hipError_t launch_attn_kv_planes(const KvChunkArgs& a, const AttnPromptPlan& pl, void* ws, hipStream_t s);

}  // namespace ggq
