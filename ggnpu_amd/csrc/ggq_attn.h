// ggq_attn.h -- launchers of the operators between the q/k/v and the output
// projections (ggq_rope.hip, ggq_kv_cache.hip, ggq_attn_prompt.hip).  All are
// asynchronous on `s`; shapes are validated by the caller (ggq_api.cpp).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/ggq.h"

namespace ggq {

// Heads turned to their positions.  turns[i]: turns of pair i per position.
struct RopeArgs {
    ggq_rope_heads set[GGQ_MAX_ROPE_SETS];
    int n_sets, n_tok, head_dim, rot_dim, layout;
    const double* turns;
    float mag, eps;
    const int32_t* pos;
};
hipError_t launch_rope(const RopeArgs& a, hipStream_t s);

// Quantized cache: one record holds 32 positions of one kv head.
constexpr int kKvTile = 32;
inline int64_t kv_record_bytes(const ggq_kv_cache& c) {
    return (int64_t)kKvTile * c.head_dim * (c.k_type + c.v_type) / 8 + 2 * c.head_dim;
}
struct KvRows {
    const int32_t* row_off;  // null: one row a sequence
    int n_rows;
    void* k;  // read by a store, written by a load
    void* v;
    int64_t ldk, ldv;
    int type;
};
hipError_t launch_kv_rows(const ggq_kv_cache& c, const ggq_kv_seqs& q, const KvRows& r, bool store, hipStream_t s);

// Attention of one row a sequence over the quantized cache.  The positions are
// taken in `splits` parts; ws holds kv_attn_ws_floats(...) floats (unused with
// one part).
struct KvAttnArgs {
    ggq_kv_cache c;
    ggq_kv_seqs q;
    const float* Q;
    int64_t ldq;
    int n_head;
    float scale;
    int window;
    float* out;
    int64_t ldo;
};
int kv_attn_splits(const KvAttnArgs& a);
size_t kv_attn_ws_floats(const KvAttnArgs& a, int splits);
hipError_t launch_kv_attn(const KvAttnArgs& a, int splits, float* ws, hipStream_t s);

// Causal attention of packed prompts: on the matrix cores with ws_bytes of
// workspace, or (few rows and keys, or no workspace) on the VALU without one.
struct AttnPromptPlan {
    bool few;
    int splits;
    size_t ws_bytes;
};
AttnPromptPlan attn_prompt_plan(const ggq_attention_prompt_params& p);
hipError_t launch_attn_prompt(const ggq_attention_prompt_params& p, const AttnPromptPlan& pl, void* ws, hipStream_t s);
hipError_t launch_attn_prompt_few(const ggq_attention_prompt_params& p, hipStream_t s);

}  // namespace ggq
