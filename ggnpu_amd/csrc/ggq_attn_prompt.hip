// ggq_attn_prompt.hip -- causal attention of packed prompts.
#include "ggq_attn.h"
#include "ggq_launch.h"

namespace ggq {
namespace {

// The sequence of a row: the number of offsets behind the first one that are not above it.  All threads
// of the workgroup call it.
__device__ __forceinline__ int seq_of(const int32_t* off, int n_seq, int row) {
    int s = 0;
    for (int i = 0; i < n_seq; i += 256) {
        const int j = i + (int)threadIdx.x;
        s += __syncthreads_count(j < n_seq && off[j + 1] <= row);
    }
    return s;
}

// One query row of four heads, a wavefront a head.  64 positions at a time: a
// lane has a position for the scores, HD / 64 values for the sum.
template <int HD, typename T>
__global__ __launch_bounds__(256) void attn_rows_kernel(ggq_attention_prompt_params a) {
    constexpr int DPL = HD / 64;
    __shared__ float sq[4][HD], sp[4][64];
    const int row = blockIdx.x, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int head = blockIdx.y * 4 + wave;
    const int seq = seq_of(a.q_off, a.n_seq, row);
    if (seq >= a.n_seq || row < a.q_off[seq]) return;
    if (head >= a.n_head) return;
    const int32_t* kvo = a.kv_off ? a.kv_off : a.q_off;
    const int64_t k0 = max(kvo[seq], 0), k1 = min(kvo[seq + 1], a.n_kv_rows);
    // behind the last position it sees
    const int64_t end = min(k1, k1 - ((int64_t)a.q_off[seq + 1] - 1 - row));
    int64_t beg = k0;
    if (a.window > 0) beg = max(beg, end - a.window);
    const int kvh = head / (a.n_head / a.n_kv_head);
    const float* q = a.q + (int64_t)row * a.ldq + (int64_t)head * HD;
    for (int i = lane; i < HD; i += 64) sq[wave][i] = q[i] * a.scale;
    __builtin_amdgcn_wave_barrier();
    float m = -INFINITY, l = 0.0f, o[DPL] = {};
    for (int64_t j0 = beg; j0 < end; j0 += 64) {
        const int n = (int)min<int64_t>(64, end - j0);
        float s = -INFINITY;
        if (lane < n) {
            const T* k = (const T*)a.k + (j0 + lane) * a.ldk + (int64_t)kvh * HD;
            s = 0.0f;
            for (int i = 0; i < HD; i++) s = fmaf(sq[wave][i], (float)k[i], s);
        }
        float mx = s;
        for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
        const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.0f : mn;
        const float al = exp2f(m - ref), p = lane < n ? exp2f(s - ref) : 0.0f;
        float ps = p;
        for (int off = 32; off > 0; off >>= 1) ps += __shfl_xor(ps, off, 64);
        l = l * al + ps;
        m = mn;
        sp[wave][lane] = p;
        __builtin_amdgcn_wave_barrier();
        for (int i = 0; i < DPL; i++) o[i] *= al;
        const T* v = (const T*)a.v + j0 * a.ldv + (int64_t)kvh * HD + lane;
        for (int j = 0; j < n; j++)
            for (int i = 0; i < DPL; i++) o[i] = fmaf(sp[wave][j], (float)v[j * a.ldv + 64 * i], o[i]);
        __builtin_amdgcn_wave_barrier();
    }
    float* out = a.out + (int64_t)row * a.ldo + (int64_t)head * HD + lane;
    for (int i = 0; i < DPL; i++) out[64 * i] = end <= beg ? 0.0f : o[i] / l;
}

}  // namespace

hipError_t launch_attn_prompt(const ggq_attention_prompt_params& p, hipStream_t s) {
    const dim3 grid((unsigned)p.n_rows, (unsigned)((p.n_head + 3) / 4));
#define L(HD_)                                                                       \
    if (p.type == GGQ_TYPE_F32) attn_rows_kernel<HD_, float><<<grid, 256, 0, s>>>(p); \
    else attn_rows_kernel<HD_, _Float16><<<grid, 256, 0, s>>>(p)
    if (p.head_dim == 64) { L(64); }
    else if (p.head_dim == 128) { L(128); }
    else { L(256); }
#undef L
    return hipGetLastError();
}

}  // namespace ggq
