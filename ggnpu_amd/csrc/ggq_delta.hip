// ggq_delta.hip -- gated delta rule over packed sequences (ggq_delta_rule_dev).
//
// Per value head a state S of k_dim x v_dim numbers; a row's step is
//   S <- a S,  u = b (v - S^T k),  S <- S + k u^T,  o = S^T q.
// The columns of S (one a value) do not know of each other: both forms cut
// v_dim into slices and a workgroup keeps its slice in registers throughout.
//
// Row by row (delta_rows_kernel): a column is spread over 16 lanes, k_dim / 16
// numbers each; both dots of a row are taken of the state before it (S^T q after
// it is a S^T q + (k.q) u), so that their sums over the lanes run side by side.
// Single tokens are bound by their states' bytes.
//
// In parts of 16 rows: with G the running sum of the decays' logarithms within
// the part and c = exp(G), the rows' u obey
//   u_i = b_i (v_i - c_i S^T k_i) - sum_{j<i} M_ij u_j,  M_ij = b_i exp(G_i - G_j) k_i.k_j
// so U = T diag(b) (V - diag(c) K S) with T = (1 + M)^-1, and
//   O = diag(c) Q S + A U,  A_ij = exp(G_i - G_j) q_i.k_j (j <= i),  S <- exp(G_15) S + K^T diag(exp(G_15 - G)) U.
// delta_parts_kernel makes T diag(b), A and the rows' factors of every part
// at once (a wavefront a part and k head, up to four of its value heads side by
// side); delta_scan_kernel goes through the parts with four products of 16 rows,
// on fp32 matrix cores: exact products, no ranges to keep.  16 rows is where the
// products are fewest: 2 k + 32 rows' products a row beside 3 k_dim for the state.
// Its four wavefronts have a quarter of k each; sums over them go through LDS,
// one barrier a part.  S^T's rows in a lane are those that the next product's operand
// wants of that lane (step e of a product takes k = 4 g + e from lane group g), so the
// state goes from product to product in its registers.
#include <algorithm>
#include <cstdlib>

#include "ggq_device.h"
#include "ggq_steps.h"

namespace ggq {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct DeltaArgs {
    ggq_delta_rule_params p;
    float scale;
    float* parts;  // records of the parts
};

constexpr int kRows = 16;  // rows of a part
// A part's record of one value head, in floats: T diag(b) and A [16][16], then factors of its rows: of K S, of Q S,
// of U on its way into the state; the state's own.
constexpr int kT = 0, kA = 256, kKc = 512, kQc = 528, kKs = 544, kDec = 560, kRecord = 576;

// Sequence s has the parts from off / 16 + s on: a bound that needs no sum over the sequences before.
struct Seq {
    int64_t row;
    int n;
    int64_t part;
};
__device__ __forceinline__ Seq seq_of(const ggq_delta_rule_params& p, int s) {
    if (!p.row_off) return Seq{s, s < p.n_rows ? 1 : 0, (int64_t)s / kRows + s};
    const int a = min(max(p.row_off[s], 0), p.n_rows), b = min(max(p.row_off[s + 1], 0), p.n_rows);
    return Seq{a, b > a ? b - a : 0, (int64_t)a / kRows + s};
}
__device__ __forceinline__ int slot_of(const ggq_delta_rule_params& p, int s) {
    const int t = p.slot ? p.slot[s] : s;
    return t >= 0 && t < p.n_slots ? t : -1;
}

// The logarithm of a row's decay and its step.
__device__ __forceinline__ float decay_of(const ggq_delta_rule_params& p, int64_t row, int h) {
    float g = p.gate[row * p.ld_gate + h];
    if (p.gate_rate) {
        const float z = g + (p.gate_bias ? p.gate_bias[h] : 0.0f);
        // softplus(z) = max(z, 0) + log(1 + exp(-|z|))
        g = p.gate_rate[h] * (fmaxf(z, 0.0f) + log1pf(expf(-fabsf(z))));
    }
    return g;
}
__device__ __forceinline__ float step_of(const ggq_delta_rule_params& p, int64_t row, int h) {
    const float b = p.beta[row * p.ld_beta + h];
    return p.flags & GGQ_DELTA_BETA_SIGMOID ? 1.0f / (1.0f + expf(-b)) : b;
}

__device__ __forceinline__ float sum16(float v) {  // over 16 neighbouring lanes
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ float dot4(float4 a, float4 b, float s) {
    return fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, s))));
}

// C columns a group of 16 lanes: 16 C a workgroup.
template <int KD, int C>
__global__ __launch_bounds__(256) void delta_rows_kernel(DeltaArgs a) {
    constexpr int N = KD / 64;  // runs of four numbers of a lane, 64 apart
    const ggq_delta_rule_params& p = a.p;
    const int h = blockIdx.x, seq = blockIdx.z, j = threadIdx.x & 15, grp = threadIdx.x >> 4;
    const int slot = slot_of(p, seq);
    if (slot < 0) return;
    const Seq sq = seq_of(p, seq);
    const int hk = h / (p.n_v_head / p.n_k_head), d0 = blockIdx.y * 16 * C + grp;
    const int64_t at = ((int64_t)slot * p.n_v_head + h) * p.v_dim;
    float4 s[C][N];
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int i = 0; i < N; i++)
            s[c][i] = d0 + 16 * c < p.v_dim ? *(const float4*)(p.state + (at + d0 + 16 * c) * KD + 64 * i + 4 * j)
                                            : make_float4(0, 0, 0, 0);
    const float *qp = p.q + sq.row * p.ldq + (int64_t)hk * KD + 4 * j, *kp = p.k + sq.row * p.ldk + (int64_t)hk * KD + 4 * j;
    const float* vp = p.v + sq.row * p.ldv + (int64_t)h * p.v_dim + d0;
    float* op = p.out + sq.row * p.ldo + (int64_t)h * p.v_dim + d0;
    struct Row {
        float4 q[N], k[N];
        float v[C], g, b;
    };
    auto load = [&](int t, Row& x) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            x.q[i] = *(const float4*)(qp + t * p.ldq + 64 * i);
            x.k[i] = *(const float4*)(kp + t * p.ldk + 64 * i);
        }
#pragma unroll
        for (int c = 0; c < C; c++) x.v[c] = d0 + 16 * c < p.v_dim ? vp[t * p.ldv + 16 * c] : 0.0f;
        x.g = decay_of(p, sq.row + t, h);
        x.b = step_of(p, sq.row + t, h);
    };
    Row cur, nxt;
    if (sq.n) load(0, cur);
    for (int t = 0; t < sq.n; t++) {
        if (t + 1 < sq.n) load(t + 1, nxt);
        float kk = 0.0f, qq = 0.0f, kq = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            kk = dot4(cur.k[i], cur.k[i], kk);
            qq = dot4(cur.q[i], cur.q[i], qq);
            kq = dot4(cur.k[i], cur.q[i], kq);
        }
        kq = sum16(kq);
        float rk = 1.0f, rq = a.scale;
        if (p.flags & GGQ_DELTA_QK_NORM) {
            rk = 1.0f / sqrtf(sum16(kk) + p.eps);
            rq = a.scale / sqrtf(sum16(qq) + p.eps);
        }
        const float al = expf(cur.g);
        float ks[C], qs[C];
#pragma unroll
        for (int c = 0; c < C; c++) {
            ks[c] = qs[c] = 0.0f;
#pragma unroll
            for (int i = 0; i < N; i++) {
                ks[c] = dot4(s[c][i], cur.k[i], ks[c]);
                qs[c] = dot4(s[c][i], cur.q[i], qs[c]);
            }
        }
#pragma unroll
        for (int c = 0; c < C; c++) {
            ks[c] = sum16(ks[c]) * rk * al;
            qs[c] = sum16(qs[c]) * rq * al;
        }
        kq *= rk * rq;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const float u = cur.b * (cur.v[c] - ks[c]), o = fmaf(kq, u, qs[c]), w = u * rk;
            if (j == c && d0 + 16 * c < p.v_dim) op[t * p.ldo + 16 * c] = o;
#pragma unroll
            for (int i = 0; i < N; i++) {
                s[c][i].x = fmaf(cur.k[i].x, w, s[c][i].x * al);
                s[c][i].y = fmaf(cur.k[i].y, w, s[c][i].y * al);
                s[c][i].z = fmaf(cur.k[i].z, w, s[c][i].z * al);
                s[c][i].w = fmaf(cur.k[i].w, w, s[c][i].w * al);
            }
        }
        cur = nxt;
    }
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int i = 0; i < N; i++)
            if (d0 + 16 * c < p.v_dim) *(float4*)(p.state_out + (at + d0 + 16 * c) * KD + 64 * i + 4 * j) = s[c][i];
}

// A sum of logarithms as multiples of 2^-8, added exactly, and what is left: differences within a part lose nothing,
// however large the sums are.
struct Log {
    float hi, lo;
};
__device__ __forceinline__ float exp_of(Log a, Log b) { return expf((a.hi - b.hi) + (a.lo - b.lo)); }

template <int KD>
__global__ __launch_bounds__(256) void delta_parts_kernel(DeltaArgs a, int n_parts) {
    constexpr int NT = KD / 16;
    __shared__ float s_kk[4][16][17], s_qk[4][16][17];
    __shared__ __attribute__((aligned(16))) float s_m[4][4][16][20];
    __shared__ float s_row[4][4][16][4];  // of a head's rows: b, hi, lo
    __shared__ float s_r[4][16][2];       // of the rows: factors of k and q
    const ggq_delta_rule_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, r = lane & 15;
    const int id = blockIdx.x;
    int seq = 0;
    for (int i = 1; i < p.n_seq; i += 256) {
        const int j = i + tid;
        seq += __syncthreads_count(j < p.n_seq && (p.row_off ? (int64_t)min(max(p.row_off[j], 0), p.n_rows) : (int64_t)j) / kRows + j <= id);
    }
    const Seq sq = seq_of(p, seq);
    const int64_t first = (id - sq.part) * kRows;
    const int hk = blockIdx.y * 4 + wave;
    if (first < 0 || first >= sq.n || hk >= p.n_k_head || slot_of(p, seq) < 0) return;  // (no barrier from here on)
    const int n = (int)min((int64_t)kRows, sq.n - first);
    const int64_t row0 = sq.row + first, row = row0 + min(r, n - 1);
    const float *kp = p.k + row * p.ldk + (int64_t)hk * KD + 4 * g, *qp = p.q + row * p.ldq + (int64_t)hk * KD + 4 * g;
    float4 k[NT], q[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) k[t] = *(const float4*)(kp + 16 * t);
#pragma unroll
    for (int t = 0; t < NT; t++) q[t] = *(const float4*)(qp + 16 * t);
    f32x4 kk{0, 0, 0, 0}, qk{0, 0, 0, 0};
    float sk = 0.0f, sq2 = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const float kv[4] = {k[t].x, k[t].y, k[t].z, k[t].w}, qv[4] = {q[t].x, q[t].y, q[t].z, q[t].w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            kk = __builtin_amdgcn_mfma_f32_16x16x4f32(kv[e], kv[e], kk, 0, 0, 0);
            qk = __builtin_amdgcn_mfma_f32_16x16x4f32(qv[e], kv[e], qk, 0, 0, 0);
        }
        sk = dot4(k[t], k[t], sk);
        sq2 = dot4(q[t], q[t], sq2);
    }
    float rk = 1.0f, rq = a.scale;
    if (p.flags & GGQ_DELTA_QK_NORM) {
        sk += __shfl_xor(sk, 16, 64);
        sk += __shfl_xor(sk, 32, 64);
        sq2 += __shfl_xor(sq2, 16, 64);
        sq2 += __shfl_xor(sq2, 32, 64);
        rk = 1.0f / sqrtf(sk + p.eps);
        rq = a.scale / sqrtf(sq2 + p.eps);
    }
    if (r >= n) rk = rq = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        s_kk[wave][4 * g + e][r] = kk[e];
        s_qk[wave][4 * g + e][r] = qk[e];
    }
    if (g == 0) { s_r[wave][r][0] = rk; s_r[wave][r][1] = rq; }
    const int G = p.n_v_head / p.n_k_head;
    for (int h0 = 0; h0 < G; h0 += 4) {
        const int h = hk * G + min(h0 + g, G - 1);
        float ld = r < n ? decay_of(p, row, h) : 0.0f;
        ld = fminf(fmaxf(ld, -1000.0f), 1000.0f) + (ld - ld == 0.0f || ld == INFINITY || ld == -INFINITY ? 0.0f : ld);  // (NaN stays)
        const float b = r < n ? step_of(p, row, h) : 0.0f;
        Log L;
        L.hi = __builtin_rintf(ld * 256.0f) * (1.0f / 256.0f);
        L.lo = ld - L.hi;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const float x = __shfl_up(L.hi, o, 16), y = __shfl_up(L.lo, o, 16);
            if (r >= o) { L.hi += x; L.lo += y; }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        s_row[wave][g][r][0] = b;
        s_row[wave][g][r][1] = L.hi;
        s_row[wave][g][r][2] = L.lo;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // this lane's column r of M and A
        float* rec = a.parts + ((int64_t)id * p.n_v_head + h) * kRecord;
        const bool mine = h0 + g < G;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float* x = s_row[wave][g][i];
            const float e = i >= r ? exp_of(Log{x[1], x[2]}, L) : 0.0f;
            s_m[wave][g][i][r] = i > r ? x[0] * s_r[wave][i][0] * e * rk * s_kk[wave][i][r] : 0.0f;
            if (mine) rec[kA + 16 * i + r] = i >= r ? s_r[wave][i][1] * e * rk * s_qk[wave][i][r] : 0.0f;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // column r of (1 + M)^-1, from the top
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float v = i == r ? 1.0f : 0.0f;
#pragma unroll
            for (int m = 0; m < i; m++) v = fmaf(-s_m[wave][g][i][m], x[m], v);
            x[i] = v;
        }
        if (!mine) continue;
#pragma unroll
        for (int i = 0; i < 16; i++) rec[kT + 16 * i + r] = x[i] * b;
        const Log end{s_row[wave][g][15][1], s_row[wave][g][15][2]};
        const float c = expf(L.hi + L.lo);
        rec[kKc + r] = c * rk;
        rec[kQc + r] = c * rq;
        rec[kKs + r] = exp_of(end, L) * rk;
        if (r == 0) rec[kDec] = expf(end.hi + end.lo);
    }
}

template <int KD>
__global__ __launch_bounds__(256) void delta_scan_kernel(DeltaArgs a) {
    constexpr int NT = KD / 64;  // tiles of 16 numbers of k of a wavefront
    __shared__ __attribute__((aligned(16))) f32x4 s_ks[2][4][64], s_o[2][4][64];
    const ggq_delta_rule_params& p = a.p;
    const int h = blockIdx.x, seq = blockIdx.z, v0 = blockIdx.y * 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, r = lane & 15;
    const int slot = slot_of(p, seq);
    if (slot < 0) return;
    const Seq sq = seq_of(p, seq);
    const int hk = h / (p.n_v_head / p.n_k_head), k0 = wave * NT * 16;
    const int64_t at = (((int64_t)slot * p.n_v_head + h) * p.v_dim + v0 + r) * KD + k0 + 4 * g;
    f32x4 s[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) s[t] = *(const f32x4*)(p.state + at + 16 * t);
    const float *kp = p.k + sq.row * p.ldk + (int64_t)hk * KD + k0, *qp = p.q + sq.row * p.ldq + (int64_t)hk * KD + k0;
    const float* vp = p.v + sq.row * p.ldv + (int64_t)h * p.v_dim + v0 + r;
    float* op = p.out + sq.row * p.ldo + (int64_t)h * p.v_dim + v0;
    const float* rec0 = a.parts + (sq.part * p.n_v_head + h) * kRecord;
    const int parts = (sq.n + kRows - 1) / kRows;
    struct In {
        f32x4 k[NT], q[NT], kt[NT], v, t, kc, qc, ks;
        float a, dec;
    };
    auto load = [&](int i, In& x) {
        const int last = sq.n - 1, n0 = i * kRows;
        const int row = min(n0 + r, last);
        const float* rec = rec0 + (int64_t)i * p.n_v_head * kRecord;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            x.k[t] = *(const f32x4*)(kp + row * p.ldk + 16 * t + 4 * g);
            x.q[t] = *(const f32x4*)(qp + row * p.ldq + 16 * t + 4 * g);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int y = min(n0 + 4 * g + e, last);
#pragma unroll
            for (int t = 0; t < NT; t++) x.kt[t][e] = kp[y * p.ldk + 16 * t + r];
            x.v[e] = vp[y * p.ldv];
        }
        x.t = *(const f32x4*)(rec + kT + 16 * r + 4 * g);
        x.a = rec[kA + 16 * r + 4 * g + wave];
        x.kc = *(const f32x4*)(rec + kKc + 4 * g);
        x.qc = *(const f32x4*)(rec + kQc + 4 * g);
        x.ks = *(const f32x4*)(rec + kKs + 4 * g);
        x.dec = rec[kDec];
    };
    auto put = [&](int i) {  // the wavefronts' parts of O, 4 rows a wavefront
        const int row = i * kRows + 4 * wave + g;
        const float* o = (const float*)s_o[i & 1] + (wave * 16 + r) * 4 + g;
        const float v = (o[0] + o[256]) + (o[512] + o[768]);
        if (row < sq.n) op[row * p.ldo + r] = v;
    };
    In cur, nxt;
    if (parts) load(0, cur);
    for (int i = 0; i < parts; i++) {
        if (i + 1 < parts) load(i + 1, nxt);
        f32x4 ks{0, 0, 0, 0}, qs{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) ks = __builtin_amdgcn_mfma_f32_16x16x4f32(cur.k[t][e], s[t][e], ks, 0, 0, 0);
        s_ks[i & 1][wave][lane] = ks;
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) qs = __builtin_amdgcn_mfma_f32_16x16x4f32(cur.q[t][e], s[t][e], qs, 0, 0, 0);
        __syncthreads();
        if (i) put(i - 1);
        const f32x4* x = &s_ks[i & 1][0][lane];
        ks = (x[0] + x[64]) + (x[128] + x[192]);
        const f32x4 rest = cur.v - cur.kc * ks;
        f32x4 u{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; e++) u = __builtin_amdgcn_mfma_f32_16x16x4f32(cur.t[e], rest[e], u, 0, 0, 0);
        const float ue = wave == 0 ? u[0] : wave == 1 ? u[1] : wave == 2 ? u[2] : u[3];
        s_o[i & 1][wave][lane] = __builtin_amdgcn_mfma_f32_16x16x4f32(cur.a, ue, qs * cur.qc, 0, 0, 0);
        u *= cur.ks;
#pragma unroll
        for (int t = 0; t < NT; t++) {
            s[t] *= cur.dec;
#pragma unroll
            for (int e = 0; e < 4; e++) s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(cur.kt[t][e], u[e], s[t], 0, 0, 0);
        }
        cur = nxt;
    }
    __syncthreads();
    if (parts) put(parts - 1);
#pragma unroll
    for (int t = 0; t < NT; t++) *(f32x4*)(p.state_out + at + 16 * t) = s[t];
}

int64_t parts_of(const ggq_delta_rule_params& p) { return (int64_t)p.n_rows / kRows + p.n_seq; }

template <int KD> hipError_t delta_launch(const DeltaArgs& a, bool parts, hipStream_t s) {
    const ggq_delta_rule_params& p = a.p;
    if (parts) {
        delta_parts_kernel<KD><<<dim3((unsigned)parts_of(p), (unsigned)((p.n_k_head + 3) / 4)), 256, 0, s>>>(a, (int)parts_of(p));
        // (heads first: the slices of one head share its rows in one XCD's L2 where there is a multiple of 8 heads)
        delta_scan_kernel<KD><<<dim3((unsigned)p.n_v_head, (unsigned)(p.v_dim / 16), (unsigned)p.n_seq), 256, 0, s>>>(a);
        return hipGetLastError();
    }
    constexpr int C = KD == 256 ? 2 : 4;
    const int64_t wide = (int64_t)p.n_seq * p.n_v_head * ((p.v_dim + 16 * C - 1) / (16 * C));
    if (wide >= 2 * cu_count())
        delta_rows_kernel<KD, C><<<dim3((unsigned)p.n_v_head, (unsigned)((p.v_dim + 16 * C - 1) / (16 * C)), (unsigned)p.n_seq), 256, 0, s>>>(a);
    else
        delta_rows_kernel<KD, 1><<<dim3((unsigned)p.n_v_head, (unsigned)(p.v_dim / 16), (unsigned)p.n_seq), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

size_t delta_ws_bytes(const ggq_delta_rule_params& p) {
    if (!p.row_off) return 0;
    const char* env = getenv("GGQ_DELTA_PARTS");
    if (env && *env ? atoi(env) == 0 : p.n_rows <= 24 * (int64_t)p.n_seq) return 0;
    return sizeof(float) * kRecord * (size_t)parts_of(p) * p.n_v_head;
}

hipError_t launch_delta(const ggq_delta_rule_params& p, void* ws, hipStream_t s) {
    DeltaArgs a{p, p.scale == 0.0f ? (float)(1.0 / sqrt((double)p.k_dim)) : p.scale, (float*)ws};
    if (p.k_dim == 64) return delta_launch<64>(a, ws != nullptr, s);
    if (p.k_dim == 128) return delta_launch<128>(a, ws != nullptr, s);
    return delta_launch<256>(a, ws != nullptr, s);
}

}  // namespace ggq
