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
// Single tokens are bound by their states' bytes: 48 of 32 heads of 128 x 128 34 us, 6 TB/s.
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
// Bound: the chain of a part's steps.  8191 rows of 32 heads of 128 x 128: parts 51 us (their rows' bytes 33), scan 343, a part 1650 cycles, of which its 29 products
// take 960 (the four products of a part's rows and the state 200 us in all); the rest is what cannot stand beside
// an fp32 product of the same wavefront: own arithmetic, the sums' way through LDS, the barrier.
#include <algorithm>
#include <climits>
#include <cstdlib>
#include <type_traits>

#include "ggq_device.h"
#include "ggq_steps.h"

namespace ggq {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

struct DeltaArgs {
    ggq_delta_rule_params p;
    float scale;
    float* parts;  // records of the parts
    // Sequences of up to `few` rows go row by row, the others in parts (-1: all in parts; INT_MAX: none).
    int few;
};

constexpr int kRows = 16;  // rows of a part
// A part's record of one value head, in floats: T diag(b) and A [16][16], then factors of its rows: of K S, of Q S,
// of U on its way into the state; the state's own.
constexpr int kT = 0, kA = 256, kKc = 512, kQc = 528, kKs = 544, kDec = 560, kRecord = 576;  // (kDec: 16 times)

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
    if (sq.n > a.few) return;
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
__global__ __launch_bounds__(256) void delta_parts_kernel(DeltaArgs a) {
    constexpr int NT = KD / 16;
    // M, then its inverse, of four heads; of their rows: step, sum of logarithms, factor of q
    __shared__ __attribute__((aligned(16))) float s_m[4][4][16][20], s_row[4][4][16][4];
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
    if (first < 0 || first >= sq.n || sq.n <= a.few || hk >= p.n_k_head || slot_of(p, seq) < 0) return;  // (no barrier from here on)
    const int n = (int)min((int64_t)kRows, sq.n - first);
    const int64_t row0 = sq.row + first, row = row0 + min(r, n - 1);
    const float *kp = p.k + row * p.ldk + (int64_t)hk * KD + 4 * g, *qp = p.q + row * p.ldq + (int64_t)hk * KD + 4 * g;
    float4 k[NT], q[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) k[t] = *(const float4*)(kp + 16 * t);
#pragma unroll
    for (int t = 0; t < NT; t++) q[t] = *(const float4*)(qp + 16 * t);
    // of the first four heads, a head a group of lanes
    const int G = p.n_v_head / p.n_k_head;
    float ld = 0.0f, b = 0.0f;
    auto gates = [&](int h0) {
        const int h = hk * G + min(h0 + g, G - 1);
        ld = r < n ? decay_of(p, row, h) : 0.0f;
        b = r < n ? step_of(p, row, h) : 0.0f;
    };
    gates(0);
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
    for (int h0 = 0; h0 < G; h0 += 4) {
        if (h0) gates(h0);
        // (NaN stays)
        ld = fminf(fmaxf(ld, -1000.0f), 1000.0f) + (ld - ld == 0.0f || ld == INFINITY || ld == -INFINITY ? 0.0f : ld);
        Log L;
        L.hi = __builtin_rintf(ld * 256.0f) * (1.0f / 256.0f);
        L.lo = ld - L.hi;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const float x = __shfl_up(L.hi, o, 16), y = __shfl_up(L.lo, o, 16);
            if (r >= o) { L.hi += x; L.lo += y; }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        *(float4*)s_row[wave][g][r] = make_float4(b * rk, L.hi, L.lo, rq);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // M and A of each head: rows 4 g + e of column r in this lane
        const int nh = min(4, G - h0);
        for (int x = 0; x < nh; x++) {
            float* rec = a.parts + ((int64_t)id * p.n_v_head + hk * G + h0 + x) * kRecord;
            const float4 cr = *(const float4*)s_row[wave][x][r];
            const Log lr{cr.y, cr.z};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = 4 * g + e;
                const float4 ci = *(const float4*)s_row[wave][x][i];
                const float d = i >= r ? exp_of(Log{ci.y, ci.z}, lr) * rk : 0.0f;
                s_m[wave][x][i][r] = i > r ? ci.x * d * kk[e] : 0.0f;
                rec[kA + 16 * i + r] = i >= r ? ci.w * d * qk[e] : 0.0f;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // column r of (1 + M)^-1 of head g, from the top
        const int mine = min(g, nh - 1);
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float v = i == r ? 1.0f : 0.0f;
#pragma unroll
            for (int m = 0; m < i; m += 4) {
                const float4 w = *(const float4*)&s_m[wave][mine][i][m];
                v = fmaf(-w.x, x[m], v);
                if (m + 1 < i) v = fmaf(-w.y, x[m + 1], v);
                if (m + 2 < i) v = fmaf(-w.z, x[m + 2], v);
                if (m + 3 < i) v = fmaf(-w.w, x[m + 3], v);
            }
            x[i] = v;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (g < nh) {
#pragma unroll
            for (int i = 0; i < 16; i++) s_m[wave][g][i][r] = x[i] * b;
            float* rec = a.parts + ((int64_t)id * p.n_v_head + hk * G + h0 + g) * kRecord;
            const float4 last = *(const float4*)s_row[wave][g][15];
            const Log end{last.y, last.z};
            const float c = expf(L.hi + L.lo);
            rec[kKc + r] = c * rk;
            rec[kQc + r] = c * rq;
            rec[kKs + r] = exp_of(end, L) * rk;
            rec[kDec + r] = expf(end.hi + end.lo);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int x = 0; x < nh; x++) {
            float* rec = a.parts + ((int64_t)id * p.n_v_head + hk * G + h0 + x) * kRecord;
            *(float4*)(rec + kT + 4 * lane) = *(const float4*)&s_m[wave][x][lane >> 2][4 * (lane & 3)];
        }
    }
}

// 64 lanes' 16 bytes at src + each lane's offset into LDS at lds + 16 lane.  The caller waits on the vector memory
// counter.  (m0 is reserved: the compiler sets it right before its own uses.)
__device__ __forceinline__ void dma16(const void* src, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(src) : "memory");
}

// A part in LDS: K, Q (16-byte runs of row i exclusive-ored with i, which keeps both ways of reading them off each
// other's banks), V's 16 columns, the record (and what lies behind it, so that all loads are alike).  `slots` parts are
// under way.
template <int KD> struct Ring {
    static constexpr int kq = kRows * KD * 4, v = 2 * kq, rec = v + 1024, bytes = rec + 3 * 1024;
    static constexpr int slots = KD == 64 ? 8 : KD == 128 ? 6 : 3;
    static constexpr int loads = KD / 32 + 1;  // of a wavefront, a part
};

// Wavefronts 0 to 3 have a quarter of k each; 4 to 7, which share their SIMDs, load the parts to come and write the
// results of those that are done, while the others wait for products.
template <int KD>
__global__ __launch_bounds__(512) void delta_scan_kernel(DeltaArgs a) {
    constexpr int NT = KD / 64;  // tiles of 16 numbers of k of a wavefront
    constexpr int RPR = KD / 4;  // 16-byte runs of a row
    typedef Ring<KD> R;
    static_assert(R::slots * R::bytes < 128 * 1024, "LDS that global_load_lds addresses");
    __shared__ __attribute__((aligned(1024))) uint8_t ring[R::slots * R::bytes];
    __shared__ __attribute__((aligned(16))) f32x4 s_ks[2][4][64], s_o[2][4][64];
    __shared__ int s_list[512], s_many[8];
    const ggq_delta_rule_params& p = a.p;
    const int h = blockIdx.x, v0 = blockIdx.y * 16;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, r = lane & 15;
    const int wave8 = __builtin_amdgcn_readfirstlane(tid >> 6), wave = wave8 & 3;
    const int hk = h / (p.n_v_head / p.n_k_head);
    auto load_and_write = [&](const Seq& sq, int parts) {
        auto after = [](int in) { return in + 1 == R::slots ? 0 : in + 1; };
        const int last_row = sq.n - 1;
        const float *kp = p.k + sq.row * p.ldk + (int64_t)hk * KD, *qp = p.q + sq.row * p.ldq + (int64_t)hk * KD;
        const float* vp = p.v + sq.row * p.ldv + (int64_t)h * p.v_dim + v0;
        float* op = p.out + sq.row * p.ldo + (int64_t)h * p.v_dim + v0;
        // (one of them loads V, the others the record)
        const float* rec0 = a.parts + (sq.part * p.n_v_head + h) * kRecord + (wave - 1) * 256;
        // loads of part i into slot `in` (behind the last part: that one again, so that their number stays).  A lane's offsets
        // from a part's first row: of whole parts, and of the last one, whose rows end with the sequence's
        constexpr int NL = KD / 64;
        const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)ring;
        uint32_t ko[2][NL], qo[2][NL], ro[2];
#pragma unroll
        for (int w = 0; w < 2; w++) {
            const int most = w ? last_row - (parts - 1) * kRows : kRows - 1;
#pragma unroll
            for (int j = 0; j < NL; j++) {
                const int x = (wave * NL + j) * 64 + lane, row = x / RPR, run = x % RPR ^ (row & 15);
                ko[w][j] = 4u * ((uint32_t)min(row, most) * (uint32_t)p.ldk + 4u * run);  // (strides of up to 2^24)
                qo[w][j] = 4u * ((uint32_t)min(row, most) * (uint32_t)p.ldq + 4u * run);
            }
            ro[w] = wave ? 16u * lane : 4u * ((uint32_t)min(lane >> 2, most) * (uint32_t)p.ldv + 4u * (lane & 3));
        }
        const int64_t rest_step = wave ? (int64_t)p.n_v_head * kRecord : (int64_t)kRows * p.ldv;
        const float* rest0 = wave ? rec0 : vp;
        auto fetch = [&](int i, int in) {
            const uint32_t to = lds_at + (uint32_t)in * R::bytes;
            const int pt = min(i, parts - 1);
            const bool end = pt == parts - 1;
            const float *kb = kp + (int64_t)pt * kRows * p.ldk, *qb = qp + (int64_t)pt * kRows * p.ldq;
#pragma unroll
            for (int j = 0; j < NL; j++) {
                dma16(kb, end ? ko[1][j] : ko[0][j], to + (uint32_t)(wave * NL + j) * 1024u);
                dma16(qb, end ? qo[1][j] : qo[0][j], to + R::kq + (uint32_t)(wave * NL + j) * 1024u);
            }
            dma16(rest0 + (int64_t)pt * rest_step, end ? ro[1] : ro[0], to + R::v + (uint32_t)wave * 1024u);
        };
        auto put = [&](int i) {  // the wavefronts' parts of O, 4 rows a wavefront
            const int row = i * kRows + 4 * wave + g;
            const float* o = (const float*)s_o[i & 1] + (wave * 16 + r) * 4 + g;
            const float v = (o[0] + o[256]) + (o[512] + o[768]);
            if (row <= last_row) op[row * p.ldo + r] = v;
        };
        // (the counter also counts this wavefront's stores: a smaller number outstanding than loads only waits longer)
        for (int i = 0; i < R::slots - 1; i++) fetch(i, i);
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((R::slots - 2) * R::loads) : "memory");
        int before = R::slots - 1;
        for (int i = 0; i < parts; i++) {
            fetch(i + R::slots - 1, before);  // over the part before i, which nobody reads any more
            before = after(before);
            if (i > 1) put(i - 2);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((R::slots - 2) * R::loads) : "memory");
        }
        // (no load may come into LDS that is another workgroup's by then)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (parts > 1) put(parts - 2);
        put(parts - 1);
    };

    const int tile0 = wave * NT;
    f32x4 s[NT];
    // Where this lane reads in a slot: a row's 16-byte runs, K's numbers transposed, the record, V
    const uint8_t *row_at[NT], *col_at[NT][4], *rec_r = ring + R::rec + 64 * r + 16 * g, *rec_g = ring + R::rec + 16 * g;
    const uint8_t *a_at = ring + R::rec + 4 * (kA + 16 * r + 4 * g + wave), *v_at = ring + R::v + 4 * (64 * g + r);
#pragma unroll
    for (int t = 0; t < NT; t++) {
        row_at[t] = ring + (r * RPR + ((4 * (tile0 + t) + g) ^ r)) * 16;
#pragma unroll
        for (int e = 0; e < 4; e++) col_at[t][e] = ring + (((4 * g + e) * RPR + ((4 * (tile0 + t) + (r >> 2)) ^ (4 * g + e))) * 4 + (r & 3)) * 4;
    }
    f32x4 k[NT], q[NT];
    // A number of T or the rest that is not finite makes a whole column of u so (a zero times it is NaN), and with it the results of the rows
    // before it.  Their results again: row i is bad if T or the rest has such a number at i or, in its triangle, before; a bad row's u is
    // taken as 0 and its result as NaN.  (The column's state is not finite any more, as it is row by row.)
    auto results_again = [&](const f32x4& tr, const f32x4& rest, float ar, f32x4 of) {
        f32x4 x{}, bad{};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool in = 4 * g + e <= r, t_is = __builtin_isfinite(tr[e]), r_is = __builtin_isfinite(rest[e]);
            x = __builtin_amdgcn_mfma_f32_16x16x4f32(in && t_is ? tr[e] : 0.0f, r_is ? rest[e] : 0.0f, x, 0, 0, 0);
            bad = __builtin_amdgcn_mfma_f32_16x16x4f32(in ? 1.0f : 0.0f, r_is ? 0.0f : 1.0f, bad, 0, 0, 0);
            bad = __builtin_amdgcn_mfma_f32_16x16x4f32(in && !t_is ? 1.0f : 0.0f, 1.0f, bad, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool is = bad[e] > 0.0f || !__builtin_isfinite(x[e]);
            x[e] = is ? 0.0f : x[e];
            of[e] = is ? __builtin_nanf("") : of[e];
        }
        return __builtin_amdgcn_mfma_f32_16x16x4f32(ar, wave & 2 ? (wave & 1 ? x[3] : x[2]) : wave & 1 ? x[1] : x[0], of, 0, 0, 0);
    };
    // One part.  Issue is in order, and an fp32 product keeps its own wavefront's other arithmetic out (an instruction
    // behind a product costs the product's end and 4 cycles each): so products stand in rows, arithmetic in a few groups, and
    // what waits (this part's other operands, the sums' way through LDS) in the shadow of products.  The slots of the ring
    // are unrolled: their addresses are constants.
    auto step = [&](auto turn) {
        constexpr int in = decltype(turn)::value % R::slots, odd = decltype(turn)::value & 1;
        constexpr int here = in * R::bytes, next = (in + 1) % R::slots * R::bytes;
        f32x4 ks[2] = {}, qs[2] = {}, v, kt[NT];
        auto q_s = [&](int first, int last) {
#pragma unroll
            for (int x = first; x < last; x++)
                qs[x & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(q[x % NT][x / NT], s[x % NT][x / NT], qs[x & 1], 0, 0, 0);
        };
#pragma unroll
        for (int x = 0; x < 4 * NT; x++)
            ks[x & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[x % NT][x / NT], s[x % NT][x / NT], ks[x & 1], 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = *(const float*)(v_at + here + 64 * e);
        const f32x4 kc = *(const f32x4*)(rec_g + here + 4 * kKc), tr = *(const f32x4*)(rec_r + here + 4 * kT);
        const f32x4 kf = *(const f32x4*)(rec_g + here + 4 * kKs), qc = *(const f32x4*)(rec_g + here + 4 * kQc);
        const float dec = *(const float*)(ring + R::rec + here + 4 * kDec), ar = *(const float*)(a_at + here);
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int t = 0; t < NT; t++) kt[t][e] = *(const float*)(col_at[t][e] + here);
        __builtin_amdgcn_sched_barrier(0);
        q_s(0, NT);
        __builtin_amdgcn_sched_barrier(0);
        const f32x4 x0 = ks[0] + ks[1];
        s_ks[odd][wave][lane] = x0;
        __builtin_amdgcn_sched_barrier(0);
        q_s(NT, 2 * NT);
        __builtin_amdgcn_sched_barrier(0);
        // the next part's loads have come and the sums are in LDS
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        // (pairs, so that all wavefronts have the same sums)
        const f32x4 x1 = s_ks[odd][wave ^ 1][lane], x2 = s_ks[odd][wave ^ 2][lane], x3 = s_ks[odd][wave ^ 3][lane];
        __builtin_amdgcn_sched_barrier(0);
        q_s(2 * NT, 4 * NT);
        __builtin_amdgcn_sched_barrier(0);
        f32x4 rest, of_q = (qs[0] + qs[1]) * qc, u{0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; e++) rest[e] = fmaf(-kc[e], (x0[e] + x1[e]) + (x2[e] + x3[e]), v[e]);
#pragma unroll
        for (int t = 0; t < NT; t++) s[t] *= dec;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < 4; e++) u = __builtin_amdgcn_mfma_f32_16x16x4f32(tr[e], rest[e], u, 0, 0, 0);
#pragma unroll
        for (int t = 0; t < NT; t++) {  // (behind the last part: that one again)
            k[t] = *(const f32x4*)(row_at[t] + next);
            q[t] = *(const f32x4*)(row_at[t] + next + R::kq);
        }
        const f32x4 w = u * kf;
        const float ue = wave & 2 ? (wave & 1 ? u[3] : u[2]) : wave & 1 ? u[1] : u[0];
        __builtin_amdgcn_sched_barrier(0);
        f32x4 of = __builtin_amdgcn_mfma_f32_16x16x4f32(ar, ue, of_q, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int t = 0; t < NT; t++) s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kt[t][e], w[e], s[t], 0, 0, 0);
        if (__any(!__builtin_isfinite(u[0]))) of = results_again(tr, rest, ar, of_q);
        s_o[odd][wave][lane] = of;
        __builtin_amdgcn_sched_barrier(0);
    };
    auto compute = [&](int slot, int parts) {
        const int64_t at = (((int64_t)slot * p.n_v_head + h) * p.v_dim + v0 + r) * KD + 16 * tile0 + 4 * g;
#pragma unroll
        for (int t = 0; t < NT; t++) s[t] = *(const f32x4*)(p.state + at + 16 * t);
        if (parts) {
            __syncthreads();
#pragma unroll
            for (int t = 0; t < NT; t++) {
                k[t] = *(const f32x4*)row_at[t];
                q[t] = *(const f32x4*)(row_at[t] + R::kq);
            }
            int left = parts;
            // (as many steps as bring the slots and the two of s_ks back to the first)
            auto steps = [&](auto self, auto turn) -> void {
                step(turn);
                left--;
                if constexpr (decltype(turn)::value + 1 < R::slots * (1 + R::slots % 2))
                    if (left) self(self, std::integral_constant<int, decltype(turn)::value + 1>());
            };
            while (left) steps(steps, std::integral_constant<int, 0>());
            __syncthreads();
        }
#pragma unroll
        for (int t = 0; t < NT; t++) *(f32x4*)(p.state_out + at + 16 * t) = s[t];
    };
    auto sequence = [&](int seq) {  // (of all threads)
        const int slot = slot_of(p, seq);
        const Seq sq = seq_of(p, seq);
        const int parts = (sq.n + kRows - 1) / kRows;
        if (slot < 0) return;
        if (wave8 < 4) compute(slot, parts);
        else if (parts) load_and_write(sq, parts);
    };
    if (a.few < 0) return sequence(blockIdx.z);
    // Each gridDim.z-th one of the longer sequences.
    int before = 0;
    for (int from = 0; from < p.n_seq; from += 512) {
        const int j = from + tid;
        const bool is = j < p.n_seq && seq_of(p, j).n > a.few;
        const u64 b = __ballot(is);
        if (lane == 0) s_many[wave8] = __popcll(b);
        __syncthreads();
        int at = 0, many = 0;
#pragma unroll
        for (int w = 0; w < 8; w++) {
            at += w < wave8 ? s_many[w] : 0;
            many += s_many[w];
        }
        if (is) s_list[at + __popcll(b & ((1ull << lane) - 1))] = j;
        __syncthreads();
        for (int i = 0; i < many; i++)
            if ((before + i) % (int)gridDim.z == (int)blockIdx.z) sequence(__builtin_amdgcn_readfirstlane(s_list[i]));
        before += many;
        __syncthreads();
    }
}

int64_t parts_of(const ggq_delta_rule_params& p) { return (int64_t)p.n_rows / kRows + p.n_seq; }

// How many rows a sequence that goes row by row has at most (DeltaArgs::few).  A row's step takes 0.9 us where the chip
// is not full, and 10 us are gone before the first part is through: one sequence of 32 heads of 128 x 128 with 8 rows takes 11.2 us
// row by row and 11.5 in parts, with 16 rows 19.1 and 12.2.  Many sequences fill the chip better row by row (16 of 16 rows 50 and
// 61 us, of 24 rows 69 and 70; 64 of 16 rows 174 and 224, of 32 rows 337 and 287).  The lengths are on the device: unless all are
// bound to be short or are long in the mean, both forms are launched and each takes its own sequences.  That costs 5 to 8 us
// where all are short (64 of 4 rows 73 us, row by row 64) and bounds what one long one costs (64 single tokens and 1024
// rows: 112 us, row by row 1840, in parts 305).
int few_rows(const ggq_delta_rule_params& p) {
    if (!p.row_off) return INT_MAX;
    const char* env = getenv("GGQ_DELTA_PARTS");
    const bool many = (int64_t)p.n_seq * p.n_v_head * (p.v_dim / 16) > 1024;
    const int few = many ? kRows : kRows / 2;
    if (env && *env) return atoi(env) == 0 ? INT_MAX : atoi(env) == 1 ? -1 : few;
    if (p.n_rows - p.n_seq < (p.n_seq == 1 ? few : kRows)) return INT_MAX;  // (none is longer, unless others have no rows: not known here)
    return p.n_rows > (many ? 64 : few) * (int64_t)p.n_seq ? -1 : few;
}

template <int KD> hipError_t delta_launch(const DeltaArgs& a, hipStream_t s) {
    const ggq_delta_rule_params& p = a.p;
    if (a.few >= 0) {
        constexpr int C = KD == 256 ? 2 : 4;
        const int64_t wide = (int64_t)p.n_seq * p.n_v_head * ((p.v_dim + 16 * C - 1) / (16 * C));
        if (wide >= 2 * cu_count())
            delta_rows_kernel<KD, C><<<dim3((unsigned)p.n_v_head, (unsigned)((p.v_dim + 16 * C - 1) / (16 * C)), (unsigned)p.n_seq), 256, 0, s>>>(a);
        else
            delta_rows_kernel<KD, 1><<<dim3((unsigned)p.n_v_head, (unsigned)(p.v_dim / 16), (unsigned)p.n_seq), 256, 0, s>>>(a);
    }
    if (a.few < INT_MAX) {
        delta_parts_kernel<KD><<<dim3((unsigned)parts_of(p), (unsigned)((p.n_k_head + 3) / 4)), 256, 0, s>>>(a);
        // (no more workgroups than sequences can be long, nor than two a CU: one that finds nothing to do takes its LDS first)
        int64_t z = p.n_seq;
        if (a.few >= 0)
            z = std::max<int64_t>(1, std::min({z, (int64_t)p.n_rows / (a.few + 1), 2 * (int64_t)cu_count() / (p.n_v_head * (p.v_dim / 16))}));
        // (heads first: the slices of one head share its rows in one XCD's L2 where there is a multiple of 8 heads)
        delta_scan_kernel<KD><<<dim3((unsigned)p.n_v_head, (unsigned)(p.v_dim / 16), (unsigned)z), 512, 0, s>>>(a);
    }
    return hipGetLastError();
}

}  // namespace

size_t delta_ws_bytes(const ggq_delta_rule_params& p) {
    if (few_rows(p) == INT_MAX) return 0;
    return sizeof(float) * (kRecord * (size_t)parts_of(p) * p.n_v_head + 256);  // (the last record's loads go 192 floats further)
}

hipError_t launch_delta(const ggq_delta_rule_params& p, void* ws, hipStream_t s) {
    DeltaArgs a{p, p.scale == 0.0f ? (float)(1.0 / sqrt((double)p.k_dim)) : p.scale, (float*)ws, ws ? few_rows(p) : INT_MAX};
    if (p.k_dim == 64) return delta_launch<64>(a, s);
    if (p.k_dim == 128) return delta_launch<128>(a, s);
    return delta_launch<256>(a, s);
}

}  // namespace ggq
