// ggq_kv_chunk.hip -- causal attention of several rows of each sequence over the
// pages of its quantized cache (ggq_attention_kv_rows_dev).
//
// As the attention of single tokens (ggq_kv_cache.hip) a wavefront computes per
// record of 32 positions, on bf16 matrix cores with exact operands,
//   S^T[position][column] = sum_d K[position][d] Q[d][column]
//   O^T[d][column]       += sum_position V[position][d] P[position][column]
// but a column is a (row, head) pair here: the rows of a sequence and the heads that
// share a kv head are numbered through, 16 a tile, and the three bf16 parts
// of q and of the weights are three products instead of three columns.  A weight is made
// once, and no column is empty where the pairs fill the tiles.
//   A workgroup has 16 CT columns; its wavefronts take the records of its part of the
// positions in turn and add up in LDS, kv_chunk_join_kernel adds up the parts.
// Two tiles where a sequence's pairs fill more than one: a record is decoded once for 32
// columns.  Calls of many rows go through planes of operands (kv_chunk_plan).
// Bound: few pairs a kv head, loads in flight (24 sequences of 4 rows over 6000 positions, 32 x 8 heads
// of 128 in 8 / 4 bits, 43 + 5 us, 4.0 TB/s); more, decoding each record a tile again (64 rows over 65000 positions 214 us in
// eight tiles).
#include <algorithm>
#include <cstdlib>

#include "ggq_attn.h"
#include "ggq_attn_device.h"
#include "ggq_launch.h"
#include "ggq_steps.h"

namespace ggq {
namespace {

// Column tiles of n of a sequence's rows off0 .. off1 - 1.
__device__ __forceinline__ int tiles_in(int off0, int off1, int n_rows, int G, int n) {
    const int rows = min(max(off1, 0), n_rows) - min(max(off0, 0), n_rows);
    return (int)(((uint32_t)max(rows, 0) * (uint32_t)G + (uint32_t)n - 1) / (uint32_t)n);
}

// Three bf16 parts of x hold all its 24 bits: x cut, what is left cut, what is left then.
__device__ __forceinline__ float cut16(float x) {
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xFFFF0000u);
}
__device__ __forceinline__ void parts_of(float a, float b, uint32_t (&w)[3]) {
    w[0] = bf16_pack(a, b);
    a -= cut16(a);
    b -= cut16(b);
    w[1] = bf16_pack(a, b);
    a -= cut16(a);
    b -= cut16(b);
    w[2] = bf16_pack(a, b);
}

template <int HD, int CT> constexpr int chunk_waves() { return 4; }
// Wavefronts of a SIMD, by their registers.  (Two records of 128-wide heads in 8 / 8 bits do not fit beside the rest four times: 9 registers
// spilled, 24 sequences of 4 rows over 6000 positions 86 us and 64 single rows over 4000 134; 74 and 100 with three wavefronts.)
template <int HD, int CT, int BITS> constexpr int chunk_side() { return HD * CT > 128 ? 2 : HD == 128 && BITS == 16 ? 3 : 4; }

template <int HD, int KB, int VB, int CT>
__global__ __launch_bounds__((chunk_waves<HD, CT>() * 64), (chunk_side<HD, CT, KB + VB>())) void kv_chunk_kernel(KvChunkArgs a, int splits, float* part) {
    constexpr int NW = chunk_waves<HD, CT>(), NC = 16 * CT;
    constexpr int KW = HD * KB / 64, VW = HD * VB / 64;  // dwords of a lane's K and V codes
    constexpr int NS = HD / 32;                          // k steps of S^T, blocks of a head
    constexpr int NO = HD / 16;                          // row tiles of O^T
    constexpr int VD = HD / 16;                          // values of a lane's V at one position
    constexpr int64_t RB = kKvTile * HD * (KB + VB) / 8 + 2 * HD;
    __shared__ float sm[NW][NC], sl[NW][NC];
    // the parts of q, and in the end the wavefronts' sums
    constexpr int SQ = CT * NS * 3 * 64 * 16, SO = NW * NC * (HD + 1) * 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[SQ > SO ? SQ : SO];
    auto sq = (bf16x8(*)[NS][3][64])lds;
    auto so = (float(*)[NC][HD + 1])lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, r = lane & 15;
    const int kvh = blockIdx.x % a.c.n_kv_head;
    const unsigned turn = blockIdx.x / (unsigned)a.c.n_kv_head;
    const int G = a.n_head / a.c.n_kv_head;  // query heads of this kv head
    const int tpp = a.c.page_len / kKvTile;
    // The tile's sequence: tiles are numbered through, once for each part, by a running sum over the offsets.  (Numbers behind the
    // last tile are the last workgroups: workgroups go round the shader engines by their numbers, and ones without work in between
    // leave some of the engines with a second round; 64 rows over 65000 positions took 296 us so, 214 now.)
    __shared__ int32_t s_sum[NW], s_find[5];
    int off0, off1, len_j, mine, run;
    auto scan = [&](int j) {  // tiles up to sequence j of this turn's threads; returns their sum
        off0 = off1 = len_j = 0;
        if (j < a.q.n_seq) {
            off0 = a.row_off ? a.row_off[j] : j;
            off1 = a.row_off ? a.row_off[j + 1] : j + 1;
            len_j = a.q.len[j];
        }
        mine = run = tiles_in(off0, off1, a.n_rows, G, NC);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int t = __shfl_up(run, o, 64);
            if (lane >= o) run += t;
        }
        __syncthreads();
        if (lane == 63) s_sum[wave] = run;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            if (w < wave) run += s_sum[w];
            all += s_sum[w];
        }
        return __builtin_amdgcn_readfirstlane(all);
    };
    int total = 0, seq = 0, split, id, r0, nr;
    int64_t len;
    if (a.q.n_seq == 1) {
        r0 = a.row_off ? min(max(a.row_off[0], 0), a.n_rows) : 0;
        nr = (a.row_off ? min(max(a.row_off[1], 0), a.n_rows) : min(1, a.n_rows)) - r0;
        len = a.q.len[0];
        total = tiles_in(r0, r0 + nr, a.n_rows, G, NC);
        if (turn >= (unsigned)total * (unsigned)splits) return;
        split = (int)(turn / (unsigned)total);
        id = (int)(turn % (unsigned)total);
    } else {
        for (int i = 0; i < a.q.n_seq; i += NW * 64) total += scan(i + tid);
        if (turn >= (unsigned)total * (unsigned)splits) return;
        split = (int)(turn / (unsigned)total);
        id = (int)(turn % (unsigned)total);
        for (int i = 0, before = 0; before <= id; i += NW * 64) {
            const int all = a.q.n_seq > NW * 64 ? scan(i + tid) : total;
            const int at = id - (before + run - mine);
            if (at >= 0 && at < mine) {
                s_find[0] = i + tid;
                s_find[1] = at;
                s_find[2] = min(max(off0, 0), a.n_rows);
                s_find[3] = min(max(off1, 0), a.n_rows);
                s_find[4] = len_j;
            }
            before += all;
        }
        __syncthreads();
        seq = __builtin_amdgcn_readfirstlane(s_find[0]);
        id = __builtin_amdgcn_readfirstlane(s_find[1]);
        r0 = __builtin_amdgcn_readfirstlane(s_find[2]);
        nr = __builtin_amdgcn_readfirstlane(s_find[3]) - r0;
        len = __builtin_amdgcn_readfirstlane(s_find[4]);
    }
    const int nf = nr * G, f0 = id * NC;
    const int64_t lim = min(min(len, (int64_t)a.q.max_len), (int64_t)a.q.table_len * a.c.page_len);
    // columns: pair f has row f / G at position len - nr + f / G; it sees positions beg .. end - 1
    auto end_of = [&](int f) { return len - nr + f / G + 1; };
    auto see = [&](int f, int& b, int& e) {
        const int64_t x = end_of(f);
        e = (int)max(min(x, lim), (int64_t)0);
        b = a.window > 0 ? (int)max(x - a.window, (int64_t)0) : 0;
    };
    int beg[CT], end[CT];
#pragma unroll
    for (int n = 0; n < CT; n++) {
        const int f = f0 + 16 * n + r;
        see(min(f, nf - 1), beg[n], end[n]);
    }
    // rows ascend with the columns: the first and the last bound what any and what all of them see
    int lo, all_hi, all_lo, hi;
    see(f0, lo, all_hi);
    see(min(f0 + NC, nf) - 1, all_lo, hi);
    const int t0 = lo / kKvTile, t1 = hi > lo ? (hi + kKvTile - 1) / kKvTile : t0;
    int per = (t1 - t0 + splits - 1) / splits;
    if (per > NW) per = (per + NW - 1) / NW * NW;
    const int first = t0 + split * per, last = min(t1, first + per);

    f32x4 o[CT][NO];
    float m[CT], l[CT];
#pragma unroll
    for (int n = 0; n < CT; n++) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < NO; i++) o[n][i] = f32x4{0, 0, 0, 0};
    }

    struct Rec {
        uint32_t k[KW], v[VW], ks[NS / 2 + (NS < 2)];
        uint2 vs;
        bool there;
    };
    const int n_it = last > first + wave ? (last - first - wave + NW - 1) / NW : 0;  // records of this wavefront
    int pages = -1;  // lane i: page of record i of the current 64
    auto look = [&](int it) {
        const int t = first + wave + NW * (it + lane);
        pages = it + lane < n_it ? a.q.pages[(int64_t)seq * a.q.table_len + t / tpp] : -1;
        if (pages >= a.c.n_pages) pages = -1;
    };
    // A record's address is the wavefront's, a lane's offset an unsigned 32-bit one: loads take both as they are.  (The empty asm
    // statements keep the offsets from being widened once for all: as 64-bit numbers they leave the 128-wide instances short of registers,
    // and a spilled one is read back behind the loads in flight, which it then waits for: 24 sequences of 4 rows over 6000 positions
    // in 8 / 4 bits 64 us so, 61 now.)
    auto load = [&](int it, Rec& x) {
        uint32_t run_at = 16u * lane, vs_at = 8u * (4u * (r * VD / 32) + g), ks_at = 2u * (16u * (g * NS / 4) + r);
        asm volatile("" : "+v"(run_at), "+v"(vs_at), "+v"(ks_at));
        const int page = __builtin_amdgcn_readlane(pages, it & 63);
        x.there = page >= 0;
        if (!x.there) return;
        const int t = first + wave + NW * it;
        const uint8_t* rec = (const uint8_t*)a.c.pages + (((int64_t)page * a.c.n_kv_head + kvh) * tpp + t % tpp) * RB;
#pragma unroll
        for (int i = 0; i < KW; i += 4) {
            const uint4 v = *(const uint4*)(rec + 256 * i + run_at);
            x.k[i] = v.x; x.k[i + 1] = v.y; x.k[i + 2] = v.z; x.k[i + 3] = v.w;
        }
        rec += kKvTile * HD * KB / 8;
        asm volatile("" : "+s"(rec));
#pragma unroll
        for (int i = 0; i < VW; i += 4) {
            const uint4 v = *(const uint4*)(rec + 256 * i + run_at);
            x.v[i] = v.x; x.v[i + 1] = v.y; x.v[i + 2] = v.z; x.v[i + 3] = v.w;
        }
        rec += kKvTile * HD * VB / 8;
        asm volatile("" : "+s"(rec));
        // K scales: a lane's quarter of the head lies in block g * NS / 4 (and the next one of 256-wide heads)
        x.ks[0] = *(const uint16_t*)(rec + ks_at);
        if constexpr (NS > 4) x.ks[1] = *(const uint16_t*)(rec + 32 + ks_at);
        x.vs = *(const uint2*)(rec + HD + vs_at);
    };
    // Positions of this lane (a bit each) with values that read back as infinite or NaN: read anew, few caches hold any.
    auto not_finite = [&](int it) {
        const int t = first + wave + NW * it;
        const uint8_t* rec = (const uint8_t*)a.c.pages +
                             (((int64_t)a.q.pages[(int64_t)seq * a.q.table_len + t / tpp] * a.c.n_kv_head + kvh) * tpp + t % tpp) * RB + kKvTile * HD * KB / 8;
        uint32_t run_at = 16u * lane, vs_at = 8u * (4u * (r * VD / 32) + g);
        asm volatile("" : "+v"(run_at), "+v"(vs_at));
        const uint8_t *run = rec + run_at, *scales = rec + kKvTile * HD * VB / 8 + HD + vs_at;
        uint32_t odd = 0;
#pragma nounroll
        for (int i = 0; i < 8 * VD; i++) {  // (in the order of the lane's codes)
            const int b = i * VB / 8;
            const uint32_t code = run[1024 * (b / 16) + b % 16] >> (i * VB % 8) & (VB == 8 ? 127u : 7u);
            odd |= (code >= first_not_finite<VB>(scales[i / VD]) ? 1u : 0u) << (i / VD);
        }
        return odd;
    };
    auto compute = [&](int it, Rec& x) {
        if (!x.there) return;
        const int base = (first + wave + NW * it) * kKvTile;
        const bool partial = base < all_lo || base + kKvTile > all_hi;
        f32x4 st[2][CT];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int n = 0; n < CT; n++) st[t][n] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NS; s++) {
            Frag f[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int blk = NS <= 4 ? 0 : s / 4;  // (256-wide: 64 values of a lane, two blocks)
                const float sc = scale_of((x.ks[blk] >> (8 * t)) & 255u);
#pragma unroll
                for (int i = 0; i < 4; i++) f[t].w[i] = pair_of<KB>(x.k + (t * (HD / 4) + 8 * s) * KB / 32, sc, i);
            }
            // (the small parts first: they do not round at the size of the sum)
#pragma unroll
            for (int j = 2; j >= 0; j--)
#pragma unroll
                for (int n = 0; n < CT; n++) {
                    const bf16x8 q = sq[n][s][j][lane];
#pragma unroll
                    for (int t = 0; t < 2; t++) st[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[t].v, q, st[t][n], 0, 0, 0);
                }
        }
        uint32_t poison = 0;  // positions with values that read back as infinite or NaN, which some columns see and some do not
        if (partial) {
            // codes of positions that no column sees, or that have such values (a weight of 0 would make NaN of them): zero, with a
            // finite scale
            uint32_t keep[8], odd = 0;
            // (but for e4m3's NaN they are under scales of 2^113 and more only: a byte's upper four bits all set)
            const uint32_t sx = x.vs.x & x.vs.x << 1, sy = x.vs.y & x.vs.y << 1;
            if (__any((((sx & sx << 2) | (sy & sy << 2)) & 0x80808080u) != 0)) odd = not_finite(it);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int pos = base + 16 * (j / 4) + 4 * g + j % 4;
                keep[j] = pos >= lo && pos < hi ? 0xFFFFFFFFu : 0u;
                uint32_t bad = odd >> j & 1u;
                if constexpr (VB == 8) {
#pragma unroll
                    for (int d = 0; d < VD; d++)
                        bad |= (x.v[(j * VD + d) / 4] >> (8 * ((j * VD + d) % 4)) & 127u) == 127u;
                }
                if (bad && keep[j]) {
                    poison |= 1u << j;
                    keep[j] = 0;
                }
            }
            constexpr int BPP = VD * VB / 8;  // bytes of a position
#pragma unroll
            for (int d = 0; d < VW; d++) {
                if constexpr (BPP >= 4) x.v[d] &= keep[d * 4 / BPP];
                else x.v[d] &= (keep[2 * d] & 0xFFFFu) | (keep[2 * d + 1] & 0xFFFF0000u);
            }
            uint32_t lo4 = 0, hi4 = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                lo4 |= (keep[j] ? (x.vs.x >> (8 * j)) & 255u : 127u) << (8 * j);
                hi4 |= (keep[j + 4] ? (x.vs.y >> (8 * j)) & 255u : 127u) << (8 * j);
            }
            x.vs = make_uint2(lo4, hi4);
            if (__any(poison != 0)) {
#pragma unroll
                for (int s = 1; s < 16; s <<= 1) poison |= (uint32_t)__shfl_xor((int)poison, s, 64);
            }
        }
        bool move = false;
        float top[CT];
#pragma unroll
        for (int n = 0; n < CT; n++) {
            if (partial) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int pos = base + 16 * (j / 4) + 4 * g + j % 4;
                    const bool sees = pos >= beg[n] && pos < end[n];
                    if (!sees) st[j / 4][n][j % 4] = -INFINITY;
                    else if (poison >> j & 1u) l[n] = __builtin_nanf("");
                }
            }
            const f32x4 x0 = st[0][n], x1 = st[1][n];
            top[n] = rows_max(max3(max3(x0[0], x0[1], x0[2]), max3(x0[3], x1[0], x1[1]), max3(x1[2], x1[3], x1[3])));
            move |= top[n] > m[n] + 8.0f;
        }
        if (__any(move)) {
#pragma unroll
            for (int n = 0; n < CT; n++) {
                const float mn = max3(m[n], top[n], top[n]);
                const float al = __builtin_amdgcn_exp2f(m[n] - (mn == -INFINITY ? 0.0f : mn));
                m[n] = mn;
                l[n] *= al;
#pragma unroll
                for (int i = 0; i < NO; i++) o[n][i] *= al;
            }
        }
        Frag pf[CT][3];
#pragma unroll
        for (int n = 0; n < CT; n++) {
            const float mm = m[n] == -INFINITY ? 0.0f : m[n];
            float e[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                e[j] = __builtin_amdgcn_exp2f(st[j / 4][n][j % 4] - mm);
                l[n] += e[j];
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t w[3];
                parts_of(e[2 * j], e[2 * j + 1], w);
#pragma unroll
                for (int i = 0; i < 3; i++) pf[n][i].w[j] = w[i];
            }
        }
        // weights times values, two row tiles (values 2 i, 2 i + 1 of a lane's run) at a time
        float vs[8];
#pragma unroll
        for (int j = 0; j < 8; j++) vs[j] = scale_of(((j < 4 ? x.vs.x : x.vs.y) >> (8 * (j & 3))) & 255u);
#pragma unroll
        for (int i = 0; i < NO / 2; i++) {
            uint32_t c[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int v = j * VD + 2 * i;  // index in the lane's run of codes, even
                if constexpr (VB == 4) c[j] = fp4_pair(x.v[v / 8], vs[j], v % 8 / 2);
                else c[j] = fp8_pair(x.v[v / 4], vs[j], v % 4 / 2);
            }
            Frag f[2];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                f[0].w[j] = __builtin_amdgcn_perm(c[2 * j + 1], c[2 * j], 0x05040100u);
                f[1].w[j] = __builtin_amdgcn_perm(c[2 * j + 1], c[2 * j], 0x07060302u);
            }
#pragma unroll
            for (int j = 2; j >= 0; j--)
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int n = 0; n < CT; n++)
                        o[n][2 * i + e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[e].v, pf[n][j].v, o[n][2 * i + e], 0, 0, 0);
        }
    };
    Rec cur, nxt;
    look(0);
    if (n_it > 0) load(0, cur);
    // the columns' parts in the order of the operands, for all wavefronts
    for (int x = tid; x < CT * NS * 64; x += NW * 64) {
        const int n = x / (NS * 64), s = x / 64 % NS, fq = min(f0 + 16 * n + (x & 15), nf - 1), qi = fq / G, h = fq - qi * G;
        const float* qp = a.Q + (int64_t)(r0 + qi) * a.ldq + (int64_t)(kvh * G + h) * HD + (x >> 4 & 3) * (HD / 4) + 8 * s;
        const float4 u = *(const float4*)qp, v = *(const float4*)(qp + 4);
        const float y[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
        Frag f[3];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t w[3];
            parts_of(y[2 * i] * a.scale, y[2 * i + 1] * a.scale, w);
#pragma unroll
            for (int j = 0; j < 3; j++) f[j].w[i] = w[j];
        }
#pragma unroll
        for (int j = 0; j < 3; j++) sq[n][s][j][x & 63] = f[j].v;
    }
    __syncthreads();
    for (int it = 0; it < n_it; it++) {
        if (it + 1 < n_it) {
            if (((it + 1) & 63) == 0) look(it + 1);
            load(it + 1, nxt);
        }
        compute(it, cur);
        cur = nxt;
    }

    // the wavefronts' parts
    __syncthreads();
#pragma unroll
    for (int n = 0; n < CT; n++) {
        float s = l[n];  // of this group's positions
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        const int c = 16 * n + r;
        if (g == 0) { sm[wave][c] = m[n]; sl[wave][c] = s; }
#pragma unroll
        for (int i = 0; i < NO; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) so[wave][c][(4 * g + e) * VD + i] = o[n][i][e];
    }
    __syncthreads();
    const int nc = min(NC, nf - f0);
    for (int e = tid; e < nc * HD; e += NW * 64) {
        const int c = e / HD, d = e % HD;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; w++) mx = fmaxf(mx, sm[w][c]);
        float ls = 0.0f, os = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float al = sm[w][c] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[w][c] - mx);
            ls = fmaf(sl[w][c], al, ls);
            os = fmaf(so[w][c][d], al, os);
        }
        const int qi = (f0 + c) / G, head = kvh * G + (f0 + c) - qi * G;
        if (splits == 1) {
            // no position at all: zeros (a NaN keeps its way through the sum)
            a.out[(int64_t)(r0 + qi) * a.ldo + (int64_t)head * HD + d] = ls == 0.0f && mx == -INFINITY ? 0.0f : os / ls;
        } else {
            float* po = part + (((int64_t)(r0 + qi) * a.n_head + head) * splits + split) * (HD + 2);
            po[d] = os;
            if (d == 0) { po[HD] = mx; po[HD + 1] = ls; }
        }
    }
}

// The parts of one row's head: their weights first, then a thread a value and group of parts, eight loads in
// flight, in an order that does not depend on timing.
constexpr int kMaxSplits = 256;
template <int HD> __global__ __launch_bounds__(256) void kv_chunk_join_kernel(KvChunkArgs a, int splits, const float* part) {
    constexpr int NG = 256 / HD, B = 8;
    __shared__ float w[kMaxSplits], red[8], go[NG][HD];
    const int row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, d = tid % HD, grp = tid / HD;
    const float* po = part + ((int64_t)row * a.n_head + head) * splits * (HD + 2);
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (tid < splits) ml = *(const float2*)(po + (int64_t)tid * (HD + 2) + HD);
    bool in = !a.row_off && row < a.q.n_seq;  // a row of some sequence
    if (a.row_off)
        for (int j = tid; j < a.q.n_seq; j += 256) in |= a.row_off[j] <= row && row < a.row_off[j + 1];
    if (!__syncthreads_or(in)) return;
    float mx = ml.x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float wt = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mx);
    if (tid < splits) w[tid] = wt;
    float ls = wt * ml.y;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ls += __shfl_xor(ls, o, 64);
    if ((tid & 63) == 0) red[4 + (tid >> 6)] = ls;
    __syncthreads();
    float os = 0.0f;
    for (int i = grp; i < splits; i += NG * B) {
        float v[B];
#pragma unroll
        for (int b = 0; b < B; b++) v[b] = i + b * NG < splits ? po[(int64_t)(i + b * NG) * (HD + 2) + d] : 0.0f;
#pragma unroll
        for (int b = 0; b < B; b++)
            if (i + b * NG < splits) os = fmaf(v[b], w[i + b * NG], os);
    }
    go[grp][d] = os;
    __syncthreads();
    if (grp) return;
    ls = (red[4] + red[5]) + (red[6] + red[7]);
#pragma unroll
    for (int i = 1; i < NG; i++) os += go[i][d];
    a.out[(int64_t)row * a.ldo + (int64_t)head * HD + d] = ls == 0.0f && mx == -INFINITY ? 0.0f : os / ls;
}

// Workgroups that the chip holds at once.
template <int HD, int KB, int VB, int CT> int64_t resident() {
    static const int64_t n = [] {
        int r = 0;
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&r, (const void*)kv_chunk_kernel<HD, KB, VB, CT>, chunk_waves<HD, CT>() * 64, 0) != hipSuccess || r < 1)
            r = 1;
        return (int64_t)r * cu_count();
    }();
    return n;
}

int64_t tiles_of(const KvChunkArgs& a, int nc) { return (int64_t)a.n_rows * (a.n_head / a.c.n_kv_head) / nc + a.q.n_seq; }

// One round of workgroups at most, four records in a part at least, where that saves more than the join costs.
// (Workgroups with work: those of sequences of the mean length.)
template <int HD, int KB, int VB, int CT> int splits_of(const KvChunkArgs& a, int64_t records) {
    constexpr int NW = chunk_waves<HD, CT>();
    const int64_t pairs = ((int64_t)a.n_rows + a.q.n_seq - 1) / a.q.n_seq * (a.n_head / a.c.n_kv_head);
    const int64_t wgs = std::max<int64_t>(1, (pairs + 16 * CT - 1) / (16 * CT)) * a.q.n_seq * a.c.n_kv_head;
    const int64_t n = std::min<int64_t>(resident<HD, KB, VB, CT>() / wgs, (records + 3) / 4);
    return n > 1 && records * (n - 1) > 3 * NW * n ? (int)std::min<int64_t>(n, kMaxSplits) : 1;
}

template <int HD, int KB, int VB> int splits_go(const KvChunkArgs& a, int ct, int64_t records) {
    if constexpr (HD < 256)
        if (ct == 2) return splits_of<HD, KB, VB, 2>(a, records);
    return splits_of<HD, KB, VB, 1>(a, records);
}

template <int HD, int KB, int VB> hipError_t chunk_go(const KvChunkArgs& a, const KvChunkPlan& pl, float* ws, hipStream_t s) {
    const dim3 grid((unsigned)(tiles_of(a, 16 * pl.tiles) * a.c.n_kv_head * pl.splits));
    bool done = false;
    if constexpr (HD < 256)
        if (pl.tiles == 2) {
            kv_chunk_kernel<HD, KB, VB, 2><<<grid, chunk_waves<HD, 2>() * 64, 0, s>>>(a, pl.splits, ws);
            done = true;
        }
    if (!done) kv_chunk_kernel<HD, KB, VB, 1><<<grid, chunk_waves<HD, 1>() * 64, 0, s>>>(a, pl.splits, ws);
    if (pl.splits > 1) kv_chunk_join_kernel<HD><<<dim3((unsigned)a.n_rows, (unsigned)a.n_head), 256, 0, s>>>(a, pl.splits, ws);
    return hipGetLastError();
}

}  // namespace

#define GGQ_BY_CACHE(HD_, F, ...)                                                                              \
    (c.k_type == GGQ_KV_MXFP4 ? (c.v_type == GGQ_KV_MXFP4 ? F<HD_, 4, 4>(__VA_ARGS__) : F<HD_, 4, 8>(__VA_ARGS__)) \
                              : (c.v_type == GGQ_KV_MXFP4 ? F<HD_, 8, 4>(__VA_ARGS__) : F<HD_, 8, 8>(__VA_ARGS__)))

KvChunkPlan kv_chunk_plan(const KvChunkArgs& a, bool workspace) {
    const ggq_kv_cache& c = a.c;
    KvChunkPlan pl{1, {}, 1, 0};
    // two tiles a wavefront where a sequence's pairs fill more than one
    const int64_t pairs = (int64_t)a.n_rows * (a.n_head / c.n_kv_head);
    if (c.head_dim < 256 && pairs > 16 * (int64_t)a.q.n_seq) pl.tiles = 2;
    if (!workspace) return pl;
    int64_t span = std::min<int64_t>(a.q.max_len, (int64_t)a.q.table_len * c.page_len);
    if (a.window > 0) span = std::min<int64_t>(span, (int64_t)a.window + a.n_rows / a.q.n_seq + kKvTile);
    const int64_t records = (span + kKvTile - 1) / kKvTile;
    // Planes of operands (codes decoded once, two fp16 products where this kernel has three) from so many pairs a sequence
    // on that they pay for the planes, in calls that are more than their launches (us, tiles -> planes; pairs: rows times heads of
    // a kv head; 8 / 8 bits):
    //   32x8x128: one of 7000 positions 512 pairs 60 -> 76, 768 93 -> 82, 2048 159 -> 142; of 65000, 384 329 -> 345, 512 369 -> 351,
    //     1024 715 -> 592; 16 of 4000, 384 281 -> 315, 512 366 -> 338, 1024 704 -> 592
    //   32x8x64: one of 7000, 2048 119 -> 124; of 65000, 1024 432 -> 487, 2048 833 -> 910
    //   16x2x256: one of 7000, 1024 57 -> 83, 4096 167 -> 162; of 65000, 512 198 -> 230, 1024 377 -> 365, 2048 736 -> 647
    const int64_t mean = ((int64_t)a.n_rows + a.q.n_seq - 1) / a.q.n_seq * (a.n_head / c.n_kv_head);
    const int64_t least = c.head_dim == 64 ? 8192 : c.head_dim == 128 ? 512 : 1024;
    const char* env = getenv("GGQ_KV_PLANES");
    if (a.row_off && (env && *env ? atoi(env) != 0 : mean >= least && mean * a.q.n_seq * c.n_kv_head * records >= 1000000)) {
        const AttnPromptPlan planes = attn_kv_planes_plan(a);
        if (planes.ws_bytes <= (size_t(1) << 30)) {
            pl.tiles = 0;
            pl.planes = planes;
            pl.ws_bytes = planes.ws_bytes;
            return pl;
        }
    }
    if (const char* e = getenv("GGQ_KV_SPLITS"); e && atoi(e) > 0)
        pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(atoi(e), kMaxSplits), records));
    else if (c.head_dim == 64) pl.splits = GGQ_BY_CACHE(64, splits_go, a, pl.tiles, records);
    else if (c.head_dim == 128) pl.splits = GGQ_BY_CACHE(128, splits_go, a, pl.tiles, records);
    else pl.splits = GGQ_BY_CACHE(256, splits_go, a, pl.tiles, records);
    if (pl.splits > 1) pl.ws_bytes = sizeof(float) * (size_t)a.n_rows * a.n_head * pl.splits * (c.head_dim + 2);
    return pl;
}

hipError_t launch_kv_chunk(const KvChunkArgs& a, const KvChunkPlan& pl, void* ws, hipStream_t s) {
    if (!pl.tiles) return launch_attn_kv_planes(a, pl.planes, ws, s);
    const ggq_kv_cache& c = a.c;
    if (c.head_dim == 64) return GGQ_BY_CACHE(64, chunk_go, a, pl, (float*)ws, s);
    if (c.head_dim == 128) return GGQ_BY_CACHE(128, chunk_go, a, pl, (float*)ws, s);
    return GGQ_BY_CACHE(256, chunk_go, a, pl, (float*)ws, s);
}
#undef GGQ_BY_CACHE

}  // namespace ggq
