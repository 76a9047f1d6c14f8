// ggq_attn_prompt.hip -- causal attention of packed prompts.
//
// The keys and values a call sees are first written as planes of fp16 operands
// (planes_kernel): 32 positions of one kv head a unit, fp32 values as hi + lo
// under a power of two of the unit (22 bits of the unit's largest), in the
// order in which the matrix cores take them, values transposed.  attn_kernel
// then computes per unit, with v_mfma_f32_32x32x16_f16,
//   S^T[position][column] = K Q^T,  O^T[value][column] += V^T P^T
// as the products hi hi + hi lo + lo hi of fp32 keys and values (two products
// with fp16 ones, which need no split), so results are as exact as fp32
// sums.  A column is one (query row, head) pair: the rows of a sequence and the
// heads that share a kv head are numbered through, 32 columns a wavefront,
// so any ratio of heads fills the tiles and all wavefronts of a workgroup share
// each unit in LDS.
//   S^T leaves a lane with 16 positions of its column, and P^T wants 8 positions a lane and
// step of the same column: the values' planes are ordered so that these are the
// same ones, and weights go from one product to the next in registers.
//   Units arrive in a ring of LDS slots straight from memory
// (global_load_lds), a barrier a unit.
//   The maximum moves only when a unit exceeds it by 2^4; weights are kept times
// 2^11 (at most 2^15), so hi + lo of a small weight keeps 2^-35 of the largest.
// The running sums are in units of the values' power of two and follow it.
// Bound: the matrix cores.
#include <algorithm>

#include "ggq_attn.h"
#include "ggq_attn_device.h"
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

// ------------------------------------------------------------ matrix cores
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kUnit = 32;  // positions
// Bytes of a unit: 64 dwords of header, K and V planes.
constexpr int64_t unit_bytes(int hd, int planes) { return (int64_t)planes * 2 * kUnit * hd * 2 + 256; }
// Header: exponents of K and V (+ 512), and whether there are values that are not
// finite, positions whose largest value is more than 2^16 below the unit's (what
// hi + lo keep of them is less than fp32), any values but zero.
enum { BAD_K = 1 << 20, BAD_V = 1 << 21, WIDE_K = 1 << 22, WIDE_V = 1 << 23, NO_V = 1 << 24 };

// Sequence s has the units from off[s] / 32 + s on (and as many column tiles of
// n from off[s] * G / n + s): a bound that needs no sum over the sequences before.
__device__ __forceinline__ int64_t bound_of(int64_t first, int64_t per, int s) { return first / per + s; }

struct PromptArgs {
    ggq_attention_prompt_params p;
    uint8_t* planes;
    float* part;
    int G, tiles, splits;
};

// A sequence's rows of an offset array, held inside [0, n].
struct Span {
    int64_t a, n;
};
__device__ __forceinline__ Span span_of(const int32_t* off, int s, int64_t most) {
    const int64_t a = min(max((int64_t)off[s], (int64_t)0), most), b = min(max((int64_t)off[s + 1], (int64_t)0), most);
    return Span{a, b > a ? b - a : 0};
}
__device__ __forceinline__ const int32_t* kv_off_of(const ggq_attention_prompt_params& p) { return p.kv_off ? p.kv_off : p.q_off; }

__device__ __forceinline__ uint32_t mag_bits(float v) {  // 0 for what is not finite
    const uint32_t u = __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu;
    return u >= 0x7F800000u ? 0u : u;
}
__device__ __forceinline__ bool finite(float v) { return (__builtin_bit_cast(uint32_t, v) & 0x7F800000u) != 0x7F800000u; }

// Exponent that brings a magnitude into [2^14, 2^15).
__device__ __forceinline__ int up_to_2_15(uint32_t bits) { return bits ? 141 - (int)(bits >> 23) : 0; }

template <int HD, typename T>
__global__ __launch_bounds__(256) void planes_kernel(PromptArgs a) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1, V = HD / 8;  // planes, values of a thread
    constexpr int PL = kUnit * HD;                         // values of a plane
    __shared__ float sv[kUnit][HD + 1];
    __shared__ uint32_t red[4][5];
    const int tid = threadIdx.x, kvh = blockIdx.y;
    const int32_t* off = kv_off_of(a.p);
    const int64_t id = blockIdx.x;
    int seq = 0;
    for (int i = 1; i < a.p.n_seq; i += 256) {
        const int j = i + tid;
        seq += __syncthreads_count(j < a.p.n_seq && bound_of(max(off[j], 0), kUnit, j) <= id);
    }
    const Span sp = span_of(off, seq, a.p.n_kv_rows);
    const int64_t u = id - bound_of(sp.a, kUnit, seq);
    if (u < 0 || u * kUnit >= sp.n) return;
    const int pos = tid / 8, d0 = tid % 8 * V;
    const bool in = u * kUnit + pos < sp.n;
    const int64_t row = sp.a + u * kUnit + pos;
    float k[V], v[V];
    uint32_t mk = 0, mv = 0, bad = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        k[i] = in ? (float)((const T*)a.p.k)[row * a.p.ldk + (int64_t)kvh * HD + d0 + i] : 0.0f;
        v[i] = in ? (float)((const T*)a.p.v)[row * a.p.ldv + (int64_t)kvh * HD + d0 + i] : 0.0f;
        mk = max(mk, mag_bits(k[i]));
        mv = max(mv, mag_bits(v[i]));
        if (!finite(k[i])) bad |= BAD_K;
        if (!finite(v[i])) {
            bad |= BAD_V;
            v[i] = 0.0f;
        }
    }
    // the unit's largest, and the least of its positions' largest (but zero): 8 threads a position first
    auto least = [](uint32_t x, uint32_t y) { return x && (!y || x < y) ? x : y; };
    uint32_t nk = 0, nv = 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        if (o == 8) {
            nk = mk;
            nv = mv;
        }
        mk = max(mk, (uint32_t)__shfl_xor((int)mk, o, 64));
        mv = max(mv, (uint32_t)__shfl_xor((int)mv, o, 64));
        bad |= (uint32_t)__shfl_xor((int)bad, o, 64);
        if (o >= 8) {
            nk = least(nk, (uint32_t)__shfl_xor((int)nk, o, 64));
            nv = least(nv, (uint32_t)__shfl_xor((int)nv, o, 64));
        }
    }
    if ((tid & 63) == 0) {
        uint32_t* r = red[tid >> 6];
        r[0] = mk; r[1] = mv; r[2] = bad; r[3] = nk; r[4] = nv;
    }
    __syncthreads();
    mk = max(max(red[0][0], red[1][0]), max(red[2][0], red[3][0]));
    mv = max(max(red[0][1], red[1][1]), max(red[2][1], red[3][1]));
    bad = red[0][2] | red[1][2] | red[2][2] | red[3][2];
    nk = least(least(red[0][3], red[1][3]), least(red[2][3], red[3][3]));
    nv = least(least(red[0][4], red[1][4]), least(red[2][4], red[3][4]));
    if (P == 2 && (mk >> 23) - (nk >> 23) > 16) bad |= WIDE_K;
    if (P == 2 && (mv >> 23) - (nv >> 23) > 16) bad |= WIDE_V;
    // fp16 values stay as they are
    const int ke = P == 2 ? up_to_2_15(mk) : 0, ve = P == 2 ? up_to_2_15(mv) : 0;
    uint8_t* out = a.planes + (id * a.p.n_kv_head + kvh) * unit_bytes(HD, P);
    if (tid < 64) ((uint32_t*)out)[tid] = (uint32_t)(ke + 512) | (uint32_t)(ve + 512) << 10 | bad | (mv ? 0 : NO_V);
    _Float16* kp = (_Float16*)(out + 256);
#pragma unroll
    for (int i = 0; i < V; i += 8) {
        h8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float x = P == 2 ? ldexpf(k[i + j], ke) : k[i + j];
            hi[j] = (_Float16)x;
            lo[j] = finite(x) ? (_Float16)(x - (float)hi[j]) : (_Float16)0.0f;
        }
        const int d = d0 + i;
        _Float16* at = kp + ((d / 16) * 64 + (d / 8 % 2) * 32 + pos) * 8;
        *(h8*)at = hi;
        if constexpr (P == 2) *(h8*)(at + PL) = lo;
    }
#pragma unroll
    for (int i = 0; i < V; i++) sv[pos][d0 + i] = P == 2 ? ldexpf(v[i], ve) : v[i];
    __syncthreads();
    _Float16* vp = kp + P * PL;
    for (int e = tid; e < HD * 4; e += 256) {  // (value, step of 16 positions, half)
        const int d = e % HD, st = e / HD / 2, h = e / HD % 2;
        h8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float x = sv[16 * st + 8 * (j / 4) + 4 * h + j % 4][d];
            hi[j] = (_Float16)x;
            lo[j] = (_Float16)(x - (float)hi[j]);
        }
        _Float16* at = vp + (((d / 32) * 2 + st) * 64 + h * 32 + d % 32) * 8;
        *(h8*)at = hi;
        if constexpr (P == 2) *(h8*)(at + PL) = lo;
    }
}

// 64 lanes' 16 (or 4) bytes at src + lane's offset into LDS at lds + 16 (4) lane.  The
// caller waits on the vector memory counter.  (m0 is reserved: the compiler
// sets it right before its own uses.)
__device__ __forceinline__ void dma16(const uint8_t* src, uint32_t lane16, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(lane16), "s"(src) : "memory");
}
__device__ __forceinline__ void dma4(const uint8_t* src, uint32_t lane4, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(lane4), "s"(src) : "memory");
}


// The weight of position `at` of a unit in this lane's column.
__device__ __forceinline__ float weight_of(const float (&e)[16], int at, int col) {
    float w = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (8 * (i / 4) + i % 4 == (at & ~4)) w = e[i];
    return __shfl(w, col + 32 * ((at >> 2) & 1), 64);
}

// Wavefronts and LDS slots of a workgroup, at most 128 KB for what global_load_lds addresses:
// three units of 128-wide fp32 heads.  256-wide heads need twice the registers.
template <int HD> constexpr int waves_of() { return HD == 256 ? 4 : 8; }
template <int HD, int P> constexpr int slots_of() { return HD * P >= 512 ? 2 : HD * P == 256 ? 3 : 4; }

template <int HD, typename T>
__global__ __launch_bounds__(waves_of<HD>() * 64) void attn_kernel(PromptArgs a) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1, NW = waves_of<HD>(), S = slots_of<HD, P>();
    constexpr int UB = (int)unit_bytes(HD, P), PL = kUnit * HD * 2;  // bytes of a unit, of a plane
    constexpr int LD = (UB - 256) / 1024 / NW;                       // loads of a wavefront a unit, and the header
    constexpr int KS = HD / 16, DB = HD / 32;
    static_assert((UB - 256) % (1024 * NW) == 0 && (S - 1) * UB + UB - 1024 < 128 * 1024, "ring");
    __shared__ __attribute__((aligned(1024))) uint8_t ring[S * UB];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;
    const ggq_attention_prompt_params& p = a.p;
    const int kvh = blockIdx.x % p.n_kv_head, split = blockIdx.y;
    const int64_t id = a.tiles - 1 - blockIdx.x / p.n_kv_head;  // late rows see most: first
    constexpr int NC = NW * 32;
    int seq = 0;
    for (int i = 1; i < p.n_seq; i += NW * 64) {
        const int j = i + tid;
        seq += __syncthreads_count(j < p.n_seq && bound_of(max((int64_t)p.q_off[j], (int64_t)0) * a.G, NC, j) <= id);
    }
    const Span qs = span_of(p.q_off, seq, p.n_rows), ks = span_of(kv_off_of(p), seq, p.n_kv_rows);
    const int64_t f0 = (id - bound_of(qs.a * a.G, NC, seq)) * NC, nf = qs.n * a.G;
    if (f0 < 0 || f0 >= nf) return;
    const int64_t shift = ks.n - qs.n + 1;  // row i sees positions below shift + i
    const int64_t i0 = f0 / a.G, i1 = (min(nf, f0 + NC) - 1) / a.G;
    const int64_t wg_end = min(max(shift + i1, (int64_t)0), ks.n);
    const int64_t wg_beg = p.window ? max(shift + i0 - p.window, (int64_t)0) : 0;
    const int all0 = (int)(wg_beg / kUnit), all1 = (int)((wg_end + kUnit - 1) / kUnit);
    const int per = (max(all1 - all0, 0) + a.splits - 1) / a.splits;
    const int u0 = all0 + split * per, u1 = min(all1, u0 + per);

    // this lane's column
    const int64_t f = f0 + wave * 32 + col;
    const bool live = f < nf;
    const int64_t qi = live ? f / a.G : i1;
    const int head = kvh * a.G + (live ? (int)(f % a.G) : 0);
    const int end = live ? (int)min(max(shift + qi, (int64_t)0), ks.n) : 0;
    const int beg = live && p.window ? (int)max(shift + qi - p.window, (int64_t)0) : 0;
    int wend = end, wbeg = live ? beg : INT32_MAX, fend = live ? end : INT32_MAX, fbeg = beg;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        wend = max(wend, __shfl_xor(wend, o, 64));
        wbeg = min(wbeg, __shfl_xor(wbeg, o, 64));
        fend = min(fend, __shfl_xor(fend, o, 64));
        fbeg = max(fbeg, __shfl_xor(fbeg, o, 64));
    }
    wend = __builtin_amdgcn_readfirstlane(wend);
    wbeg = __builtin_amdgcn_readfirstlane(wbeg);
    fend = __builtin_amdgcn_readfirstlane(fend);
    fbeg = __builtin_amdgcn_readfirstlane(fbeg);

    const float* qrow = p.q + (qs.a + qi) * p.ldq + (int64_t)head * HD;
    h8 qh[KS], ql[KS];
    int qe;
    {
        uint32_t m = 0;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) m = max(m, mag_bits(qrow[16 * s + 8 * h + j] * p.scale));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        qe = up_to_2_15(m);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float x = live ? ldexpf(qrow[16 * s + 8 * h + j] * p.scale, qe) : 0.0f;
                qh[s][j] = (_Float16)x;
                ql[s][j] = finite(x) ? (_Float16)(x - (float)qh[s][j]) : (_Float16)0.0f;
            }
    }

    const uint32_t ring_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)ring;
    const uint8_t* units = a.planes + (bound_of(ks.a, kUnit, seq) * p.n_kv_head + kvh) * UB;
    auto fetch = [&](int i) {  // unit u0 + i (past the end the last one: every unit the same number of loads)
        const int u = min(u0 + i, u1 - 1), slot = i % S * UB;
        const uint8_t* src = units + (int64_t)u * p.n_kv_head * UB;
#pragma unroll
        for (int j = 0; j < LD; j++)
            dma16(src + 256 + (wave * LD + j) * 1024, (uint32_t)lane * 16u, ring_at + (uint32_t)(slot + 256 + (wave * LD + j) * 1024));
        dma4(src, (uint32_t)lane * 4u, ring_at + (uint32_t)slot);
    };

    f16v o[DB];
#pragma unroll
    for (int d = 0; d < DB; d++) o[d] = f16v{};
    float m = -INFINITY, l = 0.0f;
    int ve = 0, least = 1 << 20;  // exponent of the sums' unit; the least one of the values so far
    bool first = true;
    const int n = u1 - u0;
    if (n > 0) {
#pragma unroll
        for (int i = 0; i < S - 1; i++) fetch(i);
    }
    for (int it = 0; it < n; it++) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * (LD + 1)) : "memory");
        fetch(it + S - 1);
        const int base = (u0 + it) * kUnit;
        if (base >= wend || base + kUnit <= wbeg) continue;
        const uint8_t* slot = ring + it % S * UB;
        const uint32_t info = __builtin_amdgcn_readfirstlane(*(const uint32_t*)slot);
        const int ke = (int)(info & 1023u) - 512, ve_u = (int)(info >> 10 & 1023u) - 512;
        const h8* kp = (const h8*)(slot + 256) + lane;
        const bool masked = base + kUnit > fend || base < fbeg;  // for a column of this wavefront
        f16v st = {};
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const h8 kh = kp[s * 64];
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qh[s], st, 0, 0, 0);
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, ql[s], st, 0, 0, 0);
            if constexpr (P == 2) st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kp[s * 64 + PL / 16], qh[s], st, 0, 0, 0);
        }
        if (info & BAD_K || (masked && info & WIDE_K)) {
            // keys that are not finite, or hidden ones that leave the others few bits: the products as they are
            const T* kr = (const T*)p.k + (ks.a + base) * p.ldk + (int64_t)kvh * HD;
#pragma unroll 1
            for (int i = 0; i < 16; i++) {
                const int at = 8 * (i / 4) + 4 * h + i % 4;
                if (base + at >= ks.n) continue;
                float s = 0.0f;
#pragma unroll 1
                for (int d = 0; d < HD; d++) s = fmaf(qrow[d] * p.scale, (float)kr[at * p.ldk + d], s);
                s = ldexpf(s, qe + ke);
#pragma unroll
                for (int j = 0; j < 16; j++) st[j] = j == i ? s : st[j];
            }
        }
        if (masked) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int at = base + 8 * (i / 4) + 4 * h + i % 4;
                if (at >= end || at < beg) st[i] = -INFINITY;
            }
        }
        // to powers of two (an exponent beyond fp32's range gives a score of 0 or an infinite one either way)
        const float cs = ldexpf(1.0f, max(-126, min(127, -(qe + ke))));
        float top = max3(st[0], st[1], st[2]);
#pragma unroll
        for (int i = 3; i < 15; i += 2) top = max3(top, st[i], st[i + 1]);
        const Two th = halves(max3(top, st[15], st[15]));
        top = max3(th.a, th.b, th.b) * cs;
        if (__any(top > m + 4.0f)) {
            const float mn = max3(m, top, top);
            const float al = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= al;
#pragma unroll
            for (int d = 0; d < DB; d++) o[d] *= al;
        }
        float pscale = 1.0f;
        if constexpr (P == 2) {
            if (!(info & NO_V)) {
                // the sums follow the values' unit when those get larger, or smaller by more than
                // 2^8 (but stay within 2^64 of the largest so far); less than that, weights shrink
                least = min(least, ve_u);
                const int to = first || ve_u < ve || ve_u > ve + 8 ? min(ve_u, least + 64) : ve;
                first = false;
                if (to != ve) {
#pragma unroll
                    for (int d = 0; d < DB; d++)
#pragma unroll
                        for (int i = 0; i < 16; i++) o[d][i] = ldexpf(o[d][i], to - ve);
                    ve = to;
                }
                if (to != ve_u) pscale = ldexpf(1.0f, max(-126, to - ve_u));
            }
        }
        const float ref = m == -INFINITY ? 0.0f : m - 11.0f;
        float e[16];
#pragma unroll
        for (int i = 0; i < 16; i++) {
            e[i] = __builtin_amdgcn_exp2f(fmaf(st[i], cs, -ref));
            l += e[i];
        }
        if (P == 2 && pscale != 1.0f) {
#pragma unroll
            for (int i = 0; i < 16; i++) e[i] *= pscale;
        }
        const h8* vp = kp + P * PL / 16;
        if (P == 2 && masked && info & WIDE_V) {
            // hidden values that leave the others few bits: the products as they are
            const T* vr = (const T*)p.v + (ks.a + base) * p.ldv + (int64_t)kvh * HD;
            const float un = 1.0f / pscale;
#pragma unroll 1
            for (int at = 0; at < kUnit; at++) {
                const float w = weight_of(e, at, col) * un;
                if (base + at >= end || base + at < beg) continue;
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        o[d][i] = fmaf(w, ldexpf((float)vr[at * p.ldv + 32 * d + 8 * (i / 4) + 4 * h + i % 4], ve), o[d][i]);
            }
            continue;
        }
#pragma unroll
        for (int t = 0; t < 2; t++) {
            h8 ph, pl;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                ph[j] = (_Float16)e[8 * t + j];
                pl[j] = (_Float16)(e[8 * t + j] - (float)ph[j]);
            }
#pragma unroll
            for (int d = 0; d < DB; d++) {
                const h8 vh = vp[(2 * d + t) * 64];
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, ph, o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh, pl, o[d], 0, 0, 0);
                if constexpr (P == 2) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vp[(2 * d + t) * 64 + PL / 16], ph, o[d], 0, 0, 0);
            }
        }
        if (info & BAD_V) {
            // values that are not finite are zero in the planes: here they come, to the rows that see them
            const T* vr = (const T*)p.v + (ks.a + base) * p.ldv + (int64_t)kvh * HD;
#pragma unroll 1
            for (int at = 0; at < kUnit; at++) {
                const float w = weight_of(e, at, col);
                if (base + at >= end || base + at < beg) continue;
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float v = (float)vr[at * p.ldv + 32 * d + 8 * (i / 4) + 4 * h + i % 4];
                        if (!finite(v)) o[d][i] += w * v;
                    }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (nothing lands in LDS behind the end)
    const Two lh = halves(l);
    l = lh.a + lh.b;
    if (!live) return;
    const bool none = end <= beg;
    const float inv = 1.0f / l;
    if (a.splits == 1) {
        float* out = p.out + (qs.a + qi) * p.ldo + (int64_t)head * HD + 4 * h;
#pragma unroll
        for (int d = 0; d < DB; d++)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                float4 r;
                r.x = none ? 0.0f : ldexpf(o[d][i] * inv, -ve);
                r.y = none ? 0.0f : ldexpf(o[d][i + 1] * inv, -ve);
                r.z = none ? 0.0f : ldexpf(o[d][i + 2] * inv, -ve);
                r.w = none ? 0.0f : ldexpf(o[d][i + 3] * inv, -ve);
                *(float4*)(out + 32 * d + 2 * i) = r;
            }
        return;
    }
    // this part's weighted mean, its maximum and its sum
    float* part = a.part + (((qs.a + qi) * p.n_head + head) * a.splits + split) * (HD + 4);
    const bool empty = m == -INFINITY && l == 0.0f;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float4 r;
            r.x = empty ? 0.0f : ldexpf(o[d][i] * inv, -ve);
            r.y = empty ? 0.0f : ldexpf(o[d][i + 1] * inv, -ve);
            r.z = empty ? 0.0f : ldexpf(o[d][i + 2] * inv, -ve);
            r.w = empty ? 0.0f : ldexpf(o[d][i + 3] * inv, -ve);
            *(float4*)(part + 32 * d + 2 * i + 4 * h) = r;
        }
    if (h == 0) { part[HD] = m; part[HD + 1] = l; }
}

// The parts of one row's head, in their order.
template <int HD> __global__ __launch_bounds__(256) void attn_join_kernel(PromptArgs a) {
    const ggq_attention_prompt_params& p = a.p;
    const int row = blockIdx.x, d = threadIdx.x;
    const int seq = seq_of(p.q_off, p.n_seq, row);
    if (seq >= p.n_seq || row < p.q_off[seq] || d >= HD) return;
    for (int head = blockIdx.y; head < p.n_head; head += gridDim.y) {
        const float* q = a.part + ((int64_t)row * p.n_head + head) * a.splits * (HD + 4);
        float mx = -INFINITY;
        for (int i = 0; i < a.splits; i++) mx = fmaxf(mx, q[(int64_t)i * (HD + 4) + HD]);
        float ls = 0.0f, os = 0.0f;
        for (int i = 0; i < a.splits; i++) {
            const float* x = q + (int64_t)i * (HD + 4);
            const float w = x[HD] == -INFINITY && x[HD + 1] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(x[HD] - mx) * x[HD + 1];
            ls += w;
            os = fmaf(x[d], w, os);
        }
        p.out[(int64_t)row * p.ldo + (int64_t)head * HD + d] = mx == -INFINITY && ls == 0.0f ? 0.0f : os / ls;
    }
}

}  // namespace

namespace {
int64_t units_of(const ggq_attention_prompt_params& p) { return (int64_t)p.n_kv_rows / kUnit + p.n_seq; }
int64_t tiles_of(const ggq_attention_prompt_params& p) {
    const int nc = (p.head_dim == 256 ? 4 : 8) * 32;
    return (int64_t)p.n_rows * (p.n_head / p.n_kv_head) / nc + p.n_seq;
}
size_t planes_bytes(const ggq_attention_prompt_params& p) {
    return (size_t)(units_of(p) * p.n_kv_head * unit_bytes(p.head_dim, p.type == GGQ_TYPE_F32 ? 2 : 1));
}
}  // namespace

AttnPromptPlan attn_prompt_plan(const ggq_attention_prompt_params& p) {
    AttnPromptPlan pl{};
    // few tiles: the positions in parts, while each keeps 8 units
    const int64_t wgs = tiles_of(p) * p.n_kv_head, units = units_of(p);
    pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>(cu_count() / wgs, units / 8));
    if (p.n_rows > 65535) pl.splits = 1;
    pl.ws_bytes = (planes_bytes(p) + 255) / 256 * 256;
    if (pl.splits > 1) pl.ws_bytes += sizeof(float) * (size_t)p.n_rows * p.n_head * pl.splits * (p.head_dim + 4);
    return pl;
}

hipError_t launch_attn_prompt(const ggq_attention_prompt_params& p, const AttnPromptPlan& pl, void* ws, hipStream_t s) {
    PromptArgs a{};
    a.p = p;
    a.planes = (uint8_t*)ws;
    a.part = (float*)((char*)ws + (planes_bytes(p) + 255) / 256 * 256);
    a.G = p.n_head / p.n_kv_head;
    a.splits = pl.splits;
    a.tiles = (int)tiles_of(p);
    const dim3 pre((unsigned)units_of(p), (unsigned)p.n_kv_head), grid((unsigned)(a.tiles * (int64_t)p.n_kv_head), (unsigned)pl.splits);
#define L(HD_, T_)                                                               \
    planes_kernel<HD_, T_><<<pre, 256, 0, s>>>(a);                               \
    attn_kernel<HD_, T_><<<grid, waves_of<HD_>() * 64, 0, s>>>(a);               \
    if (pl.splits > 1) attn_join_kernel<HD_><<<dim3((unsigned)p.n_rows, (unsigned)std::min(p.n_head, 8)), HD_, 0, s>>>(a)
#define BY_T(HD_)                                        \
    if (p.type == GGQ_TYPE_F32) { L(HD_, float); }       \
    else { L(HD_, _Float16); }
    if (p.head_dim == 64) { BY_T(64) }
    else if (p.head_dim == 128) { BY_T(128) }
    else { BY_T(256) }
#undef BY_T
#undef L
    return hipGetLastError();
}

hipError_t launch_attn_prompt_rows(const ggq_attention_prompt_params& p, hipStream_t s) {
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
