// ggq_attn_prompt.hip -- causal attention of packed prompts.
//
// The keys and values a call sees are first written as planes of fp16 operands
// (planes_kernel): 32 positions of one kv head a unit, fp32 values as hi + lo
// under a power of two of their position (22 bits of its largest), in the
// order in which the matrix cores take them, values transposed.  attn_kernel
// then computes per unit, with v_mfma_f32_32x32x16_f16,
//   S^T[position][column] = K Q^T,  O^T[value][column] += V^T P^T
// as the products hi lo + lo hi + hi hi of fp32 keys and values (hi lo + hi hi with fp16
// ones, which need no split).  Queries and weights are cut to hi (11 bits) and lo, keys and
// values rounded to hi and lo: 22 bits of the largest value of a row each, and lo lo is left
// out, so a product is off by up to 2^-20 of it where fp32 has 2^-24.  The small products of a score
// come first, which leaves a rounding a step of 16 hi hi products; against 64 bits the results
// are off by 2.8e-7 in the mean over 720 drawn calls where elementary fp32 operations are by 5.0e-7.
//   A column is one (query row, head) pair: the rows of a sequence and the
// heads that share a kv head are numbered through, 32 columns a wavefront,
// so any ratio of heads fills the tiles and all wavefronts of a workgroup share
// each unit in LDS.
//   S^T leaves a lane with 16 positions of its column, and P^T wants 8 positions a lane and
// step of the same column: the values' planes are ordered so that these are the
// same ones, and weights go from one product to the next in registers.
//   Units arrive straight from memory (global_load_lds) in two LDS slots for keys
// and two for values.  A wavefront's unit has two phases, weights (VALU: maximum,
// exponentials, split) and products (this unit's O^T, the next one's S^T); the second half of a
// workgroup's wavefronts, which share the SIMDs with the first, runs a phase behind
// it, so that one of two is always at the matrix cores while the other is not.
//   The maximum moves only when a unit exceeds it by 2^4; weights are kept times
// 2^11 (at most 2^15), so hi + lo of a small weight keeps 2^-36 of the largest (with values
// that the planes do not bring closer than 2^8: 2^-28 of the largest product).
// Scores take their position's power of two back; weights take the values', relative to
// the unit of the row's running sums, which follows the largest product of weight and value
// that the row has seen: neither a position that it does not see nor one of next to no
// weight has a say in what it keeps of the others.
// Bound: the matrix cores, at the clock that their load leaves (8191 rows of 32
// heads of 128 in fp32: 1.38 to 1.48 ms on several cards, 1.1 to 1.2 PFLOP/s of fp16 products, what the
// library's matmul reaches; a unit about 5100 cycles, three fifths of them products).
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "ggq_attn.h"
#include "ggq_attn_device.h"
#include "ggq_launch.h"

namespace ggq {
namespace {

// ------------------------------------------------------------ matrix cores
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr int kUnit = 32;  // positions
// Header of a unit: for each position how many powers of two its K and V planes
// are scaled beyond those of the unit's largest values, as negative numbers
// (32 of K, 32 of V; 16 bits each where 32 would bring the LDS of a workgroup to 128 KB), then
// dwords, all alike: those ones' exponents (+ 512), whether some values are not
// finite (zero in the planes), whether there are any but zero, whether any of
// the numbers before is not zero.  (Up to 2^8 below the unit's largest hi + lo
// keep all that matters: zero.)
template <int HD> struct Head {
    typedef int num;
    static constexpr int bytes = 512, info = 256;
};
template <> struct Head<256> {
    typedef int16_t num;
    static constexpr int bytes = 256, info = 128;
};
// Bytes of a unit: header, K and V planes.
template <int HD> constexpr int64_t unit_bytes(int planes) { return (int64_t)planes * 2 * kUnit * HD * 2 + Head<HD>::bytes; }
// Exponents between that of an all-zero row of values and its unit's (an int16_t with the sign changed).
constexpr int kZero = 4096;
enum { BAD_V = 1 << 20, NO_V = 1 << 21, OWN_K = 1 << 22, OWN_V = 1 << 23 };

// Sequence s has the units from off[s] / 32 + s on (and as many column tiles of
// n from off[s] * G / n + s): a bound that needs no sum over the sequences before.
__device__ __forceinline__ int64_t bound_of(int64_t first, int64_t per, int s) { return first / per + s; }

struct PromptArgs {
    ggq_attention_prompt_params p;
    uint8_t* planes;
    float* part;
    int G, tiles, splits;
    int kv0, kvn;  // the kv heads of this launch, whose planes there is room for
};

// A sequence's rows of an offset array, held inside [0, n].
struct Span {
    int64_t a, n;
};
__device__ __forceinline__ Span span_of(const int32_t* off, int s, int64_t most) {
    const int64_t a = min(max((int64_t)off[s], (int64_t)0), most), b = min(max((int64_t)off[s + 1], (int64_t)0), most);
    return Span{a, b > a ? b - a : 0};
}
// The first position that a row with `below` positions at or before its own sees (below < 1: none are).  A window
// may be anything up to INT32_MAX: nothing is subtracted from a negative number.
__device__ __forceinline__ int first_of(int below, int window) { return window ? max(max(below, 0) - window, 0) : 0; }
__device__ __forceinline__ const int32_t* kv_off_of(const ggq_attention_prompt_params& p) { return p.kv_off ? p.kv_off : p.q_off; }

__device__ __forceinline__ uint32_t mag_bits(float v) {  // 0 for what is not finite
    const uint32_t u = __builtin_bit_cast(uint32_t, v) & 0x7FFFFFFFu;
    return u >= 0x7F800000u ? 0u : u;
}
__device__ __forceinline__ bool finite(float v) { return (__builtin_bit_cast(uint32_t, v) & 0x7F800000u) != 0x7F800000u; }

// Exponent that brings a magnitude into [2^14, 2^15).
__device__ __forceinline__ int up_to_2_15(uint32_t bits) { return bits ? 141 - (int)(bits >> 23) : 0; }

// Few rows, few keys, or no workspace: kCols columns of one sequence and kv head a
// workgroup, on the VALU in fp32.  The four wavefronts take 16 positions each in turn, keys
// and values in flight together; four lanes share a position for the scores (its key
// against all columns' queries), a lane has HD / 64 values for the sums, and the
// wavefronts' sums meet in LDS.  One launch of few dependent loads.
constexpr int kCols = 4;
template <int HD, typename T>
__global__ __launch_bounds__(256) void attn_few_kernel(PromptArgs a) {
    constexpr int DPL = HD / 64, C = kCols, PR = 16 / sizeof(T);
    static_assert(C == 4, "a quad of lanes writes a position's weights");
    __shared__ __attribute__((aligned(16))) float sq[C][HD], sp[4][16][C], so[4][C][HD], sm[4][C], sl[4][C];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const ggq_attention_prompt_params& p = a.p;
    const int kvh = blockIdx.x % p.n_kv_head, G = a.G;
    const int id = a.tiles - 1 - (int)(blockIdx.x / p.n_kv_head);
    int seq = 0;
    for (int i = 1; i < p.n_seq; i += 256) {
        const int j = i + tid;
        seq += __syncthreads_count(j < p.n_seq && (int)((uint32_t)max(min(p.q_off[j], p.n_rows), 0) * G / C) + j <= id);
    }
    const Span qs = span_of(p.q_off, seq, p.n_rows), ks = span_of(kv_off_of(p), seq, p.n_kv_rows);
    const int nf = (int)qs.n * G, f0 = (id - ((int)((uint32_t)qs.a * G / C) + seq)) * C;
    if (f0 < 0 || f0 >= nf) return;
    const int n_keys = (int)ks.n, shift = n_keys - (int)qs.n + 1, nc = min(C, nf - f0);
    int beg[C], end[C], first = n_keys, last = 0, all = n_keys, none = 0;
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int qi = (int)((uint32_t)min(f0 + c, nf - 1) / G);
        end[c] = min(max(shift + qi, 0), n_keys);
        beg[c] = min(first_of(shift + qi, p.window), n_keys);
        first = min(first, beg[c]);
        last = max(last, end[c]);
        none = max(none, beg[c]);  // every column sees [none, all)
        all = min(all, end[c]);
    }
    for (int e = tid; e < C * HD; e += 256) {
        const int f = min(f0 + e / HD, nf - 1), qi = (int)((uint32_t)f / G);
        sq[e / HD][e % HD] = p.q[(qs.a + qi) * p.ldq + (int64_t)(kvh * G + f - qi * G) * HD + e % HD] * p.scale;
    }
    __syncthreads();
    const T* kb = (const T*)p.k + ks.a * p.ldk + (int64_t)kvh * HD;
    const T* vb = (const T*)p.v + ks.a * p.ldv + (int64_t)kvh * HD + lane * DPL;
    float m[C], l[C], o[C][DPL];
#pragma unroll
    for (int c = 0; c < C; c++) {
        m[c] = -INFINITY;
        l[c] = 0.0f;
#pragma unroll
        for (int d = 0; d < DPL; d++) o[c][d] = 0.0f;
    }
    struct alignas(16) Run { T x[PR]; };
    struct alignas(DPL * sizeof(T)) Vals { T x[DPL]; };
    constexpr int NR = HD / 4 / PR;  // runs of a lane: the ones 4 i + lane % 4 of its key
    const int quad = lane & 3, at = lane >> 2;
    for (int base = first + wave * 16; base < last; base += 64) {
        const int pos = base + at, n = min(16, last - base);
        const Run* kr = (const Run*)(kb + (int64_t)min(pos, last - 1) * p.ldk) + quad;
        Run k[NR];
#pragma unroll
        for (int i = 0; i < NR; i++) k[i] = kr[4 * i];
        constexpr int VJ = HD == 256 ? 8 : 16;  // values in flight
        Vals v[VJ];
        auto values = [&](int j0) {
#pragma unroll
            for (int j = 0; j < VJ; j++) v[j] = *(const Vals*)(vb + (int64_t)(base + min(j0 + j, n - 1)) * p.ldv);
        };
        values(0);
        float s[C] = {};
#pragma unroll
        for (int i = 0; i < NR; i++)
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int j = 0; j < PR; j++) s[c] = fmaf(sq[c][(4 * i + quad) * PR + j], (float)k[i].x[j], s[c]);
#pragma unroll
        for (int c = 0; c < C; c++) {
            float t = s[c];
            t += __shfl_xor(t, 1, 64);
            t += __shfl_xor(t, 2, 64);
            if (pos < beg[c] || pos >= end[c]) t = -INFINITY;
            float mx = t;
            mx = max3(mx, __shfl_xor(mx, 4, 64), mx);
            mx = max3(mx, __shfl_xor(mx, 8, 64), mx);
            const Two x = rows16(mx), y = halves(max3(x.a, x.b, x.b));
            mx = max3(y.a, y.b, y.b);
            const float mn = max3(m[c], mx, mx), ref = mn == -INFINITY ? 0.0f : mn;
            const float al = __builtin_amdgcn_exp2f(m[c] - ref), e = __builtin_amdgcn_exp2f(t - ref);
            m[c] = mn;
            l[c] = l[c] * al + (quad == 0 ? e : 0.0f);  // (a lane's share)
            if (quad == c) sp[wave][at][c] = e;
#pragma unroll
            for (int d = 0; d < DPL; d++) o[c][d] *= al;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const bool seen = base >= none && base + 16 <= all;  // by every column
        auto add = [&](auto whole) {
#pragma unroll
            for (int j = 0; j < 16; j++) {
                if (j == VJ) values(j);
                const float4 w = *(const float4*)sp[wave][j];
                const float wc[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int d = 0; d < DPL; d++) {
                        // (a value that is not seen may be anything)
                        const float t = fmaf(wc[c], (float)v[j % VJ].x[d], o[c][d]);
                        o[c][d] = whole || wc[c] != 0.0f ? t : o[c][d];
                    }
            }
        };
        if (seen) add(std::true_type{});
        else add(std::false_type{});
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int c = 0; c < C; c++) {
#pragma unroll
        for (int o_ = 1; o_ < 64; o_ <<= 1) l[c] += __shfl_xor(l[c], o_, 64);
        if (lane == 0) { sm[wave][c] = m[c]; sl[wave][c] = l[c]; }
#pragma unroll
        for (int d = 0; d < DPL; d++) so[wave][c][lane * DPL + d] = o[c][d];
    }
    __syncthreads();
    for (int e = tid; e < nc * HD; e += 256) {
        const int c = e / HD, d = e % HD, f = f0 + c, qi = (int)((uint32_t)f / G);
        const float mx = max3(max3(sm[0][c], sm[1][c], sm[2][c]), sm[3][c], sm[3][c]);
        float ls = 0.0f, os = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float al = sm[w][c] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[w][c] - mx);
            ls = fmaf(sl[w][c], al, ls);
            os = fmaf(so[w][c][d], al, os);
        }
        bool sees = false;
#pragma unroll
        for (int i = 0; i < C; i++) sees |= i == c && beg[i] < end[i];
        p.out[(qs.a + qi) * p.ldo + (int64_t)(kvh * G + f - qi * G) * HD + d] = sees ? os / ls : 0.0f;
    }
}

template <int HD, typename T>
__global__ __launch_bounds__(256) void planes_kernel(PromptArgs a) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1, V = HD / 8;  // planes, values of a thread
    constexpr int PL = kUnit * HD;                         // values of a plane
    __shared__ float sv[kUnit][HD + 1];
    __shared__ uint32_t red[4][3];
    const int tid = threadIdx.x, kvh = a.kv0 + blockIdx.y;
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
    const int64_t row = sp.a + min(u * kUnit + pos, sp.n - 1);
    struct alignas(16) Run { T x[16 / sizeof(T)]; };
    constexpr int PR = 16 / sizeof(T), NR = V / PR;
    const Run* kr = (const Run*)((const T*)a.p.k + row * a.p.ldk + (int64_t)kvh * HD + d0);
    const Run* vr = (const Run*)((const T*)a.p.v + row * a.p.ldv + (int64_t)kvh * HD + d0);
    Run kin[NR], vin[NR];
#pragma unroll
    for (int i = 0; i < NR; i++) { kin[i] = kr[i]; vin[i] = vr[i]; }
    float k[V], v[V];
    uint32_t mk = 0, mv = 0, bad = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        k[i] = in ? (float)kin[i / PR].x[i % PR] : 0.0f;
        v[i] = in ? (float)vin[i / PR].x[i % PR] : 0.0f;
        mk = max(mk, mag_bits(k[i]));
        mv = max(mv, mag_bits(v[i]));
        if (!finite(v[i])) {
            bad |= BAD_V;
            v[i] = 0.0f;
        }
    }
    // the positions' largest (8 threads each), the unit's
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        mk = max(mk, (uint32_t)__shfl_xor((int)mk, o, 64));
        mv = max(mv, (uint32_t)__shfl_xor((int)mv, o, 64));
    }
    uint32_t uk = mk, uv = mv;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        if (o >= 8) {
            uk = max(uk, (uint32_t)__shfl_xor((int)uk, o, 64));
            uv = max(uv, (uint32_t)__shfl_xor((int)uv, o, 64));
        }
        bad |= (uint32_t)__shfl_xor((int)bad, o, 64);
    }
    if ((tid & 63) == 0) {
        uint32_t* r = red[tid >> 6];
        r[0] = uk; r[1] = uv; r[2] = bad;
    }
    __syncthreads();
    uk = max(max(red[0][0], red[1][0]), max(red[2][0], red[3][0]));
    uv = max(max(red[0][1], red[1][1]), max(red[2][1], red[3][1]));
    bad = red[0][2] | red[1][2] | red[2][2] | red[3][2];
    // fp16 values stay as they are
    const int ku = P == 2 ? up_to_2_15(uk) : 0, vu = P == 2 ? up_to_2_15(uv) : 0;
    int ke = P == 2 && mk ? up_to_2_15(mk) : ku, ve = P == 2 && mv ? up_to_2_15(mv) : vu;
    if (ke <= ku + 8) ke = ku;
    if (ve <= vu + 8) ve = vu;
    // values that are all zero have any exponent: one that stands for no value (of a unit with others: hidden ones
    // must not lend it theirs)
    if (P == 2 && in && !mv && uv) ve = vu + kZero;
    const int own_k = __syncthreads_or(ke != ku), own_v = __syncthreads_or(ve != vu);
    typedef typename Head<HD>::num num;
    uint8_t* out = a.planes + (id * a.kvn + (kvh - a.kv0)) * unit_bytes<HD>(P);
    if (tid % 8 == 0) {
        ((num*)out)[pos] = (num)(ku - ke);
        ((num*)out)[32 + pos] = (num)(vu - ve);
    }
    if (tid < (Head<HD>::bytes - Head<HD>::info) / 4)
        ((uint32_t*)(out + Head<HD>::info))[tid] = (uint32_t)(ku + 512) | (uint32_t)(vu + 512) << 10 | bad | (uv ? 0 : NO_V) |
                                                    (own_k ? OWN_K : 0) | (own_v ? OWN_V : 0);
    _Float16* kp = (_Float16*)(out + Head<HD>::bytes);
#pragma unroll
    for (int i = 0; i < V; i += 8) {
        h8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float x = P == 2 ? ldexpf(k[i + j], ke) : k[i + j];
            hi[j] = (_Float16)x;
            lo[j] = (_Float16)(x - (float)hi[j]);  // (NaN for an infinity)
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


// fp16 parts j and j + 1 of a pair of values: hi cut, lo rounded (2^-22 of the value).
// minus1 is -1 where the compiler does not see it, which makes value - hi one
// instruction on the packed halves (v_fma_mix_f32).
__device__ __forceinline__ void split_pair(float a, float b, h2 minus1, h8& hi, h8& lo, int j) {
    const auto p = __builtin_amdgcn_cvt_pkrtz(a, b);
    const h2 q = __builtin_bit_cast(h2, p);
    hi[j] = q[0];
    hi[j + 1] = q[1];
    lo[j] = (_Float16)fmaf((float)q[0], (float)minus1[0], a);
    lo[j + 1] = (_Float16)fmaf((float)q[1], (float)minus1[1], b);
}

// Wavefronts of a workgroup: two a SIMD, or one of 256-wide heads, whose sums and
// queries take more than half of the registers.
template <int HD> constexpr int waves_of() { return HD == 256 ? 4 : 8; }

// All of this wavefront's reads of LDS are done, and with `loads` its loads into it; then
// the workgroup's.
__device__ __forceinline__ void phase_end(bool loads) {
    if (loads) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int HD, typename T>
__global__ __launch_bounds__(waves_of<HD>() * 64) void attn_kernel(PromptArgs a) {
    constexpr int P = sizeof(T) == 4 ? 2 : 1, NW = waves_of<HD>(), PL = kUnit * HD * 2;  // PL: bytes of a plane
    constexpr int64_t UB = unit_bytes<HD>(P);
    typedef typename Head<HD>::num num;
    constexpr int HB = Head<HD>::bytes, KB = HB + P * PL, VB = P * PL;          // LDS bytes of a unit's header and keys, of its values
    constexpr int KC = P * PL / 1024, LD = 2 * KC / 4;       // 1 KB loads of the keys; of a loading wavefront a unit (and the header)
    constexpr int KS = HD / 16, DB = HD / 32;
    static_assert(2 * KC % 4 == 0 && 2 * (KB + VB) - 1024 < 128 * 1024, "LDS that global_load_lds addresses");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * (KB + VB)];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, h = lane >> 5;
    const bool behind = NW == 8 && wave >= 4;  // runs a phase behind the others
    const bool loads = NW == 4 || behind;      // (those have time while the others are at the matrix cores)
    const ggq_attention_prompt_params& p = a.p;
    const int kvi = (int)(blockIdx.x % (unsigned)a.kvn), kvh = a.kv0 + kvi, split = blockIdx.y, G = a.G;
    const int id = a.tiles - 1 - (int)(blockIdx.x / (unsigned)a.kvn);  // late rows see most: first
    constexpr int NC = NW * 32;
    int seq = 0;
    for (int i = 1; i < p.n_seq; i += NW * 64) {
        const int j = i + tid;
        seq += __syncthreads_count(j < p.n_seq && (int)((uint32_t)max(min(p.q_off[j], p.n_rows), 0) * G / NC) + j <= id);
    }
    const Span qs = span_of(p.q_off, seq, p.n_rows), ks = span_of(kv_off_of(p), seq, p.n_kv_rows);
    // (n_rows * G fits 31 bits: the caller sees to it)
    const int nf = (int)qs.n * G, f0 = (id - ((int)((uint32_t)qs.a * G / NC) + seq)) * NC;
    if (f0 < 0 || f0 >= nf) return;
    const int n_keys = (int)ks.n, shift = n_keys - (int)qs.n + 1;  // row i sees positions below shift + i
    const int i0 = (int)((uint32_t)f0 / G), i1 = (int)((uint32_t)(min(nf, f0 + NC) - 1) / G);
    const int wg_end = min(max(shift + i1, 0), n_keys);
    const int wg_beg = first_of(shift + i0, p.window);
    const int all0 = wg_beg / kUnit, all1 = (wg_end + kUnit - 1) / kUnit;
    const int per = (max(all1 - all0, 0) + a.splits - 1) / a.splits;
    const int u0 = all0 + split * per, u1 = min(all1, u0 + per), n = u1 - u0;

    // loads for iteration it: the keys of its next but one unit, the values of its next (outside of what
    // there is, the nearest unit: the same number of loads each time).  Two of the four wavefronts
    // that load take the keys, two the values, LD KB in a row each.
    const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
    const uint8_t* units = a.planes + ((bound_of(ks.a, kUnit, seq) + u0) * a.kvn + kvi) * UB;
    const int64_t stride = a.kvn * UB;
    const int share = wave & 3;
    const bool of_k = share < 2;
    const uint8_t* const mine = units + (of_k ? HB + share * LD * 1024 : KB + (share * LD - KC) * 1024);
    const uint32_t to = lds_at + (of_k ? (uint32_t)(HB + share * LD * 1024) : (uint32_t)(2 * KB + (share * LD - KC) * 1024));
    auto fetch = [&](int it) {
        const int uk = min(it + 2, n - 1), uv = max(min(it + 1, n - 1), 0);
        const uint8_t* src = mine + (of_k ? uk : uv) * stride;
        const uint32_t dst = to + (uint32_t)(of_k ? (it & 1) * KB : ((it + 1) & 1) * VB);
        const uint8_t* head = units + uk * stride;
        const uint32_t hdst = lds_at + (uint32_t)((it & 1) * KB);
        dma4(head, (uint32_t)lane * 4u, hdst);
        if constexpr (HB == 512) dma4(head + 256, (uint32_t)lane * 4u, hdst + 256u);
#pragma unroll
        for (int j = 0; j < LD; j++) dma16(src + j * 1024, (uint32_t)lane * 16u, dst + (uint32_t)j * 1024u);
    };
    if (n > 0 && loads) {
        fetch(-2);
        fetch(-1);
    }

    // this lane's column
    const int f = f0 + wave * 32 + col;
    const bool live = f < nf;
    const int qi = live ? (int)((uint32_t)f / G) : i1;
    const int head = kvh * G + (live ? f - qi * G : 0);
    const int end = live ? min(max(shift + qi, 0), n_keys) : 0;
    const int beg = live ? first_of(shift + qi, p.window) : 0;
    // rows ascend with the columns: the first and the last live one bound what the wavefront sees
    const int fl = f0 + wave * 32, last = min(fl + 31, nf - 1);
    const bool any = fl < nf, full = fl + 31 < nf;
    const int ra = any ? (int)((uint32_t)fl / G) : 0, rb = any ? (int)((uint32_t)last / G) : 0;
    const int wend = any ? min(max(shift + rb, 0), n_keys) : 0, wbeg = first_of(shift + ra, p.window);
    const int fend = full ? min(max(shift + ra, 0), n_keys) : 0;  // (with columns that are no rows: masked throughout)
    const int fbeg = first_of(shift + rb, p.window);

    h2 minus1 = {(_Float16)-1.0f, (_Float16)-1.0f};
    asm volatile("" : "+v"(minus1));
    const float* qrow = p.q + (qs.a + qi) * p.ldq + (int64_t)head * HD;
    h8 qh[KS], ql[KS];
    int qe;
    {
        float4 x[2 * KS];
        uint32_t m = 0;
#pragma unroll
        for (int s = 0; s < 2 * KS; s++) x[s] = *(const float4*)(qrow + 16 * (s / 2) + 8 * h + 4 * (s % 2));
#pragma unroll
        for (int s = 0; s < 2 * KS; s++) {
            x[s] = make_float4(x[s].x * p.scale, x[s].y * p.scale, x[s].z * p.scale, x[s].w * p.scale);
            m = max(max(max(m, mag_bits(x[s].x)), mag_bits(x[s].y)), max(mag_bits(x[s].z), mag_bits(x[s].w)));
        }
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        qe = up_to_2_15(m);
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const float v[8] = {x[2 * s].x, x[2 * s].y, x[2 * s].z, x[2 * s].w, x[2 * s + 1].x, x[2 * s + 1].y, x[2 * s + 1].z, x[2 * s + 1].w};
#pragma unroll
            for (int j = 0; j < 8; j += 2)  // (NaN for an infinity, and so is its row)
                split_pair(ldexpf(v[j], qe), ldexpf(v[j + 1], qe), minus1, qh[s], ql[s], j);
        }
    }

    f16v o[DB], st;
#pragma unroll
    for (int d = 0; d < DB; d++) o[d] = f16v{};
    float m = -INFINITY, l = 0.0f;
    // the column's sums are in units of 2^-ve; `least`: the unit in which what they hold would be at its limit
    constexpr int kNone = 1 << 20;
    int ve = 0, least = kNone;
    uint32_t info = 0, bad = 0;
    auto skips = [&](int it) {  // none of the wavefront's columns sees anything of the unit
        const int base = (u0 + it) * kUnit;
        return base >= wend || base + kUnit <= wbeg;
    };
    auto masks = [&](int it) {  // one of them does not see all of it
        const int base = (u0 + it) * kUnit;
        return base + kUnit > fend || base < fbeg;
    };
    // this lane's 16 of a header's 32 numbers
    auto numbers = [&](const uint8_t* from, int (&x)[16]) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            struct alignas(4 * sizeof(num)) Four { num x[4]; };
            const Four v = *(const Four*)(from + sizeof(num) * (2 * i + 4 * h));
#pragma unroll
            for (int j = 0; j < 4; j++) x[i + j] = v.x[j];
        }
    };
    int dv[P == 2 ? 16 : 1];
    auto open = [&](int it) { info = __builtin_amdgcn_readfirstlane(*(const uint32_t*)(lds + (it & 1) * KB + Head<HD>::info)); };
    auto scores = [&](int it) {
        const h8* kp = (const h8*)(lds + (it & 1) * KB + HB) + lane;
        // the small products first: the hi hi ones alone round at the size of the sum (head_dim / 16 of them)
        st = f16v{};
#pragma unroll
        for (int s = 0; s < KS; s++) {
            st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kp[s * 64], ql[s], st, 0, 0, 0);
            if constexpr (P == 2) st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kp[s * 64 + PL / 16], qh[s], st, 0, 0, 0);
        }
#pragma unroll
        for (int s = 0; s < KS; s++) st = __builtin_amdgcn_mfma_f32_32x32x16_f16(kp[s * 64], qh[s], st, 0, 0, 0);
    };
    auto powers = [&](int it) {
        const uint8_t* slot = lds + (it & 1) * KB;
        // (the slot is loaded over before the weights of the wavefronts behind)
        if constexpr (P == 2) {
            if (info & OWN_K) {  // (scores in one step: the unit's exponent may be that of hidden keys, far from the seen ones')
                const int ku = (int)(info & 1023u) - 512;
                int dk[16];
                numbers(slot, dk);
#pragma unroll
                for (int i = 0; i < 16; i++) st[i] = ldexpf(st[i], dk[i] - ku - qe);
            }
            if (info & OWN_V) numbers(slot + 32 * sizeof(num), dv);
        }
    };
    h8 ph[2], pl[2];
    auto weights = [&](int it) {
        const int base = (u0 + it) * kUnit;
        const bool masked = masks(it);
        const int ku = (int)(info & 1023u) - 512, vu = (int)(info >> 10 & 1023u) - 512;
        bad |= info;
        if (masked) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int at = base + 8 * (i / 4) + 4 * h + i % 4;
                if (at >= end || at < beg) st[i] = -INFINITY;
            }
        }
        // to powers of two, where powers() has not (an exponent beyond fp32's range gives a score of 0 or an infinite one
        // either way)
        const float cs = P == 2 && (info & OWN_K) ? 1.0f : ldexpf(1.0f, max(-126, min(127, -(qe + ku))));
        float top = max3(st[0], st[1], st[2]);
#pragma unroll
        for (int i = 3; i < 15; i += 2) top = max3(top, st[i], st[i + 1]);
        const Two th = halves(max3(top, st[15], st[15]));
        top = max3(th.a, th.b, th.b) * cs;
        if (__any(top > m + 4.0f)) {
            const float mn = max3(m, top, top);
            const float al = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
            if (P == 2 && m > -INFINITY) least = min(least + (int)fminf(mn - m, 4096.0f), kNone);  // (so much do the sums shrink)
            m = mn;
            l *= al;
#pragma unroll
            for (int d = 0; d < DB; d++) o[d] *= al;
        }
        // the weights' power of two besides 2^(11 - m)
        int c = 0;
        if constexpr (P == 2) {
            // In the sums' unit a position's weight times value is 2^(s - m + ve - its exponent): `heavy` is the largest
            // s - m - (exponent - vu) that the column sees, `roof` the ve up to which its weight stays within 2^15.
            float heavy = top - m;
            if (info & OWN_V) {
                heavy = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; i++) heavy = fmaxf(heavy, fmaf(st[i], cs, (float)dv[i]));
                const Two x = halves(heavy);
                heavy = fmaxf(x.a, x.b) - m;
            }
            // (below: zeros only, nothing, or weights that are)
            const bool some = !(info & NO_V) && heavy > -kZero / 2;
            const int roof = vu + 4 - (int)ceilf(fmaxf(heavy, -(float)kZero));
            // The sums move to a smaller unit when weights would pass 2^15, to a larger one when what there is to add
            // (for values of one size: the values) gets smaller by more than 2^8, but stay within 2^64 of the largest that
            // they hold; less than that, weights shrink.
            const bool first = least >= kNone;
            least = some ? min(least, roof) : least;
            const int up = info & OWN_V ? roof - 4 : vu;
            const int to = !some ? ve : first ? up : roof < ve ? roof - 4 : up > ve + 8 ? min(up, least + 64) : ve;
            if (__any(to != ve)) {
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[d][i] = ldexpf(o[d][i], to - ve);
                ve = to;
            }
            // (below 2^-100 weights are nothing)
            c = some && !(info & OWN_V) ? max(ve - vu, -100) : 0;
        }
        const float ref = m == -INFINITY ? 0.0f : m - 11.0f - (float)c;
        float e[16], sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 16; i++) {
            e[i] = __builtin_amdgcn_exp2f(fmaf(st[i], cs, -ref));
            sum[i & 1] += e[i];
        }
        l += P == 2 ? ldexpf(sum[0] + sum[1], -c) : sum[0] + sum[1];
        if constexpr (P == 2) {
            if (info & OWN_V) {
#pragma unroll
                for (int i = 0; i < 16; i++) e[i] = ldexpf(e[i], dv[i] + (ve - vu));
            }
        }
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int j = 0; j < 8; j += 2) split_pair(e[8 * t + j], e[8 * t + j + 1], minus1, ph[t], pl[t], j);
    };
    auto sums = [&](int it) {
        const h8* vp = (const h8*)(lds + 2 * KB + (it & 1) * VB) + lane;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int d0 = 0; d0 < DB; d0 += 2) {
                h8 vh[2];
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    vh[d] = vp[(2 * (d0 + d) + t) * 64];
                    o[d0 + d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh[d], ph[t], o[d0 + d], 0, 0, 0);
                }
#pragma unroll
                for (int d = 0; d < 2; d++) o[d0 + d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vh[d], pl[t], o[d0 + d], 0, 0, 0);
                if constexpr (P == 2) {
#pragma unroll
                    for (int d = 0; d < 2; d++)
                        o[d0 + d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vp[(2 * (d0 + d) + t) * 64 + PL / 16], ph[t], o[d0 + d], 0, 0, 0);
                }
            }
    };
    // Phases of the workgroup, by number: the wavefronts in front have weights(i) in 2 i and
    // products(i) in 2 i + 1, those behind one later.  In 2 i + 1 nobody uses the keys of unit i or
    // the values of unit i - 1 any more: those behind load over them, and wait at the end
    // of 2 i + 2, before the ones in front need what came.  Without any behind, all do so in
    // weights(i) and at the end of products(i); the first scores are then a phase of their own, because
    // the loads of weights(0) go over their keys, and its end is where the values of unit 0 have come.
    if (n > 0) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LD + HB / 256) : "memory");
        open(0);
        if (!skips(0)) {
            scores(0);
            powers(0);
        }
        if (NW == 4 || behind) phase_end(true);
        for (int it = 0; it < n; it++) {
            if (loads) fetch(it);
            const bool on = !skips(it);
            if (on) weights(it);
            else ph[0] = ph[1] = pl[0] = pl[1] = h8{};
            phase_end(false);
            __builtin_amdgcn_s_setprio(1);
            const bool next = it + 1 < n && !skips(it + 1);
            if (it + 1 < n) open(it + 1);
            if (on || next) {  // (in one piece, so that the second's reads of LDS go beside the first's products)
                sums(it);
                scores(it + 1);
                // operands are read AHEAD of their products: a read takes longer than the two products that
                // the compiler would leave it.  (The order is that of P + 1 products for the P planes of an operand; the
                // second look at the keys' hi planes is left to the compiler.  us, 2048 rows of 32x8x128, of 16x2x256: no
                // order 159, 213, this one 149, 198, one that counts the second look 149, 227.)
                constexpr int AHEAD = 8, NG = KS + 2 * DB;  // reads; operands
                __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
                for (int i = 0; i < NG - AHEAD / P; i++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, P + 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, P, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, (P + 1) * (AHEAD / P), 0);
            }
            if (next) powers(it + 1);
            __builtin_amdgcn_s_setprio(0);
            phase_end(loads);
        }
        if (NW == 8 && !behind) phase_end(false);
    }
    const Two lh = halves(l);
    l = lh.a + lh.b;
    if (!live) return;
    if (bad & BAD_V) {
        // infinities and NaN among the values are zero in the planes: here they come, to the rows that see them
        for (int u = u0; u < u1; u++) {
            if (!(*(const uint32_t*)(units + (u - u0) * stride + Head<HD>::info) & BAD_V)) continue;
            for (int at = max(u * kUnit, beg); at < min((u + 1) * kUnit, end); at++) {
                const T* vr = (const T*)p.v + (ks.a + at) * p.ldv + (int64_t)kvh * HD + 4 * h;
#pragma unroll
                for (int d = 0; d < DB; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float v = (float)vr[32 * d + 8 * (i / 4) + i % 4];
                        if (!finite(v)) o[d][i] += v;
                    }
            }
        }
    }
    const float inv = 1.0f / l;
    const bool none = end <= beg;
    float* part = a.part + (((qs.a + qi) * p.n_head + head) * a.splits + split) * (HD + 4);
    const bool whole = a.splits == 1, empty = whole ? none : m == -INFINITY && l == 0.0f;
    // the row's result, or this part's weighted mean with its maximum and its sum
    float* out = (whole ? p.out + (qs.a + qi) * p.ldo + (int64_t)head * HD : part) + 4 * h;
#pragma unroll
    for (int d = 0; d < DB; d++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            float4 r;
            r.x = empty ? 0.0f : ldexpf(o[d][i] * inv, -ve);
            r.y = empty ? 0.0f : ldexpf(o[d][i + 1] * inv, -ve);
            r.z = empty ? 0.0f : ldexpf(o[d][i + 2] * inv, -ve);
            r.w = empty ? 0.0f : ldexpf(o[d][i + 3] * inv, -ve);
            *(float4*)(out + 32 * d + 2 * i) = r;
        }
    if (!whole && h == 0) { part[HD] = m; part[HD + 1] = l; }
}

// The parts of one row's head, in their order: a wavefront each, HD / 64 values a lane.
template <int HD> __global__ __launch_bounds__(256) void attn_join_kernel(PromptArgs a) {
    constexpr int DPL = HD / 64;
    const ggq_attention_prompt_params& p = a.p;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int row = (int)(w / p.n_head), head = (int)(w % p.n_head), lane = threadIdx.x & 63;
    if (row >= p.n_rows) return;
    bool in = false;  // a row of some sequence
    for (int i = 0; i < p.n_seq && !in; i += 64) {
        const int j = i + lane;
        in = __any(j < p.n_seq && p.q_off[j] <= row && row < p.q_off[j + 1]);
    }
    if (!in) return;
    const float* q = a.part + w * a.splits * (HD + 4);
    float mx = -INFINITY;
    for (int i = 0; i < a.splits; i++) mx = fmaxf(mx, q[(int64_t)i * (HD + 4) + HD]);
    float ls = 0.0f, os[DPL] = {};
    for (int i = 0; i < a.splits; i++) {
        const float* x = q + (int64_t)i * (HD + 4);
        const float wt = x[HD] == -INFINITY && x[HD + 1] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(x[HD] - mx) * x[HD + 1];
        ls += wt;
#pragma unroll
        for (int d = 0; d < DPL; d++) os[d] = fmaf(x[lane + 64 * d], wt, os[d]);
    }
    float* out = p.out + (int64_t)row * p.ldo + (int64_t)head * HD + lane;
#pragma unroll
    for (int d = 0; d < DPL; d++) out[64 * d] = mx == -INFINITY && ls == 0.0f ? 0.0f : os[d] / ls;
}

}  // namespace

namespace {
int64_t units_of(const ggq_attention_prompt_params& p) { return (int64_t)p.n_kv_rows / kUnit + p.n_seq; }
int64_t tiles_of(const ggq_attention_prompt_params& p) {
    const int nc = (p.head_dim == 256 ? 4 : 8) * 32;
    return (int64_t)p.n_rows * (p.n_head / p.n_kv_head) / nc + p.n_seq;
}
// Planes of one kv head, and how many heads' there are at a time: 256 MB of them, or
// one head's.
size_t head_bytes(const ggq_attention_prompt_params& p) {
    const int planes = p.type == GGQ_TYPE_F32 ? 2 : 1;
    return (size_t)units_of(p) *
           (p.head_dim == 64 ? unit_bytes<64>(planes) : p.head_dim == 128 ? unit_bytes<128>(planes) : unit_bytes<256>(planes));
}
int heads_at_once(const ggq_attention_prompt_params& p) {
    return (int)std::max<size_t>(1, std::min<size_t>((size_t)p.n_kv_head, (size_t(256) << 20) / head_bytes(p)));
}
size_t planes_bytes(const ggq_attention_prompt_params& p) { return (head_bytes(p) * heads_at_once(p) + 255) / 256 * 256; }
}  // namespace

AttnPromptPlan attn_prompt_plan(const ggq_attention_prompt_params& p) {
    AttnPromptPlan pl{};
    // The VALU's one launch up to 2^27 products of rows, heads, keys and values, while a wavefront
    // does not go through the keys too often (us, few -> matrix cores; fp32, heads x kv heads x width):
    //   19 rows: 32x8x64 6.0 -> 11.0, 16x2x256 8.5 -> 23.3; 128 rows: 32x8x128 16.5 -> 24.7
    //   256 rows: 32x8x64 20.3 -> 22.0, 32x8x128 (2^28) 39.3 -> 30.0; 40 prompts of 150 rows,
    //   8x8x64 (2^28.8) 94 -> 43; 512 rows 4x1x128 21.0 -> 29.8; 1000 rows 2x1x64 31.1 -> 26.2
    //   one row: 501 keys 32x8x128 20.5 -> 22.7, 2001 keys 67 -> 37
    // Lengths are known as a mean only: one long sequence among short ones is taken like them (63 rows of 5
    // keys with 4 rows of 20000, 32x8x128: 630 -> 1072).
    const char* env = getenv("GGQ_PROMPT_MFMA");
    const double keys = (double)p.n_kv_rows / p.n_seq;
    if (env && *env) pl.few = atoi(env) == 0;
    else pl.few = keys <= 640 && keys * p.n_rows * p.n_head * p.head_dim <= (double)(1 << 27) * 1.01;
    if (pl.few) return pl;
    // few tiles: the positions in parts of four units at least, where that saves a workgroup
    // more units than the join costs (us with 1, 2, 3, 4 parts; * the rule's: 512 rows 32x8x128 47, 42,
    // 40*, 39; 16x2x256 66, 52, 48*, 46; 5 packed prompts 12x2x128 f16 52, 48*, 60, 63; one row of 4001 keys
    // 225, 127, 94, 79, .., 48 with 16, 49 with 31*)
    const int64_t wgs = tiles_of(p) * p.n_kv_head, units = units_of(p) / p.n_seq;
    const int64_t n = std::min<int64_t>(cu_count() / wgs, units / 4);
    pl.splits = n > 1 && units * (n - 1) > 4 * n ? (int)n : 1;
    if (const char* e = getenv("GGQ_PROMPT_SPLITS"); e && atoi(e) > 0)
        pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(atoi(e), 256), units_of(p)));
    pl.ws_bytes = planes_bytes(p);
    if (pl.splits > 1) pl.ws_bytes += sizeof(float) * (size_t)p.n_rows * p.n_head * pl.splits * (p.head_dim + 4);
    return pl;
}

hipError_t launch_attn_prompt(const ggq_attention_prompt_params& p, const AttnPromptPlan& pl, void* ws, hipStream_t s) {
    PromptArgs a{};
    a.p = p;
    a.planes = (uint8_t*)ws;
    a.part = (float*)((char*)ws + planes_bytes(p));
    a.G = p.n_head / p.n_kv_head;
    a.splits = pl.splits;
    a.tiles = (int)tiles_of(p);
    const int at_once = heads_at_once(p);
#define L(HD_, T_)                                                                                                        \
    for (a.kv0 = 0; a.kv0 < p.n_kv_head; a.kv0 += at_once) {                                                              \
        a.kvn = std::min(at_once, p.n_kv_head - a.kv0);                                                                   \
        planes_kernel<HD_, T_><<<dim3((unsigned)units_of(p), (unsigned)a.kvn), 256, 0, s>>>(a);                           \
        attn_kernel<HD_, T_><<<dim3((unsigned)(a.tiles * (int64_t)a.kvn), (unsigned)pl.splits), waves_of<HD_>() * 64, 0, s>>>(a); \
    }                                                                                                                     \
    if (pl.splits > 1) attn_join_kernel<HD_><<<dim3((unsigned)(((int64_t)p.n_rows * p.n_head + 3) / 4)), 256, 0, s>>>(a)
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

hipError_t launch_attn_prompt_few(const ggq_attention_prompt_params& p, hipStream_t s) {
    PromptArgs a{};
    a.p = p;
    a.G = p.n_head / p.n_kv_head;
    a.splits = 1;
    a.tiles = (int)((int64_t)p.n_rows * a.G / kCols + p.n_seq);
    const dim3 grid((unsigned)(a.tiles * (int64_t)p.n_kv_head));
#define L(HD_)                                                                    \
    if (p.type == GGQ_TYPE_F32) attn_few_kernel<HD_, float><<<grid, 256, 0, s>>>(a); \
    else attn_few_kernel<HD_, _Float16><<<grid, 256, 0, s>>>(a)
    if (p.head_dim == 64) { L(64); }
    else if (p.head_dim == 128) { L(128); }
    else { L(256); }
#undef L
    return hipGetLastError();
}

}  // namespace ggq
