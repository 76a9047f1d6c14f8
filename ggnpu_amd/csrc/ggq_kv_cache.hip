// ggq_kv_cache.hip -- a layer's quantized KV cache: rows into its pages and
// back, and the attention of one token of each sequence over it.
//
// Formats (include/ggq.h): blocks of 32 values along a head share a power of
// two; codes are e2m1 (4 bits) or e4m3 (8 bits).  gfx950 converts both to
// bf16, f16 and fp32 with that scale in one instruction for two values, and the
// result is exact, because a code has at most 4 significant bits: no rounding
// happens between the cache and the matrix cores.  A scale byte of 255 gives
// an infinite scale operand, which the conversion turns into NaN.
#include <algorithm>
#include <cstdlib>

#include "ggq_attn.h"
#include "ggq_attn_device.h"
#include "ggq_launch.h"

namespace ggq {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float scale_of(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

// The address of a position's record and its place there.
struct Place {
    uint8_t* rec;  // null: there is none
    int p;         // 0..31
};
template <uint32_t RB>
__device__ __forceinline__ Place place_of(const ggq_kv_cache& c, const ggq_kv_seqs& q, int seq, int64_t pos, int head) {
    if (pos < 0 || pos >= (int64_t)q.table_len * c.page_len) return Place{nullptr, 0};
    const uint32_t at = (uint32_t)pos / (uint32_t)c.page_len, in = (uint32_t)pos - at * (uint32_t)c.page_len;
    const int32_t page = q.pages[(uint64_t)(uint32_t)seq * (uint32_t)q.table_len + at];
    if (page < 0 || page >= c.n_pages) return Place{nullptr, 0};
    // (fewer than 2^32 records: they have a kilobyte or more)
    const uint32_t r = ((uint32_t)page * (uint32_t)c.n_kv_head + (uint32_t)head) * ((uint32_t)c.page_len / kKvTile) + in / kKvTile;
    return Place{(uint8_t*)c.pages + (uint64_t)r * RB, (int)(in % kKvTile)};
}

// Rows to or from the pages.  A workgroup takes U times 2048 values of one kv
// head, K (z = 0) or V, a thread 8 consecutive ones of each of U rows; 4 threads share a
// block of 32.  The rows' sequences are found by all threads together: one
// strided look over row_off for the first row, a step forward for each
// sequence that ends among the rows (in LDS for up to 256).  A row's place is three dependent
// loads away (offsets and length, page, codes), so large calls have U = 4 of
// them in flight a thread.
template <int HD, int KB, int VB, bool VALUE, bool STORE, int U, typename T>
__device__ __forceinline__ void rows_body(const ggq_kv_cache& c, const ggq_kv_seqs& q, const KvRows& r) {
    constexpr int BITS = VALUE ? VB : KB;
    constexpr uint32_t RB = kKvTile * HD * (KB + VB) / 8 + 2 * HD;
    constexpr int kNear = 256;  // sequences whose offsets and lengths are looked up in LDS
    __shared__ int32_t s_off[kNear + 1], s_len[kNear];
    constexpr int RPW = 2048 / HD;  // rows of a workgroup's pass
    constexpr int TPR = HD / 8;     // threads of a row
    const int tid = threadIdx.x, head = blockIdx.y, d = tid % TPR * 8;
    const int row0 = blockIdx.x * RPW * U;
    int first = 0;
    const bool near = q.n_seq <= kNear;
    if (r.row_off) {
        for (int i = 0; i < q.n_seq; i += 256) {
            const int j = i + tid;
            int32_t o = 0, l = 0;
            if (j < q.n_seq) {
                o = r.row_off[j + 1];
                if (near) l = q.len[j];
            }
            if (near && j < q.n_seq) {
                s_off[j + 1] = o;
                s_len[j] = l;
                if (j == 0) s_off[0] = r.row_off[0];
            }
            first += __syncthreads_count(j < q.n_seq && o <= row0);
        }
    }
    Place pl[U];
    auto find = [&](auto off, auto len) {  // (apart for LDS and memory: one access for both would be a generic one)
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int row = row0 + i * RPW + tid / TPR;
            int64_t pos = -1;
            while (first < q.n_seq && off(first + 1) <= row) first++;
            if (row < r.n_rows && first < q.n_seq && row >= off(first)) pos = (int64_t)len(first) - off(first + 1) + row;
            pl[i] = pos >= 0 ? place_of<RB>(c, q, first, pos, head) : Place{nullptr, 0};
        }
    };
    if (!r.row_off) {
#pragma unroll
        for (int i = 0; i < U; i++) {
            const int row = row0 + i * RPW + tid / TPR;
            const bool in = row < r.n_rows && row < q.n_seq;
            pl[i] = in ? place_of<RB>(c, q, row, (int64_t)q.len[row] - 1, head) : Place{nullptr, 0};
        }
    } else if (near) {
        find([&](int i) { return s_off[i]; }, [&](int i) { return s_len[i]; });
    } else {
        find([&](int i) { return r.row_off[i]; }, [&](int i) { return q.len[i]; });
    }
    // codes of this thread: 8 in one run, or two runs of 4 (V of 64-wide heads)
    constexpr int RUN = VALUE && HD == 64 ? 4 : 8;
    auto at = [&](int p, int e) {  // byte offset of the code of value e at position p
        int lane, n;
        if (VALUE) {
            lane = 16 * (p % 16 / 4) + e / (HD / 16);
            n = (4 * (p / 16) + p % 4) * (HD / 16) + e % (HD / 16);
        } else {
            lane = 16 * (e / (HD / 4)) + p % 16;
            n = p / 16 * (HD / 4) + e % (HD / 4);
        }
        const int b = n * BITS / 8;
        return 1024 * (b / 16) + 16 * lane + b % 16;
    };
    const int blk = d / 32;
    auto codes_of = [&](const Place& x) { return x.rec + (VALUE ? kKvTile * HD * KB / 8 : 0); };
    auto scale_at = [&](const Place& x) {
        const int p = x.p;
        return x.rec + kKvTile * HD * (KB + VB) / 8 +
               (VALUE ? HD + (4 * blk + p % 16 / 4) * 8 + 4 * (p / 16) + p % 4 : (16 * blk + p % 16) * 2 + p / 16);
    };
    T* const row_base = (T*)(VALUE ? r.v : r.k) + (int64_t)(row0 + tid / TPR) * (VALUE ? r.ldv : r.ldk) + head * HD + d;
    auto row_at = [&](int i) { return row_base + (int64_t)(i * RPW) * (VALUE ? r.ldv : r.ldk); };
    struct alignas(16) Run { T x[16 / sizeof(T)]; };
    constexpr int NR = 8 * sizeof(T) / 16, PR = 16 / sizeof(T);  // 16-byte runs of 8 values
    if constexpr (STORE) {
        Run in[U][NR];
#pragma unroll
        for (int i = 0; i < U; i++)
#pragma unroll
            for (int j = 0; j < NR; j++) in[i][j] = pl[i].rec ? *((const Run*)row_at(i) + j) : Run{};
#pragma unroll
        for (int i = 0; i < U; i++) {
            float v[8];
            uint32_t m = 0;  // the largest magnitude's bits; infinities and NaN are the largest
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[j] = (float)in[i][j / PR].x[j % PR];
                m = max(m, __builtin_bit_cast(uint32_t, v[j]) & 0x7FFFFFFFu);
            }
            m = max(m, (uint32_t)__shfl_xor((int)m, 1, 64));
            m = max(m, (uint32_t)__shfl_xor((int)m, 2, 64));
            if (!pl[i].rec) continue;
            // smallest e with amax <= 1.75 * 2^(e + 2), or 1.8125 * 2^(e + 8)
            const int ex = (int)(m >> 23), over = (m & 0x7FFFFFu) > (BITS == 4 ? 0x600000u : 0x680000u);
            const bool bad = ex == 255;
            const int byte = bad ? 255 : max(1, ex - (BITS == 4 ? 2 : 8) + over);
            const float s = scale_of((uint32_t)byte);
            uint32_t w[2] = {0, 0};
            if (!bad) {
                if constexpr (BITS == 4) {
                    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], v[0], v[1], s, 0);
                    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], v[2], v[3], s, 1);
                    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], v[4], v[5], s, 2);
                    w[0] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w[0], v[6], v[7], s, 3);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        s16x2 o = {0, 0};
                        o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, v[4 * h], v[4 * h + 1], s, false);
                        o = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(o, v[4 * h + 2], v[4 * h + 3], s, true);
                        w[h] = __builtin_bit_cast(uint32_t, o);
                    }
                }
            }
            uint8_t* codes = codes_of(pl[i]);
            const int p = pl[i].p;
            if constexpr (BITS == 4 && RUN == 8) {
                *(uint32_t*)(codes + at(p, d)) = w[0];
            } else if constexpr (BITS == 4) {
                *(uint16_t*)(codes + at(p, d)) = (uint16_t)w[0];
                *(uint16_t*)(codes + at(p, d + 4)) = (uint16_t)(w[0] >> 16);
            } else if constexpr (RUN == 8) {
                *(uint2*)(codes + at(p, d)) = make_uint2(w[0], w[1]);
            } else {
                *(uint32_t*)(codes + at(p, d)) = w[0];
                *(uint32_t*)(codes + at(p, d + 4)) = w[1];
            }
            if (d % 32 == 0) *scale_at(pl[i]) = (uint8_t)byte;
        }
    } else {
        uint32_t w[U][2];
        uint8_t sb[U];
#pragma unroll
        for (int i = 0; i < U; i++) {
            if (!pl[i].rec) continue;
            const uint8_t* codes = codes_of(pl[i]);
            const int p = pl[i].p;
            sb[i] = *scale_at(pl[i]);
            if constexpr (BITS == 4 && RUN == 8) {
                w[i][0] = *(const uint32_t*)(codes + at(p, d));
            } else if constexpr (BITS == 4) {
                w[i][0] = *(const uint16_t*)(codes + at(p, d)) | (uint32_t)*(const uint16_t*)(codes + at(p, d + 4)) << 16;
            } else if constexpr (RUN == 8) {
                const uint2 x = *(const uint2*)(codes + at(p, d));
                w[i][0] = x.x;
                w[i][1] = x.y;
            } else {
                w[i][0] = *(const uint32_t*)(codes + at(p, d));
                w[i][1] = *(const uint32_t*)(codes + at(p, d + 4));
            }
        }
#pragma unroll
        for (int i = 0; i < U; i++) {
            if (!pl[i].rec) continue;
            const float s = scale_of(sb[i]);
            f32x2 o[4];
            if constexpr (BITS == 4) {
                o[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i][0], s, 0);
                o[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i][0], s, 1);
                o[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i][0], s, 2);
                o[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i][0], s, 3);
            } else {
                o[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i][0], s, false);
                o[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i][0], s, true);
                o[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i][1], s, false);
                o[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[i][1], s, true);
            }
#pragma unroll
            for (int j = 0; j < NR; j++) {
                Run out;
#pragma unroll
                for (int e = 0; e < PR; e++) out.x[e] = (T)o[(j * PR + e) / 2][e % 2];
                *((Run*)row_at(i) + j) = out;
            }
        }
    }
}

template <int HD, int KB, int VB, bool STORE, int U, typename T>
__global__ __launch_bounds__(256) void kv_rows_kernel(ggq_kv_cache c, ggq_kv_seqs q, KvRows r) {
    if (blockIdx.z == 0) rows_body<HD, KB, VB, false, STORE, U, T>(c, q, r);
    else rows_body<HD, KB, VB, true, STORE, U, T>(c, q, r);
}

template <int HD, int KB, int VB, int U, typename T>
void rows_go(const ggq_kv_cache& c, const ggq_kv_seqs& q, const KvRows& r, bool store, hipStream_t s) {
    const int per = U * 2048 / HD;
    const dim3 grid((unsigned)((r.n_rows + per - 1) / per), (unsigned)c.n_kv_head, 2);
    if (store) kv_rows_kernel<HD, KB, VB, true, U, T><<<grid, 256, 0, s>>>(c, q, r);
    else kv_rows_kernel<HD, KB, VB, false, U, T><<<grid, 256, 0, s>>>(c, q, r);
}

template <int HD, int KB, int VB> hipError_t rows_launch(const ggq_kv_cache& c, const ggq_kv_seqs& q, const KvRows& r,
                                                         bool store, hipStream_t s) {
    // four rows a thread once that leaves every CU two workgroups: their loads overlap (16 x 4001 fp16 rows of 2 heads of
    // 128 in 8 bits: load 30.2 us with one row, 18.6 with four, store 25.8 and 20.9); below that one row, for the shorter chain
    const bool many = (int64_t)r.n_rows * c.n_kv_head * HD * 2 / (4 * 2048) >= 2 * cu_count();
    if (r.type == GGQ_TYPE_F32) many ? rows_go<HD, KB, VB, 4, float>(c, q, r, store, s) : rows_go<HD, KB, VB, 1, float>(c, q, r, store, s);
    else many ? rows_go<HD, KB, VB, 4, _Float16>(c, q, r, store, s) : rows_go<HD, KB, VB, 1, _Float16>(c, q, r, store, s);
    return hipGetLastError();
}

}  // namespace

#define GGQ_BY_CACHE(HD_, F, ...)                                                                              \
    (c.k_type == GGQ_KV_MXFP4 ? (c.v_type == GGQ_KV_MXFP4 ? F<HD_, 4, 4>(__VA_ARGS__) : F<HD_, 4, 8>(__VA_ARGS__)) \
                              : (c.v_type == GGQ_KV_MXFP4 ? F<HD_, 8, 4>(__VA_ARGS__) : F<HD_, 8, 8>(__VA_ARGS__)))

hipError_t launch_kv_rows(const ggq_kv_cache& c, const ggq_kv_seqs& q, const KvRows& r, bool store, hipStream_t s) {
    if (c.head_dim == 64) return GGQ_BY_CACHE(64, rows_launch, c, q, r, store, s);
    if (c.head_dim == 128) return GGQ_BY_CACHE(128, rows_launch, c, q, r, store, s);
    return GGQ_BY_CACHE(256, rows_launch, c, q, r, store, s);
}

// ================================================================ attention
// One token of each sequence over the pages of its cache.
//
// Per 32 positions (one record) a wavefront computes, on bf16 matrix cores with
// exact operands,
//   S^T[position][column] = sum_d K[position][d] Qc[d][column]
//   O^T[d][column]       += sum_position V[position][d] P[position][column]
// A column is one of three bf16 parts of a query head (x = x0 + x1 + x2 holds
// all 24 bits); the fourth of a head's four columns is zero.  A head's
// scores are the sum of its four columns, four neighbouring lanes.  Each of them then
// makes its own part of the weight exp2(s - m), and the parts of O^T are added at the end.
//   The positions of S^T's rows in a lane are the ones that O^T's product wants
// of that lane (the record's V order is made for that), so scores become
// weights without leaving their registers.  K operands are the record's K
// bytes as they are loaded; V operands take one v_perm a pair of positions on top.
//   The maximum moves only when a record exceeds it by more than 8 (in powers of
// two): the weights stay below 2^8 and the sum below 2^8 * positions, and the
// accumulators are rescaled a few times a sequence.
// A workgroup has 8 wavefronts (4 where their registers allow no more) that take the records of its part of the
// positions in turn and add up in LDS; kv_join_kernel adds up the parts.
// Bound: HBM with 128-wide heads (64 sequences of up to 8191 positions, K in 8
// and V in 4 bits: 566 MB in 103 us, 5.5 TB/s); with 64-wide ones the VALU, whose
// work on scores does not shrink with the head (131001 positions: 238
// instructions a record, 71 MB in 21 us and 4 us for the join).
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

union Frag {
    uint32_t w[4];
    bf16x8 v;
};

__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float s, int b) {
    bf16x2 r;
    switch (b) {  // the byte is an immediate
    case 0: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0); break;
    case 1: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1); break;
    case 2: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2); break;
    default: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3); break;
    }
    return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, float s, int half) {
    const bf16x2 r = half ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, true)
                          : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, false);
    return __builtin_bit_cast(uint32_t, r);
}
// Values 2i and 2i + 1 of a run of codes.
template <int BITS> __device__ __forceinline__ uint32_t pair_of(const uint32_t* w, float s, int i) {
    if constexpr (BITS == 4) return fp4_pair(w[i / 4], s, i % 4);
    else return fp8_pair(w[i / 2], s, i % 2);
}

template <int CTRL> __device__ __forceinline__ float quad_perm(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}
__device__ __forceinline__ float quad_sum(float v) {
    v += quad_perm<0xB1>(v);  // lanes 1 0 3 2
    return v + quad_perm<0x4E>(v);  // lanes 2 3 0 1
}
// Over the four groups of 16 lanes.
__device__ __forceinline__ float rows_max(float v) {
    const Two x = rows16(v), y = halves(max3(x.a, x.b, x.b));
    return max3(y.a, y.b, y.b);
}

// A part of x, its upper 16 bits: three cuts of 8 bits each hold all 24, x0 = x
// cut, x1 = (x - x0) cut, x2 = x - x0 - x1.  A lane's part is chosen by its masks:
// what they cut off is subtracted (everything for the column that is zero).
struct Cuts {
    uint32_t a, b;
};
__device__ __forceinline__ Cuts cuts_of(int part) {
    return Cuts{part == 0 ? 0u : part == 3 ? 0xFFFFFFFFu : 0xFFFF0000u, part == 2 ? 0xFFFF0000u : 0u};
}
__device__ __forceinline__ float bf16_part(float x, Cuts c) {
    x -= __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & c.a);
    return x - __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & c.b);
}
__device__ __forceinline__ uint32_t bf16_pack(float a, float b) {  // upper halves
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}

// Wavefronts of a workgroup, by their registers.
template <int HD, int NT> constexpr int kv_waves() { return HD == 256 ? 4 : 8; }

template <int HD, int KB, int VB, int NT>
__global__ __launch_bounds__((kv_waves<HD, NT>() * 64)) void kv_attn_kernel(KvAttnArgs a, int splits, float* part) {
    constexpr int NW = kv_waves<HD, NT>();
    constexpr int KW = HD * KB / 64, VW = HD * VB / 64;  // dwords of a lane's K and V codes
    constexpr int NS = HD / 32;                          // k steps of S^T, blocks of a head
    constexpr int NO = HD / 16;                          // row tiles of O^T
    constexpr int VD = HD / 16;                          // values of a lane's V at one position
    constexpr int64_t RB = kKvTile * HD * (KB + VB) / 8 + 2 * HD;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, r = lane & 15;
    const int kvh = blockIdx.y % a.c.n_kv_head, hz = blockIdx.y / a.c.n_kv_head * 4 * NT, seq = blockIdx.z;
    const int split = blockIdx.x;
    const int G = a.n_head / a.c.n_kv_head;  // query heads of this kv head
    const int tpp = a.c.page_len / kKvTile;
    int64_t hi = a.q.len[seq];
    hi = min(hi, (int64_t)a.q.max_len);
    hi = min(hi, (int64_t)a.q.table_len * a.c.page_len);
    int64_t lo = a.window > 0 ? (int64_t)a.q.len[seq] - a.window : 0;
    if (lo < 0) lo = 0;
    const int t0 = (int)(lo / kKvTile), t1 = hi > lo ? (int)((hi + kKvTile - 1) / kKvTile) : t0;
    int per = (t1 - t0 + splits - 1) / splits;
    if (per > NW) per = (per + NW - 1) / NW * NW;
    const int first = t0 + split * per, last = min(t1, first + per);

    // columns: query heads hz + 4 n + r / 4, part r % 4
    const int part_i = r & 3;
    const Cuts cut = cuts_of(part_i);
    bf16x8 qf[NT][NS];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int h = hz + 4 * n + (r >> 2);
        const float* qp = a.Q + (int64_t)seq * a.ldq + (int64_t)(kvh * G + (h < G ? h : 0)) * HD + g * (HD / 4);
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const float4 u = *(const float4*)(qp + 8 * s), v = *(const float4*)(qp + 8 * s + 4);
            const float x[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
            Frag f;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float c0 = h < G ? x[2 * i] * a.scale : 0.0f, c1 = h < G ? x[2 * i + 1] * a.scale : 0.0f;
                f.w[i] = bf16_pack(bf16_part(c0, cut), bf16_part(c1, cut));
            }
            qf[n][s] = f.v;
        }
    }
    f32x4 o[NT][NO];
    float m[NT], l[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
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
    auto load = [&](int it, Rec& x) {
        const int page = __builtin_amdgcn_readlane(pages, it & 63);
        x.there = page >= 0;
        if (!x.there) return;
        const int t = first + wave + NW * it;
        const uint8_t* rec = (const uint8_t*)a.c.pages +
                             (((int64_t)page * a.c.n_kv_head + kvh) * tpp + t % tpp) * RB;
#pragma unroll
        for (int i = 0; i < KW; i += 4) {
            const uint4 v = *(const uint4*)(rec + 256 * i + 16 * lane);
            x.k[i] = v.x; x.k[i + 1] = v.y; x.k[i + 2] = v.z; x.k[i + 3] = v.w;
        }
        rec += kKvTile * HD * KB / 8;
#pragma unroll
        for (int i = 0; i < VW; i += 4) {
            const uint4 v = *(const uint4*)(rec + 256 * i + 16 * lane);
            x.v[i] = v.x; x.v[i + 1] = v.y; x.v[i + 2] = v.z; x.v[i + 3] = v.w;
        }
        rec += kKvTile * HD * VB / 8;
        // K scales: a lane's quarter of the head lies in block g * NS / 4 (and the next one of 256-wide heads)
        if constexpr (NS <= 4) x.ks[0] = *(const uint16_t*)(rec + (16 * (g * NS / 4) + r) * 2);
        else {
            x.ks[0] = *(const uint16_t*)(rec + (16 * (2 * g) + r) * 2);
            x.ks[1] = *(const uint16_t*)(rec + (16 * (2 * g + 1) + r) * 2);
        }
        x.vs = *(const uint2*)(rec + HD + (4 * (r * VD / 32) + g) * 8);
    };
    auto compute = [&](int it, Rec& x) {
        if (!x.there) return;
        const int64_t base = (int64_t)(first + wave + NW * it) * kKvTile;
        const bool partial = base < lo || base + kKvTile > hi;
        // scores
        f32x4 st[2][NT];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int n = 0; n < NT; n++) st[t][n] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const int blk = NS <= 4 ? 0 : s / 4;  // (256-wide: 64 values of a lane, two blocks)
                const float sc = scale_of((x.ks[blk] >> (8 * t)) & 255u);
                Frag f;
#pragma unroll
                for (int i = 0; i < 4; i++) f.w[i] = pair_of<KB>(x.k + (t * (HD / 4) + 8 * s) * KB / 32, sc, i);
#pragma unroll
                for (int n = 0; n < NT; n++)
                    st[t][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.v, qf[n][s], st[t][n], 0, 0, 0);
            }
        if (partial) {
            // codes of positions that are not seen: zero, with a finite scale
            uint32_t keep[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int64_t pos = base + 16 * (j / 4) + 4 * g + j % 4;
                keep[j] = pos >= lo && pos < hi ? 0xFFFFFFFFu : 0u;
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
        }
        Frag pf[NT];
        bool move = false;
        float sv[NT][8], top[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float v = quad_sum(st[j / 4][n][j % 4]);
                if (partial) {
                    const int64_t pos = base + 16 * (j / 4) + 4 * g + j % 4;
                    if (pos < lo || pos >= hi) v = -INFINITY;
                }
                sv[n][j] = v;
            }
            const float* x = sv[n];
            top[n] = rows_max(max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], x[7])));
            move |= top[n] > m[n] + 8.0f;
        }
        if (__any(move)) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const float mn = max3(m[n], top[n], top[n]);
                const float al = __builtin_amdgcn_exp2f(m[n] - (mn == -INFINITY ? 0.0f : mn));
                m[n] = mn;
                l[n] *= al;
#pragma unroll
                for (int i = 0; i < NO; i++) o[n][i] *= al;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const float mm = m[n] == -INFINITY ? 0.0f : m[n];
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float e = __builtin_amdgcn_exp2f(sv[n][j] - mm);
                l[n] += e;
                w[j] = bf16_part(e, cut);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) pf[n].w[j] = bf16_pack(w[2 * j], w[2 * j + 1]);
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
            Frag f0, f1;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                f0.w[j] = __builtin_amdgcn_perm(c[2 * j + 1], c[2 * j], 0x05040100u);
                f1.w[j] = __builtin_amdgcn_perm(c[2 * j + 1], c[2 * j], 0x07060302u);
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                o[n][2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f0.v, pf[n].v, o[n][2 * i], 0, 0, 0);
                o[n][2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f1.v, pf[n].v, o[n][2 * i + 1], 0, 0, 0);
            }
        }
    };
    Rec cur, nxt;
    look(0);
    if (n_it > 0) load(0, cur);
    for (int it = 0; it < n_it; it++) {
        if (it + 1 < n_it) {
            if (((it + 1) & 63) == 0) look(it + 1);
            load(it + 1, nxt);
        }
        compute(it, cur);
        cur = nxt;
    }

    // the wavefronts' parts
    __shared__ float sm[NW][4 * NT], sl[NW][4 * NT], so[NW][4 * NT][HD];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        float s = l[n];  // of this group's positions; the quad's four lanes hold the same
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        const int h = 4 * n + (r >> 2);
        if (g == 0 && part_i == 0) { sm[wave][h] = m[n]; sl[wave][h] = s; }
#pragma unroll
        for (int i = 0; i < NO; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float v = quad_sum(o[n][i][e]);
                if (part_i == 0) so[wave][h][(4 * g + e) * VD + i] = v;
            }
    }
    __syncthreads();
    for (int e = tid; e < 4 * NT * HD; e += NW * 64) {
        const int h = e / HD, d = e % HD;
        if (hz + h >= G) break;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; w++) mx = fmaxf(mx, sm[w][h]);
        float ls = 0.0f, os = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float al = sm[w][h] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[w][h] - mx);
            ls = fmaf(sl[w][h], al, ls);
            os = fmaf(so[w][h][d], al, os);
        }
        const int head = kvh * G + hz + h;
        if (splits == 1) {
            // no position at all: zeros (a NaN keeps its way through the sum)
            a.out[(int64_t)seq * a.ldo + (int64_t)head * HD + d] = ls == 0.0f && mx == -INFINITY ? 0.0f : os / ls;
        } else {
            float* po = part + (((int64_t)seq * a.n_head + head) * splits + split) * (HD + 2);
            po[d] = os;
            if (d == 0) { po[HD] = mx; po[HD + 1] = ls; }
        }
    }
}

// The parts of one head: their weights first, then a thread a value and group of parts,
// in an order that does not depend on timing.
constexpr int kKvMaxSplits = 256;
template <int HD> __global__ __launch_bounds__(512) void kv_join_kernel(KvAttnArgs a, int splits, const float* part) {
    constexpr int NG = 512 / HD, B = 8;
    __shared__ float w[kKvMaxSplits], red[8], go[NG][HD];
    const int head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, d = tid % HD, grp = tid / HD;
    const float* po = part + ((int64_t)seq * a.n_head + head) * splits * (HD + 2);
    const float2 ml = tid < splits ? *(const float2*)(po + (int64_t)tid * (HD + 2) + HD) : make_float2(-INFINITY, 0.0f);
    float mx = ml.x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    if ((tid & 63) == 0) red[tid >> 6] = mx;
    __syncthreads();
    mx = red[0];
#pragma unroll
    for (int i = 1; i < 8; i++) mx = fmaxf(mx, red[i]);
    const float wt = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mx);
    if (tid < splits) w[tid] = wt;
    float ls = wt * ml.y;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ls += __shfl_xor(ls, o, 64);
    __syncthreads();
    if ((tid & 63) == 0) red[tid >> 6] = ls;
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
    ls = red[0];
#pragma unroll
    for (int i = 1; i < 8; i++) ls += red[i];
#pragma unroll
    for (int i = 1; i < NG; i++) os += go[i][d];
    a.out[(int64_t)seq * a.ldo + (int64_t)head * HD + d] = ls == 0.0f && mx == -INFINITY ? 0.0f : os / ls;
}

// Workgroups that the chip holds at once.
template <int HD, int KB, int VB, int NT> int64_t resident() {
    static const int64_t n = [] {
        int r = 0;
        if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&r, (const void*)kv_attn_kernel<HD, KB, VB, NT>, kv_waves<HD, NT>() * 64, 0) != hipSuccess || r < 1)
            r = 1;
        return (int64_t)r * cu_count();
    }();
    return n;
}

// One round of workgroups at most, four records in a part at least; and only where
// the rounds of records that it saves a wavefront are worth the join (in us, one sequence,
// 8 kv heads of 128 in 4 bits: 500 positions 7.3 with one part, 8.1 with 4; 1000: 9.8,
// 8.3 with 8; 4000: 25.0, 8.7 with 32; 16 sequences of 1000: 9.9, 10.7 with 2; of 6000: 38, 27).
template <int HD, int KB, int VB> int attn_splits(const KvAttnArgs& a, int64_t records) {
    const int G = a.n_head / a.c.n_kv_head, NW = G <= 4 ? kv_waves<HD, 1>() : kv_waves<HD, 2>();
    const int64_t wgs = (int64_t)a.q.n_seq * a.c.n_kv_head * ((G + 7) / 8);
    const int64_t fit = G <= 4 ? resident<HD, KB, VB, 1>() : resident<HD, KB, VB, 2>();
    const int64_t n = std::min<int64_t>(fit / wgs, (records + 3) / 4);
    return n > 1 && records * (n - 1) > 3 * NW * n ? (int)std::min<int64_t>(n, kKvMaxSplits) : 1;
}

template <int HD, int KB, int VB> hipError_t attn_launch(const KvAttnArgs& a, int splits, float* ws, hipStream_t s) {
    const int G = a.n_head / a.c.n_kv_head;
    const dim3 grid((unsigned)splits, (unsigned)(a.c.n_kv_head * ((G + 7) / 8)), (unsigned)a.q.n_seq);
    if (G <= 4) kv_attn_kernel<HD, KB, VB, 1><<<grid, kv_waves<HD, 1>() * 64, 0, s>>>(a, splits, ws);
    else kv_attn_kernel<HD, KB, VB, 2><<<grid, kv_waves<HD, 2>() * 64, 0, s>>>(a, splits, ws);
    if (splits > 1) kv_join_kernel<HD><<<dim3((unsigned)a.n_head, (unsigned)a.q.n_seq), 512, 0, s>>>(a, splits, ws);
    return hipGetLastError();
}

}  // namespace

int kv_attn_splits(const KvAttnArgs& a) {
    const ggq_kv_cache& c = a.c;
    int64_t span = std::min<int64_t>(a.q.max_len, (int64_t)a.q.table_len * c.page_len);
    if (a.window > 0) span = std::min<int64_t>(span, (int64_t)a.window + kKvTile);
    const int64_t records = (span + kKvTile - 1) / kKvTile;
    if (const char* e = getenv("GGQ_KV_SPLITS"); e && atoi(e) > 0)
        return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(atoi(e), kKvMaxSplits), records));
    if (c.head_dim == 64) return GGQ_BY_CACHE(64, attn_splits, a, records);
    if (c.head_dim == 128) return GGQ_BY_CACHE(128, attn_splits, a, records);
    return GGQ_BY_CACHE(256, attn_splits, a, records);
}

size_t kv_attn_ws_floats(const KvAttnArgs& a, int splits) {
    return splits <= 1 ? 0 : (size_t)a.q.n_seq * a.n_head * splits * (a.c.head_dim + 2);
}

hipError_t launch_kv_attn(const KvAttnArgs& a, int splits, float* ws, hipStream_t s) {
    const ggq_kv_cache& c = a.c;
    if (c.head_dim == 64) return GGQ_BY_CACHE(64, attn_launch, a, splits, ws, s);
    if (c.head_dim == 128) return GGQ_BY_CACHE(128, attn_launch, a, splits, ws, s);
    return GGQ_BY_CACHE(256, attn_launch, a, splits, ws, s);
}
#undef GGQ_BY_CACHE

}  // namespace ggq
