// ggq_norm.hip -- what stands between two layers' matmuls: the residual's
// addition, RMSNorm of rows or of their heads, a SiLU gate, and the int8 codes
// that the next matmul reads (ggq_norm_dev).
//
// A workgroup holds one row in registers, R runs of four values a thread, so
// each input is read once and nothing is written that the caller did not ask
// for.  Values are made in 64 bits from the fp32 sum on and rounded once: the
// order of the square sum then does not show in the codes, whose borders an fp32
// last bit would move values across.  gfx950 has fp64 FMAs at the rate of
// single fp32 ones, and a row is a few of them a value.
// Bound: HBM (measured figures at launch_norm below).
#include <algorithm>

#include "ggq_device.h"
#include "ggq_steps.h"

namespace ggq {
namespace {

struct NormArgs {
    ggq_norm_params p;
    int len;    // values that are normalised together
    int lanes;  // a group's lanes where it is a power of two of up to a wavefront's (reduced by shuffles), else 0
};

// Over neighbouring lanes (a power of two of them), by data-parallel moves: pairs, quads, halves and rows of 16 turned round, then
// rows and halves swapped.  All lanes get the result.
template <int CTRL, typename T> __device__ __forceinline__ T turned(T v) {
    constexpr int W = sizeof(T) / 4;
    struct Words { int w[W]; } x = __builtin_bit_cast(Words, v);
#pragma unroll
    for (int i = 0; i < W; i++) x.w[i] = __builtin_amdgcn_update_dpp(0, x.w[i], CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(T, x);
}
template <bool HALVES, typename T, typename F> __device__ __forceinline__ T swapped(T v, F f) {
    constexpr int W = sizeof(T) / 4;
    struct Words { uint32_t w[W]; } x = __builtin_bit_cast(Words, v), y = x;
#pragma unroll
    for (int i = 0; i < W; i++) {
        const auto r = HALVES ? __builtin_amdgcn_permlane32_swap(x.w[i], x.w[i], false, false)
                              : __builtin_amdgcn_permlane16_swap(x.w[i], x.w[i], false, false);
        x.w[i] = r[0];
        y.w[i] = r[1];
    }
    return f(__builtin_bit_cast(T, x), __builtin_bit_cast(T, y));
}
template <typename T, typename F> __device__ __forceinline__ T lanes_reduce(T v, int lanes, F f) {
    if (lanes > 1) v = f(v, turned<0xB1>(v));
    if (lanes > 2) v = f(v, turned<0x4E>(v));
    if (lanes > 4) v = f(v, turned<0x141>(v));
    if (lanes > 8) v = f(v, turned<0x140>(v));
    if (lanes > 16) v = swapped<false>(v, f);
    if (lanes > 32) v = swapped<true>(v, f);
    return v;
}

template <int TPB, typename T, typename F> __device__ __forceinline__ T wg_reduce(T v, T* red, F f) {
    v = lanes_reduce(v, 64, f);
    if constexpr (TPB > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < TPB / 64; i++) v = f(v, red[i]);
    }
    return v;
}

// (a row's values may all be so small that the reciprocal of its step is infinite: zeros stay zeros there)
__device__ __forceinline__ uint32_t code_of(float y, float inv) { return (uint32_t)(uint8_t)to_i8(y == 0.0f ? 0.0f : __fmul_rn(y, inv)); }
__device__ __forceinline__ uint32_t codes_of(const float4& y, float inv) {
    return code_of(y.x, inv) | code_of(y.y, inv) << 8 | code_of(y.z, inv) << 16 | code_of(y.w, inv) << 24;
}
__device__ __forceinline__ float step_of(float amax) { return amax > 0.0f ? __fdiv_rn(amax, 127.0f) : 1.0f; }
// z / (1 + exp(-z)) within 2^-44, in half the instructions of the library's exp and division: a row's gate is most of its
// arithmetic.  exp(x) = 2^n exp(r) with |r| <= ln(2) / 2, eleven terms (the next one is 2^-47 of the sum); a reciprocal and one step of Newton's.
// (Beyond 700 the result is 0 after rounding to fp32, and the quotient of infinities NaN as it is.)
__device__ __forceinline__ double silu64(float z) {
    const double x = fmin(fmax(-(double)z, -700.0), 700.0), n = rint(x * 1.44269504088896340736);
    const double r = fma(n, -1.6465949582897082e-12, fma(n, -0.6931471805582987, x));
    double e = 1.0 / 39916800.0;
    e = fma(e, r, 1.0 / 3628800.0);
    e = fma(e, r, 1.0 / 362880.0);
    e = fma(e, r, 1.0 / 40320.0);
    e = fma(e, r, 1.0 / 5040.0);
    e = fma(e, r, 1.0 / 720.0);
    e = fma(e, r, 1.0 / 120.0);
    e = fma(e, r, 1.0 / 24.0);
    e = fma(e, r, 1.0 / 6.0);
    e = fma(e, r, 0.5);
    e = fma(e, r, 1.0);
    e = fma(e, r, 1.0);
    const double d = 1.0 + ldexp(e, (int)n);
    double q = __builtin_amdgcn_rcp(d);
    q = fma(q, fma(-d, q, 1.0), q);
    return (double)(z == -INFINITY ? __builtin_nanf("") : z) * q;
}

// 1 / sqrt(x) to 2^-50: the reciprocal root and two steps of Newton's (of 0: infinity, of infinity: 0).
__device__ __forceinline__ double one_over_root(double x) {
    double q = __builtin_amdgcn_rsq(x);
    if (!(x > 0.0 && x < INFINITY)) return q;
#pragma unroll
    for (int i = 0; i < 2; i++) q = fma(0.5 * q, fma(-x * q, q, 1.0), q);
    return q;
}

template <int TPB, int R>
__global__ __launch_bounds__(TPB) void norm_kernel(NormArgs a) {
    __shared__ double red[TPB / 64];
    __shared__ float redf[TPB / 64];
    extern __shared__ double parts[];  // a square sum a run, where groups are neither the row nor a power of two of lanes
    const ggq_norm_params& p = a.p;
    const int64_t m = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (m >= a.p.n_rows) return;
    const int tid = threadIdx.x, K = p.n_cols;
    const float* xr = p.x + m * p.ldx;
    // (the longest rows fill the registers: their gate is read where it is used)
    constexpr int NG = R > 4 ? 1 : R;
    float4 v[R], g[NG];
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int k = 4 * (tid + TPB * i);
        v[i] = k < K ? *(const float4*)(xr + k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    if (p.add) {
        const float* ar = p.add + m * p.ld_add;
        constexpr int B = R > 4 ? 4 : R;
#pragma unroll
        for (int j = 0; j < R; j += B) {
            float4 b[B];
#pragma unroll
            for (int i = 0; i < B; i++) {
                const int k = 4 * (tid + TPB * (i + j));
                b[i] = k < K ? *(const float4*)(ar + k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int i = 0; i < B; i++) {
                float4& x = v[i + j];
                x = make_float4(x.x + b[i].x, x.y + b[i].y, x.z + b[i].z, x.w + b[i].w);
            }
        }
    }
    const float* gr = p.gate + m * p.ld_gate;
    if (p.gate && NG == R) {
#pragma unroll
        for (int i = 0; i < NG; i++) {
            const int k = 4 * (tid + TPB * i);
            g[i] = k < K ? *(const float4*)(gr + k) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
    if (p.sum) {
        float* sr = p.sum + m * p.ld_sum;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int k = 4 * (tid + TPB * i);
            if (k < K) *(float4*)(sr + k) = v[i];
        }
    }
    // each run's factor
    double f[R];
#pragma unroll
    for (int i = 0; i < R; i++) {
        const double x = v[i].x, y = v[i].y, z = v[i].z, w = v[i].w;
        f[i] = fma(w, w, fma(z, z, fma(y, y, x * x)));
    }
    const double n = (double)a.len, eps = (double)p.eps;
    if (a.len == K) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < R; i++) ss += f[i];
        ss = wg_reduce<TPB>(ss, red, [](double s, double t) { return s + t; });
        const double r = one_over_root(ss / n + eps);
#pragma unroll
        for (int i = 0; i < R; i++) f[i] = r;
    } else if (a.lanes) {
#pragma unroll
        for (int i = 0; i < R; i++) {
            f[i] = lanes_reduce(f[i], a.lanes, [](double s, double t) { return s + t; });
            f[i] = one_over_root(fma(f[i], 1.0 / n, eps));
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; i++)
            if (tid + TPB * i < K / 4) parts[tid + TPB * i] = f[i];
        __syncthreads();
        const int runs = a.len / 4;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int k = tid + TPB * i;
            if (k >= K / 4) break;
            double ss = 0.0;
            for (int j = k / runs * runs, e = j + runs; j < e; j++) ss += parts[j];
            f[i] = one_over_root(ss / n + eps);
        }
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int k = 4 * (tid + TPB * i);
        if (k >= K) break;
        double y[4] = {(double)v[i].x * f[i], (double)v[i].y * f[i], (double)v[i].z * f[i], (double)v[i].w * f[i]};
        if (p.norm_w) {
            const float4 w = *(const float4*)(p.norm_w + k % a.len);
            y[0] *= (double)w.x; y[1] *= (double)w.y; y[2] *= (double)w.z; y[3] *= (double)w.w;
        }
        if (p.gate) {
            const float4 z = NG == R ? g[NG == R ? i : 0] : *(const float4*)(gr + k);
            y[0] *= silu64(z.x); y[1] *= silu64(z.y); y[2] *= silu64(z.z); y[3] *= silu64(z.w);
        }
        v[i] = make_float4((float)y[0], (float)y[1], (float)y[2], (float)y[3]);
    }
    if (p.out) {
        float* o = p.out + m * p.ldo;
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int k = 4 * (tid + TPB * i);
            if (k < K) *(float4*)(o + k) = v[i];
        }
    }
    if (p.act_mode == GGQ_ACT_F32) return;
    float top[R], amax = 0.0f;
#pragma unroll
    for (int i = 0; i < R; i++) {
        top[i] = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
        amax = fmaxf(amax, top[i]);
    }
    uint32_t* q = (uint32_t*)(p.codes + m * K);
    if (p.act_mode == GGQ_ACT_Q8_ROW) {
        amax = wg_reduce<TPB>(amax, redf, [](float s, float t) { return fmaxf(s, t); });
        const float sc = step_of(amax), inv = __fdiv_rn(1.0f, sc);
        if (tid == 0) p.scales[m] = sc;
#pragma unroll
        for (int i = 0; i < R; i++)
            if (tid + TPB * i < K / 4) q[tid + TPB * i] = codes_of(v[i], inv);
    } else {
#pragma unroll
        for (int i = 0; i < R; i++) {
            float t = top[i];
            t = lanes_reduce(t, 8, [](float s, float u) { return fmaxf(s, u); });
            const int k = tid + TPB * i;
            const float sc = step_of(t);
            if (k >= K / 4) continue;
            if ((tid & 7) == 0) p.scales[m * (K / 32) + k / 8] = sc;
            q[k] = codes_of(v[i], __fdiv_rn(1.0f, sc));
        }
    }
}

}  // namespace

// A wavefront where four values a thread and run are enough (no barrier), else as many threads as leave a thread four
// runs: loads of 64 bytes in flight a thread, and several rows a CU up to 8192 columns.  Measured (us): one row of 2048 4.3, of which 3 are the
// launch; 2047 rows of 4096 with addition and codes 22 (4.9 TB/s); 2048 of 8192 42; 512 of 16384 24, of 30000 45 (4.4
// TB/s: one row a CU, 25 of its registers spilled); 513 rows of 32 gated heads of 128 9.5, 2.6 TB/s: two rows a CU, whose loads, arithmetic and
// stores follow one another (4096 such rows 38, for bytes worth 39).
hipError_t launch_norm(const ggq_norm_params& p, hipStream_t s) {
    NormArgs a{p, p.norm_len ? p.norm_len : p.n_cols, 0};
    const int lanes = a.len / 4;
    if (lanes <= 64 && !(lanes & (lanes - 1))) a.lanes = lanes;
    const size_t lds = a.len == p.n_cols || a.lanes ? 0 : sizeof(double) * (size_t)(p.n_cols / 4);
    // (a grid has fewer than 2^32 threads a dimension)
    const unsigned x = (unsigned)std::min(p.n_rows, 1 << 20), y = ((unsigned)p.n_rows + x - 1) / x;
#define L(TPB_, R_) norm_kernel<TPB_, R_><<<dim3(x, y), TPB_, lds, s>>>(a)
    if (p.n_cols <= 256) L(64, 1);
    else if (p.n_cols <= 512) L(64, 2);
    else if (p.n_cols <= 1024) L(64, 4);
    else if (p.n_cols <= 2048) L(256, 2);
    else if (p.n_cols <= 4096) L(256, 4);
    else if (p.n_cols <= 8192) L(512, 4);
    else if (p.n_cols <= 16384) L(1024, 4);
    else L(1024, 8);
#undef L
    return hipGetLastError();
}

}  // namespace ggq
