// ggq_sample.hip -- a token of each row of logits by temperature, top-k, top-p,
// min-p and a given random number (ggq_sample_dev).
//
// Nothing is sorted.  What is kept of a row is a head of its tokens in order of
// their logits, so a border between two tokens says all, and the tokens are
// drawn in order of their indices.
//   A logit l has z = 8 log2(e) l / T in 64 bits; its bin is floor(z) counted
// down from the largest one's, its weight 2^(-bin / 8) * 2^(frac / 8), the
// second factor (1 .. 1.09) in 36 bits after the point: sums over a bin are
// integers, which no order of additions changes.  frac is of the product before it was rounded to z: logits
// millions of temperatures away from 0 keep the bits of their differences.
//   sample_bins_kernel: parts of 4096 tokens; a part counts its tokens and
// adds up their factors in 512 bins below its own largest (64 powers of two: what
// is below counts as nothing), count and sum in one 64-bit LDS atomic, and puts its
// tokens in order of their bins.  A row of which all is kept needs its parts' sums only.
//   sample_pick_kernel: a workgroup a row adds up the parts' bins and finds the
// bin that holds the border.  Of up to 128 tokens a group of 16 lanes each counts what
// stands before it: where no more reach as far as the border, that is all there is to do.  Else
// the border's bin alone is looked through, if it is cut at all, by digits of its tokens' places in the
// order until 128 are left; then the part in which the running sum passes u, and the token in it.
// Bound: the row is read once by the first kernel (HBM), the second is a chain of
// short dependent steps (measured figures at launch_sample below).
#include <algorithm>

#include "ggq_device.h"
#include "ggq_steps.h"

namespace ggq {
namespace {

constexpr int kPart = 4096, kBins = 512, kRest = kBins - 1;  // the last bin: everything below
constexpr int kMaxParts = 1024;
constexpr int kList = 4096;  // tokens of a border's bin that are looked through in LDS
constexpr int kCount = 50;   // bits below a bin's count; a part's factors add up to less than 2^49
typedef unsigned long long u64;

struct PartInfo {
    double top;  // floor(z) of the part's largest logit, -infinity: no token
    float max;
    int32_t at;  // its first index
    int32_t count;  // tokens that are above -infinity
    int32_t pad;
    double mass;    // rows that are kept whole: weights, the unit that of bin 0
};

struct SampleArgs {
    ggq_sample_params p;
    int parts;
    PartInfo* info;  // [n_rows][parts]
    u64* bins;       // [n_rows][parts][kBins]
    double* upto;    // [n_rows][parts][kBins]: weights of a bin and those before it, in the part's own unit
    uint16_t* starts;  // [n_rows][parts][kBins]: where a bin's tokens begin in `order`
    uint16_t* order;   // [n_rows][parts][kPart]: tokens by their bins
};

// Across a wavefront by data-parallel moves, which cost a few cycles where a shuffle through LDS waits for a hundred: lanes
// take what lies 1, 2, 4 and 8 lanes before them in their row of 16 (nothing: 0), then the last of the row and of the half before.
template <int CTRL, int ROWS, typename T> __device__ __forceinline__ T from_before(T v) {
    constexpr int W = sizeof(T) / 4;
    struct Words { int w[W]; } x = __builtin_bit_cast(Words, v);
#pragma unroll
    for (int i = 0; i < W; i++) x.w[i] = __builtin_amdgcn_update_dpp(0, x.w[i], CTRL, ROWS, 0xF, false);
    return __builtin_bit_cast(T, x);
}
template <typename T, typename F> __device__ __forceinline__ T scan_by(T v, F f) {
    v = f(v, from_before<0x111, 0xF>(v));
    v = f(v, from_before<0x112, 0xF>(v));
    v = f(v, from_before<0x114, 0xF>(v));
    v = f(v, from_before<0x118, 0xF>(v));
    v = f(v, from_before<0x142, 0xA>(v));
    return f(v, from_before<0x143, 0xC>(v));
}
template <typename T> __device__ __forceinline__ T lane_of(T v, int lane) {  // (a uniform lane)
    constexpr int W = sizeof(T) / 4;
    struct Words { int w[W]; } x = __builtin_bit_cast(Words, v);
#pragma unroll
    for (int i = 0; i < W; i++) x.w[i] = __builtin_amdgcn_readlane(x.w[i], lane);
    return __builtin_bit_cast(T, x);
}
template <typename T> __device__ __forceinline__ T scan_add(T v) { return scan_by(v, [](T a, T b) { return a + b; }); }  // itself included
template <typename T> __device__ __forceinline__ T wave_sum(T v) { return lane_of(scan_add(v), 63); }
template <typename T> __device__ __forceinline__ T wave_max(T v) { return lane_of(scan_by(v, [](T a, T b) { return max(a, b); }), 63); }

// Whether a logit can have a weight: above -infinity.  (On its bits: this compiler's ballot of v > -INFINITY lets NaN through.)
__device__ __forceinline__ bool there(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    return (u & 0x7FFFFFFFu) <= 0x7F800000u && u != 0xFF800000u;
}
// Keys in order of the values (no NaN).
__device__ __forceinline__ uint32_t key_of(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v == 0.0f ? 0.0f : v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
// Eighths of an octave that a logit of 1 is worth at a row's temperature (0 where that is infinite); -1: greedy.
__device__ __forceinline__ double eighths_of(const ggq_sample_params& p, int row) {
    const float t = p.temperature ? p.temperature[row] : 1.0f;
    return t > 0.0f ? 8.0 * 1.44269504088896340736 / (double)t : -1.0;
}
struct Bin {
    double top;  // floor(z)
    u64 factor;  // 2^(frac / 8) in units of 2^-36
    __device__ double weight() const { return (__builtin_bit_cast(double, factor + __builtin_bit_cast(u64, 65536.0)) - 65536.0) * 68719476736.0; }
};
// 2^(x / 8), x from 0 to 1, within 3e-13: the polynomial of degree 5 that meets it in Chebyshev's six places
__device__ __forceinline__ double factor_of(double x) {
    double e = 4.2495173672986884e-08;
    e = fma(e, x, 2.3461308667386375e-06);
    e = fma(e, x, 0.00010840752642405686);
    e = fma(e, x, 0.003753538921359355);
    e = fma(e, x, 0.08664339759143012);
    return fma(e, x, 0.9999999999997022);
}
// What the product l c has above fl, which is floor of it rounded: from 0 to 1 but for that rounding.  (Where that is as large as 1, z beyond
// 2^53, bins of different logits are 2^28 apart and more, and only equal ones, whose factors are equal, count: any factor will do.)
__device__ __forceinline__ double frac_of(float l, double c, double fl) { return fmin(fmax(fma((double)l, c, -fl), -1.0), 2.0); }
__device__ __forceinline__ Bin bin_of(float l, double c) {
    const double fl = floor((double)l * c);
    if (l == INFINITY) return Bin{INFINITY, u64(1) << 36};
    // (a sum of 2^16 and more has its last bit at 2^-36)
    return Bin{fl, __builtin_bit_cast(u64, factor_of(frac_of(l, c, fl)) + 65536.0) - __builtin_bit_cast(u64, 65536.0)};
}
__device__ __forceinline__ double floor_of(float l, double c) { return l == INFINITY ? INFINITY : floor((double)l * c); }
// Bins that `at` lies below `top`, at most kRest.
__device__ __forceinline__ int below(double top, double at) {
    return at == top ? 0 : (int)fmin(top - at, (double)kRest);
}

// 2^(-j / 8)
__device__ __forceinline__ double step_down(int j) {
    constexpr double r[8] = {1.0, 0.91700404320467123174, 0.84089641525371454303, 0.77110541270397041179,
                             0.70710678118654752440, 0.64841977732550483297, 0.59460355750136053336, 0.54525386633262882960};
    double v = r[0];
#pragma unroll
    for (int i = 1; i < 8; i++) v = (j & 7) == i ? r[i] : v;
    return ldexp(v, -(j >> 3));
}

struct Filters {
    int k;
    float p, m;
    bool by_k, by_p, by_m;
    __device__ bool any() const { return by_k || by_p || by_m; }
};
__device__ __forceinline__ Filters filters_of(const ggq_sample_params& p, int row) {
    Filters f;
    f.k = p.top_k ? p.top_k[row] : 0;
    f.p = p.top_p ? p.top_p[row] : 1.0f;
    f.m = p.min_p ? p.min_p[row] : 0.0f;
    f.by_k = f.k > 0 && f.k < p.n_vocab;
    f.by_p = f.p < 1.0f;
    f.by_m = f.m > 0.0f;
    return f;
}

constexpr int kBinThreads = 512;
static_assert(kBinThreads == kBins && kPart == 8 * kBinThreads, "a thread a bin, and eight tokens");
__global__ __launch_bounds__(kBinThreads) void sample_bins_kernel(SampleArgs a) {
    constexpr int V = kPart / kBinThreads, NW = kBinThreads / 64;
    __shared__ u64 bins[kBins];
    __shared__ __attribute__((aligned(16))) uint16_t starts[kBins], order[kPart];
    __shared__ uint32_t red[NW][3];
    __shared__ double sums[NW];
    const ggq_sample_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, row = blockIdx.y, part = blockIdx.x, base = part * kPart;
    const float* x = p.logits + (int64_t)row * p.ld;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int k = base + tid + kBinThreads * i;
        v[i] = k < p.n_vocab ? x[k] : -INFINITY;
    }
    const double c = eighths_of(p, row);
    const bool whole = !filters_of(p, row).any();
    if (!whole) {
        bins[tid] = 0;
    }
    uint32_t top = 0, at = 0xFFFFFFFFu, n = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const bool in = there(v[i]);
        n += (uint32_t)__popcll(__ballot(in));
        const uint32_t key = in ? key_of(v[i]) : 0u;
        if (key > top) {
            top = key;
            at = (uint32_t)(base + tid + kBinThreads * i);
        }
    }
    const uint32_t own_top = top;
    top = wave_max(top);
    at = ~wave_max(own_top == top ? ~at : 0u);
    if (lane == 0) { red[tid >> 6][0] = top; red[tid >> 6][1] = at; red[tid >> 6][2] = n; }
    __syncthreads();
    n = 0;
    top = 0;
#pragma unroll
    for (int i = 0; i < NW; i++) {
        n += red[i][2];
        if (red[i][0] > top || (red[i][0] == top && red[i][1] < at)) { top = red[i][0]; at = red[i][1]; }
    }
    const int64_t id = (int64_t)row * a.parts + part;
    const float mx = n ? of_key(top) : -INFINITY;
    const double first = n && c >= 0.0 ? bin_of(mx, c).top : -INFINITY;
    PartInfo info{first, mx, (int32_t)at, (int32_t)n, 0, 0.0};
    if (c < 0.0) {  // greedy rows need no more
        if (tid == 0) a.info[id] = info;
        return;
    }
    if (whole) {
        // (the bins' LDS holds the bins' weights)
        bins[tid] = __builtin_bit_cast(u64, tid == kRest ? 0.0 : step_down(tid));
        __syncthreads();
        double m = 0.0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const double fl = floor_of(v[i], c);
            const double w = there(v[i]) ? __builtin_bit_cast(double, bins[below(first, fl)]) : 0.0;
            m = fma(v[i] == INFINITY || !there(v[i]) ? 1.0 : factor_of(frac_of(v[i], c, fl)), w, m);
        }
        m = wave_sum(m);
        if (lane == 0) sums[tid >> 6] = m;
        __syncthreads();
        m = 0.0;
#pragma unroll
        for (int i = 0; i < NW; i++) m += sums[i];
        info.mass = m * 68719476736.0;  // (2^36, as the factors)
        if (tid == 0) a.info[id] = info;
        return;
    }
    uint32_t spot[V];  // bin and place in it
#pragma unroll
    for (int i = 0; i < V; i++) {
        spot[i] = 0xFFFFFFFFu;
        if (!there(v[i])) continue;
        const Bin b = bin_of(v[i], c);
        const int j = below(first, b.top);
        const u64 old = atomicAdd(&bins[j], (u64(1) << kCount) + (j == kRest ? 0 : b.factor));
        spot[i] = (uint32_t)j << 16 | (uint32_t)(old >> kCount);
    }
    __syncthreads();
    // where the bins begin, and the weights up to them
    const u64 w = bins[tid];
    const uint32_t nb = (uint32_t)(w >> kCount);
    const double mb = (double)(w & ((u64(1) << kCount) - 1)) * step_down(tid);
    const uint32_t run = scan_add(nb);
    double runw = scan_add(mb);
    if (lane == 63) { red[tid >> 6][0] = run; sums[tid >> 6] = runw; }
    __syncthreads();
    uint32_t start = run - nb;
#pragma unroll
    for (int i = 0; i < NW; i++)
        if (i < tid >> 6) { start += red[i][0]; runw += sums[i]; }
    starts[tid] = (uint16_t)start;
    a.upto[id * kBins + tid] = runw;
    a.bins[id * kBins + tid] = w;
    a.starts[id * kBins + tid] = (uint16_t)start;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; i++)
        if (spot[i] != 0xFFFFFFFFu) order[starts[spot[i] >> 16] + (spot[i] & 0xFFFFu)] = (uint16_t)(tid + kBinThreads * i);
    __syncthreads();
    ((uint4*)(a.order + id * kPart))[tid] = ((const uint4*)order)[tid];
    if (tid == 0) a.info[id] = info;
}

// A token's place in the order: larger ones come first.
__device__ __forceinline__ u64 place_of(uint32_t key, uint32_t idx) { return (u64)key << 32 | ~idx; }
// The border of what is kept: bins before `bin` whole, of `bin` the tokens from this place on.
struct Border {
    int bin;
    u64 place;
};
__device__ __forceinline__ bool nearer(const Border& a, const Border& b) { return a.bin != b.bin ? a.bin < b.bin : a.place > b.place; }

constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kFew = 128;      // tokens that are compared with each other
constexpr int kDigits = 256;
// Over 16 lanes, in the last of them.
template <typename T> __device__ __forceinline__ T sum16(T v) {
    v += from_before<0x111, 0xF>(v);
    v += from_before<0x112, 0xF>(v);
    v += from_before<0x114, 0xF>(v);
    return v + from_before<0x118, 0xF>(v);
}

__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleArgs a) {
    // factors of a bin, in units of 2^-36, and its count; a lane's eight are followed by a gap, which keeps lanes off each other's banks
    __shared__ u64 mass[kBins / 8 * 9];
    __shared__ uint32_t count[kBins / 8 * 9];
    auto apart = [](int j) { return j + (j >> 3); };
    __shared__ double tab[kBins];     // 2^(-j / 8)
    __shared__ int32_t shift[kMaxParts];
    __shared__ uint32_t run_at[kMaxParts], run_from[kMaxParts];  // of the tokens that are looked through: each part's first
    __shared__ double pmass[kMaxParts];
    __shared__ u64 inside[kMaxParts];  // kept factors of the border's bin, of each part
    __shared__ u64 place[kList];
    __shared__ u64 dmass[kDigits];
    __shared__ uint32_t dcount[kDigits];
    __shared__ u64 few[kFew];
    __shared__ double few_w[kFew];
    __shared__ uint32_t few_rank[kFew];
    __shared__ double wave_d[kWaves];
    __shared__ uint32_t wave_u[kWaves], wave_v[kWaves];
    __shared__ u64 s_place, s_mass;
    __shared__ uint32_t s_n, s_digit, s_count, s_need;
    __shared__ u64 s_left;
    __shared__ double s_total;
    const ggq_sample_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.x;
    const float* x = p.logits + (int64_t)row * p.ld;
    const u64* bins = a.bins + (int64_t)row * a.parts * kBins;
    const PartInfo* info = a.info + (int64_t)row * a.parts;
    PartInfo own{};
    if (tid < a.parts) own = info[tid];
    const double c = eighths_of(p, row);
    const Filters flt = filters_of(p, row);
    const float t_row = p.temperature ? p.temperature[row] : 1.0f;
    float u = p.u[row];
    if (!(u > 0.0f)) u = 0.0f;

    // the row's largest token, and how many there are
    u64 top = own.count ? place_of(key_of(own.max), (uint32_t)own.at) : 0;
    uint32_t n_all = (uint32_t)own.count;
    for (int q = tid + kThreads; q < a.parts; q += kThreads) {
        const PartInfo i = info[q];
        if (i.count) top = max(top, place_of(key_of(i.max), (uint32_t)i.at));
        n_all += (uint32_t)i.count;
    }
    top = wave_max(top);
    n_all = wave_sum(n_all);
    if (lane == 0) { few[wave] = top; wave_u[wave] = n_all; }
    static_assert(kThreads == kBins, "a thread a bin");
    tab[tid] = step_down(tid);
    __syncthreads();
    n_all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
        n_all += wave_u[i];
        top = max(top, few[i]);
    }
    if (c < 0.0 || n_all == 0) {
        if (tid == 0) {
            p.token[row] = n_all ? (int32_t)~(uint32_t)top : 0;
            if (p.prob) p.prob[row] = n_all ? 1.0f : 0.0f;
        }
        return;
    }
    const uint32_t top_key = (uint32_t)(top >> 32);
    const float mx = of_key(top_key);
    const double first = bin_of(mx, c).top;
    for (int q = tid; q < a.parts; q += kThreads) {
        if (q != tid) own = info[q];
        const int sh = own.count ? below(first, own.top) : kRest;
        shift[q] = sh;
        inside[q] = 0;
        if (!flt.any()) pmass[q] = sh < kRest ? own.mass * tab[sh] : 0.0;
    }
    __syncthreads();
    auto factor = [&](u64 place) { return bin_of(of_key((uint32_t)(place >> 32)), c).factor; };

    Border border{kRest, 0};  // all that has a weight
    if (flt.any()) {
        {  // the row's bins
            uint32_t n = 0;
            u64 m = 0;
            if (tid < kRest)
#pragma unroll 32
                for (int q = 0; q < a.parts; q++) {
                    const int j = tid - shift[q];
                    const u64 w = j >= 0 ? bins[(int64_t)q * kBins + j] : 0;
                    n += (uint32_t)(w >> kCount);
                    m += w & ((u64(1) << kCount) - 1);
                }
            count[apart(tid)] = n;
            mass[apart(tid)] = m;
            __syncthreads();
        }
        // running sums, eight bins a lane (in every wavefront)
        uint32_t nb[8], n_before, n_own = 0;
        double wb[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            nb[i] = 8 * lane + i < kRest ? count[9 * lane + i] : 0;
            wb[i] = 8 * lane + i < kRest ? (double)mass[9 * lane + i] * ldexp(step_down(i), -lane) : 0.0;
            n_own += nb[i];
        }
        n_before = scan_add(n_own) - n_own;
        // top-k's bin (kRest: all are kept), and the count before it
        int bin_k = kRest;
        uint32_t before_k = 0;
        if (flt.by_k) {
            uint32_t b = n_before;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (bin_k == kRest && nb[i] && b + nb[i] >= (uint32_t)flt.k) { bin_k = 8 * lane + i; before_k = b; }
                b += nb[i];
            }
            const u64 any = __ballot(bin_k < kRest);
            const int l = any ? __ffsll(any) - 1 : 0;
            bin_k = lane_of(bin_k, l);
            before_k = lane_of(before_k, l);
        }
        Border border_m{kRest, 0};
        if (flt.by_m) {
            // the smallest value with (value - largest) / T >= ln min_p
            // (at an infinite T all finite ones have the weight 1)
            const double lim = t_row == INFINITY ? -INFINITY : flt.m >= 1.0f ? 0.0 : (double)t_row * log((double)flt.m);
            float v = (float)((double)mx + lim);
            if (!(v <= mx) || mx == INFINITY) v = mx;
            uint32_t key = key_of(v);
            if (v > -INFINITY && mx < INFINITY) {
                // A step or two from here, but half a billion where v is next to nothing beside the largest (differences from
                // that round to the same): strides that double, then halve.  (0x00800000: the smallest finite number's key.)
                auto within = [&](uint32_t k) { return (double)of_key(k) - (double)mx >= lim; };
                while (key < top_key && !within(key)) key++;
                uint32_t stride = 1;
                for (; key - 0x00800000u >= stride && within(key - stride); stride *= 2) key -= stride;
                for (; stride; stride /= 2)
                    if (key - 0x00800000u >= stride && within(key - stride)) key -= stride;
            }
            v = of_key(key);
            if (v > -INFINITY) {
                const int bin = below(first, floor_of(v, c));
                if (bin < kRest) border_m = Border{bin, (u64)key << 32};
            }
            if (flt.m > 1.0f) border_m = Border{0, top};  // (no weight is so large: the first token alone)
        }
        // What the filters look through, one after the other: the border of top-k, then of top-p, then what is kept of the
        // border's bin by parts; or, first of all, everything up to the border where that is little.
        enum { ALL = -1, TOP_K = 0, TOP_P = 1, KEEP = 2 };
        int listed_lo = -1, listed_hi = -1;
        int bin = kRest;  // top_p's
        u64 left_p = 0;
        const int most = a.parts > 1 ? 1 << (31 - __builtin_clz(a.parts - 1)) : 0;  // the largest power of two below the parts
        u64 kmass = bin_k < kRest ? mass[apart(bin_k)] : 0;  // factors that top-k keeps of its bin
        border.bin = bin_k;
#pragma nounroll
        for (int phase = ALL; phase <= KEEP; phase++) {
            int lo = 0, hi = 0;
            uint32_t n = 0, need = 0;
            u64 left = 0;
            bool by_mass = false;
            if (phase == TOP_K) {
                if (bin_k == kRest) continue;
                lo = hi = bin_k;
                n = count[apart(bin_k)];
                need = (uint32_t)flt.k - before_k;
                if (need >= n) continue;
            } else if (phase == KEEP) {
                if (border_m.bin < kRest && nearer(border_m, border)) border = border_m;
                if (border.bin == kRest) break;
                lo = hi = border.bin;
                n = count[apart(lo)];
            } else {
                // the first bin in which the weights reach top_p of their sum, by what is known of top-k's border
                if (flt.by_p && (phase == ALL || bin_k < kRest)) {
                    double w[8], mine = 0.0;
                    const double cut = border.bin < kRest ? (double)kmass * tab[border.bin] : 0.0;
                    bin = kRest;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int j = 8 * lane + i;
                        w[i] = j > border.bin ? 0.0 : j == border.bin && j < kRest ? cut : wb[i];
                        mine += w[i];
                    }
                    const double run = scan_add(mine);
                    const double want = fmax(0.0, (double)flt.p) * lane_of(run, 63);
                    double b = run - mine, hb = 0.0;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int j = 8 * lane + i;
                        if (bin == kRest && nb[i] && j <= border.bin && b + w[i] >= want) { bin = j; hb = b; }
                        b += w[i];
                    }
                    const u64 any = __ballot(bin < kRest);
                    const int l = any ? __ffsll(any) - 1 : 0;
                    bin = lane_of(bin, l);
                    const double in = (want - lane_of(hb, l)) / tab[bin];  // in the bin's own units, rounded up
                    left_p = in > 0.0 ? (u64)ceil(in) : 0;
                }
                left = left_p;
                if (phase == TOP_P) {
                    if (bin == kRest) continue;
                    lo = hi = bin;
                    n = count[apart(bin)];
                    by_mass = true;
                } else {
                    // (top_p's share is of exactly what top-k leaves)
                    hi = flt.by_k && flt.by_p ? bin_k : min(min(bin_k, bin), border_m.bin);
                    if (hi == kRest) continue;
#pragma unroll
                    for (int i = 0; i < 8; i++) n += 8 * lane + i <= hi ? nb[i] : 0;
                    n = wave_sum(n);
                    if (n > kFew) continue;
                }
            }
            // The tokens of the bins lo .. hi are runs of the parts' orders, numbered through; in LDS if they are no more
            // than kList.
            if (listed_lo != lo || listed_hi != hi) {
                __syncthreads();
                uint32_t before = 0;
                for (int q0 = 0; q0 < a.parts; q0 += kThreads) {
                    const int q = q0 + tid;
                    uint32_t from = 0, len = 0;
                    if (q < a.parts && shift[q] <= hi) {
                        const uint16_t* st = a.starts + ((int64_t)row * a.parts + q) * kBins;
                        from = st[max(lo - shift[q], 0)];
                        len = st[hi - shift[q] + 1] - from;  // (hi < kRest)
                    }
                    const uint32_t run = scan_add(len);
                    if (lane == 63) wave_u[wave] = run;
                    __syncthreads();
                    uint32_t at = before + run - len;
#pragma unroll
                    for (int i = 0; i < kWaves; i++) {
                        at += i < wave ? wave_u[i] : 0;
                        before += wave_u[i];
                    }
                    if (q < a.parts) { run_at[q] = at; run_from[q] = from; }
                    __syncthreads();
                }
            }
            auto part_at = [&](uint32_t i) {  // the last part whose run begins at i or before (parts without any share their begin with the next)
                int q = 0;
                for (int s = most; s > 0; s >>= 1)
                    if (q + s < a.parts && run_at[q + s] <= i) q += s;
                return q;
            };
            auto index_at = [&](int q, uint32_t i) {
                return q * kPart + a.order[((int64_t)row * a.parts + q) * kPart + run_from[q] + i - run_at[q]];
            };
            auto token_at = [&](uint32_t i) {
                const int idx = index_at(part_at(i), i);
                return place_of(key_of(x[idx]), (uint32_t)idx);
            };
            if (listed_lo != lo || listed_hi != hi) {
                listed_lo = lo;
                listed_hi = hi;
                if (n <= kList) {
                    // (four of a thread at a time: their loads depend on each other)
                    for (uint32_t i = tid; i < n; i += 4 * kThreads) {
                        int idx[4];
                        float v[4];
#pragma unroll
                        for (int t = 0; t < 4; t++) idx[t] = i + t * kThreads < n ? index_at(part_at(i + t * kThreads), i + t * kThreads) : 0;
#pragma unroll
                        for (int t = 0; t < 4; t++) v[t] = x[idx[t]];
#pragma unroll
                        for (int t = 0; t < 4; t++)
                            if (i + t * kThreads < n) place[i + t * kThreads] = place_of(key_of(v[t]), (uint32_t)idx[t]);
                    }
                    __syncthreads();
                }
            }
            auto each = [&](auto f) {
                for (uint32_t i = tid; i < n; i += kThreads) f(n <= kList ? place[i] : token_at(i));
            };
            if (phase == KEEP) {
                auto add = [&](u64 pl) {
                    if (pl >= border.place) atomicAdd(&inside[~(uint32_t)pl / kPart], factor(pl));
                };
                each(add);
                break;
            }
            // Digits of the places, the largest first, until few are left in [base, base + 2^bits)
            u64 base = 0, taken = 0;
            int bits = 64;
            uint32_t in_range = n;
            if (n > kFew) {
                u64 least = ~u64(0), most = 0;
                each([&](u64 pl) {
                    least = min(least, pl);
                    most = max(most, pl);
                });
                least = ~wave_max(~least);
                most = wave_max(most);
                if (lane == 0) { few[2 * wave] = least; few[2 * wave + 1] = most; }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < kWaves; i++) {
                    least = min(least, few[2 * i]);
                    most = max(most, few[2 * i + 1]);
                }
                base = least;
                bits = 64 - __builtin_clzll((most - least) | 1);  // (below 64: places differ in less than the keys' sign and all)
            }
            while (in_range > kFew) {
                const int low = max(0, bits - 8);
                __syncthreads();
                for (int d = tid; d < kDigits; d += kThreads) {
                    dmass[d] = 0;
                    dcount[d] = 0;
                }
                __syncthreads();
                each([&](u64 pl) {
                    if (pl < base || (bits < 64 && (pl - base) >> bits)) return;
                    const uint32_t d = (uint32_t)((pl - base) >> low);
                    atomicAdd(&dcount[d], 1u);
                    atomicAdd(&dmass[d], factor(pl));
                });
                __syncthreads();
                if (wave == 0) {  // four digits a lane, the largest first
                    uint32_t own_n = 0;
                    u64 own_m = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) { own_n += dcount[kDigits - 1 - 4 * lane - i]; own_m += dmass[kDigits - 1 - 4 * lane - i]; }
                    uint32_t before = scan_add(own_n) - own_n, hb = 0, lb = 0;
                    u64 beforem = scan_add(own_m) - own_m, hm = 0, lm = 0;
                    int hit = -1, last = -1;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int d = kDigits - 1 - 4 * lane - i;
                        const uint32_t dn = dcount[d];
                        const u64 dm = dmass[d];
                        if (dn) {
                            if (hit < 0 && (by_mass ? beforem + dm >= left : before + dn >= need)) { hit = d; hb = before; hm = beforem; }
                            last = d;
                            lb = before;
                            lm = beforem;
                        }
                        before += dn;
                        beforem += dm;
                    }
                    const u64 any = __ballot(hit >= 0), some = __ballot(last >= 0);
                    const int l = any ? __ffsll(any) - 1 : 63 - __builtin_clzll(some);
                    const int d = lane_of(any ? hit : last, l);
                    hb = lane_of(any ? hb : lb, l);
                    hm = lane_of(any ? hm : lm, l);
                    if (lane == 0) {  // (none, only by mass: rounding left something over, so all of them)
                        s_digit = (uint32_t)d;
                        s_need = need - hb;
                        s_left = any ? left - hm : dmass[d];
                        s_mass = hm;
                        s_count = dcount[d];
                    }
                }
                __syncthreads();
                base += (u64)s_digit << low;
                need = s_need;
                left = s_left;
                taken += s_mass;
                in_range = s_count;
                bits = low;
            }
            // those few, side by side
            __syncthreads();
            if (tid == 0) s_n = 0;
            __syncthreads();
            auto gather = [&](u64 pl) {
                if (pl < base || (bits < 64 && (pl - base) >> bits)) return;
                const uint32_t i = atomicAdd(&s_n, 1u);
                if (i < kFew) few[i] = pl;
            };
            each(gather);
            __syncthreads();
            const int nf = (int)min(s_n, (uint32_t)kFew), sub = tid & 15;
            for (int i = tid >> 4; i < nf; i += kThreads / 16) {  // 16 lanes a token: what stands before it
                const u64 mine = few[i];
                uint32_t r = 0;
                for (int j = sub; j < nf; j += 16) r += few[j] > mine ? 1u : 0u;
                r = sum16(r);
                if (sub == 15) {
                    const Bin b = bin_of(of_key((uint32_t)(mine >> 32)), c);
                    few_rank[i] = r;
                    if (phase == ALL) {  // (in their order: sums in 64 bits depend on it)
                        place[r] = mine;
                        few_w[r] = flt.by_k && r >= (uint32_t)flt.k ? 0.0 : (double)b.factor * tab[below(first, b.top)];
                    } else {
                        few_w[i] = __builtin_bit_cast(double, b.factor);
                    }
                }
            }
            __syncthreads();
            if (phase != ALL) {
                for (int i = tid >> 4; i < nf; i += kThreads / 16) {
                    const uint32_t r = few_rank[i];
                    u64 before = 0;
                    for (int j = sub; j < nf; j += 16) before += few_rank[j] < r ? __builtin_bit_cast(u64, few_w[j]) : 0;
                    before = sum16(before);
                    const u64 upto = before + __builtin_bit_cast(u64, few_w[i]);
                    // (by mass: the last of them where rounding left something over; none before it reached)
                    const bool hit = by_mass ? (upto >= left && (before < left || r == 0)) || (r + 1 == (uint32_t)nf && before < left && upto < left)
                                             : r + 1 == need;
                    if (hit && sub == 15) { s_place = few[i]; s_mass = upto; }
                }
                __syncthreads();
                const Border found{lo, s_place};
                if (phase == TOP_K) kmass = taken + s_mass;
                if (phase == TOP_K || nearer(found, border)) border = found;
                __syncthreads();
                continue;
            }
            if (tid < nf) {
                few[tid] = place[tid];
                few_rank[tid] = (uint32_t)tid;
            }
            __syncthreads();
            double whole = 0.0;
            if (flt.by_p && !flt.by_k) {  // top_p's share is of the whole row
#pragma unroll
                for (int i = 0; i < 8; i++) whole += wb[i];
                whole = wave_sum(whole);
            }
            double kept[kFew * 16 / kThreads];
#pragma unroll
            for (int t = 0; t < kFew * 16 / kThreads; t++) {
                const int i = (tid >> 4) + t * (kThreads / 16);
                kept[t] = 0.0;
                if (i < nf) {
                    const uint32_t r = few_rank[i];
                    double ahead = 0.0, total = 0.0;
                    for (int j = sub; j < nf; j += 16) {
                        total += few_w[j];
                        ahead += few_rank[j] < r ? few_w[j] : 0.0;
                    }
                    ahead = sum16(ahead);
                    total = flt.by_k ? sum16(total) : whole;
                    bool keep = r == 0 || ((!flt.by_p || ahead < fmax(0.0, (double)flt.p) * total) && few[i] >= border_m.place);
                    kept[t] = keep ? few_w[i] : 0.0;
                }
            }
            __syncthreads();
#pragma unroll
            for (int t = 0; t < kFew * 16 / kThreads; t++) {
                const int i = (tid >> 4) + t * (kThreads / 16);
                if (i < nf && sub == 15) few_w[i] = kept[t];
            }
            if (tid < kWaves) { wave_u[tid] = 0xFFFFFFFFu; wave_v[tid] = 0; }
            __syncthreads();
            // weights up to each token in order of the indices (complements, here)
            double sums = 0.0;
#pragma unroll
            for (int t = 0; t < kFew * 16 / kThreads; t++) {
                const int i = (tid >> 4) + t * (kThreads / 16);
                if (i < nf) {
                    const uint32_t mine = ~(uint32_t)few[i];
                    double upto = 0.0, sum = 0.0;
                    for (int j = sub; j < nf; j += 16) {
                        sum += few_w[j];
                        upto += ~(uint32_t)few[j] <= mine ? few_w[j] : 0.0;
                    }
                    upto = sum16(upto);
                    sums = sum16(sum);
                    if (sub == 15 && few_w[i] > 0.0) {
                        if (upto > (double)u * sums) atomicMin(&wave_u[0], mine);
                        atomicMax(&wave_v[0], mine + 1);
                    }
                }
            }
            __syncthreads();
            const uint32_t hit = wave_u[0] != 0xFFFFFFFFu ? wave_u[0] : wave_v[0] ? wave_v[0] - 1 : ~(uint32_t)top;
#pragma unroll
            for (int t = 0; t < kFew * 16 / kThreads; t++) {
                const int i = (tid >> 4) + t * (kThreads / 16);
                if (i < nf && sub == 15 && ~(uint32_t)few[i] == hit) {
                    p.token[row] = (int32_t)hit;
                    if (p.prob) p.prob[row] = (float)(few_w[i] / sums);
                }
            }
            return;
        }
        __syncthreads();
        // kept weights of the parts
        for (int q = tid; q < a.parts; q += kThreads) {
            const int j = border.bin - 1 - shift[q];
            pmass[q] = (j >= 0 ? a.upto[((int64_t)row * a.parts + q) * kBins + j] * tab[shift[q]] : 0.0) +
                       (border.bin < kRest ? (double)inside[q] * tab[border.bin] : 0.0);
        }
        __syncthreads();
    }
    // running sums of the parts by one wavefront: the first that passes u times the whole (else the last that has any)
    if (wave == 0) {
        const int per = (a.parts + 63) / 64;
        double mine = 0.0;
        for (int i = 0; i < per; i++) mine += per * lane + i < a.parts ? pmass[per * lane + i] : 0.0;
        const double run = scan_add(mine);
        const double total = lane_of(run, 63), want = (double)u * total;
        double b = run - mine, hb = 0.0;
        int hit = -1, last = -1;
        double lb = 0.0;
        for (int i = 0; i < per; i++) {
            const int q = per * lane + i;
            const double m = q < a.parts ? pmass[q] : 0.0;
            if (m > 0.0) {
                if (hit < 0 && b + m > want) { hit = q; hb = b; }
                last = q;
                lb = b;
            }
            b += m;
        }
        // (the largest token has a weight; its part where nothing should have one)
        const u64 any = __ballot(hit >= 0), some = __ballot(last >= 0);
        const int l = any ? __ffsll(any) - 1 : some ? 63 - __builtin_clzll(some) : 0;
        int q = lane_of(any ? hit : last, l);
        if (q < 0) q = (int)(~(uint32_t)top / kPart);
        const double before = lane_of(any ? hb : lb, l);
        if (lane == 0) {
            s_digit = (uint32_t)q;
            s_total = total;
            wave_d[0] = want - before;
        }
    }
    __syncthreads();
    const int part = (int)s_digit;
    const double total = s_total, want = wave_d[0];
    // and the token in it: eight in a row a thread
    constexpr int V = kPart / kThreads;
    const int base = part * kPart + V * tid;
    float l[V];
    static_assert(V % 4 == 0, "runs of four");
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        float4 y;
        if (((uintptr_t)x & 15) == 0 && base + i + 3 < p.n_vocab) {
            y = *(const float4*)(x + base + i);
        } else {
            float z[4];
#pragma unroll
            for (int e = 0; e < 4; e++) z[e] = base + i + e < p.n_vocab ? x[base + i + e] : -INFINITY;
            y = make_float4(z[0], z[1], z[2], z[3]);
        }
        l[i] = y.x; l[i + 1] = y.y; l[i + 2] = y.z; l[i + 3] = y.w;
    }
    double w[V], mine = 0.0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        w[i] = 0.0;
        if (there(l[i])) {
            const Bin b = bin_of(l[i], c);
            const int j = below(first, b.top);
            if (j < kRest && (j < border.bin || (j == border.bin && place_of(key_of(l[i]), (uint32_t)(base + i)) >= border.place)))
                w[i] = b.weight() * tab[j];
        }
        mine += w[i];
    }
    const double run = scan_add(mine);
    __syncthreads();
    if (lane == 63) wave_d[wave] = run;
    __syncthreads();
    double b = run - mine;
    {
        double before[kWaves];
#pragma unroll
        for (int i = 0; i < kWaves; i++) before[i] = wave_d[i];
#pragma unroll
        for (int i = 0; i < kWaves; i++) b += i < wave ? before[i] : 0.0;
    }
    uint32_t hit = 0xFFFFFFFFu, last = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        if (w[i] > 0.0) {
            if (hit == 0xFFFFFFFFu && b + w[i] > want) hit = (uint32_t)(base + i);
            last = (uint32_t)(base + i) + 1;
        }
        b += w[i];
    }
    // (the wavefront's first and last: indices ascend with the lanes)
    const u64 any = __ballot(hit != 0xFFFFFFFFu), some = __ballot(last != 0);
    hit = any ? lane_of(hit, __ffsll(any) - 1) : 0xFFFFFFFFu;
    last = some ? lane_of(last, 63 - __builtin_clzll(some)) : 0;
    if (lane == 0) { wave_u[wave] = hit; wave_v[wave] = last; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
        hit = min(hit, wave_u[i]);
        last = max(last, wave_v[i]);
    }
    const uint32_t token = hit != 0xFFFFFFFFu ? hit : last ? last - 1 : ~(uint32_t)top;
#pragma unroll
    for (int i = 0; i < V; i++)
        if (token == (uint32_t)(base + i)) {
            p.token[row] = (int32_t)token;
            if (p.prob) p.prob[row] = (float)(w[i] / total);
        }
}

}  // namespace

namespace {
int parts_of(const ggq_sample_params& p) { return (p.n_vocab + kPart - 1) / kPart; }
size_t info_bytes(const ggq_sample_params& p) { return (sizeof(PartInfo) * (size_t)p.n_rows * parts_of(p) + 255) / 256 * 256; }
}  // namespace
size_t sample_ws_bytes(const ggq_sample_params& p) {
    return info_bytes(p) + ((sizeof(u64) + sizeof(double)) * kBins + sizeof(uint16_t) * (kBins + kPart)) * (size_t)p.n_rows * parts_of(p);
}
// Measured (us, first + second kernel): one row of 128256 by top-k, top-p and min-p 6 + 13; 33 rows by top-p 16 + 22; 200 rows of 32003
// kept whole 17 + 8; 256 rows of 128256 by top-p 106, whole 69, greedy 34 (their bytes take 26).  The first is arithmetic (90 vector
// instructions a token of a row kept whole, 106 where there are filters) and LDS atomics, the second up to nine loads that wait for each other at about 1 us each.  Where a
// border's bin holds more than kList tokens (temperatures above 4 at such sizes, logits all alike) it is read anew for
// each digit by the row's one workgroup: one row of 151936 equal logits 583.
hipError_t launch_sample(const ggq_sample_params& p, void* ws, hipStream_t s) {
    const size_t parts = (size_t)p.n_rows * parts_of(p);
    SampleArgs a{p, parts_of(p), (PartInfo*)ws, nullptr, nullptr, nullptr, nullptr};
    a.bins = (u64*)((char*)ws + info_bytes(p));
    a.upto = (double*)(a.bins + kBins * parts);
    a.order = (uint16_t*)(a.upto + kBins * parts);
    a.starts = a.order + kPart * parts;
    sample_bins_kernel<<<dim3((unsigned)a.parts, (unsigned)p.n_rows), kBinThreads, 0, s>>>(a);
    sample_pick_kernel<<<dim3((unsigned)p.n_rows), kThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace ggq
