// ggq_sample.hip -- a token of each row of logits by temperature, top-k, top-p,
// min-p and a given random number (ggq_sample_dev).
//
// Nothing is sorted.  What is kept of a row is a head of its tokens in order of
// their logits, so a border between two tokens says all, and the tokens are
// drawn in order of their indices.
//   A logit l has z = 8 log2(e) l / T in 64 bits; its bin is floor(z) counted
// down from the largest one's, its weight 2^(-bin / 8) * 2^(frac / 8), the
// second factor (1 .. 1.09) in 36 bits after the point: sums over a bin are
// integers, which no order of additions changes.
//   sample_bins_kernel: parts of 4096 tokens; a part counts its tokens and
// adds up their factors in 512 bins below its own largest (64 powers of two: what
// is below counts as nothing), count and sum in one 64-bit LDS atomic.
//   sample_pick_kernel: a workgroup a row adds up the parts' bins, finds the
// bin that holds the border and, only where the border is inside of a bin, looks
// through that bin's tokens (the parts that have any) by digits of their
// keys; then the part in which the running sum passes u, and the token in it.
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
};

struct SampleArgs {
    ggq_sample_params p;
    int parts;
    PartInfo* info;  // [n_rows][parts]
    u64* bins;       // [n_rows][parts][kBins]
};

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
};
__device__ __forceinline__ Bin bin_of(float l, double c) {
    const double z = (double)l * c, fl = floor(z);
    if (l == INFINITY) return Bin{INFINITY, u64(1) << 36};
    const double x = (z - fl) * (0.69314718055994530942 / 8.0);  // below 0.0867: the next term is 8e-14
    double e = 1.0 / 5040.0;
    e = fma(e, x, 1.0 / 720.0);
    e = fma(e, x, 1.0 / 120.0);
    e = fma(e, x, 1.0 / 24.0);
    e = fma(e, x, 1.0 / 6.0);
    e = fma(e, x, 0.5);
    e = fma(e, x, 1.0);
    e = fma(e, x, 1.0);
    // (a sum of 2^16 and more has its last bit at 2^-36)
    return Bin{fl, __builtin_bit_cast(u64, e + 65536.0) - __builtin_bit_cast(u64, 65536.0)};
}
// Bins that `at` lies below `top`, at most kRest.
__device__ __forceinline__ int below(double top, double at) {
    return at == top ? 0 : (int)fmin(top - at, (double)kRest);
}

__global__ __launch_bounds__(256) void sample_bins_kernel(SampleArgs a) {
    constexpr int V = kPart / 256;
    __shared__ u64 bins[kBins];
    __shared__ uint32_t red[4][3];
    const ggq_sample_params& p = a.p;
    const int tid = threadIdx.x, row = blockIdx.y, part = blockIdx.x, base = part * kPart;
    const float* x = p.logits + (int64_t)row * p.ld;
    const double c = eighths_of(p, row);
    float v[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int k = base + tid + 256 * i;
        v[i] = k < p.n_vocab ? x[k] : -INFINITY;
    }
    bins[tid] = 0;
    bins[tid + 256] = 0;
    uint32_t top = 0, at = 0xFFFFFFFFu, n = 0;
#pragma unroll
    for (int i = 0; i < V; i++) {
        if (!(v[i] > -INFINITY)) continue;
        const uint32_t k = key_of(v[i]);
        n++;
        if (k > top) {
            top = k;
            at = (uint32_t)(base + tid + 256 * i);
        }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t t = (uint32_t)__shfl_xor((int)top, o, 64), w = (uint32_t)__shfl_xor((int)at, o, 64);
        n += (uint32_t)__shfl_xor((int)n, o, 64);
        if (t > top || (t == top && w < at)) { top = t; at = w; }
    }
    if ((tid & 63) == 0) { red[tid >> 6][0] = top; red[tid >> 6][1] = at; red[tid >> 6][2] = n; }
    __syncthreads();
    n = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        n += red[i][2];
        if (red[i][0] > top || (red[i][0] == top && red[i][1] < at)) { top = red[i][0]; at = red[i][1]; }
    }
    const int64_t id = (int64_t)row * a.parts + part;
    const float mx = n ? of_key(top) : -INFINITY;
    const double first = n && c >= 0.0 ? bin_of(mx, c).top : -INFINITY;
    if (tid == 0) a.info[id] = PartInfo{first, mx, (int32_t)at, (int32_t)n, 0};
    if (c < 0.0) return;  // greedy rows need no bins
#pragma unroll
    for (int i = 0; i < V; i++) {
        if (!(v[i] > -INFINITY)) continue;
        const Bin b = bin_of(v[i], c);
        const int j = below(first, b.top);
        atomicAdd(&bins[j], (u64(1) << kCount) + (j == kRest ? 0 : b.factor));
    }
    __syncthreads();
    u64* out = a.bins + id * kBins;
    out[tid] = bins[tid];
    out[tid + 256] = bins[tid + 256];
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

// The border of what is kept: bins before `bin` whole, of `bin` the tokens with a larger key, and those
// with this key up to the index `last`.
struct Border {
    int bin;
    uint32_t key;
    uint32_t last;
};
__device__ __forceinline__ bool nearer(const Border& a, const Border& b) {
    return a.bin != b.bin ? a.bin < b.bin : a.key != b.key ? a.key > b.key : a.last < b.last;
}

constexpr int kThreads = 1024, kWaves = kThreads / 64;
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(SampleArgs a) {
    __shared__ u64 mass[kBins];       // factors of a bin, in units of 2^-36; digits' later
    __shared__ uint32_t count[kBins];
    __shared__ double tab[kBins];     // 2^(-j / 8)
    __shared__ int32_t shift[kMaxParts];
    __shared__ double pmass[kMaxParts];
    __shared__ u64 inside[kMaxParts];  // kept factors of the border's bin, of each part
    __shared__ uint32_t lkey[kList], lidx[kList];
    __shared__ double wave_d[kWaves];
    __shared__ uint32_t s_n, s_found, s_digit, s_need;
    __shared__ u64 s_left, s_mass;
    __shared__ double s_total;
    const ggq_sample_params& p = a.p;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.x;
    const float* x = p.logits + (int64_t)row * p.ld;
    const PartInfo* info = a.info + (int64_t)row * a.parts;
    const u64* bins = a.bins + (int64_t)row * a.parts * kBins;
    const double c = eighths_of(p, row);

    // the row's largest token, and how many there are
    uint32_t top = 0, at = 0xFFFFFFFFu, n_all = 0;
    if (tid < a.parts) {
        const PartInfo i = info[tid];
        if (i.count) { top = key_of(i.max); at = (uint32_t)i.at; n_all = (uint32_t)i.count; }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t t = (uint32_t)__shfl_xor((int)top, o, 64), w = (uint32_t)__shfl_xor((int)at, o, 64);
        n_all += (uint32_t)__shfl_xor((int)n_all, o, 64);
        if (t > top || (t == top && w < at)) { top = t; at = w; }
    }
    if (lane == 0) { lkey[wave] = top; lidx[wave] = at; count[wave] = n_all; }
    __syncthreads();
    n_all = 0;
#pragma unroll
    for (int i = 0; i < kWaves; i++) {
        n_all += count[i];
        if (lkey[i] > top || (lkey[i] == top && lidx[i] < at)) { top = lkey[i]; at = lidx[i]; }
    }
    if (c < 0.0 || n_all == 0) {
        if (tid == 0) {
            p.token[row] = n_all ? (int32_t)at : 0;
            if (p.prob) p.prob[row] = n_all ? 1.0f : 0.0f;
        }
        return;
    }
    const float mx = of_key(top);
    const double first = bin_of(mx, c).top;
    __syncthreads();
    if (tid < kBins) tab[tid] = step_down(tid);
    if (tid < a.parts) {
        const PartInfo i = info[tid];
        shift[tid] = i.count ? below(first, i.top) : kRest;
        inside[tid] = 0;
    }
    __syncthreads();

    Border border{kRest, 0u, 0xFFFFFFFFu};  // all that has a weight
    const int top_k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f, min_p = p.min_p ? p.min_p[row] : 0.0f;
    const bool by_k = top_k > 0 && (uint32_t)top_k < n_all, by_p = top_p < 1.0f, by_m = min_p > 0.0f;

    // f(key, index) for the tokens of a bin: from the list, or from the row's parts that have any
    int listed = -1;
    uint32_t n_listed = 0;
    auto scan = [&](int bin, auto f) {
        for (int q = wave; q < a.parts; q += kWaves) {
            const int j = bin - shift[q];
            if (j < 0 || !(uint32_t)(bins[(int64_t)q * kBins + j] >> kCount)) continue;
            const int base = q * kPart;
            for (int i0 = 0; i0 < kPart; i0 += 64 * 16) {
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int k = base + i0 + 64 * i + lane;
                    v[i] = k < p.n_vocab ? x[k] : -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (v[i] > -INFINITY && below(first, bin_of(v[i], c).top) == bin) f(key_of(v[i]), (uint32_t)(base + i0 + 64 * i + lane));
            }
        }
    };
    auto list = [&](int bin, uint32_t n) {  // (n: the bin's tokens)
        if (n > kList) { listed = -1; return; }
        if (listed == bin) return;
        __syncthreads();
        if (tid == 0) s_n = 0;
        __syncthreads();
        scan(bin, [&](uint32_t key, uint32_t idx) {
            const uint32_t i = atomicAdd(&s_n, 1u);
            if (i < kList) { lkey[i] = key; lidx[i] = idx; }
        });
        __syncthreads();
        n_listed = min(s_n, (uint32_t)kList);
        listed = bin;
    };
    auto each = [&](int bin, auto f) {
        if (listed == bin)
            for (uint32_t i = tid; i < n_listed; i += kThreads) f(lkey[i], lidx[i]);
        else scan(bin, f);
    };
    // Digits of 8 bits, from the highest: the shortest head of the bin's tokens that has `need` of them, or factors of
    // `left` (whichever is asked for; the other one 0).
    __shared__ u64 dmass[256];
    __shared__ uint32_t dcount[256];
    auto select = [&](int bin, uint32_t n, uint32_t need, u64 left, bool by_mass) -> Border {
        list(bin, n);
        uint32_t prefix = 0;
        uint32_t equal = 0;
        for (int s = 24; s >= 0; s -= 8) {
            __syncthreads();
            if (tid < 256) { dmass[tid] = 0; dcount[tid] = 0; }
            __syncthreads();
            each(bin, [&](uint32_t key, uint32_t) {
                if (s < 24 && key >> (s + 8) != prefix) return;
                const uint32_t d = key >> s & 255u;
                atomicAdd(&dcount[d], 1u);
                if (by_mass) atomicAdd(&dmass[d], bin_of(of_key(key), c).factor);
            });
            __syncthreads();
            if (wave == 0) {  // four digits a lane, the largest first
                uint32_t own = 0;
                u64 ownm = 0;
                for (int i = 0; i < 4; i++) { own += dcount[255 - 4 * lane - i]; ownm += dmass[255 - 4 * lane - i]; }
                uint32_t run = own;
                u64 runm = ownm;
                for (int o = 1; o < 64; o <<= 1) {
                    const uint32_t t = (uint32_t)__shfl_up((int)run, o, 64);
                    const u64 tm = __shfl_up(runm, o, 64);
                    if (lane >= o) { run += t; runm += tm; }
                }
                uint32_t before = run - own, hb = 0;
                u64 beforem = runm - ownm, hm = 0;
                int hit = -1, last = -1;
                for (int i = 0; i < 4; i++) {
                    const int d = 255 - 4 * lane - i;
                    if (dcount[d]) {
                        if (hit < 0 && (by_mass ? beforem + dmass[d] >= left : before + dcount[d] >= need)) { hit = d; hb = before; hm = beforem; }
                        last = d;
                    }
                    before += dcount[d];
                    beforem += dmass[d];
                }
                const u64 any = __ballot(hit >= 0), some = __ballot(last >= 0);
                const int l = any ? __ffsll(any) - 1 : 63 - __builtin_clzll(some);
                const int d = __shfl(any ? hit : last, l, 64);
                hb = (uint32_t)__shfl((int)hb, l, 64);
                hm = __shfl(hm, l, 64);
                if (lane == 0) {  // (none: rounding left something over, so all of them)
                    s_digit = (uint32_t)d;
                    s_need = need - hb;
                    s_left = any ? left - hm : dmass[d];
                    s_found = dcount[d];
                }
            }
            __syncthreads();
            prefix = prefix << 8 | s_digit;
            need = s_need;
            left = s_left;
            equal = s_found;
        }
        const uint32_t key = prefix;
        if (by_mass) {
            const u64 one = bin_of(of_key(key), c).factor;
            need = (uint32_t)min((left + one - 1) / one, (u64)equal);
            if (need == 0) need = 1;
        }
        if (need >= equal) return Border{bin, key, 0xFFFFFFFFu};
        // tokens that are alike: the ones of lowest index
        prefix = 0;
        for (int s = 16; s >= 0; s -= 8) {
            __syncthreads();
            if (tid < 256) dcount[tid] = 0;
            __syncthreads();
            each(bin, [&](uint32_t k, uint32_t idx) {
                if (k != key || (s < 16 && idx >> (s + 8) != prefix)) return;
                atomicAdd(&dcount[idx >> s & 255u], 1u);
            });
            __syncthreads();
            if (wave == 0) {
                uint32_t own = 0;
                for (int i = 0; i < 4; i++) own += dcount[4 * lane + i];
                uint32_t run = own;
                for (int o = 1; o < 64; o <<= 1) {
                    const uint32_t t = (uint32_t)__shfl_up((int)run, o, 64);
                    if (lane >= o) run += t;
                }
                uint32_t before = run - own, hb = 0;
                int hit = -1;
                for (int i = 0; i < 4; i++) {
                    if (hit < 0 && before + dcount[4 * lane + i] >= need) { hit = 4 * lane + i; hb = before; }
                    before += dcount[4 * lane + i];
                }
                const u64 any = __ballot(hit >= 0);  // (need is at most what there is)
                const int l = any ? __ffsll(any) - 1 : 0;
                hit = __shfl(hit, l, 64);
                hb = (uint32_t)__shfl((int)hb, l, 64);
                if (lane == 0) { s_digit = (uint32_t)max(hit, 0); s_need = need - hb; }
            }
            __syncthreads();
            prefix = prefix << 8 | s_digit;
            need = s_need;
        }
        return Border{bin, key, prefix};
    };
    auto kept_in = [&](const Border& b, uint32_t key, uint32_t idx) { return key > b.key || (key == b.key && idx <= b.last); };
    // factors of the border's bin that are kept, in all
    auto mass_in = [&](const Border& b, uint32_t n) -> u64 {
        list(b.bin, n);
        __syncthreads();
        if (tid == 0) s_mass = 0;
        __syncthreads();
        each(b.bin, [&](uint32_t key, uint32_t idx) {
            if (kept_in(b, key, idx)) atomicAdd(&s_mass, bin_of(of_key(key), c).factor);
        });
        __syncthreads();
        return s_mass;
    };

    if (by_k || by_p || by_m) {
        // the row's bins
        for (int h = 0; h < 2; h++) {  // (two threads a bin: halves of the parts)
            const int b = tid & (kBins - 1), half = tid >> 9;
            if (h == 0) {
                uint32_t n = 0;
                u64 m = 0;
                if (b < kRest)
                    for (int q = half; q < a.parts; q += 2) {
                        const int j = b - shift[q];
                        if (j < 0) continue;
                        const u64 w = bins[(int64_t)q * kBins + j];
                        n += (uint32_t)(w >> kCount);
                        m += w & ((u64(1) << kCount) - 1);
                    }
                if (half == 0) { count[b] = n; mass[b] = m; }
                __syncthreads();
                if (half == 1) { count[b] += n; mass[b] += m; }
                __syncthreads();
            }
        }
        // the first bin in which a running sum reaches something, by one wavefront: eight bins a lane
        auto reach_count = [&](uint32_t k, int& bin, uint32_t& before) {
            uint32_t own = 0;
            for (int i = 0; i < 8; i++) own += 8 * lane + i < kRest ? count[8 * lane + i] : 0;
            uint32_t run = own;
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t t = (uint32_t)__shfl_up((int)run, o, 64);
                if (lane >= o) run += t;
            }
            uint32_t b = run - own;
            int hit = kRest;
            uint32_t hb = 0;
            for (int i = 0; i < 8; i++) {
                const int j = 8 * lane + i;
                const uint32_t n = j < kRest ? count[j] : 0;
                if (hit == kRest && j < kRest && b + n >= k) { hit = j; hb = b; }
                b += n;
            }
            const u64 any = __ballot(hit < kRest);
            if (!any) { bin = kRest; before = 0; return; }
            const int l = __ffsll(any) - 1;
            bin = __shfl(hit, l, 64);
            before = (uint32_t)__shfl((int)hb, l, 64);
        };
        u64 kmass = 0;  // factors kept of the border's bin by top-k
        if (by_k) {
            int bin;
            uint32_t before;
            reach_count((uint32_t)top_k, bin, before);
            if (bin < kRest) {
                const uint32_t need = (uint32_t)top_k - before, n = count[bin];
                if (need < n) {
                    border = select(bin, n, need, 0, false);
                    kmass = mass_in(border, n);
                } else {
                    border = Border{bin, 0u, 0xFFFFFFFFu};
                    kmass = mass[bin];
                }
            }
        }
        if (by_p) {
            // sums of weights up to each bin
            double own = 0.0, w[8];
            for (int i = 0; i < 8; i++) {
                const int j = 8 * lane + i;
                const u64 m = j >= kRest || j > border.bin ? 0 : j == border.bin ? kmass : mass[j];
                w[i] = (double)m * tab[min(j, kRest)];
                own += w[i];
            }
            double run = own;
            for (int o = 1; o < 64; o <<= 1) {
                const double t = __shfl_up(run, o, 64);
                if (lane >= o) run += t;
            }
            const double want = fmax(0.0, (double)top_p) * __shfl(run, 63, 64);
            double b = run - own, hb = 0.0;
            int hit = kRest;
            for (int i = 0; i < 8; i++) {
                const int j = 8 * lane + i;
                if (hit == kRest && j < kRest && count[j] && j <= border.bin && b + w[i] >= want) { hit = j; hb = b; }
                b += w[i];
            }
            const u64 any = __ballot(hit < kRest);
            if (any) {
                const int l = __ffsll(any) - 1;
                const int bin = __shfl(hit, l, 64);
                hb = __shfl(hb, l, 64);
                // in the bin's own units, rounded up
                const double in = (want - hb) / tab[bin];
                const u64 left = in > 0.0 ? (u64)ceil(in) : 0;
                const Border n = select(bin, count[bin], 0, left, true);
                if (nearer(n, border)) border = n;
            }
        }
        if (by_m) {
            // the smallest value with (value - largest) / T >= ln min_p
            const float t = p.temperature ? p.temperature[row] : 1.0f;
            const double lim = min_p >= 1.0f ? 0.0 : (double)t * log((double)min_p);
            float v = (float)((double)mx + lim);
            if (!(v <= mx) || mx == INFINITY) v = mx;
            uint32_t key = key_of(v);
            if (v > -INFINITY && mx < INFINITY) {
                while (key < top && (double)of_key(key) - (double)mx < lim) key++;
                while (key > 0x00800000u && (double)of_key(key - 1) - (double)mx >= lim) key--;
            }
            v = of_key(key);
            if (v > -INFINITY) {
                const int bin = below(first, bin_of(v, c).top);
                const Border n{bin, key, 0xFFFFFFFFu};
                if (bin < kRest && nearer(n, border)) border = n;
            }
        }
        // what is kept of the border's bin, by parts
        if (border.bin < kRest) {
            list(border.bin, count[border.bin]);
            __syncthreads();
            each(border.bin, [&](uint32_t key, uint32_t idx) {
                if (kept_in(border, key, idx)) atomicAdd(&inside[idx / kPart], bin_of(of_key(key), c).factor);
            });
        }
        __syncthreads();
    }

    // kept weights of the parts, a wavefront a part
    for (int q = wave; q < a.parts; q += kWaves) {
        const int s = shift[q];
        double m = 0.0;
        if (s < kRest)
#pragma unroll
            for (int i = 0; i < kBins / 64; i++) {
                const int j = 64 * i + lane;
                const u64 w = bins[(int64_t)q * kBins + j] & ((u64(1) << kCount) - 1);
                if (j < kRest && j + s < border.bin) m = fma((double)w, tab[j + s], m);
            }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) m += __shfl_xor(m, o, 64);
        if (lane == 0) pmass[q] = m + (border.bin < kRest ? (double)inside[q] * tab[border.bin] : 0.0);
    }
    __syncthreads();
    // running sums of the parts by one wavefront: the first that passes u times the whole (else the last that has any)
    float u = p.u[row];
    if (!(u > 0.0f)) u = 0.0f;
    if (wave == 0) {
        const int per = (a.parts + 63) / 64;
        double own = 0.0;
        for (int i = 0; i < per; i++) own += per * lane + i < a.parts ? pmass[per * lane + i] : 0.0;
        double run = own;
        for (int o = 1; o < 64; o <<= 1) {
            const double t = __shfl_up(run, o, 64);
            if (lane >= o) run += t;
        }
        const double total = __shfl(run, 63, 64), want = (double)u * total;
        double b = run - own, hb = 0.0;
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
        const u64 any = __ballot(hit >= 0), some = __ballot(last >= 0);
        const int l = any ? __ffsll(any) - 1 : 63 - __builtin_clzll(some);
        const int q = __shfl(any ? hit : last, l, 64);
        const double before = __shfl(any ? hb : lb, l, 64);
        if (lane == 0) {
            s_found = (uint32_t)q;
            s_total = total;
            wave_d[0] = want - before;
        }
    }
    __syncthreads();
    const int part = (int)s_found;
    const double total = s_total, want = wave_d[0];
    __syncthreads();
    // and the token in it: four in a row a thread
    const int base = part * kPart + 4 * tid;
    double w[4], own = 0.0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int k = base + i;
        const float l = k < p.n_vocab ? x[k] : -INFINITY;
        w[i] = 0.0;
        if (l > -INFINITY) {
            const Bin b = bin_of(l, c);
            const int j = below(first, b.top);
            if (j < kRest && (j < border.bin || (j == border.bin && kept_in(border, key_of(l), (uint32_t)k))))
                w[i] = (double)b.factor * tab[j];
        }
        own += w[i];
    }
    double run = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double t = __shfl_up(run, o, 64);
        if (lane >= o) run += t;
    }
    if (lane == 63) wave_d[wave] = run;
    if (tid == 0) { s_found = 0xFFFFFFFFu; s_need = 0; }
    __syncthreads();
    double b = run - own;
    for (int i = 0; i < wave; i++) b += wave_d[i];
    uint32_t hit = 0xFFFFFFFFu, last = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (w[i] > 0.0) {
            if (hit == 0xFFFFFFFFu && b + w[i] > want) hit = (uint32_t)(base + i);
            last = (uint32_t)(base + i) + 1;
        }
        b += w[i];
    }
    if (hit != 0xFFFFFFFFu) atomicMin(&s_found, hit);
    if (last) atomicMax(&s_need, last);
    __syncthreads();
    const uint32_t token = s_found != 0xFFFFFFFFu ? s_found : s_need - 1;
#pragma unroll
    for (int i = 0; i < 4; i++)
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
    return info_bytes(p) + sizeof(u64) * kBins * (size_t)p.n_rows * parts_of(p);
}
hipError_t launch_sample(const ggq_sample_params& p, void* ws, hipStream_t s) {
    SampleArgs a{p, parts_of(p), (PartInfo*)ws, (u64*)((char*)ws + info_bytes(p))};
    sample_bins_kernel<<<dim3((unsigned)a.parts, (unsigned)p.n_rows), 256, 0, s>>>(a);
    sample_pick_kernel<<<dim3((unsigned)p.n_rows), kThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace ggq
