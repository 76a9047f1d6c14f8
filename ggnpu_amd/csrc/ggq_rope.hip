// ggq_rope.hip -- rotary positions of query and key heads, behind an optional
// RMSNorm of each head, in one pass over the rows.
//
// A head of head_dim values is taken by LPH lanes (head_dim / 8, rounded up to
// a power of two) of 8 values each, so a wavefront has 64 / LPH heads in flight and the norm's
// sum of squares stays inside a group of lanes.  The lanes of the rotated part
// hold both values of four pairs (two 16-byte runs rot_dim / 2 apart, or 8
// consecutive values), the others 8 values that pass through: every value is
// read and written by one lane, which makes in-place calls safe.
//
// The angle of pair i at position p is p * turns_i turns.  The product is taken
// in 64 bits and its whole turns are dropped there, so the 32-bit sine and
// cosine see an angle within half a turn at any position; what that loses of the
// angle (up to 2^-25 of half a turn) is put back along the tangent.  A lane's pairs
// are the same for all heads of a row: they are made once and used for
// `passes` groups of heads.
//
// Bound: HBM (2049 rows of 24 heads of 128 with norms: 50 MB in 11.2 us, 4.5
// TB/s); one token 3.8 us, a launch with two dependent loads.
#include "ggq_attn.h"
#include "ggq_launch.h"

namespace ggq {
namespace {

struct alignas(8) Half4 { _Float16 v[4]; };

template <int LPH>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, int heads, int passes) {
    constexpr int HPW = 64 / LPH;  // heads of a wavefront's pass
    const int lane = threadIdx.x & 63, u = lane % LPH, sub = lane / LPH;
    const int chunks = (heads + HPW * passes - 1) / (HPW * passes);
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = (int)(w / chunks), h0 = (int)(w % chunks) * HPW * passes;
    if (t >= a.n_tok) return;
    const int hd = a.head_dim, rot = a.rot_dim;
    const bool live = u * 8 < hd, turned = u * 8 < rot;
    // the two runs of 4 values
    const int i0 = !turned || a.layout == GGQ_ROPE_INTERLEAVED ? 8 * u : 4 * u;
    const int i1 = !turned || a.layout == GGQ_ROPE_INTERLEAVED ? 8 * u + 4 : rot / 2 + 4 * u;
    float cs[4], sn[4];
    if (turned) {
        const double p = (double)a.pos[t];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const double turn = p * a.turns[4 * u + j], half = 2.0 * (turn - rint(turn));
            const float at = (float)half, rest = (float)((half - (double)at) * 3.14159265358979323846);
            float s, c;
            sincospif(at, &s, &c);
            cs[j] = fmaf(-s, rest, c) * a.mag;
            sn[j] = fmaf(c, rest, s) * a.mag;
        }
    }
    const int n0 = a.set[0].n_head;
    for (int i = 0; i < passes; i++) {
        const int h = h0 + i * HPW + sub;
        if (h0 + i * HPW >= heads) break;  // (the same for the whole wavefront)
        const ggq_rope_heads& set = h < n0 ? a.set[0] : a.set[1];
        const int hs = h < n0 ? h : h - n0;
        const bool on = live && h < heads;
        float4 x0 = {0, 0, 0, 0}, x1 = {0, 0, 0, 0};
        if (on) {
            const float* x = set.x + (int64_t)t * set.ldx + (int64_t)hs * hd;
            x0 = *(const float4*)(x + i0);
            x1 = *(const float4*)(x + i1);
        }
        const float* nw = on ? set.norm_w : nullptr;
        if (a.set[0].norm_w || a.set[1].norm_w) {
            float q = x0.x * x0.x + x0.y * x0.y + x0.z * x0.z + x0.w * x0.w + x1.x * x1.x + x1.y * x1.y +
                      x1.z * x1.z + x1.w * x1.w;
#pragma unroll
            for (int o = 1; o < LPH; o <<= 1) q += __shfl_xor(q, o, 64);
            if (nw) {
                const float r = 1.0f / sqrtf(q / (float)hd + a.eps);
                const float4 w0 = *(const float4*)(nw + i0), w1 = *(const float4*)(nw + i1);
                x0 = make_float4(x0.x * r * w0.x, x0.y * r * w0.y, x0.z * r * w0.z, x0.w * r * w0.w);
                x1 = make_float4(x1.x * r * w1.x, x1.y * r * w1.y, x1.z * r * w1.z, x1.w * r * w1.w);
            }
        }
        if (!on) continue;
        float v[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
        if (turned) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int ia = a.layout == GGQ_ROPE_INTERLEAVED ? 2 * j : j;
                const int ib = a.layout == GGQ_ROPE_INTERLEAVED ? 2 * j + 1 : j + 4;
                const float p = v[ia], q = v[ib];
                v[ia] = fmaf(p, cs[j], -(q * sn[j]));
                v[ib] = fmaf(p, sn[j], q * cs[j]);
            }
        }
        const int64_t o = (int64_t)t * set.ldo + (int64_t)hs * hd;
        if (set.out_type == GGQ_TYPE_F32) {
            float* y = (float*)set.out + o;
            *(float4*)(y + i0) = make_float4(v[0], v[1], v[2], v[3]);
            *(float4*)(y + i1) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            _Float16* y = (_Float16*)set.out + o;
            *(Half4*)(y + i0) = Half4{{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]}};
            *(Half4*)(y + i1) = Half4{{(_Float16)v[4], (_Float16)v[5], (_Float16)v[6], (_Float16)v[7]}};
        }
    }
}

template <int LPH> hipError_t launch(const RopeArgs& a, hipStream_t s) {
    constexpr int HPW = 64 / LPH;
    const int heads = a.set[0].n_head + (a.n_sets > 1 ? a.set[1].n_head : 0);
    const int64_t groups = (int64_t)(heads + HPW - 1) / HPW;  // passes of a row
    // one pass a wavefront while that leaves CUs without work, up to 4 then
    int passes = 1;
    while (passes < 4 && groups * a.n_tok / (2 * passes) >= (int64_t)cu_count() * 16) passes *= 2;
    const int64_t chunks = (groups + passes - 1) / passes, waves = chunks * a.n_tok;
    rope_kernel<LPH><<<dim3((unsigned)((waves + 3) / 4)), 256, 0, s>>>(a, heads, passes);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_rope(const RopeArgs& a, hipStream_t s) {
    const int lanes = a.head_dim / 8;
    if (lanes <= 8) return launch<8>(a, s);
    if (lanes <= 16) return launch<16>(a, s);
    if (lanes <= 32) return launch<32>(a, s);
    return launch<64>(a, s);
}

}  // namespace ggq
