// vbs_kern_rope_axes.hip — rotary positions with several axes for n tokens, and
// their K and V rows into the f16 cache, in one launch.
//
// Pair p (elements 2p, 2p + 1, as src/vbs_host_math.h:38-51) of every head of
// token i turns by a = pos[axis(p)][i] * theta^(-2p / hd), axis(p) the axis whose
// section of pairs holds p. q is rotated in place; k is rotated, and k and v
// are stored with the cache's rounding (src/vbs_host_math.h:150-159).
//
// The angle of a far position needs more than 24 bits (position 1e6 times a
// frequency of 1 leaves 0.06 rad of f32's spacing), so it is formed in 64 bits,
// reduced there to [-pi/4, pi/4] and its sine and cosine are taken there too;
// only they are rounded to f32 (half a step, 2^-24). The reference's own
// rotation (vbs_gfx950_rope) forms its angles in f32 and so differs from this
// one by up to position * 2^-23 rad.
#include <math.h>

#include "vbs_dev_common.h"
#include "vbs_steps.h"

namespace vbs {

struct RopeFreqs {
    double f[kRopeMaxPairs];
};

// (cos a, sin a): a = k pi/2 + r with pi/2 in two parts (53 and 53 bits). k times the first part and a are both multiples
// of 2^-52 while |a| < 2^52, so the first difference is exact; what the parts lack of pi/2 is 2^-107 |k|. k is off by one
// at most where |a| nears 2^52 (theta of 2^-21; for theta >= 1 |a| is 2^31 at most and |r| <= pi/4). Then the Taylor
// series of sine and cosine, whose first dropped terms are r^15 / 15! < 2.1e-14 and r^16 / 16! < 1.1e-15 for
// |r| <= pi/4 and below 1e-8 for the |r| < 1.9 of the farthest.
__device__ __forceinline__ float2 cos_sin(double a) {
    const double k = rint(a * 0.63661977236758134308);  // 2 / pi
    double r = fma(k, -1.5707963267948965580, a);
    r = fma(k, -6.1232339957367660359e-17, r);
    const double z = r * r;
    double s = 1.0 / 6227020800.0;
    s = fma(s, z, -1.0 / 39916800.0);
    s = fma(s, z, 1.0 / 362880.0);
    s = fma(s, z, -1.0 / 5040.0);
    s = fma(s, z, 1.0 / 120.0);
    s = fma(s, z, -1.0 / 6.0);
    s = fma(s * z, r, r);
    double c = -1.0 / 87178291200.0;
    c = fma(c, z, 1.0 / 479001600.0);
    c = fma(c, z, -1.0 / 3628800.0);
    c = fma(c, z, 1.0 / 40320.0);
    c = fma(c, z, -1.0 / 720.0);
    c = fma(c, z, 1.0 / 24.0);
    c = fma(c, z, -0.5);
    c = fma(c, z, 1.0);
    const int quad = (int)((long long)k & 3);
    const double cs = quad & 1 ? s : c, sn = quad & 1 ? c : s;
    return make_float2((float)(quad == 1 || quad == 2 ? -cs : cs), (float)(quad >= 2 ? -sn : sn));
}

// grid (parts, tokens): a workgroup takes kRopeRows of a token's nqh + nkh heads; what it rotates is on its way while
// the angles are formed.
constexpr uint32_t kRopeRows = 8, kRopeMine = kRopeRows * kRopeMaxPairs / 256u;

__global__ __launch_bounds__(256) void k_rope_axes(RopeAxesArgs a, RopeFreqs fr) {
    __shared__ float2 cs[kRopeMaxPairs];
    const uint32_t pairs = a.hd / 2u, i = blockIdx.y, t = threadIdx.x;
    const uint32_t heads = (a.q ? a.nqh : 0u) + (a.k ? a.nkh : 0u), r0 = blockIdx.x * kRopeRows;
    const uint32_t mine = min(kRopeRows, heads - r0) * pairs, nq = a.q ? a.nqh : 0u;
    float x0[kRopeMine], x1[kRopeMine], v0[kRopeMine], v1[kRopeMine];
#pragma unroll
    for (uint32_t n = 0; n < kRopeMine; n++) {
        const uint32_t e = t + 256u * n, h = r0 + e / pairs, d = 2u * (e % pairs);
        if (e >= mine) break;
        const float *x = h < nq ? a.q + (uint64_t)i * a.q_stride + (uint64_t)h * a.hd + d
                                : a.k + (uint64_t)i * a.kv_stride + (uint64_t)(h - nq) * a.hd + d;
        x0[n] = x[0], x1[n] = x[1];
        if (h >= nq) {
            const float *v = a.v + (uint64_t)i * a.kv_stride + (uint64_t)(h - nq) * a.hd + d;
            v0[n] = v[0], v1[n] = v[1];
        }
    }
    if (t < pairs) {
        uint32_t axis = 0;
        while (t >= a.end[axis]) axis++;
        cs[t] = cos_sin((double)a.pos[(uint64_t)axis * a.n + i] * fr.f[t]);
    }
    __syncthreads();
#pragma unroll
    for (uint32_t n = 0; n < kRopeMine; n++) {
        const uint32_t e = t + 256u * n, h = r0 + e / pairs, p = e % pairs;
        if (e >= mine) break;
        const float2 w = cs[p];
        const float y0 = __fsub_rn(__fmul_rn(x0[n], w.x), __fmul_rn(x1[n], w.y));
        const float y1 = __fadd_rn(__fmul_rn(x0[n], w.y), __fmul_rn(x1[n], w.x));
        if (h < nq) {
            float *x = a.q + (uint64_t)i * a.q_stride + (uint64_t)h * a.hd + 2u * p;
            x[0] = y0, x[1] = y1;
            continue;
        }
        const uint64_t to = ((uint64_t)i * a.nkh + (h - nq)) * a.hd + 2u * p;
        a.kc[to] = vbs_f2h(y0);
        a.kc[to + 1u] = vbs_f2h(y1);
        a.vc[to] = vbs_f2h(v0[n]);
        a.vc[to + 1u] = vbs_f2h(v1[n]);
    }
}

hipError_t launch_rope_axes(const RopeAxesArgs &a, float theta, hipStream_t s) {
    const uint32_t pairs = a.hd / 2u, heads = (a.q ? a.nqh : 0u) + (a.k ? a.nkh : 0u);
    // A thread's last table, by its values: 64 powers anew are 0.4 us of a call's 5.4 (back to back; one token, 32/8 heads
    // of 128), which two thetas in turn pay. One power and products in 64 bits of mantissa instead, with nothing kept:
    // 5.3 back to back, but 9.7 for 8.6 between other work of the host.
    static thread_local RopeFreqs fr;
    static thread_local float fr_theta = 0.f;
    static thread_local uint32_t fr_hd = 0;
    if (fr_theta != theta || fr_hd != a.hd) {
        for (uint32_t p = 0; p < pairs; p++) fr.f[p] = pow((double)theta, -2.0 * p / a.hd);
        fr_theta = theta;
        fr_hd = a.hd;
    }
    k_rope_axes<<<dim3((heads + kRopeRows - 1u) / kRopeRows, a.n), 256, 0, s>>>(a, fr);
    return hipGetLastError();
}

}  // namespace vbs
