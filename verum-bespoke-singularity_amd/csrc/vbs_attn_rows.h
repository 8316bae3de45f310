// vbs_attn_rows.h — what the kernels of several query rows over the f16 cache
// share (vbs_kern_attn_rows.hip): which slots a row sees, its scores, and one row in
// plain f32 for rows whose sums are not finite.
#pragma once

#include "vbs_dev_common.h"
#include "vbs_steps.h"

namespace vbs {

constexpr float kLog2e = 1.44269504088896341f;

typedef _Float16 rh8 __attribute__((ext_vector_type(8)));
typedef _Float16 rh2 __attribute__((ext_vector_type(2)));
typedef float rf2 __attribute__((ext_vector_type(2)));
typedef float rf4 __attribute__((ext_vector_type(4)));
typedef uint32_t ru4 __attribute__((ext_vector_type(4)));

// r / group, the token of row r of a kv head: r + 1/2 is exact, at least 1/2 / group from where the quotient turns, and
// the two roundings lose less than 2^20 / group * 2^-23 (rows are fewer than 2^20).
__device__ __forceinline__ uint32_t row_token(const RowsArgs &a, uint32_t r) {
    return (uint32_t)(((float)r + 0.5f) * a.rgroup);
}

// Whether row i (slot past + i) sees slot j.
__device__ __forceinline__ bool row_sees(const RowsArgs &a, uint32_t i, uint32_t j) {
    if (a.mask) {
        if (j < a.past) return true;
        const uint32_t t = j - a.past;
        return (a.mask[(uint64_t)i * a.words + (t >> 6)] >> (t & 63u)) & 1u;
    }
    if (j > a.past + i && j >= a.prefix) return false;
    return !a.docs || a.docs[j] == a.docs[a.past + i];
}
// The slots behind the last that row i can see.
__host__ __device__ __forceinline__ uint32_t row_end(const RowsArgs &a, uint32_t i) {
    if (a.mask) return a.past + a.n;
    const uint32_t own = a.past + i + 1u;
    return own > a.prefix ? own : a.prefix;
}

// tanh by an odd polynomial on |x| < kTanhPoly (off by at most 1.3e-8 of the value, at
// 0.78, and by 1.4 of f32's half steps with its own roundings), and as
// 1 - 2 / (e^(2 |x|) + 1) beyond, where that loses less than 4 half steps.
constexpr float kTanhPoly = 0.8f;
__device__ __forceinline__ float tanh_poly(float x) {
    const float z = x * x;
    float p = 0.0015847564209252596f;
    p = fmaf(p, z, -0.0074095577001571655f);
    p = fmaf(p, z, 0.02130299061536789f);
    p = fmaf(p, z, -0.05385233089327812f);
    p = fmaf(p, z, 0.13332220911979675f);
    p = fmaf(p, z, -0.33333298563957214f);
    return fmaf(x, z * p, x);
}
__device__ __forceinline__ float tanh_any(float x) {
    const float e = __builtin_amdgcn_exp2f(fabsf(x) * (2.f * kLog2e));
    const float far = fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f);
    return fabsf(x) < kTanhPoly ? tanh_poly(x) : copysignf(far, x);
}

// The score (natural units) from scale q.k: capped, less the distance's share.
__device__ __forceinline__ float row_far(float s, float slope, uint32_t at, uint32_t j) {
    return fmaf(-slope, fabsf((float)(int32_t)(at - j)), s);  // (slots are at most 2^31)
}
// The score capped. s / cap is a subnormal of few bits where the cap is far above s (and 1 / cap from 2^126 on): from
// kFarCap on a score below 2^-13 of the cap is left as it is, of which the cap takes less than (s / cap)^2 / 3 < 2^-27.
constexpr float kFarCap = 0x1p40f;
__device__ __forceinline__ float capped(const RowsArgs &a, float s) {
    const float t = a.cap * tanh_any(s * a.rcap);
    return a.cap >= kFarCap && fabsf(s) < a.cap * 0x1p-13f ? s : t;
}
__device__ __forceinline__ float row_score(const RowsArgs &a, float s, float slope, uint32_t at, uint32_t j) {
    if (a.cap > 0.f) s = capped(a, s);
    return a.slopes ? row_far(s, slope, at, j) : s;
}

// The score from a product x of the matrix cores (x c1: scale q.k), in units of score_unit: by the operations of RowTile's
// step one for one, so that the weights that k_mass adds are the numbers that l counted, at any size of a score.
__device__ __forceinline__ float score_unit(const RowsArgs &a) { return a.cap > 0.f && a.cap < kFarCap && !a.slopes ? a.cap : 1.f; }
__device__ __forceinline__ float parts_score(const RowsArgs &a, float x, float c1, float slope, uint32_t at, uint32_t j) {
    if (a.cap >= kFarCap) {
        x = capped(a, x * c1);
    } else if (a.cap > 0.f) {
        x = tanh_any(x * (c1 * a.rcap));
        if (a.slopes) x *= a.cap;
    } else {
        x *= c1;
    }
    return a.slopes ? row_far(x, slope, at, j) : x;
}

__device__ __forceinline__ float row_dot(const float *q, const uint16_t *k, uint32_t hd) {
    float dot = 0.f;
    for (uint32_t d = 0; d < hd; d++) dot = fmaf(q[d], h2f(k[d]), dot);
    return dot;
}

// A maximum (in units of log2) from which a row is taken in f32 products and rounded scores (row_whole). The matrix-core
// path subtracts the rounded maximum from products that are not rounded: what that leaves, up to half a step of m, is
// the same for every weight of the row and cancels as long as the weights hold it. From 2^24 on it reaches one and
// more in log2 and the weights leave f16's range: such rows came out as 0 or not finite.
constexpr float kFarScore = 0x1p24f;
__device__ __forceinline__ bool far_row(float m) { return fabsf(m) > kFarScore && m > -INFINITY; }
// Beyond this maximum a row that row_whole took is marked (its sum l goes on with its sign turned): its weights have to
// come from the same f32 scores again, which differ from the matrix cores' by about 2^-22 of their size.
constexpr float kMarkScore = 0x1p12f;

// Row i, q head h over the slots [s0, s1), by one whole wave in f32 products: the
// scores of 64 slots at a time, a slot per lane, a running maximum and sum, then
// the lanes take the dims (lane + 64 c in acc[c]). For rows whose sums came out not
// finite: an infinity in q or K meets the two f16 parts of the matrix-core path
// as inf - inf or 0 * inf, and one in V the weight 0 of the rows that do not see
// it. Here an unseen slot is never touched. And for rows of far scores: y is rounded
// before the maximum is taken off, so that the greatest weighs exactly 1. m is in units of
// log2, as the scores of the slots it sees, that go to scores[j] (if not NULL).
template <uint32_t HD>
__device__ __forceinline__ void row_whole(const RowsArgs &a, uint32_t i, uint32_t h, uint32_t s0, uint32_t s1,
                                          uint32_t lane, float &m_out, float &l_out, float (&acc)[(HD + 63) / 64],
                                          float *scores = nullptr) {
    const uint32_t kvh = h / a.group;
    const float *q = a.q + (uint64_t)i * a.q_stride + (uint64_t)h * a.hd;
    const uint64_t rstride = (uint64_t)a.nkh * a.hd, base = (uint64_t)kvh * a.hd;
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (uint32_t c = 0; c < (HD + 63u) / 64u; c++) acc[c] = 0.f;
    for (uint32_t j0 = s0; j0 < s1; j0 += 64u) {
        const uint32_t j = j0 + lane;
        const bool sees = j < s1 && j < row_end(a, i) && row_sees(a, i, j);
        float y = -INFINITY;
        if (sees)
            y = kLog2e * row_score(a, row_dot(q, a.kc + (uint64_t)j * rstride + base, a.hd) * a.scale, slope,
                                   a.past + i, j);
        if (scores && sees) scores[j] = y;
        const uint64_t seen = __ballot(sees);
        if (!seen) continue;
        // (fmaxf drops a NaN: a NaN score comes through the sum instead)
        const float mn = fmaxf(m, wave_max(y)), top = mn == -INFINITY ? 0.f : mn;
        const float r = exp2f(m - top), p = sees ? exp2f(y - top) : 0.f;
        l = l * r + wave_sum(p);
        m = mn;
#pragma unroll
        for (uint32_t c = 0; c < (HD + 63u) / 64u; c++) {
            const uint32_t d = 64u * c + lane;
            float x = acc[c] * r;
            for (uint32_t t = 0; t < 64u; t++) {
                const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), (int)t));
                if ((seen >> t & 1u) && d < a.hd) x = fmaf(w, h2f(a.vc[(uint64_t)(j0 + t) * rstride + base + d]), x);
            }
            acc[c] = x;
        }
    }
    m_out = m;
    l_out = l;
}

}  // namespace vbs
