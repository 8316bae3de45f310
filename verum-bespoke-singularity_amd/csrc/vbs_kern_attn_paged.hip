// vbs_kern_attn_paged.hip — the attention of single tokens over the paged cache.
//
// Row r (one token; its q heads of one kv head are up to eight columns of a product):
// out = sum_j w_j v_j, w = softmax(scale q.k_j) over the slots j < lens[r]. A row's units
// of 32 slots are split over workgroups and over their four waves; each keeps the running
// maximum m (in log2), the sum l and O of its own units, the four are joined through LDS and
// the workgroups' by k_attn_paged_merge.
//
// Products: S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_16x16x32_f16, whose operands the
// page's layout holds as they are (vbs_pages.h), so K and V go from memory to the registers
// they are used from. The outputs are f32: q and the weights enter as two f16 parts (22 bits),
// columns 0-7 the high parts of eight heads and columns 8-15 the low parts, which costs nothing
// where eight columns would be idle. q's head is scaled by a power of two so that its greatest
// element is about 2^14, and the weights by 2^14 (relative to the running maximum), so a slot
// reaches V's sum down to 2^-38 of the greatest weight.
// Q8_0: int8 becomes f16 exactly (as 1024 + 128 + q, less 1152); K's scales multiply the products
// of their block, V's the weights, over a running power of two above all scales (2^E), which keeps
// them in f16's range: then 2^-38 of the greatest weight times the greatest scale.
//
// Values that the parts cannot carry (infinities and NaN in q, K or V meet a part that is 0,
// or whose sign differs) leave a sum that is not finite: the workgroup then takes its slots
// again in plain f32 (slow_tile).
//
// Bound: HBM.
#include <math.h>

#include "vbs_dev_common.h"
#include "vbs_pages.h"

namespace vbs {

namespace {

typedef _Float16 ph8 __attribute__((ext_vector_type(8)));
typedef _Float16 ph2 __attribute__((ext_vector_type(2)));
typedef float pf4 __attribute__((ext_vector_type(4)));
typedef uint32_t pu4 __attribute__((ext_vector_type(4)));

constexpr float kPagedLog2e = 1.44269504088896341f;
constexpr uint32_t kHeads = 8, kWaves = 4;
constexpr int kWeightBits = 14;  // weights stand 2^14 high

__device__ __forceinline__ float row_ror8(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x128, 0xF, 0xF, false));
}
__device__ __forceinline__ float over_groups_max(float v) {
    v = fmaxf(v, lane_xor<16>(v));
    return fmaxf(v, lane_xor<32>(v));
}
__device__ __forceinline__ float over_groups_sum(float v) {
    v += lane_xor<16>(v);
    return v + lane_xor<32>(v);
}

// Eight int8 as f16: with its sign bit turned over, a byte u = q + 128 under the exponent of 1024 is the f16 1024 + u.
__device__ __forceinline__ ph8 int8_to_f16(uint32_t lo, uint32_t hi) {
    lo ^= 0x80808080u, hi ^= 0x80808080u;
    const uint32_t e = 0x64646464u;
    ph2 p[4];
    p[0] = __builtin_bit_cast(ph2, __builtin_amdgcn_perm(e, lo, 0x04010400u));
    p[1] = __builtin_bit_cast(ph2, __builtin_amdgcn_perm(e, lo, 0x04030402u));
    p[2] = __builtin_bit_cast(ph2, __builtin_amdgcn_perm(e, hi, 0x04010400u));
    p[3] = __builtin_bit_cast(ph2, __builtin_amdgcn_perm(e, hi, 0x04030402u));
    const ph2 off = {(_Float16)1152.f, (_Float16)1152.f};
    ph8 r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        p[i] = p[i] - off;
        r[2 * i] = p[i][0], r[2 * i + 1] = p[i][1];
    }
    return r;
}

// The high or the low f16 part of eight values.
__device__ __forceinline__ ph8 parts(const float x[8], bool low) {
    ph8 r;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const _Float16 h = (_Float16)x[e];
        const _Float16 l = (_Float16)(x[e] - (float)h);
        r[e] = low ? l : h;
    }
    return r;
}

// What a workgroup is to do: the units [u0, u1) of a row.
struct Span {
    int32_t seq;
    uint32_t len, u0, u1;
    bool bad;  // a length or sequence out of range: the row is NaN
};
__device__ __forceinline__ Span row_span(const PagedAttnArgs &a, uint32_t row) {
    Span s;
    s.seq = a.seq ? a.seq[row] : (int32_t)row;
    const int32_t len = a.lens[row];
    s.bad = len < 0 || (uint32_t)len > a.max_len || (uint32_t)s.seq >= a.p.n_seqs;
    s.len = s.bad ? 0u : (uint32_t)len;
    s.u0 = 0u;
    s.u1 = (s.len + kUnit - 1u) / kUnit;
    return s;
}
__device__ __forceinline__ uint32_t row_splits(const PagedAttnArgs &a, const Span &s) {
    return max(1u, (s.u1 + a.per_split - 1u) / a.per_split);
}

template <uint32_t NB, bool Q8>
struct Unit {
    pu4 k[Q8 ? NB : 2 * NB], v[Q8 ? NB : 2 * NB];
    pu4 ks[Q8 ? NB : 1], vs[Q8 ? NB : 1];

    __device__ __forceinline__ void load_k(const uint8_t *p, uint32_t lane) {
#pragma unroll
        for (uint32_t i = 0; i < (Q8 ? NB : 2 * NB); i++) k[i] = *reinterpret_cast<const pu4 *>(p + i * 1024u + lane * 16u);
        if constexpr (Q8) {
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) ks[b] = *reinterpret_cast<const pu4 *>(p + NB * 1024u + b * 64u + (lane >> 4) * 16u);
        }
    }
    __device__ __forceinline__ void load_v(const uint8_t *p, uint32_t lane) {
#pragma unroll
        for (uint32_t i = 0; i < (Q8 ? NB : 2 * NB); i++) v[i] = *reinterpret_cast<const pu4 *>(p + i * 1024u + lane * 16u);
        if constexpr (Q8) {
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) vs[b] = *reinterpret_cast<const pu4 *>(p + NB * 1024u + b * 64u + (lane >> 4) * 16u);
        }
    }
};

}  // namespace

// The workgroup's slots [32 u0, min(32 u1, len)) again for one q head, in f32 products and sums: m, l and O (thread d
// holds element d). `w` holds 256 floats.
template <bool Q8>
__device__ __noinline__ void slow_tile(const PagedAttnArgs &a, const Span &sp, uint32_t kvh, const float *q, float *w, float &m,
                                       float &l, float &o) {
    const uint32_t tid = threadIdx.x, hd = a.p.hd, nb = a.p.nb, end = min(sp.u1 * kUnit, sp.len);
    m = -INFINITY, l = 0.f, o = 0.f;
    for (uint32_t j0 = sp.u0 * kUnit; j0 < end; j0 += 256u) {
        const uint32_t j = j0 + tid, count = min(256u, end - j0);
        float s = 0.f;
        if (j < end) {
            const int32_t page = page_at(a.p, sp.seq, j / kUnit);
            if (page < 0) {
                s = NAN;
            } else {
                const uint8_t *unit = a.p.k + unit_offset(a.p, page, j / kUnit, kvh);
                const uint32_t slot = j & (kUnit - 1u);
                for (uint32_t d = 0; d < hd; d++) {
                    float k;
                    if constexpr (Q8)
                        k = (float)(int8_t)unit[k_place<true>(nb, slot, d)] *
                            (float)reinterpret_cast<const _Float16 *>(unit + nb * 1024u)[(d & ~31u) + slot];
                    else
                        k = vbs_h2f(reinterpret_cast<const uint16_t *>(unit)[k_place<false>(nb, slot, d)]);
                    s = fmaf(q[d], k, s);
                }
                s *= a.scale * kPagedLog2e;
            }
            w[tid] = s;
        }
        __syncthreads();
        float top = m;
        for (uint32_t i = 0; i < count; i++) top = fmaxf(top, w[i]);
        __syncthreads();
        const float ref = top == -INFINITY ? 0.f : top;
        if (j < end) w[tid] = __builtin_amdgcn_exp2f(s - ref);
        __syncthreads();
        const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - ref);
        l *= keep, o *= keep;
        m = top;
        for (uint32_t i = 0; i < count; i++) {
            const float p = w[i];
            l += p;
            const uint32_t jj = j0 + i;
            const int32_t page = page_at(a.p, sp.seq, jj / kUnit);
            if (tid >= hd || page < 0) continue;
            const uint8_t *unit = a.p.v + unit_offset(a.p, page, jj / kUnit, kvh);
            const uint32_t slot = jj & (kUnit - 1u);
            float v;
            if constexpr (Q8)
                v = (float)(int8_t)unit[v_place<true>(slot, tid)] *
                    (float)reinterpret_cast<const _Float16 *>(unit + nb * 1024u)[(tid & ~31u) + slot];
            else
                v = vbs_h2f(reinterpret_cast<const uint16_t *>(unit)[v_place<false>(slot, tid)]);
            o = fmaf(p, v, o);
        }
        __syncthreads();
    }
}

// grid (splits x kv heads x tiles of eight q heads, rows)
template <uint32_t NB, bool Q8>
__global__ __launch_bounds__(256, 2) void k_attn_paged(PagedAttnArgs a) {
    __shared__ float so[kWaves][kHeads][NB * 32u + 4u];
    __shared__ float sm[kWaves][kHeads], sl[kWaves][kHeads];
    __shared__ uint32_t odd;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, c = lane & 15u;
    const uint32_t tiles = (a.group + kHeads - 1u) / kHeads, split = blockIdx.x % a.splits, hx = blockIdx.x / a.splits;
    const uint32_t kvh = hx / tiles, tile = hx % tiles, row = blockIdx.y, hd = a.p.hd;
    Span sp = row_span(a, row);
    if (split >= row_splits(a, sp)) return;
    const uint32_t nsplit = row_splits(a, sp);
    sp.u0 = split * a.per_split;
    sp.u1 = min(sp.u0 + a.per_split, sp.u1);
    const uint32_t head0 = kvh * a.group + tile * kHeads, heads = min(kHeads, a.group - tile * kHeads);
    const float *q0 = a.q + (uint64_t)row * a.q_stride + (uint64_t)head0 * hd;
    if (tid == 0) odd = 0u;

    // q's parts: column c the head c & 7, its elements 32 b + 8 g ..
    ph8 qf[NB];
    float unscale;
    {
        const uint32_t h = c & 7u;
        float x[NB][8], top = 0.f;
#pragma unroll
        for (uint32_t b = 0; b < NB; b++)
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) {
                const uint32_t d = b * 32u + g * 8u + e;
                x[b][e] = h < heads && d < hd ? q0[(uint64_t)h * hd + d] : 0.f;
                top = fmaxf(top, fabsf(x[b][e]));
            }
        top = over_groups_max(top);
        const int up = 13 + 127 - (int)max(vbs_float_to_bits(top) >> 23, 1u);  // (an infinity stays one)
#pragma unroll
        for (uint32_t b = 0; b < NB; b++) {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) x[b][e] = __builtin_ldexpf(x[b][e], up);
            qf[b] = parts(x[b], c >= 8u);
        }
        unscale = __builtin_ldexpf(a.scale * kPagedLog2e, -up);
    }

    pf4 o[2 * NB];
#pragma unroll
    for (uint32_t i = 0; i < 2 * NB; i++) o[i] = pf4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    int top_e = -60;  // Q8_0: V's scales are below 2^top_e
    bool lost = false;
    for (uint32_t u = sp.u0 + wave; u < sp.u1; u += kWaves) {
        const int32_t page = __builtin_amdgcn_readfirstlane(page_at(a.p, sp.seq, u));
        if (page < 0) {
            lost = true;
            break;
        }
        const uint64_t at = unit_offset(a.p, page, u, kvh);
        Unit<NB, Q8> f;
        f.load_k(a.p.k + at, lane);
        f.load_v(a.p.v + at, lane);
        // scores: lane (g, c) holds slots 8 g + e of column c
        float s[8];
        if constexpr (Q8) {
#pragma unroll
            for (int e = 0; e < 8; e++) s[e] = 0.f;
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) {
                const ph8 d = __builtin_bit_cast(ph8, f.ks[b]);
                const pf4 zero = {0.f, 0.f, 0.f, 0.f};
                const pf4 s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(int8_to_f16(f.k[b][0], f.k[b][1]), qf[b], zero, 0, 0, 0);
                const pf4 s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(int8_to_f16(f.k[b][2], f.k[b][3]), qf[b], zero, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    s[i] = fmaf(s0[i], (float)d[i], s[i]);
                    s[4 + i] = fmaf(s1[i], (float)d[4 + i], s[4 + i]);
                }
            }
        } else {
            pf4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) {
                s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, f.k[b]), qf[b], s0, 0, 0, 0);
                s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, f.k[NB + b]), qf[b], s1, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) s[i] = s0[i], s[4 + i] = s1[i];
        }
        const uint32_t mine = u * kUnit + g * 8u;  // the lane's first slot
        const bool tail = (u + 1u) * kUnit > sp.len;
        float top = m;
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) {
            s[e] = (s[e] + row_ror8(s[e])) * unscale;
            if (tail && mine + e >= sp.len) s[e] = -INFINITY;
            top = fmaxf(top, s[e]);
        }
        top = over_groups_max(top);
        const float ref = top == -INFINITY ? 0.f : top;
        if (tail) {  // what lies behind the last slot may be anything
#pragma unroll
            for (uint32_t i = 0; i < (Q8 ? 0u : 2 * NB); i++)
#pragma unroll
                for (uint32_t w = 0; w < 4; w++) {
                    const uint32_t j = mine + 2u * w;
                    f.v[i][w] &= (j < sp.len ? 0xFFFFu : 0u) | (j + 1u < sp.len ? 0xFFFF0000u : 0u);
                }
#pragma unroll
            for (uint32_t i = 0; i < (Q8 ? NB : 0u); i++)
#pragma unroll
                for (uint32_t w = 0; w < 4; w++) {
                    const uint32_t j = mine + 2u * w;
                    f.vs[i][w] &= (j < sp.len ? 0xFFFFu : 0u) | (j + 1u < sp.len ? 0xFFFF0000u : 0u);
                }
        }
        float p[8], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = __builtin_amdgcn_exp2f(s[e] - ref);
            sum += p[e];
        }
        float keep = __builtin_amdgcn_exp2f(m - ref);
        l = l * keep + sum;
        m = top;
        if constexpr (Q8) {
            uint32_t big = 0u;
#pragma unroll
            for (uint32_t b = 0; b < NB; b++)
#pragma unroll
                for (int w = 0; w < 4; w++) big = max(big, max(f.vs[b][w] & 0x7FFFu, (f.vs[b][w] >> 16) & 0x7FFFu));
            big = max(big, lane_xor<16>(big));
            big = max(big, lane_xor<32>(big));
            const int e = __builtin_amdgcn_readfirstlane((int)min(big >> 10, 30u)) - 14;
            if (e > top_e) {
                keep = __builtin_ldexpf(keep, top_e - e);
                top_e = e;
            }
        }
        if (__any(keep != 1.f)) {
#pragma unroll
            for (uint32_t i = 0; i < 2 * NB; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) o[i][r] *= keep;
        }
        if constexpr (Q8) {
#pragma unroll
            for (int e = 0; e < 8; e++) p[e] = __builtin_ldexpf(p[e], kWeightBits - top_e);
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) {
                const ph8 d = __builtin_bit_cast(ph8, f.vs[b]);
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = p[e] * (float)d[e];
                const ph8 w = parts(x, c >= 8u);
                o[2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(int8_to_f16(f.v[b][0], f.v[b][1]), w, o[2 * b], 0, 0, 0);
                o[2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(int8_to_f16(f.v[b][2], f.v[b][3]), w, o[2 * b + 1], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) p[e] *= (float)(1 << kWeightBits);
            const ph8 w = parts(p, c >= 8u);
#pragma unroll
            for (uint32_t i = 0; i < 2 * NB; i++)
                o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, f.v[i]), w, o[i], 0, 0, 0);
        }
    }
    l = over_groups_sum(l);
    const float down = __builtin_ldexpf(1.f, (Q8 ? top_e : 0) - kWeightBits);
    bool fine = fabsf(l) < INFINITY;
#pragma unroll
    for (uint32_t i = 0; i < 2 * NB; i++) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            o[i][r] = (o[i][r] + row_ror8(o[i][r])) * down;
            fine = fine && fabsf(o[i][r]) < INFINITY;
        }
        if (c < 8u) *reinterpret_cast<pf4 *>(&so[wave][c][i * 16u + g * 4u]) = o[i];
    }
    if (g == 0u && c < 8u) sm[wave][c] = m, sl[wave][c] = l;
    fine = fine || (c & 7u) >= heads;
    __syncthreads();  // (odd is 0)
    if ((lost || __any(!fine)) && lane == 0u) odd = 1u;
    __syncthreads();
    const bool again = odd != 0u, direct = nsplit == 1u && a.splits == 1u;
    for (uint32_t h = 0; h < heads; h++) {
        float mm, ll, oo;
        if (again) {
            __syncthreads();
            slow_tile<Q8>(a, sp, kvh, q0 + (uint64_t)h * hd, &so[0][0][0], mm, ll, oo);
        } else {
            mm = fmaxf(fmaxf(sm[0][h], sm[1][h]), fmaxf(sm[2][h], sm[3][h]));
            ll = 0.f, oo = 0.f;
            const float ref = mm == -INFINITY ? 0.f : mm;
#pragma unroll
            for (uint32_t w = 0; w < kWaves; w++) {
                const float f = __builtin_amdgcn_exp2f(sm[w][h] - ref);
                ll = fmaf(f, sl[w][h], ll);
                if (tid < hd) oo = fmaf(f, so[w][h][tid], oo);
            }
        }
        if (sp.bad) ll = NAN;
        const uint32_t head = head0 + h;
        if (direct) {
            if (tid < hd) a.out[(uint64_t)row * a.out_stride + (uint64_t)head * hd + tid] = ll == 0.f ? 0.f : oo / ll;
        } else {
            const uint64_t at = ((uint64_t)row * a.nqh + head) * a.splits + split;
            if (tid < hd) a.part[at * hd + tid] = oo;
            if (tid == 0u) a.ml[at] = make_float2(mm, ll);
        }
    }
}

// The splits of a row joined: grid (q heads, rows).
__global__ __launch_bounds__(256) void k_attn_paged_merge(PagedAttnArgs a) {
    const uint32_t head = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, hd = a.p.hd;
    const Span sp = row_span(a, row);
    const uint32_t n = row_splits(a, sp);
    const uint64_t at = ((uint64_t)row * a.nqh + head) * a.splits;
    float m = -INFINITY;
    for (uint32_t i = 0; i < n; i++) m = fmaxf(m, a.ml[at + i].x);
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f, o = 0.f;
    for (uint32_t i = 0; i < n; i++) {
        const float2 x = a.ml[at + i];
        const float f = __builtin_amdgcn_exp2f(x.x - ref);
        l = fmaf(f, x.y, l);
        if (tid < hd) o = fmaf(f, a.part[(at + i) * hd + tid], o);
    }
    if (tid < hd) a.out[(uint64_t)row * a.out_stride + (uint64_t)head * hd + tid] = l == 0.f ? 0.f : o / l;
}

size_t plan_attn_paged(PagedAttnArgs &a) {
    const uint32_t units = (a.max_len + kUnit - 1u) / kUnit, tiles = (a.group + kHeads - 1u) / kHeads;
    const uint64_t all = (uint64_t)units * a.rows * a.p.nkh * tiles;
    uint64_t per = (all + 1023u) / 1024u;
    per = (per + kWaves - 1u) / kWaves * kWaves;
    if (per < kWaves) per = kWaves;
    if ((uint64_t)units > per * 256u) per = ((uint64_t)units + 255u) / 256u;
    a.per_split = (uint32_t)per;
    a.splits = units ? (uint32_t)((units + per - 1u) / per) : 1u;
    if (a.splits == 1u) return 0;
    return (uint64_t)a.rows * a.nqh * a.splits * (sizeof(float2) + 4ull * a.p.hd);
}

template <bool Q8>
static void launch_nb(const PagedAttnArgs &a, dim3 grid, hipStream_t s) {
    switch (a.p.nb) {
        case 1: k_attn_paged<1, Q8><<<grid, 256, 0, s>>>(a); break;
        case 2: k_attn_paged<2, Q8><<<grid, 256, 0, s>>>(a); break;
        case 3: k_attn_paged<3, Q8><<<grid, 256, 0, s>>>(a); break;
        case 4: k_attn_paged<4, Q8><<<grid, 256, 0, s>>>(a); break;
        case 5: k_attn_paged<5, Q8><<<grid, 256, 0, s>>>(a); break;
        case 6: k_attn_paged<6, Q8><<<grid, 256, 0, s>>>(a); break;
        case 7: k_attn_paged<7, Q8><<<grid, 256, 0, s>>>(a); break;
        default: k_attn_paged<8, Q8><<<grid, 256, 0, s>>>(a); break;
    }
}

hipError_t launch_attn_paged(PagedAttnArgs a, void *scratch, hipStream_t s) {
    const uint32_t tiles = (a.group + kHeads - 1u) / kHeads;
    a.ml = static_cast<float2 *>(scratch);
    a.part = reinterpret_cast<float *>(a.ml + (uint64_t)a.rows * a.nqh * a.splits);
    const dim3 grid(a.splits * a.p.nkh * tiles, a.rows);
    if (a.p.q8) launch_nb<true>(a, grid, s);
    else launch_nb<false>(a, grid, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1u) return e;
    k_attn_paged_merge<<<dim3(a.nqh, a.rows), (a.p.hd + 63u) / 64u * 64u, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace vbs
