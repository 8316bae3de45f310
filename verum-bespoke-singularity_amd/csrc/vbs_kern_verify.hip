// vbs_kern_verify.hip — drafted tokens accepted or refused against the target's
// probabilities, from given random numbers.
//
// With p_i = softmax(target row i / T) and q_i = softmax(draft row i / T) (or q_i = 1 at the
// drafted token x_i, where no draft rows are given): x_i stays while u_i q_i(x_i) < p_i(x_i);
// the token behind the last that stays is the lowest x with sum_{y <= x} r(y) > u_n sum_y r(y),
// r = max(p_i - q_i, 0) at the first refusal (p_i where that is 0 everywhere), r = p_i at the
// draft's end. The tokens then are distributed as the target's own.
//
// Probabilities and sums are held in 64 bits: a token is chosen by on which side of a border a
// number lies, there are `vocab` borders, and a sum in f32 would move them by as much as small
// probabilities are wide. T = 0: the greatest logit (lowest place) has p = 1.
//
// Three launches: every row's maximum and sum by chunks of 4096; acceptance, from those, and what
// is left in each chunk of 1024 of the row to draw from; the chunk, and the place in it.
// Bound: HBM and, close behind, the vector units (about 27 instructions a logit, 13 of them in 64 bits) where the
// rows are many and long: 32 sequences of 7 drafted tokens of 131072 take 77 us, 53 of them the rows' sums at 4.5 TB/s
// (two chunks a workgroup, with half the joins of lanes: the same). The three launches and their round trips
// where they are few: one sequence of 4 of 32000 takes 15 us.
#include <math.h>

#include "vbs_dev_common.h"
#include "vbs_pages.h"

namespace vbs {

namespace {

constexpr uint32_t kThreads = 256, kWaves = 4, kGroups = 4;  // a lane takes kGroups times four neighbours
constexpr uint32_t kChunk = 256 * kGroups;       // of a wave: what is left is summed by these
constexpr uint32_t kRowChunk = kWaves * kChunk;  // of a workgroup: rows are summed by these

typedef float vf4 __attribute__((ext_vector_type(4)));

// 2^(j / 32); in LDS, where the 32 entries lie in banks of their own, less j 2^15 in their upper words (see power_of).
__constant__ double kTwo[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0, 0x1.172b83c7d517bp+0,
    0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0, 0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0,
    0x1.3dea64c123422p+0, 0x1.44e086061892dp+0, 0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0,
    0x1.6247eb03a5585p+0, 0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0, 0x1.ae89f995ad3adp+0,
    0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0, 0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0,
    0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0};
__device__ __forceinline__ void load_two(double *two) {
    if (threadIdx.x < 32u)
        two[threadIdx.x] = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, kTwo[threadIdx.x]) - ((uint64_t)threadIdx.x << 47));
}

// 2^(t / 32) for t <= 0 as two factors, from t = 32 n + j + f, |f| <= 1/2: w = 2^(n + j / 32) from the table, and the polynomial
// that interpolates 2^(f / 32) at the six Chebyshev nodes, its first coefficient 1 (off by 1.4e-16 of the value,
// beside the roundings'). From t = kFar down, and for NaN, 2^(kFar / 32). 13 operations in 64 bits with the sum, where a
// polynomial for the whole octave took 22.
constexpr double kFar = -32000.0;
struct Power {
    double w, p;
};
__device__ __forceinline__ Power power_of(double t, const double *two) {
    t = fmax(t, kFar);
    const double r = t + 0x1.8p52;
    const int32_t n = (int32_t)(uint32_t)__builtin_bit_cast(uint64_t, r);
    const double f = t - (r - 0x1.8p52);
    double p = 0x1.5d885e6ef14a6p-35;
    p = fma(p, f, 0x1.3b2b301f1eb9cp-27);
    p = fma(p, f, 0x1.c6b08d70380ddp-20);
    p = fma(p, f, 0x1.ebfbdff7feebap-13);
    p = fma(p, f, 0x1.62e42fefa39efp-6);
    p = fma(p, f, 1.0);
    const uint64_t w = __builtin_bit_cast(uint64_t, two[n & 31]);  // (n = 32 m + j adds m to the exponent and j 2^15 beside it)
    const uint32_t high = (uint32_t)(w >> 32) + ((uint32_t)n << 15);
    return Power{__builtin_bit_cast(double, (uint64_t)high << 32 | (uint32_t)w), p};
}
// The product, and 0 from kFar down.
__device__ __forceinline__ double exp2_neg(double t, const double *two) {
    const Power x = power_of(t, two);
    return t <= kFar ? 0.0 : x.w * x.p;
}

// The drafted tokens before the first that is none (an id outside the vocabulary); n is at most 64.
__device__ __forceinline__ uint32_t draft_length(const VerifyArgs &a, uint32_t b) {
    const uint32_t lane = threadIdx.x & 63u;
    const bool none = lane >= a.n || (uint32_t)a.drafted[(uint64_t)b * a.n + lane] >= a.vocab;
    const uint64_t at = __ballot(none);
    return at ? (uint32_t)__ffsll((unsigned long long)at) - 1u : 64u;
}
__device__ __forceinline__ const float *row_of(const VerifyArgs &a, uint32_t b, uint32_t r) {
    return r <= a.n ? a.logits + ((uint64_t)b * (a.n + 1u) + r) * a.stride
                    : a.draft + ((uint64_t)b * a.n + (r - a.n - 1u)) * a.draft_stride;
}
// Four logits from e on, `step` apart; -inf behind the last. Rows that can be read 16 bytes at a time give a lane four
// neighbours (step 1); others, where the order does not matter, every 64th, so that a wave's words are neighbours (32
// sequences of 7 of 131071: 99 -> 83 us).
template <bool VEC>
__device__ __forceinline__ vf4 four(const VerifyArgs &a, const float *x, uint32_t e, uint32_t step = VEC ? 1u : 64u) {
    if (VEC && e + 4u <= a.vocab) return *reinterpret_cast<const vf4 *>(x + e);
    vf4 v;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) v[j] = x[min(e + j * step, a.vocab - 1u)];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) v[j] = e + j * step < a.vocab ? v[j] : -INFINITY;
    return v;
}

// A wave's chunk from c0 on: of group i lane l has the four from c0 + 256 i + 4 l (VEC; else c0 + 256 i + l) on.
template <bool VEC>
__device__ __forceinline__ void whole_chunk(const VerifyArgs &a, const float *x, uint32_t c0, uint32_t lane, vf4 v[kGroups]) {
    if (VEC && c0 + kChunk <= a.vocab) {
#pragma unroll
        for (uint32_t i = 0; i < kGroups; i++) v[i] = *reinterpret_cast<const vf4 *>(x + c0 + i * 256u + lane * 4u);
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < kGroups; i++) v[i] = four<VEC>(a, x, c0 + i * 256u + (VEC ? lane * 4u : lane));
}

}  // namespace

// grid (chunks of 4096, rows of a sequence, sequences)
template <bool GREEDY, bool VEC>
__global__ __launch_bounds__(kThreads) void k_verify_sum(VerifyArgs a) {
    __shared__ float tops[kWaves];
    __shared__ uint32_t places[kWaves];
    __shared__ double sums[kWaves], two[32];
    const uint32_t b = blockIdx.z, r = blockIdx.y, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t c0 = __builtin_amdgcn_readfirstlane(blockIdx.x * kRowChunk + wave * kChunk);
    const float *x = row_of(a, b, r);
    vf4 v[kGroups];
    whole_chunk<VEC>(a, x, c0, lane, v);
    const uint32_t n = draft_length(a, b);
    if (r <= a.n ? r > n : r - a.n - 1u >= n) return;  // (a row behind the draft's end)
    const uint64_t to = ((uint64_t)b * (2u * a.n + 1u) + r) * a.chunks + blockIdx.x;
    float top = -INFINITY;
    if constexpr (GREEDY) {
        uint32_t at = 0xFFFFFFFFu;
#pragma unroll
        for (uint32_t i = 0; i < kGroups; i++)
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const uint32_t e = c0 + i * 256u + (VEC ? lane * 4u + j : j * 64u + lane);
                if (e < a.vocab && (v[i][j] > top || (v[i][j] == top && e < at))) top = v[i][j], at = e;
            }
        for (uint32_t o = 32; o; o >>= 1) {
            const float t = __shfl_xor(top, (int)o, 64);
            const uint32_t p = __shfl_xor(at, (int)o, 64);
            if (t > top || (t == top && p < at)) top = t, at = p;
        }
        if (lane == 0u) tops[wave] = top, places[wave] = at;
        __syncthreads();
        if (tid) return;
        for (uint32_t w = 1; w < kWaves; w++)
            if (tops[w] > top || (tops[w] == top && places[w] < at)) top = tops[w], at = places[w];
        a.tops[to] = top, a.arg[to] = (int32_t)at;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kGroups; i++)
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) top = fmaxf(top, v[i][j]);
        top = wave_max(top);
        if (lane == 0u) tops[wave] = top;
        load_two(two);
        __syncthreads();
        top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const double ref = top == -INFINITY ? 0.0 : (double)top;
        double s[2] = {0.0, 0.0};
#pragma unroll
        for (uint32_t i = 0; i < kGroups; i++)
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const Power x = power_of(((double)v[i][j] - ref) * a.rate, two);
                s[j & 1u] = fma(x.w, x.p, s[j & 1u]);
            }
        bool nan = false;
#pragma unroll
        for (uint32_t i = 0; i < kGroups; i++)
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) nan = nan || v[i][j] != v[i][j];
        double sum = wave_sum_d(s[0] + s[1]);
        if (__any(nan) || top == INFINITY) sum = NAN;  // (no distribution)
        else if (top == -INFINITY) sum = 0.0;
        if (lane == 0u) sums[wave] = sum;
        __syncthreads();
        if (tid == 0u) a.tops[to] = top, a.sums[to] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    }
}

// What a row sums to: its maximum, its sum relative to it, the maximum's place (temperature 0).
struct RowSum {
    float top;
    int32_t at;
    double sum;
};
// Of row r by `width` neighbouring lanes (a power of two, up to 64), `i` the lane among them.
__device__ __forceinline__ RowSum row_sum(const VerifyArgs &a, uint32_t b, uint32_t r, uint32_t i, uint32_t width, const double *two) {
    const uint64_t from = ((uint64_t)b * (2u * a.n + 1u) + r) * a.chunks;
    RowSum s{-INFINITY, -1, 0.0};
    if (a.temp == 0.f) {
        uint32_t at = 0xFFFFFFFFu;
        for (uint32_t k = i; k < a.chunks; k += width) {
            const float t = a.tops[from + k];
            const uint32_t p = (uint32_t)a.arg[from + k];
            if (t > s.top || (t == s.top && p < at)) s.top = t, at = p;
        }
        for (uint32_t o = width >> 1; o; o >>= 1) {
            const float t = __shfl_xor(s.top, (int)o, 64);
            const uint32_t p = __shfl_xor(at, (int)o, 64);
            if (t > s.top || (t == s.top && p < at)) s.top = t, at = p;
        }
        s.at = (int32_t)at;
        return s;
    }
    // (the sums of up to two chunks a lane are on their way with the maxima)
    double first = 0.0, second = 0.0;
    float t0 = -INFINITY, t1 = -INFINITY;
    if (i < a.chunks) t0 = a.tops[from + i], first = a.sums[from + i];
    if (i + width < a.chunks) t1 = a.tops[from + i + width], second = a.sums[from + i + width];
    s.top = fmaxf(t0, t1);
    for (uint32_t k = i + 2u * width; k < a.chunks; k += width) s.top = fmaxf(s.top, a.tops[from + k]);
    for (uint32_t o = width >> 1; o; o >>= 1) s.top = fmaxf(s.top, __shfl_xor(s.top, (int)o, 64));
    const double ref = s.top == -INFINITY ? 0.0 : (double)s.top;
    auto part = [&](float t, double v) { return t == -INFINITY && !(v != v) ? 0.0 : v * exp2_neg(((double)t - ref) * a.rate, two); };
    s.sum = part(t0, first) + part(t1, second);
    for (uint32_t k = i + 2u * width; k < a.chunks; k += width) s.sum += part(a.tops[from + k], a.sums[from + k]);
    for (uint32_t o = width >> 1; o; o >>= 1) s.sum += __shfl_xor(s.sum, (int)o, 64);
    if (s.top == -INFINITY) s.sum = NAN;  // (no distribution)
    return s;
}

// What is left to draw from: r(x) of the row the draft stopped at.
struct Left {
    const float *x, *y;  // the target's row; the draft's, or NULL
    double top, rsum, ytop, yrsum;
    int32_t without;  // the token of a certain draft that was refused, or -1
    const double *two;
    __device__ __forceinline__ void at(const VerifyArgs &a, uint32_t e, float lx, float ly, double &p, double &less) const {
        p = exp2_neg(((double)lx - top) * a.rate, two) * rsum;
        less = p;
        if (y) less = fmax(p - exp2_neg(((double)ly - ytop) * a.rate, two) * yrsum, 0.0);
        if ((int32_t)e == without) less = 0.0;
    }
};

// grid (chunks of 1024 / 4, sequences)
template <bool VEC>
__global__ __launch_bounds__(kThreads) void k_verify_accept(VerifyArgs a) {
    __shared__ RowSum rows[2 * kMaxDraft + 1];
    __shared__ uint32_t stop_w;
    __shared__ double two[32];
    const uint32_t b = blockIdx.y, tid = threadIdx.x, lane = tid & 63u;
    const uint32_t n = draft_length(a, b), count = n + 1u + (a.draft ? n : 0u);
    uint32_t width = 4u;
    while (width < 64u && width < a.chunks) width *= 2u;
    load_two(two);
    __syncthreads();
    int32_t token = 0;
    float u = 0.f, lx = 0.f, ly = 0.f;
    if (tid < n) {
        token = a.drafted[(uint64_t)b * a.n + tid];
        u = a.u[(uint64_t)b * (a.n + 1u) + tid];
        lx = row_of(a, b, tid)[token];
        if (a.draft) ly = row_of(a, b, a.n + 1u + tid)[token];
    }
    for (uint32_t i0 = 0; i0 < count; i0 += kThreads / width) {
        const uint32_t i = i0 + tid / width, in = min(i, count - 1u);  // (all lanes work together)
        const RowSum s = row_sum(a, b, in <= n ? in : a.n + in - n, tid & (width - 1u), width, two);
        if ((tid & (width - 1u)) == 0u && i < count) rows[i] = s;
    }
    __syncthreads();
    if (tid < 64u) {
        bool yes = tid >= n;
        if (yes) {
        } else if (a.temp > 0.f) {
            // u q < p, both sides times the two sums
            const RowSum p = rows[tid], q = a.draft ? rows[n + 1u + tid] : RowSum{0.f, 0, 1.0};
            const double qx = a.draft ? exp2_neg(((double)ly - (double)q.top) * a.rate, two) : 1.0;
            yes = (double)u * qx * p.sum < exp2_neg(((double)lx - (double)p.top) * a.rate, two) * q.sum;
        } else {
            yes = rows[tid].at == token && u < 1.f;
        }
        const uint64_t no = __ballot(!yes);
        if (tid == 0u) stop_w = no ? (uint32_t)__ffsll((unsigned long long)no) - 1u : n;
    }
    __syncthreads();
    const uint32_t stop = stop_w;
    const bool refused = stop < n;
    if (a.temp == 0.f) {
        const int32_t at = rows[stop].at;
        for (uint32_t i = tid; i <= a.n; i += kThreads)
            a.tokens[(uint64_t)b * (a.n + 1u) + i] = i < stop ? a.drafted[(uint64_t)b * a.n + i] : i == stop && (uint32_t)at < a.vocab ? at : -1;
        if (tid == 0u) a.accepted[b] = (int32_t)stop;
        return;
    }
    Left left;
    left.x = row_of(a, b, stop);
    left.y = refused && a.draft ? row_of(a, b, a.n + 1u + stop) : nullptr;
    left.top = (double)rows[stop].top;
    left.rsum = 1.0 / rows[stop].sum;
    left.ytop = left.y ? (double)rows[n + 1u + stop].top : 0.0;
    left.yrsum = left.y ? 1.0 / rows[n + 1u + stop].sum : 0.0;
    left.without = refused && !a.draft ? a.drafted[(uint64_t)b * a.n + stop] : -1;
    left.two = two;
    if (blockIdx.x == 0u && tid == 0u) {
        a.stop[b] = (int32_t)(stop | (refused ? 1u << 16 : 0u));
        double *st = a.stats + (uint64_t)b * 4u;
        st[0] = left.top, st[1] = left.rsum, st[2] = left.ytop, st[3] = left.yrsum;
    }
    const uint32_t chunk = blockIdx.x * kWaves + (tid >> 6);
    if (chunk >= a.small) return;
    const uint32_t c0 = __builtin_amdgcn_readfirstlane(chunk * kChunk);
    vf4 x[kGroups], y[kGroups];
    whole_chunk<VEC>(a, left.x, c0, lane, x);
    if (left.y) {
        whole_chunk<VEC>(a, left.y, c0, lane, y);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kGroups; i++) y[i] = vf4{0.f, 0.f, 0.f, 0.f};
    }
    double all = 0.0, less = 0.0;  // (behind the last, logits of -inf add 0)
#pragma unroll
    for (uint32_t i = 0; i < kGroups; i++)
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            double p, l;
            left.at(a, c0 + i * 256u + (VEC ? lane * 4u + j : j * 64u + lane), x[i][j], y[i][j], p, l);
            all += p, less += l;
        }
    all = wave_sum_d(all);
    less = wave_sum_d(less);
    if (lane == 0u) {
        a.left[((uint64_t)b * 2u) * a.small + chunk] = less;
        a.left[((uint64_t)b * 2u + 1u) * a.small + chunk] = all;
    }
}

__device__ __forceinline__ double scan_64(double v, uint32_t lane) {
    for (uint32_t o = 1; o < 64u; o <<= 1) {
        const double t = __shfl_up(v, (int)o, 64);
        if (lane >= o) v += t;
    }
    return v;
}

// grid (sequences): every wave finds the chunk; a thread then takes four neighbours of it.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void k_verify_pick(VerifyArgs a) {
    __shared__ double ends[kWaves], two[32];
    __shared__ uint32_t found[kWaves], last[kWaves];
    const uint32_t b = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t stop = (uint32_t)a.stop[b] & 0xFFFFu;
    const bool refused = (uint32_t)a.stop[b] >> 16;
    const double *st = a.stats + (uint64_t)b * 4u;
    Left left;
    left.x = row_of(a, b, stop);
    left.y = refused && a.draft ? row_of(a, b, a.n + 1u + stop) : nullptr;
    left.top = st[0], left.rsum = st[1], left.ytop = st[2], left.yrsum = st[3];
    left.without = refused && !a.draft ? a.drafted[(uint64_t)b * a.n + stop] : -1;
    left.two = two;
    load_two(two);
    __syncthreads();
    const double *sums = a.left + (uint64_t)b * 2u * a.small;
    const float u = a.u[(uint64_t)b * (a.n + 1u) + a.n];
    double less = 0.0, all = 0.0;
    for (uint32_t k = lane; k < a.small; k += 64u) less += sums[k], all += sums[a.small + k];
    less = wave_sum_d(less);
    const bool whole = !(less > 0.0) && !(less != less);  // nothing left: the target's own
    const double total = whole ? wave_sum_d(all) : less;
    if (whole) sums += a.small;
    int32_t next = -1;
    if (total > 0.0) {
        const double want = fmax((double)u, 0.0) * total;
        // the first chunk that passes `want`, or the last that holds anything
        double run = 0.0, before = 0.0;
        uint32_t chunk = 0;
        for (uint32_t k0 = 0; k0 < a.small; k0 += 64u) {
            const double s = k0 + lane < a.small ? sums[k0 + lane] : 0.0, to = run + scan_64(s, lane);
            const uint64_t some = __ballot(s > 0.0), past = __ballot(to > want && s > 0.0);
            if (some) {
                const uint32_t at = past ? (uint32_t)__ffsll((unsigned long long)past) - 1u : 63u - (uint32_t)__clzll((unsigned long long)some);
                chunk = k0 + at;
                before = __shfl(to - s, (int)at, 64);
            }
            if (past) break;
            run = __shfl(to, 63, 64);
        }
        const uint32_t e = chunk * kChunk + tid * 4u;
        const vf4 x = four<VEC>(a, left.x, e, 1u), y = left.y ? four<VEC>(a, left.y, e, 1u) : vf4{0.f, 0.f, 0.f, 0.f};
        double r[4], mine = 0.0;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            double p, l;
            left.at(a, e + j, x[j], y[j], p, l);
            mine += r[j] = whole ? p : l;
        }
        double at = scan_64(mine, lane);
        if (lane == 63u) ends[wave] = at;
        __syncthreads();
        at += before - mine;
        for (uint32_t k = 0; k < wave; k++) at += ends[k];
        constexpr uint32_t none = 0xFFFFFFFFu;
        uint32_t here = none, some = none;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            at += r[j];
            if (r[j] > 0.0) {
                some = e + j;
                if (at > want && here == none) here = e + j;
            }
        }
        const uint64_t past = __ballot(here != none), any = __ballot(some != none);
        here = __shfl(here, past ? __ffsll((unsigned long long)past) - 1 : 0, 64);
        some = __shfl(some, any ? 63 - __clzll((unsigned long long)any) : 0, 64);
        if (lane == 0u) found[wave] = past ? here : none, last[wave] = any ? some : none;
        __syncthreads();
        uint32_t pick = none;
        for (uint32_t k = 0; k < kWaves; k++) pick = min(pick, found[k]);
        if (pick == none)  // (the sums' roundings: the last that holds anything)
            for (uint32_t k = 0; k < kWaves; k++)
                if (last[k] != none) pick = last[k];
        next = (int32_t)pick;
    }
    for (uint32_t i = tid; i <= a.n; i += kThreads)
        a.tokens[(uint64_t)b * (a.n + 1u) + i] = i < stop ? a.drafted[(uint64_t)b * a.n + i] : i == stop ? next : -1;
    if (tid == 0u) a.accepted[b] = (int32_t)stop;
}

size_t plan_verify(VerifyArgs &a) {
    a.chunks = (a.vocab + kRowChunk - 1u) / kRowChunk;
    a.small = (a.vocab + kChunk - 1u) / kChunk;
    const uint64_t parts = (uint64_t)a.batch * (2u * a.n + 1u) * a.chunks;
    return parts * 16u + (uint64_t)a.batch * (a.small * 16u + 40u);
}

hipError_t launch_verify(VerifyArgs a, void *scratch, hipStream_t s) {
    const uint64_t parts = (uint64_t)a.batch * (2u * a.n + 1u) * a.chunks;
    a.sums = static_cast<double *>(scratch);
    a.left = a.sums + parts;
    a.stats = a.left + 2u * (uint64_t)a.batch * a.small;
    a.tops = reinterpret_cast<float *>(a.stats + 4u * (uint64_t)a.batch);
    a.arg = reinterpret_cast<int32_t *>(a.tops + parts);
    a.stop = a.arg + parts;
    if (a.temp == 0.f) a.draft = nullptr;
    a.rate = a.temp > 0.f ? 32.0 * 1.4426950408889634074 / (double)a.temp : 0.0;  // 32 log2 e / T
    const bool vec = !(((uintptr_t)a.logits & 15u) | (a.stride & 3u) | ((uintptr_t)a.draft & 15u) | (a.draft ? a.draft_stride & 3u : 0u));
    const dim3 grid(a.chunks, a.n + 1u + (a.draft ? a.n : 0u), a.batch);
    if (a.temp == 0.f) (vec ? k_verify_sum<true, true> : k_verify_sum<true, false>)<<<grid, kThreads, 0, s>>>(a);
    else (vec ? k_verify_sum<false, true> : k_verify_sum<false, false>)<<<grid, kThreads, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    (vec ? k_verify_accept<true> : k_verify_accept<false>)<<<dim3(a.temp == 0.f ? 1u : a.chunks, a.batch), kThreads, 0, s>>>(a);
    e = hipGetLastError();
    if (e != hipSuccess || a.temp == 0.f) return e;
    (vec ? k_verify_pick<true> : k_verify_pick<false>)<<<a.batch, kThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace vbs
