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
// Three launches: every row's maximum and sum by chunks; acceptance, from those, and what is
// left in each chunk of the row to draw from; the chunk, and the place in it.
#include <math.h>

#include "vbs_dev_common.h"
#include "vbs_pages.h"

namespace vbs {

namespace {

constexpr uint32_t kChunk = 4096, kThreads = 256, kEach = kChunk / kThreads;

// e^x for x <= 0 (and 0 for -inf, NaN for NaN).
__device__ __forceinline__ double exp_neg(double x) { return exp(x); }

__device__ __forceinline__ double block_sum(double v, double *w) {
    v = wave_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) w[threadIdx.x >> 6] = v;
    __syncthreads();
    return (w[0] + w[1]) + (w[2] + w[3]);
}

// The drafted tokens before the first that is none (an id outside the vocabulary).
__device__ __forceinline__ uint32_t draft_length(const VerifyArgs &a, uint32_t b) {
    uint32_t n = 0;
    while (n < a.n && (uint32_t)a.drafted[(uint64_t)b * a.n + n] < a.vocab) n++;
    return n;
}
__device__ __forceinline__ const float *row_of(const VerifyArgs &a, uint32_t b, uint32_t r) {
    return r <= a.n ? a.logits + ((uint64_t)b * (a.n + 1u) + r) * a.stride
                    : a.draft + ((uint64_t)b * a.n + (r - a.n - 1u)) * a.draft_stride;
}

}  // namespace

// grid (chunks, rows of a sequence, sequences)
__global__ __launch_bounds__(kThreads) void k_verify_sum(VerifyArgs a) {
    __shared__ double w[4];
    __shared__ float top_w[4];
    __shared__ int32_t at_w[4];
    const uint32_t b = blockIdx.z, r = blockIdx.y, tid = threadIdx.x, c0 = blockIdx.x * kChunk;
    const uint32_t n = draft_length(a, b);
    if (r <= a.n ? r > n : r - a.n - 1u >= n) return;
    const float *x = row_of(a, b, r);
    float v[kEach], top = -INFINITY;
    int32_t at = 0x7FFFFFFF;
#pragma unroll
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t e = c0 + i * kThreads + tid;
        v[i] = e < a.vocab ? x[e] : -INFINITY;
        if (v[i] > top || (v[i] == top && (int32_t)e < at && e < a.vocab)) top = v[i], at = (int32_t)e;
    }
    for (uint32_t o = 32; o; o >>= 1) {
        const float t = __shfl_xor(top, (int)o, 64);
        const int32_t p = __shfl_xor(at, (int)o, 64);
        if (t > top || (t == top && p < at)) top = t, at = p;
    }
    if ((tid & 63u) == 0u) top_w[tid >> 6] = top, at_w[tid >> 6] = at;
    __syncthreads();
    top = top_w[0], at = at_w[0];
    for (uint32_t i = 1; i < 4; i++)
        if (top_w[i] > top || (top_w[i] == top && at_w[i] < at)) top = top_w[i], at = at_w[i];
    const uint64_t to = ((uint64_t)b * (2u * a.n + 1u) + r) * a.chunks + blockIdx.x;
    double sum = 0.0;
    if (a.temp > 0.f) {
        const double rt = 1.0 / (double)a.temp, ref = top == -INFINITY ? 0.0 : (double)top;
#pragma unroll
        for (uint32_t i = 0; i < kEach; i++) sum += exp_neg(((double)v[i] - ref) * rt);
        sum = block_sum(sum, w);
    }
    if (tid == 0u) a.tops[to] = top, a.arg[to] = at, a.sums[to] = sum;
}

// What row r of a sequence sums to, by a wave: its maximum, its sum relative to it, the maximum's place.
struct RowSum {
    float top;
    double sum;
    int32_t at;
};
__device__ __forceinline__ RowSum row_sum(const VerifyArgs &a, uint32_t b, uint32_t r, uint32_t lane) {
    const uint64_t from = ((uint64_t)b * (2u * a.n + 1u) + r) * a.chunks;
    RowSum s{-INFINITY, 0.0, 0x7FFFFFFF};
    for (uint32_t i = lane; i < a.chunks; i += 64u) {
        const float t = a.tops[from + i];
        const int32_t p = a.arg[from + i];
        if (t > s.top || (t == s.top && p < s.at)) s.top = t, s.at = p;
    }
    for (uint32_t o = 32; o; o >>= 1) {
        const float t = __shfl_xor(s.top, (int)o, 64);
        const int32_t p = __shfl_xor(s.at, (int)o, 64);
        if (t > s.top || (t == s.top && p < s.at)) s.top = t, s.at = p;
    }
    if (a.temp > 0.f) {
        const double rt = 1.0 / (double)a.temp, ref = s.top == -INFINITY ? 0.0 : (double)s.top;
        for (uint32_t i = lane; i < a.chunks; i += 64u) {
            const float t = a.tops[from + i];
            s.sum += a.sums[from + i] * exp_neg(((t == -INFINITY ? ref : (double)t) - ref) * rt);
        }
        s.sum = wave_sum_d(s.sum);
    }
    return s;
}

// What is left to draw from: r(x) of the row the draft stopped at.
struct Left {
    const float *x, *y;  // the target's row; the draft's, or NULL
    double rt, top, rsum, ytop, yrsum;
    int32_t without;  // the token of a certain draft that was refused, or -1
    __device__ __forceinline__ void at(uint32_t e, double &p, double &less) const {
        p = exp_neg(((double)x[e] - top) * rt) * rsum;
        less = p;
        if (y) less = fmax(p - exp_neg(((double)y[e] - ytop) * rt) * yrsum, 0.0);
        if ((int32_t)e == without) less = 0.0;
    }
};

// grid (chunks, sequences)
__global__ __launch_bounds__(kThreads) void k_verify_accept(VerifyArgs a) {
    __shared__ double w[4];
    __shared__ RowSum rows[2 * kMaxDraft + 1];
    __shared__ uint32_t stop_w;
    const uint32_t b = blockIdx.y, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, c0 = blockIdx.x * kChunk;
    const uint32_t n = draft_length(a, b), with = a.draft ? n : 0u;
    for (uint32_t i = wave; i < n + 1u + with; i += 4u) {
        const uint32_t r = i <= n ? i : a.n + 1u + (i - n - 1u);
        const RowSum s = row_sum(a, b, r, lane);
        if (lane == 0u) rows[i] = s;
    }
    if (tid == 0u) stop_w = n;
    __syncthreads();
    const double rt = a.temp > 0.f ? 1.0 / (double)a.temp : 0.0;
    if (tid < n) {
        const uint32_t x = (uint32_t)a.drafted[(uint64_t)b * a.n + tid];
        bool yes;
        if (a.temp > 0.f) {
            const double p = exp_neg(((double)row_of(a, b, tid)[x] - (double)rows[tid].top) * rt) / rows[tid].sum;
            double q = 1.0;
            if (a.draft) q = exp_neg(((double)row_of(a, b, a.n + 1u + tid)[x] - (double)rows[n + 1u + tid].top) * rt) / rows[n + 1u + tid].sum;
            yes = (double)a.u[(uint64_t)b * (a.n + 1u) + tid] * q < p;
        } else {
            yes = rows[tid].at == (int32_t)x && a.u[(uint64_t)b * (a.n + 1u) + tid] < 1.f;
        }
        if (!yes) atomicMin(&stop_w, tid);
    }
    __syncthreads();
    const uint32_t stop = stop_w;
    const bool refused = stop < n;
    if (a.temp == 0.f) {
        if (blockIdx.x == 0u) {
            int32_t *out = a.tokens + (uint64_t)b * (a.n + 1u);
            const int32_t at = rows[stop].at;
            for (uint32_t i = tid; i <= a.n; i += kThreads)
                out[i] = i < stop ? a.drafted[(uint64_t)b * a.n + i] : i == stop && (uint32_t)at < a.vocab ? at : -1;
            if (tid == 0u) a.accepted[b] = (int32_t)stop;
        }
        return;
    }
    Left left;
    left.x = row_of(a, b, stop);
    left.y = refused && a.draft ? row_of(a, b, a.n + 1u + stop) : nullptr;
    left.rt = rt;
    left.top = (double)rows[stop].top;
    left.rsum = 1.0 / rows[stop].sum;
    left.ytop = left.y ? (double)rows[n + 1u + stop].top : 0.0;
    left.yrsum = left.y ? 1.0 / rows[n + 1u + stop].sum : 0.0;
    left.without = refused && !a.draft ? a.drafted[(uint64_t)b * a.n + stop] : -1;
    double all = 0.0, less = 0.0;
    for (uint32_t i = 0; i < kEach; i++) {
        const uint32_t e = c0 + i * kThreads + tid;
        if (e >= a.vocab) break;
        double p, l;
        left.at(e, p, l);
        all += p, less += l;
    }
    all = block_sum(all, w);
    less = block_sum(less, w);
    if (tid == 0u) {
        a.left[((uint64_t)b * 2u) * a.chunks + blockIdx.x] = less;
        a.left[((uint64_t)b * 2u + 1u) * a.chunks + blockIdx.x] = all;
        if (blockIdx.x == 0u) {
            a.stop[b] = (int32_t)(stop | (refused ? 1u << 16 : 0u));
            double *st = a.stats + (uint64_t)b * 4u;
            st[0] = left.top, st[1] = left.rsum, st[2] = left.ytop, st[3] = left.yrsum;
        }
    }
}

// grid (sequences)
__global__ __launch_bounds__(kThreads) void k_verify_pick(VerifyArgs a) {
    __shared__ double scan[kThreads];
    __shared__ uint32_t found, last;
    const uint32_t b = blockIdx.x, tid = threadIdx.x;
    const uint32_t stop = (uint32_t)a.stop[b] & 0xFFFFu;
    const bool refused = (uint32_t)a.stop[b] >> 16;
    const double *st = a.stats + (uint64_t)b * 4u;
    Left left;
    left.x = row_of(a, b, stop);
    left.y = refused && a.draft ? row_of(a, b, a.n + 1u + stop) : nullptr;
    left.rt = 1.0 / (double)a.temp;
    left.top = st[0], left.rsum = st[1], left.ytop = st[2], left.yrsum = st[3];
    left.without = refused && !a.draft ? a.drafted[(uint64_t)b * a.n + stop] : -1;
    const double *sums = a.left + (uint64_t)b * 2u * a.chunks;
    double total = 0.0;
    for (uint32_t i = 0; i < a.chunks; i++) total += sums[i];
    const bool whole = !(total > 0.0) && !(total != total);  // nothing left: the target's own
    if (whole) {
        sums += a.chunks;
        total = 0.0;
        for (uint32_t i = 0; i < a.chunks; i++) total += sums[i];
    }
    int32_t next = -1;
    if (total > 0.0) {
        const double want = fmax((double)a.u[(uint64_t)b * (a.n + 1u) + a.n], 0.0) * total;
        double before = 0.0, run = 0.0;
        uint32_t chunk = 0;
        bool in = false;
        for (uint32_t i = 0; i < a.chunks && !in; i++) {
            const double to = run + sums[i];
            if (sums[i] > 0.0) chunk = i, before = run;
            in = to > want;
            run = to;
        }
        if (tid == 0u) found = 0xFFFFFFFFu, last = 0u;
        // each thread takes kEach neighbouring elements
        const uint32_t e0 = chunk * kChunk + tid * kEach;
        double mine = 0.0;
        for (uint32_t i = 0; i < kEach; i++) {
            if (e0 + i >= a.vocab) break;
            double p, l;
            left.at(e0 + i, p, l);
            mine += whole ? p : l;
        }
        scan[tid] = mine;
        __syncthreads();
        double at = before;
        for (uint32_t i = 0; i < tid; i++) at += scan[i];
        for (uint32_t i = 0; i < kEach; i++) {
            if (e0 + i >= a.vocab) break;
            double p, l;
            left.at(e0 + i, p, l);
            const double r = whole ? p : l;
            at += r;
            if (r > 0.0) atomicMax(&last, e0 + i);
            if (at > want) {
                atomicMin(&found, e0 + i);
                break;
            }
        }
        __syncthreads();
        next = (int32_t)(found != 0xFFFFFFFFu ? found : last);
    }
    int32_t *out = a.tokens + (uint64_t)b * (a.n + 1u);
    for (uint32_t i = tid; i <= a.n; i += kThreads)
        out[i] = i < stop ? a.drafted[(uint64_t)b * a.n + i] : i == stop ? next : -1;
    if (tid == 0u) a.accepted[b] = (int32_t)stop;
}

size_t plan_verify(VerifyArgs &a) {
    a.chunks = (a.vocab + kChunk - 1u) / kChunk;
    const uint64_t parts = (uint64_t)a.batch * (2u * a.n + 1u) * a.chunks;
    return parts * 16u + (uint64_t)a.batch * (a.chunks * 16u + 40u);
}

hipError_t launch_verify(VerifyArgs a, void *scratch, hipStream_t s) {
    const uint64_t parts = (uint64_t)a.batch * (2u * a.n + 1u) * a.chunks;
    a.sums = static_cast<double *>(scratch);
    a.left = a.sums + parts;
    a.stats = a.left + 2u * (uint64_t)a.batch * a.chunks;
    a.tops = reinterpret_cast<float *>(a.stats + 4u * (uint64_t)a.batch);
    a.arg = reinterpret_cast<int32_t *>(a.tops + parts);
    a.stop = a.arg + parts;
    if (a.temp == 0.f) a.draft = nullptr;
    k_verify_sum<<<dim3(a.chunks, a.n + 1u + (a.draft ? a.n : 0u), a.batch), kThreads, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    k_verify_accept<<<dim3(a.chunks, a.batch), kThreads, 0, s>>>(a);
    e = hipGetLastError();
    if (e != hipSuccess || a.temp == 0.f) return e;
    k_verify_pick<<<a.batch, kThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace vbs
