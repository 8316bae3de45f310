// vbs_kern_rows.hip — attention of several tokens over the f16 KV cache: a chunk
// of consecutive tokens (causal, with a prefix, documents, capped scores, a bias
// that depends on distance) or a tree of drafted tokens (a mask of bits), and the
// attention weight that each slot received.
//
// Row i (a token) and q head h of kv head h / group, over the slots j that the row
// sees: s_j = scale q.k_j, capped c tanh(s_j / c), less slope_h |i - j|; m = max s_j,
// l = sum e^(s_j - m), out = sum e^(s_j - m) v_j / l, and 0 where nothing is seen
// (m = -inf). The weight of slot j, e^(s_j - m) / l, is summed over the rows and
// the q heads of its kv head into mass[j]. Rows that do not see a slot take
// nothing from it, whatever is in its K and V.
#include "vbs_dev_common.h"
#include "vbs_steps.h"

namespace vbs {

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
__device__ __forceinline__ uint32_t row_end(const RowsArgs &a, uint32_t i) {
    if (a.mask) return a.past + a.n;
    return max(a.past + i + 1u, a.prefix);
}
// The score from scale q.k.
__device__ __forceinline__ float row_score(const RowsArgs &a, float s, float slope, uint32_t i, uint32_t j) {
    if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
    const uint32_t at = a.past + i;
    return fmaf(-slope, (float)(at > j ? at - j : j - at), s);
}

// ---- every shape: a wave per row and q head, a slot per lane -----------------------
// The scores of 64 slots at a time (f32 FMA chains in element order), a running
// maximum and sum, then the lanes take the head's dims and walk the 64 weights.
constexpr uint32_t kRowHd = 256;

__global__ __launch_bounds__(64) void k_row_any(RowsArgs a, float *__restrict__ stats) {
    __shared__ float qs[kRowHd], ps[64];
    const uint32_t lane = threadIdx.x, i = blockIdx.y, h = blockIdx.x, kvh = h / (a.nqh / a.nkh);
    const float *q = a.q + (uint64_t)i * a.q_stride + (uint64_t)h * a.hd;
    for (uint32_t d = lane; d < a.hd; d += 64u) qs[d] = q[d];
    __syncthreads();
    const uint64_t rstride = (uint64_t)a.nkh * a.hd, base = (uint64_t)kvh * a.hd;
    const float slope = a.slopes ? a.slopes[h] : 0.f;
    float m = -INFINITY, l = 0.f, acc[kRowHd / 64] = {};
    const uint32_t end = row_end(a, i);
    for (uint32_t j0 = 0; j0 < end; j0 += 64u) {
        const uint32_t j = j0 + lane;
        const bool sees = j < end && row_sees(a, i, j);
        float s = -INFINITY;
        if (sees) {
            const uint16_t *k = a.kc + (uint64_t)j * rstride + base;
            float dot = 0.f;
            for (uint32_t d = 0; d < a.hd; d++) dot = fmaf(qs[d], h2f(k[d]), dot);
            s = row_score(a, dot * a.scale, slope, i, j);
        }
        const uint64_t seen = __ballot(sees);
        if (!seen) continue;
        // fmaxf drops a NaN: a NaN score must come through the sum instead
        const float mn = fmaxf(m, wave_max(s)), top = mn == -INFINITY ? 0.f : mn;
        const float r = expf(m - top), p = sees ? expf(s - top) : 0.f;
        l = l * r + wave_sum(p);
        m = mn;
        ps[lane] = p;
        __syncthreads();
#pragma unroll
        for (uint32_t c = 0; c < kRowHd / 64u; c++) {
            const uint32_t d = 64u * c + lane;
            if (d >= a.hd) break;
            float x = acc[c] * r;
            for (uint32_t t = 0; t < 64u; t++)
                if (seen >> t & 1u) x = fmaf(ps[t], h2f(a.vc[(uint64_t)(j0 + t) * rstride + base + d]), x);
            acc[c] = x;
        }
        __syncthreads();
    }
#pragma unroll
    for (uint32_t c = 0; c < kRowHd / 64u; c++) {
        const uint32_t d = 64u * c + lane;
        if (d < a.hd) a.out[(uint64_t)i * a.out_stride + (uint64_t)h * a.hd + d] = l == 0.f ? 0.f : acc[c] / l;
    }
    if (stats && lane == 0) {
        float *st = stats + 2u * ((uint64_t)i * a.nqh + h);
        st[0] = m, st[1] = l;
    }
}

// The weights of one slot: a wave per slot and kv head, the lanes over (row, q head).
__global__ __launch_bounds__(64) void k_mass_any(RowsArgs a, const float *__restrict__ stats) {
    const uint32_t lane = threadIdx.x, j = blockIdx.x, kvh = blockIdx.y, group = a.nqh / a.nkh;
    const uint64_t rstride = (uint64_t)a.nkh * a.hd;
    const uint16_t *k = a.kc + (uint64_t)j * rstride + (uint64_t)kvh * a.hd;
    float sum = 0.f;
    for (uint32_t e = lane; e < a.n * group; e += 64u) {
        const uint32_t i = e / group, h = kvh * group + e % group;
        if (j >= row_end(a, i) || !row_sees(a, i, j)) continue;
        const float *q = a.q + (uint64_t)i * a.q_stride + (uint64_t)h * a.hd;
        float dot = 0.f;
        for (uint32_t d = 0; d < a.hd; d++) dot = fmaf(q[d], h2f(k[d]), dot);
        const float s = row_score(a, dot * a.scale, a.slopes ? a.slopes[h] : 0.f, i, j);
        const float m = stats[2u * ((uint64_t)i * a.nqh + h)], l = stats[2u * ((uint64_t)i * a.nqh + h) + 1u];
        if (l != 0.f) sum += expf(s - (m == -INFINITY ? 0.f : m)) / l;
    }
    sum = wave_sum(sum);
    if (lane == 0) a.mass[(uint64_t)kvh * a.max_ctx + j] += sum;
}

size_t rows_scratch_bytes(const RowsArgs &a) {
    return a.mass ? (size_t)a.n * a.nqh * 2u * sizeof(float) : 0u;
}

hipError_t launch_rows(const RowsArgs &a, void *scratch, hipStream_t s) {
    float *stats = a.mass ? static_cast<float *>(scratch) : nullptr;
    k_row_any<<<dim3(a.nqh, a.n), 64, 0, s>>>(a, stats);
    if (a.mass) k_mass_any<<<dim3(a.past + a.n, a.nkh), 64, 0, s>>>(a, stats);
    return hipGetLastError();
}

}  // namespace vbs
