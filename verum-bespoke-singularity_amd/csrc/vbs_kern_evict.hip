// vbs_kern_evict.hip — the f16 KV cache cut to a budget of slots by the attention
// weight they accumulated.
//
// Per layer and kv head: the first and the last slots stay, and of those between
// the ones of the greatest weight (the lowest slot among equals; a NaN counts
// as the lowest weight there is). Two launches: k_evict_select writes the kept
// slots in order (one workgroup per layer and head: the weight of the last slot
// taken by a radix selection over the 32-bit order of floats, then one ordered
// pass), k_evict_move moves their K and V rows to the front.
//
// The move is in place. A kept slot never moves up (its new place is the number
// of kept slots before it), so rows taken in ascending order are safe as long as
// every row of a batch is in registers before the first of them is written: what
// earlier batches wrote lies below this batch's first place, and so below its
// slots. A workgroup owns a column slice of one head's rows (of K or of V) and
// walks all kept slots; the slices share nothing.
#include "vbs_dev_common.h"
#include "vbs_steps.h"

namespace vbs {

constexpr uint32_t kSelThreads = 1024, kSelWaves = kSelThreads / 64;

// The order of weights as unsigned numbers: -0 as 0, NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (__builtin_isnan(w)) return 0u;
    const uint32_t u = vbs_float_to_bits(w == 0.f ? 0.f : w);
    return u >> 31 ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kSelThreads) void k_evict_select(EvictArgs a) {
    __shared__ uint32_t hist[256], waves[2][kSelWaves], s_prefix, s_need;
    const uint32_t t = threadIdx.x, wave = t >> 6, lane = t & 63u, h = blockIdx.x, l = blockIdx.y;
    const float *mass = a.mass + ((uint64_t)l * a.nkh + h) * a.max_ctx;
    float *mass_out = a.mass_out ? a.mass_out + ((uint64_t)l * a.nkh + h) * a.max_ctx : nullptr;
    uint32_t *kept = a.kept + ((uint64_t)l * a.nkh + h) * a.budget;
    const uint32_t lo = a.first, hi = a.len - a.last;  // the slots that are chosen among
    uint32_t need = a.budget - a.first - a.last;       // as many of them

    // the key of the need-th greatest, eight bits a pass; `need` becomes how many of
    // that key are taken
    uint32_t prefix = 0;
    if (need > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (t < 256u) hist[t] = 0;
            __syncthreads();
            for (uint32_t j = lo + t; j < hi; j += kSelThreads) {
                const uint32_t key = weight_key(mass[j]);
                if (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[key >> shift & 255u], 1u);
            }
            __syncthreads();
            if (t == 0) {
                uint32_t b = 255u, n = need;
                while (b > 0u && hist[b] < n) n -= hist[b--];
                s_prefix = prefix | b << shift;
                s_need = n;
            }
            __syncthreads();
            prefix = s_prefix;
            need = s_need;
        }
    }
    const bool any = a.budget > a.first + a.last;

    // one ordered pass: ties of the last key in slot order, kept slots in slot order
    uint32_t ties0 = 0, kept0 = 0;
    for (uint32_t j0 = 0; j0 < a.len; j0 += kSelThreads) {
        const uint32_t j = j0 + t;
        const float w = j < a.len ? mass[j] : 0.f;
        const uint32_t key = weight_key(w);
        const bool open = j >= lo && j < hi, tie = any && open && key == prefix;
        const uint64_t tb = __ballot(tie), below = (1ull << lane) - 1ull;
        if (lane == 0) waves[0][wave] = (uint32_t)__popcll(tb);
        __syncthreads();
        uint32_t before = ties0;
        for (uint32_t v = 0; v < kSelWaves; v++) {
            if (v < wave) before += waves[0][v];
            ties0 += waves[0][v];
        }
        before += (uint32_t)__popcll(tb & below);
        const bool keep = j < a.len && (!open || (any && (key > prefix || (tie && before < need))));
        const uint64_t kb = __ballot(keep);
        if (lane == 0) waves[1][wave] = (uint32_t)__popcll(kb);
        __syncthreads();
        uint32_t at = kept0;
        for (uint32_t v = 0; v < kSelWaves; v++) {
            if (v < wave) at += waves[1][v];
            kept0 += waves[1][v];
        }
        at += (uint32_t)__popcll(kb & below);
        if (keep) {
            kept[at] = j;
            if (mass_out) mass_out[at] = w;  // (at <= j: read above, or by an earlier pass)
        }
    }
    __syncthreads();
    if (mass_out)
        for (uint32_t j = a.budget + t; j < a.len; j += kSelThreads) mass_out[j] = 0.f;
}

// A slice: `lanes` units of type U of one head's rows. Threads: (row, unit).
constexpr uint32_t kMoveThreads = 512, kMoveDepth = 4;

template <class U>
__global__ __launch_bounds__(kMoveThreads) void k_evict_move(EvictArgs a, uint32_t lanes, uint32_t slices) {
    const uint32_t t = threadIdx.x, rows = kMoveThreads / lanes, row = t / lanes;
    const uint32_t slice = blockIdx.x % slices, h = blockIdx.x / slices;
    const uint32_t units = a.hd * 2u / (uint32_t)sizeof(U), u = slice * lanes + t % lanes;
    const uint32_t *kept = a.kept + ((uint64_t)blockIdx.y * a.nkh + h) * a.budget;
    U *c = reinterpret_cast<U *>(blockIdx.z ? a.vc : a.kc) + ((uint64_t)blockIdx.y * a.max_ctx * a.nkh + h) * units + u;
    const uint64_t stride = (uint64_t)a.nkh * units;
    const bool mine = row < rows && u < units;
    U v[2][kMoveDepth];
    uint32_t from[2][kMoveDepth];
    auto load = [&](uint32_t b, U(&x)[kMoveDepth], uint32_t(&f)[kMoveDepth]) {
#pragma unroll
        for (uint32_t k = 0; k < kMoveDepth; k++) {
            const uint32_t i = (b * kMoveDepth + k) * rows + row;
            f[k] = mine && i < a.budget ? kept[i] : i;
            if (f[k] != i) x[k] = c[f[k] * stride];
        }
    };
    auto store = [&](uint32_t b, const U(&x)[kMoveDepth], const uint32_t(&f)[kMoveDepth]) {
#pragma unroll
        for (uint32_t k = 0; k < kMoveDepth; k++) {
            const uint32_t i = (b * kMoveDepth + k) * rows + row;
            if (f[k] != i) c[i * stride] = x[k];
        }
    };
    const uint32_t per = kMoveDepth * rows, batches = (a.budget + per - 1u) / per;
    load(0u, v[0], from[0]);
    for (uint32_t b = 0; b < batches; b += 2u) {
#pragma unroll
        for (uint32_t o = 0; o < 2u; o++) {
            if (b + o >= batches) break;
            // every row of this batch has arrived, in every wave, before the first is written
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            // the next batch's rows lie above every place of this one
            if (b + o + 1u < batches) load(b + o + 1u, v[1u - o], from[1u - o]);
            store(b + o, v[o], from[o]);
        }
    }
}

hipError_t launch_evict(const EvictArgs &a, hipStream_t s) {
    k_evict_select<<<dim3(a.nkh, a.n_layers), kSelThreads, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const bool wide = a.hd % 8u == 0 && (((uintptr_t)a.kc | (uintptr_t)a.vc) & 15u) == 0;
    const uint32_t units = wide ? a.hd / 8u : a.hd, want = wide ? 4u : 32u;
    const uint32_t lanes = units < want ? units : want, slices = (units + lanes - 1u) / lanes;
    const dim3 grid(a.nkh * slices, a.n_layers, 2);
    if (wide)
        k_evict_move<uint4><<<grid, kMoveThreads, 0, s>>>(a, lanes, slices);
    else
        k_evict_move<uint16_t><<<grid, kMoveThreads, 0, s>>>(a, lanes, slices);
    return hipGetLastError();
}

}  // namespace vbs
