// vbs_kern_evict.hip — the f16 KV cache cut to a budget of slots by the attention
// weight they accumulated.
//
// Per layer and kv head: the first and the last slots stay, and of those between
// the ones of the greatest weight (the lowest slot among equals; a NaN counts
// as the lowest weight there is). k_evict_select writes the kept
// slots in order (one workgroup per layer and head: the weight of the last slot
// taken by a radix selection over the 32-bit order of floats, then one ordered
// pass), k_evict_move moves their K and V rows to the front; k_evict does both, for
// few heads or long moves.
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

constexpr uint32_t kSelThreads = 1024, kSelWaves = kSelThreads / 64, kSelBins = 2048;
constexpr uint32_t kSelKeys = 8, kSelRun = kSelThreads * kSelKeys;  // most slots a thread and a workgroup hold at once

// The order of weights as unsigned numbers: -0 as 0, NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (__builtin_isnan(w)) return 0u;
    const uint32_t u = vbs_float_to_bits(w == 0.f ? 0.f : w);
    return u >> 31 ? ~u : u | 0x80000000u;
}

// Inclusive sum over the lanes up to each: within the rows of 16 lanes, then the rows before added (DPP row_shr and
// row_bcast; lanes without a source add 0). The whole wave must be active.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // lane 15 of rows 0, 2 to rows 1, 3
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);  // lane 31 to rows 2, 3
    return v;
}
// The sum of the waves' entries before `wave`, and of all.
__device__ __forceinline__ uint2 waves_before(const uint32_t *waves, uint32_t wave) {
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t v = 0; v < kSelWaves; v++) {
        const uint32_t x = waves[v];
        if (v < wave) before += x;
        all += x;
    }
    return make_uint2(before, all);
}

// The selection of one layer and head by a workgroup: put(place, slot, weight) for every kept slot.
template <uint32_t KEYS, class Put>
__device__ __forceinline__ void evict_select(const EvictArgs &a, const float *mass, Put put) {
    __shared__ uint32_t hist[kSelBins], waves[2][kSelWaves], s_bin, s_need, s_count;
    const uint32_t t = threadIdx.x, wave = t >> 6, lane = t & 63u;
    const uint32_t lo = a.first, hi = a.len - a.last;  // the slots that are chosen among
    uint32_t need = a.budget - a.first - a.last;       // as many of them

    // a run of slots in registers, 64 KEYS in a row to each wave; the weights stay there if one run holds them all
    constexpr uint32_t RUN = kSelThreads * KEYS;
    const uint32_t runs = (a.len + RUN - 1u) / RUN;
    float w[KEYS];
    uint32_t key[KEYS], is_open = 0;  // (bits of the slots that are chosen among)
    auto slot = [&](uint32_t run, uint32_t k) { return run * RUN + (wave * KEYS + k) * 64u + lane; };
    auto load = [&](uint32_t run) {
        is_open = 0;
#pragma unroll
        for (uint32_t k = 0; k < KEYS; k++) w[k] = slot(run, k) < a.len ? mass[slot(run, k)] : 0.f;
#pragma unroll
        for (uint32_t k = 0; k < KEYS; k++) {
            key[k] = weight_key(w[k]);
            is_open |= (slot(run, k) >= lo && slot(run, k) < hi ? 1u : 0u) << k;
        }
    };
    load(0u);

    // the first bits of the key of the need-th greatest, up to 11 a pass: every key with
    // greater bits is kept, and `need` of those that share them (all, once `whole`)
    uint32_t prefix = 0, bits = 0;
    bool whole = false;
    for (uint32_t pass = 0; pass < 3u && need > 0u && !whole; pass++) {
        const uint32_t width = pass < 2u ? 11u : 10u, shift = 32u - bits - width;
        for (uint32_t i = t; i < kSelBins; i += kSelThreads) hist[i] = 0;
        __syncthreads();
        for (uint32_t run = 0; run < runs; run++) {
            if (runs > 1u) load(run);
#pragma unroll
            for (uint32_t k = 0; k < KEYS; k++)
                if ((is_open >> k & 1u) && (bits == 0u || key[k] >> (32u - bits) == prefix))
                    atomicAdd(&hist[key[k] >> shift & ((1u << width) - 1u)], 1u);
        }
        __syncthreads();
        // thread t takes the bins 2 t and 2 t + 1 counted from the greatest
        const uint32_t top = kSelBins - 1u - 2u * t, n0 = hist[top], n1 = hist[top - 1u];
        const uint32_t sum = wave_scan(n0 + n1);
        if (lane == 63u) waves[0][wave] = sum;
        __syncthreads();
        const uint32_t before = waves_before(waves[0], wave).x + sum - n0 - n1;
        if (before < need && need <= before + n0 + n1) {  // (one thread)
            const bool first = need <= before + n0;
            s_bin = first ? top : top - 1u;
            s_need = need - before - (first ? 0u : n0);
            s_count = first ? n0 : n1;
        }
        __syncthreads();
        prefix = prefix << width | s_bin;
        bits += width;
        need = s_need;
        whole = need == s_count;
    }
    const bool any = bits > 0u;
    const uint32_t down = 32u - bits;

    // ordered passes over the runs: ties of the last key in slot order, kept slots in slot order
    uint32_t ties0 = 0, kept0 = 0;
    for (uint32_t run = 0; run < runs; run++) {
        if (runs > 1u) load(run);  // (what earlier runs wrote lies below this run's slots)
        uint32_t tie = 0, keep = 0, n = 0;  // bits per key; the wave's count
#pragma unroll
        for (uint32_t k = 0; k < KEYS; k++) {
            const uint32_t head = any ? key[k] >> down : 0u;
            const bool open = is_open >> k & 1u;
            if (any && open && head == prefix) tie |= 1u << k;
            if (slot(run, k) < a.len && (!open || (any && head > prefix))) keep |= 1u << k;
        }
        if (whole) {
            keep |= tie;
        } else if (any) {
#pragma unroll
            for (uint32_t k = 0; k < KEYS; k++) n += (uint32_t)__popcll(__ballot(tie >> k & 1u));
            if (lane == 0) waves[0][wave] = n;
            __syncthreads();
            const uint2 b = waves_before(waves[0], wave);
            uint32_t at = ties0 + b.x;
            ties0 += b.y;
#pragma unroll
            for (uint32_t k = 0; k < KEYS; k++) {
                const uint64_t m = __ballot(tie >> k & 1u);
                if ((tie >> k & 1u) && at + (uint32_t)__popcll(m & ((1ull << lane) - 1ull)) < need) keep |= 1u << k;
                at += (uint32_t)__popcll(m);
            }
        }
        n = 0;
#pragma unroll
        for (uint32_t k = 0; k < KEYS; k++) n += (uint32_t)__popcll(__ballot(keep >> k & 1u));
        if (lane == 0) waves[1][wave] = n;
        __syncthreads();  // (every weight of this run is in a register)
        const uint2 b = waves_before(waves[1], wave);
        uint32_t at = kept0 + b.x;
        kept0 += b.y;
#pragma unroll
        for (uint32_t k = 0; k < KEYS; k++) {
            const uint64_t m = __ballot(keep >> k & 1u);
            if (keep >> k & 1u) {
                const uint32_t to = at + (uint32_t)__popcll(m & ((1ull << lane) - 1ull));
                put(to, slot(run, k), w[k]);  // (to <= the slot)
            }
            at += (uint32_t)__popcll(m);
        }
        if (runs > 1u) __syncthreads();  // (the counts are read before the next run's)
    }
    __syncthreads();
}

template <uint32_t KEYS>
__global__ __launch_bounds__(kSelThreads) void k_evict_select(EvictArgs a) {
    const uint64_t lh = (uint64_t)blockIdx.y * a.nkh + blockIdx.x;
    float *mass_out = a.mass_out ? a.mass_out + lh * a.max_ctx : nullptr;
    uint32_t *kept = a.kept + lh * a.budget;
    evict_select<KEYS>(a, a.mass + lh * a.max_ctx, [&](uint32_t to, uint32_t slot, float w) {
        kept[to] = slot;
        if (mass_out) mass_out[to] = w;
    });
    if (mass_out)
        for (uint32_t j = a.budget + threadIdx.x; j < a.len; j += kSelThreads) mass_out[j] = 0.f;
}

// A slice: `lanes` units of type U of one head's rows, of K or of V. Threads: (row, unit).
// Workgroups whose slices share rows follow each other by the number of XCDs, so
// that they run on one, which then has the rows' other bytes in its L2.
constexpr uint32_t kMoveThreads = 512, kMoveDepth = 4, kXcds = 8;
typedef uint32_t eu4 __attribute__((ext_vector_type(4)));

struct MoveOf {  // whose rows this workgroup moves: the unit (layer, head, K or V) and the slice of them
    uint32_t unit, slice;
    bool any;
    __device__ MoveOf(const EvictArgs &a, uint32_t slices)
        : unit(blockIdx.x / (kXcds * slices) * kXcds + blockIdx.x % kXcds), slice(blockIdx.x / kXcds % slices),
          any(unit < 2u * a.nkh * a.n_layers) {}  // (the grid is whole groups of kXcds units)
};

template <class U, uint32_t THREADS, class Id>
__device__ __forceinline__ void evict_move(const EvictArgs &a, MoveOf of, uint32_t lanes, const Id *kept) {
    const uint32_t t = threadIdx.x, rows = THREADS / lanes, row = t / lanes, unit = of.unit;
    const uint32_t l = (unit >> 1) / a.nkh, h = (unit >> 1) % a.nkh;
    const uint32_t units = a.hd * 2u / (uint32_t)sizeof(U), u = of.slice * lanes + t % lanes;
    U *c = reinterpret_cast<U *>(unit & 1u ? a.vc : a.kc) + ((uint64_t)l * a.max_ctx * a.nkh + h) * units + u;
    const uint64_t stride = (uint64_t)a.nkh * units;
    const uint32_t budget = row < rows && u < units ? a.budget : 0u;  // (threads past the slice have nothing)
    // the slots of the batch to write, of the one whose rows are on their way and of the one behind it
    uint32_t fa[kMoveDepth], fb[kMoveDepth], fc[kMoveDepth];
    U v0[kMoveDepth], v1[kMoveDepth];
    auto place = [&](uint32_t b, uint32_t k) { return (b * kMoveDepth + k) * rows + row; };
    auto ids = [&](uint32_t b, uint32_t(&f)[kMoveDepth]) {
#pragma unroll
        for (uint32_t k = 0; k < kMoveDepth; k++) f[k] = place(b, k) < budget ? kept[place(b, k)] : place(b, k);
    };
    auto load = [&](uint32_t b, U(&x)[kMoveDepth]) {
#pragma unroll
        for (uint32_t k = 0; k < kMoveDepth; k++)
            if (fb[k] != place(b, k)) x[k] = c[fb[k] * stride];
    };
    const uint32_t per = kMoveDepth * rows, batches = (a.budget + per - 1u) / per;
    // every row of the batch at hand has arrived, in every wave, before the first is written;
    // the next batch's rows lie above every place of it
    auto turn = [&](uint32_t b, const U(&x)[kMoveDepth], U(&y)[kMoveDepth]) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < kMoveDepth; k++) fa[k] = fb[k], fb[k] = fc[k];
        if (b + 1u < batches) load(b + 1u, y);
        ids(b + 2u, fc);
#pragma unroll
        for (uint32_t k = 0; k < kMoveDepth; k++)
            if (fa[k] != place(b, k)) c[place(b, k) * stride] = x[k];
    };
    ids(0u, fb);
    load(0u, v0);
    ids(1u, fc);
    for (uint32_t b = 0; b < batches; b += 2u) {
        turn(b, v0, v1);
        if (b + 1u < batches) turn(b + 1u, v1, v0);
    }
}

template <class U>
__global__ __launch_bounds__(kMoveThreads) void k_evict_move(EvictArgs a, uint32_t lanes, uint32_t slices) {
    const MoveOf of(a, slices);
    if (of.any) evict_move<U, kMoveThreads>(a, of, lanes, a.kept + (uint64_t)(of.unit >> 1) * a.budget);
}

// Both in one launch, where a run holds every slot: each workgroup of a head selects for itself, and one of them
// writes what the caller gets. Not where mass_out is mass, which the others may still have to read.
template <class U, uint32_t KEYS>
__global__ __launch_bounds__(kSelThreads) void k_evict(EvictArgs a, uint32_t lanes, uint32_t slices) {
    __shared__ uint16_t ids[kSelThreads * KEYS];
    const MoveOf of(a, slices);
    if (!of.any) return;
    const uint64_t lh = of.unit >> 1;
    const bool tells = !(of.unit & 1u) && of.slice == 0u;
    float *mass_out = tells && a.mass_out ? a.mass_out + lh * a.max_ctx : nullptr;
    uint32_t *kept = a.kept + lh * a.budget;
    evict_select<KEYS>(a, a.mass + lh * a.max_ctx, [&](uint32_t to, uint32_t slot, float w) {
        ids[to] = (uint16_t)slot;
        if (tells) kept[to] = slot;
        if (mass_out) mass_out[to] = w;
    });
    if (mass_out)
        for (uint32_t j = a.budget + threadIdx.x; j < a.len; j += kSelThreads) mass_out[j] = 0.f;
    evict_move<U, kSelThreads>(a, of, lanes, ids);
}

hipError_t launch_evict(const EvictArgs &a, hipStream_t s) {
    const bool wide = a.hd % 8u == 0 && (((uintptr_t)a.kc | (uintptr_t)a.vc) & 15u) == 0;
    // Whole rows a workgroup where that gives a workgroup per CU (32 layers of 8 heads of 128, 8192
    // slots to 4096: 223 us, 4.8 TB/s read and written; half rows 253, quarters 303, eighths 335), else
    // narrower slices, down to 32 bytes (one such layer, 2049 to 1024, the move as a launch of its own: 3.5 us; whole
    // rows 11.2).
    const uint32_t units = wide ? a.hd / 8u : a.hd, pairs = 2u * a.nkh * a.n_layers, least = wide ? 2u : 16u;
    uint32_t lanes = units;
    while (lanes > least && pairs * ((units + lanes - 1u) / lanes) < 256u) lanes = (lanes + 1u) / 2u;
    const uint32_t slices = (units + lanes - 1u) / lanes;
    const uint32_t grid = (pairs + kXcds - 1u) / kXcds * kXcds * slices;
    // Four slots a thread where they hold every slot: every pass is half as long (2049 slots: the selection 9.2 us under
    // the tracer with eight, 6.7 with four). One launch for up to two workgroups per CU (2049 to 1024 of 8 heads 8.7 us,
    // two launches 10.0; 32 layers of 8192 to 4096 229 and 236), or where the move is long beside the selection, which
    // one launch does for K and for V (64 layers of 8 heads, 4096 to 2048: 232 and 241; but 8192 to 256 57 and 50, 1024
    // to 512 53 and 50, 128 layers of 512 to 256 59 and 39).
    const bool small = a.len <= kSelThreads * 4u, one = grid <= 512u || (a.budget >= 1024u && a.len / 2u <= a.budget);
    if (a.len <= kSelRun && a.mass_out != a.mass && one) {
        if (small && wide)
            k_evict<eu4, 4><<<grid, kSelThreads, 0, s>>>(a, lanes, slices);
        else if (wide)
            k_evict<eu4, 8><<<grid, kSelThreads, 0, s>>>(a, lanes, slices);
        else if (small)
            k_evict<uint16_t, 4><<<grid, kSelThreads, 0, s>>>(a, lanes, slices);
        else
            k_evict<uint16_t, 8><<<grid, kSelThreads, 0, s>>>(a, lanes, slices);
        return hipGetLastError();
    }
    if (small)
        k_evict_select<4><<<dim3(a.nkh, a.n_layers), kSelThreads, 0, s>>>(a);
    else
        k_evict_select<8><<<dim3(a.nkh, a.n_layers), kSelThreads, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (wide)
        k_evict_move<eu4><<<grid, kMoveThreads, 0, s>>>(a, lanes, slices);
    else
        k_evict_move<uint16_t><<<grid, kMoveThreads, 0, s>>>(a, lanes, slices);
    return hipGetLastError();
}

}  // namespace vbs
