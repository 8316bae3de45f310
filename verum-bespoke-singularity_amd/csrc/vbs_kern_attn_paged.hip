// vbs_kern_attn_paged.hip — the attention of single tokens over the paged cache.
//
// Row r (one token; up to eight of its q heads of one kv head are the columns of a product, 9 to 16 those of two):
// out = sum_j w_j v_j, w = softmax(scale q.k_j) over the slots j < lens[r]. The units of 32
// slots of all rows and heads are shared out evenly over the workgroups that run at once, and
// within one over its four waves; each keeps the running maximum m (in log2), the sum l and O of
// its own units, the four are joined through LDS and the workgroups' by k_attn_paged_merge.
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
// Bound: HBM where the caches are large (a workgroup reads its next unit while it computes, 64 KB or
// more in flight a CU): 64 sequences of 4096 slots, 32/8 heads of 128, 5.7 TB/s of F16 (188 us) and 5.2 of
// Q8_0 (111); launches and round trips where they are small: one sequence of 2048 slots 11.6 us, of which
// the merge 4. Workgroups of fewer units each, in more than one round, cost 12 us of start each (lengths, table, first
// unit, one after the other) under load: 264 us for 111 at four units a workgroup.
#include <math.h>

#include "vbs_dev_common.h"
#include "vbs_pages.h"

namespace vbs {

namespace {

typedef _Float16 ph8 __attribute__((ext_vector_type(8)));
typedef _Float16 ph2 __attribute__((ext_vector_type(2)));
typedef float pf2 __attribute__((ext_vector_type(2)));
typedef float pf4 __attribute__((ext_vector_type(4)));
typedef uint32_t pu4 __attribute__((ext_vector_type(4)));

constexpr float kPagedLog2e = 1.44269504088896341f;
constexpr uint32_t kWaves = 4;
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
    const ph2 off = {(_Float16)1152.f, (_Float16)1152.f};
    const ph2 p0 = __builtin_bit_cast(ph2, __builtin_amdgcn_perm(e, lo, 0x04010400u)) - off;
    const ph2 p1 = __builtin_bit_cast(ph2, __builtin_amdgcn_perm(e, lo, 0x04030402u)) - off;
    const ph2 p2 = __builtin_bit_cast(ph2, __builtin_amdgcn_perm(e, hi, 0x04010400u)) - off;
    const ph2 p3 = __builtin_bit_cast(ph2, __builtin_amdgcn_perm(e, hi, 0x04030402u)) - off;
    return ph8{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

// Of eight values the high f16 part where low is 0, and the low part, of what the high one leaves, where it is -1.
__device__ __forceinline__ ph8 parts(const float x[8], float low) {
    ph2 r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const ph2 h = __builtin_convertvector((pf2{x[2 * i], x[2 * i + 1]}), ph2);
        const float l0 = fmaf(low, (float)h[0], x[2 * i]), l1 = fmaf(low, (float)h[1], x[2 * i + 1]);
        r[i] = __builtin_convertvector((pf2{l0, l1}), ph2);
    }
    return ph8{r[0][0], r[0][1], r[1][0], r[1][1], r[2][0], r[2][1], r[3][0], r[3][1]};
}

// A row: its sequence, its slots (0 where one of the two is out of range: the row is NaN) and units.
struct Row {
    int32_t seq;
    uint32_t len, units;
    bool bad;
};
__device__ __forceinline__ Row row_at(const PagedAttnArgs &a, uint32_t row) {
    Row r;
    r.seq = a.seq ? a.seq[row] : (int32_t)row;
    const int32_t len = a.lens[row];
    r.bad = len < 0 || (uint32_t)len > a.max_len || (uint32_t)r.seq >= a.p.n_seqs;
    r.len = r.bad ? 0u : (uint32_t)len;
    r.units = (r.len + kUnit - 1u) / kUnit;
    return r;
}

// What every lane holds, told to the compiler.
__device__ __forceinline__ uint64_t same(uint64_t v) {
    return (uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32 | __builtin_amdgcn_readfirstlane((uint32_t)v);
}

// How the units of all rows and heads are shared out. They lie in one line: row by row, within a row kv head (and tile of q
// heads) by head, within that slot by slot, and a workgroup takes `share` of them, so all have the same work whatever the
// lengths. Shares of few units (kAlignedShare) begin and end with their head, which `grain` pads in the line: a
// second piece's start would take as long as the share: one row of 600 slots takes 11.9 us and without 15.6, 4 of 1500
// 14.6 and 18.9 (Q8_0, 32 q and 8 kv heads of 128). With up to 64 units instead of 16, 40 rows of 1500 take 53.2 for 42.0 and 20
// of up to 3000 take 35.6 for 30.9, but 4 of 9000 take 24.8 for 29.0, 40 of 600 22.6 for 29.6 and one of 20000 20.7 for 25.0:
// those whose padded shares are still one round of the workgroups that run at once (480, 320 and 256 of 512), where 40
// of 1500 have 640. 16 keeps the first two from their loss and leaves the others' gain. One workgroup
// a CU where the line is short: 8 heads of one row of 8192 slots take 18.2 us with 256 workgroups (Q8_0, 128 elements) and
// 23.4 with 512, of 8 rows 44.6 and 38.5.
constexpr uint32_t kAlignedShare = 16, kShortLine = 8192;

struct Shares {
    uint64_t share, grain;
};
__device__ __forceinline__ Shares shares(const PagedAttnArgs &a, uint64_t units, uint32_t line) {  // units: of a head, all rows
    const uint64_t all = units * line;
    const uint32_t workgroups = all < kShortLine ? min(a.workgroups, 256u) : a.workgroups;
    Shares s;
    s.share = (all + workgroups - 1u) / workgroups;
    s.share = max((s.share + kWaves - 1u) / kWaves, (uint64_t)1) * kWaves;  // (not 0 where no row has a unit: `grain` divides)
    s.grain = a.aligned && s.share <= kAlignedShare ? s.share : 1u;
    return s;
}
__device__ __forceinline__ uint64_t padded(const Shares &s, uint32_t units) {
    return s.grain == 1u ? units : (units + s.grain - 1u) / s.grain * s.grain;
}
// The sum of v over a workgroup of 256 threads; w: 4 words.
__device__ __forceinline__ uint64_t sum_of_256(uint64_t v, uint64_t *w) {
    for (uint32_t o = 32; o; o >>= 1) v += __shfl_xor((unsigned long long)v, (int)o, 64);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) w[threadIdx.x >> 6] = v;
    __syncthreads();
    return same((w[0] + w[1]) + (w[2] + w[3]));
}
__device__ __forceinline__ uint64_t wave_total(uint64_t v) {
    for (uint32_t o = 32; o; o >>= 1) v += __shfl_xor((unsigned long long)v, (int)o, 64);
    return same(v);
}
// v summed over the lanes up to each.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v, uint32_t lane) {
    for (uint32_t o = 1; o < 64u; o <<= 1) {
        const uint64_t t = __shfl_up((unsigned long long)v, (int)o, 64);
        if (lane >= o) v += t;
    }
    return v;
}

// The row that unit `at` of the line lies in, and where the row begins (padded units of a head before it); false where
// the line ends before. Up to 64 rows every wave looks by itself, a row a lane; beyond, the workgroup's
// 256 threads, thread t the rows t R .. t R + R - 1.
struct Found {
    uint32_t row;
    uint64_t before;
};
__device__ __forceinline__ bool find_row(const PagedAttnArgs &a, uint32_t line, uint32_t workgroup, Shares &sh, uint64_t &at, uint64_t &end,
                                         Found &f, uint64_t *sums) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    if (a.rows <= 64u) {
        const uint32_t units = lane < a.rows ? row_at(a, lane).units : 0u;
        if (a.rows == 1u) {
            const uint32_t n = __builtin_amdgcn_readfirstlane(units);
            sh = shares(a, n, line);
            at = workgroup * sh.share, end = padded(sh, n) * line;
            end = min(end, at + sh.share);
            f.row = 0u, f.before = 0u;
            return at < end;
        }
        sh = shares(a, wave_total(units), line);
        const uint64_t mine = padded(sh, units), to = wave_scan(mine, lane);
        at = workgroup * sh.share;
        const uint64_t here = __ballot(at < to * line);
        if (here == 0u) return false;
        const uint64_t all = __shfl((unsigned long long)to, 63, 64), before = __shfl((unsigned long long)(to - mine), __ffsll((unsigned long long)here) - 1, 64);
        end = min(at + sh.share, same(all) * line);
        f.row = (uint32_t)__ffsll((unsigned long long)here) - 1u, f.before = same(before);
        return true;
    }
    __shared__ Found found;
    const uint32_t each = (a.rows + 255u) / 256u, r0 = min(tid * each, a.rows), r1 = min(r0 + each, a.rows);
    uint64_t mine = 0;
    for (uint32_t r = r0; r < r1; r++) mine += row_at(a, r).units;
    sh = shares(a, sum_of_256(mine, sums), line);
    if (sh.grain != 1u) {
        mine = 0;
        for (uint32_t r = r0; r < r1; r++) mine += padded(sh, row_at(a, r).units);
    }
    uint64_t to = wave_scan(mine, lane), all = 0;
    __syncthreads();
    if (lane == 63u) sums[wave] = to;
    __syncthreads();
    for (uint32_t w = 0; w < kWaves; w++) {
        if (w < wave) to += sums[w];
        all += sums[w];
    }
    at = workgroup * sh.share;
    end = min(at + sh.share, same(all) * line);
    if (at >= end) return false;
    uint64_t before = to - mine;
    if (before * line <= at && at < to * line) {
        uint32_t r = r0;
        for (;; r++) {
            const uint64_t n = padded(sh, row_at(a, r).units);
            if ((before + n) * line > at) break;
            before += n;
        }
        found = Found{r, before};
    }
    __syncthreads();
    f.row = __builtin_amdgcn_readfirstlane(found.row), f.before = same(found.before);
    return true;
}
// Workgroups of a CU, by the registers of a unit in flight (64 sequences of 4096 slots, 8 kv heads, Q8_0: heads of 32
// take 43 us with four and 53 with two, of 128 111 with two and 121 with three, of 192 162 with two and 193 with one, of
// 224 and 256, which spill with two, 220 and 249 with one, 230 and 338 with two).
constexpr uint32_t per_cu(uint32_t nb) { return nb == 1u ? 4u : nb <= 6u ? 2u : 1u; }

// A unit of K or of V on its way: its values as an operand takes them, and (Q8_0) its 32 NB scales, two in a dword, dword
// 64 i + lane in ds[i].
template <uint32_t NB, bool Q8>
struct Half {
    static constexpr uint32_t kValues = Q8 ? NB : 2 * NB, kScales = Q8 ? (NB + 3u) / 4u : 1u;
    pu4 x[kValues];
    uint32_t ds[kScales];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (uint32_t i = 0; i < kValues; i++) x[i] = pu4{0u, 0u, 0u, 0u};
#pragma unroll
        for (uint32_t i = 0; i < kScales; i++) ds[i] = 0u;
    }
    __device__ __forceinline__ void load(const uint8_t *p, uint32_t lane) {
#pragma unroll
        for (uint32_t i = 0; i < kValues; i++) x[i] = *reinterpret_cast<const pu4 *>(p + i * 1024u + lane * 16u);
        if constexpr (Q8) {
#pragma unroll
            for (uint32_t i = 0; i < kScales; i++)
                if (64u * i + lane < NB * 16u) ds[i] = *reinterpret_cast<const uint32_t *>(p + NB * 1024u + i * 256u + lane * 4u);
        }
    }
    // The scales through LDS (a wave's own words): every lane reads the eight of its slots, block by block.
    __device__ __forceinline__ void spread(uint32_t *w, uint32_t lane) const {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (uint32_t i = 0; i < kScales; i++)
            if (64u * i + lane < NB * 16u) w[64u * i + lane] = ds[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
};

}  // namespace

// The slots [32 u0, min(32 u1, len)) of a sequence again for one q head, in f32 products and sums: m, l and O (thread d
// holds element d). `w` holds 256 floats.
template <bool Q8>
__device__ __forceinline__ void slow_tile(const PagedAttnArgs &a, int32_t seq, uint32_t u0, uint32_t u1, uint32_t len, uint32_t kvh,
                                       const float *q, float *w, float &m, float &l, float &o) {
    const uint32_t tid = threadIdx.x, hd = a.p.hd, nb = a.p.nb, end = min(u1 * kUnit, len);
    m = -INFINITY, l = 0.f, o = 0.f;
    for (uint32_t j0 = u0 * kUnit; j0 < end; j0 += 256u) {
        const uint32_t j = j0 + tid, count = min(256u, end - j0);
        float s = 0.f;
        if (j < end) {
            const int32_t page = page_at(a.p, seq, j / kUnit);
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
            const int32_t page = page_at(a.p, seq, jj / kUnit);
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

// o is written and the scales are read 16 bytes at a time.
template <uint32_t NB, uint32_t CT>
struct Shared {
    alignas(16) float o[kWaves][8u * CT][NB * 32u + 4u];
    float m[kWaves][8u * CT], l[kWaves][8u * CT];
    alignas(16) uint32_t scales[kWaves][2][NB * 16u];
    uint32_t odd;
    static_assert((NB * 32u + 4u) % 4u == 0u && NB * 16u % 4u == 0u, "rows of 16 bytes");
};

// Units [u0, u1) of a row and a kv head (and tile of its q heads), by a workgroup: to out, or as a partial
// result if part is given. False, and nothing written, where sums are not finite (slow_units then does it).
template <uint32_t NB, bool Q8, uint32_t CT>
__device__ __forceinline__ bool attend_units(const PagedAttnArgs &a, Shared<NB, CT> &sh, uint32_t row, uint32_t hx, int32_t seq, uint32_t len,
                                             uint32_t u0, uint32_t u1, float *part, float2 *ml) {
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t lane = tid & 63u;
    asm volatile("" : "+v"(lane));  // (else what depends on the lane alone is kept from piece to piece: 60 registers more, and spills)
    const uint32_t g = lane >> 4, c = lane & 15u;
    const uint32_t tiles = (a.group + a.tile - 1u) / a.tile, kvh = hx / tiles, tile = hx % tiles, hd = a.p.hd;
    const uint32_t head0 = kvh * a.group + tile * a.tile, heads = min(a.tile, a.group - tile * a.tile);
    const float *q0 = a.q + (uint64_t)row * a.q_stride + (uint64_t)head0 * hd;
    if (tid == 0) sh.odd = 0u;

    uint32_t u = u0 + wave;
    int32_t page = u < u1 ? page_at(a.p, seq, u) : 0;
    bool lost = page < 0;
    Half<NB, Q8> k, v;
    k.clear(), v.clear();  // (so that nothing of them lives from one piece to the next)
    uint32_t *ks = sh.scales[wave][0], *vs = sh.scales[wave][1];
    if (u < u1 && !lost) {
        const uint64_t at = unit_offset(a.p, page, u, kvh);
        k.load(a.p.k + at, lane);
        v.load(a.p.v + at, lane);
    }

    // q's parts: column c the head c & 7, its elements 32 b + 8 g ..
    const float low = c < 8u ? 0.f : -1.f;
    ph8 qf[CT][NB];
    float unscale[CT];
#pragma unroll
    for (uint32_t ct = 0; ct < CT; ct++) {
        const uint32_t h = ct * 8u + (c & 7u);
        float x[NB][8], top = 0.f;
        if (a.q_vec) {
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) {
                const uint32_t d = b * 32u + g * 8u;
                pf4 y0 = {0.f, 0.f, 0.f, 0.f}, y1 = y0;
                if (h < heads && d < hd) {
                    const pf4 *from = reinterpret_cast<const pf4 *>(q0 + h * hd + d);
                    y0 = from[0], y1 = from[1];
                }
#pragma unroll
                for (int e = 0; e < 4; e++) x[b][e] = y0[e], x[b][4 + e] = y1[e];
            }
        } else {
#pragma unroll
            for (uint32_t b = 0; b < NB; b++)
#pragma unroll
                for (uint32_t e = 0; e < 8; e++) {
                    const uint32_t d = b * 32u + g * 8u + e;
                    x[b][e] = h < heads && d < hd ? q0[h * hd + d] : 0.f;
                }
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; b++)
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[b][e]));
        top = over_groups_max(top);
        const int up = 13 + 127 - (int)max(vbs_float_to_bits(top) >> 23, 1u);  // (an infinity stays one)
#pragma unroll
        for (uint32_t b = 0; b < NB; b++) {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) x[b][e] = __builtin_ldexpf(x[b][e], up);
            qf[ct][b] = parts(x[b], low);
        }
        unscale[ct] = __builtin_ldexpf(a.scale * kPagedLog2e, -up);
    }

    pf4 o[CT][2 * NB];
    float m[CT], l[CT];
#pragma unroll
    for (uint32_t t = 0; t < CT; t++) {
#pragma unroll
        for (uint32_t i = 0; i < 2 * NB; i++) o[t][i] = pf4{0.f, 0.f, 0.f, 0.f};
        m[t] = -INFINITY, l[t] = 0.f;
    }
    int top_e = -60;  // Q8_0: V's scales are below 2^top_e
    while (u < u1 && !lost) {
        const uint32_t next = u + kWaves;
        page = next < u1 ? page_at(a.p, seq, next) : 0;
        // scores: lane (g, c) holds slots 8 g + e of column c
        float s[CT][8];
        if constexpr (Q8) {
#pragma unroll
            for (uint32_t t = 0; t < CT; t++)
#pragma unroll
                for (int e = 0; e < 8; e++) s[t][e] = 0.f;
            k.spread(ks, lane);
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) {
                const ph8 d = *reinterpret_cast<const ph8 *>(ks + b * 16u + g * 4u);
                const ph8 k0 = int8_to_f16(k.x[b][0], k.x[b][1]), k1 = int8_to_f16(k.x[b][2], k.x[b][3]);
                const pf4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (uint32_t t = 0; t < CT; t++) {
                    const pf4 s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[t][b], zero, 0, 0, 0);
                    const pf4 s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[t][b], zero, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        s[t][i] = fmaf(s0[i], (float)d[i], s[t][i]);
                        s[t][4 + i] = fmaf(s1[i], (float)d[4 + i], s[t][4 + i]);
                    }
                }
            }
        } else {
#pragma unroll
            for (uint32_t t = 0; t < CT; t++) {
                pf4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
#pragma unroll
                for (uint32_t b = 0; b < NB; b++) {
                    s0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, k.x[b]), qf[t][b], s0, 0, 0, 0);
                    s1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, k.x[NB + b]), qf[t][b], s1, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) s[t][i] = s0[i], s[t][4 + i] = s1[i];
            }
        }
        // the next unit's K is on its way during the softmax and the second product, its V during the next scores
        lost = page < 0;
        const uint64_t at = lost ? 0u : unit_offset(a.p, page, next, kvh);
        const bool more = next < u1 && !lost;
        if (more) k.load(a.p.k + at, lane);
        const uint32_t mine = u * kUnit + g * 8u;  // the lane's first slot
        const bool tail = (u + 1u) * kUnit > len;
#pragma unroll
        for (uint32_t t = 0; t < CT; t++)
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) s[t][e] = (s[t][e] + row_ror8(s[t][e])) * unscale[t];
        if (tail) {  // what lies behind the last slot may be anything
#pragma unroll
            for (uint32_t t = 0; t < CT; t++)
#pragma unroll
                for (uint32_t e = 0; e < 8; e++)
                    if (mine + e >= len) s[t][e] = -INFINITY;
            auto kept = [&](uint32_t j) { return (j < len ? 0xFFFFu : 0u) | (j + 1u < len ? 0xFFFF0000u : 0u); };
            if constexpr (Q8) {
#pragma unroll
                for (uint32_t &d : v.ds) d &= kept(u * kUnit + 2u * (lane & 15u));
            } else {
#pragma unroll
                for (uint32_t w = 0; w < 4; w++) {
                    const uint32_t keep = kept(mine + 2u * w);
#pragma unroll
                    for (pu4 &x : v.x) x[w] &= keep;
                }
            }
        }
        // weights, in place of the scores
        float keep[CT];
#pragma unroll
        for (uint32_t t = 0; t < CT; t++) {
            float top = m[t], sum = 0.f;
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) top = fmaxf(top, s[t][e]);
            top = over_groups_max(top);
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                s[t][e] = __builtin_amdgcn_exp2f(s[t][e] - ref);
                sum += s[t][e];
            }
            keep[t] = __builtin_amdgcn_exp2f(m[t] - ref);
            l[t] = fmaf(l[t], keep[t], sum);
            m[t] = top;
        }
        if constexpr (Q8) {
            uint32_t e5 = 0u;
#pragma unroll
            for (uint32_t d : v.ds) e5 = max(e5, max(d & 0x7FFFu, (d >> 16) & 0x7FFFu));
            e5 = wave_butterfly(e5, [](uint32_t x, uint32_t y) { return max(x, y); });
            const int e = __builtin_amdgcn_readfirstlane((int)min(e5 >> 10, 30u)) - 14;
            if (e > top_e) {
#pragma unroll
                for (uint32_t t = 0; t < CT; t++) keep[t] = __builtin_ldexpf(keep[t], top_e - e);
                top_e = e;
            }
        }
        // 2^14 high (Q8_0: less what V's scales may add)
        const float raise = __builtin_ldexpf(1.f, kWeightBits - (Q8 ? top_e : 0));
#pragma unroll
        for (uint32_t t = 0; t < CT; t++) {
            if (__any(keep[t] != 1.f)) {
#pragma unroll
                for (uint32_t i = 0; i < 2 * NB; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) o[t][i][r] *= keep[t];
            }
#pragma unroll
            for (int e = 0; e < 8; e++) s[t][e] *= raise;
        }
        if constexpr (Q8) {
            v.spread(vs, lane);
#pragma unroll
            for (uint32_t b = 0; b < NB; b++) {
                const ph8 d = *reinterpret_cast<const ph8 *>(vs + b * 16u + g * 4u);
                const ph8 v0 = int8_to_f16(v.x[b][0], v.x[b][1]), v1 = int8_to_f16(v.x[b][2], v.x[b][3]);
#pragma unroll
                for (uint32_t t = 0; t < CT; t++) {
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = fmaf(s[t][e], (float)d[e], 0.f);
                    const ph8 w = parts(x, low);
                    o[t][2 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, w, o[t][2 * b], 0, 0, 0);
                    o[t][2 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, w, o[t][2 * b + 1], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (uint32_t t = 0; t < CT; t++) {
                const ph8 w = parts(s[t], low);
#pragma unroll
                for (uint32_t i = 0; i < 2 * NB; i++)
                    o[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(ph8, v.x[i]), w, o[t][i], 0, 0, 0);
            }
        }
        if (more) v.load(a.p.v + at, lane);
        u = next;
    }
    const float down = __builtin_ldexpf(1.f, (Q8 ? top_e : 0) - kWeightBits);
    bool fine = true;
#pragma unroll
    for (uint32_t t = 0; t < CT; t++) {
        const float sum = over_groups_sum(l[t]);
        bool good = fabsf(sum) < INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < 2 * NB; i++) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                o[t][i][r] = (o[t][i][r] + row_ror8(o[t][i][r])) * down;
                good = good && fabsf(o[t][i][r]) < INFINITY;
            }
            if (c < 8u) *reinterpret_cast<pf4 *>(&sh.o[wave][t * 8u + c][i * 16u + g * 4u]) = o[t][i];
        }
        if (g == 0u && c < 8u) sh.m[wave][t * 8u + c] = m[t], sh.l[wave][t * 8u + c] = sum;
        fine = fine && (good || t * 8u + (c & 7u) >= heads);
    }
    __syncthreads();  // (odd is 0)
    if ((lost || __any(!fine)) && lane == 0u) sh.odd = 1u;
    __syncthreads();
    if (__builtin_amdgcn_readfirstlane(sh.odd)) return false;
    float *out = a.out + (uint64_t)row * a.out_stride + (uint64_t)head0 * hd;
    for (uint32_t i = tid; i < heads * NB * 32u; i += 256u) {
        const uint32_t h = i / (NB * 32u), d = i % (NB * 32u);
        const float mm = fmaxf(fmaxf(sh.m[0][h], sh.m[1][h]), fmaxf(sh.m[2][h], sh.m[3][h])), ref = mm == -INFINITY ? 0.f : mm;
        float ll = 0.f, oo = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; w++) {
            const float k = __builtin_amdgcn_exp2f(sh.m[w][h] - ref);
            ll = fmaf(k, sh.l[w][h], ll);
            oo = fmaf(k, sh.o[w][h][d], oo);
        }
        if (!part) {
            if (d < hd) out[h * hd + d] = ll == 0.f ? 0.f : oo / ll;
        } else {
            if (d < hd) part[h * hd + d] = oo;
            if (d == 0u) ml[h] = make_float2(mm, ll);
        }
    }
    return true;
}

// The same in plain f32.
template <uint32_t NB, bool Q8, uint32_t CT>
__device__ __forceinline__ void slow_units(const PagedAttnArgs &a, Shared<NB, CT> &sh, uint32_t row, uint32_t hx, int32_t seq, uint32_t len,
                                           uint32_t u0, uint32_t u1, float *part, float2 *ml) {
    const uint32_t tiles = (a.group + a.tile - 1u) / a.tile, kvh = hx / tiles, tile = hx % tiles, hd = a.p.hd, tid = threadIdx.x;
    const uint32_t head0 = kvh * a.group + tile * a.tile, heads = min(a.tile, a.group - tile * a.tile);
    const float *q0 = a.q + (uint64_t)row * a.q_stride + (uint64_t)head0 * hd;
    float *out = a.out + (uint64_t)row * a.out_stride + (uint64_t)head0 * hd;
    for (uint32_t h = 0; h < heads; h++) {
        float mm, ll, oo;
        __syncthreads();
        slow_tile<Q8>(a, seq, u0, u1, len, kvh, q0 + h * hd, &sh.o[0][0][0], mm, ll, oo);
        if (!part) {
            if (tid < hd) out[h * hd + tid] = ll == 0.f ? 0.f : oo / ll;
        } else {
            if (tid < hd) part[h * hd + tid] = oo;
            if (tid == 0u) ml[h] = make_float2(mm, ll);
        }
    }
}

// Rows of few units: a workgroup for each row and head, nothing to join. grid (kv heads x tiles of its q heads, rows)
template <uint32_t NB, bool Q8, uint32_t CT>
__global__ __launch_bounds__(256, per_cu(NB)) void k_attn_paged_whole(PagedAttnArgs a) {
    __shared__ Shared<NB, CT> sh;
    const uint32_t row = blockIdx.y, hd = a.p.hd;
    const Row r = row_at(a, row);
    if (r.units) {
        if (!attend_units<NB, Q8, CT>(a, sh, row, blockIdx.x, r.seq, r.len, 0u, r.units, nullptr, nullptr))
            slow_units<NB, Q8, CT>(a, sh, row, blockIdx.x, r.seq, r.len, 0u, r.units, nullptr, nullptr);
        return;
    }
    const uint32_t tiles = (a.group + a.tile - 1u) / a.tile, kvh = blockIdx.x / tiles, tile = blockIdx.x % tiles;
    const uint32_t n = min(a.tile, a.group - tile * a.tile) * hd;
    float *out = a.out + (uint64_t)row * a.out_stride + (uint64_t)(kvh * a.group + tile * a.tile) * hd;
    for (uint32_t i = threadIdx.x; i < n; i += 256u) out[i] = r.bad ? NAN : 0.f;
}

// All rows' units in equal shares, one a workgroup. What lies whole in a share is done with it; the piece of a row and head
// that goes on in the next share is the workgroup's second partial result, one that began in an earlier share its first. Of
// the first kind there is one at most, which `joins` names, with the number of its pieces, for the merge.
template <uint32_t NB, bool Q8, uint32_t CT>
__global__ __launch_bounds__(256, per_cu(NB)) void k_attn_paged(PagedAttnArgs a) {
    __shared__ Shared<NB, CT> sh;
    __shared__ uint64_t sums[kWaves];
    const uint32_t line = a.p.nkh * ((a.group + a.tile - 1u) / a.tile);  // heads (tiles) of a row
    Shares sh_;
    uint64_t at, end;
    Found f;
    uint32_t open_row = 0u, open_hx = 0u, pieces = 0u;
    if (find_row(a, line, blockIdx.x, sh_, at, end, f, sums)) {
        const uint32_t row0 = f.row;
        const Row first = row_at(a, row0);
        const uint64_t in = at - f.before * line, long0 = padded(sh_, first.units);
        const uint32_t hx0 = (uint32_t)(in / long0), u00 = (uint32_t)(in % long0);
        // the share's pieces one after the other; in the second round, if there is one, those that were not finite (the
        // 64th and all behind it together)
        uint64_t odd = 0;
        for (uint32_t round = 0; round < 2u; round++) {
            Row r = first;
            uint32_t row = row0, hx = hx0, u0 = u00, n = 0;
            uint64_t left = end - at;
            while (true) {
                const uint32_t u1 = r.units - u0 < left ? r.units : u0 + (uint32_t)left;
                const bool begun = u0 != 0u, whole = !begun && u1 == r.units;
                const uint64_t slot = ((uint64_t)blockIdx.x * 2u + (begun ? 0u : 1u)) * a.tile;
                float *part = whole ? nullptr : a.part + slot * a.p.hd;
                const uint64_t bit = 1ull << min(n, 63u);
                if (!begun && !whole)
                    open_row = row, open_hx = hx, pieces = 1u + (uint32_t)((r.units - u1 + sh_.share - 1u) / sh_.share);
                if (round == 0u) {
                    if (!attend_units<NB, Q8, CT>(a, sh, row, hx, r.seq, r.len, u0, u1, part, a.ml + slot)) odd |= bit;
                } else if (odd & bit) {
                    slow_units<NB, Q8, CT>(a, sh, row, hx, r.seq, r.len, u0, u1, part, a.ml + slot);
                }
                left -= u1 - u0;
                if (left == 0u || sh_.grain != 1u) break;
                n++;
                u0 = 0u;
                if (++hx == line) {
                    hx = 0u;
                    do r = row_at(a, ++row);
                    while (r.units == 0u);
                }
                __syncthreads();
            }
            if (!odd) break;
        }
    }
    const uint32_t tid = threadIdx.x;
    if (tid == 0u) a.joins[blockIdx.x] = make_uint4(open_row, open_hx, pieces, 0u);
    // rows without units: row w + gridDim t is thread t's of workgroup w to look at
    if (blockIdx.x >= a.rows) return;
    __syncthreads();
    uint32_t *empty = reinterpret_cast<uint32_t *>(&sh.o[0][0][0]), &count = sh.odd;
    if (tid == 0u) count = 0u;
    __syncthreads();
    const uint64_t mine = blockIdx.x + (uint64_t)gridDim.x * tid;
    if (mine < a.rows) {
        const Row r = row_at(a, (uint32_t)mine);
        if (r.units == 0u) empty[atomicAdd(&count, 1u)] = (uint32_t)mine * 2u + r.bad;
    }
    __syncthreads();
    for (uint32_t k = 0; k < count; k++) {
        float *out = a.out + (uint64_t)(empty[k] >> 1) * a.out_stride;
        for (uint32_t i = tid; i < a.nqh * a.p.hd; i += 256u) out[i] = empty[k] & 1u ? NAN : 0.f;
    }
}

// The pieces of a row and head that lie in several shares, joined: grid (the workgroups they begin in, q heads of a tile).
// Threads of 256 / W groups (W: hd in whole waves) take every so many pieces of an element each; their first values are
// on their way while the weights are formed.
constexpr uint32_t kAhead = 8;

__global__ __launch_bounds__(256) void k_attn_paged_merge(PagedAttnArgs a) {
    __shared__ float w[256], so[256], sx[8];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6, hd = a.p.hd, w0 = blockIdx.x, in = blockIdx.y;
    const uint4 join = a.joins[w0];
    const uint32_t n = join.z, tiles = (a.group + a.tile - 1u) / a.tile, kvh = join.y / tiles, h = join.y % tiles * a.tile + in;
    if (n == 0u || h >= a.group) return;
    float *out = a.out + (uint64_t)join.x * a.out_stride + (uint64_t)(kvh * a.group + h) * hd;
    // piece k: workgroup w0 + k's first partial result, for k = 0 its second
    auto piece = [&](uint32_t k) { return ((uint64_t)(w0 + k) * 2u + (k ? 0u : 1u)) * a.tile + in; };
    const uint32_t width = (hd + 63u) & ~63u, groups = 256u / width, d = tid % width, grp = tid / width;
    const bool mine = d < hd && grp < groups;
    float x[kAhead];
    auto eight = [&](uint32_t from, uint32_t to) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; i++) {
            const uint32_t k = from + i * groups;
            x[i] = mine && k < to ? a.part[piece(k) * hd + d] : 0.f;
        }
    };
    eight(grp, min(n, 256u));
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (uint32_t k0 = 0; k0 < n; k0 += 256u) {  // (once, but for more than 256 pieces)
        const float2 ml = k0 + tid < n ? a.ml[piece(k0 + tid)] : make_float2(-INFINITY, 0.f);
        float top = wave_max(ml.x);
        __syncthreads();
        if (lane == 0u) sx[wave] = top;
        __syncthreads();
        top = fmaxf(fmaxf(fmaxf(sx[0], sx[1]), fmaxf(sx[2], sx[3])), m);
        const float ref = top == -INFINITY ? 0.f : top, keep = __builtin_amdgcn_exp2f(m - ref), f = __builtin_amdgcn_exp2f(ml.x - ref);
        w[tid] = f;
        const float sum = wave_sum(k0 + tid < n ? f * ml.y : 0.f);
        if (lane == 0u) sx[4u + wave] = sum;
        __syncthreads();
        l = fmaf(l, keep, (sx[4] + sx[5]) + (sx[6] + sx[7]));
        o *= keep;
        m = top;
        const uint32_t k1 = min(n, k0 + 256u);
        for (uint32_t k = k0 + grp; k < k1; k += kAhead * groups) {
            if (k != grp) eight(k, k1);
#pragma unroll
            for (uint32_t i = 0; i < kAhead; i++)
                if (k + i * groups < k1) o = fmaf(w[k - k0 + i * groups], x[i], o);
        }
    }
    so[tid] = o;
    __syncthreads();
    if (tid >= hd) return;
    for (uint32_t k = 1; k < groups; k++) o += so[tid + k * width];
    out[tid] = l == 0.f ? 0.f : o / l;
}

// Heads of up to so many blocks have 9 to 16 q heads of a kv head in one pass over its slots (two tiles of columns); larger
// ones in two passes (two tiles of them were not tried): 64 sequences of 4096 slots, 96/8 heads of 128, 202 us for 373 in two passes
// (F16), 143 for 217 (Q8_0).
constexpr uint32_t kTwoTiles = 4;
// Rows of at most so many units are not split: one of 512 slots takes 9.7 us (8 heads of 128, Q8_0), in shares 11.2.
constexpr uint32_t kWholeUnits = 16;

size_t plan_attn_paged(PagedAttnArgs &a) {
    a.tile = a.group > 8u && a.p.nb <= kTwoTiles ? 16u : 8u;
    const uint32_t units = (a.max_len + kUnit - 1u) / kUnit, tiles = (a.group + a.tile - 1u) / a.tile;
    a.workgroups = 0;
    const uint32_t most = 256u * per_cu(a.p.nb);
    if (units <= kWholeUnits) return 0;
    const uint64_t heads = (uint64_t)a.rows * a.p.nkh * tiles, each = (units * heads + kWaves - 1u) / kWaves;
    a.workgroups = each < most ? (uint32_t)each : most;
    a.aligned = heads <= most;
    a.grid = a.workgroups + (a.aligned ? (uint32_t)heads : 0u);  // (each head's last share may be short)
    return (uint64_t)a.grid * (sizeof(uint4) + 2u * a.tile * (sizeof(float2) + 4ull * a.p.hd));
}

template <uint32_t NB, bool Q8, uint32_t CT>
static void launch_one(const PagedAttnArgs &a, hipStream_t s) {
    const uint32_t tiles = (a.group + a.tile - 1u) / a.tile;
    if (a.workgroups) k_attn_paged<NB, Q8, CT><<<a.grid, 256, 0, s>>>(a);
    else k_attn_paged_whole<NB, Q8, CT><<<dim3(a.p.nkh * tiles, a.rows), 256, 0, s>>>(a);
}
template <uint32_t NB, bool Q8>
static void launch_tile(const PagedAttnArgs &a, hipStream_t s) {
    if constexpr (NB <= kTwoTiles) {
        if (a.tile == 16u) return launch_one<NB, Q8, 2>(a, s);
    }
    launch_one<NB, Q8, 1>(a, s);
}
template <bool Q8>
static void launch_nb(const PagedAttnArgs &a, hipStream_t s) {
    switch (a.p.nb) {
        case 1: launch_tile<1, Q8>(a, s); break;
        case 2: launch_tile<2, Q8>(a, s); break;
        case 3: launch_tile<3, Q8>(a, s); break;
        case 4: launch_tile<4, Q8>(a, s); break;
        case 5: launch_tile<5, Q8>(a, s); break;
        case 6: launch_tile<6, Q8>(a, s); break;
        case 7: launch_tile<7, Q8>(a, s); break;
        default: launch_tile<8, Q8>(a, s); break;
    }
}

hipError_t launch_attn_paged(PagedAttnArgs a, void *scratch, hipStream_t s) {
    a.q_vec = !(((uintptr_t)a.q & 15u) | (a.q_stride & 3u) | (a.p.hd & 7u));
    a.joins = static_cast<uint4 *>(scratch);
    a.ml = reinterpret_cast<float2 *>(a.joins + a.grid);
    a.part = reinterpret_cast<float *>(a.ml + (uint64_t)a.grid * 2u * a.tile);
    if (a.p.q8) launch_nb<true>(a, s);
    else launch_nb<false>(a, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.workgroups == 0u) return e;
    k_attn_paged_merge<<<dim3(a.grid, a.group < a.tile ? a.group : a.tile), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace vbs
