// vbs_kern_pages.hip — rows of k and v into pages (as f16, or quantised to 8 bits
// as they are written) and out of them.
//
// Q8_0 (src/vbs_dequant.c:134-147): per token, kv head and 32 elements a scale d and
// 32 int8, value q d. Here d = f16(max |x| / 127) and q = the integer nearest x / d,
// both rounded once from the exact quotient, ties to even: a quotient that is rounded
// to f32 on the way would end on the other side of some borders. A block that holds a
// NaN or an infinity, or whose d would pass f16's range, gets d = NaN; d = 0 (all
// below 127 * 2^-25) holds zeros.
//
// K lies in a page so that eight elements of a slot are neighbours, V so that eight slots of
// an element are: tokens in consecutive slots (a prompt) have V turned in LDS, to be
// stored and loaded 16 bytes at a time like K; others (a decode step) go element by element.
// Bound: HBM (each row read and written once) for prompts; for few tokens one launch and three
// round trips (the token's place, the table, the row).
#include <math.h>

#include <type_traits>

#include "vbs_dev_common.h"
#include "vbs_pages.h"

namespace vbs {

namespace {

typedef float gf4 __attribute__((ext_vector_type(4)));
typedef uint32_t gu4 __attribute__((ext_vector_type(4)));
typedef uint32_t gu2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kTile = 32;      // tokens of a workgroup
constexpr uint32_t kOctets = 5;     // runs of eight slots that they can lie in
constexpr uint32_t kMaxWide = 256;  // elements of a head, padded

// f16(top / 127), as bits: the f32 quotient rounded to odd (its last bit set unless
// it is exact, after a step towards the true value where it lies beyond), whose 13
// extra bits then round to f16 as the true quotient would.
__device__ __forceinline__ uint16_t q8_scale(float top) {
    if (!(top < INFINITY)) return 0x7E00u;
    float d = __fdiv_rn(top, 127.f);
    const float rest = fmaf(-d, 127.f, top);
    uint32_t u = vbs_float_to_bits(d);
    if (rest < 0.f) u--;
    if (rest != 0.f) u |= 1u;
    const uint16_t h = __builtin_bit_cast(uint16_t, (_Float16)vbs_half_bits_to_float(u));
    return h >= 0x7C00u ? (uint16_t)0x7E00u : h;
}
// The integers nearest x / d, ties to even, within 127, as the low bytes of w. x rd is within 2^-23 of the quotient, so within
// 1.6e-5, and rounds (by the addition of 2^23 + 2^22) as that does unless it lies closer to a border; there, and
// where d is subnormal (up to a third below max |x| / 127, so quotients pass 127), the whole wave looks again: x - q d is
// exact (d has 11 bits, q 8, and |x - q d| < |x| unless q = 0), q at most one off.
__device__ __forceinline__ void q8_round(const float x[8], float d, float rd, uint32_t w[8]) {
    constexpr float kMagic = 12582912.f;
    float far = 0.f, q[8];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float t = x[j] * rd, r = t + kMagic;
        w[j] = vbs_float_to_bits(r);
        q[j] = r - kMagic;
        far = fmaxf(far, fabsf(t - q[j]));
    }
    if (!__any(far > 0.49995f || (d > 0.f && d < 0x1p-14f))) return;
    const float half = 0.5f * d;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float c = fminf(fmaxf(q[j], -300.f), 300.f);
        const float rest = fmaf(-c, d, x[j]);
        const bool odd = (int)c & 1;
        if (fabsf(rest) > half || (fabsf(rest) == half && odd)) c += copysignf(1.f, rest);
        w[j] = (uint32_t)(int)fminf(fmaxf(c, -127.f), 127.f);
    }
}

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
}

// vbs_f2h by the hardware's conversion where the two agree: zeros, and from the least normal f16 on (both to nearest even).
__device__ __forceinline__ uint16_t cache_half(float f) {
    const uint32_t m = vbs_float_to_bits(f) & 0x7FFFFFFFu;
    if (m == 0u || m - 0x38800000u <= 0x7F800000u - 0x38800000u) return __builtin_bit_cast(uint16_t, (_Float16)f);
    return vbs_f2h(f);
}

struct Place {
    int32_t at;       // the token's slot, -1: none
    uint64_t offset;  // of its unit
};

// The places of the workgroup's tokens; whether all have one and they are consecutive slots of one sequence.
__device__ __forceinline__ bool tile_places(const PageRowsArgs &a, uint32_t t0, uint32_t count, uint32_t h, Place *pl) {
    bool run = count > 1u;
    if (threadIdx.x < count) {
        const uint32_t i = t0 + threadIdx.x;
        const int32_t seq = a.seq ? a.seq[i] : (int32_t)i, at = a.at[i];
        const int32_t page = at < 0 ? -1 : page_at(a.p, seq, (uint32_t)at / kUnit);
        Place &p = pl[threadIdx.x];
        p.at = page < 0 ? -1 : at;
        p.offset = page < 0 ? 0u : unit_offset(a.p, page, (uint32_t)at / kUnit, h);
        const int32_t seq0 = a.seq ? a.seq[t0] : (int32_t)t0, at0 = a.at[t0];
        run = run && page >= 0 && seq == seq0 && (int64_t)at - at0 == (int64_t)threadIdx.x;
    }
    return __syncthreads_and(run);
}

// V of a tile turned: the element d of the token in octet place p (its slot, counted from the first octet's beginning)
// at [d][p], an octet 8 (int8) or 16 (f16) bytes.
template <bool Q8>
using Turned = std::conditional_t<Q8, uint8_t, uint16_t>;
constexpr uint32_t kTurn = 8u * kOctets;

}  // namespace

// grid (tiles of 32 tokens, kv heads, K or V); four neighbouring lanes hold a token's block of 32, eight elements each.
template <bool Q8>
__global__ __launch_bounds__(256) void k_page_store(PageRowsArgs a) {
    __shared__ Place pl[kTile];
    __shared__ __align__(16) Turned<Q8> turn[kMaxWide * kTurn];
    const uint32_t t0 = blockIdx.x * kTile, h = blockIdx.y, tid = threadIdx.x, count = min(kTile, a.n - t0);
    const bool is_v = blockIdx.z;
    const float *src = is_v ? a.v : a.k;
    uint8_t *pool = is_v ? a.p.v : a.p.k;
    const uint32_t hd = a.p.hd, nb = a.p.nb, items = kTile * nb * 4u;
    // the first rows are on their way while the places are looked up
    auto row8 = [&](uint32_t e, float x[8]) {
        const uint32_t t = (e >> 2) & (kTile - 1u), d0 = (e >> 7) * 32u + (e & 3u) * 8u;
        const float *from = src + (uint64_t)(t0 + t) * a.stride + (uint64_t)h * hd + d0;
        if (a.vec) {
            gf4 x0 = {0.f, 0.f, 0.f, 0.f}, x1 = x0;
            if (t < count && d0 < hd) x0 = reinterpret_cast<const gf4 *>(from)[0], x1 = reinterpret_cast<const gf4 *>(from)[1];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) x[j] = x0[j], x[4 + j] = x1[j];
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) x[j] = t < count && d0 + j < hd ? from[j] : 0.f;
        }
    };
    float x[8], next[8];
    row8(tid, x);  // (at least 128 items: lanes behind them read the first tokens again, in vain)
    const bool run = tile_places(a, t0, count, h, pl), turned = is_v && run;
    const uint32_t first = run ? (uint32_t)pl[0].at & 7u : 0u;  // of the run, in its octet
    for (uint32_t e = tid; e < items; e += 256u) {  // (every lane of a wave, or none: 128 nb lanes)
        if (e + 256u < items) row8(e + 256u, next);
        const uint32_t t = (e >> 2) & (kTile - 1u), b = e >> 7, d0 = b * 32u + (e & 3u) * 8u;
        const bool there = t < count && pl[t].at >= 0;
        uint16_t dh = 0;
        uint32_t w[8];
        if constexpr (Q8) {
            uint32_t top = 0u;
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) top = max(top, vbs_float_to_bits(x[j]) & 0x7FFFFFFFu);
            dh = q8_scale(vbs_half_bits_to_float(quad_max(top)));
            const float d = (float)__builtin_bit_cast(_Float16, dh);
            const bool some = d > 0.f;  // (else all are stored as 0)
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) x[j] = some ? x[j] : 0.f;
            q8_round(x, some ? d : 0.f, some ? 1.f / d : 0.f, w);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) w[j] = cache_half(x[j]);
        }
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) x[j] = next[j];
        if (!there) continue;
        const uint32_t slot = (uint32_t)pl[t].at & (kUnit - 1u);
        uint8_t *unit = pool + pl[t].offset;
        if constexpr (Q8) {
            if ((e & 3u) == 0u) *reinterpret_cast<uint16_t *>(unit + nb * 1024u + (b * 32u + slot) * 2u) = dh;
        }
        if (turned) {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) turn[(d0 + j) * kTurn + first + t] = (Turned<Q8>)w[j];
        } else if (!is_v) {
            if constexpr (Q8) {
                gu2 o;
#pragma unroll
                for (uint32_t j = 0; j < 2; j++)
                    o[j] = (w[4 * j] & 0xFFu) | (w[4 * j + 1] & 0xFFu) << 8 | (w[4 * j + 2] & 0xFFu) << 16 | w[4 * j + 3] << 24;
                *reinterpret_cast<gu2 *>(unit + k_place<true>(nb, slot, d0)) = o;
            } else {
                gu4 o;
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) o[j] = w[2 * j] | w[2 * j + 1] << 16;
                *reinterpret_cast<gu4 *>(unit + 2u * k_place<false>(nb, slot, d0)) = o;
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                if constexpr (Q8) unit[v_place<true>(slot, d0 + j)] = (uint8_t)w[j];
                else reinterpret_cast<uint16_t *>(unit)[v_place<false>(slot, d0 + j)] = (uint16_t)w[j];
            }
        }
    }
    if (!turned) return;
    __syncthreads();
    // octet by octet, 16 bytes a lane where all eight slots are the run's: for int8 the elements d and d + 16 together
    const uint32_t octets = (first + count + 7u) / 8u, per = Q8 ? nb * 16u : nb * 32u;
    for (uint32_t i = tid; i < octets * per; i += 256u) {
        const uint32_t oc = i / per, k = i % per, lead = oc * 8u, t = max(lead, first) - first;
        const uint32_t lo = max(lead, first) - lead, hi = min(lead + 8u, first + count) - lead;  // the run's slots of the octet
        const uint32_t slot = ((uint32_t)pl[t].at & (kUnit - 1u)) & ~7u;
        uint8_t *unit = pool + pl[t].offset;
        if constexpr (Q8) {
            const uint32_t d = (k >> 4) * 32u + (k & 15u);
            const uint8_t *f0 = turn + d * kTurn + lead, *f1 = f0 + 16u * kTurn;
            uint8_t *to = unit + v_place<true>(slot, d);
            if (lo == 0u && hi == 8u) {
                const gu2 x0 = *reinterpret_cast<const gu2 *>(f0), x1 = *reinterpret_cast<const gu2 *>(f1);
                *reinterpret_cast<gu4 *>(to) = gu4{x0[0], x0[1], x1[0], x1[1]};
            } else {
                for (uint32_t j = lo; j < hi; j++) to[j] = f0[j], to[8u + j] = f1[j];
            }
        } else {
            const uint16_t *from = turn + k * kTurn + lead;
            uint16_t *to = reinterpret_cast<uint16_t *>(unit) + v_place<false>(slot, k);
            if (lo == 0u && hi == 8u) *reinterpret_cast<gu4 *>(to) = *reinterpret_cast<const gu4 *>(from);
            else
                for (uint32_t j = lo; j < hi; j++) to[j] = from[j];
        }
    }
}

// The same grid.
template <bool Q8, bool H>
__global__ __launch_bounds__(256) void k_page_load(PageRowsArgs a) {
    __shared__ Place pl[kTile];
    __shared__ __align__(16) Turned<Q8> turn[kMaxWide * kTurn];
    const uint32_t t0 = blockIdx.x * kTile, h = blockIdx.y, tid = threadIdx.x, count = min(kTile, a.n - t0);
    const bool is_v = blockIdx.z, run = tile_places(a, t0, count, h, pl), turned = is_v && run;
    const uint8_t *pool = is_v ? a.p.v : a.p.k;
    void *out = is_v ? a.out_v : a.out_k;
    const uint32_t hd = a.p.hd, nb = a.p.nb, first = run ? (uint32_t)pl[0].at & 7u : 0u;
    if (turned) {
        const uint32_t octets = (first + count + 7u) / 8u, per = Q8 ? nb * 16u : nb * 32u;
        for (uint32_t i = tid; i < octets * per; i += 256u) {
            const uint32_t oc = i / per, k = i % per, lead = oc * 8u, t = max(lead, first) - first;
            const uint32_t slot = ((uint32_t)pl[t].at & (kUnit - 1u)) & ~7u;
            const uint8_t *unit = pool + pl[t].offset;
            if constexpr (Q8) {
                const uint32_t d = (k >> 4) * 32u + (k & 15u);
                const gu4 x = *reinterpret_cast<const gu4 *>(unit + v_place<true>(slot, d));
                *reinterpret_cast<gu2 *>(turn + d * kTurn + lead) = gu2{x[0], x[1]};
                *reinterpret_cast<gu2 *>(turn + (d + 16u) * kTurn + lead) = gu2{x[2], x[3]};
            } else {
                *reinterpret_cast<gu4 *>(turn + k * kTurn + lead) =
                    *reinterpret_cast<const gu4 *>(unit + 2u * v_place<false>(slot, k));
            }
        }
        __syncthreads();
    }
    for (uint32_t e = tid; e < kTile * nb * 4u; e += 256u) {
        const uint32_t t = (e >> 2) & (kTile - 1u), b = e >> 7, d0 = b * 32u + (e & 3u) * 8u;
        if (t >= count || d0 >= hd || a.at[t0 + t] < 0) continue;
        const bool there = pl[t].at >= 0;
        const uint32_t slot = (uint32_t)pl[t].at & (kUnit - 1u);
        const uint8_t *unit = pool + pl[t].offset;
        uint16_t w[8];  // int8 or f16 bits
        float d = NAN;
        if (Q8 && there) d = (float)*reinterpret_cast<const _Float16 *>(unit + nb * 1024u + (b * 32u + slot) * 2u);
        if (!there) {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) w[j] = Q8 ? 0u : 0x7E00u;
        } else if (turned) {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) w[j] = turn[(d0 + j) * kTurn + first + t];
        } else if (!is_v) {
            if constexpr (Q8) {
                const gu2 x = *reinterpret_cast<const gu2 *>(unit + k_place<true>(nb, slot, d0));
#pragma unroll
                for (uint32_t j = 0; j < 8; j++) w[j] = (uint8_t)(x[j >> 2] >> (8u * (j & 3u)));
            } else {
                const gu4 x = *reinterpret_cast<const gu4 *>(unit + 2u * k_place<false>(nb, slot, d0));
#pragma unroll
                for (uint32_t j = 0; j < 8; j++) w[j] = (uint16_t)(x[j >> 1] >> (16u * (j & 1u)));
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++)
                w[j] = Q8 ? unit[v_place<Q8>(slot, d0 + j)] : reinterpret_cast<const uint16_t *>(unit)[v_place<Q8>(slot, d0 + j)];
        }
        const uint64_t to = (uint64_t)(t0 + t) * a.stride + (uint64_t)h * hd + d0;
        if constexpr (H) {
            uint16_t y[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) y[j] = Q8 ? cache_half((float)(int8_t)w[j] * d) : w[j];
            uint16_t *o = static_cast<uint16_t *>(out) + to;
            if (a.vec) {
                gu4 x;
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) x[j] = y[2 * j] | (uint32_t)y[2 * j + 1] << 16;
                *reinterpret_cast<gu4 *>(o) = x;
            } else {
                for (uint32_t j = 0; j < 8 && d0 + j < hd; j++) o[j] = y[j];
            }
        } else {
            float y[8];
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) y[j] = Q8 ? (float)(int8_t)w[j] * d : vbs_h2f(w[j]);
            float *o = static_cast<float *>(out) + to;
            if (a.vec) {
                reinterpret_cast<gf4 *>(o)[0] = gf4{y[0], y[1], y[2], y[3]};
                reinterpret_cast<gf4 *>(o)[1] = gf4{y[4], y[5], y[6], y[7]};
            } else {
                for (uint32_t j = 0; j < 8 && d0 + j < hd; j++) o[j] = y[j];
            }
        }
    }
}

// Whether eight elements of a row can be read or written 16 bytes at a time.
static int rows_vec(const void *k, const void *v, uint32_t stride, uint32_t hd, uint32_t size) {
    return !((((uintptr_t)k | (uintptr_t)v) & 15u) | ((uint64_t)stride * size & 15u) | (hd & 7u));
}

hipError_t launch_page_store(PageRowsArgs a, hipStream_t s) {
    a.vec = rows_vec(a.k, a.v, a.stride, a.p.hd, 4u);
    const dim3 grid((a.n + kTile - 1u) / kTile, a.p.nkh, 2);
    if (a.p.q8) k_page_store<true><<<grid, 256, 0, s>>>(a);
    else k_page_store<false><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_page_load(PageRowsArgs a, hipStream_t s) {
    a.vec = rows_vec(a.out_k, a.out_v, a.stride, a.p.hd, a.out_f16 ? 2u : 4u);
    const dim3 grid((a.n + kTile - 1u) / kTile, a.p.nkh, 2);
    if (a.p.q8) {
        if (a.out_f16) k_page_load<true, true><<<grid, 256, 0, s>>>(a);
        else k_page_load<true, false><<<grid, 256, 0, s>>>(a);
    } else {
        if (a.out_f16) k_page_load<false, true><<<grid, 256, 0, s>>>(a);
        else k_page_load<false, false><<<grid, 256, 0, s>>>(a);
    }
    return hipGetLastError();
}

}  // namespace vbs
