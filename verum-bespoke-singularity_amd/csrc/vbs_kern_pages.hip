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
// Bound: HBM (each row read and written once); one launch for few tokens.
#include <math.h>

#include "vbs_dev_common.h"
#include "vbs_pages.h"

namespace vbs {

namespace {

constexpr uint32_t kTile = 32;  // tokens of a workgroup

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
// The integer nearest x / d, ties to even, within 127: rint of an approximate quotient is
// at most one off, and x - q d is exact (d has 11 bits, q 8, and |x - q d| < |x| unless q = 0).
__device__ __forceinline__ int q8_round(float x, float d, float rd) {
    float q = rintf(x * rd);
    q = fminf(fmaxf(q, -300.f), 300.f);  // (a subnormal d may be up to a third below max |x| / 127)
    const float rest = fmaf(-q, d, x), half = 0.5f * d;
    const bool odd = (int)q & 1;
    if (fabsf(rest) > half || (fabsf(rest) == half && odd)) q += copysignf(1.f, rest);
    return (int)fminf(fmaxf(q, -127.f), 127.f);
}

__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
}

struct Place {
    int32_t at;       // the token's slot, -1: none
    uint64_t offset;  // of its unit
};

// The places of the workgroup's tokens.
__device__ __forceinline__ void tile_places(const PageRowsArgs &a, uint32_t t0, uint32_t count, uint32_t h, Place *pl) {
    if (threadIdx.x < count) {
        const uint32_t i = t0 + threadIdx.x;
        const int32_t seq = a.seq ? a.seq[i] : (int32_t)i, at = a.at[i];
        const int32_t page = at < 0 ? -1 : page_at(a.p, seq, (uint32_t)at / kUnit);
        Place &p = pl[threadIdx.x];
        p.at = page < 0 ? -1 : at;
        p.offset = page < 0 ? 0u : unit_offset(a.p, page, (uint32_t)at / kUnit, h);
    }
    __syncthreads();
}

}  // namespace

// grid (tiles of 32 tokens, kv heads, K or V); four neighbouring lanes hold a token's block of 32, eight elements each.
template <bool Q8>
__global__ __launch_bounds__(256) void k_page_store(PageRowsArgs a) {
    __shared__ Place pl[kTile];
    const uint32_t t0 = blockIdx.x * kTile, h = blockIdx.y, tid = threadIdx.x, count = min(kTile, a.n - t0);
    const bool is_v = blockIdx.z;
    tile_places(a, t0, count, h, pl);
    const float *src = is_v ? a.v : a.k;
    uint8_t *pool = is_v ? a.p.v : a.p.k;
    const uint32_t hd = a.p.hd, nb = a.p.nb;
    for (uint32_t e = tid; e < kTile * nb * 4u; e += 256u) {  // (every lane of a wave, or none: 128 nb lanes)
        const uint32_t t = (e >> 2) & (kTile - 1u), b = e >> 7, d0 = b * 32u + (e & 3u) * 8u;
        const bool there = t < count && pl[t].at >= 0;
        float x[8];
        uint32_t top = 0u;
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) {
            x[j] = there && d0 + j < hd ? src[(uint64_t)(t0 + t) * a.stride + (uint64_t)h * hd + d0 + j] : 0.f;
            top = max(top, vbs_float_to_bits(x[j]) & 0x7FFFFFFFu);
        }
        uint16_t dh = 0;
        uint16_t w[8];
        if constexpr (Q8) {
            dh = q8_scale(vbs_half_bits_to_float(quad_max(top)));
            const float d = (float)__builtin_bit_cast(_Float16, dh);
            const bool zero = !(d > 0.f);
            const float rd = zero ? 0.f : 1.f / d;
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) w[j] = (uint8_t)(zero ? 0 : q8_round(x[j], d, rd));
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) w[j] = vbs_f2h(x[j]);
        }
        if (!there) continue;
        const uint32_t slot = (uint32_t)pl[t].at & (kUnit - 1u);
        uint8_t *unit = pool + pl[t].offset;
        if constexpr (Q8) {
            if ((e & 3u) == 0u) *reinterpret_cast<uint16_t *>(unit + nb * 1024u + (b * 32u + slot) * 2u) = dh;
        }
        if (!is_v) {
            if constexpr (Q8) {
                uint64_t o = 0;
#pragma unroll
                for (uint32_t j = 0; j < 8; j++) o |= (uint64_t)w[j] << (8u * j);
                *reinterpret_cast<uint64_t *>(unit + k_place<true>(nb, slot, d0)) = o;
            } else {
                uint4 o;
                o.x = w[0] | (uint32_t)w[1] << 16, o.y = w[2] | (uint32_t)w[3] << 16;
                o.z = w[4] | (uint32_t)w[5] << 16, o.w = w[6] | (uint32_t)w[7] << 16;
                *reinterpret_cast<uint4 *>(unit + 2u * k_place<false>(nb, slot, d0)) = o;
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8; j++) {
                if constexpr (Q8) unit[v_place<true>(slot, d0 + j)] = (uint8_t)w[j];
                else reinterpret_cast<uint16_t *>(unit)[v_place<false>(slot, d0 + j)] = w[j];
            }
        }
    }
}

template <bool Q8, bool H>
__global__ __launch_bounds__(256) void k_page_load(PageRowsArgs a) {
    __shared__ Place pl[kTile];
    const uint32_t t0 = blockIdx.x * kTile, h = blockIdx.y, tid = threadIdx.x, count = min(kTile, a.n - t0);
    const bool is_v = blockIdx.z;
    tile_places(a, t0, count, h, pl);
    const uint8_t *pool = is_v ? a.p.v : a.p.k;
    void *out = is_v ? a.out_v : a.out_k;
    const uint32_t hd = a.p.hd, nb = a.p.nb;
    for (uint32_t e = tid; e < kTile * nb * 4u; e += 256u) {
        const uint32_t t = (e >> 2) & (kTile - 1u), b = e >> 7, d0 = b * 32u + (e & 3u) * 8u;
        if (t >= count || a.at[t0 + t] < 0) continue;
        const bool there = pl[t].at >= 0;
        const uint32_t slot = (uint32_t)pl[t].at & (kUnit - 1u);
        const uint8_t *unit = pool + pl[t].offset;
#pragma unroll
        for (uint32_t j = 0; j < 8; j++) {
            if (d0 + j >= hd) break;
            const uint32_t at = is_v ? v_place<Q8>(slot, d0 + j) : k_place<Q8>(nb, slot, d0 + j);
            const uint64_t to = (uint64_t)(t0 + t) * a.stride + (uint64_t)h * hd + d0 + j;
            if constexpr (Q8) {
                const float f = there ? (float)(int8_t)unit[at] *
                                            (float)*reinterpret_cast<const _Float16 *>(unit + nb * 1024u + (b * 32u + slot) * 2u)
                                      : NAN;
                if constexpr (H) static_cast<uint16_t *>(out)[to] = vbs_f2h(f);
                else static_cast<float *>(out)[to] = f;
            } else {
                const uint16_t w = there ? reinterpret_cast<const uint16_t *>(unit)[at] : (uint16_t)0x7E00u;
                if constexpr (H) static_cast<uint16_t *>(out)[to] = w;
                else static_cast<float *>(out)[to] = vbs_h2f(w);
            }
        }
    }
}

hipError_t launch_page_store(const PageRowsArgs &a, hipStream_t s) {
    const dim3 grid((a.n + kTile - 1u) / kTile, a.p.nkh, 2);
    if (a.p.q8) k_page_store<true><<<grid, 256, 0, s>>>(a);
    else k_page_store<false><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_page_load(const PageRowsArgs &a, hipStream_t s) {
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
