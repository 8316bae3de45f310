// vbs_kern_rows.hip — attention of several tokens over the f16 KV cache: a chunk
// of consecutive tokens (causal, with a prefix, documents, capped scores, a bias
// that depends on distance) or a tree of drafted tokens (a mask of bits), and the
// attention weight that each slot received.
//
// Row i (a token) and q head h of kv head h / group, over the slots j that the row
// sees: s_j = scale q.k_j, capped c tanh(s_j / c), less slope_h |i - j|; m = max s_j,
// l = sum e^(s_j - m), out = sum e^(s_j - m) v_j / l, and 0 where nothing is seen
// (l = 0). The weight of slot j, e^(s_j - m) / l, is summed over the rows and
// the q heads of its kv head into mass[j]. Rows that do not see a slot take
// nothing from it, whatever is in its K and V.
//
// The (token, q head) pairs of a kv head are its rows, n * group of them, row r =
// i * group + g. A workgroup takes 64 CT rows of one kv head (16 CT a wave) and a
// range of slots, 64 (32 for head_dim above 128) at a time through LDS, on
// v_mfma_f32_16x16x32_f16:
// * S^T = K Q^T: A = 16 slots x 32 dims of K (the cache's f16, exact), B = 32 dims
//   x 16 rows of q' = q 2^s, s so that the row's largest |q'| lies in [2^14, 2^15),
//   as two f16 parts hi + lo (22 bits; the two products add up in the same f32
//   sums). A lane then holds the scores of one row (column lane & 15) at slots
//   16 hf + 4 (lane >> 4) + r, so the softmax needs no row-wise exchange but for the
//   maximum.
// * the running maximum moves only where a score passes it by more than 8 in
//   log2: then the sums are rescaled. The weights are 2^(y - m + 7) <= 2^15, so that
//   small ones keep their low part in f16.
// * O^T += V^T P^T: B = P^T, the lane's own weights (hi, then lo), A = V^T with the
//   k slots in the same order, by transposed LDS reads.
// Each range of slots ends in m, l and acc per row; where a kv head's rows are few
// the slots are split over several workgroups and k_rows_merge adds them up,
// scaled to the common maximum.
#include "vbs_lds_dma.h"
#include "vbs_rows_common.h"

namespace vbs {

constexpr float kLazy = 8.f, kLift = 7.f;  // log2: how far a score may pass m; the weights' scale

// p - h[0] and p - h[1], the halves widened on the way (exact: h is p rounded).
__device__ __forceinline__ float less_low(float p, rh2 h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(p));
    return r;
}
__device__ __forceinline__ float less_high(float p, rh2 h) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(p));
    return r;
}

__device__ __forceinline__ uint64_t ones_below(int64_t x) {
    return x <= 0 ? 0ull : x >= 64 ? ~0ull : (1ull << x) - 1ull;
}

// The slots [p0, p0 + 64) that a row of token i sees, as bits, documents aside.
__device__ __forceinline__ uint64_t seen_bits(const RowsArgs &a, uint32_t i, uint32_t p0, uint32_t s1) {
    const uint64_t in = ones_below((int64_t)s1 - p0);
    if (!a.mask) return in & ones_below((int64_t)row_end(a, i) - p0);
    const int64_t off = (int64_t)p0 - a.past;
    const uint64_t *row = a.mask + (uint64_t)i * a.words;
    uint64_t v = ones_below(-off);
    if (off >= 0) {
        const uint64_t w = (uint64_t)off >> 6;
        const uint32_t sh = (uint32_t)off & 63u;
        if (w < a.words) v |= row[w] >> sh;
        if (sh && w + 1u < a.words) v |= row[w + 1u] << (64u - sh);
    } else if (off > -64) {
        v |= row[0] << (uint32_t)-off;
    }
    return in & v;
}

// The q' parts of one row (column lane & 15) for lane group g: dims 32 kk + 8 g ...
// `row` NULL: zeros. c: |scale| 2^-s, what a product of the parts is to be scaled by.
template <uint32_t KK>
__device__ __forceinline__ void row_parts(const float *row, uint32_t hd, bool wide, float scale, uint32_t g,
                                          rh8 (&hi)[KK], rh8 (&lo)[KK], float &c) {
    float x[KK][8], top = 0.f;
#pragma unroll
    for (uint32_t kk = 0; kk < KK; kk++) {
        const uint32_t d0 = 32u * kk + 8u * g;
        if (row && wide && d0 < hd) {
            const float4 u = *reinterpret_cast<const float4 *>(row + d0), v = *reinterpret_cast<const float4 *>(row + d0 + 4u);
            x[kk][0] = u.x, x[kk][1] = u.y, x[kk][2] = u.z, x[kk][3] = u.w;
            x[kk][4] = v.x, x[kk][5] = v.y, x[kk][6] = v.z, x[kk][7] = v.w;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8u; e++) x[kk][e] = row && !wide && d0 + e < hd ? row[d0 + e] : 0.f;
        }
#pragma unroll
        for (uint32_t e = 0; e < 8u; e++) top = fmaxf(top, fabsf(x[kk][e]));
    }
    top = fmaxf(top, lane_xor<16>(top));
    top = fmaxf(top, lane_xor<32>(top));
    int e2 = 0;
    (void)frexpf(top, &e2);  // top < 2^e2
    // (a row below 2^-111 scores nothing that an f32 sum keeps; 2^-sq must stay a number)
    const int sq = top > 0.f && top < INFINITY ? (15 - e2 < 126 ? 15 - e2 : 126) : 0;
    c = fmaxf(ldexpf(fabsf(scale), -sq), 0x1p-126f);  // (not 0: masked scores are -inf times it)
    const float sign = scale < 0.f ? -1.f : 1.f;
#pragma unroll
    for (uint32_t kk = 0; kk < KK; kk++)
#pragma unroll
        for (uint32_t e = 0; e < 8u; e++) {
            const float y = ldexpf(x[kk][e] * sign, sq);
            const _Float16 h = (_Float16)y;
            hi[kk][e] = h;
            lo[kk][e] = (_Float16)(y - (float)h);
        }
}

// Eight cache elements of a row from element d0 on (zeros from hd on).
__device__ __forceinline__ ru4 cache8(const uint16_t *p, uint32_t d0, uint32_t hd, bool wide) {
    if (wide) return d0 < hd ? *reinterpret_cast<const ru4 *>(p + d0) : ru4{0u, 0u, 0u, 0u};
    ru4 v;
#pragma unroll
    for (uint32_t k = 0; k < 4u; k++) {
        const uint32_t x = d0 + 2u * k < hd ? p[d0 + 2u * k] : 0u, y = d0 + 2u * k + 1u < hd ? p[d0 + 2u * k + 1u] : 0u;
        v[k] = x | y << 16;
    }
    return v;
}

struct RowsSplit {
    uint32_t len, n;  // slots per range (a multiple of 64), ranges
};

// How the launch's scratch is laid out: (m, l) then acc per (kv head, range, row),
// then (m, 1 / l) per (kv head, row).
struct RowsPart {
    float2 *ml;
    float *acc;
    float2 *stats;
};

// Floats from one partial row to the next.
__host__ __device__ __forceinline__ uint32_t part_stride(uint32_t hd) { return (hd + 3u) / 4u * 4u; }

template <uint32_t HD>
constexpr uint32_t kTile = HD > 128u ? 32u : 64u;  // slots per LDS tile

// The place of 16-byte chunk c of row r in an LDS tile of HD-element rows without
// padding (the DMA writes whole runs): so that the rows of an A operand of K (eight
// at a time) and the 32-byte runs of four rows that a transposed read of V takes lie
// in different banks. It goes by the row's last three bits alone.
template <uint32_t HD>
__device__ __forceinline__ uint32_t tile_place(uint32_t r, uint32_t c) {
    if constexpr (HD == 96u) {
        const uint32_t s = c + 2u * (r >> 2 & 1u);
        return s >= 12u ? s - 12u : s;
    }
    return c ^ 2u * (HD >= 128u ? r & 7u : HD == 64u ? r >> 1 & 3u : r >> 2 & 1u);
}
// The chunk at place s of row r.
template <uint32_t HD>
__device__ __forceinline__ uint32_t tile_chunk(uint32_t r, uint32_t s) {
    if constexpr (HD == 96u) {
        const uint32_t o = 2u * (r >> 2 & 1u);
        return s >= o ? s - o : s + 12u - o;
    }
    return tile_place<HD>(r, s);
}

// Four 16-bit elements a lane, transposed within each 16 lanes: lane i receives
// element i % 4 of what the lanes 4 e + i / 4 address, e = 0 .. 3.
typedef short rs4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ rs4 lds_transposed(const uint8_t *p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) rs4 *)(uint32_t)(uintptr_t)p);
}

// The rows of one wave: CT column tiles of 16, their q' parts and their running sums.
template <uint32_t HD, uint32_t CT>
struct RowTiles {
    static constexpr uint32_t KK = HD / 32u, DT = HD / 16u, RB = HD * 2u;
    static constexpr uint32_t NK = KK < 4u ? KK : 4u, NV = DT < 8u ? DT : 8u;  // (dims from 128 on lie 256 bytes on)
    rh8 qh[CT][KK], ql[CT][KK];
    float c1[CT], slope[CT], m[CT], l[CT];
    uint32_t tok[CT];
    int32_t doc[CT];
    bool real[CT];
    rf4 acc[DT][CT];
    uint32_t kat[NK], vat[NV];  // where the lane reads in LDS, from a tile's first byte of K
    // below `clear` every row sees every slot (documents aside); from `last` on, none
    uint32_t clear, last;

    // v_at: from a tile's first byte of K to its first of V
    __device__ __forceinline__ void init(const RowsArgs &a, uint32_t kvh, uint32_t row0, bool wide_q, uint32_t lane,
                                         uint32_t v_at) {
        const uint32_t col = lane & 15u, g = lane >> 4, group = a.nqh / a.nkh, rows = a.n * group;
#pragma unroll
        for (uint32_t x = 0; x < CT; x++) {
            const uint32_t r = row0 + 16u * x + col;
            real[x] = r < rows;
            tok[x] = real[x] ? r / group : 0u;
            const uint32_t h = kvh * group + (real[x] ? r % group : 0u);
            row_parts<KK>(real[x] ? a.q + (uint64_t)tok[x] * a.q_stride + (uint64_t)h * a.hd : nullptr, a.hd, wide_q,
                          a.scale, g, qh[x], ql[x], c1[x]);
            slope[x] = a.slopes ? a.slopes[h] : 0.f;
            doc[x] = a.docs ? a.docs[a.past + tok[x]] : 0;
            m[x] = -INFINITY, l[x] = 0.f;
#pragma unroll
            for (uint32_t d = 0; d < DT; d++) acc[d][x] = rf4{0.f, 0.f, 0.f, 0.f};
        }
        clear = a.docs ? 0u : a.mask ? a.past : row_end(a, min(row0, rows - 1u) / group);
        last = row0 < rows ? row_end(a, (min(row0 + 16u * CT, rows) - 1u) / group) : 0u;
        // its chunk of K per slice (row `col` of a 16-row tile), and per 16 dims its part of the
        // transposed V read: slot 4 g + col / 4, dims 4 (col % 4) ..
#pragma unroll
        for (uint32_t kk = 0; kk < NK; kk++) kat[kk] = col * RB + 16u * tile_place<HD>(col, 4u * kk + g);
#pragma unroll
        for (uint32_t d = 0; d < NV; d++) {
            const uint32_t r = 4u * g + (col >> 2);
            vat[d] = v_at + r * RB + 16u * tile_place<HD>(r, 2u * d + (col >> 1 & 1u)) + 8u * (col & 1u);
        }
    }

    __device__ __forceinline__ void turn(uint32_t by) {  // on to another buffer
#pragma unroll
        for (uint32_t kk = 0; kk < NK; kk++) kat[kk] += by;
#pragma unroll
        for (uint32_t d = 0; d < NV; d++) vat[d] += by;
    }

    // 32 slots from p0 on, in LDS from row `at` of the tile; full: every row sees them all, else vis
    // holds their bits per column tile and docs (or NULL) their documents
    __device__ __forceinline__ void step(const RowsArgs &a, const uint8_t *lds, uint32_t at, uint32_t p0,
                                         const uint32_t (&vis)[CT], bool full, const int32_t *docs, uint32_t lane) {
        const uint32_t g = lane >> 4;
        const bool terms = a.cap > 0.f || a.slopes;
        rf4 S[2][CT];
#pragma unroll
        for (uint32_t hf = 0; hf < 2u; hf++)
#pragma unroll
            for (uint32_t x = 0; x < CT; x++) S[hf][x] = rf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (uint32_t kk = 0; kk < KK; kk++) {
            rh8 ka[2];
#pragma unroll
            for (uint32_t hf = 0; hf < 2u; hf++)
                ka[hf] = *reinterpret_cast<const rh8 *>(lds + kat[kk & 3u] + 256u * (kk >> 2) + (at + 16u * hf) * RB);
#pragma unroll
            for (uint32_t hf = 0; hf < 2u; hf++)
#pragma unroll
                for (uint32_t x = 0; x < CT; x++)
                    S[hf][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[hf], qh[x][kk], S[hf][x], 0, 0, 0);
#pragma unroll
            for (uint32_t hf = 0; hf < 2u; hf++)
#pragma unroll
                for (uint32_t x = 0; x < CT; x++)
                    S[hf][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[hf], ql[x][kk], S[hf][x], 0, 0, 0);
        }
        // the score in units of log2 is cm S: S the plain product, or what the terms make of it
        float cm[CT];
#pragma unroll
        for (uint32_t x = 0; x < CT; x++) cm[x] = c1[x] * kLog2e;
        if (terms) {
            float unit = 1.f;
            if (a.cap > 0.f) {
                float far = 0.f;
#pragma unroll
                for (uint32_t x = 0; x < CT; x++)
#pragma unroll
                    for (uint32_t hf = 0; hf < 2u; hf++) {
                        S[hf][x] *= c1[x] * a.rcap;
#pragma unroll
                        for (uint32_t k = 0; k < 4u; k++) far = fmaxf(far, fabsf(S[hf][x][k]));
                    }
                // (most scores lie well below the cap: the polynomial alone then serves the wave)
                if (__any(far >= kTanhPoly)) {
#pragma unroll
                    for (uint32_t x = 0; x < CT; x++)
#pragma unroll
                        for (uint32_t j = 0; j < 8u; j++) S[j >> 2][x][j & 3u] = tanh_any(S[j >> 2][x][j & 3u]);
                } else {
#pragma unroll
                    for (uint32_t x = 0; x < CT; x++)
#pragma unroll
                        for (uint32_t j = 0; j < 8u; j++) S[j >> 2][x][j & 3u] = tanh_poly(S[j >> 2][x][j & 3u]);
                }
                unit = a.cap;
            } else {
#pragma unroll
                for (uint32_t x = 0; x < CT; x++) S[0][x] *= c1[x], S[1][x] *= c1[x];
            }
            if (a.slopes) {
#pragma unroll
                for (uint32_t x = 0; x < CT; x++)
#pragma unroll
                    for (uint32_t j = 0; j < 8u; j++)
                        S[j >> 2][x][j & 3u] = row_far(S[j >> 2][x][j & 3u] * unit, slope[x], a.past + tok[x],
                                                       p0 + 16u * (j >> 2) + 4u * g + (j & 3u));
                unit = 1.f;
            }
#pragma unroll
            for (uint32_t x = 0; x < CT; x++) cm[x] = unit * kLog2e;
        }
        if (!full) {
#pragma unroll
            for (uint32_t x = 0; x < CT; x++)
#pragma unroll
                for (uint32_t j = 0; j < 8u; j++) {
                    const uint32_t o = 16u * (j >> 2) + 4u * g + (j & 3u);
                    bool sees = vis[x] >> o & 1u;
                    if (docs) sees = sees && docs[o] == doc[x];
                    if (!sees) S[j >> 2][x][j & 3u] = -INFINITY;
                }
        }
        float top[CT];
        bool up = false;
#pragma unroll
        for (uint32_t x = 0; x < CT; x++) {
            float v = S[0][x][0];
#pragma unroll
            for (uint32_t j = 1; j < 8u; j++) v = fmaxf(v, S[j >> 2][x][j & 3u]);
            top[x] = v * cm[x];
            up = up || top[x] > m[x] + kLazy;
        }
        if (__any(up)) {
#pragma unroll
            for (uint32_t x = 0; x < CT; x++) {
                float v = fmaxf(top[x], lane_xor<16>(top[x]));
                v = fmaxf(v, lane_xor<32>(v));
                const float mn = v > m[x] + kLazy ? v : m[x];
                const float f = mn == -INFINITY ? 1.f : exp2f(m[x] - mn);
                m[x] = mn;
                l[x] *= f;
#pragma unroll
                for (uint32_t d = 0; d < DT; d++) acc[d][x] *= f;
            }
        }
        rh8 ph[CT], pl[CT];
#pragma unroll
        for (uint32_t x = 0; x < CT; x++) {
            const float ms = m[x] == -INFINITY ? 0.f : m[x] - kLift;
#pragma unroll
            for (uint32_t j = 0; j < 8u; j += 2u) {
                rf2 p;
                p[0] = __builtin_amdgcn_exp2f(fmaf(S[j >> 2][x][j & 3u], cm[x], -ms));
                p[1] = __builtin_amdgcn_exp2f(fmaf(S[j >> 2][x][(j & 3u) + 1u], cm[x], -ms));
                l[x] += p[0];
                l[x] += p[1];
                const rh2 h = __builtin_convertvector(p, rh2);
                const rf2 r = {less_low(p[0], h), less_high(p[1], h)};
                const rh2 q = __builtin_convertvector(r, rh2);
                ph[x][j] = h[0], ph[x][j + 1u] = h[1];
                pl[x][j] = q[0], pl[x][j + 1u] = q[1];
            }
        }
#pragma unroll
        for (uint32_t d = 0; d < DT; d++) {
            const uint8_t *v = lds + vat[d & 7u] + 256u * (d >> 3) + at * RB;
            const rs4 v0 = lds_transposed(v), v1 = lds_transposed(v + 16u * RB);
            const rh8 va = __builtin_bit_cast(rh8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (uint32_t x = 0; x < CT; x++) acc[d][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, ph[x], acc[d][x], 0, 0, 0);
#pragma unroll
            for (uint32_t x = 0; x < CT; x++) acc[d][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pl[x], acc[d][x], 0, 0, 0);
        }
    }

    // l over the four lane groups of a row
    __device__ __forceinline__ void sum_l() {
#pragma unroll
        for (uint32_t x = 0; x < CT; x++) {
            l[x] += lane_xor<16>(l[x]);
            l[x] += lane_xor<32>(l[x]);
        }
    }
};

// Where the results of row r of kv head kvh over range `split` go: the partials, or
// (one range) out, divided by l, and what the mass needs.
struct RowsTo {
    float *acc;
    float2 *ml;     // NULL: out
    float2 *stats;  // NULL: not wanted
    __device__ __forceinline__ RowsTo(const RowsArgs &a, const RowsSplit &sp, const RowsPart &pt, uint32_t kvh,
                                      uint32_t split, uint32_t r) {
        const uint32_t group = a.nqh / a.nkh, rows = a.n * group;
        const uint64_t at = ((uint64_t)kvh * sp.n + split) * rows + r;
        ml = sp.n > 1u ? pt.ml + at : nullptr;
        acc = sp.n > 1u ? pt.acc + at * part_stride(a.hd)
                        : a.out + (uint64_t)(r / group) * a.out_stride + (uint64_t)(kvh * group + r % group) * a.hd;
        stats = sp.n == 1u && pt.stats ? pt.stats + (uint64_t)kvh * rows + r : nullptr;
    }
    __device__ __forceinline__ float scale(float l) const { return ml ? 1.f : l == 0.f ? 0.f : __fdiv_rn(1.f, l); }
    __device__ __forceinline__ void put_ml(float m, float l) const {
        if (ml) *ml = make_float2(m, l);
        if (stats) *stats = make_float2(m, l == 0.f ? 0.f : __fdiv_rn(1.f, l));
    }
};
// The row again in f32 products, by a whole wave (row_whole), to the same place.
template <uint32_t HD>
__device__ __forceinline__ void row_again(const RowsArgs &a, const RowsSplit &sp, const RowsPart &pt, uint32_t kvh,
                                          uint32_t split, uint32_t r, uint32_t s0, uint32_t s1, uint32_t lane) {
    const uint32_t group = a.nqh / a.nkh;
    float m, l, o[(HD + 63u) / 64u];
    row_whole<HD>(a, r / group, kvh * group + r % group, s0, s1, lane, m, l, o);
    const RowsTo to(a, sp, pt, kvh, split, r);
#pragma unroll
    for (uint32_t k = 0; k < (HD + 63u) / 64u; k++)
        if (64u * k + lane < a.hd) to.acc[64u * k + lane] = to.ml ? o[k] : l == 0.f ? 0.f : o[k] / l;
    if (lane == 0) to.put_ml(m, l);
}

// ---- many rows: four waves with rows of their own, slots through two shared buffers ------
template <uint32_t HD, uint32_t CT>
__global__ __launch_bounds__(256, 2) void k_rows(RowsArgs a, RowsSplit sp, RowsPart pt, uint32_t tiles, bool wide_kv,
                                                 bool wide_q) {
    constexpr uint32_t DT = HD / 16u, T = kTile<HD>, CPR = HD / 8u, NC = T * CPR / 256u;
    constexpr uint32_t RB = HD * 2u, TB = T * RB;  // bytes of a row and of a tile
    __shared__ __align__(1024) uint8_t kv[2][2][TB];  // two buffers of K and V
    __shared__ int32_t dl[2][T];
    const uint32_t t = threadIdx.x, wave = t >> 6, lane = t & 63u, col = lane & 15u, g = lane >> 4;
    const uint32_t kvh = blockIdx.x % a.nkh, rest = blockIdx.x / a.nkh;
    const uint32_t split = rest % sp.n, tile = tiles - 1u - rest / sp.n;  // (the longest rows first)
    const uint32_t group = a.nqh / a.nkh, rows = a.n * group, row_tile = tile * 64u * CT;
    const uint32_t end = row_end(a, (min(row_tile + 64u * CT, rows) - 1u) / group);
    const uint32_t s0 = split * sp.len, s1 = min(s0 + sp.len, end);
    if (s0 >= s1) return;  // (the whole workgroup; the merge counts the ranges the same way)
    const uint32_t slots = a.past + a.n, row0 = row_tile + wave * 16u * CT;
    RowTiles<HD, CT> R;
    R.init(a, kvh, row0, wide_q, lane, TB);

    // ---- staging: tile p0 into buffer b, by LDS DMA (no registers; it arrives by the next wait) or,
    // where rows are not whole aligned chunks, through registers
    const uint64_t rstride = (uint64_t)a.nkh * a.hd;
    const uint16_t *kb = a.kc + (uint64_t)kvh * a.hd, *vb = a.vc + (uint64_t)kvh * a.hd;
    int32_t ds = 0;
    uint32_t from[NC];  // a thread's chunks: bytes from the tile's first row
    bool in[NC];        // (dims past head_dim stay 0)
#pragma unroll
    for (uint32_t k = 0; k < NC; k++) {
        const uint32_t id = t + 256u * k, r = id / CPR, d = 8u * tile_chunk<HD>(r, id % CPR);
        from[k] = (uint32_t)(2u * (r * rstride + d));
        in[k] = d < a.hd;
        if (!in[k])
#pragma unroll
            for (uint32_t b = 0; b < 4u; b++) *reinterpret_cast<ru4 *>(&kv[b >> 1][b & 1u][16u * id]) = ru4{0u, 0u, 0u, 0u};
    }
    auto fetch = [&](uint32_t p0, uint32_t b) {
        if (wide_kv && p0 + T <= slots) {
            const uint16_t *kp = kb + p0 * rstride, *vp = vb + p0 * rstride;
#pragma unroll
            for (uint32_t k = 0; k < NC; k++) {
                const uint32_t to = 16u * (256u * k + 64u * wave);
                if (HD == a.hd || in[k]) {
                    dma16s(kp, from[k], (uint32_t)(uintptr_t)&kv[b][0][to]);
                    dma16s(vp, from[k], (uint32_t)(uintptr_t)&kv[b][1][to]);
                }
            }
        } else {
#pragma unroll 1
            for (uint32_t k = 0; k < NC; k++) {
                const uint32_t id = t + 256u * k, r = id / CPR, d = 8u * tile_chunk<HD>(r, id % CPR);
                // (slots behind the last repeat it: what lies there may be no number)
                const uint64_t at = (uint64_t)min(p0 + r, slots - 1u) * rstride;
                *reinterpret_cast<ru4 *>(&kv[b][0][16u * id]) = cache8(kb + at, d, a.hd, wide_kv);
                *reinterpret_cast<ru4 *>(&kv[b][1][16u * id]) = cache8(vb + at, d, a.hd, wide_kv);
            }
        }
        if (a.docs && t < T) ds = a.docs[min(p0 + t, slots - 1u)];
    };
    // every wave's part of the tile has arrived and every wave is done with the other buffer
    auto arrive = [&](uint32_t b) {
        if (a.docs && t < T) dl[b][t] = ds;
        vmcnt_le<0>();
        __syncthreads();
    };

    fetch(s0, 0u);
    arrive(0u);
    for (uint32_t p0 = s0, b = 0; p0 < s1; p0 += T, b ^= 1u) {
        const bool more = p0 + T < s1;
        if (more) fetch(p0 + T, b ^ 1u);
        if (p0 < R.last) {
            const bool full = p0 + T <= min(R.clear, s1);
            uint64_t vis[CT];
#pragma unroll
            for (uint32_t x = 0; x < CT; x++) vis[x] = full ? ~0ull : R.real[x] ? seen_bits(a, R.tok[x], p0, s1) : 0ull;
#pragma unroll
            for (uint32_t h = 0; h < T / 32u; h++) {
                uint32_t v[CT];
#pragma unroll
                for (uint32_t x = 0; x < CT; x++) v[x] = (uint32_t)(vis[x] >> (32u * h));
                R.step(a, &kv[0][0][0], 32u * h, p0 + 32u * h, v, full, a.docs ? &dl[b][32u * h] : nullptr, lane);
            }
        }
        if (more) arrive(b ^ 1u);
        R.turn(b ? 0u - 2u * TB : 2u * TB);
    }
    if (row0 >= rows) return;

    // ---- the rows' sums
    R.sum_l();
    const bool wide_to = a.hd % 4u == 0 && (a.out_stride % 4u == 0 && ((uintptr_t)a.out & 15u) == 0);
#pragma unroll
    for (uint32_t x = 0; x < CT; x++) {
        float nan = R.l[x] * 0.f;
#pragma unroll
        for (uint32_t d = 0; d < DT; d++)
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) nan = fmaf(R.acc[d][x][k], 0.f, nan);
        const uint64_t bad = __ballot(R.real[x] && nan != 0.f);  // (0 times anything finite is 0)
        const uint32_t cols = (uint32_t)(bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xFFFFu;
        if (R.real[x] && !(cols >> col & 1u)) {
            const RowsTo to(a, sp, pt, kvh, split, row0 + 16u * x + col);
            const float inv = to.scale(R.l[x]);
#pragma unroll
            for (uint32_t d = 0; d < DT; d++) {
                const uint32_t d0 = 16u * d + 4u * g;
                if (to.ml || wide_to) {  // (the partials' rows are whole float4s)
                    if (d0 < a.hd) *reinterpret_cast<rf4 *>(to.acc + d0) = R.acc[d][x] * inv;
                } else {
#pragma unroll
                    for (uint32_t k = 0; k < 4u; k++)
                        if (d0 + k < a.hd) to.acc[d0 + k] = R.acc[d][x][k] * inv;
                }
            }
            if (g == 0) to.put_ml(R.m[x] - kLift, R.l[x]);
        }
        // rows whose sums are not finite, one at a time
        for (uint32_t c = 0; cols >> c; c++)
            if (cols >> c & 1u) row_again<HD>(a, sp, pt, kvh, split, row0 + 16u * x + c, s0, s1, lane);
    }
}

// ---- few rows: four waves with the same 16 CT rows, each with slots of its own ---------------
// A wave takes the 32-slot tiles wave, wave + 4, ... of the range, in an LDS buffer of its own (no barrier
// until the end), then the waves' sums are added in LDS.
template <uint32_t HD, uint32_t CT>
__global__ __launch_bounds__(256, 2) void k_rows_few(RowsArgs a, RowsSplit sp, RowsPart pt, bool wide_q) {
    constexpr uint32_t DT = HD / 16u, T = 32u, CPR = HD / 8u, NC = T * CPR / 64u, RB = HD * 2u, TB = T * RB;
    constexpr uint32_t RS = HD + 4u;  // floats of a row's sums in LDS (the rows of a store in different banks)
    constexpr uint32_t OWN = 2u * TB > 16u * CT * RS * 4u ? 2u * TB : 16u * CT * RS * 4u;
    __shared__ __align__(1024) uint8_t kv[4][OWN];
    __shared__ float2 mls[4][16u * CT];
    __shared__ uint32_t bad[16u * CT];
    const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63u, col = lane & 15u, g = lane >> 4;
    const uint32_t kvh = blockIdx.x % a.nkh, rest = blockIdx.x / a.nkh, split = rest % sp.n, row0 = rest / sp.n * 16u * CT;
    const uint32_t group = a.nqh / a.nkh, rows = a.n * group, slots = a.past + a.n;
    const uint32_t end = row_end(a, (min(row0 + 16u * CT, rows) - 1u) / group);
    const uint32_t s0 = split * sp.len, s1 = min(s0 + sp.len, end);
    if (s0 >= s1) return;  // (the whole workgroup)
    uint8_t *const own = &kv[wave][0];
    const uint64_t rstride = (uint64_t)a.nkh * a.hd;
    const uint16_t *kb = a.kc + (uint64_t)kvh * a.hd, *vb = a.vc + (uint64_t)kvh * a.hd;
#pragma unroll
    for (uint32_t k = 0; k < NC; k++) {  // (dims past head_dim stay 0)
        const uint32_t id = lane + 64u * k, r = id / CPR;
        if (8u * tile_chunk<HD>(r, id % CPR) < a.hd) continue;
        *reinterpret_cast<ru4 *>(own + 16u * id) = ru4{0u, 0u, 0u, 0u};
        *reinterpret_cast<ru4 *>(own + TB + 16u * id) = ru4{0u, 0u, 0u, 0u};
    }
    auto fetch = [&](uint32_t p0) {
        const uint16_t *kp = kb + p0 * rstride, *vp = vb + p0 * rstride;
        const uint32_t most = min(slots - p0, T) - 1u;  // (slots behind the last repeat it)
#pragma unroll
        for (uint32_t k = 0; k < NC; k++) {
            const uint32_t id = lane + 64u * k, r = id / CPR, d = 8u * tile_chunk<HD>(r, id % CPR);
            const uint32_t from = (uint32_t)(2u * (min(r, most) * rstride + d));
            if (HD == a.hd || d < a.hd) {
                dma16s(kp, from, (uint32_t)(uintptr_t)(own + 1024u * k));
                dma16s(vp, from, (uint32_t)(uintptr_t)(own + TB + 1024u * k));
            }
        }
    };
    uint32_t p0 = s0 + T * wave;
    if (p0 < s1) fetch(p0);
    RowTiles<HD, CT> R;
    R.init(a, kvh, row0, wide_q, lane, TB);
    while (p0 < s1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (p0 < R.last) {
            const bool full = p0 + T <= min(R.clear, s1);
            uint32_t vis[CT];
#pragma unroll
            for (uint32_t x = 0; x < CT; x++) vis[x] = full ? ~0u : R.real[x] ? (uint32_t)seen_bits(a, R.tok[x], p0, s1) : 0u;
            R.step(a, own, 0u, p0, vis, full, a.docs ? a.docs + p0 : nullptr, lane);
        }
        p0 += 4u * T;
        if (p0 >= s1) break;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the tile has been read)
        fetch(p0);
    }
    // ---- the waves' sums: M = max m_w, sum acc_w 2^(m_w - M), in the order of the waves
    R.sum_l();
    float *const sums = reinterpret_cast<float *>(own);
#pragma unroll
    for (uint32_t x = 0; x < CT; x++) {
#pragma unroll
        for (uint32_t d = 0; d < DT; d++)
            *reinterpret_cast<rf4 *>(sums + (16u * x + col) * RS + 16u * d + 4u * g) = R.acc[d][x];
        if (g == 0) mls[wave][16u * x + col] = make_float2(R.m[x], R.l[x]);
    }
    if (t < 16u * CT) bad[t] = 0;
    __syncthreads();
    const bool wide_to = a.hd % 4u == 0 && a.out_stride % 4u == 0 && ((uintptr_t)a.out & 15u) == 0;
    for (uint32_t e = t; e < 16u * CT * (HD / 4u); e += 256u) {
        const uint32_t r = e / (HD / 4u), d0 = 4u * (e % (HD / 4u));
        if (row0 + r >= rows || d0 >= a.hd) continue;
        float M = -INFINITY, l = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < 4u; w++) M = fmaxf(M, mls[w][r].x);
        const float ref = M == -INFINITY ? 0.f : M;
        rf4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (uint32_t w = 0; w < 4u; w++) {
            const float2 v = mls[w][r];
            const float f = exp2f(v.x - ref);
            l = fmaf(v.y, f, l);
            o += *reinterpret_cast<const rf4 *>(reinterpret_cast<const float *>(&kv[w][0]) + r * RS + d0) * f;
        }
        const RowsTo to(a, sp, pt, kvh, split, row0 + r);
        const float inv = to.scale(l);
        const float nan = fmaf(o[0], 0.f, fmaf(o[1], 0.f, fmaf(o[2], 0.f, fmaf(o[3], 0.f, l * 0.f))));
        if (nan != 0.f) bad[r] = 1u;
        o *= inv;
        if (to.ml || wide_to) {
            *reinterpret_cast<rf4 *>(to.acc + d0) = o;
        } else {
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++)
                if (d0 + k < a.hd) to.acc[d0 + k] = o[k];
        }
        if (d0 == 0) to.put_ml(M - kLift, l);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (a row that is taken again is written after this)
    __syncthreads();
    for (uint32_t r = wave; r < 16u * CT; r += 4u)
        if (bad[r]) row_again<HD>(a, sp, pt, kvh, split, row0 + r, s0, s1, lane);
}

// ---- the ranges of a row added up ----------------------------------------------------
// TPR threads per row: M = max m_c, L = sum l_c 2^(m_c - M), out = sum acc_c 2^(m_c - M) / L. Every wave holds the
// weights of the ranges in its lanes; lane groups of a row's float4s take the ranges in turn, eight at a time in
// flight, and the groups are added in order.
constexpr uint32_t kMostRanges = 128;

template <uint32_t TPR>
__global__ __launch_bounds__(256) void k_rows_merge(RowsArgs a, RowsSplit sp, RowsPart pt, uint32_t tile_rows, uint32_t width) {
    __shared__ rf4 part[256];
    const uint32_t t = threadIdx.x, lane = t & 63u, in = t % TPR, kvh = blockIdx.y;
    const uint32_t group = a.nqh / a.nkh, rows = a.n * group, r = min(blockIdx.x * (256u / TPR) + t / TPR, rows - 1u);
    const uint32_t end = row_end(a, (min(r / tile_rows * tile_rows + tile_rows, rows) - 1u) / group);
    const uint32_t n = (end + sp.len - 1u) / sp.len;
    const uint32_t q = in % width, grp = in / width, groups = TPR / width, ps = part_stride(a.hd);
    const float2 *ml = pt.ml + (uint64_t)kvh * sp.n * rows + r;
    const float *acc = pt.acc + ((uint64_t)kvh * sp.n * rows + r) * ps + 4u * q;
    const bool mine = 4u * q < a.hd;
    rf4 v[8];
    auto load = [&](uint32_t c0) {
#pragma unroll
        for (uint32_t k = 0; k < 8u; k++) {
            const uint32_t c = c0 + k * groups;
            v[k] = mine && c < n ? *reinterpret_cast<const rf4 *>(acc + (uint64_t)c * rows * ps) : rf4{0.f, 0.f, 0.f, 0.f};
        }
    };
    load(grp);
    const float2 none = make_float2(-INFINITY, 0.f);
    const float2 x0 = lane < n ? ml[(uint64_t)lane * rows] : none;
    const float2 x1 = lane + 64u < n ? ml[(uint64_t)(lane + 64u) * rows] : none;
    const float M = wave_max(fmaxf(x0.x, x1.x)), ref = M == -INFINITY ? 0.f : M;
    const float w0 = exp2f(x0.x - ref), w1 = exp2f(x1.x - ref);
    const float L = wave_sum(fmaf(x0.y, w0, x1.y * w1));
    rf4 o = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t c0 = grp; c0 < n + grp; c0 += 8u * groups) {  // (the same count in every lane)
        if (c0 != grp) load(c0);
#pragma unroll
        for (uint32_t k = 0; k < 8u; k++) {
            const uint32_t c = c0 + k * groups;
            const float f0 = __shfl(w0, (int)(c & 63u), 64), f1 = __shfl(w1, (int)(c & 63u), 64);
            if (c < n) o += v[k] * (c < 64u ? f0 : f1);
        }
    }
    part[t] = o;
    __syncthreads();
    if (grp || !mine || blockIdx.x * (256u / TPR) + t / TPR >= rows) return;
    for (uint32_t k = 1; k < groups; k++) o += part[t + k * width];
    const float inv = L == 0.f ? 0.f : __fdiv_rn(1.f, L);
    float *to = a.out + (uint64_t)(r / group) * a.out_stride + (uint64_t)(kvh * group + r % group) * a.hd + 4u * q;
#pragma unroll
    for (uint32_t k = 0; k < 4u; k++)
        if (4u * q + k < a.hd) to[k] = L == 0.f ? 0.f : o[k] * inv;
    if (q == 0 && pt.stats) pt.stats[(uint64_t)kvh * rows + r] = make_float2(M, inv);
}

// ---- the weights that slots received ---------------------------------------------------
// A workgroup takes 64 (32 for head_dim above 128) slots of a kv head, their K rows as A operands in registers;
// its waves take the row tiles of 16 in turn (S^T as above) and each lane adds up
// 2^(y - m) / l for its slots; the 16 columns, then the waves, are summed at the end
// in a fixed order. A slot whose sum is not finite is taken again in f32 products.
constexpr uint32_t kMassWaves = 8;

template <uint32_t HD>
constexpr uint32_t kMassTiles = HD > 128u ? 2u : 4u;

template <uint32_t HD>
__global__ __launch_bounds__(64 * kMassWaves) void k_mass(RowsArgs a, const float2 *__restrict__ stats, bool wide_kv,
                                                          bool wide_q) {
    constexpr uint32_t KK = HD / 32u, NT = kMassTiles<HD>, NP = 16u * NT;  // tiles of 16 slots; slots
    __shared__ float sums[kMassWaves][NP];
    const uint32_t t = threadIdx.x, wave = t >> 6, lane = t & 63u, col = lane & 15u, g = lane >> 4;
    const uint32_t waves = blockDim.x >> 6, kvh = blockIdx.x % a.nkh, p0 = blockIdx.x / a.nkh * NP;
    const uint32_t group = a.nqh / a.nkh, rows = a.n * group, slots = a.past + a.n;
    const uint64_t rstride = (uint64_t)a.nkh * a.hd;
    rh8 ka[NT][KK];
    int32_t ds[NT][4];
#pragma unroll
    for (uint32_t hf = 0; hf < NT; hf++) {
        const uint16_t *k = a.kc + (uint64_t)min(p0 + 16u * hf + col, slots - 1u) * rstride + (uint64_t)kvh * a.hd;
#pragma unroll
        for (uint32_t kk = 0; kk < KK; kk++)
            ka[hf][kk] = __builtin_bit_cast(rh8, cache8(k, 32u * kk + 8u * g, a.hd, wide_kv));
#pragma unroll
        for (uint32_t r = 0; r < 4u; r++)
            ds[hf][r] = a.docs ? a.docs[min(p0 + 16u * hf + 4u * g + r, slots - 1u)] : 0;
    }
    float sum[NT][4] = {};
    const bool terms = a.cap > 0.f || a.slopes;
    // the rows before the first that sees p0 (without a mask or a prefix beyond it) are left out
    const uint32_t r0 = a.mask || p0 < a.prefix || p0 <= a.past ? 0u : (p0 - a.past) * group / 16u;
    for (uint32_t rt = r0 + wave; 16u * rt < rows; rt += waves) {
        const uint32_t r = 16u * rt + col;
        const bool real = r < rows;
        const uint32_t i = real ? r / group : 0u, h = kvh * group + (real ? r % group : 0u);
        rh8 qh[KK], ql[KK];
        float c1;
        const float2 st = real ? stats[(uint64_t)kvh * rows + r] : make_float2(0.f, 0.f);
        row_parts<KK>(real ? a.q + (uint64_t)i * a.q_stride + (uint64_t)h * a.hd : nullptr, a.hd, wide_q, a.scale, g, qh,
                      ql, c1);
        const bool full = !a.docs && 16u * rt + 16u <= rows &&
                          p0 + NP <= (a.mask ? a.past : row_end(a, 16u * rt / group));
        const uint64_t vis = full ? ~0ull : real ? seen_bits(a, i, p0, slots) : 0ull;
        const int32_t doc = a.docs ? a.docs[a.past + i] : 0;
        const float slope = a.slopes ? a.slopes[h] : 0.f, ms = st.x == -INFINITY ? 0.f : st.x;
#pragma unroll
        for (uint32_t hf = 0; hf < NT; hf++) {
            rf4 S = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t kk = 0; kk < KK; kk++) S = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[hf][kk], qh[kk], S, 0, 0, 0);
#pragma unroll
            for (uint32_t kk = 0; kk < KK; kk++) S = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[hf][kk], ql[kk], S, 0, 0, 0);
#pragma unroll
            for (uint32_t k = 0; k < 4u; k++) {
                const uint32_t o = 16u * hf + 4u * g + k;
                float y;
                if (full && !terms) {
                    y = fmaf(S[k], c1 * kLog2e, -ms);
                } else {
                    float s = S[k] * c1;
                    if (terms) s = row_score(a, s, slope, a.past + i, p0 + o);
                    const bool sees = (vis >> o & 1ull) && (!a.docs || ds[hf][k] == doc);
                    y = sees ? fmaf(s, kLog2e, -ms) : -INFINITY;
                }
                sum[hf][k] = fmaf(__builtin_amdgcn_exp2f(y), st.y, sum[hf][k]);
            }
        }
    }
    // the 16 columns: each lane group's row of 16 lanes
#pragma unroll
    for (uint32_t hf = 0; hf < NT; hf++)
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) {
            float v = sum[hf][k];
            v += bfly_partner<8>(v, lane);
            v += bfly_partner<4>(v, lane);
            v += bfly_partner<2>(v, lane);
            v += bfly_partner<1>(v, lane);
            if (col == 0) sums[wave][16u * hf + 4u * g + k] = v;
        }
    __syncthreads();
    if (wave) return;
    const uint32_t j = p0 + lane;
    const bool in = lane < NP && j < slots;
    float v = 0.f;
    for (uint32_t w = 0; w < waves; w++) v += sums[w][lane % NP];
    const uint64_t bad = __ballot(in && v * 0.f != 0.f);
    for (uint32_t c = 0; c < 64u && bad >> c; c++) {
        if (!(bad >> c & 1ull)) continue;
        const uint32_t jj = p0 + c;
        const uint16_t *k = a.kc + (uint64_t)jj * rstride + (uint64_t)kvh * a.hd;
        float whole = 0.f;
        for (uint32_t r = lane; r < rows; r += 64u) {
            const uint32_t i = r / group, h = kvh * group + r % group;
            if (jj >= row_end(a, i) || !row_sees(a, i, jj)) continue;
            const float s = row_score(a, row_dot(a.q + (uint64_t)i * a.q_stride + (uint64_t)h * a.hd, k, a.hd) * a.scale,
                                      a.slopes ? a.slopes[h] : 0.f, a.past + i, jj);
            const float2 st = stats[(uint64_t)kvh * rows + r];
            whole += exp2f(fmaf(s, kLog2e, -(st.x == -INFINITY ? 0.f : st.x))) * st.y;
        }
        whole = wave_sum(whole);
        if (lane == c) v = whole;
    }
    if (in) a.mass[(uint64_t)kvh * a.max_ctx + j] += v;
}

// ---- launches -------------------------------------------------------------------------------

struct RowsPlan {
    uint32_t hd, ct, tiles;  // template head size, column tiles a wave, row tiles a kv head
    bool few;
    RowsSplit sp;
    size_t ml, acc, stats;  // bytes
};

// Whether rows of the caches and of q may be read 16 bytes at a time.
static bool rows_wide_kv(const RowsArgs &a) {
    return a.hd % 8u == 0 && (((uintptr_t)a.kc | (uintptr_t)a.vc) & 15u) == 0;
}
static bool rows_wide_q(const RowsArgs &a) {
    return a.hd % 8u == 0 && a.q_stride % 4u == 0 && ((uintptr_t)a.q & 15u) == 0;
}

static RowsPlan rows_plan(const RowsArgs &a) {
    RowsPlan p{};
    p.hd = a.hd <= 32u ? 32u : a.hd <= 64u ? 64u : a.hd <= 96u ? 96u : a.hd <= 128u ? 128u : 256u;
    const uint32_t rows = a.n * (a.nqh / a.nkh), slots = a.past + a.n;
    p.few = rows <= 16u && rows_wide_kv(a);
    p.ct = p.few || rows <= 64u || p.hd > 128u ? 1u : 2u;
    const uint32_t tile_rows = (p.few ? 16u : 64u) * p.ct;
    p.tiles = (rows + tile_rows - 1u) / tile_rows;
    // ranges: until about 512 workgroups share the work, at least a tile a wave or workgroup each
    const uint32_t least = p.few ? 128u : 64u, most = (slots + least - 1u) / least, wgs = p.tiles * a.nkh;
    uint32_t n = 512u / wgs;
    n = n < 1u ? 1u : n > most ? most : n > kMostRanges ? kMostRanges : n;
    p.sp.len = ((slots + n - 1u) / n + least - 1u) / least * least;
    p.sp.n = (slots + p.sp.len - 1u) / p.sp.len;
    const size_t all = (size_t)rows * a.nkh;
    const auto round = [](size_t b) { return (b + 255u) & ~(size_t)255u; };
    if (p.sp.n > 1u) {
        p.ml = round(all * p.sp.n * sizeof(float2));
        p.acc = round(all * p.sp.n * part_stride(a.hd) * sizeof(float));
    }
    if (a.mass) p.stats = round(all * sizeof(float2));
    return p;
}

size_t rows_scratch_bytes(const RowsArgs &a) {
    const RowsPlan p = rows_plan(a);
    return p.ml + p.acc + p.stats;
}

template <uint32_t HD>
static void start_rows(const RowsArgs &a, const RowsPlan &p, const RowsPart &pt, hipStream_t s) {
    const bool wide_kv = rows_wide_kv(a), wide_q = rows_wide_q(a);
    const uint32_t grid = p.tiles * p.sp.n * a.nkh;
    if (p.few) {
        k_rows_few<HD, 1><<<grid, 256, 0, s>>>(a, p.sp, pt, wide_q);
        return;
    }
    if constexpr (HD <= 128u) {
        if (p.ct == 2u) {
            k_rows<HD, 2><<<grid, 256, 0, s>>>(a, p.sp, pt, p.tiles, wide_kv, wide_q);
            return;
        }
    }
    k_rows<HD, 1><<<grid, 256, 0, s>>>(a, p.sp, pt, p.tiles, wide_kv, wide_q);
}

template <uint32_t HD>
static void start_mass(const RowsArgs &a, const RowsPart &pt, hipStream_t s) {
    const uint32_t tiles = (a.n * (a.nqh / a.nkh) + 15u) / 16u;
    const uint32_t np = 16u * kMassTiles<HD>;
    k_mass<HD><<<(a.past + a.n + np - 1u) / np * a.nkh, 64u * (tiles < kMassWaves ? tiles : kMassWaves), 0, s>>>(
        a, pt.stats, rows_wide_kv(a), rows_wide_q(a));
}

hipError_t launch_rows(const RowsArgs &a, void *scratch, hipStream_t s) {
    const RowsPlan p = rows_plan(a);
    uint8_t *at = static_cast<uint8_t *>(scratch);
    RowsPart pt{};
    if (p.sp.n > 1u) pt.ml = reinterpret_cast<float2 *>(at), pt.acc = reinterpret_cast<float *>(at + p.ml);
    if (a.mass) pt.stats = reinterpret_cast<float2 *>(at + p.ml + p.acc);
    switch (p.hd) {
        case 32: start_rows<32>(a, p, pt, s); break;
        case 64: start_rows<64>(a, p, pt, s); break;
        case 96: start_rows<96>(a, p, pt, s); break;
        case 128: start_rows<128>(a, p, pt, s); break;
        default: start_rows<256>(a, p, pt, s); break;
    }
    hipError_t e = hipGetLastError();
    const uint32_t rows = a.n * (a.nqh / a.nkh);
    if (e == hipSuccess && p.sp.n > 1u) {
        const uint32_t tile_rows = (p.few ? 16u : 64u) * p.ct;
        const uint32_t width = a.hd <= 32u ? 8u : a.hd <= 64u ? 16u : a.hd <= 128u ? 32u : 64u;  // float4s of a row
        // a wave per row where its lanes hold every range in one round of loads
        if (p.sp.n <= 8u * (64u / width))
            k_rows_merge<64><<<dim3((rows + 3u) / 4u, a.nkh), 256, 0, s>>>(a, p.sp, pt, tile_rows, width);
        else
            k_rows_merge<256><<<dim3(rows, a.nkh), 256, 0, s>>>(a, p.sp, pt, tile_rows, width);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a.mass) {
        switch (p.hd) {
            case 32: start_mass<32>(a, pt, s); break;
            case 64: start_mass<64>(a, pt, s); break;
            case 96: start_mass<96>(a, pt, s); break;
            case 128: start_mass<128>(a, pt, s); break;
            default: start_mass<256>(a, pt, s); break;
        }
        e = hipGetLastError();
    }
    return e;
}

}  // namespace vbs
