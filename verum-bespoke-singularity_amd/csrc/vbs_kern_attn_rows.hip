// vbs_kern_attn_rows.hip — attention of several tokens over the f16 KV cache: a chunk
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
// i * group + g. A workgroup takes 64 rows of one kv head (16 a wave) and a range of
// slots, 64 (32 for head_dim above 128) at a time through LDS, on
// v_mfma_f32_16x16x32_f16:
// * S^T = K Q^T: A = 16 slots x 32 dims of K (the cache's f16, exact), B = 32 dims
//   x 16 rows of q' = q 2^s, s so that the row's largest |q'| lies in [2^14, 2^15),
//   as two f16 parts hi + lo (22 bits; the two products add up in the same f32
//   sums). A lane then holds the scores of one row (column lane & 15) at slots
//   16 i + 4 (lane >> 4) + k, so the softmax needs no row-wise exchange but for the
//   maximum.
// * the running maximum moves only where a score passes it by more than 4 in
//   log2: then the sums are rescaled. The weights are 2^(y - m + 11) <= 2^15, so that
//   small ones keep their low part in f16: what lies 2^-36 below the greatest is in l
//   but no longer in V's sum, 1e-6 of V over 65536 such slots in one range (8 and 2^7:
//   2^-32 and 1.5e-5; 2 and 2^13: 2^-38). Moving it more often costs little: 2048 tokens over
//   8192 slots, 32/8 heads of 128, 457 to 460 us, over 4096 of heads of 64 130 to 133.
// * O^T += V^T P^T: B = P^T, the lane's own weights (hi, then lo), A = V^T with the
//   k slots in the same order, by transposed LDS reads.
// Each range of slots ends in m, l and acc per row; where a kv head's rows are few
// the slots are split over several workgroups and k_attn_rows_merge adds them up,
// scaled to the common maximum.
//
// Precision: q and the weights keep 22 bits, everything else f32; error against 64
// bits 2.6e-7 to 1.1e-6 over scores of a few units, the same in f32 matrix products
// 3.8e-7 to 2.1e-6.
// Bound, long chunks: the matrix cores and the vector unit share a SIMD's issue; a
// 64-slot tile of 16 rows is 64 products (1024 cycles) and about 335 vector
// instructions with the cap. 2048 tokens over 8192 slots, 32/8 heads of 128, capped:
// 540-570 us, 840-890 TFLOP/s of f16 products (a library product of 8192^3: 1120-1165).
// Measured beside it: 32 rows a wave 614, 16 rows and four waves a SIMD 842 (registers
// spill), three waves a SIMD 667, a ring of four tiles 581, V transposed by permutes
// instead of by the LDS read 857.
// A row that is taken again (row_whole) costs a wave of its own: 1024 tokens over 2048 slots, 32/8 heads of 128, of
// which every row shares a tile with an unseen infinite V: 26.8 ms for 87 us; one token of far scores: 3.1 ms.
// Short ones: launches and one round trip to memory each; 16 tokens over 2048 slots
// 10.9 + 4.2 us under the tracer.
#include "vbs_lds_dma.h"
#include "vbs_attn_rows.h"

namespace vbs {

constexpr float kLazy = 4.f, kLift = 11.f;  // log2: how far a score may pass m; the weights' scale

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

// One row of q (column lane & 15), lane group g's part: dims 32 kk + 8 g ..
template <uint32_t KK>
struct RowQ {
    float x[KK][8];
    // `row` NULL: zeros
    __device__ __forceinline__ void load(const float *row, uint32_t hd, bool wide, uint32_t g) {
#pragma unroll
        for (uint32_t kk = 0; kk < KK; kk++) {
            const uint32_t d0 = 32u * kk + 8u * g;
            if (row && wide && d0 < hd) {
                const rf4 u = *reinterpret_cast<const rf4 *>(row + d0), v = *reinterpret_cast<const rf4 *>(row + d0 + 4u);
#pragma unroll
                for (uint32_t e = 0; e < 4u; e++) x[kk][e] = u[e], x[kk][4u + e] = v[e];
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 8u; e++) x[kk][e] = row && !wide && d0 + e < hd ? row[d0 + e] : 0.f;
            }
        }
    }
    // its parts, and c: |scale| 2^-s, what a product of the parts is to be scaled by
    __device__ __forceinline__ void split(float scale, rh8 (&hi)[KK], rh8 (&lo)[KK], float &c) const {
        float top = 0.f;
#pragma unroll
        for (uint32_t kk = 0; kk < KK; kk++)
#pragma unroll
            for (uint32_t e = 0; e < 8u; e++) top = fmaxf(top, fabsf(x[kk][e]));
        top = fmaxf(top, lane_xor<16>(top));
        top = fmaxf(top, lane_xor<32>(top));
        int e2 = 0;
        (void)frexpf(top, &e2);  // top < 2^e2
        // (a row below 2^-111 scores nothing that an f32 sum keeps; 2^-sq must stay a number)
        const int sq = top > 0.f && top < INFINITY ? (15 - e2 < 126 ? 15 - e2 : 126) : 0;
        c = ldexpf(fabsf(scale), -sq);
        if (c < 0x1p-126f) c = 0x1p-126f;  // (not 0: masked scores are -inf times it; a NaN stays)
        const float sign = scale < 0.f ? -1.f : 1.f;
#pragma unroll
        for (uint32_t kk = 0; kk < KK; kk++)
#pragma unroll
            for (uint32_t e = 0; e < 8u; e += 2u) {
                const rf2 y = {ldexpf(x[kk][e] * sign, sq), ldexpf(x[kk][e + 1u] * sign, sq)};
                const rh2 h = __builtin_convertvector(y, rh2);
                const rf2 r = {less_low(y[0], h), less_high(y[1], h)};
                const rh2 q = __builtin_convertvector(r, rh2);
                hi[kk][e] = h[0], hi[kk][e + 1u] = h[1];
                lo[kk][e] = q[0], lo[kk][e + 1u] = q[1];
            }
    }
};

// The documents of the tokens i0 .. i1 lie in [lo, hi]: slots of others are not looked at.
struct DocRange {
    int32_t lo, hi;
    // which of the four runs of 64 slots from `win` on (a multiple of 64) hold a slot of the range
    uint32_t win, runs;

    // (the first window's documents are asked for with the tokens': one round trip)
    __device__ __forceinline__ DocRange(const RowsArgs &a, uint32_t i0, uint32_t i1, uint32_t s0, uint32_t s1, uint32_t lane) {
        lo = 0x7FFFFFFF, hi = -0x7FFFFFFF - 1, win = s0, runs = 0;
        if (!a.docs) return;
        int32_t d[4];
        read(a, s0, s1, lane, d);
        for (uint32_t i = i0 + lane; i <= i1; i += 64u) {
            const int32_t own = a.docs[a.past + i];
            lo = min(lo, own), hi = max(hi, own);
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) lo = min(lo, __shfl_xor(lo, o, 64)), hi = max(hi, __shfl_xor(hi, o, 64));
        look(s0, s1, lane, d);
    }
    __device__ __forceinline__ static void read(const RowsArgs &a, uint32_t p, uint32_t s1, uint32_t lane, int32_t (&d)[4]) {
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) d[k] = a.docs[min(p + 64u * k + lane, s1 - 1u)];
    }
    __device__ __forceinline__ void look(uint32_t p, uint32_t s1, uint32_t lane, const int32_t (&d)[4]) {
        win = p, runs = 0;
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++)
            if (__any(p + 64u * k + lane < s1 && d[k] >= lo && d[k] <= hi)) runs |= 1u << k;
    }
    // The first slot from p on (a multiple of 32) whose run of 64 holds a slot of the range, a multiple of 64 unless it
    // is p itself; s1 if there is none. Slots are looked at 256 in one round of loads.
    __device__ __forceinline__ uint32_t next(const RowsArgs &a, uint32_t p, uint32_t s1, uint32_t lane) {
        if (!a.docs) return p;
        while (p < s1) {
            if (p - win >= 256u) {
                int32_t d[4];
                read(a, p / 64u * 64u, s1, lane, d);
                look(p / 64u * 64u, s1, lane, d);
            }
            const uint32_t k = (p - win) / 64u, left = runs >> k;
            if (left & 1u) return p;
            if (left) return win + 64u * (k + (uint32_t)__builtin_ctz(left));
            p = win + 256u;
        }
        return s1;
    }
};

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
    uint32_t len, n;  // slots per range (a multiple of 128), ranges
};

// How the launch's scratch is laid out: (m, l) then acc per (kv head, range, row),
// then (m, 1 / l) per (kv head, row), then what the mass needs.
__host__ __device__ __forceinline__ uint64_t score_stride(uint32_t slots) { return ((uint64_t)slots + 31u) / 32u * 32u; }
struct RowsPart {
    float2 *ml;
    float *acc;
    float2 *stats;
    float *scores;  // few rows with a mass: (kv head, row, score_stride(slots)), else NULL
    // many rows with a mass: the parts of q as the matrix cores take them (kv head, 16-row tile, slice of 32 dims,
    // lane; 16 bytes of the high part, then 16 of the low) and the rows' c, else NULL
    ru4 *qparts;
    float *qc;
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

// Sixteen rows of a wave (one a column): their q' parts and their running sums.
template <uint32_t HD>
struct RowTile {
    static constexpr uint32_t KK = HD / 32u, DT = HD / 16u, RB = HD * 2u;
    // where the lane reads in LDS, from a tile's first byte of K: where places are xors, one address
    // each for K and V and the slice or dim tile xored in, else (96) one per slice and dim tile
    static constexpr bool XOR = HD != 96u;
    static constexpr uint32_t NK = XOR ? 1u : KK, NV = XOR ? 1u : DT;
    rh8 qh[KK], ql[KK];
    float c1, slope, m, l;
    uint32_t tok;
    int32_t doc;
    bool real;
    rf4 acc[DT];
    uint32_t kat[NK], vat[NV];
    // below `clear` every row sees every slot (documents aside); from `last` on, none
    uint32_t clear, last;

    // what is read of q (its loads are to be under way before the first tile's, behind which they would wait)
    __device__ __forceinline__ static void load(const RowsArgs &a, uint32_t kvh, uint32_t row0, bool wide_q, uint32_t lane,
                                                RowQ<KK> &x) {
        const uint32_t group = a.group, r = row0 + (lane & 15u), i = row_token(a, r);
        x.load(r < a.n * group ? a.q + (uint64_t)i * a.q_stride + (uint64_t)(kvh * group + r - i * group) * a.hd : nullptr,
               a.hd, wide_q, lane >> 4);
    }
    // v_at: from a tile's first byte of K to its first of V
    __device__ __forceinline__ void init(const RowsArgs &a, uint32_t kvh, uint32_t row0, const RowQ<KK> &x, uint32_t lane,
                                         uint32_t v_at) {
        const uint32_t col = lane & 15u, g = lane >> 4, group = a.group, rows = a.n * group;
        const uint32_t r = row0 + col;
        real = r < rows;
        tok = real ? row_token(a, r) : 0u;
        const uint32_t h = kvh * group + (real ? r - tok * group : 0u);
        slope = a.slopes ? a.slopes[h] : 0.f;
        doc = a.docs ? a.docs[a.past + tok] : 0;
        x.split(a.scale, qh, ql, c1);
        m = -INFINITY, l = 0.f;
#pragma unroll
        for (uint32_t d = 0; d < DT; d++) acc[d] = rf4{0.f, 0.f, 0.f, 0.f};
        clear = a.docs ? 0u : a.mask ? a.past : row_end(a, row_token(a, min(row0, rows - 1u)));
        last = row0 < rows ? row_end(a, row_token(a, min(row0 + 16u, rows) - 1u)) : 0u;
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

    // (dims from 128 on lie 256 bytes on)
    __device__ __forceinline__ uint32_t k_at(uint32_t kk) const {
        return XOR ? (kat[0] ^ 64u * (kk & 3u)) + 256u * (kk >> 2) : kat[XOR ? 0u : kk];
    }
    __device__ __forceinline__ uint32_t v_at(uint32_t d) const {
        return XOR ? (vat[0] ^ 32u * (d & 7u)) + 256u * (d >> 3) : vat[XOR ? 0u : d];
    }

    __device__ __forceinline__ void turn(uint32_t by) {  // on to another buffer
#pragma unroll
        for (uint32_t kk = 0; kk < NK; kk++) kat[kk] += by;
#pragma unroll
        for (uint32_t d = 0; d < NV; d++) vat[d] += by;
    }

    // 32 NH slots from p0 on, in LDS; full: every row sees them all, else vis holds their bits and docs (or NULL)
    // their documents. Slot 16 i + 4 g + k is element S[i][k]. `scores` (or NULL): where the row's scores of these
    // slots go, in units of log2.
    template <uint32_t NH, bool DOCS_LDS>
    __device__ __forceinline__ void step(const RowsArgs &a, const uint8_t *lds, uint32_t p0, uint64_t vis, bool full,
                                         const int32_t *docs, uint32_t lane, float *scores = nullptr) {
        // 16-slot tiles; dim tiles at a time (two at head_dim 256, which leave 21 registers in memory; four
        // 39)
        constexpr uint32_t NS = 2u * NH, ND = DT < 4u ? DT : DT % 4u || DT > 8u ? 2u : 4u;
        const uint32_t g = lane >> 4;
        // A product waits for the one before it into the same sums: the tiles are taken in turn, the high parts
        // then the low, so that four products lie between. Each slice's K is read while the one before it is
        // multiplied, and V a group of dim tiles ahead: left to itself the compiler waits for every read in turn.
        rf4 S[NS];
        rh8 ka[2][NS], va[2][ND];
#pragma unroll
        for (uint32_t i = 0; i < NS; i++) S[i] = rf4{0.f, 0.f, 0.f, 0.f};
        auto read_k = [&](uint32_t kk) {
#pragma unroll
            for (uint32_t i = 0; i < NS; i++) ka[kk & 1u][i] = *reinterpret_cast<const rh8 *>(lds + k_at(kk) + 16u * i * RB);
        };
        // group u of V: ND dim tiles of half u % NH
        auto read_v = [&](uint32_t u) {
#pragma unroll
            for (uint32_t d = 0; d < ND; d++) {
                const uint8_t *v = lds + v_at(u / NH * ND + d) + u % NH * 32u * RB;
                const rs4 v0 = lds_transposed(v), v1 = lds_transposed(v + 16u * RB);
                va[u & 1u][d] = __builtin_bit_cast(rh8, __builtin_shufflevector(v0, v1, 0, 1, 2, 3, 4, 5, 6, 7));
            }
        };
        read_k(0u);
#pragma unroll
        for (uint32_t kk = 0; kk < KK; kk++) {
            if (kk + 1u < KK)
                read_k(kk + 1u);
            else
                read_v(0u);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (uint32_t i = 0; i < NS; i++) S[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[kk & 1u][i], qh[kk], S[i], 0, 0, 0);
#pragma unroll
            for (uint32_t i = 0; i < NS; i++) S[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[kk & 1u][i], ql[kk], S[i], 0, 0, 0);
        }
        // the score in units of log2 is cm S: S the plain product, or what the terms make of it
        float cm = c1 * kLog2e;
        if (a.cap > 0.f || a.slopes) {
            float unit = 1.f;
            if (a.cap >= kFarCap) {
#pragma unroll
                for (uint32_t i = 0; i < NS; i++)
#pragma unroll
                    for (uint32_t k = 0; k < 4u; k++) S[i][k] = capped(a, S[i][k] * c1);
            } else if (a.cap > 0.f) {
                float far = 0.f;
#pragma unroll
                for (uint32_t i = 0; i < NS; i++) {
                    S[i] *= c1 * a.rcap;
#pragma unroll
                    for (uint32_t k = 0; k < 4u; k++) far = fmaxf(far, fabsf(S[i][k]));
                }
                // (most scores lie well below the cap: the polynomial alone then serves the wave)
                if (__any(far >= kTanhPoly)) {
#pragma unroll
                    for (uint32_t i = 0; i < NS; i++)
#pragma unroll
                        for (uint32_t k = 0; k < 4u; k++) S[i][k] = tanh_any(S[i][k]);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < NS; i++)
#pragma unroll
                        for (uint32_t k = 0; k < 4u; k++) S[i][k] = tanh_poly(S[i][k]);
                }
                unit = a.cap;
            } else {
#pragma unroll
                for (uint32_t i = 0; i < NS; i++) S[i] *= c1;
            }
            if (a.slopes) {
#pragma unroll
                for (uint32_t i = 0; i < NS; i++)
#pragma unroll
                    for (uint32_t k = 0; k < 4u; k++)
                        S[i][k] = row_far(S[i][k] * unit, slope, a.past + tok, p0 + 16u * i + 4u * g + k);
                unit = 1.f;
            }
            cm = unit * kLog2e;
        }
        if (!full) {
#pragma unroll
            for (uint32_t i = 0; i < NS; i++) {
                typedef int32_t ri4 __attribute__((ext_vector_type(4)));
                ri4 d = {doc, doc, doc, doc};
                if (docs && DOCS_LDS) d = *reinterpret_cast<const ri4 *>(docs + 16u * i + 4u * g);
#pragma unroll
                for (uint32_t k = 0; k < 4u; k++) {
                    const uint32_t o = 16u * i + 4u * g + k;
                    const bool in = vis >> o & 1ull;
                    if (docs && !DOCS_LDS && in) d[k] = docs[o];  // (behind the last slot there is none)
                    S[i][k] = in & (d[k] == doc) ? S[i][k] : -INFINITY;
                }
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < NS; i++) top = fmaxf(top, fmaxf(fmaxf(S[i][0], S[i][1]), fmaxf(S[i][2], S[i][3])));
        top *= cm;
        if (scores) {
            // (k_mass_few forms the weights from the rounded scores: from 2^10 on, where the rounding would show beside
            // l, they are rounded here too)
            if (__any(fabsf(top) > 1024.f && top > -INFINITY)) {
#pragma unroll
                for (uint32_t i = 0; i < NS; i++) S[i] *= cm;
                cm = 1.f;
            }
            if (real)
#pragma unroll
                for (uint32_t i = 0; i < NS; i++) *reinterpret_cast<rf4 *>(scores + 16u * i + 4u * g) = S[i] * cm;
        }
        if (__any(top > m + kLazy)) {
            top = fmaxf(top, lane_xor<16>(top));
            top = fmaxf(top, lane_xor<32>(top));
            const float mn = top > m + kLazy ? top : m, f = mn == -INFINITY ? 1.f : exp2f(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (uint32_t d = 0; d < DT; d++) acc[d] *= f;
        }
        rh8 ph[NH], pl[NH];
        const float ms = m == -INFINITY ? 0.f : m - kLift;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (uint32_t j = 0; j < 8u * NH; j += 2u) {
            const uint32_t i = j >> 2, k = j & 3u, e = j & 7u;
            rf2 p;
            p[0] = __builtin_amdgcn_exp2f(fmaf(S[i][k], cm, -ms));
            p[1] = __builtin_amdgcn_exp2f(fmaf(S[i][k + 1u], cm, -ms));
            sum[0] += p[0];
            sum[1] += p[1];
            const rh2 h = __builtin_convertvector(p, rh2);
            const rf2 r = {less_low(p[0], h), less_high(p[1], h)};
            const rh2 q = __builtin_convertvector(r, rh2);
            ph[j >> 3][e] = h[0], ph[j >> 3][e + 1u] = h[1];
            pl[j >> 3][e] = q[0], pl[j >> 3][e + 1u] = q[1];
        }
        l += sum[0] + sum[1];
#pragma unroll
        for (uint32_t u = 0; u < DT / ND * NH; u++) {
            if (u + 1u < DT / ND * NH) read_v(u + 1u);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (uint32_t d = 0; d < ND; d++)
                acc[u / NH * ND + d] =
                    __builtin_amdgcn_mfma_f32_16x16x32_f16(va[u & 1u][d], ph[u % NH], acc[u / NH * ND + d], 0, 0, 0);
#pragma unroll
            for (uint32_t d = 0; d < ND; d++)
                acc[u / NH * ND + d] =
                    __builtin_amdgcn_mfma_f32_16x16x32_f16(va[u & 1u][d], pl[u % NH], acc[u / NH * ND + d], 0, 0, 0);
        }
    }

    // l over the four lane groups of a row
    __device__ __forceinline__ void sum_l() {
        l += lane_xor<16>(l);
        l += lane_xor<32>(l);
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
        const uint32_t group = a.group, rows = a.n * group;
        const uint32_t i = row_token(a, r);
        const uint64_t at = ((uint64_t)kvh * sp.n + split) * rows + r;
        ml = sp.n > 1u ? pt.ml + at : nullptr;
        acc = sp.n > 1u ? pt.acc + at * part_stride(a.hd)
                        : a.out + (uint64_t)i * a.out_stride + (uint64_t)(kvh * group + r - i * group) * a.hd;
        stats = sp.n == 1u && pt.stats ? pt.stats + (uint64_t)kvh * rows + r : nullptr;
    }
    __device__ __forceinline__ float scale(float l) const { return ml ? 1.f : l == 0.f ? 0.f : __fdiv_rn(1.f, l); }
    // `mark`: l or 1 / l with its sign turned
    __device__ __forceinline__ void put_ml(float m, float l, bool mark = false) const {
        const float sign = mark ? -1.f : 1.f;
        if (ml) *ml = make_float2(m, sign * l);
        if (stats) *stats = make_float2(m, l == 0.f ? 0.f : __fdiv_rn(sign, l));
    }
};
// The row again in f32 products, by a whole wave (row_whole), to the same place.
template <uint32_t HD>
__device__ __forceinline__ void row_again(const RowsArgs &a, const RowsSplit &sp, const RowsPart &pt, uint32_t kvh,
                                          uint32_t split, uint32_t r, uint32_t s0, uint32_t s1, uint32_t lane) {
    const uint32_t group = a.group, i = row_token(a, r);
    float m, l, o[(HD + 63u) / 64u];
    row_whole<HD>(a, i, kvh * group + r - i * group, s0, s1, lane, m, l, o,
                  pt.scores ? pt.scores + ((uint64_t)kvh * a.n * group + r) * score_stride(a.past + a.n) : nullptr);
    const RowsTo to(a, sp, pt, kvh, split, r);
#pragma unroll
    for (uint32_t k = 0; k < (HD + 63u) / 64u; k++)
        if (64u * k + lane < a.hd) to.acc[64u * k + lane] = to.ml ? o[k] : l == 0.f ? 0.f : o[k] / l;
    if (lane == 0) to.put_ml(m, l, m > -INFINITY && fabsf(m) > kMarkScore);
}

// ---- many rows: four waves with rows of their own, slots through two shared buffers ------
template <uint32_t HD>
__global__ __launch_bounds__(256, 2) void k_attn_rows(RowsArgs a, RowsSplit sp, RowsPart pt, bool wide_kv,
                                                 bool wide_q) {
    constexpr uint32_t DT = HD / 16u, T = kTile<HD>, CPR = HD / 8u, NC = T * CPR / 256u;
    constexpr uint32_t RB = HD * 2u, TB = T * RB;  // bytes of a row and of a tile
    __shared__ __align__(1024) uint8_t kv[2][2][TB];  // two buffers of K and V
    __shared__ __align__(16) int32_t dl[2][T];
    const uint32_t t = threadIdx.x, wave = t >> 6, lane = t & 63u, col = lane & 15u, g = lane >> 4;
    const uint32_t kvh = blockIdx.x, split = blockIdx.y, tile = gridDim.z - 1u - blockIdx.z;  // (the longest rows first)
    const uint32_t group = a.group, rows = a.n * group, row_tile = tile * 64u;
    const uint32_t end = row_end(a, row_token(a, min(row_tile + 64u, rows) - 1u));
    const uint32_t s0 = split * sp.len, s1 = min(s0 + sp.len, end);
    if (s0 >= s1) return;  // (the whole workgroup; the merge counts the ranges the same way)
    const uint32_t slots = a.past + a.n, row0 = row_tile + wave * 16u;
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

    DocRange of(a, row_token(a, row_tile), row_token(a, min(row_tile + 64u, rows) - 1u), s0, s1, lane);
    uint32_t p0 = of.next(a, s0, s1, lane);
    RowQ<HD / 32u> x;
    RowTile<HD>::load(a, kvh, row0, wide_q, lane, x);
    if (p0 < s1) fetch(p0, 0u);
    RowTile<HD> R;
    R.init(a, kvh, row0, x, lane, TB);
    if (pt.qparts && split == 0u && row0 < rows) {  // (the mass multiplies them again)
        const uint64_t rt = (uint64_t)kvh * ((rows + 15u) / 16u) + row0 / 16u;
        ru4 *to = pt.qparts + (rt * (HD / 32u) * 64u + lane) * 2u;
#pragma unroll
        for (uint32_t kk = 0; kk < HD / 32u; kk++) {
            to[128u * kk] = __builtin_bit_cast(ru4, R.qh[kk]);
            to[128u * kk + 1u] = __builtin_bit_cast(ru4, R.ql[kk]);
        }
        if (g == 0) pt.qc[rt * 16u + col] = R.c1;
    }
    if (p0 < s1) arrive(0u);
    for (uint32_t b = 0; p0 < s1; b ^= 1u) {
        const uint32_t p1 = of.next(a, p0 + T, s1, lane);
        if (p1 < s1) fetch(p1, b ^ 1u);
        if (p0 < R.last) {
            const bool full = p0 + T <= min(R.clear, s1);
            const uint64_t vis = full ? ~0ull : R.real ? seen_bits(a, R.tok, p0, s1) : 0ull;
            R.template step<T / 32u, true>(a, &kv[0][0][0], p0, vis, full, a.docs ? dl[b] : nullptr, lane);
        }
        if (p1 < s1) arrive(b ^ 1u);
        R.turn(b ? 0u - 2u * TB : 2u * TB);
        p0 = p1;
    }
    if (row0 >= rows) return;

    // ---- the rows' sums
    R.sum_l();
    const bool wide_to = a.hd % 4u == 0 && (a.out_stride % 4u == 0 && ((uintptr_t)a.out & 15u) == 0);
    float nan = R.l * 0.f;
#pragma unroll
    for (uint32_t d = 0; d < DT; d++)
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) nan = fmaf(R.acc[d][k], 0.f, nan);
    const uint64_t bad = __ballot(R.real && (nan != 0.f || far_row(R.m)));  // (0 times anything finite is 0)
    const uint32_t cols = (uint32_t)(bad | bad >> 16 | bad >> 32 | bad >> 48) & 0xFFFFu;
    if (R.real && !(cols >> col & 1u)) {
        const RowsTo to(a, sp, pt, kvh, split, row0 + col);
        const float inv = to.scale(R.l);
#pragma unroll
        for (uint32_t d = 0; d < DT; d++) {
            const uint32_t d0 = 16u * d + 4u * g;
            if (to.ml || wide_to) {  // (the partials' rows are whole float4s)
                if (d0 < a.hd) *reinterpret_cast<rf4 *>(to.acc + d0) = R.acc[d] * inv;
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 4u; k++)
                    if (d0 + k < a.hd) to.acc[d0 + k] = R.acc[d][k] * inv;
            }
        }
        if (g == 0) to.put_ml(R.m - kLift, R.l);
    }
    // rows whose sums are not finite or whose scores are far, one at a time
    for (uint32_t c = 0; cols >> c; c++)
        if (cols >> c & 1u) row_again<HD>(a, sp, pt, kvh, split, row0 + c, s0, s1, lane);
}

// ---- few rows: four waves with the same 16 rows, each with slots of its own ---------------
// A wave takes the 32-slot tiles wave, wave + 4, ... of the range, in an LDS buffer of its own (no barrier
// until the end), then the waves' sums are added in LDS. At most 16 rows a kv head: single tokens and the
// smallest drafts, that read the cache once and compute little. One token over 8192 slots, 64/8 heads of 128,
// capped: 11.7 us under the tracer and the merge's 3.9 (33.6 MB: 6.9 us at the rate of a copy); on the kernel
// above, whose other three waves then have no rows, 13.7.
template <uint32_t HD>
__global__ __launch_bounds__(256, 2) void k_attn_few(RowsArgs a, RowsSplit sp, RowsPart pt, bool wide_q) {
    constexpr uint32_t DT = HD / 16u, T = 32u, CPR = HD / 8u, NC = T * CPR / 64u, RB = HD * 2u, TB = T * RB;
    constexpr uint32_t RS = HD + 4u;  // floats of a row's sums in LDS (the rows of a store in different banks)
    constexpr uint32_t OWN = 2u * TB > 16u * RS * 4u ? 2u * TB : 16u * RS * 4u;
    __shared__ __align__(1024) uint8_t kv[4][OWN];
    __shared__ float2 mls[4][16u];
    __shared__ uint32_t bad[16u];
    const uint32_t t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63u, col = lane & 15u, g = lane >> 4;
    const uint32_t kvh = blockIdx.x, split = blockIdx.y, row0 = 16u * blockIdx.z;
    const uint32_t group = a.group, rows = a.n * group, slots = a.past + a.n;
    const uint32_t end = row_end(a, row_token(a, min(row0 + 16u, rows) - 1u));
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
    const DocRange of(a, row_token(a, row0), row_token(a, min(row0 + 16u, rows) - 1u), s0, s1, lane);
    // (the wave's next tile, past those without a slot of the rows' documents)
    auto next = [&](uint32_t p) {
        if (a.docs)
            while (p < s1) {
                const int32_t d = a.docs[min(p + (lane & 31u), s1 - 1u)];
                if (__any(d >= of.lo && d <= of.hi)) break;
                p += 4u * T;
            }
        return p;
    };
    uint32_t p0 = next(s0 + T * wave);
    RowQ<HD / 32u> x;
    RowTile<HD>::load(a, kvh, row0, wide_q, lane, x);
    if (p0 < s1) fetch(p0);
    RowTile<HD> R;
    R.init(a, kvh, row0, x, lane, TB);
    while (p0 < s1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (p0 < R.last) {
            const bool full = p0 + T <= min(R.clear, s1);
            const uint64_t vis = full ? ~0ull : R.real ? seen_bits(a, R.tok, p0, s1) : 0ull;
            R.template step<1u, false>(a, own, p0, vis, full, a.docs ? a.docs + p0 : nullptr, lane,
                                pt.scores ? pt.scores + ((uint64_t)kvh * rows + row0 + col) * score_stride(slots) + p0 : nullptr);
        }
        p0 = next(p0 + 4u * T);
        if (p0 >= s1) break;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (the tile has been read)
        fetch(p0);
    }
    // ---- the waves' sums: M = max m_w, sum acc_w 2^(m_w - M), in the order of the waves
    R.sum_l();
    float *const sums = reinterpret_cast<float *>(own);
#pragma unroll
    for (uint32_t d = 0; d < DT; d++) *reinterpret_cast<rf4 *>(sums + col * RS + 16u * d + 4u * g) = R.acc[d];
    if (g == 0) mls[wave][col] = make_float2(R.m, R.l);
    if (t < 16u) bad[t] = 0;
    __syncthreads();
    const bool wide_to = a.hd % 4u == 0 && a.out_stride % 4u == 0 && ((uintptr_t)a.out & 15u) == 0;
    for (uint32_t e = t; e < 16u * (HD / 4u); e += 256u) {
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
        if (nan != 0.f || far_row(M)) bad[r] = 1u;
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
    for (uint32_t r = wave; r < 16u; r += 4u)
        if (bad[r]) row_again<HD>(a, sp, pt, kvh, split, row0 + r, s0, s1, lane);
}

// ---- the ranges of a row added up ----------------------------------------------------
// TPR threads per row: M = max m_c, L = sum l_c 2^(m_c - M), out = sum acc_c 2^(m_c - M) / L. Every wave holds the
// weights of the ranges in its lanes; lane groups of a row's float4s take the ranges in turn, eight at a time in
// flight, and the groups are added in order.
constexpr uint32_t kMostRanges = 128;

template <uint32_t TPR>
__global__ __launch_bounds__(256) void k_attn_rows_merge(RowsArgs a, RowsSplit sp, RowsPart pt, uint32_t tile_bits, uint32_t width_bits) {
    __shared__ rf4 part[256];
    const uint32_t t = threadIdx.x, lane = t & 63u, in = t % TPR, kvh = blockIdx.y;
    const uint32_t group = a.group, rows = a.n * group, r = min(blockIdx.x * (256u / TPR) + t / TPR, rows - 1u);
    const uint32_t end = row_end(a, row_token(a, min((r >> tile_bits) + 1u << tile_bits, rows) - 1u)), i = row_token(a, r);
    const uint32_t width = 1u << width_bits, q = in & (width - 1u), grp = in >> width_bits, groups = TPR >> width_bits;
    const uint32_t ps = part_stride(a.hd);
    auto has = [&](uint32_t c) { return c < sp.n && c * sp.len < end; };  // (sp.n ranges pass the last slot by less than one)
    const float2 *ml = pt.ml + (uint64_t)kvh * sp.n * rows + r;
    const float *acc = pt.acc + ((uint64_t)kvh * sp.n * rows + r) * ps + min(4u * q, ps - 4u);
    const bool mine = 4u * q < a.hd;
    rf4 v[8];
    auto load = [&](uint32_t c0) {  // (range 0, which every row has, for one that is not there)
#pragma unroll
        for (uint32_t k = 0; k < 8u; k++) {
            const uint32_t c = c0 + k * groups;
            v[k] = *reinterpret_cast<const rf4 *>(acc + (uint64_t)((has(c) ? c : 0u) * rows) * ps);
        }
    };
    load(grp);
    const float2 y0 = ml[(has(lane) ? lane : 0u) * rows], y1 = ml[(has(lane + 64u) ? lane + 64u : 0u) * rows];
    const float m0 = has(lane) ? y0.x : -INFINITY, m1 = has(lane + 64u) ? y1.x : -INFINITY;
    const float M = wave_max(fmaxf(m0, m1)), ref = M == -INFINITY ? 0.f : M;
    const float w0 = exp2f(m0 - ref), w1 = exp2f(m1 - ref);
    const float L = wave_sum(fmaf(has(lane) ? fabsf(y0.y) : 0.f, w0, (has(lane + 64u) ? fabsf(y1.y) : 0.f) * w1));
    const bool mark = __any((y0.y < 0.f && m0 == M) || (y1.y < 0.f && m1 == M));  // (the range of the maximum decides)
    rf4 o = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t c0 = grp;;) {  // (the same rounds in every lane)
#pragma unroll
        for (uint32_t k = 0; k < 8u; k++) {
            const uint32_t c = c0 + k * groups;
            float f = __shfl(w0, (int)(c & 63u), 64);
            if (TPR > 64u) {  // (a wave per row takes at most 64 ranges)
                const float f1 = __shfl(w1, (int)(c & 63u), 64);
                f = c < 64u ? f : f1;
            }
            const rf4 sum = o + v[k] * f;
            const bool is = has(c);
#pragma unroll
            for (uint32_t x = 0; x < 4u; x++) o[x] = is ? sum[x] : o[x];
        }
        c0 += 8u * groups;
        if (c0 - grp >= sp.n) break;
        load(c0);
    }
    part[t] = o;
    __syncthreads();
    if (grp || !mine || blockIdx.x * (256u / TPR) + t / TPR >= rows) return;
    for (uint32_t k = 1; k < groups; k++) o += part[t + k * width];
    const float inv = L == 0.f ? 0.f : __fdiv_rn(1.f, L);
    float *to = a.out + (uint64_t)i * a.out_stride + (uint64_t)(kvh * group + r - i * group) * a.hd + 4u * q;
#pragma unroll
    for (uint32_t k = 0; k < 4u; k++)
        if (4u * q + k < a.hd) to[k] = L == 0.f ? 0.f : o[k] * inv;
    if (q == 0 && pt.stats) pt.stats[(uint64_t)kvh * rows + r] = make_float2(M, mark ? -inv : inv);
}

// ---- the weights that slots received ---------------------------------------------------
// A workgroup takes 64 (32 for head_dim above 128) slots of a kv head, their K rows as A operands in registers;
// its waves take the row tiles of 16 in turn (S^T as above) and each lane adds up
// 2^(y - m) / l for its slots; the 16 columns, then the waves, are summed at the end
// in a fixed order. A slot whose sum is not finite is taken again in f32 products, and
// marked rows (kMarkScore) and rows whose sum is no number are added in f32 products alone.
// q's parts come from k_attn_rows, as the matrix cores take them: splitting q again for every 64 slots costs more
// than the products (1024 tokens over 5120 slots, 32/8 heads of 128: 269 us under the tracer, 144 from the parts).
// Where slots are few, the rows are split over `parts` workgroups and k_mass_add sums
// what they leave in `part`. At most 16 rows leave their scores on the way instead, and
// k_mass_few adds up their weights without a second product (one token over 2047 slots,
// 32/8 heads of 128: 17.6 -> 13.7 us).
constexpr uint32_t kMassWaves = 8;

template <uint32_t HD>
constexpr uint32_t kMassTiles = HD > 128u ? 2u : 4u;

template <uint32_t HD>
__global__ __launch_bounds__(64 * kMassWaves) void k_mass(RowsArgs a, RowsPart pt, float *__restrict__ part, uint32_t parts,
                                                          bool wide_kv) {
    constexpr uint32_t KK = HD / 32u, NT = kMassTiles<HD>, NP = 16u * NT;  // tiles of 16 slots; slots
    __shared__ float sums[kMassWaves][NP];
    __shared__ uint32_t apart[kMassWaves];  // whether the wave left rows out
    const uint32_t t = threadIdx.x, wave = t >> 6, lane = t & 63u, col = lane & 15u, g = lane >> 4;
    const uint32_t waves = blockDim.x >> 6, kvh = blockIdx.x % a.nkh, rest = blockIdx.x / a.nkh;
    const uint32_t mine = rest % parts, p0 = rest / parts * NP;
    const uint32_t group = a.group, rows = a.n * group, slots = a.past + a.n;
    const uint64_t rstride = (uint64_t)a.nkh * a.hd;
    const float2 *stats = pt.stats + (uint64_t)kvh * rows;
    rh8 ka[NT][KK];
    int32_t ds[NT][4];
#pragma unroll
    for (uint32_t i = 0; i < NT; i++) {
        const uint16_t *k = a.kc + (uint64_t)min(p0 + 16u * i + col, slots - 1u) * rstride + (uint64_t)kvh * a.hd;
#pragma unroll
        for (uint32_t kk = 0; kk < KK; kk++)
            ka[i][kk] = __builtin_bit_cast(rh8, cache8(k, 32u * kk + 8u * g, a.hd, wide_kv));
#pragma unroll
        for (uint32_t r = 0; r < 4u; r++)
            ds[i][r] = a.docs ? a.docs[min(p0 + 16u * i + 4u * g + r, slots - 1u)] : 0;
    }
    float sum[NT][4] = {};
    bool left_out = false;
    const bool terms = a.cap > 0.f || a.slopes;
    int32_t lo = 0, hi = 0;  // the slots' documents
    if (a.docs) {
        const int32_t d = a.docs[min(p0 + lane % NP, slots - 1u)];
        lo = hi = d;
#pragma unroll
        for (int o = 32; o; o >>= 1) lo = min(lo, __shfl_xor(lo, o, 64)), hi = max(hi, __shfl_xor(hi, o, 64));
    }
    // this part's row tiles; those before the first that sees p0 (without a mask or a prefix beyond it) are left out
    const uint32_t all = (rows + 15u) / 16u;
    const uint32_t first = min(a.mask || p0 < a.prefix || p0 <= a.past ? 0u : (p0 - a.past) * group / 16u, all);
    const uint32_t per = (all - first + parts - 1u) / parts, t0 = first + mine * per, t1 = min(t0 + per, all);
    // The wave's tiles are t0 + wave, + waves, ...; 64 of them at a time, a tile to a lane, are looked through for a
    // document of the slots', and the next one's q is on its way while one is worked on.
    ru4 qn[KK][2];
    auto fetch = [&](uint32_t rt) {
        const ru4 *from = pt.qparts + (((uint64_t)kvh * all + rt) * KK * 64u + lane) * 2u;
#pragma unroll
        for (uint32_t kk = 0; kk < KK; kk++) qn[kk][0] = from[128u * kk], qn[kk][1] = from[128u * kk + 1u];
    };
    for (uint32_t base = t0 + wave; base < t1; base += 64u * waves) {
        const uint32_t lt = base + lane * waves;
        bool need = lt < t1;
        if (a.docs && need) {
            need = false;
            for (uint32_t i = row_token(a, 16u * lt); i <= row_token(a, min(16u * lt + 16u, rows) - 1u); i++) {
                const int32_t d = a.docs[a.past + i];
                need = need || (d >= lo && d <= hi);
            }
        }
        uint64_t left = __ballot(need);
        if (left) fetch(base + (uint32_t)__builtin_ctzll(left) * waves);
        while (left) {
            const uint32_t rt = base + (uint32_t)__builtin_ctzll(left) * waves;
            left &= left - 1ull;
            const uint32_t r = 16u * rt + col;
            const bool real = r < rows;
            const uint32_t i = real ? row_token(a, r) : 0u, h = kvh * group + (real ? r - i * group : 0u);
            const float2 st = real ? stats[r] : make_float2(0.f, 0.f);
            const float c1 = pt.qc[((uint64_t)kvh * all + rt) * 16u + col];
            rh8 qh[KK], ql[KK];
#pragma unroll
            for (uint32_t kk = 0; kk < KK; kk++)
                qh[kk] = __builtin_bit_cast(rh8, qn[kk][0]), ql[kk] = __builtin_bit_cast(rh8, qn[kk][1]);
            if (left) fetch(base + (uint32_t)__builtin_ctzll(left) * waves);
            const bool full = !a.docs && 16u * rt + 16u <= rows &&
                              p0 + NP <= (a.mask ? a.past : row_end(a, row_token(a, 16u * rt)));
            const uint64_t vis = full ? ~0ull : real ? seen_bits(a, i, p0, slots) : 0ull;
            const int32_t doc = a.docs ? a.docs[a.past + i] : 0;
            // (a row that is left out: weights 2^-inf times 0)
            const bool out = !(st.y >= 0.f);
            left_out = left_out || out;
            const float slope = a.slopes ? a.slopes[h] : 0.f, ms = out ? INFINITY : st.x == -INFINITY ? 0.f : st.x;
            const float inv = out ? 0.f : st.y;
            rf4 S[NT];
#pragma unroll
            for (uint32_t j = 0; j < NT; j++) S[j] = rf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (uint32_t kk = 0; kk < KK; kk++)
#pragma unroll
                for (uint32_t v = 0; v < 2u; v++)
#pragma unroll
                    for (uint32_t j = 0; j < NT; j++)
                        S[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[j][kk], v ? ql[kk] : qh[kk], S[j], 0, 0, 0);
            float cm = c1 * kLog2e;
            if (terms) {
#pragma unroll
                for (uint32_t j = 0; j < NT; j++)
#pragma unroll
                    for (uint32_t k = 0; k < 4u; k++)
                        S[j][k] = parts_score(a, S[j][k], c1, slope, a.past + i, p0 + 16u * j + 4u * g + k);
                cm = score_unit(a) * kLog2e;
            }
#pragma unroll
            for (uint32_t j = 0; j < NT; j++)
#pragma unroll
                for (uint32_t k = 0; k < 4u; k++) {
                    const uint32_t o = 16u * j + 4u * g + k;
                    float y = fmaf(S[j][k], cm, -ms);
                    if (!full) y = (vis >> o & 1ull) & (ds[j][k] == doc) ? y : -INFINITY;  // (0 == 0 without documents)
                    sum[j][k] = fmaf(__builtin_amdgcn_exp2f(y), inv, sum[j][k]);
                }
        }
    }
    // the 16 columns: each lane group's row of 16 lanes
#pragma unroll
    for (uint32_t j = 0; j < NT; j++)
#pragma unroll
        for (uint32_t k = 0; k < 4u; k++) {
            float v = sum[j][k];
            v += bfly_partner<8>(v, lane);
            v += bfly_partner<4>(v, lane);
            v += bfly_partner<2>(v, lane);
            v += bfly_partner<1>(v, lane);
            if (col == 0) sums[wave][16u * j + 4u * g + k] = v;
        }
    const uint32_t any_left_out = __any(left_out);
    if (lane == 0) apart[wave] = any_left_out;
    __syncthreads();
    if (wave) return;
    const uint32_t j = p0 + lane;
    const bool in = lane < NP && j < slots;
    float v = 0.f;
    uint32_t some = 0;
    for (uint32_t w = 0; w < waves; w++) v += sums[w][lane % NP], some |= apart[w];
    const uint64_t bad = __ballot(in && v * 0.f != 0.f);
    const uint64_t again = some ? __ballot(in) : bad;
    for (uint32_t c = 0; c < 64u && again >> c; c++) {
        if (!(again >> c & 1ull)) continue;
        const bool every = bad >> c & 1ull;  // (else the rows that were left out)
        const uint32_t jj = p0 + c;
        const uint16_t *k = a.kc + (uint64_t)jj * rstride + (uint64_t)kvh * a.hd;
        float whole = 0.f;
        for (uint32_t r = 16u * t0 + lane; r < min(16u * t1, rows); r += 64u) {
            const float2 st = stats[r];
            if (!every && st.y >= 0.f) continue;
            const uint32_t i = row_token(a, r), h = kvh * group + r - i * group;
            if (jj >= row_end(a, i) || !row_sees(a, i, jj)) continue;
            const float s = row_score(a, row_dot(a.q + (uint64_t)i * a.q_stride + (uint64_t)h * a.hd, k, a.hd) * a.scale,
                                      a.slopes ? a.slopes[h] : 0.f, a.past + i, jj);
            // (the product rounded, as row_whole's)
            whole += exp2f(__fsub_rn(__fmul_rn(s, kLog2e), st.x == -INFINITY ? 0.f : st.x)) * fabsf(st.y);
        }
        whole = wave_sum(whole);
        if (lane == c) v = every ? whole : v + whole;
    }
    if (!in) return;
    if (parts > 1u)
        part[((uint64_t)mine * a.nkh + kvh) * slots + j] = v;
    else
        a.mass[(uint64_t)kvh * a.max_ctx + j] += v;
}

// Few rows: their scores are there (k_attn_few), a thread takes a slot.
__global__ __launch_bounds__(256) void k_mass_few(RowsArgs a, RowsPart pt) {
    const uint32_t j = blockIdx.x * 256u + threadIdx.x, kvh = blockIdx.y, slots = a.past + a.n, group = a.group;
    if (j >= slots) return;
    const float *y = pt.scores + (uint64_t)kvh * a.n * group * score_stride(slots) + j;
    const float2 *stats = pt.stats + (uint64_t)kvh * a.n * group;
    float v = 0.f;
    for (uint32_t i = 0; i < a.n; i++) {
        if (j >= row_end(a, i) || !row_sees(a, i, j)) continue;  // (its scores may not have been written)
        for (uint32_t r = i * group; r < (i + 1u) * group; r++) {
            const float2 st = stats[r];
            v = fmaf(__builtin_amdgcn_exp2f(y[r * score_stride(slots)] - (st.x == -INFINITY ? 0.f : st.x)), fabsf(st.y), v);
        }
    }
    a.mass[(uint64_t)kvh * a.max_ctx + j] += v;
}

__global__ __launch_bounds__(256) void k_mass_add(RowsArgs a, const float *__restrict__ part, uint32_t parts) {
    const uint32_t j = blockIdx.x * 256u + threadIdx.x, kvh = blockIdx.y, slots = a.past + a.n;
    if (j >= slots) return;
    float v = 0.f;
    for (uint32_t c = 0; c < parts; c += 8u) {
        float x[8];
#pragma unroll
        for (uint32_t k = 0; k < 8u; k++) x[k] = c + k < parts ? part[((uint64_t)(c + k) * a.nkh + kvh) * slots + j] : 0.f;
#pragma unroll
        for (uint32_t k = 0; k < 8u; k++) v += x[k];
    }
    a.mass[(uint64_t)kvh * a.max_ctx + j] += v;
}


// ---- launches -------------------------------------------------------------------------------

struct RowsPlan {
    uint32_t hd, tiles;  // template head size, row tiles a kv head
    bool few;
    RowsSplit sp;
    uint32_t parts;               // of the rows, for the mass
    size_t ml, acc, stats, mass, qparts, qc;  // bytes (mass: the scores of few rows, or the parts' sums)
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
    const uint32_t rows = a.n * a.group, slots = a.past + a.n;
    // (up to 64 rows the two kernels are within 15% of each other either way, the few-row one ahead over short
    // contexts: 32 rows over 500 slots 10.9 and 12.5 us, over 2048 13.8 and 12.2)
    p.few = rows <= 16u && rows_wide_kv(a);
    const uint32_t tile_rows = p.few ? 16u : 64u;
    p.tiles = (rows + tile_rows - 1u) / tile_rows;
    // Ranges: until about 512 workgroups, two a CU, share the work (64 tokens over 8255 slots, 64/8 heads of 128: 47 us;
    // until 256 59, until 768 54). A range is at least a tile a wave (few) or two tiles of a
    // workgroup (16 tokens over 2048 slots, 32/8 heads of 128: 11.5 us, one tile 14.5), and, where half the CUs have a
    // workgroup already, so many slots that sharing their products is worth the merge: 1024 at heads of 64 (777 tokens
    // in documents, 16 heads: 22 us whole, 22 and the merge's 10 in two ranges), 512 at 128 (2010 tokens, 4 heads, in
    // documents: 52 us in ranges of 1024, 40 in ranges of 512), 256 at 256 (1024 tokens over 2048 slots, 8/1 heads: 95
    // and 66; 130 tokens over 536 slots, 64/8 heads: 46 whole, 45 in two).
    const uint32_t wgs = p.tiles * a.nkh;
    const uint32_t least = p.few || wgs < 128u ? 128u : p.hd <= 64u ? 1024u : 65536u / p.hd / 128u * 128u;
    const uint32_t most = (slots + least - 1u) / least;
    uint32_t n = 512u / wgs;
    n = n < most ? n : most;
    n = n < 1u ? 1u : n < kMostRanges ? n : kMostRanges;  // (what the merge adds up)
    p.sp.len = ((slots + n - 1u) / n + 127u) / 128u * 128u;
    p.sp.n = (slots + p.sp.len - 1u) / p.sp.len;
    const size_t all = (size_t)rows * a.nkh;
    const auto round = [](size_t b) { return (b + 255u) & ~(size_t)255u; };
    if (p.sp.n > 1u) {
        p.ml = round(all * p.sp.n * sizeof(float2));
        p.acc = round(all * p.sp.n * part_stride(a.hd) * sizeof(float));
    }
    if (a.mass) {
        p.stats = round(all * sizeof(float2));
        if (p.few) {
            p.mass = round(all * score_stride(slots) * sizeof(float));
            return p;
        }
        // about 256 workgroups of eight waves, at least a row tile a wave (2560 rows over 643 slots, 2 kv heads of 80:
        // 12.1 us under the tracer; 512 workgroups 15.0, 128 16.4)
        const uint32_t np = p.hd > 128u ? 32u : 64u, blocks = (slots + np - 1u) / np * a.nkh, waves = (rows + 127u) / 128u;
        p.parts = blocks >= 256u ? 1u : 256u / blocks;
        p.parts = p.parts < waves ? p.parts : waves;
        if (p.parts > 1u) p.mass = round((size_t)p.parts * a.nkh * slots * sizeof(float));
        const size_t tiles = (size_t)((rows + 15u) / 16u) * a.nkh;
        p.qparts = round(tiles * p.hd * 64u);
        p.qc = round(tiles * 16u * sizeof(float));
    }
    return p;
}

size_t attn_rows_scratch_bytes(const RowsArgs &a) {
    const RowsPlan p = rows_plan(a);
    return p.ml + p.acc + p.stats + p.mass + p.qparts + p.qc;
}

template <uint32_t HD>
static void start_rows(const RowsArgs &a, const RowsPlan &p, const RowsPart &pt, hipStream_t s) {
    const bool wide_kv = rows_wide_kv(a), wide_q = rows_wide_q(a);
    const dim3 grid(a.nkh, p.sp.n, p.tiles);
    if (p.few) {
        k_attn_few<HD><<<grid, 256, 0, s>>>(a, p.sp, pt, wide_q);
        return;
    }
    k_attn_rows<HD><<<grid, 256, 0, s>>>(a, p.sp, pt, wide_kv, wide_q);
}

template <uint32_t HD>
static void start_mass(const RowsArgs &a, const RowsPlan &p, const RowsPart &pt, float *part, hipStream_t s) {
    const uint32_t tiles = (a.n * a.group + 15u) / 16u, np = 16u * kMassTiles<HD>;
    k_mass<HD><<<(a.past + a.n + np - 1u) / np * a.nkh * p.parts, 64u * (tiles < kMassWaves ? tiles : kMassWaves), 0, s>>>(
        a, pt, part, p.parts, rows_wide_kv(a));
}

hipError_t launch_attn_rows(const RowsArgs &a, void *scratch, hipStream_t s) {
    const RowsPlan p = rows_plan(a);
    uint8_t *at = static_cast<uint8_t *>(scratch);
    RowsPart pt{};
    if (p.sp.n > 1u) pt.ml = reinterpret_cast<float2 *>(at), pt.acc = reinterpret_cast<float *>(at + p.ml);
    if (a.mass) pt.stats = reinterpret_cast<float2 *>(at + p.ml + p.acc);
    float *const mass = reinterpret_cast<float *>(at + p.ml + p.acc + p.stats);
    if (a.mass && p.few) pt.scores = mass;
    if (a.mass && !p.few) {
        pt.qparts = reinterpret_cast<ru4 *>(at + p.ml + p.acc + p.stats + p.mass);
        pt.qc = reinterpret_cast<float *>(at + p.ml + p.acc + p.stats + p.mass + p.qparts);
    }
    switch (p.hd) {
        case 32: start_rows<32>(a, p, pt, s); break;
        case 64: start_rows<64>(a, p, pt, s); break;
        case 96: start_rows<96>(a, p, pt, s); break;
        case 128: start_rows<128>(a, p, pt, s); break;
        default: start_rows<256>(a, p, pt, s); break;
    }
    hipError_t e = hipGetLastError();
    const uint32_t rows = a.n * a.group;
    if (e == hipSuccess && p.sp.n > 1u) {
        const uint32_t tile_bits = p.few ? 4u : 6u;
        const uint32_t width_bits = a.hd <= 32u ? 3u : a.hd <= 64u ? 4u : a.hd <= 128u ? 5u : 6u;  // float4s of a row
        // a wave per row where its lanes hold every range in one round of loads
        if (p.sp.n <= 8u * (64u >> width_bits))
            k_attn_rows_merge<64><<<dim3((rows + 3u) / 4u, a.nkh), 256, 0, s>>>(a, p.sp, pt, tile_bits, width_bits);
        else
            k_attn_rows_merge<256><<<dim3(rows, a.nkh), 256, 0, s>>>(a, p.sp, pt, tile_bits, width_bits);
        e = hipGetLastError();
    }
    if (e == hipSuccess && a.mass && p.few) {
        k_mass_few<<<dim3((a.past + a.n + 255u) / 256u, a.nkh), 256, 0, s>>>(a, pt);
        e = hipGetLastError();
    } else if (e == hipSuccess && a.mass) {
        switch (p.hd) {
            case 32: start_mass<32>(a, p, pt, mass, s); break;
            case 64: start_mass<64>(a, p, pt, mass, s); break;
            case 96: start_mass<96>(a, p, pt, mass, s); break;
            case 128: start_mass<128>(a, p, pt, mass, s); break;
            default: start_mass<256>(a, p, pt, mass, s); break;
        }
        e = hipGetLastError();
        if (e == hipSuccess && p.parts > 1u)
            k_mass_add<<<dim3((a.past + a.n + 255u) / 256u, a.nkh), 256, 0, s>>>(a, mass, p.parts);
        if (e == hipSuccess) e = hipGetLastError();
    }
    return e;
}

}  // namespace vbs
