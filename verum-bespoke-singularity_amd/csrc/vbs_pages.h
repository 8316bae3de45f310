// vbs_pages.h — the paged KV cache: its layout, and the launchers of the operators
// over it (rows into and out of pages, the attention of single tokens, the
// verification of drafted tokens), shared between the runtime (vbs_gfx950_rt.hip)
// and their kernels. As in vbs_internal.h, every launcher enqueues on `s`; the
// C-ABI entry points have checked the arguments.
//
// A page holds page_slots (32 to 1024, a power of two) of every kv head in units
// of 32 slots of one head: [kv head][unit]. Within a unit the elements lie in the
// order in which the attention's matrix instructions take them, so that every load
// of a wave is 1 KB of consecutive bytes that lands in the registers of an operand,
// without LDS and without exchange between lanes (v_mfma_f32_16x16x32_f16: lane
// 16 g + r holds row r, elements 8 g .. 8 g + 7 of the products' 32):
//   K (rows: slots; products over the elements of a block of 32): two 16-row tiles
//     t with row 4 h + j the slot 8 h + 4 t + j, whose scores then lie, lane by lane,
//     as the weights' operand of the second product wants them;
//   V (rows: elements; products over the 32 slots): slot 8 g + e.
// F16:  K [t 2][b nb][g 4][r 16][e 8], V [b nb][t 2][g 4][r 16][e 8] halves
// Q8_0: K and V int8 [b nb][g 4][r 16][t 2][8], then f16 scales [b nb][slot 32]
// nb = ceil(head_dim / 32); elements behind head_dim are stored as zeros.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace vbs {

constexpr uint32_t kUnit = 32;  // slots of a unit, and elements of a block

struct PageArgs {
    uint8_t *k, *v;  // at the layer's first page
    int q8;
    uint32_t n_pages, shift;  // a page holds 1 << shift units
    uint32_t nkh, hd, nb;
    uint32_t unit_bytes;
    uint64_t page_bytes;
    const int32_t *table;  // [n_seqs][per_seq]
    uint32_t n_seqs, per_seq;
};

inline uint32_t page_unit_bytes(bool q8, uint32_t hd) { return ((hd + kUnit - 1u) / kUnit) * (q8 ? 1088u : 2048u); }

#ifdef __HIPCC__
// The page of unit u of sequence `seq`, or -1 where the table has none for it.
__device__ __forceinline__ int32_t page_at(const PageArgs &a, int32_t seq, uint32_t u) {
    const uint32_t i = u >> a.shift;
    if ((uint32_t)seq >= a.n_seqs || i >= a.per_seq) return -1;
    const int32_t p = a.table[(uint64_t)(uint32_t)seq * a.per_seq + i];
    return (uint32_t)p < a.n_pages ? p : -1;
}
// Where unit u (of a sequence) of kv head h begins in a pool, given its page.
__device__ __forceinline__ uint64_t unit_offset(const PageArgs &a, int32_t page, uint32_t u, uint32_t h) {
    return (uint64_t)(uint32_t)page * a.page_bytes +
           (uint64_t)((h << a.shift) + (u & ((1u << a.shift) - 1u))) * a.unit_bytes;
}
// The places (in elements) of a slot's element d within a unit.
template <bool Q8>
__device__ __forceinline__ uint32_t k_place(uint32_t nb, uint32_t slot, uint32_t d) {
    const uint32_t lane = (d & 24u) * 2u + (slot >> 3) * 4u + (slot & 3u), t = (slot >> 2) & 1u, b = d >> 5;
    return Q8 ? (((b * 64u + lane) * 2u + t) << 3) + (d & 7u) : (((t * nb + b) * 64u + lane) << 3) + (d & 7u);
}
template <bool Q8>
__device__ __forceinline__ uint32_t v_place(uint32_t slot, uint32_t d) {
    const uint32_t lane = (slot >> 3) * 16u + (d & 15u), t = (d >> 4) & 1u, b = d >> 5;
    return Q8 ? (((b * 64u + lane) * 2u + t) << 3) + (slot & 7u) : (((b * 2u + t) * 64u + lane) << 3) + (slot & 7u);
}
#endif

struct PageRowsArgs {
    PageArgs p;
    const int32_t *seq, *at;  // seq NULL: token i is of sequence i
    uint32_t n;
    const float *k, *v;  // rows to store
    void *out_k, *out_v;  // rows to fill
    int out_f16;
    int vec;  // eight elements of a row can be read or written 16 bytes at a time
    uint32_t stride;
};
hipError_t launch_page_store(PageRowsArgs a, hipStream_t s);
hipError_t launch_page_load(PageRowsArgs a, hipStream_t s);

struct PagedAttnArgs {
    PageArgs p;
    const float *q;
    uint32_t q_stride;
    float *out;
    uint32_t out_stride;
    const int32_t *seq, *lens;
    uint32_t rows, max_len, nqh, group;
    float scale;
    int q_vec;  // q's rows can be read 16 bytes at a time, eight elements of a head together
    uint32_t workgroups;  // that share all rows' units; 0: one for each row and head
    uint32_t grid;        // of the launch: some more where shares may end with their head (`aligned`)
    int aligned;
    uint32_t tile;  // q heads of a kv head that are taken together, 8 or 16
    uint4 *joins;   // [grid]: row and head (tile) that begin in the share and go on, and their pieces (0: none)
    float2 *ml;     // [grid][2][tile]: maximum (log2) and sum of partial results
    float *part;    // [grid][2][tile][hd]
};
// Sets workgroups, grid, aligned and tile; the bytes of joins, ml and part together (0: none needed).
size_t plan_attn_paged(PagedAttnArgs &a);
hipError_t launch_attn_paged(PagedAttnArgs a, void *scratch, hipStream_t s);

constexpr uint32_t kMaxDraft = 64;  // drafted tokens of a sequence

struct VerifyArgs {
    const float *logits, *draft;  // draft NULL: drafted tokens were certain
    uint32_t stride, draft_stride;
    const int32_t *drafted;
    const float *u;
    uint32_t batch, n, vocab;
    float temp;
    int32_t *accepted, *tokens;
    double rate;      // 32 log2 e / T
    uint32_t chunks, small;  // of a row, and of what is left of one
    double *sums;   // [batch][2 n + 1][chunks]: target rows, then draft rows
    float *tops;    // the same, the maxima
    int32_t *arg;   // the same, their places (temperature 0)
    double *left;   // [batch][2][small]: what is left to draw from, and the target alone
    double *stats;  // [batch][4]: maximum and reciprocal sum of the row to draw from, of the target and of the draft
    int32_t *stop;  // [batch]: the row drawn from | refused << 16
};
size_t plan_verify(VerifyArgs &a);
hipError_t launch_verify(VerifyArgs a, void *scratch, hipStream_t s);

}  // namespace vbs
