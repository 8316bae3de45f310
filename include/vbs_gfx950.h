/* vbs_gfx950.h — C ABI of libvbs_gfx950.so, the MI355X (gfx950) device
 * library behind Verum's HIP backend slot.
 *
 * The reference's HIP backend (src/vbs_backend_hip.c) dlopens the ROCm
 * runtime and host-stages every op through src/vbs_host_math.h. This library
 * replaces that: it owns one device, one in-order HIP stream and the
 * hand-written gfx950 kernels, and exposes them through plain pointers and
 * sizes (no HIP or torch types). The C11 shim
 * (host/vbs_backend_gfx950.c) dlopens it, checks vbs_gfx950_abi_version()
 * and every symbol below, and maps the vbs_backend_ops_t slots onto it.
 *
 * Conventions
 *   - Every function returns 1 on success and 0 on failure; the reason is
 *     then in vbs_gfx950_last_error(). Nothing aborts or throws.
 *   - Device pointers come from vbs_gfx950_alloc (or point inside such an
 *     allocation). All work is enqueued on the library's single stream in
 *     call order; copies to the host wait for it, so results are visible to
 *     the caller exactly as with the reference's synchronous backends.
 *   - `type` values are GGUF type ids (vbs_ggml_type_t): F32 0, F16 1,
 *     Q4_0 2, Q4_1 3, Q8_0 8, Q4_K 12, Q6_K 14, LNS8 40.
 */
#ifndef VBS_GFX950_H
#define VBS_GFX950_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define VBS_GFX950_ABI_VERSION 3

/* ---- library / device ------------------------------------------------ */

/* ABI version of the loaded library; the shim refuses a mismatch, as
 * vbs_hot_load does for the CPU hot table (src/vbs_hotpath.c:96-101). */
int vbs_gfx950_abi_version(void);

/* Probe and open the first gfx950 device. Idempotent; a failure is sticky and
 * explained by vbs_gfx950_last_error(). Replaces hip_init
 * (src/vbs_backend_hip.c:149-225). */
int vbs_gfx950_init(void);

/* Last failure reason ("ok" when none). Replaces vbs_hip_last_error
 * (src/vbs_backend_hip.c:110). */
const char *vbs_gfx950_last_error(void);

/* Number of usable devices (0 or 1: the backend drives one GPU). Replaces
 * hip_get_device_count (src/vbs_backend_hip.c:227). */
int vbs_gfx950_device_count(void);

/* Name, total and free HBM of device `index`. Fills what the reference's HIP
 * backend left unset (max_working_set_bytes / max_buffer_bytes,
 * src/vbs_backend_hip.c:214-220). */
int vbs_gfx950_device_info(int index, char *name, size_t name_cap, uint64_t *total_bytes,
                           uint64_t *free_bytes);

/* ---- memory (src/vbs_backend_hip.c:230-264) ---------------------------- */

void *vbs_gfx950_alloc(size_t bytes);          /* device memory, 256-B aligned */
int vbs_gfx950_free(void *dptr);
void *vbs_gfx950_host_alloc(size_t bytes);     /* pinned host memory */
int vbs_gfx950_host_free(void *hptr);
/* Stream-ordered copies that have completed when they return. */
int vbs_gfx950_copy_h2d(void *dst, const void *src, size_t bytes);
int vbs_gfx950_copy_d2h(void *dst, const void *src, size_t bytes);
int vbs_gfx950_copy_d2d(void *dst, const void *src, size_t bytes);
/* Wait for all enqueued work (src/vbs_backend_hip.c:548-551). */
int vbs_gfx950_synchronize(void);

/* ---- hot-path kernels --------------------------------------------------- */

/* 1 if `type` has a gfx950 linear kernel: F32, F16, Q4_0, Q4_1, Q8_0, Q4_K,
 * Q6_K, and LNS8 (the bridge's seventh dispatch type). Mirrors the reference's refusal contract (vbs_host_type_supported,
 * src/vbs_host_math.h:69-89, and the Q8_K refusal checked by
 * src/vbs_backend_test.c:952-955). */
int vbs_gfx950_linear_supported(int type);

/* y[row_off + r] (+)= sum_c deq(W[r, c]) * x[col_off + c] for r < rows,
 * W row-major in native GGUF blocks, row stride = (cols / block) * bytes.
 * Replaces hip_dispatch_linear_tile (src/vbs_backend_hip.c:346-394); same
 * meaning as vbs_host_linear_tile (src/vbs_host_math.h:223-267) with fp32
 * accumulation. */
int vbs_gfx950_linear(int type, const void *w, const float *x, float *y, uint32_t cols,
                      uint32_t rows, uint32_t col_off, uint32_t row_off, int accumulate);

/* out[0..dim) = deq(row `token` of table w), bit-identical to
 * vbs_host_embed_row (src/vbs_host_math.h:136-142). The EMBEDDING op of
 * src/vbs_backend_hip.c:405-423. */
int vbs_gfx950_embed(int type, const void *w, uint32_t token, float *out, uint32_t dim);

/* rms_norm (src/vbs_host_math.h:28-36; NORMALIZE, src/vbs_backend_hip.c:424-439). */
int vbs_gfx950_rms_norm(const float *in, const float *w, float *out, uint32_t dim, float eps);

/* In-place RoPE on n_heads x head_dim (src/vbs_host_math.h:38-51; ROTARY,
 * src/vbs_backend_hip.c:440-454). head_dim <= 512. */
int vbs_gfx950_rope(float *x, uint32_t pos, uint32_t head_dim, uint32_t n_heads, float theta);

/* f16 KV store at ((layer*max_ctx + pos)*kv_dim + i) with the reference
 * rounding (src/vbs_host_math.h:150-159; CACHE, src/vbs_backend_hip.c:455-481). */
int vbs_gfx950_cache_store(const float *k, const float *v, uint16_t *kc, uint16_t *vc,
                           uint32_t pos, uint32_t layer, uint32_t max_ctx, uint32_t kv_dim);

/* Single-query GQA attention over the f16 cache (src/vbs_host_math.h:170-209;
 * ATTENTION, src/vbs_backend_hip.c:482-512). */
int vbs_gfx950_attention(const float *q, const uint16_t *kc, const uint16_t *vc, float *out,
                         uint32_t seq_len, uint32_t layer, uint32_t max_ctx,
                         uint32_t n_q_heads, uint32_t n_kv_heads, uint32_t head_dim,
                         float scale);

/* vbs_gfx950_attention without any device allocation: no counterpart in the
 * reference. For callers that cannot allocate (code under HIP graph capture,
 * tight serving loops, harnesses that forbid hipMalloc). Same arguments and
 * result as vbs_gfx950_attention; the per-chunk partial results live in a
 * fixed 8 MiB device array of the library instead of the growable scratch, so
 * calls whose partials exceed it (nqh x max(ceil(640 / nkh), ceil(seq_len /
 * 64)) x (head_dim + 2) x 4 bytes, 640 being the workgroup target of the
 * sequence split, kMfmaTargetWgs in csrc/vbs_attn_common.h; e.g. 70B shapes
 * up to seq_len 16128) fail with a reason and launch nothing. Every call on the device shares that
 * array: calls that overlap on the device race (the library's own calls are
 * ordered on its one stream and never overlap). */
int vbs_gfx950_attention_noalloc(const float *q, const uint16_t *kc, const uint16_t *vc,
                                 float *out, uint32_t seq_len, uint32_t layer, uint32_t max_ctx,
                                 uint32_t n_q_heads, uint32_t n_kv_heads, uint32_t head_dim,
                                 float scale);

/* out = gate / (1 + expf(-gate)) * up (src/vbs_host_math.h:53-57; ACTIVATION). */
int vbs_gfx950_silu_mul(const float *gate, const float *up, float *out, uint32_t n);

/* out = a + b, out may alias a (src/vbs_host_math.h:59-62; ELEMENTWISE). */
int vbs_gfx950_add(const float *a, const float *b, float *out, uint32_t n);

/* ---- extensions (no slot in vbs_backend_ops_t) -------------------------- */

/* Dequantise rows of a packed tensor: out[i*dim .. +dim) = deq(row ids[i])
 * (ids == NULL means rows 0..n_rows-1). `ids` is a device array. The batched
 * form of the one-token-per-dispatch EMBEDDING op, and the bit-exactness
 * probe of every block decoder. */
int vbs_gfx950_dequant_rows(int type, const void *w, const uint32_t *ids, uint32_t n_rows,
                            uint32_t dim, float *out);

/* The neighbours of a linear matvec that vbs_gfx950_linear_fused takes into
 * the same launch; NULL / 0 fields are absent. */
typedef struct vbs_gfx950_linear_join {
    const float *norm_w;   /* NORMALIZE before: x_normed = rms_norm(x, norm_w, norm_eps) */
    float norm_eps;
    float *x_normed;
    float *acc;            /* ELEMENTWISE after: acc = acc + y */
    int rope;              /* ROTARY after: y rotated at pos in heads of head_dim, base theta */
    uint32_t pos, head_dim;
    float theta;
    const float *gate;     /* ACTIVATION after: hidden = silu(gate) * y */
    float *hidden;
    const float *k_row;    /* CACHE after: kc[kv_off + i] = f16(k_row[i]), vc[kv_off + i] = f16(y[i]) */
    uint16_t *kc, *vc;
    uint64_t kv_off;       /* (layer * max_ctx + pos) * kv_dim */
} vbs_gfx950_linear_join_t;

/* The linear matvec y = W x fused with its neighbours in the bridge's op
 * sequence, for the backend shim's per-dispatch path (no counterpart in the
 * reference: the shim holds back one op and joins it with the next when they
 * fit one of these kernels; results are bit-identical to the ops one by one,
 * and y is always written):
 *   - norm_w and x_normed: the NORMALIZE before it (src/vbs_host_math.h:28-36),
 *     x_normed stored as that op would, then y = W x_normed; alone or with rope;
 *   - acc: the ELEMENTWISE add after it (src/vbs_host_math.h:59-62);
 *   - rope: the ROTARY after it (src/vbs_host_math.h:38-51);
 *   - gate and hidden: the ACTIVATION after the up matvec
 *     (src/vbs_host_math.h:53-57);
 *   - k_row, kc, vc: the CACHE after the V matvec, with the reference's f16
 *     rounding (src/vbs_host_math.h:150-159).
 * At most one of acc / rope / gate / k_row. Q4_K and Q6_K rows of a multiple
 * of 256; returns 1 when launched, 0 with a reason on an error, and 2
 * (nothing launched) when no fused kernel takes this combination or shape.
 * The RoPE rows live in a device table the library builds for (theta,
 * head_dim) and regrows for later positions (it allocates; not for graph
 * capture). */
int vbs_gfx950_linear_fused(int type, const void *w, const float *x, float *y, uint32_t cols,
                            uint32_t rows, const vbs_gfx950_linear_join_t *join);

/* Grouped ops of the backend shim's per-dispatch path (no counterpart in the
 * reference: the shim holds back the bridge's attention-input and FFN-input
 * runs and issues each as one launch; results are bit-identical to the ops
 * one by one, and every buffer those ops write is written):
 *
 * vbs_gfx950_qkv_fused -- NORMALIZE (when norm_w and x_normed are given),
 * LINEAR q, ROTARY q, LINEAR k, ROTARY k, LINEAR v, CACHE
 * (src/vbs_specializer.c:282-302): x_normed = rms_norm(x), q = rope(Wq xn),
 * k = rope(Wk xn), v = Wv xn, and f16(k), f16(v) stored at
 * ((layer * max_ctx + pos) * kv_rows + i) of kc / vc, the rotations at pos
 * in heads of head_dim with base theta. The three matrices share the type. */
int vbs_gfx950_qkv_fused(int type, const void *wq, const void *wk, const void *wv, const float *x,
                         uint32_t cols, uint32_t q_rows, uint32_t kv_rows, const float *norm_w,
                         float eps, float *x_normed, float *q, float *k, float *v, uint32_t pos,
                         uint32_t head_dim, float theta, uint16_t *kc, uint16_t *vc,
                         uint32_t layer, uint32_t max_ctx);

/* vbs_gfx950_gate_up_fused -- NORMALIZE (optional, as above), LINEAR gate,
 * LINEAR up, ACTIVATION (src/vbs_specializer.c:282-284, 319-329): gate = Wg xn,
 * up = Wu xn, hidden = silu(gate) * up.
 *
 * Both: Q4_K and Q6_K rows of a multiple of 256, row counts of a multiple
 * of 16; 1 when launched, 0 with a reason on an error, 2 (nothing launched)
 * when no grouped kernel takes the shape. The RoPE rows come from the same
 * device table as vbs_gfx950_linear_fused's (it allocates; not for graph
 * capture). */
int vbs_gfx950_gate_up_fused(int type, const void *wg, const void *wu, const float *x,
                             uint32_t cols, uint32_t rows, const float *norm_w, float eps,
                             float *x_normed, float *gate, float *up, float *hidden);

/* Batched decode: Y[b*y_stride + r] = sum_c deq(W[r,c]) * X[b*x_stride + c]
 * for b < batch (<= 16). Equal to `batch` calls of vbs_gfx950_linear; the
 * weights are read once. The reference has no batched matvec
 * (src/vbs_specializer.c:353-357 loops tokens one by one). */
int vbs_gfx950_linear_batch(int type, const void *w, const float *x, uint32_t x_stride,
                            float *y, uint32_t y_stride, uint32_t cols, uint32_t rows,
                            uint32_t batch);

/* Up to three matrices of one type and column count over the same vectors
 * (Q, K and V, or gate and up): for m < n_mat, Y_m[b*y_stride[m] + r] =
 * sum_c deq(W_m[r,c]) * X[b*x_stride + c], b < batch (<= 16). As n_mat calls
 * of vbs_gfx950_linear_batch (F32 and LNS8 bit for bit; the other types within the
 * rounding of f32 sums, whose order goes by all of a call's matrices); for Q4_K
 * and Q6_K, and for Q4_0, Q4_1, Q8_0 and F16 where it is sooner done, the vectors are
 * prepared once and every matrix shares one matrix-core launch, as the batched
 * decoder runs a layer's Q/K/V and gate/up. w, rows, y and y_stride are host
 * arrays of n_mat entries (w[m] and y[m] device pointers). No counterpart in
 * the reference (it has no batched matvec). */
int vbs_gfx950_linear_batch_multi(int type, uint32_t n_mat, const void *const *w,
                                  const uint32_t *rows, const float *x, uint32_t x_stride,
                                  float *const *y, const uint32_t *y_stride, uint32_t cols,
                                  uint32_t batch);

/* ---- steps of several tokens over the cache (extension) --------------------
 * The reference's loop takes one token at a time (src/vbs_specializer.c:353-357):
 * ROTARY and CACHE one position, ATTENTION one query. These operators take n
 * tokens over the same f16 caches ([layer][max_ctx][n_kv_heads * head_dim]): the
 * chunk of a prompt, the drafted tokens of speculative decoding, and single
 * tokens whose attention the plain op does not have. A token is stored in a
 * slot of the cache; its position (for the rotation) may be any number. All:
 * n <= 65535 (0: nothing is done), at most 2^31 slots, head_dim even and <= 256, at most 16 q heads
 * per kv head, at most 2^28 rows (tokens x q heads) of an attention; a row of q, k, v or out is
 * n_heads x head_dim floats and rows lie
 * a stride (in floats, at least a row) apart, so that the rows of a fused Q/K/V
 * product can be given as they are. No call waits for the device. */

/* Rotary positions with several axes (time, height, width): pair p (elements 2p
 * and 2p + 1, as vbs_gfx950_rope) of every head of token i turns by
 * pos[axis(p)][i] * theta^(-2p / head_dim), where axis x owns sections[x] pairs,
 * in order (n_axes <= 4; the sections add up to head_dim / 2; a host array). pos
 * is a device array [n_axes][n]. q is rotated in place; k is rotated, and k and v
 * are stored as f16, with vbs_gfx950_cache_store's rounding, in the slots slot ..
 * slot + n - 1 of `layer` (k itself is left as it was). q may be NULL (k and v
 * alone), or k, v, kc and vc (q alone). Angles are formed in 64 bits, which far
 * positions need; vbs_gfx950_rope forms them in f32, as the reference does, and
 * differs by up to pos * 2^-23 rad: a loop takes one of the two throughout.
 * theta is at least 2^-21. */
int vbs_gfx950_rope_axes(float *q, uint32_t q_stride, const float *k, const float *v,
                         uint32_t kv_stride, const int32_t *pos, uint32_t n, uint32_t n_axes,
                         const uint32_t *sections, uint16_t *kc, uint16_t *vc, uint32_t slot,
                         uint32_t layer, uint32_t max_ctx, uint32_t n_q_heads,
                         uint32_t n_kv_heads, uint32_t head_dim, float theta);

/* Attention of a tree of n drafted tokens, in the slots past .. past + n - 1:
 * row i sees every slot below past, and slot past + t where bit t % 64 of
 * mask[i * ceil(n / 64) + t / 64] is set (a device array; a tree sets the bits of
 * a token's ancestors and its own). out row i, per q head: sum_j w_j v_j with
 * w = softmax(scale q.k_j) over the slots it sees, in f32 as
 * vbs_gfx950_attention; a row that sees nothing, or whose scores are all -inf, gives
 * 0, and what a row does not see does not reach it, infinities and NaN included. out must not overlap q.
 * Scores are held in f32 and in units of log2: up to 2e38 in size. A row with a score beyond 1.1e7, or with an infinity or
 * a NaN in a K or V row among the slots its workgroup looks at, is right but slow: it is taken again by one wave (about
 * 3 ms for the heads of one such token over 2048 slots, where a whole chunk takes 0.1). */
int vbs_gfx950_attention_tree(const float *q, uint32_t q_stride, const uint16_t *kc,
                              const uint16_t *vc, float *out, uint32_t out_stride, uint32_t n,
                              uint32_t past, const uint64_t *mask, uint32_t layer,
                              uint32_t max_ctx, uint32_t n_q_heads, uint32_t n_kv_heads,
                              uint32_t head_dim, float scale);

/* What vbs_gfx950_attention_chunk adds to plain causal attention; 0 / NULL
 * fields are absent. Device arrays. */
typedef struct vbs_gfx950_attn_terms {
    float cap;             /* s = cap * tanh(s / cap) */
    const float *slopes;   /* n_q_heads: then s = s - slopes[h] * |i - j| in slots */
    const int32_t *docs;   /* past + n: slots of another document than the row's are not seen */
    uint32_t prefix;       /* slots below it are seen by every row (of their document) */
    float *mass;           /* [layer][n_kv_heads][max_ctx]: the weights added up, see below */
} vbs_gfx950_attn_terms_t;

/* Attention of n consecutive tokens in the slots past .. past + n - 1 (n = 1: one
 * decode step): the row of slot i sees the slots j <= i, and j < prefix, of its
 * document; s_j = scale q.k_j with the terms above (terms may be NULL), out as
 * for the tree. With mass, the weight that each slot received is added to
 * mass[(layer * n_kv_heads + kv head) * max_ctx + slot], summed over the rows
 * and the q heads of the kv head in a fixed order: what vbs_gfx950_cache_evict
 * chooses by (for at most 2^27 slots x kv heads). */
int vbs_gfx950_attention_chunk(const float *q, uint32_t q_stride, const uint16_t *kc,
                               const uint16_t *vc, float *out, uint32_t out_stride, uint32_t n,
                               uint32_t past, uint32_t layer, uint32_t max_ctx,
                               uint32_t n_q_heads, uint32_t n_kv_heads, uint32_t head_dim,
                               float scale, const vbs_gfx950_attn_terms_t *terms);

/* Cut the first len slots of the layers layer .. layer + n_layers - 1 to budget
 * slots, per layer and kv head: the first `first` and the last `last` stay, and of
 * the others those of the greatest mass (the lowest slot among equals, NaN the
 * least of all). The kept rows of K and V move, in slot order and in place, to
 * the slots 0 .. budget - 1 of their kv head; the rows behind are left as they
 * were. kept (device, [n_layers][n_kv_heads][budget]) receives the slots they came
 * from, and mass_out, if not NULL (it may be mass itself), their mass, and 0 for
 * the slots budget .. len - 1, so that tokens stored there start from 0. Each
 * head has its own slots afterwards: distances and documents by slot
 * (vbs_gfx950_attn_terms_t) then no longer mean the tokens' own. At most 2^20
 * layers x kv heads. */
int vbs_gfx950_cache_evict(uint16_t *kc, uint16_t *vc, const float *mass, float *mass_out,
                           uint32_t *kept, uint32_t len, uint32_t budget, uint32_t first,
                           uint32_t last, uint32_t layer, uint32_t n_layers, uint32_t max_ctx,
                           uint32_t n_kv_heads, uint32_t head_dim);

/* ---- a paged cache (extension) ---------------------------------------------
 * The reference's cache is one run of max_ctx rows per layer
 * (src/vbs_host_math.h:150-159). These operators serve several sequences from one
 * pool of pages: a page holds page_slots tokens of every kv head of one layer, a
 * table gives each sequence's pages in order, and the same page may stand in
 * several rows of it (a shared prefix). Values are held as F16, or as Q8_0: per
 * token, kv head and 32 elements an f16 scale d and 32 int8 q, value q d.
 *
 * Layout of a page of K or V: [kv head][unit], a unit being 32 slots of one head,
 * nb = ceil(head_dim / 32) blocks of 32 elements (those behind head_dim are 0):
 *   F16  K [t 2][b nb][g 4][h 4][j 4][e 8]: slot 8 h + 4 t + j, element 32 b + 8 g + e
 *        V [b nb][t 2][g 4][r 16][e 8]:     slot 8 g + e, element 32 b + 16 t + r
 *   Q8_0 K int8 [b nb][g 4][h 4][j 4][t 2][e 8], then scales [b nb][slot 32]
 *        V int8 [b nb][g 4][r 16][t 2][e 8],     then scales [b nb][slot 32]
 * (the order in which the attention's matrix instructions take them: pages are
 * read without LDS). 2048 nb bytes a unit for F16, 1088 nb for Q8_0. */
typedef struct vbs_gfx950_pages {
    void *k, *v;           /* device: [layer][n_pages] pages each, 16-byte aligned, apart */
    int type;              /* F16 or Q8_0 */
    uint32_t page_slots;   /* 32 to 1024, a power of two */
    uint32_t n_pages;
    uint32_t n_kv_heads, head_dim;  /* head_dim even and <= 256 */
    const int32_t *table;  /* device: [n_seqs][table_stride] pages */
    uint32_t n_seqs, table_stride;
} vbs_gfx950_pages_t;

/* Bytes of one page of K, and of one of V (0: not a shape that pages take). */
uint64_t vbs_gfx950_page_bytes(int type, uint32_t page_slots, uint32_t n_kv_heads, uint32_t head_dim);

/* Store k and v (f32 rows of n_kv_heads x head_dim, kv_stride floats apart) of n
 * tokens (<= 65535) in `layer`: token i becomes slot at[i] of sequence seq[i] (seq
 * NULL: of sequence i; device arrays). A negative slot stores nothing (padding), nor
 * does a place that the table has no page for, or a page outside 0 .. n_pages - 1
 * (no memory but the pool's is touched). Two tokens of a call must not have the same place, nor
 * may the rows overlap the layer's pages. F16
 * takes vbs_gfx950_cache_store's rounding. Q8_0: d = f16(max |x| / 127) and q the
 * integer nearest x / d within 127, both rounded once from the exact quotient, ties to
 * even; a block with a NaN or an infinity, or whose d passes f16's range, reads back as NaN. */
int vbs_gfx950_page_store(const vbs_gfx950_pages_t *pages, uint32_t layer, const float *k,
                          const float *v, uint32_t kv_stride, const int32_t *seq,
                          const int32_t *at, uint32_t n);

/* Read back the rows of n tokens, as F32 or F16 rows (out_type; k and v of that type,
 * kv_stride elements apart), for instance into a cache of one sequence for the
 * attention of several tokens. F16 pages come as they are; q d is rounded to f16 as
 * vbs_gfx950_cache_store does. Rows of a negative slot are left as they were; a place without a
 * page gives NaN. The rows of k and v must not share elements with each other (they may lie
 * between each other's) or overlap the layer's pages. */
int vbs_gfx950_page_load(const vbs_gfx950_pages_t *pages, uint32_t layer, int out_type, void *k,
                         void *v, uint32_t kv_stride, const int32_t *seq, const int32_t *at,
                         uint32_t n);

/* Attention of `rows` single tokens (<= 65535, 0: nothing is done; at most 2^28 rows x q heads):
 * row r sees the slots below lens[r] of sequence seq[r] (seq NULL: of sequence r),
 * out = sum_j w_j v_j, w = softmax(scale q.k_j), per q head (at most 16 per kv head),
 * in f32 as vbs_gfx950_attention. A decode step has one row per sequence; the drafted tokens of a
 * sequence are several rows of it, each one slot longer. No lens[r] may pass max_len, by which the work is
 * split (a captured call's is the most that its sequences will grow to). A row of length 0, or whose
 * scores are all -inf, gives 0; a row whose length or sequence is out of range, or one of whose
 * pages is, gives NaN. What lies behind a row's last slot does not reach it, infinities and
 * NaN included. Scores are held in f32 in units of log2, up to 2e38 in size. Weights down to 2^-38 of a
 * row's greatest count (Q8_0: of the greatest weight times the greatest of V's scales); q's elements are
 * held to 2^-22 of themselves or 2^-38 of their head's greatest, whichever is more. Infinities and NaN in a row's
 * own q, K or V are right but slow. out must not overlap q or the layer's pages. No call waits for the device. */
int vbs_gfx950_attention_paged(const vbs_gfx950_pages_t *pages, uint32_t layer, const float *q,
                               uint32_t q_stride, float *out, uint32_t out_stride,
                               const int32_t *seq, const int32_t *lens, uint32_t rows,
                               uint32_t max_len, uint32_t n_q_heads, float scale);

/* Drafted tokens (each behind the one before: several rows of vbs_gfx950_attention_paged, a chunk, or one
 * path through vbs_gfx950_attention_tree's; the branches of a tree are not compared) accepted or refused so that
 * what stays is distributed as the target's own tokens, at one temperature for all sequences of a call. Per sequence b < batch (<= 65535): n drafted tokens (<= 64), ids
 * drafted[b n + i], of which the first id outside 0 .. vocab - 1 ends the draft; target logits in rows
 * b (n + 1) + i (`stride` floats apart), row i the distribution of the token that drafted token i is
 * compared with, and the last that of the token behind the draft; the draft's logits in rows b n + i, or NULL where drafted
 * tokens were certain (looked up); random numbers u[b (n + 1) + i] in [0, 1), n for the drafted tokens and one to draw
 * with. p_i, q_i = softmax(row / temperature). Token x_i stays while u_i q_i(x_i) < p_i(x_i);
 * behind the last that stays comes the lowest x with sum_{y <= x} r(y) > u_n sum r, r = max(p_i - q_i, 0)
 * at the first refusal (p_i where nothing is left of it), p_i at the draft's end. Temperature 0: the greatest
 * logit (the lowest place among equals) is certain, the draft's logits are not read. accepted[b] receives how many stay, tokens[b (n + 1) ..] them,
 * the token drawn, and -1s. A row with a NaN or +inf, or of -inf alone, has no distribution: the target's refuses and
 * draws -1, the draft's refuses (at temperature 0 a NaN is the least of all; only a row of NaN draws -1).
 * Probabilities and sums are held in 64 bits. vocab <= 2^24. accepted and tokens must not overlap each other or what is
 * read (nor drafted: a sequence's tokens are one more than its drafted ones). No call waits for the device. */
int vbs_gfx950_verify_draft(const float *logits, uint32_t stride, const float *draft,
                            uint32_t draft_stride, const int32_t *drafted, const float *u,
                            uint32_t batch, uint32_t n, uint32_t vocab, float temperature,
                            int32_t *accepted, int32_t *tokens);

/* XOR checksum of a device region, as partial words, for
 * i < vbs_gfx950_checksum_partials(bytes): the region is cut into consecutive
 * spans of up to 112 KB, one per workgroup of 16 waves, and partials[16 w + v]
 * is the XOR of the 32-bit words of wave v's share of span w (its interleaved
 * 1 KB runs v, v + 16, v + 32, ... of the span). Their XOR is the region's. p is 16-byte aligned and bytes a multiple of 16; partials is
 * device memory.
 * Verifies uploads (the host XORs the same words) and, reading every byte
 * exactly once and nothing else, it is the read floor beside the matvec
 * roofline. No counterpart in the reference. */
uint32_t vbs_gfx950_checksum_partials(size_t bytes);
int vbs_gfx950_checksum(const void *p, size_t bytes, uint32_t *partials);
/* The same checksum read in another shape, to show how tight the read floor
 * is: variant 0 is vbs_gfx950_checksum; 1 reads 56 KB spans with two 8-wave
 * workgroups per CU (8 partials per workgroup); 2 is variant 0's shape with
 * 16-byte vector loads into registers instead of LDS DMA. The XOR of the
 * partials is the region's in every variant. No counterpart in the
 * reference. */
uint32_t vbs_gfx950_checksum_variant_partials(size_t bytes, int variant);
int vbs_gfx950_checksum_variant(const void *p, size_t bytes, uint32_t *partials, int variant);

/* The library's stream (a hipStream_t), for callers that time kernels with
 * HIP events or capture the stream into a graph.
 *
 * Capture and the library's scratch: vbs_gfx950_linear_batch (Q4_K / Q6_K) and
 * vbs_gfx950_attention keep intermediate results in a device scratch that the
 * library owns. It only grows, and a buffer that a larger call replaces stays
 * allocated until the process ends, so a captured graph keeps valid memory
 * whatever is called after the capture; but graphs that use it must not run
 * beside each other or beside such calls on another stream. Growing allocates,
 * so a call made while the stream is being captured fails (0, reason "operation
 * not permitted when stream is capturing") if it needs more scratch than
 * earlier uncaptured calls have sized: make one uncaptured call of the
 * largest shape before capturing. Batched Q4_0, Q4_1, Q8_0 and F16 calls take
 * memory of the graph's own while captured, at any size, which is given back
 * with the graph and its executables: such graphs may run beside each other
 * and beside any call. So do vbs_gfx950_attention_tree, _chunk and _paged, and
 * vbs_gfx950_verify_draft. */
void *vbs_gfx950_stream(void);

/* ---- graph-replayed decode step (extension) -------------------------------
 * The caller side of one token (src/vbs_specializer.c:231-359) issues ~16
 * dispatches per layer through the ops table, each a separate host launch.
 * The decoder below runs the same sequence, with the same kernels and the
 * same arithmetic, from one HIP graph per model: the token and position live
 * in device memory (RoPE angles come from a table computed once with the host
 * libm, exactly as src/vbs_host_math.h:43-44), and a greedy argmax kernel
 * (first maximum, as main.c:929-932) writes the next token and advances the
 * position, so consecutive tokens replay the graph back to back. */
typedef struct {
    uint32_t n_layers, hidden, ffn, n_heads, n_kv_heads, head_dim, vocab, max_ctx;
    float rope_theta, rms_eps;
    int embd_type;
    const void *tok_embd;            /* device: vocab x hidden packed */
    const float *out_norm;           /* device: hidden */
    int head_type;
    const void *lm_head;             /* device: vocab x hidden packed */
    const float *const *attn_norm;   /* host array of n_layers device pointers */
    const float *const *ffn_norm;    /* host array of n_layers device pointers */
    const int *wtype;                /* host array n_layers x 7 (q,k,v,o,gate,up,down) */
    const void *const *wdata;        /* host array n_layers x 7 device pointers */
    uint16_t *kc, *vc;               /* device f16 caches [n_layers][max_ctx][n_kv_heads*head_dim] */
} vbs_gfx950_model_t;

/* Build the per-token graph (the model's device memory is borrowed, not
 * copied). max_steps bounds one vbs_gfx950_decoder_greedy call. */
int vbs_gfx950_decoder_create(const vbs_gfx950_model_t *m, uint32_t max_steps, void **handle);
/* One token at `pos`; logits (vocab floats, host) may be NULL. */
int vbs_gfx950_decoder_step(void *handle, uint32_t token, uint32_t pos, float *logits);
/* Greedy: feed `token` at `pos`, then n-1 further argmax tokens; tokens[i]
 * is the i-th argmax, margins (may be NULL) top-1 minus top-2 logit. */
int vbs_gfx950_decoder_greedy(void *handle, uint32_t token, uint32_t pos, uint32_t n,
                              uint32_t *tokens, float *margins);
/* The same steps as vbs_gfx950_decoder_greedy, each kernel launched directly
 * instead of replaying the graph (identical results; for tools that trace
 * kernel launches but not graph replays). */
int vbs_gfx950_decoder_greedy_eager(void *handle, uint32_t token, uint32_t pos, uint32_t n,
                                    uint32_t *tokens, float *margins);
/* No counterpart in the reference (a diagnostic of this decoder). Where every
 * layer's O is Q4_K over a 4096-wide q of 128-dim heads, the decoder merges
 * the attention partials inside the O launch: each workgroup merges one head
 * and the workgroups on one XCD share the heads through its L2; a workgroup
 * whose bounded wait for them runs out (one placed or started unexpectedly)
 * merges every head itself, with identical results. Returns 1 when the
 * decoder takes that path, with *count (may be NULL) the workgroups that
 * merged every head themselves since it was created, 0 when it does not, -1
 * on error. The environment variable VBS_ATTN_O_SPIN, read at create, sets
 * the wait's bound in polls (0: no workgroup waits). */
int vbs_gfx950_decoder_attn_o_fallbacks(void *handle, uint32_t *count);
int vbs_gfx950_decoder_destroy(void *handle);

/* ---- batched decode (extension) --------------------------------------------
 * The decode step above for `batch` (1..8) independent sequences over one copy
 * of the weights (the Llama-70B case at batch 8): each sequence has its own
 * caches, m->kc / m->vc + b * kv_seq_stride elements (the model's layout per
 * sequence), its own token and position. Every matrix must be Q4_K or Q6_K
 * (the batched matrix-core kernels; q/k/v and gate/up pairwise of one type).
 * The reference has no batched decode (src/vbs_specializer.c:353-357 loops
 * tokens one by one); each sequence computes the single-sequence step. */
int vbs_gfx950_bdecoder_create(const vbs_gfx950_model_t *m, uint32_t batch, uint64_t kv_seq_stride,
                               uint32_t max_steps, void **handle);
/* Greedy for every sequence: feed tokens0[b] at pos0[b], then n-1 further
 * argmax tokens; tokens[i * batch + b] is sequence b's i-th argmax, margins
 * (may be NULL) its top-1 minus top-2 logit. */
int vbs_gfx950_bdecoder_greedy(void *handle, const uint32_t *tokens0, const uint32_t *pos0,
                               uint32_t n, uint32_t *tokens, float *margins);
/* The same with every kernel launched directly (for kernel tracers). */
int vbs_gfx950_bdecoder_greedy_eager(void *handle, const uint32_t *tokens0, const uint32_t *pos0,
                                     uint32_t n, uint32_t *tokens, float *margins);
/* One step of every sequence with the given tokens[b] at pos[b] (teacher
 * forcing: the graph of vbs_gfx950_bdecoder_greedy, replayed once); the caches
 * at pos[b] are written as by a greedy step, and logits (batch x vocab floats,
 * host, sequence b at b * vocab) may be NULL. */
int vbs_gfx950_bdecoder_step(void *handle, const uint32_t *tokens, const uint32_t *pos,
                             float *logits);
int vbs_gfx950_bdecoder_destroy(void *handle);

/* ---- CPU hot-kernel table on the device (parity adapter) --------------------
 * The arithmetic of the reference's CPU hot-kernel ABI v1
 * (include/vbs_hotpath.h:38-57, src/hotkernels/vbs_hot_ref_impl.h:49-129) on
 * device buffers, bit-identical to its built-in table; the host-pointer
 * module over these is lib/libvbs_hot_gfx950.so (host/vbs_hot_gfx950.c). */

/* Q8 activations of x as the CPU model forms them (src/vbs_cpu.c:166-182):
 * per 32-element block d = amax/127, xq = round(x/d) clamped to +-127,
 * qd = f16(d), qsum = f16(sum(xq)*d) (round to nearest even). cols must be a
 * multiple of 32; x is assumed finite (the CPU model screens non-finite
 * inputs first, src/vbs_cpu.c:185-190). All buffers 4-byte aligned. */
int vbs_gfx950_quantize_q8(const float *x, uint32_t cols, int8_t *xq, float *qd, float *qsum);

/* y[r] = the hot table's matvec of row r (replaces matvec_q8_0 / q4_0 / q4_1 /
 * f32 / f16 of vbs_hot_kernels_t). type Q8_0, Q4_0, Q4_1: act = xq (int8),
 * qd and (Q4_1) qsum as vbs_gfx950_quantize_q8 makes them, cols a multiple
 * of 32; type F32, F16: act = x (f32). w packed row-major. */
int vbs_gfx950_hot_matvec(int type, const void *w, uint32_t rows, uint32_t cols, const void *act,
                          const float *qd, const float *qsum, float *y);

#ifdef __cplusplus
}
#endif
#endif
