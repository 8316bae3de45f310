// vbs_steps.h — launchers of the operators for steps of several tokens over the
// f16 KV cache (rotary positions with several axes, attention of a tree or a
// chunk of tokens, eviction by accumulated weight), shared between the runtime
// (vbs_gfx950_rt.hip) and their kernels. As in vbs_internal.h, every launcher
// enqueues on `s`; the C-ABI entry points have checked the arguments.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace vbs {

constexpr uint32_t kRopeAxes = 4;       // position axes of one call
constexpr uint32_t kRopeMaxPairs = 128;  // head_dim 256, as the attentions
constexpr float kRopeLeastTheta = 0x1p-21f;  // positions of 31 bits then turn by less than 2^52, which the reduction holds

struct RopeAxesArgs {
    float *q;  // NULL: k and v alone
    uint32_t q_stride;
    const float *k, *v;  // NULL with the caches: q alone
    uint32_t kv_stride;
    const int32_t *pos;  // [n_axes][n]
    uint32_t n;
    uint32_t end[kRopeAxes];  // the first pair behind each axis's section
    uint16_t *kc, *vc;        // at the first row to write
    uint32_t nqh, nkh, hd;
};
hipError_t launch_rope_axes(const RopeAxesArgs &a, float theta, hipStream_t s);

// Attention of n rows over the slots [0, past + n) of one layer's caches. Row i
// is the token in slot past + i. With `mask` (a tree) it sees the slots below
// past and past + t where bit t of its `words` mask words is set; without, the
// slots up to its own and those below `prefix`, of its own document where
// `docs` is given.
struct RowsArgs {
    const float *q;
    uint32_t q_stride;
    const uint16_t *kc, *vc;  // at the layer's first row
    float *out;
    uint32_t out_stride;
    uint32_t n, past, nqh, nkh, hd;
    uint32_t group;  // nqh / nkh
    float rgroup;    // 1 / group
    float scale;
    const uint64_t *mask;
    uint32_t words;
    float cap, rcap;      // 0: none; 1 / cap
    const float *slopes;  // NULL: none
    const int32_t *docs;  // NULL: none
    uint32_t prefix;
    float *mass;  // at the layer's first row of max_ctx floats per kv head, or NULL
    uint32_t max_ctx;
};
size_t attn_rows_scratch_bytes(const RowsArgs &a);
// `scratch`: attn_rows_scratch_bytes(a) of device memory (may be NULL if that is 0).
hipError_t launch_attn_rows(const RowsArgs &a, void *scratch, hipStream_t s);

struct EvictArgs {
    uint16_t *kc, *vc;  // at the first layer
    const float *mass;
    float *mass_out;  // NULL: not wanted
    uint32_t *kept;
    uint32_t len, budget, first, last, n_layers, max_ctx, nkh, hd;
};
hipError_t launch_evict(const EvictArgs &a, hipStream_t s);

}  // namespace vbs
