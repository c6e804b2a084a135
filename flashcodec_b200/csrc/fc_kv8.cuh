// Paged 8-bit KV cache: the format and the pieces its kernels share.
//
// A page holds `page_size` tokens of one layer: int8 codes (pages, 2, Hk, page_size, D),
// keys and values, in plain order, and one fp32 scale for every 16 tokens of a head,
// (pages, 2, Hk, page_size / 16).  With amax over the tokens that the block holds so far
// and all channels,
//
//     scale = 2^e, e the smallest integer >= -126 with amax < 128 * 2^e  (0 for amax = 0),
//     code  = floor(x / scale) in -128..127, and stands for (code + 1/2) * scale,
//
// off by at most scale / 2 <= amax / 128.  A block with an infinity or a NaN has a NaN
// scale.  Why a floor and powers of two: floors nest, floor(floor(x / s) / 2^j) =
// floor(x / (s 2^j)), so when a token raises the scale of a block that is still filling,
// the codes held are shifted right, and equal those of the block quantised in one go.
// What is stored does not depend on how tokens are split into calls.  (A step is up to
// twice that of a scale of amax / 127, which would have to be rounded anew with every
// token that raises it.)
#pragma once

#include "fc_kv4.cuh"

namespace fc {
namespace kv8 {

using kv4::Rows;
using kv4::Table;
using kv4::by_dtype;
using kv4::by_head_dim;
using kv4::ilog2;
using kv4::rows_aligned;
using kv4::rows_meet;
using kv4::rows_repeat;
using kv4::same_rows;
using kv4::warp_find;

constexpr int kBlock = 16;  // tokens of a scale

// What the tensors of a pool are indexed by: (page, K or V, head).
struct Pool {
    signed char *codes;
    float *scales;
    int Hk, log_page;

    __device__ __forceinline__ int64_t head(int page, int kv, int h) const {
        return ((int64_t)page * 2 + kv) * Hk + h;
    }
};

// Biased exponent of the scale of a block with this amax: 0 for 0, 255 where it is no number.
__device__ __forceinline__ int scale_exponent(float amax) {
    const int E = (int)(__float_as_uint(amax) >> 23);  // amax in [2^(E - 127), 2^(E - 126))
    return amax == 0.f ? 0 : E == 255 ? 255 : max(E - 6, 1);
}

__device__ __forceinline__ float max_nan(float x, float y) {  // a NaN stays
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}

inline int check_pool(const char *what, int64_t B, int64_t Hk, int64_t D, int64_t page_size, int64_t num_pages,
                      int64_t max_pages, const void *codes, const void *scales, const int *page_table,
                      const int *status) {
    const int rc = kv4::check_cache(what, B, Hk, D, page_size, num_pages, max_pages, codes, page_table, status);
    if (rc) return rc;
    if (!scales || !aligned(scales, 4)) {
        set_error("%s: the scales are required", what);
        return FC_EINVAL;
    }
    return FC_OK;
}

}  // namespace kv8
}  // namespace fc
