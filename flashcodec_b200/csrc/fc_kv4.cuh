// Paged 4-bit KV cache: the page format and the pieces its kernels share.
//
// A page holds `page_size` tokens (a multiple of 16) of one layer.  The pool is
// (pages, Hk, page_size / 16) tiles, contiguous; a tile holds 16 tokens of one
// KV head, K and V.  Channels are quantised in groups of 32 with one fp16 scale
// for each token and group:
//
//     scale = fp16(min(amax * fl(1/7), 65504)),  code = clamp(rint(x / scale), -7, 7)
//
// and stand for code * scale (exact in fp32).  A group that holds an infinity or
// a NaN gets a NaN scale.  Codes are stored as nibbles, code + 8.
//
// A tile is laid out so that a warp's lane finds in whole 4- to 16-byte words the
// operands that an m16n8k16 matrix instruction wants from it, after an AND and an
// OR per pair of codes (W = D / 32; lane = 4 r + c, r = 0..7, c = 0..3):
//
//   K codes, 16 rows of 16 W bytes.  Row t (token t of the tile) is 4 W words;
//     word c W + j holds channels 32 j + 8 c + i (i = 0..7), channel i in nibble
//     (i >> 1) + 4 (i & 1): a masked word is a pair of neighbouring channels.
//   V codes, 256 W bytes: word m of lane l (m = 0..2W-1) at word
//     (m / VW) 32 VW + l VW + m % VW, VW = 4 (2 where W is odd).  It holds channels
//     16 m + r and 16 m + r + 8 of tokens 2c, 2c+1, 2c+8, 2c+9: channel half x
//     (0, 1), token half y (0: 2c.., 1: 2c+8..), parity e in nibble x + 2 y + 4 e.
//   K scales, 32 W bytes: token t, group g at half (2 (t & 7) + (t >> 3)) W + g,
//     so that the scales of rows r and r + 8 are neighbours.
//   V scales, 32 W bytes: token t, group g at half 4 (c W + g) + 2 y + e with
//     c = (t & 7) >> 1, y = t >> 3, e = t & 1, so that a pair of tokens is a word.
//
// Optional page bounds: for every page and KV head the least and the largest
// value of every key channel, as int8 multiples of one power of two 2^e (least
// rounded down, largest up; e the smallest integer >= -40 for which all fit in
// -127..127); a group whose scale is NaN counts as zeros.  Rounding by powers of two
// nests exactly, so the bounds of a page do not depend on how its tokens were split
// into calls.
#pragma once

#include <algorithm>

#include "fc_common.cuh"

namespace fc {
namespace kv4 {

// status bits (fc_kv4_* `status`)
constexpr int kBadPage = FC_KV4_BAD_PAGE;
constexpr int kBadLength = FC_KV4_BAD_LENGTH;
constexpr int kBadPosition = FC_KV4_BAD_POSITION;

__host__ __device__ constexpr int tile_bytes(int W) { return 576 * W; }
__host__ __device__ constexpr int v_off(int W) { return 256 * W; }
__host__ __device__ constexpr int ks_off(int W) { return 512 * W; }
__host__ __device__ constexpr int vs_off(int W) { return 544 * W; }
__host__ __device__ constexpr int v_vec(int W) { return W % 2 ? 2 : 4; }

inline bool head_dim_ok(int64_t D) { return D == 64 || D == 96 || D == 128 || D == 192 || D == 256; }
inline bool page_size_ok(int64_t P) { return P >= 16 && P <= 1024 && (P & (P - 1)) == 0; }

// word index of word m of lane l in a tile's V codes
template <int W>
__device__ __forceinline__ int v_word(int m, int l) {
    constexpr int VW = v_vec(W);
    return (m / VW) * (32 * VW) + l * VW + m % VW;
}

// Where a page table and the lengths lead: bad entries set a status bit and are
// clamped, so that no access leaves the pool.
struct Table {
    const int *pages;     // (B, max_pages), row stride
    int64_t stride;
    int max_pages, num_pages, log_page;
    int *status;

    __device__ __forceinline__ int page(int64_t b, int i) const {
        if (i >= max_pages) {
            atomicOr(status, kBadLength);
            i = max_pages - 1;
        }
        const int p = pages[b * stride + i];
        if ((unsigned)p >= (unsigned)num_pages) {
            atomicOr(status, kBadPage);
            return 0;
        }
        return p;
    }
    // tokens that the table can hold for a sequence of `len` (negative: none)
    __device__ __forceinline__ int length(int len) const {
        if (len <= 0) return 0;
        if (((int64_t)len + (1 << log_page) - 1) >> log_page > max_pages) {
            atomicOr(status, kBadLength);
            return max_pages << log_page;
        }
        return len;
    }
};

// Smallest integer e >= least with amax <= 127 * 2^e (amax finite, >= 0).
__device__ __forceinline__ int bound_exponent(float amax, int least) {
    if (!(amax > 0.f)) return least;
    const uint32_t u = __float_as_uint(amax);
    int x = (int)(u >> 23);
    uint32_t m = u & 0x7fffffu;
    if (x == 0) {  // subnormal: 2^-126 and less
        const int n = __clz(m) - 8;
        m = (m << n) & 0x7fffffu;
        x = 1 - n;
    }
    // amax = (1 + m / 2^23) 2^(x - 127); 127 * 2^e = 1.984375 * 2^(e + 6)
    const int e = x - 127 - 6 + (m > 0x7e0000u ? 1 : 0);
    return max(e, least);
}

__device__ __forceinline__ float pow2f(int e) {  // 2^e, e in -126..127
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Of sorted keys key(0) <= key(1) <= ... <= key(n - 1) with key(0) <= x: the last
// index whose key is <= x.  All lanes of a warp call it with the same x; every
// step reads 32 keys.
template <typename F>
__device__ __forceinline__ int warp_find(F key, int n, int64_t x) {
    const int lane = threadIdx.x & 31;
    int lo = 0;
    int64_t len = n;
    while (len > 1) {
        const int step = (int)((len + 31) / 32);
        const int64_t i = lo + (int64_t)lane * step;
        const bool le = (int64_t)lane * step < len && key((int)i) <= x;
        const int k = 31 - __clz(__ballot_sync(0xffffffffu, le) | 1u);
        len = min((int64_t)step, len - (int64_t)k * step);
        lo += k * step;
    }
    return lo;
}

// ------------------------------------------------------------------ host side
// Workspaces begin with a header and arrival counters for this many (sequence, head, ..)
// units, whatever a call's sizes: what a call writes behind them is never a later call's
// counters.
constexpr int64_t kMaxUnits = 1 << 18;
constexpr int64_t kCounterBytes = 256 + kMaxUnits * 4;

template <typename F>
int by_head_dim(int64_t D, F f) {
    switch (D) {
        case 64: return f(std::integral_constant<int, 2>());
        case 96: return f(std::integral_constant<int, 3>());
        case 128: return f(std::integral_constant<int, 4>());
        case 192: return f(std::integral_constant<int, 6>());
        default: return f(std::integral_constant<int, 8>());
    }
}

template <typename F>
int by_dtype(int dt, F f) {
    switch (dt) {
        case FC_F32: return f(float());
        case FC_BF16: return f(__nv_bfloat16());
        default: return f(__half());
    }
}

// 16-byte accesses are possible at every row of (base, strides in elements)
inline bool rows_aligned(const void *p, int dtype, int64_t s0, int64_t s1, int64_t s2) {
    const int64_t n = 16 / dtype_size(dtype);
    return aligned(p, 16) && s0 % n == 0 && s1 % n == 0 && s2 % n == 0;
}

inline int ilog2(int64_t x) {
    int n = 0;
    while ((int64_t(1) << n) < x) n++;
    return n;
}

inline int check_cache(const char *what, int64_t B, int64_t Hk, int64_t D, int64_t page_size,
                int64_t num_pages, int64_t max_pages, const void *pool, const int *page_table,
                const int *status) {
    if (!head_dim_ok(D)) {
        set_error("%s: head dim %lld is not one of 64, 96, 128, 192, 256", what, (long long)D);
        return FC_ENOTSUP;
    }
    if (!page_size_ok(page_size)) {
        set_error("%s: page size %lld is not a power of two from 16 to 1024", what, (long long)page_size);
        return FC_EINVAL;
    }
    if (B < 0 || Hk <= 0 || num_pages <= 0 || max_pages <= 0 || B > (1 << 24) || Hk > 65535 ||
        num_pages > 0x7fffffff || max_pages > 0x7fffffff || max_pages * page_size > 0x7fffff00) {
        set_error("%s: bad shape", what);
        return FC_EINVAL;
    }
    if (!pool || (!page_table && B) || !status || !aligned(pool, 16)) {
        set_error("%s: the pool (16-byte aligned), the page table and the status word are required", what);
        return FC_EINVAL;
    }
    return FC_OK;
}

// Rows (sequence, token, head) of D elements, strides in elements.
struct Rows {
    const void *p;
    int64_t sb, ss, sh, H;
};

// The same rows in the same places.
inline bool same_rows(const Rows &x, const Rows &y, int64_t B, int64_t S) {
    return x.p == y.p && (x.H == 1 || x.sh == y.sh) && (S == 1 || x.ss == y.ss) && (B == 1 || x.sb == y.sb);
}

// Rows of an expanded tensor: several in one place.
inline bool rows_repeat(const Rows &x, int64_t B, int64_t S) {
    return (B > 1 && x.sb == 0) || (S > 1 && x.ss == 0) || (x.H > 1 && x.sh == 0);
}

// For slices of the heads of one buffer, its dims in any order: whether they have heads in
// common (0, 1), or -1 for sets that are no such slices.
inline int heads_meet(const Rows &x, const Rows &y, int64_t B, int64_t S, int64_t D, int64_t size) {
    const int64_t sh = x.H > 1 ? x.sh : y.sh;
    const int64_t d = (int64_t)reinterpret_cast<uintptr_t>(y.p) - (int64_t)reinterpret_cast<uintptr_t>(x.p);
    if ((B > 1 && x.sb != y.sb) || (S > 1 && x.ss != y.ss) || (y.H > 1 && y.sh != sh) || sh <= 0 ||
        d % (sh * size))
        return -1;
    const int64_t h = d / (sh * size);  // of x, where y begins
    // their rows lie apart when each dim's stride passes all that the ones inside it reach
    struct { int64_t n, stride; } dim[3] = {{B, x.sb}, {S, x.ss}, {(x.H > h + y.H ? x.H : h + y.H) - (h < 0 ? h : 0), sh}};
    for (auto &z : dim)
        if (z.n <= 1) z.stride = 0;
    std::sort(dim, dim + 3, [](const auto &a, const auto &b) { return a.stride < b.stride; });
    int64_t reach = D;
    for (const auto &z : dim) {
        if (z.n <= 1) continue;
        if (z.stride < reach) return -1;
        reach += (z.n - 1) * z.stride;
    }
    return h < x.H && h + y.H > 0;
}

// Whether two sets of B x S rows (packed: 1 x T) can share a byte.  Sets whose spans meet
// are told apart where they are slices of the heads of one buffer, or have equal strides from
// token to token and heads in runs that do not meet within one.
inline bool rows_meet(const Rows &x, const Rows &y, int64_t B, int64_t S, int64_t D, int64_t size) {
    auto span = [&](const Rows &r, int64_t &lo, int64_t &hi) {
        lo = hi = 0;
        for (int64_t e : {(B - 1) * r.sb, (S - 1) * r.ss, (r.H - 1) * r.sh}) (e < 0 ? lo : hi) += e;
        const int64_t base = (int64_t)reinterpret_cast<uintptr_t>(r.p);
        lo = base + lo * size;
        hi = base + (hi + D) * size;
    };
    int64_t x0, x1, y0, y1;
    span(x, x0, x1);
    span(y, y0, y1);
    if (x0 >= y1 || y0 >= x1) return false;
    const int slices = heads_meet(x, y, B, S, D, size);
    if (slices >= 0) return slices;
    const int64_t step = S > 1 ? x.ss : x.sb;  // from token to token
    const bool same = (S == 1 || x.ss == y.ss) && (B == 1 || x.sb == y.sb) &&
                      (S == 1 || B == 1 || x.sb % (step ? step : 1) == 0);
    if (!same || (S * B > 1 && step <= 0) || x.sh < 0 || y.sh < 0) return true;
    const int64_t xw = ((x.H - 1) * x.sh + D) * size, yw = ((y.H - 1) * y.sh + D) * size;
    int64_t d = (int64_t)reinterpret_cast<uintptr_t>(y.p) - (int64_t)reinterpret_cast<uintptr_t>(x.p);
    if (S * B == 1) return d < xw && -d < yw;
    const int64_t pitch = step * size;
    d = (d % pitch + pitch) % pitch;
    return d < xw || d + yw > pitch;
}

}  // namespace kv4
}  // namespace fc
