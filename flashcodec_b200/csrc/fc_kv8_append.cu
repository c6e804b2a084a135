// Paged 8-bit KV cache: new tokens into the pages, and the values held back out.
//
// Append: RMS norm of the query and key heads, rotary positions of one or several axes,
// 8-bit codes with one scale for 16 tokens of a head (fc_kv8.cuh), in one launch.
//
//   norm      y = x r w, r = 1 / sqrt(sum(x^2) fl(1/D) + eps), the sum a tree over neighbours
//   rotation  (a, b) -> (a c - b s, b c + a s) for pairs (i, i + R/2) or (2i, 2i + 1), with the
//             angle of the position, or of positions[axes[i]]
//   every product and sum rounded by itself
//
// Bytes bound it: q is read and written, k and v are read, one byte a value is written.
// A scale belongs to 16 tokens of a head, so a block of threads owns the tokens that a call
// adds to one such run (a warp 4 of its rows, 8 channels a lane): the largest |value| goes
// through shared memory and nothing is read twice or added with atomics.  Where the run held
// tokens before and its scale grows, their codes are shifted by the same block.
#include "fc_kv8.cuh"

namespace fc {
namespace kv8 {
namespace {

constexpr int kThreads = 256;
constexpr int kQPasses = 4;  // passes of a query warp: that many loads of 8 channels on their way in a lane

struct AppendArgs {
    const void *q, *k, *v;
    void *qo;
    int64_t q_sb, q_ss, q_sh, qo_sb, qo_ss, qo_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
    int64_t T, S;  // tokens in all; tokens of each sequence (0: ragged, by cu)
    int B, Hq, Hk, D, per, slots, q_units;  // per: runs of a sequence; q_units: warps of a token
    const int *cu, *lengths, *positions, *axes;
    int n_axes, axes_vec;
    const void *qw, *kw;
    int w_dtype;
    float eps, inv_d;
    const float *rotary;
    int64_t rotary_rows;
    int R, interleaved;
    Pool pool;
    Table table;
    int vec;  // bits: q, q_out, k, v rows and norm weights can be read in 16-byte words
};

template <int W> struct Lay {
    static constexpr int D = 32 * W;
    static constexpr int LPR = W == 2 ? 8 : W <= 4 ? 16 : 32;  // lanes of a row (of D = 96 and 192 some idle)
    static constexpr int RP = 32 / LPR;                        // rows of a warp's pass
};

template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, float x[8]) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = Elem<T>::to_f32(p[i]);
    } else if constexpr (sizeof(T) == 4) {
        load_vec_f32<T, 4>(p, x);
        load_vec_f32<T, 4>(p + 4, x + 4);
    } else {
        load_vec_f32<T, 8>(p, x);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, bool vec, const float x[8]) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 8; i++) store_from_f32(p, i, Elem<T>::code, x[i]);
    } else if constexpr (sizeof(T) == 4) {
        store_vec_from_f32<T, 4>(p, x);
        store_vec_from_f32<T, 4>(p + 4, x + 4);
    } else {
        uint4 w;
        uint32_t *u = reinterpret_cast<uint32_t *>(&w);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                u[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                u[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        *reinterpret_cast<uint4 *>(p) = w;
    }
}

// Where a lane's 8 channels lie in the rotation: part 0 outside of it, 1 and 2 the halves,
// 3 pairs; the lane of the other half; the first of its pairs.
struct Place {
    int part, lane, pair;
};

template <int W>
__device__ __forceinline__ Place place_of(const AppendArgs &a, int lane) {
    const int ci = lane % Lay<W>::LPR, shift = a.R / 16;
    Place p;
    p.part = ci * 8 >= a.R ? 0 : a.interleaved ? 3 : ci < shift ? 1 : 2;
    p.lane = p.part == 1 ? lane + shift : p.part == 2 ? lane - shift : lane;
    p.pair = p.part == 3 ? ci * 4 : (p.part == 2 ? ci - shift : ci) * 8;
    return p;
}

// Cosines and sines of a lane's pairs (four in c[0..3] with pairs of neighbours).
struct Angles {
    float c[8], s[8];
};

__device__ __forceinline__ const float *angle_row(const AppendArgs &a, int64_t pos) {
    if (pos < 0 || pos >= a.rotary_rows) {
        atomicOr(a.table.status, kv4::kBadPosition);
        pos = pos < 0 ? 0 : a.rotary_rows - 1;
    }
    return a.rotary + pos * a.R;
}

// Of token t of the call; `at`: its place in the cache.
__device__ __forceinline__ void load_angles(Angles &g, const AppendArgs &a, const Place &p, int64_t t, int64_t at) {
    if (p.part == 0) return;
    int ax = 0;
    bool one = true;  // all of the lane's pairs turn by one axis
    if (a.axes) {
        int x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if (i < 4 || p.part != 3) x[i] = min(max(a.axes[p.pair + i], 0), a.n_axes - 1);
            else x[i] = x[0];
        }
#pragma unroll
        for (int i = 1; i < 8; i++) one = one && x[i] == x[0];
        ax = x[0];
        if (!one) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if (i >= 4 && p.part == 3) break;
                const float *row = angle_row(a, a.positions[x[i] * a.T + t]) + p.pair + i;
                g.c[i] = row[0];
                g.s[i] = row[a.R / 2];
            }
        }
    }
    if (one) {
        const float *row = angle_row(a, a.positions ? (int64_t)a.positions[ax * a.T + t] : at) + p.pair;
        load_vec_f32<float, 4>(row, g.c);
        load_vec_f32<float, 4>(row + a.R / 2, g.s);
        if (p.part != 3) {
            load_vec_f32<float, 4>(row + 4, g.c + 4);
            load_vec_f32<float, 4>(row + a.R / 2 + 4, g.s + 4);
        }
    }
}

// Norm weights of the lane's channels.
template <typename T>
__device__ __forceinline__ void load_weights(const AppendArgs &a, const void *w, int ch, bool on, float x[8]) {
    if (!w || !on) return;
    if (a.w_dtype == Elem<T>::code) {
        load8(static_cast<const T *>(w) + ch, a.vec & 16, x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = load_as_f32(w, ch + i, a.w_dtype);
    }
}

// x r w of one head.  All lanes of the warp call it (those without channels hold zeros).
template <int W>
__device__ __forceinline__ void norm_row(float x[8], const float w[8], const AppendArgs &a) {
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) s[i] = __fmul_rn(x[i], x[i]);
#pragma unroll
    for (int n = 4; n; n /= 2)
#pragma unroll
        for (int i = 0; i < n; i++) s[i] = __fadd_rn(s[2 * i], s[2 * i + 1]);
#pragma unroll
    for (int m = 1; m < Lay<W>::LPR; m *= 2) s[0] = __fadd_rn(s[0], __shfl_xor_sync(0xffffffffu, s[0], m));
    const float r = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fmul_rn(s[0], a.inv_d), a.eps)));
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = __fmul_rn(__fmul_rn(x[i], r), w[i]);
}

__device__ __forceinline__ float turn(float x, float c, float y, float s) {  // x c + y s
    return __fadd_rn(__fmul_rn(x, c), __fmul_rn(y, s));
}

// Rotation of one head.  All lanes of the warp call it.
__device__ __forceinline__ void rotate_row(float x[8], const Angles &g, const Place &p, const AppendArgs &a) {
    if (a.interleaved) {
        if (p.part) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float u = x[2 * i], v = x[2 * i + 1];
                x[2 * i] = turn(u, g.c[i], v, -g.s[i]);
                x[2 * i + 1] = turn(v, g.c[i], u, g.s[i]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float y = __shfl_sync(0xffffffffu, x[i], p.lane);
            if (p.part) x[i] = turn(x[i], g.c[i], y, p.part == 1 ? -g.s[i] : g.s[i]);
        }
    }
}

// floor(code / 2^n) of four codes.
__device__ __forceinline__ uint32_t shift_codes(uint32_t w, int n) {
    n = min(n, 7);  // from 7 on: -1 or 0
    const uint32_t u = ((w ^ 0x80808080u) >> n) & (0x01010101u * (0xffu >> n));  // floor((code + 128) / 2^n)
    return __vsub4(u, 0x01010101u * (128u >> n));
}

// ------------------------------------------------------------------ keys and values
// Sequence b's run k of 16 positions: what of it the call adds.
struct Run {
    int64_t pos, lo, hi, t0;  // first position; the positions added; row of the call's token at position 0
};

template <typename T, int W>
__device__ __forceinline__ void append_run(const AppendArgs &a, const Run &r, int page, int h) {
    using L = Lay<W>;
    constexpr int PASSES = 4 / L::RP;
    __shared__ float tops[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kv = warp >> 2;
    const int ch = lane % L::LPR * 8, row0 = (warp & 3) * 4 + lane / L::LPR;
    const bool lane_on = ch < L::D;
    const int in_page = (int)(r.pos & ((1 << a.pool.log_page) - 1));
    const int64_t head = a.pool.head(page, kv, h);
    signed char *codes = a.pool.codes + ((head << a.pool.log_page) + in_page) * L::D + ch;
    float *scale = a.pool.scales + (head << (a.pool.log_page - 4)) + (in_page >> 4);
    const int held = (int)max((int64_t)0, r.lo - r.pos);
    const float old = held ? *scale : 0.f;
    const T *src = static_cast<const T *>(kv ? a.v : a.k);
    const int64_t sb = kv ? a.v_sb : a.k_sb, ss = kv ? a.v_ss : a.k_ss, sh = kv ? a.v_sh : a.k_sh;
    float x[PASSES][8];
    bool on[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int64_t pos = r.pos + row0 + i * L::RP, t = r.t0 + pos;
        on[i] = pos >= r.lo && pos < r.hi && lane_on;
#pragma unroll
        for (int j = 0; j < 8; j++) x[i][j] = 0.f;
        if (on[i]) {
            const int64_t b = a.S ? t / a.S : 0;
            load8(src + b * sb + (a.S ? t - b * a.S : t) * ss + h * sh + ch, a.vec & (kv ? 8 : 4), x[i]);
        }
    }
    float top = 0.f;
    if (kv == 0) {
        float w[8] = {};
        load_weights<T>(a, a.kw, ch, lane_on, w);
        const Place p = place_of<W>(a, lane);
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            Angles g;
            const int64_t pos = r.pos + row0 + i * L::RP;
            if (a.R && on[i]) load_angles(g, a, p, r.t0 + pos, pos);
            if (a.kw) norm_row<W>(x[i], w, a);
            if (a.R) {
                if (!on[i])
#pragma unroll
                    for (int j = 0; j < 8; j++) g.c[j] = g.s[j] = 0.f;
                rotate_row(x[i], g, p, a);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < PASSES; i++)
        if (on[i])
#pragma unroll
            for (int j = 0; j < 8; j++) top = max_nan(top, fabsf(x[i][j]));
#pragma unroll
    for (int m = 1; m < 32; m *= 2) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, m));
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    top = max_nan(max_nan(tops[4 * kv], tops[4 * kv + 1]), max_nan(tops[4 * kv + 2], tops[4 * kv + 3]));
    // biased exponents: 0 no value but zero, 255 no number
    const int e_old = (int)(__float_as_uint(old) >> 23) & 255;
    const int e = max(e_old, top == top ? scale_exponent(top) : 255);
    const float inv = e == 0 || e == 255 ? 0.f : __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int row = row0 + i * L::RP;
        if (on[i]) {
            uint32_t c[8];
            // x / scale + 1.5 * 2^23 rounded down: its low byte is the floor
#pragma unroll
            for (int j = 0; j < 8; j++)
                c[j] = inv > 0.f ? __float_as_uint(__fmaf_rd(x[i][j], inv, 12582912.f)) : 0u;
            uint2 w;
            w.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
            w.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
            *reinterpret_cast<uint2 *>(codes + (int64_t)row * L::D) = w;
        } else if (row < held && lane_on && e_old && e > e_old && e < 255) {
            uint2 *p = reinterpret_cast<uint2 *>(codes + (int64_t)row * L::D);
            uint2 w = *p;
            w.x = shift_codes(w.x, e - e_old);
            w.y = shift_codes(w.y, e - e_old);
            *p = w;
        }
    }
    if ((warp & 3) == 0 && lane == 0) *scale = __uint_as_float(e == 255 ? 0x7fc00000u : (uint32_t)e << 23);
}

template <typename T, int W>
__device__ __forceinline__ void keys_and_values(const AppendArgs &a, int slot, int h) {
    int b, k;
    int64_t c0, n;
    if (a.S) {
        b = slot / a.per;
        k = slot - b * a.per;
        c0 = (int64_t)b * a.S;
        n = a.S;
    } else {
        // a sequence of n tokens has at most n / 16 + 2 runs: slots from cu / 16 + 2 b on are its own
        const int *cu = a.cu;
        b = warp_find([=](int i) { return (int64_t)(cu[i] >> 4) + 2 * i; }, a.B, slot);
        c0 = cu[b];
        k = slot - (int)((c0 >> 4) + 2 * b);
        n = cu[b + 1] - c0;
        if (k < 0) return;
    }
    const int len = a.lengths[b];
    if (len < 0) return;
    // tokens without a row are skipped
    int64_t i0 = 0, i1 = n;
    if (c0 < 0 || c0 + n > a.T) {
        if (threadIdx.x == 0) atomicOr(a.table.status, kv4::kBadLength);
        i0 = max((int64_t)0, -c0);
        i1 = min(n, a.T - c0);
    }
    Run r;
    r.pos = (int64_t)((len >> 4) + k) << 4;
    r.lo = max(r.pos, len + i0);
    r.hi = min(r.pos + kBlock, len + i1);
    r.t0 = c0 - len;
    if (r.lo >= r.hi) return;
    const int64_t i = r.pos >> a.table.log_page;
    if (i >= a.table.max_pages) {
        if (threadIdx.x == 0) atomicOr(a.table.status, kv4::kBadLength);
        return;
    }
    const int page = a.table.pages[b * a.table.stride + i];
    if ((unsigned)page >= (unsigned)a.table.num_pages) {
        if (threadIdx.x == 0) atomicOr(a.table.status, kv4::kBadPage);
        return;
    }
    append_run<T, W>(a, r, page, h);
}

// ------------------------------------------------------------------------- queries
// kQPasses passes of heads of one token: its angles are read once.
template <typename T, int W>
__device__ __forceinline__ void queries(const AppendArgs &a, int64_t unit) {
    using L = Lay<W>;
    const int64_t t = unit / a.q_units;
    if (t >= a.T) return;
    const int lane = threadIdx.x & 31, ch = lane % L::LPR * 8;
    const int h0 = (int)(unit - t * a.q_units) * kQPasses * L::RP + lane / L::LPR;
    int64_t b = 0, s = t, at = 0;
    bool none = false;  // a row of no sequence
    if (a.S) {
        b = t / a.S;
        s = t - b * a.S;
        if (a.R && !a.positions) at = (int64_t)max(0, a.lengths[b]) + s;
    } else {
        const int *cu = a.cu;
        int i = 0;
        if (a.B) i = warp_find([=](int j) { return (int64_t)cu[j]; }, a.B, t);
        none = a.B == 0 || t < cu[i] || t >= cu[i + 1];
        if (!none && a.R && !a.positions) at = (int64_t)max(0, a.lengths[i]) + t - cu[i];
    }
    float x[kQPasses][8];
    const T *src = static_cast<const T *>(a.q) + b * a.q_sb + s * a.q_ss + ch;
    T *dst = static_cast<T *>(a.qo) + b * a.qo_sb + s * a.qo_ss + ch;
    const bool lane_on = ch < L::D;
#pragma unroll
    for (int i = 0; i < kQPasses; i++) {
        const int h = h0 + i * L::RP;
#pragma unroll
        for (int j = 0; j < 8; j++) x[i][j] = 0.f;
        if (lane_on && h < a.Hq && !none) load8(src + h * a.q_sh, a.vec & 1, x[i]);
    }
    const Place p = place_of<W>(a, lane);
    Angles g;
    float w[8] = {};
    if (!none) {
        if (a.R) load_angles(g, a, p, t, at);
        load_weights<T>(a, a.qw, ch, lane_on, w);
    }
#pragma unroll
    for (int i = 0; i < kQPasses; i++) {
        const int h = h0 + i * L::RP;
        if (!none) {
            if (a.qw) norm_row<W>(x[i], w, a);
            if (a.R) rotate_row(x[i], g, p, a);
        }
        if (lane_on && h < a.Hq) store8(dst + h * a.qo_sh, a.vec & 2, x[i]);
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ AppendArgs a) {
    const int64_t runs = (int64_t)a.slots * a.Hk;
    if (blockIdx.x < runs) {
        const int slot = (int)(blockIdx.x / a.Hk);
        keys_and_values<T, W>(a, slot, (int)(blockIdx.x - (int64_t)slot * a.Hk));
    } else {
        queries<T, W>(a, ((int64_t)blockIdx.x - runs) * (kThreads / 32) + (threadIdx.x >> 5));
    }
}

// ---------------------------------------------------------------------------- read
struct ReadArgs {
    int B, Hk;
    int64_t T, S;
    const int *starts, *cu;
    void *k, *v;
    int64_t o_sb, o_ss, o_sh;
    Pool pool;
    Table table;
    int vec;
};

// A warp reads the keys or the values of a token, all heads: 8 codes a lane.
template <typename T, int W>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadArgs a) {
    constexpr int CH = 4 * W;  // lanes of a row
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5), t = unit >> 1;
    const int kv = (int)unit & 1;
    if (t >= a.T) return;
    int64_t b = 0, s = t;
    int i = 0;
    int64_t pos = -1;  // no sequence, or a negative start
    if (a.S) {
        i = (int)(t / a.S);
        b = i;
        s = t - b * a.S;
        const int start = a.starts ? a.starts[i] : 0;
        if (start >= 0) pos = start + s;
    } else if (a.B) {
        const int *cu = a.cu;
        if (unit == 0 && lane == 0 && (cu[0] < 0 || cu[a.B] > a.T)) atomicOr(a.table.status, kv4::kBadLength);
        i = warp_find([=](int j) { return (int64_t)cu[j]; }, a.B, t);
        if (t >= cu[i] && t < cu[i + 1]) {
            const int start = a.starts ? a.starts[i] : 0;
            if (start >= 0) pos = start + t - cu[i];
        }
    }
    int page = -1;
    if (pos >= 0) {
        const int64_t at = pos >> a.table.log_page;
        if (at >= a.table.max_pages) {
            if (lane == 0) atomicOr(a.table.status, kv4::kBadLength);
        } else {
            page = a.table.pages[i * a.table.stride + at];
            if ((unsigned)page >= (unsigned)a.table.num_pages) {
                if (lane == 0) atomicOr(a.table.status, kv4::kBadPage);
                page = -1;
            }
        }
    }
    const int row = (int)(pos & ((1 << a.table.log_page) - 1));
    T *dst = static_cast<T *>(kv ? a.v : a.k) + b * a.o_sb + s * a.o_ss;
    for (int c = lane; c < a.Hk * CH; c += 32) {
        const int h = c / CH, ch = (c - h * CH) * 8;
        float x[8] = {};
        if (page >= 0) {
            const int64_t head = a.pool.head(page, kv, h);
            const float f = a.pool.scales[(head << (a.pool.log_page - 4)) + (row >> 4)];
            const uint2 w = *reinterpret_cast<const uint2 *>(a.pool.codes + ((head << a.pool.log_page) + row) * (32 * W) + ch);
            s8x4_to_f32(w.x, x);
            s8x4_to_f32(w.y, x + 4);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = (x[j] + 0.5f) * f;
        }
        store8(dst + h * a.o_sh + ch, a.vec, x);
    }
}

inline bool tokens_ok(int64_t B, int64_t S, int64_t T, const int *cu) {
    return S >= 0 && T >= 0 && (cu || T == B * S) && T <= 0x7fffffff;
}

}  // namespace
}  // namespace kv8
}  // namespace fc

using namespace fc;
using namespace fc::kv8;

extern "C" int fc_kv8_append(const void *q, int64_t q_sb, int64_t q_ss, int64_t q_sh, void *q_out, int64_t qo_sb,
                             int64_t qo_ss, int64_t qo_sh, int64_t Hq, const void *k, int64_t k_sb, int64_t k_ss,
                             int64_t k_sh, const void *v, int64_t v_sb, int64_t v_ss, int64_t v_sh, int dtype,
                             int64_t B, int64_t S, int64_t T, const int *cu_seqlens, const int *lengths,
                             const int *positions, const int *axes, int n_axes, const void *q_weight,
                             const void *k_weight, int w_dtype, float eps, const float *rotary, int64_t rotary_rows,
                             int rotary_dim, int interleaved, signed char *codes, float *scales, int64_t num_pages,
                             int64_t Hk, int64_t D, int64_t page_size, const int *page_table, int64_t table_stride,
                             int64_t max_pages, int *status, void *stream) {
    clear_error();
    int rc = check_pool("kv8_append", B, Hk, D, page_size, num_pages, max_pages, codes, scales, page_table, status);
    if (rc) return rc;
    if (!is_float_dtype(dtype)) { set_error("kv8_append: dtype must be fp32, bf16 or fp16"); return FC_EINVAL; }
    if (!tokens_ok(B, S, T, cu_seqlens) || Hq < 0 || Hq > 65535) {
        set_error("kv8_append: bad token counts");
        return FC_EINVAL;
    }
    if (T == 0 || (B == 0 && !cu_seqlens)) return FC_OK;
    if (!k || !v || (!lengths && B) || (Hq && (!q || !q_out))) { set_error("kv8_append: null pointer"); return FC_EINVAL; }
    if ((q_weight || k_weight) && !is_float_dtype(w_dtype)) {
        set_error("kv8_append: norm weights must be fp32, bf16 or fp16");
        return FC_EINVAL;
    }
    if (rotary) {
        if (rotary_dim < 16 || rotary_dim > D || rotary_dim % 16) {
            set_error("kv8_append: rotary dim %d is not a multiple of 16 up to the head dim", rotary_dim);
            return FC_EINVAL;
        }
        if (rotary_rows <= 0 || !aligned(rotary, 16)) {
            set_error("kv8_append: the rotary table must have rows and be 16-byte aligned");
            return FC_EINVAL;
        }
    }
    if (axes && (!positions || !rotary || n_axes < 1)) {
        set_error("kv8_append: axes go with a rotary table and positions for each of them");
        return FC_EINVAL;
    }
    if (Hq) {
        const int64_t nb = cu_seqlens ? 1 : B, ns = cu_seqlens ? T : S, size = dtype_size(dtype);
        const Rows out{q_out, qo_sb, qo_ss, qo_sh, Hq}, in{q, q_sb, q_ss, q_sh, Hq};
        if ((!same_rows(out, in, nb, ns) && rows_meet(out, in, nb, ns, D, size)) ||
            rows_meet(out, Rows{k, k_sb, k_ss, k_sh, Hk}, nb, ns, D, size) ||
            rows_meet(out, Rows{v, v_sb, v_ss, v_sh, Hk}, nb, ns, D, size)) {
            set_error("kv8_append: q_out overlaps an input (it may be q itself)");
            return FC_EINVAL;
        }
        if (rows_repeat(out, nb, ns)) { set_error("kv8_append: q_out has rows in one place"); return FC_EINVAL; }
    }
    AppendArgs a{};
    a.q = q; a.k = k; a.v = v; a.qo = q_out;
    a.q_sb = q_sb; a.q_ss = q_ss; a.q_sh = q_sh;
    a.qo_sb = qo_sb; a.qo_ss = qo_ss; a.qo_sh = qo_sh;
    a.k_sb = k_sb; a.k_ss = k_ss; a.k_sh = k_sh;
    a.v_sb = v_sb; a.v_ss = v_ss; a.v_sh = v_sh;
    a.T = T; a.S = cu_seqlens ? 0 : S;
    a.B = (int)B; a.Hq = (int)Hq; a.Hk = (int)Hk; a.D = (int)D;
    a.cu = cu_seqlens; a.lengths = lengths; a.positions = positions;
    a.axes = axes; a.n_axes = n_axes;
    a.qw = q_weight; a.kw = k_weight; a.w_dtype = w_dtype;
    a.eps = eps; a.inv_d = (float)(1.0 / (double)D);
    a.rotary = rotary; a.rotary_rows = rotary_rows; a.R = rotary ? rotary_dim : 0;
    a.interleaved = interleaved;
    a.pool = Pool{codes, scales, (int)Hk, ilog2(page_size)};
    a.table = Table{page_table, table_stride, (int)max_pages, (int)num_pages, ilog2(page_size), status};
    a.vec = (Hq && rows_aligned(q, dtype, q_sb, q_ss, q_sh) ? 1 : 0) |
            (Hq && rows_aligned(q_out, dtype, qo_sb, qo_ss, qo_sh) ? 2 : 0) |
            (rows_aligned(k, dtype, k_sb, k_ss, k_sh) ? 4 : 0) | (rows_aligned(v, dtype, v_sb, v_ss, v_sh) ? 8 : 0) |
            (aligned(q_weight, 16) && aligned(k_weight, 16) ? 16 : 0);
    // runs of 16 positions that n tokens can meet, wherever they begin: (n + 30) / 16
    a.per = (int)((S + 30) / 16);
    const int64_t slots = a.S ? B * a.per : B ? T / 16 + 2 * B : 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_dtype(dtype, [&](auto t) {
        return by_head_dim(D, [&](auto w) {
            using E = decltype(t);
            constexpr int W = decltype(w)::value, heads = kQPasses * Lay<W>::RP;
            a.q_units = (int)((Hq + heads - 1) / heads);
            const int64_t blocks = slots * Hk + (T * a.q_units + kThreads / 32 - 1) / (kThreads / 32);
            if (blocks > 0x7fffffff) {
                set_error("kv8_append: too many tokens for one call");
                return FC_ENOTSUP;
            }
            if (blocks == 0) return FC_OK;
            a.slots = (int)slots;
            append_kernel<E, W><<<(unsigned)blocks, kThreads, 0, st>>>(a);
            return check_launch("kv8_append");
        });
    });
}

extern "C" int fc_kv8_read(const signed char *codes, const float *scales, int64_t num_pages, int64_t Hk, int64_t D,
                           int64_t page_size, const int *page_table, int64_t table_stride, int64_t max_pages,
                           const int *starts, int64_t B, int64_t S, int64_t T, const int *cu_seqlens, void *k_out,
                           void *v_out, int dtype, int64_t o_sb, int64_t o_ss, int64_t o_sh, int *status,
                           void *stream) {
    clear_error();
    int rc = check_pool("kv8_read", B, Hk, D, page_size, num_pages, max_pages, codes, scales, page_table, status);
    if (rc) return rc;
    if (!is_float_dtype(dtype)) { set_error("kv8_read: dtype must be fp32, bf16 or fp16"); return FC_EINVAL; }
    if (!tokens_ok(B, S, T, cu_seqlens)) { set_error("kv8_read: bad token counts"); return FC_EINVAL; }
    if (T == 0 || (B == 0 && !cu_seqlens)) return FC_OK;
    if (!k_out || !v_out) { set_error("kv8_read: null pointer"); return FC_EINVAL; }
    ReadArgs a{};
    a.B = (int)B; a.Hk = (int)Hk; a.T = T; a.S = cu_seqlens ? 0 : S;
    a.starts = starts; a.cu = cu_seqlens; a.k = k_out; a.v = v_out;
    a.o_sb = o_sb; a.o_ss = o_ss; a.o_sh = o_sh;
    a.pool = Pool{const_cast<signed char *>(codes), const_cast<float *>(scales), (int)Hk, ilog2(page_size)};
    a.table = Table{page_table, table_stride, (int)max_pages, (int)num_pages, ilog2(page_size), status};
    a.vec = rows_aligned(k_out, dtype, o_sb, o_ss, o_sh) && rows_aligned(v_out, dtype, o_sb, o_ss, o_sh);
    const int64_t blocks = (2 * T + kThreads / 32 - 1) / (kThreads / 32);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_dtype(dtype, [&](auto t) {
        return by_head_dim(D, [&](auto w) {
            read_kernel<decltype(t), decltype(w)::value><<<(unsigned)blocks, kThreads, 0, st>>>(a);
            return check_launch("kv8_read");
        });
    });
}
