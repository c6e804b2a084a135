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
//
// 8191 packed tokens, 32/8 heads, D = 128, norm and three axes (188 MB with the angles): 50 us, 58 % of the
// copy rate, queries 28 us of them, keys and values 22; one token 3.2 us, a launch.  The latency of 24 warps'
// instructions and loads an SM (2.6 of 4 a cycle) is what is left.
#include "fc_kv8.cuh"

namespace fc {
namespace kv8 {
namespace {

constexpr int kThreads = 256;
constexpr int kQPasses = 4;  // passes of a query warp, at most: that many loads on their way in a lane

struct AppendArgs {
    const void *q, *k, *v;
    void *qo;
    int64_t q_sb, q_ss, q_sh, qo_sb, qo_ss, qo_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
    int64_t T, S;  // tokens in all; tokens of each sequence (0: ragged, by cu)
    int B, Hq, Hk, D, per, slots, q_units, q_passes, heads;  // per: runs of a sequence; q_units: warps of a token; heads: of a block
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

// A lane has 8 channels of a row; FULL, where the whole head turns by halves, 16: both channels of
// its pairs, so that none go from lane to lane.
template <int W, bool FULL> struct Lay {
    static constexpr int D = 32 * W, CH = FULL ? 2 : 1;
    static constexpr int LPR = FULL ? D / 16 : W == 2 ? 8 : W <= 4 ? 16 : 32;  // lanes of a row (of D = 96 and 192 some idle)
    static constexpr int RP = 32 / LPR;                                        // rows of a warp's pass
    static constexpr int HALF = FULL ? D / 2 : 0;                              // from a lane's first channels to its second ones
};

// 8 elements as they came.
template <typename T> struct Raw {
    uint4 w[sizeof(T) == 4 ? 2 : 1];
};

template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T *p, bool vec) {
    Raw<T> r;
    if (vec) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(Raw<T>) / 16); i++) r.w[i] = reinterpret_cast<const uint4 *>(p)[i];
    } else {
        using U = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
        const U *u = reinterpret_cast<const U *>(p);
        uint32_t *w = reinterpret_cast<uint32_t *>(&r);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(Raw<T>) / 4); i++) {
            if constexpr (sizeof(T) == 4) w[i] = u[i];
            else w[i] = u[2 * i] | (uint32_t)u[2 * i + 1] << 16;
        }
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void widen(const Raw<T> &r, float x[8]) {
    if constexpr (sizeof(T) == 4) {
        load_vec_f32<T, 4>(reinterpret_cast<const T *>(&r.w[0]), x);
        load_vec_f32<T, 4>(reinterpret_cast<const T *>(&r.w[1]), x + 4);
    } else {
        load_vec_f32<T, 8>(reinterpret_cast<const T *>(&r.w[0]), x);
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

template <int W, bool FULL>
__device__ __forceinline__ Place place_of(const AppendArgs &a, int lane) {
    const int ci = lane % Lay<W, FULL>::LPR, shift = a.R / 16;
    Place p;
    if constexpr (FULL) return Place{1, lane, ci * 8};
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
        widen(load_raw(static_cast<const T *>(w) + ch, a.vec & 16), x);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = load_as_f32(w, ch + i, a.w_dtype);
    }
}

// x r w of one head.  All lanes of the warp call it (those without channels hold zeros).
template <int W, bool FULL>
__device__ __forceinline__ void norm_row(float x[][8], const float w[][8], const AppendArgs &a) {
    using L = Lay<W, FULL>;
    float sum[L::CH];
#pragma unroll
    for (int c = 0; c < L::CH; c++) {
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; i++) s[i] = __fmul_rn(x[c][i], x[c][i]);
#pragma unroll
        for (int n = 4; n; n /= 2)
#pragma unroll
            for (int i = 0; i < n; i++) s[i] = __fadd_rn(s[2 * i], s[2 * i + 1]);
        sum[c] = s[0];
    }
    if constexpr (FULL) {
        // the two halves' sums: each lane of a pair goes on with one of them
        const bool up = threadIdx.x & 1;
        const float give = up ? sum[0] : sum[1], mine = up ? sum[1] : sum[0];
        float s = __fadd_rn(mine, __shfl_xor_sync(0xffffffffu, give, 1));
#pragma unroll
        for (int m = 2; m < L::LPR; m *= 2) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, m));
        sum[0] = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, 1));
    } else {
#pragma unroll
        for (int m = 1; m < L::LPR; m *= 2) sum[0] = __fadd_rn(sum[0], __shfl_xor_sync(0xffffffffu, sum[0], m));
    }
    const float r = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fmul_rn(sum[0], a.inv_d), a.eps)));
#pragma unroll
    for (int c = 0; c < L::CH; c++)
#pragma unroll
        for (int i = 0; i < 8; i++) x[c][i] = __fmul_rn(__fmul_rn(x[c][i], r), w[c][i]);
}

__device__ __forceinline__ float turn(float x, float c, float y, float s) {  // x c + y s
    return __fadd_rn(__fmul_rn(x, c), __fmul_rn(y, s));
}

// Rotation of one head.  All lanes of the warp call it.
template <bool FULL>
__device__ __forceinline__ void rotate_row(float x[][8], const Angles &g, const Place &p, const AppendArgs &a) {
    if constexpr (FULL) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float u = x[0][i], v = x[1][i];
            x[0][i] = turn(u, g.c[i], v, -g.s[i]);
            x[1][i] = turn(v, g.c[i], u, g.s[i]);
        }
    } else if (a.interleaved) {
        if (p.part) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float u = x[0][2 * i], v = x[0][2 * i + 1];
                x[0][2 * i] = turn(u, g.c[i], v, -g.s[i]);
                x[0][2 * i + 1] = turn(v, g.c[i], u, g.s[i]);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float y = __shfl_sync(0xffffffffu, x[0][i], p.lane);
            if (p.part) x[0][i] = turn(x[0][i], g.c[i], y, p.part == 1 ? -g.s[i] : g.s[i]);
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

// ... for n heads from h on: their tokens' angles are read once, and a head's rows while the one before it is
// worked on.
template <typename T, int W, bool FULL>
__device__ __forceinline__ void append_run(const AppendArgs &a, const Run &r, int page, int h, int n) {
    using L = Lay<W, FULL>;
    constexpr int PASSES = L::RP > 4 ? 1 : 4 / L::RP, CH = L::CH;
    __shared__ float tops[2][8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kv = warp >> 2;
    const int ch = lane % L::LPR * 8, row0 = (warp & 3) * 4 + lane / L::LPR;
    const bool lane_on = ch < L::D && lane / L::LPR < 4;
    const int in_page = (int)(r.pos & ((1 << a.pool.log_page) - 1));
    const int64_t head = a.pool.head(page, kv, h);
    signed char *codes = a.pool.codes + ((head << a.pool.log_page) + in_page) * L::D + ch;
    float *scale = a.pool.scales + (head << (a.pool.log_page - 4)) + (in_page >> 4);
    const int held = (int)max((int64_t)0, r.lo - r.pos);
    const int64_t sb = kv ? a.v_sb : a.k_sb, ss = kv ? a.v_ss : a.k_ss, sh = kv ? a.v_sh : a.k_sh;
    const T *src[PASSES];
    bool on[PASSES];
    Raw<T> raw[PASSES][CH];
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
        const int64_t pos = r.pos + row0 + i * L::RP, t = r.t0 + pos;
        on[i] = pos >= r.lo && pos < r.hi && lane_on;
        const int64_t b = on[i] && a.S ? t / a.S : 0;
        src[i] = static_cast<const T *>(kv ? a.v : a.k) + b * sb + (a.S ? t - b * a.S : t) * ss + h * sh + ch;
    }
    auto load = [&] {
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            if (on[i])
#pragma unroll
                for (int c = 0; c < CH; c++) raw[i][c] = load_raw(src[i] + c * L::HALF, a.vec & (kv ? 8 : 4));
            src[i] += sh;
        }
    };
    load();
    float old = held ? *scale : 0.f;
    float w[CH][8] = {};
    const Place p = place_of<W, FULL>(a, lane);
    Angles g[PASSES];
    if (kv == 0) {
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const int64_t pos = r.pos + row0 + i * L::RP;
#pragma unroll
            for (int j = 0; j < 8; j++) g[i].c[j] = g[i].s[j] = 0.f;
            if (a.R && on[i]) load_angles(g[i], a, p, r.t0 + pos, pos);
        }
#pragma unroll
        for (int c = 0; c < CH; c++) load_weights<T>(a, a.kw, ch + c * L::HALF, lane_on, w[c]);
    }
    for (int y = 0; y < n; y++) {
        float x[PASSES][CH][8];
#pragma unroll
        for (int i = 0; i < PASSES; i++)
#pragma unroll
            for (int c = 0; c < CH; c++) {
                if (on[i]) {
                    widen(raw[i][c], x[i][c]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) x[i][c][j] = 0.f;
                }
            }
        float next = 0.f;
        if (y + 1 < n) {
            load();
            if (held) next = scale[(int64_t)1 << (a.pool.log_page - 4)];
        }
        if (kv == 0) {
#pragma unroll
            for (int i = 0; i < PASSES; i++) {
                if (a.kw) norm_row<W, FULL>(x[i], w, a);
                if (a.R) rotate_row<FULL>(x[i], g[i], p, a);
            }
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < PASSES; i++)
            if (on[i])
#pragma unroll
                for (int c = 0; c < CH; c++)
#pragma unroll
                    for (int j = 0; j < 8; j++) top = max_nan(top, fabsf(x[i][c][j]));
#pragma unroll
        for (int m = 1; m < 32; m *= 2) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, m));
        float *z = tops[y & 1];  // (who writes to it the next time has met the others once more)
        if (lane == 0) z[warp] = top;
        if (kv) asm volatile("bar.sync 2, 128;" ::: "memory");  // the 4 warps of the values,
        else asm volatile("bar.sync 1, 128;" ::: "memory");     // or of the keys
        top = max_nan(max_nan(z[4 * kv], z[4 * kv + 1]), max_nan(z[4 * kv + 2], z[4 * kv + 3]));
        // biased exponents: 0 no value but zero, 255 no number
        const int e_old = (int)(__float_as_uint(old) >> 23) & 255;
        const int e = max(e_old, top == top ? scale_exponent(top) : 255);
        const float inv = e == 0 || e == 255 ? 0.f : __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
        for (int i = 0; i < PASSES; i++) {
            const int row = row0 + i * L::RP;
#pragma unroll
            for (int k = 0; k < CH; k++) {
                signed char *at = codes + (int64_t)row * L::D + k * L::HALF;
                if (on[i]) {
                    uint32_t c[8];
                    // x / scale + 1.5 * 2^23 rounded down: its low byte is the floor
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        c[j] = inv > 0.f ? __float_as_uint(__fmaf_rd(x[i][k][j], inv, 12582912.f)) : 0u;
                    uint2 v;
                    v.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
                    v.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
                    *reinterpret_cast<uint2 *>(at) = v;
                } else if (row < held && lane_on && e_old && e > e_old && e < 255) {
                    uint2 v = *reinterpret_cast<uint2 *>(at);
                    v.x = shift_codes(v.x, e - e_old);
                    v.y = shift_codes(v.y, e - e_old);
                    *reinterpret_cast<uint2 *>(at) = v;
                }
            }
        }
        if ((warp & 3) == 0 && lane == 0) *scale = __uint_as_float(e == 255 ? 0x7fc00000u : (uint32_t)e << 23);
        codes += (int64_t)L::D << a.pool.log_page;
        scale += (int64_t)1 << (a.pool.log_page - 4);
        old = next;
    }
}

// A slot's sequence, and which of its runs of 16 positions: of B sequences of S tokens, `per` runs
// each, or by cu.  False: none.
struct Slot {
    int b, k;
    int64_t c0, n, i0, i1;  // first row and tokens of the sequence; those of them that have a row
};

__device__ __forceinline__ bool find_slot(Slot &x, int slot, int B, int64_t S, int64_t T, int per, const int *cu, int *status) {
    if (S) {
        x.b = slot / per;
        x.k = slot - x.b * per;
        x.c0 = (int64_t)x.b * S;
        x.n = S;
    } else {
        // a sequence of n tokens has at most n / 16 + 2 runs: slots from cu / 16 + 2 b on are its own
        x.b = warp_find([=](int i) { return (int64_t)(cu[i] >> 4) + 2 * i; }, B, slot);
        x.c0 = cu[x.b];
        x.k = slot - (int)((x.c0 >> 4) + 2 * x.b);
        x.n = cu[x.b + 1] - x.c0;
        if (x.k < 0) return false;
    }
    // tokens without a row are skipped
    x.i0 = 0;
    x.i1 = x.n;
    if (x.c0 < 0 || x.c0 + x.n > T) {
        if (threadIdx.x == 0) atomicOr(status, kv4::kBadLength);
        x.i0 = max((int64_t)0, -x.c0);
        x.i1 = min(x.n, T - x.c0);
    }
    return true;
}

// The run's positions, for a sequence whose tokens begin at position `start`.
__device__ __forceinline__ bool run_of(Run &r, const Slot &x, int start) {
    r.pos = (int64_t)((start >> 4) + x.k) << 4;
    r.lo = max(r.pos, start + x.i0);
    r.hi = min(r.pos + kBlock, start + x.i1);
    r.t0 = x.c0 - start;
    return r.lo < r.hi;
}

// The page of a run, or -1, noted in status.
__device__ __forceinline__ int page_of(const Table &t, int b, int64_t pos) {
    const int64_t i = pos >> t.log_page;
    if (i >= t.max_pages) {
        if (threadIdx.x == 0) atomicOr(t.status, kv4::kBadLength);
        return -1;
    }
    const int page = t.pages[b * t.stride + i];
    if ((unsigned)page < (unsigned)t.num_pages) return page;
    if (threadIdx.x == 0) atomicOr(t.status, kv4::kBadPage);
    return -1;
}

template <typename T, int W, bool FULL>
__device__ __forceinline__ void keys_and_values(const AppendArgs &a, int slot, int h) {
    Slot x;
    if (!find_slot(x, slot, a.B, a.S, a.T, a.per, a.cu, a.table.status)) return;
    const int len = a.lengths[x.b];
    Run r;
    if (len < 0 || !run_of(r, x, len)) return;
    const int page = page_of(a.table, x.b, r.pos);
    if (page >= 0) append_run<T, W, FULL>(a, r, page, h, min(a.heads, a.Hk - h));
}

// ------------------------------------------------------------------------- queries
// q_passes passes of heads of one token: its angles are read once.
template <typename T, int W, bool FULL>
__device__ __forceinline__ void queries(const AppendArgs &a, int64_t unit) {
    using L = Lay<W, FULL>;
    constexpr int CH = L::CH;
    const int64_t t = unit / a.q_units;
    if (t >= a.T) return;
    const int lane = threadIdx.x & 31, ch = lane % L::LPR * 8;
    const int h0 = (int)(unit - t * a.q_units) * a.q_passes * L::RP + lane / L::LPR;
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
    const T *src = static_cast<const T *>(a.q) + b * a.q_sb + s * a.q_ss + ch;
    T *dst = static_cast<T *>(a.qo) + b * a.qo_sb + s * a.qo_ss + ch;
    const bool lane_on = ch < L::D;
    Raw<T> raw[kQPasses][CH];
#pragma unroll
    for (int i = 0; i < kQPasses; i++) {
        const int h = h0 + i * L::RP;
        if (i < a.q_passes && lane_on && h < a.Hq && !none)
#pragma unroll
            for (int c = 0; c < CH; c++) raw[i][c] = load_raw(src + h * a.q_sh + c * L::HALF, a.vec & 1);
    }
    const Place p = place_of<W, FULL>(a, lane);
    Angles g;
    float w[CH][8] = {};
    if (!none) {
        if (a.R) load_angles(g, a, p, t, at);
#pragma unroll
        for (int c = 0; c < CH; c++) load_weights<T>(a, a.qw, ch + c * L::HALF, lane_on, w[c]);
    }
#pragma unroll
    for (int i = 0; i < kQPasses; i++) {
        if (i >= a.q_passes) break;
        const int h = h0 + i * L::RP;
        const bool on = lane_on && h < a.Hq;
        float x[CH][8];
#pragma unroll
        for (int c = 0; c < CH; c++) {
            if (on && !none) {
                widen(raw[i][c], x[c]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) x[c][j] = 0.f;
            }
        }
        if (!none) {
            if (a.qw) norm_row<W, FULL>(x, w, a);
            if (a.R) rotate_row<FULL>(x, g, p, a);
        }
        if (on)
#pragma unroll
            for (int c = 0; c < CH; c++) store8(dst + h * a.qo_sh + c * L::HALF, a.vec & 2, x[c]);
    }
}

template <typename T, int W, bool FULL>
__global__ void __launch_bounds__(kThreads, W <= 4 ? 3 : 2) append_kernel(const __grid_constant__ AppendArgs a) {
    const int parts = (a.Hk + a.heads - 1) / a.heads;
    const int64_t runs = (int64_t)a.slots * parts;
    if (blockIdx.x < runs) {
        const int slot = (int)(blockIdx.x / parts);
        keys_and_values<T, W, FULL>(a, slot, (int)(blockIdx.x - (int64_t)slot * parts) * a.heads);
    } else {
        queries<T, W, FULL>(a, ((int64_t)blockIdx.x - runs) * (kThreads / 32) + (threadIdx.x >> 5));
    }
}

// ---------------------------------------------------------------------------- read
struct ReadArgs {
    int B, Hk, per, slots;
    int64_t T, S;
    const int *starts, *cu;
    void *k, *v;
    int64_t o_sb, o_ss, o_sh;
    Pool pool;
    Table table;
    int vec;
};

// A warp reads the keys or the values of a head and run of 16 positions: 2 KB in a row at D = 128. 32000
// tokens of 8 heads, 197 MB, take 39 us, 78 % of the copy rate (a warp a token, whose heads lie a page apart: 45
// us).
template <typename T, int W>
__device__ __forceinline__ void read_run(const ReadArgs &a, int slot, int part) {
    constexpr int UNITS = 2 * W;  // 16 codes each, of a row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Slot x;
    if (!find_slot(x, slot, a.B, a.S, a.T, a.per, a.cu, a.table.status)) return;
    const int start = a.starts ? a.starts[x.b] : 0;
    Run r;
    if (!run_of(r, x, max(start, 0))) return;
    const int page = start < 0 ? -1 : page_of(a.table, x.b, r.pos);
    const int in_page = (int)(r.pos & ((1 << a.pool.log_page) - 1));
    const int64_t b = a.S ? x.b : 0, s0 = r.t0 + r.pos - b * a.S;  // the run's first row, if it is one
    const int u = part * (kThreads / 32) + warp;
    if (u < 2 * a.Hk) {
        const int kv = u >= a.Hk, h = u - kv * a.Hk;
        uint4 w[W];
        float f = 0.f;
        if (page >= 0) {
            const int64_t head = a.pool.head(page, kv, h);
            const uint4 *src = reinterpret_cast<const uint4 *>(a.pool.codes + ((head << a.pool.log_page) + in_page) * (32 * W));
            f = a.pool.scales[(head << (a.pool.log_page - 4)) + (in_page >> 4)];
#pragma unroll
            for (int y = 0; y < W; y++) w[y] = src[32 * y + lane];
        }
        T *dst = static_cast<T *>(kv ? a.v : a.k) + b * a.o_sb + s0 * a.o_ss + h * a.o_sh;
#pragma unroll
        for (int y = 0; y < W; y++) {
            const int row = (32 * y + lane) / UNITS, ch = (32 * y + lane - row * UNITS) * 16;
            if (r.pos + row < r.lo || r.pos + row >= r.hi) continue;
            float z[16] = {};
            if (page >= 0) {
                const uint32_t c[4] = {w[y].x, w[y].y, w[y].z, w[y].w};
#pragma unroll
                for (int i = 0; i < 4; i++) s8x4_to_f32(c[i], z + 4 * i);
#pragma unroll
                for (int i = 0; i < 16; i++) z[i] = (z[i] + 0.5f) * f;
            }
            store8(dst + row * a.o_ss + ch, a.vec, z);
            store8(dst + row * a.o_ss + ch + 8, a.vec, z + 8);
        }
    }
}

template <typename T, int W>
__global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ ReadArgs a) {
    const int parts = (2 * a.Hk + kThreads / 32 - 1) / (kThreads / 32), runs = a.slots * parts;
    if ((int)blockIdx.x < runs) {
        const int slot = blockIdx.x / parts;
        read_run<T, W>(a, slot, blockIdx.x - slot * parts);
        return;
    }
    // rows of no sequence: zeros
    const int64_t lo = a.B ? min(max((int64_t)a.cu[0], (int64_t)0), a.T) : a.T, hi = a.B ? min(max((int64_t)a.cu[a.B], lo), a.T) : a.T;
    const int64_t rows = lo + a.T - hi, warps = (int64_t)(gridDim.x - runs) * (kThreads / 32);
    for (int64_t i = (int64_t)(blockIdx.x - runs) * (kThreads / 32) + (threadIdx.x >> 5); i < rows; i += warps) {
        const int64_t at = (i < lo ? i : i - lo + hi) * a.o_ss;
        for (int c = threadIdx.x & 31; c < 2 * a.Hk * 4 * W; c += 32) {
            const int u = c / (4 * W), kv = u >= a.Hk;
            const float z[8] = {};
            store8(static_cast<T *>(kv ? a.v : a.k) + at + (u - kv * a.Hk) * a.o_sh + (c - u * 4 * W) * 8, a.vec, z);
        }
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
            constexpr int W = decltype(w)::value;
            auto launch = [&](auto full) {
                constexpr bool FULL = decltype(full)::value;
                constexpr int heads = Lay<W, FULL>::RP;  // of a pass
                // passes of a query warp: one where there are few tokens, more where there are enough for
                // 32 warps an SM
                const int64_t loads = (Hq + heads - 1) / heads, want = (32 * (int64_t)num_sms() + T - 1) / T;
                a.q_passes = (int)((loads + want - 1) / want);
                if (a.q_passes > kQPasses) a.q_passes = kQPasses;
                a.q_units = a.q_passes ? (int)((loads + a.q_passes - 1) / a.q_passes) : 0;
                // heads of a block: as many as leave 3 blocks an SM, up to 8 (8191 tokens, 8 heads: 67 us with
                // one, 57 with 2, 50 with 8; a single token: 4.1 us with 2, 3.2 with one)
                a.heads = 1;
                while (a.heads < 8 && slots * ((Hk + 2 * a.heads - 1) / (2 * a.heads)) >= 3 * (int64_t)num_sms()) a.heads *= 2;
                const int64_t blocks = slots * ((Hk + a.heads - 1) / a.heads) + (T * a.q_units + kThreads / 32 - 1) / (kThreads / 32);
                if (blocks > 0x7fffffff) {
                    set_error("kv8_append: too many tokens for one call");
                    return FC_ENOTSUP;
                }
                if (blocks == 0) return FC_OK;
                a.slots = (int)slots;
                append_kernel<E, W, FULL><<<(unsigned)blocks, kThreads, 0, st>>>(a);
                return check_launch("kv8_append");
            };
            if constexpr (W == 4 || W == 8) {
                if (rotary && rotary_dim == D && !interleaved) return launch(std::true_type());
            }
            return launch(std::false_type());
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
    a.per = (int)((S + 30) / 16);
    a.slots = (int)(a.S ? B * a.per : B ? T / 16 + 2 * B : 0);
    // (blocks for rows of no sequence)
    const int64_t rest = cu_seqlens ? (T + 63) / 64 < 32 ? (T + 63) / 64 : 32 : 0, blocks = a.slots * ((2 * Hk + 7) / 8) + rest;
    if (blocks > 0x7fffffff) { set_error("kv8_read: too many tokens for one call"); return FC_ENOTSUP; }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_dtype(dtype, [&](auto t) {
        return by_head_dim(D, [&](auto w) {
            read_kernel<decltype(t), decltype(w)::value><<<(unsigned)blocks, kThreads, 0, st>>>(a);
            return check_launch("kv8_read");
        });
    });
}
