// Paged 4-bit KV cache: append (head norms, rotary positions, quantisation and
// the page write in one launch) and read (the held values, gathered back).
//
// Append, for every new token (x a query or key head of D channels, fp32):
//   norm      y = x * r * w,  r = 1 / sqrt(mean(x^2) + eps), the sum of squares
//             as a tree over neighbours (pairs, fours, ...) so that its rounding
//             does not depend on the launch
//   rotation  (a, b) -> (a cos - b sin, b cos + a sin) for the pairs
//             (i, i + R/2) or (2 i, 2 i + 1) of the first R channels, cos and sin
//             from row `position` of the table
//   query     rounded to its type; key and value quantised (fc_kv4.cuh)
// Every product and sum is rounded by itself (no contraction), so codes, scales
// and bounds are the same bits for every way of splitting tokens into calls.
//
// The launch moves each input and output byte once.  8191 packed tokens of 32/8 heads of
// 128, bf16 (177 MB, 27.5 us at the copy rate), take 56 us: the queries 22 us, at the rate of
// memory, keys and values 32 us, bound by the latency of the instructions and loads of 16
// warps an SM (2.2 of 4 instructions a cycle).  A decode step's 64 tokens take 8.0 us, one
// 6.6: a chain of dependent loads.  Its blocks have two roles.  One block per (page that gets tokens, KV head) owns everything
// it writes: codes that share a word with older tokens and the page bounds are
// read, merged and written without atomics.  The other blocks take query heads,
// one warp for one token's heads.
#include "fc_kv4.cuh"

namespace fc {
namespace kv4 {
namespace {

// How a head lies over lanes: chunks of 8 channels, one in a lane, or, where the whole
// head turns by halves (FULL), two, D / 2 channels apart: then a lane holds both channels
// of its pairs and exchanges only sums, with half as many lanes.  (Two need a power of two
// of chunks, as the sum of squares goes by halves.)
template <int W, bool FULL>
struct Lay {
    static constexpr int CH = FULL ? 2 : 1, half = 4 * W / CH;
    static constexpr int LPT = half <= 4 ? 4 : half <= 8 ? 8 : half <= 16 ? 16 : 32;  // lanes of a head
    static constexpr int TPP = 32 / LPT;                                             // heads of a warp
};
constexpr bool can_be_full(int W) { return (W & (W - 1)) == 0; }

// 8 neighbouring channels of a head in one lane, as pairs for the paired fp32
// instructions: even channels (0, 2), (4, 6) and odd ones (1, 3), (5, 7).
struct Row {
    float2 e[2], o[2];
};

__device__ __forceinline__ float2 pair(float x, float y) { return make_float2(x, y); }

// A row as it is in memory: 8 elements of T.
template <typename T>
struct Raw {
    uint32_t w[2 * sizeof(T)];
};

template <typename T>
__device__ __forceinline__ Raw<T> load_raw(const T *p, bool vec) {
    Raw<T> r;
    if (vec) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
            r.w[4 * i] = v.x; r.w[4 * i + 1] = v.y; r.w[4 * i + 2] = v.z; r.w[4 * i + 3] = v.w;
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; i++) r.w[i] = reinterpret_cast<const uint32_t *>(p)[i];
    } else {
        const uint16_t *q = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
        for (int i = 0; i < 4; i++) r.w[i] = q[2 * i] | (uint32_t)q[2 * i + 1] << 16;
    }
    return r;
}

template <typename T>
__device__ __forceinline__ Raw<T> zero_raw() {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < 2 * (int)sizeof(T); i++) r.w[i] = 0u;
    return r;
}

template <typename T>
__device__ __forceinline__ Row widen(const Raw<T> &r) {
    float x[8];
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __uint_as_float(r.w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x[2 * i] = __uint_as_float(r.w[i] << 16);
            x[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r.w[i]));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
    return Row{{pair(x[0], x[2]), pair(x[4], x[6])}, {pair(x[1], x[3]), pair(x[5], x[7])}};
}

template <typename T>
__device__ __forceinline__ void store_row(T *p, bool vec, const Row &x) {
    const float y[8] = {x.e[0].x, x.o[0].x, x.e[0].y, x.o[0].y, x.e[1].x, x.o[1].x, x.e[1].y, x.o[1].y};
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 8; i++) store_from_f32(p, i, Elem<T>::code, y[i]);
    } else if constexpr (sizeof(T) == 4) {
        store_vec_from_f32<T, 4>(p, y);
        store_vec_from_f32<T, 4>(p + 4, y + 4);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(y[2 * i], y[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&h);
            }
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

struct AppendArgs {
    const void *q, *k, *v;
    void *qo;
    int64_t q_sb, q_ss, q_sh, qo_sb, qo_ss, qo_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
    int64_t T, S;                    // tokens in all; tokens of each sequence (0: ragged, by cu)
    int B, Hq, Hk, D;
    const int *cu, *lengths, *positions;
    const void *qw, *kw;
    int w_dtype;
    float eps, inv_d;
    const float *rotary;
    int64_t rotary_rows;
    int R, interleaved, norm_q, norm_k;
    unsigned char *pool;
    Table table;
    signed char *bounds;
    int *exps;
    int vec;                         // 1 q, 2 q_out, 4 k, 8 v, 16 weights: rows on 16-byte boundaries
    int slots;                       // page slots; blocks < slots * Hk write the cache
    int q_units, q_heads;            // warps of a token, heads of each
};

// Cosines and sines of a lane's channels.  Halves: c.e, c.o and s.e, s.o as the
// channels, the sines negative in the first half (not where a lane has both halves);
// pairs: c.e and s.e for the four pairs.
struct Angles {
    Row c, s;
};

// What the place of a chunk in the head makes of the rotation: 0 outside of it, 1 and 2
// the halves, 3 pairs; the lane of the other half; where its angles are in the table's row.
struct Place {
    int part, lane, index;
};

template <int W, bool FULL>
__device__ __forceinline__ Place place_of(const AppendArgs &a, int lane) {
    const int ci = lane % Lay<W, FULL>::LPT, shift = a.R / 16;
    Place p;
    p.part = ci * 8 >= a.R ? 0 : a.interleaved ? 3 : FULL || ci < shift ? 1 : 2;
    p.lane = p.part == 1 ? lane + shift : p.part == 2 ? lane - shift : lane;
    p.index = p.part == 3 ? ci * 4 : (p.part == 2 ? ci - shift : ci) * 8;
    return p;
}

// Norm weights of chunk ci.
__device__ __forceinline__ Row load_weights(const AppendArgs &a, const void *w, int ci) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = w && ci * 8 < a.D ? load_as_f32(w, ci * 8 + i, a.w_dtype) : 0.f;
    return Row{{pair(x[0], x[2]), pair(x[4], x[6])}, {pair(x[1], x[3]), pair(x[5], x[7])}};
}

// ... in every pass: those of the tokens' own type come in whole words.
template <typename T>
__device__ __forceinline__ Row load_weights_again(const AppendArgs &a, const void *w, int ci) {
    if (a.w_dtype == Elem<T>::code && ci * 8 < a.D)
        return widen(load_raw(static_cast<const T *>(w) + ci * 8, a.vec & 16));
    return load_weights(a, w, ci);
}

template <bool FULL>
__device__ __forceinline__ void load_angles(Angles &t, const AppendArgs &a, const Place &p, int64_t pos) {
    if (p.part == 0) return;
    if (pos < 0 || pos >= a.rotary_rows) {
        atomicOr(a.table.status, kBadPosition);
        pos = pos < 0 ? 0 : a.rotary_rows - 1;
    }
    const float *row = a.rotary + pos * a.R + p.index;
    const float4 c = *reinterpret_cast<const float4 *>(row);
    const float4 s = *reinterpret_cast<const float4 *>(row + a.R / 2);
    if (!FULL && p.part == 3) {
        t.c.e[0] = pair(c.x, c.y);
        t.c.e[1] = pair(c.z, c.w);
        t.s.e[0] = pair(s.x, s.y);
        t.s.e[1] = pair(s.z, s.w);
    } else {
        const float4 d = *reinterpret_cast<const float4 *>(row + 4);
        const float4 u = *reinterpret_cast<const float4 *>(row + a.R / 2 + 4);
        const float2 g = !FULL && p.part == 1 ? pair(-1.f, -1.f) : pair(1.f, 1.f);
        t.c = Row{{pair(c.x, c.z), pair(d.x, d.z)}, {pair(c.y, c.w), pair(d.y, d.w)}};
        t.s = Row{{__fmul2_rn(pair(s.x, s.z), g), __fmul2_rn(pair(u.x, u.z), g)},
                  {__fmul2_rn(pair(s.y, s.w), g), __fmul2_rn(pair(u.y, u.w), g)}};
    }
}

// x c + y s, every operation rounded.  (The sums are scalar: the compiler joins paired
// products and paired sums into fused ones, whatever rounding they are written with.)
__device__ __forceinline__ float2 turn2(float2 x, float2 c, float2 y, float2 s) {
    const float2 u = __fmul2_rn(x, c), v = __fmul2_rn(y, s);
    return pair(__fadd_rn(u.x, v.x), __fadd_rn(u.y, v.y));
}

__device__ __forceinline__ float2 shfl2(float2 x, int from) {
    return pair(__shfl_sync(0xffffffffu, x.x, from), __shfl_sync(0xffffffffu, x.y, from));
}

// Sum of a lane's 8 squares: neighbours first, then pairs of them, then fours.
__device__ __forceinline__ float squares(const Row &x) {
    const float2 u = turn2(x.e[0], x.e[0], x.o[0], x.o[0]);
    const float2 v = turn2(x.e[1], x.e[1], x.o[1], x.o[1]);
    return __fadd_rn(__fadd_rn(u.x, u.y), __fadd_rn(v.x, v.y));
}

__device__ __forceinline__ float norm_factor(float ss, const AppendArgs &a) {
    return __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fmul_rn(ss, a.inv_d), a.eps)));
}

__device__ __forceinline__ void norm_row(Row &x, float r, const Row &w) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        x.e[i] = __fmul2_rn(__fmul2_rn(x.e[i], pair(r, r)), w.e[i]);
        x.o[i] = __fmul2_rn(__fmul2_rn(x.o[i], pair(r, r)), w.o[i]);
    }
}

// Norms of N heads; `w`: the lane's weights.  All lanes of the warp call it.  The lanes
// share the sums out while they add (the two halves of an exchange keep one half of them
// each), so that a lane sums, and takes the root of, one head.
template <int W, bool FULL, int N, typename Weights>
__device__ __forceinline__ void norm_rows(Row x[N][Lay<W, FULL>::CH], Weights w, const AppendArgs &a) {
    using L = Lay<W, FULL>;
    constexpr int V = N * L::CH;
    static_assert(V <= L::LPT && (V & (V - 1)) == 0, "every lane ends with one sum");
    const int lane = threadIdx.x & 31;
    float s[V];  // sum k N + p: chunk k of head p
#pragma unroll
    for (int k = 0; k < L::CH; k++)
#pragma unroll
        for (int p = 0; p < N; p++) s[k * N + p] = squares(x[p][k]);
    int n = V;  // sums this lane still adds
#pragma unroll
    for (int m = 1; m < L::LPT; m *= 2) {
        if (n > 1) {
            const bool up = lane & m;
            n /= 2;
#pragma unroll
            for (int i = 0; i < V / 2; i++) {
                if (i >= n) break;
                const float give = up ? s[i] : s[i + n], mine = up ? s[i + n] : s[i];
                s[i] = __fadd_rn(mine, __shfl_xor_sync(0xffffffffu, give, m));
            }
        } else {
            s[0] = __fadd_rn(s[0], __shfl_xor_sync(0xffffffffu, s[0], m));
        }
    }
    // the first halving was by chunk
    if constexpr (L::CH == 2) s[0] = __fadd_rn(s[0], __shfl_xor_sync(0xffffffffu, s[0], 1));
    const float r = norm_factor(s[0], a);
    // head p is with the lanes whose next bits, the last halving first, spell p
#pragma unroll
    for (int p = 0; p < N; p++) {
        int from = 0;
#pragma unroll
        for (int m = L::CH, h = N / 2; h; m *= 2, h /= 2) from += p & h ? m : 0;
        const float f = __shfl_sync(0xffffffffu, r, from, L::LPT);
#pragma unroll
        for (int k = 0; k < L::CH; k++) norm_row(x[p][k], f, w(k));
    }
}

// Rotation of one head.  All lanes of the warp call it.
template <int W, bool FULL>
__device__ __forceinline__ void rotate_row(Row x[Lay<W, FULL>::CH], const Angles &t, const Place &p,
                                           const AppendArgs &a) {
    if constexpr (FULL) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float2 e = x[0].e[i], o = x[0].o[i], u = x[1].e[i], v = x[1].o[i];
            const float2 s = t.s.e[i], r = t.s.o[i];
            x[0].e[i] = turn2(e, t.c.e[i], u, pair(-s.x, -s.y));
            x[0].o[i] = turn2(o, t.c.o[i], v, pair(-r.x, -r.y));
            x[1].e[i] = turn2(u, t.c.e[i], e, s);
            x[1].o[i] = turn2(v, t.c.o[i], o, r);
        }
    } else if (a.interleaved) {
        if (p.part == 3) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float2 e = x[0].e[i], o = x[0].o[i], s = t.s.e[i];
                x[0].e[i] = turn2(e, t.c.e[i], o, pair(-s.x, -s.y));
                x[0].o[i] = turn2(o, t.c.e[i], e, s);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float2 e = shfl2(x[0].e[i], p.lane), o = shfl2(x[0].o[i], p.lane);
            if (p.part) {
                x[0].e[i] = turn2(x[0].e[i], t.c.e[i], e, t.s.e[i]);
                x[0].o[i] = turn2(x[0].o[i], t.c.o[i], o, t.s.o[i]);
            }
        }
    }
}

__device__ __forceinline__ float max_nan(float x, float y) {  // a NaN stays
    float z;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(z) : "f"(x), "f"(y));
    return z;
}

__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Codes of a lane's 8 channels, left in x as whole numbers, and the scale of their group,
// which 4 lanes share; returns the word of the K layout: channel i in nibble
// (i >> 1) + 4 (i & 1).
//
// The code is rint(x / scale) of the rounded quotient.  Halves are common (a bf16 input and
// an fp16 scale have few bits: 1 in 700 quotients is one), so the quotient has to be right
// there: t = x * inv, inv about 1 / scale, is off by 2^-22; one Newton step for t * scale = x
// adds (x - t * scale) * inv, whose residual is exact, and leaves 2^-44, so that a half comes
// out as itself.  No other quotient comes out as a half: (c + 1/2) * scale has at most 15
// bits, its fp32 neighbours x differ from it by an ulp, and their quotients from the half by
// more than half an ulp times 1 + 2^-11.  Scales at either end of fp16's range, where codes
// would pass 7, and groups that are no numbers go the long way.
__device__ __forceinline__ uint32_t quantise(Row &x, __half &scale) {
    float top = max_nan(max_nan(fabsf(x.e[0].x), fabsf(x.e[0].y)), max_nan(fabsf(x.e[1].x), fabsf(x.e[1].y)));
    top = max_nan(top, max_nan(max_nan(fabsf(x.o[0].x), fabsf(x.o[0].y)), max_nan(fabsf(x.o[1].x), fabsf(x.o[1].y))));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const bool bad = !(top < INFINITY);
    scale = bad ? __ushort_as_half(0x7fff) : __float2half_rn(fminf(__fmul_rn(top, 1.f / 7.f), 65504.f));
    const float s = __half2float(scale);
    const float inv = s > 0.f ? rcp_fast(s) : 0.f;
    float2 y[4];
    const float2 inv2 = pair(inv, inv), up = pair(12582912.f, 12582912.f), down = pair(-12582912.f, -12582912.f);
    float2 *const z[4] = {&x.e[0], &x.e[1], &x.o[0], &x.o[1]};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float2 t = __fmul2_rn(*z[i], inv2);
        t = __ffma2_rn(__ffma2_rn(pair(-t.x, -t.y), pair(s, s), *z[i]), inv2, t);
        y[i] = __fadd2_rn(__fadd2_rn(t, up), down);  // to the nearest whole number, halves to even
    }
    if (!(top * inv <= 7.4f)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            y[i].x = bad ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(z[i]->x, s)), -7.f), 7.f);
            y[i].y = bad ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(z[i]->y, s)), -7.f), 7.f);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) *z[i] = y[i];
    // four codes (+8) as one number below 2^16, twice
    const float2 u = __ffma2_rn(x.e[1], pair(256.f, 256.f), x.e[0]);
    const float2 v = __ffma2_rn(x.o[1], pair(256.f, 256.f), x.o[0]);
    const float lo = fmaf(u.y, 16.f, u.x) + (8388608.f + 34952.f), hi = fmaf(v.y, 16.f, v.x) + (8388608.f + 34952.f);
    return __byte_perm(__float_as_uint(lo), __float_as_uint(hi), 0x5410);
}

template <typename T, int W, bool FULL>
__device__ __forceinline__ void write_page(const AppendArgs &a, unsigned char *smem) {
    using L = Lay<W, FULL>;
    constexpr int D = 32 * W, ROW = 4 * W + 4, CH = L::CH, LPT = L::LPT, TPP = L::TPP;  // TPP tokens a pass
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int g = lane / LPT, li = lane % LPT;
    const bool live = li < L::half;
    const int P = 1 << a.table.log_page;

    // the page slot: sequence b, its page-th page that gets new tokens
    const int slot = blockIdx.x / a.Hk, h = blockIdx.x % a.Hk;
    int b, n;
    int64_t first, t0;  // first page slot of b, its first token row
    if (a.S) {
        const int per = (int)((a.S + 2 * P - 2) >> a.table.log_page);
        b = slot / per;
        first = (int64_t)b * per;
        n = (int)a.S;
        t0 = 0;
    } else {
        const int *cu = a.cu;
        const int lp = a.table.log_page;
        b = warp_find([=](int i) { return (int64_t)(cu[i] >> lp) + 2 * i; }, a.B, slot);
        const int c0 = cu[b], c1 = cu[b + 1];
        first = (int64_t)(c0 >> lp) + 2 * b;
        n = max(0, (int)min((int64_t)c1, a.T) - max(0, c0));
        t0 = max(0, c0);
        if ((c0 < 0 || c1 > a.T) && threadIdx.x == 0) atomicOr(a.table.status, kBadLength);  // tokens that are not there
    }
    const int len = a.lengths[b];
    if (len < 0 || n <= 0 || slot < first) return;
    const int64_t end = (int64_t)len + n;
    const int64_t page = (len >> a.table.log_page) + (slot - first);  // of the sequence
    if (page << a.table.log_page >= end) return;
    if (page >= a.table.max_pages) {
        if (threadIdx.x == 0) atomicOr(a.table.status, kBadLength);
        return;
    }
    const int id = a.table.pages[b * a.table.stride + page];
    const int base = (int)page << a.table.log_page;  // position of the page's first token
    const int lo = max(len, base), hi = (int)min(end, (int64_t)base + P);

    const T *k0 = static_cast<const T *>(a.k) + b * (a.S ? a.k_sb : 0) + h * a.k_sh + li * 8;
    const T *v0 = static_cast<const T *>(a.v) + b * (a.S ? a.v_sb : 0) + h * a.v_sh + li * 8;
    const Place place = place_of<W, FULL>(a, lane);
    Raw<T> kr[CH], vr[CH];  // of the next pass
    // pass p of a tile at position tb: token p + g of it
    auto load = [&](int tb, int p) {
        const int t = tb + p + g;
        const bool on = live && t >= lo && t < hi;
        const int64_t row = t0 + (t - len);
#pragma unroll
        for (int k = 0; k < CH; k++) {
            kr[k] = on ? load_raw(k0 + row * a.k_ss + k * L::half * 8, a.vec & 4) : zero_raw<T>();
            vr[k] = on ? load_raw(v0 + row * a.v_ss + k * L::half * 8, a.vec & 8) : zero_raw<T>();
        }
    };
    // the first tile of this warp that gets tokens
    int tile = max(warp, (lo - base) / 16);
    tile += ((warp - tile) % warps + warps) % warps;
    if (tile < P / 16 && base + tile * 16 < hi) load(base + tile * 16, max(lo - base - tile * 16, 0) / TPP * TPP);

    if ((unsigned)id >= (unsigned)a.table.num_pages) {
        if (threadIdx.x == 0) atomicOr(a.table.status, kBadPage);
        return;
    }
    const int64_t record = (int64_t)id * a.Hk + h;
    unsigned char *tiles = a.pool + record * (P / 16) * tile_bytes(W);
    const bool older = lo > base;
    const int e0 = a.bounds && older ? a.exps[record] : -40;
    float2 mn[CH][4], mx[CH][4];
#pragma unroll
    for (int k = 0; k < CH; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            mn[k][i] = pair(INFINITY, INFINITY);
            mx[k][i] = pair(-INFINITY, -INFINITY);
        }

    uint32_t *stage = reinterpret_cast<uint32_t *>(smem) + warp * 16 * ROW;
    const int r = lane >> 2, c = lane & 3;
    for (; tile < P / 16 && base + tile * 16 < hi; tile += warps) {
        const int tb = base + tile * 16;  // position of the tile's first token
        const int tlo = max(lo, tb) - tb, thi = min(hi, tb + 16) - tb;
        unsigned char *out = tiles + (int64_t)tile * tile_bytes(W);
        uint32_t *vw = reinterpret_cast<uint32_t *>(out + v_off(W));
        for (int p = tlo / TPP * TPP; p < thi; p += TPP) {
            Row x[1][CH], y[CH];
#pragma unroll
            for (int k = 0; k < CH; k++) {
                x[0][k] = widen(kr[k]);
                y[k] = widen(vr[k]);
            }
            const int t = p + g;
            const bool on = live && t >= tlo && t < thi;
            if (p + TPP < thi)
                load(tb, p + TPP);
            else if (tile + warps < P / 16 && tb + 16 * warps < hi)
                load(tb + 16 * warps, 0);
            if (a.norm_k)
                norm_rows<W, FULL, 1>(x, [&](int k) { return load_weights_again<T>(a, a.kw, li + k * L::half); }, a);
            if (a.R) {
                Angles angles;
                if (on) {
                    const int64_t row = t0 + (tb + t - len);
                    const int64_t pos = a.positions ? (int64_t)a.positions[a.S ? b * a.S + row : row] : tb + t;
                    load_angles<FULL>(angles, a, place, pos);
                }
                rotate_row<W, FULL>(x[0], angles, place, a);
            }
#pragma unroll
            for (int k = 0; k < CH; k++) {
                __half ks, vs;
                const uint32_t kc = quantise(x[0][k], ks), vc = quantise(y[k], vs);
                if (on) {
                    const int ci = li + k * L::half, j = ci / 4, q = ci % 4;
                    reinterpret_cast<uint32_t *>(out)[t * 4 * W + q * W + j] = kc;
                    stage[t * ROW + ci] = vc;
                    if (q == 0) {
                        reinterpret_cast<__half *>(out + ks_off(W))[(2 * (t & 7) + (t >> 3)) * W + j] = ks;
                        reinterpret_cast<__half *>(out + vs_off(W))[4 * (((t & 7) >> 1) * W + j) +
                                                                    2 * (t >> 3) + (t & 1)] = vs;
                    }
                    if (a.bounds) {
                        const float s = __hisnan(ks) ? 0.f : __half2float(ks);  // no numbers: zeros
                        const Row &u = x[0][k];
                        const float2 z[4] = {__fmul2_rn(u.e[0], pair(s, s)), __fmul2_rn(u.e[1], pair(s, s)),
                                             __fmul2_rn(u.o[0], pair(s, s)), __fmul2_rn(u.o[1], pair(s, s))};
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            mn[k][i] = pair(fminf(mn[k][i].x, z[i].x), fminf(mn[k][i].y, z[i].y));
                            mx[k][i] = pair(fmaxf(mx[k][i].x, z[i].x), fmaxf(mx[k][i].y, z[i].y));
                        }
                    }
                }
            }
        }
        __syncwarp();
        // The V words of this lane: channels 16 m + r and + 8 of tokens 2c, 2c + 1, 2c + 8,
        // 2c + 9, turned from their place in the staged words to nibble x + 2 y + 4 e.
        uint32_t word[2 * W], mask = 0;
#pragma unroll
        for (int m = 0; m < 2 * W; m++) word[m] = 0u;
        const int from = (r >> 1) + 4 * (r & 1);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int tok = 2 * c + 8 * (u >> 1) + (u & 1), to = 2 * (u >> 1) + 4 * (u & 1);
            if (tok >= tlo && tok < thi) mask |= 0xffu << (4 * to);
            const uint4 *z = reinterpret_cast<const uint4 *>(stage + tok * ROW);
            const int s0 = 4 * (from - to), s1 = 4 * (from - to - 1);  // the funnel shifts take them mod 32
#pragma unroll
            for (int i = 0; i < W; i++) {
                const uint4 y = z[i];
                word[2 * i] |= (__funnelshift_r(y.x, y.x, s0) & (0x0fu << (4 * to))) |
                               (__funnelshift_r(y.y, y.y, s1) & (0xf0u << (4 * to)));
                word[2 * i + 1] |= (__funnelshift_r(y.z, y.z, s0) & (0x0fu << (4 * to))) |
                                   (__funnelshift_r(y.w, y.w, s1) & (0xf0u << (4 * to)));
            }
        }
        if (mask) {
#pragma unroll
            for (int m = 0; m < 2 * W; m++) {
                const int at = v_word<W>(m, lane);
                vw[at] = (word[m] & mask) | (tlo > 0 ? vw[at] & ~mask : 0u);  // older tokens share words
            }
        }
        __syncwarp();
    }

    if (a.bounds) {
        // the block's tokens: over the lanes that share channels, then over the warps
#pragma unroll
        for (int k = 0; k < CH; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int m = LPT; m < 32; m *= 2) {
                    const float2 u = shfl2(mn[k][i], lane ^ m), v = shfl2(mx[k][i], lane ^ m);
                    mn[k][i] = pair(fminf(mn[k][i].x, u.x), fminf(mn[k][i].y, u.y));
                    mx[k][i] = pair(fmaxf(mx[k][i].x, v.x), fmaxf(mx[k][i].y, v.y));
                }
        __syncthreads();
        float *lo_s = reinterpret_cast<float *>(smem), *hi_s = lo_s + warps * D;
        if (g == 0 && live) {
#pragma unroll
            for (int k = 0; k < CH; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {  // channels 0 2, 4 6, 1 3, 5 7
                    const int d = warp * D + (li + k * L::half) * 8 + (i & 1) * 4 + (i >> 1);
                    lo_s[d] = mn[k][i].x;
                    lo_s[d + 2] = mn[k][i].y;
                    hi_s[d] = mx[k][i].x;
                    hi_s[d + 2] = mx[k][i].y;
                }
        }
        __syncthreads();
        if (warp == 0) {
            signed char *out = a.bounds + record * 2 * D;
            float u[W], v[W], top = 0.f;
            int o0[W], o1[W];
#pragma unroll
            for (int i = 0; i < W; i++) {
                const int d = lane + 32 * i;
                o0[i] = older ? out[d] : 0;
                o1[i] = older ? out[D + d] : 0;
                u[i] = lo_s[d];
                v[i] = hi_s[d];
                for (int w = 1; w < warps; w++) {
                    u[i] = fminf(u[i], lo_s[w * D + d]);
                    v[i] = fmaxf(v[i], hi_s[w * D + d]);
                }
                top = fmaxf(top, fmaxf(fabsf(u[i]), fabsf(v[i])));
            }
#pragma unroll
            for (int m = 16; m; m /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
            const int e = max(bound_exponent(top, -40), e0);
            const float f = pow2f(-e);
#pragma unroll
            for (int i = 0; i < W; i++) {
                int x = (int)floorf(u[i] * f), y = (int)ceilf(v[i] * f);
                if (older) {
                    x = min(x, o0[i] >> min(e - e0, 31));
                    y = max(y, -(-o1[i] >> min(e - e0, 31)));
                }
                out[lane + 32 * i] = (signed char)x;
                out[D + lane + 32 * i] = (signed char)y;
            }
            if (lane == 0) a.exps[record] = e;
        }
    }
}

// Query heads: one warp for some heads of a token, kQPasses rows of lanes at a time, the
// next ones on their way while these are turned.
template <typename T, bool FULL>
constexpr int kQPasses = (sizeof(T) == 4 ? 2 : 4) / (FULL ? 2 : 1);

template <typename T, int W, bool FULL>
__device__ __forceinline__ void turn_queries(const AppendArgs &a) {
    using L = Lay<W, FULL>;
    constexpr int CH = L::CH, TPP = L::TPP, N = kQPasses<T, FULL>;
    const int lane = threadIdx.x & 31, g = lane / L::LPT, li = lane % L::LPT;
    const bool live = li < L::half;
    const int64_t unit = ((int64_t)blockIdx.x - (int64_t)a.slots * a.Hk) * (blockDim.x >> 5) +
                         (threadIdx.x >> 5);
    const int64_t t = (uint32_t)unit / (uint32_t)a.q_units;
    if (t >= a.T) return;
    int h = (int)((uint32_t)unit - (uint32_t)t * a.q_units) * a.q_heads + g;
    const int end = min(h - g + a.q_heads, a.Hq);
    int64_t b, row;
    bool none = false;  // a row of no sequence
    if (a.S) {
        b = (uint32_t)t / (uint32_t)a.S;
        row = t - b * a.S;
    } else {
        const int *cu = a.cu;
        b = warp_find([=](int i) { return (int64_t)cu[i]; }, a.B, t);
        row = t;
        none = a.B == 0 || t < cu[b] || t >= cu[b + 1];
    }
    const T *q = static_cast<const T *>(a.q) + (a.S ? b * a.q_sb : 0) + row * a.q_ss + li * 8;
    T *qo = static_cast<T *>(a.qo) + (a.S ? b * a.qo_sb : 0) + row * a.qo_ss + li * 8;
    Raw<T> raw[N][CH];
    auto load = [&](int h0) {
#pragma unroll
        for (int p = 0; p < N; p++)
#pragma unroll
            for (int k = 0; k < CH; k++)
                raw[p][k] = live && h0 + p * TPP < end
                                ? load_raw(q + (h0 + p * TPP) * a.q_sh + k * L::half * 8, a.vec & 1)
                                : zero_raw<T>();
    };
    load(h);
    if (none) {
        const float2 o = pair(0.f, 0.f);
        for (; live && h < end; h += TPP)
#pragma unroll
            for (int k = 0; k < CH; k++)
                store_row(qo + h * a.qo_sh + k * L::half * 8, a.vec & 2, Row{{o, o}, {o, o}});
        return;
    }
    const Place place = place_of<W, FULL>(a, lane);
    Row w[CH];
    Angles angles;
    int64_t pos = 0;
    if (a.R)
        pos = a.positions ? (int64_t)a.positions[t]
                          : (int64_t)max(0, a.lengths[b]) + (a.S ? row : t - a.cu[b]);
#pragma unroll
    for (int k = 0; k < CH; k++) w[k] = load_weights(a, a.norm_q ? a.qw : nullptr, li + k * L::half);
    if (a.R && live) load_angles<FULL>(angles, a, place, pos);
    for (; h - g < end; h += N * TPP) {
        Row x[N][CH];
#pragma unroll
        for (int p = 0; p < N; p++)
#pragma unroll
            for (int k = 0; k < CH; k++) x[p][k] = widen(raw[p][k]);
        if (h - g + N * TPP < end) load(h + N * TPP);
        if (a.norm_q) norm_rows<W, FULL, N>(x, [&](int k) { return w[k]; }, a);
#pragma unroll
        for (int p = 0; p < N; p++) {
            if (a.R) rotate_row<W, FULL>(x[p], angles, place, a);
            if (live && h + p * TPP < end) {
#pragma unroll
                for (int k = 0; k < CH; k++)
                    store_row(qo + (h + p * TPP) * a.qo_sh + k * L::half * 8, a.vec & 2, x[p][k]);
            }
        }
    }
}

template <typename T, int W, bool FULL>
__global__ void __launch_bounds__(256, 2) append_kernel(const __grid_constant__ AppendArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    if ((int64_t)blockIdx.x < (int64_t)a.slots * a.Hk)
        write_page<T, W, FULL>(a, smem);
    else
        turn_queries<T, W, FULL>(a);
}

// ------------------------------------------------------------------------ read
struct ReadArgs {
    const unsigned char *pool;
    Table table;
    const int *starts, *cu;
    int64_t T, S;
    int B, Hk, slots;
    void *k, *v;
    int64_t o_sb, o_ss, o_sh;  // of k and v
    int vec;
};

// Pairs of codes (+8, nibbles 0 and 4 of w) as exact fp16 codes.
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(w), "r"(0x000f000fu), "r"(0x64006400u));
    const __half2 z = __hadd2(*reinterpret_cast<__half2 *>(&y), __float2half2_rn(-1032.f));
    return *reinterpret_cast<const uint32_t *>(&z);
}

// 8 codes (fp16 pairs) times their scale, rounded to T, to p.
template <typename T>
__device__ __forceinline__ void store_codes(T *p, bool vec, const uint32_t c[4], __half scale) {
    const float s = __half2float(scale);
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&c[i]));
        x[2 * i] = f.x * s;  // exact
        x[2 * i + 1] = f.y * s;
    }
    store_row(p, vec, Row{{pair(x[0], x[2]), pair(x[4], x[6])}, {pair(x[1], x[3]), pair(x[5], x[7])}});
}

// One warp for 16 tokens (a tile) of one KV head: each byte of the tile is loaded once, in
// whole words; a lane turns a row's chunk c of W words into W runs of 8 channels, and the
// 8 value words that hold 8 channels of 4 tokens, by way of shared memory, into 4.  Bound by
// HBM, most of it the stores: 32,000 tokens of 8 x 128 in bf16 (168 MB) take 33 us, 79 % of the
// copy rate (39 us with a load for every code word and token).
template <typename T, int W>
__global__ void __launch_bounds__(128) read_kernel(const __grid_constant__ ReadArgs a) {
    __shared__ __align__(16) uint32_t values[4][64 * W];
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (unit >= (int64_t)a.slots * a.Hk) return;
    const int slot = (int)(unit / a.Hk), h = (int)(unit % a.Hk);
    T *ko = static_cast<T *>(a.k) + h * a.o_sh;
    T *vo = static_cast<T *>(a.v) + h * a.o_sh;
    auto clear = [&](int64_t row, int64_t end) {  // rows that nothing is read for
        const float2 o = pair(0.f, 0.f);
        const Row zero{{o, o}, {o, o}};
        const int n = (int)(end - row) * 4 * W;
        for (int u = lane; u < n; u += 32) {
            const int64_t at = (row + u / (4 * W)) * a.o_ss + u % (4 * W) * 8;
            store_row(ko + at, a.vec & 1, zero);
            store_row(vo + at, a.vec & 2, zero);
        }
    };
    int b, n;
    int64_t first, t0;
    if (a.S) {
        const int per = (int)((a.S + 30) / 16);
        b = slot / per;
        first = (int64_t)b * per;
        n = (int)a.S;
        t0 = 0;
        ko += b * a.o_sb;
        vo += b * a.o_sb;
    } else {
        const int *cu = a.cu;
        // slots before and behind the sequences' are for the rows of none
        const int64_t c0 = min((int64_t)max(cu[0], 0), a.T), cB = max(cu[a.B], 0);
        const int64_t behind = (cB >> 4) + 2 * a.B;
        if (slot < c0 >> 4) return clear((int64_t)slot * 16, (int64_t)slot * 16 + 16);
        if (slot == a.slots - 1) return clear(c0 & ~15, c0);
        if (slot >= behind) {
            const int64_t row = cB + (slot - behind) * 16;
            if (row < a.T) clear(row, min(row + 16, a.T));
            return;
        }
        b = warp_find([=](int i) { return (int64_t)(cu[i] >> 4) + 2 * i; }, a.B, slot);
        first = (int64_t)(cu[b] >> 4) + 2 * b;
        n = max(0, (int)min((int64_t)cu[b + 1], a.T) - max(0, cu[b]));
        t0 = max(0, cu[b]);
        if ((cu[b] < 0 || cu[b + 1] > a.T) && lane == 0) atomicOr(a.table.status, kBadLength);
    }
    int start = a.starts ? a.starts[b] : 0;
    const bool skipped = start < 0;
    if (skipped) start = 0;
    if (n <= 0 || slot < first) return;
    const int64_t tile64 = (start >> 4) + (slot - first), tb = tile64 * 16, end = (int64_t)start + n;
    if (tb >= end) return;
    const int lo = (int)(max((int64_t)start, tb) - tb), hi = (int)min(end - tb, (int64_t)16);
    const int64_t row0 = t0 + (tb - start);
    if (skipped) return clear(row0 + lo, row0 + hi);
    int bad = 0, id = 0;
    const int tpp = a.table.log_page - 4;
    const int64_t page = tile64 >> tpp;
    if (page >= a.table.max_pages) {
        bad = kBadLength;
    } else {
        id = a.table.pages[b * a.table.stride + page];
        if ((unsigned)id >= (unsigned)a.table.num_pages) bad = kBadPage;
    }
    if (bad) {
        if (lane == 0) atomicOr(a.table.status, bad);
        return clear(row0 + lo, row0 + hi);
    }
    const int tile = (int)tile64;
    const unsigned char *in = a.pool + ((((int64_t)id * a.Hk + h) << tpp) + (tile & ((1 << tpp) - 1))) *
                                           tile_bytes(W);
    // values: to shared memory while the keys are turned
    uint32_t *vs = values[threadIdx.x >> 5];
    {
        const uint4 *p = reinterpret_cast<const uint4 *>(in + v_off(W));
#pragma unroll
        for (int i = 0; i < (16 * W + 31) / 32; i++)
            if (32 * i + 31 < 16 * W || 32 * i + lane < 16 * W)
                reinterpret_cast<uint4 *>(vs)[32 * i + lane] = p[32 * i + lane];
    }
    const __half *ksc = reinterpret_cast<const __half *>(in + ks_off(W));
    const __half *vsc = reinterpret_cast<const __half *>(in + vs_off(W));
#pragma unroll
    for (int y = 0; y < 2; y++) {
        const int t = (lane >> 2) + 8 * y, c = lane & 3;
        if (t < lo || t >= hi) continue;
        const uint32_t *p = reinterpret_cast<const uint32_t *>(in) + (t * 4 + c) * W;
        T *out = ko + (row0 + t) * a.o_ss + 8 * c;
#pragma unroll
        for (int j = 0; j < W; j++) {
            // channels 0 1, 2 3, 4 5, 6 7 of the word: nibbles 0 4, 1 5, 2 6, 3 7
            const uint32_t w = p[j];
            const uint32_t z[4] = {codes2(w), codes2(w >> 4), codes2(w >> 8), codes2(w >> 12)};
            store_codes(out + 32 * j, a.vec & 1, z, ksc[(2 * (t & 7) + y) * W + j]);
        }
    }
    __syncwarp();
    // a lane's chunk li of 8 channels, for the tokens 2c, 2c + 1, 2c + 8, 2c + 9
    for (int u = lane; u < 16 * W; u += 32) {
        const int c = u & 3, li = u >> 2, m = li >> 1, x = li & 1;
        uint32_t z[2][8];  // [2c.., 2c+8..][channel]: codes of a pair of tokens
#pragma unroll
        for (int r = 0; r < 8; r++) {
            const uint32_t w = vs[v_word<W>(m, 4 * r + c)] >> (4 * x);
            z[0][r] = codes2(w);
            z[1][r] = codes2(w >> 8);
        }
        const __half *s = vsc + 4 * (c * W + li / 4);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int t = 2 * c + 8 * (k >> 1) + (k & 1);
            if (t < lo || t >= hi) continue;
            uint32_t q[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                q[i] = __byte_perm(z[k >> 1][2 * i], z[k >> 1][2 * i + 1], k & 1 ? 0x7632 : 0x5410);
            store_codes(vo + (row0 + t) * a.o_ss + li * 8, a.vec & 2, q, s[k]);
        }
    }
}

}  // namespace
}  // namespace kv4
}  // namespace fc

using namespace fc;
using namespace fc::kv4;

extern "C" int64_t fc_kv4_page_bytes(int64_t Hk, int64_t D, int64_t page_size) {
    clear_error();
    if (!head_dim_ok(D) || !page_size_ok(page_size) || Hk <= 0) {
        set_error("kv4_page_bytes: head dim 64, 96, 128, 192 or 256 and a page size that is a power of "
                  "two from 16 to 1024 are needed");
        return -1;
    }
    return Hk * (page_size / 16) * tile_bytes((int)(D / 32));
}

extern "C" int fc_kv4_append(const void *q, int64_t q_sb, int64_t q_ss, int64_t q_sh, void *q_out,
                             int64_t qo_sb, int64_t qo_ss, int64_t qo_sh, int64_t Hq,
                             const void *k, int64_t k_sb, int64_t k_ss, int64_t k_sh,
                             const void *v, int64_t v_sb, int64_t v_ss, int64_t v_sh, int dtype,
                             int64_t B, int64_t S, int64_t T, const int *cu_seqlens,
                             const int *lengths, const int *positions,
                             const void *q_weight, const void *k_weight, int w_dtype, float eps,
                             const float *rotary, int64_t rotary_rows, int rotary_dim,
                             int interleaved, void *pool, int64_t num_pages, int64_t Hk, int64_t D,
                             int64_t page_size, const int *page_table, int64_t table_stride,
                             int64_t max_pages, signed char *bounds, int *exponents, int *status,
                             void *stream) {
    clear_error();
    int rc = check_cache("kv4_append", B, Hk, D, page_size, num_pages, max_pages, pool, page_table, status);
    if (rc) return rc;
    if (!is_float_dtype(dtype)) { set_error("kv4_append: dtype must be fp32, bf16 or fp16"); return FC_EINVAL; }
    if (S < 0 || T < 0 || (cu_seqlens == nullptr && T != B * S) || T > 0x7fffffff || Hq < 0 || Hq > 65535) {
        set_error("kv4_append: bad token counts");
        return FC_EINVAL;
    }
    if (T == 0 || (B == 0 && !cu_seqlens)) return FC_OK;
    if (!k || !v || (!lengths && B) || (Hq && (!q || !q_out))) { set_error("kv4_append: null pointer"); return FC_EINVAL; }
    if ((bounds == nullptr) != (exponents == nullptr)) {
        set_error("kv4_append: bounds and their exponents go together");
        return FC_EINVAL;
    }
    if ((q_weight || k_weight) && !is_float_dtype(w_dtype)) {
        set_error("kv4_append: norm weights must be fp32, bf16 or fp16");
        return FC_EINVAL;
    }
    if (rotary) {
        if (rotary_dim < 16 || rotary_dim > D || rotary_dim % 16) {
            set_error("kv4_append: rotary dim %d is not a multiple of 16 up to the head dim", rotary_dim);
            return FC_EINVAL;
        }
        if (rotary_rows <= 0 || !aligned(rotary, 16)) {
            set_error("kv4_append: the rotary table must have rows and be 16-byte aligned");
            return FC_EINVAL;
        }
    }
    if (Hq) {
        const int64_t nb = cu_seqlens ? 1 : B, ns = cu_seqlens ? T : S, size = dtype_size(dtype);
        const Rows out{q_out, qo_sb, qo_ss, qo_sh, Hq};
        const Rows in{q, q_sb, q_ss, q_sh, Hq};
        if ((!same_rows(out, in, nb, ns) && rows_meet(out, in, nb, ns, D, size)) ||
            rows_meet(out, Rows{k, k_sb, k_ss, k_sh, Hk}, nb, ns, D, size) ||
            rows_meet(out, Rows{v, v_sb, v_ss, v_sh, Hk}, nb, ns, D, size)) {
            set_error("kv4_append: q_out overlaps an input (it may be q itself)");
            return FC_EINVAL;
        }
        if (rows_repeat(out, nb, ns)) { set_error("kv4_append: q_out has rows in one place"); return FC_EINVAL; }
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
    a.qw = q_weight; a.kw = k_weight; a.w_dtype = w_dtype;
    a.norm_q = q_weight != nullptr; a.norm_k = k_weight != nullptr;
    a.eps = eps; a.inv_d = (float)(1.0 / (double)D);
    a.rotary = rotary; a.rotary_rows = rotary_rows; a.R = rotary ? rotary_dim : 0;
    a.interleaved = interleaved;
    a.pool = static_cast<unsigned char *>(pool);
    a.table = Table{page_table, table_stride, (int)max_pages, (int)num_pages, ilog2(page_size), status};
    a.bounds = bounds; a.exps = exponents;
    a.vec = (Hq && rows_aligned(q, dtype, q_sb, q_ss, q_sh) ? 1 : 0) |
            (Hq && rows_aligned(q_out, dtype, qo_sb, qo_ss, qo_sh) ? 2 : 0) |
            (rows_aligned(k, dtype, k_sb, k_ss, k_sh) ? 4 : 0) |
            (rows_aligned(v, dtype, v_sb, v_ss, v_sh) ? 8 : 0) |
            (aligned(q_weight, 16) && aligned(k_weight, 16) ? 16 : 0);
    const int64_t slots = a.S ? B * ((S + 2 * page_size - 2) / page_size) : B ? T / page_size + 2 * B : 0;
    const int warps = (int)(page_size / 16 < 8 ? page_size / 16 : 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_dtype(dtype, [&](auto t) {
        return by_head_dim(D, [&](auto w) {
            using E = decltype(t);
            constexpr int W = decltype(w)::value;
            a.slots = (int)slots;
            auto launch = [&](auto full) {
                constexpr bool FULL = decltype(full)::value;
                // heads of a query warp: all of a token's where there are tokens enough for
                // 32 warps an SM, else fewer, down to one load's worth
                constexpr int per = kQPasses<E, FULL> * Lay<W, FULL>::TPP;
                const int64_t loads = (Hq + per - 1) / per, want = (32 * (int64_t)num_sms() + T - 1) / T;
                a.q_heads = (int)(per * ((loads + want - 1) / want));
                a.q_units = a.q_heads ? (int)((Hq + a.q_heads - 1) / a.q_heads) : 0;
                const int64_t blocks = slots * Hk + (T * a.q_units + warps - 1) / warps;
                if (slots * Hk > 0x7fffffff || blocks * warps > 0x7fffffff) {
                    set_error("kv4_append: too many tokens for one call");
                    return FC_ENOTSUP;
                }
                if (blocks == 0) return FC_OK;
                const size_t stage = (size_t)warps * 16 * (4 * W + 4) * 4, red = (size_t)warps * 32 * W * 8;
                append_kernel<E, W, FULL><<<(unsigned)blocks, warps * 32, stage > red ? stage : red, st>>>(a);
                return check_launch("kv4_append");
            };
            if constexpr (can_be_full(W)) {
                if (a.R == D && !interleaved) return launch(std::true_type());
            }
            return launch(std::false_type());
        });
    });
}

extern "C" int fc_kv4_read(const void *pool, int64_t num_pages, int64_t Hk, int64_t D,
                           int64_t page_size, const int *page_table, int64_t table_stride,
                           int64_t max_pages, const int *starts, int64_t B, int64_t S, int64_t T,
                           const int *cu_seqlens, void *k_out, void *v_out, int dtype, int64_t o_sb,
                           int64_t o_ss, int64_t o_sh, int *status, void *stream) {
    clear_error();
    int rc = check_cache("kv4_read", B, Hk, D, page_size, num_pages, max_pages, pool, page_table, status);
    if (rc) return rc;
    if (!is_float_dtype(dtype)) { set_error("kv4_read: dtype must be fp32, bf16 or fp16"); return FC_EINVAL; }
    if (S < 0 || T < 0 || (cu_seqlens == nullptr && T != B * S) || T > 0x7fffffff) {
        set_error("kv4_read: bad token counts");
        return FC_EINVAL;
    }
    if (T == 0 || (B == 0 && !cu_seqlens)) return FC_OK;
    if (!k_out || !v_out) { set_error("kv4_read: null pointer"); return FC_EINVAL; }
    ReadArgs a{};
    a.pool = static_cast<const unsigned char *>(pool);
    a.table = Table{page_table, table_stride, (int)max_pages, (int)num_pages, ilog2(page_size), status};
    a.starts = starts; a.cu = cu_seqlens;
    a.T = T; a.S = cu_seqlens ? 0 : S;
    a.B = (int)B; a.Hk = (int)Hk;
    a.k = k_out; a.v = v_out; a.o_sb = o_sb; a.o_ss = o_ss; a.o_sh = o_sh;
    a.vec = (rows_aligned(k_out, dtype, o_sb, o_ss, o_sh) ? 1 : 0) |
            (rows_aligned(v_out, dtype, o_sb, o_ss, o_sh) ? 2 : 0);
    const int64_t slots = a.S ? B * ((S + 30) / 16) : T / 16 + 2 * B + 2;
    const int64_t blocks = (slots * Hk + 3) / 4;
    if (slots > 0x7fffffff || blocks > 0x7fffffff) {
        set_error("kv4_read: too many tokens for one call");
        return FC_ENOTSUP;
    }
    a.slots = (int)slots;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_dtype(dtype, [&](auto t) {
        return by_head_dim(D, [&](auto w) {
            read_kernel<decltype(t), decltype(w)::value><<<(unsigned)blocks, 128, 0, st>>>(a);
            return check_launch("kv4_read");
        });
    });
}
