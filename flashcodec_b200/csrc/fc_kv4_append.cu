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
// The launch moves each input and output byte once and is bound by HBM for long
// prompts (queries are most of it) and by latency for a decode step.  Its blocks
// have two roles.  One block per (page that gets tokens, KV head) owns everything
// it writes: codes that share a word with older tokens and the page bounds are
// read, merged and written without atomics.  The other blocks take query heads,
// one warp for one token's heads.
#include "fc_kv4.cuh"

namespace fc {
namespace kv4 {
namespace {

template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, float x[8]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            load_vec_f32<T, 4>(p, x);
            load_vec_f32<T, 4>(p + 4, x + 4);
        } else {
            load_vec_f32<T, 8>(p, x);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = Elem<T>::to_f32(p[i]);
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *p, bool vec, const float x[8]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            store_vec_from_f32<T, 4>(p, x);
            store_vec_from_f32<T, 4>(p + 4, x + 4);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if constexpr (std::is_same<T, __half>::value) {
                    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
                    w[i] = *reinterpret_cast<const uint32_t *>(&h);
                } else {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
                    w[i] = *reinterpret_cast<const uint32_t *>(&h);
                }
            }
            *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) store_from_f32(p, i, Elem<T>::code, x[i]);
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
    int vec;                         // 1 q, 2 q_out, 4 k, 8 v: rows on 16-byte boundaries
    int slots;                       // page slots; blocks < slots * Hk write the cache
    int q_units;                     // head chunks of one token
};

// What a lane needs to norm and rotate its 8 channels of a head.
struct Turn {
    float w[8], c[8], s[8];
    int part;   // rotary halves: 0 outside, 1 first half, 2 second half, 3 pairs
    int shift;  // lanes to the partner half
};

template <int LPT>
__device__ __forceinline__ void turn_weights(Turn &t, const AppendArgs &a, const void *w, int li) {
#pragma unroll
    for (int i = 0; i < 8; i++)
        t.w[i] = w && li * 8 < a.D ? load_as_f32(w, li * 8 + i, a.w_dtype) : 0.f;
    const int d = li * 8;
    t.shift = a.R / 16;
    t.part = d >= a.R ? 0 : a.interleaved ? 3 : li < t.shift ? 1 : 2;
}

__device__ __forceinline__ void turn_angles(Turn &t, const AppendArgs &a, int li, int64_t pos) {
    if (t.part == 0) return;
    if (pos < 0 || pos >= a.rotary_rows) {
        atomicOr(a.table.status, kBadPosition);
        pos = pos < 0 ? 0 : a.rotary_rows - 1;
    }
    const float *row = a.rotary + pos * a.R;
    if (t.part == 3) {
        const float4 c = *reinterpret_cast<const float4 *>(row + li * 4);
        const float4 s = *reinterpret_cast<const float4 *>(row + a.R / 2 + li * 4);
        t.c[0] = c.x; t.c[1] = c.y; t.c[2] = c.z; t.c[3] = c.w;
        t.s[0] = s.x; t.s[1] = s.y; t.s[2] = s.z; t.s[3] = s.w;
    } else {
        const int i = (t.part == 1 ? li : li - t.shift) * 8;
        load_vec_f32<float, 4>(row + i, t.c);
        load_vec_f32<float, 4>(row + i + 4, t.c + 4);
        load_vec_f32<float, 4>(row + a.R / 2 + i, t.s);
        load_vec_f32<float, 4>(row + a.R / 2 + i + 4, t.s + 4);
    }
}

// Norm and rotation of one head held by LPT lanes (8 channels each).  All lanes
// of the warp call it.
template <int LPT>
__device__ __forceinline__ void turn_row(float x[8], const Turn &t, bool norm, float inv_d, float eps) {
    if (norm) {
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; i++) s[i] = __fmul_rn(x[i], x[i]);
        float ss = __fadd_rn(__fadd_rn(__fadd_rn(s[0], s[1]), __fadd_rn(s[2], s[3])),
                             __fadd_rn(__fadd_rn(s[4], s[5]), __fadd_rn(s[6], s[7])));
#pragma unroll
        for (int m = 1; m < LPT; m *= 2) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, m));
        const float r = __fdiv_rn(1.f, __fsqrt_rn(__fadd_rn(__fmul_rn(ss, inv_d), eps)));
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = __fmul_rn(__fmul_rn(x[i], r), t.w[i]);
    }
    if (t.shift == 0) return;  // no rotation (uniform over the launch)
    const int lane = threadIdx.x & 31;
    const int from = t.part == 1 ? lane + t.shift : t.part == 2 ? lane - t.shift : lane;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = __shfl_sync(0xffffffffu, x[i], from);
    if (t.part == 3) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float u = x[2 * i], v = x[2 * i + 1];
            x[2 * i] = __fsub_rn(__fmul_rn(u, t.c[i]), __fmul_rn(v, t.s[i]));
            x[2 * i + 1] = __fadd_rn(__fmul_rn(v, t.c[i]), __fmul_rn(u, t.s[i]));
        }
    } else if (t.part == 1) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            x[i] = __fsub_rn(__fmul_rn(x[i], t.c[i]), __fmul_rn(y[i], t.s[i]));
    } else if (t.part == 2) {
#pragma unroll
        for (int i = 0; i < 8; i++)
            x[i] = __fadd_rn(__fmul_rn(x[i], t.c[i]), __fmul_rn(y[i], t.s[i]));
    }
}

// Codes (+8, one per byte) of a lane's 8 channels and the scale of their group,
// which the 4 lanes of the group share.  x / scale is taken as a product with
// 1 / scale; only where that is within 1e-5 of a half (its error is under 2e-6)
// does the division itself decide, so the codes are those of rint(x / scale).
__device__ __forceinline__ void quantise8(const float x[8], uint32_t code[2], __half &scale) {
    uint32_t top = 0;  // of the bit patterns: a NaN is above an infinity is above a number
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const bool bad = top >= 0x7f800000u;
    scale = __float2half_rn(fminf(__fmul_rn(__uint_as_float(top), 1.f / 7.f), 65504.f));
    const float s = __half2float(scale);
    if (bad) scale = __ushort_as_half(0x7fff);
    const float inv = bad || !(s > 0.f) ? 0.f : 1.f / s;
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float t = x[i] * inv;
        float n = rintf(t);
        if (fabsf(fabsf(t - n) - 0.5f) < 1e-5f) n = rintf(__fdiv_rn(x[i], s));
        n = fminf(fmaxf(n, -7.f), 7.f);
        c[i] = bad ? 8u : (uint32_t)((int)n + 8);
    }
    code[0] = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
    code[1] = c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24;
}

// 8 codes in bytes -> the K word: channel i in nibble (i >> 1) + 4 (i & 1)
__device__ __forceinline__ uint32_t pack_k(const uint32_t code[2]) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; i++)
        w |= ((code[i >> 2] >> (8 * (i & 3))) & 15u) << (4 * ((i >> 1) + 4 * (i & 1)));
    return w;
}

template <typename T, int W, int LPT>
__device__ __forceinline__ void write_page(const AppendArgs &a, unsigned char *smem) {
    constexpr int D = 32 * W, ROW = D + 8, TPP = 32 / LPT;  // tokens of a pass
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int g = lane / LPT, li = lane % LPT;
    const bool live = li * 8 < D;
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
        first = (int64_t)(cu[b] >> lp) + 2 * b;
        n = max(0, (int)min((int64_t)cu[b + 1], a.T) - max(0, cu[b]));
        t0 = max(0, cu[b]);
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
    if ((unsigned)id >= (unsigned)a.table.num_pages) {
        if (threadIdx.x == 0) atomicOr(a.table.status, kBadPage);
        return;
    }
    const int64_t record = (int64_t)id * a.Hk + h;
    unsigned char *tiles = a.pool + record * (P / 16) * tile_bytes(W);
    const int base = (int)page << a.table.log_page;  // position of the page's first token
    const int lo = max(len, base), hi = (int)min(end, (int64_t)base + P);

    Turn turn;
    turn_weights<LPT>(turn, a, a.norm_k ? a.kw : nullptr, li);
    float mn[8], mx[8];
#pragma unroll
    for (int i = 0; i < 8; i++) { mn[i] = INFINITY; mx[i] = -INFINITY; }

    unsigned char *stage = smem + warp * 16 * ROW;
    const T *k0 = static_cast<const T *>(a.k) + b * (a.S ? a.k_sb : 0) + h * a.k_sh;
    const T *v0 = static_cast<const T *>(a.v) + b * (a.S ? a.v_sb : 0) + h * a.v_sh;
    for (int tile = warp; tile < P / 16; tile += warps) {
        const int tb = base + tile * 16;  // position of the tile's first token
        const int tlo = max(lo, tb) - tb, thi = min(hi, tb + 16) - tb;
        if (tlo >= thi) continue;
        unsigned char *out = tiles + (int64_t)tile * tile_bytes(W);
        for (int p = tlo / TPP * TPP; p < thi; p += TPP) {
            const int t = p + g;
            const bool on = t >= tlo && t < thi;
            const int64_t row = t0 + (tb + t - len);
            float x[8], y[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = y[i] = 0.f;
            if (on && live) {
                load8(k0 + row * a.k_ss + li * 8, a.vec & 4, x);
                load8(v0 + row * a.v_ss + li * 8, a.vec & 8, y);
                if (a.R)
                    turn_angles(turn, a, li, a.positions ? a.positions[a.S ? b * a.S + row : row]
                                                         : (int64_t)(tb + t));
            }
            turn_row<LPT>(x, turn, a.norm_k, a.inv_d, a.eps);
            uint32_t kc[2], vc[2];
            __half ks, vs;
            quantise8(x, kc, ks);
            quantise8(y, vc, vs);
            if (on && live) {
                const int j = li / 4, c = li % 4;
                reinterpret_cast<uint32_t *>(out)[t * 4 * W + c * W + j] = pack_k(kc);
                *reinterpret_cast<uint2 *>(stage + t * ROW + li * 8) = make_uint2(vc[0], vc[1]);
                if (c == 0) {
                    reinterpret_cast<__half *>(out + ks_off(W))[(2 * (t & 7) + (t >> 3)) * W + j] = ks;
                    reinterpret_cast<__half *>(out + vs_off(W))[4 * (((t & 7) >> 1) * W + j) +
                                                                2 * (t >> 3) + (t & 1)] = vs;
                }
                if (a.bounds) {
                    const float s = __half2float(ks);
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float z = (float)((int)((kc[i >> 2] >> (8 * (i & 3))) & 15u) - 8) * s;
                        mn[i] = fminf(mn[i], z);
                        mx[i] = fmaxf(mx[i], z);
                    }
                }
            }
        }
        __syncwarp();
        // the V words: this lane's channels and tokens, older tokens kept
        {
            const int r = lane >> 2, c = lane & 3;
            const int tok[4] = {2 * c, 2 * c + 1, 2 * c + 8, 2 * c + 9};
            uint32_t mask = 0;  // nibbles 2 y + 4 e and the next one: both channel halves
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (tok[u] >= tlo && tok[u] < thi) mask |= 0xffu << (4 * (2 * (u >> 1) + 4 * (u & 1)));
            uint32_t *vw = reinterpret_cast<uint32_t *>(out + v_off(W));
            const bool merge = tlo > 0;
#pragma unroll
            for (int m = 0; m < 2 * W; m++) {
                uint32_t w = 0;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const unsigned char *s = stage + tok[u] * ROW + 16 * m + r;
                    const int sh = 4 * (2 * (u >> 1) + 4 * (u & 1));
                    w |= (uint32_t)(s[0] & 15) << sh | (uint32_t)(s[8] & 15) << (sh + 4);
                }
                const int at = v_word<W>(m, lane);
                if (mask) vw[at] = (w & mask) | (merge ? vw[at] & ~mask : 0u);
            }
        }
        __syncwarp();
    }

    if (a.bounds) {
        // the block's tokens: over the lanes that share channels, then over the warps
#pragma unroll
        for (int i = 0; i < 8; i++) {
#pragma unroll
            for (int m = LPT; m < 32; m *= 2) {
                mn[i] = fminf(mn[i], __shfl_xor_sync(0xffffffffu, mn[i], m));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], m));
            }
        }
        __syncthreads();
        float *lo_s = reinterpret_cast<float *>(smem), *hi_s = lo_s + warps * D;
        if (g == 0 && live) {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                lo_s[warp * D + li * 8 + i] = mn[i];
                hi_s[warp * D + li * 8 + i] = mx[i];
            }
        }
        __syncthreads();
        if (warp == 0) {
            float top = 0.f;
            for (int d = lane; d < D; d += 32) {
                float u = lo_s[d], v = hi_s[d];
                for (int w = 1; w < warps; w++) {
                    u = fminf(u, lo_s[w * D + d]);
                    v = fmaxf(v, hi_s[w * D + d]);
                }
                if (u > v) u = v = 0.f;  // no number among them
                lo_s[d] = u;
                hi_s[d] = v;
                top = fmaxf(top, fmaxf(fabsf(u), fabsf(v)));
            }
#pragma unroll
            for (int m = 16; m; m /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
            int e = bound_exponent(top, -40);
            const bool older = lo > base;
            const int e0 = older ? a.exps[record] : e;
            e = max(e, e0);
            const float f = pow2f(-e);
            signed char *out = a.bounds + record * 2 * D;
            for (int d = lane; d < D; d += 32) {
                int u = (int)floorf(lo_s[d] * f), v = (int)ceilf(hi_s[d] * f);
                if (older) {
                    u = min(u, (int)out[d] >> min(e - e0, 31));
                    v = max(v, -(-(int)out[D + d] >> min(e - e0, 31)));
                }
                out[d] = (signed char)u;
                out[D + d] = (signed char)v;
            }
            __syncwarp();
            if (lane == 0) a.exps[record] = e;
        }
    }
}

constexpr int kQPasses = 4;  // passes of a warp over a token's query heads

template <typename T, int W, int LPT>
__device__ __forceinline__ void turn_queries(const AppendArgs &a) {
    constexpr int D = 32 * W, TPP = 32 / LPT;
    const int lane = threadIdx.x & 31, g = lane / LPT, li = lane % LPT;
    const bool live = li * 8 < D;
    const int64_t unit = ((int64_t)blockIdx.x - (int64_t)a.slots * a.Hk) * (blockDim.x >> 5) +
                         (threadIdx.x >> 5);
    const int64_t t = unit / a.q_units;
    if (t >= a.T) return;
    const int h0 = (int)(unit % a.q_units) * (kQPasses * TPP);
    int64_t b, row;
    if (a.S) {
        b = t / a.S;
        row = t % a.S;
    } else {
        const int *cu = a.cu;
        b = warp_find([=](int i) { return (int64_t)cu[i]; }, a.B, t);
        row = t;
    }
    const T *q = static_cast<const T *>(a.q) + (a.S ? b * a.q_sb : 0) + row * a.q_ss + li * 8;
    T *qo = static_cast<T *>(a.qo) + (a.S ? b * a.qo_sb : 0) + row * a.qo_ss + li * 8;
    float x[kQPasses][8];
#pragma unroll
    for (int p = 0; p < kQPasses; p++) {
        const int h = h0 + p * TPP + g;
#pragma unroll
        for (int i = 0; i < 8; i++) x[p][i] = 0.f;
        if (live && h < a.Hq) load8(q + h * a.q_sh, a.vec & 1, x[p]);
    }
    Turn turn;
    turn_weights<LPT>(turn, a, a.norm_q ? a.qw : nullptr, li);
    if (a.R) {
        int64_t pos = a.positions ? (int64_t)a.positions[t]
                                  : (int64_t)max(0, a.lengths[b]) + (a.S ? row : t - a.cu[b]);
        turn_angles(turn, a, li, pos);
    }
#pragma unroll
    for (int p = 0; p < kQPasses; p++) {
        const int h = h0 + p * TPP + g;
        turn_row<LPT>(x[p], turn, a.norm_q, a.inv_d, a.eps);
        if (live && h < a.Hq) store8(qo + h * a.qo_sh, a.vec & 2, x[p]);
    }
}

template <typename T, int W, int LPT>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    if ((int64_t)blockIdx.x < (int64_t)a.slots * a.Hk)
        write_page<T, W, LPT>(a, smem);
    else
        turn_queries<T, W, LPT>(a);
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

// One warp for 16 tokens (a tile) of one KV head.
template <typename T, int W>
__global__ void __launch_bounds__(128) read_kernel(const __grid_constant__ ReadArgs a) {
    constexpr int D = 32 * W;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (unit >= (int64_t)a.slots * a.Hk) return;
    const int slot = (int)(unit / a.Hk), h = (int)(unit % a.Hk);
    int b, n;
    int64_t first, t0;
    if (a.S) {
        const int per = (int)((a.S + 30) / 16);
        b = slot / per;
        first = (int64_t)b * per;
        n = (int)a.S;
        t0 = 0;
    } else {
        const int *cu = a.cu;
        b = warp_find([=](int i) { return (int64_t)(cu[i] >> 4) + 2 * i; }, a.B, slot);
        first = (int64_t)(cu[b] >> 4) + 2 * b;
        n = max(0, (int)min((int64_t)cu[b + 1], a.T) - max(0, cu[b]));
        t0 = max(0, cu[b]);
    }
    const int start = a.starts ? a.starts[b] : 0;
    if (start < 0 || n <= 0 || slot < first) return;
    const int64_t tile64 = (start >> 4) + (slot - first), end = (int64_t)start + n;
    if (tile64 * 16 >= end) return;
    if (tile64 * 16 >= (int64_t)a.table.max_pages << a.table.log_page) {
        if (lane == 0) atomicOr(a.table.status, kBadLength);
        return;
    }
    const int tile = (int)tile64, tb = tile * 16;
    const int lo = max(start, tb) - tb, hi = (int)min(end - tb, (int64_t)16);
    if (lo >= hi) return;
    const int tpp = a.table.log_page - 4;
    const int id = a.table.page(b, tile >> tpp);
    const unsigned char *in = a.pool + ((((int64_t)id * a.Hk + h) << tpp) + (tile & ((1 << tpp) - 1))) *
                                           tile_bytes(W);
    T *ko = static_cast<T *>(a.k) + (a.S ? b * a.o_sb : 0) + h * a.o_sh;
    T *vo = static_cast<T *>(a.v) + (a.S ? b * a.o_sb : 0) + h * a.o_sh;
    const uint32_t *kw = reinterpret_cast<const uint32_t *>(in);
    const uint32_t *vw = reinterpret_cast<const uint32_t *>(in + v_off(W));
    const __half *ksc = reinterpret_cast<const __half *>(in + ks_off(W));
    const __half *vsc = reinterpret_cast<const __half *>(in + vs_off(W));
    constexpr int CH = D / 8;  // 8-channel chunks of a token
    for (int u = lo * CH + lane; u < hi * CH; u += 32) {
        const int t = u / CH, li = u % CH, j = li / 4, c = li % 4;
        const int64_t row = t0 + (tb + t - start);
        float x[8];
        {
            const float s = __half2float(ksc[(2 * (t & 7) + (t >> 3)) * W + j]);
            const uint32_t w = kw[t * 4 * W + c * W + j];
#pragma unroll
            for (int i = 0; i < 8; i++)
                x[i] = (float)((int)((w >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u) - 8) * s;
            store8(ko + row * a.o_ss + li * 8, a.vec & 1, x);
        }
        {
            const int vc = (t & 7) >> 1;
            const float s = __half2float(vsc[4 * (vc * W + j) + 2 * (t >> 3) + (t & 1)]);
            const int sh = 4 * ((li & 1) + 2 * (t >> 3) + 4 * (t & 1));
#pragma unroll
            for (int i = 0; i < 8; i++)
                x[i] = (float)((int)((vw[v_word<W>(li >> 1, i * 4 + vc)] >> sh) & 15u) - 8) * s;
            store8(vo + row * a.o_ss + li * 8, a.vec & 2, x);
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
    if (T == 0 || B == 0) return FC_OK;
    if (!k || !v || !lengths || (Hq && (!q || !q_out))) { set_error("kv4_append: null pointer"); return FC_EINVAL; }
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
            (rows_aligned(v, dtype, v_sb, v_ss, v_sh) ? 8 : 0);
    const int64_t slots = a.S ? B * ((S + 2 * page_size - 2) / page_size) : T / page_size + 2 * B;
    const int warps = (int)(page_size / 16 < 8 ? page_size / 16 : 8);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_dtype(dtype, [&](auto t) {
        return by_head_dim(D, [&](auto w) {
            using E = decltype(t);
            constexpr int W = decltype(w)::value, LPT = lanes_per_head(W);
            a.slots = (int)slots;
            a.q_units = (int)((Hq + kQPasses * (32 / LPT) - 1) / (kQPasses * (32 / LPT)));
            const int64_t blocks = slots * Hk + (T * a.q_units + warps - 1) / warps;
            if (slots > 0x7fffffff || blocks > 0x7fffffff) {
                set_error("kv4_append: too many tokens for one call");
                return FC_ENOTSUP;
            }
            const size_t stage = (size_t)warps * 16 * (32 * W + 8), red = (size_t)warps * 32 * W * 8;
            append_kernel<E, W, LPT><<<(unsigned)blocks, warps * 32, stage > red ? stage : red, st>>>(a);
            return check_launch("kv4_append");
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
    if (T == 0 || B == 0) return FC_OK;
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
    const int64_t slots = a.S ? B * ((S + 30) / 16) : T / 16 + 2 * B;
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
