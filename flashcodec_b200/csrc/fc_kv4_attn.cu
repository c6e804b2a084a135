// Paged 4-bit KV cache: attention of one or a few new tokens.
//
//   out = softmax(scale * q . K^T) . V,  K = code * scale per group of 32 channels
//
// Every held byte is read once per KV head (4.5 bits a value, so HBM bounds it from
// below at 144 bytes a token and head at D = 128), and each value takes part in
// Hq / Hk products on each side.  What competes with HBM is the issue rate: at
// 6.4 TB/s an SM receives 46 values a cycle to unpack.  So the pages are stored in
// the operand order of mma.m16n8k16 (fc_kv4.cuh): a lane's words become operands by
// an AND and an OR per two values (fp16 1024 + code), tokens (K) or channels (V) in
// the 16 rows, the group's query rows in the 8 columns, and nothing is exchanged
// between lanes but a transposition of the weights (movmatrix).  Matrix instructions
// that read shared memory (tcgen05) would need the unpacked values written back to
// shared memory, 4 bytes moved for every half byte that arrives.
//
// Scores.  A group of 32 channels is two matrix instructions; its fp16 scales come
// in after it, in fp32.  With bf16 queries the +1032 that unpacking leaves on a code
// is taken off by starting the group's sum from -1032 * (sum of q): exact products,
// fp32 sums, an error of about 2^-24 * 1032 of the largest |q| of the group.  With
// fp16 and fp32 queries the codes are made exact first, and a query is two fp16
// parts in neighbouring columns (22 bits).  Queries are scaled by a power of two per
// row so that fp16 holds them.
//
// Weights.  Base-2 softmax with a running reference per row, moved only when a score
// passes it by 2^4, and a running power of two above the values' scales, so that
// weight * scale, an fp16 operand, stays in 2^-14 .. 2^15.  One rounding of the weight
// and one of the product for bf16 queries (2^-11 each), two fp16 parts otherwise.
//
// Work.  The chunks (32 tokens) of all (sequence, KV head, row block) are one line,
// cut into equal pieces for one wave of blocks, whatever the lengths; the lengths are
// read on the device.  A block's 4 warps take the chunks of its piece in turn, each
// with its own ring of asynchronous copies and its own running state.  Pieces of one
// (sequence, head) are joined by the last block to finish, in order: the result does
// not depend on timing.  No block waits for another.
#include "fc_kv4.cuh"

namespace fc {
namespace kv4 {
namespace {

struct AttnArgs {
    const void *q;
    int64_t q_sb, q_ss, q_sh;
    int B, Sq, Hq, Hk, G, rows, row_blocks, dtype, q_vec;
    const unsigned char *pool;
    Table table;
    const int *lengths, *selected;
    int n_selected;
    float scale;  // softmax_scale * log2(e), >= 0
    float sign;   // of softmax_scale, folded into the queries
    void *out;
    int64_t o_sb, o_ss, o_sh;
    float *lse;
    int *counters;  // one per (sequence, KV head, row block), zero between calls
    float *parts;   // two per block: [row][D], then the references and the sums
};

constexpr int kWarps = 4, kThreads = 32 * kWarps, kStages = 3;
constexpr int kMinChunks = 8;    // of a block's piece
constexpr float kSlack = 4.f;    // log2 of how far a score may pass the reference

__device__ __forceinline__ void mma16816(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t u32(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 h2(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

// (x & mask) | 0x64006400: fp16 pairs 1024 + nibble (or + 16 nibble)
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask) {
    return (x & mask) | 0x64006400u;
}

// The four pairs of a word as 1024 + u, 1024 + 16 u, 1024 + u, 1024 + 16 u.
__device__ __forceinline__ void unpack_raw(uint32_t w, uint32_t p[4]) {
    const uint32_t s = w >> 8;
    p[0] = and_or(w, 0x000f000fu);
    p[1] = and_or(w, 0x00f000f0u);
    p[2] = and_or(s, 0x000f000fu);
    p[3] = and_or(s, 0x00f000f0u);
}

// ... as codes (u - 8), exact
__device__ __forceinline__ void unpack(uint32_t w, uint32_t p[4]) {
    unpack_raw(w, p);
    const __half2 one = __float2half2_rn(-1032.f), sixteenth = __float2half2_rn(0.0625f),
                  off = __float2half2_rn(-72.f);
    p[0] = u32(__hadd2(h2(p[0]), one));
    p[1] = u32(__hfma2(h2(p[1]), sixteenth, off));
    p[2] = u32(__hadd2(h2(p[2]), one));
    p[3] = u32(__hfma2(h2(p[3]), sixteenth, off));
}

__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// N 32-bit words from shared memory by the widest loads that their alignment
// (N * 4 bytes per lane or row) allows.
template <int N>
__device__ __forceinline__ void load_words(const void *p, uint32_t w[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = static_cast<const uint4 *>(p)[i];
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const uint2 v = static_cast<const uint2 *>(p)[i];
            w[2 * i] = v.x; w[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = static_cast<const uint32_t *>(p)[i];
    }
}

template <int W, int NT, int LIMBS>
struct Attn {
    static constexpr int D = 32 * W, TILE = tile_bytes(W), STAGE = 2 * TILE;
    static constexpr int RPC = 8 * NT / LIMBS;  // query rows of a block
    static constexpr int RING = kStages * STAGE;
    static constexpr int SMEM = kWarps * RING;

    const AttnArgs &a;
    unsigned char *ring;  // of this warp
    int *pos_s;           // (kStages, 2) first positions of the staged tiles
    int warp, lane, r, c;
    // this segment
    int b, h, rb, len, chunk0, chunk1;
    int log_tpp, pages;
    // queries: operand words, offsets of a group's sum, factors and lengths seen
    uint32_t qb[NT][2 * W][2];
    float off[LIMBS == 1 ? NT : 1][LIMBS == 1 ? W : 1][2];
    float f[NT][2];
    int seen[NT][2], min_seen;
    // running state
    float M[NT][2], l[NT][2], acc[NT][2 * W][4];
    float lim, slim;

    __device__ __forceinline__ Attn(const AttnArgs &args, unsigned char *smem, int *pos)
        : a(args) {
        warp = threadIdx.x >> 5;
        lane = threadIdx.x & 31;
        r = lane >> 2;
        c = lane & 3;
        ring = smem + warp * RING;
        pos_s = pos + warp * kStages * 2;
        log_tpp = a.table.log_page - 4;
    }

    __device__ __forceinline__ int row_of(int nt, int col) const {
        return rb * RPC + (LIMBS == 1 ? nt * 8 + col : nt * 4 + col / 2);
    }

    // ---------------------------------------------------------------- queries
    __device__ __forceinline__ void load_queries() {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int row = row_of(nt, r);  // the operand's column is lane / 4
            float x[8 * W];
            const bool on = row < a.rows;
            const int s = row / a.G, g = row - s * a.G;
            const int64_t o = b * a.q_sb + s * a.q_ss + (int64_t)(h * a.G + g) * a.q_sh + 8 * c;
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < W; j++) {
                if (on && a.q_vec) {
                    if constexpr (LIMBS == 1) {
                        load_vec_f32<__nv_bfloat16, 8>(static_cast<const __nv_bfloat16 *>(a.q) + o + 32 * j, x + 8 * j);
                    } else if (a.dtype == FC_F16) {
                        load_vec_f32<__half, 8>(static_cast<const __half *>(a.q) + o + 32 * j, x + 8 * j);
                    } else {
                        load_vec_f32<float, 4>(static_cast<const float *>(a.q) + o + 32 * j, x + 8 * j);
                        load_vec_f32<float, 4>(static_cast<const float *>(a.q) + o + 32 * j + 4, x + 8 * j + 4);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[8 * j + i] = on ? load_as_f32(a.q, o + 32 * j + i, a.dtype) : 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[8 * j + i]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^e above the largest |q|: queries times 2^(14 - e)
            int e = (int)(__float_as_uint(top) >> 23) - 126;
            e = top > 0.f ? max(e, -100) : 0;
            const float up = pow2f(min(14 - e, 126)) * a.sign, down = pow2f(-min(14 - e, 126));
            float sum[W];
#pragma unroll
            for (int j = 0; j < W; j++) {
                sum[j] = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    float u = x[8 * j + i] * up, v = x[8 * j + i + 1] * up;
                    __half2 p = __floats2half2_rn(u, v);
                    if constexpr (LIMBS == 2) {
                        if (r & 1) {
                            const float2 hi = __half22float2(p);
                            p = __floats2half2_rn(u - hi.x, v - hi.y);
                        }
                    } else {
                        const bool sixteen = (i >> 1) & 1;  // its codes come as 1024 + 16 u
                        if (sixteen) p = __floats2half2_rn(u * 0.0625f, v * 0.0625f);
                        const float2 z = __half22float2(p);
                        sum[j] -= (sixteen ? 1152.f : 1032.f) * (z.x + z.y);
                    }
                    qb[nt][2 * j + (i >> 2)][(i >> 1) & 1] = u32(p);
                }
                if constexpr (LIMBS == 1) {
                    sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
                    sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
                }
            }
            // what belongs to a column, from the lanes that hold it to those that score it
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const int from = (2 * c + y) * 4;
                f[nt][y] = __shfl_sync(0xffffffffu, down, from) * a.scale;
                if constexpr (LIMBS == 1) {
#pragma unroll
                    for (int j = 0; j < W; j++) off[nt][j][y] = __shfl_sync(0xffffffffu, sum[j], from);
                }
                const int sq = min(row_of(nt, 2 * c + y), a.rows - 1) / a.G;
                seen[nt][y] = len - (a.Sq - 1 - sq);
            }
        }
        // row blocks hold rows in order: the first one sees least
        min_seen = len - (a.Sq - 1 - min(rb * RPC, a.rows - 1) / a.G);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int y = 0; y < 2; y++) { M[nt][y] = -1e30f; l[nt][y] = 0.f; }
#pragma unroll
            for (int m = 0; m < 2 * W; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[nt][m][i] = 0.f;
        }
        lim = 15.f;
        slim = 1.f;
    }

    // ------------------------------------------------------------------ copies
    // Lanes 0 and 1 look the tiles of a chunk up (the others follow lane 1): the
    // page of the sequence, and where it lies.
    __device__ __forceinline__ int logical(int chunk) const {
        const int tile = 2 * chunk + (lane & 1);
        int page = tile >> log_tpp;
        if (a.selected) {
            if (page >= a.n_selected) return -1;
            page = a.selected[((int64_t)b * a.Hk + h) * a.n_selected + page];
        }
        return page < pages ? page : -1;
    }
    __device__ __forceinline__ int physical(int page) const {
        return page < 0 ? -1 : a.table.page(b, page);
    }
    __device__ __forceinline__ void issue(int chunk, int page, int id, int stage) {
        const int tile = (2 * chunk + (lane & 1)) & ((1 << log_tpp) - 1);
        int pos = page < 0 ? 0x7fffffff - 64 : (page << a.table.log_page) + tile * 16;
        if (pos >= len) id = -1;  // nothing there
        if (id < 0) pos = 0x7fffffff - 64;
        const int64_t at = ((((int64_t)max(id, 0) * a.Hk + h) << log_tpp) + tile) * TILE;
        if (lane < 2) pos_s[stage * 2 + lane] = pos;
        const int id0 = __shfl_sync(0xffffffffu, id, 0), id1 = __shfl_sync(0xffffffffu, id, 1);
        const unsigned char *s0 = a.pool + __shfl_sync(0xffffffffu, at, 0);
        const unsigned char *s1 = a.pool + __shfl_sync(0xffffffffu, at, 1) - TILE;
        const uint32_t dst = static_cast<uint32_t>(__cvta_generic_to_shared(ring + stage * STAGE));
        constexpr int N = TILE / 16;  // 36 W pieces of a tile
#pragma unroll
        for (int i = 0; i < (2 * N + 31) / 32; i++) {
            const int p = 32 * i + lane;
            const bool second = 32 * i >= N || (32 * i + 31 >= N && p >= N);
            if ((32 * i + 31 < 2 * N || p < 2 * N) && (second ? id1 : id0) >= 0)
                copy16(dst + p * 16, (second ? s1 : s0) + p * 16);
        }
    }

    // ------------------------------------------------------------------- chunk
    __device__ __forceinline__ void score(const unsigned char *tile, float S[NT][4]) const {
        uint32_t k0[W], k1[W], sc[W];
        load_words<W>(tile + lane * 4 * W, k0);  // row r: 16 W bytes, chunk c of 4 W
        load_words<W>(tile + 128 * W + lane * 4 * W, k1);
        load_words<W>(tile + ks_off(W) + r * 4 * W, sc);  // W scales of row r, W of row r + 8
        float s[2 * W];
#pragma unroll
        for (int i = 0; i < W; i++) {
            const float2 z = __half22float2(h2(sc[i]));
            s[2 * i] = z.x;
            s[2 * i + 1] = z.y;
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 4; i++) S[nt][i] = 0.f;
#pragma unroll
        for (int j = 0; j < W; j++) {
            uint32_t x[4], y[4];
            if constexpr (LIMBS == 1) {
                unpack_raw(k0[j], x);
                unpack_raw(k1[j], y);
            } else {
                unpack(k0[j], x);
                unpack(k1[j], y);
            }
            const uint32_t a0[4] = {x[0], y[0], x[1], y[1]}, a1[4] = {x[2], y[2], x[3], y[3]};
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float t[4];
                if constexpr (LIMBS == 1) {
                    t[0] = t[2] = off[nt][j][0];
                    t[1] = t[3] = off[nt][j][1];
                } else {
                    t[0] = t[1] = t[2] = t[3] = 0.f;
                }
                mma16816(t, a0, qb[nt][2 * j][0], qb[nt][2 * j][1]);
                mma16816(t, a1, qb[nt][2 * j + 1][0], qb[nt][2 * j + 1][1]);
                S[nt][0] = fmaf(s[j], t[0], S[nt][0]);
                S[nt][1] = fmaf(s[j], t[1], S[nt][1]);
                S[nt][2] = fmaf(s[W + j], t[2], S[nt][2]);
                S[nt][3] = fmaf(s[W + j], t[3], S[nt][3]);
            }
        }
        if constexpr (LIMBS == 2) {  // the two parts of a query are neighbouring columns
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                S[nt][0] = S[nt][1] = S[nt][0] + S[nt][1];
                S[nt][2] = S[nt][3] = S[nt][2] + S[nt][3];
            }
        }
    }

    // Tokens that a row does not see, and scales of tokens that are not there.
    __device__ __forceinline__ void mask(unsigned char *tile, int pos, float S[NT][4]) const {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (pos + r + 8 * (i >> 1) >= seen[nt][i & 1]) S[nt][i] = -INFINITY;
        if (pos + 16 > len) {
            __half *vs = reinterpret_cast<__half *>(tile + vs_off(W));
#pragma unroll
            for (int i = 0; i < 16 * W / 32 + (16 * W % 32 != 0); i++) {
                const int at = 32 * i + lane;
                const int t = 2 * (at / (4 * W)) + 8 * ((at >> 1) & 1) + (at & 1);
                if (at < 16 * W && pos + t >= len) vs[at] = __ushort_as_half(0);
            }
        }
    }

    // acc += V . weights of one tile; p: the weights, in place of the scores
    __device__ __forceinline__ void gather(const unsigned char *tile, const float p[NT][4],
                                           float out[NT][2 * W][4]) const {
        uint32_t v[2 * W];
        constexpr int VW = v_vec(W);
#pragma unroll
        for (int i = 0; i < 2 * W / VW; i++) load_words<VW>(tile + v_off(W) + (i * 32 + lane) * 4 * VW, v + i * VW);
        uint32_t w[NT][W][2];
        if constexpr (LIMBS == 1) {
            uint32_t sc[2 * W];
            load_words<2 * W>(tile + vs_off(W) + c * 8 * W, sc);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const uint32_t lo = transpose8(u32(__floats2half2_rn(p[nt][0], p[nt][1])));
                const uint32_t hi = transpose8(u32(__floats2half2_rn(p[nt][2], p[nt][3])));
#pragma unroll
                for (int j = 0; j < W; j++) {
                    w[nt][j][0] = u32(__hmul2(h2(lo), h2(sc[2 * j])));
                    w[nt][j][1] = u32(__hmul2(h2(hi), h2(sc[2 * j + 1])));
                }
            }
        } else {
            const __half *vs = reinterpret_cast<const __half *>(tile + vs_off(W)) + (r >> 1) * 4 * W + (r & 1);
#pragma unroll
            for (int j = 0; j < W; j++) {
                const float s0 = __half2float(vs[4 * j]), s1 = __half2float(vs[4 * j + 2]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float u = p[nt][0] * s0, v2 = p[nt][2] * s1;
                    const __half uh = __float2half_rn(u), vh = __float2half_rn(v2);
                    w[nt][j][0] = transpose8(u32(__halves2half2(uh, __float2half_rn(u - __half2float(uh)))));
                    w[nt][j][1] = transpose8(u32(__halves2half2(vh, __float2half_rn(v2 - __half2float(vh)))));
                }
            }
        }
#pragma unroll
        for (int m = 0; m < 2 * W; m++) {
            uint32_t x[4];
            unpack(v[m], x);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) mma16816(out[nt][m], x, w[nt][m / 2][0], w[nt][m / 2][1]);
        }
    }

    __device__ __forceinline__ void chunk(int stage) {
        unsigned char *tile = ring + stage * STAGE;
        const int p0 = pos_s[stage * 2], p1 = pos_s[stage * 2 + 1];
        if (p0 >= len && p1 >= len) return;
        float S[2][NT][4];
        score(tile, S[0]);
        score(tile + TILE, S[1]);
        if (max(p0, p1) + 16 > min_seen) {
            mask(tile, p0, S[0]);
            mask(tile + TILE, p1, S[1]);
            __syncwarp();
        }
        // does a score pass its reference, or a scale of the values the running bound?
        uint32_t sv[W];
        const int half = lane >> 4;
        {
            const unsigned char *p = tile + half * TILE + vs_off(W) + (lane & 15) * 2 * W;
            if constexpr (W % 2 == 0) {
                load_words<W / 2>(p, sv);
            } else {
#pragma unroll
                for (int i = 0; i < (W + 1) / 2; i++)  // 2 W bytes: W halves, the last word overlaps
                    sv[i] = reinterpret_cast<const uint16_t *>(p)[2 * i] |
                            (uint32_t)reinterpret_cast<const uint16_t *>(p)[min(2 * i + 1, W - 1)] << 16;
            }
        }
        __half2 st = h2(sv[0]);
#pragma unroll
        for (int i = 1; i < (W + 1) / 2; i++) st = __hmax2(st, h2(sv[i]));
        const float sm = __half2float(__hmax(__low2half(st), __high2half(st)));
        bool pass = sm > slim;
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                top[nt][y] = fmaxf(fmaxf(S[0][nt][y], S[0][nt][y + 2]), fmaxf(S[1][nt][y], S[1][nt][y + 2]));
                pass = pass || fmaf(top[nt][y], f[nt][y], -M[nt][y]) > lim;
            }
        if (__any_sync(0xffffffffu, pass)) {
            float s = sm;
#pragma unroll
            for (int o = 16; o; o /= 2) s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, o));
            const float old = lim;
            if (s > slim && s <= 65504.f) {
                const uint32_t u = __float_as_uint(s);
                const int e = (int)(u >> 23) - 127 + ((u & 0x7fffffu) != 0);  // s <= 2^e
                slim = pow2f(e);
                lim = 15.f - (float)e;
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    float t = top[nt][y];
#pragma unroll
                    for (int o = 4; o < 32; o *= 2) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
                    float m = M[nt][y] + (old - lim);
                    if (t > -INFINITY) m = fmaxf(m, fmaf(t, f[nt][y], -(lim - kSlack)));
                    const float g = exp2_fast(M[nt][y] - m);
                    M[nt][y] = m;
                    l[nt][y] *= g;
#pragma unroll
                    for (int i = 0; i < 2 * W; i++) {
                        acc[nt][i][y] *= g;
                        acc[nt][i][y + 2] *= g;
                    }
                }
        }
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = exp2_fast(fmaf(S[t][nt][i], f[nt][i & 1], -M[nt][i & 1]));
                    S[t][nt][i] = p;
                    l[nt][i & 1] += p;
                }
        if constexpr (LIMBS == 1) {
            gather(tile, S[0], acc);
            gather(tile + TILE, S[1], acc);
        } else {
            // a chunk's sum by itself: the long sum is then in rounded fp32 additions
            float part[NT][2 * W][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int m = 0; m < 2 * W; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++) part[nt][m][i] = 0.f;
            gather(tile, S[0], part);
            gather(tile + TILE, S[1], part);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int m = 0; m < 2 * W; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[nt][m][i] += part[nt][m][i];
        }
    }

    // This warp's chunks of the segment: chunk0 + warp, + 4, ...
    __device__ __forceinline__ void run() {
        int next = chunk0 + warp;  // the next chunk to copy
        int page = next < chunk1 ? logical(next) : -1;
        int id = physical(page);
        int page2 = next + kWarps < chunk1 ? logical(next + kWarps) : -1;
        auto fetch = [&](int stage) {
            if (next < chunk1) issue(next, page, id, stage);
            asm volatile("cp.async.commit_group;" ::: "memory");
            next += kWarps;
            page = page2;
            id = physical(page);
            page2 = next + kWarps < chunk1 ? logical(next + kWarps) : -1;
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; i++) fetch(i);
        int stage = 0;
        for (int i = chunk0 + warp; i < chunk1; i += kWarps) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncwarp();
            fetch(stage == 0 ? kStages - 1 : stage - 1);
            chunk(stage);
            __syncwarp();
            stage = stage == kStages - 1 ? 0 : stage + 1;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }

    // -------------------------------------------------------------------- joins
    // The block's sums of this segment: rows' outputs o(row, d), references and sums
    // in shared memory.
    static constexpr int PART = RPC * (D + 2);  // floats of a partial result

    __device__ __forceinline__ void write_row(int row, int d, float v) const {
        const int s = row / a.G, g = row - s * a.G;
        store_from_f32(a.out, b * a.o_sb + s * a.o_ss + (int64_t)(h * a.G + g) * a.o_sh + d,
                       LIMBS == 1 ? FC_BF16 : a.dtype, v);
    }
    __device__ __forceinline__ void write_lse(int row, float m, float sum) const {
        const int s = row / a.G, g = row - s * a.G;
        a.lse[((int64_t)b * a.Sq + s) * a.Hq + h * a.G + g] =
            sum > 0.f ? (m + log2f(sum)) * 0.693147180559945309f : sum == 0.f ? -INFINITY : sum;
    }

    // Joins the warps; whole: the outputs are final, else they go to `part`.
    __device__ __forceinline__ void join(unsigned char *smem, float *ml, bool whole, float *part) {
        // ml: [warp][row][2]
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float s = l[nt][y];
#pragma unroll
                for (int o = 4; o < 32; o *= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
                l[nt][y] = s;
                const int col = nt * 8 + 2 * c + y;
                if (r == 0 && (LIMBS == 1 || y == 0)) {
                    ml[(warp * RPC + col / LIMBS) * 2] = M[nt][y];
                    ml[(warp * RPC + col / LIMBS) * 2 + 1] = s;
                }
            }
        __syncthreads();  // also: every warp has left its ring
        float *o = reinterpret_cast<float *>(smem);  // [warp][row][D]
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int y = 0; y < 2 / LIMBS; y++) {
                const int row = (nt * 8 + 2 * c + y) / LIMBS;
                float m = ml[row * 2];
#pragma unroll
                for (int w = 1; w < kWarps; w++) m = fmaxf(m, ml[(w * RPC + row) * 2]);
                const float g = exp2_fast(M[nt][y] - m);
#pragma unroll
                for (int i = 0; i < 2 * W; i++) {
                    float u = acc[nt][i][y], v = acc[nt][i][y + 2];
                    if constexpr (LIMBS == 2) { u += acc[nt][i][1]; v += acc[nt][i][3]; }
                    o[(warp * RPC + row) * D + 16 * i + r] = u * g;
                    o[(warp * RPC + row) * D + 16 * i + r + 8] = v * g;
                }
            }
        __syncthreads();
        const int rows = min(RPC, a.rows - rb * RPC);
        for (int i = threadIdx.x; i < rows * D; i += kThreads) {
            const int row = i / D;
            float m = ml[row * 2], s = 0.f, v = 0.f;
#pragma unroll
            for (int w = 1; w < kWarps; w++) m = fmaxf(m, ml[(w * RPC + row) * 2]);
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                s += ml[(w * RPC + row) * 2 + 1] * exp2_fast(ml[(w * RPC + row) * 2] - m);
                v += o[w * RPC * D + i];
            }
            if (whole) {
                write_row(rb * RPC + row, i % D, s == 0.f ? 0.f : v / s);
                if (a.lse && i % D == 0) write_lse(rb * RPC + row, m, s);
            } else {
                part[i] = v;
                if (i % D == 0) {
                    part[RPC * D + 2 * row] = m;
                    part[RPC * D + 2 * row + 1] = s;
                }
            }
        }
    }
};

// Chunks of sequence b, 0 where it holds nothing.
__device__ __forceinline__ int chunks_of(const AttnArgs &a, int64_t b) {
    const int len = a.table.length(a.lengths[b]);
    if (len <= 0) return 0;
    if (a.selected) return ((a.n_selected << (a.table.log_page - 4)) + 1) / 2;
    return (len + 31) / 32;
}

template <int W, int NT, int LIMBS>
__global__ void __launch_bounds__(kThreads) attn_kernel(const __grid_constant__ AttnArgs a) {
    using A = Attn<W, NT, LIMBS>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int64_t sums[kThreads], pre_s;
    __shared__ int b_s, last_s;
    __shared__ int pos[kWarps * kStages * 2];
    __shared__ float ml[kWarps * A::RPC * 2];

    // the line of chunks: before each thread's sequences, and in all
    const int HR = a.Hk * a.row_blocks;
    const int per = (a.B + kThreads - 1) / kThreads;
    const int b0 = min((int)threadIdx.x * per, a.B), b1 = min(b0 + per, a.B);
    int64_t mine = 0;
    for (int b = b0; b < b1; b++) mine += chunks_of(a, b);
    sums[threadIdx.x] = mine;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int i = 0; i < kThreads; i++) {
        if (i < (int)threadIdx.x) before += sums[i];
        all += sums[i];
    }
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {  // nothing held: zeros
        if (chunks_of(a, b)) continue;
        for (int i = threadIdx.x; i < a.Sq * a.Hq * A::D; i += kThreads) {
            const int row = i / A::D, s = row / a.Hq;
            store_from_f32(a.out, b * a.o_sb + s * a.o_ss + (row - s * a.Hq) * a.o_sh + i % A::D, a.dtype, 0.f);
            if (a.lse && i % A::D == 0) a.lse[(int64_t)b * a.Sq * a.Hq + row] = -INFINITY;
        }
    }
    const int64_t U = all * HR;
    const int64_t blocks = min((int64_t)gridDim.x, (U + kMinChunks - 1) / kMinChunks);
    if ((int64_t)blockIdx.x >= blocks) return;
    int64_t x = U * blockIdx.x / blocks;
    const int64_t end = U * (blockIdx.x + 1) / blocks;
    const int64_t start = x;
    // the sequence that x falls in
    {
        int64_t at = before * HR;
        if (x >= at && x < at + mine * HR) {
            int b = b0;
            for (;; b++) {
                const int64_t n = (int64_t)chunks_of(a, b) * HR;
                if (x < at + n) break;
                at += n;
            }
            b_s = b;
            pre_s = at;
        }
    }
    __syncthreads();
    int b = b_s;
    int64_t base = pre_s;  // where the line of sequence b begins

    A t(a, smem, pos);
    while (x < end) {
        int n = chunks_of(a, b);
        while (x >= base + (int64_t)n * HR) {
            base += (int64_t)n * HR;
            n = chunks_of(a, ++b);
        }
        const int unit = (int)((x - base) / n);
        const int64_t u0 = base + (int64_t)unit * n;
        t.b = b;
        t.h = unit / a.row_blocks;
        t.rb = unit % a.row_blocks;
        t.len = a.table.length(a.lengths[b]);
        t.pages = (t.len + (1 << a.table.log_page) - 1) >> a.table.log_page;
        t.chunk0 = (int)(x - u0);
        t.chunk1 = (int)min((int64_t)n, end - u0);
        const bool whole = t.chunk0 == 0 && t.chunk1 == n;
        t.load_queries();
        t.run();
        float *part = a.parts + ((int64_t)blockIdx.x * 2 + (x == start ? 0 : 1)) * A::PART;
        t.join(smem, ml, whole, part);
        if (!whole) {
            // blocks that share this unit: from the one its first chunk falls to
            const int64_t i0 = ((u0 + 1) * blocks - 1) / U, i1 = ((u0 + n) * blocks - 1) / U;
            int *counter = a.counters + ((int64_t)b * HR + unit);
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) last_s = atomicAdd(counter, 1) == (int)(i1 - i0);
            __syncthreads();
            if (last_s) {
                __threadfence();
                const int rows = min(A::RPC, a.rows - t.rb * A::RPC);
                for (int i = threadIdx.x; i < rows * A::D; i += kThreads) {
                    const int row = i / A::D;
                    auto of = [&](int64_t k) {
                        const bool first = U * k / blocks >= u0;
                        return a.parts + (k * 2 + (first ? 0 : 1)) * A::PART;
                    };
                    float m = -INFINITY, s = 0.f, v = 0.f;
                    for (int64_t k = i0; k <= i1; k++) m = fmaxf(m, __ldcg(of(k) + A::RPC * A::D + 2 * row));
                    for (int64_t k = i0; k <= i1; k++) {
                        const float *p = of(k);
                        const float g = exp2_fast(__ldcg(p + A::RPC * A::D + 2 * row) - m);
                        s += g * __ldcg(p + A::RPC * A::D + 2 * row + 1);
                        v += g * __ldcg(p + i);
                    }
                    t.write_row(t.rb * A::RPC + row, i % A::D, s == 0.f ? 0.f : v / s);
                    if (a.lse && i % A::D == 0) t.write_lse(t.rb * A::RPC + row, m, s);
                }
                if (threadIdx.x == 0) *counter = 0;
            }
        }
        __syncthreads();
        x = u0 + t.chunk1;
    }
}

constexpr int kMaxBlocksPerSm = 8;

// Blocks of a wave: what of the kernel fits on the device.
template <int W, int NT, int LIMBS>
int wave() {
    static int cache[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (cache[dev] == 0) {
        constexpr int smem = Attn<W, NT, LIMBS>::SMEM;
        int n = 0;
        if (cudaFuncSetAttribute(attn_kernel<W, NT, LIMBS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
                cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attn_kernel<W, NT, LIMBS>, kThreads, smem) !=
                cudaSuccess || n < 1)
            return 0;
        cache[dev] = num_sms() * (n < kMaxBlocksPerSm ? n : kMaxBlocksPerSm);
    }
    return cache[dev];
}

int64_t counter_bytes(int64_t units) { return 256 + (units * 4 + 255) / 256 * 256; }

}  // namespace
}  // namespace kv4
}  // namespace fc

using namespace fc;
using namespace fc::kv4;

extern "C" size_t fc_kv4_attn_workspace_size(int64_t B, int64_t Sq, int64_t Hq, int64_t Hk, int64_t D) {
    if (B <= 0 || Sq <= 0 || Hk <= 0 || Hq < Hk) return 256;
    const int64_t rows = Sq * (Hq / Hk);
    // the smaller of the row blocks the kernels use holds 4 rows; 16 rows are the largest
    return (size_t)(counter_bytes(B * Hk * ((rows + 3) / 4)) +
                    (int64_t)num_sms() * kMaxBlocksPerSm * 2 * 16 * (D + 2) * 4);
}

extern "C" int fc_kv4_attn(const void *q, int dtype, int64_t B, int64_t Sq, int64_t Hq, int64_t q_sb,
                           int64_t q_ss, int64_t q_sh, const void *pool, int64_t num_pages, int64_t Hk,
                           int64_t D, int64_t page_size, const int *page_table, int64_t table_stride,
                           int64_t max_pages, const int *lengths, const int *selected,
                           int64_t n_selected, float softmax_scale, void *out, int64_t o_sb,
                           int64_t o_ss, int64_t o_sh, float *lse, void *workspace,
                           size_t workspace_bytes, int *status, void *stream) {
    clear_error();
    int rc = check_cache("kv4_attn", B, Hk, D, page_size, num_pages, max_pages, pool, page_table, status);
    if (rc) return rc;
    if (!is_float_dtype(dtype)) { set_error("kv4_attn: dtype must be fp32, bf16 or fp16"); return FC_EINVAL; }
    if (Hq <= 0 || Hq % Hk) {
        set_error("kv4_attn: query heads (%lld) must be a multiple of kv heads (%lld)", (long long)Hq, (long long)Hk);
        return FC_EINVAL;
    }
    if (Sq < 0 || Sq > 65535 || Hq > 65535) { set_error("kv4_attn: bad query count"); return FC_EINVAL; }
    if (!(softmax_scale == softmax_scale) || softmax_scale - softmax_scale != 0.f) {
        set_error("kv4_attn: the softmax scale must be finite");
        return FC_EINVAL;
    }
    if (B == 0 || Sq == 0) return FC_OK;
    if (!q || !out || !lengths) { set_error("kv4_attn: null pointer"); return FC_EINVAL; }
    if (selected && (Sq != 1 || n_selected < 0 || n_selected * page_size > 0x7fffffff)) {
        set_error("kv4_attn: selected pages go with one query per sequence");
        return FC_EINVAL;
    }
    if (!workspace || !aligned(workspace, 16)) { set_error("kv4_attn: null or misaligned workspace"); return FC_EINVAL; }
    if (workspace_bytes < fc_kv4_attn_workspace_size(B, Sq, Hq, Hk, D)) {
        set_error("kv4_attn: workspace of %zu bytes is too small", workspace_bytes);
        return FC_ERANGE;
    }
    const int64_t rows = Sq * (Hq / Hk);
    const int limbs = dtype == FC_BF16 ? 1 : 2;
    // One column block of 8 serves up to 8 (4) rows.  More rows take two: they double
    // the matrix instructions but share the unpacking, against reading the pages twice.
    const int nt = rows * limbs > 8 ? 2 : 1;
    const int rpc = 8 * nt / limbs;
    const int64_t row_blocks = (rows + rpc - 1) / rpc;
    if (B * Hk * row_blocks > 0x7fffffff) { set_error("kv4_attn: too many rows"); return FC_ENOTSUP; }
    char *ws = static_cast<char *>(workspace);
    AttnArgs a{};
    a.q = q; a.q_sb = q_sb; a.q_ss = q_ss; a.q_sh = q_sh;
    a.B = (int)B; a.Sq = (int)Sq; a.Hq = (int)Hq; a.Hk = (int)Hk; a.G = (int)(Hq / Hk);
    a.rows = (int)rows; a.row_blocks = (int)row_blocks; a.dtype = dtype;
    a.q_vec = rows_aligned(q, dtype, q_sb, q_ss, q_sh);
    a.pool = static_cast<const unsigned char *>(pool);
    a.table = Table{page_table, table_stride, (int)max_pages, (int)num_pages, ilog2(page_size), status};
    a.lengths = lengths; a.selected = selected; a.n_selected = (int)n_selected;
    const float s = softmax_scale * 1.44269504088896341f;
    // a factor of zero would turn a masked score into a NaN; this one rounds every score to zero
    a.scale = s < 0.f ? -s : s > 1e-30f ? s : 1e-30f;
    a.sign = s < 0.f ? -1.f : 1.f;
    a.out = out; a.o_sb = o_sb; a.o_ss = o_ss; a.o_sh = o_sh; a.lse = lse;
    a.counters = reinterpret_cast<int *>(ws + 256);
    a.parts = reinterpret_cast<float *>(ws + counter_bytes(B * Hk * ((rows + 3) / 4)));
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_head_dim(D, [&](auto w) {
        auto launch = [&](auto n, auto lm) {
            constexpr int W = decltype(w)::value, NT = decltype(n)::value, L = decltype(lm)::value;
            const int blocks = wave<W, NT, L>();
            if (!blocks) { set_error("kv4_attn: the kernel does not fit this device"); return FC_ECUDA; }
            attn_kernel<W, NT, L><<<blocks, kThreads, Attn<W, NT, L>::SMEM, st>>>(a);
            return check_launch("kv4_attn");
        };
        using I1 = std::integral_constant<int, 1>;
        using I2 = std::integral_constant<int, 2>;
        if (limbs == 1) return nt == 1 ? launch(I1(), I1()) : launch(I2(), I1());
        return nt == 1 ? launch(I1(), I2()) : launch(I2(), I2());
    });
}
