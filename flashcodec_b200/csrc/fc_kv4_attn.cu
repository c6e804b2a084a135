// Paged 4-bit KV cache: attention of one or a few new tokens.
//
//   out = softmax(scale * q . K^T) . V,  K = code * scale per group of 32 channels
//
// Every held byte is read once per KV head and block of 8 query rows (4 of fp16 or fp32;
// twice that with two column blocks): 4.5 bits a value, so HBM bounds it from below at 144
// bytes a token and head at D = 128, and each value takes part in Hq / Hk products on each
// side.  What competes with HBM is the issue rate: at
// 6.4 TB/s an SM receives 46 values a cycle to unpack.  So the pages are stored in
// the operand order of mma.m16n8k16 (fc_kv4.cuh): tokens (K) or channels (V) in the 16
// rows, the group's query rows in the 8 columns, and nothing is exchanged between lanes
// but a transposition of the weights (movmatrix).  Matrix instructions that read shared
// memory (tcgen05) would need the unpacked values written back there, 4 bytes moved for
// every half byte that arrives.
//
// Codes.  A nibble in the low bits of an fp16 is a subnormal, its multiple of 2^-24, so
// with bf16 queries a word becomes operands by five ANDs and shifts, and the products are
// exact.  What is left is the 8 that is on every stored code: for the scores a product of
// the tokens' scales with -8 * (sum of q of each group), one more matrix instruction for
// 16 tokens; for the output the groups' sums of weight * scale, one with an operand of
// eights for each group, taken off every 256 tokens.  The tensor cores add subnormal
// products with about 2^-17 of the largest, enough beside 2^-9 of a bf16 query; fp16 and
// fp32 queries get codes made exact (fp16 1024 + u, minus 1032) and two fp16 parts in
// neighbouring columns (22 bits).
// Queries are scaled by a power of two per row so that fp16 holds them.  A group of 32
// channels is two matrix instructions; its scale comes in after it, in fp32.
//
// Weights.  Base-2 softmax with a running reference per row, moved only when a score
// passes it by 2^4, and a running power of two above the values' scales, so that
// weight * scale, an fp16 operand, is at most 2^15.  fp16 and fp32 queries: the product is
// rounded once, to two fp16 parts; the power of two follows the scales from fp16's least on,
// so that the largest weight and scale make 2^10 or more.  bf16 queries: the weight is
// rounded to fp16 and the product again (2^-11 each); a weight has to fit fp16 by itself, so
// the power of two is 1 at least, and where all scales are below 2^-10 the products of
// weights under 2^-14 of the largest are subnormal.
//
// Work.  The chunks (64 tokens; 32 where pages are smaller, heads wider than 128 or pages
// selected) of all (sequence, KV head, row block) are one line, cut into equal pieces for one wave of blocks, whatever the lengths; the lengths are
// read on the device.  A block's 4 warps take the chunks of its piece in turn, each
// with its own ring of asynchronous copies and its own running state.  Pieces of one
// (sequence, head) are joined by the last block to finish, in order: the result does
// not depend on timing.  No block waits for another.
//
// 16 sequences of 32768 tokens, 32/8 heads, D = 128, bf16 (604 MB): 124 us under sustained
// load, 4.9 TB/s, 76 % of the copy rate, where the power cap holds the SMs at 1.75 GHz; 107.5
// us, 87 %, in short runs (fp16 queries 125).  The copies alone take 100 us; the rest is the
// latency of 12 warps' own instructions (1.9 of 4 a cycle and SM, 228 for 16 tokens).  3 blocks of 168 registers an
// SM; 4 of 128 spill (121 us), 5 warps a block too.  Bulk copies in place of cp.async were
// slower (127 us against 123 at that time), chunks of 32 tokens are by 6 %.
#include "fc_attn_common.cuh"
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
    float *aside;   // one per warp: the state of its earlier spans
};

constexpr int kWarps = 4, kThreads = 32 * kWarps;
// What a segment costs beyond its chunks (queries, the pipeline's start, the joins), in
// chunks of its block's 4 warps; a block's least piece is a chunk for every warp more.
// Times in us for 0 / 8 / 16 / 32 chunks of 32 tokens (one column block): 16 sequences of
// 32768 tokens 115 / 113 / 112 / 111, 61 of 1..12000 58 / 23 / 20 / 21; with two column
// blocks, whose joins are twice as long: 24 sequences of 1..9000 with 16 rows 194 / 52 /
// 41 / 36.
constexpr int overhead(int NT, int TILES) { return (NT == 1 ? 32 : 64) / TILES; }
constexpr float kSlack = 4.f;    // log2 of how far a score may pass the reference
constexpr float kNone = -3e38f;  // the reference of a row that has seen no token
// Beyond this a reference 2^11 (2^35) below a score and the score cannot both be told from their
// neighbours: scores of 2^27 and more came out as zeros or NaN.  The reference is then the
// largest rounded score itself and weights are at most 1, which fits fp16 with every scale.
constexpr float kLarge = 0x1p22f;

__device__ __forceinline__ void mma16816(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ... with nothing to add to
__device__ __forceinline__ void mma16816_first(float d[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(y) : "r"(x), "r"(mask), "r"(0x64006400u));
    return y;
}

// The four pairs of a word.  RAW: as fp16 subnormals u 2^-24, 16 u 2^-24, u 2^-24,
// 16 u 2^-24 (u = code + 8: a nibble in the low bits of a half is that multiple of
// 2^-24); else as codes.
template <bool RAW>
__device__ __forceinline__ void unpack(uint32_t w, uint32_t p[4]) {
    const uint32_t s = w >> 8;
    if constexpr (RAW) {
        p[0] = w & 0x000f000fu;
        p[1] = w & 0x00f000f0u;
        p[2] = s & 0x000f000fu;
        p[3] = s & 0x00f000f0u;
    } else {
        const __half2 one = __float2half2_rn(-1032.f), sixteenth = __float2half2_rn(0.0625f),
                      off = __float2half2_rn(-72.f);
        p[0] = u32(__hadd2(h2(and_or(w, 0x000f000fu)), one));
        p[1] = u32(__hfma2(h2(and_or(w, 0x00f000f0u)), sixteenth, off));
        p[2] = u32(__hadd2(h2(and_or(s, 0x000f000fu)), one));
        p[3] = u32(__hfma2(h2(and_or(s, 0x00f000f0u)), sixteenth, off));
    }
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

template <int W, int NT, int LIMBS, int TILES, bool RUNS>
struct Attn {
    static constexpr int D = 32 * W, TILE = tile_bytes(W), STAGE = TILES * TILE;
    static constexpr int kStages = TILES == 4 ? 2 : 3;
    static constexpr int RPC = 8 * NT / LIMBS;  // query rows of a block
    static constexpr int H = (W + 1) / 2;       // pairs of groups
    static constexpr bool RAW = LIMBS == 1;     // how codes become operands
    static constexpr int RING = kStages * STAGE;
    static constexpr int SMEM = kWarps * RING;

    const AttnArgs &a;
    unsigned char *ring;  // of this warp
    int *pos_s;           // (kStages, TILES) first positions of the staged tiles
    // Where the bound above the values' scales begins: weight * scale <= kSlim * 2^kLim = 2^15.
    // Two fp16 parts of a product hold 22 bits of it down to about 2^-2, so the bound follows the
    // scales from the least there is; from 1 on, values near 1e-4 lost half of those bits and
    // values near 1e-5 all but a few.  A weight that is an fp16 operand itself stays below 2^15.
    static constexpr float kLim = LIMBS == 2 ? 39.f : 15.f, kSlim = LIMBS == 2 ? 0x1p-24f : 1.f;
    int warp, lane, r, c;
    // this segment
    int b, h, rb, len, chunk0, chunk1;
    int log_tpp, pages;
    const unsigned char *base_ptr;
    uint32_t page_stride;  // bytes
    // queries: operand words, those of the groups' offsets, factors and lengths seen
    uint32_t qb[NT][2 * W][2], qo[RAW ? NT : 1][2];
    float f[NT][2];
    int seen[NT][2], min_seen;
    // running state: references, sums, outputs, sums of weight * scale of each group
    float M[NT][2], l[NT][2], acc[NT][2 * W][4], ws[RAW ? NT : 1][W][2];
    float lim, slim;
    bool large;  // a row of this warp has a reference beyond kLarge

    __device__ __forceinline__ Attn(const AttnArgs &args, unsigned char *smem, int *pos)
        : a(args) {
        warp = threadIdx.x >> 5;
        lane = threadIdx.x & 31;
        r = lane >> 2;
        c = lane & 3;
        ring = smem + warp * RING;
        pos_s = pos + warp * kStages * TILES;
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
                    const bool sixteen = RAW && (i >> 1) & 1;  // codes that come as 16 u
                    float u = x[8 * j + i] * up, v = x[8 * j + i + 1] * up;
                    if (sixteen) { u *= 0.0625f; v *= 0.0625f; }
                    __half2 p = __floats2half2_rn(u, v);
                    if constexpr (LIMBS == 2) {
                        if (r & 1) {
                            const float2 hi = __half22float2(p);
                            p = __floats2half2_rn(u - hi.x, v - hi.y);
                        }
                    }
                    const float2 z = __half22float2(p);
                    sum[j] -= (sixteen ? 128.f : 8.f) * 0x1p-24f * (z.x + z.y);
                    qb[nt][2 * j + (i >> 2)][(i >> 1) & 1] = u32(p);
                }
                if constexpr (RAW) {
                    sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
                    sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
                }
            }
            // -8 sum(q) of every group, as two fp16 parts: slot c (and c + 4) of the offsets'
            // operand holds part slot / H of the groups 2 (slot % H) and the next
#pragma unroll
            for (int y = 0; y < (RAW ? 2 : 0); y++) {
                float lo[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int slot = c + 4 * y, g = 2 * (slot % H) + e;
                    float v = 0.f;
#pragma unroll
                    for (int j = 0; j < W; j++)
                        if (g == j) v = sum[j];
                    if (slot >= H) v -= __half2float(__float2half_rn(v));
                    if (slot >= 2 * H) v = 0.f;
                    lo[e] = v;
                }
                qo[nt][y] = u32(__floats2half2_rn(lo[0], lo[1]));
            }
            // what belongs to a column, from the lanes that hold it to those that score it
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const int from = (2 * c + y) * 4;
                // neither zero, which would make a masked score a NaN, nor infinity, which would a
                // score of zero: scores beyond those are ones that round to zero, and ones whose
                // weights are one and zeros at this factor too (their logarithm is not kept)
                f[nt][y] = __shfl_sync(0xffffffffu, down, from) * a.scale * (RAW ? 0x1p24f : 1.f);
                f[nt][y] = fminf(fmaxf(f[nt][y], 1e-37f), 3.4028234e38f);
                const int sq = min(row_of(nt, 2 * c + y), a.rows - 1) / a.G;
                seen[nt][y] = len - (a.Sq - 1 - sq);
            }
        }
        // row blocks hold rows in order: the first one sees least
        min_seen = len - (a.Sq - 1 - min(rb * RPC, a.rows - 1) / a.G);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int y = 0; y < 2; y++) { M[nt][y] = kNone; l[nt][y] = 0.f; }
#pragma unroll
            for (int m = 0; m < 2 * W; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[nt][m][i] = 0.f;
            if constexpr (RAW) {
#pragma unroll
                for (int j = 0; j < W; j++) ws[nt][j][0] = ws[nt][j][1] = 0.f;
            }
        }
        lim = kLim;
        slim = kSlim;
        large = false;
    }

    // ------------------------------------------------------------------ copies
    // The page of the sequence that holds tile `tile` (of its tokens, or of the
    // selected pages), or -1; where that lies in the pool.
    __device__ __forceinline__ int logical(int tile) const {
        int page = tile >> log_tpp;
        if (a.selected) {
            if (page >= a.n_selected) return -1;
            page = a.selected[((int64_t)b * a.Hk + h) * a.n_selected + page];
        }
        return (unsigned)page < (unsigned)pages ? page : -1;
    }
    __device__ __forceinline__ int physical(int page) const {
        return page < 0 ? -1 : a.table.page(b, page);
    }
    static constexpr int kNowhere = 0x7fffffff - 64;  // a position past every length

    // The common case: all tokens of the sequence, pages of a chunk's tokens and more, so
    // that a chunk is one run of bytes.  `tile`: of the page; n: tokens held from there on.
    __device__ __forceinline__ void issue_run(int tile, int id, int n, int stage) const {
        constexpr int N = TILE / 16;  // 36 W pieces of a tile
        unsigned char *dst = ring + stage * STAGE + lane * 16;
        const unsigned char *s =
            base_ptr + lane * 16 + (uint64_t)(uint32_t)id * page_stride + (uint32_t)(tile * TILE);
        const int tiles = (n + 15) / 16;
        if (tiles >= TILES) {
#pragma unroll
            for (int i = 0; i < (TILES * N + 31) / 32; i++)
                if (32 * i + 31 < TILES * N || lane < TILES * N - 32 * i) cp_async16(dst + 512 * i, s + 512 * i);
        } else {
            const int left = tiles * N - lane;
#pragma unroll 1
            for (int i = 0; 32 * i < left; i++) cp_async16(dst + 512 * i, s + 512 * i);
        }
    }

    // Any other: lane y has looked tile y up (`page` of the sequence, `id`).
    __device__ __forceinline__ void issue_tiles(int chunk, int page, int id, int stage) const {
        constexpr int N = TILE / 16;
        const int tile = (TILES * chunk + lane % TILES) & ((1 << log_tpp) - 1);
        const int p = (page << a.table.log_page) + tile * 16;
        if (page < 0 || p >= len) id = -1;
        if (lane < TILES) pos_s[stage * TILES + lane] = id < 0 ? kNowhere : p;
        const unsigned char *s = base_ptr + (uint64_t)(uint32_t)id * page_stride + (uint32_t)(tile * TILE);
#pragma unroll
        for (int y = 0; y < TILES; y++) {
            const unsigned char *z = reinterpret_cast<const unsigned char *>(
                __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(s), y));
            if (__shfl_sync(0xffffffffu, id, y) < 0) continue;
#pragma unroll
            for (int i = 0; i < (N + 31) / 32; i++)
                if (32 * i + 31 < N || lane < N - 32 * i)
                    cp_async16(ring + stage * STAGE + y * TILE + lane * 16 + 512 * i, z + lane * 16 + 512 * i);
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
        if constexpr (RAW) {
            // the offsets of all groups: a product of the tokens' scales with -8 sum(q)
            uint32_t o[4];
            if constexpr (W % 2 == 0) {
                const uint32_t *p = reinterpret_cast<const uint32_t *>(tile + ks_off(W)) + r * W;
                o[0] = p[c % H];
                o[1] = p[H + c % H];
                o[2] = H > 2 ? p[(c + 4) % H] : o[0];
                o[3] = H > 2 ? p[H + (c + 4) % H] : o[1];
            } else {
                const uint16_t *p = reinterpret_cast<const uint16_t *>(tile + ks_off(W)) + r * 2 * W;
                const int g = 2 * (c % H), g1 = min(g + 1, W - 1);
                o[0] = o[2] = p[g] | (uint32_t)p[g1] << 16;
                o[1] = o[3] = p[W + g] | (uint32_t)p[W + g1] << 16;
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++) mma16816_first(S[nt], o, qo[nt][0], qo[nt][1]);
        }
#pragma unroll
        for (int j = 0; j < W; j++) {
            uint32_t x[4], y[4];
            unpack<RAW>(k0[j], x);
            unpack<RAW>(k1[j], y);
            const uint32_t a0[4] = {x[0], y[0], x[1], y[1]}, a1[4] = {x[2], y[2], x[3], y[3]};
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float t[4];
                mma16816_first(t, a0, qb[nt][2 * j][0], qb[nt][2 * j][1]);
                mma16816(t, a1, qb[nt][2 * j + 1][0], qb[nt][2 * j + 1][1]);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    S[nt][i] = RAW || j ? fmaf(s[(i >> 1) * W + j], t[i], S[nt][i]) : s[(i >> 1) * W + j] * t[i];
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

    // out += V . weights of one tile; p: the weights.  RAW: in units of 2^-24 (channels
    // r + 8: 2^-20) and without the 8 off every code; ws gets 8 times the groups' sums of
    // weight * scale, in 2^-24 too.  MASKED: some weights are of tokens not seen, whose
    // scales may be NaN.
    template <bool MASKED>
    __device__ __forceinline__ void gather(const unsigned char *tile, const float p[NT][4],
                                           float out[NT][2 * W][4]) {
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
                    if constexpr (MASKED) {
                        w[nt][j][0] &= __hne2_mask(h2(lo), h2(0u));
                        w[nt][j][1] &= __hne2_mask(h2(hi), h2(0u));
                    }
                }
            }
        } else {
            const __half *vs = reinterpret_cast<const __half *>(tile + vs_off(W)) + (r >> 1) * 4 * W + (r & 1);
#pragma unroll
            for (int j = 0; j < W; j++) {
                const float s0 = __half2float(vs[4 * j]), s1 = __half2float(vs[4 * j + 2]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float u = MASKED && p[nt][0] == 0.f ? 0.f : p[nt][0] * s0;
                    const float z = MASKED && p[nt][2] == 0.f ? 0.f : p[nt][2] * s1;
                    const __half uh = __float2half_rn(u), zh = __float2half_rn(z);
                    w[nt][j][0] = transpose8(u32(__halves2half2(uh, __float2half_rn(u - __half2float(uh)))));
                    w[nt][j][1] = transpose8(u32(__halves2half2(zh, __float2half_rn(z - __half2float(zh)))));
                }
            }
        }
        if constexpr (RAW) {
            const uint32_t eight[4] = {0x00080008u, 0x00080008u, 0x00080008u, 0x00080008u};
#pragma unroll
            for (int j = 0; j < W; j++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float sum[4];  // of every row
                    mma16816_first(sum, eight, w[nt][j][0], w[nt][j][1]);
                    const float2 s = __fadd2_rn(make_float2(ws[nt][j][0], ws[nt][j][1]), make_float2(sum[0], sum[1]));
                    ws[nt][j][0] = s.x;
                    ws[nt][j][1] = s.y;
                }
        }
#pragma unroll
        for (int m = 0; m < 2 * W; m++) {
            uint32_t x[4];
            unpack<RAW>(v[m], x);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) mma16816(out[nt][m], x, w[nt][m / 2][0], w[nt][m / 2][1]);
        }
    }

    // All tiles of a chunk.
    template <bool MASKED>
    __device__ __forceinline__ void gather_chunk(const unsigned char *tile, const float S[TILES][NT][4]) {
        if constexpr (RAW) {
#pragma unroll
            for (int t = 0; t < TILES; t++) gather<MASKED>(tile + t * TILE, S[t], acc);
        } else {
            // a chunk's sum by itself: the long sum is then in rounded fp32 additions
            float part[NT][2 * W][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int m = 0; m < 2 * W; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++) part[nt][m][i] = 0.f;
#pragma unroll
            for (int t = 0; t < TILES; t++) gather<MASKED>(tile + t * TILE, S[t], part);
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int m = 0; m < 2 * W; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[nt][m][i] += part[nt][m][i];
        }
    }

    // The staged chunk, whose tile t holds the positions from p[t].
    __device__ __forceinline__ void chunk(int stage, const int p[TILES]) {
        unsigned char *tile = ring + stage * STAGE;
        float S[TILES][NT][4];
        int last = p[0];
#pragma unroll
        for (int t = 0; t < TILES; t++) {
            score(tile + t * TILE, S[t]);
            last = max(last, p[t]);
        }
        const bool masked = last + 16 > min_seen;
        if (masked) {
#pragma unroll
            for (int t = 0; t < TILES; t++) mask(tile + t * TILE, p[t], S[t]);
            __syncwarp();
        }
        // does a score pass its reference, or a scale of the values the running bound?
        // (this lane's share of the scales: TILES W / 2 of a tile)
        constexpr int SH = TILES * W / 2, LT = 32 / TILES;
        uint32_t sv[(SH + 1) / 2];
        {
            const unsigned char *q = tile + lane / LT * TILE + vs_off(W) + lane % LT * 2 * SH;
            if constexpr (SH % 2 == 0) {
                load_words<SH / 2>(q, sv);
            } else {
#pragma unroll
                for (int i = 0; i < (SH + 1) / 2; i++)  // an odd number: the last word holds one twice
                    sv[i] = reinterpret_cast<const uint16_t *>(q)[2 * i] |
                            (uint32_t)reinterpret_cast<const uint16_t *>(q)[min(2 * i + 1, SH - 1)] << 16;
            }
        }
        __half2 st = h2(sv[0]);
#pragma unroll
        for (int i = 1; i < (SH + 1) / 2; i++) st = __hmax2(st, h2(sv[i]));
        const float sm = __half2float(__hmax(__low2half(st), __high2half(st)));
        bool pass = sm > slim || large;
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                top[nt][y] = fmaxf(S[0][nt][y], S[0][nt][y + 2]);
#pragma unroll
                for (int t = 1; t < TILES; t++) top[nt][y] = fmaxf(top[nt][y], fmaxf(S[t][nt][y], S[t][nt][y + 2]));
                pass = pass || fmaf(top[nt][y], f[nt][y], -M[nt][y]) > lim;
            }
        if (__any_sync(0xffffffffu, pass)) {
            float s = sm;
#pragma unroll
            for (int o = 16; o; o /= 2) s = fmaxf(s, __shfl_xor_sync(0xffffffffu, s, o));
            const float old = lim;
            bool far = false;
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
                    const bool any = t > -INFINITY;
                    float m = M[nt][y] + (old - lim);
                    if (any) m = fmaxf(m, fmaf(t, f[nt][y], -(lim - kSlack)));
                    if (fabsf(m) > kLarge) {  // a number that no score is above
                        m = fabsf(M[nt][y]) > kLarge ? M[nt][y] : M[nt][y] + fmaxf(old, 0.f);
                        if (any) m = fmaxf(m, __fmul_rn(t, f[nt][y]));
                        far = far || m > kNone;
                    }
                    const float g = exp2_fast(M[nt][y] - m);
                    M[nt][y] = m;
                    l[nt][y] *= g;
                    if constexpr (RAW) {
#pragma unroll
                        for (int j = 0; j < W; j++) ws[nt][j][y] *= g;
                    }
#pragma unroll
                    for (int i = 0; i < 2 * W; i++) {
                        acc[nt][i][y] *= g;
                        acc[nt][i][y + 2] *= g;
                    }
                }
            large = __any_sync(0xffffffffu, far);
        }
        auto weights = [&](auto exponents) {
#pragma unroll
            for (int t = 0; t < TILES; t++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        const float2 x = exponents(make_float2(S[t][nt][i], S[t][nt][i + 1]), nt);
                        S[t][nt][i] = exp2_fast(x.x);
                        S[t][nt][i + 1] = exp2_fast(x.y);
                        const float2 s = __fadd2_rn(make_float2(l[nt][0], l[nt][1]),
                                                    make_float2(S[t][nt][i], S[t][nt][i + 1]));
                        l[nt][0] = s.x;
                        l[nt][1] = s.y;
                    }
        };
        if (large)
            weights([&](float2 x, int nt) {
                return make_float2(__fsub_rn(__fmul_rn(x.x, f[nt][0]), M[nt][0]),
                                   __fsub_rn(__fmul_rn(x.y, f[nt][1]), M[nt][1]));
            });
        else
            weights([&](float2 x, int nt) {
                return __ffma2_rn(x, make_float2(f[nt][0], f[nt][1]), make_float2(-M[nt][0], -M[nt][1]));
            });
        if (masked)
            gather_chunk<true>(tile, S);
        else
            gather_chunk<false>(tile, S);
    }

    // The 8 on every code comes off the sums.  The tensor cores cut what they add to, so a
    // sum that only grows (8 times the weights, where the codes themselves cancel) would lose
    // an ulp of itself at every step, always downward: flat weights over 262,144 tokens were
    // half off.  Centred every 256 tokens, it loses below 2^-16 of a code's step.
    static constexpr int kCentre = 16 / TILES;
    __device__ __forceinline__ void centre() {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < W; j++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
#pragma unroll
                    for (int m = 2 * j; m < 2 * j + 2; m++) {
                        acc[nt][m][y] -= ws[nt][j][y];
                        acc[nt][m][y + 2] = fmaf(-16.f, ws[nt][j][y], acc[nt][m][y + 2]);  // these came as 16 u
                    }
                    ws[nt][j][y] = 0.f;
                }
    }

    // Centred sums still grow where the values have a mean, and lose to the same cut: values
    // around 3, then around -3, over 262,144 tokens of a warp were 2e-3 off.  So a segment is
    // run in spans of 4096 tokens a warp (256 steps: below 2^-16 of the sum on average), whose
    // states are joined in rounded fp32 in the workspace, as the registers are the loop's and the
    // rings fill shared memory.  200 x 65536 tokens of one head (two spans a segment): 285 us
    // with and without.
    static constexpr int kSpan = 4096 / (16 * TILES) * kWarps;  // chunks
    static constexpr int ASIDE = (4 + 8 * W) * NT * 32;  // floats of a warp: references, sums, outputs
    // Joins the state with the one put aside (`more`: there is one); `last`: stays in registers.
    __device__ __forceinline__ void put_aside(bool more, bool last) {
        centre();
        float *z = a.aside + ((int64_t)blockIdx.x * kWarps + warp) * ASIDE + lane;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float g[2], h[2];
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const float held = more ? z[32 * y] : M[nt][y], m = fmaxf(held, M[nt][y]);
                g[y] = exp2_fast(M[nt][y] - m);
                h[y] = exp2_fast(held - m);
                M[nt][y] = m;
                l[nt][y] = fmaf(l[nt][y], g[y], more ? z[32 * (2 + y)] * h[y] : 0.f);
                if (!last) {
                    z[32 * y] = m;
                    z[32 * (2 + y)] = l[nt][y];
                }
            }
#pragma unroll
            for (int m = 0; m < 2 * W; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float *v = z + 32 * (4 + 4 * m + i);
                    acc[nt][m][i] = fmaf(acc[nt][m][i], g[i & 1], more ? *v * h[i & 1] : 0.f);
                    if (!last) *v = acc[nt][m][i];
                }
            z += 32 * (4 + 8 * W);
        }
    }

    // This warp's chunks of the segment: chunk0 + warp, + 4, ..., each copied
    // kStages - 1 rounds before it is used.
    __device__ __forceinline__ void run() {
        pages = (len + (1 << a.table.log_page) - 1) >> a.table.log_page;
        base_ptr = a.pool + ((int64_t)h << log_tpp) * TILE;
        page_stride = (uint32_t)((a.Hk << log_tpp) * TILE);
        if constexpr (RUNS)
            run_pages();
        else
            run_tiles();
    }

    // fetch(stage) copies the next chunk, use(i, stage) works on chunk i.
    template <typename Fetch, typename Use>
    __device__ __forceinline__ void rounds(Fetch fetch, Use use) {
#pragma unroll
        for (int i = 0; i < kStages - 1; i++) {
            if (chunk0 + warp + i * kWarps < chunk1) fetch(i);
            cp_async_commit();
        }
        load_queries();  // while the first chunks are on their way
        int stage = 0;
        for (int i = chunk0 + warp; i < chunk1; i += kWarps) {
            cp_async_wait<kStages - 2>();
            __syncwarp();
            if (i + (kStages - 1) * kWarps < chunk1) fetch(stage == 0 ? kStages - 1 : stage - 1);
            cp_async_commit();
            use(i, stage);
            if constexpr (RAW) {
                if (i / kWarps % kCentre == kCentre - 1) centre();
            }
            __syncwarp();
            stage = stage == kStages - 1 ? 0 : stage + 1;
        }
        cp_async_wait<0>();
    }

    __device__ __forceinline__ void run_pages() {
        // lane i holds the page of the chunk i rounds into a window of 32 rounds; the
        // window after it is on its way
        constexpr int LOG = TILES == 4 ? 2 : 1;
        const int shift = log_tpp - LOG;
        int next = chunk0 + warp, round = 0;
        auto window = [&](int first) {
            const int chunk = first + kWarps * lane;
            return chunk < chunk1 ? a.table.page(b, chunk >> shift) : 0;
        };
        int ids = window(next), ids2 = window(next + 32 * kWarps);
        rounds(
            [&](int stage) {
                const int id = __shfl_sync(0xffffffffu, ids, round);
                issue_run((next & ((1 << shift) - 1)) << LOG, id, len - 16 * TILES * next, stage);
                next += kWarps;
                if (++round == 32) {
                    round = 0;
                    ids = ids2;
                    ids2 = window(next + 32 * kWarps);
                }
            },
            [&](int i, int stage) {
                int p[TILES];
#pragma unroll
                for (int t = 0; t < TILES; t++) p[t] = 16 * (TILES * i + t);
                chunk(stage, p);
            });
    }

    __device__ __forceinline__ void run_tiles() {
        const int y = lane % TILES;
        int next = chunk0 + warp;  // the next chunk to copy
        int page = next < chunk1 ? logical(TILES * next + y) : -1;
        int id = physical(page);
        int page2 = next + kWarps < chunk1 ? logical(TILES * (next + kWarps) + y) : -1;
        rounds(
            [&](int stage) {
                issue_tiles(next, page, id, stage);
                next += kWarps;
                page = page2;
                id = physical(page);
                page2 = next + kWarps < chunk1 ? logical(TILES * (next + kWarps) + y) : -1;
            },
            [&](int, int stage) {
                int p[TILES], least = kNowhere;
#pragma unroll
                for (int t = 0; t < TILES; t++) {
                    p[t] = pos_s[stage * TILES + t];
                    least = min(least, p[t]);
                }
                if (least < len) chunk(stage, p);
            });
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
                const float g = exp2_fast(M[nt][y] - m) * (RAW ? 0x1p24f : 1.f);
#pragma unroll
                for (int i = 0; i < 2 * W; i++) {
                    float u = acc[nt][i][y], v = acc[nt][i][y + 2];
                    if constexpr (RAW) {
                        u -= ws[nt][i / 2][y];
                        v = fmaf(v, 0.0625f, -ws[nt][i / 2][y]);
                    } else {
                        u += acc[nt][i][1];
                        v += acc[nt][i][3];
                    }
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

    // Joins `count` parts of this unit: block `first`'s second one, then the first
    // ones of the blocks after it.
    __device__ __forceinline__ void merge(int first, int count) const {
        const float *p0 = a.parts + ((int64_t)first * 2 + 1) * PART;
        const float *p1 = a.parts + (int64_t)first * 2 * PART;  // block first + k: + 2 k PART
        const int rows = min(RPC, a.rows - rb * RPC);
        for (int i = threadIdx.x * 4; i < rows * D; i += kThreads * 4) {
            const int row = i / D, at = RPC * D + 2 * row;
            float m = __ldcg(p0 + at);
#pragma unroll 4
            for (int k = 1; k < count; k++) m = fmaxf(m, __ldcg(p1 + (int64_t)2 * k * PART + at));
            float s = 0.f;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int k = 0; k < count; k++) {
                const float *p = k ? p1 + (int64_t)2 * k * PART : p0;
                const float2 z = __ldcg(reinterpret_cast<const float2 *>(p + at));
                const float4 o = __ldcg(reinterpret_cast<const float4 *>(p + i));
                const float g = exp2_fast(z.x - m);
                s = fmaf(g, z.y, s);
                v.x = fmaf(g, o.x, v.x);
                v.y = fmaf(g, o.y, v.y);
                v.z = fmaf(g, o.z, v.z);
                v.w = fmaf(g, o.w, v.w);
            }
            const float inv = s == 0.f ? 0.f : 1.f / s;
            const float x[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
#pragma unroll
            for (int j = 0; j < 4; j++) write_row(rb * RPC + row, i % D + j, x[j]);
            if (a.lse && i % D == 0) write_lse(rb * RPC + row, m, s);
        }
    }
};

// A sequence, in the sums of the line's lengths (at most 2^18 of up to 2^26).
constexpr int64_t kOne = int64_t(1) << 44;

// Chunks of sequence b, 0 where it holds nothing.
template <int TILES>
__device__ __forceinline__ int chunks_of(const AttnArgs &a, int64_t b) {
    const int len = a.table.length(a.lengths[b]);
    if (len <= 0) return 0;
    if (a.selected) return ((a.n_selected << (a.table.log_page - 4)) + TILES - 1) / TILES;
    return (len + 16 * TILES - 1) / (16 * TILES);
}

// Where a block is on the line.
struct Plan {
    int64_t U, blocks, x, end, base;  // base: where the line of sequence b begins
    int b, n, unit;                   // n: chunks of a unit of b
};

// The line: unit (sequence, KV head, row block) u of n > 0 chunks is n + OVERHEAD
// long, the first OVERHEAD standing for what a segment costs beyond its chunks.
// Block i of `blocks` has the piece [U i / blocks, U (i + 1) / blocks).
template <int W, int NT, int LIMBS, int TILES, bool RUNS>
__global__ void __launch_bounds__(kThreads, NT == 1 && W <= 4 ? 3 : 2) attn_kernel(const __grid_constant__ AttnArgs a) {
    using A = Attn<W, NT, LIMBS, TILES, RUNS>;
    constexpr int OVERHEAD = overhead(NT, TILES), MIN_PIECE = OVERHEAD + kWarps;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int64_t sums[kWarps];
    __shared__ Plan plan;
    __shared__ int first_s, last_s, most[kWarps];
    __shared__ int pos[kWarps * A::kStages * TILES];
    __shared__ float ml[kWarps * A::RPC * 2];

    const int HR = a.Hk * a.row_blocks;
    const int per = (a.B + kThreads - 1) / kThreads;
    const int b0 = min((int)threadIdx.x * per, a.B), b1 = min(b0 + per, a.B);
    int64_t mine = 0;
    int longest = 0;
    for (int b = b0; b < b1; b++) {
        const int n = chunks_of<TILES>(a, b);
        longest = max(longest, n + OVERHEAD);
        mine += n ? n + OVERHEAD + kOne : 0;
    }
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if ((threadIdx.x & 31) >= o) upto += v;
    }
    if ((threadIdx.x & 31) == 31) sums[threadIdx.x >> 5] = upto;
    longest = __reduce_max_sync(0xffffffffu, longest);
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = longest;
    for (int b = blockIdx.x; b < a.B; b += gridDim.x) {  // nothing held: zeros
        if (chunks_of<TILES>(a, b)) continue;
        for (int64_t i = threadIdx.x; i < (int64_t)a.Sq * a.Hq * A::D; i += kThreads) {
            const int64_t row = i / A::D, s = row / a.Hq;
            store_from_f32(a.out, b * a.o_sb + s * a.o_ss + (row - s * a.Hq) * a.o_sh + i % A::D, a.dtype, 0.f);
            if (a.lse && i % A::D == 0) a.lse[(int64_t)b * a.Sq * a.Hq + row] = -INFINITY;
        }
    }
    __syncthreads();
    int64_t before = upto - mine, all = 0;  // lengths, and sequences from kOne on
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
        if (w < (int)(threadIdx.x >> 5)) before += sums[w];
        all += sums[w];
        longest = max(longest, most[w]);
    }
    before &= kOne - 1;
    mine &= kOne - 1;
    const int64_t U = (all & (kOne - 1)) * HR, units = (all / kOne) * HR;
    int64_t blocks = min((int64_t)gridDim.x, (U + MIN_PIECE - 1) / MIN_PIECE);
    // Equal units that are short: one block for each, no piece crossing from one to the
    // next (one sequence of 517 tokens: 11.4 us, 12.6 across; 3 of one token: 7.6, 11.4).
    if (units && units <= gridDim.x && longest < 2 * MIN_PIECE && U == units * longest) blocks = units;
    if ((int64_t)blockIdx.x >= blocks) return;
    const int64_t x0 = U * blockIdx.x / blocks;
    // the sequence that the piece begins in
    if (x0 >= before * HR && x0 < (before + mine) * HR) {
        int64_t at = before * HR;
        int b = b0, n;
        for (;; b++) {
            n = chunks_of<TILES>(a, b);
            const int64_t w = n ? (int64_t)(n + OVERHEAD) * HR : 0;
            if (x0 < at + w) break;
            at += w;
        }
        plan.U = U;
        plan.blocks = blocks;
        plan.x = x0;
        plan.end = U * (blockIdx.x + 1) / blocks;
        plan.base = at;
        plan.b = b;
        plan.n = n;
        plan.unit = (int)((x0 - at) / (n + OVERHEAD));
    }
    __syncthreads();

    // (the plan stays in shared memory: its registers are the segment's)
    A t(a, smem, pos);
    while (plan.x < plan.end) {
        auto first_chunk = [&] { return plan.base + (int64_t)plan.unit * (plan.n + OVERHEAD) + OVERHEAD; };
        auto begin = [&] { return (int)max(plan.x - first_chunk(), (int64_t)0); };
        auto end = [&] { return (int)min(plan.end - first_chunk(), (int64_t)plan.n); };
        if (begin() < end()) {
            t.b = plan.b;
            t.h = plan.unit / a.row_blocks;
            t.rb = plan.unit - t.h * a.row_blocks;
            t.len = a.table.length(a.lengths[t.b]);
            if constexpr (A::RAW) {
                t.chunk1 = begin();
                do {
                    t.chunk0 = t.chunk1;
                    t.chunk1 = min(t.chunk0 + A::kSpan, end());
                    t.run();
                    if (end() - begin() > A::kSpan) t.put_aside(t.chunk0 > begin(), t.chunk1 == end());
                } while (t.chunk1 < end());
            } else {
                t.chunk0 = begin();
                t.chunk1 = end();
                t.run();
            }
            const bool whole = begin() == 0 && end() == plan.n;
            // parts of a block: 0 of a unit that began in an earlier one, 1 of one that ends in a later one
            t.join(smem, ml, whole, a.parts + ((int64_t)blockIdx.x * 2 + (begin() == 0)) * A::PART);
            if (!whole) {
                __syncthreads();
                if (threadIdx.x == 0) {
                    // the blocks with chunks of this unit: i0 (its first chunk) to i1
                    const int64_t u0 = first_chunk(), u1 = u0 + plan.n;
                    const int64_t i0 = ((u0 + 1) * plan.blocks - 1) / plan.U, i1 = (u1 * plan.blocks - 1) / plan.U;
                    __threadfence();
                    int *counter = a.counters + ((int64_t)plan.b * HR + plan.unit);
                    const bool last = atomicAdd(counter, 1) == (int)(i1 - i0);
                    if (last) *counter = 0;
                    __threadfence();
                    last_s = last ? (int)(i1 - i0) + 1 : 0;
                    first_s = (int)i0;
                }
                __syncthreads();
                if (last_s) t.merge(first_s, last_s);
            }
        }
        // Every thread has read the plan, and left shared memory, before the next unit is
        // planned: also where the piece ends among the chunks that stand for this unit's
        // overhead, and so has none of its chunks.
        __syncthreads();
        if (threadIdx.x == 0) {
            const int64_t u1 = first_chunk() + plan.n;
            plan.x = max(plan.x, u1);
            if (++plan.unit == HR) {
                plan.unit = 0;
                plan.base = u1;
                if (plan.x < plan.end) do { plan.n = chunks_of<TILES>(a, ++plan.b); } while (plan.n == 0);
            }
        }
        __syncthreads();
    }
}

constexpr int kMaxBlocksPerSm = 4;
// Floats that a launch can need of the workspace: 16 rows are the largest row block, two parts of
// a block; two column blocks (up to D = 128) put aside as much as one of twice the head dim.
inline int64_t parts_floats(int64_t D) { return (int64_t)num_sms() * kMaxBlocksPerSm * 2 * 16 * (D + 2); }
inline int64_t aside_floats(int64_t D) {
    return (int64_t)num_sms() * kMaxBlocksPerSm * kWarps * 32 * (4 + D / 4) * (D <= 128 ? 2 : 1);
}

// Blocks of a wave: what of the kernel fits on the device.
template <int W, int NT, int LIMBS, int TILES, bool RUNS>
int wave() {
    static int cache[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (cache[dev] == 0) {
        constexpr int smem = Attn<W, NT, LIMBS, TILES, RUNS>::SMEM;
        int n = 0;
        if (cudaFuncSetAttribute(attn_kernel<W, NT, LIMBS, TILES, RUNS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
                cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attn_kernel<W, NT, LIMBS, TILES, RUNS>, kThreads, smem) !=
                cudaSuccess || n < 1)
            return 0;
        cache[dev] = num_sms() * (n < kMaxBlocksPerSm ? n : kMaxBlocksPerSm);
    }
    return cache[dev];
}

}  // namespace
}  // namespace kv4
}  // namespace fc

using namespace fc;
using namespace fc::kv4;

extern "C" size_t fc_kv4_attn_workspace_size(int64_t B, int64_t Sq, int64_t Hq, int64_t Hk, int64_t D) {
    return (size_t)(kCounterBytes + (parts_floats(D) + aside_floats(D)) * 4);
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
    const Rows to{out, o_sb, o_ss, o_sh, Hq}, from{q, q_sb, q_ss, q_sh, Hq};
    if (!same_rows(to, from, B, Sq) && rows_meet(to, from, B, Sq, D, dtype_size(dtype))) {
        set_error("kv4_attn: out overlaps q (it may be q itself)");
        return FC_EINVAL;
    }
    if (rows_repeat(to, B, Sq)) { set_error("kv4_attn: out has rows in one place"); return FC_EINVAL; }
    if (Hk * page_size * (tile_bytes((int)(D / 32)) / 16) > 0x7fffffff) {
        set_error("kv4_attn: pages over 2 GiB");
        return FC_ENOTSUP;
    }
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
    // One column block of 8 serves up to 8 (4) rows.  More rows can take two, which double
    // the matrix instructions but share the unpacking, against reading the pages again for
    // the next rows.  Two need 255 registers, 8 warps an SM instead of 12, so they pay where
    // sequences are long.  The host knows the table's width alone, so short sequences get two
    // as well where the table could hold long ones.  16 rows, us with two / one: 16 x 32768
    // tokens, 8 heads 179 / 206; 24 x 1..9000 36 / 34; 4 x 4096 30 / 22.  At D = 256 they spill (8 x 8192: 62 / 35).
    const int64_t tokens = B * Hk * (selected ? n_selected : max_pages) * page_size;
    const int nt = rows * limbs > 8 && D <= 128 && tokens >= 1 << 21 ? 2 : 1;
    const int rpc = 8 * nt / limbs;
    const int64_t row_blocks = (rows + rpc - 1) / rpc;
    if (B * Hk * row_blocks > kMaxUnits) { set_error("kv4_attn: too many rows"); return FC_ENOTSUP; }
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
    a.parts = reinterpret_cast<float *>(ws + kCounterBytes);
    a.aside = a.parts + parts_floats(D);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_head_dim(D, [&](auto w) {
        constexpr int W = decltype(w)::value;
        using std::integral_constant;
        auto launch = [&](auto n, auto lm, auto tiles, auto runs) {
            constexpr int NT = decltype(n)::value, L = decltype(lm)::value, T = decltype(tiles)::value;
            constexpr bool R = decltype(runs)::value;
            const int blocks = wave<W, NT, L, T, R>();
            if (!blocks) { set_error("kv4_attn: the kernel does not fit this device"); return FC_ECUDA; }
            attn_kernel<W, NT, L, T, R><<<blocks, kThreads, Attn<W, NT, L, T, R>::SMEM, st>>>(a);
            return check_launch("kv4_attn");
        };
        auto of_kind = [&](auto tiles, auto runs) {
            integral_constant<int, 1> one;
            integral_constant<int, 2> two;
            if constexpr (W <= 4) {
                if (nt == 2) return limbs == 1 ? launch(two, one, tiles, runs) : launch(two, two, tiles, runs);
            }
            return limbs == 1 ? launch(one, one, tiles, runs) : launch(one, two, tiles, runs);
        };
        // Chunks of 64 tokens where pages hold them whole and rings of them fit; of 32 else.
        if constexpr (W <= 4) {
            if (page_size >= 64 && !selected) return of_kind(integral_constant<int, 4>(), std::true_type());
        }
        return page_size >= 32 && !selected ? of_kind(integral_constant<int, 2>(), std::true_type())
                                            : of_kind(integral_constant<int, 2>(), std::false_type());
    });
}
