// Paged 8-bit KV cache: attention of one or a few new tokens.
//
//   out = softmax(scale * q . K^T) . V,  K, V = (code + 1/2) * (scale of 16 tokens and head)
//
// Every held byte is read once per KV head and block of 8 query rows (16 with two column
// blocks): HBM bounds it, at 2 D + 1/2 bytes a token and head.
//
// Operands.  mma.m16n8k16 in fp16, tokens (K) or channels (V) in the 16 rows, the group's
// query rows in the 8 columns.  Pages hold plain rows of codes; ldmatrix, which moves 16-bit
// elements, gives a lane two neighbouring channels of two tokens or of one, as it is asked to
// transpose or not, and the bytes of such a word that belong together are every second one:
// two byte permutations that put them under the exponent of 1024 (code + 128 in the low bits
// of an fp16 is 1024 + that) and an fp16 subtraction make two pairs of exact codes.  The order
// of the channels this leaves is met by the queries' order and by where outputs are written.
// The half that is on every code comes in as half the sum of the query, which the scores'
// accumulators begin with, and as half the sum of the weights, added to the outputs.
// Queries are scaled by a power of two per row so that fp16 holds them (bf16 exactly, down to
// 2^-39 of the row's largest); fp16 and fp32 ones are two fp16 parts (22 bits).
//
// Weights.  Base-2 softmax with a running maximum per row, and a running maximum r of the
// values' scales: weight * scale / r * 2^14, at most 2^14, is the fp16 operand (powers of two: the
// product is rounded once, to 11 bits; for fp16 and fp32 queries to two parts).  Those bits are
// kept of values down to 2^-28 of the largest, whose weight may be nothing.  The products
// of a chunk are summed by themselves and added in rounded fp32, which takes the factor of a
// new maximum along for nothing.
//
// Work.  The chunks of all (sequence, KV head, row block) are one line, cut into equal pieces
// for one wave of blocks, whatever the lengths; the lengths are read on the device.  A
// block's warps take the chunks of its piece in turn, each with its own ring of asynchronous
// copies and its own running state.  Pieces of one (sequence, head) are joined by the last
// block to finish, in order: the result does not depend on timing.  No block waits for another.
//
// 16 sequences of 32768 tokens, 32/8 heads, D = 128, bf16 (1.08 GB): 185 us in short runs, 5.8 TB/s, 90 %
// of the copy rate; 198 to 214 us (78 %) under sustained load, where the power cap lowers the clock.  8 warps an
// SM with three stages of 32 tokens each, as much as shared memory holds; 12 warps with two stages took 187 us,
// 12 with four of 16 tokens 182 (and spill with more query rows), 6 with four 220.
#include "fc_attn_common.cuh"
#include "fc_kv8.cuh"

namespace fc {
namespace kv8 {
namespace {

struct AttnArgs {
    const void *q;
    int64_t q_sb, q_ss, q_sh;
    int B, Sq, Hq, Hk, G, rows, row_blocks, dtype, q_vec;
    Pool pool;
    Table table;
    const int *lengths;
    float scale;  // softmax_scale * log2(e), > 0
    float sign;   // of softmax_scale, folded into the queries
    void *out;
    int64_t o_sb, o_ss, o_sh;
    float *lse;
    int *counters;  // one per (sequence, KV head, row block), zero between calls
    float *parts;   // two per block
};

constexpr int kWarps = 8, kThreads = 32 * kWarps;
constexpr float kNone = -3e38f;  // the maximum of a row that has seen no token
constexpr float kUp = 0x1p14f;   // what an fp16 weight is multiplied by

__device__ __forceinline__ void mma16816(float c[4], const uint32_t a[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 8x8 matrices of 16-bit elements whose rows the lanes point to.
__device__ __forceinline__ void ldmatrix4(uint32_t w[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t w[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
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

// The codes of bytes 0 and 2, and of bytes 1 and 3, as pairs.
__device__ __forceinline__ void unpack(uint32_t w, uint32_t &even, uint32_t &odd) {
    const uint32_t u = w ^ 0x80808080u;  // code + 128
    const __half2 off = __float2half2_rn(-1152.f);
    even = u32(__hadd2(h2(__byte_perm(u, 0x64646464u, 0x4240)), off));
    odd = u32(__hadd2(h2(__byte_perm(u, 0x64646464u, 0x4341)), off));
}

__device__ __forceinline__ void cp_async4(void *dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}

// PARTS: fp16 parts of a query and of a weight; NT: blocks of 8 query rows.
template <int W, int NT, int PARTS>
struct Attn {
    static constexpr int D = 32 * W;
    static constexpr int BLOCKS = W <= 4 ? 2 : 1;  // runs of 16 tokens in a chunk
    static constexpr int CH = 16 * BLOCKS;
    static constexpr int PITCH = D + 16;  // bytes of a row in shared memory: 8 rows lie in different banks
    static constexpr int STAGE = 2 * CH * PITCH + 16;  // keys, values, scales
    static constexpr int kStages = W == 6 ? 4 : 3;
    static constexpr int RING = kStages * STAGE, SMEM = kWarps * RING;
    static constexpr int RPB = 8 * NT;                   // rows of a block
    static constexpr int PART = RPB * (D + 4);           // floats of a partial result
    static_assert(SMEM >= kWarps * RPB * D * 4, "the joins use the rings' memory");

    const AttnArgs &a;
    unsigned char *ring;  // of this warp
    int warp, lane, r, c;
    // this segment
    int b, h, rb, len, chunk0, chunk1;
    uint32_t qb[NT][PARTS][2 * W][2];
    float f[NT][2], half_sum[NT][2];
    int seen[NT][2], min_seen;
    float M[NT][2], l[NT][2], ws[NT][2], acc[NT][2 * W][4], ref, inv_ref;

    __device__ __forceinline__ Attn(const AttnArgs &args, unsigned char *smem) : a(args) {
        warp = threadIdx.x >> 5;
        lane = threadIdx.x & 31;
        r = lane >> 2;
        c = lane & 3;
        ring = smem + warp * RING;
    }

    // ---------------------------------------------------------------- queries
    // Slot m, word e of lane (r, c): channels 16 m + 4 c + {0, 2} (e = 0), {1, 3} of row r.
    __device__ __forceinline__ void load_queries() {
        float total[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int row = rb * RPB + nt * 8 + r;
            const bool on = row < a.rows;
            const int s = row / a.G, g = row - s * a.G;
            const int64_t o = b * a.q_sb + s * a.q_ss + (int64_t)(h * a.G + g) * a.q_sh + 4 * c;
            float x[8 * W], top = 0.f;
#pragma unroll
            for (int m = 0; m < 2 * W; m++) {
#pragma unroll
                for (int i = 0; i < 4; i++) x[4 * m + i] = 0.f;
                if (on && a.q_vec) {
                    if (PARTS == 1) load_vec_f32<__nv_bfloat16, 4>(static_cast<const __nv_bfloat16 *>(a.q) + o + 16 * m, x + 4 * m);
                    else if (a.dtype == FC_F16) load_vec_f32<__half, 4>(static_cast<const __half *>(a.q) + o + 16 * m, x + 4 * m);
                    else load_vec_f32<float, 4>(static_cast<const float *>(a.q) + o + 16 * m, x + 4 * m);
                } else if (on) {
#pragma unroll
                    for (int i = 0; i < 4; i++) x[4 * m + i] = load_as_f32(a.q, o + 16 * m + i, a.dtype);
                }
#pragma unroll
                for (int i = 0; i < 4; i++) top = fmaxf(top, fabsf(x[4 * m + i]));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // 2^e above the largest |q|: queries times 2^(14 - e)
            int e = (int)(__float_as_uint(top) >> 23) - 126;
            e = top > 0.f ? max(e, -100) : 0;
            const int up_e = min(14 - e, 126);
            const float up = kv4::pow2f(up_e) * a.sign, down = kv4::pow2f(-up_e);
            float sum = 0.f;
#pragma unroll
            for (int m = 0; m < 2 * W; m++)
#pragma unroll
                for (int e2 = 0; e2 < 2; e2++) {
                    const float u = x[4 * m + e2] * up, v = x[4 * m + 2 + e2] * up;
                    const __half2 p = __floats2half2_rn(u, v);
                    const float2 z = __half22float2(p);
                    qb[nt][0][m][e2] = u32(p);
                    sum += z.x + z.y;
                    if constexpr (PARTS == 2) {
                        const __half2 p2 = __floats2half2_rn(u - z.x, v - z.y);
                        const float2 y = __half22float2(p2);
                        qb[nt][1][m][e2] = u32(p2);
                        sum += y.x + y.y;
                    }
                }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            total[nt] = sum;
            // what belongs to a column, from the lanes that hold it to those that score it
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const int from = (2 * c + y) * 4;
                f[nt][y] = __shfl_sync(0xffffffffu, down, from) * a.scale;
                half_sum[nt][y] = 0.5f * __shfl_sync(0xffffffffu, total[nt], from);
                const int sq = min(rb * RPB + nt * 8 + 2 * c + y, a.rows - 1) / a.G;
                seen[nt][y] = len - (a.Sq - 1 - sq);
                M[nt][y] = kNone;
                l[nt][y] = ws[nt][y] = 0.f;
            }
#pragma unroll
            for (int m = 0; m < 2 * W; m++)
#pragma unroll
                for (int i = 0; i < 4; i++) acc[nt][m][i] = 0.f;
        }
        // row blocks hold rows in order: the first one sees least
        min_seen = len - (a.Sq - 1 - min(rb * RPB, a.rows - 1) / a.G);
        ref = 0x1p-126f;
        inv_ref = 0x1p126f;
    }

    // ------------------------------------------------------------------ copies
    // Chunk i into a stage; lane (i % BLOCKS) of the ids holds the page of each of its runs.
    __device__ __forceinline__ void fetch(int i, const int page[BLOCKS], int stage) {
        unsigned char *dst = ring + stage * STAGE;
        constexpr int UNITS = D / 16;  // 16-byte words of a row
#pragma unroll
        for (int y = 0; y < BLOCKS; y++) {
            const int pos = i * CH + 16 * y;
            if (pos >= len) break;  // stale codes are finite, and their weights 0
            const int row = pos & ((1 << a.pool.log_page) - 1);
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                const int64_t head = a.pool.head(page[y], kv, h);
                const signed char *src = a.pool.codes + ((head << a.pool.log_page) + row) * D;
                unsigned char *to = dst + (kv * CH + 16 * y) * PITCH;
#pragma unroll
                for (int j = 0; j < 16 * UNITS / 32; j++) {
                    const int u = j * 32 + lane, rr = u / UNITS;
                    cp_async16(to + rr * PITCH + (u - rr * UNITS) * 16, src + u * 16);
                }
                if (lane == 0)
                    cp_async4(dst + 2 * CH * PITCH + (2 * y + kv) * 4,
                              a.pool.scales + (head << (a.pool.log_page - 4)) + (row >> 4));
            }
        }
    }

    // ------------------------------------------------------------------- a chunk
    __device__ __forceinline__ void chunk(int i, int stage) {
        const unsigned char *at = ring + stage * STAGE;
        // matrices: rows 0-7, 8-15 of one 16-byte column, then of the next
        const uint32_t rows = smem_addr(at) + (lane & 15) * PITCH + (lane >> 4) * 16;
        const float *scales = reinterpret_cast<const float *>(at + 2 * CH * PITCH);
        float s[BLOCKS][NT][4], vs[BLOCKS];
#pragma unroll
        for (int y = 0; y < BLOCKS; y++) {
            const bool any = i * CH + 16 * y < len;
            const float ks = any ? scales[2 * y] : 0.f;
            vs[y] = any ? scales[2 * y + 1] : 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[y][nt][j] = half_sum[nt][j & 1];
#pragma unroll
            for (int m = 0; m < W; m++) {
                uint32_t w[4], k0[4], k1[4];
                ldmatrix4(w, rows + 16 * y * PITCH + 32 * m);
                unpack(w[0], k0[0], k0[2]);
                unpack(w[1], k0[1], k0[3]);
                unpack(w[2], k1[0], k1[2]);
                unpack(w[3], k1[1], k1[3]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int p = 0; p < PARTS; p++) {
                        mma16816(s[y][nt], k0, qb[nt][p][2 * m][0], qb[nt][p][2 * m][1]);
                        mma16816(s[y][nt], k1, qb[nt][p][2 * m + 1][0], qb[nt][p][2 * m + 1][1]);
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[y][nt][j] *= f[nt][j & 1] * ks;
        }
        if ((i + 1) * CH > min_seen) {
#pragma unroll
            for (int y = 0; y < BLOCKS; y++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (i * CH + 16 * y + r + (j >> 1) * 8 >= seen[nt][j & 1]) s[y][nt][j] = -INFINITY;
        }
        // the largest scale of the values so far (a NaN stays with its weights)
        float top = ref;
#pragma unroll
        for (int y = 0; y < BLOCKS; y++) top = fmaxf(top, vs[y]);
        const float shrink = ref * __uint_as_float((254u << 23) - __float_as_uint(top));
        ref = top;
        inv_ref = __uint_as_float((254u << 23) - __float_as_uint(top));
        float ratio[BLOCKS];
#pragma unroll
        for (int y = 0; y < BLOCKS; y++) ratio[y] = vs[y] * inv_ref * kUp;
        float g[NT][2];
        uint32_t wb[BLOCKS][NT][PARTS][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float m = M[nt][y];
#pragma unroll
                for (int k = 0; k < BLOCKS; k++) m = fmaxf(m, fmaxf(s[k][nt][y], s[k][nt][y + 2]));
#pragma unroll
                for (int o = 4; o < 32; o *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                const float k = exp2_fast(M[nt][y] - m);
                M[nt][y] = m;
                l[nt][y] *= k;
                g[nt][y] = k * shrink;
                ws[nt][y] *= g[nt][y];
            }
#pragma unroll
            for (int y = 0; y < BLOCKS; y++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float w[2];
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const float z = s[y][nt][2 * j + x], p = exp2_fast(z - M[nt][x]);
                        l[nt][x] += p;
                        // A token that is not seen has no weight, whatever the scale: it may be behind the last
                        // one.  (Not every weight of zero: values that are no numbers stay so where a weight is
                        // below fp32, as it may be beside one block's largest score and not beside another's.)
                        w[x] = z == -INFINITY ? 0.f : p * ratio[y];
                        ws[nt][x] += w[x];
                    }
                    const __half2 hi = __floats2half2_rn(w[0], w[1]);
                    wb[y][nt][0][j] = transpose8(u32(hi));
                    if constexpr (PARTS == 2) {
                        const float2 z = __half22float2(hi);
                        wb[y][nt][1][j] = transpose8(u32(__floats2half2_rn(w[0] - z.x, w[1] - z.y)));
                    }
                }
        }
        // outputs: channels 16 m + 2 r (+ 1 in rows r + 8)
#pragma unroll
        for (int m = 0; m < 2 * W; m += 2) {
            float t[NT][2][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 4; j++) t[nt][0][j] = t[nt][1][j] = 0.f;
#pragma unroll
            for (int y = 0; y < BLOCKS; y++) {
                uint32_t w[4], v0[4], v1[4];
                ldmatrix4_trans(w, rows + (CH + 16 * y) * PITCH + 16 * m);
                unpack(w[0], v0[0], v0[1]);
                unpack(w[1], v0[2], v0[3]);
                unpack(w[2], v1[0], v1[1]);
                unpack(w[3], v1[2], v1[3]);
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int p = 0; p < PARTS; p++) {
                        mma16816(t[nt][0], v0, wb[y][nt][p][0], wb[y][nt][p][1]);
                        mma16816(t[nt][1], v1, wb[y][nt][p][0], wb[y][nt][p][1]);
                    }
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[nt][m + e][j] = fmaf(acc[nt][m + e][j], g[nt][j & 1], t[nt][e][j]);
        }
    }

    // This warp's chunks of the segment: chunk0 + warp, + kWarps, ..., each copied
    // kStages - 1 rounds before it is used.
    __device__ __forceinline__ void run() {
        // lane l holds the page of run l % BLOCKS of the chunk l / BLOCKS rounds into a window;
        // the window after it is on its way
        constexpr int WINDOW = 32 / BLOCKS;
        auto window = [&](int first) {
            const int chunk = first + kWarps * (lane / BLOCKS), pos = chunk * CH + 16 * (lane % BLOCKS);
            return chunk < chunk1 && pos < len ? a.table.page(b, pos >> a.table.log_page) : 0;
        };
        int next = chunk0 + warp, round = 0;
        int ids = window(next), ids2 = window(next + WINDOW * kWarps);
        auto copy = [&](int stage) {
            if (next < chunk1) {
                int page[BLOCKS];
#pragma unroll
                for (int y = 0; y < BLOCKS; y++) page[y] = __shfl_sync(0xffffffffu, ids, round * BLOCKS + y);
                fetch(next, page, stage);
            }
            cp_async_commit();
            next += kWarps;
            if (++round == WINDOW) {
                round = 0;
                ids = ids2;
                ids2 = window(next + WINDOW * kWarps);
            }
        };
#pragma unroll
        for (int i = 0; i < kStages - 1; i++) copy(i);
        load_queries();  // while the first chunks are on their way
        int stage = 0;
        for (int i = chunk0 + warp; i < chunk1; i += kWarps) {
            cp_async_wait<kStages - 2>();
            __syncwarp();
            copy(stage == 0 ? kStages - 1 : stage - 1);
            chunk(i, stage);
            __syncwarp();
            stage = stage == kStages - 1 ? 0 : stage + 1;
        }
        cp_async_wait<0>();
    }

    // -------------------------------------------------------------------- joins
    __device__ __forceinline__ void write_row(int row, int d, float v) const {
        const int s = row / a.G, g = row - s * a.G;
        store_from_f32(a.out, b * a.o_sb + s * a.o_ss + (int64_t)(h * a.G + g) * a.o_sh + d, a.dtype, v);
    }
    __device__ __forceinline__ void write_lse(int row, float m, float sum) const {
        const int s = row / a.G, g = row - s * a.G;
        a.lse[((int64_t)b * a.Sq + s) * a.Hq + h * a.G + g] =
            sum > 0.f ? (m + log2f(sum)) * 0.693147180559945309f : sum == 0.f ? -INFINITY : sum;
    }
    // v / s in units of u
    __device__ __forceinline__ static float result(float v, float s, float u) {
        return s == 0.f ? 0.f : v / s * (u / kUp);
    }

    // Joins the warps; whole: the outputs are final, else they go to `part`: [row][D], then
    // maximum, sum and unit of each row.
    __device__ __forceinline__ void join(unsigned char *smem, float *mlr, bool whole, float *part) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                float s = l[nt][y], w = ws[nt][y];
#pragma unroll
                for (int o = 4; o < 32; o *= 2) {
                    s += __shfl_xor_sync(0xffffffffu, s, o);
                    w += __shfl_xor_sync(0xffffffffu, w, o);
                }
                ws[nt][y] = 0.5f * w;
                if (r == 0) {
                    float *z = mlr + (warp * RPB + nt * 8 + 2 * c + y) * 3;
                    z[0] = M[nt][y];
                    z[1] = s;
                    z[2] = ref;
                }
            }
        __syncthreads();  // also: every warp has left its ring
        float *o = reinterpret_cast<float *>(smem);  // [warp][row][D]
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const int row = nt * 8 + 2 * c + y;
#pragma unroll
                for (int m = 0; m < 2 * W; m++)
                    *reinterpret_cast<float2 *>(o + (warp * RPB + row) * D + 16 * m + 2 * r) =
                        make_float2(acc[nt][m][y] + ws[nt][y], acc[nt][m][y + 2] + ws[nt][y]);
            }
        __syncthreads();
        const int rows = min(RPB, a.rows - rb * RPB);
        for (int i = threadIdx.x; i < rows * D; i += kThreads) {
            const int row = i / D;
            float m = mlr[row * 3], u = mlr[row * 3 + 2], s = 0.f, v = 0.f;
#pragma unroll
            for (int w = 1; w < kWarps; w++) {
                m = fmaxf(m, mlr[(w * RPB + row) * 3]);
                u = fmaxf(u, mlr[(w * RPB + row) * 3 + 2]);
            }
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                const float *z = mlr + (w * RPB + row) * 3;
                const float k = exp2_fast(z[0] - m);
                s = fmaf(z[1], k, s);
                v = fmaf(o[w * RPB * D + i], k * (z[2] / u), v);
            }
            if (whole) {
                write_row(rb * RPB + row, i % D, result(v, s, u));
                if (a.lse && i % D == 0) write_lse(rb * RPB + row, m, s);
            } else {
                part[i] = v;
                if (i % D == 0) *reinterpret_cast<float4 *>(part + RPB * D + 4 * row) = make_float4(m, s, u, 0.f);
            }
        }
    }

    // Joins `count` parts of this unit: block `first`'s second one, then the first ones of
    // the blocks after it.
    __device__ __forceinline__ void merge(int first, int count) const {
        const float *p0 = a.parts + ((int64_t)first * 2 + 1) * PART;
        const float *p1 = a.parts + (int64_t)first * 2 * PART;  // block first + k: + 2 k PART
        const int rows = min(RPB, a.rows - rb * RPB);
        for (int i = threadIdx.x * 4; i < rows * D; i += kThreads * 4) {
            const int row = i / D, at = RPB * D + 4 * row;
            float m = kNone, u = 0.f;
#pragma unroll 4
            for (int k = 0; k < count; k++) {
                const float4 z = __ldcg(reinterpret_cast<const float4 *>((k ? p1 + (int64_t)2 * k * PART : p0) + at));
                m = fmaxf(m, z.x);
                u = fmaxf(u, z.z);
            }
            float s = 0.f, v[4] = {};
#pragma unroll 4
            for (int k = 0; k < count; k++) {
                const float *p = k ? p1 + (int64_t)2 * k * PART : p0;
                const float4 z = __ldcg(reinterpret_cast<const float4 *>(p + at));
                const float4 o = __ldcg(reinterpret_cast<const float4 *>(p + i));
                const float e = exp2_fast(z.x - m), k2 = e * (z.z / u);
                s = fmaf(e, z.y, s);
                v[0] = fmaf(k2, o.x, v[0]);
                v[1] = fmaf(k2, o.y, v[1]);
                v[2] = fmaf(k2, o.z, v[2]);
                v[3] = fmaf(k2, o.w, v[3]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) write_row(rb * RPB + row, i % D + j, result(v[j], s, u));
            if (a.lse && i % D == 0) write_lse(rb * RPB + row, m, s);
        }
    }
};

// What a segment costs beyond its chunks (queries, the pipeline's start, the joins), in chunks
// of its block's warps; a block's least piece is a chunk for every warp more.
constexpr int kOverhead = 32, kMinPiece = kOverhead + kWarps;
// A sequence, in the sums of the line's lengths (at most 2^18 of up to 2^26).
constexpr int64_t kOne = int64_t(1) << 44;

// Chunks of sequence b, 0 where it holds nothing.
template <int CH>
__device__ __forceinline__ int chunks_of(const AttnArgs &a, int64_t b) {
    const int len = a.table.length(a.lengths[b]);
    return len <= 0 ? 0 : (len + CH - 1) / CH;
}

// Where a block is on the line.
struct Plan {
    int64_t U, blocks, x, end, base;  // base: where the line of sequence b begins
    int b, n, unit;                   // n: chunks of a unit of b
};

// The line: unit (sequence, KV head, row block) u of n > 0 chunks is n + kOverhead long, the
// first kOverhead standing for what a segment costs beyond its chunks.  Block i of `blocks`
// has the piece [U i / blocks, U (i + 1) / blocks).
template <int W, int NT, int PARTS>
__global__ void __launch_bounds__(kThreads, 1) attn_kernel(const __grid_constant__ AttnArgs a) {
    using A = Attn<W, NT, PARTS>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int64_t sums[kWarps];
    __shared__ Plan plan;
    __shared__ int first_s, last_s, most[kWarps];
    __shared__ float mlr[kWarps * A::RPB * 3];

    const int HR = a.Hk * a.row_blocks;
    const int per = (a.B + kThreads - 1) / kThreads;
    const int b0 = min((int)threadIdx.x * per, a.B), b1 = min(b0 + per, a.B);
    int64_t mine = 0;
    int longest = 0;
    for (int b = b0; b < b1; b++) {
        const int n = chunks_of<A::CH>(a, b);
        longest = max(longest, n + kOverhead);
        mine += n ? n + kOverhead + kOne : 0;
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
        if (chunks_of<A::CH>(a, b)) continue;
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
    int64_t blocks = min((int64_t)gridDim.x, (U + kMinPiece - 1) / kMinPiece);
    // Equal units that are short: one block for each, no piece crossing from one to the next.
    if (units && units <= gridDim.x && longest < 2 * kMinPiece && U == units * longest) blocks = units;
    if ((int64_t)blockIdx.x >= blocks) return;
    const int64_t x0 = U * blockIdx.x / blocks;
    // the sequence that the piece begins in
    if (x0 >= before * HR && x0 < (before + mine) * HR) {
        int64_t at = before * HR;
        int b = b0, n;
        for (;; b++) {
            n = chunks_of<A::CH>(a, b);
            const int64_t w = n ? (int64_t)(n + kOverhead) * HR : 0;
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
        plan.unit = (int)((x0 - at) / (n + kOverhead));
    }
    __syncthreads();

    A t(a, smem);
    while (plan.x < plan.end) {
        auto first_chunk = [&] { return plan.base + (int64_t)plan.unit * (plan.n + kOverhead) + kOverhead; };
        auto begin = [&] { return (int)max(plan.x - first_chunk(), (int64_t)0); };
        auto end = [&] { return (int)min(plan.end - first_chunk(), (int64_t)plan.n); };
        if (begin() < end()) {
            t.b = plan.b;
            t.h = plan.unit / a.row_blocks;
            t.rb = plan.unit - t.h * a.row_blocks;
            t.len = a.table.length(a.lengths[t.b]);
            t.chunk0 = begin();
            t.chunk1 = end();
            t.run();
            const bool whole = begin() == 0 && end() == plan.n;
            // parts of a block: 0 of a unit that began in an earlier one, 1 of one that ends in a later one
            t.join(smem, mlr, whole, a.parts + ((int64_t)blockIdx.x * 2 + (begin() == 0)) * A::PART);
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
        // every thread has read the plan, and left shared memory, before the next unit is planned
        __syncthreads();
        if (threadIdx.x == 0) {
            const int64_t u1 = first_chunk() + plan.n;
            plan.x = max(plan.x, u1);
            if (++plan.unit == HR) {
                plan.unit = 0;
                plan.base = u1;
                if (plan.x < plan.end) do { plan.n = chunks_of<A::CH>(a, ++plan.b); } while (plan.n == 0);
            }
        }
        __syncthreads();
    }
}

constexpr int kMaxBlocksPerSm = 4;
// Floats that a launch can need of the workspace: 16 rows are the largest row block, two parts of a block.
inline int64_t parts_floats(int64_t D) { return (int64_t)num_sms() * kMaxBlocksPerSm * 2 * 16 * (D + 4); }

// Blocks of a wave: what of the kernel fits on the device.
template <int W, int NT, int PARTS>
int wave() {
    static int cache[64] = {0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (cache[dev] == 0) {
        constexpr int smem = Attn<W, NT, PARTS>::SMEM;
        int n = 0;
        if (cudaFuncSetAttribute(attn_kernel<W, NT, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, attn_kernel<W, NT, PARTS>, kThreads, smem) != cudaSuccess || n < 1)
            return 0;
        cache[dev] = num_sms() * (n < kMaxBlocksPerSm ? n : kMaxBlocksPerSm);
    }
    return cache[dev];
}

}  // namespace
}  // namespace kv8
}  // namespace fc

using namespace fc;
using namespace fc::kv8;

extern "C" size_t fc_kv8_attn_workspace_size(int64_t B, int64_t Sq, int64_t Hq, int64_t Hk, int64_t D) {
    return (size_t)(kv4::kCounterBytes + parts_floats(D) * 4);
}

extern "C" int fc_kv8_attn(const void *q, int dtype, int64_t B, int64_t Sq, int64_t Hq, int64_t q_sb, int64_t q_ss,
                           int64_t q_sh, const signed char *codes, const float *scales, int64_t num_pages, int64_t Hk,
                           int64_t D, int64_t page_size, const int *page_table, int64_t table_stride,
                           int64_t max_pages, const int *lengths, float softmax_scale, void *out, int64_t o_sb,
                           int64_t o_ss, int64_t o_sh, float *lse, void *workspace, size_t workspace_bytes,
                           int *status, void *stream) {
    clear_error();
    int rc = check_pool("kv8_attn", B, Hk, D, page_size, num_pages, max_pages, codes, scales, page_table, status);
    if (rc) return rc;
    if (!is_float_dtype(dtype)) { set_error("kv8_attn: dtype must be fp32, bf16 or fp16"); return FC_EINVAL; }
    if (Hq <= 0 || Hq % Hk) {
        set_error("kv8_attn: query heads (%lld) must be a multiple of kv heads (%lld)", (long long)Hq, (long long)Hk);
        return FC_EINVAL;
    }
    if (Sq < 0 || Sq > 65535 || Hq > 65535) { set_error("kv8_attn: bad query count"); return FC_EINVAL; }
    if (!(softmax_scale == softmax_scale) || softmax_scale - softmax_scale != 0.f) {
        set_error("kv8_attn: the softmax scale must be finite");
        return FC_EINVAL;
    }
    if (B == 0 || Sq == 0) return FC_OK;
    if (!q || !out || !lengths) { set_error("kv8_attn: null pointer"); return FC_EINVAL; }
    const Rows to{out, o_sb, o_ss, o_sh, Hq}, from{q, q_sb, q_ss, q_sh, Hq};
    if (!same_rows(to, from, B, Sq) && rows_meet(to, from, B, Sq, D, dtype_size(dtype))) {
        set_error("kv8_attn: out overlaps q (it may be q itself)");
        return FC_EINVAL;
    }
    if (rows_repeat(to, B, Sq)) { set_error("kv8_attn: out has rows in one place"); return FC_EINVAL; }
    if (!workspace || !aligned(workspace, 16)) { set_error("kv8_attn: null or misaligned workspace"); return FC_EINVAL; }
    if (workspace_bytes < fc_kv8_attn_workspace_size(B, Sq, Hq, Hk, D)) {
        set_error("kv8_attn: workspace of %zu bytes is too small", workspace_bytes);
        return FC_ERANGE;
    }
    const int64_t rows = Sq * (Hq / Hk);
    // A column block of 8 serves up to 8 rows; two share the unpacking and the read (up to D = 128: beyond it
    // their registers spill).
    const int nt = rows > 8 && D <= 128 ? 2 : 1, rpb = 8 * nt;
    const int64_t row_blocks = (rows + rpb - 1) / rpb;
    if (B * Hk * row_blocks > kv4::kMaxUnits) { set_error("kv8_attn: too many rows"); return FC_ENOTSUP; }
    char *ws = static_cast<char *>(workspace);
    AttnArgs a{};
    a.q = q; a.q_sb = q_sb; a.q_ss = q_ss; a.q_sh = q_sh;
    a.B = (int)B; a.Sq = (int)Sq; a.Hq = (int)Hq; a.Hk = (int)Hk; a.G = (int)(Hq / Hk);
    a.rows = (int)rows; a.row_blocks = (int)row_blocks; a.dtype = dtype;
    a.q_vec = rows_aligned(q, dtype, q_sb, q_ss, q_sh);
    a.pool = Pool{const_cast<signed char *>(codes), const_cast<float *>(scales), (int)Hk, ilog2(page_size)};
    a.table = Table{page_table, table_stride, (int)max_pages, (int)num_pages, ilog2(page_size), status};
    a.lengths = lengths;
    const float s = softmax_scale * 1.44269504088896341f;
    a.scale = s < 0.f ? -s : s;
    a.sign = s < 0.f ? -1.f : 1.f;
    a.out = out; a.o_sb = o_sb; a.o_ss = o_ss; a.o_sh = o_sh; a.lse = lse;
    a.counters = reinterpret_cast<int *>(ws + 256);
    a.parts = reinterpret_cast<float *>(ws + kv4::kCounterBytes);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_head_dim(D, [&](auto w) {
        constexpr int W = decltype(w)::value;
        auto launch = [&](auto n, auto p) {
            constexpr int NT = decltype(n)::value, PARTS = decltype(p)::value;
            const int blocks = wave<W, NT, PARTS>();
            if (!blocks) { set_error("kv8_attn: the kernel does not fit this device"); return FC_ECUDA; }
            attn_kernel<W, NT, PARTS><<<blocks, kThreads, Attn<W, NT, PARTS>::SMEM, st>>>(a);
            return check_launch("kv8_attn");
        };
        std::integral_constant<int, 1> one;
        std::integral_constant<int, 2> two;
        if constexpr (W <= 4) {
            if (nt == 2) return dtype == FC_BF16 ? launch(two, one) : launch(two, two);
        }
        return dtype == FC_BF16 ? launch(one, one) : launch(one, two);
    });
}
