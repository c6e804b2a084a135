// Attention over whole prompts: packed sequences of different lengths, grouped heads, causal.
//
//   out = softmax(scale * q . K^T + mask) . V
//
// Query i of a sequence of n_q queries and n_k keys is at position n_k - n_q + i and sees the
// keys up to it (all of them where not causal).
//
// 4 D operations a visible pair and head, on tcgen05; what competes with the matrix unit is
// the softmax: at D = 128 a 128 x 128 tile takes it 512 cycles, and 16384 exponentials take the
// 16 lanes of the special function units 1024.
//
// Tiles.  The heads of a group share their keys, so a tile's 128 rows are TQ = 128 / G tokens
// times the G heads (row = token * G + head; one TMA box of a 4- or 5-dimensional map): fewer
// partly filled tiles in short prompts, and less of the diagonal computed in vain.  A block
// holds one or two query tiles ("streams") and walks the keys in tiles of 128:
//
//   warp   TMA: queries, then K and V tiles through a ring
//   warp   MMA: S = Q K^T into TMEM; O += P V with P read from TMEM, where it replaces S
//   group of 4 warps a stream: a thread a row; S to registers, running maximum, exp2, P back
//          in 16 bits; O scaled by it only when the maximum grows by more than 2^8
//   2 warps: the next item of work, and the V tiles of the diagonal (below)
//
// With two streams (D <= 128) one's softmax runs while the other's products do; with wider
// heads O leaves room for one, whose scores are in two buffers instead.
//
// What is masked.  Scores are replaced, not added to, so a NaN there is gone.  A value that no
// weight but zero meets could still turn a sum into a NaN, so the tiles that hold masked keys
// (one or two of an item) are looked through in shared memory: what is no number becomes zero
// there, and is added in plain arithmetic to the rows that do see it (an infinity whose weight is nothing then
// makes an infinity, where one in a tile without a mask makes a NaN).
//
// Work.  Items (sequence, KV head, TQ or 2 TQ tokens) are dealt out to one block an SM, the
// longest first, back and forth; every block finds its own from the lengths, which are on the
// device, by counting the items of more than a number of tiles.  Fewer items than blocks are cut along
// their keys, and the last warp to finish a row's pieces joins them, in order.  No block waits for
// another.
//
// 16384 tokens, 32/8 heads, D = 128, bf16, causal (2.2 TFLOP): 1.77 ms in short runs, 1.25 PFLOP/s, 75 % of
// the burst rate of a library product; 2.0 ms (1.1 PFLOP/s, 80 % of its sustained rate) under sustained
// load, where the power cap holds the clock near 1.5 GHz.  A pair of tiles takes 2970 cycles where the products
// alone would take 2050: a stream's softmax (1790: 200 to read the scores, 230 for the maximum, 600 for each
// half's weights, 150 to store them) and its next two products follow one another, and two streams are all
// that TMEM holds.  517 tokens 16 us, 8191 packed in 7 prompts 168 us, 512 tokens over up to 30000 keys
// (14/2 heads, D = 64, fp16) 98 us.  Heads of 64: 0.67 PFLOP/s, half a tile's products for the same softmax.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "fc_attn_common.cuh"
#include "fc_kv4.cuh"

namespace fc {
namespace prompt {
namespace {

using kv4::Rows;
using kv4::rows_aligned;
using kv4::rows_meet;
using kv4::rows_repeat;
using kv4::same_rows;

// Whether n x Sx rows x and n x Sy rows y can share a byte.
inline bool meets(const Rows &x, int64_t Sx, const Rows &y, int64_t Sy, int64_t n, int64_t D, int64_t size) {
    auto span = [&](const Rows &r, int64_t S, int64_t &lo, int64_t &hi) {
        lo = hi = 0;
        for (int64_t e : {(n - 1) * r.sb, (S - 1) * r.ss, (r.H - 1) * r.sh}) (e < 0 ? lo : hi) += e * size;
        lo += (int64_t)reinterpret_cast<uintptr_t>(r.p);
        hi += (int64_t)reinterpret_cast<uintptr_t>(r.p) + D * size;
    };
    int64_t x0, x1, y0, y1;
    span(x, Sx, x0, x1);
    span(y, Sy, y0, y1);
    return x0 < y1 && y0 < x1 && rows_meet(x, y, n, Sx > Sy ? Sx : Sy, D, size);
}

struct Args {
    const void *v;
    void *out;
    float *lse;
    int64_t v_sb, v_ss, v_sh, o_sb, o_ss, o_sh;
    int Sq, Sk, Tq, Tk;
    int B, D, Hq, Hk, G, TQ, causal, o_vec;
    const int *cu_q, *cu_k;
    float scale;  // |softmax_scale| * log2(e), > 0
    int negative;
    int *status;
    int epoch;
    int split;        // items may be cut along their keys,
    int items;        // if there are no more (item, head) than this: what the workspace is made for
    int *counters;    // by (item, head), stream and warp: pieces done, zero between calls
    int *slots;       // by (item, head) and piece: where its results are
    float *parts;     // results of pieces, kPart floats each
};

constexpr int kTile = 128;          // rows of a query tile, keys of a tile
constexpr int kBox = kTile * 128;   // bytes of 128 rows of 64 channels
constexpr int kItems = 3;           // items known ahead
constexpr uint64_t kItemNs = 100 * kWaitNs;  // bound on waits for an item
constexpr int kMaxPieces = 256;     // of an item: no more than blocks
constexpr int kNoRow = 0x7fffffff;   // keys that a row of no query sees
// fp16 weights are held 2^7 times larger (at most 2^15, the largest being above 2^6): each is off by 2^-11 of
// itself or by 2^-25, 2^-31 of the row's sum, so that a tail of 2^20 keys costs no more than another 2^-11.
// (Unscaled, 32768 keys of 2^-25 the largest's weight were nothing, in a sum that counted them as 2^-10.)
template <bool F16> constexpr float kUp = F16 ? 7.f : 0.f;
// Every kPolyStep-th pair of weights of a tile without a mask is a polynomial.  8192 tokens, 32/8 heads, D = 128,
// bf16: 440 us, 452 with none; fp16 462 and 467; 16/8 heads, D = 64, fp16 202 and 205, bf16 no difference.
constexpr int kPolyStep = 4;

template <int DP> struct Cfg {
    static constexpr int NQ = DP <= 128 ? 2 : 1;         // streams
    static constexpr int LA = NQ == 2 ? 1 : 2;           // score tiles ahead of the softmax
    static constexpr int UC = DP == 256 ? 128 : DP;      // channels of a ring stage
    static constexpr int NU = DP / UC;                   // stages of a tile
    static constexpr int STAGE = kTile * UC * 2;
    static constexpr int NST = DP == 64 ? 8 : DP == 192 ? 3 : 5;
    static constexpr int QB = kTile * DP * 2;            // bytes of a query tile
    
    static constexpr int THREADS = 128 * NQ + 128;
    static constexpr int O_COL = 256;                    // TMEM: scores at 0 and 128, outputs from here
    // Heads of 64 leave room for weights beside the scores: the next scores are made while these are turned
    // into weights.  Else weights replace scores.
    static constexpr bool BESIDE = DP == 64;
    static constexpr int P_COL = BESIDE ? O_COL + NQ * DP : 0, P_STEP = BESIDE ? 64 : kTile;
    static_assert(O_COL + NQ * DP + (BESIDE ? NQ * 64 : 0) <= 512, "TMEM");
};

// ------------------------------------------------------------------------ PTX
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, int v,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(smem_addr(bar))
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Shared-memory matrix descriptor, 128-byte swizzle; 1024 bytes between groups of 8 rows, and,
// where the operand is wider than 64 elements along its contiguous dim, 16 KB from box to box.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)(kBox >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// M = 128, N = n, fp32 sums; bf16 (or fp16) operands, B K-major or MN-major.
__host__ __device__ constexpr uint32_t idesc(int n, bool f16, int b_mn) {  // (bit 13: -A)
    return (1u << 4) | (f16 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
           ((128u >> 4) << 24);
}
// Issued by the one lane whose `lead` is not 0, in code that the whole warp runs: operands stay in
// uniform registers (from a branch of one lane every one of them had to be moved there first, and
// issuing took as long as the products: 3100 cycles for the 32 of two tiles).
__device__ __forceinline__ uint32_t elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p;
}
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(acc), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(acc), "r"(lead)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t lead, uint64_t *bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)), "r"(lead)
        : "memory");
}

#define FC_R16(v, o) "=f"(v[o]), "=f"(v[o + 1]), "=f"(v[o + 2]), "=f"(v[o + 3]), "=f"(v[o + 4]), "=f"(v[o + 5]), \
    "=f"(v[o + 6]), "=f"(v[o + 7]), "=f"(v[o + 8]), "=f"(v[o + 9]), "=f"(v[o + 10]), "=f"(v[o + 11]),           \
    "=f"(v[o + 12]), "=f"(v[o + 13]), "=f"(v[o + 14]), "=f"(v[o + 15])
#define FC_W16(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]),      \
    "r"(v[o + 6]), "r"(v[o + 7]), "r"(v[o + 8]), "r"(v[o + 9]), "r"(v[o + 10]), "r"(v[o + 11]),                 \
    "r"(v[o + 12]), "r"(v[o + 13]), "r"(v[o + 14]), "r"(v[o + 15])
// 32 columns of the warp's 32 TMEM lanes, one lane a thread.
__device__ __forceinline__ void tmem_ld32(uint32_t at, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : FC_R16(v, 0), FC_R16(v, 16) : "r"(at));
}
__device__ __forceinline__ void tmem_ld16(uint32_t at, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : FC_R16(v, 0) : "r"(at));
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::FC_W16(v, 0), FC_W16(v, 16), "r"(at)
        : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::FC_W16(v, 0),
        "r"(at)
        : "memory");
}
// Waits for this thread's loads from TMEM.  N registers that they write are named, so that no use of
// them moves in front of it: to the compiler a load is done where it stands.
#define FC_U16(v, o) "+f"(v[o]), "+f"(v[o + 1]), "+f"(v[o + 2]), "+f"(v[o + 3]), "+f"(v[o + 4]), "+f"(v[o + 5]),   \
    "+f"(v[o + 6]), "+f"(v[o + 7]), "+f"(v[o + 8]), "+f"(v[o + 9]), "+f"(v[o + 10]), "+f"(v[o + 11]),           \
    "+f"(v[o + 12]), "+f"(v[o + 13]), "+f"(v[o + 14]), "+f"(v[o + 15])
template <int N>
__device__ __forceinline__ void tmem_landed(float *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i += 16) asm volatile("" : FC_U16(v, i));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^x without the special function units, whose 16 lanes would otherwise take as long as both
// products of a tile: 2^round(x) put into the exponent, 2^f on [-1/2, 1/2] as a polynomial
// (least largest relative error, by reweighted least squares: 2^-13.7 of degree 3 for bf16
// weights, 2^-18.5 of degree 4 for fp16 ones).  From -127 down the result is 0.  The power of two is a factor, not
// an addition to the exponent's bits, which would turn a NaN into a number.  x is at most 15 or no number.
template <bool F16>
__device__ __forceinline__ float2 exp2_poly(float2 x) {
    auto low = [](float v) {
        float y;
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(v), "f"(-127.f));
        return y;
    };
    x = make_float2(low(x.x), low(x.y));
    const float2 magic = make_float2(12582912.f, 12582912.f), minus = make_float2(-12582912.f, -12582912.f);
    const float2 t = __fadd2_rn(x, magic), n = __fadd2_rn(t, minus);
    const float2 f = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
    auto c2 = [](float v) { return make_float2(v, v); };
    float2 p;
    if constexpr (F16) {
        p = __ffma2_rn(f, c2(0.009570101276040077f), c2(0.05591785907745361f));
        p = __ffma2_rn(f, p, c2(0.240247443318367f));
        p = __ffma2_rn(f, p, c2(0.6931217908859253f));
        p = __ffma2_rn(f, p, c2(0.9999992847442627f));
    } else {
        p = __ffma2_rn(f, c2(0.0551716685295105f), c2(0.2426111251115799f));
        p = __ffma2_rn(f, p, c2(0.6932609677314758f));
        p = __ffma2_rn(f, p, c2(0.9999280571937561f));
    }
    // (t = 1.5 * 2^23 + n: its low bits are n, in two's complement; at n = -127 the factor is 0)
    auto power = [](float v) { return __int_as_float((__float_as_int(v) << 23) + 0x3f800000); };
    return __fmul2_rn(p, make_float2(power(t.x), power(t.y)));
}

template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (F16) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// ------------------------------------------------------------------------ work
struct Sequence {
    int q0, nq, k0, nk;  // rows, cut to those that there are
};

__device__ __forceinline__ Sequence sequence(const Args &a, int b) {
    Sequence s;
    if (!a.cu_q) return Sequence{0, a.Sq, 0, a.Sk};
    s.q0 = min(max(a.cu_q[b], 0), a.Tq);
    s.nq = max(min(a.cu_q[b + 1], a.Tq) - s.q0, 0);
    s.k0 = min(max(a.cu_k[b], 0), a.Tk);
    s.nk = max(min(a.cu_k[b + 1], a.Tk) - s.k0, 0);
    return s;
}

struct Item {
    int b, h, t;         // sequence, KV head, first token
    Sequence s;
    int nt[2];           // key tiles of the streams
    int tiles, first;    // key tiles; the first that holds masked keys
    int valid;           // 0: no more work
    // an item cut along its keys: the first key, which piece, of how many; its number among the pieces of
    // all items, and that of the (item, head)
    int base, piece, pieces, unit, line;
    // a masked value was no number: set by the helpers, which may be as far ahead of the softmax as items are
    // known, so it has its place with the item
    int bad;
};

// Keys that token i sees.
__device__ __forceinline__ int visible(const Args &a, const Sequence &s, int i) {
    return a.causal ? max(min(s.nk - s.nq + i + 1, s.nk), 0) : s.nk;
}

__device__ __forceinline__ int tiles_of(int keys) { return (int)(((unsigned)keys + kTile - 1) / kTile); }

// A piece of an item is no shorter than this many tiles (16/8 heads, D = 128: 1000 tokens, of at most 8 tiles,
// 31 us with 6, 24 us with 8; 64 tokens over 4096 49 and 45, 48 with 16).
constexpr int kLeastPiece = 8;

// The line of work, as a warp finds its way on it.  Items (sequence, TP tokens) come by their number of
// tiles, the ones of most first, items of none last.  Where there are fewer than blocks they are cut
// along their keys, into P = NT * blocks / (all tiles) pieces each, at least 1, and all items' first pieces
// come first, then the second ones of those that have two, and so on.  More sequences than a warp has lanes
// are not sorted: counting them took longer than the items of 1000 short ones.  Their items are numbered by
// where the tokens lie, some numbers being left out.
struct Line {
    const Args &a;
    int TP, most;
    unsigned inv;     // 2^32 / TP, rounded up (not of 1)
    Sequence mine;    // of this lane, where there are no more sequences than lanes
    int all;          // its items
    // Items are cut along their keys.  (cu_seqlens that fall again are sequences that overlap, and more items
    // than the rows that there are could be: the workspace has no room for their pieces.)
    bool split;
    int64_t tiles;    // of all items and heads, where they are cut

    __device__ __forceinline__ Line(const Args &args, int tp) : a(args), TP(tp), most(0), inv(0xffffffffu / (unsigned)tp + 1), mine{}, all(0), split(false), tiles(1) {
        const int lane = threadIdx.x & 31;
        if (a.B > 32) return;
        if (lane < a.B) mine = sequence(a, lane);
        all = over((unsigned)mine.nq + TP - 1);
        most = __reduce_max_sync(0xffffffffu, tiles_of(mine.nk));
        split = a.split && (int64_t)__reduce_add_sync(0xffffffffu, all) * a.Hk <= a.items;
        if (split) {
            int64_t n = 0;
            for (int t = TP; t - TP < mine.nq; t += TP) n += tiles_of(visible(a, mine, min(t, mine.nq) - 1));
#pragma unroll
            for (int o = 16; o; o /= 2) n += __shfl_xor_sync(0xffffffffu, n, o);
            tiles = max(n * a.Hk, (int64_t)1);
        }
    }

    // n / TP: the product is right up to 2^24 at least, since TP * inv passes 2^32 by less than 2^8.
    __device__ __forceinline__ int over(unsigned n) const {
        return (int)(TP == 1 ? n : n < 1u << 24 ? __umulhi(n, inv) : n / (unsigned)TP);
    }

    // Items of this lane's sequence with at least w key tiles: those from a token on.
    __device__ __forceinline__ int items_from(int w) const {
        if (w == 0) return all;
        if (tiles_of(mine.nk) < w) return 0;
        if (!a.causal) return all;
        // item t's last token sees min(nk, nk - nq + (t + 1) TP) keys: more than (w - 1) kTile
        const int need = (w - 1) * kTile - mine.nk + mine.nq;  // (t + 1) TP > need, which is below nq
        return all - (need < 0 ? 0 : over((unsigned)need));
    }
    __device__ __forceinline__ int count(int w) const { return __reduce_add_sync(0xffffffffu, items_from(w)); }
    // Tiles from which on an item has a piece p > 0.
    __device__ __forceinline__ int of_piece(int p) const {
        const int64_t n = ((p + 1) * tiles + gridDim.x - 1) / gridDim.x;
        return (int)max(min(n, (int64_t)0x7fffffff), (int64_t)(kLeastPiece * p + 1));
    }

    // Number `rank` of the line: sequence, head, first token (behind the last one: nothing to do), and piece.
    __device__ __forceinline__ bool find(int rank, Item &x) const {
        const int lane = threadIdx.x & 31;
        x.unit = rank;
        if (a.B > 32) {
            const int item = rank / a.Hk;
            x.h = rank - item * a.Hk;
            if (!a.cu_q) {
                const int each = (a.Sq + TP - 1) / TP;
                x.b = item / max(each, 1);
                x.t = (item - x.b * each) * TP;
                return x.b < a.B;
            }
            // a sequence of n tokens has at most n / TP + 1 items: numbers from cu / TP + b on are its own
            if (item >= a.Tq / TP + a.B) return false;
            const int *cu = a.cu_q, tp = TP, T = a.Tq;
            x.b = kv4::warp_find([=](int i) { return (int64_t)(min(max(cu[i], 0), T) / tp) + i; }, a.B, item);
            const int64_t t = (int64_t)(item - min(max(cu[x.b], 0), T) / tp - x.b) * TP;
            // (a number of none: before the first sequence's, or left out)
            x.t = (int)(t < 0 ? (int64_t)0x7fffff00 : min(t, (int64_t)0x7fffff00));
            return true;
        }
        int p = 0, n = count(0) * a.Hk;
        while (rank >= n) {
            if (!split || n == 0) return false;
            rank -= n;
            n = count(of_piece(++p)) * a.Hk;
        }
        x.line = rank;
        x.piece = p;
        const int item = rank / a.Hk;
        x.h = rank - item * a.Hk;
        int lo = 0, hi = most + 1;  // count(lo) > item >= count(hi)
        while (hi - lo > 1) {
            const int mid = lo + (hi - lo) / 2;
            (count(mid) > item ? lo : hi) = mid;
        }
        const int left = item - count(lo + 1);  // among the items of lo tiles, by sequence
        const int ge = items_from(lo), m = ge - items_from(lo + 1);
        const int t0 = a.causal ? all - ge : 0;
        int upto = m;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned here = __ballot_sync(0xffffffffu, left < upto);
        if (!here) return false;
        x.b = __ffs(here) - 1;
        x.t = (__shfl_sync(0xffffffffu, t0, x.b) + left - __shfl_sync(0xffffffffu, upto - m, x.b)) * TP;
        return true;
    }

    // Cuts item x, whose tiles are set, to its piece.
    __device__ __forceinline__ void cut(Item &x, int streams) const {
        const int NT = x.tiles;
        x.pieces = 1;
        x.base = 0;
        if (!split) return;
        x.pieces = (int)max(min((int64_t)NT * gridDim.x / tiles, (int64_t)((NT - 1) / kLeastPiece + 1)), (int64_t)1);
        const int j0 = (int)((int64_t)NT * x.piece / x.pieces), n = (int)((int64_t)NT * (x.piece + 1) / x.pieces) - j0;
        for (int s = 0; s < streams; s++) x.nt[s] = min(max(x.nt[s] - j0, 0), n);
        x.tiles = n;
        x.first = max(x.first - j0, 0);
        x.base = j0 * kTile;
    }
};

// What of shared memory is not tiles.
template <int DP> struct Small {
    using C = Cfg<DP>;
    // tile copies landed, stages free; tiles to be looked through landed, half of one is done
    uint64_t kv_full[C::NST], kv_empty[C::NST], v_raw[C::NST], v_half[C::NST];
    uint64_t q_full[2], q_free[2];  // by stream
    uint64_t s_full[2], p_full[4];  // by score buffer: scores; either half of the weights are there
    uint64_t s_free[2];             // the scores have been read
    uint64_t o_done[2];             // by stream: a product P V is done
    uint64_t item_full[kItems], item_empty[kItems];
    Item items[kItems];
    int abort_s;
    uint32_t tmem;
};

template <int DP, bool F16>
struct Block {
    using C = Cfg<DP>;
    static constexpr int NQ = C::NQ, LA = C::LA, NU = C::NU, UC = C::UC, NST = C::NST;
    static constexpr int kPart = kTile * (DP + 2);  // floats of a stream of a piece

    const Args &a;
    const uint32_t q_a, ring_a;  // shared memory: queries, ring
    unsigned char *ring;
    Small<DP> *small;
    uint32_t tmem;

    __device__ __forceinline__ Block(const Args &args, unsigned char *smem)
        : a(args), q_a(smem_addr(smem)), ring_a(smem_addr(smem) + NQ * C::QB), ring(smem + NQ * C::QB),
          small(reinterpret_cast<Small<DP> *>(smem + NQ * C::QB + NST * C::STAGE)) {}

    // Every wait is bounded; one that gives up records the launch and ends the block's work.
    // (What waits for the end of an item has more time: kWaitNs are 60,000 tiles.)
    __device__ __forceinline__ bool wait(uint64_t *bar, unsigned parity, uint64_t limit = kWaitNs) const {
        if (mbar_try_wait(bar, parity)) return true;
        const uint64_t t0 = global_ns();
        for (;;) {
            if (mbar_try_wait_sleep(bar, parity, 20000)) return true;
            if (*static_cast<volatile int *>(&small->abort_s)) return false;
            if (global_ns() - t0 > limit) {
                atomicMax(a.status, a.epoch);
                *static_cast<volatile int *>(&small->abort_s) = 1;
                return false;
            }
        }
    }

    // The same for a whole warp, which goes on or gives up together.
    __device__ __forceinline__ bool wait_warp(uint64_t *bar, unsigned parity, uint64_t limit = kWaitNs) const {
        return __all_sync(0xffffffffu, wait(bar, parity, limit));
    }

    // Item `it`, in the ring of items until its readers are done with it; null: no more work, or given up.
    template <bool WARP>
    __device__ __forceinline__ const Item *next(int it) const {
        const int slot = it % kItems;
        const unsigned parity = (it / kItems) & 1;
        if (!(WARP ? wait_warp(small->item_full + slot, parity, kItemNs) : wait(small->item_full + slot, parity, kItemNs))) return nullptr;
        return small->items[slot].valid ? small->items + slot : nullptr;
    }
    template <bool WARP>
    __device__ __forceinline__ void done(int it) const {
        if constexpr (WARP) __syncwarp();
        if (!WARP || (threadIdx.x & 31) == 0) mbar_arrive(small->item_empty + it % kItems);
    }

    // A place in the ring: its stage and the parity of its use.
    struct Place {
        int st = 0;
        unsigned phase = 0;
        __device__ __forceinline__ void next() {
            if (++st == NST) {
                st = 0;
                phase ^= 1;
            }
        }
        __device__ __forceinline__ void skip(int n) {
            for (int i = 0; i < n; i++) next();
        }
    };

    // ---------------------------------------------------------------- TMA warp
    __device__ __forceinline__ void load(const CUtensorMap *mq, const CUtensorMap *mk, const CUtensorMap *mv) {
        Place at;
        bool round = false;  // the ring has been filled once
        unsigned q_uses[2] = {0, 0};
        const Item *item;
        for (int it = 0; (item = next<false>(it)); it++) {
            const Item x = *item;
            done<false>(it);
            if (!x.tiles) continue;
            const int bb = a.cu_q ? 0 : x.b;
            auto queries = [&](int s) {
                if (!x.nt[s]) return true;
                if (q_uses[s] && !wait(small->q_free + s, (q_uses[s] - 1) & 1)) return false;
                q_uses[s]++;
                mbar_expect_tx(small->q_full + s, a.TQ * a.G * 128 * (DP / 64));
#pragma unroll
                for (int c = 0; c < DP / 64; c++)
                    tma_load_5d(q_a + s * C::QB + c * kBox, mq, 64 * c, 0, x.h, x.s.q0 + x.t + s * a.TQ, bb, small->q_full + s);
                return true;
            };
            // (a tile that is looked through first arrives there instead)
            auto tile = [&](const CUtensorMap *m, int j, uint64_t *full) {
#pragma unroll
                for (int u = 0; u < NU; u++) {
                    if (round && !wait(small->kv_empty + at.st, at.phase ^ 1)) return false;
                    mbar_expect_tx(full + at.st, C::STAGE);
#pragma unroll
                    for (int c = 0; c < UC / 64; c++)
                        tma_load_4d(ring_a + at.st * C::STAGE + c * kBox, m, u * UC + 64 * c, x.h, x.s.k0 + x.base + j * kTile, bb, full + at.st);
                    at.next();
                    round = round || at.st == 0;
                }
                return true;
            };
            if (!queries(0) || !tile(mk, 0, small->kv_full)) return;
            if (NQ == 2 && !queries(1)) return;
            for (int j = 1; j < min(LA, x.tiles); j++)
                if (!tile(mk, j, small->kv_full)) return;
            for (int j = 0; j < x.tiles; j++) {
                if (!tile(mv, j, j >= x.first ? small->v_raw : small->kv_full)) return;
                if (j + LA < x.tiles && !tile(mk, j + LA, small->kv_full)) return;
            }
        }
    }

    // ---------------------------------------------------------------- MMA warp
    __device__ __forceinline__ void multiply() {
        Place at;
        const uint32_t lead = elect();
        unsigned q_uses[2] = {0, 0}, p_uses[2] = {0, 0}, f_uses[2] = {0, 0};
        constexpr uint32_t id_o = idesc(UC, F16, 1);
        const uint32_t id_s = idesc(kTile, F16, 0) | (uint32_t)a.negative << 13;
        const uint64_t ring_d = sw128_desc(ring_a), q_d = sw128_desc(q_a);
        const Item *item;
        for (int it = 0; (item = next<true>(it)); it++) {
            auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
            const int tiles = uniform(item->tiles), nt[2] = {uniform(item->nt[0]), uniform(item->nt[1])};
            done<true>(it);
            if (!tiles) continue;
            auto full = [&](Place p) {
#pragma unroll
                for (int u = 0; u < NU; u++, p.next())
                    if (!wait_warp(small->kv_full + p.st, p.phase)) return false;
                return true;
            };
            auto release = [&](Place p) {
#pragma unroll
                for (int u = 0; u < NU; u++, p.next()) mma_commit(lead, small->kv_empty + p.st);
            };
            auto scores = [&](int s, int j, Place p) {  // K tile j is at p
                if (j >= nt[s]) return true;
                if (j == 0 && !wait_warp(small->q_full + s, q_uses[s]++ & 1)) return false;
                tc_fence_after();
                const int slot = NQ == 2 ? s : j & 1;
#pragma unroll
                for (int u = 0; u < NU; u++, p.next()) {
                    const uint64_t kd = ring_d + p.st * (C::STAGE >> 4), qd = q_d + ((s * C::QB + u * (UC / 64) * kBox) >> 4);
#pragma unroll
                    for (int k = 0; k < UC / 16; k++) {
                        constexpr int step = 32 >> 4;
                        const int off = (k >> 2) * (kBox >> 4) + (k & 3) * step;
                        mma_ss(lead, tmem + slot * kTile, qd + off, kd + off, id_s, u + k > 0);
                    }
                }
                mma_commit(lead, small->s_full + slot);
                if (j == nt[s] - 1) mma_commit(lead, small->q_free + s);
                return true;
            };
            for (int j = 0; j < min(LA, tiles); j++) {
                if (!full(at)) return;
                for (int s = 0; s < NQ; s++)
                    if (!scores(s, j, at)) return;
                release(at);
                at.skip(NU);
            }
            for (int j = 0; j < tiles; j++) {
                const Place vp = at;
                at.skip(NU);
                const Place kp = at;
                const bool more = j + LA < tiles;
                if (more) at.skip(NU);
                auto product = [&](int s) {
                    if (j >= nt[s]) return true;
                    const int slot = NQ == 2 ? s : j & 1;
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        if (!wait_warp(small->p_full + 2 * slot + half, p_uses[slot] & 1)) return false;
                        tc_fence_after();
                        Place p = vp;
#pragma unroll
                        for (int u = 0; u < NU; u++, p.next()) {
                            const uint64_t vd = ring_d + p.st * (C::STAGE >> 4);
#pragma unroll
                            for (int k = 4 * half; k < 4 * half + 4; k++)
                                mma_ts(lead, tmem + C::O_COL + s * DP + u * UC, tmem + C::P_COL + slot * C::P_STEP + k * 8,
                                       vd + k * (2048 >> 4), id_o, j > 0 || k > 0);
                        }
                    }
                    p_uses[slot]++;
                    mma_commit(lead, small->o_done + s);
                    return true;
                };
                if constexpr (C::BESIDE) {
                    if (more) {
                        if (!full(kp)) return;
#pragma unroll
                        for (int s = 0; s < NQ; s++)
                            if (j + 1 < nt[s] && (!wait_warp(small->s_free + s, (f_uses[s] + j) & 1) || !scores(s, j + 1, kp))) return;
                        release(kp);
                    }
                    if (!full(vp)) return;
#pragma unroll
                    for (int s = 0; s < NQ; s++)
                        if (!product(s)) return;
                    release(vp);
                    continue;
                }
                if (!full(vp)) return;
#pragma unroll
                for (int s = 0; s < NQ; s++) {
                    if (!product(s)) return;
                    if (s == NQ - 1) release(vp);
                    if (more) {
                        if (s == 0 && !full(kp)) return;
                        if (!scores(s, j + LA, kp)) return;
                        if (s == NQ - 1) release(kp);
                    }
                }
            }
            for (int s = 0; s < NQ; s++) f_uses[s] += nt[s];
        }
    }

    // ------------------------------------------------------------ softmax warps
    // A thread has a row.  Its reference and the factors are powers of two: O is scaled without rounding.
    struct Row {
        float ref, l;  // log2 of the reference (a whole number; -inf: nothing seen), sum of weights
    };

    // Weights of 64 scores, packed; POLY: some as polynomials.
    template <bool POLY>
    __device__ __forceinline__ void weigh(const float *z, float2 off, uint32_t *w, float2 sum[2]) const {
        const float2 scale = make_float2(a.scale, a.scale);
#pragma unroll
        for (int k = 0; k < 32; k++) {
            float2 u = __ffma2_rn(make_float2(z[2 * k], z[2 * k + 1]), scale, off);
            if (POLY && k % kPolyStep == kPolyStep - 1) {
                u = exp2_poly<F16>(u);
            } else {
                u.x = exp2_fast(u.x);
                u.y = exp2_fast(u.y);
            }
            sum[k & 1] = __fadd2_rn(sum[k & 1], u);
            w[k] = pack2<F16>(u.x, u.y);
        }
    }

    // One tile of scores into weights.  The scores are read once, in one go: a load from TMEM takes 300
    // cycles while products are running (four of 32 keys, each waited for: 1800 cycles a tile instead of
    // 1400).  The product with V begins when the first 64 keys' weights are there.
    template <bool MASK>
    __device__ __forceinline__ bool tile(Row &r, int s, int slot, uint32_t lanes, int lim, bool on, bool first, unsigned o_count) const {
        const uint32_t at = tmem + lanes + slot * kTile, to = tmem + lanes + C::P_COL + slot * C::P_STEP;
        float z[kTile];
#pragma unroll
        for (int c = 0; c < kTile; c += 32) tmem_ld32(at + c, z + c);
        tmem_landed<kTile>(z);
        if constexpr (C::BESIDE) {
            tc_fence_before();
            __syncwarp();
            if ((threadIdx.x & 31) == 0) mbar_arrive(small->s_free + slot);
        }
        if constexpr (MASK) {  // 32 keys at a time, where one of the warp's rows does not see them all
            const int least = __reduce_min_sync(0xffffffffu, lim);
#pragma unroll
            for (int c = 0; c < kTile; c += 32)
                if (least < c + 32) {
#pragma unroll
                    for (int k = c; k < c + 32; k++) z[k] = k < lim ? z[k] : -INFINITY;
                }
        }
        float m[8] = {z[0], z[1], z[2], z[3], z[4], z[5], z[6], z[7]};
#pragma unroll
        for (int k = 8; k < 120; k += 16)
#pragma unroll
            for (int e = 0; e < 8; e++) m[e] = fmaxf(fmaxf(m[e], z[k + e]), z[k + 8 + e]);
#pragma unroll
        for (int e = 0; e < 8; e++) m[e] = fmaxf(m[e], z[120 + e]);
        const float top = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), fmaxf(fmaxf(m[4], m[5]), fmaxf(m[6], m[7])));
        // The reference follows only a maximum that is 2^8 above it: weights stay below 2^8.  A warp's rows move
        // theirs together; rows of no query, which hold the next sequence's queries or nothing that was written,
        // do not ask for it: another reference is another rounding of the weights.
        float f = 1.f;
        const bool moved = __any_sync(0xffffffffu, on && fmaf(top, a.scale, -r.ref) > 8.f);
        if (moved) {
            const float n = fmaxf(r.ref, ceilf(top * a.scale)), d = r.ref - n;  // d <= 0, no number where both are infinite
            f = d == 0.f ? 1.f : d > -126.f ? __int_as_float(((int)d + 127) << 23) : 0.f;
            r.ref = n;
            r.l *= f;
        }
        const float off = r.ref == -INFINITY ? 0.f : kUp<F16> - r.ref;
        const float2 off2 = make_float2(off, off);
        float2 sum[2] = {};
        uint32_t w[32];
        weigh<!MASK>(z, off2, w, sum);
        // O, and weights beside the scores, wait for the last product.  So does every tile whose scores came
        // ahead of it: at most one product may be open when the next is waited for, a parity tells no more apart.
        if (!first && (C::BESIDE || NQ == 1 || moved)) {
            if (!wait_warp(small->o_done + s, (o_count - 1) & 1)) return false;
            tc_fence_after();
        }
        tmem_st32(to, w);
        if (moved && !first) {
#pragma unroll 1
            for (int c = 0; c < DP; c += 16) {
                float o[16];
                const uint32_t oat = tmem + lanes + C::O_COL + s * DP + c;
                tmem_ld16(oat, o);
                tmem_landed<16>(o);
#pragma unroll
                for (int k = 0; k < 16; k++) o[k] *= f;
                tmem_st16(oat, reinterpret_cast<const uint32_t *>(o));
            }
        }
        ready(slot, 0);
        weigh<!MASK>(z + 64, off2, w, sum);
        tmem_st32(to + 32, w);
        r.l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        ready(slot, 1);
        return true;
    }
    // Half a tile's weights are there.
    __device__ __forceinline__ void ready(int slot, int half) const {
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(small->p_full + 2 * slot + half);
    }

    __device__ __forceinline__ void softmax(int s) {
        const int row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(row & ~31) << 16;  // of this warp
        const int tok = row / a.G, head = row - tok * a.G;
        unsigned s_uses[2] = {0, 0}, o_count = 0;
        const Item *item;
        for (int it = 0; (item = next<true>(it)); it++) {
            // (rows of no query need no mask: their results go nowhere)
            const int i = item->t + s * a.TQ + tok;
            const int vis = tok < a.TQ && i < item->s.nq ? visible(a, item->s, i) - item->base : kNoRow;
            Row r{-INFINITY, 0.f};
            const int nt = item->nt[s];
            for (int j = 0; j < nt; j++) {
                const int slot = NQ == 2 ? s : j & 1;
                // (the first scores come when the other stream is done with its tiles of the item before)
                if (!wait_warp(small->s_full + slot, s_uses[NQ == 2 ? 0 : slot]++ & 1, j ? kWaitNs : kItemNs)) return;
                tc_fence_after();
                const int lim = vis - j * kTile;
                const bool on = vis != kNoRow;
                if (__any_sync(0xffffffffu, lim < kTile) ? !tile<true>(r, s, slot, lanes, lim, on, j == 0, o_count)
                                                         : !tile<false>(r, s, slot, lanes, lim, on, j == 0, o_count))
                    return;
                o_count++;
            }
            if (nt && !wait_warp(small->o_done + s, (o_count - 1) & 1)) return;
            tc_fence_after();
            write(*item, s, tok, head, nt, r, lanes);
            done<true>(it);
        }
    }

    // Outputs of one row, or what they are joined from.
    __device__ __forceinline__ void write(const Item &x, int s, int tok, int head, int nt, const Row &r, uint32_t lanes) const {
        using T = typename std::conditional<F16, __half, __nv_bfloat16>::type;
        const int i = x.t + s * a.TQ + tok, h = x.h * a.G + head, row = threadIdx.x & 127;
        const bool on = tok < a.TQ && i < x.s.nq, cut = x.pieces > 1;
        const int64_t at = a.cu_q ? x.s.q0 + i : i;
        T *out = static_cast<T *>(a.out) + (a.cu_q ? 0 : x.b * a.o_sb) + at * a.o_ss + h * a.o_sh;
        // 32 columns of the warp's rows, in 16-byte pieces that four lanes exchange: a store then has 64 bytes of
        // 8 rows each, not 16 of 32 (with those an item's outputs took 3 us).
        const int lane = threadIdx.x & 31, r4 = lane & 3;
        T *to[4];
        unsigned rows = __ballot_sync(0xffffffffu, on) >> (lane & ~3);
#pragma unroll
        for (int k = 0; k < 4; k++)
            to[k] = reinterpret_cast<T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), (lane & ~3) + k));
        auto store = [&](float *o, int c, float inv, bool zero) {
            uint32_t w[4][4];
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    w[k][e] = zero ? 0u : pack2<F16>(o[8 * k + 2 * e] * inv, o[8 * k + 2 * e + 1] * inv);
            if (!a.o_vec) {
                if (on)
#pragma unroll
                    for (int k = 0; k < 4; k++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            reinterpret_cast<uint16_t *>(out)[c + 8 * k + 2 * e] = (uint16_t)w[k][e];
                            reinterpret_cast<uint16_t *>(out)[c + 8 * k + 2 * e + 1] = (uint16_t)(w[k][e] >> 16);
                        }
                return;
            }
#pragma unroll
            for (int m = 1; m < 4; m *= 2)  // transposed: piece r4 of the four lanes' rows
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (k & m) continue;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t give = r4 & m ? w[k][e] : w[k + m][e];
                        const uint32_t got = __shfl_xor_sync(0xffffffffu, give, m);
                        if (r4 & m) w[k][e] = got;
                        else w[k + m][e] = got;
                    }
                }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (rows >> k & 1) *reinterpret_cast<uint4 *>(to[k] + c + 8 * r4) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
        };
        auto log_sum = [&](float ref, float l) {
            if (on && a.lse)
                a.lse[(a.cu_q ? at : (int64_t)x.b * a.Sq + i) * a.Hq + h] = l == 0.f ? -INFINITY : (ref - kUp<F16> + log2f(l)) * 0.693147180559945309f;
        };
        const float inv = r.l == 0.f ? 0.f : 1.f / r.l;
        const bool fix = nt && *const_cast<const volatile int *>(&x.bad);
        float *part = a.parts + ((int64_t)x.unit * NQ + s) * kPart + row;  // columns of 128 rows, then references and sums
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
            if (c >= a.D) break;
            float o[32];
            if (nt) {
                tmem_ld32(tmem + lanes + C::O_COL + s * DP + c, o);
                tmem_landed<32>(o);
            }
            if (fix && on) {  // values of the masked tiles that are no numbers
                const T *v = static_cast<const T *>(a.v) + (a.cu_q ? 0 : x.b * a.v_sb) + x.h * a.v_sh + c;
                for (int j = x.base + x.first * kTile, n = min(visible(a, x.s, i), x.base + nt * kTile); j < n; j++)
#pragma unroll
                    for (int k = 0; k < 32; k++) {
                        const float y = Elem<T>::to_f32(v[(int64_t)(x.s.k0 + j) * a.v_ss + k]);
                        if (!(fabsf(y) < INFINITY)) o[k] += y;
                    }
            }
            if (!cut) {
                store(o, c, inv, r.l == 0.f);
            } else if (nt) {
#pragma unroll
                for (int k = 0; k < 32; k++) part[(c + k) * kTile] = o[k];
            }
        }
        tc_fence_before();
        if (!cut) {
            log_sum(r.ref, r.l);
            return;
        }
        // The warp that is the last one of its rows joins the pieces, in order.
        part[DP * kTile] = r.ref;
        part[(DP + 1) * kTile] = nt ? r.l : 0.f;
        int last = 0;
        int *slots = a.slots + x.line * kMaxPieces;
        if ((threadIdx.x & 31) == 0) slots[x.piece] = x.unit;
        __threadfence();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) {
            int *counter = a.counters + (x.line * 2 + s) * 4 + (row >> 5);
            last = atomicAdd(counter, 1) == x.pieces - 1;
            if (last) *counter = 0;
            __threadfence();
        }
        if (!__shfl_sync(0xffffffffu, last, 0)) return;
        auto of = [&](int p) { return a.parts + ((int64_t)__ldcg(slots + p) * NQ + s) * kPart + row; };
        float ref = -INFINITY, l = 0.f;
        for (int p = 0; p < x.pieces; p++) {
            const float *z = of(p);
            if (__ldcg(z + (DP + 1) * kTile) != 0.f) ref = fmaxf(ref, __ldcg(z + DP * kTile));
        }
        auto factor = [&](const float *z) {  // references are whole numbers
            const float e = __ldcg(z + DP * kTile);
            return e == ref ? 1.f : exp2_fast(e - ref);
        };
        for (int p = 0; p < x.pieces; p++) {
            const float *z = of(p), y = __ldcg(z + (DP + 1) * kTile);
            if (y != 0.f) l = fmaf(y, factor(z), l);
        }
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
            if (c >= a.D) break;
            float o[32] = {};
#pragma unroll 1
            for (int p = 0; p < x.pieces; p++) {
                const float *z = of(p);
                if (__ldcg(z + (DP + 1) * kTile) == 0.f) continue;
                const float f = factor(z);
#pragma unroll
                for (int k = 0; k < 32; k++) o[k] = fmaf(__ldcg(z + (c + k) * kTile), f, o[k]);
            }
            store(o, c, l == 0.f ? 0.f : 1.f / l, l == 0.f);
        }
        log_sum(ref, l);
    }

    // ------------------------------------------------------------- helper warps
    // Warp 0 of the two also finds the items, one ahead of the values that it looks through.
    __device__ __forceinline__ void help(int w) {
        const int lane = threadIdx.x & 31;
        int64_t pos = 0;  // where the item's tiles begin
        const Line line(a, NQ * a.TQ);
        auto publish = [&](int it) {
            const int slot = it % kItems;
            if (it >= kItems && !wait_warp(small->item_empty + slot, (it / kItems - 1) & 1, kItemNs)) return false;
            const int n = gridDim.x, c = blockIdx.x;
            Item x{};
            x.valid = line.find(it * n + (it & 1 ? n - 1 - c : c), x);
            if (x.valid) {
                x.s = sequence(a, x.b);
                x.t = min(x.t, x.s.nq);
                for (int s = 0; s < NQ; s++) {
                    const int t0 = x.t + s * a.TQ;
                    x.nt[s] = t0 < x.s.nq ? tiles_of(visible(a, x.s, min(t0 + a.TQ, x.s.nq) - 1)) : 0;
                }
                x.tiles = max(x.nt[0], x.nt[1]);
                x.first = visible(a, x.s, x.t) / kTile;
                line.cut(x, NQ);
            }
            if (lane == 0) {
                small->items[slot] = x;
                mbar_arrive(small->item_full + slot);
            }
            return true;
        };
        if (w == 0 && !publish(0)) return;
        unsigned seen = 0;  // by stage: the parity of the tiles looked through
        const Item *item;
        for (int it = 0; (item = next<true>(it)); it++) {
            const Item x = *item;
            done<true>(it);
            if (w == 0 && !publish(it + 1)) return;
            bool any = false;
            for (int j = x.first; j < x.tiles; j++)
                for (int u = 0; u < NU; u++) {
                    // order: K0 .. K(LA - 1), then V(j), K(j + LA) for every j
                    const int st = (int)((pos + NU * (min(LA, x.tiles) + j + min(j, max(x.tiles - LA, 0))) + u) % NST);
                    // (A barrier for these tiles alone: their next use waits for this one, so no phase of
                    // it can be missed, and none passed by a warp that is ahead.)
                    const unsigned parity = seen >> st & 1;
                    seen ^= 1u << st;
                    if (!wait_warp(small->v_raw + st, parity, kItemNs)) return;
                    uint4 *v = reinterpret_cast<uint4 *>(ring + st * C::STAGE) + w * 32 + lane;
                    constexpr uint32_t E = F16 ? 0x7c007c00u : 0x7f807f80u, ONE = F16 ? 0x04000400u : 0x00800080u;
#pragma unroll 4
                    for (int i = 0; i < C::STAGE / 16 / 64; i++) {
                        uint4 y = v[i * 64];
                        // an exponent of all ones carries into the sign bit
                        auto odd = [](uint32_t z) { return ((z & E) + ONE) & 0x80008000u; };
                        if (odd(y.x) | odd(y.y) | odd(y.z) | odd(y.w)) {
                            any = true;
                            auto zero = [&](uint32_t z) {
                                const uint32_t m = odd(z);
                                return z & ~((m >> 15) * 0xffffu);
                            };
                            v[i * 64] = make_uint4(zero(y.x), zero(y.y), zero(y.z), zero(y.w));
                        }
                    }
                    if (any) *const_cast<volatile int *>(&item->bad) = 1;
                    fence_async_smem();
                    __syncwarp();
                    if (w == 0 && !wait_warp(small->v_half + st, parity)) return;
                    if (lane == 0) mbar_arrive(w == 0 ? small->kv_full + st : small->v_half + st);
                }
            pos += 2 * (int64_t)NU * x.tiles;
        }
    }
};

template <int DP, bool F16>
__global__ void __launch_bounds__(Cfg<DP>::THREADS, 1)
prompt_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
              const __grid_constant__ CUtensorMap mv, const __grid_constant__ Args a) {
    using C = Cfg<DP>;
    extern __shared__ __align__(1024) unsigned char smem[];
    Block<DP, F16> k(a, smem);
    Small<DP> &m = *k.small;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int SW = 4 * C::NQ;  // softmax warps
    if (k.q_a & 1023) {  // tiles of 128-byte swizzle begin at multiples of 1024
        if (threadIdx.x == 0) atomicMax(a.status, a.epoch);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NST; i++) {
            mbar_init(m.kv_full + i, 1);
            mbar_init(m.kv_empty + i, 1);
            mbar_init(m.v_raw + i, 1);
            mbar_init(m.v_half + i, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(m.q_full + i, 1);
            mbar_init(m.q_free + i, 1);
            mbar_init(m.s_full + i, 1);
            mbar_init(m.p_full + 2 * i, 4);
            mbar_init(m.p_full + 2 * i + 1, 4);
            mbar_init(m.s_free + i, 4);
            mbar_init(m.o_done + i, 1);
        }
        for (int i = 0; i < kItems; i++) {
            mbar_init(m.item_full + i, 1);
            mbar_init(m.item_empty + i, SW + 4);
        }
        m.abort_s = 0;
        fence_mbar_init();
    }
    if (warp == SW + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&m.tmem)));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // rows of no sequence: zeros
    if (a.cu_q) {
        const int lo = a.B ? min(max(a.cu_q[0], 0), a.Tq) : a.Tq, hi = a.B ? min(max(a.cu_q[a.B], 0), a.Tq) : a.Tq;
        const int64_t n = (int64_t)(lo + a.Tq - hi) * a.Hq;
        for (int64_t r = (int64_t)blockIdx.x * (C::THREADS / 32) + warp; r < n; r += (int64_t)gridDim.x * (C::THREADS / 32)) {
            const int64_t t = r / a.Hq, row = t < lo ? t : t - lo + hi, h = r - t * a.Hq;
            uint16_t *out = static_cast<uint16_t *>(a.out) + row * a.o_ss + h * a.o_sh;
            for (int d = lane; d < a.D; d += 32) out[d] = 0;
            if (a.lse && lane == 0) a.lse[row * a.Hq + h] = -INFINITY;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    k.tmem = m.tmem;
    // Two streams: 384 threads of 168 registers, shared out as 256 of 208 and 128 of 88.
    if (warp < SW) {
        if constexpr (C::NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        k.softmax(warp >> 2);
    } else {
        if constexpr (C::NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == SW) {
            if (lane == 0) {
                asm volatile("prefetch.tensormap [%0];" ::"l"(&mq) : "memory");
                asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
                asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
                k.load(&mq, &mk, &mv);
            }
        } else if (warp == SW + 1) {
            k.multiply();
        } else {
            k.help(warp - SW - 2);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (m.abort_s) {  // copies and products in flight end (within microseconds) before their memory is given back
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 2000000) {}
    }
    if (warp == SW + 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(k.tmem));
    }
}

// ------------------------------------------------------------------ host side
PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// A map of `rank` dims, the channels first; boxes of 64 of them.
bool encode(CUtensorMap *map, bool f16, const void *p, int rank, const int64_t *dims, const int64_t *strides, const int64_t *box) {
    cuuint64_t d[5], s[4];
    cuuint32_t b[5], e[5];
    for (int i = 0; i < rank; i++) {
        d[i] = (cuuint64_t)dims[i];
        b[i] = (cuuint32_t)box[i];
        e[i] = 1;
        if (i) s[i - 1] = (cuuint64_t)(dims[i] > 1 ? strides[i] * 2 : 16);
    }
    auto fn = get_encode();
    return fn && fn(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void *>(p),
                    d, s, b, e, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What a map can walk: rows on 16-byte boundaries, apart from one another.
bool walkable(const void *p, int64_t sb, int64_t nb, int64_t ss, int64_t ns, int64_t sh, int64_t nh) {
    auto ok = [](int64_t s, int64_t n) { return n <= 1 || (s > 0 && s % 8 == 0 && s < (int64_t(1) << 38)); };
    return aligned(p, 16) && ok(sb, nb) && ok(ss, ns) && ok(sh, nh);
}

template <int DP, bool F16>
int launch(const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, const Args &a, int64_t blocks, cudaStream_t st) {
    using C = Cfg<DP>;
    constexpr int smem = C::NQ * C::QB + C::NST * C::STAGE + (int)sizeof(Small<DP>);
    static_assert(smem <= 232448, "shared memory");
    static bool ready[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { set_error("prompt_attn: no device"); return FC_ECUDA; }
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(prompt_kernel<DP, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
            set_error("prompt_attn: the kernel does not fit this device");
            return FC_ECUDA;
        }
        // warps that ask for more registers wait for what others give back: a kernel that was built
        // with too few to share out is never launched
        cudaFuncAttributes attr;
        if (cudaFuncGetAttributes(&attr, prompt_kernel<DP, F16>) != cudaSuccess || (C::NQ == 2 && attr.numRegs != 168)) {
            set_error("prompt_attn: the kernel was built with another number of registers");
            return FC_ECUDA;
        }
        ready[dev] = true;
    }
    prompt_kernel<DP, F16><<<(unsigned)blocks, C::THREADS, smem, st>>>(mq, mk, mv, a);
    return check_launch("prompt_attn");
}

}  // namespace
}  // namespace prompt
}  // namespace fc

using namespace fc;
using namespace fc::prompt;

namespace {
// Tokens of an item, and a bound of the number of (item, head), whatever the lengths.
int64_t item_tokens(int64_t D, int64_t G) { return (D <= 128 ? 2 : 1) * (kTile / G); }
int64_t most_items(int64_t B, int64_t Tq, int64_t Hk, int64_t TP) {
    const int64_t n = (Tq / TP + B) * Hk;
    return n > 0 ? n : 1;
}
// Items are cut along their keys where they are fewer than blocks; there are at most twice as many pieces as blocks then.
int64_t parts_bytes(int64_t D, int64_t items) {
    const int64_t DP = D <= 64 ? 64 : D <= 128 ? 128 : D;
    return items < num_sms() ? 2 * (int64_t)num_sms() * (D <= 128 ? 2 : 1) * kTile * (DP + 2) * 4 : 0;
}
constexpr int64_t kSlotsBytes = (int64_t)kMaxPieces * kMaxPieces * 4;
}  // namespace

extern "C" size_t fc_prompt_attn_workspace_size(int64_t B, int64_t Tq, int64_t Hq, int64_t Hk, int64_t D) {
    if (Hk <= 0 || Hq < Hk || Hq / Hk > kTile) return kWsHeader + kWsUnits * 4;
    const int64_t parts = parts_bytes(D, most_items(B, Tq, Hk, item_tokens(D, Hq / Hk)));
    return (size_t)(kWsHeader + kWsUnits * 4 + (parts ? kSlotsBytes + parts : 0));
}

extern "C" int fc_prompt_attn(const void *q, int64_t q_sb, int64_t q_ss, int64_t q_sh, const void *k, int64_t k_sb,
                              int64_t k_ss, int64_t k_sh, const void *v, int64_t v_sb, int64_t v_ss, int64_t v_sh,
                              int dtype, int64_t B, int64_t Sq, int64_t Sk, int64_t Tq, int64_t Tk, int64_t Hq,
                              int64_t Hk, int64_t D, const int *cu_seqlens_q, const int *cu_seqlens_k, int causal,
                              float softmax_scale, void *out, int64_t o_sb, int64_t o_ss, int64_t o_sh, float *lse,
                              void *workspace, size_t workspace_bytes, void *stream) {
    clear_error();
    if (!kv4::head_dim_ok(D)) {
        set_error("prompt_attn: head dim %lld is not one of 64, 96, 128, 192, 256", (long long)D);
        return FC_ENOTSUP;
    }
    if (dtype != FC_BF16 && dtype != FC_F16) { set_error("prompt_attn: dtype must be bf16 or fp16"); return FC_ENOTSUP; }
    if (B < 0 || B > (1 << 24) || Tq < 0 || Tk < 0 || Sq < 0 || Sk < 0 || Tq > 0x7fffff00 || Tk > 0x7fffff00 ||
        (cu_seqlens_q == nullptr) != (cu_seqlens_k == nullptr) ||
        (!cu_seqlens_q && (Tq != B * Sq || Tk != B * Sk))) {
        set_error("prompt_attn: bad shape");
        return FC_EINVAL;
    }
    if (Hk <= 0 || Hq <= 0 || Hq > 65535 || Hq % Hk) {
        set_error("prompt_attn: query heads (%lld) must be a multiple of kv heads (%lld)", (long long)Hq, (long long)Hk);
        return FC_EINVAL;
    }
    if (Hq / Hk > kTile) { set_error("prompt_attn: more than %d query heads to a kv head", kTile); return FC_ENOTSUP; }
    if (!(softmax_scale == softmax_scale) || softmax_scale - softmax_scale != 0.f) {
        set_error("prompt_attn: the softmax scale must be finite");
        return FC_EINVAL;
    }
    if (Tq == 0) return FC_OK;
    if (!q || !out || (Tk && (!k || !v))) { set_error("prompt_attn: null pointer"); return FC_EINVAL; }
    const int64_t size = dtype_size(dtype), nb = cu_seqlens_q ? 1 : B, nq = cu_seqlens_q ? Tq : Sq,
                  nk = cu_seqlens_q ? Tk : Sk;
    const Rows to{out, o_sb, o_ss, o_sh, Hq}, from{q, q_sb, q_ss, q_sh, Hq};
    if (!same_rows(to, from, nb, nq) && rows_meet(to, from, nb, nq, D, size)) {
        set_error("prompt_attn: out overlaps q (it may be q itself)");
        return FC_EINVAL;
    }
    if (rows_repeat(to, nb, nq)) { set_error("prompt_attn: out has rows in one place"); return FC_EINVAL; }
    if (Tk && (meets(to, nq, Rows{k, k_sb, k_ss, k_sh, Hk}, nk, nb, D, size) ||
               meets(to, nq, Rows{v, v_sb, v_ss, v_sh, Hk}, nk, nb, D, size))) {
        set_error("prompt_attn: out overlaps k or v");
        return FC_EINVAL;
    }
    if (!workspace || !aligned(workspace, 16)) { set_error("prompt_attn: null or misaligned workspace"); return FC_EINVAL; }
    if (workspace_bytes < fc_prompt_attn_workspace_size(B, Tq, Hq, Hk, D)) {
        set_error("prompt_attn: workspace of %zu bytes is too small", workspace_bytes);
        return FC_ERANGE;
    }
    if (!walkable(q, q_sb, nb, q_ss, nq, q_sh, Hq) ||
        (Tk && (!walkable(k, k_sb, nb, k_ss, nk, k_sh, Hk) || !walkable(v, v_sb, nb, v_ss, nk, v_sh, Hk)))) {
        set_error("prompt_attn: rows of q, k and v must lie on 16-byte boundaries, with positive strides");
        return FC_EINVAL;
    }
    const bool f16 = dtype == FC_F16;
    Args a{};
    a.v = v; a.out = out; a.lse = lse;
    a.v_sb = v_sb; a.v_ss = v_ss; a.v_sh = v_sh;
    a.o_sb = o_sb; a.o_ss = o_ss; a.o_sh = o_sh;
    a.Sq = (int)Sq; a.Sk = (int)Sk; a.Tq = (int)Tq; a.Tk = (int)Tk;
    a.B = (int)B; a.D = (int)D; a.Hq = (int)Hq; a.Hk = (int)Hk; a.G = (int)(Hq / Hk); a.TQ = kTile / a.G;
    a.causal = causal;
    a.o_vec = rows_aligned(out, dtype, o_sb, o_ss, o_sh);
    a.cu_q = cu_seqlens_q; a.cu_k = cu_seqlens_k;
    const float s = softmax_scale * 1.44269504088896341f;
    a.negative = s < 0.f;
    // a factor of zero would turn a masked score into a NaN; this one rounds every score to zero
    a.scale = s < 0.f ? -s : s > 1e-30f ? s : 1e-30f;
    a.status = static_cast<int *>(workspace);
    a.epoch = next_epoch();
    const int64_t one = 1;
    CUtensorMap mq, mk, mv;
    {
        const int64_t dims[5] = {D, a.G, Hk, nq, nb}, st[5] = {1, q_sh, a.G * q_sh, q_ss, q_sb}, box[5] = {64, a.G, 1, a.TQ, 1};
        bool ok = encode(&mq, f16, q, 5, dims, st, box);
        const int64_t kd[4] = {D, Hk, nk > one ? nk : one, nb}, kb[4] = {64, 1, kTile, 1};
        const int64_t ks[4] = {1, k_sh, k_ss, k_sb}, vs[4] = {1, v_sh, v_ss, v_sb};
        ok = ok && encode(&mk, f16, Tk ? k : q, 4, kd, ks, kb) && encode(&mv, f16, Tk ? v : q, 4, kd, vs, kb);
        if (!ok) { set_error("prompt_attn: the tensor maps cannot be made"); return FC_ECUDA; }
    }
    const int64_t items = most_items(B, Tq, Hk, item_tokens(D, a.G));
    if (items > 0x3fffffff) { set_error("prompt_attn: too many rows"); return FC_ENOTSUP; }
    // (blocks for pieces: one an SM, where the keys are long enough to be cut at all)
    const int sms = num_sms() < kMaxPieces ? num_sms() : kMaxPieces;
    const int64_t keys = cu_seqlens_q ? Tk : Sk;
    a.split = items < num_sms() && B <= 32 && keys > kLeastPiece * kTile;
    a.items = (int)items;
    char *ws = static_cast<char *>(workspace) + kWsHeader;
    a.counters = reinterpret_cast<int *>(ws);
    a.slots = reinterpret_cast<int *>(ws + kWsUnits * 4);
    a.parts = reinterpret_cast<float *>(ws + kWsUnits * 4 + kSlotsBytes);
    const int64_t blocks = a.split ? sms : items < num_sms() ? items : num_sms();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        return f16 ? launch<DP, true>(mq, mk, mv, a, blocks, st) : launch<DP, false>(mq, mk, mv, a, blocks, st);
    };
    if (D == 64) return go(std::integral_constant<int, 64>());
    if (D <= 128) return go(std::integral_constant<int, 128>());
    if (D == 192) return go(std::integral_constant<int, 192>());
    return go(std::integral_constant<int, 256>());
}
