// Paged 4-bit KV cache: the pages of each sequence and KV head worth attending to.
//
// A page's bounds give an upper bound of z . k over its keys, z the rounded queries:
// the sum over channels of max(z * least, z * largest).  Summed over the heads of a group this is linear
// in the positive and the negative parts of the queries, so a page costs one dot
// product of 2 D bytes with two vectors, P = sum_heads max(z, 0) and N = sum_heads
// min(z, 0), whatever the number of heads:
//     score = (P . largest + N . least) * 2^exponent
// z is the query in whole numbers (|z| <= 127, common power of two of the group),
// so the sums are exact (below 2^24, also as fp32) and the choice of pages does not
// depend on the order of any sum.
//
// The bounds, 2 D bytes a page, are read once; HBM bounds the scoring, a chain of short
// steps the choice.  A lane takes 16 bytes of a page, 8 two-way integer dot products; a
// warp 32 pages.  The block that finishes a (sequence, head) last chooses: the keys (scores
// in unsigned order) are counted in 1024 equal bins between the least and the largest, the
// bin that holds the last key wanted is counted in the same way, until what is wanted of it
// is all or one value; one prefix sum over the pages then writes the indices in order.
// 2048 pages of 4 x 8 (sequence, head)s at D = 128 (17 MB): 13.6 us, of which the choice
// takes some 8; keys kept in shared memory between its passes did not shorten it.
#include "fc_kv4.cuh"

namespace fc {
namespace kv4 {
namespace {

struct SelectArgs {
    const void *q;
    int dtype;
    int64_t q_sb, q_sh;
    int Hq, Hk;
    const signed char *bounds;
    const int *exps;
    Table table;
    const int *lengths;
    int count, sink, recent;
    int *out;
    int *counters;   // (B, Hk), zero between calls
    uint32_t *keys;  // (B, Hk, max_pages)
    int shift;       // ceil(log2(G * D / 1024)) where positive
};

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBlockPages = 32 * kWarps;  // pages of a block
constexpr int kBins = 1024;
constexpr int kHold = 16;                 // keys of a thread at a time

// Order-preserving map of finite fp32 to unsigned.
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct PickShared {
    uint32_t hist[kBins];
    uint32_t part[kWarps], part2[kWarps];
    uint32_t bin, above, inside;
};

// Sum over the threads before this one, and over all of them.
__device__ __forceinline__ uint32_t scan_before(uint32_t x, uint32_t *part, uint32_t &all) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t upto = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
    }
    __syncthreads();  // earlier readers of part are done
    if (lane == 31) part[warp] = upto;
    __syncthreads();
    uint32_t before = upto - x;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
        if (w < warp) before += part[w];
        all += part[w];
    }
    return before;
}

// The choice for one (sequence, KV head): n > count keys.
__device__ void pick(const SelectArgs &a, const uint32_t *keys, int n, int *out, PickShared &s) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int first = a.sink, last = n - a.recent;  // the pages between stand for choice
    uint32_t rest = (uint32_t)(a.count - a.sink - a.recent);
    // f(key, page) of every page that stands for choice, this thread's of each window
    auto each = [&](auto f) {
        for (int i0 = 0; i0 < n; i0 += kThreads * kHold) {
            uint32_t k[kHold];
#pragma unroll
            for (int j = 0; j < kHold; j++) {
                const int i = i0 + j * kThreads + (int)threadIdx.x;
                k[j] = i >= first && i < last ? __ldcg(keys + i) : 0u;
            }
#pragma unroll
            for (int j = 0; j < kHold; j++) {
                const int i = i0 + j * kThreads + (int)threadIdx.x;
                if (i >= first && i < last) f(k[j]);
            }
        }
    };
    // from `from` on a key is taken, but of those equal to `from` only `rest` if `some`
    uint32_t from = 0xffffffffu;
    bool some = false;
    if (rest) {
        uint32_t lo = 0xffffffffu, hi = 0;
        each([&](uint32_t k) { lo = min(lo, k); hi = max(hi, k); });
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0) { s.part[warp] = lo; s.part2[warp] = hi; }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; w++) { lo = min(lo, s.part[w]); hi = max(hi, s.part2[w]); }
        uint32_t range = hi - lo;
        for (;;) {
            const int shift = max(0, 22 - __clz(range));  // range >> shift < 1024
            for (int i = threadIdx.x; i < kBins; i += kThreads) s.hist[i] = 0;
            __syncthreads();
            each([&](uint32_t k) {
                if (k - lo <= range) atomicAdd(&s.hist[(k - lo) >> shift], 1u);
            });
            __syncthreads();
            // bins from the top: this thread's four are 1023 - 4 t and the ones below
            const int top = kBins - 1 - 4 * (int)threadIdx.x;
            const uint32_t h[4] = {s.hist[top], s.hist[top - 1], s.hist[top - 2], s.hist[top - 3]};
            uint32_t all, above = scan_before(h[0] + h[1] + h[2] + h[3], s.part, all);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (above < rest && rest <= above + h[i]) {
                    s.bin = top - i;
                    s.above = above;
                    s.inside = h[i];
                }
                above += h[i];
            }
            __syncthreads();
            rest -= s.above;
            from = lo + (s.bin << shift);
            if (rest == s.inside) break;  // all of the bin
            if (shift == 0) { some = true; break; }
            lo = from;
            range = (1u << shift) - 1;
            __syncthreads();  // s.bin is read
        }
    }
    // indices in ascending order: a thread takes neighbouring pages
    uint32_t done = 0, equal = 0;  // of the windows before
    for (int i0 = 0; i0 < n; i0 += kThreads * kHold) {
        const int per = min(kHold, (n - i0 + kThreads - 1) / kThreads);
        const int b = i0 + (int)threadIdx.x * per, e = min(b + per, n);
        uint32_t over = 0, same = 0;  // bit j: page b + j is taken; equals the last key
#pragma unroll
        for (int j = 0; j < kHold; j++) {
            const int i = b + j;
            if (i >= e || j >= per) continue;
            if (i < first || i >= last) {
                over |= 1u << j;
            } else if (a.count > a.sink + a.recent) {
                const uint32_t k = __ldcg(keys + i);
                if (k > from || (k == from && !some)) over |= 1u << j;
                if (k == from && some) same |= 1u << j;
            }
        }
        uint32_t all;
        const uint32_t eq = equal + scan_before(__popc(same), s.part, all);
        equal += all;
        // of the equal ones the first `rest`
        uint32_t take = over, left = eq < rest ? rest - eq : 0u;
        for (uint32_t m = same; m && left; m &= m - 1, left--) take |= m & -m;
        uint32_t at = done + scan_before(__popc(take), s.part2, all);
        done += all;
        for (uint32_t m = take; m; m &= m - 1) out[at++] = b + __ffs(m) - 1;
    }
}

// Lanes that share a page, 16 bytes each: a power of two of at least 4 W.
constexpr int lanes_per_page(int W) { return W <= 2 ? 8 : W <= 4 ? 16 : 32; }

template <int W>
__global__ void __launch_bounds__(kThreads) select_kernel(const __grid_constant__ SelectArgs a) {
    constexpr int D = 32 * W, GRP = lanes_per_page(W), PPW = 32 / GRP;
    __shared__ __align__(16) short z[16 * GRP];  // N then P, as the bounds: least then largest
    __shared__ float wmax[kWarps];
    __shared__ PickShared pick_s;
    __shared__ int last_s;
    const int h = blockIdx.y;
    const int64_t b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.Hq / a.Hk;
    const int64_t q0 = b * a.q_sb + (int64_t)h * G * a.q_sh;
    const int len = a.table.length(a.lengths[b]);
    const int n = (len + (1 << a.table.log_page) - 1) >> a.table.log_page;
    int *out = a.out + (b * a.Hk + h) * a.count;
    if (n <= a.count) {  // everything is taken: no scores needed
        if (blockIdx.x == 0)
            for (int i = threadIdx.x; i < a.count; i += kThreads) out[i] = i < n ? i : -1;
        return;
    }
    const int p0 = blockIdx.x * kBlockPages;
    if (p0 >= n) return;
    // this lane's page, its record and exponent
    const int page = p0 + warp * 32 + lane;
    int rec = 0, e_page = 0;
    if (page < n) {
        rec = a.table.page(b, page);
        e_page = a.exps[(int64_t)rec * a.Hk + h];
    }

    float top = 0.f;
    for (int i = threadIdx.x; i < G * D; i += kThreads)
        top = fmaxf(top, fabsf(load_as_f32(a.q, q0 + (i / D) * a.q_sh + i % D, a.dtype)));
    for (int o = 16; o; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) wmax[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; w++) top = fmaxf(top, wmax[w]);
    const int e = bound_exponent(fminf(top, 3e38f), -100) + a.shift;
    for (int d = threadIdx.x; d < 8 * GRP; d += kThreads) {
        int neg = 0, pos = 0;
        if (d < D)
            for (int g = 0; g < G; g++) {
                const float x = load_as_f32(a.q, q0 + g * a.q_sh + d, a.dtype);
                const int v = (int)fminf(fmaxf(rintf(ldexpf(x, -e)), -127.f), 127.f);
                neg += min(v, 0);
                pos += max(v, 0);
            }
        if (d < D) {
            z[d] = (short)neg;
            z[D + d] = (short)pos;
        }
    }
    __syncthreads();
    const int li = lane % GRP, grp = lane / GRP;
    const bool live = li < 4 * W;
    int zr[8];
#pragma unroll
    for (int i = 0; i < 8; i++) zr[i] = live ? reinterpret_cast<const int *>(z)[li * 8 + i] : 0;
    int mine = 0;
    if (p0 + warp * 32 < n) {
        constexpr int AHEAD = 8;  // loads on their way at a time
#pragma unroll 1
        for (int i0 = 0; i0 < GRP; i0 += AHEAD) {  // PPW pages at a time, one a group
            int4 v[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int id = __shfl_sync(0xffffffffu, rec, (i0 + i) * PPW + grp);
                v[i] = make_int4(0, 0, 0, 0);
                if (live)
                    v[i] = __ldg(reinterpret_cast<const int4 *>(a.bounds + ((int64_t)id * a.Hk + h) * 2 * D) + li);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                int sum = 0;
                const int w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    sum = __dp2a_lo(zr[2 * j], w[j], sum);
                    sum = __dp2a_hi(zr[2 * j + 1], w[j], sum);
                }
#pragma unroll
                for (int o = GRP / 2; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                const int s = __shfl_sync(0xffffffffu, sum, (lane % PPW) * GRP);
                if (lane / PPW == i0 + i) mine = s;
            }
        }
    }
    uint32_t *keys = a.keys + (b * a.Hk + h) * a.table.max_pages;
    if (page < n) keys[page] = order_key((float)mine * pow2f(e_page));
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        int *counter = a.counters + b * a.Hk + h;
        const int blocks = (n + kBlockPages - 1) / kBlockPages;
        last_s = atomicAdd(counter, 1) == blocks - 1;
        if (last_s) *counter = 0;
        __threadfence();
    }
    __syncthreads();
    if (last_s) pick(a, keys, n, out, pick_s);
}

}  // namespace
}  // namespace kv4
}  // namespace fc

using namespace fc;
using namespace fc::kv4;

extern "C" size_t fc_kv4_select_workspace_size(int64_t B, int64_t Hk, int64_t max_pages) {
    return (size_t)(kCounterBytes + B * Hk * max_pages * 4);
}

extern "C" int fc_kv4_select(const void *q, int dtype, int64_t B, int64_t Hq, int64_t q_sb, int64_t q_sh,
                             const signed char *bounds, const int *exponents, int64_t num_pages,
                             int64_t Hk, int64_t D, int64_t page_size, const int *page_table,
                             int64_t table_stride, int64_t max_pages, const int *lengths, int64_t count,
                             int64_t sink, int64_t recent, int *pages, void *workspace,
                             size_t workspace_bytes, int *status, void *stream) {
    clear_error();
    int rc = check_cache("kv4_select", B, Hk, D, page_size, num_pages, max_pages, bounds, page_table, status);
    if (rc) return rc;
    if (!is_float_dtype(dtype)) { set_error("kv4_select: dtype must be fp32, bf16 or fp16"); return FC_EINVAL; }
    if (Hq <= 0 || Hq % Hk || Hq / Hk > 256) {
        set_error("kv4_select: query heads (%lld) must be a multiple (at most 256) of kv heads (%lld)",
                  (long long)Hq, (long long)Hk);
        return FC_EINVAL;
    }
    if (count <= 0 || sink < 0 || recent < 0 || sink + recent > count || count > 0x7fffffff) {
        set_error("kv4_select: count must be positive and hold the sink and recent pages");
        return FC_EINVAL;
    }
    if (B == 0) return FC_OK;
    if (B > 65535 || B * Hk > kMaxUnits) {
        set_error("kv4_select: more than 65535 sequences, or 2^18 of them and KV heads");
        return FC_ENOTSUP;
    }
    if (!q || !exponents || !lengths || !pages || !workspace || !aligned(workspace, 16)) {
        set_error("kv4_select: null pointer or misaligned workspace");
        return FC_EINVAL;
    }
    if (workspace_bytes < fc_kv4_select_workspace_size(B, Hk, max_pages)) {
        set_error("kv4_select: workspace of %zu bytes is too small", workspace_bytes);
        return FC_ERANGE;
    }
    SelectArgs a{q, dtype, q_sb, q_sh, (int)Hq, (int)Hk, bounds, exponents,
                 Table{page_table, table_stride, (int)max_pages, (int)num_pages, ilog2(page_size), status},
                 lengths, (int)count, (int)sink, (int)recent, pages,
                 reinterpret_cast<int *>(static_cast<char *>(workspace) + 256),
                 reinterpret_cast<uint32_t *>(static_cast<char *>(workspace) + kCounterBytes),
                 Hq / Hk * D > 1024 ? ilog2((Hq / Hk * D + 1023) / 1024) : 0};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_head_dim(D, [&](auto w) {
        select_kernel<decltype(w)::value><<<dim3((unsigned)((max_pages + kBlockPages - 1) / kBlockPages),
                                                 (unsigned)Hk, (unsigned)B), kThreads, 0, st>>>(a);
        return check_launch("kv4_select");
    });
}
