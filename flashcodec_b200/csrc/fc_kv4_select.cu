// Paged 4-bit KV cache: the pages of each sequence and KV head worth attending to.
//
// A page's bounds give an upper bound of q . k over its keys: the sum over channels
// of max(q * least, q * largest).  Summed over the heads of a group this is linear
// in the positive and the negative parts of the queries, so a page costs one dot
// product of 2 D bytes with two vectors, P = sum_heads max(z, 0) and N = sum_heads
// min(z, 0), whatever the number of heads:
//     score = (P . largest + N . least) * 2^exponent
// z is the query in whole numbers (|z| <= 127, common power of two of the group),
// so the sums are exact (below 2^24, also as fp32) and the choice of pages does not
// depend on the order of any sum.
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
    uint32_t *keys;  // (B, Hk, max_pages)
    int shift;       // ceil(log2(G * D / 1024)) where positive
};

constexpr int kScoreThreads = 256;
constexpr int kScorePages = 128;  // pages of a scoring block

// Order-preserving map of finite fp32 to unsigned.
__device__ __forceinline__ uint32_t order_key(float f) {
    const uint32_t u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int W>
__global__ void __launch_bounds__(kScoreThreads) score_kernel(const __grid_constant__ SelectArgs a) {
    constexpr int D = 32 * W;
    __shared__ short z[2 * D];  // N then P, as the bounds: least then largest
    __shared__ float wmax[kScoreThreads / 32];
    const int h = blockIdx.y;
    const int64_t b = blockIdx.z;
    const int len = a.table.length(a.lengths[b]);
    const int n = (len + (1 << a.table.log_page) - 1) >> a.table.log_page;
    const int p0 = blockIdx.x * kScorePages;
    if (p0 >= n || n <= a.count) return;  // everything is taken: no scores needed
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.Hq / a.Hk;
    const int64_t q0 = b * a.q_sb + (int64_t)h * G * a.q_sh;
    float top = 0.f;
    for (int i = threadIdx.x; i < G * D; i += kScoreThreads)
        top = fmaxf(top, fabsf(load_as_f32(a.q, q0 + (i / D) * a.q_sh + i % D, a.dtype)));
    for (int o = 16; o; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) wmax[warp] = top;
    __syncthreads();
    for (int w = 0; w < kScoreThreads / 32; w++) top = fmaxf(top, wmax[w]);
    const int e = bound_exponent(fminf(top, 3e38f), -100) + a.shift;
    for (int d = threadIdx.x; d < D; d += kScoreThreads) {
        int neg = 0, pos = 0;
        for (int g = 0; g < G; g++) {
            const float x = load_as_f32(a.q, q0 + g * a.q_sh + d, a.dtype);
            const int v = (int)fminf(fmaxf(rintf(ldexpf(x, -e)), -127.f), 127.f);
            neg += min(v, 0);
            pos += max(v, 0);
        }
        z[d] = (short)neg;
        z[D + d] = (short)pos;
    }
    __syncthreads();
    const int p1 = min(p0 + kScorePages, n);
    for (int p = p0 + warp; p < p1; p += kScoreThreads / 32) {
        const int64_t rec = (int64_t)a.table.page(b, p) * a.Hk + h;
        int sum = 0;
        for (int d = lane; d < 2 * D; d += 32) sum += (int)a.bounds[rec * 2 * D + d] * z[d];
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0) {
            uint32_t k = order_key((float)sum * pow2f(a.exps[rec]));
            if (p < a.sink || p >= n - a.recent) k = 0xffffffffu;
            a.keys[(b * a.Hk + h) * a.table.max_pages + p] = k;
        }
    }
}

constexpr int kPickThreads = 1024;

// The `count` largest keys, equal ones by index, in ascending order of index.
__global__ void __launch_bounds__(kPickThreads) pick_kernel(const __grid_constant__ SelectArgs a) {
    __shared__ uint32_t hist[256], want_s, rest_s, base[2], sums[2][kPickThreads / 32];
    const int h = blockIdx.x;
    const int64_t b = blockIdx.y;
    const int len = a.table.length(a.lengths[b]);
    const int n = (len + (1 << a.table.log_page) - 1) >> a.table.log_page;
    int *out = a.out + (b * a.Hk + h) * a.count;
    if (n <= a.count) {
        for (int i = threadIdx.x; i < a.count; i += kPickThreads) out[i] = i < n ? i : -1;
        return;
    }
    const uint32_t *keys = a.keys + (b * a.Hk + h) * a.table.max_pages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t prefix = 0, rest = (uint32_t)a.count;  // of keys with this prefix, `rest` are wanted
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kPickThreads) hist[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kPickThreads) {
            const uint32_t k = keys[i];
            if (shift == 24 || k >> (shift + 8) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int i = 255;
            uint32_t left = rest;
            while (hist[i] < left) left -= hist[i--];
            want_s = (uint32_t)i;
            rest_s = left;
        }
        __syncthreads();
        prefix = prefix << 8 | want_s;
        rest = rest_s;
        __syncthreads();
    }
    // prefix is the smallest key taken, `rest` of its equals are
    if (threadIdx.x < 2) base[threadIdx.x] = 0;
    __syncthreads();
    for (int i0 = 0; i0 < n; i0 += kPickThreads) {
        const int i = i0 + threadIdx.x;
        const uint32_t k = i < n ? keys[i] : 0u;
        const bool over = i < n && k > prefix, same = i < n && k == prefix;
        const uint32_t below = (1u << lane) - 1;
        const uint32_t mo = __ballot_sync(0xffffffffu, over), ms = __ballot_sync(0xffffffffu, same);
        if (lane == 0) { sums[0][warp] = __popc(mo); sums[1][warp] = __popc(ms); }
        __syncthreads();
        uint32_t no = base[0], ns = base[1];
        for (int w = 0; w < warp; w++) { no += sums[0][w]; ns += sums[1][w]; }
        no += __popc(mo & below);
        ns += __popc(ms & below);
        if (over || (same && ns < rest)) out[no + min(ns, rest)] = i;
        __syncthreads();
        if (threadIdx.x == 0)
            for (int w = 0; w < kPickThreads / 32; w++) { base[0] += sums[0][w]; base[1] += sums[1][w]; }
        __syncthreads();
    }
}

}  // namespace
}  // namespace kv4
}  // namespace fc

using namespace fc;
using namespace fc::kv4;

extern "C" size_t fc_kv4_select_workspace_size(int64_t B, int64_t Hk, int64_t max_pages) {
    return 256 + (size_t)B * Hk * max_pages * sizeof(uint32_t);
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
    if (B > 65535) { set_error("kv4_select: more than 65535 sequences"); return FC_ENOTSUP; }
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
                 reinterpret_cast<uint32_t *>(static_cast<char *>(workspace) + 256),
                 Hq / Hk * D > 1024 ? ilog2((Hq / Hk * D + 1023) / 1024) : 0};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_head_dim(D, [&](auto w) {
        score_kernel<decltype(w)::value><<<dim3((unsigned)((max_pages + kScorePages - 1) / kScorePages),
                                                (unsigned)Hk, (unsigned)B), kScoreThreads, 0, st>>>(a);
        int e = check_launch("kv4_select");
        if (e) return e;
        pick_kernel<<<dim3((unsigned)Hk, (unsigned)B), kPickThreads, 0, st>>>(a);
        return check_launch("kv4_select");
    });
}
