// Paged 4-bit KV cache: attention of one or a few new tokens.
//
//   out = softmax(scale * q . K^T) . V,  K = code * scale per group of 32 channels
//
// One block for a query row and KV head; its warps take the tiles of 16 tokens in
// turn, a lane scores one token, and every warp keeps a running maximum, sum and
// output (fp32) that are joined at the end.
#include "fc_kv4.cuh"

namespace fc {
namespace kv4 {
namespace {

struct AttnArgs {
    const void *q;
    int64_t q_sb, q_ss, q_sh;
    int Sq, Hq, Hk, dtype;
    const unsigned char *pool;
    Table table;
    const int *lengths, *selected;
    int n_selected;
    float scale;
    void *out;
    int64_t o_sb, o_ss, o_sh;
    float *lse;
};

constexpr int kThreads = 128;

template <int W>
__global__ void __launch_bounds__(kThreads) attn_kernel_simple(const __grid_constant__ AttnArgs a) {
    constexpr int D = 32 * W, WARPS = kThreads / 32;
    __shared__ float qs[D], part[WARPS][D], mx[WARPS], sm[WARPS];
    const int G = a.Hq / a.Hk;
    const int h = blockIdx.x / G, g = blockIdx.x % G, s = blockIdx.y;
    const int64_t b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int P = 1 << a.table.log_page, tpp = P / 16;
    const int64_t qoff = b * a.q_sb + s * a.q_ss + (int64_t)(h * G + g) * a.q_sh;
    for (int d = threadIdx.x; d < D; d += kThreads) qs[d] = load_as_f32(a.q, qoff + d, a.dtype) * a.scale;
    __syncthreads();
    const int len = a.table.length(a.lengths[b]);
    const int seen = len - (a.Sq - 1 - s);
    const int pages = (len + P - 1) >> a.table.log_page;
    const int tiles = a.selected ? a.n_selected * tpp : (max(seen, 0) + 15) / 16;
    float m = -INFINITY, sum = 0.f, acc[2 * W][2];
#pragma unroll
    for (int i = 0; i < 2 * W; i++) acc[i][0] = acc[i][1] = 0.f;
    for (int i = warp; i < tiles; i += WARPS) {
        int page = i / tpp;
        if (a.selected) {
            page = a.selected[(b * a.Hk + h) * a.n_selected + page];
            if (page < 0 || page >= pages) continue;
        }
        const int tile = i % tpp;
        const int pos = page * P + tile * 16 + (lane & 15);
        const unsigned char *in =
            a.pool + (((int64_t)a.table.page(b, page) * a.Hk + h) * tpp + tile) * tile_bytes(W);
        const int t = lane & 15;
        float x = 0.f;
        const uint32_t *kw = reinterpret_cast<const uint32_t *>(in) + t * 4 * W;
        const __half *ks = reinterpret_cast<const __half *>(in + ks_off(W)) + (2 * (t & 7) + (t >> 3)) * W;
        for (int j = 0; j < W; j++) {
            float y = 0.f;
            for (int cc = 0; cc < 4; cc++) {
                const uint32_t w = kw[cc * W + j];
                for (int e = 0; e < 8; e++)
                    y += (float)((int)((w >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u) - 8) * qs[32 * j + 8 * cc + e];
            }
            x += y * __half2float(ks[j]);
        }
        if (pos >= seen) x = -INFINITY;
        float top = x;
        for (int o = 8; o; o /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        top = fmaxf(top, m);
        if (top == -INFINITY) continue;
        const float f = __expf(m - top);
        const float p = expf(x - top);
        float ps = p;
        for (int o = 8; o; o /= 2) ps += __shfl_xor_sync(0xffffffffu, ps, o);
        sum = sum * f + ps;
        m = top;
        const uint32_t *vw = reinterpret_cast<const uint32_t *>(in + v_off(W));
        const __half *vs = reinterpret_cast<const __half *>(in + vs_off(W));
        for (int mt = 0; mt < 2 * W; mt++) {
            const uint32_t w = vw[v_word<W>(mt, lane)];
            acc[mt][0] *= f;
            acc[mt][1] *= f;
            for (int u = 0; u < 4; u++) {
                const int tok = 2 * c + 8 * (u >> 1) + (u & 1);
                const float pt = __shfl_sync(0xffffffffu, p, tok);
                if (pt == 0.f) continue;
                const float sc = pt * __half2float(vs[4 * (c * W + mt / 2) + u]);
                const int sh = 4 * (2 * (u >> 1) + 4 * (u & 1));
                acc[mt][0] += sc * (float)((int)((w >> sh) & 15u) - 8);
                acc[mt][1] += sc * (float)((int)((w >> (sh + 4)) & 15u) - 8);
            }
        }
    }
    for (int mt = 0; mt < 2 * W; mt++)
        for (int x = 0; x < 2; x++) {
            float v = acc[mt][x];
            v += __shfl_xor_sync(0xffffffffu, v, 1);
            v += __shfl_xor_sync(0xffffffffu, v, 2);
            if (c == 0) part[warp][16 * mt + r + 8 * x] = v;
        }
    if (lane == 0) { mx[warp] = m; sm[warp] = sum; }
    __syncthreads();
    float top = -INFINITY, all = 0.f;
    for (int w = 0; w < WARPS; w++) top = fmaxf(top, mx[w]);
    for (int w = 0; w < WARPS; w++) all += top == -INFINITY ? 0.f : sm[w] * expf(mx[w] - top);
    for (int d = threadIdx.x; d < D; d += kThreads) {
        float o = 0.f;
        for (int w = 0; w < WARPS; w++) o += top == -INFINITY ? 0.f : part[w][d] * expf(mx[w] - top);
        store_from_f32(a.out, b * a.o_sb + s * a.o_ss + (int64_t)(h * G + g) * a.o_sh + d, a.dtype,
                       top == -INFINITY ? 0.f : o / all);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[(b * a.Sq + s) * a.Hq + h * G + g] = top == -INFINITY ? -INFINITY : top + logf(all);
}

}  // namespace
}  // namespace kv4
}  // namespace fc

using namespace fc;
using namespace fc::kv4;

extern "C" size_t fc_kv4_attn_workspace_size(int64_t B, int64_t Sq, int64_t Hq, int64_t Hk, int64_t D) {
    return 256;
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
    if (Sq < 0 || Sq > 65535) { set_error("kv4_attn: bad query count"); return FC_EINVAL; }
    if (B == 0 || Sq == 0) return FC_OK;
    if (!q || !out || !lengths) { set_error("kv4_attn: null pointer"); return FC_EINVAL; }
    if (selected && (Sq != 1 || n_selected < 0)) {
        set_error("kv4_attn: selected pages go with one query per sequence");
        return FC_EINVAL;
    }
    if (!workspace || !aligned(workspace, 16)) { set_error("kv4_attn: null or misaligned workspace"); return FC_EINVAL; }
    if (workspace_bytes < fc_kv4_attn_workspace_size(B, Sq, Hq, Hk, D)) {
        set_error("kv4_attn: workspace of %zu bytes is too small", workspace_bytes);
        return FC_ERANGE;
    }
    if (B > 65535) { set_error("kv4_attn: more than 65535 sequences"); return FC_ENOTSUP; }
    AttnArgs a{q, q_sb, q_ss, q_sh, (int)Sq, (int)Hq, (int)Hk, dtype,
               static_cast<const unsigned char *>(pool),
               Table{page_table, table_stride, (int)max_pages, (int)num_pages, ilog2(page_size), status},
               lengths, selected, (int)n_selected, softmax_scale, out, o_sb, o_ss, o_sh, lse};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_head_dim(D, [&](auto w) {
        attn_kernel_simple<decltype(w)::value><<<dim3((unsigned)Hq, (unsigned)Sq, (unsigned)B), kThreads, 0, st>>>(a);
        return check_launch("kv4_attn");
    });
}
