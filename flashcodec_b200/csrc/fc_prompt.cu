// Attention over whole prompts: packed sequences of different lengths, grouped heads, causal.
//
//   out = softmax(scale * q . K^T + mask) . V
//
// Query i of a sequence of n_q queries and n_k keys is at position n_k - n_q + i and sees the
// keys up to it (all of them where not causal).
#include "fc_attn_common.cuh"
#include "fc_kv4.cuh"

namespace fc {
namespace prompt {
namespace {

using kv4::Rows;
using kv4::rows_meet;
using kv4::rows_repeat;
using kv4::same_rows;
using kv4::warp_find;

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
    const void *q, *k, *v;
    void *out;
    float *lse;
    int64_t q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, o_sb, o_ss, o_sh;
    int64_t Sq, Sk, Tq, Tk;
    int B, Hq, Hk, G, causal;
    const int *cu_q, *cu_k;
    float scale;  // softmax_scale * log2(e)
};

// One warp a query and head.
template <typename T, int W>
__global__ void __launch_bounds__(256) prompt_simple_kernel(const __grid_constant__ Args a) {
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), t = unit / a.Hq;
    if (t >= a.Tq) return;
    const int lane = threadIdx.x & 31, h = (int)(unit - t * a.Hq), hk = h / a.G;
    int64_t k0 = 0, n = 0, b = 0, i = t;
    if (!a.cu_q) {
        b = t / a.Sq;
        i = t - b * a.Sq;
        n = a.Sk;
        if (a.causal) n = max(n - a.Sq + i + 1, (int64_t)0);
    } else if (a.B) {
        const int *cu = a.cu_q;
        const int w = warp_find([=](int j) { return (int64_t)cu[j]; }, a.B, t);
        if (t >= cu[w] && t < cu[w + 1]) {
            k0 = max(a.cu_k[w], 0);
            n = max(min((int64_t)a.cu_k[w + 1], a.Tk) - k0, (int64_t)0);
            if (a.causal) n = max(n - (min((int64_t)cu[w + 1], a.Tq) - 1 - t), (int64_t)0);
        }
    }
    const T *q = static_cast<const T *>(a.q) + b * a.q_sb + i * a.q_ss + h * a.q_sh;
    float x[W], o[W], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < W; w++) {
        x[w] = Elem<T>::to_f32(q[lane + 32 * w]) * a.scale;
        o[w] = 0.f;
    }
    for (int64_t j = k0; j < k0 + n; j++) {
        const T *k = static_cast<const T *>(a.k) + b * a.k_sb + j * a.k_ss + hk * a.k_sh;
        const T *v = static_cast<const T *>(a.v) + b * a.v_sb + j * a.v_ss + hk * a.v_sh;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < W; i++) s = fmaf(x[i], Elem<T>::to_f32(k[lane + 32 * i]), s);
#pragma unroll
        for (int d = 1; d < 32; d *= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        const float top = fmaxf(m, s), ref = top == -INFINITY ? 0.f : top;
        const float f = exp2f(m - ref), p = exp2f(s - ref);
        m = top;
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < W; i++) o[i] = fmaf(o[i], f, p * Elem<T>::to_f32(v[lane + 32 * i]));
    }
    T *out = static_cast<T *>(a.out) + b * a.o_sb + i * a.o_ss + h * a.o_sh;
#pragma unroll
    for (int i = 0; i < W; i++) store_from_f32(out, lane + 32 * i, Elem<T>::code, l == 0.f ? 0.f : o[i] / l);
    if (a.lse && lane == 0) a.lse[t * a.Hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
}

}  // namespace
}  // namespace prompt
}  // namespace fc

using namespace fc;
using namespace fc::prompt;

extern "C" size_t fc_prompt_attn_workspace_size(int64_t B, int64_t Tq, int64_t Hq, int64_t Hk, int64_t D) {
    return kWsHeader + kWsUnits * 4;
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
    Args a{};
    a.q = q; a.k = k; a.v = v; a.out = out; a.lse = lse;
    a.q_sb = q_sb; a.q_ss = q_ss; a.q_sh = q_sh;
    a.k_sb = k_sb; a.k_ss = k_ss; a.k_sh = k_sh;
    a.v_sb = v_sb; a.v_ss = v_ss; a.v_sh = v_sh;
    a.o_sb = o_sb; a.o_ss = o_ss; a.o_sh = o_sh;
    a.Sq = Sq; a.Sk = Sk; a.Tq = Tq; a.Tk = Tk; a.B = (int)B; a.Hq = (int)Hq; a.Hk = (int)Hk; a.G = (int)(Hq / Hk); a.causal = causal;
    a.cu_q = cu_seqlens_q; a.cu_k = cu_seqlens_k;
    a.scale = softmax_scale * 1.44269504088896341f;
    const int64_t blocks = (Tq * Hq + 7) / 8;
    if (blocks > 0x7fffffff) { set_error("prompt_attn: too many rows"); return FC_ENOTSUP; }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return kv4::by_head_dim(D, [&](auto w) {
        constexpr int W = decltype(w)::value;
        if (dtype == FC_BF16) prompt_simple_kernel<__nv_bfloat16, W><<<(unsigned)blocks, 256, 0, st>>>(a);
        else prompt_simple_kernel<__half, W><<<(unsigned)blocks, 256, 0, st>>>(a);
        return check_launch("prompt_attn");
    });
}
