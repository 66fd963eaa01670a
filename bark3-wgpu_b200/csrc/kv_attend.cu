// kv_attend.cu — b3_kv_attend: attention over the paged 8-bit cache.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j - m_i)
// with k_j = code * 2^e of the page, in one pass over the keys with a running
// maximum m and sum.  One warp for each (token, query head).
#include "kv_attend.cuh"

namespace b3 {
namespace {

constexpr int kThreads = 128;

template <typename T, int DIM>
__global__ void __launch_bounds__(kThreads) k_kv_attend_row(const __grid_constant__ AttendParams p) {
    constexpr int kPer = DIM / 32;
    const int lane = threadIdx.x & 31;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
    if (id >= static_cast<int64_t>(p.b.tokens) * p.a.q_heads) return;
    const int token = static_cast<int>(id / p.a.q_heads), head = static_cast<int>(id % p.a.q_heads);
    const int kv_head = head / (p.a.q_heads / p.c.kv_heads), page = p.c.page_tokens;
    const int s = kv_seq_of(p.b, token);
    const int first = __ldg(p.b.cu_q + s), n = __ldg(p.b.cu_q + s + 1) - first, len = __ldg(p.b.kv_lens + s);
    if (len < 0 || len > static_cast<int64_t>(p.b.table_width) * page) {
        kv_flag(p.c.status, B3_KV_BAD_LENGTH);
        return;
    }
    if (n > p.a.max_q) kv_flag(p.c.status, B3_KV_BAD_LENGTH);
    int hi = len, lo = 0;   // the keys this token sees
    if (p.a.causal) {
        const int pos = len - n + token - first;
        hi = min(len, max(pos + 1, 0));
        if (p.a.window > 0) lo = max(0, pos + 1 - p.a.window);
    }
    const T* q = static_cast<const T*>(p.a.q) + token * p.a.q_token_stride + head * p.a.q_head_stride + lane * kPer;
    float x[kPer], o[kPer], m = -INFINITY, l = 0.f;
    for (int i = 0; i < kPer; ++i) {
        x[i] = to_f32(q[i]) * p.a.scale;
        o[i] = 0.f;
    }
    for (int j = lo; j < hi; ++j) {
        const int to = __ldg(p.b.page_table + s * p.b.table_stride + j / page);
        if (to < 0 || to >= p.c.pages) {
            kv_flag(p.c.status, B3_KV_BAD_PAGE);
            continue;
        }
        const int64_t slab = static_cast<int64_t>(to) * p.c.kv_heads + kv_head;
        const int64_t at = (slab * page + j % page) * DIM + lane * kPer;
        float dot = 0.f;
        for (int i = 0; i < kPer; i += 2) {
            const float2 k = __half22float2(decode2(*reinterpret_cast<const uint16_t*>(p.c.k + at + i)));
            dot = fmaf(x[i], k.x, fmaf(x[i + 1], k.y, dot));
        }
        for (int w = 16; w; w >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, w);
        dot *= p.c.k_scale[slab];
        const float top = fmaxf(m, dot), old = m == top ? 1.f : expf(m - top), e = dot == top ? 1.f : expf(dot - top);
        l = l * old + e;
        const float ev = e * p.c.v_scale[slab];
        for (int i = 0; i < kPer; i += 2) {
            const float2 v = __half22float2(decode2(*reinterpret_cast<const uint16_t*>(p.c.v + at + i)));
            o[i] = fmaf(ev, v.x, o[i] * old);
            o[i + 1] = fmaf(ev, v.y, o[i + 1] * old);
        }
        m = top;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    T* out = static_cast<T*>(p.a.out) + (static_cast<int64_t>(token) * p.a.q_heads + head) * DIM + lane * kPer;
    for (int i = 0; i < kPer; ++i) from_f32(o[i] * inv, out[i]);
    if (p.a.lse && lane == 0) p.a.lse[id] = hi > lo ? m + logf(l) : -INFINITY;
}

int check(const b3_kv_cache* cache, const b3_kv_batch* batch, const b3_kv_attend_args* args) {
    if (int rc = kv_check(cache, batch)) return rc;
    if (!args) return set_error(B3_EINVAL, "null arguments");
    const b3_kv_attend_args& a = *args;
    if (a.dtype != B3_DTYPE_F16 && a.dtype != B3_DTYPE_BF16) return set_error(B3_EINVAL, "dtype %d (f16 or bf16)", a.dtype);
    if (a.q_heads <= 0 || a.q_heads % cache->kv_heads)
        return set_error(B3_EINVAL, "q_heads %d is no multiple of kv_heads %d", a.q_heads, cache->kv_heads);
    if (a.max_q <= 0) return set_error(B3_EINVAL, "max_q %d", a.max_q);
    if (a.window < 0 || (a.window && !a.causal)) return set_error(B3_EINVAL, "window %d (needs causal)", a.window);
    return 0;
}

template <typename T>
int launch(const AttendParams& p, cudaStream_t st) {
    const int64_t blocks = (static_cast<int64_t>(p.b.tokens) * p.a.q_heads + 3) / 4;
    if (blocks > 0x7fffffffll) return set_error(B3_EINVAL, "b3_kv_attend: too many tokens for one call");
    if (p.c.head_dim == 128)
        k_kv_attend_row<T, 128><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(p);
    else
        k_kv_attend_row<T, 64><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : set_cuda_error("k_kv_attend_row", e);
}

}  // namespace
}  // namespace b3

using namespace b3;

static bool few_rows(const b3_kv_cache& c, const b3_kv_attend_args& a) {
    return static_cast<int64_t>(a.max_q) * (a.q_heads / c.kv_heads) <= 16;
}

extern "C" int64_t b3_kv_attend_workspace(const b3_kv_cache* cache, const b3_kv_batch* batch,
                                          const b3_kv_attend_args* args) {
    if (int rc = check(cache, batch, args)) return rc;
    const AttendParams p{*cache, *batch, *args};
    return few_rows(*cache, *args) ? attend_rows_workspace(p) : 0;
}

extern "C" int b3_kv_attend(const b3_kv_cache* cache, const b3_kv_batch* batch, const b3_kv_attend_args* args,
                            void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = check(cache, batch, args)) return rc;
    if (batch->tokens == 0) return 0;
    if (!args->q || !args->out) return set_error(B3_EINVAL, "null q or out");
    if (reinterpret_cast<uintptr_t>(args->out) & 15) return set_error(B3_EINVAL, "out must be 16-byte aligned");
    const AttendParams p{*cache, *batch, *args};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (few_rows(*cache, *args)) {
        const int64_t need = attend_rows_workspace(p);
        if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15))
            return set_error(B3_EINVAL, "workspace of %lld bytes, 16-byte aligned, is needed (got %lld)",
                             static_cast<long long>(need), static_cast<long long>(workspace_bytes));
        return launch_attend_rows(p, workspace, st);
    }
    return args->dtype == B3_DTYPE_F16 ? launch<__half>(p, st) : launch<__nv_bfloat16>(p, st);
}
