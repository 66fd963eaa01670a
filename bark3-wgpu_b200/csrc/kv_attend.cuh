// kv_attend.cuh — what the attention kernels over the paged 8-bit cache share.
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j),
//   k_j = kc_j 2^ke, v_j = vc_j 2^ve with e4m3 codes kc, vc and the exponents
//   of j's page.
//
// The tensor cores multiply the codes themselves: e4m3 -> f16 is exact, and a
// query row is exact in f16 too (bf16 rows are moved by a power of two, see
// row_shift).  Scores are kept in log2 units,
//   x_ij = (scale log2(e) 2^ke) (q_i . kc_j),   x'_ij = x_ij + ve,
// and the running maximum m is taken of x', so the probabilities that the
// second product multiplies by codes already carry the value's scale:
//   p'_ij = 2^(x'_ij - m) <= 1  (f16 for the product),   o = sum p' vc / l,
//   l = sum p' 2^-ve = sum 2^(x_ij - m).
// With ve in [-40, 40] a p' that underflows f32 has a share below 2^-46 of l.
#pragma once
#include "kv_cache.cuh"

namespace b3 {

struct AttendParams {
    b3_kv_cache c;
    b3_kv_batch b;
    b3_kv_attend_args a;
};

__device__ __forceinline__ float ex2_approx(float x) {   // relative error below 2^-22; 0 below 2^-126
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// The power of two that brings a bf16 row of largest magnitude amax into
// [2^14, 2^15): channels down to 2^-28 of the largest keep their 8 bits in
// f16, smaller ones lose what is 2^-39 of the largest.
__device__ __forceinline__ int row_shift(float amax) {
    const int e = static_cast<int>(__float_as_uint(amax) >> 23) - 127;
    return amax > 0.f && e < 128 ? min(14 - e, 100) : 0;
}

// A sequence's part in an attention call: its first query row, new tokens and
// cached length; lengths that do not fit leave it empty (and are flagged).
struct SeqSpan {
    int first, n, len;
};
__device__ __forceinline__ SeqSpan attend_span(const AttendParams& p, int s) {
    SeqSpan r;
    r.first = __ldg(p.b.cu_q + s);
    r.n = __ldg(p.b.cu_q + s + 1) - r.first;
    r.len = __ldg(p.b.kv_lens + s);
    if (r.first < 0 || r.n < 0 || r.n > p.b.tokens - r.first || r.n > p.a.max_q) {
        kv_flag(p.c.status, B3_KV_BAD_LENGTH);
        r.n = 0;
    }
    if (r.len < 0 || r.len > p.b.table_width * p.c.page_tokens) {
        kv_flag(p.c.status, B3_KV_BAD_LENGTH);
        r.len = 0;
    }
    return r;
}

// The keys [lo, hi) that new token i of a sequence sees.
__device__ __forceinline__ void seen_keys(const AttendParams& p, const SeqSpan& s, int i, int& lo, int& hi) {
    lo = 0;
    hi = s.len;
    if (p.a.causal) {
        const int pos = s.len - s.n + i;
        hi = max(pos + 1, 0);
        if (p.a.window > 0) lo = max(0, pos + 1 - p.a.window);
    }
}

// One query row by one warp in plain arithmetic, a key at a time: the keys of
// [k0, k1) that the row sees, m in the units above, o and l against it, o in
// DIM / 32 channels a lane.  A masked key does not touch the row, whatever it
// holds; in the tensor cores' sums 0 * NaN of a value that other rows see is
// NaN, so rows whose output came out NaN are taken again by this.
template <typename T, int DIM>
__device__ __noinline__ void attend_row_exact(const AttendParams& p, int seq, int token, int i, int q_head, int k0, int k1,
                                              float (&o)[DIM / 32], float& m, float& l) {
    constexpr int kPer = DIM / 32;
    const int lane = threadIdx.x & 31, page = p.c.page_tokens, kv_head = q_head / (p.a.q_heads / p.c.kv_heads);
    const SeqSpan sp = attend_span(p, seq);
    int lo, hi;
    seen_keys(p, sp, i, lo, hi);
    const T* q = static_cast<const T*>(p.a.q) + token * p.a.q_token_stride + q_head * p.a.q_head_stride + lane * kPer;
    float x[kPer];
    for (int c = 0; c < kPer; ++c) {
        x[c] = to_f32(q[c]) * (p.a.scale * kLog2e);
        o[c] = 0.f;
    }
    m = -INFINITY;
    l = 0.f;
    for (int j = max(lo, k0); j < min(hi, k1); ++j) {
        int id = __ldg(p.b.page_table + seq * p.b.table_stride + j / page);
        if (id < 0 || id >= p.c.pages) id = 0;   // flagged where it was met first
        const int64_t slab = static_cast<int64_t>(id) * p.c.kv_heads + kv_head;
        const int64_t at = (slab * page + j % page) * DIM + lane * kPer;
        float dot = 0.f;
        for (int c = 0; c < kPer; c += 2) {
            const float2 k = __half22float2(decode2(*reinterpret_cast<const uint16_t*>(p.c.k + at + c)));
            dot = fmaf(x[c], k.x, fmaf(x[c + 1], k.y, dot));
        }
        for (int w = 16; w; w >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, w);
        const int ve = stored_exp(p.c.v_scale[slab]);
        dot = fmaf(dot, p.c.k_scale[slab], static_cast<float>(ve));
        const float top = fmaxf(m, dot), ref = top == -INFINITY ? 0.f : top;
        const float old = m == top ? 1.f : ex2_approx(m - top), e = ex2_approx(dot - ref);
        l = fmaf(e, exp2_int(-ve), l * old);
        for (int c = 0; c < kPer; c += 2) {
            const float2 v = __half22float2(decode2(*reinterpret_cast<const uint16_t*>(p.c.v + at + c)));
            o[c] = fmaf(e, v.x, o[c] * old);
            o[c + 1] = fmaf(e, v.y, o[c + 1] * old);
        }
        m = top;
    }
}

// The float of a finished row: o / l, zeros where nothing was seen.
__device__ __forceinline__ float row_inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float row_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2; }

// kv_attend_rows.cu: at most 16 query rows (new tokens x heads of a group) a key head.
int64_t attend_rows_workspace(const AttendParams& p);
int launch_attend_rows(const AttendParams& p, void* workspace, cudaStream_t st);
// kv_attend_tiles.cu: any number of query rows, in tiles of 256.
int64_t attend_tiles_workspace(const AttendParams& p);
int launch_attend_tiles(const AttendParams& p, void* workspace, cudaStream_t st);

}  // namespace b3
