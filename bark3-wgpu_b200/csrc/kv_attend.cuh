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

// kv_attend_rows.cu: at most 16 query rows (new tokens x heads of a group) a key head.
int64_t attend_rows_workspace(const AttendParams& p);
int launch_attend_rows(const AttendParams& p, void* workspace, cudaStream_t st);

}  // namespace b3
