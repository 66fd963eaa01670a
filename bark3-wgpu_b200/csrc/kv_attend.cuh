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
//
// p' is rounded to f16 for the second product, l is summed from the unrounded
// ones.  f16 keeps 2^-11 of a p' down to 2^-14; below that p' is a multiple of
// 2^-24.  Because p' carries ve, that is where a key's probability times its
// value page's scale is 2^-14 of the row's largest such product: a page whose
// scale is so far below another's contributes with an error of up to 2^-25 of
// the largest product times its codes, whatever its own size.  Operands of more
// bits would double the tensor cores' work (tf32) for terms that small.
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

// Flags a cu_q that does not lead from 0 to the number of tokens without a step
// back: some rows would be nobody's, or two sequences'.  By `threads` threads.
__device__ __forceinline__ void check_cu_q(const AttendParams& p, int thread, int threads) {
    for (int s = thread; s < p.b.n_seq; s += threads) {
        const int a = __ldg(p.b.cu_q + s), b = __ldg(p.b.cu_q + s + 1);
        if (a > b || (s == 0 && a != 0) || (s == p.b.n_seq - 1 && b != p.b.tokens)) kv_flag(p.c.status, B3_KV_BAD_LENGTH);
    }
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

// What the new tokens i0 .. i1 of a sequence see together: each key of
// [any_lo, any_hi) some of them, each of [lo_max, hi_min) all of them.
struct SeenByRows {
    int any_lo, lo_max, hi_min, any_hi;
    __device__ __forceinline__ bool whole(int key, int n) const { return key >= lo_max && key + n <= hi_min; }
    // keys [key, key + n) that not all rows see, where rows see different keys at all
    __device__ __forceinline__ bool split(int key, int n) const {
        return (any_lo != lo_max || any_hi != hi_min) && !whole(key, n);
    }
};
__device__ __forceinline__ SeenByRows seen_by_rows(const AttendParams& p, const SeqSpan& s, int i0, int i1) {
    SeenByRows r;
    seen_keys(p, s, i0, r.any_lo, r.hi_min);
    seen_keys(p, s, i1, r.lo_max, r.any_hi);
    return r;
}

// NaN values.  In the tensor cores' sums 0 * NaN of a value that a row does not
// see would be NaN, so in blocks of keys that only some rows see (SeenByRows::
// split) NaN codes of V go into the product as 0, and the rows that do see them
// get their NaN back at the end, by nan_channels over those blocks: their
// number depends on the rows of a tile, not on the length of the sequence.
__device__ __forceinline__ uint32_t nan_codes(uint32_t four) {   // bit 7 of each byte that is an e4m3 NaN
    return ((four & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ uint32_t without_codes(uint32_t four, uint32_t nans) { return four & ~((nans >> 7) * 0xffu); }

// By a whole warp; each lane has a row that sees the keys [lo, hi).  Sets bit b
// of mask[c] where one of these among [k0, k1) holds NaN in channel
// b * (DIM / 32) + c of V.
template <int DIM>
__device__ __noinline__ void nan_channels(const AttendParams& p, int seq, int kv_head, int k0, int k1, int lo, int hi,
                                          uint32_t (&mask)[DIM / 32]) {
    constexpr int kPer = DIM / 32, kAhead = 4;
    const int lane = threadIdx.x & 31, page = p.c.page_tokens;
    for (int j0 = k0; j0 < k1; j0 += kAhead) {
        uint32_t nans[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int j = j0 + i;
            uint32_t w = 0;
            if (j < k1) {
                int id = __ldg(p.b.page_table + seq * p.b.table_stride + j / page);
                if (id < 0 || id >= p.c.pages) id = 0;   // flagged where it was met first
                const uint8_t* v = p.c.v + ((static_cast<int64_t>(id) * p.c.kv_heads + kv_head) * page + j % page) * DIM + lane * kPer;
                w = kPer == 4 ? *reinterpret_cast<const uint32_t*>(v) : *reinterpret_cast<const uint16_t*>(v);
            }
            nans[i] = nan_codes(w);
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (!__any_sync(0xffffffffu, nans[i])) continue;
            const bool sees = j0 + i >= lo && j0 + i < hi;
#pragma unroll
            for (int c = 0; c < kPer; ++c) {
                const uint32_t m = __ballot_sync(0xffffffffu, nans[i] >> (8 * c + 7) & 1);
                if (sees) mask[c] |= m;
            }
        }
    }
}

// NaN into the channels of mask of a row at `out`.
template <int DIM, typename U>
__device__ __forceinline__ void put_nan(U* out, const uint32_t (&mask)[DIM / 32]) {
#pragma unroll
    for (int c = 0; c < DIM / 32; ++c)
        for (uint32_t m = mask[c]; m; m &= m - 1) from_f32(__uint_as_float(0x7fffffffu), out[(__ffs(m) - 1) * (DIM / 32) + c]);
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
