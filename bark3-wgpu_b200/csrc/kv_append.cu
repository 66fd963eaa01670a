// kv_append.cu — b3_kv_append: norms of queries and keys for each head, the
// position rotation, and the new keys and values into the paged 8-bit cache.
//
//   x' = R(pos) (x / sqrt(mean(x^2) + eps) * w)     for each head of q and k
//   q_out = round16(q'),  k' and v' = v -> code = e4m3(x' / 2^e), scale 2^e
// with e of a (page, head) from the largest finite magnitude that the page
// holds.  Bound by memory: each value leaves as two bytes (q) or one (k, v)
// and is read once, but for pages that one warp fills by many rows (GROUP = 1
// below); the arithmetic is some ten operations a value.
//
// One launch.  The first blocks own the cache: a (page, key head, k or v) that
// receives tokens belongs to one group of warps, which finds the page's new
// exponent over all its new rows before it writes a code, so no atomics order
// the scale.  The other blocks own q, 8 heads of 128 channels (16 of 64) of a
// token for each warp.  A row of head_dim channels is held by
// head_dim / 8 lanes, eight channels each; the norm's sum by shuffles within
// the row.  PAIRED (the usual rotation of all channels, i with i + head_dim / 2)
// gives a lane four channels and their four partners, so the rotation stays in
// the lane; otherwise a lane has eight neighbours and shuffles for partners.
//   GROUP = 1     a warp a (page, head).  Decode brings one row to each page;
//                 more rows than 256 / head_dim are read, normed and turned
//                 again after the exponent is known.
//   GROUP = 4, 8  that many warps, the page's rows in registers between the
//                 exponent and the codes.  Prompts fill whole pages; four warps
//                 hold 16 rows of 64 channels.
// The host takes groups from four new tokens a sequence on average: one choice
// for the call, so of a mixed batch one part goes the wrong way (32 + 2 x 8 heads
// of 128 in bf16: 127 sequences of one token 4.0 us, a prompt of 512 tokens 5.1,
// both in one call, in groups, 24; 255 sequences 5.8, a prompt of 700 5.1, both
// by single warps 44).
//
// Measured: 16384 tokens of 32 + 2 x 8 heads of 128 in bf16 84 us (378 MB at
// 4.5 TB/s), 29 of 64 warps resident at 64 registers, most often waiting for
// loads; one token for each of 256 sequences of the same heads
// 5.7 us: the launch, then loads one behind the other (lengths, page number and,
// behind the page's check though its address does not need it, the row).
#include "kv_cache.cuh"

namespace b3 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kQRows = 4;   // q: passes of a warp over a token's heads

struct AppendParams {
    b3_kv_cache c;
    b3_kv_batch b;
    b3_kv_append_args a;
    int unit_by_token;   // cache units: one a token (live at a page's first new token), else by page counts
    int units;
    int kv_blocks;
    int q_chunks;        // warps a token of q
    int angles16;        // cos and sin are 16-byte aligned
};

// A lane's eight channels of a row: PAIRED [4 l, 4 l + 4) and the same plus
// DIM / 2, else [8 l, 8 l + 8).
template <int DIM, bool PAIRED>
struct Piece {
    static __device__ __forceinline__ int low(int l) { return PAIRED ? 4 * l : 8 * l; }
    static __device__ __forceinline__ int high(int l) { return PAIRED ? DIM / 2 + 4 * l : 8 * l + 4; }

    template <bool VEC, typename T>
    static __device__ __forceinline__ void load(const T* row, int l, float2 (&x)[4]) {
        T v[8];
        if (VEC && !PAIRED) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
                reinterpret_cast<uint4*>(v)[i] = __ldcs(reinterpret_cast<const uint4*>(row + 8 * l) + i);
        } else if (VEC) {
            if (sizeof(T) == 4) {
                reinterpret_cast<uint4*>(v)[0] = __ldcs(reinterpret_cast<const uint4*>(row + low(l)));
                reinterpret_cast<uint4*>(v)[sizeof(T) / 4] = __ldcs(reinterpret_cast<const uint4*>(row + high(l)));
            } else {
                reinterpret_cast<uint2*>(v)[0] = __ldcs(reinterpret_cast<const uint2*>(row + low(l)));
                reinterpret_cast<uint2*>(v)[1] = __ldcs(reinterpret_cast<const uint2*>(row + high(l)));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = row[low(l) + i];
                v[4 + i] = row[high(l) + i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = make_float2(to_f32(v[2 * i]), to_f32(v[2 * i + 1]));
    }
    template <typename T>   // T of 16 bits, row 16-byte aligned
    static __device__ __forceinline__ void store(T* row, int l, const float2 (&x)[4]) {
        T v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            from_f32(x[i].x, v[2 * i]);
            from_f32(x[i].y, v[2 * i + 1]);
        }
        if (PAIRED) {
            *reinterpret_cast<uint2*>(row + low(l)) = reinterpret_cast<uint2*>(v)[0];
            *reinterpret_cast<uint2*>(row + high(l)) = reinterpret_cast<uint2*>(v)[1];
        } else {
            *reinterpret_cast<uint4*>(row + 8 * l) = *reinterpret_cast<uint4*>(v);
        }
    }
    static __device__ __forceinline__ void store_codes(uint8_t* row, int l, const float2 (&x)[4], float inv) {
        const float y[8] = {x[0].x, x[0].y, x[1].x, x[1].y, x[2].x, x[2].y, x[3].x, x[3].y};
        const uint2 c = encode8(y, inv);
        if (PAIRED) {
            *reinterpret_cast<uint32_t*>(row + low(l)) = c.x;
            *reinterpret_cast<uint32_t*>(row + high(l)) = c.y;
        } else {
            *reinterpret_cast<uint2*>(row + 8 * l) = c;
        }
    }
    static __device__ __forceinline__ void load_norm(float2 (&w)[4], const float* norm, int l) {
        if (!norm) return;
        const float4 a = __ldg(reinterpret_cast<const float4*>(norm + low(l))), b = __ldg(reinterpret_cast<const float4*>(norm + high(l)));
        w[0] = make_float2(a.x, a.y), w[1] = make_float2(a.z, a.w), w[2] = make_float2(b.x, b.y), w[3] = make_float2(b.z, b.w);
    }
};

// A lane's cosines and sines: of its four pairs (PAIRED, interleaved) or of its
// eight channels (half-split with partners in other lanes).
struct Angles {
    float2 c[4], s[4];
};
template <int DIM, bool PAIRED>
__device__ __forceinline__ void load_angles(Angles& g, int l, int pos, const AppendParams& p) {
    const b3_kv_append_args& a = p.a;
    const int half = a.rot_dim >> 1, ch = Piece<DIM, PAIRED>::low(l);
    if (!a.cos || ch >= a.rot_dim) return;
    const bool four = PAIRED || a.interleaved;
    const int64_t at = static_cast<int64_t>(pos) * half + (PAIRED ? ch : a.interleaved ? ch >> 1 : ch < half ? ch : ch - half);
    const float *c = a.cos + at, *s = a.sin + at;
    if (p.angles16) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (i && four) break;
            const float4 u = __ldg(reinterpret_cast<const float4*>(c) + i), v = __ldg(reinterpret_cast<const float4*>(s) + i);
            g.c[2 * i] = make_float2(u.x, u.y), g.c[2 * i + 1] = make_float2(u.z, u.w);
            g.s[2 * i] = make_float2(v.x, v.y), g.s[2 * i + 1] = make_float2(v.z, v.w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i > 1 && four) break;
            g.c[i] = make_float2(__ldg(c + 2 * i), __ldg(c + 2 * i + 1));
            g.s[i] = make_float2(__ldg(s + 2 * i), __ldg(s + 2 * i + 1));
        }
    }
}

__device__ __forceinline__ float2 neg2(float2 x) { return make_float2(-x.x, -x.y); }

// Norm and rotation of one row piece; the row's lanes are consecutive and every
// lane of the warp takes part.
template <int DIM, bool PAIRED>
__device__ __forceinline__ void turn_row(float2 (&x)[4], int l, const float* norm, const float2 (&w)[4], const Angles& g,
                                         const b3_kv_append_args& a) {
    if (norm) {
        float2 ss2 = __fmul2_rn(x[0], x[0]);
#pragma unroll
        for (int i = 1; i < 4; ++i) ss2 = __ffma2_rn(x[i], x[i], ss2);
        float ss = ss2.x + ss2.y;
#pragma unroll
        for (int m = DIM / 16; m; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        const float r = rsqrtf(ss * (1.f / DIM) + a.eps);   // within 2 units in the last place
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __fmul2_rn(__fmul2_rn(x[i], make_float2(r, r)), w[i]);
    }
    if (PAIRED) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 u = x[i], v = x[2 + i];
            x[i] = __ffma2_rn(u, g.c[i], neg2(__fmul2_rn(v, g.s[i])));
            x[2 + i] = __ffma2_rn(v, g.c[i], __fmul2_rn(u, g.s[i]));
        }
    } else if (a.cos) {
        const int half = a.rot_dim >> 1, ch = 8 * l;
        if (a.interleaved) {
            if (ch < a.rot_dim) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float c = i & 1 ? g.c[i >> 1].y : g.c[i >> 1].x, s = i & 1 ? g.s[i >> 1].y : g.s[i >> 1].x;
                    x[i] = make_float2(x[i].x * c - x[i].y * s, x[i].y * c + x[i].x * s);
                }
            }
        } else {
            // channels ch and ch + half turn together, half / 8 lanes apart
            const bool low = ch < half;
            const int lane = threadIdx.x & 31;
            const int from = low ? lane + (half >> 3) : lane - (half >> 3);
            float2 y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                y[i].x = __shfl_sync(0xffffffffu, x[i].x, from & 31);
                y[i].y = __shfl_sync(0xffffffffu, x[i].y, from & 31);
            }
            if (ch < a.rot_dim) {
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = __ffma2_rn(x[i], g.c[i], __fmul2_rn(low ? neg2(y[i]) : y[i], g.s[i]));
            }
        }
    }
}

__device__ __forceinline__ int token_position(const AppendParams& p, int token, int slot) {
    if (!p.a.cos) return 0;
    const int pos = p.a.positions ? __ldg(p.a.positions + token) : slot;
    if (pos < 0 || pos >= p.a.rot_rows) {
        kv_flag(p.c.status, B3_KV_BAD_POSITION);
        return min(max(pos, 0), p.a.rot_rows - 1);
    }
    return pos;
}

// [begin, end) slots of sequence s that are new, its first token's row; false
// (and a flag) if its lengths do not fit the batch.
__device__ __forceinline__ bool seq_span(const AppendParams& p, int s, int& first, int& begin, int& end) {
    first = __ldg(p.b.cu_q + s);
    const int n = __ldg(p.b.cu_q + s + 1) - first;
    end = __ldg(p.b.kv_lens + s);
    begin = end - n;
    // n <= end and not begin >= 0: of a length near -2^31 the difference would wrap around to a large one
    const bool fits = first >= 0 && n >= 0 && n <= p.b.tokens - first && n <= end &&
                      end <= static_cast<int64_t>(p.b.table_width) * p.c.page_tokens;
    if (!fits) kv_flag(p.c.status, B3_KV_BAD_LENGTH);
    return fits;
}

template <typename T, int DIM, bool VEC, bool PAIRED>
__device__ __forceinline__ void q_rows(const AppendParams& p, int warp_id) {
    using P = Piece<DIM, PAIRED>;
    constexpr int kLanes = DIM / 8, kRows = 32 / kLanes;
    const int token = warp_id / p.q_chunks;
    if (token >= p.b.tokens) return;
    const int lane = threadIdx.x & 31, l = lane % kLanes;
    const int h0 = (warp_id % p.q_chunks) * kQRows * kRows + lane / kLanes;
    const T* q = static_cast<const T*>(p.a.q) + token * p.a.q_token_stride + h0 * p.a.q_head_stride;
    float2 x[kQRows][4];
#pragma unroll
    for (int r = 0; r < kQRows; ++r) {
        if (h0 + r * kRows < p.a.q_heads)
            P::template load<VEC>(q + r * kRows * p.a.q_head_stride, l, x[r]);
        else
            x[r][0] = x[r][1] = x[r][2] = x[r][3] = make_float2(0.f, 0.f);
    }
    const int s = kv_seq_of(p.b, token);
    int first, begin, end;
    if (!seq_span(p, s, first, begin, end)) return;
    if (token < first || token - first >= end - begin) {   // a row that cu_q gives to no sequence
        kv_flag(p.c.status, B3_KV_BAD_LENGTH);
        return;
    }
    Angles g;
    float2 w[4];
    load_angles<DIM, PAIRED>(g, l, token_position(p, token, begin + token - first), p);
    P::load_norm(w, p.a.q_norm, l);
    const int64_t at = (static_cast<int64_t>(token) * p.a.q_heads + h0) * DIM;
#pragma unroll
    for (int r = 0; r < kQRows; ++r) {
        turn_row<DIM, PAIRED>(x[r], l, p.a.q_norm, w, g, p.a);
        if (h0 + r * kRows < p.a.q_heads) {
            if (p.a.out_dtype == B3_DTYPE_F16)
                P::store(static_cast<__half*>(p.a.q_out) + at + r * kRows * DIM, l, x[r]);
            else
                P::store(static_cast<__nv_bfloat16*>(p.a.q_out) + at + r * kRows * DIM, l, x[r]);
        }
    }
}

// One (page, key head, k or v).  GROUP warps of the block (all of it, or each
// warp on its own), `gw` this warp's place in the group.  ROWS: passes of the
// group over a full page; with ROWS > 0 the rows stay in registers.
template <typename T, int DIM, bool VEC, bool PAIRED, int GROUP, int ROWS>
__device__ __forceinline__ void cache_unit(const AppendParams& p, int item, int gw, float* xmax) {
    using P = Piece<DIM, PAIRED>;
    constexpr int kLanes = DIM / 8, kRows = 32 / kLanes, kStep = kRows * GROUP;
    const int heads = p.c.kv_heads, page = p.c.page_tokens;
    const int unit = item / (2 * heads), which = (item / heads) & 1, head = item % heads;
    if (unit >= p.units) return;
    const int lane = threadIdx.x & 31, l = lane % kLanes, row = gw * kRows + lane / kLanes;

    // the unit's page: [lo, hi) are the sequence's slots that are new in it
    int s, first, begin, end, lo;
    if (p.unit_by_token) {
        s = kv_seq_of(p.b, unit);
        if (!seq_span(p, s, first, begin, end)) return;
        lo = begin + unit - first;
        if (unit < first || lo >= end || (lo != begin && lo % page)) return;
    } else {
        s = kv_search([&](int i) { return __ldg(p.b.cu_q + i) / page + 2 * i; }, p.b.n_seq, unit);
        if (!seq_span(p, s, first, begin, end)) return;
        const int nth = unit - (first / page + 2 * s);
        const int64_t at = static_cast<int64_t>(begin / page + nth) * page;
        if (nth < 0 || at >= end || end == begin) return;
        lo = max(begin, static_cast<int>(at));
    }
    const int hi = min(end, (lo / page + 1) * page), held = lo % page, rows = hi - lo;
    const int to = __ldg(p.b.page_table + s * p.b.table_stride + lo / page);
    if (to < 0 || to >= p.c.pages) {
        kv_flag(p.c.status, B3_KV_BAD_PAGE);
        return;
    }
    const int64_t slab = static_cast<int64_t>(to) * heads + head;
    float* const scale_at = (which ? p.c.v_scale : p.c.k_scale) + slab;
    uint8_t* const codes = (which ? p.c.v : p.c.k) + slab * page * DIM;
    const float old_scale = held ? *scale_at : 0.f;

    const int token0 = first + lo - begin;
    const T* const from = which ? static_cast<const T*>(p.a.v) + token0 * p.a.v_token_stride + head * p.a.v_head_stride
                                : static_cast<const T*>(p.a.k) + token0 * p.a.k_token_stride + head * p.a.k_head_stride;
    const int64_t stride = which ? p.a.v_token_stride : p.a.k_token_stride;
    auto load_row = [&](int r, float2 (&x)[4]) {   // new row r of the page, zero past the last; whole warps
        if (r < rows)
            P::template load<VEC>(from + r * stride, l, x);
        else
            x[0] = x[1] = x[2] = x[3] = make_float2(0.f, 0.f);
    };
    float2 w[4];
    if (!which) P::load_norm(w, p.a.k_norm, l);
    auto turn = [&](int r, float2 (&x)[4]) {
        if (which) return;
        Angles g;
        load_angles<DIM, PAIRED>(g, l, r < rows ? token_position(p, token0 + r, lo + r) : 0, p);
        turn_row<DIM, PAIRED>(x, l, p.a.k_norm, w, g, p.a);
    };
    auto code_row = [&](int r, const float2 (&x)[4], float inv) {
        if (r < rows) P::store_codes(codes + static_cast<int64_t>(held + r) * DIM, l, x, inv);
    };

    constexpr int kKeep = ROWS > 0 ? ROWS : 1;
    float2 x[kKeep][4];
    float amax = 0.f;
    if (ROWS > 0) {
#pragma unroll
        for (int k = 0; k < kKeep; ++k) load_row(row + k * kStep, x[k]);
#pragma unroll
        for (int k = 0; k < kKeep; ++k) {
            turn(row + k * kStep, x[k]);
#pragma unroll
            for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(fabsf(x[k][i].x), fabsf(x[k][i].y)));
        }
        if (__any_sync(0xffffffffu, amax == INFINITY)) {   // infinities have no say in a scale (nor NaN, which fmaxf passes over)
            amax = 0.f;
#pragma unroll
            for (int k = 0; k < kKeep; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(finite_abs(x[k][i].x), finite_abs(x[k][i].y)));
        }
    } else {
        for (int r = row; r - lane / kLanes < rows; r += kStep) {
            load_row(r, x[0]);
            turn(r, x[0]);
#pragma unroll
            for (int i = 0; i < 4; ++i) amax = fmaxf(amax, fmaxf(finite_abs(x[0][i].x), finite_abs(x[0][i].y)));
        }
    }
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    if (GROUP > 1) {   // the group's warps are all here: the early exits above are the same for all of them
        if (lane == 0) xmax[gw] = amax;
        asm volatile("bar.sync %0, %1;" ::"r"(1 + static_cast<int>(threadIdx.x) / (32 * GROUP)), "n"(32 * GROUP) : "memory");
#pragma unroll
        for (int w = 0; w < GROUP; ++w) amax = fmaxf(amax, xmax[w]);
    }
    int e = scale_exp(amax);
    if (held) {
        const int old = stored_exp(old_scale);
        if (e <= old) {
            e = old;
        } else {
            // the scale grows: the codes held so far follow it
            const float f = exp2_int(max(old - e, -126));
            for (int r = row; r < held; r += kStep) {
                uint2* at = reinterpret_cast<uint2*>(codes + static_cast<int64_t>(r) * DIM + 8 * l);
                float y[8];
                decode8(*at, y);
                *at = encode8(y, f);
            }
        }
    }
    const float inv = exp2_int(-e);
    if (ROWS > 0) {
#pragma unroll
        for (int k = 0; k < kKeep; ++k) code_row(row + k * kStep, x[k], inv);
    } else if (rows <= kStep) {
        code_row(row, x[0], inv);
    } else {
        for (int r = row; r - lane / kLanes < rows; r += kStep) {
            load_row(r, x[0]);
            turn(r, x[0]);
            code_row(r, x[0], inv);
        }
    }
    if (gw == 0 && lane == 0) *scale_at = exp2_int(e);
}

template <typename T, int DIM, bool VEC, bool PAIRED, int GROUP, int ROWS>
__global__ void __launch_bounds__(kThreads, ROWS >= 8 ? 2 : 4) k_kv_append(const __grid_constant__ AppendParams p) {
    __shared__ float xmax[kWarps];
    const int warp = threadIdx.x >> 5;
    if (static_cast<int>(blockIdx.x) < p.kv_blocks) {
        const int group = warp / GROUP;
        cache_unit<T, DIM, VEC, PAIRED, GROUP, ROWS>(p, blockIdx.x * (kWarps / GROUP) + group, warp % GROUP, xmax + group * GROUP);
    } else {
        q_rows<T, DIM, VEC, PAIRED>(p, (blockIdx.x - p.kv_blocks) * kWarps + warp);
    }
}

template <typename T, int DIM, bool VEC, bool PAIRED, int GROUP, int ROWS>
int launch(const AppendParams& p, int64_t blocks, cudaStream_t st) {
    k_kv_append<T, DIM, VEC, PAIRED, GROUP, ROWS><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : set_cuda_error("k_kv_append", e);
}

template <typename T, int DIM, bool VEC, bool PAIRED>
int launch_dim(AppendParams& p, cudaStream_t st) {
    constexpr int kRows = 32 / (DIM / 8);
    const int page = p.c.page_tokens;
    // units: every (sequence, page) pair that receives tokens has one.  Either
    // one a token, or cu_q[i] / page + 2 i before sequence i's first: a span
    // of n tokens touches at most (n - 2) / page + 2 pages.
    const int64_t by_page = p.b.tokens / page + 2ll * p.b.n_seq;
    p.unit_by_token = p.b.tokens <= by_page;
    p.units = static_cast<int>(p.unit_by_token ? p.b.tokens : by_page);
    p.q_chunks = (p.a.q_heads + kQRows * kRows - 1) / (kQRows * kRows);
    const int64_t items = static_cast<int64_t>(p.units) * 2 * p.c.kv_heads;
    const int64_t q_warps = static_cast<int64_t>(p.b.tokens) * p.q_chunks;
    const bool whole = p.b.tokens >= 4ll * p.b.n_seq;
    const int passes = page / (kRows * kWarps);
    const int group = !whole ? 1 : passes ? kWarps : 4;
    const int64_t kv_blocks = (items * group + kWarps - 1) / kWarps;
    const int64_t blocks = kv_blocks + (q_warps + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffffll || items > 0x7fffffffll || q_warps > 0x7fffffffll)
        return set_error(B3_EINVAL, "b3_kv_append: %lld tokens are too many for one call",
                         static_cast<long long>(p.b.tokens));
    p.kv_blocks = static_cast<int>(kv_blocks);
    if (!whole) return launch<T, DIM, VEC, PAIRED, 1, 0>(p, blocks, st);
    // pages of 16 to 128 tokens: 1 to 8 passes of 16 rows of 128 channels, 0 to 4 of 32 rows of 64
    if constexpr (DIM == 128) {
        if (passes == 8) return launch<T, DIM, VEC, PAIRED, kWarps, 8>(p, blocks, st);
    } else {
        if (passes == 0) return launch<T, DIM, VEC, PAIRED, 4, 1>(p, blocks, st);
    }
    switch (passes) {
        case 4: return launch<T, DIM, VEC, PAIRED, kWarps, 4>(p, blocks, st);
        case 2: return launch<T, DIM, VEC, PAIRED, kWarps, 2>(p, blocks, st);
        default: return launch<T, DIM, VEC, PAIRED, kWarps, 1>(p, blocks, st);
    }
}

template <typename T>
int launch_type(AppendParams& p, cudaStream_t st) {
    const b3_kv_append_args& a = p.a;
    const int per16 = 16 / static_cast<int>(sizeof(T));
    const uintptr_t bases = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
    const int64_t strides = a.q_token_stride | a.q_head_stride | a.k_token_stride | a.k_head_stride |
                            a.v_token_stride | a.v_head_stride;
    const bool vec = bases % 16 == 0 && strides % per16 == 0;
    const bool paired = a.cos && !a.interleaved && a.rot_dim == p.c.head_dim;
    if (p.c.head_dim == 128) {
        if (paired) return vec ? launch_dim<T, 128, true, true>(p, st) : launch_dim<T, 128, false, true>(p, st);
        return vec ? launch_dim<T, 128, true, false>(p, st) : launch_dim<T, 128, false, false>(p, st);
    }
    if (paired) return vec ? launch_dim<T, 64, true, true>(p, st) : launch_dim<T, 64, false, true>(p, st);
    return vec ? launch_dim<T, 64, true, false>(p, st) : launch_dim<T, 64, false, false>(p, st);
}

}  // namespace

int kv_check(const b3_kv_cache* c, const b3_kv_batch* b) {
    if (!c || !b) return set_error(B3_EINVAL, "null cache or batch");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !b->cu_q || !b->kv_lens || !b->page_table)
        return set_error(B3_EINVAL, "null buffer in the cache or the batch");
    if (c->head_dim != 64 && c->head_dim != 128)
        return set_error(B3_EINVAL, "head_dim %d (64 and 128 are supported)", c->head_dim);
    if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
        return set_error(B3_EINVAL, "page_tokens %d (16, 32, 64 and 128 are supported)", c->page_tokens);
    if (c->pages <= 0 || c->kv_heads <= 0 ||
        static_cast<int64_t>(c->pages) * c->kv_heads > 0x7fffffffll / c->page_tokens)
        return set_error(B3_EINVAL, "cache of %d pages x %d heads x %d tokens (need 1 .. 2^31 - 1 rows)", c->pages,
                         c->kv_heads, c->page_tokens);
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
        return set_error(B3_EINVAL, "the cache's codes must be 16-byte aligned");
    if (b->n_seq <= 0 || b->tokens < 0 || b->table_width <= 0 || (b->table_stride < b->table_width && b->table_stride != 0))
        return set_error(B3_EINVAL, "batch of %d sequences, %d tokens, page table %d wide with stride %lld", b->n_seq,
                         b->tokens, b->table_width, static_cast<long long>(b->table_stride));
    // what is left up to 2^31 lets the kernels round a token's place up to a block or a tile
    if (static_cast<int64_t>(b->table_width) * c->page_tokens > kMostTokens)
        return set_error(B3_EINVAL, "a page table of %d entries passes %lld tokens", b->table_width,
                         static_cast<long long>(kMostTokens));
    return 0;
}

}  // namespace b3

using namespace b3;

extern "C" int b3_kv_append(const b3_kv_cache* cache, const b3_kv_batch* batch, const b3_kv_append_args* args,
                            void* stream) {
    if (int rc = kv_check(cache, batch)) return rc;
    if (!args) return set_error(B3_EINVAL, "null arguments");
    const b3_kv_append_args& a = *args;
    if (batch->tokens == 0) return 0;
    if (!a.q || !a.k || !a.v || !a.q_out) return set_error(B3_EINVAL, "null q, k, v or q_out");
    if (a.q_heads <= 0 || a.q_heads % cache->kv_heads)
        return set_error(B3_EINVAL, "q_heads %d is no multiple of kv_heads %d", a.q_heads, cache->kv_heads);
    if (a.out_dtype != B3_DTYPE_F16 && a.out_dtype != B3_DTYPE_BF16)
        return set_error(B3_EINVAL, "out_dtype %d (f16 or bf16)", a.out_dtype);
    if (reinterpret_cast<uintptr_t>(a.q_out) & 15) return set_error(B3_EINVAL, "q_out must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(a.q_norm) | reinterpret_cast<uintptr_t>(a.k_norm)) & 15)
        return set_error(B3_EINVAL, "norm weights must be 16-byte aligned");
    if (!a.cos != !a.sin) return set_error(B3_EINVAL, "cos and sin come together");
    if (a.cos && (a.rot_dim <= 0 || a.rot_dim > cache->head_dim || a.rot_dim % 16 || a.rot_rows <= 0))
        return set_error(B3_EINVAL, "rot_dim %d (a multiple of 16, at most head_dim %d), rot_rows %d", a.rot_dim,
                         cache->head_dim, a.rot_rows);
    AppendParams p{};
    p.c = *cache;
    p.b = *batch;
    p.a = a;
    p.angles16 = ((reinterpret_cast<uintptr_t>(a.cos) | reinterpret_cast<uintptr_t>(a.sin)) & 15) == 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (a.dtype) {
        case B3_DTYPE_F32: return launch_type<float>(p, st);
        case B3_DTYPE_F16: return launch_type<__half>(p, st);
        case B3_DTYPE_BF16: return launch_type<__nv_bfloat16>(p, st);
        default: return set_error(B3_EINVAL, "dtype %d", a.dtype);
    }
}
