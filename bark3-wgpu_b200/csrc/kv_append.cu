// kv_append.cu — b3_kv_append: norms of queries and keys for each head, the
// position rotation, and the new keys and values into the paged 8-bit cache.
//
//   x' = R(pos) (x / sqrt(mean(x^2) + eps) * w)     for each head of q and k
//   q_out = round16(q'),  k' and v' = v -> code = e4m3(x' / 2^e), scale 2^e
// with e of a (page, head) from the largest finite magnitude that the page
// holds.  Bound by memory: each value is read once and leaves as two bytes
// (q) or one (k, v); the arithmetic is some ten operations a value.
//
// One launch.  The first blocks own the cache: a (page, key head, k or v) that
// receives tokens belongs to one group of warps, which finds the page's new
// exponent over all its new rows before it writes a code, so no atomics and no
// second pass over memory order the scale.  The other blocks own q, a few
// heads of a token for each warp.  A row of head_dim channels is held by
// head_dim / 8 lanes, eight channels each: 16-byte loads of 16-bit types, the
// norm and the rotation's partner channels by shuffles within the row.
//   GROUP = 1: a warp a (page, head).  Decode brings one row to each page.
//   GROUP = 8: a whole block, the page's rows in registers between the
//              exponent and the codes.  Prompts fill whole pages.
// The host takes GROUP = 8 from four new tokens a sequence on average.
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
};

// Norm and rotation of one row piece: channels [8 l, 8 l + 8) of a row whose
// lanes are consecutive; every lane of the warp takes part.
template <int DIM>
__device__ __forceinline__ void turn_row(float (&x)[8], int l, const float* norm, int pos, const b3_kv_append_args& a) {
    if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
        for (int m = DIM / 16; m; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        const float r = 1.f / sqrtf(ss * (1.f / DIM) + a.eps);
        const float4 w0 = __ldg(reinterpret_cast<const float4*>(norm) + 2 * l);
        const float4 w1 = __ldg(reinterpret_cast<const float4*>(norm) + 2 * l + 1);
        const float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = x[i] * r * w[i];
    }
    if (a.cos) {
        const int half = a.rot_dim >> 1;
        const int64_t row = static_cast<int64_t>(pos) * half;
        const int ch = 8 * l;
        if (a.interleaved) {
            if (ch < a.rot_dim) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float c = __ldg(a.cos + row + (ch >> 1) + i), s = __ldg(a.sin + row + (ch >> 1) + i);
                    const float u = x[2 * i], v = x[2 * i + 1];
                    x[2 * i] = u * c - v * s;
                    x[2 * i + 1] = v * c + u * s;
                }
            }
        } else {
            // channels ch and ch + half turn together, half / 8 lanes apart
            const bool low = ch < half;
            const int lane = threadIdx.x & 31;
            const int from = low ? lane + (half >> 3) : lane - (half >> 3);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], from & 31);
            if (ch < a.rot_dim) {
                const int64_t at = row + (low ? ch : ch - half);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float c = __ldg(a.cos + at + i), s = __ldg(a.sin + at + i);
                    x[i] = low ? x[i] * c - y[i] * s : x[i] * c + y[i] * s;
                }
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
    const bool fits = first >= 0 && n >= 0 && n <= p.b.tokens - first && begin >= 0 &&
                      end <= static_cast<int64_t>(p.b.table_width) * p.c.page_tokens;
    if (!fits) kv_flag(p.c.status, B3_KV_BAD_LENGTH);
    return fits;
}

template <typename T, int DIM, bool VEC>
__device__ __forceinline__ void q_rows(const AppendParams& p, int warp_id) {
    constexpr int kLanes = DIM / 8, kRows = 32 / kLanes;
    const int token = warp_id / p.q_chunks;
    if (token >= p.b.tokens) return;
    const int lane = threadIdx.x & 31, l = lane % kLanes;
    const int s = kv_seq_of(p.b, token);
    int first, begin, end;
    if (!seq_span(p, s, first, begin, end) || token - first < 0 || token - first >= end - begin) return;
    const int pos = token_position(p, token, begin + token - first);
    const int h0 = (warp_id % p.q_chunks) * kQRows * kRows + lane / kLanes;
    float x[kQRows][8];
#pragma unroll
    for (int r = 0; r < kQRows; ++r) {
        const int h = h0 + r * kRows;
        if (h < p.a.q_heads)
            load8<VEC>(static_cast<const T*>(p.a.q) + token * p.a.q_token_stride + h * p.a.q_head_stride + 8 * l, x[r]);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) x[r][i] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < kQRows; ++r) {
        const int h = h0 + r * kRows;
        turn_row<DIM>(x[r], l, p.a.q_norm, pos, p.a);
        if (h < p.a.q_heads) {
            const int64_t at = (static_cast<int64_t>(token) * p.a.q_heads + h) * DIM + 8 * l;
            if (p.a.out_dtype == B3_DTYPE_F16)
                store8(static_cast<__half*>(p.a.q_out) + at, x[r]);
            else
                store8(static_cast<__nv_bfloat16*>(p.a.q_out) + at, x[r]);
        }
    }
}

// One (page, key head, k or v).  GROUP warps of the block (all of it, or each
// warp on its own), `gw` this warp's place in the group.  ROWS: passes of the
// group over a full page; with ROWS > 0 the rows stay in registers.
template <typename T, int DIM, bool VEC, int GROUP, int ROWS>
__device__ __forceinline__ void cache_unit(const AppendParams& p, int item, int gw, float* xmax) {
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

    auto load_row = [&](int r, float (&x)[8]) {   // new row r of the page, zero past the last; whole warps
        const int token = first + lo - begin + r;
        if (r < rows) {
            if (which)
                load8<VEC>(static_cast<const T*>(p.a.v) + token * p.a.v_token_stride + head * p.a.v_head_stride + 8 * l, x);
            else
                load8<VEC>(static_cast<const T*>(p.a.k) + token * p.a.k_token_stride + head * p.a.k_head_stride + 8 * l, x);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.f;
        }
    };
    auto turn = [&](int r, float (&x)[8]) {
        if (!which) turn_row<DIM>(x, l, p.a.k_norm, r < rows ? token_position(p, first + lo - begin + r, lo + r) : 0, p.a);
    };
    auto code_row = [&](int r, const float (&x)[8], float inv) {
        if (r < rows) *reinterpret_cast<uint2*>(codes + static_cast<int64_t>(held + r) * DIM + 8 * l) = encode8(x, inv);
    };

    constexpr int kKeep = ROWS > 0 ? ROWS : 1;
    float x[kKeep][8];
    float amax = 0.f;
    if (ROWS > 0) {
#pragma unroll
        for (int k = 0; k < kKeep; ++k) load_row(row + k * kStep, x[k]);
#pragma unroll
        for (int k = 0; k < kKeep; ++k) {
            turn(row + k * kStep, x[k]);
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(x[k][i]));
        }
    } else {
        for (int r = row; r - lane / kLanes < rows; r += kStep) {
            load_row(r, x[0]);
            turn(r, x[0]);
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(x[0][i]));
        }
    }
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
    if (GROUP > 1) {   // every thread of the block is here: the early exits above are the same for all of it
        if (lane == 0) xmax[gw] = amax;
        __syncthreads();
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

template <typename T, int DIM, bool VEC, int GROUP, int ROWS>
__global__ void __launch_bounds__(kThreads) k_kv_append(const __grid_constant__ AppendParams p) {
    __shared__ float xmax[kWarps];
    const int warp = threadIdx.x >> 5;
    if (static_cast<int>(blockIdx.x) < p.kv_blocks) {
        if (GROUP > 1)
            cache_unit<T, DIM, VEC, GROUP, ROWS>(p, blockIdx.x, warp, xmax);
        else
            cache_unit<T, DIM, VEC, GROUP, ROWS>(p, blockIdx.x * kWarps + warp, 0, xmax);
    } else {
        q_rows<T, DIM, VEC>(p, (blockIdx.x - p.kv_blocks) * kWarps + warp);
    }
}

template <typename T, int DIM, bool VEC, int GROUP, int ROWS>
int launch(const AppendParams& p, int64_t blocks, cudaStream_t st) {
    k_kv_append<T, DIM, VEC, GROUP, ROWS><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : set_cuda_error("k_kv_append", e);
}

template <typename T, int DIM, bool VEC>
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
    const int64_t kv_blocks = whole ? items : (items + kWarps - 1) / kWarps;
    const int64_t blocks = kv_blocks + (q_warps + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffffll || items > 0x7fffffffll || q_warps > 0x7fffffffll)
        return set_error(B3_EINVAL, "b3_kv_append: %lld tokens are too many for one call",
                         static_cast<long long>(p.b.tokens));
    p.kv_blocks = static_cast<int>(kv_blocks);
    if (!whole) return launch<T, DIM, VEC, 1, 0>(p, blocks, st);
    switch (page / (kRows * kWarps)) {
        case 8: return launch<T, DIM, VEC, kWarps, 8>(p, blocks, st);
        case 4: return launch<T, DIM, VEC, kWarps, 4>(p, blocks, st);
        case 2: return launch<T, DIM, VEC, kWarps, 2>(p, blocks, st);
        default: return launch<T, DIM, VEC, kWarps, 1>(p, blocks, st);
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
    if (p.c.head_dim == 128) return vec ? launch_dim<T, 128, true>(p, st) : launch_dim<T, 128, false>(p, st);
    return vec ? launch_dim<T, 64, true>(p, st) : launch_dim<T, 64, false>(p, st);
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
    if (b->n_seq <= 0 || b->tokens < 0 || b->table_width <= 0 || b->table_stride < b->table_width)
        return set_error(B3_EINVAL, "batch of %d sequences, %d tokens, page table %d wide with stride %lld", b->n_seq,
                         b->tokens, b->table_width, static_cast<long long>(b->table_stride));
    if (static_cast<int64_t>(b->table_width) * c->page_tokens > 0x7fffffffll)
        return set_error(B3_EINVAL, "a page table of %d entries passes 2^31 tokens", b->table_width);
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
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (a.dtype) {
        case B3_DTYPE_F32: return launch_type<float>(p, st);
        case B3_DTYPE_F16: return launch_type<__half>(p, st);
        case B3_DTYPE_BF16: return launch_type<__nv_bfloat16>(p, st);
        default: return set_error(B3_EINVAL, "dtype %d", a.dtype);
    }
}
