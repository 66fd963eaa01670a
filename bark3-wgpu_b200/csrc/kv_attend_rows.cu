// kv_attend_rows.cu — attention over the paged 8-bit cache for few query rows:
// the decode step (one or a few new tokens a sequence).
//
// Bound by memory: a key head's cached codes are read once for all the query
// rows that share it (new tokens x heads of the group, at most 16: one MMA
// tile).  The mathematics is in kv_attend.cuh.
//
// Work.  The steps of 32 keys of all (sequence, key head) items, laid end to
// end, are cut into equal runs, one for each resident warp, so ragged batches
// and one long sequence keep every SM reading to the end.  A warp carries the
// running maximum, sum and output of its item in registers; a run that covers
// an item from end to end stores the result, other runs leave partial results
// that k_join adds up in run order (same bits every time).
//
// A step.  Each warp has its own ring of stages in shared memory, filled by
// TMA boxes of a page's rows, lines of 128 bytes in the 128-byte swizzle.
//   scores  S[rows, 8 keys] += Q[rows, 16 dims] K^T   mma m16n8k16, B = K codes
//   output  O[rows, 8 dims] += P[rows, 16 keys] V     mma m16n8k16, B = V codes
// The S tile's accumulator layout is P's operand layout, so probabilities never
// leave registers.  Which 16 channels an MMA step takes and which output
// channel a column stands for are free choices: a lane takes 16 consecutive
// bytes of a K row as four steps' operands, and of a V row as the same column
// of 16 tiles, so both come by 16-byte loads; a V operand pairs two keys, two
// byte permutes for four channels.  Which key a score column stands for is
// free as well (key_of_col): chosen so that both kinds of load touch every
// bank once.  m16n8k16 on mma.sync suffices here: at 16 rows the products need
// a third of its rate when memory is saturated, and tcgen05's 128-row tiles
// would multiply zeros.
#include <algorithm>
#include <type_traits>

#include "b3_ptx.cuh"
#include "kv_attend.cuh"

namespace b3 {
namespace {

constexpr int kStep = 32;           // keys
constexpr int kMaxSeqs = 1024;      // sequences a launch
constexpr int kMinRun = 2;          // steps a run at least

template <int DIM>
struct Cfg {
    static constexpr int kWarps = 8;
    static constexpr int kStages = DIM == 128 ? 3 : 6;
    static constexpr uint32_t kHalf = kStep * DIM;             // K (or V) bytes of a stage
    static constexpr uint32_t kStage = 2 * kHalf;
    static constexpr uint32_t kRing = kWarps * kStages * kStage;
    static constexpr uint32_t kBars = kRing;
    static constexpr uint32_t kPrefix = kBars + kWarps * kStages * 8;
    static constexpr uint32_t kSmem = kPrefix + (kMaxSeqs + 1) * 4 + 64 + 1024;
};

struct RowsParams {
    AttendParams p;
    int seq0, seqs;        // this launch's sequences
    int workers, rows;     // warps of the grid; row capacity of a partial result (8 or 16)
    float* part;           // [workers][2][rows][DIM] outputs, then [workers][2][rows][2] (m, l)
};

// Score column c (0..7) of a tile stands for this key of the tile's eight.
template <int DIM>
__device__ __forceinline__ int key_of_col(int c) {
    return DIM == 128 ? c ^ ((c & 1) << 2) : c ^ ((c >> 1) & 1);
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t codes2(uint32_t two) {   // two e4m3 codes -> f16x2
    const __half2 h = decode2(two & 0xffffu);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}

// The keys [lo, hi) that any row of a sequence sees, lo down to a step.
__device__ __forceinline__ void item_keys(const AttendParams& p, const SeqSpan& s, int& lo, int& hi) {
    int a, b;
    seen_keys(p, s, 0, lo, a);
    seen_keys(p, s, s.n - 1, b, hi);
    lo = min(lo, hi) / kStep * kStep;
}

// Steps of one key head of a sequence: at least one where it has queries, so
// that rows that see nothing are written too.
__device__ __forceinline__ int seq_steps(const RowsParams& r, int s) {
    SeqSpan sp = attend_span(r.p, r.seq0 + s);
    if (sp.n == 0) return 0;
    int lo, hi;
    item_keys(r.p, sp, lo, hi);
    return max(1, (hi - lo + kStep - 1) / kStep);
}

// prefix[i] = steps of one key head in the sequences before i, by the whole block.
__device__ __forceinline__ void make_prefix(const RowsParams& r, int* prefix, int* warp_sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nwarps = blockDim.x >> 5;
    int carry = 0;
    for (int base = 0; base < r.seqs; base += blockDim.x) {
        const int s = base + tid;
        int v = s < r.seqs ? seq_steps(r, s) : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += u;
        }
        if (lane == 31) warp_sums[warp] = v;
        __syncthreads();
        int before = carry, all = carry;
        for (int w = 0; w < nwarps; ++w) {
            const int t = warp_sums[w];
            before += w < warp ? t : 0;
            all += t;
        }
        if (s < r.seqs) prefix[s + 1] = before + v;
        carry = all;
        __syncthreads();
    }
    if (tid == 0) prefix[0] = 0;
    __syncthreads();
}

// Item and first step of global step g: heads of a sequence follow one another.
struct Place {
    int seq, head;       // seq within the launch
    int64_t begin;       // global step of the item's first
    int steps;
};
__device__ __forceinline__ Place place_of(const int* prefix, int n, int heads, int64_t g) {
    int lo = 0, hi = n;   // prefix[lo] * heads <= g < prefix[hi] * heads
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (static_cast<int64_t>(prefix[mid]) * heads <= g) lo = mid; else hi = mid;
    }
    Place q;
    q.seq = lo;
    q.steps = prefix[lo + 1] - prefix[lo];
    const int64_t base = static_cast<int64_t>(prefix[lo]) * heads;
    q.head = static_cast<int>((g - base) / q.steps);
    q.begin = base + static_cast<int64_t>(q.head) * q.steps;
    return q;
}

__device__ __forceinline__ int64_t run_length(int64_t total, int workers) {
    return max(static_cast<int64_t>(kMinRun), (total + workers - 1) / workers);
}

template <typename T>
__device__ __forceinline__ void store_row(const AttendParams& p, int token, int head, int d, const float* o, int n, float inv) {
    T* out = static_cast<T*>(p.a.out) + (static_cast<int64_t>(token) * p.a.q_heads + head) * p.c.head_dim + d;
    for (int i = 0; i < n; i += 8) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = o[i + j] * inv;
        store8(out + i, x);
    }
}

template <typename T, int DIM, int ROWS>
__global__ void __launch_bounds__(Cfg<DIM>::kWarps * 32, 1)
    k_attend_rows(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ RowsParams r) {
    using C = Cfg<DIM>;
    constexpr int kTiles = DIM / 8;      // output tiles of 8 channels; also 2 x the MMA steps over the channels
    constexpr int kHalves = ROWS / 8;    // 1: rows 8..15 of the MMA tile are empty
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    int* prefix = reinterpret_cast<int*>(smem + C::kPrefix);
    const AttendParams& p = r.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * C::kStages * C::kStage;
    const uint32_t bars = smem_u32(smem + C::kBars) + warp * C::kStages * 8;
    if (lane == 0) {
        for (int s = 0; s < C::kStages; ++s) mbar_init(bars + 8 * s, 1);
        fence_mbar_init();
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
    }
    pdl_launch_dependents();
    make_prefix(r, prefix, prefix + kMaxSeqs + 1);

    const int heads = p.c.kv_heads, group = p.a.q_heads / heads, page = p.c.page_tokens;
    const int64_t total = static_cast<int64_t>(prefix[r.seqs]) * heads;
    const int64_t run = run_length(total, r.workers);
    const int worker = warp * gridDim.x + blockIdx.x;   // neighbours in work on different SMs
    int64_t at = worker * run;
    const int64_t end = min(at + run, total);
    const int log_page = 31 - __clz(page);
    uint32_t issued = 0, used = 0;   // stages over the warp's life

    while (at < end) {
        const Place it = place_of(prefix, r.seqs, heads, at);
        const int seq = r.seq0 + it.seq;
        const SeqSpan sp = attend_span(p, seq);
        int key_lo, key_hi;
        item_keys(p, sp, key_lo, key_hi);
        const int s0 = static_cast<int>(at - it.begin);
        const int s1 = static_cast<int>(min(end - it.begin, static_cast<int64_t>(it.steps)));
        const int key0 = key_lo + s0 * kStep;                 // this run's keys of the item: [key0, key1)
        const int key1 = min(key_lo + s1 * kStep, key_hi);
        const int n_steps = key1 > key0 ? (key1 - key0 + kStep - 1) / kStep : 0;
        const int n_rows = sp.n * group;

        // pages: lane i of a group of 32 holds page `page0 + i`, its number and scales
        const int page_last = (key1 - 1) >> log_page;
        int page0 = key0 >> log_page;
        auto load_pages = [&](int from, int& id, float& ks, float& vs) {
            id = 0;
            ks = vs = 1.f;
            if (from + lane <= page_last) {
                id = __ldg(p.b.page_table + seq * p.b.table_stride + from + lane);
                if (id < 0 || id >= p.c.pages) {
                    kv_flag(p.c.status, B3_KV_BAD_PAGE);
                    id = 0;
                }
                const int64_t slab = static_cast<int64_t>(id) * heads + it.head;
                ks = __ldg(p.c.k_scale + slab);
                vs = __ldg(p.c.v_scale + slab);
            }
        };
        int id_a, id_b;
        float ks_a, vs_a, ks_b, vs_b;
        if (n_steps) {
            load_pages(page0, id_a, ks_a, vs_a);
            load_pages(page0 + 32, id_b, ks_b, vs_b);
        }
        auto page_id = [&](int pg) {
            const int i = pg - page0;
            const int a = __shfl_sync(0xffffffffu, id_a, i & 31), b = __shfl_sync(0xffffffffu, id_b, i & 31);
            return i < 32 ? a : b;
        };
        auto issue = [&](int step) {   // whole warp; step of this run
            const int key = key0 + step * kStep;
            const uint32_t st = issued % C::kStages;
            ++issued;
            const uint32_t bar = bars + 8 * st, dst = ring + st * C::kStage;
            if (page >= kStep) {
                const int id = page_id(key >> log_page);
                if (lane == 0) {
                    const int row = (id * heads + it.head) * page + (key & (page - 1));
                    const int line = DIM == 128 ? row : row >> 1;
                    mbar_arrive_expect_tx(bar, C::kStage);
                    tma_load_2d(dst, &map_k, bar, 0, line);
                    tma_load_2d(dst + C::kHalf, &map_v, bar, 0, line);
                }
            } else {   // two pages of 16
                const int pg = key >> log_page;
                const int id0 = page_id(pg), id1 = page_id(pg + 1);
                if (lane == 0) {
                    const bool two = key + 16 < key1;
                    mbar_arrive_expect_tx(bar, two ? C::kStage : C::kStage / 2);
                    int row = (id0 * heads + it.head) * page;
                    int line = DIM == 128 ? row : row >> 1;
                    tma_load_2d(dst, &map_k, bar, 0, line);
                    tma_load_2d(dst + C::kHalf, &map_v, bar, 0, line);
                    if (two) {
                        row = (id1 * heads + it.head) * page;
                        line = DIM == 128 ? row : row >> 1;
                        tma_load_2d(dst + C::kHalf / 2, &map_k, bar, 0, line);
                        tma_load_2d(dst + C::kHalf + C::kHalf / 2, &map_v, bar, 0, line);
                    }
                }
            }
        };
        for (int i = 0; i < C::kStages && i < n_steps; ++i) issue(i);

        // queries: row r of the tile is new token r / group, head r % group
        uint32_t qa[kTiles / 2][4];
        float qscale[kHalves];
        int row_lo[kHalves], row_hi[kHalves], lo_max = 0, hi_min = key_hi;
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf) {
            const int row = g + 8 * hf;
            const bool live = row < n_rows;
            const int i = live ? row / group : 0;
            const T* q = static_cast<const T*>(p.a.q) + static_cast<int64_t>(sp.first + i) * p.a.q_token_stride +
                         static_cast<int64_t>(it.head * group + (live ? row % group : 0)) * p.a.q_head_stride + 16 * t;
            T v[DIM / 4];
            const bool vec = ((reinterpret_cast<uintptr_t>(p.a.q) | (p.a.q_token_stride * 2) | (p.a.q_head_stride * 2)) & 15) == 0;
#pragma unroll
            for (int c = 0; c < DIM / 64; ++c) {
                if (!live) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) from_f32(0.f, v[16 * c + k]);
                } else if (vec) {
                    reinterpret_cast<uint4*>(v)[2 * c] = __ldg(reinterpret_cast<const uint4*>(q + 64 * c));
                    reinterpret_cast<uint4*>(v)[2 * c + 1] = __ldg(reinterpret_cast<const uint4*>(q + 64 * c + 8));
                } else {
#pragma unroll
                    for (int k = 0; k < 16; ++k) v[16 * c + k] = q[64 * c + k];
                }
            }
            int shift = 0;
            if (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
                float amax = 0.f;
#pragma unroll
                for (int k = 0; k < DIM / 4; ++k) amax = fmaxf(amax, fabsf(to_f32(v[k])));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                shift = row_shift(amax);
            }
            const float mul = exp2_int(shift);
            qscale[hf] = p.a.scale * kLog2e * exp2_int(-shift);
#pragma unroll
            for (int k = 0; k < kTiles / 2; ++k) {
                // MMA step k = 4 c + i: channels 64 c + 16 t + 4 i + {0, 1 | 2, 3}
                __half2 h0, h1;
                if (std::is_same<T, __half>::value) {
                    h0 = reinterpret_cast<const __half2*>(v)[2 * k];
                    h1 = reinterpret_cast<const __half2*>(v)[2 * k + 1];
                } else {
                    h0 = __floats2half2_rn(to_f32(v[4 * k]) * mul, to_f32(v[4 * k + 1]) * mul);
                    h1 = __floats2half2_rn(to_f32(v[4 * k + 2]) * mul, to_f32(v[4 * k + 3]) * mul);
                }
                qa[k][hf] = *reinterpret_cast<uint32_t*>(&h0);
                qa[k][2 + hf] = *reinterpret_cast<uint32_t*>(&h1);
                if (kHalves == 1) qa[k][1] = qa[k][3] = 0;
            }
            seen_keys(p, sp, i, row_lo[hf], row_hi[hf]);
        }
        {   // keys that every row sees: [lo_max, hi_min)
            int lo, hi;
            seen_keys(p, sp, 0, lo, hi);
            hi_min = hi;
            seen_keys(p, sp, sp.n - 1, lo, hi);
            lo_max = lo;
        }
        int any_lo, any_hi;   // keys that some row sees
        {
            int x;
            seen_keys(p, sp, 0, any_lo, x);
            seen_keys(p, sp, sp.n - 1, x, any_hi);
        }

        float o[kTiles][2 * kHalves], m[kHalves], l[kHalves];
#pragma unroll
        for (int j = 0; j < kTiles; ++j)
#pragma unroll
            for (int e = 0; e < 2 * kHalves; ++e) o[j][e] = 0.f;
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf) {
            m[hf] = -INFINITY;
            l[hf] = 0.f;
        }

        bool ok = true;
        for (int step = 0; step < n_steps && ok; ++step) {
            const int key = key0 + step * kStep;
            if ((key >> log_page) - page0 >= 32) {
                page0 += 32;
                id_a = id_b, ks_a = ks_b, vs_a = vs_b;
                load_pages(page0 + 32, id_b, ks_b, vs_b);
            }
            // scales of the two 16-key halves
            float ks[2], vs[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int i = ((key + 16 * u) >> log_page) - page0;
                const float ka = __shfl_sync(0xffffffffu, ks_a, i & 31), kb = __shfl_sync(0xffffffffu, ks_b, i & 31);
                const float va = __shfl_sync(0xffffffffu, vs_a, i & 31), vb = __shfl_sync(0xffffffffu, vs_b, i & 31);
                ks[u] = i < 32 ? ka : kb;
                vs[u] = i < 32 ? va : vb;
            }
            const uint32_t st = used % C::kStages;
            const uint32_t kbase = ring + st * C::kStage, vbase = kbase + C::kHalf;
            ok = __all_sync(0xffffffffu, mbar_wait(bars + 8 * st, (used / C::kStages) & 1, 0x60));
            ++used;
            if (!ok) {
                kv_flag(p.c.status, B3_KV_TIMEOUT);
                break;
            }

            // ── scores ──
            float s[4][4];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
                const int kk = 8 * n + key_of_col<DIM>(g);
#pragma unroll
                for (int c = 0; c < DIM / 64; ++c) {
                    const uint32_t line = DIM == 128 ? kk : kk >> 1;
                    const uint32_t piece = DIM == 128 ? t + 4 * c : (kk & 1) * 4 + t;
                    const uint4 w = lds128(kbase + line * 128 + ((piece ^ (line & 7)) << 4));
                    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) mma16816(s[n], qa[4 * c + i], codes2(ww[i]), codes2(ww[i] >> 16));
                }
            }
            const bool whole = key >= lo_max && key + kStep <= hi_min;   // no row masks any key here
            float ve[2], rv[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int e = stored_exp(vs[u]);
                ve[u] = static_cast<float>(e);
                rv[u] = exp2_int(-e);
            }
            float top[kHalves];
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf) {
                top[hf] = m[hf];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const float f = fminf(qscale[hf] * ks[n >> 1], 3.4e38f);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = fmaf(s[n][2 * hf + e], f, ve[n >> 1]);
                        if (!whole) {
                            const int j = key + 8 * n + key_of_col<DIM>(2 * t + e);
                            if (j < row_lo[hf] || j >= row_hi[hf]) x = -INFINITY;
                        }
                        s[n][2 * hf + e] = x;
                        top[hf] = fmaxf(top[hf], x);
                    }
                }
                top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 1));
                top[hf] = fmaxf(top[hf], __shfl_xor_sync(0xffffffffu, top[hf], 2));
            }
            bool moved = false;
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf) moved = moved || top[hf] > m[hf];
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int hf = 0; hf < kHalves; ++hf) {
                    const float corr = m[hf] == top[hf] ? 1.f : ex2_approx(m[hf] - top[hf]);
                    m[hf] = top[hf];
                    l[hf] *= corr;
#pragma unroll
                    for (int j = 0; j < kTiles; ++j) {
                        o[j][2 * hf] *= corr;
                        o[j][2 * hf + 1] *= corr;
                    }
                }
            }
            uint32_t pa[2][4];
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf) {
                const float ref = m[hf] == -INFINITY ? 0.f : m[hf];   // nothing seen yet: every x is -inf
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const float p0 = ex2_approx(s[n][2 * hf] - ref), p1 = ex2_approx(s[n][2 * hf + 1] - ref);
                    l[hf] = fmaf(p0 + p1, rv[n >> 1], l[hf]);
                    const __half2 h = __floats2half2_rn(p0, p1);
                    pa[n >> 1][2 * (n & 1) + hf] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            if (kHalves == 1)
#pragma unroll
                for (int u = 0; u < 2; ++u) pa[u][1] = pa[u][3] = 0;

            // ── output ──
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t w[4][DIM / 32];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int kk = 16 * u + 8 * (i >> 1) + key_of_col<DIM>(2 * t + (i & 1));
                    const uint32_t line = DIM == 128 ? kk : kk >> 1;
                    if (DIM == 128) {
                        const uint4 q4 = lds128(vbase + line * 128 + ((g ^ (line & 7)) << 4));
                        w[i][0] = q4.x, w[i][1] = q4.y, w[i][DIM / 32 - 2] = q4.z, w[i][DIM / 32 - 1] = q4.w;
                    } else {
                        const uint32_t piece = (kk & 1) * 4 + (g >> 1);
                        const uint2 q2 = lds64(vbase + line * 128 + ((piece ^ (line & 7)) << 4) + (g & 1) * 8);
                        w[i][0] = q2.x, w[i][1] = q2.y;
                    }
                    // a key that no row sees may hold anything, NaN codes among it: 0 * NaN is no zero
                    if (!whole && (key + kk < any_lo || key + kk >= any_hi))
#pragma unroll
                        for (int j = 0; j < DIM / 32; ++j) w[i][j] = 0;
                }
#pragma unroll
                for (int j = 0; j < DIM / 32; ++j) {
                    const uint32_t x01 = prmt(w[0][j], w[1][j], 0x5140), y01 = prmt(w[0][j], w[1][j], 0x7362);
                    const uint32_t x23 = prmt(w[2][j], w[3][j], 0x5140), y23 = prmt(w[2][j], w[3][j], 0x7362);
                    const uint32_t b01[4] = {codes2(x01), codes2(x01 >> 16), codes2(y01), codes2(y01 >> 16)};
                    const uint32_t b23[4] = {codes2(x23), codes2(x23 >> 16), codes2(y23), codes2(y23 >> 16)};
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        float d[4] = {o[4 * j + b][0], o[4 * j + b][1], 0.f, 0.f};
                        if (kHalves == 2) d[2] = o[4 * j + b][2 * kHalves - 2], d[3] = o[4 * j + b][2 * kHalves - 1];
                        mma16816(d, pa[u], b01[b], b23[b]);
                        o[4 * j + b][0] = d[0], o[4 * j + b][1] = d[1];
                        if (kHalves == 2) o[4 * j + b][2 * kHalves - 2] = d[2], o[4 * j + b][2 * kHalves - 1] = d[3];
                    }
                }
            }
            __syncwarp();   // every lane has read the stage
            if (step + C::kStages < n_steps) issue(step + C::kStages);
        }

        // ── the run's end: rows' sums over the four lanes that share them ──
        const bool all = s0 == 0 && s1 == it.steps;
        const int64_t slot = 2ll * worker + (at > worker * run ? 1 : 0);
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf) {
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 1);
            l[hf] += __shfl_xor_sync(0xffffffffu, l[hf], 2);
            const int row = g + 8 * hf;
            if (row >= n_rows) continue;
            // columns 2t and 2t + 1 of tile j: channels kTiles (2t) + j and kTiles (2t + 1) + j
            float x[2][kTiles];
#pragma unroll
            for (int j = 0; j < kTiles; ++j) x[0][j] = o[j][2 * hf], x[1][j] = o[j][2 * hf + 1];
            if (all) {
                const int token = sp.first + row / group, head = it.head * group + row % group;
                const float inv = l[hf] == 0.f ? 0.f : 1.f / l[hf];
                store_row<T>(p, token, head, kTiles * 2 * t, x[0], kTiles, inv);
                store_row<T>(p, token, head, kTiles * (2 * t + 1), x[1], kTiles, inv);
                if (p.a.lse && t == 0)
                    p.a.lse[static_cast<int64_t>(token) * p.a.q_heads + head] =
                        l[hf] == 0.f ? -INFINITY : (m[hf] + log2f(l[hf])) * kLn2;
            } else {
                float* po = r.part + (slot * ROWS + row) * DIM + kTiles * 2 * t;
#pragma unroll
                for (int j = 0; j < 2 * kTiles; j += 4)
                    *reinterpret_cast<float4*>(po + j) =
                        make_float4(x[j / kTiles][j % kTiles], x[j / kTiles][j % kTiles + 1], x[j / kTiles][j % kTiles + 2],
                                    x[j / kTiles][j % kTiles + 3]);
                if (t == 0)
                    *reinterpret_cast<float2*>(r.part + 2ll * r.workers * ROWS * DIM + (slot * ROWS + row) * 2) =
                        make_float2(m[hf], l[hf]);
            }
        }
        if (!ok) break;
        at = it.begin + s1;
    }
}

// Adds up the partial results of the items that more than one run worked on:
// block w takes the item that starts in run w and goes on past it.  Eight
// warps share the runs; each lane keeps DIM / 32 channels.
template <typename T, int DIM, int ROWS>
__global__ void __launch_bounds__(256) k_attend_join(const __grid_constant__ RowsParams r) {
    constexpr int kPer = DIM / 32;
    __shared__ int prefix[kMaxSeqs + 1 + 16];
    __shared__ float so[8][DIM], sl[8];
    make_prefix(r, prefix, prefix + kMaxSeqs + 1);
    const AttendParams& p = r.p;
    const int heads = p.c.kv_heads, group = p.a.q_heads / heads;
    const int64_t total = static_cast<int64_t>(prefix[r.seqs]) * heads;
    const int64_t run = run_length(total, r.workers);
    const int w0 = blockIdx.x;
    const int64_t edge = (w0 + 1) * run;          // first step of the next run
    Place it = {};
    if (edge < total) it = place_of(prefix, r.seqs, heads, edge - 1);
    pdl_wait();   // the partial results are complete (and this kernel ends after the one before it)
    if (edge >= total || it.begin < w0 * run || it.begin + it.steps <= edge) return;
    const int w1 = static_cast<int>((it.begin + it.steps - 1) / run);
    const int slot0 = it.begin > w0 * run ? 1 : 0;
    const SeqSpan sp = attend_span(p, r.seq0 + it.seq);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* ml = r.part + 2ll * r.workers * ROWS * DIM;
    for (int row = 0; row < sp.n * group; ++row) {
        auto slot = [&](int w) { return (2ll * w + (w == w0 ? slot0 : 0)) * ROWS + row; };
        float m = -INFINITY;
        for (int w = w0 + lane; w <= w1; w += 32) m = fmaxf(m, ml[slot(w) * 2]);
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        const float ref = m == -INFINITY ? 0.f : m;
        float l = 0.f, o[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) o[i] = 0.f;
#pragma unroll 4
        for (int w = w0 + warp; w <= w1; w += 8) {
            const float2 x = *reinterpret_cast<const float2*>(ml + slot(w) * 2);
            const float f = ex2_approx(x.x - ref);
            l = fmaf(x.y, f, l);
            const float* po = r.part + slot(w) * DIM + lane * kPer;
            float v[kPer];
            if (kPer == 4) {
                const float4 y = *reinterpret_cast<const float4*>(po);
                v[0] = y.x, v[1] = y.y, v[kPer - 2] = y.z, v[kPer - 1] = y.w;
            } else {
                const float2 y = *reinterpret_cast<const float2*>(po);
                v[0] = y.x, v[1] = y.y;
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) o[i] = fmaf(v[i], f, o[i]);
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) so[warp][lane * kPer + i] = o[i];
        if (lane == 0) sl[warp] = l;
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < DIM) {
            float a = 0.f;
            l = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                a += so[w][threadIdx.x];
                l += sl[w];
            }
            const int token = sp.first + row / group, head = it.head * group + row % group;
            const int64_t at = static_cast<int64_t>(token) * p.a.q_heads + head;
            from_f32(l == 0.f ? 0.f : a / l, static_cast<T*>(p.a.out)[at * DIM + threadIdx.x]);
            if (p.a.lse && threadIdx.x == 0) p.a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
        __syncthreads();
    }
}

template <int DIM>
int workers_of() { return device_sms() * Cfg<DIM>::kWarps; }

int row_capacity(const AttendParams& p) { return p.a.max_q * (p.a.q_heads / p.c.kv_heads) <= 8 ? 8 : 16; }

template <typename T, int DIM, int ROWS>
int launch(const AttendParams& p, void* workspace, cudaStream_t st) {
    using C = Cfg<DIM>;
    static PerDeviceOnce smem_once;
    int rc = set_smem_limit_once(smem_once, k_attend_rows<T, DIM, ROWS>, C::kSmem, "cudaFuncSetAttribute(k_attend_rows)");
    if (rc) return rc;
    CUtensorMap mk, mv;
    const uint64_t lines = static_cast<uint64_t>(p.c.pages) * p.c.kv_heads * p.c.page_tokens * DIM / 128;
    const uint32_t box = (p.c.page_tokens < kStep ? p.c.page_tokens : kStep) * DIM / 128;
    rc = make_map_2d(&mk, p.c.k, kMapU8, 128, lines, 128, 128, box, true);
    if (!rc) rc = make_map_2d(&mv, p.c.v, kMapU8, 128, lines, 128, 128, box, true);
    if (rc) return rc;
    RowsParams r{p, 0, 0, workers_of<DIM>(), ROWS, static_cast<float*>(workspace)};
    // sequences a launch: the prefix array's room, and all their steps in 31 bits
    const int64_t most = static_cast<int64_t>(p.b.table_width) * p.c.page_tokens / kStep + 1;
    const int at_once = static_cast<int>(std::min<int64_t>(kMaxSeqs, 0x7fffffffll / most));
    for (; r.seq0 < p.b.n_seq; r.seq0 += at_once) {
        r.seqs = std::min(at_once, p.b.n_seq - r.seq0);
        k_attend_rows<T, DIM, ROWS><<<device_sms(), C::kWarps * 32, C::kSmem, st>>>(mk, mv, r);
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return set_cuda_error("k_attend_rows", e);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(r.workers);
        cfg.blockDim = dim3(256);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, k_attend_join<T, DIM, ROWS>, r);
        if (e != cudaSuccess) return set_cuda_error("k_attend_join", e);
    }
    return 0;
}

template <typename T>
int launch_type(const AttendParams& p, void* workspace, cudaStream_t st) {
    const bool few = row_capacity(p) == 8;
    if (p.c.head_dim == 128) return few ? launch<T, 128, 8>(p, workspace, st) : launch<T, 128, 16>(p, workspace, st);
    return few ? launch<T, 64, 8>(p, workspace, st) : launch<T, 64, 16>(p, workspace, st);
}

}  // namespace

int64_t attend_rows_workspace(const AttendParams& p) {
    const int64_t workers = p.c.head_dim == 128 ? workers_of<128>() : workers_of<64>();
    return workers * 2 * row_capacity(p) * (p.c.head_dim + 2) * 4;
}

int launch_attend_rows(const AttendParams& p, void* workspace, cudaStream_t st) {
    return p.a.dtype == B3_DTYPE_F16 ? launch_type<__half>(p, workspace, st) : launch_type<__nv_bfloat16>(p, workspace, st);
}

}  // namespace b3
