// kv_attend_rows.cu — attention over the paged 8-bit cache for few query rows:
// the decode step (one or a few new tokens a sequence).
//
// Bound by memory: a key head's cached codes are read once for all the query
// rows that share it (new tokens x heads of the group, at most 16: one MMA
// tile).  The mathematics is in kv_attend.cuh.
//
// Work.  The steps of 32 keys of all (sequence, key head) items, laid end to
// end with four more units for the start of each item (without them the warps
// that get the shortest sequences, a dozen of them, finish last: 94 against 63
// us for a ragged batch of 128), are cut into equal runs, one for each resident
// warp, so ragged batches and one long sequence keep every SM reading to the end.  A warp carries the
// running maximum, sum and output of its item in registers; a run that covers
// an item from end to end stores the result, other runs leave partial results
// that k_attend_join adds up in run order (same bits every time).
//
// A step.  Each warp has its own ring of stages in shared memory, filled by
// TMA boxes of a page's rows, lines of 128 bytes in the 128-byte swizzle.  Both
// products are transposed, the codes being the MMA's 16-row operand, so a tile
// of eight query rows wastes nothing (mma m16n8k16, f16 -> f32):
//   S^T[16 keys, 8 rows] += K[16 keys, 16 channels] Q^T
//   O^T[16 channels, 8 rows] += V^T[16 channels, 16 keys] P^T
// P^T's operand layout is S^T's accumulator layout with each 8 x 8 block
// transposed (movmatrix), so probabilities never leave registers.  Which 16
// channels an MMA step takes and which channel an output row stands for are
// free choices: a lane takes 16 consecutive bytes of a K row as four steps'
// operands, and of a V row as the same row of 16 tiles' columns, so both come
// by 16-byte loads; a V operand pairs two keys, two byte permutes for four
// channels.  Which key a score row stands for is free as well (key_of_row):
// chosen so that both kinds of load touch every bank once.  mma.sync suffices
// here: at eight rows the products need a sixth of its rate when memory is
// saturated, and tcgen05's 128-row tiles would hold one token's few rows.
//
// Measured (32 query heads, 8 key heads of 128): 128 sequences of 16 to 7504
// tokens 63 us (320 MB at 5.1 TB/s); one of 100,003 tokens 48 us (205 MB at
// 4.2 TB/s), where start, first loads and join take some 15 us.
#include <algorithm>
#include <type_traits>

#include "b3_ptx.cuh"
#include "kv_attend.cuh"

namespace b3 {
namespace {

constexpr int kStep = 32;           // keys
constexpr int kTilesM = kStep / 16; // MMA tiles of 16 keys
constexpr int kMaxSeqs = 1024;      // sequences a launch
constexpr int kItem = 4;            // what starting an item costs, in steps (measured on a decode batch of head_dim 128)

template <int DIM, int ROWS>
struct Cfg {
    // eight rows leave registers for ten warps: one sequence of 100,003 tokens took 50 us with ten of two
    // stages, 51 with eight of three, 52 with twelve of two (the ragged batch 94, 101 and 96, all before item
    // starts were counted into the runs); the ring takes what shared memory there is
    static constexpr int kWarps = ROWS == 8 ? 10 : 8;
    static constexpr int kStages = (ROWS == 8 ? 2 : 3) * 128 / DIM;
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
    int workers;           // warps of the grid
    float* part;           // [workers][2][ROWS][DIM] outputs, then [workers][2][ROWS][2] (m, l)
};

// Score row c (0..7) of a tile's half stands for this key of the half's eight.
template <int DIM>
__device__ __forceinline__ int key_of_row(int c) {
    return DIM == 128 ? c ^ ((c & 1) << 2) : c ^ ((c >> 1) & 1);
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {   // of an 8 x 8 block of 16-bit values over the warp
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
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

// Units of one key head of a sequence: kItem and its steps, of which there is
// at least one where it has queries, so that rows that see nothing are written.
__device__ __forceinline__ int seq_units(const RowsParams& r, int s) {
    SeqSpan sp = attend_span(r.p, r.seq0 + s);
    if (sp.n == 0) return 0;
    int lo, hi;
    item_keys(r.p, sp, lo, hi);
    return kItem + max(1, (hi - lo + kStep - 1) / kStep);
}

// prefix[i] = units of one key head in the sequences before i, by the whole block.
__device__ __forceinline__ void make_prefix(const RowsParams& r, int* prefix, int* warp_sums) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nwarps = blockDim.x >> 5;
    int carry = 0;
    for (int base = 0; base < r.seqs; base += blockDim.x) {
        const int s = base + tid;
        int v = s < r.seqs ? seq_units(r, s) : 0;
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

// The item of global unit g: heads of a sequence follow one another.
struct Place {
    int seq, head;       // seq within the launch
    int64_t begin;       // global unit of the item's first
    int units;
};
__device__ __forceinline__ Place place_of(const int* prefix, int n, int heads, int64_t g) {
    int lo = 0, hi = n;   // prefix[lo] * heads <= g < prefix[hi] * heads
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (static_cast<int64_t>(prefix[mid]) * heads <= g) lo = mid; else hi = mid;
    }
    Place q;
    q.seq = lo;
    q.units = prefix[lo + 1] - prefix[lo];
    const int64_t base = static_cast<int64_t>(prefix[lo]) * heads;
    q.head = static_cast<int>((g - base) / q.units);
    q.begin = base + static_cast<int64_t>(q.head) * q.units;
    return q;
}

__device__ __forceinline__ int64_t run_length(int64_t total, int workers) {
    return max(static_cast<int64_t>(1), (total + workers - 1) / workers);
}

template <typename T, int N>
__device__ __forceinline__ void store_row(const AttendParams& p, int token, int head, int d, const float (&o)[N], float inv) {
    T* out = static_cast<T*>(p.a.out) + (static_cast<int64_t>(token) * p.a.q_heads + head) * p.c.head_dim + d;
#pragma unroll
    for (int i = 0; i < N; i += 8) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = o[i + j] * inv;
        store8(out + i, x);
    }
}

// NaN codes out of a staged V of `bytes`, by a warp; true if this lane met one.
// Out of line: few steps need it, and in line the compiler predicates it.
__device__ __noinline__ bool clean_v(uint32_t v, uint32_t bytes) {
    uint32_t any = 0;
    for (uint32_t at = v + 16 * (threadIdx.x & 31); at < v + bytes; at += 512) {
        const uint4 x = lds128(at), n = make_uint4(nan_codes(x.x), nan_codes(x.y), nan_codes(x.z), nan_codes(x.w));
        if (!(n.x | n.y | n.z | n.w)) continue;
        any = 1;
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(without_codes(x.x, n.x)),
                     "r"(without_codes(x.y, n.y)), "r"(without_codes(x.z, n.z)), "r"(without_codes(x.w, n.w))
                     : "memory");
    }
    if (any) fence_async_shared();   // the next TMA box into this stage comes after these stores
    return any;
}

// NaN back into the rows of an item, where a key of [key0, key1) that the row
// sees holds it; lane i has row i.  The rows have been stored, by all lanes, as
// output (slot < 0) or partial results.
template <typename T, int DIM, int ROWS>
__device__ __noinline__ void restore_nan(const RowsParams& r, int seq, int head, int key0, int key1, int64_t slot) {
    const AttendParams& p = r.p;
    const SeqSpan sp = attend_span(p, seq);
    const SeenByRows see = seen_by_rows(p, sp, 0, sp.n - 1);
    const int lane = threadIdx.x & 31, group = p.a.q_heads / p.c.kv_heads;
    const bool live = lane < sp.n * group;
    uint32_t mask[DIM / 32] = {};
    int lo = 0, hi = 0;
    if (live) seen_keys(p, sp, lane / group, lo, hi);
    for (int key = key0; key < key1; key += kStep)
        if (see.split(key, kStep)) nan_channels<DIM>(p, seq, head, max(key, see.any_lo), min(key + kStep, key1), lo, hi, mask);
    __syncwarp();
    if (live && slot < 0)
        put_nan<DIM>(static_cast<T*>(p.a.out) +
                         (static_cast<int64_t>(sp.first + lane / group) * p.a.q_heads + head * group + lane % group) * DIM, mask);
    else if (live)
        put_nan<DIM>(r.part + (slot * ROWS + lane) * DIM, mask);
}

template <typename T, int DIM, int ROWS>
__global__ void __launch_bounds__(Cfg<DIM, ROWS>::kWarps * 32, 1)
    k_attend_rows(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const __grid_constant__ RowsParams r) {
    using C = Cfg<DIM, ROWS>;
    constexpr int kSteps = DIM / 16;     // MMA steps over the channels; also output tiles of 16 channels
    constexpr int kHalves = ROWS / 8;    // tiles of eight query rows
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
        const int64_t upto = min(end, it.begin + it.units), from = at;
        at = upto;
        const int s0 = max(0, static_cast<int>(from - it.begin) - kItem), s1 = static_cast<int>(upto - it.begin) - kItem;
        if (s1 <= s0) continue;   // only the item's start
        const int seq = r.seq0 + it.seq;
        const SeqSpan sp = attend_span(p, seq);
        int key_lo, key_hi;
        item_keys(p, sp, key_lo, key_hi);
        const int key0 = key_lo + s0 * kStep;                 // this run's keys of the item: [key0, key1)
        const int key1 = min(key_lo + s1 * kStep, key_hi);
        const int n_steps = key1 > key0 ? (key1 - key0 + kStep - 1) / kStep : 0;
        const int n_rows = sp.n * group;

        // pages: lane i holds the number and scales of page `page0 + i`, and the number of page `page0 + 32 + i`
        const int page_last = (key1 - 1) >> log_page;
        int page0 = key0 >> log_page;
        auto load_id = [&](int pg) {
            int id = 0;
            if (pg <= page_last) {
                id = __ldg(p.b.page_table + seq * p.b.table_stride + pg);
                if (id < 0 || id >= p.c.pages) {
                    kv_flag(p.c.status, B3_KV_BAD_PAGE);
                    id = 0;
                }
            }
            return id;
        };
        auto load_scale = [&](const float* scale, int id) { return __ldg(scale + static_cast<int64_t>(id) * heads + it.head); };
        int id_a = 0, id_b = 0;
        float ks_a = 1.f, vs_a = 1.f;
        if (n_steps) {
            id_a = load_id(page0 + lane);
            id_b = load_id(page0 + 32 + lane);
            ks_a = load_scale(p.c.k_scale, id_a);
            vs_a = load_scale(p.c.v_scale, id_a);
        }
        auto page_id = [&](int pg) {
            const int i = pg - page0;
            return __shfl_sync(0xffffffffu, i < 32 ? id_a : id_b, i & 31);
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

        // queries: row r of the item is new token r / group, head r % group; this lane loads rows g and
        // g + 8 (the product's columns), and keeps the scores of rows 2t, 2t + 1, + 8
        uint32_t qb[kHalves][kSteps][2];
        float qscale[kHalves][2];
        int row_lo[kHalves][2], row_hi[kHalves][2];
        const bool vec = ((reinterpret_cast<uintptr_t>(p.a.q) | (p.a.q_token_stride * 2) | (p.a.q_head_stride * 2)) & 15) == 0;
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf) {
            const int row = g + 8 * hf;
            const bool live = row < n_rows;
            const T* q = static_cast<const T*>(p.a.q) +
                         static_cast<int64_t>(sp.first + (live ? row / group : 0)) * p.a.q_token_stride +
                         static_cast<int64_t>(it.head * group + (live ? row % group : 0)) * p.a.q_head_stride + 16 * t;
            T v[DIM / 4];
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
            if (!std::is_same<T, __half>::value) {
                float amax = 0.f;
#pragma unroll
                for (int k = 0; k < DIM / 4; ++k) amax = fmaxf(amax, fabsf(to_f32(v[k])));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                shift = row_shift(amax);
            }
            const float mul = exp2_int(shift);
            const float qs = p.a.scale * kLog2e * exp2_int(-shift);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                // MMA step k = 4 c + i: channels 64 c + 16 t + 4 i + {0, 1 | 2, 3}
                __half2 h0, h1;
                if (std::is_same<T, __half>::value) {
                    h0 = reinterpret_cast<const __half2*>(v)[2 * k];
                    h1 = reinterpret_cast<const __half2*>(v)[2 * k + 1];
                } else {
                    h0 = __floats2half2_rn(to_f32(v[4 * k]) * mul, to_f32(v[4 * k + 1]) * mul);
                    h1 = __floats2half2_rn(to_f32(v[4 * k + 2]) * mul, to_f32(v[4 * k + 3]) * mul);
                }
                qb[hf][k][0] = *reinterpret_cast<uint32_t*>(&h0);
                qb[hf][k][1] = *reinterpret_cast<uint32_t*>(&h1);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                qscale[hf][e] = __shfl_sync(0xffffffffu, qs, 4 * (2 * t + e));
                const int mine = 2 * t + e + 8 * hf;
                seen_keys(p, sp, mine < n_rows ? mine / group : 0, row_lo[hf][e], row_hi[hf][e]);
            }
        }
        const SeenByRows see = seen_by_rows(p, sp, 0, sp.n - 1);
        bool nans = false;   // this lane has taken NaN codes of V out

        float o[kHalves][kSteps][4], m[kHalves][2], l[kHalves][2];
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf) {
#pragma unroll
            for (int j = 0; j < kSteps; ++j) o[hf][j][0] = o[hf][j][1] = o[hf][j][2] = o[hf][j][3] = 0.f;
            m[hf][0] = m[hf][1] = -INFINITY;
            l[hf][0] = l[hf][1] = 0.f;
        }

        bool ok = true;
        for (int step = 0; step < n_steps && ok; ++step) {
            const int key = key0 + step * kStep;
            if ((key >> log_page) - page0 >= 32) {
                page0 += 32;
                id_a = id_b;
                id_b = load_id(page0 + 32 + lane);
                ks_a = load_scale(p.c.k_scale, id_a);
                vs_a = load_scale(p.c.v_scale, id_a);
            }
            // scales of the step's page, or of its two pages of 16
            float ks[kTilesM];
            int ve[kTilesM];
            {
                const int i = (key >> log_page) - page0;
                ks[0] = __shfl_sync(0xffffffffu, ks_a, i);
                ve[0] = stored_exp(__shfl_sync(0xffffffffu, vs_a, i));
#pragma unroll
                for (int mt = 1; mt < kTilesM; ++mt) {
                    ks[mt] = ks[0];
                    ve[mt] = ve[0];
                    if (page < kStep) {
                        ks[mt] = __shfl_sync(0xffffffffu, ks_a, i + mt);
                        ve[mt] = stored_exp(__shfl_sync(0xffffffffu, vs_a, i + mt));
                    }
                }
            }
            const uint32_t st = used % C::kStages;
            const uint32_t kbase = ring + st * C::kStage, vbase = kbase + C::kHalf;
            ok = __all_sync(0xffffffffu, mbar_wait(bars + 8 * st, (used / C::kStages) & 1, 0x60));
            ++used;
            if (!ok) {
                kv_flag(p.c.status, B3_KV_TIMEOUT);
                // the block must not leave before its copies have landed: this one and those behind it, each with the same limit
                for (uint32_t u = used - 1; u != issued; ++u) mbar_wait(bars + 8 * (u % C::kStages), (u / C::kStages) & 1, 0x61);
                break;
            }

            // ── scores ──
            float s[kHalves][kTilesM][4];
#pragma unroll
            for (int mt = 0; mt < kTilesM; ++mt) {
#pragma unroll
                for (int hf = 0; hf < kHalves; ++hf) s[hf][mt][0] = s[hf][mt][1] = s[hf][mt][2] = s[hf][mt][3] = 0.f;
#pragma unroll
                for (int c = 0; c < DIM / 64; ++c) {
                    uint32_t w[2][4];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int kk = 16 * mt + 8 * u + key_of_row<DIM>(g);
                        const uint32_t line = DIM == 128 ? kk : kk >> 1;
                        const uint32_t piece = DIM == 128 ? t + 4 * c : (kk & 1) * 4 + t;
                        const uint4 x = lds128(kbase + line * 128 + ((piece ^ (line & 7)) << 4));
                        w[u][0] = x.x, w[u][1] = x.y, w[u][2] = x.z, w[u][3] = x.w;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t a0 = codes2(w[0][i]), a1 = codes2(w[1][i]);
                        const uint32_t a2 = codes2(w[0][i] >> 16), a3 = codes2(w[1][i] >> 16);
#pragma unroll
                        for (int hf = 0; hf < kHalves; ++hf)
                            mma16816(s[hf][mt], a0, a1, a2, a3, qb[hf][4 * c + i][0], qb[hf][4 * c + i][1]);
                    }
                }
            }
            const bool whole = see.whole(key, kStep);   // no row masks any key here
            float top[kHalves][2];
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    top[hf][e] = m[hf][e];
#pragma unroll
                    for (int mt = 0; mt < kTilesM; ++mt) {
                        const float f = fminf(qscale[hf][e] * ks[mt], 3.4e38f);
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            float x = fmaf(s[hf][mt][2 * u + e], f, static_cast<float>(ve[mt]));
                            if (!whole) {
                                const int j = key + 16 * mt + 8 * u + key_of_row<DIM>(g);
                                if (j < row_lo[hf][e] || j >= row_hi[hf][e]) x = -INFINITY;
                            }
                            s[hf][mt][2 * u + e] = x;
                            top[hf][e] = fmaxf(top[hf][e], x);
                        }
                    }
                }
#pragma unroll
            for (int d = 4; d < 32; d <<= 1)
#pragma unroll
                for (int hf = 0; hf < kHalves; ++hf)
#pragma unroll
                    for (int e = 0; e < 2; ++e) top[hf][e] = fmaxf(top[hf][e], __shfl_xor_sync(0xffffffffu, top[hf][e], d));
            bool moved = false;
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf) moved = moved || top[hf][0] > m[hf][0] || top[hf][1] > m[hf][1];
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int hf = 0; hf < kHalves; ++hf)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float corr = m[hf][e] == top[hf][e] ? 1.f : ex2_approx(m[hf][e] - top[hf][e]);
                        m[hf][e] = top[hf][e];
                        l[hf][e] *= corr;
#pragma unroll
                        for (int j = 0; j < kSteps; ++j) {
                            o[hf][j][e] *= corr;
                            o[hf][j][2 + e] *= corr;
                        }
                    }
            }
            uint32_t pb[kHalves][kTilesM][2];
#pragma unroll
            for (int hf = 0; hf < kHalves; ++hf) {
                // nothing seen yet: every x is -inf
                const float ref0 = m[hf][0] == -INFINITY ? 0.f : m[hf][0], ref1 = m[hf][1] == -INFINITY ? 0.f : m[hf][1];
#pragma unroll
                for (int mt = 0; mt < kTilesM; ++mt) {
                    float p4[4];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        p4[2 * u] = ex2_approx(s[hf][mt][2 * u] - ref0);
                        p4[2 * u + 1] = ex2_approx(s[hf][mt][2 * u + 1] - ref1);
                        const __half2 h = __floats2half2_rn(p4[2 * u], p4[2 * u + 1]);
                        pb[hf][mt][u] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h));
                    }
                    const float rv = exp2_int(-ve[mt]);
                    l[hf][0] = fmaf(p4[0] + p4[2], rv, l[hf][0]);
                    l[hf][1] = fmaf(p4[1] + p4[3], rv, l[hf][1]);
                }
            }

            // ── output ──
            if (see.split(key, kStep)) {
                nans |= clean_v(vbase, C::kHalf);
                __syncwarp();
            }
#pragma unroll
            for (int mt = 0; mt < kTilesM; ++mt) {
                uint32_t w[4][DIM / 32];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int kk = 16 * mt + 8 * (i >> 1) + key_of_row<DIM>(2 * t + (i & 1));
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
                    if (!whole && (key + kk < see.any_lo || key + kk >= see.any_hi))
#pragma unroll
                        for (int j = 0; j < DIM / 32; ++j) w[i][j] = 0;
                }
#pragma unroll
                for (int j = 0; j < DIM / 32; ++j) {   // channels (DIM / 8) g + 4 j + {0, 1 | 2, 3}
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const uint32_t lo = prmt(w[0][j], w[1][j], b ? 0x7362 : 0x5140);
                        const uint32_t hi = prmt(w[2][j], w[3][j], b ? 0x7362 : 0x5140);
                        const uint32_t a0 = codes2(lo), a1 = codes2(lo >> 16), a2 = codes2(hi), a3 = codes2(hi >> 16);
#pragma unroll
                        for (int hf = 0; hf < kHalves; ++hf)
                            mma16816(o[hf][2 * j + b], a0, a1, a2, a3, pb[hf][mt][0], pb[hf][mt][1]);
                    }
                }
            }
            __syncwarp();   // every lane has read the stage
            if (step + C::kStages < n_steps) issue(step + C::kStages);
        }

        // ── the run's end: rows' sums over the eight lanes that share them ──
        const bool all = s0 == 0 && s1 == it.units - kItem;
        const int64_t slot = 2ll * worker + (from > worker * run ? 1 : 0);
#pragma unroll
        for (int hf = 0; hf < kHalves; ++hf)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = l[hf][e];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                const int row = 2 * t + e + 8 * hf;
                if (row >= n_rows) continue;
                float x[2 * kSteps];   // channels [2 kSteps g, + 2 kSteps)
#pragma unroll
                for (int j = 0; j < kSteps; ++j) x[2 * j] = o[hf][j][e], x[2 * j + 1] = o[hf][j][2 + e];
                if (all) {
                    const int token = sp.first + row / group, head = it.head * group + row % group;
                    store_row<T>(p, token, head, 2 * kSteps * g, x, row_inverse(sum));
                    if (p.a.lse && g == 0)
                        p.a.lse[static_cast<int64_t>(token) * p.a.q_heads + head] =
                            row_lse(m[hf][e], sum);
                } else {
                    float* po = r.part + (slot * ROWS + row) * DIM + 2 * kSteps * g;
#pragma unroll
                    for (int j = 0; j < 2 * kSteps; j += 4)
                        *reinterpret_cast<float4*>(po + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                    if (g == 0)
                        *reinterpret_cast<float2*>(r.part + 2ll * r.workers * ROWS * DIM + (slot * ROWS + row) * 2) =
                            make_float2(m[hf][e], sum);
                }
            }
        if (!ok) break;
        if (__any_sync(0xffffffffu, nans)) restore_nan<T, DIM, ROWS>(r, seq, it.head, key0, key1, all ? -1 : slot);
    }
}

// Adds up the partial results of the items that more than one run worked on,
// a block an item (few items: a block an item and row), its warps shared out
// among the rows and of each row among its runs.  Each lane keeps DIM / 32
// channels.
constexpr int kJoinMax = 32;   // warps

template <typename T, int DIM, int ROWS>
__global__ void __launch_bounds__(kJoinMax * 32) k_attend_join(const __grid_constant__ RowsParams r) {
    constexpr int kPer = DIM / 32;
    __shared__ int prefix[kMaxSeqs + 1 + kJoinMax];
    __shared__ float so[kJoinMax][DIM], sl[kJoinMax];
    make_prefix(r, prefix, prefix + kMaxSeqs + 1);
    const AttendParams& p = r.p;
    const int heads = p.c.kv_heads, group = p.a.q_heads / heads;
    const int seq = blockIdx.x / heads, head = blockIdx.x % heads, units = prefix[seq + 1] - prefix[seq];
    const int64_t run = run_length(static_cast<int64_t>(prefix[r.seqs]) * heads, r.workers);
    const int64_t begin = static_cast<int64_t>(prefix[seq]) * heads + static_cast<int64_t>(head) * units;
    // the runs that hold its first and its last step
    const int w0 = static_cast<int>((begin + kItem) / run), w1 = static_cast<int>((begin + units - 1) / run);
    const int slot0 = begin > w0 * run ? 1 : 0;
    const SeqSpan sp = attend_span(p, r.seq0 + seq);
    if (blockIdx.x == 0 && blockIdx.y == 0 && r.seq0 == 0) check_cu_q(p, threadIdx.x, blockDim.x);
    pdl_wait();   // the partial results are complete (and this kernel ends after the one before it)
    if (units == 0 || w0 == w1) return;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int rows = sp.n * group;
    const int share = min(warps, max(1, warps * static_cast<int>(gridDim.y) / rows));   // warps a row
    const int at_once = warps / share;                                                  // rows at once
    const float* ml = r.part + 2ll * r.workers * ROWS * DIM;
    for (int row0 = blockIdx.y * at_once; row0 < rows; row0 += at_once * gridDim.y) {
        const int row = row0 + warp / share, mine = warp % share;
        auto slot = [&](int w) { return (2ll * w + (w == w0 ? slot0 : 0)) * ROWS + row; };
        float m = -INFINITY, l = 0.f, o[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) o[i] = 0.f;
        const bool live = row < rows && warp / share < at_once;
        if (live) {
#pragma unroll 4
            for (int w = w0 + lane; w <= w1; w += 32) m = fmaxf(m, ml[slot(w) * 2]);
#pragma unroll
            for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll 8
            for (int w = w0 + mine; w <= w1; w += share) {
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
        }
        if (share > 1) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) so[warp][lane * kPer + i] = o[i];
            if (lane == 0) sl[warp] = l;
            __syncthreads();
            if (live && mine == 0)
                for (int w = 1; w < share; ++w) {
#pragma unroll
                    for (int i = 0; i < kPer; ++i) o[i] += so[warp + w][lane * kPer + i];
                    l += sl[warp + w];
                }
            __syncthreads();
        }
        if (live && mine == 0) {
            const int token = sp.first + row / group, q_head = head * group + row % group;
            const int64_t at = static_cast<int64_t>(token) * p.a.q_heads + q_head;
            const float inv = row_inverse(l);
#pragma unroll
            for (int i = 0; i < kPer; ++i) from_f32(o[i] * inv, static_cast<T*>(p.a.out)[at * DIM + lane * kPer + i]);
            if (p.a.lse && lane == 0) p.a.lse[at] = row_lse(m, l);
        }
    }
}

template <int DIM>
int workers_of(int rows) { return device_sms() * (rows == 8 ? Cfg<DIM, 8>::kWarps : Cfg<DIM, 16>::kWarps); }

int row_capacity(const AttendParams& p) { return p.a.max_q * (p.a.q_heads / p.c.kv_heads) <= 8 ? 8 : 16; }

template <typename T, int DIM, int ROWS>
int launch(const AttendParams& p, void* workspace, cudaStream_t st) {
    using C = Cfg<DIM, ROWS>;
    static PerDeviceOnce smem_once;
    int rc = set_smem_limit_once(smem_once, k_attend_rows<T, DIM, ROWS>, C::kSmem, "cudaFuncSetAttribute(k_attend_rows)");
    if (rc) return rc;
    CUtensorMap mk, mv;
    const uint64_t lines = static_cast<uint64_t>(p.c.pages) * p.c.kv_heads * p.c.page_tokens * DIM / 128;
    const uint32_t box = (p.c.page_tokens < kStep ? p.c.page_tokens : kStep) * DIM / 128;
    rc = make_map_2d(&mk, p.c.k, kMapU8, 128, lines, 128, 128, box, true);
    if (!rc) rc = make_map_2d(&mv, p.c.v, kMapU8, 128, lines, 128, 128, box, true);
    if (rc) return rc;
    RowsParams r{p, 0, 0, workers_of<DIM>(ROWS), static_cast<float*>(workspace)};
    // sequences a launch: the prefix array's room, and all their units in 31 bits
    const int64_t most = static_cast<int64_t>(p.b.table_width) * p.c.page_tokens / kStep + 2 + kItem;
    const int at_once = static_cast<int>(std::min<int64_t>(kMaxSeqs, 0x7fffffffll / most));
    for (; r.seq0 < p.b.n_seq; r.seq0 += at_once) {
        r.seqs = std::min(at_once, p.b.n_seq - r.seq0);
        k_attend_rows<T, DIM, ROWS><<<device_sms(), C::kWarps * 32, C::kSmem, st>>>(mk, mv, r);
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return set_cuda_error("k_attend_rows", e);
        cudaLaunchConfig_t cfg = {};
        const int items = r.seqs * p.c.kv_heads;
        cfg.gridDim = dim3(items, items * ROWS <= device_sms() ? ROWS : 1);
        // few items are cut into many runs each: more warps to read them
        cfg.blockDim = dim3(32 * (items > 4 * device_sms() ? 4 : items > device_sms() ? 8 : kJoinMax));
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
    const int rows = row_capacity(p);
    const int64_t workers = p.c.head_dim == 128 ? workers_of<128>(rows) : workers_of<64>(rows);
    return workers * 2 * rows * (p.c.head_dim + 2) * 4;
}

int launch_attend_rows(const AttendParams& p, void* workspace, cudaStream_t st) {
    return p.a.dtype == B3_DTYPE_F16 ? launch_type<__half>(p, workspace, st) : launch_type<__nv_bfloat16>(p, workspace, st);
}

}  // namespace b3
