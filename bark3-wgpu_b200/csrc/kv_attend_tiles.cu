// kv_attend_tiles.cu — attention over the paged 8-bit cache for many query
// rows: prompts, chunks of prompts, decode steps with more than 16 rows a key
// head.  The mathematics is in kv_attend.cuh.
//
// Bound by arithmetic: 4 head_dim operations a (row, key) pair on tcgen05 and
// one exponential, of which an SM makes 16 a clock, as long as 512 (head_dim
// 128) of its tensor operations.
//
// An item is 256 query rows (new token x head of the group, so K and V are
// read, expanded and staged once for all heads that share them) of one key
// head; it walks its keys in blocks of 128.  Its two halves of 128 rows take
// turns: while the softmax warps of one work on a block's scores, the tensor
// cores multiply for the other.
//   warps 0..3, 4..7   softmax of half 0 and 1: a thread owns a row, so the
//                      running maximum and sum need no exchange.  They stage
//                      the half's queries (f16, 128-byte swizzle), read the
//                      scores from TMEM twice (maximum, then exponentials),
//                      write P (f16) over them, move the reference maximum only
//                      when a row's grows by more than 2^8 (and then rescale O
//                      in TMEM), and store the output.
//   warps 8..14        expand codes to f16 operands in tasks of 16 keys: 16-byte
//                      loads of a page's rows two tasks ahead in registers, K
//                      and V both as 128-byte swizzled rows of 64 channels
//                      (K-major for S, MN-major for PV).
//   warp 15            one thread issues S = Q K^T (M128 N128 K128) and
//                      O += P V (M128 N128 K128, P from TMEM).
// TMEM: S/P of both halves 2 x 128 columns, O 2 x 128.
//
// Work.  k_attend_plan lists the items with their blocks; all blocks of all
// (item, key head) pairs, laid end to end with three more units for the start
// and end of each item (105 against 74 us for eight prompts without them), are
// cut into equal runs, one a CTA, so causal triangles, ragged prompts and few
// rows over many keys end together.  A run that covers an item from end to end stores it, other runs
// leave partial results that k_attend_tiles_join adds up in run order.
//
// Measured: 2048 tokens over 16384, 32 query and 8 key heads of 128, 583 us
// (884 TFLOP/s).  The chain softmax, PV, S of a half sets the pace: a half's
// softmax takes 3600 cycles a block beside the other half's, PV and S 1240.
// Reading the scores twice (593 us then) beat reading them once (794), two
// threads a row (648), exponentials by groups of 16 keys (619), 64-key blocks (713).
#include <type_traits>

#include "b3_ptx.cuh"
#include "kv_attend.cuh"

namespace b3 {
namespace {

constexpr int kRows = 256;          // query rows of an item
constexpr int kKeys = 128;          // keys of a block
// 16 warps, four on each scheduler: a 17th would cut every thread's registers from 128 to 96
constexpr int kThreads = 512;
constexpr int kExpWarp0 = 8, kExpWarps = 7, kMmaWarp = 15;
constexpr int kItem = 3;            // what an item's start and end cost, in blocks (measured on prompts of head_dim 64)
constexpr float kMove = 8.f;        // log2: how far a maximum may pass the reference

struct Tile {
    int seq, first, n, len;         // sequence, its first query row, new tokens, cached tokens
    int row0, steps, key_lo, pad;   // first query row of the item in the sequence, blocks, first key
    int64_t begin, pad2;            // units (of one key head) of the items before: kItem and an item's blocks
};

struct TilesParams {
    AttendParams p;
    int tiles;              // entries of `tile`; tile[tiles].begin is the total
    int runs;
    Tile* tile;
    float* part;            // [runs][2][kRows][DIM], then [runs][2][kRows][2] (m, l)
};

template <int DIM>
struct Cfg {
    static constexpr uint32_t kHalf = kKeys * 128;               // 64 channels of 128 rows (keys or queries)
    static constexpr uint32_t kOperand = kHalf * (DIM / 64);
    static constexpr uint32_t kQ = 0;                            // 2 halves of rows
    static constexpr uint32_t kK = 2 * kOperand;                 // 2 stages
    static constexpr uint32_t kV = 4 * kOperand;                 // 2 stages
    static constexpr uint32_t kBar = 6 * kOperand;
    static constexpr uint32_t kSmem = kBar + 256 + 1024;
    static constexpr uint32_t kTmemS = 0, kTmemO = 256;
    static constexpr uint32_t kIdescS = idesc_f16_f32_b<128, 128, 0>();
    static constexpr uint32_t kIdescPV = idesc_f16_f32_b<128, DIM, 1>();
};

// ───────────────────────────── the plan ─────────────────────────────

__global__ void __launch_bounds__(1024) k_attend_plan(const __grid_constant__ TilesParams r) {
    __shared__ int64_t sums[32];
    const AttendParams& p = r.p;
    const int group = p.a.q_heads / p.c.kv_heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    int64_t carry = 0;
    // items before sequence i's: cu_q[i] * group / kRows + i, room for every sequence's last, part-filled one
    auto key = [&](int i) { return static_cast<int64_t>(__ldg(p.b.cu_q + i)) * group / kRows + i; };
    for (int base = 0; base < r.tiles; base += 1024) {
        const int u = base + tid;
        Tile t = {};
        if (u < r.tiles) {
            int lo = 0, hi = p.b.n_seq;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (key(mid) <= u) lo = mid; else hi = mid;
            }
            const SeqSpan sp = attend_span(p, lo);
            const int64_t row0 = (u - key(lo)) * kRows;
            if (row0 >= 0 && row0 < static_cast<int64_t>(sp.n) * group) {
                t.seq = lo, t.first = sp.first, t.n = sp.n, t.len = sp.len;
                t.row0 = static_cast<int>(row0);
                const int last = static_cast<int>(min(row0 + kRows, static_cast<int64_t>(sp.n) * group)) - 1;
                int a, hi_key, lo_key;
                seen_keys(p, sp, t.row0 / group, lo_key, a);
                seen_keys(p, sp, last / group, a, hi_key);
                t.key_lo = min(lo_key, hi_key) / kKeys * kKeys;
                t.steps = max(1, (hi_key - t.key_lo + kKeys - 1) / kKeys);   // rows that see nothing are written too
            }
        }
        const int units = t.steps ? kItem + t.steps : 0;
        int64_t v = units;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += x;
        }
        if (lane == 31) sums[warp] = v;
        __syncthreads();
        int64_t before = carry, all = carry;
        for (int w = 0; w < 32; ++w) {
            before += w < warp ? sums[w] : 0;
            all += sums[w];
        }
        t.begin = before + v - units;
        if (u < r.tiles) r.tile[u] = t;
        carry = all;
        __syncthreads();
    }
    if (tid == 0) r.tile[r.tiles].begin = carry;
}

__device__ __forceinline__ int64_t run_length(int64_t total, int runs) {
    return max(static_cast<int64_t>(1), (total + runs - 1) / runs);
}

// Walks the items of a run: [s0, s1) are the blocks of the item in it.  All in
// units: an item has kItem of them and then its blocks.
struct Walk {
    const Tile* tile;
    int tiles, heads;
    int64_t start, at, upto, end;   // the run's first unit; this part's; the next part's; the run's end
    int u, head, s0, s1;
    Tile t;

    // the whole warp; false where the run has no blocks
    __device__ __forceinline__ bool init(const TilesParams& r, int run_id) {
        tile = r.tile;
        tiles = r.tiles;
        heads = r.p.c.kv_heads;
        const int64_t total = __ldg(&tile[tiles].begin) * heads, run = run_length(total, r.runs);
        at = start = run_id * run;
        end = min(at + run, total);
        if (at >= end) return false;
        // the last item that begins at or before `at` (items without blocks begin where the next one does)
        const int lane = threadIdx.x & 31;
        int lo = 0, len = tiles;
        while (len > 1) {
            const int step = (len + 31) >> 5, i = lane * step;
            const unsigned m = __ballot_sync(0xffffffffu, i < len && __ldg(&tile[lo + i].begin) * heads <= at);
            const int k = m ? (31 - __clz(m)) * step : 0;
            lo += k;
            len = min(step, len - k);
        }
        u = lo;
        load();
        const int64_t in = at - t.begin * heads;
        head = static_cast<int>(in / (t.steps + kItem));
        if (set(static_cast<int>(in % (t.steps + kItem)))) return true;
        return next();
    }
    __device__ __forceinline__ void load() {
        const int4* q = reinterpret_cast<const int4*>(tile + u);
        const int4 a = __ldg(q), b = __ldg(q + 1);
        t.seq = a.x, t.first = a.y, t.n = a.z, t.len = a.w, t.row0 = b.x, t.steps = b.y, t.key_lo = b.z;
        t.begin = __ldg(&tile[u].begin);
    }
    // the item's units from `from`; false where they hold no block
    __device__ __forceinline__ bool set(int from) {
        const int last = static_cast<int>(min(static_cast<int64_t>(t.steps + kItem), from + (end - at)));
        upto = at + last - from;
        s0 = max(0, from - kItem);
        s1 = last - kItem;
        return s1 > s0;
    }
    __device__ __forceinline__ bool next() {
        for (;;) {
            at = upto;
            if (at >= end) return false;
            if (++head == heads) {
                head = 0;
                do ++u; while (__ldg(&tile[u].steps) == 0);   // at < end: an item with blocks follows
                load();
            }
            if (set(0)) return true;
        }
    }
};

// ───────────────────────────── the kernel ─────────────────────────────

__device__ __forceinline__ uint32_t h2u(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t at) {
    uint4 x;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
    return x;
}

// NaN out of the f16 values that a lane has staged of a task of V: LOADS times
// 16 channels of every KEYS-th key; sets *seen if there was one.  Out of line:
// in line the compiler predicates it, and every task pays (2048 tokens over
// 16384 660 us instead of 595).
template <int LOADS, int KEYS>
__device__ __noinline__ void clean_v(uint32_t to, int sub, int c0, volatile uint32_t* seen) {
#pragma unroll 1
    for (int i = 0; i < 2 * LOADS; ++i) {
        const uint32_t at = to + (i >> 1) * KEYS * 128 + (((c0 + (i & 1)) ^ ((sub + (i >> 1) * KEYS) & 7)) << 4);
        uint4 x = lds128(at);
        auto nan = [](uint32_t two) { return ((two & 0x7fff7fffu) + 0x03ff03ffu) & 0x80008000u; };   // bit 15 of a half that is NaN
        const uint4 n = make_uint4(nan(x.x), nan(x.y), nan(x.z), nan(x.w));
        if (!(n.x | n.y | n.z | n.w)) continue;
        *seen = 1;
        sts128(at, x.x & ~((n.x >> 15) * 0xffffu), x.y & ~((n.y >> 15) * 0xffffu), x.z & ~((n.z >> 15) * 0xffffu),
               x.w & ~((n.w >> 15) * 0xffffu));
    }
}

// NaN back into row i of an item, where a key of the blocks [s0, s1) that the
// row sees holds it; a row a lane.  The row has been stored as output (slot < 0)
// or partial result.
template <typename T, int DIM>
__device__ __noinline__ void restore_nan(const TilesParams& r, const Tile& t, int head, int s0, int s1, int i, bool live, int64_t slot) {
    const AttendParams& p = r.p;
    const int group = p.a.q_heads / p.c.kv_heads, last = min(t.row0 + kRows, t.n * group) - 1, row = min(t.row0 + i, last);
    const SeqSpan sp = {t.first, t.n, t.len};
    const SeenByRows see = seen_by_rows(p, sp, t.row0 / group, last / group);
    int lo, hi;
    seen_keys(p, sp, row / group, lo, hi);
    uint32_t mask[DIM / 32] = {};
    for (int j = s0; j < s1; ++j) {
        const int key = t.key_lo + j * kKeys;
        if (see.split(key, kKeys))
            nan_channels<DIM>(p, t.seq, head, max(key, see.any_lo), min(key + kKeys, see.any_hi), lo, hi, mask);
    }
    if (live && slot < 0)
        put_nan<DIM>(static_cast<T*>(p.a.out) +
                         (static_cast<int64_t>(t.first + row / group) * p.a.q_heads + head * group + row % group) * DIM, mask);
    else if (live)
        put_nan<DIM>(r.part + (slot * kRows + i) * DIM, mask);
}

template <typename T, int DIM>
__global__ void __launch_bounds__(kThreads, 1) k_attend_tiles(const __grid_constant__ TilesParams r) {
    using C = Cfg<DIM>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const AttendParams& p = r.p;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Barriers.  k, v: two stages each, phases over the CTA's blocks; q: a half's
    // queries are staged (an item); s: a half's scores are in TMEM, p: its
    // probabilities of the first 64 keys, and of all, are (a block; PV starts on
    // the first while the softmax is at the rest); o: its last product is done
    // (an item).
    const uint32_t bars = smem_u32(smem + C::kBar);
    auto k_full = [&](int s) { return bars + 8 * s; };
    auto k_empty = [&](int s) { return bars + 16 + 8 * s; };
    auto v_full = [&](int s) { return bars + 32 + 8 * s; };
    auto v_empty = [&](int s) { return bars + 48 + 8 * s; };
    auto q_full = [&](int h) { return bars + 64 + 8 * h; };
    auto s_full = [&](int h) { return bars + 80 + 8 * h; };
    auto p_half = [&](int h) { return bars + 96 + 8 * h; };
    auto p_full = [&](int h) { return bars + 112 + 8 * h; };
    auto o_full = [&](int h) { return bars + 128 + 8 * h; };
    const uint32_t drained = bars + 144;   // after a wait that ran out: every product issued is done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kBar + 160);
    // set when NaN codes of V have gone into a product as 0: before v_full of their block, read behind o_full
    volatile uint32_t* nan_seen = reinterpret_cast<uint32_t*>(smem + C::kBar + 164);
    if (threadIdx.x == 0) {
        *nan_seen = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full(i), 8);
            mbar_init(v_full(i), 8);
            mbar_init(k_empty(i), 1);
            mbar_init(v_empty(i), 1);
            mbar_init(q_full(i), 4);
            mbar_init(s_full(i), 1);
            mbar_init(p_half(i), 4);
            mbar_init(p_full(i), 4);
            mbar_init(o_full(i), 1);
        }
        mbar_init(drained, 1);
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc<512>(smem_u32(tmem_slot));
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    pdl_wait();   // the plan is complete

    const int group = p.a.q_heads / p.c.kv_heads, heads = p.c.kv_heads, page = p.c.page_tokens;
    const int log_page = 31 - __clz(page);
    Walk w;
    const bool any = w.init(r, blockIdx.x);
    auto halves = [&]() { return w.t.n * group - w.t.row0 > 128 ? 2 : 1; };
    bool ok = any;

    if (!any) {
        // no run for this CTA
    } else if (warp == kMmaWarp) {
        // ── MMA issuer ──
        if (lane == 0) {
            const uint32_t sq = smem_u32(smem + C::kQ), sk = smem_u32(smem + C::kK), sv = smem_u32(smem + C::kV);
            uint32_t g = 0, items[2] = {0, 0}, blocks[2] = {0, 0};   // blocks of the CTA; items and blocks of each half
            auto scores = [&](int h, uint32_t gb) {   // S of half h for the CTA's block gb
                const uint64_t a0 = smem_desc_sw128(sq + h * C::kOperand), b0 = smem_desc_sw128(sk + (gb & 1) * C::kOperand);
#pragma unroll
                for (int k = 0; k < DIM / 16; ++k) {
                    const uint32_t off = (k >> 2) * C::kHalf + (k & 3) * 32;
                    mma_f16_ss(tmem + C::kTmemS + 128 * h, desc_advance(a0, off), desc_advance(b0, off), C::kIdescS, k > 0);
                }
                mma_commit(s_full(h));
            };
            do {
                const int nh = halves(), n = w.s1 - w.s0;
                for (int h = 0; h < nh && ok; ++h) {
                    ok = mbar_wait(q_full(h), items[h] & 1, 0x70);
                    ++items[h];
                    if (ok && h == 0) ok = mbar_wait(k_full(g & 1), (g >> 1) & 1, 0x71);
                    if (!ok) break;
                    tc_fence_after();
                    scores(h, g);
                }
                if (ok) mma_commit(k_empty(g & 1));
                for (int j = 0; j < n && ok; ++j, ++g) {
                    const uint32_t st = g & 1;
                    for (int h = 0; h < nh && ok; ++h) {
                        const uint64_t bv = smem_desc_sw128_mn(sv + st * C::kOperand, C::kHalf, 1024);
                        for (int part = 0; part < 2 && ok; ++part) {   // 64 keys each
                            ok = mbar_wait(part ? p_full(h) : p_half(h), blocks[h] & 1, 0x72);
                            if (ok && h == 0 && part == 0) ok = mbar_wait(v_full(st), (g >> 1) & 1, 0x73);
                            if (!ok) break;
                            tc_fence_after();
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                mma_f16_ts(tmem + C::kTmemO + 128 * h, tmem + C::kTmemS + 128 * h + 32 * part + 8 * k,
                                           desc_advance(bv, 8192 * part + 2048 * k), C::kIdescPV, j > 0 || part > 0 || k > 0);
                        }
                        if (!ok) break;
                        ++blocks[h];
                        if (h == nh - 1) mma_commit(v_empty(st));
                        if (j == n - 1) mma_commit(o_full(h));
                        if (j + 1 < n) {
                            if (h == 0) {
                                ok = mbar_wait(k_full((g + 1) & 1), ((g + 1) >> 1) & 1, 0x74);
                                if (!ok) break;
                                tc_fence_after();
                            }
                            scores(h, g + 1);   // over P of this block: the products run in order
                            if (h == nh - 1) mma_commit(k_empty((g + 1) & 1));
                        }
                    }
                }
            } while (ok && w.next());
            if (!ok) {
                kv_flag(p.c.status, B3_KV_TIMEOUT);
                // products in flight still read and write the memory that the block gives back
                mma_commit(drained);
                mbar_wait(drained, 0, 0x7A);
            }
        }
    } else if (warp >= kExpWarp0) {
        // ── codes to f16 operands ──
        // Tasks of 16 keys of K or V: the eight of a block's K, then of its V, dealt out to the warps in
        // turn, so 16 keys are one page and one table entry.  A task's loads are two tasks ahead of its
        // stores.  A load of a warp covers four keys x 128 bytes (eight x 64); a lane takes 16 bytes, the
        // lanes of a quarter-warp four pieces of 64 channels of two keys, so that the swizzled 16-byte
        // stores of each quarter touch every bank once.
        constexpr int kLoads = DIM / 32;                   // loads a thread and task
        constexpr int kKeysLoad = 16 / kLoads;             // keys of a load
        const int piece = DIM == 128 ? (lane & 3) + 4 * ((lane >> 3) & 1) : lane & 3;   // 16 channels
        const int sub = DIM == 128 ? ((lane >> 2) & 1) + 2 * (lane >> 4) : lane >> 2;
        const uint32_t dst = smem_u32(smem) + (piece >> 2) * C::kHalf + sub * 128;
        const int c0 = 2 * (piece & 3);
        uint32_t block = 0;
        // of the item that the loads are at: keys that some row sees; its blocks before and from which rows see
        // different keys (SeenByRows::split)
        int any_lo, any_hi, split_lo, split_hi;
        const int32_t* pages;
        auto item = [&]() {
            const SeqSpan sp = {w.t.first, w.t.n, w.t.len};
            const SeenByRows see = seen_by_rows(p, sp, w.t.row0 / group, (min(w.t.row0 + kRows, w.t.n * group) - 1) / group);
            any_lo = see.any_lo, any_hi = see.any_hi;
            const bool differ = see.split(see.hi_min, kKeys);
            split_lo = differ ? (see.lo_max - w.t.key_lo + kKeys - 1) / kKeys : 0;
            split_hi = differ ? (see.hi_min - w.t.key_lo) / kKeys : 0x7fffffff;
            pages = p.b.page_table + w.t.seq * p.b.table_stride;
        };
        item();
        bool more = true;
        enum { kNone, kPlain, kSplitV };
        auto fetch = [&](uint32_t q, uint4 (&c)[kLoads]) -> int {   // kNone where the run has no such task
            if ((q >> 4) != block && more) {
                ++block;
                if (++w.s0 == w.s1) {
                    more = w.next();
                    if (more) item();
                }
            }
            if (!more) return kNone;
            const int key = w.t.key_lo + w.s0 * kKeys + 16 * (q & 7);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) c[i] = make_uint4(0, 0, 0, 0);   // a key that no row sees: 0, whatever its place holds
            if (key + 16 > any_lo && key < any_hi) {
                int id = __ldg(pages + (key >> log_page));
                if (id < 0 || id >= p.c.pages) {
                    kv_flag(p.c.status, B3_KV_BAD_PAGE);
                    id = 0;
                }
                const int line = (id * heads + w.head) * page + (key & (page - 1)) + sub;
                const uint8_t* from = ((q & 8) ? p.c.v : p.c.k) + static_cast<int64_t>(line) * DIM + 16 * piece;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int k = key + sub + i * kKeysLoad;
                    if (k >= any_lo && k < any_hi) c[i] = __ldg(reinterpret_cast<const uint4*>(from + i * kKeysLoad * DIM));
                }
            }
            return (q & 8) && (w.s0 < split_lo || w.s0 >= split_hi) ? kSplitV : kPlain;
        };
        auto expand = [&](uint32_t q, const uint4 (&c)[kLoads], int kind) {
            const uint32_t g = q >> 4, st = g & 1, v = (q >> 3) & 1, key = 16 * (q & 7);
            if (g >= 2) ok = __all_sync(0xffffffffu, mbar_wait(v ? v_empty(st) : k_empty(st), ((g >> 1) - 1) & 1, 0x75));
            if (!ok) return;
            const uint32_t to = dst + (v ? C::kV : C::kK) + st * C::kOperand + key * 128;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t in[4] = {c[i].x, c[i].y, c[i].z, c[i].w};
                uint32_t out[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const __half2 a = decode2(in[k] & 0xffffu), b = decode2(in[k] >> 16);
                    out[2 * k] = *reinterpret_cast<const uint32_t*>(&a);
                    out[2 * k + 1] = *reinterpret_cast<const uint32_t*>(&b);
                }
                const int sw = (sub + i * kKeysLoad) & 7;
                sts128(to + i * kKeysLoad * 128 + ((c0 ^ sw) << 4), out[0], out[1], out[2], out[3]);
                sts128(to + i * kKeysLoad * 128 + (((c0 + 1) ^ sw) << 4), out[4], out[5], out[6], out[7]);
            }
            if (kind == kSplitV) clean_v<kLoads, kKeysLoad>(to, sub, c0, nan_seen);
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(v ? v_full(st) : k_full(st));
        };
        uint4 ca[kLoads], cb[kLoads];
        const uint32_t first = warp - kExpWarp0;
        int a = fetch(first, ca), b = a != kNone ? fetch(first + kExpWarps, cb) : kNone;
        for (uint32_t q = first; a != kNone && ok; q += 2 * kExpWarps) {
            expand(q, ca, a);
            if (!ok || b == kNone) break;
            a = fetch(q + 2 * kExpWarps, ca);
            expand(q + kExpWarps, cb, b);
            if (!ok) break;
            b = a != kNone ? fetch(q + 3 * kExpWarps, cb) : kNone;
        }
        if (!ok && lane == 0) kv_flag(p.c.status, B3_KV_TIMEOUT);
    } else {
        // ── softmax: half h, a row a thread ──
        const int h = warp >> 2, mine = (warp & 3) * 32 + lane;
        const uint32_t lrow = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + lrow + C::kTmemS + 128 * h, to = tmem + lrow + C::kTmemO + 128 * h;
        uint8_t* sq = smem + C::kQ + h * C::kOperand + mine * 128;
        const bool vec = ((reinterpret_cast<uintptr_t>(p.a.q) | (p.a.q_token_stride * 2) | (p.a.q_head_stride * 2)) & 15) == 0;
        float qscale = 0.f;
        // stages this thread's query row of the walk's item
        auto stage = [&]() {
            const int row = w.t.row0 + 128 * h + mine;
            const bool live = row < w.t.n * group;
            const T* q = static_cast<const T*>(p.a.q) + static_cast<int64_t>(w.t.first + (live ? row / group : 0)) * p.a.q_token_stride +
                         static_cast<int64_t>(w.head * group + (live ? row % group : 0)) * p.a.q_head_stride;
            auto piece = [&](int c, float (&x)[8]) {
                if (vec)
                    load8<true>(q + 8 * c, x);
                else
                    load8<false>(q + 8 * c, x);
            };
            const float sign = p.a.scale < 0.f ? -1.f : 1.f;   // scores are scaled by what is positive: order is kept
            int shift = 0;
            if (live && !std::is_same<T, __half>::value) {
                float amax = 0.f;
                for (int c = 0; c < DIM / 8; ++c) {
                    float x[8];
                    piece(c, x);
#pragma unroll
                    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
                }
                shift = row_shift(amax);
            }
            const float mul = sign * exp2_int(shift);
            qscale = fabsf(p.a.scale) * kLog2e * exp2_int(-shift);
#pragma unroll 4
            for (int c = 0; c < DIM / 8; ++c) {
                float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (live) piece(c, x);
                *reinterpret_cast<uint4*>(sq + (c >> 3) * C::kHalf + (((c & 7) ^ (mine & 7)) << 4)) =
                    make_uint4(h2u(x[0] * mul, x[1] * mul), h2u(x[2] * mul, x[3] * mul), h2u(x[4] * mul, x[5] * mul),
                               h2u(x[6] * mul, x[7] * mul));
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full(h));
        };
        uint32_t items = 0, blocks = 0;
        bool more = true, mine_next = halves() > h;
        if (mine_next) stage();
        while (ok && more) {
            if (!mine_next) {   // an item without a second half
                more = w.next();
                mine_next = more && halves() > h;
                if (mine_next) stage();
                continue;
            }
            const Tile t = w.t;
            const int head = w.head, s0 = w.s0, s1 = w.s1;
            const SeqSpan sp = {t.first, t.n, t.len};
            const int rows = min(128, t.n * group - t.row0 - 128 * h);
            const int row = t.row0 + 128 * h + min(mine, rows - 1);
            int row_lo, row_hi, any_lo, any_hi, x;
            seen_keys(p, sp, row / group, row_lo, row_hi);
            const SeenByRows half = seen_by_rows(p, sp, (t.row0 + 128 * h) / group, (t.row0 + 128 * h + rows - 1) / group);
            seen_keys(p, sp, t.row0 / group, any_lo, x);
            seen_keys(p, sp, (min(t.row0 + kRows, t.n * group) - 1) / group, x, any_hi);
            const int32_t* pages = p.b.page_table + t.seq * p.b.table_stride;
            // lane i (0..7) brings the scales of the block's keys [16 i, 16 i + 16)
            auto scales = [&](int block, float& ks, int& ve) {
                const int key = t.key_lo + block * kKeys + 16 * (lane & 7);
                ks = 1.f;
                ve = 0;
                if (block < s1 && key + 16 > any_lo && key < any_hi) {
                    int id = __ldg(pages + (key >> log_page));
                    if (id < 0 || id >= p.c.pages) id = 0;   // flagged by the expanding warps
                    ks = __ldg(p.c.k_scale + static_cast<int64_t>(id) * heads + head);
                    ve = stored_exp(__ldg(p.c.v_scale + static_cast<int64_t>(id) * heads + head));
                }
            };
            float ks, ks_next;
            int ve, ve_next;
            scales(s0, ks_next, ve_next);
            float m = -INFINITY, l = 0.f;
            const float qs = qscale;
            auto factor = [&](float k) { return fminf(fmaxf(qs * k, 1e-37f), 3.4e38f); };   // finite and positive
            for (int j = s0; j < s1; ++j) {
                ks = ks_next, ve = ve_next;
                scales(j + 1, ks_next, ve_next);
                ok = __all_sync(0xffffffffu, mbar_wait(s_full(h), blocks & 1, 0x77));
                ++blocks;
                if (!ok) break;
                tc_fence_after();
                const int key = t.key_lo + j * kKeys;
                if (!half.whole(key, kKeys)) {   // scores of keys that a row does not see become -inf in TMEM
#pragma unroll 1
                    for (int c = 0; c < 4; ++c) {
                        const int from = row_lo - key - 32 * c, to_ = row_hi - key - 32 * c;
                        if (__all_sync(0xffffffffu, from <= 0 && to_ >= 32)) continue;
                        uint32_t a[32];
                        tmem_ld_32x32b_x32(ts + 32 * c, a);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (i < from || i >= to_) a[i] = 0xff800000u;
                        tmem_st_32x32b_x32(ts + 32 * c, a);
                    }
                    tmem_wait_st();
                }
                // maximum: of the raw products in each 16 keys, then scaled (the factor is positive)
                float top = -INFINITY;
                uint32_t a[2][32];
                tmem_ld_32x32b_x32(ts, a[0]);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    tmem_wait_ld();
                    if (c < 3) tmem_ld_32x32b_x32(ts + 32 * (c + 1), a[(c + 1) & 1]);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float f = factor(__shfl_sync(0xffffffffu, ks, 2 * c + u));
                        const float e = static_cast<float>(__shfl_sync(0xffffffffu, ve, 2 * c + u));
                        float g0 = -INFINITY, g1 = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            g0 = fmaxf(g0, __uint_as_float(a[c & 1][16 * u + i]));
                            g1 = fmaxf(g1, __uint_as_float(a[c & 1][16 * u + i + 1]));
                        }
                        top = fmaxf(top, fmaf(fmaxf(g0, g1), f, e));
                    }
                }
                tmem_ld_32x32b_x32(ts, a[0]);   // again, for the exponentials
                const bool grow = top > m + kMove || (m == -INFINITY && top > -INFINITY);
                if (__any_sync(0xffffffffu, grow)) {
                    const float m_new = grow ? top : m;
                    const float corr = m_new == m ? 1.f : ex2_approx(m - m_new);
                    m = m_new;
                    l *= corr;
                    if (j > s0) {   // the products so far are done: S was issued after them
#pragma unroll 1
                        for (int c = 0; c < DIM / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld_32x32b_x16(to + 16 * c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                            tmem_st_32x32b_x16(to + 16 * c, o);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t b[16];
                    tmem_wait_ld();
                    if (c < 3) tmem_ld_32x32b_x32(ts + 32 * (c + 1), a[(c + 1) & 1]);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const float f = factor(__shfl_sync(0xffffffffu, ks, 2 * c + u));
                        const int ei = __shfl_sync(0xffffffffu, ve, 2 * c + u);
                        const float e = static_cast<float>(ei) - ref;
                        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float2 y = __ffma2_rn(make_float2(__uint_as_float(a[c & 1][16 * u + i]),
                                                              __uint_as_float(a[c & 1][16 * u + i + 1])),
                                                  make_float2(f, f), make_float2(e, e));
                            y = make_float2(ex2_approx(y.x), ex2_approx(y.y));
                            sum = __fadd2_rn(sum, y);
                            b[8 * u + (i >> 1)] = h2u(y.x, y.y);
                        }
                        l = fmaf(sum.x + sum.y, exp2_int(-ei), l);
                    }
                    tmem_st_32x32b_x16(ts + 16 * c, b);   // over scores that were read
                    if (c == 1) {                         // the first 64 keys' probabilities are there
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_half(h));
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(h));
            }
            if (!ok) break;
            // the next item's queries, then this one's output
            const int64_t slot = 2ll * blockIdx.x + (w.at > w.start ? 1 : 0);
            more = w.next();
            mine_next = more && halves() > h;
            if (mine_next) stage();
            ok = __all_sync(0xffffffffu, mbar_wait(o_full(h), items & 1, 0x78));
            ++items;
            if (!ok) break;
            tc_fence_after();
            const bool all = s0 == 0 && s1 == t.steps, live = mine < rows;
            const int token = t.first + row / group, q_head = head * group + row % group;
            const float inv = row_inverse(l);
            T* out = static_cast<T*>(p.a.out) + (static_cast<int64_t>(token) * p.a.q_heads + q_head) * DIM;
            float* po = r.part + (slot * kRows + 128 * h + mine) * DIM;
            float* ml = r.part + 2ll * r.runs * kRows * DIM + (slot * kRows + 128 * h + mine) * 2;
#pragma unroll
            for (int c = 0; c < DIM / 32; ++c) {
                uint32_t a[32];
                tmem_ld_32x32b_x32(to + 32 * c, a);
                tmem_wait_ld();
                if (live && all) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float x8[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) x8[k] = __uint_as_float(a[i + k]) * inv;
                        store8(out + 32 * c + i, x8);
                    }
                } else if (live) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4*>(po + 32 * c + i) = make_uint4(a[i], a[i + 1], a[i + 2], a[i + 3]);
                }
            }
            tc_fence_before();
            if (live && all) {
                if (p.a.lse) p.a.lse[static_cast<int64_t>(token) * p.a.q_heads + q_head] = row_lse(m, l);
            } else if (live) {
                *reinterpret_cast<float2*>(ml) = make_float2(m, l);
            }
            if (__any_sync(0xffffffffu, *nan_seen))   // by this item or one before: each row gets its NaN back
                restore_nan<T, DIM>(r, t, head, s0, s1, 128 * h + mine, live, all ? -1 : slot);
        }
        if (!ok && lane == 0) kv_flag(p.c.status, B3_KV_TIMEOUT);
    }

    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc<512>(tmem);
    }
}

// Adds up partial results: block (w, y) takes 32 rows, four a warp at once, of
// the item that starts in run w and goes on past it.
template <typename T, int DIM>
__global__ void __launch_bounds__(256) k_attend_tiles_join(const __grid_constant__ TilesParams r) {
    constexpr int kPer = DIM / 32;
    const AttendParams& p = r.p;
    // beside the tiles; inputs of the call, which were there before its first kernel
    if (blockIdx.x == 0 && blockIdx.y == 0) check_cu_q(p, threadIdx.x, blockDim.x);
    pdl_wait();
    const int heads = p.c.kv_heads, group = p.a.q_heads / heads;
    const int64_t total = __ldg(&r.tile[r.tiles].begin) * heads, run = run_length(total, r.runs);
    const int w0 = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t edge = (w0 + 1) * run;
    if (edge >= total) return;
    const int64_t want = edge - 1;
    int lo = 0, len = r.tiles;
    while (len > 1) {
        const int step = (len + 31) >> 5, i = lane * step;
        const unsigned m = __ballot_sync(0xffffffffu, i < len && __ldg(&r.tile[lo + i].begin) * heads <= want);
        const int k = m ? (31 - __clz(m)) * step : 0;
        lo += k;
        len = min(step, len - k);
    }
    const Tile t = r.tile[lo];
    const int units = t.steps + kItem, head = static_cast<int>((want - t.begin * heads) / units);
    const int64_t begin = t.begin * heads + static_cast<int64_t>(head) * units;
    // the runs that hold its first and its last block
    if ((begin + kItem) / run != w0 || begin + units <= edge) return;
    const int w1 = static_cast<int>((begin + units - 1) / run);
    const int slot0 = begin > w0 * run ? 1 : 0;
    const float* ml = r.part + 2ll * r.runs * kRows * DIM;
    const int i0 = 32 * blockIdx.y + 4 * warp, row0 = t.row0 + i0, rows = min(4, t.n * group - row0);
    if (rows <= 0) return;
    float m[4], l[4], o[4][kPer];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < kPer; ++c) o[i][c] = 0.f;
    }
    // an item is rarely in more than three runs: the reference moves along
    for (int w = w0; w <= w1; ++w) {
        const int64_t at = (2ll * w + (w == w0 ? slot0 : 0)) * kRows + i0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i >= rows) break;
            const float2 x = *reinterpret_cast<const float2*>(ml + (at + i) * 2);
            const float top = fmaxf(m[i], x.x), ref = top == -INFINITY ? 0.f : top;
            const float old = ex2_approx(m[i] - ref), f = ex2_approx(x.x - ref);
            l[i] = fmaf(x.y, f, l[i] * old);
#pragma unroll
            for (int c = 0; c < kPer; ++c) o[i][c] = fmaf(r.part[(at + i) * DIM + 32 * c + lane], f, o[i][c] * old);
            m[i] = top;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= rows) break;
        const int row = row0 + i;
        const int64_t at = static_cast<int64_t>(t.first + row / group) * p.a.q_heads + head * group + row % group;
#pragma unroll
        for (int c = 0; c < kPer; ++c) from_f32(o[i][c] * row_inverse(l[i]), static_cast<T*>(p.a.out)[at * DIM + 32 * c + lane]);
        if (p.a.lse && lane == 0) p.a.lse[at] = row_lse(m[i], l[i]);
    }
}

int64_t tile_count(const AttendParams& p) {
    return static_cast<int64_t>(p.b.tokens) * (p.a.q_heads / p.c.kv_heads) / kRows + p.b.n_seq;
}
int64_t tile_bytes(const AttendParams& p) { return ((tile_count(p) + 1) * static_cast<int64_t>(sizeof(Tile)) + 255) / 256 * 256; }

template <typename T, int DIM>
int launch(const AttendParams& p, void* workspace, cudaStream_t st) {
    using C = Cfg<DIM>;
    static PerDeviceOnce smem_once;
    const int rc = set_smem_limit_once(smem_once, k_attend_tiles<T, DIM>, C::kSmem, "cudaFuncSetAttribute(k_attend_tiles)");
    if (rc) return rc;
    if (tile_count(p) > 0x7ffffffell) return set_error(B3_EINVAL, "b3_kv_attend: too many tokens for one call");
    TilesParams r{p, static_cast<int>(tile_count(p)), device_sms(), static_cast<Tile*>(workspace),
                  reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + tile_bytes(p))};
    k_attend_plan<<<1, 1024, 0, st>>>(r);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error("k_attend_plan", e);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(r.runs);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, k_attend_tiles<T, DIM>, r);
    if (e != cudaSuccess) return set_cuda_error("k_attend_tiles", e);
    cfg.gridDim = dim3(r.runs, kRows / 32);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, k_attend_tiles_join<T, DIM>, r);
    return e == cudaSuccess ? 0 : set_cuda_error("k_attend_tiles_join", e);
}

}  // namespace

int64_t attend_tiles_workspace(const AttendParams& p) {
    return tile_bytes(p) + static_cast<int64_t>(device_sms()) * 2 * kRows * (p.c.head_dim + 2) * 4;
}

int launch_attend_tiles(const AttendParams& p, void* workspace, cudaStream_t st) {
    if (p.a.dtype == B3_DTYPE_F16)
        return p.c.head_dim == 128 ? launch<__half, 128>(p, workspace, st) : launch<__half, 64>(p, workspace, st);
    return p.c.head_dim == 128 ? launch<__nv_bfloat16, 128>(p, workspace, st) : launch<__nv_bfloat16, 64>(p, workspace, st);
}

}  // namespace b3
