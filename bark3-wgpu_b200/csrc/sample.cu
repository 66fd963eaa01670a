// sample.cu — b3_sample: the next token of every row of logits by temperature,
// top-k, top-p and min-p from a given random number.
//
//   w_i = exp((l_i - m) / T) as a whole number of 2^-31 (W_i),  sums exact
// Sums of whole numbers do not depend on their order, so the answer is the
// same however a row is split over threads and blocks.  The kept tokens are a
// beginning of the order (falling logit, rising index); the answer is the
// first kept token, by index, at which the running sum of W passes u times the
// total.
//
// A row is read once, into the shared memory of a cluster of 1 to 8 blocks of
// 512 threads (a column of vectors for each thread, in their own type, touched
// by it alone; a warp's values are neighbours in the row, in index order over
// (vector, lane, place)).  Shared memory and not registers: loops over 32
// values unrolled with an exponential in each miss the instruction cache.
// Bound by instructions for many rows (55 a value on average, at 0.57 of the
// issue rate), by the chain of block- and cluster-wide steps for few.  Measured,
// settings of each kind mixed: 256 rows x 131072 in 16 bits 125 us (one read takes
// 10), 256 x 8193 in f32 24, one row 11; all rows of one kind, 131072 and 8193:
// no filter 81 and 11, top-k 50 89 and 13, top-k 5000 173 and 23, top-p 197 and
// 26, greedy 41 and 6.
//   top_k <= 512   Each warp's j-th largest thread maximum, j = ceil(k / warps),
//                  bounds the k-th largest logit from below (the warps hold k
//                  values that large); what reaches the bound, a few hundred
//                  candidates, goes to a list in the first block, which ranks
//                  it by counting and does the rest alone: no weight of the
//                  row's bulk is ever computed.
//   top_p, larger  A histogram of weights (or counts) over 2048 steps of
//   top_k          l_i below the largest, to where weights end at 2^-31: a
//                  bell of logits spreads over hundreds of bins, so atomics
//                  rarely meet.  The members of the bin where the sum reaches
//                  its goal go to the list and are ranked; what is kept is then
//                  one comparison with the last kept (logit, index).
//   long ties      A list that overflows (thousands of equal logits) falls back
//                  to a search over the bits of (logit, index).
#include <cooperative_groups.h>

#include <type_traits>

#include "kv_cache.cuh"

namespace cg = cooperative_groups;

namespace b3 {
namespace {

using u32 = uint32_t;
using u64 = unsigned long long;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBlocks = 8;        // of a cluster: the portable limit
constexpr int kList = 2048;          // candidates
constexpr int kBins = 2048;
constexpr int kMostValues = 64;      // of a thread
constexpr int kTopList = 512;        // top_k up to here ranks candidates: one a thread afterwards

struct Shared {
    union {
        struct {
            u64 key[kList];              // (order of the logit, ~index)
            u32 weight[kList];           // by rank
        } list;
        struct {
            u32 lo[kBins], hi[kBins];    // sums of W's lower and upper 16 bits (or counts and nothing)
        } hist;
    };
    u64 warp_sum[kWarps];
    u64 vec_sum[kWarps][kMostValues / 4];   // a warp's sums of each of its vectors
    float warp_f[2 * kWarps];
    // written by the other blocks of the cluster
    float peak[kMaxBlocks], bound[kMaxBlocks];
    u64 part[2][kMaxBlocks];
    u64 cut_before, cut_key;
    int cut_bin, count, best;
};

// Order-preserving bits of a logit: larger logits, larger keys; -0 = +0.
__device__ __forceinline__ u32 key_of(float x) {
    const u32 b = __float_as_uint(x == 0.f ? 0.f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(u32 key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ u64 rank_key(float x, int i) { return static_cast<u64>(key_of(x)) << 32 | static_cast<u32>(~i); }

// exp((x - peak) / t) with the division rounded as IEEE's.  inv = 1 / t
// correctly rounded: then q = a inv is next to a / t, r = a - q t is exact in
// one fused multiply-add, and q + r inv is a / t correctly rounded unless t's
// significand is all ones (P. Markstein, "Computation of elementary functions
// on the IBM RISC System/6000 processor", 1990); such t, and ones so far out
// that a residual could leave the normal range, are divided by.
struct Weigh {
    float peak, t, inv, least;
    bool divide, infinite;
    __device__ __forceinline__ void set(float p, float temperature) {
        peak = p;
        t = temperature;
        inv = __frcp_rn(t);
        least = -64.f * t;   // exp(-64) is no weight: what is further down is held here
        divide = (__float_as_uint(t) & 0x7fffffu) == 0x7fffffu || !(t > 0x1p-60f && t < 0x1p60f);
        infinite = peak == INFINITY;
    }
    // the usual row: no branch and no division, in loops over all values
    __device__ __forceinline__ bool usual() const { return !divide && !infinite; }
    __device__ __forceinline__ float usual_power(float x) const {
        const float a = fmaxf(x - peak, least), q = a * inv;
        return fmaf(fmaf(-q, t, a), inv, q);
    }
    __device__ __forceinline__ float power(float x) const {
        if (infinite) return x == peak ? 0.f : -INFINITY;
        return divide ? (x - peak) / t : usual_power(x);
    }
    template <bool USUAL>
    __device__ __forceinline__ float weight(float x) const { return expf(USUAL ? usual_power(x) : power(x)); }
};
__device__ __forceinline__ u32 whole(float w) { return static_cast<u32>(w * 2147483648.f); }

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
// Inclusive sums over the block's threads; `all` their total.
__device__ __forceinline__ u64 block_scan(u64 v, u64* sums, u64& all) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += x;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    u64 before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        before += w < warp ? sums[w] : 0;
        all += sums[w];
    }
    return before + v;
}

template <typename T>
struct Row {
    static constexpr int kVec = 16 / sizeof(T);      // values of a load
    const T* x;            // the row
    int n, off;            // off: values from the 16-byte boundary before the row to its start
    int base;              // place of this thread's first value
    int count;             // values a thread, a multiple of kVec
    bool by_one;           // values one by one: off is 0 wherever the row starts
    // place of value e: index + off
    __device__ __forceinline__ int index(int e) const { return base + (e / kVec) * 32 * kVec + e % kVec - off; }

    // The thread's values into its column, their maximum; what is no number, or outside the row, is -inf.
    __device__ __forceinline__ float load(uint4* col) const {
        T least;
        from_f32(-INFINITY, least);
        float top = -INFINITY;
        constexpr int kAhead = 8;      // vectors in flight
        for (int c0 = 0; c0 < count; c0 += kAhead * kVec) {
            uint4 raw[kAhead];
#pragma unroll
            for (int c = 0; c < kAhead; ++c) {
                const int e = c0 + c * kVec, i = index(e);
                if (e < count && i >= 0 && i + kVec <= n && !by_one) raw[c] = __ldcs(reinterpret_cast<const uint4*>(x + i));
            }
#pragma unroll
            for (int c = 0; c < kAhead; ++c) {
                const int e = c0 + c * kVec, i = index(e);
                if (e >= count) break;
                const bool vector = i >= 0 && i + kVec <= n && !by_one;
                T* t = reinterpret_cast<T*>(&raw[c]);
#pragma unroll
                for (int k = 0; k < kVec; ++k) {
                    if (!vector) t[k] = i + k >= 0 && i + k < n ? x[i + k] : least;
                    const float f = to_f32(t[k]);
                    top = fmaxf(top, f);
                    if (f != f) t[k] = least;
                }
                col[e / kVec * kThreads] = raw[c];
            }
        }
        return top;
    }
};

// Ranks of the list's entries, largest key first: entry i of thread `tid`,
// tid + 512, ... ; f(rank, key).  Keys differ.
template <typename F>
__device__ __forceinline__ void rank_list(const u64* key, int n, F f) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const u64 mine = key[i];
        int rank = 0;
        int j = 0;
        for (; j + 4 <= n; j += 4)
            rank += (key[j] > mine) + (key[j + 1] > mine) + (key[j + 2] > mine) + (key[j + 3] > mine);
        for (; j < n; ++j) rank += key[j] > mine;
        f(rank, mine);
    }
}

__device__ __forceinline__ float log_weight(u64 total) { return logf(static_cast<float>(total) * (1.f / 2147483648.f)); }

// u total, so that the first token whose running sum exceeds it is the answer;
// below 0 or no number: the first kept token, 1 and above: the last.
__device__ __forceinline__ u64 mark_of(float u, u64 total) {
    const double all = static_cast<double>(total);
    return static_cast<u64>(fmin(fmax(static_cast<double>(u), 0.) * all, all - 1.));
}
__device__ __forceinline__ u64 mass_goal(float p, u64 total) {   // what the kept beginning has to reach
    const double mass = static_cast<double>(p) * static_cast<double>(total);
    return mass > 0. ? static_cast<u64>(ceil(mass)) : 1;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) k_sample(const __grid_constant__ b3_sample_args a, int count, bool by_one) {
    extern __shared__ uint4 values[];
    __shared__ Shared s;
    const cg::cluster_group cluster = cg::this_cluster();
    const int blocks = cluster.num_blocks(), me = cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x / blocks;
    if (blocks > 1) cluster.barrier_arrive();   // this block runs: its shared memory may be written from outside
    Shared* const first = cluster.map_shared_rank(&s, 0);
    constexpr int kVec = Row<T>::kVec;
    uint4* const col = values + tid;      // vector c of the thread at col[c * kThreads]
    auto each = [&](auto f) {             // f(value, e) for the thread's values, rising indices
#pragma unroll 2
        for (int c = 0; c < count / kVec; ++c) {
            const uint4 raw = col[c * kThreads];
            const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
            for (int k = 0; k < kVec; ++k) f(to_f32(t[k]), c * kVec + k);
        }
    };

    Row<T> r;
    r.x = static_cast<const T*>(a.logits) + row * a.row_stride;
    r.n = a.vocab;
    r.by_one = by_one;
    r.off = by_one ? 0 : static_cast<int>((reinterpret_cast<uintptr_t>(r.x) & 15) / sizeof(T));
    r.count = count;
    r.base = (me * kWarps + warp) * 32 * count + lane * Row<T>::kVec;
    float peak = r.load(col);
    const float t = a.temperature ? __ldg(a.temperature + row) : 1.f;
    const int top_k = a.top_k ? __ldg(a.top_k + row) : 0;
    const float top_p = a.top_p ? __ldg(a.top_p + row) : 1.f;
    const float min_p = a.min_p ? __ldg(a.min_p + row) : 0.f;
    const float u = __ldg(a.uniform + row);
    const bool sampled = t > 0.f;
    const bool by_list = sampled && top_k > 0 && top_k <= kTopList && top_k < r.n;

    // ── the largest logit, and a lower bound of the k-th ──
    float jth = -INFINITY;
    const int full = min(max((r.n + r.off) / (32 * count) - me * kWarps, 0), kWarps);   // warps of this block full of values
    const int j = full ? (top_k + full - 1) / full : 33;
    if (by_list && j <= 32) {
        // bitonic sort of the warp's thread maxima, largest in lane 0
        float x = peak;
#pragma unroll
        for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
            for (int d = k >> 1; d; d >>= 1) {
                const float y = __shfl_xor_sync(0xffffffffu, x, d);
                const bool larger = ((lane & d) == 0) == ((lane & k) == 0);
                x = larger ? fmaxf(x, y) : fminf(x, y);
            }
        jth = __shfl_sync(0xffffffffu, x, j - 1);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, d));
    if (lane == 0) {
        s.warp_f[warp] = peak;
        s.warp_f[kWarps + warp] = jth;
    }
    if (tid == 0) {
        s.count = 0;
        s.best = r.n;
    }
    __syncthreads();
    jth = INFINITY;
    for (int w = 0; w < kWarps; ++w) {
        peak = fmaxf(peak, s.warp_f[w]);
        if (w < full) jth = fminf(jth, s.warp_f[kWarps + w]);
    }
    if (j > 32) jth = -INFINITY;
    if (blocks > 1) {
        cluster.barrier_wait();   // every block of the cluster runs; reached behind the row's loads, so long since done
        if (tid < blocks) {
            Shared* const to = cluster.map_shared_rank(&s, tid);
            to->peak[me] = peak;
            to->bound[me] = jth;
        }
        cluster.sync();
        for (int b = 0; b < blocks; ++b) {
            peak = fmaxf(peak, s.peak[b]);
            jth = fmaxf(jth, s.bound[b]);
        }
    }
    auto write = [&](int id, float logprob) {
        a.ids[row] = id;
        if (a.logprob) a.logprob[row] = logprob;
    };
    const float no_number = __uint_as_float(0x7fffffffu);
    if (!(peak > -INFINITY)) {   // uniform over the cluster, like every choice by the row's settings below
        if (me == 0 && tid == 0) write(-1, no_number);
        return;
    }
    if (!sampled) {
        int best = r.n;
        each([&](float x, int e) {
            if (x == peak) best = min(best, r.index(e));
        });
        best = __reduce_min_sync(0xffffffffu, best);
        if (lane == 0 && best < r.n) atomicMin(&first->best, best);
        cluster.sync();
        if (me == 0 && tid == 0) write(s.best, 0.f);
        return;
    }
    Weigh weigh;
    weigh.set(peak, t);

    // adds an entry to the first block's list
    auto enlist = [&](float x, int i) {
        const int at = atomicAdd(&first->count, 1);
        if (at < kList) first->list.key[at] = rank_key(x, i);
    };

    // ── small top_k: candidates only ──
    if (by_list) {
        each([&](float x, int e) {
            if (x >= jth && x > -INFINITY) enlist(x, r.index(e));
        });
        cluster.sync();
        const int n = first->count;
        if (n <= kList) {
            if (blocks > 1) cluster.sync();   // every block has read the count: the others may leave
            if (me) return;
            const int k = min(top_k, n);
            u64 mine = 0;                     // the entry of rank tid
            // rank_list reads all keys; the ranked ones are written behind a barrier
            u64 found[kList / kThreads];
            int where[kList / kThreads], c = 0;
            rank_list(s.list.key, n, [&](int rank, u64 key) {
                found[c] = key;
                where[c++] = rank;
            });
            __syncthreads();
            for (int i = 0; i < c; ++i)
                if (where[i] < k) s.list.key[where[i]] = found[i];
            __syncthreads();
            float w = 0.f;
            if (tid < k) {
                mine = s.list.key[tid];
                w = weigh.weight<false>(logit_of(static_cast<u32>(mine >> 32)));
            }
            u32 W = tid < k ? whole(w) : 0;
            if (top_p < 1.f) {
                u64 total;
                const u64 upto = block_scan(W, s.warp_sum, total);
                if (tid > 0 && upto - W >= mass_goal(top_p, total)) W = 0;
            }
            if (!(w >= min_p)) W = 0;
            __syncthreads();
            s.list.weight[tid] = W;
            __syncthreads();
            u64 total = 0, before = 0;
            for (int j = 0; j < k; ++j) {
                const u32 x = s.list.weight[j];
                total += x;
                before += static_cast<u32>(s.list.key[j]) > static_cast<u32>(mine) ? x : 0;   // ~index: larger comes first
            }
            if (total == 0) {
                if (tid == 0) write(-1, no_number);
                return;
            }
            const u64 mark = mark_of(u, total);
            if (W && before <= mark && mark < before + W) {
                const float x = logit_of(static_cast<u32>(mine >> 32));
                write(static_cast<int>(~static_cast<u32>(mine)), (x == peak ? 0.f : weigh.power(x)) - log_weight(total));
            }
            return;
        }
        cluster.sync();
        if (me == 0 && tid == 0) s.count = 0;
    }

    auto rest = [&](auto usual) {
    constexpr bool kUsual = decltype(usual)::value;
    // ── top_k (by counts), then top_p (by weights): a beginning of the order ──
    float cut_x = -INFINITY;   // kept: logits above it, and equal ones up to index cut_i
    int cut_i = -1;
    auto kept = [&](float x, int e) { return x > cut_x || (x == cut_x && r.index(e) <= cut_i); };
    auto weight = [&](float x) { return whole(weigh.template weight<kUsual>(x)); };
    // steps below the largest logit, the last one all of what weighs nothing: exp(-21.6) < 2^-31
    const float step = static_cast<float>(kBins - 1) / (21.6f * t);
    auto bin_of = [&](float x) {
        const float y = x == peak ? 0.f : fminf((peak - x) * step, static_cast<float>(kBins - 1));
        return static_cast<int>(__float_as_uint(y + 8388608.f) & 0x7fffffu);   // rounded: 2^23 shifts the fraction out
    };
    for (int stage = 0; stage < 2; ++stage) {
        if (stage == 0 ? !(top_k > 0 && top_k < r.n) : !(top_p < 1.f)) continue;
        __syncthreads();
        for (int i = tid; i < kBins; i += kThreads) s.hist.lo[i] = s.hist.hi[i] = 0;
        if (tid == 0) s.cut_bin = -1;
        __syncthreads();
        each([&](float x, int e) {
            if (!kept(x, e)) return;
            const int b = bin_of(x);
            if (stage == 0) {
                atomicAdd(&s.hist.lo[b], 1u);
            } else if (b < kBins - 1) {
                const u32 w = weight(x);
                atomicAdd(&s.hist.lo[b], w & 0xffffu);
                if (w >> 16) atomicAdd(&s.hist.hi[b], w >> 16);
            }
        });
        cluster.sync();
        // each block adds up its share of the bins, the largest logits first, over all blocks
        const int share = kBins / blocks, per = (share + kThreads - 1) / kThreads;
        u64 sums[kBins / kThreads], mine = 0;
        for (int i = 0; i < per; ++i) {
            const int bin = me * share + tid * per + i;
            sums[i] = 0;
            if (tid * per + i < share)
                for (int b = 0; b < blocks; ++b) {
                    const Shared* const from = cluster.map_shared_rank(&s, b);
                    sums[i] += from->hist.lo[bin] + (static_cast<u64>(from->hist.hi[bin]) << 16);
                }
            mine += sums[i];
        }
        u64 all;
        u64 upto = block_scan(mine, s.warp_sum, all);
        if (tid < blocks) cluster.map_shared_rank(&s, tid)->part[0][me] = all;
        cluster.sync();
        u64 total = 0, before = 0;
        for (int b = 0; b < blocks; ++b) {
            before += b < me ? s.part[0][b] : 0;
            total += s.part[0][b];
        }
        const u64 goal = stage == 0 ? static_cast<u64>(top_k) : mass_goal(top_p, total);
        u64 at = before + upto - mine;
        for (int i = 0; i < per; ++i) {
            if (at < goal && at + sums[i] >= goal)
                for (int b = 0; b < blocks; ++b) {
                    Shared* const to = cluster.map_shared_rank(&s, b);
                    to->cut_bin = me * share + tid * per + i;
                    to->cut_before = at;
                }
            at += sums[i];
        }
        cluster.sync();   // the cut is known, and the histograms (where the list lies) have been read
        const int cut = s.cut_bin;
        if (cut < 0 || cut == kBins - 1) continue;   // only what weighs nothing would go
        const u64 above = s.cut_before;
        auto member = [&](float x, int e) { return kept(x, e) && bin_of(x) == cut; };
        each([&](float x, int e) {
            if (member(x, e)) enlist(x, r.index(e));
        });
        cluster.sync();
        const int n = first->count;
        u64 cut_key;
        if (n <= kList) {
            if (me == 0) {
                u64 found[kList / kThreads];
                int where[kList / kThreads], c = 0;
                rank_list(s.list.key, n, [&](int rank, u64 key) {
                    found[c] = key;
                    where[c++] = rank;
                });
                __syncthreads();
                for (int i = 0; i < c; ++i) {
                    s.list.key[where[i]] = found[i];
                    s.list.weight[where[i]] = stage == 0 ? 1u : weight(logit_of(static_cast<u32>(found[i] >> 32)));
                }
                __syncthreads();
                constexpr int kPer = kList / kThreads;
                u64 own = 0, sum;
                for (int i = 0; i < kPer; ++i) own += kPer * tid + i < n ? s.list.weight[kPer * tid + i] : 0;
                u64 at_ = above + block_scan(own, s.warp_sum, sum) - own;
                for (int i = 0; i < kPer && kPer * tid + i < n; ++i) {
                    const u32 x = s.list.weight[kPer * tid + i];
                    if (at_ < goal && at_ + x >= goal)   // the last that stays
                        for (int b = 0; b < blocks; ++b) cluster.map_shared_rank(&s, b)->cut_key = s.list.key[kPer * tid + i];
                    at_ += x;
                }
            }
            cluster.sync();
            cut_key = s.cut_key;
        } else {
            // bit by bit, the largest key whose entries and those above it reach the goal
            cut_key = 0;
            for (int bit = 63, turn = 0; bit >= 0; --bit, turn ^= 1) {
                const u64 want = cut_key | 1ull << bit;
                u64 own = 0;
                each([&](float x, int e) {
                    if (member(x, e) && rank_key(x, r.index(e)) >= want) own += stage == 0 ? 1 : weight(x);
                });
                u64 sum;
                block_scan(own, s.warp_sum, sum);
                if (tid < blocks) cluster.map_shared_rank(&s, tid)->part[turn][me] = sum;
                cluster.sync();
                sum = above;
                for (int b = 0; b < blocks; ++b) sum += s.part[turn][b];
                if (sum >= goal) cut_key = want;
            }
        }
        cut_x = logit_of(static_cast<u32>(cut_key >> 32));
        cut_i = static_cast<int>(~static_cast<u32>(cut_key));
        cluster.sync();
        if (me == 0 && tid == 0) s.count = 0;
        cluster.sync();
    }

    // ── the token ──
    const bool cut = cut_x > -INFINITY;
    auto final_weight = [&](float x, int i) -> u32 {   // i: the index
        if (cut && !(x > cut_x || (x == cut_x && i <= cut_i))) return 0;
        const float w = weigh.template weight<kUsual>(x);
        return w >= min_p ? whole(w) : 0;
    };
    auto vector_sum = [&](int c) {
        const uint4 raw = col[c * kThreads];
        const T* y = reinterpret_cast<const T*>(&raw);
        const int i = r.index(c * kVec);
        u64 own = 0;
#pragma unroll
        for (int k = 0; k < kVec; ++k) own += final_weight(to_f32(y[k]), i + k);
        return own;
    };
    u64 mine = 0;
#pragma unroll 2
    for (int c = 0; c < count / kVec; ++c) {
        const u64 own = warp_sum(vector_sum(c));
        if (lane == 0) s.vec_sum[warp][c] = own;
        mine += own;
    }
    __syncthreads();
    if (lane == 0) s.warp_sum[warp] = mine;
    __syncthreads();
    u64 total = 0, before = 0;
    for (int w = 0; w < kWarps; ++w) {
        before += w < warp ? s.warp_sum[w] : 0;
        total += s.warp_sum[w];
    }
    if (blocks > 1) {
        if (tid < blocks) cluster.map_shared_rank(&s, tid)->part[1][me] = total;
        cluster.sync();
        total = 0;
        for (int b = 0; b < blocks; ++b) {
            before += b < me ? s.part[1][b] : 0;
            total += s.part[1][b];
        }
    }
    if (total == 0) {
        if (me == 0 && tid == 0) write(-1, no_number);
        return;
    }
    const u64 mark = mark_of(u, total);
    if (mark < before || mark >= before + mine) return;
    // this warp has it: its values in index order are (vector, lane, place)
    int c = 0;
    for (;; ++c) {
        const u64 x = s.vec_sum[warp][c];
        if (mark < before + x) break;
        before += x;
    }
    const u64 own = vector_sum(c);
    u64 upto = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
    }
    const int src = __ffs(__ballot_sync(0xffffffffu, mark < before + upto)) - 1;
    before += __shfl_sync(0xffffffffu, upto - own, src);
    // that lane's vector, a value a lane
    const int i = __shfl_sync(0xffffffffu, r.index(c * kVec), src) + lane;
    const float x = lane < kVec ? to_f32(reinterpret_cast<const T*>(col + c * kThreads + (src - lane))[lane]) : -INFINITY;
    upto = lane < kVec ? final_weight(x, i) : 0;
#pragma unroll
    for (int d = 1; d < kVec; d <<= 1) {
        const u64 y = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += y;
    }
    const int at = __ffs(__ballot_sync(0xffffffffu, lane < kVec && mark < before + upto)) - 1;
    if (lane == at) write(i, (x == peak ? 0.f : weigh.power(x)) - log_weight(total));
    };
    if (weigh.usual())
        rest(std::true_type{});
    else
        rest(std::false_type{});
}

// Values a thread: at most 32 of 32 bits or 64 of 16 (64 KB, two blocks an SM)
// where the row fits a cluster so.  Fewer, longer blocks are better than more:
// 256 rows x 131072 in 16 bits with top_k 94 us in clusters of four, 162 of eight
// (with every value divided by the temperature, as unusual rows still are).
template <typename T>
int launch(const b3_sample_args& a, cudaStream_t st) {
    constexpr int kVec = Row<T>::kVec;
    static PerDeviceOnce smem_once;
    const int rc = set_smem_limit_once(smem_once, k_sample<T>, kMostValues * kThreads * sizeof(T), "cudaFuncSetAttribute(k_sample)");
    if (rc) return rc;
    if (static_cast<int64_t>(a.rows) * kMaxBlocks > 0x7fffffff) return set_error(B3_EINVAL, "%d rows are too many for one call", a.rows);
    // a row that starts within a 16-byte vector takes up to a vector more places
    const bool aligned = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.row_stride % kVec == 0;
    bool by_one = false;
    int places = a.vocab + (aligned ? 0 : kVec - 1);
    if (places > kMaxBlocks * kThreads * kMostValues) {
        by_one = true;   // the largest vocabulary in unaligned rows
        places = a.vocab;
    }
    auto values = [&](int blocks) {
        const int per = kThreads * kVec * blocks;
        return (places + per - 1) / per * kVec;
    };
    // few rows: short columns on more SMs; many: few blocks a row, so that a row's steps stay inside a block
    int blocks = 1;
    while (blocks < kMaxBlocks && (values(blocks) > 128 / static_cast<int>(sizeof(T)) || (values(blocks) > 8 && 2 * blocks * static_cast<int64_t>(a.rows) <= device_sms())))
        blocks *= 2;
    const int count = values(blocks);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * blocks);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(count) * kThreads * sizeof(T);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {static_cast<unsigned>(blocks), 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k_sample<T>, a, count, by_one);
    return e == cudaSuccess ? 0 : set_cuda_error("k_sample", e);
}

}  // namespace
}  // namespace b3

using namespace b3;

extern "C" int b3_sample(const b3_sample_args* args, void* stream) {
    if (!args) return set_error(B3_EINVAL, "null arguments");
    const b3_sample_args& a = *args;
    if (a.rows == 0) return 0;
    if (!a.logits || !a.uniform || !a.ids) return set_error(B3_EINVAL, "null logits, uniform or ids");
    if (a.rows < 0 || a.vocab <= 0 || a.vocab > B3_SAMPLE_MAX_VOCAB || (a.row_stride < a.vocab && a.row_stride != 0))
        return set_error(B3_EINVAL, "logits of %d rows x %d (at most %d), row stride %lld", a.rows, a.vocab,
                         B3_SAMPLE_MAX_VOCAB, static_cast<long long>(a.row_stride));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (a.dtype) {
        case B3_DTYPE_F32: return launch<float>(a, st);
        case B3_DTYPE_F16: return launch<__half>(a, st);
        case B3_DTYPE_BF16: return launch<__nv_bfloat16>(a, st);
        default: return set_error(B3_EINVAL, "dtype %d", a.dtype);
    }
}
