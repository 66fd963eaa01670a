// sample.cu — b3_sample: the next token of every row of logits by temperature,
// top-k, top-p and min-p from a given random number.
//
//   w_i = exp((l_i - m) / T) as a whole number of 2^-31, W = their exact sum
// Sums of whole numbers do not depend on their order, so the answer is the
// same however the row is split over threads.  The kept tokens are a beginning
// of the order (falling logit, rising index); it is found by a search over the
// logits' order-preserving bit patterns, eight bits a pass, then over indices
// among equals.  One block a row.
#include "kv_cache.cuh"

namespace b3 {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;

// Order-preserving bits of a logit: larger logits, larger keys; -0 = +0; NaN
// and -inf give 0 (they weigh nothing and are never taken).
__device__ __forceinline__ uint32_t key_of(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float weight_of(float x, float peak, float t) { return x == peak ? 1.f : expf((x - peak) / t); }
__device__ __forceinline__ unsigned long long whole(float w) { return static_cast<unsigned long long>(w * 2147483648.f); }

template <typename V>
__device__ __forceinline__ V block_sum(V v, V* sh) {
    for (int m = 16; m; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    V t = 0;
    for (int w = 0; w < kWarps; ++w) t += sh[w];
    return t;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample(const b3_sample_args a) {
    __shared__ float shf[kWarps];
    __shared__ unsigned long long shu[kWarps], bin_w[256];
    __shared__ int found;
    const int row = blockIdx.x, tid = threadIdx.x, n = a.vocab;
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    auto at = [&](int i) { return to_f32(x[i]); };

    uint32_t kmax = 0;
    for (int i = tid; i < n; i += kThreads) kmax = max(kmax, key_of(at(i)));
    kmax = __reduce_max_sync(0xffffffffu, kmax);
    if ((tid & 31) == 0) shf[tid >> 5] = __uint_as_float(kmax);
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) kmax = max(kmax, __float_as_uint(shf[w]));
    if (tid == 0) found = n;
    __syncthreads();
    if (kmax == 0) {
        if (tid == 0) {
            a.ids[row] = -1;
            if (a.logprob) a.logprob[row] = __uint_as_float(0x7fffffffu);
        }
        return;
    }
    const float peak = __uint_as_float(kmax & 0x80000000u ? kmax & 0x7fffffffu : ~kmax);
    const float t = a.temperature ? a.temperature[row] : 1.f;
    if (!(t > 0.f)) {
        for (int i = tid; i < n; i += kThreads)
            if (key_of(at(i)) == kmax) atomicMin(&found, i);
        __syncthreads();
        if (tid == 0) {
            a.ids[row] = found;
            if (a.logprob) a.logprob[row] = 0.f;
        }
        return;
    }
    const int top_k = a.top_k ? a.top_k[row] : 0;
    const float top_p = a.top_p ? a.top_p[row] : 1.f;
    const float min_p = a.min_p ? a.min_p[row] : 0.f;

    // kept: key > cut, or key == cut and index <= last
    uint32_t cut = 1;
    int last = n;
    for (int stage = 0; stage < 2; ++stage) {
        if (stage == 0 ? !(top_k > 0 && top_k < n) : !(top_p < 1.f)) continue;
        unsigned long long sum = 0, goal;   // keep the shortest beginning that reaches `goal`
        if (stage == 0) {
            goal = top_k;
        } else {
            for (int i = tid; i < n; i += kThreads) {
                const uint32_t k = key_of(at(i));
                if (k > cut || (k == cut && i <= last)) sum += whole(weight_of(at(i), peak, t));
            }
            sum = block_sum(sum, shu);
            const double mass = static_cast<double>(top_p) * static_cast<double>(sum);
            goal = mass > 0. ? static_cast<unsigned long long>(ceil(mass)) : 1;
        }
        uint32_t prefix = 0;
        unsigned long long before = 0;   // weight of the keys above the prefix
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            for (int i = tid; i < 256; i += kThreads) bin_w[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const uint32_t k = key_of(at(i));
                if (k && (shift == 24 || (k >> (shift + 8)) == prefix) && (k > cut || (k == cut && i <= last)))
                    atomicAdd(&bin_w[(k >> shift) & 255], stage == 0 ? 1ull : whole(weight_of(at(i), peak, t)));
            }
            __syncthreads();
            int b = 255;
            for (; b > 0 && before + bin_w[b] < goal; --b) before += bin_w[b];
            prefix = prefix << 8 | b;
        }
        // among equals, by index
        int lo = -1, hi = n - 1;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            sum = 0;
            for (int i = tid; i <= mid; i += kThreads)
                if (key_of(at(i)) == prefix) sum += stage == 0 ? 1ull : whole(weight_of(at(i), peak, t));
            if (before + block_sum(sum, shu) >= goal) hi = mid; else lo = mid;
        }
        last = prefix == cut ? min(last, hi) : hi;
        cut = max(prefix, 1u);
    }

    auto kept = [&](int i) -> unsigned long long {
        const float v = at(i);
        const uint32_t k = key_of(v);
        if (!(k > cut || (k == cut && i <= last))) return 0;
        const float w = weight_of(v, peak, t);
        return w >= min_p ? whole(w) : 0;
    };
    unsigned long long total = 0;
    for (int i = tid; i < n; i += kThreads) total += kept(i);
    total = block_sum(total, shu);
    // below 0 or no number: the first kept token; 1 and above: the last
    const double mark = fmin(fmax(static_cast<double>(a.uniform[row]), 0.) * static_cast<double>(total),
                             static_cast<double>(total) - 1.);
    int lo = -1, hi = n - 1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        unsigned long long sum = 0;
        for (int i = tid; i <= mid; i += kThreads) sum += kept(i);
        if (static_cast<double>(block_sum(sum, shu)) > mark) hi = mid; else lo = mid;
    }
    if (tid == 0) {
        a.ids[row] = total ? hi : -1;
        if (a.logprob)
            a.logprob[row] = total ? (at(hi) == peak ? 0.f : (at(hi) - peak) / t) - logf(static_cast<float>(total) * (1.f / 2147483648.f))
                                   : __uint_as_float(0x7fffffffu);
    }
}

}  // namespace
}  // namespace b3

using namespace b3;

extern "C" int b3_sample(const b3_sample_args* args, void* stream) {
    if (!args) return set_error(B3_EINVAL, "null arguments");
    const b3_sample_args& a = *args;
    if (a.rows == 0) return 0;
    if (!a.logits || !a.uniform || !a.ids) return set_error(B3_EINVAL, "null logits, uniform or ids");
    if (a.rows < 0 || a.vocab <= 0 || a.vocab > B3_SAMPLE_MAX_VOCAB || a.row_stride < a.vocab)
        return set_error(B3_EINVAL, "logits of %d rows x %d (at most %d), row stride %lld", a.rows, a.vocab,
                         B3_SAMPLE_MAX_VOCAB, static_cast<long long>(a.row_stride));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (a.dtype) {
        case B3_DTYPE_F32: k_sample<float><<<a.rows, kThreads, 0, st>>>(a); break;
        case B3_DTYPE_F16: k_sample<__half><<<a.rows, kThreads, 0, st>>>(a); break;
        case B3_DTYPE_BF16: k_sample<__nv_bfloat16><<<a.rows, kThreads, 0, st>>>(a); break;
        default: return set_error(B3_EINVAL, "dtype %d", a.dtype);
    }
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : set_cuda_error("k_sample", e);
}
