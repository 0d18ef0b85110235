// Rules on the logits of a decoder, in one pass over them: with count = how
// often v stands among the tokens of row n,
//   l = logits[n][v]
//   count > 0:  l = l > 0 ? l / repetition : l * repetition
//               l = l - presence - frequency * count
//   l = l + bias[v];  not allowed: l = -infinity
// Bound by HBM, or by the launch where the logits are few.  A workgroup takes
// `segment` columns of a row: it counts those of the row's tokens that fall into
// them in LDS (integers: the order does not matter), then streams its columns.
#include "network.h"
#include "rows.h"

namespace wctct {

namespace {

constexpr int kThreads = 256;

template <typename B>
__device__ __forceinline__ float bias_at(const void *bias, long at) {
    return to_float(static_cast<const B *>(bias)[at]);
}
__device__ __forceinline__ float bias_of(const void *bias, int type, long at) {
    return type == kIoF32 ? bias_at<float>(bias, at)
                          : type == kIoF16 ? bias_at<f16>(bias, at) : bias_at<bf16>(bias, at);
}

template <typename IO, bool VEC>
__global__ __launch_bounds__(kThreads) void adjust_kernel(warpctct_adjust_t p, int segment) {
    constexpr int EV = VEC ? kVec<IO> : 1;
    extern __shared__ unsigned counts[];
    const int n = blockIdx.y, from = blockIdx.x * segment, to = min(from + segment, p.V);
    const bool history = p.tokens && p.H > 0;
    float repetition = p.repetition, presence = p.presence, frequency = p.frequency;
    if (history) {
        for (int k = threadIdx.x; k < to - from; k += kThreads) counts[k] = 0u;
        __syncthreads();
        const int h = p.tokens_lengths ? min(max(p.tokens_lengths[n], 0), p.H) : p.H;
        const long row = (long)n * p.tokens_n;
        for (int i = threadIdx.x; i < h; i += kThreads) {
            const long v = p.tokens_64 ? (long)static_cast<const long long *>(p.tokens)[row + i]
                                       : (long)static_cast<const int *>(p.tokens)[row + i];
            if (v >= from && v < to) atomicAdd(&counts[v - from], 1u);
        }
        __syncthreads();
        if (p.repetitions) repetition = p.repetitions[n];
        if (p.presences) presence = p.presences[n];
        if (p.frequencies) frequency = p.frequencies[n];
    }
    const IO *in = static_cast<const IO *>(p.logits) + (long)n * p.logits_n;
    IO *out = static_cast<IO *>(p.out) + (long)n * p.V;
    const unsigned char *flags =
        p.allowed && !p.allowed_packed ? static_cast<const unsigned char *>(p.allowed) + (long)n * p.allowed_n : nullptr;
    const unsigned *words =
        p.allowed && p.allowed_packed ? static_cast<const unsigned *>(p.allowed) + (long)n * p.allowed_n : nullptr;
    for (int at = from + threadIdx.x * EV; at < to; at += kThreads * EV) {
        float l[EV];
        load_n<EV>(in + at, l);
        // (from is a multiple of 32 and EV divides 32: the bits lie in one word)
        const unsigned bits = words ? words[at >> 5] >> (at & 31) : 0u;
#pragma unroll
        for (int i = 0; i < EV; ++i) {
            const int v = at + i;
            if (history) {
                const unsigned count = counts[v - from];
                if (count) {
                    l[i] = l[i] > 0.0f ? l[i] / repetition : l[i] * repetition;
                    l[i] = l[i] - presence - frequency * (float)count;
                }
            }
            if (p.bias) l[i] += bias_of(p.bias, p.bias_dtype, (long)n * p.bias_n + v);
            if (words && !((bits >> i) & 1u)) l[i] = -__builtin_huge_valf();
            if (flags && !flags[v]) l[i] = -__builtin_huge_valf();
        }
        store_n<EV>(out + at, l);
    }
}

// Columns of a workgroup, a multiple of 2048.  Every workgroup of a row reads
// the row's whole history, which should stay the smaller part of its traffic; but
// there should be two workgroups for every compute unit first, and the counts of
// 16384 columns take all the LDS that two workgroups on a compute unit can have.
int segment_of(long N, int V, int H, bool history) {
    long segment = 2048;
    while (segment < V && segment < 16384 && N * ((V + 2 * segment - 1) / (2 * segment)) >= 512 &&
           (!history || 2L * H > segment || segment < 4096))
        segment *= 2;
    return (int)segment;
}

template <typename IO, bool VEC>
hipError_t start(const warpctct_adjust_t &p, hipStream_t stream) {
    const bool history = p.tokens && p.H > 0;
    const int segment = segment_of(p.N, p.V, p.H, history);
    const dim3 grid((p.V + segment - 1) / segment, p.N);
    const size_t shared = history ? sizeof(unsigned) * (size_t)(p.V < segment ? p.V : segment) : 0;
    auto kernel = adjust_kernel<IO, VEC>;
    TIMED_LAUNCH(kernel, grid, dim3(kThreads), shared, stream, p, segment);
    return hipGetLastError();
}

template <typename IO>
hipError_t start(const warpctct_adjust_t &p, hipStream_t stream) {
    const auto aligned = [](const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
    const bool vec = p.V % kVec<IO> == 0 && p.logits_n % kVec<IO> == 0 && aligned(p.logits) && aligned(p.out);
    return vec ? start<IO, true>(p, stream) : start<IO, false>(p, stream);
}

}  // namespace

hipError_t launch_adjust(const warpctct_adjust_t &p, hipStream_t stream) {
    if (p.dtype == kIoF32) return start<float>(p, stream);
    if (p.dtype == kIoF16) return start<f16>(p, stream);
    return start<bf16>(p, stream);
}

}  // namespace wctct
