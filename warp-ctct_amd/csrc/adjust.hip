// Rules on the logits of a decoder, in one pass over them: with count = how
// often v stands among the tokens of row n,
//   l = logits[n][v]
//   count > 0:  l = l > 0 ? l / repetition : l * repetition
//               l = l - presence - frequency * count
//   l = l + bias[v];  not allowed: l = -infinity
// Bound by HBM, or by the launch where the logits are few.  A workgroup takes one
// 16-byte vector a thread (2048 columns of 2-byte elements) of a row, asks for
// everything that belongs to it first, counts meanwhile those of the row's tokens
// that fall into its columns in LDS (integers: the order does not matter), and
// applies the rules.  More columns a workgroup would read the history less often,
// but fewer wavefronts would share a compute unit: 128 rows of 65536 bfloat16
// logits with 300 tokens each take 10.5 us with one vector a thread, 11.5 with two,
// 13.2 with four.
#include "network.h"
#include "rows.h"

namespace wctct {

namespace {

constexpr int kThreads = 256;
constexpr int kVectors = 1;      // 16-byte vectors of a thread

// EV columns of a bias of any of the three types, all of them asked for at once
template <typename B, int EV>
__device__ __forceinline__ void load_bias(const void *bias, long at, float (&b)[EV]) {
    B v[EV];
#pragma unroll
    for (int i = 0; i < EV; ++i) v[i] = static_cast<const B *>(bias)[at + i];
#pragma unroll
    for (int i = 0; i < EV; ++i) b[i] = to_float(v[i]);
}

template <typename IO, bool VEC>
__global__ __launch_bounds__(kThreads) void adjust_kernel(warpctct_adjust_t p) {
    constexpr int EV = VEC ? kVec<IO> : 1, U = VEC ? kVectors : kVectors * kVec<IO>, SEGMENT = kThreads * EV * U;
    __shared__ unsigned counts[SEGMENT];
    const int n = blockIdx.y, from = blockIdx.x * SEGMENT, t = threadIdx.x;
    const bool history = p.tokens && p.H > 0;
    const IO *in = static_cast<const IO *>(p.logits) + (long)n * p.logits_n;
    Raw<IO, EV> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u].load(in + min(from + (u * kThreads + t) * EV, p.V - EV), true, 0);
    // the bias, and a bit for every column that is allowed
    float bias[U][EV];
    unsigned bits[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int at = min(from + (u * kThreads + t) * EV, p.V - EV);
        const long b = (long)n * p.bias_n + at, m = (long)n * p.allowed_n;
        if (p.bias && p.bias_dtype == kIoF32) load_bias<float>(p.bias, b, bias[u]);
        if (p.bias && p.bias_dtype == kIoF16) load_bias<f16>(p.bias, b, bias[u]);
        if (p.bias && p.bias_dtype == kIoBF16) load_bias<bf16>(p.bias, b, bias[u]);
        bits[u] = ~0u;
        if (p.allowed && p.allowed_packed) {
            // (at is a multiple of EV, which divides 32: the bits lie in one word)
            bits[u] = static_cast<const unsigned *>(p.allowed)[m + (at >> 5)] >> (at & 31);
        } else if (p.allowed) {
            unsigned char flag[EV];
#pragma unroll
            for (int i = 0; i < EV; ++i) flag[i] = static_cast<const unsigned char *>(p.allowed)[m + at + i];
            bits[u] = 0u;
#pragma unroll
            for (int i = 0; i < EV; ++i) bits[u] |= (flag[i] ? 1u : 0u) << i;
        }
    }
    float repetition = p.repetition, presence = p.presence, frequency = p.frequency;
    if (history) {
        const int to = min(from + SEGMENT, p.V);
        for (int k = t; k < to - from; k += kThreads) counts[k] = 0u;
        const int h = p.tokens_lengths ? min(max(p.tokens_lengths[n], 0), p.H) : p.H;
        const long row = (long)n * p.tokens_n;
        __syncthreads();
        for (int i = t; i < h; i += kThreads) {
            const long v = p.tokens_64 ? (long)static_cast<const long long *>(p.tokens)[row + i]
                                       : (long)static_cast<const int *>(p.tokens)[row + i];
            if (v >= from && v < to) atomicAdd(&counts[v - from], 1u);
        }
        if (p.repetitions) repetition = p.repetitions[n];
        if (p.presences) presence = p.presences[n];
        if (p.frequencies) frequency = p.frequencies[n];
        __syncthreads();
    }
    IO *out = static_cast<IO *>(p.out) + (long)n * p.V;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int at = from + (u * kThreads + t) * EV;
        if (at >= p.V) break;
        float l[EV];
#pragma unroll
        for (int i = 0; i < EV; ++i) l[i] = raw[u][i];
        if (history) {
            // (of a vector's columns together: most of them have no count)
            unsigned count[EV], any = 0u;
#pragma unroll
            for (int i = 0; i < EV; ++i) any |= count[i] = counts[at - from + i];
            if (any) {
#pragma unroll
                for (int i = 0; i < EV; ++i) {
                    const float scaled = l[i] > 0.0f ? l[i] / repetition : l[i] * repetition;
                    const float less = scaled - presence - frequency * (float)count[i];
                    l[i] = count[i] ? less : l[i];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < EV; ++i) {
            if (p.bias) l[i] += bias[u][i];
            l[i] = (bits[u] >> i) & 1u ? l[i] : -__builtin_huge_valf();
        }
        store_n<EV>(out + at, l);
    }
}

template <typename IO, bool VEC>
hipError_t start(const warpctct_adjust_t &p, hipStream_t stream) {
    const int segment = kThreads * kVec<IO> * kVectors;
    auto kernel = adjust_kernel<IO, VEC>;
    TIMED_LAUNCH(kernel, dim3((p.V + segment - 1) / segment, p.N), dim3(kThreads), 0, stream, p);
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
