// Short causal convolution along time, every channel with its own K taps:
//   pre[t] = bias + sum_k weight[k] x[t - (K-1) + k],  out = pre or silu(pre)
//   gp = g act'(pre),  gx[t] = sum_k weight[k] gp[t + K-1 - k],
//   gweight[k] = sum_t gp[t] x[t - (K-1) + k],  gbias = sum_t gp[t]
// Bound by HBM: x is read and out written once, in the backward x and g read and
// gx written.  A thread takes a few channels next to each other and walks down a
// tile of time with the last K-1 inputs in registers, so that every row is
// loaded once but for the K-1 rows where two tiles meet.  Four channels a thread:
// with eight of 2-byte elements there are too few wavefronts to keep the memory
// busy (32 ragged sequences of up to 400 steps, 2048 channels, bfloat16: forward
// 39.5 us instead of 26, 3.5 TB/s; backward 41 us, 3.2 TB/s).
#include "network.h"
#include "rows.h"

namespace wctct {

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 4;        // rows asked for at once

struct Tile {
    int n, t0, e;      // sequence, first step, first channel
    bool in;
};

// Thread -> (channels, tile): the channels of a tile first, so that neighbouring
// lanes read neighbouring channels, and narrow problems still fill wavefronts.
template <int EV>
__device__ __forceinline__ Tile tile_of(int E, int tiles, int steps) {
    const unsigned per = (unsigned)((E + EV - 1) / EV);
    const unsigned long long i = (unsigned long long)blockIdx.x * kThreads + threadIdx.x;
    Tile a;
    a.in = i < (unsigned long long)per * (unsigned)tiles;
    const unsigned tile = a.in ? (unsigned)(i / per) : 0u;
    a.n = blockIdx.y;
    a.t0 = (int)tile * steps;
    a.e = a.in ? (int)(i - (unsigned long long)tile * per) * EV : 0;
    return a;
}

__device__ __forceinline__ int length_of(const int *lengths, int n, int L) {
    return lengths ? min(max(lengths[n], 0), L) : L;
}

// Row t of a sequence with the K-1 rows of `initial` in front of it.
template <int EV, int K, typename IO>
__device__ __forceinline__ void load_row(const IO *x, long x_t, const IO *initial, int E, int t, float *v) {
    if (t >= 0) {
        load_n<EV>(x + (long)t * x_t, v);
    } else if (initial) {
        load_n<EV>(initial + (long)(t + K - 1) * E, v);
    } else {
#pragma unroll
        for (int i = 0; i < EV; ++i) v[i] = 0.0f;
    }
}

template <int EV, int K>
__device__ __forceinline__ void load_taps(const float *weight, const float *bias, int e, float (&w)[K][EV],
                                          float (&b)[EV]) {
#pragma unroll
    for (int i = 0; i < EV; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][i] = weight[(long)(e + i) * K + k];
        b[i] = bias ? bias[e + i] : 0.0f;
    }
}

template <typename IO, int K, int EV>
__global__ __launch_bounds__(kThreads) void conv_kernel(warpctct_conv_t p, int tiles, int steps) {
    const Tile a = tile_of<EV>(p.E, tiles, steps);
    if (!a.in) return;
    const int len = length_of(p.lengths, a.n, p.L);
    const IO *x = static_cast<const IO *>(p.x) + (long)a.n * p.x_n + a.e;
    const IO *initial =
        p.initial ? static_cast<const IO *>(p.initial) + (long)a.n * (K - 1) * p.E + a.e : nullptr;
    IO *out = static_cast<IO *>(p.out) + (long)a.n * p.L * p.E + a.e;
    if (p.last && a.t0 == 0) {
        IO *last = static_cast<IO *>(p.last) + (long)a.n * (K - 1) * p.E + a.e;
        for (int r = 0; r < K - 1; ++r) {
            float v[EV];
            load_row<EV, K>(x, p.x_t, initial, p.E, len - (K - 1) + r, v);
            store_n<EV>(last + (long)r * p.E, v);
        }
    }
    const int end = min(a.t0 + steps, p.L), live = min(end, len);
    int t = a.t0;
    if (t < live) {
        // the rows asked for, and those being worked on
        Raw<IO, EV> next[kAhead];
        auto request = [&](int from) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j) next[j].load(x + (long)min(from + j, live - 1) * p.x_t, true, 0);
        };
        request(t);
        float w[K][EV], b[EV], v[K - 1 + kAhead][EV];
        load_taps<EV, K>(p.weight, p.bias, a.e, w, b);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) load_row<EV, K>(x, p.x_t, initial, p.E, t - (K - 1) + k, v[k]);
        for (; t < live; t += kAhead) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
#pragma unroll
                for (int i = 0; i < EV; ++i) v[K - 1 + j][i] = next[j][i];
            if (t + kAhead < live) request(t + kAhead);
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (t + j >= live) break;
                float y[EV];
#pragma unroll
                for (int i = 0; i < EV; ++i) {
                    y[i] = b[i];
#pragma unroll
                    for (int k = 0; k < K; ++k) y[i] = fmaf(w[k][i], v[j + k][i], y[i]);
                    if (p.silu) y[i] *= sigmoid(y[i]);
                }
                store_n<EV>(out + (long)(t + j) * p.E, y);
            }
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
#pragma unroll
                for (int i = 0; i < EV; ++i) v[k][i] = v[k + kAhead][i];
        }
        t = live;
    }
    const float zero[EV] = {};
    for (; t < end; ++t) store_n<EV>(out + (long)t * p.E, zero);
}

// A thread walks its tile and K-1 steps past it: at step t it forms gp[t], adds
// to its sums if t is its own, and has with gp[t-K+1 .. t] all that gx[t-K+1]
// takes.  The tile that starts a sequence goes on to the rows in front of it,
// whose gradient is that of `initial`.
template <typename IO, int K, int EV>
__global__ __launch_bounds__(kThreads) void conv_grad_kernel(warpctct_conv_t p, warpctct_conv_grad_t g,
                                                             float *__restrict__ partial, int tiles, int steps) {
    const Tile a = tile_of<EV>(p.E, tiles, steps);
    if (!a.in) return;
    const int len = length_of(p.lengths, a.n, p.L);
    const IO *x = static_cast<const IO *>(p.x) + (long)a.n * p.x_n + a.e;
    const IO *up = static_cast<const IO *>(g.grad_out) + (long)a.n * g.grad_n + a.e;
    const long before = (long)a.n * (K - 1) * p.E + a.e;
    const IO *initial = p.initial ? static_cast<const IO *>(p.initial) + before : nullptr;
    const IO *glast = g.grad_last ? static_cast<const IO *>(g.grad_last) + before : nullptr;
    IO *ginitial = g.grad_initial ? static_cast<IO *>(g.grad_initial) + before : nullptr;
    IO *gx = static_cast<IO *>(g.grad_x) + (long)a.n * p.L * p.E + a.e;
    const int end = min(a.t0 + steps, p.L);
    // windows of x and gp: K-1 rows behind, kAhead being worked on
    float w[K][EV], b[EV], v[K - 1 + kAhead][EV], gp[K - 1 + kAhead][EV], gw[K][EV], gb[EV];
    Raw<IO, EV> next_x[kAhead], next_g[kAhead];
    auto request = [&](int from) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const long t = min(from + j, len - 1);
            next_x[j].load(x + t * p.x_t, true, 0);
            next_g[j].load(up + t * g.grad_t, true, 0);
        }
    };
    if (a.t0 < len) request(a.t0);
    load_taps<EV, K>(p.weight, p.bias, a.e, w, b);
#pragma unroll
    for (int i = 0; i < EV; ++i) {
        gb[i] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) gw[k][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < K - 1; ++k) gp[k][i] = v[k][i] = 0.0f;
    }
    if (a.t0 < len) {
#pragma unroll
        for (int k = 0; k < K - 1; ++k) load_row<EV, K>(x, p.x_t, initial, p.E, a.t0 - (K - 1) + k, v[k]);
    }
    // behind the sequence there is nothing but zeros to write
    const int work = a.t0 < len || a.t0 == 0 ? min(end, len) + K - 1 : a.t0;
    for (int t0 = a.t0; t0 < work; t0 += kAhead) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const bool in = t0 + j < len;
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                v[K - 1 + j][i] = in ? next_x[j][i] : 0.0f;
                gp[K - 1 + j][i] = in ? next_g[j][i] : 0.0f;
            }
        }
        if (t0 + kAhead < min(len, work)) request(t0 + kAhead);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int t = t0 + j;
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                float &e = gp[K - 1 + j][i];
                if (p.silu) {
                    float y = b[i];
#pragma unroll
                    for (int k = 0; k < K; ++k) y = fmaf(w[k][i], v[j + k][i], y);
                    const float s = sigmoid(y);
                    e *= s * fmaf(y, 1.0f - s, 1.0f);
                    if (t >= len) e = 0.0f;
                }
                const float own = t < end ? e : 0.0f;
                gb[i] += own;
#pragma unroll
                for (int k = 0; k < K; ++k) gw[k][i] = fmaf(own, v[j + k][i], gw[k][i]);
            }
            const int s = t - (K - 1);      // gx[s] is complete
            if (s >= min(end, len) || (s < a.t0 && a.t0 > 0) || (s < 0 && !ginitial)) continue;
            float d[EV];
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                d[i] = 0.0f;
#pragma unroll
                for (int k = 0; k < K; ++k) d[i] = fmaf(w[K - 1 - k][i], gp[j + k][i], d[i]);
            }
            const int r = s - len + K - 1;   // row s is row r of the state that was handed on
            if (glast && r >= 0 && r < K - 1) {
                float last[EV];
                load_n<EV>(glast + (long)r * p.E, last);
#pragma unroll
                for (int i = 0; i < EV; ++i) d[i] += last[i];
            }
            store_n<EV>(s >= 0 ? gx + (long)s * p.E : ginitial + (long)(s + K - 1) * p.E, d);
        }
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int i = 0; i < EV; ++i) {
                v[k][i] = v[k + kAhead][i];
                gp[k][i] = gp[k + kAhead][i];
            }
    }
    const float zero[EV] = {};
    for (int s = max(a.t0, len); s < end; ++s) store_n<EV>(gx + (long)s * p.E, zero);
    if (!partial) return;
    float *mine = partial + ((size_t)a.n * tiles + a.t0 / steps) * (size_t)p.E * (K + 1);
#pragma unroll
    for (int i = 0; i < EV; ++i) {
#pragma unroll
        for (int k = 0; k < K; ++k) mine[(long)(a.e + i) * K + k] = gw[k][i];
        mine[(long)p.E * K + a.e + i] = gb[i];
    }
}

template <typename IO, int K, int EV>
__global__ __launch_bounds__(kThreads) void conv_step_kernel(warpctct_conv_step_t p) {
    const unsigned per = (unsigned)((p.E + EV - 1) / EV);
    const unsigned long long i0 = (unsigned long long)blockIdx.x * kThreads + threadIdx.x;
    if (i0 >= (unsigned long long)per * (unsigned)p.N) return;
    const int n = (int)(i0 / per), e = (int)(i0 - (unsigned long long)n * per) * EV;
    IO *out = static_cast<IO *>(p.out) + (long)n * p.E + e;
    float y[EV];
#pragma unroll
    for (int i = 0; i < EV; ++i) y[i] = 0.0f;
    if (!p.advance || p.advance[n]) {
        IO *state = static_cast<IO *>(p.state) + (long)n * (K - 1) * p.E + e;
        float w[K][EV], v[K][EV];
        load_taps<EV, K>(p.weight, p.bias, e, w, y);
#pragma unroll
        for (int k = 0; k < K - 1; ++k) load_n<EV>(state + (long)k * p.E, v[k]);
        load_n<EV>(static_cast<const IO *>(p.x) + (long)n * p.x_n + e, v[K - 1]);
#pragma unroll
        for (int i = 0; i < EV; ++i) {
#pragma unroll
            for (int k = 0; k < K; ++k) y[i] = fmaf(w[k][i], v[k][i], y[i]);
            if (p.silu) y[i] *= sigmoid(y[i]);
        }
#pragma unroll
        for (int k = 0; k < K - 1; ++k) store_n<EV>(state + (long)k * p.E, v[k + 1]);
    }
    store_n<EV>(out, y);
}

bool aligned(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Steps of a tile: 32, fewer where that would leave compute units without work.
int conv_steps(long N, long L, long vectors) {
    int steps = 32;
    while (steps > 4 && N * ((L + steps - 1) / steps) * vectors < 256L * 1024) steps /= 2;
    return steps;
}
int conv_grad_steps(int N, int L, int E) {
    int steps = 64;
    while (steps > 8 && (long)N * ((L + steps - 1) / steps) * ((E + 3) / 4) < 256L * 512) steps /= 2;
    return steps;
}

template <typename IO, int K, int EV>
hipError_t start(const warpctct_conv_t &p, hipStream_t stream) {
    const long per = (p.E + EV - 1) / EV;
    const int steps = conv_steps(p.N, p.L, per), tiles = p.L > 0 ? (p.L + steps - 1) / steps : 1;
    const dim3 grid((unsigned)((per * tiles + kThreads - 1) / kThreads), p.N);
    auto kernel = conv_kernel<IO, K, EV>;
    TIMED_LAUNCH(kernel, grid, dim3(kThreads), 0, stream, p, tiles, steps);
    return hipGetLastError();
}

template <typename IO, int K, int EV>
hipError_t start_grad(const warpctct_conv_t &p, const warpctct_conv_grad_t &g, float *partial, hipStream_t stream) {
    const long per = (p.E + EV - 1) / EV;
    const int steps = conv_grad_steps(p.N, p.L, p.E), tiles = conv_grad_tiles(p.N, p.L, p.E);
    const dim3 grid((unsigned)((per * tiles + kThreads - 1) / kThreads), p.N);
    auto kernel = conv_grad_kernel<IO, K, EV>;
    TIMED_LAUNCH(kernel, grid, dim3(kThreads), 0, stream, p, g, partial, tiles, steps);
    return hipGetLastError();
}

template <typename IO, int K, int EV>
hipError_t start_step(const warpctct_conv_step_t &p, hipStream_t stream) {
    const unsigned long long all = (unsigned long long)((p.E + EV - 1) / EV) * (unsigned)p.N;
    auto kernel = conv_step_kernel<IO, K, EV>;
    TIMED_LAUNCH(kernel, dim3((unsigned)((all + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, p);
    return hipGetLastError();
}

// Whether EV channels can be loaded and stored at once: E is a whole number of
// them, and every row of every operand starts where such an access may.
template <typename IO>
bool fits(const warpctct_conv_t &p, int ev) {
    const size_t bytes = ev * sizeof(IO);
    return p.E % ev == 0 && p.x_n % ev == 0 && p.x_t % ev == 0 && aligned(p.x, bytes) && aligned(p.initial, bytes) &&
           aligned(p.out, bytes) && aligned(p.last, bytes);
}

template <typename IO, int K>
hipError_t run(const warpctct_conv_t &p, hipStream_t stream) {
    return fits<IO>(p, 4) ? start<IO, K, 4>(p, stream) : start<IO, K, 1>(p, stream);
}
template <typename IO, int K>
hipError_t run(const warpctct_conv_t &p, const warpctct_conv_grad_t &g, float *partial, hipStream_t stream) {
    const size_t bytes = 4 * sizeof(IO);
    warpctct_conv_t q = p;
    q.out = q.last = nullptr;
    const bool four = fits<IO>(q, 4) && g.grad_n % 4 == 0 && g.grad_t % 4 == 0 && aligned(g.grad_out, bytes) &&
                      aligned(g.grad_last, bytes) && aligned(g.grad_x, bytes) && aligned(g.grad_initial, bytes);
    return four ? start_grad<IO, K, 4>(p, g, partial, stream) : start_grad<IO, K, 1>(p, g, partial, stream);
}
template <typename IO, int K>
hipError_t run(const warpctct_conv_step_t &p, hipStream_t stream) {
    const size_t bytes = 4 * sizeof(IO);
    const bool four = p.E % 4 == 0 && p.x_n % 4 == 0 && aligned(p.x, bytes) && aligned(p.state, bytes) &&
                      aligned(p.out, bytes);
    return four ? start_step<IO, K, 4>(p, stream) : start_step<IO, K, 1>(p, stream);
}

template <typename IO, typename... Args>
hipError_t by_taps(int K, const Args &...args) {
    switch (K) {
        case 1: return run<IO, 1>(args...);
        case 2: return run<IO, 2>(args...);
        case 3: return run<IO, 3>(args...);
        case 4: return run<IO, 4>(args...);
        case 5: return run<IO, 5>(args...);
        case 6: return run<IO, 6>(args...);
        case 7: return run<IO, 7>(args...);
        case 8: return run<IO, 8>(args...);
        default: return hipErrorInvalidValue;
    }
}
template <typename... Args>
hipError_t by_type(int dtype, int K, const Args &...args) {
    if (dtype == kIoF32) return by_taps<float>(K, args...);
    if (dtype == kIoF16) return by_taps<f16>(K, args...);
    return by_taps<bf16>(K, args...);
}

}  // namespace

int conv_grad_tiles(int N, int L, int E) {
    const int steps = conv_grad_steps(N, L, E);
    return L > 0 ? (L + steps - 1) / steps : 1;
}

hipError_t launch_conv(const warpctct_conv_t &p, hipStream_t stream) { return by_type(p.dtype, p.K, p, stream); }

hipError_t launch_conv_grad(const warpctct_conv_t &p, const warpctct_conv_grad_t &g, float *partial,
                            hipStream_t stream) {
    hipError_t e = hipSuccess;
    if (p.N > 0) e = by_type(p.dtype, p.K, p, g, partial, stream);
    if (e != hipSuccess || !(g.grad_weight || g.grad_bias)) return e;
    // (of no sequences the sums are zero: the launch reads nothing then)
    return launch_column_sums(partial, (long)p.N * conv_grad_tiles(p.N, p.L, p.E), {g.grad_weight, p.E * p.K, kIoF32},
                              {g.grad_bias, p.E, kIoF32}, {}, stream);
}

hipError_t launch_conv_step(const warpctct_conv_step_t &p, hipStream_t stream) {
    return by_type(p.dtype, p.K, p, stream);
}

}  // namespace wctct
