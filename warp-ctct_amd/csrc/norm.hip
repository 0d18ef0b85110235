// Layer norm over the last dimension, and its backward pass:
//   m = mean x,  r = (mean (x - m)^2 + eps)^(-1/2),  h = (x - m) r,  out = h weight + bias
//   u = g weight,  gx = r (u - mean u - h mean(u h)),  gweight = sum_rows g h,  gbias = sum_rows g
// Bound by HBM: a row is read once into registers (twice in the backward: x and
// g) and written once.  The mean is taken twice, the second time of x - m, so
// that rows whose mean is large against their deviation lose nothing to the
// rounding of the first; sums, statistics and the column sums of the weight's
// gradient are fp32.  12800 rows of 2048 bfloat16 elements: forward 24 us (4.4
// TB/s), backward 36 us (4.3 TB/s) and 5 us for the column sums.
#include "network.h"
#include "rows.h"

// A product is fused into a sum only where fmaf says so: a mean that is rounded
// in one place and part of a fused x - sum * inv in another would put rows far
// from zero off by half a step of their mean.
#pragma clang fp contract(off)

namespace wctct {

namespace {

constexpr int kThreads = 256;        // of a workgroup whose wavefronts take a row each
constexpr int kWide = 1024;          // the largest number of threads on one row
constexpr unsigned kGroups = 1024;   // workgroups of the forward pass, at most
constexpr unsigned kWideGroups = 1u << 20;      // and where a row does not fit into their registers
// and of the backward pass: four on a compute unit where they take a row each, two
// where their wavefronts do (12800 rows of 2048 elements: 36.6 us with 1024, 42.0
// with 512; 2592 rows of 641: 16.2 with 1024, 11.4 with 512).  Measured at these
// widths alone: at several times 2048 the 8 bytes a column that every workgroup
// leaves come to as much as the rows.
constexpr int kGradGroups = 1024, kGradGroupsOfWaves = 512;

// Sums of two values over the threads of a row: a wavefront (threads == 64) or
// the whole workgroup.  `shared` holds 2 floats per wavefront and is free again
// when the call returns.
__device__ __forceinline__ void row_sums(float &a, float &b, int threads, float *shared) {
    a = wave_sum(a);
    b = wave_sum(b);
    if (threads == 64) return;
    const int wave = threadIdx.x >> 6, waves = threads >> 6;
    if ((threadIdx.x & 63) == 0) {
        shared[2 * wave] = a;
        shared[2 * wave + 1] = b;
    }
    __syncthreads();
    a = 0.0f;
    b = 0.0f;
    for (int w = 0; w < waves; ++w) {
        a += shared[2 * w];
        b += shared[2 * w + 1];
    }
    __syncthreads();
}

// What the backward pass keeps of a row: the first mean, what it was off by, and
// the inverse deviation.  (Their sum as one float would shift every normalised
// value of a row by up to |mean| / deviation units in the last place.)
struct RowStats {
    float m, c, r;
    __device__ __forceinline__ float normalise(float x) const { return ((x - m) - c) * r; }
};
__device__ __forceinline__ RowStats row_stats(const float *stats, unsigned row) {
    const float *s = stats + 3 * (size_t)row;
    return RowStats{s[0], s[1], s[2]};
}
__device__ __forceinline__ void keep_stats(float *stats, unsigned row, float m, float c, float r) {
    float *s = stats + 3 * (size_t)row;
    s[0] = m;
    s[1] = c;
    s[2] = r;
}

// How the elements of a row are dealt to its threads: slot i of thread t is
// element (i / EV * threads + t) * EV + i % EV, EV = 1 or a 16-byte vector.
template <typename IO, bool VEC, int CAP>
struct Slots {
    static constexpr int EV = VEC ? kVec<IO> : 1;
    static constexpr int NV = CAP / EV;
    static __device__ __forceinline__ int first(int j, int t, int threads) {
        return (j * threads + t) * EV;
    }
    // A row as it was loaded.  All loads are issued together, those past the row
    // at its last elements; unpack() masks them.
    struct Row {
        Raw<IO, EV> v[NV];
    };
    static __device__ __forceinline__ void load(Row &r, const IO *row, int width, int t, int threads) {
#pragma unroll
        for (int j = 0; j < NV; ++j) r.v[j].load(row + min(first(j, t, threads), width - EV), true, 0);
    }
    static __device__ __forceinline__ void unpack(const Row &r, int width, int t, int threads, float (&x)[CAP]) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const bool in = first(j, t, threads) < width;
#pragma unroll
            for (int i = 0; i < EV; ++i) x[j * EV + i] = in ? r.v[j][i] : 0.0f;
        }
    }
    static __device__ __forceinline__ void store(IO *row, int width, int t, int threads, const float (&x)[CAP]) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = first(j, t, threads);
            if (at < width) {
                store_n<EV>(row + at, x + j * EV);
            }
        }
    }
    // a parameter of the columns, `other` where there is none (its start need not
    // be aligned)
    template <typename W>
    static __device__ __forceinline__ void load_param(const W *p, float other, int width, int t, int threads,
                                                      float (&x)[CAP]) {
#pragma unroll
        for (int i = 0; i < CAP; ++i) x[i] = other;
        if (!p) return;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = min(first(j, t, threads), width - EV);
#pragma unroll
            for (int i = 0; i < EV; ++i) x[j * EV + i] = to_float(p[at + i]);
        }
    }
};

template <typename IO, typename W, bool VEC, int CAP, int BLOCK>
__global__ __launch_bounds__(BLOCK) void norm_kernel(const IO *__restrict__ x, RowAddress at,
                                                     const W *__restrict__ weight, const W *__restrict__ bias,
                                                     float eps, IO *__restrict__ out, float *__restrict__ stats,
                                                     unsigned rows, int width, int threads) {
    typedef Slots<IO, VEC, CAP> S;
    __shared__ float shared[2 * kWide / 64];
    const int t = threads == 64 ? threadIdx.x & 63 : threadIdx.x;
    const unsigned per = threads == 64 ? blockDim.x >> 6 : 1u;
    const unsigned stride = gridDim.x * per;
    unsigned row = blockIdx.x * per + (threads == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
    if (row >= rows) return;      // whole wavefronts; a workgroup on one row always has one
    const float inv = 1.0f / (float)width;
    typename S::Row raw;
    S::load(raw, x + at.at(row), width, t, threads);
    float w[CAP], b[CAP];
    S::load_param(weight, 1.0f, width, t, threads, w);
    S::load_param(bias, 0.0f, width, t, threads, b);
    for (; row < rows; row += stride) {
        float v[CAP];
        S::unpack(raw, width, t, threads, v);
        // the next row, while this one is worked on
        if (rows - row > stride) S::load(raw, x + at.at(row + stride), width, t, threads);
        float sum = 0.0f, none = 0.0f;
#pragma unroll
        for (int i = 0; i < CAP; ++i) sum += v[i];
        row_sums(sum, none, threads, shared);
        const float m = sum * inv;
        float off = 0.0f, sq = 0.0f;
#pragma unroll
        for (int j = 0; j < S::NV; ++j) {
            const bool in = S::first(j, t, threads) < width;
#pragma unroll
            for (int i = 0; i < S::EV; ++i) {
                float &e = v[j * S::EV + i];
                e = in ? e - m : 0.0f;
                off += e;
                sq = fmaf(e, e, sq);
            }
        }
        row_sums(off, sq, threads, shared);
        const float c = off * inv;                       // what the first mean was off by
        const float var = fmaxf(sq * inv - c * c, 0.0f);
        const float r = 1.0f / sqrtf(var + eps);
        if (stats && t == 0) keep_stats(stats, row, m, c, r);
#pragma unroll
        for (int i = 0; i < CAP; ++i) v[i] = fmaf((v[i] - c) * r, w[i], b[i]);
        S::store(out + (long)row * width, width, t, threads, v);
    }
}

// Rows too wide for the registers of one workgroup: three passes over the row.
// (As in the backward pass, a workgroup takes more rows than one where there are
// more than a launch has workgroups.)
template <typename IO, typename W>
__global__ __launch_bounds__(kWide) void norm_wide_kernel(const IO *__restrict__ x, RowAddress at,
                                                          const W *__restrict__ weight,
                                                          const W *__restrict__ bias, float eps,
                                                          IO *__restrict__ out, float *__restrict__ stats, unsigned rows,
                                                          int width) {
    __shared__ float shared[2 * kWide / 64];
    const float inv = 1.0f / (float)width;
    for (unsigned row = blockIdx.x; row < rows; row += gridDim.x) {
        const IO *in = x + at.at(row);
        float sum = 0.0f, none = 0.0f;
        for (int k = threadIdx.x; k < width; k += kWide) sum += to_float(in[k]);
        row_sums(sum, none, kWide, shared);
        const float m = sum * inv;
        float off = 0.0f, sq = 0.0f;
        for (int k = threadIdx.x; k < width; k += kWide) {
            const float d = to_float(in[k]) - m;
            off += d;
            sq = fmaf(d, d, sq);
        }
        row_sums(off, sq, kWide, shared);
        const float c = off * inv;
        const float r = 1.0f / sqrtf(fmaxf(sq * inv - c * c, 0.0f) + eps);
        if (stats && threadIdx.x == 0) keep_stats(stats, row, m, c, r);
        for (int k = threadIdx.x; k < width; k += kWide) {
            float v = (to_float(in[k]) - m - c) * r * (weight ? to_float(weight[k]) : 1.0f);
            if (bias) v += to_float(bias[k]);
            out[(long)row * width + k] = from_float<IO>(v);
        }
    }
}

// The backward pass: a wavefront (or workgroup) walks over rows, a fixed number
// apart, and keeps the column sums of its rows in registers; the wavefronts of a
// workgroup add theirs up in LDS, in order, and a workgroup leaves one row of
// 2 * width partial sums, which column_sums_kernel adds up: no atomics, the same
// result on every call.
template <typename IO, typename W, bool VEC, int CAP, int BLOCK>
__global__ __launch_bounds__(BLOCK) void norm_grad_kernel(
    const IO *__restrict__ x, RowAddress x_at, const IO *__restrict__ g, RowAddress g_at,
    const W *__restrict__ weight, const float *__restrict__ stats,
    IO *__restrict__ gx, float *__restrict__ partial, unsigned rows, int width, int threads) {
    typedef Slots<IO, VEC, CAP> S;
    __shared__ float shared[2 * kWide / 64];
    extern __shared__ float columns[];               // 2 * width, where wavefronts take rows each
    const int t = threads == 64 ? threadIdx.x & 63 : threadIdx.x;
    const int per = threads == 64 ? blockDim.x >> 6 : 1;      // rows of this workgroup at a time
    const int wave = threads == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const float inv = 1.0f / (float)width;
    float w[CAP], gw[CAP], gb[CAP];
    S::load_param(weight, 1.0f, width, t, threads, w);
#pragma unroll
    for (int i = 0; i < CAP; ++i) gw[i] = gb[i] = 0.0f;
    const unsigned stride = gridDim.x * per;
    unsigned row = blockIdx.x * per + wave;
    typename S::Row xr, gr;
    if (row < rows) {
        S::load(xr, x + x_at.at(row), width, t, threads);
        S::load(gr, g + g_at.at(row), width, t, threads);
    }
    for (; row < rows; row += stride) {
        float h[CAP], e[CAP];
        S::unpack(xr, width, t, threads, h);
        S::unpack(gr, width, t, threads, e);
        if (rows - row > stride) {      // the next row, while this one is worked on
            S::load(xr, x + x_at.at(row + stride), width, t, threads);
            S::load(gr, g + g_at.at(row + stride), width, t, threads);
        }
        const RowStats s = row_stats(stats, row);
        float su = 0.0f, suh = 0.0f;
#pragma unroll
        for (int i = 0; i < CAP; ++i) {
            h[i] = s.normalise(h[i]);
            gb[i] += e[i];                            // (e is 0 past the row)
            gw[i] = fmaf(e[i], h[i], gw[i]);
            e[i] *= w[i];
            su += e[i];
            suh = fmaf(e[i], h[i], suh);
        }
        if (!gx) continue;
        row_sums(su, suh, threads, shared);
        su *= inv;
        suh *= inv;
#pragma unroll
        for (int i = 0; i < CAP; ++i) e[i] = s.r * (e[i] - su - h[i] * suh);
        S::store(gx + (long)row * width, width, t, threads, e);
    }
    if (!partial) return;
    float *mine = partial + (size_t)blockIdx.x * 2 * width;
    for (int turn = 0; turn < per; ++turn) {
        if (turn == wave) {
            float *to = per == 1 ? mine : columns;
#pragma unroll
            for (int j = 0; j < S::NV; ++j) {
                const int at = S::first(j, t, threads);
                if (at < width) {
#pragma unroll
                    for (int i = 0; i < S::EV; ++i) {
                        const int k = at + i;
                        to[k] = gw[j * S::EV + i] + (turn ? to[k] : 0.0f);
                        to[width + k] = gb[j * S::EV + i] + (turn ? to[width + k] : 0.0f);
                    }
                }
            }
        }
        if (per > 1) __syncthreads();
    }
    if (per > 1)
        for (int k = threadIdx.x; k < 2 * width; k += blockDim.x) mine[k] = columns[k];
}

// The same for rows too wide for registers: gx in two passes over a row, the
// column sums by threads that walk down their columns.
template <typename IO, typename W>
__global__ __launch_bounds__(kWide) void norm_wide_grad_kernel(
    const IO *__restrict__ x, RowAddress x_at, const IO *__restrict__ g, RowAddress g_at,
    const W *__restrict__ weight, const float *__restrict__ stats,
    IO *__restrict__ gx, unsigned rows, int width) {
    __shared__ float shared[2 * kWide / 64];
    const float inv = 1.0f / (float)width;
    for (unsigned row = blockIdx.x; row < rows; row += gridDim.x) {
        const IO *in = x + x_at.at(row), *up = g + g_at.at(row);
        const RowStats s = row_stats(stats, row);
        float su = 0.0f, suh = 0.0f;
        for (int k = threadIdx.x; k < width; k += kWide) {
            const float u = to_float(up[k]) * (weight ? to_float(weight[k]) : 1.0f);
            su += u;
            suh = fmaf(u, s.normalise(to_float(in[k])), suh);
        }
        row_sums(su, suh, kWide, shared);
        su *= inv;
        suh *= inv;
        for (int k = threadIdx.x; k < width; k += kWide) {
            const float u = to_float(up[k]) * (weight ? to_float(weight[k]) : 1.0f);
            gx[(long)row * width + k] = from_float<IO>(s.r * (u - su - s.normalise(to_float(in[k])) * suh));
        }
    }
}
template <typename IO>
__global__ __launch_bounds__(kThreads) void norm_wide_columns_kernel(
    const IO *__restrict__ x, RowAddress x_at, const IO *__restrict__ g, RowAddress g_at,
    const float *__restrict__ stats, float *__restrict__ partial, unsigned rows,
    int width) {
    const int k = blockIdx.x * kThreads + threadIdx.x;
    if (k >= width) return;
    float gw = 0.0f, gb = 0.0f;
    for (unsigned row = blockIdx.y; row < rows; row += gridDim.y) {
        const float e = to_float(g[g_at.at(row) + k]);
        gb += e;
        gw = fmaf(e, row_stats(stats, row).normalise(to_float(x[x_at.at(row) + k])), gw);
    }
    float *mine = partial + (size_t)blockIdx.y * 2 * width;
    mine[k] = gw;
    mine[width + k] = gb;
}

RowAddress address(long rows, long inner_rows, long outer_stride, long inner_stride) {
    RowAddress a;
    a.inner = inner_rows >= rows ? 0u : (unsigned)inner_rows;
    a.outer_stride = outer_stride;
    a.inner_stride = inner_stride;
    return a;
}

// Every row of a strided operand starts on a 16-byte boundary.
bool rows_aligned(const void *p, const RowAddress &a, size_t size) {
    const size_t ev = 16 / size;
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && a.inner_stride % (long)ev == 0 &&
           (a.inner == 0u || a.outer_stride % (long)ev == 0);
}

// Threads on a row and elements of each: a wavefront, 256 or 1024 threads, with as
// many elements as leave them their registers (a lane of 1024 threads has 128).
// A wavefront alone saves the exchanges through LDS; the backward pass, which
// holds five values an element, and rows that are not loaded in vectors, whose
// elements take a register each until they are used, are better off with more
// threads (12800 rows of 2048 bfloat16: forward 24.2 us by wavefronts against 27.4
// by 256 threads, backward 50.3 against 42.2).  0: no shape holds the row.
int threads_for(int width, bool backward, bool vec) {
    const int most = !backward && vec ? 32 : 16;
    if (width <= most * 64) return 64;
    if (width <= most * kThreads) return kThreads;
    return width <= most / 2 * kWide ? kWide : 0;
}

template <typename IO, typename W, bool VEC, int CAP, int BLOCK>
hipError_t start(const warpctct_norm_t &p, const RowAddress &at, int threads, hipStream_t stream) {
    const unsigned rows = (unsigned)p.rows;
    const unsigned groups = threads == 64 ? (rows + 3) / 4 : rows;
    const dim3 grid(groups < kGroups ? groups : kGroups), block(BLOCK);
    auto kernel = norm_kernel<IO, W, VEC, CAP, BLOCK>;
    TIMED_LAUNCH(kernel, grid, block, 0, stream, static_cast<const IO *>(p.x), at, static_cast<const W *>(p.weight),
                 static_cast<const W *>(p.bias), p.eps, static_cast<IO *>(p.out), p.stats, rows, p.width,
                 threads);
    return hipGetLastError();
}

template <typename IO, typename W>
hipError_t start(const warpctct_norm_t &p, hipStream_t stream) {
    const RowAddress at = address(p.rows, p.x_inner_rows, p.x_outer_stride, p.x_inner_stride);
    const bool vec = p.width % kVec<IO> == 0 && rows_aligned(p.x, at, sizeof(IO)) &&
                     (reinterpret_cast<uintptr_t>(p.out) & 15u) == 0;
    const int threads = threads_for(p.width, false, vec);
    if (threads == 0) {
        auto kernel = norm_wide_kernel<IO, W>;
        const unsigned rows = (unsigned)p.rows;
        TIMED_LAUNCH(kernel, dim3(rows < kWideGroups ? rows : kWideGroups), dim3(kWide), 0, stream,
                     static_cast<const IO *>(p.x), at, static_cast<const W *>(p.weight),
                     static_cast<const W *>(p.bias), p.eps, static_cast<IO *>(p.out), p.stats, rows, p.width);
        return hipGetLastError();
    }
    if (threads == kWide)
        return vec ? start<IO, W, true, 16, kWide>(p, at, threads, stream)
                   : start<IO, W, false, 8, kWide>(p, at, threads, stream);
    if (p.width <= 8 * threads)
        return vec ? start<IO, W, true, 8, kThreads>(p, at, threads, stream)
                   : start<IO, W, false, 8, kThreads>(p, at, threads, stream);
    if (p.width <= 16 * threads)
        return vec ? start<IO, W, true, 16, kThreads>(p, at, threads, stream)
                   : start<IO, W, false, 16, kThreads>(p, at, threads, stream);
    return start<IO, W, true, 32, kThreads>(p, at, threads, stream);
}

template <typename IO, typename W, bool VEC, int CAP, int BLOCK>
hipError_t start_grad(const warpctct_norm_t &p, const warpctct_norm_grad_t &g, const RowAddress &x_at,
                      const RowAddress &g_at, int threads, float *partial, hipStream_t stream) {
    const dim3 grid(norm_grad_groups(p.rows, p.width)), block(BLOCK);
    const size_t shared = threads == 64 && partial ? 2 * sizeof(float) * p.width : 0;
    auto kernel = norm_grad_kernel<IO, W, VEC, CAP, BLOCK>;
    TIMED_LAUNCH(kernel, grid, block, shared, stream, static_cast<const IO *>(p.x), x_at,
                 static_cast<const IO *>(g.grad_out), g_at, static_cast<const W *>(p.weight), p.stats,
                 static_cast<IO *>(g.grad_x), partial, (unsigned)p.rows, p.width, threads);
    return hipGetLastError();
}

template <typename IO, typename W>
hipError_t start_grad(const warpctct_norm_t &p, const warpctct_norm_grad_t &g, float *partial, hipStream_t stream) {
    const RowAddress x_at = address(p.rows, p.x_inner_rows, p.x_outer_stride, p.x_inner_stride);
    const RowAddress g_at = address(p.rows, g.inner_rows, g.outer_stride, g.inner_stride);
    const bool vec = p.width % kVec<IO> == 0 && rows_aligned(p.x, x_at, sizeof(IO)) &&
                     rows_aligned(g.grad_out, g_at, sizeof(IO)) &&
                     (reinterpret_cast<uintptr_t>(g.grad_x) & 15u) == 0;
    const int threads = threads_for(p.width, true, vec);
    if (threads == 0) {
        const unsigned rows = (unsigned)p.rows;
        if (g.grad_x) {
            auto kernel = norm_wide_grad_kernel<IO, W>;
            TIMED_LAUNCH(kernel, dim3(rows < kWideGroups ? rows : kWideGroups), dim3(kWide), 0, stream,
                         static_cast<const IO *>(p.x), x_at, static_cast<const IO *>(g.grad_out), g_at,
                         static_cast<const W *>(p.weight), p.stats, static_cast<IO *>(g.grad_x), rows, p.width);
        }
        if (partial) {
            auto kernel = norm_wide_columns_kernel<IO>;
            const dim3 grid((p.width + kThreads - 1) / kThreads, norm_grad_groups(p.rows, p.width));
            TIMED_LAUNCH(kernel, grid, dim3(kThreads), 0, stream, static_cast<const IO *>(p.x), x_at,
                         static_cast<const IO *>(g.grad_out), g_at, p.stats, partial, rows, p.width);
        }
        return hipGetLastError();
    }
    if (threads == kWide)
        return vec ? start_grad<IO, W, true, 8, kWide>(p, g, x_at, g_at, threads, partial, stream)
                   : start_grad<IO, W, false, 8, kWide>(p, g, x_at, g_at, threads, partial, stream);
    if (p.width <= 8 * threads)
        return vec ? start_grad<IO, W, true, 8, kThreads>(p, g, x_at, g_at, threads, partial, stream)
                   : start_grad<IO, W, false, 8, kThreads>(p, g, x_at, g_at, threads, partial, stream);
    return vec ? start_grad<IO, W, true, 16, kThreads>(p, g, x_at, g_at, threads, partial, stream)
               : start_grad<IO, W, false, 16, kThreads>(p, g, x_at, g_at, threads, partial, stream);
}

}  // namespace

int norm_grad_groups(long rows, int width) {
    const long per = threads_for(width, true, false) == 64 ? 4 : 1;      // rows of a workgroup at a time
    const long groups = (rows + per - 1) / per;
    const long most = per == 1 ? kGradGroups : kGradGroupsOfWaves;
    return (int)(groups < most ? groups : most);
}

hipError_t launch_layer_norm(const warpctct_norm_t &p, hipStream_t stream) {
    const bool same = p.weight_dtype == p.dtype;
    if (p.dtype == kIoF32) return start<float, float>(p, stream);
    if (p.dtype == kIoF16) return same ? start<f16, f16>(p, stream) : start<f16, float>(p, stream);
    return same ? start<bf16, bf16>(p, stream) : start<bf16, float>(p, stream);
}

hipError_t launch_layer_norm_grad(const warpctct_norm_t &p, const warpctct_norm_grad_t &g, float *partial,
                                  hipStream_t stream) {
    const bool same = p.weight_dtype == p.dtype;
    hipError_t e;
    if (p.dtype == kIoF32)
        e = start_grad<float, float>(p, g, partial, stream);
    else if (p.dtype == kIoF16)
        e = same ? start_grad<f16, f16>(p, g, partial, stream) : start_grad<f16, float>(p, g, partial, stream);
    else
        e = same ? start_grad<bf16, bf16>(p, g, partial, stream) : start_grad<bf16, float>(p, g, partial, stream);
    if (e != hipSuccess || !partial) return e;
    return launch_column_sums(partial, norm_grad_groups(p.rows, p.width), {g.grad_weight, p.width, p.weight_dtype},
                              {g.grad_bias, p.width, p.weight_dtype}, {}, stream);
}

}  // namespace wctct
