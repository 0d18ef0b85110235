// Selective state space scan and its backward pass.  Channel e has S states,
//   d_t = softplus(dt_t + dt_bias)  (or the sum itself)
//   h_t[s] = exp(d_t a[s]) h_{t-1}[s] + d_t x_t b_t[s]
//   y_t = sum_s c_t[s] h_t[s] + skip x_t,   out_t = y_t silu(gate_t)
// and, with gy = g silu(gate) and k_t[s] = exp(d_t a[s]),
//   gh_t[s] = c_t[s] gy_t + k_{t+1}[s] gh_{t+1}[s]
//   gc_t[s] = sum_e gy_t h_t[s],  gb_t[s] = sum_e gh_t[s] d_t x_t
//   gx_t = skip gy_t + d_t sum_s gh_t[s] b_t[s]
//   gd_t = x_t sum_s gh_t[s] b_t[s] + sum_s a[s] gh_t[s] k_t[s] h_{t-1}[s]
//   ga[s] = sum_t d_t gh_t[s] k_t[s] h_{t-1}[s],  gskip = sum_t gy_t x_t
// b and c are shared by the channels of a group.
//
// Bound by arithmetic: a state and a step cost an exponential (two issue slots)
// and four multiply-adds forwards, more than twice that backwards, against 8
// bytes a channel and a step of 2-byte elements for 16 states.  A channel lies on
// LANES lanes next to each other, four states on each, so that the states'
// products are independent work of a lane and their sum a few lane exchanges.  A
// workgroup takes 256 / LANES channels of one group and one sequence and walks
// down time in tiles of 16 steps: what depends on the step and the channel alone
// (softplus, silu, the products with x) is computed once an element, by threads
// that load and store the tile's rows in wide pieces, and handed over in LDS.
// States, sums and exponents are fp32.
//
// Few long sequences are cut into chunks of tiles.  The states behind a chunk
// are exp(a sum d) times those in front of it plus what it makes of zeros, so a
// first pass takes every chunk from zeros (without c and y), a small kernel joins
// them one after the other, and the second pass starts every chunk from its own
// states; the reverse recurrence of gh alike.
//
// Measured with 16 states, bfloat16 and a gate: 32 ragged sequences of 200 to 400
// steps, 1024 channels: forward 58 us, backward 147 us (65 and 176 beside a
// profiler), of which the vector units cannot do without 39 and 112
// (SQ_ACTIVE_INST_VALU); one sequence of 16384 steps, 2048 channels: 242 us in two
// passes, 224 of them the vector units'; one step of 256 sequences, 70 % of which
// advance, 2048 channels: 12.6 us, 4.0 TB/s of what is read and written.
#include <algorithm>
#include <cmath>

#include "network.h"
#include "rows.h"

// products are fused into sums where fmaf says so
#pragma clang fp contract(off)

namespace wctct {

namespace {

constexpr int kThreads = 256;
constexpr int kSteps = 16;                      // of a tile
constexpr int kStates = 4;                      // of a lane
constexpr float kLog2e = 1.4426950408889634f;

// Steps of a tile of the backward pass, which is also how far apart the states
// lie that the forward pass keeps for it: the states and factors of a tile take
// 8 registers a step, and a thread has up to 4 elements.  With 8 steps the kernel
// takes 184 registers, two wavefronts on a SIMD; with 16 it spilled (training on
// the sequences above: 708 us instead of 392 at the time).
constexpr int back_steps(int lanes) { return lanes == 1 ? 4 : lanes == 16 ? 16 : 8; }

// Channels of a row in LDS that the lanes of a channel write at four steps at a
// time: as far apart as a wavefront's channels, so that the four fall into
// different banks.
constexpr int padded(int lanes) { return kThreads / lanes + 64 / lanes; }

// Tiles in LDS at a time.  With two, a tile's results are formed while the next
// tile is worked on, and one barrier a tile is enough; with few or many states they
// take the LDS of the second or third workgroup of a compute unit (32 sequences
// all of 400 steps, 1024 channels, bfloat16, training, one / two: 16 states 273 /
// 268 us, 32 states 465 / 456; 64 states 861 / 866, forwards 180 / 182; of 200 to
// 400 steps, 16 states: 222 / 217).
constexpr int buffers(int lanes) { return lanes == 4 || lanes == 8 ? 2 : 1; }

__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }

// v held within [-most, most]; not a number as it is
__device__ __forceinline__ float within(float v, float most) { return fabsf(v) > most ? copysignf(most, v) : v; }

// a of a state as the power of two that its factor is formed from, finite where a
// log2 e is not: d = 0 (a step that does not count has it) leaves every state as
// it is.
__device__ __forceinline__ float rate_of(float a) { return within(a * kLog2e, 3.402823466e38f); }

// log(1 + e^v) and its derivative.  log1p(q), q = e^-|v| in [0, 1], is
// 2 atanh(q / (2 + q)), whose argument r is at most 1/3.  atanh(r) / r as a
// polynomial of degree 4 in r^2, its coefficients found by Remez exchange for the
// least relative error over [0, 1/9], is off by 8e-9; log2(1 + q) on the
// transcendental unit would lose q itself to the rounding of the sum.
struct Softplus {
    float value, slope;
};
__device__ __forceinline__ Softplus softplus(float v) {
    const float q = exp2_hw(-kLog2e * fabsf(v));
    const float r = q * __builtin_amdgcn_rcpf(2.0f + q), r2 = r * r;
    float s = 0.140891984f;
    s = fmaf(s, r2, 0.139802948f);
    s = fmaf(s, r2, 0.200124562f);
    s = fmaf(s, r2, 0.333331585f);
    s = fmaf(s, r2, 1.0f);
    Softplus p;
    p.value = fmaf(2.0f * r, s, fmaxf(v, 0.0f));
    const float inv = __builtin_amdgcn_rcpf(1.0f + q);
    p.slope = v >= 0.0f ? inv : q * inv;
    return p;
}

// Sum over the LANES lanes of a channel, the same in all of them.
template <int LANES>
__device__ __forceinline__ float channel_sum(float v) {
    if constexpr (LANES >= 2) v += dpp<kDppXor1>(v);
    if constexpr (LANES >= 4) v += dpp<kDppXor2>(v);
    if constexpr (LANES >= 8) v += dpp<0x141 /* row_half_mirror */>(v);
    if constexpr (LANES >= 16) v += dpp<kDppRor8>(v);
    return v;
}

__device__ __forceinline__ float swap_add32(float a, float b) {      // lanes < 32: a's sum, others: b's
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap_add16(float a, float b) {      // even rows of 16: a's, odd rows: b's
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Four values summed over the channels of a wavefront (lanes LANES apart): row r
// of 16 lanes receives value (r & 1) * 2 + (r >> 1).  Halving the values while
// doubling the distance takes 6 exchanges for the first two steps, not 8.
template <int LANES>
__device__ __forceinline__ float sum_over_channels(const float (&v)[kStates]) {
    float s = swap_add16(swap_add32(v[0], v[1]), swap_add32(v[2], v[3]));
    if constexpr (LANES <= 8) s += dpp<kDppRor8>(s);
    if constexpr (LANES <= 4) s += dpp<kDppRor4>(s);
    if constexpr (LANES <= 2) s += dpp<kDppXor2>(s);
    if constexpr (LANES <= 1) s += dpp<kDppXor1>(s);
    return s;
}

// Where a workgroup works: sequence n, channels [first, end) of group g, chunk
// blockIdx.z of the sequence: steps [from, to) of the `len` that count and
// [clear, over) of those that do not.
struct Place {
    int n, g, block, first, end, len, from, to, clear, over;
};
template <int LANES>
__device__ __forceinline__ Place place_of(const warpctct_scan_t &p, int chunk_tiles) {
    constexpr int CH = kThreads / LANES;
    const int per = p.E / p.G, blocks = (per + CH - 1) / CH;
    Place w;
    // First one half of the batch, then the other from its end: of a batch sorted
    // by length a CU that takes two workgroups is given a long sequence and a short
    // one (training on 32 sequences of 200 to 400 steps: 225 us, in order 227).
    const int half = (p.N + 1) / 2;
    w.n = (int)blockIdx.y < half ? blockIdx.y : p.N - 1 - (blockIdx.y - half);
    w.block = blockIdx.x;
    w.g = blockIdx.x / blocks;
    w.first = w.g * per + (blockIdx.x - w.g * blocks) * CH;
    w.end = (w.g + 1) * per;
    w.len = p.lengths ? min(max(p.lengths[w.n], 0), p.L) : p.L;
    const int first = min((int)blockIdx.z * chunk_tiles * kSteps, p.L);
    w.over = blockIdx.z + 1 == gridDim.z ? p.L : min(first + chunk_tiles * kSteps, p.L);
    w.from = min(first, w.len);
    w.to = min(w.over, w.len);
    w.clear = max(first, w.len);
    return w;
}

// A thread's elements of a tile: EPT channels next to each other of one step.
template <int LANES, int STEPS>
struct Elements {
    static constexpr int CH = kThreads / LANES, EPT = STEPS * CH / kThreads;
    int j, c;        // step in the tile, first channel in the workgroup
    __device__ __forceinline__ Elements() {
        const int at = threadIdx.x * EPT;
        j = at / CH;
        c = at % CH;
    }
};

// N elements of a row, in the widest pieces where `wide`; those at or past `have`
// are not written.
template <int N, typename IO>
__device__ __forceinline__ void store_row(IO *p, int have, bool wide, const float (&v)[N]) {
    constexpr int piece = N < 4 ? 1 : (N < kVec<IO> ? 4 : kVec<IO>);
    if (wide && have >= N) {
#pragma unroll
        for (int i = 0; i < N; i += piece) store_n<piece>(p + i, v + i);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < have) p[i] = from_float<IO>(v[i]);
    }
}

// Zeros to the elements of rows [from + j, to) of every `by`: the steps that do not
// count.  (The zeros are opaque to the compiler, which would otherwise write them
// again between two wide stores of them.)
template <int N, typename IO>
__device__ __forceinline__ void clear_rows(IO *p, long stride, int from, int to, int by, int have, bool wide) {
    float zero[N] = {};
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(zero[i]));
    for (int t = from; t < to; t += by) store_row<N>(p + t * stride, have, wide, zero);
}

// The tile's rows of b and c, STEPS x 2 SP values, by all threads: a thread has
// one column of b or of c, and of every kRows steps one.  Where there is nothing
// to read (behind the sequence, past the states) it reads row `safe` of its
// column, or the last state, and puts zero.
template <typename IO, int LANES, int STEPS>
struct Sides {
    static constexpr int SP = kStates * LANES, kRows = kThreads / (2 * SP);
    static constexpr int PER = STEPS > kRows ? STEPS / kRows : 1;
    const IO *at, *safe;
    long stride;
    int j, k;
    bool in;
    IO v[PER];
    __device__ __forceinline__ Sides(const warpctct_scan_t &p, const Place &w, int t0, int safe_row) {
        j = threadIdx.x / (2 * SP);
        k = threadIdx.x % (2 * SP);
        const int s = min(k % SP, p.S - 1);
        in = k % SP < p.S && j < STEPS;
        const IO *base = (k < SP ? static_cast<const IO *>(p.b) + (long)w.n * p.b_n + (long)w.g * p.b_g
                                 : static_cast<const IO *>(p.c) + (long)w.n * p.c_n + (long)w.g * p.c_g) + s;
        stride = k < SP ? p.b_t : p.c_t;
        at = base + (long)(t0 + j) * stride;
        safe = base + safe_row * stride;
    }
    __device__ __forceinline__ void load(int t0, int len) {
#pragma unroll
        for (int i = 0; i < PER; ++i) v[i] = *(t0 + j + i * kRows < len ? at + i * kRows * stride : safe);
    }
    // of the tile at t0, which load() was asked for
    __device__ __forceinline__ void put(float (*bc)[2 * SP], int t0, int len) const {
        if (kRows > STEPS && j >= STEPS) return;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            bc[j + i * kRows][k] = in && t0 + j + i * kRows < len ? to_float(v[i]) : 0.0f;
    }
    __device__ __forceinline__ void advance(int steps) { at += steps * stride; }
};

// A thread's elements of x, dt, gate or grad_out, tile after tile, from a row that
// counts.  In the tile that ends the sequence some threads have none: they are
// shifted onto its last row for that load, and mask what they make of it, as do
// threads past the workgroup's channels, which read its first ones.
template <typename IO, int EPT>
struct Column {
    const IO *at;
    long stride;
    __device__ __forceinline__ Column(const void *base, long start, long t_stride, long row) {
        stride = t_stride;
        at = static_cast<const IO *>(base) + start + row * stride;
    }
    __device__ __forceinline__ void shift(long rows) { at += rows * stride; }
    // the present row, and on by `steps`
    __device__ __forceinline__ void next(Raw<IO, EPT> &v, bool wide, int most, int steps) {
        v.load(at, wide, most);
        at += steps * stride;
    }
};

// Four steps of a tile as a lane takes them out of LDS.
struct Four {
    float2 s[4];                 // d, d x
    float b[4][kStates], c[4][kStates];
};
template <int LANES, bool WITH_C>
__device__ __forceinline__ void load_four(Four &f, const float2 (*steps)[kThreads / LANES],
                                          const float (*bc)[2 * kStates * LANES], int j0, int ch, int q) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f.s[j] = steps[j0 + j][ch];
        *reinterpret_cast<float4 *>(f.b[j]) = *reinterpret_cast<const float4 *>(&bc[j0 + j][q * kStates]);
        if (WITH_C)
            *reinterpret_cast<float4 *>(f.c[j]) =
                *reinterpret_cast<const float4 *>(&bc[j0 + j][kStates * LANES + q * kStates]);
    }
}

// What four lanes q = 0..3 of a channel (or two, or one) hold for four steps,
// summed over the channel's lanes: each step's sum ends on one lane (of every
// four), which holds `kept` of them, the first of them `step`.  Three selects and
// exchanges where a sum for every lane would take two a step, and no branch.
template <int LANES>
struct StepSums {
    static constexpr int kept = LANES >= 4 ? 1 : 4 / LANES;
    static __device__ __forceinline__ int step(int q) {
        return LANES == 1 ? 0 : LANES == 2 ? 2 * q : (q & 1) * 2 + ((q >> 1) & 1);
    }
    static __device__ __forceinline__ void add(const float (&v)[4], int q, float (&r)[kept]) {
        if constexpr (LANES == 1) {
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = v[j];
        } else {
            const bool odd = q & 1, high = q & 2;
            const float u0 = (odd ? v[2] : v[0]) + dpp<kDppXor1>(odd ? v[0] : v[2]);
            const float u1 = (odd ? v[3] : v[1]) + dpp<kDppXor1>(odd ? v[1] : v[3]);
            if constexpr (LANES == 2) {
                r[0] = u0;
                r[1] = u1;
            } else {
                float w = (high ? u1 : u0) + dpp<kDppXor2>(high ? u0 : u1);
                // lane ^ 4: the mirror image within 8 lanes, its quads turned round
                if constexpr (LANES >= 8) w += dpp<0x1B>(dpp<0x141>(w));
                if constexpr (LANES >= 16) w += dpp<kDppRor8>(w);
                r[0] = w;
            }
        }
    }
};

// The first pass over chunks: where a chunk leads from zeros, and its sum of d.
// local (N, chunks, E, SP), total (N, chunks, E).
struct Chunks {
    float *local, *total;
    int tiles;                   // of a chunk
};

// CARRY: the first pass over chunks.  Otherwise from `starts` (laid out like
// Chunks::local, the states in front of every chunk) or, without it, from
// p.initial.
template <typename IO, int LANES, bool CARRY>
__global__ __launch_bounds__(kThreads) void scan_kernel(warpctct_scan_t p, float *__restrict__ keep, Chunks chunks,
                                                        const float *__restrict__ starts, bool wide) {
    constexpr int CH = kThreads / LANES, SP = kStates * LANES, EPT = Elements<LANES, kSteps>::EPT;
    constexpr int PAD = padded(LANES);
    constexpr int BUFS = buffers(LANES);
    __shared__ float2 steps[BUFS][kSteps][CH];     // d, d x
    __shared__ __align__(16) float bc[BUFS][kSteps][2 * SP];
    __shared__ float ys[CARRY ? 1 : BUFS][kSteps][CARRY ? 1 : PAD];
    constexpr int BACK = back_steps(LANES);
    const Place w = place_of<LANES>(p, chunks.tiles);
    const Elements<LANES, kSteps> el;
    // as a lane: a channel and four of its states
    const int ch = threadIdx.x / LANES, q = threadIdx.x % LANES, e = w.first + ch;
    const bool live = e < w.end;
    float a[kStates], h[kStates], total = 0.0f;
    const long state = ((long)w.n * p.E + e) * p.S + q * kStates;
    const long chunk = ((long)w.n * gridDim.z + blockIdx.z) * p.E + e;
#pragma unroll
    for (int i = 0; i < kStates; ++i) {
        const bool in = live && q * kStates + i < p.S;
        a[i] = in ? rate_of(p.a[(long)e * p.S + q * kStates + i]) : 0.0f;
        h[i] = 0.0f;
        if (!CARRY && in && starts)
            h[i] = starts[chunk * SP + q * kStates + i];
        else if (!CARRY && in && p.initial)
            h[i] = p.initial[state + i];
    }
    // as a thread of elements: its channels' parameters and rows
    const int e0 = w.first + el.c, have = max(0, min(EPT, w.end - e0));
    float skip[EPT], bias[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        skip[i] = !CARRY && p.skip && i < have ? p.skip[e0 + i] : 0.0f;
        bias[i] = p.dt_bias && i < have ? p.dt_bias[e0 + i] : 0.0f;
    }
    const int el0 = have > 0 ? e0 : w.first, most = max(have - 1, 0), t1 = w.from + el.j;
    const bool gated = !CARRY && p.gate;
    typedef Raw<IO, EPT> Row;
    Column<IO, EPT> xs(p.x, (long)w.n * p.x_n + el0, p.x_t, t1);
    Column<IO, EPT> ds(p.dt, (long)w.n * p.dt_n + el0, p.dt_t, t1);
    Column<IO, EPT> zs(p.gate, (long)w.n * p.gate_n + el0, p.gate_t, t1);
    IO *out = static_cast<IO *>(p.out) + ((long)w.n * p.L + t1) * p.E + e0;
    typedef Sides<IO, LANES, kSteps> Side;
    Side sides(p, w, w.from, w.from);
    Row x, d, z;
    auto request = [&](int t0) {
        if (t0 + kSteps > w.to) {       // the last tile
            const long past = min(w.to - 1 - t0 - el.j, 0);
            xs.shift(past);
            ds.shift(past);
            zs.shift(past);
        }
        xs.next(x, wide, most, kSteps);
        ds.next(d, wide, most, kSteps);
        if (gated) zs.next(z, wide, most, kSteps);
        sides.load(t0, w.len);
        sides.advance(kSteps);
    };
    // the results of a tile whose sums are in ys
    Row xk, zk;
    bool on = false;
    auto emit = [&](int buf) {
        if (on) {
            float o[EPT];
#pragma unroll
            for (int i = 0; i < EPT; ++i) {
                o[i] = fmaf(skip[i], xk[i], ys[buf][el.j][el.c + i]);
                if (gated) o[i] *= zk[i] * sigmoid(zk[i]);
            }
            store_row<EPT>(out, have, wide, o);
        }
        out += (long)kSteps * p.E;
    };
    if (w.from < w.to) request(w.from);
    int buf = 0;
    for (int t0 = w.from; t0 < w.to; t0 += kSteps) {
        const bool counts = t0 + el.j < w.to;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            float v = d[i] + bias[i];
            if (p.softplus) v = softplus(v).value;
            const bool in = counts && i < have;     // otherwise a step that leaves the state as it is
            v = in ? v : 0.0f;
            steps[buf][el.j][el.c + i] = make_float2(v, in ? v * x[i] : 0.0f);
        }
        sides.put(bc[buf], t0, w.len);
        __syncthreads();
        if (!CARRY && BUFS == 2 && t0 > w.from) emit(buf ^ 1);
        on = counts;
        xk = x;
        zk = z;
        if (t0 + kSteps < w.to) request(t0 + kSteps);
        Four f[2];
        load_four<LANES, !CARRY>(f[0], steps[buf], bc[buf], 0, ch, q);
#pragma unroll
        for (int j0 = 0; j0 < kSteps; j0 += 4) {
            if (t0 + j0 >= w.to) break;
            if (!CARRY && keep && live && j0 % BACK == 0)
                *reinterpret_cast<float4 *>(
                    keep + (((long)w.n * ((p.L + BACK - 1) / BACK) + (t0 + j0) / BACK) * p.E + e) * SP + q * kStates) =
                    make_float4(h[0], h[1], h[2], h[3]);
            const Four &g = f[(j0 / 4) & 1];
            if (j0 + 4 < kSteps) load_four<LANES, !CARRY>(f[(j0 / 4 + 1) & 1], steps[buf], bc[buf], j0 + 4, ch, q);
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                y[j] = 0.0f;
#pragma unroll
                for (int i = 0; i < kStates; ++i) {
                    h[i] = fmaf(exp2_hw(g.s[j].x * a[i]), h[i], g.s[j].y * g.b[j][i]);
                    if (!CARRY) y[j] = fmaf(g.c[j][i], h[i], y[j]);
                }
                if (CARRY) total += g.s[j].x;
            }
            if (!CARRY) {
                float r[StepSums<LANES>::kept];
                StepSums<LANES>::add(y, q, r);
                // (with more than four lanes a channel, groups of four write the same)
#pragma unroll
                for (int j = 0; j < StepSums<LANES>::kept; ++j)
                    ys[buf][j0 + StepSums<LANES>::step(q) + j][ch] = r[j];
            }
        }
        if (BUFS == 1) {
            __syncthreads();
            if (!CARRY) emit(0);
        } else {
            buf ^= 1;
        }
    }
    if (!CARRY && BUFS == 2 && w.from < w.to) {
        __syncthreads();
        emit(buf ^ 1);
    }
    if (CARRY) {
        if (live) {
            *reinterpret_cast<float4 *>(chunks.local + chunk * SP + q * kStates) =
                make_float4(h[0], h[1], h[2], h[3]);
            if (q == 0) chunks.total[chunk] = total;
        }
        return;
    }
    out = static_cast<IO *>(p.out) + (long)w.n * p.L * p.E + e0;
    clear_rows<EPT>(out, p.E, w.clear + el.j, w.over, kSteps, have, wide);
    if (blockIdx.z + 1 != gridDim.z) return;
    if (p.last && live) {
#pragma unroll
        for (int i = 0; i < kStates; ++i)
            if (q * kStates + i < p.S) p.last[state + i] = h[i];
    }
}

// 2^x v as the steps that x is the sum of would leave it: the power alone may be
// beyond the range where the product is not (2^200 times 0, or times 2^-120).
// |x| > 300 takes every v to zero, or what is not zero out of range.
__device__ __forceinline__ float times_exp2(float v, float x) {
    x = within(x, 300.0f);
    const float whole = rintf(x);
    return ldexpf(v * exp2_hw(x - whole), (int)whole);
}

// Joins chunks: turns what each makes of zeros into what stands in front of it,
// in place; backwards for the reverse recurrence, whose end (in front of the
// sequence) goes to `end`.  A thread has one state, and asks for kJoin chunks while
// it joins the kJoin in front of them.
constexpr int kJoin = 16;
__global__ __launch_bounds__(kThreads) void scan_join_kernel(const float *__restrict__ a,
                                                             const float *__restrict__ first,
                                                             Chunks chunks, int count, int E, int S, int SP,
                                                             bool backwards, float *__restrict__ end) {
    const long i = (long)blockIdx.x * kThreads + threadIdx.x;
    if (i >= (long)E * SP) return;
    const int n = blockIdx.y, e = (int)(i / SP), k = (int)(i - (long)e * SP);
    if (k >= S) return;
    const float rate = rate_of(a[(long)e * S + k]);
    const long state = ((long)n * E + e) * S + k;
    float h = first ? first[state] : 0.0f;
    float local[2][kJoin], total[2][kJoin];
    auto request = [&](int c0, float (&l)[kJoin], float (&d)[kJoin]) {
#pragma unroll
        for (int c = 0; c < kJoin; ++c) {
            const int i = min(c0 + c, count - 1), at = backwards ? count - 1 - i : i;
            const long chunk = ((long)n * count + at) * E + e;
            l[c] = chunks.local[chunk * SP + k];
            d[c] = chunks.total[chunk];
        }
    };
    auto join = [&](int c0, const float (&l)[kJoin], const float (&d)[kJoin]) {
#pragma unroll
        for (int c = 0; c < kJoin; ++c) {
            if (c0 + c >= count) break;
            const int at = backwards ? count - 1 - c0 - c : c0 + c;
            chunks.local[(((long)n * count + at) * E + e) * SP + k] = h;
            h = times_exp2(h, rate * d[c]) + l[c];
        }
    };
    request(0, local[0], total[0]);
    for (int c0 = 0; c0 < count; c0 += 2 * kJoin) {
        if (c0 + kJoin < count) request(c0 + kJoin, local[1], total[1]);
        join(c0, local[0], total[0]);
        if (c0 + 2 * kJoin < count) request(c0 + 2 * kJoin, local[0], total[0]);
        join(c0 + kJoin, local[1], total[1]);
    }
    if (end) end[state] = h;
}

// The backward pass walks up time.  A tile's states are computed again from the
// one that the forward pass kept in front of it, into registers, together with
// the factors k; then the tile is walked backwards with gh in registers.  gb and
// gc, sums over channels, are added up within a wavefront by lane exchanges,
// within the workgroup in LDS, and leave as partial sums of the workgroup (row:
// 2 SP floats a step); the sums over time stay in registers until the end.
template <typename IO, int LANES>
__global__ __launch_bounds__(kThreads, 2) void scan_grad_kernel(warpctct_scan_t p, warpctct_scan_grad_t g,
                                                                const float *__restrict__ keep,
                                                                float *__restrict__ part_bc,
                                                                float *__restrict__ part_sums, int chunk_tiles,
                                                                const float *__restrict__ starts, bool wide) {
    constexpr int STEPS = back_steps(LANES);
    constexpr int CH = kThreads / LANES, SP = kStates * LANES, EPT = Elements<LANES, STEPS>::EPT;
    constexpr int WAVES = kThreads / 64;
    constexpr int PAD = padded(LANES);
    constexpr int BUFS = buffers(LANES);
    __shared__ float4 steps[BUFS][STEPS][CH];       // d, d x, gy, -
    __shared__ float ys[BUFS][STEPS][PAD];          // y without the skip
    __shared__ float2 back[BUFS][STEPS][PAD];       // sum gh b, sum a gh k h
    __shared__ __align__(16) float bc[BUFS][STEPS][2 * SP];
    __shared__ float sums[BUFS][WAVES][STEPS][2 * SP];     // gb, gc of a wavefront
    const Place w = place_of<LANES>(p, chunk_tiles);
    const Elements<LANES, STEPS> el;
    const int ch = threadIdx.x / LANES, q = threadIdx.x % LANES, e = w.first + ch;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row16 = lane >> 4;
    const int s_at = q * kStates + (row16 & 1) * 2 + (row16 >> 1);      // see sum_over_channels
    const bool live = e < w.end;
    const int tiles = (p.L + STEPS - 1) / STEPS;
    float a[kStates], carry[kStates], ga[kStates];
    const long state = ((long)w.n * p.E + e) * p.S + q * kStates;
#pragma unroll
    for (int i = 0; i < kStates; ++i) {
        const bool in = live && q * kStates + i < p.S;
        a[i] = in ? p.a[(long)e * p.S + q * kStates + i] : 0.0f;
        carry[i] = 0.0f;
        if (in && starts)
            carry[i] = starts[(((long)w.n * gridDim.z + blockIdx.z) * p.E + e) * SP + q * kStates + i];
        else if (in && g.grad_last)
            carry[i] = g.grad_last[state + i];
        ga[i] = 0.0f;
    }
    const int e0 = w.first + el.c, have = max(0, min(EPT, w.end - e0));
    float skip[EPT], bias[EPT], gskip[EPT], gbias[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        skip[i] = p.skip && i < have ? p.skip[e0 + i] : 0.0f;
        bias[i] = p.dt_bias && i < have ? p.dt_bias[e0 + i] : 0.0f;
        gskip[i] = gbias[i] = 0.0f;
    }
    const long rows = (long)w.n * p.L * p.E + e0;
    IO *gx = static_cast<IO *>(g.grad_x) + rows, *gd = static_cast<IO *>(g.grad_dt) + rows;
    IO *gz = p.gate ? static_cast<IO *>(g.grad_gate) + rows : nullptr;

    clear_rows<EPT>(gx, p.E, w.clear + el.j, w.over, STEPS, have, wide);
    clear_rows<EPT>(gd, p.E, w.clear + el.j, w.over, STEPS, have, wide);
    if (gz) clear_rows<EPT>(gz, p.E, w.clear + el.j, w.over, STEPS, have, wide);
    // the rows of a tile and the states in front of it are asked for while the
    // tile behind it is worked on
    const int top = (w.to + STEPS - 1) / STEPS - 1, bottom = w.from < w.to ? w.from / STEPS : top + 1;
    const long t1 = (long)top * STEPS + el.j;
    const int el0 = have > 0 ? e0 : w.first, most = max(have - 1, 0);
    const bool gated = p.gate;
    typedef Raw<IO, EPT> Row;
    const long past = max(t1 - (w.to - 1), 0L);      // rows from the last one that counts
    Column<IO, EPT> xs(p.x, (long)w.n * p.x_n + el0, p.x_t, t1 - past);
    Column<IO, EPT> ds(p.dt, (long)w.n * p.dt_n + el0, p.dt_t, t1 - past);
    Column<IO, EPT> zs(p.gate, (long)w.n * p.gate_n + el0, p.gate_t, t1 - past);
    Column<IO, EPT> us(g.grad_out, (long)w.n * g.grad_n + el0, g.grad_t, t1 - past);
    const float *fronts = keep + (((long)w.n * tiles + top) * p.E + (live ? e : w.first)) * SP + q * kStates;
    long row = t1 * p.E;         // of the tile that is written next
    typedef Sides<IO, LANES, STEPS> Side;
    Side sides(p, w, top * STEPS, w.from);
    Row x, raw, z, u;
    float4 front;
    auto request = [&](int tile) {
        xs.next(x, wide, most, -STEPS);
        ds.next(raw, wide, most, -STEPS);
        us.next(u, wide, most, -STEPS);
        if (gated) zs.next(z, wide, most, -STEPS);
        sides.load(tile * STEPS, w.len);
        front = *reinterpret_cast<const float4 *>(fronts);
        fronts -= (long)p.E * SP;
        sides.advance(-STEPS);
    };
    if (top >= bottom) {
        request(top);
        xs.shift(past);
        ds.shift(past);
        us.shift(past);
        zs.shift(past);
    }
    // the results of a tile whose sums are in `back`, `ys` and `sums`
    float d[EPT], slope[EPT];
    Row xk, uk, zk;
    bool on = false;
    auto emit = [&](int buf, int tile) {
        if (on) {
            float ox[EPT], od[EPT], oz[EPT];
#pragma unroll
            for (int i = 0; i < EPT; ++i) {
                const float2 s = back[buf][el.j][el.c + i];
                ox[i] = fmaf(d[i], s.x, skip[i] * steps[buf][el.j][el.c + i].z);
                od[i] = fmaf(xk[i], s.x, s.y) * slope[i];
                if (i < have) gbias[i] += od[i];
                if (gated) {
                    const float sg = sigmoid(zk[i]);
                    oz[i] = uk[i] * fmaf(skip[i], xk[i], ys[buf][el.j][el.c + i]) *
                            (sg * fmaf(zk[i], 1.0f - sg, 1.0f));
                }
            }
            store_row<EPT>(gx + row, have, wide, ox);
            store_row<EPT>(gd + row, have, wide, od);
            if (gz) store_row<EPT>(gz + row, have, wide, oz);
        }
        row -= (long)STEPS * p.E;
        float *to = part_bc + (((long)w.n * gridDim.x + w.block) * tiles + tile) * (STEPS * 2 * SP);
        for (int at = threadIdx.x; at < STEPS * 2 * SP; at += kThreads) {
            float s = 0.0f;
#pragma unroll
            for (int v = 0; v < WAVES; ++v) s += sums[buf][v][at / (2 * SP)][at % (2 * SP)];
            to[at] = s;
        }
    };
    int buf = 0;
    for (int tile = top; tile >= bottom; --tile) {
        const bool counts = tile * STEPS + el.j < w.to;
        float dk[EPT], slopek[EPT];
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const float v = raw[i] + bias[i];
            dk[i] = v;
            slopek[i] = 1.0f;
            if (p.softplus) {
                const Softplus s = softplus(v);
                dk[i] = s.value;
                slopek[i] = s.slope;
            }
            float gy = u[i], xi = x[i];
            if (gated) gy *= z[i] * sigmoid(z[i]);
            if (!(counts && i < have)) dk[i] = gy = xi = 0.0f;
            steps[buf][el.j][el.c + i] = make_float4(dk[i], dk[i] * xi, gy, 0.0f);
            gskip[i] = fmaf(gy, xi, gskip[i]);
        }
        sides.put(bc[buf], tile * STEPS, w.len);
        const float h0[kStates] = {live ? front.x : 0.0f, live ? front.y : 0.0f, live ? front.z : 0.0f,
                                   live ? front.w : 0.0f};
        __syncthreads();
        if (BUFS == 2 && tile < top) emit(buf ^ 1, tile + 1);
        on = counts;
        xk = x;
        uk = u;
        zk = z;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            d[i] = dk[i];
            slope[i] = slopek[i];
        }
        if (tile > bottom) request(tile - 1);
        float k[STEPS][kStates], h[STEPS][kStates];
#pragma unroll
        for (int j0 = 0; j0 < STEPS; j0 += 4) {
            float y[4];
#pragma unroll
            for (int j = j0; j < j0 + 4; ++j) {
                const float2 s = *reinterpret_cast<const float2 *>(&steps[buf][j][ch]);
                const float4 b4 = *reinterpret_cast<const float4 *>(&bc[buf][j][q * kStates]);
                const float b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
                for (int i = 0; i < kStates; ++i) {
                    k[j][i] = exp2_hw(s.x * rate_of(a[i]));
                    h[j][i] = fmaf(k[j][i], j ? h[j - 1][i] : h0[i], s.y * b[i]);
                }
                const float4 c4 = *reinterpret_cast<const float4 *>(&bc[buf][j][SP + q * kStates]);
                y[j - j0] = fmaf(c4.w, h[j][3], fmaf(c4.z, h[j][2], fmaf(c4.y, h[j][1], c4.x * h[j][0])));
            }
            if (gated) {
                float r[StepSums<LANES>::kept];
                StepSums<LANES>::add(y, q, r);
#pragma unroll
                for (int j = 0; j < StepSums<LANES>::kept; ++j) ys[buf][j0 + StepSums<LANES>::step(q) + j][ch] = r[j];
            }
        }
#pragma unroll
        for (int j0 = STEPS - 4; j0 >= 0; j0 -= 4) {
            float ghb[4], akh[4];
#pragma unroll
            for (int j = j0 + 3; j >= j0; --j) {
                const float4 s = steps[buf][j][ch];
                const float4 b4 = *reinterpret_cast<const float4 *>(&bc[buf][j][q * kStates]);
                const float4 c4 = *reinterpret_cast<const float4 *>(&bc[buf][j][SP + q * kStates]);
                const float b[4] = {b4.x, b4.y, b4.z, b4.w}, c[4] = {c4.x, c4.y, c4.z, c4.w};
                float vb[kStates], vc[kStates];
                ghb[j - j0] = akh[j - j0] = 0.0f;
#pragma unroll
                for (int i = 0; i < kStates; ++i) {
                    const float gh = fmaf(c[i], s.z, carry[i]);
                    ghb[j - j0] = fmaf(gh, b[i], ghb[j - j0]);
                    vb[i] = gh * s.y;
                    vc[i] = h[j][i] * s.z;
                    carry[i] = gh * k[j][i];
                    const float r = carry[i] * (j ? h[j - 1][i] : h0[i]);
                    akh[j - j0] = fmaf(a[i], r, akh[j - j0]);
                    ga[i] = fmaf(s.x, r, ga[i]);
                }
                const float sb = sum_over_channels<LANES>(vb), sc = sum_over_channels<LANES>(vc);
                // (lanes of a row that hold the same sum write it to the same place)
                sums[buf][wave][j][s_at] = sb;
                sums[buf][wave][j][SP + s_at] = sc;
            }
            float rb[StepSums<LANES>::kept], ra[StepSums<LANES>::kept];
            StepSums<LANES>::add(ghb, q, rb);
            StepSums<LANES>::add(akh, q, ra);
#pragma unroll
            for (int j = 0; j < StepSums<LANES>::kept; ++j)
                back[buf][j0 + StepSums<LANES>::step(q) + j][ch] = make_float2(rb[j], ra[j]);
        }
        if (BUFS == 1) {
            __syncthreads();
            emit(0, tile);
        } else {
            buf ^= 1;
        }
    }
    if (BUFS == 2 && top >= bottom) {
        __syncthreads();
        emit(buf ^ 1, bottom);
    }
    if (g.grad_initial && !starts && live) {
#pragma unroll
        for (int i = 0; i < kStates; ++i)
            if (q * kStates + i < p.S) g.grad_initial[state + i] = carry[i];
    }
    // the sums over time: a row of E S + 2 E floats for every chunk
    float *mine = part_sums + ((size_t)w.n * gridDim.z + blockIdx.z) * p.E * (p.S + 2);
    if (live) {
#pragma unroll
        for (int i = 0; i < kStates; ++i)
            if (q * kStates + i < p.S) mine[(long)e * p.S + q * kStates + i] = ga[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EPT; ++i) steps[0][el.j][el.c + i] = make_float4(gskip[i], gbias[i], 0.0f, 0.0f);
    __syncthreads();
    for (int c = threadIdx.x; c < CH; c += kThreads) {
        if (w.first + c >= w.end) continue;
        float s = 0.0f, b = 0.0f;
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
            s += steps[0][j][c].x;
            b += steps[0][j][c].y;
        }
        mine[(long)p.E * p.S + w.first + c] = s;
        mine[(long)p.E * p.S + p.E + w.first + c] = b;
    }
}

// The first pass of the reverse recurrence over chunks: what each makes of zeros
// behind it, k_t gh_t of its first step, and its sum of d.
template <typename IO, int LANES>
__global__ __launch_bounds__(kThreads) void scan_grad_carry_kernel(warpctct_scan_t p, warpctct_scan_grad_t g,
                                                                   Chunks chunks, bool wide) {
    constexpr int CH = kThreads / LANES, SP = kStates * LANES, EPT = Elements<LANES, kSteps>::EPT;
    __shared__ float2 steps[kSteps][CH];           // d, gy
    __shared__ __align__(16) float bc[kSteps][2 * SP];
    const Place w = place_of<LANES>(p, chunks.tiles);
    const Elements<LANES, kSteps> el;
    const int ch = threadIdx.x / LANES, q = threadIdx.x % LANES, e = w.first + ch;
    const bool live = e < w.end;
    float a[kStates], carry[kStates], total = 0.0f;
#pragma unroll
    for (int i = 0; i < kStates; ++i) {
        const bool in = live && q * kStates + i < p.S;
        a[i] = in ? rate_of(p.a[(long)e * p.S + q * kStates + i]) : 0.0f;
        carry[i] = 0.0f;
    }
    const int e0 = w.first + el.c, have = max(0, min(EPT, w.end - e0));
    float bias[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) bias[i] = p.dt_bias && i < have ? p.dt_bias[e0 + i] : 0.0f;
    const int last = w.from + (w.to - w.from - 1) / kSteps * kSteps;
    const long t1 = last + el.j;
    const int el0 = have > 0 ? e0 : w.first, most = max(have - 1, 0);
    const bool gated = p.gate;
    const long past = max(t1 - (w.to - 1), 0L);
    Column<IO, EPT> ds(p.dt, (long)w.n * p.dt_n + el0, p.dt_t, t1 - past);
    Column<IO, EPT> zs(p.gate, (long)w.n * p.gate_n + el0, p.gate_t, t1 - past);
    Column<IO, EPT> us(g.grad_out, (long)w.n * g.grad_n + el0, g.grad_t, t1 - past);
    typedef Sides<IO, LANES, kSteps> Side;
    Side sides(p, w, last, w.from);
    Raw<IO, EPT> d, u, z;
    auto request = [&](int t0) {
        ds.next(d, wide, most, -kSteps);
        us.next(u, wide, most, -kSteps);
        if (gated) zs.next(z, wide, most, -kSteps);
        sides.load(t0, w.len);
        sides.advance(-kSteps);
    };
    if (w.from < w.to) {
        request(last);
        ds.shift(past);
        us.shift(past);
        zs.shift(past);
    }
    for (int t0 = w.from < w.to ? last : -1; t0 >= w.from; t0 -= kSteps) {
        const bool on = t0 + el.j < w.to;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            float v = d[i] + bias[i];
            if (p.softplus) v = softplus(v).value;
            float y = u[i];
            if (gated) y *= z[i] * sigmoid(z[i]);
            if (!(on && i < have)) v = y = 0.0f;
            steps[el.j][el.c + i] = make_float2(v, y);
        }
        sides.put(bc, t0, w.len);
        __syncthreads();
        if (t0 - kSteps >= w.from) request(t0 - kSteps);
#pragma unroll
        for (int j = kSteps - 1; j >= 0; --j) {
            const float2 s = steps[j][ch];
            const float4 c4 = *reinterpret_cast<const float4 *>(&bc[j][SP + q * kStates]);
            const float c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
            for (int i = 0; i < kStates; ++i) carry[i] = exp2_hw(s.x * a[i]) * fmaf(c[i], s.y, carry[i]);
            total += s.x;
        }
        __syncthreads();
    }
    if (!live) return;
    const long chunk = ((long)w.n * gridDim.z + blockIdx.z) * p.E + e;
    *reinterpret_cast<float4 *>(chunks.local + chunk * SP + q * kStates) =
        make_float4(carry[0], carry[1], carry[2], carry[3]);
    if (q == 0) chunks.total[chunk] = total;
}

// gb, gc (N, L, G, S): the workgroups' partial sums of a group added up, zero
// behind a sequence.  A thread has one value; `rows` steps a workgroup.
template <typename IO>
__global__ __launch_bounds__(kThreads) void scan_grad_bc_kernel(warpctct_scan_t p, warpctct_scan_grad_t g,
                                                                const float *__restrict__ part_bc, int blocks,
                                                                int SP, int rows) {
    const int n = blockIdx.y, GS = p.G * p.S;
    const long i = (long)blockIdx.x * kThreads + threadIdx.x;
    if (i >= (long)p.L * 2 * GS) return;
    const int t = (int)(i / (2 * GS)), k = (int)(i - (long)t * 2 * GS), v = k % GS, grp = v / p.S, s = v % p.S;
    const int len = p.lengths ? min(max(p.lengths[n], 0), p.L) : p.L;
    float sum = 0.0f;
    if (t < len) {
        const float *from =
            part_bc + (((long)n * p.G + grp) * blocks * rows + t) * (2 * SP) + (k < GS ? 0 : SP) + s;
#pragma unroll 4
        for (int b = 0; b < blocks; ++b) sum += from[(long)b * rows * 2 * SP];
    }
    IO *to = static_cast<IO *>(k < GS ? g.grad_b : g.grad_c);
    to[((long)n * p.L + t) * GS + v] = from_float<IO>(sum);
}

// One step of N sequences; a channel lies on LANES lanes, and a thread takes its
// four states of `BATCH` sequences, so that a is read once for them.  WIDE: b, c,
// a and the states in pieces of four.
template <typename IO, int LANES, int BATCH, bool WIDE>
__global__ __launch_bounds__(kThreads) void scan_step_kernel(warpctct_scan_step_t p) {
    const long i0 = (long)blockIdx.x * kThreads + threadIdx.x;
    if (i0 >= (long)p.E * LANES) return;           // all lanes of a channel
    const int e = (int)(i0 / LANES), q = threadIdx.x % LANES, s0 = q * kStates, grp = e / (p.E / p.G);
    const int most = max(min(kStates, p.S - s0) - 1, 0), s1 = min(s0, p.S - 1);
    const float *ap = p.a + (long)e * p.S + s1;
    float a[kStates];
    Raw<float, kStates> ar;
    ar.load(ap, WIDE, most);
#pragma unroll
    for (int i = 0; i < kStates; ++i) a[i] = rate_of(ar[i]);
    const float bias = p.dt_bias ? p.dt_bias[e] : 0.0f, skip = p.skip ? p.skip[e] : 0.0f;
    for (long n0 = (long)blockIdx.y * BATCH; n0 < p.N; n0 += (long)gridDim.y * BATCH) {
        Raw<float, kStates> h[BATCH];
        Raw<IO, kStates> b[BATCH], c[BATCH];
        IO x[BATCH], d[BATCH], z[BATCH];
        bool go[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const long n = min(n0 + k, (long)p.N - 1);
            // (the same for the whole workgroup: a sequence that stays is not read)
            go[k] = __builtin_amdgcn_readfirstlane(n0 + k < p.N && (!p.advance || p.advance[n]));
            if (!go[k]) continue;
            h[k].load(p.state + (n * p.E + e) * p.S + s1, WIDE, most);
            b[k].load(static_cast<const IO *>(p.b) + n * p.b_n + grp * p.b_g + s1, WIDE, most);
            c[k].load(static_cast<const IO *>(p.c) + n * p.c_n + grp * p.c_g + s1, WIDE, most);
            x[k] = static_cast<const IO *>(p.x)[n * p.x_n + e];
            d[k] = static_cast<const IO *>(p.dt)[n * p.dt_n + e];
            if (p.gate) z[k] = static_cast<const IO *>(p.gate)[n * p.gate_n + e];
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            if (n0 + k >= p.N) break;
            float y = 0.0f;
            if (go[k]) {
                const float xv = to_float(x[k]);
                float dv = to_float(d[k]) + bias;
                if (p.softplus) dv = softplus(dv).value;
                const float dx = dv * xv;
                float hv[kStates];
#pragma unroll
                for (int i = 0; i < kStates; ++i) {
                    hv[i] = fmaf(exp2_hw(dv * a[i]), h[k][i], dx * b[k][i]);
                    y = s0 + i < p.S ? fmaf(c[k][i], hv[i], y) : y;
                }
                float *to = p.state + ((n0 + k) * p.E + e) * p.S + s0;
                if (WIDE) {
                    store_n<kStates>(to, hv);
                } else {
#pragma unroll
                    for (int i = 0; i < kStates; ++i)
                        if (s0 + i < p.S) to[i] = hv[i];
                }
                y = fmaf(skip, xv, channel_sum<LANES>(y));
                if (p.gate) {
                    const float zv = to_float(z[k]);
                    y *= zv * sigmoid(zv);
                }
            }
            if (q == 0) static_cast<IO *>(p.out)[(n0 + k) * p.E + e] = from_float<IO>(y);
        }
    }
}

// steps, rounded up to whole tiles of the backward pass
int back_rows(int L, int lanes) {
    const int steps = back_steps(lanes);
    return (L + steps - 1) / steps * steps;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int lanes_of(int S) {
    int lanes = 1;
    while (lanes * kStates < S) lanes *= 2;
    return lanes;
}
int blocks_of(const warpctct_scan_t &p) {      // of a group
    const int ch = kThreads / lanes_of(p.S);
    return (p.E / p.G + ch - 1) / ch;
}

// Rows may be read and written in 16-byte pieces: so are they spaced and aligned,
// every group starts at a multiple of 16 bytes, and a thread has all of its `ept`
// channels or none.
template <typename IO>
bool rows_wide(const warpctct_scan_t &p, int ept) {
    constexpr int V = kVec<IO>;
    return p.E % V == 0 && (p.E / p.G) % V == 0 && (p.E / p.G) % ept == 0 && p.x_n % V == 0 &&
           p.x_t % V == 0 && p.dt_n % V == 0 && p.dt_t % V == 0 && p.gate_n % V == 0 && p.gate_t % V == 0 &&
           aligned16(p.x) && aligned16(p.dt) && aligned16(p.gate) && aligned16(p.out);
}

// Chunks that a sequence is cut into.  Two passes cost twice the arithmetic
// forwards and a quarter more backwards, but a wavefront alone on its SIMD waits
// most of the time: sequences are cut up to 768 wavefronts of them uncut (1024
// SIMDs) forwards and 1024 backwards, into as many chunks as put eight wavefronts
// on each, of two tiles at least.  The limits are those that long sequences gain by
// without short ones losing much.  Measured with 1024 channels, 16 states, 1500
// steps (us, uncut / cut): forwards 512 wavefronts 186 / 102, 768 186 / 139, 1024
// 188 / 178, 1536 245 / 272; backwards 1024 595 / 454, 1536 746 / 711, 2048
// 751 / 885; with 300 steps forwards 768 41 / 45 (a loss), backwards 1024
// 130 / 111, 1536 157 / 162.  Fewer than 8 tiles are not worth the two launches more, and more
// than 8 sqrt(tiles) chunks take longer to join than they save (2 us a tile for a
// wavefront on its own).
struct Cut {
    int count, tiles;
};
Cut cut_of(const warpctct_scan_t &p, bool backward) {
    const long waves = (long)p.N * p.G * blocks_of(p) * (kThreads / 64), tiles = ((long)p.L + kSteps - 1) / kSteps;
    Cut c = {1, (int)tiles};
    if (waves <= 0 || waves > (backward ? 1024 : 768) || tiles < 8) return c;
    const long count = std::min(std::min(8192 / waves, tiles / 2), (long)(8.0 * std::sqrt((double)tiles)));
    c.tiles = (int)((tiles + count - 1) / count);
    c.count = (int)((tiles + c.tiles - 1) / c.tiles);
    return c;
}
size_t chunk_floats(const warpctct_scan_t &p, bool backward) {
    const Cut c = cut_of(p, backward);
    return c.count > 1 ? (size_t)p.N * c.count * p.E * (kStates * lanes_of(p.S) + 1) : 0;
}
Chunks chunks_of(const warpctct_scan_t &p, const Cut &c, float *workspace) {
    Chunks k;
    k.local = workspace;
    k.total = workspace + (c.count > 1 ? (size_t)p.N * c.count * p.E * (kStates * lanes_of(p.S)) : 0);
    k.tiles = c.tiles;
    return k;
}
hipError_t join_chunks(const warpctct_scan_t &p, const float *first, const Chunks &chunks, int count, bool backwards,
                       float *end, hipStream_t stream) {
    const int SP = kStates * lanes_of(p.S);
    const long threads = (long)p.E * SP;
    TIMED_LAUNCH(scan_join_kernel, dim3((unsigned)((threads + kThreads - 1) / kThreads), p.N), dim3(kThreads), 0,
                 stream, p.a, first, chunks, count, p.E, p.S, SP, backwards, end);
    return hipGetLastError();
}

template <typename IO, int LANES>
hipError_t start(const warpctct_scan_t &p, float *keep, float *workspace, hipStream_t stream) {
    const Cut cut = cut_of(p, false);
    const Chunks chunks = chunks_of(p, cut, workspace);
    const dim3 grid(p.G * blocks_of(p), p.N, cut.count);
    const bool wide = rows_wide<IO>(p, Elements<LANES, kSteps>::EPT);
    if (cut.count > 1) {
        auto carry = scan_kernel<IO, LANES, true>;
        TIMED_LAUNCH(carry, grid, dim3(kThreads), 0, stream, p, nullptr, chunks, nullptr, wide);
        const hipError_t e = join_chunks(p, p.initial, chunks, cut.count, false, nullptr, stream);
        if (e != hipSuccess) return e;
    }
    auto kernel = scan_kernel<IO, LANES, false>;
    TIMED_LAUNCH(kernel, grid, dim3(kThreads), 0, stream, p, keep, chunks, cut.count > 1 ? chunks.local : nullptr,
                 wide);
    return hipGetLastError();
}

template <typename IO, int LANES>
hipError_t start(const warpctct_scan_t &p, const warpctct_scan_grad_t &g, const float *keep, float *part_bc,
                 float *part_sums, float *workspace, hipStream_t stream) {
    constexpr int V = kVec<IO>;
    const bool wide = rows_wide<IO>(p, Elements<LANES, kSteps>::EPT) && g.grad_n % V == 0 &&
                      g.grad_t % V == 0 && aligned16(g.grad_out) &&
                      aligned16(g.grad_x) && aligned16(g.grad_dt) && aligned16(g.grad_gate);
    const int blocks = blocks_of(p);
    if (p.N == 0) return hipSuccess;
    const Cut cut = cut_of(p, true);
    const Chunks chunks = chunks_of(p, cut, workspace);
    const dim3 grid(p.G * blocks, p.N, cut.count);
    hipError_t e;
    if (cut.count > 1) {
        auto carry = scan_grad_carry_kernel<IO, LANES>;
        TIMED_LAUNCH(carry, grid, dim3(kThreads), 0, stream, p, g, chunks, wide);
        e = join_chunks(p, g.grad_last, chunks, cut.count, true, g.grad_initial, stream);
        if (e != hipSuccess) return e;
    }
    auto kernel = scan_grad_kernel<IO, LANES>;
    TIMED_LAUNCH(kernel, grid, dim3(kThreads), 0, stream, p, g, keep, part_bc, part_sums, cut.tiles,
                 cut.count > 1 ? chunks.local : nullptr, wide);
    e = hipGetLastError();
    if (e != hipSuccess || p.L == 0) return e;
    auto join = scan_grad_bc_kernel<IO>;
    const long values = (long)p.L * 2 * p.G * p.S;
    TIMED_LAUNCH(join, dim3((unsigned)((values + kThreads - 1) / kThreads), p.N), dim3(kThreads), 0, stream, p, g,
                 part_bc, blocks, kStates * LANES, back_rows(p.L, LANES));
    return hipGetLastError();
}

template <typename IO, int LANES, int BATCH>
hipError_t start_step(const warpctct_scan_step_t &p, hipStream_t stream) {
    const long groups = ((long)p.E * LANES + kThreads - 1) / kThreads, batches = ((long)p.N + BATCH - 1) / BATCH;
    const size_t four = kStates * sizeof(IO);
    const bool wide = p.S == kStates * LANES && aligned16(p.state) && aligned16(p.a) && p.b_n % kStates == 0 &&
                      p.b_g % kStates == 0 && p.c_n % kStates == 0 && p.c_g % kStates == 0 &&
                      (reinterpret_cast<uintptr_t>(p.b) | reinterpret_cast<uintptr_t>(p.c)) % four == 0;
    auto kernel = wide ? scan_step_kernel<IO, LANES, BATCH, true> : scan_step_kernel<IO, LANES, BATCH, false>;
    TIMED_LAUNCH(kernel, dim3((unsigned)groups, (unsigned)std::min(batches, 65535L)), dim3(kThreads), 0, stream, p);
    return hipGetLastError();
}
template <typename IO, int LANES>
hipError_t start(const warpctct_scan_step_t &p, hipStream_t stream) {
    // two sequences a thread once there are eight workgroups a compute unit with them
    const long groups = ((long)p.E * LANES + kThreads - 1) / kThreads * p.N;
    return groups >= 4096 ? start_step<IO, LANES, 2>(p, stream) : start_step<IO, LANES, 1>(p, stream);
}

template <typename IO, typename... Args>
hipError_t by_states(int S, const Args &...args) {
    switch (lanes_of(S)) {
        case 1: return start<IO, 1>(args...);
        case 2: return start<IO, 2>(args...);
        case 4: return start<IO, 4>(args...);
        case 8: return start<IO, 8>(args...);
        case 16: return start<IO, 16>(args...);
        default: return hipErrorInvalidValue;
    }
}
template <typename... Args>
hipError_t by_type(int dtype, int S, const Args &...args) {
    if (dtype == kIoF32) return by_states<float>(S, args...);
    if (dtype == kIoF16) return by_states<f16>(S, args...);
    return by_states<bf16>(S, args...);
}

size_t part_bc_floats(const warpctct_scan_t &p) {
    const int lanes = lanes_of(p.S);
    return (size_t)p.N * p.G * blocks_of(p) * back_rows(p.L, lanes) * 2 * kStates * lanes;
}

}  // namespace

size_t scan_keep_floats(int N, int L, int E, int S) {
    const int lanes = lanes_of(S);
    return (size_t)N * (back_rows(L, lanes) / back_steps(lanes)) * E * (kStates * lanes);
}

size_t scan_floats(const warpctct_scan_t &p) { return chunk_floats(p, false); }

size_t scan_grad_floats(const warpctct_scan_t &p) {
    return part_bc_floats(p) + chunk_floats(p, true) +
           column_sums_floats((long)p.N * cut_of(p, true).count, (long)p.E * (p.S + 2));
}

hipError_t launch_scan(const warpctct_scan_t &p, float *keep, float *workspace, hipStream_t stream) {
    return by_type(p.dtype, p.S, p, keep, workspace, stream);
}

hipError_t launch_scan_grad(const warpctct_scan_t &p, const warpctct_scan_grad_t &g, const float *keep,
                            float *workspace, hipStream_t stream) {
    float *part_bc = workspace, *local = part_bc + part_bc_floats(p), *part_sums = local + chunk_floats(p, true);
    const hipError_t e = by_type(p.dtype, p.S, p, g, keep, part_bc, part_sums, local, stream);
    if (e != hipSuccess) return e;
    return launch_column_sums(part_sums, (long)p.N * cut_of(p, true).count, {g.grad_a, p.E * p.S, kIoF32},
                              {g.grad_skip, p.E, kIoF32}, {g.grad_dt_bias, p.E, kIoF32}, stream);
}

hipError_t launch_scan_step(const warpctct_scan_step_t &p, hipStream_t stream) {
    return by_type(p.dtype, p.S, p, stream);
}

}  // namespace wctct
