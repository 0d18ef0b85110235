// Loads, stores and reductions shared by the operators that work on rows of
// float, half or bfloat16 elements in 16-byte vectors (norm.hip, conv.hip,
// scan.hip, adjust.hip).  All arithmetic is in fp32; a store rounds to nearest
// even, once.
#pragma once

#include <hip/hip_runtime.h>

namespace wctct {

typedef __bf16 bf16;
typedef _Float16 f16;
typedef unsigned int raw16 __attribute__((ext_vector_type(4)));

// elements per 16-byte vector
template <typename IO>
constexpr int kVec = 16 / (int)sizeof(IO);

template <typename IO>
__device__ __forceinline__ float to_float(IO v) { return (float)v; }
template <typename IO>
__device__ __forceinline__ IO from_float(float v) { return (IO)v; }

// two floats rounded to nearest even into one word of 2-byte elements
__device__ __forceinline__ unsigned pack_two(const f16 *, float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef f16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f2){a, b}, h2));
}
__device__ __forceinline__ unsigned pack_two(const bf16 *, float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(unsigned, __builtin_convertvector((f2){a, b}, b2));
}
__device__ __forceinline__ raw16 pack16(const float *, const float *x) {
    return raw16{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]),
                 __float_as_uint(x[3])};
}
template <typename IO>
__device__ __forceinline__ raw16 pack16(const IO *p, const float *x) {
    return raw16{pack_two(p, x[0], x[1]), pack_two(p, x[2], x[3]), pack_two(p, x[4], x[5]),
                 pack_two(p, x[6], x[7])};
}
// N elements next to each other (1, 4, or a 16-byte vector), aligned to their size
template <int N, typename IO>
__device__ __forceinline__ void load_n(const IO *p, float *x) {
    if constexpr (N == 1) {
        x[0] = to_float(*p);
    } else {
        typedef IO piece __attribute__((ext_vector_type(N)));
        const piece v = *reinterpret_cast<const piece *>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (float)v[i];
    }
}
template <int N, typename IO>
__device__ __forceinline__ void store_n(IO *p, const float *x) {
    if constexpr (N == 1) {
        *p = from_float<IO>(x[0]);
    } else if constexpr (N == kVec<IO>) {
        *reinterpret_cast<raw16 *>(p) = pack16(p, x);
    } else {
        static_assert(N == 4 && sizeof(IO) == 2, "1, 4 elements or a vector");
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack_two(p, x[0], x[1]), pack_two(p, x[2], x[3]));
    }
}

// N elements next to each other as they are loaded, not yet converted: a
// conversion waits for its load, so loads that are to be in flight together, or
// while something else is worked on, are kept in this form.  `wide`: the start is
// aligned for pieces of up to 16 bytes; otherwise element i is p[min(i, most)].
template <typename IO, int N>
struct Raw {
    static constexpr int kPiece = N * (int)sizeof(IO) > 16 ? kVec<IO> : N;
    typedef IO piece __attribute__((ext_vector_type(kPiece)));
    piece v[N / kPiece];
    __device__ __forceinline__ void load(const IO *p, bool wide, int most) {
        if (wide) {
#pragma unroll
            for (int k = 0; k < N / kPiece; ++k) v[k] = *reinterpret_cast<const piece *>(p + k * kPiece);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i / kPiece][i % kPiece] = p[min(i, most)];
        }
    }
    __device__ __forceinline__ float operator[](int i) const { return (float)v[i / kPiece][i % kPiece]; }
};
template <typename IO>
struct Raw<IO, 1> {
    IO v;
    __device__ __forceinline__ void load(const IO *p, bool, int) { v = *p; }
    __device__ __forceinline__ float operator[](int) const { return (float)v; }
};

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __uint_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E;        // quad_perm [1,0,3,2], [2,3,0,1]
constexpr int kDppRor4 = 0x124, kDppRor8 = 0x128;      // rotations within 16 lanes

// v of lane l plus v of lane l ^ 16 / l ^ 32, in every lane
__device__ __forceinline__ float add_xor16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_xor32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Sum over the wavefront, the same bits in every lane: each step adds the two
// halves of a pair of lanes.  (The rotation by 8 comes before that by 4, which
// pairs lanes l and l ^ 4 only once l and l ^ 8 hold the same.)
__device__ __forceinline__ float wave_sum(float v) {
    v += dpp<kDppXor1>(v);
    v += dpp<kDppXor2>(v);
    v += dpp<kDppRor8>(v);
    v += dpp<kDppRor4>(v);
    return add_xor32(add_xor16(v));
}

__device__ __forceinline__ float sigmoid(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
}

// Rows of a tensor whose leading dimensions are addressed by two strides (in
// elements): row i starts at (i / inner) * outer_stride + (i % inner) * inner_stride.
struct RowAddress {
    unsigned inner;      // rows per outer index; 0: all rows lie inner_stride apart
    long outer_stride, inner_stride;
    __device__ __forceinline__ long at(unsigned row) const {
        if (inner == 0u) return (long)row * inner_stride;
        const unsigned o = row / inner;
        return (long)o * outer_stride + (long)(row - o * inner) * inner_stride;
    }
};

}  // namespace wctct
