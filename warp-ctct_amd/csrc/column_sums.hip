// Sums down the columns of a matrix of partial sums: what the backward passes of
// layer norm, the causal convolution and the selective scan leave for gradients
// of parameters, which every row or sequence contributes to.  No atomics: the
// order of the additions is fixed by the sizes.
#include "network.h"
#include "rows.h"

namespace wctct {

namespace {

// A workgroup takes 64 columns by 16 strands of rows; the strands are added up
// in order.  Up to kDirect rows one launch does it; beyond, a first launch leaves
// kParts rows (4096 rows of 380 columns: 6 workgroups alone would walk down 256
// rows each).
constexpr int kStrands = 16;
constexpr long kDirect = 1024;
constexpr int kParts = 64;

__device__ __forceinline__ void store_as(void *p, int type, int at, float v) {
    if (type == kIoF32)
        static_cast<float *>(p)[at] = v;
    else if (type == kIoF16)
        static_cast<f16 *>(p)[at] = (f16)v;
    else
        static_cast<bf16 *>(p)[at] = (bf16)v;
}

__global__ __launch_bounds__(64 * kStrands) void column_sums_kernel(const float *__restrict__ partial, long rows,
                                                                    int columns, SumsTo first, SumsTo second,
                                                                    SumsTo third) {
    __shared__ float strands[kStrands][64];
    const int lane = threadIdx.x & 63, strand = threadIdx.x >> 6, k = blockIdx.x * 64 + lane;
    // the rows of this part (all of them where gridDim.y is 1)
    const long per = (rows + gridDim.y - 1) / gridDim.y;
    const long from = blockIdx.y * per, to = min(rows, from + per);
    float sum = 0.0f;
    if (k < columns) {
#pragma unroll 8
        for (long r = from + strand; r < to; r += kStrands) sum += partial[r * columns + k];
    }
    strands[strand][lane] = sum;
    __syncthreads();
    if (strand != 0 || k >= columns) return;
    for (int s = 1; s < kStrands; ++s) sum += strands[s][lane];
    if (gridDim.y > 1) {
        static_cast<float *>(first.p)[(long)blockIdx.y * columns + k] = sum;
        return;
    }
    const int j = k - first.count;
    if (j < 0) {
        if (first.p) store_as(first.p, first.type, k, sum);
    } else if (j < second.count) {
        if (second.p) store_as(second.p, second.type, j, sum);
    } else if (third.p) {
        store_as(third.p, third.type, j - second.count, sum);
    }
}

}  // namespace

size_t column_sums_floats(long rows, long columns) {
    return (size_t)(rows > kDirect ? rows + kParts : rows) * (size_t)columns;
}

hipError_t launch_column_sums(float *partial, long rows, SumsTo first, SumsTo second, SumsTo third,
                              hipStream_t stream) {
    const int columns = first.count + second.count + third.count;
    const unsigned groups = (columns + 63) / 64;
    if (rows > kDirect) {
        float *fewer = partial + (size_t)rows * columns;
        const SumsTo all = {fewer, columns, kIoF32}, none = {};
        TIMED_LAUNCH(column_sums_kernel, dim3(groups, kParts), dim3(64 * kStrands), 0, stream, partial, rows,
                     columns, all, none, none);
        partial = fewer;
        rows = kParts;
    }
    TIMED_LAUNCH(column_sums_kernel, dim3(groups), dim3(64 * kStrands), 0, stream, partial, rows, columns, first,
                 second, third);
    return hipGetLastError();
}

}  // namespace wctct
