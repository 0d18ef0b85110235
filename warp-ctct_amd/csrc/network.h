// Internal launch interface of the operators beside the losses (layer norm,
// causal convolution, selective scan, rules on logits) between the C ABI
// (network_api.hip) and their kernels.  Structs of device pointers and sizes;
// each launcher enqueues on the given stream and returns hipGetLastError().
#pragma once

#include <hip/hip_runtime.h>

#include "launch.h"
#include "warp_ctct_hip.h"

namespace wctct {

hipError_t launch_layer_norm(const warpctct_norm_t &p, hipStream_t stream);
// workgroups of the backward pass, each of which leaves 2 * width partial sums
int norm_grad_groups(long rows, int width);
hipError_t launch_layer_norm_grad(const warpctct_norm_t &p, const warpctct_norm_grad_t &g,
                                  float *partial, hipStream_t stream);

// Where the sums of a run of columns go: `count` of them in an element type, or
// nowhere (null).
struct SumsTo {
    void *p;
    int count, type;
};
// Sums down `rows` rows of partial (rows, columns), in a fixed order; the columns
// are those of to[0], then to[1], then to[2].  `partial` holds
// column_sums_floats(rows, columns) floats: the rows, and behind them room for a
// second level where there are many.
size_t column_sums_floats(long rows, long columns);
hipError_t launch_column_sums(float *partial, long rows, SumsTo first, SumsTo second, SumsTo third,
                              hipStream_t stream);

hipError_t launch_conv(const warpctct_conv_t &p, hipStream_t stream);
// tiles of time that a sequence is cut into by the backward pass, each of which
// leaves (K + 1) * E partial sums per sequence
int conv_grad_tiles(int N, int L, int E);
hipError_t launch_conv_grad(const warpctct_conv_t &p, const warpctct_conv_grad_t &g, float *partial,
                            hipStream_t stream);
hipError_t launch_conv_step(const warpctct_conv_step_t &p, hipStream_t stream);

// floats that the forward pass keeps for the backward: the states in front of every tile
size_t scan_keep_floats(int N, int L, int E, int S);
// floats of scratch that the two passes take (16-byte aligned)
size_t scan_floats(const warpctct_scan_t &p);
size_t scan_grad_floats(const warpctct_scan_t &p);
hipError_t launch_scan(const warpctct_scan_t &p, float *keep, float *workspace, hipStream_t stream);
hipError_t launch_scan_grad(const warpctct_scan_t &p, const warpctct_scan_grad_t &g, const float *keep,
                            float *workspace, hipStream_t stream);
hipError_t launch_scan_step(const warpctct_scan_step_t &p, hipStream_t stream);

hipError_t launch_adjust(const warpctct_adjust_t &p, hipStream_t stream);

}  // namespace wctct
