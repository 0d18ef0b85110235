// extern "C" surface of the operators beside the losses (declared in
// include/warp_ctct_hip.h).  Host code only: argument validation and kernel
// launches.  No allocation, no host synchronisation, no process exit.
#include <hip/hip_runtime.h>

#include "network.h"
#include "warp_ctct_hip.h"

namespace {

using namespace wctct;

inline hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }

inline int done(hipError_t e) {
    if (e == hipSuccess) return WARPCTCT_OK;
    return e == hipErrorInvalidValue ? WARPCTCT_EINVAL : WARPCTCT_ELAUNCH;
}

constexpr long kMostRows = 0x7fffffffL;
constexpr int kMostBatch = 65535;      // a grid dimension, as for the losses
// A launch has fewer than 2^32 threads: the sums down columns take 16 a column,
// other kernels one a value.
constexpr long kMostColumns = (1L << 28) - 64, kMostThreads = (1L << 32) - 1024;

bool norm_ok(const warpctct_norm_t *p) {
    return p && io_valid(p->dtype) && (p->weight_dtype == p->dtype || p->weight_dtype == WARPCTCT_F32) &&
           p->width >= 1 && 2L * p->width <= kMostColumns && p->rows >= 0 && p->rows <= kMostRows &&
           (p->rows == 0 || (p->x && p->x_inner_rows >= 1));
}

bool conv_ok(const warpctct_conv_t *p) {
    return p && io_valid(p->dtype) && p->N >= 0 && p->N <= kMostBatch && p->L >= 0 && p->E >= 1 && p->K >= 1 &&
           p->K <= WARPCTCT_CONV_MAX_TAPS && (long)p->E * (p->K + 1) <= kMostColumns && p->L <= (1 << 30) &&
           (long)p->L * p->E <= kMostThreads && (p->N == 0 || (p->weight && (p->x || p->L == 0)));
}

bool scan_sizes_ok(int dtype, int N, int L, int E, int S, int G) {
    return io_valid(dtype) && N >= 0 && N <= kMostBatch && L >= 0 && E >= 1 && E < (1 << 24) && S >= 1 &&
           S <= WARPCTCT_SCAN_MAX_STATES && G >= 1 && E % G == 0 && 2L * L * G * S <= kMostThreads &&
           (long)E * (S + 2) <= kMostColumns && L <= (1 << 30);
}
bool scan_ok(const warpctct_scan_t *p) {
    return p && scan_sizes_ok(p->dtype, p->N, p->L, p->E, p->S, p->G) &&
           (p->N == 0 || (p->a && (p->L == 0 || (p->x && p->dt && p->b && p->c))));
}

}  // namespace

extern "C" {

int warpctct_layer_norm(const warpctct_norm_t *p, void *stream) {
    if (!norm_ok(p)) return WARPCTCT_EINVAL;
    if (p->rows == 0) return WARPCTCT_OK;
    if (!p->out) return WARPCTCT_EINVAL;
    return done(launch_layer_norm(*p, as_stream(stream)));
}

size_t warpctct_layer_norm_workspace_bytes(long rows, int width) {
    if (rows < 0 || rows > kMostRows || width < 1) return 0;
    const long groups = rows > 0 ? norm_grad_groups(rows, width) : 1;
    return column_sums_floats(groups, 2L * width) * sizeof(float);
}

int warpctct_layer_norm_grad(const warpctct_norm_t *p, const warpctct_norm_grad_t *g, void *workspace,
                             size_t workspace_bytes, void *stream) {
    if (!norm_ok(p) || !g) return WARPCTCT_EINVAL;
    const bool columns = g->grad_weight || g->grad_bias;
    if (p->rows > 0 && (!p->stats || !g->grad_out || g->inner_rows < 1)) return WARPCTCT_EINVAL;
    if (columns && !workspace) return WARPCTCT_EINVAL;
    if (columns && workspace_bytes < warpctct_layer_norm_workspace_bytes(p->rows, p->width))
        return WARPCTCT_EWORKSPACE;
    float *partial = columns ? static_cast<float *>(workspace) : nullptr;
    if (p->rows == 0) {     // the sums of no rows: zeros
        if (!columns) return WARPCTCT_OK;
        return done(launch_column_sums(partial, 0, {g->grad_weight, p->width, p->weight_dtype},
                                       {g->grad_bias, p->width, p->weight_dtype}, {}, as_stream(stream)));
    }
    if (!g->grad_x && !columns) return WARPCTCT_OK;
    return done(launch_layer_norm_grad(*p, *g, partial, as_stream(stream)));
}

int warpctct_causal_conv(const warpctct_conv_t *p, void *stream) {
    if (!conv_ok(p)) return WARPCTCT_EINVAL;
    if (p->N == 0) return WARPCTCT_OK;
    if (!p->out && p->L > 0) return WARPCTCT_EINVAL;
    return done(launch_conv(*p, as_stream(stream)));
}

size_t warpctct_causal_conv_workspace_bytes(int N, int L, int E, int K) {
    if (N < 0 || L < 0 || E < 1 || K < 1 || K > WARPCTCT_CONV_MAX_TAPS) return 0;
    return column_sums_floats((long)N * conv_grad_tiles(N, L, E), (long)E * (K + 1)) * sizeof(float);
}

int warpctct_causal_conv_grad(const warpctct_conv_t *p, const warpctct_conv_grad_t *g, void *workspace,
                              size_t workspace_bytes, void *stream) {
    if (!conv_ok(p) || !g) return WARPCTCT_EINVAL;
    const bool columns = g->grad_weight || g->grad_bias;
    if (p->N > 0 && p->L > 0 && (!g->grad_out || !g->grad_x)) return WARPCTCT_EINVAL;
    const size_t need = warpctct_causal_conv_workspace_bytes(p->N, p->L, p->E, p->K);
    if (columns && need > 0 && !workspace) return WARPCTCT_EINVAL;
    if (columns && workspace_bytes < need) return WARPCTCT_EWORKSPACE;
    float *partial = columns ? static_cast<float *>(workspace) : nullptr;
    return done(launch_conv_grad(*p, *g, partial, as_stream(stream)));
}

int warpctct_causal_conv_step(const warpctct_conv_step_t *p, void *stream) {
    if (!p || !io_valid(p->dtype) || p->N < 0 || p->E < 1 || p->K < 1 || p->K > WARPCTCT_CONV_MAX_TAPS ||
        (long)p->N * p->E > kMostThreads)
        return WARPCTCT_EINVAL;
    if (p->N == 0) return WARPCTCT_OK;
    if (!p->x || !p->weight || !p->out || (p->K > 1 && !p->state)) return WARPCTCT_EINVAL;
    return done(launch_conv_step(*p, as_stream(stream)));
}

int warpctct_adjust_logits(const warpctct_adjust_t *p, void *stream) {
    if (!p || !io_valid(p->dtype) || p->N < 0 || p->N > kMostBatch || p->V < 1 || p->V > (1 << 30) || p->H < 0 ||
        p->H > (1 << 30) || (p->bias && !io_valid(p->bias_dtype)))
        return WARPCTCT_EINVAL;
    if (p->N == 0) return WARPCTCT_OK;
    if (!p->logits || !p->out) return WARPCTCT_EINVAL;
    return done(launch_adjust(*p, as_stream(stream)));
}

size_t warpctct_selective_scan_keep_bytes(int N, int L, int E, int S) {
    if (!scan_sizes_ok(WARPCTCT_F32, N, L, E, S, 1)) return 0;
    return scan_keep_floats(N, L, E, S) * sizeof(float);
}

size_t warpctct_selective_scan_workspace_bytes(int N, int L, int E, int S, int G, int backward) {
    if (!scan_sizes_ok(WARPCTCT_F32, N, L, E, S, G)) return 0;
    warpctct_scan_t p = {};
    p.N = N;
    p.L = L;
    p.E = E;
    p.S = S;
    p.G = G;
    return (backward ? scan_grad_floats(p) : scan_floats(p)) * sizeof(float);
}

int warpctct_selective_scan(const warpctct_scan_t *p, void *keep, size_t keep_bytes, void *workspace,
                            size_t workspace_bytes, void *stream) {
    if (!scan_ok(p)) return WARPCTCT_EINVAL;
    if (p->N == 0) return WARPCTCT_OK;
    if (p->L > 0 && !p->out) return WARPCTCT_EINVAL;
    if ((reinterpret_cast<uintptr_t>(keep) | reinterpret_cast<uintptr_t>(workspace)) & 15u) return WARPCTCT_EINVAL;
    const size_t need = scan_floats(*p) * sizeof(float);
    if (need > 0 && !workspace) return WARPCTCT_EINVAL;
    if ((keep && keep_bytes < scan_keep_floats(p->N, p->L, p->E, p->S) * sizeof(float)) || workspace_bytes < need)
        return WARPCTCT_EWORKSPACE;
    return done(launch_scan(*p, static_cast<float *>(keep), static_cast<float *>(workspace), as_stream(stream)));
}

int warpctct_selective_scan_grad(const warpctct_scan_t *p, const warpctct_scan_grad_t *g, const void *keep,
                                 size_t keep_bytes, void *workspace, size_t workspace_bytes, void *stream) {
    if (!scan_ok(p) || !g || !g->grad_a) return WARPCTCT_EINVAL;
    if (p->N > 0 && p->L > 0 &&
        (!g->grad_out || !g->grad_x || !g->grad_dt || !g->grad_b || !g->grad_c || (p->gate && !g->grad_gate) || !keep))
        return WARPCTCT_EINVAL;
    if ((reinterpret_cast<uintptr_t>(keep) | reinterpret_cast<uintptr_t>(workspace)) & 15u) return WARPCTCT_EINVAL;
    // (without steps too, the sequences' partial sums go through it)
    const size_t need = scan_grad_floats(*p) * sizeof(float);
    if (need > 0 && !workspace) return WARPCTCT_EINVAL;
    if (keep_bytes < scan_keep_floats(p->N, p->L, p->E, p->S) * sizeof(float) || workspace_bytes < need)
        return WARPCTCT_EWORKSPACE;
    return done(launch_scan_grad(*p, *g, static_cast<const float *>(keep), static_cast<float *>(workspace),
                                 as_stream(stream)));
}

int warpctct_selective_scan_step(const warpctct_scan_step_t *p, void *stream) {
    // (the batch is no grid dimension here)
    if (!p || p->N < 0 || !scan_sizes_ok(p->dtype, 0, 1, p->E, p->S, p->G) || (long)p->N * p->E >= (1L << 34))
        return WARPCTCT_EINVAL;
    if (p->N == 0) return WARPCTCT_OK;
    if (!p->x || !p->dt || !p->a || !p->b || !p->c || !p->state || !p->out) return WARPCTCT_EINVAL;
    return done(launch_scan_step(*p, as_stream(stream)));
}

}  // extern "C"
