"""Host-side argument checks of the C entry points beside the losses: wrong
arguments are refused before any launch, empty problems are no-ops.  Nothing
touches a device."""
import ctypes

import hip_lib

EINVAL, EWORKSPACE = 1, 3
F32, F16, BF16 = 0, 1, 2
P = ctypes.c_void_p
HOST = (ctypes.c_float * 64)()
SOME = ctypes.cast(HOST, P).value       # an address that is never followed


class Norm(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("weight_dtype", ctypes.c_int), ("width", ctypes.c_int),
                ("eps", ctypes.c_float), ("rows", ctypes.c_long), ("x_inner_rows", ctypes.c_long),
                ("x_outer_stride", ctypes.c_long), ("x_inner_stride", ctypes.c_long), ("x", P), ("weight", P),
                ("bias", P), ("out", P), ("stats", P)]


class NormGrad(ctypes.Structure):
    _fields_ = [("inner_rows", ctypes.c_long), ("outer_stride", ctypes.c_long), ("inner_stride", ctypes.c_long),
                ("grad_out", P), ("grad_x", P), ("grad_weight", P), ("grad_bias", P)]


def norm(**over):
    fields = dict(dtype=F32, weight_dtype=F32, width=8, eps=1e-5, rows=4, x_inner_rows=4, x_outer_stride=0,
                  x_inner_stride=8, x=SOME, weight=None, bias=None, out=SOME, stats=SOME)
    fields.update(over)
    return Norm(**fields)


def test_layer_norm_arguments():
    lib = hip_lib.lib()
    call = lambda **over: lib.warpctct_layer_norm(ctypes.byref(norm(**over)), P(0))  # noqa: E731
    assert lib.warpctct_layer_norm(P(0), P(0)) == EINVAL
    for bad in (dict(dtype=3), dict(weight_dtype=F16), dict(width=0), dict(rows=-1), dict(rows=2 ** 31),
                dict(x=None), dict(out=None), dict(x_inner_rows=0)):
        assert call(**bad) == EINVAL, bad
    assert call(rows=0, x=None, out=None) == 0


def test_layer_norm_gradient_arguments():
    lib = hip_lib.lib()
    size = lib.warpctct_layer_norm_workspace_bytes
    size.restype, size.argtypes = ctypes.c_size_t, [ctypes.c_long, ctypes.c_int]
    assert size(4, 8) == 64 and size(-1, 8) == 0 and size(4, 0) == 0
    assert size(1 << 20, 8) == 512 * 64      # a workgroup walks over rows: the scratch does not grow with them

    def call(p=None, workspace=SOME, have=1 << 20, **over):
        fields = dict(inner_rows=4, outer_stride=0, inner_stride=8, grad_out=SOME, grad_x=SOME, grad_weight=SOME,
                      grad_bias=SOME)
        fields.update(over)
        return lib.warpctct_layer_norm_grad(ctypes.byref(p or norm()), ctypes.byref(NormGrad(**fields)),
                                            P(workspace), ctypes.c_size_t(have), P(0))

    assert call(norm(stats=None)) == EINVAL
    assert call(grad_out=None) == EINVAL
    assert call(inner_rows=0) == EINVAL
    assert call(workspace=0) == EINVAL
    assert call(have=63) == EWORKSPACE
    assert call(grad_x=None, grad_weight=None, grad_bias=None) == 0
    assert call(norm(rows=0), grad_weight=None, grad_bias=None) == 0


class Conv(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int) for k in ("dtype", "N", "L", "E", "K", "silu")] + [
        ("x_n", ctypes.c_long), ("x_t", ctypes.c_long), ("x", P), ("weight", P), ("bias", P), ("lengths", P),
        ("initial", P), ("out", P), ("last", P)]


class ConvGrad(ctypes.Structure):
    _fields_ = [("grad_n", ctypes.c_long), ("grad_t", ctypes.c_long)] + [
        (k, P) for k in ("grad_out", "grad_last", "grad_x", "grad_initial", "grad_weight", "grad_bias")]


class ConvStep(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int) for k in ("dtype", "N", "E", "K", "silu")] + [("x_n", ctypes.c_long)] + [
        (k, P) for k in ("x", "state", "weight", "bias", "advance", "out")]


def conv(**over):
    fields = dict(dtype=BF16, N=2, L=5, E=4, K=4, silu=1, x_n=20, x_t=4, x=SOME, weight=SOME, out=SOME)
    fields.update(over)
    return Conv(**fields)


def test_causal_conv_arguments():
    lib = hip_lib.lib()
    call = lambda **over: lib.warpctct_causal_conv(ctypes.byref(conv(**over)), P(0))  # noqa: E731
    assert lib.warpctct_causal_conv(P(0), P(0)) == EINVAL
    for bad in (dict(dtype=-1), dict(N=-1), dict(N=65536), dict(L=-1), dict(E=0), dict(K=0), dict(K=9), dict(x=None),
                dict(weight=None), dict(out=None), dict(E=1 << 29), dict(L=1 << 30, E=1 << 20)):
        assert call(**bad) == EINVAL, bad
    assert call(N=0, x=None, weight=None, out=None) == 0


def test_causal_conv_gradient_and_step_arguments():
    lib = hip_lib.lib()
    size = lib.warpctct_causal_conv_workspace_bytes
    size.restype = ctypes.c_size_t
    assert size(2, 5, 4, 4) == 2 * 20 * 4 and size(2, 5, 4, 9) == 0 and size(-1, 5, 4, 4) == 0
    assert size(0, 5, 4, 4) == 0

    def call(p=None, workspace=SOME, have=1 << 20, **over):
        fields = dict(grad_n=20, grad_t=4, grad_out=SOME, grad_x=SOME, grad_weight=SOME, grad_bias=SOME)
        fields.update(over)
        return lib.warpctct_causal_conv_grad(ctypes.byref(p or conv()), ctypes.byref(ConvGrad(**fields)),
                                             P(workspace), ctypes.c_size_t(have), P(0))

    assert call(conv(K=9)) == EINVAL
    assert call(grad_out=None) == EINVAL and call(grad_x=None) == EINVAL
    assert call(workspace=0) == EINVAL and call(have=159) == EWORKSPACE
    assert call(conv(N=0), grad_weight=None, grad_bias=None) == 0

    def step(**over):
        fields = dict(dtype=F16, N=2, E=4, K=4, silu=0, x_n=4, x=SOME, state=SOME, weight=SOME, out=SOME)
        fields.update(over)
        return lib.warpctct_causal_conv_step(ctypes.byref(ConvStep(**fields)), P(0))

    assert lib.warpctct_causal_conv_step(P(0), P(0)) == EINVAL
    for bad in (dict(dtype=4), dict(N=-1), dict(E=0), dict(K=0), dict(K=9), dict(x=None), dict(state=None),
                dict(weight=None), dict(out=None)):
        assert step(**bad) == EINVAL, bad
    assert step(N=0, x=None, state=None) == 0


class Adjust(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int) for k in ("dtype", "N", "V", "H", "tokens_64", "bias_dtype", "allowed_packed")] + [
        (k, ctypes.c_float) for k in ("repetition", "presence", "frequency")] + [
        (k, ctypes.c_long) for k in ("logits_n", "tokens_n", "bias_n", "allowed_n")] + [
        (k, P) for k in ("logits", "tokens", "tokens_lengths", "repetitions", "presences", "frequencies", "bias",
                         "allowed", "out")]


def test_adjust_logits_arguments():
    lib = hip_lib.lib()

    def call(**over):
        fields = dict(dtype=F32, N=2, V=8, H=0, repetition=1.0, logits_n=8, logits=SOME, out=SOME)
        fields.update(over)
        return lib.warpctct_adjust_logits(ctypes.byref(Adjust(**fields)), P(0))

    assert lib.warpctct_adjust_logits(P(0), P(0)) == EINVAL
    for bad in (dict(dtype=3), dict(N=-1), dict(N=65536), dict(V=0), dict(V=(1 << 30) + 1), dict(H=-1),
                dict(bias=SOME, bias_dtype=3), dict(logits=None), dict(out=None)):
        assert call(**bad) == EINVAL, bad
    assert call(N=0, logits=None, out=None) == 0


SCAN_SIZES = ("dtype", "N", "L", "E", "S", "G", "softplus")
SCAN_STRIDES = ("x_n", "x_t", "dt_n", "dt_t", "gate_n", "gate_t", "b_n", "b_t", "b_g", "c_n", "c_t", "c_g")


class Scan(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int) for k in SCAN_SIZES] + [(k, ctypes.c_long) for k in SCAN_STRIDES] + [
        (k, P) for k in ("x", "dt", "gate", "b", "c", "a", "skip", "dt_bias", "lengths", "initial", "out", "last")]


class ScanGrad(ctypes.Structure):
    _fields_ = [("grad_n", ctypes.c_long), ("grad_t", ctypes.c_long)] + [
        (k, P) for k in ("grad_out", "grad_last", "grad_x", "grad_dt", "grad_gate", "grad_b", "grad_c", "grad_a",
                         "grad_skip", "grad_dt_bias", "grad_initial")]


class ScanStep(ctypes.Structure):
    _fields_ = [(k, ctypes.c_int) for k in ("dtype", "N", "E", "S", "G", "softplus")] + [
        (k, ctypes.c_long) for k in ("x_n", "dt_n", "gate_n", "b_n", "b_g", "c_n", "c_g")] + [
        (k, P) for k in ("x", "dt", "gate", "b", "c", "a", "skip", "dt_bias", "state", "advance", "out")]


ALIGNED = SOME + 15 & ~15


def scan(**over):
    fields = dict(dtype=F32, N=2, L=20, E=8, S=16, G=2, x=SOME, dt=SOME, b=SOME, c=SOME, a=SOME, out=SOME)
    fields.update(over)
    return Scan(**fields)


BAD_SCANS = (dict(dtype=3), dict(N=-1), dict(N=65536), dict(L=-1), dict(E=0), dict(E=9), dict(S=0), dict(S=65),
             dict(G=0), dict(x=None), dict(dt=None), dict(a=None), dict(b=None), dict(c=None), dict(E=(1 << 24) + 2))


def test_selective_scan_arguments():
    lib = hip_lib.lib()
    size = lib.warpctct_selective_scan_keep_bytes
    size.restype = ctypes.c_size_t
    assert size(2, 20, 8, 16) == 2 * 3 * 8 * 16 * 4 and size(2, 20, 8, 5) == 2 * 3 * 8 * 8 * 4
    assert size(2, 0, 8, 16) == 0 and size(2, 20, 8, 65) == 0

    def call(keep=0, have=0, workspace=0, scratch=0, **over):
        return lib.warpctct_selective_scan(ctypes.byref(scan(**over)), P(keep), ctypes.c_size_t(have), P(workspace),
                                           ctypes.c_size_t(scratch), P(0))

    none = ctypes.c_size_t(0)
    assert lib.warpctct_selective_scan(P(0), P(0), none, P(0), none, P(0)) == EINVAL
    for bad in BAD_SCANS + (dict(out=None),):
        assert call(**bad) == EINVAL, bad
    assert call(keep=ALIGNED, have=3071) == EWORKSPACE
    assert call(keep=ALIGNED + 4, have=1 << 20) == EINVAL
    # few long sequences take scratch: at least the states and the sum of every chunk but one
    size = lib.warpctct_selective_scan_workspace_bytes
    size.restype = ctypes.c_size_t
    need = size(1, 20000, 8, 16, 2, 0)
    assert need >= 2 * 8 * 17 * 4 and need % (8 * 17 * 4) == 0 and size(2, 20, 8, 16, 2, 0) == 0
    long = dict(N=1, L=20000)
    assert call(**long) == EINVAL and call(workspace=ALIGNED, scratch=need - 1, **long) == EWORKSPACE
    assert call(workspace=ALIGNED + 4, scratch=need, **long) == EINVAL
    assert call(N=0, x=None, dt=None, b=None, c=None, a=None, out=None) == 0


def test_selective_scan_gradient_and_step_arguments():
    lib = hip_lib.lib()
    size = lib.warpctct_selective_scan_workspace_bytes
    size.restype = ctypes.c_size_t
    need = size(2, 20, 8, 16, 2, 1)
    assert need == 4 * (2 * 2 * 24 * 32 + 2 * 8 * 18) and size(2, 20, 9, 16, 2, 1) == 0

    def call(p=None, keep=ALIGNED, kept=1 << 20, workspace=ALIGNED, have=1 << 20, **over):
        fields = dict(grad_out=SOME, grad_x=SOME, grad_dt=SOME, grad_b=SOME, grad_c=SOME, grad_a=SOME)
        fields.update(over)
        return lib.warpctct_selective_scan_grad(ctypes.byref(p or scan()), ctypes.byref(ScanGrad(**fields)), P(keep),
                                                ctypes.c_size_t(kept), P(workspace), ctypes.c_size_t(have), P(0))

    for bad in BAD_SCANS:
        assert call(scan(**bad)) == EINVAL, bad
    for bad in ("grad_out", "grad_x", "grad_dt", "grad_b", "grad_c", "grad_a"):
        assert call(**{bad: None}) == EINVAL, bad
    assert call(scan(gate=SOME)) == EINVAL
    assert call(keep=0) == EINVAL and call(workspace=0) == EINVAL and call(workspace=ALIGNED + 4) == EINVAL
    assert call(kept=3071) == EWORKSPACE and call(have=need - 1) == EWORKSPACE

    def step(**over):
        fields = dict(dtype=F16, N=2, E=8, S=16, G=1, x=SOME, dt=SOME, b=SOME, c=SOME, a=SOME, state=SOME, out=SOME)
        fields.update(over)
        return lib.warpctct_selective_scan_step(ctypes.byref(ScanStep(**fields)), P(0))

    assert lib.warpctct_selective_scan_step(P(0), P(0)) == EINVAL
    for bad in (dict(dtype=3), dict(N=-1), dict(E=0), dict(S=65), dict(G=3), dict(x=None), dict(dt=None), dict(a=None),
                dict(b=None), dict(c=None), dict(state=None), dict(out=None)):
        assert step(**bad) == EINVAL, bad
    assert step(N=0, x=None, state=None) == 0


def test_sizes_that_no_launch_holds():
    lib = hip_lib.lib()
    none = ctypes.c_size_t(0)
    assert lib.warpctct_layer_norm(ctypes.byref(norm(width=(1 << 27) - 31)), P(0)) == EINVAL
    for bad in (dict(L=(1 << 30) + 1, E=1), dict(L=1 << 20, E=1 << 12), dict(L=1, E=1 << 26, K=4)):
        assert lib.warpctct_causal_conv(ctypes.byref(conv(**bad)), P(0)) == EINVAL, bad
    p = ConvStep(dtype=F16, N=1 << 17, E=1 << 15, K=4, x=SOME, state=SOME, weight=SOME, out=SOME)
    assert lib.warpctct_causal_conv_step(ctypes.byref(p), P(0)) == EINVAL
    for bad in (dict(E=1 << 24, S=1, G=1), dict(E=1 << 23, S=64, G=1), dict(L=(1 << 30) + 1, E=1, S=1, G=1),
                dict(L=1 << 20, E=32, S=64, G=32)):
        assert lib.warpctct_selective_scan(ctypes.byref(scan(**bad)), P(0), none, P(0), none, P(0)) == EINVAL, bad


def test_the_scans_gradient_of_no_steps_takes_scratch_too():
    # the parameters' partial sums (zeros) go through it where there are sequences
    lib = hip_lib.lib()
    size = lib.warpctct_selective_scan_workspace_bytes
    size.restype = ctypes.c_size_t
    need = size(2, 0, 8, 16, 2, 1)
    assert need > 0 and size(0, 20, 8, 16, 2, 1) == 0
    grads = ScanGrad(grad_a=SOME)

    def call(workspace, have):
        return lib.warpctct_selective_scan_grad(ctypes.byref(scan(L=0)), ctypes.byref(grads), P(0), ctypes.c_size_t(0),
                                                P(workspace), ctypes.c_size_t(have), P(0))

    assert call(0, need) == EINVAL and call(0, 0) == EINVAL
    assert call(ALIGNED, need - 1) == EWORKSPACE


def test_histories_that_no_index_holds():
    # a workgroup walks over the history in steps of its 256 threads, counted in 32 bits
    lib = hip_lib.lib()
    for H in ((1 << 30) + 1, (1 << 31) - 1):
        p = Adjust(dtype=F32, N=2, V=8, H=H, repetition=1.0, logits_n=8, logits=SOME, out=SOME, tokens=SOME)
        assert lib.warpctct_adjust_logits(ctypes.byref(p), P(0)) == EINVAL, H
