"""causal_conv, its backward pass and its single step against the definitions in
float64.

Tolerances, in units of 2^-24: a sum of K products and the bias is off by at
most (K + 2) units of the sum of the magnitudes; silu has a slope of at most 1.1
and its own value and slope are formed with an error of at most ~20 units (exp2
of an argument rounded to a unit, a reciprocal, three products), the slope
changing by at most half of what its argument does.  The parameters' gradients
are sums over at most 64 steps of a tile and then over the tiles, 16 strands of
which are added up one after the other.  A result rounded to a type is off by
half a step of it."""
import pytest
import torch

import warp_ctct

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT = 2.0 ** -24


def f64(t):
    return None if t is None else t.detach().double().cpu()


def oracle(x, weight, bias, lengths, initial, silu, g=None, glast=None):
    """Results and the tolerances they are given before they are rounded."""
    x, weight, bias, initial, g, glast = (f64(t) for t in (x, weight, bias, initial, g, glast))
    (N, T, E), K = x.shape, weight.shape[1]
    lengths = [T] * N if lengths is None else [min(max(int(l), 0), T) for l in lengths.cpu()]
    if initial is None:
        initial = torch.zeros(N, K - 1, E, dtype=torch.float64)
    bias = torch.zeros(E, dtype=torch.float64) if bias is None else bias
    val, tol = {}, {}
    for name, shape in (("out", (N, T, E)), ("state", (N, K - 1, E)), ("gx", (N, T, E)), ("gw", (E, K)), ("gb", (E,)),
                        ("ginitial", (N, K - 1, E))):
        val[name], tol[name] = torch.zeros(shape, dtype=torch.float64), torch.zeros(shape, dtype=torch.float64)
    for n in range(N):
        l = lengths[n]
        ext = torch.cat([initial[n], x[n, :l]])
        win = torch.stack([ext[k:k + l] for k in range(K)], -1)               # (l, E, K)
        pre = (win * weight).sum(-1) + bias
        pre_off = (K + 2) * UNIT * ((win * weight).abs().sum(-1) + bias.abs())
        s = torch.sigmoid(pre)
        val["out"][n, :l] = pre * s if silu else pre
        tol["out"][n, :l] = (1.1 * pre_off + (20 + 3 * pre.abs()) * UNIT * (pre * s).abs()) if silu else pre_off
        val["state"][n] = ext[l:]
        if g is None:
            continue
        slope = s * (1 + pre * (1 - s)) if silu else torch.ones_like(pre)
        gp = g[n, :l] * slope
        gp_off = g[n, :l].abs() * (0.5 * pre_off + 20 * UNIT * (1 + pre.abs()) * s if silu else 0 * pre)
        gext, gext_off = torch.zeros_like(ext), torch.zeros_like(ext)
        for k in range(K):
            gext[k:k + l] += weight[:, k] * gp
            gext_off[k:k + l] += weight[:, k].abs() * (gp_off + (K + 2) * UNIT * gp.abs())
        if glast is not None:
            gext[l:] += glast[n]
            gext_off[l:] += UNIT * (glast[n].abs() + gext[l:].abs())
        val["gx"][n, :l], tol["gx"][n, :l] = gext[K - 1:], gext_off[K - 1:]
        val["ginitial"][n], tol["ginitial"][n] = gext[:K - 1], gext_off[:K - 1]
        val["gw"] += (gp[..., None] * win).sum(0)
        val["gb"] += gp.sum(0)
        tol["gw"] += ((gp_off + 200 * UNIT * gp.abs())[..., None] * win.abs()).sum(0)
        tol["gb"] += (gp_off + 200 * UNIT * gp.abs()).sum(0)
    return val, tol


def check(got, val, tol, name):
    want, dtype = val[name], got.dtype
    assert got.shape == want.shape, name
    far = (f64(got) - want).abs() - tol[name] - torch.finfo(dtype).eps / 2 * want.abs() - 2.0 ** -25
    if dtype == torch.float32:
        far += 2.0 ** -25       # the last term is float16's smallest step only
    assert torch.isfinite(got).all() and (got.numel() == 0 or float(far.max()) <= 0), (name, float(far.max()))


def leaf(t):
    return t.detach().requires_grad_(True)


def make(N, T, E, K, dtype, seed=0, initial=True, params=torch.float32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x = leaf(draw(N, T, E).to(dtype))
    weight, bias = leaf((draw(E, K) * K ** -0.5).to(params)), leaf((0.3 * draw(E)).to(params))
    first = leaf(draw(N, K - 1, E).to(dtype)) if initial else None
    return x, weight, bias, first, draw(N, T, E).to(dtype), draw(N, K - 1, E).to(dtype)


def run(x, weight, bias, first, g, glast, lengths=None, activation="silu"):
    out, state = warp_ctct.causal_conv(x, weight, bias, lengths, first, activation, return_state=True)
    leaves = [t for t in (x, weight, bias, first) if t is not None]
    ends, ups = ([out, state], [g, glast]) if glast is not None and glast.numel() else ([out], [g])
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(ends, leaves, ups, allow_unused=True)))
    named = {"gx": grads[id(x)], "gw": grads[id(weight)]}
    if bias is not None:
        named["gb"] = grads[id(bias)]
    if first is not None and first.numel():
        named["ginitial"] = grads[id(first)]
    return dict(named, out=out.detach(), state=state.detach())


def compare(x, weight, bias, first, g, glast, lengths=None, activation="silu"):
    val, tol = oracle(x, weight, bias, lengths, first, activation == "silu", g, glast)
    for name, got in run(x, weight, bias, first, g, glast, lengths, activation).items():
        check(got, val, tol, name)
    assert torch.equal(warp_ctct.causal_conv(x, weight, bias, lengths, first, activation).detach(),
                       run(x, weight, bias, first, g, glast, lengths, activation)["out"])


SHAPES = [(1, 1, 1, 4), (2, 1, 8, 4), (2, 2, 5, 4), (3, 3, 16, 3), (2, 33, 7, 4), (3, 65, 24, 2), (2, 130, 40, 4),
          (1, 200, 260, 8), (4, 17, 12, 5), (2, 40, 64, 1), (2, 9, 33, 6), (1, 500, 4, 7), (130, 70, 8, 4)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,T,E,K", SHAPES)
def test_against_the_definition(N, T, E, K, dtype):
    lengths = torch.tensor([(T * (i + 1)) // N for i in range(N)], device="cuda")
    compare(*make(N, T, E, K, dtype, seed=T), lengths=lengths)
    compare(*make(N, T, E, K, dtype, seed=T + 1, initial=False), activation=None)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_of_nothing_and_out_of_range(dtype):
    args = make(6, 20, 16, 4, dtype)
    compare(*args, lengths=torch.tensor([0, 1, 2, 20, 25, -3], device="cuda", dtype=torch.int64))
    x, weight, bias, first, g, glast = make(2, 20, 16, 4, dtype)
    # what lies behind a sequence is not read
    lengths = torch.tensor([5, 0], device="cuda", dtype=torch.int32)
    with torch.no_grad():
        x[0, 5:], x[1], g[0, 5:], g[1] = float("nan"), float("inf"), float("nan"), float("nan")
    got = run(x, weight, bias, first, g, glast, lengths)
    val, tol = oracle(x[:, :5], weight, bias, lengths, first, True, g[:, :5], glast)
    for name in got:
        cut = got[name][:, :5] if name in ("out", "gx") else got[name]
        check(cut, val, tol, name)
    assert not got["out"][:, 5:].any() and not got["gx"][:, 5:].any()


@gpu
def test_no_steps_and_no_sequences():
    x, weight, bias, first, g, glast = make(2, 0, 8, 4, torch.float32)
    got = run(x, weight, bias, first, g, glast)
    assert got["out"].shape == (2, 0, 8) and torch.equal(got["state"], first) and torch.equal(got["ginitial"], glast)
    assert not got["gw"].any() and not got["gb"].any()
    x, weight, bias, first, g, glast = make(0, 5, 8, 4, torch.float32)
    got = run(x, weight, bias, first, g, None)
    assert got["out"].shape == (0, 5, 8) and not got["gw"].any()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_inputs_and_gradients(dtype):
    wide = torch.randn(3, 21, 100, device="cuda").to(dtype)
    _, weight, bias, first, g, glast = make(3, 21, 32, 4, dtype)
    for view in (wide[..., 8:40], wide[..., 3:35], wide[..., ::3][..., :32],
                 wide.transpose(0, 1).contiguous().transpose(0, 1)[..., :32], wide[:1, :, :32].expand(3, 21, 32)):
        compare(leaf(view), weight, bias, first, g, glast)
        compare(leaf(view), weight, None, first, torch.randn(3, 21, 48, device="cuda").to(dtype)[..., 5:37], glast)
    compare(leaf(wide[..., 8:40]), weight, bias, first, torch.ones(1, device="cuda", dtype=dtype).expand(3, 21, 32),
            glast)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_parameters_in_the_inputs_type_and_the_state_alone(dtype):
    x, weight, bias, first, g, glast = make(2, 30, 16, 4, dtype, params=dtype)
    compare(x, weight, bias, first, g, glast)
    out, state = warp_ctct.causal_conv(x, weight, bias, None, first, None, return_state=True)
    gx, gfirst = torch.autograd.grad(state, [x, first], glast)
    assert torch.equal(gx[:, -3:], glast) and not gx[:, :-3].any() and not gfirst.any()


@gpu
def test_gradients_of_some_of_the_inputs_and_twice():
    args = make(3, 40, 24, 4, torch.float16)
    want = run(*args)
    for keep, name in enumerate(("gx", "gw", "gb", "ginitial")):
        some = [leaf(t) if i == keep else t.detach() for i, t in enumerate(args[:4])]
        out, state = warp_ctct.causal_conv(some[0], some[1], some[2], None, some[3], "silu", return_state=True)
        for again in (True, False):     # the state does not depend on the parameters
            ends, ups = ([out, state], args[4:]) if state.requires_grad else ([out], args[4:5])
            got, = torch.autograd.grad(ends, some[keep], ups, retain_graph=again)
            assert torch.equal(got, want[name])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,K", [(24, 4), (7, 3), (16, 1), (8, 8)])
def test_steps_and_pieces_are_the_whole(E, K, dtype):
    x, weight, bias, first, _, _ = make(5, 23, E, K, dtype)
    lengths = torch.tensor([23, 11, 0, 1, 19], device="cuda", dtype=torch.int32)
    with torch.no_grad():
        whole, last = warp_ctct.causal_conv(x, weight, bias, lengths, first, "silu", return_state=True)
        head, mid = warp_ctct.causal_conv(x[:, :9], weight, bias, lengths.clamp(max=9), first, "silu", True)
        tail, end = warp_ctct.causal_conv(x[:, 9:], weight, bias, (lengths - 9).clamp(min=0), mid, "silu", True)
        assert torch.equal(torch.cat([head, tail], 1), whole) and torch.equal(end, last)
        state = first.detach().clone()
        for t in range(23):
            out = warp_ctct.causal_conv_step(x[:, t], state, weight, bias, "silu", advance=lengths > t)
            assert torch.equal(out, whole[:, t]), t
        assert torch.equal(state, last)
        val, tol = oracle(x[:, :1], weight, bias, None, first, False)
        state = first.detach().clone()
        check(warp_ctct.causal_conv_step(x[:, 0], state, weight, bias)[:, None], val, tol, "out")
        check(state, val, tol, "state")


@gpu
def test_the_same_call_gives_the_same_bits():
    args = make(300, 200, 24, 4, torch.bfloat16)
    first, again = run(*args), run(*args)
    assert all(torch.equal(first[k], again[k]) for k in first)


@gpu
def test_on_a_stream_of_its_own_and_in_a_graph():
    x, weight, bias, first, g, glast = make(4, 90, 32, 4, torch.float16)
    lengths = torch.tensor([90, 45, 3, 77], device="cuda", dtype=torch.int32)
    want = run(x, weight, bias, first, g, glast, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, weight, bias, first, g, glast, lengths)
    side.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want)
    state, token = first.detach().clone(), x[:, 0].detach().clone()
    with torch.no_grad():
        warp_ctct.causal_conv_step(token, state, weight, bias, "silu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = run(x, weight, bias, first, g, glast, lengths)
        with torch.no_grad():
            step = warp_ctct.causal_conv_step(token, state, weight, bias, "silu")
    for seed in range(3):
        fresh = make(4, 90, 32, 4, torch.float16, seed=seed + 3)
        with torch.no_grad():
            for to, of in zip((x, weight, bias, first, g, glast), fresh):
                to.copy_(of)
            lengths.copy_(torch.tensor([1 + 20 * seed, 90, 0, 50], dtype=torch.int32))
            twin = state.clone()
            token.copy_(x[:, 1])
        graph.replay()
        torch.cuda.synchronize()
        want = run(x, weight, bias, first, g, glast, lengths)
        assert all(torch.equal(kept[k], want[k]) for k in want)
        with torch.no_grad():
            assert torch.equal(step, warp_ctct.causal_conv_step(token, twin, weight, bias, "silu"))
        assert torch.equal(state, twin)


@gpu
def test_gradient_against_differences():
    args = make(2, 12, 6, 4, torch.float32)
    g, glast = args[4], args[5]
    got = run(*args)
    for k, name in ((0, "gx"), (1, "gw"), (2, "gb"), (3, "ginitial")):
        way = torch.randn_like(args[k])
        value = []
        for step in (1e-2, -1e-2):
            moved = [t.detach() + (step * way if i == k else 0) for i, t in enumerate(args[:4])]
            out, state = warp_ctct.causal_conv(moved[0], moved[1], moved[2], None, moved[3], "silu", True)
            value.append(float((f64(out) * f64(g)).sum() + (f64(state) * f64(glast)).sum()))
        want = float((f64(got[name]) * f64(way)).sum())
        assert abs((value[0] - value[1]) / 2e-2 - want) < 0.02 * (1 + abs(want)), name


@gpu
def test_refusals_on_the_gpu():
    x, weight, bias, first, g, glast = make(2, 10, 8, 4, torch.float32)
    ones = lambda *s, **k: torch.ones(*s, device="cuda", **k)  # noqa: E731
    for bad in (dict(x=ones(2, 8)), dict(weight=ones(7, 4)), dict(weight=ones(8, 9)), dict(weight=ones(8, 0)),
                dict(bias=ones(7)), dict(lengths=ones(3, dtype=torch.int32)), dict(lengths=ones(2)),
                dict(initial_state=ones(2, 4, 8)), dict(initial_state=ones(2, 3, 8, dtype=torch.float16)),
                dict(activation="relu"), dict(weight=torch.ones(8, 4)), dict(lengths=torch.ones(2, dtype=torch.int32))):
        with pytest.raises(RuntimeError):
            warp_ctct.causal_conv(**{**dict(x=x, weight=weight), **bad})
    state = ones(2, 3, 8)
    with torch.no_grad():
        for bad in (dict(x=ones(2, 1, 8)), dict(state=ones(2, 4, 8)), dict(state=ones(2, 3, 8, dtype=torch.float16)),
                    dict(state=ones(2, 8, 3).transpose(1, 2)), dict(advance=ones(2)), dict(weight=ones(8, 3)),
                    dict(advance=ones(3, dtype=torch.bool)), dict(state=torch.ones(2, 3, 8))):
            with pytest.raises(RuntimeError):
                warp_ctct.causal_conv_step(**{**dict(x=ones(2, 8), state=state, weight=weight), **bad})
    with pytest.raises(RuntimeError, match="no_grad"):
        warp_ctct.causal_conv_step(ones(2, 8), state, weight)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(warp_ctct.causal_conv(x, weight), [x], g, create_graph=True)


@gpu
def test_a_step_counts_up_the_version_of_its_state():
    x, weight, bias, first, _, _ = make(2, 10, 8, 4, torch.float32)
    state = torch.ones(2, 3, 8, device="cuda")
    out = warp_ctct.causal_conv(x, weight, bias, initial_state=state)
    with torch.no_grad():
        warp_ctct.causal_conv_step(x[:, 0], state, weight, bias)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()      # the graph had saved the state
    with torch.no_grad(), pytest.raises(RuntimeError, match="complex"):
        warp_ctct.causal_conv_step(x[:, 0], state, weight.to(torch.complex64), bias)


def test_refusals_without_a_gpu():
    with pytest.raises(RuntimeError, match="GPU"):
        warp_ctct.causal_conv(torch.zeros(1, 2, 3), torch.zeros(3, 4))
    with pytest.raises(RuntimeError, match="GPU"):
        warp_ctct.causal_conv_step(torch.zeros(1, 3), torch.zeros(1, 3, 3), torch.zeros(3, 4))
    with pytest.raises(RuntimeError, match="activation"):
        warp_ctct.causal_conv(torch.zeros(1, 2, 3), torch.zeros(3, 4), activation="gelu")
