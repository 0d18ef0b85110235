"""selective_scan, its backward pass and its single step against the recurrence
in float64.

Tolerances follow the recurrence: next to every quantity the oracle carries a
bound of its error in the kernel's fp32 arithmetic (UNIT = 2^-24), from the
roundings that each formula makes and the bounds of what goes into it.  So a
state's bound decays and grows with the state itself, and a gradient's with the
reverse recurrence.  Sums over time are taken one after the other (T units of
the sum of magnitudes), sums over channels in a tree within a workgroup and
then one after the other over the workgroups.  The exponential that the factors and
the sigmoids are formed from gives zero (or infinity, whose reciprocal is zero)
where the result lies below TINY = 2^-126: such a factor is off by TINY, silu by
|gate| TINY, its slope by (1 + |gate|) TINY, in absolute terms.  Products of two errors are left
out and covered by the factor 1.1 at the end."""
import ctypes
import math

import pytest
import torch

import hip_lib
import warp_ctct

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT, TINY = 2.0 ** -24, 2.0 ** -126


def f64(t):
    return None if t is None else t.detach().double().cpu()


class Case:
    """Inputs of a call, by the names of its arguments, and the upstream gradients."""

    def __init__(self, N, T, E, S, G=1, dtype=torch.float32, gate=True, skip=True, dt_bias=True, softplus=True,
                 initial=True, lengths=None, seed=0, grouped=True, decay=1.0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        draw = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
        self.args = {
            "x": draw(N, T, E).to(dtype),
            "dt": (draw(N, T, E) - 2.0 if softplus else 0.1 * draw(N, T, E).abs()).to(dtype),
            "a": -decay * (torch.rand(E, S, device="cuda", generator=gen) * S + 0.1),
            "b": (draw(N, T, G, S) if grouped else draw(N, T, S)).to(dtype),
            "c": (draw(N, T, G, S) if grouped else draw(N, T, S)).to(dtype),
            "skip": draw(E) if skip else None, "gate": draw(N, T, E).to(dtype) if gate else None,
            "dt_bias": 0.3 * draw(E).abs() if dt_bias else None,
            "initial_state": draw(N, E, S) if initial else None}
        self.softplus = softplus
        self.lengths = None if lengths is None else torch.tensor(lengths, device="cuda")
        self.g, self.glast = draw(N, T, E).to(dtype), draw(N, E, S)
        self.track()

    def track(self):
        self.args = {k: None if v is None else v.detach().requires_grad_(True) for k, v in self.args.items()}

    def call(self, **over):
        return warp_ctct.selective_scan(**{**self.args, **over}, softplus=self.softplus, lengths=self.lengths,
                                        return_state=True)

    def run(self):
        out, state = self.call()
        names = [k for k, v in self.args.items() if v is not None]
        ends, ups = ([out, state], [self.g, self.glast]) if self.glast is not None else ([out], [self.g])
        grads = torch.autograd.grad(ends, [self.args[k] for k in names], ups)
        return dict({"grad_" + k: v for k, v in zip(names, grads)}, out=out.detach(), state=state.detach())


def oracle(case):
    """Values and bounds by name; outputs behind a sequence are zero with bound zero."""
    p = {k: f64(v) for k, v in case.args.items()}
    x, a = p["x"], p["a"]
    (N, T, E), S = x.shape, a.shape[1]
    b, c = (t if t.dim() == 4 else t.unsqueeze(2) for t in (p["b"], p["c"]))
    G = b.shape[2]
    b, c = (t.repeat_interleave(E // G, 2) for t in (b, c))
    lengths = [T] * N if case.lengths is None else [min(max(int(l), 0), T) for l in case.lengths]
    live = (torch.arange(T)[None] < torch.tensor(lengths)[:, None])[..., None]
    zero = torch.zeros((), dtype=torch.float64)
    clean = lambda t: torch.where(live if t.dim() == 3 else live[..., None], t, zero)  # noqa: E731
    x, b, c = clean(x), clean(b), clean(c)
    raw = clean(p["dt"]) + (p["dt_bias"] if p["dt_bias"] is not None else 0)
    d = clean(torch.nn.functional.softplus(raw, threshold=1e6) if case.softplus else raw)
    slope = clean(torch.sigmoid(raw) if case.softplus else torch.ones_like(raw))
    dd = clean(2 * UNIT * raw.abs() * slope + 16 * UNIT * d.abs())
    z = clean(p["gate"]) if p["gate"] is not None else None
    sg = torch.sigmoid(z) if z is not None else None
    silu = z * sg if z is not None else torch.ones_like(x)
    dsilu = sg * (1 + z * (1 - sg)) if z is not None else torch.zeros_like(x)
    zu = UNIT * (12 + 3 * z.abs()) if z is not None else torch.zeros_like(x)
    skip = p["skip"] if p["skip"] is not None else torch.zeros(E, dtype=torch.float64)
    k = torch.exp(d[..., None] * a)
    kk = k * (a.abs() * dd[..., None] + 4 * UNIT * (d[..., None] * a).abs() + 4 * UNIT)
    kk = (kk + TINY) * live[..., None]
    u = (d * x)[..., None] * b
    h0 = p["initial_state"] if p["initial_state"] is not None else torch.zeros(N, E, S, dtype=torch.float64)
    hs, hhs, h, hh = [h0], [torch.zeros_like(h0)], h0, torch.zeros_like(h0)
    for t in range(T):
        on = live[:, t][..., None]
        new = k[:, t] * h + u[:, t]
        newer = (k[:, t] * hh + kk[:, t] * h.abs() + (x[:, t].abs() * dd[:, t])[..., None] * b[:, t].abs()
                 + 3 * UNIT * u[:, t].abs() + UNIT * new.abs())
        h, hh = torch.where(on, new, h), torch.where(on, newer, hh)
        hs.append(h)
        hhs.append(hh)
    H, HH = torch.stack(hs[1:], 1), torch.stack(hhs[1:], 1)
    P, PP = torch.stack(hs[:-1], 1), torch.stack(hhs[:-1], 1)
    y = (c * H).sum(-1) + skip * x
    yy = (c.abs() * HH).sum(-1) + (S + 2) * UNIT * (c * H).abs().sum(-1) + 2 * UNIT * (skip * x).abs()
    val = {"out": y * silu, "state": h}
    za = TINY * z.abs() if z is not None else torch.zeros_like(x)
    tol = {"out": yy * silu.abs() + (y * silu).abs() * (zu + 2 * UNIT) + y.abs() * za, "state": hh}
    g, glast = clean(f64(case.g)), f64(case.glast)
    gy = g * silu
    gg = gy.abs() * (zu + UNIT) + g.abs() * za
    gh, ee = [None] * T, [None] * T
    carry, off = (glast if glast is not None else torch.zeros_like(h0)), torch.zeros_like(h0)
    for t in reversed(range(T)):
        on = live[:, t][..., None]
        new = c[:, t] * gy[:, t][..., None] + carry
        newer = c[:, t].abs() * gg[:, t][..., None] + off + 2 * UNIT * (c[:, t] * gy[:, t][..., None]).abs() + UNIT * new.abs()
        gh[t], ee[t] = torch.where(on, new, 0 * new), torch.where(on, newer, 0 * newer)
        off = torch.where(on, k[:, t] * newer + kk[:, t] * new.abs() + UNIT * (k[:, t] * new).abs(), off)
        carry = torch.where(on, k[:, t] * new, carry)
    val["grad_initial_state"], tol["grad_initial_state"] = carry, off
    if T == 0:
        gh, ee = torch.zeros(N, 0, E, S, dtype=torch.float64), torch.zeros(N, 0, E, S, dtype=torch.float64)
    else:
        gh, ee = torch.stack(gh, 1), torch.stack(ee, 1)
    ghb = (gh * b).sum(-1)
    ghb_off = (ee * b.abs()).sum(-1) + (S + 4) * UNIT * (gh * b).abs().sum(-1)
    r = gh * k * P
    rr = ee * k * P.abs() + gh.abs() * kk * P.abs() + gh.abs() * k * PP + 3 * UNIT * r.abs()
    ar, ar_off = (a * r).sum(-1), (a.abs() * (rr + (S + 4) * UNIT * r.abs())).sum(-1)
    val["grad_x"] = skip * gy + d * ghb
    tol["grad_x"] = skip.abs() * gg + dd * ghb.abs() + d.abs() * ghb_off + 3 * UNIT * ((skip * gy).abs() + (d * ghb).abs())
    gd = x * ghb + ar
    gd_off = x.abs() * ghb_off + ar_off + 2 * UNIT * ((x * ghb).abs() + ar.abs())
    val["grad_dt"] = gd * slope
    tol["grad_dt"] = gd_off * slope + UNIT * (12 + 2 * raw.abs()) * (gd * slope).abs()
    if z is not None:
        val["grad_gate"] = g * y * dsilu
        tol["grad_gate"] = g.abs() * (yy * dsilu.abs() + y.abs() * UNIT * (20 * (1 + z.abs()) * sg + 3 * dsilu.abs()))
        tol["grad_gate"] = tol["grad_gate"] + (g * y).abs() * (TINY + za)
    wide = lambda t: t.unflatten(2, (G, E // G)).sum(3)  # noqa: E731
    deep = 24 + E / 16
    dx = (d * x)[..., None]
    dx_off = (x.abs() * dd)[..., None] + 2 * UNIT * dx.abs()
    val["grad_b"] = wide(gh * dx)
    tol["grad_b"] = wide(ee * dx.abs() + gh.abs() * dx_off + deep * UNIT * (gh * dx).abs())
    val["grad_c"] = wide(gy[..., None] * H * live[..., None])
    tol["grad_c"] = wide((gy.abs()[..., None] * HH + gg[..., None] * H.abs() + deep * UNIT * (gy[..., None] * H).abs()) * live[..., None])
    long = T + N + 40
    val["grad_a"] = (d[..., None] * r).sum((0, 1))
    tol["grad_a"] = (dd[..., None] * r.abs() + d.abs()[..., None] * (rr + long * UNIT * r.abs())).sum((0, 1))
    val["grad_skip"] = (gy * x).sum((0, 1))
    tol["grad_skip"] = (gg * x.abs() + long * UNIT * (gy * x).abs()).sum((0, 1))
    val["grad_dt_bias"] = val["grad_dt"].sum((0, 1))
    tol["grad_dt_bias"] = (tol["grad_dt"] + long * UNIT * val["grad_dt"].abs()).sum((0, 1))
    for name in ("b", "c"):
        if case.args[name].dim() == 3:
            val["grad_" + name], tol["grad_" + name] = val["grad_" + name][:, :, 0], tol["grad_" + name][:, :, 0]
    return val, tol


def check(got, val, tol, name):
    want, dtype = val[name], got.dtype
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), name
    far = (f64(got) - want).abs() - 1.1 * tol[name] - torch.finfo(dtype).eps / 2 * want.abs()
    far = far - (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)      # half of the smallest step; denormals
    assert got.numel() == 0 or float(far.max()) <= 0, (name, float(far.max()))


def compare(case):
    val, tol = oracle(case)
    got = case.run()
    for name in got:
        check(got[name], val, tol, name)
    with torch.no_grad():
        out, state = case.call()
        assert torch.equal(out, got["out"]) and torch.equal(state, got["state"])
    return got


SHAPES = [(1, 1, 1, 1, 1), (2, 1, 8, 16, 1), (2, 15, 6, 3, 2), (1, 16, 64, 16, 1), (3, 17, 65, 16, 1), (2, 33, 10, 5, 2),
          (2, 40, 260, 4, 1), (2, 50, 130, 8, 1), (1, 100, 96, 16, 3), (2, 37, 40, 20, 1), (2, 20, 34, 32, 2),
          (1, 35, 20, 33, 1), (2, 48, 24, 64, 1), (1, 300, 16, 12, 1), (70, 18, 4, 2, 1), (140, 70, 6, 16, 1),
          (1, 1100, 10, 16, 1)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,T,E,S,G", SHAPES)
def test_against_the_recurrence(N, T, E, S, G, dtype):
    compare(Case(N, T, E, S, G, dtype, seed=T, lengths=[(T * (i + 1)) // N for i in range(N)]))
    compare(Case(N, T, E, S, G, dtype, seed=T + 1, gate=False, softplus=False, initial=False))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_arguments_left_out(dtype):
    for over in (dict(skip=False), dict(dt_bias=False), dict(gate=False, skip=False, dt_bias=False),
                 dict(grouped=False), dict(softplus=False, dt_bias=False)):
        compare(Case(2, 35, 24, 16, 1, dtype, **over))
    case = Case(2, 35, 24, 16, 1, dtype)
    case.glast = None
    compare(case)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_of_nothing_and_out_of_range(dtype):
    got = compare(Case(7, 40, 12, 16, 1, dtype, lengths=[0, 1, 16, 17, 40, 99, -2]))
    assert not got["out"][0].any() and not got["grad_b"][0].any() and not got["out"][1, 1:].any()
    case = Case(2, 40, 12, 16, 1, dtype, lengths=[18, 0])
    bad = {"x": float("nan"), "dt": float("inf"), "b": float("nan"), "c": float("inf"), "gate": float("nan")}
    with torch.no_grad():       # what lies behind a sequence is not read
        for name, value in bad.items():
            case.args[name][0, 18:], case.args[name][1] = value, value
        case.g[0, 18:], case.g[1] = float("nan"), float("inf")
    compare(case)


@gpu
def test_no_steps_and_no_sequences():
    got = Case(2, 0, 8, 16).run()
    case = Case(2, 0, 8, 16)
    got = case.run()
    assert got["out"].shape == (2, 0, 8) and torch.equal(got["state"], case.args["initial_state"])
    assert torch.equal(got["grad_initial_state"], case.glast) and not got["grad_a"].any() and not got["grad_skip"].any()
    case = Case(0, 5, 8, 16)
    case.glast = None
    got = case.run()
    assert got["out"].shape == (0, 5, 8) and not got["grad_a"].any() and not got["grad_dt_bias"].any()


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_inputs_and_gradients(dtype):
    N, T, E, S = 3, 29, 32, 16
    wide = torch.randn(N, T, 160, device="cuda").to(dtype)
    both = torch.randn(N, T, 2 * S + 6, device="cuda").to(dtype)
    views = [wide[..., 8:40], wide[..., 3:35], wide[..., ::3][..., :32],
             wide.transpose(0, 1).contiguous().transpose(0, 1)[..., :32], wide[:1, :, 64:96].expand(N, T, E)]
    for i, view in enumerate(views):
        case = Case(N, T, E, S, 1, dtype, seed=i, grouped=False)
        case.args.update(x=view, gate=views[(i + 1) % 5], dt=(views[(i + 2) % 5].abs() * 0.5 - 2).to(dtype),
                         b=both[..., 6:6 + S], c=both[..., 6 + S:])
        case.track()
        case.g = views[(i + 3) % 5]
        compare(case)
    case = Case(N, T, E, S, 2, dtype)
    case.args["b"] = torch.randn(N, T, S, 2, device="cuda").to(dtype).transpose(2, 3)     # not dense: copied
    case.args["c"] = torch.randn(N, T, 2, S + 3, device="cuda").to(dtype)[..., 1:1 + S]
    case.track()
    case.g = torch.ones(1, device="cuda", dtype=dtype).expand(N, T, E)
    compare(case)


@gpu
def test_gradients_of_some_of_the_inputs_and_twice():
    case = Case(3, 40, 24, 16, 2, torch.bfloat16)
    want = case.run()
    for name in list(case.args):
        some = {k: v.detach().requires_grad_(k == name) for k, v in case.args.items()}
        out, state = warp_ctct.selective_scan(**some, softplus=True, return_state=True)
        for again in (True, False):
            got, = torch.autograd.grad([out, state], some[name], [case.g, case.glast], retain_graph=again)
            assert torch.equal(got, want["grad_" + name]), name


@gpu
def test_the_state_alone_and_parameters_of_another_type():
    case = Case(2, 40, 24, 16, dtype=torch.float16)
    for name in ("a", "skip", "dt_bias"):
        case.args[name] = case.args[name].to(torch.bfloat16)
    case.track()
    val, tol = oracle(case)
    got = case.run()
    assert got["grad_a"].dtype == torch.bfloat16
    for name in got:
        check(got[name], val, tol, name)
    case.g = torch.zeros_like(case.g)
    val, tol = oracle(case)
    _, state = case.call()
    names = ("x", "dt", "a", "b", "dt_bias", "initial_state")
    for name, g in zip(names, torch.autograd.grad(state, [case.args[k] for k in names], case.glast)):
        check(g, val, tol, "grad_" + name)


@gpu
def test_extreme_steps():
    case = Case(2, 40, 16, 16, softplus=True)
    with torch.no_grad():
        case.args["dt"][0, ::5] = -200.0      # d = 0: the state stays
        case.args["dt"][0, 1::5] = 60.0       # d = 60: the state is forgotten
        case.args["gate"][1, ::3] = -90.0
        case.args["gate"][1, 1::3] = 90.0
        case.args["a"][3] = 0.0
    compare(case)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,S,G", [(24, 16, 1), (10, 5, 2), (40, 64, 1), (6, 1, 3), (16, 4, 1), (8, 32, 1)])
def test_steps_and_pieces_are_the_whole(E, S, G, dtype):
    N, T, cut = 5, 37, 21
    lengths = [37, 20, 0, 1, 30]
    case = Case(N, T, E, S, G, dtype, lengths=lengths)
    val, tol = oracle(case)
    names = ("x", "dt", "b", "c", "gate")
    fixed = {k: v for k, v in case.args.items() if k not in names + ("initial_state",)}
    with torch.no_grad():
        head, mid = warp_ctct.selective_scan(**fixed, **{k: case.args[k][:, :cut] for k in names}, softplus=True,
                                             lengths=case.lengths.clamp(max=cut), return_state=True,
                                             initial_state=case.args["initial_state"])
        tail, last = warp_ctct.selective_scan(**fixed, **{k: case.args[k][:, cut:] for k in names}, softplus=True,
                                              lengths=(case.lengths - cut).clamp(min=0), return_state=True,
                                              initial_state=mid)
        check(torch.cat([head, tail], 1), val, tol, "out")
        check(last, val, tol, "state")
        state, outs = case.args["initial_state"].detach().clone(), []
        for t in range(T):
            before = state.clone()
            outs.append(warp_ctct.selective_scan_step(state=state, **fixed, **{k: case.args[k][:, t] for k in names},
                                                      softplus=True, advance=case.lengths > t))
            still = (case.lengths <= t).nonzero().flatten()
            assert torch.equal(state[still], before[still]) and not outs[-1][still].any()
        check(torch.stack(outs, 1), val, tol, "out")
        check(state, val, tol, "state")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_step_without_its_optional_arguments_and_from_views(dtype):
    N, E, S = 9, 30, 16
    case = Case(N, 1, E, S, 1, dtype, gate=False, skip=False, dt_bias=False, softplus=False, grouped=False)
    val, tol = oracle(case)
    wide = torch.zeros(N, 2 * E + 1, device="cuda", dtype=dtype)
    wide[:, 1:1 + E] = case.args["x"][:, 0]
    with torch.no_grad():
        state = case.args["initial_state"].detach().clone()
        out = warp_ctct.selective_scan_step(wide[:, 1:1 + E], state, case.args["dt"][:, 0], case.args["a"],
                                            case.args["b"][:, 0], case.args["c"][:, 0])
        check(out[:, None], val, tol, "out")
        check(state, val, tol, "state")


@gpu
def test_the_same_call_gives_the_same_bits():
    case = Case(20, 90, 130, 16, dtype=torch.bfloat16)
    first, again = case.run(), case.run()
    assert all(torch.equal(first[k], again[k]) for k in first)


@gpu
def test_on_a_stream_of_its_own_and_in_a_graph():
    make = lambda seed: Case(3, 70, 24, 16, 1, torch.float16, lengths=[70, 33, 5], seed=seed)  # noqa: E731
    case = make(0)
    case.lengths = case.lengths.int()
    want = case.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = case.run()
    side.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want)
    state = case.args["initial_state"].detach().clone()
    token = {k: case.args[k][:, 0].detach().clone() for k in ("x", "dt", "b", "c", "gate")}
    fixed = {k: case.args[k].detach() for k in ("a", "skip", "dt_bias")}
    step = lambda s: warp_ctct.selective_scan_step(state=s, **token, **fixed, softplus=True)  # noqa: E731
    step(state)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = case.run()
        out = step(state)
    for seed in range(3):
        fresh = make(seed + 1)
        with torch.no_grad():
            for k, v in fresh.args.items():
                case.args[k].copy_(v)
            case.g.copy_(fresh.g)
            case.glast.copy_(fresh.glast)
            case.lengths.copy_(torch.tensor([1 + 9 * seed, 70, 0], dtype=torch.int32))
            for k in token:
                token[k].copy_(fresh.args[k][:, 1])
            twin = state.clone()
        graph.replay()
        torch.cuda.synchronize()
        want = case.run()
        assert all(torch.equal(kept[k], want[k]) for k in want)
        assert torch.equal(out, step(twin)) and torch.equal(state, twin)


@gpu
def test_gradient_against_differences():
    case = Case(2, 20, 6, 8, 2)
    got = case.run()
    for name, of in case.args.items():
        way = torch.randn_like(of) * (0.1 if name == "a" else 1.0)
        value = []
        for step in (4e-3, -4e-3):
            with torch.no_grad():
                out, state = case.call(**{name: of + step * way})
            value.append(float((f64(out) * f64(case.g)).sum() + (f64(state) * f64(case.glast)).sum()))
        want = float((f64(got["grad_" + name]) * f64(way)).sum())
        assert abs((value[0] - value[1]) / 8e-3 - want) < 0.02 * (1 + abs(want)), name


@gpu
def test_rates_at_the_ends_of_the_range():
    low = torch.finfo(torch.float32).min
    for lengths in ([40, 18, 3], [40 * 8, 18 * 8, 0]):       # whole, and cut into chunks
        case = Case(3, lengths[0], 16, 16, lengths=lengths)
        with torch.no_grad():
            case.args["a"][3], case.args["a"][4, 2], case.args["a"][5, 3:] = low, -3e38, -2.5e38
        compare(case)
        with torch.no_grad():
            kept = case.call()
            case.args["a"][3] = -math.inf
            got = case.call()
            assert torch.equal(got[0], kept[0]) and torch.equal(got[1], kept[1])
            case.args["a"][7, 5] = math.nan
            out = case.call()[0]
            assert out[:2, 0, 7].isnan().all() and torch.equal(out[..., :7], kept[0][..., :7])
            case.args["a"][7, 5] = -1.0
            case.args["a"][3] = low
            case.args["dt"][:, ::5] = -200.0      # d = 0: the state stays, whatever its rate
            val, tol = oracle(case)
            out, state = case.call()
            check(out, val, tol, "out")
            check(state, val, tol, "state")
    case = Case(3, 1, 16, 16)
    with torch.no_grad():
        case.args["a"][3], case.args["dt"][1:] = low, -200.0
        val, tol = oracle(case)
        state = case.args["initial_state"].detach().clone()
        steps = ("x", "dt", "b", "c", "gate")
        fixed = {k: v for k, v in case.args.items() if k not in steps + ("initial_state",)}
        out = warp_ctct.selective_scan_step(state=state, **fixed, **{k: case.args[k][:, 0] for k in steps}, softplus=True)
        check(out[:, None], val, tol, "out")
        check(state, val, tol, "state")


def growing():
    """400 steps of one sequence, cut into chunks of 48, with exponents above zero and nothing to grow.  What a chunk
    does to a state goes by the sum of its d, formed one after the other: off by up to 24 units of the sum, where the
    oracle allows every step 20 units of its d a and 4 more.  Twice the oracle's bound covers both; with d = 0.01
    the 4 units a step do."""
    case = Case(1, 400, 8, 16, gate=False, softplus=False, initial=False, dt_bias=False)
    case.glast = None
    with torch.no_grad():
        case.args["a"].fill_(1.0)
        case.args["x"].zero_()
        case.args["dt"].fill_(0.01)
    return case


@gpu
@pytest.mark.parametrize("first", [None, 1e-36])
def test_growth_of_nothing_and_of_little_over_a_chunk(first):
    case = growing()
    with torch.no_grad():
        case.args["dt"][:, :200 if first is None else 35] = 4.0      # 2^277 over a chunk, 2^202
        if first is None:
            case.args["x"][:, 200:] = 1.0
        else:
            case.args["initial_state"] = torch.full((1, 8, 16), first, device="cuda")
        val, tol = oracle(case)
        out, state = case.call()
    for name, got in (("out", out), ("state", state)):
        check(got, val, {name: 2 * tol[name]}, name)


@gpu
def test_growth_of_gradients_of_zero_over_a_chunk():
    case = growing()
    with torch.no_grad():
        case.args["dt"][:, 200:] = 4.0
    case.g[:, 200:] = 0
    compare(case)


@gpu
def test_refusals_on_the_gpu():
    case = Case(2, 10, 8, 16)
    ones = lambda *s, **k: torch.ones(*s, device="cuda", **k)  # noqa: E731
    for bad in (dict(x=ones(2, 8)), dict(dt=ones(2, 10, 7)), dict(dt=ones(2, 10, 8, dtype=torch.float16)),
                dict(a=ones(8, 65)), dict(a=ones(7, 16)), dict(a=ones(8, 0)), dict(b=ones(2, 10, 3, 16)),
                dict(b=ones(2, 10, 1, 15)), dict(c=ones(2, 9, 1, 16)), dict(c=ones(2, 10, 2, 16)), dict(skip=ones(7)),
                dict(gate=ones(2, 10, 9)), dict(dt_bias=ones(8, 1)), dict(initial_state=ones(2, 8, 15)),
                dict(initial_state=ones(2, 8, 16, dtype=torch.float16)), dict(a=torch.ones(8, 16)),
                dict(b=ones(2, 10, 1, 16, dtype=torch.bfloat16))):
        with pytest.raises(RuntimeError):
            case.call(**bad)
    for lengths in (ones(3, dtype=torch.int32), ones(2), torch.ones(2, dtype=torch.int32)):
        with pytest.raises(RuntimeError):
            warp_ctct.selective_scan(**case.args, lengths=lengths)
    with torch.no_grad():
        good = dict(x=ones(2, 8), state=ones(2, 8, 16), dt=ones(2, 8), a=-ones(8, 16), b=ones(2, 16), c=ones(2, 16))
        warp_ctct.selective_scan_step(**good)
        for bad in (dict(x=ones(2, 1, 8)), dict(state=ones(2, 8, 15)), dict(state=ones(2, 8, 16, dtype=torch.float16)),
                    dict(state=ones(2, 16, 8).transpose(1, 2)), dict(b=ones(2, 3, 16)), dict(c=ones(3, 16)),
                    dict(advance=ones(2)), dict(state=torch.ones(2, 8, 16)), dict(gate=ones(2, 7))):
            with pytest.raises(RuntimeError):
                warp_ctct.selective_scan_step(**{**good, **bad})
    with pytest.raises(RuntimeError, match="no_grad"):
        warp_ctct.selective_scan_step(**dict(good, x=ones(2, 8, requires_grad=True)))
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(case.call()[0], [case.args["x"]], case.g, create_graph=True)


@gpu
def test_a_step_counts_up_the_version_of_its_state():
    x, b = torch.rand(2, 10, 8, device="cuda"), torch.rand(2, 10, 16, device="cuda")
    a, state = -torch.rand(8, 16, device="cuda"), torch.ones(2, 8, 16, device="cuda")
    out = warp_ctct.selective_scan(x.requires_grad_(True), x, a, b, b, initial_state=state)
    with torch.no_grad():
        warp_ctct.selective_scan_step(x[:, 0], state, x[:, 0], a, b[:, 0], b[:, 0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()      # the graph had saved the state


def test_refusals_without_a_gpu():
    t = torch.zeros
    with pytest.raises(RuntimeError, match="GPU"):
        warp_ctct.selective_scan(t(1, 2, 3), t(1, 2, 3), t(3, 4), t(1, 2, 4), t(1, 2, 4))
    with pytest.raises(RuntimeError, match="GPU"):
        warp_ctct.selective_scan_step(t(1, 3), t(1, 3, 4), t(1, 3), t(3, 4), t(1, 4), t(1, 4))


# Few long sequences are cut into chunks, in both directions.  Two groups, odd and
# even batches, rows in wide pieces and not, 1 to 16 lanes a channel; more channels
# in a group than a workgroup takes; sequences that end inside an earlier chunk, at
# the end of one and one step behind it, and that have one step or none.
CUT = [(6, 250, 10, 3, 2), (6, 240, 64, 3, 2), (3, 400, 600, 4, 2), (6, 250, 24, 8, 2), (5, 260, 40, 16, 2),
       (6, 230, 64, 16, 1), (6, 230, 20, 24, 2), (3, 200, 12, 64, 2), (5, 140, 40, 64, 2)]


def chunk_steps(N, T, E, S, G):
    """Steps of a chunk, forwards and backwards, from the scratch that the two passes take."""
    size = hip_lib.lib().warpctct_selective_scan_workspace_bytes
    size.restype = ctypes.c_size_t
    lanes = next(n for n in (1, 2, 4, 8, 16) if 4 * n >= S)
    tile, blocks = {1: 4, 16: 16}.get(lanes, 8), -(-(E // G) // (256 // lanes))
    states, sums = E * (4 * lanes + 1), E * (S + 2)      # of a sequence and chunk
    forward, rest = divmod(size(N, T, E, S, G, 0) // 4, N * states)
    backward, left = divmod(size(N, T, E, S, G, 1) // 4 - N * G * blocks * -(-T // tile) * tile * 8 * lanes, N * (states + sums))
    assert rest == left == 0 and forward > 1 and backward > 1      # (else it is not cut)
    return [16 * -(-(-(-T // 16)) // n) for n in (forward, backward)]


@pytest.mark.parametrize("shape", CUT)
def test_the_shapes_below_are_cut(shape):
    assert all(32 <= steps <= shape[1] - 16 for steps in chunk_steps(*shape))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", CUT)
def test_few_long_sequences(shape, dtype):
    # A chunk's factor goes by the sum of its d, formed one after the other: off by up to steps/2 units of the sum,
    # where the oracle allows every step 20 units of its d a.
    loose = 1 + max(chunk_steps(*shape)) / 40
    N, T, E, S, G = shape
    lengths = [T, T // 3, 0, 64, 65, 1][:N]
    for start, end in ((True, False), (False, True)):
        case = Case(*shape, dtype, seed=T, lengths=lengths, initial=start, gate=end)
        if not end:
            case.glast = None
        with torch.no_grad():       # what lies behind a sequence is not read
            for n, length in enumerate(lengths):
                for rows in [case.args[k] for k in ("x", "dt", "b", "c")] + [case.g] + [case.args["gate"]] * end:
                    rows[n, length:] = math.nan
        val, tol = oracle(case)
        got, again = case.run(), case.run()
        for name in got:
            check(got[name], val, {name: loose * tol[name]}, name)
            assert torch.equal(got[name], again[name])
        with torch.no_grad():
            out, state = case.call()
        assert torch.equal(out, got["out"]) and torch.equal(state, got["state"])
