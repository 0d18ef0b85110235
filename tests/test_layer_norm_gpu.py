"""layer_norm and its backward pass against the definitions in float64.

Tolerances.  With h the normalised value, every h the kernel forms is off by at
most ~64 units of 2^-24 (1 + |h|): the deviations from the first mean are exact
to half a unit each, the mean of them and of their squares is a sum of at most
54 additions in sequence (32 in a lane, 6 across a wavefront, 16 across a
workgroup), and the root and the two products add four roundings.  A result
rounded to a type is off by half a step of it, eps/2 |value|."""
import pytest
import torch

import warp_ctct

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def oracle(x, weight, bias, g, eps):
    """out, gx, gweight, gbias in float64, and how far each may be off but for
    the rounding of the result."""
    D = x.shape[-1]
    x, g = x.detach().double().reshape(-1, D).cpu(), g.detach().double().reshape(-1, D).cpu()
    w = weight.detach().double().cpu() if weight is not None else torch.ones(D, dtype=torch.float64)
    b = bias.detach().double().cpu() if bias is not None else torch.zeros(D, dtype=torch.float64)
    m = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + eps)
    h = (x - m) * r
    out = h * w + b
    u = g * w
    gx = r * (u - u.mean(1, keepdim=True) - h * (u * h).mean(1, keepdim=True))
    off = 64 * UNIT * (1 + h.abs())
    tol_out = off * w.abs() + 2 * UNIT * (out.abs() + b.abs())
    mean_off = (u.abs() * (off + 64 * UNIT * h.abs())).mean(1, keepdim=True)
    tol_gx = r * (64 * UNIT * (u.abs() + u.abs().mean(1, keepdim=True)) + h.abs() * mean_off
                  + off * (u * h).mean(1, keepdim=True).abs() + 4 * UNIT * (h * (u * h).mean(1, keepdim=True)).abs())
    deep = 128 + x.shape[0] / 512
    tol_gw = (g.abs() * (off + deep * UNIT * h.abs())).sum(0)
    tol_gb = deep * UNIT * g.abs().sum(0)
    return (out, gx, (g * h).sum(0), g.sum(0)), (tol_out, tol_gx, tol_gw, tol_gb)


def check(got, want, tol, dtype, name):
    got = got.detach().double().cpu().reshape(want.shape)
    far = (got - want).abs() - tol - half_step(dtype) * want.abs() - torch.finfo(dtype).tiny * 2 ** -9
    assert torch.isfinite(got).all() and float(far.max() if far.numel() else 0) <= 0, (name, float(far.max()))


def run(x, weight, bias, g, eps=1e-5):
    leaves = [t for t in (x, weight, bias) if t is not None]
    out = warp_ctct.layer_norm(x, weight, bias, eps)
    grads = dict(zip([id(t) for t in leaves], torch.autograd.grad(out, leaves, g)))
    # (detached: a backward pass cannot be captured while an eager graph of the same leaves lives)
    return out.detach(), [grads.get(id(t)) if t is not None else None for t in (x, weight, bias)]


def compare(x, weight, bias, g, eps=1e-5):
    want, tol = oracle(x, weight, bias, g, eps)
    out, grads = run(x, weight, bias, g, eps)
    assert out.dtype == x.dtype and out.shape == x.shape
    check(out, want[0], tol[0], x.dtype, "out")
    for got, of, k, name in zip(grads, (x, weight, bias), (1, 2, 3), ("gx", "gweight", "gbias")):
        if of is not None:
            assert got.dtype == of.dtype and got.shape == of.shape
            check(got, want[k], tol[k], of.dtype, name)
    with torch.no_grad():
        assert torch.equal(warp_ctct.layer_norm(x, weight, bias, eps), out)


def leaf(t):
    return t.detach().requires_grad_(True)


def make(shape, dtype, params, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x, g = leaf((draw(*shape) * 1.5 + 0.5).to(dtype)), draw(*shape).to(dtype)
    pt = {"none": None, "f32": torch.float32, "same": dtype}[params]
    weight = leaf((1 + 0.3 * draw(shape[-1])).to(pt)) if pt else None
    bias = leaf((0.3 * draw(shape[-1])).to(pt)) if pt else None
    return x, weight, bias, g


SHAPES = [(1, 1), (3, 2), (4, 7), (5, 64), (2, 3, 129), (9, 512), (3, 641), (2, 2048), (3, 2049), (2, 4097),
          (2, 5000), (3, 8192), (2, 8200), (2, 16384), (2, 16385), (1, 20000), (700, 40), (5000, 256)]


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_definition(shape, dtype):
    for params in ("none", "f32", "same"):
        compare(*make(shape, dtype, params, seed=shape[-1]))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_one_parameter_without_the_other_and_mixed_types(dtype):
    x, weight, bias, g = make((6, 96), dtype, "f32")
    compare(x, weight, None, g)
    compare(x, None, bias, g)
    mixed = leaf(bias.detach().to(dtype))       # weight float32, bias of the input's type: both read as float32
    compare(x, weight, mixed, g)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_inputs_and_gradients(dtype):
    wide = torch.randn(5, 9, 200, device="cuda").to(dtype)
    weight, bias = leaf(torch.randn(64, device="cuda")), leaf(torch.randn(64, device="cuda"))
    views = [wide[..., :64].transpose(0, 1), wide[:, ::2, 3:67], wide[:, 1, 8:72], wide[..., ::3][..., :64],
             wide[:1].expand(4, 9, 200)[..., 64:128], wide.reshape(5, 3, 3, 200)[:, :, 1:, :64].transpose(0, 2)]
    for view in views:
        x = leaf(view)
        compare(x, weight, bias, torch.randn(*x.shape, device="cuda").to(dtype))
        g = torch.randn(*x.shape[:-1], 80, device="cuda").to(dtype)[..., 7:71]
        compare(x, weight, bias, g)
        compare(x, weight, bias, torch.ones(1, device="cuda", dtype=dtype).expand(x.shape))


@gpu
def test_rows_far_from_zero_and_constant_rows():
    x = torch.randn(8, 700, device="cuda") + 1e4
    x[3] = 5.0
    x[4] = 0.0
    compare(leaf(x), leaf(torch.ones(700, device="cuda")), leaf(torch.zeros(700, device="cuda")),
            torch.randn(8, 700, device="cuda"))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_a_row_that_is_not_finite_stays_alone(dtype):
    x, weight, bias, g = make((6, 130), dtype, "f32")
    with torch.no_grad():
        x[2, 5], x[4, 7] = float("nan"), float("inf")
    out, (gx, _, _) = run(x, weight, bias, g)
    keep = [0, 1, 3, 5]
    want, tol = oracle(x[keep], weight, bias, g[keep], 1e-5)
    check(out[keep], want[0], tol[0], dtype, "out")
    check(gx[keep], want[1], tol[1], dtype, "gx")
    assert torch.isnan(out[2]).all() and torch.isnan(out[4]).any()


@gpu
def test_no_rows():
    weight, bias = leaf(torch.ones(16, device="cuda")), leaf(torch.ones(16, device="cuda"))
    x = leaf(torch.empty(0, 3, 16, device="cuda"))
    out, (gx, gw, gb) = run(x, weight, bias, torch.empty(0, 3, 16, device="cuda"))
    assert out.shape == gx.shape == (0, 3, 16)
    assert torch.equal(gw, torch.zeros_like(gw)) and torch.equal(gb, torch.zeros_like(gb))


@gpu
def test_the_same_call_gives_the_same_bits():
    args = make((3000, 257), torch.bfloat16, "same")
    first, again = run(*args), run(*args)
    assert torch.equal(first[0], again[0])
    assert all(torch.equal(a, b) for a, b in zip(first[1], again[1]))


@gpu
def test_other_types_are_converted():
    x = torch.randn(4, 10, device="cuda", dtype=torch.float64)
    out = warp_ctct.layer_norm(x)
    assert out.dtype == torch.float32 and torch.equal(out, warp_ctct.layer_norm(x.float()))


@gpu
def test_on_a_stream_of_its_own_and_in_a_graph():
    x, weight, bias, g = make((40, 384), torch.float16, "f32")
    want = run(x, weight, bias, g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, weight, bias, g)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = run(x, weight, bias, g)
    for seed in range(3):
        fresh = make((40, 384), torch.float16, "f32", seed=seed + 5)
        with torch.no_grad():
            for to, of in zip((x, weight, bias, g), fresh):
                to.copy_(of)
        graph.replay()
        torch.cuda.synchronize()
        want = run(x, weight, bias, g)
        assert torch.equal(kept[0], want[0]) and all(torch.equal(a, b) for a, b in zip(kept[1], want[1]))


@gpu
def test_gradient_against_differences():
    x, weight, bias, g = make((3, 24), torch.float32, "f32")
    _, grads = run(x, weight, bias, g)
    for of, grad in zip((x, weight, bias), grads):
        way = torch.randn_like(of)
        step = 1e-2
        up, down = [warp_ctct.layer_norm(*[t.detach() + s * way if t is of else t.detach() for t in (x, weight, bias)])
                    for s in (step, -step)]
        slope = float(((up.double() - down.double()) * g.double()).sum() / (2 * step))
        want = float((grad.double() * way.double()).sum())
        # third derivatives times step^2, and the rounding of the outputs over 2 step
        assert abs(slope - want) < 0.05 * (1 + abs(want)), (slope, want)


@gpu
@pytest.mark.parametrize("shape", [(50, 96), (3, 20000)])
def test_gradients_of_some_of_the_inputs_and_twice(shape):
    args = make(shape, torch.bfloat16, "f32")
    _, want = run(*args)
    for keep in range(3):
        some = [leaf(t) if i == keep else t.detach() for i, t in enumerate(args[:3])]
        out = warp_ctct.layer_norm(*some)
        first = torch.autograd.grad(out, some[keep], args[3], retain_graph=True)[0]
        assert torch.equal(first, want[keep])
        assert torch.equal(first, torch.autograd.grad(out, some[keep], args[3])[0])


@gpu
def test_refusals_on_the_gpu():
    x, weight, bias, g = make((4, 12), torch.float32, "f32")
    for bad in (dict(weight=torch.ones(11, device="cuda")), dict(bias=torch.ones(12, 1, device="cuda")),
                dict(weight=torch.ones(12)), dict(eps=-1.0), dict(x=torch.ones(4, 12, device="cuda", dtype=torch.cfloat))):
        with pytest.raises(RuntimeError):
            warp_ctct.layer_norm(**{**dict(x=x), **bad})
    with pytest.raises(RuntimeError):
        warp_ctct.layer_norm(torch.zeros(4, 0, device="cuda"))
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(warp_ctct.layer_norm(x, weight, bias), [x], g, create_graph=True)


def test_refusals_without_a_gpu():
    with pytest.raises(RuntimeError, match="GPU"):
        warp_ctct.layer_norm(torch.zeros(3, 4))
    with pytest.raises(TypeError):
        warp_ctct.layer_norm([1.0, 2.0])
