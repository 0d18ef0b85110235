"""Offsets beyond 32 bits: tensors of more than 2^31 elements through every
operator.  What the end of such a tensor gives must be what the end alone gives,
taken from the state in front of it (bit for bit, but for the scan, whose long
run is cut into chunks: half a step of bfloat16 more)."""
import pytest
import torch

import warp_ctct

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def big(*shape):
    return torch.empty(*shape, device="cuda", dtype=BF16).normal_(generator=torch.Generator("cuda").manual_seed(1))


def leaf(t):
    return t.detach().requires_grad_(True)


def test_layer_norm():
    rows, width = 2 ** 21 + 5, 1024
    x, g = leaf(big(rows, width)), big(rows, width)
    weight = torch.randn(width, device="cuda")
    out = warp_ctct.layer_norm(x, weight)
    gx, = torch.autograd.grad(out, x, g)
    for part in (slice(0, 3), slice(rows - 7, rows)):
        few = leaf(x[part])
        small = warp_ctct.layer_norm(few, weight)
        assert torch.equal(out[part], small)
        assert torch.equal(gx[part], torch.autograd.grad(small, few, g[part])[0])


def test_causal_conv():
    L, E, end = 2 ** 20 + 9, 2048, 6
    x, g = leaf(big(1, L, E)), big(1, L, E)
    weight = torch.randn(E, 4, device="cuda")
    out, state = warp_ctct.causal_conv(x, weight, activation="silu", return_state=True)
    gx, = torch.autograd.grad(out, x, g)
    few, first = leaf(x[:, L - end:]), x[:, L - end - 3:L - end].detach()
    small, last = warp_ctct.causal_conv(few, weight, initial_state=first, activation="silu", return_state=True)
    assert torch.equal(out[:, L - end:], small) and torch.equal(state, last)
    assert torch.equal(gx[:, L - end:], torch.autograd.grad(small, few, g[:, L - end:])[0])


def test_selective_scan():
    L, E, S, end = 2 ** 20 + 9, 2048, 4, 7
    x, g = leaf(big(1, L, E)), big(1, L, E)
    b, c = big(1, L, S), big(1, L, S)
    a = -torch.rand(E, S, device="cuda")
    call = lambda x, b, c, h, **k: warp_ctct.selective_scan(x, x.detach(), a, b, c, gate=x.detach(), softplus=True,  # noqa: E731
                                                            initial_state=h, **k)
    out, state = call(x, b, c, None, return_state=True)
    gx, = torch.autograd.grad(out, x, g)
    cut = slice(L - end, L)
    with torch.no_grad():
        _, mid = call(x[:, :L - end], b[:, :L - end], c[:, :L - end], None, return_state=True)
    few = leaf(x[:, cut])
    small, last = call(few, b[:, cut], c[:, cut], mid, return_state=True)
    gfew, = torch.autograd.grad(small, few, g[:, cut])
    for got, want in ((out[:, cut], small), (gx[:, cut], gfew), (state, last)):
        got, want = got.detach().float(), want.detach().float()
        # two float32 computations of the same value, each rounded once: a step of the type apart at most
        assert bool(((got - want).abs() <= 2 ** -8 * (got.abs() + want.abs()) / 2 * 1.01 + 1e-4).all())
    del gx, g, out
    state = mid.clone()
    with torch.no_grad():
        step = warp_ctct.selective_scan_step(x[:, L - end], state, x[:, L - end], a, b[:, L - end], c[:, L - end],
                                             gate=x[:, L - end], softplus=True)
    assert bool(((step - small[:, 0].detach()).float().abs() <= 2 ** -8 * step.float().abs() * 1.01 + 1e-4).all())


def test_adjust_logits():
    N, V = 33000, 65536
    logits = big(N, V)
    tokens = torch.randint(0, V, (N, 5), device="cuda")
    bias = torch.randn(V, device="cuda")
    out = warp_ctct.adjust_logits(logits, tokens, repetition_penalty=1.5, presence_penalty=0.5, bias=bias)
    part = slice(N - 4, N)
    assert torch.equal(out[part], warp_ctct.adjust_logits(logits[part], tokens[part], repetition_penalty=1.5,
                                                          presence_penalty=0.5, bias=bias))


def test_layer_norm_of_more_wide_rows_than_workgroups():
    rows, width, many = 5, 8193, 2 ** 20 + 5      # rows in no multiple of a vector, a workgroup each
    x, g = big(rows, width).half(), big(rows, width).half()
    x[1:], g[1:] = x[0], g[0]
    few, weight = leaf(x), leaf(torch.randn(width, device="cuda"))
    small = warp_ctct.layer_norm(few, weight)
    gsmall, = torch.autograd.grad(small, few, g)
    row = leaf(x[:1])
    out = warp_ctct.layer_norm(row.expand(many, width), weight)
    assert bool((out[:5] == small).all()) and bool((out[many - 5:] == small).all())
    wide = leaf(x[:1].expand(many, width))
    gx, = torch.autograd.grad(warp_ctct.layer_norm(wide, weight), wide, g[:1].expand(many, width))
    assert bool((gx[:5] == gsmall).all()) and bool((gx[many - 5:] == gsmall).all())
