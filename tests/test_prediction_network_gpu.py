"""The operators beside the losses as they are used together: a prediction
network (embedding, norm, projection, causal convolution, selective scan,
projection) that makes the label scores g of ctct_simple_loss, in training over
padded label rows, and in decoding one token at a time with rules on the logits.

Tolerance of the training run: every operator's result is off by at most ~200
units of 2^-24 of the magnitudes that go into it (the operators' own tests), a
matrix product over 64 elements by 64; ten of them in a row, forwards and
backwards, stay below 20 * 200 units = 2.4e-4 of a tensor's norm."""
import pytest
import torch

import warp_ctct
from oracle import ctct_oracle as O

pytestmark = pytest.mark.gpu
V, D, E, S, K, R = 48, 32, 64, 16, 4, 6


def parameters(seed=0):
    gen = torch.Generator().manual_seed(seed)
    draw = lambda *s, scale=1.0: torch.randn(*s, generator=gen) * scale  # noqa: E731
    p = {"embedding": draw(V, D), "norm_weight": 1 + draw(D, scale=0.1), "norm_bias": draw(D, scale=0.1),
         "into": draw(D, 2 * E, scale=D ** -0.5), "taps": draw(E, K, scale=K ** -0.5), "tap_bias": draw(E, scale=0.1),
         "select": draw(E, R + 2 * S, scale=E ** -0.5), "rate": draw(R, E, scale=R ** -0.5),
         "a_log": torch.log(torch.arange(1, S + 1.0)).repeat(E, 1), "skip": draw(E), "dt_bias": draw(E) - 3,
         "out": draw(E, V, scale=E ** -0.5), "end_weight": 1 + draw(V, scale=0.1), "end_bias": draw(V, scale=0.1)}
    return p


def network(p, tokens, lengths, norm, conv, scan):
    """Scores (N, L, V) for rows of tokens, by the three operators that are handed in."""
    h = norm(p["embedding"][tokens], p["norm_weight"], p["norm_bias"])
    both = h @ p["into"]
    x = conv(both[..., :E], p["taps"], p["tap_bias"], lengths)
    sel = x @ p["select"]
    y = scan(x, sel[..., :R] @ p["rate"], -torch.exp(p["a_log"]), sel[..., R:R + S], sel[..., R + S:], p["skip"],
             both[..., E:], p["dt_bias"], lengths)
    return norm(y @ p["out"], p["end_weight"], p["end_bias"])


def own(p, tokens, lengths, return_state=False):
    states = []

    def conv(x, weight, bias, lengths):
        out, state = warp_ctct.causal_conv(x, weight, bias, lengths, activation="silu", return_state=True)
        states.append(state)
        return out

    def scan(x, dt, a, b, c, skip, gate, dt_bias, lengths):
        out, state = warp_ctct.selective_scan(x, dt, a, b, c, skip=skip, gate=gate, dt_bias=dt_bias, softplus=True,
                                              lengths=lengths, return_state=True)
        states.append(state)
        return out

    g = network(p, tokens, lengths, warp_ctct.layer_norm, conv, scan)
    return (g, states) if return_state else g


def plain(p, tokens, lengths):
    """The same from the definitions, differentiable, in the type of the parameters."""
    live = (torch.arange(tokens.shape[1])[None] < lengths[:, None])[..., None]

    def norm(x, weight, bias):
        mid = x - x.mean(-1, keepdim=True)
        return mid / torch.sqrt((mid ** 2).mean(-1, keepdim=True) + 1e-5) * weight + bias

    def conv(x, weight, bias, _):
        wide = torch.cat([torch.zeros_like(x[:, :1]).expand(-1, K - 1, -1), x], 1)
        pre = sum(weight[:, k] * wide[:, k:k + x.shape[1]] for k in range(K)) + bias
        return pre * torch.sigmoid(pre) * live

    def scan(x, dt, a, b, c, skip, gate, dt_bias, _):
        d = torch.nn.functional.softplus(dt + dt_bias)
        h, ys = torch.zeros(x.shape[0], E, S, dtype=x.dtype), []
        for t in range(x.shape[1]):
            h = torch.exp(d[:, t, :, None] * a) * h + (d * x)[:, t, :, None] * b[:, t, None]
            ys.append((h * c[:, t, None]).sum(-1))
        return (torch.stack(ys, 1) + skip * x) * gate * torch.sigmoid(gate) * live

    return network(p, tokens, lengths, norm, conv, scan)


def close(got, want, name):
    want = want.double()
    assert float((got.detach().double().cpu() - want).norm()) <= 2.4e-4 * float(want.norm()), name


def test_training_on_padded_label_rows():
    N, T, U = 5, 40, 17
    gen = torch.Generator().manual_seed(3)
    labels = torch.randint(1, V, (N, U), generator=gen)
    ly = torch.tensor([17, 9, 1, 0, 13])
    lx = torch.tensor([40, 31, 40, 22, 25])
    f = torch.randn(N, T, V, generator=gen)
    tokens = torch.cat([torch.zeros(N, 1, dtype=torch.long), labels], 1)      # the start, then the labels
    cpu = {k: v.double().requires_grad_(True) for k, v in parameters().items()}
    gpu = {k: v.cuda().requires_grad_(True) for k, v in parameters().items()}
    g = own(gpu, tokens.cuda(), (ly + 1).cuda())
    want = plain(cpu, tokens, ly + 1)
    for n in range(N):
        close(g[n, :ly[n] + 1], want[n, :ly[n] + 1].detach(), "g")
    fg = f.cuda().requires_grad_(True)
    loss = warp_ctct.ctct_simple_loss(fg, g, labels.cuda(), lx.cuda(), ly.cuda(), reduction="sum")
    ref = O.ctct_simple_loss(f.double().numpy(), want.detach().numpy(), labels.int().numpy(), lx.int().numpy(),
                             ly.int().numpy(), reduction="sum", normalized=True)[0]
    assert abs(float(loss.detach()) - float(ref)) <= 2.4e-4 * abs(float(ref))
    names = list(gpu)
    grads = torch.autograd.grad(loss, [g] + [gpu[k] for k in names])
    wanted = torch.autograd.grad(want, [cpu[k] for k in names], grads[0].double().cpu())
    for name, got, ref in zip(names, grads[1:], wanted):
        assert got.shape == ref.shape
        close(got, ref, name)


def test_decoding_a_token_at_a_time_under_rules():
    N, T = 6, 25
    gen = torch.Generator().manual_seed(5)
    p = {k: v.cuda() for k, v in parameters(1).items()}
    f = torch.randn(N, T, V, generator=gen).cuda() * 2
    f[..., 0] += 1.5                                   # blank is taken now and then
    bias = torch.randn(V, generator=gen).cuda() * 0.3
    parity = torch.arange(V, device="cuda") % 2 == 0   # the grammar: even and odd labels take turns, blank always
    states = [torch.zeros(N, K - 1, E, device="cuda"), torch.zeros(N, E, S, device="cuda")]

    def step(token, advance):
        h = warp_ctct.layer_norm(p["embedding"][token], p["norm_weight"], p["norm_bias"])
        both = h @ p["into"]
        x = warp_ctct.causal_conv_step(both[:, :E], states[0], p["taps"], p["tap_bias"], "silu", advance)
        sel = x @ p["select"]
        y = warp_ctct.selective_scan_step(x, states[1], sel[:, :R] @ p["rate"], -torch.exp(p["a_log"]),
                                          sel[:, R:R + S], sel[:, R + S:], p["skip"], both[:, E:], p["dt_bias"], True,
                                          advance)
        return warp_ctct.layer_norm(y @ p["out"], p["end_weight"], p["end_bias"])

    history = torch.zeros(N, T + 1, dtype=torch.int32, device="cuda")     # the start, then what was taken
    count = torch.ones(N, dtype=torch.int32, device="cuda")
    g = step(history[:, 0].long(), torch.ones(N, dtype=torch.bool, device="cuda"))
    for t in range(T):
        last = history.gather(1, (count - 1).long()[:, None])
        allowed = torch.where((last % 2 == 0), ~parity, parity)
        allowed[:, 0] = True
        logits = warp_ctct.adjust_logits(f[:, t] + g, history[:, 1:], count - 1, repetition_penalty=1.3,
                                         frequency_penalty=0.2, bias=bias, allowed=allowed)
        token = logits.argmax(-1)
        assert bool(allowed.gather(1, token[:, None]).all())
        advance = token != 0
        g = torch.where(advance[:, None], step(token, advance), g)
        at = torch.where(advance, count, T).long()[:, None]
        history.scatter_(1, at, torch.where(advance, token, 0).int()[:, None])
        count += advance.int()
    assert int(count.max()) > 5 and int(count.min()) < T      # labels were taken, and blanks
    # the same labels as a padded batch: scores behind the last label, and the states
    with torch.no_grad():
        scores, whole = own(p, history[:, :T].long(), count, return_state=True)
    rows = scores[torch.arange(N, device="cuda"), (count - 1).long()]
    close(g, rows.cpu(), "g")
    close(states[0], whole[0].cpu(), "convolution state")
    close(states[1], whole[1].cpu(), "scan state")
