"""adjust_logits against the rules written out in float64.

Tolerance: five roundings to float32 (the quotient or product, the product with
the count, two differences and a sum), each of at most one unit of 2^-24 of the
magnitudes that meet there, and half a step of the result's type."""
import math

import pytest
import torch

import warp_ctct

gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT = 2.0 ** -24


def rows(v, n):
    """A number, or one for each row, as a list."""
    return [float(v)] * n if not torch.is_tensor(v) else [float(x) for x in v.float().cpu()]


def oracle(logits, tokens=None, tokens_lengths=None, repetition_penalty=1.0, presence_penalty=0.0,
           frequency_penalty=0.0, bias=None, allowed=None):
    l = logits.detach().double().cpu()
    (N, V), size = l.shape, l.abs()
    if tokens is not None:
        rep, pre, fre = (rows(v, N) for v in (repetition_penalty, presence_penalty, frequency_penalty))
        for n in range(N):
            H = tokens.shape[1]
            h = H if tokens_lengths is None else min(max(int(tokens_lengths[n]), 0), H)
            count = {}
            for v in tokens[n, :h].tolist():
                if 0 <= v < V:
                    count[v] = count.get(v, 0) + 1
            for v, c in count.items():
                x = float(l[n, v])
                x = x / rep[n] if x > 0 else x * rep[n]
                size[n, v] = abs(x) + abs(pre[n]) + abs(fre[n]) * c
                l[n, v] = x - pre[n] - fre[n] * c
    if bias is not None:
        l = l + bias.double().cpu()
        size = size + bias.double().cpu().abs()
    if allowed is not None:
        if allowed.dtype == torch.int32:
            bits = allowed.cpu().reshape(-1, allowed.shape[-1])
            at = torch.arange(V)
            allowed = ((bits[:, at // 32].long() >> (at % 32)) & 1) != 0
        l = torch.where(allowed.cpu(), l, -math.inf)
    return l, 6 * UNIT * size


def compare(logits, **rules):
    got = warp_ctct.adjust_logits(logits, **rules)
    assert got.dtype == logits.dtype and got.shape == logits.shape and got.is_contiguous()
    want, tol = oracle(logits, **rules)
    got = got.double().cpu()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    far = (got - want).abs() <= tol + torch.finfo(logits.dtype).eps / 2 * want.abs() + 2.0 ** -25
    assert bool((same | far).all()), (got - want)[~(same | far)][:5]


def pack(allowed):
    V = allowed.shape[-1]
    wide = torch.nn.functional.pad(allowed.long(), (0, -V % 32)).unflatten(-1, (-1, 32))
    words = (wide << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def make(N, V, H, dtype, seed=0, many=torch.int32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    few = max(1, min(V, 2 * H))
    return dict(logits=(3 * draw(N, V)).to(dtype),
                tokens=torch.randint(0, few, (N, H), device="cuda", generator=gen).to(many) * (V // few),
                tokens_lengths=torch.randint(0, H + 1, (N,), device="cuda", generator=gen),
                repetition_penalty=0.7 + draw(N).abs(), presence_penalty=draw(N) * 0.3,
                frequency_penalty=draw(N).abs() * 0.2, bias=draw(V), allowed=draw(N, V) < 0.8)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,V,H", [(1, 1, 1), (2, 7, 3), (3, 32, 40), (4, 33, 5), (2, 1000, 600), (5, 2048, 17),
                                   (2, 2056, 80), (1, 30001, 200), (40, 8192, 70), (300, 4100, 9)])
def test_against_the_rules(N, V, H, dtype):
    rules = make(N, V, H, dtype, seed=V, many=torch.int64 if N % 2 else torch.int32)
    compare(**rules)
    packed = dict(rules, allowed=pack(rules["allowed"]))
    assert torch.equal(warp_ctct.adjust_logits(**packed), warp_ctct.adjust_logits(**rules))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_each_rule_alone(dtype):
    rules = make(6, 515, 30, dtype)
    logits, tokens = rules["logits"], rules["tokens"]
    assert torch.equal(warp_ctct.adjust_logits(logits), logits)
    assert torch.equal(warp_ctct.adjust_logits(logits, tokens), logits)
    for rule in (dict(repetition_penalty=1.7), dict(presence_penalty=0.25), dict(frequency_penalty=-0.5),
                 dict(repetition_penalty=rules["repetition_penalty"].double()),
                 dict(tokens_lengths=rules["tokens_lengths"].int(), presence_penalty=2)):
        compare(logits, tokens=tokens, **rule)
    compare(logits, bias=rules["bias"])
    compare(logits, bias=rules["bias"].to(dtype).expand(6, 515))
    compare(logits, bias=torch.randn(6, 520, device="cuda")[:, 3:518])
    compare(logits, allowed=rules["allowed"])
    compare(logits, allowed=rules["allowed"][2])
    compare(logits, allowed=pack(rules["allowed"])[1])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_allow_nothing_and_values_that_are_not_finite(dtype):
    rules = make(5, 200, 50, dtype)
    rules["allowed"][1] = False
    low = torch.finfo(dtype).min
    rules["logits"][0, :4] = torch.tensor([low, -math.inf, math.inf, math.nan], device="cuda", dtype=dtype)
    rules["logits"][2] = -math.inf
    rules["allowed"][0, 3] = False              # what is not allowed is minus infinity, a NaN too
    rules["tokens"][0, :4] = torch.arange(4, device="cuda", dtype=torch.int32)
    rules["tokens_lengths"][0] = 50
    rules.update(repetition_penalty=1.5, bias=torch.where(rules["bias"] > 1, -math.inf, rules["bias"]))
    rules["bias"][:4] = 0
    if dtype != torch.bfloat16 and dtype != torch.float32:
        rules["logits"][0, 0] = low / 2         # (low * 1.5 is beyond the type: it becomes minus infinity there)
    got = warp_ctct.adjust_logits(**rules)
    assert bool((got[1] == -math.inf).all()) and bool((got[2] == -math.inf).all())
    assert float(got[0, 1]) == -math.inf and float(got[0, 3]) == -math.inf
    assert float(got[0, 2]) == (math.inf if rules["allowed"][0, 2] else -math.inf)
    keep = [1, 2, 3, 4]
    compare(**{k: v[keep] if torch.is_tensor(v) and v.shape[0] == 5 else v for k, v in rules.items()})


@gpu
def test_tokens_out_of_range_and_lengths_out_of_range():
    rules = make(4, 100, 12, torch.float32)
    rules["tokens"][:, ::3] = -1
    rules["tokens"][:, 1::3] = 100
    rules["tokens"][0, 2] = 2 ** 31 - 1
    rules["tokens_lengths"] = torch.tensor([12, 50, -4, 0], device="cuda")
    compare(**rules)
    wide = dict(rules, tokens=rules["tokens"].long())
    wide["tokens"][1, 0] = 2 ** 40 + 5          # not 5
    compare(**wide)
    compare(**dict(wide, tokens=wide["tokens"][:, :0], tokens_lengths=None))
    compare(**dict(rules, tokens=torch.full((4, 12), 7, device="cuda", dtype=torch.int16), tokens_lengths=None))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_inputs(dtype):
    rules = make(6, 96, 20, dtype)
    wide = torch.randn(6, 300, device="cuda").to(dtype)
    for view in (wide[:, :96], wide[:, 3:99], wide[:, ::3][:, :96], wide[:1, :96].expand(6, 96)):
        compare(**dict(rules, logits=view))
    compare(**dict(rules, tokens=torch.randint(0, 96, (20, 6), device="cuda").t(),
                   allowed=torch.rand(6, 200, device="cuda")[:, 50:146] < 0.5))


@gpu
def test_no_rows_and_a_graph():
    assert warp_ctct.adjust_logits(torch.zeros(0, 5, device="cuda")).shape == (0, 5)
    rules = make(9, 3000, 64, torch.bfloat16)
    warp_ctct.adjust_logits(**rules)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    rules["tokens_lengths"] = rules["tokens_lengths"].int()
    with torch.cuda.graph(graph):
        kept = warp_ctct.adjust_logits(**rules)
    for seed in range(3):
        for k, v in make(9, 3000, 64, torch.bfloat16, seed=seed + 1).items():
            rules[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kept, warp_ctct.adjust_logits(**rules))


@gpu
def test_refusals_on_the_gpu():
    ones = lambda *s, **k: torch.ones(*s, device="cuda", **k)  # noqa: E731
    x = ones(3, 64)
    for bad in (dict(logits=ones(64)), dict(tokens=ones(3, 4)), dict(tokens=ones(2, 4, dtype=torch.int32)),
                dict(tokens_lengths=ones(3, dtype=torch.int32)), dict(repetition_penalty=0.0),
                dict(repetition_penalty=-1.0), dict(presence_penalty=ones(2)), dict(bias=ones(63)),
                dict(bias=ones(2, 64)), dict(allowed=ones(64)), dict(allowed=ones(3, 3, dtype=torch.int32)),
                dict(allowed=ones(63, dtype=torch.bool)), dict(bias=torch.ones(64)),
                dict(logits=ones(3, 64, requires_grad=True)), dict(bias=ones(64, requires_grad=True)),
                dict(tokens=ones(3, 4, dtype=torch.int32), tokens_lengths=ones(4, dtype=torch.int32))):
        with pytest.raises(RuntimeError):
            warp_ctct.adjust_logits(**{**dict(logits=x), **bad})


def test_refusals_without_a_gpu():
    with pytest.raises(RuntimeError, match="GPU"):
        warp_ctct.adjust_logits(torch.zeros(2, 8))
