"""Arguments that the operators beside the losses have in common: what all of them
refuse, and what each converts."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import warp_ctct

pytestmark = pytest.mark.gpu
N, T, E, K, S = 3, 20, 8, 4, 16


def rand(*shape, **options):
    return torch.rand(*shape, device="cuda", **options)


def calls():
    """Every operator with its floating inputs by name: all of them."""
    scan = lambda *lead: dict(x=rand(*lead, E), dt=rand(*lead, E), a=-rand(E, S), b=rand(*lead, S), c=rand(*lead, S),  # noqa: E731
                              skip=rand(E), gate=rand(*lead, E), dt_bias=rand(E))
    taps = dict(weight=rand(E, K), bias=rand(E))
    return [(warp_ctct.layer_norm, dict(x=rand(N, E), weight=rand(E), bias=rand(E))),
            (warp_ctct.causal_conv, dict(x=rand(N, T, E), initial_state=rand(N, K - 1, E), **taps)),
            (warp_ctct.causal_conv_step, dict(x=rand(N, E), state=rand(N, K - 1, E), **taps)),
            (warp_ctct.selective_scan, dict(initial_state=rand(N, E, S), **scan(N, T))),
            (warp_ctct.selective_scan_step, dict(state=rand(N, E, S), **scan(N))),
            (lambda **a: warp_ctct.adjust_logits(tokens=torch.ones(N, 2, device="cuda", dtype=torch.int32), **a),
             dict(logits=rand(N, E), repetition_penalty=1 + rand(N), presence_penalty=rand(N),
                  frequency_penalty=rand(N), bias=rand(E)))]


def test_tangents_are_refused():
    for operator, inputs in calls():
        for name, value in inputs.items():
            with forward_ad.dual_level():
                dual = dict(inputs, **{name: forward_ad.make_dual(value, torch.ones_like(value))})
                for tracking in (True, False):
                    with torch.set_grad_enabled(tracking), pytest.raises(RuntimeError, match="forward-mode"):
                        operator(**dual)
                operator(**inputs)
            operator(**inputs)


def with_lengths():
    """Every operator with lengths, as a function of them: outputs over T steps or tokens of N rows."""
    x, weight, dt, b = rand(N, T, E), rand(E, K), rand(N, T, E), rand(N, T, S)
    a, logits, tokens = -rand(E, S), rand(N, 16), torch.randint(0, 16, (N, T), device="cuda")
    return [lambda l: warp_ctct.causal_conv(x, weight, lengths=l, return_state=True),
            lambda l: warp_ctct.selective_scan(x, dt, a, b, b, lengths=l, return_state=True),
            lambda l: (warp_ctct.adjust_logits(logits, tokens, l, presence_penalty=0.5, frequency_penalty=0.1),)]


def test_lengths_out_of_the_range_of_int32_are_clamped():
    lengths = lambda values, dtype: torch.tensor(values, dtype=dtype).cuda()  # noqa: E731
    for operator in with_lengths():
        for dtype, values, clamped in (
                (torch.int64, [2 ** 32, 2 ** 63 - 1, 2 ** 33 + 5], [T, T, T]),
                (torch.int64, [-2 ** 32 - 5 + 2 ** 31, -2 ** 63, -2 ** 32 + 7], [0, 0, 0]),
                (torch.int64, [T + 1, 3, 0], [T, 3, 0]), (torch.uint32, [2 ** 32 - 1, 2 ** 31, 3], [T, T, 3]),
                (torch.uint64, [2 ** 64 - 1, 2 ** 63 + 2, 2 ** 32 + 4], [T, T, T]),
                (torch.uint64, [7, 0, T], [7, 0, T]), (torch.uint16, [65535, 2, 0], [T, 2, 0]),
                (torch.uint8, [255, 2, 0], [T, 2, 0]), (torch.int16, [-1, 300, 5], [0, T, 5])):
            got, want = operator(lengths(values, dtype)), operator(lengths(clamped, torch.int32))
            assert all(torch.equal(x, y) for x, y in zip(got, want)), (dtype, values)


def test_lengths_that_are_no_whole_numbers_are_refused():
    for operator in with_lengths():
        for dtype in (torch.bool, torch.complex64, torch.float32):
            with pytest.raises(RuntimeError, match="whole numbers"):
                operator(torch.ones(N, device="cuda", dtype=dtype))


def test_tokens_of_other_types():
    logits = rand(1, 8)
    tokens = lambda values, dtype: torch.tensor([values], dtype=dtype).cuda()  # noqa: E731
    rule = lambda t: warp_ctct.adjust_logits(logits, t, presence_penalty=0.5)  # noqa: E731
    want = rule(tokens([3, -1, 9], torch.int32))
    for dtype, values in ((torch.uint64, [3, 2 ** 32 + 5, 2 ** 64 - 7]), (torch.uint32, [3, 2 ** 32 - 6, 2 ** 31]),
                          (torch.uint16, [3, 65530, 8]), (torch.uint8, [3, 250, 8]), (torch.int8, [3, -3, -8]),
                          (torch.int16, [3, -3, 99]), (torch.int64, [3, 2 ** 32 + 5, -2 ** 63])):
        assert torch.equal(rule(tokens(values, dtype)), want), dtype
    for dtype in (torch.bool, torch.complex64, torch.float32):
        with pytest.raises(RuntimeError, match="whole numbers"):
            rule(torch.ones(1, 3, device="cuda", dtype=dtype))


def test_float64_is_float32():
    for operator, inputs in calls():
        if "state" in inputs:       # moved on in place: never converted
            narrow, wide = inputs["state"].clone(), inputs["state"].double()
            rest = {k: v for k, v in inputs.items() if k != "state"}
            want = operator(state=narrow, **rest)
            assert torch.equal(operator(state=inputs["state"], **{k: v.double() for k, v in rest.items()}), want)
            assert torch.equal(inputs["state"], narrow)
            with pytest.raises(RuntimeError, match="state"):
                operator(state=wide, **rest)
            continue
        leaves = {k: v.detach().requires_grad_(operator.__name__ != "<lambda>") for k, v in inputs.items()}
        wide = {k: v.detach().double().requires_grad_(v.requires_grad) for k, v in leaves.items()}
        want, got = operator(**leaves), operator(**wide)
        assert got.dtype == torch.float32 and torch.equal(got, want)
        if got.requires_grad:
            g = torch.rand_like(got)
            for x, y in zip(torch.autograd.grad(got, list(wide.values()), g),
                            torch.autograd.grad(want, list(leaves.values()), g)):
                assert x.dtype == torch.float64 and torch.equal(x.float(), y)


def test_states_of_integers_and_of_narrow_types():
    for operator, inputs in calls():
        if "initial_state" not in inputs:
            continue
        whole = torch.randint(-3, 4, inputs["initial_state"].shape, device="cuda")
        assert torch.equal(operator(**dict(inputs, initial_state=whole)),
                           operator(**dict(inputs, initial_state=whole.float())))
        with pytest.raises(RuntimeError, match="initial_state"):
            operator(**dict(inputs, initial_state=whole.half()))
