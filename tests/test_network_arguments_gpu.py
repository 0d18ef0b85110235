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
