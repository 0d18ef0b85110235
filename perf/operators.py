"""The operators beside the losses, case by case: what makes the label scores g (layer norm, short causal
convolution, selective scan) and what is done to the joiner's logits before a token is taken from them.

``run`` computes a case either in plain elementary torch operations (``own`` false) or through
``warp_ctct`` (``own`` true); ``exact`` gives the same outputs from the definitions in 64 bits.
"""
import math
import os
import sys

import torch

own = False

_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _package():
    """The framework's package, from the source tree."""
    at = os.path.join(os.getcwd(), "warp-ctct_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import warp_ctct
    return warp_ctct


# ---- cases --------------------------------------------------------------------------------------

def listed():
    return [
        # the prediction network's norm for the four hypotheses of a beam, one token each
        {"name": "norm_token_f32", "op": "norm", "rows": 4, "width": 512, "dtype": "f32", "train": False},
        # training on label rows (32 utterances, 80 labels and the start), a width that is no power of two
        {"name": "norm_labels_f16", "op": "norm", "rows": 2592, "width": 641, "dtype": "f16", "train": True},
        # training on encoder frames (32 utterances of 400 frames) at the vocabulary's width
        {"name": "norm_frames_bf16", "op": "norm", "rows": 12800, "width": 2048, "dtype": "bf16", "train": True},
        # one token for each of 32 utterances; those that emitted blank do not advance
        {"name": "conv_token_f16", "op": "conv_step", "n": 32, "e": 1024, "k": 4, "dtype": "f16"},
        # training on ragged frames
        {"name": "conv_frames_bf16", "op": "conv", "n": 32, "l": 400, "e": 2048, "k": 4, "dtype": "bf16",
         "silu": True, "train": True},
        # one token for the eight hypotheses of a beam
        {"name": "scan_token_f32", "op": "scan_step", "n": 8, "e": 512, "s": 16, "g": 1, "dtype": "f32"},
        # one token for each of 256 utterances served together
        {"name": "scan_tokens_bf16", "op": "scan_step", "n": 256, "e": 2048, "s": 16, "g": 1, "dtype": "bf16"},
        # training on label rows in float32, without a gate, an odd width and two groups
        {"name": "scan_labels_f32", "op": "scan", "n": 32, "l": 81, "e": 500, "s": 16, "g": 2, "dtype": "f32",
         "gate": False, "train": True},
        # training on ragged frames
        {"name": "scan_frames_bf16", "op": "scan", "n": 32, "l": 400, "e": 1024, "s": 16, "g": 1, "dtype": "bf16",
         "gate": True, "train": True},
        # one long recording read in before decoding starts
        {"name": "scan_prompt_bf16", "op": "scan", "n": 1, "l": 16384, "e": 2048, "s": 16, "g": 1, "dtype": "bf16",
         "gate": True, "train": False},
        # the logits of a beam of eight with their label histories
        {"name": "logits_beam_f32", "op": "logits", "n": 8, "v": 1024, "h": 80, "dtype": "f32", "packed": False},
        # the logits of 128 utterances over a large vocabulary, each with penalties and a grammar of its own
        {"name": "logits_batch_bf16", "op": "logits", "n": 128, "v": 65536, "h": 300, "dtype": "bf16",
         "packed": True},
    ]


def _between(rng, lo, hi):
    """A whole number, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "conv", "conv_step", "scan", "scan", "prompt", "scan_step", "logits"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "norm":
        width = _between(rng, 16, 12000)
        rows = _between(rng, 1, max(1, min(40000, 20000000 // width)))
        return {"op": "norm", "rows": rows, "width": width, "dtype": dtype, "train": rng.random() < 0.6}
    if op == "conv_step":
        return {"op": "conv_step", "n": _between(rng, 1, 300), "e": _between(rng, 16, 4096),
                "k": rng.randint(1, 8), "dtype": dtype}
    if op == "conv":
        e, n = _between(rng, 16, 4096), _between(rng, 1, 64)
        most = max(1, min(4096, 20000000 // (e * n)))
        return {"op": "conv", "n": n, "l": _between(rng, 1, most), "e": e, "k": rng.randint(2, 6), "dtype": dtype,
                "silu": rng.random() < 0.5, "train": rng.random() < 0.7}
    if op == "scan":
        e, n, s = 2 * _between(rng, 8, 1024), _between(rng, 1, 64), rng.choice([4, 7, 8, 16, 16, 24, 32, 64])
        most = max(1, min(1500, 150000000 // (e * n * s)))
        return {"op": "scan", "n": n, "l": _between(rng, 1, most), "e": e, "s": s, "g": rng.choice([1, 1, 2]),
                "dtype": dtype, "gate": rng.random() < 0.6, "train": True}
    if op == "prompt":
        e, n = _between(rng, 64, 2048), _between(rng, 1, 8)
        most = max(64, min(16384, 400000000 // (e * n * 16)))
        return {"op": "scan", "n": n, "l": _between(rng, 64, most), "e": e, "s": 16, "g": 1, "dtype": dtype,
                "gate": rng.random() < 0.8, "train": False}
    if op == "scan_step":
        return {"op": "scan_step", "n": _between(rng, 1, 256), "e": 2 * _between(rng, 16, 1024),
                "s": rng.choice([4, 9, 16, 16, 32, 64]), "g": rng.choice([1, 2]), "dtype": dtype}
    return {"op": "logits", "n": _between(rng, 1, 128), "v": _between(rng, 32, 65536), "h": _between(rng, 1, 1500),
            "dtype": dtype, "packed": rng.random() < 0.5}


def _lengths(n, l):
    """Ragged lengths from half of `l` up to `l`, the same for every seed."""
    return [max(1, l - (i * (l // 2)) // max(1, n - 1)) if n > 1 else l for i in range(n)]


# ---- inputs -------------------------------------------------------------------------------------

def prepare(case, seed):
    op, dtype = case["op"], _DTYPE[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, to=dtype, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(to)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, device="cuda", generator=gen) * (hi - lo) + lo

    def whole(lo, hi, *shape, to=torch.int32):
        return torch.randint(lo, hi, shape, device="cuda", generator=gen).to(to)

    st = {"case": case}
    f32 = torch.float32
    if op == "norm":
        r, d = case["rows"], case["width"]
        st["x"] = (torch.randn(r, d, device="cuda", generator=gen) * 2 + uniform(r, 1, lo=-1.0)).to(dtype)
        st["weight"] = uniform(d, lo=0.5, hi=1.5)
        st["bias"] = normal(d, to=f32, scale=0.2)
        grads = ["x", "weight", "bias"]
        if case["train"]:
            st["gout"] = normal(r, d)
    elif op == "conv":
        n, l, e, k = case["n"], case["l"], case["e"], case["k"]
        st["x"] = normal(n, l, e)
        st["weight"] = normal(e, k, to=f32, scale=k ** -0.5)
        st["bias"] = normal(e, to=f32, scale=0.2)
        st["initial"] = normal(n, k - 1, e)
        st["lengths"] = torch.tensor(_lengths(n, l), dtype=torch.int32, device="cuda")
        grads = ["x", "weight", "bias", "initial"]
        if case["train"]:
            st["gout"], st["gstate"] = normal(n, l, e), normal(n, k - 1, e)
    elif op == "conv_step":
        n, e, k = case["n"], case["e"], case["k"]
        st["x"], st["state"] = normal(n, e), normal(n, k - 1, e)
        st["weight"] = normal(e, k, to=f32, scale=k ** -0.5)
        st["bias"] = normal(e, to=f32, scale=0.2)
        st["advance"] = uniform(n) < 0.7
    elif op in ("scan", "scan_step"):
        n, e, s, g = case["n"], case["e"], case["s"], case["g"]
        lead = (n, case["l"]) if op == "scan" else (n,)
        # x and the gate are the halves of one projection, b and c of another
        both = normal(*lead, 2 * e)
        st["x"] = both[..., :e]
        st["gate"] = both[..., e:] if op == "scan_step" or case["gate"] else None
        parts = normal(*lead, 2 * g * s)
        st["b"] = parts[..., :g * s].unflatten(-1, (g, s))
        st["c"] = parts[..., g * s:].unflatten(-1, (g, s))
        st["dt"] = normal(*lead, e, scale=0.5)
        st["a"] = -torch.arange(1, s + 1, device="cuda", dtype=f32) * uniform(e, 1, lo=0.5, hi=1.5)
        st["skip"] = normal(e, to=f32)
        st["dt_bias"] = torch.log(torch.expm1(torch.exp(uniform(e, lo=math.log(1e-3), hi=math.log(1e-1)))))
        grads = ["x", "dt", "a", "b", "c", "skip", "gate", "dt_bias", "initial"]
        if op == "scan_step":
            st["state"] = normal(n, e, s, to=f32)
            st["advance"] = uniform(n) < 0.7
        else:
            st["initial"] = normal(n, e, s, to=f32, scale=0.5)
            st["lengths"] = torch.tensor(_lengths(n, case["l"]), dtype=torch.int32, device="cuda")
            if case["train"]:
                st["gout"] = normal(n, case["l"], e)
                st["gstate"] = normal(n, e, s, to=f32, scale=0.1)
    else:
        n, v, h = case["n"], case["v"], case["h"]
        st["logits"] = normal(n, v, scale=3.0)
        st["tokens"] = whole(0, v, n, h, to=torch.int64 if case["packed"] else torch.int32)
        st["tokens"][:, h // 2:] = st["tokens"][:, :h - h // 2].clone()   # histories repeat themselves
        st["tokens_lengths"] = whole(0, h + 1, n)
        st["repetition"] = uniform(n, lo=0.8, hi=1.6)
        st["presence"] = uniform(n, lo=-0.2, hi=0.6)
        st["frequency"] = uniform(n, hi=0.3)
        st["bias"] = normal(v, to=f32, scale=0.5)
        if case["packed"]:
            st["allowed"] = whole(-2 ** 31, 2 ** 31, n, (v + 31) // 32, to=torch.int32)
        else:
            st["allowed"] = uniform(v) < 0.8
    if case.get("train"):
        st["leaves"] = [k for k in grads if st.get(k) is not None]
        for k in st["leaves"]:
            st[k] = st[k].detach().requires_grad_(True)
    return st


# ---- one pass -----------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


def _run_own(st):
    w, case = _package(), st["case"]
    op = case["op"]
    if op == "norm":
        out = w.layer_norm(st["x"], st["weight"], st["bias"], 1e-5)
        ends, given = [out], [st.get("gout")]
        got = {"out": out}
    elif op == "conv":
        out, last = w.causal_conv(st["x"], st["weight"], st["bias"], lengths=st["lengths"],
                                  initial_state=st["initial"], activation="silu" if case["silu"] else None,
                                  return_state=True)
        ends, given = [out, last], [st.get("gout"), st.get("gstate")]
        got = {"out": out, "state": last}
    elif op == "scan":
        out, last = w.selective_scan(st["x"], st["dt"], st["a"], st["b"], st["c"], skip=st["skip"], gate=st["gate"],
                                     dt_bias=st["dt_bias"], softplus=True, lengths=st["lengths"],
                                     initial_state=st["initial"], return_state=True)
        ends, given = [out, last], [st.get("gout"), st.get("gstate")]
        got = {"out": out, "state": last}
    elif op == "conv_step":
        out = w.causal_conv_step(st["x"], st["state"], st["weight"], st["bias"], activation="silu",
                                 advance=st["advance"])
        return {"out": out, "state": st["state"]}
    elif op == "scan_step":
        out = w.selective_scan_step(st["x"], st["state"], st["dt"], st["a"], st["b"], st["c"], skip=st["skip"],
                                    gate=st["gate"], dt_bias=st["dt_bias"], softplus=True, advance=st["advance"])
        return {"out": out, "state": st["state"]}
    else:
        return {"out": w.adjust_logits(st["logits"], st["tokens"], st["tokens_lengths"],
                                       repetition_penalty=st["repetition"], presence_penalty=st["presence"],
                                       frequency_penalty=st["frequency"], bias=st["bias"], allowed=st["allowed"])}
    if case["train"]:
        grads = torch.autograd.grad(ends, [st[k] for k in st["leaves"]], given)
        got.update({"grad_" + k: g for k, g in zip(st["leaves"], grads)})
    return got


def _sigmoid(v):
    return 1 / (1 + torch.exp(-v))


def _plain_norm(st):
    dtype = st["x"].dtype
    x, weight, bias = st["x"].float(), st["weight"], st["bias"]
    mid = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((mid * mid).mean(-1, keepdim=True) + 1e-5)
    xh = mid * r
    got = {"out": (xh * weight + bias).to(dtype)}
    if st["case"]["train"]:
        g = st["gout"].float()
        u = g * weight
        gx = r * (u - u.mean(-1, keepdim=True) - xh * (u * xh).mean(-1, keepdim=True))
        got.update(grad_x=gx.to(dtype), grad_weight=(g * xh).sum(0), grad_bias=g.sum(0))
    return got


def _valid(lengths, l):
    return (torch.arange(l, device=lengths.device) < lengths[:, None])[..., None]


def _plain_conv(st):
    case, dtype = st["case"], st["x"].dtype
    (n, l, e), k = st["x"].shape, case["k"]
    ok = _valid(st["lengths"], l)
    ext = torch.cat([st["initial"].float(), st["x"].float()], 1)            # (n, k-1+l, e)
    windows = ext.unfold(1, k, 1)                                           # (n, l, e, k)
    pre = (windows * st["weight"]).sum(-1) + st["bias"]
    out = pre * _sigmoid(pre) if case["silu"] else pre
    at = (st["lengths"].long()[:, None] + torch.arange(k - 1, device=ext.device))[..., None].expand(n, k - 1, e)
    got = {"out": torch.where(ok, out, 0).to(dtype), "state": ext.gather(1, at).to(dtype)}
    if case["train"]:
        g = torch.where(ok, st["gout"].float(), 0)
        if case["silu"]:
            sig = _sigmoid(pre)
            g = g * sig * (1 + pre * (1 - sig))
        wide = torch.nn.functional.pad(g, (0, 0, k - 1, k - 1))
        gext = (wide.unfold(1, k, 1) * st["weight"].flip(1)).sum(-1)        # (n, l+k-1, e)
        gext = gext.scatter_add(1, at, st["gstate"].float())
        got.update(grad_x=gext[:, k - 1:].to(dtype), grad_weight=(windows * g[..., None]).sum((0, 1)),
                   grad_bias=g.sum((0, 1)), grad_initial=gext[:, :k - 1].to(dtype))
    return got


def _plain_conv_step(st):
    dtype, go = st["x"].dtype, st["advance"][:, None]
    ext = torch.cat([st["state"], st["x"][:, None]], 1)
    pre = (ext.float() * st["weight"].t()).sum(1) + st["bias"]
    out = torch.where(go, pre * _sigmoid(pre), 0).to(dtype)
    st["state"].copy_(torch.where(go[..., None], ext[:, 1:], st["state"]))
    return {"out": out, "state": st["state"]}


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _linear_scan(a, u):
    """h[t] = a[t] h[t-1] + u[t] along dim 1, in log2(l) rounds over the whole tensors."""
    d, l = 1, a.shape[1]
    while d < l:
        u = torch.cat([u[:, :d], u[:, d:] + a[:, d:] * u[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return u


def _of_group(v, e):
    """(..., g, s) for every one of e channels: (..., e, s)."""
    return v.float().repeat_interleave(e // v.shape[-2], -2)


def _plain_scan(st):
    case, dtype = st["case"], st["x"].dtype
    n, l, e = st["x"].shape
    g, s = st["b"].shape[-2:]
    ok = _valid(st["lengths"], l)
    x = st["x"].float()
    raw = st["dt"].float() + st["dt_bias"]
    d = torch.where(ok, _softplus(raw), 0)
    b, c = _of_group(st["b"], e), _of_group(st["c"], e)
    a = torch.exp(d[..., None] * st["a"])                                   # (n, l, e, s)
    u = (d * x)[..., None] * b
    u[:, 0] += a[:, 0] * st["initial"]
    h = _linear_scan(a, u)
    del u
    y = (h * c).sum(-1) + st["skip"] * x
    z = st["gate"].float() if st["gate"] is not None else None
    out = y if z is None else y * z * _sigmoid(z)
    got = {"out": torch.where(ok, out, 0).to(dtype), "state": h[:, -1].clone()}
    if not case["train"]:
        return got
    go = torch.where(ok, st["gout"].float(), 0)
    gy = go if z is None else go * z * _sigmoid(z)
    gu = c * gy[..., None]
    gu[:, -1] += st["gstate"]
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    gh = _linear_scan(later.flip(1), gu.flip(1)).flip(1)
    del gu, later
    back = gh * a
    got["grad_initial"] = back[:, 0].clone()
    back[:, 0] *= st["initial"]
    back[:, 1:] *= h[:, :-1]                                                # gh a h[t-1]
    ghb = (gh * b).sum(-1)
    gd = x * ghb + (back * st["a"]).sum(-1)
    graw = torch.where(ok, gd * _sigmoid(raw), 0)
    sums = lambda v: v.unflatten(2, (g, e // g)).sum(3)                     # noqa: E731
    got.update(grad_x=torch.where(ok, st["skip"] * gy + d * ghb, 0).to(dtype), grad_dt=graw.to(dtype),
               grad_a=(back * d[..., None]).sum((0, 1)),
               grad_b=torch.where(ok[..., None], sums(gh * (d * x)[..., None]), 0).to(dtype),
               grad_c=torch.where(ok[..., None], sums(h * gy[..., None]), 0).to(dtype),
               grad_skip=(gy * x).sum((0, 1)), grad_dt_bias=graw.sum((0, 1)))
    if z is not None:
        sig = _sigmoid(z)
        got["grad_gate"] = (go * y * sig * (1 + z * (1 - sig))).to(dtype)
    return got


def _plain_scan_step(st):
    dtype, e, go = st["x"].dtype, st["x"].shape[1], st["advance"][:, None]
    x, z = st["x"].float(), st["gate"].float()
    d = _softplus(st["dt"].float() + st["dt_bias"])
    h = torch.exp(d[..., None] * st["a"]) * st["state"] + (d * x)[..., None] * _of_group(st["b"], e)
    y = (h * _of_group(st["c"], e)).sum(-1) + st["skip"] * x
    st["state"].copy_(torch.where(go[..., None], h, st["state"]))
    return {"out": torch.where(go, y * z * _sigmoid(z), 0).to(dtype), "state": st["state"]}


def _plain_logits(st):
    l = st["logits"].float()
    (n, v), h = l.shape, st["tokens"].shape[1]
    here = torch.arange(h, device=l.device) < st["tokens_lengths"][:, None]
    count = torch.zeros_like(l).scatter_add_(1, st["tokens"].long(), here.float())
    seen = count > 0
    rep = st["repetition"][:, None]
    l = torch.where(seen, torch.where(l > 0, l / rep, l * rep), l)
    l = l - torch.where(seen, st["presence"][:, None], 0) - st["frequency"][:, None] * count
    l = l + st["bias"]
    allowed = st["allowed"]
    if st["case"]["packed"]:
        bits = (allowed[..., None] >> torch.arange(32, device=l.device, dtype=torch.int32)) & 1
        allowed = bits.flatten(1)[:, :v] != 0
    return {"out": torch.where(allowed, l, -math.inf).to(st["logits"].dtype)}


_PLAIN = {"norm": _plain_norm, "conv": _plain_conv, "conv_step": _plain_conv_step, "scan": _plain_scan,
          "scan_step": _plain_scan_step, "logits": _plain_logits}


# ---- what a pass cannot do without --------------------------------------------------------------

def work(case):
    op, w = case["op"], _SIZE[case["dtype"]]
    train = bool(case.get("train"))
    if op == "norm":
        cells = case["rows"] * case["width"]
        return {"bytes": cells * w * (4 if train else 2) + case["width"] * (16 if train else 8),
                "flops": cells * (22 if train else 8)}
    if op == "conv":
        live, cells = sum(_lengths(case["n"], case["l"])) * case["e"], case["n"] * case["l"] * case["e"]
        small = case["e"] * (4 * case["k"] + 4) + case["n"] * (2 * w * (case["k"] - 1) * case["e"])
        return {"bytes": (live + cells) * w * (2 if train else 1) + small * (2 if train else 1),
                "flops": live * (2 * case["k"] + 6) * (3 if train else 1)}
    if op == "conv_step":
        cells = case["n"] * case["e"]
        return {"bytes": cells * w * (2 + 2 * (case["k"] - 1)) + case["e"] * 4 * (case["k"] + 1),
                "flops": cells * (2 * case["k"] + 6)}
    if op == "scan":
        steps, n, e, s, g = sum(_lengths(case["n"], case["l"])), case["n"], case["e"], case["s"], case["g"]
        z = 1 if case["gate"] else 0
        all_steps, small = n * case["l"], 8 * n * e * s + 4 * e * (s + 2)
        if not train:
            return {"bytes": w * (steps * (e * (2 + z) + 2 * g * s) + all_steps * e) + small,
                    "flops": steps * e * (7 * s + 20)}
        return {"bytes": w * (steps * (e * (3 + z) + 2 * g * s) + all_steps * (e * (3 + z) + 2 * g * s)) + 2 * small,
                "flops": steps * e * (25 * s + 50)}
    if op == "scan_step":
        cells, s = case["n"] * case["e"], case["s"]
        return {"bytes": cells * (8 * s + 4 * w) + case["n"] * 2 * case["g"] * s * w + case["e"] * 4 * (s + 2),
                "flops": cells * (7 * s + 20)}
    cells = case["n"] * case["v"]
    mask = cells // 8 if case["packed"] else case["v"]
    return {"bytes": cells * w * 2 + mask + 4 * case["v"] + case["n"] * case["h"] * (8 if case["packed"] else 4) // 2,
            "flops": cells * 6}


# ---- from the definitions, in 64 bits -----------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    for k, v in list(st.items()):
        if torch.is_tensor(v) and v.is_floating_point():
            st[k] = v.detach().double()
    leaves = st.get("leaves") or []
    for k in leaves:
        st[k] = st[k].contiguous().requires_grad_(True)
    with torch.set_grad_enabled(bool(leaves)):
        got, ends, given = _EXACT[case["op"]](st)
        if leaves:
            grads = torch.autograd.grad(ends, [st[k] for k in leaves], given)
            got.update({"grad_" + k: v for k, v in zip(leaves, grads)})
    return {k: v.detach() for k, v in got.items()}


def _exact_norm(st):
    x, d = st["x"], st["x"].shape[1]
    mean = x.sum(1, keepdim=True) / d
    var = ((x - mean) ** 2).sum(1, keepdim=True) / d
    out = (x - mean) / torch.sqrt(var + 1e-5) * st["weight"] + st["bias"]
    return {"out": out}, [out], [st.get("gout")]


def _silu64(v):
    return v * torch.sigmoid(v)


def _exact_conv(st):
    case, x = st["case"], st["x"]
    (n, l, e), k = x.shape, case["k"]
    ext = torch.cat([st["initial"], x], 1)
    pre = st["bias"]
    for i in range(k):
        pre = pre + st["weight"][:, i] * ext[:, i:i + l]
    out = _silu64(pre) if case["silu"] else pre
    steps = st["lengths"].tolist()
    live = torch.zeros(n, l, 1, dtype=torch.bool, device=x.device)
    for i, t in enumerate(steps):
        live[i, :t] = True
    out = out.masked_fill(~live, 0.0)
    last = torch.stack([ext[i, t:t + k - 1] for i, t in enumerate(steps)])
    return {"out": out, "state": last}, [out, last], [st.get("gout"), st.get("gstate")]


def _exact_conv_step(st):
    pre = st["bias"] + st["weight"][:, -1] * st["x"]
    for i in range(st["state"].shape[1]):
        pre = pre + st["weight"][:, i] * st["state"][:, i]
    keep = ~st["advance"]
    out = _silu64(pre)
    out[keep] = 0.0
    after = torch.cat([st["state"][:, 1:], st["x"][:, None]], 1) if st["state"].shape[1] else st["state"].clone()
    after[keep] = st["state"][keep]
    return {"out": out, "state": after}, None, None


def _exact_step(h, x, d, a, b, c):
    e = x.shape[1]
    b, c = (v.repeat_interleave(e // v.shape[1], 1) for v in (b, c))
    h = h * torch.exp(d[..., None] * a) + (d * x)[..., None] * b
    return h, torch.einsum("nes,nes->ne", h, c)


def _exact_scan(st):
    x, l = st["x"], st["x"].shape[1]
    d = torch.nn.functional.softplus(st["dt"] + st["dt_bias"], threshold=1e6)
    h, ys = st["initial"], []
    for t in range(l):
        live = (t < st["lengths"])[:, None]
        new, y = _exact_step(h, x[:, t], d[:, t], st["a"], st["b"][:, t], st["c"][:, t])
        h = torch.where(live[..., None], new, h)
        y = y + st["skip"] * x[:, t]
        if st["gate"] is not None:
            y = y * _silu64(st["gate"][:, t])
        ys.append(y.masked_fill(~live, 0.0))
    out = torch.stack(ys, 1)
    return {"out": out, "state": h}, [out, h], [st.get("gout"), st.get("gstate")]


def _exact_scan_step(st):
    d = torch.nn.functional.softplus(st["dt"] + st["dt_bias"], threshold=1e6)
    h, y = _exact_step(st["state"], st["x"], d, st["a"], st["b"], st["c"])
    out = (y + st["skip"] * st["x"]) * _silu64(st["gate"])
    keep = ~st["advance"]
    out[keep] = 0.0
    h[keep] = st["state"][keep]
    return {"out": out, "state": h}, None, None


def _exact_logits(st):
    l, (n, v) = st["logits"].clone(), st["logits"].shape
    for i in range(n):
        history = st["tokens"][i, :int(st["tokens_lengths"][i])].long()
        token, count = history.unique(return_counts=True)
        old, rep = l[i, token], st["repetition"][i]
        l[i, token] = torch.where(old > 0, old / rep, old * rep) - st["presence"][i] - st["frequency"][i] * count
    l = l + st["bias"]
    at = torch.arange(v, device=l.device)
    if st["case"]["packed"]:
        banned = torch.bitwise_and(st["allowed"].long()[:, at // 32], 1 << (at % 32)) == 0
    else:
        banned = (~st["allowed"]).expand(n, v)
    return {"out": l.masked_fill(banned, -math.inf)}, None, None


_EXACT = {"norm": _exact_norm, "conv": _exact_conv, "conv_step": _exact_conv_step, "scan": _exact_scan,
          "scan_step": _exact_scan_step, "logits": _exact_logits}
