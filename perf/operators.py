"""The dense side of a MoE block on one B200, as measurable cases: three operators, each through its public entry point.

  norm      ``fused.add_rms_norm``: residual sum and RMS norm of a token's row, optionally with the row in e4m3 (one scale per 128 columns)
  balance   ``fused.balance_loss``: the router's balance loss and the experts' counts
  linear    ``fused.linear``: a matrix product with bias, activation and residual in its epilogue (SwiGLU: tiles of 128 gate rows and
            128 up rows in the weight, as the experts have them)

Each as a forward pass alone (serving) and as a forward and backward pass (training). Where ``own`` is false, ``run`` computes the same from
elementary torch operations. Shapes: the Mixtral-8x7B-shaped block (hidden 4096, FFN 14336, 8 experts, 2 a token), the DeepSeek-V3-like layer
(hidden 7168, FFN 2048, 256 experts, 8 a token) and odd ones.
"""
from __future__ import annotations

import math

import torch

own = False
EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _norm(name, rows, hidden, mode, dtype="bf16", residual=True):
    """mode: serve (y and the sum), fp8 (those and the e4m3 rows), train (and gradients)."""
    return {"name": name, "op": "norm", "rows": rows, "hidden": hidden, "mode": mode, "dtype": dtype, "residual": residual}


def _balance(name, rows, experts, k, scores, train=True, padded=0.0, dtype="fp32"):
    return {"name": name, "op": "balance", "rows": rows, "experts": experts, "k": k, "scores": scores, "train": train, "padded": padded, "dtype": dtype}


def _linear(name, rows, inputs, outputs, activation, bias=False, residual=False, train=False):
    """outputs: rows of the weight (swiglu: the result has half as many columns)."""
    return {"name": name, "op": "linear", "rows": rows, "inputs": inputs, "outputs": outputs, "activation": activation, "bias": bias, "residual": residual, "train": train}


def listed():
    return [
        # The norm in front of the block in a decode step of one user: latency alone.
        _norm("norm_decode_1", 1, 4096, "serve"),
        # A prefill whose rows leave in e4m3 through the dispatch.
        _norm("norm_prefill_4096_fp8", 4096, 7168, "fp8"),
        # The training benchmark's step: eight sequences of 4096 tokens, the residual stream in bf16.
        _norm("norm_train_32768", 32768, 4096, "train"),
        # A small model in fp32 with an odd hidden size and no residual.
        _norm("norm_train_odd_fp32", 1777, 1001, "train", "fp32", residual=False),
        # Monitoring the routing of a small evaluation batch.
        _balance("balance_eval_61", 61, 64, 6, "softmax", train=False),
        # The training benchmark's router.
        _balance("balance_train_32768x8", 32768, 8, 2, "softmax"),
        # A padded batch through the router of many experts, normalised sigmoid scores.
        _balance("balance_train_16384x256", 16384, 256, 8, "sigmoid", padded=0.2),
        # Shared expert's first projection, decode step of one token: the weight's bytes are the time.
        _linear("linear_decode_1", 1, 7168, 4096, "swiglu"),
        # Its second projection for a decode batch, on top of the routed experts' output.
        _linear("linear_decode_48", 48, 2048, 7168, "none", residual=True),
        # An odd prompt through an FFN layer with biases, sizes that fill no tile.
        _linear("linear_prefill_1235_odd", 1235, 1000, 2760, "silu", bias=True, residual=True),
        # A prefill through the shared expert's first projection.
        _linear("linear_prefill_4096", 4096, 7168, 4096, "swiglu"),
        # Training a dense FFN layer of the Mixtral size, forward and all gradients.
        _linear("linear_train_8192", 8192, 4096, 14336, "gelu", bias=True, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("norm", "balance", "linear", "linear"))
    if op == "norm":
        mode = rng.choice(("serve", "fp8", "train"))
        hidden = _log_int(rng, 1, 112) * 128 if mode == "fp8" else _log_int(rng, 64, 16384)
        if mode != "fp8" and rng.random() < 0.7:
            hidden = (hidden + 7) // 8 * 8
        c = _norm("", min(_log_int(rng, 1, 32768), 2**27 // hidden), hidden, mode, rng.choice(("bf16", "bf16", "fp32")), rng.random() < 0.7)
    elif op == "balance":
        experts = _log_int(rng, 2, 512)
        c = _balance("", min(_log_int(rng, 1, 65536), 2**23 // experts), experts, rng.randint(1, min(8, experts - 1)), rng.choice(("softmax", "sigmoid")), rng.random() < 0.7,
                     rng.choice((0.0, 0.1, 0.5)), rng.choice(("fp32", "fp32", "bf16")))
    else:
        activation = rng.choice(("none", "relu", "silu", "gelu", "swiglu"))
        inputs = _log_int(rng, 8, 1024) * 8
        outputs = _log_int(rng, 1, 32) * 256 if activation == "swiglu" else _log_int(rng, 8, 1024) * 8
        train = rng.random() < 0.4
        rows = min(_log_int(rng, 1, 8192), 2**38 // (inputs * outputs))
        c = _linear("", rows, inputs, outputs, activation, activation != "swiglu" and rng.random() < 0.5, activation != "swiglu" and rng.random() < 0.5, train)
    del c["name"]
    return c


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = case["rows"]
    s = {"case": case}
    if case["op"] == "norm":
        H, dt = case["hidden"], TYPES[case["dtype"]]
        train = case["mode"] == "train"
        s["x"] = _randn(g, T, H).to(dt).requires_grad_(train)
        # the stream grows with depth
        s["residual"] = _randn(g, T, H, std=3.0).to(dt).requires_grad_(train) if case["residual"] else None
        s["weight"] = (1.0 + _randn(g, H, std=0.1)).to(dt).requires_grad_(train)
        if train:
            s["dy"] = _randn(g, T, H).to(dt)
            s["dh"] = _randn(g, T, H).to(dt) if case["residual"] else None
    elif case["op"] == "balance":
        E, dt = case["experts"], TYPES[case["dtype"]]
        # popular experts and unpopular ones
        logits = (_randn(g, T, E) + _randn(g, E, std=0.5)).to(dt)
        s["topk_idx"] = logits.float().topk(case["k"], dim=-1).indices.to(torch.int32)
        s["logits"] = logits.requires_grad_(case["train"])
        s["mask"] = torch.rand(T, generator=g, device="cuda") >= case["padded"] if case["padded"] else None
        s["dloss"] = torch.rand((), generator=g, device="cuda") + 0.01
    else:
        N, K, train = case["outputs"], case["inputs"], case["train"]
        cols = N // 2 if case["activation"] == "swiglu" else N
        bf = torch.bfloat16
        s["x"] = _randn(g, T, K).to(bf).requires_grad_(train)
        s["weight"] = _randn(g, N, K, std=K**-0.5).to(bf).requires_grad_(train)
        s["bias"] = _randn(g, N, std=0.5).to(bf).requires_grad_(train) if case["bias"] else None
        s["residual"] = _randn(g, T, cols).to(bf).requires_grad_(train) if case["residual"] else None
        s["dy"] = _randn(g, T, cols).to(bf) if train else None
    return s


def run(s):
    return (_run_own if own else _run_plain)(s)


# ---- the framework's calls ------------------------------------------------------------------------------------------
def _run_own(s):
    from fast_b200.ops import fused

    case = s["case"]
    if case["op"] == "norm":
        quantise = case["mode"] == "fp8"
        r = fused.add_rms_norm(s["x"], s["weight"], EPS, residual=s["residual"], quantise=quantise)
        out = {"y": r.y}
        if s["residual"] is not None:
            out["h"] = r.h
        if quantise:
            out["q"] = fused.dequantise_rows(r.q, r.scales)
        if case["mode"] == "train":
            res = s["residual"] is not None
            grads = torch.autograd.grad([r.y, r.h] if res else [r.y], [s["x"], s["weight"]] + [s["residual"]] * res, [s["dy"], s["dh"]] if res else [s["dy"]])
            out.update(zip(("dx", "dweight", "dresidual"), grads))
        return out
    if case["op"] == "balance":
        loss, counts = fused.balance_loss(s["logits"], s["topk_idx"], mask=s["mask"], scores=case["scores"])
        out = {"loss": loss, "counts": counts}
        if case["train"]:
            out["dlogits"] = torch.autograd.grad(loss, s["logits"], s["dloss"])[0]
        return out
    y = fused.linear(s["x"], s["weight"], bias=s["bias"], activation=None if case["activation"] == "none" else case["activation"], residual=s["residual"])
    out = {"y": y}
    if case["train"]:
        leaves = {k: s[k] for k in ("x", "weight", "bias", "residual") if s[k] is not None}
        out.update(zip(("d" + k for k in leaves), torch.autograd.grad(y, list(leaves.values()), s["dy"])))
    return out


# ---- plain forms ------------------------------------------------------------------------------------------------------
def _quantised(y):
    """Rows of y through e4m3 and back. Per 128 columns the scale is the fp32 product of the largest magnitude and 1/448, rounded up to a bf16 value, and
    the numbers rounded to e4m3 are the fp32 products of y and 1/scale; their rounding, next to a border, in 64 bits."""
    b = y.float().view(y.shape[0], -1, 128)
    want = (b.abs().amax(-1, keepdim=True).clamp_min(1e-12) * (1.0 / 448.0)).double()
    step = torch.exp2(torch.floor(torch.log2(want)) - 7)          # distance of bf16 values there
    scale = torch.ceil(want / step) * step
    v = (b * (1.0 / scale.float())).double()
    ulp = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)   # of e4m3; below 2^-6 its values are evenly spaced
    return (torch.round(v / ulp) * ulp * scale).view(y.shape).to(torch.bfloat16)


@torch.no_grad()
def _run_plain(s):
    case = s["case"]
    if case["op"] == "norm":
        dt = s["x"].dtype
        h = s["x"].float()
        if s["residual"] is not None:
            h = (h + s["residual"].float()).to(dt).float()
        r = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
        w = s["weight"].float()
        y = (h * r * w).to(dt)
        out = {"y": y}
        if s["residual"] is not None:
            out["h"] = h.to(dt)
        if case["mode"] == "fp8":
            out["q"] = _quantised(y)
        if case["mode"] == "train":
            dy, hat = s["dy"].float(), h * r
            gw = dy * w
            dx = r * (gw - hat * (gw * hat).mean(-1, keepdim=True))
            if s["dh"] is not None:
                dx = dx + s["dh"].float()
            out["dx"], out["dweight"] = dx.to(dt), (dy * hat).sum(0).to(dt)
            if s["residual"] is not None:
                out["dresidual"] = out["dx"]
        return out
    if case["op"] == "balance":
        T, E = s["logits"].shape
        live = torch.ones(T, device="cuda") if s["mask"] is None else s["mask"].float()
        n = live.sum().clamp_min(1.0)
        counts = torch.zeros(E, device="cuda", dtype=torch.int32)
        weight = live.to(torch.int32).unsqueeze(1).expand_as(s["topk_idx"]).reshape(-1)
        counts.index_add_(0, s["topk_idx"].reshape(-1), weight)
        l = s["logits"].float()
        if case["scores"] == "softmax":
            e = torch.exp(l - l.amax(-1, keepdim=True))
            p = e / e.sum(-1, keepdim=True)
            slope = p
        else:
            sig = 1.0 / (1.0 + torch.exp(-l))
            total = sig.sum(-1, keepdim=True)
            p = sig / total
            slope = sig * (1.0 / (1.0 + torch.exp(l))) / total
        factor = E / (case["k"] * n * n)
        loss = factor * (counts.float() * (p * live.unsqueeze(1)).sum(0)).sum()
        out = {"loss": loss, "counts": counts}
        if case["train"]:
            # scores of a token sum to one, so counts may be taken relative to their mean: no cancellation of large numbers
            c = (counts.double() - counts.double().mean()).float()
            out["dlogits"] = (s["dloss"] * factor * live.unsqueeze(1) * slope * (c - (p * c).sum(-1, keepdim=True))).to(s["logits"].dtype)
        return out
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    act, slope, up = _activate(z, case["activation"])
    y = act if s["residual"] is None else act + s["residual"].float()
    out = {"y": y.to(torch.bfloat16)}
    if case["train"]:
        dy = s["dy"].float()
        if case["activation"] == "swiglu":
            dz = torch.stack([_tiles(dy * slope), _tiles(dy * up)], dim=2).reshape(z.shape)
        else:
            dz = dy * slope
        out["dx"], out["dweight"] = (dz @ w).to(torch.bfloat16), (dz.t() @ x).to(torch.bfloat16)
        if s["bias"] is not None:
            out["dbias"] = dz.sum(0).to(torch.bfloat16)
        if s["residual"] is not None:
            out["dresidual"] = s["dy"]
    return out


def _tiles(v):
    return v.reshape(v.shape[0], -1, 128)


def _activate(z, kind):
    """Value and slope of the activation of z; swiglu: value, slope towards the gate, slope towards the up half."""
    if kind == "none":
        return z, torch.ones_like(z), None
    if kind == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on, None
    if kind == "gelu":
        phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi)), None
    if kind == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        return z * sig, sig * (1.0 + z * (1.0 - sig)), None
    t = z.reshape(z.shape[0], -1, 2, 128)
    gate, up = t[:, :, 0].reshape(z.shape[0], -1), t[:, :, 1].reshape(z.shape[0], -1)
    sig = 1.0 / (1.0 + torch.exp(-gate))
    return gate * sig * up, up * sig * (1.0 + gate * (1.0 - sig)), gate * sig


def work(case):
    T = case["rows"]
    if case["op"] == "norm":
        H, b, res = case["hidden"], TYPES[case["dtype"]].itemsize, case["residual"]
        n = T * H
        fwd = n * b * (4 if res else 2) + H * b + (n + n // 128 * 4 if case["mode"] == "fp8" else 0)
        # backward: dy, dh and, again, what was normalised; dx and the weight's gradient
        bwd = n * b * (4 if res else 3) + H * b if case["mode"] == "train" else 0
        return {"bytes": fwd + bwd, "flops": n * (6 + (12 if case["mode"] == "train" else 0))}
    if case["op"] == "balance":
        E, b = case["experts"], TYPES[case["dtype"]].itemsize
        n = T * E
        mask = T if case["padded"] else 0
        return {"bytes": n * b * (3 if case["train"] else 1) + T * case["k"] * 4 + mask + E * 4 + 4, "flops": n * (6 + (10 if case["train"] else 0))}
    N, K = case["outputs"], case["inputs"]
    cols = N // 2 if case["activation"] == "swiglu" else N
    fwd = 2 * (T * K + N * K + T * cols * (2 if case["residual"] else 1) + (N if case["bias"] else 0))
    if not case["train"]:
        return {"bytes": fwd, "flops": 2 * T * N * K}
    # backward: dy, x, weight and what the activation was of; three gradients
    kept = T * N if case["activation"] != "none" else 0
    bwd = 2 * (T * cols + 2 * T * K + 2 * N * K + kept + (N if case["bias"] else 0))
    return {"bytes": fwd + 2 * kept + bwd, "flops": 6 * T * N * K}


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------------
def _to_type(v, like):
    return v.to(like.dtype).double()


def _e4m3_exact(y):
    """Nearest e4m3 number times its scale, by looking the neighbours up in a table of all of them. Scale and quotient are fp32 numbers by definition."""
    codes = torch.arange(127, device=y.device)
    exponent, mantissa = codes // 8, (codes % 8).double()
    table = torch.where(exponent == 0, mantissa / 8 * 2.0**-6, (1 + mantissa / 8) * torch.pow(2.0, (exponent - 7).double()))
    groups = y.unflatten(-1, (-1, 128))
    reciprocal = torch.tensor(1 / 448, dtype=torch.float32, device=y.device).double()
    largest = (torch.clamp(groups.abs().max(dim=-1, keepdim=True).values, min=1e-12) * reciprocal).float().double()
    fraction, power = torch.frexp(largest)
    scale = torch.ldexp(torch.ceil(fraction * 256) / 256, power)
    a = (groups.abs() * (1 / scale).float().double()).float().double()
    hi = torch.searchsorted(table, a.contiguous()).clamp(1, 126)
    below, above = table[hi - 1], table[hi]
    middle = (below + above) / 2
    take_above = (a > middle) | ((a == middle) & (hi % 2 == 0))   # a tie goes to the even code
    return (torch.where(take_above, above, below) * torch.sign(groups) * scale).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "norm":
        h = d["x"] if not case["residual"] else _to_type(d["x"] + d["residual"], s["x"])
        leaf_h, leaf_w = h.clone().requires_grad_(), d["weight"].clone().requires_grad_()
        y = leaf_h / torch.sqrt(leaf_h.pow(2).mean(dim=1, keepdim=True) + EPS) * leaf_w
        out = {"y": y.detach()}
        if case["residual"]:
            out["h"] = d["x"] + d["residual"]
        if case["mode"] == "fp8":
            out["q"] = _e4m3_exact(_to_type(y.detach(), s["x"]))
        if case["mode"] == "train":
            gh, gw = torch.autograd.grad(y, [leaf_h, leaf_w], d["dy"])
            out["dx"] = gh + d["dh"] if case["residual"] else gh
            out["dweight"] = gw
            if case["residual"]:
                out["dresidual"] = out["dx"]
        return out
    if case["op"] == "balance":
        leaf = d["logits"].clone().requires_grad_()
        p = torch.softmax(leaf, dim=1) if case["scores"] == "softmax" else torch.nn.functional.normalize(torch.sigmoid(leaf), p=1, dim=1)
        keep = slice(None) if s["mask"] is None else s["mask"]
        n = p[keep].shape[0]
        counts = torch.bincount(s["topk_idx"][keep].flatten().long(), minlength=case["experts"])
        share = counts.double() / max(case["k"] * n, 1)
        loss = case["experts"] * torch.dot(share, p[keep].sum(dim=0) / max(n, 1))
        out = {"loss": loss.detach(), "counts": counts.to(torch.int32)}
        if case["train"]:
            # a part of all counts that is the same for every expert has no gradient: taken out in whole numbers
            uneven = (counts * case["experts"] - counts.sum()).double() / (case["k"] * max(n, 1))
            out["dlogits"] = torch.autograd.grad(torch.dot(uneven, p[keep].sum(dim=0) / max(n, 1)), leaf, d["dloss"])[0]
        return out
    leaves = {k: d[k].clone().requires_grad_(case["train"]) for k in ("x", "weight", "bias", "residual") if k in d}
    z = torch.nn.functional.linear(leaves["x"], leaves["weight"], leaves.get("bias"))
    if case["activation"] == "swiglu":
        pairs = z.unflatten(1, (-1, 2, 128))
        y = (torch.nn.functional.silu(pairs[:, :, 0]) * pairs[:, :, 1]).flatten(1)
    else:
        y = {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[case["activation"]](z)
    if "residual" in leaves:
        y = y + leaves["residual"]
    out = {"y": y.detach()}
    if case["train"]:
        out.update(zip(("d" + k for k in leaves), torch.autograd.grad(y, list(leaves.values()), d["dy"])))
    return out
