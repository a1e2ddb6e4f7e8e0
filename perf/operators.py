"""Performance cases of the operators that apply decoded weights: ``rms_norm`` and ``matvec``.

A model's state dict, as this package decodes it, holds norm vectors and, where the model is microscaled, matrices of 4-bit
values with a scale per group: MXFP4 (an E8M0 scale per 32) and NVFP4 (an E4M3 scale per 16 and one fp32 scale).  ``op`` is

* ``norm``: the residual's addition, the root-mean-square norm and its weight, into the input's type (``quant`` "none") or into
  E4M3 with a fp32 scale per row ("row") or an E8M0 scale per 32 values ("block");
* ``norm_step``: the same into the input's type, with the gradients of x (which the residual shares) and of the weight;
* ``matvec``: products of one 4-bit matrix with a few or many tokens, which come in bf16, fp16, fp32, or in 8 bits with scales;
* ``matvec_step``: such a product and the gradient that goes back to the tokens;
* ``layer``: the norm in front of a feed-forward block with both matrices that read its 8-bit output.

Shapes are those of the Llama-3-8B layers the package is benchmarked on, and ragged ones.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-5
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _norm_case(name, op, rows, cols, dtype, quant, residual):
    return dict(name=name, op=op, rows=rows, cols=cols, dtype=dtype, quant=quant, residual=residual)


def _mat_case(name, op, tokens, n, k, kind, x):
    return dict(name=name, op=op, tokens=tokens, n=n, k=k, kind=kind, x=x)


def listed():
    return [
        # One token on its way into a block of an 8-bit pipeline: the smallest call, all latency.
        _norm_case("norm_token_block8", "norm", 1, 4096, "bf16", "block", True),
        # A long prompt, or a batch of them, into 8 bits with a scale per token.
        _norm_case("norm_8192_row8", "norm", 8192, 4096, "bf16", "row", True),
        # Rows of an odd length, which no wide load fits, without a residual.
        _norm_case("norm_ragged_row8", "norm", 333, 10501, "fp16", "row", False),
        # Fine-tuning: forward and backward over a batch of sequences.
        _norm_case("norm_step_4096", "norm_step", 4096, 4096, "bf16", "none", True),
        # Generating one token: an up or gate projection in MXFP4.
        _mat_case("matvec_token_mx", "matvec", 1, 14336, 4096, "mxfp4", "bf16"),
        # Generating one token: the down projection in NVFP4, rows much longer than they are many.
        _mat_case("matvec_token_nv", "matvec", 1, 4096, 14336, "nvfp4", "bf16"),
        # A key or value projection of one token whose norm wrote 8 bits: the smallest matrix.
        _mat_case("matvec_small_nv8", "matvec", 1, 1024, 4096, "nvfp4", "block8"),
        # A batch of sequences that generate together, activations in 8 bits with a scale per token.
        _mat_case("matvec_16_mx8", "matvec", 16, 4096, 4096, "mxfp4", "row8"),
        # A few drafted tokens in fp32, a matrix of ragged sizes whose rows end in half a pair of groups.
        _mat_case("matvec_ragged_fp32", "matvec", 5, 10501, 2992, "nvfp4", "fp32"),
        # A prompt of 512 tokens.
        _mat_case("matvec_512_mx", "matvec", 512, 14336, 4096, "mxfp4", "bf16"),
        # Training in front of frozen 4-bit weights: the product and the gradient of its input.
        _mat_case("matvec_step_nv", "matvec_step", 256, 14336, 4096, "nvfp4", "bf16"),
        # The way into a feed-forward block for two sequences: norm into 8 bits, then the gate and up projections.
        _mat_case("layer_2_mx", "layer", 2, 14336, 4096, "mxfp4", "bf16"),
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi], odd ones among them."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "norm", "norm_step", "matvec", "matvec", "matvec", "matvec", "matvec_step", "layer"))
    if op.startswith("norm"):
        quant = "none" if op == "norm_step" else rng.choice(("none", "row", "block"))
        cols = _log_int(rng, 64, 14336)
        cols = max(64, cols // 32 * 32) if quant == "block" else cols
        most = 8192 * 4096 if op == "norm" else 4096 * 4096
        rows = _log_int(rng, 1, min(8192, max(2, most // cols)))
        return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), quant=quant, residual=rng.random() < 0.7)
    kind = rng.choice(("mxfp4", "nvfp4"))
    group = 32 if kind == "mxfp4" else 16
    if op == "layer":
        k = max(256, _log_int(rng, 256, 4096) // 32 * 32)
        return dict(op=op, tokens=_log_int(rng, 1, 64), n=_log_int(rng, 256, 14336), k=k, kind=kind, x="bf16")
    n, k = _log_int(rng, 64, 14336), max(64, _log_int(rng, 64, 14336) // group * group)
    while n * k > 14336 * 4096:
        n, k = n // 2 + 1, max(64, k // 2 // group * group)
    tokens = _log_int(rng, 1, 512) if rng.random() < 0.6 else _log_int(rng, 1, 8)
    if op == "matvec_step":
        return dict(op=op, tokens=max(1, tokens // 2), n=n, k=k, kind=kind, x=rng.choice(("bf16", "bf16", "fp16", "fp32")))
    x = rng.choice(("bf16", "bf16", "fp16", "fp32", "row8", "block8"))
    if x == "block8":
        k = max(64, k // 32 * 32)
    return dict(op=op, tokens=tokens, n=n, k=k, kind=kind, x=x)


# ---- inputs -----------------------------------------------------------------------------------------
def _activations(rows, cols, g):
    """Values of a residual stream: normal, with a few channels that are some twenty times as large."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    return x * torch.where(torch.rand(cols, generator=g, device="cuda") < 0.003, 20.0, 1.0)


def _matrix(n, k, kind, g):
    """values [n, k/2], scales and the fp32 scale (or None) of normal weights with a sigma of its own for each row."""
    lo, hi = math.log(0.005), math.log(0.05)
    w = torch.randn(n, k, generator=g, device="cuda") * torch.exp(torch.rand(n, 1, generator=g, device="cuda") * (hi - lo) + lo)
    group, top = (32, None) if kind == "mxfp4" else (16, (w.abs().amax() / (448.0 * 6.0)).reshape(1))
    b = w.reshape(n, k // group, group)
    most = b.abs().amax(-1)
    if kind == "mxfp4":
        scales = (127 + torch.ceil(torch.log2(most.clamp_min(1e-30) / 6.0))).clamp(0, 254).to(torch.uint8)
        s = torch.exp2(scales.float() - 127)
    else:
        scales = (most / 6.0 / top).to(torch.float8_e4m3fn)
        s = scales.float() * top
    x = (b / torch.where(s == 0, torch.ones_like(s), s).unsqueeze(-1)).reshape(n, k)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")
    c = torch.bucketize(x.abs(), edges, out_int32=True).to(torch.uint8) | ((x < 0).to(torch.uint8) << 3)
    return c[:, 0::2] | (c[:, 1::2] << 4), scales, top


def _to_8_bits(x, how):
    """E4M3 values of x and their scales: fp32 per row, or powers of two per 32 values."""
    if how == "row8":
        s = x.abs().amax(-1, keepdim=True) / 448.0
        return (x / s).to(torch.float8_e4m3fn), s.reshape(-1)
    b = x.reshape(x.shape[0], -1, 32)
    e = torch.ceil(torch.log2(b.abs().amax(-1) / 448.0))
    return (b / torch.exp2(e).unsqueeze(-1)).reshape(x.shape).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op.startswith("norm"):
        rows, cols, dt = case["rows"], case["cols"], _DTYPES[case["dtype"]]
        state = {"op": op, "quant": case["quant"], "x": _activations(rows, cols, g).to(dt), "residual": _activations(rows, cols, g).to(dt) if case["residual"] else None,
                 "weight": (1 + 0.01 * torch.randn(cols, generator=g, device="cuda")).to(dt)}
        if op == "norm_step":
            state["dy"] = (torch.randn(rows, cols, generator=g, device="cuda") * 0.01).to(dt)
            state["dh"] = (torch.randn(rows, cols, generator=g, device="cuda") * 0.01).to(dt) if case["residual"] else None
            if own:
                for name in ("x", "residual", "weight"):
                    if state[name] is not None:
                        state[name].requires_grad_()
        return state
    tokens, n, k = case["tokens"], case["n"], case["k"]
    state = {"op": op, "kind": case["kind"], "w": [_matrix(n, k, case["kind"], g) for _ in range(2 if op == "layer" else 1)]}
    x = _activations(tokens, k, g)
    if case["x"] in _DTYPES:
        state["x"] = x.to(_DTYPES[case["x"]])
    else:
        state["x"], state["x_scales"] = _to_8_bits(x, case["x"])
    if op == "layer":
        state["residual"] = _activations(tokens, k, g).to(torch.bfloat16)
        state["weight"] = (1 + 0.01 * torch.randn(k, generator=g, device="cuda")).to(torch.bfloat16)
    if op == "matvec_step":
        state["dy"] = (torch.randn(tokens, n, generator=g, device="cuda") * 0.01).to(state["x"].dtype)
    if own:  # the handles a program keeps; they hold the tensors above
        import ptwm_b200
        state["handles"] = [ptwm_b200.ScaledWeight(*w) for w in state["w"]]
        if op == "matvec_step":
            state["x"].requires_grad_()
        if op == "layer":
            state["projection"] = ptwm_b200.Projection(state["weight"], state["handles"], eps=_EPS, quant="block")
        if "x_scales" in state:
            state["x"] = ptwm_b200.ScaledActivations(state["x"], state["x_scales"])
    return state


# ---- the plain forms -----------------------------------------------------------------------------------
def _plain_quantise(y, quant):
    """y in fp32 -> E4M3 values and scales."""
    if quant == "row":
        s = y.abs().amax(-1, keepdim=True) / 448.0
        q = torch.where(s > 0, y / s, torch.zeros_like(y)).clamp(-448.0, 448.0)
        return q.to(torch.float8_e4m3fn), s.reshape(-1)
    b = y.reshape(y.shape[0], -1, 32)
    m, p = torch.frexp(b.abs().amax(-1))  # in [0.5, 1), and the power of two
    e = (p - 9 + (m > 0.875).to(torch.int32)).clamp(-127, 127)
    e = torch.where(m > 0, e, torch.full_like(e, -127))
    q = (b.double() * torch.exp2(-e.double()).unsqueeze(-1)).float().clamp(-448.0, 448.0)
    return q.reshape(y.shape).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _plain_norm(x, residual, weight):
    """The sum with the residual, its inverse root mean square and the normed values, the last two in fp32."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    r = torch.rsqrt((h.float() * h.float()).mean(-1, keepdim=True) + _EPS)
    return h, r, h.float() * r * weight.float()


def _plain_matrix(values, scales, top):
    """The matrix in fp32."""
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=values.device)
    codes = torch.stack((values & 15, values >> 4), dim=-1).reshape(values.shape[0], -1)
    if top is None:
        s = torch.exp2(scales.double() - 127).float()
    else:
        s = scales.float() * top
    w = table[codes.int()]
    return (w.reshape(s.shape[0], s.shape[1], -1) * s.unsqueeze(-1)).reshape(w.shape)


def _plain_tokens(x, scales):
    if scales is None:
        return x.float()
    if scales.dtype == torch.float32:
        return x.float() * scales.unsqueeze(-1)
    s = torch.exp2(scales.view(torch.uint8).double() - 127).float()
    return (x.float().reshape(s.shape[0], s.shape[1], 32) * s.unsqueeze(-1)).reshape(x.shape)


def _run_plain(state):
    op, x = state["op"], state["x"]
    if op == "norm":
        h, _, y = _plain_norm(x, state["residual"], state["weight"])
        out = [y.to(x.dtype)] if state["quant"] == "none" else list(_plain_quantise(y, state["quant"]))
        return out + ([h] if state["residual"] is not None else [])
    if op == "norm_step":
        w, dy = state["weight"].float(), state["dy"].float()
        h, r, y = _plain_norm(x, state["residual"], state["weight"])
        hf, gw = h.float(), dy * w
        dx = r * gw - hf * (r * r * r * (gw * hf).mean(-1, keepdim=True))
        if state["dh"] is not None:
            dx = dx + state["dh"].float()
        dw = (dy * hf * r).sum(0)
        return [y.to(x.dtype), dx.to(x.dtype), dw.to(state["weight"].dtype)] + ([h] if state["dh"] is not None else [])
    if op == "layer":
        h, _, y = _plain_norm(x, state["residual"], state["weight"])
        q, s = _plain_quantise(y, "block")
        t = _plain_tokens(q, s)
        return [(t @ _plain_matrix(*w).t()).to(torch.bfloat16) for w in state["w"]] + [h]
    w = _plain_matrix(*state["w"][0])
    out = x.dtype if state.get("x_scales") is None else torch.bfloat16
    y = (_plain_tokens(x, state.get("x_scales")) @ w.t()).to(out)
    if op == "matvec":
        return [y]
    return [y, (state["dy"].float() @ w).to(out)]


# ---- the framework's calls -------------------------------------------------------------------------------
def _run_own(state):
    import ptwm_b200
    op, x = state["op"], state["x"]
    if op == "norm":
        quant = state["quant"]
        got = ptwm_b200.rms_norm(x, state["weight"], _EPS, residual=state["residual"], quant=None if quant == "none" else quant)
        y, more = got if state["residual"] is not None else (got, None)
        out = [y] if quant == "none" else [y.values, y.scales]
        return out + ([more] if more is not None else [])
    if op == "norm_step":
        leaves = [x, state["weight"]]
        if state["residual"] is None:
            y = ptwm_b200.rms_norm(x, state["weight"], _EPS)
            dx, dw = torch.autograd.grad(y, leaves, state["dy"])
            return [y, dx, dw]
        y, h = ptwm_b200.rms_norm(x, state["weight"], _EPS, residual=state["residual"])
        dx, dw, _ = torch.autograd.grad((y, h), leaves + [state["residual"]], (state["dy"], state["dh"]))
        return [y, dx, dw, h]
    if op == "layer":
        (gate, up), h = state["projection"](x, state["residual"])
        return [gate, up, h]
    y = ptwm_b200.matvec(x, state["handles"][0])
    if op == "matvec":
        return [y]
    return [y, torch.autograd.grad(y, x, state["dy"])[0]]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits -----------------------------------------------------------------------------
def _exact_codes(nibbles):
    """The number an E2M1 code stands for: a sign, two bits of exponent, one of mantissa."""
    c = nibbles.to(torch.int64)
    e, m = (c >> 1) & 3, (c & 1).double()
    size = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * (2.0 ** (e - 1).double()))
    return torch.where(c >= 8, -size, size)


def _exact_matrix(values, scales, top):
    n, half = values.shape
    w = torch.empty(n, 2 * half, dtype=torch.float64, device=values.device)
    w[:, 0::2], w[:, 1::2] = _exact_codes(values % 16), _exact_codes(values // 16)
    s = 2.0 ** (scales.double() - 127) if top is None else scales.double() * top.double()
    return w.mul_(s.repeat_interleave(2 * half // s.shape[1], dim=1))


def _exact_tokens(x, scales):
    if scales is None:
        return x.double()
    if scales.dtype == torch.float32:
        return x.double() * scales.double()[:, None]
    return x.double() * (2.0 ** (scales.view(torch.uint8).double() - 127)).repeat_interleave(32, dim=1)


def _exact_norm(state):
    x, h = state["x"], state["x"].double()
    if state["residual"] is not None:
        h = (h + state["residual"].double()).to(x.dtype).double()
    rms = ((h ** 2).sum(1, keepdim=True) / h.shape[1] + _EPS).sqrt()
    return h, rms, h / rms * state["weight"].double()


def _exact_8_bits(y, quant):
    if quant == "row":
        s = y.abs().max(1, keepdim=True).values / 448
        return (y / s).clamp(-448, 448).to(torch.float8_e4m3fn), s[:, 0]
    rows, cols = y.shape
    most = y.abs().reshape(rows, cols // 32, 32).max(-1).values
    e = torch.ceil(torch.log2(most / 448)).clamp(-127, 127)
    return (y * (2.0 ** -e).repeat_interleave(32, dim=1)).to(torch.float8_e4m3fn), 2.0 ** e


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    op = state["op"]
    if op == "norm":
        h, _, y = _exact_norm(state)
        out = [y] if state["quant"] == "none" else [v.double() for v in _exact_8_bits(y, state["quant"])]
        return out + ([h] if state["residual"] is not None else [])
    if op == "norm_step":
        h, rms, y = _exact_norm(state)
        dy, cols = state["dy"].double(), h.shape[1]
        unit = h / rms
        dunit = dy * state["weight"].double()
        dx = (dunit - unit * (dunit * unit).sum(1, keepdim=True) / cols) / rms
        if state["dh"] is not None:
            dx = dx + state["dh"].double()
        return [y, dx, (dy * unit).sum(0)] + ([h] if state["dh"] is not None else [])
    if op == "layer":
        h, _, y = _exact_norm(state)
        q, s = _exact_8_bits(y, "block")
        t = q.double() * s.repeat_interleave(32, dim=1)
        return [t @ _exact_matrix(*w).T for w in state["w"]] + [h]
    w = _exact_matrix(*state["w"][0])
    y = _exact_tokens(state["x"], state.get("x_scales")) @ w.T
    return [y] if op == "matvec" else [y, state["dy"].double() @ w]


# ---- what a pass cannot do without --------------------------------------------------------------------------
def work(case):
    """Inputs read once, outputs written once.  Norms: five operations a value, twelve for a step.  Products: two operations for
    each weight and token, twice that for a step."""
    op = case["op"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if op.startswith("norm"):
        rows, cols, b = case["rows"], case["cols"], size[case["dtype"]]
        values = rows * cols
        if op == "norm_step":  # x, residual, dy, dh in; y, h, dx, dw out
            return {"bytes": values * b * (7 if case["residual"] else 4) + 2 * cols * b, "flops": 12 * values}
        out = {"none": b, "row": 1 + 4 / cols, "block": 1 + 1 / 32}[case["quant"]]
        return {"bytes": values * (b * (3 if case["residual"] else 1) + out) + cols * b, "flops": 5 * values}
    m, n, k = case["tokens"], case["n"], case["k"]
    weights = n * k / 2 + (n * k / 32 if case["kind"] == "mxfp4" else n * k / 16 + 4)
    if op == "layer":
        return {"bytes": 2 * weights + 3 * 2 * m * k + 2 * k + 2 * 2 * m * n, "flops": 4 * m * n * k}
    x = size.get(case["x"], 1 + (1 / 32 if case["x"] == "block8" else 4 / k))
    out = size.get(case["x"], 2)
    if op == "matvec":
        return {"bytes": weights + m * k * x + m * n * out, "flops": 2 * m * n * k}
    return {"bytes": weights + 2 * m * k * x + 2 * m * n * out, "flops": 4 * m * n * k}
