"""What is measured of the MXFP4 operators, and their plain forms.

The operators: ``mxfp4_quantize`` with ``mxfp4_dequantize`` (OCP microscaled
4-bit floats: e2m1 codes, one e8m0 scale for each 32 values along the
contraction), ``mxfp4_linear`` (the Block-ELL product of quantised rows and
tiles, and its differentiable form ``mxfp4_linear_ad``), ``mxfp4_swiglu_fwd``
(the gated feed-forward block for serving) and ``mxfp4_swiglu`` (the same
block in training: forward and straight-through backward).

A Block-ELL weight is ``values [R, K, B, B]`` (tiles ``[B_in, B_out]``) and
``cols [R, K]``, -1 for a dead slot: the logical weight is ``[R*B, C*B]``.
"""

import sys

import torch

own = False

BLOCK = 32


def listed():
    return [
        # one token's activations on the way into a quantised product: latency
        dict(name="quantize_one", op="quantize", T=1, d=4096, B=128, dtype="bf16"),
        # a prompt's hidden states at the widest d_ff of the configurations
        dict(name="quantize_prompt", op="quantize", T=8192, d=16384, B=128, dtype="bf16"),
        # an odd batch of fp32 states, a width that is an odd number of 64-wide tiles
        dict(name="quantize_ragged_f32", op="quantize", T=4001, d=2112, B=64, dtype="f32"),
        # decoding: the down projection of one token, residual added
        dict(name="linear_one", op="linear", T=1, d=16384, out=4096, B=128, K=32, dead=0, residual=True, dtype="bf16"),
        # a long prompt through the down projection
        dict(name="linear_long", op="linear", T=16384, d=16384, out=4096, B=128, K=32, dead=0, residual=True,
             dtype="bf16"),
        # quantisation-aware training of one projection: odd token count, pruned slots, gradients of x and tiles
        dict(name="linear_train", op="linear_train", T=2047, d=2048, out=8192, B=64, K=4, dead=9, residual=False,
             dtype="bf16"),
        # decoding one token through the whole block, large configuration
        dict(name="ffn_one", op="ffn", T=1, d=4096, F=16384, B=128, Kg=8, Kd=32, dead=0, residual=True),
        # a small serving batch on the loop configuration
        dict(name="ffn_batch", op="ffn", T=24, d=1024, F=4096, B=64, Kg=4, Kd=16, dead=0, residual=True),
        # a ragged prompt on the tile-64 configuration, some slots pruned
        dict(name="ffn_prompt", op="ffn", T=4133, d=2048, F=8192, B=64, Kg=4, Kd=16, dead=17, residual=True),
        # bulk prefill on the large configuration
        dict(name="ffn_long", op="ffn", T=32768, d=4096, F=16384, B=128, Kg=8, Kd=32, dead=0, residual=True),
        # a training step of the block on the loop configuration, one micro-batch with an odd length
        dict(name="train_small", op="train", T=777, d=1024, F=4096, B=64, Kg=4, Kd=16, dead=5, residual=True),
        # a training step on the large configuration
        dict(name="train_large", op="train", T=8192, d=4096, F=16384, B=128, Kg=8, Kd=32, dead=0, residual=True),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear_train", "ffn", "train"])
    B = rng.choice([64, 128])
    if op == "quantize":
        return dict(op=op, T=_log(rng, 1, 12000), d=B * rng.randint(1, 8192 // B), B=B, dtype=rng.choice(["bf16", "f32"]))
    C = rng.randint(2, 4096 // B)
    if op in ("linear", "linear_train"):
        R, K = rng.randint(1, 8192 // B), rng.randint(1, C)
        return dict(op=op, T=_log(rng, 1, 8000), d=C * B, out=R * B, B=B, K=K, dead=rng.choice([0, 1, R * K // 8]),
                    residual=rng.random() < 0.5, dtype="bf16" if op == "linear_train" else rng.choice(["bf16", "f32"]))
    R = rng.randint(2, 8192 // B)
    return dict(op=op, T=_log(rng, 1, 6000), d=C * B, F=R * B, B=B, Kg=rng.randint(1, max(1, C // 2)),
                Kd=rng.randint(1, max(1, R // 2)), dead=rng.choice([0, 1, R]), residual=rng.random() < 0.5)


# ------------------------------------------------------------------- inputs


def _package():
    if "looped-blockell-tpu_b200" not in sys.path:
        sys.path.insert(0, "looped-blockell-tpu_b200")
    from looped_blockell import kernels
    return kernels


def _activations(g, T, d, dtype):
    """N(0, 1) hidden states with a few strong channels, as transformers have them."""
    strong = torch.where(torch.rand(d, generator=g, device="cuda") < 0.01, 8.0, 1.0)
    x = torch.randn(T, d, generator=g, device="cuda") * strong
    return x.to(torch.bfloat16 if dtype == "bf16" else torch.float32)


def _ell(g, R, C, K, B, dead):
    """Random tiles N(0, 0.02^2) in bf16 and their sorted distinct columns, `dead` slots pruned."""
    cols = torch.sort(torch.topk(torch.rand(R, C, generator=g, device="cuda"), K, dim=1).indices, dim=1).values
    if dead:
        at = torch.randint(R * K, (dead,), generator=g, device="cuda")
        cols.view(-1)[at] = -1
    values = torch.randn(R, K, B, B, generator=g, device="cuda") * 0.02
    return values.to(torch.bfloat16), cols.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, B, d = case["op"], case["B"], case["d"]
    s = dict(case)
    s["x"] = _activations(g, case["T"], d, case.get("dtype", "bf16"))
    if op in ("linear", "linear_train"):
        s["w"] = _ell(g, case["out"] // B, d // B, case["K"], B, case["dead"])
        s["res"] = _activations(g, case["T"], case["out"], case["dtype"]) if case["residual"] else None
        s["dy"] = _activations(g, case["T"], case["out"], "bf16") if op == "linear_train" else None
    if op in ("ffn", "train"):
        F = case["F"]
        s["gate"] = _ell(g, F // B, d // B, case["Kg"], B, case["dead"])
        s["up"] = _ell(g, F // B, d // B, case["Kg"], B, case["dead"])
        s["down"] = _ell(g, d // B, F // B, case["Kd"], B, case["dead"])
        s["dy"] = _activations(g, case["T"], d, "bf16") if op == "train" else None
    if op in ("linear", "ffn"):  # a server keeps its weights quantised: packed for the kernels, or as plain fp32 values
        pack = _package().make_mxfp4 if own else _dense_quantized
        for name, C in (("w", d // B), ("gate", d // B), ("up", d // B), ("down", case.get("F", 0) // B)):
            if name in s:
                s[name] = pack(*s[name], C)
    if op in ("linear_train", "train") and own:  # leaves of the user's graph
        s["x"].requires_grad_(True)
        for name in ("w", "gate", "up", "down"):
            if name in s:
                s[name][0].requires_grad_(True)
    return s


# --------------------------------------------------------------- plain form


def _quantized(v):
    """The fp32 values that MXFP4 holds for v, along its last axis."""
    b = v.float().reshape(*v.shape[:-1], -1, BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    byte = ((top.view(torch.int32) >> 23) - 2).clamp(min=0)  # biased exponent of the scale, 2^-127 for 0
    inverse = ((254 - byte) << 23).view(torch.float32)
    m = (b * inverse).abs()
    code = (0.5 * (m > 0.25) + 0.5 * (m >= 0.75) + 0.5 * (m > 1.25) + 0.5 * (m >= 1.75) + (m > 2.5).float()
            + (m >= 3.5).float() + 2.0 * (m > 5.0))
    scale = torch.where(byte > 0, byte << 23, 0x00400000).view(torch.float32)
    q = torch.copysign(code, b) * scale
    return torch.where(torch.isfinite(top), q, float("nan")).reshape(v.shape)


def _dense(values, cols, C):
    """fp32 [R*B, C*B] of the live tiles."""
    R, K, B, _ = values.shape
    blocks = torch.zeros(R, C + 1, B, B, device=values.device)
    rows = torch.arange(R, device=values.device)[:, None].expand(R, K)
    blocks[rows, torch.where(cols >= 0, cols, C).long()] = values.float()  # [B_in, B_out]; dead slots in column C
    return blocks[:, :C].permute(0, 3, 1, 2).reshape(R * B, C * B)


def _quantized_tiles(values):
    return _quantized(values.transpose(-1, -2)).transpose(-1, -2)


def _dense_quantized(values, cols, C):
    return _dense(_quantized_tiles(values), cols, C)


def _tiles(dense, cols, B):
    """The tiles [B_in, B_out] of a dense [R*B, C*B] at cols, zeros in dead slots."""
    R, K = cols.shape
    blocks = dense.reshape(R, B, -1, B).permute(0, 2, 3, 1)
    rows = torch.arange(R, device=cols.device)[:, None]
    return blocks[rows, cols.clamp(min=0).long()] * (cols >= 0)[:, :, None, None]


def _plain_linear(x, w, res):
    y = _quantized(x) @ w.T
    return y if res is None else y + res.float()


def _plain_train(s):
    B, d, F = s["B"], s["d"], s["F"]
    (vg, cg), (vu, cu), (vd, cd) = s["gate"], s["up"], s["down"]
    wg, wu, wd = _dense_quantized(vg, cg, d // B), _dense_quantized(vu, cu, d // B), _dense_quantized(vd, cd, F // B)
    x, dy = _quantized(s["x"]), s["dy"].float()
    g, u = x @ wg.T, x @ wu.T
    sig = 1 / (1 + torch.exp(-g))
    h = _quantized(g * sig * u)
    y = h @ wd.T
    dh = dy @ wd
    du = dh * (g * sig)
    dg = dh * u * (sig * (1 + g * (1 - sig)))
    dx = dg @ wg + du @ wu
    if s["residual"]:
        y, dx = y + s["x"].float(), dx + dy
    grads = _tiles(dg.T @ x, cg, B), _tiles(du.T @ x, cu, B), _tiles(dy.T @ h, cd, B)
    return dict(zip(("out", "dx", "dgate", "dup", "ddown"), (t.to(torch.bfloat16) for t in (y, dx, *grads))))


def _plain(s):
    op, x = s["op"], s["x"]
    if op == "quantize":
        return _quantized(x).to(x.dtype)
    if op == "linear":
        return _plain_linear(x, s["w"], s["res"]).to(x.dtype)
    if op == "linear_train":
        values, cols = s["w"]
        w, dy = _dense_quantized(values, cols, s["d"] // s["B"]), s["dy"].float()
        out = dict(out=_plain_linear(x, w, s["res"]), dx=dy @ w, dw=_tiles(dy.T @ _quantized(x), cols, s["B"]))
        return {k: v.to(torch.bfloat16) for k, v in out.items()}
    if op == "ffn":
        g, u = _plain_linear(x, s["gate"], None), _plain_linear(x, s["up"], None)
        return _plain_linear(g / (1 + torch.exp(-g)) * u, s["down"], x if s["residual"] else None).to(x.dtype)
    return _plain_train(s)


# ---------------------------------------------------------------------- run


def _own(s):
    K, op, x = _package(), s["op"], s["x"]
    if op == "quantize":
        return K.mxfp4_dequantize(K.mxfp4_quantize(x, tile=s["B"]), dtype=x.dtype)
    if op == "linear":
        return K.mxfp4_linear(x, s["w"], residual=s["res"])
    if op == "ffn":
        return K.mxfp4_swiglu_fwd(x, s["gate"], s["up"], s["down"], add_residual=s["residual"])
    if op == "linear_train":
        values, cols = s["w"]
        y = K.mxfp4_linear_ad(x, values, cols, residual=s["res"])
        dx, dw = torch.autograd.grad(y, (x, values), s["dy"])
        return dict(out=y, dx=dx, dw=dw)
    (vg, cg), (vu, cu), (vd, cd) = s["gate"], s["up"], s["down"]
    y = K.mxfp4_swiglu(x, vg, cg, vu, cu, vd, cd, add_residual=s["residual"])
    grads = torch.autograd.grad(y, (x, vg, vu, vd), s["dy"])
    return dict(zip(("out", "dx", "dgate", "dup", "ddown"), (y, *grads)))


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------- work


def work(case):
    T, d, B, op = case["T"], case["d"], case["B"], case["op"]
    e = 4 if case.get("dtype") == "f32" else 2
    q = 0.5 + 1 / BLOCK  # bytes of a quantised value with its share of the scale
    if op == "quantize":
        return {"bytes": 2 * e * T * d, "flops": 4 * T * d}
    if op in ("linear", "linear_train"):
        out, live = case["out"], case["out"] // B * case["K"] * B * B
        if op == "linear":
            return {"bytes": e * T * (d + (2 if case["residual"] else 1) * out) + q * live, "flops": 2 * T * live}
        # x, residual, dy and the tiles in; y, dx and the tiles' gradient out
        return {"bytes": 2 * (T * (2 * d + (3 if case["residual"] else 2) * out) + 2 * live), "flops": 6 * T * live}
    live = B * B * (2 * (case["F"] // B) * case["Kg"] + (d // B) * case["Kd"])
    if op == "ffn":
        return {"bytes": 4 * T * d + q * live, "flops": 2 * T * live}
    return {"bytes": 8 * T * d + 4 * live, "flops": 6 * T * live}


# -------------------------------------------------------------------- exact


def _exact_quantized(v):
    """MXFP4 by its definition in 64 bits: exponents from frexp, rounding half to even on the e2m1 step."""
    v = v.double()
    b = v.reshape(*v.shape[:-1], v.shape[-1] // BLOCK, BLOCK)
    top = b.abs().max(dim=-1, keepdim=True).values
    powers = torch.tensor([2.0 ** k for k in range(-140, 141)], dtype=torch.float64, device=v.device)
    E = torch.where(top > 0, torch.frexp(top).exponent.long() - 3, -127).clamp(-127, 127)
    r = b / powers[E + 140]
    step = powers[(torch.frexp(r.abs()).exponent.long() - 1).clamp(0, 2) - 1 + 140]
    return ((r / step).round() * step).clamp(-6.0, 6.0).mul(powers[E + 140]).reshape(v.shape)


def _exact_weight(values, cols, C):
    R, K, B, _ = values.shape
    q = _exact_quantized(values.mT.contiguous())  # [R, K, B_out, B_in]
    w = torch.zeros(R * B, C * B, dtype=torch.float64, device=values.device)
    for r, row in enumerate(cols.tolist()):
        for k, c in enumerate(row):
            if c >= 0:
                w[r * B:(r + 1) * B, c * B:(c + 1) * B] = q[r, k]
    return w


def _exact_tile_grads(dense, cols, B):
    out = torch.zeros(*cols.shape, B, B, dtype=torch.float64, device=cols.device)
    for r, row in enumerate(cols.tolist()):
        for k, c in enumerate(row):
            if c >= 0:
                out[r, k] = dense[r * B:(r + 1) * B, c * B:(c + 1) * B].mT
    return out


def exact(case, seed):
    global own
    kept, own = own, False
    try:  # the inputs as they were made; weights before any layout
        s = prepare(dict(case, op={"linear": "linear_train", "ffn": "train"}.get(case["op"], case["op"])), seed)
    finally:
        own = kept
    op, B, d = case["op"], case["B"], case["d"]
    x = _exact_quantized(s["x"])
    if op == "quantize":
        return x
    if op in ("linear", "linear_train"):
        w = _exact_weight(*s["w"], d // B)
        y = torch.matmul(x, w.mT)
        if case["residual"]:
            y = y + s["res"].double()
        if op == "linear":
            return y
        dy = s["dy"].double()
        return dict(out=y, dx=torch.matmul(dy, w), dw=_exact_tile_grads(torch.matmul(dy.mT, x), s["w"][1], B))
    wg, wu, wd = (_exact_weight(*s[n], C) for n, C in (("gate", d // B), ("up", d // B), ("down", case["F"] // B)))
    g, u = torch.matmul(x, wg.mT), torch.matmul(x, wu.mT)
    sig = torch.sigmoid(g)
    h = _exact_quantized(g * sig * u)
    y = torch.matmul(h, wd.mT)
    if case["residual"]:
        y = y + s["x"].double()
    if op == "ffn":
        return y
    dy = s["dy"].double()
    dh = torch.matmul(dy, wd)
    du, dg = dh * g * sig, dh * u * (sig + g * sig * (1 - sig))
    dx = torch.matmul(dg, wg) + torch.matmul(du, wu)
    if case["residual"]:
        dx = dx + dy
    grads = (_exact_tile_grads(torch.matmul(t.mT, a), s[n][1], B) for t, a, n in ((dg, x, "gate"), (du, x, "up"), (dy, h, "down")))
    return dict(zip(("out", "dx", "dgate", "dup", "ddown"), (y, dx, *grads)))
