"""Cases for the operators of the answer path: residual add + RMS norm (training, and with an 8-bit output), 4-bit block
scaled tables (quantisation and products) and sampling from scores.

`run` computes an operator in plain torch (`own = False`) or through the package's entry points (`own = True`) on what
`prepare` made.  Formats: "mx8" is e4m3 with one power-of-two scale (a byte, exponent + 127) per 32 values along the last
axis, "mx4" is e2m1 (two values per byte, the even one in the low half) with the same scales; the scale is the least power
of two 2^e, -126 <= e <= 127, with amax <= limit * 2^e (limit 448 / 6; 1 for a block of zeros).
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # a training step's last norm over the loss rows of a small batch: launches count
        {"name": "norm_train_small", "op": "norm_train", "rows": 1024, "d": 64, "dtype": "f32"},
        # every position of the benchmark's train batch (1024 sequences x 100 positions, hidden size 64)
        {"name": "norm_train_batch", "op": "norm_train", "rows": 102400, "d": 64, "dtype": "f32"},
        # a wide encoder in bf16, as long sequences in large batches give it
        {"name": "norm_train_wide", "op": "norm_train", "rows": 16384, "d": 4096, "dtype": "bf16"},
        # one new event of one user: the latency of a single row
        {"name": "norm_mx8_token", "op": "norm_mx8", "rows": 1, "d": 4096, "dtype": "bf16"},
        # a ragged serving batch whose width ends inside a block of 32
        {"name": "norm_mx8_ragged", "op": "norm_mx8", "rows": 8191, "d": 1000, "dtype": "f32"},
        # refreshing the 4-bit copy of the whole item table after a training step
        {"name": "quant_table", "op": "quant_mx4", "n": 4000001, "k": 64, "dtype": "f32"},
        # scoring one user against the whole item table
        {"name": "linear_catalogue_1", "op": "linear_mx4", "m": 1, "n": 4000001, "k": 64, "x": "f32"},
        # a small batch of users at the default hidden size 60, a quarter of the items
        {"name": "linear_catalogue_16", "op": "linear_mx4", "m": 16, "n": 1000003, "k": 60, "x": "bf16"},
        # a square layer for a batch of single tokens whose activations are in 8 bits
        {"name": "linear_layer_32", "op": "linear_mx4", "m": 32, "n": 8192, "k": 8192, "x": "mx8"},
        # one user, a pre-selected set of items, the usual short list: latency
        {"name": "sample_short", "op": "sample", "b": 1, "v": 50000, "draws": 1, "dtype": "f32", "temperature": 1.0,
         "top_k": 50, "top_p": 1.0, "min_p": 0.0, "spread": 3.0, "per_row": False},
        # a serving batch, every request with its own settings
        {"name": "sample_batch", "op": "sample", "b": 256, "v": 131072, "draws": 1, "dtype": "bf16", "temperature": 0.8,
         "top_k": 0, "top_p": 0.9, "min_p": 0.0, "spread": 3.0, "per_row": True},
        # a slate of 16 for each of four users over the whole item table
        {"name": "sample_catalogue", "op": "sample", "b": 4, "v": 4000001, "draws": 16, "dtype": "f32",
         "temperature": 1.0, "top_k": 1000, "top_p": 0.95, "min_p": 0.001, "spread": 2.0, "per_row": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_train", "norm_mx8", "quant_mx4", "linear_mx4", "linear_mx4", "sample", "sample"])
    if op in ("norm_train", "norm_mx8"):
        most = 1 << 26 if op == "norm_train" else 1 << 23
        d = _log_int(rng, 16, 8192)
        return {"op": op, "rows": _log_int(rng, 1, min(131072, most // d)), "d": d, "dtype": rng.choice(["f32", "bf16"])}
    if op == "quant_mx4":
        k = _log_int(rng, 16, 4096)
        return {"op": op, "n": _log_int(rng, 16, min(4000001, 256000064 // k)), "k": k, "dtype": rng.choice(["f32", "bf16"])}
    if op == "linear_mx4":
        m = _log_int(rng, 1, 64)
        if rng.random() < 0.5:                                    # scores of a table
            k = _log_int(rng, 16, 128)
            n = _log_int(rng, 1000, min(4000001, 16000048 // m, 256000064 // k))
        else:                                                     # a layer
            n, k = _log_int(rng, 200, 8192), _log_int(rng, 200, 8192)
            m = min(m, 32)
        return {"op": op, "m": m, "n": n, "k": k, "x": rng.choice(["f32", "bf16", "mx8"])}
    b = _log_int(rng, 1, 256)
    v = _log_int(rng, 100, min(4000001, 33554432 // b))
    kind = rng.randrange(4)
    return {"op": op, "b": b, "v": v, "draws": _log_int(rng, 1, 32), "dtype": rng.choice(["f32", "bf16"]),
            "temperature": round(rng.uniform(0.5, 1.5), 3),
            "top_k": _log_int(rng, 1, 2000) if kind in (0, 3) else 0,
            "top_p": round(rng.uniform(0.5, 0.99), 3) if kind in (1, 3) else 1.0,
            "min_p": round(rng.uniform(0.001, 0.2), 4) if kind in (2, 3) else 0.0,
            "spread": round(rng.uniform(1.0, 4.0), 2), "per_row": rng.random() < 0.5}


# ------------------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    op = case["op"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEVICE)

    if op in ("norm_train", "norm_mx8"):
        dt = DTYPES[case["dtype"]]
        rows, d = case["rows"], case["d"]
        st = {"op": op, "eps": 1e-6, "x": randn(rows, d).to(dt), "r": (2.0 * randn(rows, d)).to(dt),
              "w": 1.0 + 0.2 * randn(d)}
        if op == "norm_train":
            for key in ("x", "r", "w"):
                st[key].requires_grad_()
            st["dy"], st["ds"] = randn(rows, d).to(dt), randn(rows, d).to(dt)
        return st
    if op == "quant_mx4":
        return {"op": op, "table": (0.1 * randn(case["n"], case["k"])).to(DTYPES[case["dtype"]])}
    if op == "linear_mx4":
        codes, scales = _pack_mx4(*_blocks(0.1 * randn(case["n"], case["k"]), 6.0))
        st = {"op": op, "k": case["k"], "codes": codes, "scales": scales, "x_scales": None}
        x = randn(case["m"], case["k"])
        if case["x"] == "mx8":
            st["x"], st["x_scales"] = _pack_mx8(*_blocks(x, 448.0))
        else:
            st["x"] = x.to(DTYPES[case["x"]])
        return st
    b, v = case["b"], case["v"]
    st = {"op": op, "logits": (case["spread"] * randn(b, v)).to(DTYPES[case["dtype"]]),
          "u": torch.rand(b, case["draws"], generator=g, device=DEVICE, dtype=torch.float64)}
    for key in ("temperature", "top_k", "top_p", "min_p"):
        st[key] = case[key]
    if case["per_row"]:                                           # settings of the same kind, different in every row
        def vary():
            return torch.rand(b, generator=g, device=DEVICE)
        st["temperature"] = case["temperature"] * (0.75 + 0.5 * vary())
        st["top_k"] = (case["top_k"] * (0.5 + vary())).ceil().to(torch.int32)
        st["top_p"] = (case["top_p"] * (0.9 + 0.1 * vary()) if case["top_p"] < 1 else torch.ones(b, device=DEVICE))
        st["min_p"] = case["min_p"] * (0.5 + vary())
    return st


# -------------------------------------------------------------------------------------------------------------- plain
def _blocks(v, limit):
    """v (rows, k) -> (values (rows, blocks, 32) fp32 padded with zeros, exponents (rows, blocks) int32; 128: not finite)."""
    rows, k = v.shape
    v = v.float()
    if k % 32:
        v = torch.cat([v, v.new_zeros(rows, 32 - k % 32)], 1)
    v = v.view(rows, -1, 32)
    amax = v.abs().amax(2)
    mant, exp = torch.frexp(amax)                                 # amax = mant * 2^exp, 0.5 <= mant < 1
    limit_mant, limit_exp = math.frexp(limit)
    e = (exp - limit_exp + (mant > limit_mant).to(exp.dtype)).clamp(-126, 127)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    return v, torch.where(torch.isfinite(amax), e, torch.full_like(e, 128))


def _scaled(v, e):
    return torch.ldexp(v, -e.unsqueeze(2).to(v.dtype))


def _round_e2m1(v):
    """Nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code), |v| <= 6."""
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, v)


def _pack_mx4(v, e):
    q = _round_e2m1(_scaled(v, e))
    a = q.abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code + 8 * torch.signbit(q).to(torch.uint8)).flatten(1)
    return code[:, 0::2] + 16 * code[:, 1::2], (e + 127).to(torch.uint8)


def _pack_mx8(v, e):
    return _scaled(v, e).to(torch.float8_e4m3fn).flatten(1), (e + 127).to(torch.uint8)


def _unpack_mx4(codes, scales, dtype=torch.float32):
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=dtype, device=codes.device)
    grid = torch.cat([grid, -grid])
    q = torch.stack([grid[(codes & 15).int()], grid[(codes >> 4).int()]], 2).flatten(1)
    return torch.ldexp(q.view(*scales.shape, 32), (scales.to(dtype) - 127).unsqueeze(2)).flatten(1)


def _unpack_mx8(codes, scales, dtype=torch.float32):
    return torch.ldexp(codes.to(dtype).view(*scales.shape, 32), (scales.to(dtype) - 127).unsqueeze(2)).flatten(1)


def _plain_norm(x, r, w, eps):
    s = (x.float() + r.float()).to(x.dtype)
    s32 = s.float()
    rstd = torch.rsqrt(s32.square().mean(1, keepdim=True) + eps)
    return s, s32, rstd, s32 * rstd * w.float()


def _plain_norm_train(st):
    with torch.no_grad():
        x, w = st["x"], st["w"]
        s, s32, rstd, y = _plain_norm(x, st["r"], w, st["eps"])
        dy = st["dy"].float()
        g = dy * w
        ds = rstd * (g - s32 * rstd.square() * (g * s32).mean(1, keepdim=True)) + st["ds"].float()
        dw = (dy * s32 * rstd).sum(0)
        dx = ds.to(x.dtype)
        return {"y": y.to(x.dtype), "s": s, "dx": dx, "dr": dx, "dw": dw}


def _plain_sample(st):
    logits, u = st["logits"], st["u"]
    b, v = logits.shape

    def column(p):
        return p.double().unsqueeze(1) if isinstance(p, torch.Tensor) else torch.full((b, 1), float(p), dtype=torch.float64, device=logits.device)

    t, k, p, min_p = (column(st[key]) for key in ("temperature", "top_k", "top_p", "min_p"))
    ranked, order = torch.sort(logits, dim=1, descending=True, stable=True)
    ranked = ranked.double()
    w = torch.exp((ranked - ranked[:, :1]) / t)
    place = torch.arange(v, device=logits.device).unsqueeze(0)
    w = torch.where((k > 0) & (place >= k), 0.0, w)
    before = torch.cumsum(w, 1) - w
    keep = ((p >= 1) | (before < p * w.sum(1, keepdim=True))) & (w >= min_p)
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    upto = torch.cumsum(w, 1)
    ids = torch.searchsorted(upto, u * upto[:, -1:], right=True)
    return {"ids": ids, "probs": (w.gather(1, ids) / upto[:, -1:]).float()}


def _run_plain(st):
    op = st["op"]
    if op == "norm_train":
        return _plain_norm_train(st)
    if op == "norm_mx8":
        s, _, _, y = _plain_norm(st["x"], st["r"], st["w"], st["eps"])
        codes, scales = _pack_mx8(*_blocks(y, 448.0))
        return {"s": s, "values": _unpack_mx8(codes, scales)[:, :y.shape[1]].to(torch.bfloat16)}
    if op == "quant_mx4":
        codes, scales = _pack_mx4(*_blocks(st["table"], 6.0))
        return {"values": _unpack_mx4(codes, scales)[:, :st["table"].shape[1]].to(torch.bfloat16)}
    if op == "linear_mx4":
        x = st["x"].float() if st["x_scales"] is None else _unpack_mx8(st["x"], st["x_scales"])
        return {"out": x[:, :st["k"]] @ _unpack_mx4(st["codes"], st["scales"])[:, :st["k"]].t()}
    return _plain_sample(st)


# ---------------------------------------------------------------------------------------------------------------- own
def _run_own(st):
    from generative_recommenders_amd import enc_ops, mx_ops, ops
    op = st["op"]
    if op == "norm_train":
        y, s = enc_ops.add_rmsnorm(st["x"], st["r"], st["w"], st["eps"])
        dx, dr, dw = torch.autograd.grad((y, s), (st["x"], st["r"], st["w"]), (st["dy"], st["ds"]))
        return {"y": y, "s": s, "dx": dx, "dr": dr, "dw": dw}
    if op == "norm_mx8":
        codes, scales, s = mx_ops.add_rmsnorm_mx8(st["x"], st["r"], st["w"], st["eps"])
        return {"s": s, "values": mx_ops.dequantize_mx8(codes, scales, st["x"].shape[1])}
    if op == "quant_mx4":
        codes, scales = mx_ops.quantize_mx4(st["table"])
        return {"values": mx_ops.dequantize_mx4(codes, scales, st["table"].shape[1])}
    if op == "linear_mx4":
        return {"out": mx_ops.linear_mx4(st["x"], st["codes"], st["scales"], x_scales=st["x_scales"])}
    ids, probs = ops.sample_logits(st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"],
                                   top_p=st["top_p"], min_p=st["min_p"])
    return {"ids": ids, "probs": probs}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# --------------------------------------------------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op in ("norm_train", "norm_mx8"):
        size = 4 if case["dtype"] == "f32" else 2
        n = case["rows"] * case["d"]
        if op == "norm_train":      # x, r, dy, ds in; y, s and the one gradient of x and r out (s need not be read again)
            return {"bytes": 7 * n * size + 8 * case["d"], "flops": 16 * n}
        return {"bytes": n * (3 * size + 1 + 2) + n // 32 + 4 * case["d"], "flops": 8 * n}       # s, codes, scales, values
    if op == "quant_mx4":
        n = case["n"] * case["k"]
        return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + n // 2 + n // 32 + 2 * n, "flops": 4 * n}
    if op == "linear_mx4":
        m, n, k = case["m"], case["n"], case["k"]
        kp = -(-k // 32) * 32
        x = {"f32": 4 * k, "bf16": 2 * k, "mx8": kp + kp // 32}[case["x"]]
        return {"bytes": n * (kp // 2 + kp // 32) + m * x + 4 * m * n, "flops": 2 * m * n * k}
    n = case["b"] * case["v"]
    return {"bytes": n * (4 if case["dtype"] == "f32" else 2) + 20 * case["b"] * case["draws"], "flops": 4 * n}


# -------------------------------------------------------------------------------------------------------------- exact
# In 64 bits, element by element from the definitions, apart from the forms above.
def _least_exponent(amax, limit):
    """The least integer e in [-126, 127] with amax <= limit 2^e (0 where amax is 0)."""
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, 1.0) / limit))
    e = torch.where(torch.exp2(e) * limit < amax, e + 1, e)
    e = torch.where(torch.exp2(e - 1) * limit >= amax, e - 1, e)
    return torch.where(amax > 0, e.clamp(-126, 127), 0.0)


def _nearest(v, mantissa_bits, least):
    """v to `mantissa_bits` fractional bits of its own binade, binades below 2^least sharing its step."""
    binade = torch.floor(torch.log2(v.abs().clamp_min(2.0 ** least))).clamp_min(least)
    step = torch.exp2(binade - mantissa_bits)
    return torch.round(v / step) * step


def _exact_mx(v, limit, mantissa_bits, least):
    rows, k = v.shape
    padded = torch.zeros(rows, -(-k // 32) * 32, dtype=torch.float64, device=v.device)
    padded[:, :k] = v
    blocks = padded.view(rows, -1, 32)
    unit = torch.exp2(_least_exponent(blocks.abs().amax(2, keepdim=True), limit))
    return (_nearest(blocks / unit, mantissa_bits, least) * unit).view(rows, -1)[:, :k]


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        if op in ("norm_train", "norm_mx8"):
            x, r, w = st["x"].double(), st["r"].double(), st["w"].double()
            s = (x + r).to(st["x"].dtype).double()
            n = s / torch.sqrt((s * s).sum(1, keepdim=True) / s.shape[1] + st["eps"])
            if op == "norm_mx8":
                return {"s": s, "values": _exact_mx(n * w, 448.0, 3, -6)}
            dy, norm = st["dy"].double(), torch.sqrt((s * s).sum(1, keepdim=True) / s.shape[1] + st["eps"])
            dn = dy * w
            ds = (dn - n * (dn * n).sum(1, keepdim=True) / s.shape[1]) / norm + st["ds"].double()
            return {"y": n * w, "s": s, "dx": ds, "dr": ds, "dw": (dy * n).sum(0)}
        if op == "quant_mx4":
            return {"values": torch.cat([_exact_mx(t.double(), 6.0, 1, 0) for t in st["table"].split(500000)])}
        if op == "linear_mx4":
            x = st["x"].double() if st["x_scales"] is None else _unpack_mx8(st["x"], st["x_scales"], torch.float64)
            x = x[:, :case["k"]]
            rows = 500000
            parts = [_unpack_mx4(c, s, torch.float64)[:, :case["k"]] @ x.t()
                     for c, s in zip(st["codes"].split(rows), st["scales"].split(rows))]
            return {"out": torch.cat(parts).t()}
        probs = []
        for i in range(case["b"]):
            row = st["logits"][i].double()
            t, k, p, mp = (float(q[i]) if isinstance(q, torch.Tensor) else float(q)
                           for q in (st["temperature"], st["top_k"], st["top_p"], st["min_p"]))
            weight = torch.exp((row - row.max()) / t)
            by_rank = torch.argsort(-row, stable=True)
            if k > 0:
                by_rank = by_rank[:int(k)]
            sums = torch.cumsum(weight[by_rank], 0)
            if p < 1:                                             # the shortest prefix that holds the share p
                by_rank = by_rank[:int((sums < p * sums[-1]).sum()) + 1]
            by_rank = by_rank[weight[by_rank] >= mp]
            kept = torch.sort(by_rank).values
            sums = torch.cumsum(weight[kept], 0)
            at = kept[(sums.unsqueeze(0) <= st["u"][i].unsqueeze(1) * sums[-1]).sum(1)] if kept.numel() < 1 << 20 else \
                kept[torch.searchsorted(sums, st["u"][i] * sums[-1], right=True)]
            probs.append((weight[at] / sums[-1]))
        return {"ids": None, "probs": torch.stack(probs)}
