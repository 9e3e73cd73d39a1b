"""Microscaled 4-bit floating point (MXFP4) around the attention, as measurable cases.

* ``quantize``       a tensor to MXFP4 and back: 4-bit codes (e2m1) with a power-of-two scale for 32 columns
* ``modulate``       RMS norm before a block with its modulation, ``xhat * w * (1 + scale)``, to MXFP4
* ``gate_modulate``  the norm after one half of a block, gated, onto the residual, and the norm before the next
  half to MXFP4
* ``linear``         ``act(x W^T + b) + r`` with ``W`` in MXFP4 and ``x`` quantized to it in the call

MXFP4 of a row: its columns in blocks of 32.  With ``amax`` the largest magnitude of a block its scale is
``2^(floor(log2 amax) - 2)`` (at least ``2^-127``), and a column becomes the nearest of ``+-{0, .5, 1, 1.5, 2, 3,
4, 6}`` times the scale, ties to the even code, what is past 6 to 6.  Codes are held two a byte, the even column
in the low half, rows padded to 256 columns; scales as ``[columns / 256, rows, 8]`` exponents biased by 127.

``train`` cases of the linear layer run it and the gradients of ``x``, the bias and the residual; the gradient
passes the rounding of ``x`` as if it were the identity, the weight is frozen.  Outputs in MXFP4 are returned as the
values they stand for.  Channels are the package's 30 heads of 128 and smaller or odd widths.
"""

import math

import torch

own = False

_EPS = 1e-5
_WIDTH = 30 * 128  # channels of the package's model shape
_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _quantize(M, K, dtype="bf16"):
    return dict(op="quantize", M=M, K=K, dtype=dtype)


def _norm(op, B, N, C, segments="", pad=0, dtype="bf16", params="bf16"):
    """``pad``: tokens of no document behind the last segment."""
    return dict(op=op, B=B, N=N, C=C, segments=segments, pad=pad, dtype=dtype, params=params)


def _linear(M, K, N, act="none", bias=False, residual=False, dtype="bf16", train=False):
    """``N``: columns of the output; a swiglu weight has two rows for each."""
    return dict(op="linear", M=M, K=K, N=N, act=act, bias=bias, residual=residual, dtype=dtype, train=train)


def listed():
    named = {
        # one row, a pooled conditioning vector: latency of the two calls
        "quantize_row": _quantize(1, _WIDTH),
        # a weight or activation of odd width, half precision
        "quantize_odd": _quantize(1337, 1001, dtype="fp16"),
        # four 1024x1024 samples (the largest memory-bound pass)
        "quantize_ktuple": _quantize(4 * 4352, _WIDTH),
        # the padded caption tokens of one prompt in the caption refiner: latency
        "modulate_caption": _norm("modulate", 1, 32, _WIDTH),
        # sampling on the packed mixed-resolution batch, a timestep per image, before the QKV projection
        "modulate_packed": _norm("modulate", 1, 6912, _WIDTH, segments="1280,1216,4416"),
        # one 1280x832 image between attention and feed-forward
        "gate_modulate_dit1280": _norm("gate_modulate", 1, 4416, _WIDTH),
        # conditioning rows of a pair of samples: few rows, every weight read once
        "linear_conditioning": _linear(2, 256, 4 * _WIDTH, bias=True),
        # the QKV projection of one prompt's caption tokens
        "linear_caption": _linear(32, _WIDTH, 3 * _WIDTH),
        # the feed-forward's gated up-projection of one 1280x832 image (hidden of 8/3 of the width; the largest)
        "linear_swiglu_dit1280": _linear(4416, _WIDTH, _WIDTH * 8 // 3, act="swiglu"),
        # the feed-forward's down-projection of one 512x512 image, onto the residual
        "linear_down_dit512": _linear(1280, _WIDTH * 8 // 3, _WIDTH, bias=True, residual=True),
        # adapters trained over the frozen QKV projection on one 1280x832 image
        "linear_qkv_train": _linear(4416, _WIDTH, 3 * _WIDTH, bias=True, train=True),
        # the same over a small odd head, half precision
        "linear_odd_train": _linear(667, 1001, 779, act="silu", bias=True, residual=True, dtype="fp16", train=True),
    }
    return [dict(c, name=name) for name, c in named.items()]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """The same operators over the range of sizes: 1 to 6912 tokens, 64 to 10240 channels, odd ones among them."""
    width = rng.choice([_log_int(rng, 64, 4200), 8 * _log_int(rng, 8, 525), 1024, 1536, 2048, _WIDTH, _WIDTH])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kind = rng.random()
    if kind < 0.2:
        return _quantize(_log_int(rng, 1, 4 * 4352), width, dtype)
    if kind < 0.5:
        n, b = _log_int(rng, 1, 6912), rng.choice([1, 1, 2, 4])
        c = _norm(rng.choice(["modulate", "gate_modulate"]), b, n, width, dtype=dtype,
                  params=rng.choice([dtype, "fp32"]))
        if n >= 16 and rng.random() < 0.5:
            pad = rng.choice([0, n % 13])
            cuts = [0] + sorted(rng.sample(range(1, n - pad), rng.choice([1, 2, 3]))) + [n - pad]
            c.update(pad=pad, segments=",".join(str(y - x) for x, y in zip(cuts, cuts[1:])))
        while work(c)["bytes"] > 4 * 4352 * _WIDTH * 5:
            c["B"] //= 2
        return c
    m = _log_int(rng, 1, 6912)
    n = rng.choice([16, _log_int(rng, 64, 4200), 8 * _log_int(rng, 8, 1280), _WIDTH, 3 * _WIDTH, _WIDTH * 8 // 3])
    k = rng.choice([256, width, width, width, _WIDTH * 8 // 3])
    c = _linear(m, k, n, act=rng.choice(["none", "none", "silu", "gelu", "swiglu"]), bias=rng.random() < 0.5,
                residual=rng.random() < 0.5, dtype=dtype, train=rng.random() < 0.4)
    while work(c)["flops"] > 4 * 4416 * _WIDTH * 3 * _WIDTH:
        c["M"] //= 2
    return c


def _held(rows, cols):
    """Bytes of MXFP4 rows: codes and scales."""
    blocks = rows * -(-cols // 32)
    return rows * cols / 2 + blocks


def work(case):
    if case["op"] == "quantize":  # both calls: the values read and written, the codes written and read
        n = case["M"] * case["K"]
        return {"bytes": 4 * n + 2 * _held(case["M"], case["K"]), "flops": 4 * n}
    if case["op"] == "linear":
        m, k, n, train = case["M"], case["K"], case["N"], case["train"]
        rows = 2 * n if case["act"] == "swiglu" else n
        nbytes = 2 * (m * k + m * n + (m * n if case["residual"] else 0) + (rows if case["bias"] else 0))
        nbytes += _held(rows, k)
        if train:  # dout in; dx, db out (the residual's gradient is dout)
            nbytes += 2 * (m * n + m * k + (rows if case["bias"] else 0))
        return {"bytes": nbytes, "flops": (4 if train else 2) * m * k * rows}
    # the norm, and its values back from MXFP4
    tokens = case["B"] * case["N"]
    each = tokens * case["C"] * 2
    tensors = 2 if case["op"] == "modulate" else 4
    return {"bytes": tensors * each + 2 * _held(tokens, case["C"]),
            "flops": tokens * case["C"] * (9 if case["op"] == "modulate" else 14)}


# ---------------------------------------------------------------- MXFP4 in elementary operations

_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _power(e):
    """2^(e - 127) of biased exponents, exactly; NaN of 255."""
    bits = torch.where(e == 0, 0x00400000, torch.where(e == 255, 0x7FC00000, e << 23))
    return bits.to(torch.int32).view(torch.float32)


def _blocks(x):
    """The exponents [rows, blocks] of rows of fp32 or fp64 values, and the codes' values [rows, blocks, 32]."""
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % 32)).unflatten(-1, (-1, 32))
    amax = x.abs().amax(-1)
    e = torch.clamp(torch.frexp(amax)[1] - 1 - 2 + 127, 0, 254)
    e = torch.where(amax == 0, 0, torch.where(torch.isfinite(amax), e, 255))
    v = x * _power(torch.where(e == 255, 127, 254 - e))[..., None].to(x.dtype)  # 254 - e: the reciprocal
    mag = v.abs()
    step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0)).to(x.dtype)
    mag = torch.clamp(torch.round(mag / step) * step, max=6.0)  # round: halves to even
    return e, torch.where(e[..., None] == 255, 0, torch.copysign(mag, v))


def _values(x, dtype):
    """What MXFP4 makes of rows of values, in their places."""
    e, v = _blocks(x)
    return (v * _power(e)[..., None].to(v.dtype)).flatten(-2)[..., :x.shape[-1]].to(dtype)


def _encode(w):
    """Codes [rows, columns / 2] and scales [columns / 256, rows, 8] of rows of fp32 values."""
    rows = w.shape[0]
    e, v = _blocks(torch.nn.functional.pad(w, (0, -w.shape[1] % 256)))
    table = torch.tensor(_VALUES, device=w.device)
    code = torch.searchsorted(table, v.abs().contiguous()).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    code = code.reshape(rows, -1, 2)
    return code[..., 0] | (code[..., 1] << 4), e.to(torch.uint8).reshape(rows, -1, 8).transpose(0, 1).contiguous()


def _decode(codes, scales, columns):
    """The fp32 values [rows, columns] of codes and scales."""
    rows = codes.shape[0]
    table = torch.tensor(_VALUES + [-x for x in _VALUES], device=codes.device)
    v = table[torch.stack([codes & 15, codes >> 4], -1).reshape(rows, -1, 32).int()]
    return (v * _power(scales.transpose(0, 1).reshape(rows, -1).int())[..., None]).reshape(rows, -1)[:, :columns]


# ---------------------------------------------------------------- inputs

def _doc_ids(case, device):
    lengths = [int(x) for x in case["segments"].split(",")]
    ids = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
    ids = torch.cat([ids, torch.full((case["pad"],), -1)])
    return ids.to(torch.int32).expand(case["B"], case["N"]).contiguous().to(device)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    dtype = _DTYPE[case["dtype"]]
    s = {"case": case, "leaves": []}
    if case["op"] == "quantize":
        # channels of unlike size, as a block's activations have them
        s["x"] = (normal(case["M"], case["K"]) * torch.exp(normal(case["K"]))).to(dtype)
    elif case["op"] == "linear":
        m, k, n = case["M"], case["K"], case["N"]
        rows = 2 * n if case["act"] == "swiglu" else n
        s["x"] = normal(m, k).to(dtype)
        s["codes"], s["scales"] = _encode(normal(rows, k) / math.sqrt(k))
        s["bias"] = (0.3 * normal(rows)).to(dtype) if case["bias"] else None
        s["residual"] = normal(m, n).to(dtype) if case["residual"] else None
        if case["train"]:
            s["dout"] = normal(m, n).to(dtype)
            s["leaves"] = [name for name in ("x", "bias", "residual") if s[name] is not None]
            for name in s["leaves"]:
                s[name].requires_grad_()
    else:
        B, N, C, params = case["B"], case["N"], case["C"], _DTYPE[case["params"]]
        s["doc_ids"] = _doc_ids(case, device) if case["segments"] else None
        docs = (len(case["segments"].split(",")),) if case["segments"] else ()
        s["x"] = (1.5 * normal(B, N, C)).to(dtype)
        s["weight"] = (1 + 0.2 * normal(C)).to(params)
        # scale and gate of both halves of a block, from one projection
        scale, gate, scale2, _ = (0.4 * normal(B, *docs, 4 * C)).to(params).chunk(4, dim=-1)
        if case["op"] == "modulate":
            s["scale"] = scale
        else:
            s["residual"] = (2 * normal(B, N, C)).to(dtype)
            s["gate"] = gate
            s["next_weight"] = (1 + 0.2 * normal(C)).to(params)
            s["next_scale"] = scale2
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    if own:
        return _framework(state)
    with torch.no_grad():
        op = state["case"]["op"]
        if op == "quantize":
            return {"values": _values(state["x"].float(), state["x"].dtype)}
        return _plain_linear(state) if op == "linear" else _plain_norm(state)


def _framework(s):
    import futudiffu_amd as F
    op = s["case"]["op"]
    if op == "quantize":
        return {"values": F.mxfp4_dequantize(F.mxfp4_quantize(s["x"]), dtype=s["x"].dtype)}
    if op == "modulate":
        q = F.rms_norm_modulate_mxfp4(s["x"], s["weight"], s["scale"], doc_ids=s["doc_ids"], eps=_EPS)
        return {"out": F.mxfp4_dequantize(q, dtype=s["x"].dtype)}
    if op == "gate_modulate":
        hidden, q = F.rms_norm_gate_residual_modulate_mxfp4(
            s["residual"], s["x"], s["weight"], s["gate"], s["next_weight"], s["next_scale"], doc_ids=s["doc_ids"],
            eps=_EPS)
        return {"out": F.mxfp4_dequantize(q, dtype=s["x"].dtype), "hidden": hidden}
    weight = F.MXFP4(s["codes"], s["scales"], s["case"]["K"])
    out = {"out": F.mxfp4_linear(s["x"], weight, s["bias"], s["residual"], activation=s["case"]["act"])}
    if s["leaves"]:
        grads = torch.autograd.grad(out["out"], [s[n] for n in s["leaves"]], s["dout"])
        out.update(("d" + n, gr) for n, gr in zip(s["leaves"], grads))
    return out


def _act(kind, z):
    """The activation and its derivative."""
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "silu":
        sig = 1 / (1 + torch.exp(-z))
        return z * sig, sig * (1 + z * (1 - sig))
    a = math.sqrt(2 / math.pi)
    t = torch.tanh(a * (z + 0.044715 * z * z * z))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)


def _plain_linear(s):
    case, dtype = s["case"], s["x"].dtype
    w = _decode(s["codes"], s["scales"], case["K"])
    z = _values(s["x"].float(), torch.float32) @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if case["act"] == "swiglu":
        z1, z2 = z.chunk(2, dim=-1)
        a1, d1 = _act("silu", z1)
        out = a1 * z2
    else:
        out, d = _act(case["act"], z)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    r = {"out": out.to(dtype)}
    if s["leaves"]:
        dout = s["dout"].float()
        dz = torch.cat([dout * z2 * d1, dout * a1], dim=-1) if case["act"] == "swiglu" else dout * d
        r["dx"] = (dz @ w).to(dtype)
        if s["bias"] is not None:
            r["dbias"] = dz.sum(0).to(dtype)
        if s["residual"] is not None:
            r["dresidual"] = s["dout"]
    return r


def _plain_norm(s):
    """In 64 bits: a value next to a border between two codes falls on its own side."""
    dtype = s["x"].dtype

    def unit(t):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + _EPS)

    def by_token(rows):
        rows = rows.double()
        if s["doc_ids"] is None:
            return rows[:, None, :]
        ids = s["doc_ids"].long()
        rows = torch.cat([rows, torch.zeros_like(rows[:, :1])], 1)
        index = torch.where((ids < 0) | (ids >= rows.shape[1] - 1), rows.shape[1] - 1, ids)
        return rows[torch.arange(rows.shape[0], device=rows.device)[:, None], index]

    y = unit(s["x"].double()) * s["weight"].double()
    if s["case"]["op"] == "modulate":
        return {"out": _values(y * (1 + by_token(s["scale"])), dtype)}
    h = s["residual"].double() + by_token(s["gate"]) * y
    return {"out": _values(unit(h) * s["next_weight"].double() * (1 + by_token(s["next_scale"])), dtype),
            "hidden": h.to(dtype)}


# ---------------------------------------------------------------- 64 bits

def _exact_values(x):
    """MXFP4's values of fp64 rows: the border that each magnitude has passed, block by block."""
    columns = x.shape[-1]
    x = torch.cat([x, x.new_zeros(*x.shape[:-1], -columns % 32)], -1)
    b = x.reshape(*x.shape[:-1], -1, 32)
    top = b.abs().max(dim=-1, keepdim=True).values
    # floor(log2 top) by the powers of two that top reaches, one halving at a time of their range
    e = torch.full_like(top, -150.0)
    for step in (256.0, 128.0, 64.0, 32.0, 16.0, 8.0, 4.0, 2.0, 1.0):
        e = torch.where(top >= torch.pow(2.0, e + step), e + step, e)
    scale = torch.pow(2.0, torch.clamp(e - 2, min=-127.0))
    ratio = b.abs() / scale
    value = torch.zeros_like(b)
    for border, even_below, above in ((0.25, True, 0.5), (0.75, False, 1.0), (1.25, True, 1.5), (1.75, False, 2.0),
                                      (2.5, True, 3.0), (3.5, False, 4.0), (5.0, True, 6.0)):
        passed = ratio > border if even_below else ratio >= border
        value = torch.where(passed, above, value)
    return (torch.sign(b) * value * scale).reshape(x.shape)[..., :columns]


def exact(case, seed):
    """The definition in 64 bits; gradients by differentiating it."""
    s = prepare(case, seed)
    v = {n: t.detach().double() for n, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}
    if case["op"] == "quantize":
        return {"values": _exact_values(v["x"])}

    def unit(t):
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + _EPS)

    def by_token(rows):
        if s["doc_ids"] is None:
            return rows.unsqueeze(1).expand(-1, case["N"], -1)
        ids = s["doc_ids"].long()
        live = (ids >= 0) & (ids < rows.shape[1])
        picked = torch.gather(rows, 1, ids.clamp(0, rows.shape[1] - 1).unsqueeze(-1).expand(-1, -1, rows.shape[2]))
        return picked * live.unsqueeze(-1)

    if case["op"] == "modulate":
        return {"out": _exact_values(unit(v["x"]) * v["weight"] * (1 + by_token(v["scale"])))}
    if case["op"] == "gate_modulate":
        h = v["residual"] + by_token(v["gate"]) * unit(v["x"]) * v["weight"]
        return {"out": _exact_values(unit(h) * v["next_weight"] * (1 + by_token(v["next_scale"]))), "hidden": h}

    # the weight's values, one code at a time
    nibbles = torch.stack([s["codes"] % 16, s["codes"] // 16], dim=-1).flatten(1).long()
    magnitude = torch.tensor(_VALUES, dtype=torch.float64, device=nibbles.device)[nibbles % 8]
    powers = torch.pow(2.0, s["scales"].double() - 127).permute(1, 0, 2).flatten(1).repeat_interleave(32, dim=1)
    w = (torch.where(nibbles >= 8, -magnitude, magnitude) * powers)[:, :case["K"]]
    leaves = {n: v[n].requires_grad_() for n in s["leaves"]}
    x = v["x"] + (_exact_values(v["x"].detach()) - v["x"]).detach()  # the rounding passes the gradient on
    z = torch.matmul(x, w.mT)
    if "bias" in v:
        z = z + v["bias"]
    if case["act"] == "swiglu":
        half = z.shape[-1] // 2
        z = z[:, :half] * torch.sigmoid(z[:, :half]) * z[:, half:]
    elif case["act"] == "silu":
        z = z * torch.sigmoid(z)
    elif case["act"] == "gelu":
        z = z * torch.sigmoid(math.sqrt(8 / math.pi) * (z + 0.044715 * z.pow(3)))
    out = {"out": z + v["residual"] if "residual" in v else z}
    if leaves:
        grads = torch.autograd.grad(out["out"], list(leaves.values()), v["dout"])
        out.update(("d" + n, gr) for n, gr in zip(leaves, grads))
    return {n: t.detach() for n, t in out.items()}
