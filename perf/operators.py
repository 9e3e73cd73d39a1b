"""The operators around the attention of a transformer block, as measurable cases.

* ``modulate``       RMS norm before a block with its modulation: ``xhat * w * (1 + scale)``
* ``gate``           RMS norm after a block with its gate and the residual: ``r + gate * xhat * w``
* ``gate_modulate``  the norm after one block and the norm before the next in one pass
* ``linear``         ``act(x W^T + b) + r``

``xhat`` is ``x / sqrt(mean(x^2) + eps)`` over the channels.  ``scale`` and
``gate`` have a row per batch item, or with document ids a row per document of
a packed sequence (tokens of no document: scale 0, gate 0).  ``train`` cases run the
operator and the gradients of everything it takes.  Channels are the package's
30 heads of 128 and smaller or odd widths; the conditioning rows are views of
one projection's output, as a block has them.
"""

import math

import torch

own = False

_EPS = 1e-5
_WIDTH = 30 * 128  # channels of the package's model shape
_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _norm(op, B, N, C, segments="", pad=0, dtype="bf16", params="bf16", train=False):
    """``pad``: tokens of no document behind the last segment."""
    return dict(op=op, B=B, N=N, C=C, segments=segments, pad=pad, dtype=dtype, params=params, train=train)


def _linear(M, K, N, act="none", bias=False, residual=False, dtype="bf16", train=False):
    """``N``: columns of the output; a swiglu weight has two rows for each."""
    return dict(op="linear", M=M, K=K, N=N, act=act, bias=bias, residual=residual, dtype=dtype, train=train)


def listed():
    named = {
        # the padded caption tokens of one prompt in the caption refiner: latency
        "modulate_caption": _norm("modulate", 1, 32, _WIDTH),
        # fine-tuning on the packed mixed-resolution batch, a timestep per image
        "modulate_packed_train": _norm("modulate", 1, 6912, _WIDTH, segments="1280,1216,4416", train=True),
        # one 1280x832 image in the sampling loop
        "gate_dit1280": _norm("gate", 1, 4416, _WIDTH),
        # fine-tuning a narrow odd-width block on a ragged pair, padded, half precision
        "gate_odd_train": _norm("gate", 2, 1337, 1001, segments="700,600", pad=37, dtype="fp16", params="fp32",
                                train=True),
        # four 1024x1024 samples between attention and feed-forward (the largest memory-bound pass)
        "gate_modulate_ktuple": _norm("gate_modulate", 4, 4352, _WIDTH),
        # the same place while fine-tuning on a pack of odd segment lengths
        "gate_modulate_train": _norm("gate_modulate", 1, 3071, _WIDTH, segments="1003,771,1297", params="fp32",
                                     train=True),
        # conditioning rows of a pair of samples: few rows, every weight read once
        "linear_conditioning": _linear(2, 256, 4 * _WIDTH, bias=True),
        # the feed-forward's gated up-projection of one 1280x832 image (hidden of 8/3 of the width)
        "linear_swiglu_dit1280": _linear(4416, _WIDTH, _WIDTH * 8 // 3, act="swiglu"),
        # the feed-forward's down-projection of one 512x512 image, onto the residual
        "linear_down_dit512": _linear(1280, _WIDTH * 8 // 3, _WIDTH, bias=True, residual=True),
        # fine-tuning the QKV projection on one 1280x832 image (the largest)
        "linear_qkv_train": _linear(4416, _WIDTH, 3 * _WIDTH, bias=True, train=True),
        # fine-tuning a small odd head, half precision
        "linear_odd_train": _linear(667, 1001, 779, act="silu", bias=True, residual=True, dtype="fp16", train=True),
        # the second product of a rank-16 adapter, added to the base projection's output
        "linear_adapter_train": _linear(4416, 16, _WIDTH, residual=True, train=True),
    }
    return [dict(c, name=name) for name, c in named.items()]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """The same operators over the range of sizes: 1 to 6912 tokens, 64 to 10240 channels, odd ones among them."""
    width = rng.choice([_log_int(rng, 64, 4200), 8 * _log_int(rng, 8, 525), 1024, 1536, 2048, _WIDTH, _WIDTH])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    train = rng.random() < 0.5
    if rng.random() < 0.5:
        op = rng.choice(["modulate", "gate", "gate_modulate"])
        n, b = _log_int(rng, 1, 6912), rng.choice([1, 1, 2, 4])
        c = _norm(op, b, n, width, dtype=dtype, params=rng.choice([dtype, "fp32"]), train=train)
        if n >= 16 and rng.random() < 0.5:
            pad = rng.choice([0, n % 13])
            cuts = [0] + sorted(rng.sample(range(1, n - pad), rng.choice([1, 2, 3]))) + [n - pad]
            c.update(pad=pad, segments=",".join(str(y - x) for x, y in zip(cuts, cuts[1:])))
        while work(c)["bytes"] > 4 * 4352 * _WIDTH * 8:
            c["B"] //= 2
        return c
    m = _log_int(rng, 1, 6912)
    n = rng.choice([16, _log_int(rng, 64, 4200), 8 * _log_int(rng, 8, 1280), _WIDTH, 3 * _WIDTH, _WIDTH * 8 // 3])
    k = rng.choice([16, 256, width, width, width])
    c = _linear(m, k, n, act=rng.choice(["none", "none", "silu", "gelu", "swiglu"]), bias=rng.random() < 0.5,
                residual=rng.random() < 0.5, dtype=dtype, train=train)
    while work(c)["flops"] > 6 * 4416 * _WIDTH * 3 * _WIDTH:
        c["M"] //= 2
    return c


def work(case):
    if case["op"] == "linear":
        m, k, n, train = case["M"], case["K"], case["N"], case["train"]
        rows = 2 * n if case["act"] == "swiglu" else n
        nbytes = 2 * (m * k + rows * k + m * n + (m * n if case["residual"] else 0) + (rows if case["bias"] else 0))
        if train:  # dout in; dx, dW, db out (the residual's gradient is dout)
            nbytes += 2 * (m * n + m * k + rows * k + (rows if case["bias"] else 0))
        return {"bytes": nbytes, "flops": (6 if train else 2) * m * k * rows}
    tokens = case["B"] * case["N"]
    each = tokens * case["C"] * 2  # bytes of one [B, N, C] tensor
    op, train = case["op"], case["train"]
    tensors = {"modulate": 2, "gate": 3, "gate_modulate": 4}[op]
    if train:  # incoming gradients read, gradients written (gate: the residual's is dout itself)
        tensors += {"modulate": 2, "gate": 2, "gate_modulate": 4}[op]
    flops = tokens * case["C"] * (8 if op == "gate_modulate" else 5) * (3 if train else 1)
    return {"bytes": tensors * each, "flops": flops}


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

    dtype, train = _DTYPE[case["dtype"]], case["train"]
    s = {"case": case}
    if case["op"] == "linear":
        m, k, n = case["M"], case["K"], case["N"]
        rows = 2 * n if case["act"] == "swiglu" else n
        s["x"] = normal(m, k).to(dtype)
        s["weight"] = (normal(rows, k) / math.sqrt(k)).to(dtype)
        s["bias"] = (0.3 * normal(rows)).to(dtype) if case["bias"] else None
        s["residual"] = normal(m, n).to(dtype) if case["residual"] else None
        if train:
            s["dout"] = normal(m, n).to(dtype)
        leaves = ("x", "weight", "bias", "residual")
    else:
        B, N, C, params = case["B"], case["N"], case["C"], _DTYPE[case["params"]]
        shape = (B, N, C)
        s["doc_ids"] = _doc_ids(case, device) if case["segments"] else None
        docs = (len(case["segments"].split(",")),) if case["segments"] else ()
        s["x"] = (1.5 * normal(*shape)).to(dtype)
        s["weight"] = (1 + 0.2 * normal(C)).to(params)
        # scale and gate of both halves of a block, from one projection
        scale, gate, scale2, _ = (0.4 * normal(B, *docs, 4 * C)).to(params).chunk(4, dim=-1)
        if case["op"] == "modulate":
            s["scale"] = scale
        else:
            s["residual"] = (2 * normal(*shape)).to(dtype)
            s["gate"] = gate
        if case["op"] == "gate_modulate":
            s["next_weight"] = (1 + 0.2 * normal(C)).to(params)
            s["next_scale"] = scale2
        if train:
            s["dout"] = normal(*shape).to(dtype)
            if case["op"] == "gate_modulate":
                s["dhidden"] = normal(*shape).to(dtype)
        leaves = ("x", "residual", "weight", "scale", "gate", "next_weight", "next_scale")
    s["leaves"] = [name for name in leaves if s.get(name) is not None] if train else []
    for name in s["leaves"]:
        s[name] = s[name].detach().requires_grad_()
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    if own:
        return _framework(state)
    with torch.no_grad():
        return _plain_linear(state) if state["case"]["op"] == "linear" else _plain_norm(state)


def _framework(s):
    import futudiffu_amd as F
    op = s["case"]["op"]
    if op == "linear":
        out = {"out": F.fused_linear(s["x"], s["weight"], s["bias"], s["residual"], activation=s["case"]["act"])}
    elif op == "modulate":
        out = {"out": F.rms_norm_modulate(s["x"], s["weight"], s["scale"], doc_ids=s["doc_ids"], eps=_EPS)}
    elif op == "gate":
        out = {"out": F.rms_norm_gate_residual(s["residual"], s["x"], s["weight"], s["gate"], doc_ids=s["doc_ids"],
                                               eps=_EPS)}
    else:
        hidden, y = F.rms_norm_gate_residual_modulate(s["residual"], s["x"], s["weight"], s["gate"],
                                                      s["next_weight"], s["next_scale"], doc_ids=s["doc_ids"],
                                                      eps=_EPS)
        out = {"out": y, "hidden": hidden}
    if s["leaves"]:
        grads = torch.autograd.grad(list(out.values()), [s[n] for n in s["leaves"]], [s["d" + n] for n in out])
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
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
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
        r["dweight"] = (dz.t() @ x).to(dtype)
        if s["bias"] is not None:
            r["dbias"] = dz.sum(0).to(dtype)
        if s["residual"] is not None:
            r["dresidual"] = s["dout"]
    return r


class _Rows:
    """Rows of a conditioning tensor by token, and the sums of a token tensor by row."""

    def __init__(self, s, docs):
        self.ids, self.docs = s["doc_ids"], docs
        if self.ids is not None:
            ids = self.ids.long()
            self.index = torch.where((ids < 0) | (ids >= docs), docs, ids)

    def of(self, rows):
        rows = rows.float()
        if self.ids is None:
            return rows[:, None, :]
        rows = torch.cat([rows, torch.zeros_like(rows[:, :1])], 1)
        return rows[torch.arange(rows.shape[0], device=rows.device)[:, None], self.index]

    def sums(self, t):
        if self.ids is None:
            return t.sum(1)
        one = (self.index[:, None, :] == torch.arange(self.docs, device=t.device)[None, :, None]).float()
        return torch.matmul(one, t)


def _norm_plain(x):
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
    return x * r, r


def _norm_plain_back(g, xhat, r):
    return r * (g - xhat * (g * xhat).mean(-1, keepdim=True))


def _plain_norm(s):
    op, dtype, params = s["case"]["op"], s["x"].dtype, s["weight"].dtype
    cond = s["scale"] if op == "modulate" else s["gate"]
    rows = _Rows(s, cond.shape[1] if cond.ndim == 3 else 0)
    w = s["weight"].float()
    xhat, rr = _norm_plain(s["x"].float())
    m = rows.of(cond)
    if op == "modulate":
        m = 1 + m
        out = {"out": (xhat * w * m).to(dtype)}
    else:
        h = s["residual"].float() + m * (xhat * w)
        out = {"out": h.to(dtype)}
    if op == "gate_modulate":
        hhat, hr = _norm_plain(h)
        w2, m2 = s["next_weight"].float(), 1 + rows.of(s["next_scale"])
        out = {"out": (hhat * w2 * m2).to(dtype), "hidden": h.to(dtype)}
    if not s["leaves"]:
        return out
    d = s["dout"].float()
    grads = {}
    if op == "gate_modulate":
        grads["dnext_weight"] = (d * hhat * m2).sum((0, 1)).to(params)
        grads["dnext_scale"] = rows.sums(d * hhat * w2).to(params)
        d = s["dhidden"].float() + _norm_plain_back(d * w2 * m2, hhat, hr)
    grads["dx"] = _norm_plain_back(d * w * m, xhat, rr).to(dtype)
    grads["dweight"] = (d * xhat * m).sum((0, 1)).to(params)
    grads["dscale" if op == "modulate" else "dgate"] = rows.sums(d * xhat * w).to(params)
    if op != "modulate":
        grads["dresidual"] = s["dout"] if op == "gate" else d.to(dtype)
    out.update(("d" + n, grads["d" + n]) for n in s["leaves"])
    return out


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    """The definition in 64 bits; gradients by differentiating it."""
    s = prepare(case, seed)
    v = {n: t.detach().double().requires_grad_(n in s["leaves"])
         for n, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}

    def unit(t):
        return t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + _EPS)

    def by_token(rows):
        if s["doc_ids"] is None:
            return rows.unsqueeze(1).expand(-1, case["N"], -1)
        ids = s["doc_ids"].long()
        live = (ids >= 0) & (ids < rows.shape[1])
        picked = torch.gather(rows, 1, ids.clamp(0, rows.shape[1] - 1).unsqueeze(-1).expand(-1, -1, rows.shape[2]))
        return picked * live.unsqueeze(-1)

    if case["op"] == "linear":
        z = torch.matmul(v["x"], v["weight"].mT)
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
    elif case["op"] == "modulate":
        out = {"out": unit(v["x"]) * v["weight"] * (1 + by_token(v["scale"]))}
    else:
        h = v["residual"] + by_token(v["gate"]) * unit(v["x"]) * v["weight"]
        out = {"out": h}
        if case["op"] == "gate_modulate":
            out = {"out": unit(h) * v["next_weight"] * (1 + by_token(v["next_scale"])), "hidden": h}
    if s["leaves"]:
        grads = torch.autograd.grad(list(out.values()), [v[n] for n in s["leaves"]], [v["d" + n] for n in out])
        out.update(("d" + n, gr) for n, gr in zip(s["leaves"], grads))
    return {n: t.detach() for n, t in out.items()}
