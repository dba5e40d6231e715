"""What the memory-saving operators of long-sequence training cost, and their plain forms.

Three operators, as a training step at long context uses them side by side:

  xent    cross entropy of a language-model head without logits in memory:
          ``functional.linear_cross_entropy`` (loss, hidden gradient, head-weight gradient; or
          per-token losses only, to score text)
  act8    activations kept in 8 bits between forward and backward: ``act8.quantize`` /
          ``dequantize`` (a checkpoint), ``act8.rms_norm`` and ``act8.swiglu`` with backward
          passes that read the 8-bit copies
  rotary  rotary positions in half or interleaved layout, over all or part of the head, from
          fp32 tables that may be scaled for long contexts: ``rotary.rotary_qk``

``run`` computes the plain form (elementary fp32 tensor operations) where ``own`` is false and
calls the framework where it is true.  ``exact`` restates each definition in 64 bits.
"""
import math

import torch

own = False

GROUPS = (32, 64, 128, 256)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one next-token probability of one sequence: the head weight is read once, latency counts
        dict(name="xent score 1 token", op="xent", grad=False, T=1, H=4096, V=32000, ignored=0.0),
        # the debug configuration's micro-batch (4 x 128 tokens): launch-bound
        dict(name="xent train tiny", op="xent", grad=True, T=512, H=256, V=2048, ignored=0.0),
        # a packed batch with padding, no dimension a multiple of a tile, odd vocabulary
        dict(name="xent train ragged", op="xent", grad=True, T=1021, H=5120, V=32003, ignored=0.1),
        # one micro-batch of the 8B configuration: 4096 tokens over its 128256-word vocabulary
        dict(name="xent train 8B", op="xent", grad=True, T=4096, H=4096, V=128256, ignored=0.0),
        # a short ragged fp32 activation kept through a forward pass and restored
        dict(name="act8 checkpoint odd", op="ckpt", T=509, N=1023, dtype="fp32", group=64),
        # the decoder-layer inputs of an 8B micro-batch of two sequences
        dict(name="act8 checkpoint 8B", op="ckpt", T=8192, N=4096, dtype="bf16", group=128),
        # RMSNorm of the 70B hidden size whose backward reads its input in 8 bits
        dict(name="act8 norm 70B", op="norm8", T=4096, H=8192, group=128),
        # SwiGLU of the debug configuration's MLP, last group of each half ragged
        dict(name="act8 swiglu tiny", op="swiglu8", T=512, F=688, group=128),
        # SwiGLU of an 8B micro-batch: the largest activation of a decoder layer
        dict(name="act8 swiglu 8B", op="swiglu8", T=4096, F=14336, group=128),
        # eight sequences each adding one token far into their context: latency
        dict(name="rotary one token", op="rotary", B=8, S=1, nq=32, nkv=8, d=128, rot=128,
             interleaved=False, inverse=False, dtype="bf16", far=131072, heads_first=False),
        # the query and key of the 8B configuration, scattered positions in a long context
        dict(name="rotary 8B long", op="rotary", B=2, S=8192, nq=32, nkv=8, d=128, rot=128,
             interleaved=False, inverse=False, dtype="bf16", far=131072, heads_first=False),
        # the backward pass of a partial, interleaved rotation in heads-first order, odd length
        dict(name="rotary partial back", op="rotary", B=3, S=1999, nq=40, nkv=40, d=128, rot=64,
             interleaved=True, inverse=True, dtype="bf16", far=8192, heads_first=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["xent", "xent", "ckpt", "norm8", "swiglu8", "rotary", "rotary"])
    if op == "xent":
        while True:
            c = dict(op=op, grad=rng.random() < 0.75, T=_log(rng, 1, 8192),
                     H=rng.choice([256, 512, 1000, 2048, 4096, 5120, 8192]),
                     V=_log(rng, 2000, 128256), ignored=rng.choice([0.0, 0.1, 0.5]))
            if c["T"] * c["H"] * c["V"] <= 4096 * 4096 * 128256 and c["H"] * c["V"] <= 4096 * 128256:
                return c
    if op == "ckpt":
        while True:
            c = dict(op=op, T=_log(rng, 1, 16384), N=_log(rng, 64, 28672),
                     dtype=rng.choice(["bf16", "fp32"]), group=rng.choice(GROUPS))
            if c["T"] * c["N"] <= 8192 * 4096:
                return c
    if op == "norm8":
        while True:
            c = dict(op=op, T=_log(rng, 1, 16384), H=8 * _log(rng, 8, 1024), group=rng.choice(GROUPS))
            if c["T"] * c["H"] <= 4096 * 8192:
                return c
    if op == "swiglu8":
        while True:
            c = dict(op=op, T=_log(rng, 1, 16384), F=8 * _log(rng, 16, 3584), group=rng.choice(GROUPS))
            if c["T"] * c["F"] <= 4096 * 14336:
                return c
    while True:
        d = rng.choice([32, 36, 64, 80, 96, 128, 192, 256])
        nkv = rng.choice([1, 4, 8, 32, 40])
        c = dict(op=op, B=rng.choice([1, 2, 3, 8]), S=_log(rng, 1, 8192),
                 nq=nkv * rng.choice([1, 4, 8]), nkv=nkv, d=d,
                 rot=rng.choice([d, d, d // 2, d // 4 * 2]), interleaved=rng.random() < 0.5,
                 inverse=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                 far=rng.choice([8192, 32768, 131072]), heads_first=rng.random() < 0.5)
        elems = c["B"] * c["S"] * (c["nq"] + c["nkv"]) * d * (2 if c["dtype"] == "fp32" else 1)
        if elems <= 2 * 8192 * 40 * 128:
            return c


# ------------------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    op = case["op"]
    s = dict(case)
    if op == "xent":
        T, H, V = case["T"], case["H"], case["V"]
        # hidden states leave an RMSNorm (unit rms); logits spread by about 2.5 around zero
        s["h"] = randn(T, H)
        s["w"] = randn(V, H, scale=2.5 / math.sqrt(H))
        labels = torch.randint(0, V, (T,), generator=g, device="cuda")
        drop = torch.rand(T, generator=g, device="cuda") < case["ignored"]
        drop[0] = False
        s["labels"] = torch.where(drop, torch.full_like(labels, -100), labels)
        if case["grad"]:
            s["h"].requires_grad_()
            s["w"].requires_grad_()
    elif op == "ckpt":
        # activations with a few channels far above the others, as hidden states have
        x = randn(case["T"], case["N"], dtype=torch.float32)
        big = torch.rand(case["N"], generator=g, device="cuda") < 0.01
        s["x"] = (x * torch.where(big, 20.0, 1.0)).to(TYPES[case["dtype"]])
    elif op == "norm8":
        x = randn(case["T"], case["H"], dtype=torch.float32)
        big = torch.rand(case["H"], generator=g, device="cuda") < 0.01
        s["x"] = (x * torch.where(big, 20.0, 1.0)).to(torch.bfloat16)
        s["w"] = (1 + 0.1 * torch.randn(case["H"], generator=g, device="cuda")).to(torch.bfloat16)
        s["dy"] = randn(case["T"], case["H"], scale=1e-2)
    elif op == "swiglu8":
        s["gu"] = randn(case["T"], 2 * case["F"], scale=1.5)
        s["dh"] = randn(case["T"], case["F"], scale=1e-2)
    else:
        B, S, nq, nkv, d = (case[k] for k in ("B", "S", "nq", "nkv", "d"))
        dt = TYPES[case["dtype"]]
        if case["heads_first"]:
            qkv = randn(B, nq + 2 * nkv, S, d, dtype=dt).transpose(1, 2)
        else:
            qkv = randn(B, S, nq + 2 * nkv, d, dtype=dt)
        s["q"], s["k"] = qkv[:, :, :nq], qkv[:, :, nq:nq + nkv]
        # tables of the whole context, frequencies stretched by a factor of 4
        inv = 1.0 / (500000.0 ** (torch.arange(0, case["rot"], 2, device="cuda").double() / case["rot"])) / 4
        angle = torch.outer(torch.arange(case["far"], device="cuda").double(), inv)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        start = torch.randint(0, case["far"] - S + 1, (B, 1), generator=g, device="cuda")
        s["pos"] = start + torch.arange(S, device="cuda")
    return s


# ------------------------------------------------------------------------------ plain forms
def _quant(x, group, f32=torch.float32):
    """The values that 8 bits keep of x: rows in groups of `group`, symmetric, largest
    magnitude at 127, ties to even; a group all below 2^-120 is kept as zeros."""
    T, n = x.shape
    m = -(-n // group)
    p = torch.zeros(T, m * group, dtype=f32, device=x.device)
    p[:, :n] = x
    p = p.view(T, m, group)
    top = p.abs().amax(-1, keepdim=True)
    inv = torch.where(top >= 2.0 ** -120, torch.reciprocal(top) * 127.0, torch.zeros_like(top))
    q = torch.round(p * inv).clamp(-127, 127)
    return (q * (top * (1.0 / 127.0))).view(T, m * group)[:, :n]


def _plain_xent(s, dt=torch.float32):
    h, w, lab = s["h"].detach().to(dt), s["w"].detach().to(dt), s["labels"]
    x = h @ w.t()
    valid = lab != -100
    at = lab.clamp(min=0)[:, None]
    top = x.amax(1, keepdim=True)
    lse = torch.log(torch.exp(x - top).sum(1, keepdim=True)) + top
    rows = torch.where(valid, (lse - x.gather(1, at))[:, 0], torch.zeros_like(lse[:, 0]))
    if not s["grad"]:
        return {"losses": rows}
    n = valid.sum()
    p = x.sub_(lse).exp_()
    p.scatter_add_(1, at, torch.full_like(lse, -1.0))
    p.mul_((valid / n)[:, None].to(dt))
    return {"loss": rows.sum() / n, "dh": p @ w, "dw": p.t() @ h}


def _plain_norm8(s, dt=torch.float32):
    x, w, dy = s["x"].to(dt), s["w"].to(dt), s["dy"].to(dt)
    rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-5)
    n = _quant(x, s["group"], dt) * rstd
    dn = dy * w
    dx = rstd * (dn - n * (dn * n).mean(1, keepdim=True))
    return {"y": x * rstd * w, "rstd": rstd[:, 0], "dx": dx, "dw": (dy * n).sum(0), "y8": n * w}


def _plain_swiglu8(s, dt=torch.float32):
    F = s["F"]
    g, u, dh = s["gu"][:, :F].to(dt), s["gu"][:, F:].to(dt), s["dh"].to(dt)
    h = g / (1 + torch.exp(-g)) * u
    g, u = _quant(g, s["group"], dt), _quant(u, s["group"], dt)
    sg = 1 / (1 + torch.exp(-g))
    dgu = torch.cat([dh * u * sg * (1 + g * (1 - sg)), dh * g * sg], 1)
    return {"h": h, "dgu": dgu, "h8": g * sg * u}


def _plain_rotary(s, dt=torch.float32):
    r = s["rot"] // 2
    c, n = s["cos"].to(dt)[s["pos"]][:, :, None], s["sin"].to(dt)[s["pos"]][:, :, None]
    n = -n if s["inverse"] else n

    def turn(x):
        x = x.to(dt)
        a, b = (x[..., 0:2 * r:2], x[..., 1:2 * r:2]) if s["interleaved"] else (x[..., :r], x[..., r:2 * r])
        ra, rb = a * c - b * n, b * c + a * n
        y = x.clone()
        if s["interleaved"]:
            y[..., 0:2 * r:2], y[..., 1:2 * r:2] = ra, rb
        else:
            y[..., :r], y[..., r:2 * r] = ra, rb
        return y
    return {"q": turn(s["q"]), "k": turn(s["k"])}


def _plain(s, dt=torch.float32):
    op = s["op"]
    if op == "xent":
        return _plain_xent(s, dt)
    if op == "ckpt":
        return {"x8": _quant(s["x"].to(dt), s["group"], dt)}
    return {"norm8": _plain_norm8, "swiglu8": _plain_swiglu8, "rotary": _plain_rotary}[op](s, dt)


def _rounded(s, out):
    """Each output once to the type that the operator gives it in."""
    if s["op"] in ("ckpt", "rotary"):
        return {k: v.to(TYPES[s["dtype"]]) for k, v in out.items()}
    return {k: v if k in ("loss", "losses", "rstd") or s["op"] == "norm8" and k == "dw"
            else v.to(torch.bfloat16) for k, v in out.items()}


def run(s):
    if not own:
        return _rounded(s, _plain(s))
    op = s["op"]
    if op == "xent":
        from femtotron_b200.ops.functional import linear_cross_entropy
        h, w = s["h"], s["w"]
        if not s["grad"]:
            with torch.no_grad():
                return {"losses": linear_cross_entropy(h, w, s["labels"], reduction="none")}
        h.grad = w.grad = None
        loss = linear_cross_entropy(h, w, s["labels"])
        loss.backward()
        return {"loss": loss.detach(), "dh": h.grad, "dw": w.grad}
    if op == "rotary":
        from femtotron_b200.ops import rotary
        q, k = rotary.rotary_qk(s["q"], s["k"], s["cos"], s["sin"], s["pos"],
                                interleaved=s["interleaved"], inverse=s["inverse"])
        return {"q": q, "k": k}
    from femtotron_b200.ops import act8
    if op == "ckpt":
        return {"x8": act8.quantize(s["x"], s["group"]).dequantize()}
    if op == "norm8":
        y, rstd, x8 = act8.rms_norm(s["x"], s["w"], 1e-5, s["group"])
        dx, dw, y8 = act8.rms_norm_bwd(s["dy"], x8, s["w"], rstd)
        return {"y": y, "rstd": rstd, "dx": dx, "dw": dw, "y8": y8}
    h, gu8 = act8.swiglu(s["gu"], s["group"])
    dgu, h8 = act8.swiglu_bwd(s["dh"], gu8)
    return {"h": h, "dgu": dgu, "h8": h8}


# ------------------------------------------------------------------------------ cost and truth
def work(case):
    op = case["op"]
    if op == "xent":
        T, H, V = case["T"], case["H"], case["V"]
        read = 2 * T * H + 2 * V * H + 8 * T
        if not case["grad"]:
            return {"bytes": read + 4 * T, "flops": 2 * T * H * V}
        # logits, hidden gradient and weight gradient: three products
        return {"bytes": read + 2 * T * H + 2 * V * H + 4, "flops": 6 * T * H * V}
    if op == "ckpt":
        # x in, the 8-bit copy and its scales out and in again, x out
        n, e = case["T"] * case["N"], 4 if case["dtype"] == "fp32" else 2
        m = case["T"] * -(-case["N"] // case["group"])
        return {"bytes": 2 * n * e + 2 * (n + 4 * m), "flops": 5 * n}
    if op == "norm8":
        # x -> y, 8 bits, rstd;  dy, 8 bits, rstd -> dx, dw, y8
        T, H = case["T"], case["H"]
        m = T * -(-H // case["group"])
        return {"bytes": T * H * (2 + 2 + 1 + 2 + 1 + 2 + 2) + 8 * m + 8 * T + 4 * H + 4 * H,
                "flops": 20 * T * H}
    if op == "swiglu8":
        # gu -> h, 8 bits;  dh, 8 bits -> dgu, h8
        T, F = case["T"], case["F"]
        m = 2 * T * -(-F // case["group"])
        return {"bytes": T * F * (4 + 2 + 2 + 2 + 2 + 4 + 2) + 8 * m, "flops": 30 * T * F}
    e = 4 if case["dtype"] == "fp32" else 2
    n = case["B"] * case["S"] * (case["nq"] + case["nkv"]) * case["d"]
    tables = case["B"] * case["S"] * (case["rot"] * 4 + 8)
    return {"bytes": 2 * n * e + tables, "flops": 3 * n}


def exact(case, seed):
    """The definitions in 64 bits, one row, group or pair at a time where that fits."""
    s = prepare(case, seed)
    op, f = s["op"], torch.float64
    if op == "xent":
        h, w, lab = s["h"].detach().to(f), s["w"].detach().to(f), s["labels"]
        logits = torch.einsum("th,vh->tv", h, w)
        keep = (lab != -100).nonzero()[:, 0]
        lse = torch.logsumexp(logits, 1)
        losses = torch.zeros(lab.shape[0], dtype=f, device="cuda")
        losses[keep] = lse[keep] - logits[keep, lab[keep]]
        if not s["grad"]:
            return {"losses": losses}
        p = torch.softmax(logits, 1)
        del logits
        p[keep, lab[keep]] -= 1
        p[lab == -100] = 0
        p /= keep.numel()
        return {"loss": losses.sum() / keep.numel(), "dh": torch.einsum("tv,vh->th", p, w),
                "dw": torch.einsum("tv,th->vh", p, h)}

    def eight(x):
        out = torch.empty_like(x)
        for a in range(0, x.shape[1], s["group"]):
            part = x[:, a:a + s["group"]]
            unit = part.abs().max(1, keepdim=True).values / 127
            out[:, a:a + s["group"]] = torch.where(unit > 0, torch.round(part / unit) * unit, 0 * part)
        return out

    if op == "ckpt":
        return {"x8": eight(s["x"].to(f))}
    if op == "norm8":
        x, w, dy = s["x"].to(f), s["w"].to(f), s["dy"].to(f)
        r = 1 / torch.sqrt(x.square().sum(1, keepdim=True) / x.shape[1] + 1e-5)
        xh = eight(x) * r
        dot = torch.einsum("th,th,h->t", dy, xh, w)[:, None] / x.shape[1]
        return {"y": w * (x * r), "rstd": r[:, 0], "dx": r * dy * w - r * xh * dot,
                "dw": torch.einsum("th,th->h", dy, xh), "y8": w * xh}
    if op == "swiglu8":
        F = s["F"]
        g, u, dh = s["gu"].to(f)[:, :F], s["gu"].to(f)[:, F:], s["dh"].to(f)
        g8, u8 = eight(g), eight(u)
        sg = torch.sigmoid(g8)
        return {"h": g * torch.sigmoid(g) * u,
                "dgu": torch.cat([dh * u8 * (sg + g8 * sg * (1 - sg)), dh * sg * g8], 1),
                "h8": g8 * sg * u8}
    r = s["rot"] // 2
    turn = torch.complex(s["cos"].to(f), s["sin"].to(f))[s["pos"].reshape(-1)]
    turn = turn.reshape(*s["pos"].shape, 1, r)
    turn = turn.conj() if s["inverse"] else turn
    out = {}
    for name in ("q", "k"):
        x = s[name].to(f)
        head, rest = x[..., :2 * r], x[..., 2 * r:]
        pairs = head.unflatten(-1, (r, 2)) if s["interleaved"] else head.unflatten(-1, (2, r)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        z = z if s["interleaved"] else z.transpose(-1, -2)
        out[name] = torch.cat([z.flatten(-2), rest], -1)
    return out
