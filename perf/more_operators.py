"""What the operators of a training step on packed documents cost, and their plain forms.

Three operators, in the order in which such a step meets them:

  embed  embedding lookup with a factor, and its gradient summed row by row in a fixed order:
         ``functional.embedding``
  attn   attention over whole sequences whose rows see what a mask of documents, a window and a
         prefix leaves them, with scores capped by a tanh or lowered by distance:
         ``masked_attention.masked_attention`` with ``masked_attention.attention_mask``
  clip   the global norm over many gradients and the gradients clipped by it:
         ``grad_norm.clip_grads``

``run`` computes the plain form (elementary fp32 tensor operations) where ``own`` is false and
calls the framework where it is true.  ``exact`` restates each definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the debug configuration's micro-batch (4 x 128 tokens) with short documents: launch-bound
        _attn("attn tiny documents", B=4, S=128, nq=8, nkv=4, d=32, doc=40),
        # one packed sequence of the 8B configuration's heads, documents of about a thousand tokens
        _attn("attn 8B documents", B=1, S=8192, nq=32, nkv=8, d=128, doc=1000),
        # the same heads in a layer with a sliding window and capped scores
        _attn("attn 8B window cap", B=2, S=4096, nq=32, nkv=8, d=128, window=1024, cap=30.0),
        # every head its own keys, a bias of distance, padded sequences of an odd length, a head size
        # that is no power of two
        _attn("attn distance ragged", B=3, S=1999, nq=40, nkv=40, d=80, alibi=True, pad=0.2),
        # a whole long sequence, the heads of one of eight tensor-parallel ranks of the 70B configuration
        _attn("attn 70B shard long", B=1, S=16384, nq=8, nkv=1, d=128),
        # prompts that see themselves in both directions, scored without gradients
        _attn("attn prefix score", B=8, S=1024, nq=12, nkv=12, d=64, prefix=0.4, grad=False),
        # the debug configuration's table and micro-batch, gradient in the weight's type: launch-bound
        dict(name="embed tiny", op="embed", T=512, V=2048, H=256, micro=1, scale=16.0, shard=1, grad="bf16"),
        # an 8B micro-batch of two sequences into the fp32 gradient buffer: the buffer is the largest
        dict(name="embed 8B", op="embed", T=8192, V=128256, H=4096, micro=1, scale=64.0, shard=1, grad="fp32"),
        # one of four vocabulary shards, two micro-batches summed, no size a multiple of a vector
        dict(name="embed shard odd", op="embed", T=3001, V=8001, H=1023, micro=2, scale=1.0, shard=4, grad="fp32"),
        # the gradients of the debug configuration: latency
        dict(name="clip tiny", op="clip", layers=4, H=256, F=688, V=2048, ranks=1, dtype="fp32", norm=3.0),
        # the fp32 gradient shards that one of eight ranks holds of the 8B configuration
        dict(name="clip 8B shard", op="clip", layers=32, H=4096, F=14336, V=128256, ranks=8, dtype="fp32", norm=40.0),
        # gradients in two types and odd lengths, of a norm that needs no clipping
        dict(name="clip mixed odd", op="clip", layers=40, H=1023, F=2731, V=32003, ranks=3, dtype="mixed", norm=0.5),
    ]


def _attn(name, *, B, S, nq, nkv, d, doc=0, window=0, cap=0.0, alibi=False, pad=0.0, prefix=0.0, causal=True, grad=True):
    c = dict(op="attn", B=B, S=S, nq=nq, nkv=nkv, d=d, doc=doc, window=window, cap=cap, alibi=alibi, pad=pad,
             prefix=prefix, causal=causal, grad=grad)
    return dict(c, name=name) if name else c


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "embed", "clip"])
    if op == "attn":
        while True:
            S, nkv = _log(rng, 1, 16384), rng.choice([1, 2, 4, 8, 12, 40])
            c = _attn(None, B=rng.choice([1, 1, 2, 3, 8]), S=S, nq=nkv * rng.choice([1, 1, 4, 8]), nkv=nkv,
                      d=rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 128]),
                      doc=rng.choice([0, _log(rng, 8, 8192)]), window=rng.choice([0, 0, _log(rng, 16, 8192)]),
                      cap=rng.choice([0.0, 0.0, 20.0, 50.0]), alibi=rng.random() < 0.25,
                      pad=rng.choice([0.0, 0.0, 0.3]), prefix=rng.choice([0.0, 0.0, 0.3]),
                      causal=rng.random() < 0.85, grad=rng.random() < 0.75)
            c["prefix"] *= c["causal"]
            if c["B"] * c["nq"] * S * S <= 8 * 16384 ** 2 and work(c)["flops"] <= work(listed()[4])["flops"]:
                return c
    if op == "embed":
        while True:
            c = dict(op=op, T=_log(rng, 1, 32768), V=_log(rng, 1000, 128256),
                     H=rng.choice([64, 256, 1000, 1023, 2048, 4096, 5120, 8192]), micro=rng.choice([1, 1, 2, 4]),
                     scale=rng.choice([1.0, 16.0, 45.25]), shard=rng.choice([1, 1, 2, 8]),
                     grad=rng.choice(["fp32", "fp32", "bf16"]))
            if c["V"] * c["H"] + c["micro"] * c["T"] * c["H"] <= 128256 * 4096:
                return c
    while True:
        c = dict(op=op, layers=_log(rng, 1, 48), H=_log(rng, 64, 8192), F=_log(rng, 128, 28672), V=_log(rng, 1000, 128256),
                 ranks=rng.choice([1, 1, 2, 8]), dtype=rng.choice(["fp32", "fp32", "bf16", "mixed"]),
                 norm=rng.choice([0.5, 3.0, 40.0]))
        if 1 <= sum(_grad_sizes(c)) <= 900_000_000:
            return c


def _grad_sizes(c):
    """Numbers of values of one rank's gradients, tensor by tensor."""
    H, F, r = c["H"], c["F"], c["ranks"]
    layer = [H * H, H * H // 4, H * H // 4, H * H, H * F, H * F, H * F, H, H]
    return [-(-n // r) for n in [c["V"] * H] + layer * c["layers"] + [H]]


# ------------------------------------------------------------------------------ the inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case)
    if case["op"] == "attn":
        B, S, nq, nkv, d = (case[k] for k in ("B", "S", "nq", "nkv", "d"))
        # queries and keys leave a projection and a rotation: scores spread by about 1.5
        s["q"], s["k"], s["v"] = randn(B, S, nq, d, scale=1.5), randn(B, S, nkv, d), randn(B, S, nkv, d)
        s["do"] = randn(B, S, nq, d, scale=1e-2)
        if case["grad"]:
            for n in "qkv":
                s[n].requires_grad_()
        s["docs"] = s["marks"] = s["slopes"] = None
        if case["doc"] or case["pad"]:
            # documents end with a fixed chance at every token; padding comes last
            begins = rand(B, S) < 1.0 / case["doc"] if case["doc"] else torch.zeros(B, S, dtype=torch.bool, device="cuda")
            kept = (S * (1 - case["pad"] * rand(B, 1))).ceil()
            place = torch.arange(S, device="cuda")[None]
            s["docs"] = torch.where(place < kept, begins.cumsum(1), torch.full_like(begins.cumsum(1), -1)).int()
        if case["prefix"]:
            # a prompt opens each sequence; what a document other than the first marks comes by chance
            ends = (S * 2 * case["prefix"] * rand(B, 1)).floor()
            s["marks"] = (torch.arange(S, device="cuda")[None] < ends) | (rand(B, S) < 0.3)
        if case["alibi"]:
            # the slopes 2^(-8 i / heads) of a bias of distance
            s["slopes"] = torch.exp2(-8.0 * torch.arange(1, nq + 1, device="cuda") / nq).float()
        if own and s["docs"] is None and s["marks"] is None:  # the same mask for every batch: a program keeps it
            from femtotron_b200.ops import masked_attention as MA
            s["mask"] = MA.attention_mask(1, S, causal=case["causal"], window=case["window"] or None, device="cuda")
    elif case["op"] == "embed":
        T, V, H, n = case["T"], case["V"], case["H"], case["micro"]
        s["weight"] = randn(V, H, scale=0.02).requires_grad_()
        # word frequencies fall with the rank (Zipf): a few words are a large part of every batch
        words = case["V"] * case["shard"]
        s["ids"] = (torch.exp(rand(n, T) * math.log(words + 1)) - 1).long().clamp_(0, words - 1)
        s["ids"] = s["ids"] * 7919 % words if math.gcd(7919, words) == 1 else s["ids"]
        s["vstart"] = case["V"] * (case["shard"] // 2)
        s["dout"] = randn(n, T, H, scale=1e-2)
        s["into"] = torch.zeros(V, H, device="cuda") if case["grad"] == "fp32" else None
    else:
        sizes = _grad_sizes(case)
        kind = ["bf16" if case["dtype"] == "bf16" or (case["dtype"] == "mixed" and i % 3) else "fp32" for i in range(len(sizes))]
        # one buffer for each type, as a sharding strategy holds gradients; every tensor on a boundary
        total = {t: sum(-(-n // 64) * 64 for n, k in zip(sizes, kind) if k == t) for t in ("bf16", "fp32")}
        rms = case["norm"] / math.sqrt(sum(sizes))
        s["flat"] = {t: randn(n, scale=rms, dtype=TYPES[t]) for t, n in total.items()}
        s["clipped"] = {t: torch.zeros_like(x) for t, x in s["flat"].items()}
        at, s["grads"], s["outs"] = {"bf16": 0, "fp32": 0}, [], []
        for n, k in zip(sizes, kind):
            s["grads"].append(s["flat"][k][at[k]:at[k] + n])
            s["outs"].append(s["clipped"][k][at[k]:at[k] + n])
            at[k] += -(-n // 64) * 64
    return s


# ------------------------------------------------------------------------------ one pass
def run(s):
    return {"attn": _run_attn, "embed": _run_embed, "clip": _run_clip}[s["op"]](s)


def _run_attn(s):
    if own:
        from femtotron_b200.ops import masked_attention as MA
        mask = s.get("mask")
        if mask is None:
            mask = MA.attention_mask(s["B"], s["S"], causal=s["causal"], window=s["window"] or None, docs=s["docs"],
                                     prefix=s["marks"], device="cuda")
        if not s["grad"]:
            with torch.no_grad():
                return MA.masked_attention(s["q"], s["k"], s["v"], mask, softcap=s["cap"], slopes=s["slopes"])
        o = MA.masked_attention(s["q"], s["k"], s["v"], mask, softcap=s["cap"], slopes=s["slopes"])
        return [o.detach(), *torch.autograd.grad(o, [s["q"], s["k"], s["v"]], s["do"])]
    with torch.no_grad():
        return _plain_attn(s)


def _visible(s):
    """[B or 1, S, S]: whether row i sees column j."""
    S = s["S"]
    i = torch.arange(S, device="cuda")
    first, end = torch.zeros(1, S, dtype=torch.long, device="cuda"), torch.full((1, S), S, device="cuda")
    alive = None
    if s["docs"] is not None:
        docs = s["docs"].long()
        new = torch.ones_like(docs, dtype=torch.bool)
        new[:, 1:] = docs[:, 1:] != docs[:, :-1]
        first = torch.where(new, i, torch.zeros_like(i)).cummax(1).values
        last = torch.ones_like(new)
        last[:, :-1] = new[:, 1:]
        end = torch.where(last, i + 1, torch.full_like(i, S)).flip(1).cummin(1).values.flip(1)
        alive = docs >= 0
    hi = end
    if s["causal"]:
        hi = (i + 1)[None]
        if s["marks"] is not None:
            stop = torch.where(s["marks"], torch.full_like(i, S), i).flip(1).cummin(1).values.flip(1)
            hi = torch.maximum(hi, torch.minimum(stop.gather(1, first.expand_as(stop)), end))
    vis = (i >= first[..., None]) & (i < hi[..., None])
    if s["window"]:
        vis &= (i[:, None] - i[None]).abs() < s["window"]
    return vis if alive is None else vis & alive[..., None]


def _plain_attn(s):
    B, S, nq, nkv, d = (s[k] for k in ("B", "S", "nq", "nkv", "d"))
    n, scale = nq // nkv, 1.0 / math.sqrt(d)

    def heads(x):  # [B, S, h, d] -> [B, nkv, (h / nkv) S, d]
        return x.float().view(B, S, nkv, -1, d).permute(0, 2, 3, 1, 4).reshape(B, nkv, -1, d)

    def back(x, h):
        return x.view(B, nkv, h // nkv, S, d).permute(0, 3, 1, 2, 4).reshape(B, S, h, d).to(torch.bfloat16)
    q, k, v = heads(s["q"]), heads(s["k"]), heads(s["v"])
    x = (q @ k.transpose(-1, -2)).mul_(scale).view(B, nkv, n, S, S)
    slope = None
    if s["cap"]:
        t = torch.tanh(x.mul_(1.0 / s["cap"]))
        slope = 1 - t * t
        x = t.mul_(s["cap"])
    if s["slopes"] is not None:
        i = torch.arange(S, device="cuda")
        x -= s["slopes"].view(nkv, n, 1, 1) * (i[:, None] - i[None]).abs().float()
    x = x.masked_fill_(~_visible(s)[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = x.sub_(top.masked_fill(top == float("-inf"), 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(total.masked_fill(total == 0, 1.0)).view(B, nkv, n * S, S)
    o = p @ v
    if not s["grad"]:
        return back(o, nq)
    do = heads(s["do"])
    dv = p.transpose(-1, -2) @ do
    ds = do @ v.transpose(-1, -2)
    ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if slope is not None:
        ds = ds.mul_(slope.view_as(ds))
    dq, dk = (ds @ k).mul_(scale), (ds.transpose(-1, -2) @ q).mul_(scale)
    return [back(o, nq), back(dq, nq), back(dk, nkv), back(dv, nkv)]


def _run_embed(s):
    w, into = s["weight"], s["into"]
    if own:
        from femtotron_b200.ops import functional as FN
        outs = []
        w.grad = None
        if into is not None:
            w.main_grad, w.grad_overwrite = into, True
        for ids, dout in zip(s["ids"], s["dout"]):
            out = FN.embedding(ids, w, scale=s["scale"], vstart=s["vstart"])
            out.backward(dout)
            outs.append(out.detach())
        return [outs, into if into is not None else w.grad]
    with torch.no_grad():
        V, H = w.shape
        local = s["ids"] - s["vstart"]
        has = (local >= 0) & (local < V)
        rows = torch.where(has, local, torch.zeros_like(local))
        out = (w[rows].float() * s["scale"] * has[..., None]).to(w.dtype)
        dw = into.zero_() if into is not None else torch.zeros(V, H, device="cuda")
        dw.index_add_(0, rows.view(-1), (s["dout"].float() * has[..., None]).view(-1, H)).mul_(s["scale"])
        return [list(out), dw if into is not None else dw.to(w.dtype)]


MAX_NORM = 1.0


def _run_clip(s):
    if own:
        from femtotron_b200.ops import grad_norm as GN
        norm = GN.clip_grads(s["grads"], MAX_NORM, out=s["outs"])
    else:
        norm = torch.stack([x.float().square().sum(dtype=torch.float64) for x in s["grads"]]).sum().sqrt().float()
        coef = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
        [o.copy_(x.float() * coef) for o, x in zip(s["outs"], s["grads"])]
    return [norm, s["clipped"]]


# ------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "attn":
        pairs = c["B"] * c["nq"] * _pairs(c)
        io = 2 * c["B"] * c["S"] * c["d"]
        ahead = io * (2 * c["nq"] + 2 * c["nkv"])
        if not c["grad"]:
            return {"bytes": ahead, "flops": 4 * c["d"] * pairs}
        # q, k, v, o and its gradient read, three gradients written; five more products
        return {"bytes": ahead + io * (4 * c["nq"] + 4 * c["nkv"]), "flops": 14 * c["d"] * pairs}
    if c["op"] == "embed":
        here = c["T"] * c["micro"] / c["shard"]
        rows = 2 * c["micro"] * c["T"] * c["H"]
        out = c["V"] * c["H"] * (4 if c["grad"] == "fp32" else 2)
        return {"bytes": int(8 * c["T"] * c["micro"] + 2 * here * c["H"] + rows + rows / c["shard"] + out),
                "flops": int(2 * here * c["H"])}
    n = sum(_grad_sizes(c))
    size = {"fp32": 4, "bf16": 2, "mixed": 8 / 3}[c["dtype"]]
    # the norm has to be known before the first gradient is scaled: read twice, written once
    return {"bytes": int(3 * size * n), "flops": 3 * n}


def _pairs(c):
    """About how many keys the rows of one sequence see in all."""
    S = c["S"]
    i = np.arange(S, dtype=np.float64)
    mean = float(c["doc"] or 1e12)
    w = float(c["window"] or 1e12)

    def reach(n):  # rows apart by less than n that a document holds together
        return -mean * np.expm1(-np.minimum(n, w) / mean)
    seen = reach(i + 1).sum()
    if not c["causal"]:
        seen += reach(S - 1 - i).sum()
    elif c["prefix"]:
        e = min(c["prefix"], 0.5) * S
        seen += reach(np.maximum(0.0, e - i)).sum()
    return max(1, int(seen * (1 - c["pad"] / 2) ** 2))


# ------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    keep, globals()["own"] = own, False
    s = prepare(case, seed)
    globals()["own"] = keep
    with torch.no_grad():
        if s["op"] == "attn":
            return _exact_attn(s)
        if s["op"] == "embed":
            return _exact_embed(s)
        total = sum(float(g.double().square().sum()) for g in s["grads"])
        norm = math.sqrt(total)
        coef = min(1.0, MAX_NORM / (norm + 1e-6))
        clipped = {t: torch.zeros_like(x, dtype=torch.float64) for t, x in s["flat"].items()}
        at = {torch.bfloat16: 0, torch.float32: 0}
        for x in s["grads"]:
            to = clipped["bf16" if x.dtype == torch.bfloat16 else "fp32"]
            to[at[x.dtype]:at[x.dtype] + x.numel()] = x.double() * coef
            at[x.dtype] += -(-x.numel() // 64) * 64
        return [torch.tensor(norm, dtype=torch.float64), clipped]


def _exact_attn(s):
    B, S, nq, nkv, d = (s[k] for k in ("B", "S", "nq", "nkv", "d"))
    o, dq, dk, dv = (torch.zeros(B, S, h, d, dtype=torch.float64, device="cuda") for h in (nq, nq, nkv, nkv))
    pos = torch.arange(S, device="cuda")
    far = (pos[:, None] - pos[None, :]).abs()
    for b in range(B):
        ok = torch.ones(S, S, dtype=torch.bool, device="cuda")
        run_of = torch.zeros(S, dtype=torch.long, device="cuda")
        if s["docs"] is not None:
            docs = s["docs"][b].long()
            run_of[1:] = (docs.diff() != 0).cumsum(0)
            ok &= (run_of[:, None] == run_of[None, :]) & (docs >= 0)[:, None]
        if s["causal"]:
            ahead = torch.zeros(S, dtype=torch.bool, device="cuda")
            if s["marks"] is not None:  # marked, as is all of the document before it
                plain = (~s["marks"][b]).long().cumsum(0)
                begin = torch.searchsorted(run_of, run_of)
                before = torch.where(begin > 0, plain[(begin - 1).clamp(min=0)], torch.zeros_like(plain))
                ahead = plain == before
            ok &= (pos[None, :] <= pos[:, None]) | ahead[None, :]
        if s["window"]:
            ok &= far < s["window"]
        for h in range(nq):
            g = h * nkv // nq
            qh, kh, vh = s["q"][b, :, h].double(), s["k"][b, :, g].double(), s["v"][b, :, g].double()
            x = qh @ kh.T / math.sqrt(d)
            if s["cap"]:
                t = torch.tanh(x / s["cap"])
                x = s["cap"] * t
            if s["slopes"] is not None:
                x = x - s["slopes"][h].double() * far
            x = torch.where(ok, x, torch.full_like(x, -math.inf))
            lse = torch.logsumexp(x, -1, keepdim=True)
            p = torch.where(ok, torch.exp(x - lse), torch.zeros_like(x))
            o[b, :, h] = p @ vh
            if s["grad"]:
                doh = s["do"][b, :, h].double()
                dp = doh @ vh.T
                ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                if s["cap"]:
                    ds = ds * (1 - t * t)
                dq[b, :, h] = ds @ kh / math.sqrt(d)
                dk[b, :, g] += ds.T @ qh / math.sqrt(d)
                dv[b, :, g] += p.T @ doh
    return [o, dq, dk, dv] if s["grad"] else o


def _exact_embed(s):
    V, H = s["weight"].shape
    outs, dw = [], torch.zeros(V, H, dtype=torch.float64, device="cuda")
    for ids, dout in zip(s["ids"], s["dout"]):
        here = torch.nonzero((ids >= s["vstart"]) & (ids < s["vstart"] + V))[:, 0]
        out = torch.zeros(ids.numel(), H, dtype=torch.float64, device="cuda")
        out[here] = s["weight"][ids[here] - s["vstart"]].double() * s["scale"]
        outs.append(out)
        dw.index_put_((ids[here] - s["vstart"],), dout[here].double() * s["scale"], accumulate=True)
    return [outs, dw]
