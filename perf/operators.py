"""The operators around the attention of a decode step, as cases to be measured.

* ``norm``   -- residual addition + RMS norm, with a float or an 8-bit output (``add_rmsnorm``).
* ``w4``     -- products with 4-bit weights and group scales (``W4Weights``).
* ``verify`` -- drafted tokens checked against the target's probabilities (``verify_drafts``).

``own`` false: the operators' plain forms in elementary torch operations. True: the framework's calls.
"""
import torch

own = False

HIDDEN = 2048      # the model's hidden size (bench.py's configurations)
VOCAB = 128000     # rows of its logits head
EPS = 1e-5


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a decode step: residual stream in f32, 8-bit output in the K-quant products' 256-wide blocks
        dict(name="norm one token", op="norm", rows=1, n=HIDDEN, dtype="f32", out="int8", group=256, residual=True),
        # a long prompt in bf16 between two layers
        dict(name="norm prompt bf16", op="norm", rows=8192, n=HIDDEN, dtype="bf16", out="bf16", group=0, residual=True),
        # a ragged batch of another width: f32, no residual, 8-bit rows with one scale each
        dict(name="norm odd rows", op="norm", rows=1037, n=2080, dtype="f32", out="int8", group=0, residual=False),
        # one token through a hidden x hidden projection
        dict(name="w4 one token", op="w4", tokens=1, n_in=HIDDEN, n_out=2048, group=32, x="f32", x_group=0, y="f32",
             scales="f16", zeros=False),
        # five rows of a speculative step through the logits head, from 8-bit activations
        dict(name="w4 head 5 rows", op="w4", tokens=5, n_in=HIDDEN, n_out=VOCAB, group=128, x="int8", x_group=256, y="f32",
             scales="f16", zeros=False),
        # one token through a large layer with zero points
        dict(name="w4 large layer", op="w4", tokens=1, n_in=8192, n_out=8192, group=128, x="bf16", x_group=0, y="bf16",
             scales="bf16", zeros=True),
        # a batch of 24 sequences, odd sizes
        dict(name="w4 batch odd", op="w4", tokens=24, n_in=2080, n_out=5003, group=32, x="f32", x_group=0, y="f32",
             scales="f16", zeros=True),
        # a prompt chunk through a wide projection
        dict(name="w4 prompt bf16", op="w4", tokens=2048, n_in=HIDDEN, n_out=8192, group=128, x="bf16", x_group=0, y="bf16",
             scales="f16", zeros=True),
        # a ragged prompt chunk with the residual stream's f32 values
        dict(name="w4 prompt f32", op="w4", tokens=777, n_in=HIDDEN, n_out=2048, group=64, x="f32", x_group=0, y="f32",
             scales="bf16", zeros=False),
        # one conversation, four drafted tokens
        dict(name="verify one", op="verify", seqs=1, drafts=4, vocab=VOCAB, temperature=0.75, probs=False, draft_rows=True),
        # a serving batch
        dict(name="verify batch", op="verify", seqs=64, drafts=8, vocab=VOCAB, temperature=1.0, probs=False, draft_rows=True),
        # probabilities in hand, an odd vocabulary, drafts looked up in the text (no rows of their own)
        dict(name="verify looked up", op="verify", seqs=24, drafts=5, vocab=32003, temperature=1.0, probs=True, draft_rows=False),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(("norm", "w4", "w4", "verify"))
    if op == "norm":
        n = _log(rng, 32, 8192)
        rows = _log(rng, 1, max(1, min(8192, 8192 * HIDDEN // n)))
        out = rng.choice(("same", "int8"))
        group = 0
        if out == "int8":
            group = rng.choice((0, 32, 64, 128, 256))
            step = group or 32
            n = max(step, n // step * step)
        dtype = rng.choice(("f32", "bf16"))
        return dict(op="norm", rows=rows, n=n, dtype=dtype, out=dtype if out == "same" else out, group=group,
                    residual=rng.random() < 0.7)
    if op == "w4":
        group = rng.choice((32, 64, 128, 256))
        n_in = group * max(1, _log(rng, 256, 8192) // group)
        n_out = min(_log(rng, 64, VOCAB), VOCAB * HIDDEN // n_in)
        tokens = min(_log(rng, 1, 2048), max(1, 2048 * HIDDEN * 8192 // (n_in * n_out)))
        x = rng.choice(("f32", "bf16", "int8"))
        x_group = rng.choice((0, group)) if x == "int8" else 0
        return dict(op="w4", tokens=tokens, n_in=n_in, n_out=n_out, group=group, x=x, x_group=x_group,
                    y="bf16" if x == "bf16" else "f32", scales=rng.choice(("f16", "bf16")), zeros=rng.random() < 0.5)
    drafts = rng.randint(1, 8)
    vocab = _log(rng, 500, VOCAB)
    seqs = _log(rng, 1, 64)
    probs = rng.random() < 0.3
    temperature = 1.0 if probs else rng.choice((0.0, 0.5, 0.75, 1.0, 1.25))
    return dict(op="verify", seqs=seqs, drafts=drafts, vocab=vocab, temperature=temperature, probs=probs,
                draft_rows=rng.random() < 0.75)


# --------------------------------------------------------------------------- inputs
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _norm_inputs(case, seed):
    g = _gen(seed)
    rows, n, dt = case["rows"], case["n"], _TYPES[case["dtype"]]
    # a residual stream: unit-scale rows with a few channels far larger than the rest
    chan = torch.exp(0.5 * torch.randn(n, device="cuda", generator=g))
    x = (torch.randn(rows, n, device="cuda", generator=g) * chan).to(dt)
    res = (torch.randn(rows, n, device="cuda", generator=g) * chan * 2).to(dt) if case["residual"] else None
    gain = 1 + 0.1 * torch.randn(n, device="cuda", generator=g)
    return x, res, gain


def _w4_inputs(case, seed):
    g = _gen(seed)
    t, k, n, gs = case["tokens"], case["n_in"], case["n_out"], case["group"]
    # rounded normal weights: most codes near the middle of the range
    c = torch.randn(n, k, device="cuda", generator=g).mul_(2.8).add_(8).round_().clamp_(0, 15).to(torch.uint8)
    codes = c[:, 0::2] | (c[:, 1::2] << 4)
    del c
    scales = (0.01 * torch.exp(0.3 * torch.randn(n, k // gs, device="cuda", generator=g))).to(_TYPES[case["scales"]])
    zeros = torch.randint(5, 12, (n, k // gs), device="cuda", generator=g, dtype=torch.uint8) if case["zeros"] else None
    if case["x"] == "int8":
        x = torch.randn(t, k, device="cuda", generator=g).mul_(32).round_().clamp_(-127, 127).to(torch.int8)
        ng = k // case["x_group"] if case["x_group"] else 1
        xs = 0.03 * torch.exp(0.3 * torch.randn(t, ng, device="cuda", generator=g))
    else:
        x, xs = torch.randn(t, k, device="cuda", generator=g).to(_TYPES[case["x"]]), None
    return codes.contiguous(), scales, zeros, x, xs


def _verify_inputs(case, seed):
    g = _gen(seed)
    b, d, v, temp = case["seqs"], case["drafts"], case["vocab"], case["temperature"]
    target = torch.randn(b, d + 1, v, device="cuda", generator=g).mul_(2.5)
    # the drafting model's logits follow the target's
    draft = target[:, :d] + 0.5 * torch.randn(b, d, v, device="cuda", generator=g)
    noise = torch.rand(b, d, v, device="cuda", generator=g).clamp_(1e-20, 1 - 1e-7)
    tokens = (draft / (temp or 1.0) - torch.log(-torch.log(noise))).argmax(-1).to(torch.int32)
    if temp == 0.0:
        tokens = draft.argmax(-1).to(torch.int32)
    del noise
    if case["probs"]:
        target, draft = torch.softmax(target, -1), torch.softmax(draft, -1)
    u = torch.rand(b, d, device="cuda", generator=g)
    u_sample = torch.rand(b, device="cuda", generator=g)
    n_drafts = torch.randint(0, d + 1, (b,), device="cuda", generator=g, dtype=torch.int32)
    n_drafts = torch.where(torch.rand(b, device="cuda", generator=g) < 0.8, torch.full_like(n_drafts, d), n_drafts)
    return target, (draft if case["draft_rows"] else None), tokens, n_drafts, u, u_sample


def prepare(case, seed):
    s = dict(case=case)
    if case["op"] == "norm":
        x, res, gain = _norm_inputs(case, seed)
        rows, n = case["rows"], case["n"]
        s.update(x=x, res=res, gain=gain, sum=torch.empty_like(x) if res is not None else None)
        if case["out"] == "int8":
            s["out"] = torch.empty(rows, n, dtype=torch.int8, device="cuda")
            s["scales"] = torch.empty(rows, n // (case["group"] or n), dtype=torch.float32, device="cuda")
        else:
            s["out"] = torch.empty(rows, n, dtype=_TYPES[case["out"]], device="cuda")
    elif case["op"] == "w4":
        codes, scales, zeros, x, xs = _w4_inputs(case, seed)
        s.update(codes=codes, scales=scales, zeros=zeros, x=x, xs=xs,
                 out=torch.empty(case["tokens"], case["n_out"], dtype=_TYPES[case["y"]], device="cuda"))
        if own:  # the weights' handle that a program keeps
            import bebelm_b200 as bb
            s["w"] = bb.W4Weights(codes, scales, zeros, group=case["group"])
    else:
        names = ("target", "draft", "tokens", "n_drafts", "u", "u_sample")
        s.update(zip(names, _verify_inputs(case, seed)))
        s["out"] = torch.empty(case["seqs"], case["drafts"] + 1, dtype=torch.int32, device="cuda")
        s["accepted"] = torch.empty(case["seqs"], dtype=torch.int32, device="cuda")
    return s


# --------------------------------------------------------------------------- the framework's calls
def _own_norm(s):
    import bebelm_b200 as bb
    case = s["case"]
    if case["out"] == "int8":
        q, scales, _ = bb.add_rmsnorm(s["x"], s["gain"], s["res"], EPS, out_dtype=bb.INT8, group=case["group"], out=s["out"],
                                      scales=s["scales"], sum_out=s["sum"])
        rows, ng = scales.shape  # what the 8 bits stand for
        return dict(y=torch.mul(q.view(rows, ng, -1), scales.view(rows, ng, 1)).view(rows, -1), scales=scales, h=s["sum"])
    y, _ = bb.add_rmsnorm(s["x"], s["gain"], s["res"], EPS, out=s["out"], sum_out=s["sum"])
    return dict(y=y, h=s["sum"])


def _own_w4(s):
    return s["w"].matmul(s["x"], s["xs"], out=s["out"])


def _own_verify(s):
    import bebelm_b200 as bb
    case = s["case"]
    tokens, accepted = bb.verify_drafts(s["target"], s["tokens"], s["u"], s["u_sample"], draft=s["draft"],
                                        n_drafts=s["n_drafts"], temperature=case["temperature"], probs=case["probs"],
                                        out=s["out"], accepted=s["accepted"])
    return dict(tokens=tokens, accepted=accepted)


# --------------------------------------------------------------------------- plain forms
def _plain_norm(s):
    """The definition's own steps, each rounded to f32 where it says so."""
    case, x, res = s["case"], s["x"], s["res"]
    h = x if res is None else (x.float() + res.float()).to(x.dtype)
    hf = h.float()
    ss = (hf * hf).double().sum(-1, keepdim=True)
    mean = (ss / torch.full_like(ss, case["n"])).float()
    r = torch.sqrt(mean + EPS).reciprocal()
    t = (hf * r) * s["gain"]
    out = dict(h=None if res is None else h)
    if case["out"] != "int8":
        return dict(out, y=t.to(_TYPES[case["out"]]))
    rows, n = t.shape
    t = t.view(rows, -1, case["group"] or n)
    a = t.abs().amax(-1, keepdim=True)
    c127 = torch.full_like(a, 127.0)
    inv = torch.where(a > 0, c127 / a, torch.zeros_like(a))
    z = t * inv
    whole = torch.trunc(z)
    q = (whole + torch.sign(z) * ((z - whole).abs() >= 0.5)).clamp(-127, 127)
    scales = a / c127
    return dict(out, y=(q * scales).view(rows, n), scales=scales.view(rows, -1))


def _plain_w4(s):
    case, codes = s["case"], s["codes"]
    n, k, g = case["n_out"], case["n_in"], case["group"]
    c = torch.stack((codes & 15, codes >> 4), -1).view(n, k // g, g).float()
    z = s["zeros"].float()[..., None] if s["zeros"] is not None else 8.0
    w = ((c - z) * s["scales"].float()[..., None]).view(n, k)
    x = s["x"].float()
    if s["xs"] is not None:
        x = (x.view(x.shape[0], s["xs"].shape[1], -1) * s["xs"][..., None]).view(x.shape[0], k)
    return (x @ w.t()).to(_TYPES[case["y"]])


def _plain_verify(s):
    """In 64 bits: a token is the place where a sum over the vocabulary passes a border."""
    case, tokens, lens = s["case"], s["tokens"].long(), s["n_drafts"].long()
    b, d, v, temp = case["seqs"], case["drafts"], case["vocab"], case["temperature"]
    at = torch.arange(d, device="cuda")
    if temp == 0.0:
        best = s["target"].argmax(-1)
        ok = best[:, :d] == tokens
    else:
        p, q = s["target"].double(), None if s["draft"] is None else s["draft"].double()
        if not case["probs"]:
            p = torch.exp((p - p.amax(-1, keepdim=True)) / temp)
            p = p / p.sum(-1, keepdim=True)
            if q is not None:
                q = torch.exp((q - q.amax(-1, keepdim=True)) / temp)
                q = q / q.sum(-1, keepdim=True)
        px = p[:, :d].gather(-1, tokens[..., None])[..., 0]
        qx = torch.ones_like(px) if q is None else q.gather(-1, tokens[..., None])[..., 0]
        ok = s["u"].double() * qx < px
    ok = ok & (at < lens[:, None])
    a = torch.cumprod(ok.long(), -1).sum(-1)
    rows = torch.arange(b, device="cuda")
    if temp == 0.0:
        nxt = best[rows, a]
    else:
        pr, last = p[rows, a], (a == lens)
        i = a.clamp(max=d - 1)
        if q is None:
            qr = torch.zeros_like(pr).scatter_(1, tokens[rows, i][:, None], float("inf"))
        else:
            qr = q[rows, i]
        w = torch.where(last[:, None], pr, (pr - qr).clamp(min=0))
        w = torch.where(w.sum(-1, keepdim=True) > 0, w, pr)
        cum = torch.cumsum(w, -1)
        nxt = (cum <= s["u_sample"].double()[:, None] * cum[:, -1:]).sum(-1).clamp(max=v - 1)
    every = torch.arange(d + 1, device="cuda")
    given = torch.cat((tokens, torch.full((b, 1), -1, device="cuda")), 1)
    out = torch.where(every < a[:, None], given, torch.where(every == a[:, None], nxt[:, None], -1))
    return dict(tokens=out.int(), accepted=a.int())


def run(state):
    op = state["case"]["op"]
    if own:
        return _own_norm(state) if op == "norm" else _own_w4(state) if op == "w4" else _own_verify(state)
    return _plain_norm(state) if op == "norm" else _plain_w4(state) if op == "w4" else _plain_verify(state)


# --------------------------------------------------------------------------- work and exact values
def work(case):
    if case["op"] == "norm":
        e = 2 if case["dtype"] == "bf16" else 4
        m = case["rows"] * case["n"]
        o = 1 if case["out"] == "int8" else 2 if case["out"] == "bf16" else 4
        scales = 4 * case["rows"] * (case["n"] // (case["group"] or case["n"])) if case["out"] == "int8" else 0
        return dict(bytes=m * (e * (3 if case["residual"] else 1) + o) + 4 * case["n"] + scales, flops=6 * m)
    if case["op"] == "w4":
        t, k, n, g = case["tokens"], case["n_in"], case["n_out"], case["group"]
        xb = {"f32": 4, "bf16": 2, "int8": 1}[case["x"]]
        xs = 4 * t * (k // case["x_group"] if case["x_group"] else 1) if case["x"] == "int8" else 0
        yb = 2 if case["y"] == "bf16" else 4
        return dict(bytes=n * k // 2 + n * (k // g) * (3 if case["zeros"] else 2) + t * k * xb + xs + t * n * yb,
                    flops=2 * t * k * n)
    rows = case["seqs"] * (case["drafts"] + 1 + (case["drafts"] if case["draft_rows"] else 0))
    if case["probs"]:  # single entries decide; one row (two with draft rows) of each sequence is summed
        rows = case["seqs"] * (2 if case["draft_rows"] else 1)
    if case["temperature"] == 0.0:
        rows = case["seqs"] * (case["drafts"] + 1)
    return dict(bytes=4 * rows * case["vocab"] + case["seqs"] * (case["drafts"] * 12 + 16), flops=4 * rows * case["vocab"])


def exact(case, seed):
    if case["op"] == "norm":
        return _exact_norm(case, seed)
    if case["op"] == "w4":
        return _exact_w4(case, seed)
    return None  # tokens and counts: no computed numbers among the outputs


def _exact_norm(case, seed):
    x, res, gain = _norm_inputs(case, seed)
    total = x.double() if res is None else x.double().add_(res.double())
    h = total.to(x.dtype).double()  # the stream is kept in its own type: that rounding is part of the definition
    if case["out"] != "int8":
        y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * gain.double()
        return dict(y=y, h=None if res is None else total)
    # 8-bit codes: the definition rounds to f32 at these places, which decides a code next to a border
    def f32(v):
        return v.float().double()
    eps = float(torch.tensor(EPS, dtype=torch.float32))
    mean = f32(f32(h.square()).sum(-1, keepdim=True) / case["n"])
    r = f32(1.0 / f32(torch.sqrt(f32(mean + eps))))
    t = f32(f32(h * r) * gain.double()).unflatten(1, (-1, case["group"] or case["n"]))
    a = t.abs().max(-1, keepdim=True).values
    z = f32(t * torch.nan_to_num(f32(127.0 / a), posinf=0.0))
    codes = torch.copysign(torch.floor(z.abs() + 0.5), z).clamp(-127, 127)
    return dict(y=(codes * (a / 127.0)).flatten(1), scales=(a / 127.0).flatten(1), h=None if res is None else total)


def _exact_w4(case, seed):
    codes, scales, zeros, x, xs = _w4_inputs(case, seed)
    n, k, g = case["n_out"], case["n_in"], case["group"]
    w = torch.empty(n, k, dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = codes.bitwise_and(0xF), codes.bitwise_right_shift(4)
    w -= 8.0 if zeros is None else zeros.double().repeat_interleave(g, 1)
    w *= scales.double().repeat_interleave(g, 1)
    x = x.double()
    if xs is not None:
        x = x * xs.double().repeat_interleave(k // xs.shape[1], 1)
    return torch.einsum("tk,nk->tn", x, w)
