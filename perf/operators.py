"""The low-bit decode step's operators, as cases that can be timed and compared: linears of a few rows with 4-bit weights, the e4m3
key/value cache (written, and read back by the attention of one token or of a tree of drafted tokens), and the logits' penalties, biases
and masks.  Sizes are those of the text encoder that the prompt prologue decodes with (hidden 3584, 28 query and 4 key/value heads of 128,
gated MLP 18944, vocabulary 152064), of smaller language models, and odd ones."""
import math

import torch

own = False

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
TINY = 2.0 ** -126            # the smallest scale of a cache row: the smallest normal number of 32 bits
EPS = 1e-6


def listed():
    return [
        # q / k / v projection of the decode step, input norm in the same launch: the shortest linear, where latency counts
        dict(name="linear_qkv_1", op="linear", m=1, n=4608, k=3584, group=128, zero=True, norm=True, bias=True, res=False, swiglu=False),
        # gate and up projection of the gated MLP for one token: the bulk of a decoder layer's weights
        dict(name="linear_gate_up_1", op="linear", m=1, n=37888, k=3584, group=128, zero=True, norm=True, bias=False, res=False, swiglu=True),
        # down projection onto the residual rows of seven drafted tokens, finer groups
        dict(name="linear_down_7", op="linear", m=7, n=3584, k=18944, group=64, zero=True, norm=False, bias=False, res=True, swiglu=False),
        # odd rows, odd outputs, a depth that is no multiple of 128, smallest groups, no zero points: a batch of 33 requests
        dict(name="linear_odd_33", op="linear", m=33, n=5001, k=3424, group=32, zero=False, norm=False, bias=True, res=False, swiglu=False),
        # one new token of the decode step: queries rotated, key and value quantised into the cache
        dict(name="append_1", op="append", b=1, t=1, hq=28, hkv=4, d=128, start=1100, cap=1536),
        # three prompts of a padded batch written at different places
        dict(name="append_prompts", op="append", b=3, t=1111, hq=28, hkv=4, d=128, start=401, cap=2368),
        # attention of the decode step in the middle of an answer
        dict(name="attention_1", op="attention", b=1, t=1, hq=28, hkv=4, d=128, rows=1500, cap=2048),
        # the longest cache that the decode step takes
        dict(name="attention_long", op="attention", b=1, t=1, hq=28, hkv=4, d=128, rows=15359, cap=15360),
        # a tree of 21 drafted tokens over three ragged contexts, the last one empty
        dict(name="attention_tree", op="attention", b=3, t=21, hq=28, hkv=4, d=128, rows=2777, cap=3136),
        # a batch of requests with heads of 64 and long ragged contexts: the most bytes
        dict(name="attention_batch", op="attention", b=24, t=1, hq=16, hkv=8, d=64, rows=40001, cap=40064),
        # greedy choice of the decode step's next token under a repetition penalty and a mask of allowed tokens
        dict(name="select_1", op="logits", rows=1, vocab=152064, half=True, counts=True, bias=False, mask=True, select=True),
        # processed scores of a batch of requests, for a sampler: every term
        dict(name="process_48", op="logits", rows=48, vocab=151937, half=False, counts=True, bias=True, mask=True, select=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "append", "attention", "logits"])
    if op == "linear":
        group, swiglu = rng.choice([32, 64, 128]), rng.random() < 0.25
        k = max(1, _log(rng, 64, 18944) // group) * group
        n = min(_log(rng, 16, 40000), 120_000_000 // k)
        n = max(n // 32, 1) * 32 if swiglu else n
        return dict(op=op, m=_log(rng, 1, 64), n=n, k=k, group=group, zero=rng.random() < 0.6, norm=rng.random() < 0.4, bias=rng.random() < 0.4,
                    res=rng.random() < 0.4 and not swiglu, swiglu=swiglu)
    hq, hkv = rng.choice([(28, 4), (16, 8), (8, 8), (5, 1), (12, 2)])
    d = rng.choice([64, 128])
    if op == "append":
        t = _log(rng, 1, 1500)
        start = rng.randrange(0, 1000)
        return dict(op=op, b=rng.randrange(1, 4), t=t, hq=hq, hkv=hkv, d=d, start=start, cap=(start + t + 63 + rng.randrange(0, 200)) // 64 * 64)
    if op == "attention":
        t = 1 if rng.random() < 0.5 else _log(rng, 2, 64)
        b = _log(rng, 1, 16)
        rows = min(_log(rng, 1, 40000), 150_000_000 // (b * hkv * d * (2 if t == 1 else 8)))
        return dict(op=op, b=b, t=t, hq=hq, hkv=hkv, d=d, rows=rows, cap=(rows + t + 63) // 64 * 64)
    return dict(op=op, rows=_log(rng, 1, 48), vocab=_log(rng, 300, 152064), half=rng.random() < 0.5, counts=rng.random() < 0.8, bias=rng.random() < 0.5,
                mask=rng.random() < 0.7, select=rng.random() < 0.5)


# ---- inputs ---------------------------------------------------------------------------------------------------------------------

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _linear_inputs(c, g):
    """codes two to a byte (even element low) with a bell-shaped histogram, scales of weights of about 0.02, rows with a few large channels"""
    groups = c["k"] // c["group"]
    low, high = ((_randn(g, c["n"], c["k"] // 2) * 2.7 + 7.5).round_().clamp_(0, 15).to(torch.uint8) for _ in range(2))
    x = _randn(g, c["m"], c["k"])
    x[:, torch.randint(0, c["k"], (8,), generator=g, device="cuda")] *= 12
    d = dict(codes=low | (high << 4), scale=(0.007 * torch.exp(0.3 * _randn(g, c["n"], groups))).to(BF), x=x.to(BF),
             zero=(_randn(g, c["n"], groups) * 1.2 + 7.5).round_().clamp_(0, 15).to(torch.uint8) if c["zero"] else None,
             bias=_randn(g, c["n"]).to(BF) if c["bias"] else None, res=_randn(g, c["m"], c["n"]).to(BF) if c["res"] else None)
    return d


def _rotary(c, g):
    angle = torch.arange(c["cap"], device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, c["d"], 2, device="cuda", dtype=torch.float64) / c["d"])
    angle = torch.cat([angle, angle], dim=1)
    return dict(cos=angle.cos().to(BF), sin=angle.sin().to(BF))


def _starts(c, rows):
    """context rows of each sequence: ragged, from `rows` down to none for the last one of a batch"""
    b = torch.arange(c["b"], device="cuda", dtype=torch.int64)
    return (rows * (c["b"] - 1 - b) // max(c["b"] - 1, 1) if c["b"] > 1 else rows + 0 * b).to(torch.int32)


def _append_inputs(c, g):
    """heads as a projection leaves them: side by side in one row per token; a channel or two of the keys far larger than the others"""
    qkv = _randn(g, c["b"], c["t"], c["hq"] + 2 * c["hkv"], c["d"])
    qkv[..., c["hq"]:c["hq"] + c["hkv"], 3] += 15
    return dict(qkv=qkv.to(BF), start=_starts(c, c["start"]), **_rotary(c, g))


def _cache_inputs(c, g):
    """a cache in hand: e4m3 codes and the scale of each (token, head), rows behind the last new token zero"""
    shape = c["b"], c["hkv"], c["cap"], c["d"]
    k, v = _randn(g, *shape).to(BF), (_randn(g, *shape) + 0.3 * _randn(g, shape[0], shape[1], 1, shape[3])).to(BF)
    start = _starts(c, c["rows"])
    here = (torch.arange(c["cap"], device="cuda") < start[:, None] + c["t"])[:, None, :, None]
    return dict(k=k * here, v=v * here, start=start, q=(1.5 * _randn(g, c["b"], c["t"], c["hq"], c["d"])).to(BF), tree=_tree(c, g) if c["t"] > 1 else None)


def _tree(c, g):
    """bit j of word i: drafted token i descends from drafted token j (or is it)"""
    i = torch.arange(c["t"], device="cuda")
    parent = (torch.rand((c["b"], c["t"]), generator=g, device="cuda") * i).long()
    up = torch.nn.functional.one_hot(parent, c["t"]).double() * (i > 0)[:, None] + torch.eye(c["t"], device="cuda", dtype=torch.float64)
    return ((torch.linalg.matrix_power(up, c["t"]) > 0.5).long() << i).sum(-1)


def _logits_inputs(c, g):
    """scores with a head of likely tokens; counts: bit 15 = in the prompt, below = how often generated; a mask that leaves about a third"""
    rows, vocab = c["rows"], c["vocab"]
    logits = (2.5 * _randn(g, rows, vocab)).to(BF if c["half"] else torch.float32)
    r = torch.rand((rows, vocab), generator=g, device="cuda")
    counts = ((r < 0.004) * (1 + (r * 1e6).long() % 5) + (r > 0.996) * -32768 + (r > 0.999) * 2).to(torch.int16)
    words = torch.randint(-2 ** 31, 2 ** 31, (2, rows, (vocab + 31) // 32), generator=g, device="cuda", dtype=torch.int64)
    return dict(logits=logits, counts=counts if c["counts"] else None,
                penalties=torch.tensor([[1.05, 0.3, 0.2]], device="cuda").expand(rows, 3).contiguous() if c["counts"] else None,
                bias=0.5 * _randn(g, vocab) if c["bias"] else None, allowed=(words[0] & words[1]).to(torch.int32) if c["mask"] else None)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"linear": _linear_inputs, "append": _append_inputs, "attention": _cache_inputs, "logits": _logits_inputs}[case["op"]](case, g)


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if case["op"] == "append":
        s |= _empty_cache(case)
    if case["op"] == "attention":
        s["kq"], s["ks"] = _quantise(s["k"].float())
        s["vq"], s["vs"] = _quantise(s["v"].float())
        if not own:
            s["k"] = s["v"] = None
    if own:
        return _prepare_own(case, s)
    return s


def _prepare_own(case, s):
    """what a program keeps: the weight in the library's layout, the cache object (filled by the library's own writes)"""
    from physicedit_amd import ops
    if case["op"] == "linear":
        s["w"] = ops.pack_w4(s["codes"], s["scale"], s["zero"], group=case["group"])
        s["codes"] = s["scale"] = s["zero"] = None
    if case["op"] in ("append", "attention"):
        s["cache"] = ops.KVCacheE4M3(case["b"], case["hkv"], case["cap"], case["d"], device="cuda")
    if case["op"] == "attention":
        ops.kv_append_e4m3(s["cache"], s["k"].transpose(1, 2), s["v"].transpose(1, 2), torch.zeros_like(s["start"]))
        s["k"] = s["v"] = s["kq"] = s["vq"] = None
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        return _run_own(c, s)
    return {"linear": _linear, "append": _append, "attention": _attention, "logits": _logits}[c["op"]](c, s)


def _run_own(c, s):
    from physicedit_amd import ops
    if c["op"] == "linear":
        return ops.gemv_w4(s["x"], s["w"], bias=s["bias"], res=s["res"], epilogue="swiglu" if c["swiglu"] else "bias", norm_eps=EPS if c["norm"] else None)
    if c["op"] == "append":
        q, k, v = s["qkv"].split([c["hq"], c["hkv"], c["hkv"]], dim=2)
        q = ops.kv_append_e4m3(s["cache"], k, v, s["start"], q=q, cos=s["cos"], sin=s["sin"])
        return dict(q=q, k=s["cache"].k, v=s["cache"].v, k_scale=s["cache"].k_scale, v_scale=s["cache"].v_scale)
    if c["op"] == "attention":
        return ops.kv_attention_e4m3(s["q"], s["cache"], s["start"], tree=s["tree"])
    if c["select"]:
        return ops.select_token(s["logits"], counts=s["counts"], penalties=s["penalties"], bias=s["bias"], allowed=s["allowed"])
    return ops.process_logits(s["logits"], counts=s["counts"], penalties=s["penalties"], bias=s["bias"], allowed=s["allowed"])


def _unpack(s):
    return torch.stack([s["codes"] & 15, s["codes"] >> 4], dim=-1).flatten(1)


def _linear(c, s):
    zero = 8.0 if s["zero"] is None else s["zero"].float()[:, :, None]
    w = (_unpack(s).view(c["n"], -1, c["group"]).float() - zero) * s["scale"].float()[:, :, None]
    x = s["x"].float()
    y = x @ w.view(c["n"], c["k"]).T
    if c["norm"]:
        y = y * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if c["swiglu"]:
        gate, up = y.chunk(2, dim=1)
        y = gate * torch.sigmoid(gate) * up
    if s["res"] is not None:
        y = y + s["res"].float()
    return y.to(BF)


def _empty_cache(c):
    shape = c["b"], c["hkv"], c["cap"], c["d"]
    return dict(kq=torch.zeros(shape, device="cuda").to(F8), vq=torch.zeros(shape, device="cuda").to(F8),
                ks=torch.zeros(shape[:3], device="cuda"), vs=torch.zeros(shape[:3], device="cuda"))


def _quantise(x):
    top = x.abs().amax(-1)
    scale = (top / 448).clamp_min(TINY).where(top.isfinite(), torch.full_like(top, math.nan))
    return torch.where(top.isfinite()[..., None], x / scale[..., None], torch.zeros_like(x)).to(F8), scale


def _rotate(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return x * cos + torch.cat([-b, a], dim=-1) * sin


def _append(c, s):
    q, k, v = s["qkv"].float().split([c["hq"], c["hkv"], c["hkv"]], dim=2)
    row = s["start"].long()[:, None] + torch.arange(c["t"], device="cuda")
    cos, sin = s["cos"].float()[row][:, :, None], s["sin"].float()[row][:, :, None]
    b = torch.arange(c["b"], device="cuda")[:, None]
    kq, ks = _quantise(_rotate(k, cos, sin))
    vq, vs = _quantise(v)
    s["kq"].view(torch.uint8)[b, :, row] = kq.view(torch.uint8)
    s["vq"].view(torch.uint8)[b, :, row] = vq.view(torch.uint8)
    s["ks"][b, :, row] = ks
    s["vs"][b, :, row] = vs
    return dict(q=_rotate(q, cos, sin).to(BF), k=s["kq"], v=s["vq"].view(c["b"], c["hkv"], c["cap"] // 64, 64, c["d"]), k_scale=s["ks"], v_scale=s["vs"])


def _visible(c, start, tree):
    """[b, t, cap]: what each new token attends to"""
    at = torch.arange(c["cap"], device="cuda")
    behind = at - start[:, None, None].long()
    bits = torch.ones((c["b"], c["t"]), dtype=torch.int64, device="cuda") if tree is None else tree
    return (behind < 0).expand(c["b"], c["t"], c["cap"]) | ((behind >= 0) & (behind < c["t"]) & ((bits[:, :, None] >> behind.clamp(0, 63)) & 1).bool())


def _attention(c, s):
    b, t, hkv, d = c["b"], c["t"], c["hkv"], c["d"]
    k, v = s["kq"].float() * s["ks"][..., None], s["vq"].float() * s["vs"][..., None]
    q = s["q"].float().view(b, t, hkv, -1, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    seen = _visible(c, s["start"], s["tree"])[:, None, None].expand(b, hkv, c["hq"] // hkv, t, c["cap"]).reshape(b, hkv, -1, c["cap"])
    score = (q @ k.transpose(2, 3) / math.sqrt(d)).masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.where(top.isfinite(), torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, p @ v / total, torch.zeros_like(total))
    return o.view(b, hkv, -1, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, c["hq"] * d).to(BF)


def _logits(c, s):
    x = s["logits"].float()
    if s["counts"] is not None:
        rep, presence, frequency = s["penalties"].unbind(1)
        made = (s["counts"] & 32767).float()
        x = torch.where(s["counts"] != 0, torch.where(x > 0, x / rep[:, None], x * rep[:, None]), x)
        x = x - frequency[:, None] * made - presence[:, None] * (made > 0)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["allowed"] is not None:
        at = torch.arange(c["vocab"], device="cuda")
        x = x.masked_fill(((s["allowed"][:, at // 32] >> (at % 32).int()) & 1) == 0, -math.inf)
    if c["select"]:
        return x.argmax(-1).to(torch.int32)
    return x


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------------

def work(c):
    if c["op"] == "linear":
        groups = c["n"] * (c["k"] // c["group"])
        out = c["n"] // 2 if c["swiglu"] else c["n"]
        return dict(bytes=c["n"] * c["k"] // 2 + 2 * groups + (groups // 2 if c["zero"] else 0) + 2 * c["m"] * (c["k"] + out + (c["n"] if c["res"] else 0)) + (2 * c["n"] if c["bias"] else 0),
                    flops=2 * c["m"] * c["n"] * c["k"])
    if c["op"] == "append":
        tokens = c["b"] * c["t"]
        return dict(bytes=tokens * (4 * c["hq"] * c["d"] + 2 * c["hkv"] * (3 * c["d"] + 4) + 4 * c["d"]) + 4 * c["b"], flops=tokens * c["d"] * (3 * (c["hq"] + c["hkv"]) + 4 * c["hkv"]))
    if c["op"] == "attention":
        b = c["b"]
        rows = sum((c["rows"] * (b - 1 - i) // max(b - 1, 1) if b > 1 else c["rows"]) + c["t"] for i in range(b))
        return dict(bytes=rows * c["hkv"] * (2 * c["d"] + 8) + 4 * b * c["t"] * c["hq"] * c["d"] + (8 * b * c["t"] if c["t"] > 1 else 0), flops=4 * rows * c["t"] * c["hq"] * c["d"])
    n = c["rows"] * c["vocab"]
    return dict(bytes=n * ((2 if c["half"] else 4) + (2 if c["counts"] else 0) + (0 if c["select"] else 4)) + (n // 8 if c["mask"] else 0) + (4 * c["vocab"] if c["bias"] else 0),
                flops=n * (6 if c["counts"] else 1))


# ---- the same in 64 bits, from the definitions ----------------------------------------------------------------------------------------

def exact(case, seed):
    s = _inputs(case, seed)
    return {"linear": _exact_linear, "append": _exact_append, "attention": _exact_attention, "logits": _exact_logits}[case["op"]](case, s)


def _exact_linear(c, s):
    """the products over blocks of output rows: out = r * sum_g scale * (sum codes * x - zero * sum x) + bias"""
    x = s["x"].double()
    groups = c["k"] // c["group"]
    xg = x.view(c["m"], groups, c["group"])
    parts = []
    for lo in range(0, c["n"], 4096):
        byte = s["codes"][lo:lo + 4096].long()
        code = torch.empty((byte.shape[0], c["k"]), dtype=torch.float64, device="cuda")
        code[:, 0::2], code[:, 1::2] = (byte % 16).double(), (byte // 16).double()
        zero = s["zero"][lo:lo + 4096].double() if c["zero"] else torch.full((byte.shape[0], groups), 8.0, dtype=torch.float64, device="cuda")
        scale = s["scale"][lo:lo + 4096].double()
        code *= scale.repeat_interleave(c["group"], dim=1)
        parts.append(x @ code.T - xg.sum(2) @ (scale * zero).T)
    y = torch.cat(parts, dim=1)
    if c["norm"]:
        y = y / ((x * x).sum(1, keepdim=True) / c["k"] + EPS).sqrt()
    if c["bias"]:
        y = y + s["bias"].double()
    if c["swiglu"]:
        half = c["n"] // 2
        y = y[:, half:] * y[:, :half] / (1 + torch.exp(-y[:, :half]))
    if c["res"]:
        y = y + s["res"].double()
    return y


def _exact_append(c, s):
    x = s["qkv"].double()
    half = c["d"] // 2
    hq, hkv = c["hq"], c["hkv"]
    row = s["start"].long()[:, None] + torch.arange(c["t"], device="cuda")
    cos, sin = s["cos"].double()[row][:, :, None, :half], s["sin"].double()[row][:, :, None, :half]
    turned = x.clone()
    turned[..., :half] = x[..., :half] * cos - x[..., half:] * sin
    turned[..., half:] = x[..., half:] * cos + x[..., :half] * sin
    shape = c["b"], hkv, c["cap"], c["d"]
    out = {}
    for name, rows in (("k", turned[:, :, hq:hq + hkv]), ("v", x[:, :, hq + hkv:])):
        scale = rows.abs().max(-1).values / 448
        codes = (rows / scale[..., None]).float().to(F8).double()
        full, scales = torch.zeros(shape, dtype=torch.float64, device="cuda"), torch.zeros(shape[:3], dtype=torch.float64, device="cuda")
        for b in range(c["b"]):
            lo = int(s["start"][b])
            full[b, :, lo:lo + c["t"]] = codes[b].transpose(0, 1)
            scales[b, :, lo:lo + c["t"]] = scale[b].T
        out[name], out[name + "_scale"] = full, scales
    return dict(q=turned[:, :, :hq], k=out["k"], v=out["v"].view(c["b"], hkv, -1, 64, c["d"]), k_scale=out["k_scale"], v_scale=out["v_scale"])


def _exact_attention(c, s):
    group = c["hq"] // c["hkv"]
    (kq, ks), (vq, vs) = _quantise(s["k"].float()), _quantise(s["v"].float())
    out = torch.zeros((c["b"], c["t"], c["hq"], c["d"]), dtype=torch.float64, device="cuda")
    i = torch.arange(c["t"], device="cuda")
    for b in range(c["b"]):
        ctx = int(s["start"][b])
        n = ctx + c["t"]
        k, v = kq[b, :, :n].double() * ks[b, :, :n, None].double(), vq[b, :, :n].double() * vs[b, :, :n, None].double()
        seen = torch.ones((c["t"], n), dtype=torch.bool, device="cuda")
        if c["t"] > 1:
            seen[:, ctx:] = (s["tree"][b][:, None] >> i) & 1 == 1
        for h in range(c["hkv"]):
            q = s["q"][b, :, h * group:(h + 1) * group].double()
            score = (q @ k[h].T / c["d"] ** 0.5).masked_fill(~seen[:, None], -math.inf)
            out[b, :, h * group:(h + 1) * group] = torch.softmax(score, -1) @ v[h]
    return out.view(c["b"], c["t"], -1)


def _exact_logits(c, s):
    if c["select"]:
        return None
    x = s["logits"].double()
    if c["counts"]:
        p = s["penalties"].double()
        count = s["counts"].long() & 0xffff
        made = count % 32768
        x = torch.where(count > 0, x * torch.where(x > 0, 1 / p[:, :1], p[:, :1]), x) - p[:, 2:] * made - p[:, 1:2] * (made > 0)
    if c["bias"]:
        x = x + s["bias"].double()
    if c["mask"]:
        bits = (s["allowed"].long()[:, :, None] >> torch.arange(32, device="cuda")) & 1
        x[bits.flatten(1)[:, :c["vocab"]] == 0] = -math.inf
    return x
