"""The trainable frame operators as they are measured: the selective state space scan with its
short causal convolution, layer norm, and the clipping of gradients by their global norm.

Every case runs one operator, once, on packed frames of utterances: `run` makes the calls of
the package where `own` is true, and computes the same in elementary torch operations in 32
bits (64 where 32 lose what matters) where it is false; `exact` computes it in 64 bits from the
definition, one frame after the other, with the gradients taken by automatic differentiation.
"""
import math
import random

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---- the cases ---------------------------------------------------------------------------

def listed():
    return [
        # one frame of eight live audio streams through one layer: latency is all that counts
        dict(name="scan_step_live", op="scan_step", dtype="bfloat16", streams=8, channels=1024, states=16,
             groups=1, gate=True),
        # one long recording, transcribed in one call: a single row, so all parallelism is in time
        dict(name="scan_long_recording", op="scan", dtype="bfloat16", utts=1, shortest=24001, longest=24001,
             channels=512, states=16, groups=1, gate=True, state=False),
        # a batch of command-word recordings (100 to 300 frames) that continue earlier pieces
        dict(name="scan_prompt_batch", op="scan", dtype="float16", utts=96, shortest=100, longest=300,
             channels=1024, states=16, groups=1, gate=True, state=True),
        # a training step's forward and backward pass over a batch of such recordings
        dict(name="scan_train_batch", op="scan_train", dtype="bfloat16", utts=64, shortest=100, longest=300,
             channels=1536, states=16, groups=1, gate=True),
        # the same for a small model in float32 with two groups and odd lengths
        dict(name="scan_train_small", op="scan_train", dtype="float32", utts=5, shortest=1, longest=119,
             channels=200, states=8, groups=2, gate=False),
        # one frame of 64 live streams through the short convolution
        dict(name="conv_step_live", op="conv_step", dtype="float16", streams=64, channels=2048, width=4),
        # the short convolution over a batch of recordings that continue earlier pieces
        dict(name="conv_prompt_batch", op="conv", dtype="bfloat16", utts=256, shortest=100, longest=300,
             channels=2048, width=4, state=True),
        # its forward and backward pass in float32
        dict(name="conv_train_batch", op="conv_train", dtype="float32", utts=64, shortest=100, longest=300,
             channels=1536, width=3),
        # the 39 features of every frame normalised: MFCC with their first and second differences
        dict(name="norm_features", op="norm", dtype="float32", rows=1310720, width=39),
        # a layer's norm in training: forward and backward with the weights' gradients
        dict(name="norm_train_batch", op="norm_train", dtype="bfloat16", rows=65536, width=1024),
        # the gradients of a small model, clipped into the optimiser's buffer: many little tensors
        dict(name="clip_small_model", op="clip", dtype="float32", layers=4, width=200),
        # those of a large one
        dict(name="clip_large_model", op="clip", dtype="bfloat16", layers=24, width=1024),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["scan_step", "scan", "scan", "scan_train", "conv_step", "conv", "conv_train", "norm",
                     "norm_train", "clip"])
    case = dict(op=op, dtype=rng.choice(sorted(TYPES)))
    if op in ("scan", "scan_train"):
        utts = _spread(rng, 1, 200)
        longest = _spread(rng, 1, min(24000, 24000 // utts if op == "scan" else 300))
        case.update(utts=utts, shortest=rng.randint(0, longest) if utts > 1 else longest, longest=longest,
                    states=rng.choice([4, 8, 16, 16, 16, 24, 32]), groups=rng.choice([1, 1, 1, 2, 4]), gate=rng.random() < 0.7)
        room = 24001 * 512 * 16 if op == "scan" else 12800 * 1536 * 16 // 2
        most = max(32, min(2048, room // (utts * longest * case["states"])))
        case["channels"] = max(1, _spread(rng, 32, most) // case["groups"]) * case["groups"]
        if op == "scan":
            case["state"] = rng.random() < 0.5
    elif op == "scan_step":
        case.update(streams=_spread(rng, 1, 512), states=rng.choice([4, 8, 16, 16, 16, 24, 32]), groups=1,
                    gate=rng.random() < 0.7, channels=_spread(rng, 32, 2048))
    elif op in ("conv", "conv_train"):
        utts = _spread(rng, 1, 256)
        longest = _spread(rng, 1, 24000 // utts)
        case.update(utts=utts, shortest=rng.randint(0, longest) if utts > 1 else longest, longest=longest,
                    channels=_spread(rng, 32, 2048), width=rng.choice([2, 3, 4, 4]))
        if op == "conv":
            case["state"] = rng.random() < 0.5
    elif op == "conv_step":
        case.update(streams=_spread(rng, 1, 512), channels=_spread(rng, 32, 4096), width=rng.choice([2, 3, 4, 4]))
    elif op in ("norm", "norm_train"):
        width = _spread(rng, 13, 8192)
        case.update(width=width, rows=_spread(rng, 1, 50000000 // width))
    else:
        case.update(layers=_spread(rng, 1, 24), width=_spread(rng, 13, 900))
    return case


def _lengths(case):
    """Frames per utterance: spread evenly over the case's range, in a mixed order."""
    r = random.Random(case["utts"] * 1000003 + case["longest"])
    span, utts = case["longest"] - case["shortest"], case["utts"]
    got = [case["shortest"] + (span * i) // max(1, utts - 1) for i in range(utts)]
    r.shuffle(got)
    return got


def _tensors(case):
    """The shapes of a model's parameters: per layer two projections, the convolution, A and the vectors."""
    w, shapes = case["width"], []
    for _ in range(case["layers"]):
        shapes += [(4 * w, w), (2 * w, 4), (2 * w,), (w // 16 + 32, 2 * w), (2 * w, 16), (2 * w,), (2 * w,),
                   (w, 2 * w), (w,), (w,)]
    return shapes


# ---- the inputs --------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev, dtype = torch.device("cuda"), TYPES[case["dtype"]]

    def randn(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * scale).to(dtype)

    s = {"case": dict(case)}
    op = case["op"]
    if op in ("scan", "scan_train", "conv", "conv_train"):
        lengths = _lengths(case)
        s["lengths"] = lengths
        n = sum(lengths)
        s["offsets"] = torch.tensor([0] + lengths, device=dev).cumsum(0)
        # what the plain form goes by: of each frame its utterance and its place in it
        of = torch.repeat_interleave(torch.arange(len(lengths), device=dev), torch.tensor(lengths, device=dev))
        s["of"], s["place"] = of, torch.arange(n, device=dev) - s["offsets"][of]
    else:
        n = case.get("streams", case.get("rows", 0))
    if op.startswith("scan"):
        c, m, groups = case["channels"], case["states"], case["groups"]
        rank = max(1, c // 16)
        s["x"] = torch.nn.functional.silu(randn(n, c)).to(dtype)
        # steps between about 0.001 and 0.2, as such layers are set up and learn
        s["dt"] = randn(n, c, dtype=dtype, scale=0.5)
        s["dt_bias"] = torch.rand(c, device=dev, generator=g) * 4.5 - 6.0
        # B and C are parts of one projection's rows, the gate is the other half of the input's
        s["rows"] = randn(n, rank + 2 * groups * m, dtype=dtype)
        s["B"] = s["rows"][:, rank:rank + groups * m].unflatten(1, (groups, m))
        s["C"] = s["rows"][:, rank + groups * m:].unflatten(1, (groups, m))
        s["gate"] = randn(n, 2 * c, dtype=dtype)[:, c:] if case["gate"] else None
        s["A"] = -torch.arange(1, m + 1, device=dev, dtype=torch.float32).repeat(c, 1) * \
            torch.exp(randn(c, m, scale=0.1))
        s["skip"] = 1 + randn(c, scale=0.1)
        if op == "scan_train":
            s["dy"] = randn(n, c, dtype=dtype)
        rows = case.get("streams") or (case["utts"] if case.get("state") else 0)
        s["state"] = randn(rows, c, m) if rows else None
    elif op.startswith("conv"):
        c, w = case["channels"], case["width"]
        s["x"] = randn(n, 2 * c, dtype=dtype)[:, :c]
        s["weight"] = randn(c, w, scale=1 / math.sqrt(w))
        s["bias"] = randn(c, scale=0.1)
        if op == "conv_train":
            s["dy"] = randn(n, c, dtype=dtype)
        rows = case.get("streams") or (case["utts"] if case.get("state") else 0)
        s["state"] = randn(rows, w - 1, c, dtype=dtype) if rows else None
    elif op.startswith("norm"):
        w = case["width"]
        # columns of their own mean and spread, like cepstra
        s["x"] = (randn(n, w) * (0.5 + torch.rand(w, device=dev, generator=g)) + randn(w)).to(dtype)
        s["weight"], s["bias"] = 1 + randn(w, scale=0.1), randn(w, scale=0.1)
        if op == "norm_train":
            s["dy"] = randn(n, w, dtype=dtype)
    else:
        s["grads"] = [randn(*shape, dtype=dtype, scale=0.01) for shape in _tensors(case)]
        s["flat"] = torch.zeros(sum(t.numel() for t in s["grads"]), device=dev)
        s["outs"], at = [], 0
        for t in s["grads"]:
            s["outs"].append(s["flat"][at:at + t.numel()].view(t.shape))
            at += t.numel()
        s["max_norm"] = 0.5 * 0.01 * math.sqrt(at)
    return s


# ---- one pass ----------------------------------------------------------------------------

def run(s):
    return _OWN[s["case"]["op"]](s) if own else _PLAIN[s["case"]["op"]](s)


def _library(s):
    import speech_recognition_amd as sra
    if "ctx" not in s:
        s["ctx"] = sra.Context.default()
    return sra, s["ctx"]


def _own_scan(s):
    sra, ctx = _library(s)
    return sra.selective_scan(ctx, s["x"], s["dt"], s["A"], s["B"], s["C"], s["offsets"], skip=s["skip"],
                              gate=s["gate"], dt_bias=s["dt_bias"], state=s["state"])


def _own_scan_train(s):
    sra, ctx = _library(s)
    y, last, saved = sra.selective_scan(ctx, s["x"], s["dt"], s["A"], s["B"], s["C"], s["offsets"], skip=s["skip"],
                                        gate=s["gate"], dt_bias=s["dt_bias"], save=True)
    grads = sra.selective_scan_backward(ctx, s["dy"], s["x"], s["dt"], s["A"], s["B"], s["C"], s["offsets"],
                                        skip=s["skip"], gate=s["gate"], dt_bias=s["dt_bias"], saved=saved)
    return y, last, {k: v for k, v in grads.items() if v is not None}


def _own_scan_step(s):
    sra, ctx = _library(s)
    y = sra.selective_scan_step(ctx, s["state"], s["x"], s["dt"], s["A"], s["B"], s["C"], skip=s["skip"],
                                gate=s["gate"], dt_bias=s["dt_bias"])
    return y, s["state"]


def _own_conv(s):
    sra, ctx = _library(s)
    return sra.causal_conv(ctx, s["x"], s["weight"], s["offsets"], bias=s["bias"], activation="silu",
                           state=s["state"])


def _own_conv_train(s):
    sra, ctx = _library(s)
    y, last = sra.causal_conv(ctx, s["x"], s["weight"], s["offsets"], bias=s["bias"], activation="silu")
    grads = sra.causal_conv_backward(ctx, s["dy"], s["x"], s["weight"], s["offsets"], bias=s["bias"],
                                     activation="silu")
    return y, last, {k: v for k, v in grads.items() if v is not None}


def _own_conv_step(s):
    sra, ctx = _library(s)
    y = sra.causal_conv_step(ctx, s["state"], s["x"], s["weight"], bias=s["bias"], activation="silu")
    return y, s["state"]


def _own_norm(s):
    sra, ctx = _library(s)
    return sra.layer_norm(ctx, s["x"], s["weight"], s["bias"])


def _own_norm_train(s):
    sra, ctx = _library(s)
    y, mean, rstd = sra.layer_norm(ctx, s["x"], s["weight"], s["bias"])
    return y, mean, rstd, sra.layer_norm_backward(ctx, s["dy"], s["x"], mean, rstd, s["weight"])


def _own_clip(s):
    sra, ctx = _library(s)
    return sra.clip_gradients(ctx, s["grads"], s["max_norm"], out=s["outs"]), s["flat"]


# ---- the plain forms ---------------------------------------------------------------------

def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-torch.abs(v)))


def _recurrence(a, b, place, longest):
    """h[t] = a[t] h[t-1] + b[t] inside every utterance, by doubling: after a round that spans k
    frames, b holds the last 2k frames' part of h, a their decay."""
    k = 1
    while k < longest:
        reach = (place[k:] >= k).view(-1, 1, 1)
        more = torch.where(reach, a[k:] * b[:-k], 0.0)
        decay = torch.where(reach, a[k:] * a[:-k], 0.0)
        a, b = torch.cat([a[:k], decay]), torch.cat([b[:k], b[k:] + more])
        k *= 2
    return b


def _per_channel(v, channels):
    """(n, groups, states) -> (n, channels, states) in 32 bits"""
    return v.float().repeat_interleave(channels // v.shape[1], dim=1)


def _scan_states(s):
    """What forward and backward have in common: step, decay, B and C per channel, all states."""
    c = s["x"].shape[1]
    raw = s["dt"].float() + s["dt_bias"]
    step = _softplus(raw)
    a = torch.exp(step[:, :, None] * s["A"])
    B, C = _per_channel(s["B"], c), _per_channel(s["C"], c)
    b = (step * s["x"].float())[:, :, None] * B
    if s["state"] is not None:
        first = (s["place"] == 0).nonzero()[:, 0]
        b[first] += a[first] * s["state"][s["of"][first]]
    h = _recurrence(a, b, s["place"], max(s["lengths"]))
    p = (C * h).sum(2) + s["skip"] * s["x"].float()
    return raw, step, a, B, C, h, p


def _scan_last(s, h):
    last = s["state"].clone() if s["state"] is not None else \
        torch.zeros(len(s["lengths"]), *s["A"].shape, device=h.device)
    some = (s["offsets"].diff() > 0).nonzero()[:, 0]
    last[some] = h[s["offsets"][some + 1] - 1]
    return last


def _plain_scan(s):
    *_, h, p = _scan_states(s)
    if s["gate"] is not None:
        z = s["gate"].float()
        p = p * (z / (1 + torch.exp(-z)))
    return p.to(s["x"].dtype), _scan_last(s, h)


def _plain_scan_train(s):
    dtype, (n, c) = s["x"].dtype, s["x"].shape
    groups = s["B"].shape[1]
    raw, step, a, B, C, h, p = _scan_states(s)
    x, dp, grads = s["x"].float(), s["dy"].float(), {}
    y = p
    if s["gate"] is not None:
        z = s["gate"].float()
        sig = 1 / (1 + torch.exp(-z))
        y = p * z * sig
        grads["gate"] = (dp * p * sig * (1 + z * (1 - sig))).to(dtype)
        dp = dp * z * sig
    # backwards in time: what the next frame's state owes to this one's
    left = (torch.tensor(s["lengths"], device=x.device)[s["of"]] - 1 - s["place"]).flip(0)
    after = torch.cat([a[1:], torch.zeros_like(a[:1])]).flip(0)
    dh = _recurrence(after, (dp[:, :, None] * C).flip(0), left, max(s["lengths"])).flip(0)
    du = (dh * B).sum(2)
    before = torch.where((s["place"] > 0).view(-1, 1, 1), torch.cat([torch.zeros_like(h[:1]), h[:-1]]), 0.0)
    m = dh * a * before
    dstep = (m * s["A"]).sum(2) + du * x
    draw = dstep / (1 + torch.exp(-raw))
    grads["x"] = (du * step + dp * s["skip"]).to(dtype)
    grads["dt"] = draw.to(dtype)
    grads["B"] = (dh * (step * x)[:, :, None]).unflatten(1, (groups, c // groups)).sum(2).to(dtype)
    grads["C"] = (h * dp[:, :, None]).unflatten(1, (groups, c // groups)).sum(2).to(dtype)
    grads["A"] = (m * step[:, :, None]).sum(0)
    grads["skip"], grads["dt_bias"] = (dp * x).sum(0), draw.sum(0)
    return y.to(dtype), _scan_last(s, h), grads


def _plain_scan_step(s):
    c = s["x"].shape[1]
    step = _softplus(s["dt"].float() + s["dt_bias"])
    x = s["x"].float()
    s["state"].copy_(torch.exp(step[:, :, None] * s["A"]) * s["state"]
                     + (step * x)[:, :, None] * _per_channel(s["B"], c))
    y = (s["state"] * _per_channel(s["C"], c)).sum(2) + s["skip"] * x
    if s["gate"] is not None:
        z = s["gate"].float()
        y = y * (z / (1 + torch.exp(-z)))
    return y.to(s["x"].dtype), s["state"]


def _conv_rows(s):
    """(n, width, channels): the frames that each output reads, oldest first; zeros or the state before the first"""
    x, w = s["x"].float(), s["weight"].shape[1]
    n, c = x.shape
    back = torch.arange(w - 1, -1, -1, device=x.device)
    at = torch.arange(n, device=x.device)[:, None] - back
    early = s["place"][:, None] < back
    if s["state"] is None:
        rows = torch.cat([x, torch.zeros(1, c, device=x.device)])
        at = torch.where(early, n, at)
    else:
        rows = torch.cat([x, s["state"].float().flatten(0, 1)])
        at = torch.where(early, n + s["of"][:, None] * (w - 1) + w - 1 + s["place"][:, None] - back, at)
    return rows[at.flatten()].view(n, w, c)


def _conv_last(s):
    """the last width - 1 frames of every utterance, those of the state or zeros before them"""
    w, x = s["weight"].shape[1], s["x"]
    utts, c = len(s["lengths"]), x.shape[1]
    lengths = s["offsets"].diff()[:, None]
    at = lengths - (w - 1) + torch.arange(w - 1, device=x.device)     # place in the utterance, negative before it
    before = s["state"] if s["state"] is not None else torch.zeros(utts, w - 1, c, dtype=x.dtype, device=x.device)
    rows = torch.cat([x, before.flatten(0, 1)])
    of = torch.arange(utts, device=x.device)[:, None]
    at = torch.where(at >= 0, s["offsets"][:-1, None] + at, x.shape[0] + of * (w - 1) + at + w - 1)
    return rows[at.flatten()].view(utts, w - 1, c)


def _plain_conv(s):
    v = (_conv_rows(s) * s["weight"].t()).sum(1) + s["bias"]
    return (v / (1 + torch.exp(-v))).to(s["x"].dtype), _conv_last(s)


def _plain_conv_train(s):
    dtype, (n, c), w = s["x"].dtype, s["x"].shape, s["weight"].shape[1]
    rows = _conv_rows(s)
    v = (rows * s["weight"].t()).sum(1) + s["bias"]
    sig = 1 / (1 + torch.exp(-v))
    g = s["dy"].float() * sig * (1 + v * (1 - sig))
    ahead = torch.arange(w - 1, -1, -1, device=g.device)
    at = torch.arange(n, device=g.device)[:, None] + ahead
    length = s["offsets"].diff()[s["of"]]
    at = torch.where(s["place"][:, None] + ahead < length[:, None], at, n)
    later = torch.cat([g, torch.zeros(1, c, device=g.device)])[at.flatten()].view(n, w, c)
    grads = {"x": (later * s["weight"].t()).sum(1).to(dtype), "weight": (g[:, None] * rows).sum(0).t().contiguous(),
             "bias": g.sum(0)}
    return (v * sig).to(dtype), _conv_last(s), grads


def _plain_conv_step(s):
    rows = torch.cat([s["state"], s["x"][:, None]], 1)
    v = (rows.float() * s["weight"].t()).sum(1) + s["bias"]
    s["state"].copy_(rows[:, 1:])
    return (v / (1 + torch.exp(-v))).to(s["x"].dtype), s["state"]


def _plain_norm(s):
    x = s["x"].float()
    mean = x.mean(1)
    away = x - mean[:, None]
    rstd = torch.rsqrt((away * away).mean(1) + 1e-5)
    return (away * rstd[:, None] * s["weight"] + s["bias"]).to(s["x"].dtype), mean, rstd


def _plain_norm_train(s):
    y, mean, rstd = _plain_norm(s)
    dy = s["dy"].float()
    unit = (s["x"].float() - mean[:, None]) * rstd[:, None]
    g = dy * s["weight"]
    dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True))
    return y, mean, rstd, (dx.to(s["x"].dtype), (dy * unit).sum(0), dy.sum(0))


def _plain_clip(s):
    norm = torch.sqrt(torch.stack([t.double().square().sum() for t in s["grads"]]).sum())
    factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    s["flat"].copy_(torch.cat([t.float().flatten() * factor.float() for t in s["grads"]]))
    return norm, s["flat"]


_OWN = {"scan": _own_scan, "scan_train": _own_scan_train, "scan_step": _own_scan_step, "conv": _own_conv,
        "conv_train": _own_conv_train, "conv_step": _own_conv_step, "norm": _own_norm,
        "norm_train": _own_norm_train, "clip": _own_clip}
_PLAIN = {"scan": _plain_scan, "scan_train": _plain_scan_train, "scan_step": _plain_scan_step, "conv": _plain_conv,
          "conv_train": _plain_conv_train, "conv_step": _plain_conv_step, "norm": _plain_norm,
          "norm_train": _plain_norm_train, "clip": _plain_clip}


# ---- what a pass cannot do without -------------------------------------------------------

def work(case):
    e, op = (4 if case["dtype"] == "float32" else 2), case["op"]
    n = sum(_lengths(case)) if "utts" in case else case.get("streams", case.get("rows", 0))
    if op.startswith("scan"):
        c, m, g = case["channels"], case["states"], case["groups"]
        wide = 3 + case["gate"]                                   # x, dt, y and the gate
        size = e * n * (wide * c + 2 * g * m) + 4 * c * (m + 2)
        flops = n * c * (7.0 * m + 12)                            # exp, two products, two multiply-adds
        if op == "scan_train":
            size += e * n * (wide * c + 2 * g * m) + 4 * c * (m + 2)   # dy; dx, ddt, dgate; dB, dC; dA, dskip, dbias
            flops += n * c * (14.0 * m + 24)
        rows = case.get("streams") or case["utts"]
        size += 4 * rows * c * m * (2 if case.get("state") or "streams" in case else 1)
    elif op.startswith("conv"):
        c, w = case["channels"], case["width"]
        size, flops = e * n * c * 2 + 4 * c * (w + 1), n * c * (2.0 * w + 6)
        if op == "conv_train":
            size, flops = size + e * n * c * 2 + 4 * c * (w + 1), flops * 3
        rows = case.get("streams") or case["utts"]
        size += e * rows * (w - 1) * c * (2 if case.get("state") or "streams" in case else 1)
    elif op.startswith("norm"):
        w = case["width"]
        size, flops = n * (2 * e * w + 8) + 8 * w, 8.0 * n * w
        if op == "norm_train":
            size, flops = size + 2 * e * n * w + 8 * w, flops * 3
    else:
        values = sum(math.prod(shape) for shape in _tensors(case))
        size, flops = (e + 4) * values + 8, 3.0 * values
    return {"bytes": size, "flops": flops}


# ---- the same in 64 bits, from the definitions -------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    train = case["op"].endswith("_train")
    names = {"scan": ["x", "dt", "A", "B", "C", "skip", "dt_bias", "gate"], "conv": ["x", "weight", "bias"],
             "norm": ["x", "weight", "bias"]}.get(case["op"].split("_")[0], [])
    v = {k: (t.double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t) for k, t in s.items()}
    if train:
        for k in names:
            if v[k] is not None:
                v[k] = v[k].detach().clone().requires_grad_()
    with torch.set_grad_enabled(train):
        if case["op"] == "clip":
            grads = [t.double() for t in s["grads"]]
            norm = math.sqrt(math.fsum(float((t * t).sum()) for t in grads))
            flat = torch.cat([t.reshape(-1) for t in grads])
            return torch.tensor(norm, dtype=torch.float64), flat * min(1.0, s["max_norm"] / (norm + 1e-6))
        y, *rest = {"scan": _exact_scan, "conv": _exact_conv, "norm": _exact_norm}[case["op"].split("_")[0]](case, v)
        if train:
            (y * v["dy"]).sum().backward()
    if not train:
        return (y, *rest)
    grads = {k: v[k].grad for k in names if v[k] is not None}
    out = (y.detach(), *(t.detach() for t in rest))
    return (*out, (grads["x"], grads["weight"], grads["bias"])) if case["op"] == "norm_train" else (*out, grads)


def _frames(case, v):
    """For a step the streams' single frames, else utterances side by side: lengths, a function
    that lays packed rows out as (utterances, frames, ...), and one that packs them again."""
    if "streams" in case:
        return [1] * case["streams"], lambda t: t.unsqueeze(1), lambda t: t.squeeze(1)
    lengths, dev = v["lengths"], v["x"].device
    longest, n = max(lengths), sum(lengths)
    at = torch.zeros(len(lengths), longest, dtype=torch.long, device=dev)
    back = torch.zeros(n, dtype=torch.long, device=dev)
    start = 0
    for u, length in enumerate(lengths):
        at[u, :length] = torch.arange(start, start + length, device=dev)
        back[start:start + length] = u * longest + torch.arange(length, device=dev)
        start += length

    def side_by_side(t):
        return t.index_select(0, at.flatten()).unflatten(0, (len(lengths), longest))

    return lengths, side_by_side, lambda t: t.flatten(0, 1).index_select(0, back)


def _exact_scan(case, v):
    lengths, wide, pack = _frames(case, v)
    per, dev = case["channels"] // case["groups"], v["x"].device
    x, raw = wide(v["x"]), wide(v["dt"] + v["dt_bias"])
    step = torch.logaddexp(raw, torch.zeros_like(raw))
    B, C = wide(v["B"]), wide(v["C"])
    length = torch.tensor(lengths, device=dev)
    h = torch.zeros(len(lengths), case["channels"], case["states"], dtype=torch.float64, device=dev)
    if v["state"] is not None:
        h = v["state"].clone()
    outs = []
    for t in range(max(lengths)):
        new = torch.exp(step[:, t, :, None] * v["A"]) * h \
            + (step[:, t] * x[:, t])[:, :, None] * B[:, t].repeat_interleave(per, 1)
        h = torch.where((t < length)[:, None, None], new, h)
        outs.append((h * C[:, t].repeat_interleave(per, 1)).sum(2) + v["skip"] * x[:, t])
    y = pack(torch.stack(outs, 1))
    if v["gate"] is not None:
        y = y * v["gate"] * torch.sigmoid(v["gate"])
    return y, h


def _exact_conv(case, v):
    lengths, wide, pack = _frames(case, v)
    w, x = case["width"], wide(v["x"])
    before = v["state"] if v["state"] is not None else \
        torch.zeros(len(lengths), w - 1, case["channels"], dtype=torch.float64, device=x.device)
    rows = torch.cat([before, x], 1)
    y = v["bias"]
    for k in range(w):
        y = y + rows[:, k:k + x.shape[1]] * v["weight"][:, k]
    last = torch.stack([rows[u, length:length + w - 1] for u, length in enumerate(lengths)])
    return pack(y * torch.sigmoid(y)), last.detach()


def _exact_norm(case, v):
    mean = v["x"].mean(1, keepdim=True)
    spread = (v["x"] - mean).square().mean(1, keepdim=True)
    y = (v["x"] - mean) / torch.sqrt(spread + 1e-5) * v["weight"] + v["bias"]
    return y, mean[:, 0].detach(), (1 / torch.sqrt(spread + 1e-5))[:, 0].detach()
