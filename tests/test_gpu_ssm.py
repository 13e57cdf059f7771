"""The trainable frame operators on the GPU against their float64 oracle.

Tolerances.  E = 2^-24 is half a step of float32.  The oracle also runs over absolute values, which
gives for each result the sum of the magnitudes that went into it (its scale); a float32 evaluation is then
off by at most K E scale, K the number of roundings on the longest path into a result:
  scan, forward:  a step of softplus is off by at most 12 E of itself (exponential, reciprocal, series), so a decay
    exp(-q) by (14 q + 2) E; over a stretch of frames the q exp(-q) sum to less than 0.37, which leaves 2 per frame,
    1 each for the product and the sum of the state, and the N-term sum of the output: K = 4 L + 2 N + 40 for
    utterances of at most L frames;
  scan, backward: the same again for the recursion backwards, and the channels of a group added up:
    2 (4 L + 2 N + 40) + c + 64; sums over n frames n more.
A result in 16 bits is rounded once more, by half a step of its own type (and of its subnormals)."""
import numpy as np
import pytest

from oracle import ssm_oracle as so

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
UNIT = {"float32": E, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 0.0, "bfloat16": 0.0, "float16": 2.0 ** -25}


@pytest.fixture(scope="module")
def sra():
    import speech_recognition_amd
    return speech_recognition_amd


@pytest.fixture(scope="module")
def ctx(sra):
    return sra.Context.default()


def _torch():
    import torch
    return torch


def _type(name):
    return getattr(_torch(), name)


def _draw(rng, shape, dtype, scale=1.0, pitch=0, shift=0):
    """(device tensor of the type, the float64 values that it holds); pitch: wider rows than shape[1:], starting
    `shift` elements into them, so that nothing is aligned."""
    torch = _torch()
    v = torch.from_numpy(np.asarray(rng.standard_normal(shape) * scale)).to(_type(dtype))
    t = v.cuda()
    if pitch:
        width = int(np.prod(shape[1:]))
        wide = torch.full((shape[0], width + pitch), float("nan"), dtype=_type(dtype), device="cuda")
        wide[:, shift:shift + width] = t.view(shape[0], width)
        t = wide[:, shift:shift + width].unflatten(1, shape[1:]) if len(shape) > 2 else wide[:, shift:shift + width]
    return t, v.double().numpy()


def _host(t):
    return t.detach().double().cpu().numpy()


def _close(got, ref, scale, k, dtype, what):
    got, ref = _host(got), np.asarray(ref)
    assert got.shape == ref.shape, what
    inside = ~np.isnan(ref)
    tol = UNIT[dtype] * np.abs(ref) * (1 if dtype != "float32" else 2) + k * E * np.abs(scale) + TINY[dtype]
    # (the rounding to 16 bits is of the computed value, which is off by the second term)
    tol = tol * (1 + UNIT[dtype])
    bad = ~(np.abs(got - ref) <= tol) & inside
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - ref) / np.where(tol > 0, tol, 1)):.3g} tolerances"


def _scan_case(rng, lengths, c, s, g, dtype, gate=True, skip=True, bias=True, state=True, pitch=0, tail=0):
    torch = _torch()
    off = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    n = int(off[-1]) + tail
    t, v = {}, {}
    t["x"], v["x"] = _draw(rng, (n, c), dtype, pitch=pitch, shift=pitch // 2)
    t["dt"], v["dt"] = _draw(rng, (n, c), dtype, pitch=pitch, shift=pitch)
    t["B"], v["B"] = _draw(rng, (n, g, s), dtype, pitch=pitch, shift=1 if pitch else 0)
    t["C"], v["C"] = _draw(rng, (n, g, s), dtype, pitch=pitch)
    f = np.float32
    v["A"] = -np.exp(rng.uniform(-2, 2.5, (c, s))).astype(f)
    v["skip"] = rng.standard_normal(c).astype(f) if skip else None
    v["dt_bias"] = (rng.standard_normal(c) - 2).astype(f) if bias else None
    v["state"] = rng.standard_normal((len(lengths), c, s)).astype(f) if state else None
    if gate:
        t["gate"], v["gate"] = _draw(rng, (n, c), dtype, pitch=pitch, shift=pitch // 2)
    else:
        t["gate"] = v["gate"] = None
    for k in ("A", "skip", "dt_bias", "state"):
        t[k] = None if v[k] is None else torch.from_numpy(v[k]).cuda()
        v[k] = None if v[k] is None else v[k].astype(np.float64)
    return off, t, v


ORDER = ("x", "dt", "A", "B", "C")
REST = ("skip", "gate", "dt_bias", "state")


def _run_scan(sra, ctx, off, t, dy=None, dso=None, softplus=True, **kw):
    torch = _torch()
    o = torch.from_numpy(off).cuda()
    rest = {k: t[k] for k in REST}
    if dy is None:
        return sra.selective_scan(ctx, *(t[k] for k in ORDER), o, dt_softplus=softplus, **rest, **kw)
    y, last, saved = sra.selective_scan(ctx, *(t[k] for k in ORDER), o, dt_softplus=softplus, save=True, **rest)
    return y, last, sra.selective_scan_backward(ctx, dy, *(t[k] for k in ORDER), o, dt_softplus=softplus, saved=saved,
                                                dstate_out=dso, **rest)


def _check_scan(sra, ctx, off, t, v, dtype, rng, backward=True, softplus=True):
    torch = _torch()
    n, c = v["x"].shape
    s, longest = v["A"].shape[1], int(np.diff(off).max())
    k = 4 * longest + 2 * s + 40
    kb = 2 * k + c + 64
    args = {q: v[q] for q in (*ORDER, *REST)}
    dy = dso = None
    if backward:
        dy, dyv = _draw(rng, (n, c), dtype)
        dsov = rng.standard_normal((len(off) - 1, c, s)).astype(np.float32)
        dso = torch.from_numpy(dsov).cuda()
        args.update(dy=dyv, dstate_out=dsov.astype(np.float64))
    ref = so.scan(off, dt_softplus=softplus, **args)
    size = so.scan(off, dt_softplus=softplus, scales=True, **args)
    got = _run_scan(sra, ctx, off, t, dy, dso, softplus)
    _close(got[0], ref["y"], size["y"], k, dtype, "y")
    _close(got[1], ref["state_out"], size["state_out"], k, "float32", "state_out")
    if backward:
        for q, grad in got[2].items():
            if v[q] is None:
                assert grad is None, q
                continue
            param = q in ("A", "skip", "dt_bias", "state")
            _close(grad, ref["d" + q], size["d" + q], kb + (n if param else 0), "float32" if param else dtype, "d" + q)
    return got


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("lengths,c,s,g", [
    ([1], 1, 1, 1), ([7], 3, 4, 1), ([0, 5, 0, 17, 1, 0], 64, 16, 1), ([16, 32, 15, 33], 65, 16, 1),
    ([8, 9], 130, 8, 2), ([40, 3], 200, 8, 2), ([31], 20, 24, 5), ([19, 2], 40, 32, 1), ([18], 24, 64, 1),
    ([65, 64], 17, 33, 1), ([3] * 40, 48, 3, 3), ([300], 66, 16, 1)])
def test_scan_against_oracle(sra, ctx, lengths, c, s, g, dtype):
    rng = np.random.default_rng(c + s)
    off, t, v = _scan_case(rng, lengths, c, s, g, dtype)
    _check_scan(sra, ctx, off, t, v, dtype, rng)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("gate,skip,bias,state,softplus", [
    (False, False, False, False, True), (True, False, False, True, True), (False, True, True, False, True),
    (False, False, True, True, False), (True, True, False, False, False)])
def test_scan_optional_arguments(sra, ctx, gate, skip, bias, state, softplus, dtype):
    rng = np.random.default_rng(5)
    off, t, v = _scan_case(rng, [9, 20], 30, 16, 1, dtype, gate, skip, bias, state)
    if not softplus:            # steps as they are: positive ones
        t["dt"], v["dt"] = t["dt"].abs() + 3, None
        v["dt"] = _host(t["dt"])
    _check_scan(sra, ctx, off, t, v, dtype, rng, softplus=softplus)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("lengths", [[1500], [700, 0, 1, 901], [129, 500]])
def test_scan_long_utterances_in_pieces(sra, ctx, lengths, dtype):
    """Few rows and long: the utterances are cut into pieces that run side by side."""
    rng = np.random.default_rng(6)
    off, t, v = _scan_case(rng, lengths, 24, 16, 1, dtype)
    _check_scan(sra, ctx, off, t, v, dtype, rng)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("c,s,g,gate", [(1650, 16, 3, True), (1665, 16, 1, False), (1700, 7, 2, True)])
def test_scan_batches_that_fill_the_device(sra, ctx, c, s, g, gate, dtype):
    """Enough rows for two channels a lane and for utterances taken by their lengths; the longest is not the first, one
    has no frame, and some are equally long."""
    rng = np.random.default_rng(c)
    lengths = rng.integers(5, 80, 40)
    lengths[[3, 30]], lengths[7], lengths[38] = 20, 0, 90
    assert lengths.sum() >= 32 * 40
    off, t, v = _scan_case(rng, lengths, c, s, g, dtype, gate=gate)
    got = _check_scan(sra, ctx, off, t, v, dtype, rng)
    y, last = _run_scan(sra, ctx, off, t)           # (without saved states: the order is kept elsewhere)
    torch = _torch()
    assert torch.equal(y, got[0]) and torch.equal(last, got[1])


def test_scan_more_short_utterances_than_a_wave_takes(sra, ctx):
    """One wave sums the parameters' gradients over several utterances."""
    rng = np.random.default_rng(25)
    off, t, v = _scan_case(rng, rng.integers(0, 5, 300), 2040, 16, 1, "float32")
    _check_scan(sra, ctx, off, t, v, "float32", rng)


@pytest.mark.parametrize("u", [0, 3])
def test_scan_of_no_frames(sra, ctx, u):
    """No utterance, or only empty ones: states pass, the parameters' gradients are 0."""
    torch = _torch()
    rng = np.random.default_rng(26)
    off, t, v = _scan_case(rng, [0] * u, 20, 16, 1, "float32")
    dso = torch.from_numpy(rng.standard_normal((u, 20, 16)).astype(np.float32)).cuda()
    y, last, g = _run_scan(sra, ctx, off, t, torch.empty(0, 20, device="cuda"), dso)
    assert y.shape == (0, 20) and torch.equal(last, t["state"])
    assert torch.equal(g["state"], dso)
    for k in ("A", "skip", "dt_bias"):
        assert not g[k].any(), k
    conv = torch.from_numpy(rng.standard_normal((20, 4)).astype(np.float32)).cuda()
    o = torch.from_numpy(off).cuda()
    first = torch.from_numpy(rng.standard_normal((u, 3, 20)).astype(np.float32)).cuda()
    y, last = sra.causal_conv(ctx, t["x"], conv, o, None, "silu", state=first)
    assert y.shape == (0, 20) and torch.equal(last, first)
    g = sra.causal_conv_backward(ctx, y, t["x"], conv, o, None, "silu", state=first)
    assert not g["weight"].any()


@pytest.mark.parametrize("pitch", [2, 3, 5])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scan_takes_rows_at_any_pitch_and_leaves_others_alone(sra, ctx, dtype, pitch):
    torch = _torch()
    rng = np.random.default_rng(7)
    off, t, v = _scan_case(rng, [12, 0, 21], 37, 7, 1, dtype, pitch=pitch, tail=4)
    _check_scan(sra, ctx, off, t, v, dtype, rng)
    wide = torch.full((v["x"].shape[0], 37 + pitch), 7.0, dtype=_type(dtype), device="cuda")
    out = wide[:, 1:38]
    y, _ = _run_scan(sra, ctx, off, t, out=out)
    assert y is out
    y2, _ = _run_scan(sra, ctx, off, t)
    assert torch.equal(out[:33], y2[:33])
    assert (wide[33:] == 7).all() and (wide[:, :1] == 7).all() and (wide[:, 38:] == 7).all()


def test_scan_offsets_that_skip_frames(sra, ctx):
    """Offsets that begin behind the first frame: those rows belong to nobody, whatever they hold."""
    torch = _torch()
    rng = np.random.default_rng(8)
    off, t, v = _scan_case(rng, [10, 6], 16, 4, 1, "float32")
    lead = {k: torch.cat([torch.full_like(t[k][:3], float("nan")), t[k]]) for k in ("x", "dt", "B", "C", "gate")}
    out = torch.full((19, 16), 5.0, device="cuda")
    y, last = _run_scan(sra, ctx, off + 3, {**t, **lead}, out=out)
    want, wlast = _run_scan(sra, ctx, off, t)
    assert (y[:3] == 5).all() and torch.equal(y[3:], want) and torch.equal(last, wlast)


def test_scan_not_a_number_stays_in_its_utterance(sra, ctx):
    torch = _torch()
    rng = np.random.default_rng(9)
    off, t, v = _scan_case(rng, [21, 18, 30], 20, 16, 1, "float32")
    clean = _run_scan(sra, ctx, off, t, _draw(np.random.default_rng(1), (69, 20), "float32")[0])
    for bad in (float("nan"), float("inf")):
        x = t["x"].clone()
        x[25] = bad
        dirty = _run_scan(sra, ctx, off, {**t, "x": x}, _draw(np.random.default_rng(1), (69, 20), "float32")[0])
        assert torch.equal(dirty[0][:25], clean[0][:25]) and torch.equal(dirty[0][39:], clean[0][39:])
        assert not torch.isfinite(dirty[0][25:39]).any()
        for k in ("x", "dt", "B", "C", "gate"):
            assert torch.equal(dirty[2][k][:21], clean[2][k][:21]) and torch.equal(dirty[2][k][39:], clean[2][k][39:]), k


@pytest.mark.parametrize("lengths", [[5, 16, 35], [1500]])
def test_scan_decays_without_bound_forget_at_once(sra, ctx, lengths):
    """An A of minus infinity, or the type's lowest value, is one whose decay is 0 at any step of ordinary size: the same
    results as with -1e30, in whole tiles and at their ends."""
    torch = _torch()
    rng = np.random.default_rng(27)
    off, t, v = _scan_case(rng, lengths, 24, 16, 1, "float32")
    dy = _draw(rng, (int(off[-1]), 24), "float32")[0]
    got = []
    for low in (-1e30, torch.finfo(torch.float32).min, float("-inf")):
        A = t["A"].clone()
        A[::3, ::2] = low
        got.append(_run_scan(sra, ctx, off, {**t, "A": A}, dy))
    for y, last, g in got[1:]:
        assert torch.isfinite(y).all() and torch.equal(y, got[0][0]) and torch.equal(last, got[0][1])
        for k in g:
            assert torch.equal(g[k], got[0][2][k]), k


def test_scan_infinity_in_the_last_frame_stays_infinity(sra, ctx):
    torch = _torch()
    rng = np.random.default_rng(28)
    for n in (5, 16, 21):
        off, t, v = _scan_case(rng, [n], 20, 16, 1, "float32")
        t["B"][n - 1] = float("inf")
        _, last = _run_scan(sra, ctx, off, t)
        want = torch.sign(t["x"][n - 1])[:, None].expand(20, 16) * float("inf")
        assert torch.equal(last[0], want), n


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_scan_in_pieces_by_the_caller_equals_the_whole(sra, ctx, dtype):
    """A recording that comes in three calls, its state handed on in place; then frame by frame."""
    torch = _torch()
    rng = np.random.default_rng(10)
    off, t, v = _scan_case(rng, [50], 33, 16, 1, dtype, state=True)
    whole, last = _run_scan(sra, ctx, off, t)
    state, parts = t["state"].clone(), []
    for a, b in ((0, 7), (7, 7), (7, 40), (40, 50)):
        cut = {k: (t[k][a:b] if k in ("x", "dt", "B", "C", "gate") else t[k]) for k in t}
        y, got = _run_scan(sra, ctx, np.array([0, b - a]), {**cut, "state": state}, state_out=state)
        assert got is state
        parts.append(y)
    assert torch.equal(torch.cat(parts), whole) and torch.equal(state, last)
    state, parts = t["state"].clone(), []
    for i in range(50):
        parts.append(sra.selective_scan_step(ctx, state, t["x"][i:i + 1], t["dt"][i:i + 1], t["A"], t["B"][i:i + 1],
                                             t["C"][i:i + 1], skip=t["skip"], gate=t["gate"][i:i + 1],
                                             dt_bias=t["dt_bias"]))
    args = {q: v[q] for q in (*ORDER, *REST)}
    ref, size = so.scan(off, **args), so.scan(off, scales=True, **args)
    _close(torch.cat(parts), ref["y"], size["y"], 4 * 50 + 2 * 16 + 40, dtype, "y")
    _close(state, ref["state_out"], size["state_out"], 4 * 50 + 2 * 16 + 40, "float32", "state")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,c,s,g", [(1, 1, 1, 1), (3, 65, 16, 1), (8, 200, 7, 2), (2, 12, 64, 3), (300, 40, 24, 1)])
def test_scan_step_against_oracle(sra, ctx, rows, c, s, g, dtype):
    rng = np.random.default_rng(rows)
    off, t, v = _scan_case(rng, [1] * rows, c, s, g, dtype, pitch=3)
    state = t["state"].clone()
    y = sra.selective_scan_step(ctx, state, *(t[k] for k in ORDER), skip=t["skip"], gate=t["gate"], dt_bias=t["dt_bias"])
    args = {q: v[q] for q in (*ORDER, *REST)}
    ref, size = so.scan(off, **args), so.scan(off, scales=True, **args)
    _close(y, ref["y"], size["y"], 4 + 2 * s + 40, dtype, "y")
    _close(state, ref["state_out"], size["state_out"], 4 + 2 * s + 40, "float32", "state")


def test_scan_gradient_is_the_difference(sra, ctx):
    """The gradients against the forward pass itself.  Along a direction v the loss changes by grad . v h
    + third derivatives h^3; with h = 1e-2 and smooth inputs of order one the second is below 1e-3 of the
    sum of the terms' magnitudes, and the loss's own rounding (K E of its magnitudes, K = 600) over h is
    4e-3 of them."""
    torch = _torch()
    rng = np.random.default_rng(11)
    off, t, v = _scan_case(rng, [60, 30], 40, 16, 1, "float32")
    dy = _draw(rng, (90, 40), "float32")[0]
    _, _, grads = _run_scan(sra, ctx, off, t, dy)
    for k in ("x", "dt", "A", "B", "C", "skip", "gate", "dt_bias", "state"):
        way = torch.from_numpy(rng.standard_normal(t[k].shape).astype(np.float32)).cuda()
        if k == "A":
            way = way * t[k].abs()
        h = 1e-2
        terms = [(_run_scan(sra, ctx, off, {**t, k: t[k] + sign * h * way})[0].double() * dy.double())
                 for sign in (1, -1)]
        want = float((terms[0].sum() - terms[1].sum()) / (2 * h))
        size = float((grads[k].double() * way.double()).abs().sum())
        noise = 600 * E * float(terms[0].abs().sum()) / h
        assert abs(float((grads[k].double() * way.double()).sum()) - want) <= 5e-3 * size + noise, k


def test_scan_backward_without_saved_states_and_twice(sra, ctx):
    torch = _torch()
    rng = np.random.default_rng(12)
    for lengths in ([30, 41, 2], [900]):
        off, t, v = _scan_case(rng, lengths, 50, 16, 2 if len(lengths) > 1 else 1, "bfloat16")
        dy = _draw(rng, (int(off[-1]), 50), "bfloat16")[0]
        a = _run_scan(sra, ctx, off, t, dy)[2]
        b = sra.selective_scan_backward(ctx, dy, *(t[k] for k in ORDER), torch.from_numpy(off).cuda(),
                                        **{k: t[k] for k in REST})
        for k in a:
            assert torch.equal(a[k], b[k]), k


def _conv_case(rng, lengths, c, w, dtype, state=True, pitch=0, tail=0):
    torch = _torch()
    off = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
    n = int(off[-1]) + tail
    t, v = {}, {}
    t["x"], v["x"] = _draw(rng, (n, c), dtype, pitch=pitch, shift=pitch)
    t["state"], v["state"] = _draw(rng, (len(lengths), w - 1, c), dtype) if state else (None, None)
    for k, shape in (("weight", (c, w)), ("bias", (c,))):
        v[k] = rng.standard_normal(shape).astype(np.float32)
        t[k] = torch.from_numpy(v[k]).cuda()
        v[k] = v[k].astype(np.float64)
    return off, t, v


@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("lengths,c,w,pitch", [
    ([1], 1, 4, 0), ([0, 2, 0, 17, 1, 3], 9, 4, 0), ([16, 32, 15, 33, 100], 64, 3, 3), ([5, 1, 2], 200, 2, 0),
    ([40], 12, 1, 1), ([19, 4, 3, 7, 0], 30, 8, 5), ([6, 61], 520, 5, 0), ([21, 9], 16, 6, 1), ([33, 4], 8, 7, 0)])
def test_conv_against_oracle(sra, ctx, lengths, c, w, pitch, dtype, activation):
    """K: the width's products and sums, the bias and, with silu, the sigmoid (at most 8 E of itself)."""
    torch = _torch()
    rng = np.random.default_rng(c + w)
    off, t, v = _conv_case(rng, lengths, c, w, dtype, pitch=pitch, tail=2)
    n = v["x"].shape[0]
    dy, dyv = _draw(rng, (n, c), dtype, pitch=pitch)
    dso, dsov = _draw(rng, (len(lengths), w - 1, c), dtype)
    o = torch.from_numpy(off).cuda()
    ref = so.conv(off, dy=dyv, dstate_out=dsov, activation=activation, **v)
    size = so.conv(off, dy=dyv, dstate_out=dsov, activation=activation, scales=True, **v)
    y, last = sra.causal_conv(ctx, t["x"], t["weight"], o, t["bias"], activation, t["state"])
    k = 2 * w + 16
    _close(y, ref["y"], size["y"], k, dtype, "y")
    assert np.array_equal(_host(last), ref["state_out"])                  # frames as they came
    grads = sra.causal_conv_backward(ctx, dy, t["x"], t["weight"], o, t["bias"], activation, t["state"], dso)
    for q, grad in grads.items():
        param = q in ("weight", "bias")
        _close(grad, ref["d" + q], size["d" + q], 2 * k + (n if param else 0), "float32" if param else dtype, "d" + q)
    # without bias and state
    bare = sra.causal_conv_backward(ctx, dy, t["x"], t["weight"], o, None, activation)
    assert bare["bias"] is None and bare["state"] is None
    ref = so.conv(off, v["x"], v["weight"], activation=activation, dy=dyv)
    size = so.conv(off, v["x"], v["weight"], activation=activation, dy=dyv, scales=True)
    _close(sra.causal_conv(ctx, t["x"], t["weight"], o, activation=activation)[0], ref["y"], size["y"], k, dtype, "y")
    _close(bare["x"], ref["dx"], size["dx"], 2 * k, dtype, "dx")
    _close(bare["weight"], ref["dweight"], size["dweight"], 2 * k + n, "float32", "dweight")


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("w", [1, 2, 4, 8])
def test_conv_in_pieces_and_frame_by_frame(sra, ctx, w, dtype):
    torch = _torch()
    rng = np.random.default_rng(w)
    off, t, v = _conv_case(rng, [40], 21, w, dtype)
    whole, last = sra.causal_conv(ctx, t["x"], t["weight"], None, t["bias"], "silu", t["state"])
    state, parts = t["state"].clone(), []
    for a, b in ((0, 1), (1, 1), (1, 3), (3, 20), (20, 40)):
        y, got = sra.causal_conv(ctx, t["x"][a:b], t["weight"], [0, b - a], t["bias"], "silu", state, state_out=state)
        assert got is state
        parts.append(y)
    assert torch.equal(torch.cat(parts), whole) and torch.equal(state, last)
    state, parts = t["state"].clone(), []
    for i in range(40):
        parts.append(sra.causal_conv_step(ctx, state, t["x"][i:i + 1], t["weight"], t["bias"], "silu"))
    assert torch.equal(torch.cat(parts), whole) and torch.equal(state, last)


def test_conv_leaves_rows_behind_the_last_utterance_alone(sra, ctx):
    torch = _torch()
    rng = np.random.default_rng(3)
    off, t, v = _conv_case(rng, [9, 4], 10, 4, "bfloat16", tail=5)
    out = torch.full((18, 10), 3.0, dtype=torch.bfloat16, device="cuda")
    sra.causal_conv(ctx, t["x"], t["weight"], off, t["bias"], None, out=out)
    assert (out[13:] == 3).all() and not (out[:13] == 3).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("n,d", [(1, 1), (5, 13), (7, 39), (100, 64), (33, 65), (9, 129), (16, 256), (3, 257), (5, 600),
                                 (2, 1024), (3, 1025), (2, 2500), (3, 4096), (2, 4097), (1, 9001), (3000, 20)])
def test_norm_against_oracle(sra, ctx, n, d, dtype):
    """K: a lane sums at most d / 16 values (d / 256 of the wide rows), the lanes as a tree, and every value goes
    through a dozen roundings: d / 16 + 40.  The normalised value is off by K E of what was subtracted and
    divided, (max |x| + |mean|) rstd, which the scales below carry into the gradients."""
    torch = _torch()
    rng = np.random.default_rng(n + d)
    x, xv = _draw(rng, (n, d), dtype, pitch=3, shift=1)
    x, xv = x + 2, None
    xv = _host(x)
    wide = torch.zeros(n, d + 3, dtype=x.dtype, device="cuda")
    wide[:, 1:d + 1] = x
    x = wide[:, 1:d + 1]
    dy, dyv = _draw(rng, (n, d), dtype, pitch=1)
    w, b = rng.standard_normal((2, d)).astype(np.float32)
    k = d / 16 + 40
    for weight, bias in ((w, b), (None, None)):
        tw, tb = (None if a is None else torch.from_numpy(a).cuda() for a in (weight, bias))
        wv = np.ones(d) if weight is None else weight.astype(np.float64)
        ref = so.norm(xv, wv, None if bias is None else bias.astype(np.float64), dy=dyv)
        y, mean, rstd = sra.layer_norm(ctx, x, tw, tb)
        r = ref["rstd"][:, None]
        top = 2 * np.abs(xv).max(1, keepdims=True) * r
        unit = (xv - ref["mean"][:, None]) * r
        _close(y, ref["y"], top * np.abs(wv) + np.abs(ref["y"]) + (0 if bias is None else np.abs(bias)), k, dtype, "y")
        _close(mean, ref["mean"], np.abs(xv).max(1), k, "float32", "mean")
        # rstd: the variance is off by K E of itself and by the mean's error times the largest deviation
        _close(rstd, ref["rstd"], ref["rstd"] * (1 + top[:, 0] * np.abs(unit).max(1)), k, "float32", "rstd")
        # (an error of rstd moves a whole row: relative to the value; that of the mean by its own size)
        spread = 1 + top * np.abs(unit).max(1, keepdims=True)
        dx, dw, db = sra.layer_norm_backward(ctx, dy, x, mean, rstd, tw)
        g = np.abs(dyv * wv)
        gu = (g * np.abs(unit)).mean(1, keepdims=True)
        size = r * ((g + g.mean(1, keepdims=True) + np.abs(unit) * gu) * spread
                    + spread * top * (gu + np.abs(unit) * g.mean(1, keepdims=True)))
        _close(dx, ref["dx"], size, 2 * k, dtype, "dx")
        _close(dw, ref["dweight"], (np.abs(dyv) * (np.abs(unit) + top) * spread).sum(0), 2 * k + n, "float32", "dweight")
        _close(db, ref["dbias"], np.abs(dyv).sum(0), n + 8, "float32", "dbias")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("n", [1, 128, 301])
def test_norm_of_narrow_rows_without_gaps(sra, ctx, n, dtype):
    """Rows that lie side by side travel as one run of memory: the same bits as rows with gaps, and nothing behind
    the last one is written."""
    torch = _torch()
    rng = np.random.default_rng(n)
    for d in (1, 2, 7, 8, 9, 15, 16, 23, 26, 31, 32, 33, 39, 47, 49, 55, 57, 63, 64):
        x = _draw(rng, (n, d), dtype)[0]
        wide = torch.zeros(n, d + 2, dtype=x.dtype, device="cuda")
        wide[:, 1:d + 1] = x
        w, b = (torch.from_numpy(rng.standard_normal(d).astype(np.float32)).cuda() for _ in range(2))
        want, mean, rstd = sra.layer_norm(ctx, wide[:, 1:d + 1], w, b)
        room = torch.full((n * d + 19,), 7.0, dtype=x.dtype, device="cuda")
        got = sra.layer_norm(ctx, x, w, b, out=room[1:1 + n * d].view(n, d))     # (of its element's alignment only)
        assert torch.equal(got[0], want) and torch.equal(got[1], mean) and torch.equal(got[2], rstd), d
        assert room[0] == 7 and (room[1 + n * d:] == 7).all(), d


def test_norm_far_from_zero_and_constant_rows(sra, ctx):
    """Rows around 1000 with a spread of one: the deviations are exact to their own size, as the mean is
    subtracted before anything is squared; a constant row gives the bias."""
    torch = _torch()
    rng = np.random.default_rng(4)
    xv = (1000 + rng.standard_normal((6, 300))).astype(np.float32)
    xv[3] = 7.25
    y, mean, rstd = sra.layer_norm(ctx, torch.from_numpy(xv).cuda(), eps=1e-5)
    ref = so.norm(xv.astype(np.float64))
    # the mean is off by half a step at 1000 (2^-15) and a few more in its sum
    assert np.abs(_host(y) - ref["y"])[[0, 1, 2, 4, 5]].max() < 4 * 2.0 ** -15
    assert (_host(y)[3] == 0).all() and abs(_host(rstd)[3] * np.sqrt(1e-5) - 1) < 4 * E


def _grads(rng, shapes, dtypes):
    torch = _torch()
    return [torch.from_numpy(rng.standard_normal(s)).to(_type(d)).cuda() for s, d in zip(shapes, dtypes)]


@pytest.mark.parametrize("shapes,dtypes", [
    ([(1,)], ["float32"]), ([(3, 5), (0,), (7,)], ["float32", "float16", "bfloat16"]),
    ([(8193,), (16384,), (1,)], ["bfloat16", "float32", "float16"]),
    ([(13,)] * 250, ["float32", "bfloat16"] * 125), ([(300, 777), (5,)], ["float16", "bfloat16"]), ([], [])])
@pytest.mark.parametrize("max_norm", [0.0, 0.5, 1e9])
def test_clip_against_oracle(sra, ctx, shapes, dtypes, max_norm):
    torch = _torch()
    rng = np.random.default_rng(len(shapes))
    grads = _grads(rng, shapes, dtypes)
    total, ref = so.clip([_host(g) for g in grads], max_norm)
    flat = torch.full((sum(g.numel() for g in grads) + 1,), 9.0, device="cuda")
    outs, at = [], 1
    for g in grads:                        # (one float into the buffer: nothing is aligned)
        outs.append(flat[at:at + g.numel()].view(g.shape))
        at += g.numel()
    norm = sra.clip_gradients(ctx, grads, max_norm, out=outs)
    assert norm.dtype == torch.float64 and norm.shape == ()
    assert abs(float(norm) - total) <= 1e-13 * max(total, 1)
    for o, r in zip(outs, ref):            # factor and product: a rounding each
        _close(o, r, r, 2, "float32", "out")
    assert flat[0] == 9
    before = [g.clone() for g in grads]
    norm = sra.clip_gradients(ctx, grads, max_norm)
    assert abs(float(norm) - total) <= 1e-13 * max(total, 1)
    for g, r, d, b in zip(grads, ref, dtypes, before):
        _close(g, r, r, 2, d, "in place")
        if max_norm == 1e9:
            assert torch.equal(g, b)


def test_clip_large_small_and_lost_gradients(sra, ctx):
    torch = _torch()
    big = [torch.full((1000,), 1e30, device="cuda"), torch.full((10,), 1e-30, device="cuda")]
    norm = sra.clip_gradients(ctx, big, 1.0)
    assert abs(float(norm) / (1e30 * np.sqrt(1000)) - 1) < 1e-6
    assert abs(float(big[0][0]) * np.sqrt(1000) - 1) < 4 * E
    for bad in (float("nan"), float("inf")):
        g = [torch.ones(100, device="cuda"), torch.full((3,), bad, device="cuda")]
        out = [torch.zeros(100, device="cuda"), torch.zeros(3, device="cuda")]
        assert not np.isfinite(float(sra.clip_gradients(ctx, g, 0.1, out=out)))
        assert (out[0] == 1).all() and not torch.isfinite(out[1]).any()
        assert not np.isfinite(float(sra.clip_gradients(ctx, g, 0.1)))
        assert (g[0] == 1).all()
    turned = torch.arange(12.0, device="cuda").view(3, 4).t()
    norm = sra.clip_gradients(ctx, [turned], 1.0)
    assert abs(float(turned.square().sum()) - 1) < 1e-5 and abs(float(norm) - np.sqrt(506)) < 1e-12 * 23


def _layer(sra, ctx, p, frames, off, dy=None):
    """One layer as a user strings it together: norm, projection, convolution, scan, projection back."""
    torch = _torch()
    c, s = p["A"].shape
    rank = p["up"].shape[1]
    u, mean, rstd = sra.layer_norm(ctx, frames, p["gamma"], p["beta"])
    both = u @ p["in"]
    v, _ = sra.causal_conv(ctx, both[:, :c], p["conv"], off, p["conv_bias"], "silu")
    rows = v @ p["rows"]
    dt = rows[:, :rank] @ p["up"].t()
    args = (v, dt, p["A"], rows[:, rank:rank + s], rows[:, rank + s:], off)
    kw = dict(skip=p["skip"], gate=both[:, c:], dt_bias=p["dt_bias"])
    y, last, saved = sra.selective_scan(ctx, *args, save=True, **kw)
    out = y @ p["out"]
    if dy is None:
        return out
    g = {"out": y.t() @ dy}
    d = sra.selective_scan_backward(ctx, dy @ p["out"].t(), *args, saved=saved, **kw)
    g.update(A=d["A"], skip=d["skip"], dt_bias=d["dt_bias"], up=d["dt"].t() @ rows[:, :rank])
    drows = torch.cat([d["dt"] @ p["up"], d["B"], d["C"]], 1)
    g["rows"] = v.t() @ drows
    dc = sra.causal_conv_backward(ctx, d["x"] + drows @ p["rows"].t(), both[:, :c], p["conv"], off, p["conv_bias"],
                                  "silu")
    g.update(conv=dc["weight"], conv_bias=dc["bias"])
    dboth = torch.cat([dc["x"], d["gate"]], 1)
    g["in"] = u.t() @ dboth
    g["x"], g["gamma"], g["beta"] = sra.layer_norm_backward(ctx, dboth @ p["in"].t(), frames, mean, rstd, p["gamma"])
    return out, g


def _layer_parameters(rng, d, c, s, rank, out, w=4):
    torch = _torch()

    def mat(*shape, scale=None):
        v = rng.standard_normal(shape) * (1 / np.sqrt(shape[0]) if scale is None else scale)
        return torch.from_numpy(v.astype(np.float32)).cuda()

    return {"gamma": 1 + mat(d, scale=0.1), "beta": mat(d, scale=0.1), "in": mat(d, 2 * c), "conv": mat(c, w, scale=0.5),
            "conv_bias": mat(c, scale=0.1), "rows": mat(c, rank + 2 * s), "up": mat(c, rank, scale=0.5),
            "A": -torch.arange(1, s + 1, dtype=torch.float32, device="cuda").repeat(c, 1),
            "skip": 1 + mat(c, scale=0.1), "dt_bias": mat(c, scale=0.5) - 2, "out": mat(c, out)}


def _plain_layer(p, frames, off):
    """The same in float64 with torch's own operations, for automatic differentiation on the CPU."""
    torch = _torch()
    nn = torch.nn.functional
    c, s = p["A"].shape
    rank = p["up"].shape[1]
    u = nn.layer_norm(frames, (frames.shape[1],), p["gamma"], p["beta"], 1e-5)
    outs = []
    for a, b in zip(off[:-1], off[1:]):
        both = u[a:b] @ p["in"]
        v = nn.conv1d(nn.pad(both[:, :c].t(), (p["conv"].shape[1] - 1, 0)), p["conv"][:, None], p["conv_bias"], groups=c)
        v = nn.silu(v.t())
        rows = v @ p["rows"]
        d = nn.softplus(rows[:, :rank] @ p["up"].t() + p["dt_bias"])
        h, ys = torch.zeros(c, s, dtype=torch.float64), []
        for t in range(b - a):
            h = torch.exp(d[t][:, None] * p["A"]) * h + (d[t] * v[t])[:, None] * rows[t, rank:rank + s]
            ys.append((h * rows[t, rank + s:]).sum(1) + p["skip"] * v[t])
        outs.append(torch.stack(ys) * nn.silu(both[:, c:]) @ p["out"])
    return torch.cat(outs)


def test_layer_forward_backward_and_clipping_together(sra, ctx):
    """A layer's gradients against automatic differentiation in float64, then clipped.  Every operation of it is
    good to K E with K below 2000 (60 frames, sums over 90 values), and a dozen of them follow one another."""
    torch = _torch()
    rng = np.random.default_rng(20)
    lengths = [40, 1, 60, 17]
    off = np.concatenate([[0], np.cumsum(lengths)])
    p = _layer_parameters(rng, 39, 90, 16, 6, 8)
    frames = torch.from_numpy(rng.standard_normal((118, 39)).astype(np.float32)).cuda()
    dy = torch.from_numpy(rng.standard_normal((118, 8)).astype(np.float32)).cuda()
    out, g = _layer(sra, ctx, p, frames, off, dy)
    q = {k: v.cpu().double().requires_grad_() for k, v in p.items()}
    x = frames.cpu().double().requires_grad_()
    want = _plain_layer(q, x, off)
    (want * dy.cpu().double()).sum().backward()
    tol = 12 * 2000 * E
    assert float((out.cpu().double() - want).norm() / want.norm()) < tol
    for k in g:
        ref = x.grad if k == "x" else q[k].grad
        assert float((g[k].cpu().double() - ref).norm() / ref.norm()) < tol, k
    names = sorted(p)
    total = float(sra.clip_gradients(ctx, [g[k].contiguous() for k in names], 1.0))
    ref = np.sqrt(sum(float(q[k].grad.square().sum()) for k in names))
    assert abs(total - ref) < tol * ref


def test_hybrid_model_from_posteriors_to_viterbi(sra, ctx):
    """The operators between this package's own ends: posteriors of an HMM as targets, the layer's
    log-densities into the dense decoder; frame-by-frame inference gives the batch's outputs."""
    torch = _torch()
    rng = np.random.default_rng(21)
    S, D, lengths = 3, 13, [30, 12, 25]
    bank = sra.HMMBank(ctx, rng.dirichlet(np.ones(S)), rng.dirichlet(np.ones(S), size=S),
                       rng.standard_normal((S, D)), rng.uniform(0.5, 1.5, (S, D)))
    data = sra.Ragged(ctx, rng.standard_normal((67, D)).astype(np.float32), lengths)
    _, target = bank.posteriors(data)
    p = _layer_parameters(rng, D, 24, 16, 4, S)

    def loss_and_grad(logits):
        logp = torch.log_softmax(logits, 1)
        return -(target * logp).sum() / 67, (logp.exp() * target.sum(1, keepdim=True) - target) / 67

    logits = _layer(sra, ctx, p, data.X, data)
    loss, dlogits = loss_and_grad(logits)
    logits, g = _layer(sra, ctx, p, data.X, data, dlogits)
    names = [k for k in p]
    grads = [g[k].contiguous() for k in names]
    # the gradient is that of the loss: a small step against it changes the loss by its square
    norm2 = sum(float((x.double() ** 2).sum()) for x in grads)
    h = 1e-3
    q = {k: p[k] - h * x for k, x in zip(names, grads)}
    change = float(loss_and_grad(_layer(sra, ctx, q, data.X, data))[0].double() - loss.double())
    # (second derivatives of order norm2 each way, and the losses' own rounding)
    assert abs(change + h * norm2) < 0.2 * h * norm2 + 200 * E * float(loss)
    assert float(sra.clip_gradients(ctx, grads, 0.5)) == pytest.approx(np.sqrt(norm2), rel=1e-6)
    loglik = torch.log_softmax(logits, 1).contiguous()
    lp, path = sra.viterbi_dense(ctx, loglik, data.offsets, bank.startprob[0], bank.transmat[0])
    assert torch.isfinite(lp).all() and int(path.min()) >= 0 and int(path.max()) < S
    # live: one frame of all three recordings at a time, as long as each lasts
    conv = torch.zeros(3, 3, 24, device="cuda")
    scan = torch.zeros(3, 24, 16, device="cuda")
    off = np.concatenate([[0], np.cumsum(lengths)])
    for t in range(12):                       # (all three have a frame)
        x = data.X[torch.from_numpy(off[:3] + t).cuda()]
        u = sra.layer_norm(ctx, x, p["gamma"], p["beta"])[0]
        both = u @ p["in"]
        v = sra.causal_conv_step(ctx, conv, both[:, :24], p["conv"], p["conv_bias"], "silu")
        rows = v @ p["rows"]
        y = sra.selective_scan_step(ctx, scan, v, rows[:, :4] @ p["up"].t(), p["A"], rows[:, 4:20], rows[:, 20:],
                                    skip=p["skip"], gate=both[:, 24:], dt_bias=p["dt_bias"])
        want = logits[torch.from_numpy(off[:3] + t).cuda()]
        assert float((y @ p["out"] - want).norm() / want.norm()) < 12 * 2000 * E


def test_two_streams_and_the_current_device(sra, ctx):
    """One context, two streams, nothing in between: scratch is per call, so they do not meet."""
    torch = _torch()
    rng = np.random.default_rng(22)
    cases = [_scan_case(rng, [2000], 64, 16, 1, "float32"), _scan_case(rng, [1200, 700], 64, 16, 1, "float32")]
    dys = [_draw(rng, (int(o[-1]), 64), "float32")[0] for o, _, _ in cases]
    want = [_run_scan(sra, ctx, o, t, dy) for (o, t, _), dy in zip(cases, dys)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for rep in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append((i, _run_scan(sra, ctx, cases[i][0], cases[i][1], dys[i])))
    torch.cuda.synchronize()
    for i, (y, last, g) in got:
        assert torch.equal(y, want[i][0]) and torch.equal(last, want[i][1])
        for k in g:
            assert torch.equal(g[k], want[i][2][k]), k
    assert torch.cuda.current_device() == 0


def test_captured_and_replayed(sra, ctx):
    """Forward, backward and clipping captured into a graph, replayed on new inputs with the program's own
    work and calls in between: every replay equals the eager call."""
    torch = _torch()
    rng = np.random.default_rng(23)
    off, t, v = _scan_case(rng, [400, 30], 40, 16, 1, "float32")
    o = torch.from_numpy(off).cuda()
    w = torch.from_numpy(rng.standard_normal((40, 4)).astype(np.float32)).cuda()
    dy = _draw(rng, (430, 40), "float32")[0]

    def step():
        u, mean, rstd = sra.layer_norm(ctx, t["x"])
        c, _ = sra.causal_conv(ctx, u, w, o, None, "silu")
        args = (c, t["dt"], t["A"], t["B"], t["C"], o)
        rest = {k: t[k] for k in REST}
        y, last, saved = sra.selective_scan(ctx, *args, save=True, **rest)
        g = sra.selective_scan_backward(ctx, dy, *args, saved=saved, **rest)
        gc = sra.causal_conv_backward(ctx, g["x"], u, w, o, None, "silu")
        dx, dw, db = sra.layer_norm_backward(ctx, gc["x"], t["x"], mean, rstd)
        grads = [g["A"], g["skip"], g["dt_bias"], gc["weight"]]
        norm = sra.clip_gradients(ctx, grads, 0.01)
        return [y, last, dx, dw, db, norm, *grads]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        held = step()
    for rep in range(4):
        t["x"].copy_(torch.from_numpy(rng.standard_normal((430, 40)).astype(np.float32)))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b), rep


def test_captured_with_offsets_that_change(sra, ctx):
    """The offsets are the device's: a replay after they have changed is a call with the new ones, pieces, order
    of the utterances and all; and two such calls on two streams do not meet."""
    torch = _torch()
    rng = np.random.default_rng(29)
    for lengths, c in ((rng.permutation(np.arange(10, 58)), 1400), (np.array([700, 3, 0, 297]), 24)):
        off, t, v = _scan_case(rng, lengths, c, 16, 1, "bfloat16")
        dy = _draw(rng, (int(off[-1]), c), "bfloat16")[0]
        o = torch.from_numpy(off).cuda()
        args, rest = [t[k] for k in ORDER], {k: t[k] for k in REST}

        def step():
            y, last, saved = sra.selective_scan(ctx, *args, o, save=True, **rest)
            g = sra.selective_scan_backward(ctx, dy, *args, o, saved=saved, **rest)
            return [y, last, *g.values()]

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            held = step()
        for rep in range(4):
            o.copy_(torch.from_numpy(np.concatenate([[0], np.cumsum(rng.permutation(lengths))])))
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            for k, (a, b) in enumerate(zip(held, want)):
                assert torch.equal(a, b), (rep, k)
        streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
        for st in streams * 2:
            with torch.cuda.stream(st):
                got.append(step())
        torch.cuda.synchronize()
        for other in got:
            for a, b in zip(other, want):
                assert torch.equal(a, b)


def test_state_offsets_beyond_32_bits(sra, ctx):
    """Rows at a pitch that puts the last ones more than 2^32 bytes behind the first."""
    torch = _torch()
    n, c, pitch = 5, 24, 2 ** 28 + 8
    room = torch.empty((n - 1) * pitch + 64, dtype=torch.float32, device="cuda")
    rng = np.random.default_rng(24)
    off, t, v = _scan_case(rng, [n], c, 16, 1, "float32")
    far = torch.as_strided(room, (n, c), (pitch, 1), 8)
    far.copy_(t["x"])
    y, last = _run_scan(sra, ctx, off, t)
    y2, last2 = _run_scan(sra, ctx, off, {**t, "x": far})
    assert torch.equal(y, y2) and torch.equal(last, last2)
    w = torch.from_numpy(rng.standard_normal((c, 4)).astype(np.float32)).cuda()
    a, b = sra.causal_conv(ctx, t["x"], w), sra.causal_conv(ctx, far, w)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert torch.equal(sra.layer_norm(ctx, t["x"])[0], sra.layer_norm(ctx, far)[0])


# ---- values without bound, in the single-frame form, in padded states and channels, behind a last frame ----------------

@pytest.mark.parametrize("low", [-3e38, -3.4028234663852886e38, float("-inf")])
def test_scan_step_decays_without_bound_forget_at_once(sra, ctx, low):
    """The single frame as the recording: a decay without bound is 0, the same results as with -1e30 (whose decay is 0
    at steps above 1e-28, and these are above e^-10); a step of 0, whatever A is, leaves the state as it was."""
    torch = _torch()
    rng = np.random.default_rng(30)
    off, t, v = _scan_case(rng, [1] * 6, 20, 16, 1, "float32")
    t["dt"][4], v["dt"][4] = float("-inf"), -np.inf
    got = []
    for a in (-1e30, low):
        A, state = t["A"].clone(), t["state"].clone()
        A[::3, ::2] = a
        y = sra.selective_scan_step(ctx, state, t["x"], t["dt"], A, t["B"], t["C"], skip=t["skip"], gate=t["gate"],
                                    dt_bias=t["dt_bias"])
        got.append((y, state))
    v["A"][::3, ::2] = -1e30
    args = {q: v[q] for q in (*ORDER, *REST)}
    ref, size = so.scan(off, **args), so.scan(off, scales=True, **args)
    _close(got[0][0], ref["y"], size["y"], 4 + 2 * 16 + 40, "float32", "y")
    _close(got[0][1], ref["state_out"], size["state_out"], 4 + 2 * 16 + 40, "float32", "state")
    assert torch.equal(got[1][0], got[0][0]) and torch.equal(got[1][1], got[0][1])
    assert torch.equal(got[1][1][4], t["state"][4])
    # a recording handed from one form to the other
    A = t["A"].clone()
    A[::3, ::2] = low
    state = _run_scan(sra, ctx, off, {**t, "A": A})[1]
    y = sra.selective_scan_step(ctx, state, t["x"], t["dt"], A, t["B"], t["C"], dt_bias=t["dt_bias"])
    assert torch.isfinite(y).all() and torch.isfinite(state).all()


@pytest.mark.parametrize("high", [89.0, 1000.0, 3.4028234663852886e38, float("inf")])
def test_scan_step_growth_without_bound_is_infinity(sra, ctx, high):
    """e^89 and more is infinity in 32 bits: infinite states of the old ones' signs, in both forms."""
    torch = _torch()
    rng = np.random.default_rng(31)
    off, t, v = _scan_case(rng, [1] * 3, 20, 16, 1, "float32")
    t["dt"] = torch.ones_like(t["dt"])
    t["A"] = torch.full_like(t["A"], high)
    args = [t["x"], t["dt"], t["A"], t["B"], t["C"]]
    want = torch.sign(t["state"]) * float("inf")
    _, last = sra.selective_scan(ctx, *args, torch.arange(4, device="cuda"), state=t["state"], dt_softplus=False)
    state = t["state"].clone()
    sra.selective_scan_step(ctx, state, *args, dt_softplus=False)
    assert torch.equal(last, want) and torch.equal(state, want)


def _same(got, ref, size, k, dtype, what):
    """Like _close where the definition is finite, of infinities the signs; what it leaves open (NaN) is not compared."""
    got, far = _host(got), np.isinf(ref)
    assert np.array_equal(got[far], ref[far]), f"{what}: {(got[far] != ref[far]).sum()} of {far.sum()} infinities differ"
    keep = np.isfinite(ref)
    assert np.isfinite(got[keep]).all(), f"{what}: {(~np.isfinite(got[keep])).sum()} of {keep.sum()} are not finite"
    _close(_torch().from_numpy(got[keep]), ref[keep], size[keep], k, dtype, what)


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("lengths,c,s", [([5], 20, 16), ([8, 13], 20, 16), ([1, 3, 16, 22], 40, 8), ([19], 70, 4), ([300], 24, 16),
                                         ([9, 7], 17, 24), ([12], 16, 64)])
def test_scan_infinity_in_a_last_frame_spares_the_gradients_before_it(sra, ctx, lengths, c, s):
    """An infinite state behind the last frame is no factor of any gradient but that frame's own: what the frames of
    an octet behind the end add to dA is nothing."""
    torch = _torch()
    rng = np.random.default_rng(32)
    off, t, v = _scan_case(rng, lengths, c, s, 1, "float32")
    dy, dyv = _draw(rng, (off[-1], c), "float32")
    dsov = rng.standard_normal((len(lengths), c, s)).astype(np.float32)
    for end in off[1:]:
        t["B"][end - 1], v["B"][end - 1] = float("inf"), np.inf
    args = {**{q: v[q] for q in (*ORDER, *REST)}, "dy": dyv, "dstate_out": dsov.astype(np.float64)}
    ref, size = so.scan(off, **args), so.scan(off, scales=True, **args)
    grads = _run_scan(sra, ctx, off, t, dy, torch.from_numpy(dsov).cuda())[2]
    assert np.isfinite(ref["dA"]).all() and np.isfinite(ref["dskip"]).all() and np.isfinite(ref["dstate"]).all()
    kb = 2 * (4 * max(lengths) + 2 * s + 40) + c + 64
    for q in ("A", "skip", "state", "B"):
        _same(grads[q], ref["d" + q], size["d" + q], kb + (off[-1] if q != "B" else 0), "float32", "d" + q)


@pytest.mark.parametrize("s", [3, 16])
def test_scan_in_pieces_that_begin_with_silence_and_grow(sra, ctx, s):
    """A state that is zero stays zero however much a piece would let it grow (e^32 and more per piece, beyond 32 bits
    over a few of them), forwards and for the gradients backwards.  A decay of e^1 is off by its exponent's two roundings
    and its own, less than 4 E, which the 4 L of the tolerance has."""
    torch = _torch()
    rng = np.random.default_rng(33)
    off, t, v = _scan_case(rng, [400], 24, s, 1, "float32", state=False, bias=False)
    t["dt"], v["dt"] = torch.ones_like(t["dt"]), np.ones_like(v["dt"])
    t["A"], v["A"] = torch.ones_like(t["A"]), np.ones_like(v["A"])
    t["x"][:380], v["x"][:380] = 0, 0
    dy, dyv = _draw(rng, (400, 24), "float32")
    dy[20:], dyv[20:] = 0, 0
    args = {**{q: v[q] for q in (*ORDER, *REST)}, "dy": dyv, "dt_softplus": False}
    ref, size = so.scan(off, **args), so.scan(off, scales=True, **args)
    y, last, grads = _run_scan(sra, ctx, off, t, dy, softplus=False)
    k = 4 * 400 + 2 * s + 40
    assert not y[:380].any()
    _close(y, ref["y"], size["y"], k, "float32", "y")
    _close(last, ref["state_out"], size["state_out"], k, "float32", "state_out")
    for q, grad in grads.items():
        if grad is not None:
            _close(grad, ref["d" + q], size["d" + q], 2 * k + 24 + 64 + 400, "float32", "d" + q)


def _check_infinity(sra, ctx, off, t, v, dtype, rng, which):
    """Forward and backward with an infinity in the last utterance, in the last channel or group, all else positive."""
    n, c = v["x"].shape
    longest = int(np.diff(off).max())
    for k in ("x", "B", "C", "gate", "skip"):
        t[k], v[k] = t[k].abs(), np.abs(v[k])
    dy, dyv = _draw(rng, (n, c), dtype)
    dy, dyv = dy.abs(), np.abs(dyv)
    for q in ({**t, "dy": dy}, {**v, "dy": dyv}):
        q[which][n - int(off[-1] - off[-2]) // 2 - 2, -1] = float("inf")
    args = {q: v[q] for q in (*ORDER, *REST)}
    ref, size = so.scan(off, dy=dyv, **args), so.scan(off, dy=dyv, scales=True, **args)
    got = _run_scan(sra, ctx, off, t, dy)
    k = 4 * longest + 2 * v["A"].shape[1] + 40
    _same(got[0], ref["y"], size["y"], k, dtype, "y")
    _same(got[1], ref["state_out"], size["state_out"], k, "float32", "state_out")
    for q, grad in got[2].items():
        if grad is not None:
            param = q in ("A", "skip", "dt_bias")
            _same(grad, ref["d" + q], size["d" + q], 2 * k + c + 64 + (n if param else 0), "float32" if param else dtype, "d" + q)


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("which", ["x", "dy"])
@pytest.mark.parametrize("lengths,c,s", [([300], 32, 16), ([704], 64, 4), ([129, 304], 16, 32)])
def test_scan_infinities_pass_from_piece_to_piece(sra, ctx, lengths, c, s, which):
    """Where the decay over a piece is 0 in 32 bits, that of every frame is not: infinity stays."""
    rng = np.random.default_rng(38)
    off, t, v = _scan_case(rng, lengths, c, s, 1, "float32", state=False)
    _check_infinity(sra, ctx, off, t, v, "float32", rng, which)


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("which", ["x", "dt", "B"])
@pytest.mark.parametrize("lengths,c,s,g", [([5, 9, 40], 20, 16, 1), ([21, 6], 70, 4, 1), ([24], 38, 8, 2), ([300], 20, 16, 1), ([19], 17, 64, 1)])
def test_scan_infinities_meet_no_channels_that_do_not_exist(sra, ctx, lengths, c, s, g, which, dtype):
    """The last channel stands in for those of a block that do not exist: an infinity of its own, or one of B, must not
    reach the sums over the channels as NaN.  All signs alike, so that the definition adds up no infinities of both."""
    torch = _torch()
    rng = np.random.default_rng(s + c)
    off, t, v = _scan_case(rng, lengths, c, s, g, dtype, state=False)
    _check_infinity(sra, ctx, off, t, v, dtype, rng, which)


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("which", ["x", "dt", "B"])
@pytest.mark.parametrize("lengths,c,s,g", [([5, 9, 40], 20, 1, 1), ([21, 6], 70, 3, 1), ([5, 30], 40, 7, 2), ([17, 9], 33, 13, 1),
                                           ([300], 20, 13, 1), ([300], 66, 2, 1), ([300], 40, 6, 2), ([300], 16, 20, 1),
                                           ([9, 19], 17, 24, 1), ([11], 16, 33, 1), ([200], 18, 40, 1)])
def test_scan_infinities_meet_no_states_that_do_not_exist(sra, ctx, lengths, c, s, g, which, dtype):
    """A wave has room for 4, 8, 16, 32 or 64 states: those that there are not must not turn an infinite input into NaN."""
    rng = np.random.default_rng(s + c)
    off, t, v = _scan_case(rng, lengths, c, s, g, dtype, state=False)
    _check_infinity(sra, ctx, off, t, v, dtype, rng, which)


@pytest.mark.filterwarnings("ignore::RuntimeWarning")
@pytest.mark.parametrize("s", [1, 2, 3, 7, 13, 16, 33])
def test_scan_step_infinities_meet_no_states_that_do_not_exist(sra, ctx, s):
    rng = np.random.default_rng(s)
    off, t, v = _scan_case(rng, [1] * 4, 9, s, 1, "float32")
    for k in ("x", "B", "C", "gate", "skip"):
        t[k], v[k] = t[k].abs(), np.abs(v[k])
    for q in (t, v):
        q["x"][1, 3] = q["dt"][2, 4] = q["B"][3, 0, s - 1] = float("inf")
    args = {q: v[q] for q in (*ORDER, *REST)}
    ref, size = so.scan(off, **args), so.scan(off, scales=True, **args)
    state = t["state"].clone()
    y = sra.selective_scan_step(ctx, state, *(t[k] for k in ORDER), skip=t["skip"], gate=t["gate"], dt_bias=t["dt_bias"])
    assert np.isinf(ref["y"][1, 3]) and np.isinf(ref["y"][2, 4]) and np.isinf(ref["y"][3]).all()
    _same(y, ref["y"], size["y"], 4 + 2 * s + 40, "float32", "y")
    _same(state, ref["state_out"], size["state_out"], 4 + 2 * s + 40, "float32", "state")


# ---- rows that belong to no utterance ------------------------------------------------------------------------------------

def _dirty(*shapes):
    """Leaves memory of these sizes full of NaN behind with torch's allocator."""
    torch = _torch()
    for _ in range(3):
        held = [torch.full(s, float("nan"), dtype=d, device="cuda") for s, d in shapes for _ in range(8)]
        del held


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("lengths,lead,tail,c,s,g", [([12, 0, 21], 3, 4, 37, 7, 1), ([700], 5, 1, 24, 16, 1), ([], 3, 4, 20, 16, 2),
                                                     ([3], 900, 1000, 40, 24, 1), (list(range(20, 60)), 1, 2, 1650, 16, 1)])
def test_results_that_are_new_are_zero_in_rows_of_no_utterance(sra, ctx, lengths, lead, tail, c, s, g, dtype):
    """Frames outside every utterance take no part: their gradients are 0, and so are their rows in results that the
    functions themselves allocate, whatever they hold as inputs; where the offsets come from does not matter."""
    torch = _torch()
    rng = np.random.default_rng(34)
    off, t, v = _scan_case(rng, lengths, c, s, g, dtype, state=False)
    inside, n = int(off[-1]), int(off[-1]) + lead + tail

    def room(a):
        wide = torch.full((n, *a.shape[1:]), float("nan"), dtype=a.dtype, device="cuda")
        wide[lead:lead + inside] = a
        return wide

    wide = {k: room(t[k]) for k in ("x", "dt", "B", "C", "gate")}
    dy = _draw(rng, (inside, c), dtype)[0]
    w = torch.from_numpy(rng.standard_normal((c, 4)).astype(np.float32)).cuda()
    want = _run_scan(sra, ctx, off, t, dy)
    grad = sra.causal_conv_backward(ctx, dy, t["x"], w, torch.from_numpy(off).cuda(), None, "silu")
    plain = sra.causal_conv(ctx, t["x"], w, torch.from_numpy(off).cuda(), None, "silu")[0]
    for offsets in (torch.from_numpy(off + lead).cuda(), off + lead):
        o = dict(offsets=offsets)
        _dirty(((n, c), t["x"].dtype), ((n, g, s), t["x"].dtype))
        rest, args = {k: {**t, **wide}[k] for k in REST}, [{**t, **wide}[k] for k in ORDER]
        y, last, saved = sra.selective_scan(ctx, *args, save=True, **o, **rest)
        _dirty(((n, c), t["x"].dtype), ((n, g, s), t["x"].dtype))
        got = sra.selective_scan_backward(ctx, room(dy), *args, saved=saved, **o, **rest)
        pairs = [("y", y, want[0]), *((k, got[k], want[2][k]) for k in ("x", "dt", "B", "C", "gate"))]
        _dirty(((n, c), t["x"].dtype))
        pairs.append(("conv", sra.causal_conv(ctx, wide["x"], w, activation="silu", **o)[0], plain))
        _dirty(((n, c), t["x"].dtype))
        back = sra.causal_conv_backward(ctx, room(dy), wide["x"], w, activation="silu", **o)
        pairs.append(("conv dx", back["x"], grad["x"]))
        for k, a, b in pairs:
            assert torch.equal(a[lead:lead + inside], b), k
            assert not a[:lead].any() and not a[lead + inside:].any(), k
        assert torch.equal(last, want[1])
        for a in (got["A"], got["skip"], got["dt_bias"], back["weight"]):        # (their sums' order may differ)
            assert torch.isfinite(a).all()


# ---- captured calls without offsets --------------------------------------------------------------------------------------

def test_captured_without_offsets(sra, ctx):
    """None is one utterance, made on the device; host numbers would be copied while a graph is captured and are refused
    before anything is recorded."""
    torch = _torch()
    rng = np.random.default_rng(37)
    off, t, v = _scan_case(rng, [50], 24, 16, 1, "float32")
    w = torch.from_numpy(rng.standard_normal((24, 4)).astype(np.float32)).cuda()
    dy = _draw(rng, (50, 24), "float32")[0]

    def step():
        u, _ = sra.causal_conv(ctx, t["x"], w, activation="silu")
        args, rest = (u, t["dt"], t["A"], t["B"], t["C"]), {k: t[k] for k in REST}
        y, last, saved = sra.selective_scan(ctx, *args, save=True, **rest)
        g = sra.selective_scan_backward(ctx, dy, *args, saved=saved, **rest)
        return [y, last, *g.values(), sra.causal_conv_backward(ctx, g["x"], t["x"], w, activation="silu")["weight"]]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        with pytest.raises(ValueError, match="captured"):
            sra.causal_conv(ctx, t["x"], w, [0, 50])
        held = step()
    for rep in range(4):
        t["x"].copy_(torch.from_numpy(rng.standard_normal((50, 24)).astype(np.float32)))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b), rep


# ---- shapes of the pieces, of utterances by length, and of whole blocks --------------------------------------------------

@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("lengths,c,s,g", [([700], 130, 4, 1), ([300, 41], 66, 3, 1), ([700], 40, 8, 1), ([129, 300], 96, 5, 2),
                                           ([700], 33, 24, 1), ([300, 0, 129], 40, 32, 2), ([500], 17, 64, 1)])
def test_scan_pieces_of_every_number_of_states(sra, ctx, lengths, c, s, g, dtype):
    rng = np.random.default_rng(35)
    off, t, v = _scan_case(rng, lengths, c, s, g, dtype)
    _check_scan(sra, ctx, off, t, v, dtype, rng)


@pytest.mark.parametrize("dtype,lengths,c,s,g", [("float32", 40, 3328, 4, 1), ("bfloat16", 40, 3300, 3, 2), ("float16", 40, 1650, 16, 1),
                                                 ("float16", 40, 832, 24, 1), ("bfloat16", 40, 840, 64, 1),
                                                 ("float32", 1100, 65, 12, 1)])
def test_scan_more_batches_that_fill_the_device(sra, ctx, dtype, lengths, c, s, g):
    """Utterances by length for the other numbers of states, and more utterances than are put in order."""
    rng = np.random.default_rng(36)
    lengths = rng.integers(25, 50, lengths) if lengths < 100 else rng.integers(0, 9, lengths)
    lengths[5], lengths[8] = 0, 60
    off, t, v = _scan_case(rng, lengths, c, s, g, dtype)
    _check_scan(sra, ctx, off, t, v, dtype, rng)
