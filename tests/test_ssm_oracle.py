"""The oracle of the trainable frame operators against automatic differentiation and against
differences, in float64 on the CPU; the refusals of the entry points, which need no GPU."""
import ctypes as C

import numpy as np
import pytest

from oracle import ssm_oracle as so

EPS = 1e-6


def _scan_problem(rng, lengths, c, s, g, gate=True, state=True):
    off = np.concatenate([[0], np.cumsum(lengths)])
    n = off[-1]
    p = dict(x=rng.standard_normal((n, c)), dt=rng.standard_normal((n, c)), A=-rng.uniform(0.2, 3, (c, s)),
             B=rng.standard_normal((n, g, s)), C=rng.standard_normal((n, g, s)), skip=rng.standard_normal(c),
             dt_bias=rng.standard_normal(c))
    if gate:
        p["gate"] = rng.standard_normal((n, c))
    if state:
        p["state"] = rng.standard_normal((len(lengths), c, s))
    return off, p


def _differences(loss, p, grads, rng):
    """Every gradient against the central difference along a random direction.  The difference is off by
    the step's square times third derivatives (of order 10 here), and by the rounding of its two losses
    over the step: each is a sum of terms that are a few dozen roundings of 2^-53 off, so
    64 x 2^-53 x the sum of the terms' magnitudes, over EPS."""
    for k, g in grads.items():
        v = rng.standard_normal(p[k].shape)
        up, down = dict(p), dict(p)
        up[k], down[k] = p[k] + EPS * v, p[k] - EPS * v
        terms = [np.concatenate([t.ravel() for t in loss(q)]) for q in (up, down)]
        want = (terms[0].sum() - terms[1].sum()) / (2 * EPS)
        size = np.abs(g * v).sum() + 1.0
        assert abs((g * v).sum() - want) < 1e-7 * size + 64 * 2.0 ** -53 * np.abs(terms[0]).sum() / EPS, k


@pytest.mark.parametrize("softplus", [True, False])
@pytest.mark.parametrize("gate", [True, False])
def test_scan_gradients_are_differences(softplus, gate):
    rng = np.random.default_rng(1)
    off, p = _scan_problem(rng, [5, 0, 1, 9], 6, 3, 2, gate=gate)
    if not softplus:
        p["dt"] = np.abs(p["dt"])
    dy, dso = rng.standard_normal(p["x"].shape), rng.standard_normal(p["state"].shape)

    def loss(q):
        r = so.scan(off, dt_softplus=softplus, **q)
        return r["y"] * dy, r["state_out"] * dso

    r = so.scan(off, dy=dy, dstate_out=dso, dt_softplus=softplus, **p)
    _differences(loss, p, {k: r["d" + k] for k in p}, rng)


@pytest.mark.parametrize("activation", [None, "silu"])
def test_conv_gradients_are_differences(activation):
    rng = np.random.default_rng(2)
    lengths, c, w = [4, 0, 1, 2, 11], 5, 4
    off = np.concatenate([[0], np.cumsum(lengths)])
    p = dict(x=rng.standard_normal((off[-1], c)), weight=rng.standard_normal((c, w)), bias=rng.standard_normal(c),
             state=rng.standard_normal((len(lengths), w - 1, c)))
    dy, dso = rng.standard_normal(p["x"].shape), rng.standard_normal(p["state"].shape)

    def loss(q):
        r = so.conv(off, activation=activation, **q)
        return r["y"] * dy, r["state_out"] * dso

    r = so.conv(off, activation=activation, dy=dy, dstate_out=dso, **p)
    _differences(loss, p, {k: r["d" + k] for k in p}, rng)


def test_norm_gradients_are_differences():
    rng = np.random.default_rng(3)
    p = dict(x=rng.standard_normal((4, 7)) + 2, weight=rng.standard_normal(7), bias=rng.standard_normal(7))
    dy = rng.standard_normal((4, 7))
    r = so.norm(dy=dy, **p)
    _differences(lambda q: [so.norm(**q)["y"] * dy], p, {k: r["d" + k] for k in p}, rng)


def test_scan_agrees_with_automatic_differentiation():
    import torch
    rng = np.random.default_rng(4)
    off, p = _scan_problem(rng, [7], 4, 3, 2)
    dy = rng.standard_normal(p["x"].shape)
    r = so.scan(off, dy=dy, **p)
    t = {k: torch.tensor(v, requires_grad=True) for k, v in p.items()}
    d = torch.nn.functional.softplus(t["dt"] + t["dt_bias"])
    h, ys = t["state"][0], []
    for i in range(7):
        h = torch.exp(d[i][:, None] * t["A"]) * h + (d[i] * t["x"][i])[:, None] * t["B"][i].repeat_interleave(2, 0)
        ys.append(((h * t["C"][i].repeat_interleave(2, 0)).sum(1) + t["skip"] * t["x"][i]))
    y = torch.stack(ys) * torch.nn.functional.silu(t["gate"])
    np.testing.assert_allclose(y.detach().numpy(), r["y"], rtol=1e-12)
    (y * torch.tensor(dy)).sum().backward()
    for k in p:
        np.testing.assert_allclose(t[k].grad.numpy(), r["d" + k], rtol=1e-9, atol=1e-12, err_msg=k)


# ---- refusals ---------------------------------------------------------------------------------

class _Stub:
    """What the functions ask of a context, on the CPU: nothing gets as far as a launch here."""

    def __init__(self):
        import torch
        self.device = torch.device("cpu")
        # a context's first two fields: device, compute units
        self._mem = (C.c_int32 * 256)(0, 256)
        self.handle = C.cast(self._mem, C.c_void_p)

    def stream_ptr(self):
        return None

    def tensor(self, a, dtype=None):
        import torch
        return torch.from_numpy(np.ascontiguousarray(a))


@pytest.fixture()
def scan_args():
    import torch
    n, c, s = 6, 4, 3
    return dict(x=torch.zeros(n, c), dt=torch.zeros(n, c), A=torch.zeros(c, s), B=torch.zeros(n, s), C=torch.zeros(n, s))


def _refused(match, call, *args, **kw):
    with pytest.raises(ValueError, match=match):
        call(_Stub(), *args, **kw)


def test_scan_refusals(scan_args):
    import torch
    import speech_recognition_amd as sra
    f, a = sra.selective_scan, scan_args
    _refused("must be float32, bfloat16 or float16", f, **{**a, "x": a["x"].double()})
    _refused("must be torch.float32", f, **{**a, "dt": a["dt"].half()})
    _refused("A must be float32", f, **{**a, "A": a["A"].double()})
    _refused("2-D", f, **{**a, "x": a["x"][0]})
    _refused("Shape mismatch: A", f, **{**a, "A": torch.zeros(5, 3)})
    _refused("Shape mismatch: B", f, **{**a, "B": torch.zeros(6, 4)})
    _refused("Shape mismatch: C", f, **{**a, "C": torch.zeros(5, 3)})
    _refused("3 groups", f, **{**a, "B": torch.zeros(6, 3, 3), "C": torch.zeros(6, 3, 3)})
    _refused("rows of x must be contiguous", f, **{**a, "x": torch.zeros(4, 6).t()})
    _refused("rows of dt overlap", f, **{**a, "dt": torch.zeros(1, 4).expand(6, 4)})
    _refused("Shape mismatch: skip", f, skip=torch.zeros(3), **a)
    _refused("Shape mismatch: gate", f, gate=torch.zeros(6, 5), **a)
    _refused("state must be", f, state=torch.zeros(2, 4, 3), **a)
    _refused("state_out must be", f, state_out=torch.zeros(1, 4, 3, dtype=torch.float64), **a)
    _refused("requires grad", f, **{**a, "x": a["x"].clone().requires_grad_()})
    _refused("offsets must lie between", f, offsets=[0, 7], **a)
    _refused("negative utterance length", f, offsets=[0, 4, 2], **a)
    _refused("int64 tensor", f, offsets=torch.zeros(2, dtype=torch.int32), **a)
    _refused("shares memory", f, out=a["x"], **a)
    _refused("shares memory", f, state_out=a["A"][None], **a)
    wide = dict(a, A=torch.zeros(4, 65), B=torch.zeros(6, 65), C=torch.zeros(6, 65))
    _refused(r"n_states 65 outside \[1, 64\]", f, **wide)
    _refused("state must be given", sra.selective_scan_step, None, **a)
    _refused("state must be", sra.selective_scan_step, torch.zeros(6, 4, 2), **a)
    _refused("Shape mismatch: dy", sra.selective_scan_backward, torch.zeros(6, 3), **a)
    _refused("saved must be", sra.selective_scan_backward, torch.zeros(6, 4), saved=torch.zeros(3), **a)


def test_scan_refuses_results_over_parameters_and_what_it_did_not_save(scan_args):
    import torch
    import speech_recognition_amd as sra
    a = scan_args
    room = torch.zeros(24)
    _refused("out shares memory", sra.selective_scan, out=room.view(6, 4), state=room[:12].view(1, 4, 3), **a)
    _refused("out shares memory", sra.selective_scan, out=room.view(6, 4), **{**a, "A": room[12:].view(4, 3)})
    _refused("out shares memory", sra.selective_scan_step, torch.zeros(6, 4, 3), out=room.view(6, 4), skip=room[:4], **a)
    wide = dict(a, A=torch.zeros(4, 65), B=torch.zeros(6, 65), C=torch.zeros(6, 65))
    _refused(r"n_states 65 outside \[1, 64\]", sra.selective_scan, save=True, **wide)
    _refused(r"n_states 65 outside \[1, 64\]", sra.selective_scan_backward, torch.zeros(6, 4), **wide)
    from speech_recognition_amd import _lib
    size = _lib.lib.srx_selective_scan_saved(C.byref(_lib.Scan(4, 3, 1, 1, 1, None, None)), 1, 6)
    for saved in (torch.zeros(2 * size)[::2], torch.zeros(1, size), torch.zeros(size).double(), [0.0] * size):
        _refused("saved must be", sra.selective_scan_backward, torch.zeros(6, 4), saved=saved, **a)


def test_a_result_beside_its_input_in_one_matrix_is_not_refused():
    """Two halves of one projection: their memory ranges overlap, their values do not."""
    import torch
    from speech_recognition_amd import ssm
    both = torch.zeros(6, 8)
    ssm._apart(both[:, :4], "out", both[:, 4:], None, both[:0])
    ssm._apart(both[:, 4:], "out", both[:, :4])
    for bad in (both[:, 2:6], both[1:, :4], both):
        with pytest.raises(ValueError, match="shares memory"):
            ssm._apart(both[:, :4], "out", bad)


def test_conv_norm_and_clip_refusals():
    import torch
    import speech_recognition_amd as sra
    x, w = torch.zeros(6, 4), torch.zeros(4, 3)
    _refused("activation", sra.causal_conv, x, w, activation="tanh")
    _refused(r"width 9 outside \[1, 8\]", sra.causal_conv, x, torch.zeros(4, 9))
    _refused(r"width 0 outside \[1, 8\]", sra.causal_conv_step, torch.zeros(6, 0, 4), x, torch.zeros(4, 0))
    _refused("Shape mismatch: weight", sra.causal_conv, x, torch.zeros(5, 3))
    _refused("weight must be float32", sra.causal_conv, x, w.half())
    _refused("state must be", sra.causal_conv, x, w, state=torch.zeros(1, 3, 4))
    _refused("shares memory", sra.causal_conv, x, w, out=x)
    _refused("Shape mismatch: dy", sra.causal_conv_backward, torch.zeros(5, 4), x, w)
    _refused("2-D", sra.layer_norm, x[0])
    _refused("eps must not be negative", sra.layer_norm, x, eps=-1.0)
    _refused("Shape mismatch: mean", sra.layer_norm_backward, x, x, torch.zeros(5), torch.zeros(6))
    clip = sra.clip_gradients
    _refused("float32, bfloat16 or float16", clip, [x.double()], 1.0)
    _refused("max_norm must not be negative", clip, [x], -1.0)
    _refused("max_norm must not be negative", clip, [x], float("nan"))
    _refused("without gaps", clip, [torch.zeros(4, 6)[:, ::2]], 1.0)
    _refused("overlap", clip, [x, x], 1.0)                       # the same tensor twice
    _refused("overlap", clip, [x, x[2:3]], 1.0)
    _refused("overlap", clip, [x, w], 1.0, out=[torch.zeros(6, 4), x.view(-1)[:12].view(4, 3)])
    _refused("1 gradients but 0 outputs", clip, [x], 1.0, out=[])
    _refused("shape and order", clip, [x], 1.0, out=[torch.zeros(4, 6)])
    _refused("type or float32", clip, [x.half()], 1.0, out=[torch.zeros(6, 4, dtype=torch.bfloat16)])


def test_c_entry_points_refuse_what_the_python_layer_cannot_pass():
    import speech_recognition_amd as sra
    from speech_recognition_amd import _lib
    lib, stub = _lib.lib, _Stub()
    scan = _lib.Scan(4, 3, 1, 1, 1, None, None)
    rows = _lib.ScanInputs()
    assert lib.srx_selective_scan(None, C.byref(scan), C.byref(rows), 0, None, 0, 0, None, None, None, 0, None, None, 0, None) \
        == _lib.SRX_EINVAL
    assert b"NULL context" in lib.srx_last_error()
    h = stub.handle
    assert lib.srx_selective_scan(h, C.byref(scan), C.byref(rows), 1, None, 0, 0, None, None, None, 0, None, None, 0, None) \
        == _lib.SRX_EINVAL and b"unknown dtype 1" in lib.srx_last_error()
    assert lib.srx_selective_scan(h, C.byref(scan), C.byref(rows), 0, None, 1, 5, None, None, None, 0, None, None, 0, None) \
        == _lib.SRX_EINVAL and b"NULL input" in lib.srx_last_error()
    rows = _lib.ScanInputs(1, 1, 1, 1, None, 3, 4, 3, 3, 0)
    assert lib.srx_selective_scan(h, C.byref(scan), C.byref(rows), 0, None, 1, 5, None, None, None, 0, None, None, 0, None) \
        == _lib.SRX_EINVAL and b"pitch" in lib.srx_last_error()
    rows.ld_x = 4
    assert lib.srx_selective_scan(h, C.byref(scan), C.byref(rows), 0, 1, 1, 5000, None, None, 1, 4, None, None, 0, None) \
        == _lib.SRX_EINVAL and b"workspace" in lib.srx_last_error()
    assert lib.srx_selective_scan_workspace(h, C.byref(_lib.Scan(4, 3, 3, 1, 1, None, None)), 1, 5) == -1
    assert lib.srx_selective_scan_workspace(h, C.byref(scan), -1, 5) == -1
    conv = _lib.Conv(4, 3, 2, 0, 1, None)
    assert lib.srx_causal_conv(h, C.byref(conv), 0, None, 4, None, 0, 0, None, None, None, 4, None) == _lib.SRX_EINVAL
    assert lib.srx_layer_norm(h, None, 4, 0, 1, 0, None, None, 1e-5, None, 4, None, None, None) == _lib.SRX_EINVAL
    assert lib.srx_clip_gradients(h, 1, None, None, None, None, None, 1.0, None, None, 0, None) == _lib.SRX_EINVAL
    for fn, args in ((lib.srx_emission_loglik, (h, None, 2, 0, None, None, None)),
                     (lib.srx_column_moments, (h, None, 3, 1, 1, None, None, None))):
        assert fn(*args) == _lib.SRX_EINVAL            # the new element types are the new operators' alone


def test_sizes_beyond_what_32_bits_count_are_refused():
    from speech_recognition_amd import _lib
    lib, h, many = _lib.lib, _Stub().handle, 2 ** 24 + 1
    scan = _lib.Scan(many, 3, 1, 1, 1, None, None)
    assert lib.srx_selective_scan_workspace(h, C.byref(scan), 1, 5) == -1 and b"2^24" in lib.srx_last_error()
    conv = _lib.Conv(many, 3, 0, 0, 1, None)
    assert lib.srx_causal_conv_step(h, C.byref(conv), 0, None, many, 0, None, None, many, None) == _lib.SRX_EINVAL
    assert b"2^24" in lib.srx_last_error()
    assert lib.srx_layer_norm(h, None, many, 0, 0, many, None, None, 1e-5, None, many, None, None, None) == _lib.SRX_EINVAL
    assert lib.srx_layer_norm_backward_workspace(h, 1, many) == -1 and b"2^24" in lib.srx_last_error()
    # a wave reaches four rows of the channels' matrices, 16 of B and C, with 32-bit offsets
    scan = _lib.Scan(4, 3, 1, 1, 1, None, None)
    for rows in (_lib.ScanInputs(1, 1, 1, 1, None, 2 ** 29, 4, 3, 3, 0), _lib.ScanInputs(1, 1, 1, 1, None, 4, 2 ** 40, 3, 3, 0),
                 _lib.ScanInputs(1, 1, 1, 1, None, 4, 4, 2 ** 27, 3, 0), _lib.ScanInputs(1, 1, 1, 1, 1, 4, 4, 3, 3, 2 ** 62)):
        assert lib.srx_selective_scan(h, C.byref(scan), C.byref(rows), 0, 1, 1, 5, None, None, 1, 4, None, None, 0, None) \
            == _lib.SRX_EINVAL and b"pitch" in lib.srx_last_error()
    rows = _lib.ScanInputs(1, 1, 1, 1, None, 4, 4, 3, 3, 0)
    assert lib.srx_selective_scan(h, C.byref(scan), C.byref(rows), 0, 1, 1, 5, None, None, 1, 2 ** 29, None, None, 0, None) \
        == _lib.SRX_EINVAL and b"pitch" in lib.srx_last_error()


def test_workspace_sizes_grow_with_the_problem():
    from speech_recognition_amd import _lib
    h = _Stub().handle
    scan = _lib.Scan(512, 16, 1, 1, 1, None, None)
    lib = _lib.lib
    assert lib.srx_selective_scan_workspace(h, C.byref(scan), 4096, 4096 * 200) == 0       # whole utterances
    one = lib.srx_selective_scan_workspace(h, C.byref(scan), 1, 24000)                     # pieces of one
    assert one > 0 and lib.srx_selective_scan_backward_workspace(h, C.byref(scan), 1, 24000) > one
    assert lib.srx_selective_scan_saved(C.byref(scan), 1, 24000) == (3000 + 1) * 512 * 16


@pytest.mark.parametrize("bad", [None, 1.0, [[0.0] * 4] * 6, np.zeros((6, 4), np.float32)])
def test_what_is_no_tensor_is_refused_by_name(scan_args, bad):
    import torch
    import speech_recognition_amd as sra
    a, x = scan_args, torch.zeros(6, 4)
    for k in ("x", "dt", "A", "B", "C"):
        _refused(f"{k} must be", sra.selective_scan, **{**a, k: bad})
        _refused(f"{k} must be", sra.selective_scan_step, torch.zeros(6, 4, 3), **{**a, k: bad})
        _refused(f"{k} must be", sra.selective_scan_backward, x, **{**a, k: bad})
    _refused("dy must be", sra.selective_scan_backward, bad, **a)
    _refused("dy must be", sra.causal_conv_backward, bad, x, torch.zeros(4, 3))
    _refused("weight must be", sra.causal_conv, x, bad)
    _refused("x must be", sra.causal_conv, bad, torch.zeros(4, 3))
    _refused("x must be", sra.layer_norm, bad)
    _refused("dy must be", sra.layer_norm_backward, bad, x, torch.zeros(6), torch.zeros(6))
    _refused("mean must be", sra.layer_norm_backward, x, x, bad, torch.zeros(6))
    _refused("rstd must be", sra.layer_norm_backward, x, x, torch.zeros(6), bad)
    _refused(r"grads\[0\] must be", sra.clip_gradients, [bad], 1.0)
    if bad is not None:
        for k in ("gate", "skip", "dt_bias", "state"):
            _refused(f"{k} must be", sra.selective_scan, **{**a, k: bad})
        _refused("out must be", sra.selective_scan, out=bad, **a)
        _refused("state_out must be", sra.selective_scan, state_out=bad, **a)
        _refused("bias must be", sra.causal_conv, x, torch.zeros(4, 3), bias=bad)


def test_conv_backward_sums_at_most_512_frames_in_a_row():
    """The taps' gradients: every thread's own sum in 32 bits, the rest in 64.  16 pieces of 32 frames a thread, as long
    as a grid's second dimension has room."""
    from speech_recognition_amd import _lib
    h = _Stub().handle
    for channels, lanes in ((256, 64), (32, 8), (1000, 64)):
        for utts, frames in ((1, 100), (64, 12800), (1, 1 << 20), (5000, 10 ** 7), (1, 10 ** 8)):
            size = _lib.lib.srx_causal_conv_backward_workspace(h, C.byref(_lib.Conv(channels, 4, 0, 0, 1, None)), utts, frames)
            parts, rows = size // (5 * channels * 4), 256 // lanes
            pieces = frames // 32 + utts
            assert -(-pieces // (parts * rows)) * 32 <= 512, (channels, utts, frames, parts)


@pytest.mark.parametrize("channels,states,groups", [(20, 16, 5), (40, 12, 40), (512, 17, 1), (100, 64, 1), (66, 3, 2), (70, 8, 1)])
def test_saved_states_take_room_for_the_widest_block_and_no_more(channels, states, groups):
    """Channels of a group up to whole blocks of 64 (up to 4 states), 32 (up to 16) or 16, states up to 4, 8, 16, 32 or 64."""
    from speech_recognition_amd import _lib
    block, room = (64 if states <= 4 else 32 if states <= 16 else 16), next(r for r in (4, 8, 16, 32, 64) if states <= r)
    for utts, frames in ((1, 1000), (3, 50), (40, 5000)):
        size = _lib.lib.srx_selective_scan_saved(C.byref(_lib.Scan(channels, states, groups, 1, 1, None, None)), utts, frames)
        wide = -(-(channels // groups) // block) * block * groups
        assert size == (frames // 8 + utts) * wide * room + (utts if utts >= 16 else 0)
