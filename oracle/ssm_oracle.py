"""CPU oracle of the trainable frame operators (test infrastructure): selective scan, short causal
convolution, layer norm and gradient clipping in float64 numpy, frame after frame from the
definitions.  The reference has no such operators; this is their definition here.

Every function also takes the ABSOLUTE problem: the recursions are sums of products, so the same run
over absolute values (``scales=True``) gives for every result the sum of the magnitudes that went into
it, which is what rounding errors are measured against."""
import numpy as np


def softplus(v):
    return np.logaddexp(v, 0.0)


def sigmoid(v):
    return 1.0 / (1.0 + np.exp(-np.clip(v, -700, 700)))


def _abs(on, *arrays):
    return [None if a is None else (np.abs(a) if on else a) for a in arrays]


def scan(off, x, dt, A, B, C, skip=None, gate=None, dt_bias=None, dt_softplus=True, state=None, dy=None,
         dstate_out=None, scales=False):
    """x, dt, gate, dy: (n, c); B, C: (n, g, s); A: (c, s); state: (U, c, s).  Returns a dict with y,
    state_out and, with dy, the gradients d<name>.  Rows outside every utterance are NaN."""
    n, c = x.shape
    g, s = B.shape[1:]
    per = c // g
    raw = dt + (0.0 if dt_bias is None else dt_bias)
    d = softplus(raw) if dt_softplus else raw
    draw = sigmoid(raw) if dt_softplus else np.ones_like(raw)
    silu = dsilu = np.ones_like(x)
    if gate is not None:
        sg = sigmoid(gate)
        silu, dsilu = gate * sg, sg * (1 + (np.abs(gate) if scales else gate) * (1 - sg))
    decay_A = A
    x, B, C, skip, state, dy, dstate_out, silu, dsilu, A, step = _abs(
        scales, x, B, C, skip, state, dy, dstate_out, silu, dsilu, A, d)
    skip0 = np.zeros(c) if skip is None else skip
    U = len(off) - 1
    out = {"y": np.full((n, c), np.nan), "state_out": np.zeros((U, c, s))}
    grads = {k: np.full(v.shape, np.nan) for k, v in
             (("dx", x), ("ddt", x), ("dB", B), ("dC", C), ("dgate", x))}
    grads.update(dA=np.zeros((c, s)), dskip=np.zeros(c), ddt_bias=np.zeros(c), dstate=np.zeros((U, c, s)))
    for u in range(U):
        a0, a1 = off[u], off[u + 1]
        h = np.zeros((c, s)) if state is None else state[u].copy()
        hs, inner = [h], np.zeros((a1 - a0, c))
        Bc, Cc = np.repeat(B[a0:a1], per, axis=1), np.repeat(C[a0:a1], per, axis=1)
        a = np.exp(d[a0:a1, :, None] * decay_A)
        for t in range(a1 - a0):
            h = a[t] * h + (step[a0 + t] * x[a0 + t])[:, None] * Bc[t]
            hs.append(h)
            inner[t] = (Cc[t] * h).sum(1) + skip0 * x[a0 + t]
        out["y"][a0:a1] = inner * silu[a0:a1]
        out["state_out"][u] = h
        if dy is None:
            continue
        dp = dy[a0:a1] * silu[a0:a1]
        grads["dgate"][a0:a1] = dy[a0:a1] * inner * dsilu[a0:a1]
        carry = np.zeros((c, s)) if dstate_out is None else dstate_out[u].copy()
        for t in range(a1 - a0 - 1, -1, -1):
            row = a0 + t
            dh = dp[t][:, None] * Cc[t] + carry
            grads["dC"][row] = (dp[t][:, None] * hs[t + 1]).reshape(g, per, s).sum(1)
            grads["dB"][row] = (dh * (step[row] * x[row])[:, None]).reshape(g, per, s).sum(1)
            du = (dh * Bc[t]).sum(1)
            carry = dh * a[t]
            m = carry * hs[t]
            dd = ((m * A).sum(1) + du * x[row]) * draw[row]
            grads["dA"] += m * step[row][:, None]
            grads["dx"][row] = du * step[row] + dp[t] * skip0
            grads["ddt"][row] = dd
            grads["ddt_bias"] += dd
            grads["dskip"] += dp[t] * x[row]
        grads["dstate"][u] = carry
    if dy is not None:
        out.update(grads)
    return out


def conv(off, x, weight, bias=None, activation=None, state=None, dy=None, dstate_out=None, scales=False):
    """x: (n, c), weight: (c, w), state: (U, w - 1, c).  Returns a dict like ``scan``'s."""
    n, c = x.shape
    w = weight.shape[1]
    U = len(off) - 1
    out = {"y": np.full((n, c), np.nan), "state_out": np.zeros((U, w - 1, c))}
    grads = {"dx": np.full((n, c), np.nan), "dweight": np.zeros((c, w)), "dbias": np.zeros(c),
             "dstate": np.zeros((U, w - 1, c))}
    for u in range(U):
        a0, a1 = off[u], off[u + 1]
        before = np.zeros((w - 1, c)) if state is None else state[u]
        rows = np.concatenate([before, x[a0:a1]])
        v = np.zeros((a1 - a0, c)) + (0.0 if bias is None else bias)
        for k in range(w):
            v = v + rows[k:k + a1 - a0] * weight[:, k]
        sg = sigmoid(v)
        size = v
        if scales:
            size = np.zeros_like(v) + (0.0 if bias is None else np.abs(bias))
            for k in range(w):
                size = size + np.abs(rows[k:k + a1 - a0] * weight[:, k])
        out["y"][a0:a1] = size * (sg if not scales else 1.1) if activation == "silu" else size
        out["state_out"][u] = rows[a1 - a0:]
        if dy is None:
            continue
        slope = sg * (1 + v * (1 - sg)) if activation == "silu" else np.ones_like(v)
        gr = dy[a0:a1] * slope
        W, R = weight, rows
        if scales:
            # (the slope moves by at most half of what its argument is off by)
            gr, W, R = np.abs(dy[a0:a1]) * (1.1 + 0.5 * size if activation == "silu" else 1.0), np.abs(weight), np.abs(rows)
        dr = np.zeros((a1 - a0 + w - 1, c))
        for k in range(w):
            dr[k:k + a1 - a0] += gr * W[:, k]
            grads["dweight"][:, k] += (gr * R[k:k + a1 - a0]).sum(0)
        grads["dbias"] += gr.sum(0)
        if dstate_out is not None:
            dr[a1 - a0:] += np.abs(dstate_out[u]) if scales else dstate_out[u]
        grads["dx"][a0:a1] = dr[w - 1:]
        grads["dstate"][u] = dr[:w - 1]
    if dy is not None:
        out.update(grads)
    return out


def norm(x, weight=None, bias=None, eps=1e-5, dy=None):
    mean = x.mean(1)
    rstd = 1 / np.sqrt(((x - mean[:, None]) ** 2).mean(1) + eps)
    unit = (x - mean[:, None]) * rstd[:, None]
    w = np.ones(x.shape[1]) if weight is None else weight
    out = {"y": unit * w + (0.0 if bias is None else bias), "mean": mean, "rstd": rstd}
    if dy is not None:
        g = dy * w
        out["dx"] = rstd[:, None] * (g - g.mean(1, keepdims=True) - unit * (g * unit).mean(1, keepdims=True))
        out["dweight"], out["dbias"] = (dy * unit).sum(0), dy.sum(0)
    return out


def clip(grads, max_norm):
    total = float(np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in grads)))
    factor = 1.0
    if np.isfinite(total) and total + 1e-6 > max_norm:
        factor = max_norm / (total + 1e-6)
    return total, [g * factor for g in grads]
