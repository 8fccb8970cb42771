"""The sequence-layer operators' definitions in 64 bits (numpy), with their gradients."""
import numpy as np


def gated_delta(q, k, v, g, beta, scale=None, state=None, grad_o=None, grad_state=None):
    """One sequence through the gated delta rule, token by token: q, k [T, Hk, dk],
    v [T, H, dv], g, beta [T, H], state [H, dk, dv].  -> (o, final state), and with ``grad_o``
    (and ``grad_state``) the gradients (dq, dk, dv, dg, dbeta, dstate) of their weighted sum."""
    q, k, v, g, beta = (np.asarray(x, np.float64) for x in (q, k, v, g, beta))
    T, hk, dk = q.shape
    h, dv = v.shape[1:]
    group = h // hk
    scale = dk ** -0.5 if scale is None else scale
    s = np.zeros((h, dk, dv)) if state is None else np.asarray(state, np.float64).copy()
    qh, kh = np.repeat(q, group, 1), np.repeat(k, group, 1)
    o, kept = np.zeros_like(v), []
    for t in range(T):
        kept.append(s)
        with np.errstate(under='ignore'):
            sd = np.exp(g[t])[:, None, None] * s
        u = beta[t][:, None] * (v[t] - np.einsum('hde,hd->he', sd, kh[t]))
        s = sd + kh[t][:, :, None] * u[:, None]
        o[t] = scale * np.einsum('hde,hd->he', s, qh[t])
    if grad_o is None:
        return o, s
    do = np.asarray(grad_o, np.float64)
    ds = np.zeros_like(s) if grad_state is None else np.asarray(grad_state, np.float64).copy()
    dqh, dkh = np.zeros_like(qh), np.zeros_like(kh)
    dvv, dg, db = np.zeros_like(v), np.zeros_like(g), np.zeros_like(beta)
    for t in reversed(range(T)):
        decay = np.exp(g[t])[:, None, None]
        sd = decay * kept[t]
        miss = v[t] - np.einsum('hde,hd->he', sd, kh[t])
        u = beta[t][:, None] * miss
        st = sd + kh[t][:, :, None] * u[:, None]
        dqh[t] = scale * np.einsum('hde,he->hd', st, do[t])
        ds = ds + scale * qh[t][:, :, None] * do[t][:, None]
        du = np.einsum('hde,hd->he', ds, kh[t])
        dmiss = beta[t][:, None] * du
        db[t] = (du * miss).sum(1)
        dvv[t] = dmiss
        dkh[t] = np.einsum('hde,he->hd', ds, u) - np.einsum('hde,he->hd', sd, dmiss)
        ds = ds - kh[t][:, :, None] * dmiss[:, None]
        dg[t] = (ds * sd).sum((1, 2))
        ds = decay * ds
    fold = lambda x: x.reshape(T, hk, group, dk).sum(2)                       # noqa: E731
    return (o, s), (fold(dqh), fold(dkh), dvv, dg, db, ds)


def norm_gate_residual(y, post=None, gate=None, scale=None, residual=None, pre=None, eps=1e-6,
                       grad_stream=None, grad_normed=None):
    """Norm, gate, scale, residual and the next norm over rows [R, D] -> (stream, normed or None),
    and with ``grad_stream`` the dict of gradients by argument."""
    f = lambda x: None if x is None else np.asarray(x, np.float64)             # noqa: E731
    y, post, gate, scale, residual, pre = map(f, (y, post, gate, scale, residual, pre))
    one = np.ones(1)
    r1 = (np.mean(y * y, 1, keepdims=True) + eps) ** -0.5 if post is not None else one
    w1 = post if post is not None else one
    sg = 1 / (1 + np.exp(-gate)) if gate is not None else one
    act = gate * sg if gate is not None else one
    c = scale if scale is not None else one
    stream = y * r1 * w1 * act * c + (residual if residual is not None else 0)
    r2 = (np.mean(stream * stream, 1, keepdims=True) + eps) ** -0.5
    normed = stream * r2 * pre if pre is not None else None
    if grad_stream is None and grad_normed is None:
        return stream, normed
    out = {}
    d = np.zeros_like(stream) if grad_stream is None else f(grad_stream)
    if pre is not None and grad_normed is not None:
        dn, n = f(grad_normed), stream * r2
        out['pre'] = (dn * n).sum(0)
        dn = dn * pre
        d = d + r2 * (dn - n * (dn * n).mean(1, keepdims=True))
    if residual is not None:
        out['residual'] = d
    if scale is not None:
        out['scale'] = (d * y * r1 * w1 * act).sum(0)
    if gate is not None:
        out['gate'] = d * c * y * r1 * w1 * sg * (1 + gate * (1 - sg))
    dp = d * c * act
    if post is not None:
        n = y * r1
        out['post'] = (dp * n).sum(0)
        dp = dp * w1
        dp = r1 * (dp - n * (dp * n).mean(1, keepdims=True))
    out['y'] = dp
    return (stream, normed), out


def int8_quantize(x):
    """Rows of x in 8 bits: a = max|x| / 127 and round-half-even of x / a = 127 x / max|x| (one
    rounding, so halves of 16-bit values are met exactly); 0 for a row of 0."""
    x = np.asarray(x, np.float64)
    top = np.abs(x).max(1, keepdims=True) if x.shape[1] else np.zeros((x.shape[0], 1))
    x8 = np.where(top > 0, np.rint(127 * x / np.where(top > 0, top, 1)), 0.0)
    return x8, top[:, 0] / 127


def int8_linear(x, w8, w_scale, bias=None):
    x8, a = int8_quantize(x)
    y = (x8 @ np.asarray(w8, np.float64).T) * a[:, None] * np.asarray(w_scale, np.float64)
    return y if bias is None else y + np.asarray(bias, np.float64)
