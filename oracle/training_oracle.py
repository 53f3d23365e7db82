"""Activations in 8 bits, the gated activation over them, token log-probabilities and the preference loss, in 64 bits on the CPU: what
tests/test_gpu_act8.py and tests/test_gpu_preference.py hold the kernels to.  Test infrastructure only."""
import numpy as np

BLOCK = 32


def least_scale(top):
    """float64 array of the least bfloat16 s with 127 s >= top, top >= 0 finite: 8 leading bits, exponents from -126 on, multiples of 2^-133 below."""
    top = np.asarray(top, dtype=np.float64)
    _, e = np.frexp(top / 127.0)                               # top / 127 = m 2^e, m in [0.5, 1)
    unit = np.ldexp(1.0, np.maximum(e - 8, -133))
    k = np.ceil(top / 127.0 / unit)
    k = np.where(127.0 * (k - 1) * unit >= top, k - 1, k)      # the quotient's own rounding; 127 k unit is exact
    k = np.where(127.0 * k * unit < top, k + 1, k)
    return np.where(top > 0, k * unit, 0.0)


def act8(x):
    """(codes int64 of x's shape, scales float64 [ceil(n / 32)]; NaN scale and codes 0 for blocks with an infinity or NaN) of float64 x."""
    x = np.asarray(x, dtype=np.float64)
    flat = x.reshape(-1)
    g = np.concatenate([flat, np.zeros(-flat.size % BLOCK)]).reshape(-1, BLOCK)
    fine = np.isfinite(g).all(1)
    g = np.where(fine[:, None], g, 0.0)
    s = least_scale(np.abs(g).max(1) if g.size else np.zeros(0))
    q = np.rint(g / np.where(s > 0, s, 1.0)[:, None])          # 64 bits hold the quotients of 24-bit values by 8-bit scales apart from ties
    return q.astype(np.int64).reshape(-1)[:flat.size].reshape(x.shape), np.where(fine, s, np.nan)


def held(x):
    """The float64 values that x's 8 bits stand for."""
    q, s = act8(x)
    return (q.reshape(-1) * np.repeat(s, BLOCK)[:q.size]).reshape(q.shape)


def sigmoid(x):
    e = np.exp(-np.abs(x))
    return np.where(x >= 0, 1.0, e) / (1.0 + e)


def silu_mul(gate, up):
    gate, up = (np.asarray(t, dtype=np.float64) for t in (gate, up))
    return gate * sigmoid(gate) * up


def silu_mul_bwd(dout, gate, up):
    """(dgate, dup) at gate, up."""
    dout, gate, up = (np.asarray(t, dtype=np.float64) for t in (dout, gate, up))
    s = sigmoid(gate)
    return dout * up * s * (1.0 + gate * (1.0 - s)), dout * gate * s


def token_logps(logits, labels):
    """(logps, softmax) float64 of logits [..., V]; logps 0 where labels are no words."""
    x = np.asarray(logits, dtype=np.float64)
    v = x.shape[-1]
    with np.errstate(all="ignore"):
        top = x.max(-1, keepdims=True)
        d = x - top
        total = np.log(np.exp(d).sum(-1, keepdims=True))
        lp = d - total
    word = (labels >= 0) & (labels < v)
    mine = np.take_along_axis(lp, np.where(word, labels, 0)[..., None], -1)[..., 0]
    return np.where(word, mine, 0.0), np.exp(lp)


def logits_grad(softmax, labels, coef):
    """coef (1[label] - softmax), zero rows where labels are no words."""
    v = softmax.shape[-1]
    word = (labels >= 0) & (labels < v)
    g = -softmax.copy()
    at = np.where(word, labels, 0)[..., None]
    np.put_along_axis(g, at, np.take_along_axis(g, at, -1) + 1.0, -1)
    return np.where(word[..., None], g * np.asarray(coef, dtype=np.float64)[..., None], 0.0)


def preference(logps, ref, labels, v, beta, smoothing):
    """(loss, rewards [2P], coef [2P]) float64."""
    word = (labels >= 0) & (labels < v)
    with np.errstate(invalid="ignore"):
        r = np.where(word, logps - np.where(word, ref, 0.0), 0.0).sum(-1)
    p = r.size // 2
    z = beta * (r[:p] - r[p:])
    soft = np.log1p(np.exp(-np.abs(z)))
    one = (1 - smoothing) * (soft + np.maximum(-z, 0)) + (smoothing * (soft + np.maximum(z, 0)) if smoothing else 0.0)
    dz = (smoothing * sigmoid(z) - (1 - smoothing) * sigmoid(-z)) * beta / p
    return one.mean(), beta * r, np.concatenate([dz, -dz])
