"""Plain 64-bit implementations of the answer operators (numpy)."""
import numpy as np


def ref_pack(w, group):
    """Weights [C, K] -> (q [K, C] in [-7, 7], a / 7 [K, G])."""
    w = np.asarray(w, dtype=np.float64).T
    K, C = w.shape
    G = -(-C // group)
    pad = np.zeros((K, G * group))
    pad[:, :C] = w
    a = np.abs(pad).reshape(K, G, group).max(-1)
    safe = np.where(a > 0, a, 1.0)
    q = np.rint(pad.reshape(K, G, group) * 7 / safe[..., None])
    return q.reshape(K, -1)[:, :C], a / 7


def nibbles(packed, C):
    return np.stack([packed & 15, packed >> 4], -1).reshape(packed.shape[0], -1)[:, :C]


def ref_votes(x, q, scales, group, bias=None):
    """(votes, sum of the magnitudes that were added) [N, K]; q signed [K, C]."""
    s = np.repeat(scales.astype(np.float64), group, axis=1)[:, :q.shape[1]]
    w = q.astype(np.float64) * s
    y, mag = x.astype(np.float64) @ w.T, np.abs(x.astype(np.float64)) @ np.abs(w).T
    return (y, mag) if bias is None else (y + bias, mag + np.abs(bias))


def ref_answer(cs, bias=None, allowed=None, history=None, lengths=None, repetition=1.0, frequency=0.0, presence=0.0,
               temperature=1.0):
    """(choice, logprob of the rounded z, z in 64 bits); knobs as float32."""
    n, k = cs.shape
    v = cs.astype(np.float64).copy()
    knob = [np.broadcast_to(np.asarray(a, np.float32).astype(np.float64), (n,)) for a in
            (repetition, frequency, presence, temperature)]
    with np.errstate(all="ignore"):
        for i in range(n):
            if history is not None:
                h = history[i] if lengths is None else history[i][:max(0, int(lengths[i]))]
                c = np.bincount(h[(h >= 0) & (h < k)], minlength=k)
                hit = np.where(v[i] > 0, v[i] / knob[0][i], v[i] * knob[0][i]) - knob[1][i] * c - knob[2][i]
                v[i] = np.where(c > 0, hit, v[i])
        if bias is not None:
            v = v + bias.astype(np.float64)
        z = v / knob[3][:, None]
        if allowed is not None:
            z = np.where(allowed, z, -np.inf)
        r = z.astype(np.float32)
        choice, logprob = np.full(n, -1, np.int64), np.full(n, -np.inf)
        for i in range(n):
            at = np.arange(k) if allowed is None else np.nonzero(np.broadcast_to(allowed, (n, k))[i])[0]
            if len(at) == 0:
                continue
            choice[i] = at[np.argmax(r[i, at])]
            top = float(r[i, choice[i]])
            others = r[i, at[at != choice[i]]].astype(np.float64)
            logprob[i] = np.nan if np.isnan(top) else -np.log1p(np.exp(others - top).sum())
    return choice, logprob, z


def ref_loss(cs, target, bias=None, allowed=None, temperature=1.0, weight=None):
    """(loss [n], dcs [n, k], dbias [k], dtemperature) of the definition."""
    n, k = cs.shape
    t = float(np.float64(temperature))
    w = np.ones(n) if weight is None else weight.astype(np.float64)
    z = (cs.astype(np.float64) + (0 if bias is None else bias.astype(np.float64))) / t
    loss, d, dt = np.zeros(n), np.zeros((n, k)), 0.0
    for i in range(n):
        y = int(target[i])
        if not 0 <= y < k or w[i] == 0:
            continue
        at = np.arange(k) if allowed is None else np.nonzero(np.broadcast_to(allowed, (n, k))[i])[0]
        if y not in at:
            loss[i] = w[i] * np.inf
            continue
        m = z[i, at].max()
        e = np.exp(z[i, at] - m)
        loss[i] = w[i] * (np.log(e.sum()) + m - z[i, y])
        d[i, at] = w[i] * e / e.sum()
        d[i, y] -= w[i]
        dt -= (d[i, at] * z[i, at]).sum() / t
    return loss, d / t, d.sum(0) / t, dt
