"""Plain 64-bit implementations of the packed-batch operators, for the tests."""
import numpy as np


def offsets(lengths, total, padded=0):
    n = np.maximum(np.asarray(lengths, np.int64), 0)
    if padded:
        n = np.minimum(n, padded)
    return np.minimum(np.concatenate([[0], np.cumsum(n)]), total)


def plan(lengths, total, padded=0):
    """offsets, doc, pos, slots (hb_pack_plan)."""
    off = offsets(lengths, total, padded)
    doc, pos = np.full(total, -1), np.zeros(total, np.int64)
    for b in range(len(lengths)):
        doc[off[b]:off[b + 1]] = b
        pos[off[b]:off[b + 1]] = np.arange(off[b + 1] - off[b])
    return off, doc, pos, np.where(doc < 0, -1, doc * padded + pos)


def blocks(off, total):
    """Blocks of up to 128 rows: (document, first row), rows behind the last as
    document B, (-1, 0) to the end of the table."""
    B, end = len(off) - 1, off[-1]
    got = [(b, t) for b in range(B) for t in range(off[b], off[b + 1], 128)] + [(B, t) for t in range(end, total, 128)]
    return np.array(got + [(-1, 0)] * (total // 128 + B + 1 - len(got)))


def angles(positions, D, base, sections):
    """cos and sin [T, D / 2] by the contract's f32 angle rule."""
    half = D // 2
    ex = (-(np.arange(half) / half).astype(np.float32).astype(np.float64) * float(np.float32(np.log2(base)))).astype(np.float32)
    inv = np.exp2(ex.astype(np.float64)).astype(np.float32).astype(np.float64)
    axis = np.repeat(np.arange(len(sections)), sections)
    th = (np.asarray(positions, np.float64)[axis].T * inv).astype(np.float32).astype(np.float64)
    return np.cos(th), np.sin(th)


def rope_at(x, positions, base, sections):
    x = np.asarray(x, np.float64)
    c, s = (a[:, None, :] for a in angles(positions, x.shape[-1], base, sections))
    a, b = np.split(x, 2, -1)
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def visible(nq, nk, causal, window, prefix):
    p, j = np.arange(nq)[:, None] + nk - nq, np.arange(nk)[None]
    m = np.ones((nq, nk), bool)
    if causal:
        m &= j <= p
    if window is not None:
        m &= np.abs(p - j) <= window // 2
    return m | (j < prefix)


def sdpa_packed(q, k, v, qoff, koff, scale, causal=False, window=None, prefix=None, cap=None, slopes=None):
    """(o, w, e): the outputs, sum_j p_j |v_j| and scale * max sum_c |q_c k_c|,
    which the tolerances scale with."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    T, H, D = q.shape
    G = H // k.shape[1]
    o, w, e = np.zeros(q.shape), np.zeros(q.shape), 0.0
    for b in range(len(qoff) - 1):
        nq, nk = qoff[b + 1] - qoff[b], koff[b + 1] - koff[b]
        if nq == 0 or nk == 0:
            continue
        m = visible(nq, nk, causal, window, 0 if prefix is None else int(np.clip(prefix[b], 0, nk)))
        far = np.abs(np.arange(nq)[:, None] + nk - nq - np.arange(nk)[None])
        for h in range(H):
            Q, K, V = q[qoff[b]:qoff[b + 1], h], k[koff[b]:koff[b + 1], h // G], v[koff[b]:koff[b + 1], h // G]
            with np.errstate(invalid="ignore"):
                x = scale * (Q @ K.T)
                if cap:
                    x = cap * np.tanh(x / cap)
                if slopes is not None:
                    x = x - float(slopes[h]) * far
                x = np.where(m, x, -np.inf)
            top = np.max(x, -1, keepdims=True)
            p = np.exp(x - np.where(np.isfinite(top), top, 0))
            p = np.where(m, p, 0)
            s = p.sum(-1, keepdims=True)
            p = p / np.where(s == 0, 1, s)
            # hidden values are not used, whatever they hold
            keep = np.where(np.isfinite(V), V, 0)
            o[qoff[b]:qoff[b + 1], h] = p @ keep
            w[qoff[b]:qoff[b + 1], h] = p @ np.abs(keep)
            with np.errstate(invalid="ignore"):
                e = max(e, float(np.nanmax(abs(scale) * (np.abs(Q) @ np.abs(np.where(np.isfinite(K), K, 0)).T))))
    return o, w, e


def lora_linear(x, w, bias, a, b, scales, index):
    """(y, mass): outputs and the sum of absolute products behind each."""
    x, w, a, b = (np.asarray(t, np.float64) for t in (x, w, a, b))
    y, mass = x @ w.T, np.abs(x) @ np.abs(w).T
    delta = np.zeros_like(y)
    if bias is not None:
        y, mass = y + bias, mass + np.abs(bias)
    for i in range(a.shape[0]):
        r = np.nonzero(index == i)[0]
        delta[r] = np.abs(scales[i]) * (np.abs(x[r]) @ np.abs(a[i]).T) @ np.abs(b[i]).T
        y[r] += scales[i] * (x[r] @ a[i].T) @ b[i].T
    return y, mass, delta
