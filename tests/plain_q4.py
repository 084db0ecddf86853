"""Plain statements, in 64 bits, of the 4- and 8-bit formats and of the verification of drafted tokens."""
import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def padded(k):
    return -(-k // 128) * 128


def scale_bytes(scales, rows):
    """The laid-out exponent bytes (uint8 [tiles, kb, 32, 4, 4]) as [rows, groups]."""
    t, kb = scales.shape[:2]
    return scales.transpose(0, 3, 2, 1, 4).reshape(t * 128, kb * 4)[:rows]


def q4_values(codes, scales):
    """uint8 codes [n, kp / 2] and bytes -> float64 [n, kp]."""
    n, half = codes.shape
    c = np.stack([codes & 15, codes >> 4], axis=2).reshape(n, 2 * half).astype(int)
    v = np.where(c >= 8, -1.0, 1.0) * MAGNITUDES[c % 8]
    return v * np.repeat(2.0 ** (scale_bytes(scales, n).astype(float) - 127), 32, axis=1)


def e4m3(byte):
    """The value of e4m3 bytes."""
    b = byte.astype(int)
    e, f = (b >> 3) & 15, b & 7
    v = np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))
    v = np.where((b & 127) == 127, np.nan, v)
    return np.where(b >= 128, -v, v)


def q8_values(codes, scales):
    return e4m3(codes) * np.repeat(2.0 ** (scale_bytes(scales, codes.shape[0]).astype(float) - 127), 32, axis=1)


def groups_of(x):
    m, k = x.shape
    wide = np.zeros((m, padded(k)))
    wide[:, :k] = x
    return wide.reshape(m, -1, 32)


def smallest_exponent(top, most):
    """The smallest e with top <= most 2^e, by trying: -127 for zeros, and never below it."""
    e = np.full(top.shape, -127.0)
    for t in range(-126, 128):
        e = np.where(top > most * 2.0 ** (t - 1), float(t), e)
    return e


def round_e4m3(v):
    step = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -20))), -6.0) - 3.0)
    return np.round(v / step) * step                      # (numpy rounds halves to even)


def q8_of(x):
    """Rows in 64 bits -> (values of the codes [m, kp], exponents [m, groups])."""
    g = groups_of(x)
    e = smallest_exponent(np.abs(g).max(axis=2), 448.0)
    return round_e4m3(g / 2.0 ** e[..., None]).reshape(x.shape[0], -1), e


def round_e2m1(v):
    """To the nearest code, halves to the even one, cut off at 6; the values."""
    edges = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    a = np.abs(v)
    code = np.searchsorted(edges, a, side="left")         # at an edge: the lower code ...
    at_edge = np.isin(a, edges)
    code = np.where(at_edge & (code % 2 == 1), code + 1, code)        # ... or the upper one where that is even
    return np.sign(v) * MAGNITUDES[code]


def softmax_kept(logits, temperature, top_k):
    """Softmax at the temperature over the top_k largest (ties: the lowest index first); NaN-free rows."""
    z = np.asarray(logits, dtype=np.float64)
    kept = np.ones(z.shape, dtype=bool)
    if 0 < top_k < z.shape[0]:
        order = np.argsort(-z, kind="stable")
        kept[order[top_k:]] = False
    top = z.max()
    if not np.isfinite(top):
        return np.full(z.shape, np.nan)
    p = np.where(kept, np.exp((z - top) / temperature), 0.0)
    return p / p.sum()


def walk(mass, draw):
    target, run = draw * mass.sum(), 0.0
    found = -1
    for i, m in enumerate(mass):
        if m > 0:
            found = i
            run += m
            if run > target:
                return i
    return found


def verify(logits, draft_logits, drafts, draws, temperature, top_k):
    """One sequence: (tokens, kept, margin).  ``margin``: how far the closest decision was from going the other way."""
    g = len(drafts)
    greedy = temperature <= 0 or top_k == 1
    top_k = max(top_k, 0)
    kept, margin = 0, 1.0
    ended = True
    for i, x in enumerate(drafts):
        if not 0 <= x < len(logits[i]):
            break
        if greedy:
            taken = int(np.argmax(logits[i])) == x
        else:
            p, q = softmax_kept(logits[i], temperature, top_k), softmax_kept(draft_logits[i], temperature, top_k)
            taken = draws[i] * q[x] < p[x]
            if p[x] > 0 or q[x] > 0:
                margin = min(margin, abs(draws[i] * q[x] - p[x]) / max(p[x], q[x]))
        if not taken:
            ended = False
            break
        kept += 1
    if greedy:
        then = int(np.argmax(logits[kept]))
    else:
        p = softmax_kept(logits[kept], temperature, top_k)
        if np.isnan(p).any():
            then = int(np.argmax(logits[kept]))
        else:
            mass = p
            if not ended:
                rest = np.maximum(p - softmax_kept(draft_logits[kept], temperature, top_k), 0.0)
                mass = rest if rest.sum() > 0 else p
            then = walk(mass, draws[g])
            run = np.cumsum(mass[mass > 0])
            margin = min(margin, float(np.abs(run / run[-1] - draws[g])[:-1].min())) if len(run) > 1 else margin
    return list(drafts[:kept]) + [then] + [-1] * (g - kept), kept, margin
