"""float64 references of the 4-bit cache's operators, from their definitions (numpy)."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def bf16_bits(x):
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    nan = np.isnan(np.asarray(x, np.float32))
    return np.where(nan, 0x7FC0, (u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def val(bits):
    return (np.asarray(bits, np.uint16).astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def norm_rope(x, w, pos, rot, theta, eps):
    """x [rows][heads][d] float64, pos [rows] -> (result, |a| + |b| of each rotated pair, |y| elsewhere)."""
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1 + w)
    out, size, half = y.copy(), np.abs(y), rot // 2
    if rot:
        ang = pos[:, None, None] * theta ** (-2.0 * np.arange(half) / rot)
        c, s = np.cos(ang), np.sin(ang)
        a, b = y[..., :half], y[..., half:rot]
        out[..., :half], out[..., half:rot] = a * c - b * s, b * c + a * s
        size[..., :half] = size[..., half:rot] = np.abs(a) + np.abs(b)
    return out, size


def scale_byte(amax):
    """Smallest b with amax <= 6 * 2^(b - 127), within 8 .. 252; 255 for what is not finite."""
    m, e = np.frexp(np.where(np.isfinite(amax), amax, 0.0))       # amax = m 2^e, m in [0.5, 1)
    b = np.clip(np.where(m > 0.75, e - 2, e - 3) + 127, 8, 252)
    return np.where(np.isfinite(amax), np.where(amax > 0, b, 8), 255).astype(np.int64)


def values(codes, scales):
    """Codes [..][d / 2] and scale bytes [..][d / 32] as read back from a cache -> float64 [..][d]."""
    lut = np.concatenate([GRID, -GRID])
    x = np.stack([lut[codes & 15], lut[codes >> 4]], -1).reshape(*codes.shape[:-1], -1)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return x * np.repeat(s, 32, -1)


def nearest_ok(x, codes, scales, slack):
    """Whether every code is a nearest value to x / 2^e (e from its scale byte), ties to even, where
    x is known within slack * |x|; saturated beyond 6."""
    v = values(codes, scales)
    s = np.repeat(np.exp2(scales.astype(np.float64) - 127), 32, -1)
    m = np.abs(x) / s
    got = np.abs(v) / s
    i = np.searchsorted(GRID, got)
    up = np.where(i < 7, (GRID[np.minimum(i + 1, 7)] + got) / 2, np.inf)
    dn = np.where(i > 0, (GRID[np.maximum(i - 1, 0)] + got) / 2, -1.0)
    e = slack * m
    tie = (i % 2 == 0)
    ok_hi = np.where(tie, m - e <= up, m - e < up)
    ok_lo = np.where(tie, m + e >= dn, m + e > dn)
    return ok_hi & ok_lo & ((np.sign(v) == np.sign(x)) | (got == 0))


def attention(q, K, V, pos, window, sinks, scale):
    """q [T][hq][d], K, V [kv][slots][d], rows at pos .. -> (out, p . |V|, largest sum |q||k| scale)."""
    T, hq, d = q.shape
    kv = K.shape[0]
    out, pv, big = np.zeros(q.shape), np.zeros(q.shape), np.zeros((T, hq))
    for t in range(T):
        p = pos + t
        j = np.arange(p + 1)
        if window:
            j = j[(j > p - window) | (j < sinks)]
        for h in range(hq):
            k, v = K[h // (hq // kv)][j], V[h // (hq // kv)][j]
            with np.errstate(invalid="ignore", over="ignore"):
                s = k @ q[t, h] * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[t, h], pv[t, h] = w @ v, w @ np.abs(v)
                big[t, h] = (np.abs(k) @ np.abs(q[t, h])).max() * abs(scale)
    return out, pv, big


def attention_bound(out, pv, big, n, d, gate=None):
    """How far a result may be: weights rounded to bf16 (2^-8), scores off by (d + 4) 2^-24 of sum |q||k| (its
    float32 sum, scale and exponent) in the weight and in its normaliser, n + 64 float32 sums, the bf16
    result (2^-8); a sigmoid in float32."""
    e = (2.0 ** -8 + 4 * (d + 4) * 2.0 ** -24 * big[..., None] + (n + 64) * 2.0 ** -24) * pv
    if gate is not None:
        sg = 1 / (1 + np.exp(-gate))
        out, e = out * sg, e * sg + 2.0 ** -20 * np.abs(out)
    return out, e + 2.0 ** -8 * np.abs(out) + 1e-30


def probs(logits, temperature):
    x = logits / temperature
    e = np.exp(x - x.max())
    return e / e.sum()


def dist(row):
    return not np.isnan(row).any() and np.isfinite(row.max())


def verify(logits, drafts, u, temperature, dlogits=None):
    """One lane: (accepted, weights of the token or None or its argmax, border in [0, 1), nearness of the
    closest decision)."""
    k, near = len(drafts), np.inf
    for j in range(k + 1):
        t = drafts[j] if j < k else -1
        row = logits[j]
        if not dist(row):
            return j, None, 0.0, near
        if t < 0:
            break
        if temperature == 0:
            if t == row.argmax():
                continue
            break
        p = probs(row, temperature)
        pd = p[t] if t < len(row) else 0.0
        if dlogits is None:
            q, qd, good = None, 1.0, True
        else:
            good = dist(dlogits[j])
            q = probs(dlogits[j], temperature) if good else None
            qd = q[t] if good and t < len(row) else 0.0
        if pd > 0:                                 # (a p of 0 is one on both sides: nothing is below it)
            near = min(near, abs(u[j] * qd - pd) / pd)
        if good and u[j] * qd < pd:
            continue
        w = p.copy()
        if dlogits is None:
            if t < len(row):
                w[t] = 0.0
        elif good:
            w = np.maximum(p - q, 0)
        return j, (w if w.sum() > 0 else p), float(u[k]), near
    if temperature == 0:
        return j, int(row.argmax()), 0.0, near
    return j, probs(row, temperature), float(u[k]), near


def token_ok(tok, w, r):
    """Whether tok holds the border r of the weights w's running sum, up to float64 rounding."""
    if w is None:
        return tok == -1
    if isinstance(w, int):
        return tok == w
    c = np.cumsum(w)
    tol = 1e-12 * c[-1]
    before = c[tok - 1] if tok else 0.0
    return 0 <= tok < len(w) and w[tok] > 0 and before - tol <= r * c[-1] <= c[tok] + tol
