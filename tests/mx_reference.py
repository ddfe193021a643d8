"""Plain numpy statements, in 64 bits, of the 4-bit format and of scored routing: what the
kernels' tests compare with.  Written from the definitions; no torch, no library code."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
VALUE = np.concatenate([E2M1, -E2M1])          # by 4-bit code


def scale_byte(block):
    """E8M0 byte of a block of float64 values: floor(log2(max)) - 2 + 127, at least 0; 255 if
    any value is no number."""
    if not np.isfinite(block).all():
        return 255
    m = np.abs(block).max()
    if m == 0:
        return 0
    return max(int(np.frexp(m)[1]) - 1 - 2 + 127, 0)


def quantize(x):
    """(codes [rows, K rounded up to 32], bytes [rows, blocks]) of float64 [rows, K]."""
    rows, k = x.shape
    blocks = -(-k // 32)
    pad = np.zeros((rows, blocks * 32))
    pad[:, :k] = x
    b = pad.reshape(rows, blocks, 32)
    finite = np.isfinite(b).all(-1)
    safe = np.where(finite[..., None], b, 0.0)
    m = np.abs(safe).max(-1)
    byte = np.where(m > 0, np.frexp(m)[1] - 3 + 127, 0)
    byte = np.where(finite, np.maximum(byte, 0), 255)
    q = np.abs(safe) / np.ldexp(1.0, np.where(finite, byte, 127)[..., None] - 127)
    # nearest of the eight magnitudes, halfway cases to the even code
    mid = (E2M1[:-1] + E2M1[1:]) / 2
    code = np.zeros(q.shape, dtype=np.int64)
    for c in range(7):
        code += (q > mid[c]) if c % 2 == 0 else (q >= mid[c])
    code += 8 * np.signbit(safe)
    return np.where(finite[..., None], code, 0).reshape(rows, -1), byte


def values(codes, byte, k):
    """float64 [rows, K] of codes [rows, K rounded up to 32] and bytes [rows, blocks]."""
    scale = np.ldexp(1.0, byte.astype(np.int64) - 127)
    scale = np.where(byte == 255, np.nan, scale)
    v = VALUE[codes].reshape(*byte.shape, 32) * scale[..., None]
    return v.reshape(codes.shape[0], -1)[:, :k]


def unpack(code_rows, scale_rows, k):
    """The kernels' rows (uint8) as (codes [rows, K rounded up to 32], bytes [rows, blocks])."""
    c = np.stack([code_rows & 15, code_rows >> 4], -1).reshape(code_rows.shape[0], -1)
    blocks = -(-k // 32)
    return c[:, :blocks * 32].astype(np.int64), scale_rows[:, :blocks].astype(np.int64)


def round_trip(x):
    codes, byte = quantize(x)
    return values(codes, byte, x.shape[1])


def boundary_distance(x):
    """|q - nearest rounding boundary| of every value of float64 [rows, K], q its quotient by
    its block's scale; -1 in blocks whose largest value is next to a power of two, where the
    scale itself is in doubt."""
    rows, k = x.shape
    codes, byte = quantize(x)
    pad = np.zeros_like(codes, dtype=np.float64)
    pad[:, :k] = x
    b = pad.reshape(rows, -1, 32)
    q = np.abs(b) / np.ldexp(1.0, byte[..., None] - 127)
    mid = (E2M1[:-1] + E2M1[1:]) / 2
    d = np.abs(q[..., None] - mid).min(-1)
    top = np.abs(b).max(-1)
    mant = np.frexp(top)[0]
    doubt = (np.abs(mant - 0.5) < 1e-4) | (np.abs(mant - 1.0) < 1e-4)
    d[doubt] = -1.0
    return d.reshape(rows, -1)[:, :k]


# ------------------------------------------------------------------ scored routing
def scores(logits, kind):
    if kind == "sigmoid":
        return 1 / (1 + np.exp(-logits))
    m = logits.max(-1, keepdims=True)
    e = np.exp(logits - np.where(np.isfinite(m), m, 0.0))
    total = e.sum(-1, keepdims=True)
    return e / np.where(total == 0, 1.0, total)


def score_topk(logits, bias, k, kind, n_group=1, top_group=1, group_best=2, renorm=True,
               scale=1.0):
    """(idx [T, k], weight [T, k], margin [T]): margin is the smallest difference on which a
    decision of the token rested."""
    t, e = logits.shape
    s = scores(logits, kind)
    v = s + (0 if bias is None else bias)
    v = np.where(np.isneginf(logits), -np.inf, v)
    idx = np.full((t, k), -1, dtype=np.int64)
    weight = np.zeros((t, k))
    margin = np.full(t, np.inf)
    size = e // n_group
    for r in range(t):
        row = v[r].copy()
        if n_group > 1 and top_group < n_group:
            value = []
            for g in range(n_group):
                part = np.sort(row[g * size:(g + 1) * size])[::-1][:group_best]
                part = part[np.isfinite(part)]
                value.append(part.sum() if len(part) else -np.inf)
            value = np.array(value)
            order = np.argsort(-value, kind="stable")
            if np.isfinite(value[order[top_group]]):
                margin[r] = min(margin[r], value[order[top_group - 1]] - value[order[top_group]])
            for g in order[top_group:]:
                row[g * size:(g + 1) * size] = -np.inf
        order = np.argsort(-row, kind="stable")
        live = [i for i in order if row[i] > -np.inf]
        for a, b in zip(live[:k], live[1:k + 1]):
            margin[r] = min(margin[r], row[a] - row[b])
        chosen = live[:k]
        idx[r, :len(chosen)] = chosen
        w = s[r, chosen]
        weight[r, :len(chosen)] = scale * (w / (w.sum() + 1e-20) if renorm else w)
    return idx, weight, margin


def score_topk_backward(dweight, logits, idx, kind, renorm=True, scale=1.0):
    s = scores(logits, kind)
    ds = np.zeros_like(s)
    for r in range(len(s)):
        live = idx[r] >= 0
        c, g = s[r, idx[r][live]], dweight[r][live]
        if renorm:
            total = c.sum() + 1e-20
            ds[r, idx[r][live]] = scale / total * (g - (g * c).sum() / total)
        else:
            ds[r, idx[r][live]] = scale * g
    if kind == "sigmoid":
        return ds * s * (1 - s)
    return s * (ds - (ds * s).sum(-1, keepdims=True))
