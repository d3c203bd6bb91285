"""Plain 64-bit forms of the 8-bit operators (vosk.ops), on the CPU."""
import numpy as np

PAD = 64


def pad(k):
    return -(-k // PAD) * PAD


def codes_of(x):
    """codes [M, pad(K)] int8 and scales float32 [M] of float rows (any float type, exactly representable in 64 bits)."""
    x = np.asarray(x, np.float64)
    m, k = x.shape
    codes, scales = np.zeros((m, pad(k)), np.int8), np.zeros(m, np.float32)
    for i in range(m):
        if not np.isfinite(x[i]).all():
            scales[i] = np.nan
            continue
        s = np.float32(np.abs(x[i]).max() / 127)
        scales[i] = s
        if s > 0:
            codes[i, :k] = np.clip(np.rint(x[i] / np.float64(s)), -127, 127)
    return codes, scales


def frame_map(lengths, first, table, page, offsets, step, low, high, clamp, rows):
    """starts, and `rows` with the output rows filled in; frame after frame."""
    out = np.array(rows)
    ring = page * table.shape[1]
    starts, at = [0], 0
    for r, length in enumerate(int(v) for v in lengths):
        n = -(-max(length, 0) // step)
        newest = int(first[r]) + step * (n - 1) + max(offsets)
        if high is not None:
            newest = min(newest, int(high[r]))
        for i in range(n):
            if at < len(out):
                for j, off in enumerate(offsets):
                    t = int(first[r]) + step * i + off
                    if clamp:
                        t = max(t, int(low[r])) if low is not None else t
                        t = min(t, int(high[r])) if high is not None else t
                    ok = -2**31 <= t < 2**31 and t > newest - ring
                    ok = ok and (low is None or t >= int(low[r])) and (high is None or t <= int(high[r]))
                    p = int(table[r, (t % ring) // page]) if ok else -1
                    out[at, j] = p * page + t % page if p >= 0 else -1
            at += 1
        starts.append(at)
    return np.array(starts), out


def linear(codes, scales, rows, w, w_scales, taps, bias=None, relu=False, gain=None, shift=None, residual=None,
           residual_scale=1.0):
    """The product and its epilogue in 64 bits, unrounded, and the sum of the
    magnitudes that its roundings are relative to."""
    c64, s64 = np.asarray(codes, np.float64), np.asarray(scales, np.float64)
    w64 = np.asarray(w, np.float64).reshape(len(w), taps, -1)
    m = len(codes) if rows is None else len(rows)
    idx = np.arange(m)[:, None] if rows is None else np.asarray(rows)
    v, size = np.zeros((m, len(w))), np.zeros((m, len(w)))
    for j in range(taps):
        ok = (idx[:, j] >= 0) & (idx[:, j] < len(codes))
        at = np.where(ok, idx[:, j], 0)
        part = (c64[at] @ w64[:, j].T) * np.where(ok, s64[at], 0.0)[:, None]
        v, size = v + part, size + np.abs(part)
    ws = np.asarray(w_scales, np.float64)
    v, size = v * ws, size * np.abs(ws)
    if bias is not None:
        v, size = v + bias, size + np.abs(bias)
    if relu:
        v = np.where(v < 0, 0.0, v)
    if gain is not None:
        v, size = v * gain + shift, size * np.abs(gain) + np.abs(shift)
    if residual is not None:
        r = residual_scale * np.asarray(residual, np.float64)
        v, size = v + r, size + np.abs(r)
    return v, size
