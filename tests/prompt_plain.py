"""A prompt's operators in plain numpy and 64 bits: the four-bit floating-point format, and attention of packed rows."""
import numpy as np

MX, NV = 0, 1
BLOCK = {MX: 32, NV: 16}
NUMBERS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)
MIDDLES = (NUMBERS[1:] + NUMBERS[:-1]) / 2
# the finite e4m3 floats that are not negative, by their code: 0..126
E4M3 = np.array([(c & 7) * 2.0**-9 if c < 8 else 2.0 ** ((c >> 3) - 7) * (1 + (c & 7) / 8) for c in range(127)])


def nearest(x, middles):
    """How many middles lie below each x; of one on a middle the neighbour of even number."""
    low = np.searchsorted(middles, x, side="left")  # middles below x
    on = np.isin(x, middles)
    return low + (on & (low % 2 == 1))


def padded(k):
    return -(-k // 128) * 128


def quantise(x, fmt, unit=1.0):
    """x [rows, k]: codes (0..15) [rows, padded k] and scale bytes [rows, padded k / block]."""
    rows, k = x.shape
    g = np.zeros((rows, padded(k)))
    g[:, :k] = x
    g = g.reshape(rows, -1, BLOCK[fmt])
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0, g)
    top = np.abs(g).max(-1)
    unit = float(np.float32(unit))
    if fmt == MX:
        byte = np.clip(np.frexp(top)[1] - 3, -127, 127) + 127
        byte = np.where(top > 0, byte, 0)
        by = 2.0 ** (byte - 127.0)
    else:
        byte = nearest(top / (6 * unit), (E4M3[1:] + E4M3[:-1]) / 2)
        by = E4M3[byte] * unit
    a = np.where(by[..., None] > 0, np.abs(g) / np.where(by > 0, by, 1)[..., None], 0)
    code = nearest(a, MIDDLES)
    code = code + np.where(np.signbit(g), 8, 0)
    code = np.where((by > 0)[..., None], code, 0)
    byte = np.where(bad, 255 if fmt == MX else 127, byte)
    return np.where(bad[..., None], 0, code).reshape(rows, -1).astype(np.uint8), byte.astype(np.uint8)


def scales(byte, fmt):
    if fmt == MX:
        return np.where(byte == 255, np.nan, 2.0 ** (np.minimum(byte, 254).astype(np.float64) - 127))
    return np.where(byte == 127, np.nan, E4M3[np.minimum(byte, 126)])


def values(code, byte, fmt, unit, k):
    """What they stand for [rows, k], in 64 bits."""
    n = NUMBERS[code & 7] * np.where(code & 8, -1, 1)
    s = scales(byte, fmt) * float(np.float32(unit))
    return (n.reshape(n.shape[0], -1, BLOCK[fmt]) * s[..., None]).reshape(n.shape)[:, :k]


def stored(code, byte):
    """As they lie in memory: codes [rows, padded / 2], and every scale's place [rows, count] in the scales' bytes."""
    rows, count = byte.shape
    r, s = np.arange(rows)[:, None], np.arange(count)[None]
    place = (r // 128 * (count // 4) + s // 4) * 512 + r % 32 * 16 + r % 128 // 32 * 4 + s % 4
    return code[:, 0::2] | (code[:, 1::2] << 4), place


def attend(q, k, v, q_lens, k_lens, heads, scale, causal, window):
    """q [rows, q_heads, width], k and v [keys, heads, width] in 64 bits, sequences one behind the other: outputs and log-sum-exp.
    A key that a row does not see has no part in it, whatever it holds."""
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    each, q0, k0 = q.shape[1] // heads, 0, 0
    for n, length in zip(q_lens, k_lens):
        for i in range(n):
            hi = max(0, min(length, length - n + i + 1)) if causal else length
            lo = max(0, length - n + i + 1 - window) if window else 0
            if hi <= lo:
                continue
            qi, ks, vs = q[q0 + i].reshape(heads, each, -1), k[k0 + lo:k0 + hi], v[k0 + lo:k0 + hi]
            s = scale * np.einsum("nhw,hew->hen", ks, qi)
            top = s.max(-1, keepdims=True)
            p = np.exp(s - top)
            total = p.sum(-1, keepdims=True)
            lse[q0 + i] = (top + np.log(total)).reshape(-1)
            out[q0 + i] = (np.einsum("hen,nhw->hew", p, vs) / total).reshape(q.shape[1:])
        q0, k0 = q0 + n, k0 + length
    return out, lse
