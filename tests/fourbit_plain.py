"""The four-bit format and operators in plain numpy, for the tests: the quantiser in the 32-bit steps that the header
describes (its codes are compared bit for bit), everything else in 64 bits."""
import numpy as np


def quantise(x, group):
    """x [..., width] (any float type) -> codes [..., width] uint8, step and low [..., width / group] f16."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, group)
    bad = ~np.isfinite(g).all(-1)
    with np.errstate(all="ignore"):
        mn, mx = np.where(bad, 0, g.min(-1)), np.where(bad, 0, g.max(-1))
        low = np.clip(mn, np.float32(-65504), np.float32(65504)).astype(np.float16)
        span = np.maximum(np.minimum(mx, np.float32(65504)) - low.astype(np.float32), np.float32(0)).astype(np.float32)
        step = (span / np.float32(15)).astype(np.float16)
        s = step.astype(np.float32)[..., None]
        code = np.rint((g - low.astype(np.float32)[..., None]) / np.where(s > 0, s, 1).astype(np.float32))
        code = np.where(s > 0, np.clip(np.where(bad[..., None], 0, code), 0, 15), 0).astype(np.uint8)
    step = np.where(bad, np.float16(0), step)
    low = np.where(bad, np.uint16(0x7E00).view(np.float16), low)
    return code.reshape(x.shape), step, low


def places(width, values):
    """For every coordinate, its nibble's place among a token's width nibbles."""
    i, units = np.arange(width), width // 32
    u, r = i // 32, i % 32
    return ((r // 4) * units + u) * 4 + r % 4 if values else ((r // 8) * units + u) * 8 + r % 8


def pack(code, values):
    width = code.shape[-1]
    nib = np.zeros_like(code)
    nib[..., places(width, values)] = code
    return nib[..., 0::2] | (nib[..., 1::2] << 4)


def unpack(raw, values):
    nib = np.stack([raw & 15, raw >> 4], -1).reshape(*raw.shape[:-1], -1)
    return nib[..., places(nib.shape[-1], values)]


def scales(step, low):
    return np.stack([step, low], -1)


def value(code, step, low, group):
    """What codes stand for, in 64 bits."""
    rep = lambda a: np.repeat(a.astype(np.float64), group, -1)  # noqa: E731
    return rep(low) + rep(step) * code


def pool_of(k, v, slots, pages, page, group, fill):
    """A pool [pages][page bytes] with rows k, v [tokens][heads][width] in their slots, `fill` bytes elsewhere, and the
    values they stand for."""
    tokens, heads, w = k.shape
    ng = w // group
    size = page * (w + 8 * ng)
    pool = np.full((pages, heads, size), fill, np.uint8)
    found = []
    for x, at, values in ((k, 0, False), (v, page * (w // 2 + 4 * ng), True)):
        code, step, low = quantise(x, group)
        found.append(value(code, step, low, group))
        raw = pack(code, values)
        sc = np.ascontiguousarray(scales(step, low)).view(np.uint8).reshape(tokens, heads, 4 * ng)
        for t, slot in enumerate(slots):
            if slot < 0:
                continue
            p, o = slot // page, slot % page
            pool[p, :, at + o * (w // 2): at + (o + 1) * (w // 2)] = raw[t]
            s = at + page * (w // 2)
            pool[p, :, s + o * 4 * ng: s + (o + 1) * 4 * ng] = sc[t]
    return pool.reshape(pages, -1), found[0], found[1]


def attend(q, k, v, n, length, scale, causal, window):
    """One sequence: q [n][q_heads][width], k, v [length][heads][width] in 64 bits -> out, lse, and for each output how
    far a relative error of 1 in every product q_c k_c could move a score (the largest over its keys)."""
    hq, h = q.shape[1], k.shape[1]
    out, lse = np.zeros(q.shape), np.full(q.shape[:2], -np.inf)
    reach = np.zeros(q.shape[:2])
    q = q.astype(np.float64)
    for i in range(n):
        end = min(length, length - n + i + 1) if causal else length
        begin = max(0, length - n + i - window + 1) if window else 0
        if end <= begin:
            continue
        for j in range(hq):
            ks, vs = k[begin:end, j // (hq // h)], v[begin:end, j // (hq // h)]
            s = ks @ q[i, j] * scale
            reach[i, j] = (np.abs(ks) @ np.abs(q[i, j])).max() * abs(scale)
            m = s.max()
            p = np.exp(s - m)
            lse[i, j] = m + np.log(p.sum())
            out[i, j] = p @ vs / p.sum()
    return out, lse, reach


def logprobs(x, labels, top, temperature):
    """One row of scores in 64 bits (NaN and +infinity not among them)."""
    x = x.astype(np.float64)
    m = x.max()
    if m == -np.inf:
        return np.where(labels < 0, 0.0, -np.inf), 0.0, np.full(top, -np.inf), np.full(top, -1)
    d = (x - m) / temperature
    e = np.exp(d)
    ls = np.log(e.sum())
    ent = ls - (e[e > 0] * d[e > 0]).sum() / e.sum()
    order = np.lexsort((np.arange(x.size), -x))[:top]
    order = order[x[order] > -np.inf]
    ids, vals = np.full(top, -1), np.full(top, -np.inf)
    ids[: order.size], vals[: order.size] = order, d[order] - ls
    return np.where(labels < 0, 0.0, d[np.maximum(labels, 0)] - ls), ent, vals, ids
