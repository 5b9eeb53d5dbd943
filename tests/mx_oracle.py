"""MXFP4, routing and the experts' feed-forward from their definitions, in 64 bits on the host."""
import numpy as np

ELEMENTS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """x [.., K] float64 -> codes uint8 [.., K / 2], scales uint8 [.., K / 32] (finite x)"""
    v = x.reshape(*x.shape[:-1], -1, 32)
    top = np.abs(v).max(axis=-1)
    with np.errstate(divide="ignore"):
        power = np.where(top > 0, np.frexp(top)[1] - 1, -10000)   # floor(log2)
    scales = np.maximum(power - 2 + 127, 0).astype(np.uint8)
    a = np.abs(v) / np.exp2(scales.astype(np.float64) - 127)[..., None]
    # the nearest element; of two as near ones that with the even code
    away = np.abs(a[..., None] - ELEMENTS)
    near = away.min(axis=-1, keepdims=True) == away
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(axis=-1), even.argmax(axis=-1), near.argmax(axis=-1)).astype(np.uint8)
    code |= ((v < 0) * 8).astype(np.uint8)
    code = code.reshape(x.shape)
    return code[..., 0::2] | code[..., 1::2] << 4, scales


def values(codes, scales):
    pair = np.stack([codes & 15, codes >> 4], axis=-1).reshape(*codes.shape[:-1], -1)
    v = np.where(pair >= 8, -1.0, 1.0) * ELEMENTS[pair & 7]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * s.repeat(32, axis=-1)


def _best(c, top):
    """indices of the `top` largest per row, in falling order, ties to the lowest"""
    return np.argsort(-c, axis=1, kind="stable")[:, :top]


def route(logits, top, scoring, bias, groups, top_groups, renormalize, scale):
    """ids, weights, and per token the smallest difference that its choice hangs on and the largest number that it compares"""
    M, E = logits.shape
    if scoring == "softmax":
        e = np.exp(logits - logits.max(axis=1, keepdims=True))
        s = e / e.sum(axis=1, keepdims=True)
    else:
        s = 1 / (1 + np.exp(-logits))
    c = s + (0 if bias is None else bias.astype(np.float64))
    gap, size = np.full(M, np.inf), np.abs(c).max(axis=1)

    def least(v, n):   # of the first n places among all
        d = -np.diff(-np.sort(-v, axis=1), axis=1)[:, :n]
        return d.min(axis=1) if d.shape[1] else np.full(M, np.inf)

    if groups > 1:
        by = c.reshape(M, groups, -1)
        worth = np.sort(by, axis=2)[:, :, -2:].sum(axis=2)
        size = np.maximum(size, np.abs(worth).max(axis=1))
        kept = np.zeros((M, groups), dtype=bool)
        np.put_along_axis(kept, _best(worth, top_groups), True, axis=1)
        if top_groups < groups:
            in_out = -np.sort(-worth, axis=1)
            gap = np.minimum(gap, in_out[:, top_groups - 1] - in_out[:, top_groups])
        c = np.where(kept[:, :, None], by, -1e9).reshape(M, E)
    gap = np.minimum(gap, least(c, top))
    ids = _best(c, top)
    w = np.take_along_axis(s, ids, axis=1)
    if renormalize:
        w = w / w.sum(axis=1, keepdims=True)
    return ids.astype(np.int32), w * scale, gap, size


def experts(x, mats, ids, w, rows16):
    """(y, bound): the feed-forward in 64 bits, and how far a computation with fp32 sums may be off before its last rounding.

    Its h differs from that in 64 bits by what fp32 sums allow, d; a block's scale and elements are those of numbers up to d away,
    so its rounding may fall on a neighbouring code. The bound follows every element: |h^ - h^'| is at most the distance between
    the roundings of h - d and h + d under the scales that a block of such numbers can have. rows16: an expert's outputs may be held
    as fp16 numbers of a unit that 32 of them share, the largest from 2^14 units up: off by at most 2^-11 of themselves, or by 2^-25
    units, which is under 2^-39 of the largest."""
    (gc, gs), (uc, us), (dc, ds) = mats
    E = gc.shape[0]
    xq = values(*quantize(x))
    y = np.zeros((x.shape[0], dc.shape[1]))
    bound = np.zeros_like(y)
    eps = 2.0 ** -24
    for e in range(E):
        t, j = np.nonzero(ids == e)
        if not len(t):
            continue
        gate, up, down = values(gc[e], gs[e]), values(uc[e], us[e]), values(dc[e], ds[e])
        a = xq[t]
        g, u = a @ gate.T, a @ up.T
        grow = 2 * (a.shape[1] / 32 + 16) * eps
        dg, du = grow * (np.abs(a) @ np.abs(gate).T), grow * (np.abs(a) @ np.abs(up).T)
        sig = 1 / (1 + np.exp(-g))
        h = g * sig * u
        # silu's slope is under 1.1; its own exp, sum, division and products: 8 roundings and exp's argument
        d = 1.1 * dg * (np.abs(u) + du) + np.abs(g * sig) * du + (8 + np.abs(g)) * eps * np.abs(h)
        hq = values(*quantize(h))
        low, high = (np.abs(h) - d).clip(0), np.abs(h) + d
        near = np.zeros_like(h)
        for top in (low, high):
            blocks = top.reshape(*top.shape[:-1], -1, 32).max(axis=-1)
            power = np.where(blocks > 0, np.frexp(np.where(blocks > 0, blocks, 1))[1] - 3, -127).clip(-127)
            unit = np.exp2(power.astype(np.float64)).repeat(32, axis=-1)
            for v in (h - d, h + d):
                r = np.abs(v) / unit
                step = np.where(r < 2, 0.5, np.where(r < 4, 1.0, 2.0))
                q = np.sign(v) * np.minimum(np.round(r / step) * step, 6) * unit
                near = np.maximum(near, np.abs(q - hq))
        o = hq @ down.T
        wj = w[t, j].astype(np.float64)[:, None]
        off = near @ np.abs(down).T + 2 * (h.shape[1] / 32 + 16) * eps * (np.abs(hq) @ np.abs(down).T)
        if rows16:
            size = np.abs(o) + off
            pad = np.pad(size, ((0, 0), (0, -o.shape[1] % 32)))
            largest = pad.reshape(len(t), -1, 32).max(axis=2).repeat(32, axis=1)[:, :o.shape[1]]
            off = off + np.maximum(2.0 ** -11 * size, 2.0 ** -39 * largest)
        np.add.at(y, t, wj * o)
        # (and the weighted sum over the token's experts, every term rounded twice per addition)
        np.add.at(bound, t, np.abs(wj) * (off + 2 * (ids.shape[1] + 1) * eps * np.abs(o)))
    return y, bound
