"""The 4-bit KV cache in numpy, in 64 bits, from its definition (include/tmg.h):
the tests' reference for tmg_kv4_*."""
import numpy as np

MAG = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def groups(hd):
    return max(1, hd // 32)


def quantize(x):
    """Codes [..., hd] (0..15) and scale bytes [..., groups] of f32 x [..., hd]."""
    x = np.asarray(x, np.float32)
    hd = x.shape[-1]
    g = x.astype(np.float64).reshape(x.shape[:-1] + (groups(hd), -1))
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    top = np.abs(g).max(-1)
    # the smallest e with top <= 7 * 2^e
    frac, e = np.frexp(top / 7.0)
    e = np.clip(np.where(top == 0, -100, np.where(frac == 0.5, e - 1, e)), -100, 125)
    a = np.abs(g) / np.exp2(e.astype(np.float64))[..., None]
    d = np.abs(a[..., None] - MAG)
    code = d.argmin(-1)  # the lower of two equally near
    tie = (code < 7) & (np.take_along_axis(d, np.minimum(code + 1, 7)[..., None], -1)[..., 0] == d.min(-1))
    code = np.where(tie & (code % 2 == 1), code + 1, code)
    code = np.where(np.signbit(g) & ~bad[..., None], code + 8, code)
    return code.reshape(x.shape), np.where(bad, 255, e + 127).astype(np.uint8)


def values(code, byte):
    """What codes [..., hd] and bytes [..., groups] stand for, f64."""
    v = MAG[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, np.exp2(byte.astype(np.float64) - 127))
    v = v.reshape(v.shape[:-1] + (byte.shape[-1], -1)) * s[..., None]
    return v.reshape(code.shape)


def stands_for(x):
    return values(*quantize(x))


def unpack(slab, cap, nkv, hd):
    """Keys and values [2][nkv][cap][hd] of one slab of bytes."""
    n, ng = nkv * cap * (hd // 2), groups(hd)
    out = []
    for i in range(2):
        c = slab[i * n:(i + 1) * n].reshape(nkv, cap, hd // 2)
        code = np.stack((c & 15, c >> 4), -1).reshape(nkv, cap, hd)
        b = slab[2 * n + i * nkv * cap * ng:][:nkv * cap * ng].reshape(nkv, cap, ng)
        out.append(values(code, b))
    return np.stack(out)


def attend(q, k, v, pos, scale=None):
    """Causal attention of rows q [rows][nq][hd] at pos .. over k, v
    [nkv][positions][hd], and the bound its f32 result keeps, [rows][nq][hd].

    The bound, in units u = 2^-24 (a rounding of f32): a score, in log2 units,
    is off by up to 3 u of its magnitude sum for the scaling of q, 2 u of the
    sum with each 32 dimensions' largest |q| for the parts left out, and about
    30 roundings of the partial sums; a weight by twice that times ln 2, and
    by 4 u for the exponential; the sums over n weights by (16 + n / 8) u, as
    no lane adds more than n / 16 of them in a row, twice (l and o)."""
    rows, nq, hd = q.shape
    nkv = k.shape[0]
    group = nq // nkv
    scale = 1 / np.sqrt(hd) if scale is None else scale
    q = np.asarray(q, np.float64)
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    u = 2.0 ** -24
    with np.errstate(all="ignore"):
        for t in range(rows):
            n = pos + t + 1
            for h in range(nq):
                kk, vv = k[h // group, :n], v[h // group, :n]
                s = kk @ q[t, h] * scale
                top = s.max() if not np.isnan(s).any() else np.nan
                w = np.zeros(n) if top == -np.inf else np.exp(s - top)
                total = w.sum()
                # a value of weight zero does not count, whatever it is: but
                # only masked positions have weight zero by definition
                out[t, h] = (w @ vv) / total if total != 0 else 0.0
                wide = np.abs(q[t, h]).reshape(groups(hd), -1).max(-1).repeat(hd // groups(hd))
                mag = np.nanmax(np.abs(kk) @ wide) * abs(scale) * 1.4426950408889634 if n else 0.0
                rel = 2 * 0.6931471805599453 * 35 * mag + 4 + 2 * (16 + n / 8)
                tol[t, h] = u * rel * ((w / total if total != 0 else w) @ np.abs(vv)) + 1e-37
    return out, tol
