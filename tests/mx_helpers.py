"""Microscaled 4-bit floating point in 64 bits with numpy, from the definition in include/cugl.h."""
import numpy as np

MXFP4, NVFP4 = 0, 1
GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6.0])
MIDPOINTS = (GRID[1:] + GRID[:-1]) / 2


def block_of(fmt):
    return 16 if fmt == NVFP4 else 32


def blocks_of(cols, fmt):
    return -(-cols // block_of(fmt))


def _round_even(v):
    return np.round(v)  # ties to even


def scale_of(amax, fmt):
    """(scale bytes, scale values) of block maxima, float64."""
    amax = np.asarray(amax, np.float64)
    fine = np.isfinite(amax) & (amax > 0)
    a = np.where(fine, amax, 1.0)
    if fmt == MXFP4:
        e = np.maximum(np.frexp(a)[1] - 1 - 2, -127)
        byte, value = e + 127, np.ldexp(1.0, e)
        nan = 255
    else:
        v = np.clip(a / 6, 2.0 ** -9, 448.0)
        e = np.maximum(np.frexp(v)[1] - 1, -6)
        value = _round_even(np.ldexp(v, 3 - e)) * np.ldexp(1.0, e - 3)
        e = np.frexp(value)[1] - 1
        byte = np.where(e < -6, np.ldexp(value, 9), (e + 7) * 8 + (np.ldexp(value, 3 - e) - 8)).astype(np.int64)
        nan = 127
    byte = np.where(fine, byte, np.where(amax == 0, 0, nan)).astype(np.uint8)
    return byte, np.where(fine, value, np.where(amax == 0, 0.0, np.nan))


def quantize(x, fmt, exponent=0):
    """Codes [rows, cols] and scale bytes [rows, blocks] of a float64 matrix."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    nb, block = blocks_of(cols, fmt), block_of(fmt)
    t = np.zeros((rows, nb * block))
    t[:, :cols] = x * 2.0 ** -exponent
    t = t.reshape(rows, nb, block)
    with np.errstate(invalid="ignore"):
        amax = np.abs(t).max(axis=2) if cols else np.zeros((rows, 0))
    amax = np.where(np.isnan(t).any(axis=2), np.nan, amax)
    byte, scale = scale_of(amax, fmt)
    q = np.abs(t) / np.where(np.isfinite(scale) & (scale > 0), scale, 1.0)[:, :, None]
    lo, hi = np.searchsorted(MIDPOINTS, q, side="left"), np.searchsorted(MIDPOINTS, q, side="right")
    code = np.where(lo % 2 == 0, lo, hi) | (np.signbit(t) << 3)
    return code.reshape(rows, -1)[:, :cols].astype(np.uint8), byte


def values(code, byte, fmt, exponent=0):
    """What codes [rows, cols] with scale bytes [rows, blocks] stand for, float64."""
    byte = byte.astype(np.int64)
    if fmt == MXFP4:
        scale = np.where(byte == 255, np.nan, np.ldexp(1.0, byte - 127))
    else:
        e, m = byte >> 3, byte & 7
        scale = np.where(byte == 127, np.nan, np.where(e == 0, m * 2.0 ** -9, np.ldexp(1 + m / 8, e - 7)))
    v = GRID[code & 7] * np.where(code & 8, -1.0, 1.0)
    return v * np.repeat(scale, block_of(fmt), axis=1)[:, :code.shape[1]] * 2.0 ** exponent


def pack(code, pitch):
    rows, cols = code.shape
    full = np.zeros((rows, 2 * pitch), np.uint8)
    full[:, :cols] = code
    return full[:, 0::2] | (full[:, 1::2] << 4)


def unpack(packed, cols):
    return np.stack([packed & 15, packed >> 4], axis=-1).reshape(packed.shape[0], -1)[:, :cols]


def _tile_index(rows, nb):
    r, b = np.arange(rows)[:, None], np.arange(nb)[None, :]
    across = -(-nb // 4)
    return ((r // 128) * across + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4


def tile(byte, fill=0):
    """Scale bytes [rows, blocks] as tiles (flat); blocks behind a row are 0, rows behind the last are `fill`."""
    rows, nb = byte.shape
    out = np.full((-(-rows // 128)) * (-(-nb // 4)) * 512, fill, np.uint8)
    padded = np.zeros((rows, -(-nb // 4) * 4), np.uint8)
    padded[:, :nb] = byte
    out[_tile_index(rows, padded.shape[1])] = padded
    return out


def untile(flat, rows, nb):
    return flat[_tile_index(rows, nb)]


def matrix(rng, rows, cols, fmt, std=1.0):
    """A random quantised matrix: (codes, scale bytes, values)."""
    code, byte = quantize(rng.standard_normal((rows, cols)) * std, fmt)
    return code, byte, values(code, byte, fmt)


# ---- expert layer -----------------------------------------------------------------------------------------
def choose(logits, top_k, renormalize):
    """Chosen experts and their weights per token: lists of (expert, weight)."""
    out = []
    for row in np.asarray(logits, np.float64):
        order = [e for e in np.lexsort((np.arange(row.size), -np.where(np.isnan(row), -np.inf, row)))
                 if not np.isnan(row[e]) and row[e] > -np.inf]
        chosen = order[:top_k]
        among = row[chosen] if renormalize else row[order]
        top = row[order[0]] if order else 0.0
        total = np.exp(among - top).sum()
        out.append([(int(e), np.exp(row[e] - top) / total) for e in chosen])
    return out


def requantized(h, err, fmt, exponent=0):
    """(values h is stored as, how far a value may be from that where h is only known within err).  A code may fall the other way
    where its midpoint lies within err; a block whose scale may change is off by at most a step of either scale."""
    rows, cols = h.shape
    code, byte = quantize(h, fmt, exponent)
    v = values(code, byte, fmt, exponent)
    block, nb = block_of(fmt), blocks_of(cols, fmt)
    pad = ((0, 0), (0, nb * block - cols))
    hb, eb = np.pad(np.abs(h), pad).reshape(rows, nb, block), np.pad(err, pad).reshape(rows, nb, block)
    low = quantize(np.maximum(hb - eb, 0).max(axis=2, keepdims=True).reshape(-1, 1), fmt, exponent)[1].reshape(rows, nb)
    high = quantize((hb + eb).max(axis=2, keepdims=True).reshape(-1, 1), fmt, exponent)[1].reshape(rows, nb)
    one = np.full((rows * nb, 1), 2, np.uint8)  # the code of 1
    s_high = values(one, high.reshape(-1, 1), fmt, exponent).reshape(rows, nb, 1)
    s = values(one, byte.reshape(-1, 1), fmt, exponent).reshape(rows, nb, 1)
    q, qe = hb / np.where(s > 0, s, 1), eb / np.where(s > 0, s, 1)
    near = (np.abs(q[..., None] - MIDPOINTS) <= qe[..., None] * (1 + 1e-9)).any(axis=3) & (s > 0)
    off = np.where(near, 2 * s, 0)          # the widest step of E2M1 is 2
    off = np.where((low != high)[:, :, None], 4 * s_high, off)
    return v, off.reshape(rows, -1)[:, :cols]


def moe(vx, logits, gate, up, down, top_k, renormalize, fmt, h_exponent=0, alphas=(1, 1, 1)):
    """(y, bound of what float sums may change): values of x and of the experts' matrices [E, rows, cols] in float64.  A product
    of K elements is off by (K / 64 + 18) steps of 2^-23 of its magnitudes (its MMAs, the parts of a split K, the factor), the
    gate's weight by 2^-20 (expf, division), silu by 2^-20 and by what its argument is off (its slope is below 1.1)."""
    T, H = vx.shape
    F = gate.shape[1]
    y, tol, size = np.zeros((T, H)), np.zeros((T, H)), np.zeros((T, H))
    steps = 2.0 ** -23 * (-(-H // 64) + 18)
    picks = choose(logits, top_k, renormalize)
    for e in range(gate.shape[0]):
        tokens = [t for t in range(T) if any(i == e for i, _ in picks[t])]
        if not tokens:
            continue
        p = np.array([[w for i, w in picks[t] if i == e] for t in tokens])
        x = vx[tokens]
        g, u = alphas[0] * (x @ gate[e].T), alphas[1] * (x @ up[e].T)
        eg, eu = steps * abs(alphas[0]) * (np.abs(x) @ np.abs(gate[e]).T), steps * abs(alphas[1]) * (np.abs(x) @ np.abs(up[e]).T)
        with np.errstate(over="ignore"):
            silu = g / (1 + np.exp(-g))
        h = p * silu * u
        err = p * ((1.1 * eg + 2.0 ** -20 * np.abs(silu)) * (np.abs(u) + eu) + np.abs(silu) * eu) + 2.0 ** -19 * np.abs(h)
        v, off = requantized(h, err, fmt, h_exponent)
        y[tokens] += alphas[2] * (v @ down[e].T)
        tol[tokens] += abs(alphas[2]) * (off @ np.abs(down[e]).T)
        size[tokens] += abs(alphas[2]) * ((np.abs(v) + off) @ np.abs(down[e]).T)
    active = len({e for pick in picks for e, _ in pick})
    return y, tol + 2.0 ** -23 * (active * -(-F // 64) + 18) * size
