"""The operators on 8-bit rows from their definitions, in 64 bits on the CPU (numpy)."""
import numpy as np

BLOCK, LOW, BIAS = 128, -117, 127


def code_values():
    """The number each e4m3 byte stands for: sign, 4 bits of exponent (bias 7), 3 of fraction; 127 and 255 are NaN."""
    c = np.arange(256)
    power, part = c >> 3 & 15, c & 7
    v = np.where(power == 0, part / 512.0, (1 + part / 8.0) * np.exp2(power - 7.0))
    v[(c & 127) == 127] = np.nan
    return np.where(c >> 7 == 1, -v, v)


def quantise(x):
    """(code values [n, dim], exponent bytes [n, blocks], rows as stored, squared norms) of a float64 matrix."""
    n, dim = x.shape
    blocks = -(-dim // BLOCK)
    mags = code_values()[:127]
    codes, exps = np.zeros((n, dim)), np.zeros((n, blocks), dtype=np.int64)
    for b in range(blocks):
        part = x[:, b * BLOCK : (b + 1) * BLOCK]
        fine = np.isfinite(part)
        top = np.where(fine, np.abs(part), 0.0).max(1)
        e = np.full(n, LOW, dtype=np.int64)
        for i in range(n):
            while top[i] > 448.0 * 2.0 ** int(e[i]):
                e[i] += 1
        scaled = np.abs(np.where(fine, part, 0.0)) / np.exp2(e.astype(np.float64))[:, None]
        up = np.clip(np.searchsorted(mags, scaled), 1, 126)
        low, high = scaled - mags[up - 1], mags[up] - scaled
        near = np.where((high < low) | ((high == low) & (up % 2 == 0)), up, up - 1)
        codes[:, b * BLOCK : (b + 1) * BLOCK] = np.where(fine, np.copysign(mags[near], part), np.nan)
        exps[:, b] = e
    rows = codes * np.exp2(np.repeat(exps, BLOCK, axis=1)[:, :dim].astype(np.float64))
    return codes, exps + BIAS, rows, (rows * rows).sum(1)


def products(a, b):
    """(a @ b.T, the sum of the magnitudes of each element's terms)."""
    return a @ b.T, np.abs(a) @ np.abs(b).T


def coverage(a, c, prior=None):
    d = np.full(a.shape[0], np.inf)
    for j in range(c.shape[0]):
        diff = ((a - c[j]) ** 2).sum(1)
        d = np.fmin(d, diff)
    return d if prior is None else np.fmin(prior, d)
