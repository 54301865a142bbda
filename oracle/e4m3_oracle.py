"""The 8-bit dense layer and the embedding rows in 64 bits, from their definitions, on the CPU (test infrastructure; nothing of the
package is used).  An e4m3 image holds, per row and block of 128 columns, the smallest power of two 2^e >= 2^-126 with
max |x| <= 448 * 2^e, and the codes of x * 2^-e."""
import numpy as np

MANTISSA_BITS, MIN_EXPONENT, MOST = 3, -6, 448.0


def code_values():
    """The 256 values of OCP e4m3, by code: sign, four exponent bits (bias 7), three mantissa bits; 0x7f and 0xff are NaN."""
    v = np.empty(256)
    for c in range(256):
        s, e, m = -1.0 if c & 128 else 1.0, (c >> 3) & 15, c & 7
        v[c] = s * (m / 8.0 * 2.0 ** -6 if e == 0 else (1.0 + m / 8.0) * 2.0 ** (e - 7))
    v[0x7F] = v[0xFF] = np.nan
    return v


def image(x):
    """x [rows, K] -> (codes uint8 [rows, Kp], exponents uint8 [rows, KB4])."""
    x = np.asarray(x, dtype=np.float64)
    rows, K = x.shape
    blocks = -(-K // 128)
    codes = np.zeros((rows, blocks * 128), np.uint8)
    exponents = np.full((rows, -(-blocks // 4) * 4), 127, np.uint8)
    steps = np.append(code_values()[:0x7F], np.inf)  # ascending non-negative values
    for b in range(blocks):
        part = x[:, b * 128:(b + 1) * 128]
        fine = np.isfinite(part)
        a = np.where(fine, np.abs(part), 0.0).max(axis=1)
        with np.errstate(divide="ignore"):
            e = np.where(a > 0, np.ceil(np.log2(a / 448.0)), -1000).astype(int)
        e += np.ldexp(448.0, e) < a  # log2's own rounding
        e -= np.ldexp(448.0, e - 1) >= a
        e = np.maximum(e, -126)
        v = np.ldexp(np.where(fine, part, 0.0), -e[:, None])
        v = np.where((e == 120)[:, None], np.clip(v, -240, 240), v)
        mag = np.abs(v)
        low = np.searchsorted(steps, mag, side="right") - 1
        down, up = mag - steps[low], steps[low + 1] - mag
        c = np.where((up < down) | ((up == down) & (low % 2 == 1)), low + 1, low).astype(np.uint8)
        c = np.where(np.signbit(np.where(fine, part, 0.0)), c | 128, c)
        c = np.where(fine, c, 0x7F)
        codes[:, b * 128:b * 128 + part.shape[1]] = c
        exponents[:, b] = e + 127
    return codes, exponents


def values(codes, exponents, K):
    rows, Kp = codes.shape
    p = np.ldexp(1.0, exponents[:, :Kp // 128].astype(int) - 127)
    return (code_values()[codes].reshape(rows, Kp // 128, 128) * p[:, :, None]).reshape(rows, Kp)[:, :K]


def linear(xv, wv, bias, relu):
    y = xv @ wv.T + (0.0 if bias is None else np.asarray(bias, np.float64))
    return np.maximum(y, 0.0) if relu else y


def pack_bits(mask):
    rows, N = mask.shape
    words = -(-N // 32)
    m = np.zeros((rows, words * 32), np.uint64)
    m[:, :N] = mask
    return (m.reshape(rows, words, 32) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32).view(np.int32)


def backward(dy, mask, xv, wv):
    dz = np.asarray(dy, np.float64) * (1.0 if mask is None else mask)
    return dz @ wv, dz.T @ xv, dz.sum(0)


def embedding(table, tokens, scale):
    table = np.asarray(table, np.float64)
    ok = (tokens >= 0) & (tokens < table.shape[0])
    return np.where(ok[:, None], table[np.where(ok, tokens, 0)], 0.0) * scale


def embedding_grad(d_out, tokens, V, scale):
    d = np.zeros((V, d_out.shape[1]))
    ok = (tokens >= 0) & (tokens < V)
    np.add.at(d, tokens[ok], np.asarray(d_out, np.float64)[ok])
    return d * scale
