"""fc_Q4A in 64 bits, with how far fp32 sums may be from it: for the tests of FCs whose weights depend on the row."""
import numpy as np

EPS = 2.0 ** -24  # half a step of fp32, relative


def quantize(x, G):
    """fp32 [rows, K] -> codes [rows, Kg, G], scales [rows, Kg] (fp32 arithmetic, which defines them), group sums in 64 bits and
    the sums of absolute values."""
    rows, K = x.shape
    Kg = -(-K // G)
    codes = np.zeros((rows, Kg, G))
    d, sums, absolute = np.zeros((rows, Kg), np.float32), np.zeros((rows, Kg)), np.zeros((rows, Kg))
    for kb in range(Kg):
        part = x[:, kb * G: (kb + 1) * G]
        amax = np.abs(part).max(1)
        d[:, kb] = amax / np.float32(127)
        inverse = np.divide(np.float32(1), d[:, kb], out=np.zeros_like(amax), where=d[:, kb] != 0)
        t = part * inverse[:, None]
        body = part.shape[1] // 8 * 8
        q = np.rint(t).astype(np.float64)
        q[:, body:] = np.trunc(t[:, body:].astype(np.float64) + np.copysign(0.5, t[:, body:]))
        codes[:, kb, : part.shape[1]] = np.clip(q, -128, 127)
        sums[:, kb], absolute[:, kb] = part.astype(np.float64).sum(1), np.abs(part).astype(np.float64).sum(1)
    return codes, d.astype(np.float64), sums, absolute


def unpack(wq, qtype, G, signed=False):
    """int8 [Ng, Kg, bytes] -> nibbles [Kg, G, Ng * 32], scales and minima [Kg, Ng * 32]."""
    u = wq.view(np.uint8)
    Ng, Kg, _ = u.shape
    word = u[..., : 16 * G].reshape(Ng, Kg, G // 8, 32, 4)
    nib = np.stack((word & 15, word >> 4), -2).astype(np.float64)  # [Ng, Kg, G/8, column, half, 4]
    if signed:
        nib = np.where(nib > 7, nib - 16, nib)
    nib = nib.transpose(1, 2, 4, 5, 0, 3).reshape(Kg, G, Ng * 32)
    d = u[..., 16 * G: 16 * G + 64].copy().view(np.float16).astype(np.float64).transpose(1, 0, 2).reshape(Kg, Ng * 32)
    m = np.zeros_like(d)
    if qtype == 1:
        m = u[..., 16 * G + 64:].copy().view(np.float16).astype(np.float64).transpose(1, 0, 2).reshape(Kg, Ng * 32)
    return nib, d, m


def fc64(x, wq, N, qtype, G, signed=False):
    """fp32 [rows, K] through one packed tensor: the product in 64 bits, and a bound of an fp32 kernel's error.

    The integers are exact.  A term of a group is a product of three factors (two roundings, or one in a fused addition), a group
    sum is a tree of at most 3 + 7 additions, and the at most 2 Kg terms of an output and what its partial sums add (warps and
    CTAs: at most 16 + 8) meet in chains no longer than that: each addition rounds by half a step of a partial sum, which the sum of
    the absolute terms bounds."""
    codes, d, sums, absolute = quantize(x, G)
    nib, wd, wm = unpack(wq, qtype, G, signed)
    rows, Kg = d.shape
    y, size, loose = np.zeros((rows, nib.shape[2])), np.zeros((rows, nib.shape[2])), np.zeros((rows, nib.shape[2]))
    for kb in range(Kg):
        term = d[:, kb, None] * (codes[:, kb] @ nib[kb]) * wd[kb]
        low = sums[:, kb, None] * wm[kb]
        y += term + low
        size += np.abs(term) + np.abs(low)
        loose += absolute[:, kb, None] * np.abs(wm[kb])
    bound = ((2 * Kg + 24) + 3) * EPS * size + 11 * EPS * loose
    return y[:, :N], bound[:, :N] + 1e-30
