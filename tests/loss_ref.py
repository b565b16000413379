"""The losses over a ternary head in 64 bits, and how far 32-bit kernels may
be from them.

Errors, with h = 2^-24 (half a step of 32 bits) and Z the largest sum of
magnitudes |product| + |bias| of a row's logits over tau: the logit's factor
is rounded four times (the constant log2(e) / (64 tau), times the row's
scale, times beta, the sum), its whole sum at most once, the bias twice, so a
logit is off by at most 8 h Z.  An exponential is off by 2 h relative besides
(one step), and by h |z - m| from its argument's rounding, which its own size
outweighs: |x| 2^x < 0.54.  A sum of positive numbers is off by h a link of
its chain: 32 in a lane, 8 joins in a tile, up to 8 tiles a thread at the sizes
tested here and 8 joins more.
"""
import numpy as np

F32, F64 = np.float32, np.float64
H = 2.0 ** -24


def quantise(x):
    """pack-act-rows' rounding: whole numbers (as float64) and the rows' scales (float32)."""
    g = (np.abs(x).max(axis=1, keepdims=True) / F32(127)).astype(F32)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(g > 0, (x / g).astype(F32), F32(0))
    return np.sign(q).astype(F64) * np.minimum(np.floor((np.abs(q) + F32(0.5)).astype(F32)), 127), g


def logits(h, w, bias, beta):
    """From rows as rounded (float64): logits, and the sums of magnitudes that make them."""
    p = (h @ w.T) * beta[None, :].astype(F64)
    b = np.zeros(w.shape[0]) if bias is None else bias.astype(F64)
    return p + b[None], np.abs(p) + np.where(np.isinf(b), 0, np.abs(b))[None]


def teacher_weights(index, teacher, teacher_lse, tau, vocab):
    """t [rows, top], zero where the index names nothing."""
    there = (index >= 0) & (index < vocab)
    if teacher is None:
        return there.astype(F64)
    y = np.where(there, teacher.astype(F64) / tau, -np.inf)
    if teacher_lse is None:
        m = y.max(axis=1, keepdims=True)
        with np.errstate(invalid="ignore"):
            e = np.where(there, np.exp(y - m), 0)
        return e / np.where(there.any(axis=1, keepdims=True), e.sum(axis=1, keepdims=True), 1)
    return np.exp(y - teacher_lse.astype(F64)[:, None])


def loss_of(h, w, bias, beta, index, t, tau):
    """loss, lse and the gradient with respect to h (for dloss 1)."""
    z = logits(h, w, bias, beta)[0] / tau
    m = z.max(axis=1, keepdims=True)
    e = np.exp(z - m)
    lse = (m + np.log(e.sum(axis=1, keepdims=True)))[:, 0]
    p = e / e.sum(axis=1, keepdims=True)
    rows = np.arange(z.shape[0])[:, None]
    at = np.where(t > 0, index, 0)
    with np.errstate(divide="ignore", invalid="ignore"):
        loss = np.where(t > 0, t * (np.log(t) - (z[rows, at] - lse[:, None])), 0).sum(axis=1)
    d = p * t.sum(axis=1, keepdims=True)
    np.add.at(d, (np.broadcast_to(rows, at.shape), at), -t)
    wb = w * beta[:, None].astype(F64)
    return loss, lse, d @ wb / tau, p


def tolerances(x, w, bias, beta, index, teacher, teacher_lse, t, tau, p):
    """Bounds [rows] of loss and lse and [rows, cols] of dx (for dloss 1)."""
    q, g = quantise(x)
    z = (logits(q * g, w, bias, beta)[1] / tau).max(axis=1)
    # a logit's error, the sum's, the logarithm's and its scaling (three roundings of the result)
    lse = H * (8 * z + 2 + 56 + 3 * (z + np.log(w.shape[0])))
    y = np.zeros_like(z)
    if teacher is not None:  # the same of the teacher's
        y = np.where((index >= 0) & (index < w.shape[0]) & np.isfinite(teacher), np.abs(teacher), 0).max(axis=1) / tau
        if teacher_lse is not None:
            y = y + np.abs(teacher_lse)
    lt = 0 if teacher is None else H * (8 * y + 64 + 3 * np.log(index.shape[1] + 1.0))
    # a target's two logarithms, its weight's error (relative: lt) times their difference, the sum over the targets
    T = t.sum(axis=1)
    apart = 2 * z + 2 * y + np.log(w.shape[0]) + np.log(index.shape[1] + 1.0)
    loss = T * (lse + 8 * H * z + lt + (lt + 12 * H) * apart)
    # a probability: its logit's and the log sum's error, the exponential, beta, two halves of 11 bits; steps of 2^-39;
    # the product's chain adds sixteen vocabulary rows twice at a time, and the parts meet
    wb = np.abs(w * beta[:, None].astype(F64))
    size = p @ wb
    e = lse + 8 * H * z + 8 * H
    dx = T[:, None] * (size * (e[:, None] + H * (w.shape[0] / 8 + 64)) + 2.0 ** -39 * wb.sum(axis=0)[None])
    # the targets' weights, subtracted one at a time
    tw = np.zeros_like(dx)
    for k in range(index.shape[1]):
        tw += t[:, k:k + 1] * wb[np.where(t[:, k] > 0, index[:, k], 0)]
    lt = np.broadcast_to(lt, z.shape)
    dx += T[:, None] * lt[:, None] * size + tw * (lt[:, None] + H * (index.shape[1] + 8)) + H * size * index.shape[1]
    return loss + H * T, lse, dx / tau * (1 + 2.0 ** -10)
