"""Plain 64-bit forms of the language-model operators, and how far a result of 32 bits may lie from them.

A rounding is off by at most half a step, 2**-24 relative in fp32 (U below), 2**-11 in fp16, 2**-8 in bf16."""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}       # of the rounding to the result's type, where it is another than fp32
LEAST = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}   # half a step of the smallest numbers


def quantize_rows(x, index=None):
    """x: float64 [rows, cols] -> (codes, scales); see zant_b200_quantize_rows."""
    if index is not None:
        known = (index >= 0) & (index < len(x))
        x = np.where(known[:, None], x[np.where(known, index, 0)] if len(x) else 0.0, 0.0)
    with np.errstate(all="ignore"):
        top = np.abs(x).max(axis=1)
        scale = (top / 127).astype(np.float32)
        bad = ~np.isfinite(x).all(axis=1)
        none = bad | (scale == 0)
        q = np.rint(x / np.where(none, 1, scale).astype(np.float64)[:, None])
        q = np.where(none[:, None], 0, np.clip(q, -127, 127)).astype(np.int8)
    return q, np.where(bad, np.float32(np.nan), scale)


def scaled_product(a, a_scale, w, w_scale, bias, kind):
    """(y, how far off y may be): the sum is exact; its conversion and two products round once each, the bias once, the result's type once."""
    p = (a.astype(np.float64) @ w.astype(np.float64).T) * a_scale.astype(np.float64)[:, None] * w_scale.astype(np.float64)
    y = p if bias is None else p + bias.astype(np.float64)
    off = 3.01 * U * np.abs(p) + (0 if bias is None else 1.01 * U * np.abs(y))
    return y, off + HALF_STEP[kind] * (np.abs(y) + off) + LEAST[kind]


def token_logprobs(x, tokens, top):
    """(logprob, entropy, ids, their log probabilities) of float64 rows."""
    n, vocab = x.shape
    with np.errstate(all="ignore"):
        m = x.max(axis=1, keepdims=True)
        m = np.where(np.isneginf(m), 0, m)
        e = np.exp(x - m)
        s = e.sum(axis=1, keepdims=True)
        logp = np.where(s == 0, -np.inf, x - m - np.log(s))
        bad = (np.isnan(x) | np.isposinf(x)).any(axis=1)
        logp[bad] = np.nan
        entropy = np.where(s[:, 0] == 0, 0, -np.where(e == 0, 0, (e / s) * logp).sum(axis=1))
        entropy[bad] = np.nan
    key = np.where(np.isnan(x), np.inf, x)
    first = np.isnan(x).astype(np.int64)
    ids = np.stack([np.lexsort((np.arange(vocab), -key[r], -first[r]))[:top] for r in range(n)]) if n else np.zeros((0, top), np.int64)
    given = None
    if tokens is not None:
        inside = (tokens >= 0) & (tokens < vocab)
        given = np.where(inside, np.take_along_axis(logp, np.where(inside, tokens, 0)[:, None].astype(np.int64), 1)[:, 0], np.where(tokens < 0, 0.0, np.nan))
    return given, entropy, ids.astype(np.int32), np.take_along_axis(logp, ids, 1)


def logprob_bound(x):
    """How far log p and entropy may be off, per row: (bound of log S alone, |x - m|'s share per unit, entropy's bound).

    Each e = exp(x - m) is off by the rounding of x - m (|d| U), of its product with log2 e (1.5 |d| U) and of the function (4 U):
    e |d| <= 0.37, so at most (4 e + 2.5 e |d|) U.  256 threads or more share a row: each adds at most vocab / 256 + 1 values one after
    the other, and the joins of lanes, warps and parts add 64 more roundings, each at most U of the sum."""
    vocab = x.shape[1]
    with np.errstate(all="ignore"):
        m = x.max(axis=1)
        d = np.where(np.isneginf(x), 0, x - np.where(np.isneginf(m), 0, m)[:, None])
        e = np.where(np.isneginf(x), 0, np.exp(d))
        s = e.sum(axis=1)
        mean_d = np.where(s > 0, (e * -d).sum(axis=1) / np.where(s > 0, s, 1), 0)
        mean_d2 = np.where(s > 0, (e * d * d).sum(axis=1) / np.where(s > 0, s, 1), 0)
        chain = vocab / 256 + 1 + 64
        rel_s = U * (chain + 4 + 2.5 * mean_d)
        log_s = rel_s + 4 * U * (1 + np.where(s > 0, np.abs(np.log(np.where(s > 0, s, 1))), 0))
        rel_w = U * ((chain + 6) * mean_d + 2.5 * mean_d2)         # of W / S, before S's own error
        entropy = log_s + rel_w + rel_s * mean_d + 4 * U * (1 + mean_d)
    return log_s, entropy
