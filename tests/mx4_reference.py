"""Float64 statements of the 4-bit KV store's operators, value by value from
their definitions -- TEST INFRASTRUCTURE."""
import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def blocks(d):
    return -(-d // 32)


def quantize(rows, heads, d):
    """Rows [count, heads * d] as (codes [count, heads, NB, 32], scale bytes
    [count, heads, NB])."""
    nb = blocks(d)
    x = np.zeros((rows.shape[0], heads, nb * 32))
    x[:, :, :d] = np.asarray(rows, np.float64).reshape(-1, heads, d)
    x = x.reshape(-1, heads, nb, 32)
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], 0.0, x)
    top = np.abs(x).max(-1)
    e = np.full(top.shape, -120)
    # The smallest exponent under which the largest magnitude rounds to at
    # most 6: below 7 (7 is a tie that goes to 8).
    while np.any(grow := (top >= 7 * np.exp2(e.astype(np.float64))) & (e < 125)):
        e = e + grow
    y = np.abs(x) / np.exp2(e.astype(np.float64))[..., None]
    # The nearest of the eight, ties to the even code.
    dist = np.abs(y[..., None] - VALUES)
    best = dist.min(-1, keepdims=True)
    code = np.where(dist == best, np.arange(8) % 2, 2).argmin(-1)
    code = code + 8 * np.signbit(x)
    return np.where(bad[..., None], 0, code).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(code, scale, d):
    """What codes and scale bytes stand for: [count, heads * d] in f64."""
    v = VALUES[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(scale == 255, np.nan, np.exp2(scale.astype(np.float64) - 127))
    x = (v * s[..., None]).reshape(code.shape[0], code.shape[1], -1)
    return x[:, :, :d].reshape(code.shape[0], -1)


def round_trip(rows, heads, d):
    return values(*quantize(rows, heads, d), d)


def pack(rows, capacity, heads, d, nbytes):
    """The bytes of a zeroed store after rows 0 .. count - 1 were written."""
    nb, groups = blocks(d), -(-capacity // 4)
    code, scale = quantize(rows, heads, d)
    out = np.zeros(nbytes, np.uint8)
    codes = out[:heads * groups * 64 * nb].reshape(heads, groups, 16, 4, nb)
    scales = out[codes.size:codes.size + heads * groups * 4 * nb].reshape(heads, groups, nb, 4)
    for r in range(rows.shape[0]):
        for p in range(nb):
            codes[:, r // 4, :, r % 4, p] = code[r, :, p, :16] | code[r, :, p, 16:] << 4
            scales[:, r // 4, p, r % 4] = scale[r, :, p]
    return out


def attention(q, k, v, heads, kv_heads, d, causal=True, window=None, scale=None):
    """q [seq, heads * d] over the held k, v [kv, kv_heads * d]: outputs, the
    attention each key received [kv_heads, kv], and the largest |score|."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    seq, kv = q.shape[0], k.shape[0]
    scale = scale if scale else 1.0 / np.sqrt(d)
    at = np.arange(seq)[:, None] + kv - seq
    key = np.arange(kv)[None, :]
    ok = np.ones((seq, kv), bool)
    if causal:
        ok = key <= at
        if window:
            ok &= key > at - window
    out = np.empty((seq, heads * d))
    received = np.zeros((kv_heads, kv))
    largest = 0.0
    for h in range(heads):
        m = h // (heads // kv_heads)
        kk, vv = k[:, m * d:(m + 1) * d], v[:, m * d:(m + 1) * d]
        with np.errstate(all="ignore"):
            s = np.where(ok, q[:, h * d:(h + 1) * d] @ kk.T * scale, -np.inf)
            fine = np.isfinite(s)
            largest = max(largest, np.abs(s[fine]).max() if fine.any() else 0.0)
            p = np.exp(s - s.max(-1, keepdims=True))
            p = p / p.sum(-1, keepdims=True)
            for i in range(seq):  # a key that is not admitted has no part, whatever it holds
                out[i, h * d:(h + 1) * d] = p[i, ok[i]] @ vv[ok[i]]
        received[m] += np.where(ok, p, 0.0).sum(0)
    return out, received, largest


def attention_tolerance(d, largest):
    """Of the relative 2-norm error. A score is 3 d products (three bf16 planes
    of a query, exact) summed in f32, each sum off by at most half a step, 2^-24:
    taken as independent, sqrt(3 d) of them times the largest score bound the
    error of the exponent, which is the weight's relative error; 16 more for the
    exponential, the weights' sum and the outputs'."""
    return 2.0 ** -24 * (np.sqrt(3 * d) * max(largest, 1.0) + 16)


def evict(weights, key_count, keep, first, recent):
    """The kept rows, in order, of one head's weights."""
    w = np.asarray(weights[:key_count], np.float64)
    w = np.where(np.isnan(w), -np.inf, w)
    lo, hi = first, key_count - recent
    order = sorted(range(lo, hi), key=lambda j: (-w[j], j))[:keep - first - recent]
    return np.array(list(range(lo)) + sorted(order) + list(range(hi, key_count)), np.int64)
