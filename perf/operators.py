"""Performance cases of the 4-bit key/value cache: rows written into a store
and read back, attention over a store (single tokens, chunks and whole
prompts, with or without the accumulated attention weights), and eviction of
the rows that were attended least.

A store holds f32 rows [capacity, kv_heads * d] as 4-bit floating-point codes
(sign, two exponent bits, one fraction bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), each
block of 32 values of a head under one power-of-two scale. Where `own` is
false the operators run in their plain form, from elementary operations.

Buffers are torch tensors; the library sees them as DeviceArray views.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "magnetar-provider-cuda_amd")
_DEVICE = None


def _lib():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import magnetar_hip
    return magnetar_hip


def _dev():
    """The program's one bound device."""
    global _DEVICE
    if _DEVICE is None:
        _DEVICE = _lib().Device(0)
    return _DEVICE


# --------------------------------------------------------------------------
# The cases
# --------------------------------------------------------------------------

def listed():
    return [
        # One decode step's key rows for a batch of four sequences: the
        # smallest call, where launches count.
        _write("write_token", batch=4, rows=1, heads=8, d=128, position=777),
        # The key rows of a whole prompt, one cache row per token and head.
        _write("write_prompt", batch=1, rows=4099, heads=32, d=128, position=0),
        # The tiny Llama-style block's heads (4 of 64), one token against a
        # short history.
        _attention("decode_short", batch=1, seq=1, kv=301, heads=4, kv_heads=4, d=64),
        # A batch of decode steps of a grouped-query model.
        _attention("decode_batch", batch=8, seq=1, kv=4096, heads=32, kv_heads=8, d=128),
        # One token against a very long history.
        _attention("decode_long", batch=1, seq=1, kv=131073, heads=32, kv_heads=8, d=128),
        # Decode steps that keep account of which rows they attended.
        _attention("decode_weights", batch=4, seq=1, kv=8191, heads=32, kv_heads=8, d=128,
                   weights=True),
        # A few drafted tokens checked at once, a head dimension of 80.
        _attention("draft_check", batch=2, seq=5, kv=3001, heads=32, kv_heads=32, d=80),
        # A whole prompt of a grouped-query model.
        _attention("prompt", batch=1, seq=2048, kv=2048, heads=32, kv_heads=8, d=128),
        # A later chunk of a prompt under a sliding window, odd length.
        _attention("prompt_chunk", batch=1, seq=509, kv=4605, heads=16, kv_heads=4, d=64,
                   window=1500),
        # A prompt that starts the account of attended rows.
        _attention("prompt_weights", batch=1, seq=1021, kv=1021, heads=32, kv_heads=32, d=128,
                   weights=True),
        # A short cache halved.
        _evict("evict_short", batch=1, kv=1024, keep=512, first=4, recent=128, heads=4, d=64),
        # A batch of long caches cut to a quarter.
        _evict("evict_batch", batch=8, kv=8192, keep=2050, first=4, recent=512, heads=8, d=128),
    ]


def _write(name, batch, rows, heads, d, position):
    return {"name": name, "kind": "write", "batch": batch, "rows": rows, "heads": heads, "d": d,
            "position": position}


def _attention(name, batch, seq, kv, heads, kv_heads, d, causal=True, window=0, weights=False):
    return {"name": name, "kind": "attention", "batch": batch, "seq": seq, "kv": kv, "heads": heads,
            "kv_heads": kv_heads, "d": d, "causal": causal, "window": window, "weights": weights}


def _evict(name, batch, kv, keep, first, recent, heads, d):
    return {"name": name, "kind": "evict", "batch": batch, "kv": kv, "keep": keep, "first": first,
            "recent": recent, "heads": heads, "d": d}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MOST_FLOPS, _MOST_BYTES = 3.4e10, 1.4e8  # of a drawn case


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES:
            del case["name"]
            return case


def _draw(rng):
    kind = rng.choice(["write", "decode", "decode", "decode", "prompt", "prompt", "prompt", "evict"])
    d = rng.choice([32, 64, 64, 80, 96, 112, 128, 128, 128, 256])
    if kind == "write":
        return _write("", _log_int(rng, 1, 16), _log_int(rng, 1, 4200), rng.choice([1, 2, 4, 8, 32]),
                      d, rng.choice([0, _log_int(rng, 1, 8000)]))
    if kind == "evict":
        kv = _log_int(rng, 64, 20000)
        keep = max(1, int(kv * rng.uniform(0.1, 0.95)))
        first = min(keep, rng.choice([0, 4]))
        return _evict("", _log_int(rng, 1, 8), kv, keep, first,
                      int((keep - first) * rng.uniform(0.0, 0.7)), rng.choice([1, 4, 8, 8]), d)
    heads = rng.choice([4, 8, 16, 32])
    kv_heads = max(1, heads // rng.choice([1, 2, 4, 4, 8]))
    weights = rng.random() < 0.3
    if kind == "decode":
        seq = rng.choice([1, 1, 1, rng.randint(2, 12)])
        return _attention("", _log_int(rng, 1, 16), seq, seq + _log_int(rng, 100, 100000), heads,
                          kv_heads, d, True, _log_int(rng, 64, 4096) if rng.random() < 0.2 else 0,
                          weights)
    seq = _log_int(rng, 16, 2048)
    kv = seq + rng.choice([0, 0, _log_int(rng, 16, 4096)])
    causal = rng.random() < 0.85
    window = _log_int(rng, 64, 2048) if causal and rng.random() < 0.25 else 0
    return _attention("", _log_int(rng, 1, 4), seq, kv, heads, kv_heads, d, causal, window, weights)


# --------------------------------------------------------------------------
# The store: codes and scales
# --------------------------------------------------------------------------
# For NB = ceil(d / 32) blocks of 32 values a head and groups of four rows,
#   codes  [kv_heads][ceil(capacity / 4)][16][4 rows][NB] bytes, then
#   scales [kv_heads][ceil(capacity / 4)][NB][4 rows] bytes,
# rounded up to 256 bytes a sequence. Byte (n, row, p) holds the codes of the
# head's values 32 p + n (low half) and 32 p + 16 + n (high half); a scale
# byte s stands for 2^(s - 127), 255 for NaN.

_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_VALUES = _VALUES + [-v for v in _VALUES]


def _blocks(d):
    return (d + 31) // 32


def _store_bytes(capacity, heads, d):
    n = heads * ((capacity + 3) // 4) * 68 * _blocks(d)
    return (n + 255) // 256 * 256


def _quantize(rows, heads, d):
    """Rows [..., heads * d] as codes [..., heads, NB, 32] and scale exponents
    [..., heads, NB] (128: not a number)."""
    nb = _blocks(d)
    x = rows.reshape(*rows.shape[:-1], heads, d)
    x = torch.nn.functional.pad(x, (0, nb * 32 - d)).reshape(*x.shape[:-1], nb, 32)
    top = x.abs().amax(-1)
    _, e = torch.frexp(top)             # top = f * 2^e, f in [0.5, 1)
    f = torch.ldexp(top, -e)
    e = e - 3 + (f >= 0.875).to(e.dtype)  # the largest value rounds to at most 6
    e = torch.where(top == 0, -120, e).clamp(-120, 125)
    bad = ~torch.isfinite(x).all(-1)
    y = torch.ldexp(x, -e.unsqueeze(-1))
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) +
            (a >= 3.5) + (a > 5.0))     # to the nearest, ties to the even code
    code = code + 8 * torch.signbit(y)
    return torch.where(bad.unsqueeze(-1), 0, code).to(torch.uint8), torch.where(bad, 128, e)


def _pack(rows, capacity, heads, d):
    """A store [batch, bytes] that holds `rows` [batch, count <= capacity, heads * d]."""
    batch, count = rows.shape[:2]
    nb, groups = _blocks(d), (capacity + 3) // 4
    code, e = _quantize(rows, heads, d)
    code = torch.nn.functional.pad(code, (0, 0, 0, 0, 0, 0, 0, 4 * groups - count))
    e = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, 0, 0, 0, 0, 4 * groups - count))
    code = code.reshape(batch, groups, 4, heads, nb, 2, 16)
    byte = code[..., 0, :] + 16 * code[..., 1, :]       # [batch, groups, 4, heads, nb, 16]
    byte = byte.permute(0, 3, 1, 5, 2, 4).reshape(batch, -1)
    scale = e.reshape(batch, groups, 4, heads, nb).permute(0, 3, 1, 4, 2).reshape(batch, -1)
    n = _store_bytes(capacity, heads, d)
    return torch.nn.functional.pad(torch.cat([byte, scale], 1), (0, n - byte.shape[1] - scale.shape[1]))


def _unpack(store, capacity, heads, d, dtype):
    """The values [batch, capacity, heads, d] that a store stands for."""
    batch = store.shape[0]
    nb, groups = _blocks(d), (capacity + 3) // 4
    n = heads * groups * 64 * nb
    byte = store[:, :n].reshape(batch, heads, groups, 16, 4, nb).permute(0, 2, 4, 1, 5, 3)
    scale = store[:, n:n + n // 16].reshape(batch, heads, groups, nb, 4).permute(0, 2, 4, 1, 3)
    code = torch.stack([byte & 15, byte >> 4], -2)      # [batch, groups, 4, heads, nb, 2, 16]
    x = torch.tensor(_VALUES, device=store.device, dtype=dtype)[code.to(torch.int64)]
    s = torch.exp2(scale.to(dtype) - 127)
    s = torch.where(scale == 255, math.nan, s)[..., None, None]
    return (x * s).reshape(batch, 4 * groups, heads, nb * 32)[:, :capacity, :, :d]


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + 29)
    return g


def _normal(g, shape, std=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g)


def _cache_rows(g, batch, count, heads, d):
    """Key or value rows: normal, some channels several times the others'."""
    x = _normal(g, (batch, count, heads, d))
    loud = torch.rand((heads, d), device="cuda", generator=g) < 0.05
    return (x * torch.where(loud, 4.0, 1.0)).reshape(batch, count, heads * d)


def _capacity(c):
    return c["kv"] + 37  # rows that a later step will write


def prepare(case, seed):
    c, g = case, _gen(seed)
    kind = c["kind"]
    st = {"case": c, "in": {}, "out": {}}
    t, out = st["in"], st["out"]
    if kind == "write":
        width = c["heads"] * c["d"]
        cap = c["position"] + c["rows"] + 5
        t["rows"] = _cache_rows(g, c["batch"], c["rows"], c["heads"], c["d"])
        t["store"] = torch.zeros((c["batch"], _store_bytes(cap, c["heads"], c["d"])),
                                 dtype=torch.uint8, device="cuda")
        out["rows"] = torch.empty((c["batch"], c["rows"], width), device="cuda")
        st["capacity"] = cap
    else:
        B, Hk, d = c["batch"], c["heads" if kind == "evict" else "kv_heads"], c["d"]
        cap = st["capacity"] = _capacity(c)
        for name in ("k", "v"):
            t[name] = _pack(_cache_rows(g, B, c["kv"], Hk, d), cap, Hk, d)
        if kind == "attention":
            t["q"] = _normal(g, (B * c["seq"], c["heads"] * d), 1.5)
            out["o"] = torch.empty_like(t["q"])
            if c["weights"]:
                t["weights"] = torch.rand((B, Hk, cap), device="cuda", generator=g) ** 4
                out["weights"] = torch.zeros_like(t["weights"])
        else:
            # Accumulated weights: heavy-tailed, many rows hardly attended
            # and some never.
            w = torch.exp(2.0 * _normal(g, (B, Hk, cap)))
            t["weights"] = torch.where(w < 0.1, 0.0, w)
            keep = c["keep"]
            for name in ("k", "v"):
                out[name + "_store"] = torch.zeros((B, _store_bytes(keep, Hk, d)), dtype=torch.uint8,
                                                   device="cuda")
                out[name] = torch.empty((B, keep, Hk * d), device="cuda")
            out["weights"] = torch.empty((B, Hk, keep), device="cuda")
            out["indices"] = torch.empty((B, Hk, keep), dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()  # the inputs were made on torch's stream
    return st


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------

def _view(t):
    """A torch tensor as the library sees it."""
    dtype = {torch.uint8: np.uint8, torch.int32: np.uint32}.get(t.dtype, np.float32)
    return _lib().DeviceArray(_dev(), t.data_ptr(), tuple(t.shape), dtype, None, owned=False)


def _handles(state):
    """The library's views of the state's buffers, which a program keeps."""
    if "handles" not in state:
        ops, c, cap = _lib().ops, state["case"], state["capacity"]
        h = {"in_" + n: _view(x) for n, x in state["in"].items()}
        h |= {"out_" + n: _view(x) for n, x in state["out"].items()}
        hk = c.get("kv_heads", c["heads"])
        for n in ("in_store", "in_k", "in_v"):
            if n in h:
                h[n] = ops.Mx4Store(_dev(), cap, hk, c["d"], c["batch"], h[n])
        for n in ("out_k_store", "out_v_store"):
            if n in h:
                h[n] = ops.Mx4Store(_dev(), c["keep"], hk, c["d"], c["batch"], h[n])
        if c["kind"] == "attention":
            h["params"] = ops.attention_params(c["seq"], cap, c["heads"], c["d"], kv_head_count=hk,
                                               causal=c["causal"], window_size=c["window"] or None,
                                               key_count=c["kv"], batch=c["batch"])
        state["handles"] = h
    return state["handles"]


def run(state):
    c = state["case"]
    if own:
        return _run_own(state)
    return {"write": _plain_write, "attention": _plain_attention, "evict": _plain_evict}[c["kind"]](state)


def _run_own(state):
    c, dev, h, out = state["case"], _dev(), _handles(state), state["out"]
    ops = _lib().ops
    if c["kind"] == "write":
        ops.kv_write_mx4(dev, h["in_store"], h["in_rows"], c["position"])
        ops.kv_read_mx4(dev, h["in_store"], c["position"], c["rows"], out=h["out_rows"])
        return out["rows"]
    if c["kind"] == "attention":
        if not c["weights"]:
            ops.attention_mx4(dev, h["in_q"], h["in_k"], h["in_v"], h["params"], out=h["out_o"])
            return out["o"]
        ops.attention_mx4(dev, h["in_q"], h["in_k"], h["in_v"], h["params"], out=h["out_o"],
                          weights=h["in_weights"], weights_out=h["out_weights"])
        return {"o": out["o"], "weights": out["weights"][:, :, :c["kv"]]}
    ops.kv_evict_mx4(dev, h["in_k"], h["in_v"], h["in_weights"], c["kv"], c["keep"],
                     h["out_k_store"], h["out_v_store"], h["out_weights"], h["out_indices"],
                     first=c["first"], recent=c["recent"])
    ops.kv_read_mx4(dev, h["out_k_store"], 0, c["keep"], out=h["out_k"])
    ops.kv_read_mx4(dev, h["out_v_store"], 0, c["keep"], out=h["out_v"])
    return {n: out[n] for n in ("k", "v", "weights", "indices")}


def _plain_write(state):
    """The written rows, as the store then holds them."""
    c, x = state["case"], state["in"]["rows"]
    code, e = _quantize(x, c["heads"], c["d"])
    value = torch.tensor(_VALUES, device="cuda")[code.to(torch.int64)]
    value = torch.ldexp(value, e.unsqueeze(-1)).reshape(*x.shape[:2], c["heads"], -1)
    return value[..., :c["d"]].reshape(x.shape)


def _admitted(c):
    """Which of the keys [kv] each query [seq] admits."""
    at = torch.arange(c["seq"], device="cuda")[:, None] + (c["kv"] - c["seq"])
    key = torch.arange(c["kv"], device="cuda")[None, :]
    if not c["causal"]:
        return torch.ones((c["seq"], c["kv"]), dtype=torch.bool, device="cuda")
    ok = key <= at
    return ok & (key > at - c["window"]) if c["window"] else ok


def _plain_attention(state):
    c, t = state["case"], state["in"]
    B, S, H, Hk, d, kv = c["batch"], c["seq"], c["heads"], c["kv_heads"], c["d"], c["kv"]
    k, v = (_unpack(t[n], state["capacity"], Hk, d, torch.float32)[:, :kv].permute(0, 2, 1, 3).contiguous()
            for n in ("k", "v"))                        # [B, Hk, kv, d]
    q = t["q"].reshape(B, S, Hk, H // Hk, d).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, d)
    s = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(d)).reshape(B, Hk, H // Hk, S, kv)
    s.masked_fill_(~_admitted(c), -math.inf)
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    p = s.div_(s.sum(-1, keepdim=True)).reshape(B, Hk, -1, kv)
    o = torch.matmul(p, v).reshape(B, Hk, H // Hk, S, d).permute(0, 3, 1, 2, 4).reshape(B * S, H * d)
    if not c["weights"]:
        return o
    return {"o": o, "weights": t["weights"][:, :, :kv] + p.sum(2)}


def _plain_evict(state):
    c, t = state["case"], state["in"]
    B, H, d, kv, keep = c["batch"], c["heads"], c["d"], c["kv"], c["keep"]
    w = t["weights"][:, :, :kv]
    # The first and the most recent rows stay; of the others those of the
    # largest weights, ties to the lowest row.
    row = torch.arange(kv, device="cuda")
    rank = torch.where((row < c["first"]) | (row >= kv - c["recent"]), math.inf, w)
    index = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    out = {"weights": torch.gather(w, -1, index), "indices": index.to(torch.int32)}
    for n in ("k", "v"):
        x = _unpack(t[n], state["capacity"], H, d, torch.float32)      # [B, capacity, H, d]
        at = index.permute(0, 2, 1).unsqueeze(-1).expand(B, keep, H, d)
        out[n] = torch.gather(x, 1, at).reshape(B, keep, H * d)
    return out


# --------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------

def _pairs(c):
    """(query, key) pairs of one head and sequence."""
    if not c["causal"]:
        return c["seq"] * c["kv"]
    reach = c["window"] or c["kv"]
    return sum(min(reach, c["kv"] - c["seq"] + i + 1) for i in range(c["seq"]))


def _rows_read(c):
    """Keys that some query admits."""
    if not c["causal"] or not c["window"]:
        return c["kv"]
    return min(c["kv"], c["seq"] + c["window"] - 1)


def work(case):
    c = case
    B, d = c["batch"], c["d"]
    packed = 17 * _blocks(d)  # bytes of one row of one head
    if c["kind"] == "write":
        n = B * c["rows"] * c["heads"]
        return {"bytes": n * (8 * d + 2 * packed), "flops": 4 * n * d}
    if c["kind"] == "evict":
        n = B * c["heads"] * c["keep"]
        # The weights once; the kept rows moved, and read as values.
        return {"bytes": B * c["heads"] * c["kv"] * 4 + n * (8 + 2 * (3 * packed + 4 * d)),
                "flops": B * c["heads"] * c["kv"] * 4}
    rows = B * c["kv_heads"] * _rows_read(c)
    kept = 8 * B * c["kv_heads"] * c["kv"] if c["weights"] else 0
    return {"bytes": 8 * B * c["seq"] * c["heads"] * d + 2 * rows * packed + kept,
            "flops": 4.0 * B * c["heads"] * _pairs(c) * d}


# --------------------------------------------------------------------------
# The same in 64 bits, from the definitions
# --------------------------------------------------------------------------

def _value_table():
    """The sixteen code values: (-1)^s 2^(x - 1) (1 + m / 2), x > 0; (-1)^s m / 2 for x = 0."""
    got = []
    for code in range(16):
        s, x, m = code >> 3, (code >> 1) & 3, code & 1
        got.append((-1.0) ** s * (2.0 ** (x - 1) * (1 + m / 2) if x else m / 2))
    return torch.tensor(got, dtype=torch.float64, device="cuda")


def _held(store, capacity, heads, d):
    """What a store holds, [batch, heads, capacity, d] in 64 bits, value by value."""
    nb, groups = _blocks(d), (capacity + 3) // 4
    row = torch.arange(capacity, device="cuda")[:, None]
    col = torch.arange(d, device="cuda")[None, :]
    p, half, n = col // 32, col % 32 // 16, col % 16
    table = _value_table()
    out = torch.empty((store.shape[0], heads, capacity, d), dtype=torch.float64, device="cuda")
    for h in range(heads):
        at = (((h * groups + row // 4) * 16 + n) * 4 + row % 4) * nb + p
        scale_at = heads * groups * 64 * nb + ((h * groups + row // 4) * nb + p) * 4 + row % 4
        for b in range(store.shape[0]):
            code = (store[b][at].to(torch.int64) >> (4 * half)) & 15
            e = store[b][scale_at].to(torch.float64) - 127
            out[b, h] = table[code] * torch.pow(torch.full_like(e, 2.0), e)
    return out


def _round_block(x):
    """Blocks [..., 32] in 64 bits, rounded to the nearest of the sixteen
    values under the smallest power of two whose largest value holds them."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -118))) - 2
    e = torch.where(top >= 7 * torch.exp2(e), e + 1, e)
    e = torch.where(top < 3.5 * torch.exp2(e), e - 1, e).clamp(-120, 125)
    y = x / torch.exp2(e)
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), y) * torch.exp2(e)


def exact(case, seed):
    st = prepare(case, seed)
    c, t = case, st["in"]
    d = c["d"]
    if c["kind"] == "write":
        x = t["rows"].to(torch.float64).reshape(c["batch"], c["rows"], c["heads"], d)
        parts = [_round_block(x[..., b:b + 32]) for b in range(0, d, 32)]
        return torch.cat(parts, -1).reshape(t["rows"].shape)
    B, kv = c["batch"], c["kv"]
    if c["kind"] == "evict":
        # Which rows stay is counted row by row: those that fewer than the
        # free places are ahead of.
        H, keep = c["heads"], c["keep"]
        w = t["weights"][:, :, :kv].to(torch.float64)
        lo, hi = c["first"], kv - c["recent"]
        index = torch.empty((B, H, keep), dtype=torch.int64, device="cuda")
        for b in range(B):
            for h in range(H):
                order = np.lexsort((np.arange(lo, hi), -w[b, h, lo:hi].cpu().numpy())) + lo
                kept = np.concatenate([np.arange(lo), np.sort(order[:keep - lo - c["recent"]]),
                                       np.arange(hi, kv)])
                index[b, h] = torch.from_numpy(kept).to(index.device)
        out = {"weights": torch.gather(w, -1, index), "indices": index}
        for n in ("k", "v"):
            x = _held(t[n], st["capacity"], H, d)
            x = torch.gather(x, 2, index.unsqueeze(-1).expand(B, H, keep, d))
            out[n] = x.permute(0, 2, 1, 3).reshape(B, keep, H * d)
        return out
    S, H, Hk = c["seq"], c["heads"], c["kv_heads"]
    held = {n: _held(t[n], st["capacity"], Hk, d)[:, :, :kv] for n in ("k", "v")}
    q = t["q"].to(torch.float64).reshape(B, S, H, d)
    o = torch.empty((B, S, H, d), dtype=torch.float64, device="cuda")
    kept = t["weights"][:, :, :kv].to(torch.float64) if c["weights"] else None
    at = torch.arange(S, device="cuda", dtype=torch.float64)[:, None] + (kv - S)
    key = torch.arange(kv, device="cuda", dtype=torch.float64)[None, :]
    low = at - c["window"] + 1 if c["window"] else torch.zeros_like(at)
    outside = (key > at) | (key < low) if c["causal"] else torch.zeros((S, kv), dtype=torch.bool, device="cuda")
    for b in range(B):
        for h in range(H):
            m = h // (H // Hk)
            p = torch.softmax((q[b, :, h] @ held["k"][b, m].T / math.sqrt(d)).masked_fill(outside, -math.inf), -1)
            o[b, :, h] = p @ held["v"][b, m]
            if kept is not None:
                kept[b, m] += p.sum(0)
    o = o.reshape(B * S, H * d)
    return o if kept is None else {"o": o, "weights": kept}
