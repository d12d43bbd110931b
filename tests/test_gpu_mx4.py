"""GPU: 4-bit KV stores -- rows written and read, attention over them with the
attention each key received, and eviction by it -- against their definitions
in 64 bits (mx4_reference.py).

Bars: what a store holds, which rows an eviction keeps and what it moves are
exact; attention's tolerance is derived in mx4_reference.attention_tolerance.
"""
import numpy as np
import pytest

import mx4_reference as ref
from conftest import assert_bitexact

pytestmark = pytest.mark.gpu


def cache_rows(seed, count, heads, d):
    """Rows of many magnitudes: some blocks loud, some near zero, some zero."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((count, heads, d)) * np.exp2(rng.integers(-3, 3, (count, heads, 1)))
    x[rng.random((count, heads)) < 0.02] = 0.0
    return x.reshape(count, heads * d).astype(np.float32)


def store_of(dev, rows, capacity, heads, d, batch=1):
    from magnetar_hip import ops
    store = ops.Mx4Store(dev, capacity, heads, d, batch)
    if rows.size:
        ops.kv_write_mx4(dev, store, dev.upload(rows.reshape(batch, -1, heads * d)), 0)
    return store


def rel(got, want):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    return np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-300)


# ---- write and read ----

@pytest.mark.parametrize("d", [1, 31, 32, 33, 64, 80, 96, 100, 128, 160, 200, 224, 256])
@pytest.mark.parametrize("offset,count", [(0, 9), (5, 1), (3, 6), (6, 2)])
def test_rows_are_held_as_defined(dev, d, offset, count):
    """Packed bytes and read values, at offsets and counts inside a group of
    four rows and across groups; the rows around them keep their bits."""
    from magnetar_hip import ops
    heads, cap = 3, 14
    old, new = cache_rows(d, cap, heads, d), cache_rows(d + 500, count, heads, d)
    store = store_of(dev, old, cap, heads, d)
    ops.kv_write_mx4(dev, store, dev.upload(new), offset)
    rows = old.copy()
    rows[offset:offset + count] = new
    assert np.array_equal(store.data.numpy(), ref.pack(rows, cap, heads, d, store.data.nbytes))
    want = ref.round_trip(rows, heads, d).astype(np.float32)
    assert_bitexact(ops.kv_read_mx4(dev, store, 0, cap).numpy()[0], want)
    assert_bitexact(ops.kv_read_mx4(dev, store, offset, count).numpy()[0], want[offset:offset + count])


def test_every_rounding_and_extreme_magnitude(dev):
    """The ties and their neighbours, and blocks at the ends of f32's range."""
    from magnetar_hip import ops
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], np.float32)
    near = np.concatenate([np.nextafter(ties, np.float32(0)), ties, np.nextafter(ties, np.float32(9))])
    base = np.zeros((1, 32), np.float32)
    base[0, :24] = np.minimum(near, np.float32(6.99))
    base[0, 24:] = -near[:8]
    rows = [base * np.float32(2.0) ** np.float32(e) for e in (-126, -118, -60, 0, 1, 50, 120, 124)]
    top = np.zeros((6, 32), np.float32)
    top[0, 5] = np.finfo(np.float32).max
    top[1, 5] = np.float32(1.75 * 2.0 ** 127)
    top[2, 5] = np.nextafter(np.float32(1.75 * 2.0 ** 127), np.float32(0))
    top[3, 5] = np.finfo(np.float32).tiny
    top[4, 5] = np.float32(1e-45)
    top[5, 5] = np.float32(-0.0)
    rows = np.concatenate(rows + [top, 0.9 * top])
    store = store_of(dev, rows, len(rows), 1, 32)
    assert np.array_equal(store.data.numpy(), ref.pack(rows, len(rows), 1, 32, store.data.nbytes))
    got = ops.kv_read_mx4(dev, store, 0, len(rows)).numpy()[0]
    assert_bitexact(got, ref.round_trip(rows, 1, 32).astype(np.float32))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_block_that_is_not_finite_is_held_as_nan(dev, bad):
    from magnetar_hip import ops
    rows = cache_rows(3, 5, 2, 80)
    rows[2, 80 + 37] = bad  # head 1, block 1
    got = ops.kv_read_mx4(dev, store_of(dev, rows, 5, 2, 80), 0, 5).numpy()[0]
    want = ref.round_trip(rows, 2, 80)
    assert np.isnan(want[2, 80 + 32:80 + 64]).all() and np.isnan(want).sum() == 32
    assert np.array_equal(got, want.astype(np.float32), equal_nan=True)


def test_a_zeroed_store_holds_zeros_and_empty_calls_do_nothing(dev):
    from magnetar_hip import ops
    store = ops.Mx4Store(dev, 6, 2, 48)
    ops.kv_write_mx4(dev, store, dev.empty((1, 0, 96)), 6)
    assert ops.kv_read_mx4(dev, store, 6, 0).size == 0
    assert not ops.kv_read_mx4(dev, store, 0, 6).numpy().any()


def test_a_batch_of_stores_apart(dev):
    """Stores at a stride of their own, what lies between them left alone."""
    from magnetar_hip import ops
    cap, heads, d, batch = 7, 2, 64, 3
    one = heads * 2 * 68 * 2
    stride = one + 48
    data = dev.upload(np.full(batch * stride, 0xAB, np.uint8))
    store = ops.Mx4Store(dev, cap, heads, d, batch, dev.upload(np.full(batch * 1024, 0xAB, np.uint8)))
    store.data, store.shape.batch_stride = data, stride
    rows = cache_rows(5, batch * cap, heads, d).reshape(batch, cap, -1)
    ops.kv_write_mx4(dev, store, dev.upload(rows), 0)
    want = np.stack([ref.round_trip(r, heads, d) for r in rows]).astype(np.float32)
    assert_bitexact(ops.kv_read_mx4(dev, store, 0, cap).numpy(), want)
    held = data.numpy().reshape(batch, stride)
    assert (held[:, one:] == 0xAB).all()


def test_overruns_write_nothing(dev):
    import magnetar_hip
    from magnetar_hip import ops
    store = store_of(dev, cache_rows(1, 4, 1, 32), 4, 1, 32)
    before = store.data.numpy()
    with pytest.raises(magnetar_hip.MagnetarHipError) as err:
        ops.kv_write_mx4(dev, store, dev.upload(cache_rows(2, 2, 1, 32)), 3)
    assert err.value.code == "ShapeUnsupported"
    assert np.array_equal(store.data.numpy(), before)


# ---- attention ----

def check_attention(dev, seed, seq, kv, heads, kv_heads, d, causal=True, window=None, batch=1,
                    capacity=None, scale=None, weights=True, qstd=1.5):
    from magnetar_hip import ops
    cap = capacity or kv
    rng = np.random.default_rng(seed)
    q = (qstd * rng.standard_normal((batch, seq, heads * d))).astype(np.float32)
    rows = {n: np.full((batch, cap, kv_heads * d), np.nan, np.float32) for n in "kv"}
    for i, n in enumerate("kv"):
        for b in range(batch):
            rows[n][b, :kv] = cache_rows(100 * seed + 10 * b + i, kv, kv_heads, d)
    stores = {n: store_of(dev, rows[n], cap, kv_heads, d, batch) for n in "kv"}
    p = ops.attention_params(seq, cap, heads, d, kv_head_count=kv_heads, causal=causal,
                             window_size=window, key_count=kv, scale=scale, batch=batch)
    w_in = rng.random((batch, kv_heads, cap)).astype(np.float32)
    w_out = dev.upload(np.full((batch, kv_heads, cap), 7.0, np.float32))
    out = dev.upload(np.full((batch * seq + 1, heads * d), 5.0, np.float32))
    kwargs = dict(weights=dev.upload(w_in), weights_out=w_out) if weights else {}
    ops.attention_mx4(dev, dev.upload(q), stores["k"], stores["v"], p, out=out, **kwargs)
    got, got_w = out.numpy(), w_out.numpy()
    assert (got[-1] == 5.0).all()
    got = got[:-1].reshape(batch, seq, -1)
    for b in range(batch):
        held = [ref.round_trip(rows[n][b, :kv], kv_heads, d) for n in "kv"]
        want, received, largest = ref.attention(q[b], *held, heads, kv_heads, d, causal, window, scale)
        tol = ref.attention_tolerance(d, largest)
        assert rel(got[b], want) <= tol, (rel(got[b], want), tol)
        # No row alone is lost: each within the same relative error of itself,
        # times 8 for the spread over rows.
        for i in range(seq):
            assert rel(got[b, i], want[i]) <= 8 * tol, i
        if weights:
            assert rel(got_w[b, :, :kv], w_in[b, :, :kv] + received) <= tol
            assert np.allclose(got_w[b, :, :kv] - w_in[b, :, :kv], received, rtol=16 * tol, atol=2.0 ** -22 * 4)
            assert (got_w[b, :, kv:] == 7.0).all()


@pytest.mark.parametrize("d", [1, 4, 32, 33, 64, 80, 96, 112, 128, 130, 192, 224, 256])
def test_attention_head_dimensions(dev, d):
    check_attention(dev, d, 1, 333, 4, 2, d)
    check_attention(dev, d + 1, 21, 150, 4, 2, d)


@pytest.mark.parametrize("kv", [1, 2, 3, 4, 5, 63, 64, 65, 127, 255, 256, 257, 1000, 4097])
def test_attention_one_token_against_any_length(dev, kv):
    check_attention(dev, kv, 1, kv, 8, 2, 64, capacity=kv + 11)


@pytest.mark.parametrize("seq,kv,heads,kv_heads", [
    (1, 700, 1, 1), (1, 700, 16, 1), (1, 700, 32, 1), (1, 700, 7, 7), (2, 700, 12, 4), (5, 66, 24, 8),
    (16, 16, 4, 4), (17, 17, 6, 2), (33, 64, 4, 4), (64, 64, 4, 1), (65, 200, 2, 2), (130, 131, 4, 2),
])
def test_attention_group_sizes_and_row_tiles(dev, seq, kv, heads, kv_heads):
    check_attention(dev, seq * 7 + kv, seq, kv, heads, kv_heads, 128)
    check_attention(dev, seq * 7 + kv + 1, seq, kv, heads, kv_heads, 64, batch=2, capacity=kv + 3)


@pytest.mark.parametrize("seq,kv,heads,kv_heads,d,kw", [
    # Long enough for the prompts' kernel: whole row tiles of it split over their
    # keys, one chunk each, odd lengths, windows, blocks that are no power of two.
    (700, 700, 32, 4, 128, {}), (513, 1500, 24, 8, 96, dict(window=333)), (1030, 1030, 16, 16, 64, {}),
    (400, 2500, 16, 2, 80, dict(batch=2, capacity=2510)), (600, 1300, 16, 4, 32, dict(causal=False)),
    (500, 900, 16, 4, 160, {}), (420, 1000, 16, 4, 192, dict(window=100)), (300, 700, 16, 4, 256, {}),
    (900, 900, 32, 8, 100, dict(scale=0.3)),
])
def test_attention_prompts(dev, seq, kv, heads, kv_heads, d, kw):
    check_attention(dev, seq + kv, seq, kv, heads, kv_heads, d, **kw)


def test_attention_prompt_with_outliers_in_q(dev):
    """Q's planes are fixed-point within a block: values 1000 times smaller than
    their block's largest keep 2^-30 of it."""
    from magnetar_hip import ops
    rng = np.random.default_rng(5)
    seq, heads, d = 600, 16, 128
    q = rng.standard_normal((seq, heads * d)).astype(np.float32)
    q[:, 7::32] *= 1000.0
    k, v = cache_rows(1, seq, heads, d), cache_rows(2, seq, heads, d)
    k[:, 7::32] *= np.float32(1e-3)
    p = ops.attention_params(seq, seq, heads, d, causal=True)
    out = ops.attention_mx4(dev, dev.upload(q), store_of(dev, k, seq, heads, d), store_of(dev, v, seq, heads, d), p).numpy()
    want, _, largest = ref.attention(q, ref.round_trip(k, heads, d), ref.round_trip(v, heads, d), heads, heads, d)
    # Each of 32 values of a block is off by at most 2^-30 of the largest, the
    # held keys are within 6 of one another's scale: under 2^-30 * 3000 * 16 * 6 /
    # sqrt(128) of a score, beside the sums' own.
    assert rel(out, want) <= ref.attention_tolerance(d, largest) + 2.0 ** -30 * 3000 * 16 * 6 / np.sqrt(d)


@pytest.mark.parametrize("causal,window", [(False, None), (True, 1), (True, 7), (True, 64), (True, 100), (True, 5000)])
@pytest.mark.parametrize("seq,kv", [(1, 500), (9, 300), (100, 230), (300, 300)])
def test_attention_masks(dev, causal, window, seq, kv):
    check_attention(dev, seq + kv, seq, kv, 4, 2, 64, causal=causal, window=window)
    check_attention(dev, seq + kv + 1, seq, kv, 4, 4, 128, causal=causal, window=window, batch=2)


def test_attention_scale_and_large_scores(dev):
    check_attention(dev, 1, 3, 200, 4, 2, 64, scale=0.5)
    check_attention(dev, 2, 3, 200, 4, 2, 64, qstd=40.0)   # one key takes all
    check_attention(dev, 3, 40, 200, 4, 2, 128, qstd=1e-3)


def test_attention_without_weights_has_the_same_outputs(dev):
    check_attention(dev, 4, 1, 900, 8, 2, 128, weights=False)
    check_attention(dev, 5, 200, 900, 8, 2, 128, weights=False)


def nonfinite_case(dev, seq, kv, heads, kv_heads, d, window, k_bad, v_bad, q_bad=()):
    from magnetar_hip import ops
    rng = np.random.default_rng(seq + kv)
    q = rng.standard_normal((seq, heads * d)).astype(np.float32)
    k, v = cache_rows(1, kv, kv_heads, d), cache_rows(2, kv, kv_heads, d)
    for row, col in k_bad:
        k[row, col] = np.nan
    for row, col in v_bad:
        v[row, col] = np.inf
    for row, col in q_bad:
        q[row, col] = np.inf
    p = ops.attention_params(seq, kv, heads, d, kv_head_count=kv_heads, causal=True, window_size=window)
    w = dev.empty((1, kv_heads, kv))
    out = ops.attention_mx4(dev, dev.upload(q), store_of(dev, k, kv, kv_heads, d), store_of(dev, v, kv, kv_heads, d),
                            p, weights_out=w).numpy()
    want, received, largest = ref.attention(q, ref.round_trip(k, kv_heads, d), ref.round_trip(v, kv_heads, d),
                                            heads, kv_heads, d, True, window)
    for got, expect in ((out, want), (w.numpy()[0], received)):
        assert np.array_equal(np.isnan(got), np.isnan(expect))
        fine = ~np.isnan(expect)
        assert np.allclose(got[fine], expect[fine], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("seq,kv", [(40, 40), (40, 200), (130, 130), (1500, 1500)])
@pytest.mark.parametrize("window", [None, 9])
def test_values_that_are_not_finite_reach_the_queries_that_admit_them(dev, seq, kv, window):
    """A NaN block of K or V next to the mask's edges: queries that admit the
    key get NaN (in the value's 32 columns, in all of them for a key), the
    others what they get without it."""
    nonfinite_case(dev, seq, kv, 4, 2, 80, window, [], [(kv - 20, 80 + 33), (kv - 7, 3)])
    nonfinite_case(dev, seq, kv, 4, 2, 80, window, [(kv - 11, 90)], [])
    nonfinite_case(dev, seq, kv, 4, 2, 64, window, [(kv - 1, 5)], [(kv - 1, 70), (0, 0)])


def test_a_query_that_is_not_finite_gives_nan_to_its_own_row(dev):
    nonfinite_case(dev, 20, 90, 4, 2, 64, None, [], [], [(3, 70), (19, 0)])


def test_sixteen_queries_and_keys_far_apart(dev):
    """Rows of very different maxima in one tile, over several chunks."""
    check_attention(dev, 9, 16, 3000, 8, 8, 64, qstd=8.0)


# ---- eviction ----

def evict_case(dev, batch, heads, d, cap, count, keep, first, recent, weights, out_cap=None, in_place=False,
               indices=True):
    from magnetar_hip import ops
    rows = {n: cache_rows(i + 31, batch * cap, heads, d).reshape(batch, cap, -1) for i, n in enumerate("kv")}
    stores = {n: store_of(dev, rows[n], cap, heads, d, batch) for n in "kv"}
    out_cap = cap if in_place else (out_cap or keep + 3)
    old = {n: cache_rows(i + 77, batch * out_cap, heads, d).reshape(batch, out_cap, -1) for i, n in enumerate("kv")}
    outs = stores if in_place else {n: store_of(dev, old[n], out_cap, heads, d, batch) for n in "kv"}
    if in_place:
        old = rows
    w = dev.upload(weights)
    w_out = w if in_place else dev.upload(np.full((batch, heads, out_cap), -3.0, np.float32))
    idx = dev.upload(np.zeros((batch, heads, keep), np.uint32)) if indices else None
    ops.kv_evict_mx4(dev, stores["k"], stores["v"], w, count, keep, outs["k"], outs["v"], w_out, idx,
                     first=first, recent=recent)
    got = {n: ops.kv_read_mx4(dev, outs[n], 0, out_cap).numpy().reshape(batch, out_cap, heads, d) for n in "kv"}
    got_w = w_out.numpy()
    for b in range(batch):
        want = {n: ref.round_trip(rows[n][b], heads, d).reshape(cap, heads, d) for n in "kv"}
        behind = {n: ref.round_trip(old[n][b], heads, d).reshape(out_cap, heads, d) for n in "kv"}
        for h in range(heads):
            at = ref.evict(weights[b, h], count, keep, first, recent)
            if indices:
                assert np.array_equal(idx.numpy()[b, h], at)
            assert np.array_equal(got_w[b, h, :keep], weights[b, h][at], equal_nan=True)
            assert not got_w[b, h, keep:].any()
            for n in "kv":
                assert np.array_equal(got[n][b, :keep, h], want[n][at, h]), (b, h, n)
                assert np.array_equal(got[n][b, keep:, h], behind[n][keep:, h]), (b, h, n)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,heads,d,cap,count,keep,first,recent", [
    (1, 1, 32, 8, 8, 3, 0, 0), (1, 2, 64, 10, 9, 9, 0, 0), (2, 3, 80, 101, 100, 37, 4, 10),
    (1, 2, 128, 2100, 2047, 1022, 4, 128), (1, 1, 256, 60, 60, 1, 0, 1), (1, 1, 33, 60, 60, 1, 1, 0),
    (1, 2, 64, 60, 60, 20, 8, 12), (1, 1, 64, 5000, 4999, 4097, 0, 0), (3, 2, 96, 300, 270, 0, 0, 0),
    # On both sides of what a workgroup's registers hold.
    (1, 1, 32, 8193, 8192, 5000, 3, 7), (1, 2, 32, 8200, 8193, 4100, 0, 100), (1, 1, 32, 16385, 16384, 9000, 0, 0), (1, 1, 32, 16387, 16385, 9000, 4, 500),
    (1, 1, 32, 40000, 39999, 30001, 0, 0),
])
def test_eviction_keeps_the_heaviest(dev, in_place, batch, heads, d, cap, count, keep, first, recent):
    rng = np.random.default_rng(cap)
    w = np.exp(2 * rng.standard_normal((batch, heads, cap))).astype(np.float32)
    evict_case(dev, batch, heads, d, cap, count, keep, first, recent, w, in_place=in_place, indices=keep % 2 == 1)


@pytest.mark.parametrize("kind", ["equal", "few", "special", "negative"])
def test_eviction_ties_and_odd_weights(dev, kind):
    """Ties go to the lowest row; NaN counts as -inf and -0 as 0."""
    rng = np.random.default_rng(8)
    if kind == "few":  # ties across the stretches of a long account
        evict_case(dev, 1, 1, 32, 33000, 32999, 20001, 5, 9, rng.integers(0, 3, (1, 1, 33000)).astype(np.float32))
    w = rng.integers(0, 3, (1, 2, 1500)).astype(np.float32)
    if kind == "equal":
        w[:] = 1.5
    elif kind == "special":
        w = rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-42, 1.0, -1.0], np.float32), (1, 2, 1500))
    elif kind == "negative":
        w = -np.abs(rng.standard_normal((1, 2, 1500))).astype(np.float32)
    for keep in (1, 700, 1400, 1490):
        evict_case(dev, 1, 2, 64, 1500, 1490, keep, 0, 0, w)
        evict_case(dev, 1, 2, 64, 1500, 1490, keep, 1, keep // 3, w) if keep > 1 else None


# ---- together ----

def test_a_conversation_over_a_bounded_cache(dev):
    """A prompt and decode steps over 4-bit stores with their account of
    attended rows, evicted whenever the cache is full, against the same in 64
    bits over the rows that the reference keeps."""
    from magnetar_hip import ops
    heads, kv_heads, d, cap, keep = 4, 2, 64, 96, 48
    rng = np.random.default_rng(12)
    k, v = (ops.Mx4Store(dev, cap, kv_heads, d) for _ in range(2))
    w = dev.zeros((1, kv_heads, cap))
    held = {n: np.zeros((kv_heads, 0, d)) for n in "kv"}
    account = np.zeros((kv_heads, 0))
    used = evictions = 0
    for seq in [37] + [1] * 40 + [19] + [1] * 30:
        if used + seq > cap:
            ops.kv_evict_mx4(dev, k, v, w, used, keep, k, v, w, first=2, recent=8)
            at = [ref.evict(account[h], used, keep, 2, 8) for h in range(kv_heads)]
            got = ops.kv_read_mx4(dev, k, 0, keep).numpy()[0].reshape(keep, kv_heads, d)
            for n in "kv":
                held[n] = np.stack([held[n][h][at[h]] for h in range(kv_heads)])
            account = np.stack([account[h][at[h]] for h in range(kv_heads)])
            assert np.array_equal(got.transpose(1, 0, 2), held["k"])
            used, evictions = keep, evictions + 1
        rows = {n: cache_rows(int(rng.integers(1 << 30)), seq, kv_heads, d) for n in "kv"}
        q = rng.standard_normal((seq, heads * d)).astype(np.float32)
        ops.kv_write_mx4(dev, k, dev.upload(rows["k"]), used)
        ops.kv_write_mx4(dev, v, dev.upload(rows["v"]), used)
        used += seq
        for n in "kv":
            new = ref.round_trip(rows[n], kv_heads, d).reshape(seq, kv_heads, d).transpose(1, 0, 2)
            held[n] = np.concatenate([held[n], new], 1)
        p = ops.attention_params(seq, cap, heads, d, kv_head_count=kv_heads, causal=True, key_count=used)
        out = ops.attention_mx4(dev, dev.upload(q), k, v, p, weights=w, weights_out=w).numpy()
        flat = [held[n].transpose(1, 0, 2).reshape(used, -1) for n in "kv"]
        want, received, largest = ref.attention(q, *flat, heads, kv_heads, d)
        assert rel(out, want) <= ref.attention_tolerance(d, largest)
        account = np.concatenate([account, np.zeros((kv_heads, seq))], 1) + received
        got = w.numpy()[0, :, :used]
        assert rel(got, account) <= 40 * ref.attention_tolerance(d, largest)
        # The account is f32 on the device: the next eviction goes by its own.
        account = got.astype(np.float64)
    assert evictions >= 1


@pytest.mark.parametrize("d,heads,kv_heads", [(64, 4, 2), (128, 8, 8), (80, 4, 1), (64, 40, 1)])
def test_a_captured_step_replays_down_the_cache(dev, d, heads, kv_heads):
    """Write, attention and account recorded once and replayed at later rows
    equal the eager calls at those rows bit for bit, eager work in between."""
    from magnetar_hip import ops
    from magnetar_hip.device import ADVANCE_KEY_COUNT, ADVANCE_ROW_OFFSET
    cap, start, steps = 700, 293, [0, 1, 2, 3, 5, 90, 290, 406]
    past = {n: cache_rows(i + 1, cap, kv_heads, d) for i, n in enumerate("kv")}
    row = {n: dev.upload(cache_rows(i + 5, 1, kv_heads, d)) for i, n in enumerate("kv")}
    q = dev.upload(np.random.default_rng(1).standard_normal((1, heads * d)).astype(np.float32))
    w_in = dev.upload(np.random.default_rng(2).random((1, kv_heads, cap)).astype(np.float32))
    stores = {n: store_of(dev, past[n], cap, kv_heads, d) for n in "kv"}
    out, w_out = dev.zeros((1, heads * d)), dev.zeros((1, kv_heads, cap))

    def step(at, stores, out, w_out):
        for n in "kv":
            ops.kv_write_mx4(dev, stores[n], row[n], at)
        p = ops.attention_params(1, cap, heads, d, kv_head_count=kv_heads, causal=True, key_count=at + 1)
        ops.attention_mx4(dev, q, stores["k"], stores["v"], p, out=out, weights=w_in, weights_out=w_out)

    step(start, {n: store_of(dev, past[n], cap, kv_heads, d) for n in "kv"}, dev.zeros((1, heads * d)),
         dev.zeros((1, kv_heads, cap)))  # the workspace has its size
    dev.capture_begin(ADVANCE_KEY_COUNT | ADVANCE_ROW_OFFSET)
    step(start, stores, out, w_out)
    captured = dev.capture_end()
    assert captured.max_offset == cap - start - 1
    for offset in steps:
        captured.launch(offset)
        dev.sync()
        got, got_w = out.numpy(), w_out.numpy()
        e_stores = {n: store_of(dev, past[n], cap, kv_heads, d) for n in "kv"}
        for earlier in steps[:steps.index(offset)]:
            for n in "kv":
                ops.kv_write_mx4(dev, e_stores[n], row[n], start + earlier)
        e_out, e_w = dev.zeros((1, heads * d)), dev.zeros((1, kv_heads, cap))
        step(start + offset, e_stores, e_out, e_w)
        assert_bitexact(got, e_out.numpy(), f"offset {offset}")
        count = start + offset + 1
        assert_bitexact(got_w[..., :count], e_w.numpy()[..., :count], f"weights at {offset}")
        for n in "kv":
            assert np.array_equal(stores[n].data.numpy(), e_stores[n].data.numpy())
    captured.close()


def test_a_captured_eviction_replays(dev):
    from magnetar_hip import ops
    rng = np.random.default_rng(4)
    k, v = (store_of(dev, cache_rows(i, 200, 2, 64), 200, 2, 64) for i in range(2))
    k2, v2 = (ops.Mx4Store(dev, 50, 2, 64) for _ in range(2))
    w, w2 = dev.upload(rng.random((1, 2, 200)).astype(np.float32)), dev.zeros((1, 2, 50))
    idx = dev.upload(np.zeros((1, 2, 50), np.uint32))
    ops.kv_evict_mx4(dev, k, v, w, 190, 50, k2, v2, w2, idx, first=1, recent=9)
    dev.capture_begin()
    ops.kv_evict_mx4(dev, k, v, w, 190, 50, k2, v2, w2, idx, first=1, recent=9)
    captured = dev.capture_end()
    for seed in range(4):
        weights = np.random.default_rng(seed).random((1, 2, 200)).astype(np.float32)
        dev.write(w, weights)
        captured.launch()
        got = idx.numpy()
        for h in range(2):
            assert np.array_equal(got[0, h], ref.evict(weights[0, h], 190, 50, 1, 9))
        dev.zeros((64,)).numpy()
    captured.close()


def test_a_fresh_context_captures_all_calls():
    """A context without scratch records the calls that need some and replays
    them with the eager call's bits; two captures share the scratch."""
    import magnetar_hip
    from magnetar_hip import ops
    heads, kv_heads, d, kv, seq = 8, 2, 64, 900, 70
    rng = np.random.default_rng(9)
    rows = {n: cache_rows(i, kv, kv_heads, d) for i, n in enumerate("kv")}
    q_host = rng.standard_normal((seq, heads * d)).astype(np.float32)

    def calls(dev, st):
        p = ops.attention_params(seq, kv, heads, d, kv_head_count=kv_heads, causal=True)
        ops.attention_mx4(dev, st["q"], st["k"], st["v"], p, out=st["o"], weights_out=st["w"])
        ops.kv_evict_mx4(dev, st["k"], st["v"], st["w"], kv, 300, st["k2"], st["v2"], st["w2"], first=2, recent=50)
        p1 = ops.attention_params(1, 300, heads, d, kv_head_count=kv_heads)
        ops.attention_mx4(dev, st["q1"], st["k2"], st["v2"], p1, out=st["o1"], weights=st["w2"], weights_out=st["w3"])

    def state(dev):
        st = {n: ops.Mx4Store(dev, kv, kv_heads, d) for n in "kv"}
        for n in "kv":
            ops.kv_write_mx4(dev, st[n], dev.upload(rows[n]), 0)
        st |= {n: ops.Mx4Store(dev, 300, kv_heads, d) for n in ("k2", "v2")}
        st |= {"q": dev.upload(q_host), "q1": dev.upload(q_host[:1]), "o": dev.zeros((seq, heads * d)),
               "o1": dev.zeros((1, heads * d)), "w": dev.zeros((1, kv_heads, kv)),
               "w2": dev.zeros((1, kv_heads, 300)), "w3": dev.zeros((1, kv_heads, 300))}
        return st

    with magnetar_hip.Device(0) as eager:
        st = state(eager)
        calls(eager, st)
        want = {n: st[n].numpy() for n in ("o", "w", "w2", "o1", "w3")}
        del st
    with magnetar_hip.Device(0) as dev:
        st = state(dev)
        graphs = []
        for _ in range(2):
            dev.capture_begin()
            calls(dev, st)
            graphs.append(dev.capture_end())
        for turn in range(4):
            for n in ("o", "o1", "w3"):
                dev.write(st[n], np.zeros(st[n].shape, np.float32))
            graphs[turn % 2].launch()
            dev.sync()
            for n, x in want.items():
                assert_bitexact(st[n].numpy(), x, f"{n}, replay {turn}")
        for g in graphs:
            g.close()
        del st


def test_two_contexts_side_by_side(dev):
    """The chunks' counters and the scratch are a context's own."""
    import magnetar_hip
    from magnetar_hip import ops
    heads, d, kv = 4, 128, 6000
    rows = [cache_rows(i, kv, heads, d) for i in range(2)]
    q = np.random.default_rng(2).standard_normal((1, heads * d)).astype(np.float32)
    with magnetar_hip.Device(0) as other:
        sides = []
        for side in (dev, other):
            sides.append((side, side.upload(q), store_of(side, rows[0], kv, heads, d), store_of(side, rows[1], kv, heads, d),
                          ops.attention_params(1, kv, heads, d), [side.zeros((1, heads * d)) for _ in range(20)]))
        for i in range(20):
            for side, x, k, v, p, outs in sides:
                ops.attention_mx4(side, x, k, v, p, out=outs[i])
        first = sides[0][5][0].numpy()
        for side in sides:
            for o in side[5]:
                assert_bitexact(o.numpy(), first)
        del side, sides, o, outs, x, k, v


def test_unaligned_rows_and_outputs(dev):
    """Queries and outputs at 4-byte addresses take the scalar forms."""
    from magnetar_hip import DeviceArray, ops
    heads, d = 4, 64
    for seq, kv in ((1, 300), (40, 300), (700, 1200)):
        k, v = (store_of(dev, cache_rows(i, kv, heads, d), kv, heads, d) for i in range(2))
        q = np.random.default_rng(seq).standard_normal((seq, heads * d)).astype(np.float32)
        p = ops.attention_params(seq, kv, heads, d, causal=True)
        want = ops.attention_mx4(dev, dev.upload(q), k, v, p).numpy()
        held = dev.upload(np.concatenate([[0.0], q.ravel()]).astype(np.float32))
        into = dev.zeros((seq * heads * d + 1,))
        ops.attention_mx4(dev, DeviceArray(dev, held.ptr + 4, q.shape, np.float32, owned=False), k, v, p,
                          out=DeviceArray(dev, into.ptr + 4, q.shape, np.float32, owned=False))
        got = into.numpy()
        assert got[0] == 0.0
        assert_bitexact(got[1:].reshape(q.shape), want)


def test_weights_of_a_window_far_down_a_long_cache(dev):
    """A window's rows are counted back from every key of the cache: 2.2 million
    keys under 1024 query heads of one KV head pass 31 bits. Zeros are held, so
    each of the 16 keys admitted gets 1/16 from each head, exactly."""
    from magnetar_hip import ops
    heads, d, kv, window = 1024, 32, 2200000, 16
    k, v = (ops.Mx4Store(dev, kv, 1, d) for _ in range(2))
    q = dev.upload(np.random.default_rng(3).standard_normal((1, heads * d)).astype(np.float32))
    w = dev.zeros((1, 1, kv))
    out = ops.attention_mx4(dev, q, k, v, ops.attention_params(1, kv, heads, d, kv_head_count=1, causal=True, window_size=window),
                            weights=w, weights_out=w)
    assert not out.numpy().any()
    got = w.numpy()[0, 0]
    assert not got[:-window].any() and (got[-window:] == heads / window).all()


@pytest.mark.parametrize("seq,kv", [(1, 300), (5, 300), (60, 300), (600, 900)])
def test_sequences_at_strides_of_their_own(dev, seq, kv):
    """Queries, outputs and stores of a batch at strides of their own: the bits
    of each sequence by itself, what lies between left alone; then an eviction
    in place of the same stores."""
    import ctypes

    from magnetar_hip import _lib, ops
    batch, heads, kv_heads, d, cap = 2, 4, 2, 64, kv + 5
    one = kv_heads * -(-cap // 4) * 68 * 2
    stride, q_bs, o_bs = one + (-one) % 16 + 32, seq * heads * d + 8, seq * heads * d + 4
    rows = [[cache_rows(10 * i + b, kv, kv_heads, d) for b in range(batch)] for i in range(2)]
    held = [dev.upload(np.full(batch * stride, 0xAB, np.uint8)) for _ in range(2)]
    alone = [[store_of(dev, rows[i][b], cap, kv_heads, d) for b in range(batch)] for i in range(2)]
    shape = _lib.Mx4StoreShape(cap, kv_heads, d, batch, stride)
    for i in range(2):
        both = dev.upload(np.stack(rows[i]))
        _lib.call("mhip_kv_write_mx4", dev.ctx, ctypes.c_void_p(held[i].ptr), ctypes.byref(shape), ctypes.c_void_p(both.ptr), kv, 0)
    q = np.random.default_rng(seq).standard_normal((batch, q_bs)).astype(np.float32)
    x = dev.upload(q)
    out, w = dev.upload(np.full((batch, o_bs), 5.0, np.float32)), dev.zeros((batch, kv_heads, cap))
    p = ops.attention_params(seq, cap, heads, d, kv_head_count=kv_heads, causal=True, key_count=kv, batch=batch)
    p.q_batch_stride, p.out_batch_stride, p.kv_batch_stride, p.v_batch_stride = q_bs, o_bs, stride, stride
    _lib.call("mhip_attention_mx4", dev.ctx, *(ctypes.c_void_p(t.ptr) for t in (x, held[0], held[1], out)), ctypes.byref(p), None,
              ctypes.c_void_p(w.ptr))
    got, got_w = out.numpy(), w.numpy()
    assert (got[:, seq * heads * d:] == 5.0).all()
    for b in range(batch):
        pb = ops.attention_params(seq, cap, heads, d, kv_head_count=kv_heads, causal=True, key_count=kv)
        w1 = dev.zeros((1, kv_heads, cap))
        want = ops.attention_mx4(dev, dev.upload(q[b, :seq * heads * d]), alone[0][b], alone[1][b], pb, weights_out=w1).numpy()
        # One sequence's chunks may be shorter: the same sums in another order.
        held_rows = [ref.round_trip(rows[i][b], kv_heads, d) for i in range(2)]
        exact, received, largest = ref.attention(q[b, :seq * heads * d].reshape(seq, -1), *held_rows, heads, kv_heads, d)
        tol = ref.attention_tolerance(d, largest)
        assert rel(got[b, :seq * heads * d], want.ravel()) <= 2 * tol
        assert rel(got[b, :seq * heads * d], exact.ravel()) <= tol
        assert rel(got_w[b, :, :kv], received) <= tol and not got_w[b, :, kv:].any()
    keep = kv // 2
    e = _lib.KvEvictParams(kv, keep, 2, 9, cap, cap)
    _lib.call("mhip_kv_evict_mx4", dev.ctx, ctypes.c_void_p(held[0].ptr), ctypes.c_void_p(held[1].ptr), ctypes.c_void_p(w.ptr),
              ctypes.byref(shape), ctypes.byref(e), ctypes.c_void_p(held[0].ptr), ctypes.c_void_p(held[1].ptr), ctypes.byref(shape),
              ctypes.c_void_p(w.ptr), None)
    for i in range(2):
        into = dev.zeros((batch, keep, kv_heads, d))
        _lib.call("mhip_kv_read_mx4", dev.ctx, ctypes.c_void_p(held[i].ptr), ctypes.byref(shape), ctypes.c_void_p(into.ptr), keep, 0)
        kept = into.numpy()
        for b in range(batch):
            full = ref.round_trip(rows[i][b], kv_heads, d).reshape(kv, kv_heads, d)
            for h in range(kv_heads):
                at = ref.evict(got_w[b, h], kv, keep, 2, 9)
                assert np.array_equal(kept[b, :, h], full[at, h])
        assert (held[i].numpy().reshape(batch, stride)[:, one:] == 0xAB).all()
