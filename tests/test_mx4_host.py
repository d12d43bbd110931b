"""4-bit KV stores without a GPU: the sizes of a store, the reference that the
device is held to, and every refusal. A refused call ends before it touches
its context, so a block of zeros stands for one here."""
import ctypes

import numpy as np
import pytest

import mx4_reference as ref


@pytest.fixture(scope="module")
def mh():
    import magnetar_hip
    return magnetar_hip


def test_store_bytes(mh):
    size = mh.lib().mhip_kv_mx4_bytes
    for cap, heads, d in [(1, 1, 1), (4, 1, 32), (5, 2, 33), (4096, 8, 128), (131072, 8, 256), (0, 3, 64)]:
        used = heads * -(-cap // 4) * 68 * ref.blocks(d)
        assert size(cap, heads, d) == -(-used // 256) * 256
    assert size(4, 0, 64) == size(4, 1, 0) == size(4, 1, 257) == size(1 << 31, 1, 64) == 0


def test_reference_rounds_to_the_nearest_code_and_ties_to_even():
    x = np.zeros((1, 32), np.float32)
    x[0, :17] = [6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, 0.2500001, 0.7499999, 4.9, 5.1, -6, -3.4, 0.1]
    got = ref.round_trip(x, 1, 32)[0]
    assert got[:17].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, -1, 0.5, 0.5, 4, 6, -6, -3, 0]


@pytest.mark.parametrize("top,exponent", [(6.0, 0), (6.999, 0), (7.0, 1), (3.5, 0), (3.4999, -1),
                                          (1.0, -2), (0.0, -120), (2.0 ** -130, -120), (3.3e38, 125)])
def test_reference_scale(top, exponent):
    x = np.zeros((1, 32), np.float32)
    x[0, 3] = top
    assert ref.quantize(x, 1, 32)[1][0, 0, 0] == exponent + 127


def _call(mh, name, *args):
    blank = ctypes.create_string_buffer(1 << 14)
    status = getattr(mh.lib(), name)(ctypes.cast(blank, ctypes.c_void_p), *args)
    return mh.STATUS_NAMES[status], mh.lib().mhip_last_error_detail().decode()


# Addresses that no refused call reads.
BUF = [ctypes.c_void_p(0x10000000 * (i + 1)) for i in range(8)]


def _shape(mh, capacity=64, heads=2, d=64, batch=1, stride=0):
    return mh._lib.Mx4StoreShape(capacity, heads, d, batch, stride)


@pytest.mark.parametrize("shape,count,offset,store,code,words", [
    (dict(), 3, 62, BUF[0], "ShapeUnsupported", "exceeds the store's 64 rows"),
    (dict(), 1, 2 ** 64 - 1, BUF[0], "ShapeUnsupported", "exceeds the store's 64 rows"),
    (dict(heads=0), 1, 0, BUF[0], "ShapeUnsupported", "must be positive"),
    (dict(d=0), 1, 0, BUF[0], "ShapeUnsupported", "must be positive"),
    (dict(d=288), 1, 0, BUF[0], "ShapeUnsupported", "head dimension 288"),
    (dict(capacity=1 << 31), 1, 0, BUF[0], "ShapeUnsupported", "too large"),
    (dict(batch=2, stride=1000), 1, 0, BUF[0], "LayoutUnsupported", "multiple of 16"),
    (dict(batch=2, stride=4096), 1, 0, BUF[0], "ShapeUnsupported", "below a store's size"),
    (dict(), 1, 0, ctypes.c_void_p(0), "ShapeUnsupported", "null buffer"),
    (dict(), 1, 0, ctypes.c_void_p(0x10000008), "LayoutUnsupported", "16-byte aligned"),
])
def test_write_and_read_refusals(mh, shape, count, offset, store, code, words):
    s = _shape(mh, **shape)
    for name, args in (("mhip_kv_write_mx4", (store, ctypes.byref(s), BUF[1], count, offset)),
                       ("mhip_kv_read_mx4", (store, ctypes.byref(s), BUF[1], count, offset))):
        got, detail = _call(mh, name, *args)
        assert got == code and words in detail, (name, got, detail)
    assert getattr(mh.lib(), "mhip_kv_write_mx4")(None, store, ctypes.byref(s), BUF[1], count, offset) == 8
    got, detail = _call(mh, "mhip_kv_write_mx4", store, None, BUF[1], count, offset)
    assert got == "ShapeUnsupported" and "null store shape" in detail


@pytest.mark.parametrize("change,weights,code,words", [
    (dict(head_count=3), (None, None), "ShapeUnsupported", "exact multiple"),
    (dict(kv_head_count=0), (None, None), "ShapeUnsupported", "must all be positive"),
    (dict(head_dimension=257, value_dimension=0), (None, None), "ShapeUnsupported", "above 256"),
    (dict(value_dimension=32), (None, None), "ShapeUnsupported", "keys' head dimension"),
    (dict(window_size=0), (None, None), "ShapeUnsupported", "window_size must be positive"),
    (dict(window_size=4, causal=0), (None, None), "ShapeUnsupported", "only defined for causal"),
    (dict(kv_seq_len=65), (None, None), "ShapeUnsupported", "key_count 65 exceeds the 64 rows"),
    (dict(kv_seq_len=2), (None, None), "ShapeUnsupported", "cannot exceed k/v sequence length"),
    (dict(scale=float("nan")), (None, None), "ShapeUnsupported", "finite and positive"),
    (dict(scale=float("inf")), (None, None), "ShapeUnsupported", "finite and positive"),
    (dict(kv_batch_stride=4100), (None, None), "LayoutUnsupported", "multiple of 16"),
    (dict(kv_rows=1 << 31, kv_seq_len=64), (None, None), "ShapeUnsupported", "too large"),
    (dict(), (BUF[4], None), "ShapeUnsupported", "without an output"),
    (dict(seq_len=0), (None, BUF[4]), "ShapeUnsupported", "no query"),
])
def test_attention_refusals(mh, change, weights, code, words):
    p = mh.ops.attention_params(3, 64, 4, 64, kv_head_count=2, causal=True, key_count=64)
    for key, value in change.items():
        setattr(p, key, value)
    got, detail = _call(mh, "mhip_attention_mx4", *BUF[:4], ctypes.byref(p), *weights)
    assert got == code and words in detail, (got, detail)


def test_attention_refuses_null_and_unaligned_buffers(mh):
    p = mh.ops.attention_params(1, 64, 4, 64, causal=True)
    for i in range(4):
        args = list(BUF[:4])
        args[i] = None
        got, detail = _call(mh, "mhip_attention_mx4", *args, ctypes.byref(p), None, None)
        assert got == "ShapeUnsupported" and "null buffer" in detail
    for i in (1, 2):
        args = list(BUF[:4])
        args[i] = ctypes.c_void_p(args[i].value + 4)
        got, detail = _call(mh, "mhip_attention_mx4", *args, ctypes.byref(p), None, None)
        assert got == "LayoutUnsupported" and "16-byte aligned" in detail
    assert _call(mh, "mhip_attention_mx4", *BUF[:4], None, None, None)[0] == "ShapeUnsupported"


@pytest.mark.parametrize("params,out,buffers,code,words", [
    (dict(key_count=65), {}, {}, "ShapeUnsupported", "exceeds the store's 64 rows"),
    (dict(keep=61), {}, {}, "ShapeUnsupported", "cannot keep 61 of 60"),
    (dict(), dict(capacity=31), {}, "ShapeUnsupported", "exceed the output store's 31"),
    (dict(first=20, recent=13), {}, {}, "ShapeUnsupported", "exceed the rows to keep"),
    (dict(first=2 ** 64 - 1, recent=2), {}, {}, "ShapeUnsupported", "exceed the rows to keep"),
    (dict(weight_stride=59), {}, {}, "ShapeUnsupported", "stride is below"),
    (dict(weight_out_stride=63), {}, {}, "ShapeUnsupported", "stride is below"),
    (dict(), dict(heads=1), {}, "ShapeUnsupported", "differ in heads"),
    (dict(), dict(d=32), {}, "ShapeUnsupported", "differ in heads"),
    (dict(), dict(batch=2), {}, "ShapeUnsupported", "differ in heads"),
    (dict(), {}, {2: None}, "ShapeUnsupported", "null buffer"),
    (dict(), {}, {5: None}, "ShapeUnsupported", "null buffer"),
    (dict(), {}, {3: ctypes.c_void_p(0x40000004)}, "LayoutUnsupported", "16-byte aligned"),
    # K in place and V not; a shifted copy; both outputs in one buffer; the
    # stores themselves under another shape; shifted weights.
    (dict(), {}, {3: BUF[0]}, "LayoutUnsupported", "overlap"),
    (dict(), {}, {3: ctypes.c_void_p(BUF[0].value + 64)}, "LayoutUnsupported", "overlap"),
    (dict(), {}, {3: BUF[4]}, "LayoutUnsupported", "overlap"),
    (dict(), {}, {3: BUF[1], 4: BUF[0]}, "LayoutUnsupported", "overlap"),
    (dict(), dict(capacity=48), {3: BUF[0], 4: BUF[1]}, "LayoutUnsupported", "overlap"),
    (dict(), {}, {5: ctypes.c_void_p(BUF[2].value + 4)}, "LayoutUnsupported", "weights overlap"),
    (dict(weight_out_stride=80), {}, {5: BUF[2]}, "LayoutUnsupported", "weights overlap"),
])
def test_evict_refusals(mh, params, out, buffers, code, words):
    s, o = _shape(mh), _shape(mh, **{**dict(capacity=64), **out})
    p = mh._lib.KvEvictParams(60, 32, 4, 8, 0, 0)
    for key, value in params.items():
        setattr(p, key, value)
    b = {i: buffers.get(i, BUF[i]) for i in range(6)}
    got, detail = _call(mh, "mhip_kv_evict_mx4", b[0], b[1], b[2], ctypes.byref(s), ctypes.byref(p), b[3],
                        b[4], ctypes.byref(o), b[5], None)
    assert got == code and words in detail, (got, detail)


@pytest.mark.parametrize("count,width,width_out", [(60, 59, 64), (1, 0, 64), (60, 64, 63), (60, 64, 0)])
def test_evict_refuses_weights_of_fewer_rows(mh, count, width, width_out):
    """Before any call: weights of no rows would else pass as the stride 0, the
    store's capacity."""
    def array(*shape):
        return mh.DeviceArray(None, 0, shape, np.float32, owned=False)

    store = object.__new__(mh.ops.Mx4Store)
    store._key = (64, 2, 32, 1)
    with pytest.raises(ValueError, match="fewer rows"):
        mh.ops.kv_evict_mx4(None, store, store, array(1, 2, width), count, 1, store, store, array(1, 2, width_out))
