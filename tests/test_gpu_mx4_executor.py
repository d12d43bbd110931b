"""GPU: 4-bit KV stores behind the executor -- kv-write and attention take one in
place of an f32 store, reads return its values, other Kernels refuse it -- and a
captured decode step over them. Attention's tolerance is derived in
mx4_reference.attention_tolerance; the rest is exact.
"""
import numpy as np
import pytest

import mx4_reference as ref
from conftest import assert_bitexact
from test_gpu_mx4 import cache_rows, rel

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ex():
    import magnetar_hip
    p = magnetar_hip.Provider()
    yield p.execution_api()
    p.close()


def inv(kernel, inputs, output, attrs=None):
    from magnetar_hip import KernelInvocation, TensorRef
    return KernelInvocation(kernel, [TensorRef(i) for i in inputs], [TensorRef(output)], attrs or {})


def attrs(heads, kv_heads, d, count):
    from magnetar_hip import Boolean, Integer
    return {"head_count": Integer(heads), "kv_head_count": Integer(kv_heads), "head_dimension": Integer(d),
            "causal": Boolean(True), "key_count": Integer(count)}


def test_a_store_is_written_read_copied_and_attended(ex):
    from magnetar_hip import Integer
    from magnetar_hip.executor import KV_MX4
    heads, kv_heads, d, cap = 8, 2, 80, 50
    for n in "kv":
        assert ex.write_zeroed_kv_store("m." + n, (cap, kv_heads * d), KV_MX4, d)
    rows = {n: cache_rows(i, 33, kv_heads, d) for i, n in enumerate("kv")}
    for n in "kv":
        ex.write_tensor("m.rows", rows[n])
        ex.execute(inv("kv-write", ["m." + n, "m.rows"], "m." + n, {"row_offset": Integer(0)}))
    held = {n: ref.round_trip(rows[n], kv_heads, d) for n in "kv"}
    want = np.zeros((cap, kv_heads * d), np.float32)
    want[:33] = held["k"]
    assert_bitexact(ex.read_tensor("m.k"), want)
    assert_bitexact(ex.read_tensor_values("m.k"), want)
    assert_bitexact(ex.read_tensor_rows("m.k", 30, 5), want[30:35])
    assert ex.resident_shape("m.k") == ((cap, kv_heads * d), 0)
    # Into another resource: a copy, the store unchanged.
    ex.write_tensor("m.rows", rows["v"][:2])
    ex.execute(inv("kv-write", ["m.k", "m.rows"], "m.k2", {"row_offset": Integer(1)}))
    assert_bitexact(ex.read_tensor("m.k"), want)
    want2 = want.copy()
    want2[1:3] = held["v"][:2]
    assert_bitexact(ex.read_tensor("m.k2"), want2)
    ex.copy_tensor("m.k2", "m.k3")
    assert_bitexact(ex.read_tensor("m.k3"), want2)
    q = np.random.default_rng(3).standard_normal((5, heads * d)).astype(np.float32)
    ex.write_tensor("m.q", q)
    ex.execute(inv("attention", ["m.q", "m.k", "m.v"], "m.o", attrs(heads, kv_heads, d, 33)))
    o, _, largest = ref.attention(q, held["k"], held["v"], heads, kv_heads, d)
    assert rel(ex.read_tensor("m.o"), o) <= ref.attention_tolerance(d, largest)


def test_refusals(ex):
    from magnetar_hip import Integer, KernelError
    from magnetar_hip.executor import KV_MX4, KV_TQ3
    for shape, d in (((4, 96), 64), ((4, 64), 0), ((4, 512), 512), ((4, 2, 32), 32)):
        with pytest.raises(KernelError) as err:
            ex.write_zeroed_kv_store("r.bad", shape, KV_MX4, d)
        assert err.value.code == "KernelShapeUnsupported", shape
    assert not ex.write_zeroed_kv_store("r.bad", (4, 64), KV_TQ3, 64)
    assert ex.write_zeroed_kv_store("r.k", (6, 64), KV_MX4, 32)
    assert ex.write_zeroed_kv_store("r.w", (6, 64), KV_MX4, 64)
    ex.write_tensor("r.f", np.ones((6, 64), np.float32))
    ex.write_tensor("r.a", np.ones((1, 6), np.float32))
    ex.write_tensor("r.b", np.ones((64, 3), np.float32))
    ex.write_tensor("r.q", np.ones((1, 64), np.float32))
    ex.write_tensor("r.rows", np.ones((3, 64), np.float32))
    cases = [
        (inv("kv-write", ["r.k", "r.rows"], "r.k", {"row_offset": Integer(4)}), "KernelShapeUnsupported"),
        (inv("kv-write", ["r.f", "r.k"], "r.f", {"row_offset": Integer(0)}), "KernelDTypeUnsupported"),
        (inv("add", ["r.k", "r.f"], "r.o"), "KernelDTypeUnsupported"),
        (inv("softmax", ["r.k"], "r.o"), "KernelDTypeUnsupported"),
        (inv("matmul", ["r.a", "r.k"], "r.o"), "KernelDTypeUnsupported"),
        (inv("matmul", ["r.k", "r.b"], "r.o"), "KernelDTypeUnsupported"),
        (inv("silu", ["r.k"], "r.o"), "KernelDTypeUnsupported"),
        (inv("rmsnorm", ["r.k"], "r.o"), "KernelDTypeUnsupported"),
        (inv("concat", ["r.f", "r.k"], "r.o"), "KernelDTypeUnsupported"),
        (inv("attention", ["r.q", "r.k", "r.f"], "r.o", attrs(2, 2, 32, 6)), "KernelLayoutUnsupported"),
        (inv("attention", ["r.q", "r.k", "r.w"], "r.o", attrs(2, 2, 32, 6)), "KernelLayoutUnsupported"),
        (inv("attention", ["r.k", "r.k", "r.k"], "r.o", attrs(2, 2, 32, 6)), "KernelDTypeUnsupported"),
    ]
    for invocation, code in cases:
        with pytest.raises(KernelError) as err:
            ex.execute(invocation)
        assert err.value.code == code, (invocation.kernel, err.value)
    assert not ex.read_tensor("r.k").any()


def test_an_output_of_the_same_size_does_not_become_a_store(ex):
    from magnetar_hip.executor import KV_MX4
    # 8 rows of 4 heads of 32: 4 * 2 * 68 bytes, rounded up to 768: 192 floats.
    assert ex.write_zeroed_kv_store("s.k", (8, 128), KV_MX4, 32)
    x = np.random.default_rng(1).standard_normal((3, 64)).astype(np.float32)
    ex.write_tensor("s.x", x)
    ex.execute(inv("add", ["s.x", "s.x"], "s.k"))
    assert_bitexact(ex.read_tensor("s.k"), x + x)


def test_a_captured_decode_step_over_4_bit_stores(ex):
    from magnetar_hip import Integer
    from magnetar_hip.executor import KV_MX4
    heads, kv_heads, d, cap, start = 8, 4, 64, 120, 70
    past = {n: cache_rows(i, start, kv_heads, d) for i, n in enumerate("kv")}
    for n in "kv":
        assert ex.write_zeroed_kv_store("c." + n, (cap, kv_heads * d), KV_MX4, d)
        ex.write_tensor("c.past", past[n])
        ex.execute(inv("kv-write", ["c." + n, "c.past"], "c." + n, {"row_offset": Integer(0)}))
    rng = np.random.default_rng(6)
    steps = [dict(q=rng.standard_normal((1, heads * d)).astype(np.float32), k=cache_rows(10 + t, 1, kv_heads, d),
                  v=cache_rows(40 + t, 1, kv_heads, d)) for t in range(8)]

    def write(t):
        for n in ("q", "k", "v"):
            ex.write_tensor("c.new_" + n, steps[t][n])

    def step(at):
        for n in "kv":
            ex.execute(inv("kv-write", ["c." + n, "c.new_" + n], "c." + n, {"row_offset": Integer(at)}))
        ex.execute(inv("attention", ["c.new_q", "c.k", "c.v"], "c.o", attrs(heads, kv_heads, d, at + 1)))

    write(0)
    step(start)  # eager: the workspace has its size
    ex.begin_step_capture(["key_count", "row_offset"])
    step(start)
    captured = ex.end_step_capture()
    for t in range(len(steps)):
        ex.replay_step(captured, t, {"c.new_" + n: steps[t][n] for n in ("q", "k", "v")})
        got = ex.read_tensor("c.o")
        held = [ref.round_trip(np.concatenate([past[n]] + [s[n] for s in steps[:t + 1]]), kv_heads, d) for n in "kv"]
        want, _, largest = ref.attention(steps[t]["q"], *held, heads, kv_heads, d)
        assert rel(got, want) <= ref.attention_tolerance(d, largest), t
    ex.release_step_capture(captured)
