"""Numbers that the bindings of rotary plans and windowed attention hand on, without a GPU:
what 32 bits do not hold is refused or limited, not wrapped."""
import ctypes as C
import types

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from ltx_amd import runtime as rt  # noqa: E402


@pytest.fixture
def calls(monkeypatch):
    """A context on the host whose library notes the calls that it gets: (name, arguments)."""
    seen = []

    class Lib:
        def __getattr__(self, name):
            def call(*args):
                seen.append((name, args))
                return 1
            return call
    monkeypatch.setattr(rt, "lib", lambda: Lib())
    ctx = rt.Context.__new__(rt.Context)
    ctx.handle, ctx.device = 1, -1
    ctx._graphs, ctx._caches, ctx._ropes = set(), set(), set()
    yield ctx, seen
    ctx._ropes.clear()
    ctx.handle = None


@pytest.mark.parametrize("window,sinks", [(5, 3), (2 ** 31 + 7, 2 ** 40), (-(2 ** 32) + 5, 0), (7, -(2 ** 32) + 5), (0, -1),
                                          (2 ** 32 + 5, 2 ** 32 + 1)])
def test_windows_beyond_32_bits(calls, window, sinks):
    """What the library is asked has the same sign, and more keys than a table holds stay more."""
    ctx, seen = calls
    kv = torch.zeros(1, dtype=torch.int32)
    batch = rt.KvBatch(kv, kv[None])
    cache = types.SimpleNamespace(handle=1, mode=rt.MODE_F16, ctx=ctx)
    q = torch.zeros(1, 128, dtype=torch.float16)
    ctx.kv_attention_window_workspace(cache, batch, 1, window, sinks)
    ctx.kv_attention_window(cache, batch, q, q, 1, window, sinks, stream=types.SimpleNamespace(cuda_stream=0))
    asked = [a[5:7] for n, a in seen if n.endswith("workspace")] + [a[7:9] for n, a in seen if n.endswith("window")]
    assert len(asked) == 2
    for pair in asked:
        for want, got in zip((window, sinks), pair):
            got = C.c_int32(got).value
            assert got == want if abs(want) <= 2 ** 30 else got >= 2 ** 30 if want > 0 else got < 0


def test_plans_beyond_32_bits(calls):
    ctx, seen = calls
    freq = np.ones((2, 64))
    for bad in [dict(axes=2 ** 32 + 1), dict(axes=-(2 ** 32) + 2), dict(axis=np.full((2, 64), 2 ** 32)),
                dict(axis=np.full((2, 64), 0.5)), dict(axis=np.full((2, 64), np.nan))]:
        with pytest.raises(rt.LtxError):
            ctx.rope(freq, **dict(dict(axes=2), **bad))
    assert not seen
    for axis in (None, np.ones((2, 64)), np.ones((2, 64), np.int64), torch.ones(2, 64, dtype=torch.int32)):
        ctx.rope(freq, axis=axis, axes=2).handle = None
    assert len(seen) == 4


def test_one_row_has_no_stride(calls):
    """A single row's stride says nothing (that of a transposed column is 1): its length is handed on."""
    ctx, seen = calls
    st = types.SimpleNamespace(cuda_stream=0)

    def row(n, dt=torch.float16):
        t = torch.zeros(n, 1, dtype=dt).T
        assert t.stride() == (1, 1)
        return t
    u8 = dict(dtype=torch.uint8)
    q, s = torch.zeros(1, 128, **u8), torch.zeros(2, 1, 4, **u8)
    ctx.mx4_quantise(row(256), q, s, stream=st)
    ctx.mx4_values(q, s, row(256), stream=st)
    plan = types.SimpleNamespace(handle=1, axes=1)
    ctx.qk_rope(plan, torch.zeros(1, 1, dtype=torch.float64), row(256), row(256), row(128), row(128), stream=st)
    kv = torch.zeros(1, dtype=torch.int32)
    batch = rt.KvBatch(kv, kv[None])
    cache = types.SimpleNamespace(handle=1, mode=rt.MODE_F16, ctx=ctx, kv_heads=2)
    ctx.kv_write(cache, batch, row(256), row(256), stream=st)
    ctx.kv_read(cache, batch, row(256), row(256), stream=st)
    ctx.kv_attention(cache, batch, row(256), row(256), 2, stream=st)
    ctx.kv_attention_window(cache, batch, row(256), row(256), 2, 9, stream=st)
    where = {"ltx_op_mx4_quantise": (2,), "ltx_op_mx4_values": (4,), "ltx_op_qk_rope": (5, 8, 11, 14),
             "ltx_op_kv_write": (4, 6), "ltx_op_kv_read": (4, 6), "ltx_op_kv_attention": (4, 9),
             "ltx_op_kv_attention_window": (4, 11)}
    assert {n for n, _ in seen} == set(where)
    for name, args in seen:
        widths = [128 if (name, i) in {("ltx_op_qk_rope", 11), ("ltx_op_qk_rope", 14)} else 256 for i in where[name]]
        assert [args[i] for i in where[name]] == widths, name
