"""The 4-bit key/value cache where it can go wrong beside the shapes of
test_gpu_kv.py: rows that see no key, scores beyond f32,
calls beside others."""
import math

import numpy as np
import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ltx_amd import runtime as rt  # noqa: E402
from ltx_amd import synth  # noqa: E402
from test_gpu_kv import HD, MODES, PAGE, Setup, any_tile, check, ints  # noqa: E402, F401


# ---- rows that see no key ---------------------------------------------------------

@pytest.mark.parametrize("mode", ["f16", "bf16"])
@pytest.mark.parametrize("keys", [[70, 9, 300, 1], [70, 9, 3000, 1]])
def test_padded_rows_with_stale_queries(any_tile, mode, keys):
    """Rows that see only pages outside the pool give zeros whatever their q holds, as
    rows of a sequence without keys do; a row with such a q that sees a key gives NaN."""
    ctx = any_tile
    say(f"kv padded, stale q {mode} {keys}")
    for rows in ([1, 1, 1, 1], [70, 3, 200, 1]):
        for bad in (math.nan, math.inf, -math.inf):
            s = Setup(ctx, mode, 2, rows, keys, seed=12)
            s.pages[1] = -1
            s.pages[2] = s.cache.pages
            s.pages[3] = -1
            q = s.queries(4)
            for causal in (True, False):
                want, tol = s.want(q, 4, causal, skip=lambda b, j: b > 0)
                stale = q.clone()
                stale[rows[0]:] = bad
                stale[rows[0] - 1, HD + 5] = bad  # the last row of the sequence that is there
                want[rows[0] - 1, HD:2 * HD] = math.nan
                check(s.attend(stale, 4, causal), want, tol)


@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_rows_before_the_first_page_of_the_pool(any_tile, mode):
    """Causal rows whose pages are outside the pool up to a later one: zeros, whatever
    their q holds; the rows behind attend to that page on."""
    ctx = any_tile
    say(f"kv first pages bad {mode}")
    for rows, keys in (([200, 150], [300, 1500]), ([300, 80], [320, 700])):
        s = Setup(ctx, mode, 2, rows, keys, seed=13)
        last = [(k - 1) // PAGE for k in keys]
        for b in range(2):
            s.pages[b, :last[b]] = -1
        q = s.queries(4)
        want, tol = s.want(q, 4, True, skip=lambda b, j: j // PAGE < last[b])
        for b in range(2):
            n, r0 = rows[b], s.row_start[b]
            blind = max(0, last[b] * PAGE - (keys[b] - n))  # rows at positions before the page
            assert 0 < blind < n
            assert (want[r0:r0 + blind] == 0).all() and (want[r0 + blind:r0 + n] != 0).any()
            q[r0:r0 + blind] = math.nan
        check(s.attend(q, 4, True), want, tol)


def test_scores_beyond_f32(any_tile):
    """bf16 q and k whose products leave f32: a key with a score of -inf among finite
    ones weighs nothing; a row all of whose scores are -inf, or with one of +inf, is NaN
    and not taken for one without keys."""
    ctx = any_tile
    say("kv scores beyond f32")
    for rows, keys in (([1, 1, 1, 2], [64, 1500, 900, 3]), ([150, 100, 70, 2], [200, 1500, 900, 3])):
        g = torch.Generator().manual_seed(6)
        total = sum(keys)
        k, v = torch.randn(2, total, 1, HD, generator=g)
        k[:, :, 0] = 0
        start = np.concatenate([[0], np.cumsum(keys)])
        huge = 2.0 ** 30
        lost = {(1, j) for j in range(0, keys[1], 3)}
        for b, j in lost:
            k[start[b] + j, 0] = 0
            k[start[b] + j, 0, 0] = -huge
        k[start[2]:start[3], 0, 0] = -huge   # all of the third sequence
        k[start[3], 0, 0] = huge             # one key of the fourth
        s = Setup(ctx, "bf16", 1, rows, keys, kv=(k, v))
        q = s.queries(2)
        q[:, 0] = q[:, HD] = 0
        s.kx[..., 0] = 0  # the finite scores: without the first dim (the lost keys are left out)
        want, tol = s.want(q, 2, False, skip=lambda b, j: (b, j) in lost)
        want[s.row_start[2]:] = math.nan
        q[:, 0] = q[:, HD] = 2.0 ** 100
        check(s.attend(q, 2, False), want, tol)


# ---- calls beside others ------------------------------------------------------------

def test_a_cache_made_inside_a_capture(block0):
    """A cache made (and another freed) while the same context's forward is being
    captured: the graph is whole, the cache holds zeros and takes rows."""
    say("kv cache made inside a capture")
    T, S = 250, 40
    inp = synth.make_inputs(T, S, seed=0, sigma=0.7)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    x = [dev(inp[n]) for n in ("x", "tstab", "tidx", "ctx", "pts2")] + [dev(t) for t in rt.rope_tables(inp["grid"])]
    y, want = torch.empty(2, T, 4096, device="cuda")
    c = rt.Context(0)
    try:
        w = c.upload(block0)
        gone = c.kv_cache(2, 3)
        c.forward(w, *x, want, mode=rt.MODE_F16)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="global"):
            c.forward(w, *x, y, mode=rt.MODE_F16)
            cache = c.kv_cache(2, 5)
            gone.free()
            y.add_(0)
        batch = rt.KvBatch(ints([130]), ints([[4, 0, 2]]), ints([0, 130]), 130)
        k, v = torch.full((2, 130, 2 * HD), 7.0, dtype=torch.float16, device="cuda")
        c.kv_read(cache, batch, k, v)
        assert (k == 0).all() and (v == 0).all()
        for _ in range(3):
            y.fill_(math.nan)
            graph.replay()
            c.kv_write(cache, batch, k + 1.5, v - 3)
            c.kv_read(cache, batch, k, v)
            torch.cuda.synchronize()
            assert torch.equal(y, want) and (k == 1.5).all() and (v == -3).all()
            k.zero_()
            v.zero_()
    finally:
        c.close()


def test_faults_beside_a_capture(ctx):
    """Read on another stream while one is captured; refused on the captured one, which
    goes on."""
    say("kv faults beside a capture")
    s = Setup(ctx, "f16", 2, [1, 3], [100, 70], seed=14)
    s.pages[1, 0] = -1
    q = s.queries(4).cuda()
    out, want = torch.zeros(2, s.total, 4 * HD, dtype=s.dt, device="cuda")
    work = torch.empty(max(16, ctx.kv_attention_workspace(s.cache, s.batch, 4)), dtype=torch.uint8, device="cuda")
    ctx.kv_attention(s.cache, s.batch, q, want, 4, work=work)
    once = s.cache.faults(reset=False)
    assert once > 0
    other, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, capture_error_mode="global"):
        ctx.kv_attention(s.cache, s.batch, q, out, 4, work=work)
        assert s.cache.faults(stream=other) == once
        with pytest.raises(rt.LtxError, match="captured"):
            s.cache.faults()
        out.mul_(2)
    for i in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want * 2)
        assert s.cache.faults() == once


def test_a_pool_that_does_not_fit(ctx):
    """Refused, and the next calls of this library and of torch know nothing of it."""
    say("kv pool beyond memory")
    before = torch.cuda.mem_get_info()[0]
    with pytest.raises(rt.LtxError):
        ctx.kv_cache(32, (1 << 25) - 1, rt.MODE_F16)  # 9.3 TB
    assert (torch.ones(1000, device="cuda") + 1).sum().item() == 2000
    c = ctx.kv_cache(32, 10, rt.MODE_F16)
    assert c.faults() == 0
    c.free()
    assert abs(torch.cuda.mem_get_info()[0] - before) < 64 << 20
