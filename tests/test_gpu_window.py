"""Attention with a sliding window and first keys over the 4-bit cache on the GPU against
the dense softmax in f64, with the bounds of test_gpu_kv.py (over the keys that a row sees);
and a streamed step of all its operators.

One term more: weights are 2^(score - maximum) in f32, where a maximum may be behind by 2^8,
and below 2^-126 they are zero (as are what products and sums of them fall below it). In f16
the term for weights below 2^-14 covers that; in bf16, whose weights have f32's exponents,
each key may lose 2^-126 of a sum of at least 2^-8: 2^-118 max |v| a key, and as much through
the denominator. It counts where values of v that are 0 meet the large weights."""
import math

import numpy as np
import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ltx_amd import runtime as rt  # noqa: E402
from test_gpu_kv import HD, MODES, PAGE, SHAPES, Setup, any_tile, check, ints  # noqa: E402, F401
from test_gpu_mx4 import streams  # noqa: E402


class Windowed(Setup):
    def seen(self, b, causal, window, sinks):
        n, L = self.rows[b], self.keys[b]
        end = (L - n + 1 + np.arange(n) if causal else np.full(n, L))[:, None]
        at = np.arange(L)[None]
        return (at < end) & ((at >= end - window) | (at < sinks))

    def want_window(self, q, heads, causal, window, sinks, gate=None, skip=None):
        """f64 attention and the bound, per value."""
        group = heads // self.kvh
        u = torch.finfo(self.dt).eps / 2
        out = np.zeros((self.total, heads, HD))
        tol = np.zeros_like(out)
        qx = q.double().cpu().numpy().reshape(self.total, heads, HD)
        for b, (n, L) in enumerate(zip(self.rows, self.keys)):
            r0, s0 = self.row_start[b], self.start[b]
            if n == 0 or L == 0:
                continue
            seen = self.seen(b, causal, window, sinks)
            if skip is not None:
                seen &= ~np.array([skip(b, j) for j in range(L)], bool)[None]
            for h in range(heads):
                k, v = self.kx[s0:s0 + L, h // group], self.vx[s0:s0 + L, h // group]
                x = qx[r0:r0 + n, h]
                bad = np.isnan(k).any(1) | np.isnan(v).any(1)
                k, v = np.where(bad[:, None], 0, k), np.where(bad[:, None], 0, v)
                s = np.where(seen, x @ k.T / math.sqrt(HD), -np.inf)
                top = s.max(1, keepdims=True)
                p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
                total = p.sum(1, keepdims=True)
                safe = np.where(total > 0, total, 1)
                o, A = p @ v / safe, p @ np.abs(v) / safe
                count = seen.sum(1, keepdims=True)
                size = (np.abs(x) @ np.abs(k).T).max(1, keepdims=True) / math.sqrt(HD) * 1.4427
                d = 128 * 2.0 ** -24 * size + 2.0 ** -22 * size + 2.0 ** -22
                t = (2 * u + 2 * d + 2 * count * 2.0 ** -24) * A + u * np.abs(o)
                if self.mode == "f16":
                    t = t + 2 * 2.0 ** -24 * count * np.abs(v).max() + 2.0 ** -24
                else:
                    t = t + 2 * 2.0 ** -118 * count * np.abs(v).max()
                o[(seen & bad[None]).any(1)] = np.nan
                gt = 1.0
                if gate is not None:
                    gt = (2 / (1 + np.exp(-gate.double().numpy()[r0:r0 + n, h])))[:, None]
                    t = t + 2.0 ** -20 * np.abs(o)
                out[r0:r0 + n, h], tol[r0:r0 + n, h] = o * gt, t * gt
        return out.reshape(self.total, -1), tol.reshape(self.total, -1)

    def look(self, q, heads, causal, window, sinks, gate=None, **kw):
        out = torch.full((self.total, heads * HD), 7.0, dtype=self.dt, device="cuda")
        self.ctx.kv_attention_window(self.cache, self.batch, q.cuda(), out, heads, window, sinks, causal=causal,
                                     glog=None if gate is None else gate.cuda(), **kw)
        return out

    def hide_pages(self, causal, window, sinks, fill):
        """The table with `fill` in every entry that no row sees a key of."""
        t = self.pages.clone()
        for b in range(len(self.keys)):
            seen = self.seen(b, causal, window, sinks).any(0) if self.rows[b] else np.zeros(self.keys[b], bool)
            for p in range(t.shape[1]):
                if not seen[PAGE * p:PAGE * p + PAGE].any():
                    t[b, p] = fill
        return t


WINDOWS = [(1, 0), (65, 4), (64, 0), (100, 64), (1, 1), (257, 3), (128, 130), (1000, 65), (63, 5000)]
_wanted = {}


def _cases():
    """Every shape with three of the windows, the types in turn."""
    for i, shape in enumerate(SHAPES):
        for j in range(3):
            yield (*shape, *WINDOWS[(2 * i + 7 * j) % len(WINDOWS)], ("f16", "bf16")[(i + j) % 2])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kvh,rows,keys,window,sinks,mode", list(_cases()))
def test_window(any_tile, mode, heads, kvh, rows, keys, window, sinks, causal):  # noqa: F811
    ctx = any_tile
    say(f"kv window {mode} heads={heads}/{kvh} rows={rows[:4]} keys={keys[:4]} window={window}+{sinks} causal={causal}")
    s = Windowed(ctx, mode, kvh, rows, keys, seed=sum(keys) + heads)
    gate = torch.randn(s.total, heads, generator=s.g) if heads != 32 else None
    q = s.queries(heads)
    case = (mode, heads, kvh, *rows, *keys, window, sinks, causal)
    if case not in _wanted:  # (one for all kernels)
        _wanted[case] = s.want_window(q, heads, causal, window, sinks, gate)
    want, tol = _wanted[case]
    got = s.look(q, heads, causal, window, sinks, gate)
    check(got, want, tol)
    # the caller's own workspace, and a table whose unseen entries hold anything: the same bits
    n = ctx.kv_attention_window_workspace(s.cache, s.batch, heads, window, sinks, causal=causal)
    work = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
    s.batch = rt.KvBatch(s.lens, s.hide_pages(causal, window, sinks, 0x7ffffff0), ints(s.row_start), s.total)
    assert torch.equal(got, s.look(q, heads, causal, window, sinks, gate, work=work))
    assert s.cache.faults() == 0


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kvh,rows,keys", [
    (32, 32, [300, 5, 130, 0, 515, 200, 1], [700, 0, 130, 9, 515, 258, 1]),
    (48, 12, [9, 260, 33, 128, 200, 64, 7, 96, 17], [90, 260, 1000, 128, 455, 64, 1200, 3, 400]),
    (64, 32, [3] * 65, [70 - i for i in range(65)]),
])
def test_more_than_a_round(any_tile, heads, kvh, rows, keys, causal):  # noqa: F811
    """More tiles than CUs."""
    ctx = any_tile
    say(f"kv window rounds heads={heads}/{kvh} rows={rows[:4]} keys={keys[:4]} causal={causal}")
    s = Windowed(ctx, "bf16", kvh, rows, keys, seed=sum(keys) + heads)
    q = s.queries(heads)
    for window, sinks in ((70, 2), (20, 64)):
        case = (heads, kvh, *rows, *keys, window, sinks, causal)
        if case not in _wanted:
            _wanted[case] = s.want_window(q, heads, causal, window, sinks)
        check(s.look(q, heads, causal, window, sinks), *_wanted[case])


@pytest.mark.parametrize("causal", [True, False])
def test_a_window_over_all_keys_is_the_call_without(any_tile, causal):  # noqa: F811
    ctx = any_tile
    say(f"kv window of all keys causal={causal}")
    s = Windowed(ctx, "f16", 2, [1, 33, 150], [700, 333, 300], seed=8)
    q = s.queries(4)
    want, tol = s.want(q, 4, causal)
    check(s.look(q, 4, causal, 700, 0), want, tol)  # narrower than the table, wider than any sequence
    whole = s.attend(q, 4, causal)
    for window, sinks in ((s.pages.shape[1] * PAGE, 5), (2 ** 31 - 1, 0), (2 ** 40, 2 ** 40)):
        assert torch.equal(s.look(q, 4, causal, window, sinks), whole)


@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_values_that_are_not_finite(any_tile, mode):  # noqa: F811
    """NaN for the rows that see them; no trace for those whose window or causal limit
    leaves them out, on pages that others of the tile read."""
    ctx = any_tile
    say(f"kv window not finite {mode}")
    g = torch.Generator().manual_seed(3)
    keys, rows = [400, 40, 70], [390, 3, 70]
    k, v = torch.randn(2, sum(keys), 2, HD, generator=g)
    k[120, 1, 5] = math.inf
    v[60, 0, 100] = -math.inf
    v[5, 1, 9] = math.inf
    v[300, 0, 3] = math.nan
    k[399, 0, 64] = math.nan
    v[400 + 40 + 69, 1, 0] = math.inf
    s = Windowed(ctx, mode, 2, rows, keys, kv=(k, v))
    for heads in (2, 8):
        q = s.queries(heads)
        for causal in (True, False):
            for window, sinks in ((30, 0), (30, 6), (100, 4), (90, 61)):
                want, tol = s.want_window(q, heads, causal, window, sinks)
                assert np.isnan(want).any() and not np.isnan(want).all()
                check(s.look(q, heads, causal, window, sinks), want, tol)


def test_rows_without_keys_and_bad_pages(any_tile):  # noqa: F811
    """Empty sequences, rows before the first position, windows whose pages are all outside
    the pool: zeros, whatever q holds. Bad pages among others are left out and counted."""
    ctx = any_tile
    say("kv window rows without keys")
    s = Windowed(ctx, "f16", 2, [1, 5, 0, 80, 2, 1], [0, 3, 10, 70, 0, 300], seed=9)
    q = s.queries(4)
    q[0] = math.nan
    for causal in (True, False):
        for window, sinks in ((1, 0), (40, 2)):
            want, tol = s.want_window(torch.nan_to_num(q), 4, causal, window, sinks)
            got = s.look(q, 4, causal, window, sinks)
            assert (got[0] == 0).all()
            check(got, want, tol)
    assert s.cache.faults() == 0
    for rows, keys in (([1, 2, 1], [300, 900, 200]), ([200, 70, 150], [300, 900, 200])):
        s = Windowed(ctx, "bf16", 2, rows, keys, seed=10)
        s.pages[0, 4] = -5
        s.pages[1, 13] = s.cache.pages
        s.pages[2] = -1
        q = s.queries(4)
        skip = lambda b, j: b == 2 or (b, j // PAGE) in ((0, 4), (1, 13))  # noqa: E731
        for causal in (True, False):
            want, tol = s.want_window(q, 4, causal, 130, 1, skip=skip)
            check(s.look(q, 4, causal, 130, 1), want, tol)
            assert s.cache.faults() > 0


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_queries_that_are_not_finite(any_tile, bad):  # noqa: F811
    """NaN for their row and head, others as without."""
    ctx = any_tile
    say(f"kv window query {bad}")
    s = Windowed(ctx, "f16", 2, [1, 100, 2], [1500, 300, 1], seed=4)
    q = s.queries(4)
    want, tol = s.want_window(q, 4, True, 90, 3)
    q[0, 3], q[50, HD + 127], q[101, 3] = bad, bad, bad  # (row 101: before the first position)
    got = s.look(q, 4, True, 90, 3)
    want[0, :HD] = want[50, HD:2 * HD] = math.nan
    assert (got[101] == 0).all()
    check(got, want, tol)


@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_peaked_scores(any_tile, mode):  # noqa: F811
    """Scores of hundreds: maxima that move, and sinks that outweigh every window."""
    ctx = any_tile
    say(f"kv window peaked {mode}")
    s = Windowed(ctx, mode, 2, [1, 33, 150], [700, 333, 300], seed=8)
    q = s.queries(4, 30.0)
    for window, sinks in ((100, 3), (20, 200)):
        want, tol = s.want_window(q, 4, True, window, sinks)
        check(s.look(q, 4, True, window, sinks), want, tol)


@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_wide_tables(any_tile, mode):  # noqa: F811
    """A table of 20,000 pages a sequence and a window of most of it: the kernels for large
    caches, with nothing behind the first few pages looked at."""
    ctx = any_tile
    say(f"kv window wide table {mode}")
    s = Windowed(ctx, mode, 2, [1, 1, 40], [700, 0, 1300], seed=29)
    wide = torch.full((3, 20000), 0x7ffffff0, dtype=torch.int32, device="cuda")
    wide[:, :s.pages.shape[1]] = s.pages
    wide[1] = -1
    s.batch = rt.KvBatch(s.lens, wide, ints(s.row_start), s.total)
    q = s.queries(4)
    for window, sinks in ((600_000, 0), (300, 600_000), (300, 20)):
        want, tol = s.want_window(q, 4, True, window, sinks)
        check(s.look(q, 4, True, window, sinks), want, tol)
    assert s.cache.faults() == 0


def test_pages_that_are_used_again(ctx):
    """A stream that keeps its sinks and a ring of pages: what slides out of the window gives
    its page to what comes. Captured once, replayed as the stream grows, against the rows that
    the ring has held."""
    say("kv window ring")
    kvh, heads, window, sinks, ring, steps = 2, 4, 150, 5, 4, 30
    cache = ctx.kv_cache(kvh, ring + 1, rt.MODE_F16)
    g = torch.Generator().manual_seed(1)
    table = ints([[0] + [1 + p % ring for p in range(40)]])
    new = 37
    lens, starts = ints([0]), ints([0, new])
    batch = rt.KvBatch(lens, table, starts, new)
    fused = torch.zeros(new, (heads + 2 * kvh) * HD, dtype=torch.float16, device="cuda")
    q, k, v = fused.split([heads * HD, kvh * HD, kvh * HD], 1)
    out = torch.zeros(new, heads * HD, dtype=torch.float16, device="cuda")
    work = torch.empty(max(16, ctx.kv_attention_window_workspace(cache, batch, heads, window, sinks)), dtype=torch.uint8,
                       device="cuda")

    def step():
        ctx.kv_write(cache, batch, k, v)
        ctx.kv_attention_window(cache, batch, q, out, heads, window, sinks, work=work)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    s = Windowed.__new__(Windowed)
    s.mode, s.dt, s.kvh, s.start, s.row_start, s.total, s.rows = "f16", torch.float16, kvh, [0], [0], new, [new]
    from test_gpu_kv import held
    rows = []
    for i in range(steps):
        x = torch.randn(new, fused.shape[1], generator=g).half()
        rows.append(x)
        fused.copy_(x)
        lens.fill_(new * (i + 1))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        every = torch.cat(rows)
        s.keys = [every.shape[0]]
        s.kx = held(every[:, heads * HD:(heads + kvh) * HD].reshape(-1, kvh, HD), "f16")
        s.vx = held(every[:, (heads + kvh) * HD:].reshape(-1, kvh, HD), "f16")
        check(out, *s.want_window(x[:, :heads * HD], heads, True, window, sinks))
        replayed = out.clone()
        out.zero_()
        step()
        assert torch.equal(out, replayed)
    assert cache.faults() == 0


def test_strides_streams_and_captures(ctx):
    """Slices of wider rows, another stream, a captured call without a workspace (it does
    not split), two calls at once with a workspace each: the bits of the call alone."""
    say("kv window strides and streams")
    s = Windowed(ctx, "f16", 2, [1, 90], [4000, 220], seed=11)
    wide = torch.randn(s.total, 3 * 4 * HD, generator=s.g).half()
    q, dev = wide[:, 4 * HD:8 * HD], wide.cuda()
    want, tol = s.want_window(q, 4, True, 2500, 3)
    out = torch.full((s.total, 5 * HD), 7.0, dtype=s.dt, device="cuda")
    args = (s.cache, s.batch, dev[:, 4 * HD:8 * HD])

    def call(o, **kw):
        ctx.kv_attention_window(*args, o[:, HD:], 4, 2500, 3, **kw)

    call(out)
    check(out[:, HD:], want, tol)
    assert (out[:, :HD] == 7).all()
    n = ctx.kv_attention_window_workspace(s.cache, s.batch, 4, 2500, 3)
    assert n > 0
    outs = [torch.zeros_like(out) for _ in range(4)]
    works = [torch.empty(n, dtype=torch.uint8, device="cuda") for _ in outs]
    sts = streams(len(outs))
    torch.cuda.synchronize()
    for _ in range(5):
        for o, w, st in zip(outs, works, sts):
            call(o, work=w, stream=st)
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o[:, HD:], out[:, HD:])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(outs[0])
    for _ in range(3):
        outs[0].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(outs[0][:, HD:], want, tol)


def test_refusals(ctx):
    say("kv window refusals")
    s = Windowed(ctx, "f16", 2, [1, 9], [40, 20], seed=1)
    q = s.queries(4).cuda()
    out = torch.full((s.total, 4 * HD), 7.0, dtype=s.dt, device="cuda")
    for heads, window, sinks, kw in [(4, 0, 0, {}), (4, -1, 0, {}), (4, 5, -1, {}), (3, 5, 0, {}),
                                     (4, 5, 0, dict(glog=torch.zeros(3, 4, device="cuda")))]:
        with pytest.raises(rt.LtxError):
            ctx.kv_attention_window(s.cache, s.batch, q, out, heads, window, sinks, **kw)
    with pytest.raises(rt.LtxError):
        ctx.kv_attention_window_workspace(s.cache, s.batch, 4, 0)
    with pytest.raises(rt.LtxError):
        ctx.kv_attention_window(s.cache, s.batch, q.float(), out, 4, 5)
    assert (out == 7).all()


# ---- a streamed step ----------------------------------------------------------------------

@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_a_streamed_step(ctx, mode):
    """Hidden state -> 4-bit q|k|v linear -> norm and positions -> cache -> windowed attention
    -> 4-bit out linear, captured once and replayed over two sequences' steps (a frame and a
    token): every operator's output within its own bound of f64 on what it was given."""
    from test_gpu_kv import held
    from test_gpu_mx4 import check as mx4_check, expected as mx4_expected, quantise, room
    from test_gpu_rope import check as rope_check, expected as rope_expected, plan
    say(f"streamed step {mode}")
    m, dt = MODES[mode]
    heads, kvh, D, window, sinks, pages = 8, 2, 512, 100, 10, 12
    rows = [70, 1]
    n = sum(rows)
    g = torch.Generator().manual_seed(7)
    p = plan(kvh, 3)
    rope = ctx.rope(*p, axes=3)
    width = (heads + 2 * kvh) * HD
    wqkv = quantise(ctx, (torch.randn(width, D, generator=g) * 0.04).cuda(), "f32")
    wout = quantise(ctx, (torch.randn(D, heads * HD, generator=g) * 0.03).cuda(), "f32")
    nq, nk = (1 + 0.2 * torch.randn(w * HD, generator=g).cuda() for w in (heads, kvh))
    cache = ctx.kv_cache(kvh, 2 * pages, m)
    lens, starts = ints([0, 0]), ints([0, rows[0], n])
    batch = rt.KvBatch(lens, ints(np.random.default_rng(0).permutation(2 * pages).reshape(2, pages)), starts, n)
    x = torch.zeros(n, D, dtype=dt, device="cuda")
    pos = torch.zeros(n, 3, dtype=torch.float64, device="cuda")
    held_x, held_o = room(n, D), room(n, heads * HD)
    fused = torch.zeros(n, width, dtype=dt, device="cuda")
    q, k, v = fused.split([heads * HD, kvh * HD, kvh * HD], 1)
    qo, ko = torch.zeros(n, heads * HD, dtype=dt, device="cuda"), torch.zeros(n, kvh * HD, dtype=dt, device="cuda")
    out, y = torch.zeros_like(qo), torch.zeros(n, D, device="cuda")
    work = torch.empty(max(16, ctx.kv_attention_window_workspace(cache, batch, heads, window, sinks)), dtype=torch.uint8,
                       device="cuda")

    def step():
        ctx.mx4_quantise(x, *held_x, mode=m)
        ctx.linear_mx4(*held_x, *wqkv, None, fused, mode=m)
        ctx.qk_rope(rope, pos, q, qo, k, ko, nq, nk, mode=m)
        ctx.kv_write(cache, batch, ko, v)
        ctx.kv_attention_window(cache, batch, qo, out, heads, window, sinks, work=work)
        ctx.mx4_quantise(out, *held_o, mode=m)
        ctx.linear_mx4(*held_o, *wout, None, y, mode=m)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    s = Windowed.__new__(Windowed)
    s.mode, s.dt, s.kvh, s.rows, s.row_start, s.total = mode, dt, kvh, rows, [0, rows[0]], n
    kept = [[], []], [[], []]
    for i in range(4):
        x.copy_(torch.randn(n, D, generator=g))
        pos.copy_(torch.rand(n, 3, generator=g, dtype=torch.float64) * 5 + 10 * i)
        lens.copy_(ints([r * (i + 1) for r in rows]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        mx4_check(fused, *mx4_expected(held_x, wqkv, None, False, dt))
        rope_check(qo, *rope_expected(p, pos, q, nq, 1e-6, dt))
        rope_check(ko, *rope_expected(p, pos, k, nk, 1e-6, dt))
        for b in range(2):
            at = slice(s.row_start[b], s.row_start[b] + rows[b])
            for which, t in enumerate((ko, v)):
                kept[which][b].append(held(t[at].reshape(rows[b], kvh, HD), mode))
        s.keys = [r * (i + 1) for r in rows]
        s.start = [0, s.keys[0]]
        s.kx, s.vx = (np.concatenate([np.concatenate(t) for t in both]) for both in kept)
        check(out, *s.want_window(qo, heads, True, window, sinks))
        mx4_check(y, *mx4_expected(held_o, wout, None, False, torch.float32))
        replayed = y.clone()
        step()
        assert torch.equal(y, replayed)
    assert cache.faults() == 0
