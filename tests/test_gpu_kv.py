"""The 4-bit key/value cache on the GPU against its definition in 64 bits.

What the cache holds of a row is exactly determined: written and read back it must
equal the oracle's bits. Attention is compared value by value with the dense softmax
in f64 over what the cache stands for. The bound counts the kernel's roundings, u =
eps / 2 of the 16-bit type:
  - the weights p are rounded to 16 bits, once, in numerator and denominator: 2 u A,
    A = sum p |v| / sum p; in f16 those below 2^-14 keep an absolute 2^-25, L of them
    against a sum of at least 1/2 (the largest weight is 1 to within 2^8 after a
    lazily moved maximum): 2^-24 L max|v|, and as much through the denominator;
  - a score q . k is a sum of 128 products in f32, 2^-24 * 128 sum |q k| at most, its
    exponent another 2^-22 of its size, exp2 2^-22: relative errors of p, so twice
    their largest, d, times A;
  - sums over keys in f32: 2^-24 times their number, L, times 2 A;
  - the output: u |o|.
"""
import math

import numpy as np
import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ltx_amd import runtime as rt  # noqa: E402

HD, PAGE = 128, 64
MODES = {"f16": (rt.MODE_F16, torch.float16), "bf16": (rt.MODE_BF16, torch.bfloat16)}
LIMITS = {"f16": (-23, 13), "bf16": (-125, 125)}
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def held(x, mode):
    """What the cache makes of x [..., 128] (any float tensor), in f64."""
    lo, hi = LIMITS[mode]
    g = x.double().cpu().numpy().reshape(-1, 32)
    out = np.empty_like(g)
    with np.errstate(invalid="ignore", divide="ignore"):
        top = np.abs(g).max(1, keepdims=True)
        m, e = np.frexp(top)
        e = np.clip(e - 3 + (m > 0.875), lo, hi)
        y = np.abs(g) / 2.0 ** e
        dist = np.abs(y[..., None] - GRID)
        i = dist.argmin(-1)
        tie = np.take_along_axis(dist, np.minimum(i + 1, 7)[..., None], -1)[..., 0] == dist.min(-1)
        i = np.where(tie & (i < 7) & (i % 2 == 1), i + 1, i)
        out = np.copysign(GRID[i], g) * 2.0 ** e
    out[~np.isfinite(g).all(1)] = np.nan
    return out.reshape(x.shape)


@pytest.fixture(params=["rule", "16", "128", "256"])
def any_tile(request, monkeypatch, ctx):
    """The context, and one for each kernel of the attention (columns of a tile)
    whatever the rule would take."""
    if request.param == "rule":
        yield ctx
        return
    monkeypatch.setenv("LTX_KV_TILE", request.param)
    c = rt.Context(0)
    yield c
    c.close()


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


class Setup:
    """A cache, ragged sequences on shuffled pages, and the f64 values of every key."""

    def __init__(self, ctx, mode, kv_heads, rows, keys, seed=0, extra=3, kv=None):
        self.ctx, self.mode, self.kvh, self.rows, self.keys = ctx, mode, kv_heads, rows, keys
        self.m, self.dt = MODES[mode]
        g = torch.Generator().manual_seed(seed + 101)
        self.g = g
        width = max(1, max(-(-k // PAGE) for k in keys))
        pool = len(keys) * width + extra
        self.pages = torch.randperm(pool, generator=g)[:len(keys) * width].reshape(len(keys), width).to(torch.int32).cuda()
        self.lens = ints(keys)
        self.cache = ctx.kv_cache(kv_heads, pool, self.m)
        total = sum(keys)
        if kv is None:
            k = torch.randn(total, kv_heads, HD, generator=g) * torch.exp(0.5 * torch.randn(kv_heads, HD, generator=g))
            v = torch.randn(total, kv_heads, HD, generator=g)
            kv = k, v
        self.k, self.v = (t.reshape(total, kv_heads * HD).to(self.dt) for t in kv)
        self.start = np.concatenate([[0], np.cumsum(keys)]).astype(int)
        if total:
            whole = rt.KvBatch(self.lens, self.pages, ints(self.start), total)
            ctx.kv_write(self.cache, whole, self.k.cuda(), self.v.cuda())
        self.kx, self.vx = (held(t.reshape(total, kv_heads, HD), mode) for t in (self.k, self.v))
        self.row_start = np.concatenate([[0], np.cumsum(rows)]).astype(int)
        self.total = int(self.row_start[-1])
        self.batch = rt.KvBatch(self.lens, self.pages, ints(self.row_start), self.total)

    def queries(self, heads, scale=1.0):
        return (torch.randn(self.total, heads * HD, generator=self.g) * scale).to(self.dt)

    def want(self, q, heads, causal, gate=None, skip=None):
        """f64 attention and the bound, per value. skip(b, key): keys left out."""
        group = heads // self.kvh
        u = torch.finfo(self.dt).eps / 2
        out = np.zeros((self.total, heads, HD))
        tol = np.zeros_like(out)
        qx = q.double().cpu().numpy().reshape(self.total, heads, HD)
        for b, (n, L) in enumerate(zip(self.rows, self.keys)):
            r0, s0 = self.row_start[b], self.start[b]
            pos = L - n + np.arange(n)
            seen = np.ones((n, L), bool) if not causal else np.arange(L)[None] <= pos[:, None]
            if skip is not None:
                seen &= ~np.array([skip(b, j) for j in range(L)], bool)[None]
            for h in range(heads):
                if n == 0 or L == 0:
                    continue
                k, v = self.kx[s0:s0 + L, h // group], self.vx[s0:s0 + L, h // group]
                x = qx[r0:r0 + n, h]
                bad = np.isnan(k).any(1) | np.isnan(v).any(1)
                k, v = np.where(bad[:, None], 0, k), np.where(bad[:, None], 0, v)
                s = np.where(seen, x @ k.T / math.sqrt(HD), -np.inf)
                top = s.max(1, keepdims=True)
                p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
                total = p.sum(1, keepdims=True)
                safe = np.where(total > 0, total, 1)
                o = p @ v / safe
                A = p @ np.abs(v) / safe
                size = (np.abs(x) @ np.abs(k).T).max(1, keepdims=True) / math.sqrt(HD) * 1.4427
                d = 128 * 2.0 ** -24 * size + 2.0 ** -22 * size + 2.0 ** -22
                t = (2 * u + 2 * d + 2 * L * 2.0 ** -24) * A + u * np.abs(o)
                if self.mode == "f16":
                    t = t + 2 * 2.0 ** -24 * L * np.abs(v).max() + 2.0 ** -24
                nan = (seen & bad[None]).any(1)
                o[nan] = np.nan
                gt = 1.0
                if gate is not None:
                    gt = (2 / (1 + np.exp(-gate.double().numpy()[r0:r0 + n, h])))[:, None]
                    t = t + 2.0 ** -20 * np.abs(o)
                out[r0:r0 + n, h] = o * gt
                tol[r0:r0 + n, h] = t * gt
        return out.reshape(self.total, -1), tol.reshape(self.total, -1)

    def attend(self, q, heads, causal, gate=None, **kw):
        out = torch.full((self.total, heads * HD), 7.0, dtype=self.dt, device="cuda")
        self.ctx.kv_attention(self.cache, self.batch, q.cuda(), out, heads, causal=causal,
                              glog=None if gate is None else gate.cuda(), **kw)
        return out


def check(got, want, tol):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(got - want)
    ok = np.isnan(want) | (off <= tol)
    assert ok.all(), (int((~ok).sum()), float(np.nanmax(off / np.maximum(tol, 1e-300))))


# ---- written and read back -------------------------------------------------------

def _edge_rows(mode):
    """Rows at the borders of the form: midpoints, the 7 2^e step, zeros, the
    largest and smallest numbers of the type."""
    dt = MODES[mode][1]
    ticks = torch.tensor([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7])
    rows = []
    for e in (-14, -3, 0, 5):
        for top in (4.0, 6.0, 7.0, 7.03125, 7.9375):
            g = torch.cat([ticks, -ticks]) * 2.0 ** e
            g = torch.where(g.abs() > top * 2.0 ** e, torch.zeros_like(g), g)
            g[31] = -top * 2.0 ** e
            rows.append(g.repeat(4))
    tiny, top = torch.finfo(dt).tiny, torch.finfo(dt).max
    sub = 2.0 ** -24 if mode == "f16" else 2.0 ** -133
    for a in (0.0, sub, 3 * sub, tiny, 5 * tiny, top, top * 0.87, top * 0.8, -top, 1.0):
        g = torch.zeros(32, dtype=torch.float64)
        g[3], g[17], g[30] = a, a * 0.25, -a * 0.4
        rows.append(g.repeat(4).float())
    return torch.stack(rows).to(dt)


@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_borders_of_the_form(ctx, mode):
    say(f"kv borders {mode}")
    x = _edge_rows(mode)
    n = x.shape[0]
    s = Setup(ctx, mode, 1, [n], [n], kv=(x[:, None], x.flip(0)[:, None]))
    k, v = torch.empty(n, HD, dtype=s.dt, device="cuda"), torch.empty(n, HD, dtype=s.dt, device="cuda")
    ctx.kv_read(s.cache, s.batch, k, v)
    assert np.array_equal(k.double().cpu().numpy(), s.kx.reshape(n, HD))
    assert np.array_equal(v.double().cpu().numpy(), s.vx.reshape(n, HD))


@pytest.mark.parametrize("mode,kvh,rows,keys", [
    ("f16", 1, [1], [1]),
    ("bf16", 8, [1, 1, 1], [64, 65, 1]),
    ("f16", 3, [5, 0, 63, 130], [9, 70, 63, 200]),
    ("bf16", 32, [17, 64], [100, 64]),
    ("f16", 8, [1] * 70, list(range(1, 71))),
    ("bf16", 2, [300], [1000]),
])
def test_write_and_read(ctx, mode, kvh, rows, keys):
    """New rows from slices of fused rows enter behind what was there; every row of
    the pool, before and after, holds what it should."""
    say(f"kv write/read {mode} heads={kvh} rows={rows[:4]} keys={keys[:4]}")
    s = Setup(ctx, mode, kvh, rows, keys, seed=len(keys) + kvh)
    w, n = kvh * HD, s.total
    fused = torch.randn(n + 2, 3 * w + 24, generator=s.g).to(s.dt)
    dev = fused.cuda()
    b = rt.KvBatch(s.lens, s.pages, ints(s.row_start), n + 2)  # two rows behind the last sequence
    ctx.kv_write(s.cache, b, dev[:, w:2 * w], dev[:, 2 * w:3 * w])
    for i, x in ((1, s.kx), (2, s.vx)):
        new = held(fused[:n, i * w:(i + 1) * w].reshape(n, kvh, HD), mode)
        for q, (c, L) in enumerate(zip(rows, keys)):
            x[s.start[q] + L - c:s.start[q] + L] = new[s.row_start[q]:s.row_start[q] + c]
    total = sum(keys)
    out = torch.full((2, total, w + 8), 9.0, dtype=s.dt, device="cuda")
    ctx.kv_read(s.cache, rt.KvBatch(s.lens, s.pages, ints(s.start), total), out[0, :, :w], out[1, :, :w])
    assert np.array_equal(out[0, :, :w].double().cpu().numpy(), s.kx.reshape(total, w))
    assert np.array_equal(out[1, :, :w].double().cpu().numpy(), s.vx.reshape(total, w))
    assert (out[:, :, w:] == 9).all()
    part = torch.full((2, n + 2, w), 9.0, dtype=s.dt, device="cuda")
    ctx.kv_read(s.cache, b, part[0], part[1])
    at = np.concatenate([np.arange(s.start[q] + L - c, s.start[q] + L) for q, (c, L) in enumerate(zip(rows, keys))])
    assert np.array_equal(part[0, :n].double().cpu().numpy(), s.kx.reshape(total, w)[at.astype(int)])
    assert (part[:, n:] == 9).all()  # rows behind the last sequence
    assert s.cache.faults() == 0


def test_rows_before_the_first_position_and_bad_pages(ctx):
    """More rows than keys: the first are left out. Page indices outside the pool:
    not followed, counted, read as zeros."""
    say("kv bad pages")
    s = Setup(ctx, "f16", 2, [6, 3], [4, 130], seed=5)
    x = torch.randn(9, 2 * HD, generator=s.g).half()
    s.pages[1, 2] = -1
    s.pages[0, 1:] = 1 << 30  # not reached
    ctx.kv_write(s.cache, s.batch, x.cuda(), x.cuda())
    assert s.cache.faults() == 2  # positions 128 and 129 of the second sequence
    k, v = torch.full((2, 9, 2 * HD), 9.0, dtype=s.dt, device="cuda")
    ctx.kv_read(s.cache, s.batch, k, v)
    assert s.cache.faults(reset=False) == 2 and s.cache.faults() == 2 and s.cache.faults() == 0
    want = held(x.reshape(9, 2, HD), "f16").reshape(9, -1)
    want[:2] = 0  # positions -2 and -1
    want[7:] = 0
    assert np.array_equal(k.double().cpu().numpy(), want) and np.array_equal(v.double().cpu().numpy(), want)


@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_values_that_are_not_finite(any_tile, mode):
    """Read back as NaN of their group; NaN for the rows that see them, and no trace
    for those that do not (causal rows before them, keys past the end, other heads)."""
    ctx = any_tile
    say(f"kv not finite {mode}")
    g = torch.Generator().manual_seed(3)
    keys, rows = [150, 40, 70], [140, 3, 70]
    k, v = torch.randn(2, sum(keys), 2, HD, generator=g)
    k[120, 1, 5] = math.inf
    v[60, 0, 100] = -math.inf
    v[130, 0, 3] = math.nan
    k[149, 0, 64] = math.nan
    v[150 + 40 + 69, 1, 0] = math.inf
    s = Setup(ctx, mode, 2, rows, keys, kv=(k, v))
    for heads in (2, 8):
        for causal in (True, False):
            q = s.queries(heads)
            want, tol = s.want(q, heads, causal)
            assert np.isnan(want).any() and not np.isnan(want).all()
            check(s.attend(q, heads, causal), want, tol)
    # the last keys leave (shorter sequences): stale rows of their pages stay unseen
    s.lens.copy_(ints([119, 40, 69]))
    s.keys = [119, 40, 69]
    s.rows, s.row_start = [60, 3, 69], np.array([0, 60, 63, 132])
    s.total = 132
    s.batch = rt.KvBatch(s.lens, s.pages, ints(s.row_start), s.total)
    for causal in (True, False):
        q = s.queries(8)
        want, tol = s.want(q, 8, causal)
        check(s.attend(q, 8, causal), want, tol)
    total = sum(keys)
    s.lens.copy_(ints(keys))
    kk, vv = torch.empty(2, total, 2 * HD, dtype=s.dt, device="cuda")
    ctx.kv_read(s.cache, rt.KvBatch(s.lens, s.pages, ints(s.start), total), kk, vv)
    assert np.array_equal(kk.double().cpu().numpy(), s.kx.reshape(total, -1), equal_nan=True)
    assert np.array_equal(vv.double().cpu().numpy(), s.vx.reshape(total, -1), equal_nan=True)


# ---- attention -------------------------------------------------------------------

SHAPES = [
    # heads, kv_heads, rows, keys
    (1, 1, [1], [1]),
    (32, 32, [1], [1000]),
    (32, 8, [1, 1, 1, 1], [1, 63, 64, 65]),
    (8, 2, [1] * 70, [3 * i + 1 for i in range(70)]),
    (6, 2, [3, 1, 7], [300, 1, 64]),          # three query heads a cached head: columns end inside a row
    (20, 1, [2, 1], [500, 129]),              # more query heads than a tile has columns
    (32, 4, [1, 5, 40], [2970, 130, 40]),
    (4, 4, [100], [100]),
    (4, 4, [257, 64, 1], [257, 600, 90]),
    (8, 2, [200, 3], [1500, 5]),
    (2, 1, [1], [9000]),
    (4, 2, [129], [4099]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("mode", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kvh,rows,keys", SHAPES)
def test_attention(any_tile, mode, heads, kvh, rows, keys, causal):
    ctx = any_tile
    say(f"kv attention {mode} heads={heads}/{kvh} rows={rows[:4]} keys={keys[:4]} causal={causal}")
    s = Setup(ctx, mode, kvh, rows, keys, seed=sum(keys) + heads)
    gate = torch.randn(s.total, heads, generator=s.g) if heads != 32 else None
    q = s.queries(heads)
    want, tol = s.want(q, heads, causal, gate)
    got = s.attend(q, heads, causal, gate)
    check(got, want, tol)
    # the caller's own workspace: the same bits
    n = ctx.kv_attention_workspace(s.cache, s.batch, heads)
    work = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(got, s.attend(q, heads, causal, gate, work=work))
    assert s.cache.faults() == 0


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kvh,rows,keys", [
    (32, 32, [300, 5, 130, 0, 515, 200, 1], [700, 0, 130, 9, 515, 258, 1]),
    (48, 12, [9, 260, 33, 128, 200, 64, 7, 96, 17], [90, 260, 1000, 128, 455, 64, 1200, 3, 400]),
    (64, 32, [5] * 64, [2 * i + 3 for i in range(64)]),
    (64, 32, [5] * 65, [131 - 2 * i for i in range(65)]),
])
def test_attention_of_more_than_a_round(any_tile, heads, kvh, rows, keys, causal):
    """More tiles than CUs."""
    ctx = any_tile
    say(f"kv attention rounds heads={heads}/{kvh} rows={rows[:4]} keys={keys[:4]} causal={causal}")
    s = Setup(ctx, "bf16", kvh, rows, keys, seed=sum(keys) + heads)
    q = s.queries(heads)
    want, tol = s.want(q, heads, causal)
    check(s.attend(q, heads, causal), want, tol)
    assert s.cache.faults() == 0


@pytest.mark.parametrize("mode", ["f16", "bf16"])
@pytest.mark.parametrize("scale", [30.0, 0.01])
def test_attention_peaked_and_flat(any_tile, mode, scale):
    """Scores of hundreds, whose maximum moves from page to page, and near zero."""
    ctx = any_tile
    say(f"kv attention {mode} q scale {scale}")
    s = Setup(ctx, mode, 2, [1, 33, 150], [700, 333, 300], seed=8)
    q = s.queries(4, scale)
    want, tol = s.want(q, 4, True)
    check(s.attend(q, 4, True), want, tol)


def test_attention_rows_without_keys(any_tile):
    """Empty sequences and rows before the first position give zeros; rows behind
    the last sequence stay."""
    ctx = any_tile
    say("kv attention rows without keys")
    s = Setup(ctx, "f16", 2, [1, 5, 0, 80, 2], [0, 3, 10, 70, 0], seed=9)
    q = s.queries(4)
    for causal in (True, False):
        want, tol = s.want(q, 4, causal)
        check(s.attend(q, 4, causal), want, tol)
    more = torch.cat([q, torch.full((3, 4 * HD), math.nan, dtype=s.dt)]).cuda()
    out = torch.full((s.total + 3, 4 * HD), 7.0, dtype=s.dt, device="cuda")
    b = rt.KvBatch(s.lens, s.pages, ints(s.row_start), s.total + 3)
    ctx.kv_attention(s.cache, b, more, out, 4, causal=False)
    check(out[:s.total], want, tol)
    assert (out[s.total:] == 7).all()


def test_attention_leaves_bad_pages_out(any_tile):
    ctx = any_tile
    say("kv attention bad pages")
    for rows, keys in (([1, 2], [300, 900]), ([200, 70], [300, 900])):
        s = Setup(ctx, "bf16", 2, rows, keys, seed=10)
        s.pages[0, 2] = -5
        s.pages[1, 0] = s.cache.pages
        s.pages[1, 14] = 0x7fffffff
        q = s.queries(4)
        skip = lambda b, j: (b, j // PAGE) in ((0, 2), (1, 0), (1, 14))  # noqa: E731
        want, tol = s.want(q, 4, False, skip=skip)
        check(s.attend(q, 4, False), want, tol)
        assert s.cache.faults() > 0


@pytest.mark.parametrize("keys", [[70, 9, 300, 1], [70, 9, 3000, 1]])
def test_attention_of_rows_whose_pages_are_all_bad(any_tile, keys):
    """A padded batch: rows that see only pages outside the pool give zeros."""
    ctx = any_tile
    say(f"kv attention padded {keys}")
    for rows in ([1, 1, 1, 1], [70, 3, 200, 1]):
        s = Setup(ctx, "f16", 2, rows, keys, seed=12)
        s.pages[1] = -1
        s.pages[2] = s.cache.pages
        s.pages[3] = -1
        q = s.queries(4)
        for causal in (True, False):
            want, tol = s.want(q, 4, causal, skip=lambda b, j: b > 0)
            assert (want[rows[0]:] == 0).all()
            check(s.attend(q, 4, causal), want, tol)
            assert s.cache.faults() > 0


@pytest.mark.parametrize("mode", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_queries_that_are_not_finite(any_tile, mode, bad):
    """NaN for their row and head, also where every score is -inf; zeros where no key
    is seen; every other row and head within the bounds that it has without (not the
    same bits: a column's weights are formed with a maximum that is behind by up to 2^8,
    moved for the columns of a wave together, and the bound holds for any such one)."""
    ctx = any_tile
    say(f"kv attention query {bad} {mode}")
    g = torch.Generator().manual_seed(4)
    for rows, keys in (([1, 1, 2], [5, 1500, 1]), ([100, 200, 2], [120, 1500, 1])):
        k, v = torch.randn(2, sum(keys), 2, HD, generator=g)
        k[:, 0, 3] = 2.0 + k[:, 0, 3].abs()
        s = Setup(ctx, mode, 2, rows, keys, kv=(k, v))
        q = s.queries(4)
        want, tol = s.want(q, 4, True)
        last = s.total - 2  # before the first position: sees nothing
        for row, dim in ((0, 3), (rows[0], HD + 127), (last, 3)):
            q[row, dim] = bad
        got = s.attend(q, 4, True)
        for row, head in ((0, 0), (rows[0], 1)):
            want[row, head * HD:(head + 1) * HD] = math.nan
        assert (got[last] == 0).all()
        check(got, want, tol)


@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_tables_wider_than_what_is_in_use(any_tile, mode):
    """A table of 10,000 pages a sequence, nothing behind the first few looked at: the
    kernel of large caches, and splits over few real pages."""
    ctx = any_tile
    say(f"kv wide table {mode}")
    s = Setup(ctx, mode, 2, [1, 1, 40], [700, 0, 1300], seed=29)
    wide = torch.full((3, 10000), 0x7ffffff0, dtype=torch.int32, device="cuda")
    wide[:, :s.pages.shape[1]] = s.pages
    wide[1] = -1
    s.pages = wide
    s.batch = rt.KvBatch(s.lens, wide, ints(s.row_start), s.total)
    assert 3 * 10000 * 2 * 8704 > 384 << 20
    for causal in (True, False):
        q = s.queries(4)
        want, tol = s.want(q, 4, causal)
        check(s.attend(q, 4, causal), want, tol)
    assert s.cache.faults() == 0


def test_strides_streams_and_repeats(ctx):
    """q and out as slices of wider rows, on another stream; equal bits every time."""
    say("kv attention strides and streams")
    s = Setup(ctx, "f16", 2, [1, 90], [400, 120], seed=11)
    wide = torch.randn(s.total, 3 * 4 * HD, generator=s.g).half()
    q = wide[:, 4 * HD:8 * HD]
    want, tol = s.want(q, 4, True)
    dev = wide.cuda()
    outs = []
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for st in (None, stream, stream):
        out = torch.full((s.total, 5 * HD), 7.0, dtype=s.dt, device="cuda")
        torch.cuda.synchronize()
        ctx.kv_attention(s.cache, s.batch, dev[:, 4 * HD:8 * HD], out[:, :4 * HD], 4, stream=st)
        torch.cuda.synchronize()
        assert (out[:, 4 * HD:] == 7).all()
        outs.append(out)
    check(outs[0][:, :4 * HD], want, tol)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_places_behind_32_bits(ctx):
    """Pages whose blocks lie more than 4 GiB into the pool."""
    say("kv 64-bit places")
    kvh, pool = 32, 16000
    assert pool * kvh * 8704 > 1 << 32
    cache = ctx.kv_cache(kvh, pool, rt.MODE_BF16)
    s = Setup(ctx, "bf16", kvh, [2], [130], seed=12)
    pages = ints([[15999, 7, 15998]])
    b = rt.KvBatch(s.lens, pages, ints([0, 130]), 130)
    ctx.kv_write(cache, b, s.k.cuda(), s.v.cuda())
    k, v = torch.empty(2, 130, kvh * HD, dtype=s.dt, device="cuda")
    ctx.kv_read(cache, b, k, v)
    assert np.array_equal(k.double().cpu().numpy(), s.kx.reshape(130, -1))
    assert np.array_equal(v.double().cpu().numpy(), s.vx.reshape(130, -1))
    q = s.queries(32)
    want, tol = s.want(q, 32, True)
    out = torch.empty(2, 32 * HD, dtype=s.dt, device="cuda")
    ctx.kv_attention(cache, rt.KvBatch(s.lens, pages, ints([0, 2]), 2), q.cuda(), out, 32)
    check(out, want, tol)
    cache.free()


def test_captured_steps_follow_the_lengths(any_tile):
    """A step (write, attention) of two contexts' worth of graphs, captured with their
    own workspaces and replayed together while the lengths grow: each replay equals
    the eager result."""
    ctx = any_tile
    say("kv graphs")
    runs = []
    for i, mode in enumerate(("f16", "bf16")):
        s = Setup(ctx, mode, 2, [1, 1, 1], [700, 130, 65], seed=20 + i, extra=9)
        s.lens.copy_(ints([690, 120, 60]))
        w, heads = 2 * HD, 8
        x = dict(q=torch.zeros(3, heads * HD, dtype=s.dt, device="cuda"), k=torch.zeros(3, w, dtype=s.dt, device="cuda"),
                 v=torch.zeros(3, w, dtype=s.dt, device="cuda"), out=torch.zeros(3, heads * HD, dtype=s.dt, device="cuda"))
        work = torch.empty(ctx.kv_attention_workspace(s.cache, s.batch, heads), dtype=torch.uint8, device="cuda")

        def step(out, s=s, x=x, work=work, heads=heads):
            ctx.kv_write(s.cache, s.batch, x["k"], x["v"])
            ctx.kv_attention(s.cache, s.batch, x["q"], out, heads, work=work)

        step(x["out"])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(x["out"])
        runs.append((s, x, graph, step, torch.cuda.Stream()))
    for it in range(5):
        for s, x, *_ in runs:
            for t in ("q", "k", "v"):
                x[t].copy_(torch.randn(x[t].shape, generator=s.g))
            s.lens.add_(1)
            x["out"].fill_(5)
        torch.cuda.synchronize()
        for s, x, graph, step, stream in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s, x, graph, step, stream in runs:
            eager = torch.empty_like(x["out"])
            step(eager)
            assert torch.equal(eager, x["out"]) and torch.isfinite(eager).all()


def test_captured_without_a_workspace(any_tile):
    """A captured call that is given no workspace does not split: within the same
    bounds, at every replay."""
    ctx = any_tile
    say("kv graph without workspace")
    s = Setup(ctx, "f16", 2, [1, 3, 130], [1500, 64, 2000], seed=25)
    q = s.queries(4)
    want, tol = s.want(q, 4, True)
    dev, out = q.cuda(), torch.zeros(s.total, 4 * HD, dtype=s.dt, device="cuda")
    ctx.kv_attention(s.cache, s.batch, dev, out, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.kv_attention(s.cache, s.batch, dev, out, 4)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        check(out, want, tol)
        eager = torch.zeros_like(out)
        ctx.kv_attention(s.cache, s.batch, dev, eager, 4)
        check(eager, want, tol)


def test_two_calls_at_once(any_tile):
    """Two eager calls on two streams, each with its own workspace, and two that share
    the context's scratch: the bits of the calls one by one."""
    ctx = any_tile
    say("kv two streams")
    a = Setup(ctx, "f16", 2, [1, 1], [3000, 1200], seed=26)
    b = Setup(ctx, "bf16", 4, [40], [2500], seed=27)
    torch.cuda.synchronize()
    cases = [(s, s.queries(8).cuda()) for s in (a, b)]
    alone = [s.attend(q, 8, True) for s, q in cases]
    works = [torch.empty(max(16, ctx.kv_attention_workspace(s.cache, s.batch, 8)), dtype=torch.uint8, device="cuda")
             for s, _ in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for shared in (False, True):
        for _ in range(5):
            outs = [torch.zeros_like(o) for o in alone]
            torch.cuda.synchronize()
            for (s, q), out, work, st in zip(cases, outs, works, streams):
                ctx.kv_attention(s.cache, s.batch, q, out, 8, work=None if shared else work, stream=st)
            torch.cuda.synchronize()
            for out, ref in zip(outs, alone):
                assert torch.equal(out, ref)


def test_rows_of_no_sequence(any_tile):
    """Rows before the first sequence's and between row_start's ends are of none: out
    and what is read back stay as they were, the cache too."""
    ctx = any_tile
    say("kv rows of no sequence")
    s = Setup(ctx, "bf16", 2, [2, 70], [100, 300], seed=28)
    q = s.queries(4)
    want, tol = s.want(q, 4, True)
    shift = 5
    wide = torch.full((s.total + shift + 2, 4 * HD), math.nan, dtype=s.dt, device="cuda")
    wide[shift:shift + s.total] = q.cuda()
    out = torch.full_like(wide, 7.0)
    b = rt.KvBatch(s.lens, s.pages, ints(s.row_start + shift), wide.shape[0])
    ctx.kv_attention(s.cache, b, wide, out, 4)
    check(out[shift:shift + s.total], want, tol)
    assert (out[:shift] == 7).all() and (out[shift + s.total:] == 7).all()
    k = torch.full((2, wide.shape[0], 2 * HD), 9.0, dtype=s.dt, device="cuda")
    ctx.kv_read(s.cache, b, k[0], k[1])
    assert (k[:, :shift] == 9).all() and (k[:, shift + s.total:] == 9).all() and (k[:, shift:shift + s.total] != 9).all()
    k[:, :shift] = math.nan
    k[:, shift + s.total:] = math.nan
    ctx.kv_write(s.cache, b, k[0], k[1])  # what is held already, and NaN in rows of none
    check(s.attend(q, 4, True), want, tol)


@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_a_decoder_step(ctx, mode):
    """The operators as one layer's step uses them: the 4-bit q|k|v projection, its k
    and v into the cache as they lie, attention, the 4-bit out projection; 20 steps of
    three sequences from a prompt each, against f64 with the roundings between the
    operators (16-bit activations) made alike. Bound: the operators' own, carried
    through the out projection (its row sums of |w|) and its f32 sum, plus the output's
    rounding."""
    say(f"decoder step {mode}")
    heads, kvh, D = 4, 2, 256
    m, dt = MODES[mode]
    s = Setup(ctx, mode, kvh, [1, 1, 1], [100, 20, 64], seed=30)
    g = s.g
    N = (heads + 2 * kvh) * HD

    def weights(n, k):
        w = torch.randint(-8, 8, (n, k), generator=g)
        sc = (torch.rand(n, k // 128, generator=g) * 0.02 + 0.002).float()
        b = (w & 15).to(torch.uint8)
        return (b[:, 0::2] | (b[:, 1::2] << 4)).contiguous(), sc, w.double().numpy() * sc.double().repeat_interleave(128, 1).numpy()

    q1, s1, w1 = weights(N, D)
    q2, s2, w2 = weights(D, heads * HD)
    dq1, ds1, dq2, ds2 = q1.cuda(), s1.cuda(), q2.cuda(), s2.cuda()
    fused = torch.empty(3, N, dtype=dt, device="cuda")
    att = torch.empty(3, heads * HD, dtype=dt, device="cuda")
    y = torch.empty(3, D, dtype=torch.float32, device="cuda")
    keys = list(s.keys)
    kx = [s.kx[s.start[b]:s.start[b + 1]] for b in range(3)]
    vx = [s.vx[s.start[b]:s.start[b + 1]] for b in range(3)]
    for it in range(20):
        keys = [min(k + 1, 108) for k in keys]  # the longest overwrites its last token in the end
        lens = ints(keys)
        b = rt.KvBatch(lens, s.pages)
        x = torch.randn(3, D, generator=g).to(dt)
        ctx.linear_q4(x.cuda(), dq1, ds1, None, fused, mode=m)
        k, v = fused[:, heads * HD:(heads + kvh) * HD], fused[:, (heads + kvh) * HD:]
        ctx.kv_write(s.cache, b, k, v)
        ctx.kv_attention(s.cache, b, fused[:, :heads * HD], att, heads)
        ctx.linear_q4(att, dq2, ds2, None, y, mode=m)
        f = fused.double().cpu().numpy()
        exact = x.double().numpy() @ w1.T
        u = torch.finfo(dt).eps / 2
        bound = u * np.abs(exact) + 2.0 ** -18 * (np.abs(x.double().numpy()) @ np.abs(w1).T) + 2.0 ** -24
        assert (np.abs(f - exact) <= bound).all()
        t = Setup.__new__(Setup)
        t.mode, t.dt, t.kvh, t.rows, t.keys, t.total = mode, dt, kvh, [1, 1, 1], keys, 3
        t.row_start = np.arange(4)
        for i in range(3):
            nk, nv = held(k[i].cpu().reshape(1, kvh, HD), mode), held(v[i].cpu().reshape(1, kvh, HD), mode)
            kx[i] = np.concatenate([kx[i], nk])[:keys[i]] if len(kx[i]) < keys[i] else np.concatenate([kx[i][:-1], nk])
            vx[i] = np.concatenate([vx[i], nv])[:keys[i]] if len(vx[i]) < keys[i] else np.concatenate([vx[i][:-1], nv])
        t.kx, t.vx = np.concatenate(kx), np.concatenate(vx)
        t.start = np.concatenate([[0], np.cumsum(keys)])
        want, tol = t.want(fused[:, :heads * HD], heads, True)
        check(att, want, tol)
        yw, yt = want @ w2.T, tol @ np.abs(w2).T + 2.0 ** -18 * (np.abs(want) @ np.abs(w2).T)
        assert (np.abs(y.double().cpu().numpy() - yw) <= yt).all()
    assert s.cache.faults() == 0


def test_refusals(ctx):
    """What the host sees is refused with its reason, and nothing runs."""
    say("kv refusals")
    s = Setup(ctx, "f16", 2, [1], [10], seed=40)
    q = s.queries(4).cuda()
    out = torch.full_like(q, 7)
    for heads, bad in ((3, q[:, :384]), (0, q[:, :0])):
        with pytest.raises(rt.LtxError, match="heads"):
            ctx.kv_attention(s.cache, s.batch, bad, bad, heads)
    with pytest.raises(rt.LtxError, match="work"):
        ctx.kv_attention(s.cache, rt.KvBatch(s.lens, s.pages.repeat(1, 40)), q, out, 4,
                         work=torch.empty(16, dtype=torch.uint8, device="cuda"))
    with pytest.raises(rt.LtxError, match="16-bit mode"):
        ctx.kv_cache(2, 4, rt.MODE_F32)
    with pytest.raises(rt.LtxError, match="type"):
        ctx.kv_attention(s.cache, s.batch, q.bfloat16(), out, 4)
    assert (out == 7).all()
