"""The 4-bit key/value cache where it can go wrong beside the shapes of
test_gpu_kv.py: rows that see no key, scores beyond f32, subnormal values, long
sequences whose answer depends on every page, and calls beside others."""
import math

import numpy as np
import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ltx_amd import runtime as rt  # noqa: E402
from ltx_amd import synth  # noqa: E402
from test_gpu_kv import HD, MODES, PAGE, Setup, any_tile, check, held, ints  # noqa: E402, F401


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


# ---- the form ---------------------------------------------------------------------

@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_subnormal_values(ctx, mode):
    """Groups of values below the type's smallest normal number, rounded as any other."""
    say(f"kv subnormal {mode}")
    dt = MODES[mode][1]
    step = 2.0 ** -24 if mode == "f16" else 2.0 ** -133
    per = 1024 if mode == "f16" else 128  # subnormals are 0 .. per - 1 times step
    g = torch.Generator().manual_seed(2)
    rows = []
    for top in (1, 2, 3, 5, per // 4, per // 2, per - 1, 2 * per, 8 * per):
        x = torch.randint(-top, top + 1, (HD,), generator=g).double()
        x[::32] = top
        rows.append(x * step)
    rows.append(torch.arange(HD).double() * (per // HD) * step)
    x = torch.stack(rows).to(dt)  # exact
    assert torch.equal(x[:8].double(), torch.stack(rows[:8]))
    n = x.shape[0]
    s = Setup(ctx, mode, 1, [n], [n], kv=(x[:, None], x.flip(0)[:, None]))
    k, v = torch.empty(2, n, HD, dtype=s.dt, device="cuda")
    ctx.kv_read(s.cache, s.batch, k, v)
    assert np.array_equal(k.double().cpu().numpy(), s.kx.reshape(n, HD))
    assert np.array_equal(v.double().cpu().numpy(), s.vx.reshape(n, HD))
    assert (s.kx != 0).any()


# ---- long sequences: every page counts ----------------------------------------------

def _unsplit(s, q, heads, causal):
    """A captured call without a workspace: no split."""
    dev, out = q.cuda(), torch.full((s.total, heads * HD), 7.0, dtype=s.dt, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.ctx.kv_attention(s.cache, s.batch, dev, out, heads, causal=causal)
    for _ in range(2):
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("mode,rows,keys", [
    ("f16", [1], [9000]), ("bf16", [1], [28672]), ("f16", [1, 2], [28671, 500]), ("f16", [70], [9001]),
    ("bf16", [300], [28600]), ("f16", [1, 1, 90], [17, 28672, 12345]),
])
def test_every_page_of_equal_scores(any_tile, mode, rows, keys, causal):
    """q = 0: every weight is 1. The keys of page p have one value, 2^(p / 128) in dim p %
    128, so a page that is left out, taken twice or in the wrong place changes a dim of the
    output by a fifteenth at least. All sums are whole numbers below 2^24, exact in f32; a
    division, a product (2^-24 and 2^-23) and the output's rounding remain."""
    ctx = any_tile
    say(f"kv every page {mode} {rows} {keys} causal={causal}")
    total = sum(keys)
    v = torch.zeros(total, 1, HD)
    at = np.concatenate([np.arange(k) for k in keys])
    page = at // PAGE
    assert page.max() < 512
    v[np.arange(total), 0, page % HD] = torch.tensor(2.0 ** (page // HD)).float()
    k = torch.randn(total, 1, HD, generator=torch.Generator().manual_seed(1))
    s = Setup(ctx, mode, 1, rows, keys, kv=(k, v))
    assert np.array_equal(s.vx.reshape(total, HD), v.reshape(total, HD).double().numpy())
    want = []
    for b, (n, L) in enumerate(zip(rows, keys)):
        sums = np.cumsum(s.vx[s.start[b]:s.start[b + 1], 0], 0)
        seen = L - n + 1 + np.arange(n) if causal else np.full(n, L)
        want.append(sums[seen - 1] / seen[:, None])
    want = np.repeat(np.concatenate(want)[:, None], 2, 1).reshape(s.total, -1)
    tol = (torch.finfo(s.dt).eps / 2 + 2.0 ** -21) * want + (2.0 ** -25 if mode == "f16" else 0)
    q = torch.zeros(s.total, 2 * HD, dtype=s.dt)
    check(s.attend(q, 2, causal), want, tol)
    check(_unsplit(s, q, 2, causal), want, tol)


@pytest.mark.parametrize("mode", ["f16", "bf16"])
@pytest.mark.parametrize("keys", [9000, 28672])
def test_every_page_by_its_own_query(any_tile, mode, keys):
    """A row a page, whose q is 16 times the signs of one key there: its score is 181 and
    every other one at least 80 below it (checked), so all but that key have weight 0 and
    the output is that key's v, exactly: a code of the page's number."""
    ctx = any_tile
    say(f"kv page by query {mode} {keys}")
    n = -(-keys // PAGE)
    g = torch.Generator().manual_seed(keys)
    sign = torch.randint(0, 2, (n, HD), generator=g).float() * 2 - 1
    cross = (sign @ sign.T).fill_diagonal_(0).abs().max().item()
    assert 16 * (HD - cross) / math.sqrt(HD) > 80
    key = torch.arange(n) * PAGE + torch.randint(0, PAGE, (n,), generator=g)
    key = key.clamp_max(keys - 1)
    k, v = torch.zeros(2, keys, 1, HD)
    k[key, 0] = sign
    v[:, 0] = 1.5
    code = ((torch.arange(n)[:, None] >> (torch.arange(HD) % 9)) & 1).float() * 2 + 1
    v[key, 0] = code * torch.where(torch.arange(HD) % 2 == 0, 1.0, -1.0)
    s = Setup(ctx, mode, 1, [n], [keys], kv=(k, v))
    q = (16 * sign).to(s.dt)
    want = v[key, 0].double().numpy()
    check(s.attend(q, 1, False), want, np.zeros_like(want))
    check(_unsplit(s, q, 1, False), want, np.zeros_like(want))


@pytest.mark.parametrize("mode,rows,keys", [("f16", 1, 200000), ("f16", 150, 60000), ("bf16", 1, 200000)])
def test_many_small_weights(any_tile, mode, rows, keys):
    """One key whose score is 25.25 (in powers of two) above all others, which share the
    rest: in f16 their weights are below its smallest number where that key's is 1, and
    together they are 6.7e-3 of the result. f16 weights are held times 2^7: their rounding is
    off by 2^-25 / 2^7 at most. bf16's range has room."""
    ctx = any_tile
    say(f"kv small weights {mode} {keys}")
    k, v = torch.zeros(2, keys, 1, HD)
    at = keys // 3
    k[at, 0, 0] = 1.0
    v[:, 0] = 1.0
    v[at] = 0
    s = Setup(ctx, mode, 1, [rows], [keys], kv=(k, v))
    gap = 25.25
    q = torch.zeros(rows, HD, dtype=s.dt)
    q[:, 0] = gap * math.sqrt(HD) / 1.4426950408889634
    score = q[0, 0].item() / math.sqrt(HD) * 1.4426950408889634  # as rounded
    rest = (keys - 1) * 2.0 ** -score
    want = np.full((rows, HD), rest / (1 + rest))
    u = torch.finfo(s.dt).eps / 2
    # exponents and sums in f32: 2^-22 of the exponent, 2^-24 a key
    tol = (2 * u + 2.0 ** -22 * (score + 2) + 2 * keys * 2.0 ** -24) * want
    if mode == "f16":
        tol = tol + 2 * keys * 2.0 ** -32
        assert (tol < 0.06 * want).all()
    check(s.attend(q, 1, False), want, tol)


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


@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_captured_step_with_values_that_are_not_finite(any_tile, mode):
    """A captured write and attention: rows that hold a NaN make the rows that see them
    NaN in that replay, and not in the next, which holds others in their place; the page's
    flag, set by the write, is seen by the attention behind it."""
    ctx = any_tile
    say(f"kv captured not finite {mode}")
    rows, keys = [3, 100], [200, 130]
    s = Setup(ctx, mode, 2, rows, keys, seed=15)
    g = s.g
    q = s.queries(4).cuda()
    k, v, out = (torch.zeros(s.total, w, dtype=s.dt, device="cuda") for w in (2 * HD, 2 * HD, 4 * HD))
    work = torch.empty(max(16, ctx.kv_attention_workspace(s.cache, s.batch, 4)), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ctx.kv_write(s.cache, s.batch, k, v)
        ctx.kv_attention(s.cache, s.batch, q, out, 4, work=work)
    for bad in (None, (1, HD + 3), (50, 7), None, (102, 0)):
        new = [torch.randn(s.total, 2 * HD, generator=g).to(s.dt) for _ in range(2)]
        if bad:
            new[1][bad] = math.nan
        k.copy_(new[0])
        v.copy_(new[1])
        for x, t in ((s.kx, new[0]), (s.vx, new[1])):
            h = held(t.reshape(s.total, 2, HD), mode)
            for b, (n, L) in enumerate(zip(rows, keys)):
                x[s.start[b] + L - n:s.start[b] + L] = h[s.row_start[b]:s.row_start[b] + n]
        out.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        want, tol = s.want(q.cpu(), 4, True)
        assert np.isnan(want).any() == (bad is not None)
        check(out, want, tol)


def test_sequences_that_share_pages(any_tile):
    """A common beginning held once: two sequences whose tables name the same pages."""
    ctx = any_tile
    say("kv shared pages")
    s = Setup(ctx, "f16", 2, [2, 70, 1], [300, 330, 64], seed=16)
    s.pages[1, :4] = s.pages[0, :4]
    s.pages[2, 0] = s.pages[0, 2]
    for x in (s.kx, s.vx):
        x[s.start[1]:s.start[1] + 256] = x[:256]
        x[s.start[2]:s.start[2] + 64] = x[128:192]
    for causal in (True, False):
        q = s.queries(4)
        want, tol = s.want(q, 4, causal)
        check(s.attend(q, 4, causal), want, tol)


def test_a_workspace_of_the_other_form(ctx):
    """Sized without row_start and used with it, and the other way round."""
    say("kv workspace forms")
    n = 16
    s = Setup(ctx, "bf16", 8, [1] * n, [100 * i + 1 for i in range(n)], seed=17)
    q = s.queries(32)
    want, tol = s.want(q, 32, True)
    wide = torch.full((n, 128), -1, dtype=torch.int32, device="cuda")
    wide[:, :s.pages.shape[1]] = s.pages
    forms = [rt.KvBatch(s.lens, wide), rt.KvBatch(s.lens, wide, ints(range(n + 1)), n)]
    for a, b in (forms, forms[::-1]):
        size = ctx.kv_attention_workspace(s.cache, a, 32)
        assert size > 0
        work = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
        s.batch = b
        check(s.attend(q, 32, True, work=work), want, tol)
