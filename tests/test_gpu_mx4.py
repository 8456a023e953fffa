"""Microscaled 4-bit operands on the GPU against their definition in 64 bits.

Rows in the form are exactly determined: codes and scale codes must equal the oracle's.
In the linear every product of two codes and two powers of two is exact. A step's 128
products are summed in f32, with at most 128 roundings of sums no larger than S_g = sum
|a w| over the step, and its sum is added to the others': G additions (and the eight waves'
sums) no larger than S = sum S_g. So |error| <= 2^-24 (128 + G + 8) S + 2^-24 (|y| + |bias|),
doubled where a matrix instruction keeps its products' sum to one bit less. GELU multiplies
by at most 1.13 (its largest slope) and rounds to 2^-20 (exp2 and a reciprocal of an ulp
each, at arguments whose own rounding moves the tail by 2^-20); a 16-bit output adds eps / 2
of its size (2^-25 at least, f16's smallest step; bf16's lies far below)."""
import math

import numpy as np
import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ltx_amd import runtime as rt  # noqa: E402

MODES = {"f16": (rt.MODE_F16, torch.float16), "bf16": (rt.MODE_BF16, torch.bfloat16),
         "f32": (rt.MODE_F32, torch.float32)}
LIMITS = {"f16": (-23, 13), "bf16": (-125, 125), "f32": (-125, 125)}
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def oracle_codes(x, mode):
    """Codes [rows, K] (0 .. 15) and scale codes [rows, K / 32] of x, by the definition."""
    lo, hi = LIMITS[mode]
    g = x.double().cpu().numpy().reshape(x.shape[0], -1, 32)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        top = np.abs(g).max(2, keepdims=True)
        bad = ~np.isfinite(g).all(2)
        m, e = np.frexp(np.where(np.isfinite(top), top, 1))
        e = np.clip(np.where(top == 0, lo, e - 3 + (m > 0.875)), lo, hi)  # (log2 of 0: -inf, limited)
        y = np.where(np.isfinite(g), np.abs(g), 0) / 2.0 ** e
        dist = np.abs(y[..., None] - GRID)
        i = dist.argmin(-1)
        tie = np.take_along_axis(dist, np.minimum(i + 1, 7)[..., None], -1)[..., 0] == dist.min(-1)
        i = np.where(tie & (i < 7) & (i % 2 == 1), i + 1, i)
    codes = (i + 8 * np.signbit(g)).astype(np.uint8).reshape(x.shape[0], -1)
    return codes, np.where(bad, 255, e[..., 0] + 127).astype(np.uint8)


def values(codes, scales):
    """What they stand for, in f64."""
    v = np.where(codes & 8, -1.0, 1.0) * GRID[codes & 7]
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return v * s.repeat(32, 1)


def unpack(q, s):
    """The library's codes and scales -> codes [rows, K], scale codes [rows, K / 32]."""
    q, s = q.cpu().numpy(), s.cpu().numpy()
    return np.stack([q & 15, q >> 4], 2).reshape(q.shape[0], -1), s.transpose(1, 0, 2).reshape(q.shape[0], -1)


def pack(codes, scales):
    q = codes[:, 0::2] | codes[:, 1::2] << 4
    s = scales.reshape(scales.shape[0], -1, 4).transpose(1, 0, 2)
    return torch.from_numpy(np.ascontiguousarray(q)).cuda(), torch.from_numpy(np.ascontiguousarray(s)).cuda()


def room(rows, K):
    return (torch.full((rows, K // 2), 0xA5, dtype=torch.uint8, device="cuda"),
            torch.full((K // 128, rows, 4), 0x5A, dtype=torch.uint8, device="cuda"))


def quantise(ctx, x, mode, **kw):
    return ctx.mx4_quantise(x, *room(*x.shape), mode=MODES[mode][0], **kw)


# ---- rows ---------------------------------------------------------------------------

def _same(q, s, want):
    codes, scales = unpack(q, s)
    assert np.array_equal(scales, want[1])
    keep = (scales != 255).repeat(32, 1)  # (a group that is not a number has codes of any value)
    assert np.array_equal(codes[keep], want[0][keep])


def streams(n):
    """n streams of a whole round of torch's 32. torch hands them out in turn, the one that
    it captures on among them: taking rounds leaves the turn where other tests count on it."""
    return [torch.cuda.Stream() for _ in range(32)][:n]


@pytest.mark.parametrize("mode", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,K", [(1, 128), (3, 256), (31, 384), (32, 512), (33, 640), (100, 128), (5, 16384), (257, 1152)])
def test_rows_into_the_form(ctx, mode, rows, K):
    """Random rows, slices of wider ones; what lies around the outputs stays."""
    say(f"mx4 quantise {mode} {rows} x {K}")
    g = torch.Generator().manual_seed(rows + K)
    wide = torch.randn(rows, K + 24, generator=g) * torch.exp(2 * torch.randn(rows, K + 24, generator=g))
    wide = wide.to(MODES[mode][1]).cuda()
    x = wide[:, 8:8 + K]
    qs = torch.full((rows * K // 2 + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    ss = torch.full((rows * K // 32 + 64,), 0x5A, dtype=torch.uint8, device="cuda")
    q, s = qs[32:-32].view(rows, K // 2), ss[32:-32].view(K // 128, rows, 4)
    ctx.mx4_quantise(x, q, s, mode=MODES[mode][0])
    _same(q, s, oracle_codes(x, mode))
    assert bool((qs[:32] == 0xA5).all()) and bool((qs[-32:] == 0xA5).all())
    assert bool((ss[:32] == 0x5A).all()) and bool((ss[-32:] == 0x5A).all())
    y = torch.full((rows, K + 16), 7.0, dtype=x.dtype, device="cuda")
    ctx.mx4_values(q, s, y[:, 8:8 + K], mode=MODES[mode][0])
    assert np.array_equal(y[:, 8:8 + K].double().cpu().numpy(), values(*unpack(q, s)))
    assert bool((y[:, :8] == 7).all()) and bool((y[:, 8 + K:] == 7).all())


def _edge_rows(mode):
    """Groups at the borders of the form: midpoints, the 7 2^e step, zeros of both signs,
    the largest and smallest numbers of the type."""
    dt = MODES[mode][1]
    ticks = torch.tensor([0, 0.25, 0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7])
    groups = []
    for e in (-14, -3, 0, 5):
        for top in (4.0, 6.0, 7.0, 7.03125, 7.9375):
            g = torch.cat([ticks, -ticks]) * 2.0 ** e
            g = torch.where(g.abs() > top * 2.0 ** e, torch.zeros_like(g), g)
            g[31] = -top * 2.0 ** e
            groups.append(g.double())
    tiny, top = torch.finfo(dt).tiny, torch.finfo(dt).max
    sub = {"f16": 2.0 ** -24, "bf16": 2.0 ** -133, "f32": 2.0 ** -149}[mode]
    for a in (0.0, -0.0, sub, 3 * sub, tiny, 5 * tiny, top, top * 0.87, top * 0.8, -top, 1.0):
        g = torch.zeros(32, dtype=torch.float64)
        g[3], g[17], g[30] = a, a * 0.25, -a * 0.4
        groups.append(g)
    while len(groups) % 4:
        groups.append(torch.zeros(32, dtype=torch.float64))
    return torch.stack(groups).reshape(-1, 128).to(dt)


@pytest.mark.parametrize("mode", ["f16", "bf16", "f32"])
def test_borders_of_the_form(ctx, mode):
    """Also as rows that a linear quantises on its way: the same bits."""
    say(f"mx4 borders {mode}")
    x = _edge_rows(mode).cuda()
    q, s = quantise(ctx, x, mode)
    _same(q, s, oracle_codes(x, mode))
    if mode == "f32":
        return
    w = quantise(ctx, torch.randn(48, 128, device="cuda"), "f32")
    a, b = torch.empty(x.shape[0], 48, device="cuda"), torch.empty(x.shape[0], 48, device="cuda")
    ctx.linear_mx4(x, None, *w, None, a, mode=MODES[mode][0])
    ctx.linear_mx4(q, s, *w, None, b, mode=MODES[mode][0])
    assert torch.equal(a, b)


@pytest.mark.parametrize("mode", ["f16", "bf16", "f32"])
def test_values_that_are_not_finite(ctx, mode):
    """They make their group NaN, and nothing else."""
    say(f"mx4 not finite {mode}")
    x = torch.randn(40, 256, device="cuda").to(MODES[mode][1])
    x[3, 5], x[7, 100], x[39, 255] = math.nan, math.inf, -math.inf
    q, s = quantise(ctx, x, mode)
    _same(q, s, oracle_codes(x, mode))
    y = torch.empty_like(x)
    ctx.mx4_values(q, s, y, mode=MODES[mode][0])
    nan = torch.zeros(40, 8, dtype=torch.bool)
    nan[3, 0] = nan[7, 3] = nan[39, 7] = True
    assert torch.equal(torch.isnan(y).cpu(), nan.repeat_interleave(32, 1))


@pytest.mark.parametrize("mode", ["f16", "bf16", "f32"])
def test_any_scale_codes(ctx, mode):
    """All 256 scale codes with all 16 codes: the value, rounded to the type (a tie to even;
    beyond its largest, infinity)."""
    say(f"mx4 any scale codes {mode}")
    codes = np.tile(np.arange(16, dtype=np.uint8), (64, 8))
    scales = np.arange(256, dtype=np.uint8).reshape(64, 4)
    q, s = pack(codes, scales)
    y = torch.empty(64, 128, dtype=MODES[mode][1], device="cuda")
    ctx.mx4_values(q, s, y, mode=MODES[mode][0])
    want = torch.from_numpy(values(codes, scales)).to(MODES[mode][1]).double()
    got = y.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, 0.5, 1e300, -1e300), torch.nan_to_num(want, 0.5, 1e300, -1e300))


# ---- the linear -----------------------------------------------------------------------

def gelu64(z):
    return z / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def expected(a, w, bias, gelu, out):
    """The product in f64 of what a and w (codes, scales) stand for, and its bound."""
    ax, wx = values(*unpack(*a)), values(*unpack(*w))
    want, size = ax @ wx.T, np.abs(ax) @ np.abs(wx).T
    bx = 0.0 if bias is None else bias.double().cpu().numpy()[None]
    want = want + bx
    tol = 2 * 2.0 ** -24 * (128 + ax.shape[1] // 128 + 8) * size + 2.0 ** -24 * (np.abs(want) + np.abs(bx))
    if gelu:
        tol = 1.13 * tol + 2.0 ** -20 * np.abs(want)
        want = gelu64(want)
    if out != torch.float32:
        tol = tol + torch.finfo(out).eps / 2 * (np.abs(want) + tol) + 2.0 ** -25
    return want, tol


def check(y, want, tol):
    got = y.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = np.isnan(want) | (np.abs(got - want) <= tol)
    assert ok.all(), (int((~ok).sum()), float(np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-300))))


@pytest.fixture(params=["rule", "16", "64", "128", "256"])
def any_tile(request, monkeypatch, ctx):
    """The context, and one for each kernel of the linear whatever the rule would take."""
    if request.param == "rule":
        yield ctx
        return
    monkeypatch.setenv("LTX_MX4_TILE", request.param)
    c = rt.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("mode,out_f32", [("f16", False), ("bf16", False), ("bf16", True), ("f32", True)])
@pytest.mark.parametrize("M,N,K,bias,gelu", [
    (1, 1, 128, True, False),
    (1, 16, 256, False, False),
    (2, 33, 384, True, True),
    (17, 100, 512, False, False),
    (48, 257, 640, True, False),
    (64, 64, 1152, True, True),
    (65, 130, 128, False, False),
    (130, 300, 2048, True, False),
    (257, 511, 896, True, True),
    (300, 520, 4224, False, False),
])
def test_linear(any_tile, mode, out_f32, M, N, K, bias, gelu):
    ctx = any_tile
    say(f"linear_mx4 {mode} M={M} N={N} K={K} bias={bias} gelu={gelu} out_f32={out_f32}")
    g = torch.Generator().manual_seed(M + N + K)
    src = "bf16" if mode == "f32" else mode
    a = torch.randn(M, K, generator=g).to(MODES[src][1]).cuda()
    w = (torch.randn(N, K, generator=g) * 0.05 * torch.exp(torch.randn(N, 1, generator=g))).cuda()
    b = torch.randn(N, generator=g).cuda() if bias else None
    qa, qw = quantise(ctx, a, src), quantise(ctx, w, "f32")
    out = torch.float32 if out_f32 else MODES[mode][1]
    y = torch.full((M, N), 7.0, dtype=out, device="cuda")
    ctx.linear_mx4(*qa, *qw, b, y, mode=MODES[mode][0], gelu=gelu)
    check(y, *expected(qa, qw, b, gelu, out))
    if M <= 64 and mode != "f32":
        z = torch.full_like(y, 7.0)
        ctx.linear_mx4(a, None, *qw, b, z, mode=MODES[mode][0], gelu=gelu)
        check(z, *expected(qa, qw, b, gelu, out))


@pytest.mark.parametrize("M,N", [(1, 20), (16, 4112), (20, 4112), (40, 8208), (64, 16400), (33, 130)])
@pytest.mark.parametrize("mode", ["f16", "bf16"])
def test_few_rows(ctx, mode, M, N):
    """Every form of the kernel of few rows (1 .. 4 times 16 rows, 1, 2 and 4 times 16
    columns), at 37 steps of k: no multiple of the waves or of the loads in flight."""
    say(f"linear_mx4 few rows {mode} M={M} N={N}")
    K = 37 * 128
    g = torch.Generator(device="cuda").manual_seed(M + N)
    a = torch.randn(M, K, generator=g, device="cuda").to(MODES[mode][1])
    w = torch.randn(N, K, generator=g, device="cuda") * 0.02
    qa, qw = quantise(ctx, a, mode), quantise(ctx, w, "f32")
    want, tol = expected(qa, qw, None, False, torch.float32)
    for aa in (qa, (a, None)):
        y = torch.full((M, N), 7.0, device="cuda")
        ctx.linear_mx4(*aa, *qw, None, y, mode=MODES[mode][0])
        check(y, want, tol)


@pytest.mark.parametrize("M,N,K", [(3, 40, 384), (200, 300, 640)])
def test_scales_far_apart(any_tile, M, N, K):
    """Scale codes of any size whose products stay in f32, 0 and 254 among them."""
    ctx = any_tile
    say(f"linear_mx4 scales {M} {N} {K}")
    r = np.random.default_rng(M)
    a = r.integers(0, 16, (M, K), dtype=np.uint8), r.integers(60, 130, (M, K // 32)).astype(np.uint8)
    w = r.integers(0, 16, (N, K), dtype=np.uint8), r.integers(90, 170, (N, K // 32)).astype(np.uint8)
    a[1][1, :], w[1][:, 1] = 0, 254  # 2^-127 and 2^127: only with each other is that in range
    a[0][[i for i in range(M) if i != 1], 32:64] = 0
    a[1][2, 0] = 0
    qa, qw = pack(*a), pack(*w)
    y = torch.full((M, N), 7.0, device="cuda")
    ctx.linear_mx4(*qa, *qw, None, y)
    check(y, *expected(qa, qw, None, False, torch.float32))


@pytest.mark.parametrize("M,N", [(4, 40), (70, 80)])
def test_groups_that_are_nan(any_tile, M, N):
    """A NaN group of a makes its row NaN, one of w its column, whatever meets it (zeros)."""
    ctx = any_tile
    say(f"linear_mx4 nan {M} {N}")
    K = 384
    a = torch.randn(M, K, device="cuda").half()
    w = torch.randn(N, K, device="cuda") * 0.1
    a[2, 300], w[7, 0] = math.inf, math.nan
    w[:, 288:320] = 0
    qa, qw = quantise(ctx, a, "f16"), quantise(ctx, w, "f32")
    for aa in [qa] + ([(a, None)] if M <= 64 else []):
        y = torch.full((M, N), 7.0, device="cuda")
        ctx.linear_mx4(*aa, *qw, None, y)
        nan = torch.zeros(M, N, dtype=torch.bool)
        nan[2], nan[:, 7] = True, True
        assert torch.equal(torch.isnan(y).cpu(), nan)


@pytest.mark.parametrize("out", [torch.float16, torch.float32])
@pytest.mark.parametrize("M,N", [(5, 17), (66, 64), (90, 81)])
def test_y_anywhere(any_tile, M, N, out):
    """y that starts on its type alone, odd rows; what lies around it stays."""
    ctx = any_tile
    say(f"linear_mx4 y anywhere {M} {N} {out}")
    K = 256
    qa = quantise(ctx, torch.randn(M, K, device="cuda").half(), "f16")
    qw = quantise(ctx, torch.randn(N, K, device="cuda"), "f32")
    buf = torch.full((M * N + 34,), 7.0, dtype=out, device="cuda")
    y = buf[17:17 + M * N].view(M, N)
    ctx.linear_mx4(*qa, *qw, None, y)
    check(y, *expected(qa, qw, None, False, out))
    assert bool((buf[:17] == 7).all()) and bool((buf[17 + M * N:] == 7).all())


@pytest.mark.parametrize("K", [128, 512, 640, 2176])
@pytest.mark.parametrize("M,N,mode,out_f32,bias,gelu", [
    (4369, 4880, "f16", False, True, False), (4096, 4608, "bf16", False, True, True), (5000, 4100, "f16", True, True, False),
    (4600, 4999, "bf16", False, False, False),
])
def test_many_tiles(ctx, M, N, mode, out_f32, bias, gelu, K):
    """More tiles than CUs: a workgroup's next tile comes in while the last one leaves.
    Called again and again, the same bits. (f64 on the GPU)"""
    say(f"linear_mx4 many tiles M={M} N={N} K={K} {mode} out_f32={out_f32}")
    g = torch.Generator(device="cuda").manual_seed(M + K)
    a = torch.randn(M, K, generator=g, device="cuda").to(MODES[mode][1])
    w = torch.randn(N, K, generator=g, device="cuda") * 0.05
    b = torch.randn(N, generator=g, device="cuda") if bias else None
    qa, qw = quantise(ctx, a, mode), quantise(ctx, w, "f32")
    ax, wx = torch.empty(M, K, device="cuda"), torch.empty(N, K, device="cuda")
    ctx.mx4_values(*qa, ax, mode=rt.MODE_F32)
    ctx.mx4_values(*qw, wx, mode=rt.MODE_F32)
    out = torch.float32 if out_f32 else MODES[mode][1]
    y = torch.full((M, N), 7.0, dtype=out, device="cuda")
    ctx.linear_mx4(*qa, *qw, b, y, mode=MODES[mode][0], gelu=gelu)
    want = ax.double() @ wx.double().T
    size = ax.double().abs() @ wx.double().abs().T
    bx = torch.zeros((), dtype=torch.float64, device="cuda") if b is None else b.double()
    want = want + bx
    tol = 2 * 2.0 ** -24 * (128 + K // 128 + 8) * size + 2.0 ** -24 * (want.abs() + bx.abs())
    if gelu:
        tol = 1.13 * tol + 2.0 ** -20 * want.abs()
        want = want / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (want + 0.044715 * want ** 3)))
    if not out_f32:
        tol = tol + torch.finfo(out).eps / 2 * (want.abs() + tol) + 2.0 ** -25
    off = (y.double() - want).abs()
    assert bool((off <= tol).all()), (int((off > tol).sum()), float((off / tol).max()))
    for _ in range(10):
        z = torch.full_like(y, 7.0)
        ctx.linear_mx4(*qa, *qw, b, z, mode=MODES[mode][0], gelu=gelu)
        assert torch.equal(y, z)


def test_captured_and_on_another_stream(ctx):
    """Quantise and multiply, replayed with other inputs, and beside it on a stream."""
    say("linear_mx4 graph and stream")
    M, N, K = 100, 272, 1024
    x = torch.randn(M, K, device="cuda").half()
    w = quantise(ctx, torch.randn(N, K, device="cuda") * 0.02, "f32")
    held, y = room(M, K), torch.zeros(M, N, dtype=torch.float16, device="cuda")

    def step(**kw):
        ctx.mx4_quantise(x, *held, **kw)
        ctx.linear_mx4(*held, *w, None, y, gelu=True, **kw)
        ctx.linear_mx4(x[:20], None, *w, None, y[:20], **kw)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(torch.randn(M, K, device="cuda").half() * (i + 1))
        y.zero_()
        step()
        eager = y.clone()
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, eager)
        st, = streams(1)
        y.zero_()
        torch.cuda.synchronize()
        step(stream=st)
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


@pytest.mark.parametrize("K", [1024, 4096])
def test_rows_in_values_at_once(ctx, K):
    """Calls on four streams, which from 2^17 values on share the context's scratch, and two
    graphs, which take none: the bits of each call alone. (The order of the sums differs, but
    f32 holds these exactly: 32 normal values have their largest within a factor of 8 of
    other groups', so products are multiples of 2^-8 of the largest scales' product, and
    4,096 of them, of 2 in the mean square and 36 at most, stay below 2^24 of those.)"""
    say(f"linear_mx4 rows in values at once K={K}")
    cases = [(17, 272), (64, 4112), (33, 96), (48, 528)]
    w = [quantise(ctx, torch.randn(N, K, device="cuda") * 0.02, "f32") for _, N in cases]
    x = [torch.randn(M, K, device="cuda").bfloat16() for M, _ in cases]
    want = [torch.empty(M, N, device="cuda") for M, N in cases]
    got = [torch.zeros_like(t) for t in want]

    def call(i, y, **kw):
        ctx.linear_mx4(x[i], None, *w[i], None, y, mode=rt.MODE_BF16, **kw)

    for i, y in enumerate(want):
        call(i, y)
    sts = streams(len(cases))
    torch.cuda.synchronize()
    for _ in range(10):
        for i, st in enumerate(sts):
            call(i, got[i], stream=st)
    torch.cuda.synchronize()
    assert all(torch.equal(g, t) for g, t in zip(got, want))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            call(i, got[i])
    for _ in range(3):
        for g in got:
            g.zero_()
        torch.cuda.synchronize()
        for graph, st in zip(graphs, sts):
            with torch.cuda.stream(st):
                graph.replay()
        for i in (2, 3):
            call(i, got[i])
        torch.cuda.synchronize()
        assert all(torch.equal(g, t) for g, t in zip(got, want))


def test_empty_and_refused(ctx):
    say("mx4 refusals")
    q, s = room(0, 256)
    ctx.mx4_quantise(torch.empty(0, 256, dtype=torch.float16, device="cuda"), q, s)
    x = torch.randn(4, 256, device="cuda").half()
    q, s = room(4, 256)
    for bad in [dict(x=x.float()), dict(x=x[:, :128]), dict(x=x.T), dict(q=q[:, :64]), dict(s=s[:1]), dict(s=s.transpose(0, 1)),
                dict(x=torch.randn(4, 264, device="cuda").half()[:, 4:260]), dict(x=x.cpu()), dict(q=q.float())]:
        args = dict(dict(x=x, q=q, s=s), **bad)
        with pytest.raises(rt.LtxError):
            ctx.mx4_quantise(args["x"], args["q"], args["s"])
    with pytest.raises(rt.LtxError):
        ctx.mx4_quantise(x[:, :96], q[:, :48].contiguous(), s[:1])
    assert bool((q == 0xA5).all()) and bool((s == 0x5A).all())
    qa, qw = quantise(ctx, x, "f16"), quantise(ctx, torch.randn(32, 256, device="cuda"), "f32")
    y = torch.full((4, 32), 7.0, dtype=torch.float16, device="cuda")
    big = torch.randn(65, 256, device="cuda").half()
    for a, a_s, w, b, out, mode in [
            (x[:, :128], None, qw, None, y, 0), (x.bfloat16(), None, qw, None, y, 0), (qa[0], qa[1][:1], qw, None, y, 0),
            (*qa, (qw[0][:, :64], qw[1]), None, y, 0), (*qa, qw, torch.zeros(31, device="cuda"), y, 0), (*qa, qw, None, y.T, 0),
            (*qa, qw, None, y, 1), (*qa, qw, None, y, 5), (*qa, qw, None, y, 2), (x.float(), None, qw, None, y.float(), 2),
            (big, None, qw, None, torch.empty(65, 32, dtype=torch.float16, device="cuda"), 0)]:
        with pytest.raises(rt.LtxError):
            ctx.linear_mx4(a, a_s, *w, b, out, mode=mode)
    assert bool((y == 7).all())
