"""The linear with 4-bit weights on the GPU against f64.

Weights are exact MFMA operands (integers / 16) and a 16-bit a is one as well (f32: its
three bf16 planes), so every product is exact. A group's 128 products are summed in
f32, at most 3 x 128 + 8 additions of partial sums no larger than S = sum |a q|; the
scale, the groups' sum and the bias round once each per group: with G groups,
|error| <= 2^-24 (3 * 128 + 8 + G + 8) sum |a q s| + 2^-24 (|y| + |bias|), doubled where
a matrix instruction keeps its products' sum to one bit less. GELU multiplies by at
most 1.13 (its largest slope) and rounds to 2^-20 (exp2 and a reciprocal of an ulp
each, at arguments whose own rounding moves the tail by 2^-20); a 16-bit output adds
eps / 2 of its size (2^-25 at least, f16's smallest step)."""
import math

import numpy as np
import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ltx_amd import runtime as rt  # noqa: E402

MODES = {"f16": (rt.MODE_F16, torch.float16), "bf16": (rt.MODE_BF16, torch.bfloat16),
         "f32": (rt.MODE_F32, torch.float32)}


def packed(w):
    b = (torch.as_tensor(w).to(torch.int32) & 15).to(torch.uint8)
    return (b[:, 0::2] | (b[:, 1::2] << 4)).contiguous()


def case(mode, M, N, K, scale="f32", seed=0):
    g = torch.Generator().manual_seed(seed + M + N + K)
    a = torch.randn(M, K, generator=g).to(MODES[mode][1])
    w = torch.randint(-8, 8, (N, K), generator=g)
    s = (torch.rand(N, K // 128, generator=g) * 0.03 + 0.001).to(torch.float16 if scale == "f16" else torch.float32)
    bias = torch.randn(N, generator=g)
    return a, w, s, bias


def run(ctx, mode, a, w, s, bias, gelu, out_f32):
    y = torch.full((a.shape[0], w.shape[0]), 7.0, dtype=torch.float32 if out_f32 else a.dtype, device="cuda")
    ctx.linear_q4(a.cuda(), packed(w).cuda(), s.cuda(), None if bias is None else bias.cuda(), y, mode=MODES[mode][0],
                  gelu=gelu)
    return y


def gelu64(z):
    return z / (1 + np.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


@pytest.mark.parametrize("mode,out_f32", [("f16", False), ("f16", True), ("bf16", False), ("bf16", True), ("f32", True)])
@pytest.mark.parametrize("M,N,K,scale,bias,gelu", [
    (1, 1, 128, "f32", True, False),
    (1, 4096, 4096, "f16", True, False),
    (2, 100, 384, "f16", False, False),
    (5, 33, 1152, "f32", True, True),
    (16, 256, 512, "f16", True, True),
    (17, 48, 16384, "f32", False, False),
    (31, 1000, 640, "f16", True, False),
    (33, 272, 256, "f32", True, True),
    (64, 512, 1024, "f16", False, False),
    (77, 4100, 128, "f16", True, True),
    (130, 160, 2048, "f32", True, False),
    (256, 130, 896, "f16", True, False),
    (300, 64, 384, "f32", False, True),
])
def test_linear_q4(ctx, mode, out_f32, M, N, K, scale, bias, gelu):
    say(f"linear_q4 {mode} M={M} N={N} K={K} scale={scale} bias={bias} gelu={gelu} out_f32={out_f32}")
    a, w, s, b = case(mode, M, N, K, scale)
    b = b if bias else None
    got = run(ctx, mode, a, w, s, b, gelu, out_f32).double().cpu().numpy()
    ws = w.double().numpy() * s.double().repeat_interleave(128, 1).numpy()
    ax = a.double().numpy()
    want = ax @ ws.T
    size = np.abs(ax) @ np.abs(ws).T
    bx = 0.0 if b is None else b.double().numpy()[None]
    want = want + bx
    tol = 2 * 2.0 ** -24 * (3 * 128 + 16 + K // 128) * size + 2.0 ** -24 * (np.abs(want) + np.abs(bx))
    if gelu:
        tol = 1.13 * tol + 2.0 ** -20 * np.abs(want)
        want = gelu64(want)
    if not out_f32:
        tol = tol + torch.finfo(a.dtype).eps / 2 * (np.abs(want) + tol) + 2.0 ** -25
    off = np.abs(got - want)
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("mode", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("M,N", [(3, 48), (40, 130)])
def test_one_hot_rows_give_the_weights(ctx, mode, M, N):
    """a = 2^j at one place: each output is one weight times its scale, exactly."""
    say(f"linear_q4 one-hot {mode} M={M}")
    K = 384
    _, w, s, _ = case(mode, M, N, K, "f16")
    for shift in range(0, K, M):
        at = (np.arange(M) + shift) % K
        a = torch.zeros(M, K)
        a[np.arange(M), at] = 4.0
        got = run(ctx, mode, a.to(MODES[mode][1]), w, s, None, False, True).double().cpu().numpy()
        ws = w.double().numpy() * s.double().repeat_interleave(128, 1).numpy()
        assert np.array_equal(got, 4 * ws[:, at].T)


def test_f32_keeps_small_and_large_values(ctx):
    """The planes hold every f32: cancelling large values leave the small ones."""
    say("linear_q4 f32 planes")
    K = 256
    a = torch.zeros(2, K)
    a[0, 0], a[0, 1], a[0, 130] = 1 + 2.0 ** -23, -1.0, 2.0 ** -60
    a[1, 5], a[1, 200] = 3.0e38, 1.2345678e-30
    w = torch.ones(16, K, dtype=torch.int64)
    w[1] = -1
    w[2, 5] = 0
    s = torch.ones(16, 2)
    got = run(ctx, "f32", a, w, s, None, False, True).double().cpu().numpy()
    ax = a.double().numpy()
    want = ax @ w.double().numpy().T
    assert np.array_equal(got[0], want[0].astype(np.float32).astype(np.float64))
    assert np.allclose(got[1], want[1], rtol=2.0 ** -23, atol=0)


@pytest.mark.parametrize("mode", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("M", [3, 20])
def test_values_that_are_not_finite_stay_in_their_row(ctx, mode, M):
    """An infinity times non-zero weights is that infinity; NaN where 0 or opposite
    signs meet it; every other row as without."""
    say(f"linear_q4 not finite {mode}")
    a, w, s, b = case(mode, M, 40, 256)
    w[w == 0] = 3
    w[7, 9] = 0
    clean = run(ctx, mode, a, w, s, b, False, True)
    a[1, 9] = math.inf
    a[2, 70] = math.nan
    got = run(ctx, mode, a, w, s, b, False, True)
    keep = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(got[keep], clean[keep])
    row = got[1].cpu()
    want = torch.where(w[:, 9] > 0, math.inf, -math.inf)
    want[7] = math.nan
    assert torch.equal(torch.nan_to_num(row, 5.0, 1e9, -1e9), torch.nan_to_num(want, 5.0, 1e9, -1e9))
    assert torch.isnan(got[2]).all()


def test_captured_and_on_another_stream(ctx):
    say("linear_q4 graph and stream")
    a, w, s, b = case("f16", 4, 272, 1024)
    eager = run(ctx, "f16", a, w, s, b, True, False)
    x, q, sc, bi = a.cuda(), packed(w).cuda(), s.cuda(), b.cuda()
    y = torch.zeros_like(eager)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    ctx.linear_q4(x, q, sc, bi, y, mode=rt.MODE_F16, gelu=True, stream=st)
    torch.cuda.synchronize()
    assert torch.equal(y, eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.linear_q4(x, q, sc, bi, y, mode=rt.MODE_F16, gelu=True)
    for i in range(4):
        y.zero_()
        x.copy_(a.cuda() * (i + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, run(ctx, "f16", (a * (i + 1)).half(), w, s, b, True, False))


def test_refusals(ctx):
    say("linear_q4 refusals")
    a, w, s, b = (t.cuda() for t in case("f16", 2, 32, 256))
    q, y = packed(w.cpu()).cuda(), torch.full((2, 32), 7.0, dtype=torch.float16, device="cuda")
    for bad in [dict(a=a[:, :128]), dict(q=q[:, :64].contiguous()), dict(s=s[:, :1].contiguous()), dict(y=y.T),
                dict(b=b[:5]), dict(a=a.bfloat16()), dict(a=a[:, ::2])]:
        args = dict(dict(a=a, q=q, s=s, b=b, y=y), **bad)
        with pytest.raises(rt.LtxError):
            ctx.linear_q4(args["a"], args["q"], args["s"], args["b"], args["y"])
    with pytest.raises(rt.LtxError):
        ctx.linear_q4(a.float(), q, s, b, y, mode=rt.MODE_F32)
    with pytest.raises(rt.LtxError, match="unknown mode|types"):
        ctx.linear_q4(a, q, s, b, y, mode=5)
    assert (y == 7).all()


@pytest.mark.parametrize("scale", ["f16", "f32"])
@pytest.mark.parametrize("N", [48, 4112, 8200])
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5, 6])
def test_f32_planes_of_few_rows(ctx, M, N, scale):
    """Up to five rows share a tile with their planes, six do not."""
    say(f"linear_q4 f32 few rows M={M} N={N} {scale}")
    a, w, s, b = case("f32", M, N, 640, scale, seed=M)
    got = run(ctx, "f32", a, w, s, b, False, True).double().cpu().numpy()
    ws = w.double().numpy() * s.double().repeat_interleave(128, 1).numpy()
    ax, bx = a.double().numpy(), b.double().numpy()[None]
    want = ax @ ws.T + bx
    size = np.abs(ax) @ np.abs(ws).T
    tol = 2 * 2.0 ** -24 * (3 * 128 + 16 + 5) * size + 2.0 ** -24 * (np.abs(want) + np.abs(bx))
    off = np.abs(got - want)
    assert (off <= tol).all(), float((off / tol).max())
