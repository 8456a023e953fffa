"""The microscaled 4-bit linear, kernel by kernel: every form that sizes select, by the name
that the launches are recorded under, and the longest k with each tile. Bounds as in
test_gpu_mx4.py; the products are formed in f64 on the GPU."""
import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ltx_amd import runtime as rt  # noqa: E402
from test_gpu_mx4 import MODES, quantise  # noqa: E402


def operands(ctx, mode, M, N, K):
    """a [M, K] of the type, both operands in the form, and a . w^T of what they stand for
    with its bound."""
    g = torch.Generator(device="cuda").manual_seed(M + N + K)
    a = torch.randn(M, K, generator=g, device="cuda").to(MODES[mode][1])
    w = torch.randn(N, K, generator=g, device="cuda") * 0.02
    qa, qw = quantise(ctx, a, mode), quantise(ctx, w, "f32")
    ax, wx = torch.empty(M, K, device="cuda"), torch.empty(N, K, device="cuda")
    ctx.mx4_values(*qa, ax, mode=rt.MODE_F32)
    ctx.mx4_values(*qw, wx, mode=rt.MODE_F32)
    want, size = ax.double() @ wx.double().T, ax.double().abs() @ wx.double().abs().T
    return a, qa, qw, want, 2 * 2.0 ** -24 * (128 + K // 128 + 8) * size + 2.0 ** -24 * want.abs()


def right(y, want, tol):
    if y.dtype != torch.float32:
        tol = tol + torch.finfo(y.dtype).eps / 2 * (want.abs() + tol) + 2.0 ** -25
    off = (y.double() - want).abs()
    assert bool((off <= tol).all()), (int((off > tol).sum()), float((off / tol).max()))


def launched(ctx, call):
    """How many kernels whose name holds `part` a call launches, as a function of `part`."""
    ctx.profile_reset()
    ctx.profile(True)
    try:
        call()
    finally:
        ctx.profile(False)
    return lambda part: ctx.profile_read(part)[1]


@pytest.mark.parametrize("mode", ["f16", "bf16"])
@pytest.mark.parametrize("M", [1, 16, 17, 32, 33, 41, 49, 64])
@pytest.mark.parametrize("N", [40, 4112, 8208, 16400])
def test_rows_in_values(ctx, mode, M, N):
    """One to four times 16 rows, one, two and four times 16 columns, at 13 steps of k: at
    most 2^17 values, so that they are quantised in the product itself; in the type and f32."""
    K, cols = 13 * 128, {40: 1, 4112: 2, 8208: 4, 16400: 4}[N]
    name = f"ltx_linear_mx4_{mode}_rows_{(M + 15) // 16}_{cols}"
    say(f"linear_mx4 {name} M={M} N={N}")
    a, _, qw, want, tol = operands(ctx, mode, M, N, K)
    for out in (torch.float32, MODES[mode][1]):
        y = torch.full((M, N), 7.0, dtype=out, device="cuda")
        count = launched(ctx, lambda: ctx.linear_mx4(a, None, *qw, None, y, mode=MODES[mode][0]))
        assert count(name) == count("") == 1
        right(y, want, tol)


@pytest.mark.parametrize("mode", ["f16", "bf16"])
@pytest.mark.parametrize("M,N", [(17, 4112), (33, 40), (48, 4112), (40, 8208), (64, 40), (64, 4112), (50, 16400)])
def test_rows_in_values_captured(ctx, mode, M, N):
    """More than 2^17 values in a captured call, which takes no scratch: the same kernels over
    37 steps of k, no multiple of the waves or of the loads in flight."""
    say(f"linear_mx4 rows captured {mode} M={M} N={N}")
    a, _, qw, want, tol = operands(ctx, mode, M, N, 37 * 128)
    y = torch.zeros(M, N, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.linear_mx4(a, None, *qw, None, y, mode=MODES[mode][0])
    for _ in range(3):
        y.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        right(y, want, tol)


@pytest.mark.parametrize("mode", ["f16", "bf16"])
@pytest.mark.parametrize("M,N,form", [(1, 40, "1_1"), (16, 4096, "1_1"), (5, 4112, "1_2"), (16, 8192, "1_2"), (17, 40, "2_1"),
                                      (32, 4096, "2_1")])
def test_few_rows_of_codes(ctx, mode, M, N, form):
    name = f"ltx_linear_mx4_{mode}_{form}"
    say(f"linear_mx4 {name} M={M} N={N}")
    _, qa, qw, want, tol = operands(ctx, mode, M, N, 37 * 128)
    for out in (torch.float32, MODES[mode][1]):
        y = torch.full((M, N), 7.0, dtype=out, device="cuda")
        count = launched(ctx, lambda: ctx.linear_mx4(*qa, *qw, None, y, mode=MODES[mode][0]))
        assert count(name) == count("") == 1
        right(y, want, tol)


@pytest.mark.parametrize("tile", ["16", "64", "128", "256"])
@pytest.mark.parametrize("M,N", [(300, 520), (77, 201)])
def test_long_k(monkeypatch, tile, M, N):
    """k of 16,384 and 16,512, an odd count of steps, with each tile; the groups of waves of
    64 and 128 share it; rows of y on 16 bytes and not."""
    say(f"linear_mx4 long k tile={tile} M={M} N={N}")
    monkeypatch.setenv("LTX_MX4_TILE", tile)
    c = rt.Context(0)
    for K in (16384, 16384 + 128):
        _, qa, qw, want, tol = operands(c, "bf16", M, N, K)
        for out in (torch.float32, torch.bfloat16):
            y = torch.full((M, N), 7.0, dtype=out, device="cuda")
            c.linear_mx4(*qa, *qw, None, y, mode=rt.MODE_BF16)
            right(y, want, tol)
            z = torch.full_like(y, 7.0)
            c.linear_mx4(*qa, *qw, None, z, mode=rt.MODE_BF16)
            assert torch.equal(y, z)
    torch.cuda.synchronize()
    c.close()


@pytest.mark.parametrize("M,N,form", [(64, 4096, "64k4"), (256, 4096, "64k4"), (512, 4096, "64k2"), (1024, 4096, "128k2"),
                                      (64, 4100, "odd"), (2048, 8192, "256")])
def test_long_k_by_the_rule(ctx, M, N, form):
    """The block's widest k with the tiles that the rule takes."""
    say(f"linear_mx4 long k M={M} N={N} {form}")
    _, qa, qw, want, tol = operands(ctx, "f16", M, N, 16384)
    y = torch.full((M, N), 7.0, dtype=torch.float16, device="cuda")
    count = launched(ctx, lambda: ctx.linear_mx4(*qa, *qw, None, y))
    assert count(f"ltx_gemm_mx4_f16_{form}") >= 1 and count("") == 1
    right(y, want, tol)


@pytest.mark.skipif(not hasattr(torch, "float4_e2m1fn_x2"), reason="torch has no 4-bit type")
@pytest.mark.parametrize("M", [5, 90])
def test_torchs_own_types(ctx, M):
    """Codes and scales as torch's types for these bytes, out of rows and into a linear: the
    same bits."""
    say(f"linear_mx4 torch's types M={M}")
    own = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
    x, w = torch.randn(M, 256, device="cuda").half(), torch.randn(48, 256, device="cuda")
    q, s = quantise(ctx, x, "f16")
    qo, so = torch.zeros_like(q).view(own[0]), torch.zeros_like(s).view(own[1])
    ctx.mx4_quantise(x, qo, so)
    assert torch.equal(qo.view(torch.uint8), q) and torch.equal(so.view(torch.uint8), s)
    a, b = torch.empty_like(x), torch.empty_like(x)
    ctx.mx4_values(q, s, a)
    ctx.mx4_values(qo, so, b)
    assert torch.equal(a, b)
    qw, sw = quantise(ctx, w, "f32")
    y, z = torch.empty(M, 48, device="cuda"), torch.empty(M, 48, device="cuda")
    ctx.linear_mx4(q, s, qw, sw, None, y)
    ctx.linear_mx4(qo, so, qw.view(own[0]), sw.view(own[1]), None, z)
    assert torch.equal(y, z)
