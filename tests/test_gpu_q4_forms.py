"""The linear with 4-bit weights: every tile form that the sizes select, and the ends
of f32's range. Bounds as in test_gpu_q4.py."""
import math

import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ltx_amd import runtime as rt  # noqa: E402
from test_gpu_q4 import MODES, packed  # noqa: E402


@pytest.mark.parametrize("scale", ["f16", "f32"])
@pytest.mark.parametrize("mode", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("N", [48, 4112, 8200, 16400])
def test_every_tile_form(ctx, mode, N, scale):
    """Rows and columns that take each of the tiles (1 and 2 times 16 rows; 1, 2 and 4
    times 16 columns; mode F32 with its planes in one tile and in three), at 37 groups of
    k: five for a wave, two for the last, no multiple of the loads in flight. The oracle is
    a product in f64."""
    g = torch.Generator(device="cuda").manual_seed(N)
    K, dt = 37 * 128, MODES[mode][1]
    w = torch.randint(-8, 8, (N, K), generator=g, device="cuda")
    s = torch.rand(N, K // 128, generator=g, device="cuda") * 0.03 + 0.001
    s = s.to(torch.float16 if scale == "f16" else torch.float32)
    bias = torch.randn(N, generator=g, device="cuda")
    q = packed(w)
    ws = w.double() * s.double().repeat_interleave(128, 1)
    for M in (1, 3, 5, 16, 17, 32, 33, 64):
        say(f"linear_q4 forms {mode} M={M} N={N} {scale}")
        a = torch.randn(M, K, generator=g, device="cuda").to(dt)
        want = a.double() @ ws.T + bias.double()
        size = a.double().abs() @ ws.abs().T
        sums = 2 * 2.0 ** -24 * (3 * 128 + 16 + K // 128) * size + 2.0 ** -24 * (want.abs() + bias.double().abs())
        for out_f32 in (True,) if mode == "f32" else (True, False):
            y = torch.full((M, N), 7.0, dtype=torch.float32 if out_f32 else dt, device="cuda")
            ctx.linear_q4(a, q, s, bias, y, mode=MODES[mode][0])
            tol = sums if out_f32 else sums + torch.finfo(dt).eps / 2 * (want.abs() + sums) + 2.0 ** -25
            off = (y.double() - want).abs()
            assert bool((off <= tol).all()), (M, out_f32, float((off / tol).max()))


@pytest.mark.parametrize("mode", ["bf16", "f32"])
@pytest.mark.parametrize("M,N", [(1, 48), (4, 4112), (5, 8200), (6, 48), (16, 4112), (17, 48), (33, 4112), (20, 8200)])
def test_the_range_of_f32(ctx, mode, M, N):
    """Values of a up to f32's largest, whose products with the weights alone leave f32
    and with the scales do not: y is right where it is finite; rows that hold an infinity
    or NaN stay those."""
    say(f"linear_q4 range {mode} M={M} N={N}")
    K, dt = 640, MODES[mode][1]
    g = torch.Generator(device="cuda").manual_seed(M + N)
    a = torch.rand(M, K, generator=g, device="cuda").double() + 0.5
    a = a * 2.0 ** torch.linspace(0, 127, M, device="cuda", dtype=torch.float64)[:, None].round()
    a[-1] = torch.finfo(dt).max
    a = a.to(dt)
    w = torch.randint(1, 8, (N, K), generator=g, device="cuda")  # one sign: the sums grow
    s = torch.rand(N, K // 128, generator=g, device="cuda") * 2.0 ** -16 + 2.0 ** -17
    y = torch.full((M, N), 7.0, device="cuda")
    ctx.linear_q4(a, packed(w), s, None, y, mode=MODES[mode][0])
    want = a.double() @ (w.double() * s.double().repeat_interleave(128, 1)).T
    assert float(want.max()) < 2.0 ** 127
    off = (y.double() - want).abs()
    tol = 2 * 2.0 ** -24 * (3 * 128 + 16 + K // 128) * want
    assert bool((off <= tol).all()), float((off / tol).max())
    if M < 4:
        return
    clean = y.clone()
    a[1, 9], a[2, 70] = math.inf, math.nan
    ctx.linear_q4(a, packed(w), s, None, y, mode=MODES[mode][0])
    assert bool(torch.isinf(y[1]).all()) and bool((y[1] > 0).all()) and bool(torch.isnan(y[2]).all())
    keep = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(y[keep], clean[keep])
