"""The norm of q and k over the whole range of the types: rows whose squares leave f32 at
either end, among ordinary ones. Bounds as in test_gpu_rope.py, whose sums of squares these
rows' are no worse than."""
import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_rope import MODES, check, expected, plan, tensors, weights  # noqa: E402


def far(x, seed, exponents):
    """Every third row times one of 2^exponents; the largest stay within the type."""
    g = torch.Generator().manual_seed(seed)
    e = torch.tensor(exponents)[torch.randint(0, len(exponents), (x.shape[0],), generator=g)]
    e = torch.where(torch.rand(x.shape[0], generator=g) < 0.34, e, torch.zeros_like(e))
    top = torch.finfo(x.dtype).max
    return (x.double().cpu() * 2.0 ** e[:, None].double()).clamp(-top, top).to(x.dtype).cuda()


@pytest.mark.parametrize("mode", ["bf16", "f32"])
@pytest.mark.parametrize("rows,heads,kv_heads", [(9, 32, 8), (1700, 32, 32), (40, 1, 4), (30, 40, 5), (21, 33, 33), (5, 96, 8)])
@pytest.mark.parametrize("eps", [1e-6, 0.0, 2.0 ** -140])
def test_rows_whose_squares_leave_f32(ctx, mode, rows, heads, kv_heads, eps):
    say(f"qk_rope range {mode} rows={rows} heads={heads}/{kv_heads} eps={eps}")
    p = plan(1, 2)
    r = ctx.rope(*p, axes=2)
    pos = (torch.rand(rows, 2, dtype=torch.float64, generator=torch.Generator().manual_seed(rows)) * 100).cuda()
    exponents = [62, 64, 90, 122, 127] + ([-60, -75, -110] if eps < 1e-30 else [])
    q, k = far(tensors(mode, rows, heads), 1, exponents), far(tensors(mode, rows, kv_heads, 1), 2, exponents)
    wq, wk = weights(heads), weights(kv_heads, 6)
    qo, ko = torch.full_like(q, 7), torch.full_like(k, 7)
    ctx.qk_rope(r, pos, q, qo, k, ko, wq, wk, eps=eps, mode=MODES[mode][0])
    check(qo, *expected(p, pos, q, wq, eps, q.dtype))
    check(ko, *expected(p, pos, k, wk, eps, k.dtype))
    # ordinary rows have the bits that they have among ordinary ones, and those of one normed alone
    z, w = torch.full_like(q, 7), torch.full_like(k, 7)
    plain = far(tensors(mode, rows, heads), 1, [0]), far(tensors(mode, rows, kv_heads, 1), 2, [0])
    ctx.qk_rope(r, pos, *(t for pair in zip(plain, (z, w)) for t in pair), wq, wk, eps=eps, mode=MODES[mode][0])
    for got, want, x, y in ((qo, z, q, plain[0]), (ko, w, k, plain[1])):
        same = (x == y).all(1)
        assert bool(same.any()) and torch.equal(got[same], want[same])
