"""Norm and rotary positions on several axes on the GPU against 64 bits.

The bound, with u = eps / 2 of the type and e = 2^-24:
  - cos and sin are off by at most 2^-21: what is left of an angle after whole quarters is
    below 0.8 and rounded twice (2 e of it), and the series are a handful of f32 operations
    on numbers below 1; the angle itself is off by 2^-50 of its size (f64, three roundings);
  - the norm: a sum of squares in f32, 16 additions a thread and 32 heads and ten to join
    them, a division, a root and a product: (16 ceil(heads / 32) + 20) e of the value;
  - a product with a weight, the rotation's two products and their sum: 4 e;
all relative to |x| + |y| of the pair (its normed values), and the output's u (2^-25 at
least in f16, 2^-134 in bf16)."""
import math

import numpy as np
import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ltx_amd import runtime as rt  # noqa: E402
from test_gpu_mx4 import streams  # noqa: E402

MODES = {"f16": (rt.MODE_F16, torch.float16), "bf16": (rt.MODE_BF16, torch.bfloat16),
         "f32": (rt.MODE_F32, torch.float32)}
E = 2.0 ** -24


def plan(heads, axes, seed=0, top=1.0):
    r = np.random.default_rng(seed + heads + axes)
    freq = top * 10000.0 ** -r.uniform(0, 1, (heads, 64))
    return freq, r.uniform(-3, 3, (heads, 64)), r.integers(0, axes, (heads, 64)).astype(np.int32)


def expected(p, pos, x, w, eps, dt):
    """f64 values and the bound, [rows, heads * 128]."""
    freq, phase, axis = p
    pos = pos.cpu().numpy()
    v = x.double().cpu().numpy()
    rows, heads = v.shape[0], v.shape[1] // 128
    rel = 4 * E
    if w is not None:
        v = v / np.sqrt((v * v).mean(1, keepdims=True) + eps) * w.double().cpu().numpy()
        rel += (16 * -(-heads // 32) + 20) * E
    angle = pos[:, axis] * freq + phase  # [rows, plan heads, 64]
    far = 2.0 ** -50 * (np.abs(pos[:, axis] * freq) + np.abs(phase))
    angle, far = (t.repeat(heads // freq.shape[0], 1) for t in (angle, far))
    v = v.reshape(rows, heads, 2, 64)
    a, b, c, s = v[:, :, 0], v[:, :, 1], np.cos(angle), np.sin(angle)
    out = np.stack([a * c - b * s, b * c + a * s], 2)
    size = (np.abs(a) + np.abs(b)) * (rel + 2.0 ** -21 + far)
    least = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dt]
    tol = np.stack([size, size], 2) * (1 + torch.finfo(dt).eps) + torch.finfo(dt).eps / 2 * np.abs(out) + least
    return out.reshape(rows, -1), tol.reshape(rows, -1)


def check(y, want, tol):
    got = y.double().cpu().numpy()
    ok = np.abs(got - want) <= tol
    assert ok.all(), (int((~ok).sum()), float((np.abs(got - want) / tol).max()))


def tensors(mode, rows, heads, seed=0, wide=0):
    g = torch.Generator().manual_seed(seed + rows + heads)
    x = torch.randn(rows, 128 * heads + wide, generator=g) * torch.exp(0.5 * torch.randn(128 * heads + wide, generator=g))
    return x.to(MODES[mode][1]).cuda()[:, wide // 2:wide // 2 + 128 * heads]


def weights(heads, seed=5):
    return 1 + 0.3 * torch.randn(128 * heads, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("mode", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,heads,kv_heads,plan_heads,axes,norm", [
    (1, 32, 32, 32, 3, True),
    (1, 1, 1, 1, 1, False),
    (7, 32, 8, 8, 3, True),
    (33, 32, 8, 1, 3, False),
    (5, 40, 5, 5, 2, True),
    (9, 96, 8, 4, 8, True),
    (64, 3, 0, 3, 1, True),
    (130, 4, 4, 1, 2, True),
    (300, 32, 32, 1, 3, False),
    (257, 8, 32, 4, 3, False),
    (20, 33, 33, 33, 1, True),
    (2100, 32, 32, 32, 3, True),
])
def test_norm_and_rotation(ctx, mode, rows, heads, kv_heads, plan_heads, axes, norm):
    say(f"qk_rope {mode} rows={rows} heads={heads}/{kv_heads}/{plan_heads} axes={axes} norm={norm}")
    p = plan(plan_heads, axes)
    r = ctx.rope(*p, axes=axes)
    pos = (torch.rand(rows, axes, dtype=torch.float64, generator=torch.Generator().manual_seed(rows)) * 2000 - 100).cuda()
    q, wq = tensors(mode, rows, heads, wide=32), weights(heads) if norm else None
    k, wk = (tensors(mode, rows, kv_heads, 1, 16), weights(kv_heads, 6) if norm else None) if kv_heads else (None, None)
    dt = q.dtype
    qo = torch.full((rows, 128 * heads + 8), 7.0, dtype=dt, device="cuda")
    ko = torch.full((rows, 128 * kv_heads + 8), 7.0, dtype=dt, device="cuda")
    ctx.qk_rope(r, pos, q, qo[:, :-8], k, ko[:, :-8] if kv_heads else None, wq, wk, eps=1e-3, mode=MODES[mode][0])
    check(qo[:, :-8], *expected(p, pos, q, wq, 1e-3, dt))
    assert bool((qo[:, -8:] == 7).all()) and bool((ko[:, -8:] == 7).all())
    if kv_heads:
        check(ko[:, :-8], *expected(p, pos, k, wk, 1e-3, dt))


@pytest.mark.parametrize("mode", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("norm", [(True, False), (False, True)])
def test_one_norm_in_place(ctx, mode, norm):
    """A norm of one of the two alone; outputs that are q and k themselves: the same bits."""
    say(f"qk_rope in place {mode} {norm}")
    p = plan(8, 3)
    r = ctx.rope(*p, axes=3)
    fused = tensors(mode, 50, 32 + 16)
    q, k = fused[:, :4096], fused[:, 4096:5120]
    rest = fused[:, 5120:].clone()
    wq, wk = weights(32) if norm[0] else None, weights(8, 6) if norm[1] else None
    pos = torch.rand(50, 3, dtype=torch.float64, device="cuda") * 30
    qo, ko = (torch.empty(t.shape, dtype=t.dtype, device="cuda") for t in (q, k))
    ctx.qk_rope(r, pos, q, qo, k, ko, wq, wk, mode=MODES[mode][0])
    check(qo, *expected(p, pos, q, wq, 1e-6, q.dtype))
    check(ko, *expected(p, pos, k, wk, 1e-6, q.dtype))
    ctx.qk_rope(r, pos, q, q, k, k, wq, wk, mode=MODES[mode][0])
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(fused[:, 5120:], rest)


def test_far_positions(ctx):
    """Angles of 10^9 and more, in f32: the same as near ones by the bound."""
    say("qk_rope far positions")
    p = plan(2, 2, top=1000.0)
    r = ctx.rope(*p, axes=2)
    pos = torch.tensor([[0.0, -0.0], [1.0, 1e6], [123456789.0, 2.0 ** 31 + 1], [-1e6, 1e-9], [1 / 3, -1e5 / 7]],
                       dtype=torch.float64, device="cuda")
    q = tensors("f32", 5, 4)
    out = torch.empty_like(q)
    ctx.qk_rope(r, pos, q, out, mode=rt.MODE_F32)
    check(out, *expected(p, pos, q, None, 0.0, torch.float32))


def test_quarter_turns_are_exact(ctx):
    say("qk_rope quarter turns")
    r = ctx.rope(np.full((1, 64), math.pi / 2))
    q = tensors("f32", 9, 1)
    out = torch.empty_like(q)
    ctx.qk_rope(r, torch.arange(-4.0, 5.0, dtype=torch.float64, device="cuda")[:, None], q, out, mode=rt.MODE_F32)
    for i, n in enumerate(range(-4, 5)):
        x, y = q[i, :64], q[i, 64:]
        want = [(x, y), (-y, x), (-x, -y), (y, -x)][n % 4]
        assert torch.equal(out[i], torch.cat(want))


def test_turned_back(ctx):
    """-pos turns back what pos has turned (no phases)."""
    say("qk_rope turned back")
    freq, _, axis = plan(4, 3)
    r = ctx.rope(freq, None, axis, axes=3)
    pos = torch.rand(40, 3, dtype=torch.float64, device="cuda") * 1000
    q = tensors("f32", 40, 8)
    out, back = torch.empty_like(q), torch.empty_like(q)
    ctx.qk_rope(r, pos, q, out, mode=rt.MODE_F32)
    ctx.qk_rope(r, -pos, out, back, mode=rt.MODE_F32)
    _, tol = expected((freq, 0 * freq, axis), pos, q, None, 0.0, torch.float32)
    size = np.abs(q.double().cpu().numpy()).reshape(40, 8, 2, 64).sum(2, keepdims=True).repeat(2, 2).reshape(40, -1)
    assert (np.abs((back - q).double().cpu().numpy()) <= 2 * tol + 2.0 ** -21 * size).all()


@pytest.mark.parametrize("mode", ["f16", "f32"])
def test_the_blocks_own_plan(ctx, mode):
    """ltx_rope_create_grid on midpoints against the tables of the block forward (f32 cos and
    sin: 2^-24 more)."""
    from ltx_amd import synth
    say(f"qk_rope grid {mode}")
    grid = synth.latent_grid(3, 4, 8)
    cos, sin = rt.rope_tables(grid)
    T = grid.shape[1]
    pos = torch.from_numpy(grid.astype(np.float64).mean(2).T.copy()).cuda()
    q, w = tensors(mode, T, 32), weights(32)
    out = torch.empty_like(q)
    ctx.qk_rope(ctx.rope_grid(), pos, q, out, None, None, w, mode=MODES[mode][0])
    v = q.double().cpu().numpy()
    v = (v / np.sqrt((v * v).mean(1, keepdims=True) + 1e-6) * w.double().cpu().numpy()).reshape(T, 32, 2, 64)
    a, b, c, s = v[:, :, 0], v[:, :, 1], cos.astype(np.float64), sin.astype(np.float64)
    want = np.stack([a * c - b * s, b * c + a * s], 2).reshape(T, -1)
    size = (np.abs(a) + np.abs(b)) * (40 * E + 2.0 ** -21 + 2.0 ** -50 * 16000 * 3 + E)
    tol = np.stack([size, size], 2).reshape(T, -1) * 1.001 + torch.finfo(q.dtype).eps / 2 * np.abs(want) + 2.0 ** -25
    check(out, want, tol)


def test_values_and_positions_that_are_not_finite(ctx):
    """A position touches the pairs on its axis, a value its pair (its row where that is
    normed), nothing else."""
    say("qk_rope not finite")
    p = plan(2, 2)
    r = ctx.rope(*p, axes=2)
    pos = torch.rand(6, 2, dtype=torch.float64, device="cuda")
    pos[1, 0], pos[2, 1] = math.nan, math.inf
    q, k = tensors("f32", 6, 2), tensors("f32", 6, 2, 3)
    q[3, 130] = math.nan
    k[4, 7] = math.inf
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    ctx.qk_rope(r, pos, q, qo, k, ko, None, weights(2), mode=rt.MODE_F32)
    axis = np.concatenate([p[2][0], p[2][0], p[2][1], p[2][1]])
    nan = np.zeros((6, 256), bool)
    nan[1], nan[2] = axis == 0, axis == 1
    bad_q, bad_k = nan.copy(), nan.copy()
    bad_q[3, [130, 194]] = True
    assert np.array_equal(torch.isnan(qo).cpu().numpy(), bad_q)
    got = torch.isnan(ko).cpu().numpy()
    assert np.array_equal(got[:4], bad_k[:4]) and np.array_equal(got[5], bad_k[5]) and got[4].any()


def test_captured_and_on_another_stream(ctx):
    say("qk_rope graph and stream")
    r = ctx.rope_grid()
    q, k, w = tensors("bf16", 70, 32), tensors("bf16", 70, 32, 1), weights(32)
    pos = torch.rand(70, 3, dtype=torch.float64, device="cuda")
    qo, ko = torch.zeros_like(q), torch.zeros_like(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.qk_rope(r, pos, q, qo, k, ko, w, w, mode=rt.MODE_BF16)
    st, = streams(1)
    for i in range(4):
        pos.copy_(torch.rand(70, 3, dtype=torch.float64, device="cuda") * 100 * i)
        ctx.qk_rope(r, pos, q, qo, k, ko, w, w, mode=rt.MODE_BF16)
        want = qo.clone(), ko.clone()
        for replay in (True, False):
            qo.zero_(), ko.zero_()
            torch.cuda.synchronize()
            graph.replay() if replay else ctx.qk_rope(r, pos, q, qo, k, ko, w, w, mode=rt.MODE_BF16, stream=st)
            torch.cuda.synchronize()
            assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])


def test_refusals(ctx):
    say("qk_rope refusals")
    for bad in [dict(freq=np.ones((1, 32))), dict(freq=np.full((1, 64), math.nan)), dict(axis=np.full((1, 64), 2)),
                dict(axis=np.full((1, 64), -1)), dict(axes=0), dict(axes=9), dict(phase=np.ones((2, 64))),
                dict(freq=np.ones((0, 64)))]:
        with pytest.raises(rt.LtxError):
            ctx.rope(**dict(dict(freq=np.ones((1, 64)), axes=2), **bad))
    r = ctx.rope(np.ones((4, 64)), None, np.ones((4, 64)), axes=2)
    q, k = tensors("f16", 6, 8), tensors("f16", 6, 4)
    pos = torch.zeros(6, 2, dtype=torch.float64, device="cuda")
    qo, ko = torch.full_like(q, 7), torch.full_like(k, 7)
    good = dict(rope=r, pos=pos, q=q, q_out=qo, k=k, k_out=ko)
    for bad in [dict(pos=pos.float()), dict(pos=pos[:5]), dict(pos=torch.zeros(6, 3, dtype=torch.float64, device="cuda")),
                dict(q=q[:, :768]), dict(q=q[:, :640], q_out=qo[:, :640]), dict(k=k[:, :256], k_out=ko[:, :256]),
                dict(q=q.float()), dict(k=None), dict(q_norm=weights(4)), dict(k_norm=weights(4).half()), dict(mode=1),
                dict(mode=7), dict(q_out=qo[:5]), dict(q=torch.empty(6, 1028, dtype=torch.float16, device="cuda")[:, 4:]),
                dict(q=q.cpu())]:
        with pytest.raises(rt.LtxError):
            ctx.qk_rope(**dict(good, **bad))
    assert bool((qo == 7).all()) and bool((ko == 7).all())
    ctx.qk_rope(r, pos[:0], q[:0], qo[:0], k[:0], ko[:0])
