"""Norm and rotary positions as an operator against the block forward's own q and k.

What the forward's norm reads (the projections, formed here in f64 from the norm_msa stage
and the weights) goes through ltx_op_qk_rope with the block's plan and norm weights; the
result is the Q1 and K1 stage. In f32 both are within the stages' gate, 1e-5 relative RMS. In
f16 each side rounds the projections (a sum apart in its last bits may round the other way: a
step, 2^-10 of the value) and its result (half a step each, 2^-11; the stage's is scaled
before): at most 4 x 2^-11 = 2e-3, the stages' gate too."""
import numpy as np
import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import blockcases  # noqa: E402
import oracle  # noqa: E402
from ltx_amd import runtime as rt  # noqa: E402
from ltx_amd import synth  # noqa: E402
from test_gpu_stages import GATE, TORCH_DT, D, dev, forward, stage  # noqa: E402


@pytest.mark.parametrize("mode", ["f16", "f32"])
@pytest.mark.parametrize("T", [256, 250])
def test_the_forwards_q_and_k(ctx, block0, mode, T):
    say(f"qk_rope against the block's stages {mode} T={T}")
    inp = synth.make_inputs(T, 64, sigma=0.7)
    cos, sin = rt.rope_tables(inp["grid"])
    w = ctx.upload(block0)
    forward(ctx, w, inp, cos, sin, mode)
    dt, f32 = TORCH_DT[mode], mode == "f32"
    x = dev(stage(ctx, "norm_msa", dt, (T, D)))
    want = {"q1": stage(ctx, "q1", dt, (T, D)) / (1.0 if f32 else rt.ATTN_C), "k1": stage(ctx, "k1", dt, (T, D))}
    w.free()
    # (f64, then the type the forward holds its projections in)
    pre = [(x @ dev(blockcases.weight64(block0, f"{n}_w")).T + dev(blockcases.bias64(block0, f"{n}_b"))).to(dt) for n in want]
    norm = [dev(blockcases.bias64(block0, f"{n[0]}n1")).float() for n in want]
    pos = dev(inp["grid"].astype(np.float64).mean(2).T)
    out = [torch.empty_like(t) for t in pre]
    ctx.qk_rope(ctx.rope_grid(), pos, pre[0], out[0], pre[1], out[1], *norm, eps=1e-6, mode=rt.MODES[mode])
    for n, y in zip(want, out):
        r = oracle.rel_rms(y.double().cpu().numpy(), want[n])
        say(f"  {n} {r:.2e}")
        assert r <= GATE[mode], (n, r)
