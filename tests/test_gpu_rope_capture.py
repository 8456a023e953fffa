"""Plans of rotary positions made and freed while a call with another one is captured."""
import pytest

from conftest import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from ltx_amd import runtime as rt  # noqa: E402
from test_gpu_rope import check, expected, plan, tensors, weights  # noqa: E402


def test_a_plan_made_inside_a_capture():
    """The graph is whole, and the plan turns what it should, in a graph of its own too."""
    say("qk_rope plan made inside a capture")
    c = rt.Context(0)
    try:
        p, other = plan(4, 3), plan(8, 2)
        r, gone = c.rope(*p, axes=3), c.rope(*other, axes=2)
        q, w = tensors("f32", 70, 8), weights(8)
        pos = torch.rand(70, 3, dtype=torch.float64, device="cuda") * 50
        want, out, out2 = (torch.zeros_like(q) for _ in range(3))
        c.qk_rope(r, pos, q, want, q_norm=w, mode=rt.MODE_F32)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, capture_error_mode="global"):
            c.qk_rope(r, pos, q, out, q_norm=w, mode=rt.MODE_F32)
            made = c.rope(*other, axes=2)
            gone.free()
            c.qk_rope(made, pos[:, :2].contiguous(), q, out2, mode=rt.MODE_F32)
        for _ in range(3):
            out.zero_()
            out2.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            check(out2, *expected(other, pos[:, :2], q, None, 0.0, torch.float32))
            c.qk_rope(made, pos[:, :2].contiguous(), q, out2, mode=rt.MODE_F32)
            check(out2, *expected(other, pos[:, :2], q, None, 0.0, torch.float32))
    finally:
        c.close()
