"""Types and shapes that the bindings of the microscaled 4-bit operands take, without a GPU."""
import pytest

torch = pytest.importorskip("torch")

from ltx_amd import runtime as rt  # noqa: E402

CODES = [t for t in (torch.uint8, getattr(torch, "float4_e2m1fn_x2", None)) if t]
SCALES = [t for t in (torch.uint8, getattr(torch, "float8_e8m0fnu", None)) if t]
CPU = -1  # where tensors of the host say they are


def held(rows=3, K=256):
    return torch.zeros(rows, K // 2, dtype=torch.uint8), torch.zeros(K // 128, rows, 4, dtype=torch.uint8)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("scales", SCALES)
def test_types_of_these_bytes_are_taken(codes, scales):
    q, s = held()
    rt._mx4_held("test", q.view(codes), s.view(scales), 3, 256, CPU)


def test_other_types_and_shapes_are_refused():
    q, s = held()
    other = [torch.float8_e4m3fn, torch.float8_e5m2]
    bad = [(q.view(t), s) for t in other + SCALES[1:]] + [(q, s.view(t)) for t in other + CODES[1:]]
    bad += [(q.to(torch.int16), s), (q, s.float()), (q[:, :64], s), (q[:2], s), (q, s[:1]), (q, s.transpose(0, 1)),
            (q.T.contiguous().T, s)]
    for q1, s1 in bad:
        with pytest.raises(rt.LtxError, match="are needed"):
            rt._mx4_held("test", q1, s1, 3, 256, CPU)
    with pytest.raises(rt.LtxError, match="device"):
        rt._mx4_held("test", q, s, 3, 256, 0)
    with pytest.raises(rt.LtxError, match="128"):
        rt._mx4_held("test", q, s, 3, 192, CPU)
