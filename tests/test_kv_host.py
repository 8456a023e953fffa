"""The 4-bit cache and linear without a GPU: refusals, workspaces and routes on the
recording stand-in for the HIP runtime (tests/host/fake_hip.hpp), the kernels' index
arithmetic on arrays of any contents, and the Python entry points' own checks."""
import pathlib
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent
PKG = ROOT / "ltx-zml_amd"


@pytest.fixture(scope="session")
def kv_paths(tmp_path_factory):
    exe = tmp_path_factory.mktemp("kv") / "kv_paths"
    subprocess.run(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-Wno-unused-result", "-rdynamic",
                    "-I/opt/rocm/include", f"-I{ROOT / 'include'}", f"-I{PKG / 'csrc'}", f"-I{PKG / 'csrc' / 'host'}",
                    str(ROOT / "tests" / "host" / "kv_paths.cpp"), "-o", str(exe), str(PKG / "libltx_amd.so"),
                    f"-Wl,-rpath,{PKG}", "-Wl,--allow-shlib-undefined", "-pthread"], check=True)

    def run(*args):
        r = subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout + r.stderr
    return run


def test_refusals(kv_paths):
    kv_paths("refusals")


def test_attention_scratch(kv_paths):
    kv_paths("scratch")


def test_cache_memory(kv_paths):
    kv_paths("memory")


def test_cache_made_inside_a_capture_of_its_context(kv_paths):
    kv_paths("own_capture")


def test_faults_beside_a_capture(kv_paths):
    kv_paths("faults_beside_a_capture")


def test_faults_are_not_lost(kv_paths):
    kv_paths("faults_are_not_lost")


def test_one_workspace_for_both_forms(kv_paths):
    kv_paths("workspace_forms")


def test_tiles_of_calls_that_cannot_split(kv_paths):
    kv_paths("unsplit_tiles")


def test_row_limit(kv_paths):
    kv_paths("row_limit")


def test_alignment_of_the_batch(kv_paths):
    kv_paths("alignment")


def test_linear_forms(kv_paths):
    kv_paths("linear_forms")


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_index_arithmetic_stays_inside(kv_paths, seed):
    kv_paths("index", seed)


def test_python_checks():
    """What the bindings refuse before a call: shapes, types and strides that the
    C interface cannot see."""
    torch = pytest.importorskip("torch")
    from ltx_amd import runtime as rt

    i32 = dict(dtype=torch.int32)
    lens, pages = torch.zeros(3, **i32), torch.zeros(3, 4, **i32)
    b = rt.KvBatch(lens, pages, torch.zeros(4, **i32), 7)
    assert (b.args.nseq, b.args.rows, b.args.max_pages) == (3, 7, 4)
    assert rt.KvBatch(lens, pages).rows == 3
    for bad in [(lens.long(), pages), (lens, pages[:2]), (lens, pages.T.contiguous().T), (lens, pages, lens, 7),
                (lens, pages, torch.zeros(4, **i32))]:
        with pytest.raises(rt.LtxError):
            rt.KvBatch(*bad)

    class Ctx:
        device = -1  # the tensors' here: the CPU

    class Cache:
        kv_heads, mode, handle, ctx = 2, rt.MODE_F16, 0, Ctx
    good = torch.zeros(7, 256, dtype=torch.float16)
    rt._rows("x", b, Cache, 2, good, torch.zeros(7, 768, dtype=torch.float16)[:, 256:512])
    for bad in [good[:6], good[:, :128], good.bfloat16(), torch.zeros(256, 7, dtype=torch.float16).T, good[0]]:
        with pytest.raises(rt.LtxError):
            rt._rows("x", b, Cache, 2, bad)
    Ctx.device = 0
    with pytest.raises(rt.LtxError, match="device"):
        rt._rows("x", b, Cache, 2, good)


def test_stream_of_the_contexts_device(monkeypatch):
    """Without a stream a call takes the current stream of the context's device, which
    need not be the current one; also on a torch without the raw handle's call."""
    torch = pytest.importorskip("torch")
    import types

    from ltx_amd import runtime as rt

    seen = []

    def faults(ctx, cache, st, n, reset):
        seen.append(st)
        return 1
    monkeypatch.setattr(rt, "_lib", types.SimpleNamespace(ltx_kv_cache_faults=faults, ltx_kv_cache_free=lambda *a: None,
                                                          ltx_block_graph_launch=lambda h, st: seen.append(st) or 1,
                                                          ltx_block_graph_destroy=lambda h: None))
    ctx = rt.Context.__new__(rt.Context)
    ctx.handle, ctx.device = 1, 3
    cache, graph = rt.KvCache(ctx, 2, 1, 1, rt.MODE_F16), rt.BlockGraph(ctx, 2, ())
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 1000 + device, raising=False)
    assert cache.faults() == 0
    graph.launch()
    assert seen == [1003, 1003]
    monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream")
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=2000 + device))
    cache.faults()
    graph.launch()
    assert seen[2:] == [2003, 2003]
    cache.faults(stream=types.SimpleNamespace(cuda_stream=5))
    assert seen[4:] == [5]
