"""Microscaled 4-bit operands, rotary positions and windowed attention without a GPU:
refusals, scratch and routes on the recording stand-in for the HIP runtime
(tests/host/fake_hip.hpp), and the window's index arithmetic."""
import pathlib
import re
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent
PKG = ROOT / "ltx-zml_amd"


@pytest.fixture(scope="session")
def paths(tmp_path_factory):
    exe = tmp_path_factory.mktemp("stream") / "stream_paths"
    subprocess.run(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-Wno-unused-result", "-rdynamic",
                    "-I/opt/rocm/include", f"-I{ROOT / 'include'}", f"-I{PKG / 'csrc'}", f"-I{PKG / 'csrc' / 'host'}",
                    str(ROOT / "tests" / "host" / "stream_paths.cpp"), "-o", str(exe), str(PKG / "libltx_amd.so"),
                    f"-Wl,-rpath,{PKG}", "-Wl,--allow-shlib-undefined", "-pthread"], check=True)

    def run(*args):
        r = subprocess.run([str(exe), *map(str, args)], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout + r.stderr
        return r.stdout.split()[:-1]
    return run


@pytest.mark.parametrize("what", ["mx4_refusals", "mx4_scratch", "rope_refusals", "rope_grid", "window_refusals"])
def test_calls(paths, what):
    paths(what)


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_pages_of_a_window(paths, seed):
    paths("window_index", seed)


def test_kernels_that_are_selected_are_those_that_are_built(paths):
    """Over the ranges of sizes and types: every kernel that a call takes is in the library,
    and every one that is built is taken."""
    taken = set(paths("kernels"))
    built = set(re.findall(rb"\n?(ltx_(?:gemm_mx4|linear_mx4|mx4|qk_rope|kv_attn|kv_join)_[a-z0-9_]+)\.kd",
                           (PKG / "libltx_amd.so").read_bytes()))
    built = {n.decode() for n in built}
    assert taken <= built, sorted(taken - built)
    new = {n for n in built if not n.startswith(("ltx_kv_",)) or "_win" in n}
    assert new <= taken, sorted(new - taken)
