"""Scratch of the microscaled 4-bit linear without a GPU (tests/host/fake_hip.hpp): both sides
of the size from which a call takes it, and a call that gets none."""
import pathlib
import subprocess

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent
PKG = ROOT / "ltx-zml_amd"


@pytest.fixture(scope="module")
def paths(tmp_path_factory):
    exe = tmp_path_factory.mktemp("mx4_scratch") / "mx4_scratch_paths"
    subprocess.run(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-Wno-unused-result", "-rdynamic",
                    "-I/opt/rocm/include", f"-I{ROOT / 'include'}", f"-I{PKG / 'csrc'}", f"-I{PKG / 'csrc' / 'host'}",
                    str(ROOT / "tests" / "host" / "mx4_scratch_paths.cpp"), "-o", str(exe), str(PKG / "libltx_amd.so"),
                    f"-Wl,-rpath,{PKG}", "-Wl,--allow-shlib-undefined", "-pthread"], check=True)

    def run(*args):
        r = subprocess.run([str(exe), *args], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0 and r.stdout == "ok\n", r.stdout + r.stderr
    return run


@pytest.mark.parametrize("what", ["threshold", "no_memory", "captured"])
def test_scratch(paths, what):
    paths(what)
