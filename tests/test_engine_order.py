"""The Llama engine's and the Sim's copies and kernels are ordered on their own
streams: run on the CPU over a runtime whose legacy-stream copies arrive as late
as CUDA allows (tests/engine_on_host.cc). No device calls."""

import subprocess

import pytest

from tests.conftest import ROOT


@pytest.fixture(scope="module")
def engine_on_host(tmp_path_factory):
    exe = tmp_path_factory.mktemp("engine") / "engine_on_host"
    csrc = ROOT / "accelep_b200" / "csrc"
    # Kernels that no case reaches stay unresolved.
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'include'}", f"-I{csrc}", "-I/usr/local/cuda/include",
                    str(ROOT / "tests" / "engine_on_host.cc"), str(csrc / "llama.cc"), str(csrc / "sim_api.cc"),
                    "-no-pie", "-Wl,--unresolved-symbols=ignore-all", "-pthread", "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    return exe


@pytest.mark.parametrize("case", ["cache_rows", "weights", "int8_weights", "sim_upload"])
def test_copies_arrive_before_the_kernels_that_read_them(engine_on_host, case):
    out = subprocess.run([str(engine_on_host), case], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout
