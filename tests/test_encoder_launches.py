"""The encoder's launches, recorded on the CPU by a stand-in for the HIP runtime (tests/launches.py)."""

import json
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    """launches([name, arguments], ...): the answers to these calls, made in a process of their own."""
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    recorder = str(tmp_path_factory.mktemp("recorder") / "liblaunch_recorder.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__", f"-I{rocm}/include",
                    os.path.join(HERE, "cpp", "launch_recorder.cc"), "-o", recorder], check=True)

    def run(*calls):
        p = subprocess.run([sys.executable, os.path.join(HERE, "launches.py"), recorder], input=json.dumps(calls),
                           capture_output=True, text=True)
        assert p.returncode == 0, p.stderr
        return json.loads(p.stdout)

    return run


def _kernels(answer):
    assert answer["status"] == 0, answer["error"]
    return [launch[0] for launch in answer["launches"]]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,dim", [(30, 50), (300_000, 100), (250_000, 128), (1_183_514, 100), (1_000_000, 1)])
def test_embed_grad_without_tokens_clears_the_rows(launches, rows, dim, dtype):
    """One launch that writes zeros, whichever way a batch of that size would take."""
    answer, = launches(["embed_grad", dict(rows=rows, dim=dim, count=0, dtype=dtype)])
    kernel, = _kernels(answer)
    grid = answer["launches"][0][1]
    assert kernel == "embed_grad_own_kernel" or (kernel == "embed_grad_sum_kernel" and grid * 64 >= rows)
