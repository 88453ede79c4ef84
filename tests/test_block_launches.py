"""The blocks' launches, recorded on the CPU by a stand-in for the HIP runtime (tests/block_launches.py)."""

import json
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
TYPES = ("fp32", "fp16", "bf16")


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    recorder = str(tmp_path_factory.mktemp("recorder") / "liblaunch_recorder.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__", f"-I{rocm}/include",
                    os.path.join(HERE, "cpp", "launch_recorder.cc"), "-o", recorder], check=True)

    def run(*calls):
        p = subprocess.run([sys.executable, os.path.join(HERE, "block_launches.py"), recorder], input=json.dumps(calls),
                           capture_output=True, text=True)
        assert p.returncode == 0, p.stderr
        run.held, answers = json.loads(p.stdout)
        return answers

    return run


def _names(answer):
    assert answer["status"] == 0, answer["error"]
    return [launch[0] for launch in answer["launches"]]


# As test_blocks_gpu.py and test_attention_gpu.py have them.
DIMS = [1, 3, 5, 8, 31, 64, 100, 129, 256, 500, 768, 1000, 1024, 1025, 2000, 2051, 4096, 4099, 8192, 8200, 16_384]
SHAPES = [(1, 1, 64, 64), (3, 1, 64, 64), (4, 2, 128, 128), (2, 2, 16, 40), (1, 1, 1, 1), (6, 3, 33, 100), (2, 1, 200, 72),
          (1, 1, 256, 256), (2, 2, 72, 130)]


def _tested(dtype):
    calls = [[name, dict(rows=37, dim=dim, dtype=dtype, block=block, gate=gate)] for dim in DIMS for name in ("block_norm", "block_norm_grad")
             for block, gate in ((False, False), (True, False), (True, True))]
    calls += [[name, dict(batch=2, tokens=t, heads=s[0], kv_heads=s[1], dk=s[2], dv=s[3], dtype=dtype, state=bool(t % 2))]
              for s in SHAPES for t in (1, 7, 200, 1_537) for name in ("attention", "attention_grad")]
    return [*calls, ["clip", dict(sizes=[3, 5], dtype=dtype)], ["clip", dict(sizes=[3_000_001, 17_000_000], dtype=dtype)],
            ["clip", dict(sizes=[0], dtype=dtype)]]


def test_tested_shapes_take_every_kernel(launches):
    """No kernel is built that the tested shapes do not take. (1,537 tokens stand for the longer texts, which are of fewer shapes.)"""
    taken = {name for dtype in TYPES for answer in launches(*_tested(dtype)) for name in _names(answer)}
    assert taken == set(launches.held)


@pytest.mark.parametrize("dtype", TYPES)
def test_segments(launches, dtype):
    """Few heads over a long text are cut, many are not; results that need the last segment's state make it too."""
    few, state, many, grad = launches(["attention", dict(batch=1, tokens=32_768, heads=16, kv_heads=16, dk=64, dv=64, dtype=dtype)],
                                      ["attention", dict(batch=1, tokens=32_768, heads=16, kv_heads=16, dk=64, dv=64, dtype=dtype, state=True)],
                                      ["attention", dict(batch=32, tokens=4_096, heads=16, kv_heads=16, dk=64, dv=64, dtype=dtype)],
                                      ["attention_grad", dict(batch=2, tokens=4_096, heads=8, kv_heads=2, dk=64, dv=64, dtype=dtype)])
    kernel = f"attention_kernel {dtype} 64"
    assert _names(few) == [kernel + " 1 1", "attention_scan_kernel", kernel + " 0 1"] == _names(state)
    assert few["launches"][0][1] < state["launches"][0][1] == state["launches"][2][1]
    assert _names(many) == [kernel + " 0 1"] and many["workspace"] == 0
    assert [n.split()[0] for n in _names(grad)] == ["attention_kernel", "attention_scan_kernel", "attention_kernel"] + ["attention_shared_kernel"] * 2
    assert grad["launches"][0][2] == grad["launches"][2][2] == 3  # three passes in one launch


def test_rows_that_are_no_whole_pieces_are_loaded_by_elements(launches):
    shape = dict(batch=1, tokens=100, heads=2, kv_heads=2, dk=64, dv=64)
    whole, odd, shifted, far = launches(["attention", shape], ["attention", dict(shape, apart=1)], ["attention", dict(shape, offset=1)],
                                        ["attention", dict(shape, tokens=4_000, apart=2**22)])
    assert _names(whole)[-1].endswith(" 1") and all(_names(a)[-1].endswith(" 0") for a in (odd, shifted, far))


def test_rows_far_apart_are_cut_to_what_a_buffer_holds(launches):
    answer, = launches(["attention", dict(batch=200, tokens=60_000, heads=2, kv_heads=2, dk=64, dv=64, apart=2**16)])
    assert _names(answer)[-1].endswith(" 1")
    segments = answer["workspace"] // (200 * 2 * 64 * 64 * 4)
    assert segments > 1 and (60_000 / segments + 128) * 2**16 * 2 < 2**31


def test_long_lists_take_several_launches(launches):
    some, = launches(["clip", dict(sizes=[1000] * 290)])
    assert _names(some) == ["clip_norm_kernel"] * 3 + ["clip_scale_kernel 0"] * 3
    large, = launches(["clip", dict(sizes=[20_000_000] * 2)])
    assert _names(large) == ["clip_norm_kernel", "clip_scale_kernel 1"]
    parts = sum(launch[1] for launch in some["launches"][:3])
    assert parts * 8 <= some["workspace"]


@pytest.mark.parametrize("name,args", [
    ("block_norm", dict(rows=10, dim=64)), ("block_norm_grad", dict(rows=10, dim=64)), ("clip", dict(sizes=[10, 0, 7])),
    ("attention", dict(batch=1, tokens=3, heads=2, kv_heads=1, dk=32, dv=32)),
    ("attention", dict(batch=1, tokens=3_000, heads=2, kv_heads=1, dk=32, dv=32, state=True)),
    ("attention_grad", dict(batch=1, tokens=3_000, heads=2, kv_heads=1, dk=32, dv=32))])
def test_the_callers_device_stays(launches, name, args):
    answer, = launches([name, args])
    assert answer["device"][0] == answer["device"][1] != 0
    assert answer["launches"] and all(launch[4] == 0 for launch in answer["launches"])
