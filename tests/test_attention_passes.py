"""The memory of linear attention's passes: what the launches are given, recorded on the CPU (tests/attention_passes.py)."""

import itertools
import json
import os
import subprocess
import sys

import pytest

from attention_passes import WORK

HERE = os.path.dirname(os.path.abspath(__file__))
WIDTHS = (16, 64, 65, 128, 200, 256)
TEXTS = (1, 3, 16, 24, 32, 48, 63, 64, 96, 128, 192, 256)


@pytest.fixture(scope="module")
def passes(tmp_path_factory):
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    recorder = str(tmp_path_factory.mktemp("recorder") / "liblaunch_recorder.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__", f"-I{rocm}/include",
                    os.path.join(HERE, "cpp", "launch_recorder.cc"), "-o", recorder], check=True)

    def run(calls):
        p = subprocess.run([sys.executable, os.path.join(HERE, "attention_passes.py"), recorder], input=json.dumps(calls),
                           capture_output=True, text=True)
        assert p.returncode == 0, p.stderr
        return list(zip(calls, json.loads(p.stdout)))

    return run


def _check(call, answer):
    """Every launch's passes keep their segments' states inside the workspace, apart from one another's and from what shared heads'
    gradients take; those of one text's length need none, and take no part in the launches that make them."""
    _, args = call
    assert answer["status"] == 0, (args, answer["error"])
    assert answer["launches"], args
    for kernel, of in answer["launches"]:
        makes = kernel.startswith("attention_scan") or kernel.split()[3] == "1"  # the states
        spans = []
        for p in of:
            # The arguments are read as they are laid out.
            assert (p["tokens"], p["batch"], p["heads"]) == (args["tokens"], args["batch"], args["heads"]), args
            assert sorted((p["dk"], p["dv"])) == sorted((args["dk"], args["dv"])), args
            assert (p["segments"] - 1) * p["segment"] < p["tokens"] <= p["segments"] * p["segment"], args
            if makes or p["segments"] > 1:
                spans.append((p["states"], p["states"] + 4 * p["segments"] * p["batch"] * p["heads"] * p["dk"] * p["dv"]))
            if p["parts"]:
                spans.append((p["parts"], p["parts"] + 4 * p["batch"] * p["tokens"] * p["heads"] * p["dv"]))
        spans.sort()
        assert all(WORK <= a and b <= WORK + answer["workspace"] for a, b in spans), (args, kernel, of, answer["workspace"])
        assert all(x[1] <= y[0] for x, y in zip(spans, spans[1:])), (args, kernel, of)


def _cuts(answer):
    return {p["segments"] for p in answer["launches"][-1][1]}


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("tokens", [449, 1_100, 4_096])
def test_states_of_every_pass_lie_in_the_workspace(passes, dtype, tokens):
    calls = [[name, dict(batch=n // h, tokens=tokens, heads=h, kv_heads=h // share, dk=dk, dv=dv, dtype=dtype, state=state)]
             for n in TEXTS for h, share in ((1, 1), (4, 2)) if n % h == 0 for dk, dv in itertools.product(WIDTHS, WIDTHS)
             for state in (False, True) for name in ("attention", "attention_grad")]
    cuts = []
    for call, answer in passes(calls):
        _check(call, answer)
        cuts.append(_cuts(answer))
    # Some cut alike, some differently, some only in part.
    assert {1} in cuts and any(len(c) == 1 and 1 not in c for c in cuts) and any(len(c) > 1 and 1 in c for c in cuts)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_states_where_one_tensors_rows_lie_far_apart(passes, dtype):
    """The passes look at three tensors of four each, and are cut by them where nothing else cuts them."""
    calls = [["attention_grad", dict(batch=n, tokens=20_000, heads=4, kv_heads=share, dk=dk, dv=dv, dtype=dtype, state=state, apart={name: 2**16})]
             for n in (1, 20, 100) for share in (4, 1) for dk, dv in ((64, 64), (128, 128), (64, 200)) for state in (False, True)
             for name in ("q", "k", "v", "grad")]
    cuts = []
    for call, answer in passes(calls):
        _check(call, answer)
        cuts.append(_cuts(answer))
    assert any(len(c) > 1 and 1 in c for c in cuts)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("batch,tokens,heads,dk,dv", [(65_536, 1_000, 1, 8, 8), (2**19, 70, 4, 1, 1), (65_535, 250_000, 1, 8, 8),
                                                      (2**21, 2_000, 1, 16, 16), (16_000, 16_000, 4, 8, 200)])
def test_many_texts_whose_rows_lie_far_apart_are_taken(passes, dtype, batch, tokens, heads, dk, dv):
    """Texts next to one another within a token, so many that no launch holds their segments: whole texts, by ordinary loads where no buffer holds one."""
    shape = dict(batch=batch, tokens=tokens, heads=heads, kv_heads=heads, dk=dk, dv=dv, dtype=dtype, state=True, by_token=True)
    for call, answer in passes([["attention", shape], ["attention_grad", shape]]):
        _check(call, answer)
        (kernel, _), = answer["launches"]
        assert kernel.startswith("attention_kernel") and kernel.endswith(" 0") or tokens == 1_000, call
