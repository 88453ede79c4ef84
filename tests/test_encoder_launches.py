"""The encoder's launches, recorded on the CPU by a stand-in for the HIP runtime (tests/launches.py)."""

import json
import math
import os
import random
import subprocess
import sys

import pytest

from encoder_paths import GRAD, LINEAR, ORTHO

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    """launches([name, arguments], ...): the answers to these calls, made in a process of their own. launches.held: the
    product kernels that the library holds."""
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    recorder = str(tmp_path_factory.mktemp("recorder") / "liblaunch_recorder.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__", f"-I{rocm}/include",
                    os.path.join(HERE, "cpp", "launch_recorder.cc"), "-o", recorder], check=True)

    def run(*calls):
        p = subprocess.run([sys.executable, os.path.join(HERE, "launches.py"), recorder], input=json.dumps(calls),
                           capture_output=True, text=True)
        assert p.returncode == 0, p.stderr
        run.held, answers = json.loads(p.stdout)
        return answers

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


# ---- the kernels that the shapes of test_encoder_paths_gpu.py take ------------------------------


def _products(answers):
    return {kernel for a in answers for kernel in _kernels(a) if kernel.startswith("gemm_kernel")}


def _calls(dtype):
    for act in ("gelu", "none"):
        for name, shapes in (("linear", LINEAR[dtype]), ("linear_grad", GRAD[dtype])):
            for m, k, n in shapes:
                yield [name, dict(m=m, k=k, n=n, dtype=dtype, act=act)]


def _any_calls(rng, count, dtype):
    """Layers and gradients over all sizes, half of the rows in whole 16-byte pieces, some not aligned to them."""
    size = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    for _ in range(count):
        whole = rng.choice([1, 8])
        m, k, n = size(1, 200_000), size(1, 20_000), size(1, 20_000)
        args = dict(m=m, k=max(whole, k // whole * whole), n=max(whole, n // whole * whole), dtype=dtype,
                    act=rng.choice(["none", "gelu"]))
        if args["m"] * max(args["n"], args["k"]) < 1 << 32:
            yield ["linear", dict(args, offset=rng.choice([0, 0, 1]))]
            yield ["linear_grad", dict(args, inputs=rng.random() < 0.8, weight=rng.random() < 0.8)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_tested_shapes_take_every_product_kernel(launches, dtype):
    tested = _products(launches(*_calls(dtype)))
    taken = _products(launches(*_any_calls(random.Random(3), 6000, dtype)))
    assert taken <= tested, sorted(taken - tested)


def test_tested_orthogonalisations_take_every_product_kernel(launches):
    tested = _products(launches(*(["orthogonalize", dict(m=m, n=n, batch=b, steps=2)] for m, n, b in ORTHO)))
    rng = random.Random(4)
    size = lambda hi: int(round(math.exp(rng.uniform(0, math.log(hi)))))  # noqa: E731
    batch = lambda: rng.choice([1, 1, 2, 6, 12, size(200)])  # noqa: E731
    taken = _products(launches(*(["orthogonalize", dict(m=size(16384), n=size(16384), steps=2, batch=batch())]
                                 for _ in range(6000))))
    assert taken <= tested, sorted(taken - tested)


def test_every_product_kernel_is_taken_by_a_call(launches):
    """Nothing is built that no call reaches."""
    calls = [c for dtype in ("bf16", "fp32") for c in _calls(dtype)]
    calls += [["orthogonalize", dict(m=m, n=n, batch=b, steps=2)] for m, n, b in ORTHO]
    taken = _products(launches(*calls))
    assert set(launches.held) == taken, sorted(set(launches.held) - taken)


def test_fp16_goes_as_bf16_does(launches):
    """The shapes that are listed for bf16 take the same kernels in fp16."""
    calls = list(_calls("bf16"))
    half = [[name, dict(args, dtype="fp16")] for name, args in calls]
    assert [_kernels(a) for a in launches(*half)] == [_kernels(a) for a in launches(*calls)]


def test_special_values_meet_operands_in_parts(launches):
    """The shapes of the tests of infinities, tiny and huge values in fp32, forwards and backwards."""
    layer, grad = launches(["linear", dict(m=2100, k=520, n=2050)], ["linear_grad", dict(m=2100, k=520, n=2050, act="silu")])
    assert all("planes 3" in kernel for kernel in _products([layer]) | _products([grad]))


# ---- sizes past one launch ----------------------------------------------------------------------


def test_the_largest_matrix_is_orthogonalised(launches):
    for steps in (0, 1):
        answer, = launches(["orthogonalize", dict(m=65536, n=65536, steps=steps)])
        assert _kernels(answer)


@pytest.mark.parametrize("name,args", [("linear", dict(m=2**31 - 1, k=1, n=1, dtype="bf16")),
                                       ("linear", dict(m=2**31 - 1, k=8, n=8, dtype="fp32")),
                                       ("linear_grad", dict(m=2**31 - 1, k=2, n=2, dtype="bf16"))])
def test_products_past_one_launch_are_refused(launches, name, args):
    """With the status of a wrong argument and words for it, before anything runs."""
    answer, = launches([name, args])
    assert answer["status"] == -22 and "too large" in answer["error"] and not answer["launches"]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("dim,count", [(1024, 80_000_000), (25, 2**31 - 1), (64, 2**31 - 1), (32_768, 1_500_000)])
def test_embed_of_very_many_tokens(launches, dim, count, dtype):
    answer, = launches(["embed", dict(rows=1000, dim=dim, count=count, dtype=dtype)])
    names = _kernels(answer)
    width = 4 if dtype == "fp32" else 8
    threads = sum(grid * block for _, grid, _, block, _, _ in answer["launches"])
    assert all(n.startswith("embed_kernel") for n in names) and 2 * threads >= count * -(-dim // width)


@pytest.mark.parametrize("rows,dim,count", [(2**30 + 70, 1, 10), (2**30 + 70, 1, 0), (2**32 - 2, 1, 5000), (2**31, 30, 100_000)])
def test_embed_grad_of_very_many_rows(launches, rows, dim, count):
    """Every row is cleared or written, in launches that the runtime takes."""
    answer, = launches(["embed_grad", dict(rows=rows, dim=dim, count=count, dtype="bf16")])
    assert "embed_grad_sum_kernel" in _kernels(answer)


# ---- the caller's device ------------------------------------------------------------------------


@pytest.mark.parametrize("name,args", [
    ("get_device", {}), ("embed", dict(rows=100, dim=64, count=10)), ("embed_grad", dict(rows=100, dim=64, count=9000)),
    ("embed_grad", dict(rows=100, dim=64, count=10)), ("linear", dict(m=3, k=64, n=64)), ("linear", dict(m=3000, k=640, n=640)),
    ("linear_grad", dict(m=300, k=64, n=64)), ("orthogonalize", dict(m=64, n=64)), ("orthogonalize", dict(m=640, n=640)),
    ("linear", dict(m=2**31 - 1, k=64, n=64))])
def test_the_callers_device_stays(launches, name, args):
    """The kernels run on the library's device (0), and the caller's current one (1) is the same after the call, a refused
    one too."""
    answer, = launches([name, args])
    assert answer["device"] == [1, 1]
    assert all(launch[5] == 0 for launch in answer["launches"])


# ---- what goes past the L2s ---------------------------------------------------------------------


@pytest.mark.parametrize("dtype,dim,count,kernel", [
    ("bf16", 9, 1_050_000, "8 x 2"), ("bf16", 9, 1_900_000, "8 x 2 past"), ("bf16", 1, 2_200_000, "1 x 2"),
    ("fp32", 100, 80_000, "4 x 1"), ("fp32", 100, 84_000, "4 x 2 past"), ("fp32", 5, 1_100_000, "4 x 2"),
    ("fp32", 5, 1_700_000, "4 x 2 past"), ("bf16", 768, 24, "8 x 1"), ("bf16", 1024, 60_000, "8 x 2 past"),
    ("fp32", 3, 20_000_000, "2 x 2")])
def test_embed_stores_large_results_past_the_caches(launches, dtype, dim, count, kernel):
    """By the result's bytes (32 MB), where its pieces are of 16 bytes."""
    answer, = launches(["embed", dict(rows=1000, dim=dim, count=count, dtype=dtype)])
    assert _kernels(answer) == ["embed_kernel " + kernel]


def test_large_results_of_any_width_go_past_the_caches(launches):
    """A layer's, where it takes the largest tile whole: also with rows that end anywhere."""
    for n in (920, 917):
        answer, = launches(["linear", dict(m=27437, k=200, n=n, dtype="bf16", act="gelu", bias=True, residual=True, keep=True)])
        assert _kernels(answer) == ["gemm_kernel rr 256x256 depth 64 planes 1 loads 16 streamed"]
