"""What the encoder's calls launch, by their C entry points, in a process without a GPU.

    python tests/launches.py RECORDER < calls > launches

Both are JSON. A call is [name, {argument: value}]. Out come the names of all product kernels that the library
holds, and an answer to each call: the status, the error's text, the workspace's size, the current device
before and after, and the launches as [kernel, grid x, grid y, threads, LDS bytes, device]. RECORDER is
tests/cpp/launch_recorder.cc, compiled. Buffers are made-up addresses: nothing reads them.
"""

from __future__ import annotations

import ctypes as C
import itertools
import json
import os
import re
import sys

LIB = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "quiver_amd", "lib", "libqvh.so")
BUF = 1 << 20
TYPES = {"fp32": 0, "fp16": 1, "bf16": 2}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


class LinearArgs(C.Structure):
    _fields_ = [("m", C.c_uint64), ("k", C.c_uint32), ("n", C.c_uint32), ("dtype", C.c_int), ("activation", C.c_int),
                ("x", C.c_void_p), ("x_stride", C.c_uint64), ("weight", C.c_void_p), ("weight_stride", C.c_uint64),
                ("bias", C.c_void_p), ("residual", C.c_void_p), ("residual_stride", C.c_uint64), ("out", C.c_void_p),
                ("out_stride", C.c_uint64), ("preactivation", C.c_void_p), ("preactivation_stride", C.c_uint64)]


class LinearGradArgs(C.Structure):
    _fields_ = [("m", C.c_uint64), ("k", C.c_uint32), ("n", C.c_uint32), ("dtype", C.c_int), ("activation", C.c_int),
                ("grad", C.c_void_p), ("grad_stride", C.c_uint64), ("preactivation", C.c_void_p),
                ("preactivation_stride", C.c_uint64), ("x", C.c_void_p), ("x_stride", C.c_uint64),
                ("weight", C.c_void_p), ("weight_stride", C.c_uint64), ("grad_x", C.c_void_p),
                ("grad_x_stride", C.c_uint64), ("grad_weight", C.c_void_p), ("grad_weight_stride", C.c_uint64),
                ("grad_bias", C.c_void_p)]


def embed(lib, rows, dim, count, dtype="fp32", index=8):
    return 0, lib.qvh_embed_device(C.c_void_p(BUF), C.c_uint64(rows), C.c_uint32(dim), C.c_uint64(dim), TYPES[dtype],
                                   C.c_void_p(BUF), index, C.c_uint64(count), C.c_float(1.0), C.c_void_p(BUF), None)


def embed_grad(lib, rows, dim, count, dtype="fp32", index=8):
    need = C.c_uint64()
    status = lib.qvh_embed_grad_workspace(C.c_uint64(rows), C.c_uint32(dim), C.c_uint64(count), C.byref(need))
    return need.value, status or lib.qvh_embed_grad_device(
        C.c_void_p(BUF), C.c_uint64(dim), C.c_void_p(BUF), index, C.c_uint64(count), C.c_uint64(rows), C.c_uint32(dim),
        TYPES[dtype], C.c_float(1.0), C.c_void_p(BUF), C.c_void_p(BUF if need.value else 0), need, None)


def linear(lib, m, k, n, dtype="fp32", act="none", bias=False, residual=False, keep=False, offset=0):
    a = LinearArgs(m=m, k=k, n=n, dtype=TYPES[dtype], activation=ACTS[act], x=BUF + offset * SIZE[dtype], x_stride=k, weight=BUF,
                   weight_stride=k, bias=BUF if bias else None, residual=BUF if residual else None, residual_stride=n, out=BUF,
                   out_stride=n, preactivation=BUF if keep else None, preactivation_stride=n)
    need = C.c_uint64()
    status = lib.qvh_linear_workspace(C.byref(a), C.byref(need))
    return need.value, status or lib.qvh_linear_device(C.byref(a), C.c_void_p(BUF if need.value else 0), need, None)


def linear_grad(lib, m, k, n, dtype="fp32", act="none", inputs=True, weight=True, bias=True):
    a = LinearGradArgs(m=m, k=k, n=n, dtype=TYPES[dtype], activation=ACTS[act], grad=BUF, grad_stride=n, preactivation=BUF,
                       preactivation_stride=n, x=BUF, x_stride=k, weight=BUF, weight_stride=k, grad_x=BUF if inputs else None,
                       grad_x_stride=k, grad_weight=BUF if weight else None, grad_weight_stride=k,
                       grad_bias=BUF if bias else None)
    need = C.c_uint64()
    status = lib.qvh_linear_grad_workspace(C.byref(a), C.byref(need))
    return need.value, status or lib.qvh_linear_grad_device(C.byref(a), C.c_void_p(BUF if need.value else 0), need, None)


def orthogonalize(lib, m, n, batch=1, dtype="fp32", steps=5):
    need = C.c_uint64()
    status = lib.qvh_orthogonalize_workspace(C.c_uint64(batch), C.c_uint32(m), C.c_uint32(n), C.byref(need))
    return need.value, status or lib.qvh_orthogonalize_device(
        C.c_void_p(BUF), C.c_uint64(batch), C.c_uint32(m), C.c_uint32(n), TYPES[dtype], C.c_uint32(steps), C.c_float(3.4445),
        C.c_float(-4.775), C.c_float(2.0315), C.c_void_p(BUF), C.c_void_p(BUF if need.value else 0), need, None)


def get_device(lib):
    device = C.c_int()
    return 0, lib.qvh_get_device(C.byref(device))


def _short(mangled):
    """The kernel's name; for a product also how its operands are read, its tile and its epilogue, for a lookup its
    pieces' elements, how many a thread has, and whether they are stored past the L2s."""
    name = re.search(r"([a-z][a-z_]*_kernel)", mangled).group(1)
    if name == "gemm_kernel":
        read = "".join("rk"[int(b)] for b in re.findall(r"Lb([01])E", mangled)[:2])  # by rows, by k
        tile = re.findall(r"Li(\d+)E", re.search(r"4TileI((?:Li\d+E)+)E", mangled).group(1))
        name += f" {read} {'x'.join(tile[:2])} depth {tile[4]} planes {tile[6]} loads {tile[7]} " + \
            re.search(r"\d([A-Z][a-z]+)Epilogue", mangled).group(1).lower()
    if name == "embed_kernel":
        elements, each = re.findall(r"Li(\d+)E", mangled)
        name += f" {elements} x {each}" + (" past" if re.search(r"Lb1E", mangled) else "")
    return name


def main():
    recorder = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
    recorder.recorder_name.restype = C.c_char_p
    recorder.recorder_kernel.restype = C.c_char_p
    lib = C.CDLL(LIB)
    lib.qvh_last_error.restype = C.c_char_p
    answers = []
    for name, args in json.load(sys.stdin):
        recorder.recorder_clear()
        before = recorder.recorder_device()
        need, status = globals()[name](lib, **args)
        launches = []
        for i in range(recorder.recorder_count()):
            shape = (C.c_ulonglong * 7)()
            recorder.recorder_shape(i, shape)
            launches.append([_short(recorder.recorder_name(i).decode()), shape[0], shape[1], shape[2], shape[4], shape[5]])
        answers.append(dict(status=status, error=lib.qvh_last_error().decode() if status else "", workspace=need,
                            device=[before, recorder.recorder_device()], launches=launches))
    held = itertools.takewhile(lambda name: name is not None, (recorder.recorder_kernel(i) for i in itertools.count()))
    json.dump([sorted({_short(name.decode()) for name in held if b"11gemm_kernel" in name}), answers], sys.stdout)


if __name__ == "__main__":
    main()
