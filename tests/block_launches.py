"""What the blocks' calls launch: tests/launches.py with the calls of norms, attention and clipping.

    python tests/block_launches.py RECORDER < calls > launches

Kernels go by name and template arguments; all of these operators' that the library holds come out first.
"""

from __future__ import annotations

import ctypes as C
import itertools
import json
import re
import sys

import launches
from launches import BUF, SIZE, TYPES

GATES = {"none": 0, "silu": 3, "sigmoid": 4}
OWN = re.compile(r"(norm_kernel|norm_grad_kernel|norm_sums_kernel|clip_\w+?_kernel|norm_result_kernel|attention_\w*?kernel)")

U3 = C.c_uint64 * 3


class NormArgs(C.Structure):
    _fields_ = [("rows", C.c_uint64), ("dim", C.c_uint32), ("dtype", C.c_int), ("gate_activation", C.c_int), ("eps", C.c_float),
                ("x", C.c_void_p), ("x_stride", C.c_uint64), ("y", C.c_void_p), ("y_stride", C.c_uint64), ("gate", C.c_void_p),
                ("gate_stride", C.c_uint64), ("weight", C.c_void_p), ("post_weight", C.c_void_p), ("scale", C.c_void_p),
                ("r", C.c_void_p), ("h", C.c_void_p)]


class NormGradArgs(C.Structure):
    _fields_ = [("rows", C.c_uint64), ("dim", C.c_uint32), ("dtype", C.c_int), ("gate_activation", C.c_int), ("eps", C.c_float),
                ("grad_h", C.c_void_p), ("grad_h_stride", C.c_uint64), ("grad_r", C.c_void_p), ("grad_r_stride", C.c_uint64),
                ("r", C.c_void_p), ("r_stride", C.c_uint64), ("y", C.c_void_p), ("y_stride", C.c_uint64), ("gate", C.c_void_p),
                ("gate_stride", C.c_uint64), ("weight", C.c_void_p), ("post_weight", C.c_void_p), ("scale", C.c_void_p),
                ("grad_x", C.c_void_p), ("grad_y", C.c_void_p), ("grad_gate", C.c_void_p), ("grad_weight", C.c_void_p),
                ("grad_post", C.c_void_p), ("grad_scale", C.c_void_p)]


class AttentionArgs(C.Structure):
    _fields_ = [("batch", C.c_uint64), ("tokens", C.c_uint64), ("heads", C.c_uint32), ("kv_heads", C.c_uint32), ("dk", C.c_uint32),
                ("dv", C.c_uint32), ("dtype", C.c_int), ("scale", C.c_float), ("q", C.c_void_p), ("q_stride", U3), ("k", C.c_void_p),
                ("k_stride", U3), ("v", C.c_void_p), ("v_stride", U3), ("log_decay", C.c_void_p), ("lengths", C.c_void_p),
                ("index_bytes", C.c_int), ("state", C.c_void_p), ("state_out", C.c_void_p), ("out", C.c_void_p)]


class AttentionGradArgs(C.Structure):
    _fields_ = [("forward", AttentionArgs), ("grad", C.c_void_p), ("grad_stride", U3), ("grad_state", C.c_void_p), ("grad_q", C.c_void_p),
                ("grad_k", C.c_void_p), ("grad_v", C.c_void_p), ("grad_first", C.c_void_p)]


class Gradient(C.Structure):
    _fields_ = [("grad", C.c_void_p), ("out", C.c_void_p), ("count", C.c_uint64), ("dtype", C.c_int)]


def block_norm(lib, rows, dim, dtype="bf16", block=True, gate=True):
    p = BUF if block else None
    a = NormArgs(rows=rows, dim=dim, dtype=TYPES[dtype], eps=1e-6, x=BUF, x_stride=dim, y=p, y_stride=dim, gate=p if gate else None,
                 gate_stride=dim, weight=BUF, post_weight=p, r=p, h=BUF)
    return 0, lib.qvh_block_norm_device(C.byref(a), None)


def block_norm_grad(lib, rows, dim, dtype="bf16", block=True, gate=True):
    p = BUF if block else None
    q = p if gate else None
    a = NormGradArgs(rows=rows, dim=dim, dtype=TYPES[dtype], eps=1e-6, grad_h=BUF, grad_h_stride=dim, grad_r=BUF, grad_r_stride=dim, r=BUF,
                     r_stride=dim, y=p, y_stride=dim, gate=q, gate_stride=dim, weight=BUF, post_weight=p, grad_x=BUF, grad_y=p, grad_gate=q,
                     grad_weight=BUF, grad_post=p)
    need = C.c_uint64()
    status = lib.qvh_block_norm_grad_workspace(C.c_uint64(rows), C.c_uint32(dim), TYPES[dtype], int(block), C.byref(need))
    return need.value, status or lib.qvh_block_norm_grad_device(C.byref(a), C.c_void_p(BUF if need.value else 0), need, None)


def _attention(batch, tokens, heads, kv_heads, dk, dv, dtype, apart=0, offset=0, state=False):
    qs, ks, vs = ((n * d + apart, d) for n, d in ((heads, dk), (kv_heads, dk), (kv_heads, dv)))
    at = BUF + offset * SIZE[dtype]
    three = lambda t, d: U3(min(t * tokens, 2**39), t, d)  # noqa: E731
    return AttentionArgs(batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, dtype=TYPES[dtype], scale=1.0, q=at,
                         q_stride=three(*qs), k=at, k_stride=three(*ks), v=at, v_stride=three(*vs), log_decay=BUF,
                         state=BUF if state else None, state_out=BUF if state else None, out=BUF)


def attention(lib, batch, tokens, heads, kv_heads, dk, dv, dtype="bf16", **more):
    a = _attention(batch, tokens, heads, kv_heads, dk, dv, dtype, **more)
    need = C.c_uint64()
    status = lib.qvh_attention_workspace(C.byref(a), C.byref(need))
    return need.value, status or lib.qvh_attention_device(C.byref(a), C.c_void_p(BUF if need.value else 0), need, None)


def attention_grad(lib, batch, tokens, heads, kv_heads, dk, dv, dtype="bf16", **more):
    f = _attention(batch, tokens, heads, kv_heads, dk, dv, dtype, **more)
    a = AttentionGradArgs(forward=f, grad=BUF, grad_stride=U3(tokens * heads * dv, heads * dv, dv), grad_q=BUF, grad_k=BUF, grad_v=BUF,
                          grad_first=f.state)
    need = C.c_uint64()
    status = lib.qvh_attention_grad_workspace(C.byref(a), C.byref(need))
    return need.value, status or lib.qvh_attention_grad_device(C.byref(a), C.c_void_p(BUF if need.value else 0), need, None)


def clip(lib, sizes, dtype="bf16"):
    at, grads = BUF, []
    for n in sizes:
        grads.append(Gradient(at, at, n, TYPES[dtype]))
        at += n * 4
    need = C.c_uint64()
    status = lib.qvh_grad_norm_workspace(C.c_uint64(len(grads)), C.byref(need))
    return need.value, status or lib.qvh_clip_grad_norm_device((Gradient * len(grads))(*grads), C.c_uint64(len(grads)), C.c_float(1.0),
                                                               C.c_float(1e-6), C.c_void_p(BUF), C.c_void_p(BUF), need, None)


def short(mangled):
    """Name, type and numbers: attention_kernel bf16 64 0 1 is of 64 dk, not the states alone, whole rows."""
    found = OWN.search(mangled)
    if not found:
        return "other"
    rest = mangled[found.end():]
    types = {"f": "fp32", "DF16_": "fp16", "DF16b": "bf16"}
    element = re.match(r"I(DF16_|DF16b|f)", rest)
    numbers = re.findall(r"L[ib](\d+)E", rest)
    if found.group(1) == "norm_kernel" and not numbers:
        return "other"  # of orthogonalisation and of rows of an index
    return " ".join([found.group(1), *([types[element.group(1)]] if element else []), *numbers])


def main():
    recorder = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
    recorder.recorder_name.restype = C.c_char_p
    recorder.recorder_kernel.restype = C.c_char_p
    lib = C.CDLL(launches.LIB)
    lib.qvh_last_error.restype = C.c_char_p
    answers = []
    for name, args in json.load(sys.stdin):
        recorder.recorder_clear()
        before = recorder.recorder_device()
        need, status = globals()[name](lib, **args)
        out = []
        for i in range(recorder.recorder_count()):
            shape = (C.c_ulonglong * 7)()
            recorder.recorder_shape(i, shape)
            out.append([short(recorder.recorder_name(i).decode()), shape[0], shape[1], shape[2], shape[5]])
        answers.append(dict(status=status, error=lib.qvh_last_error().decode() if status else "", workspace=need,
                            device=[before, recorder.recorder_device()], launches=out))
    held = itertools.takewhile(lambda name: name is not None, (recorder.recorder_kernel(i) for i in itertools.count()))
    json.dump([sorted({short(name.decode()) for name in held} - {"other"}), answers], sys.stdout)


if __name__ == "__main__":
    main()
