"""Which memory the passes of linear attention's launches keep their segments' states in, in a process without a GPU.

    python tests/attention_passes.py RECORDER < calls > launches

As tests/block_launches.py, with the launches' arguments: a call is [name, {argument: value}], name attention or attention_grad, and
its answer {status, error, workspace, launches}, each launch [kernel, passes]. A pass has what the kernels take of it and the
shape it was made for. The workspace lies at WORK, every other buffer at another address.
"""

from __future__ import annotations

import ctypes as C
import json
import sys

import block_launches
import launches
from block_launches import U3, AttentionArgs, AttentionGradArgs
from launches import BUF, TYPES

WORK = 1 << 44


class TokenTensor(C.Structure):
    _fields_ = [("base", C.c_void_p), ("batch", C.c_uint64), ("token", C.c_uint64), ("head", C.c_uint64), ("share", C.c_uint32)]


class Pass(C.Structure):
    """As AttentionPass in quiver_amd/csrc/hip/attention.hip."""
    _fields_ = [("tokens", C.c_uint64), ("batch", C.c_uint32), ("heads", C.c_uint32), ("dk", C.c_uint32), ("dv", C.c_uint32),
                ("q", TokenTensor), ("k", TokenTensor), ("v", TokenTensor), ("out", C.c_void_p), ("out_fp32", C.c_bool),
                ("exact", C.c_bool), ("wide", C.c_bool), ("log_decay", C.c_void_p), ("lengths", C.c_void_p), ("index_bytes", C.c_int),
                ("state", C.c_void_p), ("state_out", C.c_void_p), ("state_dk", C.c_uint32), ("state_dv", C.c_uint32),
                ("reverse", C.c_bool), ("ahead", C.c_uint32), ("kv_scale", C.c_float), ("near_scale", C.c_float),
                ("far_scale", C.c_float), ("segments", C.c_uint32), ("segment", C.c_uint64), ("states", C.c_void_p)]


def _forward(batch, tokens, heads, kv_heads, dk, dv, dtype, state, apart, by_token):
    """apart: elements between the rows of a tensor by its name, where they are further apart than its heads; by_token: texts lie
    next to one another within a token."""
    def strides(name, n, d):
        row = max(n * d, apart.get(name, 0))
        return U3(n * d, batch * n * d, d) if by_token else U3(min(tokens * row, 2**39), row, d)

    p = BUF if state else None
    return AttentionArgs(batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, dtype=TYPES[dtype], scale=1.0, q=BUF,
                         q_stride=strides("q", heads, dk), k=BUF, k_stride=strides("k", kv_heads, dk), v=BUF,
                         v_stride=strides("v", kv_heads, dv), log_decay=BUF, state=p, state_out=p, out=BUF), strides("grad", heads, dv)


def attention(lib, batch, tokens, heads, kv_heads, dk, dv, dtype="bf16", state=False, apart={}, by_token=False):
    a, _ = _forward(batch, tokens, heads, kv_heads, dk, dv, dtype, state, apart, by_token)
    need = C.c_uint64()
    status = lib.qvh_attention_workspace(C.byref(a), C.byref(need))
    return need.value, status or lib.qvh_attention_device(C.byref(a), C.c_void_p(WORK), need, None)


def attention_grad(lib, batch, tokens, heads, kv_heads, dk, dv, dtype="bf16", state=False, apart={}, by_token=False):
    f, grad = _forward(batch, tokens, heads, kv_heads, dk, dv, dtype, state, apart, by_token)
    a = AttentionGradArgs(forward=f, grad=BUF, grad_stride=grad, grad_state=f.state, grad_q=BUF, grad_k=BUF, grad_v=BUF, grad_first=f.state)
    need = C.c_uint64()
    status = lib.qvh_attention_grad_workspace(C.byref(a), C.byref(need))
    return need.value, status or lib.qvh_attention_grad_device(C.byref(a), C.c_void_p(WORK), need, None)


def main():
    recorder = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
    recorder.recorder_name.restype = C.c_char_p
    recorder.recorder_argument.restype = C.c_void_p
    lib = C.CDLL(launches.LIB)
    lib.qvh_last_error.restype = C.c_char_p
    recorder.recorder_keep(b"AttentionPasses", C.c_size_t(C.sizeof(Pass * 3)))
    answers = []
    for name, args in json.load(sys.stdin):
        recorder.recorder_clear()
        need, status = globals()[name](lib, **args)
        out = []
        for i in range(recorder.recorder_count()):
            at = recorder.recorder_argument(i)
            if not at:
                continue
            shape = (C.c_ulonglong * 7)()
            recorder.recorder_shape(i, shape)
            kernel = block_launches.short(recorder.recorder_name(i).decode())
            count = shape[3] if kernel.startswith("attention_scan") else shape[1]
            out.append([kernel, [dict(tokens=p.tokens, batch=p.batch, heads=p.heads, dk=p.dk, dv=p.dv, segments=p.segments, segment=p.segment,
                                      states=p.states or 0, parts=(p.out or 0) if p.out_fp32 else 0) for p in (Pass * 3).from_address(at)[:count]]])
        answers.append(dict(status=status, error=lib.qvh_last_error().decode() if status else "", workspace=need, launches=out))
    json.dump(answers, sys.stdout)


if __name__ == "__main__":
    main()
