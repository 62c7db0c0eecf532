"""Refusals of the block operators, on the CPU: every argument check runs before the first CUDA
call, so the pointers here are numbers that are never followed."""
from __future__ import annotations

import ctypes as C
import math

import pytest

P = 1 << 20  # 16-byte aligned, never followed
OK, INVALID, UNSUPPORTED, NULL = 0, 3, 10, 11


def _lib():
    from gliner_decide_metal_b200._lib import lib
    return lib


ATTENTION = dict(dtype=2, q=P, ldq=512, k=P, ldk=128, v=P, ldv=128, out=P, ldo=512, q_off=P, k_off=None, batch=2, q_rows=10, k_rows=10,
                 heads=8, kv_heads=2, head_dim=64, causal=1, scale=0.125, workspace=P, workspace_bytes=1 << 40, stream=None)
LINEAR = dict(dtype=5, a=P, lda=64, w=P, ldw=64, bias=None, residual=P, ldr=100, out=P, ldo=100, M=3, rows_dev=None, N=100, K=60, act=3,
              stream=None)
NORM = dict(dtype=2, y=P, ldy=64, x=P, ldx=64, post_norm=1, post_weight=None, post_bias=None, gate=P, gate_rows=1, gate_index=None,
            scale=1.0, pre_norm=2, pre_weight=None, pre_bias=None, x_out=P, ldxo=64, n_out=P, ldno=64, rows=9, rows_dev=None, cols=64,
            eps=1e-6, stream=None)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=3), UNSUPPORTED), (dict(dtype=99), UNSUPPORTED), (dict(batch=-1), INVALID), (dict(q_rows=-1), INVALID),
    (dict(k_rows=-1), INVALID), (dict(q_rows=1 << 31), INVALID), (dict(heads=0), INVALID), (dict(heads=9), INVALID),
    (dict(kv_heads=0), INVALID), (dict(heads=129, kv_heads=1, ldq=1 << 14, ldo=1 << 14), UNSUPPORTED), (dict(head_dim=32), UNSUPPORTED),
    (dict(head_dim=96), UNSUPPORTED), (dict(scale=0.0), INVALID), (dict(scale=-1.0), INVALID), (dict(scale=math.nan), INVALID),
    (dict(scale=math.inf), INVALID), (dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL), (dict(out=None), NULL),
    (dict(q_off=None), NULL), (dict(ldq=504), INVALID), (dict(ldk=120), INVALID), (dict(ldv=64), INVALID), (dict(ldo=8), INVALID),
    (dict(ldq=516), INVALID), (dict(ldk=132), INVALID), (dict(q=P + 2), INVALID), (dict(k=P + 8), INVALID), (dict(v=P + 4), INVALID),
    (dict(out=P + 2), INVALID), (dict(q_off=P + 2), INVALID), (dict(k_off=P + 1), INVALID), (dict(workspace=None), NULL), (dict(workspace_bytes=0), INVALID), (dict(workspace=P + 16), INVALID),
    (dict(batch=0), OK), (dict(q_rows=0, q=None, out=None), OK)])
def test_attention_refuses(change, status):
    assert _lib().gdc_packed_attention(*{**ATTENTION, **change}.values()) == status
    if status != OK:
        assert _lib().gdc_last_error()


def test_attention_workspace_query():
    n = C.c_size_t()
    assert _lib().gdc_packed_attention_workspace(2, 10, 10, 8, 2, 64, None) == NULL
    assert _lib().gdc_packed_attention_workspace(2, 10, 10, 8, 3, 64, C.byref(n)) == INVALID
    assert _lib().gdc_packed_attention_workspace(2, 10, 10, 8, 2, 80, C.byref(n)) == UNSUPPORTED
    for batch, q_rows, k_rows in ((0, 0, 0), (1, 1, 1), (64, 64, 1 << 20), (4, 8192, 8192), (1 << 20, 1 << 30, 1 << 30)):
        assert _lib().gdc_packed_attention_workspace(batch, q_rows, k_rows, 8, 2, 64, C.byref(n)) == OK
        assert n.value < 1 << 30


@pytest.mark.parametrize("change,status", [
    (dict(dtype=0), UNSUPPORTED), (dict(M=-1), INVALID), (dict(N=0), INVALID), (dict(K=0), INVALID), (dict(act=4), INVALID),
    (dict(act=-1), INVALID), (dict(a=None), NULL), (dict(w=None), NULL), (dict(out=None), NULL), (dict(lda=56), INVALID),
    (dict(ldw=56), INVALID), (dict(lda=68), INVALID), (dict(ldw=65), INVALID), (dict(ldr=99), INVALID), (dict(ldo=99), INVALID),
    (dict(a=P + 2), INVALID), (dict(w=P + 8), INVALID), (dict(bias=P + 1), INVALID), (dict(residual=P + 1), INVALID),
    (dict(out=P + 1), INVALID), (dict(rows_dev=P + 2), INVALID), (dict(ldo=1 << 33), UNSUPPORTED), (dict(M=0, a=None), OK)])
def test_linear_refuses(change, status):
    assert _lib().gdc_linear_residual(*{**LINEAR, **change}.values()) == status


@pytest.mark.parametrize("change,status", [
    (dict(dtype=4), UNSUPPORTED), (dict(rows=-1), INVALID), (dict(cols=0), INVALID), (dict(cols=16385), INVALID),
    (dict(post_norm=3), INVALID), (dict(pre_norm=-1), INVALID), (dict(scale=math.nan), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=math.nan), INVALID), (dict(x=None), NULL), (dict(x_out=None), NULL), (dict(n_out=None), INVALID),
    (dict(pre_norm=0), INVALID), (dict(pre_norm=0, n_out=None, x_out=None, y=None, gate=None, post_norm=0), NULL),
    (dict(gate_rows=0), INVALID), (dict(gate_rows=8), INVALID), (dict(gate=None, gate_index=P), INVALID),
    (dict(y=None), INVALID), (dict(y=None, gate=None), INVALID), (dict(ldy=63), INVALID), (dict(ldx=63), INVALID),
    (dict(ldxo=63), INVALID), (dict(ldno=0), INVALID), (dict(x=P + 1), INVALID), (dict(gate=P + 1), INVALID),
    (dict(gate_index=P + 2), INVALID), (dict(rows_dev=P + 1), INVALID), (dict(rows=0), OK)])
def test_norm_refuses(change, status):
    assert _lib().gdc_gated_residual_norm(*{**NORM, **change}.values()) == status


def test_outputs_laid_over_inputs_at_another_pitch_are_refused():
    norm = {**NORM, "x_out": 2 * P, "n_out": 3 * P, "x": 4 * P}
    for change in (dict(x_out=4 * P, ldxo=72), dict(n_out=P, ldno=65), dict(n_out=2 * P)):
        assert _lib().gdc_gated_residual_norm(*{**norm, **change}.values()) == INVALID
        assert _lib().gdc_last_error()
    assert _lib().gdc_linear_residual(*{**LINEAR, "ldo": 104}.values()) == INVALID


def test_other_entry_points_still_refuse_the_new_type():
    """GDC_BFLOAT16 belongs to the block operators: a classify input of that type is refused."""
    from gliner_decide_metal_b200 import _lib as b
    assert b.GDC_BFLOAT16 == 5
    inp = b.GdcInput(1, 4, 1, 1, P, b.GDC_INT32, P, b.GDC_BFLOAT16, P, b.GDC_INT32, P, b.GDC_FLOAT32)
    out = b.GdcOutput(P, None, 0, None, 0, 0)
    import numpy as np
    keep = np.zeros(8, np.float32)
    out.logits = keep.ctypes.data
    h = C.c_void_p(P)
    models = (C.c_void_p * 1)(h)
    st = (C.c_int * 1)()
    assert _lib().gdc_classify_sharded(models, 1, C.byref(inp), C.byref(out), st) == INVALID
