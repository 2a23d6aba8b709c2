"""Refusals of kb_matmul, kb_rope and kb_cross_attention that need no GPU: sizes, strides and views are looked at before anything else."""
import ctypes

import pytest

from katago_b200 import capi

FP32, FP16 = capi.PRECISION_FP32, capi.PRECISION_FP16
P = 0x10000000  # an address that nothing looks at before the sizes are found to be right


def matmul(precision=FP32, m=4, n=4, k=4, ldx=4, ldw=4, ldy=4, act=0, residual=0, ldr=4):
    capi.matmul(precision, m, n, k, P, ldx, P, ldw, P, ldy, act=act, residual=residual, ldr=ldr)


@pytest.mark.parametrize("given,says", [
    (dict(precision=7), "unknown precision"), (dict(m=-1), "m is -1"), (dict(k=(1 << 30) + 1, ldx=1 << 31, ldw=1 << 31), "k is 1073741825"), (dict(n=2 ** 31 - 1), "n is 2147483647"), (dict(n=0), "n is 0"), (dict(k=0), "k is 0"), (dict(act=4), "unknown activation"),
    (dict(ldx=3), "row stride of x or w"), (dict(ldw=3), "row stride of x or w"), (dict(ldy=3), "row stride of y"), (dict(residual=P, ldr=3), "row stride of y or the residual"),
])
def test_matmul_refuses(given, says):
    with pytest.raises(capi.KBError, match=says):
        matmul(**given)


def rope(precision=FP32, batch=1, tokens=2, dim=8, rot=8, axes=1, tables=1, halves=0, q_heads=2, k_heads=0, stride=16, pos_stride=0, q="view", out="view"):
    v = capi.View(P, 2 * stride, stride, 8)
    capi.rope(precision, batch, tokens, dim, rot, P, pos_stride, axes, P, tables, halves, v if q else None, v if out else None, q_heads, None, None, k_heads)


@pytest.mark.parametrize("given,says", [
    (dict(precision=3), "unknown precision"), (dict(batch=-1), "batch is -1"), (dict(tokens=-2), "tokens is -2"), (dict(rot=7), "rotDim is odd"), (dict(rot=10), "rotDim is 10"),
    (dict(rot=0), "rotDim is 0"), (dict(dim=1, rot=1), "headDim is 1"), (dict(axes=0), "axes is 0"), (dict(axes=17), "axes is 17"), (dict(tables=0), "freqHeads is 0"),
    (dict(tables=2, q_heads=3), "freqHeads does not divide"), (dict(halves=2), "unknown pair layout"), (dict(q_heads=-1), "qHeads is -1"), (dict(q=None), "q in is NULL"),
    (dict(out=None), "q out is NULL"), (dict(k_heads=1), "k in is NULL|no CUDA device|could not be looked up|not device memory"), (dict(stride=-16), "stride of q in"),
    (dict(pos_stride=-1), "batch stride of the positions"), (dict(batch=1 << 20, tokens=1 << 20), r"more than 2\^31"),
])
def test_rope_refuses(given, says):
    with pytest.raises(capi.KBError, match=says):
        rope(**given)


def attention(precision=FP32, batch=1, q_len=2, k_len=2, heads=2, kv_heads=1, dq=8, dv=8, scale=1.0, views=4, stride=16):
    v = [capi.View(P, 2 * stride, stride, 8) if i < views else None for i in range(4)]
    capi.cross_attention(precision, batch, q_len, k_len, heads, kv_heads, dq, dv, scale, *v)


@pytest.mark.parametrize("given,says", [
    (dict(precision=-1), "unknown precision"), (dict(batch=-1), "batch is -1"), (dict(q_len=-1), "qLen is -1"), (dict(k_len=-1), "kLen is -1"), (dict(heads=0), "heads is 0"),
    (dict(kv_heads=0), "kvHeads is 0"), (dict(heads=3, kv_heads=2), "does not divide"), (dict(dq=0), "qkDim is 0"), (dict(dq=257), "qkDim is 257"), (dict(dv=257), "vDim is 257"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(views=0), "q is NULL"),
    (dict(views=3), "out is NULL"), (dict(stride=-8), "stride of q"), (dict(q_len=1 << 30, heads=8), r"more than 2\^31 rows"), (dict(batch=1 << 30, q_len=1 << 20), "too many rows"),
])
def test_attention_refuses(given, says):
    with pytest.raises(capi.KBError, match=says):
        attention(**given)


def test_calls_of_nothing_do_nothing():
    matmul(m=0)
    rope(batch=0)
    rope(tokens=0)
    rope(q_heads=0)
    attention(batch=0)
    attention(q_len=0)


def test_workspace_refuses_what_the_call_refuses():
    with pytest.raises(capi.KBError, match="qkDim is 300"):
        capi.cross_attention_workspace(FP16, 1, 1, 1, 1, 1, 300, 64)
    with pytest.raises(capi.KBError, match="bytes is NULL"):
        capi._check(capi.lib().kb_cross_attention_workspace(FP16, 1, 1, 1, 1, 1, 64, 64, None), "kb_cross_attention_workspace")
    assert capi.cross_attention_workspace(FP16, 0, 1, 1, 1, 1, 64, 64) == 0


def test_pointers_are_not_taken_without_a_device():
    """Whatever the machine: an address that is no device memory is refused, not read."""
    import numpy as np
    host = np.zeros(64, np.float32)
    at = host.ctypes.data_as(ctypes.c_void_p).value
    with pytest.raises(capi.KBError, match="no CUDA device|not device memory|could not be looked up"):
        capi.matmul(FP32, 2, 2, 2, at, 2, at + 64, 2, at + 128, 2)
