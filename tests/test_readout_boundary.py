"""The readout operators' C entry points refuse bad arguments before they touch a GPU."""

from __future__ import annotations

import ctypes

import pytest

from mdescriptor_b200 import _lib
from mdescriptor_b200._lib import INVALID_ARGUMENT, OK, lib

P = 1 << 20  # a 16-byte aligned address that no refused call reads


def refused(status, text):
    assert status == INVALID_ARGUMENT
    assert text in _lib.last_error()
    with pytest.raises(ValueError, match="readout"):
        _lib.raise_for(status)


def norm(x=P, rows=4, width=8, stride=8, dtype=_lib.FLOAT32, weight=P, eps=1e-6, out=P, out_stride=16, scales=P,
         scale_stride=1):
    return lib.mdsoap_rms_norm(x, rows, width, stride, None, 0, dtype, weight, eps, None, 0, None, out, out_stride, scales,
                               scale_stride, 0, None)


def test_norm_refusals():
    refused(norm(x=None), "norm input")
    refused(norm(rows=-1), "norm input")
    refused(norm(stride=7), "norm input")
    refused(norm(weight=None), "weight")
    refused(norm(eps=0.0), "eps")
    refused(norm(eps=float("nan")), "eps")
    refused(norm(out_stride=8), "multiple of 16")
    refused(norm(out=P + 8), "16-byte aligned")
    refused(norm(scale_stride=0), "one scale")
    refused(norm(scales=None, out=None), "norm output")
    refused(lib.mdsoap_rms_norm_backward(P, 4, 8, 8, P, 8, P, P, None, 0, _lib.FLOAT32, P, 7, P, P, 1 << 20, 0, None), "dx")
    refused(lib.mdsoap_rms_norm_backward(P, 4, 8, 8, P, 8, None, P, None, 0, _lib.FLOAT32, P, 8, P, P, 1 << 20, 0, None),
            "rstd")


def test_quantize_refusals():
    def quantize(tiles=0, row=None, codes=P, codes_t=P, stride=16, stride_t=16, scale_t_stride=1):
        return lib.mdsoap_quantize(P, 4, 8, 8, _lib.FLOAT32, row, None, tiles, codes, stride, P, 1, codes_t, stride_t, P,
                                   scale_t_stride, 0, None)

    refused(quantize(codes=None, codes_t=None), "output")
    refused(quantize(tiles=1, row=P), "factors")
    refused(quantize(tiles=1, codes_t=None), "transpose")
    refused(quantize(stride=24), "8-bit rows")
    refused(quantize(stride_t=4), "8-bit columns")
    refused(quantize(codes_t=P + 4), "8-bit columns")


def test_product_refusals():
    def matmul(a=P, m=4, n=4, k=32, stride=32, scales=P, dtype=_lib.FLOAT32, accumulate=0, out=P, out_stride=4):
        return lib.mdsoap_matmul(a, m, stride, scales, 1, P, n, 32, P, 1, 0, k, dtype, accumulate, out, out_stride, None, 0,
                                 0, None)

    refused(matmul(m=-1), "shape")
    refused(matmul(k=1 << 40), "shape")
    refused(matmul(dtype=_lib.FLOAT16), "float32 or bfloat16")
    refused(matmul(dtype=_lib.BFLOAT16, accumulate=1), "added to")
    refused(matmul(out=None), "output")
    refused(matmul(out_stride=3), "output")
    refused(matmul(a=None), "operands")
    refused(matmul(a=P + 8), "operands")
    refused(matmul(stride=40), "operands")
    refused(matmul(scales=None), "operands")
    size = ctypes.c_int64()
    assert lib.mdsoap_matmul_bytes(-1, 4, 32, 0, 0, ctypes.byref(size)) == INVALID_ARGUMENT


def test_optimizer_refusals_and_lifetime():
    pointers, counts = (ctypes.c_void_p * 2)(P, P), (ctypes.c_int64 * 2)(10, 20)

    def create(tensors=2, dtype=_lib.FLOAT32, bits=32, counts=counts, scales=None, params=pointers, decay=None):
        handle = ctypes.c_void_p()
        address = [ctypes.cast(v, ctypes.c_void_p) if v is not None else None for v in (params, scales, counts, decay)]
        args = _lib.AdamWParams(tensors, address[0], ctypes.cast(pointers, ctypes.c_void_p),
                                ctypes.cast(pointers, ctypes.c_void_p), address[1], address[1], address[2], address[3],
                                dtype, bits, 0, 0)
        return lib.mdsoap_adamw_create(ctypes.byref(args), ctypes.byref(handle)), handle

    refused(create(bits=16)[0], "32 or 8")
    refused(create(bits=8)[0], "scales")
    refused(create(dtype=_lib.FLOAT64)[0], "element type")
    refused(create(params=None)[0], "tensors")
    refused(create(params=(ctypes.c_void_p * 2)(P, None))[0], "null")
    refused(create(counts=(ctypes.c_int64 * 2)(10, -1))[0], "size")
    refused(create(decay=(ctypes.c_float * 2)(0.0, -0.5))[0], "weight decay")
    status, handle = create()  # touches no GPU
    assert status == OK

    def step(grads=pointers, dtype=_lib.FLOAT32, step=1, lr=1e-3, beta=0.9, eps=1e-8, scale=1.0):
        return lib.mdsoap_adamw_step(handle, grads, dtype, step, lr, beta, 0.999, eps, scale, None)

    refused(step(step=0), "count from 1")
    refused(step(beta=1.0), "betas")
    refused(step(lr=float("inf")), "settings")
    refused(step(scale=float("nan")), "settings")
    refused(step(grads=None), "gradients")
    refused(step(grads=(ctypes.c_void_p * 2)(P, None)), "null gradient")
    refused(step(dtype=_lib.FLOAT64), "element type")
    lib.mdsoap_adamw_destroy(handle)
    lib.mdsoap_adamw_destroy(None)
