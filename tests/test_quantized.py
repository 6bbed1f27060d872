"""What the norm, the row quantisation and the e4m3 and 4-bit products refuse. Every check here comes before
anything that needs a device, so the refusals run on a machine without one."""
import numpy as np
import pytest

from basalt_b200 import kernels

X, Y, Z, S, W = 0x10000000, 0x20000000, 0x30000000, 0x40000000, 0x50000000   # far apart, never followed


def norm(**k):
    a = dict(x=X, y=Y, rows=4, cols=64, dtype="f16")
    a.update(k)
    kernels.rms_norm(**a)


@pytest.mark.parametrize("change, message", [
    (dict(dtype="f64"), "unknown type"),
    (dict(rows=-1), "rows must lie"),
    (dict(rows=2**31), "rows must lie"),
    (dict(cols=0), "cols must lie"),
    (dict(x=None), "are needed"),
    (dict(y=None), "are needed"),
    (dict(ldx=63), "row stride"),
    (dict(ldy=63), "row stride"),
    (dict(residual=Z, ldr=10), "row stride"),
    (dict(x=X + 1), "aligned"),
    (dict(dtype="f32", x=X + 2), "aligned"),
    (dict(scales=S + 2), "aligned"),
    (dict(weight=W + 1), "aligned"),
    (dict(total=Z), "total is written only"),
    (dict(eps=-1e-6), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(y=X + 64), "overlaps"),
    (dict(y=X, ldy=72), "overlaps"),
    (dict(y=X, scales=S), "overlaps"),
    (dict(residual=Z, total=Z + 2), "overlaps"),
    (dict(residual=Z, total=Y), "outputs overlap"),
    (dict(weight=Y), "the weight"),
    (dict(y=S, scales=S), "scales overlap"),
])
def test_rms_norm_refuses(change, message):
    with pytest.raises(kernels.KernelError, match=message):
        norm(**change)


@pytest.mark.parametrize("change, message", [
    (dict(scales=None), "scales are needed"),
    (dict(q=X), "overlaps"),
    (dict(ldq=63), "row stride"),
    (dict(rows=-3), "rows must lie"),
    (dict(cols=2**31), "cols must lie"),
    (dict(scales=X), "scales overlap"),
])
def test_quantize_refuses(change, message):
    a = dict(x=X, q=Y, scales=S, rows=4, cols=64, dtype="bf16")
    a.update(change)
    with pytest.raises(kernels.KernelError, match=message):
        kernels.quantize_e4m3(**a)


@pytest.mark.parametrize("change, message", [
    (dict(out="e4m3"), "unknown type"),
    (dict(M=-1), "negative"),
    (dict(N=-1), "negative"),
    (dict(K=0), "K must be"),
    (dict(A=None), "are needed"),
    (dict(a_scales=None), "are needed"),
    (dict(A=X + 8), "multiples of 16"),
    (dict(K=40), "multiples of 16"),
    (dict(lda=48), "row stride"),
    (dict(ldc=7), "row stride"),
    (dict(Cm=Z + 1), "aligned"),
    (dict(out="f32", Cm=Z + 2), "aligned"),
    (dict(status=W + 1), "aligned"),
    (dict(Cm=X), "overlaps"),
    (dict(Cm=S), "overlaps"),
])
def test_matmul_e4m3_refuses(change, message):
    a = dict(A=X, a_scales=S, B=Y, b_scales=S + 4096, Cm=Z, M=4, N=8, K=64)
    a.update(change)
    with pytest.raises(kernels.KernelError, match=message):
        kernels.matmul_e4m3(**a)


@pytest.mark.parametrize("change, message", [
    (dict(dtype="f32"), "f16 or bf16"),
    (dict(M=-1), "negative"),
    (dict(K=0), "K must be"),
    (dict(group=0), "multiple of 32"),
    (dict(group=48), "multiple of 32"),
    (dict(group=-32), "multiple of 32"),
    (dict(W=None), "are needed"),
    (dict(scales=None), "are needed"),
    (dict(X=X + 8), "multiples of 16"),
    (dict(ldx=68), "multiples of 16"),
    (dict(ldw=33), "multiples of 16"),
    (dict(ldx=56), "row stride"),
    (dict(ldw=16), "row stride"),
    (dict(ldc=7), "row stride"),
    (dict(Cm=Z + 1), "aligned"),
    (dict(scales=S + 2), "multiple of 4"),
    (dict(zeros=W + 1), "multiple of 4"),
    (dict(Cm=X), "overlaps"),
    (dict(Cm=Y), "overlaps"),
])
def test_matmul_w4_refuses(change, message):
    a = dict(X=X, W=Y, scales=S, Cm=Z, M=4, N=8, K=64, group=32)
    a.update(change)
    with pytest.raises(kernels.KernelError, match=message):
        kernels.matmul_w4(**a)


def test_nothing_to_do_is_no_error():
    norm(rows=0)
    kernels.quantize_e4m3(X, Y, S, 0, 64, "f32")
    kernels.matmul_e4m3(X, S, Y, S, Z, 0, 8, 64)
    kernels.matmul_e4m3(X, S, Y, S, Z, 4, 0, 64)
    kernels.matmul_w4(X, Y, S, Z, 0, 8, 64, 32)


def test_arguments_that_fit_no_parameter():
    with pytest.raises(OverflowError):
        kernels.matmul_w4(X, Y, S, Z, 2**32 + 1, 8, 64, 32)     # must not wrap to one row
    with pytest.raises(OverflowError):
        kernels.rms_norm(-16, Y, 1, 64, "f16")
    with pytest.raises(TypeError):
        kernels.quantize_e4m3(X, Y, S, None, 64, "f16")
    with pytest.raises(TypeError):
        norm(eps="small")
    with pytest.raises(AttributeError):
        norm(x="x")
    norm(x=np.uint64(X), rows=np.int64(0))                       # whatever is an integer passes
