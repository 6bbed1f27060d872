"""Matrices beside one another in the rows of one buffer: what is refused as an overlap and what is not. Everything here comes before
anything that needs a device: a call that passes the argument checks stops at its first pointer, which is no device memory."""
import pytest

from basalt_b200 import kernels

X, Y, Z, S, W = 0x10000000, 0x20000000, 0x30000000, 0x40000000, 0x50000000   # far apart, never followed


def passes(call, *a, **k):
    """The argument checks let the call through: what stops it is the pointer check, or that there is no device."""
    with pytest.raises(kernels.KernelError) as e:
        call(*a, **k)
    assert "overlap" not in str(e.value) and ("device" in str(e.value) or "driver" in str(e.value)), e.value


def refuses(call, *a, **k):
    with pytest.raises(kernels.KernelError, match="overlap"):
        call(*a, **k)


@pytest.mark.parametrize("shift", [64, 64 + 128 * 3, 64 - 128 * 2])   # columns 64 .. 127 of the same rows, of rows further down or further up
def test_norm_beside_its_input(shift):
    passes(kernels.rms_norm, X, X + 2 * shift, 8, 64, "f16", ldx=128, ldy=128)
    refuses(kernels.rms_norm, X, X + 2 * (shift - 1), 8, 64, "f16", ldx=128, ldy=128)     # one column in common
    refuses(kernels.rms_norm, X, X + 2 * (shift + 1), 8, 64, "f16", ldx=128, ldy=128)     # the last one is the next row's first
    passes(kernels.rms_norm, X, X + 2 * (shift + 1), 8, 63, "f16", ldx=128, ldy=128)


def test_norm_and_total_beside_one_another():
    passes(kernels.rms_norm, Z, X, 8, 64, "bf16", residual=X + 512, total=X + 512, ldx=64, ldy=512, ldr=512, ldt=512)
    refuses(kernels.rms_norm, Z, X, 8, 64, "bf16", residual=W, total=X + 64, ldx=64, ldy=512, ldr=512, ldt=512)
    refuses(kernels.rms_norm, X, X + 128, 8, 64, "f16", ldx=128, ldy=136)                  # other strides meet somewhere


def test_bytes_beside_wider_elements():
    passes(kernels.quantize_e4m3, X, X + 128, S, 8, 64, "f16", ldx=128, ldq=256)           # 256 bytes a row, both
    refuses(kernels.quantize_e4m3, X, X + 127, S, 8, 64, "f16", ldx=128, ldq=256)
    refuses(kernels.quantize_e4m3, X, X + 128, S, 8, 64, "f16", ldx=128, ldq=128)


def test_product_beside_its_input():
    passes(kernels.matmul_w4, X, Y, S, X + 256, 16, 128, 128, 32, "f16", ldx=256, ldc=256)
    refuses(kernels.matmul_w4, X, Y, S, X + 254, 16, 128, 128, 32, "f16", ldx=256, ldc=256)
    passes(kernels.matmul_e4m3, X, S, Y, S + 4096, X + 64, 16, 32, 64, "f16", lda=128, ldc=64)
    refuses(kernels.matmul_e4m3, X, S, Y, S + 4096, X + 62, 16, 32, 64, "f16", lda=128, ldc=64)


def test_one_row_and_scales_inside_a_gap_stay_refused():
    refuses(kernels.rms_norm, X, X, 1, 64, "f16", scales=S)
    refuses(kernels.quantize_e4m3, X, Y, X + 128, 8, 64, "f16", ldx=128)                   # scales have no stride to lie beside
