"""Calls of the quantised layer's operators at the ends of their ranges: the largest rows, exact ties, weights from cold
memory, long sums, matrices that share a buffer."""
import numpy as np
import pytest
import torch

from basalt_b200 import kernels
from test_gpu_quantized import T, U, check_e4m3, down, exact_norm, gen, rows, up

pytestmark = pytest.mark.gpu

# widths of every path through the row kernels: whole vectors in registers, element by element, and read twice
WIDTHS = [64, 77, 4096, 9001, 40000]


def quantized(gpu, x, t):
    n, cols = x.shape
    y, s = torch.full((n, cols), 0x55, dtype=torch.uint8), torch.full((n,), 5.0)
    dx, dy, ds = up(gpu, x.contiguous()), up(gpu, y), up(gpu, s)
    kernels.quantize_e4m3(dx, dy, ds, n, cols, t)
    gpu.synchronize()
    return down(dy, y), down(ds, s)


def largest_rows(cols, t):
    """Rows whose largest magnitude is 2^125, just above 2^126, 2^127 and the type's largest number, and one masked with the lowest."""
    top = torch.finfo(T[t]).max
    most = [2.0 ** 125, 2.0 ** 126 * 1.25, 2.0 ** 127, top, top]
    x = (torch.rand(len(most), cols, generator=gen(cols)) * 2 - 1).double()
    x = (x * torch.tensor(most, dtype=torch.float64)[:, None]).to(T[t])
    x[:, cols // 3] = torch.tensor(most, dtype=torch.float64).to(T[t])
    x[4] = -top
    return x


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("cols", WIDTHS)
def test_quantize_of_the_largest_rows(gpu, cols, t):
    """The reciprocal of a row's maximum above 2^126 is a subnormal number, that of its scale is not."""
    x = largest_rows(cols, t)
    q, s = quantized(gpu, x, t)
    check_e4m3(q, s, x.double(), 0.0)
    assert (q[4] == 0xFE).all()   # -448


@pytest.mark.parametrize("cols", WIDTHS)
def test_norm_to_e4m3_of_the_largest_weights(gpu, cols):
    """y reaches 2^127 through the weight, h * w with it. The norm's f32 arithmetic is allowed for as everywhere: half a sum's error and ten more."""
    g = gen(cols + 1)
    x = rows(g, 3, cols, torch.float32).clamp(-2, 2)
    w = (torch.rand(cols, generator=g) - 0.5) * 2.0 ** 127
    y, s = torch.full((3, cols), 0x55, dtype=torch.uint8), torch.full((3,), 5.0)
    dy, ds = up(gpu, y), up(gpu, s)
    kernels.rms_norm(up(gpu, x.contiguous()), dy, 3, cols, "f32", weight=up(gpu, w), scales=ds)
    gpu.synchronize()
    _, want = exact_norm(x, None, w, 1e-6)
    assert want.abs().amax(1).min() > 2.0 ** 126
    check_e4m3(down(dy, y), down(ds, s), want, (cols / 2 + 10) * U)
