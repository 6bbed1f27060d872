"""Calls of the quantised layer's operators at the ends of their ranges: the largest rows, exact ties, weights from cold
memory, long sums, matrices that share a buffer."""
import os
import subprocess
import sys

import pytest
import torch

from basalt_b200 import kernels
from test_gpu_quantized import T, U, check_e4m3, down, e4m3_rows, exact_norm, gen, rows, run_e4m3, up

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

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


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("cols", WIDTHS)
def test_norm_of_rows_whose_squares_exceed_f32_is_zero(gpu, cols, t):
    """Their mean is infinite in f32; the rows beside them are what they are alone."""
    x = rows(gen(cols), 4, cols, T[t])
    x[1], x[2, cols - 1] = -torch.finfo(T[t]).max, 2.0 ** 64
    for out8 in (False, True):
        got = []
        for v in (x, x[[0, 3]]):
            n = v.shape[0]
            y, s = torch.full((n, cols), 0x55, dtype=torch.uint8) if out8 else torch.full((n, cols), 7.0, dtype=T[t]), torch.full((n,), 5.0)
            dy, ds = up(gpu, y), up(gpu, s)
            kernels.rms_norm(up(gpu, v.contiguous()), dy, n, cols, t, scales=ds if out8 else None)
            gpu.synchronize()
            got.append((down(dy, y), down(ds, s)))
        (y, s), (alone, s_alone) = got
        assert torch.equal(y[[0, 3]], alone) and torch.equal(s[[0, 3]], s_alone)
        assert ((y[1:3] & 0x7F if out8 else y[1:3]) == 0).all() and (not out8 or (s[1:3] == 2.0 ** -126).all())


def e4m3_of_the_quotient(y, s):
    """y / s in f32, as the CPU divides, then e4m3 to the nearest, ties to even."""
    return (y.float() / s[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def rows_of_ties(cols, t, exponent):
    """Rows whose largest magnitude is 448 * 2^exponent, so that the scale is 2^exponent, and whose other values are e4m3 numbers and the points
    half-way between two of them, of both signs: odd multiples of half a step, the subnormals' among them, and zeros."""
    e4m3 = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    points = torch.cat([e4m3, (e4m3[1:] + e4m3[:-1]) / 2])
    points = torch.cat([points, -points])
    x = points[torch.randint(0, len(points), (3, cols), generator=gen(cols))]
    x[:, cols - 1] = 448.0
    x = (x * 2.0 ** exponent).to(T[t])
    assert torch.equal((x.double() * 2.0 ** -exponent * 1024).frac(), torch.zeros(3, cols, dtype=torch.float64))   # nothing was rounded
    return x


@pytest.mark.parametrize("t,exponent", [("f16", 0), ("f16", 6), ("bf16", 0), ("bf16", 119), ("bf16", -100), ("f32", 0), ("f32", -126), ("f32", -91), ("f32", -90), ("f32", 100)])
@pytest.mark.parametrize("cols", WIDTHS)
def test_quantize_ties_go_to_even(gpu, cols, t, exponent):
    x = rows_of_ties(cols, t, exponent)
    q, s = quantized(gpu, x, t)
    assert (s == 2.0 ** exponent).all()
    assert torch.equal(q, e4m3_of_the_quotient(x, s))


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -9, 700.0])
def test_quantize_is_the_quotient_by_the_stored_scale(gpu, cols, t, scale):
    """The scale is the f32 quotient max / 448, the bytes are those of the f32 quotient x / scale. (A quotient that f32 holds is met exactly and
    any other within half a step and 2^-45 of it, so that a byte could differ from these only where a division comes as near as that
    to the middle of two f32 numbers; none of 24 bits by 24 does outside subnormals.) 16-bit rows meet ties often."""
    x = rows(gen(cols), 40 if cols < 9000 else 5, cols, T[t], 0, scale)
    q, s = quantized(gpu, x, t)
    assert torch.equal(s, x.float().abs().amax(1) / torch.full((x.shape[0],), 448.0))
    assert torch.equal(q, e4m3_of_the_quotient(x, s))


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_to_e4m3_ties_go_to_even(gpu, cols, t, residual):
    """h = +-1 and eps = 0: the mean of squares and its root are exactly one, y is the weight with h's sign, and ties are ties."""
    w = rows_of_ties(cols, t, 0)[0]
    h = torch.where(torch.rand(3, cols, generator=gen(cols)) < 0.5, -1.0, 1.0).to(T[t])
    r = torch.randint(-4, 5, (3, cols), generator=gen(cols + 1)).to(T[t])
    x = h - r if residual else h
    y, s = torch.full((3, cols), 0x55, dtype=torch.uint8), torch.full((3,), 5.0)
    dy, ds = up(gpu, y), up(gpu, s)
    total = up(gpu, torch.zeros_like(x)) if residual else None
    kernels.rms_norm(up(gpu, x), dy, 3, cols, t, weight=up(gpu, w), eps=0.0, residual=up(gpu, r) if residual else None, total=total, scales=ds)
    gpu.synchronize()
    q, s = down(dy, y), down(ds, s)
    assert (s == 1.0).all()
    assert torch.equal(q, e4m3_of_the_quotient(h.float() * w.float(), s))


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("K", [14720, 14848])   # groups of 32, 64 and 128 in whole aligned pieces in the second only
@pytest.mark.parametrize("group", [32, 64, 96, 128])
def test_matmul_w4_in_every_form_from_cold_memory(gpu, group, K, zeros, t):
    """Every launch is compared, the caches overwritten before it: the scales of a slab take longest to come then, and have to be waited for. M
    goes through tiles of 8 and 16 rows and through narrow, middling and wide tiles of the tcgen05 kernel."""
    N, dev = 14931, "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(group + K)
    groups = -(-K // group)
    q = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8, device=dev)
    s = (2.0 ** torch.randint(-2, 2, (N, groups), generator=g, device=dev).float()).to(T[t])
    z = torch.randint(0, 16, (N, groups), generator=g, dtype=torch.uint8, device=dev) if zeros else None
    at = torch.arange(K, device=dev) // group
    w = (q.float() - (8.0 if z is None else z.float()[:, at])) * s.float()[:, at]
    packed = q[:, 0::2] | (q[:, 1::2] << 4)
    caches = torch.empty(256 << 20, dtype=torch.uint8, device=dev)
    stream = torch.cuda.current_stream().cuda_stream
    for M in (1, 9, 64, 150, 300):
        x = torch.randint(-2, 3, (M, K), generator=g, device=dev).to(T[t])
        want = (x.float() @ w.T).to(T[t])   # quarters below 2^20: exact in 32 bits in any order
        c = torch.empty(M, N, dtype=T[t], device=dev)
        for i in range(60):
            caches.fill_(i)
            kernels.matmul_w4(x.data_ptr(), packed.data_ptr(), s.data_ptr(), c.data_ptr(), M, N, K, group, t, zeros=None if z is None else z.data_ptr(), stream=stream)
            assert torch.equal(c, want), (M, i, int((c != want).sum()))


@pytest.mark.parametrize("ldc_pad", [0, 4, 3])   # C's rows are whole 16-byte pieces, with a gap or without one, or not
@pytest.mark.parametrize("shape", [(1000, 2600, 16300), (1030, 2100, 8200), (600, 4100, 24600), (150, 700, 20000), (5, 68, 16400)])
def test_matmul_e4m3_parts_are_added_to_f32(gpu, shape, ldc_pad):
    """A K beyond 8192 in two, three and four parts, the later ones added to what C holds: on pairs of CTAs (the first three shapes) in whole pieces and element by
    element, and in narrower tiles. Sums of small integers below 2^24 are exact whatever their order."""
    M, N, K = shape
    g = gen(M + K)
    a, b = torch.randint(-3, 4, (M, K), generator=g).float(), torch.randint(-2, 3, (N, K), generator=g).float()
    sa, sb = 2.0 ** torch.randint(-3, 3, (M,), generator=g).float(), 2.0 ** torch.randint(-2, 3, (N,), generator=g).float()
    want = (a @ b.T) * sa[:, None] * sb
    got = run_e4m3(gpu, e4m3_rows(a, 5), sa, e4m3_rows(b, 0), sb, K, "f32", ldc_pad)
    assert torch.equal(got, want), int((got != want).sum())


@pytest.mark.parametrize("cols", [64, 77, 4096, 9001])
def test_norm_beside_its_input_in_one_buffer(gpu, cols):
    g = gen(cols)
    both = torch.cat([rows(g, 5, cols, torch.bfloat16), torch.full((5, cols), 3.0, dtype=torch.bfloat16)], 1)
    w = rows(g, 1, cols, torch.bfloat16)
    db, dw, dx, dy = up(gpu, both), up(gpu, w), up(gpu, both[:, :cols].contiguous()), up(gpu, both[:, cols:].contiguous())
    kernels.rms_norm(db, db.device_ptr() + 2 * cols, 5, cols, "bf16", weight=dw, ldx=2 * cols, ldy=2 * cols)
    kernels.rms_norm(dx, dy, 5, cols, "bf16", weight=dw)
    gpu.synchronize()
    got = down(db, both)
    assert torch.equal(got[:, :cols], both[:, :cols]) and torch.equal(got[:, cols:], down(dy, torch.empty(5, cols, dtype=torch.bfloat16)))


@pytest.mark.parametrize("M", [3, 20, 300])
def test_products_beside_their_input_in_one_buffer(gpu, M):
    K = N = 256
    g = gen(M)
    x, q, s = torch.randint(-2, 3, (M, K), generator=g).half(), torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8), torch.ones(N, K // 32, dtype=torch.float16)
    both = torch.cat([x, torch.full((M, N), 7.0, dtype=torch.float16)], 1)
    db = up(gpu, both)
    kernels.matmul_w4(db, up(gpu, q[:, 0::2] | (q[:, 1::2] << 4)), up(gpu, s), db.device_ptr() + 2 * K, M, N, K, 32, "f16", ldx=2 * K, ldc=2 * K)
    got = down(db, both)
    assert torch.equal(got[:, :K], x) and torch.equal(got[:, K:], (x.float() @ (q.float() - 8).T).half())
    a, b = torch.randint(-3, 4, (M, K), generator=g).float(), torch.randint(-2, 3, (N // 2, K), generator=g).float()
    both = torch.cat([e4m3_rows(a, 0), torch.full((M, N), 1, dtype=torch.uint8)], 1)   # 256 bytes of A, 128 f16 of C
    db = up(gpu, both)
    kernels.matmul_e4m3(db, up(gpu, torch.ones(M)), up(gpu, e4m3_rows(b, 0)), up(gpu, torch.ones(N // 2)), db.device_ptr() + K, M, N // 2, K, "f16", lda=2 * K, ldc=K)
    got = down(db, both)
    assert torch.equal(got[:, :K], both[:, :K]) and torch.equal(got[:, K:].contiguous().view(torch.float16), (a @ b.T).half())


@pytest.mark.parametrize("M", [1, 40, 600])
def test_the_scales_of_the_norm_before_reach_the_product(gpu, M):
    """The product's kernel begins while the norm still runs; what it reads of the scales has to be this norm's, not the one's before."""
    K, N, n = 4096, 520, 40
    g = gen(M)
    b = e4m3_rows((torch.randn(N, K, generator=g) * 40).clamp(-448, 448), 0)
    db, dbs, dq, dqs = up(gpu, b), up(gpu, torch.full((N,), 0.01)), up(gpu, torch.zeros(M, K, dtype=torch.uint8)), up(gpu, torch.zeros(M))
    xs = [up(gpu, torch.randn(M, K, generator=g).half() * 1.5 ** (i % 7)) for i in range(n)]
    out = []
    for wait in (True, False):
        cs = [up(gpu, torch.zeros(M, N)) for _ in range(n)]
        for x, c in zip(xs, cs):
            kernels.quantize_e4m3(x, dq, dqs, M, K, "f16")
            if wait:
                gpu.synchronize()
            kernels.matmul_e4m3(dq, dqs, db, dbs, c, M, N, K, "f32")
            if wait:
                gpu.synchronize()
        gpu.synchronize()
        out.append([down(c, torch.empty(M, N)) for c in cs])
    for apart, together in zip(*out):
        assert torch.equal(apart, together)


FIRST_CALL_CAPTURED = """
import torch
from basalt_b200 import kernels
x, w, q, s = torch.randn(4, 512, device="cuda").half(), torch.ones(512, device="cuda").half(), torch.empty(4, 512, dtype=torch.uint8, device="cuda"), torch.empty(4, device="cuda")
b, bs, c = torch.zeros(256, 512, dtype=torch.uint8, device="cuda"), torch.ones(256, device="cuda"), torch.ones(4, 256, device="cuda").half()
w4, w4s, c4 = torch.full((256, 256), 0x99, dtype=torch.uint8, device="cuda"), torch.ones(256, 4, device="cuda").half(), torch.zeros(4, 256, device="cuda").half()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    st = torch.cuda.current_stream().cuda_stream
    kernels.rms_norm(x.data_ptr(), q.data_ptr(), 4, 512, "f16", weight=w.data_ptr(), scales=s.data_ptr(), stream=st)
    kernels.matmul_e4m3(q.data_ptr(), s.data_ptr(), b.data_ptr(), bs.data_ptr(), c.data_ptr(), 4, 256, 512, "f16", stream=st)
    kernels.matmul_w4(x.data_ptr(), w4.data_ptr(), w4s.data_ptr(), c4.data_ptr(), 4, 256, 512, 128, "f16", stream=st)
graph.replay()
torch.cuda.synchronize()
assert (c == 0).all() and (s > 0).all() and torch.allclose(c4.float(), x.float().sum(1, keepdim=True).expand(4, 256), rtol=2**-10, atol=2**-10)
"""


def test_the_first_call_of_a_process_may_be_captured(gpu):
    done = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr
