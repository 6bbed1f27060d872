"""The norm, the row quantisation and the e4m3 and 4-bit products against plain 64-bit arithmetic on the CPU.

Tolerances count roundings. u = 2^-24 is half an f32 step. A norm's f32 arithmetic before the one rounding of y: a sum of at
most `cols` squares costs cols * u of the mean at worst, half of that in its root, and ten more operations are 10 u. A product
of K terms costs at most K * u * sum|a b| (every partial sum is below sum|a b|, and each of the K additions is off by at most
u of it, twice that where the adder truncates; the products themselves are exact in f32), and three more roundings
for scales. On top comes half a step of the output's type."""
import ctypes
import threading

import numpy as np
import pytest
import torch

from basalt_b200 import kernels

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
T = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}      # half a step, relative
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "f32": 2.0 ** -150}  # half a step of the subnormals
SCALE_MIN = 2.0 ** -126


def up(gpu, t):
    """A CPU tensor's bytes on the device; its strides are kept by uploading its whole storage."""
    base = t if t._base is None else t._base
    raw = base.contiguous().view(torch.uint8).reshape(-1).numpy()
    return gpu.upload(raw if raw.size else np.zeros(16, np.uint8))


def down(buf, like):
    base = like if like._base is None else like._base
    raw = torch.from_numpy(buf.to_numpy(np.uint8).copy())[: base.numel() * base.element_size()]
    return raw.view(base.dtype).reshape(base.shape)


def rows(g, n, cols, t, pad=0, scale=1.0, fill=float("nan")):
    """n x cols values of type t inside rows of cols + pad that end in `fill`."""
    buf = torch.full((n, cols + pad), fill, dtype=t)
    buf[:, :cols] = (torch.randn(n, cols, generator=g) * scale).to(t)
    return buf[:, :cols]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def exact_norm(x, res, w, eps):
    h = x.double() if res is None else x.double() + res.double()
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    return h, y if w is None else y * w.double()


def check_e4m3(q_bytes, scales, y, rel):
    """q * s against y: half an e4m3 step (2^-4 of the value, 2^-10 below 2^-6), and the f32 error of y / s."""
    want_scale = torch.clamp(y.abs().amax(1) / 448.0, min=SCALE_MIN)
    assert ((scales.double() - want_scale).abs() <= want_scale * (rel + 2 * U)).all()
    v = y / scales.double()[:, None]
    q = q_bytes.view(torch.float8_e4m3fn).double()
    assert ((q - v).abs() <= torch.maximum(v.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10)) * (1 + 2.0 ** -6) + v.abs() * (rel + 4 * U)).all()
    top = q.abs().amax(1)
    assert ((top == 448) | (y.abs().amax(1) / 448.0 < SCALE_MIN)).all()


NORM_SHAPES = [(1, 1), (3, 7), (5, 8), (2, 64), (130, 64), (7, 128), (33, 96), (9, 1000), (4, 2048), (1, 4096), (3, 5003), (2, 8192), (2, 11008), (2, 32768), (1, 40000), (1, 70000)]


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("out8", [False, True])
@pytest.mark.parametrize("pad", [0, 8, 5])
def test_rms_norm(gpu, t, out8, pad):
    for i, (n, cols) in enumerate(NORM_SHAPES):
        for residual, weight in ((True, True), (False, True), (True, False)):
            g = gen(100 * i + pad)
            x = rows(g, n, cols, T[t], pad)
            res = rows(g, n, cols, T[t], pad + 16, 3.0) if residual else None
            w = (1 + 0.3 * torch.randn(cols, generator=g)).to(T[t]) if weight else None
            y = torch.full((n + 1, cols + pad), 0x55 if out8 else 7.0, dtype=torch.uint8 if out8 else T[t])
            total = torch.full((n, cols + pad), 9.0, dtype=T[t])
            scales = torch.full((n + 1,), 5.0)
            dx, dy, dt, ds = up(gpu, x), up(gpu, y), up(gpu, total), up(gpu, scales)
            dr, dw = up(gpu, res) if residual else None, up(gpu, w) if weight else None
            kernels.rms_norm(dx, dy, n, cols, t, weight=dw, eps=1e-5, residual=dr, total=dt if residual else None, scales=ds if out8 else None, ldx=cols + pad,
                             ldy=cols + pad, ldr=cols + pad + 16, ldt=cols + pad)
            gpu.synchronize()
            h, want = exact_norm(x, res, w, 1e-5)
            got, rel = down(dy, y), (cols / 2 + 10) * U
            what = (t, out8, pad, n, cols, residual, weight)
            if out8:
                check_e4m3(got[:n, :cols].contiguous(), down(ds, scales)[:n], want, rel)
                assert down(ds, scales)[n] == 5.0, what
            else:
                assert ((got[:n, :cols].double() - want).abs() <= want.abs() * (HALF[t] * (1 + 2 ** -7) + rel) + TINY[t]).all(), what
            assert torch.equal(got[n], y[n]) and torch.equal(got[:, cols:], y[:, cols:]), what   # nothing beyond the rows and columns
            if residual:
                back = down(dt, total)
                assert ((back[:, :cols].double() - h).abs() <= h.abs() * (HALF[t] + U) * (1 + 2 ** -7) + TINY[t]).all() and (back[:, cols:] == 9.0).all(), what


@pytest.mark.parametrize("cols", [64, 1001, 4096])
def test_rms_norm_in_place(gpu, cols):
    """total may be the residual's buffer and y the input's: the values are those of separate buffers."""
    g = gen(3)
    x, res, w = rows(g, 5, cols, torch.bfloat16), rows(g, 5, cols, torch.bfloat16), rows(g, 1, cols, torch.bfloat16)
    dx, dr, dw, dy, dt = (up(gpu, v) for v in (x, res, w, x, res))
    kernels.rms_norm(dx, dy, 5, cols, "bf16", weight=dw, residual=dr, total=dt)
    apart = down(dy, x), down(dt, res)
    kernels.rms_norm(dx, dx, 5, cols, "bf16", weight=dw, residual=dr, total=dr)
    gpu.synchronize()
    assert torch.equal(down(dx, x), apart[0]) and torch.equal(down(dr, res), apart[1])
    dx, dr = up(gpu, x), up(gpu, res)
    kernels.rms_norm(dx, dy, 5, cols, "bf16", weight=dw, residual=dr, total=dx)
    assert torch.equal(down(dy, x), apart[0]) and torch.equal(down(dx, res), apart[1])


@pytest.mark.parametrize("cols", [64, 77, 4096])
def test_rows_of_zeros_infinities_and_nans_stay_among_themselves(gpu, cols):
    x = rows(gen(4), 6, cols, torch.float16)
    x[1] = 0
    x[2, cols // 2] = float("inf")
    x[3, cols - 1] = float("nan")
    x[4] = 6e-8   # f16's smallest subnormal
    clean = x.clone()
    clean[2:4] = 1.0
    out = []
    for v in (x, clean):
        y, s = torch.zeros(6, cols, dtype=torch.uint8), torch.zeros(6)
        dx, dy, ds = up(gpu, v.contiguous()), up(gpu, y), up(gpu, s)
        kernels.quantize_e4m3(dx, dy, ds, 6, cols, "f16")
        out.append((down(dy, y), down(ds, s)))
    (y, s), (yc, sc) = out
    ok = [0, 1, 4, 5]
    assert torch.equal(y[ok], yc[ok]) and torch.equal(s[ok], sc[ok])
    check_e4m3(y[ok], s[ok], x[ok].double(), 0.0)
    assert (y[1] == 0).all() and s[1] == SCALE_MIN
    assert torch.isinf(s[2]) and torch.isnan(s[3])
    v = y.view(torch.float8_e4m3fn).float()
    assert torch.isnan(v[2, cols // 2]) and (v[2, : cols // 2] == 0).all() and torch.isnan(v[3]).all()
    w, dy16 = torch.ones(cols, dtype=torch.float16), up(gpu, torch.zeros(6, cols, dtype=torch.float16))
    kernels.rms_norm(up(gpu, x.contiguous()), dy16, 6, cols, "f16", weight=up(gpu, w))
    n = down(dy16, torch.zeros(6, cols, dtype=torch.float16))
    assert torch.isfinite(n[ok]).all() and (n[1] == 0).all() and torch.isnan(n[3]).all() and torch.isnan(n[2, cols // 2]) and (n[2, : cols // 2] == 0).all()


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("cols", [1, 64, 77, 4096, 9001])
def test_norm_of_rows_that_cancel_or_nearly(gpu, t, cols):
    """Rows whose sum with the residual is zero (a padded batch), or so small that the norm's factor times the inverse scale exceeds f32: zeros
    stay zeros, and small values are what the formula says. The small ones are exact in their type, and so are their products with r
    up to one rounding, because they stay normal numbers of f32."""
    x = rows(gen(6), 6, cols, T[t])
    res = torch.zeros_like(x)
    res[1], x[3], res[4] = -x[1], 0, 1.0
    x[4] = -1.0
    if t != "f16":
        x[2] = torch.randint(1, 4, (cols,), generator=gen(7)).to(T[t]) * 2.0 ** -127
        x[5] = 2.0 ** -122
    for residual in (res, None):
        y, sc, total = torch.full((6, cols), 0x55, dtype=torch.uint8), torch.full((6,), 5.0), torch.zeros(6, cols, dtype=T[t])
        dy, ds, dx, w = up(gpu, y), up(gpu, sc), up(gpu, x), up(gpu, torch.ones(cols, dtype=T[t]))
        kernels.rms_norm(dx, dy, 6, cols, t, weight=w, eps=1e-6, residual=None if residual is None else up(gpu, residual), total=None if residual is None else up(gpu, total), scales=ds)
        gpu.synchronize()
        _, want = exact_norm(x, residual, torch.ones(cols, dtype=T[t]), 1e-6)
        check_e4m3(down(dy, y), down(ds, sc), want, (cols / 2 + 10) * U)
        zero = (want == 0).all(1)
        assert (down(dy, y)[zero] & 0x7F == 0).all() and (down(ds, sc)[zero] == SCALE_MIN).all() and zero.sum() >= (1 if residual is None else 3)


@pytest.mark.parametrize("t", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("pad", [0, 5])
def test_quantize(gpu, t, pad):
    for i, (n, cols) in enumerate(NORM_SHAPES):
        x = rows(gen(i), n, cols, T[t], pad)
        y, s = torch.full((n + 1, cols + pad), 0x55, dtype=torch.uint8), torch.full((n + 1,), 5.0)
        dx, dy, ds = up(gpu, x), up(gpu, y), up(gpu, s)
        kernels.quantize_e4m3(dx, dy, ds, n, cols, t, ldx=cols + pad, ldq=cols + pad)
        got, sc = down(dy, y), down(ds, s)
        check_e4m3(got[:n, :cols].contiguous(), sc[:n], x.double(), 0.0)
        assert torch.equal(got[n], y[n]) and (got[:, cols:] == 0x55).all() and sc[n] == 5.0, (t, pad, n, cols)


def e4m3_rows(v, pad):
    """v as e4m3 bytes inside rows whose stride is a multiple of 16 and whose rest is NaN."""
    n, k = v.shape
    buf = torch.full((n, (k + pad + 15) // 16 * 16), 0x7F, dtype=torch.uint8)
    buf[:, :k] = v.to(torch.float8_e4m3fn).view(torch.uint8)
    return buf


def run_e4m3(gpu, a, sa, b, sb, K, out, ldc_pad=3):
    M, N = a.shape[0], b.shape[0]
    c = torch.full((M + 2, N + ldc_pad), 7.0, dtype=T[out])
    status = gpu.upload(np.zeros(1, np.int32))
    da, dsa, db, dsb, dc = up(gpu, a), up(gpu, sa), up(gpu, b), up(gpu, sb), up(gpu, c)
    kernels.matmul_e4m3(da, dsa, db, dsb, dc, M, N, K, out, lda=a.shape[1], ldb=b.shape[1], ldc=N + ldc_pad, status=status)
    gpu.synchronize()
    assert status.to_numpy(np.int32)[0] == 0, "a bounded wait inside the kernel expired"
    got = down(dc, c)
    assert (got[M:] == 7.0).all() and (got[:, N:] == 7.0).all(), "rows or columns beyond the result were written"
    return got[:M, :N]


E4M3_SHAPES = [(1, 1, 1), (1, 128, 128), (2, 127, 16), (7, 129, 31), (16, 300, 127), (17, 64, 129), (33, 260, 1000), (64, 128, 2048), (65, 257, 640), (129, 130, 256), (200, 520, 515),
               (256, 256, 128), (300, 700, 1152), (515, 512, 384), (1, 1000, 8192), (5, 200, 16384), (20, 9000, 2100), (250, 3000, 2200), (120, 4100, 4200), (1000, 2000, 1500),
               (600, 4000, 300), (65, 4100, 4200), (2600, 2100, 1000)]   # the last ones: each tile width with K whole and shared, and pairs of CTAs


@pytest.mark.parametrize("out", ["f32", "f16"])
@pytest.mark.parametrize("shape", E4M3_SHAPES)
def test_matmul_e4m3_exact_on_small_integers(gpu, shape, out):
    M, N, K = shape
    g = gen(M + N + K)
    a = torch.randint(-3, 4, (M, K), generator=g).float()
    b = torch.randint(-2, 3, (N, K), generator=g).float()
    sa, sb = 2.0 ** torch.randint(-3, 3, (M,), generator=g).float(), 2.0 ** torch.randint(-2, 3, (N,), generator=g).float()
    want = ((a.double() @ b.double().T) * sa.double()[:, None] * sb.double()).to(T[out])   # exact sums, one rounding
    got = run_e4m3(gpu, e4m3_rows(a, 5), sa, e4m3_rows(b, 0), sb, K, out)
    bad = (got != want).nonzero()
    assert len(bad) == 0, (len(bad), bad[:5].tolist())


@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("shape", [(1, 300, 4096), (19, 129, 777), (130, 400, 2049), (384, 640, 1024), (2600, 2104, 999)])
def test_matmul_e4m3_random(gpu, shape, out):
    M, N, K = shape
    g = gen(K)
    a, b = (torch.randn(M, K, generator=g) * 60).clamp(-448, 448), (torch.randn(N, K, generator=g) * 60).clamp(-448, 448)
    qa, qb = e4m3_rows(a, 0), e4m3_rows(b, 0)
    sa, sb = torch.rand(M, generator=g) * 0.01 + 1e-4, torch.rand(N, generator=g) * 0.01 + 1e-4
    va, vb = (q.view(torch.float8_e4m3fn).double()[:, :K] for q in (qa, qb))
    scale = sa.double()[:, None] * sb.double()
    want, size = (va @ vb.T) * scale, (va.abs() @ vb.abs().T) * scale
    got = run_e4m3(gpu, qa, sa, qb, sb, K, out, 0).double()
    assert ((got - want).abs() <= want.abs() * (HALF[out] * (1 + 2 ** -7) + 3 * U) + size * 2 * K * U + TINY[out]).all()
    assert float((got - want).norm() / want.norm()) <= 0.6 * HALF[out] + 2.0 ** -19   # what errors of random signs leave: a uniform rounding's spread, and 32 u


@pytest.mark.parametrize("shape", [(3, 130, 16384), (520, 2600, 16300), (150, 140, 20000), (300, 300, 8193)])
def test_matmul_e4m3_long_sums_in_f32(gpu, shape):
    """K in parts of at most 8192, added to C one after the other. The bound is a part's worst: every one of its additions truncated (2 u each)."""
    M, N, K = shape
    g = gen(K)
    qa, qb = e4m3_rows(torch.rand(M, K, generator=g) + 0.5, 0), e4m3_rows(torch.rand(N, K, generator=g) + 0.5, 0)
    sa, sb = torch.rand(M, generator=g) + 0.5, torch.rand(N, generator=g) + 0.5
    va, vb = (q.view(torch.float8_e4m3fn).double()[:, :K] for q in (qa, qb))
    want = (va @ vb.T) * (sa.double()[:, None] * sb.double())
    got = run_e4m3(gpu, qa, sa, qb, sb, K, "f32").double()
    assert ((got - want).abs() <= want * (8192 + 4) * 2 * U).all()


def test_matmul_e4m3_nan_and_infinite_scales_stay_in_their_rows(gpu):
    a, b = e4m3_rows(torch.ones(20, 64), 0), e4m3_rows(torch.ones(140, 64), 0)
    a[3, 10], b[130, 5] = 0x7F, 0xFF
    sa, sb = torch.ones(20), torch.ones(140)
    sa[7], sb[9] = float("inf"), 0.0
    got = run_e4m3(gpu, a, sa, b, sb, 64, "f32")
    want = torch.full((20, 140), 64.0)
    want[:, 9], want[7] = 0.0, float("inf")
    want[7, 9] = want[3] = want[:, 130] = float("nan")
    assert torch.equal(torch.nan_to_num(got, nan=-1.0), torch.nan_to_num(want, nan=-1.0))


def pack(q):
    """Four-bit numbers [N x K], packed two to a byte (k even low) in rows of a multiple of 16 bytes whose rest is ones."""
    N, K = q.shape
    full = torch.full((N, ((K + 1) // 2 + 15) // 16 * 32), 15, dtype=torch.uint8)
    full[:, :K] = q
    return full[:, 0::2] | (full[:, 1::2] << 4)


def run_w4(gpu, x, q, s, z, group, t, ldc_pad=3):
    (M, K), N = x.shape, q.shape[0]
    c = torch.full((M + 2, N + ldc_pad), 7.0, dtype=T[t])
    xb = torch.full((M, (K + 7) // 8 * 8 + 8), float("nan"), dtype=T[t])
    xb[:, :K] = x
    w = pack(q).contiguous()
    status = gpu.upload(np.zeros(1, np.int32))
    dx, dw, ds, dc, dz = up(gpu, xb), up(gpu, w), up(gpu, s), up(gpu, c), None if z is None else up(gpu, z)
    kernels.matmul_w4(dx, dw, ds, dc, M, N, K, group, t, zeros=dz, ldx=xb.shape[1], ldw=w.shape[1], ldc=N + ldc_pad, status=status)
    gpu.synchronize()
    assert status.to_numpy(np.int32)[0] == 0, "a bounded wait inside the kernel expired"
    got = down(dc, c)
    assert (got[M:] == 7.0).all() and (got[:, N:] == 7.0).all(), "rows or columns beyond the result were written"
    return got[:M, :N]


def w4_weights(g, N, K, group, zeros, t, exact):
    groups = -(-K // group)
    q = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    s = (2.0 ** torch.randint(-2, 2, (N, groups), generator=g).float() if exact else 0.01 * (0.5 + torch.rand(N, groups, generator=g))).to(T[t])
    z = torch.randint(0, 16, (N, groups), generator=g, dtype=torch.uint8) if zeros else None
    at = torch.arange(K) // group
    w = (q.double() - (8.0 if z is None else z.double()[:, at])) * s.double()[:, at]
    return q, s, z, w


W4_SHAPES = [(1, 1, 1, 32), (1, 128, 256, 128), (2, 127, 33, 32), (8, 130, 255, 64), (9, 64, 257, 128), (16, 300, 1000, 32), (17, 129, 512, 96), (32, 200, 2048, 128), (33, 140, 300, 64),
             (70, 260, 640, 128), (129, 128, 384, 1024), (200, 300, 1111, 128), (1, 500, 8192, 128), (3, 96, 4096, 64), (1, 140, 16000, 32), (2, 20000, 4500, 128), (13, 19000, 4100, 64), (20, 260, 17000, 96), (31, 20000, 2200, 32), (9, 7000, 129, 128), (5, 129, 2560, 256), (40, 300, 2816, 256), (6, 131, 2048, 64), (70, 130, 4096, 32), (3, 128, 1024, 192),
             # the tcgen05 kernel: wide and narrow tiles, one tile and several a CTA, K whole and shared by two, four and eight
             (520, 4100, 70, 32), (520, 9000, 130, 64), (520, 2100, 777, 96), (400, 520, 8200, 128), (100, 19000, 64, 64), (520, 520, 1111, 128), (700, 130, 3001, 192), (700, 130, 4100, 32),
             (300, 3000, 1400, 256), (2000, 260, 600, 64)]


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("shape", W4_SHAPES)
def test_matmul_w4_exact_on_small_integers(gpu, shape, zeros, t):
    M, N, K, group = shape
    g = gen(M + N + K)
    x = torch.randint(-2, 3, (M, K), generator=g).to(T[t])
    q, s, z, w = w4_weights(g, N, K, group, zeros, t, True)
    want = (x.double() @ w.T).to(T[t])   # quarters below 2^22: exact sums, one rounding
    got = run_w4(gpu, x, q, s, z, group, t)
    bad = (got != want).nonzero()
    assert len(bad) == 0, (len(bad), bad[:5].tolist())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M", [1, 9])
def test_matmul_w4_from_cold_memory(gpu, group, M):
    """Two copies of weights in turn, together more than the L2 cache: the scales of a slab take longest to come, and have to be waited for."""
    N, K, t = 14931, 14720, "bf16"
    g = gen(group + M)
    x = torch.randint(-2, 3, (M, K), generator=g).to(T[t])
    q = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    groups = K // group
    s = (2.0 ** torch.randint(-2, 2, (N, groups), generator=g).float()).to(T[t])
    z = torch.randint(0, 16, (N, groups), generator=g, dtype=torch.uint8)
    want = torch.empty(M, N, dtype=T[t])
    for n in range(0, N, 1024):   # a group's sum times its scale: quarters, exact in 32 bits
        w = (q[n : n + 1024].float().view(-1, groups, group) - z[n : n + 1024].float()[:, :, None]) * s[n : n + 1024].float()[:, :, None]
        want[:, n : n + 1024] = (x.double() @ w.view(-1, K).double().T).to(T[t])
    packed = pack(q).contiguous()
    sets = [[up(gpu, v) for v in (packed, s, z)] for _ in range(2)]
    c = torch.zeros(M, N, dtype=T[t])
    dx, dc = up(gpu, x), up(gpu, c)
    for i in range(100):
        w, sc, zp = sets[i % 2]
        kernels.matmul_w4(dx, w, sc, dc, M, N, K, group, t, zeros=zp, ldw=packed.shape[1])
        gpu.synchronize()
        if i % 2 == 0 or i > 90:
            assert torch.equal(down(dc, c), want), i


@pytest.mark.parametrize("zeros,t", [(True, "f16"), (False, "bf16")])
@pytest.mark.parametrize("K", [300, 330, 407, 450])
def test_matmul_w4_several_wide_tiles_a_cta_and_a_ragged_last_slab(gpu, K, zeros, t):
    """Tiles of 256 rows of X, three for each CTA, where K ends in a slab of which 1, 2, 3 or all of its 64-k tiles are needed."""
    M, N = 768, 148 * 128
    g = gen(K)
    x = torch.randint(-2, 3, (M, K), generator=g).to(T[t])
    q, s, z, w = w4_weights(g, N, K, 128, zeros, t, True)
    want = (x.float() @ w.float().T).to(T[t])   # quarters below 2^20: exact in 32 bits too
    for _ in range(3):
        assert torch.equal(run_w4(gpu, x, q, s, z, 128, t), want)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 300, 4096, 128), (13, 129, 777, 32), (16, 260, 1500, 96), (25, 140, 600, 64), (40, 257, 2049, 64), (150, 100, 900, 64), (300, 384, 1024, 128), (520, 520, 1111, 64), (400, 520, 8200, 128), (100, 19000, 65, 32)])
def test_matmul_w4_random(gpu, shape, t):
    M, N, K, group = shape
    g = gen(K)
    x = torch.randn(M, K, generator=g).to(T[t])
    q, s, z, w = w4_weights(g, N, K, group, M != 1, t, False)
    want, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    got = run_w4(gpu, x, q, s, z, group, t, 0).double()
    # beyond 16 rows a weight may be rounded to X's type before the product: half a step of |w| each
    weight = HALF[t] if M > 16 else 0.0
    assert ((got - want).abs() <= want.abs() * (HALF[t] * (1 + 2 ** -7) + 2 * U) + size * (2 * K * U + weight) + TINY[t]).all()


def test_matmul_w4_infinities_and_nans_stay_in_their_rows(gpu):
    g = gen(9)
    x = torch.randn(10, 300, generator=g).to(torch.float16)
    q, s, z, w = w4_weights(g, 140, 300, 64, True, "f16", False)
    want = run_w4(gpu, x, q, s, z, 64, "f16")
    x[3, 299], s[5, 4] = float("nan"), float("inf")
    got = run_w4(gpu, x, q, s, z, 64, "f16")
    keep = torch.ones(10, 140, dtype=torch.bool)
    keep[3], keep[:, 5] = False, False
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[3]).all() and not torch.isfinite(got[:, 5]).any()


def layer(gpu, dev, rows_n, hidden, width, stream=None):
    """norm -> e4m3 product, and norm -> 4-bit product, on the buffers of `dev`."""
    kernels.rms_norm(dev["x"], dev["q"], rows_n, hidden, "bf16", weight=dev["w"], residual=dev["res"], total=dev["total"], scales=dev["qs"], stream=stream)
    kernels.matmul_e4m3(dev["q"], dev["qs"], dev["b"], dev["bs"], dev["c"], rows_n, width, hidden, "bf16", stream=stream)
    kernels.quantize_e4m3(dev["c"], dev["q2"], dev["q2s"], rows_n, width, "bf16", stream=stream)
    kernels.rms_norm(dev["total"], dev["y"], rows_n, hidden, "bf16", weight=dev["w"], stream=stream)
    kernels.matmul_w4(dev["y"], dev["w4"], dev["w4s"], dev["c4"], rows_n, width, hidden, 128, "bf16", stream=stream)


LAYER_OUT = ("q", "qs", "total", "c", "q2", "q2s", "y", "c4")


def layer_buffers(seed, rows_n, hidden, width):
    g = gen(seed)
    q, s, _, w4 = w4_weights(g, width, hidden, 128, False, "bf16", False)
    b = (torch.randn(width, hidden, generator=g) * 40).clamp(-448, 448).to(torch.float8_e4m3fn)
    host = {"x": rows(g, rows_n, hidden, torch.bfloat16).contiguous(), "res": rows(g, rows_n, hidden, torch.bfloat16).contiguous(), "w": (1 + 0.2 * torch.randn(hidden, generator=g)).bfloat16(),
            "b": b.view(torch.uint8), "bs": torch.rand(width, generator=g) * 1e-3 + 1e-4, "w4": pack(q).contiguous(), "w4s": s}
    host.update(q=torch.zeros(rows_n, hidden, dtype=torch.uint8), qs=torch.zeros(rows_n), total=torch.zeros(rows_n, hidden, dtype=torch.bfloat16),
                c=torch.zeros(rows_n, width, dtype=torch.bfloat16), q2=torch.zeros(rows_n, width, dtype=torch.uint8), q2s=torch.zeros(rows_n),
                y=torch.zeros(rows_n, hidden, dtype=torch.bfloat16), c4=torch.zeros(rows_n, width, dtype=torch.bfloat16))
    return host, w4


@pytest.mark.parametrize("rows_n", [1, 12, 150])
def test_a_layer_of_them(gpu, rows_n):
    """Each step against 64 bits on what the step before it really wrote, so every tolerance is the operator's own."""
    hidden, width = 512, 384
    host, w4 = layer_buffers(rows_n, rows_n, hidden, width)
    dev = {k: up(gpu, v) for k, v in host.items()}
    layer(gpu, dev, rows_n, hidden, width)
    gpu.synchronize()
    got = {k: down(dev[k], host[k]) for k in LAYER_OUT}
    rel, half = (hidden / 2 + 10) * U, HALF["bf16"]
    h, y = exact_norm(host["x"], host["res"], host["w"], 1e-6)
    assert ((got["total"].double() - h).abs() <= h.abs() * (half + U) * (1 + 2 ** -7)).all()
    check_e4m3(got["q"], got["qs"], y, rel)
    a = got["q"].view(torch.float8_e4m3fn).double() * got["qs"].double()[:, None]
    b = host["b"].view(torch.float8_e4m3fn).double() * host["bs"].double()[:, None]
    want = a @ b.T
    assert ((got["c"].double() - want).abs() <= want.abs() * (half * (1 + 2 ** -7) + 3 * U) + 2 * hidden * U * (a.abs() @ b.abs().T)).all()
    check_e4m3(got["q2"], got["q2s"], got["c"].double(), 0.0)
    _, y = exact_norm(got["total"], None, host["w"], 1e-6)
    assert ((got["y"].double() - y).abs() <= y.abs() * (half * (1 + 2 ** -7) + rel)).all()
    x = got["y"].double()
    want, size = x @ w4.T, x.abs() @ w4.abs().T
    weight = half if rows_n > 16 else 0.0
    assert ((got["c4"].double() - want).abs() <= want.abs() * (half * (1 + 2 ** -7) + 2 * U) + size * (2 * hidden * U + weight)).all()


@pytest.mark.parametrize("size", [(12, 1024, 640), (520, 2048, 1030)])
def test_two_streams_at_once_and_again_give_the_same_bits(gpu, size):
    """Also where both products share K among clusters, and one of them takes all tensor memory of its SMs."""
    streams = [gpu.create_stream(), gpu.create_stream()]
    hosts = [layer_buffers(s, *size)[0] for s in (1, 2)]
    alone = []
    for h in hosts:
        dev = {k: up(gpu, v) for k, v in h.items()}
        layer(gpu, dev, *size)
        gpu.synchronize()
        alone.append({k: down(dev[k], h[k]) for k in LAYER_OUT})
    devs = [{k: up(gpu, v) for k, v in h.items()} for h in hosts]
    for _ in range(20):
        for d, s in zip(devs, streams):
            layer(gpu, d, *size, stream=s)
    gpu.synchronize()
    for d, h, want in zip(devs, hosts, alone):
        assert all(torch.equal(down(d[k], h[k]).view(torch.uint8), want[k].view(torch.uint8)) for k in LAYER_OUT)
    for s in streams:
        gpu.destroy_stream(s)


def test_captured_into_a_graph_and_replayed_on_new_inputs(gpu):
    host, _ = layer_buffers(5, 12, 1024, 640)
    other, _ = layer_buffers(6, 12, 1024, 640)
    dev = {k: v.cuda() for k, v in host.items()}
    ptr = {k: v.data_ptr() for k, v in dev.items()}
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        layer(gpu, ptr, 12, 1024, 640, stream=torch.cuda.current_stream().cuda_stream)
    for inputs in (host, other):
        for k, v in inputs.items():
            dev[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        got = {k: dev[k].cpu() for k in LAYER_OUT}
        fresh = {k: up(gpu, v) for k, v in inputs.items()}
        layer(gpu, fresh, 12, 1024, 640)
        gpu.synchronize()
        assert all(torch.equal(got[k].view(torch.uint8), down(fresh[k], inputs[k]).view(torch.uint8)) for k in LAYER_OUT)


def test_rows_a_gigabyte_apart(gpu):
    """Offsets past 2^31 elements in every matrix that has a row stride."""
    ld, n, k, cols = 2**30 + 16, 200, 300, 1000
    g = gen(11)
    x, res, w = rows(g, 3, cols, torch.float16), rows(g, 3, cols, torch.float16), rows(g, 1, cols, torch.float16)[0]
    big = [torch.empty(2 * ld + 4096, dtype=torch.float16, device="cuda") for _ in range(2)]
    apart = lambda b, r, c, t=torch.float16: b.view(t)[: 2 * ld + c].as_strided((r, c), (ld, 1))  # noqa: E731
    near = {name: v.cuda() for name, v in (("x", x.contiguous()), ("res", res.contiguous()), ("w", w))}
    out = {}
    for far in (False, True):
        xs = apart(big[0], 3, cols) if far else near["x"]
        xs.copy_(x)
        ys = apart(big[1], 3, cols) if far else torch.empty(3, cols, dtype=torch.float16, device="cuda")
        kernels.rms_norm(xs.data_ptr(), ys.data_ptr(), 3, cols, "f16", weight=near["w"].data_ptr(), residual=near["res"].data_ptr(), ldx=xs.stride(0), ldy=ys.stride(0))
        out.setdefault("norm", []).append(ys.clone())
        q = apart(big[1], 3, cols, torch.uint8) if far else torch.empty(3, cols, dtype=torch.uint8, device="cuda")
        s = torch.empty(3, device="cuda")
        kernels.quantize_e4m3(xs.data_ptr(), q.data_ptr(), s.data_ptr(), 3, cols, "f16", ldx=xs.stride(0), ldq=q.stride(0))
        out.setdefault("quantize", []).append(q.clone())
    a = torch.randint(-3, 4, (3, k), generator=g).float().to(torch.float8_e4m3fn).view(torch.uint8)
    b = torch.randint(-3, 4, (3, k), generator=g).float().to(torch.float8_e4m3fn).view(torch.uint8)
    x4, w4 = torch.randint(-3, 4, (3, k), generator=g).half(), torch.randint(0, 256, (3, k // 2), generator=g, dtype=torch.uint8)
    one = torch.ones(n, device="cuda")
    s4 = torch.ones(3, 10, dtype=torch.float16, device="cuda")
    pad = lambda t, to: torch.nn.functional.pad(t, (0, to - t.shape[1])).contiguous().cuda()  # noqa: E731
    for far in (False, True):
        aa, bb = (apart(big[0], 3, k, torch.uint8), apart(big[1], 3, k, torch.uint8)) if far else (pad(a, 304), pad(b, 304))
        aa[:, :k].copy_(a), bb[:, :k].copy_(b)
        c = torch.empty(3, 3, dtype=torch.float32, device="cuda")
        kernels.matmul_e4m3(aa.data_ptr(), one.data_ptr(), bb.data_ptr(), one.data_ptr(), c.data_ptr(), 3, 3, k, "f32", lda=aa.stride(0), ldb=bb.stride(0))
        out.setdefault("e4m3", []).append(c)
        xx, ww = (apart(big[0], 3, k), apart(big[1], 3, k // 2, torch.uint8)) if far else (pad(x4, 304), pad(w4, 160))
        xx[:, :k].copy_(x4), ww[:, : k // 2].copy_(w4)
        c = torch.empty(3, 3, dtype=torch.float16, device="cuda")
        kernels.matmul_w4(xx.data_ptr(), ww.data_ptr(), s4.data_ptr(), c.data_ptr(), 3, 3, k, 32, "f16", ldx=xx.stride(0), ldw=ww.stride(0))
        out.setdefault("w4", []).append(c)
    far_c = apart(big[0], 3, 3)
    kernels.matmul_w4(pad(x4, 304).data_ptr(), ww.data_ptr(), s4.data_ptr(), far_c.data_ptr(), 3, 3, k, 32, "f16", ldx=304, ldw=ww.stride(0), ldc=ld)
    out["w4"].append(far_c)
    for name, got in out.items():
        assert all(torch.equal(v, got[0]) for v in got[1:]), name


def test_a_thread_that_has_made_no_call_before(gpu):
    host, _ = layer_buffers(7, 12, 1024, 640)
    dev = {k: up(gpu, v) for k, v in host.items()}
    layer(gpu, dev, 12, 1024, 640)
    gpu.synchronize()
    want = {k: down(dev[k], host[k]) for k in LAYER_OUT}
    fresh, trouble = {k: up(gpu, v) for k, v in host.items()}, []

    def run():
        try:
            layer(gpu, fresh, 12, 1024, 640)
        except Exception as e:
            trouble.append(e)

    thread = threading.Thread(target=run)
    thread.start()
    thread.join()
    gpu.synchronize()
    assert not trouble, trouble
    assert all(torch.equal(down(fresh[k], host[k]).view(torch.uint8), want[k].view(torch.uint8)) for k in LAYER_OUT)


def test_pointers_outside_device_memory_are_refused(gpu):
    host = np.zeros(4096, np.float16)
    p = host.ctypes.data_as(ctypes.c_void_p).value & ~15
    d = gpu.upload(np.zeros(4096, np.float32))
    with pytest.raises(kernels.KernelError, match="device memory"):
        kernels.rms_norm(p, d, 1, 64, "f16")
    with pytest.raises(kernels.KernelError, match="device memory"):
        kernels.matmul_e4m3(d, p, d.device_ptr() + 1024, d.device_ptr() + 4096, d.device_ptr() + 8192, 1, 16, 64)
    with pytest.raises(kernels.KernelError, match="device memory"):
        kernels.matmul_w4(d, d.device_ptr() + 1024, p, d.device_ptr() + 8192, 1, 16, 64, 32)
