"""The operators of a quantised linear layer, as they are timed and checked: the root-mean-square norm that feeds
it, the quantisation of rows to e4m3, the e4m3 product with row scales and the product with 4-bit weights.

`run` takes what `prepare` gives through one operator: in elementary torch operations where `own` is false, through
basalt_b200.kernels where it is true. `exact` says what the result is in 64 bits."""
import math

import torch

own = False

E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4, "e4m3": 1}


def listed():
    return [
        # The norm before a layer while one sequence decodes: one token, its residual stream, 8-bit output.
        {"name": "norm_token", "op": "norm", "rows": 1, "cols": 4096, "type": "f16", "residual": True, "out": "e4m3", "pad": 0},
        # The same for a batch of decoding sequences, its output in 16 bits for the 4-bit product.
        {"name": "norm_batch", "op": "norm", "rows": 48, "cols": 8192, "type": "bf16", "residual": True, "out": "same", "pad": 0},
        # An odd width, rows that start at no vector boundary, no residual: the first norm of a ragged model.
        {"name": "norm_ragged", "op": "norm", "rows": 1023, "cols": 5003, "type": "bf16", "residual": False, "out": "e4m3", "pad": 0},
        # A long prompt.
        {"name": "norm_prefill", "op": "norm", "rows": 8192, "cols": 8192, "type": "f16", "residual": True, "out": "e4m3", "pad": 0},
        # The activation before the second product of a feed-forward block, one token.
        {"name": "quantize_token", "op": "quantize", "rows": 1, "cols": 11008, "type": "f16", "pad": 0},
        # The same over a long prompt, read from inside a wider buffer.
        {"name": "quantize_prefill", "op": "quantize", "rows": 4096, "cols": 14336, "type": "bf16", "pad": 64},
        # A projection while one sequence decodes: the weights are read for one row.
        {"name": "e4m3_token", "op": "e4m3", "M": 1, "N": 8192, "K": 8192, "out": "f16"},
        # A small ragged batch on odd widths, nothing a multiple of a tile.
        {"name": "e4m3_ragged", "op": "e4m3", "M": 77, "N": 4100, "K": 4104, "out": "bf16"},
        # A long prompt through a square projection: the size of the fp16 matmul of the benchmark.
        {"name": "e4m3_prefill", "op": "e4m3", "M": 8192, "N": 8192, "K": 8192, "out": "f16"},
        # One token through 4-bit weights.
        {"name": "w4_token", "op": "w4", "M": 1, "N": 8192, "K": 8192, "group": 128, "zeros": False, "type": "f16"},
        # A batch of decoding sequences, weights with zero points in small groups.
        {"name": "w4_batch", "op": "w4", "M": 16, "N": 14336, "K": 4096, "group": 64, "zeros": True, "type": "bf16"},
        # A prompt through 4-bit weights.
        {"name": "w4_prefill", "op": "w4", "M": 2048, "N": 4096, "K": 11008, "group": 128, "zeros": False, "type": "f16"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _width(rng, lo, hi):
    """Mostly widths that a model has (multiples of 128), a third of them any number."""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.34 or n < 128 else n // 128 * 128


def draw(rng):
    op = rng.choice(["norm", "norm", "quantize", "e4m3", "e4m3", "w4", "w4"])
    if op in ("norm", "quantize"):
        cols = _width(rng, 1, 16384)
        rows = _log(rng, 1, max(1, min(8192, (1 << 26) // cols)))
        case = {"op": op, "rows": rows, "cols": cols, "type": rng.choice(["f16", "bf16", "f32"]), "pad": rng.choice([0, 0, 8, 5])}
        if op == "norm":
            case["residual"] = rng.random() < 0.7
            case["out"] = rng.choice(["e4m3", "same"])
        return case
    N, K = _width(rng, 1, 16384), _width(rng, 16, 16384)
    if op == "e4m3":
        M = _log(rng, 1, min(8192, (1 << 39) // (N * K)))
        return {"op": op, "M": M, "N": N, "K": K, "out": rng.choice(["f16", "bf16", "f32"])}
    M = _log(rng, 1, min(4096, (1 << 36) // (N * K)))
    return {"op": op, "M": M, "N": N, "K": K, "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5, "type": rng.choice(["f16", "bf16"])}


def _up(n, to):
    return -(-n // to) * to


def _rows(g, rows, cols, kind, pad, scale=1.0):
    """Rows of activations: normal values, a few channels much larger, inside rows of cols + pad elements that end in NaN."""
    t = TYPES[kind]
    buf = torch.full((rows, cols + pad), float("nan"), device="cuda", dtype=t)
    channel = torch.ones(cols, device="cuda")
    channel[torch.randint(0, cols, (max(1, cols // 200),), device="cuda", generator=g)] = 12.0
    x = torch.randn(rows, cols, device="cuda", generator=g)
    buf[:, :cols] = (x.mul_(channel).mul_(scale)).to(t)
    return buf[:, :cols]


def _e4m3(x):
    """x (f32) as e4m3 rows in a buffer whose rows are 16-byte multiples (the rest NaN), and their scales."""
    rows, cols = x.shape
    scale = (x.abs().amax(1) / E4M3_MAX).clamp(min=SCALE_MIN)
    buf = torch.full((rows, _up(cols, 16)), 0x7F, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    buf[:, :cols] = x.div_(scale[:, None]).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return buf[:, :cols], scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] in ("norm", "quantize"):
        rows, cols, kind, pad = case["rows"], case["cols"], case["type"], case["pad"]
        s["x"] = _rows(g, rows, cols, kind, pad)
        eight = case.get("out", "e4m3") == "e4m3"
        s["y"] = torch.empty(rows, _up(cols, 16) if eight else cols + pad, device="cuda", dtype=torch.float8_e4m3fn if eight else TYPES[kind])[:, :cols]
        s["scales"] = torch.empty(rows, device="cuda") if eight else None
        if case["op"] == "norm":
            s["weight"] = (1.0 + 0.3 * torch.randn(cols, device="cuda", generator=g)).to(TYPES[kind])
            s["res"] = _rows(g, rows, cols, kind, pad, 3.0) if case["residual"] else None
            s["sum"] = torch.empty(rows, cols + pad, device="cuda", dtype=TYPES[kind])[:, :cols] if case["residual"] else None
        return s
    M, N, K = case["M"], case["N"], case["K"]
    if case["op"] == "e4m3":
        s["a"], s["a_scales"] = _e4m3(_rows(g, M, K, "f32", 0).contiguous())
        s["b"], s["b_scales"] = _e4m3(torch.randn(N, K, device="cuda", generator=g).mul_(0.02))
        s["c"] = torch.empty(M, N, device="cuda", dtype=TYPES[case["out"]])
        return s
    groups = -(-K // case["group"])
    s["x"] = _rows(g, M, K, case["type"], _up(K, 8) - K)
    q = torch.randn(N, _up(K, 32), device="cuda", generator=g).mul_(2.6).add_(8.0).round_().clamp_(0, 15).to(torch.uint8)
    s["w"] = q[:, 0::2] | (q[:, 1::2] << 4)
    s["w_scales"] = (0.008 * (0.5 + torch.rand(N, groups, device="cuda", generator=g))).to(TYPES[case["type"]])
    s["w_zeros"] = torch.randint(5, 12, (N, groups), device="cuda", generator=g, dtype=torch.uint8) if case["zeros"] else None
    s["c"] = torch.empty(M, N, device="cuda", dtype=TYPES[case["type"]])
    return s


def _own_run(s):
    from basalt_b200 import kernels

    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "norm":
        x, y, res, total, scales = s["x"], s["y"], s["res"], s["sum"], s["scales"]
        kernels.rms_norm(x.data_ptr(), y.data_ptr(), s["rows"], s["cols"], s["type"], weight=s["weight"].data_ptr(), eps=1e-6,
                         residual=None if res is None else res.data_ptr(), total=None if total is None else total.data_ptr(),
                         scales=None if scales is None else scales.data_ptr(), ldx=x.stride(0), ldy=y.stride(0),
                         ldr=None if res is None else res.stride(0), ldt=None if total is None else total.stride(0), stream=stream)
        return {k: v for k, v in (("y", y), ("scales", scales), ("sum", total)) if v is not None}
    if s["op"] == "quantize":
        x, y = s["x"], s["y"]
        kernels.quantize_e4m3(x.data_ptr(), y.data_ptr(), s["scales"].data_ptr(), s["rows"], s["cols"], s["type"], ldx=x.stride(0), ldq=y.stride(0), stream=stream)
        return {"y": y, "scales": s["scales"]}
    if s["op"] == "e4m3":
        a, b, c = s["a"], s["b"], s["c"]
        kernels.matmul_e4m3(a.data_ptr(), s["a_scales"].data_ptr(), b.data_ptr(), s["b_scales"].data_ptr(), c.data_ptr(), s["M"], s["N"], s["K"], s["out"],
                            lda=a.stride(0), ldb=b.stride(0), ldc=c.stride(0), stream=stream)
        return c
    x, w, c, zeros = s["x"], s["w"], s["c"], s["w_zeros"]
    kernels.matmul_w4(x.data_ptr(), w.data_ptr(), s["w_scales"].data_ptr(), c.data_ptr(), s["M"], s["N"], s["K"], s["group"], s["type"],
                      zeros=None if zeros is None else zeros.data_ptr(), ldx=x.stride(0), ldw=w.stride(0), ldc=c.stride(0), stream=stream)
    return c


def _to_e4m3(y):
    scale = (y.abs().amax(1) / E4M3_MAX).clamp(min=SCALE_MIN)
    return (y / scale[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def run(s):
    if own:
        return _own_run(s)
    if s["op"] == "norm":
        h = s["x"].float()
        if s["res"] is not None:
            h = h + s["res"].float()
        y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + 1e-6) * s["weight"].float()
        got = dict(zip(("y", "scales"), _to_e4m3(y))) if s["out"] == "e4m3" else {"y": y.to(s["x"].dtype)}
        return got if s["res"] is None else {**got, "sum": h.to(s["x"].dtype)}
    if s["op"] == "quantize":
        return dict(zip(("y", "scales"), _to_e4m3(s["x"].float())))
    if s["op"] == "e4m3":
        return ((s["a"].float() @ s["b"].float().T) * s["a_scales"][:, None] * s["b_scales"]).to(s["c"].dtype)
    K, w = s["K"], s["w"]
    q = torch.stack([w & 15, w >> 4], 2).reshape(w.shape[0], -1)[:, :K].float()
    spread = lambda t: t.float().repeat_interleave(s["group"], 1)[:, :K]  # noqa: E731
    q = q - (8.0 if s["w_zeros"] is None else spread(s["w_zeros"]))
    return (s["x"].float() @ (q * spread(s["w_scales"])).T).to(s["c"].dtype)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "quantize"):
        h, got = s["x"].double(), {}
        if case["op"] == "norm":
            if s["res"] is not None:
                h = h + s["res"].double()
                got["sum"] = h
            y = s["weight"].double() * h / torch.sqrt(h.pow(2).sum(1) / case["cols"] + 1e-6).unsqueeze(1)
        else:
            y = h
        if s["scales"] is None:
            return {**got, "y": y}
        got["scales"] = torch.maximum(y.abs().max(1).values / E4M3_MAX, torch.tensor(SCALE_MIN, dtype=torch.float64, device=y.device))
        return {**got, "y": y / got["scales"].unsqueeze(1)}  # the values that the 8 bits stand for, before their rounding
    if case["op"] == "e4m3":
        a = s["a"].double() * s["a_scales"].double().unsqueeze(1)
        return torch.matmul(a, (s["b"].double() * s["b_scales"].double().unsqueeze(1)).transpose(0, 1))
    k = torch.arange(case["K"], device="cuda")
    weight = torch.bitwise_and(s["w"][:, k // 2].int() >> (4 * (k % 2)).int(), 15).double()
    weight -= 8.0 if s["w_zeros"] is None else s["w_zeros"].double()[:, k // case["group"]]
    weight *= s["w_scales"].double()[:, k // case["group"]]
    return torch.matmul(s["x"].double(), weight.transpose(0, 1))


def work(case):
    if case["op"] in ("norm", "quantize"):
        n, size = case["rows"] * case["cols"], BYTES[case["type"]]
        out = case.get("out", "e4m3")
        moved = n * size + n * (1 if out == "e4m3" else size) + (4 * case["rows"] if out == "e4m3" else 0)
        if case["op"] == "norm":
            moved += size * case["cols"] + (2 * n * size if case["residual"] else 0)
        return {"bytes": moved, "flops": (6 if case["op"] == "norm" else 2) * n}
    M, N, K = case["M"], case["N"], case["K"]
    if case["op"] == "e4m3":
        return {"bytes": M * K + N * K + 4 * (M + N) + M * N * BYTES[case["out"]], "flops": 2 * M * N * K}
    groups = -(-K // case["group"])
    return {"bytes": N * -(-K // 2) + N * groups * (3 if case["zeros"] else 2) + 2 * M * (K + N), "flops": 2 * M * N * K}
