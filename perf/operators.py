"""Linear layers in 8-bit integers, as cases that can be timed and compared: what a decoder whose weights and activations are
int8 adds to the 16-bit path.

  norm   RMS norm of 16-bit rows (`add`: after the residual's addition, which the stream keeps), int8 out, a scale per token
  quant  rows to int8 with a scale per row: attention results, gated results, weights when they are loaded
  gemm   matrix product of int8 rows with int8 weights, a scale per token and per output channel; `bias`, and with `silu` the
         gated product silu(gate) * up of weight rows [gate | up]

A row's codes are q = round(127 t / max|t|), to the nearest, ties to even, with t the row (norm: the row times the norm's
weight); 1 / rms multiplies numerator and maximum alike and appears in the scale alone.  t is exact in 32 bits, and the quotient
is taken in 64, so that values next to a border fall on the right side: codes are whole numbers and compared as such.
"""
import math

import torch

own = False

DEV = "cuda"
EPS = 1e-5
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one user chatting: the norm before a layer's qkv projection, where launches and latency count
        dict(name="norm_1_token", kind="norm", rows=1, width=4096, dtype="f16", add=True),
        # the headline batch of the benchmark at the 70B width
        dict(name="norm_32_tokens", kind="norm", rows=32, width=8192, dtype="bf16", add=True),
        # a long prompt at the 70B width: bandwidth
        dict(name="norm_prompt_8192", kind="norm", rows=8192, width=8192, dtype="bf16", add=True),
        # a ragged batch of prompt portions, the first norm of a model (no residual yet), a width that fills no block evenly
        dict(name="norm_ragged_1003", kind="norm", rows=1003, width=2056, dtype="f16", add=False),
        # a decode batch's gated results before the down projection
        dict(name="quant_32_tokens", kind="quant", rows=32, width=14336, dtype="f16"),
        # a prompt's gated results; the size of a projection's weights, too
        dict(name="quant_prompt_8192", kind="quant", rows=8192, width=14336, dtype="bf16"),
        # the fused q | k | v projection of a single token: weights are read once, latency counts
        dict(name="gemm_1_token_qkv", kind="gemm", m=1, n=6144, k=4096, dtype="f16", bias=False, silu=False),
        # gate | up of the headline batch, activation included
        dict(name="gemm_32_tokens_gate_up", kind="gemm", m=32, n=28672, k=4096, dtype="f16", bias=False, silu=True),
        # logits of the headline batch
        dict(name="gemm_32_tokens_logits", kind="gemm", m=32, n=128256, k=4096, dtype="f32", bias=False, silu=False),
        # a short prompt beside decoded tokens, through the down projection
        dict(name="gemm_257_tokens_down", kind="gemm", m=257, n=4096, k=14336, dtype="bf16", bias=False, silu=False),
        # a ragged batch of prompt portions through a 70B-sized q | k | v with bias
        dict(name="gemm_1003_tokens_qkv", kind="gemm", m=1003, n=10240, k=8192, dtype="bf16", bias=True, silu=False),
        # a long prompt through gate | up: most of the time to the first token
        dict(name="gemm_prompt_8192_gate_up", kind="gemm", m=8192, n=28672, k=4096, dtype="bf16", bias=False, silu=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "quant", "gemm", "gemm"])
    if kind != "gemm":
        width = _log_int(rng, 64, 16384)
        if rng.random() < 0.7:
            width = max(64, width // 8 * 8)                 # the others are odd sizes
        rows = _log_int(rng, 1, min(16384, 8192 * 14336 // width))
        c = dict(kind=kind, rows=rows, width=width, dtype=rng.choice(["f16", "bf16"]))
        if kind == "norm":
            c["rows"] = min(rows, max(1, 8192 * 8192 // width))
            c["add"] = rng.random() < 0.6
        return c
    k = _log_int(rng, 64, 16384) // 16 * 16
    n = _log_int(rng, 64, 32768)
    if rng.random() < 0.7:
        n = max(64, n // 64 * 64)
    m = _log_int(rng, 1, 8192)
    m = max(1, min(m, 8192 * 28672 * 4096 // (n * k)))
    silu = rng.random() < 0.3
    return dict(kind="gemm", m=m, n=n // 2 * 2 if silu else n, k=k, dtype=rng.choice(["f16", "bf16"]) if silu else
                rng.choice(["f16", "bf16", "bf16", "f32"]), bias=rng.random() < 0.3, silu=silu)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _codes(g, rows, width):
    """Codes as a per-row quantiser leaves them for Gaussian rows: sigma about a quarter of the range."""
    out = torch.empty(rows, width, dtype=torch.int8, device=DEV)
    step = max(1, (1 << 26) // width)
    for r in range(0, rows, step):
        part = out[r:r + step]
        part.copy_(torch.randn(part.shape, generator=g, device=DEV).mul_(32).round_().clamp_(-127, 127))
    return out


def _rows(g, rows, width, dtype):
    """Activations: Gaussian, tokens of unlike size, a few channels far larger than the rest."""
    x = torch.randn(rows, width, generator=g, device=DEV)
    x *= 0.5 + torch.rand(rows, 1, generator=g, device=DEV)
    hot = torch.rand(width, generator=g, device=DEV) < 0.002
    return x.mul_(torch.where(hot, 12.0, 1.0)).to(dtype)


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    s = dict(case)
    if case["kind"] == "norm":
        s["x"] = _rows(g, case["rows"], case["width"], dt)
        s["w"] = (1.0 + 0.3 * torch.randn(case["width"], generator=g, device=DEV)).to(dt)
        if case["add"]:
            s["residual"] = _rows(g, case["rows"], case["width"], dt)
    elif case["kind"] == "quant":
        s["x"] = _rows(g, case["rows"], case["width"], dt)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["w"] = _codes(g, m, k), _codes(g, n, k)
        s["a_scales"] = (0.5 + torch.rand(m, generator=g, device=DEV)) / 32
        s["w_scales"] = (0.5 + torch.rand(n, generator=g, device=DEV)) / (32 * math.sqrt(k))
        s["bias_"] = torch.randn(n, generator=g, device=DEV).to(dt) if case["bias"] else None
    return s


def _to_codes(t):
    """Codes of fp32 rows, and the rows' maxima."""
    top = t.abs().amax(-1)
    q = torch.round(t.double() * 127.0 / top.double()[:, None])
    return torch.nan_to_num(q).to(torch.int8), top


def _plain(s):
    if s["kind"] == "norm":
        x = s["x"]
        if s["add"]:
            s["residual"].copy_(s["residual"].float() + x.float())
            x = s["residual"]
        f = x.float()
        q, top = _to_codes(f * s["w"].float())
        scales = top * torch.rsqrt((f * f).mean(-1) + EPS) / 127.0
        return (q, scales, s["residual"]) if s["add"] else (q, scales)
    if s["kind"] == "quant":
        q, top = _to_codes(s["x"].float())
        return q, top / 127.0
    y = (s["a"].float() @ s["w"].float().t()) * s["a_scales"][:, None] * s["w_scales"]
    if s["bias_"] is not None:
        y = y + s["bias_"].float()
    if s["silu"]:
        gate, up = y.chunk(2, -1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y.to(DTYPES[s["dtype"]])


def run(s):
    if own:
        from vllm_rs_b200 import ops
        if s["kind"] == "norm":
            if s["add"]:
                return (*ops.add_rmsnorm_i8(s["residual"], s["x"], s["w"], EPS), s["residual"])
            return ops.rmsnorm_i8(s["x"], s["w"], EPS)
        if s["kind"] == "quant":
            return ops.quant_rows_i8(s["x"])
        return ops.gemm_i8(s["a"], s["a_scales"], s["w"], s["w_scales"], bias=s["bias_"], dtype=DTYPES[s["dtype"]],
                           epilogue=ops.EPI_SILU_MUL if s["silu"] else ops.EPI_NONE)
    return _plain(s)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "gemm":
        out = torch.matmul(s["a"].to(torch.float64), s["w"].to(torch.float64).T)
        out *= torch.outer(s["a_scales"].to(torch.float64), s["w_scales"].to(torch.float64))
        if case["bias"]:
            out += s["bias_"].to(torch.float64)
        if case["silu"]:
            half = case["n"] // 2
            out = out[:, :half] * torch.sigmoid(out[:, :half]) * out[:, half:]
        return out
    r = s["x"].to(torch.float64)
    if case["kind"] == "norm":
        kept = r
        if case["add"]:
            # the stream is kept in 16 bits, and the norm is that of the stream as kept
            total = r + s["residual"].to(torch.float64)
            r = total.to(s["x"].dtype).to(torch.float64)
            kept = total
        normed = r / torch.sqrt(torch.mean(r ** 2, dim=1, keepdim=True) + EPS) * s["w"].to(torch.float64)
    else:
        normed = r
    scales = torch.max(torch.abs(normed), dim=1).values / 127
    codes = torch.where(scales[:, None] > 0, torch.round(normed / scales[:, None]), torch.zeros_like(normed)).to(torch.int8)
    return (codes, scales, kept) if case.get("add") else (codes, scales)


def work(case):
    if case["kind"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        elem = 4 if case["dtype"] == "f32" else 2
        cols = n // 2 if case["silu"] else n
        return {"bytes": (m + n) * k + 4 * (m + n) + elem * m * cols + (elem * n if case["bias"] else 0), "flops": 2 * m * n * k}
    rows, width = case["rows"], case["width"]
    per = 3 if case["kind"] == "quant" or not case["add"] else 7          # 16-bit reads, the stream's write, the codes
    return {"bytes": rows * (width * per + 4) + (2 * width if case["kind"] == "norm" else 0), "flops": 6 * rows * width}
