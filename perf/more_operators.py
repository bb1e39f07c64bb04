"""The 8-bit linear layers of a language model that this package is measured by:
the rows that enter them (RMS norm with the residual's addition, SwiGLU's gated
product, and rows as they are or times a gate, each rounded to 8 bits with a scale
for each block of 128 columns) and their product with weights in 8 bits with a
scale for each block of 128 by 128.

A case is a dict of plain values; `kind` names the operator.  `own` False: the
operator's plain form in torch, in 32 bits; `own` True: this package's call.

Formulas
  8-bit block   128 numbers x of a row (a weight: 128 rows of 128) become e4m3
                numbers c with one scale s = 2^e, the smallest power of two with
                max|x| <= 448 s (1 for a block of zeros): c is x / s rounded.  Rows
                are filled up to whole blocks with zeros; scales are kept as e8m0
                bytes, 2^(byte - 127), a row of them filled up to whole words with 1
  norm8         t = x + r in x's type where there is a residual r, else x;
                t rsqrt(mean t^2 + eps) (1 + w) in 8 bits
  silu8         a c / (1 + e^-c) in 8 bits
  rows8         x, or x gate, in 8 bits
  linear8       y[m, n] = sum_b s_x[m, b] s_w[n / 128, b] sum_k c_x c_w + bias[n]
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
FP8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
EPS = 1e-6


def listed():
    return [
        # a decode step of a small batch: the residual's addition, the next norm and
        # its rows for the layer behind it; launches count
        dict(name="norm8_step", kind="norm8", rows=4, dim=1024, residual=True, dtype="bfloat16"),
        # the same over a batch of prompts
        dict(name="norm8_prompt", kind="norm8", rows=32768, dim=1024, residual=True, dtype="bfloat16"),
        # SwiGLU's product before its last layer, one step and a batch of prompts
        dict(name="silu8_step", kind="silu8", rows=4, dim=4096),
        dict(name="silu8_prompt", kind="silu8", rows=32768, dim=4096),
        # attention's output times its gate before the output projection
        dict(name="rows8_step", kind="rows8", rows=4, dim=1024, gated=True, dtype="bfloat16"),
        # an SSM block's output before its projection: ragged prompts, columns off the blocks
        dict(name="rows8_prompt", kind="rows8", rows=8191, dim=2056, gated=False, dtype="bfloat16"),
        # a projection of one token of a small model
        dict(name="linear8_one", kind="linear8", rows=1, inner=1024, outer=1024, bias=True, given="rows"),
        # a decode step's widest layer (an SSM block's input projection)
        dict(name="linear8_step", kind="linear8", rows=4, inner=1024, outer=4384, bias=True, given="rows"),
        # a vocabulary projection for a serving batch
        dict(name="linear8_head", kind="linear8", rows=32, inner=4096, outer=32000, bias=False,
             given="rows"),
        # a short prompt, or a step's rows of many requests, still in bfloat16; odd sizes
        dict(name="linear8_chunk", kind="linear8", rows=500, inner=2050, outer=4383, bias=True,
             given="bfloat16"),
        # a batch of prompts through SwiGLU's first layer
        dict(name="linear8_prompt", kind="linear8", rows=32768, inner=1024, outer=4096, bias=True,
             given="rows"),
        # a large product
        dict(name="linear8_large", kind="linear8", rows=8192, inner=8192, outer=8192, bias=False,
             given="rows"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed kinds, no larger than the largest listed."""
    kind = rng.choice(["norm8", "norm8", "silu8", "rows8", "linear8", "linear8", "linear8", "linear8"])
    odd = rng.random() < 0.3
    if kind == "linear8":
        size = (lambda lo, hi: _log_int(rng, lo, hi)) if odd else (  # noqa: E731
            lambda lo, hi: 64 * max(1, _log_int(rng, lo, hi) // 64))
        inner, outer = size(100, 8192), size(50, 32000)
        most = min(32768, (1 << 39) // (inner * outer), (1 << 28) // outer)
        rows = _log_int(rng, 1, 64) if rng.random() < 0.4 else _log_int(rng, 1, max(2, most))
        return dict(kind=kind, rows=rows, inner=inner, outer=outer, bias=rng.random() < 0.5,
                    given=rng.choice(["rows", "rows", "bfloat16"]))
    dim = _log_int(rng, 64, 16384)
    dim = dim if odd else 64 * max(1, dim // 64)
    rows = _log_int(rng, 1, min(65536, (1 << 27) // dim))
    if kind == "silu8":
        return dict(kind=kind, rows=rows, dim=dim)
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if kind == "norm8":
        return dict(kind=kind, rows=rows, dim=dim, residual=rng.random() < 0.6, dtype=dtype)
    return dict(kind=kind, rows=rows, dim=dim, gated=rng.random() < 0.5, dtype=dtype)


# --- inputs -------------------------------------------------------------------
def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _stream(gen, rows, dim, dtype):
    """Rows of a residual stream: columns of unlike size, a few of them large."""
    col = torch.exp(0.5 * _normal(gen, dim)) * (1 + 20 * (torch.rand(dim, generator=gen, device="cuda") < 0.01))
    return _normal(gen, rows, dim).mul_(col).to(dtype)


def _blocks(n):
    return (n + 127) // 128


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, M, bf16 = case["kind"], case["rows"], torch.bfloat16
    s = dict(case=case)
    if kind == "linear8":
        K, N = case["inner"], case["outer"]
        x = _stream(gen, M, K, bf16)
        if case["given"] == "rows":
            s["codes"], s["scales"] = _rows(x)
        else:
            s["x"] = x
        w = _normal(gen, N, K) / K ** 0.5
        s["packed"], s["w_scales"] = _weight(w)
        s["bias"] = _normal(gen, N, dtype=bf16) if case["bias"] else None
        return s
    D = case["dim"]
    if kind == "silu8":
        s["a"], s["c"] = _normal(gen, M, D, dtype=bf16), (2 * _normal(gen, M, D)).to(bf16)
        return s
    dtype = DTYPES[case["dtype"]]
    s["x"] = _stream(gen, M, D, dtype)
    if kind == "norm8":
        s["weight"] = 0.2 * _normal(gen, D)
        s["residual"] = _stream(gen, M, D, dtype) if case["residual"] else None
    else:
        s["gate"] = torch.sigmoid(_normal(gen, M, D) + 1.0).to(dtype) if case["gated"] else None
    return s


# --- plain forms --------------------------------------------------------------
def _scale_of(top):
    """The smallest power of two s with top <= 448 s, as a float and as its e8m0 byte."""
    part, power = torch.frexp(top)                      # top = part 2^power, part in [0.5, 1)
    power = (power - 9 + (part > 0.875)).clamp(min=-126)
    power = torch.where(top > 0, power, 0)
    return torch.ldexp(torch.ones_like(top), power), (power + 127).to(torch.uint8)


def _words(byte):
    """Scales' bytes (n, blocks) filled up to whole words of four with 127, 2^0."""
    return torch.nn.functional.pad(byte, (0, -byte.shape[1] % 4), value=127).view(E8)


def _rows(x):
    """x (rows, dim) -> codes (rows, 128 blocks) e4m3, scales (rows, words of four) e8m0."""
    M, D = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -D % 128)).view(M, -1, 128)
    s, byte = _scale_of(x.abs().amax(2))
    return (x / s[..., None]).to(FP8).view(M, -1), _words(byte)


def _weight(w):
    """w (N, K) -> packed (N / 16, K / 128, 8, 16, 16) bytes and scales (N / 128, words
    of four): tiles of 16 rows and 128 columns; in a tile, 16 columns of its 16 rows
    after each other."""
    N, K = w.shape
    nb, kb = _blocks(N), _blocks(K)
    w = torch.nn.functional.pad(w, (0, -K % 128, 0, -N % 128)).view(nb, 128, kb, 128)
    s, byte = _scale_of(w.abs().amax((1, 3)))
    code = (w / s[:, None, :, None]).to(FP8).view(torch.uint8).view(nb * 8, 16, kb, 8, 16)
    return code.permute(0, 2, 3, 1, 4)[:(N + 15) // 16].contiguous(), _words(byte)


def _norm8_plain(s):
    t = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    f = t.float()
    f = f * torch.rsqrt(f.pow(2).mean(1, keepdim=True) + EPS) * (1.0 + s["weight"])
    codes, scales = _rows(f)
    out = {"codes": codes, "scales": scales}
    return out if s["residual"] is None else {**out, "sum": t}


def _linear8_plain(s):
    c = s["case"]
    N, K = c["outer"], c["inner"]
    codes, scales = (s["codes"], s["scales"]) if c["given"] == "rows" else _rows(s["x"])
    kb = _blocks(K)
    x = codes.float().view(-1, kb, 128) * scales.float()[:, :kb, None]
    w = s["packed"].view(FP8).float().permute(0, 3, 1, 2, 4)                   # tile, row, block, piece, column
    w = w.reshape(-1, kb, 128) * s["w_scales"].float()[:, :kb, None].repeat_interleave(128, 0)[:w.shape[0] * 16]
    y = x.flatten(1) @ w.flatten(1)[:N].t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(torch.bfloat16)


# --- one pass -----------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        if kind == "linear8":
            return _linear8_plain(s)
        if kind == "norm8":
            return _norm8_plain(s)
        if kind == "silu8":
            a, g = s["a"].float(), s["c"].float()
            codes, scales = _rows(a * (g / (1.0 + torch.exp(-g))))
        else:
            codes, scales = _rows(s["x"].float() if s["gate"] is None else s["x"].float() * s["gate"].float())
        return {"codes": codes, "scales": scales}
    ops = _ops()
    if kind == "linear8":
        x = ops.Fp8Rows(s["codes"], s["scales"]) if c["given"] == "rows" else s["x"]
        return ops.fp8_linear(x, s["packed"], s["w_scales"], s["bias"], out_features=c["outer"])
    if kind == "norm8":
        if s["residual"] is None:
            r = ops.rms_norm_fp8(s["x"], s["weight"], EPS)
            return {"codes": r.codes, "scales": r.scales}
        t, r = ops.rms_norm_fp8(s["x"], s["weight"], EPS, residual=s["residual"])
        return {"codes": r.codes, "scales": r.scales, "sum": t}
    r = ops.silu_mul_fp8(s["a"], s["c"]) if kind == "silu8" else ops.quantize_rows_fp8(s["x"], s["gate"])
    return {"codes": r.codes, "scales": r.scales}


def _ops():
    package = os.path.join(ROOT, "selective-attention_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    import selective_attention.ops as ops
    return ops


# --- what a pass cannot do without --------------------------------------------
def work(case):
    kind, M = case["kind"], case["rows"]
    if kind == "linear8":
        K, N = case["inner"], case["outer"]
        x = M * (K + _blocks(K)) if case["given"] == "rows" else 2 * M * K
        return {"bytes": x + N * K + _blocks(N) * _blocks(K) + 2 * N * case["bias"] + 2 * M * N,
                "flops": 2 * M * K * N}
    D = case["dim"]
    out = M * (D + _blocks(D))
    if kind == "silu8":
        return {"bytes": out + 4 * M * D, "flops": 8 * M * D}
    size = 4 if case["dtype"] == "float32" else 2
    if kind == "norm8":
        return {"bytes": out + size * M * D * (3 if case["residual"] else 1) + 4 * D, "flops": 8 * M * D}
    return {"bytes": out + size * M * D * (2 if case["gated"] else 1), "flops": 4 * M * D}


# --- the definitions in 64 bits -----------------------------------------------
def _e4m3(y):
    """The nearest e4m3 number (ties to even) of |y| <= 448, in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(y / step) * step


def _rows64(x):
    """Codes and scales of x (rows, dim) in 64 bits, a block of columns after another."""
    M, D = x.shape
    kb = _blocks(D)
    codes = torch.zeros(M, 128 * kb, dtype=torch.float64, device=x.device)
    scales = torch.ones(M, 4 * ((kb + 3) // 4), dtype=torch.float64, device=x.device)
    for b in range(kb):
        y = x[:, 128 * b:128 * (b + 1)]
        top = y.abs().amax(1)
        e = torch.ceil(torch.log2(top / 448.0)).clamp(min=-126.0)
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)         # (a logarithm rounded)
        e = torch.where((top <= 224.0 * torch.exp2(e)) & (e > -126), e - 1, e)
        s = torch.where(top > 0, torch.exp2(e), 1.0)
        scales[:, b] = s
        codes[:, 128 * b:128 * b + y.shape[1]] = _e4m3(y / s[:, None])
    return codes, scales


def _exact_rows(case, s):
    if case["kind"] == "silu8":
        c = s["c"].double()
        return _rows64(s["a"].double() * c * torch.sigmoid(c))
    x = s["x"].double()
    if case["kind"] == "rows8":
        return _rows64(x if s["gate"] is None else x * s["gate"].double())
    if s["residual"] is not None:
        x = (s["x"] + s["residual"]).double()
    return _rows64(x / torch.sqrt((x * x).sum(1, keepdim=True) / case["dim"] + EPS) * (1.0 + s["weight"].double()))


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] != "linear8":
        codes, scales = _exact_rows(case, s)
        out = {"codes": codes, "scales": scales}
        if case["kind"] == "norm8" and s["residual"] is not None:
            out["sum"] = (s["x"] + s["residual"]).double()
        return out
    N, K = case["outer"], case["inner"]
    kb = _blocks(K)
    if case["given"] == "rows":
        codes, scales = s["codes"].double(), s["scales"].double()
    else:
        codes, scales = _rows64(s["x"].double())
    y = torch.zeros(case["rows"], N, dtype=torch.float64, device="cuda")
    for b in range(kb):
        tile = s["packed"][:, b].view(FP8).double()                            # (tile, piece, row, column)
        w = tile.transpose(1, 2).reshape(-1, 128)[:N]
        of = s["w_scales"].double()[:, b][torch.arange(N, device="cuda") // 128]
        x = codes[:, 128 * b:128 * (b + 1)] * scales[:, b, None]
        y += torch.matmul(x, (w * of[:, None]).t().contiguous())
    return y if s["bias"] is None else y + s["bias"].double()
