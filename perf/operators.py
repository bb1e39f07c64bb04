"""The serving and scoring operators of a language model that this package is
measured by: paged decode attention over a cache held in 8 bits, the writes that
fill that cache, linear layers with 4-bit weights for few rows, and the log
probabilities of given tokens with their entropy, alternatives and gradient.

A case is a dict of plain values; `kind` names the operator.  `own` False: the
operator's plain form in torch, in 32 bits; `own` True: this package's call.

Formulas
  8-bit cache   a block is one page of tokens of one kv head.  Its keys (and its
                values) are e4m3 numbers c with one scale s = 2^e for the block,
                the smallest power of two with max|x| <= 448 s; x stands as c s.
                Tokens whose gate is -inf are left out (stored as 0), except the
                block's last one.  A row's open block (the tokens behind its last
                full page) is kept in bfloat16 until it is full.
  attention     o = softmax_j(scale q.k_j + [j not the newest] gate_j) v_j
  4-bit layer   y = x W^T + bias, W[n, k] = s[n, k // group] (c[n, k] - z), z = 8
                or z[n, k // group]
  log probs     l_t = x_t - log sum_j e^x_j,  H = -sum_j p_j log p_j, and the
                largest x_j with their l_j, ties to the lowest j
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
FP8 = torch.float8_e4m3fn
PENALTY, GATE_STD = 2.0, 1.0
IGNORE = -100


def listed():
    return [
        # one request's next token in one layer of a small model: launches count
        dict(name="attend8_one", kind="attend8", batch=1, heads=16, kv_heads=16, headdim=64,
             page=64, shortest=200, longest=200, gated=True, pack=1),
        # SelectiveMHA's gated decode step, a small batch behind long prompts
        dict(name="attend8_gated", kind="attend8", batch=4, heads=16, kv_heads=16, headdim=64,
             page=64, shortest=5000, longest=8193, gated=True, pack=2),
        # a serving batch with grouped heads and long contexts
        dict(name="attend8_long", kind="attend8", batch=64, heads=32, kv_heads=8, headdim=128,
             page=64, shortest=1024, longest=32768, gated=False, pack=3),
        # one decode step's tokens into the cache of a serving batch
        dict(name="append8", kind="append8", batch=64, kv_heads=8, headdim=128, page=64,
             shortest=30, longest=2048, gated=False, pack=4),
        # a prompt's keys and values into the cache after prefill, ragged rows
        dict(name="build8", kind="build8", batch=4, kv_heads=16, headdim=64, page=64, seqlen=8192,
             gated=True, pack=5),
        # a projection of one token of a small model
        dict(name="int4_one", kind="int4", rows=1, inner=1024, outer=1024, group=128, zeros=False,
             bias=True),
        # a decode step's widest layer (an SSM block's input projection) for a small
        # batch, weights with zero points
        dict(name="int4_step", kind="int4", rows=4, inner=1024, outer=4384, group=64, zeros=True,
             bias=True),
        # a vocabulary projection for a serving batch
        dict(name="int4_head", kind="int4", rows=32, inner=4096, outer=32000, group=128,
             zeros=False, bias=False),
        # what a decode step answers with: the chosen tokens and their alternatives
        dict(name="logprobs_step", kind="logprobs", rows=4, vocab=32000, top=8, dtype="bfloat16",
             train=False),
        # scoring a batch of prompts
        dict(name="logprobs_score", kind="logprobs", rows=8192, vocab=32000, top=20,
             dtype="bfloat16", train=False),
        # a training step's loss with an entropy term, and the logits' gradient
        dict(name="logprobs_train", kind="logprobs", rows=8192, vocab=32000, top=0,
             dtype="bfloat16", train=True),
        # the same in float32 with an odd vocabulary (rows off a 16-byte boundary)
        dict(name="logprobs_train_fp32", kind="logprobs", rows=1500, vocab=32003, top=0,
             dtype="float32", train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed kinds, no larger than the largest listed."""
    kind = rng.choice(["attend8", "attend8", "attend8", "append8", "build8", "int4", "int4", "int4",
                       "logprobs", "logprobs", "logprobs"])
    pack = rng.randrange(1, 1 << 20)
    if kind in ("attend8", "append8"):
        kv, dim = rng.choice([4, 8, 16]), rng.choice([64, 128])
        batch = _log_int(rng, 1, 64)
        most = (1 << 30) // (batch * kv * dim * (1 if kind == "attend8" else 16))
        longest = _log_int(rng, 1, max(2, min(32768, most)))
        c = dict(kind=kind, batch=batch, kv_heads=kv, headdim=dim, page=rng.choice([64, 64, 128]),
                 shortest=rng.randrange(1, longest + 1), longest=longest,
                 gated=rng.random() < 0.5, pack=pack)
        if kind == "attend8":
            c["heads"] = kv * rng.choice([1, 1, 2, 4, 8, 16])
        return c
    if kind == "build8":
        return dict(kind=kind, batch=rng.choice([1, 2, 3, 4]), kv_heads=rng.choice([4, 8, 16]),
                    headdim=rng.choice([64, 128]), page=rng.choice([64, 64, 128]),
                    seqlen=_log_int(rng, 1, 4096), gated=rng.random() < 0.5, pack=pack)
    if kind == "int4":
        return dict(kind=kind, rows=_log_int(rng, 1, 64), inner=_log_int(rng, 100, 4096),
                    outer=_log_int(rng, 50, 32000), group=rng.choice([32, 64, 128, 128]),
                    zeros=rng.random() < 0.5, bias=rng.random() < 0.5)
    vocab = _log_int(rng, 100, 131072)
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    train = rng.random() < 0.5
    return dict(kind=kind, rows=_log_int(rng, 1, min(8192, (1 << 27) // vocab)), vocab=vocab,
                top=0 if train else rng.choice([0, 1, 5, 20, 32]), dtype=dtype, train=train)


# --- inputs -------------------------------------------------------------------
def _lengths(case):
    """The rows' token counts, from the case itself."""
    r = random.Random(case["pack"])
    if case["kind"] == "build8":
        hi = case["seqlen"]
        return [hi] + [r.randint(max(1, hi // 2), hi) for _ in range(case["batch"] - 1)]
    lo, hi = case["shortest"], case["longest"]
    return [hi] + [r.randint(lo, hi) for _ in range(case["batch"] - 1)]


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def _gates(gen, *shape):
    """log(gate) * std * penalty of gates sigmoid(N(2, 1)); about a tenth of them
    stand below the threshold and are dropped."""
    g = torch.sigmoid(2.0 + _normal(gen, *shape))
    return torch.where(g < 0.67, -math.inf, torch.log(g) * GATE_STD * PENALTY)


def _pool(case, lens, gen, more):
    """Page tables over a shuffled pool, `more` tokens of room behind each row."""
    ps, n = case["page"], [(x + more + case["page"] - 1) // case["page"] for x in lens]
    total, width = sum(n), max(n)
    perm = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    count = torch.tensor(n, device="cuda")
    col = torch.arange(width, device="cuda")[None, :]
    first = (torch.cumsum(count, 0) - count)[:, None]
    inside = col < count[:, None]
    table = torch.where(inside, perm[(first + col).clamp(max=total - 1)], -1)
    return total, table.to(torch.int32).contiguous(), torch.tensor(lens, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind = case["kind"]
    if kind in ("attend8", "append8", "build8"):
        lens = _lengths(case)
        b, H, D, ps = case["batch"], case["kv_heads"], case["headdim"], case["page"]
        pages, table, seq_lens = _pool(case, lens, gen, 1 if kind == "append8" else 0)
        bf16 = torch.bfloat16
        s = dict(case=case, table=table, lens=seq_lens)
        if kind == "build8":
            L = case["seqlen"]
            s["k"] = _normal(gen, b, L, H, D, dtype=bf16).transpose(1, 2)
            s["v"] = _normal(gen, b, L, H, D, dtype=bf16).transpose(1, 2)
            s["log_gate"] = _gates(gen, b, H, L) if case["gated"] else None
            s["k_tail"] = torch.zeros(b, H, ps, D, dtype=bf16, device="cuda")
            s["v_tail"] = torch.zeros(b, H, D, ps, dtype=bf16, device="cuda")
            s["k_pages"] = torch.zeros(pages, H, ps, D, device="cuda").to(FP8)
            s["v_pages"] = torch.zeros(pages, H, D, ps, device="cuda").to(FP8)
            s["k_scale"] = torch.zeros(pages, H, device="cuda")
            s["v_scale"] = torch.zeros(pages, H, device="cuda")
            s["gates"] = torch.full((pages, H, ps), -math.inf, device="cuda") if case["gated"] else None
            return s
        s["gates"] = _gates(gen, pages, H, ps) if case["gated"] else None
        s["k_pages"], s["k_scale"] = _quantised(_normal(gen, pages, H, ps, D, dtype=bf16), s["gates"])
        v, s["v_scale"] = _quantised(_normal(gen, pages, H, ps, D, dtype=bf16), s["gates"])
        s["v_pages"] = v.view(torch.uint8).transpose(2, 3).contiguous().view(FP8)
        s["k_tail"] = _normal(gen, b, H, ps, D, dtype=bf16)
        s["v_tail"] = _normal(gen, b, H, D, ps, dtype=bf16)
        if kind == "attend8":
            s["q"] = _normal(gen, b, case["heads"], D, dtype=bf16)
        else:
            s["k"] = _normal(gen, b, H, D, dtype=bf16)
            s["v"] = _normal(gen, b, H, D, dtype=bf16)
            s["log_gate"] = _gates(gen, b, H) if case["gated"] else None
        return s
    if kind == "int4":
        M, K, N, G = case["rows"], case["inner"], case["outer"], case["group"]
        nt, kb = (N + 15) // 16, (K + 127) // 128
        s = dict(case=case, x=_normal(gen, M, K, dtype=torch.bfloat16))
        # packed codes and scales in the order the layer keeps them (see _codes)
        s["packed"] = torch.randint(0, 256, (nt, kb, 64, 16), generator=gen, device="cuda",
                                    dtype=torch.uint8)
        step = (0.5 + torch.rand(nt, kb * 128 // G, 16, generator=gen, device="cuda")) / (4.6 * K ** 0.5)
        s["scales"] = step.to(torch.bfloat16)
        s["zeros"] = (torch.randint(4, 12, step.shape, generator=gen, device="cuda").to(torch.bfloat16)
                      if case["zeros"] else None)
        s["bias"] = _normal(gen, N, dtype=torch.bfloat16) if case["bias"] else None
        return s
    rows, V = case["rows"], case["vocab"]
    x = _normal(gen, rows, V).mul_(2.0)
    targets = torch.randint(0, V, (rows,), generator=gen, device="cuda")
    # the model prefers the target in half of the rows; one token in 50 is ruled out
    x[torch.arange(rows, device="cuda"), targets] += 8.0 * (torch.rand(rows, generator=gen, device="cuda") < 0.5)
    banned = torch.rand(V, generator=gen, device="cuda") < 0.02
    x.masked_fill_(banned[None, :], -math.inf)
    targets = torch.where(banned[targets], IGNORE, targets)
    s = dict(case=case, logits=x.to(DTYPES[case["dtype"]]), targets=targets)
    if case["train"]:
        s["logits"].requires_grad_(True)
        s["g_logprob"] = -(0.5 + torch.rand(rows, generator=gen, device="cuda")) / rows
        s["g_entropy"] = 0.1 * _normal(gen, rows) / rows
    return s


# --- plain forms --------------------------------------------------------------
def _quantised(x, gates):
    """x (..., tokens, dim), gates (..., tokens) or None -> (e4m3 codes, scale (...))."""
    x = x.float()
    if gates is not None:
        keep = gates > -math.inf
        keep[..., -1] = True
        x = torch.where(keep[..., None], x, 0.0)
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax((-2, -1))
    part, power = torch.frexp(top)                      # top = part 2^power, part in [0.5, 1)
    power = (power - 9 + (part > 0.875)).clamp(min=-126)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), power), 1.0)
    return (x / scale[..., None, None]).to(FP8), scale


def _attend8_plain(s):
    c = s["case"]
    b, Hq, Hkv, D, ps = c["batch"], c["heads"], c["kv_heads"], c["headdim"], c["page"]
    table, lens = s["table"].long().clamp(min=0), s["lens"].long()
    width = table.shape[1]
    k = s["k_pages"][table].float() * s["k_scale"][table][..., None, None]     # (b, width, Hkv, ps, D)
    v = s["v_pages"][table].float() * s["v_scale"][table][..., None, None]     # (b, width, Hkv, D, ps)
    open_page = (torch.arange(width, device="cuda")[None, :] == (lens // ps)[:, None])[:, :, None, None, None]
    k = torch.where(open_page, s["k_tail"].float()[:, None], k)
    v = torch.where(open_page, s["v_tail"].float()[:, None], v)
    q = s["q"].float().view(b, 1, Hkv, Hq // Hkv, D)
    score = (q @ k.transpose(-1, -2)) * D ** -0.5                              # (b, width, Hkv, grp, ps)
    pos = (torch.arange(width, device="cuda")[:, None] * ps + torch.arange(ps, device="cuda"))[None]
    if s["gates"] is not None:
        newest = pos == (lens - 1)[:, None, None]
        score = score + torch.where(newest[:, :, None], 0.0, s["gates"][table])[:, :, :, None]
    score = torch.where((pos < lens[:, None, None])[:, :, None, None], score, -math.inf)
    p = torch.exp(score - score.amax((1, 4), keepdim=True))
    p = p / p.sum((1, 4), keepdim=True)
    o = (p @ v.transpose(-1, -2)).sum(1)                                       # (b, Hkv, grp, D)
    return o.reshape(b, Hq, D).to(torch.bfloat16)


def _cache_of(s, lens):
    names = ("k_pages", "v_pages", "k_scale", "v_scale", "k_tail", "v_tail", "gates")
    return {**{n: s[n] for n in names}, "lens": lens}


def _append8_plain(s, lens):
    ps = s["case"]["page"]
    row = torch.arange(lens.shape[0], device="cuda")
    t = lens.long()
    slot, page = t % ps, s["table"].long()[row, t // ps]
    s["k_tail"][row, :, slot] = s["k"]
    s["v_tail"][row, :, :, slot] = s["v"]
    if s["gates"] is not None:
        s["gates"][page, :, slot] = s["log_gate"]
    full = slot == ps - 1
    page, gates = page[full], None
    if s["gates"] is not None:
        gates = s["gates"][page]
    code, s["k_scale"][page] = _quantised(s["k_tail"][full], gates)
    s["k_pages"].view(torch.uint8)[page] = code.view(torch.uint8)
    code, s["v_scale"][page] = _quantised(s["v_tail"][full].transpose(-1, -2), gates)
    s["v_pages"].view(torch.uint8)[page] = code.view(torch.uint8).transpose(-1, -2)
    lens += 1
    return _cache_of(s, lens)


def _build8_plain(s):
    c = s["case"]
    b, H, D, ps, L = c["batch"], c["kv_heads"], c["headdim"], c["page"], c["seqlen"]
    lens, width = s["lens"].long(), s["table"].shape[1]
    pad = width * ps - L
    rows = lambda x, fill: torch.nn.functional.pad(x, (0, 0, 0, pad), value=fill).view(  # noqa: E731
        b, H, width, ps, -1).transpose(1, 2)                                   # (b, width, H, ps, .)
    inside = (torch.arange(width * ps, device="cuda")[None, :] < lens[:, None]).view(b, width, 1, ps, 1)
    k = torch.where(inside, rows(s["k"], 0.0), 0.0)
    v = torch.where(inside, rows(s["v"], 0.0), 0.0)
    col = torch.arange(width, device="cuda")[None, :]
    full, tail = col < (lens // ps)[:, None], col == (lens // ps)[:, None]
    gates = None
    if s["gates"] is not None:
        gates = torch.where(inside, rows(s["log_gate"][..., None], 0.0), -math.inf)[..., 0]
        used = full | (tail & (lens % ps > 0)[:, None])
        s["gates"][s["table"].long()[used]] = gates[used]
        gates = gates[full]
    page = s["table"].long()[full]
    code, s["k_scale"][page] = _quantised(k[full], gates)
    s["k_pages"].view(torch.uint8)[page] = code.view(torch.uint8)
    code, s["v_scale"][page] = _quantised(v[full], gates)
    s["v_pages"].view(torch.uint8)[page] = code.view(torch.uint8).transpose(-1, -2)
    has = tail.any(1) & (lens % ps > 0)
    s["k_tail"][has] = k[tail & has[:, None]]
    s["v_tail"][has] = v[tail & has[:, None]].transpose(-1, -2)
    return _cache_of(s, s["lens"])


def _codes(packed, N, K):
    """The codes (N, K) of a packed weight.  packed (N / 16, K / 128, 64, 16) bytes:
    byte 4 j + i of lane 16 g + c holds, in its low and high half, the codes of row
    c, columns 32 j + 8 g + 2 i and + 1, of a tile of 16 rows and 128 columns."""
    nt, kb = packed.shape[:2]
    p = packed.view(nt, kb, 4, 16, 4, 4)                                       # g, c, j, i
    both = torch.stack((p & 15, p >> 4), -1)                                   # g, c, j, i, half
    w = both.permute(0, 3, 1, 4, 2, 5, 6).reshape(nt * 16, kb * 128)           # c, kb, j, g, i, half
    return w[:N, :K]


def _int4_plain(s):
    c = s["case"]
    N, K, G = c["outer"], c["inner"], c["group"]
    code = _codes(s["packed"], N, K).float()
    each = lambda t: t.float().transpose(1, 2).flatten(0, 1).repeat_interleave(G, 1)[:N, :K]  # noqa: E731
    w = each(s["scales"]) * (code - (8.0 if s["zeros"] is None else each(s["zeros"])))
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(torch.bfloat16)


def _logprobs_plain(s):
    c = s["case"]
    x = s["logits"].detach().float()
    asked = s["targets"] != IGNORE
    top = x.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    lp = torch.where(asked, x.gather(1, s["targets"].clamp(min=0)[:, None])[:, 0] - lse[:, 0], 0.0)
    p, logp = torch.exp(x - lse), x - lse
    plogp = torch.where(p > 0, p * logp, 0.0)
    H = -plogp.sum(1)
    if not c["train"]:
        if not c["top"]:
            return {"logprob": lp, "entropy": H}
        value, index = torch.sort(x, dim=1, descending=True, stable=True)
        index = index[:, :c["top"]].contiguous()
        return {"logprob": lp, "entropy": H, "top_ids": index,
                "top_logprobs": value[:, :c["top"]] - lse}
    ga = torch.where(asked, s["g_logprob"], 0.0)[:, None]
    d = -p * ga - s["g_entropy"][:, None] * (plogp + p * H[:, None])
    d.scatter_add_(1, s["targets"].clamp(min=0)[:, None], ga)
    return {"logprob": lp, "entropy": H, "dlogits": d.to(s["logits"].dtype)}


# --- one pass -----------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if not own:
        if kind == "attend8":
            return _attend8_plain(s)
        if kind == "append8":
            return _append8_plain(s, s["lens"].clone())
        if kind == "build8":
            return _build8_plain(s)
        return _int4_plain(s) if kind == "int4" else _logprobs_plain(s)
    ops = _ops()
    if kind == "attend8":
        return ops.paged_decode_attn_fp8(s["q"], s["k_pages"], s["v_pages"], s["k_scale"],
                                         s["v_scale"], s["k_tail"], s["v_tail"], s["table"],
                                         s["lens"], key_bias=s["gates"])
    if kind in ("append8", "build8"):
        lens = s["lens"].clone() if kind == "append8" else s["lens"]
        call = ops.paged_kv_append_fp8 if kind == "append8" else ops.paged_kv_build_fp8
        call(s["k"], s["v"], s["log_gate"], s["table"], lens, s["k_pages"], s["v_pages"],
             s["k_scale"], s["v_scale"], s["k_tail"], s["v_tail"], s["gates"])
        return _cache_of(s, lens)
    if kind == "int4":
        return ops.int4_linear(s["x"], s["packed"], s["scales"], s["zeros"], s["bias"],
                               out_features=c["outer"])
    out = ops.token_logprobs(s["logits"], s["targets"], top=c["top"], ignore_index=IGNORE)
    if c["train"]:
        (d,) = torch.autograd.grad((out.logprob, out.entropy), (s["logits"],),
                                   (s["g_logprob"], s["g_entropy"]))
        return {"logprob": out.logprob, "entropy": out.entropy, "dlogits": d}
    if not c["top"]:
        return {"logprob": out.logprob, "entropy": out.entropy}
    return {"logprob": out.logprob, "entropy": out.entropy, "top_ids": out.top_ids,
            "top_logprobs": out.top_logprobs}


def _ops():
    package = os.path.join(ROOT, "selective-attention_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    import selective_attention.ops as ops
    return ops


# --- what a pass cannot do without --------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "attend8":
        H, Hq, D, ps = case["kv_heads"], case["heads"], case["headdim"], case["page"]
        lens = _lengths(case)
        closed, tail = sum(n // ps * ps for n in lens), sum(n % ps for n in lens)
        blocks = sum(n // ps for n in lens)
        size = H * D * 2 * (closed + 2 * tail) + 8 * H * blocks + 4 * case["batch"] * Hq * D
        return {"bytes": size + 4 * (closed + tail) * H * case["gated"] + 4 * blocks,
                "flops": 4 * Hq * D * (closed + tail)}
    if kind == "append8":
        H, D, ps = case["kv_heads"], case["headdim"], case["page"]
        full = sum(n % ps == ps - 1 for n in _lengths(case))
        size = case["batch"] * H * (8 * D + 8 * case["gated"]) + full * H * ps * (6 * D + 4 * case["gated"])
        return {"bytes": size + 8 * case["batch"], "flops": 4 * full * H * ps * D}
    if kind == "build8":
        H, D, ps = case["kv_heads"], case["headdim"], case["page"]
        lens = _lengths(case)
        closed, tail = sum(n // ps * ps for n in lens), sum(n % ps for n in lens)
        return {"bytes": H * (D * (6 * closed + 8 * tail) + 8 * (closed + tail) * case["gated"]),
                "flops": 4 * H * D * closed}
    if kind == "int4":
        M, K, N, G = case["rows"], case["inner"], case["outer"], case["group"]
        groups = (K + G - 1) // G
        return {"bytes": N * K / 2 + N * groups * (4 if case["zeros"] else 2) + 2 * M * (K + N),
                "flops": 2 * M * K * N}
    cells = case["rows"] * case["vocab"]
    size = 4 if case["dtype"] == "float32" else 2
    # a training step reads the logits for the loss and again for the gradient
    return {"bytes": cells * size * (3 if case["train"] else 1) + case["rows"] * (16 + 12 * case["top"]),
            "flops": cells * (10 if case["train"] else 5)}


# --- the definitions in 64 bits -----------------------------------------------
def _e4m3(y):
    """The nearest e4m3 number (ties to even) of |y| <= 448, in 64 bits."""
    a = y.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3.0)
    return torch.round(y / step) * step


def _block64(x, keep):
    """One block x (tokens, dim) in 64 bits, keep (tokens,) -> (codes, scale)."""
    x = torch.where(keep[:, None], x, 0.0)
    top = float(x.abs().max())
    scale = 2.0 ** max(-126, math.ceil(math.log2(top / 448.0))) if top > 0 else 1.0
    return _e4m3(x / scale), scale


def _exact_attend8(case, s):
    b, Hq, Hkv, D, ps = (case[n] for n in ("batch", "heads", "kv_heads", "headdim", "page"))
    out = torch.zeros(b, Hq, D, dtype=torch.float64, device="cuda")
    for r, n in enumerate(_lengths(case)):
        ids = s["table"][r, :(n + ps - 1) // ps].long()
        full = n // ps
        k = s["k_pages"][ids[:full]].double() * s["k_scale"][ids[:full]].double()[:, :, None, None]
        v = s["v_pages"][ids[:full]].double() * s["v_scale"][ids[:full]].double()[:, :, None, None]
        k = torch.cat([k.transpose(0, 1).reshape(Hkv, full * ps, D),
                       s["k_tail"][r, :, :n % ps].double()], 1)
        v = torch.cat([v.permute(1, 0, 3, 2).reshape(Hkv, full * ps, D),
                       s["v_tail"][r, :, :, :n % ps].double().transpose(1, 2)], 1)
        score = torch.matmul(s["q"][r].double().view(Hkv, Hq // Hkv, D), k.transpose(1, 2).contiguous())
        score = score / math.sqrt(D)
        if s["gates"] is not None:
            gate = s["gates"][ids].double().transpose(0, 1).reshape(Hkv, -1)[:, :n].clone()
            gate[:, n - 1] = 0.0
            score = score + gate[:, None]
        out[r] = torch.matmul(torch.softmax(score, -1), v).reshape(Hq, D)
    return out


def _exact_cache(case, s):
    H, ps = case["kv_heads"], case["page"]
    build = case["kind"] == "build8"
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    ks, vs = s["k_scale"].double(), s["v_scale"].double()
    kt, vt = s["k_tail"].double(), s["v_tail"].double()
    gates = None if s["gates"] is None else s["gates"].double()
    for r, n in enumerate(_lengths(case)):
        ids = s["table"][r].tolist()
        if build:
            pages = range((n + ps - 1) // ps)
        else:
            kt[r, :, n % ps], vt[r, :, :, n % ps] = s["k"][r].double(), s["v"][r].double()
            if gates is not None:
                gates[ids[n // ps], :, n % ps] = s["log_gate"][r].double()
            pages = range(n // ps, (n + 1) // ps)
        for j in pages:
            m = min(ps, n - j * ps) if build else ps
            if build and gates is not None:
                gates[ids[j]] = -math.inf
                gates[ids[j], :, :m] = s["log_gate"][r, :, j * ps:j * ps + m].double()
            for h in range(H):
                if build:
                    k = torch.zeros(ps, kt.shape[-1], dtype=torch.float64, device="cuda")
                    v = torch.zeros_like(k)
                    k[:m] = s["k"][r, h, j * ps:j * ps + m].double()
                    v[:m] = s["v"][r, h, j * ps:j * ps + m].double()
                else:
                    k, v = kt[r, h], vt[r, h].t()
                if m < ps:
                    kt[r, h], vt[r, h] = k, v.t()
                    continue
                keep = torch.ones(ps, dtype=torch.bool, device="cuda")
                if gates is not None:
                    keep = gates[ids[j], h] > -math.inf
                    keep[-1] = True
                kp[ids[j], h], ks[ids[j], h] = _block64(k, keep)
                c, vs[ids[j], h] = _block64(v, keep)
                vp[ids[j], h] = c.t()
    return {"k_pages": kp, "v_pages": vp, "k_scale": ks, "v_scale": vs, "k_tail": kt, "v_tail": vt,
            "gates": gates, "lens": None}


def _exact_logprobs(case, s):
    x, rows = s["logits"].detach(), case["rows"]
    lp = torch.zeros(rows, dtype=torch.float64, device="cuda")
    H = torch.zeros_like(lp)
    tops = torch.zeros(rows, case["top"], dtype=torch.float64, device="cuda")
    grad = torch.zeros(x.shape, dtype=torch.float64, device="cuda") if case["train"] else None
    for a in range(0, rows, 512):
        y = x[a:a + 512].double()
        logp = y - torch.logsumexp(y, 1, keepdim=True)
        p = logp.exp()
        t = s["targets"][a:a + 512]
        ok = t != IGNORE
        hit = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0) * ok[:, None]
        H[a:a + 512] = -torch.xlogy(p, p).sum(1)
        lp[a:a + 512] = torch.where(hit > 0, logp, 0.0).sum(1)
        if case["top"]:
            tops[a:a + 512] = torch.topk(logp, case["top"], 1).values
        if grad is not None:
            g = s["g_logprob"][a:a + 512].double()[:, None] * ok[:, None]
            e = s["g_entropy"][a:a + 512].double()[:, None]
            grad[a:a + 512] = g * (hit - p) - e * (torch.xlogy(p, p) + p * H[a:a + 512, None])
    if case["train"]:
        return {"logprob": lp, "entropy": H, "dlogits": grad}
    if not case["top"]:
        return {"logprob": lp, "entropy": H}
    return {"logprob": lp, "entropy": H, "top_ids": None, "top_logprobs": tops}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "attend8":
        return _exact_attend8(case, s)
    if case["kind"] in ("append8", "build8"):
        return _exact_cache(case, s)
    if case["kind"] == "logprobs":
        return _exact_logprobs(case, s)
    N, K, G = case["outer"], case["inner"], case["group"]
    code = _codes(s["packed"], N, K).double()
    group = torch.arange(K, device="cuda") // G
    scale = s["scales"].double().permute(0, 2, 1).reshape(-1, s["scales"].shape[1])[:N][:, group]
    zero = 8.0
    if s["zeros"] is not None:
        zero = s["zeros"].double().permute(0, 2, 1).reshape(-1, s["zeros"].shape[1])[:N][:, group]
    w = torch.matmul(s["x"].double(), ((code - zero) * scale).t().contiguous())
    return w if s["bias"] is None else w + s["bias"].double()
