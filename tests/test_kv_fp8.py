"""The paged KV cache held in 8 bits (ops/kv_fp8.py): its two writes, code for
code, and the decode attention over it, against oracle/kv_fp8.py in float64.

Tolerance of the attention: with A = sum_j p_j |v_j| / l, the weights p are
rounded to bf16 (half a step, 2^-8, of each term) and the output once more
(2^-8 of it); a score of D products summed in fp32 is off by at most
e = (D + 4) 2^-24 (scale sum|q k| + |bias|), which moves numerator and
denominator by e each.
"""
import math

import pytest
import torch

from oracle import kv_fp8 as ref
from selective_attention.ops import (paged_decode_attn_fp8, paged_kv_append_fp8,
                                     paged_kv_build_fp8)

FP8 = torch.float8_e4m3fn
INF = math.inf


def make_cache(b, H, D, ps, width, gated, device, seed=0, fill=False):
    """A pool of b * width pages in shuffled order; fill: every byte of it random."""
    g = torch.Generator().manual_seed(seed)
    n = b * width
    table = torch.randperm(n, generator=g).to(torch.int32).view(b, width)
    c = dict(k_pages=torch.zeros(n, H, ps, D, dtype=torch.uint8),
             v_pages=torch.zeros(n, H, D, ps, dtype=torch.uint8),
             k_scale=torch.zeros(n, H), v_scale=torch.zeros(n, H),
             k_tail=torch.zeros(b, H, ps, D, dtype=torch.bfloat16),
             v_tail=torch.zeros(b, H, D, ps, dtype=torch.bfloat16),
             gate_pages=torch.full((n, H, ps), -INF) if gated else None)
    if fill:
        for name in ("k_pages", "v_pages"):
            c[name] = torch.randint(0, 256, c[name].shape, generator=g, dtype=torch.uint8)
        for name in ("k_scale", "v_scale", "k_tail", "v_tail"):
            c[name].fill_(math.nan)
        if gated:
            c["gate_pages"].fill_(7.0)
    c = {k: None if t is None else t.to(device) for k, t in c.items()}
    c["k_pages"], c["v_pages"] = c["k_pages"].view(FP8), c["v_pages"].view(FP8)
    return table.to(device), c


def tokens(b, H, L, D, gated, seed=0, spread=True):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(b, H, L, D, generator=g)
    v = torch.randn(b, H, L, D, generator=g)
    if spread:   # blocks and heads of very different sizes
        k = k * torch.exp2(torch.randint(-12, 13, (b, H, L, 1), generator=g).float() / 4)
        v = v * torch.exp2(torch.randint(-60, 60, (b, H, 1, 1), generator=g).float())
    lg = None
    if gated:
        lg = -torch.rand(b, H, L, generator=g) * 3
        lg[torch.rand(b, H, L, generator=g) < 0.2] = -INF
        lg[:, 0] = -INF     # one head drops every key
    return k.to(torch.bfloat16), v.to(torch.bfloat16), lg


def refs(k, v, lg, lens, ps):
    b, H, L, D = k.shape
    out = []
    for r in range(b):
        row = []
        for h in range(H):
            c = ref.CacheRef(ps, lg is not None)
            for t in range(min(lens[r], L)):
                c.append(k[r, h, t], v[r, h, t], 0.0 if lg is None else lg[r, h, t])
            row.append(c)
        out.append(row)
    return out


def same(got, want, name):
    """Equal value for value, NaN where NaN is wanted."""
    got, want = got.double().cpu(), want.double().cpu()
    ok = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert ok.all(), f"{name}: {int((~ok).sum())} of {ok.numel()} values differ"


def check_cache(c, table, rows, lens, before=None):
    """Every page, scale, tail slot and gate of the rows; the rest as before."""
    D, ps = c["k_pages"].shape[3], c["k_pages"].shape[2]
    gp = c["gate_pages"]
    seen_pages, table = set(), table.cpu()
    for r, row in enumerate(rows):
        n = lens[r]
        for h, cr in enumerate(row):
            for p, (kc, ks, vc, vs) in enumerate(cr.blocks()):
                pid = int(table[r, p])
                seen_pages.add(pid)
                same(c["k_pages"][pid, h].float(), kc, f"k codes {r} {h} {p}")
                same(c["v_pages"][pid, h].float(), vc.t(), f"v codes {r} {h} {p}")
                assert float(c["k_scale"][pid, h]) == ks and float(c["v_scale"][pid, h]) == vs
            m = n % ps
            if m:
                at = slice(n - m, n)
                same(c["k_tail"][r, h, :m], torch.stack(cr.k[at]), f"k tail {r} {h}")
                same(c["v_tail"][r, h, :, :m], torch.stack(cr.v[at]).t(), f"v tail {r} {h}")
            if gp is not None:
                for p in range((n + ps - 1) // ps):
                    pid = int(table[r, p])
                    seen_pages.add(pid)
                    g = torch.tensor(cr.g[p * ps:(p + 1) * ps])
                    same(gp[pid, h, :len(g)], g.float(), f"gates {r} {h} {p}")
    if before is not None:
        rest = [i for i in range(c["k_pages"].shape[0]) if i not in seen_pages]
        for name in ("k_pages", "v_pages", "k_scale", "v_scale", "gate_pages"):
            if c[name] is not None:
                a, b_ = c[name][rest], before[name][rest]
                if a.dtype == FP8:
                    a, b_ = a.view(torch.uint8), b_.view(torch.uint8)
                same(a, b_, f"{name} behind the rows")


def build(k, v, lg, table, lens, c, device="cuda"):
    paged_kv_build_fp8(k, v, lg, table, lens, c["k_pages"], c["v_pages"], c["k_scale"],
                       c["v_scale"], c["k_tail"], c["v_tail"], c["gate_pages"])


def append(k, v, lg, table, lens, c):
    paged_kv_append_fp8(k, v, lg, table, lens, c["k_pages"], c["v_pages"], c["k_scale"],
                        c["v_scale"], c["k_tail"], c["v_tail"], c["gate_pages"])


def attend(q, c, table, lens, **kw):
    kw.setdefault("key_bias", c["gate_pages"])
    return paged_decode_attn_fp8(q, c["k_pages"], c["v_pages"], c["k_scale"], c["v_scale"],
                                 c["k_tail"], c["v_tail"], table, lens, **kw)


def check_attention(o, q, rows, lens, scale=None, live=None):
    """o (b, Hq, D) against the rows' CacheRefs; live(r) -> bool per token or None."""
    b, Hq, D = q.shape
    Hkv = len(rows[0])
    sc = D ** -0.5 if scale is None else scale
    for r in range(b):
        for h in range(Hq):
            cr = rows[r][h // (Hq // Hkv)]
            if lens[r] == 0:
                assert torch.equal(o[r, h].cpu(), torch.zeros(D, dtype=o.dtype))
                continue
            k, v = cr.keys_values()
            g = torch.tensor(cr.g, dtype=torch.float64) if cr.gated else None
            want = ref.attend(q[r, h].cpu(), k, v, g, sc)
            on = torch.ones(len(k), dtype=torch.bool)
            if g is not None:
                on = g > -INF
                on[-1] = True
            A = ref.attend(q[r, h].cpu(), k[on], v[on].abs(), None if g is None else g[on], sc)
            big = sc * (k[on].abs() @ q[r, h].double().cpu().abs())
            if g is not None:
                big = big + g[on].abs()
            e = (D + 4) * 2.0 ** -24 * float(big.max())
            tol = (2.0 ** -8 + 2.5 * e) * A + 2.0 ** -8 * want.abs()
            err = (o[r, h].double().cpu() - want).abs()
            assert (err <= tol).all(), (r, h, float((err - tol).max()), float(err.max()))


# --- the oracle itself, on the CPU ---------------------------------------------
def test_oracle_rounds_as_e4m3():
    """Every e4m3 number, every midpoint of two neighbours, and bf16 values between."""
    codes = torch.arange(256, dtype=torch.int64).to(torch.uint8).view(FP8).double()
    codes = codes[torch.isfinite(codes)].unique()
    assert torch.equal(ref.e4m3(codes), codes)
    x = torch.cat([codes, (codes[1:] + codes[:-1]) / 2,
                   torch.randn(2000, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).double() * 60])
    x = x[x.abs() <= 448]
    assert torch.equal(ref.e4m3(x), x.float().to(FP8).double())


def test_oracle_scale_is_the_smallest_power_of_two():
    for top, want in ((448.0, 1.0), (449.0, 2.0), (224.0, 0.5), (225.0, 1.0), (0.0, 1.0),
                      (2.0 ** -133, 2.0 ** -126)):
        assert ref.block(torch.tensor([[top, -top / 2]]))[1] == want


# --- refusals: argument errors before any launch -------------------------------
def _args(b=2, H=2, D=64, ps=64, width=2, gated=True, device="cpu"):
    table, c = make_cache(b, H, D, ps, width, gated, device)
    return table, torch.zeros(b, dtype=torch.int32, device=device), c


@pytest.mark.parametrize("what", ["D", "ps", "dtype", "table", "lens", "gate", "strided", "k", "cpu",
                                  "empty"])
def test_append_and_build_refuse(what):
    table, lens, c = _args(D=96 if what == "D" else 64, ps=32 if what == "ps" else 64)
    D = c["k_pages"].shape[3]
    k = torch.zeros(2, 2, D, dtype=torch.bfloat16)
    lg = torch.zeros(2, 2)
    if what == "dtype":
        c["k_pages"] = c["k_pages"].view(torch.uint8)
    elif what == "table":
        table = table.long()
    elif what == "lens":
        lens = lens[:1]
    elif what == "gate":
        lg = None
    elif what == "strided":
        c["k_tail"] = c["k_tail"].transpose(2, 3).contiguous().transpose(2, 3)
    elif what == "k":
        k = k[:, :1]
    elif what == "empty":
        c = {n: t[:0] if n not in ("k_tail", "v_tail") else t for n, t in c.items()}
    with pytest.raises((ValueError, TypeError)):
        append(k, k, lg, table, lens, c)
    with pytest.raises((ValueError, TypeError)):
        k4 = k[:, :, None].expand(-1, -1, 5, -1)
        build(k4, k4, None if lg is None else lg[..., None].expand(-1, -1, 5), table, lens, c)


def test_attention_refuses_a_workspace_too_small():
    from selective_attention import _lib
    lib = _lib.load()
    assert lib.sa_paged_decode_fp8_workspace_size(1, 8, 8, 64, 64, 16) == 0    # 1024 keys: one launch
    need = lib.sa_paged_decode_fp8_workspace_size(2, 8, 8, 64, 64, 17)
    assert need == lib.sa_paged_decode_workspace_size(2, 8, 8, 64, 17) > 0
    at = 4096   # refused before any pointer is read
    for ws, nbytes in ((at, need - 1), (None, need)):
        assert lib.sa_paged_decode_fp8_fwd(at, at, at, at, at, at, at, at, at, None, 2, 8, 8, 64, 64, 17, 9,
                                           -1.0, at, ws, nbytes, None) == 1
    assert b"workspace" in lib.sa_last_error()


def test_append_refuses_tables_beyond_the_length_bits():
    from selective_attention import _lib
    lib = _lib.load()
    at = 4096   # refused before any pointer is read
    for pages, rows, rc in ((1 << 21, 0, 1), ((1 << 21) - 1, 0, 0), (1, 1 << 21, 1)):
        assert lib.sa_paged_kv_append_fp8(at, at, None, at, at, rows, 1, 64, 64, pages, 1, at, at, at,
                                          at, at, at, None, None) == rc
    assert b"too large" in lib.sa_last_error()


@pytest.mark.parametrize("what", ["heads", "group", "dtype", "D", "bias", "lens", "scale",
                                  "softmax", "cpu"])
def test_attention_refuses(what):
    table, lens, c = _args()
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    if what == "heads":
        q = q[:, :3]
    elif what == "group":
        q = torch.zeros(2, 34, 64, dtype=torch.bfloat16)
    elif what == "dtype":
        q = q.float()
    elif what == "D":
        q = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    elif what == "bias":
        c["gate_pages"] = c["gate_pages"].double()
    elif what == "lens":
        lens = torch.zeros(3, dtype=torch.int32)
    elif what == "scale":
        c["v_scale"] = c["v_scale"][:, :1]
    kw = dict(softmax_scale=0.0) if what == "softmax" else {}
    with pytest.raises((ValueError, TypeError)):
        attend(q, c, table, lens, **kw)


# --- the writes ------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("D,ps,gated", [(64, 64, True), (64, 128, False), (128, 64, False),
                                        (128, 128, True)])
def test_build_codes(D, ps, gated):
    lens = [0, 1, ps - 1, ps, ps + 1, 3 * ps, 2 * ps + 17]
    b, H, L = len(lens), 3, 3 * ps
    k, v, lg = tokens(b, H, L, D, gated)
    table, c = make_cache(b, H, D, ps, 4, gated, "cuda", fill=True)
    before = {n: None if t is None else t.clone() for n, t in c.items()}
    rows_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2).cuda()   # noqa: E731
    build(rows_first(k), rows_first(v), None if lg is None else lg.cuda(), table,
          torch.tensor(lens, dtype=torch.int32, device="cuda"), c)
    check_cache(c, table, refs(k, v, lg, lens, ps), lens, before)
    assert torch.isnan(c["k_tail"][0].float()).all()          # a row without tokens: as it was
    assert torch.isnan(c["v_tail"][3].float()).all()          # a row of full blocks: no open one
    assert not c["k_tail"][1, :, 1:].float().any()            # slots behind the open block's tokens
    if gated:
        pid = int(table[1, 0])
        assert (c["gate_pages"][pid, :, 1:] == -INF).all()


@pytest.mark.gpu
def test_build_clamps_lengths_and_skips_bad_pages():
    """Lengths beyond the tokens given, negative ones, and ids outside the pool."""
    b, H, D, ps, L = 4, 2, 64, 64, 100
    k, v, lg = tokens(b, H, L, D, True)
    table, c = make_cache(b, H, D, ps, 2, True, "cuda", fill=True)
    own = table.clone()
    table[2, 0], table[3, 1] = -1, table.numel()
    before = {n: t.clone() for n, t in c.items()}
    build(k.cuda(), v.cuda(), lg.cuda(), table,
          torch.tensor([1000, -5, 100, 100], dtype=torch.int32, device="cuda"), c)
    rows = refs(k, v, lg, [100, 0, 0, 0], ps)
    check_cache(c, own, rows, [100, 0, 0, 0])
    for name in ("k_pages", "gate_pages"):
        for pid in (int(own[1, 0]), int(own[2, 0]), int(own[3, 1])):
            a, b_ = c[name][pid], before[name][pid]
            same(a.float(), b_.float(), name)
    assert torch.isnan(c["k_tail"][3].float()).all()          # its open block has no page


@pytest.mark.gpu
@pytest.mark.parametrize("D,ps,gated", [(64, 64, True), (128, 64, False), (128, 128, True)])
def test_append_gives_the_codes_of_build(D, ps, gated):
    """Token by token from nothing, and behind a prompt, over two closings."""
    lens, H = [0, ps - 2, ps, 5], 2
    b, steps = len(lens), ps + 3
    k, v, lg = tokens(b, H, 2 * ps + 3, D, gated, seed=3)
    table, c = make_cache(b, H, D, ps, 3, gated, "cuda", fill=True)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), None if lg is None else lg.cuda(), table, sl, c)
    at = torch.tensor(lens)
    for s in range(steps):
        i = at + s
        r = torch.arange(b)
        append(k[r, :, i].cuda(), v[r, :, i].cuda(), None if lg is None else lg[r, :, i].cuda(),
               table, sl, c)
    end = [n + steps for n in lens]
    assert sl.tolist() == end
    check_cache(c, table, refs(k, v, lg, end, ps), end)


@pytest.mark.gpu
def test_append_at_the_tables_end_and_bad_pages():
    """A row whose table is full, and one whose page id is outside the pool: no
    page changes, the other rows are right."""
    b, H, D, ps = 3, 2, 64, 64
    k, v, lg = tokens(b, H, 130, D, True, seed=4)
    table, c = make_cache(b, H, D, ps, 2, True, "cuda")
    sl = torch.tensor([128, 127, 63], dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), lg.cuda(), table, sl, c)
    keep = {n: t.clone() for n, t in c.items()}
    bad = table.clone()
    bad[1, 1] = table.numel() + 3
    r = torch.arange(b)
    i = torch.tensor([128, 127, 63])
    append(k[r, :, i].cuda(), v[r, :, i].cuda(), lg[r, :, i].cuda(), bad, sl, c)
    assert sl.tolist() == [129, 128, 64]
    for name in ("k_pages", "gate_pages", "k_scale"):
        for row in (0, 1):
            ids = table[row].long()
            same(c[name][ids].float(), keep[name][ids].float(), name)
    rows = refs(k, v, lg, [0, 0, 64], ps)
    check_cache(c, table, rows, [0, 0, 64])


@pytest.mark.gpu
@pytest.mark.parametrize("H,D,ps,gated", [(3, 64, 64, True), (1, 128, 128, False), (9, 64, 128, True)])
def test_append_to_many_rows(H, D, ps, gated):
    """Rows at every place of a block, some closing; a row of length -1 stays."""
    b = 131
    lens = [(17 * r) % (2 * ps) for r in range(b)]
    lens[3], lens[50], lens[b - 1] = ps - 1, 2 * ps - 1, -1
    k, v, lg = tokens(b, H, 2 * ps, D, gated, seed=22)
    table, c = make_cache(b, H, D, ps, 2, gated, "cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), None if lg is None else lg.cuda(), table, sl, c)
    keep = {n: None if t is None else t.clone() for n, t in c.items()}
    r, i = torch.arange(b), torch.tensor(lens).clamp(min=0)
    append(k[r, :, i].cuda(), v[r, :, i].cuda(), None if lg is None else lg[r, :, i].cuda(), table, sl, c)
    assert sl.tolist() == [n + 1 if n >= 0 else -1 for n in lens]
    same(c["k_tail"][b - 1], keep["k_tail"][b - 1], "tail")
    same(c["v_tail"][b - 1], keep["v_tail"][b - 1], "tail")
    check_cache(c, table, refs(k, v, lg, [n + 1 for n in lens], ps), [n + 1 for n in lens])


@pytest.mark.gpu
def test_values_that_are_no_numbers():
    """Infinities and NaN: stored as NaN where the key is kept, as 0 where it is
    dropped, and without effect on the block's scale."""
    H, D, ps = 2, 64, 64
    k, v, _ = tokens(1, H, ps, D, False, spread=False)
    lg = torch.zeros(1, H, ps)
    k[0, 0, 5, 3], k[0, 0, 9, 1], v[0, 0, 7, 2] = math.nan, INF, -INF
    k[0, 1, 5], v[0, 1, 6], lg[0, 1, 5:7] = math.nan, INF, -INF
    table, c = make_cache(1, H, D, ps, 1, True, "cuda")
    sl = torch.full((1,), ps, dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), lg.cuda(), table, sl, c)
    check_cache(c, table, refs(k, v, lg, [ps], ps), [ps])
    table2, c2 = make_cache(1, H, D, ps, 1, True, "cuda")
    sl = torch.zeros(1, dtype=torch.int32, device="cuda")
    for t in range(ps):
        append(k[:, :, t].cuda(), v[:, :, t].cuda(), lg[:, :, t].cuda(), table2, sl, c2)
    check_cache(c2, table2, refs(k, v, lg, [ps], ps), [ps])


@pytest.mark.gpu
def test_sizes_at_the_ends_of_the_range():
    """All zeros, the smallest bf16 numbers, large ones, and the borders of a scale."""
    D, ps = 64, 64
    tops = [0.0, 2.0 ** -133, 2.0 ** -120, 448.0, 450.0, 446.0, 2.0 ** 100, 2.0 ** 127]
    H = len(tops)
    g = torch.Generator().manual_seed(1)
    k = torch.rand(1, H, ps, D, generator=g) * 2 - 1
    k = k * torch.tensor(tops)[None, :, None, None]
    k[..., 11, 5] = torch.tensor(tops)
    k = k.to(torch.bfloat16)
    table, c = make_cache(1, H, D, ps, 1, False, "cuda")
    build(k.cuda(), k.flip(1).cuda(), None, table,
          torch.full((1,), ps, dtype=torch.int32, device="cuda"), c)
    check_cache(c, table, refs(k, k.flip(1), None, [ps], ps), [ps])


# --- the attention -------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("D,ps,Hkv,grp,gated", [(64, 64, 2, 1, True), (64, 128, 2, 3, False),
                                                (128, 64, 2, 4, False), (128, 128, 1, 16, True),
                                                (128, 64, 2, 8, True), (64, 64, 3, 2, False)])
def test_attention(D, ps, Hkv, grp, gated):
    lens = [0, 1, 5, 63, 64, 65, 127, 128, 129, 200, 300]
    b = len(lens)
    k, v, lg = tokens(b, Hkv, max(lens), D, gated, seed=D + ps, spread=False)
    table, c = make_cache(b, Hkv, D, ps, (max(lens) + ps - 1) // ps, gated, "cuda", fill=True)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), None if lg is None else lg.cuda(), table, sl, c)
    q = torch.randn(b, Hkv * grp, D, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    rows = refs(k, v, lg, lens, ps)
    check_attention(attend(q.cuda(), c, table, sl), q, rows, lens)
    check_attention(attend(q.cuda(), c, table, sl, softmax_scale=0.3), q, rows, lens, scale=0.3)


@pytest.mark.gpu
def test_attention_many_rows():
    """More than 64 rows: the row plan has a kernel of its own."""
    g = torch.Generator().manual_seed(2)
    lens = [int(x) for x in torch.randint(0, 150, (70,), generator=g)]
    k, v, _ = tokens(70, 1, 150, 64, False, seed=5, spread=False)
    table, c = make_cache(70, 1, 64, 64, 3, False, "cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), None, table, sl, c)
    q = torch.randn(70, 2, 64, generator=g).to(torch.bfloat16)
    check_attention(attend(q.cuda(), c, table, sl), q, refs(k, v, None, lens, 64), lens)


@pytest.mark.gpu
def test_attention_one_long_row():
    """One row over every wave of the launch: 40,000 keys, checked in float64."""
    L, H, D, ps = 40000, 2, 64, 64
    k, v, lg = tokens(1, H, L, D, True, seed=6, spread=False)
    width = (L + ps - 1) // ps
    table, c = make_cache(1, H, D, ps, width, True, "cuda")
    sl = torch.full((1,), L, dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), lg.cuda(), table, sl, c)
    q = torch.randn(1, H, D, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    o = attend(q.cuda(), c, table, sl)
    ids, full = table[0].long(), L // ps
    for h in range(H):
        kk = (c["k_pages"][ids[:full], h].double() * c["k_scale"][ids[:full], h].double()[:, None, None]).reshape(-1, D)
        vv = (c["v_pages"][ids[:full], h].double() * c["v_scale"][ids[:full], h].double()[:, None, None]).transpose(1, 2).reshape(-1, D)
        assert L % ps == 0
        want = ref.attend(q[0, h], kk.cpu(), vv.cpu(), lg[0, h])
        A = ref.attend(q[0, h], kk.cpu(), vv.cpu().abs(), lg[0, h])
        err = (o[0, h].double().cpu() - want).abs()
        # fp32 scores of 64 products up to |s| < 8, off by 68 2^-24 8 < 2^-14 each way
        assert (err <= (2.0 ** -8 + 2.0 ** -13) * A + 2.0 ** -8 * want.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("D,ps", [(64, 64), (128, 128)])
def test_masked_places_hold_anything(D, ps):
    """NaN codes and NaN tail slots under -inf gates, behind a row's tokens and in
    pages of invalid ids change nothing."""
    lens = [ps * 2 + 9, ps + 1, ps * 2]
    b, H = len(lens), 2
    k, v, lg = tokens(b, H, max(lens), D, True, seed=8, spread=False)
    table, c = make_cache(b, H, D, ps, 3, True, "cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), lg.cuda(), table, sl, c)
    q = torch.randn(b, 2 * H, D, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16).cuda()
    clean = attend(q, c, table, sl)
    assert torch.isfinite(clean.float()).all()
    ku, vu = c["k_pages"].view(torch.uint8), c["v_pages"].view(torch.uint8)
    for r, n in enumerate(lens):
        dead = lg[r, :, :n] == -INF
        dead[:, n - 1] = False
        for h in range(H):
            for t in dead[h].nonzero()[:, 0].tolist():
                if t < n // ps * ps:
                    pid = int(table[r, t // ps])
                    ku[pid, h, t % ps], vu[pid, h, :, t % ps] = 0x7f, 0xff
                else:
                    c["k_tail"][r, h, t % ps], c["v_tail"][r, h, :, t % ps] = math.nan, INF
        c["k_tail"][r, :, n % ps:], c["v_tail"][r, :, :, n % ps:] = math.nan, math.nan
    assert torch.equal(attend(q, c, table, sl), clean)
    # a page outside the pool: its keys are gone, in a row's middle and at its end
    table2 = table.clone()
    table2[0, 0], table2[1, 1] = -1, table.numel()
    got = attend(q, c, table2, sl)
    rows = refs(k, v, lg, lens, ps)
    for cr in rows[0]:
        cr.g[:ps] = [-INF] * ps
    o0 = got[:1]
    # the refs round page 0 of row 0 anew without its gates, which takes no part
    check_attention(o0, q[:1], rows[:1], lens[:1])
    assert torch.equal(got[2], clean[2])


@pytest.mark.gpu
def test_no_rows_and_no_pages():
    table, c = make_cache(2, 2, 64, 64, 2, True, "cuda")
    z = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    empty = dict(c, k_tail=c["k_tail"][:0], v_tail=c["v_tail"][:0])
    assert attend(z, empty, table[:0], torch.zeros(0, **i32)).shape == (0, 2, 64)
    append(z, z, torch.zeros(0, 2, device="cuda"), table[:0], torch.zeros(0, **i32), empty)
    q = torch.ones(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    assert not attend(q, c, table[:, :0], torch.zeros(2, **i32)).any()


@pytest.mark.gpu
def test_other_index_types_and_strides_of_q():
    """int64 lengths and tables, q as a transposed view: the same answer."""
    b, H, D, ps = 2, 4, 64, 64
    k, v, lg = tokens(b, H, 100, D, True, seed=13, spread=False)
    table, c = make_cache(b, H, D, ps, 2, True, "cuda")
    sl = torch.tensor([100, 70], dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), lg.cuda(), table, sl, c)
    q = torch.randn(b, H, D, device="cuda").to(torch.bfloat16)
    want = attend(q, c, table, sl)
    assert torch.equal(attend(q.transpose(0, 1).contiguous().transpose(0, 1), c, table.long(), sl.long()), want)


@pytest.mark.gpu
def test_rows_that_the_mask_leaves_empty():
    """Every key dropped: the newest alone answers (its gate does not count)."""
    b, H, D, ps = 2, 2, 64, 64
    k, v, _ = tokens(b, H, 128, D, True, seed=11, spread=False)
    lg = torch.full((b, H, 128), -INF)
    table, c = make_cache(b, H, D, ps, 2, True, "cuda")
    lens = [128, 70]
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), lg.cuda(), table, sl, c)
    q = torch.randn(b, H, D).to(torch.bfloat16)
    o = attend(q.cuda(), c, table, sl).cpu()
    rows = refs(k, v, lg, lens, ps)
    for r in range(b):
        for h in range(H):
            assert torch.equal(o[r, h].double(), rows[r][h].keys_values()[1][-1])
    # the type's lowest value in place of -inf: the same answer
    low = torch.full_like(lg, torch.finfo(torch.float32).min)
    build(k.cuda(), v.cuda(), low.cuda(), table, sl, c)
    o = attend(q.cuda(), c, table, sl).cpu()
    rows = refs(k, v, low, lens, ps)
    for r in range(b):
        for h in range(H):
            assert torch.equal(o[r, h].double(), rows[r][h].keys_values()[1][-1])


@pytest.mark.gpu
def test_step_in_a_graph_and_on_another_stream():
    """append and attend captured once and replayed over a block's end, against
    the same calls eagerly, with other GPU work between the replays."""
    b, H, D, ps, steps = 3, 2, 64, 64, 70
    k, v, lg = (t.cuda() for t in tokens(b, H, 200, D, True, seed=12, spread=False))
    qs = torch.randn(steps, b, 2 * H, D, device="cuda").to(torch.bfloat16)
    start = torch.tensor([10, 60, 64], dtype=torch.int32, device="cuda")

    def fresh():
        table, c = make_cache(b, H, D, ps, 4, True, "cuda")
        sl = start.clone()
        build(k, v, lg, table, sl, c)
        return table, c, sl

    tok = lambda s: (k[:, :, 100 + s].contiguous(), v[:, :, 100 + s].contiguous(),   # noqa: E731
                     lg[:, :, 100 + s].contiguous())
    table, c, sl = fresh()
    want = []
    for s in range(steps):
        append(*tok(s), table, sl, c)
        want.append(attend(qs[s], c, table, sl))
    table, c, sl = fresh()
    kk, vv, gg = (t.clone() for t in tok(0))
    q = qs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        append(kk, vv, gg, table, sl, c)
        o = attend(q, c, table, sl)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        append(kk, vv, gg, table, sl, c)
        o = attend(q, c, table, sl)
    for s in range(1, steps):
        for dst, src in zip((kk, vv, gg), tok(s)):
            dst.copy_(src)
        q.copy_(qs[s])
        graph.replay()
        torch.randn(64, 64, device="cuda").sum()
        assert torch.equal(o, want[s]), s
    assert sl.tolist() == [x + steps for x in start.tolist()]


@pytest.mark.gpu
@pytest.mark.parametrize("run", [
    lambda: test_attention(64, 64, 2, 1, True), lambda: test_attention(64, 128, 2, 3, False),
    lambda: test_attention(128, 64, 2, 4, False), lambda: test_attention(128, 128, 1, 16, True),
    lambda: test_attention_many_rows(), lambda: test_masked_places_hold_anything(64, 64),
    lambda: test_masked_places_hold_anything(128, 128), lambda: test_no_rows_and_no_pages(),
    lambda: test_other_index_types_and_strides_of_q(), lambda: test_rows_that_the_mask_leaves_empty(),
    lambda: test_step_in_a_graph_and_on_another_stream()])
def test_attention_behind_wide_tables(monkeypatch, run):
    """The same checks with tables of at least 2304 keys, the rows' pages first:
    wide tables have a kernel of their own."""
    narrow = attend

    def wide(q, c, table, lens, **kw):
        pad = torch.full((table.shape[0], 36), -1, dtype=table.dtype, device=table.device)
        return narrow(q, c, torch.cat([table, pad], 1), lens, **kw)

    monkeypatch.setitem(globals(), "attend", wide)
    run()


@pytest.mark.gpu
@pytest.mark.parametrize("b,H,D,ps,lens,gated", [
    (1, 2, 64, 64, [1024], True), (2, 2, 128, 128, [1024, 1000], False), (1, 1, 128, 64, [961], True),
    (2, 64, 64, 128, [2048, 1930], True), (2, 64, 128, 64, [2047, 1], False)])
def test_attention_rows_as_long_as_a_short_table(b, H, D, ps, lens, gated):
    """Several tiles a wave, closed and open ones, where one workgroup takes a row."""
    L = max(lens)
    width = (L + ps - 1) // ps
    k, v, lg = tokens(b, H, L, D, gated, seed=21, spread=False)
    table, c = make_cache(b, H, D, ps, width, gated, "cuda", fill=True)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), None if lg is None else lg.cuda(), table, sl, c)
    q = torch.randn(b, H, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    o = attend(q.cuda(), c, table, sl).cpu()
    c = {name: None if t is None else t.cpu() for name, t in c.items()}
    for r, n in enumerate(lens):
        ids, full = table[r].long().cpu(), n // ps
        for h in sorted({0, 1 % H, H // 2, H - 1}):
            kk = (c["k_pages"][ids[:full], h].double() * c["k_scale"][ids[:full], h].double()[:, None, None]).reshape(-1, D)
            vv = (c["v_pages"][ids[:full], h].double() * c["v_scale"][ids[:full], h].double()[:, None, None]).transpose(1, 2).reshape(-1, D)
            kk = torch.cat([kk, c["k_tail"][r, h, :n - full * ps].double()])
            vv = torch.cat([vv, c["v_tail"][r, h, :, :n - full * ps].t().double()])
            on = torch.ones(n, dtype=torch.bool)
            if gated:
                on = lg[r, h, :n] > -INF
                on[-1] = True
            g = lg[r, h, :n][on] if gated else None
            want = ref.attend(q[r, h], kk[on], vv[on], g)
            A = ref.attend(q[r, h], kk[on], vv[on].abs(), g)
            big = D ** -0.5 * (kk[on].abs() @ q[r, h].double().abs())
            if gated:   # the newest key's gate does not count
                big[:-1] += g[:-1].double().abs()
            e = (D + 4) * 2.0 ** -24 * float(big.max())
            err = (o[r, h].double() - want).abs()
            assert (err <= (2.0 ** -8 + 2.5 * e) * A + 2.0 ** -8 * want.abs()).all(), (r, h)


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("D,ps,gated", [(64, 64, True), (64, 128, False), (128, 64, False), (128, 128, True)])
def test_attention_keeps_its_weights(D, ps, gated, wide):
    """Outputs that are small differences of large sums: as many values of 1 as of
    -1, under weights e^s of scores s in steps of 2^-7.  A weight stands in the
    products as two bf16 numbers, which is off by 2^-16 of it; s by 2.5 e A as in
    check_attention, e^s by 2^-21, the sums over the keys by (n / 32 + 40) 2^-24
    (n at most 600): below (2^-15 + 2.5 e) A together, and one rounding to bf16."""
    lens, H = [2, 10, 64, 70, 128, 256, 600], 2
    b, L = len(lens), max(lens)
    g = torch.Generator().manual_seed(D)
    k = torch.zeros(b, H, L, D)
    k[..., 0] = torch.randint(0, 16, (b, H, L), generator=g).float()   # exact in e4m3
    q = torch.zeros(b, H, D, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    v = torch.empty(b, H, L, D)
    for r, n in enumerate(lens):
        sign = torch.ones(H, D, n)
        sign[..., n // 2:] = -1.0
        at = torch.rand(H, D, n, generator=g).argsort(-1)
        v[r, :, :n] = sign.gather(-1, at).transpose(1, 2)
    k, v, lg = k.to(torch.bfloat16), v.to(torch.bfloat16), torch.zeros(b, H, L) if gated else None
    width = (L + ps - 1) // ps
    table, c = make_cache(b, H, D, ps, width, gated, "cuda")
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    build(k.cuda(), v.cuda(), None if lg is None else lg.cuda(), table, sl, c)
    if wide:
        table = torch.cat([table, torch.full((b, 36), -1, dtype=torch.int32, device="cuda")], 1)
    sc = 2.0 ** -7
    o = attend(q.cuda(), c, table, sl, softmax_scale=sc).double().cpu()
    e = (D + 4) * 2.0 ** -24 * sc * 15
    for r, cr in enumerate(refs(k, v, lg, lens, ps)):
        for h in range(H):
            kk, vv = cr[h].keys_values()
            want = ref.attend(q[r, h], kk, vv, None, sc)
            err = (o[r, h] - want).abs()      # A = 1
            assert (err <= 2.0 ** -15 + 2.5 * e + 2.0 ** -8 * want.abs()).all(), (lens[r], h, float(err.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("wide", [False, True])
def test_infinite_values_of_an_open_block(D, wide):
    """They stand as they are until the block is rounded: the output has them, in
    their own dimension alone, and NaN where both signs meet."""
    H, ps, n = 2, 64, 90
    k, v, _ = tokens(1, H, n, D, False, seed=14, spread=False)
    clean_v = v.clone()
    v[0, 0, 70, 3], v[0, 0, 80, 5], v[0, 0, 64, 9], v[0, 0, 89, 9] = INF, -INF, INF, -INF
    q = torch.randn(1, H, D, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16)
    sl = torch.full((1,), n, dtype=torch.int32, device="cuda")
    out = []
    for values in (clean_v, v):
        table, c = make_cache(1, H, D, ps, 2, False, "cuda")
        build(k.cuda(), values.cuda(), None, table, sl, c)
        if wide:
            table = torch.cat([table, torch.full((1, 36), -1, dtype=torch.int32, device="cuda")], 1)
        out.append(attend(q.cuda(), c, table, sl).float().cpu())
    clean, o = out
    assert o[0, 0, 3] == INF and o[0, 0, 5] == -INF and torch.isnan(o[0, 0, 9])
    rest = [d for d in range(D) if d not in (3, 5, 9)]
    assert torch.equal(o[0, 0, rest], clean[0, 0, rest]) and torch.equal(o[0, 1], clean[0, 1])
