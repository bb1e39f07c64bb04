"""4-bit linear layers (ops/int4.py) against oracle/int4.py in float64.

Tolerance of the kernel: the products of x and 1 + c / 16 (1 to 1.94) are exact
and summed in fp32, as is sum x; their difference stands for terms of |c - z| / 16
down to 1/16.  With A1 = sum_k s |x_k| 16 (1.94 + 1.94) the sums' rounding is at
most (K / 32 + 36) 2^-24 of A1 (32 terms a step on the matrix cores, K / 32
steps and groups, then at most 36 sums of groups and waves), and the result is
rounded once to bf16, half a step, 2^-8 of it at most.
"""
import pytest
import torch

from oracle import int4 as ref
from selective_attention.modules.layers import Int4Linear, Linear, project
from selective_attention.ops import (dequantize_int4, int4_linear, int4_linear_multi, pack_int4,
                                     quantize_int4)


def make(N, K, G, zeros, seed=0, bias=False):
    g = torch.Generator().manual_seed(seed)
    groups = (K + G - 1) // G
    codes = torch.randint(0, 16, (N, K), generator=g)
    scales = (torch.randn(N, groups, generator=g) * 0.02).to(torch.bfloat16)
    z = torch.randint(0, 16, (N, groups), generator=g).to(torch.bfloat16) if zeros else None
    b = torch.randn(N, generator=g).to(torch.bfloat16) if bias else None
    return codes, scales, z, b


def bound(x, w, want, scales, K, xscale=None):
    xx = (x if xscale is None else x * xscale).double().abs()
    G = 128 * ((K + 127) // 128) // scales.shape[1]
    of = torch.arange(K) // G
    s = scales.double().abs().transpose(1, 2).reshape(-1, scales.shape[1])[:w.shape[0]][:, of]
    A1 = 16 * 3.9 * (xx @ s.t())
    return (K / 32 + 36) * 2.0 ** -24 * A1 + 2.0 ** -8 * want.abs() + 2.0 ** -133


def check(y, x, packed, N, K, bias=None, xscale=None):
    w = ref.weight(*packed, N, K)
    want, _ = ref.linear(x, w, bias, xscale)
    err = (y.double().cpu() - want).abs()
    tol = bound(x, w, want, packed[1], K, xscale)
    assert y.shape == want.shape and (err <= tol).all(), (float((err - tol).max()), float(err.max()))


def dev(packed):
    return tuple(None if t is None else t.cuda() for t in packed)


# --- layout and rounding, on the CPU ---------------------------------------------
@pytest.mark.parametrize("N,K,G,zeros", [(16, 128, 128, False), (33, 100, 32, True), (1, 1, 64, True),
                                         (50, 300, 64, False)])
def test_pack_keeps_codes_and_factors(N, K, G, zeros):
    codes, scales, z, _ = make(N, K, G, zeros)
    packed, s, zz = pack_int4(codes, scales, z, G)
    assert packed.shape == ((N + 15) // 16, (K + 127) // 128, 64, 16)
    assert torch.equal(ref.unpack(packed, N, K), codes)
    of = torch.arange(K) // G
    want = scales.double()[:, of] * (codes.double() - (8.0 if z is None else z.double()[:, of]))
    assert torch.equal(ref.weight(packed, s, zz, N, K), want)
    assert torch.isfinite(s.float()).all()


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("G", [32, 128])
def test_quantize_rounds_to_the_nearest_code(symmetric, G):
    g = torch.Generator().manual_seed(1)
    N, K = 20, 200
    w = torch.randn(N, K, generator=g)
    w[3] = 0.0
    w[4] = w[4].abs()
    packed = quantize_int4(w, G, symmetric)
    got = ref.weight(*packed, N, K)
    of = torch.arange(K) // G
    s = packed[1].double().transpose(1, 2).reshape(-1, packed[1].shape[1])[:N][:, of]
    # half a step; the range's ends stand off by the bf16 rounding of the scale
    # (2^-8 of 7, 8 or 15 steps) and, with zero points, by their rounding
    ends = 15 * 2.0 ** -8 + (0.0 if symmetric else 0.5)
    assert ((got - w.double()).abs() <= s * (0.5 + ends)).all()
    inner = (w.double() / s).abs() <= 6.0
    if symmetric:
        assert ((got - w.double()).abs() <= s * (0.5 + 1e-6))[inner].all()
    assert not got[3].any()


@pytest.mark.parametrize("what", ["dtype", "rows", "packed", "scales", "zeros", "group", "bias",
                                  "xscale", "mixed", "count", "cpu"])
def test_linear_refuses(what):
    codes, scales, z, b = make(32, 128, 64, True, bias=True)
    p = list(pack_int4(codes, scales, z, 64))
    x = torch.zeros(2, 128, dtype=torch.bfloat16)
    kw = dict(out_features=32)
    if what == "dtype":
        x = x.float()
    elif what == "rows":
        kw = dict(out_features=48)
    elif what == "packed":
        p[0] = p[0].view(torch.int8)
    elif what == "scales":
        p[1] = p[1].float()
    elif what == "zeros":
        p[2] = p[2][:, :1]
    elif what == "group":
        p[1] = p[2] = torch.zeros(2, 3, 16, dtype=torch.bfloat16)
    elif what == "bias":
        kw["bias"] = b[:31]
    elif what == "xscale":
        kw["xscale"] = x[:1]
    with pytest.raises((ValueError, TypeError)):
        if what == "mixed":
            int4_linear_multi(x, [tuple(p), (p[0], p[1], None)], [None, None], [32, 32])
        elif what == "count":
            int4_linear_multi(x, [tuple(p)] * 5, [None] * 5, [32] * 5)
        else:
            int4_linear(x, *p, **kw)


@pytest.mark.parametrize("what", ["range", "float", "group", "scales"])
def test_pack_refuses(what):
    codes, scales, z, _ = make(32, 128, 64, True)
    kw = dict(group_size=64)
    if what == "range":
        codes[0, 0] = 16
    elif what == "float":
        codes = codes.float()
    elif what == "group":
        kw = dict(group_size=48)
    else:
        scales = scales[:, :1]
    with pytest.raises((ValueError, TypeError)):
        pack_int4(codes, scales, z, **kw)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_quantize_refuses_weights_that_are_no_numbers(bad):
    w = torch.ones(16, 64)
    w[3, 5] = bad
    with pytest.raises(ValueError):
        quantize_int4(w, 32)


# --- the kernel ------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 7, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("N,K,G,zeros", [(64, 256, 128, False), (100, 1000, 32, True),
                                         (17, 72, 64, True), (257, 2055, 128, True),
                                         (1, 1, 32, False), (48, 640, 64, False)])
def test_linear(M, N, K, G, zeros):
    codes, scales, z, b = make(N, K, G, zeros, seed=M, bias=M % 2 == 1)
    packed = pack_int4(codes, scales, z, G)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(torch.bfloat16)
    y = int4_linear(x.cuda(), *dev(packed), bias=None if b is None else b.cuda(), out_features=N)
    check(y, x, packed, N, K, b)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 20, 64])
@pytest.mark.parametrize("N,K,G,zeros", [(40, 4096, 64, True), (5000, 1100, 128, False),
                                         (40, 4100, 128, False), (50, 2100, 32, True)])
def test_linear_long(M, N, K, G, zeros):
    """The widest x that stays in registers, more tiles than workgroups, and the
    columns behind that."""
    codes, scales, z, b = make(N, K, G, zeros, seed=M, bias=True)
    packed = pack_int4(codes, scales, z, G)
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(torch.bfloat16)
    y = int4_linear(x.cuda(), *dev(packed), bias=b.cuda(), out_features=N)
    check(y, x, packed, N, K, b)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 40])
@pytest.mark.parametrize("K", [384, 4300])
def test_multi_with_xscale(M, K):
    """Four weights of one x * xscale in one launch, outputs of their own."""
    G, sizes = 64, [16, 100, 33, 1]
    g = torch.Generator().manual_seed(5)
    x, f = (torch.randn(M, K, generator=g).to(torch.bfloat16) for _ in range(2))
    ws, bs = [], []
    for i, N in enumerate(sizes):
        codes, scales, z, b = make(N, K, G, True, seed=i, bias=i != 1)
        ws.append(pack_int4(codes, scales, z, G))
        bs.append(b)
    ys = int4_linear_multi(x.cuda(), [dev(w) for w in ws], [None if b is None else b.cuda() for b in bs],
                           sizes, xscale=f.cuda())
    for y, w, b, N in zip(ys, ws, bs, sizes):
        check(y, x, w, N, K, b, f)
        assert y.is_contiguous()


@pytest.mark.gpu
def test_strides_and_alignment():
    """x transposed, off a 16-byte boundary, with leading dimensions, and empty."""
    N, K, G = 40, 200, 64
    codes, scales, z, _ = make(N, K, G, False)
    packed = pack_int4(codes, scales, z, G)
    d = dev(packed)
    x = torch.randn(6, K, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    xg = x.cuda()
    want = int4_linear(xg, *d, out_features=N)
    check(want, x, packed, N, K)
    assert torch.equal(int4_linear(xg.t().contiguous().t(), *d, out_features=N), want)
    off = torch.zeros(6 * K + 3, dtype=torch.bfloat16, device="cuda")
    off[3:] = xg.flatten()
    assert torch.equal(int4_linear(off[3:].view(6, K), *d, out_features=N), want)
    assert torch.equal(int4_linear(xg.view(2, 3, K), *d, out_features=N), want.view(2, 3, N))
    assert int4_linear(xg[:0], *d, out_features=N).shape == (0, N)


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,G,zeros", [(1, 40, 999, 128, False), (20, 40, 1001, 64, True), (5, 50, 2047, 32, False),
                                           (40, 33, 3999, 128, True), (3, 40, 4097, 64, False), (64, 20, 2050, 32, True),
                                           (33, 24, 5002, 128, False), (2, 16, 1, 32, False), (7, 16, 1024, 64, False)])
def test_rows_off_every_boundary(M, N, K, G, zeros):
    """Odd lengths, strides and offsets; what stands beside the rows is not read
    into them."""
    codes, scales, z, b = make(N, K, G, zeros, seed=K, bias=True)
    packed = pack_int4(codes, scales, z, G)
    d, bias = dev(packed), b.cuda()
    g = torch.Generator().manual_seed(M)
    x, f = (torch.randn(M, K, generator=g).to(torch.bfloat16) for _ in range(2))
    want = int4_linear(x.cuda(), *d, bias=bias, out_features=N)
    check(want, x, packed, N, K, b)
    for shift in (1, 2, 3, 8):
        flat = torch.full((M * K + shift + 9,), float("nan"), dtype=torch.bfloat16, device="cuda")
        flat[shift:shift + M * K] = x.cuda().flatten()
        rows = flat[shift:shift + M * K].view(M, K)
        assert torch.equal(int4_linear(rows, *d, bias=bias, out_features=N), want)
        wide = torch.full((M, K + 2 * shift), float("nan"), dtype=torch.bfloat16, device="cuda")
        wide[:, shift:shift + K] = x.cuda()
        assert torch.equal(int4_linear(wide[:, shift:shift + K], *d, bias=bias, out_features=N), want)
        y = int4_linear(rows, *d, bias=bias, out_features=N, xscale=f.cuda())
        check(y, x, packed, N, K, b, f)
        got = int4_linear(wide[:, shift:shift + K], *d, bias=bias, out_features=N, xscale=f.cuda())
        assert torch.equal(got, y)


@pytest.mark.gpu
def test_what_is_no_number_stays_in_its_row():
    N, K, G = 32, 256, 128
    codes, scales, z, _ = make(N, K, G, True)
    d = dev(pack_int4(codes, scales, z, G))
    x = torch.randn(20, K).to(torch.bfloat16).cuda()
    clean = int4_linear(x, *d, out_features=N)
    x[3, 7], x[17, 200] = float("nan"), float("inf")
    y = int4_linear(x, *d, out_features=N)
    rows = [i for i in range(20) if i not in (3, 17)]
    assert torch.equal(y[rows], clean[rows])
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[17]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("N,K,G,zeros", [(100, 1000, 32, True), (16, 128, 128, False), (33, 77, 64, True)])
def test_dequantize(N, K, G, zeros):
    codes, scales, z, _ = make(N, K, G, zeros)
    packed = pack_int4(codes, scales, z, G)
    got = dequantize_int4(*dev(packed), out_features=N, in_features=K)
    # scale (8 bits) times a difference of codes (4 bits) is exact in fp32: one rounding
    assert torch.equal(got.cpu(), ref.weight(*packed, N, K).to(torch.bfloat16))


@pytest.mark.gpu
def test_many_rows_and_gradients():
    """More than 64 rows, and rows that take a gradient: a plain product with the
    widened weights."""
    N, K, G = 96, 256, 64
    codes, scales, z, b = make(N, K, G, True, bias=True)
    packed = pack_int4(codes, scales, z, G)
    d = dev(packed)
    w = ref.weight(*packed, N, K)
    x = torch.randn(100, K, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    y = int4_linear(x.cuda(), *d, bias=b.cuda(), out_features=N)
    want, A = ref.linear(x, w, b)
    # bf16 weights (2^-8 of each term) and the result's rounding; fp32 sums
    assert ((y.double().cpu() - want).abs() <= (2.0 ** -8 + K * 2.0 ** -24) * A + 2.0 ** -8 * want.abs()).all()
    xg = x[:4].cuda().requires_grad_(True)
    dy = torch.randn(4, N, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    (dx,) = torch.autograd.grad(int4_linear(xg, *d, out_features=N), xg, dy.cuda())
    want, A = dy.double() @ w, dy.double().abs() @ w.abs()
    assert ((dx.double().cpu() - want).abs() <= (2.0 ** -8 + N * 2.0 ** -24) * A + 2.0 ** -8 * want.abs()).all()


@pytest.mark.gpu
def test_graph_replays():
    N, K, G = 200, 512, 128
    codes, scales, z, b = make(N, K, G, False, bias=True)
    d = dev(pack_int4(codes, scales, z, G))
    b = b.cuda()
    xs = torch.randn(5, 3, K, device="cuda").to(torch.bfloat16)
    want = [int4_linear(x, *d, bias=b, out_features=N) for x in xs]
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        int4_linear(x, *d, bias=b, out_features=N)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = int4_linear(x, *d, bias=b, out_features=N)
    for i in range(5):
        x.copy_(xs[i])
        graph.replay()
        torch.randn(64, 64, device="cuda").sum()
        assert torch.equal(y, want[i])


# --- the layer ---------------------------------------------------------------------
def test_layer_state_dict_round_trip():
    lin = Linear(100, 40)
    q = Int4Linear.from_linear(lin, group_size=32)
    assert not list(q.parameters())
    other = Int4Linear(100, 40, group_size=32)
    other.load_state_dict(q.state_dict())
    assert torch.equal(other.packed, q.packed) and torch.equal(other.scales, q.scales)
    assert torch.equal(other.bias, q.bias)
    q.to(torch.float32).to(torch.float64)     # a cast of the module leaves the weight as it is
    assert q.scales.dtype == torch.bfloat16 and q.bias.dtype == torch.bfloat16


@pytest.mark.gpu
def test_layer_matches_linear_on_its_own_weights():
    """Int4Linear.forward, split_forward and project against nn.Linear with the
    weights that the codes stand for."""
    torch.manual_seed(0)
    K, sizes = 256, [48, 17, 64]
    lin = Linear(K, sum(sizes)).cuda().to(torch.bfloat16)
    q = Int4Linear.from_linear(lin, group_size=64)
    w = ref.weight(q.packed.cpu(), q.scales.cpu(), None, sum(sizes), K)
    x = torch.randn(4, K).to(torch.bfloat16)
    with torch.no_grad():
        y = q(x.cuda())
        check(y, x, (q.packed.cpu(), q.scales.cpu(), None), sum(sizes), K, q.bias.cpu())
        parts = q.split_forward(x.cuda(), sizes)
        assert torch.equal(torch.cat(parts, -1), y) and all(p.is_contiguous() for p in parts)
        f = torch.randn(4, K).to(torch.bfloat16)
        a, b = project(x.cuda(), [q, q], xscale=f.cuda())
        check(a, x, (q.packed.cpu(), q.scales.cpu(), None), sum(sizes), K, q.bias.cpu(), f)
        assert torch.equal(a, b)
        mixed = project(x.cuda(), [q, lin])
        assert torch.equal(mixed[0], y)
        assert torch.equal(mixed[1], lin(x.cuda()))
    assert (w - lin.weight.double().cpu()).abs().max() <= 0.55 * q.scales.double().abs().max()


# --- groups without a weight -------------------------------------------------------
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("G", [32, 64, 128])
def test_quantize_gives_a_group_of_zeros_the_scale_zero(G, symmetric):
    w = torch.randn(20, 300, generator=torch.Generator().manual_seed(2))
    w[3] = 0.0
    w[:, G:2 * G] = 0.0
    packed = quantize_int4(w, G, symmetric)
    s = packed[1].float().transpose(1, 2).reshape(-1, packed[1].shape[1])[:20, :(300 + G - 1) // G]
    zero = torch.zeros_like(s, dtype=torch.bool)
    zero[3], zero[:, 1] = True, True
    assert not s[zero].any() and (s[~zero] > 0).all()
    assert not ref.weight(*packed, 20, 300)[w == 0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("M,K,G", [(1, 256, 128), (7, 1000, 32), (20, 2055, 64), (64, 4300, 128), (80, 512, 64)])
def test_groups_of_zeros_add_nothing(M, K, G, symmetric):
    """A weight's rows and groups of zeros beside large activations: exactly nothing."""
    g = torch.Generator().manual_seed(K)
    w = torch.randn(40, K, generator=g) * 0.02
    w[[0, 17, 39]] = 0.0
    w[:, G:2 * G] = 0.0
    b = torch.randn(40, generator=g).to(torch.bfloat16)
    x = torch.randn(M, K, generator=g).to(torch.bfloat16)
    packed = quantize_int4(w, G, symmetric)
    d = dev(packed)
    base = int4_linear(x.cuda(), *d, bias=b.cuda(), out_features=40)
    x[:, G:2 * G] *= 10000.0
    y = int4_linear(x.cuda(), *d, bias=b.cuda(), out_features=40)
    assert torch.equal(y, base)
    x *= 10000.0
    y = int4_linear(x.cuda(), *d, bias=b.cuda(), out_features=40).cpu()
    assert torch.equal(y[:, [0, 17, 39]], b[[0, 17, 39]].expand(M, 3))


def test_linear_refuses_grids_beyond_the_launch():
    """Tile by tile (K of more than 4096) two tiles are a workgroup of 512 threads, and
    a launch has fewer than 2^32; the kernel that streams its tiles has no such limit."""
    import ctypes

    from selective_attention import _lib
    lib, at = _lib.load(), 4096   # refused before any pointer is read
    words = [at, at, 0, 0, at, 1 << 26] * 4
    rc = lib.sa_int4_linear_bf16(at, None, 1, 4352, 4352, 128, 4, (ctypes.c_int64 * 24)(*words), None)
    assert rc == 1 and b"too many columns" in lib.sa_last_error()
    words = [at, at, 0, 0, at, 1 << 30] * 4
    rc = lib.sa_int4_linear_bf16(at, None, 1, 128, 128, 128, 4, (ctypes.c_int64 * 24)(*words), None)
    assert rc == 1 and b"too many columns" in lib.sa_last_error()
