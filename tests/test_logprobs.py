"""Token log probabilities (ops/logprobs.py) against oracle/logprobs.py in
float64.

Tolerances (half a step of fp32 is u = 2^-24).  With d = x - m the relative error
of e^d is at most (3 |d| + 4) u: log2(e)'s rounding, the exponent's, exp2's.  Summed
over the terms, s is off by (3 |t / s| + 4) u, |t / s| <= log V < 12, and by the
sum's order, 64 terms a thread, then 20 levels: 84 u.  So log s is off by
(40 + 84) u < 8e-6, a logprob by that and two roundings of its own (4 u of it).
t's terms are off by (3 |d| + 6) u each, sum d^2 e^d / s < 250: 3 250 + 6 12 + 84
12 u < 1.2e-4, the entropy's bound.  In a gradient p is off by 8e-6 + (3 40 + 4)
u < 1.6e-5 and log p + H, below 52, by 1.3e-4: p |g| (52 1.6e-5 + 1.3e-4) < 1e-3
p |g|; where a target's or alternative's own term stands, 4 u |g| more; and one
rounding to the logits' type.
"""
import math

import pytest
import torch

from oracle import logprobs as ref
from selective_attention.ops import token_logprobs

INF = math.inf
E_LP, E_H, E_P = 8e-6, 1.2e-4, 1e-3


def make(rows, V, dtype, seed=0, banned=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, V, generator=g) * 3
    if banned:
        x[torch.rand(rows, V, generator=g) < banned] = -INF
        x[:, 0] = 1.0
    t = torch.randint(0, V, (rows,), generator=g)
    return x.to(dtype), t


def near(got, want, name, tol=E_LP):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, name
    fin = torch.isfinite(want)
    assert torch.equal(fin, torch.isfinite(got)), f"{name}: not the same finite places"
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{name}: NaN"
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), name
    err = (got - want).abs()[fin]
    bad = err > tol + 2.0 ** -22 * want.abs()[fin]
    assert not bad.any(), (name, float(err.max()))


def check(x, t, top, **kw):
    out = token_logprobs(x.cuda(), t.cuda(), top=top, **kw)
    lp, H, ids, tl = ref.forward(x, t.long(), top, kw.get("ignore_index", -100))
    near(out.logprob, lp, "logprob")
    near(out.entropy, H, "entropy", E_H)
    assert torch.equal(out.top_ids.cpu(), ids)
    near(out.top_logprobs, tl, "top_logprobs")
    return out


# --- refusals ------------------------------------------------------------------
def test_refuses_rows_beyond_the_kernels_offsets():
    x = torch.zeros(1, 1, dtype=torch.bfloat16).expand(1, (1 << 28) + 1)
    with pytest.raises(ValueError, match="vocabulary"):
        token_logprobs(x, torch.zeros(1, dtype=torch.int64))
    from selective_attention import _lib
    lib, at = _lib.load(), 4096   # refused before any pointer is read
    assert lib.sa_token_logprobs_fwd(1, at, 8, at, 1 << 23, 8, 0, -100, at, at, at, None, None, None, 0, None) == 1
    assert b"bad sizes" in lib.sa_last_error()


@pytest.mark.parametrize("what", ["dtype", "targets", "shape", "top", "vocab", "empty", "cpu"])
def test_refuses(what):
    x, t = make(3, 50, torch.float32)
    top = 5
    if what == "dtype":
        x = x.double()
    elif what == "targets":
        t = t.float()
    elif what == "shape":
        t = t[:2]
    elif what == "top":
        top = 65
    elif what == "vocab":
        x, top = x[:, :4], 5
    elif what == "empty":
        x, top = x[:, :0], 0
    with pytest.raises((ValueError, TypeError)):
        token_logprobs(x, t, top=top)


def test_oracle_gradient_against_differences():
    x, t = make(2, 9, torch.float64, seed=3)
    g_lp, g_h, g_top = torch.randn(2), torch.randn(2), torch.randn(2, 3)
    d = ref.backward(x, t, g_lp, g_h, g_top, top=3)

    def f(x):
        lp, H, _, tl = ref.forward(x, t, 3)
        return float((g_lp * lp + g_h * H).sum() + (g_top * tl).sum())
    for r in range(2):
        for j in range(9):
            e = torch.zeros_like(x)
            e[r, j] = 1e-5
            assert abs((f(x + e) - f(x - e)) / 2e-5 - float(d[r, j])) < 1e-6


# --- forward -------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,top", [(1, 1), (2, 2), (7, 3), (64, 64), (100, 20), (1001, 5), (4096, 64),
                                   (4100, 64), (16384, 20), (16390, 1), (32000, 20), (33003, 64),
                                   (70001, 33), (131072, 0)])
def test_forward(V, top, dtype):
    x, t = make(5, V, dtype, seed=V, banned=0.1 if V > 2 else 0.0)
    check(x, t, top)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [50, 4096, 20000, 40000])
@pytest.mark.parametrize("order", ["equal", "ascending", "descending", "two", "zeros", "few", "block"])
def test_alternatives_in_hard_orders(V, order):
    """Ties go to the lowest id; sorted rows and clusters defeat the threshold."""
    top = 32
    j = torch.arange(V).float()
    if order == "equal":
        x = torch.full((1, V), 1.5)
    elif order == "ascending":
        x = (j / V)[None]
    elif order == "descending":
        x = (-j / V)[None]
    elif order == "two":
        x = (j % 2)[None]
    elif order == "zeros":
        x = torch.where(j % 3 == 0, 0.0, -0.0)[None]
    elif order == "few":      # fewer than top tokens are allowed
        x = torch.full((1, V), -INF)
        x[0, [3, V // 2, V - 1]] = torch.tensor([0.5, 2.0, 0.5])
    else:                     # every large value inside one thread's and one lane's logits
        x = torch.randn(1, V, generator=torch.Generator().manual_seed(0))
        lanes = (torch.arange(V) // 8) % 64
        x[0, lanes < 20] += 10.0
    for dtype in (torch.float32, torch.bfloat16):
        one = check(x.to(dtype), torch.tensor([V - 1]), top)
        # many rows: another split of the row, the same answer
        many = token_logprobs(x.to(dtype).cuda().expand(512, V).contiguous(),
                              torch.full((512,), V - 1, device="cuda"), top=top)
        assert torch.equal(many.top_ids, one.top_ids.expand(512, top))
        # (rows stand at different places to a 16-byte boundary: other threads add
        # other logits, each row within the bound of the exact value)
        assert (many.logprob - many.logprob[:1]).abs().max() <= 2 * E_LP
        for a, b, tol in zip(many, one, (E_LP, E_H, 0, E_LP)):
            near(a[:1], b.cpu(), "many rows", 2 * tol)


@pytest.mark.gpu
@pytest.mark.parametrize("V,top", [(20001, 7), (40001, 0), (40001, 20)])
def test_many_rows_of_several_pieces(V, top):
    x, t = make(515, V, torch.bfloat16, seed=V, banned=0.1)
    check(x, t, top)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [6, 600])
def test_rows_of_no_numbers(rows):
    """Rows of -inf alone, with NaN, with +inf: NaN; the rows beside them stand."""
    for V in (100, 5000, 40000):
        x, t = make(rows, V, torch.float32, seed=1)
        x[1] = -INF
        x[2, V // 3] = math.nan
        x[3, V // 2] = INF
        x[4, t[4]] = -INF
        out = token_logprobs(x.cuda(), t.cuda(), top=4)
        want = ref.forward(x[[0, 4, 5]], t[[0, 4, 5]], 4)
        for got, w, name in zip(out, want, out._fields):
            if name != "top_ids":
                near(got[[0, 4, 5]], w, name, E_H if name == "entropy" else E_LP)
        assert torch.equal(out.top_ids[[0, 4, 5]].cpu(), want[2])
        for r in (1, 2, 3):
            assert torch.isnan(out.logprob[r]) and torch.isnan(out.entropy[r])
        assert out.top_ids[1].tolist() == [0, 1, 2, 3]
        assert out.top_ids[2, 0] == V // 3 and out.top_ids[3, 0] == V // 2


@pytest.mark.gpu
def test_one_large_logit():
    """All the probability at one token, at any size of its logit: log p is 0 to
    fp32's step at 1, never above, and the entropy 0, never below."""
    for size in (30.0, 127.5, 1000.0, -1000.0, 3.0e4):
        x = torch.full((3, 500), size - 50.0)
        x[:, 7] = size
        out = token_logprobs(x.cuda(), torch.tensor([7, 8, 7]).cuda(), top=2)
        assert (out.logprob[[0, 2]] <= 0).all() and (out.logprob[[0, 2]] >= -2.0 ** -23).all()
        assert abs(float(out.logprob[1]) + 50.0) <= 2.0 ** -22 * 50
        assert (out.entropy >= 0).all() and (out.entropy <= 2.0 ** -22).all()
        assert (out.top_logprobs <= 0).all() and out.top_ids[0].tolist() == [7, 0]


@pytest.mark.gpu
def test_targets_outside_and_ignored():
    x, t = make(6, 300, torch.bfloat16)
    t[1], t[2], t[3], t[4] = -100, 300, -1, 7
    out = check(x, t, 3)
    assert out.logprob[1] == 0 and torch.isnan(out.logprob[2:4]).all()
    check(x, t, 0, ignore_index=7)
    check(x, t.to(torch.int32), 0)


@pytest.mark.gpu
def test_strides_shapes_and_alignment():
    """Row strides, rows off a 16-byte boundary, expanded rows, leading dimensions, none."""
    for dtype in (torch.float32, torch.bfloat16):
        base, _ = make(8, 1003, dtype)
        t = torch.randint(0, 990, (8,))
        for x in (base[:, 5:1000], base[::2, :1000], base[:, ::2], base[:1].expand(8, 1003),
                  base.t().contiguous().t()):
            tt = (t % x.shape[1])[:x.shape[0]]
            lp, H, ids, _ = ref.forward(x, tt, 5)
            mine = x.untyped_storage().data_ptr() == base.untyped_storage().data_ptr()
            src = base if mine else x.t()     # the same strides on the GPU
            xg = torch.as_strided(src.cuda().contiguous(), x.shape, x.stride(), x.storage_offset())
            out = token_logprobs(xg, tt.cuda(), top=5)
            near(out.logprob, lp, "logprob")
            near(out.entropy, H, "entropy", E_H)
            assert torch.equal(out.top_ids.cpu(), ids)
        out = token_logprobs(base.cuda().view(2, 4, 1003), t.cuda().view(2, 4), top=2)
        assert out.logprob.shape == (2, 4) and out.top_ids.shape == (2, 4, 2)
        one = token_logprobs(base[0].cuda(), t[0].cuda(), top=2)
        assert torch.equal(one.logprob, out.logprob[0, 0]) and one.top_ids.shape == (2,)
        assert token_logprobs(base[:0].cuda(), t[:0].cuda(), top=2).top_ids.shape == (0, 2)


# --- gradient ------------------------------------------------------------------
def check_grad(x, t, top=0, use=(1, 1, 1), view=None, ignore_index=-100):
    rows, V = x.shape
    g = torch.Generator().manual_seed(7)
    up = [torch.randn(rows, generator=g) if use[0] else None, torch.randn(rows, generator=g) if use[1] else None,
          torch.randn(rows, top, generator=g) if use[2] and top else None]
    leaf = x.cuda().requires_grad_(True)
    out = token_logprobs(leaf if view is None else view(leaf), t.cuda(), top=top, ignore_index=ignore_index)
    pairs = [(o, u.cuda()) for o, u in zip((out.logprob, out.entropy, out.top_logprobs), up) if u is not None]
    (dx,) = torch.autograd.grad([p[0] for p in pairs], leaf, [p[1] for p in pairs])
    want = ref.backward(x if view is None else view(x), t, *up, top=top, ignore_index=ignore_index)
    if view is not None:
        z = x.double().clone().requires_grad_(True)
        (want,) = torch.autograd.grad(view(z), z, want)
    assert dx.dtype == x.dtype
    size = sum(float(u.abs().max()) * max(1, u.shape[-1] if u.dim() > 1 else 1) for u in up if u is not None)
    half = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -24
    z = x.double() if view is None else view(x.double())
    _, _, ids, _ = ref.forward(z, t, top, ignore_index)
    own = torch.zeros_like(z).scatter_(1, t.clamp(0, z.shape[1] - 1)[:, None], 1.0).scatter_(1, ids, 1.0)
    tol = E_P * size * torch.softmax(z, 1) + 4 * 2.0 ** -24 * size * own
    if view is not None:      # outside the view nothing is touched
        w = torch.zeros_like(x.double())
        view(w).copy_(tol)
        tol = w
    err = (dx.double().cpu() - want).abs()
    assert (err <= tol + half * want.abs() + 1e-38).all(), float((err - tol - half * want.abs()).max())
    return dx


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,top", [(1, 1), (9, 3), (1000, 20), (8192, 0), (8199, 64), (32003, 5), (70000, 0)])
def test_gradient(V, top, dtype):
    x, t = make(4, V, dtype, seed=V, banned=0.05 if V > 9 else 0.0)
    t[1] = -100
    check_grad(x, t, top)
    check_grad(x, t, top, use=(1, 0, 0))
    check_grad(x, t, top, use=(0, 1, 0))
    if top:
        check_grad(x, t, top, use=(0, 0, 1))


@pytest.mark.gpu
def test_gradient_of_views():
    """Rows with a stride, off a boundary, and one row used for all (its gradient
    is the sum over its uses)."""
    for dtype in (torch.float32, torch.bfloat16):
        x, _ = make(4, 203, dtype)
        t = torch.randint(0, 100, (4,))
        check_grad(x, t, 3, view=lambda z: z[:, 3:200])
        check_grad(x, t, 0, view=lambda z: z[:, ::2])
    x, _ = make(1, 64, torch.float32)
    t = torch.randint(0, 64, (4,))
    leaf = x.cuda().requires_grad_(True)
    token_logprobs(leaf.expand(4, 64), t.cuda()).logprob.sum().backward()
    want = ref.backward(x.expand(4, 64), t, torch.ones(4)).sum(0, keepdim=True)
    near(leaf.grad, want, "dlogits", tol=4 * E_P * torch.softmax(x.double(), 1).max() + 16 * 2.0 ** -24)


@pytest.mark.gpu
def test_targets_outside_give_no_number_and_double_backward_is_refused():
    x, t = make(3, 40, torch.float32)
    t[1] = 40
    leaf = x.cuda().requires_grad_(True)
    out = token_logprobs(leaf, t.cuda())
    (d,) = torch.autograd.grad(out.logprob.sum(), leaf, retain_graph=True)
    assert torch.isnan(d[1]).all() and torch.isfinite(d[[0, 2]]).all()
    (d,) = torch.autograd.grad(out.logprob.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), leaf)
    assert not token_logprobs(x.cuda(), t.cuda()).logprob.requires_grad
    out = token_logprobs(leaf, t.cuda())
    with pytest.raises(RuntimeError):     # batched upstream gradients
        torch.autograd.grad(out.logprob, leaf, torch.eye(3, device="cuda"), is_grads_batched=True)
    import torch.autograd.forward_ad as fwd
    with pytest.raises(RuntimeError), fwd.dual_level():
        token_logprobs(fwd.make_dual(x.cuda(), torch.ones_like(x).cuda()), t.cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ignored_rows_take_no_gradient_whatever_they_hold(dtype):
    """Padded places may hold anything: logprob 0 and a gradient of zeros, also where
    other rows' entropy and alternatives are asked for."""
    x, t = make(4, 203, dtype)
    x[1, 7], x[2] = math.nan, -math.inf
    t[1:3] = -100
    leaf = x.cuda().requires_grad_(True)
    out = token_logprobs(leaf, t.cuda(), top=3)
    assert out.logprob[1:3].tolist() == [0.0, 0.0]
    ones = torch.tensor([1.0, 0.0, 0.0, 1.0], device="cuda")
    for outs, gs in (((out.logprob,), (torch.ones(4, device="cuda"),)),
                     ((out.logprob, out.entropy, out.top_logprobs), (ones, ones, ones[:, None].expand(4, 3)))):
        (d,) = torch.autograd.grad(outs, leaf, gs, retain_graph=True)
        assert not d[1:3].any() and torch.isfinite(d).all() and d[0].any()


@pytest.mark.gpu
def test_graph_of_forward_and_backward():
    """Captured and replayed over new logits, with eager work between."""
    V, rows = 5003, 6
    xs = [make(rows, V, torch.bfloat16, seed=i)[0].cuda() for i in range(5)]
    t = torch.randint(0, V, (rows,), device="cuda")
    g = torch.randn(rows, device="cuda")

    def step(leaf):
        out = token_logprobs(leaf, t, top=4)
        return (*out, *torch.autograd.grad((out.logprob, out.entropy), leaf, (g, g)))
    want = [[o.clone() for o in step(x.clone().requires_grad_(True))] for x in xs]
    leaf = xs[0].clone().requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaf)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(leaf)
    for x, w in zip(xs, want):
        with torch.no_grad():
            leaf.copy_(x)
        graph.replay()
        torch.randn(64, 64, device="cuda").sum()
        for a, b in zip(got, w):
            assert torch.equal(a, b)


# --- finite logits of any size ---------------------------------------------------
def shifted(x):
    """x in float64 less each row's maximum: the same distribution.  Beside 1e30 the
    logarithm of a sum is below float64's own step."""
    x = x.double()
    return x - x.amax(1, keepdim=True)


def near_shifted(out, x, t, top):
    """The results for x against those for shifted(x), rounded to fp32 (differences
    of two logits may pass its range)."""
    lp, H, ids, tl = ref.forward(shifted(x), t, top)
    near(out.logprob, lp.float(), "logprob")
    near(out.entropy, H, "entropy", E_H)
    assert torch.equal(out.top_ids.cpu(), ids)
    near(out.top_logprobs, tl.float(), "top_logprobs")


def masked_rows(V, dtype, mask):
    """Rows where all but ten tokens hold `mask`, the ten first, last, in the
    middle and spread over the row, and one where every token does."""
    low = torch.finfo(dtype).min if mask == "lowest" else mask
    x = torch.full((5, V), low, dtype=torch.float64)
    g = torch.Generator().manual_seed(V)
    keep = [torch.arange(10), torch.arange(V - 10, V), torch.arange(V // 2, V // 2 + 10),
            torch.randperm(V, generator=g)[:10]]
    for r, j in enumerate(keep):
        x[r, j] = torch.randn(10, generator=g).double() * 3
    t = torch.tensor([int(j[3]) for j in keep] + [V // 3])
    return x.to(dtype), t


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-1e10, -1e30, "lowest"])
@pytest.mark.parametrize("V,rows,top", [(5000, 1, 0), (5000, 600, 20), (40000, 1, 20), (40000, 600, 0),
                                        (40000, 600, 20), (131072, 1, 0), (131072, 1, 20), (131072, 600, 20)])
def test_finite_masks(V, rows, top, mask, dtype):
    """Masks of a large finite value, over whole pieces of a row and over all of it
    (then the row is uniform): what -inf in their place gives, and -log V."""
    x, t = masked_rows(V, dtype, mask)
    if rows == 1:
        for r in range(5):
            near_shifted(token_logprobs(x[r:r + 1].cuda(), t[r:r + 1].cuda(), top=top), x[r:r + 1], t[r:r + 1], top)
        return
    of = torch.arange(rows) % 5
    out = token_logprobs(x.cuda()[of.cuda()], t[of].cuda(), top=top)
    for a, name in zip(out, out._fields):
        want = a[:5]
        for i in range(5, rows, 5):   # rows stand at different places to a 16-byte boundary
            if name == "top_ids":
                assert torch.equal(a[i:i + 5], want)
            else:
                near(a[i:i + 5], want.cpu(), name, 2 * (E_H if name == "entropy" else E_LP))
    near_shifted(type(out)(*(a[:5] for a in out)), x, t, top)


def grad_near(x, t, top):
    g = torch.Generator().manual_seed(7)
    rows = x.shape[0]
    up = [torch.randn(rows, generator=g), torch.randn(rows, generator=g),
          torch.randn(rows, top, generator=g) if top else None]
    leaf = x.cuda().requires_grad_(True)
    out = token_logprobs(leaf, t.cuda(), top=top)
    pairs = [(o, u.cuda()) for o, u in zip((out.logprob, out.entropy, out.top_logprobs), up) if u is not None]
    (dx,) = torch.autograd.grad([p[0] for p in pairs], leaf, [p[1] for p in pairs])
    z = shifted(x)
    want = ref.backward(z, t, *up, top=top)
    size = sum(float(u.abs().max()) * (u.shape[-1] if u.dim() > 1 else 1) for u in up if u is not None)
    half = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -24
    own = torch.zeros_like(z).scatter_(1, t[:, None], 1.0).scatter_(1, ref.forward(z, t, top)[2], 1.0)
    tol = E_P * size * torch.softmax(z, 1) + 4 * 2.0 ** -24 * size * own
    err = (dx.double().cpu() - want).abs()
    assert (err <= tol + half * want.abs() + 1e-38).all(), float((err - tol - half * want.abs()).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [-1e10, -1e30, "lowest"])
@pytest.mark.parametrize("V,top", [(5000, 0), (40000, 20), (131072, 3)])
def test_gradient_of_finite_masks(V, top, mask, dtype):
    grad_near(*masked_rows(V, dtype, mask), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [500, 70001])
def test_logits_of_any_finite_size(V, dtype):
    """Three equal largest logits of any size, in different pieces where the row
    has several: each has probability 1 / 3, the others none.  And logits from
    one end of the type's range to the other."""
    sizes = [1e7, 1e8, 5e9, -5e9, 1e20, 1e30, -1e30, 3e38, -3e38]
    x = torch.tensor(sizes, dtype=torch.float64)[:, None].expand(-1, V).clone()
    x -= 0.125 * x.abs()
    for j in (7, V // 2, V - 1):
        x[:, j] = torch.tensor(sizes, dtype=torch.float64)
    x = x.to(dtype)
    t = torch.full((len(sizes),), 7)
    t[1::2] = 8
    for n in (1, len(sizes)):
        near_shifted(token_logprobs(x[:n].cuda(), t[:n].cuda(), top=2), x[:n], t[:n], 2)
    grad_near(x, t, 2)
    ends = torch.full((2, V), -3e38, dtype=torch.float64)
    ends[:, V - 3] = 3e38
    ends, t = ends.to(dtype), torch.tensor([V - 3, 0])
    near_shifted(token_logprobs(ends.cuda(), t.cuda(), top=1), ends, t, 1)


@pytest.mark.gpu
def test_distributions_far_from_zero():
    """Rows moved by a number that keeps every difference exact: the distribution of
    the row around zero."""
    g = torch.Generator().manual_seed(3)
    near0 = torch.randint(-64, 65, (4, 33000), generator=g).double() / 8
    t = torch.randint(0, 33000, (4,), generator=g)
    for by in (2.0 ** 17, -2.0 ** 17, 2.0 ** 20 - 8):     # steps of 2^-7 to 2^-4 there
        x = (near0 + by).float()
        assert torch.equal(x.double() - by, near0)
        near_shifted(token_logprobs(x.cuda(), t.cuda(), top=5), x, t, 5)
        grad_near(x, t, 5)
