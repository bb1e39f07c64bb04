"""8-bit linear layers and the rows that enter them (ops/fp8.py) against
oracle/fp8.py in float64.

Rows: quantize_rows_fp8 and rms_norm_fp8 round a value known to some 2^-45 of itself
(products of two fp32 or bf16 numbers are taken with their remainder, the norm's
in fp64 where fp32 may not do) to odd and then to e4m3, so the codes and scales are the
oracle's own, bit for bit; the inputs here are random, no exact norm lies within
2^-40 of a tie.  silu_mul_fp8's value has seven fp32 roundings (e^-c 1 ulp and the
remainder's product, the sum, a reciprocal with one correction, two products): it
is off by at most 8 2^-24 of itself, so a code by half a step and that.

Products: codes and scales are exact.  The matrix cores take the products of 8
columns, 8 i to 8 i + 7, together: aligned to the largest of their exponent sums and cut
below 2^-13 of it (a product 2^-13 of the largest counts, one of 2^-14 does not), so
each of the other seven is off by less than 2^-13 of the largest, 7 2^-13 of the
magnitudes' sum A over all groups at most.  K / 8 such sums are added in fp32, each
addition off by at most 2^-23 of A, the waves' sums by eight more, and the result is
rounded once to bf16, 2^-8 of it at most.  Where all products of a group lie within
2^13 of each other and no sum passes 2^24 of the last bit, nothing is lost but that
last rounding: whole numbers give the oracle's own result.
"""
import math

import pytest
import torch

from oracle import fp8 as ref
from selective_attention.ops import (Fp8Rows, dequantize_fp8, fp8_linear, fp8_linear_multi, pack_fp8,
                                     quantize_fp8, quantize_rows_fp8, rms_norm_fp8, silu_mul_fp8)

E4, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def rand(*shape, seed=0, dtype=torch.bfloat16, big=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g)
    if big and len(shape) > 1:   # columns of unlike size
        x = x * torch.exp(2.0 * torch.randn(shape[-1], generator=g))
    return x.to(dtype)


def make_rows(M, K, seed=0):
    """Rows in 8 bits made by the oracle, on the CPU."""
    codes, scales = ref.rows(rand(M, K, seed=seed))
    return Fp8Rows(codes.to(E4), (torch.log2(scales) + 127).to(torch.uint8).view(E8), K)


def on(r: Fp8Rows) -> Fp8Rows:
    return Fp8Rows(r.codes.cuda(), r.scales.cuda(), r.features)


def same_rows(r: Fp8Rows, v: torch.Tensor):
    codes, scales = ref.rows(v.reshape(-1, v.shape[-1]))
    assert r.shape == v.shape
    assert r.codes.dtype == E4 and r.scales.dtype == E8
    assert torch.equal(r.scales.cpu().double().reshape(scales.shape), scales)
    got = r.codes.cpu().double().reshape(codes.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(codes))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(codes))


def check_linear(y, rows, packed, scales, N, bias=None):
    K = rows.codes.shape[-1]
    w = torch.nn.functional.pad(ref.weight(packed, scales, N, 128 * packed.shape[1]), (0, 0))
    want, A = ref.linear(ref.values(rows.codes.reshape(-1, K), rows.scales.reshape(-1, rows.scales.shape[-1]), K),
                         w, bias)
    tol = 7 * 2.0 ** -13 * A + (K / 8 + 8) * 2.0 ** -23 * A + 2.0 ** -8 * want.abs() + 2.0 ** -133
    err = (y.double().cpu().reshape(want.shape) - want).abs()
    assert (err <= tol).all(), (float((err - tol).max()), float(err.max()))


# --- layout and rounding, on the CPU ---------------------------------------------
@pytest.mark.parametrize("N,K", [(16, 128), (33, 100), (1, 1), (130, 300)])
def test_pack_keeps_codes_and_scales(N, K):
    g = torch.Generator().manual_seed(3)
    codes = torch.randn(N, K, generator=g).to(E4)
    nb, kb = (N + 127) // 128, (K + 127) // 128
    e = torch.randint(-126, 128, (nb, kb), generator=g)
    byte = (e + 127).to(torch.uint8)
    for scales in (byte, byte.view(E8), torch.exp2(e.double()), torch.exp2(e.float())):
        packed, s = pack_fp8(codes, scales)
        assert packed.shape == ((N + 15) // 16, kb, 8, 16, 16) and s.shape == (nb, (kb + 3) // 4 * 4)
        assert torch.equal(ref.unpack(packed, N, K), codes.double())
        assert torch.equal(s.view(torch.uint8)[:, :kb], byte)
        assert (s.view(torch.uint8)[:, kb:] == 127).all()
    whole = ref.unpack(packed, packed.shape[0] * 16, kb * 128)
    assert not whole[N:].any() and not whole[:, K:].any()


@pytest.mark.parametrize("N,K", [(128, 128), (200, 300), (5, 129)])
def test_quantize_rounds_to_the_nearest_code(N, K):
    w = rand(N, K, seed=1, dtype=torch.float32)
    w[3] = 0.0
    packed, scales = quantize_fp8(w)
    s = torch.exp2(scales.view(torch.uint8).double() - 127)[torch.arange(N) // 128][:, torch.arange(K) // 128]
    assert torch.equal(ref.unpack(packed, N, K), ref.e4m3(w.double() / s))
    for i in range(0, N, 128):
        for j in range(0, K, 128):
            top = w[i:i + 128, j:j + 128].abs().max().double()
            assert ref.scale_of(top[None])[0] == s[i, j]


def test_quantize_borders_and_zeros():
    """448 2^e keeps the scale, the next number doubles it; a block of zeros has 1."""
    w = torch.zeros(128, 512)
    w[0, 0], w[0, 128], w[0, 256] = 448 * 2.0 ** -9, math.nextafter(448.0, 1e9), 1e-45
    w[0, 128] = torch.nextafter(torch.tensor(448.0), torch.tensor(1e9))
    byte = quantize_fp8(w)[1].view(torch.uint8)
    assert byte.tolist() == [[127 - 9, 128, 1, 127]]


@pytest.mark.parametrize("what", ["type", "nan", "scales", "power", "range", "zero", "int", "empty"])
def test_pack_refuses(what):
    codes, scales = torch.zeros(130, 128).to(E4), torch.ones(2, 1)
    if what == "type":
        codes = codes.view(torch.uint8)
    elif what == "nan":
        codes.view(torch.uint8)[7, 7] = 0x7f
    elif what == "scales":
        scales = scales[:1]
    elif what == "power":
        scales[1] = 0.75
    elif what == "range":
        scales = torch.full((2, 1), 255, dtype=torch.uint8)
    elif what == "zero":
        scales[0] = 0.0
    elif what == "int":
        scales = scales.int()
    elif what == "empty":
        codes = codes[:0]
    with pytest.raises((ValueError, TypeError)):
        pack_fp8(codes, scales)


@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_quantize_refuses_what_is_not_finite(value):
    w = torch.zeros(4, 4)
    w[1, 2] = value
    with pytest.raises(ValueError):
        quantize_fp8(w)
    with pytest.raises(ValueError):
        quantize_fp8(w[:0])


@pytest.mark.parametrize("what", ["dtype", "features", "outs", "packed", "layout", "scales", "scale type", "bias",
                                  "bias type", "xscale", "rows xscale", "codes", "rows scales", "count", "cpu",
                                  "rows cpu", "no features"])
def test_linear_refuses(what):
    packed, scales = quantize_fp8(rand(32, 256, dtype=torch.float32))
    x, kw = torch.zeros(2, 256, dtype=torch.bfloat16), dict(out_features=32)
    if what == "dtype":
        x = x.float()
    elif what == "features":
        x = x[:, :128]
    elif what == "outs":
        kw = dict(out_features=48)
    elif what == "packed":
        packed = packed.view(torch.int8)
    elif what == "layout":
        packed = packed.transpose(2, 3)
    elif what == "scales":
        scales = scales[:, :2]
    elif what == "scale type":
        scales = scales.float()
    elif what == "bias":
        kw["bias"] = torch.zeros(31, dtype=torch.bfloat16)
    elif what == "bias type":
        kw["bias"] = torch.zeros(32)
    elif what == "xscale":
        kw["xscale"] = x[:1]
    elif what == "rows xscale":
        x, kw["xscale"] = make_rows(2, 256), x
    elif what == "codes":
        x = Fp8Rows(make_rows(2, 256).codes.float(), make_rows(2, 256).scales)
    elif what == "rows scales":
        x = Fp8Rows(make_rows(2, 256).codes, make_rows(2, 256).scales[:1])
    elif what == "rows cpu":
        x = make_rows(2, 256)
    elif what == "no features":
        x = x[:, :0]
    with pytest.raises((ValueError, TypeError)):
        if what == "count":
            fp8_linear_multi(x, [(packed, scales)] * 5, [None] * 5, [32] * 5)
        else:
            fp8_linear(x, packed, scales, **kw)


def test_rows_of_wrong_shapes():
    """Codes and scales whose leading sizes or lengths do not belong together."""
    packed, scales = quantize_fp8(rand(32, 256, dtype=torch.float32))
    r = make_rows(6, 256)
    c, s = r.codes, r.scales
    for codes, sc in ((c, s[0]), (c[0], s), (c[0], s[0, 0]), (c[0, 0], s), (c.view(2, 3, 256), s), (c, s.view(2, 3, 4)),
                      (c.view(2, 3, 256), s.view(3, 2, 4)), (c, s[:, :2]), (c[:, :128], s)):
        with pytest.raises(ValueError):
            fp8_linear(Fp8Rows(codes, sc, 256), packed, scales, out_features=32)


@pytest.mark.gpu
def test_tensors_elsewhere_are_refused():
    """One tensor of a call on the CPU: told before any launch."""
    packed, scales = weight(32, 256)
    x, b = rand(2, 256), rand(32, big=False)
    r = make_rows(2, 256)
    w = torch.zeros(256)
    for i in range(4):
        at = [t.cuda() if i != j else t for j, t in enumerate((x, packed, scales, b))]
        with pytest.raises(ValueError):
            fp8_linear(at[0], *at[1:], out_features=32)
        with pytest.raises(ValueError):
            fp8_linear(Fp8Rows(r.codes if i == 0 else r.codes.cuda(), r.scales.cuda(), 256), *at[1:], out_features=32)
    calls = (lambda: fp8_linear(Fp8Rows(r.codes.cuda(), r.scales, 256), packed.cuda(), scales.cuda()),
             lambda: fp8_linear(x.cuda(), packed.cuda(), scales.cuda(), xscale=x), lambda: quantize_rows_fp8(x.cuda(), x),
             lambda: silu_mul_fp8(x, x.cuda()), lambda: rms_norm_fp8(x.cuda(), w), lambda: rms_norm_fp8(x, w.cuda()),
             lambda: rms_norm_fp8(x.cuda(), w.cuda(), residual=x), lambda: dequantize_fp8(packed.cuda(), scales),
             lambda: dequantize_fp8(packed, scales))
    for call in calls:
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("what", ["norm weight", "norm residual", "norm eps", "norm dtype", "norm wide", "norm cpu",
                                  "norm grad", "silu dtype", "silu shape", "silu grad", "rows dtype", "rows gate",
                                  "rows grad", "rows none", "rows cpu"])
def test_rows_refuse(what):
    x, w = torch.zeros(2, 8), torch.zeros(8)
    h = x.to(torch.bfloat16)
    calls = {
        "norm weight": lambda: rms_norm_fp8(x, w[:7]), "norm residual": lambda: rms_norm_fp8(x, w, residual=h),
        "norm eps": lambda: rms_norm_fp8(x, w, -1.0), "norm dtype": lambda: rms_norm_fp8(x.double().cuda() if torch.cuda.is_available() else x.int(), w),
        "norm wide": lambda: rms_norm_fp8(torch.zeros(1, 65537), torch.zeros(65537)),
        "norm cpu": lambda: rms_norm_fp8(x, w), "norm grad": lambda: rms_norm_fp8(x, w.requires_grad_()),
        "silu dtype": lambda: silu_mul_fp8(x, x), "silu shape": lambda: silu_mul_fp8(h, h[:1]),
        "silu grad": lambda: silu_mul_fp8(h.requires_grad_(), h), "rows dtype": lambda: quantize_rows_fp8(x.half()),
        "rows gate": lambda: quantize_rows_fp8(x, h), "rows grad": lambda: quantize_rows_fp8(x.requires_grad_()),
        "rows none": lambda: quantize_rows_fp8(x[:, :0]), "rows cpu": lambda: quantize_rows_fp8(x),
    }
    with pytest.raises((ValueError, TypeError, RuntimeError)):
        calls[what]()


def off_by(t, n):
    """t's values n bytes behind a 16-byte boundary."""
    raw = torch.empty(t.numel() * t.element_size() + 16 + n, dtype=torch.uint8)
    at = -raw.data_ptr() % 16 + n
    out = raw[at:at + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
    return out.copy_(t)


# what is wrong, and what the call says of it; "" names nothing: the call is whole, and
# only a device is missing
LINEAR_SAYS = {
    "": "no CPU path", "bias given": "no CPU path", "gated": "no CPU path", "rows": "no CPU path", "one row": "no CPU path",
    "uint8 scales": "no CPU path",
    "dtype": "x must be bfloat16", "features": "packed must be", "more features": "packed must be", "outs": "packed must be",
    "no outs": "packed must be", "packed type": "packed must be", "packed layout": "packed must be",
    "packed flat": "packed must be", "packed strides": "must be contiguous on 16- and 4-byte", "packed place": "must be contiguous on 16- and 4-byte",
    "scales": "scales must be", "scales rows": "scales must be", "scale type": "scales must be .* or its bytes",
    "scales strides": "must be contiguous on 16- and 4-byte", "scales place": "must be contiguous on 16- and 4-byte",
    "bias": r"\[bias\] Shape mismatch", "bias type": "bias must be bfloat16", "xscale": "xscale must be", "xscale type": "xscale must be",
    "rows xscale": "xscale goes with x as a tensor", "codes": "codes must be", "codes short": "codes must be", "codes long": "codes must be",
    "rows scales": "scales must be .* beside codes", "rows scales short": "scales must be .* beside codes",
    "rows scales type": "scales must be .* beside codes", "no features": "x must have features", "no x": "x must have features",
    "none": "1..4 weights", "five": "1..4 weights", "biases": "1..4 weights", "sizes": "1..4 weights", "second": "packed must be",
}


@pytest.mark.parametrize("what", LINEAR_SAYS)
def test_linear_says_what_is_wrong(what):
    """Each check by its own words: without it the call would get as far as its device."""
    packed, scales = quantize_fp8(rand(160, 256, dtype=torch.float32))
    x, bias, xscale, N = torch.zeros(3, 256, dtype=torch.bfloat16), None, None, 160
    r = make_rows(3, 256)
    if what == "bias given":
        bias = torch.zeros(160, dtype=torch.bfloat16)
    elif what == "gated":
        xscale = x
    elif what == "rows":
        x = r
    elif what == "one row":
        x = Fp8Rows(r.codes[0], r.scales[0])
    elif what == "uint8 scales":
        x, scales = Fp8Rows(r.codes, r.scales.view(torch.uint8)), scales.view(torch.uint8)
    elif what == "dtype":
        x = x.float()
    elif what == "features":
        x = x[:, :128]
    elif what == "more features":
        x = torch.zeros(3, 257, dtype=torch.bfloat16)
    elif what == "outs":
        N = 161
    elif what == "no outs":
        packed, scales, N = packed[:0], scales[:0], 0
    elif what == "packed type":
        packed = packed.view(torch.int8)
    elif what == "packed layout":
        packed = packed.transpose(2, 3)
    elif what == "packed flat":
        packed = packed.flatten(3)
    elif what == "packed strides":
        packed = packed.transpose(3, 4)
    elif what == "packed place":
        packed = off_by(packed, 8)
    elif what == "scales":
        scales = scales[:, :2]
    elif what == "scales rows":
        scales = scales[:1]
    elif what == "scale type":
        scales = scales.float()
    elif what == "scales strides":
        scales = scales.view(torch.uint8).t().contiguous().t()
    elif what == "scales place":
        scales = off_by(scales.view(torch.uint8), 2)
    elif what == "bias":
        bias = torch.zeros(159, dtype=torch.bfloat16)
    elif what == "bias type":
        bias = torch.zeros(160)
    elif what == "xscale":
        xscale = x[:1]
    elif what == "xscale type":
        xscale = x.float()
    elif what == "rows xscale":
        x, xscale = r, x
    elif what == "codes":
        x = Fp8Rows(r.codes.float(), r.scales)
    elif what == "codes short":
        x = Fp8Rows(r.codes[:, :128], r.scales, 256)
    elif what == "codes long":
        x = Fp8Rows(r.codes, r.scales, 128)
    elif what == "rows scales":
        x = Fp8Rows(r.codes, r.scales[:1])
    elif what == "rows scales short":
        x = Fp8Rows(r.codes, r.scales[:, :2])
    elif what == "rows scales type":
        x = Fp8Rows(r.codes, r.scales.float())
    elif what == "no features":
        x = x[:, :0]
    elif what == "no x":
        x = x[0, 0]
    ws, bs, sizes = [(packed, scales)], [bias], [N]
    if what == "none":
        ws, bs, sizes = [], [], []
    elif what == "five":
        ws, bs, sizes = ws * 5, bs * 5, sizes * 5
    elif what == "biases":
        bs = []
    elif what == "sizes":
        sizes = sizes * 2
    elif what == "second":
        ws, bs, sizes = ws * 2, bs * 2, [160, 176]
    calls = [lambda: fp8_linear_multi(x, ws, bs, sizes, xscale)]
    if len(ws) == len(bs) == len(sizes) == 1:
        calls.append(lambda: fp8_linear(x, packed, scales, bias, N, xscale))
    for call in calls:
        with pytest.raises((ValueError, TypeError), match=LINEAR_SAYS[what]):
            call()


def test_rows_that_do_not_belong_together_are_named():
    """Codes and scales of different leading sizes, each by the words of its own check."""
    packed, scales = quantize_fp8(rand(32, 256, dtype=torch.float32))
    r = make_rows(6, 256)
    c, s = r.codes, r.scales
    for codes, sc in ((c, s[0]), (c[0], s), (c[0], s[0, 0]), (c, s.view(2, 3, 4)), (c.view(2, 3, 256), s),
                      (c.view(2, 3, 256), s.view(3, 2, 4)), (c, s[:, :2]), (c, s[:5]), (c[:5], s)):
        with pytest.raises(ValueError, match="beside codes"):
            fp8_linear(Fp8Rows(codes, sc, 256), packed, scales, out_features=32)
    for codes in (c[:, :128], c[0, 0], c.view(6, 2, 128)):
        with pytest.raises(ValueError, match="codes must be"):
            fp8_linear(Fp8Rows(codes, s, 256), packed, scales, out_features=32)
    with pytest.raises(ValueError, match="no CPU path"):
        fp8_linear(Fp8Rows(c, s, 256), packed, scales, out_features=32)


def test_rows_say_what_is_wrong():
    x, w = torch.zeros(2, 8), torch.zeros(8)
    h = x.to(torch.bfloat16)
    g, hg = x.clone().requires_grad_(), h.clone().requires_grad_()
    wide = torch.zeros(1, 65537)
    says = [
        ("no CPU path", lambda: quantize_rows_fp8(x)), ("no CPU path", lambda: quantize_rows_fp8(h, h)),
        ("no CPU path", lambda: silu_mul_fp8(h, h)), ("no CPU path", lambda: rms_norm_fp8(x, w)),
        ("no CPU path", lambda: rms_norm_fp8(h, w, 0.0, h)), ("no CPU path", lambda: rms_norm_fp8(wide[:, 1:], wide[0, 1:])),
        ("no CPU path", lambda: rms_norm_fp8(x, w.to(torch.bfloat16))),
        ("x must have features", lambda: quantize_rows_fp8(x[:, :0])), ("x must have features", lambda: quantize_rows_fp8(x[0, 0])),
        ("x must have features", lambda: silu_mul_fp8(h[:, :0], h[:, :0])), ("x must have features", lambda: rms_norm_fp8(x[:, :0], w[:0])),
        ("xscale must be", lambda: quantize_rows_fp8(x, h)), ("xscale must be", lambda: quantize_rows_fp8(x, x[:1])),
        ("c must be", lambda: silu_mul_fp8(h, h[:1])), ("c must be", lambda: silu_mul_fp8(h, x)),
        ("a and c must be bfloat16", lambda: silu_mul_fp8(x, x)),
        ("residual must be", lambda: rms_norm_fp8(x, w, residual=h)), ("residual must be", lambda: rms_norm_fp8(x, w, residual=x[:1])),
        (r"\[weight\] Shape mismatch", lambda: rms_norm_fp8(x, w[:7])), (r"\[weight\] Shape mismatch", lambda: rms_norm_fp8(x, w[None])),
        ("at most 65536", lambda: rms_norm_fp8(wide, wide[0])),
        ("must not be negative", lambda: rms_norm_fp8(x, w, -1e-9)), ("must not be negative", lambda: rms_norm_fp8(x, w, math.nan)),
        ("codes have no gradient", lambda: quantize_rows_fp8(g)), ("codes have no gradient", lambda: quantize_rows_fp8(x, g)),
        ("codes have no gradient", lambda: silu_mul_fp8(hg, h)), ("codes have no gradient", lambda: silu_mul_fp8(h, hg)),
        ("codes have no gradient", lambda: rms_norm_fp8(g, w)), ("codes have no gradient", lambda: rms_norm_fp8(x, g[0])),
        ("codes have no gradient", lambda: rms_norm_fp8(x, w, residual=g)),
    ]
    for words, call in says:
        with pytest.raises((ValueError, TypeError, RuntimeError), match=words):
            call()
    with torch.no_grad():
        for call in (lambda: quantize_rows_fp8(g), lambda: silu_mul_fp8(hg, hg), lambda: rms_norm_fp8(g, g[0], residual=g)):
            with pytest.raises(ValueError, match="no CPU path"):
                call()


def test_weights_say_what_is_wrong():
    codes, ones = torch.zeros(130, 128).to(E4), torch.ones(2, 1)
    w = torch.zeros(4, 4)
    packed, scales = quantize_fp8(torch.ones(32, 256))
    x = torch.zeros(3, 256, dtype=torch.bfloat16)
    bad = w.clone()
    bad[1, 2] = math.inf
    says = [
        (r"\[codes\] Dim mismatch", lambda: pack_fp8(codes[0], ones)), ("pack_fp8: empty weight", lambda: pack_fp8(codes[:0], ones[:0])),
        ("pack_fp8: empty weight", lambda: pack_fp8(codes[:, :0], ones[:, :0])),
        ("codes must be", lambda: pack_fp8(codes.float(), ones)), (r"\[scales\] Shape mismatch", lambda: pack_fp8(codes, ones[:1])),
        ("codes hold NaN", lambda: pack_fp8(torch.full((130, 128), math.nan).to(E4), ones)),
        ("powers of two", lambda: pack_fp8(codes, 3 * ones)), ("powers of two", lambda: pack_fp8(codes, -ones)),
        ("powers of two", lambda: pack_fp8(codes, 2.0 ** -127 * ones.double())), ("floating or e8m0", lambda: pack_fp8(codes, ones.long())),
        (r"scales must be 2\^-126", lambda: pack_fp8(codes, torch.zeros(2, 1, dtype=torch.uint8))),
        (r"\[weight\] Dim mismatch", lambda: quantize_fp8(w[0])), ("quantize_fp8: empty weight", lambda: quantize_fp8(w[:0])),
        ("quantize_fp8: empty weight", lambda: quantize_fp8(w[:, :0])), ("quantize_fp8: the weight holds", lambda: quantize_fp8(bad)),
        ("packed must be", lambda: dequantize_fp8(packed.flatten(3), scales)), ("packed must be", lambda: dequantize_fp8(packed, scales, 33, 256)),
        ("packed must be", lambda: dequantize_fp8(packed, scales, 32, 257)), ("scales must be", lambda: dequantize_fp8(packed, scales[:, :1])),
        ("no CPU path", lambda: dequantize_fp8(packed, scales)), ("no CPU path", lambda: dequantize_fp8(packed, scales, 17, 129)),
        ("packed must be", lambda: dequantize_fp8(packed.flatten()[0], scales)),
        ("packed must be", lambda: fp8_linear(x, packed.flatten()[0], scales)),
        ("packed must be", lambda: fp8_linear(x, packed.flatten(3), scales)), ("no CPU path", lambda: fp8_linear(x, packed, scales)),
    ]
    for words, call in says:
        with pytest.raises((ValueError, TypeError), match=words):
            call()


@pytest.mark.gpu
def test_rows_of_other_types_are_refused():
    x, w = torch.zeros(2, 8, device="cuda"), torch.zeros(8, device="cuda")
    for t in (torch.float64, torch.float16, torch.int32):
        y = x.to(t)
        for call in (lambda: quantize_rows_fp8(y), lambda: quantize_rows_fp8(y, y), lambda: rms_norm_fp8(y, w),
                     lambda: rms_norm_fp8(y, w, residual=y)):
            with pytest.raises(TypeError, match="unsupported activation dtype"):
                call()


def test_grids_stay_below_their_limit():
    """2^24 workgroups of 256 are 2^32 threads, one more than a grid may have: the calls
    that would launch them are refused by their sizes (nothing is read: the addresses
    are none), the largest that would not pass this check and fail the next."""
    from selective_attention import _lib

    def rows(n, dim, ldx):
        return lambda: _lib.call("sa_rows_fp8", 1, 4096, None, 0, n, dim, ldx, dim, 4096, 4096, None)

    def norm(n, dim, ldx):
        return lambda: _lib.call("sa_rms_norm_fp8", 1, 4096, None, 4096, n, dim, ldx, 1e-6, None, 4096, 4096, None)
    most = (1 << 24) - 1
    for make, n, dim in ((rows, 16 * most, 128), (rows, 16 * most, 5), (rows, most, 2048), (rows, 5 * most, 300),
                         (norm, 4 * most, 100), (norm, 4 * most, 512), (norm, (1 << 24) - 1, 2000), (norm, (1 << 21) - 1, 16384),
                         (norm, 16 * most // 12, 1536)):
        with pytest.raises(RuntimeError, match="row stride"):
            make(n, dim, dim - 1)()
    for make, n, dim in ((rows, 16 * most + 1, 128), (rows, (1 << 28) - 1, 7), (rows, most + 1, 2048), (norm, 4 * most + 1, 100),
                         (norm, (1 << 26) - 1, 512), (norm, 1 << 24, 2000), (norm, 1 << 22, 16384), (rows, 1 << 40, 1 << 26)):
        with pytest.raises(RuntimeError, match="too many"):
            make(n, dim, dim - 1)()


# --- rows on the GPU ---------------------------------------------------------------
SHAPES = [(1, 1), (3, 127), (2, 128), (5, 130), (1, 512), (4, 1000), (7, 1024), (3, 2056), (65, 4096), (2, 4100),
          (3, 8200), (2, 16384), (1, 20000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize_rows(shape, gated, dtype):
    x = rand(*shape, seed=5, dtype=dtype)
    gate = torch.sigmoid(rand(*shape, seed=6, dtype=torch.float32, big=False)).to(dtype) if gated else None
    r = quantize_rows_fp8(x.cuda(), None if gate is None else gate.cuda())
    same_rows(r, x.double() if gate is None else x.double() * gate.double())


@pytest.mark.gpu
def test_quantize_rows_borders():
    """Ties, both ends of a block's range, subnormal codes, zeros, and blocks at fp32's ends."""
    x = torch.zeros(6, 256)
    ties = torch.arange(8, 16, dtype=torch.float32)
    x[0, 0], x[0, 1:9], x[0, 9:17] = 448.0, ties + 0.5, -(ties + 0.5) * 2.0 ** -8
    x[1, 0], x[1, 130] = 448.0, float(torch.nextafter(torch.tensor(448.0), torch.tensor(1e9)))
    x[2, 0], x[2, 1:65] = 1.0, torch.arange(64, dtype=torch.float32) * 2.0 ** -18
    x[3, 5], x[3, 200] = 1e-45, 2.0 ** -130
    x[4, 5], x[4, 6] = 3.4e38, -1e30
    x[5, 1], x[5, 2] = 447.99997, 16.499998
    same_rows(quantize_rows_fp8(x.cuda()), x)
    same_rows(quantize_rows_fp8(x.to(torch.bfloat16).cuda()), x.to(torch.bfloat16).double())


@pytest.mark.gpu
def test_quantize_rows_next_to_ties():
    """fp32 products whose rounding to fp32 is a tie of e4m3: the remainder decides."""
    a = torch.full((1, 128), 448.0)
    b = torch.ones(1, 128)
    # (1 + 2^-4 + 2^-12) (1 - 2^-12 + ..): exact products around 1.0625, the tie of 1 and 1.125
    for i in range(1, 120):
        u = 1.0625 * (1.0 + i * 2.0 ** -20)
        a[0, i] = torch.tensor(u)
        b[0, i] = torch.tensor(1.0625) / a[0, i]
    exact = a.double() * b.double()
    near = (exact - 1.0625).abs()[0, 1:120]
    assert (near[near > 0] < 2.0 ** -23).any()
    same_rows(quantize_rows_fp8(a.cuda(), b.cuda()), exact)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tiny_gated_rows_next_to_ties(dtype):
    """Products below fp32's normal numbers, beside ties of the smallest scale by less than
    half of fp32's last step there, or half of it: fp32's own product is the tie.  Up to 16 rows of bfloat16 in the product too, whose
    weight of ones and twos adds codes that fp32 holds."""
    e = torch.exp2(torch.linspace(20, 60, 128).floor().double())
    if dtype == torch.bfloat16:     # 145 226 = 2^15 (1 + 2^-14): half of fp32's last step above half of the codes'
        tie = torch.full((128,), 2.0 ** -136).double()
        over, f = torch.full((128,), 2.0 ** -14).double(), (145 / 128, 226 / 256)
    else:
        tie = ((torch.arange(8) * 2.0 + 1.0) * 2.0 ** -136).double().repeat(16)
        over = torch.where(torch.arange(128) % 3 == 0, -1.0, 1.0).double() * 2.0 ** -20
        f = 1 + over, 1.0
    sign = torch.where(torch.arange(128) % 5 == 0, -1.0, 1.0).double()
    x = torch.stack([f[0] / e, 1 / e, torch.zeros(128).double()]).to(dtype)
    gate = torch.stack([f[1] * tie * e * sign, tie * e, torch.ones(128).double()]).to(dtype)
    v = x.double() * gate.double()
    assert torch.equal(v[0], tie * (1 + over) * sign) and torch.equal(v[1], tie)
    assert ((x.float() * gate.float()).double()[0] == tie * sign).all()
    v = torch.where(v.abs() <= 2.0 ** -150, 0.0, v)
    r = quantize_rows_fp8(x.cuda(), gate.cuda())
    same_rows(r, v)
    if dtype == torch.bfloat16:
        ws = tuple(t.cuda() for t in pack_fp8(torch.ones(16, 128).to(E4), torch.full((1, 1), 247, dtype=torch.uint8)))
        for rows in (1, 2, 3):
            got = fp8_linear(x[:rows].cuda(), *ws, xscale=gate[:rows].cuda())
            assert torch.equal(got, fp8_linear(Fp8Rows(r.codes[:rows], r.scales[:rows]), *ws))
            assert torch.equal(got.double().cpu()[:, 0], (ref.values(r.codes[:rows], r.scales[:rows], 128).sum(1) * 2.0 ** 120).to(torch.bfloat16).double())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_are_not_finite(dtype):
    x = rand(6, 300, seed=8, dtype=dtype)
    x[1, 7], x[2, 140], x[3, 299] = math.inf, -math.inf, math.nan
    x[4, 128:256] = math.inf
    same_rows(quantize_rows_fp8(x.cuda()), x.double())
    one = torch.ones_like(x)
    same_rows(quantize_rows_fp8(x.cuda(), one.cuda()), x.double())
    same_rows(quantize_rows_fp8(one.cuda(), x.cuda()), x.double())


@pytest.mark.gpu
@pytest.mark.parametrize("fn", ["rows", "gated", "silu", "norm"])
def test_rows_of_a_stride(fn):
    """Slices of longer rows, on and off 16-byte boundaries, views and expanded rows."""
    wide = rand(9, 600, seed=9)
    other = rand(9, 600, seed=10, big=False)
    w = 0.1 * rand(256, seed=1, dtype=torch.float32)
    for a, b in ((0, 0), (8, 16), (3, 8), (1, 1)):
        x, c = wide[:, a:a + 256], other[:, b:b + 256]
        xg, cg = wide.cuda()[:, a:a + 256], other.cuda()[:, b:b + 256]
        if fn == "rows":
            same_rows(quantize_rows_fp8(xg), x.double())
        elif fn == "gated":
            same_rows(quantize_rows_fp8(xg, cg), x.double() * c.double())
        elif fn == "silu":
            check_silu(silu_mul_fp8(xg, cg), x, c)
        else:
            same_rows(rms_norm_fp8(xg, w.cuda(), 1e-6), ref.rms_norm(x, w, 1e-6)[1])
            t, v = ref.rms_norm(x, w, 1e-6, c)
            got, r = rms_norm_fp8(xg, w.cuda(), 1e-6, residual=cg)
            assert torch.equal(got.cpu(), t)
            same_rows(r, v)
    if fn == "rows":
        x3 = wide[:8].view(2, 4, 600).transpose(0, 1)
        same_rows(quantize_rows_fp8(wide[:8].cuda().view(2, 4, 600).transpose(0, 1)), x3.double())
        same_rows(quantize_rows_fp8(wide[:1].cuda().expand(5, 600)), wide[:1].expand(5, 600).double())
        same_rows(quantize_rows_fp8(wide[0].cuda()), wide[0].double())


def check_silu(r, a, c):
    a, c = a.double(), c.double()
    v = (a * c * torch.sigmoid(c)).reshape(-1, a.shape[-1])
    K = v.shape[1]
    kb = (K + 127) // 128
    got = r.codes.cpu().double().reshape(v.shape[0], -1)
    s = r.scales.cpu().double().reshape(v.shape[0], -1)
    v = torch.nn.functional.pad(v, (0, 128 * kb - K))
    top = v.abs().view(-1, kb, 128).amax(2)
    off = 8 * 2.0 ** -24
    lo, hi = ref.scale_of(top * (1 - off)), ref.scale_of(top * (1 + off))
    assert ((s[:, :kb] >= lo) & (s[:, :kb] <= hi)).all() and (s[:, kb:] == 1).all()
    u = v / s[:, :kb].repeat_interleave(128, 1)
    tol = ref.half_step(u.abs() * (1 + off)) + off * u.abs()
    assert ((got - u).abs() <= tol).all() and not got[:, K:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_silu_mul(shape):
    a, c = rand(*shape, seed=11), (3 * rand(*shape, seed=12, big=False)).to(torch.bfloat16)
    check_silu(silu_mul_fp8(a.cuda(), c.cuda()), a, c)


@pytest.mark.gpu
def test_silu_mul_ends():
    """Far gates, where e^-c leaves fp32; infinities and NaN."""
    c = torch.linspace(-120, 120, 256).to(torch.bfloat16)[None].repeat(2, 1)
    a = torch.ones_like(c)
    a[0, :128] = 2.0 ** -100
    r = silu_mul_fp8(a.cuda(), c.cuda())
    keep = c.double() > -86          # (below, e^-c may pass fp32's range and the product is 0)
    v = torch.where(keep, a.double() * c.double() * torch.sigmoid(c.double()), 0.0)
    got = torch.where(keep, r.dequantize().cpu().double(), 0.0)
    s = r.scales.cpu().double()[:, :2].repeat_interleave(128, 1)
    assert ((got - v).abs() <= s * (ref.half_step(v / s) + 1e-6 * (v / s).abs())).all()
    assert torch.isfinite(r.codes.float()).all()
    bad = torch.tensor([[math.inf, -math.inf, math.nan, 1.0]]).to(torch.bfloat16)
    fine = torch.ones_like(bad)
    for x, y in ((bad, fine), (fine, bad)):
        assert torch.isnan(silu_mul_fp8(x.cuda(), y.cuda()).codes.float().cpu()[0, :4]).tolist() == [True, True, True, False]


@pytest.mark.gpu
def test_silu_mul_where_a_c_passes_fp32():
    """a c beyond fp32's range, a silu(c) within it; and far gates, whose product is 0."""
    c = -torch.linspace(0.25, 86, 256).to(torch.bfloat16)[None].repeat(2, 1)
    a = torch.full_like(c, 2.0 ** 127)
    a[1] = -a[1]
    check_silu(silu_mul_fp8(a.cuda(), c.cuda()), a, c)
    far = torch.full_like(c, -2.0 ** 100)
    r = silu_mul_fp8(a.cuda(), far.cuda())
    assert not r.codes.float().any() and (r.scales.float() == 1).all()


def check_silu_of_all(r, a, c):
    """check_silu where a product may lie below fp32's range: 2^-150 and less counts as 0."""
    v = a.double() * c.double() * torch.sigmoid(c.double())
    check_silu(r, torch.where(v.abs() <= 2.0 ** -150, 0.0, a.double()), c)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", range(-30, 101, 10))
def test_silu_mul_of_far_gates(shift):
    """Gates to both ends of bfloat16 beside every size of a that leaves a finite product: a
    product from 2^-136 on, half a step of the smallest scale, has its code."""
    big = torch.tensor([17.0, 88.0, 100.0, 127.0, 128.0, 200.0, 2.3e38, 2.4e38, 3.38e38])
    far = -torch.cat([torch.arange(80, 92, 0.5), torch.arange(92, 200, 4.0), torch.tensor([1e3, 1e30, 2.4e38, 3.38e38])])
    c = torch.cat([big, far, torch.linspace(-79, 16, 20)]).to(torch.bfloat16)
    top = torch.where(c > 1, 2.0 ** 127 / c.double(), 2.0 ** 127)
    a = (top * 2.0 ** -shift if shift >= 0 else torch.full_like(top, 2.0 ** (4 * shift))).clamp(max=2.0 ** 127)
    a = (a * torch.where(torch.arange(len(c)) % 2 == 0, 1.0, -1.0)).to(torch.bfloat16)
    assert torch.isfinite((a.double() * c.double() * torch.sigmoid(c.double())).float()).all()
    # a block for each pair, so that each has the scale of its own
    x, g = torch.zeros(len(c), 128).to(torch.bfloat16), torch.ones(len(c), 128).to(torch.bfloat16)
    x[:, 9], g[:, 9] = a, c
    check_silu_of_all(silu_mul_fp8(x.cuda(), g.cuda()), x, g)
    # and all in one row, beside ordinary ones, which stay as they are alone
    x, g = rand(2, 256, seed=1), rand(2, 256, seed=2, big=False)
    alone = silu_mul_fp8(x[1:].cuda(), g[1:].cuda())
    x[0, :len(c)], g[0, :len(c)] = a, c
    r = silu_mul_fp8(x.cuda(), g.cuda())
    check_silu_of_all(r, x, g)
    assert torch.equal(r.codes[1:].view(torch.uint8), alone.codes.view(torch.uint8))


@pytest.mark.gpu
def test_silu_mul_of_tiny_numbers():
    """Products below fp32's normal numbers, of tiny factors of either kind."""
    g = torch.Generator().manual_seed(3)
    e = torch.arange(-133, -60).double()[:, None]
    x = (torch.randn(len(e), 128, generator=g).double() * torch.exp2(e)).to(torch.bfloat16)
    for c in (torch.randn(len(e), 128, generator=g) * 4 - 2, -80 - 8 * torch.rand(len(e), 128, generator=g)):
        check_silu_of_all(silu_mul_fp8(x.cuda(), c.to(torch.bfloat16).cuda()), x, c.to(torch.bfloat16))
    c = (torch.randn(len(e), 128, generator=g).double() * torch.exp2(-60 - e / 2)).to(torch.bfloat16)
    check_silu_of_all(silu_mul_fp8(x.cuda(), c.cuda()), x, c)
    check_silu_of_all(silu_mul_fp8(c.cuda(), x.cuda()), c, x)


@pytest.mark.gpu
def test_silu_mul_of_gates_without_end():
    """An infinite or NaN gate, or a, gives NaN, beside far gates too."""
    inf = math.inf
    a = torch.tensor([[1.0, 1.0, 1.0, inf, -inf, math.nan, inf, 0.0, 1.0, 2.0]]).to(torch.bfloat16)
    c = torch.tensor([[inf, -inf, math.nan, -100.0, 100.0, -100.0, -3e38, inf, -100.0, 1.0]]).to(torch.bfloat16)
    for x, y in ((a, c), (a[:, :8], c[:, :8])):
        r = silu_mul_fp8(x.cuda(), y.cuda())
        assert torch.isnan(r.codes.float().cpu()[0, :8]).all() and not torch.isnan(r.codes[0, 8:].float()).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", SHAPES + [(1, 65536), (2, 33000), (513, 1000), (600, 1024), (530, 1999),
                                            (520, 4095), (515, 4096), (514, 8191), (523, 1301), (515, 2560), (514, 2057),
                                            (513, 6100), (3, 10001), (2, 30001)])
def test_rms_norm(shape, residual, dtype):
    x, w = rand(*shape, seed=13, dtype=dtype), 0.3 * rand(shape[-1], seed=14, dtype=torch.float32)
    res = rand(*shape, seed=15, dtype=dtype) if residual else None
    t, v = ref.rms_norm(x, w, 1e-6, res)
    got = rms_norm_fp8(x.cuda(), w.cuda(), 1e-6, residual=None if res is None else res.cuda())
    if residual:
        assert torch.equal(got[0].cpu(), t)
        got = got[1]
    same_rows(got, v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1500, 4096), (6000, 1024), (5, 30000)])
def test_rms_norm_of_many_numbers(shape, dtype):
    """Enough numbers that some hundred lie within a few fp32 steps of a tie (2^-19 of
    them a step), and tiny ones: blocks below fp32's normal numbers, rows below 2^-100."""
    x, w = rand(*shape, seed=33, dtype=dtype), 0.3 * rand(shape[-1], seed=34, dtype=torch.float32)
    x[0] = x[0].double().div(x[0].double().abs().max()).mul(3.2e38).to(dtype)   # (near the type's end)
    x[1] *= 2.0 ** -100
    x[2, :512] *= 2.0 ** -110
    x[2, 512:1024] *= 2.0 ** -125
    w[512:640] = -1.0
    _, v = ref.rms_norm(x, w, 1e-12)
    same_rows(rms_norm_fp8(x.cuda(), w.cuda(), 1e-12), v)


@pytest.mark.gpu
def test_rms_norm_of_odd_rows():
    """A row of zeros, tiny and large rows, one with an infinity or a NaN; its neighbours stand."""
    x = rand(6, 640, seed=16, dtype=torch.float32)
    w = 0.2 * rand(640, seed=17, dtype=torch.float32)
    x[0] = 0.0
    x[1] *= 1e-20
    x[2] *= 1e15
    x[3, 5] = math.nan
    r = rms_norm_fp8(x.cuda(), w.cuda(), 1e-6)
    keep = [0, 1, 2, 4, 5]
    v = ref.rms_norm(x, w, 1e-6)[1]
    for i in keep:
        same_rows(Fp8Rows(r.codes[i:i + 1], r.scales[i:i + 1]), v[i:i + 1])
    assert torch.isnan(r.codes[3].float()).all()
    x[4, 9] = math.inf               # the factor is 0: zeros, and NaN where 0 meets the infinity
    r = rms_norm_fp8(x.cuda(), w.cuda(), 1e-6)
    want = torch.zeros(640)
    want[9] = math.nan
    assert torch.equal(torch.isnan(r.codes[4].float()).cpu(), torch.isnan(want))
    assert not torch.nan_to_num(r.codes[4].float()).any()
    same_rows(Fp8Rows(r.codes[5:], r.scales[5:]), v[5:])
    big = x[5:] * 1e25                                   # squares beyond fp32
    same_rows(rms_norm_fp8(big.cuda(), w.cuda(), 1e-6), ref.rms_norm(big, w, 1e-6)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dim", [1, 130, 640, 1500, 2500, 9000])
def test_rms_norm_of_tiny_rows(dim, residual, dtype):
    """Rows below fp32's normal numbers, whose factor passes fp32, with eps 0 and near it."""
    x = rand(6, dim, seed=18, dtype=torch.float32, big=False)
    for i, e in enumerate((-126, -130, -133, -140, -143, 0)):
        x[i] *= 2.0 ** e
    x[4, 0] = 2.0 ** -133 if dtype == torch.bfloat16 else 1e-45     # (not all zeros)
    x = x.to(dtype)
    res = rand(6, dim, seed=19, dtype=dtype, big=False) * 2.0 ** -130 if residual else None
    w = 0.3 * rand(dim, seed=20, dtype=torch.float32, big=False)
    for eps in (0.0, 2.0 ** -149):
        t, v = ref.rms_norm(x, w, eps, res)
        got = rms_norm_fp8(x.cuda(), w.cuda(), eps, residual=None if res is None else res.cuda())
        if residual:
            assert torch.equal(got[0].cpu(), t)
            got = got[1]
        keep = t.double().abs().sum(1) > 0 if eps == 0 else torch.ones(6, dtype=torch.bool)
        assert keep.sum() >= 4
        same_rows(Fp8Rows(got.codes.cpu()[keep], got.scales.cpu().view(torch.uint8)[keep].view(E8), dim), v[keep])
        assert torch.isnan(got.codes.float().cpu()[~keep, :dim]).all()      # (0 / 0)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [1e-6, 1e-5, 1e-60])
def test_rms_norm_takes_eps_as_given(eps):
    """Rows that eps alone scales, each number next to a tie, on the side that the given eps
    puts it on: half as far from it as eps in fp32 would move it."""
    e32 = float(torch.tensor(eps, dtype=torch.float32))
    off = (eps / e32) ** 0.5 - 1 if e32 else 1e-9
    side = 1e-9 if abs(off) < 1e-10 else off
    tie = (torch.arange(8, 16).double() + 0.5).repeat(16) * 2.0 ** -20
    g = torch.Generator().manual_seed(7)
    w = 1e-3 * (0.5 + torch.rand(128, generator=g).double())
    x = (tie * eps ** 0.5 / (1 + w)).float()
    w = (tie * (1 - side / 2) * eps ** 0.5 / x.double() - 1).float()      # (finer than x: its steps are 2^-33)
    v = ref.rms_norm(x[None], w, eps)[1]
    assert ((v / tie - 1).abs() < abs(side)).all() and ((v < tie) == (side > 0)).all()
    same_rows(rms_norm_fp8(x[None].cuda(), w.cuda(), eps), v)


@pytest.mark.gpu
def test_rms_norm_of_large_weights():
    """Numbers that the factor takes below fp32 and the weight brings back."""
    x, w = rand(3, 512, seed=21, dtype=torch.float32, big=False) * 1e-18, rand(512, seed=22, dtype=torch.float32, big=False)
    x[:, 3] = 1e30
    w[128:256] *= 1e25
    w[256:] *= 1e10
    same_rows(rms_norm_fp8(x.cuda(), w.cuda(), 1e-6), ref.rms_norm(x, w, 1e-6)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("fn", [lambda x: quantize_rows_fp8(x), lambda x: silu_mul_fp8(x, x),
                                lambda x: rms_norm_fp8(x, torch.zeros(200, device="cuda"))])
def test_no_rows(fn):
    r = fn(torch.zeros(0, 3, 200, dtype=torch.bfloat16, device="cuda"))
    assert r.shape == (0, 3, 200) and r.codes.shape == (0, 3, 256) and r.scales.shape == (0, 3, 4)
    packed = tuple(t.cuda() for t in quantize_fp8(rand(40, 200, dtype=torch.float32)))
    assert fp8_linear(r, *packed, out_features=40).shape == (0, 3, 40)


# --- products ------------------------------------------------------------------------
def weight(N, K, seed=20):
    w = rand(N, K, seed=seed, dtype=torch.float32) / K ** 0.5
    return quantize_fp8(w)


SIZES = [(1, 1, 1), (1, 128, 16), (2, 1000, 17), (3, 130, 300), (15, 512, 64), (16, 1024, 129), (17, 640, 100),
         (31, 4096, 48), (33, 2050, 65), (64, 1024, 4384), (65, 384, 130), (100, 129, 257), (128, 256, 128),
         (130, 1024, 140), (255, 2048, 255), (300, 700, 600), (513, 1152, 520), (1000, 128, 1000)]


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear(M, K, N, bias):
    rows, (packed, scales) = make_rows(M, K, seed=M), weight(N, K)
    b = rand(N, seed=2) if bias else None
    y = fp8_linear(on(rows), packed.cuda(), scales.cuda(), None if b is None else b.cuda(), out_features=N)
    assert y.shape == (M, N) and y.dtype == torch.bfloat16
    check_linear(y, rows, packed, scales, N, b)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", SIZES)
def test_linear_of_whole_numbers(M, K, N):
    """Sums that fp32 holds: the result is the exact one, rounded once."""
    g = torch.Generator().manual_seed(M + N)
    x, w = torch.randint(-4, 5, (M, K), generator=g).float(), torch.randint(-4, 5, (N, K), generator=g).float()
    kb = (K + 127) // 128
    xs = torch.randint(127, 130, (M, (kb + 3) // 4 * 4), generator=g).to(torch.uint8)
    rows = Fp8Rows(torch.nn.functional.pad(x, (0, -K % 128)).to(E4), xs.view(E8), K)
    packed, scales = pack_fp8(w.to(E4), torch.randint(126, 129, ((N + 127) // 128, kb), generator=g).to(torch.uint8))
    b = torch.randint(-8, 9, (N,), generator=g).to(torch.bfloat16)
    y = fp8_linear(on(rows), packed.cuda(), scales.cuda(), b.cuda(), out_features=N)
    want, _ = ref.linear(ref.values(rows.codes, rows.scales, K), ref.weight(packed, scales, N, K), b)
    assert torch.equal(y.cpu().double(), want.to(torch.bfloat16).double())


# (M, K, [N_i]), the kernel: few rows, tiles of each shape, odd borders, long K, many rows
TILES = [(61, 4000, [4090], "few"), (120, 3970, [1800, 1, 1000, 1090], "ring"), (30, 900, [1, 4000], "few"),
         (16, 1024, [20000], "few"), (32, 11008, [500], "few"), (64, 700, [12287], "ring"), (17, 256, [12289], "ring"),
         (64, 4096, [32000], "ring"), (66, 33000, [70], "few"), (257, 16384, [300], "few"), (500, 2050, [4383], "ring"),
         (1111, 1030, [4383], "ring"), (2001, 1024, [4384], "ring"), (2047, 4096, [4096], "ring"), (2047, 4096, [4100], "large"),
         (700, 4200, [1111], "ring"), (70000, 128, [64], "ring"), (8100, 1024, [4384], "ring"),
         (4100, 1408, [4097], "ring"), (8192, 2100, [4104], "ring"), (4095, 4096, [4095], "large"),
         (300, 640, [128, 1, 1000, 333], "ring"), (4096, 2048, [1111, 2000, 77, 900], "ring"), (2040, 6000, [2000, 1027, 77, 900], "large"),
         (3000, 1, [5000], "ring"), (5000, 130, [5001], "ring"), (300, 100, [1111], "ring"), (900, 300, [900], "ring"),
         (129, 2100, [30001], "ring"), (200, 1300, [9000, 5000], "ring"), (70, 1500, [37000], "ring"), (3000, 5000, [1030], "ring"),
         (4, 1204, [36073], "few"), (720, 714, [1933], "ring"),
         (100, 11000, [3900], "few"), (97, 9000, [1800, 1, 1000, 1090], "few"), (22001, 1090, [61], "ring"), (20000, 1700, [29, 1], "ring"),
         (16, 4100, [24003], "few"), (1, 9000, [8001, 3000], "few"), (33, 4096, [24001], "ring"), (33, 4090, [9000, 14001], "ring")]


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,sizes,kernel", TILES)
def test_linear_tiles(M, K, sizes, kernel):
    """Whole numbers as above, against float64 on the GPU; every kernel and its borders."""
    from selective_attention.profiling import kernel_timer
    g = torch.Generator(device="cuda").manual_seed(M + K)
    draw = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, device="cuda")  # noqa: E731
    kb, K8 = (K + 127) // 128, -K % 128
    x = draw(-3, 4, M, K).float()
    xs = draw(127, 129, M, (kb + 3) // 4 * 4).to(torch.uint8)
    rows = Fp8Rows(torch.nn.functional.pad(x, (0, K8)).to(E4), xs.view(E8), K)
    xv = x.double() * torch.exp2(xs.double() - 127)[:, torch.arange(K, device="cuda") // 128]
    ws, bs, want = [], [], []
    for N in sizes:
        w, s = draw(-3, 4, N, K).float(), draw(126, 129, (N + 127) // 128, kb).to(torch.uint8)
        ws.append(pack_fp8(w.to(E4), s))
        bs.append(draw(-8, 9, N).to(torch.bfloat16) if N % 2 else None)
        at = torch.arange(N, device="cuda")[:, None] // 128, torch.arange(K, device="cuda")[None] // 128
        y = torch.matmul(xv, (w.double() * torch.exp2(s.double() - 127)[at]).t().contiguous())
        want.append(y if bs[-1] is None else y + bs[-1].double())
    with kernel_timer() as kt:
        ys = fp8_linear_multi(rows, ws, bs, sizes)
    assert list(kt.stats) == ["fp8_" + kernel]
    for y, v in zip(ys, want):
        assert torch.equal(y, v.to(torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_few_bfloat16_rows_of_a_large_weight(gated):
    """Whole numbers again: rows rounded by the product, weights that pass the caches by."""
    g = torch.Generator(device="cuda").manual_seed(5)
    M, K, N = 5, 9001, 11003
    x = torch.randint(-3, 4, (M, K), generator=g, device="cuda").to(torch.bfloat16)
    gate = torch.randint(0, 3, (M, K), generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randint(-3, 4, (N, K), generator=g, device="cuda").float()
    packed, scales = pack_fp8(w.to(E4), torch.full(((N + 127) // 128, (K + 127) // 128), 127, dtype=torch.uint8, device="cuda"))
    v = x.double() * gate.double() if gated else x.double()
    y = fp8_linear(x, packed, scales, out_features=N, xscale=gate if gated else None)
    assert torch.equal(y, torch.matmul(v, w.double().t().contiguous()).to(torch.bfloat16))


@pytest.mark.gpu
def test_linear_results_next_to_others():
    """Outputs stop at their matrix's last row and column."""
    for M, K, N in ((5, 256, 33), (70, 256, 65), (300, 384, 129), (4100, 1408, 4097), (4095, 4096, 4095)):
        packed, scales = (t.cuda() for t in weight(N, K))
        x = make_rows(M, K) if M < 1000 else Fp8Rows(torch.ones(M, K).to(E4), torch.full((M, (K + 511) // 512 * 4), 127, dtype=torch.uint8).view(E8))
        x = on(x)
        pool = torch.full((M * N + 4096,), 7.0, dtype=torch.bfloat16, device="cuda")
        from selective_attention.kernels.fp8 import linear_multi
        want = linear_multi(x.codes, x.scales, [(packed, scales)], [None], [N])[0]
        import ctypes
        from selective_attention import _lib
        words = (ctypes.c_int64 * 5)(packed.data_ptr(), scales.data_ptr(), 0, pool.data_ptr() + 2 * 1025, N)
        _lib.call("sa_fp8_linear", x.codes.data_ptr(), x.scales.data_ptr(), M, K, 1, words, _lib.stream_of(pool))
        assert torch.equal(pool[1025:1025 + M * N].view(M, N), want)     # (rows off every boundary)
        assert (pool[:1025] == 7).all() and (pool[1025 + M * N:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_cuts_within_eight_columns_alone(M):
    """Large terms that cancel leave what stands outside their groups of eight columns,
    down to 2^-20 of them, also in other blocks: 2^16 + 2^-4 has 21 bits, fp32 holds 24
    (of 2^-13, 2^-29 of 2^16, it could hold none)."""
    K, N = 640, 16
    x, w = torch.zeros(M, K), torch.ones(N, K)
    x[:, 0], x[:, 88] = 256.0, -256.0
    for i, k in enumerate((8, 40, 64, 96, 127, 128, 300, 639)):
        x[:, k] = 2.0 ** (i - 4)
    scales = torch.full((M, 8), 127, dtype=torch.uint8).view(E8)
    sel = torch.zeros(K, dtype=torch.bool)
    sel[0] = sel[88] = True
    packed, ws = pack_fp8(torch.where(sel, 256 * w, w).to(E4), torch.ones(1, 5))
    y = fp8_linear(Fp8Rows(x.to(E4).cuda(), scales.cuda()), packed.cuda(), ws.cuda(), out_features=N)
    assert (y.cpu().double() == 255 * 2.0 ** -4).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 40, 200])
def test_linear_of_tensors_and_gates(M):
    K, N = 333, 77
    packed, scales = weight(N, K)
    x, gate = rand(2, M, K, seed=3), torch.sigmoid(rand(2, M, K, seed=4, big=False))
    for g in (None, gate):
        v = x.double() if g is None else x.double() * g.double()
        codes, s = ref.rows(v.reshape(-1, K))
        rows = Fp8Rows(codes.to(E4), (torch.log2(s) + 127).to(torch.uint8).view(E8), K)
        y = fp8_linear(x.cuda(), packed.cuda(), scales.cuda(), out_features=N, xscale=None if g is None else g.cuda())
        assert y.shape == (2, M, N)
        check_linear(y, rows, packed, scales, N)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 1024), (5, 333), (16, 130), (16, 4104), (9, 2048), (17, 500)])
def test_few_rows_are_rounded_as_by_the_rows_op(M, K, gated):
    """Up to 16 bf16 rows go through one launch that rounds them itself: the same codes
    and, at these widths, the same order of sums; on and off 16-byte boundaries, with what
    is not finite, several matrices and a bias."""
    wide, other = rand(M, K + 24, seed=M), torch.sigmoid(rand(M, K + 24, seed=3, big=False))
    if M > 2:
        wide[1, K // 2 + 8], wide[2, 8] = math.inf, math.nan
        wide[0] = 0.0
    ws = [tuple(t.cuda() for t in weight(n, K, seed=n)) for n in (64, 1, 300)]
    bs = [rand(64, seed=1).cuda(), None, rand(300, seed=2).cuda()]
    for a, b in ((0, 0), (8, 16), (3, 8), (1, 2)):
        x, g = wide.cuda()[:, a:a + K], other.cuda()[:, b:b + K] if gated else None
        want = fp8_linear_multi(quantize_rows_fp8(x, g), ws, bs, [64, 1, 300])
        for y, v in zip(fp8_linear_multi(x, ws, bs, [64, 1, 300], g), want):
            assert torch.equal(torch.isnan(y), torch.isnan(v))
            assert torch.equal(torch.nan_to_num(y), torch.nan_to_num(v))


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
def test_few_rows_at_both_ends_of_their_type(gated):
    """Subnormal bfloat16 numbers and those next to its end, rounded by the product as by the
    rows op, which is the oracle's: a weight of one code a row brings each block's codes out."""
    e = torch.tensor([-133, -130, -127, -126, -124, -120, -100, 100, 120, 125, 126, 127])
    g = torch.Generator().manual_seed(2)
    x = ((torch.rand(12, 384, generator=g) + 1).double() * torch.exp2(e.double())[:, None]
         * torch.exp2(-torch.randint(0, 9, (12, 384), generator=g).double())).to(torch.bfloat16)
    x[:, ::7] *= -1
    assert torch.isfinite(x).all()
    gate = (2.0 ** torch.randint(-1, 1, (12, 384), generator=g)).to(torch.bfloat16) if gated else None
    v = x.double() if gate is None else x.double() * gate.double()
    codes, s = ref.rows(v)
    w = torch.zeros(384, 384)
    w[torch.arange(384), torch.arange(384)] = 1.0
    # one scale for both ends would leave bf16: two weights
    for byte, at in ((247, slice(0, 7)), (7, slice(7, 12))):
        packed, ws = pack_fp8(w.to(E4), torch.full((3, 3), byte, dtype=torch.uint8))
        y = fp8_linear(x[at].cuda(), packed.cuda(), ws.cuda(), xscale=None if gate is None else gate[at].cuda())
        want = codes[at] * s[at, :3].repeat_interleave(128, 1) * 2.0 ** (byte - 127)
        assert torch.equal(y.cpu().double(), want.to(torch.bfloat16).double())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 20, 300])
def test_linear_multi(M):
    K, sizes = 600, [128, 1, 300, 513]
    ws = [weight(N, K, seed=N) for N in sizes]
    bs = [None, rand(1, seed=1), rand(300, seed=2), None]
    rows = make_rows(M, K)
    ys = fp8_linear_multi(on(rows), [(p.cuda(), s.cuda()) for p, s in ws], [None if b is None else b.cuda() for b in bs],
                          sizes)
    for y, w, b, N in zip(ys, ws, bs, sizes):
        assert y.is_contiguous()
        check_linear(y, rows, *w, N, b)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 64, 257])
def test_linear_scales(M):
    """Every block with a scale of its own, far apart."""
    g = torch.Generator().manual_seed(4)
    K, N = 1300, 400
    rows = make_rows(M, K)
    rows.scales = torch.randint(90, 160, rows.scales.shape, generator=g).to(torch.uint8).view(E8)
    codes = torch.randn(N, K, generator=g).to(E4)
    packed, scales = pack_fp8(codes, torch.randint(90, 160, (4, 11), generator=g).to(torch.uint8))
    y = fp8_linear(on(rows), packed.cuda(), scales.cuda(), out_features=N)
    check_linear(y, rows, packed, scales, N)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [4, 70, 300])
def test_linear_keeps_nan_in_its_row(M):
    K, N = 500, 200
    x = rand(M, K, seed=7)
    x[1, 130] = math.inf
    x[M - 1, 3] = math.nan
    packed, scales = (t.cuda() for t in weight(N, K))
    y = fp8_linear(x.cuda(), packed, scales, out_features=N)
    bad = torch.zeros(M, dtype=torch.bool)
    bad[1] = bad[M - 1] = True
    assert torch.equal(torch.isnan(y).all(1).cpu(), bad) and torch.equal(torch.isnan(y).any(1).cpu(), bad)
    x[1, 130] = x[M - 1, 3] = 0.0
    z = fp8_linear(x.cuda(), packed, scales, out_features=N)
    assert torch.equal(y.cpu()[~bad], z.cpu()[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("M", [4, 90])
def test_linear_of_views(M):
    """Rows and scales that are slices are copied; uint8 scales are taken as they are."""
    K, N = 256, 96
    rows, (packed, scales) = make_rows(2 * M, K), weight(N, K)
    cut = Fp8Rows(on(rows).codes[::2], on(rows).scales.view(torch.uint8)[::2])
    y = fp8_linear(cut, packed.cuda(), scales.view(torch.uint8).cuda(), out_features=N)
    check_linear(y, Fp8Rows(rows.codes[::2], rows.scales.view(torch.uint8)[::2].contiguous()), packed, scales, N)


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(1, 1), (40, 200), (128, 128), (300, 515)])
def test_dequantize(N, K):
    packed, scales = weight(N, K)
    got = dequantize_fp8(packed.cuda(), scales.cuda(), N, K)
    assert got.dtype == torch.bfloat16 and torch.equal(got.cpu().double(), ref.weight(packed, scales, N, K))
    with pytest.raises(ValueError):
        dequantize_fp8(packed.cuda(), scales.cuda(), N + 16, K)


@pytest.mark.gpu
def test_dequantize_of_the_widest_weight():
    """2^31 - 1 columns: the last piece of a row stops at its end."""
    from selective_attention import _lib
    K = (1 << 31) - 1
    packed = torch.zeros(1, 1 << 24, 8, 16, 16, dtype=torch.uint8, device="cuda")
    packed[0, -1, :, 0] = torch.ones(8, 16).to(E4).view(torch.uint8)
    scales = torch.full((1, 1 << 24), 128, dtype=torch.uint8, device="cuda")
    pool = torch.full((K + 9,), 7.0, dtype=torch.bfloat16, device="cuda")
    _lib.call("sa_fp8_dequant_bf16", packed.data_ptr(), scales.data_ptr(), 1, K, pool.data_ptr(), _lib.stream_of(pool))
    assert (pool[K:] == 7).all() and (pool[K - 127:K] == 2).all() and not pool[K - 4096:K - 127].any()
    assert not pool[:4096].any()


# --- gradients -------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 100])
def test_gradients_are_the_formulas(M):
    K, N = 300, 70
    packed, scales = weight(N, K)
    w = ref.weight(packed, scales, N, K)
    x, gate = rand(M, K, seed=1, big=False).cuda().requires_grad_(), torch.sigmoid(rand(M, K, seed=2, big=False)).cuda().requires_grad_()
    b, dy = rand(N, seed=3).cuda().requires_grad_(), rand(M, N, seed=4, big=False)
    y = fp8_linear(x, packed.cuda(), scales.cuda(), b, out_features=N)
    with torch.no_grad():
        assert torch.equal(y, fp8_linear(x, packed.cuda(), scales.cuda(), b, out_features=N))
    dx, db = torch.autograd.grad(y, (x, b), dy.cuda())
    want, A = ref.linear(dy.double(), w.t())
    # N products summed in fp32 and one rounding; the bias M
    assert ((dx.cpu().double() - want).abs() <= (N + 8) * 2.0 ** -23 * A + 2.0 ** -8 * want.abs()).all()
    want = dy.double().sum(0)
    assert ((db.cpu().double() - want).abs() <= (M + 8) * 2.0 ** -23 * dy.double().abs().sum(0) + 2.0 ** -8 * want.abs()).all()
    y = fp8_linear(x, packed.cuda(), scales.cuda(), out_features=N, xscale=gate)
    dxs = torch.autograd.grad(y, (x, gate), dy.cuda())
    want, A = ref.linear(dy.double(), w.t())
    for got, f in zip(dxs, (gate, x)):
        f = f.detach().cpu().double()
        # the product's gradient is rounded before and after it meets the other factor
        tol = ((N + 8) * 2.0 ** -23 * A + 2.0 ** -8 * want.abs()) * (1 + 2.0 ** -8) * f.abs() + 2.0 ** -8 * (want * f).abs()
        assert ((got.cpu().double() - want * f).abs() <= tol).all()
    rows = make_rows(M, K)
    y = fp8_linear(on(rows), packed.cuda(), scales.cuda(), b, out_features=N)
    (db,) = torch.autograd.grad(y, b, dy.cuda())
    want = dy.double().sum(0)
    assert ((db.cpu().double() - want).abs() <= (M + 8) * 2.0 ** -23 * dy.double().abs().sum(0) + 2.0 ** -8 * want.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 1), (7, 33), (64, 300), (65, 256), (3, 700, 257), (20000, 300), (70000, 5), (300, 70000)])
def test_bias_gradient(shape):
    """M numbers summed in fp32 (each addition off by half an ulp of at most the
    magnitudes' sum), rounded once."""
    N, M = shape[-1], math.prod(shape[:-1])
    packed, scales = (t.cuda() for t in weight(N, 1))
    b, dy = torch.zeros(N, dtype=torch.bfloat16, device="cuda").requires_grad_(), rand(*shape, seed=4, big=False)
    x = torch.ones(*shape[:-1], 1, dtype=torch.bfloat16, device="cuda")
    y = fp8_linear(x, packed, scales, b, out_features=N)
    (db,) = torch.autograd.grad(y, b, dy.cuda(), retain_graph=True)
    d = dy.double().reshape(M, N)
    want = d.sum(0)
    assert ((db.cpu().double() - want).abs() <= M * 2.0 ** -24 * d.abs().sum(0) + 2.0 ** -8 * want.abs()).all()
    assert torch.equal(db, torch.autograd.grad(y, b, dy.cuda(), retain_graph=True)[0])
    (db,) = torch.autograd.grad(y.sum(), b)      # (a gradient of one number in all places)
    assert torch.equal(db, torch.full_like(db, M))


@pytest.mark.gpu
@pytest.mark.parametrize("M", [12, 6000])
def test_gradients_captured(M):
    """A captured forward and backward, replayed on new inputs with eager work between."""
    K, N = 256, 384
    packed, scales = (t.cuda() for t in weight(N, K))
    x, b, dy = rand(M, K, big=False).cuda().requires_grad_(), rand(N, big=False).cuda().requires_grad_(), rand(M, N, seed=1).cuda()

    def run(x, b, dy):
        return torch.autograd.grad(fp8_linear(x, packed, scales, b, out_features=N), (x, b), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(x, b, dy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = run(x, b, dy)
    for turn in range(4):
        with torch.no_grad():
            x.copy_(rand(M, K, seed=10 + turn, big=False))
            dy.copy_(rand(M, N, seed=20 + turn))
        graph.replay()
        torch.cuda.synchronize()
        want = run(x.detach().clone().requires_grad_(), b.detach().clone().requires_grad_(), dy.clone())
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(out, want))


@pytest.mark.gpu
def test_gradient_is_the_difference():
    """Where x and x + d are both codes (whole numbers to 8, 448 in each block so that
    the scale is 1), the layer is linear in x and its difference is the gradient's:
    weights of whole numbers keep every sum exact."""
    K, N = 256, 32
    g = torch.Generator().manual_seed(0)
    x = torch.randint(-4, 5, (2, K), generator=g).float()
    x[:, 0] = x[:, 128] = 448.0
    codes = torch.randint(-2, 3, (N, K), generator=g).float()
    codes[:, 0] = codes[:, 128] = 0.0
    packed, scales = (t.cuda() for t in pack_fp8(codes.to(E4), torch.ones(1, 2)))
    d = torch.randint(-4, 5, (2, K), generator=g).float()
    d[:, 0] = d[:, 128] = 0.0
    xg = x.to(torch.bfloat16).cuda().requires_grad_()
    y = fp8_linear(xg, packed, scales, out_features=N)
    dy = torch.randint(-1, 2, (2, N), generator=g).to(torch.bfloat16)
    (dx,) = torch.autograd.grad(y, xg, dy.cuda())
    # the outputs' own rounding to bf16 is kept out by taking the difference of their exact values
    w = codes.double()
    diff = (((x + d).double() @ w.t() - x.double() @ w.t()) * dy.double()).sum()
    assert torch.equal(y.detach().cpu().double(), (x.double() @ w.t()).to(torch.bfloat16).double())
    y2 = fp8_linear((x + d).to(torch.bfloat16).cuda(), packed, scales, out_features=N)
    assert torch.equal(y2.cpu().double(), ((x + d).double() @ w.t()).to(torch.bfloat16).double())
    assert (dx.cpu().double() * d.double()).sum() == diff


def _second(packed, scales, N, K, M, dev):
    """The gradient by dy of |dx|^2 + |db|^2, whole numbers: dx = dy W and db the column sums."""
    g = torch.Generator().manual_seed(N)
    x = torch.randint(-4, 5, (M, K), generator=g).to(torch.bfloat16).to(dev).requires_grad_()
    b = torch.zeros(N, dtype=torch.bfloat16, device=dev).requires_grad_()
    dy = torch.randint(-1, 2, (M, N), generator=g).to(torch.bfloat16).to(dev).requires_grad_()
    w = dequantize_fp8(packed.to(dev), scales.to(dev), N, K).double().cpu()
    got = []
    for ts in ((x, b), (b,), (x,)):
        y = fp8_linear(x, packed.to(dev), scales.to(dev), b, out_features=N)
        ds = torch.autograd.grad(y, ts, dy, create_graph=True)
        (d2,) = torch.autograd.grad(sum(d.float().square().sum() for d in ds), dy)
        d = dy.detach().double().cpu()
        want = torch.zeros_like(d)
        if ts[0] is x:
            want = want + 2 * (d @ w @ w.t())
        if ts[-1] is b:
            want = want + 2 * d.sum(0)
        got.append((d2.cpu().double(), want))
    return got


def _whole_weight(N, K):
    g = torch.Generator().manual_seed(K)
    return pack_fp8(torch.randint(-1, 2, (N, K), generator=g).float().to(E4), torch.ones((N + 127) // 128, (K + 127) // 128))


def test_second_derivatives_on_the_cpu(monkeypatch):
    """The launches replaced by their arithmetic, without history as theirs: what is left
    is how the backward joins them.  Sums below 2^8 are exact in bfloat16."""
    from selective_attention.ops import fp8 as op
    packed, scales = _whole_weight(9, 6)
    w = ref.weight(packed, scales, 9, 6).to(torch.bfloat16)
    monkeypatch.setattr(op._k, "dequantize", lambda p, s, N, K: w.clone())
    monkeypatch.setattr(op._k, "linear_multi_bf16", lambda x, g, ws, bs, Ns: [(x.detach() @ w.t() + bs[0].detach())])
    monkeypatch.setattr(op._k, "column_sums", lambda d: d.detach().reshape(-1, 9).float().sum(0).to(torch.bfloat16))
    for d2, want in _second(packed, scales, 9, 6, 5, "cpu"):
        assert want.abs().max() <= 256 and torch.equal(d2, want) and want.any()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 40])
def test_second_derivatives(M):
    """Of both gradients together and each alone, exact below 2^8."""
    packed, scales = _whole_weight(9, 6)
    for d2, want in _second(packed, scales, 9, 6, M, "cuda"):
        assert want.abs().max() <= 256 and torch.equal(d2, want) and want.any()


@pytest.mark.gpu
def test_tangents_and_batches_of_the_gradient():
    """A dual dy keeps its tangent through both gradients; dys of a batch likewise."""
    import torch.autograd.forward_ad as fwd
    M, N, K = 7, 9, 6
    packed, scales = (t.cuda() for t in _whole_weight(N, K))
    g = torch.Generator().manual_seed(1)
    x = torch.ones(M, K, dtype=torch.bfloat16, device="cuda").requires_grad_()
    b = torch.zeros(N, dtype=torch.bfloat16, device="cuda").requires_grad_()
    dys = torch.randint(-1, 2, (3, M, N), generator=g).to(torch.bfloat16).cuda()
    y = fp8_linear(x, packed, scales, b, out_features=N)
    one = [torch.autograd.grad(y, (x, b), d, retain_graph=True) for d in dys]
    both = torch.autograd.grad(y, (x, b), dys, retain_graph=True, is_grads_batched=True)
    assert all(torch.equal(both[i][j], one[j][i]) for i in range(2) for j in range(3))
    with fwd.dual_level():
        ds = torch.autograd.grad(y, (x, b), fwd.make_dual(dys[0], dys[1]))
        for d, p, t in zip(ds, one[0], one[1]):
            got = fwd.unpack_dual(d)
            assert torch.equal(got.primal, p) and torch.equal(got.tangent, t)


@pytest.mark.gpu
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fwd
    packed, scales = (t.cuda() for t in weight(16, 128))
    x = torch.ones(1, 128, dtype=torch.bfloat16, device="cuda")
    with fwd.dual_level():
        dual = fwd.make_dual(x, x)
        for call in (lambda: fp8_linear(dual, packed, scales), lambda: quantize_rows_fp8(dual),
                     lambda: silu_mul_fp8(dual, dual), lambda: rms_norm_fp8(dual, torch.zeros(128, device="cuda"))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()


# --- a run of them, streams and graphs ---------------------------------------------------
def chain(x, res, w, ws, bs):
    """A pre-norm SwiGLU layer in 8 bits."""
    t, n = rms_norm_fp8(x, w, 1e-6, residual=res)
    a, c = fp8_linear_multi(n, ws[:2], bs[:2], [384, 384])
    return t + fp8_linear(silu_mul_fp8(a, c), *ws[2], bs[2], out_features=256)


def chain_inputs(M, seed=0):
    x, res = rand(M, 256, seed=seed).cuda(), rand(M, 256, seed=seed + 1).cuda()
    w = 0.1 * rand(256, seed=2, dtype=torch.float32).cuda()
    ws = [tuple(t.cuda() for t in weight(n, k, seed=i)) for i, (n, k) in enumerate(((384, 256), (384, 256), (256, 384)))]
    bs = [rand(n, seed=9, big=False).cuda() for n in (384, 384, 256)]
    return x, res, w, ws, bs


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 6, 80, 700])
def test_a_run_of_them(M):
    """Each step against the oracle on the step's own inputs."""
    x, res, w, ws, bs = chain_inputs(M)
    t, n = rms_norm_fp8(x, w, 1e-6, residual=res)
    want, v = ref.rms_norm(x.cpu(), w.cpu(), 1e-6, res.cpu())
    assert torch.equal(t.cpu(), want)
    same_rows(n, v)
    a, c = fp8_linear_multi(n, ws[:2], bs[:2], [384, 384])
    for y, p, b in ((a, ws[0], bs[0]), (c, ws[1], bs[1])):
        check_linear(y, n, *p, 384, b.cpu())
    r = silu_mul_fp8(a, c)
    check_silu(r, a.cpu(), c.cpu())
    y = fp8_linear(r, *ws[2], bs[2], out_features=256)
    check_linear(y, r, *ws[2], 256, bs[2].cpu())
    assert torch.equal(chain(x, res, w, ws, bs), t + y)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 300])
def test_captured_on_another_stream(M):
    """Two graphs of the run, replayed with eager work between, on new inputs."""
    ins = [chain_inputs(M, seed=s) for s in (0, 40)]
    eager = [chain(*i) for i in ins]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert all(torch.equal(chain(*i), e) for i, e in zip(ins, eager))
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(chain(*i))
        graphs.append(g)
    for turn in range(3):
        for k in (0, 1):
            x = rand(M, 256, seed=100 + turn + 10 * k).cuda()
            ins[k][0].copy_(x)
            graphs[k].replay()
            want = chain(*ins[k])
            torch.cuda.synchronize()
            assert torch.equal(outs[k], want)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows and outputs behind 2^32 bytes."""
    M, K, N = (1 << 25) // 2 + 5, 256, 128
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[-3:] = rand(3, K, seed=1).cuda()
    packed, scales = weight(N, K)
    r = quantize_rows_fp8(x)
    same_rows(Fp8Rows(r.codes[-3:], r.scales[-3:], K), x[-3:].cpu().double())
    del x
    y = fp8_linear(Fp8Rows(r.codes[:1 << 24], r.scales[:1 << 24]), packed.cuda(), scales.cuda(), out_features=N)
    assert not y[-1].any()
    y = fp8_linear(Fp8Rows(r.codes[5:], r.scales[5:]), packed.cuda(), scales.cuda(), out_features=N)
    check_linear(y[-3:], Fp8Rows(r.codes[-3:], r.scales[-3:]), packed, scales, N)
    assert not y[:-3].any()
    with pytest.raises(RuntimeError):
        fp8_linear(r, packed.cuda(), scales.cuda(), out_features=N)
