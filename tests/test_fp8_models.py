"""Models with 8-bit linear layers (quantize_fp8): each module against the ops it
stands for, and whole models, eager, captured and in training."""
import pytest
import torch

from selective_attention.inference import CausalBlockCache, GenerationConfig, InferenceState
from selective_attention.models import CausalLM, CausalLMConfig, Seq2SeqLM, Seq2SeqLMConfig
from selective_attention.modules.layers import Fp8Linear, Linear, RMSNorm, SwiGLU, project, quantize_linears_fp8
from selective_attention.ops import (Fp8Rows, dequantize_fp8, fp8_linear, fp8_linear_multi, quantize_rows_fp8,
                                     rms_norm_fp8, silu_mul_fp8)


def _model(layers=2):
    torch.manual_seed(0)
    return CausalLM(CausalLMConfig(vocab_size=500, model_dim=256, head_dim=64, ssm_state_dim=64, ssm_chunk_size=64,
                                   num_layers=layers, dropout_rate=0.0, device="cuda")).to_bf16().cuda().eval()


def _prompt(b, L, seed=1):
    return torch.randint(3, 300, (b, L), generator=torch.Generator().manual_seed(seed)).cuda()


def _gen(**kw):
    return GenerationConfig(bos_token_id=0, eos_token_id=1, pad_token_id=2, max_new_tokens=16,
                            attn_gate_thresholds=[0.88, 0.88], **kw)


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


# --- on the CPU ---------------------------------------------------------------------
def test_layer_keeps_its_types():
    lin = Linear(200, 300)
    q = Fp8Linear.from_linear(lin)
    assert q.packed.shape == (19, 2, 8, 16, 16) and q.scales.shape == (3, 4)
    before = {k: v.clone() for k, v in q.state_dict().items()}
    q.to(torch.float16).float()
    assert q.packed.dtype == q.scales.dtype == torch.uint8 and q.bias.dtype == torch.bfloat16
    other = Fp8Linear(200, 300)
    other.load_state_dict(before)
    assert all(torch.equal(v, other.state_dict()[k]) for k, v in q.state_dict().items())
    assert Fp8Linear(128, 16, bias=False).bias is None and "in_features=200" in repr(q)


def test_every_linear_layer_is_replaced():
    m = SwiGLU(64, 128)
    assert not m.takes_rows
    quantize_linears_fp8(m)
    assert m.takes_rows and all(isinstance(x, Fp8Linear) for x in (m.w1, m.w2, m.out))
    kept = m.w1
    assert quantize_linears_fp8(m).w1 is kept


class _Mixer(torch.nn.Module):
    """Stands for an SSM, an attention or a feed-forward that takes a tensor."""

    def __init__(self, two):
        super().__init__()
        self.two = two

    def forward(self, x, **kw):
        assert isinstance(x, torch.Tensor)
        return (x, None) if self.two else x


class _Sum(torch.nn.Identity):
    """A norm of another kind, with the two calls that a block makes of one."""

    def add_forward(self, x, y):
        return x + y, self(x + y)


def _plain_blocks():
    from selective_attention.modules import BiBlock, CausalBlock, CrossBlock
    kw = dict(layer_idx=0, model_dim=64, head_dim=32, ssm_state_dim=16, ssm_chunk_size=16, device="cpu")
    for cls in (CausalBlock, BiBlock, CrossBlock):
        b = cls(**kw).eval()
        b.ssm, b.mha, b.ffn = _Mixer(True), _Mixer(False), _Mixer(False)
        if cls is CrossBlock:
            b.cross_mha = _Mixer(False)
        yield b, dict(context=None, context_lengths=None, ssm_hiddens=None) if cls is CrossBlock else {}


def test_norms_are_called_as_norms():
    """Where no layer takes rows in 8 bits a norm is called with x alone: its hooks see one
    argument, and any module may stand in its place."""
    seen = []
    for block, kw in _plain_blocks():
        norms = [m for m in block.modules() if isinstance(m, RMSNorm)]
        for m in norms:
            m.register_forward_pre_hook(lambda m, args: seen.append(len(args)))
        x = torch.randn(2, 5, 64)
        block(x, **kw)                       # (with a gradient wanted, add_forward calls the norm)
        assert seen == [1] * len(norms) and len(norms) >= 3
        seen.clear()
        for name, m in list(block.named_children()):
            if isinstance(m, RMSNorm):
                setattr(block, name, _Sum())
        y = block(x, **kw)
        y = y if torch.is_tensor(y) else y[0]
        assert torch.equal(y, x * 2 ** len(norms))


def test_models_with_a_norm_of_another_kind():
    m = CausalLM(CausalLMConfig(vocab_size=20, model_dim=64, head_dim=32, ssm_state_dim=16, ssm_chunk_size=16,
                                num_layers=0, device="cpu")).eval()
    ids = torch.tensor([[3, 4, 5]])
    m.norm = torch.nn.LayerNorm(64)
    assert torch.equal(m(ids), m.lm_head(m.norm(m.embedding(ids))))
    quantize_linears_fp8(m)                  # (a layer that takes rows, a norm that has none)
    m.lm_head.forward = lambda x: x
    assert torch.equal(m(ids), m.norm(m.embedding(ids)))
    s = Seq2SeqLM(Seq2SeqLMConfig(vocab_size=20, model_dim=64, head_dim=32, ssm_state_dim=16, ssm_chunk_size=16,
                                  num_layers=0, device="cpu")).eval()
    s.ssm, s.norm1, s.norm4 = _Mixer(True), torch.nn.Identity(), torch.nn.Identity()
    s.norm3.forward = lambda x: x
    s.ssm.forward = lambda x, **kw: (x, torch.zeros(1, 4, 32, 16))
    h = s.embedding(ids)
    assert torch.equal(s.encode(ids, None)[0], s.norm2(h + h))
    assert torch.equal(s.decode(ids, None, None, None), s.lm_head(h))


# --- modules ------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 100])
def test_layer_is_the_op(rows):
    lin = Linear(300, 800).to(torch.bfloat16).cuda()
    q = Fp8Linear.from_linear(lin)
    x = _rand(2, rows, 300).cuda()
    with torch.no_grad():
        want = fp8_linear(x, q.packed, q.scales, q.bias, 800)
        assert torch.equal(q(x), want) and torch.equal(q(quantize_rows_fp8(x)), want)
        for sizes in ([128, 640, 32], [256, 544], [100, 700]):
            cut = q.split_forward(x, sizes)
            assert all(c.is_contiguous() for c in cut) and torch.equal(torch.cat(cut, -1), want)
        gate = torch.sigmoid(_rand(2, rows, 300, seed=1)).cuda()
        two = project(x, [q, q], xscale=gate)
        assert torch.equal(two[0], fp8_linear(quantize_rows_fp8(x, gate), *q.weights(), q.bias, 800))
        assert torch.equal(two[0], two[1])
        five = project(x, [q] * 5)
        assert all(torch.equal(y, want) for y in five)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 200])
def test_norm_and_swiglu(rows):
    torch.manual_seed(0)
    ffn = quantize_linears_fp8(SwiGLU(256, 1024).to(torch.bfloat16).cuda())
    norm = RMSNorm(256).cuda()
    with torch.no_grad():
        norm.weight.normal_(0, 0.2)
        x, y = _rand(2, rows, 256).cuda(), _rand(2, rows, 256, seed=1).cuda()
        n = norm(x, ffn)
        assert isinstance(n, Fp8Rows) and isinstance(norm(x), torch.Tensor) and n.shape == x.shape
        t, m = norm.add_forward(x, y, ffn)
        tt, mm = rms_norm_fp8(x, norm.weight, norm.eps, residual=y)
        assert torch.equal(t, tt) and torch.equal(t, x + y) and torch.equal(m.codes.view(torch.uint8), mm.codes.view(torch.uint8))
        a, c = fp8_linear_multi(m, [ffn.w1.weights(), ffn.w2.weights()], [ffn.w1.bias, ffn.w2.bias], [1024, 1024])
        want = fp8_linear(silu_mul_fp8(a, c), *ffn.out.weights(), ffn.out.bias, 256)
        assert torch.equal(ffn(m), want)
    # with a gradient the norm stays a tensor, and the layers pass it on
    x.requires_grad_()
    assert isinstance(norm(x, ffn), torch.Tensor)
    (g,) = torch.autograd.grad(ffn(norm(x, ffn)).float().sum(), x)
    assert torch.isfinite(g).all() and g.abs().max() > 0


# --- models -------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("batch", [1, 3])
def test_generate_captured_equals_eager(kv, batch):
    m, ids = _model().quantize_fp8(), _prompt(batch, 90)
    assert isinstance(m.lm_head, Fp8Linear) and not any(isinstance(x, torch.nn.Linear) for x in m.modules())
    kept = m.lm_head
    assert m.quantize_fp8().lm_head is kept
    cfg = _gen(kv_cache_dtype=kv)
    a, la = m.generate(ids, cfg, logprobs=3)
    b, lb = m.generate(ids, cfg, use_graph=False, logprobs=3)
    assert torch.equal(a, b) and a.shape == (batch, 106)
    assert all(torch.equal(x, y) for x, y in zip(la, lb))


@pytest.mark.gpu
@pytest.mark.parametrize("L", [40, 300])
def test_model_near_the_model_of_its_weights(L):
    """Against bf16 layers of the weights that the codes stand for.  What remains is the
    rows' rounding: each entry off by up to 2^-4 of itself, 2^-4 / sqrt(3) at random, in
    at most three of them on the way through a residual branch; three branches a block,
    two blocks and the head, each at most as large as the stream: sqrt(3 6 + 1) 2^-4 /
    sqrt(3) = 0.16 of the logits, and twice that as the bound."""
    m, ids = _model().quantize_fp8(), _prompt(2, L)
    w = _model()
    for (_, a), (_, b) in zip(m.named_modules(), list(w.named_modules())):
        if isinstance(a, Fp8Linear):
            b.weight = torch.nn.Parameter(dequantize_fp8(*a.weights(), a.out_features, a.in_features))
    with torch.no_grad():
        got = []
        for model in (m, w):
            cache = [CausalBlockCache() for _ in model.layers]
            h = model._hidden(ids, None, [0.88, 0.88], cache)
            st = InferenceState(torch.full((2,), L, device="cuda"))
            st.step = 1
            got.append((model.lm_head(model.norm(h, model.lm_head)).float(),
                        model.step(ids[:, 0], cache, st, _gen()).float()))
    for a, b in zip(*got):
        off = float((a - b).norm() / b.norm())
        assert 0 < off <= 0.32


@pytest.mark.gpu
def test_scores_and_gradients():
    """score() over quantised layers, and a gradient through them to the embedding: norm
    and layer as tensors, the layer's part the formula's dy W."""
    m, ids = _model().quantize_fp8(), _prompt(2, 70)
    with torch.no_grad():
        plain = m.score(ids)
    assert torch.isfinite(plain.logprob).all() and (plain.logprob <= 0).all()
    ssm, norm = m.layers[0].ssm, m.layers[0].norm1
    h = m.embedding(ids)                                  # (the embedding takes a gradient)
    (g,) = torch.autograd.grad(ssm(norm(h, ssm))[0].float().square().sum(), m.embedding.weight)
    assert torch.isfinite(g).all() and g.abs().max() > 0
    x = _rand(5, 256).cuda().requires_grad_()
    dy = _rand(5, 500, seed=2).cuda()
    (dx,) = torch.autograd.grad(m.lm_head(x), x, dy)
    want = dy.float() @ dequantize_fp8(*m.lm_head.weights(), 500, 256).float()
    assert (dx.float() - want).abs().max() <= 2.0 ** -8 * want.abs().max() + 1e-4


@pytest.mark.gpu
def test_seq2seq_generates():
    cfg = Seq2SeqLMConfig(vocab_size=300, model_dim=128, head_dim=64, ssm_state_dim=64, ssm_chunk_size=64,
                          num_layers=1, dropout_rate=0.0, device="cuda")
    torch.manual_seed(0)
    m = Seq2SeqLM(cfg).to_bf16().cuda().eval().quantize_fp8()
    assert not any(isinstance(x, torch.nn.Linear) for x in m.modules())
    gen = GenerationConfig(bos_token_id=0, eos_token_id=1, pad_token_id=2, max_new_tokens=12, kv_cache_dtype="fp8")
    ids = _prompt(2, 60)
    a = m.generate(ids, gen)
    assert torch.equal(a, m.generate(ids, gen, use_graph=False)) and a.shape == (2, 12)


@pytest.mark.gpu
def test_training_and_ragged_prompts():
    """In training the layers take tensors and pass their gradient on; a padded prompt's
    rows stay finite whatever stands behind their lengths, and padding changes nothing
    before them."""
    m, ids = _model().quantize_fp8(), _prompt(2, 70)
    lengths = torch.tensor([70, 33], device="cuda")
    m.train()
    y = m(ids, lengths=lengths)
    y.float().logsumexp(-1).sum().backward()
    g = m.embedding.weight.grad
    assert torch.isfinite(y).all() and torch.isfinite(g).all() and g.abs().max() > 0
    m.eval()
    other = ids.clone()
    other[1, 33:] = 7
    with torch.no_grad():
        a, b = m(ids, lengths=lengths), m(other, lengths=lengths)
    assert torch.isfinite(a).all() and torch.equal(a[0], b[0]) and torch.equal(a[1, :33], b[1, :33])
