"""The 8-bit cache, the 4-bit layers and the token log probabilities together, as
the models use them: SelectiveMHA's cache object, CausalLM.generate and score,
Seq2SeqLM.generate."""
import math

import pytest
import torch

from oracle import kv_fp8 as kv_ref
from oracle import logprobs as lp_ref
from selective_attention.inference import (CausalBlockCache, GenerationConfig, InferenceState,
                                           SelectiveAttnCache)
from selective_attention.models import CausalLM, CausalLMConfig
from selective_attention.modules import Int4Linear
from selective_attention.ops import (PagedSelectiveAttnCache, PagedSelectiveAttnCacheFP8,
                                     dequantize_int4)

INF = math.inf


# --- the cache object: bookkeeping on the CPU ------------------------------------
def test_cache_refuses():
    with pytest.raises(ValueError):
        PagedSelectiveAttnCacheFP8(1, 2, 96, 100, "cpu")
    with pytest.raises(ValueError):
        PagedSelectiveAttnCacheFP8(1, 2, 64, 100, "cpu", page_size=32)
    with pytest.raises(ValueError):
        SelectiveAttnCache(kv_dtype="int8")
    c = PagedSelectiveAttnCacheFP8(2, 2, 64, 100, "cpu")
    k = torch.zeros(2, 2, 10, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):           # no CPU path
        c.build(k, k, torch.zeros(2, 2, 10))
    with pytest.raises(ValueError):
        c.build(k, k, torch.zeros(2, 2, 9))
    with pytest.raises(ValueError):
        c.append(k[:, :, 0], k[:, :1, 0], torch.zeros(2, 2))
    with pytest.raises(RuntimeError):         # nothing to take back
        c.unappend()


def test_cache_growth_keeps_its_pages():
    c = PagedSelectiveAttnCacheFP8(1, 2, 64, 64, "cpu", grow=True)
    c.k_pages.view(torch.uint8).fill_(7)
    c.k_scale.fill_(4.0)
    first = c._alloc()
    more = [c._alloc() for _ in range(3)]
    assert c.k_pages.shape[0] == 4 and len({first, *more}) == 4
    assert (c.k_pages[:1].view(torch.uint8) == 7).all() and (c.k_scale[0] == 4.0).all()
    assert c.k_pages.dtype == torch.float8_e4m3fn and c.v_pages.shape[0] == 4
    assert (c.gate_pages == -INF).all() and not c.k_pages[1:].view(torch.uint8).any()


def test_generation_config_names_the_cache():
    cfg = GenerationConfig(bos_token_id=0, eos_token_id=1, pad_token_id=2, kv_cache_dtype="fp8")
    c = CausalBlockCache(reserve=4, kv_dtype=cfg.kv_cache_dtype)
    assert c.attn_cache.kv_dtype == "fp8"
    assert CausalBlockCache().attn_cache.kv_dtype == "bf16"


# --- the cache object on the GPU -------------------------------------------------
def _step_inputs(b, H, D, L, seed):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(b, H, L, D, generator=g).to(torch.bfloat16)
    v = torch.randn(b, H, L, D, generator=g).to(torch.bfloat16)
    lg = -torch.rand(b, H, L, generator=g)
    lg[torch.rand(b, H, L, generator=g) < 0.2] = -INF
    q = torch.randn(b, H, D, generator=g).to(torch.bfloat16)
    return k, v, lg, q


def _want(rows, q):
    out = torch.zeros(len(rows), len(rows[0]), q.shape[-1], dtype=torch.float64)
    for r, row in enumerate(rows):
        for h, c in enumerate(row):
            k, v = c.keys_values()
            out[r, h] = kv_ref.attend(q[r, h], k, v, torch.tensor(c.g, dtype=torch.float64))
    return out


def _close(o, want):
    """Weights and the result in bf16 (2^-8 each, |v| < 5 weighted by p), fp32 scores."""
    err = (o.double().cpu() - want).abs().max()
    assert err <= 2 * 2.0 ** -8 * 5.0, float(err)


@pytest.mark.gpu
@pytest.mark.parametrize("device_mode", [False, True])
def test_cache_object(device_mode):
    """build, append over a block's end, unappend, compaction and attend."""
    b, H, D, ps, lens = 3, 2, 64, 64, [62, 64, 5]
    k, v, lg, q = _step_inputs(b, H, D, 200, seed=1)
    c = PagedSelectiveAttnCacheFP8(b, H, D, 70, "cuda", page_size=ps, grow=True)
    rows = [[kv_ref.CacheRef(ps, True) for _ in range(H)] for _ in range(b)]

    def note(i, t):
        for h in range(H):
            rows[i][h].append(k[i, h, t], v[i, h, t], lg[i, h, t])
    c.build(k[:, :, :64].cuda(), v[:, :, :64].cuda(), lg[:, :, :64].cuda(), torch.tensor(lens))
    for i, n in enumerate(lens):
        for t in range(n):
            note(i, t)
    with pytest.raises(RuntimeError):
        c.unappend([1])                       # its block is rounded, no open one stands
    if device_mode:
        c.enter_device_mode(80)
        with pytest.raises(RuntimeError):
            c.unappend()
    for s in range(70):
        t = 100 + s
        c.append(k[:, :, t].cuda(), v[:, :, t].cuda(), lg[:, :, t].cuda())
        if s % 9 == 4:                        # taken back, and appended again
            c.unappend()
            c.append(k[:, :, t].cuda(), v[:, :, t].cuda(), lg[:, :, t].cuda())
        for i in range(b):
            note(i, t)
        if s in (0, 1, 30, 69):
            _close(c.attend(q.cuda()), _want(rows, q))
    if device_mode:
        c.exit_device_mode()
    assert c.lens == [n + 70 for n in lens]
    _close(c.attend(q.cuda()), _want(rows, q))


@pytest.mark.gpu
def test_unappend_over_a_blocks_end_is_refused():
    b, H, D, ps = 1, 2, 64, 64
    k, v, lg, q = _step_inputs(b, H, D, 70, seed=2)
    c = PagedSelectiveAttnCacheFP8(b, H, D, 200, "cuda", page_size=ps)
    for t in range(65):
        c.append(k[:, :, t].cuda(), v[:, :, t].cuda(), lg[:, :, t].cuda())
    c.unappend()                              # 64: the rounded block alone
    rows = [[kv_ref.CacheRef(ps, True) for _ in range(H)]]
    for h in range(H):
        for t in range(64):
            rows[0][h].append(k[0, h, t], v[0, h, t], lg[0, h, t])
    _close(c.attend(q.cuda()), _want(rows, q))
    with pytest.raises(RuntimeError):         # 63: its tokens in bf16 are gone
        c.unappend()
    assert c.lens == [64]


@pytest.mark.gpu
def test_dropped_pages_leave_the_open_block():
    b, H, D, ps = 2, 2, 64, 64
    k, v, lg, q = _step_inputs(b, H, D, 200, seed=3)
    lg[0, :, :64] = -INF                      # row 0 drops its first page
    c = PagedSelectiveAttnCacheFP8(b, H, D, 220, "cuda", page_size=ps)
    c.build(k[:, :, :150].cuda(), v[:, :, :150].cuda(), lg[:, :, :150].cuda())
    before = c.attend(q.cuda())
    assert c.drop_evicted_pages() == 1 and c.lens == [86, 150]
    assert torch.equal(c.attend(q.cuda()), before)
    for t in (150, 151):
        c.append(k[:, :, t].cuda(), v[:, :, t].cuda(), lg[:, :, t].cuda())
    c.unappend()
    rows = [[kv_ref.CacheRef(ps, True) for _ in range(H)] for _ in range(b)]
    for r in range(b):
        for h in range(H):
            for t in range(64 if r == 0 else 0, 151):
                rows[r][h].append(k[r, h, t], v[r, h, t], lg[r, h, t])
    _close(c.attend(q.cuda()), _want(rows, q))


# --- the models ------------------------------------------------------------------
def _model(seed=0, **kw):
    cfg = CausalLMConfig(vocab_size=300, model_dim=128, head_dim=64, ssm_state_dim=64,
                         ssm_chunk_size=64, num_layers=2, dropout_rate=0.0, device="cuda")
    torch.manual_seed(seed)
    m = CausalLM(cfg)
    with torch.no_grad():
        for blk in m.layers:
            blk.mha.score_std_ema.fill_(1.0)
    return m.to_bf16().cuda().eval()


def _gen(**kw):
    return GenerationConfig(bos_token_id=0, eos_token_id=1, pad_token_id=2, max_new_tokens=20,
                            attn_gate_thresholds=[0.88, 0.88], **kw)


def _prompt(b=3, L=120):
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(3, 300, (b, L), generator=g)
    ids[1, 100:] = 2                          # a padded row
    return ids.cuda()


@pytest.mark.gpu
def test_score_is_the_logits_log_softmax():
    m, ids = _model(), _prompt()
    lens = torch.tensor([120, 100, 1], device="cuda")
    with torch.no_grad():
        s = m.score(ids, lens, [0.88, 0.88], top=5)
        logits = m(ids, lens, [0.88, 0.88])
    assert s.logprob.shape == (3, 119) and s.top_ids.shape == (3, 119, 5)
    for r, n in enumerate(lens.tolist()):
        t = torch.full((119,), -100)
        t[:n - 1] = ids[r, 1:n].cpu()
        lp, H, top, tl = lp_ref.forward(logits[r, :-1].cpu(), t, 5)
        assert (s.logprob[r].double().cpu() - lp).abs().max() < 1e-4
        assert (s.entropy[r].double().cpu() - H).abs().max() < 1e-3
        assert torch.equal(s.top_ids[r].cpu(), top)
    assert not s.logprob[2].any()


@pytest.mark.gpu
def test_score_as_a_training_loss():
    """Gradients of minus the mean logprob against torch's cross entropy on the
    same logits (fp32; both are sums of the same terms)."""
    cfg = CausalLMConfig(vocab_size=130, model_dim=64, head_dim=32, ssm_state_dim=32,
                         ssm_chunk_size=32, num_layers=1, dropout_rate=0.0, device="cuda")
    torch.manual_seed(0)
    m = CausalLM(cfg).cuda().train()
    ids = torch.randint(0, 130, (2, 40), device="cuda")
    lens = torch.tensor([40, 25], device="cuda")
    state = {k: t.clone() for k, t in m.state_dict().items()}
    s = m.score(ids, lens)
    n = 39 + 24
    (-s.logprob.sum() / n).backward()
    got = {k: p.grad.clone() for k, p in m.named_parameters() if p.grad is not None}
    m.load_state_dict(state)                  # (the score std's running mean moved)
    m.zero_grad()
    logits = m(ids, lens)
    mask = torch.arange(1, 40, device="cuda")[None, :] < lens[:, None]
    loss = torch.nn.functional.cross_entropy(logits[:, :-1][mask], ids[:, 1:][mask])
    loss.backward()
    assert abs(float(loss.detach()) + float(s.logprob.detach().sum()) / n) < 1e-5
    assert set(got) == {k for k, p in m.named_parameters() if p.grad is not None}
    for k, p in m.named_parameters():
        if p.grad is not None:
            scale = float(p.grad.abs().max())
            assert float((got[k] - p.grad).abs().max()) <= 2e-3 * scale + 1e-9, k


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("soft", [False, True])
def test_generate_captured_equals_eager(kv, int4, soft):
    """Tokens, log probabilities and alternatives of the captured decode step are
    the eager step's, and those of the logits that the model gives.  (With the
    head tied to a random embedding one token has all the probability, entropy 0
    in fp32; soft: a tenth of the logits.)"""
    m, ids = _model(), _prompt()
    if soft:
        with torch.no_grad():
            m.norm.weight.fill_(-0.9)
    if int4:
        m.quantize_int4(group_size=64).quantize_int4(group_size=64)     # (the second finds none)
        assert isinstance(m.lm_head, Int4Linear) and isinstance(m.layers[0].mha.q_proj, Int4Linear)
    cfg = _gen(kv_cache_dtype=kv)
    a, la = m.generate(ids, cfg, logprobs=4)
    b, lb = m.generate(ids, cfg, use_graph=False, logprobs=4)
    plain = m.generate(ids, cfg)
    assert torch.equal(a, b) and torch.equal(a, plain)
    assert a.shape == (3, 140) and la.top_ids.shape == (3, 20, 4)
    for x, y in zip(la, lb):
        assert torch.equal(x, y)
    eos_before = (a[:, 119:-1] == cfg.eos_token_id).cumsum(1) > 0
    assert not la.logprob[eos_before].any()
    live = ~eos_before
    assert (la.logprob[live] <= 0).all() and (la.entropy[live] >= 0).all()
    assert not soft or (la.entropy[live] > 0).all()
    assert (la.top_logprobs[..., 0][live] >= la.logprob[live] - 1e-6).all()
    # greedy: the chosen token's probability is the largest, up to the argmax's
    # bf16 softmax (half a step of the probability each: 2 2^-8, and ties)
    assert (la.top_logprobs[..., 0][live] - la.logprob[live] <= 2.0 ** -6).all()


@pytest.mark.gpu
def test_int4_model_is_the_model_of_its_weights():
    """The quantised model's logits against the same model with the bf16 weights
    that the codes stand for: both round every layer's output to bf16, the 4-bit
    kernel keeps scale (code - zero) itself where the other has it rounded."""
    m, ids = _model(), _prompt(2, 40)
    m.quantize_int4(group_size=32, symmetric=False)
    w = _model()
    for (_, a), (_, b) in zip(m.named_modules(), list(w.named_modules())):
        if isinstance(a, Int4Linear):
            b.weight = torch.nn.Parameter(dequantize_int4(*a.weights(), a.out_features, a.in_features))
    cfg = _gen()
    with torch.no_grad():
        state = [InferenceState(torch.full((2,), 40, device="cuda")) for _ in range(2)]
        got = []
        for model, st in ((m, state[0]), (w, state[1])):
            cache = [CausalBlockCache() for _ in model.layers]
            h = model._hidden(ids, None, [0.88, 0.88], cache)
            pre = model.lm_head(model.norm(h))
            st.step = 1
            got.append((pre, model.step(ids[:, 0], cache, st, cfg)))
    for a, b, name in zip(got[0], got[1], ("prompt", "step")):
        scale = float(b.float().abs().max())
        # the prompts run the same products (the widened weights); a step's differ
        # by the weights' rounding, 2^-9 of each at random, through 2 blocks
        assert float((a.float() - b.float()).abs().max()) <= (0.0 if name == "prompt" else 3e-2) * scale, name


@pytest.mark.gpu
def test_fp8_cache_step_near_bf16():
    """One decode step over both caches after the same prompt."""
    m, ids = _model(), _prompt(2, 150)
    out = []
    for kv in ("bf16", "fp8"):
        cache = [CausalBlockCache(kv_dtype=kv) for _ in m.layers]
        with torch.no_grad():
            m._hidden(ids, None, [0.88, 0.88], cache)
            st = InferenceState(torch.full((2,), 150, device="cuda"))
            st.step = 1
            out.append(m.step(ids[:, 0], cache, st, _gen()).float())
        assert isinstance(cache[0].attn_cache.pages,
                          PagedSelectiveAttnCacheFP8 if kv == "fp8" else PagedSelectiveAttnCache)
    # keys and values off by at most 2^-4 of themselves each, averaged over the keys
    scale = float(out[0].abs().max())
    assert 0 < float((out[0] - out[1]).abs().max()) <= 2.0 ** -4 * scale


@pytest.mark.gpu
def test_seq2seq_generates_with_both():
    from selective_attention.models import Seq2SeqLM, Seq2SeqLMConfig
    cfg = Seq2SeqLMConfig(vocab_size=300, model_dim=128, head_dim=64, ssm_state_dim=64,
                          ssm_chunk_size=64, num_layers=1, dropout_rate=0.0, device="cuda")
    torch.manual_seed(0)
    m = Seq2SeqLM(cfg).to_bf16().cuda().eval().quantize_int4(group_size=64)
    assert not any(type(x) is torch.nn.Linear for x in m.modules())
    gen = GenerationConfig(bos_token_id=0, eos_token_id=1, pad_token_id=2, max_new_tokens=12,
                           kv_cache_dtype="fp8")
    ids = _prompt(2, 60)
    a = m.generate(ids, gen)
    assert torch.equal(a, m.generate(ids, gen, use_graph=False)) and a.shape == (2, 12)
