"""Decoding on the GPU from 8-bit caches, with scores, through the model's public calls."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _model(**kw):
    from hippolm_b200.config import HippoConfig
    from hippolm_b200.models.model import HippoModel
    base = dict(vocab_size=4096, hidden_size=512, num_heads=4, head_dim=128, num_layers=4, num_blocks=2, intermediate_size=1024,
                full_attn_interval=2)
    base.update(kw)
    return HippoModel(HippoConfig(**base), device="cuda", dtype=torch.bfloat16, seed=5).eval()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("kw", [dict(), dict(head_dim=64, num_heads=8)])
def test_decoding_from_8_bit_caches_follows_the_16_bit_ones(kind, kw):
    """The same tokens through both caches: keys and values rounded to 8 bits move the logits by little."""
    from hippolm_b200.ops import _ext
    _ext.clear_device_status()
    m = _model(**kw)
    g = torch.Generator(device="cuda").manual_seed(0)
    lens = [37, 1, 130]
    prompts = [torch.randint(0, 4096, (n,), device="cuda", generator=g) for n in lens]
    cu = torch.tensor([0, 37, 38, 168], dtype=torch.int32, device="cuda")
    cu1 = torch.arange(4, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        both = [m.new_decode_caches(200, 3, kv_cache=k) for k in (None, kind)]
        got = [m.hidden(torch.cat(prompts), cu_seqlens=cu, caches=c) for c in both]
        for step in range(5):
            nxt = torch.randint(0, 4096, (3,), device="cuda", generator=g)
            pos = torch.tensor(lens, device="cuda") + step
            got = [m.hidden(nxt, cu_seqlens=cu1, kda_states=s, caches=c, position_offset=pos) for (_, s), c in zip(got, both)]
            a, b = (m.lm_head.logits(h).float() for h, _ in got)
            assert torch.isfinite(b).all() and float(F.cosine_similarity(a, b, dim=-1).min()) > 0.99, step
    torch.cuda.synchronize()
    assert _ext.device_status()[0] == 0


@pytest.mark.parametrize("kind", [None, "int8", "e4m3"])
def test_generation_with_scores(kind):
    m = _model()
    g = torch.Generator(device="cuda").manual_seed(1)
    prompts = [torch.randint(0, 4096, (n,), device="cuda", generator=g) for n in (20, 3, 64)]
    limits = [7, 12, 1]
    seqs, scores = m.generate_batch(prompts, limits, kv_cache=kind, logprobs=5)
    again = m.generate_batch(prompts, limits, kv_cache=kind)
    for p, lim, s, sc, a in zip(prompts, limits, seqs, scores, again):
        assert s.tolist() == a.tolist() and s.numel() == p.numel() + lim
        new = s[p.numel():]
        assert sc.logprob.shape == (lim,) and sc.top_ids.shape == (lim, 5)
        hit = sc.top_ids == new[:, None]                                      # greedy: the token is among those that tie for the top
        assert bool(hit.any(1).all()) and torch.equal(sc.top_logprobs[:, 0], sc.logprob)
        assert bool((sc.entropy > 0).all())
    text = torch.cat(prompts)
    cu = torch.tensor([0, 20, 23, 87], dtype=torch.int32, device="cuda")
    got = m.token_logprobs(text, cu_seqlens=cu, top_k=3, chunk_rows=50)
    lp = torch.log_softmax(m(text, cu_seqlens=cu)["logits"].float(), -1)
    for s, e in ((0, 20), (20, 23), (23, 87)):
        want = lp[s:e - 1].gather(1, text[s + 1:e, None])[:, 0]
        # the same bf16 logits but for the row tiling of the head product: a bf16 step of the logits
        assert float((got.logprob[s + 1:e] - want).abs().max()) < 0.05 and float(got.logprob[s]) == 0.0
