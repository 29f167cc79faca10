"""8-bit caches and log probabilities through the model, the server, the evaluation script and tensor-parallel ranks (CPU)."""
import json
import math
import threading
import urllib.error
import urllib.request

import pytest
import torch

import kv8_plain as plain
from hippolm_b200 import ops
from hippolm_b200.config import HippoConfig
from hippolm_b200.data.tokenizer import ByteTokenizer
from hippolm_b200.models import kv_pages
from hippolm_b200.models.model import HippoModel
from hippolm_b200.ref import kv8 as ref
from hippolm_b200.serve.eval_server import EvalService, serve

BASE = dict(vocab_size=96, hidden_size=32, num_heads=2, head_dim=16, num_layers=4, num_blocks=2, intermediate_size=64, full_attn_interval=2)


def model(**kw):
    torch.manual_seed(0)
    return HippoModel(HippoConfig(**dict(BASE, **kw)), seed=4).eval()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("kw", [dict(), dict(use_short_conv=True)])
def test_cached_keys_and_values_are_the_layers_own(kind, kw, monkeypatch):
    """Every attention call of a batched decode sees, for every sequence that still runs, all keys and values of its tokens in order,
    rounded to codes; sequences that are done see none, and their blocks are free again."""
    m = model(**kw)
    prompts = [torch.randint(0, 96, (n,)) for n in (1, 70, 12, 64, 3)]
    limits = [6, 3, 8, 2, 0]
    hist, calls = {}, []
    write, attend, plan = ops.kv8_write, ops.attention_decode_kv8, ops.kv8_plan
    per_pass = {}

    def on_plan(table, lens, new, *a, **k):
        p = plan(table, lens, new, *a, **k)
        per_pass.update(new=new.tolist(), served=p.served.tolist(), table=table)
        return p

    def on_write(k, v, slots, codes, scales):
        write(k, v, slots, codes, scales)
        rows, at = hist.setdefault(codes.data_ptr(), [[] for _ in prompts]), 0
        for n, c in enumerate(per_pass["new"]):
            if per_pass["served"][n]:
                rows[n] += [(k[at + i], v[at + i]) for i in range(c)]
            at += c

    def on_attend(q, codes, scales, table, lens, scale):
        for n, rows in enumerate(hist[codes.data_ptr()]):
            ln = int(lens[n])
            assert ln == (len(rows) if per_pass["served"][n] else 0), n
            if ln == 0:
                continue
            for got, want in zip(ref.gather(codes, scales, table[n, :-(-ln // 64)], ln), zip(*rows)):
                want = torch.stack(want)
                size = torch.stack([x.abs().amax((0, 2)) for x in want.split(64)]).repeat_interleave(64, 0)[:ln]     # of a block and head
                # int8: half a step of at most 2 / 127 of the block's largest, twice (codes may be rounded anew as it fills);
                # e4m3: half of 2^-3 of the value, twice, or of the subnormals' step
                tol = size[..., None] * (2 / 127) if kind == "int8" else want.abs() * 2 * 2.0 ** -4 + size[..., None] * 2.0 ** -15
                assert bool(((got - want).abs() <= tol).all())
        calls.append(lens.tolist())
        return attend(q, codes, scales, table, lens, scale)

    monkeypatch.setattr(kv_pages.ops, "kv8_plan", on_plan)
    monkeypatch.setattr(kv_pages.ops, "kv8_write", on_write)
    monkeypatch.setattr(kv_pages.ops, "attention_decode_kv8", on_attend)
    out = m.generate_batch(prompts, limits, kv_cache=kind)
    assert [o.numel() for o in out] == [p.numel() + lim for p, lim in zip(prompts, limits)]
    assert len(calls) == 2 * 7 and calls[0] == [2, 71, 13, 65, 0] and calls[-1] == [0, 0, 19, 0, 0]


def test_pages_hold_what_the_limits_need():
    pages = kv_pages.KV8Pages([130, 0, 64, 1], block_size=64)
    assert pages.blocks == 3 + 0 + 1 + 1
    cu = torch.tensor([0, 100, 103, 167, 168], dtype=torch.int32)
    pages.release = torch.tensor([False, True, False, False])
    pages.plan(cu, 168)
    assert pages.lens.tolist() == [100, 0, 64, 1] and pages.slots[100:103].tolist() == [-1] * 3 and int(pages.free_count) == 1
    pages.release = torch.tensor([False, True, True, True])
    for i in range(30):
        pages.plan(torch.arange(5, dtype=torch.int32), 4)
    assert pages.lens.tolist() == [130, 0, 0, 0] and int(pages.free_count) == 2 and int(pages.slots[0]) >= 0
    used = pages.table[0, :3].tolist()
    assert sorted(used + pages.free[:2].tolist()) == list(range(5))


@pytest.mark.parametrize("kind", [None, "int8", "e4m3"])
def test_scores_of_generated_tokens(kind):
    m = model()
    prompts = [torch.randint(0, 96, (n,)) for n in (5, 9)]
    seqs, scores = m.generate_batch(prompts, [4, 6], logprobs=3, kv_cache=kind)
    again = m.generate_batch(prompts, [4, 6], kv_cache=kind)
    for p, s, sc, a in zip(prompts, seqs, scores, again):
        n = s.numel() - p.numel()
        assert s.tolist() == a.tolist() and sc.logprob.shape == (n,) and sc.top_ids.shape == (n, 3)
        assert sc.top_ids[:, 0].tolist() == s[p.numel():].tolist()            # greedy: the likeliest token
        assert torch.equal(sc.top_logprobs[:, 0], sc.logprob)
        if kind is None:                                                       # fp32 both ways: the full forward's distribution
            lp = torch.log_softmax(m(s)["logits"].float(), -1)[p.numel() - 1:-1]
            assert torch.allclose(sc.logprob, lp.gather(1, s[p.numel():, None])[:, 0], atol=2e-4)
            assert torch.allclose(sc.entropy, -(lp.exp() * lp).sum(-1), atol=2e-3)
    none, empty = m.generate_batch(prompts, 0, logprobs=2)
    assert [x.numel() for x in none] == [5, 9] and empty[0].top_ids.shape == (0, 2)
    assert m.generate_batch([], 3, logprobs=1) == ([], [])
    for bad in (-1, 33):
        with pytest.raises(ValueError):
            m.generate_batch(prompts, 2, logprobs=bad)
    with pytest.raises(ValueError):
        m.generate_batch(prompts, 2, kv_cache="int4")


def test_model_scores_of_packed_text():
    m = model()
    lens = [7, 1, 12]
    ids = torch.randint(0, 96, (20,))
    cu = torch.tensor([0, 7, 8, 20], dtype=torch.int32)
    got = m.token_logprobs(ids, cu_seqlens=cu, top_k=2, chunk_rows=6)
    at = 0
    for ln in lens:
        lp = torch.log_softmax(m(ids[at:at + ln])["logits"].float(), -1)
        assert float(got.logprob[at]) == 0.0
        assert torch.allclose(got.logprob[at + 1:at + ln], lp[:-1].gather(1, ids[at + 1:at + ln, None])[:, 0], atol=2e-4)
        assert torch.allclose(got.top_logprobs[at + 1:at + ln], lp[:-1].topk(2, -1).values, atol=2e-4)
        at += ln
    rows = m.token_logprobs(ids.view(2, 10))
    assert rows.top_ids is None and float(rows.logprob[10]) == 0.0 and rows.logprob.shape == (20,)


def small_service(**kw):
    cfg = HippoConfig(vocab_size=258, hidden_size=32, num_heads=2, head_dim=16, num_layers=2, num_blocks=1, intermediate_size=64,
                      full_attn_interval=2)
    return EvalService(HippoModel(cfg, seed=1).eval(), ByteTokenizer(), max_new_tokens=6, **kw)


@pytest.mark.parametrize("kv_cache", [None, "int8"])
def test_server_answers_with_log_probabilities(kv_cache):
    svc = small_service(kv_cache=kv_cache)
    srv = serve(svc, port=0)
    url = f"http://127.0.0.1:{srv.server_address[1]}/v1/"

    def post(path, body):
        req = urllib.request.Request(url + path, json.dumps(body).encode(), {"Content-Type": "application/json"})
        with urllib.request.urlopen(req, timeout=60) as r:
            return json.loads(r.read())["choices"][0]

    c = post("completions", {"prompt": "hello", "max_tokens": 5, "logprobs": 4})
    lp = c["logprobs"]
    assert len(lp["tokens"]) == len(lp["token_logprobs"]) == len(lp["top_logprobs"]) == len(lp["text_offset"]) >= 1
    assert all(x <= 0 and max(t.values()) == pytest.approx(x) for x, t in zip(lp["token_logprobs"], lp["top_logprobs"]))
    assert "".join(lp["tokens"]) == c["text"] or any(ord(ch) > 127 for ch in c["text"])
    plain_c = post("completions", {"prompt": "hello", "max_tokens": 5})
    assert plain_c["text"] == c["text"] and "logprobs" not in plain_c
    zero = post("completions", {"prompt": "hello", "max_tokens": 5, "logprobs": 0})["logprobs"]
    assert zero["token_logprobs"] == lp["token_logprobs"] and zero["top_logprobs"] is None
    chat = post("chat/completions", {"messages": [{"role": "user", "content": "hi"}], "max_tokens": 3, "logprobs": True, "top_logprobs": 2})
    item = chat["logprobs"]["content"][0]
    assert len(item["top_logprobs"]) == 2 and item["logprob"] == pytest.approx(item["top_logprobs"][0]["logprob"]) and item["bytes"]
    for path, body in (("completions", {"prompt": "a", "logprobs": 33}), ("completions", {"prompt": "a", "logprobs": "x"}),
                       ("completions", {"prompt": "a", "logprobs": True}),
                       ("chat/completions", {"messages": [], "top_logprobs": 2}), ("chat/completions", {"messages": [], "logprobs": True, "top_logprobs": -1})):
        with pytest.raises(urllib.error.HTTPError) as e:
            post(path, body)
        assert e.value.code == 400
    srv.shutdown()
    svc.close()


def test_requests_with_and_without_log_probabilities_share_a_pass():
    svc = small_service(max_batch=8)
    bodies = [{"prompt": "ab", "max_tokens": 4}, {"prompt": "abc", "max_tokens": 3, "logprobs": 2}, {"prompt": "x", "max_tokens": 5, "logprobs": 5}]
    alone = [svc.complete(b, chat=False)["choices"][0] for b in bodies]
    got = [None] * 3
    with svc.lock:
        ts = [threading.Thread(target=lambda i=i: got.__setitem__(i, svc.complete(bodies[i], chat=False)["choices"][0])) for i in range(3)]
        for t in ts:
            t.start()
    for t in ts:
        t.join(timeout=60)
    for a, g in zip(alone, got):
        assert a["text"] == g["text"] and ("logprobs" in a) == ("logprobs" in g)
        if "logprobs" in a:
            assert a["logprobs"]["token_logprobs"] == pytest.approx(g["logprobs"]["token_logprobs"], abs=2e-4)
            assert [len(t) for t in a["logprobs"]["top_logprobs"]] == [len(t) for t in g["logprobs"]["top_logprobs"]]
    svc.close()


def test_token_scores_of_documents(tmp_path):
    from hippolm_b200.serve.perplexity import evaluate_perplexity, score_documents
    cfg = HippoConfig(vocab_size=258, hidden_size=32, num_heads=2, head_dim=16, num_layers=2, num_blocks=1, intermediate_size=64,
                      full_attn_interval=2)
    m, tok = HippoModel(cfg, seed=1), ByteTokenizer()
    docs = ["some words to score", "b", "a longer document that is cut in pieces " * 5]
    rows = list(score_documents(m, tok, docs, seq_len=64, batch_tokens=50, top_logprobs=2))
    lp = [x for r in rows for x in r["logprobs"] if x is not None]
    want = evaluate_perplexity(m, tok, docs, seq_len=64)
    assert len(lp) == want["tokens"] and -sum(lp) / len(lp) == pytest.approx(want["nll"], abs=1e-4)
    assert m.training and [r["document"] for r in rows] == sorted(r["document"] for r in rows)
    for r in rows:
        assert r["logprobs"][0] is None and len(r["tokens"]) == len(r["entropy"]) == len(r["top_tokens"])
        assert all(len(t) == 2 for t in r["top_tokens"][1:]) and all(0 <= e <= math.log(258) + 1e-4 for e in r["entropy"][1:])


def test_scores_of_no_text_and_of_a_few_rows():
    from hippolm_b200.serve.perplexity import score_documents
    m = model()
    got = m.token_logprobs(torch.empty(0, dtype=torch.long), top_k=3)
    assert got.logprob.shape == got.entropy.shape == (0,) and got.top_ids.shape == got.top_logprobs.shape == (0, 3)
    cfg = HippoConfig(vocab_size=258, hidden_size=32, num_heads=2, head_dim=16, num_layers=2, num_blocks=1, intermediate_size=64,
                      full_attn_interval=2)
    m = HippoModel(cfg, seed=1)
    rows = score_documents(m, ByteTokenizer(), ["one text", "another"], batch_tokens=4)
    assert next(rows)["document"] == 0
    rows.close()                                                               # what stops early leaves the model as it was
    assert m.training


def test_requests_served_one_by_one_have_the_same_answers():
    body = {"prompt": "abc", "max_tokens": 4, "logprobs": 2}
    want, got = small_service(kv_cache="int8"), small_service(kv_cache="int8")
    got._batched = False
    for b in (body, {"prompt": "abc", "max_tokens": 4}):
        assert got.complete(b, chat=False)["choices"] == want.complete(b, chat=False)["choices"]
    want.close()
    got.close()


def _tp_worker(rank, world, port, out_path):
    import os
    os.environ.update({"RANK": str(rank), "WORLD_SIZE": str(world), "LOCAL_RANK": str(rank), "MASTER_ADDR": "127.0.0.1",
                       "MASTER_PORT": str(port), "HIPPO_TP_SIM": "1"})
    torch.set_num_threads(1)
    from hippolm_b200.parallel.mesh import init_distributed_from_env, init_mesh
    init_distributed_from_env(backend="gloo")
    init_mesh(tp=world)
    m = model()
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, 96, (n,), generator=g) for n in (5, 2, 8)]
    seqs, scores = m.generate_batch(prompts, [4, 6, 3], kv_cache="int8", logprobs=2)
    packed = torch.cat(prompts + [torch.zeros(1, dtype=torch.long)])
    text = m.token_logprobs(packed, cu_seqlens=torch.tensor([0, 5, 7, 15, 16], dtype=torch.int32))
    torch.save({"seqs": [s.tolist() for s in seqs], "lp": [s.logprob.tolist() for s in scores], "text": text.logprob.tolist()}, out_path + f".{rank}")
    import torch.distributed as dist
    dist.barrier()
    dist.destroy_process_group()


def test_tensor_parallel_ranks_decode_from_8_bit_caches(tmp_path):
    import torch.multiprocessing as mp
    from test_context_parallel import _free_port
    out = str(tmp_path / "tp")
    mp.spawn(_tp_worker, args=(2, _free_port(), out), nprocs=2, join=True)
    a, b = torch.load(out + ".0"), torch.load(out + ".1")
    assert a == b
    m = model()
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, 96, (n,), generator=g) for n in (5, 2, 8)]
    seqs, scores = m.generate_batch(prompts, [4, 6, 3], kv_cache="int8", logprobs=2)
    assert [s.tolist() for s in seqs] == a["seqs"]                            # heads do not share a block: the same codes on one rank
    for s, lp in zip(scores, a["lp"]):
        assert torch.allclose(s.logprob, torch.tensor(lp), atol=1e-3)
    assert len(a["text"]) == 16 and a["text"][0] == a["text"][5] == 0.0


def scorer(**kw):
    cfg = HippoConfig(vocab_size=258, hidden_size=32, num_heads=2, head_dim=16, num_layers=2, num_blocks=1, intermediate_size=64,
                      full_attn_interval=2, **kw)
    return HippoModel(cfg, seed=1).eval()


def passes_of(m, monkeypatch):
    """The token counts of a model's scoring passes, as they happen."""
    sizes, call = [], m.token_logprobs

    def on_call(ids, **k):
        sizes.append(ids.numel())
        return call(ids, **k)
    monkeypatch.setattr(m, "token_logprobs", on_call)
    return sizes


def test_scoring_a_long_document_runs_in_bounded_passes(monkeypatch):
    from hippolm_b200.serve.perplexity import score_documents
    m = scorer()
    sizes = passes_of(m, monkeypatch)
    doc = "".join(chr(97 + i % 26) for i in range(2999))
    rows = list(score_documents(m, ByteTokenizer(), [doc, "short", doc[:700]], seq_len=64, batch_tokens=256))
    assert max(sizes) < 256 + 64 and sum(sizes) == 3000 + 6 + 701
    assert [t for r in rows if r["document"] == 0 for t in r["tokens"]] == list(doc.encode()) + [256]


def test_scoring_stops_inside_a_long_document(monkeypatch):
    from hippolm_b200.serve.perplexity import score_documents
    m = scorer()
    sizes = passes_of(m, monkeypatch)
    rows = list(score_documents(m, ByteTokenizer(), ["x" * 4000, "y" * 4000], seq_len=64, batch_tokens=256, max_tokens=300))
    scored = sum(len(r["tokens"]) - 1 for r in rows)
    assert 300 <= scored < 300 + 64 and sum(sizes) == sum(len(r["tokens"]) for r in rows)
    assert all(r["document"] == 0 for r in rows)


@pytest.mark.parametrize("seq_len", [100, 64, 10, 200])
def test_token_scores_and_perplexity_cut_documents_alike(seq_len):
    from hippolm_b200.serve.perplexity import evaluate_perplexity, score_documents
    m, tok = scorer(), ByteTokenizer()
    docs = ["".join(chr(97 + (i * i + k) % 26) for i in range(n)) for k, n in enumerate((333, 20, 64, 150))]
    rows = list(score_documents(m, tok, docs, seq_len=seq_len, batch_tokens=150))
    lp = [x for r in rows for x in r["logprobs"] if x is not None]
    want = evaluate_perplexity(m, tok, docs, seq_len=seq_len)
    assert len(lp) == want["tokens"] and -sum(lp) / len(lp) == pytest.approx(want["nll"], abs=1e-4)


def forced(svc, tokens, monkeypatch):
    """A service whose next answers consist of ``tokens``; token i has log probability -i - 1, its alternatives are itself and 65."""
    n = len(tokens)
    scores = ops.TokenLogprobs(-1.0 - torch.arange(n, dtype=torch.float32), torch.zeros(n),
                               torch.stack([-1.0 - torch.arange(n, dtype=torch.float32), torch.full((n,), -99.0)], 1),
                               torch.tensor([[t, 65] for t in tokens], dtype=torch.int64).reshape(n, 2))
    monkeypatch.setattr(svc, "_generate", lambda *a, **k: (list(tokens), "length") + ((scores,) if "logprobs" in k else ()))
    return svc


@pytest.mark.parametrize("text,offsets", [("ab€", [0, 1, 2, 2, 2]), ("日本", [0, 0, 0, 1, 1, 1]), ("é", [0, 0]), ("日a本b", [0, 0, 0, 1, 2, 2, 2, 3])])
@pytest.mark.parametrize("ends", [False, True])
def test_log_probabilities_of_characters_of_several_tokens(text, offsets, ends, monkeypatch):
    """Every token of the answer has its log probability, also where a character's bytes are tokens of their own."""
    tokens = list(text.encode()) + [256] * ends
    svc = forced(small_service(), tokens, monkeypatch)
    c = svc.complete({"prompt": "x", "logprobs": 2}, chat=False)["choices"][0]
    n = len(text.encode())
    assert c["text"] == text and c["logprobs"]["token_logprobs"] == [-1.0 - i for i in range(n)]
    assert c["logprobs"]["text_offset"] == offsets and len(c["logprobs"]["tokens"]) == len(c["logprobs"]["top_logprobs"]) == n
    chat = svc.complete({"messages": [{"role": "user", "content": "x"}], "logprobs": True, "top_logprobs": 1}, chat=True)["choices"][0]
    assert [x["logprob"] for x in chat["logprobs"]["content"]] == [-1.0 - i for i in range(n)]
    # a stop string ends the list with the tokens of the text before it
    if text == "日a本b":
        for stop, left in (("b", 7), ("本", 4), ("a", 3)):
            c = svc.complete({"prompt": "x", "logprobs": 2, "stop": stop}, chat=False)["choices"][0]
            assert len(c["logprobs"]["tokens"]) == left and c["finish_reason"] == "stop", stop
    svc.close()


def test_no_log_probabilities_before_a_stop_string_at_the_start(monkeypatch):
    svc = forced(small_service(), list("stop it".encode()), monkeypatch)
    c = svc.complete({"prompt": "x", "logprobs": 2, "stop": ["it", "sto"]}, chat=False)["choices"][0]
    assert c["text"] == "" and c["logprobs"]["tokens"] == c["logprobs"]["token_logprobs"] == c["logprobs"]["text_offset"] == []
    chat = svc.complete({"messages": [], "logprobs": True, "stop": "s"}, chat=True)["choices"][0]
    assert chat["message"]["content"] == "" and chat["logprobs"] == {"content": []}
    svc.close()


def test_bytes_of_chat_tokens_are_the_tokens_own(monkeypatch):
    from hippolm_b200.data import bpe
    svc = forced(small_service(), list("aé€".encode()), monkeypatch)
    ask = {"messages": [{"role": "user", "content": "x"}], "logprobs": True, "top_logprobs": 2}
    items = svc.complete(ask, chat=True)["choices"][0]["logprobs"]["content"]
    assert [x["bytes"] for x in items] == [[b] for b in "aé€".encode()]
    assert [[y["bytes"] for y in x["top_logprobs"]] for x in items] == [[[b], [65]] for b in "aé€".encode()]
    svc.close()

    tok = bpe.load_default()
    svc = small_service()
    svc.tok = tok
    text = "some words, 日本 é"
    forced(svc, tok.encode(text), monkeypatch)
    items = svc.complete(ask, chat=True)["choices"][0]["logprobs"]["content"]
    assert b"".join(bytes(x["bytes"]) for x in items).decode() == text
    special = next(iter(tok.special.items()))
    assert tok.token_bytes(special[1]) == special[0].encode() and ByteTokenizer().token_bytes(256) is None and tok.token_bytes(1 << 30) is None
    svc.close()

    class Other(ByteTokenizer):                                               # a tokenizer that does not tell its tokens' bytes
        token_bytes = None
    svc = small_service()
    svc.tok = Other()
    forced(svc, list("aé".encode()), monkeypatch)
    items = svc.complete(ask, chat=True)["choices"][0]["logprobs"]["content"]
    assert [x["bytes"] for x in items] == [[97], None, None]
    svc.close()


def test_caches_that_cannot_be_kept_are_refused_at_once(monkeypatch):
    """A cache type or head size that no pass could use is refused where the cache is asked for, not by the first pass."""
    m = model()
    for call in (lambda: m.generate_batch([], 3, kv_cache="int4"), lambda: m.generate_batch([torch.tensor([1])], 0, kv_cache="fp8"),
                 lambda: m.new_decode_caches(8, 1, kv_cache="int4"), lambda: small_service(kv_cache="int4")):
        with pytest.raises(ValueError, match="int8 or e4m3"):
            call()
    kv_pages.check_cache(None, 96, torch.device("cuda"))
    kv_pages.check_cache("int8", 16, torch.device("cpu"))
    for dim in (64, 128):
        kv_pages.check_cache("e4m3", dim, torch.device("cuda"))
    with pytest.raises(ValueError, match="head_dim 96"):
        kv_pages.check_cache("int8", 96, torch.device("cuda"))
    kv_pages.check_cache("int8", None, torch.device("cuda"))                  # nothing is kept
    seen = []
    monkeypatch.setattr("hippolm_b200.models.model.check_cache", lambda *a: seen.append(a))       # what the model asks, before anything else
    m.new_decode_caches(8, 1, kv_cache="int8")
    assert seen == [("int8", 16, m.norm.weight.device)]
    # a model without full attention keeps no keys, and takes no unknown type either
    monkeypatch.undo()
    with pytest.raises(ValueError):
        model(full_attn_interval=5).new_decode_caches(8, 1, kv_cache="int4")


def test_generate_does_not_ignore_a_cache_type():
    m = model()
    ids = torch.tensor([1, 2, 3])
    for kw in (dict(max_new_tokens=0, kv_cache="int4"), dict(max_new_tokens=2, kv_cache="int4", use_cache=False),
               dict(max_new_tokens=2, kv_cache="int8", use_cache=False)):
        with pytest.raises(ValueError):
            m.generate(ids, **kw)
    assert m.generate(ids, 0, kv_cache="int8").tolist() == [1, 2, 3]
    assert m.generate(ids, 2, use_cache=False).numel() == m.generate(ids, 2, kv_cache="int8").numel() == 5


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_a_refused_pass_leaves_the_pages_as_they_were(kind):
    m = model()
    prompts = [torch.randint(0, 96, (n,)) for n in (5, 9)]
    caches = m.new_decode_caches(40, 2, kv_cache=kind)
    cu = torch.tensor([0, 5, 14], dtype=torch.int32)
    cu1 = torch.arange(3, dtype=torch.int32)
    with torch.no_grad():
        _, st = m.hidden(torch.cat(prompts), cu_seqlens=cu, caches=caches)
        pages = kv_pages.pages_of(caches)
        layers = [c for c in caches if "pages" in c]

        def held():
            return [pages.lens.clone(), pages.free_count.clone(), pages.table.clone()] + [c[k].clone() for c in layers for k in ("codes", "scales")]
        before = held()
        with pytest.raises(ValueError):                                       # three tokens for two sequences
            m.hidden(torch.tensor([1, 2, 3]), cu_seqlens=torch.tensor([0, 2, 3], dtype=torch.int32), kda_states=st, caches=caches)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, held()))
        other = m.new_decode_caches(40, 2, kv_cache=kind)
        _, st2 = m.hidden(torch.cat(prompts), cu_seqlens=cu, caches=other)
        pos, nxt = torch.tensor([5, 9]), torch.tensor([1, 2])
        a, _ = m.hidden(nxt, cu_seqlens=cu1, kda_states=st, caches=caches, position_offset=pos)
        b, _ = m.hidden(nxt, cu_seqlens=cu1, kda_states=st2, caches=other, position_offset=pos)
        assert torch.equal(a, b)


def test_scores_of_documents_that_do_not_cover_the_text_are_refused():
    m = model()
    ids = torch.randint(0, 96, (20,))
    for cu in ([0, 7, 12], [3, 20], [0, 7, 30], [0, 9, 7, 20], [0, -1, 20], [0], []):
        with pytest.raises(ValueError, match="cu_seqlens"):
            m.token_logprobs(ids, cu_seqlens=torch.tensor(cu, dtype=torch.int32))
    with pytest.raises(ValueError, match="cu_seqlens"):
        m.token_logprobs(ids[:0], cu_seqlens=torch.tensor([0, 3], dtype=torch.int32))
    with pytest.raises(ValueError, match="cu_seqlens"):
        m.token_logprobs(ids, cu_seqlens=torch.tensor([0, 20]).float())
    full = m.token_logprobs(ids, cu_seqlens=torch.tensor([0, 7, 20], dtype=torch.int32))
    empty = m.token_logprobs(ids, cu_seqlens=torch.tensor([0, 0, 7, 7, 20, 20]))               # documents without tokens, 64-bit ends
    assert torch.allclose(full.logprob, empty.logprob, atol=1e-4)
    assert m.token_logprobs(ids[:0], cu_seqlens=torch.tensor([0], dtype=torch.int32)).logprob.shape == (0,)


def test_scores_of_a_text_are_refused_before_its_pass(monkeypatch):
    from hippolm_b200.serve.perplexity import score_documents
    m = scorer()
    monkeypatch.setattr(m, "hidden", lambda *a, **k: pytest.fail("the pass ran"))
    ids = torch.arange(8)
    for kw in (dict(top_k=33), dict(top_k=-1), dict(chunk_rows=0), dict(chunk_rows=-4)):
        with pytest.raises(ValueError):
            m.token_logprobs(ids, **kw)
    with pytest.raises(ValueError):
        list(score_documents(m, ByteTokenizer(), ["some text"], top_logprobs=33))


def _eval_args(tmp_path, *more):
    (tmp_path / "c.yml").write_text("vocab_size: 258\nhidden_size: 32\nnum_heads: 2\nhead_dim: 16\nnum_layers: 2\nnum_blocks: 1\n"
                                    "intermediate_size: 64\nfull_attn_interval: 2\n")
    (tmp_path / "d.txt").write_text("a first document\n\nand a second, longer one " + "with words " * 20)
    return ["--config", str(tmp_path / "c.yml"), "--device", "cpu", "--data_files", str(tmp_path / "d.txt"),
            "--work-dir", str(tmp_path / "w"), "--seq_len", "100", *more]


def test_evaluation_script_writes_token_scores_where_no_folder_is_yet(tmp_path):
    from hippolm_b200.serve import eval_driver
    out = tmp_path / "w" / "scores" / "s.jsonl"
    assert eval_driver.main(_eval_args(tmp_path, "--perplexity", "--token_scores", str(out), "--top_logprobs", "2")) == 0
    rows = [json.loads(line) for line in out.read_text().splitlines()]
    lp = [x for r in rows for x in r["logprobs"] if x is not None]
    want = json.loads((tmp_path / "w" / "perplexity.json").read_text())
    assert len(lp) == want["tokens"] and -sum(lp) / len(lp) == pytest.approx(want["nll"], abs=1e-4)
    assert all(len(t) == 2 for r in rows for t in r["top_tokens"][1:])


def test_evaluation_script_refuses_scores_that_it_cannot_write(tmp_path, monkeypatch):
    from hippolm_b200.serve import eval_driver
    out = tmp_path / "s.jsonl"
    out.write_text("kept")
    monkeypatch.setattr("hippolm_b200.serve.eval_server.build_model_and_load", lambda *a: pytest.fail("the model was loaded"))
    monkeypatch.setattr(eval_driver, "server_command", lambda *a: pytest.fail("a server was started"))
    for more in (["--perplexity", "--token_scores", str(out), "--top_logprobs", "33"],
                 ["--perplexity", "--token_scores", str(out), "--top_logprobs", "-1"],
                 ["--perplexity", "--top_logprobs", "2"], ["--token_scores", str(out)]):
        with pytest.raises(SystemExit) as e:
            eval_driver.main(_eval_args(tmp_path, *more))
        assert e.value.code not in (0, None), more
    assert out.read_text() == "kept"


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_sequences_beyond_their_limit_are_refused(kind):
    """The pool holds what the limits need: what goes beyond had no block, and was left out of the attention without a word."""
    m = model()
    cu1 = torch.arange(3, dtype=torch.int32)
    cu = torch.tensor([0, 60, 66], dtype=torch.int32)
    ids = torch.randint(0, 96, (66,))
    with torch.no_grad():
        with pytest.raises(ValueError, match="sequence 1"):
            m.hidden(ids, cu_seqlens=cu, caches=m.new_decode_caches(64, 2, kv_cache=kind, limits=[64, 5]))
        with pytest.raises(ValueError, match="1 sequences"):
            m.hidden(ids, cu_seqlens=cu[::2], caches=m.new_decode_caches(64, 2, kv_cache=kind))
        caches = m.new_decode_caches(64, 2, kv_cache=kind, limits=[64, 64])
        _, st = m.hidden(ids, cu_seqlens=cu, caches=caches)
        pages = kv_pages.pages_of(caches)
        for step in range(4):
            pos = torch.tensor([60, 6]) + step
            _, st = m.hidden(torch.tensor([1, 2]), cu_seqlens=cu1, kda_states=st, caches=caches, position_offset=pos)
        before = pages.lens.clone(), pages.free_count.clone()
        with pytest.raises(ValueError, match="sequence 0"):
            m.hidden(torch.tensor([1, 2]), cu_seqlens=cu1, kda_states=st, caches=caches, position_offset=torch.tensor([64, 10]))
        assert torch.equal(pages.lens, before[0]) and torch.equal(pages.free_count, before[1])
        pages.release = torch.tensor([True, False])                           # the full one is done: the other goes on
        m.hidden(torch.tensor([1, 2]), cu_seqlens=cu1, kda_states=st, caches=caches, position_offset=torch.tensor([64, 10]))
        assert pages.lens.tolist() == [0, 11]
