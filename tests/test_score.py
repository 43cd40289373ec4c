"""Scoring of texts through the engine: batch plan, model, output matrix, log-probabilities as one run."""
import json
import math
import os
import subprocess
import sys

import pytest
import torch

from sllm_b200 import ops
from sllm_b200.engine.batch import PageLists, make_prefill_batch
from sllm_b200.engine.engine import Engine, build_engine
from sllm_b200.models import config as MC
from sllm_b200.ops import _lib

DEV = "cuda"
TEXTS = [[5, 9, 3, 7, 2, 8], [11], list(range(3, 60)), [4, 4]]


def _bf16(**kw):
    return MC.ModelConfig(**{**dict(name="t", n_layers=2, d_model=256, n_heads=4, n_kv_heads=2, head_dim=64, ffn=512, vocab=1000,
                                    weight_format="bf16", kv_format="bf16", max_context=256), **kw})


def _families():
    from sllm_b200.models.fekolorn import tiny_fekolorn
    from sllm_b200.models.kegorax import tiny_kegorax
    from sllm_b200.models.moe import tiny_moe
    from sllm_b200.models.qwen35 import tiny_qwen35
    from sllm_b200.models.sepedra import tiny_sepedra
    from sllm_b200.models.zokuvik import tiny_zokuvik
    gemma = _bf16(name="g", family="gemma4", act="gelu_tanh", tie_embeddings=True, embedding_scale=16.0, logit_softcap=5.0, qk_norm=True,
                  post_norms=True)
    fp8 = _bf16(name="f", d_model=512, head_dim=128, ffn=1024, vocab=2048, weight_format="fp8", kv_format="fp8")
    return [_bf16(), gemma, fp8, tiny_moe(), tiny_qwen35(), tiny_zokuvik(), tiny_sepedra(), tiny_kegorax(), tiny_fekolorn()]


def forwarded(eng, ids):
    """Logits after every token but the last, from the model's forward pass, in 64 bits."""
    s = eng.new_sequence(ids[:-1])
    try:
        return eng.extend([s], sample=False)[0].double().cpu() if len(ids) > 1 else torch.empty((0, eng.cfg.vocab), dtype=torch.float64)
    finally:
        eng.free_sequence(s)


def check(eng, got, ids, tol_z, top):
    """tol_z: how far a logit of `score` may be from the forward pass's."""
    z = forwarded(eng, ids)
    n = len(ids) - 1
    assert got.logprob.shape == (n,) and got.entropy.shape == (n,) and got.logprob.device.type == "cpu"
    if not n:
        return
    logp = torch.log_softmax(z, 1)
    want = logp.gather(1, torch.tensor(ids[1:])[:, None])[:, 0]
    assert float((got.logprob.double() - want).abs().max()) <= 2 * tol_z + 1e-5
    spread = float(z.max() - z.min())
    entropy = -(logp.exp() * logp).sum(1)
    assert float((got.entropy.double() - entropy).abs().max()) <= 2 * tol_z * (1 + spread) + 1e-4
    if top:
        assert got.top_ids.shape == (n, top)
        assert float((got.top_logprobs.double() - logp.gather(1, got.top_ids.long())).abs().max()) <= 2 * tol_z + 1e-5
        assert bool((got.top_logprobs[:, :-1] >= got.top_logprobs[:, 1:]).all())
        best = logp.max(1).values                          # no alternative was passed over by more than the logits may be off
        assert bool((got.top_logprobs[:, 0].double() >= best - 2 * tol_z - 1e-5).all())


def test_score_on_cpu():
    eng = build_engine(MC.tiny_llama(), "cpu", num_pages=32, max_batch=2)
    for top in (0, 4):
        for rows in (Engine.SCORE_ROWS, 10):               # together, and the long text in portions
            for ids, got in zip(TEXTS, eng.score(TEXTS, top, rows)):
                check(eng, got, ids, 1e-4, top)
    assert eng.score([]) == [] and eng.cache.pool.stats()["sequences"] == 0


def test_score_where_cpu_tensors_are_refused(monkeypatch):
    """Nothing of the result's assembly on the host goes through an op (a server on a GPU refuses CPU tensors in ops)."""
    eng = build_engine(MC.tiny_llama(), "cpu", num_pages=8, max_batch=2)
    monkeypatch.setattr(eng, "_row_logprobs", lambda b, h, rows, tokens, top: ops.TokenLogprobs(
        torch.zeros(rows.numel()), torch.zeros(rows.numel()), torch.zeros((rows.numel(), top), dtype=torch.int32), torch.zeros((rows.numel(), top))))
    monkeypatch.setattr(eng.model, "hidden", lambda b, cache: None)
    _lib.set_fail_closed(True)
    try:
        got = eng.score([[3], [1, 2, 3]], 2)
    finally:
        _lib.set_fail_closed(False)
    assert got[0].logprob.shape == (0,) and got[0].top_ids.shape == (0, 2) and got[1].logprob.shape == (2,)


def test_score_refusals_leave_nothing_behind():
    eng = build_engine(MC.tiny_llama(), "cpu", num_pages=4, max_batch=2)
    v = eng.cfg.vocab
    for bad in (dict(prompts=[[]]), dict(prompts=[[1, v]]), dict(prompts=[[-1]]), dict(prompts=[[1] * (eng.cfg.max_context + 1)]),
                dict(prompts=[[1]], top=33), dict(prompts=[[1]], top=-1), dict(prompts=[[1]], max_rows=0)):
        with pytest.raises(ValueError):
            eng.score(**bad)
    from sllm_b200.cache.paged import OutOfPages
    with pytest.raises(OutOfPages):
        eng.score([[1, 2], [3] * 200])
    st = eng.cache.pool.stats()
    assert st["sequences"] == 0 and st["free"] == st["pages"]


def test_score_runs_as_many_texts_as_there_is_room_for(monkeypatch):
    """Texts that fit alone but not together, beside a live sequence; in groups that fill the pages."""
    eng = build_engine(MC.tiny_llama(), "cpu", num_pages=9, max_batch=4)
    texts = [[3 + (7 * i + k) % 50 for k in range(n)] for i, n in enumerate((60, 50, 64, 1, 33, 64, 2, 16))]
    want = [build_engine(MC.tiny_llama(), "cpu", num_pages=9, max_batch=4).score([t], 2)[0] for t in texts]
    live = eng.new_sequence([1, 2, 3])
    eng.prefill([live])
    groups = []
    run = eng._score_together
    monkeypatch.setattr(eng, "_score_together", lambda prompts, *a: groups.append([len(p) for p in prompts]) or run(prompts, *a))
    got = eng.score(texts, 2)
    assert groups == [[60, 50], [64, 1, 33], [64, 2, 16]]
    for a, b in zip(got, want):
        assert torch.equal(a.top_ids, b.top_ids) and torch.allclose(a.logprob, b.logprob, atol=1e-4) and torch.allclose(a.entropy, b.entropy, atol=1e-4)
    from sllm_b200.cache.paged import OutOfPages
    groups.clear()
    with pytest.raises(OutOfPages):
        eng.score([[1, 2], [3] * 129])
    assert groups == []                                    # refused ahead of any work
    st = eng.cache.pool.stats()
    assert st["sequences"] == 1 and st["free"] == 8


def test_score_runs_as_many_texts_as_there_are_state_slots():
    from sllm_b200.models.qwen35 import tiny_qwen35
    make = lambda: build_engine(tiny_qwen35(), "cpu", num_pages=32, max_batch=2)
    eng, texts = make(), [[5, 9, 3], [11, 4], [8, 8, 8, 1]]
    want = [make().score([t])[0] for t in texts]
    live = [eng.new_sequence([1]) for _ in range(eng.cache.free_slots - 1)]
    for a, b in zip(eng.score(texts), want):
        assert torch.allclose(a.logprob, b.logprob, atol=1e-4)
    assert eng.cache.free_slots == 1
    last = eng.new_sequence([1])
    with pytest.raises(RuntimeError, match="slot"):
        eng.score(texts)
    assert eng.score([]) == [] and eng.cache.pool.stats()["sequences"] == len(live) + 1
    eng.free_sequence(last)
    assert len(eng.score(texts)) == 3


def test_accounting_counts_every_static_input():
    eng = build_engine(MC.tiny_llama(), "cpu", num_pages=8, max_batch=2)
    held = sum(t.numel() * t.element_size() for n, t in vars(eng).items() if n.startswith("d_") and isinstance(t, torch.Tensor))
    assert eng.accounting()["device_staging"] == held


def test_page_lists():
    eng = build_engine(MC.tiny_llama(), "cpu", num_pages=16, max_batch=2)
    pool = eng.cache.pool
    a, b = pool.new_seq(), pool.new_seq()
    pool.reserve(a, 40)
    pool.reserve(b, 16)
    assert pool.list_pages([b, a], [16, 33]).tolist() == pool.pages(b) + pool.pages(a)
    assert pool.list_pages([a], [17]).tolist() == pool.pages(a)[:2] and pool.list_pages([], []).numel() == 0
    out = torch.full((2, 3), -1, dtype=torch.int32)
    assert pool.list_pages([a, b], [40, 1], out=out).tolist() == pool.pages(a) + pool.pages(b) and out[1].tolist()[1:] == [-1, -1]
    for seqs, lens, o in (([a], [49], None), ([99], [1], None), ([a], [40], out[:1, :2].contiguous()), ([a], [17], out[0, :1].expand(9)),
                          ([a], [17], out.long())):
        with pytest.raises(ValueError):
            pool.list_pages(seqs, lens, o)


def test_batches_from_page_lists_on_the_host():
    pages = torch.tensor([7, 3, 9, 4], dtype=torch.int32)
    b = make_prefill_batch([[1] * 20, [2]], PageLists(pages, 3, 16), "cpu")
    assert b.block_table.tolist() == [[7, 3, 0], [9, 0, 0]]
    b = make_prefill_batch([[1], [2] * 3], PageLists(pages, 3, 16), "cpu", [16, 29])
    assert b.block_table.tolist() == [[7, 3, 0], [9, 4, 0]] and b.kv_lens.tolist() == [17, 30, 31, 32]


def test_score_runner(tmp_path, capsys):
    from sllm_b200.cli import convert
    from sllm_b200.evidence import score
    g, l = str(tmp_path / "m.gguf"), str(tmp_path / "m.json")
    assert convert.main(["--kind", "random-llama", "--artifact", "tiny-llama", "--weight-format", "fp32", "--output", g, "--derived-lock", l,
                         "--converter-commit", "test"]) == 0
    capsys.readouterr()
    src = ["--gguf", g, "--derived-lock", l, "--cpu"]
    assert score.main(src + ["--text", "hello", "--input-token-ids", "1 2 3", "--top", "2"]) == 0
    rep = json.loads(capsys.readouterr().out)
    a, b = rep["texts"]
    assert rep["schema"] == score.SCHEMA and b["tokens"] == [1, 2, 3] and len(b["logprobs"]) == 2 and len(b["top"][0]) == 2
    assert math.isclose(a["perplexity"], math.exp(-sum(a["logprobs"]) / len(a["logprobs"])), rel_tol=1e-6)
    assert score.main(src) == 2 and score.main(src + ["--input-token-ids", "1 x"]) == 2 and score.main(src + ["--input-token-ids", "999999"]) == 2
    assert score.main(["--gguf", g, "--derived-lock", str(tmp_path / "none"), "--cpu", "--text", "a"]) == 3


def test_score_records_are_json():
    """What no JSON number stands for - a token that is shut out, a row of NaN, a likelihood beyond the perplexity's range - is null."""
    from sllm_b200.evidence.score import score_texts
    inf, nan = float("inf"), float("nan")

    class Stub:
        def score(self, texts, top):
            t = torch.tensor
            return [ops.TokenLogprobs(t([-1.0, -inf]), t([0.5, 0.0]), t([[3, -1], [-1, -1]]), t([[-0.25, -inf], [-inf, -inf]])),
                    ops.TokenLogprobs(t([nan, -2.0]), t([nan, 1.0]), t([[-1, -1], [4, 2]]), t([[nan, nan], [-0.5, -inf]])),
                    ops.TokenLogprobs(t([-800.0]), t([0.0]), t([[1, 2]]), t([[0.0, -3.0]])),
                    ops.TokenLogprobs(torch.empty(0), torch.empty(0), torch.empty((0, 2), dtype=torch.int32), torch.empty((0, 2)))]

    got = json.loads(json.dumps(score_texts(Stub(), [[1, 2, 3], [4, 5, 6], [7, 8], [9]], 2), allow_nan=False))
    assert got[0]["logprobs"] == [-1.0, None] and got[0]["nll_mean"] is None and got[0]["perplexity"] is None
    assert got[0]["top"] == [[{"token": 3, "logprob": -0.25}], []]
    assert got[1]["logprobs"] == [None, -2.0] and got[1]["entropy"] == [None, 1.0] and got[1]["nll_mean"] is None and got[1]["perplexity"] is None
    assert got[1]["top"][1] == [{"token": 4, "logprob": -0.5}, {"token": 2, "logprob": None}]
    assert got[2]["nll_mean"] == 800.0 and got[2]["perplexity"] is None
    assert got[3]["logprobs"] == [] and got[3]["nll_mean"] is None and got[3]["perplexity"] is None


def test_score_is_mirrored_to_follower_ranks():
    worker = os.path.join(os.path.dirname(os.path.abspath(__file__)), "score_worker.py")
    proc = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1",
                           "--master-port", "29847", worker], capture_output=True, text=True, timeout=240)
    assert proc.returncode == 0 and "SCORE_OK" in proc.stdout, proc.stdout[-2000:] + proc.stderr[-3000:]


def test_score_without_room_leaves_the_followers_serving():
    worker = os.path.join(os.path.dirname(os.path.abspath(__file__)), "score_room_worker.py")
    proc = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1",
                           "--master-port", "29849", worker], capture_output=True, text=True, timeout=240)
    assert proc.returncode == 0 and "SCORE_ROOM_OK" in proc.stdout, proc.stdout[-2000:] + proc.stderr[-3000:]


def test_score_of_a_head_sharded_over_ranks():
    worker = os.path.join(os.path.dirname(os.path.abspath(__file__)), "score_tp_worker.py")
    proc = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1",
                           "--master-port", "29851", worker], capture_output=True, text=True, timeout=240)
    assert proc.returncode == 0 and "SCORE_TP_OK" in proc.stdout, proc.stdout[-2000:] + proc.stderr[-3000:]


# ------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
def test_prefill_batches_are_the_same_on_the_gpu():
    eng = build_engine(MC.tiny_llama(), "cpu", num_pages=64, max_batch=4)
    pool = eng.cache.pool
    for lens, starts in (([3], None), ([1, 40, 17], [5, 0, 31]), ([4, 0, 2], [0, 3, 16]), ([0], [2])):
        at = starts or [0] * len(lens)
        seqs = [pool.new_seq() for _ in lens]
        for s, n, a in zip(seqs, lens, at):
            pool.reserve(s, n + a)
        ends = [n + a for n, a in zip(lens, at)]
        table = torch.zeros((len(lens), 9), dtype=torch.int32)
        pool.fill_block_table(seqs, table)
        prompts = [[i + 7] * n for i, n in enumerate(lens)]
        for last_only in (True, False):
            want = make_prefill_batch(prompts, table, "cpu", starts, last_only)
            for given in (table.to(DEV), PageLists(pool.list_pages(seqs, ends), 9, 16)):
                got = make_prefill_batch(prompts, given, DEV, starts, last_only)
                for f in ("tokens", "positions", "seq_index", "kv_lens", "block_table", "logit_rows", "cu_seqlens", "row_off"):
                    a, b = getattr(want, f), getattr(got, f)
                    assert (a is None and b is None) or (a.dtype == b.dtype and torch.equal(a, b.cpu())), f
                    assert b is None or f == "block_table" or b.data_ptr() % 16 == 0 or b.numel() == 0
                for f in ("max_kv", "max_seqlen", "cu_seqlens_host", "row_off_host", "starts_host"):
                    assert getattr(want, f) == getattr(got, f), f


@pytest.mark.gpu
def test_score_of_every_family():
    """A row's logits differ between the two ways by their rounding to bf16 (2^-9 of a logit) and by the order of sums, also in the
    layers, where the rows of a batch take other kernels: 2^-5 of the largest logit covers both (activations of 8 bits included)."""
    for cfg in _families():
        eng = build_engine(cfg, DEV, seed=1, num_pages=64, max_batch=4)
        for top in (0, 3):
            for rows in (Engine.SCORE_ROWS, 40):
                for ids, got in zip(TEXTS, eng.score(TEXTS, top, rows)):
                    z = forwarded(eng, ids)
                    check(eng, got, ids, 2 ** -5 * float(z.abs().max()) if z.numel() else 0.0, top)
        assert eng.cache.pool.stats()["sequences"] == 0
        assert ops.device_status(torch.device(DEV)) == 0
        out = eng.generate([[3, 4, 5]], 4)                 # the engine serves on
        assert out == eng.generate([[3, 4, 5]], 4)


@pytest.mark.gpu
@pytest.mark.parametrize("which", [0, 1])
def test_alternatives_do_not_change_a_tokens_score(which):
    """Both ways sum the products in 32 bits: with a row's largest sum of magnitudes (at most the product of the norms), every 16 of d products
    are rounded once towards zero, on either way, and the joint sums as in the ops' own tests."""
    cfg = _families()[which]
    eng = build_engine(cfg, DEV, seed=1, num_pages=64, max_batch=4)
    m = eng.model.w
    mag = float(m.lm_head.w.double().norm(dim=1).max() * (m.final_norm.double().abs().max() + cfg.norm_offset_one) * cfg.d_model ** 0.5)
    dz, rel = mag * (cfg.d_model / 16 + 8) * 2 ** -23, (cfg.vocab / 256 + 64) * 2 ** -24
    texts = TEXTS + [[(7 * k) % 900 for k in range(200)]]
    for a, b in zip(eng.score(texts, 0), eng.score(texts, 3)):
        if not a.logprob.numel():
            continue
        assert float((a.logprob - b.logprob).abs().max()) <= 4 * dz + 2 * rel + 16 * 2 ** -24 * (float(a.logprob.abs().max()) + cfg.logit_softcap)
        assert float((a.entropy - b.entropy).abs().max()) <= 4 * (dz + rel) * (1 + 2 * mag + float(a.entropy.max()))


@pytest.mark.gpu
def test_wide_tables_decode_the_same():
    eng = build_engine(_bf16(max_context=4096), DEV, seed=1, num_pages=200, max_batch=8)
    prompts = [list(range(3, 40)), [5, 6, 7, 8], [9] * 15]
    want = eng.generate(prompts, 20)                       # (three sequences: a row of padding)
    eng.WIDE_TABLE = 1
    eng._table_key = None
    eng.d_table.fill_(77)
    assert eng.generate(prompts, 20) == want
    n = eng._padded(3)
    host = torch.zeros((8, eng.max_blocks), dtype=torch.int32)
    seqs = [eng.new_sequence(p) for p in prompts]
    for s, t in zip(seqs, eng.prefill(seqs)):
        s.tokens.append(t)
    eng.decode(seqs)
    eng.cache.pool.fill_block_table([s.seq_id for s in seqs], host)
    host[3:n] = host[0]
    assert torch.equal(eng.d_table[:n].cpu(), host[:n])
