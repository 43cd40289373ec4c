"""`score` of a model sharded over two ranks on CPU (gloo), its head with it (logits are gathered) or whole on each: the single rank's numbers,
with and without alternatives, in one pass and in portions, called by both ranks and through the leader / follower protocol."""
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from sllm_b200 import ops  # noqa: E402
from sllm_b200.engine.distributed import LeaderEngine, follow  # noqa: E402
from sllm_b200.engine.engine import build_engine  # noqa: E402
from sllm_b200.models.config import ModelConfig  # noqa: E402
from sllm_b200.models.qwen35 import tiny_qwen35  # noqa: E402
from sllm_b200.parallel.tp import NcclTP  # noqa: E402


def run(rank, world, cfg, sharded):
    g = torch.Generator().manual_seed(3)
    texts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (9, 1, 37, 5)]
    make = lambda tp=None: build_engine(cfg, "cpu", seed=2, max_batch=4, num_pages=32, use_cuda_graphs=False, tp=tp)
    eng = make(NcclTP(world, rank, torch.device("cpu")))
    assert (eng.model.w.lm_head.out_features < cfg.vocab) == sharded

    def check(score):
        for top in (0, 3):
            for rows in (64, 10):
                for a, b in zip(score(texts, top, rows), make().score(texts, top, rows)):
                    # partial products are rounded before they are summed over the ranks
                    assert all(torch.allclose(x, y, atol=2e-2) for x, y in ((a.logprob, b.logprob), (a.entropy, b.entropy)))
                    assert not top or torch.allclose(a.top_logprobs, b.top_logprobs, atol=2e-2)

    whole = ops.logprobs.CHUNK_LOGITS
    for chunk in (whole, 3 * cfg.vocab):                       # (rows gathered three at a time)
        ops.logprobs.CHUNK_LOGITS = chunk
        check(eng.score)
    if rank == 0:
        lead = LeaderEngine(eng)
        check(lead.score)
        lead.stop_followers()
    else:
        assert follow(eng) == 5
    ops.logprobs.CHUNK_LOGITS = whole
    assert eng.cache.pool.stats()["sequences"] == 0


def main():
    rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
    dist.init_process_group("gloo")
    cfg = tiny_qwen35()
    cfg.weight_format, cfg.kv_format = "fp32", "fp32"
    cfg.n_kv_heads, cfg.gdn_qk_heads, cfg.gdn_heads = 2, 2, 4
    run(rank, world, cfg, False)
    dense = dict(name="t", n_layers=2, d_model=64, n_heads=4, n_kv_heads=2, head_dim=16, ffn=128, vocab=96, weight_format="fp32", kv_format="fp32",
                 max_context=128)
    run(rank, world, ModelConfig(**dense), True)
    run(rank, world, ModelConfig(**{**dense, "family": "gemma4", "act": "gelu_tanh", "tie_embeddings": True, "embedding_scale": 8.0,
                                    "logit_softcap": 2.0, "qk_norm": True, "post_norms": True}), True)
    dist.barrier()
    if rank == 0:
        print("SCORE_TP_OK", flush=True)
    dist.destroy_process_group()


main()
