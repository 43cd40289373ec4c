"""`score` through the leader / follower protocol on CPU (gloo): both ranks run the same passes and end with the same pages."""
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from sllm_b200.engine.distributed import LeaderEngine, follow  # noqa: E402
from sllm_b200.engine.engine import build_engine  # noqa: E402
from sllm_b200.models import config as MC  # noqa: E402


def main():
    rank = int(os.environ["RANK"])
    dist.init_process_group("gloo")
    cfg = MC.tiny_llama()
    cfg.max_context = 128
    make = lambda: build_engine(cfg, "cpu", seed=1, num_pages=64, max_batch=4, use_cuda_graphs=False)
    eng = make()
    if rank == 0:
        lead, texts = LeaderEngine(eng), [[1, 2, 3, 4, 5], [9] * 40]
        for top in (0, 2):
            for a, b in zip(lead.score(texts, top, 16), make().score(texts, top, 16)):
                assert all((x is None and y is None) or torch.equal(x, y) for x, y in zip(a, b))
        try:
            lead.score([[cfg.vocab]])
            raise SystemExit("not refused")
        except ValueError:
            pass                                               # refused ahead of the command: the follower is still there
        lead.score([[3, 2, 1]])
        lead.stop_followers()
    else:
        assert follow(eng) == 4
    st = eng.cache.pool.stats()
    assert st["sequences"] == 0 and st["free"] == st["pages"], st
    marks = [None, None]
    dist.all_gather_object(marks, st["high_water"])
    assert marks[0] == marks[1], marks
    dist.barrier()
    if rank == 0:
        print("SCORE_OK", flush=True)
    dist.destroy_process_group()


main()
