"""`score` without room through the leader / follower protocol on CPU (gloo): the leader refuses it ahead of the command, whether pages or
recurrent-state slots are short or the engine is quarantined, and the follower serves on."""
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from sllm_b200.cache.paged import OutOfPages  # noqa: E402
from sllm_b200.engine.distributed import LeaderEngine, follow  # noqa: E402
from sllm_b200.engine.engine import EngineQuarantined, build_engine  # noqa: E402
from sllm_b200.models import config as MC  # noqa: E402
from sllm_b200.models.qwen35 import tiny_qwen35  # noqa: E402


def refused(error, call):
    try:
        call()
    except error:
        return
    raise SystemExit("not refused")


def run(make, rank, leader):
    eng = make()
    if rank == 0:
        lead = LeaderEngine(eng)
        leader(lead)
        lead.stop_followers()
    else:
        follow(eng)                                        # (raises where a command fails here)
    free = [None, None]
    dist.all_gather_object(free, (eng.cache.pool.stats(), getattr(eng.cache, "free_slots", None)))
    assert free[0] == free[1], free


def main():
    rank = int(os.environ["RANK"])
    dist.init_process_group("gloo")
    texts = [[1, 2, 3, 4, 5], [9] * 40, [7] * 50]

    def pages(lead):
        make = lambda: build_engine(MC.tiny_llama(), "cpu", seed=1, num_pages=6, max_batch=4, use_cuda_graphs=False)
        refused(OutOfPages, lambda: lead.score([[1, 2], [3] * 200]))
        for a, b in zip(lead.score(texts), make().score(texts)):      # (in two groups, on both ranks)
            assert torch.equal(a.logprob, b.logprob)
        lead._e.quarantine = {"reason": "test"}
        refused(EngineQuarantined, lambda: lead.score(texts))
        lead._e.quarantine = None
        lead.score(texts)

    def slots(lead):
        live = []
        while lead._e.cache.free_slots:
            live.append(lead.new_sequence([1]))
        refused(RuntimeError, lambda: lead.score([[1, 2]]))
        lead.free_sequence(live.pop())
        assert len(lead.score(texts)) == 3

    run(lambda: build_engine(MC.tiny_llama(), "cpu", seed=1, num_pages=6, max_batch=4, use_cuda_graphs=False), rank, pages)
    run(lambda: build_engine(tiny_qwen35(), "cpu", seed=1, num_pages=24, max_batch=2, use_cuda_graphs=False), rank, slots)
    dist.barrier()
    if rank == 0:
        print("SCORE_ROOM_OK", flush=True)
    dist.destroy_process_group()


main()
