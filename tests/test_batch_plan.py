"""The structure of a batch from request lengths, against a walk over the requests."""
import pytest
import torch

from sllm_b200 import ops
from sllm_b200.ops import _lib, plan as PL

DEV = "cuda"


def walk(new, starts, pages, rows, blocks, page):
    out, table, off, last, at = [], [], [0], [], 0
    for i, (n, s0) in enumerate(zip(new, starts)):
        n, s0 = max(n, 0), max(s0, 0)
        used = -(-(s0 + n) // page)
        mine = [pages[c] if c < len(pages) else 0 for c in range(at, at + used)]
        at += used
        out += [(s0 + j, i, s0 + j + 1, mine[(s0 + j) // page] * page + (s0 + j) % page) for j in range(n)]
        last.append(off[-1] + n - 1 if n else -1)
        off.append(off[-1] + n)
        table.append((mine + [0] * blocks)[:blocks])
    out = (out + [(-1, -1, 0, -1)] * (rows - len(out)))[:rows]
    col = list(zip(*out)) if out else [(), (), (), ()]
    t = lambda x, dt=torch.int32: torch.tensor(list(x), dtype=dt)
    return [t(off), t(col[0]), t(col[1]), t(col[2]), t(col[3], torch.int64), t(last, torch.int64),
            torch.tensor(table, dtype=torch.int32).reshape(len(new), blocks)]


def case(new, starts, page, seed=0, short=0):
    count = sum(-(-(max(s, 0) + max(n, 0)) // page) for n, s in zip(new, starts))
    pages = torch.randperm(count + 40, generator=torch.Generator().manual_seed(seed))[:max(0, count - short)].tolist()
    return new, starts, pages


def lens(s, hi, seed, lo=0):
    return torch.randint(lo, hi + 1, (s,), generator=torch.Generator().manual_seed(seed)).tolist()


CASES = [case([1], [0], 16) + (0, 1, 16), case([1], [15], 16) + (0, 1, 16), case([1], [16], 16) + (3, 2, 16), case([0], [5], 16) + (2, 4, 16),
         case([5000], [0], 16) + (0, 320, 16), case([3, 0, 17, 1], [0, 4, 31, 16], 16) + (5, 9, 16), case(lens(64, 1, 0, 1), lens(64, 900, 1), 16) + (0, 64, 16),
         case(lens(300, 40, 2), lens(300, 70, 3), 16) + (11, 7, 16), case(lens(1000, 3, 4), lens(1000, 20, 5), 1) + (1, 24, 1),
         case(lens(2100, 2, 6), lens(2100, 5, 7), 4) + (0, 2, 4), case(lens(7, 900, 8), lens(7, 900, 9), 48, short=9) + (0, 33, 48),
         case([4, -3, 2], [-8, 20, 3], 16) + (1, 3, 16), case([0, 0, 0], [0, 0, 0], 16) + (4, 2, 16), case([20, 3], [0, 0], 16) + (-9, 3, 16),
         case(lens(9, 4000, 10), [0] * 9, 16) + (0, 0, 16), case([1] * 40 + [30000] + [2] * 40, [17] * 81, 16) + (600, 1900, 16),
         case(lens(16384, 2, 11), lens(16384, 9, 12), 4) + (7, 4, 4), case([9, 1, 600], [0, 4095, 70000], 16) + (0, 5000, 16)]


def same(got, want):
    for name, a, b in zip(PL.BatchPlan._fields, got, want):
        assert a.dtype == b.dtype and torch.equal(a.cpu(), b), name


def tensors(new, starts, pages, device):
    return [torch.tensor(x, dtype=torch.int32, device=device) for x in (new, starts, pages)]


@pytest.mark.parametrize("new,starts,pages,pad,blocks,page", CASES)
def test_cpu_matches_the_walk(new, starts, pages, pad, blocks, page):
    rows = max(0, sum(max(n, 0) for n in new) + pad)
    same(ops.batch_plan(*tensors(new, starts, pages, "cpu"), rows, blocks, page), walk(new, starts, pages, rows, blocks, page))


def test_refusals():
    i = lambda *x: torch.tensor(x, dtype=torch.int32)
    good = dict(new_lens=i(2, 3), starts=i(0, 0), pages=i(0, 1), rows=5, max_blocks=2, page_size=16)
    ops.batch_plan(**good)
    for bad in (dict(new_lens=i(2, 3).long()), dict(starts=i(0)), dict(pages=i(0, 1).float()), dict(new_lens=i(2, 3).view(1, 2)), dict(rows=-1),
                dict(rows=2 ** 31), dict(new_lens=torch.zeros(20000, dtype=torch.int32), starts=torch.zeros(20000, dtype=torch.int32)), dict(max_blocks=-1), dict(page_size=0), dict(starts=torch.zeros(4, dtype=torch.int32)[::2]),
                dict(table=torch.zeros((2, 3), dtype=torch.int32)), dict(table=torch.zeros((2, 2))), dict(table=torch.zeros((2, 2), dtype=torch.int32).t()),
                dict(table=torch.zeros((1, 2), dtype=torch.int32).expand(2, 2))):
        with pytest.raises(ValueError):
            ops.batch_plan(**{**good, **bad})


def test_the_launcher_refuses():
    if not _lib.kernels_available():
        pytest.skip("the kernel library is not built")
    f = PL._k().sllm_batch_plan
    ok = [256, 256, 256, 4, 2, 5, 2, 2, 16, 256, 256, 256, 256, 256, 256, 256, None]
    assert f(*(ok[:4] + [16385] + ok[5:])) == 7 and f(*(ok[:5] + [2 ** 31 - 1] + ok[6:])) == 7 and f(*(ok[:3] + [2 ** 31] + ok[4:])) == 7
    for at, value in ((0, None), (1, None), (2, None), (3, -1), (4, -1), (5, -1), (6, -1), (7, 1), (8, 0), (9, None), (10, None), (13, None),
                      (14, None), (15, None)):
        a = list(ok)
        a[at] = value
        assert f(*a) == 1, (at, value)


@pytest.mark.gpu
@pytest.mark.parametrize("new,starts,pages,pad,blocks,page", CASES)
def test_kernel_matches_the_walk(new, starts, pages, pad, blocks, page):
    rows = max(0, sum(max(n, 0) for n in new) + pad)
    same(ops.batch_plan(*tensors(new, starts, pages, DEV), rows, blocks, page), walk(new, starts, pages, rows, blocks, page))


@pytest.mark.gpu
def test_table_of_the_caller_and_what_lies_around_it():
    new, starts, pages = case([3, 40, 1], [20, 0, 15], 16)
    big = torch.full((5, 11), 77, dtype=torch.int32, device=DEV)
    got = ops.batch_plan(*tensors(new, starts, pages, DEV), 44, 6, 16, table=big[1:4, 2:8])
    assert got.block_table.data_ptr() == big[1:4, 2:8].data_ptr()
    want = walk(new, starts, pages, 44, 6, 16)
    same(got, want)
    ring = big.clone()
    ring[1:4, 2:8] = 77
    assert bool((ring == 77).all())


@pytest.mark.gpu
def test_no_requests():
    e = torch.empty(0, dtype=torch.int32, device=DEV)
    got = ops.batch_plan(e, e, e, 3, 2)
    same(got, walk([], [], [], 3, 2, 16))


@pytest.mark.gpu
def test_captured_plan_follows_its_inputs():
    a, b = case([3, 1, 9], [4, 31, 0], 16), case([2, 10, 1], [14, 20, 17], 16, seed=5)
    n = max(len(a[2]), len(b[2]))
    held = tensors(a[0], a[1], a[2] + [0] * (n - len(a[2])), DEV)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.batch_plan(*held, 16, 4)
    for c in (b, a):
        for t, v in zip(held, tensors(c[0], c[1], c[2] + [0] * (n - len(c[2])), DEV)):
            t.copy_(v)
        g.replay()
        same(got, walk(c[0], c[1], c[2], 16, 4, 16))


@pytest.mark.gpu
def test_calls_from_two_threads():
    import threading
    cases = [case(lens(9000, 2, 13), lens(9000, 9, 14), 4), case(lens(16384, 2, 15), lens(16384, 9, 16), 4)]
    want = [walk(*c, sum(c[0]), 4, 4) for c in cases]
    held = [tensors(*c, DEV) for c in cases]
    torch.cuda.synchronize()
    failed = []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(200):
                    got = ops.batch_plan(*held[i], sum(cases[i][0]), 4, 4)
                torch.cuda.current_stream().synchronize()
                same(got, want[i])
        except BaseException as e:
            failed.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


AROUND = """
import sys, torch
sys.path.insert(0, {root!r})
from sllm_b200 import ops
for s in {sizes}:
    new, starts = torch.arange(s, dtype=torch.int32) % 3, torch.arange(s, dtype=torch.int32) % 7
    pages = torch.randperm(int(((new + starts + 3) // 4).sum())).to(torch.int32)
    want = ops.batch_plan(new, starts, pages, int(new.sum()) + 1, 3, 4)
    got = ops.batch_plan(new.cuda(), starts.cuda(), pages.cuda(), int(new.sum()) + 1, 3, 4)
    assert all(torch.equal(a, b.cpu()) for a, b in zip(want, got)), s
print("PLANS_OK")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[4095, 4096, 6134, 6135], [6136], [6143], [6144], [6137, 6140, 6142, 6145, 16384, 6139, 1]])
def test_plans_around_the_default_shared_memory(sizes):
    """Running sums of 6135 requests and the kernel's own 64 bytes are 48 KB; in a process of its own, since a larger plan raises the
    allowance for what follows."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    proc = subprocess.run([sys.executable, "-c", AROUND.format(root=root, sizes=sizes)], capture_output=True, text=True, timeout=240)
    assert proc.returncode == 0 and "PLANS_OK" in proc.stdout, proc.stderr[-2000:]
