"""Log-probabilities of given tokens, entropies and alternatives against the definition in 64 bits."""
import math

import pytest
import torch

from sllm_b200 import ops
from sllm_b200.ops import _lib, logprobs as LP

DEV = "cuda"
INF, NAN = float("inf"), float("nan")
EPS = 2.0 ** -24


def oracle(z, ids, top):
    """Row by row from p = exp(z) / sum exp(z), in 64 bits."""
    lps, hs, tids, tlps = [], [], [], []
    for row, given in zip(z.double().cpu(), (ids if ids.dim() == 2 else ids[:, None]).tolist()):
        v = row.numel()
        if torch.isnan(row).any():
            logp, h = torch.full((v,), NAN, dtype=torch.float64), NAN
        elif (row == INF).any():
            n = int((row == INF).sum())
            logp, h = torch.where(row == INF, -math.log(n), -INF).double(), math.log(n)
        elif (row == -INF).all():
            logp, h = row, 0.0
        else:
            w = torch.exp(row - row.max())
            p = w / w.sum()
            logp = (row - row.max()) - torch.log(w.sum())
            h = -float((p[p > 0] * logp[p > 0]).sum())
        lps.append([0.0 if t < 0 else NAN if t >= v else float(logp[t]) for t in given])
        hs.append(h)
        order = [] if math.isnan(h) or not top else [i for i in torch.argsort(row, descending=True, stable=True)[:top].tolist() if row[i] != -INF]
        tids.append(order + [-1] * (top - len(order)))
        tlps.append([float(logp[i]) for i in order] + [NAN if math.isnan(h) else -INF] * (top - len(order)))
    t = lambda x: torch.tensor(x, dtype=torch.float64)
    return t(lps).reshape(ids.shape), t(hs), torch.tensor(tids).reshape(z.shape[0], top), t(tlps).reshape(z.shape[0], top)


def same(got, want, tol):
    got = got.double().cpu()
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, torch.sign(want) * INF, want)      # beyond fp32's range
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and torch.equal(got[torch.isinf(got)], want[torch.isinf(want)])
    ok = torch.isfinite(want)
    err = (got - want).abs()[ok]
    limit = (torch.as_tensor(tol, dtype=torch.float64).expand(want.shape))[ok]
    assert bool((err <= limit).all()), f"off by {float((err - limit).max()):.3g} beyond the limit"


def check(z, ids, top, got):
    """Sums of V terms: a chain of at most V / 256 additions per thread and 16 more to join them, each off by 2^-24; an exponential by
    2^-22; differences and the result by 2^-24 of their size.  The entropy's second sum has the same relative error for each term, the
    terms having one sign."""
    lp, h, tid, tlp = oracle(z, ids, top)
    rel = (z.shape[1] / 256 + 32) * EPS
    same(got.logprob, lp, rel + 4 * EPS * torch.nan_to_num(lp.abs(), posinf=0.0))
    same(got.entropy, h, 4 * (rel + 8 * EPS) * (1 + torch.nan_to_num(h)))
    if top:
        assert torch.equal(got.top_ids.cpu().long(), tid)
        same(got.top_logprobs, tlp, rel + 4 * EPS * torch.nan_to_num(tlp.abs(), posinf=0.0))
    else:
        assert got.top_ids is None and got.top_logprobs is None


def rows(r, v, dtype, seed, gap=0, shift=0, std=2.5, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    store = torch.randn(shift + r * (v + gap), generator=g).mul_(std).to(dtype).to(device)
    return store[shift:].view(r, v + gap)[:, :v], torch.randint(0, v, (r,), generator=g).to(device)


def special(v, dtype):
    """Rows at the edges: shut out in part, but for one token, as a whole, at the type's ends, all equal, infinities, NaN, zeros of both
    signs."""
    lowest, highest = torch.finfo(dtype).min, torch.finfo(dtype).max
    z = torch.randn(13, v, generator=torch.Generator().manual_seed(3)) * 3
    z[0, ::2] = -INF
    z[1] = -INF
    z[1, v // 2] = 1.5
    z[2] = -INF
    z[3] = lowest
    z[4] = lowest
    z[4, v - 1] = 0.25
    z[5] = 2.0
    z[6, v // 3] = INF
    z[7] = INF
    z[8, v // 2] = NAN
    z[9] = torch.where(torch.arange(v) % 3 == 0, -0.0, 0.0)
    z[10] = lowest
    z[10, 0] = highest
    z[11, v - 1] = INF
    z[11, 0] = -INF
    z[12] = torch.arange(v) / 64.0
    return z.to(dtype)


@pytest.mark.parametrize("v", [1, 2, 7, 300])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_cpu_matches_the_definition(v, top):
    z, ids = rows(4, v, torch.float32, v)
    check(z, ids, top, ops.token_logprobs(z, ids, top))
    z = special(v, torch.float32)
    ids = torch.randint(-1, v + 1, (13, 3), generator=torch.Generator().manual_seed(1))
    check(z, ids, top, ops.token_logprobs(z, ids, top))


def test_linear_on_cpu_is_the_product_and_its_logprobs():
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(9, 24, generator=g), torch.randn(70, 24, generator=g)
    ids = torch.randint(0, 70, (9,), generator=g)
    for cap in (0.0, 2.0):
        z = x.double() @ w.double().t()
        z = cap * torch.tanh(z / cap) if cap else z
        got = ops.linear_logprobs(x, ops.LinearWeight("dense", w), ids, softcap=cap, top=3)
        lp, h, tid, _ = oracle(z, ids, 3)
        same(got.logprob, lp, 1e-5)       # 24 products of about 1, rounded to 2^-24 each, in both the row's token and its sum
        same(got.entropy, h, 1e-4)
        assert torch.equal(got.top_ids.long(), tid)


def test_linear_in_chunks_gives_the_same(monkeypatch):
    g = torch.Generator().manual_seed(0)
    x, w = torch.randn(11, 16, generator=g), ops.LinearWeight("dense", torch.randn(40, 16, generator=g))
    ids = torch.randint(0, 40, (11,), generator=g)
    whole = ops.linear_logprobs(x, w, ids, top=2)
    monkeypatch.setattr(LP, "CHUNK_LOGITS", 160)
    parts = ops.linear_logprobs(x, w, ids, top=2)
    assert all(torch.allclose(a, b, atol=1e-6) for a, b in zip(whole, parts))
    none = ops.linear_logprobs(x[:0], w, ids[:0], top=2)
    assert none.logprob.shape == (0,) and none.top_ids.shape == (0, 2)


def test_logits_of_one_chunk_are_held_at_a_time(monkeypatch):
    """The chunk's size bounds the memory only if a chunk is gone before the next one is made."""
    import weakref
    from sllm_b200.engine.engine import build_engine
    from sllm_b200.models import config as MC
    from sllm_b200.ops import core
    held = []
    monkeypatch.setattr(LP, "CHUNK_LOGITS", 160)

    def watched(make):
        def call(*a, **kw):
            assert not any(r() is not None for r in held)
            z = make(*a, **kw)
            held.append(weakref.ref(z))
            return z
        return call

    monkeypatch.setattr(core, "linear", watched(core.linear))
    x, w = torch.randn(11, 16), ops.LinearWeight("dense", torch.randn(40, 16))
    ops.linear_logprobs(x, w, torch.zeros(11, dtype=torch.int64), top=2)
    assert len(held) == 3
    monkeypatch.undo()
    held.clear()
    eng = build_engine(MC.tiny_llama(), "cpu", num_pages=8, max_batch=2)
    monkeypatch.setattr(LP, "CHUNK_LOGITS", 4 * eng.cfg.vocab)
    monkeypatch.setattr(eng.model.w.lm_head, "kind", "fp8x")                # (a head that goes through the model's logits)
    head = torch.zeros((eng.cfg.vocab, eng.cfg.d_model))
    monkeypatch.setattr(eng.model, "logits", watched(lambda h, b: h.index_select(0, b.logit_rows).float() @ head.t()))
    got = eng.score([[1, 2, 3, 4, 5, 6, 7, 8, 9, 10]], 2)[0]
    assert len(held) == 3 and got.logprob.shape == (9,)


def test_refusals():
    z, ids = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    w = ops.LinearWeight("dense", torch.zeros(8, 4))
    for bad in (lambda: ops.token_logprobs(z[0], ids), lambda: ops.token_logprobs(z.double(), ids), lambda: ops.token_logprobs(z.t(), ids),
                lambda: ops.token_logprobs(z[:, :0], ids), lambda: ops.token_logprobs(z, ids[:2]), lambda: ops.token_logprobs(z, ids.float()),
                lambda: ops.token_logprobs(z, ids, -1), lambda: ops.token_logprobs(z, ids, 33),
                lambda: ops.token_logprobs(z, ids.view(3, 1, 1)), lambda: ops.linear_logprobs(torch.zeros(3, 5), w, ids),
                lambda: ops.linear_logprobs(torch.zeros(3, 4), w, ids.view(3, 1)), lambda: ops.linear_logprobs(torch.zeros(3, 4), w, ids, softcap=-1.0),
                lambda: ops.linear_logprobs(torch.zeros(3, 4), w, ids, softcap=NAN), lambda: ops.linear_logprobs(torch.zeros(3, 4), w, ids, softcap=1e31),
                lambda: ops.linear_logprobs(torch.zeros(3, 4), w, ids, softcap=INF), lambda: ops.linear_logprobs(torch.zeros(3, 4), w, ids, softcap=1e-40),
                lambda: ops.linear_logprobs(torch.zeros(3, 4), ops.LinearWeight("dense", torch.zeros((8, 4), device="meta")), ids),
                lambda: ops.linear_logprobs(torch.zeros(3, 4), w, ids, top=40)):
        with pytest.raises(ValueError):
            bad()


def test_the_launcher_refuses():
    """Arguments that the C entry turns into errors before anything is launched."""
    if not _lib.kernels_available():
        pytest.skip("the kernel library is not built")
    f = LP._k().sllm_token_logprobs
    ok = [256, 8, 3, 8, 0, 256, 1, 1, 4, 256, 256, 256, 256, None]
    for at, value, code in ((0, None, 1), (1, -1, 1), (2, 0, 1), (3, 0, 1), (3, (1 << 30) + 1, 7), (4, 3, 1), (5, None, 1), (7, -1, 1), (8, 33, 7), (9, None, 1),
                            (10, None, 1), (11, None, 1), (12, None, 1), (0, 257, 3)):
        a = list(ok)
        a[at] = value
        assert f(*a) == code, (at, value)


def test_the_head_launcher_refuses():
    if not _lib.kernels_available():
        pytest.skip("the kernel library is not built")
    f, floats = LP._k().sllm_head_logprobs, LP._k().sllm_head_logprobs_floats
    for bn in (0, 128, 256):
        assert floats(0, 8, bn) == 0 and floats(5, 70000, bn) % 5 == 0
    assert floats(5, 8, 64) == 0 and floats(5, (1 << 30) + 1, 0) == 0
    ok = [256, 256, 256, 100, 1000, 64, 64, 0.0, 256, 256, 1 << 20, 256, 256, 256, None]
    for at, value, code in ((0, None, 1), (1, None, 1), (2, None, 1), (3, 0, 1), (4, 0, 1), (5, 0, 1), (6, 63, 1), (7, -1.0, 1), (7, NAN, 1), (7, INF, 1), (7, 1e-40, 1),
                            (8, 64, 1), (9, None, 1), (11, None, 1), (12, None, 1), (3, (1 << 24) + 1, 7), (4, (1 << 30) + 1, 7), (6, 68, 3), (0, 264, 3),
                            (1, 264, 3), (9, 264, 3), (10, floats(100, 1000, 256) - 1, 4)):
        a = list(ok)
        a[at] = value
        assert f(*a) == code, (at, value)
    assert f(*(ok[:3] + [129] + ok[4:8] + [0] + ok[9:])) == 1          # more rows than the kernel for few takes


def test_rejected_launches_are_errors():
    """Every entry's refusal reaches the caller, whichever path a call takes (a stand-in for the library counts them)."""
    z, ids = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int32)
    x, w = torch.zeros((3, 8), dtype=torch.bfloat16), ops.LinearWeight("dense", torch.zeros((5, 8), dtype=torch.bfloat16))
    i = lambda *v: torch.tensor(v, dtype=torch.int32)
    for name, call in (("sllm_token_logprobs", lambda: ops.token_logprobs(z, ids, 2)), ("sllm_head_logprobs", lambda: ops.linear_logprobs(x, w, ids)),
                       ("sllm_batch_plan", lambda: ops.batch_plan(i(1), i(0), i(0), 1, 1))):
        fake = _lib.FakeKernelLibrary({name: [0, 5]})
        _lib.install_fake(fake)
        try:
            call()
            assert fake.count(name) == 1
            with pytest.raises(_lib.KernelError):
                call()
        finally:
            _lib.install_fake(None)


def test_launches_go_to_the_device_of_their_tensors(monkeypatch):
    """Two devices stood in for: the entry gets the stream that is current on the tensors' device, which is current while it runs."""
    from sllm_b200.ops import core
    now = [0]

    class On:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *exc):
            now[0] = self.before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda i: 100 + i, raising=False)
    seen = []
    for index in (0, 1):
        assert core._launch(torch.device("cuda", index), lambda *a: seen.append((now[0], a)) or 0, 7) == 0
    assert seen == [(0, (7, 100)), (1, (7, 101))] and now == [0]


# ------------------------------------------------------------------------------------------ kernels
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("r,v,gap,shift,top", [(1, 1, 0, 0, 3), (2, 5, 3, 1, 2), (3, 31, 0, 0, 32), (5, 257, 1, 1, 1), (4, 2048, 0, 0, 5),
                                               (7, 4099, 5, 3, 20), (1, 32000, 0, 0, 32), (300, 1000, 24, 8, 4), (700, 515, 0, 1, 0), (2, 131077, 11, 7, 20),
                                               (160, 9001, 0, 0, 7), (650, 9001, 5, 3, 6), (1250, 8400, 0, 0, 0), (593, 12289, 7, 1, 32),
                                               (700, 12289, 7, 1, 32), (2000, 16500, 1, 3, 5), (80, 40001, 3, 5, 5), (100, 17000, 0, 0, 32),
                                               (148, 70000, 1, 1, 3), (160, 33001, 0, 2, 32), (197, 20000, 0, 0, 4), (118, 20011, 0, 0, 20), (30, 60000, 5, 0, 32)])
def test_kernel_matches_the_definition(dtype, r, v, gap, shift, top):
    z, ids = rows(r, v, dtype, r * v, gap, shift, device=DEV)
    check(z, ids, top, ops.token_logprobs(z, ids.int() if r % 2 else ids, top))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("v", [1, 2, 33, 1000, 20011])
@pytest.mark.parametrize("top", [0, 6, 32])
def test_kernel_at_the_edges(dtype, v, top):
    z = special(v, dtype).to(DEV)
    ids = torch.randint(-1, v + 1, (13, 3), generator=torch.Generator().manual_seed(1)).to(DEV)
    check(z, ids, top, ops.token_logprobs(z, ids, top))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,v", [(torch.bfloat16, 65543), (torch.bfloat16, 70001), (torch.float32, 32771)])
@pytest.mark.parametrize("top", [0, 6, 32])
def test_many_long_rows(dtype, v, top):
    """Rows enough for the kernel that takes them in parts: a sample of them against the definition, all of them against the kernel for
    fewer (the order of additions is the same, the alternatives are whole numbers and values of the logits)."""
    r = 2400
    store = torch.randn(r * v + 5, device=DEV, generator=torch.Generator(device=DEV).manual_seed(v)).mul_(2.5).to(dtype)
    z = store[5:].view(r, v)
    z[7] = special(v, dtype)[8].to(DEV)
    z[8] = -INF
    z[9, 100:] = -INF
    z[10] = 1.0
    z[11] = torch.arange(v, device=DEV) / 256
    ids = torch.randint(0, v, (r,), device=DEV)
    got = ops.token_logprobs(z, ids, top)
    few = slice(5, 13)
    check(z[few], ids[few], top, ops.TokenLogprobs(*(None if f is None else f[few] for f in got)))
    for lo in range(0, r, 600):
        part = slice(lo, lo + 600)
        want = ops.token_logprobs(z[part], ids[part], top)
        for a, b in zip(got, want):
            assert a is None or torch.allclose(a[part].double(), b.double(), rtol=1e-5, atol=1e-4, equal_nan=True)
        assert not top or torch.equal(got.top_ids[part], want.top_ids)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("top", [0, 6])
def test_many_rows_at_the_edges(dtype, top):
    """Rows of every kind one after another in the same CTAs."""
    v = 9007
    one = special(v, dtype)
    z = one.repeat(60, 1).to(DEV)
    ids = torch.randint(-1, v + 1, (13, 2), generator=torch.Generator().manual_seed(1)).to(DEV)
    got = ops.token_logprobs(z, ids.repeat(60, 1), top)
    for k in (0, 31, 59):
        part = ops.TokenLogprobs(*(None if f is None else f[13 * k:13 * k + 13] for f in got))
        check(one, ids, top, part)
    # a row's sums go by its 16-byte units, so rows of one alignment (8 x 13 apart: 8 x 9007 elements are whole units) have the same bits
    for k in (8, 56):
        assert all(f is None or torch.equal(torch.nan_to_num(f[13 * k:13 * k + 13]), torch.nan_to_num(f[:13])) for f in got)
    assert ops.device_status(z.device) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["rising", "falling", "equal", "runs", "few"])
@pytest.mark.parametrize("v", [700, 40000])
def test_alternatives_of_ordered_rows(order, v):
    """Rows in which many tokens pass for candidates: sorted ones, ties of all or most of the row, fewer tokens than alternatives."""
    i = torch.arange(v)
    z = {"rising": i * 0.5, "falling": -i * 0.5, "equal": i * 0.0, "runs": (i // 97 % 5) * 1.0,
         "few": torch.where(i % (v // 3) == 1, i * 1.0, torch.tensor(-INF))}[order]
    z = torch.stack([z, z.flip(0)]).to(DEV)
    ids = torch.tensor([0, v - 1], device=DEV)
    for x in (z, z.bfloat16()):
        got = ops.token_logprobs(x, ids, 32)
        _, _, tid, _ = oracle(x, ids, 32)
        assert torch.equal(got.top_ids.cpu().long(), tid)
        got = ops.token_logprobs(x.repeat(300, 1), ids.repeat(300), 32)
        assert torch.equal(got.top_ids.cpu().long(), tid.repeat(300, 1))


@pytest.mark.gpu
def test_rows_whose_offsets_pass_32_bits():
    store = torch.empty((1 << 31) + 5000, dtype=torch.bfloat16, device=DEV)
    z = store.as_strided((2, 4100), (1 << 31, 1), 3)
    z.copy_(torch.randn(2, 4100, generator=torch.Generator().manual_seed(0)))
    ids = torch.tensor([[0, 4099], [17, 4098]], device=DEV)
    check(z, ids, 5, ops.token_logprobs(z, ids, 5))


@pytest.mark.gpu
def test_broadcast_rows_streams_and_graphs():
    z, ids = rows(6, 5003, torch.bfloat16, 0, device=DEV)
    one = z[:1].expand(6, -1)
    check(one, ids, 3, ops.token_logprobs(one, ids, 3))
    want = ops.token_logprobs(z, ids, 3)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        a = ops.token_logprobs(z, ids, 3)
    b = ops.token_logprobs(z, ids, 3)                       # two calls at once
    torch.cuda.synchronize()
    assert all(torch.equal(p, w) and torch.equal(q, w) for p, q, w in zip(a, b, want))
    static, g = z.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.token_logprobs(static, ids, 3)
    static.copy_(z.flip(0))
    g.replay()
    want = ops.token_logprobs(z.flip(0), ids, 3)
    assert all(torch.equal(p, w) for p, w in zip(got, want))


@pytest.mark.gpu
def test_no_rows():
    got = ops.token_logprobs(torch.empty((0, 9), device=DEV), torch.empty(0, dtype=torch.int32, device=DEV), 2)
    assert got.logprob.shape == (0,) and got.top_ids.shape == (0, 2)
    got = ops.token_logprobs(torch.zeros((2, 9), device=DEV), torch.empty((2, 0), dtype=torch.int32, device=DEV))
    assert got.logprob.shape == (2, 0) and torch.allclose(got.entropy.cpu(), torch.tensor(math.log(9.0)))


def head_case(r, d, v, seed, std=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((r, d), generator=g).bfloat16()
    w = (torch.randn((v, d), generator=g) * std / math.sqrt(d)).bfloat16()
    return x.to(DEV), w.to(DEV), torch.randint(0, v, (r,), generator=g, dtype=torch.int32).to(DEV)


def head_check(x, w, ids, cap, got, extra=0):
    """A logit is a sum of d exact products: every 16 of them are added with one rounding towards zero (2^-23 of a partial sum, which
    is at most the sum of magnitudes), so it is off by d / 16 + 8 such roundings; log p moves by the errors of the token's logit and of
    the weighted logits, H by the logits' errors times 2 (1 + spread of the logits)."""
    z = x.double() @ w.double().t()
    mag = (x.double().abs() @ w.double().abs().t()).max()
    dz = float(mag) * (x.shape[1] / 16 + 8) * 2 ** -23
    if cap:
        z = cap * torch.tanh(z / cap)
    lp, h, _, _ = oracle(z, ids, 0)
    spread = float(z.max() - z.min())
    rel = (w.shape[0] / 256 + 64) * EPS
    same(got.logprob, lp, 2 * dz + rel + 8 * EPS * (lp.abs() + cap))
    same(got.entropy, h, 2 * (dz + 8 * EPS * cap) * (1 + spread) + 4 * rel * (1 + h))


HEADS = [(1, 8, 1), (1, 64, 300), (3, 72, 1000), (16, 512, 2048), (17, 128, 777), (128, 64, 257), (129, 200, 1025), (300, 1024, 5000), (513, 8, 40),
         (40, 4096, 3001), (5, 64, 100003), (128, 40, 76001), (600, 64, 20000), (257, 1536, 9001)]


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("r,d,v", HEADS)
def test_head_matches_the_definition(r, d, v, cap):
    x, w, ids = head_case(r, d, v, r + d + v)
    head_check(x, w, ids, cap, ops.linear_logprobs(x, ops.LinearWeight("dense", w), ids, softcap=cap))


@pytest.mark.gpu
@pytest.mark.parametrize("cap", [1e-20, 0.5, 3.0, 1e25])
@pytest.mark.parametrize("r", [6, 150])
def test_head_with_caps_of_any_size(r, cap):
    """Logits far below the cap, about it and far beyond: the polynomial, both forms in one group of columns, and saturation."""
    x, w, ids = head_case(r, 64, 700, 11)
    head_check(x, w, ids, cap, ops.linear_logprobs(x, ops.LinearWeight("dense", w), ids, softcap=cap)) if cap < 1e3 else \
        head_check(x, w, ids, 0.0, ops.linear_logprobs(x, ops.LinearWeight("dense", w), ids, softcap=cap))     # (tanh(u) = u to 2^-24 there)


@pytest.mark.gpu
@pytest.mark.parametrize("d,v", [(12, 50), (33, 300)])
def test_head_of_odd_widths_and_fp32(d, v):
    x, w, ids = head_case(5, d, v, 1)
    head_check(x, w, ids, 0.0, ops.linear_logprobs(x, ops.LinearWeight("dense", w), ids))
    head_check(x, w, ids, 0.0, ops.linear_logprobs(x.float(), ops.LinearWeight("dense", w.float()), ids))


@pytest.mark.gpu
def test_head_with_alternatives_and_quantised_weights():
    x, w, ids = head_case(40, 256, 3000, 2)
    got = ops.linear_logprobs(x, ops.LinearWeight("dense", w), ids, top=4)
    z = ops.linear(x, ops.LinearWeight("dense", w), out_fp32=True)
    want = ops.token_logprobs(z, ids, 4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    fp8 = ops.LinearWeight.from_dense(w.cpu().float(), "fp8").to(DEV)
    for rows_ in (x, ops.quant_fp8(x)):
        got = ops.linear_logprobs(rows_, fp8, ids, top=4)
        want = ops.token_logprobs(ops.linear(rows_, fp8), ids, 4)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("r", [7, 200])
def test_head_at_the_edges(r):
    """Tokens of no row and none, int64 tokens, rows of a wider matrix, off 16 bytes and in reverse order, infinities and NaN."""
    x, w, ids = head_case(r, 64, 999, 5)
    lw = ops.LinearWeight("dense", w)
    want = ops.linear_logprobs(x, lw, ids)
    odd = ids.long()
    odd[0], odd[1], odd[2] = -1, 999, 1 << 40
    got = ops.linear_logprobs(x, lw, odd)
    assert float(got.logprob[0]) == 0.0 and bool(torch.isnan(got.logprob[1:3]).all()) and torch.equal(got.logprob[3:], want.logprob[3:])
    assert torch.equal(got.entropy, want.entropy)
    wide = torch.zeros((r, 80), dtype=torch.bfloat16, device=DEV)
    for view in (wide[:, 8:72], wide[:, 3:67], torch.zeros((r, 64 + 1), dtype=torch.bfloat16, device=DEV)[:, 1:]):
        view.copy_(x)
        got = ops.linear_logprobs(view, lw, ids)
        assert torch.equal(got.logprob, want.logprob) and torch.equal(got.entropy, want.entropy)
    got = ops.linear_logprobs(x.t().contiguous().t(), lw, ids)
    assert torch.equal(got.logprob, want.logprob)
    x = x.clone()
    x[0, 0], x[1, 5], x[2] = INF, NAN, 0.0
    w2 = w.clone()
    w2[:, 0] = w2[:, 0].abs()                              # row 0: every logit +inf
    z = x.double() @ w2.double().t()
    got = ops.linear_logprobs(x, ops.LinearWeight("dense", w2), ids)
    lp, h, _, _ = oracle(z[:3], ids[:3], 0)
    same(got.logprob[:3], lp, 1e-5)                        # logarithms of 999, rounded to 2^-24 twice, and sums of 999 equal terms
    same(got.entropy[:3], h, 1e-5)
    assert bool(torch.isfinite(got.logprob[3:]).all())     # a row's values reach no other row


@pytest.mark.gpu
def test_head_of_nothing_but_minus_infinity():
    x = torch.ones((2, 8), dtype=torch.bfloat16, device=DEV)
    w = torch.full((300, 8), -INF, dtype=torch.bfloat16, device=DEV)
    for rows_ in (x, x.repeat(100, 1)):
        got = ops.linear_logprobs(rows_, ops.LinearWeight("dense", w), torch.zeros(rows_.shape[0], dtype=torch.int32, device=DEV))
        assert bool((got.logprob == -INF).all()) and bool((got.entropy == 0).all())
        w2 = w.clone()
        w2[::3] = 0.25                                     # 100 tokens of one logit each
        got = ops.linear_logprobs(rows_, ops.LinearWeight("dense", w2), torch.ones(rows_.shape[0], dtype=torch.int32, device=DEV))
        assert bool((got.logprob == -INF).all())
        same(got.entropy, torch.full((rows_.shape[0],), math.log(100.0), dtype=torch.float64), 1e-5)


@pytest.mark.gpu
def test_head_in_chunks_streams_and_graphs(monkeypatch):
    x, w, ids = head_case(700, 72, 1111, 6)
    lw = ops.LinearWeight("dense", w)
    want = ops.linear_logprobs(x, lw, ids)
    monkeypatch.setattr(LP, "CHUNK_ROWS", 256)
    got = ops.linear_logprobs(x, lw, ids)
    monkeypatch.undo()
    assert torch.equal(got.logprob, want.logprob) and torch.equal(got.entropy, want.entropy)
    few = x[:9].clone()
    first = ops.linear_logprobs(few, lw, ids[:9])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        a, b = ops.linear_logprobs(few, lw, ids[:9]), ops.linear_logprobs(x, lw, ids)
    c, d = ops.linear_logprobs(x, lw, ids), ops.linear_logprobs(few, lw, ids[:9])
    torch.cuda.synchronize()
    for got, whole in ((a, first), (b, want), (c, want), (d, first)):
        assert torch.equal(got.logprob, whole.logprob) and torch.equal(got.entropy, whole.entropy)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        p = ops.linear_logprobs(few, lw, ids[:9])
    with torch.cuda.graph(g2):
        q = ops.linear_logprobs(x, lw, ids)
    few.copy_(x[100:109])
    for g in (g1, g2, g1):
        g.replay()
    again = ops.linear_logprobs(x[100:109], lw, ids[:9])
    assert torch.equal(p.logprob, again.logprob) and torch.equal(q.logprob, want.logprob) and torch.equal(q.entropy, want.entropy)
    assert ops.device_status(x.device) == 0


def far(v, dtype, seed=0):
    """Rows whose largest logit, or whose masks, lie where a product with log2(e) is rounded by more than an exponential bears: beyond 1e9 on
    either side, and on both sides of the border (2^23; of fp16 -59000) between the sums' two references, in every part of a row."""
    g = torch.Generator().manual_seed(seed)
    noise = torch.randn(v, generator=g) * 2
    first = torch.arange(v) < v // 2
    half = torch.finfo(dtype).max < 1e6
    out = []
    for top in (6e4, -6e4) if half else (5e9, 1e10, 1e12, 1e20, 1e28, -3e9):
        z = noise.clone()
        z[v // 3] = top
        out += [z, z.flip(0)]
    for level in (-59000.0, -60000.0, -65504.0) if half else (-3e9, -1e10, -1e11, -1e12, -1e15, 1e10, 1e20):
        out.append(torch.full((v,), level))
    for mask in (-59000.0, -6e4) if half else (-1e7, -1.7e9, -2.5e9, -1e10, -1e15):
        out += [torch.where(first, mask, noise), torch.where(first, noise, mask), torch.where(torch.arange(v) % 64 < 40, mask, noise)]
    step = 32.0 if half else 1.0                           # (a unit in the last place there)
    for border in (-59008.0,) if half else (2.0 ** 23, -2.0 ** 23):
        ladder = border + step * torch.randint(-3, 4, (v,), generator=g)
        low, high = border - step * (1 + torch.arange(v) % 2), border + step * (1 + torch.arange(v) % 2)
        out += [ladder, torch.where(first, low, high), torch.where(first, high, low), torch.where(torch.arange(v) == v - 1, high, low),
                torch.where(torch.arange(v) == 0, high, low)]
    return torch.stack(out).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("v", [5, 33, 1000, 20011, 131077])
@pytest.mark.parametrize("top", [0, 6])
def test_rows_far_from_zero(dtype, v, top):
    z = far(v, dtype, v)
    ids = torch.stack([torch.zeros(len(z)), torch.full((len(z),), v - 1), torch.full((len(z),), v // 3), torch.full((len(z),), v // 2)], 1).long()
    check(z, ids, top, ops.token_logprobs(z.to(DEV), ids.to(DEV), top))
    for i in range(len(z)):                                # a row by itself: as many CTAs share it as may
        check(z[i:i + 1], ids[i:i + 1], top, ops.token_logprobs(z[i:i + 1].to(DEV), ids[i:i + 1].to(DEV), top))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,v", [(torch.float32, 32771), (torch.bfloat16, 65543), (torch.float16, 65543)])
@pytest.mark.parametrize("top", [0, 6])
def test_many_rows_far_from_zero(dtype, v, top):
    """In the form for many long rows."""
    z = far(v, dtype, v)
    n = len(z)
    ids = torch.stack([torch.zeros(n), torch.full((n,), v - 1), torch.full((n,), v // 3)], 1).long()
    times = 2400 // n + 1
    got = ops.token_logprobs(z.to(DEV).repeat(times, 1), ids.to(DEV).repeat(times, 1), top)
    for k in (0, times - 1):
        check(z, ids, top, ops.TokenLogprobs(*(None if f is None else f[n * k:n * (k + 1)] for f in got)))


def _w4(w, fmt="nvfp4"):
    from sllm_b200.ops.w4 import W4Weight
    return ops.LinearWeight("w4", None, None, W4Weight.quantize(fmt, w))


def test_operand_types_of_linear_logprobs():
    """Types that a kernel would read as others are refused: on the CPU what no product takes, with a stand-in for the library what the
    kernels take in one type only."""
    ids = torch.zeros(3, dtype=torch.int64)
    dense = lambda dt: ops.LinearWeight("dense", torch.zeros((8, 128), dtype=dt))
    fp8 = ops.LinearWeight.from_dense(torch.randn(8, 128), "fp8")
    rows_ = lambda dt: torch.zeros((3, 128), dtype=dt)
    q = ops.quant_fp8(torch.randn(3, 128))
    never = [(rows_(torch.float16), dense(torch.bfloat16)), (rows_(torch.float16), dense(torch.float16)), (rows_(torch.float32), dense(torch.float16)),
             (rows_(torch.int32), dense(torch.float32)), (rows_(torch.float64), dense(torch.float64)), (rows_(torch.float16), fp8), (q, dense(torch.bfloat16)),
             (ops.QTensor(q.data, q.scale[:, :2]), fp8), (ops.QTensor(q.data, q.scale.double()), fp8), (ops.QTensor(q.data.float(), q.scale), fp8),
             (ops.QTensor(q.data[0], q.scale), fp8), (rows_(torch.float16), _w4(torch.randn(8, 128))), (q, _w4(torch.randn(8, 128))), (None, fp8),
             (rows_(torch.float32), ops.LinearWeight("fp8", fp8.w, fp8.scale_t.to("meta"))), (rows_(torch.float32).to("meta"), _w4(torch.randn(8, 128)))]
    on_a_gpu = [(rows_(torch.float32), dense(torch.bfloat16)), (rows_(torch.bfloat16), dense(torch.float32)), (rows_(torch.float32), fp8),
                (rows_(torch.float32), _w4(torch.randn(8, 128))),
                (rows_(torch.bfloat16), ops.LinearWeight("dense", torch.zeros((8, 256), dtype=torch.bfloat16)[:, :128])),
                (rows_(torch.float32), ops.LinearWeight("dense", torch.zeros((128, 8)).t())),
                (rows_(torch.bfloat16), ops.LinearWeight("fp8", torch.zeros((8, 256), dtype=torch.uint8)[:, :128], fp8.scale_t))]
    for x, w in on_a_gpu[:4]:
        ops.linear_logprobs(x, w, ids)                     # (the CPU's oracle takes them as they are)
    fake = _lib.FakeKernelLibrary()
    for x, w in never:
        with pytest.raises(ValueError):
            ops.linear_logprobs(x, w, ids)
    _lib.install_fake(fake)
    try:
        for x, w in never + on_a_gpu:
            for top in (0, 2):
                with pytest.raises(ValueError):
                    ops.linear_logprobs(x, w, ids, top=top)
        assert not [c for c in fake.calls if c[0] != "sllm_head_logprobs_floats"]
        # rows that the quantiser, which takes no stride, would read from elsewhere
        wide = torch.zeros((3, 256), dtype=torch.bfloat16)
        for x in (wide[:, :128], wide[:, ::2], torch.zeros((128, 3), dtype=torch.bfloat16).t(), torch.zeros((3, 129), dtype=torch.bfloat16)[:, 1:]):
            fake.calls.clear()
            ops.linear_logprobs(x, fp8, ids)
            at = [c[1][0] for c in fake.calls if c[0] == "sllm_quant_fp8_1x128"]
            assert len(at) == 1 and getattr(at[0], "value", at[0]) != x.data_ptr()
    finally:
        _lib.install_fake(None)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["dense", "fp32", "fp8", "w4"])
@pytest.mark.parametrize("top", [0, 3])
@pytest.mark.parametrize("r", [1, 5, 140])
def test_rows_of_any_strides_give_the_same(kind, top, r):
    x, w, ids = head_case(r, 128, 1000, 4)
    lw = {"dense": lambda: ops.LinearWeight("dense", w), "fp32": lambda: ops.LinearWeight("dense", w.float()),
          "fp8": lambda: ops.LinearWeight.from_dense(w.cpu().float(), "fp8").to(DEV), "w4": lambda: _w4(w.cpu().float()).to(DEV)}[kind]()
    x = x.float() if kind == "fp32" else x
    want = ops.linear_logprobs(x, lw, ids, top=top)
    new = lambda *shape: torch.full(shape, 9.0, dtype=x.dtype, device=DEV)
    for view in (new(r, 256)[:, 8:136], new(r, 256)[:, ::2], new(r, 256)[:, 3:131], new(128, r).t(), new(r, 129)[:, 1:], new(r, 1, 128)[:, 0]):
        view.copy_(x)
        got = ops.linear_logprobs(view, lw, ids, top=top)
        assert all(a is None or torch.equal(a, b) for a, b in zip(got, want))
    one = x[:1].expand(r, -1)
    assert all(a is None or torch.equal(a, b) for a, b in zip(ops.linear_logprobs(one, lw, ids, top=top), ops.linear_logprobs(one.contiguous(), lw, ids, top=top)))


def test_products_run_on_the_device_of_their_rows(monkeypatch):
    """A device that is not current stood in for: it is current while the logits are made."""
    now, seen = [0], []

    class On:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *exc):
            now[0] = self.before

    class Rows:
        is_cuda, dtype, device, shape = True, torch.float32, torch.device("cuda", 1), (3, 8)

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(LP, "_check_operands", lambda x, w: None)
    monkeypatch.setattr(LP, "_check_tokens", lambda *a: None)
    monkeypatch.setattr(LP, "_through_logits", lambda *a: seen.append(now[0]))
    ops.linear_logprobs(Rows(), ops.LinearWeight("dense", torch.zeros(5, 8)), torch.zeros(3, dtype=torch.int64), top=1)
    assert seen == [1] and now == [0]


@pytest.mark.gpu
@pytest.mark.parametrize("r", [8, 200])
def test_head_sums_leave_the_tensor_core_every_512_columns(r):
    """One product of 1 and 4095 of 2^-26, which next to it a tensor core's sum loses: those of its chain of 512 columns, 511 of them, while
    the others reach the token's logit whole.  A chain of 1024 loses 1023, 1.4e-5 of the log-probability (the token has 0.07 of the row).
    Beside the loss: 8 chains added to about 1; 40 terms of the row's sum, added in pairs by a thread and joined (20 + 8 roundings, an
    exponential's 2^-22), and 8 roundings of numbers of the result's size."""
    d, v = 4096, 40
    w = torch.zeros((v, d))
    w[0] = 2.0 ** -26
    w[0, 0] = 1.0
    x, w = torch.ones((r, d), dtype=torch.bfloat16, device=DEV), w.bfloat16().to(DEV)
    ids = torch.zeros(r, dtype=torch.int32, device=DEV)
    got = ops.linear_logprobs(x, ops.LinearWeight("dense", w), ids)
    lp = torch.log_softmax(x.double() @ w.double().t(), 1)[:, 0].cpu()
    tol = 511 * 2.0 ** -26 + (8 + 20 + 8 + 4) * EPS + 8 * EPS * float(lp.abs().max())
    assert tol < 1023 * 2.0 ** -26 * (1 - math.exp(float(lp.max()))) - 2e-6
    same(got.logprob, lp, tol)
