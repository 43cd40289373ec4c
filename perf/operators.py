"""What the operators around a model's step are judged by: the step's batch laid out on the GPU from request lengths
(`ops.batch_plan`), log-probabilities of given tokens from logits (`ops.token_logprobs`) and from hidden rows and the output
matrix without writing logits (`ops.linear_logprobs`).

A case's `op`:
  plan    `requests` with `new` tokens each (`ragged`: between 1 and `new`) behind up to `cached` tokens of their pages; the batch has
          `pad` rows more than tokens, the table `blocks` columns
  tokens  `rows` of `vocab` logits of type `dtype`, `given` tokens per row (0: one, without an axis for it), `top` alternatives;
          rows lie `gap` elements apart beyond their length, the first one `shift` elements into its storage; `banned` of every 16 tokens
          are shut out with -inf (a grammar's mask)
  head    `rows` of `width` hidden values against a matrix of `vocab` rows, `cap` the soft cap of the logits (0: none)
"""
import math

import torch

own = False
DEV = "cuda"
PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def plan(name, requests, new, ragged, cached, pad, blocks):
    return {"name": name, "op": "plan", "requests": requests, "new": new, "ragged": ragged, "cached": cached, "pad": pad, "blocks": blocks}


def tokens(name, rows, vocab, dtype="bf16", given=0, top=0, gap=0, shift=0, banned=0):
    return {"name": name, "op": "tokens", "rows": rows, "vocab": vocab, "dtype": dtype, "given": given, "top": top, "gap": gap,
            "shift": shift, "banned": banned}


def head(name, rows, width, vocab, cap=0.0):
    return {"name": name, "op": "head", "rows": rows, "width": width, "vocab": vocab, "cap": cap}


def listed():
    return [
        # one token for each of 64 running requests, a context of up to 8192
        plan("plan_decode", 64, 1, False, 8000, 0, 512),
        # requests in every phase at once, a context of 131072, rows rounded up for a captured step
        plan("plan_mixed", 300, 200, True, 100000, 37, 8192),
        # one long fresh prompt
        plan("plan_prompt", 1, 65536, False, 0, 0, 4096),
        # the answer to one streamed token, with its alternatives
        tokens("tokens_one", 1, 128256, top=20),
        # a step of 64 requests that ask for five alternatives; a grammar shuts out most of the vocabulary
        tokens("tokens_batch", 64, 201088, top=5, banned=15),
        # odd sizes: logits of an unpadded vocabulary in fp32, which starts in the middle of a 16-byte unit
        tokens("tokens_odd", 37, 50021, dtype="fp32", top=8, gap=3, shift=1),
        # choices of a multiple-choice question at every place of some prompts, in fp16
        tokens("tokens_choices", 1500, 32768, dtype="fp16", given=4),
        # every token of a long text with its alternatives
        tokens("tokens_prompt", 4096, 128256, top=5),
        # one token against the whole output matrix
        head("head_one", 1, 4096, 128256),
        # the last places of 48 prompts, a width of no power of two
        head("head_batch", 48, 2880, 201088),
        # a prompt of odd length, capped logits
        head("head_odd", 777, 2560, 151936, cap=30.0),
        # every token of a long text
        head("head_prompt", 4096, 4096, 128256),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "tokens", "tokens", "head", "head"])
    if op == "plan":
        requests = _log(rng, 1, 1024)
        new = rng.choice([1, _log(rng, 1, max(1, 65536 // requests))])
        blocks = _log(rng, 256, min(8192, 2500000 // requests))
        cached = rng.choice([0, max(0, min(100000, blocks * PAGE - new))])
        new = min(new, blocks * PAGE - cached)
        c = plan("", requests, new, rng.random() < 0.7, cached, rng.choice([0, _log(rng, 1, 100)]), blocks)
    elif op == "tokens":
        rows = _log(rng, 1, 4096)
        vocab = _log(rng, 1000, min(262144, 4096 * 128256 // (2 * rows)))
        c = tokens("", rows, vocab, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice([0, 0, 1, 5]), rng.choice([0, 1, 5, 20, 32]),
                   rng.choice([0, 0, 8, 13]), rng.choice([0, 0, 3, 5]), rng.choice([0, 0, 8, 15]))
    else:
        rows = _log(rng, 1, 4096)
        c = head("", rows, 8 * _log(rng, 32, 512), _log(rng, 1000, 128256), rng.choice([0.0, 0.0, 30.0]))
    del c["name"]
    return c


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def prepare(case, seed):
    g = _generator(seed)
    st = {"case": case}
    if case["op"] == "plan":
        s = case["requests"]
        new = torch.full((s,), case["new"], dtype=torch.int32, device=DEV)
        if case["ragged"]:                                         # the same lengths in another order, so that the batch keeps its size
            spread = 1 + torch.arange(s, device=DEV) * case["new"] // s
            new = spread[torch.randperm(s, generator=g, device=DEV)].to(torch.int32)
        starts = torch.randint(0, case["cached"] + 1, (s,), generator=g, dtype=torch.int32, device=DEV)
        count = int(((starts + new + PAGE - 1) // PAGE).sum())
        pool = max(count, 1) + 64
        # what a program holds: the requests' lengths, what is cached of each, and their pages one after another
        st.update(new=new, starts=starts, pages=torch.randperm(pool, generator=g, device=DEV)[:count].to(torch.int32),
                  rows=int(new.sum()) + case["pad"])
    elif case["op"] == "tokens":
        r, v = case["rows"], case["vocab"]
        ld = v + case["gap"]
        store = torch.empty(case["shift"] + r * ld, dtype=DTYPES[case["dtype"]], device=DEV)
        for i in range(0, store.numel(), 1 << 27):                 # (in parts: fp32 normals of the largest would be 2 GB)
            part = store[i:i + (1 << 27)]
            part.copy_(torch.randn(part.numel(), generator=g, device=DEV) * 2.5)
        logits = store[case["shift"]:].view(r, ld)[:, :v]
        ids = torch.randint(0, v, (r, max(1, case["given"])), generator=g, device=DEV, dtype=torch.int32)
        if case["banned"]:
            shut = torch.rand(v, generator=g, device=DEV) < case["banned"] / 16
            shut[int(torch.randint(0, v, (1,), generator=g, device=DEV))] = False
            logits[:, shut] = float("-inf")
            allowed = torch.nonzero(~shut)[:, 0].to(torch.int32)   # a grammar's tokens are among the allowed ones
            ids = allowed[ids.long() % allowed.numel()]
        # a trained model is sure of some tokens: a third of the rows has one that stands out
        sure = torch.arange(0, r, 3, device=DEV)
        logits[sure, ids[sure, 0].long()] = 14.0
        st.update(logits=logits, ids=ids if case["given"] else ids[:, 0].contiguous())
    else:
        r, d, v = case["rows"], case["width"], case["vocab"]
        w = torch.empty((v, d), dtype=torch.bfloat16, device=DEV)
        for i in range(0, v, 16384):
            w[i:i + 16384] = torch.randn((min(16384, v - i), d), generator=g, device=DEV) * (2.5 / math.sqrt(d))
        x = torch.randn((r, d), generator=g, device=DEV).to(torch.bfloat16)
        st.update(x=x, w=w, ids=torch.randint(0, v, (r,), generator=g, device=DEV, dtype=torch.int32))
        if own:
            from sllm_b200.ops import LinearWeight
            st["weight"] = LinearWeight("dense", w)
    return st


def _plain_plan(new, starts, pages, rows, blocks):
    new, starts, pages = new.long(), starts.long(), pages.long()
    s, count = new.numel(), (starts + new + PAGE - 1) // PAGE
    ends, page_ends = torch.cumsum(new, 0), torch.cumsum(count, 0)
    row_off = torch.cat([ends.new_zeros(1), ends])
    at = torch.arange(rows, device=new.device)
    seq = torch.searchsorted(ends, at, right=True)
    live = seq < s
    seq = torch.where(live, seq, torch.zeros_like(seq))
    pos = starts[seq] + at - row_off[seq]
    first = page_ends - count
    slot = pages[torch.where(live, first[seq] + pos // PAGE, torch.zeros_like(at))] * PAGE + pos % PAGE
    col = torch.arange(blocks, device=new.device)
    used = col[None, :] < count[:, None]
    table = torch.where(used, pages[torch.where(used, first[:, None] + col[None, :], torch.zeros_like(col)[None, :])], torch.zeros_like(col)[None, :])
    neg = torch.full_like(at, -1)
    i32 = lambda t: t.to(torch.int32)
    return {"row_off": i32(row_off), "positions": i32(torch.where(live, pos, neg)), "seq_index": i32(torch.where(live, seq, neg)),
            "kv_lens": i32(torch.where(live, pos + 1, torch.zeros_like(pos))), "slots": torch.where(live, slot, neg),
            "last_rows": ends - 1, "block_table": i32(table)}


def _logp(z, ids):
    """z [R, V] fp32 -> log-probabilities of ids [R, N] and the entropy."""
    m = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - m)
    s = e.sum(dim=1, keepdim=True)
    d = torch.where(e > 0, z - m, torch.zeros_like(z))
    entropy = torch.log(s[:, 0]) - (e * d).sum(dim=1) / s[:, 0]
    return z.gather(1, ids.long()) - m - torch.log(s), entropy, m + torch.log(s)


def _plain_tokens(logits, ids, top):
    z = logits.float()
    many = ids if ids.dim() == 2 else ids[:, None]
    lp, entropy, lse = _logp(z, many)
    out = {"logprob": lp if ids.dim() == 2 else lp[:, 0], "entropy": entropy}
    if top:
        bits = (z + 0.0).view(torch.int32).long()                  # order of the values (-0 is 0), ties to the lower id
        key = torch.where(bits < 0, -1 - (bits & 0x7fffffff), bits) * (1 << 20) - torch.arange(z.shape[1], device=z.device)
        best = torch.topk(key, top, dim=1).indices
        val = z.gather(1, best)
        none = torch.isinf(val) & (val < 0)
        out["top_ids"] = torch.where(none, torch.full_like(best, -1), best).to(torch.int32)
        out["top_logprobs"] = val - lse
    return out


def run(state):
    case = state["case"]
    if case["op"] == "plan":
        if own:
            from sllm_b200 import ops
            p = ops.batch_plan(state["new"], state["starts"], state["pages"], rows=state["rows"], max_blocks=case["blocks"], page_size=PAGE)
            return p._asdict()
        return _plain_plan(state["new"], state["starts"], state["pages"], state["rows"], case["blocks"])
    if case["op"] == "tokens":
        if own:
            from sllm_b200 import ops
            p = ops.token_logprobs(state["logits"], state["ids"], top=case["top"])
            return {k: v for k, v in p._asdict().items() if v is not None}
        return _plain_tokens(state["logits"], state["ids"], case["top"])
    if own:
        from sllm_b200 import ops
        p = ops.linear_logprobs(state["x"], state["weight"], state["ids"], softcap=case["cap"])
        return {"logprob": p.logprob, "entropy": p.entropy}
    z = state["x"].float() @ state["w"].float().t()
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    lp, entropy, _ = _logp(z, state["ids"][:, None])
    return {"logprob": lp[:, 0], "entropy": entropy}


def work(case):
    if case["op"] == "plan":
        s, new = case["requests"], case["new"]
        rows = sum(1 + i * new // s for i in range(s)) if case["ragged"] else s * new
        pages = s * (case["cached"] / 2 + rows / s) / PAGE
        # lengths and pages in; offsets, last rows and the table out, and position, request, keys and slot of every row
        nbytes = 8 * s + 4 * pages + 4 * (s + 1) + 8 * s + 4 * s * case["blocks"] + 20 * (rows + case["pad"])
        return {"bytes": int(nbytes), "flops": int(2 * (rows + case["pad"]) + s * case["blocks"])}
    if case["op"] == "tokens":
        r, v, n = case["rows"], case["vocab"], max(1, case["given"])
        size = DTYPES[case["dtype"]].itemsize
        # difference, exponential, two sums and a product per logit
        return {"bytes": r * v * size + r * (8 * n + 4 + 8 * case["top"]), "flops": 5 * r * v}
    r, d, v = case["rows"], case["width"], case["vocab"]
    return {"bytes": 2 * d * (r + v) + 12 * r, "flops": 2 * r * d * v + 5 * r * v}


def _exact_rows(z, ids, top):
    """fp64 logits of some rows, from the definition: p = exp(z) / sum exp(z), entropy = - sum p log p."""
    logp = z - torch.logsumexp(z, dim=1, keepdim=True)
    p = torch.exp(logp)
    out = {"logprob": logp.gather(1, ids.long()), "entropy": -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(dim=1)}
    if top:
        val, at = torch.sort(z, dim=1, descending=True, stable=True)
        val, at = val[:, :top], at[:, :top].to(torch.int32)
        out["top_ids"] = torch.where(torch.isinf(val), torch.full_like(at, -1), at)
        out["top_logprobs"] = logp.gather(1, at.long())
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "plan":
        new, starts, pages = (st[k].tolist() for k in ("new", "starts", "pages"))
        rows, table, off = [], [], [0]
        at = 0
        for i, (n, s0) in enumerate(zip(new, starts)):
            used = -(-(s0 + n) // PAGE)
            mine = pages[at:at + used]
            at += used
            rows += [(s0 + j, i, s0 + j + 1, mine[(s0 + j) // PAGE] * PAGE + (s0 + j) % PAGE) for j in range(n)]
            off.append(off[-1] + n)
            table.append(mine + [0] * (case["blocks"] - used))
        rows += [(-1, -1, 0, -1)] * case["pad"]
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
        i64 = lambda x: torch.tensor(x, dtype=torch.int64, device=DEV)
        col = list(zip(*rows))
        return {"row_off": i32(off), "positions": i32(col[0]), "seq_index": i32(col[1]), "kv_lens": i32(col[2]), "slots": i64(col[3]),
                "last_rows": i64([o - 1 for o in off[1:]]), "block_table": i32(table)}
    r, v = case["rows"], case["vocab"]
    step = max(1, (1 << 26) // v)
    ids = st["ids"]
    many = ids if ids.dim() == 2 else ids[:, None]
    top = case.get("top", 0)
    w = st["w"].double() if case["op"] == "head" else None
    parts = []
    for i in range(0, r, step):
        if w is None:
            z = st["logits"][i:i + step].double()
        else:
            z = st["x"][i:i + step].double() @ w.t()
            if case["cap"]:
                z = case["cap"] * torch.tanh(z / case["cap"])
        parts.append(_exact_rows(z, many[i:i + step], top))
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if ids.dim() == 1:
        out["logprob"] = out["logprob"][:, 0]
    return out
