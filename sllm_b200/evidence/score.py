"""Score runner: the log-probabilities that a model gives the tokens of texts, and their perplexity.

    python -m sllm_b200.evidence.score --gguf M --derived-lock L [--text T]... [--input-token-ids "1 2 3"]... [--top K] [--cpu]

Prints one JSON line (schema ``sllm-score-v1``): per text its tokens, the log-probability of every token after the first, the
entropy of the distribution it was taken from, the mean negative log-likelihood and the perplexity (null for a text of one
token), and with ``--top`` the likeliest tokens of every place.  Numbers that are not finite (a token that is shut out, logits
that are NaN) are null.  Exit codes as the command line's (2 usage, 3 model file, 4 device).
"""
from __future__ import annotations

import math
import sys

from ..cli.common import CliError, StrictParser, add_model_source, emit, open_model, run_main

SCHEMA = "sllm-score-v1"


def _finite(x):
    return [_finite(v) for v in x] if isinstance(x, list) else x if x is not None and math.isfinite(x) else None


def score_texts(eng, token_lists: list, top: int = 0) -> list:
    """One record per token list, from `Engine.score`."""
    out = []
    for ids, lp in zip(token_lists, eng.score(token_lists, top)):
        n = lp.logprob.numel()
        nll = -float(lp.logprob.double().sum()) / n if n else None
        rec = {"tokens": list(ids), "logprobs": _finite(lp.logprob.tolist()), "entropy": _finite(lp.entropy.tolist()), "nll_mean": _finite(nll),
               "perplexity": math.exp(nll) if n and nll < 700 else None}
        if top:
            rec["top"] = [[{"token": t, "logprob": _finite(p)} for t, p in zip(ts, ps) if t >= 0]
                          for ts, ps in zip(lp.top_ids.tolist(), lp.top_logprobs.tolist())]
        out.append(rec)
    return out


def main(argv=None) -> int:
    def go():
        p = StrictParser(prog="python -m sllm_b200.evidence.score")
        add_model_source(p)
        p.add_argument("--text", action="append", default=[])
        p.add_argument("--input-token-ids", action="append", default=[])
        p.add_argument("--top", type=int, default=0)
        a = p.parse_args(argv)
        if not a.text and not a.input_token_ids:
            raise CliError("give --text or --input-token-ids")
        eng, tok, g, lock = open_model(a)
        lists = [tok.encode(t) for t in a.text]
        try:
            lists += [[int(x) for x in s.replace(",", " ").split()] for s in a.input_token_ids]
        except ValueError:
            raise CliError("--input-token-ids must be integers") from None
        try:
            recs = score_texts(eng, lists, a.top)
        except ValueError as exc:
            raise CliError(str(exc)) from None
        emit({"schema": SCHEMA, "model": lock["semantic_model_id"], "texts": recs})

    return run_main(go)


if __name__ == "__main__":
    sys.exit(main())
