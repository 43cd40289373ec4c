"""Log-probabilities of given tokens with the entropy of their rows and the likeliest alternatives: from logits
(csrc/logprobs.cu) and from hidden rows and the output matrix.  CPU tensors run the restatement below, in 64 bits."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib, core
from .core import _launch

P, I, L = C.c_void_p, C.c_int, C.c_longlong
_SIGS = {
    "sllm_token_logprobs": (I, [P, L, I, I, I, P, I, I, I, P, P, P, P, P]),
    "sllm_head_logprobs_floats": (L, [I, I, I]),
    "sllm_head_logprobs": (I, [P, P, P, I, I, I, L, C.c_float, I, P, L, P, P, P, P]),
}
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_TOP = 32
MAX_VOCAB = 1 << 30
MIN_CAP, MAX_CAP = 1e-30, 1e30 # whose reciprocals are normal numbers
FEW_ROWS = 128                 # up to here a row's tile is shared by no CTA pair (csrc/head_logprobs.cu)
CHUNK_LOGITS = 1 << 27         # logits that `linear_logprobs` holds at a time where it writes them
CHUNK_FLOATS = 1 << 25         # floats of its workspace where it does not (a thirty-second of the logits' number, with narrow tiles a sixteenth),
CHUNK_ROWS = 1 << 15           # and rows of a launch


_lib.EXTRA_KERNEL_SIGNATURES.update(_SIGS)
_k = _lib.kernels


class TokenLogprobs(NamedTuple):
    """fp32, in nats.  ``top_ids`` / ``top_logprobs`` [R, top]: the largest logits, equal ones by id; -1 / -inf where a row has fewer
    tokens."""
    logprob: torch.Tensor                          # of the given tokens, in their shape
    entropy: torch.Tensor                          # [R]
    top_ids: Optional[torch.Tensor] = None         # int32
    top_logprobs: Optional[torch.Tensor] = None


def chunk_rows(vocab: int) -> int:
    """Rows whose logits are written at a time: whole tiles of 256 where there are that many."""
    rows = max(1, CHUNK_LOGITS // vocab)
    return rows // 256 * 256 or rows


def _check_tokens(tokens: torch.Tensor, rows: int, device) -> None:
    if tokens.dtype not in (torch.int32, torch.int64) or tokens.dim() not in (1, 2) or tokens.shape[0] != rows or tokens.device != device:
        raise ValueError("tokens are int32 or int64 [rows] or [rows, n] on the device of the rows")


def _cpu(logits: torch.Tensor, tokens: torch.Tensor, top: int) -> TokenLogprobs:
    z = logits.double()
    r, v = z.shape
    inf = float("inf")
    nan = torch.isnan(z).any(1)
    up = (z == inf).any(1)
    z = torch.where(up[:, None], torch.where(z == inf, torch.zeros_like(z), torch.full_like(z, -inf)), z)
    empty = (z == -inf).all(1)
    d = z - z.max(1, keepdim=True).values                  # (first: the logarithm is lost next to a logit of the type's lowest value)
    logp = torch.where(empty[:, None], z, d - torch.logsumexp(d, 1, keepdim=True))
    p = torch.exp(logp)
    entropy = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    logp = torch.where(nan[:, None], torch.full_like(logp, float("nan")), logp)
    entropy = torch.where(nan, torch.full_like(entropy, float("nan")), entropy)
    ids = tokens.long() if tokens.dim() == 2 else tokens.long()[:, None]
    lp = logp.gather(1, ids.clamp(0, v - 1))
    lp = torch.where(ids < 0, torch.zeros_like(lp), torch.where(ids >= v, torch.full_like(lp, float("nan")), lp))
    out = [lp.float().reshape(tokens.shape), entropy.float(), None, None]
    if top:
        n = min(top, v)
        val, at = torch.sort(torch.nan_to_num(logits.double(), nan=-inf, posinf=inf, neginf=-inf), dim=1, descending=True, stable=True)
        none = (val[:, :n] == -inf) | nan[:, None]
        top_ids = torch.full((r, top), -1, dtype=torch.int32)
        top_lp = torch.full((r, top), -inf)
        top_ids[:, :n] = torch.where(none, -1, at[:, :n]).to(torch.int32)
        top_lp[:, :n] = torch.where(none, torch.tensor(-inf, dtype=torch.float64), logp.gather(1, at[:, :n])).float()
        top_lp[nan] = float("nan")
        out[2:] = [top_ids, top_lp]
    return TokenLogprobs(*out)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Log-probabilities of ``tokens`` (int32 / int64 [R] or [R, n]) under the rows of ``logits`` (bf16, fp16 or fp32 [R, V], rows of
    any stride), the rows' entropies and their ``top`` (0 to 32) likeliest tokens.  -inf logits are shut out: a row of nothing else has
    log-probabilities of -inf, entropy 0 and no alternatives.  A row with +inf is uniform over those; one with NaN gives NaN and no
    alternatives.  A token below 0 stands for none (0, so that padded places drop out of sums), one from V on gives NaN."""
    if (logits.dim() != 2 or logits.dtype not in _DTYPES or not 1 <= logits.shape[1] <= MAX_VOCAB
            or (logits.shape[1] > 1 and logits.stride(1) != 1) or logits.shape[0] >= 2 ** 31):
        raise ValueError(f"logits are bf16, fp16 or fp32 [rows, vocabulary] with contiguous rows of at most {MAX_VOCAB}")
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top lies between 0 and {MAX_TOP}")
    _check_tokens(tokens, logits.shape[0], logits.device)
    if _lib.on_cpu(logits):
        return _cpu(logits, tokens, top)
    r, v = logits.shape
    dev = logits.device
    tokens = tokens.contiguous()
    given = tokens.shape[1] if tokens.dim() == 2 else 1
    n = r * given
    out = torch.empty(n + r + 2 * r * top, dtype=torch.float32, device=dev)      # (one allocation: four cost more than a row's kernel)
    lp = out.as_strided(tokens.shape, (given, 1) if tokens.dim() == 2 else (1,), 0)
    entropy = out.as_strided((r,), (1,), n)
    ids = tlp = None
    if top:
        tlp = out.as_strided((r, top), (top, 1), n + r)
        ids = out.view(torch.int32).as_strided((r, top), (top, 1), n + r + r * top)
    if r:
        at = out.data_ptr()
        rc = _launch(dev, _k().sllm_token_logprobs, logits.data_ptr(), logits.stride(0), r, v, _DTYPES[logits.dtype], tokens.data_ptr(),
                     tokens.dtype == torch.int64, given, top, at, at + 4 * n, at + 4 * (n + r + r * top) if top else None,
                     at + 4 * (n + r) if top else None)
        _lib.check(rc, "token_logprobs")
        if _lib.audit_enabled():
            _lib.record_dispatch("token_logprobs", "logprobs_kernel", rows=r, vocab=v, top=top)
    return TokenLogprobs(lp, entropy, ids, tlp)


_head_sizes: dict = {}         # (n, bn) -> floats of workspace per row


def _head_floats(n: int, bn: int) -> int:
    floats = _head_sizes.get((n, bn))
    if floats is None:
        floats = int(_k().sllm_head_logprobs_floats(1, n, bn))
        if floats and len(_head_sizes) < 256:        # (0: a stand-in for the library)
            _head_sizes[n, bn] = floats
    return floats


def _check_operands(x, w) -> None:
    """The kernels read rows and weights as bytes of the types and in the order that they expect."""
    xd = x.data if isinstance(x, core.QTensor) else x
    if not isinstance(xd, torch.Tensor) or xd.dim() != 2 or xd.shape[1] != w.in_features:
        raise ValueError("x is [rows, in_features]")
    stored = w.w4.tiles if w.kind == "w4" else w.w
    if any(t is not None and t.device != xd.device for t in (stored, w.scale_t, x.scale if isinstance(x, core.QTensor) else None)):
        raise ValueError("rows and weight are on one device")
    on_gpu = xd.is_cuda or _lib.fake_active()
    if isinstance(x, core.QTensor):
        if w.kind != "fp8" or xd.dtype not in (torch.uint8, torch.float8_e4m3fn) or x.scale.dtype != torch.float32 \
                or x.scale.shape != ((w.in_features + 127) // 128, xd.shape[0]):
            raise ValueError("quantised rows are E4M3 with fp32 scales [width / 128, rows], for FP8 weights")
    elif xd.dtype not in (torch.bfloat16, torch.float32) or (w.kind == "dense" and w.w.dtype not in (torch.bfloat16, torch.float32)):
        raise ValueError("rows and dense weights are bf16 or fp32")
    elif on_gpu and xd.dtype != (w.w.dtype if w.kind == "dense" else torch.bfloat16):
        raise ValueError("on a GPU, rows have a dense weight's type and are bf16 for quantised ones")
    if on_gpu and w.kind != "w4" and not w.w.is_contiguous():
        rows_of_any_stride = w.kind == "dense" and (xd.dtype == torch.float32 or w.in_features % 8 != 0) and w.w.stride(1) == 1
        if not rows_of_any_stride:
            raise ValueError("the weight is contiguous")


def _plain_rows(x: torch.Tensor, strided: bool) -> torch.Tensor:
    """Rows that a TMA copy can address: whole 16-byte units from a 16-byte boundary on, with ``strided`` any number of them apart."""
    if not strided or x.stride(1) != 1 or x.stride(0) % 8 or x.stride(0) < x.shape[1]:
        x = x.contiguous()
        if x.stride(0) != x.shape[1]:                      # (a single row keeps whichever stride it had)
            x = x.as_strided(x.shape, (x.shape[1], 1))
    return x.clone() if x.data_ptr() % 16 else x


def _head(x: torch.Tensor, w: torch.Tensor, tokens: torch.Tensor, softcap: float) -> TokenLogprobs:
    """bf16 rows against a dense matrix on the tensor cores, without logits in memory."""
    r, n, dev = x.shape[0], w.shape[0], x.device
    out = torch.empty(2 * r, dtype=torch.float32, device=dev)
    lp, entropy = out.as_strided((r,), (1,), 0), out.as_strided((r,), (1,), r)
    if not r:
        return TokenLogprobs(lp, entropy)
    x = _plain_rows(x, True)
    if tokens.dtype == torch.int64:
        tokens = tokens.clamp(-1, n).to(torch.int32)
    tokens = tokens.contiguous()
    # tiles of CTA pairs by the rule of products of many rows, which holds here too (us with 128 / 256 columns: 129 x 2000 x 4096 25.3 / 29.2, 129 x
    # 5000 x 4096 24.8 / 27.7, 300 x 5000 x 4096 42.8 / 28.7, 129 x 128256 x 4096 260 / 205; of 90 sizes it lost one, 256 x 9001 x 1536 21.0 / 20.5)
    bn = 0 if r <= FEW_ROWS else core._prompt_tile(min(r, CHUNK_ROWS), n, False)
    per_row = _head_floats(n, bn)
    step = max(256, min(CHUNK_ROWS, CHUNK_FLOATS // max(1, per_row)) // 256 * 256)
    ws = torch.empty(per_row * min(r, step), dtype=torch.float32, device=dev)
    status = core.workspace(dev).status
    for lo in range(0, r, step):
        m = min(step, r - lo)
        rc = _launch(dev, _k().sllm_head_logprobs, x.data_ptr() + 2 * lo * x.stride(0), w.data_ptr(), tokens.data_ptr() + 4 * lo, m, n, x.shape[1],
                     x.stride(0) if r > 1 else x.shape[1], softcap, bn, ws.data_ptr(), ws.numel(), lp.data_ptr() + 4 * lo,
                     entropy.data_ptr() + 4 * lo, status.data_ptr())
        _lib.check(rc, "head_logprobs")
        if _lib.audit_enabled():
            _lib.record_dispatch("linear_logprobs", "head_logprobs_kernel" if bn else "head_few_kernel", m=m, n=n, k=x.shape[1], bn=bn)
    return TokenLogprobs(lp, entropy)


def linear_logprobs(x, w, tokens: torch.Tensor, softcap: float = 0.0, top: int = 0) -> TokenLogprobs:
    """`token_logprobs` of the logits x W^T (``softcap`` > 0: softcap * tanh(logit / softcap)) for one token per row, in memory that
    does not grow with rows * vocabulary.  ``x``: hidden rows [R, d] of any strides, of the weight's type (bf16 or fp32) for a dense
    ``w``, bf16 or a `QTensor` for FP8, bf16 for 4 bits; ``tokens`` [R].  Logits of dense weights are not rounded on the way (those of
    FP8 and 4-bit weights are bf16).  All but bf16 heads without alternatives go through `ops.linear`, whose workspace serves one
    stream at a time."""
    _check_operands(x, w)
    xd = x.data if isinstance(x, core.QTensor) else x
    if softcap != 0.0 and not MIN_CAP <= softcap <= MAX_CAP:
        raise ValueError(f"the soft cap lies between {MIN_CAP} and {MAX_CAP}, or is 0 for none")
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top lies between 0 and {MAX_TOP}")
    _check_tokens(tokens, xd.shape[0], xd.device)
    if tokens.dim() != 1:
        raise ValueError("one token per row")
    if (not top and w.kind == "dense" and not _lib.on_cpu(xd) and xd.dtype == w.w.dtype == torch.bfloat16 and w.in_features % 8 == 0
            and w.w.is_contiguous() and w.w.data_ptr() % 16 == 0):
        return _head(xd, w.w, tokens, softcap)
    if xd.is_cuda and xd.device.index != torch.cuda.current_device():      # (the products launch on the current device)
        with torch.cuda.device(xd.device):
            return _through_logits(x, w, tokens, softcap, top)
    return _through_logits(x, w, tokens, softcap, top)


def _through_logits(x, w, tokens: torch.Tensor, softcap: float, top: int) -> TokenLogprobs:
    """Products of some rows at a time, and the log-probabilities of their logits."""
    if isinstance(x, core.QTensor):
        xd = _plain_rows(x.data, False)
        x = core.QTensor(xd, x.scale)
    else:
        xd = x = _plain_rows(x, w.kind == "dense")
    step = chunk_rows(w.out_features)
    parts = []
    for lo in range(0, xd.shape[0], step):
        hi = min(lo + step, xd.shape[0])
        if isinstance(x, core.QTensor):
            rows = core.QTensor(x.data[lo:hi], x.scale[:, lo:hi].contiguous())
        else:
            rows = x[lo:hi]
        if w.kind == "dense":
            z = core.linear(rows, w, act="softcap" if softcap else None, act_arg=softcap, out_fp32=True)
        else:
            z = core.linear(rows, w)
            if softcap:
                z = core.elementwise("tanh_softcap", z, s=softcap)
        parts.append(token_logprobs(z, tokens[lo:hi], top))
        del z                                              # (ahead of the next rows' logits)
    if not parts:
        z = torch.empty((0, w.out_features), dtype=torch.float32, device=xd.device)
        return token_logprobs(z, tokens, top)
    if len(parts) == 1:
        return parts[0]
    return TokenLogprobs(*(None if f[0] is None else torch.cat(f) for f in zip(*parts)))
