"""Answers out of a vocabulary of discrete choices, and learning them from a teacher: rows of logits under rules.

The reference's discrete answers stop at the critic's best-of-N — argmax, or ``jax.random.categorical`` as argmax of logits plus
Gumbel noise, over a handful of unconstrained candidates (flowrl/agent/offline/dql.py:151-161, :func:`flowrl_hip.critic_select`).
This module makes the same choice among any number of entries (candidate actions, action tokens, a text vocabulary), with
penalties for repeats, biases and a mask of what is allowed, and gives the loss that trains a student on a teacher's best entries.

    rules = Constraints(history=tokens, lengths=n, repetition=1.2, allowed=grammar_words)
    z = constrain(logits, rules)                                                    # the constrained logits
    token, logprob = choose(logits, rules, temperature=0.8, gumbel=noise)           # one entry per row, nothing written in between
    loss, grad = distill_loss(student, ids, teacher, temperature=2.0, want_grad=True)

``include/flowrl_hip.h`` (frl_logits_constrain, frl_logits_choose, frl_distill_fwd / _bwd) states the arithmetic.  No arithmetic
lives here; the kernels are csrc/logits.hip and csrc/distill.hip, there is no CPU path.  Logits are float32, bfloat16 or float16 with
any leading dimensions (below: "rows"); a row is contiguous, its start and the distance between rows are free.  Every call only
enqueues work on the current stream of the logits' device, so it can be captured into a graph.  :func:`flowrl_hip.autograd.distill_loss` is
the differentiable form of the loss.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch

from . import _lib

PerRow = Union[float, torch.Tensor]
_ELT = {torch.float32: _lib.FRL_ELT_F32, torch.bfloat16: _lib.FRL_ELT_BF16, torch.float16: _lib.FRL_ELT_F16}
_KIND = {"logits": _lib.FRL_DISTILL_TOP, "logprobs": _lib.FRL_DISTILL_REST}
_REDUCTION = {"none": _lib.FRL_REDUCE_NONE, "sum": _lib.FRL_REDUCE_SUM, "mean": _lib.FRL_REDUCE_MEAN}


@dataclass(eq=False)
class Constraints:
    """The rules of a batch of rows; every field may be left out.

    history         (rows, L) int32 / int64 tokens so far.  ``lengths`` (rows,) int32: how many of a row's entries are filled (default
                    all); ``prompt_lengths`` (rows,) int32: how many of those are the prompt (default none).  Tokens outside the
                    vocabulary are padding.
    repetition      > 0: a token seen anywhere in the history has its positive logit divided, its negative one multiplied by it
    frequency       subtracted once per time the token was generated (stands behind the prompt)
    presence        subtracted once if it was generated at all
                    (each of the three a number, or a float32 tensor (rows,); without a history they do nothing)
    bias            float32 (vocab,) or (rows, vocab), added
    bias_tokens, bias_values   (K,) or (rows, K) tokens and their float32 biases, K <= 2048; a token listed twice gets the sum
    allowed         bool (vocab,) or (rows, vocab), or int32 words (ceil(vocab / 32),) or (rows, ceil(vocab / 32)) with bit ``v % 32`` of word
                    ``v // 32`` set where v is allowed; everything else becomes -inf, NaN included
    """
    history: Optional[torch.Tensor] = None
    lengths: Optional[torch.Tensor] = None
    prompt_lengths: Optional[torch.Tensor] = None
    repetition: PerRow = 1.0
    frequency: PerRow = 0.0
    presence: PerRow = 0.0
    bias: Optional[torch.Tensor] = None
    bias_tokens: Optional[torch.Tensor] = None
    bias_values: Optional[torch.Tensor] = None
    allowed: Optional[torch.Tensor] = None


_NO_RULES = Constraints()


def _check_logits(logits: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int]:
    """(rows x vocab view with contiguous rows, rows, vocab)"""
    if not logits.is_cuda:
        raise RuntimeError("flowrl_hip runs on the GPU only; there is no CPU fallback")
    if logits.dtype not in _ELT:
        raise TypeError(f"{what}: float32, bfloat16 or float16 required (got {logits.dtype})")
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"{what}: (..., vocab) with at least one entry expected, got {tuple(logits.shape)}")
    V = logits.shape[-1]
    z = logits if logits.dim() == 2 else logits.reshape(-1, V) if logits.numel() else logits.reshape(math.prod(logits.shape[:-1]), V)
    R = z.shape[0]
    if (V > 1 and z.stride(1) != 1) or (R > 1 and z.stride(0) < V):
        z = z.contiguous()
    return z, R, V


def _on(t: torch.Tensor, dev: torch.device, what: str) -> torch.Tensor:
    if t.device != dev:
        raise ValueError(f"{what}: on {t.device}, expected {dev}")
    return t


def _row_values(t: torch.Tensor, R: int, dev: torch.device, dtype: torch.dtype, what: str) -> torch.Tensor:
    """A tensor of one value per row."""
    if t.dtype != dtype or t.numel() != R:
        raise TypeError(f"{what}: {R} values of {dtype} expected (got {tuple(t.shape)} of {t.dtype})")
    _on(t, dev, what)
    return t if t.dim() == 1 and (R <= 1 or t.stride(0) == 1) else t.reshape(R).contiguous()


def _rows_of(t: torch.Tensor, R: int, n: int, dev: torch.device, what: str, shared: bool) -> Tuple[torch.Tensor, int]:
    """(tensor, row stride) of an (n,) or (rows, n) operand; stride 0 where one row serves all."""
    _on(t, dev, what)
    if shared and t.dim() == 1 and t.shape[0] == n:
        return (t if n <= 1 or t.stride(0) == 1 else t.contiguous()), 0
    if t.dim() < 1 or t.shape[-1] != n or t.numel() != R * n:
        raise ValueError(f"{what}: ({'' if not shared else f'{n},) or ('}{R}, {n}) expected, got {tuple(t.shape)}")
    t = t if t.dim() == 2 else t.reshape(R, n)
    if n > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _ids(t: torch.Tensor, what: str) -> torch.Tensor:
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{what}: int32 or int64 tokens required (got {t.dtype})")
    return t


def _no_grad(what: str, *ts) -> None:
    if torch.is_grad_enabled() and any(torch.is_tensor(t) and t.requires_grad for t in ts):
        raise NotImplementedError(f"flowrl_hip.logits: {what} is not differentiated here; detach it")


def _marshal(z: torch.Tensor, R: int, V: int, c: Constraints):
    """FrlLogitsDesc / FrlLogitsBufs of one call, and the tensors that they point into."""
    dev = z.device
    d, b, keep = _lib.FrlLogitsDesc(), _lib.FrlLogitsBufs(), [z]
    d.abi_version, d.dtype, d.vocab, d.rows, d.logits_stride = _lib.FRL_ABI_VERSION, _ELT[z.dtype], V, R, z.stride(0)
    b.logits = z.data_ptr()
    history, tokens = c.history, c.bias_tokens
    if history is not None and tokens is not None and history.dtype != tokens.dtype:
        history, tokens = _ids(history, "history").long(), _ids(tokens, "bias_tokens").long()
    if history is not None:
        L = _ids(history, "history").shape[-1] if history.dim() else 0
        history, d.history_stride = _rows_of(history, R, L, dev, "history", shared=False)
        keep.append(history)
        d.history_len, d.ids64, b.history = L, int(history.dtype == torch.int64), history.data_ptr()
        for name in ("lengths", "prompt_lengths"):
            t = getattr(c, name)
            if t is not None:
                t = _row_values(t, R, dev, torch.int32, name)
                keep.append(t)
                setattr(b, name, t.data_ptr())
        for name in ("repetition", "frequency", "presence"):
            v = getattr(c, name)
            if torch.is_tensor(v):
                v = _row_values(v, R, dev, torch.float32, name)
                keep.append(v)
                setattr(b, name, v.data_ptr())
            else:
                setattr(d, name, float(v))
    elif c.lengths is not None or c.prompt_lengths is not None:
        raise ValueError("lengths / prompt_lengths without a history")
    if c.bias is not None:
        if c.bias.dtype != torch.float32:
            raise TypeError(f"bias: float32 required (got {c.bias.dtype})")
        t, d.bias_stride = _rows_of(c.bias, R, V, dev, "bias", shared=True)
        keep.append(t)
        b.bias = t.data_ptr()
    if (tokens is None) != (c.bias_values is None):
        raise ValueError("bias_tokens and bias_values come together")
    if tokens is not None:
        if c.bias_values.dtype != torch.float32 or c.bias_values.shape != tokens.shape:
            raise TypeError(f"bias_values: float32 of bias_tokens' shape {tuple(tokens.shape)} required (got {tuple(c.bias_values.shape)} of {c.bias_values.dtype})")
        K = _ids(tokens, "bias_tokens").shape[-1] if tokens.dim() else 0
        t, d.sparse_stride = _rows_of(tokens, R, K, dev, "bias_tokens", shared=True)
        u, stride = _rows_of(c.bias_values, R, K, dev, "bias_values", shared=True)
        if stride != d.sparse_stride:
            t, u = t.contiguous(), u.contiguous()
            d.sparse_stride = 0 if t.dim() == 1 else K
        keep += [t, u]
        d.n_sparse, d.ids64, b.bias_tokens, b.bias_values = K, int(t.dtype == torch.int64), t.data_ptr(), u.data_ptr()
    if c.allowed is not None:
        if c.allowed.dtype == torch.bool:
            d.mask, n = _lib.FRL_MASK_BYTES, V
        elif c.allowed.dtype == torch.int32:
            d.mask, n = _lib.FRL_MASK_WORDS, (V + 31) // 32
        else:
            raise TypeError(f"allowed: bool entries or int32 words of 32 entries required (got {c.allowed.dtype})")
        t, d.mask_stride = _rows_of(c.allowed, R, n, dev, "allowed", shared=True)
        keep.append(t)
        b.allowed = t.data_ptr()
    return d, b, keep


def _call(fn, dev: torch.device, *args) -> None:
    """The entry point on dev's current stream, with dev as the current device while it is called."""
    stream = torch.cuda.current_stream(dev).cuda_stream
    if torch.cuda.current_device() == dev.index:
        _lib.check(fn(*args, stream))
    else:
        with torch.cuda.device(dev):
            _lib.check(fn(*args, stream))


def constrain(logits: torch.Tensor, rules: Optional[Constraints] = None, *, out: Optional[torch.Tensor] = None,
              out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The logits with ``rules`` applied, in the logits' type or float32 (``out_dtype``), rounded once.  ``out``: where they go, a
    tensor of the logits' shape with contiguous rows; it may be ``logits`` itself."""
    rules = _NO_RULES if rules is None else rules
    _no_grad("logits / bias", logits, rules.bias, rules.bias_values)
    z, R, V = _check_logits(logits, "logits")
    if out is None:
        dtype = logits.dtype if out_dtype is None else out_dtype
        out = torch.empty(logits.shape, dtype=dtype, device=logits.device)
        o = out.view(R, V)
    else:
        if out_dtype is not None and out.dtype != out_dtype:
            raise TypeError(f"out is {out.dtype}, out_dtype {out_dtype}")
        if out.shape != logits.shape:
            raise ValueError(f"out: {tuple(logits.shape)} expected, got {tuple(out.shape)}")
        _on(out, logits.device, "out")
        if out.dim() > 2 and not out.is_contiguous():
            raise ValueError("out: contiguous, or two-dimensional with contiguous rows")
        o = out if out.dim() == 2 else out.view(R, V)
        if (V > 1 and o.stride(1) != 1) or (R > 1 and o.stride(0) < V):
            raise ValueError("out: contiguous rows that do not overlap expected")
    if out.dtype != logits.dtype and out.dtype != torch.float32:
        raise TypeError(f"constrain: {logits.dtype} logits go to {logits.dtype} or float32, not {out.dtype}")
    d, b, keep = _marshal(z, R, V, rules)
    d.out_dtype, d.out_stride, b.out = _ELT[out.dtype], o.stride(0), o.data_ptr()
    _call(_lib.load().frl_logits_constrain, z.device, C.byref(d), C.byref(b))
    del keep
    return out


def choose(logits: torch.Tensor, rules: Optional[Constraints] = None, *, temperature: PerRow = 0.0,
           gumbel: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One entry per row of the constrained logits and its log-probability: (token int32, logprob float32) of the logits'
    leading shape.  Rows with ``temperature`` (a number, or float32 (rows,)) <= 0 take the argmax; the others draw
    argmax(y + gumbel) with y = logits / (1e-6 + temperature) and ``gumbel`` (rows, vocab) float32 Gumbel(0, 1) noise, finite
    (:func:`flowrl_hip.random.gumbel`); without noise every row is greedy, and a number > 0 for the temperature is refused.  The
    first of equal maxima; NaN counts as the largest.  logprob is log softmax of y (of the constrained logits for a greedy row).  A row
    that the rules leave nothing answers token -1 with logprob -inf."""
    rules = _NO_RULES if rules is None else rules
    _no_grad("logits / bias", logits, rules.bias, rules.bias_values)
    z, R, V = _check_logits(logits, "logits")
    dev = z.device
    d, b, keep = _marshal(z, R, V, rules)
    if torch.is_tensor(temperature):
        t = _row_values(temperature, R, dev, torch.float32, "temperature")
        keep.append(t)
        b.temperature = t.data_ptr()
    else:
        d.temperature = float(temperature)
    if gumbel is not None:
        if gumbel.dtype != torch.float32:
            raise TypeError(f"gumbel: float32 required (got {gumbel.dtype})")
        g, stride = _rows_of(gumbel, R, V, dev, "gumbel", shared=False)
        if R > 1 and stride < V:
            g = g.contiguous()
            stride = V
        keep.append(g)
        d.gumbel_stride, b.gumbel = stride, g.data_ptr()
    lead = logits.shape[:-1]
    token = torch.empty(lead, dtype=torch.int32, device=dev)
    logprob = torch.empty(lead, dtype=torch.float32, device=dev)
    b.token, b.logprob = token.data_ptr(), logprob.data_ptr()
    lib = _lib.load()
    # a tensor of this call's own: calls on two streams, and graphs captured from them, share no scratch
    need = lib.frl_logits_workspace_bytes(C.byref(d))
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(lib.frl_logits_choose, dev, C.byref(d), C.byref(b), ws.data_ptr() if need else None, need)
    del keep
    return token, logprob


def _distill_marshal(logits: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, kind: str, temperature: float,
                     weights: Optional[torch.Tensor], reduction: str):
    if kind not in _KIND:
        raise ValueError(f"kind {kind!r}: 'logits' or 'logprobs'")
    if reduction not in _REDUCTION:
        raise ValueError(f"reduction {reduction!r}: 'mean', 'sum' or 'none'")
    z, R, V = _check_logits(logits, "logits")
    dev = z.device
    if teacher.dtype not in _ELT:
        raise TypeError(f"teacher: float32, bfloat16 or float16 required (got {teacher.dtype})")
    K = _ids(ids, "ids").shape[-1] if ids.dim() else 0
    if K < 1:
        raise ValueError(f"ids: (rows, top) with at least one entry expected, got {tuple(ids.shape)}")
    d, b = _lib.FrlDistillDesc(), _lib.FrlDistillBufs()
    i, d.ids_stride = _rows_of(ids, R, K, dev, "ids", shared=False)
    t, d.teacher_stride = _rows_of(teacher, R, K, dev, "teacher", shared=False)
    d.abi_version, d.dtype, d.teacher_dtype, d.ids64 = _lib.FRL_ABI_VERSION, _ELT[z.dtype], _ELT[t.dtype], int(i.dtype == torch.int64)
    d.kind, d.reduction, d.vocab, d.top, d.rows = _KIND[kind], _REDUCTION[reduction], V, K, R
    d.logits_stride, d.temperature = z.stride(0), float(temperature)
    b.logits, b.ids, b.teacher = z.data_ptr(), i.data_ptr(), t.data_ptr()
    keep = [z, i, t]
    if weights is not None:
        w = _row_values(weights, R, dev, torch.float32, "weights")
        keep.append(w)
        b.weights = w.data_ptr()
    return d, b, keep


def distill_forward(logits, ids, teacher, kind, temperature, weights, reduction, want_grad=False, want_stats=False):
    """(loss, grad or None, row statistics or None): frl_distill_fwd."""
    d, b, keep = _distill_marshal(logits, ids, teacher, kind, temperature, weights, reduction)
    dev, R, V = logits.device, d.rows, d.vocab
    loss = torch.empty(logits.shape[:-1] if reduction == "none" else (), dtype=torch.float32, device=dev)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=dev) if want_grad else None
    stats = torch.empty((R + 1, _lib.FRL_DISTILL_STATS), dtype=torch.float32, device=dev) if want_stats else None
    b.loss = loss.data_ptr()
    if R == 0 and reduction == "none":
        return loss, grad, stats
    if want_grad:
        b.grad, d.grad_stride = grad.data_ptr() or None, V
    if want_stats:
        b.row_stats = stats.data_ptr()
    lib = _lib.load()
    need = lib.frl_distill_workspace_bytes(C.byref(d))
    ws = torch.empty(max(need, 256), dtype=torch.uint8, device=dev)
    _call(lib.frl_distill_fwd, dev, C.byref(d), C.byref(b), ws.data_ptr(), ws.numel())
    del keep
    return loss, grad, stats


def distill_backward(logits, ids, teacher, kind, temperature, weights, reduction, stats, g_loss):
    """d loss / d logits times ``g_loss`` from the forward's row statistics: frl_distill_bwd."""
    d, b, keep = _distill_marshal(logits, ids, teacher, kind, temperature, weights, reduction)
    grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    g = _row_values(g_loss, d.rows if reduction == "none" else 1, logits.device, torch.float32, "g_loss")
    b.row_stats, b.g_loss, b.grad, d.grad_stride = stats.data_ptr(), g.data_ptr(), grad.data_ptr(), d.vocab
    _call(_lib.load().frl_distill_bwd, logits.device, C.byref(d), C.byref(b))
    del keep
    return grad


def distill_loss(logits: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, *, kind: str = "logits", temperature: float = 1.0,
                 weights: Optional[torch.Tensor] = None, reduction: str = "mean", want_grad: bool = False):
    """KL divergence of softmax(logits / temperature) from a teacher that names its ``top`` best entries of each row.

    ``ids`` (rows, top) int32 / int64 (entries outside the vocabulary are padding), ``teacher`` (rows, top), top <= 1024:
      kind "logits"    the teacher's logits; p = softmax(teacher / temperature) over the named entries
      kind "logprobs"  its log-probabilities (at the temperature meant); what they leave of 1 is one more class, "the rest", which
                       the student fills with all entries that are not named
    ``weights`` (rows,) float32: a row of weight 0 is not read.  ``reduction`` "mean" divides by the sum of the weights; "none" returns
    the rows' weighted divergences.  With ``want_grad`` also d loss / d logits in the logits' type, in the same pass ("none": of
    the rows' sum).  Like ``mse_loss`` a value without a graph; :func:`flowrl_hip.autograd.distill_loss` differentiates."""
    _no_grad("logits (use flowrl_hip.autograd.distill_loss) / teacher / weights", logits, teacher, weights)
    loss, grad, _ = distill_forward(logits, ids, teacher, kind, temperature, weights, reduction, want_grad)
    return (loss, grad) if want_grad else loss
