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
import struct
from dataclasses import dataclass
from typing import Optional, Tuple, Union

import torch
from torch.autograd import forward_ad as _forward_ad

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
    repetition      > 0 (and no subnormal number): a token seen anywhere in the history has its positive logit divided, its negative one multiplied by it
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
# torch.cuda.current_stream(index).cuda_stream without the Stream object, and torch.cuda.current_device() without its initialisation check (the logits
# are on the device already), where torch has the shorter ways
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)

# A decoding step's call is as short as its host side.  The C structs are therefore filled with one pack each (their ctypes layout,
# checked here once) and every operand takes one cheap test on the way to its pointer; only an operand that fails it is looked at closely.
_DESC, _BUFS = struct.Struct("@4iq4i7q4f"), struct.Struct("@16Q")
_DDESC, _DBUFS = struct.Struct("@8i5qf4x"), struct.Struct("@8Q")
for _s, _t in ((_DESC, _lib.FrlLogitsDesc), (_BUFS, _lib.FrlLogitsBufs), (_DDESC, _lib.FrlDistillDesc), (_DBUFS, _lib.FrlDistillBufs)):
    assert _s.size == C.sizeof(_t), _t


def _check_logits(logits: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int, int]:
    """(logits with contiguous rows that do not overlap, rows, vocab, row stride)"""
    if not logits.is_cuda:
        raise RuntimeError("flowrl_hip runs on the GPU only; there is no CPU fallback")
    if logits.dtype not in _ELT:
        raise TypeError(f"{what}: float32, bfloat16 or float16 required (got {logits.dtype})")
    shape = logits.shape
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError(f"{what}: (..., vocab) with at least one entry expected, got {tuple(shape)}")
    V = shape[-1]
    R = shape[0] if len(shape) == 2 else math.prod(shape[:-1])
    if logits.is_contiguous():
        return logits, R, V, V
    z = logits if len(shape) == 2 else logits.reshape(R, V)
    if (V > 1 and z.stride(1) != 1) or (R > 1 and z.stride(0) < V):
        z = z.contiguous()
    return z, R, V, z.stride(0)


def _on(t: torch.Tensor, index: int, what: str) -> None:
    if t.get_device() != index:
        raise ValueError(f"{what}: on {t.device}, expected device {index}")


def _row_values(t: torch.Tensor, R: int, index: int, dtype: torch.dtype, what: str) -> torch.Tensor:
    """A tensor of one value per row, contiguous."""
    if t.dtype is not dtype or t.numel() != R:
        raise TypeError(f"{what}: {R} values of {dtype} expected (got {tuple(t.shape)} of {t.dtype})")
    if t.get_device() != index:
        _on(t, index, what)
    return t if t.is_contiguous() else t.contiguous()


def _rows_of(t: torch.Tensor, R: int, n: int, index: int, what: str, shared: bool) -> Tuple[torch.Tensor, int]:
    """(tensor, row stride) of an (n,) or (rows, n) operand; stride 0 where one row serves all."""
    if t.get_device() != index:
        _on(t, index, what)
    shape = t.shape
    if len(shape) == 2 and shape[1] == n and shape[0] == R:
        if t.is_contiguous():
            return t, n
    elif shared and len(shape) == 1 and shape[0] == n:
        return (t if t.is_contiguous() else t.contiguous()), 0
    elif len(shape) < 1 or shape[-1] != n or t.numel() != R * n:
        raise ValueError(f"{what}: ({'' if not shared else f'{n},) or ('}{R}, {n}) expected, got {tuple(shape)}")
    else:
        t = t.reshape(R, n)
    if n > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t, t.stride(0)


_IDS = {torch.int32: 0, torch.int64: 1}


def _ids(t: torch.Tensor, what: str) -> int:
    """1 for int64 tokens, 0 for int32"""
    wide = _IDS.get(t.dtype)
    if wide is None:
        raise TypeError(f"{what}: int32 or int64 tokens required (got {t.dtype})")
    return wide


def _allowed(t: torch.Tensor, R: int, V: int, index: int) -> Tuple[torch.Tensor, int, int]:
    """(tensor, FRL_MASK_*, row stride) of a mask over V entries"""
    if t.dtype is torch.bool:
        mask, n = _lib.FRL_MASK_BYTES, V
    elif t.dtype is torch.int32:
        mask, n = _lib.FRL_MASK_WORDS, (V + 31) // 32
    else:
        raise TypeError(f"allowed: bool entries or int32 words of 32 entries required (got {t.dtype})")
    t, stride = _rows_of(t, R, n, index, "allowed", True)
    return t, mask, stride


def _no_tangent(what: str, *ts) -> None:
    """Refuse operands that carry a forward-mode tangent (no_grad leaves those alone): it would be dropped."""
    if getattr(_forward_ad, "_current_level", 0) < 0:      # outside of every dual_level
        return
    for t in ts:
        if isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"flowrl_hip.logits: {what} has a forward-mode tangent, which is not carried on; unpack_dual it")


def _no_grad(what: str, *ts) -> None:
    """Refuse operands whose derivative would be lost."""
    _no_tangent(what, *ts)
    if not torch.is_grad_enabled():
        return
    for t in ts:
        if isinstance(t, torch.Tensor) and t.requires_grad:
            raise NotImplementedError(f"flowrl_hip.logits: {what} is not differentiated here; detach it")


def _differentiable(c: Constraints):
    return c.bias, c.bias_values, c.repetition, c.frequency, c.presence


def _marshal(z: torch.Tensor, R: int, V: int, c: Constraints, z_stride: Optional[int] = None, out_elt: int = 0, out_stride: int = 0, out: int = 0,
             temperature: float = 0.0, temperature_ptr: int = 0, gumbel_stride: int = 0, gumbel: int = 0, token: int = 0, logprob: int = 0):
    """FrlLogitsDesc / FrlLogitsBufs of one call, and the copies that they point into."""
    index, keep = z.get_device(), ()
    ids64 = L = K = mask = h_stride = b_stride = s_stride = m_stride = 0
    h_ptr = len_ptr = prompt_ptr = rep_ptr = freq_ptr = pres_ptr = b_ptr = t_ptr = v_ptr = a_ptr = 0
    rep, freq, pres = 1.0, 0.0, 0.0
    history, tokens, values = c.history, c.bias_tokens, c.bias_values
    lengths, prompt = c.lengths, c.prompt_lengths
    if history is not None:
        if tokens is not None and history.dtype is not tokens.dtype:
            _ids(history, "history"), _ids(tokens, "bias_tokens")
            history, tokens = history.long(), tokens.long()
        ids64 = _ids(history, "history")
        L = history.shape[-1] if history.dim() else 0
        history, h_stride = _rows_of(history, R, L, index, "history", False)
        h_ptr = history.data_ptr()
        if lengths is not None:
            lengths = _row_values(lengths, R, index, torch.int32, "lengths")
            len_ptr = lengths.data_ptr()
        if prompt is not None:
            prompt = _row_values(prompt, R, index, torch.int32, "prompt_lengths")
            prompt_ptr = prompt.data_ptr()
        rep, freq, pres = c.repetition, c.frequency, c.presence
        keep = [history, lengths, prompt]
        if isinstance(rep, torch.Tensor):
            t = _row_values(rep, R, index, torch.float32, "repetition")
            rep_ptr, rep = t.data_ptr(), 1.0
            keep.append(t)
        if isinstance(freq, torch.Tensor):
            t = _row_values(freq, R, index, torch.float32, "frequency")
            freq_ptr, freq = t.data_ptr(), 0.0
            keep.append(t)
        if isinstance(pres, torch.Tensor):
            t = _row_values(pres, R, index, torch.float32, "presence")
            pres_ptr, pres = t.data_ptr(), 0.0
            keep.append(t)
    elif lengths is not None or prompt is not None:
        raise ValueError("lengths / prompt_lengths without a history")
    bias = c.bias
    if bias is not None:
        if bias.dtype is not torch.float32:
            raise TypeError(f"bias: float32 required (got {bias.dtype})")
        bias, b_stride = _rows_of(bias, R, V, index, "bias", True)
        b_ptr = bias.data_ptr()
    if tokens is not None:
        if values is None or values.dtype is not torch.float32 or values.shape != tokens.shape:
            got = "none" if values is None else f"{tuple(values.shape)} of {values.dtype}"
            raise (ValueError if values is None else TypeError)(f"bias_values: float32 of bias_tokens' shape {tuple(tokens.shape)} required (got {got})")
        ids64 = _ids(tokens, "bias_tokens")
        K = tokens.shape[-1] if tokens.dim() else 0
        tokens, s_stride = _rows_of(tokens, R, K, index, "bias_tokens", True)
        values, stride = _rows_of(values, R, K, index, "bias_values", True)
        if stride != s_stride:
            tokens, values, s_stride = tokens.contiguous(), values.contiguous(), K
        t_ptr, v_ptr = tokens.data_ptr(), values.data_ptr()
    elif values is not None:
        raise ValueError("bias_values without bias_tokens")
    allowed = c.allowed
    if allowed is not None:
        allowed, mask, m_stride = _allowed(allowed, R, V, index)
        a_ptr = allowed.data_ptr()
    d, b = _lib.FrlLogitsDesc(), _lib.FrlLogitsBufs()
    _DESC.pack_into(d, 0, _lib.FRL_ABI_VERSION, _ELT[z.dtype], out_elt, V, R, ids64, L, K, mask, V if z_stride is None else z_stride, out_stride, gumbel_stride,
                    h_stride, b_stride, s_stride, m_stride, rep, freq, pres, temperature)
    _BUFS.pack_into(b, 0, z.data_ptr(), out, h_ptr, len_ptr, prompt_ptr, rep_ptr, freq_ptr, pres_ptr, b_ptr, t_ptr, v_ptr, a_ptr, temperature_ptr, gumbel, token, logprob)
    return d, b, (keep, bias, tokens, values, allowed)


def _call(fn, index: int, *args) -> None:
    """The entry point on the device's current stream, with the device as the current one while it is called."""
    stream = _current_stream(index)
    if _current_device() == index:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = fn(*args, stream)
    if rc:
        _lib.check(rc)


def constrain(logits: torch.Tensor, rules: Optional[Constraints] = None, *, out: Optional[torch.Tensor] = None,
              out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The logits with ``rules`` applied, in the logits' type or float32 (``out_dtype``), rounded once.  ``out``: where they go, a
    tensor of the logits' shape with contiguous rows; it may be ``logits`` itself."""
    rules = _NO_RULES if rules is None else rules
    _no_grad("logits / a rule / out", logits, out, *_differentiable(rules))
    z, R, V, stride = _check_logits(logits, "logits")
    index = logits.get_device()
    given = out is not None
    if not given:
        dtype = logits.dtype if out_dtype is None else out_dtype
        out = torch.empty_like(logits, dtype=dtype, memory_format=torch.contiguous_format)
        o_stride = V
    else:
        dtype = out.dtype
        if out_dtype is not None and dtype != out_dtype:
            raise TypeError(f"out is {dtype}, out_dtype {out_dtype}")
        if out.shape != logits.shape:
            raise ValueError(f"out: {tuple(logits.shape)} expected, got {tuple(out.shape)}")
        _on(out, index, "out")
        if out.dim() != 2 and not out.is_contiguous():
            raise ValueError("out: contiguous, or two-dimensional with contiguous rows")
        o_stride = V if out.dim() != 2 else out.stride(0)
        if out.dim() == 2 and ((V > 1 and out.stride(1) != 1) or (R > 1 and o_stride < V)):
            raise ValueError("out: contiguous rows that do not overlap expected")
    if dtype != logits.dtype and dtype != torch.float32:
        raise TypeError(f"constrain: {logits.dtype} logits go to {logits.dtype} or float32, not {dtype}")
    d, b, keep = _marshal(z, R, V, rules, stride, _ELT[dtype], o_stride, out.data_ptr())
    _call(_lib.load().frl_logits_constrain, index, C.byref(d), C.byref(b))
    if given and not out.is_inference():
        torch.autograd.graph.increment_version(out)        # written behind torch's back: a graph that saved it has to notice
    return out


def choose(logits: torch.Tensor, rules: Optional[Constraints] = None, *, temperature: PerRow = 0.0,
           gumbel: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One entry per row of the constrained logits and its log-probability: (token int32, logprob float32) of the logits'
    leading shape.  Rows whose ``temperature`` (a number, or float32 (rows,)) is not > 0 take the argmax; the others draw
    argmax(y + gumbel) with y = logits / (1e-6 + temperature) and ``gumbel`` (rows, vocab) float32 Gumbel(0, 1) noise, finite
    (:func:`flowrl_hip.random.gumbel`); without noise every row is greedy, and a number > 0 for the temperature is refused.  The
    first of equal maxima; NaN counts as the largest.  logprob is log softmax of y (of the constrained logits for a greedy row).  A row
    that the rules leave nothing answers token -1 with logprob -inf."""
    rules = _NO_RULES if rules is None else rules
    _no_grad("logits / a rule / the temperature", logits, temperature, *_differentiable(rules))      # nothing that has a derivative depends on the noise
    z, R, V, stride = _check_logits(logits, "logits")
    index = logits.get_device()
    t = g = None
    t_ptr = g_ptr = g_stride = 0
    if isinstance(temperature, torch.Tensor):
        t = _row_values(temperature, R, index, torch.float32, "temperature")
        t_ptr, temperature = t.data_ptr(), 0.0
    if gumbel is not None:
        if gumbel.dtype is not torch.float32:
            raise TypeError(f"gumbel: float32 required (got {gumbel.dtype})")
        g, g_stride = _rows_of(gumbel, R, V, index, "gumbel", False)
        if R > 1 and g_stride < V:
            g, g_stride = g.contiguous(), V
        g_ptr = g.data_ptr()
    lead = logits.shape[:-1]
    token = logits.new_empty(lead, dtype=torch.int32)
    logprob = logits.new_empty(lead, dtype=torch.float32)
    d, b, keep = _marshal(z, R, V, rules, stride, 0, 0, 0, temperature, t_ptr, g_stride, g_ptr, token.data_ptr(), logprob.data_ptr())
    lib = _lib.load()
    # a tensor of this call's own: calls on two streams, and graphs captured from them, share no scratch
    need = lib.frl_logits_workspace_bytes(C.byref(d))
    ws = logits.new_empty(need, dtype=torch.uint8) if need > 256 else None
    _call(lib.frl_logits_choose, index, C.byref(d), C.byref(b), None if ws is None else ws.data_ptr(), need)
    return token, logprob


def _distill_marshal(logits, ids, teacher, kind, temperature, weights, reduction, loss=0, stats=0, g_loss=0, grad=0):
    """FrlDistillDesc / FrlDistillBufs of one call, its rows, and the copies that they point into."""
    z, R, V, stride = _check_logits(logits, "logits")
    index = logits.get_device()
    if teacher.dtype not in _ELT:
        raise TypeError(f"teacher: float32, bfloat16 or float16 required (got {teacher.dtype})")
    ids64 = _ids(ids, "ids")
    K = ids.shape[-1] if ids.dim() else 0
    if K < 1:
        raise ValueError(f"ids: (rows, top) with at least one entry expected, got {tuple(ids.shape)}")
    i, i_stride = _rows_of(ids, R, K, index, "ids", False)
    t, t_stride = _rows_of(teacher, R, K, index, "teacher", False)
    w = None if weights is None else _row_values(weights, R, index, torch.float32, "weights")
    d, b = _lib.FrlDistillDesc(), _lib.FrlDistillBufs()
    _DDESC.pack_into(d, 0, _lib.FRL_ABI_VERSION, _ELT[z.dtype], _ELT[t.dtype], ids64, _KIND[kind], _REDUCTION[reduction], V, K, R, stride, V, i_stride, t_stride, temperature)
    _DBUFS.pack_into(b, 0, z.data_ptr(), i.data_ptr(), t.data_ptr(), 0 if w is None else w.data_ptr(), loss, stats, g_loss, grad)
    return d, b, (z, i, t, w)


def distill_forward(logits, ids, teacher, kind, temperature, weights, reduction, want_grad=False, want_stats=False):
    """(loss, grad or None, row statistics or None): frl_distill_fwd."""
    if kind not in _KIND:
        raise ValueError(f"kind {kind!r}: 'logits' or 'logprobs'")
    if reduction not in _REDUCTION:
        raise ValueError(f"reduction {reduction!r}: 'mean', 'sum' or 'none'")
    if not logits.is_cuda:
        raise RuntimeError("flowrl_hip runs on the GPU only; there is no CPU fallback")
    lead = logits.shape[:-1]
    loss = logits.new_empty(lead if reduction == "none" else (), dtype=torch.float32)
    grad = torch.empty_like(logits, memory_format=torch.contiguous_format) if want_grad else None
    stats = logits.new_empty((math.prod(lead) + 1, _lib.FRL_DISTILL_STATS), dtype=torch.float32) if want_stats else None
    d, b, keep = _distill_marshal(logits, ids, teacher, kind, temperature, weights, reduction, loss.data_ptr(), stats.data_ptr() if want_stats else 0, 0,
                                  grad.data_ptr() if want_grad else 0)
    if reduction == "none" and loss.numel() == 0:
        return loss, grad, stats
    lib = _lib.load()
    need = lib.frl_distill_workspace_bytes(C.byref(d))
    ws = logits.new_empty(need or 256, dtype=torch.uint8)              # need == 0: the entry point says why
    _call(lib.frl_distill_fwd, logits.get_device(), C.byref(d), C.byref(b), ws.data_ptr(), need)
    return loss, grad, stats


def distill_backward(logits, ids, teacher, kind, temperature, weights, reduction, stats, g_loss):
    """d loss / d logits times ``g_loss`` from the forward's row statistics: frl_distill_bwd."""
    grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
    index = logits.get_device()
    g = _row_values(g_loss, math.prod(logits.shape[:-1]) if reduction == "none" else 1, index, torch.float32, "g_loss")
    d, b, keep = _distill_marshal(logits, ids, teacher, kind, temperature, weights, reduction, 0, stats.data_ptr(), g.data_ptr(), grad.data_ptr())
    if grad.numel():
        _call(_lib.load().frl_distill_bwd, index, C.byref(d), C.byref(b))
    return grad


def distill_loss(logits: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, *, kind: str = "logits", temperature: float = 1.0,
                 weights: Optional[torch.Tensor] = None, reduction: str = "mean", want_grad: bool = False):
    """KL divergence of softmax(logits / temperature) from a teacher that names its ``top`` best entries of each row.

    ``ids`` (rows, top) int32 / int64 (entries outside the vocabulary are padding), ``teacher`` (rows, top), top <= 1024:
      kind "logits"    the teacher's logits; p = softmax(teacher / temperature) over the named entries
      kind "logprobs"  its log-probabilities (at the temperature meant); what they leave of 1 is one more class, "the rest", which
                       the student fills with all entries that are not named (a teacher that names the whole vocabulary leaves none:
                       its log-probabilities times the temperature go as "logits")
    ``weights`` (rows,) float32: a row of weight 0 is not read.  ``reduction`` "mean" divides by the sum of the weights; "none" returns
    the rows' weighted divergences.  With ``want_grad`` also d loss / d logits in the logits' type, in the same pass ("none": of
    the rows' sum).  Like ``mse_loss`` a value without a graph; :func:`flowrl_hip.autograd.distill_loss` differentiates."""
    _no_grad("logits (use flowrl_hip.autograd.distill_loss) / teacher / weights", logits, teacher, weights)
    loss, grad, _ = distill_forward(logits, ids, teacher, kind, temperature, weights, reduction, want_grad)
    return (loss, grad) if want_grad else loss
