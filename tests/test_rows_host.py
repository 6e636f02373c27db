"""CPU: refusals of the entry points beside rows of logits, before any launch."""
import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as fad

import flowrl_hip as fh
from flowrl_hip import _lib


def _critic():
    d = _lib.FrlCriticDesc()
    d.abi_version, d.particles, d.n_states, d.obs_dim, d.act_dim, d.n_hidden, d.act, d.ensemble = _lib.FRL_ABI_VERSION, 8, 4, 5, 2, 2, _lib.FRL_ACT["mish"], 2
    d.hidden[0] = d.hidden[1] = 256
    return d


@pytest.mark.parametrize("allowed,mask,stride", [(None, _lib.FRL_MASK_BYTES, 8), (None, _lib.FRL_MASK_WORDS, 1), (1 << 20, _lib.FRL_MASK_NONE, 8),
                                                 (1 << 20, 3, 8), (1 << 20, -1, 8), (1 << 20, _lib.FRL_MASK_BYTES, -1)])
def test_masked_selection_refuses(lib, allowed, mask, stride):
    d, p, b = _critic(), _lib.FrlCriticParams(), _lib.FrlSelectBufs()
    need = lib.frl_critic_workspace_bytes(C.byref(d))
    assert need > 0
    assert lib.frl_critic_select_masked(C.byref(d), C.byref(p), C.byref(b), allowed, mask, stride, 4096, need, None) == _lib.FRL_EINVAL
    assert b"mask" in lib.frl_last_error()
    # and what the entry point without a mask refuses
    assert lib.frl_critic_select_masked(C.byref(d), C.byref(p), C.byref(b), None, _lib.FRL_MASK_NONE, 0, None, 0, None) == _lib.FRL_EWORKSPACE


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("where", ["logits", "rule", "out", "temperature", "teacher", "weights", "leaf"])
def test_forward_mode_tangents_are_refused(where, grad):
    """A dual operand needs no requires_grad, and no_grad leaves its tangent alone: it must not be dropped in silence."""
    z, ids, t, w = torch.zeros((2, 8)), torch.zeros((2, 1), dtype=torch.int32), torch.zeros((2, 1)), torch.ones(2)
    with fad.dual_level(), torch.set_grad_enabled(grad):
        dual = lambda x: fad.make_dual(x, torch.ones_like(x))  # noqa: E731
        calls = {
            "logits": [lambda: fh.logits.constrain(dual(z)), lambda: fh.logits.choose(dual(z)), lambda: fh.logits.distill_loss(dual(z), ids, t),
                       lambda: fh.autograd.distill_loss(dual(z), ids, t)],
            "rule": [lambda: fh.logits.constrain(z, fh.logits.Constraints(bias=dual(z[0]))), lambda: fh.logits.choose(z, fh.logits.Constraints(presence=dual(w)))],
            "out": [lambda: fh.logits.constrain(z, out=dual(z.clone()))],
            "temperature": [lambda: fh.logits.choose(z, temperature=dual(w))],
            "teacher": [lambda: fh.logits.distill_loss(z, ids, dual(t)), lambda: fh.autograd.distill_loss(z, ids, dual(t))],
            "weights": [lambda: fh.logits.distill_loss(z, ids, t, weights=dual(w)), lambda: fh.autograd.distill_loss(z, ids, t, weights=dual(w))],
            "leaf": [lambda: fh.autograd.distill_loss(dual(z.clone().requires_grad_(True)), ids, t)],
        }[where]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="GPU only"):
            fh.logits.choose(z)


V = 1000


def _rows(**kw):
    d = _lib.FrlLogitsDesc()
    d.abi_version, d.dtype, d.out_dtype, d.vocab, d.rows, d.repetition = _lib.FRL_ABI_VERSION, _lib.FRL_ELT_BF16, _lib.FRL_ELT_BF16, V, 7, 1.0
    d.logits_stride = d.out_stride = 2 * V
    for k, v in kw.items():
        setattr(d, k, v)
    return d


# entries from the first logit to the first result; two bytes each
@pytest.mark.parametrize("off,kw", [(V - 1, {}), (1, {}), (V + 1, {}), (2 * V - 1, {}), (-1, {}), (-(V - 1), {}), (-(V + 1), {}), (2 * V, {}), (-2 * V, {}), (12 * V, {}),
                                    (13 * V - 1, {}), (-12 * V, {}), (-(13 * V - 1), {}), (V, dict(out_stride=2 * V + 1)), (V, dict(out_dtype=_lib.FRL_ELT_F32, out_stride=V)),
                                    (V, dict(out_dtype=_lib.FRL_ELT_F32, out_stride=2 * V)), (V - 1, dict(rows=1)), (0, dict(out_stride=2 * V + 2))])
def test_results_that_share_entries_with_logits_are_refused(lib, off, kw):
    d, b = _rows(**kw), _lib.FrlLogitsBufs()
    b.logits, b.out = 1 << 30, (1 << 30) + 2 * off
    assert lib.frl_logits_constrain(C.byref(d), C.byref(b), None) == _lib.FRL_EINVAL
    assert b"overlaps" in lib.frl_last_error()
    if not kw:
        d = _lib.FrlDistillDesc()
        d.abi_version, d.dtype, d.vocab, d.top, d.rows, d.temperature = _lib.FRL_ABI_VERSION, _lib.FRL_ELT_BF16, V, 4, 7, 1.0
        d.logits_stride = d.grad_stride = 2 * V
        b = _lib.FrlDistillBufs()
        b.logits, b.ids, b.teacher, b.loss, b.grad, b.row_stats, b.g_loss = 1 << 30, 1 << 12, 1 << 13, 1 << 14, (1 << 30) + 2 * off, 1 << 16, 1 << 15
        for rc in (lib.frl_distill_fwd(C.byref(d), C.byref(b), 4096, 1 << 30, None), lib.frl_distill_bwd(C.byref(d), C.byref(b), None)):
            assert rc == _lib.FRL_EINVAL and b"overlaps" in lib.frl_last_error()


@pytest.mark.parametrize("repetition", [1e-39, 1e-45, 0.0, -1.0, float("nan")])
def test_repetition_without_a_reciprocal_is_refused(lib, repetition):
    """1 / 1e-39 is no float32 number: every quotient would be infinite."""
    d, b = _rows(history_len=3, repetition=repetition), _lib.FrlLogitsBufs()
    b.logits, b.out, b.history, b.token = 1 << 30, 1 << 40, 1 << 13, 1 << 12
    assert lib.frl_logits_constrain(C.byref(d), C.byref(b), None) == _lib.FRL_EINVAL and b"repetition" in lib.frl_last_error()
    assert lib.frl_logits_choose(C.byref(d), C.byref(b), 4096, 1 << 20, None) == _lib.FRL_EINVAL and b"repetition" in lib.frl_last_error()
