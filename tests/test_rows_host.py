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
