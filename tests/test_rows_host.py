"""CPU: refusals of the entry points beside rows of logits, before any launch."""
import ctypes as C

import pytest

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
