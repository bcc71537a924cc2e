"""The rule for what autograd has to see of a call."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from pasa_b200 import _launch


def test_forward_mode_tangents_are_refused():
    t = torch.ones(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, t)
        assert not _launch.wants_grad("f", t, None)
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward"):
                _launch.wants_grad("f", t, None, dual)
    assert not _launch.wants_grad("f", t)
