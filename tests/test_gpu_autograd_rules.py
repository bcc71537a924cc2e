"""What autograd has to know of the operators: writes in place, targets that require a gradient, forward-mode tangents."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from pasa_b200 import ops
from test_gpu_kv8 import Pages, i32, randn
from test_gpu_lora import Problem

pytestmark = pytest.mark.gpu


def changed_after_it_was_saved(t, change):
    """Whether autograd notices that ``change`` writes t, which an operation before it has saved."""
    w = torch.ones_like(t, requires_grad=True)
    product = (w * t).sum()
    with torch.no_grad():
        change(t)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()


def test_writes_in_place_are_noticed(cuda_device):
    p = Problem([100], 64, 64, 8, 1)
    changed_after_it_was_saved(p.y, lambda t: ops.lora_update(t, *p.args, out=t))
    changed_after_it_was_saved(torch.zeros_like(p.y), lambda t: ops.lora_update(p.y, *p.args, out=t))
    changed_after_it_was_saved(torch.zeros_like(p.x), lambda t: ops.lora_update_backward(p.dy, *p.args, dx=t))
    rope = dict(axes=(8, 8), grid=(4, 5), inplace=True)
    changed_after_it_was_saved(randn(1, 2, 20, 32), lambda t: ops.rope_axes(t, **rope))
    changed_after_it_was_saved(randn(1, 2, 20, 32), lambda t: ops.rope_axes(randn(1, 2, 20, 32), t, **rope))
    c = Pages([100], 2, 64).fill()
    changed_after_it_was_saved(randn(1, 2, 7, 64), lambda t: ops.kv8_attention(t, c.cache, c.table, i32([100]), out=t))
    before = [t._version for t in c.cache]
    ops.kv8_write(c.cache, randn(1, 2, 3, 64), randn(1, 2, 3, 64), c.table, i32([97]))
    assert all(t._version > v for t, v in zip(c.cache, before))
    with torch.inference_mode():  # tensors without a counter
        q = randn(1, 2, 20, 32)
        assert ops.rope_axes(q, **rope) is q


def test_targets_that_require_a_gradient(cuda_device):
    p = Problem([100], 64, 64, 8, 1)
    c = Pages([100], 2, 64).fill()
    q = randn(1, 2, 7, 64)
    for call, like in ((lambda t: ops.lora_update(p.y, *p.args, out=t), p.y),
                       (lambda t: ops.lora_update_backward(p.dy, *p.args, dx=t), p.x),
                       (lambda t: ops.kv8_attention(q, c.cache, c.table, i32([100]), out=t), q)):
        with pytest.raises(ValueError, match="require"):
            call(torch.zeros_like(like, requires_grad=True))
        leaf = torch.zeros_like(like, requires_grad=True)
        with pytest.raises(ValueError, match="require"):
            call(leaf * 1)
        with torch.no_grad():
            call(leaf)


def test_forward_mode_is_refused(cuda_device):
    p = Problem([100], 64, 64, 8, 1)
    c = Pages([100], 2, 64).fill()
    q = randn(1, 2, 20, 64)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: ops.rope_axes(dual(q), axes=(8, 8), grid=(4, 5)),
                     lambda: ops.rope_axes(q, dual(q.clone()), axes=(8, 8), grid=(4, 5)),
                     lambda: ops.rope_axes(dual(q), axes=(8, 8), grid=(4, 5), inplace=True),
                     lambda: ops.lora_update(dual(p.y), *p.args), lambda: ops.lora_update(p.y, dual(p.x), *p.args[1:]),
                     lambda: ops.lora_update(p.y, p.x, dual(p.a), *p.args[2:]),
                     lambda: ops.lora_update(p.y, *p.args[:5], dual(p.scale)),
                     lambda: ops.lora_update_backward(dual(p.dy), *p.args),
                     lambda: ops.kv8_attention(dual(q), c.cache, c.table, i32([100])),
                     lambda: ops.kv8_write(c.cache, dual(q[:, :, :3]), q[:, :, :3], c.table, i32([97]))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward"):
                    call()
        ops.rope_axes(q, axes=(8, 8), grid=(4, 5))
        ops.lora_update(p.y, *p.args)
        ops.kv8_attention(q, c.cache, c.table, i32([100]))


def test_a_scale_that_requires_a_gradient(cuda_device):
    """It has none; without gradients it is a scale like any other."""
    p = Problem([100], 64, 64, 8, 1)
    want = ops.lora_update(p.y, *p.args)
    p.scale.requires_grad_()
    with pytest.raises(ValueError, match="scale"):
        ops.lora_update(p.y, *p.args)
    with torch.no_grad():
        assert torch.equal(ops.lora_update(p.y, *p.args), want)
