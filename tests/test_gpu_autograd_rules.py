"""What autograd has to know of the operators: writes in place, targets that require a gradient, forward-mode tangents."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from pasa_b200 import ops
from test_gpu_kv8 import Pages, i32, randn
from test_gpu_lora import Problem

pytestmark = pytest.mark.gpu


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
