"""Lengths of texts that are not theirs."""
import pytest
import torch

from pasa_b200 import dit, ops
from test_gpu_dit_requests import CFG, _dense, _setup
from test_gpu_kv8 import i32

pytestmark = pytest.mark.gpu


def test_lengths_above_the_text_are_cut(cuda_device):
    """A text of 70 tokens has 128 places in its pages; 90 and more tokens are its 70, below zero none."""
    x, txt, blocks, emb, rope, _ = _setup(cuda_device)
    t = torch.tensor([700, 300, 50], device=cuda_device)
    steps = []
    for lengths in ([70, 70, 0], [90, 1 << 30, -5]):
        kv = dit.text_cache(txt, emb, blocks, CFG, lengths=i32(lengths))
        assert kv.lengths.tolist() == [70, 70, 0]
        steps.append(dit.step(x, t, None, rope, emb, blocks, CFG, _dense, fused=True, text_kv=kv))
    ops.check_operator_errors()
    assert torch.equal(*steps)
