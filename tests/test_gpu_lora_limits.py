"""The adapters' operators where there are many adapters, infinities, memory that overlaps or row offsets that go back."""
import ctypes

import pytest
import torch

from pasa_b200 import _lib, ops
from test_gpu_lora import Problem

pytestmark = pytest.mark.gpu


def workspace(m, k, n, rank, adapters, requests):
    size = ctypes.c_size_t()
    assert _lib.load().pasa_lora_backward_workspace_size(m, k, n, rank, adapters, requests, ctypes.byref(size)) == _lib.OK
    return size.value


@pytest.mark.parametrize("m,k,n,rank,requests", [(4096, 5120, 5120, 16, 64), (32760, 5120, 5120, 128, 64),
                                                 (8000, 64, 72, 128, 4096)])
def test_workspace_does_not_grow_with_the_adapters(cuda_device, m, k, n, rank, requests):
    """Two sums a share at most, over all its blocks: 3 waves of blocks of 256 columns and more, 128 ranks."""
    most = 2 * m * 128 * 2 + 256 + 2 * 3 * 160 * 512 * 128 * 4
    assert workspace(m, k, n, rank, 4096, requests) <= most


@pytest.mark.parametrize("lengths,adapters,slots", [
    ([64] * 90, 90, None), ([40, 7, 300, 1, 33] * 30, 60, [(7 * i) % 61 - 1 for i in range(150)]),
    ([5000, 3, 3, 3, 6000], 4000, [3999, 1, 2, 1, 0]), ([31, 33] * 200, 400, None)])
def test_gradients_of_many_adapters(cuda_device, lengths, adapters, slots):
    """Shares that begin and end in the middle of an adapter, on its first row, and hold many whole ones."""
    for k, n, rank in ((72, 328, 24), (264, 64, 120)):
        p = Problem(lengths, k, n, rank, adapters, slots)
        grads = ops.lora_update_backward(p.dy, *p.args)
        p.check_grads(*grads)
        assert all(torch.equal(u, v) for u, v in zip(grads, ops.lora_update_backward(p.dy, *p.args)))
    ops.check_operator_errors()


@pytest.mark.parametrize("rows", [3, 100, 300])
@pytest.mark.parametrize("rank", [8, 24, 16])
def test_an_infinity_stays_one(cuda_device, rank, rows):
    """An infinite x or dy of one row with positive weights makes that row's results +infinity, and no other row's."""
    p = Problem([rows], 64, 72, rank, 1)
    p.a.abs_()
    p.b.abs_()
    clean = ops.lora_update(p.y, *p.args)
    grads = ops.lora_update_backward(p.dy, *p.args)
    p.x[2, 5] = float("inf")
    out = ops.lora_update(p.y, *p.args)
    keep = torch.arange(rows, device="cuda") != 2
    assert (out[2] == float("inf")).all() and torch.equal(out[keep], clean[keep])
    p.x[2, 5] = 0.5
    p.dy[2, 5] = float("inf")
    dx, da, db = ops.lora_update_backward(p.dy, *p.args)
    assert (dx[2] == float("inf")).all() and torch.equal(dx[keep], grads[0][keep])
    assert torch.equal(da[0].double(), float("inf") * p.x[2].double().sign().expand(rank, -1))
    assert not db[0, 5].isfinite().any() and db[0, 6:].isfinite().all()


def test_gradients_of_a_alone_without_h(cuda_device):
    """The C entry needs h for the gradients of B only."""
    p = Problem([200, 30], 72, 64, 16, 2)
    dx, da, _ = ops.lora_update_backward(p.dy, *p.args)
    size = workspace(p.m, p.k, p.n, p.rank, 2, 2)
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    got, db = torch.empty_like(p.a), torch.empty_like(p.b)
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731

    def call(h, dx, da, db):
        return _lib.load().pasa_lora_update_backward(
            torch.cuda.current_stream().cuda_stream, ptr(p.dy), p.n, ptr(p.x), p.k, ptr(p.a), ptr(p.b), ptr(p.scale), p.m,
            p.k, p.n, p.rank, 2, ptr(p.rows), ptr(p.slots), 2, ptr(h), 0, None, 0, ptr(dx), p.k, ptr(da), ptr(db),
            space.data_ptr(), size)

    assert call(None, None, got, None) == _lib.OK
    assert torch.equal(got, da)
    other = torch.empty_like(p.x)
    assert call(None, other, None, None) == _lib.OK
    assert torch.equal(other, dx)
    assert call(None, None, None, db) == _lib.ERR_NULL


def test_targets_that_overlap_what_is_read(cuda_device):
    p = Problem([100], 64, 64, 8, 1)
    want = ops.lora_update(p.y, *p.args)
    wide = torch.zeros(101, 200, device="cuda", dtype=torch.bfloat16)
    x, rest = wide[:100, :64], p.args[1:]
    x.copy_(p.x)
    for out in (wide[:100, 32:96], wide[1:, :64], wide[:100, 56:120], wide[:100, 192:193].expand(-1, 64)):
        with pytest.raises(ValueError):
            ops.lora_update(p.y, x, *rest, out=out)
        with pytest.raises(ValueError):
            ops.lora_update_backward(p.dy, x, *rest, dx=out)
    assert torch.equal(ops.lora_update(p.y, x, *rest, out=wide[:100, 64:128]), want)  # beside x in the same rows
    assert torch.equal(x, p.x)
    tall = torch.zeros(205, 64, device="cuda", dtype=torch.bfloat16)
    y = tall[:100]
    y.copy_(p.y)
    for out in (tall[1:101], tall[99:199]):
        with pytest.raises(ValueError):
            ops.lora_update(y, *p.args, out=out)
        with pytest.raises(ValueError):
            ops.lora_update_backward(y, *p.args, dx=out)
    assert torch.equal(ops.lora_update(y, *p.args, out=tall[100:200]), want)
    assert torch.equal(ops.lora_update(y, *p.args, out=y), want)
    one = Problem([1], 64, 64, 8, 1)
    line = torch.zeros(64 + 32, device="cuda", dtype=torch.bfloat16)
    line[:64] = one.x[0]
    with pytest.raises(ValueError):
        ops.lora_update(one.y, line[None, :64], *one.args[1:], out=line[None, 32:])


def test_row_offsets_that_go_back_end(cuda_device):
    """Offsets must not decrease.  Where they do, the calls end all the same, here with 2^31 stages to sum by the
    requests' sizes, and what lies behind the tensors stays as it is."""
    m, half = 1 << 20, 1 << 16
    rows = torch.tensor([0, m] * half + [0], dtype=torch.int32, device="cuda")
    slots = torch.arange(2 * half, dtype=torch.int32, device="cuda") // 2 % 2
    x, dy = (torch.zeros(m, 8, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    a, b = torch.zeros(2, 8, 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 8, 8, dtype=torch.bfloat16, device="cuda")
    h = torch.zeros(2, m, 16, dtype=torch.bfloat16, device="cuda")
    dx, da, db = ops.lora_update_backward(dy, x, a, b, rows, slots, h=h)
    torch.cuda.synchronize()
    assert dx.shape == x.shape and da.shape == a.shape and db.shape == b.shape
    p = Problem([100, 200], 64, 64, 8, 2)
    p.check_grads(*ops.lora_update_backward(p.dy, *p.args))
