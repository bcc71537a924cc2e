"""rope_axes on the GPU against a plain rotation in fp64."""
import math

import pytest
import torch

from pasa_b200 import ops

pytestmark = pytest.mark.gpu


def plain(x, positions, axes, theta=10000.0, pairs="interleaved", inverse=False):
    """positions [B or 1, T, axes] -> the exact rotation, fp64."""
    theta = list(theta) if isinstance(theta, (list, tuple)) else [theta] * len(axes)
    angle = torch.cat([positions[..., i, None].double() * torch.tensor(
        [t ** (-2 * j / d) for j in range(d // 2)], dtype=torch.float64, device=x.device)
        for i, (d, t) in enumerate(zip(axes, theta))], dim=-1)[:, None]
    if inverse:
        angle = -angle
    n = sum(axes)
    out = x.double().clone()
    u, v = (x[..., :n // 2], x[..., n // 2:n]) if pairs == "halves" else (x[..., 0:n:2], x[..., 1:n:2])
    u, v = u.double(), v.double()
    a, b = u * angle.cos() - v * angle.sin(), u * angle.sin() + v * angle.cos()
    if pairs == "halves":
        out[..., :n // 2], out[..., n // 2:n] = a, b
    else:
        out[..., 0:n:2], out[..., 1:n:2] = a, b
    return out


def grid_positions(grid, origin, device):
    r = [torch.arange(o, o + n, device=device) for n, o in zip(grid, origin)]
    return torch.stack(torch.meshgrid(*r, indexing="ij"), -1).flatten(0, -2)[None]


def check(got, x, exact, axes, pairs="interleaved"):
    """Bound: |u|, |v| <= r for each pair's length r.  Sine and cosine are off by at most 4 steps of 2^-24 (2 ulp of
    sincospif, the rest of the angle, one rounding), the two products and their sum by 3 more, together 2 * 7 * 2^-24
    of r; the store by half a step of the result's own type, eps / 2 of its value."""
    n = sum(axes)
    u, v = (x[..., :n // 2], x[..., n // 2:n]) if pairs == "halves" else (x[..., 0:n:2], x[..., 1:n:2])
    r = (u.double() ** 2 + v.double() ** 2).sqrt()
    r = torch.cat((r, r), -1) if pairs == "halves" else r.repeat_interleave(2, -1)
    half_step = 0.0 if x.dtype == torch.float32 else torch.finfo(x.dtype).eps / 2
    bound = 14 * 2.0 ** -24 * r * (1 + half_step) + half_step * exact[..., :n].abs() + 1e-38
    assert ((got[..., :n].double() - exact[..., :n]).abs() <= bound).all()
    assert torch.equal(got[..., n:], x[..., n:])


def randn(*shape, dtype=torch.bfloat16, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return torch.randn(shape, generator=g, device=device, dtype=torch.float32).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("dim,axes", [(128, (44, 42, 42)), (128, (16, 56, 56)), (64, (16, 8, 8)), (80, (16, 24, 24)),
                                      (96, (0, 32, 32)), (6, (2,)), (10, (2, 4, 2, 2)), (256, (256,)), (34, (6, 10))])
def test_grid_and_positions(cuda_device, dtype, pairs, inverse, dim, axes):
    grid, origin = [(3, 5, 2, 2)[i] for i in range(len(axes))], [(7, 0, 100, 3)[i] for i in range(len(axes))]
    tokens = math.prod(grid)
    q, k = randn(2, 5, tokens, dim, dtype=dtype), randn(2, 3, tokens, dim, dtype=dtype, seed=1)
    where = grid_positions(grid, origin, q.device)
    a = ops.rope_axes(q, k, axes=axes, grid=grid, origin=origin, pairs=pairs, inverse=inverse)
    b = ops.rope_axes(q, k, axes=axes, positions=where[0].int(), pairs=pairs, inverse=inverse)
    for x, got, same in zip((q, k), a, b):
        check(got, x, plain(x, where, axes, pairs=pairs, inverse=inverse), axes, pairs)
        assert torch.equal(got, same)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32, torch.float64])
def test_position_types_far_and_negative(cuda_device, dtype):
    where = torch.tensor([[[0, 1, 1 << 20], [-5, 77777, 3]], [[1 << 24, -1, 2], [9, 8, -(1 << 22)]]], device="cuda")
    if dtype.is_floating_point:
        where = where.to(dtype) + 0.5
    else:
        where = where.to(dtype)
    x = randn(2, 3, 2, 64, dtype=torch.float32)
    check(ops.rope_axes(x, axes=(16, 24, 24), positions=where), x, plain(x, where, (16, 24, 24)), (16, 24, 24))


@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 40), (255, 7), (1560, 24), (4097, 33)])
def test_lengths_and_heads(cuda_device, tokens, heads):
    x = randn(1, heads, tokens, 128)
    where = grid_positions((tokens, 1), (0, 0), x.device)
    check(ops.rope_axes(x, axes=(64, 64), grid=(tokens, 1)), x, plain(x, where, (64, 64)), (64, 64))


def test_theta_of_each_axis(cuda_device):
    x = randn(1, 2, 12, 32, dtype=torch.float32)
    where = grid_positions((3, 4), (0, 0), x.device)
    check(ops.rope_axes(x, axes=(16, 16), grid=(3, 4), theta=(100.0, 5e5)), x,
          plain(x, where, (16, 16), (100.0, 5e5)), (16, 16))


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
@pytest.mark.parametrize("inplace", [False, True])
def test_views(cuda_device, pairs, inplace):
    """Token-major storage, a text tail left as it is, rows that are not 16-byte aligned, a batch slice."""
    where = grid_positions((4, 5), (0, 0), "cuda")
    views = []
    base = randn(2, 27, 6, 64)
    views.append(base.transpose(1, 2)[:, :, :20])
    odd = randn(2, 6, 20, 67)
    views.append(odd[..., 3:])
    qkv = randn(2, 20, 3, 6, 64)
    views.append(qkv[:, :, 1].transpose(1, 2))
    views.append(randn(6, 4, 20, 64).transpose(0, 1)[::2])
    for x in views:
        before = x.clone()
        got = ops.rope_axes(x, axes=(32, 32), grid=(4, 5), pairs=pairs, inplace=inplace)
        check(got, before, plain(before, where, (32, 32), pairs=pairs), (32, 32), pairs)
        assert (got.data_ptr() == x.data_ptr()) == inplace
        assert inplace or torch.equal(x, before)
    if inplace:  # what the views leave out is untouched
        assert torch.equal(base[:, 20:], randn(2, 27, 6, 64)[:, 20:])
        assert torch.equal(odd[..., :3], randn(2, 6, 20, 67)[..., :3])
        assert torch.equal(qkv[:, :, ::2], randn(2, 20, 3, 6, 64)[:, :, ::2])


def test_broadcast_and_permuted_inputs(cuda_device):
    where = grid_positions((4, 5), (0, 0), "cuda")
    for x in (randn(1, 1, 20, 32).expand(3, 4, -1, -1), randn(1, 4, 32, 20).transpose(2, 3)):
        check(ops.rope_axes(x, axes=(32, 0), grid=(4, 5)), x, plain(x, where, (32, 0)), (32, 0))


def test_nothing_and_empty(cuda_device):
    assert ops.rope_axes(randn(1, 2, 0, 16), axes=(8, 8), grid=(0, 4)).shape == (1, 2, 0, 16)
    q, k = ops.rope_axes(randn(1, 2, 4, 16), randn(1, 0, 4, 16), axes=(8, 8), grid=(1, 4))
    assert q.shape[1] == 2 and k.shape[1] == 0


def test_values_behind_the_pairs_do_not_mix(cuda_device):
    x = randn(1, 2, 4, 16, dtype=torch.float32)
    x[..., 6:] = float("nan")
    got = ops.rope_axes(x, axes=(6,), grid=(4,))
    assert torch.isfinite(got[..., :6]).all() and torch.isnan(got[..., 6:]).all()


def test_offsets_past_32_bits(cuda_device):
    """The last head of a view whose elements reach past 2^31."""
    big = torch.zeros(34, 1 << 26, dtype=torch.bfloat16, device="cuda")  # 4.6 GB
    x = big.view(34, 1 << 19, 128)[None, :, -16:]
    x.copy_(randn(1, 34, 16, 128))
    before = x.clone()
    where = grid_positions((16,), (5,), "cuda")
    check(ops.rope_axes(x, axes=(128,), grid=(16,), origin=(5,), inplace=True), before, plain(before, where, (128,)),
          (128,))


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
def test_gradient(cuda_device, pairs):
    """Against the transpose of the plain rotation, and against differences in a random direction."""
    q, k = (randn(2, h, 20, 24, dtype=torch.float32, seed=h).requires_grad_() for h in (4, 2))
    where = grid_positions((4, 5), (0, 0), "cuda")
    args = dict(axes=(8, 12), grid=(4, 5), pairs=pairs)
    a, b = ops.rope_axes(q, k, **args)
    da, db = randn(*a.shape, dtype=torch.float32, seed=7), randn(*b.shape, dtype=torch.float32, seed=8)
    gq, gk = torch.autograd.grad((a, b), (q, k), (da, db))
    for g, d in ((gq, da), (gk, db)):
        check(g, d, plain(d, where, (8, 12), pairs=pairs, inverse=True), (8, 12), pairs)
    with torch.no_grad():
        step = randn(*q.shape, dtype=torch.float32, seed=9)
        slope = ((plain(q + step, where, (8, 12), pairs=pairs) - plain(q - step, where, (8, 12), pairs=pairs)) / 2
                 * da).sum()
        # a sum of n products of unit size, each off by about 14 * 2^-24
        assert abs(slope - (gq.double() * step).sum()) <= 14 * 2.0 ** -24 * (da.abs() * step.abs()).sum() * 2
    # only one of the two outputs used; an expanded gradient; the gradient of a broadcast input
    assert torch.equal(torch.autograd.grad(ops.rope_axes(q, k, **args)[0], q, da)[0], gq)
    ones = torch.autograd.grad(ops.rope_axes(q, **args).sum(), q)[0]
    check(ones, torch.ones_like(q), plain(torch.ones_like(q), where, (8, 12), pairs=pairs, inverse=True), (8, 12), pairs)
    shared = randn(2, 1, 20, 24, dtype=torch.float32).requires_grad_()
    g = torch.autograd.grad(ops.rope_axes(shared.expand(-1, 4, -1, -1), **args), shared, da)[0]
    assert torch.allclose(g, gq.sum(1, keepdim=True), rtol=0, atol=1e-5)


def test_positions_changed_before_the_gradient_are_noticed(cuda_device):
    x, where = randn(1, 1, 4, 8).requires_grad_(), torch.zeros(4, 1, device="cuda")
    y = ops.rope_axes(x, axes=(8,), positions=where)
    where += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals(cuda_device):
    x = randn(1, 2, 4, 16)
    good = dict(axes=(8, 8), grid=(2, 2))
    for bad in (dict(axes=(8, 9), grid=(2, 2)), dict(axes=(8, 10), grid=(2, 2)), dict(axes=(8, 8)),
                dict(axes=(8, 8), grid=(2, 3)), dict(axes=(8, 8), grid=(4,)), dict(good, origin=(1,)),
                dict(good, positions=torch.zeros(4, 2, device="cuda")), dict(good, pairs="both"),
                dict(good, theta=-1.0), dict(good, theta=(1.0, 2.0, 3.0)), dict(axes=(), grid=()),
                dict(axes=(8, 8), positions=torch.zeros(4, 3, device="cuda")),
                dict(axes=(8, 8), positions=torch.zeros(4, 2)),
                dict(axes=(8, 8), positions=torch.zeros(4, 2, device="cuda", dtype=torch.int16))):
        with pytest.raises(ValueError):
            ops.rope_axes(x, **bad)
    with pytest.raises(ValueError, match="bfloat16"):
        ops.rope_axes(x.half(), **good)
    with pytest.raises(ValueError):
        ops.rope_axes(x[0], **good)
    for k in (x.float(), x.cpu(), randn(1, 2, 3, 16), randn(2, 2, 4, 16), randn(1, 2, 4, 8)):
        with pytest.raises(ValueError):
            ops.rope_axes(x, k, **good)
    for t in (randn(1, 1, 4, 16).expand(1, 2, 4, 16), randn(1, 2, 16, 4).transpose(2, 3)):
        with pytest.raises(ValueError):
            ops.rope_axes(t, inplace=True, **good)
    with pytest.raises(ValueError):
        ops.rope_axes(x, x, inplace=True, **good)
    with pytest.raises(ValueError):
        ops.rope_axes(x.float().requires_grad_(), inplace=True, **good)


def test_stream_and_graph(cuda_device):
    """On another stream than the tensors' own, and captured and replayed on new values; autograd is refused there."""
    x, where = randn(1, 3, 24, 32), grid_positions((4, 6), (0, 0), "cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.rope_axes(x, axes=(16, 16), grid=(4, 6))
    torch.cuda.current_stream().wait_stream(side)
    check(y, x, plain(x, where, (16, 16)), (16, 16))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.rope_axes(x, axes=(16, 16), positions=where[0])
        with pytest.raises(RuntimeError, match="no_grad"):
            ops.rope_axes(x.detach().requires_grad_(), axes=(16, 16), grid=(4, 6))
    x.copy_(randn(1, 3, 24, 32, seed=5))
    graph.replay()
    check(y, x, plain(x, where, (16, 16)), (16, 16))
