"""lora_update and its gradients on the GPU against the formulas in fp64."""
import pytest
import torch

from pasa_b200 import ops

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8    # half a step of bf16, relative to the value
ADD = 2.0 ** -23    # one fp32 addition of a tensor core, which may truncate
SPLIT = 2.0 ** -18  # two bf16 terms: half a step of the second, relative to the first's half step


class Problem:
    def __init__(self, lengths, k, n, rank, adapters, slots=None, lead=0, tail=0, seed=0, scale=True):
        g = torch.Generator(device="cuda").manual_seed(seed)
        randn = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
        self.m, self.k, self.n, self.rank = lead + sum(lengths) + tail, k, n, rank
        starts = [lead]
        for length in lengths:
            starts.append(starts[-1] + length)
        self.starts, self.slot_list = starts, slots or [i % adapters for i in range(len(lengths))]
        self.rows = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.slots = torch.tensor(self.slot_list, dtype=torch.int32, device="cuda")
        self.x, self.y, self.dy = randn(self.m, k), randn(self.m, n), randn(self.m, n)
        self.a, self.b = randn(adapters, rank, k) * k ** -0.5, randn(adapters, n, rank) * 0.25
        self.scale = 0.5 + torch.rand(adapters, generator=g, device="cuda") if scale else None

    @property
    def args(self):
        return self.x, self.a, self.b, self.rows, self.slots, self.scale

    def requests(self):
        for first, last, slot in zip(self.starts, self.starts[1:], self.slot_list):
            if last > first and 0 <= slot < len(self.a):
                s = 1.0 if self.scale is None else self.scale[slot].double()
                yield slice(first, last), slot, s, self.a[slot].double(), self.b[slot].double()

    def check_out(self, out):
        want, bound = self.y.double(), torch.zeros_like(self.y, dtype=torch.float64)
        same = torch.ones(self.m, dtype=torch.bool, device="cuda")
        for r, _, s, a, b in self.requests():
            same[r] = False
            x = self.x[r].double()
            h = s * (x @ a.T)
            h_off = (self.k + 1) * ADD * s * (x.abs() @ a.abs().T) + SPLIT * h.abs()
            want[r] += h @ b.T
            bound[r] = h_off @ b.abs().T + (2 * self.rank + 2) * ADD * (self.y[r].double().abs() + h.abs() @ b.abs().T)
        check(out, want, bound, ~same)
        assert torch.equal(out.view(torch.int16)[same], self.y.view(torch.int16)[same])

    def check_grads(self, dx, da, db, base=None):
        want = torch.zeros_like(self.x, dtype=torch.float64) if base is None else base.double()
        bound = torch.zeros_like(want)
        wa, wb = torch.zeros_like(self.a, dtype=torch.float64), torch.zeros_like(self.b, dtype=torch.float64)
        ba, bb = torch.zeros_like(wa), torch.zeros_like(wb)
        for r, slot, s, a, b in self.requests():
            x, dy = self.x[r].double(), self.dy[r].double()
            h, g = s * (x @ a.T), s * (dy @ b)
            h_off = (self.k + 1) * ADD * s * (x.abs() @ a.abs().T) + SPLIT * h.abs()
            g_off = (self.n + 1) * ADD * s * (dy.abs() @ b.abs()) + SPLIT * g.abs()
            bound[r] = g_off @ a.abs() + (2 * self.rank + 2) * ADD * (want[r].abs() + g.abs() @ a.abs())
            want[r] += g @ a
            count = 2 * (self.m + 64 * len(self.starts))  # terms of a sum, zeros of partial stages among them
            wa[slot] += g.T @ x
            wb[slot] += dy.T @ h
            ba[slot] += g_off.T @ x.abs() + count * ADD * (g.abs().T @ x.abs())
            bb[slot] += dy.abs().T @ h_off + count * ADD * (dy.abs().T @ h.abs())
        check(dx, want, bound)
        check(da, wa, ba)
        check(db, wb, bb)


def check(got, want, bound, rows=slice(None)):
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    off = (got.double() - want).abs()[rows]
    most = (bound + HALF * (want.abs() + bound))[rows]
    assert (off <= most).all(), (off / most.clamp_min(1e-300)).max().item()


CASES = {
    "one row": dict(lengths=[1], k=8, n=8, rank=8, adapters=1),
    "least sizes": dict(lengths=[3], k=16, n=24, rank=16, adapters=1),
    "ragged": dict(lengths=[0, 5, 128, 1, 0, 127, 130, 64, 33], k=200, n=136, rank=24, adapters=4),
    "lead and tail": dict(lengths=[100, 40], k=328, n=264, rank=40, adapters=2, lead=17, tail=150),
    "no adapter": dict(lengths=[40, 40, 40, 40], k=64, n=72, rank=8, adapters=2, slots=[1, -1, 2, 0], tail=3),
    "all without": dict(lengths=[40, 90], k=64, n=72, rank=8, adapters=2, slots=[-1, 7]),
    "one adapter, many requests": dict(lengths=[7] * 70, k=512, n=128, rank=72, adapters=2, slots=[1] * 70),
    "single rows": dict(lengths=[1] * 40, k=1536, n=512, rank=64, adapters=16),
    "widest rank": dict(lengths=[300, 211], k=1000, n=776, rank=128, adapters=2),
    "rank 56": dict(lengths=[129], k=648, n=520, rank=56, adapters=1, scale=False),
    "long k, few rows": dict(lengths=[9, 2], k=13824, n=64, rank=32, adapters=2),
    "long n, few rows": dict(lengths=[9, 2], k=64, n=13824, rank=112, adapters=2),
    "many rows": dict(lengths=[20001, 13, 9000], k=136, n=320, rank=16, adapters=3),
    "uneven adapters": dict(lengths=[3000, 1, 64, 9000, 31, 700, 2, 33], k=520, n=1048, rank=64, adapters=9,
                            slots=[7, 0, 3, 7, 5, 2, 3, 8]),
    "more adapters than rows": dict(lengths=[1, 2, 1], k=72, n=64, rank=8, adapters=300, slots=[299, 0, 150]),
    "requests and nothing in them": dict(lengths=[0, 0], k=64, n=64, rank=8, adapters=1, tail=5),
}


@pytest.mark.parametrize("name", CASES)
def test_update(cuda_device, name):
    p = Problem(**CASES[name])
    out = ops.lora_update(p.y, *p.args)
    p.check_out(out)
    y = p.y.clone()
    assert ops.lora_update(y, *p.args, out=y) is y
    assert torch.equal(y, out)
    ops.check_operator_errors()


@pytest.mark.parametrize("name", CASES)
def test_backward(cuda_device, name):
    p = Problem(**CASES[name])
    _, h = ops.lora_update(p.y, *p.args, return_h=True)
    grads = ops.lora_update_backward(p.dy, *p.args, h=h)
    p.check_grads(*grads)
    again = ops.lora_update_backward(p.dy, *p.args)  # h computed again
    assert all(torch.equal(u, v) for u, v in zip(grads, again))
    base = torch.randn_like(p.x)
    dx = base.clone()
    got = ops.lora_update_backward(p.dy, *p.args, h=h, dx=dx)
    assert got[0] is dx
    p.check_grads(*got, base=base)
    ops.check_operator_errors()


def test_other_rows_do_not_leak(cuda_device):
    """NaN in rows of no request and of requests without an adapter, and an infinity in one request: the others'
    results and gradients are what they were."""
    p = Problem(lengths=[70, 50, 90], k=264, n=136, rank=24, adapters=2, slots=[0, -1, 1], lead=9, tail=30)
    clean = ops.lora_update(p.y, *p.args), *ops.lora_update_backward(p.dy, *p.args)
    for t in (p.x, p.dy):
        t[:9] = t[79:129] = t[-30:] = float("nan")
    bad = ops.lora_update(p.y, *p.args), *ops.lora_update_backward(p.dy, *p.args)
    assert all(torch.equal(u, v) for u, v in zip(clean, bad))
    p.x[130, 5] = float("inf")
    out, (dx, da, db) = ops.lora_update(p.y, *p.args), ops.lora_update_backward(p.dy, *p.args)
    mine = torch.arange(p.m, device="cuda") != 130
    assert torch.equal(out[mine], clean[0][mine]) and not torch.isfinite(out[130]).any()
    assert torch.equal(dx, clean[1]) and torch.equal(da[0], clean[2][0]) and torch.equal(db[0], clean[3][0])
    assert torch.equal(da[1][:, 6:], clean[2][1][:, 6:]) and not torch.isfinite(da[1][:, 5]).any()


def test_views_and_leading_dimensions(cuda_device):
    p = Problem(lengths=[60, 36], k=64, n=72, rank=16, adapters=2)
    want = ops.lora_update(p.y, *p.args)
    grads = ops.lora_update_backward(p.dy, *p.args)
    wide = torch.zeros(p.m, 200, dtype=torch.bfloat16, device="cuda")
    x, y = wide[:, 8:72], wide[:, 104:176]
    x.copy_(p.x), y.copy_(p.y)
    assert torch.equal(ops.lora_update(y, x, *p.args[1:]), want)
    odd = torch.zeros(p.m, 67, dtype=torch.bfloat16, device="cuda")[:, 3:]
    odd.copy_(p.x)
    assert torch.equal(ops.lora_update(p.y, odd, *p.args[1:]), want)               # copied
    turned = p.x.T.contiguous().T
    assert torch.equal(ops.lora_update(p.y, turned, *p.args[1:]), want)
    spread = p.x[:1].expand(p.m, -1)
    assert torch.equal(ops.lora_update(p.y, spread, *p.args[1:]),
                       ops.lora_update(p.y, spread.contiguous(), *p.args[1:]))
    ops.lora_update(y, x, *p.args[1:], out=y)
    assert torch.equal(y, want) and not wide[:, 72:104].any() and not wide[:, 176:].any()
    deep = ops.lora_update(p.y.view(3, 8, 4, 72), p.x.view(3, 8, 4, 64), *p.args[1:])
    assert deep.shape == (3, 8, 4, 72) and torch.equal(deep.view(96, 72), want)
    dx, da, db = ops.lora_update_backward(p.dy.view(2, 48, 72), p.x.view(2, 48, 64), *p.args[1:])
    assert torch.equal(dx.view(96, 64), grads[0]) and torch.equal(da, grads[1]) and torch.equal(db, grads[2])
    assert torch.equal(ops.lora_update(p.y, p.x, p.a.transpose(1, 2).contiguous().transpose(1, 2), *p.args[2:]), want)


def test_nothing(cuda_device):
    p = Problem(lengths=[0], k=16, n=8, rank=8, adapters=2)
    assert ops.lora_update(p.y, *p.args).shape == (0, 8)
    dx, da, db = ops.lora_update_backward(p.dy, *p.args)
    assert dx.shape == (0, 16) and not da.any() and not db.any()
    p = Problem(lengths=[], k=16, n=8, rank=8, adapters=2, lead=5)  # rows but no requests
    assert torch.equal(ops.lora_update(p.y, *p.args), p.y)
    dx, da, db = ops.lora_update_backward(p.dy, *p.args)
    assert not dx.any() and not da.any() and not db.any()


def test_offsets_past_the_rows_are_cut(cuda_device):
    """Offsets below zero and behind the last row: as if cut there."""
    p = Problem(lengths=[50, 50], k=64, n=64, rank=8, adapters=2)
    want = ops.lora_update(p.y, *p.args), *ops.lora_update_backward(p.dy, *p.args)
    p.rows.copy_(torch.tensor([-7, 50, 1 << 30]))
    got = ops.lora_update(p.y, *p.args), *ops.lora_update_backward(p.dy, *p.args)
    assert all(torch.equal(u, v) for u, v in zip(want, got))


def test_repeated_calls_agree(cuda_device):
    p = Problem(lengths=[3000, 500], k=520, n=264, rank=40, adapters=1, slots=[0, 0])
    first = ops.lora_update(p.y, *p.args), *ops.lora_update_backward(p.dy, *p.args)
    for _ in range(3):
        got = ops.lora_update(p.y, *p.args), *ops.lora_update_backward(p.dy, *p.args)
        assert all(torch.equal(u, v) for u, v in zip(first, got))


@pytest.mark.parametrize("n,rank", [(128, 16), (136, 72), (1024, 8), (5120, 16)])
def test_spans_with_and_without_adapters_in_turn(cuda_device, n, rank):
    """Blocks that go from a span with an adapter to one without and back, over and over: the same every time."""
    lengths = [700, 90, 33, 1000, 5, 260, 128, 640, 300, 1500] * 4
    p = Problem(lengths, k=64, n=n, rank=rank, adapters=3, slots=[(0, -1, 1, -1, -1, 2, 0)[i % 7] for i in range(40)],
                tail=400)
    first = ops.lora_update(p.y, *p.args)
    p.check_out(first)
    outs = [ops.lora_update(p.y, *p.args) for _ in range(40)]
    assert all(torch.equal(first, out) for out in outs)
    grads = [ops.lora_update_backward(p.dy, *p.args) for _ in range(10)]
    p.check_grads(*grads[0])
    assert all(torch.equal(u, v) for g in grads for u, v in zip(grads[0], g))
    ops.check_operator_errors()


def test_autograd(cuda_device):
    """The same gradients as the explicit call, through a projection, and the formula's against differences."""
    p = Problem(lengths=[40, 24], k=64, n=72, rank=8, adapters=2)
    dx, da, db = ops.lora_update_backward(p.dy, *p.args)
    y, x, a, b = (t.clone().requires_grad_() for t in (p.y, p.x, p.a, p.b))
    out = ops.lora_update(y, x, a, b, p.rows, p.slots, p.scale)
    got = torch.autograd.grad(out, (y, x, a, b), p.dy, retain_graph=True)
    assert all(torch.equal(u, v) for u, v in zip(got, (p.dy, dx, da, db)))
    assert torch.equal(torch.autograd.grad(out, a, p.dy)[0], da)
    w = torch.randn(72, 64, device="cuda").to(torch.bfloat16)
    out = ops.lora_update(torch.nn.functional.linear(x, w), x, a, b, p.rows, p.slots, p.scale)
    total = torch.autograd.grad(out, x, p.dy)[0]
    assert torch.equal(total, (p.dy @ w) + dx)  # one bf16 addition of the two
    ones = torch.autograd.grad(ops.lora_update(y, x, a, b, p.rows, p.slots).sum(), x)[0]  # an expanded gradient
    want = ops.lora_update_backward(torch.ones_like(p.y), p.x, p.a, p.b, p.rows, p.slots)[0]
    assert torch.equal(ones, want)

    def loss(x, a, b):
        out = p.y.double()
        for r, slot, s, _, _ in p.requests():
            out[r] = out[r] + s * (x[r] @ a[slot].T) @ b[slot].T
        return (out * p.dy.double()).sum()
    args = [t.double() for t in (p.x, p.a, p.b)]
    for i, g in enumerate((dx, da, db)):
        step = torch.randn_like(args[i]) * 1e-3
        up = loss(*[t + step if j == i else t for j, t in enumerate(args)])
        down = loss(*[t - step if j == i else t for j, t in enumerate(args)])
        slope = (up - down) / 2  # exact: the loss is linear in each of the three
        assert abs(slope - (g.double() * step).sum()) <= 1.1 * HALF * (g.double().abs() * step.abs()).sum()


def test_refusals(cuda_device):
    p = Problem(lengths=[10, 6], k=64, n=72, rank=8, adapters=2)
    x, a, b, rows, slots, scale = p.args
    bad = [
        (p.y, x.float(), a, b, rows, slots), (p.y.float(), x, a, b, rows, slots), (p.y, x, a.float(), b, rows, slots),
        (p.y[:15], x, a, b, rows, slots), (p.y[:, :64], x, a, b, rows, slots), (p.y, x, a[:1], b, rows, slots),
        (p.y, x, a[:, :, :32], b, rows, slots), (p.y, x, a[:, :4], b[:, :, :4], rows, slots),
        (p.y, x, a, b, rows[:2], slots), (p.y, x, a, b, rows.long(), slots), (p.y, x, a, b, rows, slots.long()),
        (p.y, x, a, b, rows.cpu(), slots), (p.y, x, a, b, rows, slots, scale[:1]), (p.y, x, a[0], b, rows, slots),
        (p.y, x, a, b, rows, slots, scale.half()), (p.y, x, a[:0], b[:0], rows, slots), (p.y[0], x[0], a, b, rows, slots),
        (p.y[:, :68], x, a, b[:, :68], rows, slots),
    ]
    for args in bad:
        with pytest.raises(ValueError):
            ops.lora_update(*args)
    wide = torch.zeros(16, 76, dtype=torch.bfloat16, device="cuda")
    for out in (p.y[:15], p.y.float(), wide[:, 4:], wide[:, :72], torch.zeros(72, 16, device="cuda").bfloat16().T,
                p.y.cpu()):
        with pytest.raises(ValueError):
            ops.lora_update(p.y, *p.args, out=out)
    square = Problem(lengths=[16], k=64, n=64, rank=8, adapters=1)
    with pytest.raises(ValueError, match="out is x"):
        ops.lora_update(square.y, *square.args, out=square.x)
    for dx in (square.x, square.dy):
        with pytest.raises(ValueError, match="dx is"):
            ops.lora_update_backward(square.dy, *square.args, dx=dx)
    with pytest.raises(ValueError, match="scale"):
        ops.lora_update(p.y, x, a, b, rows, slots, scale.clone().requires_grad_())
    with pytest.raises(ValueError, match="out"):
        ops.lora_update(p.y, x, a.clone().requires_grad_(), b, rows, slots, out=torch.empty_like(p.y))
    for h in (torch.zeros(2, 16, 8, dtype=torch.bfloat16, device="cuda"), torch.zeros(2, 16, 16, device="cuda")):
        with pytest.raises(ValueError):
            ops.lora_update_backward(p.dy, *p.args, h=h)
    with pytest.raises(ValueError):
        ops.lora_update_backward(p.dy[:, :64], *p.args)


def test_stream_and_graph(cuda_device):
    """On a stream of its own; captured, and replayed with other values, lengths and slots; two graphs in turn."""
    p = Problem(lengths=[130, 70], k=264, n=136, rank=24, adapters=2)
    q = Problem(lengths=[50, 150], k=264, n=136, rank=24, adapters=2, slots=[1, 1], seed=5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.lora_update(p.y, *p.args)
    torch.cuda.current_stream().wait_stream(side)
    p.check_out(out)
    eager = [t.clone().requires_grad_() for t in (p.x, p.a, p.b)]
    alive = ops.lora_update(p.y, *eager, p.rows, p.slots, p.scale)  # an eager graph of the same inputs stays alive
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, h = ops.lora_update(p.y, *p.args, return_h=True)
            results = out, *ops.lora_update_backward(p.dy, *p.args, h=h)
            with pytest.raises(RuntimeError, match="no_grad"):
                ops.lora_update(p.y, *eager, p.rows, p.slots, p.scale)
        graphs.append((g, results))
    for problem in (p, q, p):
        for name in ("x", "y", "dy", "a", "b", "scale", "rows", "slots"):
            getattr(p, name).copy_(getattr(problem, name).clone())
        p.starts, p.slot_list = problem.starts, problem.slot_list
        for g, _ in graphs:
            g.replay()
        for _, results in graphs:
            p.check_out(results[0])
            p.check_grads(*results[1:])
    assert torch.isfinite(alive).all()
    ops.check_operator_errors()


@pytest.mark.parametrize("most", [1, 9])
def test_many_requests(cuda_device, most):
    """More requests than a warp or a block looks through at once, single rows and none among them."""
    lengths = [(7 * i) % (most + 1) for i in range(700)]
    p = Problem(lengths, 128, 192, 16, 37, slots=[(11 * i) % 39 - 1 for i in range(700)], lead=3, tail=5)
    p.check_out(ops.lora_update(p.y, *p.args))
    p.check_grads(*ops.lora_update_backward(p.dy, *p.args))
