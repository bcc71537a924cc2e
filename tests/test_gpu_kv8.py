"""kv8_write and kv8_attention on the GPU: the pages bit for bit, the attention against the formula in fp64."""
import math

import pytest
import torch

from pasa_b200 import ops

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def randn(*shape, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def page_scale(amax: float) -> float:
    if not math.isfinite(amax):
        return float("nan")
    if amax == 0:
        return 2.0 ** -100
    fraction, exponent = math.frexp(amax)
    return 2.0 ** max(exponent - 9 + (fraction > 0.875), -100)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Pages:
    """A cache whose unused rows and pages hold NaN bits, with a shuffled block table."""

    def __init__(self, lengths, heads, dim, room=0, seed=0, spare=3, width=None):
        need = [-(-(n + room) // 64) for n in lengths]
        self.pages = sum(need) + spare
        self.cache = ops.kv8_cache(self.pages, heads, dim)
        for t in self.cache[:2]:
            t.view(torch.uint8).fill_(0x7F)
        g = torch.Generator().manual_seed(seed)
        order = torch.randperm(self.pages, generator=g).tolist()
        width = max(1, max(need)) if width is None else width
        self.rows, at = [], 0
        for n in need:
            self.rows.append(order[at:at + n] + [-1] * (width - n))
            at += n
        self.table, self.lengths, self.heads, self.dim = i32(self.rows), list(lengths), heads, dim

    def fill(self, seed=1, spread=False):
        """Tokens for all lengths; with ``spread`` the pages' scales differ by powers of two."""
        most = max(self.lengths)
        k, v = (randn(len(self.lengths), self.heads, most, self.dim, seed=seed + i) for i in range(2))
        if spread:
            page = torch.arange(most, device="cuda") // 64
            v = v * (2.0 ** (page % 7 - 3))[:, None].to(v.dtype)
            k = k * (2.0 ** ((page + 3) % 5 - 3))[:, None].to(k.dtype)
        if most:
            ops.kv8_write(self.cache, k, v, self.table, i32([0] * len(self.lengths)), i32(self.lengths))
        ops.check_operator_errors()
        return self

    def values(self, i, head, n):
        """fp64 keys, values and values' scales of a request's first n tokens."""
        pages = self.rows[i][:-(-n // 64)]
        k, v, ks, vs = self.cache
        return tuple((t[pages, head].double() * s[pages, head].double()[:, None, None]).flatten(0, 1)[:n]
                     for t, s in ((k, ks), (v, vs))) + (vs[pages, head].double().repeat_interleave(64)[:n],)


ADD = 2.0 ** -23  # one fp32 addition of a tensor core, which may truncate


def check_attention(out, q, p, lengths=None, scale=None):
    """The bound, for a row with scores x_j, probabilities p_j (p_top the largest) and n tokens:
    * a score: q's two terms miss it by 2^-17 of its largest element at most; 2 D additions;
    * a probability: that, and 2^-21 (exp2, its argument's rounding is added: 2^-23 of |x| + |x_top|); held to 2^-8 of
      itself and 2^-11 (through fp16), and to 2^-16 of the largest one times the largest value scale over its own;
    * the sums over 2 n terms, the denominator's over n;
    * the result: half a step of bf16, 2^-8 of its value."""
    lengths = p.lengths if lengths is None else lengths
    group = q.shape[1] // p.heads
    scale = p.dim ** -0.5 if scale is None else scale
    assert out.dtype == torch.bfloat16 and out.shape == q.shape
    for i, n in enumerate(lengths):
        for h in range(q.shape[1]):
            if n == 0:
                assert not out[i, h].any()
                continue
            k, v, vs = p.values(i, h // group, n)
            x = q[i, h].double()
            s = scale * x @ k.T
            s_off = scale * (2.0 ** -17 * x.abs().amax(1, keepdim=True) * k.abs().sum(1)
                             + 2 * p.dim * ADD * 1.07 * (x.abs() @ k.abs().T))
            w = torch.softmax(s, dim=1)
            w_off = s_off.exp() - 1 + 2.0 ** -21 + 2 * ADD * (s.abs() + s.amax(1, keepdim=True).abs())
            want = w @ v
            held = 2.0 ** -8 + 2.0 ** -11
            bound = (w * (w_off + held + 2 * n * ADD)) @ v.abs() \
                + 2.0 ** -16 * w.amax(1, keepdim=True) * (v.abs() / vs[:, None]).sum(0) * vs.max() \
                + want.abs() * (w_off.amax(1, keepdim=True) + n * ADD)
            off = (out[i, h].double() - want).abs()
            most = bound + 2.0 ** -8 * (want.abs() + bound) + 1e-30
            assert (off <= most).all(), (i, h, (off / most).max().item())


# ---------------------------------------------------------------------------
# write
# ---------------------------------------------------------------------------
def plain_write(store, scales, new, rows, starts, counts):
    """One tensor of the cache (fp32 values of its bytes, fp32 scales) on the CPU, token by token."""
    new = new.float().cpu()
    for b, (start, count) in enumerate(zip(starts, counts)):
        for h in range(new.shape[1]):
            for at in range(start // 64 * 64, start + count if count else 0, 64):
                page = rows[b][at // 64]
                mine = new[b, h, max(0, at - start):min(count, at + 64 - start)]
                held = max(0, start - at)
                scale = page_scale(mine.abs().max().item())
                if held:
                    old = scales[page, h].item()
                    scale = float("nan") if math.isnan(old) or math.isnan(scale) else max(scale, old)
                    store[page, h, :held] = (store[page, h, :held] * (old / scale)).to(E4M3).float()
                store[page, h, held:held + len(mine)] = (mine / scale).to(E4M3).float()
                scales[page, h] = scale


def check_write(p, k, v, starts, counts=None):
    ks, vs = ([t.float().cpu(), s.cpu().clone()] for t, s in ((p.cache.k, p.cache.k_scale), (p.cache.v, p.cache.v_scale)))
    full = [k.shape[2]] * k.shape[0] if counts is None else counts
    plain_write(*ks, k, p.rows, starts, full)
    plain_write(*vs, v, p.rows, starts, full)
    ops.kv8_write(p.cache, k, v, p.table, i32(starts), None if counts is None else i32(counts))
    ops.check_operator_errors()
    for got, want in ((p.cache.k.float().cpu(), ks[0]), (p.cache.v.float().cpu(), vs[0]),
                      (p.cache.k_scale.cpu(), ks[1]), (p.cache.v_scale.cpu(), vs[1])):
        assert torch.equal(got.nan_to_num(nan=1e9), want.nan_to_num(nan=1e9))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("starts,tokens,counts", [
    ([0], 1, None), ([0, 0], 64, None), ([0, 0], 65, [65, 3]), ([5, 64, 63, 130], 7, None), ([1, 0, 127], 300, [300, 0, 1]),
    ([60], 4, None), ([60], 5, None), ([0, 1, 2], 200, [0, 0, 0])])
def test_write(cuda_device, dim, starts, tokens, counts):
    p = Pages(starts, heads=3, dim=dim, room=tokens)
    if max(starts):
        p.fill(seed=5)
    k, v = (randn(len(starts), 3, tokens, dim, seed=s) * f for s, f in ((2, 30.0), (3, 0.02)))  # a larger, a smaller scale
    check_write(p, k, v, starts, counts)


def test_write_token_by_token(cuda_device):
    """A page filled one token at a time, growing: each step rounds the page again."""
    p = Pages([0], heads=2, dim=64, room=70)
    for i in range(70):
        k, v = (randn(1, 2, 1, 64, seed=i) * 1.1 ** (i % 50) for _ in range(2))
        check_write(p, k, v, [i])


def test_write_special_values(cuda_device):
    p = Pages([0, 0, 0, 0], heads=1, dim=64, room=128)
    x = randn(4, 1, 100, 64)
    x[0, 0, 3, 5] = float("inf")
    x[1, 0, 70, 1] = float("nan")
    x[2] = 0
    x[3] = torch.tensor([448.0, 449.0, 1e-30, 3e38, -3e38, 1e-38, 2.0 ** -140, -0.0] * 8, device="cuda").bfloat16()
    check_write(p, x, x.flip(2), [0] * 4)
    check_write(p, randn(4, 1, 5, 64), randn(4, 1, 5, 64), [100] * 4)  # behind them, in the same pages
    p = Pages([0], heads=1, dim=64, room=3)
    for edge in (448.0, 450.0, 1.75 * 2.0 ** 5, 1.7578125 * 2.0 ** 5, 2.0 ** 10):
        x = torch.full((1, 1, 3, 64), edge, device="cuda").bfloat16()
        check_write(p, x, -x, [0])


def test_write_views(cuda_device):
    p, same = (Pages([0, 0], heads=3, dim=64, room=90) for _ in range(2))
    qkv = randn(2, 90, 3, 3, 64)
    k, v = qkv[:, :, 1].transpose(1, 2), qkv[:, :, 2].transpose(1, 2)
    check_write(p, k, v, [0, 0])
    odd = torch.zeros(2, 3, 90, 67, device="cuda", dtype=torch.bfloat16)[..., 3:]
    odd.copy_(k)
    check_write(same, odd, v.contiguous(), [0, 0])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(p.cache[:2], same.cache[:2]))
    check_write(p, randn(1, 1, 70, 64).expand(2, 3, -1, -1), v[:, :, :70], [0, 0])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,heads,group,queries", [
    ([1], 1, 1, 1), ([0], 2, 1, 3), ([64], 1, 1, 1), ([63, 65, 127, 128, 129], 2, 1, 1), ([1000, 0, 3, 257], 2, 5, 1),
    ([300], 1, 8, 16), ([700, 90], 2, 1, 128), ([700, 90, 0], 1, 1, 129), ([200, 64], 2, 2, 200), ([513], 1, 1, 256),
    ([77, 512], 3, 1, 700), ([130] * 40, 1, 2, 3), ([2049], 2, 3, 100)])
def test_attention(cuda_device, dim, lengths, heads, group, queries):
    p = Pages(lengths, heads, dim).fill(spread=True)
    q = randn(len(lengths), heads * group, queries, dim, seed=9)
    out = ops.kv8_attention(q, p.cache, p.table, i32(lengths))
    ops.check_operator_errors()
    check_attention(out, q, p)
    assert torch.equal(out, ops.kv8_attention(q, p.cache, p.table, i32(lengths)))


@pytest.mark.parametrize("lengths,heads,group,queries", [([20000, 7, 3000], 2, 4, 1), ([5000], 1, 1, 600),
                                                         ([40000], 1, 2, 2)])
def test_long(cuda_device, lengths, heads, group, queries):
    """Units over many blocks: their parts are joined."""
    p = Pages(lengths, heads, 128).fill()
    q = randn(len(lengths), heads * group, queries, 128, seed=9)
    out = ops.kv8_attention(q, p.cache, p.table, i32(lengths))
    ops.check_operator_errors()
    check_attention(out, q, p)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group,queries", [(4, 1, 1), (3, 5, 1), (2, 4, 9), (2, 1, 70), (1, 3, 40)])
def test_many_short_requests(cuda_device, dim, heads, group, queries):
    """Several units of few rows and steps for each block, of one step and of more in turn."""
    lengths = [(37 * i) % 131 if i % 5 else (101 * i) % 700 for i in range(400)]
    p = Pages(lengths, heads, dim).fill(spread=True)
    q = randn(len(lengths), heads * group, queries, dim, seed=9)
    out = ops.kv8_attention(q, p.cache, p.table, i32(lengths))
    ops.check_operator_errors()
    check_attention(out, q, p)
    for _ in range(5):
        assert torch.equal(out, ops.kv8_attention(q, p.cache, p.table, i32(lengths)))


def test_sharp_and_wide_scores(cuda_device):
    """One token takes all; scores of some hundreds that grow along the tokens; q's elements far apart; zeros."""
    p = Pages([700], 1, 64).fill()
    for q in (p.values(0, 0, 700)[0][300][None, None, None].bfloat16() * 20, randn(1, 1, 40, 64) * 30,
              randn(1, 1, 40, 64) * torch.logspace(-6, 2, 64, device="cuda").bfloat16(),
              torch.zeros(1, 1, 3, 64, device="cuda").bfloat16(), randn(1, 1, 200, 64) * 1e-20):
        check_attention(ops.kv8_attention(q, p.cache, p.table, i32([700])), q, p)
    k = torch.arange(700, device="cuda")[:, None] * torch.ones(64, device="cuda") * 0.05
    k = k.bfloat16()[None, None]
    ops.kv8_write(p.cache, k, randn(1, 1, 700, 64), p.table, i32([0]))
    for sign in (1.0, -1.0):
        q = torch.full((1, 1, 130, 64), sign, device="cuda").bfloat16()
        check_attention(ops.kv8_attention(q, p.cache, p.table, i32([700])), q, p)


def test_far_scales(cuda_device):
    """Pages whose scales are 2^60 and more apart, smallest first and last."""
    for order in (1, -1):
        p = Pages([256], 1, 64)
        f = torch.tensor([1e-18, 1.0, 1e-25, 1e20][::order], device="cuda").repeat_interleave(64)[:, None]
        ops.kv8_write(p.cache, randn(1, 1, 256, 64), (randn(1, 1, 256, 64, dtype=torch.float32) * f).bfloat16(), p.table,
                      i32([0]))
        for n in (64, 130, 256):
            q = randn(1, 1, 5, 64)
            check_attention(ops.kv8_attention(q, p.cache, p.table, i32([n])), q, p, [n])


def test_pages_with_nan_stay_among_themselves(cuda_device):
    p = Pages([300, 300], 2, 64).fill()
    q = randn(2, 4, 150, 64)
    clean = ops.kv8_attention(q, p.cache, p.table, i32([300, 300]))
    bad = randn(1, 2, 1, 64)
    bad[0, 1] = float("nan")
    ops.kv8_write(p.cache, bad, randn(1, 2, 1, 64), p.table[1:], i32([299]))  # keys of request 1, head 1
    out = ops.kv8_attention(q, p.cache, p.table, i32([300, 300]))
    ops.check_operator_errors()
    assert torch.equal(out[0], clean[0]) and out[1, 2:].isnan().all() and not out[1, :2].isnan().any()
    out = ops.kv8_attention(q, p.cache, p.table, i32([300, 256]))  # before that page
    assert torch.equal(out[1, 2:], ops.kv8_attention(q, p.cache, p.table, i32([256, 256]))[1, 2:])
    assert not out.isnan().any()
    q[0, 0, 7, 3] = float("inf")
    out = ops.kv8_attention(q, p.cache, p.table, i32([300, 0]))
    assert out[0, 0, 7].isnan().all()
    keep = torch.arange(150, device="cuda") != 7
    assert torch.equal(out[0, 0, keep], clean[0, 0, keep]) and torch.equal(out[0, 1:], clean[0, 1:]) and not out[1].any()


def test_views_out_and_scale(cuda_device):
    p = Pages([200, 100], 2, 64).fill()
    q = randn(2, 4, 150, 64)
    n = i32([200, 100])
    want = ops.kv8_attention(q, p.cache, p.table, n, scale=0.3)
    check_attention(want, q, p, scale=0.3)
    token_major = q.transpose(1, 2).contiguous().transpose(1, 2)
    got = ops.kv8_attention(token_major, p.cache, p.table, n, scale=0.3)
    assert torch.equal(got, want) and got.stride() == token_major.stride()
    odd = torch.zeros(2, 4, 150, 67, device="cuda").bfloat16()[..., 3:]
    odd.copy_(q)
    assert torch.equal(ops.kv8_attention(odd, p.cache, p.table, n, scale=0.3), want)
    assert torch.equal(ops.kv8_attention(q.transpose(2, 3).contiguous().transpose(2, 3), p.cache, p.table, n, 0.3), want)
    same = q[:, :1].expand(-1, 4, -1, -1)
    assert torch.equal(ops.kv8_attention(same, p.cache, p.table, n),
                       ops.kv8_attention(same.contiguous(), p.cache, p.table, n))
    store = torch.full((2, 150, 6, 64), 7.0, device="cuda").bfloat16()
    out = store[:, :, 1:5].transpose(1, 2)
    assert ops.kv8_attention(q, p.cache, p.table, n, 0.3, out=out) is out
    assert torch.equal(out, want) and (store[:, :, 0] == 7).all() and (store[:, :, 5] == 7).all()
    whole = q.clone()
    ops.kv8_attention(whole, p.cache, p.table, n, 0.3, out=whole)
    assert torch.equal(whole, want)


def test_shared_pages_and_lengths(cuda_device):
    """Several requests read one page; a length behind the table is cut; one below zero is none."""
    p = Pages([200], 2, 128).fill()
    q = randn(4, 2, 9, 128)
    table = p.table.expand(4, -1)
    out = ops.kv8_attention(q, p.cache, table, i32([200, 70, -3, 1 << 30]))
    p.rows, lengths = p.rows * 4, [200, 70, 0, 64 * p.table.shape[1]]
    p.cache.k.view(torch.uint8)[p.rows[0][-1], :, 8:] = 0  # rows behind the last token, now read
    p.cache.v.view(torch.uint8)[p.rows[0][-1], :, 8:] = 0
    out = ops.kv8_attention(q, p.cache, table, i32([200, 70, -3, 1 << 30]))
    check_attention(out, q, p, lengths)


def test_nothing(cuda_device):
    p = Pages([100], 2, 64).fill()
    for q in (randn(1, 4, 0, 64), randn(0, 4, 3, 64)):
        n = q.shape[0]
        assert ops.kv8_attention(q, p.cache, p.table[:n], i32([100][:n])).shape == q.shape
    empty = ops.kv8_cache(0, 2, 64)
    q = randn(2, 2, 300, 64)
    assert not ops.kv8_attention(q, empty, torch.zeros(2, 0, dtype=torch.int32, device="cuda"), i32([5, 0])).any()
    assert not ops.kv8_attention(q, empty, torch.zeros(2, 3, dtype=torch.int32, device="cuda"), i32([5, 0])).any()
    ops.kv8_write(p.cache, randn(1, 2, 0, 64), randn(1, 2, 0, 64), p.table, i32([100]))
    ops.check_operator_errors()


def test_errors_are_reported(cuda_device):
    p = Pages([200], 2, 64, room=100).fill()
    before = [t.view(torch.uint8).clone() for t in p.cache[:2]]
    q, n = randn(1, 2, 5, 64), i32([200])
    for bad in (-1, p.pages, 1 << 30):
        table = p.table.clone()
        table[0, 3] = bad
        assert ops.kv8_attention(q, p.cache, table, i32([192])).isfinite().all()  # not needed
        ops.check_operator_errors()
        ops.kv8_attention(q, p.cache, table, n)
        with pytest.raises(RuntimeError, match="page that does not exist"):
            ops.check_operator_errors()
        ops.kv8_write(p.cache, randn(1, 2, 3, 64), randn(1, 2, 3, 64), table, i32([197]))
        with pytest.raises(RuntimeError, match="page that does not exist"):
            ops.check_operator_errors()
    assert all(torch.equal(a, t.view(torch.uint8)) for a, t in zip(before, p.cache[:2]))
    ops.kv8_write(p.cache, randn(1, 2, 100, 64), randn(1, 2, 100, 64), p.table[:, :4], i32([200]))  # behind the table
    with pytest.raises(RuntimeError, match="page that does not exist"):
        ops.check_operator_errors()
    for bad in (0.3, 0.0, -1.0, float("inf")):
        scales = p.cache.v_scale.clone()
        scales[p.rows[0][1], 1] = bad
        out = ops.kv8_attention(q, p.cache._replace(v_scale=scales), p.table, n)
        with pytest.raises(RuntimeError, match="power of two"):
            ops.check_operator_errors()
        assert out[0, 1].isnan().all() and out[0, 0].isfinite().all()
    ops.check_operator_errors()


def test_refusals(cuda_device):
    p = Pages([100, 50], 2, 64).fill()
    k, n = randn(2, 2, 5, 64), i32([100, 50])
    c = p.cache
    bad_caches = (c._replace(k=c.k[:, :1]), c._replace(v=c.v[1:]), c._replace(k_scale=c.k_scale[:, :1]),
                  c._replace(k=c.k.view(torch.uint8)), c._replace(v_scale=c.v_scale.double()),
                  c._replace(k=c.k.transpose(0, 1).contiguous().transpose(0, 1)), c._replace(v=c.v.cpu()),
                  ops.KV8Cache(*(t[:, :, :32] for t in c[:2]), *c[2:]))
    for cache in bad_caches:
        with pytest.raises(ValueError):
            ops.kv8_write(cache, k, k, p.table, n)
        with pytest.raises(ValueError):
            ops.kv8_attention(k, cache, p.table, n)
    for args in ((k.float(), k, p.table, n), (k, k[:, :, :4], p.table, n), (k[:, :1], k[:, :1], p.table, n),
                 (k[..., :32], k[..., :32], p.table, n), (k, k, p.table[:1], n), (k, k, p.table.long(), n),
                 (k, k, p.table, n[:1]), (k, k, p.table, n.long()), (k, k, p.table, n, n[:1]), (k, k, p.table, n.cpu()),
                 (k.clone().requires_grad_(), k, p.table, n)):
        with pytest.raises(ValueError):
            ops.kv8_write(c, *args)
    wide = torch.zeros(2, 2, 5, 68, device="cuda").bfloat16()
    for q, args, kw in ((k.float(), (p.table, n), {}), (k[..., :32], (p.table, n), {}), (randn(2, 3, 5, 64), (p.table, n), {}),
                        (k[:1], (p.table, n), {}), (k, (p.table, n[:1]), {}), (k, (p.table[0], n), {}),
                        (k, (p.table, n), dict(scale=0.0)), (k, (p.table, n), dict(scale=-1.0)),
                        (k, (p.table, n), dict(scale=float("nan"))), (k, (p.table, n), dict(out=k[:1])),
                        (k, (p.table, n), dict(out=k.float())), (k, (p.table, n), dict(out=wide[..., 4:])),
                        (k, (p.table, n), dict(out=randn(2, 1, 5, 64).expand(-1, 2, -1, -1))),
                        (randn(2, 0, 5, 64), (p.table, n), {}), (k.clone().requires_grad_(), (p.table, n), {})):
        with pytest.raises(ValueError):
            ops.kv8_attention(q, c, *args, **kw)
    for args in ((3, 2, 96), (3, 0, 64), (-1, 2, 64)):
        with pytest.raises(ValueError):
            ops.kv8_cache(*args)


def test_streams_and_graph(cuda_device):
    """Two calls at once on streams of their own; write and attention captured, and replayed with other lengths and
    tokens; two graphs in turn."""
    p = Pages([3064, 564], 2, 128, width=60).fill()  # every token that a length below counts has been written
    q = randn(2, 8, 1, 128)
    n = i32([3000, 500])
    want = ops.kv8_attention(q, p.cache, p.table, n)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.kv8_attention(q, p.cache, p.table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    k, v, starts, after = randn(2, 2, 1, 128), randn(2, 2, 1, 128), n.clone(), n + 1
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.kv8_write(p.cache, k, v, p.table, starts)
            out = ops.kv8_attention(q, p.cache, p.table, after)
        graphs.append((g, out))
    for lengths in ([3000, 500], [3001, 501], [64, 0], [3050, 130]):
        starts.copy_(i32(lengths))
        after.copy_(starts + 1)
        k.copy_(randn(2, 2, 1, 128, seed=lengths[0]))
        v.copy_(randn(2, 2, 1, 128, seed=lengths[1]))
        for g, out in graphs:
            g.replay()
            check_attention(out, q, p, [x + 1 for x in lengths])
    ops.check_operator_errors()


def test_pages_past_4_gib(cuda_device):
    """A cache of more than 2^32 bytes for keys and for values, its last pages in use; 2^31 elements between the
    queries' requests."""
    heads, dim, tokens = 8, 128, 700
    cache = ops.kv8_cache(66000, heads, dim)
    assert cache.k.numel() > 1 << 32
    p = Pages([tokens], heads, dim)
    p.cache, p.pages = cache, 66000
    p.rows = [[66000 - 1 - 5 * i for i in range(11)]]
    p.table = i32(p.rows)
    p.fill(spread=True)
    store = torch.empty(2 * (1 << 31) + 64 * heads * dim, dtype=torch.bfloat16, device="cuda")
    q = store.as_strided((2, heads, 3, dim), ((1 << 31) + 512, dim, heads * dim, 1))
    q.copy_(randn(2, heads, 3, dim, seed=4))
    out = ops.kv8_attention(q, cache, p.table.expand(2, -1), i32([tokens, 130]))
    ops.check_operator_errors()
    p.rows = p.rows * 2
    check_attention(out, q, p, [tokens, 130])


@pytest.mark.parametrize("queries,group", [(1, 33), (1, 32), (4, 8), (127, 1), (43, 3)])
def test_row_counts_at_the_kernels_edges(cuda_device, queries, group):
    """32 and 33, 127 to 129 rows: quarters of a step, copies of the rows, two tiles."""
    for n in (1, 31, 33, 64, 97, 129, 385):
        p = Pages([n, 0, n + 700], 1, 64).fill(spread=True)
        q = randn(3, group, queries, 64, seed=n)
        out = ops.kv8_attention(q, p.cache, p.table, i32(p.lengths))
        ops.check_operator_errors()
        check_attention(out, q, p)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths,heads,group,queries", [
    ([1], 1, 1, 129), ([0], 2, 1, 300), ([63, 65, 127, 128, 129], 2, 1, 200), ([700, 90, 0], 1, 1, 129),
    ([200, 64], 2, 2, 200), ([513], 1, 1, 256), ([77, 512], 3, 1, 700), ([130, 1, 257] * 40, 1, 2, 150), ([6000, 300], 1, 3, 100)])
def test_wide_tables(cuda_device, dim, lengths, heads, group, queries):
    """Tables of many pages for each request, of which few are in use; several units of two tiles, and of one that is
    not full, for each block."""
    p = Pages(lengths, heads, dim, width=100).fill(spread=True)
    q = randn(len(lengths), heads * group, queries, dim, seed=9)
    out = ops.kv8_attention(q, p.cache, p.table, i32(lengths))
    ops.check_operator_errors()
    check_attention(out, q, p)
    for _ in range(3):
        assert torch.equal(out, ops.kv8_attention(q, p.cache, p.table, i32(lengths)))
    if lengths != [6000, 300]:
        narrow = p.table[:, :max(1, -(-max(lengths) // 64))]
        check_attention(ops.kv8_attention(q, p.cache, narrow, i32(lengths)), q, p)


def test_wide_tables_sharp_scores_and_nan(cuda_device):
    p = Pages([700, 300], 1, 64, width=40).fill()
    for q in (p.values(0, 0, 700)[0][300].bfloat16().expand(2, 1, 300, 64) * 20, randn(2, 1, 300, 64) * 30,
              torch.zeros(2, 1, 300, 64, device="cuda").bfloat16()):
        check_attention(ops.kv8_attention(q, p.cache, p.table, i32([700, 300])), q, p)
    q = randn(2, 1, 300, 64)
    clean = ops.kv8_attention(q, p.cache, p.table, i32([700, 300]))
    q[0, 0, 7, 3] = float("inf")
    out = ops.kv8_attention(q, p.cache, p.table, i32([700, 300]))
    keep = torch.arange(300, device="cuda") != 7
    assert out[0, 0, 7].isnan().all() and torch.equal(out[0, 0, keep], clean[0, 0, keep]) and torch.equal(out[1], clean[1])
