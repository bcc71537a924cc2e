"""kv8_attention where one key dominates a long tail: the small probabilities count as the denominator counts them."""
import pytest
import torch

from pasa_b200 import ops

pytestmark = pytest.mark.gpu
ADD = 2.0 ** -23  # one fp32 addition of a tensor core, which may truncate


def filled(k, v):
    """A cache of one request's k and v [H, L, D] and its table."""
    heads, tokens, dim = k.shape
    pages = -(-tokens // 64)
    cache = ops.kv8_cache(pages, heads, dim)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").flip(0)[None]
    ops.kv8_write(cache, k[None].bfloat16(), v[None].bfloat16(), table, torch.zeros(1, dtype=torch.int32, device="cuda"))
    return cache, table


def held(cache, table, tokens):
    """fp64 keys and values [H, L, D] of the cache, and the values' scales [H, L]."""
    pages = table[0].long()
    k, v = ((t[pages].double() * s[pages].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :tokens]
            for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    return k, v, cache.v_scale[pages].double().T.repeat_interleave(64, dim=1)[:, :tokens]


def check(out, q, k, v, vs):
    """out [B, L, D] of one head, all from the same q [L, D], k, v.  For a row with probabilities w_j over n tokens:
    * a score: q's two terms miss it by 2^-17 of its largest element at most; 2 D additions; exp2 and the rounding of
      its argument;
    * a probability: half a step of fp16, 2^-11 of itself, or 2^-36 of the largest one times the largest value scale over
      its own where that is more (half the smallest step, 2^-25, under a reference that is held at 2^11);
    * the sums over n terms, and the denominator's;
    * the result: half a step of bf16, 2^-8 of its value.
    Nothing here but fp32's additions grows with the number of tokens that weigh next to nothing."""
    n, dim = k.shape
    scale = dim ** -0.5
    x = q.double()
    s = scale * x @ k.T
    s_off = scale * (2.0 ** -17 * x.abs().amax(1, keepdim=True) * k.abs().sum(1)
                     + 2 * dim * ADD * 1.07 * (x.abs() @ k.abs().T))
    w = torch.softmax(s, dim=1)
    w_off = s_off.exp() - 1 + 2.0 ** -21 + 2 * ADD * (s.abs() + s.amax(1, keepdim=True).abs())
    want = w @ v
    bound = (w * (w_off + 2.0 ** -11 + n * ADD)) @ v.abs() \
        + 2.0 ** -36 * w.amax(1, keepdim=True) * (v.abs() / vs[:, None]).sum(0) * vs.max() \
        + want.abs() * ((w * w_off).sum(1, keepdim=True) + n * ADD)
    most = bound + 2.0 ** -8 * (want.abs() + bound) + 1e-30
    off = (out.double() - want).abs()
    assert (off <= most).all(), (off / most).max().item()


@pytest.mark.parametrize("tokens,first", [(512, 0), (512, 300), (4096, 0), (18720, 0), (18720, 9000), (32767, 0)])
@pytest.mark.parametrize("rows,group", [(1, 1), (8, 4), (100, 1), (128, 2), (300, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_dominating_key_over_a_flat_tail(cuda_device, dim, rows, group, tokens, first):
    """Every row has another gap of 8 to 13 nats between the one key and the others, which score alike; among the
    gaps those whose probabilities lie next to powers of two.  Values of mean 1, and nothing but the tail in the last
    dimensions.  Enough requests, all of the same pages, that most are one block's whole, and one that is cut."""
    heads_b = 200 if tokens < 10000 else 150
    k = torch.zeros(1, tokens, dim, device="cuda")
    k[0, first, 0] = 4.0
    g = torch.Generator(device="cuda").manual_seed(tokens)
    v = 0.75 + 0.5 * torch.rand(1, tokens, dim, generator=g, device="cuda")
    v[0, first, dim // 2:] = 0
    cache, table = filled(k, v)
    gaps = torch.linspace(8, 13, rows, device="cuda") if rows > 1 else torch.full((1,), 10.3, device="cuda")
    gaps[::3] = (gaps[::3] / 0.693147).round() * 0.693147 + 0.004  # the tail just below a power of two
    q = torch.zeros(rows, dim, device="cuda")
    q[:, 0] = gaps * dim ** 0.5 / 4
    q = q.bfloat16()
    for batch in (1, heads_b):
        some = q.view(1, rows // group, group, dim).transpose(1, 2).expand(batch, -1, -1, -1)
        out = ops.kv8_attention(some, cache, table.expand(batch, -1),
                                torch.full((batch,), tokens, dtype=torch.int32, device="cuda"))
        ops.check_operator_errors()
        check(out.transpose(1, 2).flatten(1, 2), q, *(t[0] for t in held(cache, table, tokens)))


@pytest.mark.parametrize("rows", [1, 100, 300])
def test_a_dominating_key_over_a_spread_tail(cuda_device, rows):
    """Scores of the tail with a spread of about a nat, pages of values whose scales differ."""
    tokens, dim, batch = 8000, 128, 150
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randn(1, tokens, dim, generator=g, device="cuda")
    k[..., 0] = 0
    k[0, 5] = 0
    k[0, 5, 0] = 4.0
    v = torch.rand(1, tokens, dim, generator=g, device="cuda") + 0.1
    v *= 2.0 ** (torch.arange(tokens, device="cuda") // 64 % 9 - 4)[:, None]
    cache, table = filled(k, v)
    q = torch.randn(rows, dim, generator=g, device="cuda")
    q[:, 0] = torch.linspace(9, 14, max(rows, 2), device="cuda")[:rows] * dim ** 0.5 / 4
    q = q.bfloat16()
    out = ops.kv8_attention(q[None, None].expand(batch, -1, -1, -1), cache, table.expand(batch, -1),
                            torch.full((batch,), tokens, dtype=torch.int32, device="cuda"))
    ops.check_operator_errors()
    check(out[:, 0], q, *(t[0] for t in held(cache, table, tokens)))


@pytest.mark.parametrize("rows,group", [(1, 1), (24, 8), (100, 1), (150, 1), (300, 2), (520, 1)])
@pytest.mark.parametrize("dim", [64, 128])
def test_units_of_many_steps_one_behind_the_other(cuda_device, dim, rows, group):
    """Every block goes through several units of 1 to 12 steps, cut ones among them, whose last pages are full, begun
    or absent, so that each place of its rings is used many times."""
    lengths = [257, 130, 1, 1500, 512, 64, 65, 700, 385, 1025, 448, 900]
    tokens, batch = max(lengths), 40 * len(lengths)
    g = torch.Generator(device="cuda").manual_seed(3)
    k, v = (torch.randn(1, tokens, dim, generator=g, device="cuda") for _ in range(2))
    v *= 2.0 ** (torch.arange(tokens, device="cuda") // 64 % 7 - 3)[:, None]
    cache, table = filled(k, v)
    q = torch.randn(rows, dim, generator=g, device="cuda").bfloat16()
    some = q.view(1, rows // group, group, dim).transpose(1, 2).expand(batch, -1, -1, -1)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda").repeat(40)
    for _ in range(3):
        out = ops.kv8_attention(some, cache, table.expand(batch, -1), n)
        ops.check_operator_errors()
        for i, length in enumerate(lengths):
            check(out[i::len(lengths)].transpose(1, 2).flatten(1, 2), q, *(t[0] for t in held(cache, table, length)))
