"""A denoising step for several requests (pasa_b200.dit, torch path): adapters and the text's cached keys and values."""
import pytest
import torch
import torch.nn.functional as F

from pasa_b200 import dit, ops

CFG = dit.DiTConfig(hidden=64, heads=4, ffn=128, layers=2, text_len=8, frames=2, height=4, width=4, in_channels=4,
                    text_dim=32, freq_dim=16)
NAMES = ("q", "k", "v", "o", "cq", "co", "ffn1", "ffn2")


def _inputs(batch=2):
    g = torch.Generator().manual_seed(0)
    lat = torch.randn((batch, CFG.in_channels, CFG.frames, 2 * CFG.height, 2 * CFG.width), generator=g)
    txt = torch.randn((batch, CFG.text_len, CFG.text_dim), generator=g)
    blocks = [dit.init_block(CFG, 10 + i, "cpu", torch.float32) for i in range(CFG.layers)]
    return dit.patchify(lat), txt, blocks, dit.init_embed(CFG, 1, "cpu", torch.float32)


def _step(x, txt, blocks, emb, **kw):
    return dit.step(x, torch.full((x.shape[0],), 500), txt, dit.rope_table(CFG, "cpu"), emb, blocks, CFG,
                    F.scaled_dot_product_attention, **kw)


def _adapters(blocks, slots, count=3, rank=8, names=NAMES, scale=(0.5, 2.0, 1.0)):
    g = torch.Generator().manual_seed(5)
    made = []
    for w in blocks:
        made.append({n: (torch.randn((count, rank, w[n].shape[1]), generator=g) * 0.1,
                         torch.randn((count, w[n].shape[0], rank), generator=g) * 0.1) for n in names})
    return dit.Adapters(torch.tensor(slots, dtype=torch.int32), None if scale is None else torch.tensor(scale), made)


def _merged(blocks, adapters, slot):
    out = []
    for w, block in zip(blocks, adapters.blocks):
        s = 1.0 if adapters.scale is None else adapters.scale[slot]
        out.append({**w, **{n: w[n] + s * (b[slot] @ a[slot]) for n, (a, b) in block.items()}})
    return out


@pytest.mark.parametrize("names", [NAMES, ("v", "ffn2"), ()])
@pytest.mark.parametrize("scale", [(0.5, 2.0, 1.0), None])
def test_adapters_are_their_merged_weights(names, scale):
    x, txt, blocks, emb = _inputs()
    adapters = _adapters(blocks, [1, -1], names=names, scale=scale)
    got = _step(x, txt, blocks, emb, adapters=adapters)
    merged = _step(x[:1], txt[:1], _merged(blocks, adapters, 1), emb)
    plain = _step(x[1:], txt[1:], blocks, emb)
    assert torch.allclose(got[:1], merged, atol=1e-4, rtol=1e-4)
    assert torch.allclose(got[1:], plain, atol=1e-5, rtol=1e-5)
    assert bool(names) != torch.allclose(got[:1], _step(x[:1], txt[:1], blocks, emb), atol=1e-4, rtol=1e-4)


def test_adapters_do_not_write_shared_outputs():
    x, txt, blocks, emb = _inputs()
    adapters = _adapters(blocks, [0, 2])
    a = _step(x, txt, blocks, emb, adapters=adapters)
    assert torch.equal(a, _step(x, txt, blocks, emb, adapters=adapters))


def _cpu_cache(txt, lengths, blocks, emb):
    """The cache of ``dit.text_cache`` with scales of 2^-7, rounded by torch."""
    text = dit.project_text(emb, txt)
    table = torch.tensor([[2], [0]], dtype=torch.int32)
    caches = []
    for w in blocks:
        cache = ops.kv8_cache(3, CFG.heads, 64, device="cpu")
        cache = ops.KV8Cache(*(t[..., :CFG.head_dim].clone() for t in cache[:2]), *(s * 2.0 ** -7 for s in cache[2:]))
        for t, new in zip(cache[:2], (dit._text_keys(text, w, CFG, False), F.linear(text, w["cv"], w["cv_b"]))):
            for b, page in enumerate(table[:, 0].tolist()):
                t[page, :, :CFG.text_len] = (dit._heads(new, CFG)[b] * 128).to(torch.float8_e4m3fn)
        caches.append(cache)
    return dit.TextCache(caches, table, torch.tensor(lengths, dtype=torch.int32))


def test_cached_text_is_attention_over_its_values():
    x, txt, blocks, emb = _inputs()
    cache = _cpu_cache(txt, [8, 3], blocks, emb)
    g = torch.Generator().manual_seed(1)
    q = torch.randn((2, CFG.heads, 5, CFG.head_dim), generator=g)
    out = dit._cached_attention_plain(q, cache.blocks[0], cache.table, cache.lengths)
    for b, n in enumerate((8, 3)):
        page = int(cache.table[b, 0])
        k, v = (t[page, :, :n].float() * s[page][:, None, None]
                for t, s in ((cache.blocks[0].k, cache.blocks[0].k_scale), (cache.blocks[0].v, cache.blocks[0].v_scale)))
        want = torch.softmax(q[b] @ k.transpose(1, 2) * CFG.head_dim ** -0.5, dim=-1) @ v
        assert torch.allclose(out[b], want, atol=1e-5, rtol=1e-5)
    none = dit._cached_attention_plain(q, cache.blocks[0], cache.table, torch.tensor([0, -2]))
    assert not none.any()


def test_step_reads_the_cache_and_no_text():
    """Cached values are within half a step of e4m3 (2^-4), and a step moves by less than that."""
    x, txt, blocks, emb = _inputs()
    cache = _cpu_cache(txt, [8, 8], blocks, emb)
    got, want = _step(x, None, blocks, emb, text_kv=cache), _step(x, txt, blocks, emb)
    assert (got - want).norm() <= 2.0 ** -4 * want.norm()
    short = _step(x, None, blocks, emb, text_kv=cache._replace(lengths=torch.tensor([8, 2], dtype=torch.int32)))
    assert torch.equal(short[:1], got[:1]) and not torch.equal(short[1:], got[1:])


def test_refusals():
    x, txt, blocks, emb = _inputs()
    adapters = _adapters(blocks, [0, 1])
    for bad in (adapters._replace(slots=adapters.slots[:1]), adapters._replace(blocks=adapters.blocks[:1]),
                adapters._replace(blocks=[{"ck": adapters.blocks[0]["q"]}, {}])):
        with pytest.raises(ValueError):
            _step(x, txt, blocks, emb, adapters=bad)
    cache = _cpu_cache(txt, [8, 8], blocks, emb)
    with pytest.raises(ValueError):
        _step(x, None, blocks, emb, text_kv=cache._replace(blocks=cache.blocks[:1]))
