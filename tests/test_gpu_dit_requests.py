"""A denoising step for several requests on the GPU: adapters, the text's keys and values in 8 bits, and the operators
of one cached video chunk in a row."""
import pytest
import torch
import torch.nn.functional as F

from pasa_b200 import dit, ops
from test_gpu_kv8 import Pages, check_attention, i32
from test_gpu_rope_axes import check as check_rope
from test_gpu_rope_axes import grid_positions, plain

pytestmark = pytest.mark.gpu
CFG = dit.DiTConfig(hidden=512, heads=4, ffn=1024, layers=2, text_len=70, frames=2, height=16, width=32,
                    in_channels=16, text_dim=64, freq_dim=32)
NAMES = ("q", "k", "v", "o", "cq", "co", "ffn1", "ffn2")


def _setup(device, batch=3):
    g = torch.Generator().manual_seed(3)
    lat = torch.randn((batch, CFG.in_channels, CFG.frames, 2 * CFG.height, 2 * CFG.width), generator=g).to(device)
    txt = torch.randn((batch, CFG.text_len, CFG.text_dim), generator=g).to(device)
    blocks = [dit.init_block(CFG, 20 + i, device) for i in range(CFG.layers)]
    adapters = []
    for w in blocks:
        adapters.append({n: ((torch.randn((2, 16, w[n].shape[1]), generator=g) * 0.02).to(device, torch.bfloat16),
                             (torch.randn((2, w[n].shape[0], 16), generator=g) * 0.2).to(device, torch.bfloat16))
                         for n in NAMES})
    adapters = dit.Adapters(i32([1, -1, 0][:batch]), torch.tensor([1.0, 0.5], device=device), adapters)
    return dit.patchify(lat), txt, blocks, dit.init_embed(CFG, 2, device), dit.rope_table(CFG, device), adapters


def _fp32(w):
    return {k: v.float() for k, v in w.items()}


def _dense(q, k, v):
    from pasa_b200 import dense_attention
    return dense_attention(q, k, v)


def _sdpa32(q, k, v):
    return F.scaled_dot_product_attention(q.float(), k.float(), v.float())


@pytest.mark.parametrize("with_adapters,cached", [(True, False), (False, True), (True, True)])
def test_fused_step_matches_fp32_torch(cuda_device, with_adapters, cached):
    """The fused step against the torch step in fp32 with the same adapters and cached bytes: bf16 activations through
    two blocks, as for the step without them."""
    x, txt, blocks, emb, rope, adapters = _setup(cuda_device)
    t = torch.tensor([700, 300, 50], device=cuda_device)
    kv = dit.text_cache(txt, emb, blocks, CFG, lengths=i32([70, 64, 3])) if cached else None
    kw = dict(adapters=adapters) if with_adapters else {}
    got = dit.step(x, t, None if cached else txt, rope, emb, blocks, CFG, _dense, fused=True, text_kv=kv, **kw).float()
    if with_adapters:
        kw = dict(adapters=adapters._replace(blocks=[{n: tuple(m.float() for m in p) for n, p in b.items()}
                                                     for b in adapters.blocks]))
    want = dit.step(x.float(), t, txt, rope, _fp32(emb), [_fp32(b) for b in blocks], CFG, _sdpa32, text_kv=kv, **kw)
    ops.check_operator_errors()
    err, ref = (got - want).abs().max().item(), want.abs().max().item()
    cos = F.cosine_similarity(got.flatten(), want.flatten(), dim=0).item()
    assert err < 3e-2 * ref and cos > 0.999, (err, ref, cos)
    base = dit.step(x, t, txt, rope, emb, blocks, CFG, _dense, fused=True).float()
    assert not torch.equal(got, base)
    if with_adapters and not cached:
        assert torch.equal(got[1], base[1])  # a request without an adapter


def test_text_cache_holds_the_text(cuda_device):
    """Half a step of e4m3: 2^-4 of a value, and 2^-10 of the page's scale for the smallest; and the same values in
    bf16 through another order of the sums (2^-7)."""
    _, txt, blocks, emb, _, _ = _setup(cuda_device)
    lengths = [70, 64, 3]
    kv = dit.text_cache(txt, emb, blocks, CFG, lengths=i32(lengths))
    text = dit.project_text(emb, txt)
    for w, cache in zip(blocks, kv.blocks):
        for t, s, want in ((cache.k, cache.k_scale, dit._text_keys(text, w, CFG, fused=True)),
                           (cache.v, cache.v_scale, F.linear(text, w["cv"], w["cv_b"]))):
            want = dit._heads(want, CFG).double()
            for b, n in enumerate(lengths):
                pages = kv.table[b].long()
                scale = s[pages].double()[:, :, None, None].expand(-1, -1, 64, 1).transpose(0, 1).flatten(1, 2)[:, :n]
                held = t[pages].double().transpose(0, 1).flatten(1, 2)[:, :n] * scale
                bound = (2.0 ** -4 + 2.0 ** -7) * want[b, :, :n].abs() + 2.0 ** -10 * scale
                assert ((held - want[b, :, :n]).abs() <= bound).all()


def test_padded_texts_are_cut(cuda_device):
    """What lies behind a text's length is not attended to: the same step, bit for bit, with other padding."""
    x, txt, blocks, emb, rope, _ = _setup(cuda_device)
    t, lengths = torch.tensor([700, 300, 50], device=cuda_device), [70, 10, 0]
    a = dit.text_cache(txt, emb, blocks, CFG, lengths=i32(lengths))
    other = txt.clone()
    for b, n in enumerate(lengths):
        other[b, n:] = float("nan")
    b = dit.text_cache(other, emb, blocks, CFG, lengths=i32(lengths))
    steps = [dit.step(x, t, None, rope, emb, blocks, CFG, _dense, fused=True, text_kv=c) for c in (a, b)]
    assert torch.equal(*steps) and steps[0].isfinite().all()


def _check_project(got, x, w, a, b, rows, slots, scale):
    """y = x w^T is rounded to bf16 once, then y + s (x a^T) b^T once more; sums of K terms in fp32 (2^-23 a term), h
    held to 2^-18."""
    x, w = x.double(), w.double()
    want, bound = x @ w.T, x.shape[1] * 2.0 ** -23 * (x.abs() @ w.abs().T)
    bound += 2.0 ** -8 * (want.abs() + bound)
    for i, slot in enumerate(slots):
        r = slice(rows[i], rows[i + 1])
        if slot >= 0:
            s, al, bl = scale[slot].double(), a[slot].double(), b[slot].double()
            h = s * x[r] @ al.T
            h_off = (x.shape[1] + 1) * 2.0 ** -23 * s * (x[r].abs() @ al.abs().T) + 2.0 ** -18 * h.abs()
            bound[r] += h_off @ bl.abs().T + (2 * a.shape[1] + 2) * 2.0 ** -23 * (want[r].abs() + h.abs() @ bl.abs().T)
            want[r] += h @ bl.T
    off = (got.double() - want).abs()
    assert (off <= bound + 2.0 ** -8 * (want.abs() + bound)).all()


@pytest.mark.parametrize("captured", [False, True])
def test_chunks_of_two_requests(cuda_device, captured):
    """A block's attention over the chunks of a video, as it is generated: projections with each request's adapter,
    rotary positions of the chunk's frames, keys and values rounded behind the earlier chunks', attention over all of
    them, output projection with its adapter.  Every stage is held against its formula on what the stage before gave.
    Captured, the same graph serves every chunk."""
    heads, dim, grid, rank = 2, 128, (1, 9, 13), 8
    axes, tokens, width = (44, 42, 42), 117, heads * dim
    g = torch.Generator(device="cuda").manual_seed(0)
    randn = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()  # noqa: E731
    p = Pages([0, 0], heads, dim, room=4 * tokens)
    w_qkv, w_o = randn(3 * width, width) * width ** -0.5, randn(width, width) * width ** -0.5
    lora = [(randn(2, rank, width) * width ** -0.5, randn(2, n, rank) * 0.3) for n in (3 * width, width)]
    scale, slots = torch.tensor([1.0, 0.5], device="cuda"), [1, 0]
    rows, slot_t = i32([0, tokens, 2 * tokens]), i32(slots)
    x, starts, after, origin = randn(2, tokens, width), i32([0, 0]), i32([0, 0]), 0
    where = torch.empty((tokens, 3), dtype=torch.int32, device="cuda")

    def chunk():
        qkv = F.linear(x, w_qkv)
        ops.lora_update(qkv, x, *lora[0], rows, slot_t, scale, out=qkv)
        q, k, v = (t.unflatten(2, (heads, dim)).transpose(1, 2) for t in qkv.chunk(3, dim=2))
        turned = ops.rope_axes(q, k, axes=axes, positions=where)
        ops.kv8_write(p.cache, turned[1], v, p.table, starts)
        o = ops.kv8_attention(turned[0], p.cache, p.table, after)
        flat = o.transpose(1, 2).flatten(2, 3)
        y = F.linear(flat, w_o)
        ops.lora_update(y, flat, *lora[1], rows, slot_t, scale, out=y)
        return qkv, q, k, turned, o, flat, y

    with torch.no_grad():
        graph = None
        for n in range(3):
            x.copy_(randn(2, tokens, width))
            starts.fill_(n * tokens)
            after.fill_((n + 1) * tokens)
            where.copy_(grid_positions(grid, (n, 0, 0), "cuda")[0])
            if captured and graph is None:
                chunk()  # (the libraries' first calls)
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    got = chunk()
            if captured:
                graph.replay()
            else:
                got = chunk()
            qkv, q, k, turned, o, flat, y = got
            _check_project(qkv.flatten(0, 1), x.flatten(0, 1), w_qkv, *lora[0], [0, tokens, 2 * tokens], slots, scale)
            for t, s in zip((q, k), turned):
                check_rope(s, t, plain(t, where[None], axes), axes)
            check_attention(o, turned[0], p, [(n + 1) * tokens] * 2)
            _check_project(y.flatten(0, 1), flat.flatten(0, 1), w_o, *lora[1], [0, tokens, 2 * tokens], slots, scale)
    ops.check_operator_errors()
