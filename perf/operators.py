"""What is measured of three operators of a diffusion transformer's block, next to its sparse attention:

* ``rope``: rotary positions with several axes (frame, row, column) of the queries and keys, and its gradient
  (the inverse rotation);
* ``lora``: the low-rank adapters of many requests beside a shared projection, out = y + scale (x A^T) B^T with each
  request's own A and B on its own rows; ``lora_step`` is the same with its backward pass, as a training step takes it;
* ``kv8``: attention over keys and values held in 8 bits, in pages of 64 tokens with a power-of-two scale for each
  page and head, and the write of new tokens into them: the text of a prompt, kept over all denoising steps, or the
  frames so far of a video that is made chunk by chunk.

``run`` computes them in elementary torch operations, or with ``own`` set through this package's entry points.
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # Wan2.1-14B at 720p, one denoising step's self-attention: 21 x 45 x 80 latent patches, head-major
        rope_case("rope_wan14b_720p", heads=40, kv_heads=40, grid=[21, 45, 80], axes=[44, 42, 42]),
        # one latent frame with HunyuanVideo's heads at 480p, the video part of a sequence whose last 256 tokens are
        # text: latency and L2
        rope_case("rope_hunyuan_frame", heads=24, kv_heads=24, grid=[1, 30, 52], axes=[16, 56, 56], theta=256.0,
                  origin=[7, 0, 0], tail=256),
        # gradients in fp32 of a packed batch with a position for every token, token-major, grouped keys
        rope_case("rope_grad_tokens_f32", batch=2, heads=16, kv_heads=4, dim=80, tokens=4111, axes=[16, 24, 24],
                  dtype="f32", token_major=True, inverse=True),
        # one new token of each of eight requests, pairs (i, i + D/2), positions far out
        rope_case("rope_one_token", batch=8, heads=40, kv_heads=8, tokens=1, axes=[32, 48, 48], pairs="halves",
                  far=1 << 20),
        # one style adapter on a square projection of Wan2.1-14B at 720p
        lora_case("lora_wan14b_720p", lengths=[75600], k=5120, n=5120, rank=32, adapters=1),
        # prompts of ragged lengths into the cross-attention's keys; some without an adapter, a padded tail
        lora_case("lora_text_ragged", lengths=[512, 77, 1, 0, 300, 509, 64, 33, 128, 512, 255, 400, 17, 226, 512, 441],
                  k=5120, n=5120, rank=16, adapters=8, pad=109, without=3),
        # the timestep projection: one row of each request
        lora_case("lora_time_rows", lengths=[1] * 24, k=5120, n=30720, rank=64, adapters=16),
        # training one adapter of Wan2.1-14B at 480p
        lora_case("lora_step_wan14b_480p", op="lora_step", lengths=[32760], k=5120, n=5120, rank=64, adapters=1),
        # training three adapters at once on ragged rows, the widest rank
        lora_case("lora_step_ragged", op="lora_step", lengths=[1560, 3000, 77, 4000, 1], k=1536, n=8960, rank=128,
                  adapters=3, pad=47, without=5),
        # cross-attention of a guided step of Wan2.1-14B at 480p: the prompt's and the negative prompt's text
        kv8_case("kv8_text_wan14b", heads=40, kv_heads=40, queries=32760, lengths=[512, 77]),
        # the next three latent frames of a video at 480p with the heads of Wan2.1-1.3B join nine before them
        kv8_case("kv8_chunk_wan1b", heads=12, kv_heads=12, queries=4680, lengths=[14040], append=True),
        # one new token of each of eight requests, grouped keys, long caches
        kv8_case("kv8_one_token", heads=40, kv_heads=8, queries=1, append=True,
                 lengths=[32767, 20000, 32000, 777, 15000, 31001, 130, 24576]),
    ]


def rope_case(name=None, *, batch=1, heads, kv_heads, dim=128, axes, grid=None, origin=None, tokens=None, tail=0,
              theta=10000.0, dtype="bf16", token_major=False, inverse=False, pairs="interleaved", far=4096):
    """``grid``: the tokens are the grid's points, frame by frame, counted from ``origin``; else ``tokens`` tokens
    with a position each, below ``far``.  ``tail``: tokens that follow in the same tensors and are not rotated."""
    case = {"op": "rope", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim, "axes": text(axes),
            "grid": text(grid or []), "origin": text(origin or [0] * len(axes)),
            "tokens": math.prod(grid) if grid else tokens, "tail": tail, "theta": theta, "dtype": dtype,
            "token_major": token_major, "inverse": inverse, "pairs": pairs, "far": far}
    return {"name": name, **case} if name else case


def lora_case(name=None, *, op="lora", lengths, k, n, rank, adapters, pad=0, without=0):
    """``lengths``: rows of each request; ``pad``: rows behind the last one; ``without``: every so manyth request
    has no adapter (0: each has one)."""
    case = {"op": op, "lengths": text(lengths), "k": k, "n": n, "rank": rank, "adapters": adapters, "pad": pad,
            "without": without}
    return {"name": name, **case} if name else case


def kv8_case(name=None, *, heads, kv_heads, dim=128, queries, lengths, append=False):
    """``lengths``: tokens that each request has in the cache; ``append``: the queries' own keys and values are
    written behind them first."""
    case = {"op": "kv8", "heads": heads, "kv_heads": kv_heads, "dim": dim, "queries": queries,
            "lengths": text(lengths), "append": append}
    return {"name": name, **case} if name else case


def text(values):
    return " ".join(map(str, values))


def numbers(values):
    return [int(v) for v in values.split()]


def log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "lora", "lora_step", "kv8"])
    return draw_rope(rng) if op == "rope" else draw_kv8(rng) if op == "kv8" else draw_lora(rng, op)


def draw_rope(rng):
    dim = rng.choice([40, 64, 80, 96, 128, 128, 128, 160, 256])
    count = rng.choice([1, 2, 3, 3, 3, 4])
    parts = [2 * rng.randint(1, max(1, dim // (2 * count))) for _ in range(count)]
    dtype = rng.choice(["bf16", "bf16", "f32"])
    heads = rng.choice([1, 5, 8, 12, 16, 24, 40])
    kv_heads = rng.choice([h for h in (1, 4, 8, heads) if heads % h == 0])
    batch = rng.choice([1, 1, 2, 3])
    room = 10 ** 9 // ((heads + kv_heads) * batch * dim * (4 if dtype == "f32" else 2))  # bytes of the inputs
    tokens = log_uniform(rng, 1, max(1, min(120000, room)))
    grid = None
    if rng.random() < 0.5:
        grid, left = [], tokens
        for _ in range(count - 1):
            grid.append(log_uniform(rng, 1, max(1, round(left ** 0.5))))
            left = max(1, left // grid[-1])
        grid.append(left)
    return rope_case(batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, axes=parts, grid=grid, tokens=tokens,
                     origin=[rng.randint(0, 50) for _ in parts], tail=rng.choice([0, 0, 1, 77, 256]),
                     theta=rng.choice([256.0, 10000.0, 500000.0]), dtype=dtype, token_major=rng.random() < 0.4,
                     inverse=rng.random() < 0.4, pairs=rng.choice(["interleaved", "interleaved", "halves"]),
                     far=rng.choice([512, 40000, 1 << 20]))


def draw_lora(rng, op):
    width = lambda: 8 * log_uniform(rng, 16, 1728)  # noqa: E731
    k, n, rank = width(), width(), 8 * rng.randint(1, 16)
    most = min(80000, 75600 * 10240 // (k + n)) if op == "lora" else min(33000, 32760 * 10240 // (k + n))
    rows = log_uniform(rng, 1, max(1, most))
    requests = min(rows, log_uniform(rng, 1, 64))
    cuts = sorted(rng.randint(0, rows) for _ in range(requests - 1))  # a request may have no rows
    lengths = [b - a for a, b in zip([0] + cuts, cuts + [rows])]
    adapters = min(log_uniform(rng, 1, 32), max(1, 2 * 10 ** 7 // (rows * rank)), max(1, 10 ** 8 // ((k + n) * rank)))
    return lora_case(op=op, lengths=lengths, k=k, n=n, rank=rank, adapters=adapters, pad=rng.choice([0, 0, 5, 130]),
                     without=rng.choice([0, 0, 3]))


def draw_kv8(rng):
    kv_heads = rng.choice([1, 4, 8, 12, 24, 40])
    heads = kv_heads * rng.choice([1] if kv_heads > 8 else [1, 2, 5, 8])
    batch = rng.choice([1, 1, 2, 5, 16])
    queries = log_uniform(rng, 1, min(33000, 2 * 10 ** 6 // (batch * heads)))
    most = max(1, min(40000, 10 ** 9 // (heads * batch * queries)))  # scores of the plain form
    lengths = [rng.choice([0, 1, 64, 1000]) if rng.random() < 0.2 else log_uniform(rng, 1, most) for _ in range(batch)]
    return kv8_case(heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 128, 128]), queries=queries,
                    lengths=[min(n, most) for n in lengths], append=queries <= most and rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def unpacked(case):
    return {name: numbers(v) if name in ("axes", "grid", "origin", "lengths") else v for name, v in case.items()}


def prepare(case, seed):
    case = unpacked(case)
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"rope": prepare_rope, "kv8": prepare_kv8}.get(case["op"], prepare_lora)(case, g)


def prepare_rope(case, g):
    """Queries and keys [B, H, tokens, D] (a view of token-major storage where ``token_major``), after their norm:
    of about unit size."""
    dtype, count = DTYPES[case["dtype"]], case["tokens"]

    def one(heads):
        length = count + case["tail"]
        shape = (case["batch"], length, heads, case["dim"]) if case["token_major"] else \
            (case["batch"], heads, length, case["dim"])
        t = torch.randn(shape, generator=g, device=DEVICE, dtype=dtype)
        return (t.transpose(1, 2) if case["token_major"] else t)[:, :, :count]

    positions = None
    if not case["grid"]:
        positions = torch.randint(0, case["far"], (case["batch"], count, len(case["axes"])), generator=g,
                                  device=DEVICE, dtype=torch.int32)
    return {"case": case, "q": one(case["heads"]), "k": one(case["kv_heads"]), "positions": positions}


def prepare_lora(case, g):
    """x, y and dy as the projection's input, its output and the output's gradient; A as a fresh adapter's, B as a
    trained one's, so that the update is a few per cent of y; scale = alpha / rank."""
    lengths, k, n, rank, adapters = (case[name] for name in ("lengths", "k", "n", "rank", "adapters"))
    rows = sum(lengths) + case["pad"]
    randn = lambda *s: torch.randn(s, generator=g, device=DEVICE, dtype=torch.bfloat16)  # noqa: E731
    turn = torch.randperm(adapters, generator=g, device=DEVICE).int()
    slots = turn[torch.arange(len(lengths), device=DEVICE) % adapters]
    if case["without"]:
        slots[case["without"] - 1::case["without"]] = -1
    starts = [0]
    for length in lengths:
        starts.append(starts[-1] + length)
    state = {"case": case, "x": randn(rows, k), "y": randn(rows, n), "a": randn(adapters, rank, k) * k ** -0.5,
             "b": randn(adapters, n, rank) * 0.1,
             "scale": 0.5 + torch.rand(adapters, generator=g, device=DEVICE, dtype=torch.float32),
             "rows": torch.tensor(starts, device=DEVICE, dtype=torch.int32), "slots": slots}
    if case["op"] == "lora_step":
        state["dy"] = randn(rows, n)
    return state


PAGE = 64


def prepare_kv8(case, g):
    """Token-major queries (a projection's output) and a cache whose pages lie in no order, filled from unit keys and
    values; the pages' rows behind a request's last token hold what an earlier owner left."""
    batch, dim, heads = len(case["lengths"]), case["dim"], case["kv_heads"]
    added = case["queries"] if case["append"] else 0
    need = [-(-(n + added) // PAGE) for n in case["lengths"]]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEVICE).int()
    table = torch.full((batch, max(1, max(need))), -1, device=DEVICE, dtype=torch.int32)
    first = 0
    for i, n in enumerate(need):
        table[i, :n] = order[first:first + n]
        first += n
    randn = lambda *shape: torch.randn(shape, generator=g, device=DEVICE, dtype=torch.bfloat16)  # noqa: E731
    cache = []
    for _ in range(2):
        values = randn(pages, heads, PAGE, dim)
        scale = page_scale(values.abs().amax(dim=(2, 3)).float())
        cache += [(values / scale[..., None, None]).to(torch.float8_e4m3fn), scale]
    state = {"case": case, "q": randn(batch, case["queries"], case["heads"], dim).transpose(1, 2),
             "cache": (cache[0], cache[2], cache[1], cache[3]), "table": table,
             "starts": torch.tensor(case["lengths"], device=DEVICE, dtype=torch.int32),
             "lengths": torch.tensor([n + added for n in case["lengths"]], device=DEVICE, dtype=torch.int32)}
    if added:
        state["k"], state["v"] = (randn(batch, added, heads, dim).transpose(1, 2) for _ in range(2))
    return state


def page_scale(amax):
    """The smallest power of two (2^-100 at least) that brings amax to 448, e4m3's largest value, or below."""
    fraction, exponent = torch.frexp(amax)
    exponent = torch.where(fraction <= 0.875, exponent - 9, exponent - 8)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, exponent, -100).clamp_min(-100))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    return {"rope": run_rope, "lora": run_lora, "lora_step": run_lora_step, "kv8": run_kv8}[op](state)


def run_rope(s):
    case = s["case"]
    if own:
        from pasa_b200 import ops
        where = {"grid": case["grid"], "origin": case["origin"]} if case["grid"] else {"positions": s["positions"]}
        return ops.rope_axes(s["q"], s["k"], axes=case["axes"], theta=case["theta"], pairs=case["pairs"],
                             inverse=case["inverse"], **where)
    if case["grid"]:
        ranges = [torch.arange(o, o + m, device=DEVICE) for o, m in zip(case["origin"], case["grid"])]
        positions = torch.stack(torch.meshgrid(*ranges, indexing="ij"), dim=-1).flatten(0, -2)[None]
    else:
        positions = s["positions"]
    # angles in 64 bits: a far position loses its fraction of a turn in 32
    angle = torch.cat([positions[..., i, None].double() * case["theta"] ** (
        -torch.arange(0, d, 2, device=DEVICE, dtype=torch.float64) / d) for i, d in enumerate(case["axes"])], dim=-1)
    angle = (-angle if case["inverse"] else angle)[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    return rotate(s["q"], cos, sin, case), rotate(s["k"], cos, sin, case)


def rotate(x, cos, sin, case):
    """The pairs of x's first sum(axes) dimensions turned by their angles, the others kept."""
    turned = sum(case["axes"])
    f, rest = x[..., :turned].float(), x[..., turned:]
    if case["pairs"] == "halves":
        u, v = f.chunk(2, dim=-1)
        f = torch.cat((u * cos - v * sin, u * sin + v * cos), dim=-1)
    else:
        u, v = f[..., 0::2], f[..., 1::2]
        f = torch.stack((u * cos - v * sin, u * sin + v * cos), dim=-1).flatten(-2)
    return torch.cat((f.to(x.dtype), rest), dim=-1)


def adapter_of_rows(s):
    """[rows, adapters, 1]: whether the row's request has this adapter."""
    row = torch.arange(s["x"].shape[0], device=DEVICE)
    request = torch.searchsorted(s["rows"], row.int(), right=True) - 1
    inside = (request >= 0) & (request < s["slots"].numel())
    slot = torch.where(inside, s["slots"][request.clamp(0, s["slots"].numel() - 1)], -1)
    return slot[:, None, None] == torch.arange(s["a"].shape[0], device=DEVICE)[:, None]


def down(x, weight, mine, scale):
    """scale x weight^T for the row's own adapter, zero for the others: [rows, adapters * rank] in fp32."""
    adapters, rank, width = weight.shape
    h = (x.float() @ weight.float().reshape(adapters * rank, width).T).unflatten(1, (adapters, rank))
    return torch.where(mine, h * scale[:, None], 0.0).flatten(1)


def run_lora(s):
    if own:
        from pasa_b200 import ops
        return ops.lora_update(s["y"], s["x"], s["a"], s["b"], s["rows"], s["slots"], s["scale"])
    h = down(s["x"], s["a"], adapter_of_rows(s), s["scale"])
    return (s["y"].float() + h @ s["b"].float().transpose(1, 2).flatten(0, 1)).to(s["y"].dtype)


def run_lora_step(s):
    """The forward pass, then the gradients of x (the adapters' part), A and B from the output's."""
    if own:
        from pasa_b200 import ops
        out, h = ops.lora_update(s["y"], s["x"], s["a"], s["b"], s["rows"], s["slots"], s["scale"], return_h=True)
        return (out, *ops.lora_update_backward(s["dy"], s["x"], s["a"], s["b"], s["rows"], s["slots"], s["scale"],
                                               h=h))
    a, b, dy, dtype = s["a"], s["b"].transpose(1, 2), s["dy"], s["y"].dtype
    mine = adapter_of_rows(s)
    h = down(s["x"], a, mine, s["scale"])
    out = (s["y"].float() + h @ b.float().flatten(0, 1)).to(dtype)
    g = down(dy, b, mine, s["scale"])
    dx = (g @ a.float().flatten(0, 1)).to(dtype)
    da = (g.T @ s["x"].float()).reshape(a.shape).to(dtype)
    db = (h.T @ dy.float()).reshape(b.shape).transpose(1, 2).contiguous().to(dtype)
    return out, dx, da, db


def run_kv8(s):
    """The attention's output, after an append the cache too."""
    case = s["case"]
    if own:
        from pasa_b200 import ops
        if case["append"]:
            ops.kv8_write(s["cache"], s["k"], s["v"], s["table"], s["starts"])
        out = ops.kv8_attention(s["q"], s["cache"], s["table"], s["lengths"])
        return (out, *s["cache"]) if case["append"] else out
    k, v, k_scale, v_scale = s["cache"]
    if case["append"]:
        append(k, k_scale, s["k"], s["table"], s["starts"])
        append(v, v_scale, s["v"], s["table"], s["starts"])
    table, lengths = s["table"].clamp_min(0).long(), s["lengths"]
    keys, values = ((c[table].float() * scale[table][..., None, None]).transpose(1, 2).flatten(2, 3)
                    for c, scale in ((k, k_scale), (v, v_scale)))  # [B, kv heads, tokens, D]
    inside = torch.arange(keys.shape[2], device=DEVICE) < lengths[:, None, None, None]
    q = s["q"].float().unflatten(1, (case["kv_heads"], -1)).flatten(2, 3)  # a group's queries share their keys
    score = (q @ keys.transpose(2, 3)) * case["dim"] ** -0.5
    score.masked_fill_(~inside, -math.inf)
    top = score.amax(dim=3, keepdim=True)
    p = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()  # a request without tokens: all zero
    total = p.sum(dim=3, keepdim=True)
    out = (p @ values) / torch.where(total > 0, total, 1.0)
    out = out.to(s["q"].dtype).unflatten(2, (-1, case["queries"])).flatten(1, 2)
    return (out, *s["cache"]) if case["append"] else out


def append(cache, scales, new, table, starts):
    """Writes new [B, H, L, D] behind ``starts`` tokens.  A page's scale is its new tokens'; where it has earlier
    tokens it is the larger of theirs and that, and they are rounded to it."""
    batch, heads, count, dim = new.shape
    token = starts[:, None].long() + torch.arange(count, device=DEVICE)  # [B, L]
    block = token // PAGE - (starts[:, None] // PAGE)
    blocks = (PAGE - 1 + count + PAGE - 1) // PAGE
    amax = torch.zeros((batch, heads, blocks), device=DEVICE).scatter_reduce(
        2, block[:, None].expand(-1, heads, -1), new.abs().amax(dim=3).float(), "amax")
    scale = page_scale(amax)
    first, held = table.long().gather(1, (starts[:, None] // PAGE).long().clamp_max(table.shape[1] - 1)), starts % PAGE
    first = first[:, 0].clamp_min(0)
    old = scales[first]  # [B, H]
    scale[:, :, 0] = torch.where(held[:, None] > 0, torch.maximum(old, scale[:, :, 0]), scale[:, :, 0])
    earlier = cache[first].float() * (old / scale[:, :, 0])[..., None, None]
    keep = (torch.arange(PAGE, device=DEVICE) < held[:, None])[:, None, :, None]
    cache[first] = torch.where(keep, earlier, cache[first].float()).to(cache.dtype)
    page = table.long().gather(1, token // PAGE)
    mine = scale.gather(2, block[:, None].expand(-1, heads, -1))  # [B, H, L]
    head = torch.arange(heads, device=DEVICE)[None, :, None]
    cache.view(torch.uint8)[page[:, None], head, (token % PAGE)[:, None]] = \
        (new.float() / mine[..., None]).to(cache.dtype).view(torch.uint8)
    scales[page[:, None], head] = mine


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the results in 64 bits
# ---------------------------------------------------------------------------
def work(case):
    case = unpacked(case)
    if case["op"] == "rope":
        values = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        size = 4 if case["dtype"] == "f32" else 2
        where = 0 if case["grid"] else case["batch"] * case["tokens"] * len(case["axes"]) * 4
        return {"bytes": 2 * values * size + where, "flops": 3 * values}
    if case["op"] == "kv8":
        added = case["queries"] if case["append"] else 0
        kv = 2 * case["kv_heads"] * case["dim"]  # values of one token's key and value
        q = len(case["lengths"]) * case["queries"] * case["heads"] * case["dim"]
        tokens = [n + added for n in case["lengths"]]
        # q and its result; each cached token once, a page's scales; a new one read in 16 bits and written in 8
        moved = 4 * q + kv * sum(case["lengths"]) + 8 * case["kv_heads"] * sum(-(-n // PAGE) for n in tokens)
        return {"bytes": moved + 3 * kv * added * len(tokens),
                "flops": 4 * case["heads"] * case["dim"] * case["queries"] * sum(tokens)}
    k, n, rank, adapters = (case[name] for name in ("k", "n", "rank", "adapters"))
    with_adapter = [i for i, length in enumerate(case["lengths"])
                    if length and not (case["without"] and (i + 1) % case["without"] == 0)]
    used = sum(case["lengths"][i] for i in with_adapter)
    rows = sum(case["lengths"]) + case["pad"]
    weights = 2 * rank * (k + n)  # of one adapter
    moved = 2 * used * k + 4 * rows * n + weights * len({i % adapters for i in with_adapter})
    flops = 2 * used * rank * (k + n)
    if case["op"] == "lora_step":  # dy is read, the gradients of x and of all adapters are written
        moved, flops = moved + 2 * used * n + 2 * rows * k + weights * adapters, 3 * flops
    return {"bytes": moved, "flops": flops}


def exact(case, seed):
    state = prepare(case, seed)
    case = state["case"]
    return {"rope": exact_rope, "kv8": exact_kv8}.get(case["op"], exact_lora)(case, state)


def exact_rope(case, s):
    """Each pair as a complex number times e^(i angle)."""
    if case["grid"]:
        index = torch.arange(case["tokens"], device=DEVICE)
        coordinates = []
        for size, first in zip(reversed(case["grid"]), reversed(case["origin"])):
            coordinates.insert(0, index % size + first)
            index = index // size
        positions = torch.stack(coordinates, dim=1).expand(case["batch"], -1, -1)
    else:
        positions = s["positions"]
    turns = []
    for axis, size in enumerate(case["axes"]):
        for pair in range(size // 2):
            turns.append(positions[:, :, axis].double() / case["theta"] ** (2 * pair / size))
    angle = torch.stack(turns, dim=-1)
    factor = torch.polar(torch.ones_like(angle), -angle if case["inverse"] else angle)
    results = []
    for x in (s["q"], s["k"]):
        result = torch.empty(x.shape, device=DEVICE, dtype=torch.float64)
        turned = sum(case["axes"])
        result[..., turned:] = x[..., turned:].double()
        for head in range(x.shape[1]):
            part = x[:, head, :, :turned].double()
            if case["pairs"] == "halves":
                z = torch.complex(part[..., :turned // 2], part[..., turned // 2:]) * factor
                result[:, head, :, :turned // 2], result[:, head, :, turned // 2:turned] = z.real, z.imag
            else:
                z = torch.complex(part[..., ::2].contiguous(), part[..., 1::2].contiguous()) * factor
                result[:, head, :, 0:turned:2], result[:, head, :, 1:turned:2] = z.real, z.imag
        results.append(result)
    return tuple(results)


def exact_lora(case, s):
    """Request by request."""
    out = s["y"].double()
    da, db = torch.zeros_like(s["a"], dtype=torch.float64), torch.zeros_like(s["b"], dtype=torch.float64)
    dx = torch.zeros_like(s["x"], dtype=torch.float64) if case["op"] == "lora_step" else None
    first = 0
    for length, slot in zip(case["lengths"], s["slots"].tolist()):
        rows = slice(first, first + length)
        first += length
        if slot < 0 or not length:
            continue
        a, b, scale = s["a"][slot].double(), s["b"][slot].double(), s["scale"][slot].double()
        x = s["x"][rows].double()
        h = x.matmul(a.T)
        out[rows] += scale * h.matmul(b.T)
        if dx is not None:
            dy = s["dy"][rows].double()
            g = dy.matmul(b)
            dx[rows] = scale * g.matmul(a)
            da[slot] += scale * g.T.matmul(x)
            db[slot] += scale * dy.T.matmul(h)
    return out if dx is None else (out, dx, da, db)


def exact_kv8(case, s):
    """Request by request and head by head.  What is rounded to 8 bits has no value in 64."""
    k, v, k_scale, v_scale = s["cache"]
    out = torch.zeros(s["q"].shape, device=DEVICE, dtype=torch.float64)
    group = case["heads"] // case["kv_heads"]
    for i, count in enumerate(case["lengths"]):
        pages = s["table"][i].tolist()
        for head in range(case["kv_heads"]):
            rows = []
            for source, scale, new in ((k, k_scale, s.get("k")), (v, v_scale, s.get("v"))):
                used = pages[:-(-count // PAGE)]
                row = (source[used, head].double() * scale[used, head].double()[:, None, None]).flatten(0, 1)[:count]
                rows.append(row if new is None else held(row, scale[used, head], new[i, head], count))
            keys, values = rows
            for h in range(head * group, (head + 1) * group):
                if len(keys):
                    weights = torch.softmax(s["q"][i, h].double().matmul(keys.T) / math.sqrt(case["dim"]), dim=1)
                    out[i, h] = weights.matmul(values)
    return (out, None, None, None, None) if case["append"] else out


def held(row, scale, new, count):
    """The values that a head's pages hold after ``new`` has been written behind its ``count`` tokens."""
    row, new = row.clone(), new.double()
    first = count // PAGE * PAGE  # of the page that the new tokens begin in
    parts = [row[:first]]
    for at in range(first, count + len(new), PAGE):
        mine = new[max(0, at - count):at + PAGE - count]
        step = page_scale(mine.abs().max().float()).double()
        kept = row[at:] if at < count else row[:0]
        if len(kept):
            step = torch.maximum(step, scale[-1].double())
        parts += [(part / step).to(torch.float8_e4m3fn).double() * step for part in (kept.float(), mine.float())]
    return torch.cat(parts)
