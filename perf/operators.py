"""Measured cases of the attention operators that stand between the quantised
linears of a block: the norm and position rotation of queries and keys
(qk_norm_rope), appending keys and values to a paged cache (kv_append), and
attention of new tokens over that cache (paged_attention).

A case is a dict of plain values.  run() computes it in its plain form
(elementary torch operations in 32 bits) or, where `own` is set, through the
calls of turbocider_b200.cuda.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # ---- norm and rotation
        # one new token of one request: what a launch costs
        dict(name="rotate one token", op="rotate", tokens=1, q_heads=32, k_heads=8, dim=128, rotary=128, layout="half",
             axes=1, span=40000, stretch=1.0, norm=True, dtype="bf16"),
        # the image and text tokens of a 1024 x 1024 picture with guidance (2 x 4224), three position axes
        dict(name="rotate image tokens", op="rotate", tokens=8448, q_heads=30, k_heads=30, dim=128, rotary=128,
             layout="interleaved", axes=3, span=512, stretch=1.0, norm=True, dtype="f16"),
        # odd sizes: a part of each head rotated, positions scaled for a long context
        dict(name="rotate part of the head", op="rotate", tokens=1237, q_heads=20, k_heads=5, dim=96, rotary=64,
             layout="half", axes=1, span=120000, stretch=8.0, norm=False, dtype="bf16"),
        # ---- appending to the cache (queries normed and rotated in the same call)
        # one decode step of a served batch, some of its places unused
        dict(name="append a decode step", op="append", batch=64, new_low=1, new=1, past_low=1, past=700, idle=5,
             q_heads=32, k_heads=8, dim=128, rotary=128, layout="half", norm=True, page=16, dtype="bf16", mix=1),
        # prompts that arrive together
        dict(name="append prompts", op="append", batch=7, new_low=90, new=2600, past_low=0, past=300, idle=0,
             q_heads=32, k_heads=8, dim=128, rotary=128, layout="half", norm=True, page=64, dtype="bf16", mix=2),
        # keys and values only, small heads, no norm, interleaved pairs
        dict(name="append small heads", op="append", batch=19, new_low=0, new=67, past_low=0, past=1500, idle=1,
             q_heads=0, k_heads=6, dim=64, rotary=32, layout="interleaved", norm=False, page=32, dtype="f16", mix=3),
        # ---- attention over the cache
        # a single user's next token
        dict(name="attend one token", op="attend", batch=1, new_low=1, new=1, past_low=3000, past=3000, idle=0,
             q_heads=32, k_heads=8, dim=128, page=16, causal=True, window=0, lse=False, dtype="bf16", mix=4),
        # a served batch of very different lengths, some of its places unused
        dict(name="attend a decode step", op="attend", batch=96, new_low=1, new=1, past_low=1, past=8191, idle=4,
             q_heads=32, k_heads=8, dim=128, page=16, causal=True, window=0, lse=True, dtype="bf16", mix=5),
        # a few drafted tokens for each request, verified in one call, sliding window
        dict(name="attend drafted tokens", op="attend", batch=23, new_low=1, new=7, past_low=100, past=6000, idle=0,
             q_heads=20, k_heads=5, dim=64, page=32, causal=True, window=2048, lse=False, dtype="f16", mix=6),
        # the next part of one long prompt
        dict(name="attend a chunk", op="attend", batch=1, new_low=1536, new=1536, past_low=30001, past=30001, idle=0,
             q_heads=32, k_heads=8, dim=128, page=16, causal=True, window=0, lse=False, dtype="bf16", mix=7),
        # whole prompts of different lengths
        dict(name="attend prompts", op="attend", batch=5, new_low=150, new=4100, past_low=0, past=0, idle=0,
             q_heads=32, k_heads=8, dim=128, page=64, causal=True, window=0, lse=True, dtype="bf16", mix=8),
        # image and text tokens that all see one another, with guidance
        dict(name="attend image tokens", op="attend", batch=2, new_low=4224, new=4224, past_low=0, past=0, idle=0,
             q_heads=30, k_heads=30, dim=128, page=128, causal=False, window=0, lse=False, dtype="f16", mix=9),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotate", "append", "attend", "attend"])
    dtype = rng.choice(["bf16", "f16"])
    dim = rng.choice([64, 80, 96, 128, 128])
    k_heads = rng.randint(1, 10)
    q_heads = k_heads * rng.choice([1, 2, 3, 4, 5, 8])
    layout = rng.choice(["half", "interleaved"])
    rotary = rng.choice([r for r in (16, 32, 64, 80, 96, 128) if r <= dim])
    if op == "rotate":
        axes = rng.choice([1, 1, 2, 3]) if rotary >= 48 else 1
        return dict(op=op, tokens=_log(rng, 1, 8448), q_heads=min(q_heads, 48), k_heads=k_heads, dim=dim, rotary=rotary,
                    layout=layout, axes=axes, span=_log(rng, 64, 120000) if axes == 1 else rng.randint(64, 1024),
                    stretch=rng.choice([1.0, 1.0, 4.0, 8.0]), norm=rng.random() < 0.7, dtype=dtype)
    page = rng.choice([8, 16, 32, 64, 128, 256])
    if op == "append":
        batch = _log(rng, 1, 128)
        new = _log(rng, 1, max(1, 9000 // batch))
        return dict(op=op, batch=batch, new_low=rng.randint(0, new), new=new, past_low=0,
                    past=_log(rng, 1, max(2, min(4000, 50000 // batch))), idle=rng.randint(0, batch // 8),
                    q_heads=rng.choice([0, min(q_heads, 48)]), k_heads=k_heads, dim=dim, rotary=rotary, layout=layout,
                    norm=rng.random() < 0.7, page=page, dtype=dtype, mix=rng.randint(10, 10 ** 6))
    # attention: single tokens, a few, or whole chunks, with a bounded number of scores in the plain form
    form = rng.choice(["decode", "few", "chunk", "all"])
    q_heads = min(q_heads, 32 // k_heads * k_heads)
    if form == "decode":
        batch, new = _log(rng, 1, 128), 1
        past = _log(rng, 1, min(30000, 700000 // batch))
    elif form == "few":
        batch, new = _log(rng, 1, 32), rng.randint(2, 40)
        past = _log(rng, 1, min(30000, 200000 // batch))
    else:
        batch, new = rng.choice([1, 1, 2, 3, 5]), _log(rng, 41, 4100)
        past = _log(rng, 1, 12000) if form == "chunk" else 0
    most = 1.3e9 / (batch * q_heads * new)      # the plain form holds batch x heads x new x (past + new) scores
    past = max(0, min(past, int(most) - new))
    return dict(op=op, batch=batch, new_low=rng.randint(0, new) if form != "decode" else 1, new=new,
                past_low=rng.randint(0, past), past=past, idle=rng.randint(0, batch // 8), q_heads=q_heads,
                k_heads=k_heads, dim=dim, page=page, causal=form != "all" or rng.random() < 0.5,
                window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), lse=rng.random() < 0.3, dtype=dtype,
                mix=rng.randint(10, 10 ** 6))


# ------------------------------------------------------------ lengths of a batch
def _batch(case):
    """[(new tokens, cached tokens with the new ones)] of the requests: the
    listed bounds occur, the rest is spread between them; `idle` places of the
    batch hold a token and no cache (a padded place of a fixed-size batch)."""
    rng, b = random.Random(case["mix"]), case["batch"]
    out = []
    for i in range(b):
        new = case["new"] if i == 0 else rng.randint(case["new_low"], case["new"])
        past = case["past"] if i == 0 else case["past_low"] if i == 1 else rng.randint(case["past_low"], case["past"])
        out.append((new, new + past))
    for i in range(case["idle"]):
        out[b - 1 - i] = (min(1, case["new"]), 0)
    rng.shuffle(out)
    return out


def _pages(case):
    return [-(-n // case["page"]) for _, n in _batch(case)]


# ------------------------------------------------------------ rotation
def _frequencies(case):
    """Radians a position step of each pair, and the amplitude.  With
    stretch > 1 the slow pairs are interpolated by it, the fast ones kept and
    those between blended (a linear ramp over the turns made in a context of
    8192), and the amplitude grows with log(stretch)."""
    half, theta, stretch = case["rotary"] // 2, 1e6 if case.get("axes", 1) == 1 else 256.0, case.get("stretch", 1.0)
    axes = case.get("axes", 1)
    sections = [half // axes + (1 if a < half % axes else 0) for a in range(axes)]
    freq, axis = [], []
    for a, n in enumerate(sections):
        freq += [theta ** (-i / n) for i in range(n)]
        axis += [a] * n
    if stretch != 1.0:
        turns = [f * 8192 / (2 * math.pi) for f in freq]
        keep = [min(1.0, max(0.0, (t - 1.0) / (32.0 - 1.0))) for t in turns]
        freq = [f * (k + (1 - k) / stretch) for f, k in zip(freq, keep)]
    return freq, axis, sections, 1.0 if stretch == 1.0 else 0.1 * math.log(stretch) + 1.0


def _rotation(case, gen, tokens, span):
    freq, axis, sections, amplitude = _frequencies(case)
    freq = torch.tensor(freq, dtype=torch.float64, device="cuda")
    s = dict(freq=freq, sections=sections, amplitude=amplitude, layout=case["layout"], rotary=case["rotary"],
             axis=torch.tensor(axis, device="cuda"), pair=torch.arange(len(axis), device="cuda"))
    if tokens is not None:
        s["positions"] = torch.randint(0, span, (tokens, len(sections)), dtype=torch.int32, device="cuda", generator=gen)
    # the plain form's table: cos and sin of every position
    angle = torch.arange(span, dtype=torch.float64, device="cuda")[:, None] * freq
    s["table"] = torch.stack((angle.cos() * amplitude, angle.sin() * amplitude)).float()
    return s


# ------------------------------------------------------------ inputs
def _normal(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen) * scale).to(DTYPES[dtype])


def _norm_weights(s, case, gen):
    for name in ("q", "k"):
        s[name + "_weight"] = None
        if case["norm"]:
            s[name + "_weight"] = 1.0 + 0.2 * torch.randn(case["dim"], device="cuda", generator=gen)


def _ragged(s, case, gen):
    """Offsets, lengths and the page table of a batch; pages in random order."""
    lens, pages = _batch(case), _pages(case)
    offsets = [0]
    for n, _ in lens:
        offsets.append(offsets[-1] + n)
    total, widest = sum(pages) + 3, max(max(pages), 1)
    order = torch.randperm(total, device="cuda", generator=gen).to(torch.int32)
    width = torch.tensor(pages, device="cuda")
    place = torch.arange(widest, device="cuda")[None] < width[:, None]
    table = torch.full((len(pages), widest), -1, dtype=torch.int32, device="cuda")
    table[place] = order[:sum(pages)]
    s.update(offsets=torch.tensor(offsets, dtype=torch.int32, device="cuda"), table_of_pages=table,
             lengths=torch.tensor([n for _, n in lens], dtype=torch.int32, device="cuda"), tokens=offsets[-1],
             max_new=max(n for n, _ in lens), max_length=max(n for _, n in lens), page=case["page"])
    shape = (total, case["k_heads"], case["page"], case["dim"])
    s["k_cache"], s["v_cache"] = _normal(gen, shape, case["dtype"]), _normal(gen, shape, case["dtype"])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 17)
    dim, hq, hk = case["dim"], case["q_heads"], case["k_heads"]
    s = dict(case=case)
    if case["op"] == "rotate":
        # what a projection to queries, keys and values wrote: one row of all heads for each token
        row = _normal(gen, (case["tokens"], (hq + 2 * hk) * dim), case["dtype"], 1.7)
        s["q"] = row[:, :hq * dim].view(-1, hq, dim)
        s["k"] = row[:, hq * dim:(hq + hk) * dim].view(-1, hk, dim)
        _norm_weights(s, case, gen)
        s["rotation"] = _rotation(case, gen, case["tokens"], case["span"])
    elif case["op"] == "append":
        _ragged(s, case, gen)
        row = _normal(gen, (s["tokens"], (hq + 2 * hk) * dim), case["dtype"], 1.7)
        s["q"] = row[:, :hq * dim].view(-1, hq, dim) if hq else None
        s["k"] = row[:, hq * dim:(hq + hk) * dim].view(-1, hk, dim)
        s["v"] = row[:, (hq + hk) * dim:].view(-1, hk, dim)
        _norm_weights(s, case, gen)
        s["rotation"] = _rotation(case, gen, None, max(s["max_length"], 1))
    else:
        _ragged(s, case, gen)
        s["q"] = _normal(gen, (s["tokens"], hq, dim), case["dtype"], 1.5)
        s["scale"] = dim ** -0.5
    return s


# ------------------------------------------------------------ plain forms
def _plain_norm_rotate(x, weight, norm, r, index):
    """x [tokens, heads, dim]; index [tokens, pairs]: each pair's position."""
    y = x.float()
    if norm:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight
    n, half = r["rotary"], r["rotary"] // 2
    cos, sin = r["table"][:, index, r["pair"]][:, :, None]
    if r["layout"] == "half":
        a, b = y[..., :half], y[..., half:n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    else:
        a, b = y[..., 0:n:2], y[..., 1:n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    return torch.cat((turned, y[..., n:]), -1).to(x.dtype)


def _plain_places(s):
    """Request and position in its cache of each new token."""
    token = torch.arange(s["tokens"], device="cuda")
    request = torch.searchsorted(s["offsets"][1:].long(), token, right=True)
    new = s["offsets"].diff().long()
    return request, s["lengths"].long()[request] - new[request] + token - s["offsets"].long()[request]


def _plain_append(s):
    r, norm = s["rotation"], s["case"]["norm"]
    request, position = _plain_places(s)
    index = position.clamp(min=0)[:, None].expand(-1, r["pair"].numel())
    k = _plain_norm_rotate(s["k"], s["k_weight"], norm, r, index)
    live = position >= 0
    page = s["table_of_pages"][request, position.clamp(min=0) // s["page"]].long()[live]
    row = (position % s["page"])[live]
    s["k_cache"][page, :, row] = k[live]
    s["v_cache"][page, :, row] = s["v"][live]
    out = [s["k_cache"], s["v_cache"]]
    if s["q"] is not None:
        out.append(_plain_norm_rotate(s["q"], s["q_weight"], norm, r, index))
    return out


def _plain_attend(s):
    case, q = s["case"], s["q"]
    b, hk, dim = case["batch"], case["k_heads"], case["dim"]
    group, width = case["q_heads"] // hk, s["table_of_pages"].shape[1] * s["page"]
    new, length, offsets = s["offsets"].diff().long(), s["lengths"].long(), s["offsets"].long()
    # keys and values of each request side by side, zero past its length
    pages = s["table_of_pages"].clamp(min=0).long()
    at = torch.arange(width, device="cuda")
    held = (at[None] < length[:, None])[:, None, :, None]
    k, v = (torch.where(held, c[pages].permute(0, 2, 1, 3, 4).reshape(b, hk, width, dim), 0.0).float()
            for c in (s["k_cache"], s["v_cache"]))
    # queries padded to the largest number of new tokens
    i = torch.arange(s["max_new"], device="cuda")
    real = i[None] < new[:, None]
    rows = (offsets[:-1, None] + i[None]).clamp(max=max(s["tokens"] - 1, 0))
    padded = q[rows].float().view(b, -1, hk, group, dim).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, dim)
    score = (padded @ k.transpose(-1, -2)).view(b, hk, group, -1, width).mul_(s["scale"])
    place = (length - new)[:, None] + i[None]
    seen = (at < length[:, None, None]) & real[:, :, None]
    if case["causal"]:
        seen = seen & (at <= place[:, :, None])
    if case["window"]:
        seen = seen & (at > place[:, :, None] - case["window"])
        if not case["causal"]:
            seen = seen & (at < place[:, :, None] + case["window"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score = score.sub_(top.clamp(min=-1e30)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score.view(b, hk, -1, width) @ v).view(b, hk, group, -1, dim) / total.clamp(min=1e-30)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, -1, hk * group, dim)[real].to(q.dtype)
    if not case["lse"]:
        return [out]
    return [out, (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(b, -1, hk * group)[real]]


# ------------------------------------------------------------ the framework's calls
_contexts = {}


def _context(tcc):
    device = torch.cuda.current_device()
    if device not in _contexts:
        _contexts[device] = tcc.Context(device)
    return _contexts[device]


def _cache(tcc, s):
    """The cache's description, which a program makes once beside its buffers."""
    if "cache" not in s:
        s["cache"] = tcc.PagedCache(s["k_cache"], s["v_cache"])
    return s["cache"]


def _own(s):
    from turbocider_b200 import cuda as tcc
    ctx, case = _context(tcc), s["case"]
    if case["op"] == "attend":
        step = tcc.PagedBatch(s["offsets"], s["lengths"], s["table_of_pages"], s["max_new"], s["max_length"])
        out = tcc.paged_attention(ctx, _cache(tcc, s), step, s["q"], scale=s["scale"], causal=case["causal"],
                                  window=case["window"], return_lse=case["lse"])
        return list(out) if case["lse"] else [out]
    r, eps = s["rotation"], EPS if case["norm"] else None
    rope = tcc.Rope(r["freq"], r.get("positions"), layout=r["layout"], sections=r["sections"], amplitude=r["amplitude"])
    if case["op"] == "rotate":
        return list(tcc.qk_norm_rope(ctx, s["q"], s["k"], rope, q_weight=s["q_weight"], k_weight=s["k_weight"], eps=eps))
    step = tcc.PagedBatch(s["offsets"], s["lengths"], s["table_of_pages"], s["max_new"], s["max_length"])
    q = tcc.kv_append(ctx, _cache(tcc, s), step, s["k"], s["v"], rope, q=s["q"], q_weight=s["q_weight"],
                      k_weight=s["k_weight"], eps=eps)
    return [s["k_cache"], s["v_cache"]] + ([q] if q is not None else [])


def run(s):
    if own:
        return _own(s)
    case = s["case"]
    if case["op"] == "attend":
        return _plain_attend(s)
    if case["op"] == "append":
        return _plain_append(s)
    r = s["rotation"]
    index = r["positions"][:, r["axis"]].long()
    return [_plain_norm_rotate(s[x], s[x + "_weight"], case["norm"], r, index) for x in ("q", "k")]


# ------------------------------------------------------------ what a pass cannot do without
def _pairs(case, new, length):
    """(query, key) pairs that attend, and the keys that any query attends, of one request."""
    first, window, pairs, low, high = length - new, case["window"], 0, length, 0
    if not case["causal"] and not window:
        return new * length, length if new else 0
    for i in range(new):
        place = first + i
        last = min(length, place + 1) if case["causal"] else min(length, place + window)
        begin = max(0, place - window + 1) if window else 0
        if last > begin:
            pairs += last - begin
            low, high = min(low, begin), max(high, last)
    return pairs, max(0, high - low)


def work(case):
    hq, hk, dim = case["q_heads"], case["k_heads"], case["dim"]
    if case["op"] == "rotate":
        elements = case["tokens"] * (hq + hk) * dim
        return {"bytes": 4 * elements + 4 * case["tokens"] * case["axes"], "flops": 9 * elements}
    lens = _batch(case)
    tokens = sum(n for n, _ in lens)
    if case["op"] == "append":
        live = sum(n for n, length in lens if length)
        elements = tokens * hq * dim + 2 * live * hk * dim
        return {"bytes": 4 * elements, "flops": 9 * (tokens * hq + live * hk) * dim}
    pairs, keys = map(sum, zip(*(_pairs(case, n, length) for n, length in lens)))
    nbytes = 4 * tokens * hq * dim + 4 * keys * hk * dim + 4 * sum(_pages(case)) + (4 * tokens * hq if case["lse"] else 0)
    return {"bytes": nbytes, "flops": 4 * pairs * hq * dim}


# ------------------------------------------------------------ the definition in 64 bits
def _exact_heads(x, weight, norm, freq, amplitude, layout, where):
    """where [tokens, pairs]: positions.  Rotation as a product of complex numbers."""
    y = x.double()
    if norm:
        y = y / ((y ** 2).sum(-1, keepdim=True) / y.shape[-1] + EPS).sqrt() * weight.double()
    n = 2 * freq.numel()
    first = torch.arange(n // 2, device=y.device) * (1 if layout == "half" else 2)
    second = first + (n // 2 if layout == "half" else 1)
    turn = torch.polar(torch.full_like(freq, amplitude).expand(where.shape), where.double() * freq)
    z = torch.complex(y[..., first], y[..., second]) * turn[:, None]
    y[..., first], y[..., second] = z.real.clone(), z.imag.clone()
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        freq, axis, _, amplitude = _frequencies(case)
        freq = torch.tensor(freq, dtype=torch.float64, device="cuda")
        where = torch.stack([s["rotation"]["positions"][:, a] for a in axis], 1)
        return [_exact_heads(s[x], s[x + "_weight"], case["norm"], freq, amplitude, case["layout"], where) for x in ("q", "k")]
    lens, table = _batch(case), s["table_of_pages"].tolist()
    if case["op"] == "append":
        freq, _, _, amplitude = _frequencies(case)
        freq = torch.tensor(freq, dtype=torch.float64, device="cuda")
        place = torch.tensor([length - new + i for new, length in lens for i in range(new)], device="cuda")
        where = place.clamp(min=0)[:, None].expand(-1, freq.numel())
        k = _exact_heads(s["k"], s["k_weight"], case["norm"], freq, amplitude, case["layout"], where)
        caches, t = [s["k_cache"].double(), s["v_cache"].double()], 0
        for b, (new, length) in enumerate(lens):
            if length:
                spots = [divmod(p, case["page"]) for p in range(length - new, length)]
                page = torch.tensor([table[b][p] for p, _ in spots], dtype=torch.long, device="cuda")
                row = torch.tensor([r for _, r in spots], dtype=torch.long, device="cuda")
                caches[0][page, :, row], caches[1][page, :, row] = k[t:t + new], s["v"][t:t + new].double()
            t += new
        if s["q"] is not None:
            caches.append(_exact_heads(s["q"], s["q_weight"], case["norm"], freq, amplitude, case["layout"], where))
        return caches
    group, out, lse = case["q_heads"] // case["k_heads"], [], []
    t = 0
    for b, (new, length) in enumerate(lens):
        q, t = s["q"][t:t + new].double(), t + new
        y = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        z = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        if new and length:
            pages = torch.tensor(table[b][:-(-length // case["page"])], dtype=torch.long, device="cuda")
            distance = (torch.arange(length, device="cuda")[None] - torch.arange(length - new, length, device="cuda")[:, None])
            hidden = torch.zeros_like(distance, dtype=torch.bool)
            if case["causal"]:
                hidden |= distance > 0
            if case["window"]:
                hidden |= distance.abs() >= case["window"]
            for h in range(case["q_heads"]):
                k, v = (c[pages, h // group].reshape(-1, case["dim"])[:length].double() for c in (s["k_cache"], s["v_cache"]))
                score = (q[:, h] @ k.T * s["scale"]).masked_fill(hidden, -math.inf)
                z[:, h] = torch.logsumexp(score, -1)
                y[:, h] = torch.softmax(score, -1) @ v
        out.append(y)
        lse.append(z)
    return [torch.cat(out), torch.cat(lse)] if case["lse"] else [torch.cat(out)]
