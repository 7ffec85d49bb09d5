"""Cases that measure the paged key-value cache and its operators.

The operators: rotary positions (and their gradient), appending rotated keys
and values to a paged cache, the cache's page operations (extending, forking,
freeing, compacting and copying pages), and the attention of one new token
over the paged cache.  ``run`` computes each of them either in a plain form,
with elementary torch operations in 32 bits, or (``own``) with the calls that
a user makes of ``jasper_b200.paged``.

The cache: keys and values are [layers, pages, page_size, kv_heads, head_dim]
tensors whose strides say how they lie in memory ("token": as written,
"head": each page keeps a head's tokens together); ``table`` [rows, max_pages]
int32 gives a row's pages (-1 for none), ``lengths`` [rows] int32 its tokens,
``refs`` [pages] int32 how many rows hold a page (0: free).
"""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


# ── cases ────────────────────────────────────────────────────────────────

def listed():
    return [
        # One conversation of a thousand tokens: the call whose latency is a token's latency.
        attention("attend_one", batch=1, longest=1000, shortest=1000, q_heads=32, kv_heads=8, dim=128,
                  page_size=16, dtype="float16"),
        # A full serving batch whose conversations have every length up to 8 k tokens.
        attention("attend_ragged", batch=64, longest=8191, shortest=1, q_heads=32, kv_heads=8, dim=128,
                  page_size=16, dtype="bfloat16"),
        # Two very long documents: the cache's length is all the parallelism there is.
        attention("attend_long", batch=2, longest=400_001, shortest=333_337, q_heads=64, kv_heads=8, dim=128,
                  page_size=64, dtype="float16", layout="head"),
        # A graph search's answer as page table: a query batch attends to the pages of its ten nearest
        # passages; unfilled answers are -1, and passages end inside their pages.
        attention("attend_retrieved", batch=1000, longest=320, shortest=320, q_heads=8, kv_heads=8, dim=128,
                  page_size=32, dtype="float16", retrieved=True, pages=16384),
        # Queries and keys of a prompt chunk, views of one projection's output, far into a scaled context.
        rotary("rotary_prompt", tokens=8192, heads=40, dim=128, rot=128, layout="half", dtype="bfloat16",
               scaling="yarn", factor=8.0, trained=16384, offset=100_000),
        # The gradient of a training batch's rotary positions, on part of each head, in 32 bits.
        rotary("rotary_gradient", tokens=4099, heads=12, dim=80, rot=32, layout="interleaved", dtype="float32",
               scaling="linear", factor=4.0, trained=2048, offset=0, gradient=True),
        # One new token of each conversation of a batch: queries rotated, keys and values into the cache.
        append("append_token", tokens=64, q_heads=32, kv_heads=8, dim=128, rot=128, layout="half",
               page_size=16, dtype="float16", prompt=False, offset=4000),
        # A prompt chunk of 16 k tokens into the cache.
        append("append_prompt", tokens=16_384, q_heads=32, kv_heads=8, dim=128, rot=64, layout="interleaved",
               page_size=16, dtype="bfloat16", prompt=True, offset=0),
        # Continuous batching: 200 finished conversations leave, and as many prompts take their pages.
        pages("pages_turnover", "turnover", rows=256, named=200, n_pages=65_536, page_size=16, layers=1, kv_heads=1,
              dim=8, mean=3000),
        # A beam step: the losing beams leave, the winners fork, and part-filled pages are copied in every layer.
        pages("pages_fork", "fork", rows=512, named=256, n_pages=2048, page_size=16, layers=16, kv_heads=8, dim=128,
              mean=50),
        # After many conversations have left: live pages move together, so that the pool's end is free.
        pages("pages_compact", "compact", rows=64, named=0, n_pages=2048, page_size=16, layers=16, kv_heads=8,
              dim=128, mean=300, layout="head"),
        # Snapshots of some pages, to be changed apart from their originals.
        pages("pages_copy", "copy", rows=8, named=301, n_pages=1024, page_size=32, layers=8, kv_heads=8, dim=128,
              mean=300),
    ]


def attention(name=None, *, batch, longest, shortest, q_heads, kv_heads, dim, page_size, dtype, layout="token",
              retrieved=False, pages=0, window=0):
    case = dict(op="attend", batch=batch, longest=longest, shortest=shortest, q_heads=q_heads, kv_heads=kv_heads,
                dim=dim, page_size=page_size, dtype=dtype, layout=layout, retrieved=retrieved, pages=pages,
                window=window)
    return dict(case, name=name) if name else case


def rotary(name=None, *, tokens, heads, dim, rot, layout, dtype, scaling, factor, trained, offset, gradient=False):
    case = dict(op="rotary", tokens=tokens, heads=heads, dim=dim, rot=rot, layout=layout, dtype=dtype,
                scaling=scaling, factor=factor, trained=trained, offset=offset, gradient=gradient)
    return dict(case, name=name) if name else case


def append(name=None, *, tokens, q_heads, kv_heads, dim, rot, layout, page_size, dtype, prompt, offset):
    case = dict(op="append", tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, dim=dim, rot=rot, layout=layout,
                page_size=page_size, dtype=dtype, prompt=prompt, offset=offset)
    return dict(case, name=name) if name else case


def pages(name, kind, *, rows, named, n_pages, page_size, layers, kv_heads, dim, mean, layout="token"):
    case = dict(op="pages", kind=kind, rows=rows, named=named, n_pages=n_pages, page_size=page_size, layers=layers,
                kv_heads=kv_heads, dim=dim, mean=mean, layout=layout)
    return dict(case, name=name) if name else case


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["attend", "attend", "attend", "rotary", "append", "pages", "pages"])
    if op == "attend":
        dim, kv_heads = rng.choice([64, 80, 96, 128, 128, 256]), rng.choice([1, 2, 4, 8])
        group, page_size = rng.choice([1, 2, 3, 4, 6, 8, 16]), rng.choice([8, 16, 16, 32, 64, 100])
        dtype, layout = rng.choice(["float16", "bfloat16"]), rng.choice(["token", "head"])
        if rng.random() < 0.25:
            k = rng.randint(2, 24)
            batch = spread(2, 600)
            return attention(batch=batch, longest=k * page_size, shortest=k * page_size, q_heads=group * kv_heads,
                             kv_heads=kv_heads, dim=dim, page_size=page_size, dtype=dtype, layout=layout,
                             retrieved=True, pages=spread(k + 1, 4000))
        batch = spread(1, 200)
        longest = spread(1, min(300_000, 300_000_000 // (batch * kv_heads * dim)))
        shortest = longest if rng.random() < 0.3 else rng.randint(0, longest)
        window = rng.choice([0, 0, rng.randint(1, longest)])
        return attention(batch=batch, longest=longest, shortest=shortest, q_heads=group * kv_heads, kv_heads=kv_heads,
                         dim=dim, page_size=page_size, dtype=dtype, layout=layout, window=window)
    if op in ("rotary", "append"):
        dim = rng.choice([64, 80, 96, 128, 256])
        rot, layout = rng.choice([dim, dim, dim // 2, 16]), rng.choice(["half", "interleaved"])
        if op == "rotary":
            scaling = rng.choice(["none", "linear", "ntk", "yarn"])
            return rotary(tokens=spread(1, 8000), heads=rng.randint(1, 40), dim=dim, rot=rot, layout=layout,
                          dtype=rng.choice(["float16", "bfloat16", "float32"]), scaling=scaling,
                          factor=rng.choice([2.0, 4.0, 8.0]), trained=rng.choice([2048, 4096, 32_768]),
                          offset=rng.choice([0, spread(1, 1_000_000)]), gradient=rng.random() < 0.5)
        kv_heads, prompt = rng.choice([1, 2, 4, 8]), rng.random() < 0.5
        return append(tokens=spread(100, 16_000) if prompt else spread(1, 500), q_heads=kv_heads * rng.choice([1, 2, 4]),
                      kv_heads=kv_heads, dim=dim, rot=rot, layout=layout, page_size=rng.choice([8, 16, 32, 64, 100]),
                      dtype=rng.choice(["float16", "bfloat16"]), prompt=prompt, offset=0 if prompt else spread(1, 8000))
    kind, page_size = rng.choice(["turnover", "fork", "compact", "copy"]), rng.choice([8, 16, 32, 50])
    layout, kv_heads, dim = rng.choice(["token", "head"]), rng.choice([1, 2, 8]), rng.choice([64, 80, 128])
    if kind == "turnover":
        rows = spread(2, 400)
        mean = spread(20, 3000)
        return pages(None, kind, rows=rows, named=rng.randint(1, rows), page_size=page_size, layers=1, kv_heads=1, dim=8,
                     n_pages=int(rows * (mean * 2 / page_size + 2)) + rng.randint(0, 9), mean=mean)
    rows, layers, n_pages = 2 * spread(1, 100), rng.randint(1, 12), spread(500, 2000)
    return pages(None, kind, rows=rows, named=rows // 2 if kind == "fork" else rng.randint(1, n_pages // 3),
                 page_size=page_size, layers=layers, kv_heads=kv_heads, dim=dim, n_pages=n_pages,
                 mean=max(1, n_pages * page_size // (8 * rows)), layout=layout)


# ── inputs ───────────────────────────────────────────────────────────────

def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    return {"attend": prepare_attend, "rotary": prepare_rotary, "append": prepare_append,
            "pages": prepare_pages}[case["op"]](case, g)


def normal(g, *shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device=DEVICE).normal_(generator=g)


def permutation(g, n):
    return torch.randperm(n, generator=g, device=DEVICE)


def store(g, layers, n_pages, page_size, heads, dim, dtype, layout):
    """Keys or values of a pool of pages, [layers, pages, tokens, heads, dim]."""
    if layout == "token":
        return normal(g, layers, n_pages, page_size, heads, dim, dtype=dtype)
    return normal(g, layers, n_pages, heads, page_size, dim, dtype=dtype).transpose(2, 3)


def held(state):
    """The framework's handle on a state's cache, which a program keeps for as long as the cache lives."""
    if own:
        from jasper_b200 import paged
        state["cache"] = paged.PagedCache(state["k"], state["v"], state["table"], state["lengths"], state["refs"])
    return state


def spread_lengths(case):
    """The batch's lengths, from the shortest to the longest in even steps."""
    n, low, high = case["batch"], case["shortest"], case["longest"]
    return [high - (high - low) * i // max(1, n - 1) for i in range(n)]


def prepare_attend(case, g):
    dtype, ps, batch = DTYPES[case["dtype"]], case["page_size"], case["batch"]
    dims = (ps, case["kv_heads"], case["dim"])
    width = -(-case["longest"] // ps)
    if case["retrieved"]:
        n_pages = case["pages"]
        table = torch.randint(0, n_pages, (batch, width), generator=g, device=DEVICE)
        table[torch.rand(batch, width, generator=g, device=DEVICE) < 0.04] = -1
        lengths = torch.full((batch,), width * ps, device=DEVICE)
        fill = torch.randint(ps // 2, ps + 1, (batch, width, 1), generator=g, device=DEVICE)
        mask = (torch.arange(ps, device=DEVICE) < fill).view(batch, width * ps)
        refs = torch.bincount(table[table >= 0].view(-1), minlength=n_pages)
    else:
        lengths = torch.tensor(spread_lengths(case), device=DEVICE)[permutation(g, batch)]
        held_pages = (lengths + ps - 1) // ps
        inside = torch.arange(width, device=DEVICE) < held_pages[:, None]
        # every page in use has one holder, and a conversation's pages lie all over the pool
        total = sum(-(-n // ps) for n in spread_lengths(case))
        n_pages = total + total // 16 + 1
        order = permutation(g, n_pages)
        rank = (inside.view(-1).cumsum(0) - 1).clamp_min(0)
        table = torch.where(inside, order[rank].view(batch, width), -1)
        refs = torch.zeros(n_pages, dtype=torch.int64, device=DEVICE)
        refs[order[:total]] = 1
        mask = None
    k = store(g, 1, n_pages, *dims, dtype, case["layout"])
    v = store(g, 1, n_pages, *dims, dtype, case["layout"])
    v += normal(g, case["kv_heads"], case["dim"], dtype=dtype)  # values have a direction of their own in each head
    q = (normal(g, batch, case["q_heads"], case["dim"]) * 2).to(dtype)
    return held({"case": case, "q": q, "k": k, "v": v, "table": table.int(), "lengths": lengths.int(),
                 "refs": refs.int(), "mask": mask, "scale": case["dim"] ** -0.5})


def frequencies(rot, scaling="none", factor=1.0, trained=0, base=10000.0):
    """Radians a position for each pair, and the factor on the rotated vectors.  "linear" divides positions;
    "ntk" raises the base so that the slowest pair slows by the factor; "yarn" divides the slow pairs'
    frequencies only, with a ramp between pairs that turn 32 times and once over the trained length."""
    pairs = rot // 2
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2))
    theta = [base ** (-2.0 * i / rot) for i in range(pairs)]
    if scaling == "linear":
        theta = [t / factor for t in theta]
    if scaling == "yarn":
        def at(turns):
            return rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(pairs)]
        theta = [t / factor * r + t * (1 - r) for t, r in zip(theta, ramp)]
        return theta, 0.1 * math.log(factor) + 1.0
    return theta, 1.0


def fixed_point(theta):
    """Turns a position in units of 2**-64 of a turn: products with whole positions wrap at whole turns."""
    return torch.tensor([int(t / (2 * math.pi) * 2.0 ** 64) for t in theta], dtype=torch.int64, device=DEVICE)


def prepare_rotary(case, g):
    theta, scale = frequencies(case["rot"], case["scaling"], case["factor"], case["trained"])
    # a projection's output: the heads that are rotated, then those that are not
    whole = normal(g, case["tokens"], case["heads"] + 2, case["dim"], dtype=DTYPES[case["dtype"]])
    spread = torch.randint(0, 1000, (1,), generator=g, device=DEVICE)
    positions = torch.arange(case["tokens"], device=DEVICE) + case["offset"] + spread
    state = {"case": case, "x": whole[:, :case["heads"]], "positions": positions, "scale": scale,
             "freq": fixed_point(theta)}
    if own:
        from jasper_b200 import paged
        scaling = None if case["scaling"] == "none" else case["scaling"]
        state["rotary"] = paged.Rotary(case["dim"], case["rot"], layout=case["layout"], scaling=scaling,
                                       factor=case["factor"], trained_length=case["trained"])
    return state


def prepare_append(case, g):
    dtype, ps, n, hq, hkv = DTYPES[case["dtype"]], case["page_size"], case["tokens"], case["q_heads"], case["kv_heads"]
    theta, scale = frequencies(case["rot"])
    if case["prompt"]:  # a few prompts, one after the other
        cuts = sorted({0, n // 3, n // 3 + n // 2, n})
        sizes = [b - a for a, b in zip(cuts, cuts[1:])]
        rows = torch.repeat_interleave(torch.arange(len(sizes), device=DEVICE),
                                       torch.tensor(sizes, device=DEVICE), output_size=n)
        index = torch.cat([torch.arange(s, device=DEVICE) for s in sizes])
    else:  # the next token of every conversation
        sizes = [case["offset"] - case["offset"] * i // (2 * n) for i in range(n)]
        rows = permutation(g, n)
        sizes_of = torch.tensor(sizes, device=DEVICE)
        index = sizes_of[rows] - 1
    held_pages = [-(-s // ps) for s in sizes]
    width, total = max(held_pages), sum(held_pages)
    inside = torch.arange(width, device=DEVICE) < torch.tensor(held_pages, device=DEVICE)[:, None]
    order = permutation(g, total + 3)
    rank = (inside.view(-1).cumsum(0) - 1).clamp_min(0)
    table = torch.where(inside, order[rank].view(-1, width), -1)
    refs = torch.zeros(total + 3, dtype=torch.int32, device=DEVICE)
    refs[order[:total]] = 1
    qkv = normal(g, n, hq + 2 * hkv, case["dim"], dtype=dtype)
    k = store(g, 1, total + 3, ps, hkv, case["dim"], dtype, "token")
    v = store(g, 1, total + 3, ps, hkv, case["dim"], dtype, "token")
    state = {"case": case, "qkv": qkv, "k": k, "v": v, "table": table.int(), "refs": refs, "scale": scale,
             "lengths": torch.tensor(sizes, dtype=torch.int32, device=DEVICE), "rows": rows.int(),
             "index": index.int(), "freq": fixed_point(theta)}
    if own:
        from jasper_b200 import paged
        state["rotary"] = paged.Rotary(case["dim"], case["rot"], layout=case["layout"])
    return held(state)


def token_counts(case):
    """Tokens of each row that holds pages, spread around the case's mean, within the pool."""
    rows = case["rows"] if case["kind"] != "fork" else case["rows"] // 2
    wanted = [1 + (case["mean"] * (2 * i + 1)) // rows for i in range(rows)]
    room = case["n_pages"] - (case["rows"] if case["kind"] == "fork" else 0)
    while sum(-(-n // case["page_size"]) for n in wanted) > room:
        wanted = [n // 2 + 1 if n > 1 else 0 for n in wanted]
    return wanted


def prepare_pages(case, g):
    ps, n_pages, rows, named = case["page_size"], case["n_pages"], case["rows"], case["named"]
    counts = token_counts(case)
    held_pages = [-(-n // ps) for n in counts]
    dims = (case["layers"], n_pages, ps, case["kv_heads"], case["dim"], torch.float16, case["layout"])
    k, v = store(g, *dims), store(g, *dims)
    holders = permutation(g, rows)[:len(counts)]
    width = 2 * max(held_pages) + 1
    inside = torch.arange(width, device=DEVICE) < torch.tensor(held_pages, device=DEVICE)[:, None]
    rank = (inside.view(-1).cumsum(0) - 1).clamp_min(0)
    order = permutation(g, n_pages)
    table = torch.full((rows, width), -1, device=DEVICE)
    table[holders] = torch.where(inside, order[rank].view(-1, width), -1)
    lengths = torch.zeros(rows, dtype=torch.int64, device=DEVICE)
    lengths[holders] = torch.tensor(counts, device=DEVICE)
    refs = torch.zeros(n_pages, dtype=torch.int64, device=DEVICE)
    refs[order[:sum(held_pages)]] = 1
    state = {"case": case, "k": k, "v": v, "table": table.int(), "lengths": lengths.int(), "refs": refs.int()}
    if case["kind"] == "turnover":  # these leave, and prompts of other lengths take their places
        state["rows"] = holders[permutation(g, len(counts))[:named]].int()
        state["tokens"] = state["lengths"][state["rows"].long()].flip(0).contiguous()
    if case["kind"] == "fork":  # every other row is a fork's place; parents come up again and again
        free = torch.ones(rows, dtype=torch.bool, device=DEVICE)
        free[holders] = False
        children = torch.argsort(free.int(), descending=True, stable=True)[:rows - len(counts)]
        state["children"] = children[:named].int()
        pick = torch.randint(0, len(counts), (len(state["children"]),), generator=g, device=DEVICE)
        state["parents"] = holders[pick].int()
    if case["kind"] == "copy":
        two = permutation(g, n_pages)[:2 * named].int()
        state["src"], state["dst"] = two[:named].contiguous(), two[named:].contiguous()
    if case["kind"] == "compact":  # the book-keeping as it was before the call, and as the call leaves it
        state["before"] = (state["table"].clone(), state["refs"].clone())
    return held(state)


# ── one pass ─────────────────────────────────────────────────────────────

def run(state):
    case = state["case"]
    if case["op"] == "attend":
        if own:
            return state["cache"].attend(0, state["q"], scale=state["scale"], window=case["window"],
                                         mask=state["mask"], return_lse=True)
        return plain_attend(state)
    if case["op"] == "rotary":
        if own:
            call = state["rotary"].grad if case["gradient"] else state["rotary"].apply
            return call(state["x"], state["positions"])
        return plain_turn(state["x"], state["positions"], state, backwards=case["gradient"])
    if case["op"] == "append":
        hq, hkv = case["q_heads"], case["kv_heads"]
        q, k, v = state["qkv"].split([hq, hkv, hkv], dim=1)
        if own:
            q = state["cache"].append(0, k, v, state["rows"], state["index"], q=q, rotary=state["rotary"])
        else:
            q = plain_append(state, q, k, v)
        return q, state["k"], state["v"]
    (run_pages_own if own else run_pages_plain)(state)
    out = {"table": state["table"], "lengths": state["lengths"], "refs": state["refs"]}
    if case["kind"] != "turnover":  # pages are moved, not computed: their bits
        out["k"], out["v"] = state["k"].view(torch.int16), state["v"].view(torch.int16)
    return out


def run_pages_own(state):
    cache, kind = state["cache"], state["case"]["kind"]
    if kind == "turnover":
        cache.free(state["rows"])
        cache.extend(state["rows"], state["tokens"])
    elif kind == "fork":
        cache.free(state["children"])
        cache.fork(state["parents"], state["children"])
    elif kind == "copy":
        cache.copy_pages(state["src"], state["dst"])
    else:
        state["table"].copy_(state["before"][0])
        state["refs"].copy_(state["before"][1])
        cache.compact()


def plain_attend(state):
    case, table, ps = state["case"], state["table"].long(), state["case"]["page_size"]
    batch, width = table.shape
    hkv, dim = case["kv_heads"], case["dim"]
    at = table.clamp_min(0)
    k = state["k"][0, at].float().reshape(batch, width * ps, hkv, dim)
    v = state["v"][0, at].float().reshape(batch, width * ps, hkv, dim)
    place = torch.arange(width * ps, device=table.device)
    length = state["lengths"][:, None].long()
    seen = (place < length) & (table >= 0).repeat_interleave(ps, dim=1)
    if case["window"]:
        seen &= place >= length - case["window"]
    if state["mask"] is not None:
        seen &= state["mask"]
    q = state["q"].float().view(batch, hkv, -1, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)) * state["scale"]  # [batch, kv head, group, token]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.transpose(1, 2)) / torch.where(total == 0, 1.0, total)
    lse = (torch.log(total) + top).view(batch, -1)
    return out.view(batch, -1, dim).to(state["q"].dtype), lse


def plain_turn(x, positions, state, backwards=False):
    case = state["case"]
    rot, half = case["rot"], case["rot"] // 2
    phase = (positions.long()[:, None] * state["freq"]) >> 32  # units of 2**-32 of a turn, signed
    angle = (phase.float() * (2 * math.pi / 2 ** 32))[:, None]
    c, s = torch.cos(angle) * state["scale"], torch.sin(angle) * state["scale"]
    s = -s if backwards else s
    x32 = x.float()
    if case["layout"] == "half":
        a, b = x32[..., :half], x32[..., half:rot]
        turned = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = x32[..., 0:rot:2], x32[..., 1:rot:2]
        turned = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([turned, x32[..., rot:]], -1).to(x.dtype)


def plain_append(state, q, k, v):
    rows, index, ps = state["rows"].long(), state["index"].long(), state["case"]["page_size"]
    page = state["table"][rows, index // ps].long()
    state["k"][0, page, index % ps] = plain_turn(k, index, state)
    state["v"][0, page, index % ps] = v
    return plain_turn(q, index, state)


def run_pages_plain(state):
    kind = state["case"]["kind"]
    if kind == "turnover":
        plain_free(state, state["rows"].long())
        plain_extend(state, state["rows"].long(), state["tokens"].long())
    elif kind == "fork":
        plain_free(state, state["children"].long())
        plain_fork(state, state["parents"].long(), state["children"].long())
    elif kind == "copy":
        src, dst = state["src"].long(), state["dst"].long()
        state["k"][:, dst] = state["k"][:, src]
        state["v"][:, dst] = state["v"][:, src]
    else:
        state["table"].copy_(state["before"][0])
        state["refs"].copy_(state["before"][1])
        plain_compact(state)


def count_holders(state, entries, by):
    """Adds `by` to the holders of every page among `entries` (-1: none)."""
    n = state["refs"].numel()
    refs = torch.cat([state["refs"], state["refs"].new_zeros(1)])
    refs.index_add_(0, torch.where(entries < 0, n, entries).view(-1).long(),
                    torch.full((entries.numel(),), by, dtype=refs.dtype, device=refs.device))
    state["refs"].copy_(refs[:n])


def plain_free(state, rows):
    count_holders(state, state["table"][rows], -1)
    state["table"][rows] = -1
    state["lengths"][rows] = 0


def free_pages(state):
    """The free pages in rising order, then the others."""
    return torch.argsort((state["refs"] > 0).int(), stable=True), (state["refs"] == 0).sum()


def plain_extend(state, rows, tokens):
    ps, width = state["case"]["page_size"], state["table"].shape[1]
    have = (state["lengths"][rows].long() + ps - 1) // ps
    need = (state["lengths"][rows].long() + tokens + ps - 1) // ps
    wanted = torch.where(need <= width, need - have, 0)
    upto = wanted.cumsum(0)
    order, n_free = free_pages(state)
    given = (need <= width) & ((upto <= n_free) | (wanted == 0))
    place = torch.arange(width, device=rows.device)
    new = (place >= have[:, None]) & (place < need[:, None]) & given[:, None]
    rank = ((upto - wanted)[:, None] + place - have[:, None]).clamp(0, order.numel() - 1)
    entries = torch.where(new, order[rank].int(), state["table"][rows])
    count_holders(state, torch.where(new, entries, -1), 1)
    state["table"][rows] = entries
    state["lengths"][rows] += torch.where(given, tokens, 0).int()


def plain_fork(state, parents, children):
    ps, width = state["case"]["page_size"], state["table"].shape[1]
    length = state["lengths"][parents].long()
    whole, part = length // ps, length % ps
    old = state["table"][parents]
    last = old.gather(1, whole.clamp_max(width - 1)[:, None])[:, 0].long()
    wanted = ((part > 0) & (last >= 0)).long()
    upto = wanted.cumsum(0)
    order, n_free = free_pages(state)
    given = (upto <= n_free) | (wanted == 0)
    place = torch.arange(width, device=parents.device)
    copies = (wanted > 0) & given
    page = order[(upto - 1).clamp(0, order.numel() - 1)]
    entries = torch.where(place < whole[:, None], old, -1)
    entries = torch.where((place == whole[:, None]) & copies[:, None], page[:, None].int(), entries)
    entries = torch.where(given[:, None], entries, -1)
    count_holders(state, entries, 1)
    state["table"][children] = entries
    state["lengths"][children] = torch.where(given, length, 0).int()
    # the tokens of each part-filled page, in every layer
    pair, slot = torch.where(copies[:, None] & (torch.arange(ps, device=parents.device) < part[:, None]))
    for cache in (state["k"], state["v"]):
        cache[:, page[pair], slot] = cache[:, last[pair], slot]


def plain_compact(state):
    refs, table = state["refs"], state["table"]
    n = refs.numel()
    live = refs > 0
    place = torch.arange(n, device=refs.device)
    n_live = live.sum()
    src, dst = torch.where(live & (place >= n_live))[0], torch.where(~live & (place < n_live))[0]
    remap = torch.where(live, place, -1)
    remap[src] = dst
    state["k"][:, dst] = state["k"][:, src]
    state["v"][:, dst] = state["v"][:, src]
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(table >= 0, remap[table.clamp_min(0).long()].int(), -1))


# ── what a pass cannot do without ────────────────────────────────────────

def work(case):
    if case["op"] == "attend":
        hq, hkv, dim = case["q_heads"], case["kv_heads"], case["dim"]
        tokens = sum(spread_lengths(case))
        read = tokens
        if case["window"]:
            tokens = read = sum(min(n, case["window"]) for n in spread_lengths(case))
        if case["retrieved"]:  # 4 % of the answers are empty, passages fill three quarters of a page, pages are shared
            tokens = int(tokens * 0.96 * 0.75)
            width = case["longest"] // case["page_size"]
            distinct = case["pages"] * (1 - (1 - 1 / case["pages"]) ** (0.96 * case["batch"] * width))
            read = min(tokens, int(0.75 * case["page_size"] * distinct))
        return {"bytes": 4 * read * hkv * dim + 4 * case["batch"] * hq * dim, "flops": 4 * tokens * hq * dim}
    size = 4 if case.get("dtype") == "float32" else 2
    if case["op"] == "rotary":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * size, "flops": 3 * n * case["rot"]}
    if case["op"] == "append":
        n, hq, hkv = case["tokens"], case["q_heads"], case["kv_heads"]
        return {"bytes": 2 * n * (hq + 2 * hkv) * case["dim"] * size, "flops": 3 * n * (hq + hkv) * case["rot"]}
    ps, counts = case["page_size"], token_counts(case)
    token = case["layers"] * 2 * case["kv_heads"] * case["dim"] * 2
    book = 4 * (sum(-(-n // ps) for n in counts) + case["n_pages"])  # the table's entries and the counts
    moved = 0
    if case["kind"] == "copy":
        moved, book = case["named"] * ps, 8 * case["named"]
    if case["kind"] == "fork":
        moved = min(case["named"], case["rows"] - len(counts)) * sum(n % ps for n in counts) / max(1, len(counts))
    if case["kind"] == "compact":
        share = sum(-(-n // ps) for n in counts) / case["n_pages"]
        moved = share * (1 - share) * case["n_pages"] * ps
    return {"bytes": int(2 * moved * token + 2 * book), "flops": 0}


# ── the definitions in 64 bits ───────────────────────────────────────────

def exact(case, seed):
    if case["op"] == "pages":  # whole numbers and bits only
        return None
    global own
    was, own = own, False
    state = prepare(case, seed)
    own = was
    if case["op"] == "attend":
        return exact_attend(case, state)
    if case["op"] == "rotary":
        return exact_turn(case, state["x"], state["positions"].cpu(), -1 if case["gradient"] else 1)
    hq, hkv, ps = case["q_heads"], case["kv_heads"], case["page_size"]
    k, v = state["k"].double(), state["v"].double()
    place = state["index"].cpu()
    turned = exact_turn(case, state["qkv"][:, :hq + hkv], place, 1)
    values = state["qkv"][:, hq + hkv:].double()
    table = state["table"].cpu()
    for n, (row, i) in enumerate(zip(state["rows"].tolist(), place.tolist())):
        page = int(table[row, i // ps])
        k[0, page, i % ps] = turned[n, hq:]
        v[0, page, i % ps] = values[n]
    return turned[:, :hq], k, v


def exact_attend(case, state):
    ps, group = case["page_size"], case["q_heads"] // case["kv_heads"]
    table, lengths = state["table"].cpu(), state["lengths"].tolist()
    outs, lses = [], []
    for b, n in enumerate(lengths):
        first = max(0, n - case["window"]) if case["window"] else 0
        tokens = torch.arange(first, n)
        page = table[b, tokens // ps]
        kept = page >= 0
        if state["mask"] is not None:
            kept &= state["mask"][b, :n].cpu()[tokens]
        tokens, page = tokens[kept].to(DEVICE), page[kept].long().to(DEVICE)
        out = torch.zeros(case["q_heads"], case["dim"], dtype=torch.float64, device=DEVICE)
        lse = torch.full((case["q_heads"],), -math.inf, dtype=torch.float64, device=DEVICE)
        if len(tokens):
            for h in range(case["kv_heads"]):
                q = state["q"][b, h * group:(h + 1) * group].double()
                keys = state["k"][0, page, tokens % ps, h].double()
                values = state["v"][0, page, tokens % ps, h].double()
                logits = q @ keys.T * state["scale"]
                lse[h * group:(h + 1) * group] = torch.logsumexp(logits, 1)
                out[h * group:(h + 1) * group] = torch.softmax(logits, 1) @ values
        outs.append(out)
        lses.append(lse)
    return torch.stack(outs), torch.stack(lses)


def exact_turn(case, x, positions, sign):
    theta, scale = frequencies(case["rot"], case.get("scaling", "none"), case.get("factor", 1.0), case.get("trained", 0))
    angle = sign * positions.double()[:, None] * torch.tensor(theta, dtype=torch.float64)
    turn = torch.polar(torch.full_like(angle, scale), angle).to(x.device)[:, None]  # a complex number for each pair
    y = x.double().clone()
    pairs = case["rot"] // 2
    if case["layout"] == "half":
        first, second = slice(0, pairs), slice(pairs, case["rot"])
    else:
        first, second = slice(0, case["rot"], 2), slice(1, case["rot"], 2)
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y
