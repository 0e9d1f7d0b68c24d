"""A cache of keys and values in pages, continued: operators that are measured one by one.

  append    keys and values of new tokens into the pages, keys and the queries beside them normed per head and rotated on the way, by positions of one
            axis or several (ops.paged_append with norms, with an axis for every pair of columns)
  prefix    attention of sequences in groups that share their first pages, which are read once for a group (ops.paged_prefix_attention)
  weights   attention that adds every row's softmax weights up, over queries and the heads that read it (ops.paged_attention_weights)
  evict     the rows of least accumulated weight leave the cache, the others close up, in every layer (ops.paged_evict)

A page table row lists the pages of a sequence in order; row r of a sequence lies in its page r // page_size. Lengths count the
rows before the new tokens. Heads, widths and layers are those of bench.py (32 and 16 query heads, 8 key / value heads of 128, 28 and 32
layers) or generic.

With `own` false, run() computes the operators in elementary torch operations, in 32 bits."""
import functools
import math
import random
import zlib

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
F64 = torch.float64
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ the cases
def _append(name, seqs, new, **more):
    return dict(dict(name=name, kind="append", seqs=seqs, new=new, before=0, heads=32, kv_heads=8, dim=128, page=64, rotary=128, neighbours=False, norm=True,
                     axes=1, mixed=False, table="f16", dtype="f16"), **more)


def _prefix(name, groups, seqs, prefix, rest, new, **more):
    return dict(dict(name=name, kind="prefix", groups=groups, seqs=seqs, prefix=prefix, rest=rest, new=new, tree=new > 1, heads=32, kv_heads=8, dim=128, page=64,
                     dtype="f16"), **more)


def _weights(name, seqs, ctx, new, **more):
    return dict(dict(name=name, kind="weights", seqs=seqs, ctx=ctx, new=new, heads=32, kv_heads=8, dim=128, page=64, dtype="f16"), **more)


def _evict(name, seqs, ctx, budget, recent, layers, **more):
    return dict(dict(name=name, kind="evict", seqs=seqs, ctx=ctx, budget=budget, recent=recent, layers=layers, kv_heads=8, dim=128, page=64, dtype="f16"), **more)


def listed():
    return [
        # one token of each of 32 sequences that a server decodes together, queries and keys normed per head: latency
        _append("append_decode_32", 32, 1, before=900, heads=16),
        # eight prompts of text and images in one forward: positions in time, height and width
        _append("append_images", 8, 1900, axes=3, dtype="bf16", table="f32"),
        # a portion of one prompt, three axes that take turns from pair to pair, no norms, neighbouring columns
        _append("append_portion", 3, 250, before=700, axes=3, mixed=True, norm=False, neighbours=True),
        # four continuations of one short prompt: latency
        _prefix("prefix_4", 1, 4, 640, 40, 1),
        # 64 users behind one long instruction
        _prefix("prefix_decode_64", 1, 64, 8192, 700, 1),
        # eight questions, eight answers to each being sampled
        _prefix("prefix_8x8", 8, 8, 3000, 500, 1, page=48, dtype="bf16"),
        # 16 users ask about one long document, trees of 26 drafted tokens each
        _prefix("prefix_trees_16", 1, 16, 30000, 300, 26, dtype="bf16"),
        # one user, one token, a short context: latency
        _weights("weights_one_token", 1, 600, 1),
        # a server's decode batch, lengths from an eighth of the longest up
        _weights("weights_decode_32", 32, 8192, 1),
        # the last 64 tokens of a long prompt say which of its rows matter
        _weights("weights_window_64", 1, 32001, 64, dtype="bf16"),
        # one user's cache back to a thousand rows, every layer
        _evict("evict_one", 1, 1100, 1000, 100, 28),
        # 16 users' prompts down to 1024 rows
        _evict("evict_16", 16, 4096, 1024, 64, 8, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "prefix", "prefix", "weights", "weights", "evict"])
    dtype = rng.choice(["f16", "bf16"])
    dim = rng.choice([64, 128, 128, 256])
    heads, kv_heads = rng.choice([(32, 8), (16, 8), (8, 8), (12, 2), (10, 2), (28, 4), (16, 1), (9, 3)])
    page = rng.choice([16, 32, 64, 128, rng.randint(5, 200)])
    if kind == "append":
        new = rng.choice([1, 1, _log(rng, 2, 1500)])
        return _append(None, _log(rng, 1, max(1, min(200, 9000 // new))), new, before=rng.choice([0, _log(rng, 1, 500)]), heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                       rotary=rng.choice([dim, dim // 2]), neighbours=rng.random() < 0.3, norm=rng.random() < 0.7, axes=rng.choice([1, 2, 3, 4]), mixed=rng.random() < 0.5,
                       table=rng.choice(["f16", "f32"]), dtype=dtype)
    if kind == "prefix":
        tree = rng.random() < 0.3
        new = _log(rng, 2, 64) if tree else 1
        groups, seqs = _log(rng, 1, 12), _log(rng, 1, 64)
        # no more products, and no more rows for all sequences, than the largest listed cases have
        rows = min(64 * 8892 * 1024 // (kv_heads * dim), 16 * 30300 * 26 * 4096 // (new * heads * dim)) // (groups * seqs)
        prefix = _log(rng, 1, max(2, min(60000, rows - 1)))
        return _prefix(None, groups, seqs, prefix, _log(rng, 1, max(2, min(1000, rows - prefix))), new, tree=tree, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if kind == "weights":
        new = rng.choice([1, 1, 1, _log(rng, 2, 100)])
        rows = min(32 * 5000 * 1024 // (kv_heads * dim), 32001 * 64 * 4096 // (new * heads * dim))
        seqs = _log(rng, 1, 48)
        return _weights(None, seqs, _log(rng, 1, max(2, min(60000, rows // seqs))), new, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    layers, kv_heads, dim = rng.randint(1, 32), rng.choice([1, 2, 3, 8]), rng.choice([64, 128])
    ctx = _log(rng, 20, 8000)
    budget = rng.randint(1, ctx)
    seqs = _log(rng, 1, max(1, min(48, 16 * 4096 * 8 * 1024 // (ctx * layers * kv_heads * dim))))
    return _evict(None, seqs, ctx, budget, rng.choice([0, rng.randint(0, budget), min(budget, 32)]), layers, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed, name):
    return torch.Generator(device="cuda").manual_seed((seed * 7919 + zlib.crc32(name.encode())) % (1 << 62))


def _randn(seed, name, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=_gen(seed, name), device="cuda", dtype=dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _spread(n, top, least=1):
    """Counts for n sequences, the first `top`, the others between an eighth of it and itself: the same for every seed."""
    r = random.Random(n * 100003 + top)
    return [top if i == 0 else r.randint(max(least, top // 8), max(least, top)) for i in range(n)]


def _lengths(c):
    """(rows before, new tokens) of every sequence."""
    if c["kind"] == "prefix":
        n = c["groups"] * c["seqs"]
        return [c["prefix"] // c["page"] * c["page"] + k for k in _spread(n, c["rest"])], [c["new"]] * n
    n = c["seqs"]
    if c["kind"] == "append":
        return (_spread(n, c["before"]) if c["before"] else [0] * n), _spread(n, c["new"])
    if c["kind"] == "weights":
        return _spread(n, c["ctx"]), (_spread(n, c["new"]) if n > 1 else [c["new"]])
    return _spread(n, c["ctx"]), [0] * n


def _pages(c, seed, per_seq, layers=1):
    """(keys, values, table) of a pool whose pages are handed out in no order."""
    n, most = len(per_seq), max(per_seq)
    total = sum(per_seq) + 3
    order = torch.randperm(total, generator=_gen(seed, "order"), device="cuda").int()
    table = torch.zeros((n, most), dtype=torch.int32, device="cuda")
    start = 0
    for i, k in enumerate(per_seq):
        table[i, :k] = order[start:start + k]
        start += k
    shape = (layers, total, c["kv_heads"], c["page"], c["dim"])
    keys, values = (torch.empty(shape, dtype=DT[c["dtype"]], device="cuda") for _ in range(2))
    for pool, name in ((keys, "keys"), (values, "values")):
        g = _gen(seed, name)
        for layer in pool:
            layer.copy_(torch.randn(layer.shape, generator=g, device="cuda"))
    return keys, values, table


def _rotation_table(c, most):
    """cos and sin [positions, dim / 2] of the angles position * 500000 ** (-2 i / rotary); the part beyond rotary / 2 is not used."""
    i = torch.arange(c["dim"] // 2, dtype=F64, device="cuda")
    angle = torch.arange(most, dtype=F64, device="cuda")[:, None] * (5e5 ** (-2.0 * i / c["rotary"]))
    return torch.cos(angle).to(DT[c["table"]]), torch.sin(angle).to(DT[c["table"]])


def _pair_axis(c):
    """The axis of every rotated pair of columns: in turns, or in runs of which the first is the shortest."""
    half, n = c["rotary"] // 2, c["axes"]
    if c["mixed"]:
        return [i % n for i in range(half)]
    first = half // (n + 1)
    return [0 if i < first else min(n - 1, 1 + (i - first) * (n - 1) // (half - first)) if n > 1 else 0 for i in range(half)]


def _tree(seed, n, count):
    """Masks of `count` trees of n nodes [count * n, words]: bit j of a node's words is set where it sees node j, an ancestor or itself."""
    r = random.Random(seed * 131 + n)
    words, rows = -(-n // 64), []
    for _ in range(count):
        sees = []
        for t in range(n):
            sees.append((sees[r.randint(max(0, t - 9), t - 1)] if t > 0 else 0) | 1 << t)
        for m in sees:
            parts = [(m >> 64 * w) & (1 << 64) - 1 for w in range(words)]
            rows.append([p - (1 << 64) if p >> 63 else p for p in parts])
    return torch.tensor(rows, dtype=torch.int64, device="cuda")


def _starts(new):
    s = [0]
    for k in new:
        s.append(s[-1] + k)
    return s


@functools.lru_cache(None)
def _device():
    """The handle that a program opens once."""
    from ironmill_b200 import ops
    return ops.Device(0)


def prepare(case, seed):
    c, kind = case, case["kind"]
    s = dict(case=c)
    lengths, new = _lengths(c)
    n, total = len(lengths), sum(new)
    room = [-(-(a + b) // c["page"]) for a, b in zip(lengths, new)]
    keys, values, table = _pages(c, seed, room, c.get("layers", 1))
    s["starts"], s["new"] = _ints(_starts(new)), max(new)
    if kind == "append":
        # one row per token as the projection leaves it: queries, keys, values; norm weights around one
        qkv = _randn(seed, "qkv", total, c["heads"] + 2 * c["kv_heads"], c["dim"]).to(DT[c["dtype"]])
        s["q"], s["k"], s["v"] = qkv.split([c["heads"], c["kv_heads"], c["kv_heads"]], 1)
        s["q_norm"], s["k_norm"] = ((1 + 0.2 * _randn(seed, x, c["dim"])).to(DT[c["dtype"]]) if c["norm"] else None for x in ("q_norm", "k_norm"))
        s["cos"], s["sin"] = _rotation_table(c, max(a + b for a, b in zip(lengths, new)) + 64)
        s["positions"], s["pair_axis"] = None, None
        if c["axes"] > 1:
            # text counts on all axes alike, an image's tokens have one time and places of their own
            row = torch.cat([torch.arange(a, a + b) for a, b in zip(lengths, new)]).to("cuda")
            place = torch.randint(64, (c["axes"], total), generator=_gen(seed, "place"), device="cuda")
            image = torch.arange(total, device="cuda") % 512 >= 100
            s["positions"] = torch.where(image, row // 32 * 32 * (torch.arange(c["axes"], device="cuda")[:, None] == 0) + place, row).int()
            s["pair_axis"] = bytes(_pair_axis(c))
    elif kind == "evict":
        rows = table.shape[1] * c["page"]
        # sums of softmax weights: few large ones, many small ones, some rows that nothing has looked at
        w = torch.exp(2 * _randn(seed, "weights", c["layers"], n, c["kv_heads"], rows))
        s["weights"] = torch.where(torch.rand(w.shape, generator=_gen(seed, "unseen"), device="cuda") < 0.05, 0.0, w)
        s["weights_out"] = torch.zeros_like(w)
    else:
        s["q"] = _randn(seed, "q", total, c["heads"], c["dim"]).to(DT[c["dtype"]])
        s["longest"] = max(a + b for a, b in zip(lengths, new))
        s["mask"] = None
        if kind == "prefix":
            shared = c["prefix"] // c["page"]
            for g in range(c["groups"]):
                at = g * c["seqs"]
                table[at:at + c["seqs"], :shared] = table[at, :shared].clone()
            s["group_start"], s["prefix_pages"] = _ints([g * c["seqs"] for g in range(c["groups"] + 1)]), _ints([shared] * c["groups"])
            s["mask"] = _tree(seed, c["new"], n) if c["tree"] else None
        else:
            s["weights"] = torch.rand((n, c["kv_heads"], table.shape[1] * c["page"]), generator=_gen(seed, "weights"), device="cuda")
    s.update(keys=keys, values=values, table=table, lengths=_ints(lengths))
    if own:
        from ironmill_b200 import ops
        s["kv"] = ops.PagedKV(_device(), keys, values, table, s["lengths"])
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"append": _run_append, "prefix": _run_prefix, "weights": _run_weights, "evict": _run_evict}[state["case"]["kind"]](state)


def _places(s, total):
    """(sequence, place among its new tokens) of every token."""
    token = torch.arange(total, device="cuda")
    seq = torch.searchsorted(s["starts"], token.int(), right=True) - 1
    return seq, token - s["starts"].long()[seq]


def _rotated(x, cos, sin, rotary, neighbours):
    """x [tokens, heads, dim] in 32 bits, its first `rotary` columns turned by the tokens' angles (cos, sin [tokens, rotary / 2])."""
    cos, sin = cos.float()[:, None], sin.float()[:, None]
    part, rest = x[..., :rotary], x[..., rotary:]
    if neighbours:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part[..., :rotary // 2], part[..., rotary // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, rest], -1)


def _run_append(s):
    c = s["case"]
    if own:
        from ironmill_b200 import ops
        q = ops.paged_append(s["kv"], 0, s["k"], s["v"], s["starts"], q=s["q"], cos=s["cos"], sin=s["sin"], positions=s["positions"], rotary_dim=c["rotary"],
                             neighbours=c["neighbours"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, pair_axis=s["pair_axis"])
        return [q, s["keys"], s["values"]]
    seq, place = _places(s, s["k"].shape[0])
    row, half = s["lengths"].long()[seq] + place, c["rotary"] // 2
    if c["axes"] > 1:
        pair = torch.arange(half, device="cuda")
        at = s["positions"].long()[torch.tensor(list(s["pair_axis"]), device="cuda")].T        # [tokens, pairs]
        cos, sin = s["cos"][at, pair], s["sin"][at, pair]
    else:
        cos, sin = s["cos"][row, :half], s["sin"][row, :half]
    got = []
    for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
        got.append(_rotated(y, cos, sin, c["rotary"], c["neighbours"]).to(x.dtype))
    page, slot = s["table"].long()[seq, row // c["page"]], row % c["page"]
    s["keys"][0][page, :, slot] = got[1]
    s["values"][0][page, :, slot] = s["v"]
    return [got[0], s["keys"], s["values"]]


def _softmax_of(s):
    """Weights [sequences, key heads, groups, new, rows] of the new tokens (zero in places without one), values [sequences, key heads, rows, dim], places."""
    c = s["case"]
    total, groups, seqs = s["q"].shape[0], c["heads"] // c["kv_heads"], s["lengths"].shape[0]
    seq, place = _places(s, total)
    row = torch.arange(s["longest"], device="cuda")
    page, slot = s["table"].long()[:, row // c["page"]], (row % c["page"])[None]
    k, v = (s[x][0][page, :, slot].float().transpose(1, 2) for x in ("keys", "values"))
    ahead = row[None] - s["lengths"][seq, None]                                               # [tokens, rows]: place among the new rows
    fits = ahead < (s["starts"][1:] - s["starts"][:-1])[seq, None]
    if s["mask"] is None:
        seen = ahead <= place[:, None]
    else:
        word = (ahead.clamp(min=0) // 64).clamp(max=s["mask"].shape[1] - 1)
        seen = (ahead < 0) | ((s["mask"].gather(1, word) >> (ahead.clamp(min=0) % 64)) & 1).bool()
    q = torch.zeros((seqs, s["new"], c["kv_heads"], groups, c["dim"]), device="cuda")
    see = torch.zeros((seqs, s["new"], s["longest"]), dtype=torch.bool, device="cuda")
    q[seq, place] = s["q"].float().view(total, c["kv_heads"], groups, c["dim"])
    see[seq, place] = seen & fits
    score = torch.matmul(q.permute(0, 2, 3, 1, 4).flatten(2, 3), k.transpose(2, 3)).unflatten(2, (groups, s["new"])) * c["dim"] ** -0.5
    score = torch.where(see[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    sums = weight.sum(-1, keepdim=True)
    return weight / torch.where(sums == 0, 1.0, sums), v, seq, place


def _outputs(s, weight, v, seq, place):
    c = s["case"]
    out = torch.matmul(weight.flatten(2, 3), v).unflatten(2, weight.shape[2:4])
    return out.permute(0, 3, 1, 2, 4)[seq, place].reshape(s["q"].shape).to(DT[c["dtype"]])


def _run_prefix(s):
    c = s["case"]
    if own:
        from ironmill_b200 import ops
        return ops.paged_prefix_attention(s["kv"], 0, s["q"], s["starts"], s["new"], c["dim"] ** -0.5, s["group_start"], c["seqs"] * c["new"], s["prefix_pages"],
                                          max_prefix=c["prefix"], mask=s["mask"], max_len=s["longest"])
    return _outputs(s, *_softmax_of(s))


def _run_weights(s):
    c = s["case"]
    if own:
        from ironmill_b200 import ops
        return [ops.paged_attention_weights(s["kv"], 0, s["q"], s["starts"], s["new"], c["dim"] ** -0.5, s["weights"], max_len=s["longest"]), s["weights"]]
    weight, v, seq, place = _softmax_of(s)
    row = torch.arange(s["longest"], device="cuda")
    before = row < s["lengths"][:, None]
    there = row < (s["lengths"] + s["starts"][1:] - s["starts"][:-1])[:, None]
    old = s["weights"][..., :s["longest"]]
    s["weights"][..., :s["longest"]] = torch.where(there[:, None], weight.sum((2, 3)) + torch.where(before[:, None], old, 0.0), old)    # a new row's sum starts here
    return [_outputs(s, weight, v, seq, place), s["weights"]]


def _run_evict(s):
    c = s["case"]
    if own:
        from ironmill_b200 import ops
        lengths, weights = ops.paged_evict(s["kv"], s["weights"], c["budget"], c["recent"], weights_out=s["weights_out"])
        return [lengths, weights, s["keys"], s["values"]]
    heavy = c["budget"] - c["recent"]                     # rows that stay for their weight
    lengths = s["lengths"].long()
    fresh = torch.minimum(lengths, lengths.clamp(max=c["budget"]))
    rows = s["weights"].shape[-1]
    row = torch.arange(rows, device="cuda")
    over = (lengths > c["budget"])[None, :, None, None]
    old = row < (lengths - c["recent"])[None, :, None, None]
    # places by weight, ties to the lowest row
    order = torch.where(old, s["weights"], -math.inf).argsort(dim=-1, descending=True, stable=True)
    stays = torch.zeros_like(s["weights"], dtype=torch.bool).scatter_(-1, order[..., :heavy], True)
    hole, mover = over & ~stays & (row < heavy), over & stays & (row >= heavy)
    source = row.expand(s["weights"].shape).clone()
    source[hole] = row.expand(s["weights"].shape)[mover]                                       # both in order of their rows
    source = torch.where(over & (row >= heavy) & (row < c["budget"]), row + (lengths - c["budget"])[None, :, None, None], source)
    live = row < fresh[None, :, None, None]
    source = torch.where(live, source, row)
    s["weights_out"].copy_(torch.where(live, s["weights"].gather(-1, source), s["weights_out"]))
    table = s["table"].long()
    for layer in range(c["layers"]):
        seq, head, to = (source[layer] != row).nonzero(as_tuple=True)
        at = source[layer][seq, head, to]
        for x in ("keys", "values"):
            moved = s[x][layer][table[seq, at // c["page"]], head, at % c["page"]]
            s[x][layer][table[seq, to // c["page"]], head, to % c["page"]] = moved
    return [fresh.int(), s["weights_out"], s["keys"], s["values"]]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, kind = case, case["kind"]
    row = 2 * 2 * c["kv_heads"] * c["dim"]      # a key and a value
    lengths, new = _lengths(c)
    if kind == "evict":
        total, moved = 0, 0.0
        for n in lengths:
            total += n + min(n, c["budget"])
            if n > c["budget"]:
                old, heavy = n - c["recent"], c["budget"] - c["recent"]
                moved += c["recent"] + heavy * (old - heavy) / old
        return dict(bytes=int(c["layers"] * (4 * c["kv_heads"] * total + 2 * moved * row)), flops=0)
    q = 2 * c["heads"] * c["dim"]
    if kind == "append":
        table = 2 * (2 if c["table"] == "f16" else 4) * c["rotary"] // 2
        heads = c["heads"] + c["kv_heads"]
        return dict(bytes=sum(new) * (2 * row + 2 * q) + min(sum(new), max(a + b for a, b in zip(lengths, new))) * table + (4 * sum(new) * c["axes"] if c["axes"] > 1 else 0),
                    flops=sum(new) * heads * (3 * c["rotary"] + (4 * c["dim"] if c["norm"] else 0)))
    tree = c.get("tree", False)
    seen = [a + b / 2 if tree else a + (b + 1) / 2 for a, b in zip(lengths, new)]
    flops = sum(4 * c["heads"] * c["dim"] * b * k for b, k in zip(new, seen))
    rows = sum(a + b for a, b in zip(lengths, new))
    if kind == "prefix":
        rows -= c["prefix"] // c["page"] * c["page"] * c["groups"] * (c["seqs"] - 1)
        return dict(bytes=rows * row + 2 * sum(new) * q, flops=flops)
    return dict(bytes=rows * (row + 8 * c["kv_heads"]) + 2 * sum(new) * q, flops=flops)


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "prefix": _exact_attention, "weights": _exact_attention, "evict": _exact_evict}[case["kind"]](case, s)


def _exact_append(c, s):
    keys, values, q_out = s["keys"].double(), s["values"].double(), s["q"].double()
    k_in, v_in = s["k"].double(), s["v"].double()
    half = c["rotary"] // 2
    first = torch.arange(half, device="cuda") * (2 if c["neighbours"] else 1)
    second = first + (1 if c["neighbours"] else half)
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for i, before in enumerate(lengths):
        a, b = starts[i], starts[i + 1]
        at = torch.arange(before, before + b - a, device="cuda")
        cos, sin = torch.empty((b - a, half), dtype=F64, device="cuda"), torch.empty((b - a, half), dtype=F64, device="cuda")
        for j in range(half):
            p = at if s["positions"] is None else s["positions"][s["pair_axis"][j], a:b].long()
            cos[:, j], sin[:, j] = s["cos"][p, j].double(), s["sin"][p, j].double()
        turned = {}
        for name, x, w in (("q", q_out[a:b], s["q_norm"]), ("k", k_in[a:b], s["k_norm"])):
            if w is not None:
                x = x / torch.sqrt(x.pow(2).sum(2, keepdim=True) / c["dim"] + EPS) * w.double()
            y = x.clone()
            y[..., first] = x[..., first] * cos[:, None] - x[..., second] * sin[:, None]
            y[..., second] = x[..., second] * cos[:, None] + x[..., first] * sin[:, None]
            turned[name] = y
        q_out[a:b] = turned["q"]
        pages, slots = s["table"][i].long()[at // c["page"]], at % c["page"]
        for h in range(c["kv_heads"]):
            keys[0, pages, h, slots] = turned["k"][:, h]
            values[0, pages, h, slots] = v_in[a:b, h]
    return [q_out, keys, values]


def _exact_attention(c, s):
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    out = torch.zeros(s["q"].shape, dtype=F64, device="cuda")
    sums = s["weights"].double() if c["kind"] == "weights" else None
    per = c["heads"] // c["kv_heads"]
    for i, before in enumerate(lengths):
        a, b = starts[i], starts[i + 1]
        n, end = b - a, before + b - a
        pages = s["table"][i, :-(-end // c["page"])].long()
        sees = torch.ones((n, end), dtype=torch.bool, device="cuda")
        if s["mask"] is None:
            sees[:, before:] = torch.ones((n, n), device="cuda").tril().bool()
        else:
            for j in range(n):
                sees[:, before + j] = (s["mask"][a:b, j // 64] >> (j % 64)) & 1 == 1
        for g in range(c["kv_heads"]):
            k, v = (s[x][0, pages, g].reshape(-1, c["dim"])[:end].double() for x in ("keys", "values"))
            if sums is not None:
                sums[i, g, before:end] = 0
            for h in range(g * per, g * per + per):
                score = (s["q"][a:b, h].double() @ k.T / math.sqrt(c["dim"])).masked_fill(~sees, -math.inf)
                e = torch.exp(score - score.max(1, keepdim=True).values.clamp(min=-1e300))
                e = e / e.sum(1, keepdim=True).clamp(min=1e-300)
                out[a:b, h] = e @ v
                if sums is not None:
                    sums[i, g, :end] += e.sum(0)
    return out if sums is None else [out, sums]


def _exact_evict(c, s):
    keys, values, weights = s["keys"].double(), s["values"].double(), s["weights_out"].double()
    heavy = c["budget"] - c["recent"]
    for i, n in enumerate(s["lengths"].tolist()):
        pages = s["table"][i].long()
        for layer in range(c["layers"]):
            for h in range(c["kv_heads"]):
                w = s["weights"][layer, i, h, :n].double()
                if n <= c["budget"]:
                    weights[layer, i, h, :n] = w
                    continue
                best = torch.sort(w[:n - c["recent"]], descending=True, stable=True).indices[:heavy]
                place = torch.full((heavy,), -1, dtype=torch.long, device="cuda")
                at_home = best[best < heavy]
                place[at_home] = at_home
                place[place < 0] = best[best >= heavy].sort().values
                source = torch.cat([place, torch.arange(n - c["recent"], n, device="cuda")])
                to = torch.arange(c["budget"], device="cuda")
                weights[layer, i, h, :c["budget"]] = w[source]
                for x in (keys, values):
                    x[layer, pages[to // c["page"]], h, to % c["page"]] = x[layer, pages[source // c["page"]], h, source % c["page"]]
    return [None, weights, keys, values]
