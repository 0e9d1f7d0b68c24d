"""A cache of keys and values in pages, and what a server does with it between two forwards: operators that are measured one by one.

  append    keys and values of new tokens into the pages, keys (and the queries beside them) rotated on the way (ops.paged_append)
  attention new tokens, a tree of drafted ones or one each, over the pages (ops.paged_attention)
  keep      the accepted path of a drafted tree moves up behind the rows it continues, in every layer (ops.paged_keep)
  select    the best continuations of a group of beams over beams and vocabulary (ops.beam_select)
  reorder   the beams take their parents' pages, in every layer (ops.paged_reorder)

A page table row lists the pages of a sequence in order; row r of a sequence lies in its page r // page_size. Lengths count the
rows before the new tokens. Heads, widths, layers and vocabularies are those of bench.py (32 and 16 query heads, 8 key / value heads of 128,
28 and 32 layers, vocabularies of 32768, 128256 and 151936) or generic.

With `own` false, run() computes the operators in elementary torch operations, in 32 bits (scores of beams in 64: they decide an order)."""
import functools
import math
import random
import zlib

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
F64 = torch.float64


# ------------------------------------------------------------------------------------------------ the cases
def _append(name, seqs, new, **more):
    return dict(dict(name=name, kind="append", seqs=seqs, new=new, before=0, heads=32, kv_heads=8, dim=128, page=64, rotary=128, neighbours=False, table="f16",
                     dtype="f16"), **more)


def _attention(name, seqs, ctx, new, **more):
    return dict(dict(name=name, kind="attention", seqs=seqs, ctx=ctx, new=new, tree=new > 1, heads=32, kv_heads=8, dim=128, page=64, dtype="f16"), **more)


def _keep(name, seqs, new, accepted, layers, **more):
    return dict(dict(name=name, kind="keep", seqs=seqs, ctx=200, new=new, accepted=accepted, layers=layers, kv_heads=8, dim=128, page=64, dtype="f16"), **more)


def _select(name, groups, beams, vocab, picks, **more):
    return dict(dict(name=name, kind="select", groups=groups, beams=beams, vocab=vocab, picks=picks, finished=0, dtype="f32"), **more)


def _reorder(name, groups, beams, parents, layers, **more):
    return dict(dict(name=name, kind="reorder", groups=groups, beams=beams, parents=parents, layers=layers, ctx=150, kv_heads=8, dim=128, page=32, dtype="f16"), **more)


def listed():
    return [
        # one token of each of 32 sequences that a server decodes together: latency
        _append("append_decode_32", 32, 1, before=900, spread=True),
        # eight prompts of different lengths in one forward
        _append("append_prompts", 8, 1900, dtype="bf16", table="f32"),
        # one user, one token, a short context: latency
        _attention("attend_one_token", 1, 600, 1),
        # a server's decode batch, lengths from an eighth of the longest up
        _attention("attend_decode_32", 32, 8192, 1),
        # drafted trees of eight users, 26 nodes each
        _attention("attend_trees_8", 8, 4001, 26, page=48, dtype="bf16"),
        # a tree of 64 nodes behind a long document
        _attention("attend_tree_long", 1, 100003, 64, dtype="bf16"),
        # one user's tree: four of its 26 nodes were right
        _keep("keep_one", 1, 26, 4, 28),
        # 64 users, trees of 64 nodes, up to eight accepted
        _keep("keep_64", 64, 64, 8, 32, dtype="bf16"),
        # a beam search of four over a small vocabulary in half precision: latency
        _select("select_4", 1, 4, 32768, 4, dtype="f16"),
        # 32 searches of eight beams over a large one, twice as many picks as beams, some beams finished
        _select("select_32x8", 32, 8, 128256, 16, finished=1),
        # the four beams of one search: three are continued
        _reorder("reorder_4", 1, 4, 3, 28),
        # eight searches of eight beams: half of them are continued
        _reorder("reorder_8x8", 8, 8, 4, 32, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "keep", "select", "select", "reorder"])
    dtype = rng.choice(["f16", "bf16"])
    dim = rng.choice([64, 128, 128, 256])
    heads, kv_heads = rng.choice([(32, 8), (16, 8), (8, 8), (12, 2), (10, 2), (28, 4), (16, 1), (9, 3)])
    page = rng.choice([16, 32, 64, 128, rng.randint(5, 200)])
    if kind == "append":
        new = rng.choice([1, 1, _log(rng, 2, 1500)])
        return _append(None, _log(rng, 1, max(1, min(200, 9000 // new))), new, before=rng.choice([0, _log(rng, 1, 500)]), heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                       rotary=rng.choice([dim, dim // 2]), neighbours=rng.random() < 0.3, table=rng.choice(["f16", "f32"]), dtype=dtype, spread=rng.random() < 0.5)
    if kind == "attention":
        tree = rng.random() < 0.5
        new = _log(rng, 2, 128) if tree else rng.choice([1, 1, 1, _log(rng, 2, 300)])
        # no more rows than the largest listed case reads, and no more products
        rows = min(32 * 5000 * 1024, 64 * 32 * 100003 * 128 // (new * heads // kv_heads)) // (kv_heads * dim)
        seqs = _log(rng, 1, 48)
        return _attention(None, seqs, _log(rng, 1, max(2, min(120000, rows // seqs))), new, tree=tree, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if kind == "keep":
        new = _log(rng, 2, 64)
        return _keep(None, _log(rng, 1, 64), new, rng.randint(1, min(8, new)), rng.randint(1, 32), ctx=_log(rng, 1, 400), kv_heads=rng.choice([1, 2, 3, 8]), dim=rng.choice([64, 128]),
                     page=page, dtype=dtype)
    if kind == "select":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        vocab = _log(rng, 500, 152000)
        groups = _log(rng, 1, max(1, min(64, 32 * 8 * 128256 // (beams * vocab))))
        return _select(None, groups, beams, vocab, rng.choice([1, 2]) * beams, finished=rng.choice([0, rng.randint(0, beams - 1)]), dtype=rng.choice(["f16", "bf16", "f32", "f32"]))
    beams = rng.choice([2, 3, 4, 5, 8])
    return _reorder(None, _log(rng, 1, 8), beams, rng.randint(1, beams), rng.randint(1, 32), ctx=_log(rng, 1, 500), kv_heads=rng.choice([1, 2, 3, 8]), dim=rng.choice([64, 128]),
                    page=rng.choice([16, 32, 64, rng.randint(5, 64)]), dtype=dtype)


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
    n = c["seqs"]
    if c["kind"] == "append":
        new = _spread(n, c["new"])
        return (_spread(n, c["before"], 0) if c.get("spread") else [c["before"]] * n), new
    if c["kind"] == "attention":
        return _spread(n, c["ctx"]), (_spread(n, c["new"]) if n > 1 and not c["tree"] else [c["new"]] * n)
    return _spread(n, c["ctx"]), [c["new"]] * n


def _counts(c):
    """Accepted nodes of every sequence."""
    r = random.Random(c["seqs"] * 31 + c["accepted"])
    return [c["accepted"] if i == 0 else r.randint(0, c["accepted"]) for i in range(c["seqs"])]


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
    if kind == "select":
        shape = (c["groups"], c["beams"], c["vocab"])
        logits = _randn(seed, "logits", *shape) * 2
        best = torch.randint(c["vocab"], (c["groups"], c["beams"], 12), generator=_gen(seed, "best"), device="cuda")
        logits.scatter_add_(2, best, 6 + 6 * torch.rand(best.shape, generator=_gen(seed, "lift"), device="cuda"))
        s.update(logits=logits.to(DT[c["dtype"]]), scores=-20 * torch.rand((c["groups"], c["beams"]), generator=_gen(seed, "scores"), device="cuda"))
        order = torch.rand((c["groups"], c["beams"]), generator=_gen(seed, "done"), device="cuda").argsort(1)
        s["done"] = (order < c["finished"]) if c["finished"] else None
        if own:
            s["dev"] = _device()
        return s
    if kind == "reorder":
        n, before = c["groups"] * c["beams"], _spread(c["groups"], c["ctx"])
        lengths = [k for k in before for _ in range(c["beams"])]
        keys, values, table = _pages(c, seed, [k // c["page"] + 1 for k in lengths], c["layers"])
        for g in range(c["groups"]):   # the full pages are the prompt's, shared by the group
            at, full = g * c["beams"], before[g] // c["page"]
            table[at:at + c["beams"], :full] = table[at, :full]
        draw_ = torch.rand((c["groups"], c["beams"]), generator=_gen(seed, "parents"), device="cuda").argsort(1)[:, :c["parents"]]
        more = torch.randint(c["parents"], (c["groups"], c["beams"] - c["parents"]), generator=_gen(seed, "more"), device="cuda")
        parents = torch.cat([draw_, draw_.gather(1, more)], 1)
        mixed = torch.rand(parents.shape, generator=_gen(seed, "mix"), device="cuda").argsort(1)
        s["parents"] = parents.gather(1, mixed).reshape(n).int()
    else:
        before, new = _lengths(c)
        lengths = before
        room = [-(-(a + b) // c["page"]) for a, b in zip(before, new)]
        keys, values, table = _pages(c, seed, room, c.get("layers", 1))
        s["starts"], s["new"] = _ints(_starts(new)), max(new)
        total = sum(new)
        if kind == "append":
            # one row per token as the projection leaves it: queries, keys, values
            qkv = _randn(seed, "qkv", total, c["heads"] + 2 * c["kv_heads"], c["dim"]).to(DT[c["dtype"]])
            s["q"], s["k"], s["v"] = qkv.split([c["heads"], c["kv_heads"], c["kv_heads"]], 1)
            s["cos"], s["sin"] = _rotation_table(c, max(a + b for a, b in zip(before, new)))
        elif kind == "attention":
            s["q"] = _randn(seed, "q", total, c["heads"], c["dim"]).to(DT[c["dtype"]])
            s["mask"] = _tree(seed, c["new"], c["seqs"]) if c["tree"] else None
            s["longest"] = max(a + b for a, b in zip(before, new))
        else:
            # places of the accepted path: the first nodes, then some of the deeper ones
            r, counts, rows = random.Random(seed), _counts(c), []
            for k in counts:
                stay = r.randint(0, k)
                rows.append(list(range(stay)) + sorted(r.sample(range(min(k, c["new"] - (k - stay)), c["new"]), k - stay)) + [0] * (c["accepted"] - k))
            s["accepted"], s["counts"] = _ints(rows), _ints(counts)
    s.update(keys=keys, values=values, table=table, lengths=_ints(lengths))
    if own:
        from ironmill_b200 import ops
        s["kv"] = ops.PagedKV(_device(), keys, values, table, s["lengths"])
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"append": _run_append, "attention": _run_attention, "keep": _run_keep, "select": _run_select, "reorder": _run_reorder}[state["case"]["kind"]](state)


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
        q = ops.paged_append(s["kv"], 0, s["k"], s["v"], s["starts"], q=s["q"], cos=s["cos"], sin=s["sin"], rotary_dim=c["rotary"], neighbours=c["neighbours"])
        return [q, s["keys"], s["values"]]
    seq, place = _places(s, s["k"].shape[0])
    row = s["lengths"].long()[seq] + place
    cos, sin = s["cos"][row, :c["rotary"] // 2], s["sin"][row, :c["rotary"] // 2]
    q, k = (_rotated(s[x].float(), cos, sin, c["rotary"], c["neighbours"]).to(s[x].dtype) for x in ("q", "k"))
    page, slot = s["table"].long()[seq, row // c["page"]], row % c["page"]
    s["keys"][0][page, :, slot] = k
    s["values"][0][page, :, slot] = s["v"]
    return [q, s["keys"], s["values"]]


def _run_attention(s):
    c = s["case"]
    scale = c["dim"] ** -0.5
    if own:
        from ironmill_b200 import ops
        return ops.paged_attention(s["kv"], 0, s["q"], s["starts"], s["new"], scale, mask=s["mask"], max_len=s["longest"])
    total, groups = s["q"].shape[0], c["heads"] // c["kv_heads"]
    seq, place = _places(s, total)
    row = torch.arange(s["longest"], device="cuda")
    page, slot = s["table"].long()[:, row // c["page"]], (row % c["page"])[None]
    k, v = (s[x][0][page, :, slot].float().transpose(1, 2) for x in ("keys", "values"))      # [sequences, key heads, rows, dim]
    ahead = row[None] - s["lengths"][seq, None]                                               # [tokens, rows]: place among the new rows
    fits = ahead < (s["starts"][1:] - s["starts"][:-1])[seq, None]
    if s["mask"] is None:
        seen = ahead <= place[:, None]
    else:
        word = (ahead.clamp(min=0) // 64).clamp(max=s["mask"].shape[1] - 1)
        seen = (ahead < 0) | ((s["mask"].gather(1, word) >> (ahead.clamp(min=0) % 64)) & 1).bool()
    q = torch.zeros((c["seqs"], s["new"], c["kv_heads"], groups, c["dim"]), device="cuda")
    see = torch.zeros((c["seqs"], s["new"], s["longest"]), dtype=torch.bool, device="cuda")
    q[seq, place] = s["q"].float().view(total, c["kv_heads"], groups, c["dim"])
    see[seq, place] = seen & fits
    score = torch.matmul(q.permute(0, 2, 3, 1, 4).flatten(2, 3), k.transpose(2, 3)).unflatten(2, (groups, s["new"])) * scale
    score = torch.where(see[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    sums = weight.sum(-1, keepdim=True)
    out = torch.matmul((weight / torch.where(sums == 0, 1.0, sums)).flatten(2, 3), v).unflatten(2, (groups, s["new"]))
    return out.permute(0, 3, 1, 2, 4)[seq, place].reshape(total, c["heads"], c["dim"]).to(DT[c["dtype"]])


def _run_keep(s):
    c = s["case"]
    if own:
        from ironmill_b200 import ops
        return [ops.paged_keep(s["kv"], s["accepted"], s["counts"]), s["keys"], s["values"]]
    live = torch.arange(c["accepted"], device="cuda")[None] < s["counts"][:, None]
    seq, j = live.nonzero(as_tuple=True)
    start = s["lengths"].long()[seq]
    source, to = start + s["accepted"].long()[seq, j], start + j
    table = s["table"].long()
    for x in ("keys", "values"):
        rows = s[x][:, table[seq, source // c["page"]], :, source % c["page"]]
        s[x][:, table[seq, to // c["page"]], :, to % c["page"]] = rows
    return [s["lengths"] + s["counts"], s["keys"], s["values"]]


def _run_select(s):
    c = s["case"]
    if own:
        from ironmill_b200 import ops
        return list(ops.beam_select(s["dev"], s["logits"], s["scores"], c["picks"], done=s["done"], end_token=2))
    x = s["logits"].double()
    x = x - x.amax(-1, keepdim=True)
    value = s["scores"].double()[..., None] + x - torch.log(torch.exp(x).sum(-1, keepdim=True))
    if s["done"] is not None:      # a finished beam has one continuation, its end token at no cost
        alone = torch.where(torch.arange(c["vocab"], device="cuda") == 2, s["scores"].double()[..., None], -math.inf)
        value = torch.where(s["done"][..., None], alone, value)
    value, at = value.flatten(1).sort(dim=1, descending=True, stable=True)
    value, at = value[:, :c["picks"]], at[:, :c["picks"]]
    return [value.float(), (at // c["vocab"]).int(), (at % c["vocab"]).int()]


def _run_reorder(s):
    c = s["case"]
    if own:
        from ironmill_b200 import ops
        table, lengths = ops.paged_reorder(s["kv"], s["parents"], c["beams"])
        return [table, lengths, s["keys"], s["values"]]
    n, beams = s["parents"].shape[0], c["beams"]
    each = torch.arange(n, device="cuda")
    source = each // beams * beams + s["parents"].long()
    lengths = s["lengths"][source]
    # the first child of a parent keeps its last page; the others take those of the beams without a child, in order
    same = (source.view(-1, beams, 1) == source.view(-1, 1, beams)).tril(-1).any(-1)                      # an earlier beam has this parent
    childless = ~(source.view(-1, 1, beams) == each.view(-1, beams, 1)).any(-1)
    free = torch.argsort(~childless, dim=1, stable=True)                                                  # the childless first
    rank = torch.cumsum(same, 1) - 1
    giver = (each.view(-1, beams)[:, :1] + free.gather(1, rank.clamp(min=0))).flatten()
    last, old = (lengths // c["page"]).long(), (s["lengths"] // c["page"]).long()
    own_page = s["table"].gather(1, old[:, None])[:, 0]
    table = s["table"][source].clone()
    copied = same.flatten()
    page_from = table.gather(1, last[:, None])[:, 0]
    page_to = torch.where(copied, own_page[giver], page_from)
    table.scatter_(1, last[:, None], page_to[:, None])
    beam, slot = (copied[:, None] & (torch.arange(c["page"], device="cuda")[None] < (lengths % c["page"])[:, None])).nonzero(as_tuple=True)
    for x in ("keys", "values"):
        s[x][:, page_to.long()[beam], :, slot] = s[x][:, page_from.long()[beam], :, slot]
    return [table, lengths, s["keys"], s["values"]]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, kind = case, case["kind"]
    if kind == "select":
        n = c["groups"] * c["beams"] * c["vocab"]
        return dict(bytes=n * torch.finfo(DT[c["dtype"]]).bits // 8 + 12 * c["groups"] * c["picks"], flops=4 * n)
    row = 2 * 2 * c["kv_heads"] * c["dim"]      # a key and a value
    if kind == "reorder":
        moved = sum((c["beams"] - c["parents"]) * (k % c["page"]) for k in _spread(c["groups"], c["ctx"]))
        table = sum(c["beams"] * (k // c["page"] + 1) for k in _spread(c["groups"], c["ctx"]))
        return dict(bytes=2 * moved * row * c["layers"] + 8 * table + 12 * c["groups"] * c["beams"], flops=0)
    before, new = _lengths(c)
    if kind == "keep":
        return dict(bytes=2 * sum(_counts(c)) * row * c["layers"] + 4 * sum(_counts(c)) + 12 * c["seqs"], flops=0)
    q = 2 * c["heads"] * c["dim"]
    if kind == "append":
        table = 2 * (2 if c["table"] == "f16" else 4) * c["rotary"] // 2
        return dict(bytes=sum(new) * (2 * row + 2 * q) + min(sum(new), max(a + b for a, b in zip(before, new))) * table, flops=3 * sum(new) * (c["heads"] + c["kv_heads"]) * c["rotary"])
    seen = [a + b / 2 if c["tree"] else a + (b + 1) / 2 for a, b in zip(before, new)]
    return dict(bytes=sum(a + b for a, b in zip(before, new)) * row + 2 * sum(new) * q, flops=sum(4 * c["heads"] * c["dim"] * b * k for b, k in zip(new, seen)))


# ------------------------------------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "keep": _exact_keep, "select": _exact_select, "reorder": _exact_reorder}[case["kind"]](case, s)


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
        cos, sin = s["cos"][at, None, :half].double(), s["sin"][at, None, :half].double()
        turned = {}
        for name, x in (("q", q_out[a:b]), ("k", k_in[a:b])):
            y = x.clone()
            y[..., first] = x[..., first] * cos - x[..., second] * sin
            y[..., second] = x[..., second] * cos + x[..., first] * sin
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
            for h in range(g * per, g * per + per):
                score = (s["q"][a:b, h].double() @ k.T / math.sqrt(c["dim"])).masked_fill(~sees, -math.inf)
                e = torch.exp(score - score.max(1, keepdim=True).values.clamp(min=-1e300))
                out[a:b, h] = (e @ v) / e.sum(1, keepdim=True).clamp(min=1e-300)
    return out


def _exact_keep(c, s):
    got = []
    for x in ("keys", "values"):
        old, new = s[x].double(), s[x].double()
        for i, (start, places, count) in enumerate(zip(s["lengths"].tolist(), s["accepted"].tolist(), s["counts"].tolist())):
            pages = s["table"][i].tolist()
            for j in range(count):
                r, t = start + places[j], start + j
                new[:, pages[t // c["page"]], :, t % c["page"]] = old[:, pages[r // c["page"]], :, r % c["page"]]
        got.append(new)
    return [None] + got


def _exact_select(c, s):
    best = []
    for g in range(c["groups"]):
        x = s["logits"][g].double()
        value = s["scores"][g].double()[:, None] + torch.log_softmax(x, -1)
        if s["done"] is not None:
            value[s["done"][g]] = -math.inf
            value[:, 2] = torch.where(s["done"][g], s["scores"][g].double(), value[:, 2])
        best.append(value.flatten().topk(c["picks"]).values)
    return [torch.stack(best), None, None]


def _exact_reorder(c, s):
    lengths, parents = s["lengths"].tolist(), s["parents"].tolist()
    keys, values = s["keys"].double(), s["values"].double()
    for g in range(0, len(parents), c["beams"]):
        taken = set(parents[g:g + c["beams"]])
        free = [g + p for p in range(c["beams"]) if p not in taken]
        met = set()
        for i in range(g, g + c["beams"]):
            p = g + parents[i]
            if p in met:
                d = free.pop(0)
                rows = lengths[p] % c["page"]
                a, b = int(s["table"][p, lengths[p] // c["page"]]), int(s["table"][d, lengths[d] // c["page"]])
                for x in (keys, values):
                    x[:, b, :, :rows] = x[:, a, :, :rows]
            met.add(p)
    return [None, None, keys, values]
