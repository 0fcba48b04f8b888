"""The streaming and masked attention operators and the page operators of their cache, as a user's program calls them.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits), or, where ``own`` is true, through
the package's entry points.  ``exact`` gives the same outputs from the definitions in 64 bits.

Formulas.  Scores x_ij = scale q_i . k_j, capped as c tanh(x / c) where a cap is given, plus the log-mass of key j, minus
slope_h |pos_i - pos_j|; row i sees the keys [begin_i, end_i) and o_i is the softmax-weighted mean of their values, zero when
it sees none.  The cache keeps the keys, values and log-masses of every stream in pages of ``page`` tokens; pages are taken
lowest number first, a shared last page is copied before it is written, and compaction moves the j-th live page beyond the
live count into the j-th free page below it.
"""
import importlib
import math
import random
import zlib

import torch

own = False

HEAD = 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _package():
    return importlib.import_module("4d_ttt_merging_b200")


# ---------------------------------------------------------------- cases

def _masked(name, **k):
    c = dict(op="masked", batch=1, heads=16, kv_heads=16, queries=1029, keys=1029, dtype="bf16", documents=1, step=0,
             prefix=0, window=0, mass=True, softcap=0.0, slope=False)
    c.update(k)
    return dict({"name": name}, **c) if name else c


def _paged(name, **k):
    c = dict(op="paged", streams=1, new_low=1, new_high=1, past_low=300, past_high=300, heads=16, kv_heads=16, page=64,
             dtype="bf16", causal=True, mass=True, softcap=0.0, slope=False)
    c.update(k)
    return dict({"name": name}, **c) if name else c


def _cache(name, **k):
    c = dict(op="append", streams=8, new_low=1029, new_high=1029, past_low=0, past_high=0, kv_heads=16, page=64,
             dtype="bf16", mass=True)
    c.update(k)
    return dict({"name": name}, **c) if name else c


def listed():
    return [
        # the 17 camera and register tokens of a frame over that frame's 1041 tokens, shared key heads, distance bias:
        # the smallest call, where latency counts
        _masked("special tokens f32", queries=17, keys=1041, kv_heads=4, dtype="f32", mass=False, slope=True),
        # four clips of merged tokens packed into one call, frame groups of 1029 merged tokens in causal order
        _masked("packed clips bf16", queries=8232, keys=8232, documents=4, step=1029),
        # four frames' queries over the merged keys of 256 frames, capped scores: the largest call
        _masked("long clip capped f16", queries=4116, keys=32928, dtype="f16", softcap=30.0),
        # one stream, one new token, a short past
        _paged("one token bf16", past_low=300, past_high=300, page=16),
        # 32 streams, one token each, ragged pasts
        _paged("32 streams bf16", streams=32, past_low=500, past_high=9000),
        # a new frame of 1041 tokens over the merged tokens of 256 frames
        _paged("frame over 32928 bf16", new_low=1041, new_high=1041, past_low=32928, past_high=32928, causal=False),
        # ragged chunks, shared key heads, cap and distance bias
        _paged("ragged chunks f16", streams=6, new_low=1, new_high=700, past_low=0, past_high=12000, kv_heads=4, page=32,
               dtype="f16", softcap=50.0, slope=True),
        # eight streams end and eight new ones take their slots with a merged frame group each
        _cache("new streams bf16", streams=8, new_low=900, new_high=1100),
        # a shared past of one frame branches into four streams of 17 tokens
        _cache("four branches bf16", op="branch", streams=4, new_low=17, new_high=17, past_low=1041, past_high=1041),
        # a shared past of 32 frames branches into 64 streams of a ragged chunk
        _cache("64 branches bf16", op="branch", streams=64, new_low=1, new_high=257, past_low=8237, past_high=8237),
        # a small pool with holes is made dense
        _cache("compact 16 streams f32", op="compact", streams=16, past_low=100, past_high=700, page=16, kv_heads=4,
               dtype="f32"),
        # a large pool with holes is made dense
        _cache("compact 64 streams bf16", op="compact", streams=64, past_low=500, past_high=4000),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["masked", "masked", "paged", "paged", "append", "branch", "compact"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "masked":
        heads = rng.choice([1, 2, 4, 8, 12, 16])
        kv = rng.choice([h for h in (1, 2, 4, 8, 12, 16) if heads % h == 0])
        most = 4200 if dtype == "f32" else 16464  # a pass costs at most what the largest listed one does
        keys = _spread(rng, 1, most)
        queries = rng.choice([keys, _spread(rng, 1, keys)])
        batch = rng.choice([1, 1, 2, 3]) if keys < 4200 else 1
        return _masked(None, batch=batch, heads=heads, kv_heads=kv, queries=min(queries, 2100 if dtype == "f32" else 8200),
                       keys=keys, dtype=dtype, documents=rng.choice([1, 1, 2, 5]), step=rng.choice([0, 1, 17, 257, 1029]),
                       prefix=rng.choice([0, 0, 5, 130]), window=rng.choice([0, 0, 0, 100, 900]), mass=rng.random() < 0.6,
                       softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), slope=rng.random() < 0.3)
    page = rng.choice([16, 32, 64, 128])
    kv = rng.choice([1, 2, 4, 8, 16])
    if kind == "paged":
        streams = _spread(rng, 1, 32)
        new = rng.choice([1, 1, _spread(rng, 1, 1041 if streams < 5 else 200)])
        past = _spread(rng, 1, 32928 if streams * new < 1100 and streams < 8 else 6000)
        if dtype == "f32":
            past = min(past, 4000)
        return _paged(None, streams=streams, new_low=max(1, new // rng.choice([1, 3])), new_high=new, past_low=past // rng.choice([1, 2, 9]),
                      past_high=past, heads=kv * rng.choice([1, 1, 2, 4]) if kv < 8 else kv, kv_heads=kv, page=page, dtype=dtype,
                      causal=rng.random() < 0.6, mass=rng.random() < 0.6, softcap=rng.choice([0.0, 0.0, 30.0]), slope=rng.random() < 0.3)
    streams = _spread(rng, 1, 64)
    past = _spread(rng, 1, 1500 if dtype == "f32" else 4000)
    new = _spread(rng, 1, 1100 if streams < 16 else 257)
    return _cache(None, op=kind, streams=streams, new_low=max(1, new // 2), new_high=new, past_low=past // 2, past_high=past, kv_heads=kv,
                  page=page, dtype=dtype, mass=rng.random() < 0.6)


# ---------------------------------------------------------------- layouts: functions of the case alone

def _rng(case):
    return random.Random(zlib.crc32(repr(sorted((k, v) for k, v in case.items() if k != "name")).encode()))


def _documents(case):
    """Ragged document offsets over the keys."""
    rng, keys = _rng(case), case["keys"]
    cuts = sorted(min(keys, max(0, round(keys * (d + rng.uniform(-0.3, 0.3)) / case["documents"]))) for d in range(1, case["documents"]))
    return [0] + cuts + [keys]


def _ranges(case):
    """[queries, 2] visible keys of each row; the queries are the last tokens of the keys."""
    cut = torch.tensor(_documents(case))
    token = torch.arange(case["keys"] - case["queries"], case["keys"])
    at = torch.searchsorted(cut[1:], token, right=True).clamp(max=len(cut) - 2)
    start, stop = cut[at], cut[at + 1]
    begin, end = start, stop
    if case["step"]:
        end = torch.minimum(stop, start + ((token - start) // case["step"] + 1) * case["step"])
    if case["prefix"]:
        end = torch.maximum(end, torch.minimum(stop, start + case["prefix"]))
    if case["window"]:
        begin = torch.maximum(start, token - case["window"] + 1)
    return torch.stack([begin, end], 1).to(torch.int32)


def _lengths(case):
    """(new, past) tokens of each stream."""
    rng = _rng(case)
    return ([rng.randint(case["new_low"], case["new_high"]) for _ in range(case["streams"])],
            [rng.randint(case["past_low"], case["past_high"]) for _ in range(case["streams"])])


def _pages(tokens, page):
    return -(-tokens // page)


# ---------------------------------------------------------------- inputs

def _normal(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device="cuda").mul_(scale).to(dtype)


def _masses(g, shape):
    return torch.randint(1, 9, shape, generator=g, device="cuda").float().log()


def _slopes(heads):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda")


def _pool(case, g, held, spare, slots, perm_seed, contiguous=False):
    """A pool whose slot i holds held[i] tokens on pages in a shuffled order, with ``spare`` free pages."""
    page, dtype = case["page"], DTYPES[case["dtype"]]
    counts = [_pages(h, page) for h in held]
    pages = sum(counts) + spare
    order = list(range(pages))
    random.Random(perm_seed).shuffle(order)
    used = order[:sum(counts)]
    width = max(1, max(slots["width"], max(counts, default=0)))
    table = torch.full((slots["count"], width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = torch.tensor(used[at:at + n], dtype=torch.int32)
        at += n
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[torch.tensor(used, dtype=torch.long)] = 1
    length = torch.zeros(slots["count"], dtype=torch.int32)
    length[:len(held)] = torch.tensor(held, dtype=torch.int32)
    shape = (pages, page, case["kv_heads"], HEAD)
    return dict(k=_normal(g, shape, dtype), v=_normal(g, shape, dtype), mass=_masses(g, (pages, page)) if case["mass"] else None,
                table=table.cuda(), length=length.cuda(), refs=refs.cuda())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "masked":
        B, Hq, Hk, Nq, Nk = (case[n] for n in ("batch", "heads", "kv_heads", "queries", "keys"))
        s.update(q=_normal(g, (B, Nq, Hq, HEAD), dtype, 2.0).transpose(1, 2), k=_normal(g, (B, Nk, Hk, HEAD), dtype).transpose(1, 2),
                 v=_normal(g, (B, Nk, Hk, HEAD), dtype).transpose(1, 2), mass=_masses(g, (Nk,)) if case["mass"] else None,
                 ranges=_ranges(case).cuda(), slope=_slopes(Hq) if case["slope"] else None)
        return s
    new, past = _lengths(case)
    page, n = case["page"], case["streams"]
    offsets = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    s.update(new=new, sequence=torch.arange(n, dtype=torch.int32, device="cuda"), offsets=offsets)
    if case["op"] == "paged":
        held = [a + b for a, b in zip(new, past)]
        s.update(_pool(case, g, held, 3, {"count": n, "width": 0}, seed), held=held,
                 q=_normal(g, (sum(new), case["heads"], HEAD), dtype, 2.0), slope=_slopes(case["heads"]) if case["slope"] else None)
        return s
    wide = (sum(new), 3 * case["kv_heads"] * HEAD)
    packed = _normal(g, wide, dtype).view(sum(new), 3, case["kv_heads"], HEAD)  # the packed q | k | v rows of a step
    s.update(new_k=packed[:, 1], new_v=packed[:, 2], new_mass=_masses(g, (sum(new),)) if case["mass"] else None)
    if case["op"] == "append":
        # the streams that end hold as much as the new ones; other streams hold pages between theirs
        held = new + [max(1, x // 2) for x in new]
        s.update(_pool(case, g, held, 5, {"count": 2 * n, "width": max(_pages(x, page) for x in new)}, seed))
    elif case["op"] == "branch":
        # slot 0 holds the shared past; slots 1.. are the branches, empty before the first pass
        root = past[0]
        spare = sum(_pages(root % page + x, page) for x in new) + 4
        s.update(_pool(case, g, [root], spare, {"count": n + 1, "width": max(_pages(root + x, page) for x in new)}, seed), root=root,
                 source=torch.zeros(n, dtype=torch.int32, device="cuda"), sequence=torch.arange(1, n + 1, dtype=torch.int32, device="cuda"))
    else:
        # every other stream has ended: its pages are holes
        held = [max(1, x) for x in past]
        s.update(_pool(case, g, held, 2, {"count": n, "width": 0}, seed))
        gone = torch.arange(0, n, 2, device="cuda")
        pages = s["table"][gone]
        s["refs"][pages[pages >= 0].long()] = 0
        s["table"][gone] = -1
        s["length"][gone] = 0
        s.update(start_table=s["table"].clone(), start_refs=s["refs"].clone())
    return s


# ---------------------------------------------------------------- one pass

def _cache_of(s):
    """The handle that a program keeps for its cache."""
    if "cache" not in s:
        s["cache"] = _package().PagedCache(s["k"], s["v"], s["mass"], s["table"], s["length"], s["refs"])
    return s["cache"]


def run(s):
    case = s["case"]
    op = case["op"]
    if op == "masked":
        if own:
            return _package().masked_attention(s["q"], s["k"], s["v"], s["mass"], key_range=s["ranges"], softcap=case["softcap"] or None,
                                               distance_slope=s["slope"])
        return _plain_masked(s)
    if op == "paged":
        if own:
            return _package().paged_attention(s["q"], _cache_of(s), s["sequence"], s["offsets"], causal=case["causal"],
                                              softcap=case["softcap"] or None, distance_slope=s["slope"])
        return _plain_paged(s)
    state = ("k", "v", "mass", "table", "length", "refs")
    if op == "compact":
        s["table"].copy_(s["start_table"])  # the bookkeeping of the pool with holes, for a pass like the one before
        s["refs"].copy_(s["start_refs"])
        used = _cache_of(s).compact() if own else _plain_compact(s)
        return [s[n] for n in state] + [used]
    if op == "append":
        if own:
            _cache_of(s).free(s["sequence"])
        else:
            _plain_free(s, s["sequence"])
    elif own:
        _cache_of(s).fork(s["source"], s["sequence"])
    else:
        _plain_fork(s, s["source"], s["sequence"])
    if own:
        _cache_of(s).append(s["sequence"], s["offsets"], s["new_k"], s["new_v"], s["new_mass"])
    else:
        _plain_append(s)
    return [s[n] for n in state]


# ---------------------------------------------------------------- plain forms

def _attend(q, k, v, bias, seen, softcap, slope, qpos, kpos, dtype):
    """q [b, h, n, d], k and v [b, g, m, d], bias [b or 1, m] or None, seen [b or 1, n, m]; in 32 bits, rounded at the end."""
    b, h, n, d = q.shape
    g, m = k.shape[1:3]
    x = torch.matmul(q.float().reshape(b, g, h // g, n, d) * (d ** -0.5), k.float()[:, :, None].transpose(-1, -2)).view(b, h, n, m)
    if softcap:
        x = x.div_(softcap).tanh_().mul_(softcap)
    if bias is not None:
        x += bias[:, None, None]
    if slope is not None:
        x -= slope[:, None, None] * (qpos[..., :, None] - kpos[..., None, :]).abs()
    hidden = ~seen[:, None]
    x.masked_fill_(hidden, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, g, h // g, n, m), v.float()[:, :, None]).view(b, h, n, d)
    return (o / total.masked_fill_(total == 0, 1.0)).to(dtype)


def _plain_masked(s):
    case = s["case"]
    Nq, Nk = case["queries"], case["keys"]
    key = torch.arange(Nk, device="cuda")
    seen = (key >= s["ranges"][:, :1]) & (key < s["ranges"][:, 1:])
    row = torch.arange(Nk - Nq, Nk, device="cuda")
    return _attend(s["q"], s["k"], s["v"], None if s["mass"] is None else s["mass"][None], seen[None], case["softcap"], s["slope"],
                   row.float(), key.float(), DTYPES[case["dtype"]])


def _plain_paged(s):
    """The streams' pages gathered into padded rows."""
    case = s["case"]
    n, page = case["streams"], case["page"]
    most, far = max(s["new"]), _pages(max(s["held"]), page) * page
    seq = s["sequence"].long()
    table = s["table"][seq, :far // page].clamp(min=0).long()
    take = lambda pool: pool[table].reshape(n, far, *pool.shape[2:])  # noqa: E731
    k, v = take(s["k"]).transpose(1, 2), take(s["v"]).transpose(1, 2)
    bias = None if s["mass"] is None else take(s["mass"])
    length, start = s["length"][seq], s["offsets"][:-1]
    count = s["offsets"][1:] - start
    i = torch.arange(most, device="cuda")
    at = (start[:, None] + i).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"][at].transpose(1, 2)  # [n, h, most, d]
    token = (length - count)[:, None] + i
    end = token + 1 if case["causal"] else length[:, None].expand(n, most)
    key = torch.arange(far, device="cuda")
    seen = (key < end[..., None]) & (key < length[:, None, None])
    o = _attend(q, k, v, bias, seen, case["softcap"], s["slope"], token[:, None].float(), key.float()[None, None], DTYPES[case["dtype"]])
    row = torch.arange(s["q"].shape[0], device="cuda")
    stream = torch.searchsorted(s["offsets"][1:].contiguous(), row.to(torch.int32), right=True)
    return o[stream, :, (row - start[stream]).long()]


def _drop(s, rows):
    """The pages of the table rows lose a reference."""
    s["refs"].index_add_(0, rows.clamp(min=0).reshape(-1).long(), -(rows >= 0).reshape(-1).to(torch.int32))


def _plain_free(s, seq):
    seq = seq.long()
    _drop(s, s["table"][seq])
    s["table"][seq] = -1
    s["length"][seq] = 0


def _plain_fork(s, source, target):
    source, target = source.long(), target.long()
    rows, length = s["table"][source], s["length"][source]
    _drop(s, s["table"][target])
    s["refs"].index_add_(0, rows.clamp(min=0).reshape(-1).long(), (rows >= 0).reshape(-1).to(torch.int32))
    s["table"][target] = rows
    s["length"][target] = length


def _plain_append(s):
    page = s["case"]["page"]
    seq, start = s["sequence"].long(), s["offsets"][:-1].long()
    table, length, refs = s["table"], s["length"], s["refs"]
    count = s["offsets"][1:].long() - start
    old = length[seq].long()
    have, want = (old + page - 1) // page, (old + count + page - 1) // page
    last = table[seq, (have - 1).clamp(min=0)].long()
    copy = (count > 0) & (old % page != 0) & (refs[last.clamp(min=0)] > 1)
    first = have - copy.long()
    need = want - first
    free = torch.argsort((refs != 0).to(torch.int8), stable=True)  # free pages first, lowest number first
    slot = torch.arange(table.shape[1], device="cuda")
    fresh = (slot >= first[:, None]) & (slot < want[:, None])
    rank = (need.cumsum(0) - need)[:, None] + slot - first[:, None]
    room = ((need.sum() <= (refs == 0).sum()) & (want <= table.shape[1]).all()).long()  # all or nothing
    fresh &= room.bool()
    pages = free[rank.clamp(0, len(free) - 1)]
    refs.index_add_(0, last.clamp(min=0), -(copy.long() * room).to(torch.int32))
    refs[pages[fresh]] = 1
    rows = table[seq]
    table[seq] = torch.where(fresh, pages.to(torch.int32), rows)
    length[seq] = (old + count * room).to(torch.int32)
    # the copied part of shared last pages, then the new tokens
    both = torch.nonzero(copy & room.bool())[:, 0]
    src, dst = last[both], table[seq[both], (have - 1)[both]].long()
    keep = torch.arange(page, device="cuda") < (old % page)[both, None]
    token = torch.arange(s["new_k"].shape[0], device="cuda")
    stream = torch.searchsorted(s["offsets"][1:].contiguous(), token.to(torch.int32), right=True)
    at = old[stream] + token - start[stream]
    where = table[seq[stream], (at // page).clamp(max=table.shape[1] - 1)].long()
    live = room.bool() & (token >= 0)
    for pool, rows in ((s["k"], s["new_k"]), (s["v"], s["new_v"]), (s["mass"], s["new_mass"])):
        if pool is not None:
            wide = keep.view(keep.shape + (1,) * (pool.ndim - 2))
            pool[dst] = torch.where(wide, pool[src], pool[dst])
            pool[where[live], (at % page)[live]] = rows[live]


def _plain_compact(s):
    refs = s["refs"]
    page = torch.arange(len(refs), device="cuda")
    live = refs > 0
    used = live.sum()
    move, hole = page[live & (page >= used)], page[~live & (page < used)]
    to = page.clone()
    to[move] = hole
    for pool in (s["k"], s["v"], s["mass"]):
        if pool is not None:
            pool[hole] = pool[move]
    refs[hole] = refs[move]
    refs[move] = 0
    table = s["table"]
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table))
    return used.to(torch.int32)[None]


# ---------------------------------------------------------------- work

def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    if case["op"] == "masked":
        r = _ranges(case).long()
        pairs = int((r[:, 1] - r[:, 0]).clamp(min=0).sum()) * case["batch"] * case["heads"]
        kv = case["batch"] * case["keys"] * case["kv_heads"] * HEAD * size * 2
        qo = case["batch"] * case["queries"] * case["heads"] * HEAD * size * 2
        return {"bytes": kv + qo + case["queries"] * 8 + (case["keys"] * 4 if case["mass"] else 0), "flops": 4 * HEAD * pairs}
    new, past = _lengths(case)
    token = case["kv_heads"] * HEAD * size * 2 + (4 if case["mass"] else 0)
    if case["op"] == "paged":
        pairs = sum(n * (n + p) - (n * (n - 1) // 2 if case["causal"] else 0) for n, p in zip(new, past)) * case["heads"]
        table = sum(_pages(n + p, case["page"]) for n, p in zip(new, past)) * 4
        return {"bytes": sum(n + p for n, p in zip(new, past)) * token + sum(new) * case["heads"] * HEAD * size * 2 + table,
                "flops": 4 * HEAD * pairs}
    if case["op"] == "append":
        return {"bytes": 2 * sum(new) * token + sum(_pages(n, case["page"]) for n in new) * 16, "flops": 0}
    if case["op"] == "branch":
        return {"bytes": 2 * (sum(new) + len(new) * (past[0] % case["page"])) * token + len(new) * _pages(past[0], case["page"]) * 16, "flops": 0}
    # compact: every other stream's pages are holes, live pages are spread over the pool: about half of the live ones move
    held = [_pages(max(1, p), case["page"]) for p in past]
    total, live = sum(held) + 2, sum(held[1::2])
    return {"bytes": max(1, round(2 * live * (total - live) / total) * case["page"] * token) + 8 * total, "flops": 0}


# ---------------------------------------------------------------- 64 bits, from the definitions

def _softmax_rows(q, k, v, bias, begin, end, softcap, slope, qpos, kpos):
    """One batch entry in 64 bits: q [h, n, d], k and v [g, m, d]."""
    h, n, d = q.shape
    g, m = k.shape[:2]
    out = torch.zeros(h, n, d, dtype=torch.float64, device=q.device)
    if not m or not n:
        return out
    j = torch.arange(m, device=q.device)
    sees = (j[None] >= begin[:, None]) & (j[None] < end[:, None])
    some = sees.any(1)
    for head in range(h):
        kk, vv = k[head // (h // g)].double(), v[head // (h // g)].double()
        x = torch.einsum("nd,md->nm", q[head].double(), kk) / math.sqrt(d)
        x = softcap * torch.tanh(x / softcap) if softcap else x
        x = x if bias is None else x + bias.double()[None]
        x = x if slope is None else x - float(slope[head]) * (qpos.double()[:, None] - kpos.double()[None]).abs()
        x = torch.where(sees, x, torch.full_like(x, -math.inf))
        w = torch.softmax(x[some], dim=1)
        out[head, some] = w @ vv
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "masked":
        Nq, Nk = case["queries"], case["keys"]
        pos = torch.arange(Nk, device="cuda")
        begin, end = s["ranges"].long().unbind(1)
        return torch.stack([_softmax_rows(s["q"][b], s["k"][b], s["v"][b], s["mass"], begin, end, case["softcap"], s["slope"],
                                          pos[Nk - Nq:], pos) for b in range(case["batch"])])
    table, length, page = s["table"].cpu(), s["length"].tolist(), case["page"]
    new = s["new"]
    if op == "paged":
        rows, at = [], 0
        for i in range(case["streams"]):
            n, total = new[i], length[i]
            where = torch.tensor([int(table[i, t // page]) * page + t % page for t in range(total)], device="cuda")
            flat = lambda pool: pool.flatten(0, 1)[where]  # noqa: E731
            token = torch.arange(total - n, total, device="cuda")
            end = token + 1 if case["causal"] else torch.full_like(token, total)
            o = _softmax_rows(s["q"][at:at + n].transpose(0, 1), flat(s["k"]).transpose(0, 1), flat(s["v"]).transpose(0, 1),
                              None if s["mass"] is None else flat(s["mass"]), torch.zeros_like(end), end, case["softcap"], s["slope"],
                              token, torch.arange(total, device="cuda"))
            rows.append(o.transpose(0, 1))
            at += n
        return torch.cat(rows)
    # the cache by hand, one token after the other: lists of pages per slot
    refs = s["refs"].tolist()
    held = [[int(p) for p in row if p >= 0] for row in table]
    moves = []  # (pool rows written, where from): ("old", row) or ("new", token)
    if op == "compact":
        live = [p for p, r in enumerate(refs) if r > 0]
        holes = [p for p, r in enumerate(refs) if r == 0 and p < len(live)]
        to = dict(zip([p for p in live if p >= len(live)], holes))
        for a, b in to.items():
            moves += [(b * page + t, "old", a * page + t) for t in range(page)]
            refs[b], refs[a] = refs[a], 0
        held = [[to.get(p, p) for p in row] for row in held]
    else:
        seq = s["sequence"].tolist()
        if op == "append":
            for i in seq:
                for p in held[i]:
                    refs[p] -= 1
                held[i], length[i] = [], 0
        else:
            for i in seq:
                held[i], length[i] = list(held[0]), length[0]
                for p in held[i]:
                    refs[p] += 1
        free = iter([p for p, r in enumerate(refs) if r == 0])
        shared = list(refs)
        token = 0
        for i, n in zip(seq, new):
            for t in range(n):
                if length[i] % page == 0:
                    held[i].append(next(free))
                    refs[held[i][-1]] = 1
                elif t == 0 and shared[held[i][-1]] > 1:
                    was = held[i][-1]
                    held[i][-1] = next(free)
                    refs[was] -= 1
                    refs[held[i][-1]] = 1
                    moves += [(held[i][-1] * page + r, "old", was * page + r) for r in range(length[i] % page)]
                moves.append((held[i][-1] * page + length[i] % page, "new", token))
                length[i] += 1
                token += 1
    out = []
    for pool, fresh in ((s["k"], s.get("new_k")), (s["v"], s.get("new_v")), (s["mass"], s.get("new_mass"))):
        if pool is None:
            out.append(None)
            continue
        flat = pool.flatten(0, 1).clone()
        for kind, rows in (("old", pool.flatten(0, 1)), ("new", fresh)):
            some = [(a, b) for a, what, b in moves if what == kind]
            if some:
                dst, src = torch.tensor(some, device="cuda").unbind(1)
                flat[dst] = rows[src]
        out.append(flat.view(pool.shape).double())
    width = table.shape[1]
    out += [torch.tensor([row + [-1] * (width - len(row)) for row in held], dtype=torch.int32),
            torch.tensor(length, dtype=torch.int32), torch.tensor(refs, dtype=torch.int32)]
    return out + [torch.tensor([sum(r > 0 for r in refs)], dtype=torch.int32)] if op == "compact" else out
