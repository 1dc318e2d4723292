"""Performance cases of what else a step of served sequences needs: the page
tables and slots of its tokens, attention of requests that share a prefix, the
pick of a token, and projections with 4-bit weights.

`own` false computes an operator from elementary torch operations; true calls
the package. Kinds:

  tables  pages of a prefix shared, pages of new tokens taken, positions and
          slots made, and all of it given back (cache.share, cache.extend,
          cache.release)
  shared  attention over the cache of requests with common prefixes
          (cache.attention with groups)
  sample  temperature, top-k, top-p and min-p, and the draw (kernels.sample)
  int4    a projection with 4-bit weights and group scales
          (kernels.linear_int4)
"""
import math
import random

import torch

own = False
DEV = "cuda:0"

# q heads, kv heads, head_dim of the checkpoints whose configurations the test
# suite holds.
HEADS = {
    "smollm2-135m": (9, 3, 64),
    "qwen2.5-0.5b": (14, 2, 64),
    "llama-3.2-1b": (32, 8, 64),
    "qwen3-0.6b": (16, 8, 128),
    "llama-3.0-8b": (32, 8, 128),
    "llama-2-7b": (32, 32, 128),
}
# (outputs, inputs) of their projections.
SHAPES = [(576, 576), (576, 1536), (896, 896), (896, 4864), (9728, 896), (2048, 2048),
          (16384, 2048), (2048, 8192), (1024, 2048), (6144, 4096), (4096, 4096), (28672, 4096),
          (4096, 14336)]
CODES = {"bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn, "int8": torch.int8}


def listed():
    return [
        # One token of every request of a served batch.
        dict(name="tables_step", kind="tables", requests=48, tokens=1, context=4096, page=16,
             common=0, mix=1),
        # Prompts that arrive behind one system prompt, its pages shared.
        dict(name="tables_prompts", kind="tables", requests=200, tokens=500, context=1, page=16,
             common=2000, mix=2),
        # A few answers to one prompt, one token each: latency.
        dict(name="shared_few", kind="shared", groups=1, members=4, common=1500, context=120,
             tokens=1, model="llama-3.2-1b", codes="bf16", page=16, tree=False, mix=3),
        # A served batch behind one long system prompt, 8-bit cache.
        dict(name="shared_batch", kind="shared", groups=1, members=64, common=8192, context=700,
             tokens=1, model="llama-3.0-8b", codes="fp8", page=64, tree=False, mix=4),
        # Drafted trees of the requests on three documents.
        dict(name="shared_trees", kind="shared", groups=3, members=7, common=5001, context=300,
             tokens=13, model="llama-3.0-8b", codes="int8", page=16, tree=True, mix=5),
        # Many samples from one long document.
        dict(name="shared_large", kind="shared", groups=1, members=256, common=16000, context=300,
             tokens=1, model="llama-3.0-8b", codes="bf16", page=64, tree=False, mix=6),
        # The tokens of a small batch, every rule in use.
        dict(name="sample_step", kind="sample", requests=4, tokens=1, vocab=128256, dtype="f32",
             rules=True, allowed=0.9, mix=7),
        # Plain draws of a batch from bfloat16 logits.
        dict(name="sample_plain", kind="sample", requests=64, tokens=1, vocab=49152, dtype="bf16",
             rules=False, allowed=1.0, mix=8),
        # Every drafted token of a batch of trees.
        dict(name="sample_trees", kind="sample", requests=8, tokens=25, vocab=151936, dtype="f32",
             rules=True, allowed=0.5, mix=9),
        # One token through a small projection: latency.
        dict(name="int4_small", kind="int4", rows=1, n=576, k=1536, group=32, zeros=False,
             bias=False, residual=True, out="f32", mix=10),
        # One token through the widest projection of a layer.
        dict(name="int4_one", kind="int4", rows=1, n=28672, k=4096, group=128, zeros=False,
             bias=False, residual=False, out="bf16", mix=11),
        # A served batch through it, weights with zero points.
        dict(name="int4_batch", kind="int4", rows=61, n=28672, k=4096, group=32, zeros=True,
             bias=True, residual=True, out="bf16", mix=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "shared", "shared", "sample", "sample", "int4", "int4"])
    mix = rng.randint(100, 1 << 20)
    page = rng.choice([16, 32, 64, 128])
    if kind == "tables":
        b = _log(rng, 1, 256)
        behind = rng.random() < 0.5
        return dict(kind=kind, requests=b, tokens=_log(rng, 1, max(1, 100000 // b)),
                    context=1 if behind else _log(rng, 1, 8000), page=page,
                    common=_log(rng, 16, 8000) if behind else 0, mix=mix)
    if kind == "shared":
        model = rng.choice(sorted(HEADS))
        hq, hkv, hd = HEADS[model]
        groups = rng.choice([1, 1, 2, 3, 5])
        members = _log(rng, 1, 200 // groups)
        tree = rng.random() < 0.3
        tokens = rng.randint(2, 40) if tree else rng.choice([1, 1, 1, 4])
        tokens = min(tokens, max(1, 6_000_000 // (groups * members * hq * hd)))
        # At most half the products and the cached values of the largest
        # listed case.
        most = 256 * 16000 * 32 * 128 // 2 // (groups * members * tokens * hq * hd)
        values = 14_000_000 // (hkv * hd * groups)
        page = min(page, 32) if groups * members > 60 else page   # tokens in no whole page
        return dict(kind=kind, groups=groups, members=members,
                    common=_log(rng, 16, max(17, min(most, values, 20000))),
                    context=_log(rng, 1, max(1, min(most, values // members, 2000))),
                    tokens=tokens, model=model,
                    codes=rng.choice(sorted(CODES)), page=page, tree=tree, mix=mix)
    if kind == "sample":
        b = _log(rng, 1, 100)
        return dict(kind=kind, requests=b, tokens=rng.choice([1, 1, rng.randint(1, max(1, 140 // b))]),
                    vocab=rng.choice([1000, 32000, 49152, 50257, 128256, 151936]),
                    dtype=rng.choice(["f32", "bf16"]), rules=rng.random() < 0.7,
                    allowed=rng.choice([1.0, 0.9, 0.5, 0.01]), mix=mix)
    n, k = rng.choice(SHAPES)
    return dict(kind=kind, rows=_log(rng, 1, 61), n=n, k=k, group=rng.choice([32, 64, 128]),
                zeros=rng.random() < 0.5, bias=rng.random() < 0.3, residual=rng.random() < 0.3,
                out=rng.choice(["f32", "bf16"]), mix=mix)


# ------------------------------------------------------------------ helpers

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEV)


def _ragged(case):
    """(new tokens, tokens before them and behind the common ones) of each
    request."""
    rng = random.Random(case["mix"])
    b = case["requests"] if "requests" in case else case["groups"] * case["members"]
    n, c = case["tokens"], case.get("context", 1)
    new = [n if i == 0 else rng.randint(max(1, n // 2), n) for i in range(b)]
    before = [c if i == 0 else _log(rng, max(1, c // 8), c) for i in range(b)]
    return new, [0 if c == 1 else x for x in before]


def _commons(case):
    """Tokens that each group shares: ragged, the first group's the most."""
    rng = random.Random(case["mix"] + 2)
    c = case["common"]
    return [c if i == 0 else rng.randint(max(1, c // 4), c) for i in range(case["groups"])]


def _offsets(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def _up(a, b):
    return (a + b - 1) // b


def _tree_bits(case, new):
    """int64 [rows, words]: bit j of a row is set where drafted token j of its
    request is one of its ancestors or itself."""
    rng = random.Random(case["mix"] + 1)
    words = _up(max(new), 64)
    rows = []
    for n in new:
        anc = []
        for i in range(n):
            up = anc[rng.randint(max(0, i - 8), i - 1)] if i else 0
            anc.append(up | (1 << i))
        rows += [[(a >> (64 * w)) & (2**64 - 1) for w in range(words)] for a in anc]
    signed = [[w - 2**64 if w >= 2**63 else w for w in r] for r in rows]
    return torch.tensor(signed, dtype=torch.int64, device=DEV)


def _quantise(x, codes):
    """Codes and scales of rows of a head: [..., head_dim] -> [...]."""
    x = x.float()
    m = x.abs().amax(-1, keepdim=True)
    if codes == "bf16":
        return x.to(torch.bfloat16), None
    if codes == "fp8":
        f, e = torch.frexp(m)
        e = (e - 9 + (f > 0.875)).clamp(-126, 119)
        scale = ((e + 127) << 23).view(torch.float32)       # 2^e
        return (x / scale).to(torch.float8_e4m3fn), scale[..., 0]
    q = torch.where(m > 0, torch.round(x * 127.0 / m.clamp(min=1e-38)), torch.zeros_like(x))
    return q.to(torch.int8), m[..., 0] / 127.0


# ------------------------------------------------------------------ prepare

def _prepare_tables(case, g, s):
    new, before = _ragged(case)
    b, page, common = case["requests"], case["page"], case["common"]
    starts = [common // page * page] * b if common else before
    width = max(_up(n + c, page) for n, c in zip(new, starts)) + 3
    taken = [0 if common else _up(c, page) for c in before]   # pages held already
    if common:
        taken[0] = _up(common, page)      # request 0 is the system prompt itself
        new[0], starts[0] = 0, common
    fresh = sum(_up(c + n, page) - _up(c, page) for n, c in zip(new, starts))
    pages = sum(taken) + fresh + 17
    order = torch.randperm(pages, generator=g, device=DEV).int()
    table = torch.full((b, width), -1, dtype=torch.int32, device=DEV)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    at = 0
    for r, n in enumerate(taken):
        table[r, :n] = order[at:at + n]
        refs[order[at:at + n].long()] = 1
        at += n
    free = torch.zeros(pages, dtype=torch.int32, device=DEV)
    free[:pages - at] = order[at:]
    s.update(page=page, table=table, new=_ints(new), starts=_ints(starts), rows=sum(new),
             free=free, count=_ints([pages - at]), refs=refs,
             sources=_ints([-1] + [0] * (b - 1)) if common else None,
             shared=_ints([common] * b),
             lens=_ints(n + c for n, c in zip(new, starts)),
             keep=_ints([common] + [0] * (b - 1)) if common else _ints(starts))
    if own:
        from ncmorph_amd import cache
        s["pool"] = cache.PagePool(free, s["count"], refs)


def _prepare_shared(case, g, s):
    hq, hkv, hd = HEADS[case["model"]]
    page, codes, members = case["page"], case["codes"], case["members"]
    new, behind = _ragged(case)
    commons = _commons(case)
    before = [c + commons[i // members] for i, c in enumerate(behind)]
    need = [_up(n + c, page) for n, c in zip(new, before)]
    whole = [c // page for c in commons]                      # pages shared
    total = 3 + sum(whole) + sum(n - whole[i // members] for i, n in enumerate(need))
    order = torch.randperm(total, generator=g, device=DEV).int()
    table = torch.full((len(new), max(need) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        w = whole[i // members]
        if i % members == 0:
            mine = order[at:at + n]
            at += n
        else:
            mine = torch.cat([table[i // members * members, :w], order[at:at + n - w]])
            at += n - w
        table[i, :n] = mine
    s.update(table=table, page=page, codes=codes, q_heads=hq)
    for name in ("k", "v"):
        pages = torch.zeros(total, hkv, page, hd, device=DEV, dtype=CODES[codes])
        scales = None if codes == "bf16" else torch.zeros(total, hkv, page, device=DEV)
        step = max(1, 30_000_000 // (hkv * page * hd))
        for a in range(0, total, step):
            b = min(total, a + step)
            q, sc = _quantise(_randn(g, b - a, hkv, page, hd).to(torch.bfloat16), codes)
            pages[a:b] = q
            if sc is not None:
                scales[a:b] = sc
        s[name + "_pages"], s[name + "_scales"] = pages, scales
    offsets = _offsets(new)
    s.update(offsets=_ints(offsets), starts=_ints(before), rows=offsets[-1],
             groups=_ints(members * i for i in range(case["groups"] + 1)),
             # Whole pages are what the tables share.
             shared=_ints(w * page for w in whole),
             q=_randn(g, offsets[-1], hq * hd).to(torch.bfloat16),
             tree_mask=_tree_bits(case, new) if case["tree"] else None)


def _prepare_sample(case, g, s):
    new, _ = _ragged(case)
    rows, b, v = sum(new), case["requests"], case["vocab"]
    sharp = 1.5 + 2.5 * _rand(g, rows, 1)
    x = sharp * _randn(g, rows, v)
    if case["allowed"] < 1.0:
        x = torch.where(_rand(g, rows, v) < case["allowed"], x, torch.full_like(x, -math.inf))
    s.update(logits=x.to(torch.float32 if case["dtype"] == "f32" else torch.bfloat16),
             uniform=_rand(g, rows), offsets=_ints(_offsets(new)), rows=rows,
             temperature=0.5 + _rand(g, b), top_k=None, top_p=None, min_p=None)
    if case["rules"]:
        # One request in eight is greedy; each rule is off for some.
        u = _rand(g, 4, b)
        s["temperature"] = torch.where(u[0] < 0.125, torch.zeros_like(u[0]), s["temperature"])
        k = torch.randint(5, 200, (b,), generator=g, device=DEV, dtype=torch.int32)
        s["top_k"] = torch.where(u[1] < 0.4, torch.zeros_like(k), k)
        s["top_p"] = torch.where(u[2] < 0.3, torch.ones_like(u[2]), 0.7 + 0.29 * _rand(g, b))
        s["min_p"] = torch.where(u[3] < 0.5, torch.zeros_like(u[3]), 0.1 * _rand(g, b))


def _prepare_int4(case, g, s):
    m, n, k, group = case["rows"], case["n"], case["k"], case["group"]
    groups = _up(k, group)
    s.update(codes=torch.randint(0, 16, (n, k), generator=g, device=DEV, dtype=torch.uint8),
             scales=((0.5 + _rand(g, n, groups)) * (0.3 / math.sqrt(k))).to(torch.bfloat16),
             zeros=torch.randint(5, 11, (n, groups), generator=g, device=DEV, dtype=torch.uint8)
             if case["zeros"] else None,
             x=_randn(g, m, k).to(torch.bfloat16),
             bias=_randn(g, n).to(torch.bfloat16) if case["bias"] else None,
             residual=_randn(g, m, n) if case["residual"] else None, out=case["out"],
             group=group)
    if own:
        from ncmorph_amd import kernels
        s["weight"] = kernels.pack_int4(s["codes"], s["scales"], group, zeros=s["zeros"])


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": case}
    {"tables": _prepare_tables, "shared": _prepare_shared, "sample": _prepare_sample,
     "int4": _prepare_int4}[case["kind"]](case, g, s)
    return s


# ---------------------------------------------------------------------- run

def _tables(s):
    table, free, count, refs, page = s["table"], s["free"], s["count"], s["refs"], s["page"]
    column = torch.arange(table.shape[1], device=DEV)
    if s["sources"] is not None:
        on = (column < (s["shared"] // page)[:, None]) & (s["sources"] >= 0)[:, None]
        theirs = table[s["sources"].long().clamp(min=0)]
        table.copy_(torch.where(on, theirs, table))
        refs.scatter_add_(0, table[on].long(), torch.ones_like(table[on]))
    # Extend.
    starts, new = s["starts"].long(), s["new"].long()
    offsets = torch.cat([torch.zeros_like(new[:1]), new.cumsum(0)])
    first, last = _up(starts, page), _up(starts + new, page)
    on = (column >= first[:, None]) & (column < last[:, None])
    rank = on.flatten().long().cumsum(0).view(on.shape) - 1
    held = free[(count.long() - 1 - rank).clamp(min=0)]
    fresh = torch.where(rank < count, held, torch.full_like(held, -1))
    table.copy_(torch.where(on, fresh, table))
    refs.scatter_add_(0, held.long().flatten(), (on & (rank < count)).int().flatten())
    total = on.sum()
    missing = (total - count).clamp(min=0).int()
    count.copy_((count - total).clamp(min=0).int())
    row = torch.arange(s["rows"], device=DEV)
    req = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
    positions = starts[req] + row - offsets[req]
    place = table[req, positions // page].long()
    slots = torch.where(place >= 0, place * page + positions % page, torch.full_like(place, -1))
    # Release.
    on = ((column >= _up(s["keep"], page)[:, None]) & (column < _up(s["lens"], page)[:, None]))
    ids = table[on].long()
    table.masked_fill_(on, -1)
    refs.scatter_add_(0, ids, torch.full_like(ids, -1).int())
    order = torch.arange(ids.numel(), device=DEV)
    lowest = torch.full_like(refs, 1 << 30).scatter_reduce_(0, ids, order.int(), "amin")
    back = ids[(refs[ids] == 0) & (lowest[ids] == order)].flip(0)
    free[(count.long() + torch.arange(back.numel(), device=DEV))] = back.int()
    count += back.numel()
    return {"offsets": offsets.int(), "positions": positions.int(), "slots": slots,
            "missing": missing, "table": table, "free": free, "count": count, "refs": refs}


def _values(s, name, page, at):
    x = s[name + "_pages"][page, :, at].float()
    sc = s[name + "_scales"]
    return x if sc is None else x * sc[page, :, at][..., None]


def _shared(s):
    members, (_, hkv, hd) = s["case"]["members"], s["k_pages"].shape[:2] + s["k_pages"].shape[3:]
    group, rows = s["q_heads"] // hkv, s["rows"]
    table, page = s["table"].long().clamp(min=0), s["page"]
    out = torch.empty(rows, s["q_heads"] * hd, dtype=torch.bfloat16, device=DEV)
    new, behind = _ragged(s["case"])
    offs = _offsets(new)
    for g, common in enumerate(_commons(s["case"])):
        shared = common // page * page
        lo, b = g * members, members
        n, reach = max(new[lo:lo + b]), max(x + y for x, y in zip(new[lo:lo + b],
                                                                  behind[lo:lo + b]))
        reach += common - shared
        offsets, starts = s["offsets"][lo:lo + b + 1].long(), s["starts"][lo:lo + b].long()
        i = torch.arange(n, device=DEV)
        count = (offsets[1:] - offsets[:-1])[:, None]
        row = (offsets[:-1, None] + i).clamp(max=rows - 1)                # [b, n]
        q = s["q"].float()[row].view(b, n, hkv, group, hd) * hd ** -0.5
        q = q.permute(2, 0, 1, 3, 4).reshape(hkv, b, n * group, hd)
        key = torch.arange(shared, device=DEV)
        k0, v0 = (_values(s, x, table[lo, key // page], key % page).transpose(0, 1).contiguous()
                  for x in ("k", "v"))                                    # [hkv, shared, hd]
        key = shared + torch.arange(reach, device=DEV)
        pages = table[lo:lo + b][:, (key // page).clamp(max=table.shape[1] - 1)]
        k1, v1 = (_values(s, x, pages, key % page).permute(2, 0, 1, 3).contiguous()
                  for x in ("k", "v"))                                    # [hkv, b, reach, hd]
        j = (key - starts[:, None])[:, None]
        if s["tree_mask"] is None:
            seen = j <= i[:, None]
        else:
            word = (j // 64).clamp(0, s["tree_mask"].shape[1] - 1).expand(b, n, -1)
            seen = (s["tree_mask"][row].gather(2, word) >> (j % 64)) & 1 != 0
        ok = (j < 0) | (seen & (j < count[:, :, None]))                   # [b, n, reach]
        own_ = torch.matmul(q, k1.transpose(2, 3).contiguous())
        own_ = own_.view(hkv, b, n, group, reach).masked_fill(~ok[None, :, :, None], -math.inf)
        score = torch.cat([torch.matmul(q.reshape(hkv, -1, hd), k0.transpose(1, 2).contiguous()),
                           own_.view(hkv, -1, reach)], -1)
        p = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-1e30))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p[..., :shared], v0)
        o = o + torch.matmul(p[..., shared:].reshape(hkv, b, n * group, reach), v1).view(o.shape)
        o = o / torch.where(total > 0, total, torch.ones_like(total))
        o = o.view(hkv, b, n, group, hd).permute(1, 2, 0, 3, 4)
        here = (i < count)
        out[offs[lo]:offs[lo + b]] = o[here].reshape(-1, s["q_heads"] * hd).to(torch.bfloat16)
    return out


def _sample(s):
    rows, v = s["logits"].shape
    req = torch.searchsorted(s["offsets"][1:].contiguous(),
                             torch.arange(rows, device=DEV).int(), right=True)
    x, order = s["logits"].float().sort(dim=-1, descending=True, stable=True)
    x = x.double()
    t = s["temperature"].double()[req][:, None]
    greedy = t <= 0
    w = torch.exp((x - x[:, :1]) / torch.where(greedy, torch.ones_like(t), t))
    place = torch.arange(v, device=DEV)
    w = torch.where(greedy & (place > 0), torch.zeros_like(w), w)
    if s["top_k"] is not None:
        k = s["top_k"][req][:, None]
        w = torch.where((k > 0) & (place >= k), torch.zeros_like(w), w)
    if s["top_p"] is not None:
        p = s["top_p"].double()[req][:, None]
        c = w.cumsum(-1)
        ahead = c - w
        w = torch.where((p < 1) & (ahead >= p * c[:, -1:]), torch.zeros_like(w), w)
    if s["min_p"] is not None:
        w = torch.where(w < s["min_p"].double()[req][:, None], torch.zeros_like(w), w)
    c = w.cumsum(-1)
    at = (c <= s["uniform"].double()[:, None] * c[:, -1:]).sum(-1, keepdim=True).clamp(max=v - 1)
    return {"tokens": order.gather(1, at)[:, 0].int(),
            "probabilities": (w.gather(1, at) / c[:, -1:])[:, 0].float()}


def _int4(s):
    group, k = s["group"], s["x"].shape[1]
    scale = s["scales"].float().repeat_interleave(group, 1)[:, :k]
    zero = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(group, 1)[:, :k]
    y = torch.matmul(s["x"].float(), ((s["codes"].float() - zero) * scale).t())
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["residual"] is not None:
        y = y + s["residual"]
    return y if s["out"] == "f32" else y.to(torch.bfloat16)


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"tables": _tables, "shared": _shared, "sample": _sample, "int4": _int4}[kind](s)
    from ncmorph_amd import cache, kernels

    if kind == "tables":
        pool, table, page = s["pool"], s["table"], s["page"]
        if s["sources"] is not None:
            cache.share(pool, table, s["sources"], s["shared"], page)
        step = cache.extend(pool, table, s["new"], s["starts"], s["rows"], page)
        cache.release(pool, table, s["lens"], s["keep"], page)
        return {"offsets": step.offsets, "positions": step.positions, "slots": step.slots,
                "missing": step.missing, "table": table, "free": s["free"], "count": s["count"],
                "refs": s["refs"]}
    if kind == "shared":
        kv = cache.KvCache(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
        return cache.attention(s["q"], kv, s["q_heads"], s["table"], s["offsets"], s["starts"],
                               tree_mask=s["tree_mask"], groups=s["groups"], shared=s["shared"])
    if kind == "sample":
        tokens, probabilities = kernels.sample(
            s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"],
            top_p=s["top_p"], min_p=s["min_p"], offsets=s["offsets"], probabilities=True)
        return {"tokens": tokens, "probabilities": probabilities}
    return kernels.linear_int4(s["x"], s["weight"], bias=s["bias"], residual=s["residual"],
                               out_mode=s["out"])


# --------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    new, before = _ragged(case) if kind != "int4" else ([], [])
    if kind == "tables":
        page, b, common = case["page"], case["requests"], case["common"]
        starts = [common // page * page] * b if common else before
        fresh = sum(_up(c + n, page) - _up(c, page) for n, c in zip(new, starts))
        lent = b * (common // page)
        # Entries written and read back with their counts, 12 bytes a new row.
        return {"bytes": 24 * b + 32 * fresh + 24 * lent + 12 * sum(new),
                "flops": sum(new) + fresh + lent}
    if kind == "shared":
        hq, hkv, hd = HEADS[case["model"]]
        size, scale = {"bf16": (2, 0), "fp8": (1, 4), "int8": (1, 4)}[case["codes"]]
        commons, page, members = _commons(case), case["page"], case["members"]
        rows = sum(new)
        keys = sum(c // page * page for c in commons)
        pairs = 0
        for i, (n, c) in enumerate(zip(new, before)):
            common = commons[i // members]
            keys += n + c + common % page
            pairs += n * (c + common) + n * (n + 1) // 2
        return {"bytes": keys * 2 * hkv * (hd * size + scale) + 4 * rows * hq * hd,
                "flops": 4 * hd * hq * pairs}
    if kind == "sample":
        rows, size = sum(new), 4 if case["dtype"] == "f32" else 2
        return {"bytes": rows * (case["vocab"] * size + 12) + 16 * case["requests"],
                "flops": 3 * rows * case["vocab"]}
    m, n, k = case["rows"], case["n"], case["k"]
    groups = _up(k, case["group"])
    size = 4 if case["out"] == "f32" else 2
    return {"bytes": n * k // 2 + n * groups * (3 if case["zeros"] else 2) + 2 * m * k
            + m * n * (size + (4 if case["residual"] else 0)) + (2 * n if case["bias"] else 0),
            "flops": 2 * m * n * k}


# -------------------------------------------------------------------- exact

def _exact_shared(s):
    offs, starts = s["offsets"].tolist(), s["starts"].tolist()
    hkv, hd, page = s["k_pages"].shape[1], s["k_pages"].shape[3], s["page"]
    group = s["q_heads"] // hkv
    out = torch.zeros(s["rows"], s["q_heads"], hd, dtype=torch.float64, device=DEV)
    for r, c in enumerate(starts):
        a, b = offs[r], offs[r + 1]
        n = b - a
        ids = s["table"][r, :(c + n + page - 1) // page].long()
        allowed = torch.ones(n, c + n, dtype=torch.bool, device=DEV)
        if s["tree_mask"] is None:
            allowed[:, c:] = torch.ones(n, n, device=DEV).tril().bool()
        else:
            for j in range(n):
                allowed[:, c + j] = (s["tree_mask"][a:b, j // 64] >> (j % 64)) & 1 == 1
        kv = []
        for name in ("k", "v"):
            x = s[name + "_pages"][ids].double()
            if s[name + "_scales"] is not None:
                x = x * s[name + "_scales"][ids].double()[..., None]
            kv.append(x.transpose(0, 1).reshape(hkv, -1, hd)[:, :c + n])
        q = s["q"][a:b].view(n, hkv, group, hd).double().transpose(0, 1)
        for h in range(hkv):
            z = torch.matmul(q[h].reshape(n * group, hd), kv[0][h].t()) / math.sqrt(hd)
            z = z.view(n, group, -1).masked_fill(~allowed[:, None], -math.inf)
            w = torch.softmax(z, -1).view(n * group, -1)
            out[a:b, h * group:(h + 1) * group] = torch.matmul(w, kv[1][h]).view(n, group, hd)
    return out.view(s["rows"], -1)


def _exact_sample(s):
    """Row by row: the kept tokens in order, and the first whose cumulative
    weight passes the uniform number's share."""
    offs = s["offsets"].tolist()
    tokens = torch.zeros(s["rows"], dtype=torch.int32, device=DEV)
    chance = torch.zeros(s["rows"], dtype=torch.float64, device=DEV)
    for r in range(len(offs) - 1):
        t = float(s["temperature"][r])
        k = int(s["top_k"][r]) if s["top_k"] is not None else 0
        p = float(s["top_p"][r]) if s["top_p"] is not None else 1.0
        least = float(s["min_p"][r]) if s["min_p"] is not None else 0.0
        for i in range(offs[r], offs[r + 1]):
            x = s["logits"][i].double()
            ids = torch.argsort(x, descending=True, stable=True)
            if t <= 0:
                tokens[i], chance[i] = ids[0], 1.0
                continue
            ids = ids[:k] if k > 0 else ids
            w = torch.softmax(x[ids] / t, 0)
            if p < 1:
                ends = torch.nonzero(w.cumsum(0) >= p)
                w = w[:int(ends[0]) + 1] if ends.numel() else w
            w = w[w >= least * w[0]]
            w = w / w.sum()
            above = torch.nonzero(w.cumsum(0) > float(s["uniform"][i]))
            j = int(above[0]) if above.numel() else w.numel() - 1
            tokens[i], chance[i] = ids[j], w[j]
    return {"tokens": tokens, "probabilities": chance}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "tables":
        return None                       # whole numbers
    if kind == "shared":
        return _exact_shared(s)
    if kind == "sample":
        return _exact_sample(s)
    group, (n, k) = s["group"], s["codes"].shape
    y = torch.zeros(case["rows"], n, dtype=torch.float64, device=DEV)
    for g, a in enumerate(range(0, k, group)):
        b = min(k, a + group)
        q = s["codes"][:, a:b].double() - (8.0 if s["zeros"] is None
                                           else s["zeros"][:, g:g + 1].double())
        y += torch.matmul(s["x"][:, a:b].double(), q.t()) * s["scales"][:, g].double()
    if s["bias"] is not None:
        y = y + s["bias"].double()
    if s["residual"] is not None:
        y = y + s["residual"].double()
    return y
