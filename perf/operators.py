"""Performance cases of the operators that continue a sequence: rotary
positions, the paged key/value cache (write, read, attention of drafted
tokens) and the rules on the logits before a token is picked.

`own` false computes an operator from elementary torch operations; true calls
the package. Kinds:

  rope     rotation of every head at given positions (kernels.rope_positions)
  append   K and V of new tokens into the cache, quantised, and read back
           (cache.write, cache.read)
  gather   the cached tokens of some requests as dense bf16 rows (cache.read)
  attend   attention of one token, a drafted tree or a chunk of each request
           over the cache (cache.attention)
  logits   penalties, biases and grammar masks (kernels.adjust_logits)
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
CODES = {"bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn, "int8": torch.int8}


def listed():
    return [
        # Four conversations, one new token each: latency.
        dict(name="rope_step", kind="rope", rows=4, model="llama-3.2-1b", rot=64, layout="half",
             dtype="bf16", far=131072, factor=32.0),
        # The q and k heads of a long prefill, pairs interleaved, a stretched context.
        dict(name="rope_prefill", kind="rope", rows=8192, model="llama-3.0-8b", rot=128,
             layout="interleaved", dtype="bf16", far=1048576, factor=8.0),
        # One step of a served batch: one token of every request into an 8-bit cache.
        dict(name="append_step", kind="append", requests=48, tokens=1, context=4096,
             model="llama-3.0-8b", codes="int8", page=16, mix=1),
        # Prompts of a batch into the cache after their prefill.
        dict(name="append_prompts", kind="append", requests=5, tokens=4097, context=1,
             model="llama-3.0-8b", codes="fp8", page=64, mix=2),
        # A cached prefix back as dense rows, for a prefill that goes on from it.
        dict(name="gather_prefix", kind="gather", requests=3, tokens=20000, context=1,
             model="llama-3.0-8b", codes="int8", page=16, mix=3),
        # One conversation, one token: latency.
        dict(name="attend_one", kind="attend", requests=1, tokens=1, context=777,
             model="llama-3.2-1b", codes="bf16", page=16, window=0, tree=False, mix=4),
        # A served batch of ragged lengths, one token each.
        dict(name="attend_batch", kind="attend", requests=64, tokens=1, context=8192,
             model="llama-3.0-8b", codes="fp8", page=64, window=0, tree=False, mix=5),
        # Drafted trees of a batch being checked.
        dict(name="attend_tree", kind="attend", requests=8, tokens=25, context=4000,
             model="llama-3.0-8b", codes="int8", page=16, window=0, tree=True, mix=6),
        # One long document, one token.
        dict(name="attend_long", kind="attend", requests=1, tokens=1, context=131000,
             model="qwen2.5-0.5b", codes="bf16", page=64, window=0, tree=False, mix=7),
        # A chunk of a prompt behind its cached part.
        dict(name="attend_chunk", kind="attend", requests=2, tokens=256, context=8000,
             model="llama-3.0-8b", codes="bf16", page=64, window=0, tree=False, mix=8),
        # The logits of a small batch, float32 as the decoder writes them.
        dict(name="logits_step", kind="logits", requests=4, tokens=1, vocab=128256, dtype="f32",
             history=1000, bias=20, mask=True, tree=False, mix=9),
        # Every drafted token's logits of a batch of trees.
        dict(name="logits_tree", kind="logits", requests=8, tokens=25, vocab=151936, dtype="f32",
             history=4000, bias=300, mask=True, tree=True, mix=10),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "gather", "attend", "attend", "attend", "logits"])
    mix = rng.randint(100, 1 << 20)
    model = rng.choice(sorted(HEADS))
    hd = HEADS[model][2]
    codes, page = rng.choice(sorted(CODES)), rng.choice([16, 32, 64, 128, 256])
    if kind == "rope":
        return dict(kind=kind, rows=_log(rng, 1, 8192), model=model,
                    rot=rng.choice([hd, hd, hd // 2, hd // 4]),
                    layout=rng.choice(["half", "interleaved"]), dtype=rng.choice(["bf16", "f32"]),
                    far=_log(rng, 1000, 1 << 20), factor=rng.choice([1.0, 4.0, 8.0, 32.0]))
    if kind == "append":
        b = _log(rng, 1, 128)
        return dict(kind=kind, requests=b, tokens=_log(rng, 1, max(1, 16000 // b)),
                    context=_log(rng, 1, 4000), model=model, codes=codes, page=page, mix=mix)
    if kind == "gather":
        b = _log(rng, 1, 64)
        return dict(kind=kind, requests=b, tokens=_log(rng, 1, 30000 // b),
                    context=_log(rng, 1, 4000), model=model, codes=codes, page=page, mix=mix)
    if kind == "attend":
        hkv = HEADS[model][1]
        form = rng.choice(["one", "one", "tree", "chunk"])
        b = _log(rng, 1, 8 if form == "chunk" else 96)
        n = {"one": 1, "tree": rng.randint(2, 80), "chunk": rng.randint(16, 256)}[form]
        # At most half the cached values of the largest listed case, and a
        # score matrix of at most that of the listed chunk.
        most = min(200_000_000 // (hkv * hd * b), 100_000_000 // (b * n * HEADS[model][0]))
        return dict(kind=kind, requests=b, tokens=n, context=_log(rng, 1, max(2, min(most, 60000))),
                    model=model, codes=codes, page=page, window=rng.choice([0, 0, 0, 1000]),
                    tree=form == "tree", mix=mix)
    b = _log(rng, 1, 64)
    tree = rng.random() < 0.5
    return dict(kind=kind, requests=b, tokens=rng.randint(2, max(2, 160 // b)) if tree else 1,
                vocab=rng.choice([32000, 49152, 50257, 128256, 151936]),
                dtype=rng.choice(["f32", "bf16"]), history=_log(rng, 8, 8000),
                bias=rng.choice([0, 5, 100, 300]), mask=rng.random() < 0.7, tree=tree, mix=mix)


# ------------------------------------------------------------------ helpers

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEV)


def _lengths(case):
    """(new tokens, tokens before them) of each request."""
    rng = random.Random(case["mix"])
    b, n, c = case["requests"], case["tokens"], case.get("context", 1)
    new = [n if i == 0 else rng.randint(max(1, n // 2), n) for i in range(b)]
    # A prompt starts at 0; a context is ragged, the first request the longest.
    before = [c if i == 0 else _log(rng, max(1, c // 8), c) for i in range(b)]
    return new, [0 if c == 1 else x for x in before]


def _offsets(new):
    out = [0]
    for n in new:
        out.append(out[-1] + n)
    return out


def _tree_bits(case, new):
    """int64 [rows, words]: bit j of a row is set where drafted token j of its
    request is one of its ancestors or itself."""
    rng = random.Random(case["mix"] + 1)
    words = (max(new) + 63) // 64
    rows, depth = [], []
    for n in new:
        anc = []
        for i in range(n):
            up = anc[rng.randint(max(0, i - 8), i - 1)] if i else 0
            anc.append(up | (1 << i))
        rows += [[(a >> (64 * w)) & (2**64 - 1) for w in range(words)] for a in anc]
        depth += [bin(a).count("1") - 1 for a in anc]
    signed = [[w - 2**64 if w >= 2**63 else w for w in r] for r in rows]
    return torch.tensor(signed, dtype=torch.int64, device=DEV), depth


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


def _values(pages, scales):
    return pages.float() if scales is None else pages.float() * scales[..., None]


def _places(s):
    """Request, page and row in the page of every new token."""
    rows = torch.arange(s["rows"], device=DEV)
    req = torch.searchsorted(s["offsets"][1:].contiguous(), rows.int(), right=True)
    pos = s["starts"].long()[req] + rows - s["offsets"].long()[req]
    return req, s["table"].long()[req, pos // s["page"]], pos % s["page"]


# ------------------------------------------------------------------ prepare

def _cache(case, g, new, before, filled):
    """Pages, scales and the page table of a cache of every request's tokens,
    its pages in any order, a few of them nobody's."""
    _, hkv, hd = HEADS[case["model"]]
    page, codes = case["page"], case["codes"]
    need = [(n + c + page - 1) // page for n, c in zip(new, before)]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device=DEV).int()
    table = torch.full((len(new), max(need) + 1), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s = {"table": table, "page": page, "codes": codes}
    for name in ("k", "v"):
        pages = torch.zeros(total, hkv, page, hd, device=DEV, dtype=CODES[codes])
        scales = None if codes == "bf16" else torch.zeros(total, hkv, page, device=DEV)
        step = max(1, 30_000_000 // (hkv * page * hd))
        for a in range(0, total, step) if filled else ():
            b = min(total, a + step)
            q, sc = _quantise(_randn(g, b - a, hkv, page, hd).to(torch.bfloat16), codes)
            pages[a:b] = q
            if sc is not None:
                scales[a:b] = sc
        s[name + "_pages"], s[name + "_scales"] = pages, scales
    return s


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind == "rope":
        hq, hkv, hd = HEADS[case["model"]]
        half, f = case["rot"] // 2, case["factor"]
        inv = 500000.0 ** (-torch.arange(half, device=DEV, dtype=torch.float64) / half)
        s.update(heads=hq + hkv, head_dim=hd, layout=case["layout"],
                 # Slow pairs stretched, fast ones kept.
                 inv_freq=torch.where(inv < 0.001, inv / f, inv).float(),
                 scale=0.1 * math.log(f) + 1.0,
                 x=_randn(g, case["rows"], (hq + hkv) * hd).to(
                     torch.bfloat16 if case["dtype"] == "bf16" else torch.float32),
                 positions=torch.randint(0, case["far"], (case["rows"],), generator=g,
                                         device=DEV, dtype=torch.int32))
        return s
    new, before = _lengths(case)
    offsets = _offsets(new)
    s.update(offsets=_ints(offsets), rows=offsets[-1], longest=max(new))
    if kind == "logits":
        rows, b, v, h = offsets[-1], case["requests"], case["vocab"], case["history"]
        dtype = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        u = torch.rand(b, h, generator=g, device=DEV)
        lens = torch.randint(h // 2, h + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
        bias = torch.rand(b, v, generator=g, device=DEV).argsort(1)[:, :case["bias"]].int()
        s.update(logits=(3.0 * _randn(g, rows, v)).to(dtype),
                 history=(u ** 3 * v).int().clamp(max=v - 1), history_lens=lens,
                 prompt_lens=lens // 3, repetition=1.05 + 0.2 * torch.rand(b, generator=g, device=DEV),
                 frequency=0.3 * torch.rand(b, generator=g, device=DEV),
                 presence=0.5 * torch.rand(b, generator=g, device=DEV),
                 bias_ids=bias if case["bias"] else None,
                 bias_values=_randn(g, b, case["bias"]) if case["bias"] else None,
                 allowed=torch.randint(-2**31, 2**31, (rows, (v + 31) // 32), generator=g,
                                       device=DEV).int() if case["mask"] else None,
                 draft_tokens=None, tree_mask=None)
        if case["tree"]:
            s["tree_mask"], _ = _tree_bits(case, new)
            s["draft_tokens"] = torch.randint(0, v, (rows,), generator=g, device=DEV,
                                              dtype=torch.int32)
        return s
    hq, hkv, hd = HEADS[case["model"]]
    s.update(_cache(case, g, new, before, kind != "append"), starts=_ints(before))
    if kind == "append":
        # K and V as the columns behind Q in the projection's output.
        qkv = _randn(g, s["rows"], (hq + 2 * hkv) * hd).to(torch.bfloat16)
        s.update(k=qkv[:, hq * hd:(hq + hkv) * hd], v=qkv[:, (hq + hkv) * hd:])
    elif kind == "attend":
        depth = [i for n in new for i in range(n)]
        tree = None
        if case["tree"]:
            tree, depth = _tree_bits(case, new)
        first = [c for n, c in zip(new, before) for _ in range(n)]
        s.update(q=_randn(g, s["rows"], hq * hd).to(torch.bfloat16), tree_mask=tree, q_heads=hq,
                 window=case["window"], positions=_ints(d + c for d, c in zip(depth, first)),
                 reach=max(n + c for n, c in zip(new, before)))
    return s


# ---------------------------------------------------------------------- run

def _rope(s):
    half = s["inv_freq"].numel()
    rows = s["x"].shape[0]
    x = s["x"].float().view(rows, s["heads"], s["head_dim"])
    angle = (s["positions"].double()[:, None] * s["inv_freq"].double())[:, None]
    c, n = (angle.cos() * s["scale"]).float(), (angle.sin() * s["scale"]).float()
    y = x.clone()
    a, b = ((slice(0, half), slice(half, 2 * half)) if s["layout"] == "half"
            else (slice(0, 2 * half, 2), slice(1, 2 * half, 2)))
    y[..., a] = x[..., a] * c - x[..., b] * n
    y[..., b] = x[..., b] * c + x[..., a] * n
    return y.view(rows, -1).to(s["x"].dtype)


def _read(s):
    _, page, at = _places(s)
    out = {}
    for name in ("k", "v"):
        sc = s[name + "_scales"]
        x = _values(s[name + "_pages"][page, :, at], None if sc is None else sc[page, :, at])
        out[name] = x.to(torch.bfloat16).reshape(s["rows"], -1)
    return out


def _append(s):
    _, page, at = _places(s)
    for name in ("k", "v"):
        hkv, hd = s["k_pages"].shape[1], s["k_pages"].shape[3]
        q, sc = _quantise(s[name].reshape(s["rows"], hkv, hd), s["codes"])
        s[name + "_pages"][page, :, at] = q
        if sc is not None:
            s[name + "_scales"][page, :, at] = sc
    return _read(s)


def _attend(s):
    offsets, starts = s["offsets"].long(), s["starts"].long()
    hkv, hd = s["k_pages"].shape[1], s["k_pages"].shape[3]
    b, n, group = starts.numel(), s["longest"], s["q_heads"] // hkv
    i, key = torch.arange(n, device=DEV), torch.arange(s["reach"], device=DEV)
    page, at = s["table"].long().clamp(min=0)[:, key // s["page"]], key % s["page"]

    def dense(name):
        sc = s[name + "_scales"]
        x = _values(s[name + "_pages"][page, :, at], None if sc is None else sc[page, :, at])
        return x.permute(0, 2, 1, 3)                              # [b, hkv, reach, hd]

    row = (offsets[:-1, None] + i).clamp(max=s["rows"] - 1)       # [b, n]
    q = s["q"].float()[row].view(b, n, hkv, group, hd).permute(0, 2, 1, 3, 4)
    score = torch.matmul(q.reshape(b, hkv, n * group, hd), dense("k").transpose(2, 3).contiguous())
    score = (score * hd ** -0.5).view(b, hkv, n, group, -1)
    j = (key - starts[:, None])[:, None]                          # drafted index of a key
    count = (offsets[1:] - offsets[:-1])[:, None, None]
    if s["tree_mask"] is None:
        seen = j <= i[:, None]
    else:
        word = (j // 64).clamp(0, s["tree_mask"].shape[1] - 1).expand(b, n, -1)
        seen = (s["tree_mask"][row].gather(2, word) >> (j % 64)) & 1 != 0
    if s["window"]:
        near = key > s["positions"].long()[row][:, :, None] - s["window"]
    else:
        near = torch.ones((), dtype=torch.bool, device=DEV)
    ok = torch.where(j < 0, near, seen & (j < count))[:, None, :, None]
    score = score.masked_fill(~ok, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, hkv, n * group, -1), dense("v")).view(b, hkv, n, group, hd)
    o = (o / torch.where(total > 0, total, torch.ones_like(total))).permute(0, 2, 1, 3, 4)
    req, _, _ = _places(s)
    mine = torch.arange(s["rows"], device=DEV) - offsets[req]
    return o[req, mine].reshape(s["rows"], -1).to(torch.bfloat16)


def _logits(s):
    rows, v = s["logits"].shape
    line = torch.arange(rows, device=DEV)
    req = torch.searchsorted(s["offsets"][1:].contiguous(), line.int(), right=True)
    at = torch.arange(s["history"].shape[1], device=DEV)
    ids = s["history"].long()[req]
    made = (at >= s["prompt_lens"][req][:, None]) & (at < s["history_lens"][req][:, None])
    count = torch.zeros(rows, v, dtype=torch.int32, device=DEV).scatter_add_(1, ids, made.int())
    prompt = (at < s["prompt_lens"][req][:, None]).int()
    seen = torch.zeros(rows, v, dtype=torch.int32, device=DEV).scatter_add_(1, ids, prompt)
    if s["draft_tokens"] is not None:
        first = s["offsets"].long()[req]
        j = torch.arange(s["longest"], device=DEV)
        bit = (s["tree_mask"][:, j // 64] >> (j % 64)) & 1
        drafted = s["draft_tokens"].long()[(first[:, None] + j).clamp(max=rows - 1)]
        count.scatter_add_(1, drafted, bit.int())
    x = s["logits"].float()
    rep = s["repetition"][req][:, None]
    x = torch.where(count + seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][req][:, None] * count.float()
    x = x - s["presence"][req][:, None] * (count > 0).float()
    if s["bias_ids"] is not None:
        x = x.scatter_add(1, s["bias_ids"].long()[req], s["bias_values"][req])
    if s["allowed"] is not None:
        token = torch.arange(v, device=DEV)
        bit = (s["allowed"][:, token // 32] >> (token % 32).int()) & 1
        x = x.masked_fill(bit == 0, -math.inf)
    return x.to(s["logits"].dtype)


def run(s):
    kind = s["case"]["kind"]
    if not own:
        return {"rope": _rope, "append": _append, "gather": _read, "attend": _attend,
                "logits": _logits}[kind](s)
    from ncmorph_amd import cache, kernels

    if kind == "rope":
        return kernels.rope_positions(s["x"], s["positions"], s["inv_freq"], s["heads"],
                                      s["head_dim"], layout=s["layout"], scale=s["scale"])
    if kind == "logits":
        return kernels.adjust_logits(
            s["logits"], history=s["history"], prompt_lens=s["prompt_lens"],
            history_lens=s["history_lens"], repetition=s["repetition"], frequency=s["frequency"],
            presence=s["presence"], bias_ids=s["bias_ids"], bias_values=s["bias_values"],
            allowed=s["allowed"], offsets=s["offsets"], draft_tokens=s["draft_tokens"],
            tree_mask=s["tree_mask"])
    kv = cache.KvCache(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
    if kind == "attend":
        return cache.attention(s["q"], kv, s["q_heads"], s["table"], s["offsets"], s["starts"],
                               tree_mask=s["tree_mask"], window=s["window"],
                               positions=s["positions"] if s["window"] else None)
    if kind == "append":
        cache.write(kv, s["k"], s["v"], s["table"], s["offsets"], s["starts"])
    k, v = cache.read(kv, s["table"], s["offsets"], s["starts"], s["rows"])
    return {"k": k, "v": v}


# --------------------------------------------------------------------- work

def work(case):
    kind = case["kind"]
    if kind == "rope":
        hq, hkv, hd = HEADS[case["model"]]
        n = case["rows"] * (hq + hkv) * hd
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": 2 * n * size + 4 * case["rows"] + 2 * case["rot"],
                "flops": 6 * n * case["rot"] // (2 * hd)}
    new, before = _lengths(case)
    rows = sum(new)
    if kind == "logits":
        size = 4 if case["dtype"] == "f32" else 2
        v, b = case["vocab"], case["requests"]
        mask = rows * ((v + 31) // 32) * 4 if case["mask"] else 0
        return {"bytes": 2 * rows * v * size + mask + b * (3 * case["history"] + 8 * case["bias"]),
                "flops": 4 * rows * v}
    hq, hkv, hd = HEADS[case["model"]]
    size, scale = {"bf16": (2, 0), "fp8": (1, 4), "int8": (1, 4)}[case["codes"]]
    per_token = 2 * hkv * (hd * size + scale)
    if kind == "append":
        # K and V in, codes out, and the values of what was written.
        return {"bytes": rows * (8 * hkv * hd + per_token), "flops": 4 * rows * hkv * hd}
    if kind == "gather":
        return {"bytes": rows * (4 * hkv * hd + per_token), "flops": 2 * rows * hkv * hd}
    keys = pairs = 0
    for n, c in zip(new, before):
        near = min(c, case["window"] + n) if case["window"] else c
        keys += near + n
        per = min(c, case["window"]) if case["window"] else c
        pairs += n * per + n * (n + 1) // 2
    return {"bytes": keys * per_token + 4 * rows * hq * hd, "flops": 4 * hd * hq * pairs}


# -------------------------------------------------------------------- exact

def _exact_rows(s):
    """(request, its first row, cache position) of every row, on the host."""
    offs, starts = s["offsets"].tolist(), s["starts"].tolist()
    return [(r, offs[r], starts[r] + i - offs[r])
            for r in range(len(starts)) for i in range(offs[r], offs[r + 1])]


def _exact_codes(x, codes):
    """The values that the codes of one head's rows stand for, in 64 bits."""
    x = x.double()
    if codes == "bf16":
        return x
    m = x.abs().max(-1, keepdim=True).values
    if codes == "int8":
        safe = torch.where(m > 0, m, torch.ones_like(m))
        return torch.round(x * 127.0 / safe) * (m / 127.0)
    # Values of eight bits: no quotient lies within 1e-9 beside a power of two,
    # so 1e-9 keeps the logarithm of one from rounding to the wrong side.
    e = torch.ceil(torch.log2(torch.where(m > 0, m, torch.ones_like(m)) / 448.0) - 1e-9)
    unit = ((e.long() + 1023) << 52).view(torch.float64)    # 2^e
    y = x / unit                                            # |y| <= 448
    low = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)) + 1e-9)
    # e4m3: three bits behind the first.
    grid = ((low.long() - 3 + 1023) << 52).view(torch.float64)
    return torch.round(y / grid) * grid * unit


def _exact_attend(s):
    offs, starts = s["offsets"].tolist(), s["starts"].tolist()
    hkv, hd, page = s["k_pages"].shape[1], s["k_pages"].shape[3], s["page"]
    group = s["q_heads"] // hkv
    out = torch.zeros(s["rows"], s["q_heads"], hd, dtype=torch.float64, device=DEV)
    for r, c in enumerate(starts):
        a, b = offs[r], offs[r + 1]
        n = b - a
        ids = s["table"][r, :(c + n + page - 1) // page].long()
        allowed = torch.zeros(n, c + n, dtype=torch.bool, device=DEV)
        allowed[:, :c] = True
        if s["window"]:
            far = s["positions"][a:b].long() - s["window"]
            allowed[:, :c] = torch.arange(c, device=DEV)[None] > far[:, None]
        if s["tree_mask"] is None:
            allowed[:, c:] = torch.ones(n, n, device=DEV).tril().bool()
        else:
            for j in range(n):
                allowed[:, c + j] = (s["tree_mask"][a:b, j // 64] >> (j % 64)) & 1 == 1
        for h in range(hkv):
            kv = []
            for name in ("k", "v"):
                x = s[name + "_pages"][ids, h].double()
                if s[name + "_scales"] is not None:
                    x = x * s[name + "_scales"][ids, h].double()[..., None]
                kv.append(x.reshape(-1, hd)[:c + n])
            q = s["q"][a:b].view(n, s["q_heads"], hd)[:, h * group:(h + 1) * group].double()
            z = torch.matmul(q.reshape(n * group, hd), kv[0].t()) / math.sqrt(hd)
            z = z.view(n, group, -1).masked_fill(~allowed[:, None], -math.inf)
            w = torch.softmax(z, -1).nan_to_num(0.0)
            out[a:b, h * group:(h + 1) * group] = torch.matmul(
                w.view(n * group, -1), kv[1]).view(n, group, hd)
    return out.view(s["rows"], -1)


def _exact_logits(s):
    rows, v = s["logits"].shape
    offs = s["offsets"].tolist()
    out = s["logits"].double()
    token = torch.arange(v, device=DEV)
    for r in range(len(offs) - 1):
        p, n = int(s["prompt_lens"][r]), int(s["history_lens"][r])
        h = s["history"][r].long()
        base = torch.bincount(h[p:n], minlength=v)
        old = torch.bincount(h[:p], minlength=v) > 0
        for i in range(offs[r], offs[r + 1]):
            count = base
            if s["draft_tokens"] is not None:
                on = [j for j in range(offs[r + 1] - offs[r])
                      if int(s["tree_mask"][i, j // 64]) >> (j % 64) & 1]
                path = s["draft_tokens"][offs[r]:offs[r + 1]].long()[on]
                count = base + torch.bincount(path, minlength=v)
            x = out[i]
            rep = float(s["repetition"][r])
            x = torch.where(old | (count > 0), torch.where(x > 0, x / rep, x * rep), x)
            x = x - float(s["frequency"][r]) * count - float(s["presence"][r]) * (count > 0)
            if s["bias_ids"] is not None:
                x[s["bias_ids"][r].long()] += s["bias_values"][r].double()
            if s["allowed"] is not None:
                words = s["allowed"][i].long()[token // 32]
                x = torch.where((words >> (token % 32)) & 1 == 1, x, -math.inf)
            out[i] = x
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        half, hd = case["rot"] // 2, s["head_dim"]
        x = s["x"].double().view(case["rows"], s["heads"], hd)
        turn = torch.outer(s["positions"].double(), s["inv_freq"].double())
        spin = torch.polar(torch.full_like(turn, s["scale"]), turn)[:, None]
        part = x[..., :2 * half]
        if s["layout"] == "half":
            z = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * spin
            part = torch.cat([z.real, z.imag], -1)
        else:
            z = torch.view_as_complex(part.reshape(case["rows"], s["heads"], half, 2)) * spin
            part = torch.view_as_real(z).flatten(2)
        return torch.cat([part, x[..., 2 * half:]], -1).view(case["rows"], -1)
    if kind == "logits":
        return _exact_logits(s)
    if kind == "attend":
        return _exact_attend(s)
    hkv, hd = s["k_pages"].shape[1], s["k_pages"].shape[3]
    if kind == "append":
        return {n: _exact_codes(s[n].reshape(-1, hkv, hd), s["codes"]).reshape(s["rows"], -1)
                for n in ("k", "v")}
    place = _exact_rows(s)
    table = s["table"].tolist()
    page = torch.tensor([table[r][p // s["page"]] for r, _, p in place], device=DEV)
    at = torch.tensor([p % s["page"] for _, _, p in place], device=DEV)
    out = {}
    for n in ("k", "v"):
        x = s[n + "_pages"][page, :, at].double()
        if s[n + "_scales"] is not None:
            x = x * s[n + "_scales"][page, :, at].double()[..., None]
        out[n] = x.reshape(s["rows"], -1)
    return out
