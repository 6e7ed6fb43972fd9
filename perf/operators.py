"""The work that is timed for the 4-bit key/value cache: one pass through each operator around it.

Fields of a case
  op       "rotary": positions into queries and keys; "plan": block tables and slots of a step from its request lengths;
           "append": new keys and values into the cache, and the same rows read back; "attention": queries against the cache
  dtype    "fp16" or "bf16": queries, keys, values and the cache's steps and offsets
  heads, kv_heads, head_dim   query heads, key/value heads, elements of a head
  group    neighbouring elements of a head that share a step and an offset
  page     tokens of a page
  tokens   rows of the call (rotary, append)
  mix      which lengths the requests have: they are part of the case, not of the seed
Further ones stand beside the functions that read them.

The cache is a uint8 tensor [pages, kv_heads, bytes of a page].  A page is a run of cells of 16 tokens, a cell holds
  key codes    [block of 128][token][4][word of 32][half] 16-bit words of four codes; element = 128 block + 32 word + 8 [4] + 4 half + code
  value codes  [block of 128][token / 8][8][token % 8 / 2][word of 64][half][token % 2], element = 128 block + 64 word + 32 half + 4 [8] + code
  key steps    [token][group] pairs (step, offset)
  value steps  [token][group] pairs (step, offset)
and an element is offset + step * code.  Codes come from the group's least and largest element: offset = least,
step = (largest - least) / 15 rounded to dtype, code = (x - offset) / step to the nearest, ties to even.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
HEADS = ((32, 8, 128), (32, 8, 128), (40, 10, 128), (64, 8, 128), (12, 12, 64), (8, 1, 128), (8, 1, 256), (24, 8, 64))


def listed():
    llama8b = dict(heads=32, kv_heads=8, head_dim=128)
    phi3 = dict(heads=40, kv_heads=10, head_dim=128)
    return [
        # one decoded token of an 8B model: the smallest call there is
        dict(name="rotary_token", op="rotary", dtype="bf16", tokens=1, layout="half", rotary_dim=128, scaling="llama3", furthest=8192, **llama8b),
        # a prefill chunk of the same model
        dict(name="rotary_chunk", op="rotary", dtype="bf16", tokens=8192, layout="half", rotary_dim=128, scaling="llama3", furthest=131072, **llama8b),
        # wide heads of which a quarter is rotated, neighbours paired, positions stretched far past the trained length
        dict(name="rotary_partial", op="rotary", dtype="fp16", tokens=1337, layout="interleaved", rotary_dim=64, scaling="yarn", furthest=1000000,
             heads=16, kv_heads=4, head_dim=256),
        # the next decode step of a served batch
        dict(name="plan_decode", op="plan", requests=64, page=64, new="one", longest=16384, mix=1),
        # a step that mixes many decoding requests with prompts
        dict(name="plan_mixed", op="plan", requests=777, page=16, new="mixed", longest=32768, mix=2),
        # one new token for each request of a batch
        dict(name="append_batch", op="append", dtype="bf16", tokens=64, group=128, page=64, pages=512, **llama8b),
        # a prefill chunk, keys and values still inside the fused projection's output
        dict(name="append_chunk", op="append", dtype="fp16", tokens=8191, group=32, page=16, pages=1024, **phi3),
        # one request, a short context: latency only
        dict(name="attend_one", op="attention", dtype="bf16", requests=1, queries="one", shortest=777, longest=777, window=0, group=128, page=64,
             mix=3, **llama8b),
        # one request at the end of a long context
        dict(name="attend_long", op="attention", dtype="fp16", requests=1, queries="one", shortest=131071, longest=131071, window=0, group=64,
             page=64, mix=4, **llama8b),
        # a served batch of decoding requests with contexts of very different lengths
        dict(name="attend_batch", op="attention", dtype="bf16", requests=64, queries="one", shortest=512, longest=16384, window=0, group=128,
             page=16, mix=5, **llama8b),
        # drafted tokens of several requests checked at once, a sliding window
        dict(name="attend_drafts", op="attention", dtype="fp16", requests=17, queries="drafts", shortest=100, longest=12000, window=4096, group=32,
             page=32, mix=6, **phi3),
        # prompts in chunks behind cached contexts, decoding requests among them
        dict(name="attend_chunks", op="attention", dtype="bf16", requests=3, queries="chunks", shortest=4096, longest=16384, most=2048,
             window=0, group=128, page=64, mix=7, **llama8b),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case; drawn again while it would move more bytes or multiply more than any listed case."""
    most = {k: max(work(c)[k] for c in listed()) for k in ("bytes", "flops")}
    widest = [max(x) for x in zip(*map(_padded, listed()))]
    while True:
        c = _draw(rng)
        if all(work(c)[k] <= most[k] for k in most) and all(x <= y for x, y in zip(_padded(c), widest)):
            return c


def _draw(rng):
    op = rng.choice(("rotary", "plan", "append", "append", "attention", "attention", "attention", "attention"))
    if op == "plan":
        return dict(op=op, requests=_log(rng, 1, 2000), page=rng.choice((16, 32, 64, 128)), new=rng.choice(("one", "mixed")),
                    longest=_log(rng, 64, 65536), mix=rng.randrange(1 << 30))
    heads, kv_heads, head_dim = rng.choice(HEADS)
    c = dict(op=op, dtype=rng.choice(("fp16", "bf16")), heads=heads, kv_heads=kv_heads, head_dim=head_dim)
    if op == "rotary":
        c.update(tokens=_log(rng, 1, 8192), layout=rng.choice(("half", "interleaved")), rotary_dim=rng.choice((head_dim, head_dim, head_dim // 2, 32)),
                 scaling=rng.choice(("none", "linear", "llama3", "yarn")), furthest=_log(rng, 64, 1000000))
        return c
    c.update(group=rng.choice([g for g in (32, 64, 128) if g <= head_dim]), page=rng.choice((16, 32, 64, 128)))
    if op == "append":
        c.update(tokens=_log(rng, 1, 8192))
        c["pages"] = -(-c["tokens"] // c["page"]) + rng.randrange(1, 200)
        return c
    queries = rng.choice(("one", "one", "one", "drafts", "chunks"))
    c.update(queries=queries, requests=_log(rng, 1, {"one": 256, "drafts": 64, "chunks": 8}[queries]),
             longest=_log(rng, 1, {"one": 131072, "drafts": 32768, "chunks": 8192}[queries]), mix=rng.randrange(1 << 30))
    c["shortest"] = _log(rng, 1, c["longest"])
    c["window"] = rng.choice((0, 0, 0, _log(rng, 16, 8192)))
    if queries == "chunks":
        c["most"] = _log(rng, 16, 2048)
    return c


def _lengths(case):
    """Cached and new tokens of each request of a "plan", all and new tokens of each of an "attention"."""
    rng = random.Random(case["mix"])
    n = case["requests"]
    if case["op"] == "plan":
        before = [_log(rng, 1, case["longest"]) if rng.random() < 0.9 else 0 for _ in range(n)]
        if case["new"] == "one":
            return before, [1] * n
        return before, [_log(rng, 2, 1024) if rng.random() < 0.15 else rng.choice((0, 1, 1, 1, 1, 5)) for _ in range(n)]
    total = [_log(rng, case["shortest"], case["longest"]) for _ in range(n)]
    if n > 1:
        total[rng.randrange(n)] = case["longest"]
    if case["queries"] == "one":
        new = [1] * n
    elif case["queries"] == "drafts":
        new = [min(t, rng.randrange(2, 9)) for t in total]
    else:
        new = [min(t, _log(rng, 1, case["most"]) if i % 2 else case["most"]) for i, t in enumerate(total)]
    return total, new


def _padded(case):
    """Elements of the keys, and of the scores, when every request is as long as the longest: what the plain form holds."""
    if case["op"] != "attention":
        return 0, 0
    total, new = _lengths(case)
    longest = case["requests"] * max(total)
    return longest * case["kv_heads"] * case["head_dim"], longest * max(new) * case["heads"]


def _seen(case):
    """Over all requests: cached tokens that some query sees, and pairs of a query and a token that it sees."""
    keys = pairs = 0
    for t, n in zip(*_lengths(case)):
        w = case["window"] or t
        keys += min(t, w + n - 1)
        short = max(0, min(n, w - (t - n) - 1))              # queries so early that the window reaches before the first token
        pairs += (n - short) * w + sum(range(t - n + 1, t - n + 1 + short))
    return keys, pairs


def work(case):
    op = case["op"]
    if op == "plan":
        before, new = _lengths(case)
        pages = sum(-(-(b + n) // case["page"]) + -(-b // case["page"]) for b, n in zip(before, new))
        given = sum(-(-(b + n) // case["page"]) - -(-b // case["page"]) for b, n in zip(before, new))
        return {"bytes": 16 * case["requests"] + 16 * sum(new) + 8 * given + 4 * min(pages, sum(new)), "flops": 4 * case["requests"] + 4 * sum(new)}
    row = (case["heads"] + case["kv_heads"]) * case["head_dim"]
    if op == "rotary":
        turned = (case["heads"] + case["kv_heads"]) * case["rotary_dim"]
        return {"bytes": case["tokens"] * (4 * row + 8) + 4 * case["rotary_dim"], "flops": 3 * case["tokens"] * turned}
    cached = case["kv_heads"] * (case["head_dim"] + 8 * case["head_dim"] // case["group"])      # keys and values of a token in the cache
    dense = 4 * case["kv_heads"] * case["head_dim"]                                             # and in 16 bits
    if op == "append":
        return {"bytes": case["tokens"] * (2 * cached + 2 * dense + 16), "flops": 10 * case["tokens"] * case["kv_heads"] * case["head_dim"]}
    keys, pairs = _seen(case)
    rows = sum(_lengths(case)[1])
    return {"bytes": keys * cached + 4 * rows * case["heads"] * case["head_dim"] + 4 * (keys // case["page"]) + 8 * case["requests"],
            "flops": 4 * pairs * case["heads"] * case["head_dim"]}


# ---- inputs -----------------------------------------------------------------------------------------------

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _keys_values(case, g, rows):
    """Keys with a few channels that are large for every token, as models have them, and plain values: [rows, kv_heads, head_dim]."""
    shape = (rows, case["kv_heads"], case["head_dim"])
    dtype = DTYPES[case["dtype"]]
    bias = torch.randn(shape[1:], generator=g, device="cuda")
    bias = torch.where(torch.rand(shape[1:], generator=g, device="cuda") < 0.05, 4 * bias, 0.2 * bias)
    k = (torch.randn(shape, generator=g, device="cuda") + bias).to(dtype)
    return k, _normal(g, shape, dtype, 0.5)


def _frequencies(case):
    """Rotation per position of each pair, 64 bits, and the factor of the rotated values."""
    r, base, far = case["rotary_dim"], 500000.0, 8192.0
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if case["scaling"] == "linear":
        return f / 8.0, 1.0
    if case["scaling"] == "llama3":          # slow pairs are slowed eightfold, fast ones kept, those between blended
        turns = far * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * (keep + (1 - keep) / 8.0), 1.0
    if case["scaling"] == "yarn":            # the same with a ramp over the pair's index, and warmer values
        def pair(turns):
            return r * math.log(far / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), r // 2 - 1)
        slow = ((torch.arange(r // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * (1 - slow + slow / 16.0), 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _attention_inputs(case, seed):
    """Keys and values by place in the cache, pages of each request in order, queries."""
    g = _generator(seed)
    total, new = _lengths(case)
    used = [-(-t // case["page"]) for t in total]
    pages = sum(used) + 3
    k, v = _keys_values(case, g, pages * case["page"])
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(total), max(used)), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    q = _normal(g, (sum(new), case["heads"], case["head_dim"]), DTYPES[case["dtype"]])
    return k, v, table, q, total, new


def prepare(case, seed):
    g = _generator(seed)
    dev = torch.device("cuda")
    if case["op"] == "plan":
        before, new = _lengths(case)
        page = case["page"]
        have = [-(-b // page) for b in before]
        width = max(-(-(b + n) // page) for b, n in zip(before, new)) + 1
        given = sum(-(-(b + n) // page) - h for b, n, h in zip(before, new, have))
        order = torch.randperm(sum(have) + given + 11, generator=g, device="cuda").to(torch.int32).cpu()
        table = torch.zeros((len(before), width), dtype=torch.int32)
        at = 0
        for b, n in enumerate(have):
            table[b, :n] = order[at:at + n]
            at += n
        return dict(case=case, lengths=torch.tensor(before, dtype=torch.int32, device=dev), new=torch.tensor(new, dtype=torch.int32, device=dev),
                    table=table.to(dev), free=order[at:].to(dev), free_count=torch.tensor([given + 11], dtype=torch.int32, device=dev),
                    tokens=sum(new) + 5)
    heads, kv_heads, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rotary":
        qkv = _normal(g, (case["tokens"], (heads + 2 * kv_heads) * d), DTYPES[case["dtype"]])
        q, k, _ = (x.unflatten(-1, (-1, d)) for x in qkv.split([heads * d, kv_heads * d, kv_heads * d], dim=-1))
        f, factor = _frequencies(case)
        start = torch.randint(0, case["furthest"], (1,), generator=g, device="cuda")
        positions = (start + torch.arange(case["tokens"], device="cuda")) % case["furthest"]
        return dict(case=case, q=q, k=k, positions=positions, frequencies=f.cuda(), factor=factor)
    if case["op"] == "append":
        k, v = _keys_values(case, g, case["tokens"])
        qkv = torch.empty((case["tokens"], (heads + 2 * kv_heads) * d), dtype=k.dtype, device="cuda")
        qkv[:, heads * d:] = torch.cat((k.flatten(1), v.flatten(1)), dim=1)
        _, k, v = (x.unflatten(-1, (-1, d)) for x in qkv.split([heads * d, kv_heads * d, kv_heads * d], dim=-1))
        page = case["page"]
        cache = torch.zeros((case["pages"], kv_heads, page // 16 * _cell_bytes(case)), dtype=torch.uint8, device="cuda")
        if case["tokens"] <= case["pages"]:                  # a token here and there: one for each request
            slots = torch.randperm(case["pages"], generator=g, device="cuda")[:case["tokens"]] * page
            slots += torch.randint(0, page, slots.shape, generator=g, device="cuda")
        else:                                                # a run of tokens over pages in any order
            pages = torch.randperm(case["pages"], generator=g, device="cuda")[:-(-case["tokens"] // page)]
            slots = (pages[:, None] * page + torch.arange(page, device="cuda")).flatten()[:case["tokens"]]
        return dict(case=case, k=k, v=v, cache=cache, slots=slots)
    k, v, table, q, total, new = _attention_inputs(case, seed)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    shape = (-1, case["page"], kv_heads, d)
    cache = _pack(case, *_codes(case, k.view(shape).transpose(1, 2)), *_codes(case, v.view(shape).transpose(1, 2)))
    return dict(case=case, q=q, cache=cache, table=table, lengths=torch.tensor(total, dtype=torch.int32, device=dev),
                starts=torch.tensor(starts, dtype=torch.int32, device=dev), longest=max(total), most=max(new))


# ---- one pass ----------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _own(case, state)
    return {"rotary": _rotary, "plan": _plan, "append": _append, "attention": _attention}[case["op"]](case, state)


def _own(case, s):
    from decdec_b200 import kv4

    if case["op"] == "rotary":
        q, k = kv4.rotary(s["q"], s["k"], s["positions"], s["frequencies"], interleaved=case["layout"] == "interleaved", factor=s["factor"])
        return {"q": q, "k": k}
    if case["op"] == "plan":
        p = kv4.plan(s["lengths"], s["new"], s["table"], s["free"], s["free_count"], case["page"], s["tokens"])
        return {"positions": p.positions, "slots": p.slots, "query_starts": p.query_starts, "lengths": p.lengths, "table": s["table"],
                "free_count": p.free_count, "status": p.status}
    if case["op"] == "append":
        kv4.append(s["cache"], s["k"], s["v"], s["slots"], case["group"])
        k, v = kv4.gather(s["cache"], s["slots"], case["head_dim"], case["group"], s["k"].dtype)
        return {"k": k, "v": v}
    out = kv4.attention(s["q"], s["cache"], s["table"], s["lengths"], s["starts"], case["group"], max_queries=s["most"], window=case["window"])
    return {"out": out}


# ---- the cache's format ------------------------------------------------------------------------------------

def _cell_bytes(case):
    return 16 * (case["head_dim"] + 8 * case["head_dim"] // case["group"])


def _codes(case, x):
    """Codes of the elements, and step and offset of each group; 64 bits, since a code next to a border must not flip."""
    y = x.unflatten(-1, (-1, case["group"]))
    lo, hi = y.amin(-1), y.amax(-1)
    step = ((hi.double() - lo.double()) / 15).to(x.dtype)
    lo = torch.where(torch.isfinite(step), lo, torch.nan)
    step = torch.where(torch.isfinite(step), step, 0)
    code = torch.where(step[..., None] > 0, (y.double() - lo.double()[..., None]) / step.double()[..., None], 0.0)
    return code.round_().clamp_(0, 15).nan_to_num_(0).to(torch.uint8).flatten(-2), step, lo


def _words(code):
    """Four codes in a 16-bit word."""
    c = code.unflatten(-1, (-1, 4)).to(torch.int32)
    w = c[..., 0] | c[..., 1] << 4 | c[..., 2] << 8 | c[..., 3] << 12
    return torch.where(w >= 32768, w - 65536, w).to(torch.int16)


def _bytes(x):
    return x.contiguous().view(torch.uint8)


def _pack(case, k, k_step, k_lo, v, v_step, v_lo):
    """[pages, kv_heads, page, head_dim] codes, [..., groups] steps and offsets -> the cache."""
    d = case["head_dim"]
    blocks = max(1, d // 128)
    kw = _words(k).unflatten(2, (-1, 16)).unflatten(-1, (blocks, -1, 4, 2))               # page, head, cell, token, block, word, four, half
    kw = kw.permute(0, 1, 2, 4, 3, 6, 5, 7)
    vw = _words(v).unflatten(2, (-1, 2, 4, 2)).unflatten(-1, (blocks, -1, 2, 8))          # page, head, cell, 8, pair, token, block, word, half, eight
    vw = vw.permute(0, 1, 2, 6, 3, 9, 4, 7, 8, 5)
    ks = torch.stack((k_step, k_lo), -1).unflatten(2, (-1, 16))
    vs = torch.stack((v_step, v_lo), -1).unflatten(2, (-1, 16))
    return torch.cat([_bytes(x.flatten(3)) for x in (kw, vw, ks, vs)], dim=-1).flatten(2)


def _unpack(case, cache):
    """The cache -> keys and values [pages, kv_heads, page, head_dim] in 32 bits."""
    d, groups = case["head_dim"], case["head_dim"] // case["group"]
    blocks = max(1, d // 128)
    cells = cache.unflatten(2, (-1, _cell_bytes(case)))
    kw, vw, ks, vs = cells.split([8 * d, 8 * d, 64 * groups, 64 * groups], dim=-1)
    shift = torch.tensor([0, 4, 8, 12], dtype=torch.int32, device=cache.device)

    def code(words):
        return ((words.contiguous().view(torch.int16).to(torch.int32)[..., None] >> shift) & 15).float()

    k = code(kw).unflatten(3, (blocks, 16, 4, -1, 2)).permute(0, 1, 2, 4, 3, 6, 5, 7, 8).flatten(4).flatten(2, 3)
    v = code(vw).unflatten(3, (blocks, 2, 8, 4, -1, 2, 2)).permute(0, 1, 2, 4, 6, 9, 3, 7, 8, 5, 10).flatten(6).flatten(2, 5)

    def value(c, steps):
        s = steps.contiguous().view(DTYPES[case["dtype"]]).float().unflatten(3, (16, groups, 2)).flatten(2, 3)
        return (s[..., 1:] + s[..., :1] * c.unflatten(-1, (groups, -1))).flatten(-2)

    return value(k, ks), value(v, vs)


# ---- plain forms -------------------------------------------------------------------------------------------

def _rotary(case, s):
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = (f(angle).float()[:, None] for f in (torch.cos, torch.sin))
    r, half = case["rotary_dim"], case["layout"] == "half"

    def turn(x):
        y = x[..., :r].float()
        a, b = y.chunk(2, -1) if half else (y[..., ::2], y[..., 1::2])
        pair = [(a * cos - b * sin) * s["factor"], (b * cos + a * sin) * s["factor"]]
        y = torch.cat(pair, -1) if half else torch.stack(pair, -1).flatten(-2)
        return torch.cat((y.to(x.dtype), x[..., r:]), -1)

    return {"q": turn(s["q"]), "k": turn(s["k"])}


def _plan(case, s):
    page, n = case["page"], s["new"].long()
    before, free_count, width = s["lengths"].long(), s["free_count"].long(), s["table"].shape[1]
    total = before + n
    have = (before + page - 1) // page
    need = (total + page - 1) // page - have
    first = need.cumsum(0) - need
    starts = torch.nn.functional.pad(n.cumsum(0), (1, 0))
    short = need.sum() > free_count
    status = short + 2 * (total > width * page).any() + 4 * (starts[-1:] > s["tokens"]) + 8 * ((n < 0) | (before < 0)).any()
    ok = status == 0
    column = torch.arange(width, device=n.device)
    fresh = ok & (column >= have[:, None]) & (column < (have + need)[:, None])
    taken = (free_count - 1 - first[:, None] - (column - have[:, None])).clamp(0, len(s["free"]) - 1)
    s["table"].copy_(torch.where(fresh, s["free"][taken], s["table"]))
    t = torch.arange(s["tokens"], device=n.device)
    request = torch.searchsorted(starts[1:], t, right=True).clamp(max=len(n) - 1)
    used = ok & (t < starts[-1])
    positions = torch.where(used, before[request] + t - starts[request], 0)
    slots = torch.where(used, s["table"][request, positions // page].long() * page + positions % page, -1)
    return {"positions": positions, "slots": slots, "query_starts": (starts * ok).int(), "lengths": torch.where(ok, total, before).int(),
            "table": s["table"], "free_count": (free_count - need.sum() * ok).int(), "status": status.int()}


def _append(case, s):
    cells = s["cache"].unflatten(2, (-1, _cell_bytes(case)))
    page, cell, token = s["slots"] // case["page"], s["slots"] % case["page"] // 16, s["slots"] % 16
    d, groups = case["head_dim"], case["head_dim"] // case["group"]
    blocks = max(1, d // 128)
    index = torch.arange(8 * d // 2, device=token.device)
    kw = index.view(blocks, 16, 4, -1, 2).permute(1, 0, 3, 2, 4).flatten(1)                            # token -> its words of the key codes
    vw = index.view(blocks, 2, 8, 4, -1, 2, 2).permute(1, 3, 6, 0, 4, 5, 2).flatten(0, 2).flatten(1)    # and of the value codes
    pairs = torch.arange(16 * groups * 2, device=token.device).view(16, -1)
    words = cells.view(torch.int16)
    for_k, for_v = (_codes(case, s[x]) for x in ("k", "v"))
    head = torch.arange(case["kv_heads"], device=token.device)[:, None]
    page, cell = page[:, None, None], cell[:, None, None]
    for_steps = [torch.stack(x[1:], -1).flatten(2).view(torch.int16) for x in (for_k, for_v)]
    for_place = [kw[token], vw[token] + 4 * d, pairs[token] + 8 * d, pairs[token] + 8 * d + 32 * groups]
    place = torch.cat(for_place, 1)[:, None]
    words[page, head, cell, place] = torch.cat((_words(for_k[0]), _words(for_v[0]), *for_steps), -1)
    row = words[page, head, cell, place]
    shift = torch.tensor([0, 4, 8, 12], dtype=torch.int32, device=token.device)
    k, v = ((row[..., :d // 2].to(torch.int32)[..., None] >> shift) & 15).flatten(2).float().split(d, -1)
    steps = row[..., d // 2:].contiguous().view(DTYPES[case["dtype"]]).float().unflatten(-1, (2, groups, 2))

    def value(c, t):
        return (t[..., 1:] + t[..., :1] * c.unflatten(-1, (groups, -1))).flatten(-2).to(s["k"].dtype)

    return {"k": value(k, steps[..., 0, :, :]), "v": value(v, steps[..., 1, :, :])}


def _attention(case, s):
    q, starts, lengths = s["q"], s["starts"].long(), s["lengths"].long()
    kv_heads, d, page = case["kv_heads"], case["head_dim"], case["page"]
    ratio = case["heads"] // kv_heads
    k, v = (x[s["table"].long()].transpose(1, 2).flatten(2, 3) for x in _unpack(case, s["cache"]))       # request, head, token, element
    token = torch.arange(k.shape[2], device=q.device)
    i = torch.arange(s["most"], device=q.device)
    new = starts[1:] - starts[:-1]
    row = (starts[:-1, None] + i).clamp(max=len(q) - 1)
    rows = q[row].float().unflatten(2, (kv_heads, ratio)).permute(0, 2, 3, 1, 4)                       # request, head, its queries, i, element
    score = (rows.flatten(2, 3) @ k.transpose(2, 3)).unflatten(2, (ratio, -1)) * d ** -0.5
    at = (lengths - new)[:, None] + i                                                                  # position of a query
    seen = (token <= at[..., None]) & (i < new[:, None])[..., None]
    if case["window"]:
        seen &= token > at[..., None] - case["window"]
    seen = seen[:, None, None]
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    weight = torch.where(seen, (score - top).exp_(), 0.0)
    total = weight.sum(-1, keepdim=True)
    out = (weight.flatten(2, 3) @ v).unflatten(2, (ratio, -1)) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3).to(q.dtype)                                         # request, i, query head, element
    t = torch.arange(len(q), device=q.device)
    request = torch.searchsorted(starts[1:], t, right=True)
    return {"out": out[request, t - starts[request]]}


# ---- results from the definitions, 64 bits -----------------------------------------------------------------

def _held(x, group):
    """What the cache holds for x: 64 bits from the definition."""
    y = x.double().unflatten(-1, (-1, group))
    least, largest = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
    step = ((largest - least) / 15).to(x.dtype).double()
    code = torch.where(step > 0, ((y - least) / torch.where(step > 0, step, 1.0)).round(), 0.0).clamp(0, 15)
    return (least + code * step).flatten(-2)


def exact(case, seed):
    if case["op"] == "plan":
        s = {k: v.cpu() if torch.is_tensor(v) else v for k, v in prepare(case, seed).items()}
        page, left, table = case["page"], int(s["free_count"]), s["table"].clone()
        positions, slots, starts, lengths = [], [], [0], []
        for b, (have, new) in enumerate(zip(s["lengths"].tolist(), s["new"].tolist())):
            for p in range(have, have + new):
                if p % page == 0:
                    left -= 1
                    table[b, p // page] = s["free"][left]
                positions.append(p)
                slots.append(int(table[b, p // page]) * page + p % page)
            starts.append(starts[-1] + new)
            lengths.append(have + new)
        rest = s["tokens"] - len(slots)
        return {"positions": torch.tensor(positions + [0] * rest), "slots": torch.tensor(slots + [-1] * rest),
                "query_starts": torch.tensor(starts, dtype=torch.int32), "lengths": torch.tensor(lengths, dtype=torch.int32), "table": table,
                "free_count": torch.tensor([left], dtype=torch.int32), "status": torch.zeros(1, dtype=torch.int32)}
    if case["op"] == "rotary":
        s = prepare(case, seed)
        angle = s["positions"].double().view(-1, 1, 1) * s["frequencies"]
        turn = torch.polar(torch.full_like(angle, s["factor"]), angle)
        found = {}
        for name in ("q", "k"):
            x, r = s[name].double(), case["rotary_dim"]
            pairs = x[..., :r].unflatten(-1, (2, -1)).transpose(-1, -2) if case["layout"] == "half" else x[..., :r].unflatten(-1, (-1, 2))
            y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            found[name] = torch.cat(((y.transpose(-1, -2) if case["layout"] == "half" else y).flatten(-2), x[..., r:]), -1)
        return found
    if case["op"] == "append":
        s = prepare(case, seed)
        return {"k": _held(s["k"], case["group"]), "v": _held(s["v"], case["group"])}
    k, v, table, q, total, new = _attention_inputs(case, seed)
    page, ratio = case["page"], case["heads"] // case["kv_heads"]
    k, v = (x.unflatten(0, (-1, page)) for x in (k, v))
    out, at = torch.empty(q.shape, dtype=torch.float64, device=q.device), 0
    for b, (t, n) in enumerate(zip(total, new)):
        pages = table[b, :-(-t // page)].long()
        first = max(0, t - n + 1 - case["window"]) if case["window"] else 0
        position = torch.arange(t - n, t, device=q.device)[:, None]
        token = torch.arange(first, t, device=q.device)
        hidden = token > position
        if case["window"]:
            hidden |= token <= position - case["window"]
        for h in range(case["kv_heads"]):
            kh, vh = (_held(x[pages, :, h].flatten(0, 1)[first:t], case["group"]) for x in (k, v))
            for j in range(h * ratio, (h + 1) * ratio):
                score = (q[at:at + n, j].double() @ kh.T / math.sqrt(case["head_dim"])).masked_fill_(hidden, -math.inf)
                out[at:at + n, j] = score.softmax(-1) @ vh
        at += n
    return {"out": out}
