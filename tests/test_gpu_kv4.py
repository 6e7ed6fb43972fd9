"""The 4-bit key/value cache on the GPU against plain 64-bit restatements: rotary positions, the plan of a step, rows into the
cache and out of it, attention, and a run of them together."""
import math

import numpy as np
import pytest
import torch

from . import kv4_reference as R

pytestmark = pytest.mark.gpu

FORMATS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128)]
TYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def kv4():
    assert torch.cuda.is_available()
    from decdec_b200 import kv4 as m
    return m


def normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


# ---- rotary positions ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(128, 128), (128, 64), (64, 16), (96, 96), (40, 12), (256, 2), (80, 32)])
@pytest.mark.parametrize("tokens", [1, 7])
def test_rotary(kv4, dtype, interleaved, d, r, tokens):
    frequencies, factor = kv4.rotary_frequencies(r, 10000.0, {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096})
    q, k = normal((tokens, 5, d), dtype, 1), normal((tokens, 2, d), dtype, 2)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=torch.Generator().manual_seed(3))
    positions[0] = (1 << 20) + 1
    got = kv4.rotary(q.cuda(), k.cuda(), positions.cuda(), frequencies, interleaved, factor)
    for x, y in zip((q, k), got):
        want = R.rotary(x, positions, frequencies.cpu(), interleaved, factor)
        # sine and cosine: an argument rounded to 24 bits of at most a turn (2 pi 2^-24 / 2), 2 units of the result; products and sums 3 roundings
        slack = 2.0 ** -24 * (math.pi + 2 + 4) * factor * 2 * x.double().abs().amax()
        assert ((y.cpu().double() - want).abs() <= R.HALF[dtype] * want.abs() + slack).all()
        assert torch.equal(y[..., r:].cpu(), x[..., r:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("at", [0, 8, 3])
def test_rotary_in_place_inside_a_fused_projection(kv4, interleaved, at):
    """Queries and keys are views of one tensor, at aligned and at odd offsets; the rest of it stays as it is."""
    frequencies, _ = kv4.rotary_frequencies(128)
    fused = normal((33, at + 8 * 128 + 5), torch.bfloat16, 4).cuda()
    before = fused.clone()
    q, k = fused[:, at:at + 512].unflatten(-1, (4, 128)), fused[:, at + 512:at + 768].unflatten(-1, (2, 128))
    positions = torch.arange(33, dtype=torch.int32, device="cuda") - 3
    wq, wk = kv4.rotary(q, k, positions, frequencies, interleaved)
    kv4.rotary(q, k, positions, frequencies, interleaved, out=(q, k))
    assert torch.equal(q, wq) and torch.equal(k, wk)
    assert torch.equal(fused[:, :at], before[:, :at]) and torch.equal(fused[:, at + 768:], before[:, at + 768:])
    want = R.rotary(before[:, at:at + 512].unflatten(-1, (4, 128)).cpu(), positions.cpu(), frequencies.cpu(), interleaved, 1.0)
    assert ((wq.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()


def test_rotary_without_keys_or_tokens(kv4):
    frequencies, _ = kv4.rotary_frequencies(64)
    q = normal((3, 2, 64), torch.float16, 5).cuda()
    pos = torch.zeros(3, dtype=torch.int64, device="cuda")
    y, none = kv4.rotary(q, None, pos, frequencies)
    assert none is None and torch.equal(y, q)                       # position 0 turns nothing
    y, k = kv4.rotary(q[:0], q[:0], pos[:0], frequencies)
    assert y.shape == (0, 2, 64) and k.shape == (0, 2, 64)
    q[1, 0, 3] = math.nan
    q[2, 1, 5] = math.inf
    y, _ = kv4.rotary(q, None, pos + 1, frequencies)
    want = R.rotary(q.cpu(), pos.cpu() + 1, frequencies.cpu(), False, 1.0)
    assert torch.equal(torch.isfinite(y).cpu(), torch.isfinite(want))


# ---- the plan of a step ----------------------------------------------------------------------------------------

def plan_by_hand(before, new, table, free, count, page, tokens):
    left, table = count, table.copy()
    positions, slots, starts, after = [], [], [0], []
    for b, (have, n) in enumerate(zip(before, new)):
        for p in range(have, have + n):
            if p % page == 0:
                left -= 1
                table[b, p // page] = free[left]
            positions.append(p)
            slots.append(int(table[b, p // page]) * page + p % page)
        starts.append(starts[-1] + n)
        after.append(have + n)
    rest = tokens - len(slots)
    return positions + [0] * rest, slots + [-1] * rest, starts, after, left, table


@pytest.mark.parametrize("requests", [0, 1, 2, 31, 511, 512, 513, 1500])
@pytest.mark.parametrize("page", [16, 48])
@pytest.mark.parametrize("seed", [0, 1])
def test_plan(kv4, requests, page, seed):
    rng = np.random.RandomState(seed + requests)
    before = [int(x) for x in rng.choice([0, 1, 15, 16, 17, 47, 48, 100, 333], requests)]
    new = [int(x) for x in rng.choice([0, 0, 1, 1, 1, 2, 16, 33, 200], requests)]
    width = max([1] + [-(-(a + b) // page) for a, b in zip(before, new)])
    wide = torch.full((requests, width + 3), -7, dtype=torch.int32)
    have = [-(-b // page) for b in before]
    need = sum(-(-(a + b) // page) - h for a, b, h in zip(before, new, have))
    order = rng.permutation(sum(have) + need + 2).astype(np.int32)
    at = 0
    for b, n in enumerate(have):
        wide[b, :n] = torch.from_numpy(order[at:at + n])
        at += n
    free = np.concatenate([order[at:], np.full(3, -99, np.int32)])         # places behind the count are not looked at
    tokens = sum(new) + seed * 7
    p, s, starts, after, left, want = plan_by_hand(before, new, wide.numpy(), free, need + 2, page, tokens)
    wide = wide.cuda()
    got = kv4.plan(torch.tensor(before, dtype=torch.int32).cuda(), torch.tensor(new, dtype=torch.int32).cuda(), wide[:, :width] if requests else wide,
                   torch.from_numpy(free).cuda(), torch.tensor([need + 2], dtype=torch.int32).cuda(), page, tokens)
    assert got.status.item() == 0 and got.free_count.item() == left
    assert got.positions.tolist() == p and got.slots.tolist() == s
    assert got.query_starts.tolist() == starts and got.lengths.tolist() == after
    assert np.array_equal(wide.cpu().numpy(), want)


@pytest.mark.parametrize("status,before,new,count,tokens", [
    (1, [16, 5], [17, 11], 1, 64),              # two pages wanted, one left
    (1, [0], [1], 99, 64),                       # a count above what the list holds
    (2, [60, 0], [5, 1], 3, 64),                 # 65 tokens in a row of four pages
    (4, [0, 0], [9, 8], 3, 16),
    (8, [-1, 0], [1, 1], 3, 64),
    (8, [3, 0], [1, -1], 3, 64),
    (3, [60, 0], [5, 40], 2, 64),
])
def test_plan_gives_all_or_nothing(kv4, status, before, new, count, tokens):
    table = torch.arange(100, 108, dtype=torch.int32).view(2, 4)[:len(before)].cuda()
    keep = table.clone()
    free = torch.arange(3, dtype=torch.int32, device="cuda")
    got = kv4.plan(torch.tensor(before, dtype=torch.int32).cuda(), torch.tensor(new, dtype=torch.int32).cuda(), table, free,
                   torch.tensor([count], dtype=torch.int32).cuda(), 16, tokens)
    assert got.status.item() == status
    assert (got.slots == -1).all() and (got.positions == 0).all() and (got.query_starts == 0).all()
    assert got.lengths.tolist() == before and got.free_count.item() == count and torch.equal(table, keep)


# ---- rows into the cache and out of it ---------------------------------------------------------------------------

def rows_with_corners(shape, dtype, seed, group):
    x = normal(shape, dtype, seed)
    tokens, heads, d = shape
    flat = x.view(tokens * heads, d // group, group)
    n = len(flat)
    big = torch.finfo(dtype).max
    flat[0 % n, 0] = 0.0
    flat[1 % n, 0] = -2.5                                             # all equal
    flat[2 % n, 0] = torch.tensor([big, -big] * (group // 2)).to(dtype)
    flat[3 % n, 0] = torch.arange(group).to(dtype)                    # codes on their borders
    flat[4 % n, 0] = torch.finfo(dtype).tiny * torch.arange(group).to(dtype)
    flat[5 % n, 0] = 1000.0
    flat[5 % n, 0, -1] = 1001.0 if dtype == torch.float16 else 1008.0
    flat[6 % n, 0, 3] = math.nan
    flat[7 % n, 0, 5] = math.inf
    flat[8 % n, 0, 1] = -math.inf
    flat[9 % n, 0] = torch.finfo(dtype).smallest_normal * 2.0 ** -7 * (torch.arange(group) % 5).to(dtype)     # subnormal
    return x


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", FORMATS)
@pytest.mark.parametrize("page,wide,strided", [(16, True, False), (48, False, True)])
def test_append_writes_the_format(kv4, dtype, d, group, page, wide, strided):
    """Every byte of the cache, those of other tokens included, and the rows read back."""
    tokens, heads, pages = 37, 3, 5
    k, v = rows_with_corners((tokens, heads, d), dtype, 11, group), rows_with_corners((tokens, heads, d), dtype, 12, group).flip(0).contiguous()
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(13))[:tokens]
    slots[5] = -1
    slots[6] = -1000
    size = page // 16 * R.cell_bytes(d, group)
    want = np.random.RandomState(14).randint(0, 256, (pages, heads, size)).astype(np.uint8)
    cache = torch.from_numpy(want).cuda()
    for t in range(tokens):
        if slots[t] >= 0:
            R.write_row(want, int(slots[t]), k[t], v[t], group, page)
    kk, vv = k.cuda(), v.cuda()
    if strided:                                                       # views of one projection at an odd offset
        fused = torch.zeros(tokens, 2 * heads * d + 3, dtype=dtype, device="cuda")
        fused[:, 1:1 + heads * d] = kk.flatten(1)
        fused[:, 1 + heads * d:1 + 2 * heads * d] = vv.flatten(1)
        kk, vv = fused[:, 1:1 + heads * d].unflatten(-1, (heads, d)), fused[:, 1 + heads * d:1 + 2 * heads * d].unflatten(-1, (heads, d))
    s = slots.cuda() if wide else slots.int().cuda()
    kv4.append(cache, kk, vv, s, group)
    got = cache.cpu().numpy()
    same = got == want
    nan = np.zeros_like(same)                                         # a NaN may have any bits
    steps = cell_steps(want, d, group, dtype)
    nan[..., :] = steps
    assert (same | nan).all()
    gk, gv = kv4.gather(cache, s, d, group, dtype)
    for x, y in ((k, gk), (v, gv)):
        ref = R.held(x, group)
        ref = torch.where(torch.isnan(ref), ref, ref.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max))
        ref[slots < 0] = 0
        y = y.cpu().double()
        assert torch.equal(torch.isnan(y), torch.isnan(ref))
        # one rounding to 32 bits and one to the type, which may have a subnormal step
        far = (y - ref).abs() > R.HALF[dtype] * 1.0001 * ref.abs() + 2.0 ** -25 * (dtype == torch.float16)
        assert not far[~torch.isnan(ref)].any()


def cell_steps(cache, d, group, dtype):
    """Marks the offsets that are NaN: two bytes each."""
    cell = R.cell_bytes(d, group)
    cells = cache.reshape(*cache.shape[:2], -1, cell)
    mark = np.zeros_like(cells, dtype=bool)
    pairs = torch.from_numpy(cells[..., 16 * d:].copy()).view(dtype).reshape(*cells.shape[:3], -1, 2)
    nan = torch.isnan(pairs[..., 1]).numpy()
    m = mark[..., 16 * d:].reshape(*cells.shape[:3], -1, 4)
    m[..., 2:4] = nan[..., None]
    mark[..., 16 * d:] = m.reshape(*cells.shape[:3], -1)
    return mark.reshape(cache.shape)


def test_append_codes_next_to_their_borders(kv4):
    """Elements on and just beside the borders between codes: offsets and steps whose quotients 32-bit division rounds onto a border."""
    for dtype in TYPES:
        g = torch.Generator().manual_seed(21)
        n = 4096
        lo = -(2.0 ** torch.randint(-2, 3, (n, 1), generator=g)) * (1 + torch.randint(0, 8, (n, 1), generator=g) / 8)
        span = 15 * 2.0 ** torch.randint(-4, 1, (n, 1), generator=g) * (1 + torch.randint(0, 4, (n, 1), generator=g) / 4)
        x = lo + span * (torch.randint(0, 31, (n, 32), generator=g) / 30)
        x[:, 0:1], x[:, 1:2] = lo, lo + span
        x = x.to(dtype)
        x[:, 2] = torch.finfo(dtype).smallest_normal
        x[:, 3] = -torch.finfo(dtype).smallest_normal
        x = x.view(-1, 2, 64)
        cache = kv4.empty_cache(len(x) // 16, 16, 2, 64, 32)
        slots = torch.arange(len(x), device="cuda")
        kv4.append(cache, x.cuda(), x.flip(0).cuda(), slots, 32)
        k, v = kv4.gather(cache, slots, 64, 32, dtype)
        for y, z in ((k, x), (v, x.flip(0))):
            ref = R.held(z, 32)
            assert ((y.cpu().double() - ref).abs() <= R.HALF[dtype] * 1.0001 * ref.abs() + 2.0 ** -24).all()


def test_append_and_gather_of_nothing(kv4):
    cache = kv4.empty_cache(2, 16, 2, 64, 32)
    x = torch.zeros(0, 2, 64, dtype=torch.float16, device="cuda")
    s = torch.zeros(0, dtype=torch.int64, device="cuda")
    kv4.append(cache, x, x, s, 32)
    k, v = kv4.gather(cache, s, 64, 32, torch.float16)
    assert k.shape == v.shape == (0, 2, 64) and not cache.any()


# ---- attention ---------------------------------------------------------------------------------------------------

class Batch:
    """Requests with keys and values of their own, entered into a cache whose other bytes are all ones (NaN steps and offsets)."""

    def __init__(self, kv4, lengths, queries, heads, kv_heads, d, group, dtype, page, seed, starts=None, scale_q=1.0):
        self.kv4, self.lengths, self.queries, self.group, self.d = kv4, lengths, queries, group, d
        self.table, pages = R.pages_of(lengths, page, 2, seed)
        self.cache = torch.full((pages, kv_heads, page // 16 * R.cell_bytes(d, group)), 255, dtype=torch.uint8, device="cuda")
        self.k = [normal((n, kv_heads, d), dtype, seed + 10 * b) for b, n in enumerate(lengths)]
        self.v = [normal((n, kv_heads, d), dtype, seed + 10 * b + 1, 0.3) + 0.1 for b, n in enumerate(lengths)]
        self.v = [x.to(dtype) for x in self.v]
        self.q = normal((sum(queries), heads, d), dtype, seed + 5, scale_q)
        self.slots = [torch.tensor([int(self.table[b, t // page]) * page + t % page for t in range(n)], dtype=torch.int64) for b, n in enumerate(lengths)]
        self.fill()
        self.starts = torch.tensor([0] + list(np.cumsum(queries)), dtype=torch.int32)

    def fill(self):
        if sum(self.lengths):
            self.kv4.append(self.cache, torch.cat(self.k).cuda(), torch.cat(self.v).cuda(), torch.cat(self.slots).cuda(), self.group)

    def run(self, q=None, **kw):
        q = self.q.cuda() if q is None else q
        # the rule that the kernel is chosen by: more than 64 rows (queries x heads of a key head) of a request, heads up to 128
        rows = min(kw.get("max_queries", len(q)), len(q)) * (q.shape[1] // self.cache.shape[1])
        self.dense = rows > 64 and self.d <= 128 and q.shape[1] // self.cache.shape[1] <= 256
        return self.kv4.attention(q, self.cache, self.table.cuda(), torch.tensor(self.lengths, dtype=torch.int32).cuda(), self.starts.cuda(), self.group, **kw)

    def check(self, out, lse=None, scale=None, window=0):
        scale = self.d ** -0.5 if scale is None else scale
        at = 0
        for b, n in enumerate(self.queries):
            want, bound, want_lse, by = R.attention(self.q[at:at + n], self.k[b], self.v[b], self.lengths[b], scale, window, self.group, self.dense)
            got = out[at:at + n].cpu().double()
            assert torch.equal(torch.isnan(got), torch.isnan(want)), b
            off = ((got - want).abs() - bound).nan_to_num(0.0)
            assert (off <= 0).all(), (b, off.max().item(), ((got - want).abs() / bound).nan_to_num(0.0).max().item())
            if lse is not None:
                l = lse[at:at + n].cpu().double()
                inf = torch.isinf(want_lse)
                assert torch.equal(inf, torch.isinf(l))
                assert ((l - want_lse)[~inf].abs() <= 2e-5 * (1 + want_lse[~inf].abs()) + by).all()
            at += n


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", FORMATS)
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (12, 1)])
def test_attention_one_query(kv4, dtype, d, group, heads, kv_heads):
    lengths = [1, 15, 16, 17, 63, 130, 700]
    b = Batch(kv4, lengths, [1] * len(lengths), heads, kv_heads, d, group, dtype, 32, 100)
    out, lse = b.run(max_queries=1, return_lse=True)
    b.check(out, lse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [0, 1, 16, 50])
@pytest.mark.parametrize("d,group,heads,kv_heads,page", [(128, 128, 8, 2, 16), (128, 32, 5, 1, 64), (64, 32, 6, 6, 48), (256, 64, 4, 2, 16)])
def test_attention_several_queries(kv4, dtype, window, d, group, heads, kv_heads, page):
    lengths, queries = [5, 40, 200, 33, 1, 257], [5, 3, 8, 0, 1, 40]
    b = Batch(kv4, lengths, queries, heads, kv_heads, d, group, dtype, page, 200)
    out, lse = b.run(window=window, return_lse=True, scale=0.2)
    b.check(out, lse, window=window, scale=0.2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d,group", FORMATS[:5])
@pytest.mark.parametrize("heads,kv_heads,window", [(4, 4, 0), (8, 2, 0), (5, 1, 0), (8, 2, 100), (33, 1, 300)])
def test_attention_of_chunks(kv4, dtype, d, group, heads, kv_heads, window):
    """Tiles of rows and steps of 128 tokens that end anywhere, requests with one query among them."""
    lengths, queries = [129, 1, 400, 128, 300, 17], [129, 1, 70, 5, 1, 17]
    b = Batch(kv4, lengths, queries, heads, kv_heads, d, group, dtype, 16, 250)
    out, lse = b.run(window=window, return_lse=True)
    assert b.dense
    b.check(out, lse, window=window)
    assert torch.equal(out, b.run(window=window))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_rows_that_see_nothing(kv4, dtype):
    """No tokens at all, no queries, and more queries than tokens: the first stand before the first token."""
    b = Batch(kv4, [0, 0, 20, 7, 3], [1, 0, 0, 7, 6], 4, 2, 128, 64, dtype, 16, 300)
    out, lse = b.run(return_lse=True)
    b.check(out, lse)
    assert (out[0] == 0).all() and (out[8:11] == 0).all() and (lse[8:11] == -math.inf).all()


@pytest.mark.parametrize("queries", [1, 4, 40])
def test_attention_poison_behind_the_mask(kv4, queries):
    """NaN and infinities in tokens that a row does not see: later ones, ones before the window."""
    b = Batch(kv4, [90, 64], [queries, queries], 8, 2, 128, 64, torch.bfloat16, 16, 400)
    window = 45
    b.k[0][3, 0, 5] = math.nan
    b.v[0][7, 1, 70] = math.inf
    b.fill()
    first = [n - queries - window + 1 for n in b.lengths]
    assert first[0] > 7 or queries == 40
    out, lse = b.run(window=window, return_lse=True, max_queries=queries)
    b.check(out, lse, window=window)
    if queries > 1:                                                    # the last token is no number: only the last row sees it
        b.k[1][-1] = math.nan
        b.v[0][-1, :, 3] = -math.inf
        b.fill()
        out = b.run(window=window, max_queries=queries)
        b.check(out, window=window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["uniform", "sharp", "rising", "large", "tiny", "silent"])
@pytest.mark.parametrize("queries", [2, 33])
def test_attention_of_extreme_scores_and_values(kv4, dtype, kind, queries):
    b = Batch(kv4, [500, 33], [1, queries], 8, 2, 128, 32, dtype, 32, 500)
    if kind == "uniform":
        b.q.zero_()
    elif kind == "sharp":
        b.q *= 40
    elif kind == "rising":                                             # the maximum moves with every cell, steps grow too
        for k, v in zip(b.k, b.v):
            k += torch.linspace(0, 6, len(k))[:, None, None].to(dtype)
            v *= torch.logspace(-3, 3, len(v))[:, None, None].to(dtype)
        b.q = b.q.abs()
    elif kind == "large":
        b.q *= 100
        for k, v in zip(b.k, b.v):
            k *= 0.01
            v *= 5000
    elif kind == "silent":                                             # no values at all for the first tokens, then some
        for k, v in zip(b.k, b.v):
            v[:20] = 0
            v[20:] *= 3
    else:
        for k, v in zip(b.k, b.v):
            v *= 2.0 ** -9
            v[::2] = 0
    b.fill()
    out, lse = b.run(return_lse=True)
    b.check(out, lse)


def test_attention_does_not_depend_on_how_the_work_is_cut(kv4):
    """The same request alone and in batches of other lengths (whose thread blocks begin elsewhere) differs by rounding only; equal calls
    give equal bits."""
    lengths = [3000, 17, 1200, 1, 801]
    b = Batch(kv4, lengths, [1] * 5, 8, 2, 128, 128, torch.float16, 16, 600)
    out = b.run(max_queries=1)
    assert torch.equal(out, b.run(max_queries=1))
    b.check(out)
    for i in range(5):
        alone = kv4.attention(b.q[i:i + 1].cuda(), b.cache, b.table[i:i + 1].cuda(), torch.tensor([lengths[i]], dtype=torch.int32).cuda(),
                              torch.tensor([0, 1], dtype=torch.int32).cuda(), 128)
        assert (alone[0].double() - out[i].double()).abs().max() <= 2.0 ** -10 * out[i].abs().max() + 2e-4


@pytest.mark.parametrize("queries", [1, 40])
def test_attention_near_the_ends_of_bf16(kv4, queries):
    """Queries, keys and values of magnitudes that fp16 does not hold: scaled to it by powers of two, here and there with zeros."""
    b = Batch(kv4, [300, 64], [queries, 1], 8, 2, 128, 64, torch.bfloat16, 16, 650)
    b.q *= 2.0 ** 90
    for k, v in zip(b.k, b.v):
        k *= 2.0 ** -90
        v *= 2.0 ** 100
        v[3::7] = 0
    b.fill()
    out, lse = b.run(return_lse=True)
    b.check(out, lse)
    for k, v in zip(b.k, b.v):
        k *= 2.0 ** 60
        v *= 2.0 ** -190
    b.q *= 2.0 ** -60
    b.fill()
    b.check(b.run())


@pytest.mark.parametrize("most", [1, 3, 500])
def test_attention_with_any_bound_of_queries(kv4, most):
    """max_queries chooses the kernel; requests with more rows, and with fewer, are computed all the same."""
    b = Batch(kv4, [150, 3, 64], [77, 1, 20], 8, 2, 128, 128, torch.bfloat16, 16, 660)
    out = b.run(max_queries=most)
    b.check(out)


def test_attention_without_requests_or_pages(kv4):
    q = normal((5, 4, 64), torch.float16, 41).cuda()
    cache = kv4.empty_cache(2, 16, 2, 64, 64)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    out, lse = kv4.attention(q, cache, none.view(0, 3), none, torch.zeros(1, dtype=torch.int32, device="cuda"), 64, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    starts = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda")
    out = kv4.attention(q, cache, none.view(2, 0), torch.zeros(2, dtype=torch.int32, device="cuda"), starts, 64)
    assert (out == 0).all()


def test_overlapping_outputs_are_refused(kv4):
    frequencies, _ = kv4.rotary_frequencies(64)
    x = normal((4, 4, 64), torch.float16, 42).cuda()
    pos = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError):
        kv4.rotary(x[:, :2], x[:, 2:], pos, frequencies, out=(x[:, :2], x[:, :2]))
    with pytest.raises(RuntimeError):
        kv4.rotary(x, None, pos, frequencies, out=(x[:1].expand(4, 4, 64), None))
    with pytest.raises(RuntimeError, match="must not share memory"):
        kv4.rotary(x[:3], None, pos[:3], frequencies, out=(x[1:], None))          # the same rows shifted by one
    packed = normal((4, 3, 3, 64), torch.float16, 43).cuda()                      # queries, keys and values side by side in every head
    q, k = packed[:, :, 0], packed[:, :, 1]
    want = kv4.rotary(q, k, pos + 5, frequencies)
    keep = packed[:, :, 2].clone()
    kv4.rotary(q, k, pos + 5, frequencies, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(packed[:, :, 2], keep)
    b = Batch(kv4, [9], [4], 4, 2, 64, 64, torch.float16, 16, 670)
    with pytest.raises(RuntimeError):
        kv4.attention(x, b.cache, b.table.cuda(), torch.tensor([9], dtype=torch.int32).cuda(), b.starts.cuda(), 64, out=x)
    one = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="must not overlap"):
        kv4.plan(n, n, one.expand(2, 4), n, n[:1], 16, 2)


def test_attention_many_requests(kv4):
    """More requests than threads of a block, most of them without queries."""
    lengths = [(i * 37) % 90 for i in range(300)]
    queries = [1 if i % 3 == 0 else 0 for i in range(300)]
    b = Batch(kv4, lengths, queries, 2, 1, 64, 64, torch.bfloat16, 16, 700)
    b.check(b.run(max_queries=1))


def test_attention_strided_queries_and_rows_behind_the_last(kv4):
    b = Batch(kv4, [40, 9], [3, 2], 4, 2, 128, 128, torch.float16, 16, 800)
    want = b.run()
    for offset in (0, 3):                                              # queries inside a wider tensor; aligned and not
        wide = torch.zeros(9, 4 * 128 + 16 + offset, dtype=torch.float16, device="cuda")
        wide[:5, offset:offset + 512] = b.q.cuda().flatten(1)
        wide[5:] = math.nan
        q = wide[:, offset:offset + 512].unflatten(-1, (4, 128))
        out = torch.full((9, 6, 128), 7.0, dtype=torch.float16, device="cuda")
        kv4.attention(q, b.cache, b.table.cuda(), torch.tensor(b.lengths, dtype=torch.int32).cuda(), b.starts.cuda(), 128, out=out[:, 1:5])
        assert torch.equal(out[:5, 1:5], want) and (out[5:] == 7).all() and (out[:, 0] == 7).all() and (out[:, 5] == 7).all()
        fresh, lse = kv4.attention(q, b.cache, b.table.cuda(), torch.tensor(b.lengths, dtype=torch.int32).cuda(), b.starts.cuda(), 128, return_lse=True)
        assert torch.equal(fresh[:5], want) and (fresh[5:] == 0).all() and (lse[5:] == -math.inf).all()
    none = kv4.attention(b.q[:0].cuda(), b.cache, b.table.cuda(), torch.tensor(b.lengths, dtype=torch.int32).cuda(), torch.zeros(3, dtype=torch.int32).cuda(), 128)
    assert none.shape == (0, 4, 128)


def test_cache_beyond_32_bit_offsets(kv4):
    """Pages that lie more than 2^32 bytes into the cache."""
    page, d, group, heads = 64, 128, 128, 8
    size = page // 16 * R.cell_bytes(d, group)
    pages = (1 << 32) // (heads * size) + 40
    cache = torch.empty((pages, heads, size), dtype=torch.uint8, device="cuda")
    assert cache.numel() > 1 << 32
    n = 200
    table = torch.tensor([[pages - 1, 1, pages - 30, pages - 7]], dtype=torch.int32)
    k, v, q = normal((n, heads, d), torch.float16, 31), normal((n, heads, d), torch.float16, 32), normal((1, 16, d), torch.float16, 33)
    slots = torch.tensor([int(table[0, t // page]) * page + t % page for t in range(n)])
    kv4.append(cache, k.cuda(), v.cuda(), slots.cuda(), group)
    gk, _ = kv4.gather(cache, slots.cuda(), d, group, torch.float16)
    assert ((gk.cpu().double() - R.held(k, group)).abs() <= 2.0 ** -10 * 1.01 * k.double().abs().amax()).all()
    out = kv4.attention(q.cuda(), cache, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda(), group)
    want, bound, _, _ = R.attention(q, k, v, n, d ** -0.5, 0, group)
    assert ((out.cpu().double() - want).abs() <= bound).all()


def test_bad_pages_slots_and_lengths_raise_the_error_of_the_stream(kv4):
    from decdec_b200 import ops
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        b = Batch(kv4, [100], [1], 4, 2, 128, 128, torch.float16, 16, 900)
        good = b.run()
        lens, starts = torch.tensor([100], dtype=torch.int32).cuda(), b.starts.cuda()
        x = torch.zeros(1, 2, 128, dtype=torch.float16, device="cuda")
        calls = []
        for page in (-1, b.cache.shape[0], 0x7fffffff):
            bad = b.table.clone()
            bad[0, 2] = page
            calls.append(lambda bad=bad.cuda(): kv4.attention(b.q.cuda(), b.cache, bad, lens, starts, 128))
        calls.append(lambda: kv4.attention(b.q.cuda(), b.cache, b.table.cuda(), lens + 1000, starts, 128))
        calls.append(lambda: kv4.append(b.cache, x, x, torch.tensor([b.cache.shape[0] * 16]).cuda(), 128))
        calls.append(lambda: kv4.gather(b.cache, torch.tensor([1 << 40]).cuda(), 128, 128, torch.float16))
        for call in calls:
            assert ops.stream_status() == 0
            call()
            torch.cuda.synchronize()
            assert ops.stream_status() == 3
            with pytest.raises(RuntimeError, match="outside the 4-bit cache"):
                b.run()
            ops.stream_reset()
            assert torch.equal(b.run(), good)


def test_captured_and_replayed_beside_other_streams(kv4):
    """Two graphs of one stream replayed at the same time, with eager calls on a third: no call uses another's workspace."""
    batches = [Batch(kv4, [900, 50], [1, 1], 8, 2, 128, 128, torch.bfloat16, 16, 1000 + i) for i in range(3)]
    inputs = [(x.q.cuda(), x.cache, x.table.cuda(), torch.tensor(x.lengths, dtype=torch.int32).cuda(), x.starts.cuda(), 128) for x in batches]
    want = [kv4.attention(*i) for i in inputs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in inputs[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kv4.attention(*i))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = kv4.attention(*inputs[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(third, want[2])


@pytest.mark.parametrize("queries", [1, 40])
def test_rows_appended_just_before_they_are_read(kv4, queries):
    """Launches begin while the call before them ends: new rows over ones that a gather and the attention before have read, without a pause."""
    lengths = [600, 131, 64]
    batches = [Batch(kv4, lengths, [queries] * 3, 8, 2, 128, 32, torch.float16, 16, 1100) for _ in range(2)]
    batches[1].k, batches[1].v = [x.flip(0) for x in batches[0].k], [x * -2 for x in batches[0].v]
    rows = [[torch.cat(x).cuda() for x in (b.k, b.v)] for b in batches]
    slots, cache = torch.cat(batches[0].slots).cuda(), batches[0].cache
    args = (batches[0].q.cuda(), cache, batches[0].table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), batches[0].starts.cuda(), 32)

    def turn(i, pause):
        held = kv4.gather(cache, slots, 128, 32, torch.float16)
        pause()
        kv4.append(cache, *rows[i], slots, 32)
        pause()
        return held + (kv4.attention(*args, max_queries=queries),)

    want = [turn(i % 2, torch.cuda.synchronize) for i in range(4)][2:]
    torch.cuda.synchronize()
    got = [turn(i % 2, lambda: None) for i in range(40)]
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(x, want[i % 2])), i


@pytest.mark.parametrize("queries", [1, 40])
@pytest.mark.parametrize("dtype,size,scale", [(torch.bfloat16, -30, None), (torch.float16, -23, None), (torch.bfloat16, -100, None), (torch.bfloat16, -60, 1e-30)])
def test_attention_of_small_queries(kv4, queries, dtype, size, scale):
    """Queries and scales whose product with the factors of keys lies below the fp32 range, at lengths that leave parts of a step without tokens."""
    b = Batch(kv4, [300, 64, 130], [queries] * 3, 8, 2, 128, 64, dtype, 16, 1200)
    b.q *= 2.0 ** size
    out, lse = b.run(return_lse=True, scale=scale)
    b.check(out, lse, scale=scale)


def test_tokens_without_values_count_in_the_sum(kv4):
    """One token in 129 has a value, 2^15, all others zeros and weights of 2^-11.5: together they are 4 % of the sum."""
    n, far = 32 + 4096, 11.5
    b = Batch(kv4, [n], [33], 2, 1, 128, 64, torch.float16, 64, 1300)
    b.q.zero_()
    b.q[:, :, 0] = 1
    b.k[0].zero_()
    b.k[0][:, :, 1::64] = 15                                           # steps of 1: the cache holds these keys and values exactly
    b.k[0][:32, :, 0] = 9
    b.v[0].zero_()
    b.v[0][:32] = 2.0 ** 15
    b.fill()
    out, lse = b.run(scale=far * math.log(2.0) / 9, return_lse=True)
    assert b.dense
    for i in range(33):
        total = 32 + (n - 32 - 32 + i) * 2.0 ** -far
        # half an fp16 step of the weights and of the output; scores in 32 bits
        assert ((out[i].double() / (2.0 ** 15 * 32 / total) - 1).abs() <= 2.0 ** -10 + 2.0 ** -16).all(), i
        assert ((lse[i].double() - (math.log(total) + far * math.log(2.0))).abs() <= 2.0 ** -16).all(), i


def test_weights_keep_their_bits_when_a_maximum_moves_within_a_step(kv4):
    """Every 32 tokens the largest score of a row grows by a factor 0.5 (1 + 0.9 * 2^-11) of its weights, whose rounding to fp16 is as large as can be, and
    that of the row beside it by 2^16, so that the sums of both are brought to another maximum four times in a step."""
    grow = 1 - math.log2(1 + 0.9 * 2.0 ** -11)
    b = Batch(kv4, [128], [33], 2, 1, 128, 64, torch.float16, 16, 1400)
    b.q.zero_()
    b.q[:, 0, 0], b.q[:, 1, 0] = 1, 16
    b.k[0].zero_()
    b.k[0][:, :, 1::64] = 15                                           # steps of 1, and of 1/16 for the values: held exactly
    b.k[0][:, 0, 0] = torch.arange(128) // 32
    b.v[0].zero_()
    b.v[0][:32] = 1 + (torch.arange(128) % 16) / 16
    b.fill()
    out = b.run(scale=grow * math.log(2.0))
    assert b.dense
    w = 2.0 ** (grow * (torch.arange(128) // 32).double())
    want = (w @ b.v[0][:, 0].double()) / w.sum()
    # half an fp16 step of the weights and of the output; scores in 32 bits
    assert ((out[32, 0].cpu().double() - want).abs() <= (2.0 ** -10 + 2.0 ** -16) * want).all()


@pytest.mark.parametrize("queries,keys,values", [(1, 0, 114), (40, 0, 125), (40, 123, 0), (1, 98, 0)])
def test_attention_of_large_bf16_numbers(kv4, queries, keys, values):
    """Values whose weighted sums, and keys whose scores, still fit 32 bits."""
    b = Batch(kv4, [70, 20], [queries, 1], 8, 2, 128, 64, torch.bfloat16, 16, 1500)
    for k, v in zip(b.k, b.v):
        k *= 2.0 ** keys
        v *= 2.0 ** values
    b.q *= 2.0 ** -min(keys, 98)
    b.fill()
    scale = 2.0 ** (min(keys, 98) - keys) * 128 ** -0.5
    out, lse = b.run(return_lse=True, max_queries=queries, scale=scale)
    assert torch.isfinite(out).all()
    b.check(out, lse, scale=scale)


def test_steps_next_to_the_middle_of_two_numbers(kv4):
    """(largest - least) / 15 a hair above, on and below the middle of two fp16 numbers: rounded as over the reals, ties to even."""
    from fractions import Fraction

    def to_half(x):                                                    # a positive number in the normal range
        e = 0
        while x >= Fraction(2) ** (e + 1):
            e += 1
        while x < Fraction(2) ** e:
            e -= 1
        n, unit = x / Fraction(2) ** (e - 10), Fraction(2) ** (e - 10)
        whole = n.numerator // n.denominator
        rest = n - whole
        return (whole + (rest > Fraction(1, 2) or (rest == Fraction(1, 2) and whole % 2 == 1))) * unit

    rng = np.random.RandomState(22)
    groups, want = [], []
    while len(groups) < 2048:
        e = int(rng.randint(-12, 8))
        span = 15 * Fraction(2 * int(rng.randint(1024, 2048)) + 1) * Fraction(2) ** (e - 11)         # 15 times a middle
        if span >= 65504:
            continue
        hi = Fraction(float(np.float16(float(span))))
        lo = float(hi - span)
        if Fraction(float(np.float16(lo))) != hi - span or lo == 0.0:
            continue
        for least in (np.float16(lo), np.nextafter(np.float16(lo), np.float16(-1)), np.nextafter(np.float16(lo), np.float16(1))):
            for sign in (1, -1):                                       # and mirrored
                ends = (float(least), float(hi)) if sign == 1 else (-float(hi), -float(least))
                groups.append(ends)
                want.append(float(to_half((Fraction(ends[1]) - Fraction(ends[0])) / 15)))
    groups.append((-3.0458e-05, 1.8671875))
    lo = float(np.float16(-3.0458e-05))
    want.append(float(to_half((Fraction(1.8671875) - Fraction(lo)) / 15)))
    groups, want = groups[:len(groups) // 16 * 16], want[:len(groups) // 16 * 16]
    x = torch.tensor(groups, dtype=torch.float64).repeat(1, 32).half().view(-1, 1, 64)       # one group of 64 a token
    cache = kv4.empty_cache(len(x) // 16, 16, 1, 64, 64)
    kv4.append(cache, x.cuda(), x.cuda(), torch.arange(len(x), device="cuda"), 64)
    steps = cache.view(len(x) // 16, -1).cpu()[:, 16 * 64:].contiguous().view(torch.float16).view(len(x) // 16, 2, 16, 2)
    for side in range(2):
        assert torch.equal(steps[:, side, :, 0].flatten().double(), torch.tensor(want, dtype=torch.float64))
        assert torch.equal(steps[:, side, :, 1].flatten(), x.amin(-1).flatten())


@pytest.mark.parametrize("queries", [2, 40])
def test_rows_before_the_first_request(kv4, queries):
    """query_starts that do not begin at 0: the rows before are nobody's, zeros in a fresh output and left as they are in a given one."""
    b = Batch(kv4, [50, 64], [queries, 1], 4, 2, 128, 128, torch.float16, 16, 810)
    want = b.run(max_queries=queries)
    q = torch.cat((torch.full((6, 4, 128), math.nan, dtype=torch.float16), b.q, torch.zeros(3, 4, 128, dtype=torch.float16))).cuda()
    b.starts += 6
    junk = [torch.full_like(q, 9.0) for _ in range(8)]                 # what a fresh output finds in its memory
    del junk
    out, lse = b.run(q=q, max_queries=queries, return_lse=True)
    assert (out[:6] == 0).all() and (lse[:6] == -math.inf).all() and torch.equal(out[6:-3], want) and (out[-3:] == 0).all()
    out = torch.full_like(q, 7.0)
    b.run(q=q, max_queries=queries, out=out)
    assert (out[:6] == 7).all() and torch.equal(out[6:-3], want) and (out[-3:] == 7).all()


def test_outputs_with_heads_before_tokens(kv4):
    """Queries, keys and outputs that are stored head by head, and rotary in place on them."""
    frequencies, _ = kv4.rotary_frequencies(64)
    q, k = normal((4, 7, 64), torch.float16, 44).cuda().transpose(0, 1), normal((2, 7, 64), torch.float16, 45).cuda().transpose(0, 1)
    pos = torch.arange(7, device="cuda")
    want = kv4.rotary(q.contiguous(), k.contiguous(), pos, frequencies)
    out = torch.empty_like(q.contiguous().transpose(0, 1).contiguous()).transpose(0, 1), torch.empty((2, 9, 64), dtype=torch.float16, device="cuda")[:, 1:8].transpose(0, 1)
    kv4.rotary(q, k, pos, frequencies, out=out)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    with pytest.raises(RuntimeError, match="must not share memory"):
        kv4.rotary(q[:6], None, pos[:6], frequencies, out=(q[1:], None))
    both = torch.cat((q, k), 1).transpose(0, 1).contiguous().transpose(0, 1)                 # queries and keys of one tensor, head by head
    kv4.rotary(both[:, :4], both[:, 4:], pos, frequencies, out=(both[:, :4], both[:, 4:]))
    assert torch.equal(both, torch.cat(want, 1))
    kv4.rotary(q, k, pos, frequencies, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    b = Batch(kv4, [40], [7], 4, 2, 64, 64, torch.float16, 16, 672)
    want = b.run()
    out = torch.full((4, 8, 64), 7.0, dtype=torch.float16, device="cuda")
    b.run(out=out[:, :7].transpose(0, 1))
    assert torch.equal(out[:, :7].transpose(0, 1), want) and (out[:, 7] == 7).all()
    with pytest.raises(RuntimeError, match="must not share memory"):
        b.run(out=out.flatten()[:448 + 64].as_strided((7, 4, 64), (64, 64, 1)))              # heads that lie over the tokens


def test_outputs_over_caches_and_tables_are_refused(kv4):
    """What a call writes may not lie over the cache, tables, lengths or slots that it reads."""
    b = Batch(kv4, [40], [4], 4, 2, 64, 64, torch.float16, 16, 674)
    memory = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    out = memory[:4 * 4 * 64 * 2].view(torch.float16).view(4, 4, 64)
    over = memory[16:48].view(torch.int32)                             # inside the output's memory
    lens, table = torch.tensor([40], dtype=torch.int32, device="cuda"), b.table.cuda()
    q, starts = b.q.cuda(), b.starts.cuda()
    with pytest.raises(RuntimeError, match="must not share memory"):
        kv4.attention(q, b.cache, table, lens, starts, 64, out=b.cache.flatten()[:out.numel() * 2].view(torch.float16).view(4, 4, 64))
    for args in ((over[:table.numel()].view(1, -1), lens, starts), (table, over[:1], starts), (table, lens, over[:2])):
        with pytest.raises(RuntimeError, match="must not share memory"):
            kv4.attention(q, b.cache, *args, 64, out=out)
    frequencies, _ = kv4.rotary_frequencies(64)
    with pytest.raises(RuntimeError, match="must not share memory"):
        kv4.rotary(q, None, over[:4], frequencies, out=(out, None))
    with pytest.raises(RuntimeError, match="must not share memory"):
        kv4.rotary(q, q[:, :2], torch.zeros(4, dtype=torch.int64, device="cuda"), memory[256:512].view(torch.float64), out=(torch.empty_like(q), out[:, :2]))
    cache = memory[:16 * R.cell_bytes(64, 64) // 16].view(1, 1, -1)
    x = memory[64:64 + 128].view(torch.float16).view(1, 1, 64)
    with pytest.raises(RuntimeError, match="must not share memory"):
        kv4.append(cache, x, torch.zeros_like(x), torch.zeros(1, dtype=torch.int64, device="cuda"), 64)
    with pytest.raises(RuntimeError, match="must not share memory"):
        kv4.append(cache, torch.zeros_like(x), torch.zeros_like(x), over[:1], 64)
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="must not share memory"):
        kv4.plan(over[1:3], n, over.view(2, 4), n, n[:1], 16, 2)
    state = torch.zeros(1, 9, dtype=torch.int32, device="cuda")        # a row beside its table is apart from it
    assert kv4.plan(state[0, :1], n[:1], state[:, 1:], n, n[:1], 16, 1).status.item() == 0
    assert not memory.any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("window", [0, 700])
def test_many_queries_of_wide_heads_at_length(kv4, dtype, window):
    b = Batch(kv4, [1500, 900], [90, 33], 8, 1, 256, 128, dtype, 48, 2200)
    out, lse = b.run(window=window, return_lse=True)
    assert not b.dense
    b.check(out, lse, window=window)
    assert torch.equal(out, b.run(window=window))


@pytest.mark.parametrize("most,dense", [(None, True), (260, True), (1, False)])
def test_long_decoding_requests_beside_a_prompt(kv4, most, dense):
    lengths, queries = [4000, 2777, 3100, 5000], [1, 260, 1, 5]
    b = Batch(kv4, lengths, queries, 8, 2, 64, 64, torch.float16, 32, 2300)
    out, lse = b.run(return_lse=True, **({} if most is None else {"max_queries": most}))
    assert b.dense == dense
    b.check(out, lse)


# ---- together ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,d,group,interleaved", [(torch.bfloat16, 128, 128, False), (torch.float16, 64, 32, True)])
def test_steps_of_a_layer(kv4, dtype, d, group, interleaved):
    """Prompts, then decoding and drafted tokens, for requests that come to an end: plan, rotary, append and attention as a layer calls
    them, captured as one graph per step shape, against dense keys and values."""
    heads, kv_heads, page, pages = 8, 2, 16, 64
    frequencies, factor = kv4.rotary_frequencies(d, 10000.0, {"type": "linear", "factor": 2.0})
    cache = torch.full((pages, kv_heads, page // 16 * R.cell_bytes(d, group)), 255, dtype=torch.uint8, device="cuda")
    table = torch.zeros((3, 12), dtype=torch.int32, device="cuda")
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int().cuda()
    lengths, left = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.tensor([pages], dtype=torch.int32, device="cuda")
    kept_k, kept_v = [[] for _ in range(3)], [[] for _ in range(3)]
    for step, new in enumerate([[37, 1, 16], [1, 1, 1], [1, 0, 5], [30, 0, 1], [1, 1, 1]]):
        n = sum(new)
        rows = n + (step == 2) * 3                                     # padded once
        q, k, v = (normal((rows, h, d), dtype, 50 * step + i).cuda() for i, h in enumerate((heads, kv_heads, kv_heads)))
        fresh = torch.tensor(new, dtype=torch.int32, device="cuda")
        result = {}

        def layer():
            p = kv4.plan(lengths, fresh, table, free, left, page, rows)
            qr, kr = kv4.rotary(q, k, p.positions, frequencies, interleaved, factor)
            kv4.append(cache, kr, v, p.slots, group)
            result.update(p=p, k=kr, q=qr, out=kv4.attention(qr, cache, table, p.lengths, p.query_starts, group, max_queries=max(new)))

        if step % 2:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                layer()
            g.replay()
        else:
            layer()
        torch.cuda.synchronize()
        p = result["p"]
        assert p.status.item() == 0
        at = 0
        before = lengths.tolist()
        for b, m in enumerate(new):
            want_k = R.rotary(k[at:at + m].cpu(), torch.arange(before[b], before[b] + m), frequencies.cpu(), interleaved, factor)
            got_k = result["k"][at:at + m].cpu()
            assert ((got_k.double() - want_k).abs() <= R.HALF[dtype] * want_k.abs() + 1e-5).all()
            kept_k[b].append(got_k)
            kept_v[b].append(v[at:at + m].cpu())
            want, bound, _, _ = R.attention(result["q"][at:at + m].cpu(), torch.cat(kept_k[b]), torch.cat(kept_v[b]), before[b] + m, d ** -0.5, 0, group,
                                             max(new) * heads // kv_heads > 64)
            assert ((result["out"][at:at + m].cpu().double() - want).abs() <= bound).all()
            at += m
        assert (result["out"][n:] == 0).all()
        lengths, left = p.lengths.clone(), p.free_count.clone()


# ---- tiles over long contexts --------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rising", "falling", "saw"])
def test_tiles_of_values_whose_size_moves_from_step_to_step(kv4, dtype, kind):
    """More than 4096 tokens and several heads, cut over many thread blocks; the values of every 32 tokens have another power of two, so that
    exponents of an earlier step, of another head or of nothing would show.  Some values are no numbers, before the window of most rows."""
    lengths, queries = [4700, 333, 1500], [40, 1, 33]
    b = Batch(kv4, lengths, queries, 8, 4, 128, 64, dtype, 64, 2100)
    for v in b.v:
        at = torch.arange(len(v)) // 32
        last = len(v) // 32
        e = {"rising": -(last - at) // 6, "falling": -(at // 6), "saw": -(at * 5 % 11)}[kind].clamp(min=-12)
        v *= (2.0 ** e.double())[:, None, None].to(dtype)
    b.fill()
    out, lse = b.run(return_lse=True)
    assert b.dense
    b.check(out, lse)
    for _ in range(5):
        assert torch.equal(out, b.run())
    window = 2000
    b.v[0][4700 - 39 - window, 1, 7] = math.inf                        # seen by the first row alone
    b.v[0][4700 - 20 - window, 2, 70] = math.nan                       # by the first twenty
    b.fill()
    out, lse = b.run(window=window, return_lse=True)
    b.check(out, lse, window=window)
