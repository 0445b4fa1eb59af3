"""The 4-bit paged cache on a GPU: scheduling, writing, reading, attention.

Scheduling is whole numbers and reading back is one rounding: both are
compared exactly.  Attention is compared element by element with float64,
within the bound that ``kv4_reference.attention`` derives.
"""
import math
import random

import pytest
import torch

import kv4_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.half, torch.bfloat16]


@pytest.fixture(scope="module")
def m():
    import csed499ii_b200

    return csed499ii_b200


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# schedule
# ---------------------------------------------------------------------------
def schedule_case(rng, batch, page, width, most, spare, kinds):
    lens, new, at = [], [], 0
    pages = list(range(batch * width + max(spare, 0) + 7))
    rng.shuffle(pages)
    tables = [[-1] * width for _ in range(batch)]
    for b in range(batch):
        n = rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, most)])
        lens.append(min(n, most, width * page))
        new.append(rng.choice(kinds)(rng))
        for i in range(-(-lens[b] // page)):
            tables[b][i] = pages[at]
            at += 1
    free = pages[at:at + spare]
    return new, lens, tables, free + [-7] * (len(pages) - len(free)), len(free)


KINDS = {
    "step": [lambda r: 1],
    "mixed": [lambda r: 1, lambda r: 0, lambda r: -1, lambda r: r.randint(2, 90)],
    "ends": [lambda r: -1],
    "prompts": [lambda r: r.randint(1, 300)],
}


def run_schedule(m, case, rows, page, in_place=False):
    new, lens, tables, free, count = case
    t_lens, t_tables, t_free, t_count = ints(lens), ints(tables), ints(free), ints([count])
    if not tables:
        t_tables = torch.empty((0, 4), dtype=torch.int32, device=DEV)
    more = {"lens_out": t_lens, "free_count_out": t_count} if in_place else {}
    step = m.kv4_schedule(ints(new), t_lens, t_tables, t_free, t_count, rows, page, **more)
    want = R.schedule(new, lens, tables, free, count, rows, page)
    got = {"lens": step.lens, "starts": step.starts, "slots": step.slots, "positions": step.positions,
           "fate": step.fate, "free": t_free, "free_count": step.free_count, "tables": t_tables}
    for name, t in got.items():
        w = want[name] if name != "free_count" else [want[name]]
        assert t.tolist() == w, name
    return want


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("batch,page,width,spare", [
    (1, 16, 30, 100), (7, 64, 9, 40), (33, 16, 30, 11), (64, 1, 400, 3000), (300, 16, 25, 2000),
    (1300, 128, 6, 900), (70, 48, 8, 0)])
def test_schedule(m, kind, batch, page, width, spare):
    rng = random.Random(f"{kind} {batch} {page}")
    for extra in (0, 5, -1):
        case = schedule_case(rng, batch, page, width, min(300, page * width), spare, KINDS[kind])
        rows = max(0, sum(max(0, x) for x in case[0]) + extra)
        run_schedule(m, case, rows, page)
        run_schedule(m, case, rows, page, in_place=True)


def test_schedule_empty_and_largest(m):
    run_schedule(m, ([], [], [], [3, 1], 2), 5, 16)
    run_schedule(m, ([], [], [], [3, 1], 2), 0, 16)
    batch = 8192
    tables = [[b] for b in range(batch)]
    case = ([(-1, 1, 20)[b % 3] for b in range(batch)], [b % 16 + 1 for b in range(batch)], tables,
            [-1] * batch, 0)
    run_schedule(m, case, 9 * batch, 16)


def test_schedule_serves_a_run_of_steps(m):
    """No page is ever held twice or lost over many steps in place."""
    rng = random.Random(3)
    batch, page, width, pages = 40, 16, 12, 200
    lens, count = ints([0] * batch), ints([pages])
    tables = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
    free = ints(rng.sample(range(pages), pages))
    for _ in range(60):
        new = [rng.choice([1, 1, 1, 0, -1, rng.randint(1, 60)]) for _ in range(batch)]
        m.kv4_schedule(ints(new), lens, tables, free, count, 900, page, lens_out=lens, free_count_out=count)
        held = [p for n, t in zip(lens.tolist(), tables.tolist()) for p in t[:-(-n // page)]]
        assert sorted(held + free.tolist()[:count.item()]) == list(range(pages))


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
def rows_of(tokens, heads, dim, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(tokens, heads, dim, generator=g, device=DEV) * 1.3
    return (x + 2 * torch.randn(1, heads, dim, generator=g, device=DEV)).to(dtype)


def some_slots(tokens, total, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(total, generator=g)[:tokens].int().to(DEV)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("tokens,heads,page", [(1, 1, 16), (3, 2, 16), (17, 5, 48), (130, 8, 64), (700, 3, 128)])
def test_append_then_read(m, dtype, dim, tokens, heads, page):
    pages = -(-tokens // page) + 2
    cache = m.kv4_cache(pages, heads, dim, page, dtype, DEV)
    k, v = rows_of(tokens, heads, dim, dtype, 1), rows_of(tokens, heads, dim, dtype, 2)
    slots = some_slots(tokens, pages * page, 3)
    m.kv4_append(k, v, cache, slots)
    k2, v2 = m.kv4_read(cache, slots)
    assert torch.equal(k2, R.values(k).float().to(dtype)) and torch.equal(v2, R.values(v).float().to(dtype))


@pytest.mark.parametrize("dim", [64, 128])
def test_the_tiles_are_as_documented(m, dim):
    heads, page, tokens = 2, 32, 40
    cache = m.kv4_cache(3, heads, dim, page, torch.half, DEV)
    k, v = rows_of(tokens, heads, dim, torch.half, 5), rows_of(tokens, heads, dim, torch.half, 6)
    slots = some_slots(tokens, 3 * page, 7)
    m.kv4_append(k, v, cache, slots)
    raw = cache.view(torch.uint8).reshape(3, heads, page // 16, 16 * dim + 128).cpu()
    for which, x in ((0, k), (1, v)):
        codes, scale, low = (t.cpu() for t in R.quantise(x))
        for i, slot in enumerate(slots.tolist()):
            tok = slot % page % 16
            for h in range(heads):
                tile = raw[slot // page, h, slot % page // 16]
                if which == 0:
                    row = tile[tok * dim // 2:(tok + 1) * dim // 2]
                else:
                    part = tile[8 * dim:16 * dim].reshape(2, 8, 8, dim // 16)
                    row = part[tok // 8, :, tok % 8].reshape(-1)
                got = torch.stack([row & 15, row >> 4], -1).reshape(-1)
                assert torch.equal(got.double(), codes[i, h])
                pair = tile[16 * dim + 64 * which + 4 * tok:][:4].clone().view(torch.half).double()
                assert pair.tolist() == [scale[i, h].item(), low[i, h].item()]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["fused", "heads first", "odd offset", "broadcast"])
def test_append_takes_any_stride(m, dtype, layout):
    tokens, heads, dim, page = 37, 3, 128, 16
    if layout == "fused":
        both = rows_of(tokens, 4 + 2 * heads, dim, dtype, 1)
        k, v = both[:, 4:4 + heads], both[:, 4 + heads:]
    elif layout == "heads first":
        k = rows_of(heads, tokens, dim, dtype, 1).transpose(0, 1)
        v = rows_of(heads, tokens, dim, dtype, 2).transpose(0, 1)
    elif layout == "odd offset":
        flat = rows_of(1, 2, tokens * heads * dim + 8, dtype, 1)
        k = flat[0, 0, 1:1 + tokens * heads * dim].view(tokens, heads, dim)
        v = flat[0, 1, 3:3 + tokens * heads * dim].view(tokens, heads, dim)
    else:
        k = rows_of(tokens, 1, dim, dtype, 1).expand(tokens, heads, dim)
        v = rows_of(1, heads, dim, dtype, 2).expand(tokens, heads, dim)
    cache = m.kv4_cache(4, heads, dim, page, dtype, DEV)
    slots = some_slots(tokens, 4 * page, 4)
    m.kv4_append(k, v, cache, slots)
    k2, v2 = m.kv4_read(cache, slots)
    assert torch.equal(k2, R.values(k).float().to(dtype)) and torch.equal(v2, R.values(v).float().to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_are_hard_to_quantise(m, dtype, dim):
    top, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x = torch.zeros(14, 1, dim, dtype=dtype, device=DEV)
    x[1] = 7.5                                   # flat
    x[2, 0, 5] = tiny                            # a range whose scale is subnormal
    x[3, 0, 5] = tiny * 2**-7                    # ... or nothing at all
    x[4, 0, :2] = torch.tensor([top, -top], dtype=dtype)
    x[5, 0, 3] = top
    x[6] = -top
    x[7, 0, 9] = math.inf
    x[8, 0, dim - 1] = -math.inf
    x[9, 0, 11] = math.nan
    x[10] = math.nan
    x[11, 0, 1::2] = -0.0
    x[12] = torch.arange(dim, device=DEV).to(dtype)          # quotients that sit on ties
    x[13] = (torch.arange(dim, device=DEV) * 0.5 - 4).to(dtype)
    cache = m.kv4_cache(1, 1, dim, 16, dtype, DEV)
    slots = ints(list(range(14)))
    m.kv4_append(x, x.flip(0), cache, slots)
    k, v = m.kv4_read(cache, slots)
    assert same(k, R.values(x).float().to(dtype)) and same(v, R.values(x.flip(0)).float().to(dtype))


def test_append_touches_its_slots_alone(m):
    pages, heads, dim, page = 5, 3, 128, 32
    cache = m.kv4_cache(pages, heads, dim, page, torch.half, DEV)
    everything = ints(list(range(pages * page)))
    old_k, old_v = rows_of(pages * page, heads, dim, torch.half, 1), rows_of(pages * page, heads, dim, torch.half, 2)
    m.kv4_append(old_k, old_v, cache, everything)
    before = m.kv4_read(cache, everything)
    slots = ints([40, -1, 7, pages * page, 159, -2**31, 2**31 - 1])
    k, v = rows_of(7, heads, dim, torch.half, 3), rows_of(7, heads, dim, torch.half, 4)
    m.kv4_append(k, v, cache, slots)
    after = m.kv4_read(cache, everything)
    there = torch.tensor([40, 7, 159], device=DEV)
    for b, a, x in zip(before, after, (k, v)):
        b[there] = R.values(x[[0, 2, 4]]).half()
        assert torch.equal(a, b)
    for x in m.kv4_read(cache, slots):
        assert not x[[1, 3, 5, 6]].any()


def test_empty_calls(m):
    cache = m.kv4_cache(2, 2, 64, 16, torch.half, DEV)
    none = torch.empty(0, 2, 64, dtype=torch.half, device=DEV)
    m.kv4_append(none, none, cache, ints([]))
    assert m.kv4_read(cache, ints([]))[0].shape == (0, 2, 64)
    tables = torch.zeros(0, 1, dtype=torch.int32, device=DEV)
    assert m.kv4_attention(none, cache, tables, ints([])).shape == (0, 2, 64)
    # rows without a request, requests without a table
    q = torch.ones(3, 4, 64, dtype=torch.half, device=DEV)
    assert not m.kv4_attention(q, cache, tables, ints([]), starts=ints([0])).any()
    wide = torch.zeros(3, 0, dtype=torch.int32, device=DEV)
    assert not m.kv4_attention(q, cache, wide, ints([5, 1, 0])).any()
    empty = m.kv4_cache(0, 2, 64, 16, torch.half, DEV)
    assert not m.kv4_attention(q, empty, wide + 0, ints([5, 1, 0])).any()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
class Problem:
    """Requests in a cache whose unused slots hold NaN, on pages in random order."""

    def __init__(self, m, lens, new, heads, group, dim, page, dtype, seed=0, sharp=1.0, pad=0):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.lens, self.new, self.page = lens, new, page
        used = [-(-n // page) for n in lens]
        order = torch.randperm(sum(used) + 2, generator=torch.Generator().manual_seed(seed)).int()
        self.cache = m.kv4_cache(sum(used) + 2, heads, dim, page, dtype, DEV)
        self.cache.view(torch.int16).fill_(-1)
        width = max(used, default=0) + 1
        tables, slots, at = torch.full((len(lens), width), -1, dtype=torch.int32), [], 0
        for b, u in enumerate(used):
            tables[b, :u] = order[at:at + u]
            slots.append((order[at:at + u, None] * page + torch.arange(page)).reshape(-1)[:lens[b]])
            at += u
        self.tables = tables.to(DEV)
        self.slots = torch.cat(slots).int().to(DEV)
        total = sum(lens)
        self.k = (torch.randn(total, heads, dim, generator=g, device=DEV)
                  + torch.randn(1, heads, dim, generator=g, device=DEV)).to(dtype)
        self.v = torch.randn(total, heads, dim, generator=g, device=DEV).to(dtype)
        m.kv4_append(self.k, self.v, self.cache, self.slots)
        self.starts = [sum(new[:i]) for i in range(len(new) + 1)]
        self.q = (sharp * torch.randn(self.starts[-1] + pad, heads * group, dim, generator=g, device=DEV)).to(dtype)

    def check(self, out, window=0, scale=None):
        assert out.shape == self.q.shape and out.dtype is self.q.dtype
        at = 0
        for b, n in enumerate(self.lens):
            rows = slice(self.starts[b], self.starts[b + 1])
            want, bound = R.attention(self.q[rows], self.k[at:at + n], self.v[at:at + n], self.new[b],
                                      window, scale)
            got = out[rows].double()
            assert torch.isfinite(got).all(), f"request {b}"
            worst = ((got - want).abs() / (bound + 2.0**-24)).max().item() if got.numel() else 0.0
            assert worst <= 1, f"request {b} of {n}: {worst} bounds off"
            at += n
        assert not out[self.starts[-1]:].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 4), (3, 7), (2, 8), (1, 16), (1, 23)])
def test_single_tokens(m, dtype, dim, heads, group):
    lens = [1, 0, 2, 15, 16, 17, 63, 64, 65, 300, 777]
    p = Problem(m, lens, [1] * len(lens), heads, group, dim, 64, dtype, seed=heads + group)
    p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens)))


@pytest.mark.parametrize("page", [16, 32, 48, 128])
@pytest.mark.parametrize("window", [0, 1, 16, 100])
def test_pages_and_windows(m, page, window):
    lens = [5, 130, 1, 257, 0, 96, 95]
    p = Problem(m, lens, [1] * len(lens), 2, 4, 128, page, torch.half, seed=page)
    p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens), window=window), window)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,group,new", [
    (2, 1, [2, 1, 0, 3, 2]), (2, 4, [4, 4, 4, 4, 4]), (1, 8, [5, 1, 0, 4, 2]), (1, 3, [40, 1, 0, 33, 90]),
    (2, 2, [1, 130, 0, 64, 300]), (5, 1, [129, 7, 0, 128, 257])])
def test_a_few_tokens_and_pieces_of_prompts(m, dtype, dim, heads, group, new):
    lens = [131, 200, 0, 128, 300]
    p = Problem(m, lens, new, heads, group, dim, 32, dtype, seed=sum(new), pad=3)
    for most in (max(new), None, 10**6):
        out = m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=most)
        p.check(out)


@pytest.mark.parametrize("window", [1, 17, 64, 200])
@pytest.mark.parametrize("dtype", TYPES)
def test_prompts_with_a_window(m, window, dtype):
    lens, new = [500, 37, 260, 1], [500, 37, 131, 1]
    p = Problem(m, lens, new, 2, 3, 64, 16, dtype, seed=window)
    p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=500,
                            window=window), window)


@pytest.mark.parametrize("dim,heads,group", [(128, 8, 4), (64, 3, 5)])
def test_whole_prompts(m, dim, heads, group):
    lens = [1, 127, 128, 129, 1000]
    p = Problem(m, lens, lens, heads, group, dim, 64, torch.half, seed=9)
    p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=1000))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,new,heads,group,window", [
    ([20000], [9], 1, 8, 0), ([5000, 0, 3, 9000], [100, 0, 3, 40], 2, 4, 0),
    ([5000, 1200, 3, 9000], [100, 300, 3, 40], 2, 4, 2500), ([7001, 6000], [1, 130], 3, 5, 1000)])
def test_few_rows_of_many_keys(m, dtype, dim, lens, new, heads, group, window):
    p = Problem(m, lens, new, heads, group, dim, 32, dtype, seed=sum(new), pad=2)
    for most in (max(new), None):
        out = m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=most,
                              window=window)
        p.check(out, window)


@pytest.mark.parametrize("lens", [[20000], [1, 30000, 5], [4097] * 3, [100] * 200])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 8)])
def test_work_of_uneven_lengths(m, lens, heads, group):
    p = Problem(m, lens, [1] * len(lens), heads, group, 128, 64, torch.half, seed=len(lens))
    p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens)))


@pytest.mark.parametrize("sharp", [0.0, 8.0, 40.0])
def test_flat_and_sharp_weights(m, sharp):
    lens, new = [1500, 700], [1, 300]
    p = Problem(m, lens, new, 2, 4, 128, 64, torch.half, seed=11, sharp=sharp)
    p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=300))


@pytest.mark.parametrize("scale", [0.01, 1.0, -0.2])
def test_scale(m, scale):
    lens, new = [333, 200], [1, 200]
    p = Problem(m, lens, new, 2, 4, 64, 64, torch.half, seed=12)
    p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=200, scale=scale),
            scale=scale)


def test_values_of_any_size(m):
    """Values far from one, and rows of very different scales in one request."""
    lens, new = [400, 150], [1, 150]
    for size in (1e-4, 3000.0):
        p = Problem(m, lens, new, 2, 2, 128, 64, torch.half, seed=13)
        p.v = (p.v.float() * size).half()
        m.kv4_append(p.k, p.v, p.cache, p.slots)
        p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=150))
    p.v = (p.v.float() * 10.0 ** torch.randint(-6, 1, (550, 2, 1), device=DEV)).half()
    m.kv4_append(p.k, p.v, p.cache, p.slots)
    p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=150))


def test_a_bad_row_stays_where_it_is_seen(m):
    """An infinity in a key or value spoils the rows that see it and no other."""
    lens, new = [200, 200], [1, 200]
    p = Problem(m, lens, new, 1, 2, 128, 64, torch.half, seed=14)
    k = p.k.clone()
    k[200 + 90, 0, 7] = math.inf  # token 90 of the second request
    m.kv4_append(k, p.v, p.cache, p.slots)
    out = m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=200)
    assert torch.isfinite(out[:1 + 90]).all() and torch.isnan(out[1 + 90:]).all()
    out = m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=200, window=50)
    assert torch.isfinite(out[:91]).all() and torch.isnan(out[91:91 + 50]).all()
    assert torch.isfinite(out[91 + 50:]).all()


def test_keys_on_pages_outside_the_cache_are_unseen(m):
    lens, new = [150, 150], [1, 150]
    p = Problem(m, lens, new, 2, 2, 128, 32, torch.half, seed=15)
    for bad in (-1, p.cache.size(0), 2**31 - 1, -2**31):
        tables = p.tables.clone()
        tables[:, 1] = bad  # tokens 32..63
        out = m.kv4_attention(p.q, p.cache, tables, ints(lens), starts=ints(p.starts), max_new=150)
        assert torch.isfinite(out).all()
        keep = [j for j in range(150) if not 32 <= j < 64]
        want, bound = R.attention(p.q[:1], p.k[keep], p.v[keep], 1)
        assert ((out[:1].double() - want).abs() <= bound + 2.0**-24).all()
        tables[:] = bad
        assert not m.kv4_attention(p.q, p.cache, tables, ints(lens), starts=ints(p.starts), max_new=150).any()


def test_lengths_past_the_table(m):
    """A length that the table cannot hold counts as what it holds."""
    p = Problem(m, [64, 64], [1, 1], 1, 4, 64, 16, torch.half, seed=16)
    tables = p.tables[:, :4].contiguous()
    out = m.kv4_attention(p.q, p.cache, tables, ints([64, 2**31 - 1]))
    assert torch.equal(out, m.kv4_attention(p.q, p.cache, tables, ints([64, 64])))
    assert not m.kv4_attention(p.q, p.cache, tables, ints([0, -5])).any()


@pytest.mark.parametrize("layout", ["fused", "heads first", "odd offset", "table rows"])
def test_attention_takes_any_stride(m, layout):
    lens, new = [70, 300], [1, 140]
    p = Problem(m, lens, new, 2, 4, 128, 16, torch.half, seed=17)
    want = m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=140)
    p.check(want)
    q, tables = p.q, p.tables
    if layout == "fused":
        q = torch.cat([q, q[:, :4]], 1)[:, :8]
    elif layout == "heads first":
        q = q.transpose(0, 1).contiguous().transpose(0, 1)
    elif layout == "odd offset":
        flat = torch.zeros(q.numel() + 8, dtype=q.dtype, device=DEV)
        flat[3:3 + q.numel()] = q.reshape(-1)
        q = flat[3:3 + q.numel()].view(p.q.shape)
    else:
        tables = torch.cat([tables, tables + 1], 1)[:, :tables.size(1)]
    out = torch.full_like(p.q, math.nan)
    got = m.kv4_attention(q, p.cache, tables, ints(lens), starts=ints(p.starts), max_new=140, out=out)
    assert got is out and torch.equal(out, want)


def test_results_do_not_change_from_call_to_call(m):
    lens, new = [5000, 17, 900, 3], [1, 1, 260, 3]
    p = Problem(m, lens, new, 2, 4, 128, 64, torch.bfloat16, seed=18)
    args = (p.q, p.cache, p.tables, ints(lens))
    first = m.kv4_attention(*args, starts=ints(p.starts), max_new=260)
    p.check(first)
    for _ in range(20):
        assert torch.equal(first, m.kv4_attention(*args, starts=ints(p.starts), max_new=260))


@pytest.mark.parametrize("lens,heads,group", [([9000, 40], 2, 8), ([9000, 8000, 7000], 3, 3), ([30000] * 5, 1, 1)])
def test_results_do_not_depend_on_timing(m, lens, heads, group):
    """Joins over CTAs while calls on other streams come between."""
    p = Problem(m, lens, [1] * len(lens), heads, group, 128, 64, torch.half, seed=20)
    args = (p.q, p.cache, p.tables, ints(lens))
    want = m.kv4_attention(*args)
    p.check(want)
    torch.cuda.synchronize()
    for _ in range(5):
        outs = []
        for s in [torch.cuda.Stream(DEV) for _ in range(3)]:
            with torch.cuda.stream(s):
                outs += [m.kv4_attention(*args) for _ in range(10)]
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_streams_and_workspaces(m):
    p = Problem(m, [9000, 40], [1, 1], 2, 8, 128, 64, torch.half, seed=19)
    lens = ints(p.lens)
    want = m.kv4_attention(p.q, p.cache, p.tables, lens)
    p.check(want)
    streams = [torch.cuda.Stream(DEV) for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for s in streams:
        with torch.cuda.stream(s):
            outs += [m.kv4_attention(p.q, p.cache, p.tables, lens) for _ in range(10)]
    space = m.kv4_workspace(DEV)
    outs.append(m.kv4_attention(p.q, p.cache, p.tables, lens, workspace=space))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    small = torch.zeros(1, dtype=torch.int32, device=DEV)
    if 4 < m._ext.load().sm100_marlin_kv4_workspace_bytes(0):
        with pytest.raises(RuntimeError, match="workspace"):
            m.kv4_attention(p.q, p.cache, p.tables, lens, workspace=small)


def test_a_step_in_a_graph(m):
    """Scheduling, writing and attention replayed from a graph, in place."""
    heads, group, dim, page, batch = 2, 4, 128, 16, 3
    cache = m.kv4_cache(40, heads, dim, page, torch.half, DEV)
    lens, count, free = ints([0] * batch), ints([40]), ints(list(range(40)))
    tables = torch.full((batch, 8), -1, dtype=torch.int32, device=DEV)
    new = ints([1] * batch)
    q = torch.zeros(batch, heads * group, dim, dtype=torch.half, device=DEV)
    k, v = (torch.zeros(batch, heads, dim, dtype=torch.half, device=DEV) for _ in range(2))

    def step():
        s = m.kv4_schedule(new, lens, tables, free, count, batch, page, lens_out=lens, free_count_out=count)
        m.kv4_append(k, v, cache, s.slots)
        return m.kv4_attention(q, cache, tables, s.lens)

    step()
    torch.cuda.synchronize()
    lens.zero_(), count.fill_(40), tables.fill_(-1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    seen = []
    for i in range(50):
        for x, seed in ((q, 3 * i), (k, 3 * i + 1), (v, 3 * i + 2)):
            x.copy_(rows_of(*x.shape, torch.half, seed))
        seen.append((k.clone(), v.clone()))
        graph.replay()
        if i % 7 == 0 or i == 49:
            for b in range(batch):
                want, bound = R.attention(q[b:b + 1], torch.stack([x[0][b] for x in seen]),
                                          torch.stack([x[1][b] for x in seen]), 1)
                assert ((out[b:b + 1].double() - want).abs() <= bound + 2.0**-24).all()
    assert lens.tolist() == [50] * batch and count.item() == 40 - batch * 4


def test_a_layer_that_serves(m):
    """The demo's layer: prompts, single tokens, a request that ends and one that takes its place,
    against plain attention over what its cache holds."""
    from csed499ii_b200.kv4_demo import CachedAttention

    heads, kv, dim, hidden = 8, 2, 64, 512
    layer = CachedAttention(hidden, heads, kv, dim, batch=3, pages=12, page_size=32, most=160, seed=5)
    g = torch.Generator(device=DEV).manual_seed(6)
    held = [[], [], []]  # (k, v) of each token, as the projection gives them
    for new in ([70, 0, 33], [1, 5, 1], [1, 1, -1], [1, 1, 40], [1, 1, 1]):
        rows = sum(max(n, 0) for n in new)
        x = torch.randn(rows, hidden, generator=g, device=DEV).half()
        y, step = layer.step(x, ints(new), max(new))
        assert step.fate.tolist() == [0, 0, 0]
        q, k, v = layer.qkv(x).view(rows, -1, dim).split([heads, kv, kv], 1)
        out = torch.zeros(rows, heads, dim, dtype=torch.double, device=DEV)
        slack, at = torch.zeros_like(out), 0
        for b, n in enumerate(new):
            if n < 0:
                held[b] = []
                continue
            held[b] += [(k[i], v[i]) for i in range(at, at + n)]
            if n:
                ks, vs = (torch.stack([t[j] for t in held[b]]) for j in (0, 1))
                out[at:at + n], slack[at:at + n] = R.attention(q[at:at + n], ks, vs, n)
            at += n
        assert step.lens.tolist() == [len(h) for h in held]
        got = m.kv4_attention(q, layer.cache, layer.tables, step.lens, starts=step.starts, max_new=max(new))
        assert ((got.double() - out).abs() <= slack + 2.0**-24).all()
        assert torch.equal(y, layer.proj(got.flatten(1)))
    assert layer.count.item() == 12 - sum(-(-len(h) // 32) for h in held)


def test_offsets_past_32_bits(m):
    """A cache of more than 4 GB, its pages used at both ends."""
    heads, dim, page = 8, 128, 64
    pages = (5 << 30) // (heads * page // 16 * 2176)
    cache = m.kv4_cache(pages, heads, dim, page, torch.half, DEV)
    p = Problem(m, [500, 700], [1, 200], heads, 2, dim, page, torch.half, seed=20)
    tables = torch.where(p.tables >= 0, pages - 1 - p.tables, p.tables)
    slots = (pages - 1 - p.slots // page) * page + p.slots % page
    m.kv4_append(p.k, p.v, cache, slots)
    k, _ = m.kv4_read(cache, slots)
    assert torch.equal(k, R.values(p.k).half())
    p.check(m.kv4_attention(p.q, cache, tables, ints(p.lens), starts=ints(p.starts), max_new=200))


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals(m):
    cache = m.kv4_cache(4, 2, 64, 16, torch.half, DEV)
    x = torch.zeros(3, 2, 64, dtype=torch.half, device=DEV)
    q = torch.zeros(3, 4, 64, dtype=torch.half, device=DEV)
    tables = torch.zeros(3, 2, dtype=torch.int32, device=DEV)
    one, slots = ints([1] * 3), ints([0, 1, 2])
    bad = RuntimeError
    for call in (
        lambda: m.kv4_append(x.bfloat16(), x, cache, slots),
        lambda: m.kv4_append(x, x[:, :1], cache, slots),
        lambda: m.kv4_append(x, x[:2], cache, slots),
        lambda: m.kv4_append(x, x, cache, slots[:2]),
        lambda: m.kv4_append(x, x, cache, slots.long()),
        lambda: m.kv4_append(x.cpu(), x, cache, slots),
        lambda: m.kv4_append(x.transpose(1, 2).contiguous().transpose(1, 2), x, cache, slots),
        lambda: m.kv4_append(x, x, cache[:, :, :, :64], slots),
        lambda: m.kv4_append(x, x, cache.float(), slots),
        lambda: m.kv4_append(x, x, cache.cpu(), slots),
        lambda: m.kv4_append(x, x, cache[:, :1], slots),
        lambda: m.kv4_read(cache, slots.cpu()),
        lambda: m.kv4_read(cache, slots.float()),
        lambda: m.kv4_attention(q[:, :3], cache, tables, one),
        lambda: m.kv4_attention(q[:, :0], cache, tables, one),
        lambda: m.kv4_attention(q[:2], cache, tables, one),
        lambda: m.kv4_attention(q, cache, tables[:2], one),
        lambda: m.kv4_attention(q, cache, tables.long(), one),
        lambda: m.kv4_attention(q, cache, tables.t().contiguous().t(), one),
        lambda: m.kv4_attention(q, cache, tables, one.long()),
        lambda: m.kv4_attention(q, cache, tables, one, starts=ints([0, 3])),
        lambda: m.kv4_attention(q, cache, tables, one, out=q[:2]),
        lambda: m.kv4_attention(q, cache, tables, one, out=q.float()),
        lambda: m.kv4_attention(q.bfloat16(), cache, tables, one),
        lambda: m.kv4_attention(q[..., :32], cache, tables, one),
        lambda: m.kv4_schedule(one.cpu(), one, tables, slots, one[:1], 3, 16),
        lambda: m.kv4_schedule(one, one[:2], tables, slots, one[:1], 3, 16),
        lambda: m.kv4_schedule(one, one, tables[:2], slots, one[:1], 3, 16),
        lambda: m.kv4_schedule(one, one, tables, slots.long(), one[:1], 3, 16),
        lambda: m.kv4_schedule(one, one, tables, slots, one, 3, 16),
        lambda: m.kv4_schedule(one, one, tables, slots, one[:1], -1, 16),
        lambda: m.kv4_schedule(one, one, tables, slots, one[:1], 3, 0),
        lambda: m.kv4_schedule(one, one, tables, slots, one[:1], 3, 16, lens_out=one[:2]),
        lambda: m.kv4_schedule(ints([0] * 8193), ints([0] * 8193), tables.new_zeros(8193, 1), slots, one[:1], 3, 16),
    ):
        with pytest.raises(bad):
            call()
    for call in (
        lambda: m.kv4_cache(4, 2, 96, 16),
        lambda: m.kv4_cache(4, 2, 64, 24),
        lambda: m.kv4_cache(4, 2, 64, 16, torch.float),
        lambda: m.kv4_cache(2**27, 2, 64, 16),
        lambda: m.kv4_attention(q, cache, tables, one, window=-1),
        lambda: m.kv4_attention(q, cache, tables, one, starts=ints([0, 1, 2, 3]), max_new=-1),
    ):
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()


def test_weights_written_before_a_cache_call(m):
    """A GEMM prefetches its weights while the call before it ends: not while the copy before that runs."""
    k, n = 4096, 22016
    g = torch.Generator(device=DEV).manual_seed(21)
    layer = m.Layer_2_4(k, n, groupsize=128).to(DEV)
    sets = []
    for _ in range(2):
        w = torch.randn(k, n, generator=g, device=DEV).half() * 0.02
        layer.pack(type("W", (), {"weight": w, "bias": None})(), (w.view(k // 128, 128, n).abs().amax(1) / 7).half())
        sets.append([t.clone() for t in (layer.B, layer.meta, layer.s)])
    x = torch.randn(16, k, generator=g, device=DEV).half()
    want = []
    for s in sets:
        for t, u in zip((layer.B, layer.meta, layer.s), s):
            t.copy_(u)
        torch.cuda.synchronize()
        want.append(layer(x))
    cache = m.kv4_cache(4, 2, 64, 16, torch.half, DEV)
    rows = torch.randn(3, 2, 64, generator=g, device=DEV).half()
    q, tables, lens = rows.repeat(1, 2, 1), ints([[0], [1], [2]]), ints([3, 2, 1])
    calls = [lambda: m.kv4_append(rows, rows, cache, ints_of_three),
             lambda: m.kv4_read(cache, ints_of_three),
             lambda: m.kv4_attention(q, cache, tables, lens),
             lambda: m.kv4_schedule(lens, lens, tables, lens, ints_of_three[:1], 6, 16)]
    ints_of_three = ints([0, 1, 2])
    for i in range(40):
        torch.cuda.synchronize()
        for t, u in zip((layer.s, layer.meta, layer.B), reversed(sets[i % 2])):
            t.copy_(u)
        calls[i // 2 % 4]()
        assert torch.equal(layer(x), want[i % 2]), i
