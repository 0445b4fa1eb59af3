"""The 4-bit cache at the edges of what it accepts, on a GPU.

Tolerances are those that ``kv4_reference.attention`` derives; where values are
scaled by a power of two, which is exact in every step of the format, results
are scaled back and held to the bound of the values before.
"""
import random

import pytest
import torch

import kv4_reference as R
from test_kv4_gpu import DEV, KINDS, TYPES, Problem, ints, m, schedule_case  # noqa: F401  (m is the fixture)

pytestmark = pytest.mark.gpu


def attend(m, p, lens, new, **kw):  # noqa: F811
    return m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=max(new), **kw)


# ---------------------------------------------------------------------------
# sizes of values
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("power", [-85, -70, -50, 0, 50, 70, 120])
def test_values_of_any_exponent(m, dim, power):  # noqa: F811
    """The same values times a power of two: the same results times it."""
    lens, new = [400, 150], [1, 150]
    p = Problem(m, lens, new, 2, 2, dim, 64, torch.bfloat16, seed=31)
    m.kv4_append(p.k, p.v * 2.0**power, p.cache, p.slots)
    # of the result; the check is of the unscaled values
    p.check((attend(m, p, lens, new).double() * 2.0**-power).to(torch.bfloat16))


@pytest.mark.parametrize("scale", [0.0, 1e-30, -1e-9])
def test_scales_next_to_zero(m, scale):  # noqa: F811
    lens, new = [333, 200], [1, 200]
    for dtype in TYPES:
        p = Problem(m, lens, new, 2, 4, 64, 64, dtype, seed=49)
        p.check(attend(m, p, lens, new, scale=scale), scale=scale)


@pytest.mark.parametrize("power", [-130, -115, -100])
def test_smallest_values(m, power):  # noqa: F811
    """A scale below 2^-90 counts as 2^-90: codes up to 15 of it."""
    lens, new = [300, 130], [1, 130]
    p = Problem(m, lens, new, 1, 2, 64, 64, torch.bfloat16, seed=32)
    v = p.v * 2.0**power
    m.kv4_append(p.k, v, p.cache, p.slots)
    out = attend(m, p, lens, new).double()
    at = 0
    for b, n in enumerate(lens):
        rows = slice(p.starts[b], p.starts[b + 1])
        want, _ = R.attention(p.q[rows], p.k[at:at + n], v[at:at + n], new[b])
        assert ((out[rows] - want).abs() <= 16 * 2.0**-90).all()
        at += n


@pytest.mark.parametrize("power", [-40, 0, 40])
def test_rows_of_zeros_between_values_of_any_exponent(m, power):  # noqa: F811
    """A row of zeros has no scale; what stands in for it must not outweigh the others'."""
    lens, new = [400, 150], [1, 150]
    p = Problem(m, lens, new, 2, 2, 128, 64, torch.bfloat16, seed=33)
    p.v[::3] = 0
    m.kv4_append(p.k, p.v * 2.0**power, p.cache, p.slots)
    p.check((attend(m, p, lens, new).double() * 2.0**-power).to(torch.bfloat16))


# ---------------------------------------------------------------------------
# weights of very different sizes
# ---------------------------------------------------------------------------
def attend_many(m, p, n, new, copies):  # noqa: F811
    """Attention of one request, and of many at once that share its pages: enough
    of them that a warp or a CTA goes over all keys of a request by itself."""
    out = attend(m, p, [n], [new])
    many = m.kv4_attention(p.q.repeat(copies, 1, 1), p.cache, p.tables.repeat(copies, 1), ints([n] * copies),
                           starts=ints([new * i for i in range(copies + 1)]), max_new=new)
    return [out, many[:new], many[-new:], many[copies // 2 * new:][:new]]


@pytest.mark.parametrize("new,copies", [(1, 2600), (100, 80)])
@pytest.mark.parametrize("dim", [64, 128])
def test_one_wide_row_among_narrow_ones(m, dim, new, copies):  # noqa: F811
    """Values next to 1 whose scales are 2^-14, one row whose scale is 64, equal weights."""
    n = 20000
    p = Problem(m, [n], [new], 1, 2, dim, 64, torch.half, seed=36, sharp=0.0)
    g = torch.Generator(device=DEV).manual_seed(37)
    p.v = (1 + 2.0**-10 * torch.randint(0, 4, p.v.shape, generator=g, device=DEV)).half()
    p.v[77] = (960 * torch.rand(p.v[77].shape, generator=g, device=DEV) - 480).half()
    m.kv4_append(p.k, p.v, p.cache, p.slots)
    for out in attend_many(m, p, n, new, copies):
        p.check(out)


@pytest.mark.parametrize("n,new,copies", [(32768, 1, 2600), (131072, 1, 2600), (32768, 100, 80), (131072, 100, 80)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("power", [18, 19, 20, 21, 22, 24, 26, 31])
def test_one_strong_key_before_many_weak_ones(m, dtype, n, power, new, copies):  # noqa: F811
    """Keys that weigh 2^-power of the first each have their part in the result too."""
    p = Problem(m, [n], [new], 1, 2, 128, 64, dtype, seed=34)
    g = torch.Generator(device=DEV).manual_seed(35)
    signs = torch.where(torch.rand(128, generator=g, device=DEV) < 0.5, -1.0, 1.0)
    p.q = signs.expand(p.q.shape).contiguous().to(dtype)
    p.k = torch.zeros_like(p.k)
    p.k[0, 0] = (signs * (power * 0.6931 / 128**0.5)).to(dtype)
    p.v[1:] = p.v[1]
    m.kv4_append(p.k, p.v, p.cache, p.slots)
    for out in attend_many(m, p, n, new, copies):
        p.check(out)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group,new", [(1, 1), (8, 1), (8, 3)])
def test_fp16_results_of_few_rows_are_rounded_once(m, dim, group, new):  # noqa: F811
    """Many keys of like weights, where each weight's rounding shows.  All but the result
    is held to 2^-14 of it or better, so the error is next to that of one rounding."""
    n = 60000
    p = Problem(m, [n], [new], 2, group, dim, 64, torch.half, seed=39, sharp=0.5)
    want, _ = R.attention(p.q, p.k, p.v, new)
    once = (want.half().double() - want).norm()
    assert (attend(m, p, [n], [new]).double() - want).norm() <= 1.15 * once


@pytest.mark.parametrize("skewed", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,new,copies,most", [
    (20000, 1, 2600, 1.15), (20000, 100, 80, 1.55), (4000, 300, 80, 1.55), (60000, 100, 1, 1.55)])
def test_fp16_results_of_values_around_zero(m, dim, n, new, copies, most, skewed):  # noqa: F811
    """Keys of like weight, so that values average out and what sums lose shows.

    Few rows have the error of one rounding.  In the prompt kernel each weight is rounded as
    the result is, which adds as much again: the root of two, and a little for all else."""
    p = Problem(m, [n], [new], 1, 4, dim, 64, torch.half, seed=46, sharp=0.3)
    if skewed:  # exponential less the mean: a row's zero is near its lowest codes
        g = torch.Generator(device=DEV).manual_seed(47)
        p.v = (-torch.log(torch.rand(p.v.shape, generator=g, device=DEV).clamp(min=1e-6)) - 1).half()
        m.kv4_append(p.k, p.v, p.cache, p.slots)
    want, _ = R.attention(p.q, p.k, p.v, new)
    once = (want.half().double() - want).norm()
    for out in attend_many(m, p, n, new, copies):
        assert (out.double() - want).norm() <= most * once


@pytest.mark.parametrize("dim", [64, 128])
def test_keys_next_to_zero(m, dim):  # noqa: F811
    """Keys whose scale is a subnormal of the type, or of 32 bits: they weigh as zeros do."""
    lens, new = [200, 150], [1, 150]
    p = Problem(m, lens, new, 2, 2, dim, 64, torch.bfloat16, seed=38)
    tiny = torch.tensor([0.0, 2.0**-133, 2.0**-129, 2.0**-126, 2.0**-120, 2.0**-60], device=DEV)
    p.k[::4] = (torch.rand(p.k[::4].shape, device=DEV) * tiny[torch.arange(88, device=DEV) % 6, None, None]).bfloat16()
    m.kv4_append(p.k, p.v, p.cache, p.slots)
    p.check(attend(m, p, lens, new))


# ---------------------------------------------------------------------------
# max_new
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
def test_a_step_without_new_tokens(m, dim):  # noqa: F811
    """Rows that only pad a step of fixed shape are zeros."""
    p = Problem(m, [40, 0, 300], [0, 0, 0], 2, 4, dim, 64, torch.half, seed=40, pad=3)
    assert not attend(m, p, [40, 0, 300], [0, 0, 0]).any()
    none = torch.zeros(0, 1, dtype=torch.int32, device=DEV)
    assert not m.kv4_attention(p.q, p.cache, none, ints([]), starts=ints([0]), max_new=0).any()


def test_requests_with_more_rows_than_max_new(m):  # noqa: F811
    """They are served, or their rows are NaN; the others' rows are what they are."""
    lens, new = [131, 200, 90, 128, 300], [2, 1, 0, 30, 300]
    p = Problem(m, lens, new, 2, 2, 64, 32, torch.half, seed=41, pad=2)
    for most in (0, 1, 2, 31):
        out = m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=most)
        assert torch.isnan(out[33:333]).all()
        out[33:333] = attend(m, p, lens, new)[33:333]
        p.check(out)
    p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=33))


@pytest.mark.parametrize("new", [[1, 2, 0], [1, 2, 300]])
def test_rows_before_the_first_request(m, new):  # noqa: F811
    lens = [131, 200, 300]
    p = Problem(m, lens, new, 2, 2, 64, 32, torch.half, seed=48, pad=2)
    q = torch.cat([torch.ones_like(p.q[:5]), p.q])
    out = m.kv4_attention(q, p.cache, p.tables, ints(lens), starts=ints([5 + x for x in p.starts]), max_new=max(new))
    assert not out[:5].any()
    p.check(out[5:])
    out = torch.full_like(q, 7.0)
    m.kv4_attention(q, p.cache, p.tables, ints(lens), starts=ints([5 + x for x in p.starts]), max_new=max(new), out=out)
    assert not out[:5].any()
    p.check(out[5:])


# ---------------------------------------------------------------------------
# a wait that runs out
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("lens,heads,group,ctas", [
    ([30000], 1, 8, (0, 30, 58)),              # one item of all CTAs that work
    ([30000] * 5, 1, 1, (0, 28, 144)),         # items with the same CTAs each
    ([9000, 8000, 7000], 3, 3, (0, 1, 77, 140))])  # CTAs that share an item on either side
def test_calls_after_a_wait_that_gave_up(m, lens, heads, group, ctas):  # noqa: F811
    """The workspace is as it was, whichever CTA gave up, and the next calls are right."""
    from csed499ii_b200 import _ext

    lib = _ext.load()
    assert m.device_status(0) == 0
    p = Problem(m, lens, [1] * len(lens), heads, group, 128, 64, torch.half, seed=42)
    space = m.kv4_workspace(DEV)
    args = (p.q, p.cache, p.tables, ints(lens))
    want = m.kv4_attention(*args, workspace=space)
    p.check(want)
    for cta in ctas:
        assert lib.sm100_marlin_kv4_stall(cta) == 0
        try:
            out = m.kv4_attention(*args, workspace=space)
        finally:
            assert lib.sm100_marlin_kv4_stall(-1) == 0
        assert m.device_status(0) != 0 and m.device_status(0) == 0
        assert not torch.equal(out, want) and not space[:1024].any()
        for _ in range(3):
            assert torch.equal(m.kv4_attention(*args, workspace=space), want)


# ---------------------------------------------------------------------------
# workspaces of graphs
# ---------------------------------------------------------------------------
def test_a_graph_has_its_own_workspace(m):  # noqa: F811
    """Also where calls on the captured stream came before: neither the module's
    workspace for that stream nor that of another graph is in it."""
    from csed499ii_b200 import kv4

    p = Problem(m, [9000, 40], [1, 1], 2, 8, 128, 64, torch.half, seed=43)
    lens = ints(p.lens)
    want = m.kv4_attention(p.q, p.cache, p.tables, lens)
    p.check(want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(DEV) for _ in range(3)]
    graphs, outs = [], []
    with torch.cuda.stream(streams[0]):
        m.kv4_attention(p.q, p.cache, p.tables, lens)
        for _ in range(2):
            streams[0].synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=streams[0]):
                outs.append(m.kv4_attention(p.q, p.cache, p.tables, lens))
            graphs.append(graph)
    torch.cuda.synchronize()
    kept = kv4._workspaces[0, streams[0].cuda_stream]
    kept[:1024] = 1  # counters that no call would join by
    for graph, out in zip(graphs, outs):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    kept[:1024] = 0
    for _ in range(20):  # both graphs and calls on the captured stream at once
        torch.cuda.synchronize()
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        got = []
        for _ in range(5):
            for graph, stream in zip(graphs, streams[1:]):
                with torch.cuda.stream(stream):
                    graph.replay()
            with torch.cuda.stream(streams[0]):
                got.append(m.kv4_attention(p.q, p.cache, p.tables, lens))
        torch.cuda.synchronize()
        assert all(torch.equal(x, want) for x in got + outs)


# ---------------------------------------------------------------------------
# large pages
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("new", [1, 150])
def test_offsets_past_32_bits_inside_a_page(m, new):  # noqa: F811
    """One page of 2^24 tokens takes 2.3 GB; the request's tokens are its last ones."""
    n, page, dim = 16384, 2**24, 128
    p = Problem(m, [n], [new], 1, 4, dim, 64, torch.half, seed=44)
    cache = torch.empty(1, 1, page // 16, 8 * dim + 64, dtype=torch.half, device=DEV)
    slots = torch.arange(page - n, page, dtype=torch.int32, device=DEV)
    m.kv4_append(p.k, p.v, cache, slots)
    k, v = m.kv4_read(cache, slots)
    assert torch.equal(k, R.values(p.k).half()) and torch.equal(v, R.values(p.v).half())
    # the window leaves the rest of the page unseen
    p.check(m.kv4_attention(p.q, cache, ints([[0]]), ints([page]), starts=ints(p.starts), max_new=new,
                            window=5000), 5000)


def test_the_longest_requests(m):  # noqa: F811
    """A table of 128 entries that are one page of 2^24 tokens holds 2^31: the last
    steps of such a request end at the limit of 32 bits."""
    page, dim, new = 2**24, 64, [1, 5, 100]
    cache = torch.zeros(1, 1, page // 16, 8 * dim + 64, dtype=torch.half, device=DEV)
    p = Problem(m, [3000] * 3, new, 1, 2, dim, 64, torch.half, seed=45)
    most = 2**31 - 256  # its last token is at 2^24 - 257 of the page
    m.kv4_append(p.k[:3000], p.v[:3000], cache, torch.arange(page - 3256, page - 256, dtype=torch.int32, device=DEV))
    p.k, p.v = p.k[:3000].repeat(3, 1, 1), p.v[:3000].repeat(3, 1, 1)
    for lens in ([most] * 3, [2**31 - 1] * 3):
        p.check(m.kv4_attention(p.q, cache, torch.zeros(3, 128, dtype=torch.int32, device=DEV), ints(lens),
                                starts=ints(p.starts), max_new=100, window=700), 700)
    assert not m.kv4_attention(p.q, cache, torch.zeros(3, 128, dtype=torch.int32, device=DEV), ints([-2**31, -5, 0]),
                               starts=ints(p.starts), max_new=100, window=700).any()


# ---------------------------------------------------------------------------
# inputs written right before
# ---------------------------------------------------------------------------
def test_keys_written_by_the_call_before(m):  # noqa: F811
    """kv4_append begins while the projection before it ends: its rows are the new ones."""
    k, heads, dim, rows = 2048, 4, 128, 48
    g = torch.Generator(device=DEV).manual_seed(46)
    layer = m.Layer_2_4(k, 2 * heads * dim, groupsize=128).to(DEV)
    w = torch.randn(k, 2 * heads * dim, generator=g, device=DEV).half() * 0.02
    layer.pack(type("W", (), {"weight": w, "bias": None})(), (w.view(k // 128, 128, -1).abs().amax(1) / 7).half())
    xs = [torch.randn(rows, k, generator=g, device=DEV).half() for _ in range(2)]
    want = [R.values(layer(x).view(rows, -1, dim)).half().split(heads, 1) for x in xs]
    workspace = torch.zeros(2 * heads * dim // 128 * 16, dtype=torch.int32, device=DEV)
    out = torch.zeros(rows, 2 * heads * dim, dtype=torch.half, device=DEV)
    cache = m.kv4_cache(3, heads, dim, 16, torch.half, DEV)
    slots = ints(list(range(rows)))
    for i in range(60):  # the same output, read by the call before, and written again
        m.mul_2_4(xs[i % 2], layer.B, layer.meta, out, layer.s, workspace)
        m.kv4_append(*out.view(rows, -1, dim).split(heads, 1), cache, slots)
        got = m.kv4_read(cache, slots)
        if i % 3 == 0:
            torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i % 2])), i


# ---------------------------------------------------------------------------
# scheduling into its inputs
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("where", ["new_lens", "lens, shifted", "new_lens, count in lens", "count first in lens"])
def test_schedule_writes_into_any_input(m, where):  # noqa: F811
    """New lengths and count that lie in what the step reads, with rows for many CTAs."""
    rng = random.Random(47)
    batch, page = 1300, 16
    for _ in range(5):
        new, lens, tables, free, count = schedule_case(rng, batch, page, 25, 300, 6000, KINDS["mixed"])
        rows = sum(max(0, x) for x in new) + 9
        want = R.schedule(new, lens, tables, free, count, rows, page)
        t_new, t_tables, t_free, t_count = ints(new), ints(tables), ints(free), ints([count])
        both = ints(lens + [0])
        t_lens, lens_out, count_out = both[:-1], t_new, None
        if where == "lens, shifted":
            lens_out = both[1:]
        elif where == "new_lens, count in lens":
            count_out = t_lens[700:701]
        elif where == "count first in lens":
            lens_out, count_out = None, t_lens[:1]
        step = m.kv4_schedule(t_new, t_lens, t_tables, t_free, t_count, rows, page, lens_out=lens_out,
                              free_count_out=count_out)
        for name in ("lens", "starts", "slots", "positions", "fate"):
            assert getattr(step, name).tolist() == want[name], name
        assert step.free_count.item() == want["free_count"]
        assert t_tables.tolist() == want["tables"] and t_free.tolist() == want["free"]


def test_schedule_refuses_rows_past_32_bits(m):  # noqa: F811
    one, tables = ints([1] * 3), ints([[0, 1]] * 3)
    for rows, page in ((2**31, 16), (2**32 + 3, 16), (3, 2**31), (3, 2**32 + 16)):
        with pytest.raises(RuntimeError, match="2\\*\\*31"):
            m.kv4_schedule(one, one, tables, ints([2, 3]), ints([2]), rows, page)
