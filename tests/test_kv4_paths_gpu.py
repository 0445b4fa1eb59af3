"""Paths of the 4-bit cache that calls of other sizes and types take, on a GPU:
rows that stand for NaN in keys and values, more requests than one launch has
room for, and the entry points without the binding that takes torch tensors."""
import math
import random

import pytest
import torch

import kv4_reference as R
from test_kv4_gpu import DEV, KINDS, TYPES, Problem, ints, m, rows_of, schedule_case, some_slots  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_a_bad_row_of_either_kind(m, dtype, dim, where, what):  # noqa: F811
    """It spoils the rows that see it and no other, in both kernels."""
    lens, new = [200, 200, 300], [1, 200, 3]
    p = Problem(m, lens, list(new), 1, 2, dim, 64, dtype, seed=50)
    k, v = p.k.clone(), p.v.clone()
    x = k if where == "key" else v
    x[200 + 90, 0, 7] = what        # token 90 of the second request
    x[400 + 298, 0, dim - 1] = what  # the last but one of the third's: its first row does not see it
    m.kv4_append(k, v, p.cache, p.slots)
    for window in (0, 50):
        out = m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=200, window=window)
        bad = torch.zeros(204, dtype=torch.bool, device=DEV)
        bad[91:201 if not window else 91 + 50] = True
        bad[202:] = True
        assert torch.isnan(out[bad]).all() and torch.isfinite(out[~bad]).all()
        # the rows before the bad one are what they are
        check_some(p, out, [0], window)
        p.new[1], p.starts[2] = 90, 91
        p.lens, keys = [200, 90, 0], (p.k, p.v)
        p.k, p.v = (x[:290] for x in keys)
        check_some(p, out, [1], window)
        p.lens, p.new, p.starts, (p.k, p.v) = lens, list(new), [0, 1, 201, 204], keys


def check_some(p, out, which, window=0):
    """Problem.check for some of the requests."""
    at = [0]
    for n in p.lens:
        at.append(at[-1] + n)
    for b in which:
        rows = slice(p.starts[b], p.starts[b + 1])
        want, bound = R.attention(p.q[rows], p.k[at[b]:at[b + 1]], p.v[at[b]:at[b + 1]], p.new[b], window)
        assert ((out[rows].double() - want).abs() <= bound + 2.0**-24).all(), b


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_starts", [False, True])
def test_more_single_tokens_than_a_launch_has_room_for(m, dtype, with_starts):  # noqa: F811
    rng = random.Random(51)
    batch = 2100
    lens = [rng.choice([0, 1, 16, 33, rng.randint(1, 90)]) for _ in range(batch)]
    p = Problem(m, lens, [1] * batch, 2, 2, 64, 16, dtype, seed=52, pad=5 if with_starts else 0)
    kw = {"starts": ints(p.starts), "max_new": 1} if with_starts else {}
    out = m.kv4_attention(p.q, p.cache, p.tables, ints(lens), **kw)
    p.check(out)


def test_more_requests_than_a_prompt_launch_has_room_for(m):  # noqa: F811
    """Single tokens, and prompts at both ends and past request 8192."""
    rng = random.Random(53)
    batch = 8300
    lens, new = [rng.randint(0, 20) for _ in range(batch)], [1] * batch
    for b, n in ((0, 70), (5, 300), (8191, 129), (8192, 257), (8299, 66)):
        lens[b], new[b] = n + b % 3, n
    p = Problem(m, lens, new, 1, 1, 64, 16, torch.half, seed=54, pad=3)
    out = m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=300)
    assert torch.isfinite(out).all() and not out[p.starts[-1]:].any()
    check_some(p, out, [0, 1, 5, 6, 1023, 1024, 2047, 2048, 8190, 8191, 8192, 8193, 8298, 8299])
    empty = [b for b in range(batch) if lens[b] == 0]
    assert not out[torch.tensor([p.starts[b] for b in empty], device=DEV)].any()


# ---------------------------------------------------------------------------
# without the binding
# ---------------------------------------------------------------------------
@pytest.fixture
def without_binding(monkeypatch):
    from csed499ii_b200 import _ext

    assert _ext.torch_fast() is not None  # the tests elsewhere ran it
    monkeypatch.setattr(_ext, "_torch_fast", None)


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_schedule_without_the_binding(m, without_binding, kind):  # noqa: F811
    rng = random.Random(kind)
    for batch, page, width, spare in ((1, 16, 30, 100), (300, 16, 25, 2000)):
        new, lens, tables, free, count = schedule_case(rng, batch, page, width, 300, spare, KINDS[kind])
        rows = sum(max(0, x) for x in new) + 5
        want = R.schedule(new, lens, tables, free, count, rows, page)
        for in_place in (False, True):
            t_lens, t_tables, t_free, t_count = ints(lens), ints(tables), ints(free), ints([count])
            more = {"lens_out": t_lens, "free_count_out": t_count} if in_place else {}
            step = m.kv4_schedule(ints(new), t_lens, t_tables, t_free, t_count, rows, page, **more)
            for name in ("lens", "starts", "slots", "positions", "fate"):
                assert getattr(step, name).tolist() == want[name], name
            assert step.free_count.item() == want["free_count"]
            assert t_tables.tolist() == want["tables"] and t_free.tolist() == want["free"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_append_read_and_attention_without_the_binding(m, without_binding, dtype, dim):  # noqa: F811
    tokens, heads, page = 130, 3, 48
    cache = m.kv4_cache(5, heads, dim, page, dtype, DEV)
    k, v = rows_of(tokens, heads, dim, dtype, 1), rows_of(tokens, heads, dim, dtype, 2)
    slots = some_slots(tokens, 5 * page, 3)
    m.kv4_append(k, v, cache, slots)
    k2, v2 = m.kv4_read(cache, slots)
    assert torch.equal(k2, R.values(k).float().to(dtype)) and torch.equal(v2, R.values(v).float().to(dtype))
    lens, new = [131, 200, 0, 128], [4, 1, 0, 90]
    p = Problem(m, lens, new, 2, 4, dim, 32, dtype, seed=55, pad=3)
    p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=90))
    p = Problem(m, lens, [1] * 4, 2, 4, dim, 32, dtype, seed=56)
    p.check(m.kv4_attention(p.q, p.cache, p.tables, ints(lens)))
