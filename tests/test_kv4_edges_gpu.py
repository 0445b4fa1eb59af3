"""The 4-bit cache at the edges of what it accepts, on a GPU.

Tolerances are those that ``kv4_reference.attention`` derives; where values are
scaled by a power of two, which is exact in every step of the format, results
are scaled back and held to the bound of the values before.
"""
import pytest
import torch

import kv4_reference as R
from test_kv4_gpu import DEV, TYPES, Problem, ints, m  # noqa: F401  (m is the fixture)

pytestmark = pytest.mark.gpu


def attend(m, p, lens, new, **kw):  # noqa: F811
    return m.kv4_attention(p.q, p.cache, p.tables, ints(lens), starts=ints(p.starts), max_new=max(new), **kw)


# ---------------------------------------------------------------------------
# sizes of values
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("power", [-85, -70, -50, 0, 50, 70])
def test_values_of_any_exponent(m, dim, power):  # noqa: F811
    """The same values times a power of two: the same results times it."""
    lens, new = [400, 150], [1, 150]
    p = Problem(m, lens, new, 2, 2, dim, 64, torch.bfloat16, seed=31)
    m.kv4_append(p.k, p.v * 2.0**power, p.cache, p.slots)
    # of the result; the check is of the unscaled values
    p.check((attend(m, p, lens, new).double() * 2.0**-power).to(torch.bfloat16))


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
