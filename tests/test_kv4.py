"""The 4-bit cache without a GPU: what the C entries refuse before they touch
CUDA, what the Python surface refuses, and the plain implementations that the
GPU tests compare with."""
import math

import pytest
import torch

import kv4_reference as R


@pytest.fixture(scope="module")
def lib():
    from csed499ii_b200 import _ext, build

    build.build()
    return _ext.load()


P = 1 << 20  # an aligned address that nothing reads: every call below is refused first


def append(lib, **kw):
    a = dict(k=P, k_row=64, k_head=64, v=P, v_row=64, v_head=64, cache=P, pages=4, heads=1, page=16, dim=64,
             dtype=0, slots=P, tokens=1, dev=0, stream=None)
    return lib.sm100_marlin_kv4_append(*{**a, **kw}.values())


def attention(lib, **kw):
    a = dict(q=P, q_row=64, q_head=64, cache=P, pages=4, heads=2, page=16, dim=64, dtype=0, tables=P, stride=4,
             width=4, lens=P, starts=P, batch=1, rows=1, q_heads=2, max_new=1, window=0, scale=1.0, out=P,
             workspace=P, bytes=1 << 30, dev=0, stream=None)
    return lib.sm100_marlin_kv4_attention(*{**a, **kw}.values())


def schedule(lib, **kw):
    a = dict(new=P, lens=P, tables=P, stride=4, width=4, batch=1, free=P, capacity=4, count=P, rows=1, page=16,
             lens_out=P, count_out=P, starts=P, slots=P, positions=P, fate=P, dev=0, stream=None)
    return lib.sm100_marlin_kv4_schedule(*{**a, **kw}.values())


def test_c_entries_refuse_before_cuda(lib):
    from csed499ii_b200 import _ext as E

    for entry in (append, attention):
        assert entry(lib, dim=96) == E.ERR_KERN_SHAPE
        assert entry(lib, dtype=2) == E.ERR_ARGUMENT
        assert entry(lib, page=8) == E.ERR_PROB_SHAPE
        assert entry(lib, page=0) == E.ERR_PROB_SHAPE
        assert entry(lib, pages=-1) == E.ERR_PROB_SHAPE
        assert entry(lib, pages=2**27) == E.ERR_PROB_SHAPE
        assert entry(lib, heads=0) == E.ERR_PROB_SHAPE
        assert entry(lib, cache=None) == E.ERR_ARGUMENT
        assert entry(lib, cache=P + 8) == E.ERR_ALIGNMENT
    assert append(lib, tokens=-1) == E.ERR_PROB_SHAPE
    assert append(lib, tokens=0, k=None) == E.OK
    for name in ("k", "v", "slots"):
        assert append(lib, **{name: None}) == E.ERR_ARGUMENT
    assert append(lib, k=P + 1) == E.ERR_ALIGNMENT
    for kw in (dict(batch=-1), dict(rows=-1), dict(width=-1), dict(q_heads=3), dict(q_heads=0), dict(max_new=-1),
               dict(starts=None, rows=2)):
        assert attention(lib, **kw) == E.ERR_PROB_SHAPE, kw
    for kw in (dict(window=-1), dict(q=None), dict(out=None), dict(lens=None), dict(tables=None)):
        assert attention(lib, **kw) == E.ERR_ARGUMENT, kw
    assert attention(lib, out=P + 2) == E.ERR_ALIGNMENT
    assert attention(lib, rows=0) == E.OK
    for kw in (dict(batch=-1), dict(batch=8193), dict(rows=-1), dict(width=-1), dict(capacity=-1), dict(page=0)):
        assert schedule(lib, **kw) == E.ERR_PROB_SHAPE, kw
    for name in ("new", "lens", "tables", "free", "count", "lens_out", "count_out", "starts", "slots", "positions",
                 "fate"):
        assert schedule(lib, **{name: None}) == E.ERR_ARGUMENT, name


def test_python_refuses_host_tensors():
    import csed499ii_b200 as m

    cache = m.kv4_cache(2, 1, 64, 16, device="cpu")
    assert cache.shape == (2, 1, 1, 576)
    x, i = torch.zeros(1, 1, 64, dtype=torch.half), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: m.kv4_append(x, x, cache, i), lambda: m.kv4_read(cache, i),
                 lambda: m.kv4_attention(x, cache, i[None], i),
                 lambda: m.kv4_schedule(i, i, i[None], i, i, 1, 16)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_reference_quantisation():
    x = torch.tensor([[0.0, 1.0, 2.0, 15.0], [3.0, 3.0, 3.0, 3.0], [0.0, 0.0, 0.0, math.inf]]).half()
    codes, scale, low = R.quantise(x)
    assert codes[0].tolist() == [0, 1, 2, 15] and scale[0].item() == 1 and low[0].item() == 0
    assert codes[1].tolist() == [0] * 4 and scale[1].item() == 0 and low[1].item() == 3
    assert torch.isnan(R.values(x)[2]).all()
    y = torch.randn(50, 128, generator=torch.Generator().manual_seed(0)).half()
    step = R.quantise(y)[1]
    assert ((R.values(y) - y.double()).abs() <= 0.501 * step + 15 * 2.0**-11 * step).all()


def test_reference_attention_by_hand():
    """Two keys, one of them hidden from the first query."""
    k = torch.tensor([[[0.0, 15.0]], [[15.0, 0.0]]]).half()
    v = torch.tensor([[[1.0, 1.0]], [[-2.0, -2.0]]]).half()
    q = torch.tensor([[[1.0, 0.0]], [[0.1, 0.0]]]).half()
    out, bound = R.attention(q, k, v, 2, scale=1.0)
    w = 1 / (1 + math.exp(-15 * float(q[1, 0, 0])))
    assert out[0, 0].tolist() == [1.0, 1.0]
    assert abs(out[1, 0, 0].item() - (1 - 3 * w)) < 1e-12
    assert R.attention(q, k, v, 2, window=1, scale=1.0)[0][1, 0].tolist() == [-2.0, -2.0]
    assert (bound > 0).all()


def test_reference_schedule_by_hand():
    got = R.schedule([1, -1, 3, 1], [4, 5, 0, 8], [[9, -1], [7, 6], [-1, -1], [1, 2]], [3, -1, -1], 1, 5, 4)
    # the ended request's pages 7 and 6 are on top of 3
    assert got["slots"] == [6 * 4, 7 * 4, 7 * 4 + 1, 7 * 4 + 2, -1] and got["fate"] == [0, 0, 0, 2]
    assert got["lens"] == [5, 0, 3, 8] and got["free_count"] == 1 and got["free"] == [3, 7, 6]
    assert got["starts"] == [0, 1, 1, 4, 5] and got["positions"] == [4, 0, 1, 2, 8]
