"""The 8-bit paged cache on the CPU: what its calls refuse before any kernel runs."""
import ctypes
import re

import numpy as np
import pytest
import torch

import kv8_ref
from antares_b200 import _lib, ops


def _entry(name, *args):
    L = _lib.load()
    return getattr(L, name)(*args), L.ab200_last_error().decode()


CACHE = dict(k=4096, v=4096, ks=4096, vs=4096, pages=8, page_rows=32, H=2)
ROWS = dict(table=4096, stride=4, max_pages=4, pos0=4096, cu=None, S=2, T=2)


def _attention(q=4096, q_stride=512, out=4096, max_rows=1, Hq=4, D=128, dtype=0, **kw):
    a = {**CACHE, **ROWS, **kw}
    return _entry("ab200_kv8_attention", q, q_stride, out, a["k"], a["v"], a["ks"], a["vs"], a["pages"], a["page_rows"], a["H"], a["table"], a["stride"], a["max_pages"],
                  a["pos0"], a["cu"], a["S"], a["T"], max_rows, Hq, D, 0.1, 0, dtype, None, 0, None)


def _append(k=4096, v=4096, k_stride=256, v_stride=256, q=None, q_stride=0, q_out=None, qo_stride=0, Hq=0, freq=None, dtype=0, **kw):
    a = {**CACHE, **ROWS, **kw}
    return _entry("ab200_kv8_append", CACHE["k"], CACHE["v"], a["ks"], a["vs"], a["pages"], a["page_rows"], a["H"], a["table"], a["stride"], a["max_pages"], a["pos0"], a["cu"],
                  a["S"], a["T"], k, v, k_stride, v_stride, q, q_stride, q_out, qo_stride, Hq, freq, 0, dtype, None)


@pytest.mark.parametrize("change,code,word", [
    (dict(page_rows=24), _lib.EINVAL, "page_rows=24"), (dict(page_rows=8), _lib.EINVAL, "page_rows=8"), (dict(page_rows=0), _lib.EINVAL, "page_rows"),
    (dict(pages=0), _lib.EINVAL, "pages=0"), (dict(H=0), _lib.EINVAL, "heads=0"), (dict(stride=3), _lib.EINVAL, "table_stride=3"), (dict(max_pages=0), _lib.EINVAL, "max_pages=0"),
    (dict(max_pages=1 << 27, stride=1 << 27), _lib.EINVAL, "2^30"), (dict(S=-1), _lib.EINVAL, "S=-1"), (dict(T=3), _lib.EINVAL, "do not divide"), (dict(table=None), _lib.EINVAL, "null"),
    (dict(pos0=None), _lib.EINVAL, "null"), (dict(ks=None), _lib.EINVAL, "null"), (dict(k=4104), _lib.EINVAL, "aligned"), (dict(Hq=3), _lib.EINVAL, "multiple of 2"),
    (dict(Hq=0), _lib.EINVAL, "query heads"), (dict(D=64), _lib.EUNSUPPORTED, "head size 64"), (dict(dtype=2), _lib.EINVAL, "dtype 2"), (dict(q=4104), _lib.EINVAL, "aligned"),
    (dict(q_stride=500), _lib.EINVAL, "at least 512"), (dict(q_stride=516), _lib.EINVAL, "16 bytes"), (dict(out=None), _lib.EINVAL, "out"), (dict(T=1 << 29, S=1), _lib.EINVAL, "limits")])
def test_attention_refuses(change, code, word):
    rc, text = _attention(**change)
    assert rc == code and word in text and "kv8_attention" in text


@pytest.mark.parametrize("change,word", [
    (dict(k_stride=128), "at least 256"), (dict(v_stride=260), "16 bytes"), (dict(k=None), "16-byte"), (dict(q=4096), "come together"), (dict(q=4096, q_out=4096), "only rotated"),
    (dict(q=4096, q_out=4096, freq=4096, Hq=4, q_stride=512, qo_stride=500), "at least 512"), (dict(dtype=7), "dtype 7"), (dict(page_rows=48), "page_rows=48")])
def test_append_refuses(change, word):
    rc, text = _append(**change)
    assert rc == _lib.EINVAL and word in text


def test_nothing_to_do_is_no_error():
    assert _attention(S=0, T=0, q=None, out=None)[0] == 0 and _attention(T=0, q=None, out=None)[0] == 0
    assert _append(S=0, T=0, k=None, v=None)[0] == 0


def _copy(src, dst, pages=8, base=4096, layers=1, ls=0, ps=64, size=64, buffers=1):
    arr = lambda ty, v: ctypes.cast((ty * max(1, len(v)))(*v), ctypes.c_void_p)  # noqa: E731
    return _entry("ab200_kv_copy_pages", buffers, arr(ctypes.c_void_p, [base]), arr(ctypes.c_int, [layers]), arr(ctypes.c_long, [ls]), arr(ctypes.c_long, [ps]),
                  arr(ctypes.c_long, [size]), pages, arr(ctypes.c_int32, src), arr(ctypes.c_int32, dst), len(src), None)


@pytest.mark.parametrize("src,dst,word", [([0], [8], "outside"), ([-1], [2], "outside"), ([0, 1], [3, 3], "twice"), ([0, 3], [3, 4], "source and a destination"), ([2], [2], "source and")])
def test_page_lists_that_are_refused(src, dst, word):
    rc, text = _copy(src, dst)
    assert rc == _lib.EINVAL and word in text


@pytest.mark.parametrize("kw", [dict(base=0), dict(layers=0), dict(size=0), dict(ps=32), dict(ls=-64), dict(buffers=0), dict(buffers=9), dict(pages=0)])
def test_page_buffers_that_are_refused(kw):
    assert _copy([0], [1], **kw)[0] == _lib.EINVAL


def test_no_pairs_is_no_copy():
    assert _copy([], [])[0] == 0


def test_tensors_on_the_cpu_are_refused():
    cache = (torch.zeros(2, 1, 16, 128, dtype=torch.int8), torch.zeros(2, 1, 16, 128, dtype=torch.int8), torch.zeros(2, 1, 1), torch.zeros(2, 1, 1))
    table, pos0 = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 128).half()
    for f in (lambda: ops.kv8_append(cache, x, x, table, pos0), lambda: ops.kv8_attention(x, cache, table, pos0), lambda: ops.kv8_step(x, x, x, cache, table, pos0),
              lambda: ops.kv8_read(cache, table, pos0, 1), lambda: ops.kv_copy_pages([x[None]], [0], [0])):
        with pytest.raises(ValueError):
            f()


def test_the_reference_keeps_half_a_step():
    """The oracle itself: what it holds is within half a step of what it was given, after growth within a step and a half."""
    rng = np.random.default_rng(0)
    c = kv8_ref.Cache([torch.zeros(3, 2, 32, 128, dtype=torch.int8), torch.zeros(3, 2, 32, 128, dtype=torch.int8), torch.zeros(3, 2, 2), torch.zeros(3, 2, 2)],
                      torch.tensor([[2, 0]], dtype=torch.int32))
    x = rng.standard_normal((40, 2, 128)).astype(np.float32)
    kv8_ref.append(c, x, -x, [0])
    k, v = c.values(0, 40)
    step = np.repeat(np.concatenate([c.ks[2], c.ks[0]], 1), 16, 1).T[:40, :, None]
    assert (np.abs(k - x) <= step * 0.5000001).all() and (np.abs(v + x) <= step * 0.5000001).all()
    y = 3 * rng.standard_normal((1, 2, 128)).astype(np.float32)
    kv8_ref.append(c, y, y, [40])
    k, _ = c.values(0, 41)
    step = np.repeat(np.concatenate([c.ks[2], c.ks[0]], 1), 16, 1).T[:41, :, None]
    assert (np.abs(k[:40] - x) <= step[:40] * 1.0001).all() and (np.abs(k[40:] - y) <= step[40:] * 0.5000001).all()


def test_workspace_sizes_are_enough_for_every_call():
    """A call without a workspace says how much it needs, which the functions that size one must cover: whichever kernels serve it."""
    import random
    L = _lib.load()
    rng, fake = random.Random(1), 4096
    for _ in range(4000):
        hkv = rng.choice([1, 1, 2, 3, 8, 32])
        hq = hkv * rng.choice([1, 2, 5, 8, 33, 64, 65, 128])
        S, n = rng.choice([1, 2, 3, 16, 500]), rng.choice([1, 2, 3, 17, 64, 300, 2000])
        T, shift, dtype = S * n, rng.randrange(4, 9), rng.randrange(2)
        if T * hq > 1 << 30:
            continue
        cu = fake if rng.random() < 0.5 else None
        most = rng.choice([0, 1, n, T]) if cu else n
        max_pages = max(1, 2 ** rng.randrange(4, 22) >> shift)
        stride = (hq + 2) * 128
        cache = (fake, fake, fake, fake, 64, 1 << shift, hkv, fake, max_pages, max_pages, fake)
        assert L.ab200_kv8_attention(fake, stride, fake, *cache, cu, S, T, most, hq, 128, 0.1, 1, dtype, None, 0, None) != 0
        need = int(re.search(r"workspace of (\d+) bytes, got 0", L.ab200_last_error().decode()).group(1))
        assert need <= L.ab200_kv8_attention_workspace_bytes(S, T, most, hq, hkv), (hkv, hq, S, n, cu, most, max_pages, shift, dtype)
        assert L.ab200_kv8_step(fake, fake, fake, stride, stride, stride, fake, *cache, S, T, hq, 128, rng.choice([None, fake]), 0.1, dtype, None, 0, None) != 0
        need = int(re.search(r"workspace of (\d+) bytes, got 0", L.ab200_last_error().decode()).group(1))
        assert need <= L.ab200_kv8_attention_workspace_bytes(S, T, n, hq, hkv), (hkv, hq, S, n, max_pages, shift, dtype)


class OnGpu(torch.Tensor):
    """A tensor that says it lies on a GPU: for the host's checks of arguments, which look no further."""
    is_cuda = property(lambda self: True)


def _gpu(t):
    return t.as_subclass(OnGpu)


def _host_cache(pages=4, heads=2, rows=16):
    return tuple(_gpu(t) for t in (torch.zeros(pages, heads, rows, 128, dtype=torch.int8), torch.zeros(pages, heads, rows, 128, dtype=torch.int8),
                                   torch.zeros(pages, heads, rows // 16), torch.zeros(pages, heads, rows // 16)))


def test_page_tables_whose_rows_overlap():
    """Sequences may share one row of a table that is only read; the kernels step through a table by its own stride."""
    cache, pos0 = _host_cache(), _gpu(torch.zeros(3, dtype=torch.int32))
    one = torch.tensor([[2, 1, 3]], dtype=torch.int32)
    table = _gpu(one.expand(3, -1))
    args = ops._kv8_args(cache, table, pos0, None, 3)
    assert args[8] == 0 and args[9] == 3 and args[12] == 3
    with pytest.raises(ValueError, match="written"):
        ops._kv8_args(cache, table, pos0, None, 3, writes=True)
    windows = _gpu(torch.arange(6, dtype=torch.int32).as_strided((3, 3), (1, 1)))
    for writes in (False, True):
        with pytest.raises(ValueError, match="overlap"):
            ops._kv8_args(cache, windows, pos0, None, 3, writes=writes)
        # one row has no stride to speak of
        assert ops._kv8_args(cache, _gpu(one.expand(1, -1)), pos0[:1], None, 1, writes=writes)[8] >= 3
        assert ops._kv8_args(cache, _gpu(torch.zeros(3, 8, dtype=torch.int32)[:, :3]), pos0, None, 3, writes=writes)[8] == 8
    # the C entry points: readers take it (and ask for a workspace next), writers do not
    rc, text = _attention(stride=0)
    assert rc == _lib.EINVAL and "workspace" in text
    rc, text = _append(stride=0)
    assert rc == _lib.EINVAL and "table_stride=0" in text
    L = _lib.load()
    assert L.ab200_kv8_step(4096, 4096, 4096, 512, 256, 256, 4096, 4096, 4096, 4096, 4096, 8, 32, 2, 4096, 0, 4, 4096, 2, 2, 4, 128, None, 0.1, 0, None, 0, None) == _lib.EINVAL
    assert "table_stride=0" in L.ab200_last_error().decode()
    assert _append(stride=-4)[0] == _lib.EINVAL and _attention(stride=-4)[0] == _lib.EINVAL


@pytest.mark.parametrize("pages,heads", [(4, 0), (0, 2)])
def test_a_cache_without_heads_or_pages_is_refused(pages, heads):
    cache, x = _host_cache(pages, heads), _gpu(torch.zeros(1, 4, 128).half())
    table, pos0 = _gpu(torch.zeros(1, 2, dtype=torch.int32)), _gpu(torch.zeros(1, dtype=torch.int32))
    k = _gpu(torch.zeros(1, heads, 128).half())
    for f in (lambda: ops.kv8_attention(x, cache, table, pos0), lambda: ops.kv8_step(x, k, k, cache, table, pos0), lambda: ops.kv8_append(cache, k, k, table, pos0),
              lambda: ops.kv8_read(cache, table, pos0, 1)):
        with pytest.raises(ValueError, match="no heads or no pages"):
            f()


def test_the_cache_is_not_read_by_read_only_loads():
    """Its kernels start while the one before them may still write (programmatic launches): loads of memory that is read-only for a
    kernel's whole life (ld.global.nc, __ldg) are not for it."""
    import glob
    import os
    from conftest import ROOT
    files = glob.glob(os.path.join(ROOT, "antares_b200", "csrc", "kv8*.cu*")) + [os.path.join(ROOT, "antares_b200", "csrc", "kv_pages.cu")]
    assert len(files) >= 6
    for name in files:
        with open(name) as f:
            assert not re.search(r"\bld\.global\.nc|\b__ldg\(|\bldg_nc", f.read()), name


def test_whether_rows_meet():
    """Against every byte of both, for layouts of any stride."""
    import random
    rng, pool = random.Random(2), torch.zeros(40000, dtype=torch.float16)
    met = 0
    for _ in range(3000):
        T = rng.randrange(1, 6)
        sets = []
        for _ in range(2):
            heads = rng.randrange(1, 4)
            stride = heads * 128 + 64 * rng.choice([0, 0, 1, 2, 6, 8])
            sets.append(pool.as_strided((T, heads, 128), (stride, 128, 1), 64 * rng.randrange(0, 40)))
        mine, other = ({t.storage_offset() + i * t.stride(0) + j for i in range(T) for j in range(t.shape[1] * 128)} for t in sets)
        assert ops._rows_meet(*sets) == bool(mine & other), [(t.shape, t.stride(), t.storage_offset()) for t in sets]
        met += bool(mine & other)
    assert 500 < met < 2500
    assert not ops._rows_meet(pool[:0].view(0, 1, 128), pool[:128].view(1, 1, 128))


def test_results_over_inputs_are_refused():
    cache, table, pos0 = _host_cache(), _gpu(torch.zeros(1, 2, dtype=torch.int32)), _gpu(torch.zeros(1, dtype=torch.int32))
    freq, both = _gpu(torch.ones(64)), _gpu(torch.zeros(4, 8, 128).half())
    q, k, v = both[:, :4], both[:, 4:6], both[:, 6:]
    append = lambda q_out, q=q, k=k, v=v: ops.kv8_append(cache, k, v, table, pos0, q=q, inv_freq=freq, q_out=q_out)  # noqa: E731
    flat = _gpu(torch.zeros(6, 4, 128).half())
    for f in (lambda: append(both[:, 3:7]), lambda: append(both[:, 4:]), lambda: append(both[:, 2:6]), lambda: append(both[:, 1:5]), lambda: append(flat[1:5], q=flat[:4]),
              lambda: append(q.as_strided((4, 4, 128), (512, 128, 1)))):
        with pytest.raises(ValueError, match="may not lie over"):
            f()
    out = _gpu(torch.zeros(4, 2, 128).half())
    over_codes = cache[0].view(-1).view(torch.float16)[:2 * 2 * 128].view(2, 2, 128)
    # the kernels never see these: what refuses them is the host (a call that is taken ends at the missing GPU instead)
    for f in (lambda: ops.kv8_read(cache, table, pos0, 4, out=(out, out)), lambda: ops.kv8_read(cache, table, pos0, 3, out=(out[:3], out[1:])),
              lambda: ops.kv8_read(cache, table, pos0, 2, out=(out[:2], over_codes)), lambda: ops.kv8_attention(_gpu(torch.zeros(2, 2, 128).half()), cache, table, pos0, out=over_codes)):
        with pytest.raises(ValueError, match="may not lie over"):
            f()
    for good in (q, _gpu(torch.zeros(4, 4, 128).half()), None):
        with pytest.raises(Exception) as e:
            append(good)
        assert "may not lie over" not in str(e.value)
