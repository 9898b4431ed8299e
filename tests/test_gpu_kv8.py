"""The 8-bit paged cache's operators against their definitions in 64 bits (kv8_ref.py)."""
import numpy as np
import pytest
import torch

import kv8_ref
from antares_b200 import _lib, ops

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
INV_FREQ = (10000.0 ** -(np.arange(0, 128, 2) / 128)).astype(np.float32)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _setup(seed, past, rows, heads, page, spare=3, filled=True):
    """A cache whose pages lie in any order, what lies outside the sequences poisoned: huge scales, codes, table entries."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-max(p + n, 1) // page) for p, n in zip(past, rows)]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(past), max(need) + 2), 0x7FFFFFF0, dtype=torch.int32)
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[:n])
        order = order[n:]
    spread = 20 + 30 * torch.rand(pages, heads, 1, 1, generator=g)
    cache = []
    for _ in range(2):
        cache.append((torch.randn(pages, heads, page, 128, generator=g) * spread).round().clamp(-127, 127).to(torch.int8))
    for _ in range(2):
        cache.append(0.01 + 0.04 * torch.rand(pages, heads, page // 16, generator=g))
    for s, (p, n) in enumerate(zip(past, rows)):  # blocks that no position lies in yet
        for b in range(need[s] * page // 16):
            if 16 * b >= (p + n if filled else max(p, 0)):
                pg, i = int(table[s, 16 * b // page]), 16 * b % page // 16
                cache[2][pg, :, i] = float("nan")
                cache[3][pg, :, i] = float("inf")
    return [t.cuda() for t in cache], table.cuda()


def _wide(table, page):
    """The same table with room for 65536 positions: rows enough for the prompt kernel then go through it.  What it adds names
    no page."""
    return torch.cat([table, torch.full((table.shape[0], 65536 // page), 0x7FFFFFF0, dtype=torch.int32, device="cuda")], 1)


def _ref(cache, table):
    return kv8_ref.Cache(cache, table)


def _randn(seed, *shape, dtype=F16, mul=1.0):
    return (mul * torch.randn(*shape, generator=torch.Generator().manual_seed(seed))).to(dtype).cuda()


def _cu(rows):
    return _ints(np.cumsum([0] + list(rows)).tolist())


def _check_attention(got, ref_cache, q, pos0, cu, keys, dtype, scale=None, inv_freq=None, norm=True):
    want, spread, score, tiny = kv8_ref.attention(ref_cache, q.double().cpu().numpy(), pos0, cu, scale, inv_freq)
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    most = max(n for _, n in kv8_ref.rows_of(len(ref_cache.table), len(q), cu))
    single = dtype == F16 and most * q.shape[1] // ref_cache.k.shape[1] > 64
    off = np.abs(got - want) / kv8_ref.bound(want, spread, score, tiny, keys, dtype, single)
    assert off.max() <= 1, "off by %.2f of the bound at %s" % (off.max(), np.unravel_index(off.argmax(), off.shape))
    if single and norm:
        # in the mean both roundings are 2^-11 / sqrt(3) of a value at most: 2.8e-4 of the result for its own, as much for p's
        # (independent of one another, the values of a row about as large as their spread over the keys)
        assert np.linalg.norm(got - want) <= 4e-4 * np.linalg.norm(want)


# past, rows: lengths of one, block and page borders, empty rows and sequences
CASES = [
    ([0], [1], 4, 4, 16), ([15], [1], 4, 4, 16), ([16], [1], 4, 2, 16), ([31, 0, 500, 63], [1] * 4, 8, 1, 64), ([383], [1], 32, 32, 16), ([1000, 7, 77], [1] * 3, 14, 2, 32),
    ([5, 200, 31], [4] * 3, 16, 4, 32), ([100, 3], [2] * 2, 5, 1, 128), ([2500], [1], 16, 1, 256), ([300] * 40, [1] * 40, 8, 8, 32), ([129, 300], [8, 8], 32, 2, 64),
    ([0], [17], 4, 4, 16), ([0], [130], 4, 2, 16), ([77], [64], 8, 2, 32), ([0, 40, 333, 0], [3, 200, 1, 129], 6, 2, 64), ([10, 20, 30], [0, 70, 0], 4, 4, 32),
    ([1200, 5, 64], [90, 1, 300], 8, 1, 128), ([0, 0], [256, 256], 2, 2, 16),
    # prompts whose keys are one CTA's (many tiles of rows) or several, beside single rows
    ([0], [150], 32, 4, 16), ([0, 3, 70], [140] * 3, 32, 32, 32), ([5, 40, 333, 0, 100], [130, 70, 1, 0, 65], 32, 4, 32), ([700], [257], 20, 4, 64), ([1100, 0], [60, 400], 12, 12, 128),
    ([0], [129], 48, 16, 256), ([2000, 31], [3, 100], 63, 9, 64),
]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("past,rows,hq,hkv,page", CASES)
def test_attention(cuda, past, rows, hq, hkv, page, dtype):
    cache, table = _setup(len(past) + sum(rows), past, rows, hkv, page)
    T, uniform = sum(rows), len(set(rows)) == 1
    q = _randn(1, T, hq, 128, dtype=dtype, mul=2)
    cu = None if uniform else np.cumsum([0] + rows)
    got = ops.kv8_attention(q, cache, table, _ints(past), cu_rows=None if uniform else _cu(rows), max_rows=max(rows))
    ref = _ref(cache, table)
    _check_attention(got, ref, q, past, cu, max(p + n for p, n in zip(past, rows)), dtype)
    # the same rows whatever the hint says and however the rows are named
    for hint, t in ((1, table), (7, table), (T, table), (T, _wide(table, page)), (None, _wide(table, page))):
        again = ops.kv8_attention(q, cache, t, _ints(past), cu_rows=None if hint is None and uniform else _cu(rows), max_rows=hint)
        _check_attention(again, ref, q, past, cu, max(p + n for p, n in zip(past, rows)), dtype)
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("past,rows,hq,hkv", [([5000], [1], 64, 64), ([int(n) for n in np.random.RandomState(1).randint(-1, 700, 150)], [1] * 150, 4, 2),
                                              ([int(n) for n in np.random.RandomState(2).randint(-3, 400, 40)], [0, 1, 2, 7] * 10, 8, 2), ([3], [1], 64, 64)])
def test_shares_of_long_and_short_items(cuda, past, rows, hq, hkv, dtype):
    """Equal shares of all work whatever room the tables have: items in one share, in two and in many, shares of many items."""
    cache, table = _setup(41, past, rows, hkv, 64)
    table, q = _wide(table, 64), _randn(1, sum(rows), hq, 128, dtype=dtype, mul=2)
    cu = None if len(set(rows)) == 1 else np.cumsum([0] + rows)
    got = ops.kv8_attention(q, cache, table, _ints(past), cu_rows=None if cu is None else _cu(rows), max_rows=max(rows))
    _check_attention(got, _ref(cache, table), q, past, cu, max(p + n for p, n in zip(past, rows)), dtype)
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("mul", [0.0, 24.0])
@pytest.mark.parametrize("past,rows,hq,hkv", [([333, 64], [1, 1], 8, 2), ([50], [140], 4, 1), ([50], [140], 32, 4), ([0, 60], [140, 140], 32, 32)])
def test_flat_and_sharp_scores(cuda, past, rows, hq, hkv, mul, dtype):
    """All scores alike, and scores spread over hundreds: the running maximum moves often."""
    cache, table = _setup(3, past, rows, hkv, 32)
    q = _randn(2, sum(rows), hq, 128, dtype=dtype, mul=mul)
    for t in (table, _wide(table, 32)):
        got = ops.kv8_attention(q, cache, t, _ints(past), max_rows=max(rows))
        _check_attention(got, _ref(cache, table), q, past, None, max(p + n for p, n in zip(past, rows)), dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows", [1, 40, 150])
def test_block_scales_far_apart(cuda, rows, dtype):
    """Scales from 2^-40 to 2^12, and blocks of zeros, side by side."""
    past, hq, hkv = 200, 32, 4
    cache, table = _setup(5, [past], [rows], hkv, 64)
    g = torch.Generator().manual_seed(8)
    for t in cache[2:]:
        e = torch.randint(-40, 13, t.shape, generator=g).float()
        t.copy_(torch.where(torch.rand(t.shape, generator=g) < 0.2, 0.0, 2.0 ** e).cuda())
    cache[2].clamp_(max=2.0 ** -4)
    q = _randn(2, rows, hq, 128, dtype=dtype, mul=0.1)
    if dtype == F16:
        cache[3].clamp_(max=2.0 ** 5)
    ref = _ref(cache, table)
    table = _wide(table, 64)
    got = ops.kv8_attention(q, cache, table, _ints([past]))
    _check_attention(got, ref, q, [past], None, past + rows, dtype, norm=False)
    # a negative scale
    _check_attention(ops.kv8_attention(q, cache, table, _ints([past]), scale=-0.05), ref, q, [past], None, past + rows, dtype, scale=-0.05, norm=False)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows", [1, 5, 150])
def test_rows_with_nothing_to_attend_to(cuda, rows, dtype):
    """Negative positions attend to nothing (zeros), positions behind the table to all of it."""
    cache, table = _setup(6, [400 - rows, 400 - rows], [rows] * 2, 2, 64)
    table = table[:, :6].contiguous()  # capacity 384
    q = _randn(3, 2 * rows, 32, 128, dtype=dtype)
    for pos0 in ([-3, 384 - rows // 2], [-rows, -1000], [0, 383], [2 ** 31 - 1, -2 ** 31]):
        if max(pos0) > 10000 and rows > 1:
            continue
        got = ops.kv8_attention(q, cache, table, _ints(pos0), max_rows=rows)
        _check_attention(got, _ref(cache, table), q, pos0, None, 400, dtype)
        if max(pos0) < 0 and pos0[0] <= -rows:
            assert not got.any()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_queries_that_are_not_finite_stay_in_their_row(cuda, value, dtype):
    for past, rows in (([90], [3]), ([20], [150])):
        cache, table = _setup(7, past, rows, 2, 32)
        q = _randn(4, rows[0], 30, 128, dtype=dtype)
        table = _wide(table, 32)
        want = ops.kv8_attention(q, cache, table, _ints(past))
        q[1, 4, 7] = value
        got = ops.kv8_attention(q, cache, table, _ints(past))
        assert not got[1, 4].isfinite().any()
        keep = torch.ones(rows[0], 30, dtype=torch.bool, device="cuda")
        keep[1, 4] = False
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("past,rows,hkv,page", [([0], [1], 4, 16), ([5], [1], 1, 16), ([0], [33], 2, 32), ([30, 0, 47, 16], [1] * 4, 5, 64), ([7, 100, 0, 31], [40, 1, 0, 17], 3, 32),
                                               ([250], [300], 2, 128)])
def test_append(cuda, past, rows, hkv, page, rope, dtype):
    """Scales and codes as the definition has them; everything else keeps its bytes."""
    cache, table = _setup(sum(rows) + hkv, past, rows, hkv, page, filled=False)
    T, hq = sum(rows), 2 * hkv
    k, v, q = _randn(1, T, hkv, 128, dtype=dtype), _randn(2, T, hkv, 128, dtype=dtype, mul=3), _randn(3, T, hq, 128, dtype=dtype)
    ref = _ref(cache, table)
    uniform = len(set(rows)) == 1
    cu = None if uniform else np.cumsum([0] + rows)
    freq = torch.from_numpy(INV_FREQ).cuda() if rope else None
    kv8_ref.append(ref, k.float().cpu().numpy(), v.float().cpu().numpy(), past, cu, INV_FREQ if rope else None)
    got_q = ops.kv8_append(cache, k, v, table, _ints(past), cu_rows=None if uniform else _cu(rows), q=q if rope else None, inv_freq=freq)
    assert ops.kernel_status() == 0
    kc, vc, ks, vs = (t.cpu().numpy() for t in cache)
    assert np.array_equal(vs, ref.vs) and np.array_equal(vc, ref.v)
    if not rope or dtype == F32:
        assert np.array_equal(ks, ref.ks, equal_nan=True) and np.array_equal(kc, ref.k)
    else:
        # sines, cosines and the rotation in 32 bits: 2^-21 of the largest value, so a scale may differ by that and a code by one
        # where the quotient, at most 127, lies within 127 * 2^-20 of the middle of two
        assert np.allclose(ks, ref.ks, rtol=2.0 ** -20, atol=0, equal_nan=True)
        off = np.abs(kc.astype(int) - ref.k.astype(int))
        assert off.max() <= 1 and off.sum() <= max(2, 2e-3 * T * hkv * 128)
    if rope:
        pos = np.concatenate([np.arange(p, p + n) for p, n in zip(past, rows)])
        want = kv8_ref.rotate(q.double().cpu().numpy(), pos, INV_FREQ)
        tol = np.abs(want) * torch.finfo(dtype).eps / 2 * 1.01 + (2.0 ** -20 if dtype == F16 else 2.0 ** -30)
        assert (np.abs(got_q.double().cpu().numpy() - want) <= tol).all()
    else:
        assert got_q is None


@pytest.mark.parametrize("dtype", [F16, F32])
def test_append_token_by_token_and_growth(cuda, dtype):
    """Rows that arrive one at a time, each larger than the last: the block is rounded again at every growth."""
    cache, table = _setup(1, [0], [40], 2, 16, filled=False)
    ref = _ref(cache, table)
    for p in range(40):
        k, v = _randn(10 + p, 1, 2, 128, dtype=dtype, mul=1 + 0.3 * p), _randn(100 + p, 1, 2, 128, dtype=dtype)
        ops.kv8_append(cache, k, v, table, _ints([p]))
        kv8_ref.append(ref, k.float().cpu().numpy(), v.float().cpu().numpy(), [p])
    kc, vc, ks, vs = (t.cpu().numpy() for t in cache)
    assert np.array_equal(kc, ref.k) and np.array_equal(vc, ref.v) and np.array_equal(ks, ref.ks, equal_nan=True) and np.array_equal(vs, ref.vs)


def test_append_values_between_codes_and_extremes(cuda):
    """Middles between two codes go to the even one; infinities, NaN, zeros, subnormals and the largest values."""
    cache, table = _setup(2, [0], [16], 1, 16, filled=False)
    x = torch.zeros(16, 1, 128)
    x[0, 0] = torch.arange(-64, 64) + 0.5
    x[0, 0, 0] = 127.0                      # scale 1: the others lie in the middle of two codes
    x[1, 0, :4] = torch.tensor([float("inf"), float("-inf"), float("nan"), 1e-30])
    ref = _ref(cache, table)
    ops.kv8_append(cache, x.cuda(), x.cuda(), table, _ints([0]))
    kv8_ref.append(ref, x.numpy(), x.numpy(), [0])
    assert np.array_equal(cache[0].cpu().numpy(), ref.k) and ref.ks[int(table[0, 0])] == 1
    assert cache[0][int(table[0, 0]), 0, 1, :4].tolist() == [127, -127, 0, 0]
    for mul in (1e-42, 1e-33, 2.5e38, 0.0):
        y = (mul * torch.randn(16, 1, 128, generator=torch.Generator().manual_seed(1)).clamp(-1.3, 1.3)).float()
        ops.kv8_append(cache, y.cuda(), y.cuda(), table, _ints([0]))
        kv8_ref.append(ref, y.numpy(), y.numpy(), [0])
        assert np.array_equal(cache[0].cpu().numpy(), ref.k) and np.array_equal(cache[2].cpu().numpy(), ref.ks, equal_nan=True)


def test_append_outside_the_table(cuda):
    """Rows at negative positions and behind the table are not stored."""
    cache, table = _setup(4, [60, 60], [8, 8], 2, 32, filled=False)
    table = table[:, :2].contiguous()
    before = [t.clone() for t in cache]
    x = _randn(1, 16, 2, 128)
    ops.kv8_append(cache, x, x, table, _ints([-8, 64]))
    ops.kv8_append(cache, x, x, table, _ints([-2 ** 31, 2 ** 31 - 1]))
    assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(cache, before))
    ref = _ref(cache, table)
    ops.kv8_append(cache, x, x, table, _ints([-3, 61]))
    kv8_ref.append(ref, x.float().cpu().numpy(), x.float().cpu().numpy(), [-3, 61])
    assert np.array_equal(cache[0].cpu().numpy(), ref.k) and np.array_equal(cache[3].cpu().numpy(), ref.vs, equal_nan=True)
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("dtype", [F16, F32])
def test_read(cuda, dtype):
    past, rows = [0, 20, 9, 33], [50, 0, 1, 31]
    cache, table = _setup(9, past, rows, 3, 32)
    ref = _ref(cache, table)
    k, v = ops.kv8_read(cache, table, _ints(past), sum(rows), cu_rows=_cu(rows), dtype=dtype)
    at = 0
    for s, (p, n) in enumerate(zip(past, rows)):
        rk, rv = ref.values(s, p + n)
        for got, want in ((k, rk), (v, rv)):
            want = torch.from_numpy(want[p:]).float().to(dtype)
            assert torch.equal(got[at:at + n].cpu(), want)
        at += n
    # outside the table: zeros; rows behind the last sequence's: as they were
    out = tuple(torch.full((6, 3, 128), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    small = table[:2, :1].contiguous()
    ops.kv8_read(cache, small, _ints([-1, 31]), 6, cu_rows=_ints([0, 2, 4]), out=out)
    assert not out[0][0].any() and not out[1][3].any() and out[0][1].any() and out[1][2].any() and (out[0][4:] == 7).all() and (out[1][4:] == 7).all()


@pytest.mark.parametrize("rows", [1, 30, 200])
def test_rows_behind_the_last_sequence(cuda, rows):
    """A padded batch: rows that are nobody's keep what `out` held, and are zeros in a new result."""
    cache, table = _setup(11, [40, 3], [rows, 2], 2, 32)
    T = rows + 2 + 9
    q = _randn(1, T, 24, 128)
    ref, table = _ref(cache, table), _wide(table, 32)
    cu = _ints([0, rows, rows + 2])
    out = torch.full_like(q, 5.0)
    ops.kv8_attention(q, cache, table, _ints([40, 3]), cu_rows=cu, out=out)
    assert (out[rows + 2:] == 5).all()
    new = ops.kv8_attention(q, cache, table, _ints([40, 3]), cu_rows=cu)
    assert torch.equal(new[:rows + 2], out[:rows + 2]) and not new[rows + 2:].any()
    _check_attention(new[:rows + 2], ref, q[:rows + 2], [40, 3], np.array([0, rows, rows + 2]), 300, F16)
    qo = torch.full_like(q, 5.0)
    k = _randn(2, T, 2, 128)
    ops.kv8_append(cache, k, k, table, _ints([40, 3]), cu_rows=cu, q=q, inv_freq=torch.from_numpy(INV_FREQ).cuda(), q_out=qo)
    assert (qo[rows + 2:] == 5).all() and (qo[:rows + 2] != 5).any()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rope", [False, True])
@pytest.mark.parametrize("past,n,hq,hkv,page", [([383], 1, 32, 32, 16), ([0, 15, 16, 600, 31], 1, 8, 2, 32), ([20, 0], 3, 6, 1, 64), ([0], 20, 4, 4, 16), ([-1, 50], 1, 16, 2, 32),
                                               ([300, 17], 1, 40, 2, 128)])
def test_step(cuda, past, n, hq, hkv, page, rope, dtype):
    """One call = append, then attention, with q, k and v slices of one projection's result."""
    S = len(past)
    cache, table = _setup(13, past, [n] * S, hkv, page, filled=False)
    both = _randn(5, S * n, hq + 2 * hkv, 128, dtype=dtype)
    q, k, v = both[:, :hq], both[:, hq:hq + hkv], both[:, hq + hkv:]
    freq = torch.from_numpy(INV_FREQ).cuda() if rope else None
    apart = [t.clone() for t in cache]
    out = ops.kv8_step(q, k, v, cache, table, _ints(past), inv_freq=freq)
    ops.kv8_append(apart, k, v, table, _ints(past), inv_freq=freq)
    for a, b in zip(cache, apart):
        assert torch.equal(a.view(torch.int8), b.view(torch.int8))
    # against the cache as it now is; a rotated query may be kept in its type: half a step of it moves every score
    ref = _ref(cache, table)
    want, spread, score, tiny = kv8_ref.attention(ref, q.double().cpu().numpy(), past, None, None, INV_FREQ if rope else None)
    if rope:
        _, _, mag, _ = kv8_ref.attention(ref, q.double().cpu().numpy(), past, None)
        score = score + 1.5 * mag * 2.0 ** 19 * (torch.finfo(dtype).eps / 2 + 2.0 ** -21)
    off = np.abs(out.double().cpu().numpy() - want) / kv8_ref.bound(want, spread, score, tiny, max(past) + n, dtype)
    assert off.max() <= 1, off.max()
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("captured,wide", [(False, False), (True, False), (False, True)])
def test_steps_in_a_row(cuda, captured, wide, dtype):
    """A step's rows are written beside its attention's start and read by it: the bits of one call after the other, step by step,
    over the ends of blocks, with scales that grow (older rows of the block change too)."""
    past, hq, hkv, steps = [int(n) for n in np.random.RandomState(3).randint(0, 900, 30)], 16, 8, 24
    past[0] = 899
    cache, table = _setup(33, past, [steps] * len(past), hkv, 32)
    table = _wide(table, 32) if wide else table
    apart = [t.clone() for t in cache]
    q, k, v = (_randn(i, steps, len(past), h, 128, dtype=dtype) for i, h in ((1, hq), (2, hkv), (3, hkv)))
    k, v = (t * (1 + 0.2 * torch.arange(steps, device="cuda")).to(dtype)[:, None, None, None] for t in (k, v))
    pos0 = [_ints([n + i for n in past]) for i in range(steps)]
    run = lambda: [ops.kv8_step(q[i], k[i], v[i], cache, table, pos0[i]) for i in range(steps)]  # noqa: E731
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        graph.replay()
    else:
        outs = run()
    torch.cuda.synchronize()
    for i in range(steps):
        ops.kv8_append(apart, k[i], v[i], table, pos0[i])
        torch.cuda.synchronize()
        assert torch.equal(outs[i], ops.kv8_attention(q[i], apart, table, pos0[i])), i
    for a, b in zip(cache, apart):
        assert torch.equal(a.view(torch.int8), b.view(torch.int8))
    assert ops.kernel_status() == 0


def test_a_bad_page_is_reported(cuda):
    """Entries that name no page: nothing is written there, the status says so, and the next call is well."""
    for rows in (1, 150):
        cache, table = _setup(15, [70], [rows], 2, 32, filled=False)
        table = _wide(table, 32)
        table[0, 2] = cache[0].shape[0]
        before = [t.clone() for t in cache]
        x, q = _randn(1, rows, 2, 128), _randn(2, rows, 32, 128)
        ops.kv8_append(cache, x, x, table, _ints([70]))
        with pytest.raises(_lib.Ab200Error, match="page table"):
            ops.kernel_status()
        if rows == 1:
            assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(cache, before))
        ops.kv8_attention(q, cache, table, _ints([70]))
        with pytest.raises(_lib.Ab200Error, match="page table"):
            ops.kernel_status()
        k, _ = ops.kv8_read(cache, table, _ints([64]), 1)
        assert not k.any()
        with pytest.raises(_lib.Ab200Error, match="page table"):
            ops.kernel_status()
        assert ops.kernel_status() == 0


@pytest.mark.parametrize("make", [
    lambda: torch.arange(2 * 7 * 3 * 16, device="cuda").half().view(2, 7, 3, 16), lambda: torch.arange(7 * 5, device="cuda", dtype=torch.int32).view(1, 7, 5).float(),
    lambda: torch.randint(-128, 128, (3, 7, 11), device="cuda", dtype=torch.int8), lambda: torch.randn(4, 7, 40000, device="cuda").half(),
    lambda: torch.randn(7, 4, 64, device="cuda").transpose(0, 1), lambda: torch.randn(2, 9, 10, 64, device="cuda")[:, 1:8]])
def test_copy_pages(cuda, make):
    a, b = make(), make()
    want = [a.clone(), b.clone()]
    src, dst = [5, 0, 5, 2], [1, 3, 4, 6]
    for t in want:
        t[:, dst] = t[:, src].clone()
    ops.kv_copy_pages([a, b], src, dst)
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])


def test_copy_many_pages_of_several_types(cuda):
    """More pairs than one launch carries, a whole 8-bit cache at once."""
    g = torch.Generator().manual_seed(0)
    P, n = 2000, 900
    cache = [torch.randint(-127, 128, (2, P, 2, 16, 128), generator=g).to(torch.int8).cuda() for _ in range(2)] + [torch.rand(2, P, 2, 1, generator=g).cuda() for _ in range(2)]
    order = torch.randperm(P, generator=g).tolist()
    src, dst = order[:n], order[n:2 * n]
    want = [t.clone() for t in cache]
    for t in want:
        t[:, dst] = t[:, src].clone()
    ops.kv_copy_pages(cache, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(cache, want))


def test_refusals_of_tensors(cuda):
    cache, table = _setup(1, [10], [1], 2, 32)
    x, q, pos0 = _randn(1, 1, 2, 128), _randn(2, 1, 4, 128), _ints([10])
    bad = [lambda: ops.kv8_attention(q[..., :64], cache, table, pos0), lambda: ops.kv8_attention(q.bfloat16(), cache, table, pos0), lambda: ops.kv8_attention(q[:, :3], cache, table, pos0),
           lambda: ops.kv8_attention(q, cache, table.long(), pos0), lambda: ops.kv8_attention(q, cache, table, pos0.long()), lambda: ops.kv8_attention(q, cache, table, _ints([1, 2])),
           lambda: ops.kv8_attention(q, cache, table, pos0, cu_rows=_ints([0])), lambda: ops.kv8_attention(q, [cache[0], cache[1], cache[2][..., :0], cache[3]], table, pos0),
           lambda: ops.kv8_attention(q, [cache[0][:, :, :24], cache[1][:, :, :24], cache[2], cache[3]], table, pos0), lambda: ops.kv8_attention(q, cache, table, pos0, out=x),
           lambda: ops.kv8_append(cache, x, x.float(), table, pos0), lambda: ops.kv8_append(cache, x, x[:, :1], table, pos0), lambda: ops.kv8_append(cache, x, x, table, pos0, q=q),
           lambda: ops.kv8_append(cache, x, x, table, pos0, inv_freq=torch.ones(10, device="cuda")), lambda: ops.kv8_append(cache, x, x, table, pos0, q_out=q),
           lambda: ops.kv8_step(q, x, x, cache, table, pos0, out=q), lambda: ops.kv8_step(q, x, x, cache, table.t(), pos0), lambda: ops.kv8_read(cache, table, pos0, 1, dtype=torch.int8),
           lambda: ops.kv_copy_pages([cache[0][None]], [0], [0, 1]), lambda: ops.kv_copy_pages([], [], []), lambda: ops.kv_copy_pages([x[0]], [0], [1]),
           lambda: ops.kv8_attention(q.expand(4, 4, 128).transpose(0, 1), cache, table, pos0)]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, _lib.Ab200Error)):
            f()
            pytest.fail("call %d was taken" % i)
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("hq,hkv", [(8, 2), (32, 32)])
def test_captured_with_other_streams_alive(cuda, hq, hkv):
    """Two captured decode steps replayed on two streams at once, and an eager call between: each has its own scratch."""
    states = []
    for i in range(2):
        cache, table = _setup(20 + i, [700, 33], [1, 1], hkv, 32, filled=False)
        q, k = _randn(i, 2, hq, 128), _randn(9 + i, 2, hkv, 128)
        pos0 = _ints([700, 33])
        want = ops.kv8_step(q, k, k, [t.clone() for t in cache], table, pos0)
        states.append((cache, table, q, k, pos0, want))
    graphs, outs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for cache, table, q, k, pos0, _ in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.kv8_step(q, k, k, cache, table, pos0))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = ops.kv8_attention(states[0][2], states[1][0], states[1][1], _ints([600, 20]))
    torch.cuda.synchronize()
    for out, st in zip(outs, states):
        assert torch.equal(out, st[5])
    assert torch.equal(eager, ops.kv8_attention(states[0][2], states[1][0], states[1][1], _ints([600, 20])))


def test_same_bits_every_time(cuda):
    for past, rows, hq, hkv in (([3000, 1, 900], [1] * 3, 32, 8), ([500], [200], 8, 2), ([500], [200], 32, 2)):
        cache, table = _setup(30, past, rows, hkv, 64)
        q = _randn(1, sum(rows), hq, 128)
        first = ops.kv8_attention(q, cache, table, _ints(past))
        assert all(torch.equal(first, ops.kv8_attention(q, cache, table, _ints(past))) for _ in range(5))


def test_a_long_cache(cuda):
    """Positions beyond 2^17, cache offsets beyond 2^31 bytes (pages far up in a large cache)."""
    P, page, hkv, hq = 9000, 256, 8, 16   # 2.4 GB each of K and V
    past = 140001
    need = -(-(past + 1) // page)
    g = torch.Generator(device="cuda").manual_seed(1)
    k = torch.randint(-127, 128, (P, hkv, page, 128), generator=g, device="cuda", dtype=torch.int8)
    v = torch.randint(-127, 128, (P, hkv, page, 128), generator=g, device="cuda", dtype=torch.int8)
    ks, vs = (0.001 + 0.02 * torch.rand(P, hkv, page // 16, generator=g, device="cuda") for _ in range(2))
    table = torch.arange(P - 1, P - 1 - need, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    q, x = _randn(1, 1, hq, 128), _randn(2, 1, hkv, 128)
    ops.kv8_append((k, v, ks, vs), x, x, table, _ints([past]))
    got = ops.kv8_attention(q, (k, v, ks, vs), table, _ints([past])).double()
    pos = torch.arange(past + 1, device="cuda")
    pg, at = table[0].long()[pos // page], pos % page
    kk, vv = ((c[pg, :, at].double() * s[pg, :, at // 16].double()[..., None]) for c, s in ((k, ks), (v, vs)))
    sc = torch.einsum("hgd,lhd->hgl", q[0].double().view(hkv, hq // hkv, 128), kk) * 128 ** -0.5
    p = torch.softmax(sc, -1)
    want, spread = torch.einsum("hgl,lhd->hgd", p, vv).view(1, hq, 128), torch.einsum("hgl,lhd->hgd", p, vv.abs()).view(1, hq, 128)
    mag = torch.einsum("hgd,lhd->hgl", q[0].double().abs().view(hkv, hq // hkv, 128), kk.abs()).amax(-1).view(1, hq, 1) * 128 ** -0.5
    b = kv8_ref.bound(want.cpu().numpy(), spread.cpu().numpy(), (mag * 2.0 ** -18).cpu().numpy(), 0.0, past, F16)
    assert (np.abs((got - want).cpu().numpy()) <= b).all()
    back, _ = ops.kv8_read((k, v, ks, vs), table, _ints([past]), 1)
    assert torch.equal(back, (kk[-1:].float()).half())
    assert (back.float() - x.float()).abs().max() <= 0.5 * max(float(ks.max()), float(x.float().abs().max()) / 127) + 0.002


def test_pages_of_many_sequences(cuda):
    """The operators together, as a server uses them: prompts, decode steps, a fork, drafted tokens taken back, a request that
    ends, compaction; every sequence's rows read back as they were written, attention as over a cache of its own."""
    from antares_b200.kv_cache import PagedKV8Cache
    L, H, HQ = 2, 2, 4
    c = PagedKV8Cache(L, 24, H, page_rows=16, max_seqs=6, max_seq=128)
    g = torch.Generator().manual_seed(0)
    seen = {}   # sequence -> k, v rows of layer 1

    def write(need):
        c.reserve(need)
        seqs = sorted(need)
        table, pos0 = c.batch(seqs)
        rows = [need[s] for s in seqs]
        cu = _cu(rows)
        for l in range(L):
            k, v = (torch.randn(sum(rows), H, 128, generator=g).half().cuda() for _ in range(2))
            ops.kv8_append(c.layer(l), k, v, table, pos0, cu_rows=cu)
        at = 0
        for s, n in zip(seqs, rows):
            c.advance(s, n)
            seen[s] = torch.cat([seen.get(s, torch.zeros(0, 2, H, 128).cuda()), torch.stack([k[at:at + n], v[at:at + n]], 1)])
            at += n

    def check():
        seqs = sorted(seen)
        table, pos0 = c.batch(seqs)
        rows = [c.rows(s) for s in seqs]
        assert rows == [len(seen[s]) for s in seqs]
        k, v = ops.kv8_read(c.layer(1), table, torch.zeros_like(pos0), sum(rows), cu_rows=_cu(rows), dtype=F32)
        at = 0
        for s, n in zip(seqs, rows):
            for i, got in enumerate((k, v)):
                # a row is rounded once when it is written and again whenever its block's scale grows: half a step each, steps
                # that grow; the last is the largest |value| of 16 rows over 127, below 4.6 / 127 here, and 16 rows bring few records
                assert (got[at:at + n] - seen[s][:, i]).abs().max() <= 3 * 4.6 / 127
            at += n
        q = torch.randn(len(seqs), HQ, 128, generator=g).half().cuda()
        got = ops.kv8_attention(q, c.layer(1), table, pos0 - 1)
        _check_attention(got, _ref(c.layer(1), table), q, [r - 1 for r in rows], None, max(rows), F16)

    a, b = c.add(), c.add()
    write({a: 37, b: 5})
    check()
    d = c.fork(a)
    seen[d] = seen[a].clone()
    write({a: 1, b: 1, d: 1})
    check()
    write({d: 4})
    c.truncate(d, c.rows(d) - 3)
    seen[d] = seen[d][:-3]
    check()
    e = c.add()
    write({e: 60, d: 20})
    c.free(a)
    del seen[a]
    assert c.compact() > 0
    check()
    write({b: 30, d: 1, e: 1})
    check()
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows,hq", [(1, 8), (3, 8), (100, 32)])
def test_a_page_table_row_that_sequences_share(cuda, rows, hq, dtype):
    """An expanded table: as many sequences over one prompt, each with its own queries."""
    S, past = 5, 300
    cache, table = _setup(51, [past], [rows], 2, 32)
    table = _wide(table, 32)
    q, pos0 = _randn(1, S * rows, hq, 128, dtype=dtype), _ints([past, 0, past - 7, 40, 299])
    shared = table.expand(S, -1)
    assert torch.equal(ops.kv8_attention(q, cache, shared, pos0), ops.kv8_attention(q, cache, shared.contiguous(), pos0))
    for a, b in zip(ops.kv8_read(cache, shared, pos0, S * rows), ops.kv8_read(cache, shared.contiguous(), pos0, S * rows)):
        assert torch.equal(a, b)
    before = [t.clone() for t in cache]
    k = q[:, :2]
    for f in (lambda: ops.kv8_append(cache, k, k, shared, pos0), lambda: ops.kv8_step(q, k, k, cache, shared, pos0),
              lambda: ops.kv8_attention(q, cache, table[0].as_strided((S, 8), (1, 1)), pos0)):
        with pytest.raises(ValueError, match="overlap|written"):
            f()
    assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(cache, before))
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("pages,heads", [(4, 0), (0, 2)])
def test_a_cache_without_heads_or_pages(cuda, pages, heads):
    """Refused by both front ends (the native one divides by the heads)."""
    i8, f32 = dict(dtype=torch.int8, device="cuda"), dict(dtype=F32, device="cuda")
    cache = (torch.zeros(pages, heads, 16, 128, **i8), torch.zeros(pages, heads, 16, 128, **i8), torch.zeros(pages, heads, 1, **f32), torch.zeros(pages, heads, 1, **f32))
    table, q, k = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), _randn(1, 1, 4, 128), torch.zeros(1, heads, 128, dtype=F16, device="cuda")
    for f in (lambda: ops.kv8_attention(q, cache, table, _ints([0])), lambda: ops.kv8_step(q, k, k, cache, table, _ints([0])), lambda: ops.kv8_append(cache, k, k, table, _ints([0])),
              lambda: ops.kv8_read(cache, table, _ints([0]), 1)):
        with pytest.raises(ValueError, match="no heads or no pages"):
            f()


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_other_rows_over_the_same_pages_call_behind_call(cuda, dtype, captured):
    """Append and read in turn with nothing between them, other values each time at the same positions: every read has the rows of
    the append right before it."""
    past, rows, heads, turns = [0, 32, 5], [48, 1, 20], 8, 12
    cache, table = _setup(61, past, rows, heads, 32, filled=False)
    # the positions before: held already, so that every block that is read has been written
    first = _randn(7, sum(past), heads, 128, dtype=dtype)
    ops.kv8_append(cache, first, first, table, _ints([0, 0, 0]), cu_rows=_cu(past))
    start = [t.clone() for t in cache]
    T, cu, pos0 = sum(rows), _cu(rows), _ints(past)
    k, v = (_randn(i, turns, T, heads, 128, dtype=dtype) for i in (8, 9))
    k, v = (t * (1 + torch.arange(turns, device="cuda")).to(dtype)[:, None, None, None] for t in (k, v))
    freq = torch.from_numpy(INV_FREQ).cuda()

    def run():
        out = []
        for i in range(turns):
            ops.kv8_append(cache, k[i], v[i], table, pos0, cu_rows=cu, inv_freq=freq)
            out.append(ops.kv8_read(cache, table, pos0, T, cu_rows=cu, dtype=dtype))
        return out
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        graph.replay()
    else:
        outs = run()
    torch.cuda.synchronize()
    for t, s in zip(cache, start):
        t.copy_(s)
    for i in range(turns):
        torch.cuda.synchronize()
        ops.kv8_append(cache, k[i], v[i], table, pos0, cu_rows=cu, inv_freq=freq)
        torch.cuda.synchronize()
        for got, want in zip(outs[i], ops.kv8_read(cache, table, pos0, T, cu_rows=cu, dtype=dtype)):
            assert torch.equal(got, want), i
    assert ops.kernel_status() == 0


# many tiles of rows (keys are one CTA's), and few (keys in shares, joined)
WHOLE_OR_SHARED = [([0, 0, 0], [140] * 3, 32, 32), ([0], [150], 8, 2)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("past,rows,hq,hkv", WHOLE_OR_SHARED)
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_every_prompt_row_with_an_infinite_query_is_nan(cuda, past, rows, hq, hkv, value, dtype):
    """Scores that are infinite have no softmax, whichever keys they are of and whatever their signs: a code of either sign or of
    zero, the only score that is not -inf at any place of a block."""
    cache, table = _setup(71, past, rows, hkv, 32)
    table = _wide(table, 32)
    sign = 1 if value != float("-inf") else -1
    for d, high in ((7, ()), (8, (6, 7)), (9, (15,)), (10, (3,)), (11, tuple(range(16)))):
        codes = torch.full((32,), -5 * sign, dtype=torch.int8, device="cuda")
        for i in high:
            codes[i], codes[16 + i] = 5 * sign, 5 * sign
        cache[0][..., d] = codes
    cache[0][..., 12] = 0
    q = _randn(4, sum(rows), hq, 128, dtype=dtype)
    want = ops.kv8_attention(q, cache, table, _ints(past))
    assert want.isfinite().all()
    for d in (7, 8, 9, 10, 11, 12):
        for every in (1, 5):
            x = q.clone()
            x[::every, 1, d] = value
            got = ops.kv8_attention(x, cache, table, _ints(past))
            bad = torch.zeros(got.shape[:2], dtype=torch.bool, device="cuda")
            bad[::every, 1] = True
            assert got[bad].isnan().all(), (d, every, got[bad].isnan().all(1).logical_not().nonzero()[:5])
            assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("hq,hkv,rows", [(80, 80, 66), (4, 1, 66), (8, 2, 1)])
def test_keys_of_no_weight_add_nothing(cuda, hq, hkv, rows, dtype):
    """One key with large values has all the weight; 2000 others far below it hold values of scale 0, whose part of the sum counts
    2^100 times what their part of the product does."""
    past = 2000
    cache, table = _setup(72, [past], [rows], hkv, 64)
    page, rest = int(table[0, 0]), table[0, :-(-(past + rows) // 64)].long()
    for t, fill in ((cache[0], -100), (cache[1], 0), (cache[2], 0.02), (cache[3], 0.0)):
        t[rest] = fill
    g = torch.Generator().manual_seed(5)
    cache[0][page, :, :1] = 100
    cache[1][page, :, :1] = torch.randint(-1, 2, (hkv, 1, 128), generator=g).to(torch.int8).cuda()
    cache[3][page, :, 0] = 2.0 ** 15
    q = torch.ones(rows, hq, 128, dtype=dtype, device="cuda")
    q[:, :, ::3] = 0.5
    got = ops.kv8_attention(q, cache, _wide(table, 64), _ints([past]))
    _check_attention(got, _ref(cache, table), q, [past], None, past + rows, dtype, norm=False)


@pytest.mark.parametrize("rows,hq,hkv", [(1, 4, 4), (3, 16, 2), (150, 8, 2), (140, 80, 80)])
@pytest.mark.parametrize("e", [124, 118, 80, -80, -95, -118])
def test_queries_of_any_size(cuda, rows, hq, hkv, e):
    """fp32 queries up to the type's largest and down to its smallest, over keys that bring their scores back to ordinary ones."""
    past = 77
    cache, table = _setup(81, [past], [rows], hkv, 32)
    cache[2].mul_(2.0 ** min(-e, 118))
    q = _randn(3, rows, hq, 128, dtype=F32).clamp_(-6, 6) * 2.0 ** e
    got = ops.kv8_attention(q, cache, _wide(table, 32), _ints([past]))
    _check_attention(got, _ref(cache, table), q, [past], None, past + rows, F32)
    step = ops.kv8_attention(q[:1], cache, table, _ints([past]))
    _check_attention(step, _ref(cache, table), q[:1], [past], None, past + rows, F32)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows", [1, 30, 200])
def test_rows_in_front_of_the_first_sequence(cuda, rows, dtype):
    """A batch whose offsets do not begin at 0: the rows before are nobody's either."""
    cache, table = _setup(12, [40, 3], [rows, 2], 2, 32)
    table, freq = _wide(table, 32), torch.from_numpy(INV_FREQ).cuda()
    front, T = 5, rows + 2 + 5 + 4
    own = slice(front, front + rows + 2)
    q, k = _randn(1, T, 24, 128, dtype=dtype), _randn(2, T, 2, 128, dtype=dtype)
    cu, pos0 = _ints([front, front + rows, front + rows + 2]), _ints([40, 3])
    want = ops.kv8_attention(q[own], cache, table, pos0, cu_rows=_ints([0, rows, rows + 2]))
    out = torch.full_like(q, 5.0)
    ops.kv8_attention(q, cache, table, pos0, cu_rows=cu, out=out)
    torch.full_like(q, 7.0)  # memory that a new result may be given
    new = ops.kv8_attention(q, cache, table, pos0, cu_rows=cu)
    turned = ops.kv8_append(cache, k, k, table, pos0, cu_rows=cu, q=q, inv_freq=freq)
    back = ops.kv8_read(cache, table, pos0, T, cu_rows=cu, dtype=dtype)
    for t in (new, turned) + back:
        assert not t[:front].any() and not t[own.stop:].any() and t[own].any()
    assert torch.equal(new[own], want) and torch.equal(out[own], want) and (out[:front] == 5).all() and (out[own.stop:] == 5).all()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_rows_of_no_sequences_at_all(cuda, dtype):
    """S = 0 with rows: new results are zeros, a given one stays as it was."""
    cache, _ = _setup(1, [10], [1], 2, 32)
    table, pos0 = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    q, k, cu = _randn(1, 6, 4, 128, dtype=dtype), _randn(2, 6, 2, 128, dtype=dtype), torch.zeros(1, dtype=torch.int32, device="cuda")
    freq = torch.from_numpy(INV_FREQ).cuda()
    for _ in range(3):
        torch.full_like(q, 7.0), torch.full_like(k, 7.0)  # memory that a new result is given
        turned = ops.kv8_append(cache, k, k, table, pos0, cu_rows=cu, q=q, inv_freq=freq)
        assert not turned.any() and not ops.kv8_attention(q, cache, table, pos0, cu_rows=cu).any()
        assert not any(t.any() for t in ops.kv8_read(cache, table, pos0, 6, cu_rows=cu, dtype=dtype))
    out = torch.full_like(q, 5.0)
    ops.kv8_append(cache, k, k, table, pos0, cu_rows=cu, q=q, inv_freq=freq, q_out=out)
    assert (out == 5).all()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_rotated_queries_may_be_the_queries(cuda, dtype):
    """q_out over q itself, slices of one projection's result: the same rows, k and v untouched."""
    cache, table = _setup(91, [7], [40], 2, 32, filled=False)
    both, freq = _randn(1, 40, 10, 128, dtype=dtype), torch.from_numpy(INV_FREQ).cuda()
    q, k, v = both[:, :6], both[:, 6:8], both[:, 8:]
    before = both.clone()
    want = ops.kv8_append([t.clone() for t in cache], k, v, table, _ints([7]), q=q, inv_freq=freq)
    assert ops.kv8_append(cache, k, v, table, _ints([7]), q=q, inv_freq=freq, q_out=q) is q
    assert torch.equal(q, want) and torch.equal(both[:, 6:], before[:, 6:])
    for bad in (both[:, 4:], both[:, 1:7]):
        with pytest.raises(ValueError, match="may not lie over"):
            ops.kv8_append(cache, k, v, table, _ints([7]), q=q, inv_freq=freq, q_out=bad)
    out = torch.zeros(4, 2, 128, dtype=dtype, device="cuda")
    with pytest.raises(ValueError, match="may not lie over"):
        ops.kv8_read(cache, table, _ints([0]), 4, out=(out, out))


def test_a_serving_step_does_not_wait_for_the_gpu(cuda):
    """reserve, batch, append, attention, step, fork, compact and advance queue their work and return; what batch() uploads is what
    it was called for, however late the copy runs."""
    from antares_b200.kv_cache import PagedKV8Cache
    k, q = _randn(1, 40, 2, 128), _randn(2, 40, 4, 128)
    cu, busy = _ints([0, 20, 40]), torch.cuda.Event()

    def serve(c):
        a, b = c.add(), c.add()
        c.reserve({a: 20, b: 20})
        table, pos0 = c.batch([a, b])
        ops.kv8_append(c.layer(0), k, k, table, pos0, cu_rows=cu)
        ops.kv8_attention(q, c.layer(0), table, pos0, cu_rows=cu)
        c.advance(a, 20), c.advance(b, 20)
        seen = []
        d = c.fork(a)
        for _ in range(12):
            seqs = [b, a, d]
            c.reserve({s: 1 for s in seqs})
            table, pos0 = c.batch(seqs)
            seen.append((table, pos0, [list(c.pool.held[s]) for s in seqs], [c.rows(s) for s in seqs]))
            ops.kv8_step(q[:3], k[:3], k[:3], c.layer(0), table, pos0)
            for s in seqs:
                c.advance(s, 1)
        c.free(b)
        c.compact()
        return seen

    make = lambda: PagedKV8Cache(1, 40, 2, page_rows=16, max_seqs=8, max_seq=256)  # noqa: E731
    keep = serve(make())   # the first call of each kind loads its kernel and gets memory from the driver, which both wait
    c = make()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        torch.cuda._sleep(3_000_000_000)   # over a second
        busy.record()
        seen = serve(c)
        idle = [busy.query()]
    finally:
        torch.cuda.set_sync_debug_mode("default")
    del keep
    assert idle == [False]
    torch.cuda.synchronize()
    for table, pos0, held, rows in seen:
        assert table.shape == (3, 16) and table.is_cuda and pos0.tolist() == rows
        for row, pages in zip(table.tolist(), held):
            assert row == pages + [-1] * (16 - len(pages))
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("rows,hq,hkv", [(300, 80, 80), (300, 8, 1)])
def test_a_maximum_that_rises_inside_a_tile_rounds_nothing_twice(cuda, rows, hq, hkv):
    """fp16 prompts: one key with values 6.4 to 8 octaves above the first 128, behind it another that makes the maximum rise: what is
    held of the first is scaled, not rounded a second time."""
    past = 260
    cache, table = _setup(95, [past], [rows], hkv, 32)
    for t, fill in zip(cache, (0, 0, 0.02, 0.25)):
        t.fill_(fill)
    g = torch.Generator().manual_seed(3)
    place = lambda p: (int(table[0, p // 32]), slice(None), p % 32)  # noqa: E731
    cache[0][place(130)], cache[0][place(250)] = 0, 0
    cache[0][place(130) + (5,)], cache[0][place(250) + (5,)] = 100, 127
    cache[1][place(130)] = torch.randint(-127, 128, (hkv, 128), generator=g).to(torch.int8).cuda()
    # 128 ** -0.5 * log2(e) * 0.02 * 100 octaves for a query of 1
    q = torch.zeros(rows, hq, 128, dtype=F16, device="cuda")
    q[..., 5] = ((6.4 + 1.55 * torch.rand(rows, hq, generator=g)) / (128 ** -0.5 * 1.4426950408889634 * 2)).half().cuda()
    got = ops.kv8_attention(q, cache, _wide(table, 32), _ints([past]))
    _check_attention(got, _ref(cache, table), q, [past], None, past + rows, F16, norm=False)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("past,hq,hkv,rope", [([367], 32, 32, True), ([367], 32, 32, False), ([0], 8, 1, True), ([30, 600, 0, 15, 250], 16, 4, True), ([30, 600, 0, 15, 250], 16, 4, False)])
def test_steps_in_a_row_of_few_requests(cuda, past, hq, hkv, rope, captured, dtype):
    """A decoder's form of the step: tables no wider than its requests need, an item to a cluster of CTAs, which in fp16 write the new
    rows themselves.  Steps of growing values behind one another, over the ends of blocks and pages, have the bits of the same steps
    one at a time, and of append and attention apart."""
    steps, S = 40, len(past)
    cache, table = _setup(34, past, [steps] * S, hkv, 32, filled=False)
    filled = sum(past)
    if filled:  # rows that are there before, as a prompt's append leaves them
        x = _randn(9, filled, hkv, 128, dtype=dtype)
        ops.kv8_append(cache, x, x, table, _ints([0] * S), cu_rows=_cu(past))
    ahead, apart = ([t.clone() for t in cache] for _ in range(2))
    q, k, v = (_randn(i, steps, S, h, 128, dtype=dtype) for i, h in ((1, hq), (2, hkv), (3, hkv)))
    k, v = (t * (1 + 0.2 * torch.arange(steps, device="cuda")).to(dtype)[:, None, None, None] for t in (k, v))
    freq = torch.from_numpy(INV_FREQ).cuda() if rope else None
    pos0 = [_ints([n + i for n in past]) for i in range(steps)]
    run = lambda: [ops.kv8_step(q[i], k[i], v[i], cache, table, pos0[i], inv_freq=freq) for i in range(steps)]  # noqa: E731
    if captured:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        graph.replay()
    else:
        outs = run()
    torch.cuda.synchronize()
    for i in range(steps):
        one = ops.kv8_step(q[i], k[i], v[i], ahead, table, pos0[i], inv_freq=freq)
        torch.cuda.synchronize()
        assert torch.equal(outs[i], one), i
        ops.kv8_append(apart, k[i], v[i], table, pos0[i], inv_freq=freq)
        torch.cuda.synchronize()
        if not rope:
            assert torch.equal(one, ops.kv8_attention(q[i], apart, table, pos0[i])), i
    for a, b, c in zip(cache, ahead, apart):
        assert torch.equal(a.view(torch.int8), b.view(torch.int8)) and torch.equal(a.view(torch.int8), c.view(torch.int8))
    want, spread, score, tiny = kv8_ref.attention(_ref(cache, table), q[-1].double().cpu().numpy(), [n + steps - 1 for n in past], None, None, INV_FREQ if rope else None)
    if rope:  # a rotated query may be kept in its type: half a step of it moves every score
        score = score + 1.5 * kv8_ref.attention(_ref(cache, table), q[-1].double().cpu().numpy(), [n + steps - 1 for n in past], None)[2] * 2.0 ** 19 * (torch.finfo(dtype).eps / 2 + 2.0 ** -21)
    off = np.abs(outs[-1].double().cpu().numpy() - want) / kv8_ref.bound(want, spread, score, tiny, max(past) + steps, dtype)
    assert off.max() <= 1, off.max()
    assert ops.kernel_status() == 0


def _prompt_kernel_serves(q, cache, table, cu, most):
    """The library's rule: rows of a sequence (times group) beyond 64 in a call of more than 2.5 million rows of heads x positions."""
    group = q.shape[1] // cache[0].shape[1]
    return most * group > 64 and q.shape[0] * q.shape[1] * table.shape[1] * cache[0].shape[2] > 2500000


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("past,rows,hq,hkv,page", [c for c in CASES if max(c[1]) > 1])
def test_fp16_rows_of_the_few_row_kernel_hold_p_in_22_bits(cuda, past, rows, hq, hkv, page, wide):
    """The bound of a P held as a pair of fp16 numbers, 2^-20, for every row that the few-row kernel serves: all rows of calls that it
    serves alone, and short sequences beside prompts."""
    cache, table = _setup(len(past) + sum(rows), past, rows, hkv, page)
    ref = _ref(cache, table)
    table = _wide(table, page) if wide else table
    q, cu = _randn(1, sum(rows), hq, 128, mul=2), np.cumsum([0] + rows)
    got = ops.kv8_attention(q, cache, table, _ints(past), cu_rows=_cu(rows), max_rows=max(rows)).double().cpu().numpy()
    want, spread, score, tiny = kv8_ref.attention(ref, q.double().cpu().numpy(), past, cu)
    single = np.zeros(got.shape, bool)
    if _prompt_kernel_serves(q, cache, table, cu, max(rows)):
        for s, n in enumerate(rows):
            single[cu[s]:cu[s + 1]] = n * (hq // hkv) > 64
    keys = max(p + n for p, n in zip(past, rows))
    tight, loose = (kv8_ref.bound(want, spread, score, tiny, keys, F16, one) for one in (False, True))
    off = np.abs(got - want) / np.where(single, loose, tight)
    assert off.max() <= 1, (off.max(), np.unravel_index(off.argmax(), off.shape))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("past,rows,hq,hkv,page", [CASES[i] for i in (2, 3, 6, 8, 14, 18, 19, 20, 22)])
def test_results_over_the_queries_and_scratch_of_the_caller(cuda, past, rows, hq, hkv, page, wide, dtype):
    """out=q and a workspace of just the size that is asked for, filled with NaN: the bits of a new result."""
    cache, table = _setup(len(past) + sum(rows), past, rows, hkv, page)
    table = _wide(table, page) if wide else table
    S, T, cu = len(past), sum(rows), None if len(set(rows)) == 1 else _cu(rows)
    q, pos0 = _randn(1, T, hq, 128, dtype=dtype), _ints(past)
    want = ops.kv8_attention(q, cache, table, pos0, cu_rows=cu, max_rows=max(rows))
    n = ops.kv8_attention_workspace_bytes(S, T, max(rows), hq, hkv)
    room = torch.full((n + 4096,), 255, dtype=torch.uint8, device="cuda")
    keep = q.clone()
    assert torch.equal(ops.kv8_attention(q, cache, table, pos0, cu_rows=cu, max_rows=max(rows), workspace=room[:n]), want) and torch.equal(q, keep)
    assert ops.kv8_attention(q, cache, table, pos0, cu_rows=cu, max_rows=max(rows), out=q, workspace=room[:n]) is q
    assert torch.equal(q, want) and (room[n:] == 255).all()
    with pytest.raises(_lib.Ab200Error, match="workspace"):
        ops.kv8_attention(q, cache, table, pos0, cu_rows=cu, max_rows=max(rows), workspace=room[:64])
    assert ops.kernel_status() == 0


def test_a_batch_is_not_captured(cuda):
    """batch() uploads what the host knows now; a graph would keep the upload and replay it from memory that is another call's."""
    from antares_b200.kv_cache import PagedKV8Cache
    c = PagedKV8Cache(1, 8, 2, page_rows=16)
    a = c.add()
    c.reserve({a: 3})
    want = c.batch([a])
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="captured"):
            c.batch([a])
    graph.replay()
    torch.cuda.synchronize()
    assert (x == 1).all() and all(torch.equal(t, w) for t, w in zip(c.batch([a]), want))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("seqs,rows,group", [(76, 66, 1), (1, 66, 1), (150, 130, 1), (76, 1, 1), (500, 1, 1), (700, 1, 16), (1, 1, 8), (20, 9, 8)])
def test_many_keys_of_scale_zero_before_one_that_counts(cuda, seqs, rows, group, dtype):
    """20000 keys without values, nearly 2^8 times the weight of the first ones, then one key beside which they all are nothing: its
    values are the result, to 2^-30."""
    past = 20000
    cache, table = _setup(73, [past], [rows], 1, 64)
    for t, fill in zip(cache, (79, 0, 0.02, 0.0)):
        t.fill_(fill)
    at = lambda p: (int(table[0, p // 64]), 0, p % 64)  # noqa: E731
    for p in range(128):
        cache[0][at(p)] = 0
    cache[2][int(table[0, past // 64]), 0, past % 64 // 16] = 0.2      # the block of position 20000, a first one: its keys alone ...
    cache[3][int(table[0, past // 64]), 0, past % 64 // 16] = 0.25
    for p in range(past + 1, past - past % 16 + 16):                   # ... the first of which counts
        cache[0][at(p)] = 0
    values = torch.randint(-127, 128, (128,), generator=torch.Generator().manual_seed(1)).to(torch.int8).cuda()
    cache[1][at(past)] = values
    # 7.9 octaves for 79 * 0.02, 79 for 79 * 0.2
    q = torch.full((seqs * rows, group, 128), 7.9 / (79 * 0.02 * 128 ** 0.5 * 1.4426950408889634), dtype=dtype, device="cuda")
    got = ops.kv8_attention(q, cache, table.expand(seqs, -1), _ints([past] * seqs))
    want = (values.double() * 0.25).expand_as(got)
    # half a step of the result, half a step of one fp16 P (fp16 rows of the prompt kernel), the pair's and the exponential's 2^-20
    off = (got.double() - want).abs() / (want.abs() * (torch.finfo(dtype).eps / 2 * 1.01 + (2.0 ** -11 if dtype == F16 else 0) + 2.0 ** -20) + 1e-30)
    assert past % 16 == 0 and off.max() <= 1, (off.max(), got.isnan().sum())
    assert ops.kernel_status() == 0


def _exact_on_gpu(q, cache, table, past, rows):
    """Rows of sequences as long as one another, float64 [S rows, Hq, 128]."""
    S, hkv, hq = len(table), cache[0].shape[1], q.shape[1]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    for s in range(S):
        k, v = ((c[table[s].long()].double() * sc[table[s].long()].double().repeat_interleave(16, -1)[..., None]).permute(1, 0, 2, 3).reshape(hkv, -1, 128)
                for c, sc in ((cache[0], cache[2]), (cache[1], cache[3])))
        limit = past + 1 + torch.arange(rows, device="cuda")
        for h in range(hq):
            x = q[s * rows:(s + 1) * rows, h].double() @ k[h // (hq // hkv), :past + rows].T * 128 ** -0.5
            x.masked_fill_(torch.arange(past + rows, device="cuda") >= limit[:, None], float("-inf"))
            out[s * rows:(s + 1) * rows, h] = torch.softmax(x, -1) @ v[h // (hq // hkv), :past + rows]
    return out


def _check_sums(seqs, past, rows, hq, hkv, hint, wide):
    g = torch.Generator(device="cuda").manual_seed(0)
    page, need = 64, -(-(past + rows) // 64)
    codes = [(40 * torch.randn(seqs * need, hkv, page, 128, device="cuda", generator=g)).round().clamp(-127, 127).to(torch.int8) for _ in range(2)]
    cache = codes + [0.02 + 0.01 * torch.rand(seqs * need, hkv, page // 16, device="cuda", generator=g) for _ in range(2)]
    table = torch.arange(seqs * need, device="cuda").int().view(seqs, need)
    q = torch.randn(seqs * rows, hq, 128, device="cuda", generator=g)
    cu = _ints([i * rows for i in range(seqs + 1)]) if hint else None
    got = ops.kv8_attention(q, cache, _wide(table, page) if wide else table, _ints([past] * seqs), cu_rows=cu, max_rows=hint).double()
    some = min(seqs, 3)
    want, got = _exact_on_gpu(q[:some * rows], cache, table[:some], past, rows), got[:some * rows]
    bias = float(((got - want) * want).sum() / (want * want).sum())
    off = float((got - want).norm() / want.norm())
    # Added up in fp32 that rounds, errors have no sign.  A product's own sum takes 8 steps (with two blocks of keys: 4), cut towards zero by
    # at most 2^-23 of what it holds, on average half of a whole sum: 2^-21.  In all: that, scores of 2^-19 of their size (a few, and
    # half of them of either sign) and 2^-20 for weights and their exponentials: 2^-19 of the result's norm.
    assert abs(bias) <= 2.0 ** -21 and off <= 2.0 ** -19, (bias, off)
    assert ops.kernel_status() == 0


@pytest.mark.parametrize("seqs,past,rows,hq,hkv", [(1, 16000, 300, 8, 2), (1, 2000, 300, 160, 160), (76, 20000, 70, 1, 1)])
def test_sums_of_fp32_prompts_over_many_keys(cuda, seqs, past, rows, hq, hkv):
    _check_sums(seqs, past, rows, hq, hkv, None, True)


@pytest.mark.parametrize("seqs,past,rows,hq,hkv,hint", [(64, 16000, 1, 32, 8, None), (400, 8000, 1, 8, 1, None), (40, 16000, 4, 32, 8, None), (1, 16000, 300, 8, 2, 1), (3, 16000, 9, 8, 8, 9),
                                                            (1, 8000, 1, 222, 222, None), (1, 7000, 1, 32, 32, None)])
def test_sums_of_few_fp32_rows_over_many_keys(cuda, seqs, past, rows, hq, hkv, hint):
    _check_sums(seqs, past, rows, hq, hkv, hint, False)
