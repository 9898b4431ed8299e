"""The barriers between the MMA warp, the tensor pipe and the softmax warps of the prompt attention kernels, on the CPU: every
order in which they can run, for a few tiles of keys.  A wait for a phase by its parity is lost for good once the phase after it
has ended too, and passes at once while the phase before has not; both only show in orders that a GPU seldom takes.

The softmax warps' waits for O are taken from the kernels' source."""
import os
import re

import pytest

from conftest import ROOT


def _source(name):
    with open(os.path.join(ROOT, "antares_b200", "csrc", name)) as f:
        return f.read()


class Stuck(Exception):
    pass


def explore(mma, warps, counts):
    """Runs every order.  mma: ("wait", barrier, parity), ("issue", product) and ("commit", barrier); warps: also ("arrive", barrier) and
    ("needs", product), which must be complete then, and ("first", product), which must not have been issued yet.  counts: arrivals that end a phase of each barrier."""
    names = sorted(counts)
    at = {b: i for i, b in enumerate(names)}
    programs = [mma] + warps

    def arrive(bars, b):
        ended, here = bars[at[b]]
        here += 1
        return bars[:at[b]] + ((ended + 1, 0) if here == counts[b] else (ended, here),) + bars[at[b] + 1:]

    # program counters, barriers (phases ended, arrivals of the present one), the pipe's queue: a prefix of what was issued
    start = ((0,) * len(programs), tuple((0, 0) for _ in names), (), frozenset())
    seen, todo = {start}, [start]
    while todo:
        pcs, bars, queue, done = todo.pop()
        nexts = []
        if queue:  # the tensor pipe ends what was issued first; a commit arrives
            kind, what = queue[0]
            nexts.append((pcs, arrive(bars, what) if kind == "commit" else bars, queue[1:], done | {what} if kind == "issue" else done))
        for i, prog in enumerate(programs):
            if pcs[i] == len(prog):
                continue
            op = prog[pcs[i]]
            b, q = bars, queue
            if op[0] == "wait":
                if bars[at[op[1]]][0] & 1 == op[2]:
                    continue
            elif op[0] == "arrive":
                b = arrive(bars, op[1])
            elif op[0] == "first":
                if op[1] in done or ("issue", op[1]) in queue:
                    raise Stuck("%s is issued too early" % (op[1],))
            elif op[0] == "needs":
                if op[1] not in done:
                    raise Stuck("%s is used before it is complete" % (op[1],))
            else:
                q = queue + (op,)
            nexts.append((pcs[:i] + (pcs[i] + 1,) + pcs[i + 1:], b, q, done))
        if not nexts and any(pc < len(p) for pc, p in zip(pcs, programs)):
            raise Stuck("waits for good: %s" % [p[pc] for pc, p in zip(pcs, programs) if pc < len(p)])
        for s in nexts:
            if s not in seen:
                seen.add(s)
                todo.append(s)


def _kv8_tail():
    """Parities that the softmax warps of kv8_prefill.cu wait for once their last P is written: offsets from the number of tiles."""
    text = _source("kv8_prefill.cu").split("// ---- O / l")[1].split("if (!good)")[0]
    return [int(n) for n in re.findall(r"kp_wait\(bar_o, \(my_n - (\d)\) & 1", text)]


def _kv8(n, parts, raises):
    mma = [("issue", ("s", 0, 0)), ("commit", "s0"), ("issue", ("s", 0, 1)), ("commit", "s1")]
    for j in range(n):
        if parts == 1 and j + 1 < n:
            mma += [("wait", "read", j & 1), ("issue", ("s", j + 1, 0)), ("commit", "s0")]
        mma += [("wait", "p", j & 1), ("issue", ("o", j)), ("commit", "o")]
        if j + 1 < n:
            mma += [("wait", "o", j & 1)]
            if parts == 2:
                mma += [("issue", ("s", j + 1, 0)), ("commit", "s0")]
            mma += [("issue", ("s", j + 1, 1)), ("commit", "s1")]
    warp = []
    for j in range(n):
        if parts == 2 and j > 0:  # fp32 rows: the product of the tile before is added to the others before the next may take its place
            warp += [("wait", "o", (j - 1) & 1), ("needs", ("o", j - 1)), ("first", ("o", j))]
        warp += [("wait", "s0", j & 1), ("needs", ("s", j, 0))]
        if raises and j > 0:  # the first half waits itself, the other's scores were only issued after the product of the tile before
            warp += ([("wait", "o", (j - 1) & 1)] if parts == 1 else []) + [("needs", ("o", j - 1))]
        warp += [("wait", "s1", j & 1), ("needs", ("s", j, 1))]
        warp += ([("needs", ("o", j - 1))] if raises and j > 0 else []) + ([("arrive", "read")] if parts == 1 else []) + [("arrive", "p")]
    for k in _kv8_tail():
        if n >= k:
            warp += [("wait", "o", (n - k) & 1)]
    return mma, [warp, list(warp)], [("needs", ("o", n - 1))]


@pytest.mark.parametrize("raises", [False, True])
@pytest.mark.parametrize("parts", [1, 2])
@pytest.mark.parametrize("n", [1, 2, 3, 4])
def test_the_prompt_kernel_over_the_8_bit_cache(n, parts, raises):
    mma, warps, last = _kv8(n, parts, raises)
    explore(mma, [w + last for w in warps], dict(s0=1, s1=1, p=2, o=1, read=2))


def test_the_model_finds_both_faults():
    """A wait for the last phase but one behind the last arrival is lost in some order; without a wait O is used too early."""
    mma, warps, last = _kv8(3, 1, False)
    bare = [[op for op in w if op[:2] != ("wait", "o")] for w in warps]
    with pytest.raises(Stuck, match="for good"):
        explore(mma, [w + [("wait", "o", 1), ("wait", "o", 0)] + last for w in bare], dict(s0=1, s1=1, p=2, o=1, read=2))
    with pytest.raises(Stuck, match="before it is complete"):
        explore(mma, [w + last for w in bare], dict(s0=1, s1=1, p=2, o=1, read=2))


def _fp16_waits():
    """What the softmax warps of attention_prefill.cu wait for of O: before their arrival with the last tile's P, and behind it; offsets
    from the number of tiles."""
    text = _source("attention_prefill.cu")
    loop, tail = text.split("// ---- softmax: thread = query row")[1].split("// ---- O / l, rounded")
    find = lambda t: [int(n) for n in re.findall(r"ap_wait\(b_odone, \(tiles - (\d)\) & 1", t)]  # noqa: E731
    return find(loop.split("ap_arrive(b_pfull")[0]), find(tail.split("if (!good)")[0])


def _fp16(n, raises):
    mma = [("issue", ("s", 0)), ("commit", "s0")]
    for j in range(n):
        if j > 0:
            mma += [("wait", "o", (j - 1) & 1)]
        if j + 1 < n:
            mma += [("issue", ("s", j + 1)), ("commit", "s%d" % (j + 1 & 1))]
        mma += [("wait", "p%d" % (j & 1), j >> 1 & 1), ("issue", ("o", j)), ("commit", "o")]
    early, late = _fp16_waits()
    warp = []
    for j in range(n):
        warp += [("wait", "s%d" % (j & 1), j >> 1 & 1), ("needs", ("s", j))]
        if raises and j > 0:
            warp += [("wait", "o", (j - 1) & 1), ("needs", ("o", j - 1))]
        if j == n - 1:
            warp += [("wait", "o", (n - k) & 1) for k in early if n >= k]
        warp += [("arrive", "p%d" % (j & 1))]
    warp += [("wait", "o", (n - k) & 1) for k in late if n >= k]
    return mma, [warp + [("needs", ("o", n - 1))] for _ in range(2)]


@pytest.mark.parametrize("raises", [False, True])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5])
def test_the_prompt_kernel_over_the_fp16_cache(n, raises):
    explore(*_fp16(n, raises), dict(s0=1, s1=1, p0=2, p1=2, o=1))
