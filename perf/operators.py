"""The operators of a paged KV cache held in 8 bits, as they are timed.

  listed()         the cases
  draw(rng)        one more case of the same kinds and ranges
  prepare(case, s) what a serving program holds before the call: the cache's pages, the page table and positions, this
                   call's rows (from the seed s)
  run(state)       one pass: the framework's calls where `own` is true, elementary torch operations otherwise
  work(case)       bytes and operations one pass cannot do without
  exact(case, s)   what run() returns for the inputs of seed s, in 64 bits

The cache: k, v int8 [pages, kv heads, page rows, 128], one fp32 scale for each 16 rows and head, value = code * scale.
Position p of sequence s is row p % page_rows of page table[s, p // page_rows].
"""
import math
import random

import torch

own = False

D, BLOCK, CODES = 128, 16, 127.0
ROPE_BASE = 10000.0


def listed():
    return [
        # a whole prompt of the decoder's shape goes into the cache: rotary positions for queries and keys, codes for 2000 rows
        {"name": "append_prompt_2000", "kind": "append", "seqs": 1, "hq": 32, "hkv": 32, "rows": 2000, "ragged": False, "past": 0, "page": 64, "rope": True,
         "dtype": "float16", "mix": 1},
        # pieces of nine prompts behind filled caches, float32, keys that are rotated already, page and block borders anywhere
        {"name": "append_ragged_f32", "kind": "append", "seqs": 9, "hq": 12, "hkv": 4, "rows": 301, "ragged": True, "past": 500, "page": 32, "rope": False,
         "dtype": "float32", "mix": 2},
        # one token of one request, the decoder's heads: the smallest call, latency is what counts
        {"name": "step_1x384", "kind": "step", "seqs": 1, "hq": 32, "hkv": 32, "rows": 1, "ragged": False, "past": 383, "page": 16, "dtype": "float16", "mix": 3},
        # one token of 48 requests of any age, four query heads to a kv head
        {"name": "step_48_ragged", "kind": "step", "seqs": 48, "hq": 32, "hkv": 8, "rows": 1, "ragged": True, "past": 4000, "page": 64, "dtype": "float16", "mix": 4},
        # one token of one very long request: few rows over a long axis
        {"name": "attend_1x131072", "kind": "attend", "seqs": 1, "hq": 32, "hkv": 8, "rows": 1, "ragged": False, "past": 131071, "page": 256, "dtype": "float16",
         "mix": 5},
        # a full batch of decoding requests, eight query heads to a kv head
        {"name": "attend_64_ragged", "kind": "attend", "seqs": 64, "hq": 64, "hkv": 8, "rows": 1, "ragged": True, "past": 8000, "page": 64, "dtype": "float16",
         "mix": 6},
        # the operator-by-operator sample's type: float32 queries
        {"name": "attend_5_f32", "kind": "attend", "seqs": 5, "hq": 32, "hkv": 32, "rows": 1, "ragged": True, "past": 1000, "page": 16, "dtype": "float32", "mix": 7},
        # four drafted tokens a request are checked at once
        {"name": "verify_16x4", "kind": "attend", "seqs": 16, "hq": 32, "hkv": 4, "rows": 4, "ragged": True, "past": 3000, "page": 32, "dtype": "float16", "mix": 8},
        # a long prompt of the decoder's heads, from an empty cache
        {"name": "prefill_2000", "kind": "attend", "seqs": 1, "hq": 32, "hkv": 32, "rows": 2000, "ragged": False, "past": 0, "page": 64, "dtype": "float16", "mix": 9},
        # prompt pieces of different lengths, single tokens among them, behind filled caches
        {"name": "prefill_7_ragged", "kind": "attend", "seqs": 7, "hq": 32, "hkv": 8, "rows": 700, "ragged": True, "past": 2300, "page": 64, "dtype": "float16",
         "mix": 10},
        # requests are forked (one prompt, several answers): their last pages are copied, K and V of every layer of an fp16 cache
        {"name": "fork_fp16_32_layers", "kind": "copy", "layers": 32, "pages": 160, "move": 24, "page": 16, "width": 4096},
        # pages of freed requests leave holes: the rest moves together in an 8-bit cache, then the moved requests are read back
        {"name": "compact_read", "kind": "compact", "seqs": 6, "hq": 8, "hkv": 8, "rows": 900, "ragged": True, "past": 0, "page": 64, "dtype": "float16", "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "step", "step", "attend", "attend", "attend", "prefill", "prefill", "copy", "compact"])
    if kind == "copy":
        move = _log_int(rng, 1, 48)
        return {"kind": kind, "layers": _log_int(rng, 1, 32), "pages": 2 * move + rng.randrange(1, 60), "move": move, "page": rng.choice([16, 32, 64]),
                "width": D * rng.choice([1, 2, 4, 8, 16])}
    hkv, group = rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([1, 2, 4, 5, 7, 8, 16])
    while hkv * group > 64:
        group = rng.choice([1, 2, 4])
    c = {"kind": "attend" if kind == "prefill" else kind, "hkv": hkv, "hq": hkv * group, "page": rng.choice([16, 32, 64, 128, 256]), "ragged": rng.random() < 0.7,
         "dtype": "float32" if rng.random() < 0.2 else "float16", "mix": rng.randrange(1000000)}
    if kind == "append":
        c.update(seqs=_log_int(rng, 1, 32), rows=_log_int(rng, 1, 700), past=_log_int(rng, 1, 2000) - 1, rope=rng.random() < 0.5)
        c["rows"] = min(c["rows"], max(1, 2000 * 32 // (c["seqs"] * c["hkv"])))
    elif kind == "compact":
        c.update(seqs=_log_int(rng, 1, 16), rows=_log_int(rng, 1, 2000), past=0)
        c["rows"] = min(c["rows"], max(1, 2000 * 32 // (c["seqs"] * c["hkv"])))
    elif kind == "prefill":
        c.update(seqs=_log_int(rng, 1, 8), rows=_log_int(rng, 17, 1000), past=_log_int(rng, 1, 2500) - 1)
        c["rows"] = min(c["rows"], max(17, 350 * 7 * 32 // (c["seqs"] * c["hq"])))
    else:
        c.update(seqs=_log_int(rng, 1, 64), rows=1 if kind == "step" else rng.choice([1, 1, 1, 2, 5]), past=_log_int(rng, 1, 16000) - 1)
        c["past"] = min(c["past"], max(64, 4000 * 64 * 8 // (c["seqs"] * max(c["hkv"], c["hq"] // 8))))
    return c


# ---- what a program's scheduler knows on the host ------------------------------------------------------------

def _plan(case):
    """Rows in the cache before the call and new rows of each sequence; the longest of each kind is in every plan."""
    r = random.Random(case["mix"])
    past, rows = [case["past"]] * case["seqs"], [case["rows"]] * case["seqs"]
    if case["ragged"]:
        past[1:] = [r.randrange(case["past"] + 1) for _ in past[1:]]
        if case["rows"] > 8:  # prompts' pieces; drafted tokens and single ones are as many for each
            rows[1:] = [r.choice([1, r.randrange(1, case["rows"] + 1), r.randrange(1, case["rows"] + 1)]) for _ in rows[1:]]
    return past, rows


def _offsets(rows):
    at = [0]
    for n in rows:
        at.append(at[-1] + n)
    return at


# ---- inputs ----------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _codes(g, pages, hkv, page):
    """Filled pages: a block of normal values has its largest 2.5 to 4.5 times as far out as their spread."""
    spread = 28 + 22 * torch.rand(pages, hkv, 1, 1, generator=g, device="cuda")
    codes = (_randn(g, pages, hkv, page, D) * spread).round_().clamp_(-CODES, CODES).to(torch.int8)
    return codes, 0.02 + 0.01 * torch.rand(pages, hkv, page // BLOCK, generator=g, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    st = {"kind": case["kind"]}
    if case["kind"] == "copy":
        shape = (case["layers"], case["pages"], case["page"], case["width"])
        st["buffers"] = [_randn(g, *shape).half() for _ in range(2)]
        order = random.Random(seed).sample(range(case["pages"]), 2 * case["move"])
        st["src"], st["dst"] = order[:case["move"]], order[case["move"]:]
        st["src_dev"], st["dst_dev"] = _ints(st["src"]).long(), _ints(st["dst"]).long()
        return st
    past, rows = _plan(case)
    dt, page = getattr(torch, case["dtype"]), case["page"]
    T, longest = sum(rows), max(p + n for p, n in zip(past, rows))
    need = [-(-(p + n) // page) for p, n in zip(past, rows)]
    pages = sum(need) + 1   # the last page is nobody's
    table = torch.zeros(case["seqs"], max(need) + 1, dtype=torch.int32)
    ids = list(range(pages - 1))
    if case["kind"] == "compact":
        # every sequence's pages lie among twice as many; those in the upper half move into the holes of the lower half
        pages = 2 * sum(need) + 1
        ids = random.Random(seed).sample(range(pages - 1), sum(need))
        holes = sorted(set(range(sum(need))) - set(ids))
        st["src"] = [p for p in ids if p >= sum(need)]
        st["dst"] = holes[:len(st["src"])]
        st["src_dev"], st["dst_dev"] = _ints(st["src"]).long(), _ints(st["dst"]).long()
        new = dict(zip(st["src"], st["dst"]))
        ids = [new.get(p, p) for p in ids]   # the table after the move
    else:
        random.Random(seed).shuffle(ids)
    at = _offsets(need)
    for s in range(case["seqs"]):
        table[s, :need[s]] = torch.tensor(ids[at[s]:at[s + 1]], dtype=torch.int32)
    k, ks = _codes(g, pages, case["hkv"], page)
    v, vs = _codes(g, pages, case["hkv"], page)
    uniform = len(set(rows)) == 1
    st.update(cache=(k, v, ks, vs), table=table.cuda(), pos0=_ints(past), cu=None if uniform else _ints(_offsets(rows)), rows=T, most=max(rows), longest=longest, dtype=dt,
              scale=1 / math.sqrt(D), inv_freq=None)
    # where each row of the call lies: sequence and position, for the plain form's indexing
    st["seq"] = _ints([s for s, n in enumerate(rows) for _ in range(n)]).long()
    st["nth"] = _ints([i for n in rows for i in range(n)]).long()
    st["counts"], st["starts"] = _ints(rows).long(), _ints(_offsets(rows)[:-1]).long()
    st["q"] = _randn(g, T, case["hq"], D).to(dt)
    if case["kind"] in ("append", "step"):
        st["k"], st["v"] = _randn(g, T, case["hkv"], D).to(dt), _randn(g, T, case["hkv"], D).to(dt)
        if case.get("rope", True):
            j = torch.arange(0, D, 2, device="cuda").float() / D
            st["inv_freq"] = torch.cat([ROPE_BASE ** -j, ROPE_BASE ** -j])
        # what is read back: every block that a new row lies in, from the block's first row on
        first, end = [p // BLOCK * BLOCK for p in past], [min(-(-(p + n) // BLOCK) * BLOCK, page * table.shape[1]) for p, n in zip(past, rows)]
        back = [e - f for f, e in zip(first, end)]
        st["back"] = {"pos0": _ints(first), "cu": _ints(_offsets(back)), "rows": sum(back), "seq": _ints([s for s, n in enumerate(back) for _ in range(n)]).long(),
                      "nth": _ints([i for n in back for i in range(n)]).long()}
    return st


# ---- one pass ----------------------------------------------------------------------------------------------------

def _rotate(x, pos, inv_freq):
    """x [T, H, 128] rotated by halves at the positions pos [T], in fp32.  Angles are float32 products; sines and the sum are
    64-bit: codes next to the middle of two would go by the last bits of a sum in 32."""
    ang = (pos.float()[:, None] * inv_freq[None]).double()[:, None]
    x = x.double()
    turned = torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1)
    return (x * ang.cos() + turned * ang.sin()).float()


def _append_plain(st):
    """Returns the rotated queries (or None) in fp32; writes codes and scales."""
    k_codes, v_codes, k_scale, v_scale = st["cache"]
    page = k_codes.shape[2]
    pos = st["pos0"].long()[st["seq"]] + st["nth"]
    k, v, q = st["k"].float(), st["v"].float(), None
    if st["inv_freq"] is not None:
        k, q = _rotate(k, pos, st["inv_freq"]), _rotate(st["q"], pos, st["inv_freq"])
    # the blocks that new rows may lie in, [seqs, blocks, 16] positions each
    n_blocks = (st["most"] + 2 * BLOCK - 2) // BLOCK
    base = st["pos0"].long() // BLOCK
    at = ((base[:, None] + torch.arange(n_blocks, device="cuda")) * BLOCK)[..., None] + torch.arange(BLOCK, device="cuda")
    nth = at - st["pos0"].long()[:, None, None]
    is_new = (nth >= 0) & (nth < st["counts"][:, None, None])
    live = is_new.any(-1)
    is_old = (nth < 0) & live[..., None]
    row = st["starts"][:, None, None] + nth.clamp(min=0).minimum(st["counts"][:, None, None] - 1)
    table = st["table"].long()
    pages = torch.gather(table, 1, (at[..., 0] // page).clamp(max=table.shape[1] - 1))
    pages = torch.where(live, pages, k_codes.shape[0] - 1)    # blocks without a new row: the page that is nobody's
    in_page, block = at % page, at[..., 0] % page // BLOCK
    for codes, scales, x in ((k_codes, k_scale, k), (v_codes, v_scale, v)):
        was = codes[pages[..., None], :, in_page]             # [seqs, blocks, 16, heads, 128]
        s_old = torch.where(is_old.any(-1)[..., None], scales[pages, :, block], 0)
        new = torch.where(is_new[..., None, None], x[row], 0)
        s = torch.maximum(s_old, new.abs().amax((2, 4)) / CODES)
        value = torch.where(is_old[..., None, None], was.float() * s_old[:, :, None, :, None], new)
        # quotients near the middle of two codes need more than 32 bits
        code = (value.double() / s.double().clamp(min=1e-300)[:, :, None, :, None]).round().clamp(-CODES, CODES).to(torch.int8)
        codes[pages[..., None], :, in_page] = torch.where((is_new | is_old)[..., None, None], code, was)
        scales[pages, :, block] = torch.where(live[..., None], s, scales[pages, :, block])
    return q


def _values_plain(codes, scales, pages, in_page):
    return codes[pages, :, in_page].float() * scales[pages, :, in_page // BLOCK][..., None]


def _read_plain(st, at):
    k_codes, v_codes, k_scale, v_scale = st["cache"]
    page = k_codes.shape[2]
    pos = at["pos0"].long()[at["seq"]] + at["nth"]
    pages = st["table"].long()[at["seq"], pos // page]
    return [_values_plain(c, s, pages, pos % page).to(st["dtype"]) for c, s in ((k_codes, k_scale), (v_codes, v_scale))]


def _attend_plain(st, q):
    k_codes, v_codes, k_scale, v_scale = st["cache"]
    page, hkv = k_codes.shape[2], k_codes.shape[1]
    S, most, hq = st["table"].shape[0], st["most"], q.shape[1]
    pos = torch.arange(st["longest"], device="cuda")
    pages = st["table"].long()[:, pos // page]
    in_page = (pos % page).expand(S, -1)
    rows = torch.zeros(S, most, hq, D, device="cuda")
    rows[st["seq"], st["nth"]] = q.float()
    rows = rows.view(S, most, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(S, hkv, -1, D)
    k = _values_plain(k_codes, k_scale, pages, in_page).permute(0, 2, 3, 1)
    p = torch.matmul(rows, k).mul_(st["scale"]).view(S, hkv, hq // hkv, most, -1)
    last = st["pos0"].long()[:, None] + torch.arange(most, device="cuda")
    p.masked_fill_((pos > last[..., None])[:, None, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True)).view(S, hkv, -1, len(pos))
    v = _values_plain(v_codes, v_scale, pages, in_page).permute(0, 2, 1, 3)
    out = torch.matmul(p, v).view(S, hq, most, D)
    return out[st["seq"], :, st["nth"]].to(st["dtype"])


def run(st):
    kind = st["kind"]
    if own:
        from antares_b200 import ops
        if kind == "copy":
            ops.kv_copy_pages(st["buffers"], st["src"], st["dst"])
            return st["buffers"]
        if kind == "compact":
            ops.kv_copy_pages([t[None] for t in st["cache"]], st["src"], st["dst"])
            return ops.kv8_read(st["cache"], st["table"], st["pos0"], st["rows"], cu_rows=st["cu"], dtype=st["dtype"])
        if kind == "append":
            q = ops.kv8_append(st["cache"], st["k"], st["v"], st["table"], st["pos0"], cu_rows=st["cu"], q=None if st["inv_freq"] is None else st["q"],
                               inv_freq=st["inv_freq"])
            back = st["back"]
            return [q] + list(ops.kv8_read(st["cache"], st["table"], back["pos0"], back["rows"], cu_rows=back["cu"], dtype=st["dtype"]))
        if kind == "step":
            out = ops.kv8_step(st["q"], st["k"], st["v"], st["cache"], st["table"], st["pos0"], inv_freq=st["inv_freq"], scale=st["scale"])
            back = st["back"]
            return [out] + list(ops.kv8_read(st["cache"], st["table"], back["pos0"], back["rows"], cu_rows=back["cu"], dtype=st["dtype"]))
        return ops.kv8_attention(st["q"], st["cache"], st["table"], st["pos0"], cu_rows=st["cu"], max_rows=st["most"], scale=st["scale"])
    if kind in ("copy", "compact"):
        for t in st["buffers"] if kind == "copy" else [t[None] for t in st["cache"]]:
            t[:, st["dst_dev"]] = t[:, st["src_dev"]]
        return st["buffers"] if kind == "copy" else _read_plain(st, st)
    if kind == "append":
        q = _append_plain(st)
        return [None if q is None else q.to(st["dtype"])] + _read_plain(st, st["back"])
    if kind == "step":
        q = _append_plain(st)
        return [_attend_plain(st, q)] + _read_plain(st, st["back"])
    return _attend_plain(st, st["q"])


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "copy":
        return {"bytes": 2.0 * 2 * case["layers"] * case["move"] * case["page"] * case["width"] * 2, "flops": 0.0}
    past, rows = _plan(case)
    T, e, hq, hkv = sum(rows), 4 if case["dtype"] == "float32" else 2, case["hq"], case["hkv"]
    held = lambda n: n * hkv * 2 * D + -(-n // BLOCK) * hkv * 2 * 4  # noqa: E731  codes and scales of n rows, K and V
    q_bytes, flops = T * hq * D * e, 0.0
    back = sum(-(-(p + n) // BLOCK) * BLOCK - p // BLOCK * BLOCK for p, n in zip(past, rows))
    if case["kind"] == "compact":
        # every page moves with a chance of a half and is then read; the rows go out once
        moved = sum(-(-n // case["page"]) * case["page"] for n in rows) / 2
        return {"bytes": 2.0 * held(moved) + held(T) + T * hkv * 2 * D * e, "flops": float(T * hkv * 2 * D)}
    if case["kind"] == "append":
        return {"bytes": float(T * hkv * 2 * D * e + held(T) + (2 * q_bytes if case["rope"] else 0) + held(back) + back * hkv * 2 * D * e), "flops": 8.0 * T * (hkv * 2 + hq) * D}
    read = sum(held(p + n) for p, n in zip(past, rows))
    keys = sum(n * p + n * (n + 1) / 2 for p, n in zip(past, rows))
    flops = 4.0 * D * hq * keys
    if case["kind"] == "step":
        return {"bytes": float(read + 2 * q_bytes + T * hkv * 2 * D * e + held(T) + back * hkv * 2 * D * e), "flops": flops}
    return {"bytes": float(read + 2 * q_bytes), "flops": flops}


# ---- the same results in 64 bits -----------------------------------------------------------------------------------

def _place(st, s, n):
    """Page and row in the page of the positions 0 .. n - 1 of sequence s."""
    p, page = torch.arange(n, device="cuda"), st["cache"][0].shape[2]
    return st["table"][s].long()[p // page], p % page


def _sequence64(st, s, n):
    """K and V of the positions 0 .. n - 1 of sequence s, [n, heads, 128]."""
    pages, at = _place(st, s, n)
    k, v, ks, vs = st["cache"]
    return [c[pages, :, at].double() * f[pages, :, at // BLOCK].double()[..., None] for c, f in ((k, ks), (v, vs))]


def _turn64(x, first, inv_freq):
    ang = (torch.arange(first, first + x.shape[0], device="cuda").float()[:, None] * inv_freq[None, :D // 2]).double()[:, None]
    a, b = x[..., :D // 2], x[..., D // 2:]
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "copy":
        for t in st["buffers"]:
            t[:, st["dst_dev"]] = t[:, st["src_dev"]]
        return [t.double() for t in st["buffers"]]
    past, rows = _plan(case)
    at = _offsets(rows)
    if case["kind"] == "compact":
        for t in st["cache"]:
            t[st["dst_dev"]] = t[st["src_dev"]]
        pairs = [_sequence64(st, s, rows[s]) for s in range(len(rows))]
        return [torch.cat([p[i] for p in pairs]) for i in range(2)]
    outs, back = [], [[], []]
    for s, (p, n) in enumerate(zip(past, rows)):
        q = st["q"][at[s]:at[s + 1]].double()
        if case["kind"] == "attend":
            k, v = _sequence64(st, s, p + n)
        else:
            first, end = p // BLOCK * BLOCK, -(-(p + n) // BLOCK) * BLOCK
            pages, in_page = _place(st, s, end)
            held = []
            for i, name in enumerate("kv"):
                codes, scales = st["cache"][i], st["cache"][i + 2]
                x = st[name][at[s]:at[s + 1]].double()
                if name == "k" and st["inv_freq"] is not None:
                    x = _turn64(x, p, st["inv_freq"]).float().double()         # a code is the quotient of two 32-bit numbers
                c = codes[pages, :, in_page].double()                          # [end, heads, 128]
                f = scales[pages, :, in_page // BLOCK].double()                # [end, heads]
                old = f[first].clone() if p > first else torch.zeros_like(f[first])
                value = c[first:] * f[first:, :, None]
                value = torch.cat([value[:p - first], x, torch.zeros_like(value[p - first + n:])]).view(-1, BLOCK, *c.shape[1:])
                most = value.clone()
                most.view(-1, *c.shape[1:])[:p - first] = 0                    # older rows do not make the scale
                new = (most.abs().amax((1, 3)).float() / CODES).double()       # held in 32 bits
                new[0] = torch.maximum(new[0], old)
                q64 = (value / new.clamp(min=1e-300)[:, None, :, None]).round().clamp(-CODES, CODES).view(-1, *c.shape[1:])
                q64[p - first + n:] = c[p + n:]                                # rows behind the new ones keep their codes
                c[first:], f[first:] = q64, new.repeat_interleave(BLOCK, 0)
                held.append(c * f[..., None])
                back[i].append(held[-1][first:])
            k, v = held[0][:p + n], held[1][:p + n]
            if st["inv_freq"] is not None:
                q = _turn64(q, p, st["inv_freq"])
            if case["kind"] == "append":
                outs.append(q)
                continue
        group = case["hq"] // case["hkv"]
        later = torch.arange(p + n, device="cuda")[None] > torch.arange(p, p + n, device="cuda")[:, None]
        heads = []
        for h in range(case["hq"]):
            score = (q[:, h] @ k[:, h // group].T * st["scale"]).masked_fill_(later, -math.inf)
            heads.append(torch.softmax(score, -1) @ v[:, h // group])
        outs.append(torch.stack(heads, 1))
    if case["kind"] == "attend":
        return torch.cat(outs)
    return [torch.cat(outs) if case["kind"] == "step" or st["inv_freq"] is not None else None] + [torch.cat(b) for b in back]
