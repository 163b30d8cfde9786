"""Operators of a serving step over independent requests against plain implementations in 64 bits.

Tolerances.  A result rounded to bfloat16 is off by at most 2^-8 of its value; float32 sums of n terms by at most n 2^-24 of the sum of
the terms' magnitudes.  What a kernel rounds besides is said at each test.
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from ade_b200 import kernels, synth
from ade_b200.decode_ops import token_logprobs
from ade_b200.kernels import bank_deltas, multi_delta_forward
from ade_b200.paged import paged_attn_decode, paged_extend, paged_write

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


# ------------------------------------------------------------------------------------ paged_extend
def _extend_by_hand(lengths, new, table, free, count, total, ps):
    """The rules one request at a time, on Python lists."""
    B, W, pages = len(lengths), len(table[0]), len(free)
    lengths, table, stack = list(lengths), [list(r) for r in table], list(free[:count])
    status, rows = [0] * B, []
    ceil = lambda a: -(-a // ps)
    bad = [not 0 <= n <= W * ps for n in lengths]
    for b in range(B):
        if new[b] < 0 and not bad[b]:
            stack += table[b][:ceil(lengths[b])]
    free = stack + list(free[len(stack):])
    asked = at = 0
    for b in range(B):
        if bad[b]:
            status[b] = 4
            continue
        if new[b] < 0:
            lengths[b] = 0
            continue
        start, at, end = at, at + new[b], lengths[b] + new[b]
        rows += [(-1, 0, -1)] * (min(at, total) - len(rows))
        if at > total:
            status[b] = 3
            continue
        if ceil(end) > W:
            status[b] = 2
            continue
        need = ceil(end) - ceil(lengths[b])
        asked += need
        if need and asked > len(stack):
            status[b] = 1
            continue
        for j in range(need):
            table[b][ceil(lengths[b]) + j] = stack[len(stack) - 1 - (asked - need + j)]
        for i in range(new[b]):
            pos = lengths[b] + i
            page = table[b][pos // ps]
            if 0 <= page < pages:
                rows[start + i] = (page * ps + pos % ps, pos, b)
        lengths[b] = end
    rows += [(-1, 0, -1)] * (total - len(rows))
    return lengths, table, free, len(stack), status, rows


def _check_extend(lengths, new, table, free, count, total, ps, in_place=False):
    """One call against the rules; returns the state behind it."""
    want_len, want_table, want_free, height, want_status, want_rows = _extend_by_hand(lengths, new, table, free, count, total, ps)
    ceil = lambda a: -(-a // ps)
    taken = sum(ceil(w) - ceil(n) for w, n, s, f in zip(want_len, lengths, want_status, new) if s == 0 and f >= 0)
    t, f, c, n = _i32(table), _i32(free), _i32([count]), _i32(lengths)
    out = paged_extend(n, _i32(new), t, f, c, total, ps, in_place=in_place)
    slots, positions, requests, new_len, new_count, status = out
    if in_place:
        assert new_len is n and new_count is c
    else:
        assert n.tolist() == list(lengths) and c.item() == count
    assert status.tolist() == want_status
    assert new_len.tolist() == want_len
    assert new_count.item() == height - taken
    assert t.tolist() == want_table
    assert f.tolist()[:height] == want_free[:height]
    assert list(zip(slots.tolist(), positions.tolist(), requests.tolist())) == want_rows
    return new_len.tolist(), t.tolist(), f.tolist(), new_count.item()


@pytest.mark.parametrize("B, width, ps, pages, seed", [(1, 3, 4, 3, 0), (5, 4, 1, 12, 1), (33, 6, 16, 90, 2), (64, 5, 24, 400, 3), (1025, 3, 8, 1500, 4), (300, 4, 16, 700, 7),
                                                       (4096, 2, 64, 8192, 5), (7, 9, 3, 20, 6)])
def test_extend_follows_the_rules_step_by_step(B, width, ps, pages, seed):
    """Requests enter, grow, rest, end and fail (no page, a full table, no row) over ten steps; no page is ever owned twice."""
    rng = random.Random(seed)
    free = list(range(pages))
    rng.shuffle(free)
    lengths, table, count = [0] * B, [[-1] * width for _ in range(B)], pages
    for step in range(10):
        most = rng.choice([1, 1, ps, 2 * ps + 1, width * ps])
        new = [rng.choice([-1, 0, 0, 1, 1, 1, rng.randint(0, most)]) for _ in range(B)]
        total = rng.choice([sum(max(n, 0) for n in new), sum(max(n, 0) for n in new) + 5, max(0, sum(max(n, 0) for n in new) - 3), B])
        lengths, table, free, count = _check_extend(lengths, new, table, free, count, total, ps, in_place=step % 2 == 1)
        owned = [p for b in range(B) for p in table[b][:-(-lengths[b] // ps)]]
        assert sorted(owned + free[:count]) == list(range(pages))


def test_extend_takes_bad_states_for_what_they_are():
    # lengths that no request can have stay as they are and cost nothing; a released request without tokens hands nothing back
    _check_extend([-1, 200, 0, 3, 8], [1, 1, -1, 2, -1], [[0, 1], [2, 3], [-1, -1], [4, -1], [5, 6]], [7, 8, 9, -1, -1, -1, -1, -1, -1, -1], 3, 6, 4)
    # a table whose entry is no page: the row of that token has no slot
    _check_extend([3, 3], [1, 1], [[99, -1], [-7, -1]], [0, 1], 2, 2, 4)
    # rows behind the last token, no rows at all, tokens that do not fit
    _check_extend([0, 0], [2, 1], [[-1], [-1]], [0, 1], 2, 9, 4)
    _check_extend([1, 1], [0, 0], [[0], [1]], [2, 3], 2, 0, 4)
    _check_extend([0, 0, 0], [2 ** 31 - 1, 2 ** 31 - 1, 1], [[-1], [-1], [-1]], [0, 1], 2, 4, 4)
    # a stack height beyond the stack, and below it
    t, f = _i32([[-1]]), _i32([0, 1])
    assert paged_extend(_i32([0]), _i32([1]), t, f, _i32([7]), 1, 4)[4].item() == 1 and t.item() == 1
    assert paged_extend(_i32([0]), _i32([1]), t, f, _i32([-3]), 1, 4)[5].item() == 1


def test_extend_counts_pages_of_any_size():
    big = 2 ** 31 - 1
    _check_extend([2 ** 30, 5, big, 0, big, 1], [3, -1, -1, 1, 1, big - 1], [[4], [3], [5], [-1], [1], [0]], [7, 6, 2, -1, -1, -1, -1, -1], 3, 5, big)


def test_extend_places_rows_by_one_launch_or_two():
    """Around the sizes at which a second launch begins, for few requests and for many."""
    for B, sums in ((3, (511, 512, 513)), (128, (513,)), (129, (2047, 2048, 2049)), (1024, (2049,)), (1025, (4096, 4097))):
        for total in sums:
            new = [total // B + (b < total % B) for b in range(B)]
            width = max(new) // 16 + 3
            _check_extend([b % 33 for b in range(B)], new, [[b * width + c for c in range(width)] for b in range(B)],
                          list(range(B * width, 2 * B * width)) + [-1] * (B * width), B * width, total, 16)


def test_extend_reads_a_table_that_is_a_slice():
    big = torch.full((6, 10), -5, dtype=torch.int32, device=DEV)
    view = big[1:5, 2:6]
    view[:] = -1
    out = paged_extend(_i32([0] * 4), _i32([3, 0, 9, 1]), view, _i32(list(range(8))), _i32([8]), 13, 4)
    assert out[5].tolist() == [0] * 4 and view.tolist() == [[7, -1, -1, -1], [-1] * 4, [6, 5, 4, -1], [3, -1, -1, -1]]
    big[1:5, 2:6] = -5
    assert bool((big == -5).all())


# ------------------------------------------------------------------------------------ paged_write
def _rot64(x, cos, sin):
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    h = x.shape[-1] // 2
    return torch.cat((x[..., :h] * c[..., :h] - x[..., h:] * s[..., :h], x[..., h:] * c[..., h:] + x[..., :h] * s[..., h:]), -1)


def _angles(T, dim, g):
    a = torch.rand(T, dim, generator=g, device=DEV) * 6.28
    return a.cos().to(torch.bfloat16), a.sin().to(torch.bfloat16)


@pytest.mark.parametrize("T, heads, dim, ps, layout, rope", [
    (1, 1, 32, 1, "plain", True), (7, 3, 64, 5, "plain", True), (130, 8, 128, 16, "fused", True), (33, 2, 256, 64, "heads first", True),
    (50, 4, 96, 24, "odd", True), (50, 4, 96, 24, "plain", False), (9, 2, 160, 7, "odd", False), (1000, 4, 64, 16, "one row for all", True)])
def test_write_puts_rows_into_their_slots(T, heads, dim, ps, layout, rope):
    g = _gen(T + dim)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)
    if layout == "fused":                        # column slices of a projection
        y = rnd(T, 2 * heads * dim + 64)
        k, v = y[:, 64:64 + heads * dim].view(T, heads, dim), y[:, 64 + heads * dim:].view(T, heads, dim)
    elif layout == "heads first":                # as a contiguous cache keeps them
        k, v = rnd(heads, T, dim).transpose(0, 1), rnd(heads, T, dim).transpose(0, 1)
    elif layout == "odd":                        # rows that begin at no 16-byte boundary
        k, v = rnd(T, heads * dim + 3)[:, 1:1 + heads * dim].view(T, heads, dim), rnd(T, heads, dim)
    elif layout == "one row for all":
        k, v = rnd(1, heads, dim).expand(T, heads, dim), rnd(1, heads, dim).expand(T, heads, dim)
    else:
        k, v = rnd(T, heads, dim), rnd(T, heads, dim)
    pages = -(-T // ps) + 2
    slots = torch.randperm(pages * ps, generator=g, device=DEV)[:T]
    slots[::5] = torch.tensor([-1, pages * ps, -2 ** 40, 2 ** 40], device=DEV).repeat(T)[: slots[::5].numel()]
    cos, sin = _angles(T, dim, g) if rope else (None, None)
    kp, vp = rnd(pages, heads, ps, dim), rnd(pages, heads, ps, dim)
    want_k, want_v = kp.double(), vp.double()
    rows = ((slots >= 0) & (slots < pages * ps)).nonzero()[:, 0]
    s = slots[rows]
    want_k[s // ps, :, s % ps] = _rot64(k, cos, sin)[rows] if rope else k.double()[rows]
    want_v[s // ps, :, s % ps] = v.double()[rows]
    before = kp.clone()
    paged_write(k, v, slots, kp, vp, cos, sin)
    assert torch.equal(vp.double(), want_v)
    touched = torch.zeros_like(kp, dtype=torch.bool)
    touched[s // ps, :, s % ps] = True
    assert torch.equal(kp[~touched], before[~touched])
    # two float32 products and their sum, then one rounding: 2^-8 of the result and 3 * 2^-24 of the products' magnitudes (at most 2 |k|max)
    assert bool(((kp.double() - want_k).abs() <= 2.0 ** -8 * want_k.abs() + 3 * 2.0 ** -24 * 2 * k.abs().max().double()).all())


@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("slot", [0, 9, 34])
def test_write_of_a_single_row(slot, odd):
    g = _gen(slot)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)
    k, v = (rnd(1, 3 * 64 + 2)[:, odd:odd + 192].view(1, 3, 64) for _ in range(2))
    cos, sin = _angles(1, 64, g)
    kp, vp = rnd(5, 3, 7, 64), rnd(5, 3, 7, 64)
    want_k, want_v, before = kp.double(), vp.clone(), kp.clone()
    want_k[slot // 7, :, slot % 7] = _rot64(k, cos, sin)[0]
    want_v[slot // 7, :, slot % 7] = v[0]
    paged_write(k, v, torch.tensor([slot], device=DEV), kp, vp, cos, sin)
    assert torch.equal(vp, want_v) and int((kp != before).any(-1).sum()) == 3
    # as above: one rounding of the result, three of products and their sum
    assert bool(((kp.double() - want_k).abs() <= 2.0 ** -8 * want_k.abs() + 3 * 2.0 ** -24 * 2 * k.abs().max().double()).all())


# ------------------------------------------------------------------------------------ paged_attn_decode
def _attend64(q, table, requests, positions, kp, vp, scale, cos, sin):
    """Row by row in float64: (out, magnitude of the weighted sum, largest magnitude of a score) of every row and head."""
    T, hq, dim = q.shape
    P, hk, ps, _ = kp.shape
    out, mag, big = (torch.zeros(T, hq, dim, dtype=torch.float64, device=DEV) for _ in range(3))
    qr = _rot64(q, cos, sin) if cos is not None else q.double()
    for t in range(T):
        b, p = int(requests[t]), int(positions[t])
        if not 0 <= b < table.shape[0] or p < 0:
            continue
        n = min(p + 1, table.shape[1] * ps)
        pages = table[b, :-(-n // ps)].long()
        real = ((pages >= 0) & (pages < P)).repeat_interleave(ps)[:n]
        if not bool(real.any()):
            continue
        k = kp[pages.clamp(0, P - 1)].transpose(0, 1).flatten(1, 2)[:, :n][:, real].double()
        v = vp[pages.clamp(0, P - 1)].transpose(0, 1).flatten(1, 2)[:, :n][:, real].double()
        k, v = k.repeat_interleave(hq // hk, 0), v.repeat_interleave(hq // hk, 0)
        s = torch.einsum("hd,hnd->hn", qr[t], k) * scale
        w = torch.softmax(s, -1)
        out[t] = torch.einsum("hn,hnd->hd", w, v)
        mag[t] = torch.einsum("hn,hnd->hd", w, v.abs())
        big[t] = (torch.einsum("hd,hnd->hn", qr[t].abs(), k.abs()).amax(-1) * abs(scale))[:, None]
    return out.view(T, -1), mag.view(T, -1), big.view(T, -1)


def _attn_case(T, hq, hk, dim, ps, lengths, seed, spare=3, spread=1.0):
    g = _gen(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)
    counts = [-(-max(n, 0) // ps) for n in lengths]
    width = max(max(counts), 1) + 1
    order = torch.randperm(sum(counts) + spare, generator=g, device=DEV).to(torch.int32)
    table = torch.full((T, width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    pages = order.numel()
    y = rnd(T, (hq + 2 * hk) * dim + 8)
    q = (y[:, :hq * dim] * spread).view(T, hq, dim)
    cos, sin = _angles(T, dim, g)
    requests = _i32([b if n > 0 else -1 for b, n in enumerate(lengths)])
    return dict(q=q, block_table=table, requests=requests, positions=torch.tensor(lengths, device=DEV) - 1, k_pages=rnd(pages, hk, ps, dim),
                v_pages=rnd(pages, hk, ps, dim), scale=1.0 / math.sqrt(dim), cos=cos, sin=sin)


def _check_attn(c):
    got = paged_attn_decode(**c)
    want, mag, big = _attend64(*c.values())
    n = int(c["positions"].max()) + 1
    dim = c["q"].shape[2]
    # One rounding of the result (2^-8 of it).  A score is a float32 sum of `dim` products of a rotated query, itself held to 2^-16 (two
    # bfloat16 parts) by two roundings in float32, with a key: off by (dim 2^-24 + 2^-16 + 2^-22) of its products' magnitudes; an error e of the
    # scores changes a probability by 2 e.  Probabilities are held to 2^-16 and expf to 2^-22 of a score's magnitude at most; sums of n terms are
    # float32, joined from pieces of at most n.
    e = 2 * big * (dim * 2.0 ** -24 + 2.0 ** -16 + 2.0 ** -21) + 2.0 ** -16 + 2 * min(n, 4096) * 2.0 ** -24 + 2.0 ** -20
    bound = 2.0 ** -8 * (want.abs() + mag * e) + mag * e
    assert got.dtype == torch.bfloat16 and got.shape == want.shape
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-30)).max())
    return got


@pytest.mark.parametrize("hq, hk, dim, ps", [(4, 4, 64, 16), (8, 2, 128, 64), (6, 2, 96, 24), (16, 1, 128, 1), (12, 1, 32, 7), (4, 2, 256, 100), (32, 32, 128, 64),
                                             (5, 5, 160, 16), (3, 1, 192, 8), (2, 2, 224, 33), (40, 2, 64, 16)])
@pytest.mark.parametrize("lengths", [[1], [0], [2, 0, 17, 1], [15, 16, 17, 31, 32, 33, 63, 64, 65], [700, 3, 129, 0, 255]], ids=str)
def test_attention_over_pages(hq, hk, dim, ps, lengths):
    c = _attn_case(len(lengths), hq, hk, dim, ps, lengths, seed=hq + dim + len(lengths))
    got = _check_attn(c)
    for t, n in enumerate(lengths):
        assert n > 0 or bool((got[t] == 0).all())
    again = paged_attn_decode(**c)
    assert torch.equal(got, again)                                   # sums in a fixed order
    _check_attn({**c, "cos": None, "sin": None})


@pytest.mark.parametrize("lengths, hq, hk, dim, ps", [([20000], 4, 1, 128, 24), ([9000, 40, 1, 3000], 8, 8, 64, 16), ([4097] * 3, 32, 8, 128, 64),
                                                      ([70] * 150, 8, 2, 64, 16), ([1] * 300, 4, 4, 32, 8), ([30000, 5], 16, 16, 128, 256)])
def test_attention_split_over_long_caches_and_many_rows(lengths, hq, hk, dim, ps):
    _check_attn(_attn_case(len(lengths), hq, hk, dim, ps, lengths, seed=len(lengths)))


@pytest.mark.parametrize("T", [1024, 1025, 2100])
def test_attention_of_more_rows_than_one_launch_takes(T):
    """Launches of up to 1024 rows share the workspace, one behind the other; rows at their ends with and without positions."""
    lengths = [(t * 37) % 91 for t in range(T)]
    lengths[1022:1026] = [300, 0, 300, 0][:T - 1022]
    c = _attn_case(T, 2, 1, 32, 16, lengths, seed=T)
    got = _check_attn(c)
    for t in (0, 1, 1023, T - 1):                                     # by itself: the same but for the order of sums
        one = {**c, **{n: c[n][t:t + 1].contiguous() for n in ("q", "requests", "positions", "cos", "sin")}}
        assert float((got[t].double() - _check_attn(one)[0].double()).abs().max()) <= 2 * 2.0 ** -8 * float(got[t].double().abs().max())


def test_attention_over_a_table_so_wide_that_a_launch_takes_fewer_rows():
    """Places of 1024 rows as long as this table allows would not fit 31 bits: two launches for a thousand rows of two short requests."""
    c = _attn_case(2, 8, 8, 64, 64, [150, 97], seed=12)
    table = torch.full((2, 70000), -1, dtype=torch.int32, device=DEV)
    table[:, :c["block_table"].shape[1]] = c["block_table"]
    g = _gen(13)
    T = 1000
    c.update(q=torch.randn(T, 8, 64, generator=g, device=DEV).to(torch.bfloat16), block_table=table, requests=_i32([t % 2 for t in range(T)]),
             positions=torch.tensor([t % (150 if t % 2 == 0 else 97) for t in range(T)], device=DEV))
    c["cos"], c["sin"] = _angles(T, 64, g)
    _check_attn(c)


def test_attention_weights_that_one_position_takes():
    """Scores hundreds apart: the running maximum moves late, early, or not at all, and what it discards adds nothing."""
    for place in (0, 100, 299):
        c = _attn_case(2, 4, 2, 64, 16, [300, 300], seed=3, spread=12.0)
        c["cos"] = c["sin"] = None
        page, off = int(c["block_table"][0, place // 16]), place % 16
        c["k_pages"][page, :, off] = c["q"][0, ::2]
        _check_attn(c)


def test_attention_rows_of_one_request_and_rows_without_one():
    c = _attn_case(6, 8, 2, 64, 16, [90, 0, 40, 5, 0, 12], seed=9)
    # several rows of request 0 at different positions, a request beyond the table, a negative position, one beyond the table's width
    c["requests"] = _i32([0, 0, 0, 99, 2, 5])
    c["positions"] = torch.tensor([0, 40, 89, 3, -4, 10 ** 12], device=DEV)
    got = _check_attn(c)
    assert bool((got[3:5] == 0).all())
    # a table entry that is no page hides its positions; a row whose every entry is none is empty
    c["block_table"][0, 1], c["block_table"][2, :] = 10 ** 6, -1
    c["requests"], c["positions"] = _i32([0, 2, 0, 0, 2, 5]), torch.tensor([89, 39, 20, 3, 0, 11], device=DEV)
    got = _check_attn(c)
    assert bool((got[1] == 0).all()) and bool((got[4] == 0).all())


def test_attention_does_not_look_behind_the_row():
    """Whatever stands behind the row's position, in its last page or in pages that no table names, NaN included, has no part in it."""
    c = _attn_case(3, 4, 2, 128, 64, [65, 10, 128], seed=2)
    clean = paged_attn_decode(**c)
    used = torch.zeros_like(c["k_pages"], dtype=torch.bool)
    for b, n in enumerate([65, 10, 128]):
        for i in range(n):
            used[c["block_table"][b, i // 64], :, i % 64] = True
    for pages in (c["k_pages"], c["v_pages"]):
        pages[~used] = float("nan")
    assert torch.equal(paged_attn_decode(**c), clean)


@pytest.mark.parametrize("lengths", [[40, 33, 70, 5], [900, 2000, 64, 1500]], ids=str)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_row_that_sees_no_number_leaves_the_others_alone(lengths, value):
    c = _attn_case(4, 8, 2, 64, 16, lengths, seed=5)
    clean = paged_attn_decode(**c)
    page = int(c["block_table"][int(c["requests"][1]), 1])
    c["k_pages"][page, :, 3], c["v_pages"][page, :, 4] = value, value
    got = paged_attn_decode(**c)
    assert bool(torch.isnan(got[1]).any())
    for t in (0, 2, 3):
        assert torch.equal(got[t], clean[t])


def test_attention_takes_strided_queries():
    c = _attn_case(5, 4, 4, 64, 16, [30, 1, 64, 7, 19], seed=4)
    want = paged_attn_decode(**c)
    q = torch.zeros(5, 4, 67, dtype=torch.bfloat16, device=DEV)
    q[..., 1:65] = c["q"]                                             # heads 67 apart, at no 16-byte boundary
    assert torch.equal(paged_attn_decode(**{**c, "q": q[..., 1:65]}), want)
    wide = torch.zeros(5, 80, dtype=torch.bfloat16, device=DEV)
    wide2 = wide.clone()
    wide[:, 3:67], wide2[:, 3:67] = c["cos"], c["sin"]
    assert torch.equal(paged_attn_decode(**{**c, "cos": wide[:, 3:67], "sin": wide2[:, 3:67]}), want)


# ------------------------------------------------------------------------------------ multi_delta_forward
def _delta64(x, y, packed, ids):
    """y + U (V x) in float64 from the unpacked codes, and how far off the operands' fixed point may put it.

    x vs is held, for each row, rank group and 128 columns, to half a unit of a grid with at least 2^14 units to the largest of the 128 (less
    0.4 %): off by 1.004 2^-15 of it.  h is held the same way for each row and group of 128 ranks.  A code less its zero-point is at most 15."""
    out, off, mag = y.double().clone(), torch.zeros(y.shape, dtype=torch.float64, device=DEV), torch.zeros(y.shape, dtype=torch.float64, device=DEV)
    for t, d in enumerate(ids):
        if not 0 <= d < len(packed):
            continue
        p = {k: v.to(DEV).double() for k, v in packed[d].items()}
        U = (p["U_codes"] - p["U_zero"].repeat_interleave(128, 1)) * p["U_scale"].repeat_interleave(128, 1)
        V = (p["Vt_codes"] - p["Vt_zero"].repeat_interleave(128, 0)) * p["Vt_scale"].repeat_interleave(128, 0)
        h = V @ x[t].double()
        out[t] += U @ h
        largest = (x[t].double() * p["Vt_scale"]).abs().view(p["Vt_scale"].shape[0], -1, 128).amax(-1)      # (rank group, 128 columns)
        habs = 15 * 128 * largest.sum(-1)                                                                 # of any rank of the group
        hmax = h.abs().view(-1, 128).amax(-1)
        off[t] = 1.004 * 2.0 ** -15 * (15 * 128 * p["U_scale"]) @ (habs + hmax)
        mag[t] = (15 * 128 * p["U_scale"]) @ habs
    return out, off, mag


def _check_delta(M, N, ranks, ids, seed):
    packed = [synth.random_packed(M, N, r, seed=seed + i, device=DEV) for i, r in enumerate(ranks)]
    bank = bank_deltas([kernels.pack_int4(p) for p in packed])
    g = _gen(seed)
    T = len(ids)
    x = torch.randn(T, N, generator=g, device=DEV).to(torch.bfloat16)
    y = torch.randn(T, M, generator=g, device=DEV).to(torch.bfloat16)
    y *= 0.02                                                          # the delta is a visible part of the result
    got = multi_delta_forward(x, y, bank, _i32(ids))
    want, off, mag = _delta64(x, y, packed, ids)
    # integers are exact; what they come to is added in float32 (N / 128 terms and the rank groups', none more than mag), one rounding at the end
    e = off + mag * (N / 128 + 16) * 2.0 ** -24
    off = (got.double() - want).abs()
    assert bool((off <= 2.0 ** -8 * (want.abs() + e) + e).all()), float((off / (2.0 ** -8 * want.abs() + e).clamp(min=1e-30)).max())
    # the typical error is that of the last rounding alone: a uniform error of half a step has a root mean square of 2^-8 / sqrt(3) of a value
    # at the lower end of its binade, and the roundings on the way add a random walk far below it
    rms = lambda v: float(v.square().mean().sqrt())
    assert rms(got.double() - want) <= 2.0 ** -8 / math.sqrt(3) * rms(want) * 1.1
    for t, d in enumerate(ids):
        if not 0 <= d < len(ranks):
            assert torch.equal(got[t], y[t])
    assert torch.equal(got, multi_delta_forward(x, y, bank, _i32(ids)))
    return x, y, bank, got


@pytest.mark.parametrize("M, N, ranks, ids", [
    (1, 128, [128], [0]), (7, 128, [256, 128], [1, 0, -1, 1]), (1000, 2048, [384, 128], [0, 1, 1]), (300, 256, [128, 640, 256], [2, 2, 0, 1, 5, 2 ** 31 - 1, -2 ** 31]),
    (129, 1152, [2048], [0, 0]), (256, 384, [128] * 5, [i % 5 for i in range(33)]), (520, 512, [256, 384], [0] * 128), (64, 11008, [128, 256], [1, 0, 1]),
    (400, 256, [128] * 40, list(range(40)) + [-1] * 3), (2048, 640, [512, 128, 1024], [(i * 7) % 4 - 1 for i in range(127)]), (16, 128, [128], [-1, -1])], ids=lambda v: str(v)[:40])
def test_each_row_gets_its_own_delta(M, N, ranks, ids):
    _check_delta(M, N, ranks, ids, seed=M + N)


@pytest.mark.parametrize("K", [127, 128, 130, 300])
def test_banks_of_many_deltas(K):
    """Up to 127 deltas their first rank groups are kept beside the rows, beyond that they are looked up."""
    T = 128
    ids = [(t * 7) % K for t in range(T)]
    ids[5:9] = [K - 1, 0, K, -1]
    ids[60:70] = [K - 1] * 10
    _check_delta(24, 256, [128 * (1 + i % 2) for i in range(K)], ids, seed=K)


def _grid(m):
    """The step of the fixed point in which values of magnitude up to m are held: 2^-14 of the power of two at or below 1.004 m."""
    return torch.exp2(torch.floor(torch.log2((1.004 * m).clamp(min=2.0 ** -100))) - 14)


def _delta_spread(x, packed):
    """(U^ V^^T x, covariance (rows, M, M) of what the two fixed-point roundings put a row's outputs off) in float64 for rows of one delta.

    A value rounded to a grid of step s is off by s / sqrt(12), independently of the others.  x vs of each column, rank group and row is rounded on the
    grid of its 128 columns, h of each rank and row on that of its 128 ranks; the codes carry both to the outputs: U V e and U f."""
    p = {k: v.to(DEV).double() for k, v in packed.items()}
    x, M = x.double(), p["U_codes"].shape[0]
    out = torch.zeros(x.shape[0], M, dtype=torch.float64, device=DEV)
    cov = torch.zeros(x.shape[0], M, M, dtype=torch.float64, device=DEV)
    for g in range(p["Vt_scale"].shape[0]):
        ranks = slice(128 * g, 128 * g + 128)
        U = (p["U_codes"][:, ranks] - p["U_zero"][:, g:g + 1]) * p["U_scale"][:, g:g + 1]
        V = p["Vt_codes"][ranks] - p["Vt_zero"][g]
        xs = x * p["Vt_scale"][g]
        h = xs @ V.t()
        out += h @ U.t()
        step = _grid(xs.abs().view(x.shape[0], -1, 128).amax(-1)).repeat_interleave(128, 1)
        step_h = _grid(h.abs().amax(-1))
        ranks_cov = torch.einsum("kn,tn,jn->tkj", V, step ** 2 / 12, V) + step_h[:, None, None] ** 2 / 12 * torch.eye(128, dtype=torch.float64, device=DEV)
        cov += U @ ranks_cov @ U.t()
    return out, cov


@pytest.mark.parametrize("T", [3, 8, 40])
@pytest.mark.parametrize("M, N, r, kind", [(512, 1024, 256, "normal"), (512, 1024, 256, "columns"), (300, 2176, 384, "one column"), (512, 1024, 256, "ranks"), (264, 4096, 128, "all"),
                                           (128, 128, 128, "normal")])
def test_deltas_are_as_exact_as_their_fixed_point(M, N, r, kind, T):
    """The shared term takes away what the delta rounds to, so the output shows what is left of it some nine bits finer.

    With columns of x that are a hundred to a thousand times larger than the others, and ranks of V^ whose h lies apart by more than two decades."""
    packed = synth.random_packed(M, N, r, seed=M + N + r, device=DEV)
    g = _gen(T + N)
    x = torch.randn(T, N, generator=g, device=DEV)
    if kind in ("columns", "all"):
        x[:, 7::101] *= 100.0
        x[:, 50::499] *= 1000.0
    if kind == "one column":
        x[:, 1000] = 1000.0
    x = x.to(torch.bfloat16)
    if kind in ("ranks", "all"):
        # a third of the ranks hardly look at x and one looks just where that of the first row is: h from near nothing to as large as it can be
        packed["Vt_zero"] = packed["Vt_zero"].clamp(max=14)
        rank = torch.arange(r, device=DEV)[:, None]
        little = packed["Vt_zero"].long().repeat_interleave(128, 0) + torch.randint(0, 2, (r, N), generator=g, device=DEV)
        codes = torch.where(rank % 3 == 0, little, packed["Vt_codes"].long())
        packed["Vt_codes"] = torch.where(rank % 128 == 5, torch.where(x[0] > 0, 15, 0), codes).to(torch.uint8)
    want, cov = _delta_spread(x, packed)
    y = (-want).to(torch.bfloat16)
    left = want + y.double()
    got = multi_delta_forward(x, y, bank_deltas([kernels.pack_int4(packed)]), _i32([0] * T)).double()
    # What else is rounded: the output (a uniform error of a step of bfloat16 of what is left, with its error) and float32 sums of N / 128 and r / 128
    # terms.  Codes less their zero-points do not average to zero, so the outputs of a row share most of their error: its root mean square is
    # that of about one number a rank group.  So it is measured by its covariance C: off^T C^-1 off has the mean M and, for sums of many roundings, the
    # deviation sqrt(2 M); over the rows, which err independently, six deviations are allowed.  x vs has 16 significant bits, so those in the grid's
    # top binade can only be off by nothing or half a step, evenly: step^2 / 8 instead of step^2 / 12.  Of 128 normal values whose largest is 2.7
    # deviations at most one in six lies there (above 1.35): 1 + 0.5 / 6 = 1.1 of the mean.  A float64 model of the two roundings gives 1.0 to 1.2; with
    # one bit less in x vs or in h it gives 1.3 to 3.1, 1.6 to 1.9 and more for normal values, and 2.4 to 3.4 with one bit less in both.
    variance = cov.diagonal(dim1=1, dim2=2)
    ulp = torch.exp2(torch.floor(torch.log2(torch.maximum(left.abs(), variance.sqrt()))) - 7)
    other = ulp ** 2 / 12 + ((N / 128 + r / 128 + 4) * 2.0 ** -24 * want.abs().amax(1, keepdim=True)) ** 2
    off = got - left
    solved = torch.linalg.solve_triangular(torch.linalg.cholesky(cov + torch.diag_embed(other)), off[..., None], upper=False)[..., 0]
    size = float(solved.square().mean())
    assert size <= 1.1 * (1 + 6 * math.sqrt(2 / (M * T))), size
    assert bool((off.abs() <= 7 * (variance + other).sqrt()).all())


def test_rows_of_one_delta_match_the_single_delta_path():
    """The factored kernel on the rows of each delta: both are within the factored path's tolerance of each other."""
    M, N, ranks, ids = 512, 1024, [256, 512], [0, 1, 1, 0, 1, 0, 0]
    packed = [synth.random_packed(M, N, r, seed=50 + i, device=DEV) for i, r in enumerate(ranks)]
    forms = [kernels.pack_int4(p) for p in packed]
    g = _gen(8)
    x, y = (torch.randn(7, n, generator=g, device=DEV).to(torch.bfloat16) for n in (N, M))
    got = multi_delta_forward(x, y, bank_deltas(forms), _i32(ids))
    for d, f in enumerate(forms):
        rows = torch.tensor([t for t, i in enumerate(ids) if i == d], device=DEV)
        want = kernels.decode_forward_packed(x[rows].contiguous(), y[rows].contiguous(), f)
        assert float((got[rows].float() - want.float()).norm() / want.float().norm()) < 1e-2


def test_values_that_are_no_numbers_stay_in_their_row():
    """NaN, infinities, zeros and tiny values in rows of one delta: each row gives what it gives alone."""
    forms = [kernels.pack_int4(synth.random_packed(200, 384, 256, seed=5, device=DEV))]
    bank = bank_deltas(forms)
    g = _gen(4)
    x = torch.randn(9, 384, generator=g, device=DEV).to(torch.bfloat16)
    y = torch.zeros(9, 200, dtype=torch.bfloat16, device=DEV)
    x[1, 7], x[3, 300], x[4, 1], x[5], x[6] = float("nan"), float("inf"), float("-inf"), 0.0, 1e-30
    got = multi_delta_forward(x, y, bank, _i32([0] * 9))
    for t in range(9):
        alone = multi_delta_forward(x[t:t + 1].contiguous(), y[:1], bank, _i32([0]))
        assert torch.equal(got[t].nan_to_num(7.0), alone[0].nan_to_num(7.0)) and torch.equal(torch.isnan(got[t]), torch.isnan(alone[0]))
    assert not bool(torch.isfinite(got[[1, 3, 4]]).any()) and bool((got[5] == 0).all()) and bool(torch.isfinite(got[[0, 2, 5, 6, 7, 8]]).all())


def test_the_output_may_be_the_shared_term_itself():
    import ctypes

    from ade_b200 import _lib

    x, y, bank, want = _check_delta(129, 256, [256, 128], [0, 1, -1, 0], seed=31)
    lib, ids = _lib.load(), _i32([0, 1, -1, 0])
    b = _lib.AdeDeltaBank(*[bank[k].data_ptr() for k in kernels.BANK_KEYS], 129, 256, bank["uq"].shape[0], 2)
    work = torch.empty(lib.ade_b200_multi_delta_workspace_bytes(4, 256), dtype=torch.uint8, device=DEV)
    out = y.clone()
    assert lib.ade_b200_multi_delta(x.data_ptr(), out.data_ptr(), ctypes.byref(b), ids.data_ptr(), out.data_ptr(), work.data_ptr(), work.numel(), 4,
                                    torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, want)


def test_delta_ids_are_read_when_the_graph_runs():
    x, y, bank, _ = _check_delta(384, 512, [128, 256, 384], [0, 1, 2, -1, 0], seed=70)
    ids = _i32([0, 1, 2, -1, 0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        multi_delta_forward(x, y, bank, ids)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = multi_delta_forward(x, y, bank, ids)
    for new in ([2, 2, 2, 2, 2], [-1] * 5, [0, 1, 0, 1, 9]):
        ids.copy_(_i32(new))
        graph.replay()
        assert torch.equal(out, multi_delta_forward(x, y, bank, _i32(new)))


# ------------------------------------------------------------------------------------ token_logprobs
def _logprobs64(x, tokens, top):
    x = x.double()
    m = x.amax(-1, keepdim=True)
    z = x - m
    e = z.exp()
    ls = e.sum(-1).log()
    entropy = ls - torch.where(e > 0, e * z, 0.0).sum(-1) / e.sum(-1)
    best, where = torch.sort(x, dim=-1, descending=True, stable=True)
    logp = z - ls[:, None]
    given = torch.where(tokens >= 0, logp.gather(1, tokens.clamp(0, x.shape[1] - 1)[:, None])[:, 0], 0.0)
    given = torch.where(tokens >= x.shape[1], float("nan"), given)
    return given, entropy, (best - m)[:, :top] - ls[:, None], where[:, :top]


def _same(got, want, tol):
    assert got.shape == want.shape
    finite = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.double()[~finite & ~torch.isnan(want)], want[~finite & ~torch.isnan(want)])
    off = (got.double() - want).abs()[finite]
    assert bool((off <= (tol if not torch.is_tensor(tol) else tol[finite])).all()), float(off.max())


def _check_logprobs(x, tokens, top):
    logp, entropy, tl, tt = token_logprobs(x, tokens, top)
    w_logp, w_entropy, w_tl, w_tt = _logprobs64(x, tokens, top)
    assert torch.equal(tt, w_tt)
    V = x.shape[1]
    # The sum of V positive terms, each expf of a float32 difference (2 units and the difference's own rounding, up to 100 2^-24 where a term
    # still counts), in partial sums of at most V / 256 + 9 terms: relative 2^-24 (104 + V / 256 + 9) at most; log and the subtractions add
    # 2^-23 of their results.
    e = 2.0 ** -24 * (113 + V / 256)
    step = lambda w: e + 2.0 ** -22 * w.nan_to_num(0, 0, 0).abs()
    _same(logp, w_logp, step(w_logp))
    _same(tl, w_tl, step(w_tl))
    # the entropy weighs differences of up to log V + H with those sums' errors
    _same(entropy, w_entropy, 3 * e * (1 + 2 * math.log(V) + w_entropy.nan_to_num(0).abs()))


@pytest.mark.parametrize("rows, V, dtype, top", [(1, 1, torch.float32, 1), (3, 5, torch.bfloat16, 5), (2, 31, torch.float16, 31), (1, 32, torch.float32, 32),
                                                 (4, 255, torch.bfloat16, 7), (5, 256, torch.float32, 0), (7, 1003, torch.float16, 32), (64, 32000, torch.bfloat16, 5),
                                                 (3, 50257, torch.float32, 20), (2, 152064, torch.bfloat16, 32), (1, 257001, torch.float32, 1), (300, 2048, torch.bfloat16, 3),
                                                 (10, 532, torch.bfloat16, 20), (9, 517, torch.float32, 32), (5, 1025, torch.float16, 32)])
def test_log_probabilities(rows, V, dtype, top):
    g = _gen(rows + V)
    x = (torch.randn(rows, V, generator=g, device=DEV) * 3).to(dtype)
    tokens = torch.randint(0, V, (rows,), generator=g, device=DEV)
    tokens[rows // 2] = -1 if rows > 1 else tokens[0]
    _check_logprobs(x, tokens, top)
    _check_logprobs(x * 20, tokens, top)                              # a few tokens hold all of the probability


@pytest.mark.parametrize("V", [40, 3000, 33001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits_come_in_the_order_of_their_tokens(V, dtype):
    g = _gen(V)
    flat = torch.zeros(1, V, device=DEV)
    few = torch.randint(0, 3, (1, V), generator=g, device=DEV).float()
    signs = torch.where(torch.rand(1, V, generator=g, device=DEV) < 0.5, -0.0, 0.0)
    stairs = (torch.arange(V, device=DEV) // 7).float()[None] / 64
    one_lane = torch.randn(1, V, generator=g, device=DEV)
    one_lane[0, 5::256] += 50                                         # the largest all in places that one thread may read
    for x in (flat, few, signs, stairs, stairs.flip(-1), one_lane):
        _check_logprobs(x.to(dtype), torch.tensor([V // 2], device=DEV), 32)


def test_infinities_and_nan():
    inf, nan = float("inf"), float("nan")
    V = 777
    g = _gen(1)
    x = torch.randn(9, V, generator=g, device=DEV)
    x[0, :] = -inf                                                    # nothing is possible
    x[1, 1:] = -inf                                                   # one token is
    x[2, 300] = inf
    x[3, 500] = nan
    x[4, ::2] = -inf
    x[5, :] = torch.finfo(torch.float32).min                          # masked with the lowest value, all of them
    x[6, 10:] = torch.finfo(torch.float32).min
    x[7, 5], x[7, 9] = nan, nan
    tokens = torch.tensor([3, 0, 300, 4, 0, 9, 2, -5, V], device=DEV)
    _check_logprobs(x, tokens, 8)
    for dtype in (torch.bfloat16, torch.float16):                     # the lowest value of each type beside -inf
        y = x.clamp(min=torch.finfo(dtype).min).to(dtype)
        y[6, 20:] = -inf
        _check_logprobs(y, tokens, 8)
    logp, entropy, _, tt = token_logprobs(x, tokens, 2)
    assert entropy[1] == 0 and logp[1] == 0 and logp[4] == -inf and logp[7] == 0 and bool(torch.isnan(logp[8]))
    assert tt[0].tolist() == [0, 1] and tt[7].tolist() == [5, 9]


def test_logits_with_strides_and_without_tokens():
    g = _gen(2)
    big = torch.randn(6, 2003, generator=g, device=DEV).to(torch.bfloat16)
    tokens = torch.randint(0, 1001, (6,), generator=g, device=DEV)
    _check_logprobs(big[:, 1:1002], tokens, 4)                        # rows at no 16-byte boundary
    _check_logprobs(big[::2, 7:], tokens[:3].contiguous(), 4)
    _check_logprobs(big[:1].expand(6, 2003), tokens, 4)
    logp, entropy, tl, tt = token_logprobs(big)
    assert logp.numel() == 0 and entropy.shape == (6,) and tl.shape == tt.shape == (6, 0)
    assert token_logprobs(big[:0], tokens[:0], 3)[2].shape == (0, 3)


def test_a_row_of_all_31_bits():
    """The places behind the row's last whole piece, and the threads that have none there, are counted beyond 31 bits."""
    V = 2 ** 31 - 1
    x = torch.zeros(1, V, dtype=torch.bfloat16, device=DEV)
    x[0, V - 1], x[0, V - 2], x[0, 0] = 3.0, 2.0, 1.0
    logp, entropy, tl, tt = token_logprobs(x, torch.tensor([V - 1], device=DEV), 3)
    assert tt.tolist() == [[V - 1, V - 2, 0]]
    # a thread adds V / 256 terms in float32, each sum off by 2^-24 of it at most: e^(+-tol) of the sum of exp
    tol = 2.0 ** -24 * (113 + V / 256)
    want = 3.0 - math.log(math.exp(3.0) + math.exp(2.0) + math.exp(1.0) + V - 3)
    assert abs(logp.item() - want) <= tol and (tl[0] - tl[0, 0]).tolist() == pytest.approx([0.0, -1.0, -2.0], abs=2.0 ** -19)
    assert tl[0, 0] == logp[0] and bool(torch.isfinite(entropy).all())


# ------------------------------------------------------------------------------------ refusals, streams, graphs
def test_arguments_are_refused_with_a_reason():
    g = _gen(0)
    bf = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)
    i64 = lambda *s: torch.zeros(*s, dtype=torch.int64, device=DEV)
    kp, q = bf(4, 2, 8, 64), bf(3, 4, 64)
    write = lambda **kw: paged_write(**{**dict(k=bf(3, 2, 64), v=bf(3, 2, 64), slots=i64(3), k_pages=kp, v_pages=kp.clone()), **kw})
    attn = lambda **kw: paged_attn_decode(**{**dict(q=q, block_table=i32(2, 4), requests=i32(3), positions=i64(3), k_pages=kp, v_pages=kp, scale=1.0), **kw})
    extend = lambda **kw: paged_extend(**{**dict(lengths=i32(2), new_tokens=i32(2), block_table=i32(2, 3), free_pages=i32(4), free_count=i32(1), total=2, page_size=8), **kw})
    bank = bank_deltas([kernels.pack_int4(synth.random_packed(32, 128, 128, 1, DEV))])
    delta = lambda **kw: multi_delta_forward(**{**dict(x=bf(3, 128), y_dense=bf(3, 32), bank=bank, ids=i32(3)), **kw})
    refused = [
        lambda: write(k=bf(3, 2, 64).float()), lambda: write(k=bf(3, 64, 2).transpose(1, 2)), lambda: write(slots=i32(3)), lambda: write(slots=i64(4)),
        lambda: write(v_pages=bf(4, 2, 9, 64)), lambda: write(k_pages=kp.transpose(1, 2)), lambda: write(cos=bf(3, 64)), lambda: write(cos=bf(2, 64), sin=bf(2, 64)),
        lambda: write(k=bf(3, 2, 64).requires_grad_()), lambda: write(k=bf(3, 2, 64).cpu()),
        lambda: attn(q=bf(3, 3, 64)), lambda: attn(q=bf(3, 4, 32)), lambda: attn(requests=i64(3)), lambda: attn(positions=i32(3)), lambda: attn(block_table=i32(4, 2).t()),
        lambda: attn(q=bf(3, 4, 64).requires_grad_()), lambda: attn(q=q.half()), lambda: attn(sin=bf(3, 64)), lambda: attn(block_table=i32(1, 4).expand(2, 4)),
        lambda: extend(lengths=i64(2)), lambda: extend(new_tokens=i32(3)), lambda: extend(total=-1), lambda: extend(free_count=i32(2)), lambda: extend(page_size=-1),
        lambda: extend(block_table=i32(2, 6)[:, ::2]), lambda: extend(free_pages=i32(8)[::2]),
        lambda: delta(x=bf(3, 256)), lambda: delta(x=bf(3, 128).float()), lambda: delta(ids=i64(3)), lambda: delta(ids=i32(2)), lambda: delta(y_dense=bf(32, 3).t()),
        lambda: delta(bank={**bank, "uz": bank["uz"].int()}), lambda: delta(bank={**bank, "M": 31}), lambda: delta(x=bf(3, 128).requires_grad_()),
        lambda: delta(bank={**bank, "start": bank["start"][:1]}),
        lambda: token_logprobs(torch.zeros(2, 9, device=DEV, dtype=torch.float64)), lambda: token_logprobs(torch.zeros(9, device=DEV)),
        lambda: token_logprobs(torch.zeros(9, 2, device=DEV).t()), lambda: token_logprobs(torch.zeros(2, 9, device=DEV), i64(3)),
        lambda: token_logprobs(torch.zeros(2, 9, device=DEV), i32(2)), lambda: token_logprobs(torch.zeros(2, 9, device=DEV), None, 10),
        lambda: token_logprobs(torch.zeros(2, 90, device=DEV), None, 33), lambda: token_logprobs(torch.zeros(2, 9, device=DEV, requires_grad=True)),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
    with torch.no_grad():
        assert token_logprobs(torch.zeros(2, 9, device=DEV, requires_grad=True))[1].shape == (2,)
    from ade_b200._lib import AdeKernelError

    for call in (lambda: write(k=bf(3, 2, 48), v=bf(3, 2, 48), k_pages=bf(4, 2, 8, 48), v_pages=bf(4, 2, 8, 48)), lambda: extend(page_size=0),
                 lambda: delta(x=bf(129, 128), y_dense=bf(129, 32), ids=i32(129))):
        with pytest.raises(AdeKernelError, match="ADE_ERR_SHAPE"):
            call()


def test_no_rows_is_no_call():
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)
    kp = bf(4, 2, 8, 64)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    paged_write(bf(0, 2, 64), bf(0, 2, 64), none, kp, kp)
    assert paged_attn_decode(bf(0, 4, 64), _i32([[0]]), none.int(), none, kp, kp, 1.0).shape == (0, 256)
    bank = bank_deltas([kernels.pack_int4(synth.random_packed(32, 128, 128, 1, DEV))])
    assert multi_delta_forward(bf(0, 128), bf(0, 32), bank, none.int()).shape == (0, 32)


def _step(s):
    """One decode step of a layer as a serving loop runs it: room for a token each, the projection's delta, the cache, attention, log probabilities."""
    slots, positions, requests, _, _, status = paged_extend(s["lengths"], s["new"], s["table"], s["free"], s["count"], s["rows"], s["ps"], in_place=True)
    qkv = multi_delta_forward(s["x"], s["y"], s["bank"], s["ids"])
    hq, hk, dim = s["heads"]
    q, k, v = qkv[:, :hq * dim].view(-1, hq, dim), qkv[:, hq * dim:(hq + hk) * dim].view(-1, hk, dim), qkv[:, (hq + hk) * dim:].view(-1, hk, dim)
    cos, sin = s["cos"][positions], s["sin"][positions]
    paged_write(k, v, slots, s["kp"], s["vp"], cos, sin)
    ctx = paged_attn_decode(q, s["table"], requests, positions, s["kp"], s["vp"], dim ** -0.5, cos, sin)
    return (ctx, *token_logprobs(torch.nn.functional.linear(ctx, s["head"]), s["given"], 3), status, slots)


def _step_state(seed):
    g = _gen(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)
    hq, hk, dim, N, R, ps = 4, 2, 64, 256, 5, 4
    M = (hq + 2 * hk) * dim
    bank = bank_deltas([kernels.pack_int4(synth.random_packed(M, N, r, seed + r, DEV)) for r in (128, 256)])
    a = torch.rand(64, dim, generator=g, device=DEV) * 6.28
    return {"lengths": _i32([0] * R), "new": _i32([1] * R), "table": torch.full((R, 8), -1, dtype=torch.int32, device=DEV), "free": _i32(list(range(40))), "count": _i32([40]),
            "rows": R, "ps": ps, "x": rnd(R, N), "y": rnd(R, M), "bank": bank, "ids": _i32([0, 1, -1, 1, 0]), "heads": (hq, hk, dim), "cos": a.cos().to(torch.bfloat16),
            "sin": a.sin().to(torch.bfloat16), "kp": rnd(40, hk, ps, dim), "vp": rnd(40, hk, ps, dim), "head": rnd(99, hq * dim),
            "given": torch.arange(R, device=DEV)}


def test_a_step_of_all_operators_replayed_from_a_graph_and_on_another_stream():
    """Twelve steps in which requests rest, end and enter: eager on the current stream, eager on another one, and replayed from a graph."""
    runs = []
    for mode in ("eager", "stream", "graph"):
        s = _step_state(11)
        rng = random.Random(3)
        side = torch.cuda.Stream()
        graph = None
        if mode == "graph":
            spare = _step_state(12)                                   # lazy initialisation outside the capture
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                _step(spare)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = _step(s)
        got = []
        for i in range(12):
            s["new"].copy_(_i32([rng.choice([1, 1, 1, 0, -1]) for _ in range(5)]))
            s["x"].copy_(torch.randn(5, 256, generator=_gen(100 + i), device=DEV).to(torch.bfloat16))
            if mode == "graph":
                graph.replay()
            elif mode == "stream":
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    out = _step(s)
                torch.cuda.current_stream().wait_stream(side)
            else:
                out = _step(s)
            got.append([t.clone() for t in out] + [s["lengths"].clone(), s["table"].clone(), s["count"].clone(), s["kp"].clone(), s["vp"].clone()])
        runs.append(got)
        assert all(int(step[5].abs().sum()) == 0 for step in got)
    for a, b, c in zip(*runs):
        for x, y, z in zip(a, b, c):
            assert torch.equal(x.nan_to_num(7), y.nan_to_num(7)) and torch.equal(x.nan_to_num(7), z.nan_to_num(7))


def test_two_graphs_at_once_do_not_share_a_workspace():
    """Two captured attentions and deltas replayed side by side on two streams give what each gives alone."""
    c = [_attn_case(2, 8, 2, 128, 16, [3000, 2000], seed=s) for s in (1, 2)]
    packed = [synth.random_packed(2048, 2048, 512, seed=s, device=DEV) for s in (1, 2)]
    bank = bank_deltas([kernels.pack_int4(p) for p in packed])
    g = _gen(6)
    xs = [torch.randn(64, 2048, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    y, ids = torch.zeros(64, 2048, dtype=torch.bfloat16, device=DEV), _i32([i % 2 for i in range(64)])
    want = [(paged_attn_decode(**c[i]), multi_delta_forward(xs[i], y, bank, ids)) for i in range(2)]
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append((paged_attn_decode(**c[i]), multi_delta_forward(xs[i], y, bank, ids)))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for o in outs:
            for t in o:
                t.zero_()
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for w, o in zip(want, outs):
            assert torch.equal(w[0], o[0]) and torch.equal(w[1], o[1])
