"""A serving step over a batch of independent requests, operator by operator, as cases that can be timed and compared.

Five operators, in the order in which a step uses them:

  extend     pages of the key-value cache for new tokens: allocation from a stack of free pages, block tables, the slot, position
             and request of every row of the packed batch;
  write      keys (rotated to their positions) and values of new tokens into those pages;
  attend     attention of single rows over the pages of their requests;
  delta      the 4-bit deltas of many fine-tuned models beside one shared projection, each row with a delta of its own;
  logprobs   log probabilities of given tokens, entropy of the distribution, the likeliest alternatives.

`run` computes them in elementary torch operations, or, where `own` is set, makes the framework's calls.  Model sizes are those of the
7B and 13B LLaMA architectures (hidden 4096 / 5120, MLP 11008 / 13824, 32 / 40 heads of 128, vocabulary 32000) and of the small models and
ragged modules of the tests; grouped key-value heads, page sizes and batch sizes are generic.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
GROUP = 128                                    # ranks per quantisation group
NIBBLES = (0, 2, 4, 6, 1, 3, 5, 7)             # nibble i of a packed 32-bit word holds code NIBBLES[i] of its eight


def listed():
    return [
        # one decode step of 64 requests of up to 2000 tokens, a few of them idle, two finished and handing their pages back
        {"name": "extend_decode_64", "op": "extend", "requests": 64, "most": 2000, "fresh": 0, "page": 64},
        # prompts of 900 requests enter at once behind an odd number of running ones: 45 000 rows
        {"name": "extend_prompts_900", "op": "extend", "requests": 1001, "most": 700, "fresh": 100, "page": 16},
        # keys and values of one decode step of 8 requests, 13B heads
        {"name": "write_decode_8", "op": "write", "rows": 8, "q_heads": 40, "kv_heads": 40, "dim": 128, "page": 64},
        # the keys and values of four 500-token prompts and two short ones, 7B heads
        {"name": "write_prompts_2050", "op": "write", "rows": 2050, "q_heads": 32, "kv_heads": 32, "dim": 128, "page": 16},
        # one user's generation, a short context: latency
        {"name": "attend_1x100", "op": "attend", "rows": 1, "q_heads": 32, "kv_heads": 32, "dim": 128, "page": 64, "least": 100, "most": 100},
        # 32 users behind contexts of very different lengths, two rows of the batch without a request
        {"name": "attend_32x4000", "op": "attend", "rows": 32, "q_heads": 32, "kv_heads": 32, "dim": 128, "page": 64, "least": 16, "most": 4000},
        # three long documents on grouped key-value heads, pages that end inside any tile
        {"name": "attend_3x60000_grouped", "op": "attend", "rows": 3, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 24, "least": 9000, "most": 60001},
        # the smallest batch: three rows of two fine-tuned models on a narrow, ragged module
        {"name": "delta_1000x2048_t3", "op": "delta", "M": 1000, "N": 2048, "rows": 3, "deltas": 2, "least": 128, "most": 384},
        # 16 users of 12 fine-tuned models at an attention projection
        {"name": "delta_4096x4096_t16", "op": "delta", "M": 4096, "N": 4096, "rows": 16, "deltas": 12, "least": 256, "most": 512},
        # a full batch on 48 fine-tuned models at an MLP projection, popular ones with many rows
        {"name": "delta_11008x4096_t128", "op": "delta", "M": 11008, "N": 4096, "rows": 128, "deltas": 48, "least": 256, "most": 768},
        # the next tokens of 8 users with their log probabilities and five alternatives
        {"name": "logprobs_8x32000_k5", "op": "logprobs", "rows": 8, "vocab": 32000, "dtype": "bfloat16", "top": 5},
        # scoring a 2048-token document over an odd, large vocabulary with masked tokens, float32 logits
        {"name": "logprobs_2048x50257_k20", "op": "logprobs", "rows": 2048, "vocab": 50257, "dtype": "float32", "top": 20},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(8, 8, 64), (8, 2, 64), (4, 4, 32), (32, 32, 128), (40, 40, 128), (32, 8, 128), (40, 8, 128), (48, 3, 96), (16, 2, 256)]


def draw(rng):
    op = rng.choice(["extend", "write", "attend", "attend", "attend", "delta", "delta", "delta", "logprobs", "logprobs"])
    if op == "extend":
        return {"op": op, "requests": _log(rng, 1, 1500), "most": _log(rng, 8, 700), "fresh": rng.choice([0, 0, 25, 70]), "page": rng.choice([1, 8, 16, 24, 64, 128])}
    if op in ("write", "attend"):
        hq, hk, dim = rng.choice(HEADS)
        case = {"op": op, "q_heads": hq, "kv_heads": hk, "dim": dim, "page": rng.choice([1, 8, 16, 24, 64, 100, 128, 256])}
        if op == "write":
            return dict(case, rows=_log(rng, 1, 2000))
        rows = _log(rng, 1, 60)
        most = _log(rng, 1, max(1, min(60000, 32 * 4000 * 4096 // (rows * hk * dim))))
        return dict(case, rows=rows, most=most, least=_log(rng, 1, most))
    if op == "delta":
        rows = _log(rng, 1, 128)
        least = 128 * rng.randint(1, 4)
        return {"op": op, "M": _log(rng, 300, 11008), "N": 128 * _log(rng, 2, 86), "rows": rows, "deltas": _log(rng, 1, 24), "least": least,
                "most": least + 128 * rng.randint(0, 4)}
    return {"op": op, "rows": _log(rng, 1, 1500), "vocab": _log(rng, 500, 60000), "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]),
            "top": rng.choice([0, 1, 5, 20, 32])}


# ------------------------------------------------------------------------------------ what a program has in hand
def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _ints(g, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=g, device=DEVICE)


def _bf16(g, *shape):
    return torch.randn(shape, generator=g, device=DEVICE).to(torch.bfloat16)


def _tables(g, counts, width, spare):
    """Block table (requests, width) with distinct random pages for the first counts[b] entries of each row, -1 behind, and the pages left over."""
    n = int(counts.sum())
    order = torch.randperm(n + spare, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((counts.shape[0], width), -1, dtype=torch.int32, device=DEVICE)
    table[torch.arange(width, device=DEVICE)[None] < counts[:, None]] = order[:n]
    return table, order[n:]


def _angles(positions, dim):
    """cos / sin tables (rows, dim) in bfloat16, as a model's rotary embedding gives them."""
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device=DEVICE, dtype=torch.float64) / dim)
    a = positions.double()[:, None] * inv[None]
    a = torch.cat((a, a), -1)
    return a.cos().to(torch.bfloat16), a.sin().to(torch.bfloat16)


def _cap(case):
    return case["most"] + 2 * case["page"]


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "extend":
        B, most, ps = case["requests"], case["most"], case["page"]
        lengths = _ints(g, 0, most, B)
        u = torch.rand(B, generator=g, device=DEVICE)
        if case["fresh"]:                                          # most requests enter with a prompt, the others rest or leave
            fresh = _ints(g, 1, case["fresh"], B)
            new = torch.where(u < 0.9, fresh, torch.where(u < 0.95, torch.zeros_like(fresh), -torch.ones_like(fresh)))
            lengths = torch.where(u < 0.85, torch.zeros_like(lengths), lengths)
        else:
            new = torch.where(u < 0.05, torch.zeros_like(lengths), torch.where(u < 0.08, -torch.ones_like(lengths), torch.ones_like(lengths)))
        width = -(-(most + case["fresh"] + 1) // ps)
        table, left = _tables(g, -(-lengths // ps), width, B + B * case["fresh"] // ps)
        pages = int(left.shape[0]) + B * width
        free = torch.full((pages,), -1, dtype=torch.int32, device=DEVICE)
        free[:left.shape[0]] = left
        return {"op": op, "lengths": lengths.int(), "new": new.int(), "table": table, "free": free, "page": ps, "total": B * max(1, case["fresh"]),
                "count": torch.tensor([left.shape[0]], dtype=torch.int32, device=DEVICE)}
    if op == "write":
        T, hk, dim, ps = case["rows"], case["kv_heads"], case["dim"], case["page"]
        # keys and values are column slices of one fused projection; a few rows of the batch have no request
        y = _bf16(g, T, (case["q_heads"] + 2 * hk) * dim)
        k, v = y[:, case["q_heads"] * dim:].view(T, 2, hk, dim).unbind(1)
        pages = -(-T // ps) + 3
        slots = torch.randperm(pages, generator=g, device=DEVICE)[:, None] * ps + torch.arange(ps, device=DEVICE)[None]
        slots = slots.reshape(-1)[:T].clone()
        slots[_ints(g, 0, 39, T) == 0] = -1
        cos, sin = _angles(_ints(g, 0, 4000, T), dim)
        return {"op": op, "k": k, "v": v, "slots": slots, "cos": cos, "sin": sin, "page": ps,
                "k_pages": _bf16(g, pages, hk, ps, dim), "v_pages": _bf16(g, pages, hk, ps, dim)}
    if op == "attend":
        T, hq, hk, dim, ps = case["rows"], case["q_heads"], case["kv_heads"], case["dim"], case["page"]
        lo, hi = math.log(case["least"]), math.log(case["most"])
        n = torch.exp(lo + (hi - lo) * torch.rand(T, generator=g, device=DEVICE, dtype=torch.float64)).round().long().clamp(1, case["most"])
        n[0] = case["most"]
        table, _ = _tables(g, -(-n // ps), -(-_cap(case) // ps), 5)
        pages = int((-(-n // ps)).sum()) + 5
        requests, positions = torch.arange(T, device=DEVICE), n - 1
        if T > 8:                                                  # rows of the batch that have no request
            requests[3], requests[T - 1] = -1, -1
        cos, sin = _angles(positions, dim)
        y = _bf16(g, T, (hq + 2 * hk) * dim)
        k_pages = _bf16(g, pages, hk, ps, dim)
        return {"op": op, "q": y[:, :hq * dim].view(T, hq, dim), "cos": cos, "sin": sin, "table": table, "requests": requests.int(), "positions": positions,
                "k_pages": k_pages, "v_pages": _bf16(g, pages, hk, ps, dim), "scale": 1.7 / math.sqrt(dim), "page": ps}
    if op == "delta":
        M, N, T, K = case["M"], case["N"], case["rows"], case["deltas"]
        ng = _ints(g, case["least"] // GROUP, case["most"] // GROUP, K)
        start = torch.zeros(K + 1, dtype=torch.int32, device=DEVICE)
        start[1:] = ng.cumsum(0)
        G = int(start[-1])
        scale = lambda *shape: (torch.exp(torch.randn(shape, generator=g, device=DEVICE) * 0.3) * 1.5e-3).to(torch.bfloat16)
        bank = {"uq": _ints(g, 0, 255, G, M, GROUP // 2).to(torch.uint8), "us": scale(G, M), "uz": _ints(g, 0, 15, G, M).to(torch.uint8),
                "vt": _ints(g, 0, 255, G, GROUP, N // 2).to(torch.uint8), "vs": scale(G, N), "vz": _ints(g, 0, 15, G, N).to(torch.uint8),
                "start": start, "M": M, "N": N}
        ids = (K * torch.rand(T, generator=g, device=DEVICE) ** 1.7).int().clamp(max=K - 1)      # some fine-tunes are more popular
        if T > 8:
            ids[_ints(g, 0, 19, T) == 0] = -1                     # a user of the base model
        return {"op": op, "x": _bf16(g, T, N), "y": (1.28 * torch.randn(T, M, generator=g, device=DEVICE)).to(torch.bfloat16), "bank": bank, "ids": ids}
    T, V = case["rows"], case["vocab"]
    dtype = getattr(torch, case["dtype"])
    x = torch.randn(T, V, generator=g, device=DEVICE) * 2.0
    rows = torch.arange(T, device=DEVICE)
    favoured = _ints(g, 0, V - 1, T)
    x[rows, favoured] += 14.0 * torch.rand(T, generator=g, device=DEVICE)
    x[:, _ints(g, 0, V - 1, 7)] = float("-inf")                    # tokens that may not be produced
    tokens = torch.where(torch.rand(T, generator=g, device=DEVICE) < 0.5, favoured, _ints(g, 0, V - 1, T))
    x[rows, tokens] = x[rows, tokens].clamp(min=-9.0)
    if T > 8:
        tokens[_ints(g, 0, 19, T) == 0] = -1                      # positions without a given token
    return {"op": op, "logits": x.to(dtype), "tokens": tokens, "top": case["top"]}


# ------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["op"]
    if own:
        if op == "extend":
            from ade_b200.paged import paged_extend

            slots, positions, requests, lengths, count, status = paged_extend(s["lengths"], s["new"], s["table"], s["free"], s["count"], s["total"], s["page"])
            return {"slots": slots, "positions": positions, "requests": requests, "lengths": lengths, "count": count, "status": status,
                    "table": s["table"], "free": s["free"]}
        if op == "write":
            from ade_b200.paged import paged_write

            paged_write(s["k"], s["v"], s["slots"], s["k_pages"], s["v_pages"], s["cos"], s["sin"])
            return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if op == "attend":
            from ade_b200.paged import paged_attn_decode

            return paged_attn_decode(s["q"], s["table"], s["requests"], s["positions"], s["k_pages"], s["v_pages"], s["scale"], s["cos"], s["sin"])
        if op == "delta":
            from ade_b200.kernels import multi_delta_forward

            return multi_delta_forward(s["x"], s["y"], s["bank"], s["ids"])
        from ade_b200.decode_ops import token_logprobs

        return token_logprobs(s["logits"], s["tokens"], s["top"])
    if op == "extend":
        return _extend(s)
    if op == "write":
        return _write(s)
    if op == "attend":
        return _attend(s)
    if op == "delta":
        return _delta(s)
    return _logprobs(s)


def _extend(s):
    lengths, new, table, free, ps, total = s["lengths"].long(), s["new"].long(), s["table"], s["free"], s["page"], s["total"]
    B, W = table.shape
    dev = table.device
    released, grow = new < 0, new.clamp(min=0)
    have, end = -(-lengths // ps), lengths + grow
    row_end = grow.cumsum(0)
    last = -(-end // ps)
    status = torch.zeros(B, dtype=torch.int32, device=dev)
    status[(last > W) & ~released] = 2
    status[(row_end > total) & ~released] = 3
    need = torch.where(released | (status > 0), torch.zeros_like(last), last - have)
    back = torch.where(released, have, torch.zeros_like(have))
    count = s["count"].long()
    available = count + back.sum()
    cum = need.cumsum(0)
    status[(need > 0) & (cum > available)] = 1
    fine = (status == 0) & ~released
    # pages handed back go on the stack
    col = torch.arange(W, device=dev)[None]
    mask = released[:, None] & (col < have[:, None])
    place = (count + back.cumsum(0) - back)[:, None] + col
    free[place[mask]] = table[mask]
    # pages taken come from its top
    mask = fine[:, None] & (col >= have[:, None]) & (col < last[:, None])
    place = available - 1 - ((cum - need)[:, None] + col - have[:, None])
    table[mask] = free[place[mask]]
    used = torch.where(fine & (need > 0), cum, torch.zeros_like(cum)).max()
    # rows of the packed batch
    row = torch.arange(total, device=dev)
    request = torch.searchsorted(row_end, row, right=True)
    inside = request < B
    request = request.clamp(max=B - 1)
    inside &= fine[request]
    position = lengths[request] + row - (row_end - grow)[request]
    position = torch.where(inside, position, torch.zeros_like(position))
    slot = table[request, (position // ps).clamp(max=W - 1)].long() * ps + position % ps
    return {"slots": torch.where(inside, slot, -torch.ones_like(slot)), "positions": position,
            "requests": torch.where(inside, request, -torch.ones_like(request)).int(),
            "lengths": torch.where(released, torch.zeros_like(end), torch.where(fine, end, lengths)).int(), "count": (available - used).int(),
            "status": status, "table": table, "free": free}


def _rotated(x, cos, sin):
    """x (rows, heads, dim) at the angles of its rows, in 32 bits."""
    x, cos, sin = x.float(), cos.float()[:, None], sin.float()[:, None]
    a, b = x.chunk(2, -1)
    return x * cos + torch.cat((-b, a), -1) * sin


def _write(s):
    rows = s["slots"] >= 0
    slot = s["slots"][rows]
    page, off = slot // s["page"], slot % s["page"]
    s["k_pages"][page, :, off] = _rotated(s["k"][rows], s["cos"][rows], s["sin"][rows]).to(torch.bfloat16)
    s["v_pages"][page, :, off] = s["v"][rows]
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _attend(s):
    q, positions, kp = s["q"], s["positions"], s["k_pages"]
    T, hq, dim = q.shape
    hk, ps = kp.shape[1], kp.shape[2]
    table = s["table"][s["requests"].long().clamp(min=0)].long().clamp(min=0)
    dense = lambda pages: pages[table].permute(0, 2, 1, 3, 4).reshape(T, hk, -1, dim).float()
    qf = _rotated(q, s["cos"], s["sin"]).view(T, hk, hq // hk, dim)
    scores = torch.matmul(qf, dense(kp).transpose(-1, -2)) * s["scale"]
    seen = torch.arange(scores.shape[-1], device=q.device)[None] <= positions[:, None]
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    w = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(w, dense(s["v_pages"])) / w.sum(-1, keepdim=True)
    out = out.masked_fill((s["requests"] < 0)[:, None, None, None], 0.0)
    return out.reshape(T, hq * dim).to(torch.bfloat16)


def _codes(packed):
    """(..., n) bytes -> (..., 2 n) codes in 32-bit floats."""
    b = packed.unflatten(-1, (-1, 4))
    nib = torch.stack((b & 15, b >> 4), -1).flatten(-2)
    return nib[..., [NIBBLES.index(j) for j in range(8)]].flatten(-2).float()


def _delta(s):
    bank, ids, x = s["bank"], s["ids"], s["x"]
    G, T = bank["uq"].shape[0], x.shape[0]
    # which rows use which rank group: those whose delta it belongs to
    owner = torch.searchsorted(bank["start"], torch.arange(G, device=x.device, dtype=torch.int32), right=True) - 1
    uses = (ids[:, None] == owner[None]).float()
    V = (_codes(bank["vt"]) - bank["vz"].float()[:, None]) * bank["vs"].float()[:, None]
    h = torch.matmul(x.float(), V.reshape(G * GROUP, -1).t()).view(T, G, GROUP) * uses[..., None]
    U = (_codes(bank["uq"]) - bank["uz"].float()[..., None]) * bank["us"].float()[..., None]
    return (s["y"].float() + torch.matmul(h.view(T, -1), U.transpose(0, 1).reshape(bank["M"], -1).t())).to(torch.bfloat16)


def _logprobs(s):
    x, tokens, top = s["logits"].float(), s["tokens"], s["top"]
    m = x.amax(-1, keepdim=True)
    z = x - m
    e = torch.exp(z)
    total = e.sum(-1)
    log_total = torch.log(total)
    entropy = log_total - torch.where(e > 0, e * z, torch.zeros_like(e)).sum(-1) / total
    given = z.gather(1, tokens.clamp(min=0)[:, None])[:, 0] - log_total
    best, where = torch.sort(z, dim=-1, descending=True, stable=True)
    return (torch.where(tokens >= 0, given, torch.zeros_like(given)), entropy, best[:, :top] - log_total[:, None], where[:, :top])


# ------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "extend":
        B, rows = case["requests"], case["requests"] * max(1, case["fresh"])
        return {"bytes": 20.0 * B + 20.0 * rows + 12.0 * rows / case["page"], "flops": 20.0 * B + 10.0 * rows}
    if op == "write":
        values = float(case["rows"]) * case["kv_heads"] * case["dim"]
        return {"bytes": 8.0 * values + case["rows"] * (8.0 + 4.0 * case["dim"]), "flops": 3.0 * values}
    if op == "attend":
        # contexts spread over the logarithm between the shortest and the longest
        lo, hi, T = case["least"], case["most"], case["rows"]
        mean = (hi - lo) / math.log(hi / lo) if hi > lo else float(hi)
        n = hi + (T - 1 - (2 if T > 8 else 0)) * mean
        return {"bytes": 4.0 * n * case["kv_heads"] * case["dim"] + T * case["dim"] * (4.0 * case["q_heads"] + 4.0),
                "flops": 4.0 * n * case["q_heads"] * case["dim"]}
    if op == "delta":
        M, N, T, K = case["M"], case["N"], case["rows"], case["deltas"]
        # deltas with at least one row, when row t takes delta floor(K u^1.7)
        used = sum(1.0 - (1.0 - (((k + 1) / K) ** (1 / 1.7) - (k / K) ** (1 / 1.7))) ** T for k in range(K))
        rank = (case["least"] + case["most"]) / 2.0
        return {"bytes": used * rank * (M + N) * (0.5 + 3.0 / GROUP) + 2.0 * T * N + 4.0 * T * M, "flops": 2.0 * T * rank * (M + N)}
    size = 4.0 if case["dtype"] == "float32" else 2.0
    return {"bytes": case["rows"] * (case["vocab"] * size + 16.0 + 12.0 * case["top"]), "flops": 5.0 * case["rows"] * case["vocab"]}


# ------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "extend":
        return None                                                # whole numbers
    if op == "write":
        k, v = s["k_pages"].double(), s["v_pages"].double()
        half = case["dim"] // 2
        for t, slot in enumerate(s["slots"].tolist()):
            if slot < 0:
                continue
            x, c, n = s["k"][t].double(), s["cos"][t].double(), s["sin"][t].double()
            first = x[:, :half] * c[:half] - x[:, half:] * n[:half]
            second = x[:, half:] * c[half:] + x[:, :half] * n[half:]
            k[slot // case["page"], :, slot % case["page"]] = torch.cat((first, second), 1)
            v[slot // case["page"], :, slot % case["page"]] = s["v"][t].double()
        return {"k_pages": k, "v_pages": v}
    if op == "attend":
        T, hq, dim = s["q"].shape
        group, half, ps = hq // case["kv_heads"], dim // 2, case["page"]
        out = torch.zeros(T, hq, dim, dtype=torch.float64, device=DEVICE)
        for t, (b, p) in enumerate(zip(s["requests"].tolist(), s["positions"].tolist())):
            if b < 0:
                continue
            pages = s["table"][b, :p // ps + 1].long()
            k = s["k_pages"][pages].transpose(0, 1).flatten(1, 2)[:, :p + 1]
            v = s["v_pages"][pages].transpose(0, 1).flatten(1, 2)[:, :p + 1]
            c, n = s["cos"][t].double(), s["sin"][t].double()
            for h in range(hq):
                x = s["q"][t, h].double()
                r = torch.cat((x[:half] * c[:half] - x[half:] * n[:half], x[half:] * c[half:] + x[:half] * n[half:]))
                weights = torch.softmax((k[h // group].double() * r).sum(-1) * s["scale"], 0)
                out[t, h] = (weights[:, None] * v[h // group].double()).sum(0)
        return out.view(T, -1)
    if op == "delta":
        bank, start = s["bank"], s["bank"]["start"].tolist()
        out, ids = s["y"].double(), s["ids"].tolist()

        def weights(packed, zero, scale):                           # nibble i of a word holds code NIBBLES[i]
            w = packed.contiguous().view(torch.int32).long() & 0xFFFFFFFF
            c = torch.empty(*w.shape, 8, dtype=torch.float64, device=DEVICE)
            for i, j in enumerate(NIBBLES):
                c[..., j] = ((w >> (4 * i)) & 15).double()
            return (c.flatten(-2) - zero.double()) * scale.double()

        for d in sorted(set(ids) - {-1}):
            rows = torch.tensor([t for t, i in enumerate(ids) if i == d], device=DEVICE)
            x = s["x"][rows].double()
            for g in range(start[d], start[d + 1]):
                h = x @ weights(bank["vt"][g], bank["vz"][g][None], bank["vs"][g][None]).t()
                out[rows] += h @ weights(bank["uq"][g], bank["uz"][g][:, None], bank["us"][g][:, None]).t()
        return out
    x = s["logits"].double()
    logp = x - torch.logsumexp(x, -1, keepdim=True)
    p = logp.exp()
    entropy = -(p * logp.clamp(min=-1e30)).sum(-1)
    given = torch.where(s["tokens"] >= 0, logp[torch.arange(x.shape[0], device=DEVICE), s["tokens"].clamp(min=0)], 0.0)
    return (given, entropy, logp.sort(-1, descending=True)[0][:, :case["top"]], None)
