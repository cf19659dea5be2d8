"""The operators around a paged key-value cache, as cases whose time and outputs can be measured.

A serving program rotates a step's queries and keys (one position axis for text, several for images
and video), writes the new keys and values into the pages of its cache, attends the new token over
them, and keeps the cache within a budget by dropping the keys that drew the least attention.  A
training program needs the rotation's gradient.

    listed()            the fixed cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs on the GPU, as a program has them before the call
    run(state)          one pass; its outputs (own: through the framework, else in plain torch)
    work(case)          bytes and operations that the pass cannot do without
    exact(case, seed)   the same outputs in float64, written from the definitions

Pages are (page, kv head, slot, dim); a sequence's key j lies in page table[b, j // page_size], slot
j % page_size.  Unused table entries are -1.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PKG = os.path.join(_ROOT, "sparse-thresholded-attention_amd")
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
THETA = 500000.0
SECTIONS = {1: (1.0,), 2: (0.5, 0.5), 3: (0.25, 0.375, 0.375)}   # shares of the frequencies per axis
NEG = float("-inf")


def _case(name, op, dtype, heads, kv_heads, d, **kw):
    c = {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "d": d}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the rotation of one decoding step: a new token of each of 16 sequences, text positions
        _case("rotary_step", "rotary", "bf16", 32, 8, 128, tokens=16, axes=1, grad=False),
        # a prompt with images: positions on time, height and width
        _case("rotary_prompt", "rotary", "fp16", 32, 8, 128, tokens=8191, axes=3, grad=False),
        # the same rotation's gradient in a training step
        _case("rotary_grad", "rotary", "bf16", 32, 32, 128, tokens=16384, axes=3, grad=True),
        # the new keys and values of a decoding step of 64 sequences
        _case("append_step", "append", "fp16", 32, 8, 128, batch=64, n=4096, new=1, page=16, shape=3),
        # several prompts of different lengths written in one call
        _case("append_prompts", "append", "bf16", 32, 8, 128, batch=12, n=64, new=4001, page=32, shape=4),
        # one user's decoding step over a short conversation: latency counts
        _case("attend_one", "attend", "bf16", 32, 8, 128, batch=1, n=1000, q=1, page=16, weights=False, shape=0),
        # a serving batch of very different lengths, some just begun
        _case("attend_batch", "attend", "bf16", 32, 8, 128, batch=40, n=12288, q=1, page=16, weights=False, shape=5),
        # two long documents without grouped heads' savings in fp16, large pages
        _case("attend_long", "attend", "fp16", 16, 8, 128, batch=2, n=131072, q=1, page=64, weights=False, shape=6),
        # a small fp32 model's step that also accumulates each key's attention weight
        _case("attend_fp32_weights", "attend", "fp32", 8, 8, 64, batch=8, n=2047, q=1, page=32, weights=True,
              shape=7),
        # the last 32 queries of a prompt weigh its keys before the cache is cut
        _case("attend_window", "attend", "bf16", 32, 8, 128, batch=4, n=12288, q=32, page=64, weights=True, shape=8),
        # prompts cut to 2048 keys a head, into pages of their own
        _case("evict_prompts", "evict", "bf16", 32, 8, 128, batch=8, n=12288, budget=2048, page=32, shape=9),
        # one decoding step of 32 sequences held at 4096 keys: rotate, append, attend with weights, evict one
        _case("step_budget", "step", "bf16", 32, 8, 128, batch=32, budget=4096, page=16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "evict", "step"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    heads, kv_heads = rng.choice([(32, 8), (32, 32), (16, 2), (40, 8), (8, 8), (28, 4), (24, 1), (12, 12)])
    d = rng.choice([128, 128, 64])
    page = rng.choice([8, 16, 32, 64, 128, 256])
    shape = rng.randrange(1, 1 << 20)
    row = kv_heads * d * SIZES[dtype] * 2                  # bytes of a token's keys and values
    if op == "rotary":
        most = (16384 * 64 * 128 * 2) // ((heads + kv_heads) * d * SIZES[dtype])
        return _case(None, op, dtype, heads, kv_heads, d, tokens=_log_int(rng, 1, most), axes=rng.randint(1, 3),
                     grad=rng.random() < 0.5)
    if op == "append":
        new = rng.choice([1, _log_int(rng, 2, 4000)])
        batch = _log_int(rng, 1, max(1, min(128, (96 << 20) // (row * new))))
        return _case(None, op, dtype, heads, kv_heads, d, batch=batch, n=_log_int(rng, 1, 1500), new=new, page=page,
                     shape=shape)
    if op == "attend":
        q = rng.choice([1, 1, 1, 2, 5, 16, 32])
        n = _log_int(rng, 16, min((512 << 20) // row, 131072 if q == 1 else 12288))
        batch = _log_int(rng, 1, max(1, min(64, (512 << 20) // (row * n), (1 << 27) // (n * heads * q))))
        return _case(None, op, dtype, heads, kv_heads, d, batch=batch, n=n, q=q, page=page,
                     weights=rng.random() < 0.5, shape=shape)
    if op == "evict":
        n = _log_int(rng, 64, min((384 << 20) // row, 32768))
        batch = _log_int(rng, 1, max(1, min(16, (384 << 20) // (row * n))))
        return _case(None, op, dtype, heads, kv_heads, d, batch=batch, n=n, budget=_log_int(rng, 48, max(49, n)),
                     page=page, shape=shape)
    budget = _log_int(rng, 128, 4096)
    batch = _log_int(rng, 1, max(1, min(32, (384 << 20) // (row * budget))))
    return _case(None, op, dtype, heads, kv_heads, d, batch=batch, budget=budget, page=page)


# -----------------------------------------------------------------------------------------------
# shapes that a case stands for
# -----------------------------------------------------------------------------------------------
def _lens(case):
    """Lengths up to n: the longest first, the others spread over their logarithm, one of them empty
    in a batch of more than 8."""
    n, batch = case["n"], case["batch"]
    rng = random.Random(case["shape"])
    lens = [n] + [min(n, _log_int(rng, max(1, n // 64), n)) for _ in range(batch - 1)]
    if batch > 8:
        lens[batch // 2] = 0
    return lens


def _new_counts(case):
    rng = random.Random(case["shape"] + 1)
    new = case["new"]
    return [new] + [new if new == 1 else _log_int(rng, max(1, new // 16), new) for _ in range(case["batch"] - 1)]


def _sections(case):
    half = case["d"] // 2
    s = [int(share * half) for share in SECTIONS[case["axes"]]]
    s[0] += half - sum(s)
    return tuple(s)


def _pages(tokens, page):
    return -(-tokens // page)


# -----------------------------------------------------------------------------------------------
# inputs
# -----------------------------------------------------------------------------------------------
def _randn(g, shape, dtype, scale=1.0):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32 if dtype == torch.float32 else dtype)
    return x.mul_(scale) if scale != 1.0 else x


def _tables(need, width, page_ids):
    """A table (batch, width): need[b] pages of the shuffled page_ids each, -1 behind them."""
    free = iter(page_ids.tolist())
    return _int32([[next(free) for _ in range(n)] + [-1] * (width - n) for n in need])


def _cache(g, case, pages, fill=True):
    shape = (pages, case["kv_heads"], case["page"], case["d"])
    dtype = DTYPES[case["dtype"]]
    if not fill:
        return torch.zeros(shape, dtype=dtype, device="cuda"), torch.zeros(shape, dtype=dtype, device="cuda")
    return _randn(g, shape, dtype), _randn(g, shape, dtype)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _inv_freq(d):
    return (1.0 / THETA ** (torch.arange(0, d, 2, dtype=torch.float64) / d)).float().cuda()


def _page_positions(table, page, kv_heads, pages, width_tokens):
    """pos pages (pages, kv_heads, page): key j of a sequence has position j."""
    pos = torch.zeros((pages + 1, page), dtype=torch.int32, device="cuda")
    slots = torch.arange(width_tokens, dtype=torch.int32, device="cuda").reshape(1, -1, page)
    pos[table.long()] = slots.expand(table.shape[0], -1, -1)          # -1 lands in the spare last page
    return pos[:pages, None].expand(pages, kv_heads, page).contiguous()


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    dtype, heads, kv, d = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["d"]
    s = {"case": case, "sm_scale": 1.0 / math.sqrt(d)}
    if case["op"] == "rotary":
        t, axes = case["tokens"], case["axes"]
        s["q"] = _randn(g, (t, heads, d), dtype)
        s["k"] = _randn(g, (t, kv, d), dtype)
        if axes == 1:                                      # tokens anywhere in their sequences
            pos = torch.randint(0, 131072, (1, t), generator=g, device="cuda", dtype=torch.int32)
        else:                                              # frames of 24 x 36 patches behind a text
            i = torch.arange(t, device="cuda")
            base = int(torch.randint(0, 4096, (1,), generator=cpu))
            pos = torch.stack([i // 864, i // 36 % 24, i % 36])[3 - axes:].to(torch.int32) + base
        s["positions"] = pos.contiguous()
        s["inv_freq"], s["sections"] = _inv_freq(d), _sections(case)
        return s
    page = case["page"]
    if case["op"] == "append":
        lens, new = _lens(case), _new_counts(case)
        need = [_pages(a + b, page) for a, b in zip(lens, new)]
        pages = sum(need) + 3
        s["k_pages"], s["v_pages"] = _cache(g, case, pages, fill=False)
        s["table"] = _tables(need, max(need) + 1, torch.randperm(pages, generator=cpu).to(torch.int32))
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        s["k"] = _randn(g, (starts[-1], kv, d), dtype)
        s["v"] = _randn(g, (starts[-1], kv, d), dtype)
        s["lens"], s["starts"] = _int32(lens), _int32(starts)
        return s
    if case["op"] == "attend":
        lens = _lens(case)
        need = [_pages(n, page) for n in lens]
        pages = sum(need) + 3
        s["k_pages"], s["v_pages"] = _cache(g, case, pages)
        s["table"] = _tables(need, max(need), torch.randperm(pages, generator=cpu).to(torch.int32))
        shape = (len(lens), heads, d) if case["q"] == 1 else (len(lens), heads, case["q"], d)
        s["q"] = _randn(g, shape, dtype, 2.0)              # scores of standard deviation 2
        s["lens"] = _int32(lens)
        if case["weights"]:
            s["weight"] = torch.zeros((pages, kv, page), device="cuda")
        return s
    batch = case["batch"]
    lens = _lens(case) if case["op"] == "evict" else [case["budget"]] * batch
    need = [_pages(n + (case["op"] == "step"), page) for n in lens]
    left = [_pages(min(n, case["budget"]), page) for n in lens] if case["op"] == "evict" else [0] * batch
    pages = sum(need) + sum(left) + 3
    ids = torch.randperm(pages, generator=cpu).to(torch.int32)
    s["k_pages"], s["v_pages"] = _cache(g, case, pages)
    s["table"] = _tables(need, max(need), ids)
    s["pos"] = _page_positions(s["table"], page, kv, pages, s["table"].shape[1] * page)
    # what a key has drawn: most little, some much
    u = torch.rand((pages, kv, page), generator=g, device="cuda").clamp_(min=1e-7)
    s["weight"] = u.log_().neg_().square_()
    s["lens"], s["spare"] = _int32(lens), int(ids[-1])
    if case["op"] == "evict":
        s["dst_table"] = _tables(left, max(left), ids[sum(need):])
        return s
    s["q"] = _randn(g, (batch, heads, d), dtype, 2.0)
    s["k"] = _randn(g, (batch, kv, d), dtype)
    s["v"] = _randn(g, (batch, kv, d), dtype)
    s["inv_freq"] = _inv_freq(d)
    s["seen"] = _int32([case["budget"] + 1000 + 37 * b for b in range(batch)])
    return s


N_GLOBAL, N_LOCAL = 4, 32        # keys that an eviction always keeps: the first and the latest


# -----------------------------------------------------------------------------------------------
# plain forms: elementary torch operations in 32 bits (angles in 64)
# -----------------------------------------------------------------------------------------------
def _plain_rotary(x, positions, inv_freq, sections, sign):
    axis = torch.repeat_interleave(torch.arange(len(sections), device=x.device),
                                   torch.tensor(sections, device=x.device), output_size=sum(sections))
    angle = positions.double()[axis].t() * inv_freq.double()                     # (T, D/2)
    c, s = angle.cos().float()[:, None], sign * angle.sin().float()[:, None]
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(x.dtype)


def _plain_rows(table, page, n):
    """Page and slot (batch, n) of the keys 0 .. n - 1; unused entries point to page 0."""
    j = torch.arange(n, device=table.device)
    return table[:, j // page].long().clamp(min=0), (j % page).expand(table.shape[0], n)


def _plain_append(k_pages, v_pages, k, v, table, lens, starts):
    page = k_pages.shape[2]
    t = torch.arange(k.shape[0], device=k.device, dtype=torch.int32)
    b = torch.searchsorted(starts, t, right=True) - 1
    j = (lens[b] + t - starts[b]).long()
    where = (table[b, j // page].long(), j % page)
    k_pages[where[0], :, where[1]] = k
    v_pages[where[0], :, where[1]] = v
    return lens + starts[1:] - starts[:-1], where, j


def _plain_attend(q, k_pages, v_pages, table, lens, sm_scale, n, weight=None):
    page, kv, d = k_pages.shape[2], k_pages.shape[1], k_pages.shape[3]
    q4 = q if q.dim() == 4 else q[:, :, None]
    batch, heads, nq, _ = q4.shape
    where = _plain_rows(table, page, n)
    k = k_pages[where[0], :, where[1]].float().permute(0, 2, 3, 1)               # (B, Hkv, D, n)
    v = v_pages[where[0], :, where[1]].float().permute(0, 2, 1, 3)
    rows = q4.float().reshape(batch, kv, heads // kv * nq, d)
    s = (rows @ k.contiguous()).mul_(sm_scale).view(batch, kv, heads // kv, nq, n)
    end = lens[:, None] - torch.arange(nq - 1, -1, -1, device=q.device)          # (B, nq): keys a query sees
    s.masked_fill_(torch.arange(n, device=q.device) >= end[:, None, None, :, None], NEG)
    m = s.amax(dim=-1, keepdim=True)
    p = s.sub_(torch.where(m == NEG, 0.0, m)).exp_()
    p.div_(p.sum(dim=-1, keepdim=True).clamp(min=1e-30))
    out = (p.view(batch, kv, -1, n) @ v.contiguous()).reshape(q.shape).to(q.dtype)
    if weight is not None:
        drawn = p.sum(dim=(2, 3)).transpose(1, 2)                                # (B, n, Hkv)
        flat = (where[0][:, :, None] * kv + torch.arange(kv, device=q.device)) * page + where[1][:, :, None]
        weight.view(-1).index_add_(0, flat.reshape(-1), drawn.reshape(-1))
    return out


def _plain_evict(k_pages, v_pages, weight, pos, table, lens, budget, n, spare, dst_table=None):
    """Keep min(len, budget) keys a head: the first N_GLOBAL positions, the latest N_LOCAL, then by
    weight, the lower slot first among equals.  In place the kept keys behind the budget move into
    the free slots before it, in order; into dst_table all kept keys move, in order."""
    page, kv = k_pages.shape[2], k_pages.shape[1]
    where = _plain_rows(table, page, n)
    at = torch.arange(n, device=lens.device)
    live = (at < lens[:, None])[:, None]                                          # (B, 1, n)
    w = weight[where[0], :, where[1]].transpose(1, 2)                             # (B, Hkv, n)
    p = pos[where[0], :, where[1]].transpose(1, 2).masked_fill(~live, -1)
    forced = (p < N_GLOBAL) | (p > p.amax(dim=-1, keepdim=True) - N_LOCAL)
    rank = torch.where(forced, float("inf"), w).masked_fill(~live, NEG)
    order = rank.sort(dim=-1, descending=True, stable=True).indices
    left = lens.clamp(max=budget)
    keep = torch.zeros_like(order, dtype=torch.bool)
    keep.scatter_(2, order, (at < left[:, None])[:, None].expand_as(order))
    m = min(n, budget)
    if dst_table is None:
        free = ~keep[:, :, :m]
        moved = keep.clone()
        moved[:, :, :m] = False
        far = torch.where(moved, at, n).sort(dim=-1).values                       # the movers, in order
        nth = (free.cumsum(dim=-1) - 1).clamp(min=0)
        src = torch.where(free, far.gather(2, nth), at[:m]).clamp(max=n - 1)
        to = (where[0][:, :m], where[1][:, :m])
    else:
        src = torch.where(keep, at, n).sort(dim=-1).values[:, :, :m].clamp(max=n - 1)
        to = _plain_rows(dst_table, page, m)
    src_page = where[0][:, None].expand(-1, kv, -1).gather(2, src)
    src_slot = where[1][:, None].expand(-1, kv, -1).gather(2, src)
    head = torch.arange(kv, device=lens.device)[None, :, None]
    index = ((src_page * kv + head) * page + src_slot)
    flat = ((to[0][:, None] * kv + head) * page + to[1][:, None])
    used = (at[:m] < left[:, None])[:, None]
    index = torch.where(used, index, spare * kv * page)                           # no sequence's page
    flat = torch.where(used, flat, spare * kv * page)
    d = k_pages.shape[3]
    k_pages.view(-1, d)[flat] = k_pages.view(-1, d)[index]
    v_pages.view(-1, d)[flat] = v_pages.view(-1, d)[index]
    weight.view(-1)[flat] = weight.view(-1)[index]
    pos.view(-1)[flat] = pos.view(-1)[index]
    return left


def _run_plain(s):
    case = s["case"]
    if case["op"] == "rotary":
        sign = -1.0 if case["grad"] else 1.0
        return {x: _plain_rotary(s[x], s["positions"], s["inv_freq"], s["sections"], sign) for x in ("q", "k")}
    if case["op"] == "append":
        lens, _, _ = _plain_append(s["k_pages"], s["v_pages"], s["k"], s["v"], s["table"], s["lens"], s["starts"])
        return {"k": s["k_pages"], "v": s["v_pages"], "lens": lens}
    if case["op"] == "attend":
        out = _plain_attend(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["sm_scale"], case["n"],
                            s.get("weight"))
        return {"out": out, "weight": s["weight"]} if case["weights"] else {"out": out}
    if case["op"] == "evict":
        lens = _plain_evict(s["k_pages"], s["v_pages"], s["weight"], s["pos"], s["table"], s["lens"],
                            case["budget"], case["n"], s["spare"], s["dst_table"])
    else:
        n = case["budget"] + 1
        positions = s["seen"][None]
        half = (case["d"] // 2,)
        q = _plain_rotary(s["q"], positions, s["inv_freq"], half, 1.0)
        k = _plain_rotary(s["k"], positions, s["inv_freq"], half, 1.0)
        starts = torch.arange(case["batch"] + 1, dtype=torch.int32, device=k.device)
        grown, where, _ = _plain_append(s["k_pages"], s["v_pages"], k, s["v"], s["table"], s["lens"], starts)
        s["weight"][where[0], :, where[1]] = 0.0
        s["pos"][where[0], :, where[1]] = s["seen"][:, None]
        out = _plain_attend(q, s["k_pages"], s["v_pages"], s["table"], grown, s["sm_scale"], n, s["weight"])
        lens = _plain_evict(s["k_pages"], s["v_pages"], s["weight"], s["pos"], s["table"], grown, case["budget"], n,
                            s["spare"])
        s["seen"] += 1
    r = {"k": s["k_pages"], "v": s["v_pages"], "weight": s["weight"], "pos": s["pos"], "lens": lens}
    if case["op"] == "step":
        r["out"] = out
    return r


# -----------------------------------------------------------------------------------------------
# the framework's calls
# -----------------------------------------------------------------------------------------------
def _run_own(s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import paged_cache as pc
    case = s["case"]
    if case["op"] == "rotary":
        call = pc.rotary_grad if case["grad"] else pc.rotary
        q, k = call(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"])
        return {"q": q, "k": k}
    if "cache" not in s:                                   # a program keeps its cache
        s["cache"] = pc.PagedCache(s["k_pages"], s["v_pages"], s.get("weight"), s.get("pos"))
    cache = s["cache"]
    if case["op"] == "append":
        lens = pc.cache_append(cache, s["k"], s["v"], s["table"], s["lens"], s["starts"])
        return {"k": cache.k, "v": cache.v, "lens": lens}
    if case["op"] == "attend":
        out = pc.paged_attention(s["q"], cache, s["table"], s["lens"], s["sm_scale"], accumulate=case["weights"],
                                 max_len=case["n"])
        return {"out": out, "weight": cache.weight} if case["weights"] else {"out": out}
    if case["op"] == "evict":
        lens = pc.cache_evict(cache, s["table"], s["lens"], case["budget"], N_GLOBAL, N_LOCAL, s["dst_table"],
                              max_len=case["n"])
    else:
        n = case["budget"] + 1
        q, k = pc.rotary(s["q"], s["k"], s["seen"][None], s["inv_freq"])
        grown = pc.cache_append(cache, k, s["v"], s["table"], s["lens"], seen=s["seen"])
        out = pc.paged_attention(q, cache, s["table"], grown, s["sm_scale"], accumulate=True, max_len=n)
        lens = pc.cache_evict(cache, s["table"], grown, case["budget"], N_GLOBAL, N_LOCAL, max_len=n)
        s["seen"] += 1
    r = {"k": cache.k, "v": cache.v, "weight": cache.weight, "pos": cache.pos, "lens": lens}
    if case["op"] == "step":
        r["out"] = out
    return r


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -----------------------------------------------------------------------------------------------
# what a pass cannot do without
# -----------------------------------------------------------------------------------------------
def work(case):
    e, heads, kv, d = SIZES[case["dtype"]], case["heads"], case["kv_heads"], case["d"]
    row = 2 * kv * d * e                                   # a token's keys and values
    if case["op"] == "rotary":
        t = case["tokens"]
        return {"bytes": 2 * t * (heads + kv) * d * e + 4 * t * case["axes"] + 2 * d,
                "flops": 3 * t * (heads + kv) * d}
    if case["op"] == "append":
        return {"bytes": 2 * sum(_new_counts(case)) * row, "flops": 0}
    if case["op"] == "attend":
        keys, q = sum(_lens(case)), case["q"]
        table = 4 * sum(_pages(n, case["page"]) for n in _lens(case))
        extra = 8 * kv * keys if case["weights"] else 0
        return {"bytes": keys * row + 2 * case["batch"] * heads * q * d * e + extra + table,
                "flops": 4 * keys * heads * q * d}
    if case["op"] == "evict":
        lens = _lens(case)
        left = sum(min(n, case["budget"]) for n in lens)
        return {"bytes": 8 * kv * sum(lens) + 2 * left * (row + 8 * kv), "flops": 0}
    keys = case["batch"] * (case["budget"] + 1)            # weights read and written, positions read
    return {"bytes": keys * row + 12 * kv * keys + case["batch"] * (4 * heads * d * e + 6 * row),
            "flops": 4 * keys * heads * d}


# -----------------------------------------------------------------------------------------------
# the definitions in 64 bits
# -----------------------------------------------------------------------------------------------
def _exact_rotary(x, positions, inv_freq, sections, inverse):
    x64, half = x.double(), x.shape[-1] // 2
    out = torch.empty_like(x64)
    first = 0
    for axis, count in enumerate(sections):
        for i in range(first, first + count):
            angle = positions[axis].double() * float(inv_freq[i])
            turn = torch.polar(torch.ones_like(angle), -angle if inverse else angle)[:, None]
            z = torch.complex(x64[..., i], x64[..., half + i]) * turn
            out[..., i], out[..., half + i] = z.real, z.imag
        first += count
    return out


def _exact_rows(pages, table_row, n):
    """(kv, n, ...) of a sequence's first n keys, from its pages in order."""
    page = pages.shape[2]
    ids = table_row[:_pages(n, page)].long()
    x = pages[ids].transpose(0, 1)
    return x.reshape(x.shape[0], -1, *x.shape[3:])[:, :n]


def _exact_attend(q, k_pages, v_pages, table, lens, sm_scale, weight):
    q4 = (q if q.dim() == 4 else q[:, :, None]).double()
    batch, heads, nq, d = q4.shape
    kv, page = k_pages.shape[1], k_pages.shape[2]
    out = torch.zeros_like(q4)
    drawn = None if weight is None else weight.double()
    for b, n in enumerate(lens):
        if n == 0:
            continue
        for h in range(kv):
            k = _exact_rows(k_pages[:, h:h + 1], table[b], n)[0].double()
            v = _exact_rows(v_pages[:, h:h + 1], table[b], n)[0].double()
            for i in range(nq):
                sees = n - (nq - 1 - i)
                if sees <= 0:
                    continue
                group = slice(h * (heads // kv), (h + 1) * (heads // kv))
                p = torch.softmax(q4[b, group, i] @ k[:sees].t() * sm_scale, dim=-1)
                out[b, group, i] = p @ v[:sees]
                if drawn is not None:
                    total = torch.zeros(_pages(n, page) * page, dtype=torch.float64, device=q.device)
                    total[:sees] = p.sum(dim=0)
                    drawn[table[b, :_pages(n, page)].long(), h] += total.view(-1, page)
    return out.reshape(q.shape), drawn


def _exact_evict(fields, table, lens, budget, dst_table):
    """fields: k, v, weight, pos pages, the weight in 64 bits; changed in place."""
    k_pages, v_pages, weight, pos = fields
    kv, page = k_pages.shape[1], k_pages.shape[2]
    for b, n in enumerate(lens):
        if n == 0 or (n <= budget and dst_table is None):
            continue
        for h in range(kv):
            w = _exact_rows(weight[:, h:h + 1], table[b], n)[0].tolist()
            p = _exact_rows(pos[:, h:h + 1], table[b], n)[0].tolist()
            last = max(p)
            by = sorted(range(n), key=lambda j: (not (p[j] < N_GLOBAL or p[j] > last - N_LOCAL), -w[j], j)
                        if not (p[j] < N_GLOBAL or p[j] > last - N_LOCAL) else (False, 0.0, j))
            kept = sorted(by[:budget])
            if dst_table is None:
                inside = set(kept)
                src = [j for j in kept if j >= budget]
                dst, target = [j for j in range(budget) if j not in inside], table
            else:
                src, dst, target = kept, list(range(len(kept))), dst_table
            src, dst = torch.tensor(src, device=pos.device), torch.tensor(dst, device=pos.device)
            if src.numel():
                a, c = table[b, src // page].long(), target[b, dst // page].long()
                for x in (k_pages, v_pages, weight, pos):
                    x[c, h, dst % page] = x[a, h, src % page]
    return None


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return {x: _exact_rotary(s[x], s["positions"], s["inv_freq"], s["sections"], case["grad"])
                for x in ("q", "k")}
    if case["op"] == "append":
        lens, new, page = _lens(case), _new_counts(case), case["page"]
        for name in ("k", "v"):
            at = 0
            for b, n in enumerate(new):
                j = torch.arange(lens[b], lens[b] + n, device="cuda")
                pages = s[name + "_pages"]
                pages[s["table"][b, j // page].long(), :, j % page] = s[name][at:at + n]
                at += n
        return {"k": s["k_pages"].double(), "v": s["v_pages"].double(), "lens": None}
    if case["op"] == "attend":
        lens = _lens(case)
        if sum(lens) * case["kv_heads"] > (1 << 23) or len(lens) * case["kv_heads"] * case["q"] > 20000:
            return None                                    # long in 64 bits
        out, drawn = _exact_attend(s["q"], s["k_pages"], s["v_pages"], s["table"], lens, s["sm_scale"],
                                   s.get("weight"))
        return {"out": out, "weight": drawn} if case["weights"] else {"out": out}
    out = None
    if case["op"] == "evict":
        lens, weight = _lens(case), s["weight"].double()
    else:
        half, budget, page = (case["d"] // 2,), case["budget"], case["page"]
        # the attention is defined on the queries and keys as the cache's type holds them
        q = _exact_rotary(s["q"], s["seen"][None], s["inv_freq"], half, False).to(s["q"].dtype)
        k = _exact_rotary(s["k"], s["seen"][None], s["inv_freq"], half, False).to(s["k"].dtype)
        lens = [budget + 1] * case["batch"]
        last = s["table"][:, budget // page].long()
        s["k_pages"][last, :, budget % page] = k
        s["v_pages"][last, :, budget % page] = s["v"]
        s["weight"][last, :, budget % page] = 0.0
        s["pos"][last, :, budget % page] = s["seen"][:, None]
        out, weight = _exact_attend(q, s["k_pages"], s["v_pages"], s["table"], lens, s["sm_scale"], s["weight"])
    _exact_evict((s["k_pages"], s["v_pages"], weight, s["pos"]), s["table"], lens, case["budget"],
                 s.get("dst_table"))
    if case["op"] == "step":                               # its pages hold rounded keys: no value in 64 bits
        return {"k": None, "v": None, "weight": weight, "pos": None, "lens": None, "out": out}
    return {"k": s["k_pages"].double(), "v": s["v_pages"].double(), "weight": weight, "pos": None, "lens": None}
