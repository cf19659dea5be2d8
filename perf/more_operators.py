"""Operators of layers with normed heads, sliding windows and shared prefixes, as cases whose time and
outputs can be measured.

A model of this kind norms each head of its queries and keys before it rotates them, attends in most of
its layers over a window of the latest keys and a few first ones (sinks), and is served to many users
whose requests begin with the same long text.  It is trained with packed sequences of different lengths.

    listed()            the fixed cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs on the GPU, as a program has them before the call
    run(state)          one pass; its outputs (own: through the framework, else in plain torch)
    work(case)          bytes and operations that the pass cannot do without
    exact(case, seed)   the same outputs in float64, written from the definitions

Packed tensors are (tokens, heads, dim); sequence b's tokens are starts[b] .. starts[b + 1] - 1.  Pages are
(page, kv head, slot, dim); a sequence's key j lies in page table[b, j // page_size], slot j % page_size.
Unused table entries are -1.  A query at position p sees key j <= p if j > p - window or j < sinks.
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
EPS = 1e-6
NEG = float("-inf")


def _case(name, op, dtype, heads, kv_heads, d, **kw):
    c = {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "d": d}
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # norm and rotation of one decoding step: a new token of each of 16 sequences
        _case("norm_rotary_step", "norm_rotary", "bf16", 32, 8, 128, tokens=16, rotated=128, weight="bf16", grad=False),
        # the same of a prompt, half of each head rotated, norm weights kept in fp32
        _case("norm_rotary_prompt", "norm_rotary", "fp16", 32, 8, 128, tokens=8191, rotated=64, weight="fp32",
              grad=False),
        # its gradient in a training step, the norm weights' among them
        _case("norm_rotary_grad", "norm_rotary", "bf16", 32, 8, 128, tokens=16384, rotated=128, weight="bf16",
              grad=True),
        # a training step's attention in a layer with a window: packed sequences of different lengths
        _case("window_train", "window", "bf16", 32, 8, 128, batch=5, tokens=8192, window=1024, sinks=4, train=True,
              shape=1),
        # the same in a layer that sees everything, one head a kv head, small heads
        _case("causal_train", "window", "fp16", 24, 24, 64, batch=3, tokens=6001, window=0, sinks=0, train=True,
              shape=2),
        # a long prompt through a layer with a window
        _case("window_prompt", "window", "bf16", 32, 8, 128, batch=1, tokens=8192, window=4096, sinks=128, train=False,
              shape=3),
        # a small fp32 model's step over short sequences: latency counts
        _case("window_fp32", "window", "fp32", 8, 8, 64, batch=4, tokens=1000, window=100, sinks=1, train=True,
              shape=4),
        # a decoding step of a layer with a window: long and short conversations in one batch
        _case("decode_window", "decode", "bf16", 32, 8, 128, batch=48, n=65536, q=1, page=16, window=4096, sinks=16,
              shape=5),
        # one user's step, two tokens checked at once: latency counts
        _case("decode_window_one", "decode", "fp16", 32, 8, 128, batch=1, n=2000, q=2, page=32, window=1000, sinks=4,
              shape=6),
        # a decoding step of a batch behind one long system text
        _case("prefix_batch", "prefix", "bf16", 32, 8, 128, batch=64, prefix=16384, n=1024, q=1, page=16, shape=7),
        # questions about one long document
        _case("prefix_long", "prefix", "fp16", 16, 8, 128, batch=8, prefix=131072, n=300, q=1, page=64, shape=8),
        # a few tokens a sequence checked at once behind a short system text
        _case("prefix_draft", "prefix", "bf16", 40, 8, 64, batch=12, prefix=2000, n=500, q=4, page=16, shape=9),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rotary", "window", "window", "window", "decode", "prefix", "prefix"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    heads, kv_heads = rng.choice([(32, 8), (32, 32), (16, 2), (40, 8), (8, 8), (28, 4), (24, 1), (12, 12)])
    d = rng.choice([128, 128, 64])
    page = rng.choice([8, 16, 32, 64, 128, 256])
    shape = rng.randrange(1, 1 << 20)
    row = kv_heads * d * SIZES[dtype] * 2                  # bytes of a token's keys and values
    if op == "norm_rotary":
        most = (16384 * 40 * 128 * 2) // ((heads + kv_heads) * d * SIZES[dtype])
        return _case(None, op, dtype, heads, kv_heads, d, tokens=_log_int(rng, 1, most),
                     rotated=rng.choice([d, d, d // 2]), weight=rng.choice([dtype, "fp32"]), grad=rng.random() < 0.5)
    if op == "window":
        # with 32 heads a product of two fp32 matrices of 8192 rows is the largest listed one
        most = math.sqrt(8192 * 8192 * 32 / heads) * (0.5 if dtype == "fp32" else 1.0)
        tokens = _log_int(rng, 64, min(8192, int(most)))
        return _case(None, op, dtype, heads, kv_heads, d, batch=_log_int(rng, 1, 8), tokens=tokens,
                     window=rng.choice([0, _log_int(rng, 1, tokens)]), sinks=rng.choice([0, 1, 4, _log_int(rng, 1, 200)]),
                     train=rng.random() < 0.7, shape=shape)
    if op == "decode":
        n = _log_int(rng, 16, min((1 << 30) // row, 65536))
        batch = _log_int(rng, 1, max(1, min(64, (2 << 30) // (row * n))))
        window = _log_int(rng, 1, max(2, min(n, 4096, (256 << 20) // (row * batch))))
        return _case(None, op, dtype, heads, kv_heads, d, batch=batch, n=n, q=rng.choice([1, 1, 1, 2, 5, 16]), page=page,
                     window=window, sinks=rng.choice([0, 4, _log_int(rng, 1, 200)]), shape=shape)
    q = rng.choice([1, 1, 1, 2, 5])
    prefix = _log_int(rng, 16, min((512 << 20) // row, 131072))
    batch = _log_int(rng, 1, max(1, min(64, (1 << 29) // (prefix * heads * q))))
    n = _log_int(rng, q, max(q + 1, min(2048, (512 << 20) // (row * batch))))
    return _case(None, op, dtype, heads, kv_heads, d, batch=batch, prefix=prefix, n=n, q=q, page=page, shape=shape)


# -----------------------------------------------------------------------------------------------
# shapes that a case stands for
# -----------------------------------------------------------------------------------------------
def _lens(case):
    """Lengths up to n: the longest first, the others spread over their logarithm, one of a batch of more
    than 8 with nothing but its new tokens."""
    n, batch = case["n"], case["batch"]
    rng = random.Random(case["shape"])
    lens = [n] + [min(n, _log_int(rng, max(1, n // 64), n)) for _ in range(batch - 1)]
    if batch > 8:
        lens[batch // 2] = 1
    return [max(x, case["q"]) for x in lens]


def _starts(case):
    """tokens shared out among the sequences unevenly; an empty one in a batch of more than 4."""
    rng = random.Random(case["shape"])
    share = [math.exp(rng.uniform(0.0, 2.0)) for _ in range(case["batch"])]
    if len(share) > 4:
        share[2] = 0.0
    starts, total, run_ = [0], sum(share), 0.0
    for x in share:
        run_ += x
        starts.append(int(round(case["tokens"] * run_ / total)))
    return starts


def _pages(tokens, page):
    return -(-tokens // page)


def _pairs(n, window, sinks):
    """Pairs of query and key in a sequence of n tokens."""
    if not window or window >= n:
        return n * (n + 1) // 2
    total = 0
    for p in range(n):
        lo = max(p - window + 1, 0)
        total += p + 1 - lo + min(sinks, lo)
    return total


# -----------------------------------------------------------------------------------------------
# inputs
# -----------------------------------------------------------------------------------------------
def _randn(g, shape, dtype, scale=1.0):
    x = torch.randn(shape, generator=g, device="cuda", dtype=dtype)
    return x.mul_(scale) if scale != 1.0 else x


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(need, width, page_ids):
    """A table (batch, width): need[b] pages of the shuffled page_ids each, -1 behind them."""
    free = iter(page_ids.tolist())
    return _int32([[next(free) for _ in range(n)] + [-1] * (width - n) for n in need])


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    dtype, heads, kv, d = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["d"]
    s = {"case": case, "sm_scale": 1.0 / math.sqrt(d)}
    if case["op"] == "norm_rotary":
        t, half = case["tokens"], case["rotated"] // 2
        s["q"], s["k"] = _randn(g, (t, heads, d), dtype, 3.0), _randn(g, (t, kv, d), dtype, 3.0)
        w = DTYPES[case["weight"]]
        s["q_weight"] = (1.0 + 0.2 * _randn(g, (d,), torch.float32)).to(w)
        s["k_weight"] = (1.0 + 0.2 * _randn(g, (d,), torch.float32)).to(w)
        s["positions"] = torch.randint(0, 131072, (t,), generator=g, device="cuda", dtype=torch.int32)
        s["inv_freq"] = (1.0 / THETA ** (torch.arange(half, dtype=torch.float64) / half)).float().cuda()
        if case["grad"]:
            s["dq"], s["dk"] = _randn(g, (t, heads, d), dtype), _randn(g, (t, kv, d), dtype)
        return s
    if case["op"] == "window":
        t = case["tokens"]
        s["q"] = _randn(g, (t, heads, d), dtype, 2.0)      # scores of standard deviation 2
        s["k"], s["v"] = _randn(g, (t, kv, d), dtype), _randn(g, (t, kv, d), dtype)
        s["starts"] = _int32(_starts(case))
        if case["train"]:
            for x in "qkv":
                s[x].requires_grad_()
            s["dout"] = _randn(g, (t, heads, d), dtype)
        return s
    page, lens = case["page"], _lens(case)
    need, first = [_pages(n, page) for n in lens], _pages(case.get("prefix", 0), page)
    pages = sum(need) + first + 3
    ids = torch.randperm(pages, generator=cpu).to(torch.int32)
    s["k_pages"] = _randn(g, (pages, kv, page, d), dtype)
    s["v_pages"] = _randn(g, (pages, kv, page, d), dtype)
    s["table"] = _tables(need, max(need), ids)
    s["lens"] = _int32(lens)
    s["q"] = _randn(g, (len(lens), heads, d) if case["q"] == 1 else (len(lens), heads, case["q"], d), dtype, 2.0)
    if case["op"] == "prefix":
        s["prefix"] = ids[sum(need):sum(need) + first].cuda()
    return s


# -----------------------------------------------------------------------------------------------
# plain forms: elementary torch operations in 32 bits (angles and long sums in 64)
# -----------------------------------------------------------------------------------------------
def _plain_turn(x, positions, inv_freq, sign):
    """The rotation of x (T, H, D) in fp32, elements behind the rotated ones as they are."""
    half = inv_freq.shape[0]
    angle = positions.double()[:, None] * inv_freq.double()
    c, s = angle.cos().float()[:, None], sign * angle.sin().float()[:, None]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], dim=-1)


def _plain_norm_rotary(x, weight, positions, inv_freq):
    f = x.float()
    r = torch.rsqrt((f * f).mean(dim=-1, keepdim=True) + EPS)
    return _plain_turn(f * r * weight.float(), positions, inv_freq, 1.0).to(x.dtype)


def _plain_norm_rotary_grad(dy, x, weight, positions, inv_freq):
    f = x.float()
    r = torch.rsqrt((f * f).mean(dim=-1, keepdim=True) + EPS)
    n = f * r
    dn = _plain_turn(dy.float(), positions, inv_freq, -1.0)
    dweight = (dn * n).sum(dim=(0, 1), dtype=torch.float64)
    dn = dn * weight.float()
    dx = r * (dn - n * (dn * n).mean(dim=-1, keepdim=True))
    return dx.to(x.dtype), dweight.to(weight.dtype)


def _plain_packed(starts, t):
    """Sequence and position of each of t packed tokens."""
    i = torch.arange(t, device=starts.device, dtype=torch.int32)
    b = torch.searchsorted(starts, i, right=True) - 1
    return b, i - starts[b]


def _plain_softmax_(s):
    """Softmax over the last dim, in place; rows without a key become zeros."""
    m = s.amax(dim=-1, keepdim=True)
    s.sub_(torch.where(m == NEG, 0.0, m)).exp_()
    return s.div_(s.sum(dim=-1, keepdim=True).clamp(min=1e-30))


def _plain_window(q, k, v, starts, window, sinks, sm_scale, dout=None):
    t, heads, d = q.shape
    kv = k.shape[1]
    group = heads // kv
    b, p = _plain_packed(starts, t)
    sees = (b[:, None] == b) & (p[:, None] >= p)
    if window:
        sees &= (p > p[:, None] - window) | (p < sinks)
    # (kv heads, group * T, D): a kv head's rows as one matrix
    rows = q.float().view(t, kv, group, d).permute(1, 2, 0, 3).reshape(kv, group * t, d)
    kf, vf = k.float().transpose(0, 1).contiguous(), v.float().transpose(0, 1).contiguous()
    prob = (rows @ kf.transpose(1, 2).contiguous()).mul_(sm_scale)
    prob.view(kv, group, t, t).masked_fill_(~sees, NEG)
    _plain_softmax_(prob)

    def packed(x, n):                                      # (kv, n * T, D) back to (T, kv * n, D)
        return x.view(kv, n, t, d).permute(2, 0, 1, 3).reshape(t, kv * n, d).to(q.dtype)
    out = packed(prob @ vf, group)
    if dout is None:
        return {"out": out}
    do = dout.float().view(t, kv, group, d).permute(1, 2, 0, 3).reshape(kv, group * t, d)
    dv = prob.transpose(1, 2) @ do
    dp = do @ vf.transpose(1, 2).contiguous()
    dp.sub_((dp * prob).sum(dim=-1, keepdim=True)).mul_(prob)
    dq = (dp @ kf).mul_(sm_scale)
    dk = (dp.transpose(1, 2) @ rows).mul_(sm_scale)
    return {"out": out, "dq": packed(dq, group), "dk": packed(dk, 1), "dv": packed(dv, 1)}


def _plain_keys(pages, table, index):
    """(B, Hkv, n, D) fp32: keys index (B, n) of each sequence; entries without a page point to page 0."""
    page = pages.shape[2]
    at = table.gather(1, (index // page).long()).long().clamp(min=0)
    return pages[at, :, (index % page).long()].float().transpose(1, 2)


def _plain_rows(q, kv):
    """q (B, H[, Q], D) as fp32 (B, Hkv, rows, D)."""
    return q.float().reshape(q.shape[0], kv, -1, q.shape[-1])


def _plain_ends(lens, nq):
    return lens[:, None] - torch.arange(nq - 1, -1, -1, device=lens.device)      # (B, nq): keys a query sees


def _plain_decode(s, case):
    q, lens, kv, nq = s["q"], s["lens"], case["kv_heads"], case["q"]
    window, sinks, n = case["window"], case["sinks"], case["n"]
    lo = (lens - (nq - 1) - window).clamp(min=0)                                 # the first query's window begins here
    first = lo.clamp(max=sinks)[:, None]
    u = torch.arange(min(n, window + nq - 1 + sinks), device=q.device, dtype=torch.int32)
    j = torch.where(u < first, u, u - first + lo[:, None])                       # (B, keys)
    k = _plain_keys(s["k_pages"], s["table"], j.clamp(max=n - 1))
    v = _plain_keys(s["v_pages"], s["table"], j.clamp(max=n - 1))
    end = _plain_ends(lens, nq)[:, :, None]
    sees = (j[:, None] < end) & ((j[:, None] >= end - window) | (j[:, None] < sinks))
    prob = (_plain_rows(q, kv) @ k.transpose(2, 3).contiguous()).mul_(s["sm_scale"])
    prob.view(len(lens), kv, -1, nq, u.shape[0]).masked_fill_(~sees[:, None, None], NEG)
    return {"out": (_plain_softmax_(prob) @ v).reshape(q.shape).to(q.dtype)}


def _plain_prefix(s, case):
    q, lens, kv, nq, d = s["q"], s["lens"], case["kv_heads"], case["q"], case["d"]
    batch, n, n0 = len(lens), case["n"], case["prefix"]
    j = torch.arange(max(n, n0), device=q.device, dtype=torch.int32)
    kp, vp = (_plain_keys(s[x], s["prefix"][None], j[None, :n0])[0] for x in ("k_pages", "v_pages"))
    ks, vs = (_plain_keys(s[x], s["table"], j[:n].expand(batch, -1)) for x in ("k_pages", "v_pages"))
    rows = _plain_rows(q, kv)                                                    # (B, Hkv, R, D)
    shared = rows.transpose(0, 1).reshape(kv, -1, d) @ kp.transpose(1, 2).contiguous()
    shared = shared.view(kv, batch, -1, n0).transpose(0, 1)
    tail = rows @ ks.transpose(2, 3).contiguous()
    sees = j[None, None, :n] < _plain_ends(lens, nq)[:, :, None]
    tail.view(batch, kv, -1, nq, n).masked_fill_(~sees[:, None, None], NEG)
    prob = _plain_softmax_(torch.cat([shared, tail], dim=-1).mul_(s["sm_scale"]))
    out = prob[..., :n0].transpose(0, 1).reshape(kv, -1, n0) @ vp
    out = out.view(kv, batch, -1, d).transpose(0, 1) + prob[..., n0:].contiguous() @ vs
    return {"out": out.reshape(q.shape).to(q.dtype)}


@torch.no_grad()
def _run_plain(s):
    case = s["case"]
    if case["op"] == "norm_rotary":
        out = {}
        for x in ("q", "k"):
            how = (s[x], s[x + "_weight"], s["positions"], s["inv_freq"])
            if case["grad"]:
                out["d" + x], out[f"d{x}_weight"] = _plain_norm_rotary_grad(s["d" + x], *how)
            else:
                out[x] = _plain_norm_rotary(*how)
        return out
    if case["op"] == "window":
        return _plain_window(s["q"], s["k"], s["v"], s["starts"], case["window"], case["sinks"], s["sm_scale"],
                             s.get("dout"))
    return _plain_decode(s, case) if case["op"] == "decode" else _plain_prefix(s, case)


# -----------------------------------------------------------------------------------------------
# the framework's calls
# -----------------------------------------------------------------------------------------------
def _run_own(s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    case = s["case"]
    if case["op"] == "window":
        import window_attention as wa
        out = wa.window_attention(s["q"], s["k"], s["v"], window=case["window"] or None, sinks=case["sinks"],
                                  starts=s["starts"], sm_scale=s["sm_scale"])
        if not case["train"]:
            return {"out": out}
        dq, dk, dv = torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    import paged_cache as pc
    if case["op"] == "norm_rotary":
        how = (s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["inv_freq"])
        if not case["grad"]:
            q, k = pc.norm_rotary(*how, eps=EPS)
            return {"q": q, "k": k}
        dq, dk, dq_weight, dk_weight = pc.norm_rotary_grad(s["dq"], s["dk"], *how, eps=EPS)
        return {"dq": dq, "dk": dk, "dq_weight": dq_weight, "dk_weight": dk_weight}
    if "cache" not in s:                                   # a program keeps its cache
        s["cache"] = pc.PagedCache(s["k_pages"], s["v_pages"])
    if case["op"] == "decode":
        return {"out": pc.paged_attention(s["q"], s["cache"], s["table"], s["lens"], s["sm_scale"],
                                          max_len=case["n"], window=case["window"], sinks=case["sinks"])}
    return {"out": pc.prefix_attention(s["q"], s["cache"], s["prefix"], case["prefix"], s["table"], s["lens"],
                                       s["sm_scale"], max_len=case["n"])}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -----------------------------------------------------------------------------------------------
# what a pass cannot do without
# -----------------------------------------------------------------------------------------------
def work(case):
    e, heads, kv, d = SIZES[case["dtype"]], case["heads"], case["kv_heads"], case["d"]
    if case["op"] == "norm_rotary":
        t, moved = case["tokens"], 3 if case["grad"] else 2
        return {"bytes": moved * t * (heads + kv) * d * e + 4 * t + 2 * case["rotated"]
                + 2 * d * SIZES[case["weight"]] * (moved - 1),
                "flops": (20 if case["grad"] else 8) * t * (heads + kv) * d}
    if case["op"] == "window":
        t, starts = case["tokens"], _starts(case)
        pairs = sum(_pairs(b - a, case["window"], case["sinks"]) for a, b in zip(starts, starts[1:]))
        q, k = t * heads * d * e, t * kv * d * e
        if not case["train"]:
            return {"bytes": 2 * q + 2 * k, "flops": 4 * pairs * heads * d}
        # q, k, v and dout read; out, dq, dk, dv written
        return {"bytes": 4 * q + 4 * k, "flops": 14 * pairs * heads * d}
    row, nq, lens = 2 * kv * d * e, case["q"], _lens(case)
    io = 2 * len(lens) * heads * nq * d * e
    if case["op"] == "decode":
        # the keys that any query of a sequence sees, and the pairs
        keys = pairs = 0
        for n in lens:
            lo = max(n - (nq - 1) - case["window"], 0)
            keys += n - lo + min(case["sinks"], lo)
            for i in range(nq):
                end = n - (nq - 1 - i)
                lo = max(end - case["window"], 0)
                pairs += end - lo + min(case["sinks"], lo)
        return {"bytes": keys * row + io, "flops": 4 * pairs * heads * d}
    pairs = sum(nq * (case["prefix"] + n) - nq * (nq - 1) // 2 for n in lens)
    return {"bytes": (sum(lens) + case["prefix"]) * row + io, "flops": 4 * pairs * heads * d}


# -----------------------------------------------------------------------------------------------
# the definitions in 64 bits
# -----------------------------------------------------------------------------------------------
def _exact_norm_rotary(x, weight, positions, inv_freq):
    half = inv_freq.shape[0]
    n = x * weight / torch.sqrt(x.square().sum(dim=-1, keepdim=True) / x.shape[-1] + EPS)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device),
                       positions.double()[:, None, None] * inv_freq.double())
    z = torch.complex(n[..., :half], n[..., half:2 * half]) * turn
    return torch.cat([z.real, z.imag, n[..., 2 * half:]], dim=-1)


def _exact_one_head(q, k, v, window, sinks, sm_scale, behind=0):
    """out of q (n, D) whose row i is at position behind + i over k, v (m, D)."""
    p = torch.arange(q.shape[0], device=q.device)[:, None] + behind
    j = torch.arange(k.shape[0], device=q.device)
    hidden = j > p
    if window:
        hidden |= (j <= p - window) & (j >= sinks)
    return torch.softmax((q @ k.t() * sm_scale).masked_fill(hidden, NEG), dim=-1) @ v


def _exact_rows(pages, table_row, index):
    """Keys index of a sequence, (Hkv, n, D) in 64 bits."""
    page = pages.shape[2]
    return pages[table_row[index // page].long(), :, index % page].double().transpose(0, 1)


def exact(case, seed):
    s = prepare(case, seed)
    heads, kv, d = case["heads"], case["kv_heads"], case["d"]
    if case["op"] == "norm_rotary":
        out = {}
        for x in ("q", "k"):
            x64, w64 = s[x].double(), s[x + "_weight"].double()
            if not case["grad"]:
                out[x] = _exact_norm_rotary(x64, w64, s["positions"], s["inv_freq"])
                continue
            y = _exact_norm_rotary(x64.requires_grad_(), w64.requires_grad_(), s["positions"], s["inv_freq"])
            out["d" + x], out[f"d{x}_weight"] = torch.autograd.grad(y, (x64, w64), s["d" + x].double())
        return out
    if case["op"] == "window":
        starts = _starts(case)
        q, k, v = (s[x].detach().double() for x in "qkv")
        out = torch.zeros_like(q)
        grads = [torch.zeros_like(x) for x in (q, k, v)]
        for a, b in zip(starts, starts[1:]):
            if a == b:
                continue
            for h in range(heads):
                hk = h // (heads // kv)
                qh, kh, vh = q[a:b, h], k[a:b, hk], v[a:b, hk]
                if not case["train"]:
                    out[a:b, h] = _exact_one_head(qh, kh, vh, case["window"], case["sinks"], s["sm_scale"])
                    continue
                qh, kh, vh = (x.clone().requires_grad_() for x in (qh, kh, vh))
                y = _exact_one_head(qh, kh, vh, case["window"], case["sinks"], s["sm_scale"])
                out[a:b, h] = y.detach()
                for total, at, dx in zip(grads, (h, hk, hk), torch.autograd.grad(y, (qh, kh, vh),
                                                                               s["dout"][a:b, h].double())):
                    total[a:b, at] += dx
        return {"out": out, "dq": grads[0], "dk": grads[1], "dv": grads[2]} if case["train"] else {"out": out}
    lens, nq = _lens(case), case["q"]
    q = (s["q"] if case["q"] > 1 else s["q"][:, :, None]).double()
    out = torch.zeros_like(q)
    if case["op"] == "prefix":
        at = torch.arange(case["prefix"], device=q.device)
        kp, vp = _exact_rows(s["k_pages"], s["prefix"], at), _exact_rows(s["v_pages"], s["prefix"], at)
        if case["batch"] * heads * nq * case["prefix"] > (1 << 29):
            return None                                    # long in 64 bits
    for b, n in enumerate(lens):
        at = torch.arange(n, device=q.device)
        window, sinks = case.get("window", 0), case.get("sinks", 0)
        if window and n > window + nq + sinks:             # what no query sees
            at = torch.cat([at[:sinks], at[max(n - nq - window, sinks):]])
        k, v = _exact_rows(s["k_pages"], s["table"][b], at), _exact_rows(s["v_pages"], s["table"][b], at)
        for h in range(kv):
            group = slice(h * (heads // kv), (h + 1) * (heads // kv))
            end = n - torch.arange(nq - 1, -1, -1, device=q.device)[:, None]
            hidden = at >= end
            if window:
                hidden |= (at < end - window) & (at >= sinks)
            kh, vh = k[h], v[h]
            if case["op"] == "prefix":
                kh, vh = torch.cat([kp[h], kh]), torch.cat([vp[h], vh])
                hidden = torch.cat([torch.zeros((nq, case["prefix"]), dtype=torch.bool, device=q.device), hidden], dim=1)
            x = (q[b, group].reshape(-1, d) @ kh.t() * s["sm_scale"]).view(-1, nq, kh.shape[0])
            out[b, group] = torch.softmax(x.masked_fill(hidden, NEG), dim=-1) @ vh
    return {"out": out.reshape(s["q"].shape)}
