"""The paged-cache operators in 64 bits from their definitions, for tests: loops over sequences, heads
and queries on host tensors."""
import torch


def rotary(x, positions, inv_freq, sections, pos_scale=1.0, rope_scale=1.0, inverse=False):
    """(rotated, |pair| sums): x (T, H, D); the second is what an error of the sine or cosine scales with."""
    x = x.double().cpu()
    half = sum(sections)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    out, size = x.clone(), torch.zeros_like(x)
    for i in range(half):
        angle = positions[axis[i]].double().cpu() * float(torch.tensor(pos_scale)) * float(inv_freq[i])
        c, s = torch.cos(angle)[:, None] * rope_scale, torch.sin(angle)[:, None] * rope_scale
        s = -s if inverse else s
        a, b = x[..., i], x[..., half + i]
        out[..., i], out[..., half + i] = a * c - b * s, b * c + a * s
        size[..., i] = size[..., half + i] = (a.abs() + b.abs()) * abs(rope_scale)
    return out, size


def keys_of(pages, table_row, n, page_size, h):
    """(rows (n, ...) of head h, exists (n,)): keys whose table entry is no page are zeros."""
    rows = torch.zeros((n, *pages.shape[3:]), dtype=torch.float64)
    exists = torch.zeros(n, dtype=torch.bool)
    for j0 in range(0, n, page_size):
        p = int(table_row[j0 // page_size])
        if 0 <= p < pages.shape[0]:
            m = min(page_size, n - j0)
            rows[j0:j0 + m] = pages[p, h, :m].double().cpu()
            exists[j0:j0 + m] = True
    return rows, exists


def attend(q, k_pages, v_pages, table, lens, sm_scale, cap):
    """out (B, H, Q, D), lse (B, H, Q), drawn: per (b, kv head) the (len,) weights, and bounds for a
    tolerance: reach (B, H, Q, D) = sum_j p_j |v_j|, score = max_j sm_scale sum_d |q_d k_jd| per row."""
    B, H, Q, D = q.shape
    Hkv, ps = k_pages.shape[1], k_pages.shape[2]
    G = H // Hkv
    out, reach = torch.zeros((B, H, Q, D), dtype=torch.float64), torch.zeros((B, H, Q, D), dtype=torch.float64)
    lse = torch.full((B, H, Q), float("-inf"), dtype=torch.float64)
    score = torch.zeros((B, H, Q), dtype=torch.float64)
    drawn = {}
    q = q.double().cpu()
    for b in range(B):
        n = min(max(int(lens[b]), 0), cap)
        for h in range(Hkv):
            k, exists = keys_of(k_pages, table[b], n, ps, h)
            v, _ = keys_of(v_pages, table[b], n, ps, h)
            total = torch.zeros(n, dtype=torch.float64)
            for g in range(G):
                for i in range(Q):
                    sees = n - (Q - 1 - i)
                    at = torch.nonzero(exists[:max(sees, 0)]).flatten()
                    if at.numel() == 0:
                        continue
                    row = q[b, h * G + g, i]
                    s = k[at] @ row * sm_scale
                    if float(s.max()) == float("-inf"):
                        continue
                    p = torch.softmax(s, 0)
                    out[b, h * G + g, i] = p @ v[at]
                    reach[b, h * G + g, i] = p @ v[at].abs()
                    lse[b, h * G + g, i] = torch.logsumexp(s, 0)
                    score[b, h * G + g, i] = (k[at].abs() @ row.abs()).max() * abs(sm_scale)
                    total[at] += p
            drawn[b, h] = total
    return out, lse, drawn, reach, score


def evict_order(weight, pos, exists, n_global, n_local):
    """The keys of one head in the order in which they stay."""
    n = len(weight)
    live = [pos[j] for j in range(n) if exists[j]]
    last = max(live) if live else 0

    def rank(j):
        if not exists[j]:
            return (3, 0.0, j)
        if pos[j] < n_global or pos[j] > last - n_local:
            return (0, 0.0, j)
        return (1, 0.0, j) if weight[j] != weight[j] else (2, -weight[j], j)
    return sorted(range(n), key=rank)


def evict(k, v, weight, pos, table, lens, budget, n_global, n_local, cap, dst_table=None):
    """Host copies (k, v, weight, pos, lens) after the eviction."""
    k, v, weight, pos = (x.detach().cpu().clone() for x in (k, v, weight, pos))
    k0, v0, w0, p0 = (x.clone() for x in (k, v, weight, pos))
    ps, pages, left = k.shape[2], k.shape[0], []
    for b in range(table.shape[0]):
        n = min(max(int(lens[b]), 0), cap)
        m = min(n, budget)
        left.append(m)
        if m == 0 or (dst_table is None and n <= budget):
            continue
        row = [int(x) for x in table[b]]
        there = [0 <= row[j // ps] < pages for j in range(n)]
        for h in range(k.shape[1]):
            w = [float(w0[row[j // ps], h, j % ps]) if there[j] else 0.0 for j in range(n)]
            p = [int(p0[row[j // ps], h, j % ps]) if there[j] else 0 for j in range(n)]
            kept = sorted(evict_order(w, p, there, n_global, n_local)[:m])
            if dst_table is None:
                inside = set(kept)
                moves = list(zip([j for j in kept if j >= m], [j for j in range(m) if j not in inside]))
                to = row
            else:
                moves = list(zip(kept, range(m)))
                to = [int(x) for x in dst_table[b]]
            for src, dst in moves:
                a, c = row[src // ps], to[dst // ps]
                if not there[src] or not 0 <= c < pages:
                    continue
                for x, x0 in ((k, k0), (v, v0), (weight, w0), (pos, p0)):
                    x[c, h, dst % ps] = x0[a, h, src % ps]
    return k, v, weight, pos, torch.tensor(left, dtype=torch.int32)
