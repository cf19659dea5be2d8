"""Attention with a sliding window and sinks and its gradients, in 64 bits from the definitions, for tests, with
bounds of what kernels that work in fp32 and round the probabilities and the scores' gradients once may be off.

u = 2^-24 and e = finfo.eps / 2 are half a step of fp32 and of the type.  S = sm_scale max_j sum_d |q_d k_jd|.
  p    a score is off by at most (D + 8) u S, the maximum or log-sum-exp that it is set against by as much and 8 u of itself,
       the sum over n keys by n + 64 roundings: p carries a factor within rp = (2 (D + 8) S + 8 (|lse| + 1) + n + 64) u of 1
  out  each p rounded once: (e + rp) R + e |out| with R = sum_j p_j |v_j|
  dv   (e + rp) sum_i p_ij |dout_i|, a sum of n products n u more, and e |dv|
  ds   p (dp - delta), dp a sum of D products, delta one of D products of out: out is off by (e + rp) R before its own rounding,
       which delta does not see but for 2 e^2 |out|.  So ds is off by rp |ds| + p (2 D u sum|dout| |v| + delta's error),
       and rounded once: e |ds|
  dq   sm_scale times the sum over j of ds's error times |k_j|, the sum's own n u, and e |dq|; dk likewise over the rows
fp16's subnormal probabilities (below 2^-14 of 2^-7 of the maximum) add 2^-31 of the largest |v|, |dout| a key or row; its ds,
scaled to below 2^14, half a step of the subnormals, 2^-25, of that scale.
"""
import torch

U = 2.0 ** -24


def spans(starts, total):
    if starts is None:
        return [(0, total)]
    s = [min(max(int(x), 0), total) for x in starts]
    return list(zip(s, s[1:]))


def visible(nq, nk, window, sinks, device):
    p = torch.arange(nq, device=device)[:, None] + (nk - nq)
    j = torch.arange(nk, device=device)[None]
    sees = j <= p
    if window is not None:
        sees = sees & ((j > p - window) | (j < sinks))
    return sees


def attention(q, k, v, window, sinks, starts, k_starts, sm_scale, dout=None):
    """{name: (value, bound)} of out, lse (T, H), and with dout of dq, dk and dv, in float64 on q's device."""
    dtype, dev = q.dtype, q.device
    e = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    half = dtype == torch.float16
    (T, H, D), Hkv = q.shape, k.shape[1]
    q, k, v = q.detach().double(), k.detach().double(), v.detach().double()
    out, lse = torch.zeros_like(q), torch.full((T, H), float("-inf"), dtype=torch.float64, device=dev)
    r = {"out": (out, torch.zeros_like(out)), "lse": (lse, torch.zeros_like(lse))}
    if dout is not None:
        do = dout.double()
        r.update(dq=(torch.zeros_like(q), torch.zeros_like(q)), dk=(torch.zeros_like(k), torch.zeros_like(k)),
                 dv=(torch.zeros_like(v), torch.zeros_like(v)))
        grow = 1.0
        if half:
            most = 2 * do.norm(dim=-1).max() * v.norm(dim=-1).max()
            grow = 2.0 ** (13 - torch.floor(torch.log2(most.clamp(min=1e-30))).item())
    for (a, b), (c, d) in zip(spans(starts, T), spans(k_starts if k_starts is not None else starts, k.shape[0])):
        nq, nk = b - a, d - c
        if nq <= 0 or nk <= 0:
            continue
        sees = visible(nq, nk, window, sinks, dev)
        some = sees.any(dim=1)
        for h in range(H):
            hk = h // (H // Hkv)
            qh, kh, vh = q[a:b, h], k[c:d, hk], v[c:d, hk]
            s = (qh @ kh.t() * sm_scale).masked_fill(~sees, float("-inf"))
            l = torch.logsumexp(s, dim=1)
            l = torch.where(some, l, torch.zeros_like(l))
            p = torch.exp(s - l[:, None]).masked_fill(~sees, 0.0)
            S = ((qh.abs() @ kh.abs().t()) * abs(sm_scale)).masked_fill(~sees, 0.0).amax(dim=1)
            rp = ((2 * (D + 8) * S + 8 * (l.abs() + 1) + nk + 64) * U)[:, None]
            o, R = p @ vh, p @ vh.abs()
            low = nk * 2.0 ** -31 * vh.abs().max() if half else 0.0
            out[a:b, h] = o
            r["out"][1][a:b, h] = ((e + rp) * R + low) * (1 + 2 * e) + e * o.abs() + tiny
            lse[a:b, h] = torch.where(some, l, torch.full_like(l, float("-inf")))
            r["lse"][1][a:b, h] = rp[:, 0]
            if dout is None:
                continue
            g = do[a:b, h]
            low_do = nq * 2.0 ** -31 * g.abs().max() if half else 0.0
            R_do = p.t() @ g.abs()
            dv = p.t() @ g
            r["dv"][0][c:d, hk] += dv
            r["dv"][1][c:d, hk] += (p * (e + rp + nq * (H // Hkv) * U)).t() @ g.abs() + low_do + 0 * R_do
            dp, delta = g @ vh.t(), (g * o).sum(dim=1, keepdim=True)
            ds = p * (dp - delta)
            delta_err = (g.abs() * ((e + rp) * R + low + 2 * e * e * o.abs() + 4 * D * U * o.abs())).sum(dim=1, keepdim=True)
            err = (e + rp) * ds.abs() + p * (2 * D * U * (g.abs() @ vh.abs().t()) + delta_err)
            err = err.masked_fill(~sees, 0.0) + (sees * 2.0 ** -25 / grow if half else 0.0)
            r["dq"][0][a:b, h] = ds @ kh * sm_scale
            r["dq"][1][a:b, h] = (err + (nk + 64) * U * ds.abs()) @ kh.abs() * abs(sm_scale)
            r["dk"][0][c:d, hk] += ds.t() @ qh * sm_scale
            r["dk"][1][c:d, hk] += (err + (nq * (H // Hkv) + 64) * U * ds.abs()).t() @ qh.abs() * abs(sm_scale)
    for name in ("dq", "dk", "dv"):
        if name in r:
            value, bound = r[name]
            r[name] = (value, bound * (1 + 2 * e) + e * value.abs() + tiny)
    return r
