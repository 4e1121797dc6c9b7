"""The sequence operators in 64 bits, from their formulas, with a bound on
the error of a computation in fp32 whose second products, as the bf16 path's,
round p and ds to the type, and whose results are rounded to it.

A bound follows the computation: a rounding to type T is off by at most
eps(T)/2 relative, a sum of n terms in fp32 by n*u times the sum of their
magnitudes (u = 2^-24), an exponential by its argument's error relative.
"""

import math

import torch

U = 2.0 ** -24
# the hardware's exponential gives zero for results under the smallest normal
# number, so a gate's small side can be off by this much, absolutely
TINY = 2.0 ** -126


def bucket(distance, buckets, max_distance):
    """One distance's bucket, in whole numbers."""
    half = buckets // 2
    exact = half // 2
    wide = half - exact
    n = min(abs(distance), max_distance)
    b = n
    if n >= exact:
        b = exact + max(m for m in range(wide)
                        if n ** wide >= exact ** (wide - m)
                        * max_distance ** m)
    return b + half if distance > 0 else b


def attention(q, k, v, lengths=None, table=None, key_step=1, query_start=0,
              max_distance=128, scale=None, dout=None):
    """(results, bounds), dicts of out and, with dout, dq, dk, dv, dtable."""
    eps = torch.finfo(q.dtype).eps / 2
    half = eps if q.dtype == torch.bfloat16 else 0.0   # of p and ds
    N, H, E, Lq = q.shape
    Hkv, Lk = k.size(1), k.size(3)
    G = H // Hkv
    dev = q.device
    scale = 1 / math.sqrt(E) if scale is None else scale
    q, k, v = q.detach().double(), k.detach().double(), v.detach().double()
    bias = torch.zeros(H, Lq, Lk, dtype=torch.float64, device=dev)
    ids = None
    if table is not None:
        kinds = {d: bucket(d, table.size(1), max_distance)
                 for d in range(-max_distance, max_distance + 1)}
        lut = torch.tensor([kinds[d] for d in sorted(kinds)], device=dev)
        d = (torch.arange(Lk, device=dev)[None] * key_step
             - torch.arange(Lq, device=dev)[:, None] - query_start)
        ids = lut[d.clamp(-max_distance, max_distance) + max_distance]
        bias = table.detach().double()[:, ids]
        bias = torch.where(bias <= -1e30, -math.inf, bias)
    res = {"out": torch.zeros_like(q)}
    err = {"out": torch.zeros_like(q)}
    if dout is not None:
        dout = dout.detach().double()
        for c, t in (("dq", q), ("dk", k), ("dv", v)):
            res[c], err[c] = torch.zeros_like(t), torch.zeros_like(t)
        if table is not None:
            res["dtable"] = torch.zeros(table.shape, dtype=torch.float64,
                                        device=dev)
            err["dtable"] = res["dtable"].clone()
    for n in range(N):
        cnt = Lk if lengths is None else max(0, min(int(lengths[n]), Lk))
        if cnt == 0:
            continue
        for h in range(H):
            g = h // G
            qi, ki, vi = q[n, h].t(), k[n, g, :, :cnt], v[n, g, :, :cnt]
            b = bias[h, :, :cnt]
            s = qi @ ki * scale
            ds_ = ((E + 8) * U * (qi.abs() @ ki.abs()) * scale
                   + 8 * U * (s.abs() + b.nan_to_num(neginf=0.0).abs()))
            s = s + b
            top = s.amax(-1, keepdim=True)
            empty = top == -math.inf
            p = torch.exp(s - torch.where(empty, 0.0, top))
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            p = torch.where(empty, 0.0, p)
            # relative error of p: its own score's, the sum's, the joint
            # logarithm's rounding
            rp = (2 * ds_.amax(-1, keepdim=True) + (cnt + 16) * U
                  + 4 * U * torch.where(empty, 0.0, top).abs())
            va = p @ vi.abs().t()
            o = p @ vi.t()
            eo = va * (rp + half + (cnt + 16) * U)
            res["out"][n, h] = o.t()
            err["out"][n, h] = (eo + (eo + o.abs()) * eps).t()
            if dout is None:
                continue
            do = dout[n, h].t()
            dp = do @ vi
            delta = (p * dp).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            edp = (E + 4) * U * (do.abs() @ vi.abs())
            edelta = (do.abs() * (eo + (eo + o.abs()) * eps)).sum(
                -1, keepdim=True) * 1.01
            eds = p * ((dp - delta).abs() * (rp + 4 * U) + edp + edelta)
            rds = eds + half * (eds + ds.abs())
            dq = ds @ ki.t() * scale
            edq = (rds + (cnt + 8) * U * ds.abs()) @ ki.abs().t() * scale
            res["dq"][n, h] = dq.t()
            err["dq"][n, h] = (edq + (edq + dq.abs()) * eps).t()
            rows = G * Lq + 64
            dv = do.t() @ p
            edv = do.abs().t() @ (p * (rp + half + rows * U))
            res["dv"][n, g, :, :cnt] += dv
            err["dv"][n, g, :, :cnt] += edv
            dk = qi.t() @ ds * scale
            edk = qi.abs().t() @ (rds + rows * U * ds.abs()) * scale
            res["dk"][n, g, :, :cnt] += dk
            err["dk"][n, g, :, :cnt] += edk
            if table is not None:
                # a bf16 table's ds come from a delta of their own p and dp
                if half:
                    eds = p * ((dp - delta).abs() * (rp + 4 * U) + edp
                               + (p * (dp.abs() * (rp + cnt * U) + edp)).sum(
                                   -1, keepdim=True))
                eds = eds + (N * Lq + cnt) * U * ds.abs()
                for c in range(table.size(1)):
                    m = (ids[:, :cnt] == c).double()
                    res["dtable"][h, c] += (ds * m).sum()
                    err["dtable"][h, c] += (eds * m).sum()
    for c in ("dk", "dv", "dtable"):
        if c in res:
            err[c] = err[c] + (err[c] + res[c].abs()) * eps
    return res, err


def scan(x, gate, state=None, lengths=None, reverse=False, dh=None,
         dstate=None):
    """(results, bounds), dicts of h, state and, with dh or dstate, dx, dgate
    and dstate."""
    eps = torch.finfo(x.dtype).eps / 2
    N, C, L = x.shape
    f64 = {"dtype": torch.float64, "device": x.device}
    x, gate = x.detach().double(), gate.detach().double()
    h0 = torch.zeros(N, C, **f64) if state is None else state.double()
    count = [L] * N if lengths is None else \
        [max(0, min(int(i), L)) for i in lengths]
    live = torch.tensor([[t < c for t in range(L)] for c in count],
                        device=x.device)[:, None, :].expand(N, C, L)
    a = torch.where(live, torch.sigmoid(gate), 1.0)
    keep = torch.where(live, torch.sigmoid(-gate), 0.0)
    x = torch.where(live, x, 0.0)
    grad = dh is not None or dstate is not None
    d = torch.zeros_like(x) if dh is None else torch.where(live, dh.double(),
                                                           0.0)
    order = list(range(L))[::-1] if reverse else list(range(L))
    # a and keep are within 6 roundings, a composed map passes at most 40
    # compositions, and a state never exceeds the largest |x| or |h0|
    most = torch.maximum(x.abs().amax(-1), h0.abs())
    h, e = h0, torch.zeros_like(h0)
    hs, es, before, ebefore = ([None] * L for _ in range(4))
    for t in order:
        before[t], ebefore[t] = h, e
        e = a[..., t] * e + 6 * U * (a[..., t] * h.abs()
                                     + keep[..., t] * x[..., t].abs()) \
            + TINY * (h.abs() + x[..., t].abs())
        h = a[..., t] * h + keep[..., t] * x[..., t]
        hs[t], es[t] = h, e
    tree = 40 * U * most
    hs = torch.where(live, torch.stack(hs, -1), 0.0)
    es = torch.where(live, torch.stack(es, -1) + tree[..., None], 0.0)
    res = {"h": hs, "state": h}
    err = {"h": es + (es + hs.abs()) * eps, "state": e + tree + U * h.abs()}
    if not grad:
        return res, err
    u = torch.zeros(N, C, **f64) if dstate is None else dstate.double()
    ua, e = u.abs(), torch.zeros_like(u)
    out = {c: [None] * L for c in ("dx", "dgate", "ex", "eg")}
    for t in order[::-1]:
        at, kt = a[..., t], keep[..., t]
        g = d[..., t] + u
        ga = d[..., t].abs() + ua
        eg = e + 46 * U * ga
        out["dx"][t] = kt * g
        out["ex"][t] = kt * (eg + 8 * U * ga) + TINY * ga
        diff = before[t] - x[..., t]
        ediff = ebefore[t] + tree + U * (before[t].abs() + x[..., t].abs())
        out["dgate"][t] = g * diff * at * kt
        out["eg"][t] = at * kt * (eg * diff.abs() + ga * ediff
                                  + 20 * U * ga * diff.abs()) \
            + TINY * ga * diff.abs()
        e = at * (e + 6 * U * ga) + TINY * ga
        u, ua = at * g, at * ga
    for c, name in (("dx", "ex"), ("dgate", "eg")):
        r = torch.where(live, torch.stack(out[c], -1), 0.0)
        b = torch.where(live, torch.stack(out[name], -1), 0.0)
        res[c], err[c] = r, b + (b + r.abs()) * eps
    res["dstate"], err["dstate"] = u, e + 46 * U * ua
    return res, err


def assert_within(got, want, bound, what):
    got, want = got.detach().double(), want.to(got.device)
    assert got.shape == want.shape, what
    over = (got - want).abs() - bound.to(got.device) - 1e-37
    worst = over.max().item() if over.numel() else -1.0
    assert worst <= 0, f"{what}: {worst} over its bound"
    assert not torch.isnan(got).any(), what
