"""The gated recurrence in 64 bits over long records, with the bounds of
_sequence_ref.scan: those are linear recurrences with the same gates, and all
of them are walked here block by block, many blocks at once.
"""

import math

import torch

from _sequence_ref import TINY, U


def walk(a, b, first):
    """y_t = a_t y_(t-1) + b_t along the last axis of (R, L), from ``first``:
    (y before each step, y after each step)."""
    r, length = a.shape
    size = math.isqrt(length - 1) + 1
    more = -length % size
    a = torch.nn.functional.pad(a, (0, more), value=1.0).view(r, -1, size)
    b = torch.nn.functional.pad(b, (0, more)).view(r, -1, size)
    end_a, end_b = torch.ones_like(a[..., 0]), torch.zeros_like(b[..., 0])
    for t in range(size):
        end_a, end_b = a[..., t] * end_a, a[..., t] * end_b + b[..., t]
    starts, y = [], first
    for c in range(a.size(1)):
        starts.append(y)
        y = end_a[:, c] * y + end_b[:, c]
    y, ys = torch.stack(starts, 1), []
    for t in range(size):
        ys.append(y)
        y = a[..., t] * y + b[..., t]
    before = torch.stack(ys, -1).view(r, -1)
    after = torch.cat([before[:, 1:], y[:, -1:]], 1)
    return before[:, :length], after[:, :length]


def scan(x, gate, state, lengths, reverse, dh, dstate):
    """As _sequence_ref.scan, of which the lines are the steps."""
    eps = torch.finfo(x.dtype).eps / 2
    N, C, L = x.shape
    count = torch.full((N,), L) if lengths is None else \
        torch.as_tensor(lengths).cpu().clamp(0, L)
    live = (torch.arange(L)[None] < count[:, None]).to(x.device)
    live = live[:, None].expand(N, C, L).reshape(-1, L)

    def take(t):
        t = t.detach().double().reshape(-1, L)
        return turn(torch.where(live, t, 0.0))

    def turn(t):
        return t.flip(-1) if reverse else t

    def give(t):
        return torch.where(live, turn(t), 0.0).view(N, C, L)

    seen = turn(live)
    x, gate, d = take(x), take(gate), take(dh)
    a = torch.where(seen, torch.sigmoid(gate), 1.0)
    keep = torch.where(seen, torch.sigmoid(-gate), 0.0)
    h0 = state.detach().double().reshape(-1)
    zero = torch.zeros_like(h0)
    most = torch.maximum(x.abs().amax(-1), h0.abs())
    before, h = walk(a, keep * x, h0)
    own = (6 * U * (a * before.abs() + keep * x.abs())
           + TINY * (before.abs() + x.abs()))
    ebefore, e = walk(a, own, zero)
    tree = (40 * U * most)[:, None]
    es = e + tree
    res = {"h": give(h), "state": h[:, -1].view(N, C)}
    err = {"h": give(es + (es + h.abs()) * eps),
           "state": (e[:, -1] + tree[:, 0] + U * h[:, -1].abs()).view(N, C)}

    # u_t = a_t (d_t + u_(t+1)), walked from the last step
    ds = dstate.detach().double().reshape(-1)
    ar, dr = a.flip(-1), d.flip(-1)
    u0, u = (t.flip(-1) for t in walk(ar, ar * dr, ds))
    ua0, ua = (t.flip(-1) for t in walk(ar, ar * dr.abs(), ds.abs()))
    g, ga = d + u0, d.abs() + ua0
    own = a * 6 * U * ga + TINY * ga
    e0, e = (t.flip(-1) for t in walk(ar, own.flip(-1), zero))
    eg = e0 + 46 * U * ga
    diff = before - x
    ediff = ebefore + tree + U * (before.abs() + x.abs())
    dgate = g * diff * a * keep
    bound = {
        "dx": keep * (eg + 8 * U * ga) + TINY * ga,
        "dgate": a * keep * (eg * diff.abs() + ga * ediff
                             + 20 * U * ga * diff.abs())
        + TINY * ga * diff.abs()}
    for name, r in (("dx", keep * g), ("dgate", dgate)):
        res[name] = give(r)
        err[name] = give(bound[name] + (bound[name] + r.abs()) * eps)
    res["dstate"] = u[:, 0].view(N, C)
    err["dstate"] = (e[:, 0] + 46 * U * ua[:, 0]).view(N, C)
    return res, err
