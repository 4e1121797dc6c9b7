"""Cases for the sequence operators: attention to the states of another
length, with or without a learned position bias, and the gated linear
recurrence.

``run`` computes a case with elementary torch operations in 32 bits, or,
where ``own`` is true, with the framework's operators. Tensors are
channels-first as everywhere in the framework: (N, H, E, L) and (N, C, L).
"""

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp32": 4}

# the largest drawn cases stay under the largest listed ones
MAX_SCORES = 1 << 30
MAX_PRODUCTS = 1 << 37
MAX_SAMPLES = 100 * 64 * 8192


def _attend(name, n, h, hkv, e, lq, lk, dtype="bf16", train=False,
            ragged=False, buckets=0, key_step=1, max_distance=0,
            query_start=0):
    return {"name": name, "op": "attend", "n": n, "h": h, "hkv": hkv, "e": e,
            "lq": lq, "lk": lk, "dtype": dtype, "train": train,
            "ragged": ragged, "buckets": buckets, "key_step": key_step,
            "max_distance": max_distance, "query_start": query_start}


def _scan(name, n, c, length, dtype="bf16", train=False, ragged=False,
          reverse=False):
    return {"name": name, "op": "scan", "n": n, "c": c, "l": length,
            "dtype": dtype, "train": train, "ragged": ragged,
            "reverse": reverse}


def listed():
    return [
        # one new query against stored states, four query heads to a key head
        _attend("attend_one_query", 16, 8, 2, 64, 1, 4096),
        # one query, its position told by the bias, records of any length
        _attend("attend_one_query_bias", 8, 12, 12, 32, 1, 2000, ragged=True,
                buckets=32, max_distance=128, query_start=1777),
        # full-rate queries on keys pooled by 16: the attention of the
        # backbone's first stage, with positions
        _attend("attend_pooled_bias", 64, 3, 3, 8, 2048, 128, buckets=32,
                key_step=16, max_distance=512),
        # a long record on itself, heads of 16 as in the backbone
        _attend("attend_record", 4, 6, 6, 16, 8192, 8192),
        # training on records of different lengths, one of them empty
        _attend("attend_train_ragged", 32, 8, 8, 32, 1024, 1024, train=True,
                ragged=True),
        # the same in full precision, odd sizes, shared heads, with positions
        _attend("attend_train_fp32_bias", 6, 6, 3, 24, 777, 501, "fp32",
                train=True, buckets=32, max_distance=200),
        # training with positions, keys at half the queries' rate
        _attend("attend_train_bias", 8, 8, 8, 64, 2048, 1000, train=True,
                ragged=True, buckets=32, key_step=2, max_distance=128),
        # the widest heads, shared by four: the largest products
        _attend("attend_train_wide", 4, 16, 4, 128, 4096, 4096, train=True),
        # a sample at a time, as a running stream is answered
        _scan("scan_one_sample", 64, 96, 1),
        # the recurrent stage of a picker: 64 steps, full precision, both
        # directions are run, here the backward one, padded records
        _scan("scan_train_short", 500, 16, 64, "fp32", train=True,
              ragged=True, reverse=True),
        # a batch of the benchmark's windows in training
        _scan("scan_train_windows", 100, 64, 8192, train=True),
        # one continuous record, odd length, in training
        _scan("scan_train_record", 1, 24, 1000003, "fp32", train=True),
    ]


def _spread(rng, low, high):
    """A whole number, spread evenly over its logarithm."""
    return min(high, int(math.exp(rng.uniform(math.log(low),
                                              math.log(high + 1)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    train = rng.random() < 0.6
    ragged = rng.random() < 0.4
    if rng.random() < 0.4:
        length = _spread(rng, 1, 1000003)
        c = _spread(rng, 1, 128)
        n = max(1, min(_spread(rng, 1, 512), MAX_SAMPLES // (c * length)))
        c = max(1, min(c, MAX_SAMPLES // (n * length)))
        return {k: v for k, v in _scan(
            "", n, c, length, dtype, train, ragged,
            rng.random() < 0.4).items() if k != "name"}
    hkv = rng.choice([1, 2, 3, 4, 6, 8])
    h = hkv * rng.choice([1, 1, 1, 2, 4])
    e = rng.choice([8, 16, 24, 32, 32, 48, 64, 64, 80, 96, 128])
    lq = 1 if rng.random() < 0.2 else _spread(rng, 1, 8192)
    # a softmax over very few keys, or a bias all in one bucket, has gradients
    # that are nothing but rounding
    lk = _spread(rng, 16 if train else 1, 8192)
    most = MAX_SCORES if train else 2 * MAX_SCORES
    most = min(most, (MAX_PRODUCTS if dtype == "bf16" else MAX_PRODUCTS >> 4)
               // e)
    n = max(1, min(_spread(rng, 1, 64), most // (h * lq * lk)))
    if n * h * lq * lk > most:
        lq = max(1, most // (n * h * lk))
    buckets, max_distance = 0, 0
    if rng.random() < 0.5:
        buckets = rng.choice([8, 16, 32, 64])
        max_distance = _spread(rng, buckets, 1024)
    return {k: v for k, v in _attend(
        "", n, h, hkv, e, lq, lk, dtype, train, ragged, buckets,
        rng.choice([1, 1, 2, 3, 16]), max_distance,
        rng.choice([0, 0, 0 if train else rng.randrange(lk)])).items()
        if k != "name"}


def _lengths(count, full):
    """Valid lengths of a padded batch, from none of it to all."""
    return [full * ((7 * i + 4) % 11) // 10 for i in range(count)]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dtype, scale=1.0, shift=0.0, leaf=False):
        t = torch.randn(*shape, device=DEV, generator=g)
        t = t.mul_(scale).add_(shift).to(dtype)
        return t.requires_grad_(leaf and case["train"])

    s = {"case": case, "lengths": None}
    n = case["n"]
    if case["op"] == "attend":
        h, hkv, e = case["h"], case["hkv"], case["e"]
        s["q"] = normal(n, h, e, case["lq"], leaf=True)
        s["k"] = normal(n, hkv, e, case["lk"], leaf=True)
        s["v"] = normal(n, hkv, e, case["lk"], leaf=True)
        s["table"] = None
        if case["buckets"]:
            s["table"] = normal(h, case["buckets"], leaf=True)
        if case["train"]:
            s["dout"] = normal(n, h, e, case["lq"])
        full = case["lk"]
    else:
        c, full = case["c"], case["l"]
        s["x"] = normal(n, c, full, leaf=True)
        # gates that remember from one sample to some hundreds
        s["gate"] = normal(n, c, full, scale=2.0, shift=2.0, leaf=True)
        s["state"] = normal(n, c, dtype=torch.float32, leaf=True)
        if case["train"]:
            s["dh"] = normal(n, c, full)
            s["dstate"] = normal(n, c, dtype=torch.float32)
    if case["ragged"]:
        s["lengths"] = torch.tensor(_lengths(n, full), dtype=torch.int32,
                                    device=DEV)
    return s


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------


def _own_attend(s):
    from seist_amd import ops
    case = s["case"]
    more = {}
    if s["table"] is not None:
        more = {"bias_table": s["table"], "key_step": case["key_step"],
                "query_start": case["query_start"],
                "max_distance": case["max_distance"]}
    out = ops.cross_attention(s["q"], s["k"], s["v"],
                              kv_lengths=s["lengths"], **more)
    if not case["train"]:
        return {"out": out}
    leaves = [t for t in (s["q"], s["k"], s["v"], s["table"])
              if t is not None]
    grads = torch.autograd.grad(out, leaves, s["dout"])
    return dict(zip(("out", "dq", "dk", "dv", "dtable"),
                    (out.detach(),) + grads))


def _own_scan(s):
    from seist_amd import ops
    case = s["case"]
    h, state = ops.gated_scan(s["x"], s["gate"], s["state"],
                              lengths=s["lengths"], reverse=case["reverse"])
    if not case["train"]:
        return {"h": h, "state": state}
    grads = torch.autograd.grad(
        [h, state], [s["x"], s["gate"], s["state"]], [s["dh"], s["dstate"]])
    return dict(zip(("h", "state", "dx", "dgate", "dstate"),
                    (h.detach(), state.detach()) + grads))


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _thresholds(buckets, max_distance):
    """Distances at which a side's buckets after the exact ones begin:
    exact * (max_distance / exact) ** (m / wide), in whole numbers."""
    exact = buckets // 4
    wide = buckets // 2 - exact
    found = []
    for m in range(1, wide):
        least = exact ** (wide - m) * max_distance ** m
        t = exact
        while t ** wide < least:
            t += 1
        found.append(t)
    return exact, found


def _bucket_ids(case):
    i = torch.arange(case["lq"], device=DEV)
    j = torch.arange(case["lk"], device=DEV)
    far = j[None, :] * case["key_step"] - (i[:, None] + case["query_start"])
    exact, found = _thresholds(case["buckets"], case["max_distance"])
    near = far.abs()
    log = exact + torch.bucketize(
        near, torch.tensor(found, dtype=torch.int64, device=DEV), right=True)
    return (torch.where(near < exact, near, log)
            + (far > 0) * (case["buckets"] // 2))


def _plain_attend(s):
    case = s["case"]
    n, h, hkv, e = (case[c] for c in ("n", "h", "hkv", "e"))
    lq, lk = case["lq"], case["lk"]
    with torch.no_grad():
        # the query heads that share keys stand side by side: (N, Hkv, G*Lq)
        g = h // hkv

        def rows(t):
            t = t.float().reshape(n * hkv, g, e, lq).transpose(2, 3)
            return t.reshape(n * hkv, g * lq, e)

        def back(t, dtype):
            t = t.reshape(n * hkv, g, lq, e).transpose(2, 3)
            return t.reshape(n, h, e, lq).to(dtype)

        q = rows(s["q"])
        k = s["k"].float().reshape(n * hkv, e, lk)
        v = s["v"].float().reshape(n * hkv, e, lk)
        scale = 1.0 / math.sqrt(e)
        score = torch.bmm(q, k).mul_(scale).view(n, h, lq, lk)
        if s["table"] is not None:
            ids = _bucket_ids(case)
            score += s["table"].float()[:, ids]
        if s["lengths"] is not None:
            hidden = (torch.arange(lk, device=DEV)[None, :]
                      >= s["lengths"][:, None])[:, None, None, :]
            score.masked_fill_(hidden, -torch.inf)
        most = score.amax(-1, keepdim=True)
        most.masked_fill_(most == -torch.inf, 0.0)
        p = score.sub_(most).exp_()
        p /= p.sum(-1, keepdim=True).clamp_min_(1e-30)
        p = p.view(n * hkv, g * lq, lk)
        out = torch.bmm(p, v.transpose(1, 2).contiguous())
        outs = {"out": back(out, s["q"].dtype)}
        if not case["train"]:
            return outs
        dout = rows(s["dout"])
        dv = torch.bmm(dout.transpose(1, 2).contiguous(), p)
        ds = torch.bmm(dout, v)
        ds -= (ds * p).sum(-1, keepdim=True)
        ds *= p
        dq = torch.bmm(ds, k.transpose(1, 2).contiguous()) * scale
        dk = torch.bmm(q.transpose(1, 2).contiguous(), ds) * scale
        outs["dq"] = back(dq, s["q"].dtype)
        outs["dk"] = dk.view(n, hkv, e, lk).to(s["k"].dtype)
        outs["dv"] = dv.view(n, hkv, e, lk).to(s["v"].dtype)
        if s["table"] is not None:
            total = ds.view(n, h, lq, lk).sum(0)
            outs["dtable"] = torch.stack(
                [(total * (ids == b)).sum((1, 2))
                 for b in range(case["buckets"])], 1).to(s["table"].dtype)
        return outs


def _prefix(a, b):
    """h_t = a_t h_(t-1) + b_t from h = 0, by doubling along the last
    axis."""
    step, length = 1, a.size(-1)
    while step < length:
        nb, na = b.clone(), a.clone()
        nb[..., step:] += a[..., step:] * b[..., :-step]
        na[..., step:] *= a[..., :-step]
        a, b, step = na, nb, 2 * step
    return b


def _plain_scan(s):
    case = s["case"]
    with torch.no_grad():
        x, gate, state = s["x"].float(), s["gate"].float(), s["state"]
        dtype = s["x"].dtype
        valid = None
        if s["lengths"] is not None:
            valid = (torch.arange(case["l"], device=DEV)[None, :]
                     < s["lengths"][:, None])[:, None, :]

        def turn(t):
            return t.flip(-1) if case["reverse"] else t

        def kept(t, other=0.0):
            return t if valid is None else torch.where(valid, t, other)

        a = turn(kept(1 / (1 + torch.exp(-gate)), 1.0))
        keep = turn(kept(1 / (1 + torch.exp(gate))))
        x = turn(kept(x))
        b = keep * x
        b[..., 0] += a[..., 0] * state
        h = _prefix(a, b)
        outs = {"h": kept(turn(h)).to(dtype), "state": h[..., -1].clone()}
        if not case["train"]:
            return outs
        dh = turn(kept(s["dh"].float())).clone()
        dh[..., -1] += s["dstate"]
        after = torch.cat([a[..., 1:], torch.zeros_like(a[..., :1])], -1)
        grad = _prefix(after.flip(-1), dh.flip(-1)).flip(-1)
        before = torch.cat([state[..., None], h[..., :-1]], -1)
        outs["dx"] = turn(keep * grad).to(dtype)
        outs["dgate"] = turn(grad * (before - x) * a * keep).to(dtype)
        outs["dstate"] = a[..., 0] * grad[..., 0]
        return outs


def run(state):
    if state["case"]["op"] == "attend":
        return _own_attend(state) if own else _plain_attend(state)
    return _own_scan(state) if own else _plain_scan(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    n, size = case["n"], SIZE[case["dtype"]]
    if case["op"] == "scan":
        full = case["l"]
        seen = sum(_lengths(n, full)) if case["ragged"] else n * full
        seen, every = case["c"] * seen, case["c"] * n * full
        moved, flops = 2 * seen + every, 8 * seen
        if case["train"]:
            moved, flops = moved + seen + 2 * every, flops + 12 * seen
        states = (4 if case["train"] else 2) * n * case["c"]
        return {"bytes": moved * size + 4 * states, "flops": flops}
    h, hkv, e, lq, lk = (case[c] for c in ("h", "hkv", "e", "lq", "lk"))
    seen = sum(_lengths(n, lk)) if case["ragged"] else n * lk
    queries, keys = n * h * e * lq, hkv * e * seen
    moved, flops = 2 * queries + 2 * keys, 4 * h * e * lq * seen
    if case["train"]:
        moved += 2 * queries + 2 * n * hkv * e * lk
        flops *= 3
    moved += h * case["buckets"] * (2 if case["train"] else 1)
    return {"bytes": moved * size, "flops": flops}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_bias(case, table):
    """The bias of every pair and the rows and columns of each bucket."""
    half = case["buckets"] // 2
    exact, most = half // 2, case["max_distance"]
    wide = half - exact
    of = []
    for d in range(most + 1):
        b = d
        if d >= exact:
            b = max(m for m in range(wide)
                    if d ** wide * exact ** m >= exact ** wide * most ** m)
            b += exact
        of.append(b)
    of = torch.tensor(of, device=DEV)
    i = torch.arange(case["lq"], device=DEV).view(-1, 1)
    j = torch.arange(case["lk"], device=DEV).view(1, -1)
    d = j * case["key_step"] - i - case["query_start"]
    ids = of[d.abs().clamp(max=most)]
    ids = torch.where(d > 0, ids + half, ids)
    return torch.index_select(table, 1, ids.flatten()).view(
        table.size(0), case["lq"], case["lk"]), ids


def _exact_attend(case, s):
    h, hkv, e = case["h"], case["hkv"], case["e"]
    lens = _lengths(case["n"], case["lk"]) if case["ragged"] \
        else [case["lk"]] * case["n"]
    q, k, v = (s[c].detach() for c in ("q", "k", "v"))
    table = s["table"]
    outs = {"out": torch.zeros(q.shape, dtype=torch.float64, device=DEV)}
    if case["train"]:
        outs.update({c: torch.zeros(s[c[1:]].shape, dtype=torch.float64,
                                    device=DEV) for c in ("dq", "dk", "dv")})
    bias = dbias = None
    if table is not None:
        bias, ids = _exact_bias(case, table.detach().double())
        dbias = torch.zeros_like(bias)
    for r, length in enumerate(lens):
        if length == 0:
            continue
        for one in range(hkv):
            heads = slice(one * (h // hkv), (one + 1) * (h // hkv))
            qr = q[r, heads].double().transpose(1, 2)          # (G, Lq, E)
            kr = k[r, one, :, :length].double()                # (E, len)
            vr = v[r, one, :, :length].double()
            z = torch.matmul(qr, kr) / e ** 0.5
            if bias is not None:
                z = z + bias[heads, :, :length]
            p = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
            out = torch.matmul(p, vr.t())                      # (G, Lq, E)
            outs["out"][r, heads] = out.transpose(1, 2)
            if not case["train"]:
                continue
            do = s["dout"][r, heads].double().transpose(1, 2)
            dz = p * (torch.matmul(do, vr)
                      - (do * out).sum(-1, keepdim=True))
            flat = (-1, length)
            outs["dv"][r, one, :, :length] = torch.matmul(
                do.reshape(-1, e).t(), p.reshape(flat))
            outs["dk"][r, one, :, :length] = torch.matmul(
                qr.reshape(-1, e).t(), dz.reshape(flat)) / e ** 0.5
            outs["dq"][r, heads] = (torch.matmul(dz, kr.t())
                                    / e ** 0.5).transpose(1, 2)
            if dbias is not None:
                dbias[heads, :, :length] += dz
    if case["train"] and table is not None:
        outs["dtable"] = torch.stack(
            [dbias[:, ids == b].sum(-1) for b in range(case["buckets"])], 1)
    return outs


def _exact_walk(a, b, first):
    """h_t = a_t h_(t-1) + b_t one step after another, many blocks at once:
    (R, L) in 64 bits, from ``first`` (R)."""
    r, length = a.shape
    block = max(1, math.isqrt(length))
    count = -(-length // block)
    more = count * block - length
    a = torch.nn.functional.pad(a, (0, more), value=1.0).view(r, count, block)
    b = torch.nn.functional.pad(b, (0, more), value=0.0).view(r, count, block)
    ends_a = torch.ones(r, count, dtype=torch.float64, device=DEV)
    ends_b = torch.zeros_like(ends_a)
    for t in range(block):
        ends_b = a[:, :, t] * ends_b + b[:, :, t]
        ends_a = a[:, :, t] * ends_a
    at = torch.empty_like(ends_a)
    now = first.double()
    for c in range(count):
        at[:, c] = now
        now = ends_a[:, c] * now + ends_b[:, c]
    h = torch.empty_like(a)
    for t in range(block):
        at = a[:, :, t] * at + b[:, :, t]
        h[:, :, t] = at
    return h.view(r, -1)[:, :length]


def _exact_scan(case, s):
    n, c, length = case["n"], case["c"], case["l"]
    back = case["reverse"]
    mask = torch.ones(n, 1, length, dtype=torch.bool, device=DEV)
    if case["ragged"]:
        for r, valid in enumerate(_lengths(n, length)):
            mask[r, :, valid:] = False
    mask = mask.expand(n, c, length).reshape(n * c, length)

    def take(t):
        t = t.detach().double().reshape(n * c, length) * mask
        return torch.flip(t, (1,)) if back else t

    def give(t):
        t = torch.flip(t, (1,)) if back else t
        return (t * mask).view(n, c, length)

    m = torch.flip(mask, (1,)) if back else mask
    a = torch.sigmoid(take(s["gate"]))
    a = torch.where(m, a, torch.ones_like(a))
    keep = torch.where(m, torch.sigmoid(-take(s["gate"])),
                       torch.zeros_like(a))
    x = take(s["x"])
    first = s["state"].detach().reshape(-1)
    h = _exact_walk(a, keep * x, first)
    outs = {"h": give(h), "state": h[:, -1].reshape(n, c)}
    if not case["train"]:
        return outs
    dh = take(s["dh"])
    dh[:, -1] += s["dstate"].reshape(-1)
    # from the last sample to the first: what arrives at t is a_(t+1) g_(t+1)
    shifted = torch.ones_like(a)
    shifted[:, :-1] = a[:, 1:]
    g = torch.flip(_exact_walk(torch.flip(shifted, (1,)),
                               torch.flip(dh, (1,)),
                               torch.zeros_like(first)), (1,))
    last = torch.empty_like(h)
    last[:, 0] = first
    last[:, 1:] = h[:, :-1]
    outs["dx"] = give(g * keep)
    outs["dgate"] = give(g * (last - x) * a * keep)
    outs["dstate"] = (a[:, 0] * g[:, 0]).reshape(n, c)
    return outs


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_attend(case, s) if case["op"] == "attend" \
            else _exact_scan(case, s)
