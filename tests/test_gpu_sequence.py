"""Attention to other lengths, its position bias and the gated recurrence:
the gfx950 kernels against their formulas in 64 bits, within the bounds that
follow from the computation's roundings."""

import math

import pytest
import torch

import _sequence_ref as ref
from seist_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, FP32 = torch.bfloat16, torch.float32


def _attention_inputs(n, h, hkv, e, lq, lk, buckets, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = [torch.randn(s, device=DEV, generator=g).to(dtype)
         for s in ((n, h, e, lq), (n, hkv, e, lk), (n, hkv, e, lk),
                   (n, h, e, lq))]
    table = None
    if buckets:
        table = torch.randn(h, buckets, device=DEV, generator=g).to(dtype)
    return t + [table]


def _check_attention(q, k, v, do, table, lens=None, **more):
    lens = None if lens is None else torch.tensor(lens, device=DEV,
                                                  dtype=torch.int32)
    with torch.no_grad():
        plain = ops.cross_attention(q, k, v, lens, table, **more)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, table)
              if t is not None]
    out = ops.cross_attention(leaves[0], leaves[1], leaves[2], lens,
                              leaves[3] if table is not None else None,
                              **more)
    grads = torch.autograd.grad(out, leaves, do)
    want, bound = ref.attention(q, k, v, lens, table, dout=do, **more)
    ref.assert_within(plain, want["out"], bound["out"], "out, no gradient")
    for name, got in zip(("out", "dq", "dk", "dv", "dtable"), (out,) + grads):
        assert got.dtype == q.dtype
        ref.assert_within(got, want[name], bound[name], name)
    return (out,) + grads


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n,h,hkv,e,lq,lk", [
    (2, 2, 2, 16, 64, 64),      # whole tiles
    (1, 1, 1, 1, 1, 1),         # the smallest of everything
    (2, 3, 3, 8, 33, 65),       # one past a tile on both sides
    (1, 4, 2, 24, 31, 63),      # one short of a tile, shared heads
    (2, 8, 2, 40, 1, 300),      # one query, four heads to a key head
    (1, 6, 1, 64, 5, 1000),     # 30 rows of six heads in one tile, split keys
    (1, 2, 1, 72, 130, 129),    # past a workgroup's rows, odd channels
    (1, 2, 2, 128, 200, 77),    # the widest heads
    (1, 2, 1, 96, 150, 300),
    (1, 1, 1, 97, 70, 200),
    (1, 1, 1, 33, 1, 2500),     # a long split of the keys
    (1, 1, 1, 17, 2500, 3),     # few keys: a long split of the queries
    (3, 33, 1, 8, 1, 40),       # 33 heads share a key head
    (8, 16, 16, 8, 1050, 100),  # few keys, rows enough for several a workgroup
    (8, 32, 16, 24, 600, 128),  # the same, across heads that share keys
])
def test_attention(dtype, n, h, hkv, e, lq, lk):
    _check_attention(*_attention_inputs(n, h, hkv, e, lq, lk, 0, dtype))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("n,h,hkv,e,lq,lk,buckets,more", [
    (1, 2, 2, 16, 40, 70, 8, dict(max_distance=20)),
    (2, 4, 2, 32, 100, 30, 32, dict(max_distance=128, key_step=4)),
    (1, 3, 1, 8, 7, 90, 16, dict(max_distance=40, query_start=33)),
    (1, 6, 2, 64, 1, 700, 32, dict(max_distance=128, query_start=699)),
    (1, 2, 2, 8, 256, 16, 64, dict(max_distance=1024, key_step=16)),
    (1, 1, 1, 128, 70, 200, 4, dict(max_distance=2, query_start=-50)),
    (1, 2, 1, 80, 65, 150, 6, dict(max_distance=1000, key_step=3)),
    (2, 2, 2, 16, 300, 500, 32, dict(max_distance=9, scale=0.3)),
    (8, 32, 16, 8, 600, 100, 8, dict(max_distance=100, key_step=6)),
])
def test_attention_with_bias(dtype, n, h, hkv, e, lq, lk, buckets, more):
    _check_attention(*_attention_inputs(n, h, hkv, e, lq, lk, buckets, dtype),
                     **more)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("buckets", [0, 8])
@pytest.mark.parametrize("lq,lk,lens", [
    (50, 80, [0, 80, 1, 63, 64, 65]),
    (1, 600, [600, 0, 257, 1, 256, 599]),
    (9, 33, [-4, 40, 33, 32, 2, 0]),     # held to 0..Lk
])
def test_attention_lengths(dtype, buckets, lq, lk, lens):
    """What is behind a length is not read: it holds NaN and inf here."""
    q, k, v, do, table = _attention_inputs(6, 2, 2, 24, lq, lk, buckets,
                                           dtype)
    for i, c in enumerate(lens):
        k[i, :, :, max(c, 0):] = math.nan
        v[i, :, :, max(c, 0):] = math.inf
    outs = _check_attention(q, k, v, do, table, lens,
                            **(dict(max_distance=30) if buckets else {}))
    for i, c in enumerate(lens):
        if c <= 0:
            assert all((t[i] == 0).all() for t in outs[:4])
        assert (outs[2][i, :, :, max(c, 0):] == 0).all()


@pytest.mark.parametrize("entry", [-math.inf, torch.finfo(BF16).min, -1e31])
def test_attention_entry_takes_pairs_out(entry):
    """No key after the query; the first queries' only keys are out, too."""
    q, k, v, do, table = _attention_inputs(1, 2, 2, 16, 70, 70, 8, BF16)
    table[:, 4:] = entry
    table[1, 0] = entry
    outs = _check_attention(q, k, v, do, table, max_distance=6)
    assert (outs[0][0, 1, :, 0] == 0).all() and (outs[1][0, 1, :, 0] == 0).all()


def test_attention_few_query_sums_stay_exact():
    """Rows whose keys are all in one bucket add nothing to its gradient."""
    q, k, v, do, table = _attention_inputs(1, 1, 1, 32, 4000, 20, 8, BF16)
    _check_attention(q, k, v, do, table, max_distance=8)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("buckets", [0, 8])
def test_attention_one_key_has_no_slope(dtype, buckets):
    # The only key has the weight p = 1 whatever the scores: dq is zero but for
    # dp - (p dp) / p, off by two roundings to 32 bits, 2 * 2^-24 |dp|, while
    # dp is at most sum |do| |v|. Twice that covers p's own last bit and the
    # roundings of ds and dq to the type.
    q, k, v, do, table = _attention_inputs(2, 2, 1, 48, 70, 40, buckets, dtype)
    lens = torch.tensor([1, 40], device=DEV)
    q.requires_grad_()
    more = {"max_distance": 20} if buckets else {}
    if buckets:
        table.requires_grad_()
    out = ops.cross_attention(q, k, v, lens, table, **more)
    dq, = torch.autograd.grad(out, [q], do)
    dp = (do[0].double().abs() * v[0, :, :, :1].double().abs()).sum(1)
    most = 4 * 2.0 ** -24 * dp[:, None] * k[0, :, :, :1].double().abs()
    assert (dq[0].double().abs() <= most / math.sqrt(48)).all()
    assert dq[1].abs().max() > 0


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_attention_views(dtype):
    """Heads cut out of one projection, steps between samples, and orders
    that need a copy, at odd addresses."""
    g = torch.Generator(device=DEV).manual_seed(2)
    both = torch.randn(2, 3 * 48 + 1, 71, device=DEV, generator=g).to(dtype)
    q = both[:, 1:49, 3:68].view(2, 3, 16, 65)
    k = both[:, 49:97, 1:].view(2, 3, 16, 70)
    v = both[:, 97:, 1:].view(2, 3, 16, 70)
    assert not q.is_contiguous()
    do = torch.randn(2, 3, 16, 65, device=DEV, generator=g).to(dtype)
    _check_attention(q, k, v, do, None)
    last = [t.transpose(2, 3).contiguous().transpose(2, 3)
            for t in (q, k, v, do)]
    _check_attention(*last, None)
    _check_attention(q, k, v, do[:, :, :, :1].expand(2, 3, 16, 65), None)


REFUSED_ATTENTION = [
    (dict(q=(1, 3, 4, 2)), "share"),
    (dict(q=(1, 2, 4)), "needed"),
    (dict(v=(1, 2, 4, 4)), "needed"),
    (dict(q=(1, 2, 5, 2)), "needed"),
    (dict(q=(1, 2, 129, 2), k=(1, 2, 129, 3), v=(1, 2, 129, 3)), "channels"),
    (dict(q=(1, 2, 0, 2), k=(1, 2, 0, 3), v=(1, 2, 0, 3)), "channels"),
    (dict(k=(1, 0, 4, 3), v=(1, 0, 4, 3)), "share"),
    (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=math.inf), "scale"),
    (dict(scale=math.nan), "scale"),
    (dict(kv_lengths=torch.zeros(2, dtype=torch.int32)), "kv_lengths"),
    (dict(kv_lengths=torch.zeros(1)), "kv_lengths"),
    (dict(bias_table=(1, 8)), "bias_table"),
    (dict(bias_table=(2, 8, 1)), "bias_table"),
    (dict(bias_table=(2, 7)), "buckets"),
    (dict(bias_table=(2, 2)), "buckets"),
    (dict(bias_table=(2, 66)), "buckets"),
    (dict(bias_table=(2, 8), max_distance=2), "max_distance"),
    (dict(bias_table=(2, 8), max_distance=1025), "max_distance"),
    (dict(bias_table=(2, 8), key_step=0), "key_step"),
    (dict(bias_table=(2, 8), key_step=2 ** 26), "positions"),
    (dict(bias_table=(2, 8), query_start=-2 ** 27), "positions"),
    (dict(bias_table=(2, 8), query_start=2 ** 62), "positions"),
]


@pytest.mark.parametrize("change,word", REFUSED_ATTENTION)
def test_attention_refuses(change, word):
    args = dict(q=(1, 2, 4, 2), k=(1, 2, 4, 3), v=(1, 2, 4, 3))
    args.update(change)
    for name, a in args.items():
        if isinstance(a, tuple):
            args[name] = torch.zeros(a, device=DEV)
        elif isinstance(a, torch.Tensor):
            args[name] = a.to(DEV)
    with pytest.raises(ValueError, match=word):
        ops.cross_attention(**args)


def test_attention_refuses_types_and_places():
    q, k, v, do, table = _attention_inputs(1, 2, 2, 8, 5, 4, 8, FP32)
    for args in ((q.half(), k.half(), v.half()), (q, k.bfloat16(), v),
                 (q, k.cpu(), v), (q, k, v, None, table.bfloat16()),
                 (q, k, v, torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.cross_attention(*args)
    q.requires_grad_()
    out = ops.cross_attention(q, k, v)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(out, q, do, create_graph=True)


def test_attention_empty():
    q, k, v, _, _ = _attention_inputs(2, 2, 2, 8, 5, 3, 0, FP32)
    q = q.requires_grad_()
    out = ops.cross_attention(q, k[..., :0], v[..., :0])
    assert out.shape == q.shape and (out == 0).all()
    (dq,) = torch.autograd.grad(out.sum(), q)
    assert (dq == 0).all()
    assert ops.cross_attention(q[..., :0], k, v).shape == (2, 2, 8, 0)
    assert ops.cross_attention(q[:0], k[:0], v[:0]).shape == (0, 2, 8, 5)


def test_attention_some_gradients():
    q, k, v, do, table = _attention_inputs(1, 2, 2, 16, 70, 50, 8, FP32)
    want, bound = ref.attention(q, k, v, None, table, max_distance=9, dout=do)
    for name, at in (("dq", 0), ("dk", 1), ("dv", 2), ("dtable", 3)):
        args = [t.detach() for t in (q, k, v, table)]
        args[at].requires_grad_()
        out = ops.cross_attention(args[0], args[1], args[2], None, args[3],
                                  max_distance=9)
        (got,) = torch.autograd.grad(out, args[at], do)
        ref.assert_within(got, want[name], bound[name], name)
        args[at].requires_grad_(False)


def test_attention_against_differences():
    """Along a direction, in fp32: a central difference of step 2^-6 is off by
    its third derivative's share, step^2/6 of it, and by the values' rounding
    over the step."""
    q, k, v, do, table = _attention_inputs(1, 2, 1, 16, 20, 30, 8, FP32)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]

    def value(*a):
        out = ops.cross_attention(a[0], a[1], a[2], None, a[3],
                                  max_distance=9)
        return (out.double() * do).sum()

    grads = torch.autograd.grad(value(*leaves), leaves)
    for at, grad in enumerate(grads):
        way = torch.randn_like(grad)
        way /= way.norm()
        step, ends = 2.0 ** -6, []
        with torch.no_grad():
            for m in (-2, -1, 1, 2):
                moved = list(leaves)
                moved[at] = leaves[at] + m * step * way
                ends.append(value(*moved).item())
        near = (ends[2] - ends[1]) / (2 * step)
        far = (ends[3] - ends[0]) / (4 * step)
        # the two differ by three times the nearer one's error
        room = abs(far - near) + 2e-4 * do.norm().item()
        assert abs(near - (grad.double() * way).sum().item()) <= room


def test_attention_is_the_same_each_time():
    for dtype in (BF16, FP32):
        args = _attention_inputs(2, 4, 2, 32, 200, 600, 32, dtype)
        runs = [_check_attention(*args, lens=[600, 123], max_distance=64)
                for _ in range(2)]
        assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_attention_other_stream_and_graph():
    """Captured with its backward pass, replayed between eager calls on other
    inputs; two graphs at once keep apart."""
    q, k, v, do, table = _attention_inputs(2, 4, 2, 32, 1, 900, 8, BF16)
    lens = torch.tensor([900, 300], device=DEV, dtype=torch.int32)

    def step(*t):
        leaves = [x.detach().requires_grad_() for x in t]
        out = ops.cross_attention(leaves[0], leaves[1], leaves[2], lens,
                                  leaves[3], query_start=700)
        return (out.detach(),) + torch.autograd.grad(out, leaves, do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step(q, k, v, table)
    torch.cuda.current_stream().wait_stream(side)
    graphs, got = [], []
    other = [t * 0.5 for t in (q, k, v, table)]
    for args in ((q, k, v, table), other):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(step(*args))
        graphs.append(graph)
    eager_other = step(*other)
    for _ in range(3):
        graphs[0].replay()
        graphs[1].replay()
        now = step(q, k, v, table)
        torch.cuda.synchronize()
        for a, b, c in zip(got[0], eager, now):
            assert torch.equal(a, b) and torch.equal(a, c)
        assert all(torch.equal(a, b) for a, b in zip(got[1], eager_other))


@pytest.mark.parametrize("lq", [1, 100])
def test_attention_in_a_long_cache(lq):
    """Records, and a head's channels, further apart than 32 bits reach: the
    offsets of the last record's last channel pass 2**32 bytes."""
    n, e, lk = 2, 128, 300
    apart, between = 2 ** 31 + 64, 2 ** 24
    store = torch.empty(apart + e * between, device=DEV, dtype=BF16)
    k = store.as_strided((n, 1, e, lk), (apart, apart, between, 1), 5)
    v = store.as_strided((n, 1, e, lk), (apart, apart, between, 1), 1005)
    q, k0, v0, do, _ = _attention_inputs(n, 2, 1, e, lq, lk, 0, BF16)
    k.copy_(k0)
    v.copy_(v0)
    got = torch.stack([ops.cross_attention(q, k, v),
                       ops.cross_attention(q, k0, v0)])
    assert torch.equal(got[0], got[1])
    leaves = [t.requires_grad_() for t in (q, k0, v0)]
    want = torch.autograd.grad(ops.cross_attention(*leaves), leaves, do)
    leaves = [q, k.detach().requires_grad_(), v.detach().requires_grad_()]
    grads = torch.autograd.grad(ops.cross_attention(*leaves), leaves, do)
    for a, b in zip(grads, want):
        assert torch.equal(a, b)


def test_attention_deep_heads_in_a_graph():
    """The largest workgroups, whose LDS has to be asked for, captured, and
    run on two streams at once."""
    args = _attention_inputs(2, 2, 1, 128, 200, 700, 32, BF16)

    def step(q, k, v, do, table):
        leaves = [x.detach().requires_grad_() for x in (q, k, v, table)]
        out = ops.cross_attention(leaves[0], leaves[1], leaves[2], None,
                                  leaves[3], max_distance=1024)
        return (out.detach(),) + torch.autograd.grad(out, leaves, do)

    eager = step(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*args)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        graph.replay()
        both = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                both.append(step(*args))
        torch.cuda.synchronize()
        for run in [got] + both:
            assert all(torch.equal(a, b) for a, b in zip(run, eager))


def _scan_inputs(n, c, length, dtype, seed=0, shift=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x, gate, dh = (torch.randn(n, c, length, device=DEV, generator=g)
                   for _ in range(3))
    gate = gate * 2 + shift
    state, ds = (torch.randn(n, c, device=DEV, generator=g) for _ in range(2))
    return x.to(dtype), gate.to(dtype), state, dh.to(dtype), ds


def _check_scan(x, gate, state, dh, ds, lens=None, reverse=False):
    lens = None if lens is None else torch.tensor(lens, device=DEV)
    with torch.no_grad():
        plain = ops.gated_scan(x, gate, state, lens, reverse)
    leaves = [t.detach().requires_grad_() for t in (x, gate, state)]
    out = ops.gated_scan(*leaves, lens, reverse)
    grads = torch.autograd.grad(out, leaves, [dh, ds])
    want, bound = ref.scan(x, gate, state, lens, reverse, dh, ds)
    names = ("h", "state", "dx", "dgate", "dstate")
    for name, got in zip(names, plain):
        ref.assert_within(got, want[name], bound[name], name + ", no gradient")
    for name, got in zip(names, out + grads):
        ref.assert_within(got, want[name], bound[name], name)
    return out + grads


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("n,c,length", [
    (3, 5, 1), (2, 3, 7), (9, 40, 8), (5, 7, 9), (3, 3, 63), (2, 5, 64),
    (2, 3, 65), (2, 2, 511), (1, 3, 513), (1, 2, 2049), (1, 1, 9001),
    (2, 1, 20480),
])
def test_scan(dtype, reverse, n, c, length):
    _check_scan(*_scan_inputs(n, c, length, dtype), reverse=reverse)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_scan_many_rows(dtype):
    """Enough rows that a wave walks one alone, over several chunks."""
    _check_scan(*_scan_inputs(70, 64, 1100, dtype))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("length", [1, 9, 70, 700, 12345])
def test_scan_lengths(dtype, reverse, length):
    """What is behind a length is not read: it holds NaN and inf here."""
    x, gate, state, dh, ds = _scan_inputs(6, 3, length, dtype)
    lens = [0, length, (length + 1) // 2, 1, -3, length + 5]
    for i, c in enumerate(lens):
        x[i, :, max(c, 0):] = math.nan
        gate[i, :, max(c, 0):] = math.inf
        dh[i, :, max(c, 0):] = math.nan
    outs = _check_scan(x, gate, state, dh, ds, lens, reverse)
    assert torch.equal(outs[1][0], state[0])
    assert torch.equal(outs[4][0], ds[0])


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_scan_views(dtype):
    """Two halves of one projection, odd addresses, and orders that need a
    copy."""
    g = torch.Generator(device=DEV).manual_seed(2)
    both = torch.randn(3, 10, 903, device=DEV, generator=g).to(dtype)
    _, _, state, dh, ds = _scan_inputs(3, 5, 901, dtype)
    x, gate = both[:, :5, 1:902], both[:, 5:, 2:]
    _check_scan(x, gate, state, dh, ds)
    last = [t.transpose(1, 2).contiguous().transpose(1, 2)
            for t in (x, gate, dh)]
    _check_scan(last[0], last[1], state, last[2], ds)


@pytest.mark.parametrize("length", [5, 50, 3000])
def test_scan_gates_at_their_ends(length):
    """Gates of +-inf and far ones: all of the state, or none of it."""
    x, gate, state, dh, ds = _scan_inputs(2, 4, length, FP32)
    gate[0, 0] = math.inf
    gate[0, 1] = -math.inf
    gate[0, 2] = 90.0
    gate[0, 3] = -90.0
    gate[1, 0] = 200.0
    outs = _check_scan(x, gate, state, dh, ds)
    assert torch.equal(outs[0][0, 0], state[0, 0].expand(length))
    assert torch.equal(outs[0][0, 1], x[0, 1])


def test_scan_one_gradient_alone():
    for length in (1, 40, 5000):
        x, gate, _, dh, ds = _scan_inputs(2, 3, length, FP32)
        for through in (0, 1):
            leaf = x.detach().requires_grad_()
            out = ops.gated_scan(leaf, gate)
            (got,) = torch.autograd.grad(out[through], leaf,
                                         dh if through == 0 else ds)
            want, bound = ref.scan(x, gate, None, None, False,
                                   dh if through == 0 else None,
                                   ds if through == 1 else None)
            ref.assert_within(got, want["dx"], bound["dx"], "dx")


@pytest.mark.parametrize("change,word", [
    (dict(x=(2, 3)), "needed"),
    (dict(gate=(2, 3, 5)), "needed"),
    (dict(x=(2, 3, 0), gate=(2, 3, 0)), "at least 1"),
    (dict(state=(2, 4)), "state"),
    (dict(state=(2, 3, 1)), "state"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.zeros(2)), "lengths"),
])
def test_scan_refuses(change, word):
    args = dict(x=(2, 3, 4), gate=(2, 3, 4))
    args.update(change)
    for name, a in args.items():
        args[name] = torch.zeros(a, device=DEV) if isinstance(a, tuple) \
            else a.to(DEV)
    with pytest.raises(ValueError, match=word):
        ops.gated_scan(**args)


def test_scan_refuses_types_and_places():
    x, gate, state, dh, _ = _scan_inputs(2, 3, 4, FP32)
    for args in ((x.half(), gate.half()), (x, gate.bfloat16()),
                 (x, gate.cpu()), (x, gate, state.bfloat16()),
                 (x, gate, state.cpu())):
        with pytest.raises(ValueError):
            ops.gated_scan(*args)
    x.requires_grad_()
    h, _ = ops.gated_scan(x, gate)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(h, x, dh, create_graph=True)


def test_scan_empty():
    x = torch.zeros(0, 3, 4, device=DEV, requires_grad=True)
    h, last = ops.gated_scan(x, x)
    assert h.shape == (0, 3, 4) and last.shape == (0, 3)
    assert torch.autograd.grad(h.sum(), x)[0].shape == x.shape


def test_scan_against_differences():
    x, gate, state, dh, ds = _scan_inputs(1, 2, 600, FP32)
    leaves = [t.requires_grad_() for t in (x, gate, state)]

    def value(*a):
        h, last = ops.gated_scan(*a)
        return (h.double() * dh).sum() + (last.double() * ds).sum()

    grads = torch.autograd.grad(value(*leaves), leaves)
    for at, grad in enumerate(grads):
        way = torch.randn_like(grad)
        way /= way.norm()
        step, ends = 2.0 ** -6, []
        with torch.no_grad():
            for m in (-2, -1, 1, 2):
                moved = list(leaves)
                moved[at] = leaves[at] + m * step * way
                ends.append(value(*moved).item())
        near = (ends[2] - ends[1]) / (2 * step)
        far = (ends[3] - ends[0]) / (4 * step)
        room = abs(far - near) + 2e-4 * dh.norm().item()
        assert abs(near - (grad.double() * way).sum().item()) <= room


def test_scan_rows_far_apart():
    """Rows further apart than 32 bits reach."""
    apart, length = 2 ** 31 + 8, 5000
    store = torch.empty(3 * 2 ** 30, device=DEV, dtype=BF16)
    x, gate = (store.as_strided((2, 2, length), (apart, 8192, 1), at)
               for at in (3, 40001))
    near = _scan_inputs(2, 2, length, BF16)
    x.copy_(near[0])
    gate.copy_(near[1])
    for a, b in zip(ops.gated_scan(x, gate),
                    ops.gated_scan(near[0], near[1])):
        assert torch.equal(a, b)


def test_scan_graph():
    x, gate, state, dh, ds = _scan_inputs(2, 3, 30000, BF16)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, gate, state)]
        out = ops.gated_scan(*leaves)
        return tuple(t.detach() for t in out) + torch.autograd.grad(
            out, leaves, [dh, ds])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
        now = step()
        torch.cuda.synchronize()
        for a, b, c in zip(got, eager, now):
            assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_run_together(dtype):
    """A block over a long record as it would be used: a projection whose
    halves drive the recurrence, and attention of its states to a pooled
    copy with positions, trained in one pass, then the same record in pieces
    of one sample without gradients."""
    g = torch.Generator(device=DEV).manual_seed(4)
    N, C, L, H, step = 2, 32, 320, 4, 8
    lens = torch.tensor([320, 200], device=DEV, dtype=torch.int32)

    def made(*shape, scale):
        t = torch.randn(*shape, device=DEV, generator=g) * scale
        return t.to(dtype).requires_grad_()

    x = made(N, C, L, scale=1.0)
    w = made(2 * C, C, 1, scale=C ** -0.5)
    table = made(H, 16, scale=1.0)

    def block(x, w, table, move):
        both = ops.pointwise_conv(x, w)
        h, last = ops.gated_scan(both[:, :C], both[:, C:], lengths=lens)
        kv = move(h)
        heads = kv.view(N, H, C // H, L // step)
        out = ops.cross_attention(h.view(N, H, C // H, L), heads, heads,
                                  lens // step, table, key_step=step,
                                  max_distance=64)
        return out.reshape(N, C, L), last, h

    out, last, h = block(x, w, table,
                         lambda t: ops.avgmax_pool1d(t, step))
    (out.float().square().mean() + last.square().mean()).backward()
    cpu = [t.detach().cpu().requires_grad_() for t in (x, w, table)]
    lens_there, lens = lens, lens.cpu()
    want, want_last, _ = block(*cpu, lambda t: ops.avgmax_pool1d(t, step))
    (want.float().square().mean() + want_last.square().mean()).backward()
    lens = lens_there
    # bf16 rounds six times on the way (projection, states, pool, p, result,
    # each gradient): at most 6 * 2^-8 of a tensor's size; fp32 has 2^16 more
    room = 6 * 2.0 ** -8 if dtype == BF16 else 6 * 2.0 ** -20
    for got, exact in ((out, want), (x.grad, cpu[0].grad),
                       (w.grad, cpu[1].grad), (table.grad, cpu[2].grad)):
        off = (got.cpu().float() - exact.float()).norm()
        assert off <= room * exact.float().norm()
    with torch.no_grad():
        both = ops.pointwise_conv(x, w)
        state = None
        for t in range(0, 40):
            one, state = ops.gated_scan(both[:, :C, t:t + 1],
                                        both[:, C:, t:t + 1], state)
            off = (one[..., 0].float() - h[..., t].float()).abs().max()
            assert off <= (2.0 ** -7 if dtype == BF16 else 1e-5) * 4
        # one query at a time against the whole
        pooled = ops.avgmax_pool1d(h, step).view(N, H, C // H, L // step)
        for t in (0, 100, 319):
            q = h[..., t:t + 1].reshape(N, H, C // H, 1)
            one = ops.cross_attention(q, pooled, pooled, lens // step, table,
                                      key_step=step, max_distance=64,
                                      query_start=t)
            whole = out.detach().view(N, H, C // H, L)[..., t:t + 1]
            off = (one.float() - whole.float()).abs().max()
            assert off <= (2.0 ** -6 if dtype == BF16 else 1e-5) * 4
