"""Calls of the sequence operators at the edges of what their documentation
allows, on the gfx950 kernels."""

import math
import warnings

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensor, FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import _sequence_ref as ref
import _sequence_walk as walk
from seist_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF16, FP32 = torch.bfloat16, torch.float32


def _inputs(*shapes, dtype=FP32, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(s, device=DEV, generator=g).to(dtype) for s in shapes]


# ---------------------------------------------------------------------------
# what autograd and the tracer are told
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("at", range(4))
def test_attention_refuses_forward_mode(at, grad):
    """A tangent is refused and not dropped, with and without gradients."""
    args = _inputs((1, 2, 4, 5), (1, 2, 4, 6), (1, 2, 4, 6), (2, 8))
    tangent = torch.ones_like(args[at])
    if grad:
        args = [t.requires_grad_() for t in args]
    with forward_ad.dual_level():
        args[at] = forward_ad.make_dual(args[at], tangent)
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match="forward-mode"):
                ops.cross_attention(args[0], args[1], args[2], None, args[3],
                                    max_distance=5)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("at", range(3))
def test_scan_refuses_forward_mode(at, grad):
    args = _inputs((1, 2, 9), (1, 2, 9), (1, 2))
    tangent = torch.ones_like(args[at])
    if grad:
        args = [t.requires_grad_() for t in args]
    with forward_ad.dual_level():
        args[at] = forward_ad.make_dual(args[at], tangent)
        for mode in (torch.enable_grad, torch.no_grad):
            with mode(), pytest.raises(RuntimeError, match="forward-mode"):
                ops.gated_scan(*args)


def test_gradients_refuse_forward_mode():
    """Forward mode through the backward pass."""
    q, k, x, gate = (t.requires_grad_() for t in _inputs(
        (1, 2, 4, 5), (1, 2, 4, 6), (1, 2, 9), (1, 2, 9)))
    out = ops.cross_attention(q, k, k)
    h, last = ops.gated_scan(x, gate)
    with forward_ad.dual_level():
        for y, leaf in ((out, q), (h, x), (last, x)):
            dy = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, dy, retain_graph=True)


def _traced(f, args):
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        return torch.jit.trace(f, args, check_trace=False)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("grad", [False, True])
def test_attention_traced(dtype, grad):
    """What is recorded computes the operator for inputs of its own, and its
    gradients."""
    shapes = (2, 4, 16, 33), (2, 2, 16, 40), (2, 2, 16, 40), (4, 8)
    lens = torch.tensor([17, 40], device=DEV)

    def f(q, k, v, table, lens):
        return ops.cross_attention(q, k, v, lens, table, key_step=2,
                                   max_distance=20)

    first = [t.requires_grad_(grad) for t in _inputs(*shapes, dtype=dtype)]
    traced = _traced(f, (*first, lens))
    args = _inputs(*shapes, dtype=dtype, seed=1)
    do = _inputs(shapes[0], dtype=dtype, seed=2)[0]
    lens = torch.tensor([40, 5], device=DEV)
    want, bound = ref.attention(*args[:3], lens, args[3], 2, 0, 20, dout=do)
    leaves = [t.requires_grad_(grad) for t in args]
    out = traced(*leaves, lens)
    ref.assert_within(out, want["out"], bound["out"], "out")
    if grad:
        grads = torch.autograd.grad(out, leaves, do)
        for name, got in zip(("dq", "dk", "dv", "dtable"), grads):
            # recorded are plain steps, which also round what they carry
            ref.assert_within(got, want[name], 2 * bound[name], name)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("grad", [False, True])
def test_scan_traced(dtype, grad):
    shapes = (2, 3, 21), (2, 3, 21)
    lens = torch.tensor([21, 4], device=DEV)

    def f(x, gate, state, lens):
        return ops.gated_scan(x, gate, state, lens)

    first = _inputs(*shapes, dtype=dtype) + _inputs((2, 3))
    traced = _traced(f, (*(t.requires_grad_(grad) for t in first), lens))
    args = _inputs(*shapes, dtype=dtype, seed=1) + _inputs((2, 3), seed=1)
    dh = _inputs(shapes[0], dtype=dtype, seed=2)[0]
    ds = _inputs((2, 3), seed=3)[0]
    lens = torch.tensor([9, 21], device=DEV)
    want, bound = ref.scan(*args, lens, False, dh, ds)
    leaves = [t.requires_grad_(grad) for t in args]
    outs = traced(*leaves, lens)
    for name, got in zip(("h", "state"), outs):
        ref.assert_within(got, want[name], bound[name], name)
    if grad:
        grads = torch.autograd.grad(outs, leaves, [dh, ds])
        for name, got in zip(("dx", "dgate", "dstate"), grads):
            ref.assert_within(got, want[name], bound[name], name)


def test_calls_that_are_recorded_or_fake():
    """Recorded by the dispatcher, the plain steps are; under a mode that
    puts fake tensors in the place of results, and on fake tensors, no kernel
    runs, which would write to their null pointers."""
    q, k, x = _inputs((1, 2, 4, 5), (1, 2, 4, 6), (1, 2, 9))
    want, bound = ref.attention(q + 1, k + 1, k + 1)
    made = make_fx(lambda q, k: ops.cross_attention(q, k, k))(q, k)
    ref.assert_within(made(q + 1, k + 1), want["out"], bound["out"], "out")
    want, bound = ref.scan(x + 1, x + 1)
    made = make_fx(lambda x: ops.gated_scan(x, x)[0])(x)
    ref.assert_within(made(x + 1), want["h"], bound["h"], "h")
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        for args in ((q, k), (mode.from_tensor(q), mode.from_tensor(k))):
            out = ops.cross_attention(args[0], args[1], args[1])
            assert isinstance(out, FakeTensor) and out.shape == q.shape
        h, last = ops.gated_scan(x, x)
        assert isinstance(h, FakeTensor) and last.shape == (1, 2)
    for f, t in ((lambda q: ops.cross_attention(q, k, k), q),
                 (lambda x: ops.gated_scan(x, x)[0], x)):
        with pytest.raises(RuntimeError, match="no memory"):
            torch.func.functionalize(f)(t)
        y = f(t.clone().requires_grad_())
        with FakeTensorMode(allow_non_fake_inputs=True), \
                pytest.raises(RuntimeError, match="no memory"):
            y.sum().backward()
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------
# pairs that the table takes out
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("h,hkv,e,lq,lk,far,more", [
    (2, 2, 16, 70, 100, 6, {}),              # distances past the last bucket
    (2, 1, 24, 70, 200, 300, {}),            # all of them within it
    (4, 2, 64, 1, 700, 128, dict(query_start=600)),   # few rows, split keys
    (4, 2, 8, 3, 90, 20, dict(query_start=40)),
    (1, 1, 128, 150, 160, 9, {}),            # deep heads, waves in pairs
    (2, 2, 40, 64, 40, 100, dict(key_step=3)),
])
def test_attention_pairs_out_whatever_their_scores(dtype, what, h, hkv, e, lq,
                                                   lk, far, more):
    """Keys after every query, with NaN or infinite scores: the results, and
    all gradients that do not multiply by the keys, are as with finite ones."""
    q, k, v, do, table = _inputs((1, h, e, lq), (1, hkv, e, lk),
                                 (1, hkv, e, lk), (1, h, e, lq), (h, 8),
                                 dtype=dtype)
    table[:, 4:] = -math.inf
    want, bound = ref.attention(q, k, v, None, table, max_distance=far,
                                dout=do, **more)
    last = more.get("query_start", 0) + lq - 1
    behind = last // more.get("key_step", 1) + 1
    assert behind < lk
    k[..., behind:] = what
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    with torch.no_grad():
        plain = ops.cross_attention(q, k, v, None, table, max_distance=far,
                                    **more)
    out = ops.cross_attention(q, k, v, None, table, max_distance=far, **more)
    grads = torch.autograd.grad(out, leaves, do)
    for name, got in zip(("out", "out", "dk", "dv", "dtable"),
                         (plain, out) + grads[1:]):
        ref.assert_within(got, want[name], bound[name], name)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("far", [3, 100])
@pytest.mark.parametrize("e", [16, 128])
def test_attention_rows_that_leave_a_key_out(dtype, far, e):
    """A NaN key reaches the queries that have it, and no other."""
    q, k, v, table = _inputs((1, 2, e, 90), (1, 2, e, 90), (1, 2, e, 90),
                             (2, 8), dtype=dtype)
    table[:, 4:] = torch.finfo(dtype).min
    want, bound = ref.attention(q, k, v, None, table, max_distance=far)
    k[..., 50] = math.nan
    out = ops.cross_attention(q, k, v, None, table, max_distance=far)
    ref.assert_within(out[..., :50], want["out"][..., :50],
                      bound["out"][..., :50], "out")
    assert torch.isnan(out[..., 50:]).all()


def test_attention_heads_with_and_without_the_pair():
    """Heads that share a key, of which one has the pair out."""
    q, k, v, table = _inputs((1, 2, 32, 1), (1, 1, 32, 200), (1, 1, 32, 200),
                             (2, 8))
    table[0, 4:] = -math.inf
    for far in (4, 300):
        want, bound = ref.attention(q, k, v, None, table, 1, 100, far)
        bad = k.clone()
        bad[..., 150] = math.nan
        out = ops.cross_attention(q, bad, v, None, table, query_start=100,
                                  max_distance=far)
        ref.assert_within(out[:, :1], want["out"][:, :1], bound["out"][:, :1],
                          "out")
        assert torch.isnan(out[:, 1]).all()


def test_attention_no_key_left_and_no_finite_score():
    """Queries that are NaN and have no key left give zeros."""
    for lq in (1, 70):
        q, k, v, table = _inputs((1, 2, 16, lq), (1, 2, 16, 90),
                                 (1, 2, 16, 90), (2, 8))
        table[:] = -math.inf
        q[..., 0] = math.nan
        out = ops.cross_attention(q, k, v, None, table, max_distance=10)
        assert (out == 0).all()


# ---------------------------------------------------------------------------
# far apart and many
# ---------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("lq", [1, 50])
@pytest.mark.parametrize("short", [128, 127, 60, -8])
def test_attention_channels_at_the_reach(dtype, lq, short):
    """A head's channels as far apart as 32 bits of bytes reach, less some
    positions: short of a staged tile's 128, and past it."""
    lk, size = 50, torch.finfo(dtype).bits // 8
    between = 2 ** 32 // size - short
    store = torch.empty(between + 4096, device=DEV, dtype=dtype)
    q0, k0, v0, do0 = _inputs((1, 1, 2, lq), (1, 1, 2, lk), (1, 1, 2, lk),
                              (1, 1, 2, lq), dtype=dtype)
    far = []
    for at, t in enumerate((q0, k0, v0, do0)):
        far.append(store.as_strided(t.shape, (4096, 4096, between, 1),
                                    1000 * at + 1))
        far[-1].copy_(t)
    grads = []
    for q, k, v, do in ((q0, k0, v0, do0), far):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = ops.cross_attention(*leaves)
        grads.append((out,) + torch.autograd.grad(out, leaves, do))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("dtype,lq", [(BF16, 2 ** 24 + 2 ** 18),
                                      (FP32, 2 ** 23 + 2 ** 17)])
def test_attention_refuses_a_head_of_over_4_gib(dtype, lq):
    """Queries that overlap in memory, as windows of one record do: they lie
    close together, their results do not."""
    (x,) = _inputs((lq + 127,), dtype=dtype)
    q = x.as_strided((1, 1, 128, lq), (0, 0, 1, 1))
    k = x[:128 * 5].view(1, 1, 128, 5)
    with pytest.raises(ValueError, match="4 GiB"):
        ops.cross_attention(q, k, k)
    apart = x.as_strided((1, 1, 128, 5), (0, 0, 0, 1))
    with pytest.raises(ValueError, match="4 GiB"):
        ops.cross_attention(q, apart, apart)


def test_attention_of_the_most_records():
    """One workgroup a record: as many as a launch holds, and one more."""
    most = 2 ** 24 - 1
    q, k, v, do = (t.requires_grad_() for t in _inputs(
        *4 * [(most, 1, 1, 1)]))
    out = ops.cross_attention(q, k, v)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), do)
    # The only key's weight p is not 1 to the last bit, as the maximum that is
    # taken off its score is rounded; so with u = 2^-24
    # out = (p v) (1 / p): three roundings;
    # dq = p (dp - (p dp) / p) k: two on dp = do v, and those of a product by
    # what they leave; dk likewise by q;
    # dv = p do, p from the logarithm, u (|s| + 5) off 1: the logarithm's
    # rounding u |s|, u each for the sum's, its logarithm's and the
    # difference's, and 2 u for the exponential.
    u = 2.0 ** -24
    with torch.no_grad():
        assert ((out - v).abs() <= 4 * u * v.abs()).all()
        assert (dq.abs() <= 4 * u * (do * v * k).abs()).all()
        assert (dk.abs() <= 4 * u * (do * v * q).abs()).all()
        assert ((dv - do).abs() <= 8 * u * (1 + (q * k).abs())
                * do.abs()).all()
    more = torch.zeros(most + 1, 1, 1, 1, device=DEV)
    with pytest.raises(ValueError, match="one launch"):
        ops.cross_attention(more, more, more)
    # deep heads, whose gradients take twice the threads
    deep = torch.zeros(2 ** 23, 1, 65, 1, device=DEV, dtype=BF16)
    out = ops.cross_attention(deep.requires_grad_(), deep, deep)
    with pytest.raises(ValueError, match="one launch"):
        torch.autograd.grad(out.sum(), deep)


# ---------------------------------------------------------------------------
# variants by size, each against the formula
# ---------------------------------------------------------------------------


def _check_attention(shape, buckets, dtype, lens=None, table_grad=True,
                     **more):
    n, h, hkv, e, lq, lk = shape
    q, k, v, do = _inputs((n, h, e, lq), (n, hkv, e, lk), (n, hkv, e, lk),
                          (n, h, e, lq), dtype=dtype)
    table = _inputs((h, buckets), dtype=dtype)[0] if buckets else None
    if lens is not None:
        lens = torch.tensor(lens, device=DEV, dtype=torch.int32)
    want, bound = ref.attention(q, k, v, lens, table, dout=do, **more)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    if buckets and table_grad:
        leaves.append(table.requires_grad_())
    out = ops.cross_attention(q, k, v, lens, table, **more)
    grads = torch.autograd.grad(out, leaves, do)
    for name, got in zip(("out", "dq", "dk", "dv", "dtable"), (out,) + grads):
        ref.assert_within(got, want[name], bound[name], name)


@pytest.mark.parametrize("shape", [
    (8, 16, 16, 64, 1050, 200), (8, 16, 16, 48, 1100, 333),
    (8, 16, 16, 16, 1050, 300), (8, 32, 16, 24, 600, 515),
])
@pytest.mark.parametrize("lens", [None, [0, 1, 63, 129, 64, 197, 77, 200]])
def test_attention_two_column_blocks(shape, lens):
    """Queries enough for two blocks of columns a wave, and several staged
    tiles of keys."""
    _check_attention(shape, 0, BF16, lens)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", [
    (1, 2, 2, 16, 70, 50), (1, 4, 2, 32, 70, 700), (1, 2, 1, 24, 130, 20),
    (2, 2, 2, 40, 33, 300), (1, 1, 1, 128, 100, 600),
])
def test_attention_with_a_bias_that_has_no_gradient(dtype, shape):
    lens = [shape[5] - 9, shape[5]][:shape[0]]
    _check_attention(shape, 8, dtype, lens, table_grad=False, max_distance=30)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", [(70, 2, 1, 8, 1000, 20),
                                   (600, 1, 1, 16, 40, 33),
                                   (5, 3, 3, 8, 14001, 7)])
def test_attention_table_of_many_rows(dtype, shape):
    """A bias gradient of more than 512 row tiles, which two steps add up."""
    _check_attention(shape, 8, dtype, max_distance=12)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("buckets", [0, 16])
@pytest.mark.parametrize("shape", [(2, 8, 2, 128, 1, 300),
                                   (1, 4, 4, 100, 7, 1100),
                                   (3, 32, 1, 128, 1, 77)])
def test_attention_few_rows_of_deep_heads(dtype, buckets, shape):
    lens = [shape[5], 0, 31][:shape[0]]
    more = dict(max_distance=40, query_start=50) if buckets else {}
    _check_attention(shape, buckets, dtype, lens, **more)


def _check_scan(dtype, n, c, length, memory, lens, reverse):
    """Gates that keep a state for about ``memory`` samples, over a drift, so
    that what comes from far shows."""
    x, gate, dh = _inputs(*3 * [(n, c, length)])
    state, ds = _inputs((n, c), (n, c), seed=1)
    drift = torch.arange(length, device=DEV) / (3.0 * memory)
    x = (x + drift.sin()).to(dtype)
    dh = (dh + drift.cos()).to(dtype)
    gate = (gate * 0.5 + math.log(memory)).to(dtype)
    if lens is not None:
        lens = torch.tensor(lens, device=DEV)
    leaves = [t.requires_grad_() for t in (x, gate, state)]
    out = ops.gated_scan(*leaves, lens, reverse)
    grads = torch.autograd.grad(out, leaves, [dh, ds])
    with torch.no_grad():
        plain = ops.gated_scan(x, gate, state, lens, reverse)
    want, bound = walk.scan(x, gate, state, lens, reverse, dh, ds)
    names = ("h", "state", "dx", "dgate", "dstate")
    for name, got in zip(names, plain):
        ref.assert_within(got, want[name], bound[name], name + ", no gradient")
    for name, got in zip(names, out + grads):
        ref.assert_within(got, want[name], bound[name], name)


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype,n,c,length,memory", [
    (BF16, 1, 3, 7000, 2000),       # 4 waves a row, 2 segments
    (FP32, 1, 3, 4000, 1000),
    (BF16, 3, 2, 73733, 8000),      # 16 waves a row, 5 segments
    (FP32, 3, 2, 40001, 4000),
    (BF16, 1, 1, 1080001, 8000),    # 66 segments, over a wave's lanes
    (FP32, 2, 1, 540001, 8000),
    (BF16, 70, 64, 1000, 300),      # many rows, a wave each, two chunks
    (FP32, 70, 64, 500, 200),
    (BF16, 40, 30, 6000, 1000),     # 4 waves a row, the last chunk short
    (FP32, 40, 30, 2900, 1000),
])
@pytest.mark.parametrize("ragged", [False, True])
def test_scan_variants(dtype, n, c, length, memory, reverse, ragged):
    lens = None
    if ragged:
        lens = [(length * (2 * i + 1) // (2 * n) + 12345 * i) % (length + 1)
                for i in range(n)]
    _check_scan(dtype, n, c, length, memory, lens, reverse)


@pytest.mark.parametrize("e", [8, 11, 16])
@pytest.mark.parametrize("h,hkv,lq,lk,buckets", [
    (4, 4, 333, 700, 0),            # keys cut, so a delta walked beforehand
    (4, 2, 777, 1024, 0),
    (4, 4, 333, 700, 16),           # the bias has a gradient
    (64, 64, 1100, 300, 16),        # the same, uncut
    (64, 64, 1100, 300, 0),
])
def test_attention_gradients_of_small_heads(e, h, hkv, lq, lk, buckets):
    """dq in bf16 has two independent roundings of one size, ds's and its own:
    sqrt(2) of the result's alone. What all of a query's ds are off by together
    would meet the mean of the keys, which small heads do not average out; 1.5
    leaves it a twentieth of the variance, and the sums' scatter room."""
    q, k, v, do = _inputs((1, h, e, lq), (1, hkv, e, lk), (1, hkv, e, lk),
                          (1, h, e, lq), dtype=BF16)
    table = _inputs((h, buckets), dtype=BF16)[0] if buckets else None
    want, _ = ref.attention(q, k, v, None, table, max_distance=64, dout=do)
    leaves = [t.requires_grad_() for t in (q, k, v, table) if t is not None]
    out = ops.cross_attention(q, k, v, None, table, max_distance=64)
    dq = torch.autograd.grad(out, leaves, do)[0]
    least = (want["dq"].to(BF16).double() - want["dq"]).norm()
    assert (dq.double() - want["dq"]).norm() <= 1.5 * least


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_lengths_by_the_sample(dtype, reverse):
    """A row's end at each place of a lane's samples, with one lane a row, 16,
    64, 4 waves and several chunks; rows follow one another without a gap."""
    for base in (1, 9, 17, 60, 120, 500, 1020, 2040, 4090, 6140):
        for length in range(base, base + 9):
            _check_scan(dtype, 3, 5, length, 40, None, reverse)
