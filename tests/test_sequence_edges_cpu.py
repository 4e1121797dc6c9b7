"""Calls of the sequence operators at the edges of what their documentation
allows, on the CPU."""

import math
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import _sequence_ref as ref
import _sequence_walk as walk
from seist_amd import ops


def _inputs(*shapes, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g) for s in shapes]


@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_attention_gradients_do_not_read_masked_places(what):
    lens = torch.tensor([0, 4, 6])
    q, k, v, do = _inputs((3, 4, 5, 7), (3, 2, 5, 6), (3, 2, 5, 6),
                          (3, 4, 5, 7))
    (table,) = _inputs((4, 8), seed=1)
    for i, c in enumerate(lens):
        k[i, :, :, c:], v[i, :, :, c:] = what, what
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = ops.cross_attention(q, k, v, lens, table, max_distance=5)
    grads = torch.autograd.grad(out, leaves, do)
    want, bound = ref.attention(q, k, v, lens, table, max_distance=5, dout=do)
    for name, got in zip(("out", "dq", "dk", "dv", "dtable"), (out,) + grads):
        # the composite also rounds what autograd carries between its steps
        ref.assert_within(got, want[name], 2 * bound[name], name)
    assert (grads[0][0] == 0).all()
    assert (grads[1][1, :, :, 4:] == 0).all()
    assert (grads[2][1, :, :, 4:] == 0).all()


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_scan_gradients_do_not_read_masked_places(what, reverse):
    lens = torch.tensor([0, 4, 7])
    x, gate, dh, state, ds = _inputs(*3 * [(3, 2, 7)], *2 * [(3, 2)])
    for i, c in enumerate(lens):
        x[i, :, c:], gate[i, :, c:], dh[i, :, c:] = what, what, what
    leaves = [t.requires_grad_() for t in (x, gate, state)]
    out = ops.gated_scan(*leaves, lens, reverse)
    grads = torch.autograd.grad(out, leaves, [dh, ds])
    want, bound = ref.scan(x, gate, state.detach(), lens, reverse, dh, ds)
    for name, got in zip(("h", "state", "dx", "dgate", "dstate"),
                         out + grads):
        ref.assert_within(got, want[name], bound[name], name)
    for grad in grads[:2]:
        assert (grad[0] == 0).all() and (grad[1, :, 4:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16,
                                   torch.int32, torch.int64, torch.float32])
def test_buckets_of_any_type(dtype):
    low, high = -2 ** 20, 2 ** 20
    if not dtype.is_floating_point:
        ends = torch.iinfo(dtype)
        low, high = max(ends.min, -2 ** 31), min(ends.max, 2 ** 31 - 1)
    d = [low, high, high // 2] + list(range(max(low, -120), 121, 7))
    for buckets, far in ((8, 100), (32, 1024)):
        got = ops.relative_position_buckets(torch.tensor(d, dtype=dtype),
                                            buckets, far)
        assert got.dtype == dtype
        assert got.tolist() == [ref.bucket(i, buckets, far) for i in d]


def test_traced_calls_compute_their_own_inputs():
    q, k, v = _inputs((2, 4, 5, 7), (2, 2, 5, 6), (2, 2, 5, 6))
    (table,) = _inputs((4, 8), seed=1)
    x, gate = _inputs((2, 3, 9), (2, 3, 9))

    def attend(q, k, v, table, lens):
        return ops.cross_attention(q, k, v, lens, table, key_step=2,
                                   max_distance=5)

    def scan(x, gate, lens):
        return ops.gated_scan(x, gate, None, lens, True)

    lens = torch.tensor([3, 6])
    for f, args in ((attend, (q, k, v, table)), (scan, (x, gate))):
        with warnings.catch_warnings():
            warnings.simplefilter("ignore")
            traced = torch.jit.trace(f, (*args, lens), check_trace=False)
        args = [t * 0.5 - 1 for t in args] + [torch.tensor([6, 0])]
        torch.testing.assert_close(traced(*args), f(*args), rtol=0, atol=0)


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_attention_pairs_out_whatever_their_scores(what):
    q, k, v, do = _inputs((1, 2, 4, 7), (1, 2, 4, 12), (1, 2, 4, 12),
                          (1, 2, 4, 7))
    (table,) = _inputs((2, 8), seed=1)
    table[:, 4:] = -math.inf              # no key after the query
    want, bound = ref.attention(q, k, v, None, table, max_distance=5, dout=do)
    k[..., 7:] = what
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = ops.cross_attention(q, k, v, None, table, max_distance=5)
    grads = torch.autograd.grad(out, leaves, do)
    for name, got in zip(("out", "dk", "dv", "dtable"), (out,) + grads[1:]):
        ref.assert_within(got, want[name], 2 * bound[name], name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [None, [0, 31, 17]])
@pytest.mark.parametrize("reverse", [False, True])
def test_walked_recurrence_is_the_formula(dtype, lens, reverse):
    """What long records are compared with, against the steps one by one."""
    x, gate, dh, state, ds = _inputs(*3 * [(3, 2, 31)], *2 * [(3, 2)])
    args = [t.to(dtype) for t in (x, gate)] + [state, lens, reverse,
                                               dh.to(dtype), ds]
    for got, want in zip(walk.scan(*args), ref.scan(*args)):
        assert got.keys() == want.keys()
        for name in want:
            torch.testing.assert_close(got[name], want[name], rtol=1e-12,
                                       atol=1e-300)


def test_tensors_without_memory_are_not_given_to_kernels():
    """Fake tensors that say they are on a GPU: shapes and types come back and
    no kernel runs, in their mode and outside of it."""
    with FakeTensorMode():
        q, k = (torch.empty(2, 4, 8, n, device="cuda", dtype=torch.bfloat16)
                for n in (5, 7))
        x = torch.empty(2, 3, 9, device="cuda")
        lens = torch.empty(2, device="cuda", dtype=torch.int32)
        table = torch.empty(4, 8, device="cuda", dtype=torch.bfloat16)
        outs = [(ops.cross_attention(q, k, k, lens, table),)
                + ops.gated_scan(x, x, None, lens)]
    outs.append((ops.cross_attention(q, k, k),) + ops.gated_scan(x, x))
    for out, h, last in outs:
        assert out.shape == q.shape and out.dtype == torch.bfloat16
        assert h.shape == x.shape and last.shape == (2, 3)
        assert all(t.device.type == "cuda" for t in (out, h, last))


def test_recorded_calls_compute_their_own_inputs():
    q, k, x = _inputs((1, 2, 4, 5), (1, 2, 4, 6), (1, 2, 9))
    for mode in ("real", "fake"):
        for f, args in ((lambda q, k: ops.cross_attention(q, k, k), (q, k)),
                        (lambda x: ops.gated_scan(x, x)[0], (x,))):
            made = make_fx(f, tracing_mode=mode)(*args)
            args = [t + 1 for t in args]
            assert torch.equal(made(*args), f(*args))


@pytest.mark.skipif(not ops.has_ext(), reason="the extension is not built")
def test_the_extension_leaves_recorded_and_fake_calls():
    def nothing(q, x):
        args = (None, None, None, 1, 0, 128, [])
        assert ops.ext().cross_attention(q, q, q, *args) is None
        assert not ops.ext().gated_scan(x, x, None, None, False)
        return q * 2

    with FakeTensorMode():
        q = torch.empty(1, 2, 4, 5, device="cuda")
        x = torch.empty(1, 2, 5, device="cuda")
        nothing(q, x)
    nothing(q, x)
    real = _inputs((1, 2, 4, 5), (1, 2, 5))
    with FakeTensorMode(allow_non_fake_inputs=True):
        nothing(*real)
    make_fx(nothing)(*real)
    torch.jit.trace(nothing, tuple(real), check_trace=False)
