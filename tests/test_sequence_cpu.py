"""Attention to other lengths, its position bias and the gated recurrence on
the CPU: the plain composites and the formulas of their gradients against 64
bits and differences, and the calls that are refused."""

import math

import pytest
import torch

import _sequence_ref as ref
from seist_amd import ops


def _attention_inputs(n, h, hkv, e, lq, lk, buckets, dtype=torch.float32):
    g = torch.Generator().manual_seed(7 * lq + lk)
    t = [torch.randn(s, generator=g).to(dtype)
         for s in ((n, h, e, lq), (n, hkv, e, lk), (n, hkv, e, lk),
                   (n, h, e, lq))]
    table = torch.randn(h, buckets, generator=g).to(dtype) if buckets else None
    return t + [table]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [None, [0, 5], [9, 1]])
def test_attention_matches_formula(dtype, lens):
    q, k, v, do, table = _attention_inputs(2, 4, 2, 5, 7, 9, 8, dtype)
    lens = None if lens is None else torch.tensor(lens)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = ops.cross_attention(q, k, v, lens, table, key_step=2, query_start=3,
                              max_distance=10)
    grads = torch.autograd.grad(out, leaves, do)
    want, bound = ref.attention(q, k, v, lens, table, 2, 3, 10, dout=do)
    for name, got in zip(("out", "dq", "dk", "dv", "dtable"), (out,) + grads):
        # the composite also rounds what autograd carries between its steps
        ref.assert_within(got, want[name], 2 * bound[name], name)


def test_attention_formula_against_differences():
    q, k, v, do, table = (t.double() for t in _attention_inputs(
        2, 2, 1, 3, 4, 6, 8))
    lens = torch.tensor([6, 4])
    want, _ = ref.attention(q, k, v, lens, table, 1, 2, 5, dout=do)

    def value(*args):
        return (ref.attention(args[0], args[1], args[2], lens, args[3], 1, 2,
                              5)[0]["out"] * do).sum()

    args, step = [q, k, v, table], 1e-6
    for at, name in enumerate(("dq", "dk", "dv", "dtable")):
        way = torch.randn(args[at].shape, dtype=torch.float64,
                          generator=torch.Generator().manual_seed(at))
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[at] = args[at] + sign * step * way
            ends.append(value(*moved))
        got = (ends[0] - ends[1]) / (2 * step)
        assert abs(got - (want[name] * way).sum()) < 1e-7


def test_attention_masked_places_are_not_read():
    q, k, v, _, _ = _attention_inputs(2, 2, 2, 4, 3, 6, 0)
    lens = torch.tensor([0, 4])
    want = ops.cross_attention(q, k, v, lens)
    assert (want[0] == 0).all()
    k[1, :, :, 4:], v[1, :, :, 4:] = math.nan, math.inf
    k[0], v[0] = math.nan, math.nan
    assert torch.equal(ops.cross_attention(q, k, v, lens), want)


@pytest.mark.parametrize("entry", [-math.inf, torch.finfo(torch.float32).min,
                                   -1e30])
def test_attention_entry_takes_pairs_out(entry):
    q, k, v, _, _ = _attention_inputs(1, 1, 1, 4, 5, 5, 0)
    table = torch.zeros(1, 8)
    table[0, 4:] = entry                  # no key after the query
    got = ops.cross_attention(q, k, v, bias_table=table, max_distance=4)
    first = ops.cross_attention(q[..., :1], k[..., :1], v[..., :1])
    torch.testing.assert_close(got[..., :1], first)
    gone = ops.cross_attention(q, k, v, bias_table=torch.full((1, 8), entry),
                               max_distance=4)
    assert (gone == 0).all()


@pytest.mark.parametrize("buckets,far", [(4, 2), (8, 20), (32, 128),
                                         (64, 1024), (6, 100), (32, 9)])
def test_buckets(buckets, far):
    d = torch.arange(-far - 5, far + 6)
    got = ops.relative_position_buckets(d, buckets, far)
    assert got.tolist() == [ref.bucket(int(i), buckets, far) for i in d]
    assert int(got.min()) == 0 and int(got.max()) == buckets - 1


@pytest.mark.parametrize("change,word", [
    (dict(q=torch.zeros(1, 3, 4, 2)), "share"),
    (dict(q=torch.zeros(1, 2, 4)), "needed"),
    (dict(v=torch.zeros(1, 2, 4, 4)), "needed"),
    (dict(q=torch.zeros(1, 2, 5, 2)), "needed"),
    (dict(q=torch.zeros(1, 2, 4, 2, dtype=torch.float64)), "float32"),
    (dict(k=torch.zeros(1, 2, 4, 3, dtype=torch.bfloat16)), "float32"),
    (dict(kv_lengths=torch.zeros(2, dtype=torch.int32)), "kv_lengths"),
    (dict(kv_lengths=torch.zeros(1)), "kv_lengths"),
    (dict(bias_table=torch.zeros(1, 8)), "bias_table"),
    (dict(bias_table=torch.zeros(2, 8, dtype=torch.bfloat16)), "bias_table"),
    (dict(bias_table=torch.zeros(2, 7)), "buckets"),
    (dict(bias_table=torch.zeros(2, 2)), "buckets"),
    (dict(bias_table=torch.zeros(2, 66)), "buckets"),
    (dict(bias_table=torch.zeros(2, 8), max_distance=2), "max_distance"),
    (dict(bias_table=torch.zeros(2, 8), max_distance=1025), "max_distance"),
    (dict(bias_table=torch.zeros(2, 8), key_step=0), "key_step"),
    (dict(bias_table=torch.zeros(2, 8), key_step=2 ** 29), "2\\*\\*27"),
    (dict(bias_table=torch.zeros(2, 8), query_start=-2 ** 30), "2\\*\\*27"),
])
def test_attention_refuses(change, word):
    args = dict(q=torch.zeros(1, 2, 4, 2), k=torch.zeros(1, 2, 4, 3),
                v=torch.zeros(1, 2, 4, 3))
    args.update(change)
    with pytest.raises(ValueError, match=word):
        ops.cross_attention(**args)


def test_attention_refuses_wide_heads():
    with pytest.raises(ValueError, match="channels"):
        ops.cross_attention(*(torch.zeros(1, 1, 129, 2) for _ in range(3)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens", [None, [0, 5, 11]])
@pytest.mark.parametrize("reverse", [False, True])
def test_scan_matches_formula(dtype, lens, reverse):
    g = torch.Generator().manual_seed(3)
    x, gate, dh = (torch.randn(3, 2, 11, generator=g).to(dtype)
                   for _ in range(3))
    state, ds = (torch.randn(3, 2, generator=g) for _ in range(2))
    lens = None if lens is None else torch.tensor(lens)
    leaves = [t.requires_grad_() for t in (x, gate, state)]
    out = ops.gated_scan(*leaves, lens, reverse)
    grads = torch.autograd.grad(out, leaves, [dh, ds])
    want, bound = ref.scan(x, gate, state.detach(), lens, reverse, dh, ds)
    for name, got in zip(("h", "state", "dx", "dgate", "dstate"),
                         out + grads):
        ref.assert_within(got, want[name], bound[name], name)


def test_scan_formula_against_differences():
    g = torch.Generator().manual_seed(5)
    x, gate, dh = (torch.randn(2, 2, 9, generator=g, dtype=torch.float64)
                   for _ in range(3))
    state, ds = (torch.randn(2, 2, generator=g, dtype=torch.float64)
                 for _ in range(2))
    lens = torch.tensor([9, 4])
    want, _ = ref.scan(x, gate, state, lens, True, dh, ds)

    def value(*args):
        r, _ = ref.scan(*args, lens, True)
        return (r["h"] * dh).sum() + (r["state"] * ds).sum()

    args, step = [x, gate, state], 1e-6
    for at, name in enumerate(("dx", "dgate", "dstate")):
        way = torch.randn(args[at].shape, dtype=torch.float64, generator=g)
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[at] = args[at] + sign * step * way
            ends.append(value(*moved))
        got = (ends[0] - ends[1]) / (2 * step)
        assert abs(got - (want[name] * way).sum()) < 1e-7


def test_scan_in_pieces_is_the_whole():
    g = torch.Generator().manual_seed(1)
    x, gate = (torch.randn(2, 3, 8, generator=g) for _ in range(2))
    h, last = ops.gated_scan(x, gate)
    state, parts = None, []
    for cut in ((0, 3), (3, 4), (4, 8)):
        p, state = ops.gated_scan(x[..., cut[0]:cut[1]],
                                  gate[..., cut[0]:cut[1]], state)
        parts.append(p)
    torch.testing.assert_close(torch.cat(parts, -1), h)
    torch.testing.assert_close(state, last)


@pytest.mark.parametrize("change,word", [
    (dict(x=torch.zeros(2, 3)), "needed"),
    (dict(gate=torch.zeros(2, 3, 5)), "needed"),
    (dict(x=torch.zeros(2, 3, 0), gate=torch.zeros(2, 3, 0)), "at least 1"),
    (dict(gate=torch.zeros(2, 3, 4, dtype=torch.bfloat16)), "float32"),
    (dict(x=torch.zeros(2, 3, 4, dtype=torch.float16),
          gate=torch.zeros(2, 3, 4, dtype=torch.float16)), "float32"),
    (dict(state=torch.zeros(2, 4)), "state"),
    (dict(state=torch.zeros(2, 3, dtype=torch.bfloat16)), "state"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (dict(lengths=torch.zeros(2)), "lengths"),
])
def test_scan_refuses(change, word):
    args = dict(x=torch.zeros(2, 3, 4), gate=torch.zeros(2, 3, 4))
    args.update(change)
    with pytest.raises(ValueError, match=word):
        ops.gated_scan(**args)
