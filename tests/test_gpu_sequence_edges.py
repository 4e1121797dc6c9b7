"""Calls of the sequence operators at the edges of what their documentation
allows, on the gfx950 kernels."""

import warnings

import pytest
import torch

import _sequence_ref as ref
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
