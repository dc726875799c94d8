"""Gradients that come from a generator, as a model's parameters give them."""
import pytest
import torch

from fastmlx_amd import ops

pytestmark = pytest.mark.gpu


def test_any_sequence_of_gradients(gpu):
    grads = [torch.full((4,), 3.0, device=gpu), torch.full((2, 8), -2.0, device=gpu).bfloat16()]
    want, norm = ops.clip_grad_norm(grads, 1.0)
    assert norm == 10
    for many in (tuple(grads), (g for g in grads), iter(grads), {i: g for i, g in enumerate(grads)}.values()):
        got, n = ops.clip_grad_norm(many, 1.0)
        assert n == 10 and len(got) == 2 and all(torch.equal(p, q) for p, q in zip(got, want))
    assert ops.grad_norm(g for g in grads) == 10
    outs = [torch.empty_like(g) for g in grads]
    ops.clip_grad_norm((g for g in grads), 1.0, outs=(o for o in outs))
    assert all(torch.equal(p, q) for p, q in zip(outs, want))
    with pytest.raises(ValueError):
        ops.clip_grad_norm((g for g in []), 1.0)
