"""The differentiable forms: prologue and sparse attention as a training step uses them, against the whole in 64 bits."""
import logging
import math
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mods():
    from moddit_b200 import autograd, ops
    return autograd, ops


def layer(mods, seed=0, N=300, H=3, D=64, bs=64, dtype=torch.float16, density=0.5):
    autograd, ops = mods
    g = torch.Generator().manual_seed(seed)
    q, k, v, dout = (torch.randn(2, H, N, D, generator=g).to(dtype).cuda() for _ in range(4))
    nb = (N + bs - 1) // bs
    mask = (torch.rand(H, nb, nb, generator=g) < density) | torch.eye(nb, dtype=torch.bool)
    lists, klists = ops.tile_lists(mask.cuda(), bs, N), ops.key_lists(mask.cuda(), bs, N)
    return q, k, v, dout, mask, lists, klists


def test_sparse_attention_is_the_two_calls(mods):
    autograd, ops = mods
    q, k, v, dout, _, lists, klists = layer(mods)
    out, lse = ops.sparse_attn_fwd(q, k, v, *lists, order=lists.order, return_lse=True)
    want = ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    got = autograd.sparse_attention(*leaves, lists, klists)
    assert torch.equal(got, out)
    got.backward(dout)
    assert all(torch.equal(leaf.grad, w) for leaf, w in zip(leaves, want))
    # inputs and gradients of other strides are copied; a leaf without a gradient gets none
    leaves = [t.transpose(1, 2).contiguous().requires_grad_(i != 1) for i, t in enumerate((q, k, v))]
    got = autograd.sparse_attention(*[t.transpose(1, 2) for t in leaves], lists, klists)
    grads = torch.autograd.grad(got, [leaves[0], leaves[2]], dout.transpose(1, 2).contiguous().transpose(1, 2))
    assert torch.equal(grads[0].transpose(1, 2), want[0]) and torch.equal(grads[1].transpose(1, 2), want[2])
    # a gradient that is one value for everything
    ones = torch.autograd.grad(autograd.sparse_attention(*[t.requires_grad_(True) for t in (q, k, v)], lists, klists).sum(), (q, k, v))
    want = ops.sparse_attn_bwd(torch.ones_like(dout), q.detach(), k.detach(), v.detach(), out, lse, lists, klists)
    assert all(torch.equal(a, b) for a, b in zip(ones, want))


def test_from_another_thread(mods):
    autograd, ops = mods
    q, k, v, dout, _, lists, klists = layer(mods, 1)
    out, lse = ops.sparse_attn_fwd(q, k, v, *lists, return_lse=True)
    want = ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists)
    got = []
    t = threading.Thread(target=lambda: got.extend(ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists)))
    t.start()
    t.join()
    assert len(got) == 3 and all(torch.equal(a, b) for a, b in zip(got, want))
