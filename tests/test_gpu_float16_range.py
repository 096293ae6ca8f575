"""float16 gradients at both ends of the type's range.

Tolerance, in the 2-norm.  With independent roundings of at most u = 2^-11 of each value, dS and the stored result add at most
sqrt(2) u; twice that for what cancels in the sums and for the float32 arithmetic, as on peaked rows.  A dS below 2^-14 is held
in steps of 2^-24: an error of at most 2^-25 for each of the n keys of a row, independent again, makes 2^-25 scale sqrt(n)
rms(k) in each value of dq; the stored value itself is off by at most 2^-25 there.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


@pytest.fixture(scope="module")
def mods():
    from moddit_b200 import autograd, ops
    return autograd, ops


def gradients(q, k, v, dout, rows):
    """(dq of the first `rows` rows, which see everything, dk, dv) in 64 bits."""
    q, k, v, dout = (t.double() for t in (q[:, :, :rows], k, v, dout[:, :, :rows]))
    scale = q.shape[-1] ** -0.5
    p = torch.softmax(q @ k.mT * scale, -1)
    ds = p * (dout @ v.mT - (dout * (p @ v)).sum(-1, keepdim=True))
    return ds @ k * scale, ds.mT @ q * scale, p.mT @ dout


def relative(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size,scaled", [(1.0, 1), (0.02, 2.0 ** 6), (0.002, 2.0 ** 9), (0.002, 1)])
def test_small_gradients_of_long_rows(mods, D, size, scaled):
    """17,000 keys.  A loss scaled so that dout is about 1 gives dq to its rounding; without, dS loses what the bound counts."""
    autograd, ops = mods
    N, bs = 17000, 128
    g = torch.Generator(device="cuda").manual_seed(D)
    q, k, v, dout = (torch.randn(1, 1, N, D, generator=g, device="cuda") for _ in range(4))
    dout = dout * size * scaled
    q, k, v, dout = (t.half() for t in (q, k, v, dout))
    nb = (N + bs - 1) // bs
    mask = torch.zeros(1, nb, nb, dtype=torch.bool, device="cuda")
    mask[:, 0] = True                                    # 128 rows that see every key
    lists, klists = ops.tile_lists(mask, bs, N), ops.key_lists(mask, bs, N)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dq, _, _ = torch.autograd.grad(autograd.sparse_attention(*leaves, lists, klists), leaves, dout)
    want, _, _ = gradients(q.detach(), k.detach(), v.detach(), dout, bs)
    bound = 2 * math.sqrt(2) * U
    steps = 2.0 ** -25 * (1 + D ** -0.5 * math.sqrt(N) * k.detach().double().square().mean().sqrt().item())
    bound += steps * math.sqrt(want.numel()) / want.norm().item()
    assert relative(dq[:, :, :bs], want) <= bound
    if scaled > 1:
        assert relative(dq[:, :, :bs], want) <= 2.1 * math.sqrt(2) * U           # the steps no longer count


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [64.0, 1024.0])
def test_large_gradients_of_short_rows(mods, D, size):
    """Four keys and a loss scaled as high as the results allow: dS reaches some thousands and none overflows."""
    autograd, ops = mods
    g = torch.Generator(device="cuda").manual_seed(D)
    q, k, v, dout = (torch.randn(1, 64, 4, D, generator=g, device="cuda") for _ in range(4))
    q, k, v, dout = (t.half() for t in (q, k, v, dout * size))
    mask = torch.ones(1, 1, 1, dtype=torch.bool, device="cuda")
    lists, klists = ops.tile_lists(mask, 64, 4), ops.key_lists(mask, 64, 4)
    want = gradients(q, k, v, dout, 4)
    assert all(w.abs().max().item() < 60000 for w in want)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(autograd.sparse_attention(*leaves, lists, klists), leaves, dout)
    for a, b in zip(got, want):
        assert torch.isfinite(a).all() and relative(a, b) <= 2 * math.sqrt(2) * U
