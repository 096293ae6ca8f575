"""Which calls queue a copy of the kernels' status words."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_deferred_backward_reports_itself(monkeypatch):
    """`check_status="deferred"` keeps a distance between the copies unless it is told not to; what a kernel within the distance
    reports is in the next copy."""
    from moddit_b200 import autograd, ops
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, dout = (torch.randn(1, 2, 300, 64, generator=g, device="cuda").half() for _ in range(4))
    mask = torch.ones(1, 3, 3, dtype=torch.bool, device="cuda")
    lists, klists = ops.tile_lists(mask, 128, 300), ops.key_lists(mask, 128, 300)
    posts, post = [], ops.post_status
    monkeypatch.setattr(ops, "post_status", lambda device, spacing=0.0: posts.append(spacing) or post(device, spacing))
    out, lse = ops.sparse_attn_fwd(q, k, v, *lists, return_lse=True, check_status="deferred")
    ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists, check_status="deferred", status_spacing=0)
    ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists, check_status="deferred")
    assert posts == [0.0, 0.0, ops.STATUS_SPACING]
    torch.cuda.synchronize()
    ops.check_posted_status(q.device)
    ops._status_words(q.device)[0] = 7                      # as a kernel of this call would leave it
    ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists, check_status="deferred", status_spacing=0)
    torch.cuda.synchronize()
    with pytest.raises(Exception, match="bounded wait expired"):
        ops.check_posted_status(q.device)
    ops.post_status(q.device)
    ops._status_words(q.device)[0] = 7
    ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists, check_status="deferred", status_spacing=60.0)
    torch.cuda.synchronize()
    ops.check_posted_status(q.device)                       # the copy is from before
    ops.sparse_attn_fwd(q, k, v, *lists, check_status="deferred")
    torch.cuda.synchronize()
    with pytest.raises(Exception, match="bounded wait expired"):
        ops.check_posted_status(q.device)
    posts.clear()
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    autograd.sparse_attention(*leaves, lists, klists).backward(dout)
    assert posts == [ops.STATUS_SPACING] * 2
    ops.check_health(q.device)
