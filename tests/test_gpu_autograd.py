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
    out, lse, residual = ops.sparse_attn_fwd(q, k, v, *lists, order=lists.order, return_residual=True)
    plain, plain_lse = ops.sparse_attn_fwd(q, k, v, *lists, order=lists.order, return_lse=True)
    assert torch.equal(plain, out) and torch.equal(plain_lse, lse)
    want = ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists, residual=residual)
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
    want = ops.sparse_attn_bwd(torch.ones_like(dout), q.detach(), k.detach(), v.detach(), out, lse, lists, klists,
                               residual=residual)
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


def dense_keep(mask, bs, N):
    return mask.repeat_interleave(bs, 1).repeat_interleave(bs, 2)[:, :N, :N]


def relative(got, want):
    return ((got.double().cpu() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N", [3, 7, 40])
def test_peaked_rows(mods, dtype, N):
    """Rows with nearly all of their weight on one key: dout v^T - delta is then a small difference.  Here the scores' spread
    makes P > 0.99 for most rows.  The result is a sum of terms that are each rounded once to the 16-bit type, the result once
    more: with independent roundings of at most u = eps / 2 each the relative error in the 2-norm is below sqrt(2) u, taken
    twice over for what cancels in the sums.  Without the residual delta alone is wrong by u |dout| |out|."""
    autograd, ops = mods
    g = torch.Generator().manual_seed(N)
    H, D = 4, 64
    q, k = (torch.randn(1, H, N, D, generator=g).mul(2.5).to(dtype) for _ in range(2))
    v, dout = (torch.randn(1, H, N, D, generator=g).to(dtype) for _ in range(2))
    mask = torch.ones(1, 1, 1, dtype=torch.bool, device="cuda")
    lists, klists = ops.tile_lists(mask, 64, N), ops.key_lists(mask, 64, N)
    ref = [t.double().requires_grad_(True) for t in (q, k, v)]
    out = torch.softmax(ref[0] @ ref[1].mT * D ** -0.5, -1) @ ref[2]
    want = torch.autograd.grad(out, ref, dout.double())
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(autograd.sparse_attention(*leaves, lists, klists), leaves, dout.cuda())
    for a, b in zip(got, want):
        assert relative(a, b) <= 2 * math.sqrt(2) * torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("norm,fused,D,bs", [("rms_head", True, 128, 128), ("layer", False, 64, 64), ("rms_all_heads", False, 64, 64),
                                             (None, True, 128, 64)])
def test_layer_against_64_bits(mods, norm, fused, D, bs):
    """Prologue and attention as a model runs them, float16 with a scaled loss.  The stored q, k, v and out are each rounded
    once, as are P, dS and every gradient on the way: a chain of at most ten roundings of at most u = 2^-11 whose effects on a
    gradient multiply with the scores' size (|s| <= 2^3: a score's relative error of 2 u moves P by 2^4 u).  2^6 u in all, in the
    2-norm."""
    autograd, ops = mods
    g = torch.Generator().manual_seed(5)
    B, S, H, dtype = 2, 330, 3, torch.float16
    W = H * D
    x = torch.randn(B, S, 3 * W, generator=g).to(dtype)
    width = W if norm == "rms_all_heads" else D
    params = [(1 + 0.1 * torch.randn(width, generator=g)).to(dtype) if norm else None for _ in range(2)]
    bias = [(0.1 * torch.randn(width, generator=g)).to(dtype) if norm == "layer" else None for _ in range(2)]
    ang = torch.rand(S - 30, D // 2, generator=g) * 6.28
    cos, sin = ang.cos(), ang.sin()
    dout = torch.randn(B, H, S, D, generator=g).to(dtype)
    nb = (S + bs - 1) // bs
    mask = (torch.rand(H, nb, nb, generator=g) < 0.5) | torch.eye(nb, dtype=torch.bool)

    def prologue(x, w, b):
        if norm == "rms_all_heads":
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        y = x.reshape(B, S, H, D)
        if norm == "rms_head":
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w
        if norm == "layer":
            y = torch.nn.functional.layer_norm(y, (D,), w, b, 1e-6)
        y = y.transpose(1, 2)
        a, c = y[:, :, :S - 30, 0::2], y[:, :, :S - 30, 1::2]
        co, si = cos.double(), sin.double()
        turned = torch.stack((a * co - c * si, a * si + c * co), -1).flatten(-2)
        return torch.cat((turned, y[:, :, S - 30:]), 2)

    x64 = x.double().requires_grad_(True)
    p64 = [None if p is None else p.double().requires_grad_(True) for p in params + bias]
    qx, kx, vx = x64.split(W, 2)
    q, k = prologue(qx, p64[0], p64[2]), prologue(kx, p64[1], p64[3])
    s = (q @ k.mT * D ** -0.5).masked_fill(~dense_keep(mask, bs, S), -math.inf)
    out64 = torch.softmax(s, -1) @ vx.reshape(B, S, H, D).transpose(1, 2)
    leaves64 = [x64] + [p for p in p64 if p is not None]
    want = torch.autograd.grad(out64, leaves64, dout.double())

    xd = x.cuda().requires_grad_(True)
    pd = [None if p is None else p.cuda().requires_grad_(True) for p in params + bias]
    lists, klists = ops.tile_lists(mask.cuda(), bs, S), ops.key_lists(mask.cuda(), bs, S)
    kw = dict(num_heads=H, norm=norm, q_weight=pd[0], k_weight=pd[1], q_bias=pd[2], k_bias=pd[3], rope_cos=cos.cuda(),
              rope_sin=sin.cuda(), rope_form="pair", rope_range=(0, S - 30))
    if fused:
        qkv = autograd.qkv_prologue(fused=xd, **kw)
    else:
        qkv = autograd.qkv_prologue(*xd.split(W, 2), **kw)
    out = autograd.sparse_attention(*qkv, lists, klists)
    got = torch.autograd.grad(out, [xd] + [p for p in pd if p is not None], dout.cuda())
    u = 2.0 ** -11
    assert relative(out.detach(), out64.detach()) <= 2 ** 6 * u
    for a, b in zip(got, want):
        assert a.shape == b.shape and relative(a, b) <= 2 ** 6 * u


def test_gradients_against_differences(mods):
    """The directional derivative of a loss against its difference quotient, both through the kernels.  out is rounded to
    float16: the quotient of the loss sum(dout * out) over 2 h carries at most u |dout . out|-like noise, a random sum of
    N H D terms of 2^-12 |dout||out| each, over 2 h; the step's own error is of third order in h.  With h = 2^-4 and
    directions of unit variance both stay below 2 % of the derivative here."""
    autograd, ops = mods
    q, k, v, dout, _, lists, klists = layer(mods, 3, N=260)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(autograd.sparse_attention(*leaves, lists, klists), leaves, dout)
    h = 2.0 ** -4
    for i in range(3):
        # along the gradient itself, rounded to signs: the derivative is then large against the noise
        step = grads[i].sign()
        plus, minus = ([t.clone() for t in (q, k, v)] for _ in range(2))
        plus[i] = (q, k, v)[i] + h * step
        minus[i] = (q, k, v)[i] - h * step
        moved = (plus[i].double() - minus[i].double())
        loss = [(ops.sparse_attn_fwd(*x, *lists).double() * dout.double()).sum() for x in (plus, minus)]
        quotient, derivative = loss[0] - loss[1], (moved * grads[i].double()).sum()
        assert abs((quotient - derivative) / derivative) <= 0.02


def test_engine_is_differentiable(mods):
    """The layer's own entry points give gradients where their inputs ask for them, and the same output where not."""
    import MoD.mod.attn_mask as am
    autograd, ops = mods
    q, k, v, dout, mask, lists, klists = layer(mods, 4, N=512, D=128, bs=128)
    valid = 430
    pad = torch.zeros(1, 512, dtype=torch.bool, device="cuda")
    pad[:, :valid] = True
    for kw, limits in (({}, {}), (dict(pre_defined_mask=pad, video_token_num=400),
                                  dict(q_split=400, kv_len_lo=448, kv_len_hi=valid))):
        plain = am.AttentionSparseEngine(q, k, v, mask.cuda(), block_size=128, **kw)
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = am.AttentionSparseEngine(*leaves, mask.cuda(), block_size=128, **kw)
        assert plain.grad_fn is None and torch.equal(out, plain)
        with torch.no_grad():
            assert am.AttentionSparseEngine(*leaves, mask.cuda(), block_size=128, **kw).grad_fn is None
        got = torch.autograd.grad(out, leaves, dout)
        other = [t.clone().requires_grad_(True) for t in (q, k, v)]
        want = torch.autograd.grad(autograd.sparse_attention(*other, lists, klists, **limits), other, dout)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # a mask of another shape stands for every block; use_dense takes the same way
    from MoD.mod.state import create_adaptive_mask_state
    state = create_adaptive_mask_state("wan", 3, 512, 0, 128, 4, warmup_steps=2, top_k=3, predict_T=5, block_size=128)
    leaves = [t[:1].clone().requires_grad_(True) for t in (q, k, v)]
    dense, _ = am.SparseAttentionWithMap(*leaves, state, logging.getLogger("t"), use_dense=True)
    engine = am.AttentionSparseEngine(*leaves, torch.ones(1, 2, 2, dtype=torch.bool, device="cuda"), block_size=128)
    for o in (dense, engine):
        got = torch.autograd.grad(o, leaves, dout[:1])
        ref = [t[:1].double().cpu().requires_grad_(True) for t in (q, k, v)]
        o64 = torch.softmax(ref[0] @ ref[1].mT * 128 ** -0.5, -1) @ ref[2]
        want = torch.autograd.grad(o64, ref, dout[:1].double().cpu())
        assert all(relative(a, b) <= 2 ** 2 * 2.0 ** -11 for a, b in zip(got, want))


def test_captured_step(mods):
    """Forward and backward in one graph, replayed on new values; a second graph captured meanwhile does not disturb it."""
    autograd, ops = mods
    q, k, v, dout, _, lists, klists = layer(mods, 6)
    static = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grad = dout.clone()

    def step():
        out = autograd.sparse_attention(*static, lists, klists)
        return (out.detach(),) + torch.autograd.grad(out, static, grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    for seed in (7, 8):
        fresh = layer(mods, seed)
        with torch.no_grad():
            for s, t in zip(static, fresh[:3]):
                s.copy_(t)
            grad.copy_(fresh[3])
        eager = [t.clone() for t in step()]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, eager))


def test_other_streams_and_repeats(mods):
    """Two steps at once on streams of their own, each as by itself; the same bits every time."""
    autograd, ops = mods
    jobs = [layer(mods, s, N=n, D=d) for s, n, d in ((10, 900, 64), (11, 500, 128))]
    alone = []
    for q, k, v, dout, _, lists, klists in jobs:
        out, lse = ops.sparse_attn_fwd(q, k, v, *lists, return_lse=True)
        alone.append((out, lse, ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        got = []
        for st, (q, k, v, dout, _, lists, klists), (out, lse, _) in zip(streams, jobs, alone):
            with torch.cuda.stream(st):
                got.append(ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists, check_status=False))
        torch.cuda.synchronize()
        for g, (_, _, want) in zip(got, alone):
            assert all(torch.equal(a, b) for a, b in zip(g, want))
    ops.raise_on_status(torch.device("cuda"))


def test_masked_places_hold_anything(mods):
    """Keys behind the padding limit are never read, and a query that attends to nothing gets and gives nothing."""
    autograd, ops = mods
    q, k, v, dout, mask, _, _ = layer(mods, 12, N=384, H=2, D=128, bs=128)
    mask = mask[:2].clone()
    mask[:, 1] = False
    lists, klists = ops.tile_lists(mask.cuda(), 128, 384), ops.key_lists(mask.cuda(), 128, 384)
    kw = dict(kv_len_lo=300, kv_len_hi=300)
    out, lse = ops.sparse_attn_fwd(q, k, v, *lists, return_lse=True, **kw)
    assert torch.isinf(lse[:, :, 128:256]).all() and (out[:, :, 128:256] == 0).all()
    want = ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists, **kw)
    assert (want[0][:, :, 128:256] == 0).all() and (want[1][:, :, 300:] == 0).all() and (want[2][:, :, 300:] == 0).all()
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:, :, 300:] = float("nan")
    bad_v[:, :, 300:] = float("inf")
    got = ops.sparse_attn_bwd(dout, q, bad_k, bad_v, out, lse, lists, klists, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    zero = ops.sparse_attn_bwd(dout, q, k, v, torch.zeros_like(out), torch.full_like(lse, -math.inf), lists, klists,
                               kv_len_lo=0, kv_len_hi=0)
    assert all((t == 0).all() for t in zero)


@pytest.mark.parametrize("norm", ["rms_head", "rms_all_heads", "layer"])
def test_frozen_norm_parameters(mods, norm):
    """Parameters that are not trained get no gradient and change nothing about the inputs'."""
    autograd, ops = mods
    g = torch.Generator().manual_seed(31)
    B, S, H, D = 2, 70, 3, 64
    x = [torch.randn(B, S, H * D, generator=g).half().cuda().requires_grad_(True) for _ in range(3)]
    width = H * D if norm == "rms_all_heads" else D
    w = [torch.randn(width, generator=g).half().cuda().requires_grad_(True) for _ in range(2)]
    dy = [torch.randn(B, H, S, D, generator=g).half().cuda() for _ in range(3)]

    def step(weights):
        return autograd.qkv_prologue(*x, num_heads=H, norm=norm, q_weight=weights[0], k_weight=weights[1])

    want = torch.autograd.grad(step(w), x, dy)
    got = torch.autograd.grad(step([t.detach() for t in w]), x, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    dx, params = ops.qkv_prologue_bwd(*dy, x[0].detach(), x[1].detach(), num_heads=H, norm=norm, q_weight=w[0].detach(),
                                      k_weight=w[1].detach(), param_grads=False)
    assert all(torch.equal(a, b) for a, b in zip(dx, want)) and all(p is None for p in params.values())


def test_a_later_step_reports_a_kernel_that_gave_up(mods):
    """The status words of an earlier kernel, set here by hand, end a later step once their copy has arrived."""
    autograd, ops = mods
    q, k, v, dout, _, lists, klists = layer(mods, 40)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(autograd.sparse_attention(*leaves, lists, klists), leaves, dout)
    torch.cuda.synchronize()
    ops.check_posted_status(q.device)
    ops._status_words(q.device).copy_(torch.tensor([3, 1, 2, 0], dtype=torch.int32))
    ops.post_status(q.device)
    torch.cuda.synchronize()
    with pytest.raises(Exception, match="bounded wait expired"):
        autograd.sparse_attention(*leaves, lists, klists)
    got = torch.autograd.grad(autograd.sparse_attention(*leaves, lists, klists), leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    ops.check_health(q.device)
