"""Gradients of the attention prologue against its derivative in 64 bits.

Tolerance.  A result is rounded once to the 16-bit type: u |value|, u = eps / 2 (bf16 2^-8, fp16 2^-11; fp16 values below its
normal range 2^-25).  The arithmetic is float32: a rotated pair, the row's factor and the two row sums of D <= 128 or
H * D <= 2^11 terms (chains of at most 2^6 additions, then a tree) are each wrong by less than 2^-17 of the sum of their terms'
magnitudes; a handful of them multiply in one value: 2^-14 of the magnitudes.  A weight gradient adds at most 2^9 terms in a
thread, then 2^5 threads, then rows of partial sums: (2^9 + 2^5 + 2^7) 2^-24 < 2^-14 of its terms' magnitudes, and the
2^-14 of those terms themselves.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from moddit_b200 import ops as _ops
    return _ops


def tables(rows, D, form, seed):
    g = torch.Generator().manual_seed(seed)
    ang = torch.rand(rows, D // 2, generator=g) * 6.28
    if form == "pair":
        return ang.cos().contiguous(), ang.sin().contiguous()
    cos, sin = ang.cos().repeat_interleave(2, 1), ang.sin().repeat_interleave(2, 1)
    return cos * torch.linspace(0.9, 1.1, D), sin * torch.linspace(1.1, 0.9, D)      # tells the forms apart


def prologue64(x, w, b, norm, eps, H, cos, sin, form, lo, hi):
    B, S, W = x.shape
    D = W // H
    if norm == "rms_all_heads":
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
        x = x if w is None else x * w
    y = x.reshape(B, S, H, D)
    if norm == "rms_head":
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
        y = y if w is None else y * w
    if norm == "layer":
        y = y - y.mean(-1, keepdim=True)
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
        y = y if w is None else y * w
        y = y if b is None else y + b
    y = y.transpose(1, 2)
    if cos is not None:
        cos, sin = cos.double(), sin.double()
        if form == "pair":
            cos, sin = cos.repeat_interleave(2, 1), sin.repeat_interleave(2, 1)
        ce, co = cos[:, 0::2], cos[:, 0::2] if form == "even_cos_odd_sin" else cos[:, 1::2]
        se, so = sin[:, 1::2] if form == "even_cos_odd_sin" else sin[:, 0::2], sin[:, 1::2]
        a, c = y[:, :, lo:hi, 0::2], y[:, :, lo:hi, 1::2]
        turned = torch.stack((a * ce - c * se, a * so + c * co), -1).flatten(-2)
        y = torch.cat((y[:, :, :lo], turned, y[:, :, hi:]), 2)
    return y


def magnitudes(x, g, w, norm, eps, H):
    """Sums of the magnitudes that add up to dx, dw and db; `g` the absolute gradient before the rotation."""
    B, S, W = x.shape
    D = W // H
    x, g = x.double().reshape(B, S, H, D), g.transpose(1, 2)
    if norm is None:
        return g.reshape(B, S, W), None, None
    dims = (2, 3) if norm == "rms_all_heads" else (3,)
    top = x.abs()
    if norm == "layer":
        top = top + x.mean(dims, keepdim=True).abs()
        x = x - x.mean(dims, keepdim=True)
    r = torch.rsqrt(x.square().mean(dims, keepdim=True) + eps)
    xhat = top * r
    gw = g * (1.0 if w is None else w.double().abs().reshape(H, D) if norm == "rms_all_heads" else w.double().abs())
    dx = r * (gw + gw.mean(dims, keepdim=True) + xhat * (gw * xhat).mean(dims, keepdim=True))
    over = (0, 1) if norm == "rms_all_heads" else (0, 1, 2)
    return dx.reshape(B, S, W), (g * xhat).sum(over).flatten(), g.sum(over).flatten()


def within(got, want, mag, dtype, what):
    u = torch.finfo(dtype).eps / 2
    got = got.double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), what
    bound = u * (1 + 2.0 ** -8) * want.abs() + 2.0 ** -14 * mag + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
    worst = ((got - want).abs() / bound).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3f} of the bound"


CASES = [
    # B, S, H, D, norm, rope form, lo, hi, rows before, fused
    (1, 1, 1, 64, "layer", None, 0, 0, 0, False),
    (1, 1, 2, 128, "rms_head", "elementwise", 0, 1, 0, True),
    (2, 1, 3, 128, "rms_all_heads", "pair", 0, 1, 5, False),
    (2, 1, 2, 64, "rms_head", "pair", 0, 1, 0, True),
    (1, 130, 3, 128, "rms_head", "elementwise", 0, 100, 0, True),
    (2, 197, 2, 64, "layer", "even_cos_odd_sin", 40, 197, 13, False),
    (2, 300, 3, 128, "layer", "pair", 0, 300, 0, True),
    (1, 333, 5, 64, "rms_all_heads", "elementwise", 7, 300, 0, True),
    (2, 77, 16, 128, "rms_all_heads", "even_cos_odd_sin", 0, 77, 128, False),
    (1, 1000, 2, 128, None, "elementwise", 0, 1000, 0, False),
    (1, 50, 3, 64, None, None, 0, 0, 0, False),
    (1, 5000, 7, 64, "rms_head", "even_cos_odd_sin", 0, 4999, 0, False),
    # wide tokens: their sums in shared memory and the kernel's own arrays pass 48 KB together, then each
    (1, 19, 80, 128, "rms_all_heads", "pair", 0, 19, 0, False),
    (1, 11, 192, 64, "rms_all_heads", "elementwise", 3, 9, 0, True),
    (1, 10, 200, 128, "rms_all_heads", None, 0, 0, 0, False),
    # a token of eight pieces; the widest that is read once, an odd number of tokens and a rotated part; one wider
    (3, 7, 1, 64, "rms_all_heads", "pair", 2, 6, 1, True),
    (2, 331, 40, 128, "rms_all_heads", "elementwise", 5, 300, 0, False),
    (2, 45, 41, 128, "rms_all_heads", "pair", 0, 45, 2, False),
    # more pairs of tokens than blocks, a sample per round of them and several
    (5, 1201, 9, 64, "rms_all_heads", "even_cos_odd_sin", 1, 1200, 3, False),
    (300, 3, 2, 128, "rms_all_heads", "pair", 0, 3, 0, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:6])))
def test_gradients(ops, dtype, case):
    B, S, H, D, norm, form, lo, hi, before, fused = case
    g = torch.Generator().manual_seed(S * H + D)
    W, eps = H * D, 1e-6
    if fused:
        x = torch.randn(B, S, 3 * W, generator=g).to(dtype).split(W, 2)
    else:
        x = [(torch.randn(B, S, W, generator=g) * (1 + i) + 0.2).to(dtype) for i in range(3)]
    dy = [torch.randn(B, H, before + S + 3, D, generator=g).to(dtype) for _ in range(3)]
    width = W if norm == "rms_all_heads" else D
    w = [(1 + 0.2 * torch.randn(width, generator=g)).to(dtype) if norm else None for _ in range(2)]
    b = [(0.2 * torch.randn(width, generator=g)).to(dtype) if norm == "layer" else None for _ in range(2)]
    cos, sin = tables(hi - lo, D, form, 3) if form else (None, None)
    cuda = lambda t: None if t is None else t.cuda()          # noqa: E731
    if fused:
        whole = torch.cat(x, 2).cuda()
        xd, buffer = whole.split(W, 2), torch.full((B, S, 3 * W + 8), 7.0, device="cuda", dtype=dtype)
        out = tuple(buffer[:, :, i * W:(i + 1) * W] for i in range(3))
    else:
        xd, out = [cuda(t) for t in x], None
    dx, grads = ops.qkv_prologue_bwd(*map(cuda, dy), xd[0], xd[1], num_heads=H, norm=norm, q_weight=cuda(w[0]), q_bias=cuda(b[0]),
                                     k_weight=cuda(w[1]), k_bias=cuda(b[1]), eps=eps, rope_cos=cuda(cos), rope_sin=cuda(sin),
                                     rope_form=form or "pair", rope_range=(lo, hi), src_row0=before, n_tokens=S, out=out)
    if fused:
        assert dx[2].data_ptr() == out[2].data_ptr()
        assert torch.equal(buffer[:, :, 3 * W:], torch.full_like(buffer[:, :, 3 * W:], 7.0))
    for i, name in enumerate(("q", "k", "v")):
        gy = dy[i][:, :, before:before + S].double()
        xi = x[i].double().requires_grad_(True)
        wi = w[i].double().requires_grad_(True) if i < 2 and norm else None
        bi = b[i].double().requires_grad_(True) if i < 2 and norm == "layer" else None
        turn = (cos, sin) if i < 2 else (None, None)
        y = prologue64(xi, wi, bi, norm if i < 2 else None, eps, H, *turn, form, lo, hi)
        want = torch.autograd.grad(y, [t for t in (xi, wi, bi) if t is not None], gy)
        # the absolute gradient before the rotation: |g0||c| + |g1||s|
        flat = gy.abs()
        if turn[0] is not None:
            probe = flat[:, :, lo:hi].unflatten(-1, (-1, 2)).sum(-1, keepdim=True).expand(-1, -1, -1, -1, 2).flatten(-2) * 1.2
            flat = torch.cat((flat[:, :, :lo], probe, flat[:, :, hi:]), 2)
        mdx, mdw, mdb = magnitudes(x[i], flat, w[i] if i < 2 else None, norm if i < 2 else None, eps, H)
        within(dx[i], want[0], mdx, dtype, "d" + name)
        if i < 2 and norm:
            within(grads[name + "_weight"], want[1], mdw, dtype, name + " weight")
        if i < 2 and norm == "layer":
            within(grads[name + "_bias"], want[2], mdb, dtype, name + " bias")


def test_missing_parts(ops):
    """One gradient alone, no parameters: the others are neither read nor written."""
    g = torch.Generator().manual_seed(1)
    dk, k = torch.randn(1, 2, 40, 64, generator=g).bfloat16().cuda(), torch.randn(1, 40, 128, generator=g).bfloat16().cuda()
    (dq_in, dk_in, dv_in), grads = ops.qkv_prologue_bwd(None, dk, None, None, k, num_heads=2, norm="rms_head")
    assert dq_in is None and dv_in is None and all(v is None for v in grads.values())
    both, _ = ops.qkv_prologue_bwd(dk, dk, dk, k, k, num_heads=2, norm="rms_head", k_weight=torch.ones(64, device="cuda", dtype=torch.bfloat16))
    assert torch.equal(both[1], dk_in) and torch.equal(both[0], dk_in)
    assert torch.equal(both[2], dk.transpose(1, 2).reshape(1, 40, 128))


@pytest.mark.parametrize("H", [5, 41])
def test_a_token_norm_of_some_tensors(ops, H):
    """q, k and v share blocks where all are given: any of them alone gives the same bits of its gradient."""
    g = torch.Generator().manual_seed(H)
    B, S, D = 2, 51, 128
    dy = [torch.randn(B, H, S, D, generator=g).half().cuda() for _ in range(3)]
    x = [torch.randn(B, S, H * D, generator=g).half().cuda() for _ in range(2)]
    w = [torch.randn(H * D, generator=g).half().cuda() for _ in range(2)]
    kw = dict(num_heads=H, norm="rms_all_heads", q_weight=w[0], k_weight=w[1])
    want, _ = ops.qkv_prologue_bwd(*dy, *x, **kw)
    for keep in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        some = [t if i in keep else None for i, t in enumerate(dy)]
        got, params = ops.qkv_prologue_bwd(*some, *x, n_tokens=S, **kw)
        for i in range(3):
            assert got[i] is None if i not in keep else torch.equal(got[i], want[i])
        assert (params["q_weight"] is None) == (0 not in keep) and (params["k_weight"] is None) == (1 not in keep)
