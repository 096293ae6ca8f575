"""Gradients of the block-sparse attention against the formula in 64 bits, and its work lists against the mask.

Tolerance.  With u = eps / 2 of the 16-bit type (bf16 2^-8, fp16 2^-11) P and dS are each rounded once (u per value) and
every output once (u).  The rounding errors of the terms of a sum are independent, but the bound below takes them as if they
all had one sign: |error(dv)| <= u * P^T|dout| + u * |dv|, |error(dq)| <= u * scale * |dS||k| + u * |dq|, and the same for dk.
Float32 arithmetic adds to that: a score is known to about (D + 4) 2^-24 of the sum of its terms' magnitudes and its exponential
doubles as much relative error in P per unit, which with |s| below 2^6 and lse rounded to float32 is below 2^-24 * (D * 2^4 + 2^7)
< 2^-12.9; dP - delta is wrong by at most (D + 2) 2^-24 of sum |dout||v| + sum |dout||out|, carried as `wide` below; float32 sums
over N <= 2^11 rows add N 2^-24 <= 2^-13 of the same sums.  Together: 2^-11.9 of P^T|dout|, and 2^-11.9 of |dS||k| plus
2^-13 of P (wide)|k|.  Values of float16 below its normal range keep an absolute error of at most 2^-25: for P, held 2^8
times larger, 2^-33 of sum |dout|; for dS 2^-25 of sum |k|; for the stored result 2^-25.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from moddit_b200 import ops as _ops
    return _ops


def make(B, H, N, D, dtype, seed, gain=1.0, grad=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k = ((torch.randn(B, H, N, D, generator=g) * gain).to(dtype) for _ in range(2))
    v = torch.randn(B, H, N, D, generator=g).to(dtype)
    dout = (torch.randn(B, H, N, D, generator=g) * grad).to(dtype)
    return q, k, v, dout


def tokens(mask, bs, N, H, q_split=None, kv_lo=None, kv_hi=None):
    """(H, N, N) bool: the pairs that the kernels keep."""
    keep = mask.repeat_interleave(bs, 1).repeat_interleave(bs, 2)[:, :N, :N].repeat(H // mask.shape[0], 1, 1)
    col, row = torch.arange(N), torch.arange(N)[:, None]
    q_split, kv_lo, kv_hi = (N if x is None else x for x in (q_split, kv_lo, kv_hi))
    return keep & torch.where(row < q_split, col < kv_lo, col < kv_hi)


def reference(q, k, v, dout, keep, scale, out=None, lse=None):
    """(out, lse, dq, dk, dv, bounds' sums) in 64 bits on the inputs' values."""
    q, k, v, do = (t.double() for t in (q, k, v, dout))
    s = torch.matmul(q, k.mT) * scale
    s = s.masked_fill(~keep, -math.inf)
    ref_lse = torch.logsumexp(s, -1)
    p = torch.where(keep, torch.exp(s - torch.where(ref_lse.isinf(), 0.0, ref_lse)[..., None]), 0.0)
    ref_out = torch.matmul(p, v)
    if lse is not None:
        p = torch.where(keep, torch.exp(s - torch.where(lse.isinf(), 0.0, lse).double()[..., None]), 0.0)
    o = ref_out if out is None else out.double()
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (torch.matmul(do, v.mT) - delta)
    wide = p * (torch.matmul(do.abs(), v.abs().mT) + (do.abs() * o.abs()).sum(-1, keepdim=True))
    sums = dict(dv=torch.matmul(p.mT, do.abs()), dq=torch.matmul(ds.abs(), k.abs()) * scale,
                dk=torch.matmul(ds.abs().mT, q.abs()) * scale, dq_wide=torch.matmul(wide, k.abs()) * scale,
                dk_wide=torch.matmul(wide.mT, q.abs()) * scale,
                dv_count=torch.matmul(keep.double().mT, do.abs()).expand_as(v), dq_count=torch.matmul(keep.double(), k.abs()) * scale,
                dk_count=torch.matmul(keep.double().mT, q.abs()) * scale)
    return (ref_out, ref_lse, torch.matmul(ds, k) * scale, torch.matmul(ds.mT, q) * scale, torch.matmul(p.mT, do), sums)


def check(got, want, sums, dtype):
    u = torch.finfo(dtype).eps / 2
    half = dtype == torch.float16
    for name, g, w in zip(("dq", "dk", "dv"), got, want):
        g = g.double().cpu()
        assert torch.isfinite(g).all(), name
        bound = (u + 2.0 ** -11.9) * sums[name] + u * w.abs() * (1 + 2.0 ** -8) + 1e-30
        if name != "dv":
            bound = bound + 2.0 ** -13 * sums[name + "_wide"]
        if half:
            bound = bound + 2.0 ** (-33 if name == "dv" else -25) * sums[name + "_count"] + 2.0 ** -25
        worst = ((g - w).abs() / bound).max().item()
        assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"


def run(ops, q, k, v, dout, mask, bs, order=True, **kw):
    dev = [t.cuda() for t in (q, k, v, dout)]
    N = q.shape[2]
    lists, klists = ops.tile_lists(mask.cuda(), bs, N), ops.key_lists(mask.cuda(), bs, N)
    out, lse = ops.sparse_attn_fwd(*dev[:3], lists.counts, lists.entries, order=lists.order, return_lse=True, **kw)
    got = ops.sparse_attn_bwd(dev[3], *dev[:3], out, lse, lists, klists, **kw)
    return out.cpu(), lse.cpu(), got


CASES = [
    # B, H, N, D, bs, density, Hm, q_split, kv_lo, kv_hi
    (1, 1, 1, 128, 128, 1.0, 1, None, None, None),
    (1, 2, 1, 64, 64, 1.0, 2, None, None, None),
    (1, 2, 127, 64, 64, 1.0, 2, None, None, None),
    (1, 2, 128, 128, 128, 1.0, 2, None, None, None),
    (2, 3, 129, 128, 64, 0.7, 1, None, None, None),
    (1, 2, 333, 64, 64, 0.5, 2, None, None, None),
    (2, 2, 640, 128, 128, 0.4, 2, None, None, None),
    (1, 3, 1000, 128, 64, 0.35, 3, None, None, None),
    (1, 2, 1000, 64, 64, 0.1, 1, None, None, None),
    (1, 2, 777, 128, 64, 0.6, 2, 600, 640, 601),
    (2, 2, 777, 64, 64, 0.6, 1, 601, 704, 650),
    (1, 2, 512, 128, 128, 1.0, 2, 300, 256, 129),
    (1, 1, 512, 64, 128, 1.0, 1, 0, 512, 65),
    (1, 1, 2048, 128, 128, 0.3, 1, None, None, None),
    # limits far apart: first queries that see few or no keys, keys that only the last queries see, and the other way round
    (1, 2, 900, 128, 64, 0.5, 2, 512, 256, 900),
    (2, 2, 900, 64, 64, 0.5, 1, 448, 130, 900),
    (1, 2, 900, 64, 128, 1.0, 2, 600, 0, 900),
    (1, 2, 900, 128, 128, 1.0, 1, 700, 900, 0),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:5])))
def test_gradients(ops, dtype, case):
    B, H, N, D, bs, density, Hm, q_split, kv_lo, kv_hi = case
    q, k, v, dout = make(B, H, N, D, dtype, N + D)
    nb = (N + bs - 1) // bs
    mask = torch.rand(Hm, nb, nb, generator=torch.Generator().manual_seed(N)) < density
    out, lse, got = run(ops, q, k, v, dout, mask, bs, q_split=q_split, kv_len_lo=kv_lo, kv_len_hi=kv_hi)
    keep = tokens(mask, bs, N, H, q_split, kv_lo, kv_hi)
    _, _, dq, dk, dv, sums = reference(q, k, v, dout, keep, D ** -0.5, out, lse)
    check(got, (dq, dk, dv), sums, dtype)


@pytest.mark.parametrize("bs,N,H,density,limit", [(128, 1, 1, 1.0, None), (128, 700, 3, 0.4, None), (64, 700, 3, 0.3, None),
                                                  (64, 5000, 2, 0.05, 60), (128, 20000, 2, 0.1, None), (64, 8192, 1, 1.0, None)])
def test_key_lists(ops, bs, N, H, density, limit):
    nb, nt = (N + bs - 1) // bs, (N + 127) // 128
    mask = torch.rand(H, nb, nb, generator=torch.Generator().manual_seed(N)) < density
    lists = ops.key_lists(mask.cuda(), bs, N, kv_block_limit=limit)
    counts, entries = lists.counts.cpu(), lists.entries.cpu()
    want = mask.clone()
    if limit is not None:
        want[:, :, limit:] = False
    per = 128 // bs
    full = torch.zeros(H, nt * per, nt * per, dtype=torch.bool)
    full[:, :nb, :nb] = want
    bits = torch.zeros(H, nt, nt, dtype=torch.int32)
    for rh in range(2):
        for ch in range(2):
            part = full[:, rh % per::per, ch % per::per]
            bits |= part.int() << (2 * rh + ch)
    for h in range(H):
        for t in range(nt):
            rows = torch.nonzero(bits[h, :, t]).flatten().int()
            assert counts[h, t].item() == rows.numel()
            assert torch.equal(entries[h, t, :rows.numel()], (rows << 8) | bits[h, rows.long(), t])
    order = lists.order.cpu().flatten()
    assert torch.equal(order.sort().values, torch.arange(H * nt, dtype=torch.int32))


def test_refusals(ops):
    """What only a device call can tell: shapes, types, layouts and lists that do not belong together."""
    q, k, v, dout = (t.cuda() for t in make(1, 2, 200, 64, torch.float16, 1))
    mask = torch.ones(2, 2, 2, dtype=torch.bool, device="cuda")
    lists, klists = ops.tile_lists(mask, 128, 200), ops.key_lists(mask, 128, 200)
    out, lse = ops.sparse_attn_fwd(q, k, v, *lists, return_lse=True)
    good = dict(dout=dout, q=q, k=k, v=v, out=out, lse=lse, lists=lists, key_lists=klists)

    def refused(error, text, **kw):
        with pytest.raises(error, match=text):
            ops.sparse_attn_bwd(**{**good, **kw})

    refused(ValueError, "identical shapes", dout=dout[:, :, :100].contiguous())
    refused(ValueError, "identical shapes", v=v.bfloat16())
    refused(ValueError, "identical shapes", residual=out.bfloat16())
    refused(ValueError, "contiguous", dout=dout.transpose(1, 2).contiguous().transpose(1, 2))
    refused(ValueError, "lse", lse=lse.half())
    refused(ValueError, "lse", lse=lse[:, :1])
    refused(TypeError, "float16 or bfloat16", **{n: good[n].float() for n in ("dout", "q", "k", "v", "out")})
    refused(TypeError, "key_lists", lists=klists, key_lists=lists)
    refused(TypeError, "key_lists", key_lists=lists)
    refused(ValueError, "sequence length", key_lists=ops.key_lists(torch.ones(2, 3, 3, dtype=torch.bool, device="cuda"), 128, 300))
    refused(ValueError, "one mask", key_lists=ops.key_lists(mask[:1], 128, 200))
    refused(ValueError, "kv_len", kv_len_lo=201)
    refused(ValueError, "softmax_scale", softmax_scale=-1.0)
    refused(ValueError, "CUDA", lse=lse.cpu())
    with pytest.raises(ValueError, match="one launch"):
        ops.sparse_attn_fwd(q, k, v, *lists, return_residual=True, pairs_beside=4)
    odd = torch.empty(q.numel() + 4, device="cuda", dtype=q.dtype)[4:].view(q.shape)      # 8 bytes off a 16-byte boundary
    refused(RuntimeError, "aligned", q=odd)
    wide = [torch.zeros(1, 2, 200, 96, device="cuda", dtype=torch.float16) for _ in range(5)]
    refused(RuntimeError, "head_dim", **dict(zip(("dout", "q", "k", "v", "out"), wide)))
    ops.sparse_attn_bwd(**good)


def test_batches_share_a_mask_head_by_head(ops):
    """Head bh of a batch of two uses mask head bh % Hm, with limits, at both head dimensions: each sample equals its own call."""
    for D in (64, 128):
        q, k, v, dout = (t.cuda() for t in make(2, 4, 450, D, torch.bfloat16, D))
        mask = (torch.rand(2, 8, 8, generator=torch.Generator().manual_seed(3)) < 0.6).cuda()
        lists, klists = ops.tile_lists(mask, 64, 450), ops.key_lists(mask, 64, 450)
        kw = dict(q_split=300, kv_len_lo=448, kv_len_hi=401)
        out, lse = ops.sparse_attn_fwd(q, k, v, *lists, order=lists.order, return_lse=True, **kw)
        got = ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists, **kw)
        for b in range(2):
            for h in range(0, 4, 2):
                part = [t[b:b + 1, h:h + 2].contiguous() for t in (dout, q, k, v, out, lse)]
                want = ops.sparse_attn_bwd(*part, lists, klists, **kw)
                assert all(torch.equal(g[b:b + 1, h:h + 2], w) for g, w in zip(got, want))


def test_long_rows_of_few_blocks(ops):
    """65,600 rows: lists of tiles far apart, a column that every row keeps and rows that keep everything, against the same
    gradients of the kept blocks gathered into a short dense problem in 64 bits."""
    N, D, bs = 65600, 128, 128
    nb = (N + bs - 1) // bs
    q, k, v, dout = (t.cuda() for t in make(1, 1, N, D, torch.bfloat16, 9))
    mask = torch.zeros(1, nb, nb, dtype=torch.bool, device="cuda")
    cols = [0, 17, 400, nb - 1]
    mask[0, 300, cols] = True
    mask[0, nb - 1, cols[1:]] = True
    lists, klists = ops.tile_lists(mask, bs, N), ops.key_lists(mask, bs, N)
    out, lse = ops.sparse_attn_fwd(q, k, v, *lists, return_lse=True)
    dq, dk, dv = ops.sparse_attn_bwd(dout, q, k, v, out, lse, lists, klists)
    rows = torch.cat([torch.arange(300 * bs, 301 * bs), torch.arange((nb - 1) * bs, N)])
    keys = torch.cat([torch.arange(c * bs, min(N, (c + 1) * bs)) for c in cols])
    keep = torch.ones(1, rows.numel(), keys.numel(), dtype=torch.bool)
    keep[:, bs:, :bs] = False
    pick = lambda t, i: t[:, :, i.to(t.device)].cpu()          # noqa: E731
    args = (pick(q, rows), pick(k, keys), pick(v, keys), pick(dout, rows), keep, D ** -0.5, pick(out, rows), pick(lse, rows))
    _, _, wq, wk, wv, sums = reference(*args)
    check((pick(dq, rows), pick(dk, keys), pick(dv, keys)), (wq, wk, wv), sums, torch.bfloat16)
    gone = torch.ones(N, dtype=torch.bool)
    gone[rows] = False
    assert (dq[:, :, gone.cuda()] == 0).all()
    gone[:] = True
    gone[keys] = False
    assert (dk[:, :, gone.cuda()] == 0).all() and (dv[:, :, gone.cuda()] == 0).all()


@pytest.mark.parametrize("D", [64, 128])
def test_rows_that_the_limits_leave_empty_hold_anything(ops, D):
    """Blocks of 64 queries that see no key because of the limits are not multiplied: NaN there reaches nothing."""
    N, split = 700, 320
    q, k, v, dout = make(1, 2, N, D, torch.bfloat16, 77)
    mask = torch.ones(2, 11, 11, dtype=torch.bool)
    kw = dict(q_split=split, kv_len_lo=0, kv_len_hi=N)
    _, _, want = run(ops, q, k, v, dout, mask, 64, **kw)
    q[:, :, :split] = float("nan")
    dout[:, :, :split] = float("inf")
    out, lse, got = run(ops, q, k, v, dout, mask, 64, **kw)
    assert (out[:, :, :split] == 0).all() and torch.isinf(lse[:, :, :split]).all()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and (got[0][:, :, :split] == 0).all()
