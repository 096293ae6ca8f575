"""What the training operators of a sparse attention layer are measured on.

Two operators and the step that joins the first one with the forward:

    bwd       gradients of block-sparse attention with respect to query, key and value, from the forward's output and
              row log-sum-exp (`ops.sparse_attn_bwd`); the probabilities are computed again, nothing of N x N is kept
    step      forward and backward of the same layer through autograd (`autograd.sparse_attention`)
    prologue  gradients of the attention prologue: per-head or whole-row normalisation of query and key, rotary embedding
              and the move to the head-major layout (`ops.qkv_prologue_bwd`)

With s = scale * q.k over the kept pairs, P = exp(s - lse), delta = sum(dout * out) per row:
    dv = P^T dout      ds = P * (dout v^T - delta)      dq = scale * ds k      dk = scale * ds^T q
The prologue rotates back, g = R^T dy, and with xhat the normalised row, r its factor, w the weight:
    rms    dx = r (g w - xhat mean(g w xhat))                  layer  dx = r (g w - mean(g w) - xhat mean(g w xhat))
    dw = sum g xhat    db = sum g
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ROWS = 1.6e9        # values of a score matrix that the plain form holds at a time


# ------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------

def _attention(op, batch, heads, head_dim, block, tokens, text, keep, *, dtype="bf16", text_first=False, pad=0,
               mask_heads=0):
    """keep: share of the blocks that a video row keeps (1.0: all); text: tokens whose rows and columns are all kept;
    pad: keys at the end that only the rows before them see rounded up to 64; mask_heads: 0 = one mask for each head."""
    return dict(op=op, batch=batch, heads=heads, head_dim=head_dim, block=block, tokens=tokens, text=text, keep=keep,
                dtype=dtype, text_first=text_first, pad=pad, mask_heads=mask_heads or heads)


def _prologue(batch, heads, head_dim, tokens, norm, rope, rope_lo, rope_hi, *, dtype="bf16", fused=True, before=0):
    """rope_lo, rope_hi: rotated tokens; fused: the projections are one tensor; before: rows of the head-major tensors
    that precede these tokens (a stream that is projected separately)."""
    return dict(op="prologue", batch=batch, heads=heads, head_dim=head_dim, tokens=tokens, norm=norm, rope=rope,
                rope_lo=rope_lo, rope_hi=rope_hi, dtype=dtype, fused=fused, before=before)


def listed():
    named = {
        # a low-rank adapter tried out on a few hundred tokens: launches and host time count
        "odd short rows": _attention("bwd", 2, 3, 128, 64, 333, 77, 0.6, dtype="fp16", mask_heads=1),
        # the smallest layer that the repository configures: two heads of 64, block 64
        "smallest layer": _attention("bwd", 1, 2, 64, 64, 4096, 0, 0.326),
        # a rank's share of heads on a short clip
        "short clip": _attention("bwd", 1, 4, 128, 128, 8448, 256, 0.315),
        # two samples of one layer under one mask, the last text tokens padding
        "padded pair": _attention("bwd", 2, 6, 64, 64, 6820, 226, 0.4, dtype="fp16", pad=101, mask_heads=1),
        # a dense warm-up step at the size of the reference's benchmark
        "dense step": _attention("step", 1, 24, 128, 128, 4096, 0, 1.0, dtype="fp16"),
        # fine-tuning on a medium clip, forward and backward
        "medium step": _attention("step", 1, 8, 128, 128, 16640, 256, 0.25),
        # a rank's heads at 44,880 video tokens and text in front, block 64, no region a whole number of blocks
        "text first": _attention("bwd", 1, 6, 64, 64, 45104, 224, 0.12, text_first=True),
        # a rank's three heads of the headline layer: 115,200 video and 256 text tokens
        "headline rank": _attention("bwd", 1, 3, 128, 128, 115456, 256, 0.152),
        # a short text stream projected on its own, normalised and appended behind the latent rows
        "text stream": _prologue(1, 30, 64, 226, "layer", "", 0, 0, dtype="fp16", fused=False, before=1350),
        # a sequence shard of a 40-head model that normalises over all heads
        "all heads": _prologue(1, 40, 128, 8640, "rms_all_heads", "pair", 0, 8640, fused=False),
        # latent and text tokens of one fused projection, per-head normalisation, text not rotated
        "per head, fused": _prologue(1, 16, 128, 57728, "rms_head", "elementwise", 0, 57600),
        # layer normalisation, two samples, text in front
        "layer norm": _prologue(2, 30, 64, 45104, "layer", "elementwise", 224, 45104, fused=False),
    }
    return [dict(c, name=n) for n, c in named.items()]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(("bf16", "fp16"))
    if rng.random() < 0.4:
        head_dim = rng.choice((64, 128))
        heads = rng.randint(2, 40 if head_dim == 128 else 48)
        norm = rng.choice(("rms_head", "rms_all_heads", "layer", ""))
        rope = rng.choice(("elementwise", "pair", "even_cos_odd_sin", "")) if norm else rng.choice(("elementwise", "pair"))
        batch = rng.randint(1, 3)
        tokens = _spread(rng, 1, min(60000, int(2.5e8 / (batch * heads * head_dim))))
        lo = rng.choice((0, rng.randint(0, tokens))) if rope else 0
        return _prologue(batch, heads, head_dim, tokens, norm, rope, lo, tokens if rope else 0, dtype=dtype,
                         fused=rng.random() < 0.5, before=rng.choice((0, 0, 128, 37)))
    op = rng.choice(("bwd", "bwd", "step"))
    head_dim, block = rng.choice((64, 128)), rng.choice((64, 128))
    batch, heads = rng.randint(1, 2), rng.randint(1, 8)
    # the largest score matrix is well below that of three heads of 115,456 tokens
    tokens = _spread(rng, 1, int(math.sqrt(6e9 / (batch * heads))))
    text = rng.choice((0, min(tokens - 1, rng.randint(1, 300))))
    keep = rng.choice((1.0, rng.uniform(0.1, 0.6)))
    pad = rng.choice((0, rng.randint(0, text))) if text else 0
    return _attention(op, batch, heads, head_dim, block, tokens, text, keep, dtype=dtype, pad=pad,
                      text_first=not pad and rng.random() < 0.3, mask_heads=rng.choice((heads, 1)))


# ------------------------------------------------------------------------------------------------
# sizes that follow from a case
# ------------------------------------------------------------------------------------------------

def _blocks(case):
    """(blocks, first and last+1 video block, kept blocks of a video row)"""
    N, bs = case["tokens"], case["block"]
    nb = (N + bs - 1) // bs
    text_blocks = (case["text"] + bs - 1) // bs
    lo, hi = (text_blocks, nb) if case["text_first"] else (0, nb - text_blocks)
    return nb, lo, hi, max(1, min(hi - lo, round(case["keep"] * nb))) if hi > lo else 0


def _limits(case):
    """(rows before this one see the first limit, the others the second)"""
    N, valid = case["tokens"], case["tokens"] - case["pad"]
    return N - case["text"], min(N, (valid + 63) // 64 * 64), valid


def work(case):
    B, H, D = case["batch"], case["heads"], case["head_dim"]
    size = B * H * D * case["tokens"]
    if case["op"] == "prologue":
        # dy of three tensors in, dx of three out, x of the normalised two in
        tables = 2 * 4 * (case["rope_hi"] - case["rope_lo"]) * (D // 2 if case["rope"] == "pair" else D)
        return {"bytes": 2 * size * (8 if case["norm"] else 6) + tables * bool(case["rope"]), "flops": 20 * size}
    nb, lo, hi, count = _blocks(case)
    share = (count * (hi - lo) + (nb * nb - (hi - lo) ** 2)) / nb ** 2
    pairs = share * case["tokens"] * (case["tokens"] - case["pad"])
    if case["op"] == "bwd":     # q, k, v, out, dout, lse in, dq, dk, dv out; five products
        return {"bytes": 16 * size + 4 * size // D, "flops": 10 * B * H * D * pairs}
    return {"bytes": 16 * size, "flops": 14 * B * H * D * pairs}     # q, k, v, dout in, out, dq, dk, dv out


# ------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------

def _mask(case, g, dev):
    """Local window, the same place in other frames and some columns that every row keeps; a fixed count for each row."""
    nb, lo, hi, count = _blocks(case)
    n, heads = hi - lo, case["mask_heads"]
    mask = torch.ones(heads, nb, nb, dtype=torch.bool, device=dev)
    if n > 0 and count < n:
        far = (torch.arange(n, device=dev)[:, None] - torch.arange(n, device=dev)).abs().float()
        frame = max(2, n // 30)
        near = torch.exp(-far / 4) + 0.7 * torch.exp(-torch.minimum(far % frame, frame - far % frame) / 2)
        score = near + 0.8 * (torch.rand(heads, 1, n, generator=g, device=dev) < 0.04) + \
            0.5 * torch.rand(heads, n, n, generator=g, device=dev)
        video = torch.zeros(heads, n, n, dtype=torch.bool, device=dev)
        mask[:, lo:hi, lo:hi] = video.scatter_(2, score.topk(count, 2).indices, True)
    return mask


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DTYPES[case["dtype"]]
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 11)
    B, H, D, N = case["batch"], case["heads"], case["head_dim"], case["tokens"]

    def normal(*shape, gain=1.0, mean=0.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=dev) * gain + mean).to(dtype)

    # gradients of a mean loss are small; with float16 a training run scales its loss
    grad = 0.02 if case["dtype"] == "bf16" else 1.0
    s = {"case": case}
    if case["op"] == "prologue":
        W = H * D
        names = ("q", "k", "v")
        if case["fused"]:
            s["x"] = tuple(normal(B, N, 3 * W).split(W, 2))
        else:
            s["x"] = tuple(normal(B, N, W, gain=1.0 + 0.3 * i) for i, _ in enumerate(names))
        s["dy"] = tuple(normal(B, H, case["before"] + N, D, gain=grad) for _ in names)
        width = W if case["norm"] == "rms_all_heads" else D
        s["weight"] = tuple(normal(width, gain=0.1, mean=1.0) if case["norm"] else None for _ in range(2))
        s["bias"] = tuple(normal(width, gain=0.1) if case["norm"] == "layer" else None for _ in range(2))
        s["tables"] = None
        if case["rope"]:
            pos = torch.arange(case["rope_hi"] - case["rope_lo"], device=dev, dtype=torch.float64)
            inv = 256.0 ** (-torch.arange(D // 2, device=dev, dtype=torch.float64) / (D // 2))
            ang = (pos[:, None] + int(seed) % 97) * inv
            ang = ang if case["rope"] == "pair" else ang.repeat_interleave(2, 1)
            s["tables"] = (ang.cos().float().contiguous(), ang.sin().float().contiguous())
        return s
    # neighbours attend to each other: a smooth code of the position in query and key
    code = torch.arange(N, device=dev)[:, None] / N * (2.0 ** torch.arange(8, device=dev)) * math.pi
    code = torch.cat((code.sin(), code.cos()), 1)
    mix = torch.randn(B, H, 16, D, generator=g, device=dev) / 4
    s["q"], s["k"] = (normal(B, H, N, D, gain=0.7, mean=torch.matmul(code, mix)) for _ in range(2))
    s["v"], s["dout"] = normal(B, H, N, D), normal(B, H, N, D, gain=grad)
    s["mask"] = _mask(case, g, dev)
    s["scale"] = D ** -0.5
    if case["op"] == "bwd":
        out, s["lse"] = _attend(s)
        s["out"] = out.to(dt)
    else:
        for name in ("q", "k", "v"):
            s[name].requires_grad_(True)
    if own:
        # a training run keeps the work lists of a mask until the mask is predicted anew
        ops = _package("ops")
        s["lists"] = ops.tile_lists(s["mask"], case["block"], N)
        s["key_lists"] = ops.key_lists(s["mask"], case["block"], N)
    return s


# ------------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------------

def _pieces(s):
    """Ranges of query rows whose score matrices fit, each with the pairs that are kept: (rows, (1 or B, H, rows, N) bool)."""
    case, mask = s["case"], s["mask"]
    B, H, N = case["batch"], case["heads"], case["tokens"]
    step = max(1, min(N, int(ROWS / (B * H * N))))
    split, first, second = _limits(case)
    key = torch.arange(N, device=mask.device)
    for lo in range(0, N, step):
        row = torch.arange(lo, min(N, lo + step), device=mask.device)
        keep = mask[:, row // case["block"]][:, :, key // case["block"]]
        yield slice(lo, lo + row.numel()), keep & (key < torch.where(row < split, first, second)[:, None])


def _attend(s):
    """(out, lse) in 32 bits; a row that keeps nothing gives zeros and minus infinity."""
    q, k, v = (s[n].detach().float() for n in ("q", "k", "v"))
    out, lse = torch.empty_like(q), torch.empty_like(q[..., 0])
    for rows, keep in _pieces(s):
        p = torch.matmul(q[:, :, rows], k.mT).mul_(s["scale"]).masked_fill_(~keep, -math.inf)
        top = p.amax(-1, keepdim=True).clamp_(min=-1e30)
        p.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        out[:, :, rows] = torch.matmul(p, v) / total.clamp(min=1e-30)
        lse[:, :, rows] = torch.where(total > 0, total.log() + top, -math.inf)[..., 0]
    return out, lse


def _attend_bwd(s, out, lse):
    q, k, v, dout = (s[n].detach().float() for n in ("q", "k", "v", "dout"))
    delta = (dout * out.float()).sum(-1, keepdim=True)
    dq, dk, dv = torch.empty_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for rows, keep in _pieces(s):
        p = torch.matmul(q[:, :, rows], k.mT).mul_(s["scale"]).sub_(lse[:, :, rows, None]).exp_().masked_fill_(~keep, 0)
        dv += torch.matmul(p.mT, dout[:, :, rows])
        ds = torch.matmul(dout[:, :, rows], v.mT).sub_(delta[:, :, rows]).mul_(p)
        dq[:, :, rows] = torch.matmul(ds, k) * s["scale"]
        dk += torch.matmul(ds.mT, q[:, :, rows])
    dt = s["q"].dtype
    return dq.to(dt), (dk * s["scale"]).to(dt), dv.to(dt)


def _prologue_bwd(s, g, x, weight):
    """(dx, dweight, dbias) of one tensor from g (B, H, N, D), the gradient of its rotated rows."""
    case = s["case"]
    B, H, D, N = case["batch"], case["heads"], case["head_dim"], case["tokens"]
    g = g[:, :, case["before"]:].float()
    if s["tables"] is not None and x is not None:
        lo, hi = case["rope_lo"], case["rope_hi"]
        cos, sin = s["tables"]
        if case["rope"] == "pair":
            cos, sin = cos.repeat_interleave(2, 1), sin.repeat_interleave(2, 1)
        if case["rope"] == "even_cos_odd_sin":
            cos, sin = cos[:, 0::2].repeat_interleave(2, 1), sin[:, 1::2].repeat_interleave(2, 1)
        a, b = g[:, :, lo:hi, 0::2], g[:, :, lo:hi, 1::2]
        back = torch.stack((a * cos[:, 0::2] + b * sin[:, 1::2], b * cos[:, 1::2] - a * sin[:, 0::2]), -1).flatten(-2)
        g = torch.cat((g[:, :, :lo], back, g[:, :, hi:]), 2)
    g = g.transpose(1, 2)                                   # (B, N, H, D)
    dt = DTYPES[case["dtype"]]
    if x is None or not case["norm"]:
        return g.reshape(B, N, H * D).to(dt), None, None
    x = x.float().reshape(B, N, H, D)
    dims = (2, 3) if case["norm"] == "rms_all_heads" else (3,)
    if case["norm"] == "layer":
        x = x - x.mean(dims, keepdim=True)
    r = torch.rsqrt(x.square().mean(dims, keepdim=True) + 1e-6)
    xhat = x * r
    gw = g * (weight.float().reshape(H, D) if weight.numel() != D else weight.float())
    dx = gw - xhat * (gw * xhat).mean(dims, keepdim=True)
    if case["norm"] == "layer":
        dx = dx - gw.mean(dims, keepdim=True)
    over = (0, 1) if case["norm"] == "rms_all_heads" else (0, 1, 2)
    dw = (g * xhat).sum(over).flatten().to(dt)
    db = g.sum(over).to(dt) if case["norm"] == "layer" else None
    return (dx * r).reshape(B, N, H * D).to(dt), dw, db


def _package(name):
    """The named module of the framework's package."""
    root = os.path.join(os.getcwd(), "mod-dit_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import importlib
    return importlib.import_module("moddit_b200." + name)


def run(s):
    case = s["case"]
    if case["op"] == "prologue":
        if own:
            cos, sin = s["tables"] or (None, None)
            dx, grads = _package("ops").qkv_prologue_bwd(
                *s["dy"], s["x"][0], s["x"][1], num_heads=case["heads"], norm=case["norm"] or None,
                q_weight=s["weight"][0], q_bias=s["bias"][0], k_weight=s["weight"][1], k_bias=s["bias"][1], eps=1e-6,
                rope_cos=cos, rope_sin=sin, rope_form=case["rope"] or "pair", rope_range=(case["rope_lo"], case["rope_hi"]),
                src_row0=case["before"])
            return {"dx": dx, "dweight": (grads["q_weight"], grads["k_weight"]), "dbias": (grads["q_bias"], grads["k_bias"])}
        each = [_prologue_bwd(s, s["dy"][i], s["x"][i] if i < 2 else None, s["weight"][i] if i < 2 else None)
                for i in range(3)]
        return {"dx": tuple(e[0] for e in each), "dweight": tuple(e[1] for e in each[:2]),
                "dbias": tuple(e[2] for e in each[:2])}
    split, first, second = _limits(case)
    if case["op"] == "bwd":
        if own:
            return _package("ops").sparse_attn_bwd(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["lists"],
                                                   s["key_lists"], softmax_scale=s["scale"], q_split=split,
                                                   kv_len_lo=first, kv_len_hi=second, check_status="deferred")
        return _attend_bwd(s, s["out"], s["lse"])
    if own:
        out = _package("autograd").sparse_attention(s["q"], s["k"], s["v"], s["lists"], s["key_lists"],
                                                    softmax_scale=s["scale"], q_split=split, kv_len_lo=first,
                                                    kv_len_hi=second)
        return (out.detach(),) + torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"])
    out, lse = _attend(s)
    return (out.to(s["q"].dtype),) + _attend_bwd(s, out, lse)


# ------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_prologue(s) if case["op"] == "prologue" else _exact_attention(s)


def _exact_prologue(s):
    """Differentiates the prologue itself."""
    case = s["case"]
    B, H, D, N = case["batch"], case["heads"], case["head_dim"], case["tokens"]
    dx, dweight, dbias = [], [], []
    for i in range(3):
        x = s["x"][i].double().requires_grad_(True)
        w = s["weight"][i].double().requires_grad_(True) if i < 2 and case["norm"] else None
        b = s["bias"][i].double().requires_grad_(True) if i < 2 and case["norm"] == "layer" else None
        y = x
        if w is not None and case["norm"] == "rms_all_heads":
            y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w
        y = y.view(B, N, H, D)
        if w is not None and case["norm"] == "rms_head":
            y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w
        if w is not None and case["norm"] == "layer":
            y = (y - y.mean(-1, keepdim=True)) / (y.var(-1, correction=0, keepdim=True) + 1e-6).sqrt() * w + b
        y = y.permute(0, 2, 1, 3)
        if i < 2 and s["tables"] is not None:
            c, n = (t.double() for t in s["tables"])
            lo, hi = case["rope_lo"], case["rope_hi"]
            at = {"pair": (slice(None),) * 4, "elementwise": (slice(0, None, 2), slice(0, None, 2), slice(1, None, 2), slice(1, None, 2)),
                  "even_cos_odd_sin": (slice(0, None, 2), slice(1, None, 2), slice(1, None, 2), slice(0, None, 2))}[case["rope"]]
            even, odd = y[:, :, lo:hi].unflatten(-1, (-1, 2)).unbind(-1)
            turned = torch.stack((even * c[:, at[0]] - odd * n[:, at[1]], even * n[:, at[2]] + odd * c[:, at[3]]), -1)
            y = torch.cat((y[:, :, :lo], turned.flatten(-2), y[:, :, hi:]), 2)
        leaves = [t for t in (x, w, b) if t is not None]
        got = list(torch.autograd.grad(y, leaves, s["dy"][i][:, :, case["before"]:].double()))
        dx.append(got.pop(0))
        if i < 2:
            dweight.append(got.pop(0) if w is not None else None)
            dbias.append(got.pop(0) if b is not None else None)
    return {"dx": tuple(dx), "dweight": tuple(dweight), "dbias": tuple(dbias)}


def _exact_attention(s):
    """One head at a time, a few thousand query rows of it at once."""
    case = s["case"]
    B, H, N, bs = case["batch"], case["heads"], case["tokens"], case["block"]
    step = max(bs, int(4e8 / N) // bs * bs)
    split, first, second = _limits(case)
    names = ("q", "k", "v", "dout")
    outs, dqs, dks, dvs = [], [], [], []
    for b in range(B):
        for h in range(H):
            q, k, v, do = (s[n].detach()[b, h].double() for n in names)
            o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
            column = torch.arange(N, device=q.device)
            blocks = s["mask"][h % case["mask_heads"]]
            for lo in range(0, N, step):
                r = slice(lo, min(N, lo + step))
                row = column[r]
                gone = ~blocks[lo // bs:(r.stop - 1) // bs + 1].repeat_interleave(bs, 0).repeat_interleave(bs, 1)[:row.numel(), :N]
                gone = gone | ((column >= first) & (row < split)[:, None]) | ((column >= second) & (row >= split)[:, None])
                e = torch.einsum("rd,cd->rc", q[r], k) * s["scale"]
                if case["op"] == "bwd":
                    p = torch.exp(e - s["lse"][b, h, r, None].double())
                    p[gone] = 0
                    o[r] = s["out"][b, h, r].double()
                else:
                    p = torch.softmax(e.masked_fill(gone, -math.inf), 1).nan_to_num(0.0)
                    o[r] = torch.einsum("rc,cd->rd", p, v)
                t = torch.einsum("rd,cd->rc", do[r], v)
                t = p * (t - torch.einsum("rd,rd->r", do[r], o[r])[:, None])
                dv += torch.einsum("rc,rd->cd", p, do[r])
                dq[r] = torch.einsum("rc,cd->rd", t, k) * s["scale"]
                dk += torch.einsum("rc,rd->cd", t, q[r]) * s["scale"]
            for to, one in zip((outs, dqs, dks, dvs), (o, dq, dk, dv)):
                to.append(one)
    whole = [torch.stack(x).view(B, H, N, -1) for x in (outs, dqs, dks, dvs)]
    return tuple(whole[1:] if case["op"] == "bwd" else whole)
