"""What the backward entry points refuse, without a GPU."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def buf():
    raw = ctypes.create_string_buffer(96)
    return raw, ctypes.c_void_p((ctypes.addressof(raw) + 15) // 16 * 16)


def attn(lib, p, *, dtype=0, BH=2, N=256, D=64, Hm=2, scale=0.1, lo=256, hi=256, ws=1 << 30, null=None, off=None):
    args = [p] * 7
    if null is not None:
        args[null] = None
    if off is not None:
        args[off] = ctypes.c_void_p(p.value + 8)
    return lib.moddit_sparse_attn_bwd(*args, dtype, BH, N, D, p, p, p, p, p, p, Hm, scale, 0, lo, hi, p, p, p, p, ws, p, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(null=0), -1, b"null"), (dict(null=3), -1, b"null"), (dict(null=5), -1, b"null"), (dict(BH=0), -1, b"out of range"),
    (dict(BH=65536), -1, b"out of range"), (dict(N=0), -1, b"out of range"), (dict(BH=3), -1, b"multiple"),
    (dict(scale=0.0), -1, b"softmax_scale"), (dict(lo=257), -1, b"kv_len"), (dict(hi=-1), -1, b"kv_len"), (dict(D=96), -2, b"head_dim"),
    (dict(dtype=2), -1, b"dtype"), (dict(off=0), -3, b"aligned"), (dict(off=4), -3, b"aligned"), (dict(off=5), -3, b"aligned"),
    (dict(ws=0), -4, b"workspace"), (dict(N=1 << 20, lo=5, hi=5), -2, b"exceeds")])
def test_attention(buf, kw, rc, text):
    from moddit_b200 import _lib
    assert attn(_lib.lib, buf[1], **kw) == rc
    assert text in _lib.lib.moddit_last_error_string()


def test_attention_workspace():
    from moddit_b200 import _lib
    f = _lib.lib.moddit_sparse_attn_bwd_workspace_bytes
    assert f(3, 300) == 2 * 3 * 384 * 4 and f(0, 300) == 0 and f(3, 0) == 0
    assert f(65535, 1 << 20) == 2 * 65535 * (1 << 20) * 4            # past 32 bits


def prologue(lib, p, *, grads=(1, 1, 1), dtype=0, B=1, S=64, H=2, D=64, stride=128, norm=1, cos=1, sin=1, form=2, lo=0, hi=64,
             N=64, row0=0, out_stride=128, x=1, params=(1, 0, 1, 0), ws=1 << 30):
    on = lambda v: p if v else None          # noqa: E731
    return lib.moddit_qkv_prologue_bwd(*[on(g) for g in grads], on(x), on(x), dtype, B, S, H, D, stride, norm, p, p, 1e-6,
                                       on(cos), on(sin), form, lo, hi, N, row0, p, p, p, out_stride, *[on(v) for v in params], p,
                                       ws, None)


@pytest.mark.parametrize("kw,rc,text", [
    (dict(grads=(0, 0, 0), params=(0, 0, 0, 0)), -1, b"no gradient"), (dict(dtype=5), -1, b"dtype"), (dict(D=32), -1, b"head_dim"),
    (dict(S=0), -1, b"positive"), (dict(norm=4), -1, b"norm_kind"), (dict(row0=1), -1, b"rows"), (dict(row0=-1), -1, b"rows"),
    (dict(out_stride=120), -1, b"out_stride"), (dict(out_stride=132), -1, b"out_stride"), (dict(stride=64), -1, b"token_stride"),
    (dict(x=0), -1, b"normalisation"), (dict(sin=0), -1, b"go together"), (dict(hi=65), -1, b"rotary range"),
    (dict(form=3), -1, b"rope_form"), (dict(params=(1, 1, 0, 0)), -1, b"no such parameter"),
    (dict(norm=0), -1, b"no such parameter"), (dict(grads=(0, 1, 1)), -1, b"without its gradient"),
    (dict(ws=16), -4, b"workspace"), (dict(norm=2, H=1024, stride=65536, out_stride=65536), -2, b"at most")])
def test_prologue(buf, kw, rc, text):
    from moddit_b200 import _lib
    assert prologue(_lib.lib, buf[1], **kw) == rc
    assert text in _lib.lib.moddit_last_error_string()


def test_key_lists(buf):
    from moddit_b200 import _lib
    f, p = _lib.lib.moddit_key_lists, buf[1]
    assert f(None, 1, 2, 2, 64, 128, 2, p, p, None, None) == -1
    assert f(p, 0, 2, 2, 64, 128, 2, p, p, None, None) == -1
    assert f(p, 1, 2, 2, 32, 128, 2, p, p, None, None) == -2
    assert f(p, 1, 2, 2, 64, 1 << 23, 2, p, p, None, None) == -2


def test_wrappers_refuse_cpu_tensors():
    from moddit_b200 import autograd, ops
    x = torch.zeros(1, 1, 64, 64, dtype=torch.bfloat16)
    mask = torch.ones(1, 1, 1, dtype=torch.bool)
    with pytest.raises(ValueError, match="CUDA"):
        ops.key_lists(mask, 64, 64)
    lists = ops.KeyLists(torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1, 1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA"):
        ops.sparse_attn_bwd(x, x, x, x, x, torch.zeros(1, 1, 64), lists, lists)
    with pytest.raises(ValueError, match="CUDA"):
        ops.qkv_prologue_bwd(x, x, x, num_heads=1)
    with pytest.raises(ValueError, match="CUDA"):
        autograd.sparse_attention(x.requires_grad_(True), x, x, lists, lists)
    with pytest.raises(ValueError, match="no gradient"):
        ops.qkv_prologue_bwd(None, None, None, num_heads=1)
    y = torch.zeros(1, 64, 192, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="either"):
        autograd.qkv_prologue(y, y, num_heads=1)
    with pytest.raises(ValueError, match="either"):
        autograd.qkv_prologue(y, y, y, fused=y, num_heads=1)
    with pytest.raises(ValueError, match="contiguous"):
        autograd.qkv_prologue(fused=y[:, :, :128], num_heads=1)
