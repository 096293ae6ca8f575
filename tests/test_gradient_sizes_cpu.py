"""Sizes that the gradients do not cover are refused where the graph is built, not in the backward pass behind a step's work."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def mods():
    from moddit_b200 import _lib, autograd, ops
    return _lib, autograd, ops


def lists_of(kind):
    return kind(torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1, 1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32))


def test_the_limits_are_the_librarys(mods):
    _lib, _, _ = mods
    text = open(os.path.join(ROOT, "include", "moddit.h")).read()
    for name in ("ATTN_BWD_MAX_ROWS", "TOKEN_NORM_BWD_MAX_WIDTH"):
        assert int(re.search(rf"#define MODDIT_{name} (\d+)", text).group(1)) == getattr(_lib, name)
    raw = ctypes.create_string_buffer(96)
    p = ctypes.c_void_p((ctypes.addressof(raw) + 15) // 16 * 16)
    for N, rc in ((_lib.ATTN_BWD_MAX_ROWS, -4), (_lib.ATTN_BWD_MAX_ROWS + 1, -2)):        # the next check is the workspace
        assert _lib.lib.moddit_sparse_attn_bwd(*[p] * 7, 0, 1, N, 64, *[p] * 6, 1, 0.1, 0, N, N, *[p] * 4, 0, p, None) == rc
    for H, rc in ((_lib.TOKEN_NORM_BWD_MAX_WIDTH // 64, -4), (_lib.TOKEN_NORM_BWD_MAX_WIDTH // 64 + 1, -2)):
        assert _lib.lib.moddit_qkv_prologue_bwd(*[p] * 5, 0, 1, 1, H, 64, H * 64, 2, p, p, 1e-6, None, None, 2, 0, 0, 1, 0, p, p, p,
                                                H * 64, p, None, p, None, p, 0, None) == rc


def test_attention(mods):
    _lib, autograd, ops = mods
    x = torch.empty(1, 1, _lib.ATTN_BWD_MAX_ROWS + 1, 64, dtype=torch.bfloat16)
    args = (lists_of(ops.TileLists), lists_of(ops.KeyLists))
    with pytest.raises(_lib.ModditError, match="gradients"):
        autograd.sparse_attention(x, x, x.detach().requires_grad_(True), *args)
    with pytest.raises(ValueError, match="CUDA"):           # the forward alone has no such limit: the next check refuses
        autograd.sparse_attention(x, x, x, *args)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        autograd.sparse_attention(x, x, x.detach().requires_grad_(True), *args)


def test_prologue(mods):
    _lib, autograd, _ = mods
    H = _lib.TOKEN_NORM_BWD_MAX_WIDTH // 64 + 1
    x = torch.zeros(1, 2, 64 * H, dtype=torch.bfloat16)
    w = torch.ones(64 * H, dtype=torch.bfloat16)
    kw = dict(num_heads=H, norm="rms_all_heads")
    for args in (dict(q_in=x.clone().requires_grad_(True), k_in=x, v_in=x), dict(q_in=x, k_in=x, v_in=x.clone().requires_grad_(True)),
                 dict(q_in=x, k_in=x, v_in=x, k_weight=w.clone().requires_grad_(True)),
                 dict(fused=torch.zeros(1, 2, 3 * 64 * H, dtype=torch.bfloat16, requires_grad=True))):
        with pytest.raises(_lib.ModditError, match="gradients"):
            autograd.qkv_prologue(**args, **kw)
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
            autograd.qkv_prologue(**args, **kw)
    with pytest.raises(ValueError, match="CUDA"):
        autograd.qkv_prologue(x.requires_grad_(True), x, x, num_heads=H, norm="rms_head")
