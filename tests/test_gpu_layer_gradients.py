"""Gradients through the layer's own entry points: every kind of step gives, where its inputs ask for gradients, the output and the
state of the same step without, bit for bit, and the gradients of `autograd.sparse_attention` under the mask that the step ran."""
import logging
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu
LOG = logging.getLogger("test")
H, GRID, D, BS, TEXT = 2, (4, 16, 16), 64, 128, 128
VIDEO = GRID[0] * GRID[1] * GRID[2]
N = VIDEO + TEXT
VALID = N - 37


@pytest.fixture(scope="module")
def mods():
    import MoD.mod.attn_mask as am
    from moddit_b200 import autograd, ops
    return am, autograd, ops


def inputs(step):
    from moddit_b200 import synth
    q, k, v = synth.make_qkv(heads=H, grid=GRID, head_dim=D, text_tokens=TEXT, seed=20 + step, device=torch.device("cuda"))
    g = torch.Generator(device="cuda").manual_seed(step)
    return q, k, v, torch.randn(q.shape, generator=g, device="cuda").to(q.dtype)


def new_state(**extra):
    from MoD.mod.state import create_adaptive_mask_state
    state = create_adaptive_mask_state("hunyuan", H, VIDEO, TEXT, GRID[1] * GRID[2], GRID[0], warmup_steps=3, top_k=4, predict_T=3,
                                       threshold=1e-3, block_size=BS, sparse_type=extra.pop("sparse_type", "mod-dit"))
    state.update(extra)
    return state


def padding():
    return (torch.arange(N) < VALID).unsqueeze(0).expand(N, N).contiguous().cuda()


def wanted(mods, q, k, v, dout, mask, **limits):
    """Gradients under a block mask; None stands for every block."""
    am, autograd, ops = mods
    if mask is None:
        mask = torch.ones(1, (N + BS - 1) // BS, (N + BS - 1) // BS, dtype=torch.bool, device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = autograd.sparse_attention(*leaves, ops.tile_lists(mask, BS, N), ops.key_lists(mask, BS, N), **limits)
    return out.detach(), torch.autograd.grad(out, leaves, dout)


def holds_no_graph(value):
    if torch.is_tensor(value):
        return not value.requires_grad
    if isinstance(value, dict):
        return all(holds_no_graph(v) for v in value.values())
    if isinstance(value, (list, tuple)):
        return all(holds_no_graph(v) for v in value)
    return True


def both(mods, state, twin, step, **kw):
    """One step with and one without gradients, each on a state of its own: (inputs, output, gradients)."""
    am, _, _ = mods
    q, k, v, dout = inputs(step)
    plain, _ = am.SparseAttentionWithMap(q, k, v, twin, LOG, current_step=step, **kw)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        out, _ = am.SparseAttentionWithMap(*leaves, state, LOG, current_step=step, **kw)
    assert plain.grad_fn is None and out.requires_grad and torch.equal(out, plain)
    with torch.no_grad():
        assert holds_no_graph(state)
    got = torch.autograd.grad(out, leaves, dout)
    return (q, k, v, dout), out.detach(), got


def same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


SPARSE = dict(q_split=VIDEO, kv_len_lo=(VALID + 63) // 64 * 64, kv_len_hi=VALID)


@pytest.mark.parametrize("threshold", [0.0, 0.3])
def test_spargeattn(mods, threshold):
    state, twin = (new_state(sparse_type="spargeattn", spargeattn_sim_threshold=threshold) for _ in range(2))
    x, out, got = both(mods, state, twin, 7)
    assert torch.equal(state["mask"], twin["mask"])
    want_out, want = wanted(mods, *x, state["mask"])
    assert torch.equal(out, want_out) and same(got, want)


@pytest.mark.parametrize("selector", ["topk_lines", "cumulative_mass"])
def test_steps_of_the_exact_map(mods, selector):
    """Dense, collecting, sparse and refreshing steps."""
    state, twin = (new_state(selector=selector) for _ in range(2))
    for step in range(8):
        mask = state["mask"]
        collects, refreshes = step in (1, 2), step in (5,)
        x, out, got = both(mods, state, twin, step, pre_defined_mask=padding())
        if step >= 2:
            assert torch.equal(state["mask"], twin["mask"])
        if step < 1:
            want_out, want = wanted(mods, *x, None, kv_len_lo=VALID, kv_len_hi=VALID)
        elif collects or refreshes:
            want_out, want = wanted(mods, *x, None)
        else:
            want_out, want = wanted(mods, *x, mask, **SPARSE)
        assert torch.equal(out, want_out) and same(got, want), step


@pytest.mark.parametrize("groups", [1, 2])
def test_steps_of_the_pooled_map(mods, groups):
    """Dense, collecting and sparse steps, with query, key and value complete or arriving in two groups of heads."""
    extra = dict(score_producer="pooled")
    kw = dict(pre_defined_mask=padding())
    if groups > 1:
        extra["_head_groups"] = groups
        kw["head_group_ready"] = [torch.cuda.Event() for _ in range(groups)]
        for e in kw["head_group_ready"]:
            e.record()
    state, twin = new_state(**extra), new_state(**extra)
    for step in range(6):
        x, out, got = both(mods, state, twin, step, **kw)
        if step < 2:
            want_out, want = wanted(mods, *x, None, kv_len_lo=VALID, kv_len_hi=VALID)
        else:
            assert torch.equal(state["mask"], twin["mask"])
            want_out, want = wanted(mods, *x, state["mask"], **SPARSE)
        assert torch.equal(out, want_out) and same(got, want), step


def test_head_groups_arrive_before_the_gradient_path_reads(mods):
    """The launch that is differentiable waits for every group's event, whatever the event's stream still does."""
    am, _, ops = mods
    q, k, v, dout = inputs(30)
    mask = torch.rand(H, 9, 9, generator=torch.Generator().manual_seed(1)).lt(0.5).cuda()
    want_out, want = wanted(mods, q, k, v, dout, mask)
    late = [torch.zeros_like(t) for t in (q, k, v)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    ready = [torch.cuda.Event() for _ in range(H)]
    with torch.cuda.stream(side):
        torch.cuda._sleep(20000000)                 # some ten milliseconds
        for h, e in enumerate(ready):
            for dst, src in zip(late, (q, k, v)):
                dst[:, h].copy_(src[:, h])
            e.record()
    leaves = [t.requires_grad_(True) for t in late]
    lists = ops.tile_lists(mask, BS, N, heads_per_group=1)
    out = am.AttentionSparseEngine(*leaves, mask, block_size=BS, _lists=lists, _group_ready=ready)
    got = torch.autograd.grad(out, leaves, dout)
    torch.cuda.synchronize()
    assert torch.equal(out, want_out) and same(got, want)


def test_radial(mods):
    state, twin = (new_state(sparse_type="radial") for _ in range(2))
    for step in (0, 3):
        x, out, got = both(mods, state, twin, step)
        want_out, want = wanted(mods, *x, None if step < 3 else state["mask"])
        assert torch.equal(out, want_out) and same(got, want)


def test_output_that_goes_to_peers_says_that_it_has_no_gradient(mods):
    """Rows stored into other tensors are not part of the graph: the call says so once its inputs ask for gradients."""
    am, _, _ = mods
    q, k, v, _ = inputs(40)
    mask = torch.rand(H, 9, 9, generator=torch.Generator().manual_seed(2)).lt(0.5).cuda()
    want = am.AttentionSparseEngine(q, k, v, mask, block_size=BS)
    for ask in (False, True):
        to = torch.zeros_like(q)
        leaves = [t.clone().requires_grad_(ask) for t in (q, k, v)]
        with warnings.catch_warnings(record=True) as seen:
            warnings.simplefilter("always")
            am.AttentionSparseEngine(*leaves, mask, block_size=BS, _scatter=([to.data_ptr()], 0))
            with torch.no_grad():
                am.AttentionSparseEngine(*leaves, mask, block_size=BS, _scatter=([to.data_ptr()], 0))
        torch.cuda.synchronize()
        assert torch.equal(to, want)
        assert [str(w.message).count("no gradient") for w in seen] == [1] * ask


def test_two_branches(mods):
    """Both guidance branches of a collecting and a sparse step in one call."""
    am, _, _ = mods
    def states():
        return [new_state() for _ in range(2)]
    mine, twins = states(), states()
    for step in (1, 2, 3):
        pairs = [inputs(50 + 2 * step + i) for i in range(2)]
        q, k, v, dout = (torch.cat([p[i] for p in pairs]) for i in range(4))
        plain, _ = am.SparseAttentionWithMapCFG(q, k, v, twins, LOG, current_step=step)
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        mask = None if step < 3 else [s["mask"] for s in mine]
        out, _ = am.SparseAttentionWithMapCFG(*leaves, mine, LOG, current_step=step)
        assert torch.equal(out, plain)
        got = torch.autograd.grad(out, leaves, dout)
        for i, p in enumerate(pairs):
            _, want = wanted(mods, *p, None if mask is None else mask[i])
            assert same([t[i:i + 1] for t in got], want)


@pytest.mark.parametrize("ask", [False, True])
def test_a_single_group_of_heads_is_waited_for(mods, ask):
    """One event for all heads: rows that another stream still writes are read behind it, with and without gradients."""
    am, _, ops = mods
    q, k, v, dout = inputs(31)
    mask = torch.rand(H, 9, 9, generator=torch.Generator().manual_seed(3)).lt(0.5).cuda()
    want_out, want = wanted(mods, q, k, v, dout, mask)
    late = [torch.zeros_like(t) for t in (q, k, v)]
    lists = ops.tile_lists(mask, BS, N)
    torch.cuda.synchronize()
    side, ready = torch.cuda.Stream(), torch.cuda.Event()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20000000)
        for dst, src in zip(late, (q, k, v)):
            dst.copy_(src)
        ready.record()
    leaves = [t.requires_grad_(ask) for t in late]
    out = am.AttentionSparseEngine(*leaves, mask, block_size=BS, _lists=lists, _group_ready=[ready])
    got = torch.autograd.grad(out, leaves, dout) if ask else want
    torch.cuda.synchronize()
    assert torch.equal(out, want_out) and same(got, want)


def test_without_a_graph_nothing_is_kept_for_one(mods, monkeypatch):
    """Under no_grad the differentiable form is the forward alone, whatever its inputs would ask for."""
    _, autograd, ops = mods
    q, k, v, _ = inputs(60)
    mask = torch.ones(1, 9, 9, dtype=torch.bool, device="cuda")
    lists, klists = ops.tile_lists(mask, BS, N), ops.key_lists(mask, BS, N)
    forward, kept = ops.sparse_attn_fwd, []
    monkeypatch.setattr(ops, "sparse_attn_fwd", lambda *a, **kw: kept.append(kw["return_residual"]) or forward(*a, **kw))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    with torch.no_grad():
        out, lse = autograd.sparse_attention(*leaves, lists, klists, return_lse=True)
    graph, graph_lse = autograd.sparse_attention(*leaves, lists, klists, return_lse=True)
    assert kept == [False, True] and not out.requires_grad and graph.requires_grad and not graph_lse.requires_grad
    assert torch.equal(out, graph) and torch.equal(lse, graph_lse)
    assert torch.equal(autograd.sparse_attention(q, k, v, lists, klists), out)


@pytest.mark.parametrize("way", ["value", "groups", "step", "step by groups"])
@pytest.mark.parametrize("ask", [False, True])
def test_copies_of_other_layouts_wait_for_the_rows(mods, way, ask):
    """Query, key and value of (B, N, H, D) order are copied: behind the events that say that their rows are there."""
    am, _, ops = mods
    q, k, v, dout = inputs(32)
    mask = torch.rand(H, 9, 9, generator=torch.Generator().manual_seed(4)).lt(0.5).cuda()
    pools = tuple(ops.pool_blocks(t, BS) for t in (q, k))
    by_groups = "groups" in way
    state = new_state(score_producer="pooled", **(dict(_head_groups=H) if by_groups else {}))
    if "step" in way:
        am.SparseAttentionWithMap(q, k, v, state, LOG, current_step=1)           # collects
    late = [torch.zeros(1, N, H, D, device="cuda", dtype=q.dtype) for _ in range(3)]
    lists = ops.tile_lists(mask, BS, N, heads_per_group=1 if by_groups else None)
    torch.cuda.synchronize()
    side, ready = torch.cuda.Stream(), [torch.cuda.Event() for _ in range(H)]
    with torch.cuda.stream(side):
        torch.cuda._sleep(20000000)
        for h, e in enumerate(ready):
            for dst, src in zip(late, (q, k, v)):
                dst[:, :, h].copy_(src[:, h])
            e.record()
    leaves = [t.transpose(1, 2).requires_grad_(ask) for t in late]
    if way == "value":
        out = am.AttentionSparseEngine(*leaves, mask, block_size=BS, _lists=lists, _value_ready=ready[-1])
    elif way == "groups":
        out = am.AttentionSparseEngine(*leaves, mask, block_size=BS, _lists=lists, _group_ready=ready)
    else:
        events = dict(head_group_ready=ready) if by_groups else dict(qk_ready=ready[-1])
        out, _ = am.SparseAttentionWithMap(*leaves, state, LOG, current_step=2, pooled_qk=pools, **events)
        mask = state["mask"]
    got = torch.autograd.grad(out, leaves, dout) if ask else None
    torch.cuda.synchronize()
    want_out, want = wanted(mods, q, k, v, dout, mask)
    assert torch.equal(out, want_out) and (not ask or same(got, want))
