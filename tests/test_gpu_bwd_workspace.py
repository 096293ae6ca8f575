"""What a workspace held before a call of the attention's backward pass reaches nothing: called through the C entry point, on
one workspace, which holds NaN or the statistics of other inputs.  The results have to be the bits of a call that found its own
statistics there already (made after a finished one on the same workspace)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

# heads, rows, block, density: statistics on a part of the SMs, on all of them, in several waves
SIZES = [(1, 1200, 64, 0.6), (6, 333, 64, 0.7), (2, 4096, 128, 0.3), (8, 9000, 128, 0.2)]


@pytest.fixture(scope="module")
def ops():
    from moddit_b200 import ops as _ops
    return _ops


def problem(ops, size, D, dtype, seed):
    H, N, bs, density = size
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v, dout = (torch.randn(1, H, N, D, generator=g, device="cuda").to(dtype) for _ in range(4))
    nb = (N + bs - 1) // bs
    mask = (torch.rand(H, nb, nb, generator=g, device="cuda") < density) | torch.eye(nb, dtype=torch.bool, device="cuda")
    lists, klists = ops.tile_lists(mask, bs, N), ops.key_lists(mask, bs, N)
    out, lse = ops.sparse_attn_fwd(q, k, v, *lists, order=lists.order, return_lse=True)
    return (q, k, v, out, dout, lse), lists, klists


def backward(ops, job, ws, grads):
    (q, k, v, out, dout, lse), lists, klists = job
    H, N, D = q.shape[1:]
    p = torch.Tensor.data_ptr
    dtype = 0 if q.dtype == torch.bfloat16 else 1
    ops.check(ops.lib.moddit_sparse_attn_bwd(
        p(q), p(k), p(v), p(out), None, p(dout), p(lse), dtype, H, N, D, p(lists.counts), p(lists.entries), p(lists.order),
        p(klists.counts), p(klists.entries), p(klists.order), lists.counts.shape[0], D ** -0.5, N, N, N, *map(p, grads), p(ws),
        ws.numel() * 4, p(ops._status_words(q.device)), torch.cuda.current_stream().cuda_stream), "moddit_sparse_attn_bwd")


def workspace(ops, q):
    return torch.empty(ops.lib.moddit_sparse_attn_bwd_workspace_bytes(q.shape[1], q.shape[2]) // 4, device="cuda")


def settled(ops, job, ws):
    grads = [torch.empty_like(job[0][0]) for _ in range(3)]
    for _ in range(2):
        backward(ops, job, ws, grads)
        torch.cuda.synchronize()
    assert all(torch.isfinite(t).all() for t in grads)
    return [t.clone() for t in grads]


def differing(got, want):
    return torch.stack([(a.view(torch.int16) != b.view(torch.int16)).sum() for a, b in zip(got, want)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s[:2])))
def test_nan_before_every_call(ops, size, D, dtype):
    job = problem(ops, size, D, dtype, 1)
    ws = workspace(ops, job[0][0])
    want = settled(ops, job, ws)
    grads, wrong = [torch.empty_like(t) for t in want], torch.zeros(3, dtype=torch.int64, device="cuda")
    for _ in range(200):
        ws.fill_(float("nan"))
        backward(ops, job, ws, grads)
        wrong += differing(grads, want)
    ops.raise_on_status(ws.device)
    assert wrong.tolist() == [0, 0, 0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s[:2])))
def test_two_sets_of_inputs_in_turn(ops, size, D, dtype):
    jobs = [problem(ops, size, D, dtype, seed) for seed in (2, 3)]
    ws = workspace(ops, jobs[0][0][0])
    wants = [settled(ops, job, ws) for job in jobs]
    grads, wrong = [torch.empty_like(t) for t in wants[0]], torch.zeros(3, dtype=torch.int64, device="cuda")
    for _ in range(100):
        for job, want in zip(jobs, wants):
            backward(ops, job, ws, grads)
            wrong += differing(grads, want)
    ops.raise_on_status(ws.device)
    assert wrong.tolist() == [0, 0, 0]
