"""Drafted-tree operators made on one stream, or inside a capture, and used elsewhere."""
import pytest
import torch

from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
from tests.tree_support import expected, make_tree_case

pytestmark = pytest.mark.gpu


def inputs(made):
    case, paths, cmp_paths, ori_scale, cmp_scale = made
    move = lambda t: None if t is None else t.to("cuda")  # noqa: E731
    return (case.to("cuda"), move(paths), move(ori_scale), move(cmp_scale)), dict(cmp_paths=move(cmp_paths), return_lse=True)


def recycled(name, shape, dtype, device):
    """Scratch that others have written to."""
    return torch.full(shape, 0x5A, dtype=dtype, device=device)


def check(op, made):
    op.status()
    want, want_lse, bound, lse_bound = expected(*made)
    assert ((op.out.cpu().double() - want).abs() - bound).max() <= 0
    assert ((op.lse.cpu().double() - want_lse).abs() - lse_bound).max() <= 0


@pytest.mark.parametrize("ratio", [1, 4, 128])
def test_made_on_a_busy_stream(ratio):
    """What the constructor queues comes after the launches, on another stream."""
    made = make_tree_case([6, 9], [700, 130], ratio=ratio, topk=40, seed=3)
    where, more = inputs(made)
    side = torch.cuda.Stream()
    scratch = {}

    def allocate(name, shape, dtype, device):
        return scratch.setdefault(name, recycled(name, shape, dtype, device))

    PreparedTreeAttention(*where, scratch_allocator=allocate, **more)             # so that the scratch has been filled
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)                                             # about ten milliseconds
        op = PreparedTreeAttention(*where, scratch_allocator=allocate, **more)
    for _ in range(3):
        op.out.fill_(float("nan"))
        op.run()
        torch.cuda.current_stream().synchronize()
        want, _, bound, _ = expected(*made)
        assert ((op.out.cpu().double() - want).abs() - bound).max() <= 0
    torch.cuda.synchronize()
    op.run()
    check(op, made)


@pytest.mark.parametrize("ratio", [1, 4, 128])
def test_made_inside_a_capture(ratio):
    """The operator is used outside before the graph has run, then by the graph, then outside again."""
    made = make_tree_case([6, 9], [700, 130], ratio=ratio, topk=40, seed=4)
    where, more = inputs(made)
    buffers = [recycled(None, (1 << 26,), torch.uint8, "cuda")]
    PreparedTreeAttention(*where, **more).run()                                   # one-time work of the library
    out, lse = torch.empty_like(where[0].q), torch.empty(where[0].q.shape[:2], device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op = PreparedTreeAttention(*where, cmp_paths=more["cmp_paths"], output=out, lse_output=lse,
                                   scratch_allocator=lambda name, shape, dtype, device: buffers[0][:shape[0]])
        op.run()
    for use in (op.run, graph.replay, graph.replay, op.run):
        out.fill_(float("nan"))
        lse.fill_(float("nan"))
        use()
        check(op, made)
