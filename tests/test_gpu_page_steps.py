"""Page-pool calls in the order a user makes them."""
from pathlib import Path
import random
import re
from types import SimpleNamespace

import pytest
import torch

from npu_sparse_attn_sharedkv_int8 import PagePool, PreparedTreeAttention
from npu_sparse_attn_sharedkv_int8.reference import SharedKVCase
from npu_sparse_attn_sharedkv_int8.tree_attention import path_masks
from tests.test_gpu_pages import check, ints, make_pool
from tests.tree_support import expected

pytestmark = pytest.mark.gpu


def test_readme_example():
    """The speculative step of README.md, as it stands there."""
    text = (Path(__file__).resolve().parents[1] / "README.md").read_text()
    example = next(block for block in re.findall(r"```python\n(.*?)```", text, re.S) if "PagePool" in block)
    gen = torch.Generator().manual_seed(2)
    parents, chosen = [-1, 0, 0, 1, 3], [0, 1, 3]
    start, n = [62, 40], len(parents)
    caches = [torch.randint(-127, 128, (12, 32, 1, 512), dtype=torch.int8, generator=gen).cuda() for _ in range(2)]
    table = torch.full((2, 4), -1, dtype=torch.int32)
    table[0, :2], table[1, :2] = torch.tensor([7, 3]), torch.tensor([1, 9])
    table, lens = table.cuda(), ints(start)
    before = [c.clone() for c in caches]
    draft = [torch.randint(-127, 128, (n, 512), dtype=torch.int8, generator=gen).cuda() for _ in caches]

    def write():
        for cache, rows in zip(caches, draft):
            for i, row in enumerate(rows):
                cache[table[0, (start[0] + i) // 32].long(), (start[0] + i) % 32, 0] = row

    scale = torch.full((512,), 4 / 127, device="cuda")
    case = SharedKVCase(q=torch.randn(n, 8, 512, generator=gen).to(torch.bfloat16).cuda(), ori=caches[0], ori_block_table=table, cu_q=ints([0, n, n]),
                        seq_lens=ints([start[0] + n, start[1]]), sink=torch.zeros(8, device="cuda"))
    names = dict(caches=caches, block_table=table, lens=lens, drafted=ints([n, 0]), writer=SimpleNamespace(run=write), case=case, parents=parents,
                 ori_scale=scale, cmp_scale=None, accepted=ints([chosen + [-1] * (n - len(chosen)), [-1] * n]), accepted_rows=ints([len(chosen), 0]),
                 parent_of=ints([0, 0]))
    exec(example, names)
    names["pool"].status()
    rows = lambda cache, b, count: torch.cat([cache[p.long(), :, 0] for p in names["block_table"][b] if p >= 0])[:count]  # noqa: E731
    end = start[0] + len(chosen)
    assert lens.tolist() == [end, end]
    for cache, old, new in zip(caches, before, draft):
        want = torch.cat([old[7, :, 0], old[3, :30, 0], new[chosen]])
        assert torch.equal(rows(cache, 0, end), want) and torch.equal(rows(cache, 1, end), want)
    plain = SharedKVCase(**{k: v.cpu() if isinstance(v, torch.Tensor) else v for k, v in vars(case).items()})
    plain.ori = torch.cat([before[0][[7, 3], :, 0].reshape(64, 512)[:62], draft[0], torch.zeros(29, 512, dtype=torch.int8, device="cuda")]).view(3, 32, 1, 512).cpu()
    plain.ori_block_table = torch.tensor([[0, 1, 2], [-1, -1, -1]], dtype=torch.int32)
    want, _, bound, _ = expected(plain, path_masks(parents), None, scale.cpu(), None)
    assert ((names["out"].cpu().double() - want).abs() - bound).max() <= 0


def test_keep_refuses_the_pools_own_lengths():
    """They include the draft once there is room for it, so that nothing would be kept."""
    cache = torch.zeros(8, 32, 1, 512, dtype=torch.int8, device="cuda")
    pool = PagePool([cache], torch.zeros(2, 3, dtype=torch.int32, device="cuda"), ints([0, 0]))
    with pytest.raises(ValueError, match="tensor of its own"):
        pool.keep(pool.lens, ints([[0], [0]]))
    pool.keep(pool.lens.clone(), ints([[0], [0]]))


def test_a_refusal_can_be_handled():
    """Too few pages; a sequence is freed; the second attempt holds and says so, also from a captured graph."""
    cache = torch.randint(-127, 128, (6, 32, 1, 512), dtype=torch.int8, device="cuda")
    table = torch.full((2, 6), -1, dtype=torch.int32, device="cuda")
    pool = PagePool([cache], table, ints([0, 0]))
    pool.resize(ints([96, 96]))
    pool.status()
    pool.resize(ints([128, 96]))
    with pytest.raises(RuntimeError, match="refused"):
        pool.status()
    pool.clear_status()
    pool.status()
    pool.resize(ints([96, 0]))
    pool.resize(ints([128, 0]))
    pool.status()
    assert pool.lens.tolist() == [128, 0] and pool.refs.sum() == 4
    wanted = ints([128, 0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.clear_status()
        pool.resize(wanted)
    for lens, holds in (([128, 64], True), ([128, 96], False), ([192, 0], True)):
        wanted.copy_(ints(lens))
        graph.replay()
        if holds:
            pool.status()
        else:
            with pytest.raises(RuntimeError, match="refused"):
                pool.status()
    assert pool.lens.tolist() == [192, 0]


@pytest.mark.parametrize("batch, width, rows", [(8192, 3, 1), (8191, 4, 2), (4097, 9, 1), (2049, 40, 1)])
def test_many_sequences(batch, width, rows):
    """Up to the most that a pool holds, where a fork moves the table two columns at a time."""
    rng = random.Random(batch)
    pool, model = make_pool(rng, batch, batch * width + 100, layers=1, rows=rows, width=width, shared=True)
    most = width * rows
    for step in range(4):
        if step % 2:
            parents = [rng.randrange(-1, batch) for _ in range(batch)]
            pool.fork(ints(parents))
            model.fork(parents)
        else:
            wanted = [max(0, min(most, n + rng.randint(-2 * rows, 2 * rows))) for n in model.lens]
            pool.resize(ints(wanted))
            model.resize(wanted)
        assert not model.refused
        check(pool, model)
