"""A speculative step as a serving loop runs it: room for the draft, its rows written, tree attention
over pages of a pool, the accepted rows kept, the rest given back, and a fork."""
import random

import pytest
import torch

from npu_sparse_attn_sharedkv_int8 import CacheQuantization, PagePool, PreparedCacheWrite, PreparedTreeAttention
from npu_sparse_attn_sharedkv_int8.reference import SharedKVCase
from npu_sparse_attn_sharedkv_int8.tree_attention import path_masks
from tests.tree_support import expected

pytestmark = pytest.mark.gpu


def test_speculative_steps():
    rng, gen = random.Random(1), torch.Generator().manual_seed(1)
    batch, pages, nodes = 4, 64, 6
    quant = [CacheQuantization((torch.rand(512, generator=gen) + 0.5) / 40) for _ in range(2)]
    caches = [torch.zeros(pages, 32, 1, 512, dtype=torch.int8, device="cuda") for _ in range(2)]
    table = torch.full((batch, 10), -1, dtype=torch.int32, device="cuda")
    pool = PagePool(caches, table, torch.zeros(batch, dtype=torch.int32, device="cuda"))
    content = [[[] for _ in range(batch)] for _ in range(2)]             # per layer and sequence: the rows, as codes
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731

    def write(start, count):
        """Rows [start, start + count) of every sequence, in both layers."""
        rows = [(b, r) for b in range(batch) for r in range(start[b], start[b] + count[b])]
        b, r = (torch.tensor(v, device="cuda") for v in zip(*rows))
        slots = table[b, r // 32].long() * 32 + r % 32
        for layer in range(2):
            new = torch.randn(len(rows), 512, generator=gen).to(torch.bfloat16)
            PreparedCacheWrite(caches[layer], new.cuda(), slots, quant[layer].inverse_scale.cuda()).run()
            for (sequence, _), codes in zip(rows, quant[layer].quantize(new)):
                content[layer][sequence].append(codes)

    lens = [5, 40, 130, 64]
    pool.resize(ints(lens))
    write([0] * batch, lens)
    for step in range(3):
        parents = [[rng.randint(-1, i - 1) for i in range(nodes)] for _ in range(batch)]
        paths = torch.cat([path_masks(p) for p in parents])
        pool.resize(ints([n + nodes for n in lens]))
        write(lens, [nodes] * batch)
        for layer in range(2):
            case = SharedKVCase(q=torch.randn(batch * nodes, 8, 512, generator=gen).to(torch.bfloat16), ori=caches[layer], ori_block_table=table,
                                cu_q=torch.arange(0, batch * nodes + 1, nodes, dtype=torch.int32),
                                seq_lens=torch.tensor([n + nodes for n in lens], dtype=torch.int32), sink=torch.linspace(-1, 1, 8))
            op = PreparedTreeAttention(case.to("cuda"), paths.cuda(), quant[layer].scale.cuda())
            op.run()
            # the same attention over the rows as the test remembers them
            width = -(-max(len(c) for c in content[layer]) // 32)
            cache = torch.zeros(batch * width, 32, 1, 512, dtype=torch.int8)
            for b, rows in enumerate(content[layer]):
                cache[b * width:(b + 1) * width].view(-1, 512)[:len(rows)] = torch.stack(rows)
            plain = SharedKVCase(**{**vars(case), "ori": cache, "ori_block_table": torch.arange(batch * width, dtype=torch.int32).view(batch, width)})
            want, _, bound, _ = expected(plain, paths, None, quant[layer].scale, None)
            assert ((op.out.cpu().double() - want).abs() - bound).max() <= 0
        accepted = []
        for b in range(batch):
            node, chain = rng.randrange(nodes), []
            while node >= 0:
                chain.insert(0, node)
                node = parents[b][node]
            accepted.append(chain)
        pool.keep(ints(lens), ints([c + [-1] * (nodes - len(c)) for c in accepted]))
        for layer in range(2):
            for b in range(batch):
                rows = content[layer][b]
                content[layer][b] = rows[:lens[b]] + [rows[lens[b] + j] for j in accepted[b]]
        lens = [n + len(c) for n, c in zip(lens, accepted)]
        pool.resize(ints(lens))
        order = [rng.randrange(batch) for _ in range(batch)]
        pool.fork(ints(order))
        lens = [lens[p] for p in order]
        content = [[list(layer[p]) for p in order] for layer in content]
    pool.resize(ints([0] * batch))
    torch.cuda.synchronize()
    pool.status()
    assert pool.refs.eq(0).all()
