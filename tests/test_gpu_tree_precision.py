"""Drafted-tree attention where its arithmetic is strained: results against float64 in fixed bands that do not
grow with the number of keys."""
import math

import pytest
import torch

from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
from npu_sparse_attn_sharedkv_int8.tree_attention import path_masks
from tests.tree_support import make_tree_case

pytestmark = pytest.mark.gpu


def launch(made):
    case, paths, cmp_paths, ori_scale, cmp_scale = made
    move = lambda t: None if t is None else t.to("cuda")  # noqa: E731
    op = PreparedTreeAttention(case.to("cuda"), move(paths), move(ori_scale), move(cmp_scale), cmp_paths=move(cmp_paths), return_lse=True)
    op.run()
    op.status()
    return op.out.cpu().double(), op.lse.cpu().double()


def definition(made):
    """(out, lse) of the live tokens of request 0 in float64."""
    case, paths, cmp_paths, ori_scale, cmp_scale = made
    n = int(case.cu_q[1])
    prefix = int(case.seq_lens[0]) - n
    whole = prefix // case.ratio

    def rows(cache, table, scale, logical):
        logical = torch.tensor(logical, dtype=torch.int64)
        return cache[table[0, logical // 32].long(), logical % 32, 0].double() * scale.double()

    out, lse = torch.zeros(n, case.q.shape[1], 512, dtype=torch.float64), torch.zeros(n, case.q.shape[1], dtype=torch.float64)
    for t in range(n):
        drafted = [j for j in range(n) if int(paths[t]) >> j & 1]
        near = list(range(max(0, prefix - case.window + len(drafted)), prefix)) + [prefix + j for j in drafted]
        v = [rows(case.ori, case.ori_block_table, ori_scale, near)]
        if case.ratio == 128:
            v.append(rows(case.cmp, case.cmp_block_table, cmp_scale, list(range(whole)) + [whole + e for e in range(64) if int(cmp_paths[t]) >> e & 1]))
        elif case.ratio == 4:
            v.append(rows(case.cmp, case.cmp_block_table, cmp_scale, [r for r in case.cmp_indices[t, 0].tolist() if 0 <= r < whole + 64]))
        v = torch.cat(v)
        s = torch.cat([case.q[t].double() @ v.T * case.softmax_scale, case.sink.double()[:, None]], 1)
        w = s.softmax(1)
        out[t], lse[t] = w[:, :-1] @ v, s.logsumexp(1)
    return out, lse


def cmp_row(case, row):
    """Where compressed row `row` of request 0 lies."""
    return int(case.cmp_block_table[0, row // 32]), row % 32, 0


@pytest.mark.parametrize("ratio", [4, 128])
@pytest.mark.parametrize("sign", [1, -1], ids=["above", "below"])
@pytest.mark.parametrize("size", [1e6, 1e8, 1e10, 1e20, 1e33])
def test_large_finite_logits(size, sign, ratio):
    """Logits far beyond what FP32 resolves to a unit, but finite: the row with the largest one is the answer.  Its
    logit is twice the others' (half of it, where all are negative), so no rounding makes another row the largest."""
    rows, best = 700, {1: 515, -1: 300}[sign]
    made = make_tree_case([3], [ratio * rows + 1], ratio=ratio, topk=600, seed=7, sink=torch.full((8,), -math.inf))
    case, gen = made[0], torch.Generator().manual_seed(1)
    direction = torch.where(torch.rand(512, generator=gen) < 0.5, -1, 1)
    # every row lies along one direction, by 40 to 60 codes; the best one by 120 (or, where logits are negative, by 20)
    for cache in (case.ori, case.cmp):
        cache.copy_((torch.randint(40, 61, (*cache.shape[:3], 1), generator=gen) * direction).to(torch.int8))
    case.cmp[cmp_row(case, best)] = ((120 if sign > 0 else 20) * direction).to(torch.int8)
    if ratio == 4:
        case.cmp_indices[:, 0, 5:8] = best                    # named three times
    scale = torch.full((512,), 2.0 ** -5)
    case.q = (sign * size / 64 * direction).expand(3, 8, 512).to(torch.bfloat16).clone()      # logits of the size of `size`
    case.q[1, 3] = torch.randn(512, generator=gen).to(torch.bfloat16)                        # a neighbour of ordinary size
    made = (case, made[1], made[2], scale, scale.clone())
    out, lse = launch(made)
    want, want_lse = definition(made)
    # out: one BF16 rounding, half a step; codes of the ordinary neighbour, whose weights are alike, are off by 1e-3 of them at most.
    # LSE: code planes in steps of a power of two leave half a step in 254 x 63, 2^-14.9; a neighbour is off by 2^-9 at most.
    assert ((out - want).abs() <= want.abs() * 2.0 ** -8 + 2.0 ** -9).all(), float((out - want).abs().max())
    assert ((lse - want_lse).abs() <= want_lse.abs() * 2.0 ** -14 + 2.0 ** -9).all()
