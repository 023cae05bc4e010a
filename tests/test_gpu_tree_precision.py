"""Drafted-tree attention where its arithmetic is strained: results against float64 in fixed bands that do not
grow with the number of keys."""
from dataclasses import replace
import math

import pytest
import torch

from npu_sparse_attn_sharedkv_int8 import PreparedAttention, PreparedTreeAttention
from npu_sparse_attn_sharedkv_int8.reference import SharedKVCase
from npu_sparse_attn_sharedkv_int8.tree_attention import path_masks
from tests.tree_support import check_dense, make_tree_case

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
    case, ori_scale, cmp_scale = case.to("cuda"), ori_scale.cuda(), None if cmp_scale is None else cmp_scale.cuda()
    n = int(case.cu_q[1])
    prefix = int(case.seq_lens[0]) - n
    whole = prefix // case.ratio

    def rows(cache, table, scale, logical):
        logical = torch.tensor(logical, dtype=torch.int64, device="cuda")
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
        out[t], lse[t] = (w[:, :-1] @ v).cpu(), s.logsumexp(1).cpu()
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


def peaked(rows, gap, *, ratio, noise, peak, period=0, seed=0):
    """A chain of three tokens over `rows` compressed rows and a window.  All rows have a common component and logits of
    deviation `noise`, but for number `peak`, which has the opposite component and a logit `gap` nats above the others' mean.
    With `period` the rows repeat."""
    gen = torch.Generator().manual_seed(seed + 1)
    whole = rows if ratio == 128 else 9000
    prefix = whole * ratio + 1
    base, u = torch.randint(-40, 41, (512,), generator=gen), torch.where(torch.rand(512, generator=gen) < 0.5, -1, 1)

    def pool(count):
        tail = torch.randn(period or count * 32, 512, generator=gen).repeat(-(-count * 32 // (period or count * 32)), 1)[:count * 32] * 20 * noise
        return (base + tail).round().clamp(-127, 127).to(torch.int8).view(count, 32, 1, 512)

    table = torch.full((1, prefix // 32 + 2), -1, dtype=torch.int32)
    near = torch.arange((prefix - 128) // 32, (prefix + 2) // 32 + 1)
    table[0, near] = torch.randperm(len(near), generator=gen).to(torch.int32)
    pages = (whole + 64) // 32 + 1
    scale = (torch.randn(512, generator=gen) * 0.3).exp() * (4 / 127)
    # queries: 1.45 x normal gives the tail's logits deviation 1; none along the common component, and the same in all along u, in
    # which the peak leaves the others
    q = torch.randn(3, 8, 512, generator=gen) * 1.45
    along, common = scale * u, scale * base
    common = common - (common @ along) / (along @ along) * along
    for v in (along, common):
        q -= (q @ v)[..., None] / (v @ v) * v
    step = u - (common @ u.float()) / (common @ common) * common
    q += step * gap * math.sqrt(512) / (40 * float(along @ step) - 2 * float((scale * base) @ step))
    case = SharedKVCase(q=q.to(torch.bfloat16), ori=pool(len(near)), ori_block_table=table, cu_q=torch.tensor([0, 3], dtype=torch.int32),
                        seq_lens=torch.tensor([prefix + 3], dtype=torch.int32), sink=torch.full((8,), -40.0), cmp=pool(pages),
                        cmp_block_table=torch.randperm(pages, generator=gen).to(torch.int32)[None].contiguous(), ratio=ratio)
    if ratio == 4:
        case.cmp_indices = torch.stack([torch.randperm(whole, generator=gen)[:rows] for _ in range(3)])[:, None].to(torch.int32)
        case.cmp_indices = torch.where(case.cmp_indices == peak, -1, case.cmp_indices)
        case.cmp_indices[:, 0, 17] = peak
    case.cmp[cmp_row(case, peak)] = (40 * u - base).to(torch.int8)
    return case, torch.tensor([1, 3, 7]), torch.zeros(3, dtype=torch.int64) if ratio == 128 else None, scale, scale.clone()


def repeated(made, times):
    """The requests `times` over: with more of them than SMs, most are worked on by one block from end to end."""
    case, paths, cmp_paths, ori_scale, cmp_scale = made
    again = lambda t: None if t is None else t.repeat(times, *[1] * (t.ndim - 1))  # noqa: E731
    starts = case.cu_q[:-1] + len(case.q) * torch.arange(times, dtype=torch.int32)[:, None]
    case = replace(case, q=again(case.q), ori_block_table=again(case.ori_block_table), cmp_block_table=again(case.cmp_block_table),
                   seq_lens=again(case.seq_lens), cu_q=torch.cat([starts.flatten(), torch.tensor([times * len(case.q)], dtype=torch.int32)]),
                   cmp_indices=again(case.cmp_indices))
    return case, again(paths), again(cmp_paths), ori_scale, cmp_scale


def row_errors(out, want):
    return (out - want).norm(dim=-1) / want.norm(dim=-1)


SHAPES = ((1, 0.0, 0), (1, 0.6, 0), (0.3, 1.0, 0), (0, 0.6, 0), (0.5, 0.4, 128))            # noise, place of the peak, period
PEAKED = [(ratio, rows, gap, *shape) for ratio, rows, gaps in ((4, 1024, (5, 9, 10)), (128, 1024, (9,)), (128, 4096, (6, 9, 10)), (128, 8192, (4, 8, 10, 11)))
          for gap in gaps for shape in (SHAPES if gap in (9, 10) else SHAPES[:2])]


@pytest.mark.parametrize("ratio, rows, gap, noise, place, period", PEAKED)
def test_peaked_rows_keep_their_tail(ratio, rows, gap, noise, place, period):
    """One row holds much of the weight and thousands of small ones the rest.  A weight code is a whole number of
    steps of 2 / 32638 of the largest weight (8 / 32638 in the tile that brings it), unbiased and off by half a step on
    the mean square at most, so that the errors of n keys add up to sqrt(n) / 2 steps: 0.0028 of the largest row at 8320 keys.
    BF16 rounds by half a step, 0.0017 over a row; together 0.0033, and the band is half as much again.  The
    denominators' weights have steps of 2^-20 and less, and the query codes move a logit by 2^-11 at most."""
    made = peaked(rows, gap, ratio=ratio, noise=noise, peak=min(int(rows * place), rows - 1), period=period)
    want, want_lse = definition(made)
    out, lse = launch(repeated(made, 200))
    worst, worst_lse = float(row_errors(out.view(200, 3, 8, 512), want).max()), float((lse.view(200, 3, 8) - want_lse).abs().max())
    print(f"ratio {ratio} rows {rows} gap {gap} noise {noise} place {place} period {period}: out {worst:.5f} lse {worst_lse:.6f}")
    assert worst <= 0.005 and worst_lse <= 2.0 ** -10


@pytest.mark.parametrize("rows, gap", [(1024, 9), (1024, 10), (4096, 9), (4096, 10), (8192, 10), (8192, 11)])
def test_peaked_rows_as_the_decode_attention(rows, gap):
    """The decode attention's codes have steps of 1 / 16129, rounded to nearest: a deviation of sqrt(1 / 12) of a step
    where weights span several, against sqrt(1 / 6) of nearly the same step here,
    and both round to BF16.  (Small weights its rounding loses, which is not asked for here.)"""
    made = peaked(rows, gap, ratio=128, noise=1, peak=rows // 2, seed=3)
    want, want_lse = definition(made)
    made = repeated(made, 200)
    out, lse = (t.view(200, 3, 8, -1) for t in launch(made))
    dev = made[0].to("cuda")
    decode = PreparedAttention(dev, made[3].cuda(), made[4].cuda(), return_lse=True)
    decode.run()
    mine, theirs = row_errors(out, want).square().mean().sqrt(), row_errors(decode.out.cpu().double().view(200, 3, 8, 512), want).square().mean().sqrt()
    mine_lse, theirs_lse = ((t.view(200, 3, 8) - want_lse).abs().max() for t in (lse, decode.lse.cpu().double()))
    print(f"rows {rows} gap {gap}: tree {float(mine):.5f} decode {float(theirs):.5f} lse {float(mine_lse):.6f} {float(theirs_lse):.6f}")
    assert mine <= math.sqrt(2) * theirs


@pytest.mark.parametrize("ratio", [4, 128])
def test_rows_that_are_not_finite_leave_the_others_alone(ratio):
    """On walks of many tiles too, where references move: the other rows' results are those of a launch without them."""
    made = make_tree_case([9, 40], [128 * 90, 128 * 70] if ratio == 128 else [9000, 7000], ratio=ratio, topk=1024, seed=12, spread=2.0)
    case = made[0]
    broken = replace(case, q=case.q.clone())
    rows = [(0, 0), (3, 2), (20, 5), (48, 7)]
    for i, (t, h) in enumerate(rows):
        broken.q[t, h, 11 * i] = (math.nan, math.inf, -math.inf)[i % 3]
    want, want_lse = launch(repeated(made, 30))
    out, lse = launch(repeated((broken, *made[1:]), 30))
    keep = torch.ones(49, 8, dtype=torch.bool)
    for t, h in rows:
        keep[t, h] = False
    keep = keep.repeat(len(out) // 49, 1)
    assert torch.equal(out[keep], want[keep]) and torch.equal(lse[keep], want_lse[keep])
    assert out[~keep].isnan().all() and lse[~keep].isnan().all()


@pytest.mark.parametrize("ratio", [4, 128])
def test_channels_without_a_scale(ratio):
    """A channel may be zero, or next to it, in one cache and not in the other."""
    case, paths, cmp_paths, ori_scale, cmp_scale = make_tree_case([9, 40], [128 * 90, 128 * 70] if ratio == 128 else [9000, 7000], ratio=ratio, topk=333,
                                                                  seed=14)
    cmp_scale[5], cmp_scale[140], cmp_scale[300], ori_scale[6], ori_scale[511] = 0, 0, 1e-36, 0, 1e-36
    ori_scale[301] = cmp_scale[301] = 0
    made = repeated((case, paths, cmp_paths, ori_scale, cmp_scale), 30)
    out, lse = launch(made)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    dev = made[0].to("cuda")
    worst = check_dense(dev, made[1].cuda(), None if cmp_paths is None else made[2].cuda(), ori_scale.cuda(), cmp_scale.cuda(), out.cuda(), lse.cuda())
    assert worst[0] <= 1 and worst[1] <= 1, worst
    assert out[..., 301].eq(0).all()


@pytest.mark.parametrize("options", [dict(counts=[64, 40, 64, 7], prefix=[128 * 2000, 128 * 900 + 77, 128 * 3000 + 5, 128 * 1500], ratio=128),
                                     dict(counts=[30, 9], prefix=[14000, 5555], ratio=4, topk=777, spread=2.5),
                                     dict(counts=[64, 31], prefix=[9000, 5000], window=4000, spread=1.5)], ids=["c128", "c4", "wide window"])
def test_every_row_is_written(options):
    """Long walks leave no element of a live row as it was (a NaN)."""
    case, paths, cmp_paths, ori_scale, cmp_scale = make_tree_case(seed=100, **options)
    move = lambda t: None if t is None else t.to("cuda")  # noqa: E731
    tokens = len(case.q)
    out, lse = (torch.full(shape, math.nan, dtype=dtype, device="cuda") for shape, dtype in (((tokens, 8, 512), torch.bfloat16), ((tokens, 8), torch.float32)))
    PreparedTreeAttention(case.to("cuda"), move(paths), move(ori_scale), move(cmp_scale), cmp_paths=move(cmp_paths), output=out, lse_output=lse).run()
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("options", [dict(prefix=[5000], window=4000), dict(prefix=[9000], ratio=4, topk=1024), dict(prefix=[128 * 2500 + 3], ratio=128)],
                         ids=["wide window", "c4", "c128"])
def test_uneven_rows(options, seed):
    """Rows that range from flat to a single key, side by side in their octets, with keys that stand out in every part of the walk.
    A row's error: BF16's half step, and the codes' of up to 4096 keys, sqrt(n) / 2 steps of 8 / 32638 of the largest weight at
    the very most (0.008 of the largest row, where the sum of a row's weighted values may be as small as that)."""
    made = make_tree_case([24], seed=seed, **options)
    case, gen = made[0], torch.Generator().manual_seed(seed + 50)
    case.q = (case.q.float() * torch.exp(torch.randn(24, 8, 1, generator=gen) * 0.8)).to(torch.bfloat16)
    for cache in (case.ori, case.cmp) if case.ratio > 1 else (case.ori,):
        rows = cache.view(-1, 512)
        for r in torch.randint(0, len(rows), (30,), generator=gen).tolist():
            t, h = int(torch.randint(0, 24, (1,), generator=gen)), int(torch.randint(0, 8, (1,), generator=gen))
            toward = case.q[t, h].float()
            rows[r] = (rows[r].float() * 0.7 + toward / toward.norm() * 22 * (10 + 30 * float(torch.rand(1, generator=gen)))).round().clamp(-127, 127).to(torch.int8)
    want, want_lse = definition(made)
    copies = 40
    out, lse = launch(repeated(made, copies))
    errors = row_errors(out.view(copies, 24, 8, 512), want)
    print(f"{options} seed {seed}: out {float(errors.max()):.5f} mean {float(errors.mean()):.5f} lse {float((lse.view(copies, 24, 8) - want_lse).abs().max()):.5f}")
    assert errors.max() <= 0.012 and errors.square().mean().sqrt() <= 0.003
    assert ((lse.view(copies, 24, 8) - want_lse).abs() <= 2.0 ** -9 + want_lse.abs() * 2.0 ** -12).all()
