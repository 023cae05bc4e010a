"""Drafted-tree attention against its definition in float64 (tree_support has the bounds)."""
from dataclasses import replace
import math
import random
from types import SimpleNamespace

import pytest
import torch

from npu_sparse_attn_sharedkv_int8 import PreparedAttention, PreparedTreeAttention, vllm_adapter
from npu_sparse_attn_sharedkv_int8.reference import SharedKVCase
from npu_sparse_attn_sharedkv_int8.tree_attention import path_masks
from tests.support import strided_pages
from tests.tree_support import check_dense, expected, make_tree_case

pytestmark = pytest.mark.gpu


def on_device(made, stride=None, offset=0, device="cuda"):
    case, paths, cmp_paths, ori_scale, cmp_scale = made
    dev = case.to(device)
    if stride:
        dev.ori = strided_pages(case.ori, device, stride, offset)
        if case.cmp is not None:
            dev.cmp = strided_pages(case.cmp, device, stride, offset)
    move = lambda t: None if t is None else t.to(device)  # noqa: E731
    return dev, move(paths), move(ori_scale), move(cmp_scale), move(cmp_paths)


def prepared(made, stride=None, offset=0, **more):
    dev, paths, ori_scale, cmp_scale, cmp_paths = on_device(made, stride, offset)
    return PreparedTreeAttention(dev, paths, ori_scale, cmp_scale, cmp_paths=cmp_paths, **more)


def check(op, made, label=""):
    op.status()
    want, want_lse, bound, lse_bound = expected(*made)
    got, got_lse = op.out.cpu().double(), op.lse.cpu().double()
    worst = ((got - want).abs() - bound).max()
    assert worst <= 0, (label, float(worst))
    finite = torch.isfinite(want_lse)
    assert torch.equal(got_lse[~finite], want_lse[~finite])
    assert ((got_lse - want_lse).abs() - lse_bound)[finite].max() <= 0, label


CASES = {
    "one token": dict(counts=[1], prefix=[200]),
    "one token, no past": dict(counts=[1], prefix=[0]),
    "short pasts": dict(counts=[1, 2, 3, 5], prefix=[1, 31, 32, 33]),
    "window edge": dict(counts=[7, 8, 9], prefix=[127, 128, 129]),
    "whole draft": dict(counts=[64, 63, 1], prefix=[300, 95, 96]),
    "more tokens than names": dict(counts=[70, 3], prefix=[130, 64]),
    "window 1": dict(counts=[4, 9], prefix=[50, 0], window=1),
    "window 300": dict(counts=[12, 3], prefix=[700, 200], window=300),
    "window below the path": dict(counts=[20], prefix=[90], window=5, paths=[(1 << i + 1) - 1 for i in range(20)]),
    "16 heads": dict(counts=[5, 17], prefix=[40, 180], heads=16),
    "24 heads": dict(counts=[3, 11], prefix=[10, 300], heads=24),
    "128 heads": dict(counts=[2, 3], prefix=[64, 131], heads=128),
    "c128": dict(counts=[8, 3], prefix=[130, 1000], ratio=128),
    "c128, no group yet": dict(counts=[2, 64], prefix=[5, 127], ratio=128),
    "c128, several tiles": dict(counts=[9, 1, 30], prefix=[128 * 130, 128 * 256 + 5, 128 * 127 + 64], ratio=128),
    "c128, 32 heads": dict(counts=[6], prefix=[128 * 40], ratio=128, heads=32),
    "c4": dict(counts=[8, 5], prefix=[400, 1200], ratio=4),
    "c4, no group yet": dict(counts=[3, 2], prefix=[0, 3], ratio=4, topk=16),
    "c4, one pick": dict(counts=[10], prefix=[90], ratio=4, topk=1),
    "c4, wide lists": dict(counts=[11, 1], prefix=[9000, 5000], ratio=4, topk=1024),
    "c4, odd lists, 16 heads": dict(counts=[13, 4], prefix=[3000, 700], ratio=4, topk=333, heads=16),
    "padding": dict(counts=[4, 2], prefix=[100, 35], ratio=128, pad=2),
    "sharp weights": dict(counts=[8, 4], prefix=[500, 128 * 70], ratio=128, spread=8.0),
}


@pytest.mark.parametrize("stride", [None, 17408, 16400], ids=["packed", "strided", "odd stride"])
@pytest.mark.parametrize("name", list(CASES))
def test_against_definition(name, stride):
    made = make_tree_case(seed=len(name), **CASES[name])
    op = prepared(made, stride, return_lse=True)
    op.out.fill_(float("nan"))
    op.run()
    torch.cuda.synchronize()
    check(op, made, name)


@pytest.mark.parametrize("seed", range(12))
def test_random_geometries(seed):
    rng = random.Random(seed)
    ratio = (1, 4, 128)[seed % 3]
    batch = rng.randint(1, 9)
    made = make_tree_case([rng.choice([1, 2, rng.randint(1, 64)]) for _ in range(batch)],
                          [rng.choice([0, 1, rng.randint(0, 300), rng.randint(0, 128 * 150)]) for _ in range(batch)], ratio=ratio,
                          heads=rng.choice([8, 8, 16]), window=rng.choice([128, 128, 33, 257]), topk=rng.choice([1, 100, 1024]), seed=seed,
                          spread=rng.choice([0.3, 1.0, 4.0]))
    op = prepared(made, rng.choice([None, 18432, 16400]), return_lse=True)
    op.run()
    torch.cuda.synchronize()
    check(op, made)


LONG = {
    "c128": dict(counts=[64, 40, 64, 7], prefix=[128 * 2000, 128 * 900 + 77, 128 * 3000 + 5, 128 * 1500], ratio=128),
    "c128, growing maxima": dict(counts=[64, 64], prefix=[128 * 1800, 128 * 2500], ratio=128, spread=3.0),
    "c128, 16 heads": dict(counts=[33, 50], prefix=[128 * 1700 + 9, 128 * 800], ratio=128, heads=16, spread=2.0),
    "c4": dict(counts=[32, 17, 24], prefix=[24000, 9000, 17001], ratio=4, topk=1024),
    "c4, odd lists": dict(counts=[30, 9], prefix=[14000, 5555], ratio=4, topk=777, spread=2.5),
    "wide window": dict(counts=[64, 31], prefix=[9000, 5000], window=4000, spread=1.5),
}


@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("name", list(LONG))
def test_many_tiles(name, seed):
    """Long walks in which references move again and again, on every row."""
    made = make_tree_case(seed=100 + seed, **LONG[name])
    dev, paths, ori_scale, cmp_scale, cmp_paths = on_device(made)
    op = PreparedTreeAttention(dev, paths, ori_scale, cmp_scale, cmp_paths=cmp_paths, return_lse=True)
    for launch in range(3):
        op.out.fill_(float("nan"))
        op.run()
        worst = check_dense(dev, paths, cmp_paths, ori_scale, cmp_scale, op.out, op.lse)
        assert worst[0] <= 1 and worst[1] <= 1, (launch, worst)
    op.status()


def test_rising_logits():
    """Every compressed row scores higher than the one before it: each tile moves every reference."""
    made = make_tree_case([9, 24], [128 * 700, 128 * 1100], ratio=128, seed=6)
    case = made[0]
    direction = (torch.randn(512, generator=torch.Generator().manual_seed(0)) * 20).round().clamp(-60, 60)
    for b in range(2):
        pages = case.cmp_block_table[b][case.cmp_block_table[b] >= 0].long()
        count = pages.numel() * 32
        slope = torch.linspace(-1, 1, count)[:, None]
        case.cmp[pages] = (slope * direction + case.cmp[pages].view(count, 512) * 0.2).round().clamp(-127, 127).to(torch.int8).view(-1, 32, 1, 512)
    case.q = (torch.sign(torch.randn(case.q.shape[:2], generator=torch.Generator().manual_seed(1)))[..., None] * direction / 20
              + torch.randn(case.q.shape, generator=torch.Generator().manual_seed(2))).to(torch.bfloat16)
    dev, paths, ori_scale, cmp_scale, cmp_paths = on_device(made)
    op = PreparedTreeAttention(dev, paths, ori_scale, cmp_scale, cmp_paths=cmp_paths, return_lse=True)
    op.run()
    worst = check_dense(dev, paths, cmp_paths, ori_scale, cmp_scale, op.out, op.lse)
    assert worst[0] <= 1 and worst[1] <= 1, worst


def test_many_requests():
    """More group slots than the plan keeps in shared memory."""
    rng = random.Random(3)
    counts = [1 + (rng.random() < 0.02) for _ in range(2200)]
    made = make_tree_case(counts, [rng.randint(0, 40) for _ in counts], seed=8)
    dev, paths, ori_scale, _, _ = on_device(made)
    op = PreparedTreeAttention(dev, paths, ori_scale, return_lse=True)
    op.run()
    keep = [b for b in range(len(counts)) if b < 40 or b % 97 == 0 or b > 2190]
    want, want_lse, bound, lse_bound = expected(*made, only=set(keep))
    rows = torch.tensor([t for b in keep for t in range(int(made[0].cu_q[b]), int(made[0].cu_q[b + 1]))])
    assert ((op.out.cpu().double() - want).abs() - bound)[rows].max() <= 0
    assert ((op.lse.cpu().double() - want_lse).abs() - lse_bound)[rows].max() <= 0


@pytest.mark.parametrize("ratio", [4, 128])
def test_contexts_beyond_a_million_rows(ratio):
    """Lists whose rows pass the span of one bitmap; long tables over a small pool."""
    gen, rng = torch.Generator().manual_seed(ratio), random.Random(ratio)
    counts, prefix = [5, 2], [1_300_003, 64]
    cu = torch.tensor([0, 5, 7], dtype=torch.int32)
    pool = lambda pages: (torch.randn(pages, 32, 1, 512, generator=gen) * 32).round().clamp(-127, 127).to(torch.int8)  # noqa: E731
    table = lambda rows, pages: torch.randint(0, pages, (2, -(-rows // 32)), generator=gen, dtype=torch.int32)  # noqa: E731
    whole = prefix[0] // ratio
    case = SharedKVCase(q=torch.randn(7, 8, 512, generator=gen).to(torch.bfloat16), ori=pool(40), ori_block_table=table(prefix[0] + 64, 40), cu_q=cu,
                        seq_lens=torch.tensor([p + n for p, n in zip(prefix, counts)], dtype=torch.int32), sink=torch.linspace(-1, 1, 8), cmp=pool(60),
                        cmp_block_table=table(whole + 96, 60), ratio=ratio)
    cmp_paths = None
    if ratio == 4:
        case.cmp_indices = torch.full((7, 1, 1024), -1, dtype=torch.int32)
        for t in range(5):
            case.cmp_indices[t, 0] = torch.randperm(whole + 64, generator=gen)[:1024].to(torch.int32)
        case.cmp_indices[5:, 0, :60] = torch.arange(60, dtype=torch.int32)
    else:
        cmp_paths = torch.tensor([rng.getrandbits(62) for _ in range(7)])
    paths = torch.cat([path_masks([-1, 0, 0, 1, 3]), path_masks([-1, -1])])
    scale = (torch.randn(512, generator=gen) * 0.3).exp() * (4 / 127)
    dev, paths, ori_scale, cmp_scale, cmp_paths = on_device((case, paths, cmp_paths, scale, scale * 1.1))
    op = PreparedTreeAttention(dev, paths, ori_scale, cmp_scale, cmp_paths=cmp_paths, return_lse=True)
    op.run()
    worst = check_dense(dev, paths, cmp_paths, ori_scale, cmp_scale, op.out, op.lse)
    assert worst[0] <= 1 and worst[1] <= 1, worst


def test_offsets_beyond_32_bits():
    """Pages more than 4 GB into their cache."""
    made = make_tree_case([9, 4], [400, 128 * 40], ratio=128, seed=31)
    dev, paths, ori_scale, cmp_scale, cmp_paths = on_device(made)
    stride = 1 << 20
    for name, table in (("ori", "ori_block_table"), ("cmp", "cmp_block_table")):
        cache, ids = getattr(dev, name), getattr(dev, table)
        far = 5000 + torch.arange(cache.shape[0], device="cuda", dtype=torch.int32)
        big = torch.empty((5000 + cache.shape[0]) * stride, dtype=torch.int8, device="cuda").as_strided((5000 + cache.shape[0], 32, 1, 512), (stride, 512, 512, 1))
        big[5000:] = cache
        setattr(dev, name, big)
        setattr(dev, table, torch.where(ids >= 0, far[ids.clamp_min(0).long()], ids))
    op = PreparedTreeAttention(dev, paths, ori_scale, cmp_scale, cmp_paths=cmp_paths, return_lse=True)
    op.run()
    check(op, made)


@pytest.mark.parametrize("ratio", [1, 4, 128])
def test_odd_metadata(ratio):
    """Tokens in front of the first request, a request without tokens, one with fewer rows than tokens, one
    without rows at all."""
    counts, prefix = [3, 0, 5, 4, 6], [200, 50, -3, -4, 77]
    made = make_tree_case(counts, [max(p, 0) for p in prefix], ratio=ratio, seed=17, topk=20)
    case = made[0]
    case.seq_lens = torch.tensor([p + n for p, n in zip(prefix, counts)], dtype=torch.int32)
    op = prepared(made, return_lse=True)
    op.run()
    torch.cuda.synchronize()
    check(op, made)
    shifted = replace(case, q=torch.cat([case.q[:3], case.q]), cu_q=case.cu_q + 3)
    if case.cmp_indices is not None:
        shifted.cmp_indices = torch.cat([case.cmp_indices[:3], case.cmp_indices])
    front = lambda t: None if t is None else torch.cat([t[:3], t])  # noqa: E731
    later = prepared((shifted, front(made[1]), front(made[2]), *made[3:]), return_lse=True)
    later.run()
    assert torch.equal(later.out[3:], op.out) and later.out[:3].eq(0).all() and torch.equal(later.lse[3:], op.lse) and later.lse[:3].eq(0).all()


@pytest.mark.parametrize("ratio", [1, 4, 128])
def test_empty_rows_and_sinks(ratio):
    """Paths without a bit, tokens without any key, no sink at all."""
    counts, prefix = [4, 3], [0, 40]
    paths = [0, 1, 0, 8, 0, 2, 7]
    sink = torch.linspace(-3, 3, 8)
    sink[1] = sink[5] = -math.inf
    made = make_tree_case(counts, prefix, ratio=ratio, paths=paths, sink=sink, topk=8, seed=5)
    if ratio == 4:
        made[0].cmp_indices[:4] = -1
    if ratio == 128:
        made[2][:4] = 0
    op = prepared(made, return_lse=True)
    op.run()
    torch.cuda.synchronize()
    check(op, made)
    assert op.out[0].eq(0).all() and op.lse[0, 1] == -math.inf


def test_missing_pages():
    """Pages that are gone, outside the cache or beyond the table are no keys."""
    made = make_tree_case([9, 6], [300, 70], ratio=128, seed=3)
    case = made[0]
    case.ori_block_table[0, 7] = -1
    case.ori_block_table[0, 8] = 10 ** 6
    case.cmp_block_table[1, 0] = 1 << 30
    case.seq_lens[1] += 64                      # rows behind the table
    op = prepared(made, return_lse=True)
    op.run()
    torch.cuda.synchronize()
    check(op, made)


def test_values_outside_the_keys_do_not_matter():
    """Codes of rows no token names, and non-finite queries of other tokens, change nothing."""
    made = make_tree_case([5, 9], [90, 200], ratio=128, seed=9)
    first = prepared(made, return_lse=True)
    want = first.run().clone()
    dev, paths, ori_scale, cmp_scale, cmp_paths = on_device(made)
    dev.q = dev.q.clone()
    dev.q[3, 2] = float("nan")
    dev.q[8, 5, 17] = float("inf")
    unused = set(range(dev.ori.shape[0])) - set(made[0].ori_block_table.flatten().tolist())
    dev.ori[list(unused)] = -128
    got = PreparedTreeAttention(dev, paths, ori_scale, cmp_scale, cmp_paths=cmp_paths).run()
    assert got[3, 2].isnan().all() and got[8, 5].isnan().all()
    keep = torch.ones(got.shape[:2], dtype=torch.bool)
    keep[3, 2] = keep[8, 5] = False
    assert torch.equal(got[keep.cuda()], want[keep.cuda()])


def test_logits_beyond_fp32_and_wide_padding():
    """A query whose logits overflow gives NaN, as the formula does; a batch of capacity 700 with three live
    requests gives what the three give alone."""
    made = make_tree_case([4, 9, 2], [300, 90, 128 * 30], ratio=128, seed=21)
    want = prepared(made).run().clone()
    case, paths, cmp_paths, ori_scale, cmp_scale = made
    wide = replace(case, q=case.q.clone(), cu_q=torch.cat([case.cu_q, torch.full((697,), 15, dtype=torch.int32)]),
                   seq_lens=torch.cat([case.seq_lens, torch.zeros(697, dtype=torch.int32)]),
                   ori_block_table=torch.cat([case.ori_block_table, torch.zeros(697, case.ori_block_table.shape[1], dtype=torch.int32)]),
                   cmp_block_table=torch.cat([case.cmp_block_table, torch.zeros(697, case.cmp_block_table.shape[1], dtype=torch.int32)]))
    assert torch.equal(prepared((wide, paths, cmp_paths, ori_scale, cmp_scale)).run(), want)
    wide.q[6, 1] = 3e38
    got = prepared((wide, paths, cmp_paths, ori_scale * 1e6, cmp_scale)).run()
    assert got[6, 1].isnan().all() and torch.isfinite(got[6, 0]).all()


def test_chain_is_the_decode_attention():
    """A draft without branches is what PreparedAttention computes for a run of query tokens."""
    made = make_tree_case([5, 3], [260, 1290], ratio=128, seed=4)
    dev, _, ori_scale, cmp_scale, _ = on_device(made)
    chain = torch.cat([path_masks(range(-1, n - 1)) for n in (5, 3)]).cuda()
    tree = PreparedTreeAttention(dev, chain, ori_scale, cmp_scale, return_lse=True)
    run = PreparedAttention(dev, ori_scale, cmp_scale, return_lse=True)
    tree.run(), run.run()
    torch.testing.assert_close(tree.out.float(), run.out.float(), rtol=0.008, atol=0.0006)
    torch.testing.assert_close(tree.lse, run.lse, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("ratio", [4, 128])
def test_captured_replays_follow_the_inputs(ratio):
    """A captured launch reads lengths, masks and lists anew; a second stream and operator run beside it."""
    made = [make_tree_case([6, 9, 2], [128 * 20, 900, 40], ratio=ratio, topk=100, seed=s) for s in (1, 2)]
    made.append(make_tree_case([3, 12, 2], [128 * 20 + 3, 600, 40], ratio=ratio, topk=100, seed=1))
    case = made[2][0]
    case.ori, case.ori_block_table, case.cmp, case.cmp_block_table = (getattr(made[0][0], n) for n in
                                                                      ("ori", "ori_block_table", "cmp", "cmp_block_table"))
    made[2] = (case, made[2][1], made[2][2], made[0][3], made[0][4])
    op, other = prepared(made[0], return_lse=True), prepared(made[1], return_lse=True)
    op.run(), other.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.run()
        op.run()
    side = torch.cuda.Stream()
    for round_, which in enumerate((0, 2, 0)):
        source = made[which]
        for name in ("q", "cu_q", "seq_lens", "cmp_indices"):
            if getattr(source[0], name) is not None:
                getattr(op.case, name).copy_(getattr(source[0], name))
        op.paths.copy_(source[1])
        if op.cmp_paths is not None:
            op.cmp_paths.copy_(source[2])
        torch.cuda.synchronize()
        op.out.fill_(float("nan"))
        graph.replay()
        with torch.cuda.stream(side):
            other.run()
        torch.cuda.synchronize()
        check(op, source, round_)
        check(other, made[1], round_)


def test_results_do_not_depend_on_the_launch():
    made = make_tree_case([64, 40, 17, 1], [128 * 90, 5000, 128 * 300, 12], ratio=128, seed=11)
    op = prepared(made, return_lse=True)
    first, lse = op.run().clone(), op.lse.clone()
    for _ in range(5):
        op.run()
        assert torch.equal(op.out, first) and torch.equal(op.lse, lse)


def test_no_tokens_and_no_requests():
    made = make_tree_case([2], [10])
    dev, paths, ori_scale, _, _ = on_device(made)
    case = replace(dev, q=dev.q[:0])
    assert PreparedTreeAttention(case, paths[:0], ori_scale).run().shape == (0, 8, 512)
    case = replace(dev, cu_q=dev.cu_q[:1], seq_lens=dev.seq_lens[:0], ori_block_table=dev.ori_block_table[:0])
    op = PreparedTreeAttention(case, paths, ori_scale, return_lse=True, output=torch.full_like(dev.q, 7))
    op.run()
    assert op.out.eq(0).all() and op.lse.eq(0).all()


def test_layer_runtime_route(tmp_path, monkeypatch):
    """The serving adapter: frozen scales by layer name, operators kept by geometry, other tensors per call."""
    made = [make_tree_case([6, 9], [700, 130], ratio=128, seed=s) for s in (1, 2)]
    scales = dict(zip(("model.layers.3.attn.ori", "model.layers.3.attn.cmp"), made[0][3:5]))
    torch.save({"protocol": "sharedkv-c8-v1", "scales": scales}, tmp_path / "scales.pt")
    monkeypatch.setenv("SHAREDKV_SCALES", str(tmp_path / "scales.pt"))
    vllm_adapter.load_scales.cache_clear()
    impl = SimpleNamespace(head_dim=512, swa_cache_layer=SimpleNamespace(prefix="model.layers.3.attn.swa_cache"))
    layer = vllm_adapter.runtime(impl)
    for which in (0, 1, 0):
        case, paths, cmp_paths = made[which][:3]
        dev = case.to("cuda")
        out, lse = layer.tree_attention(
            dev.q, paths.cuda(), cmp_paths=cmp_paths.cuda(), layout_q="TND", layout_kv="PA_ND", ori_kv=dev.ori, ori_block_table=dev.ori_block_table,
            cu_seqlens_q=dev.cu_q, seqused_kv=dev.seq_lens, sinks=dev.sink, cmp_kv=dev.cmp, cmp_block_table=dev.cmp_block_table, cmp_ratio=128,
            ori_win_left=127, softmax_scale=dev.softmax_scale, return_softmax_lse=True)
        source = (case, paths, cmp_paths, *made[0][3:5])
        want, want_lse, bound, lse_bound = expected(*source)
        assert ((out.cpu().double() - want).abs() - bound).max() <= 0
        assert ((lse[..., 0].cpu().double() - want_lse).abs() - lse_bound).max() <= 0
    assert len(layer.tree_ops) <= 2
    vllm_adapter.load_scales.cache_clear()


@pytest.mark.parametrize("change, text", [
    (dict(paths=torch.int32), "INT64 paths"), (dict(heads=12), "multiple of eight"), (dict(window=70000), "window"),
    (dict(cmp_paths=True), "ratio-128"), (dict(page=16), "32-row pages"), (dict(lse=True), "LSE"), (dict(offset=8), "16-byte")])
def test_refusals(change, text):
    made = make_tree_case([2, 2], [10, 40], heads=change.get("heads", 8))
    dev, paths, ori_scale, _, _ = on_device(made, 16384 + 512 if "offset" in change else None, change.get("offset", 0))
    dev.window = change.get("window", 128)
    more = {}
    if "paths" in change:
        paths = paths.to(change["paths"])
    if "cmp_paths" in change:
        more["cmp_paths"] = paths
    if "page" in change:
        dev.ori = dev.ori[:, :16]
    if "lse" in change:
        more["lse_output"] = torch.empty(3, 8, device="cuda")
    with pytest.raises(ValueError, match=text):
        PreparedTreeAttention(dev, paths, ori_scale, **more)
