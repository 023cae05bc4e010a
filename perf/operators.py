"""Workloads of the drafted-tree and page operators, with their plain forms.

`listed()` and `draw()` give cases, `prepare()` a program's state for one, `run()` one pass through the
operator: as elementary torch operations, or, where `own` is set, through the framework's own calls.

  tree    attention of a tree of drafted tokens over the INT8 shared-KV cache (PreparedTreeAttention)
  copy    pages copied inside every cache of a pool                           (PagePool.copy)
  fork    sequences that continue other sequences: a beam step                (PagePool.fork)
  resize  room for drafted rows, then the rejected ones given back            (PagePool.resize)
  keep    the accepted rows of a drafted tree packed behind the committed     (PagePool.keep)
"""
import math
import os
import random
import statistics
import sys

import torch

own = False

DIM = 512            # channels of a cache row
PAGE = 32            # rows of a page
DRAFT = 64           # drafted rows a path mask can name


def listed():
    return [
        # one user, a short draft of a C128 layer: what a single verification step waits for
        dict(name="tree c128, one request", op="tree", ratio=128, batch=1, nodes=8, ragged=False, shortest=6000, longest=8000,
             heads=8, window=128, topk=0, stride=16384),
        # a sliding-window layer under a ragged batch: some requests have just begun, some draft one token
        dict(name="tree window, ragged", op="tree", ratio=1, batch=48, nodes=63, ragged=True, shortest=1, longest=4096,
             heads=16, window=128, topk=0, stride=17408),
        # a C4 layer: every drafted token brings its own top-k list, lists of one tree overlap
        dict(name="tree c4, batch", op="tree", ratio=4, batch=16, nodes=32, ragged=False, shortest=16384, longest=65536,
             heads=8, window=128, topk=1024, stride=16384),
        # a full serving batch with long contexts on a C128 layer
        dict(name="tree c128, batch", op="tree", ratio=128, batch=64, nodes=64, ragged=False, shortest=32768, longest=524288,
             heads=8, window=128, topk=0, stride=622592),
        # one page of two layers: the latency of a single copy
        dict(name="copy, one page", op="copy", layers=2, pages=512, pairs=1, stride=16384),
        # a prefix duplicated for a batch of sequences in every layer
        dict(name="copy, many pages", op="copy", layers=16, pages=4096, pairs=700, stride=16384),
        # one request, four beams
        dict(name="fork, one request", op="fork", layers=2, pages=1024, requests=1, beams=4, shortest=300, longest=2000, width=128, stride=16384),
        # a beam step of a serving batch
        dict(name="fork, batch", op="fork", layers=8, pages=32768, requests=128, beams=4, shortest=500, longest=8000, width=320, stride=16384),
        # one sequence makes room for its draft
        dict(name="resize, one sequence", op="resize", layers=2, pages=512, batch=1, nodes=63, shortest=1000, longest=3000, width=128, stride=16384),
        # a draft step of a batch: fresh pages for the drafted rows of every sequence, then most of them back
        dict(name="resize, batch", op="resize", layers=2, pages=32768, batch=512, nodes=63, shortest=33, longest=4000, width=256, stride=17408),
        # one verified tree in two layers
        dict(name="keep, one tree", op="keep", layers=2, pages=128, batch=1, kept=5, nodes=31, shortest=500, longest=3000, stride=16384),
        # a batch of verified trees in all the layers that share a block table
        dict(name="keep, batch of trees", op="keep", layers=24, pages=4096, batch=256, kept=17, nodes=64, shortest=1, longest=400, stride=16384),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "copy", "fork", "resize", "keep"])
    if op == "tree":
        ratio = rng.choice([1, 4, 128])
        nodes = _spread(rng, 1, 64)
        batch = _spread(rng, 1, 48 if ratio != 4 else 16)
        longest = _spread(rng, 64, {1: 65536, 4: 65536, 128: 200000}[ratio])
        return dict(op=op, ratio=ratio, batch=batch, nodes=nodes, ragged=rng.random() < 0.5, shortest=_spread(rng, 1, longest), longest=longest,
                    heads=rng.choice([8, 8, 16, 32]) if batch * nodes <= 256 else 8, window=rng.choice([128, 128, 64, 200]),
                    topk=rng.choice([1024, 512, _spread(rng, 5, 1000)]) if ratio == 4 else 0, stride=rng.choice([16384, 17408, 16400, 32768]))
    layers, stride = _spread(rng, 1, 12), rng.choice([16384, 17408, 16400])
    if op == "copy":
        return dict(op=op, layers=layers, pages=4096, pairs=_spread(rng, 1, 600), stride=stride)
    if op == "fork":
        requests, beams = _spread(rng, 1, 100), rng.choice([2, 3, 4, 5, 8])
        longest = _spread(rng, 40, 1500)
        return dict(op=op, layers=min(layers, 6), pages=requests * beams * (longest // PAGE + 4) + 64, requests=requests, beams=beams,
                    shortest=_spread(rng, 1, longest), longest=longest, width=longest // PAGE + rng.randint(2, 90), stride=stride)
    if op == "resize":
        batch, longest = _spread(rng, 1, 400), _spread(rng, 40, 2000)
        return dict(op=op, layers=min(layers, 4), pages=batch * (longest // PAGE + 6) + 64, batch=batch, nodes=rng.randint(1, 64),
                    shortest=_spread(rng, 1, longest), longest=longest, width=longest // PAGE + rng.randint(4, 90), stride=stride)
    nodes = rng.randint(1, 64)
    return dict(op=op, layers=layers, pages=4096, batch=_spread(rng, 1, 250), kept=rng.randint(1, min(nodes, 20)), nodes=nodes,
                shortest=1, longest=_spread(rng, 30, 400), stride=stride)


# ------------------------------------------------------------------ states

def _lengths(rng, case, count):
    low, high = math.log(case["shortest"]), math.log(case["longest"])
    return [max(1, int(round(math.exp(rng.uniform(low, high))))) for _ in range(count)]


def _pages(gen, count, stride):
    """INT8 pages [count, 32, 1, 512], `stride` bytes apart, filled as a calibrated cache is: codes of
    normal values whose scale puts four deviations at 127."""
    raw = torch.empty(count * stride, dtype=torch.int8, device="cuda")
    for first in range(0, raw.numel(), 1 << 28):
        part = raw[first:first + (1 << 28)]
        part.copy_((torch.randn(part.numel(), generator=gen, device="cuda") * 32).round_().clamp_(-127, 127))
    return raw.as_strided((count, PAGE, 1, DIM), (stride, DIM, DIM, 1))


def _layers(gen, case):
    """Pages [layers, pages, 32, 1, 512] of arbitrary codes, for operators that only move them; a pool
    has one cache per layer."""
    layers, count, stride = case["layers"], case["pages"], case["stride"]
    raw = torch.randint(-2 ** 62, 2 ** 62, (layers * count * stride // 8,), dtype=torch.int64, generator=gen, device="cuda").view(torch.int8)
    stack = raw.as_strided((layers, count, PAGE, 1, DIM), (count * stride, stride, DIM, DIM, 1))
    return dict(stack=stack, caches=list(stack.unbind(0)))


def _signed(mask):
    return mask - (1 << 64) if mask >> 63 else mask


def _trees(rng, counts):
    """Random drafts: per token the path mask (itself and its ancestors), and the parents."""
    paths = []
    for n in counts:
        masks = []
        for i in range(n):
            parent = rng.randint(-1, i - 1) if i and rng.random() < 0.6 else i - 1
            masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
        paths.append(masks)
    return paths


def _group_rows(paths, prefix, ratio):
    """Per token a mask of the drafted compressed rows on its path: row e belongs to the e-th drafted
    token whose path ends at a group boundary."""
    ends = [i for i, mask in enumerate(paths) if (prefix + mask.bit_count()) % ratio == 0]
    return [sum(1 << e for e, i in enumerate(ends) if mask >> i & 1) for mask in paths]


def _prepare_tree(case, seed):
    rng = random.Random(seed * 7919 + 1)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    batch, ratio, heads, window = case["batch"], case["ratio"], case["heads"], case["window"]
    ragged = random.Random(batch * 64 + case["nodes"])                           # how many tokens a request drafts belongs to the case
    counts = [ragged.randint(1, case["nodes"]) if case["ragged"] else case["nodes"] for _ in range(batch)]
    prefix = _lengths(rng, case, batch)
    paths = _trees(rng, counts)
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    tokens = cu[-1]

    def table_of(rows_from, rows_to):
        """Pages for rows [from, to) of each request in a shuffled pool; older pages are gone (-1)."""
        width = max(1, max(-(-r // PAGE) for r in rows_to))
        table = torch.full((batch, width), -1, dtype=torch.int32)
        spans = [(f // PAGE, max(f // PAGE + 1, -(-t // PAGE))) for f, t in zip(rows_from, rows_to)]
        total = sum(b - a for a, b in spans)
        order = list(range(total))
        rng.shuffle(order)
        order = torch.tensor(order, dtype=torch.int32)
        at = 0
        for b, (first, last) in enumerate(spans):
            table[b, first:last] = order[at:at + last - first]
            at += last - first
        return table.cuda(), total

    s = dict(op="tree", counts=counts, most=max(counts), ratio=ratio, window=window, softmax_scale=1 / math.sqrt(DIM))
    s["ori_table"], pages = table_of([max(0, p - window) for p in prefix], [p + n for p, n in zip(prefix, counts)])
    s["ori"] = _pages(gen, pages, case["stride"])
    scale = lambda: (torch.randn(DIM, generator=gen, device="cuda") * 0.3).exp() * (4 / 127)  # noqa: E731
    s["ori_scale"], s["cmp_scale"] = scale(), scale()
    s["q"] = torch.randn(tokens, heads, DIM, generator=gen, device="cuda").to(torch.bfloat16)
    s["sink"] = torch.linspace(-2, 2, heads, device="cuda")
    s["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    s["seq"] = torch.tensor([p + n for p, n in zip(prefix, counts)], dtype=torch.int32, device="cuda")
    s["paths"] = torch.tensor([_signed(m) for masks in paths for m in masks], dtype=torch.int64, device="cuda")
    s["cmp"] = s["cmp_table"] = s["cmp_paths"] = s["picks"] = None
    if ratio > 1:
        whole = [p // ratio for p in prefix]
        drafted = [_group_rows(masks, p, ratio) for masks, p in zip(paths, prefix)]
        s["most_compressed"] = max(whole) + DRAFT
        s["cmp_table"], pages = table_of([0] * batch, [w + DRAFT for w in whole])
        s["cmp"] = _pages(gen, pages, case["stride"])
    if ratio == 128:
        s["cmp_paths"] = torch.tensor([_signed(m) for masks in drafted for m in masks], dtype=torch.int64, device="cuda")
    if ratio == 4:
        # the tokens of a tree score the rows alike, not the same: a shared score and each token's own
        picks = torch.full((tokens, 1, case["topk"]), -1, dtype=torch.int32, device="cuda")
        for b, (n, rows) in enumerate(zip(counts, whole)):
            score = torch.randn(rows, generator=gen, device="cuda") + 0.5 * torch.randn(n, rows, generator=gen, device="cuda")
            best = score.topk(min(case["topk"], rows)).indices
            picks[cu[b]:cu[b + 1], 0, :best.shape[1]] = best.to(torch.int32)
        own_rows = [(t, k, rows + e) for b, rows in enumerate(whole) for t, mask in enumerate(drafted[b], cu[b])
                    for k, e in enumerate(e for e in range(DRAFT) if mask >> e & 1) if k < case["topk"]]
        if own_rows:
            t, k, row = (torch.tensor(v, device="cuda") for v in zip(*own_rows))
            picks[t, 0, case["topk"] - 1 - k] = row.to(torch.int32)
        s["picks"] = picks
    return s


def _prepare_copy(case, seed):
    rng = random.Random(seed * 7919 + 2)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    order = rng.sample(range(case["pages"]), 2 * case["pairs"])
    sources = order[:case["pairs"]]
    sources[: case["pairs"] // 4] = [sources[-1]] * (case["pairs"] // 4)         # some pages are copied more than once
    pairs = torch.tensor(list(zip(sources, order[case["pairs"]:])), dtype=torch.int32, device="cuda")
    return dict(_layers(gen, case), op="copy", pairs=pairs)


def _pool(rng, gen, case, lens, groups):
    """Pages dealt at random to sequences of `lens` rows; the sequences of a group share the full pages
    of their common beginning."""
    rows, width = len(lens), case["width"]
    order = list(range(case["pages"]))
    rng.shuffle(order)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    at = 0
    for members in groups:
        common = min(lens[b] for b in members) // PAGE if len(members) > 1 else 0
        shared = order[at:at + common]
        at += common
        for b in members:
            mine = -(-lens[b] // PAGE) - common
            table[b, :common + mine] = torch.tensor(shared + order[at:at + mine], dtype=torch.int32)
            at += mine
    live = torch.arange(width)[None] < -(-torch.tensor(lens)[:, None] // PAGE)
    refs = torch.bincount(table[live].long(), minlength=case["pages"]).to(torch.int32)
    return dict(_layers(gen, case), table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), refs=refs.cuda())


def _prepare_fork(case, seed):
    rng = random.Random(seed * 7919 + 3)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens, groups, parents = [], [], []
    for length in _lengths(rng, case, case["requests"]):
        first = len(lens)
        groups.append(range(first, first + case["beams"]))
        lens += [length] * case["beams"]                                         # the beams of a request are equally long
        parents += sorted(rng.randrange(first, first + case["beams"]) for _ in range(case["beams"]))
    s = _pool(rng, gen, case, lens, groups)
    return dict(s, op="fork", parents=torch.tensor(parents, dtype=torch.int32, device="cuda"))


def _prepare_resize(case, seed):
    rng = random.Random(seed * 7919 + 4)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens = _lengths(rng, case, case["batch"])
    s = _pool(rng, gen, case, lens, [range(b, min(b + 2, len(lens))) for b in range(0, len(lens), 2)])
    grown = torch.tensor([n + rng.randint(1, case["nodes"]) for n in lens], dtype=torch.int32, device="cuda")
    return dict(s, op="resize", grown=grown, back=s["lens"].clone())


def _prepare_keep(case, seed):
    rng = random.Random(seed * 7919 + 5)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    base = _lengths(rng, case, case["batch"])
    width = max(-(-(b + case["nodes"]) // PAGE) for b in base)
    order = rng.sample(range(case["pages"]), min(case["pages"], case["batch"] * width))
    table = torch.full((case["batch"], width), -1, dtype=torch.int32)
    kept = torch.full((case["batch"], case["kept"]), -1, dtype=torch.int32)
    at = 0
    for b, rows in enumerate(base):
        first, last = rows // PAGE, -(-(rows + case["nodes"]) // PAGE)           # only the pages that hold drafted rows matter
        table[b, first:last] = torch.tensor(order[at:at + last - first], dtype=torch.int32)
        at += last - first
        chosen = sorted(rng.sample(range(case["nodes"]), rng.randint(1, case["kept"])))
        kept[b, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return dict(_layers(gen, case), op="keep", table=table.cuda(), base=torch.tensor(base, dtype=torch.int32, device="cuda"), kept=kept.cuda())


def _framework():
    root = os.path.join(os.getcwd(), "ascend-int8-attention_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import npu_sparse_attn_sharedkv_int8 as package
    return package


def prepare(case, seed):
    s = {"tree": _prepare_tree, "copy": _prepare_copy, "fork": _prepare_fork, "resize": _prepare_resize,
         "keep": _prepare_keep}[case["op"]](case, seed)
    if not own:
        return s
    # what a serving program keeps between calls: prepared operators with their workspaces
    package = _framework()
    if s["op"] == "tree":
        from npu_sparse_attn_sharedkv_int8.reference import SharedKVCase
        data = SharedKVCase(q=s["q"], ori=s["ori"], ori_block_table=s["ori_table"], cu_q=s["cu"], seq_lens=s["seq"], sink=s["sink"],
                            cmp=s["cmp"], cmp_block_table=s["cmp_table"], cmp_indices=s["picks"], ratio=s["ratio"], window=s["window"],
                            softmax_scale=s["softmax_scale"])
        s["operator"] = package.PreparedTreeAttention(data, s["paths"], s["ori_scale"], s["cmp_scale"] if s["ratio"] > 1 else None,
                                                      cmp_paths=s["cmp_paths"])
    elif s["op"] in ("copy", "keep"):
        s["pool"] = package.PagePool(s["caches"], s.get("table"))
    else:
        s["pool"] = package.PagePool(s["caches"], s["table"], s["lens"], s["refs"])
    return s


# ------------------------------------------------------------------ plain forms

def _rows(cache, table, scale, rows):
    """Dequantised rows [B, L, 512] for logical rows [B, L], and which of them exist."""
    page = (rows // PAGE).clamp(0, table.shape[1] - 1)
    ids = table.gather(1, page).long()
    there = (rows >= 0) & (rows // PAGE < table.shape[1]) & (ids >= 0) & (ids < cache.shape[0])
    return cache[ids.clamp_min(0), (rows % PAGE), 0].float() * scale, there


def _bits(masks, count):
    return (masks[..., None] >> torch.arange(count, device=masks.device)) & 1 != 0


def _plain_tree(s):
    q, cu, window = s["q"], s["cu"].long(), s["window"]
    tokens, heads, _ = q.shape
    n = cu[1:] - cu[:-1]
    prefix = s["seq"].long() - n
    at = torch.arange(s["most"], device=q.device)
    live = at < n[:, None]                                                       # [B, N]
    token = (cu[:-1, None] + at).clamp_max(tokens - 1)
    qf = q.float()[token]                                                        # [B, N, H, 512]
    mine = _bits(s["paths"][token], DRAFT) & (torch.arange(DRAFT, device=q.device) < n[:, None, None])
    length = mine.sum(-1)                                                        # rows of the path

    back = torch.arange(window, device=q.device)                                 # committed rows of the window
    rows = torch.cat([prefix[:, None] - window + back, prefix[:, None] + torch.arange(DRAFT, device=q.device)], 1)
    kv, there = _rows(s["ori"], s["ori_table"], s["ori_scale"], rows)
    seen = torch.cat([(back >= length[..., None]), mine], 2) & there[:, None]
    score = torch.einsum("bnhd,bld->bnhl", qf, kv) * s["softmax_scale"]
    score = score.masked_fill(~seen[:, :, None], -math.inf)
    parts, values = [score], [kv]
    if s["ratio"] == 128:
        whole = prefix.clamp_min(0) // 128
        rows = torch.arange(s["most_compressed"], device=q.device).expand(len(n), -1)
        kc, there = _rows(s["cmp"], s["cmp_table"], s["cmp_scale"], rows)
        drafted = rows - whole[:, None]
        named = (s["cmp_paths"][token][..., None] >> drafted.clamp(0, DRAFT - 1)[:, None]) & 1 != 0
        seen = there[:, None] & ((drafted < 0)[:, None] | (named & (drafted >= 0)[:, None] & (drafted < DRAFT)[:, None]))
        score = torch.einsum("bnhd,bld->bnhl", qf, kc) * s["softmax_scale"]
        parts.append(score.masked_fill(~seen[:, :, None], -math.inf))
        values.append(kc)
    score = torch.cat(parts, -1)[live]                                           # [T, H, L]
    out_rows = token[live]
    if s["ratio"] == 4:
        owner = torch.arange(len(n), device=q.device)[:, None].expand(-1, s["most"])[live]
        picks = s["picks"][out_rows, 0].long()
        kc, there = _rows(s["cmp"], s["cmp_table"][owner], s["cmp_scale"], picks)
        there &= picks < (prefix[owner, None].clamp_min(0) // 4 + DRAFT)
        own_score = torch.einsum("thd,tkd->thk", q.float()[out_rows], kc) * s["softmax_scale"]
        score = torch.cat([score, own_score.masked_fill(~there[:, None], -math.inf)], -1)
    sink = s["sink"][None, :, None].expand(score.shape[0], -1, -1)
    top = torch.maximum(score.amax(-1, keepdim=True), sink)
    weight = (score - top).exp()
    total = weight.sum(-1, keepdim=True) + (sink - top).exp()
    split = weight.split([v.shape[1] for v in values] + ([kc.shape[1]] if s["ratio"] == 4 else []), -1)
    result = 0
    spread = torch.zeros(len(n), s["most"], heads, 1, device=q.device)
    for part, v in zip(split, values):
        dense = spread.expand(-1, -1, -1, v.shape[1]).clone()
        dense[live] = part
        result = result + torch.einsum("bnhl,bld->bnhd", dense, v)[live]
    if s["ratio"] == 4:
        result = result + torch.einsum("thk,tkd->thd", split[-1], kc)
    out = torch.zeros_like(q)
    out[out_rows] = (result / total).to(torch.bfloat16)
    return out


def _copy_pages(stack, sources, targets):
    stack[:, targets] = stack[:, sources]


def _live(lens):
    return (lens.long() + PAGE - 1) // PAGE


def _plain_copy(s):
    _copy_pages(s["stack"], s["pairs"][:, 0].long(), s["pairs"][:, 1].long())
    return s["stack"]


def _plain_fork(s):
    table, lens, refs, parents = s["table"], s["lens"], s["refs"], s["parents"].long()
    rows, width = table.shape
    at = torch.arange(width, device=table.device)
    index = torch.arange(rows, device=table.device)
    goes_on = parents >= 0
    children = torch.zeros(rows, dtype=torch.int64, device=table.device).index_add_(0, parents.clamp_min(0), goes_on.long())
    first = torch.full((rows,), rows, device=table.device).scatter_reduce_(0, parents.clamp_min(0), torch.where(goes_on, index, rows), "amin")
    full, live = lens.long() // PAGE, _live(lens)
    change = torch.where(at < full[:, None], children[:, None] - 1, torch.where(children[:, None] == 0, -1, 0))
    inside = at < live[:, None]
    after = refs.clone().index_add_(0, table[inside].long(), change[inside].to(torch.int32))
    of = parents.clamp_min(0)
    copies = goes_on & (first[of] != index) & (lens[of] % PAGE != 0)
    fresh = (after == 0).nonzero()[:, 0][: int(copies.sum())]
    taken = table[of]
    last = full[of].clamp_max(width - 1)
    sources = taken.gather(1, last[:, None])[copies, 0].long()
    _copy_pages(s["stack"], sources, fresh)
    taken[copies, last[copies]] = fresh.to(torch.int32)
    after[fresh] = 1
    refs.copy_(after)
    lens.copy_(torch.where(goes_on, lens[of], 0))
    table.copy_(torch.where(at < _live(lens)[:, None], taken, table))
    return [table, lens, refs, s["stack"]]


def _plain_resize(s, wanted):
    table, lens, refs = s["table"], s["lens"], s["refs"]
    width = table.shape[1]
    at = torch.arange(width, device=table.device)
    before, after = _live(lens), _live(wanted)
    gone = (at >= after[:, None]) & (at < before[:, None])
    refs.index_add_(0, table[gone].long(), torch.full((1,), -1, dtype=torch.int32, device=table.device).expand(int(gone.sum())))
    last = (before - 1).clamp_min(0)
    ends = table.gather(1, last[:, None])[:, 0].long()
    split = (wanted > lens) & (lens % PAGE != 0) & (refs[ends.clamp_min(0)] > 1)
    need = ((at >= before[:, None]) & (at < after[:, None])) | ((at == last[:, None]) & split[:, None])
    fresh = (refs == 0).nonzero()[:, 0][: int(need.sum())]
    refs.index_add_(0, ends[split], torch.full((1,), -1, dtype=torch.int32, device=table.device).expand(int(split.sum())))
    table[need] = fresh.to(torch.int32)                                          # in (sequence, page) order
    refs[fresh] = 1
    _copy_pages(s["stack"], ends[split], table.gather(1, last[:, None])[split, 0].long())
    lens.copy_(wanted)


def _plain_keep(s):
    table, base, kept = s["table"], s["base"].long()[:, None], s["kept"].long()
    to = base + torch.arange(kept.shape[1], device=kept.device)
    source = base + kept.clamp_min(0)
    moves = kept >= 0
    page = lambda rows: table.gather(1, rows // PAGE).long()[moves]  # noqa: E731
    from_page, to_page = page(source), page(to.clamp_max(table.shape[1] * PAGE - 1))
    s["stack"][:, to_page, (to % PAGE)[moves]] = s["stack"][:, from_page, (source % PAGE)[moves]]
    return s["stack"]


def run(s):
    if own:
        if s["op"] == "tree":
            return s["operator"].run()
        pool = s["pool"]
        if s["op"] == "copy":
            pool.copy(s["pairs"])
            return s["stack"]
        if s["op"] == "keep":
            pool.keep(s["base"], s["kept"])
            return s["stack"]
        if s["op"] == "fork":
            pool.fork(s["parents"])
        else:
            pool.resize(s["grown"])
            pool.resize(s["back"])
        return [s["table"], s["lens"], s["refs"], s["stack"]]
    if s["op"] == "tree":
        return _plain_tree(s)
    if s["op"] == "copy":
        return _plain_copy(s)
    if s["op"] == "keep":
        return _plain_keep(s)
    if s["op"] == "fork":
        return _plain_fork(s)
    _plain_resize(s, s["grown"])
    _plain_resize(s, s["back"])
    return [s["table"], s["lens"], s["refs"], s["stack"]]


# ------------------------------------------------------------------ floors

def _mean_length(case):
    low, high = case["shortest"], case["longest"]
    return float(low) if low == high else (high - low) / math.log(high / low)


def _union(rows, picks, tokens):
    """Expected number of rows that at least one of `tokens` lists names, for scores as _prepare_tree makes them."""
    if picks >= rows:
        return rows
    normal = statistics.NormalDist()
    border = math.sqrt(1.25) * normal.inv_cdf(1 - picks / rows)
    steps = [normal.inv_cdf((i + 0.5) / 400) for i in range(400)]
    return rows * sum(1 - normal.cdf((border - z) / 0.5) ** tokens for z in steps) / 400


def work(case):
    row, layers = DIM, case.get("layers", 1)
    if case["op"] == "tree":
        nodes = (1 + case["nodes"]) / 2 if case["ragged"] else case["nodes"]
        tokens, prefix = case["batch"] * nodes, _mean_length(case)
        near = min(prefix, case["window"])
        keys, rows = near, near + nodes
        if case["ratio"] == 128:
            keys, rows = keys + prefix / 128, rows + prefix / 128
        if case["ratio"] == 4:
            whole = prefix / 4
            keys, rows = keys + min(case["topk"], whole), rows + _union(whole, min(case["topk"], whole), nodes)
        return dict(bytes=case["batch"] * rows * row + tokens * (case["heads"] * DIM * 4 + 8 + case["topk"] * 4),
                    flops=tokens * case["heads"] * keys * DIM * 4)
    page = PAGE * row
    if case["op"] == "copy":
        return dict(bytes=(case["pairs"] - case["pairs"] // 4 + case["pairs"]) * layers * page + case["pairs"] * 8, flops=0)
    if case["op"] == "keep":
        return dict(bytes=case["batch"] * (case["kept"] + 1) / 2 * layers * 2 * row, flops=0)
    pages = _mean_length(case) / PAGE
    if case["op"] == "fork":
        beams = case["beams"]
        distinct = beams * (1 - (1 - 1 / beams) ** beams)
        copies = case["requests"] * (beams - distinct)
        return dict(bytes=copies * 2 * page * layers + case["requests"] * beams * pages * 8 + case["pages"] * 4, flops=0)
    grown = case["batch"] * (case["nodes"] / 2 / PAGE)
    return dict(bytes=2 * (grown * 8 + case["batch"] * 8 + case["pages"] * 4), flops=0)


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    """Tree attention request by request in float64.  The page operators move codes and page numbers:
    nothing they return is a computed value."""
    if case["op"] != "tree":
        return None
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    q = s["q"].double()
    out = torch.zeros_like(q)
    prefix = [int(v) - n for v, n in zip(s["seq"].tolist(), s["counts"])]

    def fetch(cache, table_row, scale, rows):
        rows = torch.as_tensor(rows, device=q.device, dtype=torch.int64)
        pages = table_row[rows // PAGE].long()
        return cache[pages, rows % PAGE, 0].double() * scale.double()

    first = 0
    for b, n in enumerate(s["counts"]):
        start = max(0, prefix[b] - s["window"])
        whole = prefix[b] // s["ratio"]
        near = fetch(s["ori"], s["ori_table"][b], s["ori_scale"], range(start, prefix[b] + n))
        far = fetch(s["cmp"], s["cmp_table"][b], s["cmp_scale"], range(whole + DRAFT)) if s["ratio"] > 1 else None
        paths = [v & (1 << 64) - 1 for v in s["paths"][first:first + n].tolist()]
        extra = [v & (1 << 64) - 1 for v in s["cmp_paths"][first:first + n].tolist()] if s["ratio"] == 128 else None
        mask = torch.zeros(n, near.shape[0], dtype=torch.float64)
        for i, path in enumerate(paths):
            mask[i, max(start, prefix[b] - s["window"] + path.bit_count()) - start:prefix[b] - start] = 1
            for j in range(n):
                mask[i, prefix[b] - start + j] = path >> j & 1
        weight, keys = mask.to(q.device), near
        if s["ratio"] == 128:
            tail = torch.tensor([[float(m >> e & 1) for e in range(DRAFT)] for m in extra], dtype=torch.float64, device=q.device)
            weight = torch.cat([weight, torch.ones(n, whole, dtype=torch.float64, device=q.device), tail], 1)
            keys = torch.cat([near, far])
        elif s["ratio"] == 4:
            picks = s["picks"][first:first + n, 0].long()
            good = (picks >= 0) & (picks < whole + DRAFT)
            count = torch.zeros(n, whole + DRAFT, dtype=torch.float64, device=q.device)
            count.scatter_add_(1, picks.clamp(0, whole + DRAFT - 1), good.double())
            weight, keys = torch.cat([weight, count], 1), torch.cat([near, far])
        score = torch.einsum("nhd,ld->nhl", q[first:first + n], keys) * s["softmax_scale"]
        sink = s["sink"].double()[None, :, None]
        top = torch.maximum(score.masked_fill(weight[:, None] == 0, -math.inf).amax(-1, keepdim=True), sink)
        p = (score - top).clamp_max(0).exp() * weight[:, None]
        out[first:first + n] = torch.einsum("nhl,ld->nhd", p, keys) / (p.sum(-1, keepdim=True) + (sink - top).exp())
        first += n
    return out
