"""Drafted-tree cases and their attention from the definition, in float64, with the error bounds the
tests hold the kernel to.

The kernel's arithmetic errors, for one query row (A = largest |q_c scale_c|, codes k, weights
w = e^(s - max s), n keys):
  query codes      two INT8 planes: |dq_c| <= A / (2 * 127 * 254), so |ds| <= Es = softmax_scale * A / 64516 * max_k sum_c |code|
                   and a weight is off by a factor of at most e^(2 Es) once the maximum moves with it;
  weight codes     steps of 8 / 32639 of the largest weight, the 8 because the reference point may stand
                   three powers of two above the largest logit; rounded to nearest: |dw| <= Ew = 4 / 32639;
  output           dw moves numerator and denominator: |dy| <= (sum dw |v| + |y| sum dw) / sum w, then one
                   rounding to BF16, half a step: 2^-8 |y|; FP32 sums of the integer products add 2^-20 relative;
  LSE              Es + n Ew / sum w, and 2^-20 of its magnitude in FP32.
"""
import math
import random

import torch

from npu_sparse_attn_sharedkv_int8.reference import SharedKVCase

DRAFT = 64
BF16_HALF_STEP = 2.0 ** -8


def signed(mask):
    return mask - (1 << 64) if mask >> 63 else mask


def random_paths(rng, n):
    masks = []
    for i in range(min(n, DRAFT)):
        parent = rng.randint(-1, i - 1) if i and rng.random() < 0.6 else i - 1
        masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
    return masks + [masks[rng.randrange(len(masks))] for _ in range(n - len(masks))]


def make_tree_case(counts, prefix, *, ratio=1, heads=8, window=128, topk=64, seed=0, paths=None, sink=None, pad=0, spread=1.0):
    """(case, paths, cmp_paths, ori_scale, cmp_scale) on the host; `pad` requests and tokens of padding."""
    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    batch, live = len(counts), sum(counts)
    tokens = live + 3 * pad
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    masks = paths if paths is not None else [m for n in counts for m in random_paths(rng, n)]
    masks = masks + [(1 << 64) - 1] * (tokens - live)

    def pool(rows):
        width = max(1, -(-max(rows) // 32))
        need = [max(1, -(-r // 32)) for r in rows]
        order = torch.randperm(sum(need) + 2, generator=gen).to(torch.int32)
        table = torch.full((batch + pad, width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        codes = (torch.randn(sum(need) + 2, 32, 1, 512, generator=gen) * 32).round().clamp(-127, 127).to(torch.int8)
        return codes, table

    scale = lambda: (torch.randn(512, generator=gen) * 0.3).exp() * (4 * spread / 127)  # noqa: E731
    ori, ori_table = pool([max(1, p + min(n, DRAFT)) for p, n in zip(prefix, counts)])
    ori_scale, cmp_scale = scale(), scale() if ratio > 1 else None
    case = SharedKVCase(
        q=torch.randn(tokens, heads, 512, generator=gen).to(torch.bfloat16), ori=ori, ori_block_table=ori_table,
        cu_q=torch.tensor(cu + [-1] * pad, dtype=torch.int32),
        seq_lens=torch.tensor([p + n for p, n in zip(prefix, counts)] + [0] * pad, dtype=torch.int32),
        sink=torch.linspace(-2, 2, heads) if sink is None else sink, ratio=ratio, window=window)
    cmp_paths = None
    if ratio > 1:
        whole = [max(p, 0) // ratio for p in prefix]
        case.cmp, case.cmp_block_table = pool([w + DRAFT for w in whole])
    if ratio == 4:
        picks = torch.full((tokens, 1, topk), -1, dtype=torch.int32)
        for b in range(batch):
            rows = whole[b] + DRAFT
            for t in range(cu[b], cu[b + 1]):
                chosen = torch.randperm(rows, generator=gen)[:topk]
                picks[t, 0, :chosen.numel()] = chosen.to(torch.int32)
                if topk >= 4:            # a hole, an entry beyond the rows and a row named twice
                    picks[t, 0, 1] = -5
                    picks[t, 0, topk // 2] = rows + 3
                    picks[t, 0, topk - 1] = picks[t, 0, 0]
        case.cmp_indices = picks
    if ratio == 128:
        cmp_paths = torch.tensor([signed(rng.getrandbits(64) & rng.getrandbits(64) & rng.getrandbits(64)) for _ in range(tokens)])
    return case, torch.tensor([signed(m) for m in masks], dtype=torch.int64), cmp_paths, ori_scale, cmp_scale


def expected(case, paths, cmp_paths, ori_scale, cmp_scale, only=None):
    """(out, lse, bound of out, bound of lse) in float64; of the requests `only` when given."""
    tokens, heads, _ = case.q.shape
    live = max([b + 1 for b in range(case.seq_lens.numel()) if case.seq_lens[b] > 0 and case.cu_q[b + 1] >= 0], default=0)
    out, lse = torch.zeros(tokens, heads, 512, dtype=torch.float64), torch.zeros(tokens, heads, dtype=torch.float64)
    out_bound, lse_bound = torch.zeros_like(out), torch.zeros_like(lse)

    def rows(kind, b, logical):
        cache, table = (case.cmp, case.cmp_block_table) if kind else (case.ori, case.ori_block_table)
        found = [(int(table[b, r // 32]), r % 32) for r in logical if 0 <= r < table.shape[1] * 32]
        found = [(p, r) for p, r in found if 0 <= p < cache.shape[0]]
        index = torch.tensor(found, dtype=torch.int64).reshape(-1, 2)
        return cache[index[:, 0], index[:, 1], 0].double()

    for b in range(live):
        if only is not None and b not in only:
            continue
        first, last = int(case.cu_q[b]), int(case.cu_q[b + 1])
        n = last - first
        prefix = int(case.seq_lens[b]) - n
        whole = max(prefix, 0) // case.ratio
        for t in range(first, last):
            path = int(paths[t]) & (1 << min(n, DRAFT)) - 1
            near = list(range(max(0, prefix - (case.window - path.bit_count())), prefix))
            near += [prefix + j for j in range(DRAFT) if path >> j & 1]
            codes, scales = [rows(0, b, near)], [ori_scale.double()]
            if case.ratio == 128:
                extra = int(cmp_paths[t]) & (1 << 64) - 1 if cmp_paths is not None else 0
                codes.append(rows(1, b, list(range(whole)) + [whole + e for e in range(64) if extra >> e & 1]))
            elif case.ratio == 4:
                codes.append(rows(1, b, [r for r in case.cmp_indices[t, 0].tolist() if 0 <= r < whole + DRAFT]))
            if case.ratio > 1:
                scales.append(cmp_scale.double())
            q = case.q[t].double()
            v = torch.cat([c * s for c, s in zip(codes, scales)])
            s = q @ v.T * case.softmax_scale
            sink = case.sink.double()[:, None]
            top = torch.maximum(s.amax(1, keepdim=True), sink) if len(v) else sink
            w = (s - top).exp()
            total = w.sum(1, keepdim=True) + torch.where(sink == -math.inf, 0.0, (sink - top).exp())
            if len(v) == 0:
                lse[t] = case.sink.double()
                continue
            out[t] = w @ v / total
            lse[t] = (top + total.log())[:, 0]
            es = max(float((q * sc).abs().amax() * c.abs().sum(1).amax()) for c, sc in zip(codes, scales) if len(c)) * case.softmax_scale / 64516
            largest = (s.amax(1, keepdim=True) - top).exp()            # weight codes count from the largest logit, not from the sink
            ew = 4 / 32639 * largest
            dw = w * (math.exp(2 * es) - 1) + ew
            out_bound[t] = (dw @ v.abs() + out[t].abs() * dw.sum(1, keepdim=True)) / total + out[t].abs() * (BF16_HALF_STEP + 2 ** -20) + 1e-30
            lse_bound[t] = es + (len(v) * ew / total)[:, 0] + lse[t].abs() * 2 ** -20 + 2 ** -20
    return out, lse, out_bound, lse_bound


def check_dense(case, paths, cmp_paths, ori_scale, cmp_scale, out, lse):
    """The bounds above for many keys and tokens, a request at a time on the tensors' device (live requests whose
    rows all have pages).  Returns the largest errors of out and lse in units of their bounds."""
    worst = [-math.inf, -math.inf]
    bits = torch.arange(DRAFT, device=case.q.device)
    for b in range(case.seq_lens.numel()):
        first, last = int(case.cu_q[b]), int(case.cu_q[b + 1])
        n, t = last - first, slice(first, last)
        prefix = int(case.seq_lens[b]) - n
        whole = prefix // case.ratio

        def rows(cache, table, logical):
            return cache[table[b, logical // 32].long(), logical % 32, 0].double()

        start = max(0, prefix - case.window)
        near = torch.arange(start, prefix + min(n, DRAFT), device=case.q.device)
        path = ((paths[t, None] >> bits) & 1).bool() & (bits < n)
        weight = torch.zeros(n, near.numel(), dtype=torch.float64, device=case.q.device)
        weight[:, :prefix - start] = (near[:prefix - start] >= prefix - (case.window - path.sum(1, keepdim=True))).double()
        weight[:, prefix - start:] = path[:, :min(n, DRAFT)].double()
        codes, scales, weights = [rows(case.ori, case.ori_block_table, near)], [ori_scale.double()], [weight]
        if case.ratio > 1:
            far = torch.arange(min(whole + DRAFT, case.cmp_block_table.shape[1] * 32), device=case.q.device)
            weight = torch.zeros(n, whole + DRAFT + 1, dtype=torch.float64, device=case.q.device)
            if case.ratio == 128:
                weight[:, :whole] = 1
                weight[:, whole:whole + DRAFT] = ((cmp_paths[t, None] >> bits) & 1).double()
            else:
                picks = case.cmp_indices[t, 0].long()
                picks = torch.where((picks >= 0) & (picks < whole + DRAFT), picks, whole + DRAFT)
                weight.scatter_add_(1, picks, torch.ones_like(picks, dtype=torch.float64))
            codes.append(rows(case.cmp, case.cmp_block_table, far))
            scales.append(cmp_scale.double())
            weights.append(weight[:, :far.numel()])
        v, w0 = torch.cat([c * s for c, s in zip(codes, scales)]), torch.cat(weights, 1)[:, None]
        q = case.q[t].double()
        s = torch.einsum("nhd,ld->nhl", q, v) * case.softmax_scale
        s = s.masked_fill(w0 == 0, -math.inf)
        sink = case.sink.double()[None, :, None]
        largest = s.amax(2, keepdim=True)
        top = torch.maximum(largest, sink)
        w = (s - top).exp() * w0
        total = w.sum(2, keepdim=True) + (sink - top).exp()
        want, want_lse = torch.einsum("nhl,ld->nhd", w, v) / total, (top + total.log())[..., 0]
        # an entry named k times carries a weight k times as large, and the reference counts from the largest of those
        lift = (s + w0.clamp_min(1).log()).amax(2, keepdim=True)
        es = torch.stack([(q * sc).abs().amax(2) * c.abs().sum(1).amax() for c, sc in zip(codes, scales)]).amax(0)[..., None] * case.softmax_scale / 64516
        dw = w * ((2 * es).exp() - 1) + 4 / 32639 * (lift - top).exp() * (w0 > 0)
        bound = (torch.einsum("nhl,ld->nhd", dw, v.abs()) + want.abs() * dw.sum(2, keepdim=True)) / total + want.abs() * (BF16_HALF_STEP + 2 ** -20) + 1e-30
        lse_bound = (es + (w0 > 0).sum(2, keepdim=True) * 4 / 32639 * (lift - top).exp() / total)[..., 0] + want_lse.abs() * 2 ** -20 + 2 ** -20
        worst[0] = max(worst[0], float(((out[t].double() - want).abs() / bound).max()))
        worst[1] = max(worst[1], float(((lse[t].double() - want_lse).abs() / lse_bound).max()))
    return worst
