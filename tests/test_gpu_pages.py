"""Page pool operations against a pool kept in Python: tables, lengths, counts and codes are exact."""
import random

import pytest
import torch

from npu_sparse_attn_sharedkv_int8 import PagePool
from npu_sparse_attn_sharedkv_int8.pages import count_references

pytestmark = pytest.mark.gpu


class Model:
    """The same pool, one step at a time."""

    def __init__(self, table, lens, refs, caches, rows):
        self.table, self.lens, self.refs = [list(r) for r in table.tolist()], lens.tolist(), refs.tolist()
        self.caches, self.rows, self.refused = [c.clone() for c in caches], rows, False

    def live(self, rows):
        return -(-rows // self.rows)

    def _take(self, count):
        free = [p for p, r in enumerate(self.refs) if r == 0][:count]
        return free if len(free) == count else None

    def _move(self, source, target):
        for cache in self.caches:
            cache[target] = cache[source]

    def resize(self, wanted):
        width = len(self.table[0])
        if any(w < 0 or self.live(w) > width for w in wanted):
            self.refused = True
            return
        before = list(self.refs)
        for b, w in enumerate(wanted):
            for k in range(self.live(w), self.live(self.lens[b])):
                self.refs[self.table[b][k]] -= 1
        split = [w > n and n % self.rows != 0 and self.refs[self.table[b][self.live(n) - 1]] > 1
                 for b, (w, n) in enumerate(zip(wanted, self.lens))]
        need = [int(s) + max(0, self.live(w) - self.live(n)) for s, w, n in zip(split, wanted, self.lens)]
        fresh = self._take(sum(need))
        if fresh is None:
            self.refs, self.refused = before, True
            return
        for b, w in enumerate(wanted):
            at = self.live(self.lens[b])
            if split[b]:
                source, page = self.table[b][at - 1], fresh.pop(0)
                self._move(source, page)
                self.refs[source] -= 1
                self.refs[page], self.table[b][at - 1] = 1, page
            for k in range(at, self.live(w)):
                page = fresh.pop(0)
                self.refs[page], self.table[b][k] = 1, page
            self.lens[b] = w

    def fork(self, parents):
        if any(p >= len(self.lens) for p in parents):
            self.refused = True
            return
        before, old, lens = list(self.refs), [list(r) for r in self.table], list(self.lens)
        children = [[b for b, p in enumerate(parents) if p == i] for i in range(len(lens))]
        for i, mine in enumerate(children):
            for k in range(self.live(lens[i])):
                full = k < lens[i] // self.rows
                self.refs[old[i][k]] += (len(mine) - 1) if full else (-1 if not mine else 0)
        copied = [b for b, p in enumerate(parents) if p >= 0 and children[p][0] != b and lens[p] % self.rows]
        fresh = self._take(len(copied))
        if fresh is None:
            self.refs, self.refused = before, True
            return
        for b, p in enumerate(parents):
            self.lens[b] = lens[p] if p >= 0 else 0
            for k in range(self.live(self.lens[b])):
                self.table[b][k] = old[p][k]
            if b in copied:
                k = self.live(lens[p]) - 1
                self.table[b][k] = fresh.pop(0)
                self.refs[self.table[b][k]] = 1
                self._move(old[p][k], self.table[b][k])


def make_pool(rng, batch, pages, *, layers=2, rows=32, width=12, stride=None, longest=None, shared=False):
    stride = stride or rows * 512
    caches = []
    for layer in range(layers):
        raw = torch.randint(-128, 128, (pages * stride,), dtype=torch.int8)
        caches.append(raw.cuda().as_strided((pages, rows, 1, 512), (stride, 512, 512, 1)))
    order = rng.sample(range(pages), pages)
    lens = [rng.randint(0, longest if longest is not None else width * rows // 2) for _ in range(batch)]
    table = [[rng.choice([-1, 10 ** 6]) for _ in range(width)] for _ in range(batch)]
    for b in range(batch):
        for k in range(-(-lens[b] // rows)):
            table[b][k] = order.pop()
        if shared and b % 2 and lens[b - 1]:                # every second sequence holds its neighbour's pages
            lens[b] = lens[b - 1]
            table[b][:] = table[b - 1]
    table, lens = torch.tensor(table, dtype=torch.int32).reshape(batch, width), torch.tensor(lens, dtype=torch.int32)
    refs = count_references(table, lens, rows, pages)
    return PagePool(caches, table.cuda(), lens.cuda(), refs.cuda()), Model(table, lens, refs, [c.cpu() for c in caches], rows)


def check(pool, model):
    torch.cuda.synchronize()
    assert pool.lens.tolist() == model.lens
    assert pool.refs.tolist() == model.refs
    assert pool.table.tolist() == model.table
    for got, want in zip(pool.caches, model.caches):
        assert torch.equal(got.cpu(), want)
    if model.refused:
        with pytest.raises(RuntimeError, match="refused"):
            pool.status()
    else:
        pool.status()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("batch, pages, options", [
    (1, 1, dict(longest=0)), (1, 40, {}), (3, 33, dict(width=3, longest=32)), (7, 129, dict(rows=16, stride=16 * 512 + 16)),
    (40, 300, dict(shared=True)), (40, 400, dict(rows=5, width=20, layers=3)), (9, 1000, dict(shared=True, rows=1, width=9)),
    (700, 9000, dict(layers=1, rows=2, width=30, shared=True)), (1100, 1200, dict(layers=1, rows=1, width=2, longest=1))])
def test_sequences_of_operations(batch, pages, options):
    rng = random.Random(batch * 1000 + pages)
    pool, model = make_pool(rng, batch, pages, **options)
    check(pool, model)
    most = pool.table.shape[1] * pool.page_rows
    for step in range(8):
        if step % 3 == 2:
            parents = [rng.randrange(-1, batch) for _ in range(batch)]
            pool.fork(ints(parents))
            model.fork(parents)
        else:
            wanted = [max(0, min(most, n + rng.randint(-2 * pool.page_rows, 2 * pool.page_rows))) for n in model.lens]
            if step == 4:
                wanted = [0 if rng.random() < 0.5 else n for n in wanted]
            pool.resize(ints(wanted))
            model.resize(wanted)
        check(pool, model)


def test_shared_last_pages_are_copied_before_they_grow():
    """Two sequences hold the same partly filled page; both grow, one is cut back into a shared page and
    grows again."""
    pool, model = make_pool(random.Random(2), 6, 100, shared=True, longest=200)
    for step in (lambda n, b: n + 3, lambda n, b: n // 2, lambda n, b: n + (b % 2) * 40):
        wanted = [step(n, b) for b, n in enumerate(model.lens)]
        pool.resize(ints(wanted))
        model.resize(wanted)
        check(pool, model)


@pytest.mark.parametrize("bad", ["no room", "too long", "negative", "unknown parent", "no room to fork"])
def test_refused_operations_change_nothing(bad):
    rng = random.Random(8)
    pool, model = make_pool(rng, 6, 40, width=12, longest=150)
    wanted = {"no room": [384] * 6, "too long": [385] + [0] * 5, "negative": [-1] + [10] * 5}.get(bad)
    if bad == "no room to fork":
        pool, model = make_pool(rng, 4, 5, width=12, longest=40)
        lens = [10, 10, 10, 10]
        for w in (lens,):
            pool.resize(ints(w)), model.resize(w)
        check(pool, model)
        pool.refs[:] = torch.where(pool.refs == 0, 1, pool.refs)        # pinned by the caller
        model.refs = [r or 1 for r in model.refs]
        parents = [0, 0, 2, 3]
        pool.fork(ints([0, 0, 2, 3]))
        model.fork(parents)                                             # sequence 1's page is released and taken
        check(pool, model)
        return
    if wanted:
        pool.resize(ints(wanted))
        model.resize(wanted)
    else:
        pool.fork(ints([0, 1, 6, 3, 4, 5]))
        model.fork([0, 1, 6, 3, 4, 5])
    assert model.refused
    check(pool, model)
    pool.resize(ints([5] * 6))                                          # and the pool goes on
    model.resize([5] * 6)
    check(pool, model)


@pytest.mark.parametrize("rows, stride", [(32, None), (32, 16400), (3, None), (40, 40 * 512 + 64)])
def test_copy(rows, stride):
    rng = random.Random(rows)
    pool, model = make_pool(rng, 1, 64, layers=3, rows=rows, stride=stride)
    order = rng.sample(range(64), 64)
    pairs = [(order[i % 7], order[20 + i]) for i in range(20)] + [(-1, order[60]), (order[0], 64), (64, order[61])]
    for source, target in pairs[:20]:
        model._move(source, target)
    bare = PagePool(pool.caches)
    bare.copy(ints(pairs))
    bare.copy(ints(pairs)[:0])
    check(pool, model)


@pytest.mark.parametrize("batch, kept, rows, stride", [(1, 1, 32, None), (5, 64, 32, None), (9, 17, 32, 16400), (300, 5, 4, None), (3, 20, 7, 7 * 512 + 16)])
def test_keep(batch, kept, rows, stride):
    rng = random.Random(kept)
    pool, model = make_pool(rng, batch, max(64, batch * 30), layers=2, rows=rows, stride=stride, width=25, longest=24 * rows)
    base = [rng.randint(0, max(0, n - 5)) for n in model.lens]
    chosen = []
    for b in range(batch):
        row = sorted(rng.sample(range(80), kept))
        row = [r if rng.random() < 0.8 else -1 for r in row]
        if b % 3 == 2:
            rng.shuffle(row)                                            # any order: read before written
        chosen.append(row)
    for cache in model.caches:
        old = cache.clone()

        def place(b, row):
            page = model.table[b][row // rows] if row < 25 * rows else -1
            return (page, row % rows) if 0 <= page < pool.pages else None

        for b in range(batch):
            for i, r in enumerate(chosen[b]):
                source, target = place(b, base[b] + max(r, 0)), place(b, base[b] + i)
                if r >= 0 and source and target:
                    cache[target] = old[source]
    pool.keep(ints(base), ints(chosen))
    check(pool, model)


def test_offsets_beyond_32_bits():
    stride, pages = 1 << 20, 5003
    cache = torch.empty(pages * stride, dtype=torch.int8, device="cuda").as_strided((pages, 32, 1, 512), (stride, 512, 512, 1))
    cache[5000:] = torch.randint(-128, 128, (3, 32, 1, 512), dtype=torch.int8, device="cuda")
    old = cache[5000:].clone()
    table = ints([[5000, 5001, 5002], [4998, 4999, 0]])
    pool = PagePool([cache], table)
    pool.copy(ints([[5001, 4999], [5002, 3]]))
    pool.keep(ints([40, 0]), ints([[3, 25], [-1, -1]]))                 # rows 43 and 65 of sequence 0 to 40 and 41
    assert torch.equal(cache[4999], old[1]) and torch.equal(cache[3], old[2])
    assert torch.equal(cache[5001, 8], old[1, 11]) and torch.equal(cache[5001, 9], old[2, 1])
    old[1, 8], old[1, 9] = old[1, 11].clone(), old[2, 1].clone()
    assert torch.equal(cache[5000:], old)


def test_captured_steps():
    """A captured grow / fork / trim step, replayed with other inputs."""
    rng = random.Random(77)
    pool, model = make_pool(rng, 12, 400, layers=2)
    grown, parents, trimmed = (ints([0] * 12) for _ in range(3))
    state = [t.clone() for t in (pool.table, pool.lens, pool.refs)]
    grown.copy_(pool.lens), trimmed.copy_(pool.lens), parents.copy_(torch.arange(12))
    pool.resize(grown), pool.fork(parents), pool.resize(trimmed)
    torch.cuda.synchronize()
    for now, then in zip((pool.table, pool.lens, pool.refs), state):
        assert torch.equal(now, then)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pool.resize(grown)
        pool.fork(parents)
        pool.resize(trimmed)
    for _ in range(4):
        steps = [n + rng.randint(0, 40) for n in model.lens]
        of = [rng.randrange(12) for _ in range(12)]
        ends = [max(0, steps[p] - rng.randint(0, 40)) for p in of]
        for tensor, values in ((grown, steps), (parents, of), (trimmed, ends)):
            tensor.copy_(ints(values))
        graph.replay()
        model.resize(steps), model.fork(of), model.resize(ends)
        check(pool, model)


def test_refusals():
    cache = torch.zeros(8, 32, 1, 512, dtype=torch.int8, device="cuda")
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    for arguments, text in (([], "at least one"), ([cache.half()], "INT8"), ([cache, cache[:4]], "one shape"), ([cache.cpu()], "CUDA"),
                            ([cache[:, :, :, 8:]], "INT8")):
        with pytest.raises(ValueError, match=text):
            PagePool(arguments)
    with pytest.raises(ValueError, match="table"):
        PagePool([cache], table.long())
    with pytest.raises(ValueError, match="lens"):
        PagePool([cache], table, lens[:1])
    with pytest.raises(ValueError, match="refs"):
        PagePool([cache], table, lens, lens)
    pool = PagePool([cache], table, lens)
    with pytest.raises(ValueError, match="lens"):
        pool.resize(lens.long())
    with pytest.raises(ValueError, match="parents"):
        pool.fork(lens[:1])
    with pytest.raises(ValueError, match="pairs"):
        pool.copy(lens)
    with pytest.raises(ValueError, match="kept"):
        pool.keep(lens, torch.zeros(2, 65, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="lengths"):
        PagePool([cache], table).resize(lens)
    with pytest.raises(ValueError, match="block table"):
        PagePool([cache]).keep(lens, table)


def test_refuses_aliases():
    """The pool's own lengths as new ones (a caller who added to them in place would get no pages), and a cache
    whose rows would move twice."""
    cache = torch.zeros(8, 32, 1, 512, dtype=torch.int8, device="cuda")
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="tensor of their own"):
        PagePool([cache], table, lens).resize(lens)
    with pytest.raises(ValueError, match="twice"):
        PagePool([cache, cache], table, lens)
