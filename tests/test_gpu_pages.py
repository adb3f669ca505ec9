"""The page pool's updates, compaction and copies (csrc/paged_cache.hip) against the rules applied row by row on the
host (oracle/serving_oracle.py): every number equal, every byte of the pages equal."""
import random

import pytest
import torch

from conftest import PKG
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
pc = PKG.models.modules.paged_cache


def i32(x, dev="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Pair:
    """A pool on the device and its copy on the host, stepped together."""

    def __init__(self, n, width, pages, ps, dev, layers=2, heads=2, dim=8, dtype=torch.bfloat16, data=True):
        self.ps, self.dev = ps, dev
        self.table, self.lens, self.refs = [[-1] * width for _ in range(n)], [0] * n, [0] * pages
        self.data = torch.randn(layers, 2, pages, heads, ps, dim).to(dtype) if data else None
        self.g = [i32(self.table, dev).view(n, width), i32(self.lens, dev), i32(self.refs, dev)]
        self.gdata = self.data.to(dev) if data else None

    def pin(self, page):
        self.refs[page] += 1
        self.g[2][page] += 1

    def update(self, parents=None, new_lens=None):
        before = [t.clone() for t in self.g]
        out = pc.pages_update(self.gdata, *self.g, parents=None if parents is None else i32(parents, self.dev),
                              new_lens=None if new_lens is None else i32(new_lens, self.dev), page_size=self.ps)
        for a, b in zip(before, self.g):
            assert torch.equal(a, b)  # inputs untouched
        self.table, self.lens, self.refs, short = O.pages_update(self.table, self.lens, self.refs, parents, new_lens,
                                                                 self.ps, self.data)
        self.g = list(out[:3])
        assert int(out[3]) == short
        self.same()
        return short

    def compact(self):
        table, refs, remap, live = pc.pages_compact(self.gdata, self.g[0], self.g[2])
        self.table, self.refs, rm, lv = O.pages_compact(self.table, self.refs, self.data)
        self.g[0], self.g[2] = table, refs
        assert int(live) == lv and remap.tolist() == rm
        self.same()

    def same(self):
        assert self.g[0].tolist() == self.table and self.g[1].tolist() == self.lens and self.g[2].tolist() == self.refs
        if self.data is not None:
            assert torch.equal(self.gdata.cpu(), self.data)


def test_grow_fork_write_on_copy(dev):
    p = Pair(4, 4, 20, 8, dev)
    p.update(new_lens=[11, 0, 8, 3])
    p.update(parents=[0, 0, 0, 0])                  # all share row 0: no page moves
    assert p.refs.count(4) == 2
    p.update(new_lens=[12, 11, 12, 12])             # row 1 keeps the old page: three copies
    p.update(parents=[3, 3, 3, 3], new_lens=[13] * 4)   # every sharer grows: the highest keeps it
    p.update(new_lens=[2, 0, 9, 32])
    p.update(new_lens=[100, -5, 9, 0])              # clamped to [0, 32]
    p.update(parents=[-1, 7, 2, 2])                 # unknown parents: empty rows
    p.update(new_lens=[0] * 4)
    assert sum(p.refs) == 0


def test_cut_to_a_shared_full_page_then_grow(dev):
    p = Pair(2, 4, 12, 8, dev)
    p.update(new_lens=[16, 0])
    p.update(parents=[0, 0])
    p.update(new_lens=[13, 16])                     # row 0 now ends inside a page that row 1 still fills
    p.update(new_lens=[14, 16])                     # so it takes a copy


def test_running_short_changes_nothing(dev):
    p = Pair(3, 4, 5, 8, dev)
    p.update(new_lens=[16, 9, 0])
    assert p.update(new_lens=[17, 10, 8]) == 1
    assert p.update(parents=[0, 0, 0], new_lens=[17, 17, 32]) == 1   # row 1's pages come free in the same step
    assert p.update(new_lens=[17, 10, 0]) == 0
    assert p.update(new_lens=[32, 32, 32]) > 0


def test_pinned_pages_are_not_given_away(dev):
    p = Pair(2, 3, 8, 4, dev)
    p.pin(0)
    p.pin(2)
    p.update(new_lens=[9, 4])
    assert p.table[0] == [1, 3, 4]
    p.pin(4)                                        # a holder outside the table: growing copies
    p.update(new_lens=[10, 4])
    p.compact()


def test_damaged_entries_hold_nothing(dev):
    p = Pair(2, 3, 8, 4, dev)
    p.update(new_lens=[9, 10])
    p.table[0][1] = -1
    p.table[1][2] = 99
    p.g[0] = i32(p.table, dev)
    p.update(new_lens=[11, 11])
    p.update(parents=[1, 0], new_lens=[12, 12])
    p.compact()


@pytest.mark.parametrize("n, width, pages, ps, seed", [(1, 1, 1, 1, 0), (5, 7, 40, 4, 1), (12, 40, 300, 1, 2),
                                                     (300, 9, 1500, 16, 3), (7, 300, 1025, 2, 4), (40, 20, 500, 32, 5),
                                                     (1200, 3, 5000, 8, 6), (100, 100, 8192, 4, 7),
                                                     (1024, 16, 8191, 16, 8), (3, 6000, 20000, 1, 9)])
def test_random_histories(dev, n, width, pages, ps, seed):
    """Forks, cuts, growth and compactions in turn; now and then more is asked for than there is."""
    r = random.Random(seed)
    torch.manual_seed(seed)
    p = Pair(n, width, pages, ps, dev, layers=1, heads=2, dim=8)
    for step in range(8):
        parents = [r.randrange(-1, n) if r.random() < 0.6 else s for s in range(n)] if r.random() < 0.7 else None
        base = p.lens if parents is None else [p.lens[x] if x >= 0 else 0 for x in parents]
        top = max(1, min(width * ps, int(2.2 * pages * ps / n)))
        new = [min(top, max(0, b + r.choice([0, 1, 1, 2, ps, -1, -ps, r.randrange(top + 1)]))) for b in base]
        p.update(parents, new if r.random() < 0.9 else None)
        if step % 3 == 2:
            p.compact()


@pytest.mark.parametrize("pages", [1, 1023, 1024, 1025, 5000])
@pytest.mark.parametrize("share", [0.0, 0.3, 1.0])
def test_compaction(dev, pages, share):
    r = random.Random(pages)
    p = Pair(1, 1, pages, 4, dev, layers=1, heads=1, dim=8)
    p.refs = [int(r.random() < share) * r.randrange(1, 3) for _ in range(pages)]
    held = [x for x in range(pages) if p.refs[x]]
    r.shuffle(held)
    p.table = [held + [-1, pages, 0 if not p.refs[0] else -5]]
    p.g[0], p.g[2] = i32(p.table, dev), i32(p.refs, dev)
    p.compact()
    p.compact()                                     # a compact pool stays as it is


@pytest.mark.parametrize("dtype, dim", [(torch.float32, 4), (torch.bfloat16, 72), (torch.float16, 128)])
def test_types_and_copy(dev, dtype, dim):
    p = Pair(3, 3, 12, 8, dev, layers=3, heads=3, dim=dim, dtype=dtype)
    p.update(new_lens=[5, 7, 1])
    p.update(parents=[1, 1, 1], new_lens=[8, 9, 17])
    src, dst = [0, 3, 99, 1, -1], [7, 9, 1, -2, 4]
    pc.pages_copy(p.gdata, i32(src, dev), i32(dst, dev))
    p.data[:, :, 7], p.data[:, :, 9] = p.data[:, :, 0], p.data[:, :, 3]
    p.same()
    pc.pages_copy(p.gdata, i32([], dev), i32([], dev))
    p.same()


def test_without_data_and_without_rows(dev):
    p = Pair(3, 3, 12, 8, dev, data=False)
    p.update(new_lens=[5, 7, 1])
    p.update(parents=[0, 0, 0], new_lens=[6, 6, 6])
    p.compact()
    t, l, f, short = pc.pages_update(None, torch.empty(0, 4, dtype=torch.int32, device=dev), i32([], dev),
                                     i32([0, 1], dev), page_size=4)
    assert t.shape == (0, 4) and f.tolist() == [0, 1] and int(short) == 0
    t, l, f, short = pc.pages_update(None, torch.full((2, 1), -1, dtype=torch.int32, device=dev), i32([0, 0], dev),
                                     i32([], dev), new_lens=i32([1, 1], dev), page_size=4)
    assert int(short) == 2 and l.tolist() == [0, 0]


def test_graph_and_stream(dev):
    p = Pair(6, 6, 60, 4, dev)
    p.update(new_lens=[9, 9, 9, 14, 0, 2])
    par, new = i32([0, 0, 3, 3, 3, 5], dev), i32([10, 11, 15, 15, 16, 3], dev)
    data0 = p.gdata.clone()
    want = pc.pages_update(p.gdata, *p.g, parents=par, new_lens=new)
    wdata = p.gdata.clone()
    p.gdata.copy_(data0)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = pc.pages_update(p.gdata, *p.g, parents=par, new_lens=new)
        comp = pc.pages_compact(None, got[0], got[2])
    for _ in range(3):
        p.gdata.copy_(data0)
        for t in got + comp:
            t.fill_(-9)
        gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert torch.equal(p.gdata, wdata)
        assert comp[1].tolist() == O.pages_compact(want[0].tolist(), want[2].tolist())[1]
        eager = pc.pages_compact(None, want[0], want[2])
        assert torch.equal(eager[0], comp[0])
    p.gdata.copy_(data0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = pc.pages_update(p.gdata, *p.g, parents=par, new_lens=new)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(other, want):
        assert torch.equal(a, b)


def test_cache_runs_a_beam_search_of_chunks(dev):
    """The operators together: a prompt chunk, forks with copies on write, single tokens, a cut, a compaction —
    each attention equal to one over every row's own dense history."""
    torch.manual_seed(0)
    n, heads, kvh, dim, ps, layers = 6, 4, 2, 32, 4, 2
    dt = torch.float32
    cache = pc.PagedKVCache(layers, n, 40, kvh, dim, page_size=ps, dtype=dt, device=dev)
    hist = [[torch.zeros(layers, 2, 0, kvh, dim)] for _ in range(n)]
    hist = [h[0] for h in hist]
    r = random.Random(3)

    def step(new_tokens, parents):
        nonlocal hist
        if parents is not None:
            hist = [hist[p].clone() for p in parents]
        lens = [h.shape[2] + m for h, m in zip(hist, new_tokens)]
        cache.update(None if parents is None else i32(parents, dev), i32(lens, dev))
        rows = max(new_tokens)
        starts = [h.shape[2] for h in hist]
        for layer in range(layers):
            q = torch.randn(n, rows, heads, dim)
            kv = torch.randn(2, n, rows, kvh, dim)
            out = cache.attend(layer, q.to(dev), kv[0].to(dev), kv[1].to(dev), starts=i32(starts, dev)).cpu()
            for s in range(n):
                new = kv[:, s, :new_tokens[s]]
                full = torch.cat([hist[s][layer], new], 1)
                table = torch.arange(max(1, full.shape[1]), dtype=torch.int32)[None]
                ref, aux, _, _ = O.paged_attention(
                    q[s:s + 1], full[0][:, :, None], full[1][:, :, None], table, i32([full.shape[1]]),
                    starts=i32([starts[s]]))
                # fp32: the terms of test_gpu_paged_attention's tolerance
                A, _, S = aux
                tol = 2.0 ** -24 * ref.abs() + A * (2 * ((dim + 8) * 2.0 ** -24 * S[..., None] + 2.0 ** -20)
                                                    + 80 * 2.0 ** -24) + 1e-30
                assert bool(((out[s:s + 1].double() - ref).abs() <= tol).all()), (s, layer)
            if layer == layers - 1:
                pad = [torch.stack([kv_l[:, s, :new_tokens[s]] for kv_l in (step.first, kv)]) for s in range(n)]
                hist = [torch.cat([h, x], 2) for h, x in zip(hist, pad)]
            step.first = kv
        assert int(cache.short) == 0

    step([5, 1, 3, 5, 4, 2], None)
    for _ in range(6):
        step([r.randrange(0, 3) for _ in range(n - 1)] + [1], [r.randrange(n) for _ in range(n)])
    cut = [max(0, h.shape[2] - 3) for h in hist]
    cache.update(new_lens=i32(cut, dev))
    hist = [h[:, :, :c] for h, c in zip(hist, cut)]
    cache.compact()
    step([1] * n, [r.randrange(n) for _ in range(n)])
    cache.update(new_lens=i32([0] * n, dev))
    assert int(cache.refs.abs().sum()) == 0


def test_compaction_of_a_large_pool(dev):
    """More than 256 MB of pages (the ranks in launches of their own), few pages enough for one workgroup's."""
    r = random.Random(1)
    pages = 600
    data = torch.randint(-9, 9, (2, 2, pages, 4, 64, 256), dtype=torch.int16, device=dev).view(torch.bfloat16)
    refs = [int(r.random() < 0.5) for _ in range(pages)]
    table = [x for x in range(pages) if refs[x]]
    want = data.clone()
    t, f, remap, live = pc.pages_compact(data, i32(table, dev), i32(refs, dev))
    ot, of, orm, ol = O.pages_compact([table], refs, want)
    assert t.tolist() == ot[0] and f.tolist() == of and remap.tolist() == orm and int(live) == ol
    assert torch.equal(data.view(torch.int16), want.view(torch.int16))
