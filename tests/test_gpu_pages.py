"""Pages and rows moved within a paged cache: bits, against indexing on the host."""

import random

import pytest
import torch

import svdmlp
from test_gpu_decoder import BF, F32, _gen, _pages, _randn

pytestmark = pytest.mark.gpu


def _pool(g, n, pages, page, K, D, dtype, kind, gpu):
    """(caches on the CPU (n, pages, page, K, D), the same on the GPU as the kind of argument, the GPU's buffer)."""
    if kind == "tensor":
        cpu = _randn(g, n, pages, page, K, D, dtype=dtype)
        buf = cpu.to(gpu)
        return cpu, buf, buf
    if kind == "list":
        cpu = _randn(g, n, pages, page, K, D, dtype=dtype)
        buf = [c.clone() for c in cpu.to(gpu)]
        return cpu, buf, buf
    if kind == "joint":  # all caches of a page side by side
        buf = _randn(g, pages, n, page, K, D, dtype=dtype)
        gb = buf.to(gpu)
        return buf.transpose(0, 1).contiguous(), list(gb.unbind(1)), gb
    # heads outside rows, rows of one value more than the heads hold
    buf = _randn(g, n, pages, K, page, D + 1, dtype=dtype)
    gb = buf.to(gpu)
    return buf[..., 1:].transpose(2, 3).contiguous(), gb[..., 1:].transpose(2, 3), gb


def _same(caches, want):
    for c, w in zip(caches, want):
        assert torch.equal(c.cpu(), w)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", ["tensor", "list", "joint", "strided"])
@pytest.mark.parametrize("n,pages,page,K,D,m", [(1, 3, 1, 1, 1, 1), (2, 40, 16, 8, 128, 17), (5, 9, 7, 3, 5, 4), (150, 12, 4, 2, 24, 6), (3, 6, 300, 2, 64, 2)])
def test_copy_pages(gpu, dtype, kind, n, pages, page, K, D, m):
    g = _gen(n * 7 + pages)
    cpu, caches, _ = _pool(g, n, pages, page, K, D, dtype, kind, gpu)
    order = torch.randperm(pages, generator=g)
    src, dst = order[:m], order[m:2 * m]
    rows = torch.randint(-1, page + 3, (m,), generator=g)
    want = cpu.clone()
    for i, j, r in zip(src.tolist(), dst.tolist(), rows.clamp(0, page).tolist()):
        want[:, j, :r] = cpu[:, i, :r]
    svdmlp.copy_pages(caches, src.int().to(gpu), dst.to(gpu), rows.to(gpu))
    _same(caches, want)
    want[:, dst] = cpu[:, src]
    svdmlp.copy_pages(caches, src.to(gpu), dst.int().to(gpu))
    _same(caches, want)


def test_copy_pages_outside_the_cache(gpu):
    """Pairs with a page outside the cache, or of a page and itself, are skipped; 64-bit numbers keep their meaning."""
    g = _gen(3)
    cpu, caches, _ = _pool(g, 2, 5, 4, 2, 16, BF, "tensor", gpu)
    src = torch.tensor([-1, 0, 5, 1, 2, 2 ** 32, 3, 2 ** 40])
    dst = torch.tensor([0, -2, 1, 5, 2, 3, 2 ** 32 + 4, 4])
    svdmlp.copy_pages(caches, src.to(gpu), dst.to(gpu))
    _same(caches, cpu)
    svdmlp.copy_pages(caches, src[:0].to(gpu), dst[:0].to(gpu))
    _same(caches, cpu)


def test_copy_pages_far_apart(gpu):
    """Pages whose byte offsets pass 2^32."""
    c = torch.zeros((1, 70000, 64, 4, 128), dtype=BF, device=gpu)
    small = _randn(_gen(4), 64, 4, 128).to(gpu)
    c[0, 69999] = small
    svdmlp.copy_pages(c, torch.tensor([69999], device=gpu), torch.tensor([69000], device=gpu))
    assert torch.equal(c[0, 69000], small) and int((c[0].flatten(1) != 0).any(dim=1).sum()) == 2


def _kept(path, drafts):
    """The accepted drafts of a row of `path`, as far as they count."""
    kept = []
    for p in path:
        if p <= (kept[-1] if kept else -1) or p >= drafts:
            break
        kept.append(p)
    return kept


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kind", ["tensor", "list", "joint", "strided"])
@pytest.mark.parametrize("lens,drafts,n,page,K,D", [
    ([1], 1, 1, 1, 1, 1), ([70, 64, 0, 3], 64, 3, 16, 2, 32), ([30, 9, 100], 8, 140, 16, 8, 16), ([50] * 70, 20, 2, 7, 3, 5), ([300, 17], 17, 4, 64, 8, 128)])
def test_keep_drafts(gpu, dtype, kind, lens, drafts, n, page, K, D):
    g, rng = _gen(sum(lens) + n), random.Random(drafts)
    table, pages = _pages(g, lens, page)
    table[table < 0] = 0  # behind a sequence's end: not followed
    cpu, caches, _ = _pool(g, n, pages, page, K, D, dtype, kind, gpu)
    paths = []
    for b in range(len(lens)):  # none, all, a chain from the first draft on, whatever a tree gives
        k = rng.randint(0, drafts)
        p = [list(range(k)), list(range(drafts)), sorted(rng.sample(range(drafts), k))][b % 3]
        paths.append((p + [-1] * drafts)[:drafts])
    want, new = cpu.clone(), []
    for b, (length, path) in enumerate(zip(lens, paths)):
        context, kept = length - drafts, _kept(path, drafts) if length >= drafts else []
        at = lambda x: (int(table[b, x // page]), x % page)  # noqa: E731
        for i, p in enumerate(kept):
            (pd, rd), (ps, rs) = at(context + i), at(context + p)
            want[:, pd, rd] = cpu[:, ps, rs]
        new.append(context + len(kept) if length >= drafts else length)
    ln, pt = torch.tensor(lens), torch.tensor(paths)
    got = svdmlp.keep_drafts(caches, table.to(gpu), ln.to(gpu), pt.to(gpu), drafts)
    assert got.dtype == torch.int32 and got.tolist() == new
    _same(caches, want)


def test_keep_drafts_broken_paths_and_tables(gpu):
    """A path ends where it stops to increase or leaves the drafts; rows in pages outside the cache are not moved; lengths beyond the table are cut."""
    g = _gen(6)
    page, drafts = 4, 6
    cpu, caches, _ = _pool(g, 2, 12, page, 2, 8, F32, "tensor", gpu)
    table = torch.tensor([[0, 1], [2, 3], [4, 5], [6, 99], [8, 9], [10, 11]])
    lens = [8, 8, 8, 8, 10 ** 10, -5]
    paths = [[1, 3, 3, 4], [2, 6, 7, 8], [3, 1, 2, 4], [1, 3, 4, 5], [5, -1, 5, 5], [1, 2, 3, 4]]
    want = cpu.clone()
    for b, kept in ((0, [1, 3]), (1, [2]), (2, [3]), (3, [1]), (4, [5])):
        for i, p in enumerate(kept):
            x, y = 2 + i, 2 + p
            want[:, table[b, x // page], x % page] = cpu[:, table[b, y // page], y % page]
    got = svdmlp.keep_drafts(caches, table.to(gpu), torch.tensor(lens).to(gpu), torch.tensor(paths).to(gpu), drafts)
    _same(caches, want)
    assert got.tolist() == [4, 3, 3, 6, 3, 0]


def test_pages_refusals(gpu):
    c = torch.zeros(4, 6, 4, 2, 8, device=gpu)
    i, t, ln = torch.zeros(2, dtype=torch.int32, device=gpu), torch.zeros(2, 3, dtype=torch.int32, device=gpu), torch.ones(2, dtype=torch.int32, device=gpu)
    path = torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    cases = [
        (lambda: svdmlp.copy_pages(c[0], i, i), "caches must have shape"),
        (lambda: svdmlp.copy_pages([], i, i), "nonempty"),
        (lambda: svdmlp.copy_pages([c], i, i), "a cache must have shape"),
        (lambda: svdmlp.copy_pages([c[0], c[1, :5]], i, i), "alike"),
        (lambda: svdmlp.copy_pages([c[0], c[1].transpose(1, 2).contiguous().transpose(1, 2)], i, i), "alike"),
        (lambda: svdmlp.copy_pages([c[0], c[0]], i, i), "overlap"),
        (lambda: svdmlp.copy_pages([c[0, :5], c[0, 1:]], i, i), "overlap"),
        (lambda: svdmlp.copy_pages(c[:1].expand(4, 6, 4, 2, 8), i, i), "overlap"),
        (lambda: svdmlp.copy_pages(c, i, i[:1]), "dst"),
        (lambda: svdmlp.copy_pages(c, i, i, i[:1]), "rows"),
        (lambda: svdmlp.copy_pages(c, i.cpu(), i), "same device"),
        (lambda: svdmlp.copy_pages(c, c.view(torch.int32)[0, 0, 0, 0, :2], i), "overlap"),
        (lambda: svdmlp.copy_pages(c.clone().requires_grad_(), i, i), "no gradient"),
        (lambda: svdmlp.keep_drafts(c, t, ln, path, 65), "1 to 64"),
        (lambda: svdmlp.keep_drafts(c, t, ln, path, 2), "path"),
        (lambda: svdmlp.keep_drafts(c, t, ln, path[:1], 4), "path"),
        (lambda: svdmlp.keep_drafts(c, t[:, :0], ln, path, 4), "block_table"),
        (lambda: svdmlp.keep_drafts(c, t, ln[:1], path, 4), "lengths"),
        (lambda: svdmlp.keep_drafts(c, t.cpu(), ln, path, 4), "same device"),
    ]
    for fn, msg in cases:
        with pytest.raises(ValueError, match=msg):
            fn()
    with pytest.raises(TypeError, match="src"):
        svdmlp.copy_pages(c, i.float(), i)
    with pytest.raises(TypeError, match="supported dtypes"):
        svdmlp.copy_pages(c.half(), i, i)
    assert svdmlp.keep_drafts(c, t[:0], ln[:0], path[:0], 4).shape == (0,)


def test_moves_in_graphs_and_on_streams(gpu):
    """Captured, replayed onto other contents and indices of the same tensors, with eager calls between; and on another stream."""
    g = _gen(8)
    n, pages, page, K, D, drafts = 6, 20, 4, 2, 64, 5
    caches = torch.zeros(n, pages, page, K, D, dtype=BF, device=gpu)
    src, dst = torch.zeros(3, dtype=torch.int32, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu)
    table = torch.arange(10, dtype=torch.int32, device=gpu).view(2, 5)
    ln, path = torch.zeros(2, dtype=torch.int32, device=gpu), torch.zeros(2, 3, dtype=torch.int32, device=gpu)

    def fill(i):
        h = _gen(100 + i)
        caches.copy_(_randn(h, n, pages, page, K, D))
        order = torch.randperm(pages, generator=h).int()
        src.copy_(order[:3]), dst.copy_(order[3:6])
        ln.copy_(torch.tensor([20 - i, 5 + i], dtype=torch.int32))
        path.copy_(torch.tensor([[0, 2, 4], [1 + i % 2, 3, -1]], dtype=torch.int32))

    def call():
        svdmlp.copy_pages(caches, src, dst)
        return svdmlp.keep_drafts(caches, table, ln, path, drafts)

    fill(0)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    side = torch.cuda.Stream()
    for i in range(4):
        fill(i)
        new = call().clone()
        want = caches.clone()
        fill(i)
        graph.replay()
        assert torch.equal(caches, want) and torch.equal(out, new)
        fill(i)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert torch.equal(call(), new)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(caches, want)


def test_page_pool(gpu):
    """Sequences that grow, fork, are cut and freed at random, with compactions between: what each holds is what was written for it."""
    g, rng = _gen(9), random.Random(9)
    n, pages, page, K, D = 4, 40, 4, 1, 8
    caches = torch.zeros(n, pages, page, K, D, dtype=F32, device=gpu)
    pool = svdmlp.PagePool(caches)
    told: dict[int, torch.Tensor] = {}  # (n, tokens, K, D) a sequence
    for step in range(300):
        what = rng.random()
        if what < 0.5 or not told:
            if not told or rng.random() < 0.2:
                told[pool.add()] = torch.zeros(n, 0, K, D)
            seqs = rng.sample(list(told), min(len(told), rng.randint(1, 3)))
            grow = [rng.randint(0, 9) for _ in seqs]
            free = pool.free_pages
            try:
                slots, positions, cu = pool.reserve(seqs, grow)
            except RuntimeError:
                assert pool.free_pages == free
                s = rng.choice(list(told))
                pool.free(s)
                del told[s]
                continue
            rows = torch.randn(n, sum(grow), K, D, generator=g)
            caches.flatten(1, 2)[:, slots] = rows.to(gpu)
            assert cu.tolist() == [sum(grow[:i]) for i in range(len(grow) + 1)]
            at = []
            for s, a, z in zip(seqs, cu.tolist(), cu.tolist()[1:]):
                at += range(told[s].shape[1], told[s].shape[1] + z - a)
                told[s] = torch.cat([told[s], rows[:, a:z]], dim=1)
            assert positions.tolist() == at
        elif what < 0.7:
            s = rng.choice(list(told))
            told[pool.fork(s)] = told[s]
        elif what < 0.8:
            s = rng.choice(list(told))
            length = rng.randint(0, told[s].shape[1])
            pool.trim(s, length)
            told[s] = told[s][:, :length]
        elif what < 0.9:
            s = rng.choice(list(told))
            pool.free(s)
            del told[s]
        else:
            used = pool.compact()
            assert used == pages - pool.free_pages
            held = {int(p) for p in pool.table(list(told))[0].flatten() if p >= 0} if told else set()
            assert held == set(range(used))
        if told and step % 7 == 0:
            table, lengths = pool.table(list(told))
            for row, length, (s, want) in zip(table.tolist(), lengths.tolist(), told.items()):
                assert length == want.shape[1] == pool.length(s) and sum(p >= 0 for p in row) == -(-length // page)
                got = caches[:, [p for p in row if p >= 0]].flatten(1, 2)[:, :length].cpu()
                assert torch.equal(got, want)
    for s in list(told):
        pool.free(s)
    assert pool.free_pages == pages and pool.compact() == 0


def test_page_pool_refusals(gpu):
    pool = svdmlp.PagePool(torch.zeros(2, 3, 4, 1, 8, device=gpu))
    a = pool.add()
    pool.reserve([a], [5])
    b = pool.fork(a)
    with pytest.raises(RuntimeError, match="2 pages needed, 1 of 3 free"):
        pool.reserve([a, b], [1, 4])  # a copy of the shared page, and one more for b
    assert pool.length(a) == pool.length(b) == 5 and pool.free_pages == 1
    with pytest.raises(KeyError, match="no sequence 7"):
        pool.fork(7)
    with pytest.raises(KeyError, match="no sequence"):
        pool.reserve([a, 9], [1, 1])
    with pytest.raises(ValueError, match="not negative"):
        pool.reserve([a], [-1])
    with pytest.raises(ValueError, match="trimmed"):
        pool.trim(a, 6)
    with pytest.raises(ValueError, match="caches"):
        svdmlp.PagePool(torch.zeros(2, 3, device=gpu))
    pool.free(a)
    with pytest.raises(KeyError):
        pool.free(a)
    pool.reserve([b], [3])  # alone again: no copy
    assert pool.free_pages == 1
    slots, positions, cu = pool.reserve([], [])
    assert slots.shape == positions.shape == (0,) and cu.tolist() == [0] and slots.is_cuda and cu.dtype is torch.int32
    slots, positions, cu = pool.reserve([b], [0])
    assert slots.shape == (0,) and cu.tolist() == [0, 0]
    table, lengths = pool.table([])
    assert table.shape == (0, 1) and lengths.shape == (0,) and table.is_cuda
    path = torch.zeros(0, 1, dtype=torch.int32, device=gpu)
    assert svdmlp.keep_drafts(pool.caches, table, lengths, path, 3).shape == (0,)
