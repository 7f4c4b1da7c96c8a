"""PageTableUpdate and PageTableCompact on the GPU against lists (paged_ref), and
the operators of the paged cache together as a server runs them."""
import random

import pytest
import torch

import paged_ref as ref
from test_gpu_paged_cache import make_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def build(rng, rows, cols, pages, page, most, fork=0.3):
    """A consistent table: rows of up to `most` pages, some of them forks of a part of another row."""
    free = list(range(pages))
    rng.shuffle(free)
    table, lengths, refs = [], [], [0] * pages
    for r in range(rows):
        n = rng.randint(0, min(most, cols) * page)
        have = []
        if table and rng.random() < fork:
            other = rng.randrange(r)
            have = [p for p in table[other][:rng.randint(0, min(-(-n // page), -(-lengths[other] // page)))]]
        while len(have) < -(-n // page) and free:
            have.append(free.pop())
        n = min(n, len(have) * page)
        have = have[:-(-n // page)]
        for p in have:
            refs[p] += 1
        table.append(have + [rng.choice([-1, -1, 12345678, 3])] * (cols - len(have)))  # what is behind a row's pages does not count
        lengths.append(n)
    return table, lengths, refs


def run_update(ctx, table, lengths, refs, source, grow, page, in_place=False):
    rows = len(table)
    t, n, c = ints(table), ints(lengths), ints(refs)
    nt, nn, nc = (t, n, c) if in_place else (torch.full_like(t, 99), torch.full_like(n, 99), torch.full_like(c, 99))
    pairs, result = torch.full((rows, 2), 99, dtype=torch.int32, device=DEV), ints([99, 99])
    ctx.page_table_update(nt, nn, nc, pairs, result, t, n, c, ints(source), ints(grow), page)
    got = [x.cpu().tolist() for x in (nt, nn, nc, pairs, result)]
    if not in_place:
        assert t.cpu().tolist() == table and n.cpu().tolist() == lengths and c.cpu().tolist() == refs
    return got


def run_compact(ctx, table, lengths, refs, page, room, in_place=False):
    t, n, c = ints(table), ints(lengths), ints(refs)
    nt, nc = (t, c) if in_place else (torch.full_like(t, 99), torch.full_like(c, 99))
    pairs, result = torch.full((room, 2), 99, dtype=torch.int32, device=DEV), ints([99, 99])
    ctx.page_table_compact(nt, nc, pairs, result, t, n, c, page)
    return [x.cpu().tolist() for x in (nt, nc, pairs, result)]


# one workgroup with 4 and with 8 entries a lane, and several launches
SIZES = [(1, 1, 1, 1, 1), (1, 5, 9, 16, 4), (7, 6, 60, 16, 5), (64, 20, 1500, 3, 15), (300, 8, 2500, 16, 6), (200, 30, 6000, 16, 20), (513, 40, 20000, 64, 30), (5000, 9, 40000, 16, 6)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rows, cols, pages, page, most", SIZES)
def test_update(ctx, rows, cols, pages, page, most, in_place):
    rng = random.Random(rows * 7 + cols)
    for trial in range(4 if rows < 1000 else 1):
        table, lengths, refs = build(rng, rows, cols, pages, page, most)
        kind = trial % 4
        source = [[r, rng.randrange(rows), rng.choice([r, r, -1, rng.randrange(rows)]), rows - 1 - r][kind] for r in range(rows)]
        grow = [rng.choice([0, 1, 1, page, rng.randint(0, 2 * page), -4]) for _ in range(rows)]
        assert run_update(ctx, table, lengths, refs, source, grow, page, in_place) == list(ref.update(table, lengths, refs, source, grow, page)), trial


@pytest.mark.parametrize("large", [False, True])
def test_update_edges(ctx, large):
    """Rows that name no row, pages that run out by one, rows too wide, entries that are no page, lengths out of range."""
    rows, cols, page = 6, 4, 16
    pages = 30000 if large else 12
    filler = pages - 12  # all in use
    refs = [1, 1, 2, 1, 0, 0, 0, 1, 0, 1, 1, 1] + [1] * filler
    table = [[0, 2, -1, -1], [1, 2, 3, -1], [7, -1, -1, -1], [-9, 99999999, 5, 5], [9, 10, 11, -1], [-1, -1, -1, -1]]
    lengths = [20, 33, 16, 0, 48, 0]
    same = list(range(rows))

    def check(source, grow, lengths=lengths, table=table, refs=refs):
        for in_place in (False, True):
            got = run_update(ctx, table, lengths, refs, source, grow, page, in_place)
            assert got == list(ref.update(table, lengths, refs, source, grow, page))
        return got[4]

    assert check(same, [0] * 6) == [0, 0]
    assert check(same, [1, 0, 0, 0, 0, 0]) == [0, 0]           # a shared last page: copied
    assert check(same, [0, 0, 1, 0, 0, 0]) == [0, 0]           # a full one: a fresh page
    assert check(same, [0, 0, 0, 64, 0, 0]) == [0, 0]          # four fresh pages, all there are
    assert check(same, [1, 0, 0, 64, 0, 0]) == [1, 0]          # one too few
    assert check(same, [0, 0, 0, 64, 0, 2 ** 31 - 1]) == [0, 1]  # wider than the table
    assert check(same, [0, 0, 49, 0, 17, 0]) == [0, 2]
    assert check([-1] * 6, [0] * 6) == [0, 0]
    assert check([-1, 6, 7, 10 ** 9, -2 ** 31, 2 ** 31 - 1], [0] * 6) == [0, 0]
    assert check([0] * 6, [1] * 6)[1] == 0                     # one row six times, each with a copy of its last page
    assert check([4, 4, 4, 4, 4, -1], [-3, 0, 0, 1, 1, 5]) == [0, 0]
    # a length beyond the table or below 0, an entry that is no page in a row's last place, and in one that is freed
    assert check(same, [1] * 6, lengths=[-4, 33, 10 ** 9, 2, 48, 0]) == [0, 1]
    assert check([0, 1, 2, 5, 4, 5], [0, 0, 0, 1, 0, 1], lengths=[20, 33, 16, 20, 48, 0]) == [0, 0]
    assert check([3, 1, 2, 3, 4, 5], [1, 0, 0, 1, 0, 0], lengths=[20, 33, 16, 20, 48, 0]) == [0, 0]


@pytest.mark.parametrize("pages", [5, 30000])
def test_update_of_no_rows(ctx, pages):
    """A batch without rows: the counts stay, and nothing lacks."""
    none, refs = torch.zeros(0, dtype=torch.int32, device=DEV), ints([p % 3 for p in range(pages)])
    table, pairs = torch.zeros(0, 4, dtype=torch.int32, device=DEV), torch.zeros(0, 2, dtype=torch.int32, device=DEV)
    for out in (torch.full_like(refs, 99), refs):
        result = ints([99, 99])
        ctx.page_table_update(table, none, out, pairs, result, table, none, refs, none, none, 16)
        assert result.tolist() == [0, 0] and out.tolist() == [p % 3 for p in range(pages)]


def test_update_that_wants_2_30_pages(ctx):
    """Pages of one token and a row that grows by 2^30 of them: it is not too wide, the pages lack."""
    cols = (1 << 30) + 3
    table = torch.full((1, cols), -1, dtype=torch.int32, device=DEV)
    refs, length, result, pairs = ints([0] * 100), ints([0]), ints([9, 9]), ints([[9, 9]])
    for grow, want in (((1 << 30) - 1, [(1 << 30) - 101, 0]), (1 << 30, [(1 << 30) - 100, 0]), ((1 << 30) + 1, [(1 << 30) - 99, 0]), ((1 << 30) + 4, [0, 1])):
        ctx.page_table_update(table, length, refs, pairs, result, table, length, refs, ints([0]), ints([grow]), 1)
        assert result.tolist() == want, grow
        assert length.tolist() == [0] and pairs.tolist() == [[-1, -1]] and int(refs.sum()) == 0


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rows, cols, pages, page, most", SIZES)
def test_compact(ctx, rows, cols, pages, page, most, in_place):
    rng = random.Random(rows + cols * 3)
    for trial in range(3 if rows < 1000 else 1):
        table, lengths, refs = build(rng, rows, cols, pages, page, most)
        room = pages // 2 + trial
        want = ref.compact(table, lengths, refs, page, room)
        assert run_compact(ctx, table, lengths, refs, page, room, in_place) == list(want), trial
        if not in_place:  # a compact table stays as it is
            again = run_compact(ctx, want[0], lengths, want[1], page, room)
            assert again[0] == want[0] and again[1] == want[1] and again[3][1] == 0


@pytest.mark.parametrize("pages", [1, 2, 63, 64, 65, 1023, 1024, 1025, 8192, 8193, 9216, 20000])
def test_compact_edges(ctx, pages):
    room = pages // 2
    for refs in ([0] * pages, [1] * pages, [0] * (pages // 2) + [2] * (pages - pages // 2), [1] * (pages // 2) + [0] * (pages - pages // 2),
                 [p % 2 for p in range(pages)], [0] * (pages - 1) + [5]):
        table, lengths = [[p, pages + 5, -1] for p in range(min(pages, 40))], [3] * min(pages, 40)
        assert run_compact(ctx, table, lengths, refs, 2, room) == list(ref.compact(table, lengths, refs, 2, room))


def test_pools_of_more_chunks_than_workgroups(ctx):
    """1.3 million pages: a workgroup goes through several chunks of 1024."""
    pages, page, rows, cols = 1300000, 16, 40, 400
    g = torch.Generator().manual_seed(9)
    refs = (torch.rand(pages, generator=g) < 0.6).int()
    refs[100000:1200000] = 1  # the free ones are far apart
    free = (refs == 0).nonzero().flatten()
    table, lengths = torch.full((rows, cols), -1, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32)
    high = (refs[1250000:] > 0).nonzero().flatten()[:rows * 3].view(rows, 3) + 1250000
    table[:, :3], lengths[:] = high.int(), 3 * page
    grow = 390 * page  # 15600 fresh pages
    assert rows * 390 <= len(free)
    t, n, c, result = table.to(DEV), lengths.to(DEV), refs.to(DEV), ints([9, 9])
    pairs = torch.empty(rows, 2, dtype=torch.int32, device=DEV)
    ctx.page_table_update(t, n, c, pairs, result, t, n, c, ints(list(range(rows))), ints([grow] * rows), page)
    assert result.tolist() == [0, 0] and (pairs == -1).all() and (n == 393 * page).all()
    want = table.clone()
    want[:, 3:393] = free[:rows * 390].view(rows, 390).int()
    assert torch.equal(t.cpu(), want)
    refs[free[:rows * 390]] = 1
    assert torch.equal(c.cpu(), refs)
    moves = torch.empty(pages // 2, 2, dtype=torch.int32, device=DEV)
    ctx.page_table_compact(t, c, moves, result, t, n, c, page)
    used = int((refs > 0).sum())
    above, below = (refs[used:] > 0).nonzero().flatten() + used, (refs[:used] == 0).nonzero().flatten()
    assert result.tolist() == [used, len(above)] and len(above) == len(below)
    assert torch.equal(moves[:len(above)].cpu(), torch.stack([above, below], 1).int()) and (moves[len(above):] == -1).all()
    goes = torch.arange(pages)
    goes[above] = below
    assert torch.equal(t.cpu(), torch.where(want >= 0, goes[want.clamp(min=0).long()].int(), want))
    assert (c[:used] == 1).all() and (c[used:] == 0).all()


def test_captured_update_and_compact(ctx):
    from operators_amd.ops import PageTableCompactPlan, PageTableUpdatePlan

    for rows, cols, pages in ((16, 8, 300), (400, 30, 30000)):
        page, rng = 4, random.Random(5)
        table, lengths, refs = build(rng, rows, cols, pages, page, cols // 2)
        t, n, c, source, grow = ints(table), ints(lengths), ints(refs), ints(list(range(rows))), ints([1] * rows)
        pairs, result = ints([[0, 0]] * rows), ints([0, 0])
        moves, moved = ints([[0, 0]] * (pages // 2)), ints([0, 0])
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        up = PageTableUpdatePlan(ctx, t, n, c, pairs, result, t, n, c, source, grow, page)
        co = PageTableCompactPlan(ctx, t, c, moves, moved, t, n, c, page)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            up(t, n, c, pairs, result, t, n, c, source, grow, stream=torch.cuda.current_stream().cuda_stream)
            co(t, c, moves, moved, t, n, c, stream=torch.cuda.current_stream().cuda_stream)
        for replay in range(4):
            s = [rng.choice([r, r, r, -1, rng.randrange(rows)]) for r in range(rows)]
            source.copy_(ints(s))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            table, lengths, refs, p, res = ref.update(table, lengths, refs, s, [1] * rows, page)
            table, refs, m, mv = ref.compact(table, lengths, refs, page, pages // 2)
            got = [x.cpu().tolist() for x in (t, n, c, pairs, result, moves, moved)]
            assert got == [table, lengths, refs, p, res, m, mv], replay
        up.close()
        co.close()


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_serving_steps(ctx, cache, dtype):
    """Prompts, decoding, forks, rows that end and begin, a compaction: two layers' caches through one page table.  Each row's
    tokens are kept apart, as a cache of its own that is appended to in the same steps, and attention is held to that."""
    rng = random.Random(13)
    rows, cols, pages, page, block, heads, kv, dim = 6, 8, 30, 32, 16, 8, 2, 64
    layers = 2
    t, n, c = ints([[-1] * cols] * rows), ints([0] * rows), ints([0] * pages)
    pairs, result, moves, moved = ints([[0, 0]] * rows), ints([0, 0]), ints([[0, 0]] * (pages // 2)), ints([0, 0])
    caches = []
    for i in range(layers):
        k, ks = make_cache(pages, kv, page, dim, block, cache, i)
        caches.append([x.to(DEV) for x in (k, k, ks, ks)])
    blank = lambda: [[ref.Cache(torch.zeros(cols, kv, page, dim).to(ref.CODE[cache]), torch.zeros(cols, kv, page // block), cache) for _ in range(2)] for _ in range(layers)]  # noqa: E731
    mine, lengths = [blank() for _ in range(rows)], [0] * rows
    g = torch.Generator().manual_seed(1)
    copied = 0
    for step in range(14):
        source = list(range(rows))
        grow = [1] * rows
        if step == 0:
            grow = [rng.randint(1, 60) for _ in range(rows)]
        elif step % 3 == 1:
            source[rng.randrange(rows)] = rng.randrange(rows)
            source[rng.randrange(rows)] = rng.randrange(rows)
        elif step % 5 == 3:
            r = rng.randrange(rows)
            source[r], grow[r] = -1, rng.randint(2, 50)
        grow[rng.randrange(rows)] = 0
        ctx.page_table_update(t, n, c, pairs, result, t, n, c, ints(source), ints(grow), page)
        assert result.cpu().tolist() == [0, 0]
        before = [(mine[s], lengths[s]) if s >= 0 else (blank(), 0) for s in source]
        mine = [[[ref.Cache(x.codes.clone(), x.scales.clone(), cache) for x in layer] for layer in m] for m, _ in before]
        lengths = [a + b for (_, a), b in zip(before, grow)]
        assert n.cpu().tolist() == lengths
        copied += int((pairs[:, 0] >= 0).sum())
        offsets = [0]
        for b in grow:
            offsets.append(offsets[-1] + b)
        for layer in range(layers):
            kc, vc, ks, vs = caches[layer]
            ctx.kv_cache_copy(kc, vc, ks, vs, pairs)
            qkv = torch.randn(offsets[-1], heads + 2 * kv, dim, generator=g).to(ref.FLOAT[dtype])
            x = qkv.to(DEV)
            ctx.kv_cache_append(kc, vc, ks, vs, x[:, heads:heads + kv], x[:, heads + kv:], t, ints(offsets), n)
            out = torch.full((offsets[-1], heads, dim), 77.0, dtype=x.dtype, device=DEV)
            ctx.paged_attention(out, x[:, :heads], kc, vc, ks, vs, t, ints(offsets), n, max(grow))
            out = out.cpu().double()
            for r in range(rows):
                lo, hi = offsets[r], offsets[r + 1]
                if lo == hi:
                    continue
                for i, side in enumerate(mine[r][layer]):
                    side.append(list(range(cols)), lengths[r] - grow[r], qkv[lo:hi, heads + i * kv:heads + (i + 1) * kv])
                k, v = (side.read(list(range(cols)), lengths[r]) for side in mine[r][layer])
                want, mean, size = ref.attention(qkv[lo:hi, :heads], k, v, dim ** -0.5)
                bound = ref.attention_bound(want, mean, size, dtype, dim, lengths[r], mine[r][layer][1].top(list(range(cols)), lengths[r]))
                assert ((out[lo:hi] - want).abs() <= bound).all(), (step, layer, r)
        if step in (5, 9):
            ctx.page_table_compact(t, c, moves, moved, t, n, c, page)
            for kc, vc, ks, vs in caches:
                ctx.kv_cache_copy(kc, vc, ks, vs, moves)
            used = moved.cpu().tolist()[0]
            assert (c[:used] > 0).all() and (c[used:] == 0).all()
    assert copied > 0
