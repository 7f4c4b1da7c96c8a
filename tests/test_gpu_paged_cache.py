"""KVCacheAppend and KVCacheCopy on the GPU against the plain statements of
tests/paged_ref.py: codes and scales exactly (each is defined by single fp32
steps), and against the values themselves in 64 bits."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make_cache(pages, heads, page, dim, block, cache, seed, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(pages, heads, page, dim, generator=g)
    scales = (torch.rand(pages, heads, page // block, generator=g) + 0.5) * 2.0 ** -5
    if cache == "e4m3":
        scales = torch.exp2(torch.floor(torch.log2(scales)) - 2)
    codes = ref.nearest(x.view(pages, heads, page // block, -1) / scales[..., None], cache).view(pages, heads, page, dim)
    return codes, scales


def same(got, want):
    return torch.equal(got.cpu().contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


def place(t, layout):
    """A tensor on the GPU in the named layout, as a view with the logical shape [pages, heads, page, ...]."""
    t = t.to(DEV)
    if layout == "dense":
        return t.clone()
    if layout == "tokens first":  # [pages, page, heads, dim]
        return t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    if layout == "wide":  # rows of codes with room behind them, every other page of a pool
        pages, heads, page, dim = t.shape
        whole = torch.zeros((pages, 2, heads, page, dim + 32), dtype=torch.uint8, device=DEV)
        whole.random_(0, 255)
        view = whole.view(t.dtype)[:, 1, :, :, 16:16 + dim]
        view.view(torch.uint8).copy_(t.view(torch.uint8))
        return view
    raise ValueError(layout)


def batch_of(rows, page, cols, pages, seed):
    """rows: (tokens before, new tokens).  Every row has pages of its own, in no order."""
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(rows), cols), -1, dtype=torch.int32)
    for r, (had, new) in enumerate(rows):
        for c in range(-(-(had + new) // page)):
            table[r, c] = perm.pop()
    offsets = [0]
    for _, new in rows:
        offsets.append(offsets[-1] + new)
    return table, torch.tensor(offsets, dtype=torch.int32), torch.tensor([a + b for a, b in rows], dtype=torch.int32)


def check_append(ctx, rows, *, heads=2, dim=64, page=32, block=16, cache="i8", dtype="f16", layout="dense", pages=None, seed=0, fill=None, behind=0, stream=None):
    cols = max(-(-(a + b) // page) for a, b in rows) + 1
    pages = pages or sum(-(-(a + b) // page) for a, b in rows) + 3
    table, offsets, lengths = batch_of(rows, page, cols, pages, seed)
    tokens = int(offsets[-1]) + behind
    g = torch.Generator().manual_seed(seed + 1)
    both = (torch.randn(tokens, 2 * heads + 1, dim, generator=g) * torch.exp2(torch.randint(-6, 7, (tokens, 1, 1), generator=g).float())).to(ref.FLOAT[dtype])
    if fill is not None:
        fill(both)
    qkv = both.to(DEV)
    sides, args = [], []
    for i in range(2):
        codes, scales = make_cache(pages, heads, page, dim, block, cache, seed + 2 + i)
        sides.append(ref.Cache(codes.clone(), scales.clone(), cache))
        args.append((place(codes, layout), scales.to(DEV)))
    x = [qkv[:, 1:1 + heads], qkv[:, 1 + heads:]]
    (kc, ks), (vc, vs) = args
    ctx.kv_cache_append(kc, vc, ks, vs, x[0], x[1], table.to(DEV), offsets.to(DEV), lengths.to(DEV), stream)
    torch.cuda.synchronize()
    for i, side in enumerate(sides):
        part = both[:, 1 + i * heads:1 + (i + 1) * heads]
        for r, (had, new) in enumerate(rows):
            side.append(table[r].tolist(), had, part[offsets[r]:offsets[r + 1]])
        assert same(args[i][1], side.scales), ("scales", i)
        assert same(args[i][0], side.codes), ("codes", i, int((args[i][0].cpu().view(torch.uint8) != side.codes.view(torch.uint8)).sum()))
    return sides, both, table, offsets


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [
    [(0, 1)], [(5, 1)], [(15, 1), (16, 1), (17, 1), (0, 16)], [(0, 200)], [(7, 130), (0, 0), (64, 0), (31, 2), (100, 33)],
], ids=str)
def test_append_lengths(ctx, cache, dtype, rows):
    check_append(ctx, rows, cache=cache, dtype=dtype, seed=len(rows))


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dim, heads, page, block", [(16, 1, 16, 16), (80, 3, 48, 16), (96, 5, 64, 32), (128, 8, 64, 64), (112, 2, 128, 128), (256, 1, 256, 256), (192, 2, 96, 48)])
def test_append_shapes(ctx, cache, dim, heads, page, block):
    check_append(ctx, [(3, 70), (page - 1, 2), (0, block), (block + 1, 2 * page + 5)], cache=cache, dtype="bf16", dim=dim, heads=heads, page=page, block=block, seed=dim)


@pytest.mark.parametrize("layout", ["tokens first", "wide"])
@pytest.mark.parametrize("cache", ["i8", "e4m3"])
def test_append_layouts(ctx, layout, cache):
    check_append(ctx, [(9, 40), (0, 3)], cache=cache, layout=layout, dim=80, heads=3)


def test_append_many_rows(ctx):
    # more rows than a workgroup has lanes, most of one token, some of none
    rows = [((7 * r) % 50, (0 if r % 11 == 3 else 1 + (r % 29 == 0) * 20)) for r in range(700)]
    check_append(ctx, rows, cache="e4m3", dim=16, heads=1, page=16)


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
def test_append_is_within_half_a_step(ctx, cache):
    """Fresh blocks: every value within half a step of its code, in 64 bits (int8: half a scale; e4m3: 2^-4 of the value, or
    half of 2^-9 of the scale below its normal numbers), beside the roundings of the scale, its inverse and the product
    (2^-24 each, of a code up to 127)."""
    sides, both, table, offsets = check_append(ctx, [(0, 100)], cache=cache, dtype="bf16", seed=11)
    for i, side in enumerate(sides):
        x = both[:, 1 + 2 * i:3 + 2 * i].double()
        y = side.read(table[0].tolist(), 100)
        step = torch.stack([side.scales[int(table[0, p // 32]), :, p % 32 // 16] for p in range(100)]).double()[..., None]
        bound = step / 2 if cache == "i8" else torch.maximum(x.abs() * 2.0 ** -4, step * 2.0 ** -10)
        assert ((x - y).abs() <= bound + 128 * step * 3 * 2.0 ** -24).all()


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
def test_append_extremes(ctx, cache):
    """Infinities, NaN, zeros, numbers near the ends of bf16 and below 2^-96, signed zeros; ties between codes."""
    def fill(x):
        x[0] = 0
        x[1] = -0.0
        x[2, :, 3] = float("inf")
        x[3, :, 4] = -float("inf")
        x[4, :, 5] = float("nan")
        x[16:32] = 1e-38
        x[17, 1] = -1.1754944e-38
        x[32:48] *= 2.0 ** 100
        x[33, 2, 1] = 3.3e38
        x[48:64] = 0
        x[64:80] = 127.0 if cache == "i8" else 448.0
        x[65] = torch.arange(64) - 31.5  # halves
        x[66] = 63.5
        x[80:96] = float("inf")
        x[96:112] = float("nan")
        x[112:] *= 2.0 ** -90

    check_append(ctx, [(0, 120)], cache=cache, dtype="bf16", fill=fill)


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
def test_append_one_by_one(ctx, cache):
    """A block that grows token by token, each call on what the last one left, among them growing, equal and falling tops."""
    heads, dim, page, block = 2, 64, 32, 32
    g = torch.Generator().manual_seed(3)
    x = torch.randn(40, heads, dim, generator=g) * torch.exp2(torch.randint(-9, 9, (40, 1, 1), generator=g).float())
    x[20] = 0
    x = x.to(torch.bfloat16)
    table = torch.tensor([[2, 0, -1]], dtype=torch.int32)
    codes, scales = make_cache(3, heads, page, dim, block, cache, 5)
    side = ref.Cache(codes.clone(), scales.clone(), cache)
    kc, ks, vc, vs = codes.to(DEV), scales.to(DEV), codes.to(DEV), scales.to(DEV)
    for t in range(40):
        one = x[t:t + 1].to(DEV)
        ctx.kv_cache_append(kc, vc, ks, vs, one, one, table.to(DEV), torch.tensor([0, 1], dtype=torch.int32, device=DEV),
                            torch.tensor([t + 1], dtype=torch.int32, device=DEV))
        side.append(table[0].tolist(), t, x[t:t + 1])
        torch.cuda.synchronize()
        assert same(ks, side.scales) and same(kc, side.codes) and same(vc, side.codes), t


def test_append_bad_pages_and_lengths(ctx):
    """Entries that are no page are passed over; more new tokens than the row is long: its last; tokens behind the last row,
    and rows whose offsets fall: none."""
    heads, dim, page, block, pages = 1, 32, 16, 16, 6
    codes, scales = make_cache(pages, heads, page, dim, block, "i8", 1)
    x = torch.randn(60, heads, dim).to(torch.float16)
    table = torch.tensor([[4, -1, 99], [2, 1, -7], [3, 0, 5]], dtype=torch.int32)
    kc, ks = codes.to(DEV), scales.to(DEV)
    vc, vs = codes.to(DEV), scales.to(DEV)
    offsets = torch.tensor([0, 40, 58, 50], dtype=torch.int32)
    lengths = torch.tensor([40, 10, 20], dtype=torch.int32)  # row 1: 18 new tokens, 10 places; row 2: offsets fall
    ctx.kv_cache_append(kc, vc, ks, vs, x.to(DEV), x.to(DEV), table.to(DEV), offsets.to(DEV), lengths.to(DEV))
    torch.cuda.synchronize()
    side = ref.Cache(codes.clone(), scales.clone(), "i8")
    side.append(table[0].tolist(), 0, x[:40])
    side.append(table[1].tolist(), 0, x[48:58])
    assert same(kc, side.codes) and same(ks, side.scales) and same(vc, side.codes)
    # a length beyond the table, and below 0
    lengths = torch.tensor([10 ** 9, -5, 0], dtype=torch.int32)
    offsets = torch.tensor([0, 3, 7, 9], dtype=torch.int32)
    table = torch.tensor([[0, 1, 2], [3, 3, 3], [4, 4, 4]], dtype=torch.int32)
    ctx.kv_cache_append(kc, vc, ks, vs, x.to(DEV), x.to(DEV), table.to(DEV), offsets.to(DEV), lengths.to(DEV))
    torch.cuda.synchronize()
    side.append(table[0].tolist(), 45, x[:3])
    assert same(kc, side.codes) and same(ks, side.scales)


def test_append_on_another_stream_and_captured(ctx):
    from operators_amd.ops import KVCacheAppendPlan

    table, offsets, lengths = batch_of([(10, 5), (0, 40)], 32, 3, 8, 0)
    codes, scales = make_cache(8, 2, 32, 64, 16, "e4m3", 1)
    caches = [t.to(DEV) for t in (codes, codes, scales, scales)]
    index = [t.to(DEV) for t in (table, offsets, lengths)]
    x = torch.randn(45, 2, 64, device=DEV).to(torch.float16)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with KVCacheAppendPlan(ctx, *caches, x, x, *index) as plan:
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            plan(*caches, x, x, *index, stream=torch.cuda.current_stream().cuda_stream)
        for replay in range(3):
            x.copy_(torch.randn(45, 2, 64, device=DEV) * (replay + 1))
            for t, s in zip(caches, (codes, codes, scales, scales)):
                t.view(torch.uint8).copy_(s.to(DEV).view(torch.uint8))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = ref.Cache(codes.clone(), scales.clone(), "e4m3")
            want.append(table[0].tolist(), 10, x.cpu()[:5])
            want.append(table[1].tolist(), 0, x.cpu()[5:])
            assert same(caches[0], want.codes) and same(caches[1], want.codes) and same(caches[3], want.scales)


def test_append_of_nothing(ctx):
    check_append(ctx, [(3, 0)], behind=0)
    codes, scales = (t.to(DEV) for t in make_cache(2, 1, 16, 16, 16, "i8", 0))
    x = torch.zeros(0, 1, 16, dtype=torch.float16, device=DEV)
    one = torch.zeros(1, 1, 16, dtype=torch.float16, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    ctx.kv_cache_append(codes, codes, scales, scales, x, x, torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV),
                        torch.zeros(1, dtype=torch.int32, device=DEV))
    ctx.kv_cache_append(codes, codes, scales, scales, one, one, torch.zeros(0, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), none)


def test_append_many_rows_of_several_tokens(ctx):
    # more than two tokens a row and more rows than a workgroup has lanes: units are found by a scan, several rows a lane
    rows = [((7 * r) % 50, (0 if r % 5 == 2 else 3 + (r % 29 == 0) * 40)) for r in range(300)]
    assert sum(b for _, b in rows) > 2 * len(rows)
    check_append(ctx, rows, cache="e4m3", dim=16, heads=1, page=16)
    check_append(ctx, rows, cache="i8", dim=32, heads=3, page=32, block=32, dtype="bf16", behind=7)


def test_append_more_than_1024_rows(ctx):
    # plain decoding of more rows than a token's row is looked up among
    rows = [((7 * r) % 50, 0 if r % 11 == 3 else 1) for r in range(1100)]
    check_append(ctx, rows, cache="e4m3", dim=16, heads=1, page=16)
    check_append(ctx, [((3 * r) % 20, 0 if r % 2 else 2) for r in range(1100)], cache="i8", dim=16, heads=1, page=16, dtype="bf16")


@pytest.mark.parametrize("page, block, dim", [(32, 32, 64), (256, 256, 64)])
@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("scale", [1e-45, 1e-40, 2.0 ** -127, 2.0 ** -110])
def test_append_onto_scales_of_next_to_nothing(ctx, scale, cache, page, block, dim):
    """Older tokens whose scale has no finite inverse, or is smaller than new values that count as 0: zeros stay zeros and what
    is beyond the codes becomes the largest."""
    for value in (0.0, 2.0 ** -97, 1e-38, float("inf"), float("nan")):
        codes, scales = make_cache(2, 2, page, dim, block, cache, 3)
        scales.fill_(scale)
        x = torch.zeros(3, 2, dim, dtype=torch.bfloat16)
        x[1, 0, ::2], x[1, 0, 1::4], x[2, 1, 5] = value, -value, value
        sides = [ref.Cache(codes.clone(), scales.clone(), cache) for _ in range(2)]
        kc, vc, ks, vs = codes.to(DEV), codes.to(DEV), scales.to(DEV), scales.to(DEV)
        ctx.kv_cache_append(kc, vc, ks, vs, x.to(DEV), -x.to(DEV), torch.tensor([[1]], dtype=torch.int32, device=DEV),
                            torch.tensor([0, 3], dtype=torch.int32, device=DEV), torch.tensor([8], dtype=torch.int32, device=DEV))
        torch.cuda.synchronize()
        for side, new, c, s in zip(sides, (x, -x), (kc, vc), (ks, vs)):
            side.append([1], 5, new)
            assert same(s, side.scales) and same(c, side.codes), value


# ---- KVCacheCopy ---------------------------------------------------------------
@pytest.mark.parametrize("layout", ["dense", "tokens first", "wide"])
@pytest.mark.parametrize("dim, heads, page, block, pages", [(16, 1, 16, 16, 5), (80, 3, 48, 16, 9), (128, 8, 64, 32, 20), (256, 2, 128, 128, 6)])
def test_copy(ctx, layout, dim, heads, page, block, pages):
    k, ks = make_cache(pages, heads, page, dim, block, "i8", 1)
    v, vs = make_cache(pages, heads, page, dim, block, "i8", 2)
    kc, vc, ksc, vsc = place(k, layout), place(v, layout), ks.to(DEV), vs.to(DEV)
    pairs = torch.tensor([[-1, 2], [0, pages - 1], [3, -1], [3, 1], [pages, 2], [0, pages], [-1, -1], [3, 4]], dtype=torch.int32)
    ctx.kv_cache_copy(kc, vc, ksc, vsc, pairs.to(DEV))
    torch.cuda.synchronize()
    for src, dst in ((0, pages - 1), (3, 1), (3, 4)):
        for t in (k, v, ks, vs):
            t[dst] = t[src]
    assert same(kc, k) and same(vc, v) and same(ksc, ks) and same(vsc, vs)


def test_copy_long_sparse_list(ctx):
    pages, count = 300, 20000
    k, ks = make_cache(pages, 1, 16, 32, 16, "e4m3", 1)
    kc, ksc = k.to(DEV), ks.to(DEV)
    vc, vsc = k.to(DEV), ks.to(DEV)
    pairs = torch.full((count, 2), -1, dtype=torch.int32)
    g = torch.Generator().manual_seed(0)
    where = torch.randperm(count, generator=g)[:100]
    pairs[where, 0] = torch.arange(100, dtype=torch.int32)
    pairs[where, 1] = torch.arange(100, 200, dtype=torch.int32)
    ctx.kv_cache_copy(kc, vc, ksc, vsc, pairs.to(DEV))
    torch.cuda.synchronize()
    k[100:200], ks[100:200] = k[:100].clone(), ks[:100].clone()
    assert same(kc, k) and same(vc, k) and same(ksc, ks) and same(vsc, ks)
    ctx.kv_cache_copy(kc, vc, ksc, vsc, pairs[:0].to(DEV))


def test_offsets_beyond_2_31(ctx):
    """Pages 17 MiB apart in a pool of 3.4 GiB: the last ones lie past 2^31 bytes."""
    pages, step = 200, 17 << 20
    pool = torch.zeros(pages * step, dtype=torch.int8, device=DEV)
    kc = pool.as_strided((pages, 1, 16, 32), (step, 512, 32, 1))
    vc = pool[1024:].as_strided((pages, 1, 16, 32), (step, 512, 32, 1))
    ks, vs = torch.zeros(pages, 1, 1, device=DEV), torch.zeros(pages, 1, 1, device=DEV)
    x = torch.randn(16, 1, 32).to(torch.float16)
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=DEV)
    span = torch.tensor([0, 16], dtype=torch.int32, device=DEV)
    ctx.kv_cache_append(kc, vc, ks, vs, x.to(DEV), x.to(DEV), table, span, span[1:].contiguous())
    ctx.kv_cache_copy(kc, vc, ks, vs, torch.tensor([[pages - 1, 150]], dtype=torch.int32, device=DEV))
    out = torch.empty(16, 1, 32, dtype=torch.float16, device=DEV)
    ctx.paged_attention(out, x.to(DEV), kc, vc, ks, vs, torch.tensor([[150]], dtype=torch.int32, device=DEV), span, span[1:].contiguous(), 16)
    torch.cuda.synchronize()
    side = ref.Cache(torch.zeros(1, 1, 16, 32, dtype=torch.int8), torch.zeros(1, 1, 1), "i8")
    side.append([0], 0, x)
    for t, s in ((kc, ks), (vc, vs)):
        for p in (150, pages - 1):
            assert same(t[p], side.codes[0]) and same(s[p], side.scales[0])
    y = side.read([0], 16)
    want, mean, size = ref.attention(x, y, y, 32 ** -0.5)
    assert ((out.cpu().double() - want).abs() <= ref.attention_bound(want, mean, size, "f16", 32, 16, side.top([0], 16))).all()
