"""PagedAttention on the GPU against attention in 64 bits over the values that
the codes stand for, element by element within what its roundings allow
(paged_ref.attention_bound)."""
import pytest
import torch

import paged_ref as ref
from test_gpu_paged_cache import batch_of, make_cache, place

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Problem:
    def __init__(self, rows, *, heads=8, kv_heads=2, dim=128, page=32, block=16, cache="i8", dtype="f16", layout="dense", seed=0, q_scale=2.0, behind=3,
                 garbage=True, spread=0):
        self.rows, self.heads, self.kv, self.dim, self.page, self.cache, self.dtype = rows, heads, kv_heads, dim, page, cache, dtype
        pages = sum(-(-(a + b) // page) for a, b in rows) + 2
        cols = max(-(-(a + b) // page) for a, b in rows) + 2
        self.table, self.offsets, self.lengths = batch_of(rows, page, cols, pages, seed)
        self.sides, self.gpu = [], []
        for i in range(2):
            codes, scales = make_cache(pages, kv_heads, page, dim, block, cache, seed + i)
            if spread:
                g = torch.Generator().manual_seed(seed + 7 + i)
                scales = scales * torch.exp2(torch.randint(-spread, spread + 1, scales.shape, generator=g).float())
            if garbage:  # what lies behind a row's end may be anything: NaN codes, and NaN scales where a whole block does
                for r, (a, b) in enumerate(rows):
                    n = a + b
                    for pos in range(n, -(-n // page) * page):
                        p = int(self.table[r, pos // page])
                        codes.view(torch.uint8)[p, :, pos % page] = 0x7F if pos % 2 else 0xFF
                        if pos % block == 0:
                            scales[p, :, pos % page // block] = float("nan")
                unused = set(range(pages)) - set(self.table.flatten().tolist())
                for p in unused:
                    codes.view(torch.uint8)[p] = 0x7F
                    scales[p] = float("nan")
            self.sides.append(ref.Cache(codes, scales, cache))
            self.gpu.append((place(codes, layout), scales.to(DEV)))
        g = torch.Generator().manual_seed(seed + 5)
        self.q = (torch.randn(int(self.offsets[-1]) + behind, heads, dim, generator=g) * q_scale).to(ref.FLOAT[dtype])
        self.scale = dim ** -0.5

    def args(self):
        (kc, ks), (vc, vs) = self.gpu
        return kc, vc, ks, vs, self.table.to(DEV), self.offsets.to(DEV), self.lengths.to(DEV)

    def run(self, ctx, max_tokens=None, q=None, out=None, stream=None):
        q = self.q.to(DEV) if q is None else q
        out = torch.full_like(self.q, 77.0, device=DEV) if out is None else out
        most = max(b for _, b in self.rows) if max_tokens is None else max_tokens
        ctx.paged_attention(out, q, *self.args(), max(most, 1), self.scale, stream)
        torch.cuda.synchronize()
        return out

    def check(self, out, rows=None, most=None):
        out = out.cpu()
        for r, (had, new) in enumerate(self.rows):
            if rows is not None and r not in rows:
                continue
            lo, n = int(self.offsets[r]), had + new
            k, v = (s.read(self.table[r].tolist(), n) for s in self.sides)
            there = ~k[:, 0, 0].isnan()
            want, mean, size = ref.attention(self.q[lo:lo + new], k, v, self.scale, there)
            got = out[lo:lo + new].double()
            upto = new if most is None else min(new, most)
            bound = ref.attention_bound(want, mean, size, self.dtype, self.dim, n, self.sides[1].top(self.table[r].tolist(), n))
            off = ((got - want).abs() - bound)[:upto]
            assert torch.isfinite(got[:upto]).all(), ("not finite", r)
            assert (off <= 0).all(), (r, had, new, float(off.max()), float(((got - want).abs() / bound)[:upto].max()))
            assert (out[lo + upto:lo + new] == 77.0).all(), ("beyond max_tokens", r)
        assert (out[int(self.offsets[-1]):] == 77.0).all(), "rows behind the last sequence"


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 127, 300, 1025, 5000])
def test_decode_lengths(ctx, cache, dtype, length):
    p = Problem([(length - 1, 1)], cache=cache, dtype=dtype, seed=length)
    p.check(p.run(ctx))


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [16, 32, 64, 80, 96, 112, 128, 144, 160, 176, 192, 208, 240, 256])
def test_head_widths(ctx, cache, dim):
    p = Problem([(70, 1), (0, 3), (200, 2)], cache=cache, dtype="bf16", dim=dim, seed=dim)
    p.check(p.run(ctx))


@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (5, 5), (8, 1), (7, 1), (16, 2), (40, 8), (17, 1), (48, 1), (6, 2)])
@pytest.mark.parametrize("new", [1, 3, 9])
def test_head_groups(ctx, heads, kv_heads, new):
    p = Problem([(50, new), (333, 1), (0, new)], heads=heads, kv_heads=kv_heads, dim=64, cache="e4m3", dtype="f16", seed=heads)
    p.check(p.run(ctx))


@pytest.mark.parametrize("page, block", [(16, 16), (48, 16), (48, 48), (64, 32), (128, 128), (256, 64), (512, 512)])
def test_pages_and_blocks(ctx, page, block):
    p = Problem([(page - 1, 1), (page, 1), (5 * page + 7, 2), (0, 1)], page=page, block=block, dim=64, cache="i8", dtype="bf16", seed=page)
    p.check(p.run(ctx))


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("new", [2, 5, 16, 33, 64, 100, 129, 257, 700])
def test_prompts(ctx, cache, new):
    p = Problem([(0, new), (300, new)], cache=cache, dtype="bf16", heads=8, kv_heads=2, dim=128, seed=new)
    p.check(p.run(ctx))


@pytest.mark.parametrize("dim", [16, 64, 80, 128, 144, 160, 192, 256])
@pytest.mark.parametrize("cache", ["i8", "e4m3"])
def test_prompt_head_widths(ctx, cache, dim):
    p = Problem([(37, 150), (0, 1), (500, 1), (0, 90)], cache=cache, dtype="f16", dim=dim, heads=6, kv_heads=2, seed=dim)
    p.check(p.run(ctx))


def test_mixed_batch_with_empty_rows(ctx):
    rows = [(0, 0), (1000, 1), (200, 180), (5, 0), (0, 1), (0, 64), (64, 0), (2047, 1), (15, 17)]
    for cache in ("i8", "e4m3"):
        p = Problem(rows, cache=cache, dtype="bf16", heads=16, kv_heads=2, dim=64, seed=9)
        p.check(p.run(ctx))


def test_many_rows(ctx):
    rows = [((37 * r) % 90, 0 if r % 13 == 5 else 1) for r in range(600)]
    p = Problem(rows, heads=2, kv_heads=1, dim=16, page=16, cache="e4m3", seed=4)
    p.check(p.run(ctx))


@pytest.mark.parametrize("layout", ["tokens first", "wide"])
@pytest.mark.parametrize("new", [1, 130])
def test_layouts(ctx, layout, new):
    p = Problem([(100, new), (30, 1)], layout=layout, dim=80, heads=6, kv_heads=3, cache="e4m3", dtype="bf16")
    # q is a slice of a fused buffer at an odd place, out lies heads first
    whole = torch.zeros(p.q.shape[0], 11, 81, dtype=p.q.dtype, device=DEV)
    q = whole[:, 2:8, 1:]
    q.copy_(p.q)
    out = torch.full((6, p.q.shape[0], 80), 77.0, dtype=p.q.dtype, device=DEV).transpose(0, 1)
    p.check(p.run(ctx, q=q, out=out))


def test_max_tokens_leaves_the_rest(ctx):
    p = Problem([(10, 5), (40, 2), (0, 90)], dim=64)
    p.check(p.run(ctx, max_tokens=3), most=3)
    p.check(p.run(ctx, max_tokens=1), most=1)
    p.check(p.run(ctx, max_tokens=60), most=60)
    p.check(p.run(ctx, max_tokens=10 ** 6))


@pytest.mark.parametrize("new", [1, 70])
def test_bad_pages_see_nothing(ctx, new):
    """Entries that are no page: their tokens do not exist; a row without a page: zeros."""
    p = Problem([(200, new), (100, new), (0, new)], dim=64, cache="e4m3", page=32)
    p.table[0, 2], p.table[0, 4] = -1, 10 ** 6
    p.table[1, :] = -5
    p.table[2, 0] = 2 ** 31 - 1
    out = p.run(ctx)
    p.check(out)
    lo = int(p.offsets[1])
    assert (out[lo:lo + new] == 0).all()


def test_more_new_tokens_than_the_row_has(ctx):
    """Tokens at places below 0 see nothing."""
    p = Problem([(0, 40), (0, 3)], dim=64)
    p.lengths[0] = 25
    out = p.run(ctx).cpu()
    assert (out[:15] == 0).all()
    k, v = (s.read(p.table[0].tolist(), 25) for s in p.sides)
    want, mean, size = ref.attention(p.q[15:40], k, v, p.scale)
    assert ((out[15:40].double() - want).abs() <= ref.attention_bound(want, mean, size, p.dtype, 64, 25, p.sides[1].top(p.table[0].tolist(), 25))).all()
    p.lengths[0] = -3
    assert (p.run(ctx)[:40] == 0).all()


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("q_scale", [0.0, 1e-6, 60.0, 3000.0])
def test_score_magnitudes(ctx, q_scale, new):
    """From equal weights to a softmax that takes one key only; bf16 carries q of any size."""
    p = Problem([(700, new)], q_scale=q_scale, dim=128, cache="i8", dtype="bf16", seed=2)
    p.check(p.run(ctx))


@pytest.mark.parametrize("new", [1, 50])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-30, 3.0])
def test_factors_of_the_scores(ctx, scale, new):
    p = Problem([(700, new), (0, 3)], dim=64, cache="e4m3", dtype="f16", seed=4)
    p.scale = scale
    p.check(p.run(ctx))


@pytest.mark.parametrize("new", [1, 50])
def test_scales_far_apart(ctx, new):
    """Blocks whose scales differ by up to 2^24, falling and rising along the row, and blocks of zeros."""
    p = Problem([(900, new)], dim=64, cache="e4m3", dtype="bf16", spread=12, q_scale=0.02, seed=3)
    for s, (_, g) in zip(p.sides, p.gpu):
        s.scales[int(p.table[0, 0])] = 0
        s.scales[int(p.table[0, 3])] = 0
        g.copy_(s.scales)
    p.check(p.run(ctx))


@pytest.mark.parametrize("rows", [[(20000, 1)], [(9999, 20)], [(30000, 1), (10, 1), (0, 5), (4000, 2)], [(6000, 200), (0, 3)]], ids=str)
def test_rows_shared_by_workgroups(ctx, rows):
    p = Problem(rows, heads=8, kv_heads=1, dim=64, page=64, block=64, cache="i8", dtype="bf16", seed=8)
    p.check(p.run(ctx))


@pytest.mark.parametrize("new", [1, 60])
def test_two_calls_give_the_same_bits(ctx, new):
    p = Problem([(8000, new), (77, 1)], heads=8, kv_heads=1, dim=128, cache="e4m3", seed=6)
    a, b = p.run(ctx), p.run(ctx)
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("rows", [[(5000, 1), (40, 1)], [(3000, 65), (2, 1)]], ids=str)
def test_captured_and_replayed_with_other_lengths(ctx, rows):
    """One graph serves whatever the index tensors hold at replay; eager calls and synchronisations in between."""
    from operators_amd.ops import PagedAttentionPlan

    p = Problem(rows, heads=8, kv_heads=2, dim=64, cache="e4m3", dtype="bf16", seed=1, garbage=False)
    kc, vc, ks, vs, table, offsets, lengths = p.args()
    q, out = p.q.to(DEV), torch.full_like(p.q, 77.0, device=DEV)
    most = max(b for _, b in rows)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with PagedAttentionPlan(ctx, out, q, kc, vc, ks, vs, table, offsets, lengths, most, p.scale) as plan:
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            plan(out, q, kc, vc, ks, vs, table, offsets, lengths, stream=torch.cuda.current_stream().cuda_stream)
        full = list(rows)
        for cut in (0, 33, 1000, 0):
            p.rows = [(max(0, full[0][0] - cut), full[0][1]), full[1]]
            p.lengths = torch.tensor([a + b for a, b in p.rows], dtype=torch.int32)
            lengths.copy_(p.lengths)
            out.fill_(77.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            p.check(out)
            assert torch.equal(p.run(ctx).view(torch.int16), out.view(torch.int16))


def test_two_calls_at_once_with_workspaces_of_their_own(ctx):
    from operators_amd.ops import PagedAttentionPlan

    ps = [Problem([(9000 + 100 * i, 1)], heads=8, kv_heads=1, dim=128, cache="i8", seed=i) for i in range(3)]
    streams = [torch.cuda.Stream() for _ in ps]
    calls = []
    for p in ps:
        q, out = p.q.to(DEV), torch.full_like(p.q, 77.0, device=DEV)
        a = p.args()
        calls.append((PagedAttentionPlan(ctx, out, q, *a, 1, p.scale), out, q, a))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (plan, out, q, a) in zip(streams, calls):
            plan(out, q, *a, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for p, (plan, out, _, _) in zip(ps, calls):
        p.check(out)
        plan.close()


def test_workspace_and_pointer_refusals(ctx):
    from operators_amd import InfiniopError
    from operators_amd.ops import PagedAttentionPlan

    p = Problem([(30, 1)], dim=64)
    a, q = p.args(), p.q.to(DEV)
    out = torch.empty_like(q)
    with PagedAttentionPlan(ctx, out, q, *a, 1) as plan:
        args = [t.data_ptr() for t in (out, q, *a)]
        call = plan.paged.infiniopPagedAttention
        assert call(plan.desc, plan.workspace.data_ptr(), plan.workspace_size - 1, *args, None) == 6
        assert call(plan.desc, None, plan.workspace_size, *args, None) == 6
        for i in range(len(args)):
            assert call(plan.desc, plan.workspace.data_ptr(), plan.workspace_size, *args[:i], None, *args[i + 1:], None) == 2, i
        for i in (2, 3):
            assert call(plan.desc, plan.workspace.data_ptr(), plan.workspace_size, *args[:i], args[i] + 8, *args[i + 1:], None) == 2, i
        assert call(plan.desc, plan.workspace.data_ptr() + 4, plan.workspace_size, *args, None) == 2
    with pytest.raises(InfiniopError):
        PagedAttentionPlan(ctx, out, q[:, :5], *a, 1)
    torch.cuda.synchronize()


def test_random_problems(ctx):
    import random

    rng = random.Random(77)
    for trial in range(40):
        kv = rng.choice([1, 2, 3, 8])
        rows = [(rng.choice([0, rng.randint(0, 100), rng.randint(0, 3000)]), rng.choice([0, 1, 1, 2, rng.randint(1, 200)])) for _ in range(rng.randint(1, 6))]
        if not any(a + b for a, b in rows):
            rows.append((3, 1))
        page = rng.choice([16, 32, 48, 64, 128])
        p = Problem(rows, heads=kv * rng.choice([1, 2, 5, 8]), kv_heads=kv, dim=16 * rng.randint(1, 16), page=page, block=rng.choice([b for b in (16, 32, 48, 64, 128) if page % b == 0]),
                    cache=rng.choice(["i8", "e4m3"]), dtype=rng.choice(["f16", "bf16"]), layout=rng.choice(["dense", "tokens first", "wide"]), seed=trial)
        print(trial, p.rows, p.heads, p.kv, p.dim, p.page, p.cache, p.dtype, flush=True)
        p.check(p.run(ctx))


@pytest.mark.parametrize("dim", [80, 128, 256])
@pytest.mark.parametrize("new", [4, 5, 8, 9, 16, 17])
def test_between_decoding_and_prompts(ctx, new, dim):
    """32, 40, 64, 72, 128 and 136 query rows of a K/V head, one sequence long enough to be shared, beside single tokens and longer chunks."""
    for rows in ([(3000, new), (10, new), (700, 1), (0, new)], [(5000, new)], [(900, new), (40, 90), (0, 1)]):
        p = Problem(rows, heads=8, kv_heads=1, dim=dim, cache="e4m3", dtype="bf16", seed=new + dim)
        p.check(p.run(ctx))


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [80, 96, 112, 192, 256])
def test_prompts_past_missing_pages(ctx, dim, cache):
    """Pages that are none inside a chunk's keys, in every width that tiles are held in, with page sizes that end inside a tile of 64 keys."""
    for page in (16, 48, 80):
        p = Problem([(300, 131), (5, 77), (0, 200)], heads=4, kv_heads=2, dim=dim, page=page, cache=cache, dtype="f16", seed=dim + page)
        p.table[0, 1], p.table[0, 3], p.table[2, 0] = -1, 10 ** 6, -7
        p.check(p.run(ctx))


class Seen(Problem):
    """A problem whose V scales are changed by `change(scales of v, pages of the rows)`, held to a bound that takes of each token's
    keys only those that it sees, by the weights that they have."""

    def __init__(self, rows, change, **more):
        super().__init__(rows, garbage=False, **more)
        side, (_, gpu) = self.sides[1], self.gpu[1]
        change(side.scales, self.table)
        gpu.copy_(side.scales)

    def check(self, out, least=0.0):
        """least: a V scale smaller than this part of the largest may count as that.  What this adds is rounded with the rest: to bf16
        (2^-8 of it), its weight to fp16 (2^-11) and by its scale's exponent (2^-16), less than 2^-7 of it together."""
        out = out.cpu()
        assert torch.isfinite(out.float()).all()
        for r, (had, new) in enumerate(self.rows):
            lo, n = int(self.offsets[r]), had + new
            if not new:
                continue
            pages = self.table[r].tolist()
            k, v = (s.read(pages, n) for s in self.sides)
            want, mean, size = ref.attention(self.q[lo:lo + new], k, v, self.scale)
            side = self.sides[1]
            scales = torch.stack([side.scales[pages[j // side.page], :, j % side.page // side.block] for j in range(n)])
            share = ref.largest_share(self.q[lo:lo + new], k, scales, self.cache, self.scale)
            bound = ref.seen_bound(want, mean, size, self.dtype, self.dim, n, share) + least * float(scales.max()) * ref.MOST[self.cache] * (1 + 2.0 ** -7)
            off = (out[lo:lo + new].double() - want).abs()
            assert (off <= bound).all(), (r, had, new, float((off / bound).max()), int((off > bound).any(-1).any(-1).nonzero()[0]))


def times(exponent, start, end=None):
    """The V scales of blocks start .. end of every row, by a power of two."""
    def change(scales, table):
        per = scales.shape[2]
        for row in table.tolist():
            held = [(p, b) for p in row if p >= 0 for b in range(per)]
            for p, b in held[start:end]:
                scales[p, :, b] *= 2.0 ** exponent
    return change


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("exponent, dim", [(-26, 64), (-34, 64), (-60, 64), (-34, 256), (-60, 256)])
@pytest.mark.parametrize("rows, heads, kv_heads", [([(14, 5), (30, 2)], 4, 2), ([(0, 12), (14, 4)], 16, 2), ([(14, 150), (0, 300)], 8, 2), ([(15, 70)], 1, 1),
                                                   ([(14, 40)], 8, 2), ([(0, 1100)], 4, 2)], ids=str)
def test_values_far_smaller_than_the_unseen(ctx, rows, heads, kv_heads, exponent, dim, cache):
    """The first block's values are smaller than all later ones by far, which the first tokens do not see."""
    p = Seen(rows, times(exponent, 0, 1), heads=heads, kv_heads=kv_heads, dim=dim, cache=cache, dtype="bf16", seed=heads)
    p.check(p.run(ctx))


@pytest.mark.parametrize("new", [1, 20, 100])
@pytest.mark.parametrize("exponent", [30, 60])
@pytest.mark.parametrize("k_scale", [1.0, 2.0 ** -6])
def test_values_far_smaller_than_the_unweighted(ctx, k_scale, exponent, new):
    """A block of huge values whose weight is next to nothing, before, between and behind the others."""
    for block in (0, 7, 20):
        p = Seen([(340, new)], times(exponent, block, block + 1), heads=8, kv_heads=2, dim=64, cache="e4m3", dtype="bf16", seed=block)
        k, (codes, _) = p.sides[0], p.gpu[0]
        page, at = int(p.table[0, block // 2]), block % 2 * 16
        low = torch.full((16,), -240.0).to(torch.float8_e4m3fn).view(torch.uint8)[0]
        k.codes.view(torch.uint8)[page, :, at:at + 16] = low  # all products far below 0
        k.scales[page, :, block % 2] = k_scale
        codes.view(torch.uint8).copy_(k.codes.view(torch.uint8))
        p.gpu[0][1].copy_(k.scales)
        p.q = p.q.abs()
        p.check(p.run(ctx))


@pytest.mark.parametrize("rows", [[(3100, 1), (2050, 3)], [(2900, 200)], [(1000, 60), (2100, 40), (3000, 33)], [(0, 1100)]], ids=str)
@pytest.mark.parametrize("steps", [(-120, -60, 0), (0, -60, -120), (-90, 0, -90), (-40, -39, 0)])
@pytest.mark.parametrize("q_scale", [0.0, 1.0, 40.0])
def test_values_that_jump_along_the_row(ctx, q_scale, steps, rows):
    """V scales that rise and fall by up to 2^120 every 1024 keys, with weights from equal ones to nearly one."""
    def change(scales, table):
        for i, e in enumerate(steps):
            times(e, i * 64, None if i == 2 else i * 64 + 64)(scales, table)
    p = Seen(rows, change, heads=2, kv_heads=1, dim=64, cache="e4m3", dtype="bf16", seed=11, q_scale=q_scale)
    p.check(p.run(ctx), least=2.0 ** -80)


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("exponent", [-135, -100, 100, 118])
@pytest.mark.parametrize("rows", [[(40, 1), (0, 3)], [(9000, 1)], [(300, 90)], [(5000, 60), (3, 1)]], ids=str)
def test_values_near_the_ends_of_the_type(ctx, rows, exponent, cache):
    """V scales from subnormal numbers up to values of 2^120: results of 16 bits hold them, and so does all on the way."""
    p = Seen(rows, times(exponent, 0), heads=8, kv_heads=1, dim=128, cache=cache, dtype="bf16", seed=5)
    p.check(p.run(ctx))


@pytest.mark.parametrize("new", [1, 50])
def test_scales_of_zero(ctx, new):
    """A V scale of 0 stands for zeros whatever the codes, all along a row and in its first and last blocks; the weights count."""
    for start, end in ((0, None), (0, 20), (30, None)):
        def change(scales, table):
            pages = [p for p in table[0].tolist() if p >= 0]
            for i in range(start, len(pages) * 2 if end is None else end):
                scales[pages[i // 2], :, i % 2] = 0
        p = Seen([(900, new)], change, heads=8, kv_heads=2, dim=64, cache="i8", dtype="bf16", seed=2)
        out = p.run(ctx)
        p.check(out)
        if start == 0 and end is None:
            assert (out[:new] == 0).all()


# ---- more than 64 rows: the units are found by a scan over the workgroup ------------
@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("count", [65, 257, 300])
def test_many_rows_some_shared_by_workgroups(ctx, count, cache):
    rows = [((37 * r) % 90, 0 if r % 13 == 5 else 1) for r in range(count)]
    rows[3], rows[40], rows[count - 1] = (6000, 1), (2500, 2), (9000, 1)
    p = Problem(rows, heads=8, kv_heads=1, dim=64, page=64, block=16, cache=cache, dtype="bf16", seed=count)
    p.check(p.run(ctx))


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("count, dim", [(65, 64), (300, 80), (600, 64), (300, 256)])
def test_many_rows_with_chunks(ctx, count, dim, cache):
    """Chunks of more than 64 query rows among them, long enough to be cut, with both kernels and both joins."""
    rows = [((37 * r) % 90, 0 if r % 13 == 5 else 1) for r in range(count)]
    rows[0], rows[30], rows[50], rows[count - 2] = (3000, 70), (0, 90), (4000, 1), (1500, 33)
    p = Problem(rows, heads=4, kv_heads=1, dim=dim, page=32, block=32, cache=cache, dtype="f16", seed=count + dim)
    p.check(p.run(ctx))


def test_many_rows_replayed_with_other_lengths(ctx):
    from operators_amd.ops import PagedAttentionPlan

    rows = [((37 * r) % 90, 1) for r in range(130)]
    rows[7], rows[100] = (5000, 1), (700, 40)
    p = Problem(rows, heads=4, kv_heads=2, dim=64, cache="e4m3", dtype="bf16", seed=1, garbage=False)
    kc, vc, ks, vs, table, offsets, lengths = p.args()
    q, out = p.q.to(DEV), torch.full_like(p.q, 77.0, device=DEV)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with PagedAttentionPlan(ctx, out, q, kc, vc, ks, vs, table, offsets, lengths, 40, p.scale) as plan:
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            plan(out, q, kc, vc, ks, vs, table, offsets, lengths, stream=torch.cuda.current_stream().cuda_stream)
        full = list(rows)
        for cut in (0, 600, 4500, 0):
            p.rows = [(max(0, had - cut) if had > 90 else had, new) for had, new in full]
            p.lengths = torch.tensor([a + b for a, b in p.rows], dtype=torch.int32)
            lengths.copy_(p.lengths)
            out.fill_(77.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            p.check(out)


@pytest.mark.parametrize("rows, heads, kv_heads, dim", [([(0, 32)], 8, 1, 64), ([(511, 1)], 8, 2, 128), ([(1000, 1), (1000, 1)], 8, 1, 64), ([(2000, 40), (2000, 40)], 8, 1, 64),
                                                        ([(700, 300)], 8, 1, 128), ([(513, 130), (60, 70)], 16, 2, 256), ([(400, 3)] * 70, 4, 2, 64)], ids=str)
def test_workspace_is_enough(ctx, rows, heads, kv_heads, dim):
    """What lies behind the workspace stays as it is: with tables just as long as the rows, also where all offsets name the same tokens."""
    from operators_amd.ops import PagedAttentionPlan

    p = Problem(rows, heads=heads, kv_heads=kv_heads, dim=dim, page=16, cache="i8", dtype="bf16", seed=1, garbage=False)
    p.table = p.table[:, :max(-(-(a + b) // 16) for a, b in rows)].contiguous()
    a, q = p.args(), p.q.to(DEV)
    out = torch.full_like(q, 77.0)
    with PagedAttentionPlan(ctx, out, q, *a, max(b for _, b in rows), p.scale) as plan:
        size = plan.workspace_size
        plan.workspace = torch.full((size + (16 << 20),), 0x5A, dtype=torch.uint8, device=DEV)
        plan(out, q, *a)
        torch.cuda.synchronize()
        p.check(out)
        assert (plan.workspace[size:] == 0x5A).all()
        most = rows[0][1]
        a[5].copy_(torch.tensor([0] + [0 if i % 2 else most for i in range(len(rows))], dtype=torch.int32))
        a[6].fill_(2 ** 31 - 1)
        plan(out, q, *a)
        torch.cuda.synchronize()
        assert (plan.workspace[size:] == 0x5A).all()
