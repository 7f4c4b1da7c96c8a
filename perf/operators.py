"""The operators of a paged key/value cache held in 8 bits, as a serving loop calls them, in their plain form (elementary torch operations) and through
this package: appending new tokens, attention over the pages, copying pages, and the two operations on the page table (update and compaction).

A cache is [pages, kv_heads, page, dim] codes (int8 or e4m3) and [pages, kv_heads, page / block] fp32 scales, one for each block of tokens and head.
Row r of a batch has its pages in table[r], `lengths[r]` tokens in all, of which the last offsets[r + 1] - offsets[r] are the call's own.
"""
import math
import random

import torch

own = False

# ---------------------------------------------------------------- cases


def listed():
    return [
        # a chat's next token: the smallest attention, 1000 cached tokens, small pages
        {"name": "decode, one sequence", "op": "attention", "rows": 1, "tokens": 1, "chunk": 1, "low": 1000, "high": 1000, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "block": 16, "dtype": "bf16", "cache": "e4m3"},
        # a batch that decodes: 48 sequences of very different age
        {"name": "decode, 48 ragged", "op": "attention", "rows": 48, "tokens": 1, "chunk": 1, "low": 100, "high": 131072, "heads": 64, "kv_heads": 8,
         "dim": 128, "page": 64, "block": 64, "dtype": "bf16", "cache": "i8"},
        # a whole prompt, the matrix units' case
        {"name": "prompt of 4096", "op": "attention", "rows": 1, "tokens": 1, "chunk": 4096, "low": 4096, "high": 4096, "heads": 64, "kv_heads": 8,
         "dim": 128, "page": 64, "block": 64, "dtype": "bf16", "cache": "e4m3"},
        # a chunk of a prompt that goes along with eight decoding sequences; an odd head width and odd lengths
        {"name": "chunk beside decodes", "op": "attention", "rows": 9, "tokens": 1, "chunk": 500, "low": 301, "high": 20011, "heads": 40, "kv_heads": 8,
         "dim": 80, "page": 32, "block": 16, "dtype": "f16", "cache": "i8"},
        # one new token of each of 256 sequences into its page
        {"name": "append, decode of 256", "op": "append", "rows": 256, "tokens": 1, "chunk": 1, "low": 50, "high": 2000, "kv_heads": 8,
         "dim": 128, "page": 16, "block": 16, "dtype": "bf16", "cache": "e4m3"},
        # prompts: one chunk of 8192 tokens beside shorter ones, that begin and end inside blocks
        {"name": "append, prompts", "op": "append", "rows": 5, "tokens": 77, "chunk": 8192, "low": 77, "high": 9001, "kv_heads": 8,
         "dim": 128, "page": 64, "block": 64, "dtype": "f16", "cache": "i8"},
        # the copies on write of one decoding step
        {"name": "copy, on write", "op": "copy", "pages": 4096, "moves": 24, "kv_heads": 8, "dim": 128, "page": 16, "block": 16, "cache": "e4m3"},
        # the moves of a compaction
        {"name": "copy, compaction", "op": "copy", "pages": 6000, "moves": 2000, "kv_heads": 8, "dim": 128, "page": 64, "block": 32, "cache": "e4m3"},
        # beam search over 8 prompts with 8 beams: each row continues one of its group
        {"name": "update, beams", "op": "update", "rows": 64, "cols": 64, "pages": 4096, "page": 16, "low": 100, "high": 1000, "kind": "beams"},
        # a large server's step: rows that end, rows that begin with a prompt, rows that decode
        {"name": "update, serving", "op": "update", "rows": 1024, "cols": 512, "pages": 262144, "page": 64, "low": 10, "high": 30000, "kind": "serving"},
        # compaction of a small and of a large pool
        {"name": "compact, small", "op": "compact", "rows": 32, "cols": 128, "pages": 4096, "page": 16, "low": 20, "high": 2000, "kind": "beams"},
        {"name": "compact, large", "op": "compact", "rows": 512, "cols": 512, "pages": 262144, "page": 64, "low": 10, "high": 30000, "kind": "serving"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "append", "copy", "update", "compact"])
    page = rng.choice([16, 32, 64, 128])
    block = rng.choice([b for b in (16, 32, 64, 128) if b <= page])
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 80, 96, 112, 128, 192, 256])
    dtype, cache = rng.choice(["bf16", "f16"]), rng.choice(["e4m3", "i8"])
    if op == "attention":
        kind = rng.choice(["decode", "decode", "prompt", "mixed"])
        rows = _log(rng, 1, 64) if kind == "decode" else 1 if kind == "prompt" else rng.randint(2, 12)
        high = _log(rng, 40, 131072 if rows < 8 else 16384) if kind == "decode" else _log(rng, 100, 4000)
        chunk = 1 if kind == "decode" else high if kind == "prompt" else rng.randint(2, high)
        tokens = rng.choice([1, 1, 1, 2, 5]) if kind == "decode" else 1
        chunk = tokens if kind == "decode" else chunk
        case = {"op": op, "rows": rows, "tokens": tokens, "chunk": chunk, "low": rng.randint(max(tokens, high // 9), high), "high": high,
                "heads": kv * rng.choice([1, 4, 5, 7, 8]), "kv_heads": kv, "dim": dim, "page": page, "block": block, "dtype": dtype, "cache": cache}
        # no larger than the listed ones, in what the operator does and in what its plain form holds
        while (work(case)["flops"] > 2.7e11 or work(case)["bytes"] > 1.8e9 or rows * case["high"] * kv * dim > 6e9
               or rows * case["chunk"] * case["high"] * case["heads"] > 6e9):
            case["high"] = case["high"] * 2 // 3
            case["chunk"] = min(case["chunk"], case["high"])
            case["low"] = min(case["low"], case["high"])
        return case
    if op == "append":
        rows = _log(rng, 1, 256)
        tokens = 1 if rng.random() < 0.5 else rng.randint(1, max(1, 4096 // rows))
        chunk = tokens if rng.random() < 0.5 else _log(rng, 1, 4096)
        high = max(tokens, chunk) + rng.randint(0, 1000)
        return {"op": op, "rows": rows, "tokens": tokens, "chunk": chunk, "low": rng.randint(tokens, high), "high": high, "kv_heads": kv, "dim": dim,
                "page": page, "block": block, "dtype": dtype, "cache": cache}
    if op == "copy":
        pages = _log(rng, 40, 6000)
        return {"op": op, "pages": pages, "moves": _log(rng, 1, pages // 3), "kv_heads": kv, "dim": dim, "page": page, "block": block, "cache": "e4m3"}
    rows, kind = _log(rng, 8, 1024) // 8 * 8, rng.choice(["beams", "serving"])
    high = rng.randint(200, 8000)
    cols = high // page + 20
    return {"op": op, "rows": rows, "cols": cols, "pages": rng.randint(rows * cols // 2, rows * cols) + 64, "page": page, "low": rng.randint(10, high), "high": high,
            "kind": kind}


# ---------------------------------------------------------------- inputs

_DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _lengths(case):
    """Lengths of the rows, from the case alone: spread evenly over the logarithm, the longest first, none shorter than its new tokens."""
    n, low, high = case["rows"], case["low"], case["high"]
    got = [int(round(high * (low / high) ** (i / max(1, n - 1)))) for i in range(n)]
    return [max(v, t) for v, t in zip(got, _tokens(case))] if "tokens" in case else got


def _tokens(case):
    return [case["chunk"]] + [case["tokens"]] * (case["rows"] - 1)


def _normal(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _pool(g, case, pages):
    """A cache whose every page holds what earlier tokens left there: codes and scales of normal values with a spread of magnitudes from block to block."""
    kv, page, dim, block = case["kv_heads"], case["page"], case["dim"], case["block"]
    codes, scales = [], []
    for _ in range(2):
        x = _normal(g, (pages, kv, page // block, block * dim), torch.bfloat16)
        spread = torch.exp2(torch.rand((pages, kv, page // block), generator=g, device="cuda") * 2 - 1)
        top = x.abs().amax(-1).float() * spread
        scale = top / 127 if case["cache"] == "i8" else _power(top)
        x = x.mul_((spread / scale).unsqueeze(-1))
        c = x.clamp_(-127, 127).round_().to(torch.int8) if case["cache"] == "i8" else x.clamp_(-448, 448).to(torch.float8_e4m3fn)
        codes.append(c.view(pages, kv, page, dim))
        scales.append(scale.contiguous())
        del x
    return codes[0], codes[1], scales[0], scales[1]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _table(g, lengths, page, cols, pages):
    """Every row's pages, taken in no order from the pool; -1 behind them."""
    need = [-(-v // page) for v in lengths]
    perm = torch.randperm(pages, generator=g, device="cuda")
    need_t = torch.tensor(need, device="cuda")
    first = torch.cumsum(need_t, 0) - need_t
    col = torch.arange(cols, device="cuda")
    at = (first[:, None] + col).clamp(max=pages - 1)
    return torch.where(col < need_t[:, None], perm[at], torch.full_like(at, -1)).to(torch.int32)


def _context():
    from operators_amd.ops import Context

    if not hasattr(_context, "kept"):
        _context.kept = Context(0)
    return _context.kept


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    if op in ("attention", "append"):
        lengths, tokens, page = _lengths(case), _tokens(case), case["page"]
        cols = max(-(-v // page) for v in lengths) + 2
        pages = sum(-(-v // page) for v in lengths) + 7
        s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"] = _pool(g, case, pages)
        s["table"] = _table(g, lengths, page, cols, pages)
        s["lengths"] = _ints(lengths)
        s["offsets"] = _ints([sum(tokens[:i]) for i in range(len(tokens) + 1)])
        total, dt = sum(tokens), _DT[case["dtype"]]
        if op == "attention":
            s["q"] = (_normal(g, (total, case["heads"], case["dim"])) * 2).to(dt)
            s["out"] = torch.empty_like(s["q"])
        else:
            # k and v lie side by side in the projection's output
            both = (_normal(g, (total, 2 * case["kv_heads"], case["dim"])) * 1.5).to(dt)
            s["k"], s["v"] = both[:, : case["kv_heads"]], both[:, case["kv_heads"]:]
    elif op == "copy":
        s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"] = _pool(g, case, case["pages"])
        perm = torch.randperm(case["pages"], generator=g, device="cuda")[: 2 * case["moves"]]
        s["pairs"] = torch.stack([perm[: case["moves"]], perm[case["moves"]:]], 1).to(torch.int32).contiguous()
    else:
        rng = random.Random(seed)
        rows, cols, pages, page = case["rows"], case["cols"], case["pages"], case["page"]
        lengths = _lengths(case)
        # what the pool has no room for is cut: two thirds of it are in use, a few pages a row are left
        room = max(page, 2 * pages // (3 * rows) * page)
        lengths = [min(v, (cols - 4) * page, room) for v in lengths]
        rng.shuffle(lengths)
        table = _table(g, lengths, page, cols, pages)
        if case["kind"] == "beams":  # the rows of a group of 8 share the pages of their first row's first half
            lead = torch.arange(rows, device="cuda") // 8 * 8
            need = (_ints(lengths) + page - 1) // page
            shared = torch.minimum(need, need[lead]) // 2
            col = torch.arange(cols, device="cuda")
            table = torch.where(col < shared[:, None], table[lead], table)
            source = [r // 8 * 8 + rng.randrange(8) for r in range(rows)]
            grow = [1] * rows
        else:
            source = [(-1 if rng.random() < 0.05 else rng.randrange(rows) if rng.random() < 0.02 else r) for r in range(rows)]
            grow = [rng.choice([0, 1, 1, 1]) if v >= 0 else rng.randint(1, 3 * page) for v in source]
        s["table"], s["lengths"] = table.contiguous(), _ints(lengths)
        held = torch.arange(cols, device="cuda") < ((s["lengths"] + page - 1) // page)[:, None]
        s["refcount"] = torch.zeros(pages, dtype=torch.int32, device="cuda").scatter_add_(0, table.clamp(min=0).flatten().long(), held.int().flatten())
        s["new_table"], s["new_refcount"] = torch.empty_like(s["table"]), torch.empty_like(s["refcount"])
        s["result"] = torch.zeros(2, dtype=torch.int32, device="cuda")
        if op == "update":
            s["source"], s["grow"], s["new_lengths"] = _ints(source), _ints(grow), torch.empty_like(s["lengths"])
            s["pairs"] = torch.empty((rows, 2), dtype=torch.int32, device="cuda")
        else:
            s["pairs"] = torch.empty((pages // 2, 2), dtype=torch.int32, device="cuda")
    if own:
        from operators_amd import ops

        plan = {"attention": ops.PagedAttentionPlan, "append": ops.KVCacheAppendPlan, "copy": ops.KVCacheCopyPlan, "update": ops.PageTableUpdatePlan,
                "compact": ops.PageTableCompactPlan}[op]
        more = {"attention": {"max_tokens": max(_tokens(case)) if op == "attention" else 0}, "update": {"page_size": case["page"]},
                "compact": {"page_size": case["page"]}}.get(op, {})
        s["plan"] = plan(_context(), *[s[k] for k in _ARGS[op]], **more)
    return s


#: The tensors of a call, in the order of the package's plans.
_ARGS = {
    "attention": ("out", "q", "k_cache", "v_cache", "k_scale", "v_scale", "table", "offsets", "lengths"),
    "append": ("k_cache", "v_cache", "k_scale", "v_scale", "k", "v", "table", "offsets", "lengths"),
    "copy": ("k_cache", "v_cache", "k_scale", "v_scale", "pairs"),
    "update": ("new_table", "new_lengths", "new_refcount", "pairs", "result", "table", "lengths", "refcount", "source", "grow"),
    "compact": ("new_table", "new_refcount", "pairs", "result", "table", "lengths", "refcount"),
}


# ---------------------------------------------------------------- one pass


def run(s):
    op = s["case"]["op"]
    if own:
        s["plan"](*[s[k] for k in _ARGS[op]], stream=torch.cuda.current_stream().cuda_stream)
    else:
        {"attention": _attention, "append": _append, "copy": _copy, "update": _update, "compact": _compact}[op](s)
    if op == "attention":
        return s["out"]
    if op == "append" and s["case"]["cache"] == "i8":
        # what int8 holds, as the values that it stands for
        return {"k": _values(s["k_cache"], s["k_scale"], s["k"].dtype), "v": _values(s["v_cache"], s["v_scale"], s["v"].dtype), "k_scale": s["k_scale"],
                "v_scale": s["v_scale"]}
    if op in ("append", "copy"):
        return {k: s[k] for k in ("k_cache", "v_cache", "k_scale", "v_scale")}
    return {k: s[k] for k in ("new_table", "new_refcount", "pairs", "result") + (("new_lengths",) if op == "update" else ())}


def _values(codes, scale, dtype):
    pages, kv, page, dim = codes.shape
    return torch.mul(codes.view(pages, kv, scale.shape[2], -1), scale.unsqueeze(-1)).to(dtype)


def _attention(s):
    c = s["case"]
    rows, kv, group, page, dim, block = c["rows"], c["kv_heads"], c["heads"] // c["kv_heads"], c["page"], c["dim"], c["block"]
    most, long = max(_tokens(c)), max(_lengths(c))
    cols = -(-long // page)
    at = s["table"][:, :cols].clamp(min=0).long()

    def whole(codes, scale):
        x = codes.view(torch.uint8)[at].view(codes.dtype).float().view(rows, cols, kv, page // block, block * dim)
        return (x * scale[at].unsqueeze(-1)).view(rows, cols, kv, page, dim).permute(0, 2, 1, 3, 4).reshape(rows, kv, cols * page, dim)

    first, length = s["offsets"][:-1].long(), s["lengths"].long()
    count = s["offsets"][1:].long() - first
    i, j = torch.arange(most, device="cuda"), torch.arange(cols * page, device="cuda")
    q = s["q"][(first[:, None] + i).clamp(max=s["q"].shape[0] - 1)].float()  # [rows, most, heads, dim]
    q = q.view(rows, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(rows, kv, group * most, dim)
    x = torch.matmul(q, whole(s["k_cache"], s["k_scale"]).transpose(2, 3).contiguous()) / math.sqrt(dim)
    seen = (j <= (length - count)[:, None, None] + i[:, None]) & (i[:, None] < count[:, None, None])  # [rows, most, keys]
    x = x.view(rows, kv, group, most, -1).masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
    total = x.sum(-1, keepdim=True)
    y = torch.matmul(x.view(rows, kv, group * most, -1), whole(s["v_cache"], s["v_scale"])).view(rows, kv, group, most, dim)
    y = (y / total.masked_fill(total == 0, 1)).permute(0, 3, 1, 2, 4).reshape(rows * most, kv * group, dim)
    token = torch.arange(s["q"].shape[0], device="cuda")
    row = torch.searchsorted(s["offsets"][1:].long(), token, right=True)
    s["out"].copy_(y[row * most + token - first[row]])


def _power(top):
    """The smallest power of two by which the largest magnitude fits e4m3 (448 = 1.75 * 2^8)."""
    m, e = torch.frexp(top)  # top = m 2^e, 0.5 <= m < 1
    return torch.where(top > 0, torch.ldexp(torch.ones_like(top), e - 9 + (m > 0.875).int()), torch.zeros_like(top))


def _append(s):
    c = s["case"]
    page, block, i8 = c["page"], c["block"], c["cache"] == "i8"
    per = page // block
    first, length = s["offsets"][:-1].long(), s["lengths"].long()
    begin = length - (s["offsets"][1:].long() - first)
    token = torch.arange(s["k"].shape[0], device="cuda")
    row = torch.searchsorted(s["offsets"][1:].long(), token, right=True)
    pos = begin[row] + token - first[row]
    where_ = s["table"][row, pos // page].long()
    key = where_ * per + pos % page // block  # the block that a token falls into
    # the block each row's first new token falls into, and whether it held tokens before
    old_page = s["table"].gather(1, (begin // page)[:, None])[:, 0].long().clamp(min=0)
    old_key, held = old_page * per + begin % page // block, (begin % block != 0) & (length > begin)
    for codes, scale, x in ((s["k_cache"], s["k_scale"], s["k"]), (s["v_cache"], s["v_scale"], s["v"])):
        x = x.float()
        pages, kv, _, dim = codes.shape
        x = torch.where(x.isnan(), 0.0, x)
        a = torch.where(x.isinf(), 0.0, x.abs()).amax(-1)  # [tokens, kv]
        top = torch.zeros((pages * per, kv), device="cuda").scatter_reduce_(0, key[:, None].expand(-1, kv), a, "amax")
        top = torch.where(top < 2.0 ** -96, 0.0, top)
        new = top / 127 if i8 else _power(top)
        flat = scale.transpose(1, 2).reshape(pages * per, kv)  # by block
        before = flat[old_key] * held[:, None]  # [rows, kv]
        new = new.scatter_reduce(0, old_key[:, None].expand(-1, kv), before, "amax")
        # the tokens that were there before, to the block's new scale
        now = new[old_key]
        ratio = torch.where((now > before) & held[:, None], before / torch.where(now > 0, now, 1.0), 1.0)
        by_block = codes.view(torch.uint8).view(pages, kv, per, block * dim)
        was = by_block[old_page, :, begin % page // block]  # [rows, kv, block * dim]
        y = was.view(codes.dtype).float() * ratio[:, :, None]
        y = (y.round().to(torch.int8) if i8 else y.to(torch.float8_e4m3fn)).view(torch.uint8)
        mine = (torch.arange(block, device="cuda")[None, :] < (begin % block)[:, None]) & held[:, None]
        y = torch.where(mine[:, None, :, None], y.view(-1, kv, block, dim), was.view(-1, kv, block, dim)).view(-1, kv, block * dim)
        # (a row without such tokens writes its block back as it was)
        head = torch.arange(kv, device="cuda")[None, :]
        by_block.index_put_((old_page[:, None], head, (begin % page // block)[:, None]), y)
        # the new tokens
        scale.index_put_((where_[:, None], head, (pos % page // block)[:, None]), new[key])
        most = 127.0 if i8 else 448.0
        inverse = torch.where(new > 0, 1 / torch.where(new > 0, new, 1.0), 0.0)
        y = (x * inverse[key][:, :, None]).clamp(-most, most)
        y = (y.round().to(torch.int8) if i8 else y.to(torch.float8_e4m3fn)).view(torch.uint8)
        codes.view(torch.uint8).index_put_((where_[:, None], head, (pos % page)[:, None]), y)


def _copy(s):
    src, dst = s["pairs"][:, 0].long(), s["pairs"][:, 1].long()
    for k in ("k_cache", "v_cache"):
        codes = s[k].view(torch.uint8)
        codes[dst] = codes[src]
    for k in ("k_scale", "v_scale"):
        s[k][dst] = s[k][src]


def _update(s):
    rows, cols, page, pages = s["table"].shape + (s["case"]["page"], s["refcount"].shape[0])
    table, lengths, source, grow = s["table"].long(), s["lengths"].long(), s["source"].long(), s["grow"].long()
    row, col = torch.arange(rows, device="cuda"), torch.arange(cols, device="cuda")
    kept = (source >= 0) & (source < rows)
    at = source.clamp(0, rows - 1)
    length = torch.where(kept, lengths[at], 0)
    count = (length + page - 1) // page
    changed = source != row
    now = torch.where((col < count[:, None]), table[at], -1)
    refs = s["refcount"].long()
    less = changed[:, None] & (col < ((lengths + page - 1) // page)[:, None])
    more = changed[:, None] & (col < count[:, None])
    refs = refs.scatter_add(0, table.clamp(min=0).flatten(), -less.long().flatten()).scatter_add_(0, now.clamp(min=0).flatten(), more.long().flatten())
    last = now.gather(1, (count - 1).clamp(min=0)[:, None])[:, 0]
    copied = (grow > 0) & (length % page != 0) & (refs[last.clamp(min=0)] > 1)
    longer = length + grow
    wanted = (longer + page - 1) // page
    copied &= wanted <= cols
    need = torch.where(wanted > cols, 0, wanted - count + copied)
    free = refs == 0
    missing = need.sum() - free.sum()
    wide = (wanted > cols).sum()
    fits = (missing <= 0) & (wide == 0)
    rank = torch.cumsum(free, 0) - 1
    lowest = torch.zeros(pages + 1, dtype=torch.long, device="cuda").scatter_(0, torch.where(free, rank, pages), torch.arange(pages, device="cuda"))
    first = torch.cumsum(need, 0) - need
    fresh = lowest[(first[:, None] + copied[:, None] + col - count[:, None]).clamp(0, pages - 1)]
    own_copy = lowest[first.clamp(0, pages - 1)]
    new = torch.where(changed[:, None], now, table)
    added = fits & (col >= count[:, None]) & (col < wanted[:, None])
    new = torch.where(added, fresh, new)
    moved = fits & copied
    at_last = moved[:, None] & (col == (count - 1)[:, None])
    new = torch.where(at_last, own_copy[:, None], new)
    refs = refs.scatter_add_(0, new.clamp(min=0).flatten(), (added | at_last).long().flatten()).scatter_add_(0, last.clamp(min=0), -moved.long())
    s["new_table"].copy_(new)
    s["new_refcount"].copy_(refs)
    s["new_lengths"].copy_(torch.where(fits, longer, length))
    s["pairs"].copy_(torch.where(moved[:, None], torch.stack([last, own_copy], 1), -1))
    s["result"].copy_(torch.stack([missing.clamp(min=0), wide]))


def _compact(s):
    cols, page, pages, most = s["table"].shape[1], s["case"]["page"], s["refcount"].shape[0], s["pairs"].shape[0]
    refs, index = s["refcount"], torch.arange(s["refcount"].shape[0], device="cuda")
    used = refs > 0
    count = used.sum()
    high, low = used & (index >= count), ~used & (index < count)
    rank_high, rank_low = torch.cumsum(high, 0) - 1, torch.cumsum(low, 0) - 1
    target = torch.zeros(pages + 1, dtype=torch.long, device="cuda").scatter_(0, torch.where(low, rank_low, pages), index)
    goes = torch.where(high, target[rank_high.clamp(min=0)], index)
    pairs = torch.full((most + 1, 2), -1, dtype=torch.long, device="cuda")
    at = torch.where(high, rank_high, most)[:, None].expand(-1, 2)
    pairs.scatter_(0, at, torch.stack([index, goes], 1))
    s["pairs"].copy_(pairs[:most])
    held = torch.arange(cols, device="cuda") < ((s["lengths"] + page - 1) // page)[:, None]
    s["new_table"].copy_(torch.where(held, goes[s["table"].clamp(min=0).long()].int(), s["table"]))
    s["new_refcount"].zero_().scatter_add_(0, goes, refs)
    s["result"].copy_(torch.stack([count, high.sum()]))


# ---------------------------------------------------------------- work


def work(case):
    op = case["op"]
    if op in ("attention", "append"):
        lengths, tokens = _lengths(case), _tokens(case)
        kv, dim, block = case["kv_heads"], case["dim"], case["block"]
    if op == "attention":
        keys, total, heads = sum(lengths), sum(tokens), case["heads"]
        cells = sum(n * v - n * (n - 1) // 2 for n, v in zip(tokens, lengths))  # (query, key) pairs that the mask keeps
        return {"bytes": 2 * keys * kv * dim + 2 * kv * 4 * (keys // block) + 2 * 2 * total * heads * dim + 4 * (keys // case["page"]) + 12 * case["rows"],
                "flops": 4 * cells * heads * dim}
    if op == "append":
        total = sum(tokens)
        return {"bytes": 2 * total * kv * dim * 3 + 2 * kv * 4 * (total // block + case["rows"]) + 16 * case["rows"], "flops": 4 * total * kv * dim}
    if op == "copy":
        page = case["kv_heads"] * (case["page"] * case["dim"] + 4 * (case["page"] // case["block"]))
        return {"bytes": 2 * 2 * case["moves"] * page + 8 * case["moves"], "flops": 0}
    # a table and the counts read and written, and the list of copies written
    pairs = case["rows"] if op == "update" else case["pages"] // 2
    return {"bytes": 8 * case["rows"] * case["cols"] + 8 * case["pages"] + 8 * pairs + 16 * case["rows"], "flops": 0}


# ---------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    if case["op"] not in ("attention", "append"):
        return None  # copies and whole numbers
    s = prepare(case, seed)
    table, offsets, lengths = s["table"].cpu(), s["offsets"].tolist(), s["lengths"].tolist()
    page, block, kv = case["page"], case["block"], case["kv_heads"]
    caches = ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"]))
    if case["op"] == "attention":
        group = case["heads"] // kv
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for r, length in enumerate(lengths):
            a, b = offsets[r], offsets[r + 1]
            at = table[r, : -(-length // page)].cuda().long()
            ends = torch.arange(length - (b - a) + 1, length + 1, device="cuda")
            dead = torch.arange(length, device="cuda")[None, :] >= ends[:, None]
            for h in range(kv):
                k, v = [codes.view(torch.uint8)[at, h].view(codes.dtype).to(torch.float32).double().reshape(-1, case["dim"])[:length]
                        * scale[at, h].double().repeat_interleave(block, 1).reshape(-1)[:length, None] for codes, scale in caches]
                for e in range(h * group, (h + 1) * group):
                    x = (s["q"][a:b, e].double() @ k.T.contiguous()) * case["dim"] ** -0.5
                    out[a:b, e] = torch.softmax(x.masked_fill(dead, -math.inf), -1) @ v
        return out
    if s["k"].shape[0] > 20000 or case["rows"] * kv > 4096:
        return None
    i8, answer = case["cache"] == "i8", {}
    steps = torch.arange(256, device="cuda").to(torch.uint8).view(torch.float8_e4m3fn).float().double()
    steps = steps[steps.isfinite()].unique()  # the values of e4m3, ascending
    middle = (steps[1:] + steps[:-1]) / 2

    def nearest(y):
        if i8:
            return torch.round(y.clamp(-127, 127))
        y = y.clamp(-448, 448)
        down, up = torch.searchsorted(middle, y), torch.searchsorted(middle, y, right=True)  # a tie lies between two values: the even code
        even = steps[up].abs() / torch.exp2(torch.floor(torch.log2(steps[up].abs().clamp(min=2.0 ** -6))) - 3) % 2 == 0
        return torch.where((down == up) | ~even, steps[down], steps[up])

    for name, x, (codes, scale) in zip("kv", (s["k"], s["v"]), caches):
        got, by = codes.float().double(), scale.double()
        for r, length in enumerate(lengths):
            a, b = offsets[r], offsets[r + 1]
            begin, at = length - (b - a), 0
            while begin + at < length:
                pos = begin + at
                n = min(block - pos % block, length - pos)
                p, blk, lo = int(table[r, pos // page]), pos % page // block, pos % block
                new = x[a + at: a + at + n].double().transpose(0, 1)  # [kv, n, dim]
                top = new.abs().amax((1, 2))
                mine = top / 127 if i8 else torch.exp2(torch.ceil(torch.log2(top / 448)))
                old = by[p, :, blk] if lo else torch.zeros_like(mine)
                now = torch.maximum(mine, old)
                part = got[p, :, blk * block: blk * block + lo + n]
                if lo:
                    part[:, :lo] = torch.where((now > old)[:, None, None], nearest(part[:, :lo] * (old / now)[:, None, None]), part[:, :lo])
                part[:, lo:] = nearest(new / now[:, None, None])
                by[p, :, blk] = now
                at += n
        if i8:
            got = got.view(got.shape[0], kv, page // block, -1) * by.unsqueeze(-1)
        answer["%s" % name if i8 else "%s_cache" % name], answer["%s_scale" % name] = got, by
    return answer
