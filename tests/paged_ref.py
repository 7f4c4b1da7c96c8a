"""Plain statements of the paged-cache operators for the tests, sequence by
sequence and number by number on the CPU: codes in the fp32 steps that the
operator is defined by, values and attention in 64 bits, page tables as lists."""
import numpy as np
import torch

MOST = {"i8": 127.0, "e4m3": 448.0}
CODE = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
FLOAT = {"f16": torch.float16, "bf16": torch.bfloat16}


def values(codes):
    return codes.to(torch.float32).double()


def nearest(y, cache):
    """fp32 -> codes: to nearest even, infinities to the ends, NaN to 0."""
    y = torch.where(y.isnan(), torch.zeros_like(y), y).clamp(-MOST[cache], MOST[cache])
    return torch.round(y).to(torch.int8) if cache == "i8" else y.to(torch.float8_e4m3fn)


def scale_for(top, cache):
    """The scale of a block whose largest finite magnitude is `top` (fp32, exact in it)."""
    top = np.float32(top)
    if top < np.float32(2.0 ** -96):
        return np.float32(0)
    if cache == "i8":
        return np.float32(top / np.float32(127))
    m, e = np.frexp(np.float64(top))  # 448 = 0.875 * 2^9
    return np.float32(np.ldexp(1.0, int(e) - 9 + (1 if m > 0.875 else 0)))


class Cache:
    """One of k, v: codes [pages, heads, page, dim] and scales [pages, heads, page / block] on the CPU."""

    def __init__(self, codes, scales, cache):
        self.codes, self.scales, self.cache = codes, scales, cache
        self.page, self.block = codes.shape[2], codes.shape[2] // scales.shape[2]

    def append(self, row_pages, begin, x):
        """x [tokens, heads, dim] of 16-bit floats to places begin .. of a row."""
        x = x.float()
        at = 0
        while at < x.shape[0]:
            pos = begin + at
            lo = pos % self.block
            n = min(self.block - lo, x.shape[0] - at)
            page = row_pages[pos // self.page]
            if 0 <= page < self.codes.shape[0]:
                for h in range(self.codes.shape[1]):
                    self._block(page, h, pos % self.page // self.block, lo, x[at:at + n, h])
            at += n

    def _block(self, page, h, b, lo, new):
        a = new.abs()
        a = torch.where(a < float("inf"), a, torch.zeros_like(a))
        old = np.float32(self.scales[page, h, b]) if lo else np.float32(0)
        now = max(scale_for(float(a.max()), self.cache), old)
        at = self.codes[page, h, b * self.block:(b + 1) * self.block]
        if lo and now > old:
            ratio = np.float32(old / now)
            at[:lo] = nearest(at[:lo].to(torch.float32) * float(ratio), self.cache)
        inv = np.float32(np.float32(1) / now) if now > 0 else np.float32(0)
        at[lo:lo + new.shape[0]] = nearest(new * float(inv), self.cache)
        self.scales[page, h, b] = float(now)

    def top(self, row_pages, length):
        """The largest value that a code of the row's places could stand for."""
        rows = [p for p in row_pages[:-(-length // self.page)] if 0 <= p < self.codes.shape[0]]
        return max([0.0] + [float(self.scales[p, :, b].max()) * MOST[self.cache] for i, p in enumerate(rows) for b in range(self.page // self.block)
                            if i * self.page + b * self.block < length])

    def read(self, row_pages, length):
        """[length, heads, dim] in 64 bits; places without a page are NaN."""
        pages, heads, page, dim = self.codes.shape
        out = torch.full((length, heads, dim), float("nan"), dtype=torch.float64)
        for pos in range(0, length, self.block):
            p, n = row_pages[pos // page], min(self.block, length - pos)
            if 0 <= p < pages:
                b = pos % page
                out[pos:pos + n] = (values(self.codes[p, :, b:b + n]) * self.scales[p, :, b // self.block].double()[:, None, None]).transpose(0, 1)
        return out


def attention(q, k, v, scale, there=None):
    """q [tokens, heads, dim] (the last tokens of the row), k, v [length, kv_heads, dim] in 64 bits.  Returns the result, the weighted
    mean of |v| and the largest sum of |scale q k| of each (token, head): what the tolerance is derived from."""
    q = q.double()
    tokens, heads, dim = q.shape
    length, kv, _ = k.shape
    group = heads // kv
    there = torch.ones(length, dtype=torch.bool) if there is None else there
    kk, vv = torch.where(there[:, None, None], k, 0.0), torch.where(there[:, None, None], v, 0.0)
    kk, vv = kk.repeat_interleave(group, 1), vv.repeat_interleave(group, 1)
    s = torch.einsum("thd,jhd->thj", q, kk) * scale
    size = torch.einsum("thd,jhd->thj", q.abs(), kk.abs()) * abs(scale)
    seen = (torch.arange(length)[None, :] <= (length - tokens + torch.arange(tokens))[:, None]) & there[None, :]
    s = s.masked_fill(~seen[:, None], -float("inf"))
    top = s.amax(-1, keepdim=True) if length else torch.zeros(tokens, heads, 1).double()
    p = torch.exp(s - torch.where(top == -float("inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    return torch.einsum("thj,jhd->thd", p, vv), torch.einsum("thj,jhd->thd", p, vv.abs()), (size * seen[:, None]).amax(-1) if length else top[..., 0]


def attention_bound(want, mean, size, dtype, dim, length, v_top):
    """What rounding allows, element by element:
      * the result to its type: half a step of it;
      * each weight to fp16: 2^-11 of it (half a step), so 2^-11 of the weighted mean of |v|;
      * a score: dim products added in fp32, and q to fp16 after scaling (2^-11 times 2^-14 of the row's largest for what falls
        below its normal numbers), its scale and exponent: (dim + 16) 2^-24 of the sum of |q k|, and 2^-22 for exp2 and its argument.
        A weight changes by twice that (its own and the sum's);
      * a weight too small for fp16's normal numbers, which is held 2^10 up: half a step of 2^-24 there, 2^-35 of the largest weight
        and so of their sum, times the largest value (code times the row's largest V scale, `v_top`), for each key;
      * prompts: a V scale goes into the exponent as its log2, relative to the largest one's.  The log2 is at most 126, so it and the two sums it
        goes through are off by at most a step and two halves of 2^-17, 2^-16 in the exponent, and the value by ln 2 of that: 2^-16 of
        the mean.  (It is taken out of the weights' own sum with the same error.)  A scale 2^-40 times smaller than the largest has
        weights that fp16 holds as 0: that is within the last point's 2^-35;
      * sums over keys in fp32: one rounding for each 32 keys and each joined part, 2^-24 of the mean each."""
    delta = (dim + 16) * 2.0 ** -24 * size + 2.0 ** -22 * (1 + size)
    eps = torch.finfo(FLOAT[dtype]).eps / 2
    tiny = torch.finfo(FLOAT[dtype]).tiny * torch.finfo(FLOAT[dtype]).eps
    inside = 2.0 ** -35 * length * v_top + (2.0 ** -11 + 2.0 ** -16 + 2.0 ** -24 * (length / 32 + 600)) * mean + 2 * delta[..., None] * mean
    return inside + eps * (want.abs() + inside) + tiny


def largest_share(q, k, v_scale, cache, scale, there=None):
    """[tokens, heads]: the largest that one key which the token sees could add to its result, weight times V scale times the largest code.
    v_scale: [length, kv_heads]."""
    tokens, heads, _ = q.shape
    length, kv, _ = k.shape
    there = torch.ones(length, dtype=torch.bool) if there is None else there
    kk = torch.where(there[:, None, None], k, 0.0).repeat_interleave(heads // kv, 1)
    s = torch.einsum("thd,jhd->thj", q.double(), kk) * scale
    seen = (torch.arange(length)[None, :] <= (length - tokens + torch.arange(tokens))[:, None]) & there[None, :]
    p = torch.softmax(s.masked_fill(~seen[:, None], -float("inf")), -1)
    one = torch.where(there[:, None], v_scale.double(), 0.0).repeat_interleave(heads // kv, 1)
    return torch.where(p.isnan(), 0.0, p * one.T[None]).amax(-1) * MOST[cache]


def seen_bound(want, mean, size, dtype, dim, length, share):
    """attention_bound with its point on small weights held to what each token sees: a weight times its V scale that is too small
    for fp16 is off by 2^-35 of the largest such product (`share`, of the token itself), times the largest code, for each key."""
    return attention_bound(want, mean, size, dtype, dim, length, share[..., None])


# ---- page tables ----------------------------------------------------------------
def update(table, lengths, refs, source, grow, page):
    """(table, lengths, refs, pairs, result) after PageTableUpdate, from lists."""
    rows, cols, pages = len(table), len(table[0]), len(refs)
    count = lambda n: -(-n // page)  # noqa: E731
    clip = lambda n: min(max(n, 0), cols * page)  # noqa: E731
    refs = list(refs)
    new, before = [], []
    for r in range(rows):
        s = source[r]
        ok = 0 <= s < rows
        before.append(clip(lengths[s]) if ok else 0)
        new.append(list(table[r]) if s == r else [table[s][c] if ok and c < count(before[r]) else -1 for c in range(cols)])
    for r in range(rows):
        if source[r] != r:
            for p in table[r][:count(clip(lengths[r]))]:
                if 0 <= p < pages:
                    refs[p] -= 1
            for p in new[r][:count(before[r])]:
                if 0 <= p < pages:
                    refs[p] += 1
    by = [max(g, 0) for g in grow]
    wide = [before[r] + by[r] > cols * page for r in range(rows)]
    copies, need = [], []
    for r in range(rows):
        last = new[r][count(before[r]) - 1] if before[r] else -1
        copies.append(not wide[r] and by[r] > 0 and before[r] % page != 0 and 0 <= last < pages and refs[last] > 1)
        need.append(0 if wide[r] else count(before[r] + by[r]) - count(before[r]) + copies[r])
    free = [p for p in range(pages) if refs[p] == 0]
    result = [max(0, sum(need) - len(free)), sum(wide)]
    pairs = [[-1, -1] for _ in range(rows)]
    if result != [0, 0]:
        return new, before, refs, pairs, result
    fresh = iter(free)
    after = list(before)
    for r in range(rows):
        have = count(before[r])
        if copies[r]:
            p = next(fresh)
            pairs[r] = [new[r][have - 1], p]
            refs[new[r][have - 1]] -= 1
            new[r][have - 1] = p
            refs[p] = 1
        after[r] = before[r] + by[r]
        for c in range(have, count(after[r])):
            new[r][c] = next(fresh)
            refs[new[r][c]] = 1
    return new, after, refs, pairs, result


def compact(table, lengths, refs, page, room):
    """(table, refs, pairs, result) after PageTableCompact, from lists."""
    pages, cols = len(refs), len(table[0]) if table else 0
    used = sum(n > 0 for n in refs)
    above = [p for p in range(used, pages) if refs[p] > 0]
    below = [p for p in range(used) if refs[p] <= 0]
    goes = dict(zip(above, below))
    new = [[goes.get(p, p) if c < -(-min(max(n, 0), cols * page) // page) else p for c, p in enumerate(row)] for row, n in zip(table, lengths)]
    refs = list(refs)
    for a, b in goes.items():
        refs[b], refs[a] = refs[a], 0
    pairs = [[a, b] for a, b in goes.items()] + [[-1, -1]] * (room - len(goes))
    return new, refs, pairs, [used, len(goes)]
