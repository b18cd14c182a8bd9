"""Keys and values in 8 bits with a scale for every 16 tokens and head: writing, reading back and attention over them, against
64-bit arithmetic."""
import math

import pytest
import torch

from air_b200.csrc import ops
from air_b200.parts.attention import plan_portions

pytestmark = pytest.mark.gpu

E4M3 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()      # 0 .. 448, rising


def nearest(x, grid):
    """x (float64) to the nearest number of `grid` (rising, from 0), ties to the one of even place."""
    a = x.abs()
    hi = torch.searchsorted(grid, a).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = (grid[hi] - a).abs(), (a - grid[lo]).abs()
    pick = torch.where(up < down, hi, torch.where(down < up, lo, torch.where(hi % 2 == 0, hi, lo)))
    return torch.copysign(grid[pick], x)


def scale_for(top):
    if top == 0:
        return 2.0 ** -110
    e = math.ceil(math.log2(top / 448))
    while 448 * 2.0 ** e < top:
        e += 1
    while 448 * 2.0 ** (e - 1) >= top:
        e -= 1
    return 2.0 ** max(-110, e)


class Pool:
    """Pages for requests of these lengths, in any order, filled with numbers of a known scale."""

    def __init__(self, lengths, K, P, d, seed, fill=True, spread=3):
        g = torch.Generator().manual_seed(seed)
        self.g, self.K, self.P, self.d = g, K, P, d
        need = [-(-n // P) for n in lengths]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g).int()
        self.slots = torch.randperm(len(lengths) + 1, generator=g).tolist()[:len(lengths)]
        table = torch.full((len(lengths) + 1, max(need) + 1), -1, dtype=torch.int32)
        at = 0
        for s, n in zip(self.slots, need):
            table[s, :n] = order[at:at + n]
            at += n
        self.table = table.cuda()
        codes = torch.randint(0, 256, (pages, 2, K, P, d), generator=g, dtype=torch.uint8)
        codes[(codes & 127) == 127] = 0
        self.scales = torch.exp2(torch.randint(-9 - spread, -9 + spread, (pages, 2, K, P // 16), generator=g).float()).cuda()
        if not fill:
            codes.fill_(0x7f)           # NaN wherever nothing has been written
            self.scales.fill_(math.nan)
        self.cache = codes.view(torch.float8_e4m3fn).cuda()

    def rows(self, slot, n):
        """float64 [2, K, n, d] on the CPU."""
        pages = self.table[slot].cpu().tolist()
        x = self.cache.cpu().float().double() * self.scales.cpu().double().repeat_interleave(16, -1)[..., None]
        return torch.cat([x[p] for p in pages[:-(-n // self.P)]], 2)[:, :, :n] if n else torch.zeros((2, self.K, 0, self.d), dtype=torch.float64)


def batch(counts, before, slots):
    pos = torch.cat([torch.arange(b, b + c) for c, b in zip(counts, before)]).int().cuda()
    seq = torch.cat([torch.full((c,), s) for c, s in zip(counts, slots)]).int().cuda()
    return pos, seq


# ---------------------------------------------------------------------------------------------- writing
def stored(pool, qkv, bias, table, pos, seq, H, status=None):
    T = qkv.shape[-2]
    q = torch.full((T, H, pool.d), math.nan, dtype=torch.bfloat16, device="cuda")
    return ops.qkv_rope_store8(qkv, bias, table, pos, seq, pool.table, q, pool.cache, pool.scales, H, pool.K, pool.d, status=status)


def rotation(n, d):
    a = torch.arange(n, dtype=torch.float64)[:, None] * torch.pow(torch.tensor(1e4, dtype=torch.float64), -torch.arange(d // 2).double() * 2 / d)
    return torch.cat([a.cos(), a.sin()], 1).float()


@pytest.mark.parametrize("d,P,H,K,parts,with_bias", [(64, 16, 3, 1, 1, False), (128, 64, 4, 2, 3, True), (128, 32, 28, 4, 1, True), (64, 128, 5, 5, 2, False)])
def test_portions_are_rounded_by_their_blocks_largest_number(d, P, H, K, parts, with_bias):
    counts, before = [1, 5, 40, 1, 16, 19], [0, 14, 3, 47, 32, 0]
    lengths = [c + b for c, b in zip(counts, before)]
    pool = Pool(lengths, K, P, d, seed=d + P)
    T, width = sum(counts), (H + 2 * K) * d
    qkv = torch.randn((parts, T, width), generator=pool.g) * torch.exp2(torch.randint(-8, 8, (1, T, 1), generator=pool.g).float())
    bias = torch.randn(width, generator=pool.g) if with_bias else None
    table = rotation(max(lengths), d)
    pos, seq = batch(counts, before, pool.slots)
    earlier = [pool.rows(s, n) for s, n in zip(pool.slots, before)]
    old_scales = pool.scales.cpu().clone()
    behind = pool.cache.cpu().view(torch.uint8).clone()
    q = stored(pool, qkv.cuda() if parts > 1 else qkv[0].cuda(), bias.cuda() if with_bias else None, table.cuda(), pos, seq, H)

    x = qkv.double().sum(0)
    size = qkv.double().abs().sum(0)
    if with_bias:
        x, size = x + bias.double(), size + bias.double().abs()
    x, size = x.view(T, H + 2 * K, d), size.view(T, H + 2 * K, d)
    cs = table.double()[pos.cpu().long()][:, None]
    c, s = cs[..., :d // 2], cs[..., d // 2:]

    def turn(v, c, s):
        a, b = v[..., :d // 2], v[..., d // 2:]
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    turned = turn(x[:, :H + K], c, s)
    spread = torch.cat([size[..., :d // 2] + size[..., d // 2:]] * 2, -1)[:, :H + K]
    # float32: a sum of parts + 1 numbers, two products and their sum, each rounded by 2^-24 of at most `spread`
    slack = spread * (parts + 4) * 2.0 ** -24
    assert ((q.cpu().double() - turned[:, :H]).abs() <= slack[:, :H] + (turned[:, :H].abs() + slack[:, :H]) * 2.0 ** -8).all()
    new = torch.stack([turned[:, H:], x[:, H + K:]], 1)                      # [T, 2, K, d]
    new_slack = torch.stack([slack[:, H:], size[:, H + K:] * (parts + 1) * 2.0 ** -24], 1)
    at = 0
    for i, (n, b, slot) in enumerate(zip(counts, before, pool.slots)):
        got = pool.rows(slot, n + b)
        mine, lax = new[at:at + n].permute(1, 2, 0, 3), new_slack[at:at + n].permute(1, 2, 0, 3)
        at += n
        # blocks that were full before are as they were
        whole = b // 16 * 16
        assert torch.equal(got[:, :, :whole], earlier[i][:, :, :whole])
        pages = pool.table[slot].cpu().tolist()
        for start in range(whole, n + b, 16):
            stop, first = min(start + 16, n + b), max(start, b)
            for w in range(2):
                for k in range(K):
                    fresh, lx = mine[w, k, first - b:stop - b], lax[w, k, first - b:stop - b]
                    place = (pages[start // P], w, k, start % P // 16)
                    unit = scale_for(float(fresh.abs().max()))
                    low, high = scale_for(float((fresh.abs() - lx).max())), scale_for(float((fresh.abs() + lx).max()))
                    if first > start:
                        unit, low, high = (max(v, float(old_scales[place])) for v in (unit, low, high))
                    assert low <= float(pool.scales[place]) <= high
                    unit = float(pool.scales[place])
                    # half a step of e4m3 (2^-4 of a number, 2^-10 of the scale below its normal ones), and float32's own rounding
                    err = (got[w, k, first:stop] - fresh).abs()
                    assert (err <= (fresh.abs() + lx) * 2.0 ** -4 + unit * 2.0 ** -10 + lx).all()
                    exact = nearest(fresh / unit, E4M3) * unit
                    assert (got[w, k, first:stop] == exact).double().mean() > 0.98       # (but where float32's rounding decides)
                    held = nearest(earlier[i][w, k, start:first] / unit, E4M3) * unit
                    assert torch.equal(got[w, k, start:first], held)
            if stop < start + 16:       # rows behind the last token: as they were
                page, off = pages[start // P], stop % P
                left = start + 16 - stop
                assert torch.equal(pool.cache.cpu().view(torch.uint8)[page, :, :, off:off + left], behind[page, :, :, off:off + left])


def test_a_block_filled_token_by_token_holds_what_its_scale_allows():
    H, K, d, P, n = 2, 1, 128, 16, 37
    pool = Pool([n], K, P, d, seed=3, fill=False)
    qkv = torch.randn((n, (H + 2 * K) * d), generator=pool.g) * torch.exp2(torch.arange(n).float() % 7)[:, None]
    table = torch.cat([torch.ones(n, d // 2), torch.zeros(n, d // 2)], 1).cuda()          # no turn: keys are what the product left
    for i in range(n):
        pos, seq = batch([1], [i], pool.slots)
        stored(pool, qkv[i:i + 1].cuda(), None, table, pos, seq, H)
    got = pool.rows(pool.slots[0], n)
    want = qkv.double().view(n, H + 2, d)[:, H:].permute(1, 0, 2)[:, None]
    unit = torch.stack([pool.scales.cpu()[p] for p in pool.table[pool.slots[0]].cpu().tolist()[:3]], 2)[:, :, :, 0].double()
    unit = unit.repeat_interleave(16, -1)[:, :, :n, None]
    # every rounding of a number is half a step; a scale that grows only shifts it, but below the scale's normal numbers, where each of
    # at most six later roundings adds half a step of the scale that it was made with
    assert ((got - want).abs() <= want.abs() * 2.0 ** -4 + 2 * unit * 2.0 ** -10).all()
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_numbers_that_are_not_finite_become_nan_alone(bad):
    H, K, d = 1, 2, 64
    pool = Pool([20], K, 32, d, seed=4)
    qkv = torch.randn((20, (H + 2 * K) * d), generator=pool.g)
    qkv[7, (H + K) * d + 3] = bad                # a value of head 0
    table = rotation(20, d).cuda()
    pos, seq = batch([20], [0], pool.slots)
    stored(pool, qkv.cuda(), None, table, pos, seq, H)
    got = pool.rows(pool.slots[0], 20)
    assert math.isnan(got[1, 0, 7, 3])
    got[1, 0, 7, 3] = 0
    assert torch.isfinite(got).all()


def test_padding_and_pages_that_are_not_held():
    H, K, d, P = 2, 2, 64, 16
    pool = Pool([16, 16], K, P, d, seed=5)
    before = pool.cache.cpu().view(torch.uint8).clone(), pool.scales.cpu().clone()
    qkv = torch.randn((3, (H + 2 * K) * d), generator=pool.g).cuda()
    table = rotation(4096, d).cuda()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    pos = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda")
    seq = torch.full((3,), -1, dtype=torch.int32, device="cuda")
    q = stored(pool, qkv, None, table, pos, seq, H, status)
    assert torch.isnan(q).all() and int(status) == 0
    for at in (16, 4000):      # a block without a page, and one beyond the table
        status.zero_()
        seq = torch.full((1,), pool.slots[0], dtype=torch.int32, device="cuda")
        q = stored(pool, qkv[:1], None, table, torch.tensor([at], dtype=torch.int32, device="cuda"), seq, H, status)
        assert torch.isfinite(q).all() and int(status) == 2
    assert torch.equal(pool.cache.cpu().view(torch.uint8), before[0]) and torch.equal(pool.scales.cpu(), before[1])


@pytest.mark.parametrize("d,P", [(64, 16), (128, 64), (128, 128)])
def test_rows_are_read_back(d, P):
    lengths = [1, 33, 200, 64]
    pool = Pool(lengths, 3, P, d, seed=6)
    pool.table[pool.slots[2], 0] = -1
    out = torch.full((4, 2, 3, 210, d), math.nan, dtype=torch.bfloat16, device="cuda")
    ops.cache8_rows(pool.cache, pool.scales, pool.table, torch.tensor(pool.slots, dtype=torch.int32, device="cuda"),
                    torch.tensor(lengths, dtype=torch.int32, device="cuda"), out)
    for i, (slot, n) in enumerate(zip(pool.slots, lengths)):
        want = pool.rows(slot, n)
        if i == 2:
            want[:, :, :P] = 0
        assert torch.equal(out[i, :, :, :n].cpu().double(), want)
        assert (out[i, :, :, n:] == 0).all()


# ---------------------------------------------------------------------------------------------- attention
def attention64(q, pos, rows, window, scale):
    """float64 (out [n, H, d], size [n, H, d] = sum of weight |value|) of n queries at positions pos over rows [2, K, L, d]."""
    n, H, d = q.shape
    K, L = rows.shape[1], rows.shape[2]
    k, v = (x.repeat_interleave(H // K, 0) for x in (rows[0], rows[1]))
    score = torch.einsum("nhd,hld->hnl", q.double(), k) * scale
    key = torch.arange(L)
    seen = key <= pos[:, None]
    if window:
        seen &= key > pos[:, None] - window
    score = score.masked_fill(~seen, -math.inf)
    w = torch.softmax(score, -1)
    return torch.einsum("hnl,hld->nhd", w, v), torch.einsum("hnl,hld->nhd", w, v.abs())


def poison(pool, slot, n):
    """What stands behind token n of the request in its pages: NaN, and scales that are no numbers."""
    page = int(pool.table[slot, (n - 1) // pool.P])
    codes = pool.cache.view(torch.uint8)
    if n % pool.P:
        codes[page, :, :, n % pool.P:] = 0x7f
    whole = -(-n // 16) * 16
    if whole % pool.P:
        pool.scales[page, :, :, whole % pool.P // 16:] = math.nan


DECODE = [(64, 16, 4, 4, None, [1, 2, 16, 17]), (128, 64, 28, 4, None, [1, 63, 64, 65, 1000]), (128, 32, 40, 8, 100, [99, 100, 101, 300, 7]),
          (64, 128, 34, 1, None, [129, 500]), (128, 16, 6, 2, 16, [16, 31, 48, 1]), (128, 64, 12, 2, None, [5000]), (64, 64, 2, 2, 1, [1, 70])]


@pytest.mark.parametrize("d,P,H,K,window,contexts", DECODE)
@pytest.mark.parametrize("splits", [None, 1, 5])
def test_single_tokens(d, P, H, K, window, contexts, splits):
    pool = Pool(contexts, K, P, d, seed=sum(contexts) + d)
    for s, n in zip(pool.slots, contexts):
        poison(pool, s, n)
        if window and n > window + P:
            pool.table[s, 0] = -1               # the window has given its first page back
    T = len(contexts)
    q = (torch.randn((T + 1, H, d), generator=pool.g) * 4).bfloat16()
    pos = torch.tensor([n - 1 for n in contexts] + [0], dtype=torch.int32, device="cuda")
    seq = torch.tensor(pool.slots + [-1], dtype=torch.int32, device="cuda")
    out = torch.full((T + 1, H, d), math.nan, dtype=torch.bfloat16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.decode_attention8(q.cuda(), pool.cache, pool.scales, pool.table, seq, pos, out, window, d ** -0.5, splits=splits, status=status)
    assert int(status) == 0 and torch.isnan(out[T]).all()
    for i, (slot, n) in enumerate(zip(pool.slots, contexts)):
        if window and n > window + P:
            pool.table[slot, 0] = int(pool.table[slot, 1])          # (never seen; the oracle wants some page there)
        rows = pool.rows(slot, n)
        if window:
            rows[:, :, :max(0, n - window)] = 0
        want, size = attention64(q[i:i + 1], torch.tensor([n - 1]), rows, window, d ** -0.5)
        # probabilities are rounded to float16 (2^-11), scores and sums in float32, the output to bfloat16 (2^-8)
        tolerance = size * (2.0 ** -11 + 2.0 ** -16) + want.abs() * 2.0 ** -8
        assert ((out[i:i + 1].cpu().double() - want).abs() <= tolerance * 1.01 + 1e-30).all()


def test_scales_far_apart_and_queries_of_any_size():
    d, P, H, K, n = 128, 64, 8, 2, 300
    pool = Pool([n], K, P, d, seed=9)
    pool.scales.copy_(torch.exp2(torch.randint(-40, -8, pool.scales.shape, generator=pool.g).float()))
    pool.scales[:, 0] = 2.0 ** -9
    q = torch.randn((1, H, d), generator=pool.g)
    q *= torch.exp2(torch.tensor([-60.0, -20, -3, 0, 3, 5, 8, 100]))[None, :, None]
    q = q.bfloat16()
    out = torch.empty((1, H, d), dtype=torch.bfloat16, device="cuda")
    pos, seq = batch([1], [n - 1], pool.slots)
    ops.decode_attention8(q.cuda(), pool.cache, pool.scales, pool.table, seq, pos, out, None, 0.125)
    rows = pool.rows(pool.slots[0], n)
    want, size = attention64(q, torch.tensor([n - 1]), rows, None, 0.125)
    # scores of up to 2^108 * 448 have float32 errors far beyond one unless a single key stands out, which it then does for every one
    gap = torch.einsum("nhd,hld->nhl", q.double(), rows[0].repeat_interleave(H // K, 0)) * 0.125
    top = gap.topk(2, -1).values
    sure = (top[..., 0] - top[..., 1] > 2.0 ** -18 * gap.abs().amax(-1)) | (gap.abs().amax(-1) < 2.0 ** 7)
    # 2^-24 of the largest score for every step of its float32 sum of eight instructions, as a relative change of a weight, doubled
    # for the numerator and the denominator; a probability times its value's scale, against the largest scale, may fall below float16's
    # normal numbers and be off by 2^-25, for each of n keys
    largest = rows[1].abs().amax((1, 2)).repeat_interleave(H // K, 0)[None, :, None]
    score_error = torch.where(gap.abs().amax(-1) < 2.0 ** 7, gap.abs().amax(-1) * 2.0 ** -19, 0.0)[..., None]
    tolerance = size * (2.0 ** -11 + 2.0 ** -16 + 2 * score_error) + want.abs() * 2.0 ** -8 + largest * n * 2.0 ** -25
    assert sure.sum() >= 6
    bad = ((out.cpu().double() - want).abs() > tolerance * 1.01) & sure[..., None]
    assert not bad.any()


PROMPTS = [(64, 64, 4, 2, None, [70], [0]), (128, 64, 7, 1, None, [300, 2, 129], [0, 63, 500]), (128, 16, 4, 4, None, [33], [15]),
           (64, 32, 8, 2, 50, [200, 16], [100, 0]), (128, 128, 5, 5, 1000, [17, 256], [1500, 130]), (128, 64, 28, 4, None, [64], [6000]),
           (64, 16, 2, 1, 8, [40], [300])]


@pytest.mark.parametrize("d,P,H,K,window,counts,before", PROMPTS)
def test_portions(d, P, H, K, window, counts, before):
    lengths = [c + b for c, b in zip(counts, before)]
    pool = Pool(lengths, K, P, d, seed=sum(lengths))
    for s, n in zip(pool.slots, lengths):
        poison(pool, s, n)
    T = sum(counts)
    q = (torch.randn((T + 3, H, d), generator=pool.g) * 4).bfloat16()
    out = torch.full((T + 3, H, d), math.nan, dtype=torch.bfloat16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    plan = plan_portions(counts, before, pool.slots, H, window, "cuda")
    ops.prefill_attention8(q.cuda(), pool.cache, pool.scales, pool.table, plan.tiles, out, window, d ** -0.5, status=status,
                           segments=plan.segments, items=plan.items, slots=plan.slots)
    assert int(status) == 0 and torch.isnan(out[T:]).all()
    at = 0
    for slot, c, b in zip(pool.slots, counts, before):
        rows = pool.rows(slot, c + b)
        want, size = attention64(q[at:at + c], torch.arange(b, b + c), rows, window, d ** -0.5)
        # probabilities are rounded to bfloat16 (2^-8) and come from 2^x within 7.5e-5, sums are theirs before rounding; the output to
        # bfloat16 (2^-8)
        tolerance = size * (2.0 ** -8 + 2 * 7.6e-5) + want.abs() * 2.0 ** -8
        assert ((out[at:at + c].cpu().double() - want).abs() <= tolerance * 1.01 + 1e-30).all()
        at += c


@pytest.mark.parametrize("exponent", [-100, 30])
def test_portions_over_blocks_of_any_scale(exponent):
    d, P, H, K, n = 128, 64, 2, 1, 100
    pool = Pool([n], K, P, d, seed=12)
    pool.scales[:, 1] = torch.exp2(torch.randint(exponent - 2, exponent + 2, pool.scales[:, 1].shape, generator=pool.g).float()).cuda()
    q = torch.randn((n, H, d), generator=pool.g).bfloat16()
    out = torch.empty((n, H, d), dtype=torch.bfloat16, device="cuda")
    plan = plan_portions([n], [0], pool.slots, H, None, "cuda")
    ops.prefill_attention8(q.cuda(), pool.cache, pool.scales, pool.table, plan.tiles, out, None, 0.1)
    want, size = attention64(q, torch.arange(n), pool.rows(pool.slots[0], n), None, 0.1)
    assert ((out.cpu().double() - want).abs() <= (size * (2.0 ** -8 + 2 * 7.6e-5) + want.abs() * 2.0 ** -8) * 1.01).all()


@pytest.mark.parametrize("which", [0, 1])
def test_nan_that_is_seen_reaches_the_output(which):
    d, P, H, K, n = 64, 64, 4, 2, 90
    pool = Pool([n], K, P, d, seed=13)
    page = int(pool.table[pool.slots[0], 0])
    pool.cache.view(torch.uint8)[page, which, 1, 20, 5] = 0xff
    q = torch.randn((n, H, d), generator=pool.g).bfloat16().cuda()
    out = torch.empty((n, H, d), dtype=torch.bfloat16, device="cuda")
    plan = plan_portions([n], [0], pool.slots, H, None, "cuda")
    ops.prefill_attention8(q, pool.cache, pool.scales, pool.table, plan.tiles, out, None, 0.1)
    assert torch.isfinite(out[:, :2]).all() and torch.isfinite(out[:20]).all()
    assert torch.isnan(out[20:, 2:] if which == 0 else out[20:, 2:, 5]).all()
    # the same where the stream of keys is cut: two segments of the one item of every head
    heads = torch.arange(H, dtype=torch.int32)
    cut = torch.cat([torch.stack([0 * heads, heads, 0 * heads, 0 * heads + 1, 2 * heads], 1),
                     torch.stack([0 * heads, heads, 0 * heads + 1, 0 * heads + (1 << 30), 2 * heads + 1], 1)]).cuda()
    items = torch.stack([0 * heads, heads, 2 * heads, 0 * heads + 2], 1).cuda()
    again = torch.empty_like(out)
    ops.prefill_attention8(q, pool.cache, pool.scales, pool.table, plan.tiles, again, None, 0.1, segments=cut, items=items, slots=2 * H)
    assert torch.equal(torch.isnan(again), torch.isnan(out))
    one = torch.empty((1, H, d), dtype=torch.bfloat16, device="cuda")
    pos, seq = batch([1], [n - 1], pool.slots)
    ops.decode_attention8(q[:1].contiguous(), pool.cache, pool.scales, pool.table, seq, pos, one, None, 0.1)
    assert torch.isfinite(one[:, :2]).all()
    assert torch.isnan(one[:, 2:] if which == 0 else one[:, 2:, 5]).all()


FRESH = [(64, 16, 4, 2, None, [1, 16, 17, 31, 64, 65, 130]), (128, 64, 28, 4, None, [1, 2, 33, 1000]), (128, 32, 40, 8, 100, [99, 250, 7]),
         (64, 128, 14, 1, 20, [15, 500]), (128, 16, 16, 1, None, [48, 700])]


@pytest.mark.parametrize("d,P,H,K,window,contexts", FRESH)
@pytest.mark.parametrize("splits,early", [(None, False), (1, False), (3, True)])
def test_single_tokens_from_the_product_are_what_two_launches_make_of_them(d, P, H, K, window, contexts, splits, early):
    T, parts = len(contexts), 3
    pools = [Pool(contexts, K, P, d, seed=sum(contexts) + d, spread=2) for _ in range(2)]
    pool = pools[0]
    qkv = torch.randn((parts, T, (H + 2 * K) * d), generator=pool.g)
    qkv *= torch.exp2(torch.randint(-9, 6, (1, T, 1), generator=pool.g).float())          # blocks whose scale grows, and does not
    qkv = qkv.cuda()
    bias = torch.randn((H + 2 * K) * d, generator=pool.g).cuda()
    table = rotation(max(contexts), d).cuda()
    pos, seq = batch([1] * T, [n - 1 for n in contexts], pool.slots)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = stored(pools[0], qkv, bias, table, pos, seq, H, status)
    want = torch.empty((T, H, d), dtype=torch.bfloat16, device="cuda")
    ops.decode_attention8(q, pools[0].cache, pools[0].scales, pools[0].table, seq, pos, want, window, d ** -0.5, splits=splits)
    out = torch.full((T, H, d), math.nan, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    ops.decode_attention8_fresh(qkv, bias, table, pools[1].cache, pools[1].scales, pools[1].table, seq, pos, out, H, window, d ** -0.5,
                                splits=splits, status=status, early=early)
    assert int(status) == 0
    assert torch.equal(pools[0].cache.view(torch.uint8), pools[1].cache.view(torch.uint8)) and torch.equal(pools[0].scales, pools[1].scales)
    assert torch.equal(out, want)
    # once more over the same pages, whose keys and values another layer has written
    again = torch.full_like(out, math.nan)
    ops.decode_attention8_fresh(qkv, bias, table, pools[1].cache, pools[1].scales, pools[1].table, seq, pos, again, H, window, d ** -0.5,
                                write_kv=False, splits=splits, status=status)
    assert torch.equal(again, want)
    assert torch.equal(pools[0].cache.view(torch.uint8), pools[1].cache.view(torch.uint8))


def test_refusals():
    pool = Pool([100], 2, 64, 64, seed=21)
    H, K, d = 4, 2, 64
    q = torch.zeros((1, H, d), dtype=torch.bfloat16, device="cuda")
    out = torch.empty_like(q)
    pos, seq = batch([1], [99], pool.slots)
    table = rotation(128, d).cuda()
    qkv = torch.zeros((1, (H + 2 * K) * d), device="cuda")
    c, s, bt = pool.cache, pool.scales, pool.table
    plan = plan_portions([1], [99], pool.slots, H, None, "cuda")
    odd = torch.zeros((3, 2, K, 48, d), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.ones((3, 2, K, 3), device="cuda")
    wide = torch.zeros((3, 2, K, 64, 256), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.ones((3, 2, K, 4), device="cuda")
    calls = [lambda: ops.decode_attention8(q, c.float(), s, bt, seq, pos, out, None, 1.0), lambda: ops.decode_attention8(q, c, s[:, :, :, :3], bt, seq, pos, out, None, 1.0),
             lambda: ops.decode_attention8(q[..., :32].contiguous(), c, s, bt, seq, pos, out, None, 1.0), lambda: ops.decode_attention8(q, *odd, bt, seq, pos, out, None, 1.0),
             lambda: ops.decode_attention8(q[:, :3].contiguous(), c, s, bt, seq, pos, out[:, :3].contiguous(), None, 1.0),
             lambda: ops.decode_attention8(torch.zeros((1, H, 256), dtype=torch.bfloat16, device="cuda"), *wide, bt, seq, pos, out, None, 1.0),
             lambda: ops.decode_attention8(q, c, s, bt, seq.long(), pos, out, None, 1.0), lambda: ops.decode_attention8(q, c, s, bt, seq, pos, out, -5, 1.0),
             lambda: ops.prefill_attention8(q, c, s, bt, plan.tiles.tiles, out, None, 1.0), lambda: ops.prefill_attention8(q, c, s, bt, plan.tiles, out.float(), None, 1.0),
             lambda: ops.qkv_rope_store8(qkv.bfloat16(), None, table, pos, seq, bt, q, c, s, H, K, d), lambda: ops.qkv_rope_store8(qkv, None, table[:, :32].contiguous(), pos, seq, bt, q, c, s, H, K, d),
             lambda: ops.qkv_rope_store8(qkv[:, :-1].contiguous(), None, table, pos, seq, bt, q, c, s, H, K, d), lambda: ops.qkv_rope_store8(qkv.cpu(), None, table, pos, seq, bt, q, c, s, H, K, d),
             lambda: ops.decode_attention8_fresh(torch.zeros((1, 38 * d), device="cuda"), None, table, c, s, bt, seq, pos, torch.zeros((1, 34, d), dtype=torch.bfloat16, device="cuda"), 34, None, 1.0),
             lambda: ops.cache8_rows(c, s, bt, seq, pos, torch.empty((1, 2, K, 4, d), device="cuda"))]
    for call in calls:
        with pytest.raises(ops.KernelError):
            call()
    # no tokens: nothing to do
    none = torch.empty((0, H, d), dtype=torch.bfloat16, device="cuda")
    i0 = pos[:0].contiguous()
    assert ops.decode_attention8(none, c, s, bt, i0, i0, none.clone(), None, 1.0).shape == (0, H, d)
    ops.qkv_rope_store8(qkv[:0].contiguous(), None, table, i0, i0, bt, none, c, s, H, K, d)


@pytest.mark.parametrize("n,splits", [(65, 2), (130, 3), (17, 1)])
def test_a_split_whose_only_key_is_nan(n, splits):
    """A block of the grid that sees no finite score must not drop out of the merge."""
    d, P, H, K = 64, 64, 4, 2
    pool = Pool([n], K, P, d, seed=31)
    q = torch.randn((1, H, d), generator=pool.g).bfloat16().cuda()
    pos, seq = batch([1], [n - 1], pool.slots)
    page = int(pool.table[pool.slots[0], (n - 1) // P])
    pool.cache.view(torch.uint8)[page, 0, 1, (n - 1) // 16 * 16 % P:, 5] = 0x7f          # head 1's keys of the last block
    out = torch.empty((1, H, d), dtype=torch.bfloat16, device="cuda")
    ops.decode_attention8(q, pool.cache, pool.scales, pool.table, seq, pos, out, None, 0.1, splits=splits)
    assert torch.isfinite(out[:, :2]).all() and torch.isnan(out[:, 2:]).all()
    # the same from a product whose key is NaN
    pool = Pool([n], K, P, d, seed=31)
    qkv = torch.randn((1, (H + 2 * K) * d), generator=pool.g).cuda()
    qkv[0, (H + 1) * d + 3] = math.nan
    ops.decode_attention8_fresh(qkv, None, rotation(n, d).cuda(), pool.cache, pool.scales, pool.table, seq, pos, out, H, None, 0.1, splits=splits)
    assert torch.isfinite(out[:, :2]).all() and torch.isnan(out[:, 2:]).all()


def test_a_step_of_padding_alone():
    d, P, H, K = 128, 64, 4, 2
    pool = Pool([10], K, P, d, seed=32)
    before = pool.cache.view(torch.uint8).clone(), pool.scales.clone()
    qkv = torch.randn((5, (H + 2 * K) * d), generator=pool.g).cuda()
    out = torch.full((5, H, d), math.nan, dtype=torch.bfloat16, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    pos, seq = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.full((5,), -1, dtype=torch.int32, device="cuda")
    for early in (False, True):
        ops.decode_attention8_fresh(qkv, None, rotation(16, d).cuda(), pool.cache, pool.scales, pool.table, seq, pos, out, H, None, 0.1,
                                    status=status, early=early)
    ops.decode_attention8(out, pool.cache, pool.scales, pool.table, seq, pos, out.clone(), None, 0.1, splits=4, status=status)
    assert int(status) == 0 and torch.isnan(out).all()
    assert torch.equal(pool.cache.view(torch.uint8), before[0]) and torch.equal(pool.scales, before[1])


def test_captured_steps_replayed_over_new_inputs_and_on_other_streams():
    """Two graphs of the same calls, replayed in turn and on two streams at once, give what eager calls give."""
    d, P, H, K, parts = 128, 64, 28, 4, 2
    contexts = [1, 17, 64, 300, 1000]
    T = len(contexts)
    table = rotation(1200, d).cuda()
    pools = [Pool(contexts, K, P, d, seed=33, spread=2) for _ in range(3)]
    width = (H + 2 * K) * d
    inputs = [torch.randn((parts, T, width), generator=pools[0].g).cuda() for _ in range(4)]

    def calls(pool, qkv, two, one):
        q = ops.qkv_rope_store8(qkv, None, table, pos, seq, pool.table, torch.empty_like(two), pool.cache, pool.scales, H, K, d)
        ops.decode_attention8(q, pool.cache, pool.scales, pool.table, seq, pos, two, None, d ** -0.5)
        ops.decode_attention8_fresh(qkv, None, table, pool.cache, pool.scales, pool.table, seq, pos, one, H, None, d ** -0.5)

    pos, seq = batch([1] * T, [n - 1 for n in contexts], pools[0].slots)
    sides = [torch.cuda.Stream() for _ in range(2)]
    states = []
    for pool, stream in zip(pools[:2], sides):
        qkv = inputs[0].clone()
        two, one = (torch.empty((T, H, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream):
            calls(pool, qkv, two, one)          # (functions' attributes are set outside of a capture)
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                calls(pool, qkv, two, one)
        states.append((qkv, two, one, graph, stream))
    torch.cuda.synchronize()
    want = []
    for x in inputs:      # eager, over pages that see the same calls (the captures' run over inputs[0] among them)
        if not want:
            two, one = (torch.empty((T, H, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
            calls(pools[2], inputs[0], two, one)
        two, one = (torch.empty((T, H, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        calls(pools[2], x, two, one)
        want.append((two, one))
    for x, (two, one) in zip(inputs, want):
        for qkv, _, _, graph, stream in states:
            with torch.cuda.stream(stream):
                qkv.copy_(x)
                graph.replay()
        torch.cuda.synchronize()
        for _, got_two, got_one, _, _ in states:
            assert torch.equal(got_two, two) and torch.equal(got_one, one)
    for pool in pools[:2]:
        assert torch.equal(pool.cache.view(torch.uint8), pools[2].cache.view(torch.uint8)) and torch.equal(pool.scales, pools[2].scales)


def test_portions_on_two_streams_at_once():
    d, P, H, K = 64, 64, 4, 2
    counts, before = [200, 70], [300, 0]
    pool = Pool([c + b for c, b in zip(counts, before)], K, P, d, seed=34)
    q = torch.randn((sum(counts), H, d), generator=pool.g).bfloat16().cuda()
    plan = plan_portions(counts, before, pool.slots, H, None, "cuda")

    def call(out):
        return ops.prefill_attention8(q, pool.cache, pool.scales, pool.table, plan.tiles, out, None, 0.125, segments=plan.segments,
                                      items=plan.items, slots=plan.slots)
    want = call(torch.empty_like(q))
    outs = [torch.empty_like(q) for _ in range(4)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            call(out)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("d,H,K", [(128, 8, 2), (64, 4, 4), (128, 24, 2)])
@pytest.mark.parametrize("tile,splits", [(0, 1), (0, None), (7, 1)])
@pytest.mark.parametrize("apart,key_scale", [(0, 4.0), (16, 4.0), (20, 4.0), (24, 4.0), (40, 4.0), (100, 4.0), (60, 0.5)])
def test_a_tile_of_large_values_costs_the_others_no_bits(d, H, K, tile, splits, apart, key_scale):
    """One tile's values have scales 2^apart above the others'; its keys point away from the queries, so that it has hardly any weight (or,
    in the last case, little enough that its values still decide)."""
    P, n = 64, 512
    pool = Pool([n], K, P, d, seed=41 + d)
    page = int(pool.table[pool.slots[0], tile])
    pool.cache[page, 0] = torch.full((K, P, d), -8.0, device="cuda").to(torch.float8_e4m3fn)
    pool.scales[page, 0] = key_scale
    pool.scales[page, 1] *= 2.0 ** apart
    q = torch.randn((1, H, d), generator=pool.g).abs().bfloat16()
    out = torch.full((1, H, d), math.nan, dtype=torch.bfloat16, device="cuda")
    pos, seq = batch([1], [n - 1], pool.slots)
    ops.decode_attention8(q.cuda(), pool.cache, pool.scales, pool.table, seq, pos, out, None, d ** -0.5, splits=splits)
    rows = pool.rows(pool.slots[0], n)
    want, size = attention64(q, torch.tensor([n - 1]), rows, None, d ** -0.5)
    # probabilities are rounded to float16 (2^-11; those below 2^-21 of their block's largest are off by 2^-32 of it, for n keys),
    # scores and sums in float32, the output to bfloat16 (2^-8); the other tiles' weights are all of the denominator
    rows[1, :, 64 * tile:64 * (tile + 1)] = 0
    largest = rows[1].abs().amax((1, 2)).repeat_interleave(H // K, 0)[None, :, None]
    tolerance = size * (2.0 ** -11 + 2.0 ** -16) + want.abs() * 2.0 ** -8 + largest * n * 2.0 ** -32
    assert ((out.cpu().double() - want).abs() <= tolerance * 1.01 + 1e-30).all()


@pytest.mark.parametrize("count,before,kernels", [(40, 10, 2), (300, 5000, 3)])
def test_launches_of_portions_are_counted(count, before, kernels):
    d, P, H, K = 64, 64, 4, 2
    pool = Pool([count + before], K, P, d, seed=50)
    q = torch.zeros((count, H, d), dtype=torch.bfloat16, device="cuda")
    plan = plan_portions([count], [before], pool.slots, H, None, "cuda")
    assert (plan.items is not None and plan.items.shape[0] > 0) == (kernels == 3)
    launched = ops.launches
    ops.prefill_attention8(q, pool.cache, pool.scales, pool.table, plan.tiles, torch.empty_like(q), None, 0.1, segments=plan.segments,
                           items=plan.items, slots=plan.slots)
    assert ops.launches - launched == kernels


@pytest.mark.parametrize("window", [None, 50])
def test_several_portions_of_one_request(window):
    d, P, H, K = 64, 32, 4, 2
    counts, before, total = [64, 37, 1, 200], [10, 74, 111, 112], 312
    pool = Pool([total, 90], K, P, d, seed=51)
    poison(pool, pool.slots[0], total)
    slots = [pool.slots[0]] * 4
    q = (torch.randn((sum(counts) + 90, H, d), generator=pool.g) * 4).bfloat16()
    out = torch.full(q.shape, math.nan, dtype=torch.bfloat16, device="cuda")
    plan = plan_portions(counts + [90], before + [0], slots + [pool.slots[1]], H, window, "cuda")
    ops.prefill_attention8(q.cuda(), pool.cache, pool.scales, pool.table, plan.tiles, out, window, d ** -0.5, segments=plan.segments,
                           items=plan.items, slots=plan.slots)
    for first, n, b, slot in ((0, 302, 10, pool.slots[0]), (302, 90, 0, pool.slots[1])):
        want, size = attention64(q[first:first + n], torch.arange(b, b + n), pool.rows(slot, b + n), window, d ** -0.5)
        tolerance = size * (2.0 ** -8 + 2 * 7.6e-5) + want.abs() * 2.0 ** -8          # (as for portions of several requests)
        assert ((out[first:first + n].cpu().double() - want).abs() <= tolerance * 1.01 + 1e-30).all()


@pytest.mark.parametrize("H,K", [(2, 4), (6, 4), (4, 0), (0, 4)])
def test_heads_that_are_not_a_multiple_are_refused(H, K):
    P, d = 64, 64
    c = torch.zeros((3, 2, K, P, d), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    s = torch.ones((3, 2, K, P // 16), device="cuda")
    bt = torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    q = torch.zeros((1, H, d), dtype=torch.bfloat16, device="cuda")
    pos, seq = batch([1], [5], [0])
    plan = plan_portions([1], [5], [0], max(H, 1), None, "cuda")
    for call in (lambda: ops.decode_attention8(q, c, s, bt, seq, pos, torch.empty_like(q), None, 1.0),
                 lambda: ops.decode_attention8(q, c, s, bt, seq, pos, torch.empty_like(q), None, 1.0, splits=2),
                 lambda: ops.prefill_attention8(q, c, s, bt, plan.tiles, torch.empty_like(q), None, 1.0),
                 lambda: ops.decode_attention8_fresh(torch.zeros((1, (H + 2 * K) * d), device="cuda"), None, rotation(8, d).cuda(), c, s, bt, seq, pos,
                                                     torch.empty_like(q), H, None, 1.0)):
        with pytest.raises(ops.KernelError):
            call()
