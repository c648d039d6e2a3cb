"""The state cache on the GPU against plain 64-bit forms (tests/state_ref.py).

Tolerances.  Codes, scales, moves, lengths and copied values have to be equal.  attend, with
u = 2^-24: a logit is a chain of at most D + 8 sums in 32 bits.  Its terms are products of q and
values (size = scale * sum |q k|, the values with one rounding of their own), or, where codes are
multiplied first, of q and codes below 144, times the scales (144 steps, steps = scale * sum |q| s),
so it is off by at most E = (D + 8) u (size + 144 steps) (32-bit inputs take the first form only:
E = (D + 8) u size).  A probability is off by exp(2 E) - 1, the hardware exp2 (2^-23, and its argument's
rounding, 3 u (size + 1)), the rounding of p times a scale to two bfloat16 terms (2^-17, not for
32-bit inputs) and sums in 32 bits (64 u): rel in all.  The output is a mean of values up to vmax
under such weights, with the same error in the sum that divides it, plus its own rounding, eps / 2."""
import math
import os

import numpy as np
import pytest
import torch

import dgs
import state_ref as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def prob_error(dim, size, steps, exact):
    e = (dim + 8) * U * (size if exact else size + 144 * steps)
    return torch.expm1(2 * e) + 2.0 ** -23 + 3 * U * (size + 1) + (0 if exact else 2.0 ** -17) + 64 * U


def states(shape, gen, dtype):
    x = torch.randn(shape, generator=gen) * (torch.rand(shape[-1], generator=gen) + 0.5)
    return (x + torch.randn(shape[-1], generator=gen) * 0.5).to(dtype).cuda()


def full_cache(pages, page, heads, dim, group, seed=0):
    """A cache whose every slot holds a row, written by the plain form."""
    gen = torch.Generator().manual_seed(seed)
    bufs = []
    for _ in range(2):
        c, s = ref.quantise(torch.randn(pages, heads, page, dim, generator=gen) +
                            torch.randn(dim, generator=gen), group)
        bufs += [ref.pack(c).cuda(), s.cuda()]
    return dgs.classes.StateCache.wrap(*bufs)


def buffers(c):
    return [c.k_codes, c.k_scales, c.v_codes, c.v_scales]


def same_bits(a, b):
    v = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[a.element_size()]
    return torch.equal(a.cpu().view(v), b.cpu().view(v))


# ------------------------------------------------------------------------------ rows
SHAPES = [(128, 64, 16, 8), (128, 128, 1, 1), (128, 32, 32, 2), (64, 64, 8, 3), (80, 40, 2, 5),
          (96, 96, 4, 2), (8, 8, 1, 1), (256, 64, 64, 2), (40, 8, 1, 4), (24, 24, 128, 1)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("dim, group, page, heads", SHAPES)
@pytest.mark.parametrize("tokens", [1, 77])
def test_write_and_read(dim, group, page, heads, tokens, dtype):
    gen = torch.Generator().manual_seed(dim + tokens)
    pages = -(-(tokens + 5) // page)
    cache = dgs.classes.StateCache(pages, page, heads, dim, group)
    before = [b.fill_(7) for b in buffers(cache)]
    before = [b.clone() for b in before]
    qkv = states((tokens, 3 * heads, dim), gen, TYPES[dtype])
    k, v = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]  # views of a fused projection
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    slots[tokens // 2] = -1 if tokens > 1 else slots[0]
    cache.write(k, v, slots.cuda())
    live = slots >= 0
    for x, codes, scales, c0, s0 in ((k, cache.k_codes, cache.k_scales, before[0], before[1]),
                                     (v, cache.v_codes, cache.v_scales, before[2], before[3])):
        qc, qs = ref.quantise(x, group)
        c0, s0 = c0.cpu(), s0.cpu()
        at = slots[live] // page, slots[live] % page
        c0[at[0], :, at[1]], s0[at[0], :, at[1]] = ref.pack(qc[live]), qs[live]
        assert same_bits(codes, c0) and same_bits(scales, s0)  # others left as they were
    for t in TYPES.values():
        got = cache.read(slots.int().cuda(), t)
        for x, g in zip((k, v), got):
            qc, qs = ref.quantise(x, group)
            want = ref.values(ref.pack(qc), qs)
            want[~live] = 0
            # s * c has 12 bits; one rounding to 32 bits, one more to a 16-bit type
            assert torch.equal(g.cpu(), want.float().to(t))


def test_quantiser_borders():
    """Groups where the code hangs on a rounding: ties, tiny, constant and wide ranges, signs."""
    gen = torch.Generator().manual_seed(3)
    n, dim, group = 4096, 64, 8
    x = torch.randn(n, 1, dim, generator=gen)
    g = x.view(n, dim // 8, 8)
    g[:512, :, 0], g[:512, :, 7] = 0, 15  # scale 1, base 0: halves are ties
    g[:512, :, 1:7] = torch.randint(0, 30, (512, dim // 8, 6), generator=gen) / 2
    g[512:700] = torch.nextafter(g[:188], torch.tensor(8.0))
    g[700:900] *= 1e-38
    g[900:1000] *= 1e-41  # below the normal range
    g[1000:1100] = g[1000:1100, :, :1]
    g[1100:1200] *= 1e37
    g[1200:1300] += 1000
    g[1300:1400] = 0
    g[1400:1500] = -0.0
    for i, bad in enumerate((math.nan, math.inf, -math.inf)):
        g[1500 + 50 * i:1550 + 50 * i, ::2, i] = bad
    g[1700:1750, :, 0], g[1700:1750, :, 1] = 3e38, -3e38
    cache = dgs.classes.StateCache(n, 1, 1, dim, group)
    cache.write(x.cuda(), x.flip(0).cuda(), torch.arange(n).cuda())
    codes, scales = ref.quantise(x, group)
    assert torch.equal(cache.k_codes.cpu()[:, 0, 0], ref.pack(codes)[:, 0])
    nan = scales.isnan()[:, 0]
    assert torch.equal(cache.k_scales.cpu()[:, 0, 0].isnan(), nan)
    got = cache.k_scales.cpu()[:, 0, 0]
    assert torch.equal(torch.where(nan, 0, got), torch.where(nan, 0, scales[:, 0]))
    k, v = cache.read(torch.arange(n).cuda())
    want = ref.values(ref.pack(codes), scales).float()
    assert torch.equal(k.cpu().isnan(), want.isnan())
    assert torch.equal(k.cpu().nan_to_num(), want.nan_to_num())
    assert torch.equal(v.cpu().nan_to_num(), want.flip(0).nan_to_num())


@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
def test_append(ids):
    gen = torch.Generator().manual_seed(5)
    n, page, heads, dim = 13, 4, 3, 64
    lens = torch.randint(0, 20, (n,), generator=gen)
    lens[0], lens[1] = 0, 19  # the first slot, the last slot of the table
    table = torch.randperm(n * 5, generator=gen).view(n, 5)
    cache = dgs.classes.StateCache(n * 5, page, heads, dim)
    other = dgs.classes.StateCache(n * 5, page, heads, dim)
    k, v = (states((n, heads, dim), gen, torch.bfloat16) for _ in range(2))
    slots = cache.append(k, v, table.to(ids).cuda(), lens.to(ids).cuda())
    want = table[torch.arange(n), lens // page] * page + lens % page
    assert torch.equal(slots.cpu(), want)
    other.write(k, v, want.cuda())
    assert all(same_bits(a, b) for a, b in zip(buffers(cache), buffers(other)))


def test_empty_calls():
    cache = dgs.classes.StateCache(2, 4, 2, 64)
    z = torch.zeros(0, 2, 64, device="cuda")
    i = torch.zeros(0, dtype=torch.int64, device="cuda")
    cache.write(z, z, i)
    assert cache.append(z, z, i.view(0, 1), i).shape == (0,)
    assert cache.read(i)[0].shape == (0, 2, 64)
    assert cache.attend(z, i.view(0, 1), i).shape == (0, 2, 64)
    q = torch.randn(3, 4, 64, device="cuda")
    out = cache.attend(q, torch.zeros(3, 0, dtype=torch.int32, device="cuda"),
                       torch.zeros(3, dtype=torch.int32, device="cuda"))
    assert torch.equal(out, torch.zeros_like(q))
    w = torch.zeros(0, 2, 8, device="cuda")
    got = dgs.ops.evict_rows([cache.k_codes], w, None, i.view(0, 2), i, 4)
    assert got[0].shape == (0, 2, 8) and got[2].shape == (0,)


# ------------------------------------------------------------------------------ attention
def check_attend(cache, q, table, lens, scale=None, weights=None, decay=1.0):
    dim = cache.head_dim
    want, prob, size, steps, vmax = ref.attend(q, cache, table, lens,
                                               dim ** -0.5 if scale is None else scale)
    before = None if weights is None else weights.clone()
    got = cache.attend(q, table, lens, scale=scale, weights=weights, decay=decay)
    assert got.dtype == q.dtype and got.shape == q.shape
    rel = prob_error(dim, size, steps, q.dtype == torch.float32)
    off = (2 * rel * vmax)[..., None]
    tol = off + torch.finfo(q.dtype).eps / 2 * (want.abs() + off)
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half a step below the normal range
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), (float(err.max()), float(tol.max()))
    if weights is not None:
        cap, g = prob.shape[2], q.shape[1] // cache.heads
        inside = torch.arange(cap) < lens.cpu().long()[:, None, None]
        old = before.cpu().double()[..., :cap]
        exp = torch.where(inside, prob + (decay * old if decay else 0.0), old)
        werr = (weights.cpu().double()[..., :cap] - exp).abs()
        wrel = 2 * rel.unflatten(1, (cache.heads, g)).amax(2)[..., None]
        wtol = wrel * prob + (g + 4) * U * exp.abs()
        assert bool((werr <= wtol)[inside.expand_as(werr)].all()), float(werr.max())
        keep = torch.ones_like(before, dtype=torch.bool)
        keep[..., :cap] = ~inside.cuda()
        assert same_bits(weights[keep], before[keep])  # behind the lengths nothing changes
    return got


ATTEND = [  # q_heads, heads, dim, group, page
    (8, 2, 128, 64, 16), (32, 8, 128, 64, 16), (4, 4, 32, 32, 1), (12, 12, 80, 40, 8),
    (7, 1, 128, 128, 64), (16, 1, 128, 32, 2), (6, 2, 64, 32, 4), (4, 1, 256, 64, 32),
    (20, 1, 64, 64, 128), (5, 5, 96, 96, 16), (2, 2, 8, 8, 1), (33, 1, 128, 64, 32),
    (9, 3, 24, 8, 4), (70, 1, 32, 32, 8), (8, 8, 128, 64, 1), (4, 2, 192, 64, 16)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("q_heads, heads, dim, group, page", ATTEND)
@pytest.mark.parametrize("keep", [False, True])
def test_attend(q_heads, heads, dim, group, page, dtype, keep):
    gen = torch.Generator().manual_seed(q_heads * dim + page)
    lens = torch.tensor([0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 130, 257, 300])
    rows, width = len(lens), -(-300 // page)
    cache = full_cache(rows * width + 1, page, heads, dim, group, seed=dim)
    table = (torch.randperm(rows * width, generator=gen) + 1).view(rows, width)
    # what lies behind a row's length must not matter: NaN in its slots, ids of no page
    for i, n in enumerate(lens.tolist()):
        for p in range(n // page, width):
            first = n - p * page if p == n // page else 0
            cache.k_scales[table[i, p], :, max(first, 0):] = math.nan
            cache.v_scales[table[i, p], :, max(first, 0):] = math.nan
            if first == 0:
                table[i, p] = -12345 if p % 2 else 2 ** 31 - 1
    q = states((rows, q_heads, dim), gen, TYPES[dtype])
    w = torch.rand(rows, heads, width * page + 3, generator=gen).cuda() if keep else None
    check_attend(cache, q, table.int().cuda(), lens.cuda(), weights=w,
                 decay=[1.0, 0.5, 0.0][dim % 3])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("q_heads, heads, dim, group, page", [
    (8, 2, 128, 64, 16), (16, 1, 64, 64, 1), (3, 3, 80, 40, 8), (40, 1, 128, 128, 64)])
def test_attend_long(q_heads, heads, dim, group, page, dtype):
    """Rows long enough to be split, beside short ones; each page used by several rows."""
    gen = torch.Generator().manual_seed(dim)
    lens = torch.tensor([20011, 1, 0, 4097, 12288, 777])
    pages = 30000 // page
    cache = full_cache(pages, page, heads, dim, group, seed=1)
    table = torch.randint(0, pages, (len(lens), -(-20480 // page)), generator=gen)
    q = states((len(lens), q_heads, dim), gen, TYPES[dtype])
    w = torch.zeros(len(lens), heads, table.shape[1] * page, device="cuda")
    check_attend(cache, q, table.cuda(), lens.int().cuda(), weights=w)
    check_attend(cache, q, table.int().cuda(), lens.cuda(), scale=0.3)


@pytest.mark.parametrize("rows, high, heads, g, page", [
    (600, 3000, 1, 2, 16), (1024, 1500, 1, 1, 4), (1025, 1500, 1, 2, 16), (1100, 500, 1, 20, 8),
    (700, 600, 1, 4, 32), (300, 900, 2, 3, 2), (1, 5000, 1, 1, 64), (2, 1100, 2, 17, 1024)])
@pytest.mark.parametrize("keep", [False, True])
def test_attend_ragged_rows(rows, high, heads, g, page, keep):
    """Many rows of very different lengths, most of them short or empty, some long: every way of
    cutting the work."""
    gen = torch.Generator().manual_seed(rows)
    lens = (torch.rand(rows, generator=gen) ** 12 * high).long()
    lens[rows // 2], lens[-1] = high, (0 if rows > 2 else high - 1)
    lens[rows // 3:rows // 3 + 70] = 0 if rows > 300 else lens[rows // 3]
    pages = 4000 // page + 1
    cache = full_cache(pages, page, heads, 64, 64, seed=3)
    table = torch.randint(0, pages, (rows, -(-high // page)), generator=gen)
    q = states((rows, heads * g, 64), gen, torch.bfloat16)
    w = torch.rand(rows, heads, table.shape[1] * page, generator=gen).cuda() if keep else None
    check_attend(cache, q, table.int().cuda(), lens.cuda(), weights=w)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("page", [1, 16])
def test_attend_scale_zero(dtype, page):
    """All logits equal: the mean of the values."""
    gen = torch.Generator().manual_seed(0)
    cache = full_cache(4096 // page, page, 2, 64, 64)
    q = states((3, 4, 64), gen, TYPES[dtype])
    table = torch.randint(0, 4096 // page, (3, 2048 // page), generator=gen).cuda()
    check_attend(cache, q, table, torch.tensor([2001, 5, 0]).cuda(), scale=0.0)
    check_attend(cache, q, table[:, :64 // page].contiguous(), torch.tensor([61, 5, 0]).cuda(),
                 scale=0.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_many_short_rows(dtype):
    """Sampled neighbours: many rows of at most 15 slots, pages of one slot."""
    gen = torch.Generator().manual_seed(2)
    rows, nodes = 3001, 5000
    cache = full_cache(nodes, 1, 4, 32, 32)
    table = torch.randint(0, nodes, (rows, 15), generator=gen)
    lens = torch.randint(0, 16, (rows,), generator=gen)
    q = states((rows, 4, 32), gen, TYPES[dtype])
    w = torch.full((rows, 4, 15), 0.25, device="cuda")
    check_attend(cache, q, table.cuda(), lens.cuda(), weights=w)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_attend_large_logits(dtype):
    """Logits far apart: one slot takes everything, also when a later chunk holds it."""
    gen = torch.Generator().manual_seed(4)
    cache = full_cache(64, 64, 2, 128, 64)
    q = (torch.randn(3, 8, 128, generator=gen) * 4).to(TYPES[dtype]).cuda()
    table = torch.randperm(64, generator=gen)[None].repeat(3, 1).cuda()
    lens = torch.tensor([4096, 4001, 5]).cuda()
    for scale in (1.0, -1.0):
        check_attend(cache, q, table, lens, scale=scale)


def test_attend_nan_and_infinity_stay_in_their_rows():
    cache = full_cache(8, 16, 2, 128, 64)
    q = torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    table = torch.arange(8).view(4, 2).cuda()
    lens = torch.tensor([32, 20, 32, 17]).cuda()
    clean = cache.attend(q, table, lens)
    cache.k_scales[3, 0, 3] = math.nan  # row 1, slot 19, head 0
    cache.v_scales[3, 1, 4] = math.nan  # behind row 1's length
    q2 = q.clone()
    q2[2, 5] = math.inf
    q2[3, 0, 7] = math.nan
    got = cache.attend(q2, table, lens)
    bad = torch.zeros(4, 8, dtype=torch.bool)
    bad[1, :4] = bad[2, 5] = bad[3, 0] = True
    assert torch.equal(got.isnan().all(-1).cpu(), bad)
    assert torch.equal(got.isnan().any(-1).cpu(), bad)
    assert torch.equal(got[~bad], clean[~bad])


def test_attend_views_and_repeats():
    """Strided queries and weights of another step; the same call twice gives the same bits."""
    gen = torch.Generator().manual_seed(9)
    cache = full_cache(40, 16, 2, 128, 64)
    qkv = states((5, 12, 128), gen, torch.bfloat16)
    table = torch.randperm(40, generator=gen).view(5, 8).cuda()
    lens = torch.tensor([128, 7, 0, 100, 33]).cuda()
    q = qkv[:, 2:10]
    a = check_attend(cache, q, table, lens)
    assert torch.equal(a, cache.attend(q.contiguous(), table, lens))
    odd = torch.empty(5 * 8 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(5, 8, 128)
    odd.copy_(q)  # rows that are not 16-byte aligned
    assert torch.equal(a, cache.attend(odd, table, lens))
    assert torch.equal(a, cache.attend(q.transpose(0, 1).contiguous().transpose(0, 1), table, lens))
    every = table.repeat_interleave(2, 1)[:, ::2]
    assert torch.equal(a, cache.attend(q, every, lens.int()))


def test_offsets_past_32_bits():
    """Rows past 2^31 and 2^32 bytes of a buffer."""
    pages, page, heads, dim = 300000, 64, 4, 128
    bufs = []
    for _ in range(2):
        bufs += [torch.empty(pages, heads, page, dim // 2, dtype=torch.uint8, device="cuda"),
                 torch.empty(pages, heads, page, 2, 2, dtype=torch.bfloat16, device="cuda")]
    assert bufs[0].numel() > 2 ** 32
    cache = dgs.classes.StateCache.wrap(*bufs)
    gen = torch.Generator().manual_seed(0)
    use = torch.tensor([3, 131071, 131073, 262145, 299999])
    slots = (use[:, None] * page + torch.arange(page)).flatten()
    k, v = (states((slots.numel(), heads, dim), gen, torch.bfloat16) for _ in range(2))
    cache.write(k, v, slots.cuda())
    got = cache.read(slots.cuda())
    small = dgs.classes.StateCache(5, page, heads, dim)
    small.write(k, v, torch.arange(5 * page).cuda())
    want = small.read(torch.arange(5 * page).cuda())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q = states((1, 16, dim), gen, torch.bfloat16)
    n = torch.tensor([5 * page - 3]).cuda()
    assert torch.equal(cache.attend(q, use[None].cuda(), n),
                       small.attend(q, torch.arange(5)[None].cuda(), n))
    # eviction moves rows out there too
    w = torch.rand(1, heads, 5 * page, generator=gen).cuda()
    a = cache.evict(w, None, use[None].cuda(), n, 100)
    b = small.evict(w, None, torch.arange(5)[None].cuda(), n, 100)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(cache.read(slots[:100].cuda())[1],
                       small.read(torch.arange(100).cuda())[1])


# ------------------------------------------------------------------------------ eviction
@pytest.mark.parametrize("rows, heads, page, width, budget, sinks, recent", [
    (7, 2, 16, 12, 64, 2, 8), (3, 1, 1, 77, 50, 0, 10), (5, 3, 8, 40, 1, 0, 0),
    (4, 2, 64, 40, 700, 4, 300), (2, 4, 32, 200, 6300, 0, 1), (3, 2, 4, 20, 80, 3, 77),
    (2, 1, 16, 8, 500, 1, 1), (3, 2, 2, 1500, 1024, 0, 0), (2, 2, 3, 30, 40, 1, 2)])
@pytest.mark.parametrize("ids", [torch.int32, torch.int64])
@pytest.mark.parametrize("given", [False, True])
def test_evict(rows, heads, page, width, budget, sinks, recent, ids, given):
    rng = np.random.default_rng(rows * width + budget)
    cap = width * page
    lens = rng.integers(0, cap + 1, rows)
    lens[0] = cap
    if rows > 2:
        lens[1], lens[2] = 0, min(budget + 1, cap)
    w = np.exp(rng.standard_normal((rows, heads, cap + 5)) * 2).astype(np.float32)
    w = np.where(rng.random(w.shape) < 0.5, np.round(w), w)  # many ties
    w[rng.random(w.shape) < 0.05] = 0.0
    w[rng.random(w.shape) < 0.02] = -0.0
    w[rng.random(w.shape) < 0.02] = np.nan
    w[rng.random(w.shape) < 0.01] = np.inf
    w[rng.random(w.shape) < 0.01] = -np.inf
    w = w.astype(np.float32)
    pos = None
    if given:
        pos = np.stack([rng.permutation(3 * cap + 15)[:cap + 5] for _ in range(rows * heads)])
        pos = pos.reshape(rows, heads, cap + 5).astype(np.int32)
    table = rng.permutation(rows * width + 3)[:rows * width].reshape(rows, width)
    pages = rows * width + 3
    gen = torch.Generator().manual_seed(1)
    stores = [torch.randn(pages, heads, page, 40, generator=gen).bfloat16().cuda(),
              torch.randint(0, 255, (pages, heads, page, 7), generator=gen).byte().cuda(),
              torch.randn(pages, heads, page, generator=gen).cuda(),
              torch.randn(pages, heads, page, 3, 5, generator=gen).cuda()]
    want_w, want_p, want_n, moves = ref.evict(w, pos, lens, budget, sinks, recent)
    expect = [s.cpu().clone() for s in stores]
    if moves:
        i, h, s, d = (torch.tensor(x) for x in zip(*moves))
        t = torch.tensor(table)
        for e in expect:
            e[t[i, d // page], h, d % page] = e[t[i, s // page], h, s % page].clone()
    tab = torch.tensor(table)
    for r, n in enumerate(lens):
        tab[r, -(-int(n) // page):] = -1
    for again in range(2):  # a second call on the same inputs gives the same
        got_w, got_p, got_n = dgs.ops.evict_rows(
            stores, torch.tensor(w).cuda(), None if pos is None else torch.tensor(pos).cuda(),
            tab.to(ids).cuda(), torch.tensor(lens).to(ids).cuda(), budget, sinks=sinks,
            recent=recent)
        assert got_n.dtype == ids and np.array_equal(got_n.cpu().numpy(), want_n)
        assert np.array_equal(got_p.cpu().numpy(), want_p)
        assert np.array_equal(got_w.cpu().numpy(), want_w, equal_nan=True)
        for a, b in zip(stores, expect):
            assert same_bits(a, b)


@pytest.mark.parametrize("value", [0.0, math.nan, math.inf, 1.0])
def test_evict_all_equal(value):
    """Only ties: the first slots stay, nothing moves."""
    st = torch.arange(64.0, device="cuda").view(4, 1, 16, 1)
    w = torch.full((1, 1, 64), value, device="cuda")
    before = st.clone()
    _, p, n = dgs.ops.evict_rows([st], w, None, torch.arange(4).view(1, 4).cuda(),
                                 torch.tensor([61]).cuda(), 20)
    assert torch.equal(st, before) and n.item() == 20
    assert p[0, 0, :20].tolist() == list(range(20)) and bool((p[0, 0, 20:] == -1).all())


def test_evict_long():
    """One long row: every digit of the selection and every chunk of the numbering."""
    rng = np.random.default_rng(0)
    cap, budget = 131072, 4096
    w = rng.random((1, 2, cap), dtype=np.float32)
    st = torch.arange(2 * cap, dtype=torch.int32, device="cuda").view(cap // 64, 2, 64, 1)
    before = st.cpu().clone()
    lens = np.array([cap - 5])
    want_w, want_p, _, moves = ref.evict(w, None, lens, budget, 4, 1000)
    t = torch.arange(cap // 64).view(1, -1).cuda()
    got_w, got_p, _ = dgs.ops.evict_rows([st], torch.tensor(w).cuda(), None, t,
                                         torch.tensor(lens).cuda(), budget, 4, 1000)
    assert np.array_equal(got_p.cpu().numpy(), want_p)
    assert np.array_equal(got_w.cpu().numpy(), want_w)
    for _, h, s, d in moves:
        before[d // 64, h, d % 64] = before[s // 64, h, s % 64]
    assert torch.equal(st.cpu(), before)


# ------------------------------------------------------------------------------ errors, streams
def raises_next(match):
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match=match):
        dgs.ops._check_async_errors()
    dgs.ops._check_async_errors()


def test_ids_outside_are_left_out_and_reported():
    """The kernels compare every page, slot and length with its bound before they use it."""
    gen = torch.Generator().manual_seed(0)
    cache = full_cache(8, 16, 2, 128, 64)
    before = [b.clone() for b in buffers(cache)]
    k = states((2, 2, 128), gen, torch.bfloat16)
    cache.write(k, k, torch.tensor([8 * 16, -1]).cuda())
    raises_next("page or slot 128, outside")
    one = torch.tensor([[3], [8]]).cuda()
    assert cache.append(k, k, one, torch.tensor([16, 0]).cuda()).tolist() == [-1, -1]
    raises_next("state cache call met")
    assert all(same_bits(a, b) for a, b in zip(buffers(cache), before))
    assert bool((cache.read(torch.tensor([128]).cuda())[0] == 0).all())
    raises_next("page or slot 128, outside")
    q = states((2, 8, 128), gen, torch.bfloat16)
    ok = cache.attend(q, torch.tensor([[1, 2], [3, 4]]).cuda(), torch.tensor([16, 32]).cuda())
    got = cache.attend(q, torch.tensor([[1, 9], [3, 4]]).cuda(), torch.tensor([32, 32]).cuda())
    raises_next("page or slot 9, outside")
    assert torch.equal(got[1], ok[1])
    torch.testing.assert_close(got[0], ok[0], rtol=2 ** -7, atol=2 ** -8)
    got = cache.attend(q, torch.tensor([[1, 2], [3, 4]]).cuda(), torch.tensor([16, 33]).cuda())
    raises_next("length 33, outside")
    assert torch.equal(got, ok)
    w = torch.rand(1, 2, 32, generator=gen).cuda()
    _, _, n = cache.evict(w, None, torch.tensor([[1, 2]]).cuda(), torch.tensor([40]).cuda(), 8)
    raises_next("length 40, outside")
    assert n.item() == 8
    w = torch.arange(32.0).expand(1, 2, 32).contiguous().cuda()
    now = [b.clone() for b in buffers(cache)]
    cache.evict(w, None, torch.tensor([[-3, 99]]).cuda(), torch.tensor([32]).cuda(), 8)
    raises_next("page or slot")
    assert all(same_bits(a, b) for a, b in zip(buffers(cache), now))


def test_streams_run_independently():
    gen = torch.Generator().manual_seed(0)
    cache = full_cache(256, 16, 2, 128, 64)
    table = torch.randperm(256, generator=gen).view(2, 128).cuda()
    lens = torch.tensor([2048, 1999]).cuda()
    qs = [states((2, 8, 128), gen, torch.bfloat16) for _ in range(4)]
    ws = [torch.zeros(2, 2, 2048, device="cuda") for _ in range(4)]
    want = [cache.attend(q, table, lens) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [None] * 4
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = cache.attend(qs[i], table, lens, weights=ws[i], decay=0.0)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graphs_replay_as_eager():
    """A captured decoding step (append, attend, evict) and a second graph on the same cache,
    replayed between eager calls with new inputs in place."""
    gen = torch.Generator().manual_seed(0)
    page, heads, dim, budget = 16, 2, 128, 40
    cache = full_cache(8, page, heads, dim, 64)
    table = torch.randperm(8, generator=gen).view(2, 4).cuda()
    lens = torch.tensor([40, 23]).cuda()
    k, v = (states((2, heads, dim), gen, torch.bfloat16) for _ in range(2))
    q = states((2, 8, dim), gen, torch.bfloat16)
    w0 = torch.rand(2, heads, 64, generator=gen).cuda()
    w = w0.clone()
    bufs0 = [b.clone() for b in buffers(cache)]

    def step():
        cache.append(k, v, table, lens)
        n = lens + 1
        w.copy_(w0)
        out = cache.attend(q, table, n, weights=w)
        return (out,) + tuple(cache.evict(w, None, table, n, budget, sinks=1, recent=4))

    def look():
        return cache.attend(q, table, lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), look()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        r1 = step()
    with torch.cuda.graph(g2):
        r2 = look()
    for turn in range(4):
        for t in (k, v, q):
            t.copy_(states(t.shape, gen, torch.bfloat16))
        for a, b in zip(buffers(cache), bufs0):
            a.copy_(b)
        want2 = look().clone()
        want = [t.clone() for t in step()]
        after = [b.clone() for b in buffers(cache)]
        for a, b in zip(buffers(cache), bufs0):
            a.copy_(b)
        g2.replay()
        got2 = r2.clone()
        g1.replay()
        torch.cuda.synchronize()
        assert torch.equal(got2, want2), turn
        assert all(torch.equal(a, b) for a, b in zip(r1, want)), turn
        assert all(same_bits(a, b) for a, b in zip(buffers(cache), after)), turn


# ------------------------------------------------------------------------------ together
def test_sampled_neighbours_attend():
    """Sample a block, hold every node's states in the cache (page = node id), attend to the
    sampled neighbours."""
    from DistGNN.dataloading.synthetic import rmat_csc_numpy
    indptr, indices = rmat_csc_numpy(10, 8, seed=3)
    n = indptr.size - 1
    sampler = dgs.classes.P2PCacheSampler(torch.from_numpy(indptr), torch.from_numpy(indices),
                                          torch.Tensor(), torch.arange(n), 0)
    dgs.ops._CAPI_set_random_seed(5)
    seeds = torch.randperm(n, generator=torch.Generator().manual_seed(0))[:200].cuda()
    blocks = sampler._CAPI_sample_node_classifiction(seeds, [15, 5], False)
    gen = torch.Generator().manual_seed(0)
    heads, dim = 4, 32
    cache = dgs.classes.StateCache(n, 1, heads, dim)
    k, v = (states((n, heads, dim), gen, torch.float32) for _ in range(2))
    cache.write(k, v, torch.arange(n).cuda())
    for block, fan_out in zip(blocks, (5, 15)):
        table, lens = dgs.ops.neighbour_table(block, fan_out)
        row, col = block[2].cpu().numpy(), block[3].cpu().numpy()
        front = block[1].cpu().numpy()
        for i in range(0, block[0].numel(), 17):
            assert sorted(table[i, :lens[i]].tolist()) == sorted(front[col[row == i]].tolist())
        q = states((block[0].numel(), heads, dim), gen, torch.float32)
        check_attend(cache, q, table, lens,
                     weights=torch.zeros(lens.numel(), heads, fan_out, device="cuda"))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decoding_with_a_full_cache(dtype):
    """Append, attend with weights, evict, over many steps; every step against the plain forms on
    the state that the step before left."""
    gen = torch.Generator().manual_seed(0)
    seqs, heads, q_heads, dim, page, budget = 3, 2, 6, 64, 8, 30
    cache = dgs.classes.StateCache(seqs * 5, page, heads, dim, 32)
    table = torch.randperm(seqs * 5, generator=gen).view(seqs, 5).int().cuda()
    cap = 5 * page
    lens = torch.tensor([0, 25, 30], dtype=torch.int32).cuda()
    start = torch.randn(cap, heads, dim, generator=gen).to(TYPES[dtype]).cuda()
    for i, n in enumerate(lens.tolist()):
        j = torch.arange(n)
        cache.write(start[:n], start[:n].flip(0), table[i, j // page].long() * page + j.cuda() % page)
    weights = torch.zeros(seqs, heads, cap, device="cuda")
    pos = torch.arange(cap, dtype=torch.int32).repeat(seqs, heads, 1).cuda()
    token = lens.clone()
    for _ in range(12):
        k, v = (states((seqs, heads, dim), gen, TYPES[dtype]) for _ in range(2))
        slots = cache.append(k, v, table, lens)
        got = cache.read(slots)
        want = ref.values(*[x if i else ref.pack(x) for i, x in enumerate(ref.quantise(k, 32))])
        assert torch.equal(got[0].cpu(), want.float())
        pos[torch.arange(seqs), :, lens.long()] = token[:, None]
        lens, token = lens + 1, token + 1
        q = states((seqs, q_heads, dim), gen, TYPES[dtype])
        check_attend(cache, q, table, lens, weights=weights)
        ww, wp, wn, moves = ref.evict(weights.cpu().numpy(), pos.cpu().numpy(),
                                      lens.cpu().numpy(), budget, 2, 5)
        expect = [b.cpu().clone() for b in buffers(cache)]
        t = table.cpu().long()
        for i, h, s, d in moves:
            for e in expect:
                e[t[i, d // page], h, d % page] = e[t[i, s // page], h, s % page]
        weights, pos, lens = cache.evict(weights, pos, table, lens, budget, sinks=2, recent=5)
        assert np.array_equal(weights.cpu().numpy(), ww) and np.array_equal(pos.cpu().numpy(), wp)
        assert np.array_equal(lens.cpu().numpy(), wn)
        assert all(same_bits(a, b) for a, b in zip(buffers(cache), expect))
    assert lens.tolist() == [12, 30, 30]


def test_a_refused_registration_is_not_reported_again():
    """Where the driver does not map memory that exists already, the call that asked for it raises,
    and the launches after it do not."""
    host = torch.zeros(4096, dtype=torch.uint8)
    try:
        dgs.ops._CAPI_tensor_pin_memory(host)
    except RuntimeError as e:
        assert "hipHostRegister" in str(e)
    else:
        dgs.ops._CAPI_tensor_unpin_memory(host)
    cache = full_cache(2, 4, 1, 64, 64)
    got = cache.read(torch.arange(8).cuda())
    assert got[0].shape == (8, 1, 64) and torch.isfinite(got[0]).all()


@pytest.mark.parametrize("dim, group, heads, g, dtype", [
    (80, 40, 3, 1, "f16"), (96, 32, 1, 3, "bf16"), (128, 64, 2, 2, "f32"), (256, 64, 1, 1, "f32"),
    (16, 8, 2, 5, "bf16"), (32, 32, 2, 4, "f32"), (40, 40, 1, 7, "f32")])
@pytest.mark.parametrize("rows, high, page", [(300, 1000, 8), (1024, 700, 16), (1025, 700, 1),
                                              (3, 6000, 64), (1, 520, 1), (40, 600, 128)])
def test_attend_ragged_rows_of_every_size(dim, group, heads, g, dtype, rows, high, page):
    """As test_attend_ragged_rows, for the channels, groups and types of the vector form."""
    gen = torch.Generator().manual_seed(rows + dim)
    lens = (torch.rand(rows, generator=gen) ** 8 * high).long()
    lens[rows // 2], lens[-1] = high, (0 if rows > 2 else high - 1)
    lens[rows // 3:rows // 3 + 70] = 0 if rows > 200 else lens[rows // 3]
    pages = 2000 // page + 1
    cache = full_cache(pages, page, heads, dim, group, seed=4)
    table = torch.randint(0, pages, (rows, -(-high // page)), generator=gen)
    q = states((rows, heads * g, dim), gen, TYPES[dtype])
    w = torch.rand(rows, heads, table.shape[1] * page, generator=gen).cuda()
    w = w if rows % 2 else None
    check_attend(cache, q, table.int().cuda() if page > 1 else table.cuda(), lens.cuda(), weights=w)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cap", [16, 64, 2048])
def test_lengths_outside_are_reported_however_the_work_is_cut(cap, dtype):
    gen = torch.Generator().manual_seed(cap)
    cache = full_cache(cap // 16, 16, 2, 64, 64)
    table = torch.arange(cap // 16, dtype=torch.int32).repeat(3, 1).cuda()
    q = states((3, 4, 64), gen, TYPES[dtype])
    for bad, shown in ((-1, "length -1, outside"), (cap + 1, f"length {cap + 1}, outside")):
        got = cache.attend(q, table, torch.tensor([bad, cap, 5]).cuda())
        raises_next(shown)
        # the nearest length inside; equal bits, as the batch is cut in the same places
        near = torch.tensor([min(max(bad, 0), cap), cap, 5]).cuda()
        assert torch.equal(got, cache.attend(q, table, near))


@pytest.mark.parametrize("dim, group, g, dtype", [
    (64, 64, 1, "f32"), (40, 40, 2, "bf16"), (96, 32, 1, "bf16"), (96, 24, 2, "f16"),
    (128, 32, 2, "f32"), (120, 40, 1, "f16"), (192, 64, 1, "f32"), (176, 88, 2, "bf16"),
    (256, 128, 2, "f32"), (248, 8, 1, "f32"), (32, 32, 1, "f32")])
@pytest.mark.parametrize("rows, high", [(600, 1000), (1100, 500)])
def test_attend_many_slots_of_every_size(dim, group, g, dtype, rows, high):
    """Batches with slots enough that a lane takes several words of a row."""
    gen = torch.Generator().manual_seed(dim)
    lens = (torch.rand(rows, generator=gen) ** 6 * high).long()
    lens[7], lens[8] = high, 0
    cache = full_cache(high // 8, 16, 2, dim, group, seed=5)
    table = torch.randint(0, high // 8, (rows, -(-high // 16)), generator=gen)
    q = states((rows, 2 * g, dim), gen, TYPES[dtype])
    w = torch.rand(rows, 2, table.shape[1] * 16, generator=gen).cuda() if g == 1 else None
    check_attend(cache, q, table.int().cuda(), lens.cuda(), weights=w)


@pytest.mark.parametrize("cols", [1, 5, 63, 64, 65, 200, 256, 257, 1000])
@pytest.mark.parametrize("share", [0.1, 0.5, 0.95])
def test_evict_short_rows(cols, share):
    """Rows of few slots with many ties: every length there can be, four stores of odd rows."""
    rng = np.random.default_rng(cols)
    lens = np.unique(np.concatenate([np.arange(min(cols, 70) + 1), [cols // 2, cols - 1, cols]]))
    rows, heads, budget = len(lens), 3, max(1, int(cols * share))
    w = rng.integers(0, 5, (rows, heads, cols)).astype(np.float32) * 0.5 - 1
    w[rng.random(w.shape) < 0.1] = np.nan
    pos = rng.permuted(np.tile(np.arange(cols, dtype=np.int32) * 2, (rows, heads, 1)), axis=-1)
    sinks, recent = budget // 3, budget // 2
    table = rng.permutation(rows * cols).reshape(rows, cols)
    stores = [torch.from_numpy(rng.integers(0, 256, (rows * cols, heads, 1, n), dtype=np.uint8)).cuda()
              for n in (3, 16, 40, 272)]
    expect = [s.cpu().clone() for s in stores]
    want_w, want_p, want_n, moves = ref.evict(w, pos, lens, budget, sinks, recent)
    t = torch.from_numpy(table)
    for i, h, s, d in moves:
        for e in expect:
            e[t[i, d], h] = e[t[i, s], h]
    got_w, got_p, got_n = dgs.ops.evict_rows(
        stores, torch.from_numpy(w).cuda(), torch.from_numpy(pos).cuda(), t.cuda(),
        torch.from_numpy(lens).cuda(), budget, sinks=sinks, recent=recent)
    assert np.array_equal(got_n.cpu().numpy(), want_n)
    assert np.array_equal(got_p.cpu().numpy(), want_p)
    assert np.array_equal(got_w.cpu().numpy(), want_w, equal_nan=True)
    for a, b in zip(stores, expect):
        assert same_bits(a, b)


@pytest.mark.parametrize("given", [False, True])
def test_evict_without_columns(given):
    """Rows that have no slots yet: nothing is read, nothing moves."""
    st = torch.arange(24, dtype=torch.uint8, device="cuda").view(3, 2, 4, 1)
    w = torch.empty(5, 2, 0, device="cuda")
    pos = torch.empty(5, 2, 0, dtype=torch.int32, device="cuda") if given else None
    lens = torch.zeros(5, dtype=torch.int32, device="cuda")
    table = torch.empty(5, 0, dtype=torch.int32, device="cuda")
    gw, gp, gn = dgs.ops.evict_rows([st], w, pos, table, lens, 3)
    assert gw.shape == gp.shape == (5, 2, 0) and gn.tolist() == [0] * 5
    assert st.flatten().tolist() == list(range(24))


@pytest.mark.parametrize("cols, budget", [(50, 20), (300, 290), (2000, 300)])
def test_evict_without_stores(cols, budget):
    """The C entry without a store: weights and positions alone."""
    from dgs._lib import c_i64, c_vp, check, lib, stream_ptr
    gen = torch.Generator().manual_seed(cols)
    rows, heads = 4, 2
    w = torch.rand(rows, heads, cols, generator=gen)
    pos = torch.arange(cols, dtype=torch.int32).repeat(rows, heads, 1)
    lens = torch.tensor([0, budget, budget + 1, cols])
    want_w, want_p, want_n, _ = ref.evict(w.numpy(), pos.numpy(), lens.numpy(), budget, 1, 2)
    dw, dl = w.cuda(), lens.cuda()
    ow, op, on = torch.empty_like(dw), torch.empty_like(dw, dtype=torch.int32), torch.empty_like(dl)
    table = torch.arange(rows * cols).view(rows, cols).cuda()
    need = c_i64()
    check(lib.dgs_evict_workspace(rows, heads, cols, budget, need))
    ws = torch.empty(max(need.value, 1), dtype=torch.uint8, device="cuda")
    check(lib.dgs_evict_rows(
        (c_vp * 1)(), (c_i64 * 1)(), 0, rows * cols, heads, 1, dw.data_ptr(), None, ow.data_ptr(),
        op.data_ptr(), rows, cols, table.data_ptr(), 8, cols, dl.data_ptr(), 8, on.data_ptr(),
        budget, 1, 2, ws.data_ptr() if need.value else None, need.value, stream_ptr(0)))
    assert np.array_equal(on.cpu().numpy(), want_n)
    assert np.array_equal(op.cpu().numpy(), want_p) and np.array_equal(ow.cpu().numpy(), want_w)


@pytest.mark.parametrize("dim, group, dtype, width", [
    (128, 64, "f32", 2), (80, 40, "f16", 2), (32, 32, "f32", 1), (128, 64, "f32", 80),
    (64, 64, "bf16", 80), (40, 8, "bf16", 80)])
def test_nan_and_infinity_stay_in_their_rows_in_every_form(dim, group, dtype, width):
    """As test_attend_nan_and_infinity_stay_in_their_rows; a row's parts are cut by lengths alone."""
    pages = 4 * width
    cache = full_cache(pages, 16, 2, dim, group)
    q = states((4, 8, dim), torch.Generator().manual_seed(1), TYPES[dtype])
    table = torch.arange(pages).view(4, width).cuda()
    full = 16 * width
    lens = torch.tensor([full, full - 5, full, full - 3]).cuda()
    w = torch.zeros(4, 2, full, device="cuda")
    clean = cache.attend(q, table, lens, weights=w)
    cache.k_scales[2 * width - 1, 0, 3] = math.nan  # row 1, slot full - 13, head 0
    cache.v_scales[2 * width - 1, 1, 12] = math.nan  # behind row 1's length
    q2 = q.clone()
    q2[2, 5] = math.inf
    q2[3, 0, 7] = math.nan
    w2 = torch.zeros_like(w)
    got = cache.attend(q2, table, lens, weights=w2)
    bad = torch.zeros(4, 8, dtype=torch.bool)
    bad[1, :4] = bad[2, 5] = bad[3, 0] = True
    assert torch.equal(got.isnan().all(-1).cpu(), bad) and torch.equal(got.isnan().any(-1).cpu(), bad)
    assert torch.equal(got[~bad], clean[~bad])
    heads = bad.view(4, 2, 4).any(-1)
    inside = (torch.arange(full) < lens.cpu()[:, None])[:, None].expand(4, 2, full)
    assert torch.equal(w2.isnan().cpu(), heads[..., None] & inside)
    assert torch.equal(w2.cpu()[~heads], w.cpu()[~heads])


@pytest.mark.parametrize("dim, group, dtype", [(128, 64, "f32"), (80, 40, "bf16"), (64, 64, "f16")])
def test_attend_offsets_past_32_bits(dim, group, dtype):
    """Rows whose bytes lie past 2^31 and 2^32, in both forms."""
    page, heads = 64, 4
    pages = 2 ** 32 // (heads * page * dim // 2) + 4000
    bufs = []
    for _ in range(2):
        bufs += [torch.empty(pages, heads, page, dim // 2, dtype=torch.uint8, device="cuda"),
                 torch.empty(pages, heads, page, dim // group, 2, dtype=torch.bfloat16, device="cuda")]
    assert bufs[0].numel() > 2 ** 32
    cache = dgs.classes.StateCache.wrap(*bufs)
    small = full_cache(12, page, heads, dim, group, seed=6)
    gen = torch.Generator().manual_seed(2)
    use = torch.cat([torch.randperm(pages - 1, generator=gen)[:11], torch.tensor([pages - 1])]).cuda()
    for b, s in zip(bufs, buffers(small)):
        b[use] = s
    table = torch.arange(12).view(2, 6).cuda()
    q = states((2, 8, dim), gen, TYPES[dtype])
    for n in (384, 301):
        lens = torch.tensor([n, 130]).cuda()
        w, w2 = torch.zeros(2, heads, 384, device="cuda"), torch.zeros(2, heads, 384, device="cuda")
        want = check_attend(small, q, table, lens, weights=w)
        got = cache.attend(q, use[table], lens, weights=w2)
        assert torch.equal(got, want) and torch.equal(w, w2)


@pytest.mark.parametrize("dim, group, dtype, cap", [
    (128, 64, "bf16", 4096), (128, 64, "f32", 4096), (80, 40, "f16", 1024), (64, 64, "bf16", 640)])
def test_graphs_of_cut_rows_follow_the_lengths(dim, group, dtype, cap):
    """Two graphs of attend with weights, and an eviction with moves of its own kernel, replayed
    between eager calls while queries and lengths change in place."""
    gen = torch.Generator().manual_seed(cap)
    rows, page, budget = 5, 16, cap // 3
    cache = full_cache(rows * cap // page, page, 2, dim, group, seed=8)
    bufs0 = [b.clone() for b in buffers(cache)]
    table = torch.randperm(rows * cap // page, generator=gen).view(rows, cap // page).int().cuda()
    lens = torch.full((rows,), cap, dtype=torch.int32, device="cuda")
    q = states((rows, 6, dim), gen, TYPES[dtype])
    w0 = torch.rand(rows, 2, cap, generator=gen).cuda()
    wa, wb = w0.clone(), w0.clone()

    def one():
        return (cache.attend(q, table, lens, weights=wa),)

    def two():
        wb.copy_(w0)
        out = cache.attend(q, table, lens, weights=wb, decay=0.5)
        return (out,) + tuple(cache.evict(wb, None, table, lens, budget, sinks=2, recent=20))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(), two()
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        r1 = one()
    with torch.cuda.graph(g2):
        r2 = two()
    for turn in range(4):
        q.copy_(states(q.shape, gen, q.dtype))
        lens.copy_(torch.randint(0, cap + 1, (rows,), generator=gen) if turn else torch.zeros(rows))
        want = []
        for i, f in enumerate((one, two)):
            for a, b in zip(buffers(cache), bufs0):
                a.copy_(b)
            wa.copy_(w0)
            want.append([t.clone() for t in f()] + [wa.clone()] + [b.clone() for b in buffers(cache)])
        torch.cuda.synchronize()
        for f, r, g in ((one, r1, g1), (two, r2, g2)):
            for a, b in zip(buffers(cache), bufs0):
                a.copy_(b)
            wa.copy_(w0)
            g.replay()
            got = list(r) + [wa] + buffers(cache)
            assert all(same_bits(x, y) for x, y in zip(got, want[f is two])), (turn, f)
