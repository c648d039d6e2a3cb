"""The state cache's calls at the edges of what it documents, against plain forms.

Tolerances of attend: those of test_state_gpu.py (prob_error), whose derivation counts the sums over
the slots that are there."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import dgs
import state_ref as ref
from test_state_gpu import TYPES, U, full_cache, prob_error, raises_next, same_bits, states

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------ eviction
@pytest.mark.parametrize("cols, budget", [(32768, 32768), (32769, 32769), (32769, 2 ** 40),
                                          (40000, 40000), (65536, 65537)])
@pytest.mark.parametrize("given", [False, True])
def test_evict_with_room_for_every_column(cols, budget, given):
    """A cache that holds all its columns, evicted after every token: copies, and nothing moves."""
    gen = torch.Generator().manual_seed(cols)
    heads, page = 2, 2 - cols % 2
    w = torch.rand(3, heads, cols, generator=gen)
    pos = torch.randint(0, 2 ** 31 - 1, (3, heads, cols), generator=gen).int() if given else None
    lens = torch.tensor([cols, 0, cols - 7])
    store = torch.randn(cols // page, heads, page, 2, generator=gen).cuda()
    before = store.clone()
    table = torch.arange(cols // page).repeat(3, 1)
    want_w, want_p, want_n, moves = ref.evict(w.numpy(), None if pos is None else pos.numpy(),
                                              lens.numpy(), budget, 3, 9)
    assert not moves
    for _ in range(2):
        got_w, got_p, got_n = dgs.ops.evict_rows(
            [store], w.cuda(), None if pos is None else pos.cuda(), table.cuda(), lens.cuda(), budget,
            sinks=3, recent=9)
        torch.cuda.synchronize()
        assert np.array_equal(got_w.cpu().numpy(), want_w)
        assert np.array_equal(got_p.cpu().numpy(), want_p)
        assert np.array_equal(got_n.cpu().numpy(), want_n)
        assert same_bits(store, before)


@pytest.mark.parametrize("cols, budget", [
    (50, 20), (64, 63), (200, 100), (256, 255), (300, 100), (1000, 999), (1000, 400), (4000, 3999),
    (5003, 1000), (8000, 7900), (12000, 6000), (20001, 20000), (30000, 200), (40000, 39999),
    (40000, 9000)])
@pytest.mark.parametrize("kind", ["few", "same", "zeros", "negative", "half"])
def test_evict_repeated_positions(cols, budget, kind):
    """Positions that repeat (timestamps, zeros behind a prompt, -1 at an appended slot) protect more
    slots than stay: of the protected ones the heaviest do."""
    rng = np.random.default_rng(cols + budget)
    lens = np.array([cols, budget + 1, cols - cols // 7])
    rows, heads, sinks, recent = 3, 2, 0, min(budget, 3)
    w = rng.integers(0, 400, (rows, heads, cols)).astype(np.float32) * 0.25 - 20  # ties too
    w[rng.random(w.shape) < 0.05] = np.nan
    w[rng.random(w.shape) < 0.02] = np.inf
    w[rng.random(w.shape) < 0.02] = -np.inf
    pos = {"few": rng.integers(0, 4, w.shape), "same": np.full(w.shape, 7),
           "zeros": np.zeros(w.shape), "negative": np.full(w.shape, -1),
           "half": np.where(rng.random(w.shape) < 0.5, rng.permutation(cols), 10 ** 9)}[kind]
    pos = pos.astype(np.int32)
    if kind in ("zeros", "negative"):
        sinks, recent = 1, 0
    store = torch.from_numpy(rng.integers(0, 2 ** 31, (rows * cols, heads, 1, 1), dtype=np.int32)).cuda()
    table = rng.permutation(rows * cols).reshape(rows, cols)
    want_w, want_p, want_n, moves = ref.evict(w, pos, lens, budget, sinks, recent)
    expect, t = store.cpu().clone(), torch.from_numpy(table)
    if moves:
        i, h, s, d = (torch.tensor(x) for x in zip(*moves))
        expect[t[i, d], h] = expect[t[i, s], h].clone()
    got_w, got_p, got_n = dgs.ops.evict_rows(
        [store], torch.from_numpy(w).cuda(), torch.from_numpy(pos).cuda(), t.cuda(),
        torch.from_numpy(lens).cuda(), budget, sinks=sinks, recent=recent)
    assert np.array_equal(got_n.cpu().numpy(), want_n)
    assert np.array_equal(got_p.cpu().numpy(), want_p)
    assert np.array_equal(got_w.cpu().numpy(), want_w, equal_nan=True)
    assert same_bits(store, expect)


def test_first_call_of_a_process_inside_a_capture():
    worker = os.path.join(os.path.dirname(os.path.abspath(__file__)), "evict_capture_worker.py")
    p = subprocess.run([sys.executable, worker], capture_output=True, text=True, timeout=100)
    assert p.returncode == 0 and "capture worker ok" in p.stdout, p.stderr[-2000:]


# ------------------------------------------------------------------------------ attention
def plain_left_out(q, cache, table, lens):
    """As ref.attend, with the slots on pages outside the cache left out (none left: zeros)."""
    kc, ks, vc, vs = [t.cpu() for t in (cache.k_codes, cache.k_scales, cache.v_codes,
                                        cache.v_scales)]
    q, table, lens = q.cpu().double(), table.cpu().long(), lens.cpu().long()
    rows, nq, dim = q.shape
    pages, heads, page = kc.shape[:3]
    group, g, scale = dim // ks.shape[3], nq // heads, dim ** -0.5
    out = torch.zeros(rows, nq, dim, dtype=torch.float64)
    prob = torch.zeros(rows, heads, table.shape[1] * page, dtype=torch.float64)
    size, steps, vmax = (torch.zeros(rows, nq, dtype=torch.float64) for _ in range(3))
    for i in range(rows):
        j = torch.arange(int(lens[i]))
        j = j[(table[i, j // page] >= 0) & (table[i, j // page] < pages)]
        if j.numel() == 0:
            continue
        p, o = table[i, j // page], j % page
        for h in range(heads):
            k, v = ref.values(kc[p, h, o], ks[p, h, o]), ref.values(vc[p, h, o], vs[p, h, o])
            mine = slice(h * g, (h + 1) * g)
            e = torch.softmax(q[i, mine] @ k.T * scale, 1)
            out[i, mine], prob[i, h, j] = e @ v, e.sum(0)
            s = ks[p, h, o, :, 0].double().repeat_interleave(group, 1)
            size[i, mine] = (q[i, mine].abs() @ k.abs().T).amax(1) * scale
            steps[i, mine] = (q[i, mine].abs() @ s.T).amax(1) * scale
            vmax[i, mine] = v.abs().max()
    return out, prob, size, steps, vmax


@pytest.mark.parametrize("page", [1, 8, 16])
@pytest.mark.parametrize("cap", [16, 64, 2048])
@pytest.mark.parametrize("dim, group, heads, g, dtype", [
    (128, 64, 2, 4, "bf16"), (64, 64, 1, 1, "f32"), (80, 40, 2, 3, "f16"), (32, 32, 2, 20, "bf16"),
    (128, 32, 1, 5, "f32"), (96, 96, 2, 2, "bf16")])
def test_slots_outside_are_left_out(page, cap, dim, group, heads, g, dtype):
    """Rows with none, one, some and all of their pages outside the cache: a row without a slot gives
    zeros, and its weights receive nothing but their decay."""
    gen = torch.Generator().manual_seed(cap + dim)
    pages, width = 4096 // page, cap // page
    cache = full_cache(pages, page, heads, dim, group, seed=7)
    table = torch.randint(0, pages, (9, width), generator=gen)
    lens = torch.tensor([cap, cap, cap, cap - 3, 0, cap, 1, cap // 2, cap])
    bad = torch.randint(1, 2 ** 31, (9, width), generator=gen) * -1
    bad[:, 1::2] = pages
    table[1] = bad[1]
    table[2, ::2] = bad[2, ::2]
    table[3] = bad[3]
    table[4] = bad[4]
    table[5, -1] = bad[5, -1]
    table[6] = bad[6]
    table[7, :-(-cap // 2 // page)] = bad[7, :-(-cap // 2 // page)]  # only what lies in the length
    table[8, 0] = bad[8, 0]
    q = states((9, heads * g, dim), gen, TYPES[dtype])
    want, prob, size, steps, vmax = plain_left_out(q, cache, table, lens)
    rel = prob_error(dim, size, steps, dtype == "f32")
    off = (2 * rel * vmax)[..., None]
    tol = off + torch.finfo(q.dtype).eps / 2 * (want.abs() + off)
    tol = tol + 2.0 ** -25 if dtype == "f16" else tol
    w0 = torch.rand(9, heads, cap, generator=gen)
    inside = (torch.arange(cap) < lens[:, None])[:, None]
    for ids in (torch.int32, torch.int64):
        for decay in (0.5, 0.0):
            w = w0.cuda()
            got = cache.attend(q, table.to(ids).cuda(), lens.cuda(), weights=w, decay=decay)
            raises_next("page or slot")
            err = (got.cpu().double() - want).abs()
            assert bool((err <= tol).all()), (float(err.max()), float(tol.max()))
            for none in (1, 3, 4, 6, 7):
                assert bool((got[none] == 0).all())
            exp = torch.where(inside, prob + decay * w0.double(), w0.double())
            wrel = 2 * rel.unflatten(1, (heads, g)).amax(2)[..., None]
            werr = (w.cpu().double() - exp).abs()
            assert bool((werr <= wrel * prob + (g + 4) * U * exp.abs()).all()), float(werr.max())
        plain = cache.attend(q, table.to(ids).cuda(), lens.cuda())
        raises_next("page or slot")
        assert bool(((plain.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("cap", [16, 256, 2048])
@pytest.mark.parametrize("g", [1, 4])
def test_infinite_logits_are_no_empty_row(cap, g):
    """Logits that are all -infinity have no softmax: NaN, not the zeros of a row without slots."""
    dim = 64
    codes = torch.full((cap, 1, 1, dim // 2), 0x11, dtype=torch.uint8, device="cuda")  # code 1
    scales = torch.tensor([1.0, 0.0]).to(torch.bfloat16).cuda().expand(cap, 1, 1, 1, 2).contiguous()
    cache = dgs.classes.StateCache.wrap(codes, scales, codes.clone(), scales.clone())  # all rows are 1
    q = torch.ones(3, g, dim, device="cuda")
    q[1, 0, 7] = -math.inf
    table = torch.arange(cap).repeat(3, 1).cuda()
    w = torch.zeros(3, 1, cap, device="cuda")
    got = cache.attend(q, table, torch.tensor([cap, cap, 0]).cuda(), weights=w)
    assert bool(got[1, 0].isnan().all()) and bool(w[1].isnan().all())
    assert torch.equal(got[2], torch.zeros(g, dim, device="cuda")) and not w[2].any()
    ones = torch.cat([got[0], got[1, 1:]])
    assert bool(((ones - 1).abs() <= (cap + 8) * U).all())  # a mean of ones


@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("cap", [16, 256, 2048, 40000])
@pytest.mark.parametrize("g", [1, 3])
def test_infinite_logits_beside_finite_ones(page, cap, g):
    """Slots whose logits overflow to -infinity, slots on pages outside and slots of logit 0, in runs that
    different parts of a row take: the last share the row evenly."""
    dim, pages = 64, 64
    half = pages // 2  # pages of keys of 1, then of 0
    codes = torch.full((pages, 1, page, dim // 2), 0x11, dtype=torch.uint8)
    codes[half:] = 0
    scales = torch.tensor([1.0, 0.0]).to(torch.bfloat16).expand(pages, 1, page, 1, 2).contiguous()
    cache = dgs.classes.StateCache.wrap(codes.cuda(), scales.cuda(), codes.flip(0).contiguous().cuda(),
                                        scales.clone().cuda())  # values of 0, then of 1
    width = cap // page
    table = torch.zeros(4, width, dtype=torch.int64)
    table[0] = torch.where(torch.arange(width) >= width - max(1, width // 4), half, 0)  # finite at the end
    table[1, 0], table[1, 1:], table[1, width // 2:] = half + 1, 3, pages  # and at the front, bad ones behind
    table[2] = torch.where(torch.arange(width) < width - 1, pages, 1)  # only -infinity is left
    table[3] = pages
    q = torch.full((4, g, dim), -3e38, device="cuda")
    w = torch.zeros(4, 1, cap, device="cuda")
    lens = torch.full((4,), cap).cuda()
    if width == 1:
        table[1, 0] = half + 1
    got = cache.attend(q, table.cuda(), lens, scale=1.0, weights=w)
    raises_next("page or slot")
    share = (table[:2] >= half) & (table[:2] < pages)
    prob = share.repeat_interleave(page, 1).double()
    prob = g * prob / prob.sum(1, keepdim=True)
    # sums of cap equal terms and of their parts
    assert bool(((w[:2, 0].cpu().double() - prob).abs() <= 8 * (cap + 8) * U * prob).all())
    assert bool(((got[:2].cpu().double() - 1).abs() <= 8 * (cap + 8) * U).all())
    assert bool(got[2].isnan().all()) and bool(w[2].isnan().all())
    assert not got[3].any() and not w[3].any()


@pytest.mark.parametrize("dim, group", [(64, 64), (40, 40), (96, 32), (128, 32), (24, 8), (256, 128)])
@pytest.mark.parametrize("g", [1, 2, 3, 4, 6])
@pytest.mark.parametrize("rows, cap", [(70, 15), (30, 200), (5, 600), (3, 3000), (600, 1000)])
def test_values_of_zero_sum_to_zero(dim, group, g, rows, cap):
    """32-bit outputs are sums of p * v with v = scale * code + base taken first: where every slot's v is
    exactly 0 (here scale * 5 - 5 * scale), so is the sum, however large scale and base are.  The
    scales are k / 8, k up to 25: 5 k has 7 bits, so bases are exact too."""
    gen = torch.Generator().manual_seed(cap + g)
    heads, pages = 2, max(cap, 64)
    ng = dim // group
    codes = torch.randint(0, 16, (pages, heads, 1, dim), generator=gen).to(torch.uint8)
    codes[..., ::3] = 5
    s = torch.randint(1, 26, (pages, heads, 1, ng), generator=gen) / 8
    vs = torch.stack([s, -5 * s], -1).to(torch.bfloat16)
    kc, ks = ref.quantise(torch.randn(pages, heads, 1, dim, generator=gen), group)
    cache = dgs.classes.StateCache.wrap(ref.pack(kc).cuda(), ks.cuda(), ref.pack(codes).cuda(),
                                        vs.cuda())
    q = torch.randn(rows, heads * g, dim, generator=gen).cuda()
    table = torch.randint(0, pages, (rows, cap), generator=gen).cuda()
    lens = torch.randint(1, cap + 1, (rows,), generator=gen).cuda()
    got = cache.attend(q, table, lens)
    assert bool((got[..., ::3] == 0).all()), float(got[..., ::3].abs().max())
    rest = torch.ones(dim, dtype=torch.bool)
    rest[::3] = False
    assert bool((got[..., rest.cuda()] != 0).any())


@pytest.mark.parametrize("page, cap", [(1, 48), (16, 48), (1, 2000), (16, 2000)])
def test_large_queries_that_cancel(page, cap):
    """The matrix form multiplies q by codes that stand 16 too high and takes the offset out again.  Two
    channels of +-2^18 with equal codes lie in different products; q (16 + c) and its sums are whole
    numbers below 2^24, the scale is a power of two and the base 0: every logit is exact, and the weights
    are off by the softmax alone.  (An offset of 128 would make the logits off by 1 / 32.)"""
    gen = torch.Generator().manual_seed(cap)
    dim, slots = 64, 4096
    codes = torch.randint(0, 16, (slots // page, 1, page, dim), generator=gen).to(torch.uint8)
    codes[..., 63] = codes[..., 0]
    ks = torch.tensor([1 / 64, 0.0]).to(torch.bfloat16).expand(slots // page, 1, page, 1, 2)
    vc, vs = ref.quantise(torch.randn(slots // page, 1, page, dim, generator=gen), 64)
    cache = dgs.classes.StateCache.wrap(ref.pack(codes).cuda(), ks.contiguous().cuda(),
                                        ref.pack(vc).cuda(), vs.cuda())
    q = torch.randint(-3, 4, (5, 4, dim), generator=gen).float()
    q[..., 0], q[..., 63] = 2.0 ** 18, -2.0 ** 18
    q = q.bfloat16().cuda()
    table = torch.randint(0, slots // page, (5, cap // page), generator=gen).cuda()
    lens = torch.tensor([cap, cap - 1, 33, 1, cap // 2]).cuda()
    w = torch.zeros(5, 1, cap, device="cuda")
    cache.attend(q, table, lens, scale=1.0, weights=w, decay=0.0)
    _, prob, _, _, _ = ref.attend(q, cache, table, lens, 1.0)
    largest = 62 * 3 * 15 / 64
    rel = 2 * (2.0 ** -23 + 3 * U * (largest + 1) + 64 * U)
    err = (w.cpu().double() - prob).abs()
    assert bool((err <= rel * prob + 8 * U * prob).all()), float((err / prob.clamp(min=1e-30)).max())


@pytest.mark.parametrize("dtype, top", [("f32", 3e38), ("bf16", 3e38), ("f16", 65504.0)])
@pytest.mark.parametrize("page, cap", [(1, 16), (16, 64), (16, 2048)])
def test_queries_near_the_types_largest_value(dtype, top, page, cap):
    """A query of +-top in two channels whose keys are alike cancels; the scale makes a small factor of
    what a third adds: logits of top * scale * code, which is 1 / 4 * code."""
    gen = torch.Generator().manual_seed(cap)
    dim, pages = 64, 4096 // page
    codes = torch.zeros(pages, 1, page, dim, dtype=torch.uint8)
    codes[..., 5] = torch.randint(0, 16, (pages, 1, page), generator=gen).to(torch.uint8)
    ks = torch.tensor([1.0, 0.0]).to(torch.bfloat16).expand(pages, 1, page, 1, 2).contiguous()
    vc, vs = ref.quantise(torch.randn(pages, 1, page, dim, generator=gen), 64)
    cache = dgs.classes.StateCache.wrap(ref.pack(codes).cuda(), ks.cuda(), ref.pack(vc).cuda(), vs.cuda())
    big = torch.tensor(top).to(TYPES[dtype])
    q = torch.zeros(2, 2, dim, dtype=TYPES[dtype])
    q[..., 5], q[:, 1, 9] = big / 16, -big / 16  # sums of codes up to 15 stay in range
    if dtype != "bf16":
        q[0, 0, 5] = big if dtype == "f16" else big / 16
    table = torch.randint(0, pages, (2, cap // page), generator=gen)
    lens = torch.tensor([cap, cap // 2 + 1])
    scale = 4 / float(big)  # logits of up to 15 * 4 (f16: 64)
    w = torch.zeros(2, 1, cap, device="cuda")
    out, prob, size, steps, vmax = ref.attend(q, cache, table, lens, scale)
    got = cache.attend(q.cuda(), table.cuda(), lens.cuda(), scale=scale, weights=w)
    rel = prob_error(dim, size, steps, dtype == "f32")
    off = (2 * rel * vmax)[..., None]
    tol = off + torch.finfo(q.dtype).eps / 2 * (out.abs() + off) + (2.0 ** -25 if dtype == "f16" else 0)
    assert bool(((got.cpu().double() - out).abs() <= tol).all())
    assert bool(((w.cpu().double() - prob).abs() <= 2 * rel.amax(1)[:, None, None] * prob + 8 * U).all())


def test_streams_keep_their_own_weights():
    gen = torch.Generator().manual_seed(0)
    cache = full_cache(256, 16, 2, 128, 64)
    table = torch.randperm(256, generator=gen).view(2, 128).cuda()
    lens = torch.tensor([2048, 1999]).cuda()
    for dtype in TYPES.values():
        qs = [states((2, 8, 128), gen, dtype) for _ in range(4)]
        want = [torch.zeros(2, 2, 2048, device="cuda") for _ in range(4)]
        for q, w in zip(qs, want):
            for _ in range(5):
                cache.attend(q, table, lens, weights=w, decay=0.5)
        torch.cuda.synchronize()
        got = [torch.zeros(2, 2, 2048, device="cuda") for _ in range(4)]
        streams = [torch.cuda.Stream() for _ in range(4)]
        torch.cuda.synchronize()
        for _ in range(5):
            for q, w, s in zip(qs, got, streams):
                with torch.cuda.stream(s):
                    cache.attend(q, table, lens, weights=w, decay=0.5)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_the_last_gather_is_no_state_call():
    """A loader tells its batches by the tag of this thread's last gather."""
    cache = full_cache(8, 16, 2, 64, 64)
    dgs.ops._CAPI_cuda_index_select(torch.arange(8.0).cuda().view(8, 1), torch.tensor([3]).cuda())
    tag = dgs.ops._last_gather_tag()
    assert tag > 0
    slots = torch.arange(4).cuda()
    k, v = cache.read(slots)
    cache.write(k, v, slots)
    table = torch.arange(8).view(1, 8).cuda()
    cache.append(k[:1], v[:1], table, slots[:1])
    w = torch.zeros(1, 2, 128, device="cuda")
    cache.attend(k[:1], table, slots[1:2], weights=w)
    cache.evict(w, None, table, slots[3:], 2)
    assert dgs.ops._last_gather_tag() == tag
    dgs.ops._CAPI_cuda_index_select(torch.arange(8.0).cuda().view(8, 1), torch.tensor([3]).cuda())
    assert dgs.ops._last_gather_tag() > tag
