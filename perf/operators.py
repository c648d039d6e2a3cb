"""The cached-state operators, as cases to measure: attention over a cache held in 4 bits, writing
rows into that cache, reading them back, and eviction of rows by accumulated attention weight.

Layout of the cache (pages of `page` slots; a slot holds one row of every head):
  codes   uint8    [pages, heads, page, D / 2]        two channels a byte, the even one low
  scales  bfloat16 [pages, heads, page, D / group, 2] scale s and base b of each group
and a channel's value is s * code + b.
"""
import math
import os
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_CHUNK = 1 << 27  # elements of a 32-bit temporary


def _dgs():
    path = os.path.join(_ROOT, "dist-gnn_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    import dgs
    return dgs


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token of one conversation: latency counts
        dict(name="attend_token", op="attend", rows=1, q_heads=32, heads=8, dim=128, group=64,
             page=16, low=700, high=700, dtype="bf16", weights=False),
        # a serving batch of very different lengths that also keeps the attention weights
        dict(name="attend_batch", op="attend", rows=64, q_heads=32, heads=8, dim=128, group=64,
             page=16, low=1, high=8192, dtype="bf16", weights=True),
        # few long contexts: the work is split over the cache's length
        dict(name="attend_long", op="attend", rows=8, q_heads=32, heads=8, dim=128, group=64,
             page=64, low=100001, high=131072, dtype="bf16", weights=False),
        # the second hop of the sampling benchmark: every frontier node attends to its at most
        # 15 sampled neighbours, whose rows are addressed by node id (pages of one slot)
        dict(name="attend_neighbours", op="attend", rows=40960, q_heads=4, heads=4, dim=32,
             group=32, page=1, low=0, high=15, dtype="f32", weights=True, nodes=2449029),
        # one head per query head, small odd heads, empty rows, pages that end inside a tile
        dict(name="attend_odd", op="attend", rows=37, q_heads=12, heads=12, dim=80, group=40,
             page=8, low=0, high=1531, dtype="f16", weights=True),
        # the rows of one decoding step, appended to their sequences
        dict(name="write_token", op="write", rows=64, q_heads=32, heads=8, dim=128, group=64,
             page=16, high=8192, dtype="bf16", append=True),
        # the states of a long prompt, cut out of the fused projection
        dict(name="write_prompt", op="write", rows=65536, q_heads=32, heads=8, dim=128, group=64,
             page=16, high=0, dtype="bf16", append=False),
        # the feature rows of a sampled batch, by node id
        dict(name="read_nodes", op="read", rows=400000, heads=1, dim=128, group=64, page=1,
             nodes=2449029, dtype="f32"),
        # one conversation's prefix, read back for a dense attention over the next prompt
        dict(name="read_prefix", op="read", rows=4099, heads=8, dim=128, group=128, page=32,
             nodes=8192, dtype="bf16"),
        # a decoding step of sequences that are full: one row of each head goes
        dict(name="evict_step", op="evict", rows=64, heads=8, dim=128, page=16, budget=4096,
             low=4000, high=4097, sinks=4, recent=256, dtype="bf16"),
        # after a prompt: most of it goes
        dict(name="evict_prompt", op="evict", rows=16, heads=8, dim=128, page=64, budget=4096,
             low=20000, high=32768, sinks=4, recent=1024, dtype="bf16"),
        # a small memory of one graph node batch, odd sizes
        dict(name="evict_small", op="evict", rows=33, heads=2, dim=40, page=1, budget=50,
             low=0, high=77, sinks=0, recent=10, dtype="f32"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "write", "read", "evict", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim, group = rng.choice([(128, 64), (128, 64), (128, 32), (128, 128), (64, 32), (64, 64),
                             (96, 32), (80, 40), (32, 32), (256, 64), (16, 8), (40, 40)])
    heads = rng.choice([1, 2, 3, 4, 5, 8, 8])
    page = 1 << rng.randrange(0, 8)
    if op == "attend":
        q_heads = heads * rng.choice([1, 1, 2, 3, 4, 4, 7, 8, 16])
        rows = _log_int(rng, 1, min(20000, 30000000 // (q_heads * dim)))
        room = min(131072, 120000000 // (rows * heads * dim))  # slots a row
        high = _log_int(rng, 1, max(2, room))
        return dict(op=op, rows=rows, q_heads=q_heads, heads=heads, dim=dim, group=group,
                    page=page, low=rng.randrange(0, high + 1), high=high, dtype=dtype,
                    weights=rng.random() < 0.6)
    if op == "write":
        append = rng.random() < 0.5
        return dict(op=op, rows=_log_int(rng, 1, 300 if append else 60000 * 128 // (dim * heads)),
                    q_heads=heads * rng.choice([1, 4]), heads=heads, dim=dim, group=group,
                    page=page, high=_log_int(rng, 1, 4000) if append else 0, dtype=dtype,
                    append=append)
    if op == "read":
        nodes = _log_int(rng, 1000, 200000)
        return dict(op=op, rows=_log_int(rng, 1, 400000 * 128 // (dim * heads)), heads=heads,
                    dim=dim, group=group, page=page, nodes=nodes, dtype=dtype)
    rows = _log_int(rng, 1, 64)
    row = heads * dim * _TYPES[dtype].itemsize
    high = _log_int(rng, 2, min(32768, max(2, 1000000000 // (rows * row))))
    budget = rng.randrange(1, high + 1)
    recent = rng.randrange(0, budget + 1)
    return dict(op=op, rows=rows, heads=heads, dim=dim, page=page, budget=budget,
                low=rng.randrange(0, high + 1), high=high,
                sinks=rng.randrange(0, min(4, budget - recent) + 1), recent=recent, dtype=dtype)


def _lengths(case):
    """The rows' lengths: spread from `low` to `high`, more of them short; the longest is `high`."""
    n, low, high = case["rows"], case["low"], case["high"]
    if n == 1:
        return [high]
    return [low + int(round((high - low) * (i / (n - 1)) ** 2)) for i in range(n)]


def work(case):
    op, heads, dim = case["op"], case["heads"], case["dim"]
    size = _TYPES[case["dtype"]].itemsize
    if op == "evict":
        lens = _lengths(case)
        budget = case["budget"]
        total = sum(lens) * heads
        row = 2 * dim * size
        moved = sum(min(budget, n) * max(n - budget, 0) // max(n, 1) for n in lens) * heads
        return {"bytes": 16 * total + 2 * moved * row, "flops": 2 * total}
    held = heads * (dim + 8 * (dim // case["group"]))  # a slot's K and V in the cache
    if op == "attend":
        slots = sum(_lengths(case))
        q = case["rows"] * case["q_heads"] * dim
        return {"bytes": slots * held + 2 * q * size + slots * heads * 4 * bool(case["weights"]),
                "flops": 4 * slots * case["q_heads"] * dim}
    values = 2 * case["rows"] * heads * dim
    if op == "write":  # the rows in, their codes out, and those codes as values
        return {"bytes": values * (size + 4) + 2 * case["rows"] * held, "flops": 6 * values}
    return {"bytes": values * size + case["rows"] * held, "flops": 2 * values}


# ------------------------------------------------------------------------------------ inputs
def _quantise(x, group):
    """[..., D] -> codes [..., D] (uint8, one a channel) and scales [..., D / group, 2]."""
    g = x.float().unflatten(-1, (-1, group))
    low, high = g.amin(-1), g.amax(-1)
    s = ((high - low) / 15).to(torch.bfloat16)
    b = low.to(torch.bfloat16)
    d = g.double() - b.double()[..., None]
    c = torch.where(s[..., None] == 0, torch.zeros_like(d), (d / s.double()[..., None]).round())
    return c.clamp(0, 15).to(torch.uint8).flatten(-2), torch.stack([s, b], -1)


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _states(shape, gen, device):
    """Projected states: a channel has its own offset and spread."""
    offset = torch.randn(shape[-1], generator=gen, device=device) * 0.5
    spread = torch.rand(shape[-1], generator=gen, device=device) + 0.5
    return torch.randn(shape, generator=gen, device=device) * spread + offset


def _fill_cache(pages, case, gen, device):
    heads, page, dim, group = case["heads"], case["page"], case["dim"], case["group"]
    out = {}
    for name in ("k", "v"):
        codes = torch.empty(pages, heads, page, dim // 2, dtype=torch.uint8, device=device)
        scales = torch.empty(pages, heads, page, dim // group, 2, dtype=torch.bfloat16,
                             device=device)
        step = max(1, _CHUNK // 4 // (heads * page * dim))
        for lo in range(0, pages, step):
            n = min(step, pages - lo)
            c, s = _quantise(_states((n, heads, page, dim), gen, device), group)
            codes[lo:lo + n], scales[lo:lo + n] = _pack(c), s
        out[name + "_codes"], out[name + "_scales"] = codes, scales
    return out


def _paged_table(lens, page, gen, device):
    """A table of distinct pages in a random order, -1 behind each row's last page."""
    need = [-(-n // page) for n in lens]
    width = max(1, max(need))
    total = max(1, sum(need))
    count = torch.tensor(need, device=device)
    used = torch.arange(width, device=device) < count[:, None]
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=device)
    table[used] = torch.randperm(total, generator=gen, device=device)[:sum(need)].int()
    return table, total


def prepare(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(seed * 1000003 + 17)
    op, rows, heads, dim = case["op"], case["rows"], case["heads"], case["dim"]
    dtype, page = _TYPES[case["dtype"]], case["page"]
    st = dict(case=case)
    if op == "evict":
        lens = _lengths(case)
        mixed = torch.randperm(rows, generator=gen, device=device)
        lens = torch.tensor(lens, dtype=torch.int32, device=device)[mixed]
        st["table"], pages = _paged_table(lens.tolist(), page, gen, device)
        st["lens"] = lens
        cap = st["table"].shape[1] * page
        # sums of attention weights: heavy tails, older rows more, a few that never got any and
        # a few that are equal
        w = torch.exp(torch.randn(rows, heads, cap, generator=gen, device=device) * 2)
        w = w / (1 + torch.arange(cap, device=device) / 64)
        u = torch.rand(rows, heads, cap, generator=gen, device=device)
        w = torch.where(u < 0.05, torch.zeros_like(w), w)
        st["weights"] = torch.where(u > 0.9, (w * 64).round() / 64, w)
        # earlier evictions left the rows out of order
        order = torch.rand(rows, heads, 2 * cap, generator=gen, device=device).argsort(-1)
        st["positions"] = order[..., :cap].int()
        st["stores"] = [torch.randn(pages, heads, page, dim, generator=gen,
                                    device=device).to(dtype) for _ in range(2)]
        return st
    if op == "attend":
        lens = torch.tensor(_lengths(case), dtype=torch.int32, device=device)
        lens = lens[torch.randperm(rows, generator=gen, device=device)]
        nodes = case.get("nodes")
        if nodes:  # sampled neighbours: ids of nodes, some of them under many rows
            width = max(1, case["high"])
            u = torch.rand(rows, width, generator=gen, device=device)
            st["table"], pages = (u * u * nodes).long().clamp(max=nodes - 1), nodes
        else:
            st["table"], pages = _paged_table(lens.tolist(), page, gen, device)
        st["lens"] = lens
        st["q"] = _states((rows, case["q_heads"], dim), gen, device).to(dtype)
        if case["weights"]:
            st["weights"] = torch.rand(rows, heads, st["table"].shape[1] * page, generator=gen,
                                       device=device)
    elif op == "write":
        fused = case["q_heads"] + 2 * heads  # a fused projection's rows
        st["qkv"] = _states((rows, fused, dim), gen, device).to(dtype)
        if case["append"]:
            lens = torch.randint(0, case["high"], (rows,), generator=gen, device=device)
            st["lens"] = lens.int()
            st["table"], pages = _paged_table((lens + 1).tolist(), page, gen, device)
        else:
            pages = -(-rows // page) + 3
            st["slots"] = torch.randperm(pages * page, generator=gen, device=device)[:rows]
    else:
        pages = -(-case["nodes"] // page)
        st["slots"] = torch.randint(0, pages * page, (rows,), generator=gen, device=device)
        st["dtype"] = dtype
    st["buffers"] = _fill_cache(pages, case, gen, device)
    if own:
        st["cache"] = _dgs().classes.StateCache.wrap(**st["buffers"])
    return st


# ------------------------------------------------------------------------------------ plain form
def _values(codes, scales):
    """Codes and scales of some rows -> their values, 32 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    s = scales.float()
    c = c.unflatten(-1, (s.shape[-2], -1))
    return (c * s[..., 0:1] + s[..., 1:2]).flatten(-2)


def _plain_attend(st):
    case, buf = st["case"], st["buffers"]
    heads, dim, page = case["heads"], case["dim"], case["page"]
    g = case["q_heads"] // heads
    q, table, lens = st["q"], st["table"], st["lens"]
    rows, width = table.shape
    cap = width * page
    out = torch.empty_like(q)
    weights = st.get("weights")
    step = max(1, _CHUNK // (heads * cap * dim))
    slot = torch.arange(cap, device=q.device)
    for lo in range(0, rows, step):
        hi = min(rows, lo + step)
        t = table[lo:hi].clamp(min=0).long()
        k = _values(buf["k_codes"][t], buf["k_scales"][t]).transpose(1, 2).flatten(2, 3)
        qs = q[lo:hi].float().view(hi - lo, heads, g, dim)
        logits = (k @ qs.transpose(2, 3).contiguous()) / math.sqrt(dim)  # [rows, heads, cap, g]
        inside = slot < lens[lo:hi, None]
        logits = logits.masked_fill(~inside[:, None, :, None], -math.inf)
        top = logits.amax(2, keepdim=True)
        p = torch.exp(logits - top.masked_fill(top == -math.inf, 0))
        p = p / p.sum(2, keepdim=True).clamp(min=1e-30)
        v = _values(buf["v_codes"][t], buf["v_scales"][t]).transpose(1, 2).flatten(2, 3)
        o = p.transpose(2, 3).contiguous() @ v
        out[lo:hi] = o.reshape(hi - lo, heads * g, dim).to(q.dtype)
        if weights is not None:
            weights[lo:hi] = torch.where(inside[:, None], p.sum(3), weights[lo:hi])
    return out if weights is None else (out, weights)


def _slot_of(table, lens, page):
    lens = lens.long()
    return table.gather(1, (lens // page)[:, None])[:, 0].long() * page + lens % page


def _plain_write(st):
    case, buf = st["case"], st["buffers"]
    page, heads, nq = case["page"], case["heads"], case["q_heads"]
    slots = _slot_of(st["table"], st["lens"], page) if case["append"] else st["slots"]
    at = slots // page, slots % page
    out = []
    for name, lo in (("k", nq), ("v", nq + heads)):
        codes, scales = _quantise(st["qkv"][:, lo:lo + heads], case["group"])
        buf[name + "_codes"][at[0], :, at[1]] = _pack(codes)
        buf[name + "_scales"][at[0], :, at[1]] = scales
        out.append(_values(buf[name + "_codes"][at[0], :, at[1]],
                           buf[name + "_scales"][at[0], :, at[1]]))
    return tuple(out)


def _plain_read(st):
    buf, page, slots = st["buffers"], st["case"]["page"], st["slots"]
    at = slots // page, slots % page
    return tuple(_values(buf[n + "_codes"][at[0], :, at[1]],
                         buf[n + "_scales"][at[0], :, at[1]]).to(st["dtype"]) for n in "kv")


def _plain_evict(st):
    case, table, lens = st["case"], st["table"], st["lens"]
    budget, page = case["budget"], case["page"]
    w, pos = st["weights"], st["positions"]
    rows, heads, cap = w.shape
    slot = torch.arange(cap, device=w.device)
    inside = (slot < lens[:, None])[:, None].expand(rows, heads, cap)
    seen = pos.masked_fill(~inside, -1).amax(-1, keepdim=True) + 1
    fixed = inside & ((pos < case["sinks"]) | (pos >= seen - case["recent"]))
    order = w.masked_fill(w.isnan(), -math.inf).argsort(dim=-1, descending=True,
                                                       stable=True)
    rank_of = inside.int() + fixed.int()  # 2 protected, 1 held, 0 behind the end
    again = rank_of.gather(-1, order).argsort(dim=-1, descending=True, stable=True)
    order = order.gather(-1, again)
    new_lens = lens.clamp(max=budget)
    kept = torch.zeros_like(inside).scatter(
        -1, order, (slot < new_lens[:, None])[:, None].expand(rows, heads, cap))
    holes = ~kept & inside & (slot < budget)
    movers = kept & (slot >= budget)
    # the i-th hole of a head takes the i-th mover (both in slot order)
    dst, src = holes.nonzero(), movers.nonzero()
    new_w, new_pos = w.clone(), pos.clone()
    new_w[dst[:, 0], dst[:, 1], dst[:, 2]] = w[src[:, 0], src[:, 1], src[:, 2]]
    new_pos[dst[:, 0], dst[:, 1], dst[:, 2]] = pos[src[:, 0], src[:, 1], src[:, 2]]
    behind = (slot >= new_lens[:, None])[:, None].expand(rows, heads, cap)
    new_w, new_pos = new_w.masked_fill(behind, 0), new_pos.masked_fill(behind, -1)
    d_page = table[dst[:, 0], dst[:, 2] // page].long()
    s_page = table[src[:, 0], src[:, 2] // page].long()
    for store in st["stores"]:
        store[d_page, dst[:, 1], dst[:, 2] % page] = store[s_page, src[:, 1], src[:, 2] % page]
    return (new_w, new_pos, new_lens, *st["stores"])


# ------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"attend": _plain_attend, "write": _plain_write, "read": _plain_read,
                "evict": _plain_evict}[op](state)
    if op == "evict":
        w, pos, lens = _dgs().ops.evict_rows(
            state["stores"], state["weights"], state["positions"], state["table"], state["lens"],
            case["budget"], sinks=case["sinks"], recent=case["recent"])
        return (w, pos, lens, *state["stores"])
    cache = state["cache"]
    if op == "attend":
        weights = state.get("weights")
        if weights is None:
            return cache.attend(state["q"], state["table"], state["lens"])
        # decay 0: the weights of this step alone, which the caller adds up as it likes
        out = cache.attend(state["q"], state["table"], state["lens"], weights=weights, decay=0.0)
        return out, weights
    if op == "read":
        return cache.read(state["slots"], state["dtype"])
    nq, heads = case["q_heads"], case["heads"]
    k, v = state["qkv"][:, nq:nq + heads], state["qkv"][:, nq + heads:]
    if case["append"]:
        slots = cache.append(k, v, state["table"], state["lens"])
    else:
        slots = state["slots"]
        cache.write(k, v, slots)
    return cache.read(slots, torch.float32)


# ------------------------------------------------------------------------------------ 64 bits
def _exact_rows(buf, name, page, head_dim, flat):
    """Rows of flat slots (page * size + offset) in 64 bits: [n, heads, dim]."""
    codes = buf[name + "_codes"]
    scales = buf[name + "_scales"].double()
    p, o = torch.div(flat, page, rounding_mode="floor"), flat.remainder(page)
    c = codes[p, :, o].long()
    full = torch.empty(*c.shape[:2], head_dim, dtype=torch.float64, device=c.device)
    full[..., 0::2] = (c % 16).double()
    full[..., 1::2] = (c // 16).double()
    sc = scales[p, :, o]
    width = head_dim // sc.shape[2]
    return full * sc[..., 0].repeat_interleave(width, 2) + sc[..., 1].repeat_interleave(width, 2)


def _exact_long(q, k, v, scale):
    """One row in 64 bits: q [heads, g, dim], k and v [n, heads, dim] -> out, summed weights."""
    out, w = torch.empty_like(q), []
    for h in range(q.shape[0]):
        x = (q[h] @ k[:, h].T.contiguous()) * scale
        e = torch.exp(x - x.max(1, keepdim=True).values)
        e = e / e.sum(1, keepdim=True)
        out[h] = e @ v[:, h].contiguous()
        w.append(e.sum(0))
    return out, torch.stack(w)


def _exact_short(q, k, v, row, scale):
    """Many short rows: q [rows, heads, g, dim], pair i joins q[row[i]] with k[i] and v[i]."""
    rows, heads, g, dim = q.shape
    x = (q[row] * k[:, :, None]).sum(-1) * scale
    at = row[:, None, None].expand_as(x)
    top = torch.full((rows, heads, g), -math.inf, dtype=x.dtype, device=x.device)
    top = top.scatter_reduce(0, at, x, "amax")
    e = torch.exp(x - top[row])
    e = e / torch.zeros_like(top).index_add_(0, row, e)[row]
    out = torch.zeros_like(q).index_add_(0, row, e[..., None] * v[:, :, None])
    return out, e.sum(2)


def _exact_attend(case, st):
    heads, dim, page = case["heads"], case["dim"], case["page"]
    rows, nq = st["q"].shape[:2]
    q = st["q"].double().view(rows, heads, nq // heads, dim)
    out = torch.zeros_like(q)
    weights = st["weights"].double() if case["weights"] else None
    lens = st["lens"].tolist()
    limit, lo = _CHUNK // (4 * nq * dim), 0
    while lo < rows:
        hi, total = lo, 0
        while hi < rows and (hi == lo or (total + lens[hi] <= limit and lens[hi] <= 64)):
            total += lens[hi]
            hi += 1
            if lens[hi - 1] > 64:
                break
        if total:
            ln = torch.tensor(lens[lo:hi], device=q.device)
            row = torch.repeat_interleave(torch.arange(hi - lo, device=q.device), ln)
            j = torch.arange(total, device=q.device) - (ln.cumsum(0) - ln)[row]
            flat = st["table"][row + lo, j // page].long() * page + j % page
            k = _exact_rows(st["buffers"], "k", page, dim, flat)
            v = _exact_rows(st["buffers"], "v", page, dim, flat)
            if hi == lo + 1:
                out[lo], w = _exact_long(q[lo], k, v, dim ** -0.5)
                w = w.T
            else:
                out[lo:hi], w = _exact_short(q[lo:hi], k, v, row, dim ** -0.5)
            if weights is not None:
                weights[row + lo, :, j] = w
        lo = hi
    out = out.view(rows, nq, dim)
    return out if weights is None else (out, weights)


def exact(case, seed):
    if case["op"] == "evict":
        return None  # rows are moved, nothing is computed
    global own
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    page, dim = case["page"], case["dim"]
    if case["op"] == "attend":
        return _exact_attend(case, st)
    if case["op"] == "read":
        return tuple(_exact_rows(st["buffers"], n, page, dim, st["slots"]) for n in "kv")
    out = []
    heads, group = case["heads"], case["group"]
    for lo in (case["q_heads"], case["q_heads"] + heads):
        x = st["qkv"][:, lo:lo + heads].double().reshape(case["rows"], heads, dim // group, group)
        low, high = x.min(3).values, x.max(3).values
        # scale and base are by definition 16-bit numbers
        s = (((high - low).float() / 15).to(torch.bfloat16)).double()
        b = low.float().to(torch.bfloat16).double()
        near = torch.round((x - b[..., None]) / s.clamp(min=1e-300)[..., None])
        near = torch.minimum(torch.maximum(near, torch.zeros_like(near)),
                             torch.full_like(near, 15))
        out.append((b[..., None] + s[..., None] * near).reshape(case["rows"], heads, dim))
    return tuple(out)
