"""The state cache's checks of arguments, which need no GPU: the binding refuses before it touches
the device, and the C ABI refuses before it launches."""
import ctypes

import pytest
import torch

import dgs
from dgs._lib import c_i64, lib
from dgs.state import StateCache, _CCache, evict_rows


def _fake(**kw):
    """A cache object without memory, for the binding's checks."""
    c = StateCache.__new__(StateCache)
    c.num_pages, c.page_size, c.heads, c.head_dim, c.group = 4, 8, 2, 64, 32
    c.device, c._index = torch.device("cuda", 0), 0
    for k, v in kw.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("args, msg", [
    ((0, 8, 2, 64, 32), "pages and heads"), ((4, 8, 0, 64, 32), "pages and heads"),
    ((4, 6, 2, 64, 32), "power of two"), ((4, 0, 2, 64, 32), "power of two"),
    ((4, 8, 2, 60, 60), "head_dim"), ((4, 8, 2, 264, 8), "head_dim"), ((4, 8, 2, 0, 8), "head_dim"),
    ((4, 8, 2, 64, 12), "group"), ((4, 8, 2, 64, 48), "group"), ((4, 8, 2, 64, 0), "group")])
def test_shapes_refused(args, msg):
    with pytest.raises(RuntimeError, match=msg):
        StateCache(*args)


def test_cpu_device_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        StateCache(4, 8, 2, 64, device="cpu")


def _buffers(pages=4, heads=2, page=8, dim=64, group=32):
    c = torch.zeros(pages, heads, page, dim // 2, dtype=torch.uint8)
    s = torch.zeros(pages, heads, page, dim // group, 2, dtype=torch.bfloat16)
    return dict(k_codes=c, k_scales=s, v_codes=c.clone(), v_scales=s.clone())


@pytest.mark.parametrize("change, msg", [
    (dict(k_codes=torch.zeros(4, 2, 8, dtype=torch.uint8)), "dimensions"),
    (dict(v_codes=torch.zeros(4, 2, 8, 32, dtype=torch.int8)), "v_codes"),
    (dict(v_codes=torch.zeros(5, 2, 8, 32, dtype=torch.uint8)), "v_codes"),
    (dict(v_scales=torch.zeros(4, 2, 8, 2, 2)), "v_scales"),
    (dict(k_scales=torch.zeros(4, 2, 8, 2, 3, dtype=torch.bfloat16)), "k_scales"),
    (dict(v_scales=torch.zeros(4, 2, 8, 1, 2, dtype=torch.bfloat16)), "v_scales"),
    (dict(v_codes=torch.zeros(4, 2, 8, 64, dtype=torch.uint8)[..., ::2]), "contiguous"),
    (dict(), "CUDA")])
def test_wrap_refusals(change, msg):
    with pytest.raises(RuntimeError, match=msg):
        StateCache.wrap(**{**_buffers(), **change})


def test_write_refusals():
    c = _fake()
    k = torch.zeros(3, 2, 64)
    s = torch.zeros(3, dtype=torch.int64)
    for bad, msg in (((k[:2], k, s), "slots must be"), ((k, k, s[:2]), "slots must be"),
                     ((k[..., :32], k, s), "k must be"), ((k, k[:, :1], s), "v must be"),
                     ((k, k.double(), s), "v must be"), ((k, k.half(), s), "alike"),
                     ((k, k, s.float()), "int32 or int64"),
                     ((k.clone().requires_grad_(), k, s), "no backward"), ((k, k, s), "CUDA")):
        with pytest.raises(RuntimeError, match=msg):
            c.write(*bad)


def test_append_and_read_refusals():
    c = _fake()
    k = torch.zeros(3, 2, 64)
    t, n = torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for bad, msg in (((k, k, t[:2], n), "table must be"), ((k, k, t[:, :0], n), "no columns"),
                     ((k, k, t, n[:2]), "lens must be"), ((k, k, t.float(), n), "int32 or int64"),
                     ((k, k, t, n), "CUDA")):
        with pytest.raises(RuntimeError, match=msg):
            c.append(*bad)
    with pytest.raises(RuntimeError, match="one dimension"):
        c.read(t)
    with pytest.raises(RuntimeError, match="read as"):
        c.read(n, torch.float64)
    with pytest.raises(RuntimeError, match="CUDA"):
        c.read(n)


def test_attend_refusals():
    c = _fake()
    q = torch.zeros(3, 4, 64)
    t, n = torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    w = torch.zeros(3, 2, 40)
    for bad, kw, msg in (
            ((q[0], t, n), {}, "q must be"), ((q[..., :32], t, n), {}, "q must be"),
            ((q[:, :3], t, n), {}, "multiple of 2"), ((q.double(), t, n), {}, "q must be float32"),
            ((q, t[:2], n), {}, "table must be"), ((q, t, n[:2]), {}, "lens must be"),
            ((q, t, n.float()), {}, "int32 or int64"),
            ((q.clone().requires_grad_(), t, n), {}, "no backward"),
            ((q, t, n), dict(weights=w[..., :39]), "weights must be"),
            ((q, t, n), dict(weights=w.double()), "weights must be"),
            ((q, t, n), dict(weights=torch.zeros(3, 40, 2).transpose(1, 2)), "contiguous"),
            ((q, t, n), {}, "CUDA")):
        with pytest.raises(RuntimeError, match=msg):
            c.attend(*bad, **kw)


def test_evict_refusals():
    st = torch.zeros(4, 2, 8, 5)
    w, p = torch.zeros(3, 2, 40), torch.zeros(3, 2, 40, dtype=torch.int32)
    t, n = torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    ok = ([st], w, p, t, n, 8)
    for i, bad, msg in ((0, [], "one to eight"), (0, [st] * 9, "one to eight"),
                        (0, [st[:, :1]], "a store must be"), (0, [st, st[:3]], "same pages"),
                        (0, [st.transpose(0, 2)], "a store must be"),
                        (0, [torch.zeros(4, 2, 8, 10)[..., ::2]], "contiguous"),
                        (1, w.double(), "weights"), (1, w[..., :39], "positions"),
                        (2, p.long(), "positions"), (3, t[:2], "table"), (4, n[:2], "lens"),
                        (4, n.float(), "int32 or int64"), (5, 0, "budget")):
        args = list(ok)
        args[i] = bad
        with pytest.raises(RuntimeError, match=msg):
            evict_rows(*args)
    with pytest.raises(RuntimeError, match="column for every slot"):
        evict_rows([st], w[..., :39], None, t, n, 8)
    for kw in (dict(sinks=5, recent=4), dict(sinks=-1), dict(recent=-1)):
        with pytest.raises(RuntimeError, match="sinks"):
            evict_rows(*ok, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        evict_rows(*ok)
    assert dgs.ops.evict_rows is evict_rows and dgs.classes.StateCache is StateCache


def _c(**kw):
    f = dict(k_codes=4096, k_scales=4096, v_codes=4096, v_scales=4096, pages=4, page_size=8,
             heads=2, head_dim=64, group=32)
    f.update(kw)
    c = _CCache(*[f[n] for n, _ in _CCache._fields_])
    return c


@pytest.mark.parametrize("change, msg", [
    (dict(pages=0), b"no pages"), (dict(heads=0), b"no pages"), (dict(page_size=6), b"power of two"),
    (dict(head_dim=68), b"head_dim"), (dict(head_dim=512), b"head_dim"), (dict(group=24), b"group"),
    (dict(v_codes=0), b"null buffer"), (dict(k_scales=4100), b"aligned")])
def test_c_abi_refuses_bad_caches(change, msg):
    c = _c(**change)
    assert lib.dgs_state_read(ctypes.addressof(c), 4096, 1, 0, 4096, 4096, None) == -1
    assert msg in lib.dgs_last_error()


def test_c_abi_refuses_bad_calls():
    c = _c()
    ref = ctypes.addressof(c)
    row = (2 * 64, 64)

    def last(rc, msg):
        assert rc == -1 and msg in lib.dgs_last_error(), lib.dgs_last_error()

    last(lib.dgs_state_write(None, 4096, 4096, 0, 1, *row, *row, 4096, None), b"null")
    last(lib.dgs_state_write(ref, 4096, 4096, 3, 1, *row, *row, 4096, None), b"dtype")
    last(lib.dgs_state_write(ref, 4096, 4096, 0, -1, *row, *row, 4096, None), b"negative")
    last(lib.dgs_state_write(ref, 4100, 4096, 0, 1, *row, *row, 4096, None), b"aligned")
    last(lib.dgs_state_write(ref, 4096, 4096, 1, 1, 128, 64, 128, 60, 4096, None), b"aligned")
    last(lib.dgs_state_write(ref, 4096, 4096, 0, 1, *row, *row, None, None), b"null slots")
    last(lib.dgs_state_append(ref, 4096, 4096, 0, 1, *row, *row, 4096, 4, 0, 4096, 4, 4096, None),
         b"no columns")
    last(lib.dgs_state_append(ref, 4096, 4096, 0, 1, *row, *row, 4096, 2, 1, 4096, 4, 4096, None),
         b"int32 or int64")
    last(lib.dgs_state_attend(ref, 4096, 0, 1, 3, 192, 64, 4096, 4, 1, 4096, 4, 1.0, None, 0, 1.0,
                              4096, None, 0, None), b"multiple")
    last(lib.dgs_state_attend(ref, 4096, 0, 1, 2, 128, 64, 4096, 4, 2, 4096, 4, 1.0, 4096, 15, 1.0,
                              4096, None, 0, None), b"column for every slot")
    last(lib.dgs_evict_rows(None, None, 9, 1, 1, 1, None, None, None, None, 1, 1, None, 4, 1, None,
                            4, None, 1, 0, 0, None, 0, None), b"at most 8")
    last(lib.dgs_evict_rows(None, None, 0, 1, 1, 1, None, None, None, None, 1, 1, None, 4, 1, None,
                            4, None, 1, 1, 1, None, 0, None), b"sinks")
    n = c_i64()
    last(lib.dgs_evict_workspace(1, 1, 1, 0, ctypes.byref(n)), b"bad sizes")
    # nothing to do: no pointer is looked at, no device is needed
    assert lib.dgs_state_write(ref, None, None, 0, 0, *row, *row, None, None) == 0
    assert lib.dgs_state_read(ref, None, 0, 0, None, None, None) == 0
    assert lib.dgs_state_attend(ref, None, 0, 0, 2, 128, 64, None, 4, 1, None, 4, 1.0, None, 0,
                                1.0, None, None, 0, None) == 0


@pytest.mark.parametrize("width", [1 << 30, 1 << 40, (1 << 61) + 1, (1 << 63) - 1, -1])
def test_c_abi_refuses_tables_whose_sizes_do_not_fit(width):
    c = _c()
    ref = ctypes.addressof(c)
    row = (2 * 64, 64)
    n = c_i64(-7)

    def last(rc, msg):
        assert rc == -1 and msg in lib.dgs_last_error(), lib.dgs_last_error()

    last(lib.dgs_state_append(ref, 4096, 4096, 0, 1, *row, *row, 4096, 4, width, 4096, 4, 4096, None),
         b"width")
    last(lib.dgs_state_attend(ref, 4096, 0, 1, 2, 128, 64, 4096, 4, width, 4096, 4, 1.0, 4096, 15,
                              1.0, 4096, None, 0, None), b"width")
    last(lib.dgs_state_attend_workspace(ref, 1, 2, width, 0, 0, ctypes.byref(n)), b"width")
    last(lib.dgs_evict_rows(None, None, 0, 1, 1, 16, 4096, None, 8192, 8192, 1, 1, 4096, 4, width,
                            4096, 4, 4096, 1, 0, 0, None, 0, None), b"width")
    if width > 0:
        last(lib.dgs_evict_workspace(1, 1, width, 1, ctypes.byref(n)), b"bad sizes")
        last(lib.dgs_state_attend_workspace(ref, width * 2 if width < 1 << 60 else width, 2, 1, 0, 0,
                                            ctypes.byref(n)), b"bad rows")
    assert n.value == -7


def test_c_abi_refuses_null_results():
    c = _c()
    assert lib.dgs_state_attend_workspace(ctypes.addressof(c), 1, 2, 1, 0, 0, None) == -1
    assert lib.dgs_evict_workspace(1, 1, 8, 1, None) == -1
    assert lib.dgs_evict_rows(None, None, 1, 1, 1, 1, 4096, None, 8192, 8192, 1, 1, 4096, 4, 1, 4096,
                              4, 4096, 1, 0, 0, None, 0, None) == -1
    assert b"null stores" in lib.dgs_last_error()


def test_neighbour_table():
    seeds = torch.tensor([7, 3, 9])
    frontier = torch.tensor([7, 3, 9, 20, 21])
    row, col = torch.tensor([0, 0, 2, 2, 2]), torch.tensor([3, 1, 4, 4, 0])
    table, lens = dgs.ops.neighbour_table((seeds, frontier, row, col), 4)
    assert lens.tolist() == [2, 0, 3]
    assert table.tolist() == [[20, 3, -1, -1], [-1] * 4, [21, 21, 7, -1]]
    short, lens = dgs.ops.neighbour_table((seeds, frontier, row.int(), col.int()), 2)
    assert lens.tolist() == [2, 0, 2] and short.tolist() == [[20, 3], [-1, -1], [21, 21]]
    with pytest.raises(RuntimeError, match="fan_out"):
        dgs.ops.neighbour_table((seeds, frontier, row, col), 0)


def test_buffers_cannot_be_replaced():
    with pytest.raises(AttributeError):
        _fake().k_codes = torch.zeros(1)
