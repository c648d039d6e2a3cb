"""The state cache's calls at the edges of what it documents, against plain forms."""
import numpy as np
import pytest
import torch

import dgs
import state_ref as ref
from test_state_gpu import same_bits

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
