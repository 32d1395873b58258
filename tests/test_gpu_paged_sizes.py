"""PagedKv::attention at the ends of its sizes: rows past what one launch of the join covers."""
import numpy as np
import pytest

import gie
from paged_plain import Cache

pytestmark = pytest.mark.gpu


def test_more_rows_than_a_join_could_take():
    """2^26 rows of q (2^32 values), which no launch of the join covers: nothing is split here, so nothing is joined.
    Every sequence has the same tokens and the same page."""
    import torch
    new, heads, dim, batch = 32, 64, 64, 1 << 15
    c = Cache([new], [new], heads=heads, kv_heads=1, dim=dim, page=32, precision="fp16", seed=21)
    one = torch.from_numpy(c.q).half().cuda()
    q = one.repeat(batch, 1, 1)
    out = torch.full_like(q, 7)
    k, v = (torch.from_numpy(t).half().cuda() for t in (c.k_pages, c.v_pages))
    starts = torch.arange(0, batch * new + 1, new, dtype=torch.int32).cuda()
    lens = torch.full((batch,), new, dtype=torch.int32).cuda()
    table = torch.full((batch, 1), int(c.table[0, 0]), dtype=torch.int32).cuda()
    p = gie.PagedKv(batch, batch * new, heads, 1, dim, 32, c.pages, 1, max_new=new, max_len=new)
    assert gie.paged_attention_workspace_size(p) == 0
    torch.cuda.synchronize()
    print("attend", p, flush=True)
    gie.paged_attention(p, q.data_ptr(), k.data_ptr(), v.data_ptr(), starts.data_ptr(), lens.data_ptr(), table.data_ptr(),
                        out.data_ptr())
    torch.cuda.synchronize()
    want, bound = c.plain()
    assert (np.abs(out[:new].float().cpu().numpy() - want) <= bound).all()
    assert bool((out.view(batch, -1) == out[:new].reshape(1, -1)).all())


def check(c, **hints):
    got = c.attend(**hints).astype(np.float64)
    want, bound = c.plain()
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("batch", [64, 65, 70])
@pytest.mark.parametrize("chunk", [1, 40])
def test_parts_are_joined_in_large_batches(batch, chunk):
    """The join finds a token's sequence by lanes up to 64 sequences and by a search past them; sequences without new
    tokens and one with a chunk among them, one context long enough to be split, the others in one part."""
    new = [b % 3 > 0 for b in range(batch)]
    new = [int(n) for n in new]
    new[batch - 4] = chunk
    lens = [n + 11 * b % 60 for b, n in enumerate(new)]
    lens[batch - 4] = 3000
    c = Cache(new, lens, heads=2, kv_heads=1, dim=64, page=32, seed=batch)
    hints = dict(max_new=max(new), max_len=3000)
    assert gie.paged_attention_workspace_size(c.p(**hints)) > 0
    check(c, **hints)


def test_more_sequences_than_two_searches_cover():
    """Past 4096 sequences the search for a row's sequence takes three steps."""
    rng = np.random.default_rng(5)
    new = rng.integers(0, 3, 4200).tolist()
    lens = [n + int(rng.integers(0, 20)) for n in new]
    check(Cache(new, lens, heads=2, kv_heads=1, dim=64, seed=6))
