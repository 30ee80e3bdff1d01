"""The paged cache's host side without a GPU: NULL handles are refused with a message, and the
plain restatement that the GPU tests compare with has the properties that define it."""
import random

import pytest
import torch

from navi_b200 import capi, engine
from oracle import pages as op


def test_null_handles_are_refused():
    L = capi.lib()
    for call in (lambda: L.navi_pages_create(None, None, None), lambda: L.navi_pages_get(None, None), lambda: L.navi_pages_plan(None, None, None),
                 lambda: L.navi_pages_store(None, None, 0, None, None), lambda: L.navi_pages_attend(None, None, 0, None, None),
                 lambda: L.navi_pages_commit(None, None, None, None)):
        assert call() == capi.NAVI_E_ARG
        assert L.navi_last_error()
    L.navi_pages_destroy(None)


def test_argument_records_know_their_fields():
    s = engine.TreeStep(n_req=3, max_rows=5)
    assert (s.s.n_req, s.s.max_rows, s.s.parent) == (3, 5, None)
    with pytest.raises(TypeError):
        engine.CommitArgs(widht=1)


@pytest.mark.parametrize("seed", range(20))
def test_pages_are_owned_once(seed):
    """After any sequence of steps every page is on the stack or in one request's row, once."""
    rng = random.Random(seed)
    B, n_pages = 5, 12
    t = op.Tables.fresh(n_pages, 16, B, 6)
    ctx = [0] * B
    for _ in range(30):
        new = [rng.choice([0, 0, 1, 5, 40]) for _ in range(B)]
        s = op.Step(ctx, new, None)
        op.plan(t, s)
        pages = t.free[:t.n_free] + [p for i in range(B) for p in t.table[i][:t.held[i]]]
        assert sorted(pages) == list(range(n_pages))
        ctx = [0 if rng.random() < 0.2 else c + n if st == op.OK else c for c, n, st in zip(ctx, new, s.status)]


def test_tree_is_its_branches():
    """A tree's row attends like the last row of the chain that its ancestors form."""
    gen = torch.Generator().manual_seed(0)
    t = op.Tables.fresh(8, 16, 1, 4)
    s = op.Step([20], [5], [-1, 0, 0, 2, 1])
    op.plan(t, s)
    assert s.anc == [{0}, {0, 1}, {0, 2}, {0, 2, 3}, {0, 1, 4}] and s.pos == [20, 21, 21, 22, 22]
    k, v = (torch.randn(8, 1, 16, 64, generator=gen).double() for _ in range(2))
    q = torch.randn(5, 2, 64, generator=gen).double()
    out, lse = op.attend(t, s, q, k, v, 0.125)
    c = op.Step([20], [3], None)
    op.plan(t, c)
    k2, v2 = k.clone(), v.clone()
    for n, j in enumerate([0, 2, 3]):
        for a, b in ((k2, k), (v2, v)):
            a[c.slot[n] // 16, :, c.slot[n] % 16] = b[s.slot[j] // 16, :, s.slot[j] % 16]
    o2, l2 = op.attend(t, c, q[[0, 2, 3]], k2, v2, 0.125)
    assert torch.allclose(out[[0, 2, 3]], o2) and torch.allclose(lse[[0, 2, 3]], l2)
    # and committing that branch makes the same cache
    tok = [[1], [2], [3], [4], [5]]
    paths, nxt = op.commit(16, s, tok, [[3], [0], [4], [9], [0]], [[1]], [k, v])
    assert paths == [[0, 2, 3]] and nxt == [[9]]
    L = [c.slot[n] for n in range(3)]
    for a, b in ((k2, k), (v2, v)):
        for x in L:
            assert torch.equal(a[x // 16, :, x % 16], b[x // 16, :, x % 16])


def test_kernels_launched_early_read_nothing_as_constant():
    """plan, store, attend and commit may be resident while the launch before them still writes what they read: loads
    through the read-only path (__ldg, ld.global.nc, restrict pointers) are for data that nobody writes meanwhile."""
    import pathlib
    import re
    src = pathlib.Path(__file__).resolve().parent.parent / "navi-tts_b200" / "csrc"
    files = sorted(src.glob("paged_attn*")) + [src / "pages.cu"]
    assert len(files) == 6
    for f in files:
        code = re.sub(r"//.*", "", f.read_text())
        assert not re.search(r"__ldg|global\.nc|__restrict__", code), f.name


def test_wrap_needs_a_v_pool_for_each_k_pool():
    for k, v in (([16], []), ([], [16]), ([16, 32], [48])):
        with pytest.raises(ValueError, match="pools"):
            engine.PagedKv.wrap(None, k, v, 4, 16, 2, 128, capi.NAVI_F16, 2, 2, 16, 16, 16, 16)


def test_copies_land_before_a_block_that_gave_up_ends():
    """A wait of any warp may give up after the warp that copies has left its loop: the copies under way (K and V, and q
    by TMA in the kernel for many rows) are waited for behind the last barrier of the block."""
    import pathlib
    src = pathlib.Path(__file__).resolve().parent.parent / "navi-tts_b200" / "csrc"
    few, many = ((src / f).read_text() for f in ("paged_attn_few.cu", "paged_attn_many.cu"))
    assert few.index("named_sync(2, 288);") < few.index("mbar_drain(") and few.count("named_sync(2, 288);") == 2
    last = many.rindex("__syncthreads();")
    assert many.index("mbar_drain(&S.full[") > last and many.index("mbar_drain(&S.q_full") > last
