"""Edges of the paged cache's calls (navi_pages_*): requests that are refused, the ends of the types'
ranges, shared buffers, graphs. Against the plain 64-bit restatement of oracle/pages.py, as
test_pages_gpu.py, whose caches and steps are used. navi_pages_check follows each attend, so that a wait
that ran out fails the test even where the results are right."""
import ctypes
import math
import random

import pytest
import torch

from navi_b200 import capi, engine
from oracle import pages as op
from test_pages_gpu import TYPES, U, Cache, GpuStep, check_attend, drafts, fill_tokens, i32, planned, tree

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


# ---- requests that are not served ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group,n", [(1, 129), (1, 256), (1, 300), (2, 65), (2, 128), (2, 150), (3, 43), (3, 86), (3, 100)])
@pytest.mark.parametrize("why", ["full", "shape", "parent"])
@pytest.mark.parametrize("first", [True, False])
def test_attend_refused_requests_of_many_rows(dev, dtype, group, n, why, first):
    """129, about 256 and 300 rows x heads of a request that is not served, before or after one that is:
    0 and -inf for it, its neighbour as without it."""
    if why == "parent" and n > 256:
        pytest.skip("a tree has at most 256 rows")
    _, _, kt, kcode = TYPES[dtype]
    need, ctx1, served = -(-n // 16), 70, 9                  # pages of 16; the other request has 70 + 9 tokens, or 16 + 9
    if why == "full":
        served = 140
        blocks, n_pages = max(need, 14), 5 + need - 1 if first else 14
    elif why == "shape":
        ctx1, blocks, n_pages = 16, need - 1, 64
    else:
        blocks, n_pages = max(need, 5), 64
    c = Cache(dev, rows=2, blocks=blocks, n_pages=n_pages, G=1, kt=kt, code=kcode)
    planned(c, [0], [ctx1], None, req=[1])
    order = [0, 1] if first else [1, 0]
    ctx, new = [0 if r == 0 else ctx1 for r in order], [n if r == 0 else served for r in order]
    par = None
    if why == "parent":
        rng = random.Random(n)
        trees = {0: tree(rng, n), 1: tree(rng, served)}
        trees[0][n - 1] = n - 1                             # not below its row
        par = sum((trees[r] for r in order), [])
    g = planned(c, ctx, new, par, req=order)
    status = g.status.tolist()
    assert status[order.index(0)] == {"full": capi.NAVI_E_KV_FULL, "shape": capi.NAVI_E_SHAPE, "parent": capi.NAVI_E_ARG}[why]
    # a later request that needs pages waits for the one that does not fit
    assert status[order.index(1)] == (capi.NAVI_E_KV_FULL if why == "full" and first else capi.NAVI_OK)
    fill_tokens(c, g, torch.Generator().manual_seed(n), kt)
    out, lse = check_attend(c, g, dtype, group)
    c.h.check(stream=0)
    a = 0 if first else served
    assert (out[a:a + n] == 0).all() and (lse[a:a + n] == -math.inf).all()


# ---- the ends of the types' ranges ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new,H", [(1, 2), (5, 2), (12, 2), (40, 2), (90, 2)])
@pytest.mark.parametrize("ctx,nats", [(700, 10.0), (8192, 18.0), (8192, 20.0), (60000, 17.0)])
def test_attend_long_tail_under_a_few_large_weights(dev, dtype, new, H, ctx, nats):
    """Every 16th key far above the others, and V zero there: the result is the others' sum alone, which a
    weight that is dropped or rounded to a multiple of 2^-24 of the largest would show.

    Weights: 2^-25 of f16's terms against 2^(13 - nats log2 e) at the least (an f16 cache), their one rounding
    (16-bit rows), scores of up to 60 in f32 (60 x 2^-23 twice, and the same of log2 e), sums over the keys of
    relative 2^-23 a 16-key step."""
    tt, _, kt, kcode = TYPES[dtype]
    D, page = 128, 64
    c = Cache(dev, rows=1, blocks=-(-(ctx + new) // page), page=page, G=1, D=D, kt=kt, code=kcode, fill=0)
    planned(c, [0], [ctx], None)
    g = planned(c, [ctx], [new])
    c.v[..., 0::2], c.v[..., 1::2] = 1.0, 1.5
    scale, q0, top = D ** -0.5, 8.0, 64.0                   # scores up to 45
    low = float(torch.tensor(top - nats / (scale * q0)).to(kt))
    c.k[..., 0] = low
    where = torch.tensor(c.t.table[0])[:-(-ctx // page)].cuda()
    keys = torch.arange(0, ctx, 16, device="cuda")
    c.k[0, where[keys // page], 0, keys % page, 0] = top
    c.v[0, where[keys // page], 0, keys % page] = 0.0
    q = torch.zeros(new, H, D)
    q[..., 0] = q0
    qd, out = q.to(tt).cuda(), torch.zeros(new, H, D, dtype=tt, device="cuda")
    c.h.attend(g.c, 0, engine.AttendArgs(q=qd.data_ptr(), out=out.data_ptr(), dtype=TYPES[dtype][1], n_head=H, scale=scale), stream=0)
    c.h.check(stream=0)
    gap = (top - low) * q0 * scale
    many = torch.tensor([len(a) for a in g.s.anc]).double() + ctx - len(keys)
    share = many * math.exp(-gap) / (many * math.exp(-gap) + len(keys))
    want = share[:, None, None] * torch.where(torch.arange(D) % 2 == 0, 1.0, 1.5).double()
    rel = 2.0 ** (gap * math.log2(math.e) - 13 - 25) if kt == torch.float16 else 0.0
    rel += 4 * 60 * 2.0 ** -23 + (ctx + new) / 16 * 2.0 ** -23 + (0 if dtype == "f32" else U[dtype])
    tiny = 2.0 ** -25 if dtype == "f16" else 0.0            # f16's own smallest step in the result
    assert ((out.cpu().double() - want).abs() <= (rel + U[dtype]) * want + tiny).all(), ((out.cpu().double() / want - 1).abs().max(), rel)


@pytest.mark.parametrize("new,H,D", [(1, 2, 128), (4, 4, 64), (7, 2, 128), (16, 2, 64), (50, 2, 128), (150, 1, 64)])
@pytest.mark.parametrize("size", [1e5, 1e-4, 1e30, 1e-20])
@pytest.mark.parametrize("ctx", [90, 1500])
def test_attend_f32_rows_of_any_size(dev, new, H, D, size, ctx):
    """f32 q far from 1, its magnitude taken out again by the scale, a row of another magnitude, a row of zeros: the
    tolerance of standard normal rows (check_attend's), as the scores are theirs."""
    c = Cache(dev, rows=1, blocks=-(-(ctx + new) // 16), G=1, D=D, fill=0)
    c.k.normal_(generator=torch.Generator("cuda").manual_seed(1))
    c.v.normal_(generator=torch.Generator("cuda").manual_seed(2))
    planned(c, [0], [ctx], None)
    g = planned(c, [ctx], [new])
    x = torch.randn(new, H, D, generator=torch.Generator().manual_seed(new))
    x[0, 0, 1:] *= 2.0 ** -9
    if new > 2:
        x[1] *= 2.0 ** -12
        x[2, H - 1] = 0
    q = x * size
    qd, out, lse = q.cuda(), torch.zeros(new, H, D, device="cuda"), torch.zeros(new, H, device="cuda")
    scale = D ** -0.5 / size
    c.h.attend(g.c, 0, engine.AttendArgs(q=qd.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(), dtype=capi.NAVI_F32, n_head=H, scale=scale), stream=0)
    c.h.check(stream=0)
    kd, vd = c.k[0].cpu().double(), c.v[0].cpu().double()
    want, wl = op.attend(c.t, g.s, q.double(), kd, vd, scale)
    ds = 2.0 ** -20 * scale * float(q.double().abs().sum(2).max()) * float(kd.abs().max())
    tol = float(vd.abs().max()) * (2 * ds + 2.0 ** -20 + (ctx + new) * 2.0 ** -24)
    assert ((out.cpu().double() - want).abs() <= tol + 2.0 ** -24 * want.abs()).all(), (out.cpu().double() - want).abs().max()
    assert ((lse.cpu().double() - wl).abs() <= ds + 2.0 ** -20 + (ctx + new) * 2.0 ** -24 + 2.0 ** -22 * wl.abs()).all()


# ---- arguments ----------------------------------------------------------------------------------------

def refused(status, fn, *a, **kw):
    with pytest.raises(capi.NaviError) as e:
        fn(*a, **kw)
    assert e.value.status == status and len(str(e.value)) > 12


def step_with(g, **kw):
    return engine.TreeStep(**{**{n: getattr(g.c.s, n) for n, _ in capi.Step._fields_}, **kw})


def test_plan_without_a_mask(dev):
    """Words of a mask without a mask are refused, whatever max_new says; max_new 0 and no words are a step whose requests
    with rows are refused, each by its status."""
    c = Cache(dev, rows=2, blocks=4)
    g = planned(c, [3, 0], [2, 0])
    for kw in (dict(max_new=0, mask_words=1, mask=0), dict(max_new=0, mask_words=4, mask=0), dict(max_new=2, mask_words=1, mask=0),
               dict(max_new=1, mask_words=0, mask=0)):
        for call in (lambda s: c.h.plan(s, stream=0), lambda s: c.h.commit(s, engine.CommitArgs(width=1), stream=0)):
            refused(capi.NAVI_E_ARG, call, step_with(g, **kw))
    c.h.plan(step_with(g, max_new=0, mask_words=0, mask=0), stream=0)
    torch.cuda.synchronize()
    assert g.status.tolist() == [capi.NAVI_E_SHAPE, capi.NAVI_OK] and g.slot.tolist() == [-1, -1]


# ---- shared buffers -------------------------------------------------------------------------------------

@pytest.mark.parametrize("width", [1, 5, 16, 40])
@pytest.mark.parametrize("B", [1, 3, 200])
def test_commit_in_place(dev, width, B):
    """One step's next_token is the next one's root_target, its new_len the next one's ctx_len: both in the same buffer.
    Few requests have hundreds of blocks, which all read the root's ids."""
    rng = random.Random(width * B)
    ctx, new = [rng.randrange(60) for _ in range(B)], [rng.randrange(13) for _ in range(B)]
    c = Cache(dev, rows=B, blocks=5, G=2, D=64, L=28, fill=0)
    planned(c, [0] * B, ctx, None)
    g = planned(c, ctx, new)
    for rep in range(8):
        tok, tgt, root = drafts(rng, g.s, width, (0.0, 0.9, 1.0)[rep % 3], vocab=3 if width == 1 else 50)
        T = max(g.s.cu[-1], 1)
        ids, tg, nx = i32(sum(tok, []) or [0]), i32(sum(tgt, []) or [0]), i32(sum(root, []))
        acc, path, nl = i32([-7] * B), i32([-7] * T), g.ctx.clone()
        c.k.normal_(generator=torch.Generator("cuda").manual_seed(rep))
        c.v.normal_(generator=torch.Generator("cuda").manual_seed(rep + 100))
        kw, vw = c.k.cpu().clone(), c.v.cpu().clone()
        c.h.commit(step_with(g, ctx_len=nl.data_ptr()), engine.CommitArgs(width=width, tokens=ids.data_ptr(), targets=tg.data_ptr(), root_target=nx.data_ptr(),
                                                                          accepted=acc.data_ptr(), path=path.data_ptr(), new_len=nl.data_ptr(),
                                                                          next_token=nx.data_ptr()), stream=0)
        torch.cuda.synchronize()
        paths, nxt = op.commit(16, g.s, tok, tgt, root, [x for l in range(28) for x in (kw[l], vw[l])])
        assert acc.tolist() == [len(p) for p in paths] and nl.tolist() == [x + len(p) for x, p in zip(ctx, paths)]
        assert nx.view(B, width).tolist() == nxt
        assert torch.equal(c.k.cpu(), kw) and torch.equal(c.v.cpu(), vw)


def test_commit_refuses_an_outcome_over_the_ids(dev):
    c = Cache(dev, rows=2, blocks=4)
    g = planned(c, [3, 0], [2, 4])
    x = i32([0] * 256)
    p = lambda n: x[n:].data_ptr()  # noqa: E731
    good = dict(width=2, tokens=p(0), targets=p(16), root_target=p(32), accepted=p(48), path=p(64), new_len=p(80), next_token=p(96))
    for kw in (dict(next_token=p(33)), dict(next_token=p(1)), dict(next_token=p(15)), dict(path=p(20)), dict(accepted=p(35)), dict(new_len=p(11))):
        refused(capi.NAVI_E_ARG, c.h.commit, g.c, engine.CommitArgs(**{**good, **kw}), stream=0)
    c.h.commit(g.c, engine.CommitArgs(**good), stream=0)
    torch.cuda.synchronize()


# ---- pools that the library allocates --------------------------------------------------------------------

@pytest.mark.parametrize("tables", ["own", "library"])
def test_rows_stored_right_after_create_stay(dev, tables):
    """Pools of 8 GB are zeroed before create returns: rows stored at once, on a stream that waits for no other, are there."""
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip("needs 30 GB free")
    G, D, page, L, blocks = 8, 128, 16, 2, 4
    n_pages = (2 << 30) // (G * D * page * 2)
    H, T = 1, 3 * page
    s = op.Step([0], [T], None)
    g = GpuStep(s)
    qkv = torch.randn(T, (H + 2 * G) * D, generator=torch.Generator().manual_seed(0)).half().cuda()
    q = torch.zeros(T, H * D, dtype=torch.float16, device="cuda")
    t = op.Tables.fresh(n_pages, page, 1, blocks)           # page 0 on top; own tables: the last page, which is zeroed last
    if tables == "own":
        t.free.sort()
    table, held, free, n_free = i32([0] * blocks), i32([0]), i32(t.free), i32([n_pages])
    op.plan(t, s)
    torch.cuda.synchronize()
    p = lambda x: x.data_ptr()  # noqa: E731
    d = capi.PagesDesc(L, n_pages, page, G, D, capi.NAVI_F16, 1, blocks)
    if tables == "own":
        d.table, d.held, d.free_pages, d.n_free = p(table), p(held), p(free), p(n_free)
    kv = engine.PagedKv(dev, d)
    kv.plan(g.c)                                            # on the engine's stream
    a = engine.StoreArgs(qkv=p(qkv), q_out=p(q), dtype=capi.NAVI_F16, n_head=H)
    for l in range(L - 1, -1, -1):
        kv.store(g.c, l, a)
    kv.check()
    desc = kv.desc()
    cudart = ctypes.CDLL("libcudart.so.12")
    for l in range(L):
        for pool, first in ((desc.k, H), (desc.v, H + G)):
            for b in range(3):
                got = torch.empty(G, page, D, dtype=torch.float16, device="cuda")
                src = pool[l] + t.table[0][b] * G * page * D * 2
                assert cudart.cudaMemcpy(ctypes.c_void_p(p(got)), ctypes.c_void_p(src), ctypes.c_size_t(got.numel() * 2), 3) == 0
                want = qkv[b * page:(b + 1) * page].view(page, H + 2 * G, D)[:, first:first + G].transpose(0, 1)
                assert torch.equal(got, want)
    kv.close()


# ---- graphs ------------------------------------------------------------------------------------------------

class Whole:
    """plan, store, attend and commit of a drafted step over a cache of its own, with buffers that stay."""

    def __init__(self, dev, seed, H=4, G=2, D=128):
        rng = random.Random(seed)
        self.H, self.G, self.D = H, G, D
        self.ctx, self.new = [2900, 1500 + seed, 20], [9, 1 + seed % 3, 4]
        self.c = Cache(dev, rows=3, blocks=200, n_pages=320, G=G, D=D, seed=seed, fill=0)
        self.c.k.normal_(generator=torch.Generator("cuda").manual_seed(seed))
        self.c.v.normal_(generator=torch.Generator("cuda").manual_seed(seed + 1))
        planned(self.c, [0] * 3, self.ctx, None)
        self.s = op.Step(self.ctx, self.new, sum((tree(rng, n) for n in self.new), []))
        self.g = GpuStep(self.s)
        T = sum(self.new)
        gen = torch.Generator().manual_seed(seed)
        self.qkv = torch.randn(T, (H + 2 * G) * D, generator=gen).half().cuda()
        self.q, self.out = (torch.zeros(T, H * D, dtype=torch.float16, device="cuda") for _ in range(2))
        self.tok = i32(rng.randrange(2) for _ in range(T))
        self.tgt, self.root = i32(rng.randrange(2) for _ in range(T)), i32(rng.randrange(2) for _ in self.ctx)
        self.acc, self.path, self.nl, self.nx = i32([-7] * 3), i32([-7] * T), i32([-7] * 3), i32([-7] * 3)
        p = lambda x: x.data_ptr()  # noqa: E731
        self.sa = engine.StoreArgs(qkv=p(self.qkv), q_out=p(self.q), dtype=capi.NAVI_F16, n_head=H)
        self.aa = engine.AttendArgs(q=p(self.q), out=p(self.out), dtype=capi.NAVI_F16, n_head=H, scale=D ** -0.5)
        self.ca = engine.CommitArgs(width=1, tokens=p(self.tok), targets=p(self.tgt), root_target=p(self.root), accepted=p(self.acc),
                                    path=p(self.path), new_len=p(self.nl), next_token=p(self.nx))
        self.state = [self.c.k, self.c.v, self.c.table, self.c.held, self.c.free, self.c.n_free]
        self.before = [x.clone() for x in self.state]

    def run(self, stream):
        self.c.h.plan(self.g.c, stream=stream)
        self.c.h.store(self.g.c, 0, self.sa, stream=stream)
        for _ in range(6):                                  # many pieces to join
            self.c.h.attend(self.g.c, 0, self.aa, stream=stream)
        self.c.h.commit(self.g.c, self.ca, stream=stream)

    def again(self):
        """The cache as it was, the results cleared; on the current stream."""
        for x, y in zip(self.state, self.before):
            x.copy_(y)
        for x in (self.out, self.q, self.acc, self.path, self.nl, self.nx, self.g.slot):
            x.zero_()

    def results(self):
        return [x.clone() for x in (self.out, self.q, self.acc, self.path, self.nl, self.nx, self.g.slot, self.c.k, self.c.v, self.c.table)]


def test_graphs_of_one_stream_side_by_side(dev):
    """Two steps captured on one stream, the first calls on it, replayed on two others while a third step is called on the
    stream itself: each as when it runs alone."""
    steps = [Whole(dev, k) for k in range(3)]
    wants = []
    for w in steps:
        w.run(0)
        w.c.h.check(stream=0)
        wants.append(w.results())
        w.again()
    # the first one's attention against the oracle; the others by it
    w = steps[0]
    op.plan(w.c.t, w.s)
    cap, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    graphs = []
    for w in steps[:2]:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=cap):
            w.run(cap.cuda_stream)
        graphs.append(gr)
    for rep in range(10):
        for w in steps:
            w.again()
        torch.cuda.synchronize()
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        steps[2].run(cap.cuda_stream)
        torch.cuda.synchronize()
        for w, want in zip(steps, wants):
            assert all(torch.equal(x, y) for x, y in zip(w.results(), want))
    w.c.h.check(stream=cap.cuda_stream)
    s, w = steps[0].s, steps[0]
    w.again()
    kd, vd = w.c.k[0].cpu().double(), w.c.v[0].cpu().double()
    T = s.cu[-1]
    q = op.store(16, s, w.qkv.cpu(), w.H, w.G, kd, vd)
    want, _ = op.attend(w.c.t, s, q, kd, vd, w.D ** -0.5)
    # check_attend's tolerance: scores by f32 sums of exact products, f16 weights and result, the sums over the keys
    ds = 2.0 ** -20 * w.D ** -0.5 * float(q.abs().sum(2).max()) * float(kd.abs().max())
    tol = float(vd.abs().max()) * (2 * ds + 2.0 ** -20 + 3000 * 2.0 ** -24 + U["f16"])
    assert ((wants[0][0].cpu().double().view(T, w.H, w.D) - want).abs() <= tol + U["f16"] * want.abs()).all()
    # the scratch of graphs that are gone serves the next ones: 20 captures take no more memory than two
    del gr, graphs
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(20):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=cap):
            steps[0].run(cap.cuda_stream)
        gr.replay()
        torch.cuda.synchronize()
        gr.reset()
    assert free - torch.cuda.mem_get_info()[0] < 10 * (39 << 20)


def test_check_refuses_a_stream_that_is_captured(dev):
    w = Whole(dev, 5)
    st, gr = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=st):
        refused(capi.NAVI_E_ARG, w.c.h.check, stream=st.cuda_stream)
        w.run(st.cuda_stream)
    gr.replay()
    w.c.h.check(stream=0)


def test_a_bad_parent_takes_pages_until_the_next_plan(dev):
    """What the header says of it: pages taken, slots for the rows above the bad one, nothing attended or accepted; a
    plan without rows gives the pages back."""
    c = Cache(dev, rows=2, blocks=4, n_pages=5, fill=0)
    planned(c, [0, 0], [10, 3], None)
    stack = c.free.tolist()[:c.n_free.item()]
    g = planned(c, [10, 3], [30, 2], [-1] + list(range(28)) + [29] + [-1, 0])
    assert g.status.tolist() == [capi.NAVI_E_ARG, capi.NAVI_OK] and c.held.tolist() == [3, 1]
    assert all(x >= 0 for x in g.slot.tolist()[:29]) and g.slot.tolist()[29] == -1
    out, lse = check_attend(c, g, "f16", 2)
    assert (out[:30] == 0).all() and (lse[:30] == -math.inf).all()
    ids, acc, path, nl, nx = i32([1] * 32), i32([-7] * 2), i32([-7] * 32), i32([-7] * 2), i32([-7] * 2)
    root = i32([1, 1])
    c.h.commit(g.c, engine.CommitArgs(width=1, tokens=ids.data_ptr(), targets=ids.data_ptr(), root_target=root.data_ptr(), accepted=acc.data_ptr(),
                                      path=path.data_ptr(), new_len=nl.data_ptr(), next_token=nx.data_ptr()), stream=0)
    c.h.check(stream=0)
    assert acc.tolist() == [0, 2] and nl.tolist() == [10, 5] and path.tolist() == [-1] * 30 + [0, 1]
    planned(c, [10, 3], [0, 0], None)
    assert c.free.tolist()[:c.n_free.item()] == stack and c.held.tolist() == [1, 1]


@pytest.mark.parametrize("n", [257, 300, 700])
def test_commit_path_of_a_refused_tree_of_many_rows(dev, n):
    """A tree of more rows than a tree may have is refused; path is -1 in all of its rows."""
    c = Cache(dev, rows=2, blocks=60, fill=0)
    g = planned(c, [0, 0], [n, 2], [x - 1 for x in range(n)] + [-1, 0], max_new=256)
    assert g.status.tolist() == [capi.NAVI_E_SHAPE, capi.NAVI_OK]
    ids, acc, path, nl, nx = i32([1] * (n + 2)), i32([-7] * 2), i32([-7] * (n + 4)), i32([-7] * 2), i32([-7] * 2)
    root = i32([1, 1])
    c.h.commit(g.c, engine.CommitArgs(width=1, tokens=ids.data_ptr(), targets=ids.data_ptr(), root_target=root.data_ptr(), accepted=acc.data_ptr(),
                                      path=path.data_ptr(), new_len=nl.data_ptr(), next_token=nx.data_ptr()), stream=0)
    torch.cuda.synchronize()
    assert acc.tolist() == [0, 2] and nl.tolist() == [0, 2] and nx.tolist() == [1, 1]
    assert path.tolist() == [-1] * n + [0, 1] + [-7] * 2


def test_layers_without_a_pool_are_refused(dev):
    """Tables without pools serve plan alone; a layer with one of two pools none of the others."""
    x = torch.zeros(1 << 16, dtype=torch.float16, device="cuda")
    table, held, free, n_free = i32([0] * 8), i32([0] * 2), i32(range(4)), i32([4])
    p = lambda t: t.data_ptr()  # noqa: E731
    s = op.Step([0, 0], [3, 2], [-1, 0, 1, -1, 0])
    g = GpuStep(s)
    ids = i32([0] * 64)
    co = engine.CommitArgs(width=1, tokens=p(ids), targets=p(ids), root_target=p(ids), accepted=p(ids[16:]), path=p(ids[24:]), new_len=p(ids[32:]),
                           next_token=p(ids[40:]))
    for k, v in (([0, 0], [0, 0]), ([p(x), 0], [p(x), p(x)]), ([p(x), p(x)], [p(x), 0])):
        kv = engine.PagedKv.wrap(dev, k, v, n_pages=4, page_size=16, n_kv_head=2, head_dim=128, dtype=capi.NAVI_F16, max_requests=2, max_blocks=4,
                                 table=p(table), held=p(held), free_pages=p(free), n_free=p(n_free))
        kv.plan(g.c, stream=0)
        torch.cuda.synchronize()
        assert g.status.tolist() == [0, 0]
        refused(capi.NAVI_E_ARG, kv.store, g.c, 1, engine.StoreArgs(qkv=p(x), q_out=p(x), dtype=capi.NAVI_F16, n_head=2), stream=0)
        refused(capi.NAVI_E_ARG, kv.attend, g.c, 1, engine.AttendArgs(q=p(x), out=p(x[8192:]), dtype=capi.NAVI_F16, n_head=2, scale=1.0), stream=0)
        refused(capi.NAVI_E_ARG, kv.commit, g.c, co, stream=0)


def test_store_refuses_q_over_other_rows(dev):
    """q in place of its rows or between them, not over rows that are still to be read: the default stride of rows in place."""
    c = Cache(dev, rows=2, blocks=4, fill=0)
    g = planned(c, [3, 0], [2, 4])
    H, G, D, T = 4, 2, 128, 6
    W = (H + 2 * G) * D
    x = torch.randn(T + 2, W + H * D, generator=torch.Generator().manual_seed(0)).cuda()
    p, f, one = x.data_ptr(), 4, x.shape[1]
    base = dict(qkv=p, dtype=capi.NAVI_F32, n_head=H)
    for kw in (dict(q_out=p), dict(q_out=p + f * D, qkv_stride=one, q_out_stride=one), dict(q_out=p + f * one, qkv_stride=one, q_out_stride=one),
               dict(q_out=p + f * (W - D), qkv_stride=one, q_out_stride=one), dict(q_out=p + f * W, qkv_stride=one),
               dict(q_out=p + f * (W + D), qkv_stride=one, q_out_stride=one), dict(q_out=p, qkv_stride=one, q_out_stride=one - 4)):
        refused(capi.NAVI_E_ARG, c.h.store, g.c, 0, engine.StoreArgs(**base, **kw), stream=0)
    kw, vw = c.k[0].cpu().double(), c.v[0].cpu().double()
    want = op.store(16, g.s, x[:T, :W].cpu(), H, G, kw, vw)
    for off in (W, 0):                                      # between the rows, then in place
        c.h.store(g.c, 0, engine.StoreArgs(**base, q_out=p + f * off, qkv_stride=one, q_out_stride=one), stream=0)
        torch.cuda.synchronize()
        assert (x[:T, off:off + H * D].cpu().double().view(T, H, D) - want).abs().max() < 1e-6
    g1 = planned(c, [0], [1], req=[1])
    y = x[T:, :].contiguous()
    want = y[:1, :H * D].clone()
    c.h.store(g1.c, 0, engine.StoreArgs(qkv=y.data_ptr(), q_out=y.data_ptr(), dtype=capi.NAVI_F32, n_head=H), stream=0)   # one row: no other
    torch.cuda.synchronize()
    assert torch.equal(y[:1, :H * D], want)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("parent", ["tree", None])
@pytest.mark.parametrize("new", [[1, 2], [70, 3], [200, 300]])
def test_attend_with_max_new_zero(dev, dtype, parent, new):
    """No request may have rows: those that have are refused, and their rows get 0 and -inf as any refused request's."""
    _, _, kt, kcode = TYPES[dtype]
    c = Cache(dev, rows=2, blocks=20, G=1, kt=kt, code=kcode)
    rng = random.Random(1)
    s = op.Step([0, 0], new, sum((tree(rng, n) for n in new), []) if parent else None, max_new=0)
    g = GpuStep(s, words=0)
    c.h.plan(g.c, stream=0)
    op.plan(c.t, s)
    torch.cuda.synchronize()
    assert g.status.tolist() == [capi.NAVI_E_SHAPE] * 2
    out, lse = check_attend(c, g, dtype, 2)
    c.h.check(stream=0)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_attend_refuses_more_rows_than_its_counts_hold(dev):
    """Room for rows whose number times the heads passes 31 bits, or the exact quotients of 32; nothing is launched."""
    c = Cache(dev, rows=1, blocks=4, G=1)
    g = planned(c, [0], [3])
    x = torch.zeros(1 << 14, device="cuda")
    for rows, H in ((1 << 30, 2), (1 << 24, 128), (1 << 29, 3), (5_000_000, 31)):
        refused(capi.NAVI_E_SHAPE, c.h.attend, step_with(g, max_rows=rows, max_new=4),
                0, engine.AttendArgs(q=x.data_ptr(), out=x.data_ptr() + 32768, dtype=capi.NAVI_F32, n_head=H, scale=0.1), stream=0)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,G,D,new", [(4, 2, 128, [1, 1, 1]), (4, 2, 64, [4, 1, 3]), (8, 1, 128, [1, 0, 1]), (3, 3, 64, [8, 5, 7])])
def test_attend_16_bit_rows_of_tiles_of_8_keep_their_weights(dev, dtype, H, G, D, new):
    """Up to 8 rows x heads: weights enter the product as two terms (2^-16 of each with bf16, 2^-22 with f16), so the error is
    that of f32 rows and the result's one rounding."""
    tt, code, kt, kcode = TYPES[dtype]
    ctx = [1500, 3, 700]
    c = Cache(dev, rows=3, blocks=100, G=G, D=D, kt=kt, code=kcode, fill=0)
    c.k.normal_(generator=torch.Generator("cuda").manual_seed(1))
    c.v.normal_(generator=torch.Generator("cuda").manual_seed(2))
    planned(c, [0] * 3, ctx, None)
    g = planned(c, ctx, new)
    T = sum(new)
    q = (torch.randn(T, H, D, generator=torch.Generator().manual_seed(3)) * 2).to(tt)
    qd, out = q.cuda(), torch.zeros(T, H, D, dtype=tt, device="cuda")
    c.h.attend(g.c, 0, engine.AttendArgs(q=qd.data_ptr(), out=out.data_ptr(), dtype=code, n_head=H, scale=D ** -0.5), stream=0)
    c.h.check(stream=0)
    kd, vd = c.k[0].cpu().double(), c.v[0].cpu().double()
    want, _ = op.attend(c.t, g.s, q.double(), kd, vd, D ** -0.5)
    ds = 2.0 ** -20 * D ** -0.5 * float(q.double().abs().sum(2).max()) * float(kd.abs().max())
    tol = float(vd.abs().max()) * (2 * ds + 2.0 ** -20 + 1510 * 2.0 ** -24) + (2.0 ** -16 if dtype == "bf16" else 2.0 ** -22) * float(vd.abs().max())
    assert ((out.cpu().double() - want).abs() <= tol + U[dtype] * want.abs()).all(), ((out.cpu().double() - want).abs().max(), tol)


# ---- pages of 64 ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,G,D", [(4, 2, 128), (2, 2, 64)])
@pytest.mark.parametrize("parent", ["tree", None])
@pytest.mark.parametrize("ctx,new", [([0, 63, 64], [1, 1, 1]), ([129, 65, 0], [12, 3, 64]), ([200], [190])])
def test_attend_pages_of_64(dev, dtype, H, G, D, parent, ctx, new):
    _, _, kt, kcode = TYPES[dtype]
    c = Cache(dev, rows=len(ctx), blocks=7, page=64, G=G, D=D, kt=kt, code=kcode)
    planned(c, [0] * len(ctx), ctx, None)
    g = planned(c, ctx, new, parent)
    fill_tokens(c, g, torch.Generator().manual_seed(7), kt)
    check_attend(c, g, dtype, H)
    c.h.check(stream=0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,D,new", [(4, 128, [1, 2]), (2, 64, [3, 5]), (8, 128, [2, 0])])
def test_attend_infinite_cached_values_stay_infinite(dev, dtype, H, D, new):
    """Infinity in a cached V (what an f16 cache makes of a value past its range) in tiles of 8 rows: that infinity in its
    dim, all else as without it. Scores are small, so that no weight is lost."""
    tt, code, kt, kcode = TYPES[dtype]
    ctx = [600, 90]
    c = Cache(dev, rows=2, blocks=50, G=2, D=D, kt=kt, code=kcode, fill=0)
    c.k.normal_(generator=torch.Generator("cuda").manual_seed(1))
    c.v.normal_(generator=torch.Generator("cuda").manual_seed(2))
    planned(c, [0, 0], ctx, None)
    g = planned(c, ctx, new)
    for i, x, dim, what in ((0, 5, 3, math.inf), (0, 130, 7, -math.inf), (0, 300, 40, math.inf), (1, 0, 1, math.inf)):
        c.v[0][c.t.table[i][x // 16], :, x % 16, dim] = what
    T = sum(new)
    q = (torch.randn(T, H, D, generator=torch.Generator().manual_seed(3))).to(tt)
    qd, out = q.cuda(), torch.zeros(T, H, D, dtype=tt, device="cuda")
    c.h.attend(g.c, 0, engine.AttendArgs(q=qd.data_ptr(), out=out.data_ptr(), dtype=code, n_head=H, scale=D ** -0.5), stream=0)
    c.h.check(stream=0)
    want, _ = op.attend(c.t, g.s, q.double(), c.k[0].cpu().double(), c.v[0].cpu().double(), D ** -0.5)
    got = out.cpu().double()
    assert want.isinf().any() and torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])
    assert not got.isnan().any() and (got - want)[want.isfinite()].abs().max() < 4 * U[dtype] + 2.0 ** -14
