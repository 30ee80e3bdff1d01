"""The paged KV cache's operators (navi_pages_plan / store / attend / commit) on the GPU against
the plain 64-bit restatement of oracle/pages.py, through the engine's Python classes.

Whole numbers are compared exactly. For the attention the tolerance follows from the arithmetic:
a score is off by at most ds = 2^-20 scale sum|q||k| (two f16 terms of q, f32 sums), a weight by
2 ds + 2^-20 relative (and, for 16-bit rows, by its one rounding, 2^-11 or 2^-8), the f32 sums by
2^-24 a key, all against the largest |v|; the result is then rounded to its type."""
import math
import random

import pytest
import torch

from navi_b200 import capi, engine
from oracle import pages as op

pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, capi.NAVI_F32, torch.float16, capi.NAVI_F16), "f16": (torch.float16, capi.NAVI_F16, torch.float16, capi.NAVI_F16),
         "bf16": (torch.bfloat16, capi.NAVI_BF16, torch.bfloat16, capi.NAVI_BF16)}
U = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32).cuda()


class Cache:
    """A cache over torch tensors and its oracle twin; every pool value that no test writes is NaN."""

    def __init__(self, dev, rows=4, blocks=8, page=16, n_pages=None, G=2, D=128, kt=torch.float16, code=capi.NAVI_F16, L=1, seed=0, fill=math.nan):
        n_pages = n_pages or rows * blocks
        self.page, self.G, self.D, self.L = page, G, D, L
        self.t = op.Tables.fresh(n_pages, page, rows, blocks)
        random.Random(seed).shuffle(self.t.free)
        self.k = torch.full((L, n_pages, G, page, D), fill, dtype=kt, device="cuda")
        self.v = torch.full((L, n_pages, G, page, D), fill, dtype=kt, device="cuda")
        self.table = i32(sum(self.t.table, [])).view(rows, blocks)
        self.held, self.free, self.n_free = i32(self.t.held), i32(self.t.free), i32([n_pages])
        self.h = engine.PagedKv.wrap(dev, [x.data_ptr() for x in self.k], [x.data_ptr() for x in self.v], n_pages, page, G, D, code, rows, blocks,
                                     self.table.data_ptr(), self.held.data_ptr(), self.free.data_ptr(), self.n_free.data_ptr())

    def check(self):
        torch.cuda.synchronize()
        assert self.held.tolist() == self.t.held
        assert self.n_free.item() == self.t.n_free
        assert self.free.tolist()[:self.t.n_free] == self.t.free[:self.t.n_free]
        for row, held, want in zip(self.table.tolist(), self.t.held, self.t.table):
            assert row[:held] == want[:held]


class GpuStep:
    def __init__(self, s: op.Step, rows=None, words=None):
        B = len(s.ctx)
        self.s = s
        self.rows = sum(max(n, 0) for n in s.new) if s.max_rows is None else s.max_rows
        most = max(s.new, default=0) if s.max_new is None else s.max_new
        self.words = (max(1, -(-most // 64)) if words is None else words) if s.parent is not None else 0
        self.ctx, self.new = i32(s.ctx), i32(s.new)
        self.parent = i32(s.parent) if s.parent is not None else None
        self.req = i32(s.req) if s.req is not None else None
        T = max(self.rows, 1)
        self.cu, self.status = i32([-7] * (B + 1)), i32([-7] * B)
        self.row_req, self.pos = i32([-7] * T), i32([-7] * T)
        self.slot = torch.full((T,), -7, dtype=torch.int64, device="cuda")
        self.mask = torch.full((T, max(self.words, 1)), -7, dtype=torch.int64, device="cuda")
        p = lambda x: x.data_ptr() if x is not None else 0  # noqa: E731
        self.c = engine.TreeStep(n_req=B, max_rows=self.rows, max_new=most, ctx_len=p(self.ctx), n_new=p(self.new), parent=p(self.parent),
                                 req=p(self.req), cu_rows=p(self.cu), row_req=p(self.row_req), pos=p(self.pos), slot=p(self.slot),
                                 mask=p(self.mask) if self.words else 0, mask_words=self.words, status=p(self.status))

    def check(self):
        torch.cuda.synchronize()
        s = self.s
        n = s.cu[-1]
        assert self.cu.tolist() == s.cu
        assert self.status.tolist() == s.status
        assert self.row_req.tolist()[:n] == s.row_req
        assert self.slot.tolist()[:n] == s.slot
        ok = [r for r in range(n) if s.slot[r] >= 0]
        pos = self.pos.tolist()
        assert [pos[r] for r in ok] == [s.pos[r] for r in ok]
        if s.parent is not None:
            m = self.mask.tolist()
            got = [{64 * w + b for w in range(self.words) for b in range(64) if m[r][w] >> b & 1} for r in range(n)]
            assert [got[r] for r in ok] == [s.anc[r] for r in ok]
        for x in (self.row_req, self.pos, self.slot):       # rows past the step's are left alone
            assert (x[n:] == -7).all()


def tree(rng, n, bushy=4):
    return [max(j - 1 - rng.randrange(bushy), -1) for j in range(n)]


def planned(c: Cache, ctx, new, parent="tree", seed=1, stream=0, **kw):
    rng = random.Random(seed)
    par = None if parent is None else sum((tree(rng, max(n, 0)) for n in new), []) if parent == "tree" else parent
    s = op.Step(list(ctx), list(new), par, **kw)
    g = GpuStep(s)
    c.h.plan(g.c, stream=stream)
    op.plan(c.t, s)
    g.check()
    c.check()
    return g


# ---- plan ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("parent", ["tree", None])
@pytest.mark.parametrize("ctx,new", [([0], [1]), ([15, 16, 17, 0], [1, 1, 1, 0]), ([0, 0, 3, 40], [17, 0, 64, 33]),
                                     ([100] * 7, [65, 1, 2, 128, 256, 0, 3]), ([5], [0]), ([0, 0], [0, 0])])
def test_plan_rows(dev, page, parent, ctx, new):
    c = Cache(dev, rows=len(ctx), blocks=-(-512 // page), page=page)
    planned(c, [0] * len(ctx), ctx, parent=None)             # the cached tokens' pages
    planned(c, ctx, new, parent)


def test_plan_grow_undo_release(dev):
    """A step that is undone leaves the stack as it was; a length of zero frees a request."""
    c = Cache(dev, rows=5, blocks=20, seed=3)
    planned(c, [0] * 5, [33, 0, 16, 100, 1], None)
    before = c.free.tolist()[:c.n_free.item()]
    planned(c, [33, 0, 16, 100, 1], [60, 64, 1, 0, 31])
    planned(c, [33, 0, 16, 100, 1], [0] * 5)
    assert c.free.tolist()[:c.n_free.item()] == before
    planned(c, [0] * 5, [0, 7, 0, 0, 40])                    # frees and takes in one call
    planned(c, [0] * 5, [0] * 5)
    assert c.n_free.item() == 100


@pytest.mark.parametrize("n_pages", [1, 4, 5, 6, 9])
def test_plan_too_few_pages(dev, n_pages):
    """First come, first served: a request that does not fit waits, and later ones that need pages."""
    c = Cache(dev, rows=5, blocks=8, n_pages=n_pages)
    g = planned(c, [0, 0, 0, 0, 0], [20, 40, 16, 1, 0])
    assert capi.NAVI_E_KV_FULL in g.status.tolist() or n_pages >= 8
    planned(c, [0, 0, 0, 0, 0], [0, 40, 0, 64, 17])          # pages given back serve the others in the same call


def test_plan_table_rows(dev):
    """A batch in another order than the table's rows, some of them absent."""
    c = Cache(dev, rows=9, blocks=8)
    planned(c, [0, 0, 0], [20, 60, 5], None, req=[7, 2, 4])
    planned(c, [5, 60, 20], [9, 30, 40], "tree", req=[4, 2, 7])
    planned(c, [0, 0], [0, 10], None, req=[2, 0])


def test_plan_refusals_on_the_device(dev):
    c = Cache(dev, rows=6, blocks=4)
    g = planned(c, [0, -1, 3, 60, 0, 0], [5, 2, -2, 9, 1, 4], "tree", req=[0, 1, 2, 3, 6, 5])
    assert g.status.tolist() == [0, capi.NAVI_E_ARG, capi.NAVI_E_ARG, capi.NAVI_E_SHAPE, capi.NAVI_E_ARG, 0]
    g = planned(c, [5, 0], [3, 6], "tree", max_new=4)        # above max_new
    assert g.status.tolist() == [0, capi.NAVI_E_SHAPE]
    g = planned(c, [5, 0, 0], [3, 4, 2], "tree", max_rows=6, max_new=4)      # rows past max_rows
    assert g.status.tolist() == [0, capi.NAVI_E_SHAPE, capi.NAVI_E_SHAPE]


@pytest.mark.parametrize("bad", [[-1, 1, 0], [-1, 0, 2], [0, 0, 1], [-1, -2, 1], [-1, 5, 1], [-1, 0, -2147483648]])
def test_plan_bad_parent(dev, bad):
    """A parent that is not below its row: the request is refused, its good rows and its neighbours stay."""
    c = Cache(dev, rows=3, blocks=4)
    g = planned(c, [4, 9, 1], [2, 3, 3], [-1, 0] + bad + [-1, 0, 1])
    assert g.status.tolist() == [0, capi.NAVI_E_ARG, 0]
    g = planned(c, [4, 9, 1], [2, 3, 3], [-1, 0] + [-1, 0, 1] + [-1, 0, 1])  # nothing of it is left for the next call
    assert g.status.tolist() == [0, 0, 0]


@pytest.mark.parametrize("B", [257, 1000, 8192])
def test_plan_many_requests(dev, B):
    rng = random.Random(B)
    c = Cache(dev, rows=B, blocks=6, n_pages=3 * B, D=64, G=1)
    ctx = [rng.randrange(40) for _ in range(B)]
    planned(c, [0] * B, ctx, None)
    planned(c, ctx, [rng.choice([0, 1, 1, 2, 9, 30]) for _ in range(B)], "tree")
    planned(c, ctx, [0] * B, None)
    planned(c, [0 if rng.random() < 0.5 else x for x in ctx], [rng.randrange(20) for _ in range(B)], "tree")


def test_plan_is_the_same_every_time(dev):
    outs = []
    for _ in range(3):
        c = Cache(dev, rows=300, blocks=4, D=64, G=1, seed=5)
        g = planned(c, [0] * 300, [x % 41 for x in range(300)])
        outs.append((g.slot.tolist(), c.table.tolist(), c.free.tolist()))
    assert outs[0] == outs[1] == outs[2]


# ---- store ---------------------------------------------------------------------------------------

def rope_table(n, D):
    ang = torch.arange(n).double()[:, None] * 1e6 ** (-torch.arange(0, D, 2).double() / D)
    return torch.cat([ang.cos(), ang.sin()], 1).float()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,G,D", [(4, 2, 128), (16, 8, 128), (3, 1, 64), (5, 5, 64), (0, 3, 128), (7, 7, 128)])
@pytest.mark.parametrize("norm,rope", [(True, True), (False, True), (True, False), (False, False)])
def test_store(dev, dtype, H, G, D, norm, rope):
    tt, code, kt, kcode = TYPES[dtype]
    c = Cache(dev, rows=3, blocks=10, page=16, G=G, D=D, kt=kt, code=kcode, L=2)
    planned(c, [0, 0, 0], [14, 0, 5], None)
    g = planned(c, [14, 0, 5], [9, 1, 20])
    T = g.rows
    gen = torch.Generator().manual_seed(T + H)
    qkv = torch.randn(T, (H + 2 * G) * D, generator=gen).to(tt)
    qn, kn, tab = torch.rand(D, generator=gen) + 0.5, torch.rand(D, generator=gen) + 0.5, rope_table(64, D)
    # rows with room between them, and a result of another stride
    wide = torch.full((T, (H + 2 * G) * D + 16), 9.0, dtype=tt, device="cuda")
    wide[:, :qkv.shape[1]] = qkv.cuda()
    q = torch.full((T, max(H * D, 8) + 8), 7.0, dtype=tt, device="cuda")
    qn_d, kn_d, tab_d = qn.cuda(), kn.cuda(), tab.cuda()
    a = engine.StoreArgs(qkv=wide.data_ptr(), qkv_stride=wide.shape[1], q_out=q.data_ptr() if H else 0, q_out_stride=q.shape[1], dtype=code, n_head=H,
                         q_norm=qn_d.data_ptr() if norm else 0, k_norm=kn_d.data_ptr() if norm else 0, eps=1e-6,
                         rope=tab_d.data_ptr() if rope else 0, rope_positions=64 if rope else 0)
    kw, vw = c.k[1].cpu().double(), c.v[1].cpu().double()
    c.h.store(g.c, 1, a, stream=0)
    torch.cuda.synchronize()
    want = op.store(16, g.s, qkv, H, G, kw, vw, qn if norm else None, kn if norm else None, 1e-6, tab if rope else None)
    # f32 arithmetic: a few units in the last place of the row's largest value; then one rounding
    def near(got, want, u):
        assert torch.equal(got.isnan(), want.isnan())
        got, want = got.nan_to_num(7.0), want.nan_to_num(7.0)
        assert ((got - want).abs() <= u * want.abs() + 2.0 ** -20 * want.abs().max() + 2.0 ** -25).all()

    if H:
        near(q[:, :H * D].cpu().double().reshape(T, H, D), want, U[dtype])
    assert (q[:, H * D:] == 7).all()
    near(c.k[1].cpu().double(), kw, U["bf16" if kt == torch.bfloat16 else "f16"])
    near(c.v[1].cpu().double(), vw, U["bf16" if kt == torch.bfloat16 else "f16"])
    assert c.k[0].isnan().all() and c.v[0].isnan().all()     # the other layer is left alone


def test_store_in_place_refused_and_outside_the_table(dev):
    """q over its own rows; rows of a refused request and of a position past the table are not stored."""
    c = Cache(dev, rows=2, blocks=2)
    g = planned(c, [0, 0], [20, 33], "tree")                 # the second does not fit the block table
    assert g.status.tolist() == [0, capi.NAVI_E_SHAPE]
    T, H, G, D = g.rows, 2, 2, 128
    qkv = torch.randn(T, (H + 2 * G) * D, generator=torch.Generator().manual_seed(0))
    d, tab = qkv.cuda(), rope_table(3, D)
    tab_d = tab.cuda()
    kw, vw = c.k[0].cpu().double(), c.v[0].cpu().double()
    want = op.store(16, g.s, qkv, H, G, kw, vw, rope=tab)
    a = engine.StoreArgs(qkv=d.data_ptr(), q_out=d.data_ptr(), q_out_stride=d.shape[1], dtype=capi.NAVI_F32, n_head=H, rope=tab_d.data_ptr(),
                         rope_positions=3)
    c.h.store(g.c, 0, a, stream=0)
    torch.cuda.synchronize()
    inside = [r for r in range(20) if g.s.pos[r] < 3]
    assert 0 < len(inside) < 20
    got = d.cpu()[:, :H * D].reshape(T, H, D).double()
    assert (got[:20] - want[:20]).abs().max() < 1e-5
    outside = [r for r in range(20) if g.s.pos[r] >= 3]
    assert (got[outside] == 0).all()
    assert torch.equal(c.k[0].cpu().isnan(), kw.isnan()) and torch.equal(c.v[0].cpu().isnan(), vw.isnan())
    assert torch.equal(d.cpu()[:, H * D:], qkv[:, H * D:])


# ---- attend --------------------------------------------------------------------------------------

def fill_tokens(c: Cache, g: GpuStep, gen, kt):
    """Random K and V for the tokens that the step's requests own; all else stays NaN."""
    s = g.s
    req = s.req if s.req is not None else range(len(s.ctx))
    for i, tr in enumerate(req):
        if s.status[i]:
            continue
        for x in range(s.ctx[i] + s.new[i]):
            p, o = c.t.table[tr][x // c.page], x % c.page
            c.k[0][p, :, o] = torch.randn(c.G, c.D, generator=gen).to(kt).cuda()
            c.v[0][p, :, o] = torch.randn(c.G, c.D, generator=gen).to(kt).cuda()


def check_attend(c, g, dtype, H, seed=0, qscale=1.0, stream=0, pad=0, want_lse=True):
    tt, code, kt, _ = TYPES[dtype]
    T, D, s = g.s.cu[-1], c.D, g.s
    gen = torch.Generator().manual_seed(seed)
    q = (torch.randn(max(g.rows, 1), H * D, generator=gen) * qscale).to(tt)
    qd = torch.full((q.shape[0], H * D + pad), math.nan, dtype=tt, device="cuda")
    qd[:, :H * D] = q.cuda()
    out = torch.full((q.shape[0], H * D + 2 * pad), 9.0, dtype=tt, device="cuda")
    lse = torch.full((q.shape[0], H), 9.0, device="cuda")
    scale = D ** -0.5
    a = engine.AttendArgs(q=qd.data_ptr(), q_stride=qd.shape[1], out=out.data_ptr(), out_stride=out.shape[1],
                          lse=lse.data_ptr() if want_lse else 0, dtype=code, n_head=H, scale=scale)
    c.h.attend(g.c, 0, a, stream=stream)
    torch.cuda.synchronize()
    kd, vd = c.k[0].cpu().double(), c.v[0].cpu().double()
    want, wl = op.attend(c.t, s, q[:T].double().reshape(T, H, D), kd, vd, scale)
    got = out.cpu()[:T, :H * D].double().reshape(T, H, D)
    kmax, vmax = kd.nan_to_num(0).abs().max(), vd.nan_to_num(0).abs().max()
    L = max(x + n for x, n in zip(s.ctx, s.new))
    ds = 2.0 ** -20 * scale * float(q.double().abs().reshape(-1, H, D).sum(2).max()) * float(kmax)
    tol = float(vmax) * (2 * ds + 2.0 ** -20 + L * 2.0 ** -24 + (0 if dtype == "f32" else U[dtype]))
    assert ((got - want).abs() <= tol + U[dtype] * want.abs()).all(), ((got - want).abs().max(), tol)
    assert (out[:T, H * D:] == 9).all() and (out[T:] == 9).all()
    if want_lse:
        gl = lse.cpu()[:T].double()
        assert torch.equal(gl.isinf(), wl.isinf())
        assert ((gl - wl).nan_to_num(0).abs() <= ds + 2.0 ** -20 + L * 2.0 ** -24 + 2.0 ** -22 * wl.nan_to_num(0, neginf=0).abs()).all()
        assert (lse[T:] == 9).all()
    return out, lse


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,G,D", [(4, 2, 128), (2, 2, 64), (8, 1, 128), (3, 1, 64), (12, 1, 128)])
@pytest.mark.parametrize("page,ctx,new", [(16, [0, 1, 15, 16, 17], [1, 1, 1, 1, 1]), (16, [63, 64, 65, 0, 127], [5, 0, 1, 3, 17]),
                                          (32, [130, 7], [33, 66]), (128, [300, 0], [2, 64])])
def test_attend_trees(dev, dtype, H, G, D, page, ctx, new):
    tt, _, kt, kcode = TYPES[dtype]
    c = Cache(dev, rows=len(ctx), blocks=-(-400 // page), page=page, G=G, D=D, kt=kt, code=kcode)
    planned(c, [0] * len(ctx), ctx, None)
    g = planned(c, ctx, new)
    fill_tokens(c, g, torch.Generator().manual_seed(7), kt)
    check_attend(c, g, dtype, H)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [63, 64, 65, 129, 200, 256])
def test_attend_large_trees(dev, dtype, n):
    tt, _, kt, kcode = TYPES[dtype]
    c = Cache(dev, rows=2, blocks=40, G=1, kt=kt, code=kcode)
    planned(c, [0, 0], [70, 31], None)
    g = planned(c, [70, 31], [n, 3])
    fill_tokens(c, g, torch.Generator().manual_seed(n), kt)
    check_attend(c, g, dtype, 2)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,G,D", [(4, 2, 128), (2, 2, 64)])
@pytest.mark.parametrize("ctx,new", [([0], [1]), ([0, 5], [130, 1]), ([100, 0, 64], [65, 129, 0]), ([0], [300])])
def test_attend_chains(dev, dtype, H, G, D, ctx, new):
    tt, _, kt, kcode = TYPES[dtype]
    c = Cache(dev, rows=len(ctx), blocks=24, G=G, D=D, kt=kt, code=kcode)
    planned(c, [0] * len(ctx), ctx, None)
    g = planned(c, ctx, new, None)
    fill_tokens(c, g, torch.Generator().manual_seed(3), kt)
    check_attend(c, g, dtype, H)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ctx", [[1500, 3, 700], [4095], [2049, 0]])
def test_attend_long(dev, dtype, ctx):
    """Lengths whose keys several blocks share out."""
    tt, _, kt, kcode = TYPES[dtype]
    c = Cache(dev, rows=len(ctx), blocks=260, G=2, kt=kt, code=kcode, fill=0)
    c.k.normal_(generator=torch.Generator("cuda").manual_seed(1))
    c.v.normal_(generator=torch.Generator("cuda").manual_seed(2))
    planned(c, [0] * len(ctx), ctx, None)
    g = planned(c, ctx, [5, 1, 33][:len(ctx)])
    a = check_attend(c, g, dtype, 4, qscale=3.0)
    b = check_attend(c, g, dtype, 4, qscale=3.0)             # the same bits again
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [8, 9, 16, 17])
@pytest.mark.parametrize("B", [70, 74, 80])
def test_attend_small_trees_of_many_requests(dev, dtype, rows, B):
    """16 to 34 rows x heads, on both sides of as many items as a B200 has multiprocessors (148 = 74 x 2)."""
    tt, _, kt, kcode = TYPES[dtype]
    ctx, new = [(37 * r) % 210 for r in range(B)], [rows - (r * 5) % (rows + 1) for r in range(B)]
    c = Cache(dev, rows=B, blocks=16, G=2, kt=kt, code=kcode)
    planned(c, [0] * B, ctx, None)
    g = planned(c, ctx, new)
    fill_tokens(c, g, torch.Generator().manual_seed(B), kt)
    check_attend(c, g, dtype, 4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_rows_that_see_nothing(dev, dtype):
    """A mask without a bit and no cached token; refused requests; a token's scores of -inf."""
    tt, _, kt, kcode = TYPES[dtype]
    c = Cache(dev, rows=4, blocks=2, kt=kt, code=kcode)
    g = planned(c, [0, 0, 0, 20], [3, 40, 2, 1])
    assert g.status.tolist()[1] == capi.NAVI_E_SHAPE
    fill_tokens(c, g, torch.Generator().manual_seed(5), kt)
    g.mask[1] = 0                                            # the second row of the first request
    g.s.anc[1] = set()
    out, lse = check_attend(c, g, dtype, 4)
    assert (out[1] == 0).all() and (lse[1] == -math.inf).all()
    assert (out[3:43] == 0).all() and (lse[3:43] == -math.inf).all()


def test_attend_large_and_infinite_scores(dev):
    """Scores far from zero, and a key whose score is -inf for every row."""
    c = Cache(dev, rows=1, blocks=4, G=1)
    planned(c, [0], [30], None)
    g = planned(c, [30], [4])
    fill_tokens(c, g, torch.Generator().manual_seed(5), torch.float16)
    c.k[0] *= 30
    check_attend(c, g, "f16", 2, qscale=20.0)
    p, o = c.t.table[0][0], 3
    c.k[0][p, 0, o] = 0
    c.k[0][p, 0, o, 0] = -math.inf
    T, H, D = 4, 2, 128
    q = torch.randn(T, H * D, generator=torch.Generator().manual_seed(1)).half().cuda()
    q.view(T, H, D)[:, :, 0] = 1
    out = torch.zeros_like(q)
    c.h.attend(g.c, 0, engine.AttendArgs(q=q.data_ptr(), out=out.data_ptr(), dtype=capi.NAVI_F16, n_head=H, scale=0.1), stream=0)
    torch.cuda.synchronize()
    kd = c.k[0].cpu().double()
    kd[p, 0, o, 0] = -1e300
    want, _ = op.attend(c.t, g.s, q.cpu().double().view(T, H, D), kd, c.v[0].cpu().double(), 0.1)
    assert (out.cpu().double().view(T, H, D) - want).abs().max() < 2.0 ** -8 * c.v[0].nan_to_num(0).abs().max()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,G,D", [(4, 2, 128), (2, 2, 64)])
@pytest.mark.parametrize("parent", ["tree", None])
@pytest.mark.parametrize("ctx,new", [([20, 0], [5, 3]), ([37, 130], [14, 9]), ([100, 3], [33, 64]), ([5, 250], [150, 40])])
def test_attend_values_that_are_not_finite_stay_with_those_who_look(dev, dtype, H, G, D, parent, ctx, new):
    """K and V of a new row that hold NaN or infinity: only rows that see it (its descendants, the later
    rows of a chain) are affected, in the dims that they concern; its siblings' results are as without it."""
    tt, _, kt, kcode = TYPES[dtype]
    c = Cache(dev, rows=2, blocks=20, G=G, D=D, kt=kt, code=kcode)
    planned(c, [0, 0], ctx, None)
    g = planned(c, ctx, new, parent)
    fill_tokens(c, g, torch.Generator().manual_seed(4), kt)
    for i, j, pool, dims, what in ((0, 2, "v", slice(None), math.nan), (1, 1, "v", slice(3, 7), math.inf), (0, new[0] - 1, "v", slice(0, 1), -math.inf),
                                   (1, new[1] - 1, "k", slice(None), math.nan)):
        slot = g.s.slot[g.s.cu[i] + j]
        getattr(c, pool)[0][slot // 16, 0, slot % 16, dims] = what
    gen = torch.Generator().manual_seed(1)
    T = g.rows
    q = torch.randn(T, H * D, generator=gen).to(tt)
    qd, out = q.cuda(), torch.zeros(T, H * D, dtype=tt, device="cuda")
    a = engine.AttendArgs(q=qd.data_ptr(), out=out.data_ptr(), dtype=TYPES[dtype][1], n_head=H, scale=D ** -0.5)
    c.h.attend(g.c, 0, a, stream=0)
    torch.cuda.synchronize()
    want, _ = op.attend(c.t, g.s, q.double().reshape(T, H, D), c.k[0].cpu().double(), c.v[0].cpu().double(), D ** -0.5)
    got = out.cpu().double().reshape(T, H, D)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[got.isinf()], want[want.isinf()])
    fine = want.isfinite()
    assert fine.any() and not fine.all()
    # the scores of standard normal values are below 8; the tolerance of the finite ones as in check_attend
    vmax, L = 6.0, max(x + n for x, n in zip(ctx, new))
    tol = vmax * (2.0 ** -19 * 8 * 12 + 2.0 ** -20 + L * 2.0 ** -24 + (0 if dtype == "f32" else U[dtype]))
    assert ((got - want)[fine].abs() <= tol + U[dtype] * want[fine].abs()).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_attend_strides_table_rows_and_no_lse(dev, dtype):
    c = Cache(dev, rows=6, blocks=8)
    planned(c, [0, 0, 0], [33, 70, 2], None, req=[5, 0, 3])
    g = planned(c, [2, 33, 70], [7, 1, 20], req=[3, 5, 0])
    fill_tokens(c, g, torch.Generator().manual_seed(9), torch.float16)
    check_attend(c, g, dtype, 4, pad=8)
    check_attend(c, g, dtype, 4, pad=16, want_lse=False)


def test_attend_room_for_more_rows(dev):
    """max_rows and max_new above what the step has: what lies past its rows is left alone."""
    c = Cache(dev, rows=2, blocks=8)
    planned(c, [0, 0], [33, 70], None)
    rng = random.Random(2)
    g = planned(c, [33, 70], [3, 5], tree(rng, 3) + tree(rng, 5) + [0] * 12, max_rows=20, max_new=64)
    fill_tokens(c, g, torch.Generator().manual_seed(9), torch.float16)
    check_attend(c, g, "f32", 4)


def test_attend_on_other_streams(dev):
    """Two streams at once, each with its own step and cache: each has its own scratch."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.ExternalStream(dev.stream)]
    for _ in range(3):
        for k, st in enumerate(streams):
            c = Cache(dev, rows=3, blocks=64, seed=k)
            planned(c, [0] * 3, [900, 500 + k, 20], None)
            g = planned(c, [900, 500 + k, 20], [9, 1, 4])
            fill_tokens(c, g, torch.Generator().manual_seed(k), torch.float16)
            torch.cuda.synchronize()
            check_attend(c, g, "f16", 4, seed=k, stream=st.cuda_stream)


def test_attend_offsets_past_32_bits(dev):
    """Pages whose byte and element offsets pass 2^32: the last pages of a pool of over 8 GB."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB free")
    G, D, page, blocks = 8, 128, 16, 8
    n_pages = (1 << 32) // (G * D * page) + 300            # > 2^32 elements
    c = Cache(dev, rows=2, blocks=blocks, page=page, n_pages=n_pages, G=G, D=D, fill=0)
    c.t.free.sort()                                         # the highest page on top
    c.free.copy_(i32(c.t.free))
    planned(c, [0, 0], [100, 17], None)
    g = planned(c, [100, 17], [6, 4])
    assert min(x for x in g.s.slot) * G * D > 1 << 32
    fill_tokens(c, g, torch.Generator().manual_seed(9), torch.float16)
    kd, vd = c.k, c.v
    # the oracle sees the pages in use alone
    used = sorted({p for row, h in zip(c.t.table, c.t.held) for p in row[:h]})
    small = {p: n for n, p in enumerate(used)}
    q = torch.randn(10, 16 * D, generator=torch.Generator().manual_seed(1))
    out = torch.zeros(10, 16 * D, device="cuda")
    qd = q.cuda()
    c.h.attend(g.c, 0, engine.AttendArgs(q=qd.data_ptr(), out=out.data_ptr(), dtype=capi.NAVI_F32, n_head=16, scale=0.1), stream=0)
    torch.cuda.synchronize()
    t = op.Tables(page, blocks, [[small.get(p, 0) for p in row] for row in c.t.table], c.t.held, [], 0, len(used))
    want, _ = op.attend(t, g.s, q.double().view(10, 16, D), kd[0][used].cpu().double(), vd[0][used].cpu().double(), 0.1)
    assert (out.cpu().double().view(10, 16, D) - want).abs().max() < 1e-4


# ---- commit --------------------------------------------------------------------------------------

def drafts(rng, s: op.Step, width, hit=0.8, vocab=50):
    T = s.cu[-1]
    tok = [[rng.randrange(vocab) for _ in range(width)] for _ in range(T)]
    tgt = [[rng.randrange(vocab) for _ in range(width)] for _ in range(T)]
    root = [[rng.randrange(vocab) for _ in range(width)] for _ in s.ctx]
    for i in range(len(s.ctx)):
        for j in [-1] + list(range(s.cu[i + 1] - s.cu[i])):
            kids = [k for k in range(s.cu[i + 1] - s.cu[i]) if s.parent[s.cu[i] + k] == j]
            if kids and rng.random() < hit:
                k = rng.choice(kids)
                if j < 0:
                    root[i] = list(tok[s.cu[i] + k])
                else:
                    tgt[s.cu[i] + j] = list(tok[s.cu[i] + k])
    return tok, tgt, root


@pytest.mark.parametrize("width", [1, 3, 16])
@pytest.mark.parametrize("page,G,D,L,ctx,new", [(16, 2, 128, 3, [0, 14, 5, 9], [1, 16, 0, 40]), (32, 3, 64, 1, [33], [64]),
                                                (16, 8, 128, 28, [7, 60], [16, 9]), (64, 1, 64, 2, [0, 100, 3], [256, 70, 2])])
def test_commit(dev, width, page, G, D, L, ctx, new):
    rng = random.Random(width + L)
    c = Cache(dev, rows=len(ctx), blocks=-(-400 // page), page=page, G=G, D=D, L=L, fill=0)
    c.k.normal_(generator=torch.Generator("cuda").manual_seed(1))
    c.v.normal_(generator=torch.Generator("cuda").manual_seed(2))
    planned(c, [0] * len(ctx), ctx, None)
    g = planned(c, ctx, new)
    total = 0
    for hit in (0.0, 0.9, 1.0):
        tok, tgt, root = drafts(rng, g.s, width, hit, vocab=3 if width == 1 else 50)     # twins among the siblings at width 1
        T, B = max(g.s.cu[-1], 1), len(ctx)
        dt, dg, dr = i32(sum(tok, [])), i32(sum(tgt, [])), i32(sum(root, []))
        acc, path, nl, nx = i32([-7] * B), i32([-7] * T), i32([-7] * B), i32([-7] * B * width)
        kw, vw = c.k.cpu().clone(), c.v.cpu().clone()
        c.h.commit(g.c, engine.CommitArgs(width=width, tokens=dt.data_ptr(), targets=dg.data_ptr(), root_target=dr.data_ptr(), accepted=acc.data_ptr(),
                                          path=path.data_ptr(), new_len=nl.data_ptr(), next_token=nx.data_ptr()), stream=0)
        torch.cuda.synchronize()
        paths, nxt = op.commit(page, g.s, tok, tgt, root, [x for l in range(L) for x in (kw[l], vw[l])])
        assert acc.tolist() == [len(p) for p in paths]
        assert nl.tolist() == [x + len(p) for x, p in zip(ctx, paths)]
        assert nx.view(B, width).tolist() == nxt
        assert path.tolist()[:g.s.cu[-1]] == sum((p + [-1] * (g.s.new[i] - len(p)) for i, p in enumerate(paths)), [])
        assert torch.equal(c.k.cpu(), kw) and torch.equal(c.v.cpu(), vw)
        total += sum(len(p) for p in paths)
    assert total > 0


def test_commit_refused_request(dev):
    c = Cache(dev, rows=2, blocks=2)
    g = planned(c, [3, 0], [2, 40], [-1, 0] + [x - 1 for x in range(40)])
    T = 42
    ids = i32([4] * T)
    root, acc, path, nl, nx = i32([4, 4]), i32([-7] * 2), i32([-7] * T), i32([-7] * 2), i32([-7] * 2)
    before = c.k.clone()
    c.h.commit(g.c, engine.CommitArgs(width=1, tokens=ids.data_ptr(), targets=ids.data_ptr(), root_target=root.data_ptr(), accepted=acc.data_ptr(),
                                      path=path.data_ptr(), new_len=nl.data_ptr(), next_token=nx.data_ptr()), stream=0)
    torch.cuda.synchronize()
    assert acc.tolist() == [2, 0] and nl.tolist() == [5, 0] and nx.tolist() == [4, 4]
    assert path.tolist() == [0, 1] + [-1] * 40
    assert torch.equal(c.k.isnan(), before.isnan())


# ---- refusals --------------------------------------------------------------------------------------

def refused(status, fn, *a, **kw):
    with pytest.raises(capi.NaviError) as e:
        fn(*a, **kw)
    assert e.value.status == status and len(str(e.value)) > 12


@pytest.mark.parametrize("kw,status", [(dict(page_size=24), capi.NAVI_E_ARG), (dict(page_size=256), capi.NAVI_E_ARG), (dict(head_dim=96), capi.NAVI_E_SHAPE),
                                       (dict(dtype=capi.NAVI_F32), capi.NAVI_E_ARG), (dict(n_layer=0), capi.NAVI_E_ARG), (dict(n_layer=129), capi.NAVI_E_ARG),
                                       (dict(n_pages=0), capi.NAVI_E_ARG), (dict(n_kv_head=0), capi.NAVI_E_ARG), (dict(max_requests=8193), capi.NAVI_E_ARG),
                                       (dict(max_requests=0), capi.NAVI_E_ARG), (dict(max_blocks=0), capi.NAVI_E_ARG),
                                       (dict(n_pages=1 << 26, page_size=16), capi.NAVI_E_SHAPE)])
def test_create_refusals(dev, kw, status):
    base = dict(n_layer=1, n_pages=4, page_size=16, n_kv_head=2, head_dim=128, max_requests=2, max_blocks=2)
    refused(status, engine.PagedKv.create, dev, **{**base, **kw})


def test_create_refuses_half_given_pointers_and_odd_addresses(dev):
    x = torch.zeros(1 << 16, dtype=torch.float16, device="cuda")
    t = i32([0] * 64)
    p, q = x.data_ptr(), t.data_ptr()
    kw = dict(n_pages=4, page_size=16, n_kv_head=2, head_dim=128, dtype=capi.NAVI_F16, max_requests=2, max_blocks=2)
    refused(capi.NAVI_E_ARG, engine.PagedKv.wrap, dev, [p], [p], table=q, held=0, free_pages=q, n_free=q, **kw)
    refused(capi.NAVI_E_ARG, engine.PagedKv.wrap, dev, [p + 2], [p], table=q, held=q, free_pages=q, n_free=q, **kw)


def test_call_refusals(dev):
    c = Cache(dev, rows=2, blocks=4)
    g = planned(c, [3, 0], [2, 4])
    x = torch.zeros(1 << 14, device="cuda")
    p = x.data_ptr()

    def step(**kw):
        f = {n: getattr(g.c.s, n) for n, _ in capi.Step._fields_}
        return engine.TreeStep(**{**f, **kw})

    E = capi.NAVI_E_ARG
    for kw in (dict(n_req=3), dict(n_req=-1), dict(max_rows=-1), dict(ctx_len=0), dict(n_new=0), dict(cu_rows=0), dict(status=0), dict(slot=0), dict(pos=0),
               dict(row_req=0), dict(mask=0), dict(mask_words=0), dict(mask_words=5)):
        refused(E, c.h.plan, step(**kw), stream=0)
    refused(capi.NAVI_E_SHAPE, c.h.plan, step(max_new=257, mask_words=4), stream=0)
    c.h.plan(step(n_req=0), stream=0)                        # nothing to do

    st = dict(qkv=p, q_out=p, dtype=capi.NAVI_F32, n_head=4)
    for kw in (dict(qkv=0), dict(q_out=0), dict(qkv=p + 4), dict(q_out=p + 8), dict(qkv_stride=100), dict(q_out_stride=512 + 2), dict(dtype=capi.NAVI_BF16),
               dict(dtype=7), dict(n_head=-1), dict(rope=p, rope_positions=0)):
        refused(E, c.h.store, g.c, 0, engine.StoreArgs(**{**st, **kw}), stream=0)
    refused(E, c.h.store, g.c, 1, engine.StoreArgs(**st), stream=0)
    refused(E, c.h.store, g.c, -1, engine.StoreArgs(**st), stream=0)

    at = dict(q=p, out=p + 4096, dtype=capi.NAVI_F32, n_head=4, scale=0.1)
    for kw in (dict(q=0), dict(out=0), dict(q=p + 4), dict(out=p + 8), dict(q_stride=100), dict(out_stride=514), dict(dtype=capi.NAVI_BF16), dict(n_head=3),
               dict(n_head=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf)):
        refused(E, c.h.attend, g.c, 0, engine.AttendArgs(**{**at, **kw}), stream=0)
    refused(E, c.h.attend, g.c, 1, engine.AttendArgs(**at), stream=0)

    co = dict(width=1, tokens=p, targets=p, root_target=p, accepted=p, path=p, new_len=p, next_token=p)
    for kw in (dict(width=0), dict(tokens=0), dict(targets=0), dict(root_target=0), dict(accepted=0), dict(path=0), dict(new_len=0), dict(next_token=0)):
        refused(E, c.h.commit, g.c, engine.CommitArgs(**{**co, **kw}), stream=0)
    refused(E, c.h.commit, step(parent=0), engine.CommitArgs(**co), stream=0)
    with pytest.raises(TypeError):
        engine.AttendArgs(quey=p)


def test_own_pools_and_tables(dev):
    """A cache that the library allocates: every page free, page 0 on top, K and V zero."""
    kv = engine.PagedKv.create(dev, 2, 6, 16, 1, 64, 3, 4)
    d = kv.desc()
    assert (d.n_layer, d.n_pages, d.page_size, d.max_blocks) == (2, 6, 16, 4) and all([d.table, d.held, d.free_pages, d.n_free, d.k[1], d.v[1]])
    s = op.Step([0, 0, 0], [17, 1, 0], None)
    g = GpuStep(s)
    kv.plan(g.c)                                             # on the engine's stream
    t = op.Tables.fresh(6, 16, 3, 4)
    op.plan(t, s)
    g.check()
    assert s.slot[0] == 0 and s.slot[16] == 16
    kv.close()
