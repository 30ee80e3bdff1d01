"""Steps of many requests through the talker over a paged cache (navi_talker_step) on the GPU:
prompts admitted together, drafted trees of different requests checked in one pass over the weights,
the branch that agrees committed, decoding continued from there. Every row is compared with the CPU
oracle's prefill of that row's own history (its request's rows, then its ancestors), so the test runs
plan, store, attend and commit together as a serving loop does.

Tolerance: rel-L2 2e-4 on hidden rows and logits, the prefill test's, and for the same reason: the
same GEMMs, and a cache rounded once to f16 on both sides."""
import numpy as np
import pytest
import torch

from navi_b200 import capi, engine
from oracle import model as om

pytestmark = pytest.mark.gpu

REL = 2e-4


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


class Session:
    def __init__(self, path, n_pages=64, page=16, requests=3, blocks=16, max_prompt=256):
        self.W = om.Weights.from_navi(path)
        self.dev = engine.Device(0)
        self.w = engine.Weights(self.dev, path)
        self.tal = engine.Talker(self.dev, self.w, max_prompt_tokens=max_prompt, max_positions=512)
        t = self.W.tl
        self.pages = engine.PagedKv.create(self.dev, t.n_layer, n_pages, page, t.n_kv_head, t.head_dim, requests, blocks)
        self.H, self.V = t.hidden, t.vocab

    def step(self, rows, ctx, new, parent=None, spare=0):
        """(hidden, logits, TreeStep) of the rows [sum(new)][H]; `spare` rows of room are left over."""
        T, B = sum(new) + spare, len(ctx)
        d = torch.zeros(T, self.H, device="cuda")
        d[:sum(new)] = rows.cuda()
        hidden, logits = torch.zeros(T, self.H, device="cuda"), torch.zeros(T, self.V, device="cuda")
        keep = dict(ctx_len=i32(ctx), n_new=i32(new), cu_rows=i32([0] * (B + 1)), row_req=i32([0] * T), pos=i32([0] * T),
                    slot=torch.zeros(T, dtype=torch.int64, device="cuda"), status=i32([0] * B))
        words = 0
        if parent is not None:
            words = -(-max(new) // 64)
            keep.update(parent=i32(list(parent) + [0] * spare), mask=torch.zeros(T, words, dtype=torch.int64, device="cuda"))
        s = engine.TreeStep(n_req=B, max_rows=T, max_new=max(new), mask_words=words, keepalive=keep, **{k: v.data_ptr() for k, v in keep.items()})
        torch.cuda.synchronize()
        self.tal.step(self.pages, s, d.data_ptr(), hidden.data_ptr(), logits.data_ptr())
        assert keep["status"].tolist() == [0] * B
        return hidden.cpu(), logits.cpu(), s

    def want(self, rows):
        t = self.W.tl
        kv = [(torch.zeros(rows.shape[0], t.n_kv_head * t.head_dim), torch.zeros(rows.shape[0], t.n_kv_head * t.head_dim)) for _ in range(t.n_layer)]
        return om.prefill(self.W, rows, kv)

    def check(self, hidden, logits, rows):
        h, lg = self.want(rows)
        assert om.rel_l2(hidden.numpy(), h) < REL, om.rel_l2(hidden.numpy(), h)
        assert om.rel_l2(logits.numpy(), lg) < REL, om.rel_l2(logits.numpy(), lg)


def rows_of(n, H, seed):
    return torch.randn(n, H, generator=torch.Generator().manual_seed(seed)) * 0.5


def branch(parent, j):
    out = []
    while j >= 0:
        out.append(j)
        j = parent[j]
    return out[::-1]


@pytest.mark.parametrize("spare", [0, 5])
def test_prompts_drafts_and_what_follows(small_navi, spare):
    S = Session(small_navi)
    lens = [23, 1, 70]
    hist = [rows_of(n, S.H, 10 + i) for i, n in enumerate(lens)]
    h, lg, _ = S.step(torch.cat(hist), [0, 0, 0], lens, spare=spare)
    at = np.cumsum(lens) - 1
    for i in range(3):
        S.check(h[at[i]], lg[at[i]], hist[i])

    # drafted trees of two of the requests, the third decodes one row
    trees = [[-1, 0, 0, 1, 2, 4, -1], [-1], [-1, 0, 1, 1, 2, 2, 0, 6, 7]]
    new = [len(t) for t in trees]
    drafts = [rows_of(n, S.H, 20 + i) for i, n in enumerate(new)]
    h, lg, step = S.step(torch.cat(drafts), lens, new, sum(trees, []), spare=spare)
    first = np.cumsum([0] + new)
    for i in range(3):
        for j in range(new[i]):
            S.check(h[first[i] + j], lg[first[i] + j], torch.cat([hist[i], drafts[i][branch(trees[i], j)]]))

    # ids of the drafts and the model's choices: 0, 2, 4 of the first, its only row of the second, none of the third
    T = sum(new) + spare
    tok, tgt, root = torch.arange(T * 2).view(T, 2).int(), torch.full((T, 2), -1).int(), torch.full((3, 2), -2).int()
    root[0], tgt[0], tgt[2] = tok[0], tok[2], tok[4]
    root[1] = tok[first[1]]
    tok, tgt, root = tok.cuda(), tgt.cuda(), root.cuda()
    out = dict(accepted=i32([0] * 3), path=i32([0] * T), new_len=i32([0] * 3), next_token=i32([0] * 6))
    torch.cuda.synchronize()
    S.pages.commit(step, engine.CommitArgs(width=2, tokens=tok.data_ptr(), targets=tgt.data_ptr(), root_target=root.data_ptr(),
                                           **{k: v.data_ptr() for k, v in out.items()}))
    S.pages.check()
    assert out["accepted"].tolist() == [3, 1, 0] and out["new_len"].tolist() == [26, 2, 70]
    assert out["path"].tolist()[:7] == [0, 2, 4, -1, -1, -1, -1]
    hist = [torch.cat([hist[0], drafts[0][[0, 2, 4]]]), torch.cat([hist[1], drafts[1]]), hist[2]]

    # one row each from there
    last = [rows_of(1, S.H, 30 + i) for i in range(3)]
    h, lg, _ = S.step(torch.cat(last), out["new_len"].tolist(), [1, 1, 1], spare=spare)
    for i in range(3):
        S.check(h[i], lg[i], torch.cat([hist[i], last[i]]))


def test_prompt_step_agrees_with_the_prefill(small_navi):
    """A prompt's rows through the pages and through the talker's own cache: the same last row."""
    S = Session(small_navi)
    cfg = S.W.cfg
    rng = np.random.default_rng(3)
    ids = [cfg.im_start_id, cfg.assistant_id, 198] + rng.integers(0, cfg.text_vocab, 30).tolist() + \
          [cfg.im_end_id, 198, cfg.im_start_id, cfg.assistant_id, 198]
    pr = S.tal.build_prompt(ids, "english", rng.standard_normal(S.H).astype(np.float32))
    n = pr.n_prefill
    host = torch.empty(n, S.H, device="cuda")
    import ctypes
    cudart = ctypes.CDLL("libcudart.so.12")

    def fetch(dst, src, count):
        assert cudart.cudaMemcpy(ctypes.c_void_p(dst.data_ptr()), ctypes.c_void_p(src), ctypes.c_size_t(count * 4), 3) == 0

    fetch(host, pr.prefill, n * S.H)
    S.tal.prefill(pr)
    hid, lg = torch.empty(S.H, device="cuda"), torch.empty(S.V, device="cuda")
    fetch(hid, S.tal.d_hidden(), S.H)
    fetch(lg, S.tal.d_logits(), S.V)
    h2, lg2, _ = S.step(host.cpu(), [0], [n])
    assert om.rel_l2(h2[n - 1].numpy(), hid.cpu()) < REL and om.rel_l2(lg2[n - 1].numpy(), lg.cpu()) < REL
    S.check(h2[n - 1], lg2[n - 1], host.cpu())


def test_step_refusals(small_navi):
    S = Session(small_navi, max_prompt=16)
    t = S.W.tl
    x = torch.zeros(64 * max(S.H, S.V), device="cuda")
    z = i32([0] * 8)
    q = torch.zeros(64, dtype=torch.int64, device="cuda")

    def call(pages, rows=4, **kw):
        f = dict(n_req=1, max_rows=rows, max_new=rows, ctx_len=z.data_ptr(), n_new=z.data_ptr(), cu_rows=z.data_ptr(), row_req=q.data_ptr(),
                 pos=q.data_ptr(), slot=q.data_ptr(), status=z.data_ptr())
        S.tal.step(pages, engine.TreeStep(**{**f, **kw}), x.data_ptr(), x.data_ptr())

    for bad in (dict(n_layer=t.n_layer + 1), dict(n_kv_head=t.n_kv_head + 1), dict(head_dim=64), dict(dtype=capi.NAVI_BF16)):
        kw = {**dict(n_layer=t.n_layer, n_pages=4, page_size=16, n_kv_head=t.n_kv_head, head_dim=t.head_dim, max_requests=2, max_blocks=2), **bad}
        with pytest.raises(capi.NaviError) as e:
            call(engine.PagedKv.create(S.dev, **kw))
        assert e.value.status == capi.NAVI_E_SHAPE
    for kw in (dict(rows=17), dict(n_req=4), dict(ctx_len=0)):
        with pytest.raises(capi.NaviError) as e:
            call(S.pages, **kw)
        assert e.value.status == capi.NAVI_E_ARG
