"""Edges of navi_talker_step: the end of the talker's positions, steps without rows, cached prompts of requests
that are refused. Rows that are served are compared with the CPU oracle's prefill as in test_step_gpu.py."""
import ctypes

import pytest
import torch

from navi_b200 import capi, engine
from test_step_gpu import Session, branch, i32, rows_of

pytestmark = pytest.mark.gpu


class Short(Session):
    """A talker of few positions; step_any() allows requests that are not served."""

    def __init__(self, path, positions):
        super().__init__(path)
        self.tal = engine.Talker(self.dev, self.w, max_prompt_tokens=64, max_positions=positions)

    def step_any(self, rows, ctx, new, parent=None):
        T, B = max(sum(new), 1), len(ctx)
        d = torch.zeros(T, self.H, device="cuda")
        d[:sum(new)] = rows.cuda()
        hidden, logits = torch.zeros(T, self.H, device="cuda"), torch.zeros(T, self.V, device="cuda")
        keep = dict(ctx_len=i32(ctx), n_new=i32(new), cu_rows=i32([0] * (B + 1)), row_req=i32([0] * T), pos=i32([0] * T),
                    slot=torch.zeros(T, dtype=torch.int64, device="cuda"), status=i32([-7] * B))
        words = 1 if parent is not None else 0
        if words:
            keep.update(parent=i32(parent), mask=torch.zeros(T, 1, dtype=torch.int64, device="cuda"))
        s = engine.TreeStep(n_req=B, max_rows=sum(new), max_new=max(new), mask_words=words, **{k: v.data_ptr() for k, v in keep.items()})
        torch.cuda.synchronize()
        self.tal.step(self.pages, s, d.data_ptr(), hidden.data_ptr(), logits.data_ptr())
        return hidden.cpu(), logits.cpu(), keep["status"].tolist(), keep["slot"].tolist()


def test_requests_at_the_end_of_the_positions(small_navi):
    """The last position is served; a row past it refuses its request, which would attend to what was never stored."""
    S = Short(small_navi, 64)
    hist = [rows_of(n, S.H, 40 + n) for n in (62, 63, 9)]
    for i, (ctx, n) in enumerate([([0, 0, 0], 62), ([62, 0, 0], 63), ([62, 63, 0], 9)]):
        _, _, st, _ = S.step_any(hist[i], ctx, [n if k == i else 0 for k in range(3)])
        assert st == [capi.NAVI_OK] * 3
    # chains: one row too many, up to the end, far from it
    x = [rows_of(n, S.H, 50 + n) for n in (3, 1, 4)]
    h, lg, st, slot = S.step_any(torch.cat(x), [62, 63, 9], [3, 1, 4])
    assert st == [capi.NAVI_E_SHAPE, capi.NAVI_OK, capi.NAVI_OK] and slot[:3] == [-1] * 3
    S.check(h[3], lg[3], torch.cat([hist[1], x[1]]))
    S.check(h[7], lg[7], torch.cat([hist[2], x[2]]))
    # trees: more rows than positions but no branch too deep; a branch too deep; a bad parent among rows too deep
    trees = [[-1, 0, 0, -1, 3], [-1, -1, 1], [-1, 0, 1, 7]]
    x = [rows_of(len(t), S.H, 60 + k) for k, t in enumerate(trees)]
    h, lg, st, _ = S.step_any(torch.cat(x), [62, 63, 62], [len(t) for t in trees], sum(trees, []))
    assert st == [capi.NAVI_OK, capi.NAVI_E_SHAPE, capi.NAVI_E_ARG]
    for j in range(5):
        S.check(h[j], lg[j], torch.cat([hist[0], x[0][branch(trees[0], j)]]))
    # nothing of that is left for the next step
    x = rows_of(2, S.H, 70)
    h, lg, st, _ = S.step_any(x, [62, 63, 9], [1, 0, 1], [-1, -1])
    assert st == [capi.NAVI_OK] * 3
    S.check(h[0], lg[0], torch.cat([hist[0], x[:1]]))
    _, _, st, _ = S.step_any(rows_of(3, S.H, 80), [62], [3])
    assert st == [capi.NAVI_E_SHAPE]


@pytest.mark.parametrize("requests", [0, 3])
def test_a_step_without_rows_waits_too(small_navi, requests):
    """A step that only gives pages back, or does nothing, has ended when the call returns; its time is its own."""
    S = Session(small_navi)
    cudart = ctypes.CDLL("libcudart.so.12")
    S.step(rows_of(200, S.H, 1), [0, 0, 0], [100, 60, 40])
    before = S.tal.last_ms()
    z, st, cu = i32([0] * 8), i32([-7] * 4), i32([0] * 4)
    torch.cuda.synchronize()
    p = z.data_ptr()
    s = engine.TreeStep(n_req=requests, max_rows=0, max_new=0, ctx_len=p, n_new=p, cu_rows=cu.data_ptr(), status=st.data_ptr())
    S.tal.step(S.pages, s, 0, 0)
    assert cudart.cudaStreamQuery(ctypes.c_void_p(S.dev.stream)) == 0
    assert st.tolist()[:requests] == [capi.NAVI_OK] * requests
    assert 0 <= S.tal.last_ms() < before
