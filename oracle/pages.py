"""Plain 64-bit restatement of the paged KV cache's operators (include/navi_b200.h, "paged KV
cache and drafted trees"): loops over requests, rows and heads on the CPU, written from the
definitions for the tests. Pools are [n_pages][n_kv_head][page_size][head_dim] float64 tensors."""
from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch

OK, E_ARG, KV_FULL, SHAPE = 0, 1, 5, 7


@dataclass
class Tables:
    """The block tables and the stack of free pages."""
    page: int
    blocks: int
    table: list                      # per table row a list of `blocks` page ids (stale past held)
    held: list
    free: list                       # the whole stack array; its top is n_free - 1
    n_free: int
    n_pages: int

    @staticmethod
    def fresh(n_pages, page, rows, blocks):
        return Tables(page, blocks, [[0] * blocks for _ in range(rows)], [0] * rows, list(range(n_pages - 1, -1, -1)), n_pages, n_pages)


@dataclass
class Step:
    ctx: list
    new: list
    parent: list | None              # flat, per row; None: a chain
    req: list | None = None          # table rows
    max_rows: int | None = None
    max_new: int | None = None
    cu: list = field(default_factory=list)
    row_req: list = field(default_factory=list)
    pos: list = field(default_factory=list)
    slot: list = field(default_factory=list)
    anc: list = field(default_factory=list)   # sets of the request's rows: the row and its ancestors
    status: list = field(default_factory=list)


def plan(t: Tables, s: Step) -> None:
    B = len(s.ctx)
    cap = s.max_rows if s.max_rows is not None else sum(max(n, 0) for n in s.new)
    most = s.max_new if s.max_new is not None else max(s.new, default=0)
    req = s.req if s.req is not None else list(range(B))
    s.cu, at = [0], 0
    s.status, need = [], []
    for i in range(B):
        at += max(s.new[i], 0)
        s.cu.append(min(at, cap))
        k = -(-(s.ctx[i] + max(s.new[i], 0)) // t.page)
        need.append(k)
        if s.new[i] < 0 or s.ctx[i] < 0 or not 0 <= req[i] < len(t.held) or not 0 <= t.held[req[i]] <= t.blocks:
            s.status.append(E_ARG)
        elif s.new[i] > most or k > t.blocks or at > cap:
            s.status.append(SHAPE)
        else:
            s.status.append(OK)
    back = [t.table[req[i]][b] for i in range(B) if s.status[i] == OK for b in range(need[i], t.held[req[i]])]
    for p in reversed(back):
        t.free[t.n_free] = p
        t.n_free += 1
    wanted, room = 0, t.n_free
    for i in range(B):
        if s.status[i] != OK:
            continue
        more = max(need[i] - t.held[req[i]], 0)
        wanted += more
        if more and wanted > room:
            s.status[i] = KV_FULL
            continue
        for b in range(t.held[req[i]], need[i]):
            t.n_free -= 1
            t.table[req[i]][b] = t.free[t.n_free]
        t.held[req[i]] = need[i]
    s.row_req, s.pos, s.slot, s.anc = [], [], [], []
    broken = set()
    for i in range(B):
        for j in range(s.cu[i + 1] - s.cu[i]):
            seen, whole, a = set(), True, j
            if s.parent is None:
                depth = j
            else:
                depth = -1
                while a >= 0 and whole:
                    seen.add(a)
                    depth += 1
                    up = s.parent[s.cu[i] + a]
                    whole = -1 <= up < a
                    a = up
                if not whole:
                    broken.add(i)
                    seen = set()
            at = s.ctx[i] + j
            ok = s.status[i] == OK and whole
            s.row_req.append(i)
            s.pos.append(s.ctx[i] + depth)
            s.slot.append(t.table[req[i]][at // t.page] * t.page + at % t.page if ok else -1)
            s.anc.append(seen)
    for i in broken:
        if s.status[i] == OK:
            s.status[i] = E_ARG


def store(page, s: Step, qkv, n_head, n_kv, k, v, q_norm=None, k_norm=None, eps=1e-6, rope=None):
    """q rows [T][n_head][D]; k and v are written in place."""
    T = len(s.slot)
    D = k.shape[-1]
    x = qkv.double().reshape(-1, n_head + 2 * n_kv, D).clone()
    q = torch.zeros(T, n_head, D, dtype=torch.float64)
    for r in range(T):
        known = rope is None or 0 <= s.pos[r] < rope.shape[0]
        for h in range(n_head + n_kv):
            y = x[r, h]
            w = q_norm if h < n_head else k_norm
            if w is not None:
                y = y / math.sqrt(float((y * y).sum()) / D + eps) * w.double()
            if rope is not None and known:
                c, sn = rope[s.pos[r], :D // 2].double(), rope[s.pos[r], D // 2:].double()
                y = torch.cat([y[:D // 2] * c - y[D // 2:] * sn, y[:D // 2] * sn + y[D // 2:] * c])
            if h < n_head:
                q[r, h] = y if known else 0.0
            elif s.slot[r] >= 0 and known:
                k[s.slot[r] // page, h - n_head, s.slot[r] % page] = y
        if s.slot[r] >= 0 and known:
            v[s.slot[r] // page, :, s.slot[r] % page] = x[r, n_head + n_kv:]
    return q


def attend(t: Tables, s: Step, q, k, v, scale):
    """(out [T][H][D], lse [T][H]) of q [T][H][D] float64."""
    T, H, D = q.shape
    G = k.shape[1]
    out = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    req = s.req if s.req is not None else list(range(len(s.ctx)))
    for i in range(len(s.ctx)):
        if s.status[i] != OK:
            continue
        n, L = s.cu[i + 1] - s.cu[i], s.ctx[i] + s.cu[i + 1] - s.cu[i]
        if n == 0 or L == 0:
            continue
        pages = torch.tensor(t.table[req[i]][:-(-L // t.page)])
        ki = k[pages].transpose(0, 1).reshape(G, -1, D)[:, :L]
        vi = v[pages].transpose(0, 1).reshape(G, -1, D)[:, :L]
        for j in range(n):
            seen = list(range(s.ctx[i])) + [s.ctx[i] + a for a in (sorted(s.anc[s.cu[i] + j]) if s.parent is not None else range(j + 1))]
            if not seen:
                continue
            sc = torch.einsum("hd,hkd->hk", q[s.cu[i] + j].double(), ki[:, seen].repeat_interleave(H // G, 0)) * scale
            lse[s.cu[i] + j] = torch.logsumexp(sc, 1)
            out[s.cu[i] + j] = torch.einsum("hk,hkd->hd", torch.softmax(sc, 1), vi[:, seen].repeat_interleave(H // G, 0))
    return out, lse


def commit(page, s: Step, tokens, targets, root, pools):
    """(paths, next ids) per request; the pools are moved in place."""
    paths, nxt = [], []
    for i in range(len(s.ctx)):
        path, at, want = [], -1, root[i]
        while s.status[i] == OK:
            kids = [j for j in range(s.cu[i + 1] - s.cu[i]) if s.parent[s.cu[i] + j] == at and list(tokens[s.cu[i] + j]) == list(want)]
            if not kids:
                break
            at = kids[0]
            want = targets[s.cu[i] + at]
            path.append(at)
        for n, j in enumerate(path):
            a, b = s.slot[s.cu[i] + j], s.slot[s.cu[i] + n]
            for p in pools:
                p[b // page, :, b % page] = p[a // page, :, a % page].clone()
        paths.append(path)
        nxt.append(list(want))
    return paths, nxt
