"""The paged KV cache operators: what is measured of them, and their plain forms.

Four operators share one step of a batch of requests (include/navi_b200.h, "paged KV cache"):

  plan    block tables, slot maps, positions and ancestor masks from the requests' lengths
  store   q/k RMSNorm and RoPE of a step's rows, keys and values into their page slots
  attend  attention of a step's rows (single tokens, drafted trees, prompt chunks) over the pages
  commit  the walk of a drafted tree against the model's choices, accepted rows moved to the front

`run` computes them with elementary torch operations in 32 bits where `own` is false, and calls
navi_b200.engine where it is true; both work on what `prepare` makes.  Lengths of a batch are
quantiles of a range, so the work of a case follows from the case alone; a seed only deals them
out to the requests.
"""
import math
import os
import sys

import torch

own = False

F32, F16, BF16 = 0, 1, 2                       # the .navi type codes
TYPES = {"f32": (torch.float32, F32), "f16": (torch.float16, F16), "bf16": (torch.bfloat16, BF16)}
KV_FULL, SHAPE = 5, 7                          # NAVI_E_KV_FULL, NAVI_E_SHAPE
EPS = 1e-6
FRAME_CODES = 16                               # ids of one frame: what a drafted node holds
ACCEPT = 0.8                                   # how often the model's choice is one of a node's children


# ---- the cases --------------------------------------------------------------------------------

def case(op, name=None, **kw):
    c = dict(op=op, reqs=4, ctx_lo=1, ctx_hi=1, new_lo=1, new_hi=1, tree=True, page=16, heads=16, kv_heads=8, dim=128, dtype="f32", layers=1)
    c.update(kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # the frame kernel's four streams one frame on: what a serving step pays before any arithmetic
        case("plan", "plan 4 streams", reqs=4, ctx_lo=10, ctx_hi=600),
        # 64 streams with a drafted tree each
        case("plan", "plan 64 trees", reqs=64, ctx_lo=100, ctx_hi=4001, new_lo=0, new_hi=61),
        # a thousand prompts admitted at once
        case("plan", "plan 1000 prompts", reqs=1000, ctx_lo=0, ctx_hi=0, new_lo=9, new_hi=1024, tree=False),
        # the talker's rows of four drafted trees (f32 activations, f16 cache)
        case("store", "store 4 trees f32", reqs=4, ctx_lo=10, ctx_hi=600, new_lo=9, new_hi=16),
        # sixteen prompts of bf16 activations
        case("store", "store 16 prompts bf16", reqs=16, ctx_lo=0, ctx_hi=77, new_lo=500, new_hi=1023, tree=False, dtype="bf16"),
        # the frame kernel's four streams at the benchmark's KV 512: latency
        case("attend", "attend 4 streams f32", reqs=4, ctx_lo=512, ctx_hi=512),
        # the talker checking four drafted trees (f32 activations)
        case("attend", "attend 4 trees f32", reqs=4, ctx_lo=200, ctx_hi=2048, new_lo=9, new_hi=16),
        # many streams of ragged lengths, odd trees, f16
        case("attend", "attend 48 trees f16", reqs=48, ctx_lo=255, ctx_hi=8191, new_lo=0, new_hi=33, dtype="f16"),
        # one long session, a small tree: the keys of one request spread over the whole GPU
        case("attend", "attend 1 long bf16", reqs=1, ctx_lo=200003, ctx_hi=200003, new_lo=5, new_hi=5, page=64, dtype="bf16"),
        # chunks of long prompts over what is cached: arithmetic
        case("attend", "attend 8 chunks bf16", reqs=8, ctx_lo=511, ctx_hi=4097, new_lo=1000, new_hi=1000, tree=False, dtype="bf16", page=32),
        # four streams' accepted frames through the talker's 28 layers
        case("commit", "commit 4 trees", reqs=4, ctx_lo=10, ctx_hi=600, new_lo=9, new_hi=16, layers=28, dtype="f16"),
        # sixty-four streams', larger trees
        case("commit", "commit 64 trees", reqs=64, ctx_lo=3, ctx_hi=90, new_lo=20, new_hi=64, layers=28, dtype="f16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most = max(weight(c) for c in listed())
    while True:
        op = rng.choice(["plan", "store", "attend", "attend", "commit"])
        heads, kv_heads, dim = rng.choice([(16, 8, 128), (16, 8, 128), (4, 2, 128), (32, 4, 128), (16, 16, 64)])
        kind = rng.choice(["token", "tree", "tree", "prompt"])
        kw = dict(page=rng.choice([16, 32, 64]), heads=heads, kv_heads=kv_heads, dim=dim, dtype=rng.choice(["f32", "f16", "bf16"]))
        if op == "plan":
            kw.update(heads=16, kv_heads=8, dim=128, dtype="f32", reqs=log(2, 1000))
        else:
            kw.update(reqs=log(2, 64))
        ctx = log(16, 16384 if op != "commit" else 512)
        kw.update(ctx_lo=rng.randint(0, ctx), ctx_hi=ctx)
        if op == "commit" or kind == "tree":
            n = log(3, 64)
            kw.update(new_lo=rng.randint(0, n), new_hi=n)
        elif kind == "prompt":
            n = log(17, 1024)
            kw.update(new_lo=rng.randint(1, n), new_hi=n, tree=False)
        if op == "commit":
            kw.update(layers=rng.choice([5, 28]), dtype="f16")
        if op == "attend" and kind == "tree" and rng.random() < 0.15:
            kw.update(reqs=1, ctx_lo=log(20000, 200000))
            kw.update(ctx_hi=kw["ctx_lo"])
        c = case(op, **kw)
        # the pools of a step, and the plain forms' padded copies of them, stay within a few GB
        if weight(c) <= most and sum(lens(c)) > 0 and pool_tokens(c) * c["layers"] * c["kv_heads"] * c["dim"] < 4e8 and \
                c["reqs"] * c["heads"] * max(lens(c)) * (max(ctxs(c)) + max(lens(c))) < 1.5e9:
            return c


def spread(lo, hi, n):
    """n lengths from lo to hi, evenly spread over their logarithm."""
    if n == 1:
        return [hi]
    return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** (i / (n - 1)))) - 1 for i in range(n)]


def ctxs(c):
    return spread(c["ctx_lo"], c["ctx_hi"], c["reqs"])


def lens(c):
    return spread(c["new_lo"], c["new_hi"], c["reqs"])


def dealt(c, seed):
    """(ctx, new) per request: the lengths in an order made from the seed."""
    g = torch.Generator().manual_seed(seed * 7919 + 13)
    n = c["reqs"]
    ctx, new = torch.tensor(ctxs(c)), torch.tensor(lens(c))
    return ctx[torch.randperm(n, generator=g)].tolist(), new[torch.randperm(n, generator=g)].tolist()


def pool_tokens(c):
    return sum(-(-(a + max(lens(c))) // c["page"]) * c["page"] for a in ctxs(c))


def weight(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def work(c):
    T, B = sum(lens(c)), c["reqs"]
    elt = 4 if c["dtype"] == "f32" else 2
    row = c["heads"] * c["dim"]
    kv_row = 2 * c["kv_heads"] * c["dim"] * 2                            # K and V of one token, 16-bit
    words = mask_words(c)
    if c["op"] == "plan":
        taken = sum(lens(c)) / c["page"]                                 # about: pages that a step takes, and gives back
        return {"bytes": T * (4 + 4 + 8 + (4 + 8 * words if c["tree"] else 0)) + 16 * B + 16 * taken, "flops": 0}
    if c["op"] == "store":
        return {"bytes": T * (row * 2 + 2 * c["kv_heads"] * c["dim"]) * elt + T * kv_row + 12 * T, "flops": T * (row + c["kv_heads"] * c["dim"]) * 8}
    if c["op"] == "attend":
        # lengths are dealt out by the seed: the mean of the pairs
        ctx = sum(ctxs(c)) / B
        seen = sum(n * (ctx + (n / 2 if not c["tree"] else 0)) for n in lens(c))
        keys = sum(a + n for a, n in zip(ctxs(c), lens(c)) if n)
        return {"bytes": keys * kv_row + T * row * 2 * elt + 4 * T * c["heads"], "flops": 4 * row * seen}
    # commit: a path takes on about as many rows as the accepted children in a row; those off their place move
    path = sum(min(n, ACCEPT / (1 - ACCEPT)) for n in lens(c))
    return {"bytes": T * FRAME_CODES * 8 + 0.7 * path * c["layers"] * kv_row * 2, "flops": 0}


def mask_words(c):
    return max(1, -(-max(lens(c)) // 64)) if c["tree"] else 0


# ---- inputs -----------------------------------------------------------------------------------

def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev = dict(device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    ctx_h, new_h = dealt(c, seed)
    B, P = c["reqs"], c["page"]
    T, N = sum(new_h), max(new_h)
    ctx, new = torch.tensor(ctx_h, **i32), torch.tensor(new_h, **i32)
    words = mask_words(c)
    s = dict(c=c, ctx=ctx, new=new, n_max=N, l_max=max(a + n for a, n in zip(ctx_h, new_h)), T=T, words=words)

    # drafted trees: a node hangs on one of the nodes just before it, a few of them on the last committed token
    row_req = torch.repeat_interleave(torch.arange(B, **dev), new.long(), output_size=T)
    cu = torch.zeros(B + 1, dtype=torch.int64, **dev)
    cu[1:] = new.long().cumsum(0)
    local = torch.arange(T, **dev) - cu[row_req]
    back = 1 + (torch.rand(T, generator=g, **dev) ** 2 * 4).long()
    parent = torch.clamp(local - back, min=-1) if c["tree"] else local - 1
    s["parent"] = parent.int() if c["tree"] else None

    # pages in a random order: what the requests hold, then the free stack
    held_h = [-(-a // P) for a in ctx_h]
    MB = max(1, -(-(max(ctxs(c)) + max(lens(c))) // P))
    n_pages = sum(held_h) + sum(-(-n // P) + 1 for n in new_h) + 5         # the same for every deal
    ids = torch.randperm(n_pages, generator=g, device="cuda").int()
    held = torch.tensor(held_h, **i32)
    table = torch.full((B, MB), -1, **i32)
    blk = torch.arange(MB, **dev)
    has = blk[None, :] < held[:, None]
    table[has] = ids[:sum(held_h)]
    s.update(table=table, held=held, free=torch.cat([ids[sum(held_h):], torch.full((sum(held_h),), -1, **i32)]),
             n_free=torch.tensor([n_pages - sum(held_h)], **i32), n_pages=n_pages, blocks=MB)
    # what plan writes
    s["out"] = dict(cu_rows=torch.zeros(B + 1, **i32), row_req=torch.zeros(T, **i32), pos=torch.zeros(T, **i32),
                    slot=torch.zeros(T, dtype=torch.int64, **dev), mask=torch.zeros((T, max(words, 1)), dtype=torch.int64, **dev),
                    status=torch.zeros(B, **i32))
    s["back"] = {k: torch.zeros_like(v) for k, v in s["out"].items()}    # the step that gives the pages back
    s["none"] = torch.zeros_like(new)
    if c["op"] != "plan":
        plain_plan(s, new, s["out"])                                     # the other operators start from a planned step

    tt, code = TYPES[c["dtype"]]
    kt = torch.float16 if c["dtype"] == "f32" else tt
    s["code"], s["kv_code"] = code, F16 if c["dtype"] == "f32" else code
    H, G, D, L = c["heads"], c["kv_heads"], c["dim"], c["layers"]
    if c["op"] != "plan":
        k = torch.empty((L, n_pages, G, P, D), dtype=kt, **dev)
        v = torch.empty((L, n_pages, G, P, D), dtype=kt, **dev)
        fill(k, g)
        fill(v, g)
        s.update(k=k, v=v)
    if c["op"] == "store":
        s["qkv"] = (torch.randn((T, (H + 2 * G) * D), generator=g, **dev) * 1.5).to(tt)
        s["q_out"] = torch.zeros((T, H * D), dtype=tt, **dev)
        s["q_norm"] = torch.rand(D, generator=g, **dev) + 0.5
        s["k_norm"] = torch.rand(D, generator=g, **dev) + 0.5
        n_pos = s["l_max"] + 1
        ang = torch.arange(n_pos, **dev)[:, None].float() * (1e6 ** (-torch.arange(0, D, 2, **dev).double() / D)).float()[None, :]
        s["rope"] = torch.cat([ang.double().cos(), ang.double().sin()], 1).float()
    if c["op"] == "attend":
        s["q"] = (torch.randn((T, H * D), generator=g, **dev) * 2).to(tt)   # scores of a few units: some keys count more than others
        s["o"] = torch.zeros((T, H * D), dtype=tt, **dev)
        s["lse"] = torch.zeros((T, H), dtype=torch.float32, **dev)
    if c["op"] == "commit":
        W = FRAME_CODES
        tokens = torch.randint(0, 2048, (T, W), generator=g, **dev).int()
        targets = torch.randint(0, 2048, (T, W), generator=g, **dev).int()
        root = torch.randint(0, 2048, (B, W), generator=g, **dev).int()
        # the model's choice at a node: one of its children's tokens most of the time
        key = row_req * (N + 1) + parent + 1
        last = torch.full((B * (N + 1),), -1, dtype=torch.int64, **dev).scatter_reduce(0, key, torch.arange(T, **dev), "amax")
        mine = last[row_req * (N + 1) + local + 1]
        hit = (mine >= 0) & (torch.rand(T, generator=g, **dev) < ACCEPT)
        targets = torch.where(hit[:, None], tokens[mine.clamp(min=0)], targets) if T else targets
        mine = last.view(B, N + 1)[:, 0]
        root = torch.where((mine >= 0)[:, None], tokens[mine.clamp(min=0)], root) if T else root
        s.update(tokens=tokens, targets=targets, root=root, n_acc=torch.zeros(B, **i32), path=torch.zeros(T, **i32),
                 new_len=torch.zeros(B, **i32), nxt=torch.zeros((B, W), **i32))
    if own:
        handles(s)
    return s


def fill(t, g):
    """Standard normal values, made in slices so that no 32-bit copy of a whole pool is needed."""
    flat = t.view(-1)
    for a in range(0, flat.numel(), 1 << 26):
        n = min(1 << 26, flat.numel() - a)
        flat[a:a + n] = torch.randn(n, generator=g, device="cuda")


device = None


def handles(s):
    """The cache's handle and the steps that a user's program keeps."""
    global device
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "navi-tts_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    from navi_b200 import engine
    if device is None:
        device = engine.Device(0)
    c, p = s["c"], lambda t: t.data_ptr() if t is not None else 0
    k = [p(x) for x in s["k"]] if "k" in s else [0]
    v = [p(x) for x in s["v"]] if "v" in s else [0]
    s["pages"] = engine.PagedKv.wrap(device, k, v, n_pages=s["n_pages"], page_size=c["page"], n_kv_head=c["kv_heads"], head_dim=c["dim"],
                                     dtype=s["kv_code"], max_requests=c["reqs"], max_blocks=s["blocks"], table=p(s["table"]),
                                     held=p(s["held"]), free_pages=p(s["free"]), n_free=p(s["n_free"]))

    def step(new, out):
        return engine.TreeStep(n_req=c["reqs"], max_rows=s["T"], max_new=s["n_max"], ctx_len=p(s["ctx"]), n_new=p(new), parent=p(s["parent"]),
                               cu_rows=p(out["cu_rows"]), row_req=p(out["row_req"]), pos=p(out["pos"]), slot=p(out["slot"]),
                               mask=p(out["mask"]) if s["words"] else 0, mask_words=s["words"], status=p(out["status"]))

    s["step"] = step(s["new"], s["out"])
    s["step_back"] = step(s["none"], s["back"])
    if c["op"] == "store":
        s["args"] = engine.StoreArgs(qkv=p(s["qkv"]), q_out=p(s["q_out"]), dtype=s["code"], n_head=c["heads"], q_norm=p(s["q_norm"]),
                                     k_norm=p(s["k_norm"]), eps=EPS, rope=p(s["rope"]), rope_positions=s["rope"].shape[0])
    if c["op"] == "attend":
        s["args"] = engine.AttendArgs(q=p(s["q"]), out=p(s["o"]), lse=p(s["lse"]), dtype=s["code"], n_head=c["heads"], scale=c["dim"] ** -0.5)
    if c["op"] == "commit":
        s["args"] = engine.CommitArgs(width=FRAME_CODES, tokens=p(s["tokens"]), targets=p(s["targets"]), root_target=p(s["root"]),
                                      accepted=p(s["n_acc"]), path=p(s["path"]), new_len=p(s["new_len"]), next_token=p(s["nxt"]))


# ---- one pass -----------------------------------------------------------------------------------

def run(s):
    op = s["c"]["op"]
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        if op == "plan":
            s["pages"].plan(s["step"], stream=stream)
            s["pages"].plan(s["step_back"], stream=stream)
        elif op == "store":
            s["pages"].store(s["step"], 0, s["args"], stream=stream)
        elif op == "attend":
            s["pages"].attend(s["step"], 0, s["args"], stream=stream)
        else:
            s["pages"].commit(s["step"], s["args"], stream=stream)
    elif op == "plan":
        # a step is planned, its pages are taken, and then given back: the drafts of a step that is dropped
        plain_plan(s, s["new"], s["out"])
        plain_plan(s, s["none"], s["back"])
    else:
        {"store": plain_store, "attend": plain_attend, "commit": plain_commit}[op](s)
    if op == "plan":
        o = s["out"]
        got = [o["cu_rows"], o["row_req"], o["pos"], o["slot"], o["status"], s["table"], s["held"], s["free"], s["n_free"], s["back"]["status"]]
        return got + [o["mask"]] if s["words"] else got
    if op == "store":
        return [s["q_out"], s["k"], s["v"]]
    if op == "attend":
        return [s["o"], s["lse"]]
    return [s["n_acc"], s["path"], s["new_len"], s["nxt"], s["k"], s["v"]]


def plain_plan(s, new, out):
    c, P = s["c"], s["c"]["page"]
    dev = dict(device="cuda")
    ctx, new, held = s["ctx"].long(), new.long(), s["held"].long()
    B, MB = s["table"].shape
    T = out["row_req"].numel()
    cu = torch.zeros(B + 1, dtype=torch.int64, **dev)
    cu[1:] = new.cumsum(0)
    need = (ctx + new + P - 1) // P
    fits = need <= MB
    surplus = torch.where(fits, (held - need).clamp(min=0), 0)
    grow = torch.where(fits, (need - held).clamp(min=0), 0)
    F = s["n_free"][0].long()
    blk = torch.arange(MB, **dev)[None, :]
    # pages past a request's need go on the stack, the first request's first page on top
    top = F + surplus.sum()
    gone = (blk >= need[:, None]) & (blk < held[:, None]) & fits[:, None]
    nth = (surplus.cumsum(0) - surplus)[:, None] + blk - need[:, None]
    s["free"][(top - 1 - nth)[gone]] = s["table"][gone]
    # pages are taken from the top, first come first served
    cum = grow.cumsum(0)
    served = fits & ((grow == 0) | (cum <= top))
    new_blk = (blk >= held[:, None]) & (blk < need[:, None]) & served[:, None]
    nth = (cum - grow)[:, None] + blk - held[:, None]
    s["table"][new_blk] = s["free"][(top - 1 - nth)[new_blk]]
    s["held"].copy_(torch.where(served, need, held))
    s["n_free"].copy_((top - torch.where(served, grow, 0).sum())[None])
    out["status"].copy_(torch.where(fits, torch.where(served, 0, KV_FULL), SHAPE))
    out["cu_rows"].copy_(cu)
    r = torch.arange(T, **dev)
    req = torch.searchsorted(cu, r, right=True) - 1
    live = req < B
    req = req.clamp(max=B - 1)
    j = r - cu[req]
    at = ctx[req] + j
    page = s["table"][req, (at // P).clamp(max=MB - 1)].long()
    slot = torch.where(served[req], page * P + at % P, -1)
    if c["tree"]:
        N = s["n_max"]
        # ancestors: the pattern of (I + parent)^N, whose entries are counts of walks
        A = torch.zeros((B, N, N), dtype=torch.float64, **dev)
        A[req[live], j[live], j[live]] = 1
        par = s["parent"].long()
        up = live & (par >= 0)
        A[req[up], j[up], par[up]] = 1
        A = torch.matrix_power(A, max(N, 1)) > 0
        rows = A[req, j.clamp(max=max(N - 1, 0))]
        pos = ctx[req] + rows.sum(1) - 1
        W = s["words"]
        bits = torch.zeros((T, W * 64), dtype=torch.int64, **dev)
        bits[:, :N] = rows
        mask = (bits.view(T, W, 64) << torch.arange(64, **dev)).sum(2)
        out["mask"].copy_(torch.where(live[:, None], mask, out["mask"]))
    else:
        pos = at
    out["row_req"].copy_(torch.where(live, req, out["row_req"].long()))
    out["pos"].copy_(torch.where(live, pos, out["pos"].long()))
    out["slot"].copy_(torch.where(live, slot, out["slot"]))


def plain_store(s):
    c, o = s["c"], s["out"]
    H, G, D, P, T = c["heads"], c["kv_heads"], c["dim"], c["page"], s["T"]
    x = s["qkv"].float().view(T, H + 2 * G, D)
    qk = x[:, :H + G]
    w = torch.cat([s["q_norm"].expand(H, D), s["k_norm"].expand(G, D)])
    qk = qk * torch.rsqrt((qk * qk).mean(2, keepdim=True) + EPS) * w
    cs = s["rope"][o["pos"].long()]
    cos, sin = cs[:, None, :D // 2], cs[:, None, D // 2:]
    a, b = qk[..., :D // 2], qk[..., D // 2:]
    qk = torch.cat([a * cos - b * sin, a * sin + b * cos], 2)
    s["q_out"].copy_(qk[:, :H].reshape(T, H * D))
    page, off = o["slot"] // P, o["slot"] % P
    s["k"][0][page, :, off] = qk[:, H:].to(s["k"].dtype)
    s["v"][0][page, :, off] = x[:, H + G:].to(s["v"].dtype)


def plain_attend(s):
    c, o = s["c"], s["out"]
    H, G, D, P, B, N, Lm, T = c["heads"], c["kv_heads"], c["dim"], c["page"], c["reqs"], s["n_max"], s["l_max"], s["T"]
    dev = dict(device="cuda")
    req = o["row_req"].long()
    j = torch.arange(T, **dev) - o["cu_rows"].long()[req]
    q = torch.zeros((B, N, H, D), dtype=torch.float32, **dev)
    q[req, j] = s["q"].float().view(T, H, D)
    at = torch.arange(Lm, **dev)
    page = s["table"].long().clamp(min=0)[:, at // P]                                # [B][Lm]
    k = s["k"][0][page, :, (at % P).expand(B, Lm)].float()                           # [B][Lm][G][D]
    sc = q.view(B, N, G, H // G, D).permute(0, 2, 1, 3, 4).reshape(B, G, N * (H // G), D) @ k.permute(0, 2, 3, 1)
    del k
    sc = sc.view(B, G, N, H // G, Lm) * D ** -0.5
    a = (at[None, :] - s["ctx"].long()[:, None])                                     # key's place among the new rows
    if c["tree"]:
        m = torch.zeros((B, N, s["words"]), dtype=torch.int64, **dev)
        m[req, j] = o["mask"]
        word = (a // 64).clamp(0, s["words"] - 1)
        bit = (torch.gather(m, 2, word[:, None, :].expand(B, N, Lm)) >> (a % 64)[:, None, :]) & 1
        seen = (a < 0)[:, None, :] | ((a >= 0) & (a < s["words"] * 64))[:, None, :] & (bit == 1)
    else:
        seen = a[:, None, :] <= torch.arange(N, **dev)[None, :, None]
    sc = sc.masked_fill(~seen[:, None, :, None, :], -math.inf)
    m = sc.amax(4, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = (sc - m).exp_()
    del sc
    l = p.sum(4, keepdim=True)
    v = s["v"][0][page, :, (at % P).expand(B, Lm)].float()
    y = (p.view(B, G, N * (H // G), Lm) @ v.permute(0, 2, 1, 3)).view(B, G, N, H // G, D) / torch.where(l == 0, torch.ones_like(l), l)
    s["o"].copy_(y.permute(0, 2, 1, 3, 4).reshape(B, N, H * D)[req, j])
    s["lse"].copy_((m + l.log()).squeeze(4).permute(0, 2, 1, 3).reshape(B, N, H)[req, j])


def plain_commit(s):
    c, o = s["c"], s["out"]
    B, N, P, T = c["reqs"], s["n_max"], c["page"], s["T"]
    dev = dict(device="cuda")
    req = o["row_req"].long()
    cu = o["cu_rows"].long()
    j = torch.arange(T, **dev) - cu[req]
    par = s["parent"].long()
    # a node matches when its token is the model's choice at its parent; the first such child goes on
    want = torch.where((par >= 0)[:, None], s["targets"][cu[req] + par.clamp(min=0)], s["root"][req])
    match = (want == s["tokens"]).all(1)
    key = torch.where(match, req * (N + 1) + par + 1, B * (N + 1))
    first = torch.full((B * (N + 1) + 1,), T, dtype=torch.int64, **dev).scatter_reduce(0, key, j, "amin")
    on = match & (first[key] == j)
    # on the path: the node and all its ancestors
    A = torch.zeros((B, N, N), dtype=torch.float32, **dev)
    bit = (o["mask"][:, :, None] >> torch.arange(64, **dev)) & 1
    A[req, j] = bit.reshape(T, -1)[:, :N].float()
    ok = torch.zeros((B, N), dtype=torch.float32, **dev)
    ok[req, j] = on.float()
    hits = (A @ ok[:, :, None]).squeeze(2)[req, j]
    depth = o["pos"].long() - s["ctx"].long()[req]
    on = hits == (depth + 1).float()
    n = torch.zeros(B, dtype=torch.int64, **dev).scatter_add(0, req, on.long())
    s["path"].fill_(-1)
    s["path"][(cu[req] + depth)[on]] = j[on].int()
    s["n_acc"].copy_(n)
    s["new_len"].copy_(s["ctx"] + n)
    last = s["path"].long()[(cu[:B] + n - 1).clamp(min=0)]
    s["nxt"].copy_(torch.where((n > 0)[:, None], s["targets"][(cu[:B] + last.clamp(min=0)).clamp(max=T - 1)], s["root"]))
    src, dst = o["slot"][on], o["slot"][(cu[req] + depth)[on]]
    for pool in (s["k"], s["v"]):
        pool[:, dst // P, :, dst % P] = pool[:, src // P, :, src % P]


# ---- the definitions in 64 bits -----------------------------------------------------------------

def exact(c, seed):
    if c["op"] == "plan":
        return None                                                     # whole numbers only
    s = prepare(c, seed)
    o = {k: v.cpu() for k, v in s["out"].items()}
    D, P, H, G = c["dim"], c["page"], c["heads"], c["kv_heads"]
    cu, ctx = o["cu_rows"].tolist(), s["ctx"].tolist()
    if c["op"] == "store":
        x = s["qkv"].double().view(-1, H + 2 * G, D)

        def norm_rope(v, w):
            v = v / torch.sqrt((v ** 2).sum(-1, keepdim=True) / D + EPS) * w.double()
            z = torch.complex(v[..., :D // 2], v[..., D // 2:])
            rot = s["rope"].double()[s["out"]["pos"].long()]
            z = z * torch.complex(rot[:, :D // 2], rot[:, D // 2:])[:, None, :]
            return torch.cat([z.real, z.imag], -1)

        k, v = s["k"].double(), s["v"].double()
        kn = norm_rope(x[:, H:H + G], s["k_norm"])
        slot = s["out"]["slot"]
        k[0].permute(0, 2, 1, 3)[slot // P, slot % P] = kn
        v[0].permute(0, 2, 1, 3)[slot // P, slot % P] = x[:, H + G:]
        return [norm_rope(x[:, :H], s["q_norm"]).reshape(-1, H * D), k, v]
    if c["op"] == "attend":
        out = torch.zeros((s["T"], H * D), dtype=torch.float64, device="cuda")
        lse = torch.zeros((s["T"], H), dtype=torch.float64, device="cuda")
        parent = s["parent"].tolist() if c["tree"] else None
        for i in range(c["reqs"]):
            a, b = cu[i], cu[i + 1]
            if a == b:
                continue
            n, L = b - a, ctx[i] + b - a
            pages = s["table"][i, :-(-L // P)].long()
            k = s["k"][0][pages].transpose(0, 1).reshape(G, -1, D)[:, :L].double()
            v = s["v"][0][pages].transpose(0, 1).reshape(G, -1, D)[:, :L].double()
            seen = torch.ones((n, L), dtype=torch.bool)
            if parent is not None:
                seen[:, ctx[i]:] = False
                for r in range(n):
                    if parent[a + r] >= 0:
                        seen[r, ctx[i]:] = seen[parent[a + r], ctx[i]:]
                    seen[r, ctx[i] + r] = True
            else:
                seen = seen.tril(ctx[i])
            seen = seen.cuda()
            q = s["q"][a:b].double().view(n, H, D)
            for h in range(H):
                sc = (q[:, h] @ k[h // (H // G)].T / math.sqrt(D)).masked_fill(~seen, -math.inf)
                lse[a:b, h] = torch.logsumexp(sc, 1)
                out[a:b, h * D:(h + 1) * D] = torch.softmax(sc, 1) @ v[h // (H // G)]
        return [out, lse]
    parent, tokens, targets, root = s["parent"].tolist(), s["tokens"].tolist(), s["targets"].tolist(), s["root"].tolist()
    src, dst = [], []
    for i in range(c["reqs"]):
        at, want, walked = -1, root[i], 0
        while True:
            child = next((r for r in range(cu[i + 1] - cu[i]) if parent[cu[i] + r] == at and tokens[cu[i] + r] == want), None)
            if child is None:
                break
            src.append(int(o["slot"][cu[i] + child]))
            dst.append(int(o["slot"][cu[i] + walked]))
            at, want, walked = child, targets[cu[i] + child], walked + 1
    src, dst = torch.tensor(src, dtype=torch.int64, device="cuda"), torch.tensor(dst, dtype=torch.int64, device="cuda")
    got = []
    for pool in (s["k"], s["v"]):
        rows = pool.double().permute(0, 1, 3, 2, 4).reshape(c["layers"], -1, G, D)
        rows[:, dst] = rows[:, src]
        got.append(rows.view(c["layers"], -1, P, G, D).permute(0, 1, 3, 2, 4))
    return [None, None, None, None] + got
