"""Performance cases of the ops that a program with its own loop over several
requests calls: pages for their tokens, head norms with the rotation and the
append to the paged cache, attention of the new rows over it, and the check of
drafted tokens.

``run`` calls the library where ``own`` is true. Where it is false it computes
the same from elementary torch operations in 32 bits (angles, sums of
probabilities and comparisons next to a border in 64), for every kind of case:

* ``assign``  -- one step's growth of every request and the roll back behind
  it (two calls, after which the pages are as before);
* ``norm``    -- q, k, v rows of a projection to rotated q and cache rows;
* ``attend``  -- new rows of every request over its cached ones;
* ``verify``  -- drafted tokens against the target's probabilities.

Heads and head sizes are those of the decoders named in ``vvli_amd.config``.
Lengths are spread between requests by a fixed rule of the case; values, the
order of pages and the random numbers come from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HEADS = [(32, 8, 64), (14, 2, 64), (28, 4, 128), (16, 16, 128)]  # heads, kv heads, head size
EPS = 1e-6
THETA = 500000.0


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed() -> list:
    return [
        # Pages of one decode step of a batch: the smallest call of a step.
        dict(name="assign-decode-48", kind="assign", R=48, ctx=2000, new=1, ps=16, short=0),
        # Prompts that start together: many rows, more pages, some requests
        # that the pool has no room for.
        dict(name="assign-prompts-300", kind="assign", R=300, ctx=900, new=130, ps=32, short=40),
        # One token of one request (Llama-3.2-1B heads), f32 cache: latency.
        dict(name="norm-1row-f32", kind="norm", rows=1, heads=32, kv=8, hd=64, cache="f32", norm=False, split=False, ps=16),
        # Drafts of a batch (Qwen2.5-7B heads), odd rows.
        dict(name="norm-75rows-bf16", kind="norm", rows=75, heads=28, kv=4, hd=128, cache="bf16", norm=True, split=True, ps=16),
        # The rows of long prompts, f16 cache.
        dict(name="norm-6000rows-f16", kind="norm", rows=6000, heads=28, kv=4, hd=128, cache="f16", norm=True, split=True, ps=64),
        # One request's decode step behind a chat turn, f32 cache: latency.
        dict(name="attend-1x1-f32", kind="attend", R=1, ctx=230, new=1, heads=32, kv=8, hd=64, cache="f32", ps=16, window=0),
        # Decode of a batch behind long contexts: the cache read once.
        dict(name="attend-40x1-bf16", kind="attend", R=40, ctx=8000, new=1, heads=28, kv=4, hd=128, cache="bf16", ps=16, window=0),
        # Five rows (a token and its drafts) of each request, f16 cache.
        dict(name="attend-24x5-f16", kind="attend", R=24, ctx=4100, new=5, heads=32, kv=8, hd=64, cache="f16", ps=64, window=0),
        # Prompt chunks behind cached text, bf16 cache: matrix-core work.
        dict(name="attend-2x2000-bf16", kind="attend", R=2, ctx=2100, new=2000, heads=28, kv=4, hd=128, cache="bf16", ps=32, window=0),
        # Chunks in f32 throughout, behind a window shorter than the context.
        dict(name="attend-3x333-f32", kind="attend", R=3, ctx=1700, new=333, heads=14, kv=2, hd=64, cache="f32", ps=48, window=1000),
        # Drafts of one request against the whole vocabulary.
        dict(name="verify-1x4", kind="verify", R=1, D=4, V=151936, certain=False),
        # Drafts of a batch.
        dict(name="verify-64x4", kind="verify", R=64, D=4, V=128256, certain=False),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["assign", "norm", "attend", "attend", "attend", "verify"])
    if kind == "assign":
        new = rng.choice([1, rng.randint(2, 8), _log_int(rng, 8, 200)])
        return dict(kind=kind, R=_log_int(rng, 1, 200 if new > 100 else 1500), ctx=_log_int(rng, 1, 4000), new=new,
                    ps=rng.choice([1, 16, 16, 24, 32, 64, 256]), short=rng.choice([0, 0, rng.randint(1, 60)]))
    h, kv, hd = rng.choice(HEADS)
    cache = rng.choice(["f32", "bf16", "f16"])
    ps = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if kind == "norm":
        return dict(kind=kind, rows=_log_int(rng, 1, 3000 if h * hd > 2048 else 6000), heads=h, kv=kv, hd=hd, cache=cache,
                    norm=rng.random() < 0.7, split=rng.random() < 0.6, ps=ps)
    if kind == "verify":
        return dict(kind=kind, R=_log_int(rng, 1, 60), D=rng.randint(0, 4), V=_log_int(rng, 1000, 128256),
                    certain=rng.random() < 0.3)
    window = rng.choice([0, 0, 0, _log_int(rng, 1, 4000)])
    what = rng.choice(["step", "drafts", "chunks"])
    if what == "step":
        R, ctx, new = _log_int(rng, 1, 40), _log_int(rng, 1, 8000), 1
        if cache == "f32" or hd == 64 or kv == 16:
            R = min(R, 20)
    elif what == "drafts":
        R, ctx, new = _log_int(rng, 1, 24), _log_int(rng, 1, 4100), rng.randint(2, 12)
        if kv == 16:
            R = min(R, 8)
    else:
        R, ctx, new = _log_int(rng, 1, 8), _log_int(rng, 1, 2500), _log_int(rng, 13, 1500)
        R = max(1, min(R, 3000 // new))
    return dict(kind=kind, R=R, ctx=ctx, new=new, heads=h, kv=kv, hd=hd, cache=cache, ps=ps, window=window)


def _lengths(case) -> tuple:
    """(cached tokens, new rows) of every request: fixed by the case."""
    R, ctx, new = case["R"], case["ctx"], case["new"]
    r = np.random.RandomState((R * 1009 + ctx * 31 + new) % (1 << 31))
    past = r.randint(ctx // 4, ctx + 1, R)
    past[-1] = ctx
    add = np.full(R, new) if new <= 1 else r.randint(1, new + 1, R)
    add[-1] = new
    if R >= 3:
        add[1] = 0    # a request that waits
        past[0] = 0   # one that starts
    return past.astype(np.int64), add.astype(np.int64)


def _rows(case) -> int:
    """Rows of the batch: the requests' and a few behind them that stay as they were."""
    return int(_lengths(case)[1].sum()) + case["R"] % 3


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _i32(x) -> torch.Tensor:
    return torch.as_tensor(np.ascontiguousarray(x), dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------------------
# prepare
# ---------------------------------------------------------------------------
def _tables(past, add, ps: int, seed: int) -> tuple:
    """(table [R, stride] with every request's pages in a random order, page count)."""
    need = -(-(past + add) // ps)
    pages = int(need.sum()) + 3
    order = np.random.RandomState(seed % (1 << 31)).permutation(pages)
    stride = int(need.max()) + 2
    table = np.full((len(past), stride), -1, np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return table, pages


def _prepare_assign(case, seed: int) -> dict:
    past, add = _lengths(case)
    R, ps = case["R"], case["ps"]
    table, pages = _tables(past, add * 0, ps, seed)
    grown = int((-(-(past + add) // ps) + (past // -ps)).sum())  # pages that the step takes
    stride = int((-(-(past + add) // ps)).max()) + 2
    full = np.full((R, stride), -1, np.int32)
    m = min(stride, table.shape[1])
    full[:, :m] = table[:, :m]
    free = max(0, grown * (100 - case["short"]) // 100)
    stack = np.full(pages + free, -1, np.int32)
    stack[:free] = pages + np.random.RandomState((seed + 1) % (1 << 31)).permutation(free)
    rows = _rows(case)
    st = dict(ps=ps, pages=pages + free, stack=_i32(stack), count=_i32([free]), table=_i32(full), past=_i32(past), add=_i32(add),
              none=_i32(np.zeros(R)), len1=_i32(np.zeros(R)), len2=_i32(np.zeros(R)), row_start=_i32(np.zeros(R + 1)),
              start=_i32(np.zeros(R)), pos=_i32(np.full(rows, -7)), slots=torch.full((rows,), -7, dtype=torch.int64, device=DEV),
              row_start2=_i32(np.zeros(R + 1)), start2=_i32(np.zeros(R)))
    return st


def _prepare_norm(case, seed: int) -> dict:
    g = _gen(seed)
    T, H, K, d = case["rows"], case["heads"], case["kv"], case["hd"]
    width = (H + 2 * K) * d
    qkv = torch.randn(T, width, device=DEV, generator=g) * 1.5
    pages = -(-(T + 5) // case["ps"])
    n = pages * case["ps"]
    r = np.random.RandomState(seed % (1 << 31))
    slots = r.permutation(n)[:T].astype(np.int64)
    if T >= 8:
        slots[3] = -1  # a row that the pool had no room for
    pos = r.randint(0, 120000, T)
    weight = lambda: (1 + 0.2 * torch.randn(d, device=DEV, generator=g)).bfloat16() if case["norm"] else None  # noqa: E731
    t = TYPES[case["cache"]]
    return dict(qkv=qkv, q_norm=weight(), k_norm=weight(), pos=_i32(pos), slots=torch.as_tensor(slots, device=DEV),
                inv=(THETA ** -(torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)).float(),
                k=torch.zeros(n, K, d, device=DEV, dtype=t), v=torch.zeros(n, K, d, device=DEV, dtype=t),
                q=torch.zeros(T, H * d, device=DEV), pages=pages)


def _prepare_attend(case, seed: int) -> dict:
    past, add = _lengths(case)
    g = _gen(seed)
    H, K, d = case["heads"], case["kv"], case["hd"]
    table, pages = _tables(past, add, case["ps"], seed)
    n = pages * case["ps"]
    t = TYPES[case["cache"]]
    rows = _rows(case)
    row_start = np.concatenate([[0], np.cumsum(add)])
    return dict(q=torch.randn(rows, H * d, device=DEV, generator=g) * 1.3, out=torch.zeros(rows, H * d, device=DEV),
                k=torch.randn(n, K, d, device=DEV, generator=g).to(t), v=torch.randn(n, K, d, device=DEV, generator=g).to(t),
                table=_i32(table), row_start=_i32(row_start), start=_i32(past), pages=pages, rows=rows, scale=d ** -0.5,
                most=int((past + add).max()), most_new=int(add.max()))


def _prepare_verify(case, seed: int) -> dict:
    g = _gen(seed)
    R, D, V = case["R"], case["D"], case["V"]
    counts = np.random.RandomState(R * 7 + D).randint(0, D + 1, R) + 1
    counts[-1] = D + 1
    if R >= 3:
        counts[1] = 0  # a request without rows
    row_start = np.concatenate([[0], np.cumsum(counts)])
    rows = int(row_start[-1]) + R % 3
    logits = 3.0 * torch.randn(rows, V, device=DEV, generator=g)
    target = torch.softmax(logits, -1)
    tokens = torch.zeros(rows, dtype=torch.int32, device=DEV)
    logits += 0.7 * torch.randn(rows, V, device=DEV, generator=g)
    draft = torch.softmax(logits, -1)
    drawn = (draft / torch.empty_like(draft).exponential_(generator=g)).argmax(-1)
    tokens[1:] = drawn[:-1].int()
    return dict(target=target, draft=None if case["certain"] else draft, tokens=tokens, row_start=_i32(row_start),
                u=torch.rand(rows, device=DEV, generator=g), us=torch.rand(R, device=DEV, generator=g),
                accepted=_i32(np.zeros(R)), out=_i32(np.full(rows, -9)), most=D + 1)


def prepare(case, seed: int) -> dict:
    st = {"assign": _prepare_assign, "norm": _prepare_norm, "attend": _prepare_attend, "verify": _prepare_verify}[case["kind"]](
        case, seed)
    st["case"] = case
    st["stream"] = torch.cuda.current_stream().cuda_stream
    st["kept"] = {}  # handles and workspaces that the program keeps from call to call
    return st


# ---------------------------------------------------------------------------
# The library's calls
# ---------------------------------------------------------------------------
def _p(t) -> int | None:
    return None if t is None else t.data_ptr()


def _cache(st, R):
    if "cache" not in st["kept"]:
        c = st["case"]
        st["kept"]["cache"] = R.PagedCache(_p(st["k"]), _p(st["v"]), c["cache"], c["kv"], c["hd"], c["ps"], st["pages"])
    return st["kept"]["cache"]


def _workspace(st, size: int):
    if "workspace" not in st["kept"]:
        st["kept"]["workspace"] = torch.zeros(max(1, size), dtype=torch.uint8, device=DEV)
    return st["kept"]["workspace"]


def _own(st):
    from vvli_amd import runtime as R

    c = st["case"]
    if c["kind"] == "assign":
        if "pool" not in st["kept"]:
            st["kept"]["pool"] = R.PagePool(_p(st["stack"]), _p(st["count"]), _p(st["table"]), c["R"], st["table"].shape[1],
                                            st["ps"], st["pages"])
        pool, rows = st["kept"]["pool"], st["pos"].numel()
        R.paged_assign(pool, _p(st["past"]), _p(st["past"]), _p(st["add"]), rows, _p(st["len1"]), _p(st["row_start"]),
                       _p(st["start"]), _p(st["pos"]), _p(st["slots"]), st["stream"])
        R.paged_assign(pool, _p(st["len1"]), _p(st["past"]), _p(st["none"]), 0, _p(st["len2"]), _p(st["row_start2"]),
                       _p(st["start2"]), None, None, st["stream"])
        return _assigned(st)
    if c["kind"] == "norm":
        H, K, d, T = c["heads"], c["kv"], c["hd"], c["rows"]
        base, ld = _p(st["qkv"]), (H + 2 * K) * d
        R.norm_rope_append(_cache(st, R), base, ld, base + 4 * H * d, ld, base + 4 * (H + K) * d, ld, T, H, _p(st["q"]), H * d,
                           _p(st["inv"]), _p(st["pos"]), _p(st["slots"]), "split_half" if c["split"] else "interleaved",
                           _p(st["q_norm"]), _p(st["k_norm"]), EPS, st["stream"])
        return {"q": st["q"], "k": st["k"], "v": st["v"]}
    if c["kind"] == "attend":
        ws = _workspace(st, R.paged_attention_workspace(st["rows"], c["R"], c["heads"], c["kv"], c["hd"]))
        ld = c["heads"] * c["hd"]
        R.paged_attention(_cache(st, R), _p(st["table"]), st["table"].shape[1], _p(st["row_start"]), _p(st["start"]), c["R"],
                          _p(st["q"]), ld, _p(st["out"]), ld, st["rows"], c["heads"], st["scale"], c["window"], ws.data_ptr(),
                          ws.numel(), st["stream"])
        return {"out": st["out"]}
    ws = _workspace(st, R.verify_drafts_workspace(c["R"], c["V"]))
    R.verify_drafts(_p(st["target"]), c["V"], _p(st["draft"]), c["V"], _p(st["tokens"]), _p(st["row_start"]), c["R"],
                    st["tokens"].numel(), c["V"], _p(st["u"]), _p(st["us"]), _p(st["accepted"]), _p(st["out"]), ws.data_ptr(),
                    ws.numel(), st["stream"])
    return {"accepted": st["accepted"], "tokens": st["out"]}


def _assigned(st) -> dict:
    return {k: st[k] for k in ("len1", "row_start", "start", "pos", "slots", "len2", "table", "stack", "count")}


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _plain_assign(st, held, keep, add, pos_out, slots_out):
    """One call: (lengths, row_start, start); stack, count, table, pos_out and slots_out change in place."""
    ps, pages = st["ps"], st["pages"]
    table = st["table"].long()
    R, stride = table.shape
    rows = 0 if pos_out is None else pos_out.numel()
    held, keep, add = held.long(), keep.long(), add.long()
    n = add.clamp(min=0)
    row_end = n.cumsum(0)
    ok = (add >= 0) & (keep >= 0) & (keep <= held) & (keep + add <= stride * ps) & (row_end <= rows)
    have, want = (held + ps - 1) // ps, (keep + add + ps - 1) // ps
    need, give = ((want - have).clamp(min=0) * ok), ((have - want).clamp(min=0) * ok)
    need_end, give_end = need.cumsum(0), give.cumsum(0)
    avail = st["count"].long() + give_end[-1]
    served = ok & ((need == 0) | (need_end <= avail))
    col = torch.arange(stride, device=DEV)
    # Given pages, the first on top of the stack; `pages` is a place for what is not one.
    stack = torch.cat([st["stack"].long(), torch.full((1,), -1, device=DEV)])
    given = ok[:, None] & (col >= want[:, None]) & (col < have[:, None])
    at = avail - 1 - ((give_end - give)[:, None] + col - want[:, None])
    stack[torch.where(given, at, pages)] = torch.where(given, table, -1)
    table = torch.where(given, -1, table)
    taken = served[:, None] & (col >= have[:, None]) & (col < want[:, None])
    at = avail - 1 - ((need_end - need)[:, None] + col - have[:, None])
    table = torch.where(taken, stack[torch.where(taken, at, pages)], table)
    st["stack"].copy_(stack[:pages])
    st["count"].copy_(avail - (need * served).sum())
    st["table"].copy_(table)
    row_start = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), row_end]).clamp(max=rows)
    if rows:
        i = torch.arange(rows, device=DEV)
        r = torch.searchsorted(row_start[1:].contiguous(), i, right=True)
        there = r < R
        r = r.clamp(max=R - 1)
        p = keep[r] + i - row_start[r]
        page = table[r, (p // ps).clamp(0, stride - 1)]
        good = served[r] & (page >= 0) & (page < pages)
        pos_out.copy_(torch.where(there, torch.where(served[r], p, -1), pos_out.long()))
        slots_out.copy_(torch.where(there, torch.where(good, page * ps + p % ps, -1), slots_out))
    return torch.where(served, keep + add, held).int(), row_start.int(), torch.where(served, keep, -n).int()


def _plain_norm(st, f=torch.float32):
    c = st["case"]
    H, K, d, T = c["heads"], c["kv"], c["hd"], c["rows"]
    q, k, v = st["qkv"].to(f).view(T, H + 2 * K, d).split([H, K, K], 1)
    if st["q_norm"] is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + EPS) * st["q_norm"].to(f)
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + EPS) * st["k_norm"].to(f)
    angle = st["pos"].double()[:, None] * st["inv"].double()
    cos, sin = angle.cos().to(f)[:, None], angle.sin().to(f)[:, None]

    def turn(x):
        if c["split"]:
            a, b = x[..., : d // 2], x[..., d // 2:]
            return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)

    return turn(q).reshape(T, H * d), turn(k), v


def _plain_attend(st):
    c = st["case"]
    H, K, d, R, ps = c["heads"], c["kv"], c["hd"], c["R"], c["ps"]
    G, L, N = H // K, st["most"], st["most_new"]
    j, i = torch.arange(L, device=DEV), torch.arange(N, device=DEV)
    start, first = st["start"].long(), st["row_start"].long()
    count = first[1:] - first[:-1]
    page = st["table"].long()[:, j // ps]
    slot = (page * ps + j % ps).clamp(min=0)
    there = (j < (start + count)[:, None]) & (page >= 0)                               # [R, L]
    k = (st["k"][slot].float() * there[..., None, None]).permute(0, 2, 3, 1).contiguous()  # [R, K, d, L]
    v = (st["v"][slot].float() * there[..., None, None]).permute(0, 2, 1, 3).contiguous()
    row = first[:-1, None] + i                                                         # [R, N]
    used = i < count[:, None]
    q = st["q"][torch.where(used, row, 0)].view(R, N, K, G, d).permute(0, 2, 3, 1, 4).reshape(R, K, G * N, d)
    s = torch.matmul(q, k).view(R, K, G, N, L) * st["scale"]
    pos = start[:, None] + i
    seen = there[:, None] & (j <= pos[..., None])
    if c["window"]:
        seen &= j > pos[..., None] - c["window"]
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-3e38)
    s = s.sub_(top).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(R, K, G * N, L), v).view(R, K, G, N, d) / total.clamp(min=1e-30)
    o = o.permute(0, 3, 1, 2, 4).reshape(R * N, H * d)
    rows = st["rows"]
    out = torch.cat([st["out"], st["out"][:1]])  # a last row for what is no request's
    out[torch.where(used, row, rows).view(-1)] = o
    st["out"].copy_(out[:rows])
    return {"out": st["out"]}


def _plain_verify(st):
    n, V = st["most"], st["target"].shape[1]
    first = st["row_start"].long()
    count = (first[1:] - first[:-1])[:, None]
    i = torch.arange(n, device=DEV)
    rows = st["tokens"].numel()
    row = (first[:-1, None] + i).clamp(max=rows - 1)
    tested = i < count - 1
    token = st["tokens"].long()[(row + 1).clamp(max=rows - 1)]
    real = (token >= 0) & (token < V)
    token = token.clamp(0, V - 1)
    p = torch.where(real, st["target"][row, token], 0).double()
    q = torch.ones_like(p) if st["draft"] is None else torch.where(real, st["draft"][row, token], 0).double()
    ok = tested & (st["u"][row].double() * q < p)
    accepted = ok.long().cumprod(1).sum(1)
    stop = (first[:-1] + accepted).clamp(max=rows - 1)
    weight = st["target"][stop].double()
    if st["draft"] is None:
        hot = torch.arange(V, device=DEV) == token.gather(1, accepted[:, None].clamp(max=n - 1))
        less = weight * ~hot
    else:
        less = weight - st["draft"][stop].double()
    weight, less = (torch.where((w > 0) & (w < math.inf), w, 0) for w in (weight, less))
    left = (accepted < count[:, 0] - 1) & (less.sum(1) > 0)
    sums = torch.where(left[:, None], less, weight).cumsum(1)
    total = sums[:, -1:]
    found = (sums <= st["us"].double()[:, None] * total).sum(1)
    found = torch.minimum(found, (sums < total).sum(1))
    found = torch.where(total[:, 0] > 0, found, -1)
    given = torch.where(i < accepted[:, None], token, torch.where(i == accepted[:, None], found[:, None], -1))
    out = torch.cat([st["out"].long(), st["out"][:1].long()])
    out[torch.where(i < count, row, rows)] = given
    st["out"].copy_(out[:rows])
    st["accepted"].copy_(accepted)
    return {"accepted": st["accepted"], "tokens": st["out"]}


def run(st):
    if own:
        return _own(st)
    kind = st["case"]["kind"]
    if kind == "assign":
        a = _plain_assign(st, st["past"], st["past"], st["add"], st["pos"], st["slots"])
        st["len1"], st["row_start"], st["start"] = a
        st["len2"], _, _ = _plain_assign(st, a[0], st["past"], st["none"], None, None)
        return _assigned(st)
    if kind == "norm":
        q, k, v = _plain_norm(st)
        st["q"].copy_(q)
        n = st["k"].shape[0]
        at = torch.where(st["slots"] < 0, n, st["slots"])
        for pool, x in (("k", k), ("v", v)):
            st[pool].copy_(torch.cat([st[pool], st[pool][:1]]).index_copy_(0, at, x.to(st[pool].dtype))[:n])
        return {"q": st["q"], "k": st["k"], "v": st["v"]}
    return _plain_attend(st) if kind == "attend" else _plain_verify(st)


# ---------------------------------------------------------------------------
# work
# ---------------------------------------------------------------------------
def work(case) -> dict:
    kind = case["kind"]
    if kind == "assign":
        past, add = _lengths(case)
        R, rows, ps = case["R"], _rows(case), case["ps"]
        moved = int((-(-(past + add) // ps) + (past // -ps)).sum())
        return {"bytes": 2 * (4 * R * 7) + 12 * rows + 4 * 4 * moved, "flops": 0}
    e = {"f32": 4, "bf16": 2, "f16": 2}.get(case.get("cache"))
    if kind == "norm":
        T, H, K, d = case["rows"], case["heads"], case["kv"], case["hd"]
        return {"bytes": T * ((H + 2 * K) * d * 4 + H * d * 4 + 2 * K * d * e + 12), "flops": T * (H + K) * d * 8}
    if kind == "attend":
        past, add = _lengths(case)
        H, K, d, w = case["heads"], case["kv"], case["hd"], case["window"] or 1 << 40
        keys = sum(int(min(p + n, w + n - 1)) for p, n in zip(past, add) if n)
        pairs = sum(int(np.minimum(p + 1 + np.arange(n), w).sum()) for p, n in zip(past, add))
        return {"bytes": 2 * keys * K * d * e + 2 * int(add.sum()) * H * d * 4, "flops": 4 * pairs * H * d}
    # One row of target probabilities for each request's last token; of about
    # half of the requests the draft's row too (a draft of theirs is refused).
    share = 0.5 if not case["certain"] and case["D"] else 0.0
    return {"bytes": case["R"] * case["V"] * 4 * (1 + share), "flops": case["R"] * case["V"]}


# ---------------------------------------------------------------------------
# The results in 64 bits
# ---------------------------------------------------------------------------
def _exact_norm(case, st) -> dict:
    """Pair by pair through complex numbers: each pair times exp(i pos f)."""
    H, K, d, T = case["heads"], case["kv"], case["hd"], case["rows"]
    x = st["qkv"].double().view(T, H + 2 * K, d)
    turn = torch.polar(torch.ones(T, d // 2, dtype=torch.float64, device=DEV), st["pos"].double()[:, None] * st["inv"].double())
    heads = x[:, : H + K].clone()
    if case["norm"]:
        heads /= heads.square().mean(-1, keepdim=True).add(EPS).sqrt()
        heads[:, :H] *= st["q_norm"].double()
        heads[:, H:] *= st["k_norm"].double()
    pair = heads.view(T, H + K, 2, d // 2).transpose(2, 3) if case["split"] else heads.view(T, H + K, d // 2, 2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn[:, None])
    y = (z.transpose(2, 3) if case["split"] else z).reshape(T, H + K, d)
    k, v = st["k"].double(), st["v"].double()
    for t, s in enumerate(st["slots"].tolist()):
        if s >= 0:
            k[s], v[s] = y[t, H:], x[t, H + K:]
    return {"q": y[:, :H].reshape(T, H * d), "k": k, "v": v}


def _exact_attend(case, st) -> dict:
    """Request by request, kv head by kv head."""
    H, K, d, ps = case["heads"], case["kv"], case["hd"], case["ps"]
    out = st["out"].double()
    past, add = _lengths(case)
    row = 0
    for r, (p, n) in enumerate(zip(past.tolist(), add.tolist())):
        if not n:
            continue
        j = torch.arange(p + n, device=DEV)
        slot = st["table"][r].long()[j // ps] * ps + j % ps
        pos = p + torch.arange(n, device=DEV)
        hidden = j[None] > pos[:, None]
        if case["window"]:
            hidden |= j[None] <= pos[:, None] - case["window"]
        for h in range(K):
            q = st["q"][row:row + n].double().view(n, K, H // K, d)[:, h].transpose(0, 1)
            s = torch.matmul(q, st["k"][slot, h].double().t().contiguous()) * st["scale"]
            w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            o = torch.matmul(w, st["v"][slot, h].double())
            out[row:row + n].view(n, K, H // K, d)[:, h] = o.transpose(0, 1)
        row += n
    return {"out": out}


def exact(case, seed: int):
    if case["kind"] not in ("norm", "attend"):
        return None  # whole numbers
    return {"norm": _exact_norm, "attend": _exact_attend}[case["kind"]](case, prepare(case, seed))
