"""Ops for several requests over a paged cache on the GPU, against plain
implementations in 64 bits.

Tolerances (u = 2^-24, half a step of f32 relative to the value):

* ``norm_rope_append``: the sum of squares passes at most 8 rounded additions
  and one product, the root, quotient and the products by it and the weight one
  each (a half of the sum's error reaches the root): under 9 u; cos and sin are
  off by at most 2 u of 1, the two products and their sum by 3 u: 16 u = 2^-20
  of |a| + |b| for the pair (a, b). A cache value adds half a step of its type.
* ``paged_attention``: a score is a sum of hd products, off by at most
  (hd + 8) u of sum |scale q_d k_d| =: S whatever the order (8: scale, split
  terms and their sums); a weight is exp of it, off by that and 4 u; sums over
  n keys add (n + 16) u. Numerator and sum both carry them:
  |error| <= 2 ((hd + 8) max S + n + 24) u * sum p_j |v_j|. The f16 cache's
  two-term split leaves 2^-22 of a term instead of u: 4 u more a product, which
  (hd + 8) covers from hd = 32 on for S >= the largest single product.
  The worst case lets an error hide that is systematic, so the 2-norm over all
  outputs is held to 1e-6 too: rounding errors of either sign grow with the
  root of their number, 4 sqrt(hd + n) u < 1.1e-5 / 10 for hd + n <= 2000 and
  scores of unit size.
"""

import numpy as np
import pytest

from vvli_amd import config as C
from vvli_amd import runtime as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # relative, at most


@pytest.fixture(scope="module")
def torch():
    import torch as t

    return t


def types(torch):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def ptr(t):
    return None if t is None else t.data_ptr()


def i32(torch, x):
    return torch.tensor(np.ascontiguousarray(x, dtype=np.int32), device="cuda")


# ---------------------------------------------------------------------------
# paged_assign
# ---------------------------------------------------------------------------
def plain_assign(stack, table, ps, pages, held, keep, add, rows):
    """The definition, request by request, on lists. Returns (len, row_start, start, pos, slots); stack (top last) and table change."""
    n_req, stride = table.shape
    n = [max(0, int(a)) for a in add]
    ends = np.cumsum(n)
    ok = [add[r] >= 0 and 0 <= keep[r] <= held[r] and held[r] <= stride * ps and keep[r] + add[r] <= stride * ps and ends[r] <= rows
          for r in range(n_req)]
    have = [-(-int(h) // ps) for h in held]
    want = [-(-int(keep[r] + add[r]) // ps) for r in range(n_req)]
    given = []
    for r in range(n_req):
        if ok[r]:
            for c in range(want[r], have[r]):
                given.append(int(table[r, c]))
                table[r, c] = -1
    stack += given[::-1]
    length, start, dry = [], [], False
    for r in range(n_req):
        need = max(0, want[r] - have[r]) if ok[r] else 0
        if need and (dry or need > len(stack)):
            dry = True
            ok[r] = False
        if ok[r]:
            for c in range(have[r], have[r] + need):
                table[r, c] = stack.pop()
        length.append(int(keep[r] + add[r]) if ok[r] else int(held[r]))
        start.append(int(keep[r]) if ok[r] else -n[r])
    row_start = [0] + [int(min(e, rows)) for e in ends]
    pos, slots = [], []
    for r in range(n_req):
        for i in range(row_start[r + 1] - row_start[r]):
            p = start[r] + i if ok[r] else -1
            page = int(table[r, p // ps]) if p >= 0 else -1
            pos.append(p)
            slots.append(page * ps + p % ps if 0 <= page < pages else -1)
    return length, row_start, start, pos, slots


class Pool:
    """A pool on the device beside the plain one."""

    def __init__(self, torch, n_req, stride, ps, pages, seed=0):
        self.torch, self.ps, self.pages = torch, ps, pages
        self.stack = np.random.RandomState(seed).permutation(pages).tolist()
        self.table = np.full((n_req, stride), -1, np.int64)
        self.d_stack, self.d_count, self.d_table = i32(torch, self.stack), i32(torch, [pages]), i32(torch, self.table)
        self.handle = R.PagePool(ptr(self.d_stack), ptr(self.d_count), ptr(self.d_table), n_req, stride, ps, pages)
        self.d_len = i32(torch, np.zeros(n_req))
        self.n_req = n_req

    def step(self, held, keep, add, rows, sync=True):
        torch = self.torch
        out = dict(len=self.d_len, row_start=i32(torch, np.full(self.n_req + 1, -5)), start=i32(torch, np.full(self.n_req, -5)),
                   pos=i32(torch, np.full(rows + 3, -7)), slots=torch.full((rows + 3,), -7, dtype=torch.int64, device="cuda"))
        d = [i32(torch, x) for x in (held, keep, add)]
        R.paged_assign(self.handle, *map(ptr, d), rows, ptr(out["len"]), ptr(out["row_start"]), ptr(out["start"]),
                       ptr(out["pos"]), ptr(out["slots"]), torch.cuda.current_stream().cuda_stream)
        want = plain_assign(self.stack, self.table, self.ps, self.pages, held, keep, add, rows)
        got = {k: v.cpu().numpy() for k, v in out.items()}
        for name, w in zip(("len", "row_start", "start", "pos", "slots"), want):
            g = got[name]
            assert g[:len(w)].tolist() == list(w), name
            assert (g[len(w):] == -7).all(), f"{name}: rows behind the last were written"
        count = int(self.d_count.item())
        assert count == len(self.stack)
        assert self.d_stack[:count].tolist() == self.stack
        assert self.d_table.cpu().numpy().tolist() == self.table.tolist()
        return got["len"]


@pytest.mark.parametrize("n_req,stride,ps,pages", [(1, 4, 16, 6), (5, 9, 1, 30), (67, 12, 24, 300), (300, 40, 16, 2000),
                                                   (1024, 3, 8, 2000), (1025, 7, 16, 5000), (2500, 5, 3, 9000)])
def test_assign_follows_the_definition(torch, n_req, stride, ps, pages):
    """Steps that grow, shrink, end and restart requests, some of them beyond the pool, the table or the rows."""
    rng = np.random.RandomState(n_req)
    pool = Pool(torch, n_req, stride, ps, pages)
    held = np.zeros(n_req, np.int64)
    most = stride * ps
    for step in range(8):
        keep = np.where(rng.rand(n_req) < 0.3, rng.randint(0, held + 1), held)
        add = np.where(rng.rand(n_req) < 0.5, rng.randint(0, 3, n_req), rng.randint(0, max(2, most // 2), n_req))
        if step % 3 == 2:
            bad = rng.rand(n_req)
            add = np.where(bad < 0.05, -rng.randint(1, 100, n_req), add)
            keep = np.where((bad > 0.05) & (bad < 0.1), held + 1, keep)
            keep = np.where((bad > 0.1) & (bad < 0.15), -1, keep)
            add = np.where((bad > 0.15) & (bad < 0.2), most + 1, add)
        total = int(np.maximum(add, 0).sum())
        rows = total + 5 if step % 2 == 0 else max(0, total * 2 // 3)
        print(f"assign {n_req} x {stride} x {ps}, step {step}, rows {rows}", flush=True)
        held = pool.step(held, keep, add, rows).astype(np.int64)


def test_assign_given_back_step_restores_the_pool(torch):
    rng = np.random.RandomState(3)
    pool = Pool(torch, 40, 30, 16, 600)
    held = pool.step(np.zeros(40), np.zeros(40), rng.randint(0, 200, 40), 40 * 200)
    stack, table = list(pool.stack), pool.table.copy()
    grown = pool.step(held, held, rng.randint(0, 60, 40), 40 * 60)
    pool.step(grown, held, np.zeros(40), 0)
    assert pool.stack == stack and (pool.table == table).all()


def test_assign_without_rows_and_with_lengths_in_place(torch):
    pool = Pool(torch, 3, 4, 16, 12)
    add, zero = i32(torch, [20, 0, 33]), i32(torch, [0, 0, 0])
    rs, st, pos = i32(torch, np.zeros(4)), i32(torch, np.zeros(3)), i32(torch, np.zeros(53))
    slots = torch.zeros(53, dtype=torch.int64, device="cuda")
    R.paged_assign(pool.handle, ptr(pool.d_len), ptr(pool.d_len), ptr(add), 53, ptr(pool.d_len), ptr(rs), ptr(st), ptr(pos), ptr(slots))
    assert pool.d_len.tolist() == [20, 0, 33]
    R.paged_assign(pool.handle, ptr(pool.d_len), ptr(zero), ptr(zero), 0, ptr(pool.d_len), ptr(rs), ptr(st), None, None)
    assert pool.d_len.tolist() == [0, 0, 0] and rs.tolist() == [0, 0, 0, 0]
    assert pool.d_stack.tolist() == pool.stack and pool.d_count.item() == 12 and (pool.d_table == -1).all()


def test_assign_damaged_pool_stays_in_bounds(torch):
    """A count outside the stack and page numbers outside the cache: no slot comes of them, nothing outside is written."""
    for count in (-4, 9, 1 << 30):
        guard = i32(torch, np.full(64, 77))
        stack, cnt, table = guard[16:24], i32(torch, [count]), i32(torch, np.full((2, 4), 1 << 20))
        stack[:] = i32(torch, [5, -1, 8, 1 << 30, 0, 1, 2, 3])
        pool = R.PagePool(ptr(stack), ptr(cnt), ptr(table), 2, 4, 16, 8)
        held, keep, add = i32(torch, [64, 64]), i32(torch, [0, 0]), i32(torch, [0, 64])
        rs, st, pos = i32(torch, np.zeros(3)), i32(torch, np.zeros(2)), i32(torch, np.zeros(64))
        slots = torch.zeros(64, dtype=torch.int64, device="cuda")
        R.paged_assign(pool, ptr(held), ptr(keep), ptr(add), 64, ptr(held), ptr(rs), ptr(st), ptr(pos), ptr(slots))
        assert 0 <= cnt.item() <= 8
        assert ((slots >= -1) & (slots < 128)).all()
        assert (guard[:16] == 77).all() and (guard[24:] == 77).all()


# ---------------------------------------------------------------------------
# norm_rope_append
# ---------------------------------------------------------------------------
def plain_norm(torch, q, k, v, pos, inv, split, wq, wk, eps):
    """(rotated q, rotated k, v, |a| + |b| of the pairs of q and of k) in 64 bits; heads in dim 1."""
    def one(x, w):
        x = x.double()
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        d = x.shape[-1]
        a, b = (x[..., : d // 2], x[..., d // 2:]) if split else (x[..., ::2], x[..., 1::2])
        ang = pos.double()[:, None] * inv.double()
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        y = torch.empty_like(x)
        m = torch.empty_like(x)
        lo, hi = (slice(0, d // 2), slice(d // 2, d)) if split else (slice(0, d, 2), slice(1, d, 2))
        y[..., lo], y[..., hi] = a * c - b * s, b * c + a * s
        m[..., lo] = m[..., hi] = a.abs() + b.abs()
        return y, m
    yq, mq = one(q, wq)
    yk, mk = one(k, wk)
    return yq, yk, v.double(), mq, mk


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd,rows", [(4, 2, 32, 5), (32, 8, 64, 1), (14, 2, 64, 130), (28, 4, 128, 37), (16, 16, 128, 3),
                                              (3, 1, 64, 700), (28, 4, 128, 1100)])
@pytest.mark.parametrize("split,normed", [(False, False), (True, True), (False, True)])
def test_norm_rope_append(torch, kind, heads, kv, hd, rows, split, normed):
    g = torch.Generator().manual_seed(rows + heads)
    pad = 12 if rows % 2 else 0
    ld = (heads + 2 * kv) * hd + pad
    qkv = torch.randn(rows, ld, generator=g) * 3
    pos = torch.randint(0, 1 << 17, (rows,), generator=g)
    pos[0] = (1 << 31) - 1  # the farthest position
    pos[-1] = 0
    ps, pages = 24, rows // 24 + 2
    slots = torch.randperm(ps * pages, generator=g)[:rows]
    if rows > 4:
        slots[1], slots[2], slots[3] = -1, ps * pages, 1 << 40  # rows that are not appended
    inv = (500000.0 ** -(torch.arange(0, hd, 2).double() / hd)).float()
    wq, wk = ((1 + 0.3 * torch.randn(hd, generator=g)).bfloat16() for _ in range(2)) if normed else (None, None)
    if normed and rows % 5 == 0:
        wk = None  # one of the two alone
    f32_weights = normed and heads == 28
    if f32_weights:
        wq, wk = wq.float(), None if wk is None else wk.float()
    t = types(torch)[kind]
    stride = 2 * kv * hd + 16
    store = torch.full((ps * pages, stride), float("nan"), device="cuda").to(t)  # k and v in one buffer
    dq = qkv.cuda()
    out = torch.full((rows, heads * hd + 4), 9.0, device="cuda")
    e = store.element_size()
    c = R.PagedCache(ptr(store), ptr(store) + kv * hd * e, kind, kv, hd, ps, pages, stride)
    dev = [x.cuda() if x is not None else None for x in (inv, pos.int(), slots, wq, wk)]
    print(f"norm {kind} {rows} x {heads}/{kv} x {hd} split={split} normed={normed}", flush=True)
    b = ptr(dq)
    R.norm_rope_append(c, b, ld, b + 4 * heads * hd, ld, b + 4 * (heads + kv) * hd, ld, rows, heads, ptr(out), heads * hd + 4, ptr(dev[0]),
                       ptr(dev[1]), ptr(dev[2]), "split_half" if split else "interleaved", ptr(dev[3]), ptr(dev[4]), 1e-6,
                       torch.cuda.current_stream().cuda_stream, 0 if f32_weights else 1)
    x = qkv[:, : (heads + 2 * kv) * hd].view(rows, heads + 2 * kv, hd)
    yq, yk, yv, mq, mk = plain_norm(torch, x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], pos, inv, split, wq, wk, 1e-6)
    got = out.cpu().double()
    assert (got[:, heads * hd:] == 9).all()
    assert ((got[:, : heads * hd].view(rows, heads, hd) - yq).abs() <= 2.0 ** -20 * mq).all()
    s = store.cpu().double()
    used = (slots >= 0) & (slots < ps * pages)
    gk = s[slots[used], : kv * hd].view(-1, kv, hd)
    gv = s[slots[used], kv * hd: 2 * kv * hd].view(-1, kv, hd)
    tiny = 2.0 ** -25 if kind == "f16" else 0  # half of f16's smallest step
    assert ((gk - yk[used]).abs() <= (2.0 ** -20 + HALF_STEP[kind]) * mk[used] + tiny).all()
    assert torch.equal(gv, yv[used].float().to(t).double())
    rest = torch.ones(ps * pages, dtype=torch.bool)
    rest[slots[used]] = False
    assert s[rest].isnan().all() and s[:, 2 * kv * hd:].isnan().all()  # nothing else is written
    # The same in place: q's rows hold the result.
    b = ptr(dq)
    R.norm_rope_append(c, b, ld, b + 4 * heads * hd, ld, b + 4 * (heads + kv) * hd, ld, rows, heads, b, ld, ptr(dev[0]), ptr(dev[1]),
                       ptr(dev[2]), "split_half" if split else "interleaved", ptr(dev[3]), ptr(dev[4]), 1e-6,
                       torch.cuda.current_stream().cuda_stream, 0 if f32_weights else 1)
    after = dq.cpu()
    assert torch.equal(after[:, : heads * hd], out.cpu()[:, : heads * hd])
    assert torch.equal(after[:, heads * hd:], qkv[:, heads * hd:])


def test_norm_rope_append_odd_values(torch):
    """A head of zeros, of values whose squares leave f32's middle, and of infinities and NaN: each stays in its own head."""
    heads, kv, hd = 4, 2, 64
    x = torch.randn(3, (heads + 2 * kv) * hd)
    x[0, :hd] = 0
    x[0, hd: 2 * hd] *= 1e15
    x[0, 2 * hd: 3 * hd] *= 1e-15
    x[0, 3 * hd + 5] = float("inf")
    x[1, 4 * hd + 1] = float("nan")
    inv, pos, slots = torch.ones(hd // 2).cuda(), i32(torch, [3, 4, 5]), torch.tensor([0, 1, 2]).cuda()
    k, v = (torch.zeros(16, kv * hd, device="cuda", dtype=torch.float16) for _ in range(2))
    out, w, dx = torch.zeros(3, heads * hd, device="cuda"), torch.ones(hd, device="cuda").bfloat16(), x.cuda()
    b, ld = ptr(dx), x.shape[1]
    R.norm_rope_append(R.PagedCache(ptr(k), ptr(v), "f16", kv, hd, 16, 1), b, ld, b + 4 * heads * hd, ld, b + 4 * (heads + kv) * hd, ld, 3,
                       heads, ptr(out), heads * hd, ptr(inv), ptr(pos), ptr(slots), "interleaved", ptr(w), ptr(w), 1e-6)
    o = out.cpu().view(3, heads, hd)
    assert (o[0, 0] == 0).all() and o[0, 1].isfinite().all() and o[0, 2].isfinite().all()
    assert abs(o[0, 1].double().square().mean().item() - 1) < 1e-5  # 1e30 in squares: eps is nothing
    assert not o[0, 3].isfinite().all() and o[1].isfinite().all()
    assert not k[1, :hd].isfinite().all() and k[1, hd:].isfinite().all() and k[0].isfinite().all()


# ---------------------------------------------------------------------------
# paged_attention
# ---------------------------------------------------------------------------
def plain_attend(torch, q, k, v, table, row_start, start, ps, pages, window, scale, out, valid=None):
    """(out, error bound) in 64 bits, row by row over exactly the keys that a row sees."""
    rows, heads, hd = q.shape
    kv = k.shape[1]
    G = heads // kv
    out, bound = out.double().clone(), torch.zeros(rows, heads, hd, dtype=torch.float64)
    q, k, v = q.double(), k.double(), v.double()
    for r in range(len(start)):
        b, e = (min(max(int(x), 0), rows) for x in row_start[r:r + 2])
        for i in range(b, e):
            p = int(start[r]) + i - b
            lo, hi = (max(0, p + 1 - window) if window else 0), min(p + 1, table.shape[1] * ps)
            page = torch.as_tensor(np.asarray(table[r])[np.arange(lo, hi) // ps] if p >= 0 and lo < hi else [], dtype=torch.int64)
            there = (page >= 0) & (page < pages)
            slot = (page * ps + torch.arange(lo, lo + len(page)) % ps)[there]
            if not len(slot):
                out[i] = 0
                continue
            kk, vv = k[slot].permute(1, 2, 0), v[slot].permute(1, 0, 2)  # [kv, hd, n], [kv, n, hd]
            qq = q[i].view(kv, G, hd) * scale
            s = torch.matmul(qq, kk)
            w = torch.softmax(s, -1)
            out[i] = torch.matmul(w, vv).view(heads, hd)
            size = torch.matmul(qq.abs(), kk.abs()).amax(-1, keepdim=True)
            n = len(slot)
            bound[i] = (2 * ((hd + 8) * size + n + 24) * U * torch.matmul(w, vv.abs())).view(heads, hd)
    return out, bound


SPECS = {
    "one": [(0, 1)],
    "step": [(5, 1), (0, 0), (63, 1), (64, 1), (200, 1), (15, 1), (0, 1), (777, 1)],
    "drafts": [(100, 5), (0, 3), (17, 1), (31, 12), (500, 2)],
    "chunks": [(0, 70), (33, 130), (500, 64), (9, 1)],
    "long": [(1500, 33)],
    "wait": [(40, 0), (-6, 3), (-2, 5), (70, 1)],  # no rows; rows that see nothing
}


def build(torch, spec, heads, kv, hd, kind, ps, seed, extra_rows=2, garbage=float("nan")):
    """Inputs of a batch: pages in a random order, `garbage` in every slot that no request fills."""
    rng = np.random.RandomState(seed)
    g = torch.Generator().manual_seed(seed)
    total = [max(0, p + n) for p, n in spec]
    need = [-(-x // ps) for x in total]
    pages = sum(need) + 2
    order = rng.permutation(pages)
    table = np.full((len(spec), max(need) + 2), -1, np.int32)
    at = 0
    t = types(torch)[kind]
    k, v = (torch.full((pages * ps, kv, hd), garbage).to(t) for _ in range(2))
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
        j = np.arange(total[r])
        slot = torch.as_tensor(table[r][j // ps].astype(np.int64) * ps + j % ps)
        k[slot] = torch.randn(len(j), kv, hd, generator=g).to(t)
        v[slot] = torch.randn(len(j), kv, hd, generator=g).to(t)
    counts = [n for _, n in spec]
    row_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    q = torch.randn(int(row_start[-1]) + extra_rows, heads, hd, generator=g) * 1.5
    return dict(q=q, k=k, v=v, table=table, row_start=row_start, start=np.array([p for p, _ in spec], np.int32), pages=pages, ps=ps)


def attend(torch, b, kind, window=0, scale=None, pad=0, stream=None, ws=None, fill=9.0):
    """The op on the GPU: out with rows `pad` values apart more than they are wide, [rows, heads, hd]."""
    rows, heads, hd = b["q"].shape
    kv = b["k"].shape[1]
    w = heads * hd
    q = torch.full((rows, w + pad), float("nan"), device="cuda")
    q[:, :w] = b["q"].reshape(rows, w).cuda()
    out = torch.full((rows, w + pad), fill, device="cuda")
    k, v = b["k"].cuda(), b["v"].cuda()
    c = R.PagedCache(ptr(k), ptr(v), kind, kv, hd, b["ps"], b["pages"])
    d = [i32(torch, b[x]) for x in ("table", "row_start", "start")]
    n = len(b["start"])
    if ws is None:
        ws = torch.zeros(R.paged_attention_workspace(rows, n, heads, kv, hd), dtype=torch.uint8, device="cuda")
    R.paged_attention(c, ptr(d[0]), b["table"].shape[1], ptr(d[1]), ptr(d[2]), n, ptr(q), w + pad, ptr(out), w + pad, rows, heads,
                      hd ** -0.5 if scale is None else scale, window, ptr(ws), ws.numel(),
                      torch.cuda.current_stream().cuda_stream if stream is None else stream)
    torch.cuda.synchronize()
    assert (out[:, w:] == fill).all()
    return out[:, :w].reshape(rows, heads, hd).cpu()


def check(torch, b, got, window=0, scale=None, fill=9.0, norm=1e-6):
    rows, heads, hd = b["q"].shape
    want, bound = plain_attend(torch, b["q"], b["k"], b["v"], b["table"], b["row_start"], b["start"], b["ps"], b["pages"], window,
                               hd ** -0.5 if scale is None else scale, torch.full((rows, heads, hd), fill))
    got = got.double()
    # Rows that several requests claim (row_start does not ascend) hold one's output; NaN is NaN where a row sees one.
    spans = [(min(max(int(x), 0), rows), min(max(int(y), 0), rows)) for x, y in zip(b["row_start"][:-1], b["row_start"][1:])]
    claims = torch.tensor([sum(x <= i < y for x, y in spans) for i in range(rows)])
    same = (claims > 1)[:, None, None] | (got.isnan() & want.isnan())
    got, want, bound = (torch.where(same, 0.0, t) for t in (got, want, bound))
    err = (got - want).abs()
    assert (err <= bound).all(), f"largest error {err.max():.3g}, {float((err / bound.clamp(min=1e-30)).max()):.3g} of its bound"
    if norm and want.norm() > 0:
        assert (err.norm() / want.norm()).item() <= norm, (err.norm() / want.norm()).item()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,hd", [(4, 2, 32), (32, 8, 64), (14, 2, 64), (28, 4, 128), (5, 5, 128), (40, 1, 64)])
@pytest.mark.parametrize("spec", sorted(SPECS))
def test_attention(torch, kind, heads, kv, hd, spec):
    ps = {32: 8, 64: 16, 128: 24}[hd] if spec != "long" else 48
    b = build(torch, SPECS[spec], heads, kv, hd, kind, ps, seed=heads + hd)
    print(f"attention {kind} {heads}/{kv} x {hd} {spec}", flush=True)
    check(torch, b, attend(torch, b, kind, pad=4 if spec == "drafts" else 0))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 5000])
@pytest.mark.parametrize("heads,kv,hd,ps", [(8, 2, 64, 16), (7, 1, 128, 64)])
def test_attention_window(torch, kind, window, heads, kv, hd, ps):
    for spec in ("step", "drafts", "chunks", "wait"):
        b = build(torch, SPECS[spec], heads, kv, hd, kind, ps, seed=window)
        check(torch, b, attend(torch, b, kind, window), window)


@pytest.mark.parametrize("ps", [1, 3, 8, 16, 17, 32, 100, 256, 1000])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_attention_page_sizes(torch, kind, ps):
    """Pages that end inside a tile of keys, and ones larger than any request."""
    for spec in ("step", "chunks"):
        b = build(torch, SPECS[spec], 8, 2, 64, kind, ps, seed=ps)
        check(torch, b, attend(torch, b, kind))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [32, 64, 128])
def test_attention_hidden_values_do_not_matter(torch, kind, hd):
    """Infinities and NaN in keys and values behind a row's position, and in front of its window, leave the row as it is."""
    b = build(torch, [(40, 90), (3, 7), (300, 1)], 4, 2, hd, kind, 16, seed=hd)
    for window in (0, 20):
        clean = attend(torch, b, kind, window)
        for value in (float("nan"), float("inf"), -float("inf")):
            for r, p in ((0, 77), (1, 8), (0, 129)):
                d = dict(b, k=b["k"].clone(), v=b["v"].clone())
                slot = b["table"][r, p // 16] * 16 + p % 16
                d["k"][slot], d["v"][slot] = value, value
                got = attend(torch, d, kind, window)
                for r2, (past, n) in enumerate([(40, 90), (3, 7), (300, 1)]):
                    first = int(b["row_start"][r2])
                    for i in range(n):
                        sees = r2 == r and past + i >= p and not (window and past + i >= p + window)
                        a, c = got[first + i], clean[first + i]
                        if sees:
                            assert value == -float("inf") or not a.isfinite().all()
                        else:
                            assert a.isfinite().all() and (a - c).abs().max() <= 1e-5 * (1 + c.abs().max()), (window, value, r, p, r2, i)


def test_attention_one_bad_value_stays_in_its_dimension(torch):
    """A value that is not finite reaches the rows that see it, in its own head and dimension."""
    for kind in ("f32", "bf16", "f16"):
        b = build(torch, [(20, 40)], 4, 2, 64, kind, 16, seed=1)
        clean = attend(torch, b, kind)
        slot = b["table"][0, 30 // 16] * 16 + 30 % 16
        b["v"][slot, 1, 17] = float("inf")
        got = attend(torch, b, kind)
        hit = torch.zeros(40, 4, 64, dtype=torch.bool)
        hit[10:, 2:, 17] = True
        assert (got[:40][hit] == float("inf")).all()
        assert (got[:40][~hit] - clean[:40][~hit]).abs().max() <= 1e-5


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_attention_bad_pages_and_rows(torch, kind):
    """Page numbers that are none are holes in a request's keys; row_start of any values stays in the batch."""
    b = build(torch, SPECS["chunks"], 8, 4, 64, kind, 16, seed=2)
    t = b["table"]
    t[0, 1], t[1, 0], t[1, 3], t[2, 5], t[2, 30], t[3, 0] = -1, b["pages"], 2**31 - 1, -2**31, -7, -1
    check(torch, b, attend(torch, b, kind))
    b["row_start"] = np.array([-5, 20, 10, 2**31 - 1, 2**31 - 1], np.int32)
    check(torch, b, attend(torch, b, kind))
    b["row_start"] = np.array([60, 30, -2**31, 0, 50], np.int32)  # one request has rows: 0 .. 49
    check(torch, b, attend(torch, b, kind))


def test_attention_positions_behind_the_table(torch):
    """A row whose position is past what the table has room for sees all of it."""
    b = build(torch, [(64, 3), (30, 2)], 4, 2, 64, "bf16", 16, seed=3)
    b["table"] = np.ascontiguousarray(b["table"][:, :4])
    check(torch, b, attend(torch, b, "bf16"))
    b["start"] = np.array([2**31 - 1, 2**31 - 2], np.int32)
    check(torch, b, attend(torch, b, "bf16"))
    check(torch, b, attend(torch, b, "bf16", window=2**32 - 1), window=2**32 - 1)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_attention_large_and_small_scores(torch, kind):
    """One key far ahead of the others, scores that would leave exp's range, values near the type's ends, and equal scores."""
    b = build(torch, [(100, 4), (0, 40)], 4, 2, 64, kind, 16, seed=4)
    check(torch, b, attend(torch, b, kind, scale=8.0), scale=8.0, norm=None)  # scores of hundreds
    check(torch, b, attend(torch, b, kind, scale=-3.0), scale=-3.0, norm=None)
    check(torch, b, attend(torch, b, kind, scale=0.0), scale=0.0)  # the mean of what is seen
    big = dict(b, v=(b["v"].double() * (1e4 if kind == "f16" else 1e30)).to(b["v"].dtype))
    check(torch, big, attend(torch, big, kind))
    small = dict(b, q=b["q"] * 1e-20, k=(b["k"].double() * (1e-4 if kind == "f16" else 1e-10)).to(b["k"].dtype))
    check(torch, small, attend(torch, small, kind, scale=1e20), scale=1e20)
    wide = dict(b, q=b["q"] * 1e20, k=(b["k"].double() * 1e-3).to(b["k"].dtype))
    check(torch, wide, attend(torch, wide, kind, scale=1e-17), scale=1e-17)


def test_attention_lowest_values(torch):
    """Keys whose scores are f32's lowest or -inf have no weight; where all of a row's are -inf it gets zeros."""
    b = build(torch, [(30, 2), (4, 1)], 2, 1, 64, "f32", 16, seed=5)
    b["q"][:] = 0
    b["q"][..., 0] = 1.0
    b["k"][..., 0] = 0.0
    slot = lambda r, p: b["table"][r, p // 16] * 16 + p % 16  # noqa: E731
    for p in range(31):
        b["k"][slot(0, p), 0, 0] = torch.finfo(torch.float32).min if p % 2 else -float("inf")
    b["k"][slot(0, 7), 0, 0] = 1.0
    for p in range(5):
        b["k"][slot(1, p), 0, 0] = -float("inf")
    got = attend(torch, b, "f32", scale=1.0)
    for i in range(2):
        want = b["v"][slot(0, 7), 0]
        if i == 1:  # (its own position's key scores 0: e^-1 of the weight)
            w = 1 / (1 + np.exp(1.0))
            want = b["v"][slot(0, 7), 0] * (1 - w) + b["v"][slot(0, 31), 0] * w
        assert (got[i] - want).abs().max() <= 1e-5
    assert (got[2] == 0).all()


def test_attention_interleaved_cache_and_long_offsets(torch):
    """k and v in one buffer whose slots lie past 2^32 bytes."""
    kv, hd, ps = 2, 64, 16
    stride = 1 << 16
    pages = 3000  # 48000 slots of 128 KiB: 6.3 GB
    store = torch.zeros(pages * ps, stride, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(0)
    table = np.array([[2999, 1, 2500, 2100]], np.int32)
    q = torch.randn(2, 4, hd, generator=g)
    k, v = (torch.zeros(pages * ps, kv, hd, dtype=torch.bfloat16) for _ in range(2))
    for p in range(60):
        s = int(table[0, p // ps]) * ps + p % ps
        k[s], v[s] = torch.randn(kv, hd, generator=g).bfloat16(), torch.randn(kv, hd, generator=g).bfloat16()
        store[s, 1000 * 8: 1000 * 8 + kv * hd] = k[s].flatten().cuda()
        store[s, 2000 * 8: 2000 * 8 + kv * hd] = v[s].flatten().cuda()
    c = R.PagedCache(ptr(store) + 16000, ptr(store) + 32000, "bf16", kv, hd, ps, pages - 1 + 1, stride)
    out, dq = torch.zeros(2, 4 * hd, device="cuda"), q.flatten(1).cuda()
    ws = torch.zeros(R.paged_attention_workspace(2, 1, 4, kv, hd), dtype=torch.uint8, device="cuda")
    d = [i32(torch, x) for x in (table, [0, 2], [58])]
    R.paged_attention(c, ptr(d[0]), 4, ptr(d[1]), ptr(d[2]), 1, ptr(dq), 4 * hd, ptr(out), 4 * hd, 2, 4, hd ** -0.5, 0, ptr(ws), ws.numel())
    b = dict(q=q, k=k, v=v, table=table, row_start=[0, 2], start=[58], ps=ps, pages=pages)
    check(torch, b, out.cpu().view(2, 4, hd))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_attention_does_not_change_from_run_to_run(torch, kind):
    b = build(torch, [(1900, 3), (10, 200), (700, 1)], 8, 2, 64, kind, 16, seed=6)
    first = attend(torch, b, kind)
    for _ in range(3):
        assert torch.equal(attend(torch, b, kind), first)


def test_attention_many_requests(torch):
    """More requests than threads of a block."""
    rng = np.random.RandomState(0)
    spec = [(int(rng.randint(0, 60)), int(rng.randint(0, 3))) for _ in range(1500)]
    b = build(torch, spec, 4, 1, 32, "f16", 8, seed=7)
    check(torch, b, attend(torch, b, "f16"))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_attention_captured_step_serves_other_batches(torch, kind):
    """One graph, replayed with other lengths, pages and values, and eager calls between, on another stream and workspace."""
    heads, kv, hd, ps = 8, 2, 64, 16
    batches = [build(torch, s, heads, kv, hd, kind, ps, seed=i) for i, s in enumerate(
        [[(30, 2), (100, 1), (0, 5)], [(500, 1), (0, 0), (77, 7)], [(0, 1), (1200, 3), (-9, 4)], [(5, 8), (0, 0), (0, 0)]])]
    rows = max(b["q"].shape[0] for b in batches)
    pages, stride = max(b["pages"] for b in batches), max(b["table"].shape[1] for b in batches)
    t = types(torch)[kind]
    k, v = (torch.zeros(pages * ps, kv, hd, dtype=t, device="cuda") for _ in range(2))
    q, out = (torch.zeros(rows, heads * hd, device="cuda") for _ in range(2))
    table, rs, st = i32(torch, np.zeros((3, stride))), i32(torch, np.zeros(4)), i32(torch, np.zeros(3))
    ws = torch.zeros(R.paged_attention_workspace(rows, 3, heads, kv, hd), dtype=torch.uint8, device="cuda")
    c = R.PagedCache(ptr(k), ptr(v), kind, kv, hd, ps, pages)

    def call():
        R.paged_attention(c, ptr(table), stride, ptr(rs), ptr(st), 3, ptr(q), heads * hd, ptr(out), heads * hd, rows, heads, hd ** -0.5, 0,
                          ptr(ws), ws.numel(), torch.cuda.current_stream().cuda_stream)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in (0, 1, 2, 3, 1, 0):
        b = batches[i]
        n = b["q"].shape[0]
        k[: b["pages"] * ps], v[: b["pages"] * ps] = b["k"].cuda(), b["v"].cuda()
        q[:n] = b["q"].flatten(1).cuda()
        out.fill_(9.0)
        table[:, : b["table"].shape[1]] = i32(torch, b["table"])
        table[:, b["table"].shape[1]:] = -1
        rs.copy_(i32(torch, b["row_start"]))
        st.copy_(i32(torch, b["start"]))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check(torch, b, out[:n].view(n, heads, hd).cpu())
        check(torch, b, attend(torch, b, kind))  # an eager call with a workspace of its own


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window", [0, 1, 33, 500])
@pytest.mark.parametrize("heads,kv,spec,ps", [(28, 4, [(0, 131), (700, 90), (33, 200)], 16), (16, 16, [(90, 513)], 40), (7, 1, [(0, 400), (1300, 3), (5, 0)], 64)])
def test_attention_prompts_of_wide_heads(torch, kind, window, heads, kv, spec, ps):
    """Chunks that fill tiles of 128 vectors, heads of 128."""
    b = build(torch, spec, heads, kv, 128, kind, ps, seed=heads)
    check(torch, b, attend(torch, b, kind, window, pad=4), window)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_attention_bad_values_in_prompts_of_wide_heads(torch, kind):
    """A NaN among the values reaches its dimension of the rows that see it, NaN in holes and behind every row none."""
    b = build(torch, [(100, 150), (0, 80)], 28, 4, 128, kind, 16, seed=3)
    for r, j, kvh, d in ((0, 7, 1, 5), (0, 200, 2, 127), (1, 79, 0, 64)):
        b["v"][int(b["table"][r][j // 16]) * 16 + j % 16, kvh, d] = float("nan")
    b["table"][0][4] = -1
    check(torch, b, attend(torch, b, kind), norm=0)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("n_req", [2, 66, 130, 700])
def test_attention_idle_requests(torch, kind, n_req):
    """Requests without rows before, between and behind those that have some."""
    for busy in ((0, n_req - 1), (n_req // 2,), (0,), (n_req - 1,), (0, 1, n_req // 2, n_req - 1)):
        for rows in (1, 40):
            spec = [(300 + 7 * i, rows) if i in busy else (20, 0) for i in range(n_req)]
            print("idle", n_req, busy, rows, flush=True)
            b = build(torch, spec, 8, 2, 64, kind, 16, seed=n_req)
            check(torch, b, attend(torch, b, kind))


@pytest.mark.parametrize("requests,rows,hd", [(1, 1, 64), (800, 1, 64), (600, 3, 128), (40, 150, 64), (40, 250, 128), (40, 100, 32)])
def test_attention_small_weights_in_f16(torch, requests, rows, hd):
    """One key whose value is 0 is 2^31 times as heavy as each of the others, whose values are 1: they make all of the output,
    as many as they are * 2^-31. f16 terms of a weight are off by half of f16's smallest step at most, 2^-25, where the
    heaviest weight is 2^11 at least: 2^-36 for every key, beside the bound of the other cases (scores of 31 ln 2 = 21.5).
    The requests share their pages and are enough for items that are not cut."""
    kv, ps, past = 2, 16, 4000
    pages = (past + rows) // ps + 2
    t = torch.float16
    k, v = torch.zeros(pages * ps, kv, hd, dtype=t, device="cuda"), torch.ones(pages * ps, kv, hd, dtype=t, device="cuda")
    k[17, :, 0], v[17] = 1.0, 0.0
    q = torch.zeros(requests * rows, 4 * hd, device="cuda")
    q[:, ::hd] = 31 * np.log(2.0)
    out = torch.full((requests * rows, 4 * hd), 9.0, device="cuda")
    table, rs = i32(torch, np.tile(np.arange(pages), (requests, 1))), i32(torch, np.arange(requests + 1) * rows)
    st = i32(torch, np.full(requests, past))
    ws = torch.zeros(R.paged_attention_workspace(requests * rows, requests, 4, kv, hd), dtype=torch.uint8, device="cuda")
    R.paged_attention(R.PagedCache(ptr(k), ptr(v), "f16", kv, hd, ps, pages), ptr(table), pages, ptr(rs), ptr(st), requests, ptr(q), 4 * hd,
                      ptr(out), 4 * hd, requests * rows, 4, 1.0, 0, ptr(ws), ws.numel(), torch.cuda.current_stream().cuda_stream)
    gap = np.exp(-np.float64(np.float32(31 * np.log(2.0))))
    n = past + np.tile(np.arange(rows), requests)[:, None]  # keys beside the heavy one
    want = n * gap / (1 + n * gap)
    err = np.abs(out.cpu().numpy().astype(np.float64) - want)
    over = err - (n * 2.0 ** -36 + 2 * ((hd + 8) * 21.5 + n + 24) * U * want)
    assert over.max() <= 0, f"{(err / want).max():.3g} of the output"


@pytest.mark.parametrize("rows,hd", [(1, 64), (2, 128), (200, 32), (200, 64), (300, 128)])
@pytest.mark.parametrize("log2", [8, 16, 20, 23, 24, 25, 26, 27, 28, 30])
def test_attention_scores_past_f32s_steps_in_f16(torch, rows, hd, log2):
    """Scores (in base 2) of 2^log2 and up to 8 above it, where f32 holds no more than some of the steps between: which keys are
    ahead is a matter of rounding, but outputs stay averages of the values, 1 .. 2."""
    kv, ps, past = 1, 16, 500
    pages, rng = (past + rows) // ps + 1, np.random.RandomState(log2)
    t = torch.float16
    k, v = torch.zeros(pages * ps, kv, hd, dtype=t), torch.tensor(1 + rng.rand(pages * ps, kv, hd)).to(t)
    k[:, :, 0], k[:, :, 1] = 1024.0, torch.tensor(rng.randint(0, 9, (pages * ps, 1))).to(t)
    q = torch.zeros(rows, 2, hd, device="cuda")
    q[..., 0], q[..., 1] = 2.0 ** (log2 - 10) * np.log(2.0), np.log(2.0)
    b = dict(q=q.cpu(), k=k, v=v, table=np.arange(pages, dtype=np.int32)[None], row_start=np.array([0, rows]), start=np.array([past]), pages=pages, ps=ps)
    out = attend(torch, b, "f16", scale=1.0)
    assert out.isfinite().all() and (out >= 1 - 1e-5).all() and (out <= 2 + 1e-5).all(), (out.min(), out.max())


def attend_exact(torch, b, window, scale):
    """As plain_attend, a request and head at a time on the GPU: (out, error bound); without holes, every row a request's."""
    rows, heads, hd = b["q"].shape
    kv, ps = b["k"].shape[1], b["ps"]
    q, k, v = b["q"].cuda().double() * scale, b["k"].cuda(), b["v"].cuda()
    out, bound = (torch.zeros(rows, heads, hd, dtype=torch.float64, device="cuda") for _ in range(2))
    for r, past in enumerate(b["start"].tolist()):
        first, end = int(b["row_start"][r]), int(b["row_start"][r + 1])
        j = torch.arange(past + end - first, device="cuda")
        slot = torch.as_tensor(b["table"][r].astype(np.int64), device="cuda")[j // ps] * ps + j % ps
        pos = past + torch.arange(end - first, device="cuda")[:, None]
        hidden = (j > pos) | ((j <= pos - window) if window else (j < 0))
        n = (~hidden).sum(1, keepdim=True)
        for h in range(heads if end > first else 0):
            kk, vv = (x[slot, h * kv // heads].double() for x in (k, v))
            qq, kt = q[first:end, h], kk.t().contiguous()
            w = torch.softmax((qq @ kt).masked_fill(hidden, -np.inf), -1)
            out[first:end, h] = w @ vv
            size = (qq.abs() @ kt.abs()).masked_fill(hidden, 0).amax(1, keepdim=True)
            bound[first:end, h] = 2 * ((hd + 8) * size + n + 24) * U * (w @ vv.abs())
    return out.cpu(), bound.cpu()


RUNS = {"tokens": [(5000 + 37 * i, 1) for i in range(44)],
        "drafts": [(8000 - 211 * i, 1 + i % 8) for i in range(36)],
        "prompts": [(1900, 1000), (400, 1500)],
        "mixed": [(6000 - 97 * i, 1) for i in range(40)] + [(700, 900), (0, 0), (3000, 5), (0, 300)]}


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("what,heads,kv,hd,window", [
    ("tokens", 28, 4, 128, 0), ("drafts", 32, 8, 64, 0), ("drafts", 28, 4, 128, 3000), ("prompts", 28, 4, 128, 0),
    ("prompts", 32, 8, 64, 1000), ("mixed", 28, 4, 128, 0), ("prompts", 16, 4, 32, 0)])
def test_attention_runs_of_many_units(torch, kind, what, heads, kv, hd, window):
    """Batches that give every block a long run, over several items or inside one."""
    spec, ps = RUNS[what], 16
    print("runs", kind, what, heads, kv, hd, flush=True)
    g = torch.Generator(device="cuda").manual_seed(hd)
    need = [-(-(p + n) // ps) for p, n in spec]
    pages = sum(need) + 2
    order, table = np.random.RandomState(hd).permutation(pages), np.full((len(spec), max(need)), -1, np.int32)
    for r, n in enumerate(need):
        table[r, :n] = order[sum(need[:r]): sum(need[:r]) + n]
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    k, v = (rnd(pages * ps, kv, hd).to(types(torch)[kind]) for _ in range(2))
    row_start = np.concatenate([[0], np.cumsum([n for _, n in spec])]).astype(np.int32)
    b = dict(q=1.5 * rnd(int(row_start[-1]), heads, hd), k=k, v=v, table=table, row_start=row_start,
             start=np.array([p for p, _ in spec], np.int32), pages=pages, ps=ps)
    want, bound = attend_exact(torch, b, window, hd ** -0.5)
    err = (attend(torch, b, kind, window).double() - want).abs()
    assert (err <= bound).all(), f"largest error {err.max():.3g}"
    assert (err.norm() / want.norm()).item() <= 1e-6


def test_attention_workspace_serves_other_sizes(torch):
    """One workspace, zeroed once, for calls of other head sizes, rows and requests in turn: no call's parts lie on another's counters."""
    ws = torch.zeros(max(R.paged_attention_workspace(200, 8, h, kv, hd) for h, kv, hd in ((28, 4, 128), (32, 8, 64), (4, 2, 32))),
                     dtype=torch.uint8, device="cuda")
    for _ in range(2):
        for heads, kv, hd, spec, kind in ((28, 4, 128, "step", "bf16"), (32, 8, 64, "chunks", "f32"), (4, 2, 32, "step", "f16"),
                                          (32, 8, 64, "long", "bf16"), (28, 4, 128, "chunks", "f16"), (32, 8, 64, "drafts", "f32")):
            b = build(torch, SPECS[spec], heads, kv, hd, kind, 16, seed=heads + hd)
            if spec == "chunks":
                b["q"] = b["q"][:200]  # the last request's rows end behind them
            print("workspace", heads, hd, spec, kind, flush=True)
            check(torch, b, attend(torch, b, kind, ws=ws))


def test_attention_on_two_streams(torch):
    """Calls that overlap, each with a workspace of its own."""
    cases = [(build(torch, SPECS["long"], 28, 4, 128, "bf16", 16, seed=1), "bf16"), (build(torch, SPECS["drafts"], 32, 8, 64, "f16", 16, seed=2), "f16")]
    sides = []
    for b, kind in cases:
        rows, heads, hd = b["q"].shape
        kv, w = b["k"].shape[1], heads * hd
        k, v, q = b["k"].cuda(), b["v"].cuda(), b["q"].cuda()
        out = torch.full((rows, w), 9.0, device="cuda")
        d = [i32(torch, b[x]) for x in ("table", "row_start", "start")]
        n = len(b["start"])
        ws = torch.zeros(R.paged_attention_workspace(rows, n, heads, kv, hd), dtype=torch.uint8, device="cuda")
        c = R.PagedCache(ptr(k), ptr(v), kind, kv, hd, b["ps"], b["pages"])
        sides.append((b, out, torch.cuda.Stream(), (k, v, q), lambda s, a=(c, ptr(d[0]), b["table"].shape[1], ptr(d[1]), ptr(d[2]), n, ptr(q), w,
                      ptr(out), w, rows, heads, hd ** -0.5, 0, ptr(ws), ws.numel()), keep=(d, ws): R.paged_attention(*a, s.cuda_stream)))
    torch.cuda.synchronize()
    for _ in range(20):
        for _, _, s, _, run in sides:
            run(s)
    torch.cuda.synchronize()
    for b, out, _, _, _ in sides:
        check(torch, b, out.view(b["q"].shape).cpu())


# ---------------------------------------------------------------------------
# verify_drafts
# ---------------------------------------------------------------------------
def plain_verify(target, draft, tokens, row_start, ua, us, vocab, out):
    """The definition, request by request, in 64 bits."""
    accepted, out = [], np.array(out)
    rows = len(tokens)
    good = lambda w: np.where((w > 0) & np.isfinite(w), w, 0.0)  # noqa: E731
    for r in range(len(us)):
        b, e = (min(max(int(x), 0), rows) for x in row_start[r:r + 2])
        if e <= b:
            accepted.append(0)
            continue
        a = 0
        while a < e - b - 1:
            x = int(tokens[b + a + 1])
            if not 0 <= x < vocab:
                break
            q = 1.0 if draft is None else np.float64(draft[b + a, x])
            if not np.float64(ua[b + a]) * q < np.float64(target[b + a, x]):
                break
            a += 1
        p = target[b + a].astype(np.float64)
        w = good(p)
        if a < e - b - 1:
            less = p - draft[b + a] if draft is not None else np.where(np.arange(vocab) == int(tokens[b + a + 1]), 0.0, p)
            w = good(less) if good(less).sum() > 0 else w
        c = w.cumsum()
        if c[-1] > 0:
            found = min(int((c <= np.float64(us[r]) * c[-1]).sum()), int((c < c[-1]).sum()))
        else:
            found = -1
        out[b:e] = -1
        out[b:b + a] = tokens[b + 1:b + a + 1]
        out[b + a] = found
        accepted.append(a)
    return accepted, out.tolist()


def verify(torch, target, draft, tokens, row_start, ua, us, vocab=None, ws=None):
    rows, ld = target.shape
    vocab = ld if vocab is None else vocab
    d = [torch.tensor(np.ascontiguousarray(x, dtype=np.float32), device="cuda") if x is not None else None for x in (target, draft, ua, us)]
    tk, rs = i32(torch, tokens), i32(torch, row_start)
    n = len(us)
    acc, out = i32(torch, np.full(n, -5)), i32(torch, np.full(rows, -9))
    if ws is None:
        ws = torch.zeros(R.verify_drafts_workspace(n, vocab), dtype=torch.uint8, device="cuda")
    for _ in range(2):  # the workspace serves call after call
        R.verify_drafts(ptr(d[0]), ld, ptr(d[1]), ld, ptr(tk), ptr(rs), n, rows, vocab, ptr(d[2]), ptr(d[3]), ptr(acc), ptr(out), ptr(ws),
                        ws.numel(), torch.cuda.current_stream().cuda_stream)
    want = plain_verify(np.asarray(target, np.float32)[:, :vocab], None if draft is None else np.asarray(draft, np.float32)[:, :vocab], tokens,
                        row_start, np.asarray(ua, np.float32), np.asarray(us, np.float32), vocab, np.full(rows, -9))
    assert acc.tolist() == want[0]
    spans = [(min(max(int(x), 0), rows), min(max(int(y), 0), rows)) for x, y in zip(row_start[:-1], row_start[1:])]
    once = [i for i in range(rows) if sum(x <= i < y for x, y in spans) <= 1]  # (rows that several claim hold one's output)
    got = out.tolist()
    assert [got[i] for i in once] == [want[1][i] for i in once]
    return want


@pytest.mark.parametrize("vocab", [1, 2, 100, 255, 1000, 1024, 4097, 32000, 151936])
@pytest.mark.parametrize("certain", [False, True])
def test_verify_follows_the_definition(torch, vocab, certain):
    rng = np.random.RandomState(vocab)
    counts = [5, 0, 1, 3, 9, 2, 1]
    row_start = np.concatenate([[0], np.cumsum(counts)])
    rows = int(row_start[-1]) + 2
    softmax = lambda x: np.exp(x - x.max(-1, keepdims=True)) / np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True)  # noqa: E731
    logits = 3 * rng.randn(rows, vocab)
    target = softmax(logits).astype(np.float32)
    draft = softmax(logits + 0.5 * rng.randn(rows, vocab)).astype(np.float32)
    tokens = np.zeros(rows, np.int64)
    for i in range(rows - 1):
        tokens[i + 1] = rng.choice(vocab, p=draft[i].astype(np.float64) / draft[i].astype(np.float64).sum())
    print(f"verify vocab {vocab} certain {certain}", flush=True)
    seen = set()
    for k in range(6):
        want = verify(torch, target, None if certain else draft, tokens, row_start, rng.rand(rows), rng.rand(7))
        seen |= {a - (c - 1) for a, c in zip(want[0], counts) if c > 1}
    assert vocab < 100 or len(seen) > 1  # some were refused, some not
    # a stride over the vocabulary: what lies behind it is not looked at
    if vocab > 2:
        verify(torch, target, None if certain else draft, np.minimum(tokens, vocab), row_start, rng.rand(rows), rng.rand(7), vocab=vocab - 1)


def test_verify_borders(torch):
    """Numbers on a border, of 0 and next to 1, ties, zeros, rows without weight, values that are not finite, tokens outside the vocabulary."""
    V = 3000
    p = np.zeros((12, V), np.float32)
    q = np.zeros((12, V), np.float32)
    p[:, [3, 700, 1023, 1024, 2999]] = [0.25, 0.25, 0.25, 0.125, 0.125]
    q[:, [3, 700]] = [0.5, 0.5]
    tokens = [0, 3, 700, 3, 0, 700, 0, -1, V, 5, 3, 0]
    below = float(np.nextafter(np.float32(1), np.float32(0)))
    row_start = [0, 4, 6, 8, 9, 12]
    for ua in (0.0, 0.25, 0.5, float(np.nextafter(np.float32(0.5), np.float32(0))), below):
        for us in (0.0, 0.25, 0.5, 0.75, 0.875, below, 1.0, 2.0, -1.0, float("nan")):
            verify(torch, p, q, tokens, row_start, np.full(12, ua), np.full(5, us))
            verify(torch, p, None, tokens, row_start, np.full(12, ua), np.full(5, us))
    same = p.copy()
    verify(torch, p, same, tokens, row_start, np.full(12, 1.0), np.full(5, 0.3))  # refused with nothing left: the target row
    verify(torch, np.zeros_like(p), q, tokens, row_start, np.full(12, 0.3), np.full(5, 0.3))
    odd = p.copy()
    odd[:, 5], odd[:, 9], odd[:, 11], odd[:, 13] = np.nan, np.inf, -np.inf, -1.0
    verify(torch, odd, q, tokens, row_start, np.full(12, 0.3), np.full(5, 0.6))
    qn = q.copy()
    qn[:, 3], qn[:, 1023] = np.nan, np.inf
    verify(torch, odd, qn, tokens, row_start, np.full(12, 0.3), np.full(5, 0.6))
    verify(torch, p, q, tokens, [-5, 3, 2, 2**31 - 1, 5, 2**31 - 1], np.full(12, 0.3), np.full(5, 0.6))  # spans of any values


def test_verify_gives_the_target_distribution(torch):
    """Given tokens follow the target whatever the draft says: 20000 draws over 8 tokens, each frequency within 5 standard deviations."""
    rng = np.random.RandomState(11)
    V, n = 8, 20000
    p, q = (x / x.sum() for x in (rng.rand(V), rng.rand(V)))
    tokens = np.zeros(2 * n, np.int64)
    tokens[1::2] = rng.choice(V, size=n, p=q)
    d = lambda x: torch.tensor(np.ascontiguousarray(x, dtype=np.float32), device="cuda")  # noqa: E731
    t, dr = d(np.tile(p, (2 * n, 1))), d(np.tile(q, (2 * n, 1)))
    ua, us = d(rng.rand(2 * n)), d(rng.rand(n))
    tk, rs, acc, out = i32(torch, tokens), i32(torch, np.arange(n + 1) * 2), i32(torch, np.zeros(n)), i32(torch, np.zeros(2 * n))
    ws = torch.zeros(R.verify_drafts_workspace(n, V), dtype=torch.uint8, device="cuda")
    R.verify_drafts(ptr(t), V, ptr(dr), V, ptr(tk), ptr(rs), n, 2 * n, V, ptr(ua), ptr(us), ptr(acc), ptr(out), ptr(ws), ws.numel())
    first = out.cpu().numpy()[0::2]
    freq = np.bincount(first, minlength=V) / n
    assert (np.abs(freq - p) <= 5 * np.sqrt(p * (1 - p) / n)).all()


def test_verify_workspace_serves_other_sizes(torch):
    """One workspace, zeroed once, for calls of more and fewer requests and of other vocabularies in turn."""
    rng = np.random.RandomState(3)
    ws = torch.zeros(R.verify_drafts_workspace(40, 40000), dtype=torch.uint8, device="cuda")
    for n, V in ((3, 40000), (40, 2000), (1, 40000), (40, 5000), (17, 100), (40, 40000), (2, 600), (40, 1)):
        p, q = (x / x.sum(-1, keepdims=True) for x in (rng.rand(3 * n, V), rng.rand(3 * n, V)))
        print("workspace", n, V, flush=True)
        verify(torch, p, q, rng.randint(0, V, 3 * n), np.arange(n + 1) * 3, rng.rand(3 * n), rng.rand(n), ws=ws)


@pytest.mark.parametrize("vocab", [700, 5000, 40000, 151936])
@pytest.mark.parametrize("refused", [False, True])
def test_verify_gives_tokens_that_have_a_weight(torch, vocab, refused):
    """Rows cut by a mask, in sums that no order of adding has exactly: u_sample of 1 and more gives the last token with a
    weight; a border at a sum in front of a masked stretch one of the two tokens beside the stretch."""
    rng = np.random.RandomState(vocab)
    n = 400 if vocab < 100000 else 60
    half, gap = vocab * 2 // 5, vocab // 20
    w = np.exp(4 * rng.randn(n, half)).astype(np.float32)
    w[:, rng.rand(half) < 0.3] = 0
    w[:, [0, -1]] = 1.0
    p = np.zeros((n, vocab), np.float32)  # weights, a masked stretch, the same weights, a masked tail
    p[:, :half], p[:, half + gap: 2 * half + gap] = w, w
    last, left, right = 2 * half + gap - 1, half - 1, half + gap
    counts = np.full(n, 2 if refused else 1)
    target, draft = np.repeat(p, counts, 0), None
    tokens = np.zeros(len(target), np.int64)
    if refused:  # a draft of weight 0 in front; q leaves half of every weight
        tokens[1::2] = vocab - 1
        draft = target / 2
    d = lambda x: torch.tensor(np.ascontiguousarray(x, dtype=np.float32), device="cuda") if x is not None else None  # noqa: E731
    dt, dd, ua = d(target), d(draft), d(np.ones(len(target)))
    tk, rs = i32(torch, tokens), i32(torch, np.concatenate([[0], np.cumsum(counts)]))
    acc, out = i32(torch, np.zeros(n)), i32(torch, np.zeros(len(target)))
    ws = torch.zeros(R.verify_drafts_workspace(n, vocab), dtype=torch.uint8, device="cuda")
    for u, want in ((1.0, (last,)), (2.0, (last,)), (float("inf"), (last,)), (0.5, (left, right)), (0.0, (0,))):
        us = d(np.full(n, u))
        R.verify_drafts(ptr(dt), vocab, ptr(dd), vocab, ptr(tk), ptr(rs), n, len(target), vocab, ptr(ua), ptr(us), ptr(acc), ptr(out),
                        ptr(ws), ws.numel(), torch.cuda.current_stream().cuda_stream)
        assert acc.tolist() == [0] * n
        got = set(out.cpu().numpy()[rs.cpu().numpy()[:-1]].tolist())
        assert got <= set(want), (u, got - set(want))
    # Numbers next to 1: whatever the sums' last bits are, no masked token.
    for u in (np.nextafter(np.float32(1), np.float32(0)), np.float32(0.999999)):
        us = d(np.full(n, u))
        R.verify_drafts(ptr(dt), vocab, ptr(dd), vocab, ptr(tk), ptr(rs), n, len(target), vocab, ptr(ua), ptr(us), ptr(acc), ptr(out),
                        ptr(ws), ws.numel(), torch.cuda.current_stream().cuda_stream)
        first = out.cpu().numpy()[rs.cpu().numpy()[:-1]]
        assert (p[np.arange(n), first] > 0).all()


@pytest.mark.parametrize("certain", [False, True])
def test_verify_values_that_are_no_probabilities(torch, certain):
    """Drafted tokens on target and draft values that are infinite, NaN, negative or 0. A target value that is not finite and
    positive counts 0; a negative draft value too; a draft value that is not finite refuses its token and leaves it no weight."""
    V = 64
    odd = [float("inf"), float("-inf"), float("nan"), -float("nan"), -0.5, -0.0, 0.0, 0.25]
    pairs = [(p, q) for p in odd for q in ([1.0] if certain else odd)]
    n = len(pairs)
    target, draft = np.full((2 * n, V), 0.0078125, np.float32), np.full((2 * n, V), 0.00390625, np.float32)
    for i, (p, q) in enumerate(pairs):
        target[2 * i, 40], draft[2 * i, 40] = p, q
    tokens = np.tile([0, 40], n)
    d = lambda x: torch.tensor(np.ascontiguousarray(x, dtype=np.float32), device="cuda") if x is not None else None  # noqa: E731
    dt, dd = d(target), None if certain else d(draft)
    tk, rs = i32(torch, tokens), i32(torch, np.arange(n + 1) * 2)
    ws = torch.zeros(R.verify_drafts_workspace(n, V), dtype=torch.uint8, device="cuda")
    for u in (0.0, 0.3, 1.0):
        for border in (0.45, 0.63):
            ua, us = d(np.full(2 * n, u)), d(np.full(n, border))
            acc, out = i32(torch, np.zeros(n)), i32(torch, np.full(2 * n, -9))
            R.verify_drafts(ptr(dt), V, ptr(dd), V, ptr(tk), ptr(rs), n, 2 * n, V, ptr(ua), ptr(us), ptr(acc), ptr(out), ptr(ws),
                            ws.numel(), torch.cuda.current_stream().cuda_stream)
            for i, (p, q) in enumerate(pairs):
                weight = target[2 * i].astype(np.float64)
                weight[40] = p if np.isfinite(p) and p > 0 else 0.0
                ok = bool(np.isfinite(q) and np.float64(np.float32(u)) * max(q, 0.0) < weight[40])
                assert acc[i].item() == ok, (p, q, u)
                if ok:
                    weight = target[2 * i + 1].astype(np.float64)
                elif certain:
                    weight[40] = 0
                else:
                    weight -= draft[2 * i]
                    weight[40] = max((p if np.isfinite(p) and p > 0 else 0.0) - max(q, 0.0), 0.0) if np.isfinite(q) else 0.0
                c = weight.cumsum()
                token = int((c <= np.float64(np.float32(border)) * c[-1]).sum())
                assert out[2 * i: 2 * i + 2].tolist() == ([40, token] if ok else [token, -1]), (p, q, u, border)


# ---------------------------------------------------------------------------
# The ops together
# ---------------------------------------------------------------------------
def test_steps_of_several_requests_match_the_runner(torch):
    """Prompts in chunks, drafts with some of them given back, and single tokens of three requests through a two-layer
    decoder of linear and these ops, against a Runner of the same weights for each request: 2e-3 of the largest logit, the
    bar of the other paths (an f32 cache, the same bf16 weights)."""
    cfg = C.Config(vocab_size=320, hidden_size=256, intermediate_size=384, num_hidden_layers=2, num_attention_heads=4,
                   num_key_value_heads=2, max_position_embeddings=128, rope_theta=10000.0, rms_norm_eps=1e-5, tie_word_embeddings=True)
    H, hd, kv, I, V = 256, 64, 2, 384, 320
    heads = 4
    blob = R.synthetic_blob(cfg, C.WEIGHT_BF16, seed=5, stddev=0.06)
    w = {(s, l): torch.from_numpy(blob[o:o + n].view(np.int16).copy()).cuda().view(torch.bfloat16)
         for s, l, o, n in R.dense_slices(cfg)}
    stacked = [torch.cat([w[(x, l)] for x in ("q", "k", "v")]) for l in range(2)]
    biases = [torch.cat([w[(x, l)] for x in ("q_bias", "k_bias", "v_bias")]) for l in range(2)]
    stream = torch.cuda.current_stream().cuda_stream
    ps, pages, n_req, most = 8, 24, 3, 64

    def linear(weight, x, n, k, bias=None):
        y = torch.empty(x.shape[0], n, device="cuda")
        R.linear(ptr(weight), ptr(x), ptr(y), x.shape[0], n, k, ptr(bias), stream)
        return y

    def rms(x, weight):
        return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * weight.float()).contiguous()

    inv = torch.tensor([1.0 / 10000.0 ** (2 * i / hd) for i in range(hd // 2)], dtype=torch.float32, device="cuda")
    caches = []
    for _ in range(2):
        k, v = (torch.full((pages * ps, kv * hd), float("nan"), device="cuda") for _ in range(2))
        caches.append((R.PagedCache(ptr(k), ptr(v), "f32", kv, hd, ps, pages), k, v))
    free, count, table = i32(torch, np.random.RandomState(0).permutation(pages)), i32(torch, [pages]), i32(torch, np.full((n_req, 12), -1))
    pool = R.PagePool(ptr(free), ptr(count), ptr(table), n_req, 12, ps, pages)
    length, row_start, start = i32(torch, np.zeros(3)), i32(torch, np.zeros(4)), i32(torch, np.zeros(3))
    pos, slots = i32(torch, np.zeros(most)), torch.zeros(most, dtype=torch.int64, device="cuda")
    ws = torch.zeros(R.paged_attention_workspace(most, n_req, heads, kv, hd), dtype=torch.uint8, device="cuda")

    def step(keep, tokens):
        """Logits of all new rows; `tokens` per request."""
        add = [len(t) for t in tokens]
        rows = sum(add)
        d_keep, d_add = i32(torch, keep), i32(torch, add)
        R.paged_assign(pool, ptr(length), ptr(d_keep), ptr(d_add), most, ptr(length), ptr(row_start), ptr(start), ptr(pos),
                       ptr(slots), stream)
        ids = torch.tensor([t for ts in tokens for t in ts], device="cuda")
        x = w[("embed", None)].view(V, H)[ids].float()
        for l, (c, _, _) in enumerate(caches):
            width = (heads + 2 * kv) * hd
            qkv = linear(stacked[l], rms(x, w[("input_norm", l)]), width, H, biases[l])
            b = ptr(qkv)
            R.norm_rope_append(c, b, width, b + 4 * H, width, b + 4 * (H + kv * hd), width, rows, heads, b, width, ptr(inv), ptr(pos),
                               ptr(slots), "split_half", None, None, 0.0, stream)
            o = torch.empty(rows, H, device="cuda")
            R.paged_attention(c, ptr(table), 12, ptr(row_start), ptr(start), n_req, b, width, ptr(o), H, rows, heads, hd ** -0.5, 0, ptr(ws),
                              ws.numel(), stream)
            x = x + linear(w[("o", l)], o, H, H)
            h = rms(x, w[("post_norm", l)])
            m = torch.nn.functional.silu(linear(w[("gate", l)], h, I, H)) * linear(w[("up", l)], h, I, H)
            x = x + linear(w[("down", l)], m.contiguous(), H, I)
        return linear(w[("embed", None)], rms(x, w[("final_norm", None)]), V, H)

    rng = np.random.RandomState(1)
    text = [rng.randint(0, V, n).tolist() for n in (40, 23, 31)]
    runners = [R.Runner(cfg, blob, 128) for _ in range(n_req)]
    done = [0, 0, 0]

    def compare(tokens, logits):
        at = 0
        for r, ts in enumerate(tokens):
            for i, t in enumerate(ts):
                want = runners[r].forward_token(int(t), done[r] + i)
                err = np.abs(logits[at].cpu().numpy() - want).max() / np.abs(want).max()
                assert err <= 2e-3, (r, done[r] + i, err)
                at += 1

    # prompts in chunks; the third request starts a step later
    for chunk in ([text[0][:17], text[1][:23], []], [text[0][17:30], [], text[2][:20]], [[text[0][30]], [5], text[2][20:30]]):
        logits = step(done, chunk)
        compare(chunk, logits)
        done = [d + len(c) for d, c in zip(done, chunk)]
    # tokens with drafts, checked against the target's probabilities; what is refused goes back
    for k in range(4):
        drafts = [[int(t) for t in rng.randint(0, V, n)] for n in (4, 1, 3)]
        logits = step(done, drafts)
        compare(drafts, logits)
        p = torch.softmax(logits, -1)
        tk = i32(torch, [t for d in drafts for t in d])
        # drafts that the target likes: its own best tokens, for the first rows
        q = torch.softmax(logits + 0.3 * torch.randn_like(logits), -1)
        ua, us = torch.rand(8, device="cuda"), torch.rand(3, device="cuda")
        acc, out = i32(torch, np.zeros(3)), i32(torch, np.zeros(8))
        vw = torch.zeros(R.verify_drafts_workspace(3, V), dtype=torch.uint8, device="cuda")
        R.verify_drafts(ptr(p), V, ptr(q), V, ptr(tk), ptr(row_start), 3, 8, V, ptr(ua), ptr(us), ptr(acc), ptr(out), ptr(vw), vw.numel(),
                        stream)
        want = plain_verify(p.cpu().numpy(), q.cpu().numpy(), tk.cpu().numpy(), row_start.cpu().numpy(), ua.cpu().numpy(), us.cpu().numpy(), V,
                            np.zeros(8))
        assert acc.tolist() == want[0] and out.tolist() == want[1]
        done = [d + 1 + a for d, a in zip(done, acc.tolist())]  # the next step keeps the token and its accepted drafts
    assert all(a >= b for a, b in zip(length.tolist(), done))
    for r in runners:
        r.close()


def test_steps_with_a_dry_pool_and_idle_requests(torch):
    """The loop of assign and verify as a host keeps it: a request that got its rows keeps them up to the last accepted draft
    (all of a prompt's); one that had none, or that the pool had no pages for, keeps what it kept before and offers its rows
    again; where nobody gets pages the last one gives up its own and starts again from its text. The calls give what plain
    ones give, and every request gets to its end."""
    rng = np.random.RandomState(5)
    n, ps, stride, pages, V, most, goal = 6, 4, 12, 26, 50, 256, 34
    pool = Pool(torch, n, stride, ps, pages)
    rs, st, pos = i32(torch, np.zeros(n + 1)), i32(torch, np.zeros(n)), i32(torch, np.zeros(most))
    slots = torch.zeros(most, dtype=torch.int64, device="cuda")
    vw = torch.zeros(R.verify_drafts_workspace(n, V), dtype=torch.uint8, device="cuda")
    acc, out = i32(torch, np.zeros(n)), i32(torch, np.zeros(most))
    stream = torch.cuda.current_stream().cuda_stream
    text = [rng.randint(0, V, 3 + r).tolist() for r in range(n)]  # the last token is never in the cache
    keep, waited, idle, restarts = np.zeros(n, np.int64), 0, 0, 0
    for step in range(400):
        ended = [len(t) > goal for t in text]
        if all(ended):
            break
        offered, prompt = [], []
        for r in range(n):
            if ended[r]:
                keep[r] = 0  # its pages go to the others
            prompt.append(keep[r] < len(text[r]) - 1)
            if ended[r] or rng.rand() < 0.2:
                offered.append([])
            elif prompt[r]:
                offered.append(text[r][keep[r]: -1])
            else:
                offered.append(text[r][-1:] + rng.randint(0, V, rng.randint(0, 4)).tolist())
        add = [len(x) for x in offered]
        held = pool.d_len.cpu().numpy().astype(np.int64)
        flat = np.array([t for x in offered for t in x] + [0] * (most - sum(add)))
        p, q, ua, us = (rng.rand(*s).astype(np.float32) for s in ((most, V), (most, V), (most,), (n,)))
        d = [i32(torch, keep), i32(torch, add), i32(torch, flat), *(torch.tensor(x, device="cuda") for x in (p, q, ua, us))]
        R.paged_assign(pool.handle, ptr(pool.d_len), ptr(d[0]), ptr(d[1]), most, ptr(pool.d_len), ptr(rs), ptr(st), ptr(pos), ptr(slots), stream)
        R.verify_drafts(ptr(d[3]), V, ptr(d[4]), V, ptr(d[2]), ptr(rs), n, most, V, ptr(d[5]), ptr(d[6]), ptr(acc), ptr(out), ptr(vw),
                        vw.numel(), stream)
        want = plain_assign(pool.stack, pool.table, ps, pages, held, keep, add, most)
        start, length, first = st.tolist(), pool.d_len.tolist(), rs.tolist()
        assert start == want[2] and length == want[0] and first == want[1]
        accepted, given = acc.tolist(), out.tolist()
        plain = plain_verify(p, q, flat, first, ua, us, V, np.zeros(most))
        assert accepted == plain[0] and given[: first[n]] == plain[1][: first[n]]
        moved = False
        for r in range(n):
            if add[r] and start[r] >= 0:
                moved = True
                if prompt[r]:
                    keep[r] = length[r]
                else:
                    keep[r] = start[r] + 1 + accepted[r]
                    text[r] += given[first[r]: first[r] + accepted[r] + 1]
                assert keep[r] == len(text[r]) - 1 <= length[r]
            else:
                waited, idle = waited + (add[r] > 0), idle + (add[r] == 0)
                assert length[r] == (held[r] if add[r] else keep[r])
        if not moved and any(add):
            keep[max(r for r in range(n) if not ended[r] and length[r])] = 0
            restarts += 1
    assert all(len(t) > goal for t in text), [len(t) for t in text]
    print(f"{step} steps, {waited} without pages, {idle} idle, {restarts} restarts", flush=True)
    assert waited > 5 and idle > 20


def test_captured_step_follows_the_eager_one(torch):
    """A whole step in one graph, for batches of fewer rows than it has room for: pages, cache, outputs and tokens are those of eager
    calls over the same inputs, replay by replay, with eager work between."""
    n, heads, kv, hd, ps, pages, stride, most, V = 4, 8, 2, 64, 8, 40, 16, 48, 3000
    width = (heads + 2 * kv) * hd
    g = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *shape: torch.rand(*shape, device="cuda", generator=g)  # noqa: E731
    order = np.random.RandomState(4).permutation(pages)
    keep, add, qkv, inv = i32(torch, np.zeros(n)), i32(torch, np.zeros(n)), torch.zeros(most, width, device="cuda"), rnd(hd // 2)
    target, draft, tokens, ua, us = rnd(most, V), rnd(most, V), i32(torch, np.zeros(most)), rnd(most), rnd(n)

    class Side:
        def __init__(self):
            self.free, self.count, self.table = i32(torch, order), i32(torch, [pages]), i32(torch, np.full((n, stride), -1))
            self.len, self.row_start, self.start = i32(torch, np.zeros(n)), i32(torch, np.zeros(n + 1)), i32(torch, np.zeros(n))
            self.pos, self.slots = i32(torch, np.zeros(most)), torch.zeros(most, dtype=torch.int64, device="cuda")
            self.k, self.v = (torch.zeros(pages * ps, kv * hd, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            self.q, self.out = (torch.zeros(most, heads * hd, device="cuda") for _ in range(2))
            self.acc, self.tok = i32(torch, np.zeros(n)), i32(torch, np.zeros(most))
            self.aw = torch.zeros(R.paged_attention_workspace(most, n, heads, kv, hd), dtype=torch.uint8, device="cuda")
            self.vw = torch.zeros(R.verify_drafts_workspace(n, V), dtype=torch.uint8, device="cuda")

        def step(self):
            s = torch.cuda.current_stream().cuda_stream
            pool = R.PagePool(ptr(self.free), ptr(self.count), ptr(self.table), n, stride, ps, pages)
            c = R.PagedCache(ptr(self.k), ptr(self.v), "bf16", kv, hd, ps, pages)
            self.slots.fill_(-1)
            R.paged_assign(pool, ptr(self.len), ptr(keep), ptr(add), most, ptr(self.len), ptr(self.row_start), ptr(self.start), ptr(self.pos),
                           ptr(self.slots), s)
            b = ptr(qkv)
            R.norm_rope_append(c, b, width, b + 4 * heads * hd, width, b + 4 * (heads + kv) * hd, width, most, heads, ptr(self.q), heads * hd,
                               ptr(inv), ptr(self.pos), ptr(self.slots), "split_half", None, None, 0.0, s)
            R.paged_attention(c, ptr(self.table), stride, ptr(self.row_start), ptr(self.start), n, ptr(self.q), heads * hd, ptr(self.out),
                              heads * hd, most, heads, hd ** -0.5, 0, ptr(self.aw), self.aw.numel(), s)
            R.verify_drafts(ptr(target), V, ptr(draft), V, ptr(tokens), ptr(self.row_start), n, most, V, ptr(ua), ptr(us), ptr(self.acc),
                            ptr(self.tok), ptr(self.vw), self.vw.numel(), s)

        def state(self):
            return {x: getattr(self, x).clone() for x in ("free", "count", "table", "len", "row_start", "start", "slots", "k", "v", "out",
                                                          "acc", "tok")}

    captured, eager = Side(), Side()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        captured.step()  # (no request has rows yet)
        eager.step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    rng = np.random.RandomState(9)
    for i, new in enumerate([(17, 5, 0, 26), (1, 9, 30, 1), (3, 0, 1, 3), (1, 1, 1, 1), (0, 40, 2, 1), (5, 1, 1, 5)]):
        held = eager.len.cpu().numpy()
        kept = np.maximum(held - rng.randint(0, 3, n), 0)
        if i == 3:
            kept[0] = 0  # a request that has ended, and the next one in its place
        keep.copy_(i32(torch, kept)), add.copy_(i32(torch, new)), tokens.copy_(i32(torch, rng.randint(0, V, most)))
        qkv.copy_(torch.randn(most, width, device="cuda", generator=g)), ua.copy_(rnd(most)), us.copy_(rnd(n))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager.step()
        torch.cuda.synchronize()
        a, b = captured.state(), eager.state()
        for x in a:
            assert torch.equal(a[x], b[x]), (i, x)
        rows = int(b["row_start"][-1])
        assert rows == sum(new) and bool((b["slots"][:rows] >= 0).all()) and bool((b["slots"][rows:] == -1).all())
