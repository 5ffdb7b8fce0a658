"""Ops around 8-bit products without a GPU: the refusals of their entry points
and the arithmetic behind them."""
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from vvli_amd import runtime as R
from vvli_amd._lib import VvliError

ROOT = Path(__file__).resolve().parents[1]
P = 0x100000  # addresses that no refused call looks behind
Q, S, T, U = 16 * P, 32 * P, 48 * P, 64 * P

CONFIG, NULL = "InvalidConfig", "NullArgument"


def refused(call, name, **kw):
    with pytest.raises(VvliError) as e:
        call(**kw)
    assert e.value.name == name, str(e.value)


def quantize(**kw):
    a = dict(x=P, kind="f32", ldx=64, rows=3, width=50, codes=Q, ldc=64, scales=S)
    a.update(kw)
    R.quantize_rows(**a)


def norm(**kw):
    a = dict(x=P, ldx=64, delta=Q, ldd=64, rows=3, width=50, weight=S, weight_kind="f32", eps=1e-6, total=T, lds=64, y=None, ldy=0,
             codes=U, ldc=64, scales=2 * U)
    a.update(kw)
    R.add_norm(**a)


def gate(**kw):
    a = dict(gate=P, ldg=128, up=P + 4 * 64, ldu=128, rows=3, width=50, codes=Q, ldc=64, scales=S)
    a.update(kw)
    R.silu_mul(**a)


def linear(**kw):
    a = dict(W=P, ldw=1024, w_scales=Q, X=S, ldx=1024, x_scales=T, bias=None, Y=U, ldy=40, M=50, N=40, K=1024, workspace=2 * U,
             workspace_bytes=1 << 30)
    a.update(kw)
    R.linear_i8(**a)


CODES = [(dict(codes=None), NULL), (dict(scales=None), NULL), (dict(ldc=48), CONFIG), (dict(ldc=72), CONFIG), (dict(codes=Q + 8), CONFIG),
         (dict(ldc=1 << 31), CONFIG), (dict(width=65), CONFIG)]
SIZES = [(dict(rows=1 << 31), CONFIG), (dict(width=0), CONFIG), (dict(width=(1 << 31) - 1, ldx=1 << 31), CONFIG)]


@pytest.mark.parametrize("bad,name", CODES + SIZES + [
    (dict(x=None), NULL), (dict(x=P + 4), CONFIG), (dict(ldx=49), CONFIG), (dict(ldx=50), CONFIG), (dict(ldx=48), CONFIG),
    (dict(ldx=60, kind="bf16"), CONFIG), (dict(ldx=1 << 31), CONFIG),
    (dict(codes=P), CONFIG), (dict(codes=P + 3 * 256 - 64), CONFIG), (dict(scales=P + 4), CONFIG), (dict(scales=Q + 8), CONFIG),
])
def test_quantize_rows_refusals(bad, name):
    refused(quantize, name, **bad)


def test_quantize_rows_unknown_kind():
    from vvli_amd import _lib

    assert _lib.lib().vvli_gpu_quantize_rows(P, 2, 64, 3, 50, Q, 64, S, None) == 1


@pytest.mark.parametrize("bad,name", CODES[:2] + CODES[2:4] + [(dict(codes=U + 8), CONFIG)] + SIZES[:2] + [
    (dict(x=None), NULL), (dict(weight=None), NULL), (dict(weight=S + 8), CONFIG), (dict(x=P + 8), CONFIG), (dict(ldx=48), CONFIG),
    (dict(ldd=54), CONFIG), (dict(delta=Q + 4), CONFIG), (dict(total=T + 4), CONFIG), (dict(lds=48), CONFIG), (dict(y=3 * U, ldy=48), CONFIG),
    (dict(y=3 * U + 4, ldy=64), CONFIG), (dict(eps=-1e-6), CONFIG), (dict(eps=float("nan")), CONFIG), (dict(eps=float("inf")), CONFIG),
    (dict(delta=None), CONFIG),                              # a sum without delta
    (dict(codes=None, scales=None), NULL),                   # nothing to compute
    (dict(y=3 * U, ldy=64, codes=None), NULL), (dict(y=3 * U, ldy=64, scales=None), NULL),
    (dict(total=P, lds=128), CONFIG), (dict(total=Q, lds=128), CONFIG),       # in place with another stride
    (dict(total=P + 16), CONFIG), (dict(y=P + 256, ldy=64), CONFIG),          # shifted
    (dict(y=T, ldy=64), CONFIG), (dict(total=P, y=P, ldy=64), CONFIG),        # sum and y in one place
    (dict(codes=P), CONFIG), (dict(codes=Q), CONFIG), (dict(codes=T), CONFIG), (dict(scales=P), CONFIG), (dict(codes=S), CONFIG),
    (dict(total=S), CONFIG), (dict(scales=S + 100), CONFIG),
])
def test_add_norm_refusals(bad, name):
    refused(norm, name, **bad)


@pytest.mark.parametrize("place", [P, Q], ids=["x", "delta"])
@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("others", [dict(total=None), dict(), dict(total=None, y=3 * U, ldy=64), dict(y=3 * U, ldy=64)],
                         ids=["codes alone", "sum", "y", "sum and y"])
def test_add_norm_refuses_codes_in_place(place, rows, others):
    """sum and y may lie where x or delta does, codes may not, whatever their stride."""
    for ldc in (64, 128, 256, 512):
        refused(norm, CONFIG, codes=place, ldc=ldc, rows=rows, **others)


def test_add_norm_unknown_weight_kind():
    from vvli_amd import _lib

    assert _lib.lib().vvli_gpu_add_norm(P, 64, None, 0, 3, 50, S, 2, 1e-6, None, 0, None, 0, U, 64, 2 * U, None) == 1


@pytest.mark.parametrize("bad,name", CODES[:6] + SIZES[:2] + [
    (dict(gate=None), NULL), (dict(up=None), NULL), (dict(gate=P + 4), CONFIG), (dict(up=P + 8), CONFIG), (dict(ldg=48), CONFIG),
    (dict(ldu=130), CONFIG), (dict(codes=P), CONFIG), (dict(codes=P + 256), CONFIG), (dict(scales=P), CONFIG),
])
def test_silu_mul_refusals(bad, name):
    refused(gate, name, **bad)


@pytest.mark.parametrize("bad,name", [
    (dict(W=None), NULL), (dict(w_scales=None), NULL), (dict(X=None), NULL), (dict(x_scales=None), NULL), (dict(Y=None), NULL),
    (dict(workspace=None), NULL), (dict(N=0), CONFIG), (dict(K=0), CONFIG), (dict(K=56), CONFIG), (dict(M=1 << 31), CONFIG),
    (dict(K=131072, ldw=131072, ldx=131072), CONFIG), (dict(K=1040), CONFIG), (dict(ldw=1032), CONFIG), (dict(ldx=1008), CONFIG),
    (dict(ldw=1 << 31), CONFIG), (dict(W=P + 8), CONFIG), (dict(X=S + 4), CONFIG), (dict(ldy=39), CONFIG), (dict(ldy=1 << 31), CONFIG),
    (dict(workspace=2 * U + 8), CONFIG), (dict(workspace_bytes=0), CONFIG), (dict(Y=P), CONFIG), (dict(Y=S + 64), CONFIG), (dict(Y=Q), CONFIG),
    (dict(Y=T), CONFIG), (dict(bias=U + 8), CONFIG), (dict(Y=2 * U + 4), CONFIG), (dict(N=1 << 31, ldy=1 << 31), CONFIG),
    (dict(workspace=P), CONFIG), (dict(workspace=S - 16), CONFIG), (dict(workspace=Q), CONFIG), (dict(workspace=T), CONFIG),
    (dict(bias=2 * U + 2), CONFIG),
])
def test_linear_i8_refusals(bad, name):
    refused(linear, name, **bad)


def test_linear_i8_workspace():
    assert R.linear_i8_workspace(1, 16, 16) == R.linear_i8_workspace(32, 16, 131056) == R.linear_i8_workspace(5000, 16, 512) == 0
    assert R.linear_i8_workspace(300, 0, 4096) == R.linear_i8_workspace(300, 16, 4104) == R.linear_i8_workspace(300, 16, 131072) == 0
    assert R.linear_i8_workspace(300, 16, 4096) > 0
    ms, ns, ks = (1, 32, 33, 64, 65, 300, 2000, 100000), (1, 16, 896, 3584, 40000, 200000), (16, 1008, 1024, 4096, 131056)
    for n in ns:  # it serves calls of any sizes up to its own
        for k in ks:
            sizes = [R.linear_i8_workspace(m, n, k) for m in ms]
            assert sizes == sorted(sizes) and max(sizes) <= 64 << 20
            assert all(R.linear_i8_workspace(m, n, k) <= R.linear_i8_workspace(m, 2 * n, k) for m in ms)
    for m in ms:
        sizes = [R.linear_i8_workspace(m, 896, k) for k in ks]
        assert sizes == sorted(sizes)


PLAN = """
#include "linear_i8_plan.hpp"
#include <cstdio>
int main() {
    unsigned long long m, n, k, ld;
    unsigned cus;
    while (scanf("%llu %llu %llu %llu %u", &m, &n, &k, &ld, &cus) == 5) {
        const vvli::I8Plan p = vvli::i8_plan(m, n, k, ld, cus);
        const vvli::I8Kernel& x = vvli::kI8Kernels[p.kernel];
        printf("%u %u %llu %d %d %d %d %llu %u %llu\\n", p.kernel, p.splits, (unsigned long long)p.blocks, (int)x.kind, x.r, x.m, x.split,
               (unsigned long long)vvli::i8_part_bytes(m, n, k), vvli::kI8KernelCount,
               (unsigned long long)p.cut);
    }
}
"""


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "t.cpp").write_text(PLAN)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'vvli_amd' / 'csrc'}", "-o", d / "t", d / "t.cpp"], check=True)

    def ask(sizes):
        text = "\n".join(" ".join(map(str, s)) for s in sizes)
        out = subprocess.run([d / "t"], input=text, capture_output=True, text=True, check=True).stdout.split("\n")
        return [tuple(map(int, line.split())) for line in out if line]

    return ask


# (M, N, K) of two calls for each kernel: odd sizes, K that ends inside a step, an odd number of tiles.
ODD = [(1, 33, 432), (5, 413, 2672), (35, 39, 624), (109, 365, 1120), (153, 43, 752), (161, 189, 3904), (1, 24713, 16),
       (1, 29723, 912), (1, 31, 16), (65, 169, 48), (173, 95, 16), (67, 32037, 16), (441, 41, 848), (209, 1751, 992),
       (261, 41, 480), (217, 725, 832), (323, 5905, 16), (129, 2383, 1936), (263, 43, 288), (861, 475, 832),
       (33, 24827, 16), (55, 32197, 208), (857, 9191, 16), (1371, 3365, 2800), (145, 41, 16), (311, 1461, 32),
       (461, 14459, 144), (295, 18253, 928), (189, 39433, 656), (395, 18565, 2480), (61, 33, 18576), (311, 401, 6768),
       (3017, 75, 10976), (687, 875, 14512), (181, 5555, 10272), (623, 3541, 16112),
       (1207, 6409, 608), (847, 2359, 1504), (395, 27229, 512), (1393, 9401, 1472), (65, 16505, 592), (133, 17291, 576),
       (131, 34373, 672), (155, 33383, 576), (133, 21, 9328), (149, 179, 16128), (73, 2793, 9920), (139, 5585, 8944)]

# Two launches of columns, the second a split K, a stream and small tiles.
CUT = [(393, 32779, 3616), (537, 21815, 4688), (409, 33031, 1728), (431, 37029, 1072), (387, 33589, 1296)]

# Results of more than 128 MiB by each of the large tiles (the last two: in two launches).
LONG = [(3551, 9743, 112), (37293, 909, 192), (683, 49517, 224), (13293, 2641, 928), (11015, 3213, 880), (645, 54647, 912),
        (1161, 29417, 1232), (669, 51443, 1168)]


def test_odd_sizes_reach_every_kernel(plan):
    got = plan([(m, n, k, max(k, 4 * n), 256) for m, n, k in ODD])
    assert {g[0] for g in got} == set(range(got[0][8])) and not any(g[9] for g in got)
    assert all(g[9] for g in plan([(m, n, k, 4 * n, 256) for m, n, k in CUT + LONG[-2:]]))
    assert all(m * n * 4 > 128 << 20 for m, n, _ in LONG)
    tiles = {(g[4], g[5]) for g in plan([(m, n, k, 4 * n, 256) for m, n, k in LONG])}
    assert tiles == {(2, 2), (3, 2), (4, 2), (3, 4), (4, 3), (4, 4)}


def test_every_kernel_is_taken_somewhere(plan):
    ms = [1, 2, 5, 8, 9, 16, 17, 24, 32, 33, 48, 64, 96, 128, 192, 256, 384, 512, 768, 1024, 1536, 2048, 4096]
    shapes = [(1152, 896), (896, 4864), (9728, 896), (2048, 2048), (2048, 8192), (16384, 2048), (4608, 3584), (3584, 18944), (37888, 3584),
              (128, 1024), (40, 131056), (128256, 2048)]
    got = plan([(m, n, k, max(k, 4 * n), 256) for m in ms for n, k in shapes])
    assert {g[0] for g in got} == set(range(got[0][8]))


def test_plans_fit_their_calls(plan):
    """Parts fit the workspace, parts have steps, tiles only where their buffers reach, few rows need nothing."""
    rng = np.random.RandomState(1)
    sizes = []
    for _ in range(4000):
        m, n = (int(np.exp(rng.uniform(0, np.log(200000)))) for _ in range(2))
        k = 16 * int(np.exp(rng.uniform(0, np.log(8191))))
        ld = max(k, 4 * n, int(np.exp(rng.uniform(0, np.log(2 ** 30)))))
        sizes.append((m, n, k, ld, int(rng.choice([256, 64, 304]))))
    cuts = 0
    for (m, n, k, ld, cus), (kernel, splits, blocks, kind, r, c, split, room, _, cut) in zip(sizes, plan(sizes)):
        if cut:  # whole rounds of large tiles, columns left for the next launch
            assert kind == 1 and not split and 0 < cut < n and cut % (64 * r) == 0 and blocks <= -(-n // (64 * r)) * -(-m // (64 * c)) // cus * cus
            n, cuts = cut, cuts + 1
        assert blocks > 0 and (splits > 1) == bool(split)
        if split:
            assert splits * m * n * 4 <= room and k >= 512 * splits and m > 32
        if kind == 1:
            assert ld * 256 <= 1 << 30 and m > 32
            assert blocks == splits * -(-n // (64 * r)) * -(-m // (64 * c))
        else:
            assert blocks == -(-(-(-n // (16 * r))) // 8) * 8 * -(-m // (8 * c))
    assert cuts > 20


def test_no_rows_launch_nothing():
    """(An address that nothing is behind: a launch would fail, here without a GPU and there with one.)"""
    quantize(rows=0)
    norm(rows=0)
    gate(rows=0)
    linear(M=0)


HARNESS = """
#include "row_bytes.hpp"
#include <cstdio>
int main() {
    unsigned long long p, lp, wp, rp, q, lq, wq, rq;
    while (scanf("%llu %llu %llu %llu %llu %llu %llu %llu", &p, &lp, &wp, &rp, &q, &lq, &wq, &rq) == 8)
        printf("%d\\n", vvli::rows_meet(vvli::RowBytes{(void*)p, lp, wp, rp}, vvli::RowBytes{(void*)q, lq, wq, rq}));
}
"""


@pytest.mark.skipif(not shutil.which("g++"), reason="no host compiler")
def test_rows_that_share_bytes_are_found(tmp_path):
    """Against sets of bytes: of one stride exactly, of two strides wherever the ranges meet."""
    (tmp_path / "t.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'vvli_amd' / 'csrc'}", "-o", tmp_path / "t", tmp_path / "t.cpp"], check=True)
    rng = np.random.RandomState(3)
    cases = []
    for _ in range(4000):
        la, lb = rng.randint(1, 12), rng.randint(1, 12)
        lb = la if rng.rand() < 0.7 else lb
        cases.append((100 + rng.randint(0, 60), la, rng.randint(1, la + 1), rng.randint(0, 5), 100 + rng.randint(0, 60), lb,
                      rng.randint(1, lb + 1), rng.randint(0, 5)))
    out = subprocess.run([tmp_path / "t"], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True,
                         check=True).stdout.split()
    met = beside = 0
    for (p, lp, wp, rp, q, lq, wq, rq), got in zip(cases, out):
        a = {p + i * lp + e for i in range(rp) for e in range(wp)}
        b = {q + i * lq + e for i in range(rq) for e in range(wq)}
        ranges = bool(a and b) and max(min(a), min(b)) <= min(max(a), max(b))
        want = bool(a & b)
        if lp != lq:
            assert int(got) == ranges
        elif want:
            assert int(got) == 1, (p, lp, wp, rp, q, lq, wq, rq)
            met += 1
        elif int(got):  # only where a row beyond the last would share one
            a = {p + i * lp + e for i in range(-9, rp + 9) for e in range(wp)}
            assert ranges and a & {q + i * lq + e for i in range(-9, rq + 9) for e in range(wq)}
        else:
            beside += ranges
    assert met > 100 and beside > 50


# Calls that leave parts of K in their workspace: tiles of each of the three sizes that have them, rows of results that are
# whole units and not.
SPLIT = [(311, 401, 6768), (687, 875, 14512), (300, 64, 131056), (623, 3541, 16112), (133, 21, 9328), (181, 5555, 10272),
         (61, 33, 18576), (448, 3584, 18944), (256, 3584, 18944)]


def test_split_sizes_leave_parts(plan):
    got = plan([(m, n, k, max(k, 4 * n), 256) for m, n, k in SPLIT])
    assert all(g[1] > 1 and g[6] for g in got)
    assert {(g[4], g[5]) for g in got} == {(1, 1), (2, 2), (4, 4)}
    assert {n % 4 == 0 for _, n, _ in SPLIT} == {True, False}
    for (m, n, k), g in zip(SPLIT, got):
        assert 0 < g[1] * m * n * 4 <= R.linear_i8_workspace(m, n, k)


# Sizes (M, N, K) with a stride of more than 4 MiB of W, X or Y, whose rows of a tile are behind what a tile's offsets reach.
FAR_STRIDE = (1 << 22) + 16  # bytes
FAR = [(33, 300, 64), (40, 65, 1040), (300, 40, 64), (300, 300, 1040), (1000, 33, 272)]


def test_far_strides_take_streams(plan):
    for ld, kinds in ((FAR_STRIDE, {0}), (1 << 22, {0, 1})):
        assert {g[3] for g in plan([(m, n, k, ld, 256) for m, n, k in FAR])} == kinds


LAUNCHES = """
#include "linear_i8_plan.hpp"
#include <cstdio>
int main() {
    unsigned long long m, n, k, ld;
    unsigned cus;
    int stop;
    while (scanf("%llu %llu %llu %llu %u %d", &m, &n, &k, &ld, &cus, &stop) == 6) {
        auto f = [&](const vvli::I8Plan& p, uint64_t m0, uint64_t M, uint64_t n0, uint64_t N) {
            printf("%u,%u,%llu,%llu,%llu,%llu,%llu ", p.kernel, p.splits, (unsigned long long)p.blocks, (unsigned long long)m0,
                   (unsigned long long)M, (unsigned long long)n0, (unsigned long long)N);
            return --stop != 0;
        };
        printf("%d\\n", (int)vvli::i8_launches(m, n, k, ld, cus, f));
    }
}
"""

# More columns, or rows, than one launch has blocks for.
HUGE = [(1, (1 << 27) + 21, 16), (1, (1 << 27) + 24, 32), ((1 << 29) + 5, 1, 16)]


def test_launches_cover_their_call_once(tmp_path):
    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    (tmp_path / "t.cpp").write_text(LAUNCHES)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT / 'vvli_amd' / 'csrc'}", "-o", tmp_path / "t", tmp_path / "t.cpp"], check=True)
    rng = np.random.RandomState(5)
    most = (1 << 31) - 1
    calls = HUGE + CUT + LONG + ODD + SPLIT + [(1, most, 16), (most, 1, 16), (40, most, 16), (most, 40, 16)]
    while len(calls) < 1000:
        m, n = (int(np.exp(rng.uniform(0, np.log(most)))) for _ in range(2))
        if m * n < 1 << 42:
            calls.append((m, n, 16 * int(np.exp(rng.uniform(0, np.log(8191))))))

    def ask(calls, stop):
        text = "\n".join(f"{m} {n} {k} {max(k, 4 * n)} 256 {stop}" for m, n, k in calls)
        out = subprocess.run([tmp_path / "t"], input=text, capture_output=True, text=True, check=True).stdout.split("\n")
        return [([tuple(map(int, x.split(","))) for x in line.split()[:-1]], line.split()[-1] == "1") for line in out if line]

    for (m, n, k), (got, whole) in zip(calls, ask(calls, 0)):
        assert whole and all(blocks < 1 << 23 for _, _, blocks, *_ in got)
        assert all(M and N and m0 % 256 == 0 and n0 % 64 == 0 and m0 + M <= m and n0 + N <= n for *_, m0, M, n0, N in got)
        assert sum(M * N for *_, M, _, N in got) == m * n
        for i, (*_, m0, M, n0, N) in enumerate(got):
            assert all(m0 + M <= m1 or m1 + M1 <= m0 or n0 + N <= n1 or n1 + N1 <= n0 for *_, m1, M1, n1, N1 in got[:i])
        assert len(got) > 1 or (m, n, k) not in HUGE + CUT
    for got, whole in ask(HUGE + CUT, 1):  # a launch that fails is the last
        assert len(got) == 1 and not whole
