"""Ops for several requests over a paged cache, without a GPU: the refusals of
their entry points and the index arithmetic that their kernels use."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

from vvli_amd import runtime as R
from vvli_amd._lib import VvliError

ROOT = Path(__file__).resolve().parents[1]
P = 0x10000  # an address that no refused call looks behind

CONFIG, NULL = "InvalidConfig", "NullArgument"


def cache(k=P, v=P, kind="bf16", kv=2, hd=64, ps=16, pages=8, stride=None):
    return R.PagedCache(k, v, kind, kv, hd, ps, pages, stride)


BAD_CACHES = [
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(kv=0), CONFIG), (dict(kv=65536), CONFIG), (dict(hd=48), CONFIG),
    (dict(hd=256), CONFIG), (dict(hd=0), CONFIG), (dict(ps=0), CONFIG), (dict(pages=0), CONFIG),
    (dict(ps=1 << 16, pages=1 << 15), CONFIG), (dict(stride=127), CONFIG), (dict(stride=132), CONFIG),
    (dict(kind="f32", stride=130), CONFIG), (dict(k=P + 8), CONFIG), (dict(v=P + 2), CONFIG), (dict(stride=1 << 31), CONFIG),
]


def norm(c=None, **kw):
    a = dict(q=P, ldq=256, k=P, ldk=128, v=P, ldv=128, rows=3, heads=4, q_out=P, ldo=256, inv_freq=P, pos=P, slots=P,
             rope_layout="interleaved", q_norm=None, k_norm=None, eps=1e-6)
    a.update(kw)
    R.norm_rope_append(c or cache(), **a)


def attend(c=None, **kw):
    a = dict(table=P, table_stride=4, row_start=P, start_pos=P, requests=2, q=P, ldq=256, out=P, ldo=256, rows=3, heads=4,
             scale=0.125, window=0, workspace=P, workspace_bytes=1 << 40)
    a.update(kw)
    R.paged_attention(c or cache(), **a)


def assign(pool=None, **kw):
    a = dict(held=P, keep=P, add=P, rows=4, length=P, row_start=P, start_pos=P, row_pos=P, slots=P)
    a.update(kw)
    p = dict(free_pages=P, free_count=P, table=P, requests=2, table_stride=4, page_size=16, pages=8)
    p.update(pool or {})
    R.paged_assign(R.PagePool(**p), **a)


def verify(**kw):
    a = dict(target=P, ldt=100, draft=P, ldd=100, tokens=P, row_start=P, requests=2, rows=5, vocab=100, u_accept=P, u_sample=P,
             accepted=P, out=2 * P, workspace=P, workspace_bytes=1 << 40)
    a.update(kw)
    R.verify_drafts(**a)


@pytest.mark.parametrize("bad,name", BAD_CACHES)
def test_bad_caches_are_refused(bad, name):
    for call in (norm, attend):
        with pytest.raises(VvliError) as e:
            call(cache(**bad))
        assert e.value.name == name


def test_unknown_cache_kind_is_refused():
    c = cache()
    c._c.kind = 3
    for call in (norm, attend):
        with pytest.raises(VvliError, match="kind"):
            call(c)


@pytest.mark.parametrize("bad,name", [
    (dict(q=None), NULL), (dict(k=None), NULL), (dict(v=None), NULL), (dict(q_out=None), NULL), (dict(inv_freq=None), NULL),
    (dict(pos=None), NULL), (dict(slots=None), NULL), (dict(heads=0), CONFIG), (dict(heads=65536), CONFIG),
    (dict(ldq=252), CONFIG), (dict(ldq=258), CONFIG), (dict(ldk=124), CONFIG), (dict(ldv=130), CONFIG), (dict(ldo=255), CONFIG),
    (dict(q=P + 4), CONFIG), (dict(k=P + 8), CONFIG), (dict(rows=1 << 31), CONFIG), (dict(ldq=260), CONFIG),
    (dict(q_norm=P, eps=-1.0), CONFIG), (dict(k_norm=P, eps=float("nan")), CONFIG), (dict(weight_kind=2), CONFIG),
])
def test_norm_rope_append_refusals(bad, name):
    with pytest.raises(VvliError) as e:
        norm(**bad)
    assert e.value.name == name


def test_norm_rope_append_rows_that_no_launch_takes_are_refused():
    """2^26 rows are 2^32 threads, which no launch has: refused before it, with what other sizes give."""
    for rows in (1 << 26, (1 << 26) + 1, (1 << 31) - 1):
        with pytest.raises(VvliError) as e:
            norm(rows=rows)
        assert e.value.name == CONFIG


@pytest.mark.parametrize("bad,name", [
    (dict(table=None), NULL), (dict(row_start=None), NULL), (dict(start_pos=None), NULL), (dict(q=None), NULL),
    (dict(out=None), NULL), (dict(workspace=None), NULL), (dict(heads=0), CONFIG), (dict(heads=5), CONFIG),
    (dict(heads=65536), CONFIG), (dict(requests=0), CONFIG), (dict(table_stride=0), CONFIG), (dict(table_stride=1 << 27), CONFIG),
    (dict(table_stride=1 << 20, requests=1 << 11), CONFIG), (dict(ldq=252), CONFIG), (dict(ldo=258), CONFIG), (dict(q=P + 4), CONFIG),
    (dict(rows=1 << 31), CONFIG), (dict(scale=float("inf")), CONFIG), (dict(scale=float("nan")), CONFIG),
    (dict(workspace_bytes=0), CONFIG), (dict(workspace=P + 4), CONFIG), (dict(q=P, out=P, ldq=256, ldo=256), CONFIG),
])
def test_paged_attention_refusals(bad, name):
    kw = dict(out=P << 8)
    kw.update(bad)
    with pytest.raises(VvliError) as e:
        attend(**kw)
    assert e.value.name == name


@pytest.mark.parametrize("bad,name", [
    (dict(held=None), NULL), (dict(keep=None), NULL), (dict(add=None), NULL), (dict(length=None), NULL), (dict(row_start=None), NULL),
    (dict(start_pos=None), NULL), (dict(row_pos=None), NULL), (dict(slots=None), NULL), (dict(rows=1 << 31), CONFIG),
    (dict(pool=dict(free_pages=None)), NULL), (dict(pool=dict(free_count=None)), NULL), (dict(pool=dict(table=None)), NULL),
    (dict(pool=dict(requests=0)), CONFIG), (dict(pool=dict(table_stride=0)), CONFIG), (dict(pool=dict(page_size=0)), CONFIG),
    (dict(pool=dict(pages=0)), CONFIG), (dict(pool=dict(requests=1 << 16, table_stride=1 << 15)), CONFIG),
    (dict(pool=dict(page_size=1 << 16, table_stride=1 << 15)), CONFIG), (dict(pool=dict(page_size=1 << 16, pages=1 << 15)), CONFIG),
])
def test_paged_assign_refusals(bad, name):
    with pytest.raises(VvliError) as e:
        assign(**bad)
    assert e.value.name == name


@pytest.mark.parametrize("bad,name", [
    (dict(target=None), NULL), (dict(tokens=None), NULL), (dict(row_start=None), NULL), (dict(u_accept=None), NULL),
    (dict(u_sample=None), NULL), (dict(accepted=None), NULL), (dict(out=None), NULL), (dict(workspace=None), NULL),
    (dict(requests=0), CONFIG), (dict(vocab=0), CONFIG), (dict(ldt=99), CONFIG), (dict(ldd=99), CONFIG), (dict(rows=1 << 31), CONFIG),
    (dict(workspace_bytes=0), CONFIG), (dict(workspace=P + 8), CONFIG), (dict(out=P), CONFIG),
])
def test_verify_drafts_refusals(bad, name):
    with pytest.raises(VvliError) as e:
        verify(**bad)
    assert e.value.name == name


@pytest.mark.parametrize("rows", [0, 1, 5])
@pytest.mark.parametrize("gap", [-5, -4, -1, 0, 1, 4, 5])
def test_verify_drafts_output_over_its_tokens_is_refused(rows, gap):
    """`rows` tokens and outputs `gap` values apart: refused where they share one (or start together)."""
    tokens = P << 4
    good = dict(tokens=tokens, out=tokens + 4 * gap, rows=rows, requests=1)
    if gap == 0 or abs(gap) < rows:
        with pytest.raises(VvliError, match="overlaps"):
            verify(**good)
    else:  # not for this: the workspace is looked at next
        with pytest.raises(VvliError, match="workspace"):
            verify(**good, workspace_bytes=0)


def test_workspace_sizes():
    assert R.paged_attention_workspace(1, 1, 32, 8, 64) > 0
    assert R.paged_attention_workspace(1, 1, 32, 7, 64) == 0   # kv_heads does not divide heads
    assert R.paged_attention_workspace(1, 1, 32, 8, 80) == 0
    assert R.paged_attention_workspace(1, 0, 32, 8, 64) == 0
    # A workspace for the largest sizes serves smaller ones.
    big = R.paged_attention_workspace(4096, 64, 32, 8, 128)
    for rows, requests in ((1, 1), (64, 64), (4096, 1), (300, 7)):
        assert R.paged_attention_workspace(rows, requests, 32, 8, 128) <= big
    assert R.verify_drafts_workspace(1, 1000) <= R.verify_drafts_workspace(64, 128256)


# ---------------------------------------------------------------------------
# paged_index.hpp through a small library of its own
# ---------------------------------------------------------------------------
SOURCE = r"""
#include "paged_index.hpp"
using namespace vvli;
extern "C" {
uint32_t t_page_of(uint32_t d, uint32_t n) { return page_of(page_div(d), n); }
uint32_t t_pages_for(uint32_t d, uint32_t n) { return pages_for(page_div(d), n); }
int32_t t_slot(const int32_t* row, uint32_t stride, uint32_t pages, uint32_t d, uint32_t pos) {
    return page_slot(row, stride, pages, page_div(d), pos);
}
void t_rows(int32_t b, int32_t e, uint32_t rows, uint32_t* out) {
    RowSpan s = row_span(b, e, rows);
    out[0] = s.first, out[1] = s.count;
}
void t_keys(int64_t pos, uint32_t window, uint32_t room, uint32_t* out) {
    KeySpan s = key_span(pos, window, room);
    out[0] = s.lo, out[1] = s.hi;
}
}
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    if not cxx:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("paged_index")
    (d / "t.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-O1", "-std=c++17", "-shared", "-fPIC", "-I", str(ROOT / "vvli_amd" / "csrc"), "-o", str(d / "t.so"),
                    str(d / "t.cpp")], check=True)
    lib = ctypes.CDLL(str(d / "t.so"))
    lib.t_page_of.restype = lib.t_pages_for.restype = ctypes.c_uint32
    lib.t_keys.argtypes = [ctypes.c_int64, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_void_p]
    return lib


def test_division_by_the_page_size(index):
    rng = np.random.RandomState(0)
    for d in [1, 2, 3, 5, 7, 8, 15, 16, 17, 24, 48, 100, 255, 256, 257, 1000, 65535, 65536, (1 << 30) + 1, (1 << 31) - 1]:
        near = [k * d + o for k in (1, 2, 3, (2**31 - 1) // d) for o in (-1, 0, 1)]
        for n in [0, 1, 2**31 - 1, 2**31 - 2] + near + rng.randint(0, 2**31 - 1, 200).tolist():
            if 0 <= n < 2**31:
                assert index.t_page_of(d, n) == n // d, (d, n)
                assert index.t_pages_for(d, n) == -(-n // d), (d, n)


def test_slots_of_bad_pages(index):
    row = np.array([3, -1, 8, 7, 2**31 - 1, -2**31, 0], np.int32)
    at = lambda pos, ps=16, pages=8: index.t_slot(ctypes.c_void_p(row.ctypes.data), row.size, pages, ps, pos)  # noqa: E731
    assert at(0) == 48 and at(15) == 63 and at(16) == -1 and at(32) == -1 and at(48) == 7 * 16 and at(63) == 7 * 16 + 15
    assert at(64) == -1 and at(80) == -1 and at(96) == 0 and at(111) == 15
    for pos in (112, 113, 1000, 2**31 - 1):  # behind the row's end
        assert at(pos) == -1
    assert at(7, ps=7) == -1 and at(21, ps=7) == 7 * 7


def test_row_spans_stay_in_the_batch(index):
    out = (ctypes.c_uint32 * 2)()
    for b in (-2**31, -1, 0, 3, 10, 11, 2**31 - 1):
        for e in (-2**31, -1, 0, 3, 10, 11, 2**31 - 1):
            index.t_rows(b, e, 10, out)
            assert out[0] + out[1] <= 10
            want = range(min(max(b, 0), 10), min(max(e, 0), 10))
            assert out[1] == len(want) and (not want or out[0] == want[0])


def test_key_spans(index):
    out = (ctypes.c_uint32 * 2)()
    for pos in (-5, -1, 0, 1, 15, 16, 99, 100, 101, 2**31, 2**32):
        for window in (0, 1, 2, 16, 100, 2**32 - 1):
            for room in (1, 16, 100, 2**31 - 1):
                index.t_keys(pos, window, room, out)
                lo = max(0, pos + 1 - window) if window else 0
                hi = min(pos + 1, room)
                want = (lo, hi) if pos >= 0 and lo < hi else (0, 0)
                assert tuple(out) == want, (pos, window, room)
