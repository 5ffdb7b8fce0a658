"""Ops around 8-bit products on the GPU, against plain implementations in 64
bits.

Tolerances: codes and scales are those of exact arithmetic wherever 64 bits tell
a value from a border. Here and there a value passes fewer than 40 roundings of
2^-53 on the way and a sum of n squares n more, half of which reach the root:
with n <= 70000 under 2^-36 relative, so that

* a code is an integer next to value / scale: |value / scale - code| is at most
  0.5 + 127 * 2^-35;
* a scale is max |value| / 127 rounded to f32: within 2^-24 + 2^-35 of it;
* the norm's f32 rows are within 2^-24 + 2^-35 of the value (or half a step of
  the denormals, 2^-150);
* rows quantised as they are pass one division: codes and scales are equal;
* the residual's sum is one f32 addition, the product a whole number followed by
  f32 operations in a given order: equal in every bit.
"""
import numpy as np
import pytest
from test_ops_i8 import CUT, FAR, FAR_STRIDE, HUGE, LONG, ODD, SPLIT

from vvli_amd import runtime as R

pytestmark = pytest.mark.gpu

EPS = float(np.float32(1e-6))
SLACK = 2.0 ** -35
HALF = 2.0 ** -24


@pytest.fixture(scope="module")
def torch():
    import torch as t

    return t


def ptr(t):
    return None if t is None else t.data_ptr()


def up(n, to):
    return -(-n // to) * to


def stream(torch):
    return torch.cuda.current_stream().cuda_stream


def gen(torch, seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Codes:
    """Codes and scales on the device with marks around them."""

    def __init__(self, torch, rows, width, pad=0):
        self.rows, self.width, self.ldc = rows, width, up(width, 16) + 16 * pad
        self.codes = torch.full((rows + 2, self.ldc), 99, dtype=torch.int8, device="cuda")
        self.scales = torch.full((rows + 2,), -5.0, device="cuda")
        self.args = (self.codes.data_ptr(), self.ldc, self.scales.data_ptr())

    def get(self):
        """(codes [rows, width], scales) in f64, with what is around them looked at."""
        c, s, n, w = self.codes.cpu().numpy(), self.scales.cpu().numpy(), self.rows, self.width
        assert (c[n:] == 99).all() and (s[n:] == -5).all(), "rows behind the last were written"
        assert (c[:n, w:up(w, 16)] == 0).all(), "the codes' tail is not 0"
        assert (c[:n, up(w, 16):] == 99).all(), "codes behind the padded width were written"
        return c[:n, :w].astype(np.float64), s[:n].astype(np.float64)


def check_codes(codes, scales, v):
    """codes and scales of rows v (f64)."""
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        top = np.abs(v).max(-1)
        whole = np.isfinite(v).all(-1)
        want = (top / 127).astype(np.float32).astype(np.float64)
        fine = whole & np.isfinite(want)
        assert np.isnan(scales[~fine]).all() and (codes[~fine] == 0).all()
        near = np.maximum(np.abs(want) * (2 * HALF + SLACK), 2.0 ** -149)  # (a neighbour where top / 127 is next to a border)
        assert (np.abs(scales - want)[fine] <= near[fine]).all()
        assert ((scales == want) | ~fine).mean() > 0.99 or len(want) < 100
        none = fine & (scales == 0)
        assert (codes[none] == 0).all() and (np.abs(codes) <= 127).all()
        some = fine & (scales > 0)
        t = v[some] / scales[some][:, None]
        assert (np.abs(np.clip(t, -127, 127) - codes[some]) <= 0.5 + 127 * SLACK).all()


def equal_codes(codes, scales, v):
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        want = (np.abs(v).max(-1) / 127).astype(np.float32).astype(np.float64)
        want[~np.isfinite(want)] = np.nan
        assert np.array_equal(scales, want, equal_nan=True)
        t = np.where((want > 0)[:, None], np.rint(v / want[:, None]), 0)
        assert np.array_equal(codes, np.clip(t, -127, 127))


WIDTHS = [1, 2, 3, 15, 16, 17, 63, 64, 255, 896, 1024, 1025, 2047, 3584, 4096, 4099, 8192, 16384, 16390, 18944, 65536, 65541, 70001]


def rows_for(width):
    return 9 if width < 5000 else 4


# ---------------------------------------------------------------------------
# quantize_rows
# ---------------------------------------------------------------------------
def odd_rows(torch, x):
    """Rows that are no ordinary ones, in place (f32)."""
    n = len(x)
    if n >= 4:
        x[1] = 0
        x[2] *= 1e-39      # denormal values and scale
        x[3] *= 1e30
    if n >= 9:
        x[4, -1] = float("inf")
        x[5, 0] = float("nan")
        x[6] = 1e-45       # a scale below f32's range
        x[7, : x.shape[1] // 2] = 0
        x[7, -1] = -127.0  # a scale of 1 and ties
        x[7, 0] = 0.5 if x.shape[1] > 1 else -127.0
        x[7, 1:2] = 1.5 if x.shape[1] > 2 else -127.0
        x[7, 2:3] = -2.5 if x.shape[1] > 3 else -127.0
    return x


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("width", WIDTHS)
def test_quantize_rows(torch, width, kind):
    rows, unit = rows_for(width), 4 if kind == "f32" else 8
    for pad in (0, 3):
        ld = up(width, unit) + unit * pad
        x = torch.full((rows, ld), float("nan"), device="cuda")  # (behind the width: not read)
        x[:, :width] = odd_rows(torch, torch.randn(rows, width, device="cuda", generator=gen(torch, width)))
        x = x if kind == "f32" else x.bfloat16()
        out = Codes(torch, rows, width, pad)
        R.quantize_rows(ptr(x), kind, ld, rows, width, *out.args, stream(torch))
        equal_codes(*out.get(), x[:, :width].double().cpu().numpy())


def test_quantize_rows_borders(torch):
    """Values on and next to the borders between codes, for scales of many last bits."""
    rng = np.random.RandomState(0)
    s = (1 + rng.rand(600)).astype(np.float32)
    top = (s.astype(np.float64) * 127).astype(np.float32)
    scale = (top.astype(np.float64) / 127).astype(np.float32)
    n = rng.randint(0, 127, (600, 400)) + 0.5
    x = (n * scale.astype(np.float64)[:, None]).astype(np.float32)
    x = np.where(rng.rand(*x.shape) < 0.5, x, np.nextafter(x, np.float32(rng.choice([0, 1e9])), dtype=np.float32))
    x[:, 0] = top
    x *= rng.choice([-1, 1], x.shape).astype(np.float32)
    d = torch.from_numpy(x).cuda()
    out = Codes(torch, 600, 400)
    R.quantize_rows(ptr(d), "f32", 400, 600, 400, *out.args, stream(torch))
    equal_codes(*out.get(), x.astype(np.float64))


@pytest.mark.parametrize("width", [7, 401, 896, 3584, 18950])
def test_quantize_rows_ties(torch, width):
    """Rows of bf16 whose quotients fall on borders by the hundred (127 / 254 of 8-bit values is one half)."""
    rng = np.random.RandomState(width)
    m = rng.randint(-255, 256, (40, width)).astype(np.float64)
    top = np.array([254, 254, 255, 128, 192, 160, 224, 250] * 5, np.float64)
    m = np.clip(m * np.exp2(-rng.randint(0, 4, m.shape)), -top[:, None], top[:, None])
    m[:, width // 2] = top
    x = torch.from_numpy((m * np.exp2(rng.randint(-20, 20, (40, 1)))).astype(np.float32)).cuda().bfloat16()
    ld = up(width, 8)
    d = torch.full((40, ld), float("nan"), dtype=torch.bfloat16, device="cuda")
    d[:, :width] = x
    out = Codes(torch, 40, width)
    R.quantize_rows(ptr(d), "bf16", ld, 40, width, *out.args, stream(torch))
    equal_codes(*out.get(), x.double().cpu().numpy())


def test_quantize_rows_many(torch):
    """More rows than one launch of a block each might take at once."""
    x = torch.randn(70001, 16, device="cuda", generator=gen(torch, 1))
    out = Codes(torch, 70001, 16)
    R.quantize_rows(ptr(x), "f32", 16, 70001, 16, *out.args, stream(torch))
    equal_codes(*out.get(), x.double().cpu().numpy())


@pytest.mark.parametrize("rows,width", [((1 << 22) + 5, 4), ((1 << 20) + 3, 1028)])
def test_quantize_rows_more_than_a_launch_has_blocks(torch, rows, width):
    """Blocks that take a row after the other (four of them at a time up to 1024 values)."""
    x = torch.zeros(rows, width + width % 8, dtype=torch.bfloat16, device="cuda")
    x.uniform_(-1, 1, generator=gen(torch, 3))
    codes, scales = torch.full((rows + 1, up(width, 16)), 99, dtype=torch.int8, device="cuda"), torch.full((rows + 1,), -5.0, device="cuda")
    R.quantize_rows(ptr(x), "bf16", x.shape[1], rows, width, ptr(codes), codes.shape[1], ptr(scales), stream(torch))
    want = (x[:, :width].abs().amax(-1).double() / 127).float()
    assert torch.equal(scales[:rows], want) and scales[rows] == -5 and (codes[rows] == 99).all()
    assert (codes[:rows, width:] == 0).all()
    for part in (slice(0, 400), slice(rows - 400, rows)):
        equal_codes(codes[part, :width].cpu().numpy().astype(np.float64), scales[part].cpu().numpy().astype(np.float64),
                    x[part, :width].double().cpu().numpy())


def test_quantize_rows_offsets_past_32_bits(torch):
    """Strides that put the last rows' elements and codes behind 2^32 bytes."""
    ld, rows = 1 << 28, 6
    x = torch.zeros(rows, ld, dtype=torch.bfloat16, device="cuda")
    codes, scales = torch.zeros(rows, (1 << 30), dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    v = torch.randn(rows, 100, device="cuda", generator=gen(torch, 2)).bfloat16()
    x[:, :100] = v
    R.quantize_rows(ptr(x), "bf16", ld, rows, 100, ptr(codes), 1 << 30, ptr(scales), stream(torch))
    equal_codes(codes[:, :100].cpu().numpy().astype(np.float64), scales.cpu().numpy().astype(np.float64), v.double().cpu().numpy())


# ---------------------------------------------------------------------------
# add_norm
# ---------------------------------------------------------------------------
def norm_value(h, w, eps=EPS):
    h = h.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        return h * w / np.sqrt((h * h).mean(-1, keepdims=True) + eps)


def check_y(y, v):
    with np.errstate(invalid="ignore", over="ignore"):
        bad = ~np.isfinite(v.astype(np.float32))
        assert np.array_equal(np.isnan(y), np.isnan(v))
        fine = ~bad & np.isfinite(y)
        assert (fine | bad).all()
        assert (np.abs(y - v)[fine] <= np.maximum(np.abs(v[fine]) * (HALF + SLACK), 2.0 ** -150)).all()


@pytest.mark.parametrize("kind,delta,total,y,codes", [
    ("bf16", True, True, False, True), ("f32", True, True, True, True), ("bf16", False, False, True, False),
    ("f32", True, False, False, True), ("bf16", False, False, True, True), ("bf16", True, True, True, False)])
@pytest.mark.parametrize("width", WIDTHS)
def test_add_norm(torch, width, kind, delta, total, y, codes):
    rows, pad = rows_for(width), (width % 3)
    ld = up(width, 4) + 4 * pad
    g = gen(torch, width)
    x = torch.full((rows, ld), float("nan"), device="cuda")
    x[:, :width] = torch.randn(rows, width, device="cuda", generator=g)
    if rows >= 9:
        odd_rows(torch, x[:, :width])
    d = torch.randn(rows, ld, device="cuda", generator=g) if delta else None
    if delta and rows >= 4:
        d[1] = 0
        d[2] *= 1e-39
    w = (1 + 0.3 * torch.randn(width, device="cuda", generator=g)).to(torch.bfloat16 if kind == "bf16" else torch.float32)
    s = torch.full((rows + 1, ld), 77.0, device="cuda") if total else None
    o = torch.full((rows + 1, ld), 77.0, device="cuda") if y else None
    out = Codes(torch, rows, width, pad)
    R.add_norm(ptr(x), ld, ptr(d), ld, rows, width, ptr(w), kind, EPS, ptr(s), ld, ptr(o), ld, *(out.args if codes else (None, 0, None)),
               stream(torch))
    h = (x + d if delta else x)[:, :width]
    if total:
        assert np.array_equal(s[:rows, :width].cpu().numpy(), h.cpu().numpy(), equal_nan=True)
        assert (s[rows] == 77).all() and (s[:, width:] == 77).all()
    v = norm_value(h.cpu().numpy(), w.double().cpu().numpy())
    if y:
        check_y(o[:rows, :width].double().cpu().numpy(), v)
        assert (o[rows] == 77).all() and (o[:, width:] == 77).all()
    if codes:
        check_codes(*out.get(), v)


@pytest.mark.parametrize("place", ["sum is x", "sum is delta", "y is x", "y is delta, sum is x", "y is x, no sum", "y is delta, no sum"])
@pytest.mark.parametrize("width", [100, 3584, 18944, 70001])
def test_add_norm_in_place(torch, width, place):
    rows, ld = 5, up(width, 4)
    g = gen(torch, 5)
    x, d = (torch.randn(rows, ld, device="cuda", generator=g) for _ in range(2))
    w = torch.randn(width, device="cuda", generator=g)
    h = (x + d)[:, :width].cpu().numpy()
    other = torch.zeros(rows, ld, device="cuda")
    total, y = {"sum is x": (x, None), "sum is delta": (d, None), "y is x": (other, x), "y is delta, sum is x": (x, d),
                "y is x, no sum": (None, x), "y is delta, no sum": (None, d)}[place]
    out = Codes(torch, rows, width)
    R.add_norm(ptr(x), ld, ptr(d), ld, rows, width, ptr(w), "f32", EPS, ptr(total), ld, ptr(y), ld, *out.args, stream(torch))
    v = norm_value(h, w.double().cpu().numpy())
    check_codes(*out.get(), v)
    if total is not None:
        assert np.array_equal(total[:, :width].cpu().numpy(), h)
    if y is not None:
        check_y(y[:, :width].double().cpu().numpy(), v)


def test_add_norm_far_values(torch):
    """Squares that leave f32, weights that do with the values, eps 0, weights of 0 and NaN."""
    rows, width = 8, 1000
    g = gen(torch, 6)
    x = torch.randn(rows, width, device="cuda", generator=g) * torch.tensor([1e30, 1e-30, 1e38, 1e-38, 1, 1e20, 1e-20, 0.0], device="cuda")[:, None]
    for w in (torch.randn(width, device="cuda", generator=g) * 1e25, torch.randn(width, device="cuda", generator=g) * 1e-30,
              torch.zeros(width, device="cuda"), torch.full((width,), float("nan"), device="cuda")):
        for eps in (EPS, 0.0):
            y, out = torch.zeros_like(x), Codes(torch, rows, width)
            R.add_norm(ptr(x), width, None, 0, rows, width, ptr(w), "f32", eps, None, 0, ptr(y), width, *out.args, stream(torch))
            v = norm_value(x.cpu().numpy(), w.double().cpu().numpy(), eps)
            check_y(y.double().cpu().numpy(), v)
            check_codes(*out.get(), v)


# ---------------------------------------------------------------------------
# silu_mul
# ---------------------------------------------------------------------------
def gate_value(g, u):
    g = g.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        return g / (1 + np.exp(-g)) * u


@pytest.mark.parametrize("width", WIDTHS)
def test_silu_mul(torch, width):
    rows = rows_for(width)
    for pad in (0, 5):
        ld = up(width, 4) + 4 * pad
        g = gen(torch, width + 1)
        a = torch.full((rows, 2 * ld), float("nan"), device="cuda")
        a[:, :width] = 3 * torch.randn(rows, width, device="cuda", generator=g)
        a[:, ld:ld + width] = odd_rows(torch, torch.randn(rows, width, device="cuda", generator=g))
        if rows >= 9:
            a[0, :width] *= 60  # gates of -150 and less
            a[8, : width // 2] = -300
        out = Codes(torch, rows, width, pad)
        R.silu_mul(ptr(a), 2 * ld, ptr(a) + 4 * ld, 2 * ld, rows, width, *out.args, stream(torch))
        check_codes(*out.get(), gate_value(a[:, :width].cpu().numpy(), a[:, ld:ld + width].double().cpu().numpy()))


def test_silu_mul_longer_than_the_caches(torch):
    """More than 128 MiB of gate and up, of an odd width."""
    rows, width, ld = 900, 18950, 2 * 18952
    g = gen(torch, 12)
    a = torch.randn(rows, ld, device="cuda", generator=g)
    a[5], a[6, :18952], a[7, 3] = 0, -60, float("inf")
    out = Codes(torch, rows, width)
    R.silu_mul(ptr(a), ld, ptr(a) + 4 * 18952, ld, rows, width, *out.args, stream(torch))
    check_codes(*out.get(), gate_value(a[:, :width].cpu().numpy(), a[:, 18952:18952 + width].double().cpu().numpy()))


@pytest.mark.parametrize("low,high,size", [(-120, -60, 1e30), (-104, -80, 1.0), (-95, -85, 3e38), (-700, -80, 1.0), (60, 120, 1e-38),
                                           (-1e-30, 1e-30, 1e-10), (-20, 20, 1e38), (-800, -740, 1e38), (-90, 90, 1e13)])
def test_silu_mul_far_values(torch, low, high, size):
    """Gates whose exponential leaves f32, products that do: a row's codes follow the values all the same."""
    rows, width = 6, 2000
    g = gen(torch, 7)
    gate = torch.empty(rows, width, device="cuda").uniform_(low, high, generator=g)
    u = torch.randn(rows, width, device="cuda", generator=g).clamp_(-1, 1) * size
    out = Codes(torch, rows, width)
    R.silu_mul(ptr(gate), width, ptr(u), width, rows, width, *out.args, stream(torch))
    check_codes(*out.get(), gate_value(gate.cpu().numpy(), u.double().cpu().numpy()))


@pytest.mark.parametrize("width", [5, 16, 2050, 18944, 40000])
def test_silu_mul_rows_without_values(torch, width):
    """Rows of zeros, of products that are 0 where f32's are none, and below what a scale holds."""
    ld = up(width, 4)
    gate, u = torch.ones(6, ld, device="cuda"), torch.ones(6, ld, device="cuda")
    gate[0] = 0
    u[1] = 0
    gate[2], u[2] = -1e4, 3e38
    gate[3], u[3] = -1e4, -3e38
    gate[3, 0], u[3, 0] = 1, 1e-30
    gate[4], u[4] = -80, 1e-20
    out = Codes(torch, 6, width)
    R.silu_mul(ptr(gate), ld, ptr(u), ld, 6, width, *out.args, stream(torch))
    codes, scales = out.get()
    check_codes(codes, scales, gate_value(gate[:, :width].cpu().numpy(), u[:, :width].double().cpu().numpy()))
    assert (scales[:3] == 0).all() and (codes[:3] == 0).all() and scales[4] == 0 and scales[5] > 0


def test_add_norm_weights_not_finite(torch):
    """A weight of infinity makes a row of zeros NaN, and any other."""
    x, w = torch.zeros(4, 700, device="cuda"), torch.ones(700, device="cuda")
    x[1:] = torch.randn(3, 700, device="cuda", generator=gen(torch, 8))
    for bad in (float("inf"), float("-inf")):
        w[333] = bad
        y, out = torch.zeros_like(x), Codes(torch, 4, 700)
        R.add_norm(ptr(x), 700, None, 0, 4, 700, ptr(w), "f32", EPS, None, 0, ptr(y), 700, *out.args, stream(torch))
        v = norm_value(x.cpu().numpy(), w.double().cpu().numpy())
        codes, scales = out.get()
        check_codes(codes, scales, v)
        assert np.isnan(scales).all() and np.isnan(y[0, 333].item()) and np.isinf(y[1:, 333].cpu().numpy()).all()


@pytest.mark.parametrize("g,u", [(float("-inf"), 1.0), (float("inf"), 1.0), (float("nan"), 1.0), (1.0, float("inf")), (-200.0, float("inf")),
                                 (3e38, 3e38), (-1e4, float("nan"))])
def test_silu_mul_not_finite(torch, g, u):
    gate, up_ = torch.ones(3, 512, device="cuda"), torch.ones(3, 512, device="cuda")
    gate[1, 300], up_[1, 300] = g, u
    out = Codes(torch, 3, 512)
    R.silu_mul(ptr(gate), 512, ptr(up_), 512, 3, 512, *out.args, stream(torch))
    check_codes(*out.get(), gate_value(gate.cpu().numpy(), up_.double().cpu().numpy()))


# Bits of NaN other than those that arithmetic makes: low bits set, a sign, signaling ones.
NANS = [0x7FC000A5, 0xFFC0FFFF, 0x7F8000A5, 0x7FFFFFFF]


def nan_of(torch, bits):
    return torch.tensor([bits - (1 << 32) if bits >> 31 else bits], dtype=torch.int32, device="cuda").view(torch.float32)


@pytest.mark.parametrize("bits", NANS, ids=hex)
@pytest.mark.parametrize("width", [1, 5, 17, 1025, 2047, 4099, 18945, 40001])
def test_nans_of_any_bits(torch, width, bits):
    """A row with a NaN has scale NaN and codes 0, zeros behind its width among them, whatever the NaN's bits."""
    rows, ld, nan = 4, up(width, 8), nan_of(torch, bits)
    g = gen(torch, width + 2)
    x, d = (torch.randn(rows, ld, device="cuda", generator=g) for _ in range(2))
    bad = x.clone()
    bad.view(torch.int32)[1, width // 2] = nan.view(torch.int32)
    bad.view(torch.int32)[2, width - 1] = nan.view(torch.int32)
    half = bad.bfloat16()
    half.view(torch.int16)[1:3, width // 2] = nan.view(torch.int32).item() >> 16 | 1  # (a signaling one's low bits are cut off)
    w = torch.randn(ld, device="cuda", generator=g)
    w_nan, w_half = w.clone(), w.bfloat16()
    w_nan.view(torch.int32)[width // 2] = nan.view(torch.int32)
    w_half.view(torch.int16)[width // 2] = nan.view(torch.int32).item() >> 16 | 1

    def looked_at(call, want):
        out = Codes(torch, rows, width, 1)
        call(out)
        codes, scales = out.get()
        assert np.array_equal(np.isnan(scales), want), scales
        assert (codes[want] == 0).all()

    some, every = np.array([False, True, True, False]), np.ones(rows, bool)
    s = stream(torch)
    looked_at(lambda o: R.quantize_rows(ptr(bad), "f32", ld, rows, width, *o.args, s), some)
    looked_at(lambda o: R.quantize_rows(ptr(half), "bf16", ld, rows, width, *o.args, s), some)
    looked_at(lambda o: R.silu_mul(ptr(bad), ld, ptr(x), ld, rows, width, *o.args, s), some)
    looked_at(lambda o: R.silu_mul(ptr(x), ld, ptr(bad), ld, rows, width, *o.args, s), some)
    total, y = torch.zeros(rows, ld, device="cuda"), torch.zeros(rows, ld, device="cuda")
    for a, b in ((bad, None), (bad, d), (x, bad), (bad, bad)):
        looked_at(lambda o: R.add_norm(ptr(a), ld, ptr(b), ld, rows, width, ptr(w), "f32", EPS, ptr(total) if b is not None else None, ld,
                                       ptr(y), ld, *o.args, s), some)
        assert torch.isnan(y[1:3, :width]).all() and torch.isfinite(y[[0, 3]]).all()
    for kind, t in (("f32", w_nan), ("bf16", w_half)):
        looked_at(lambda o: R.add_norm(ptr(x), ld, None, 0, rows, width, ptr(t), kind, EPS, None, 0, None, 0, *o.args, s), every)


# ---------------------------------------------------------------------------
# linear_i8
# ---------------------------------------------------------------------------
class Product:
    def __init__(self, torch, M, N, K, bias=False, padw=0, padx=0, pady=0, seed=0, least=False, space=None):
        g = gen(torch, seed * 1000 + M + N + K)
        self.torch, self.sizes, self.strides = torch, (M, N, K), (K + 16 * padw, K + 16 * padx, N + pady)
        r = lambda n, ld: torch.randint(-128 if least else -127, 128, (n, ld), dtype=torch.int8, device="cuda", generator=g)  # noqa: E731
        self.W, self.X = r(N, self.strides[0]), r(M, self.strides[1])
        if least:
            self.W[:, ::2], self.X[:, ::2] = -128, -128
        self.ws = torch.empty(N, device="cuda").uniform_(1e-4, 2e-3, generator=g)
        self.xs = torch.empty(M, device="cuda").uniform_(1e-3, 1e-1, generator=g)
        self.bias = torch.randn(N, device="cuda", generator=g).bfloat16() if bias else None
        self.Y = torch.full((M + 1, self.strides[2]), 55.0, device="cuda")
        self.space = torch.zeros(R.linear_i8_workspace(M, N, K), dtype=torch.uint8, device="cuda") if space is None else space

    def run(self, stream_=None):
        R.linear_i8(ptr(self.W), self.strides[0], ptr(self.ws), ptr(self.X), self.strides[1], ptr(self.xs), ptr(self.bias), ptr(self.Y),
                    self.strides[2], *self.sizes, ptr(self.space), self.space.numel(), stream_ or stream(self.torch))

    def want(self):
        M, N, K = self.sizes
        y = self.torch.empty(M, N, device="cuda")
        w = self.W[:, :K].double().t().contiguous()
        for m in range(0, M, 256):
            y[m:m + 256] = (self.X[m:m + 256, :K].double() @ w).float()
        y = (y * self.xs[:, None]) * self.ws
        return y if self.bias is None else y + self.bias.float()

    def check(self):
        M, N, K = self.sizes
        want, got = self.want().cpu().numpy(), self.Y.cpu().numpy()
        bad = np.argwhere(~((got[:M, :N] == want) | (np.isnan(want) & np.isnan(got[:M, :N]))))
        assert not len(bad), f"{len(bad)} of {M * N} differ, first at {bad[0]}: {got[tuple(bad[0])]} for {want[tuple(bad[0])]}"
        assert (got[M:] == 55).all() and (got[:, N:] == 55).all(), "written behind the output"
        self.Y.fill_(55.0)


ROWS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 200, 255, 257, 333, 600]


@pytest.mark.parametrize("N,K", [(1, 16), (3, 32), (15, 48), (16, 64), (17, 80), (33, 112), (64, 128), (65, 144), (130, 256), (256, 272),
                                 (300, 1008), (896, 896), (1152, 4864), (2048, 2048)])
def test_linear_i8(torch, N, K):
    for i, M in enumerate(ROWS):
        p = Product(torch, M, N, K, bias=i % 2 == 0, padw=i % 3, padx=i % 4, pady=i % 5)
        p.run()
        p.check()


@pytest.mark.parametrize("M,N,K", [(1, 37888, 3584), (4, 4608, 3584), (2, 3584, 18944), (8, 2048, 8192), (48, 4608, 3584), (64, 3584, 18944),
                                   (128, 16384, 2048), (200, 6144, 2048), (1, 16, 131056), (9, 40, 131056), (300, 64, 131056),
                                   (1000, 1152, 896), (2049, 4608, 3584), (4096, 9728, 896), (777, 3584, 3600), (5000, 257, 528),
                                   (70000, 16, 16), (1, 70001, 32)])
def test_linear_i8_large(torch, M, N, K):
    p = Product(torch, M, N, K, bias=N % 3 == 0, seed=1)
    p.run()
    p.check()


@pytest.mark.parametrize("M,N,K", ODD + CUT)
def test_linear_i8_every_kernel(torch, M, N, K):
    for pad in ((0, 0, 0), (1, 3, 5)):
        p = Product(torch, M, N, K, True, *pad, seed=2)
        for _ in range(2):
            p.run()
            p.check()


@pytest.mark.parametrize("M,N,K", LONG)
def test_linear_i8_long_results(torch, M, N, K):
    p = Product(torch, M, N, K, True, pady=3, seed=6)
    want = p.want()
    for _ in range(2):
        p.run()
        assert torch.equal(p.Y[:M, :N], want) and (p.Y[M:] == 55).all() and (p.Y[:, N:] == 55).all()
        p.Y.fill_(55.0)


@pytest.mark.parametrize("M", [1, 5, 20, 70, 300])
def test_linear_i8_most_negative(torch, M):
    """Codes of -128, and sums next to the ends of 32 bits."""
    p = Product(torch, M, 40, 131056, least=True)
    p.run()
    p.check()
    p.W.fill_(-128), p.X.fill_(-128)
    p.run()
    p.check()
    p.X.fill_(127)
    p.run()
    p.check()


@pytest.mark.parametrize("M", [1, 6, 40, 130, 700])
def test_linear_i8_scales(torch, M):
    """Rows whose scale is 0 or NaN, codes of zeros."""
    p = Product(torch, M, 100, 640)
    p.xs[0] = float("nan")
    if M > 3:
        p.xs[1], p.X[1] = 0, 0
        p.xs[2] = float("inf")
    p.ws[3], p.ws[5] = 0, float("nan")
    p.run()
    p.check()


def test_linear_i8_one_workspace_for_all_sizes(torch):
    """A workspace made for the largest call serves all others, in any order."""
    sizes = [(300, 896, 4864), (1, 2048, 2048), (48, 1152, 8192), (5, 40, 131056), (64, 3584, 3584), (17, 16, 65536), (129, 300, 4096)]
    space = torch.zeros(max(R.linear_i8_workspace(*s) for s in sizes), dtype=torch.uint8, device="cuda")
    products = [Product(torch, *s, space=space, seed=i) for i, s in enumerate(sizes)]
    for _ in range(3):
        for p in products:
            p.run()
        torch.cuda.synchronize()
        for p in products:
            p.check()
        products = products[3:] + products[:3]


def test_linear_i8_two_streams(torch):
    streams = [torch.cuda.Stream() for _ in range(2)]
    products = [Product(torch, 48, 2048, 8192, seed=3), Product(torch, 20, 1152, 18944, seed=4)]
    torch.cuda.synchronize()
    for _ in range(20):
        for p, s in zip(products, streams):
            p.run(s.cuda_stream)
    torch.cuda.synchronize()
    for p in products:
        p.check()


def test_linear_i8_unaligned_output(torch):
    """Y at an address and with a stride that no vector store fits."""
    for M, N in ((1, 33), (5, 64), (70, 130), (300, 257), (600, 512)):
        p = Product(torch, M, N, 512, bias=True)
        want = p.want()
        flat = torch.full((M * (N + 1) + 9,), 55.0, device="cuda")
        R.linear_i8(ptr(p.W), 512, ptr(p.ws), ptr(p.X), 512, ptr(p.xs), ptr(p.bias), ptr(flat) + 4, N + 1, M, N, 512, ptr(p.space),
                    p.space.numel(), stream(torch))
        got = flat[1:1 + M * (N + 1)].view(M, N + 1)
        assert torch.equal(got[:, :N], want) and flat[0] == 55 and (got[:, N] == 55).all() and (flat[1 + M * (N + 1):] == 55).all()


@pytest.mark.parametrize("M", [33, 65, 129, 193, 257, 300, 513])
@pytest.mark.parametrize("N,K", [(40, 96), (333, 1536), (8200, 256)])
def test_linear_i8_rows_behind_the_last(torch, M, N, K):
    """A tile's rows that there are none of lie in memory that is not Y's."""
    p = Product(torch, M, N, K, True, pady=3)
    p.Y = torch.full((M + 300, N + 3), 55.0, device="cuda")
    p.run()
    p.check()


@pytest.mark.parametrize("M,N,K", [(1, 33, 64), (20, 50, 256), (70, 130, 144), (300, 270, 512), (311, 401, 6768)])
def test_linear_i8_scales_at_any_address(torch, M, N, K):
    p = Product(torch, M, N, K, True)
    for name, t in (("xs", p.xs), ("ws", p.ws), ("bias", p.bias)):
        setattr(p, name, torch.cat([t[:1], t])[1:])
        assert ptr(getattr(p, name)) % 16
    p.run()
    p.check()


@pytest.mark.parametrize("M", [1, 9, 50, 300])
@pytest.mark.parametrize("width", [1, 100, 897, 2030])
def test_products_of_odd_widths(torch, M, width):
    """Rows of a width that is no multiple of 16 multiply as the next one: the codes behind them are 0."""
    N, K = 70, up(width, 16)
    g = gen(torch, 9)
    rows = lambda n: torch.randn(n, up(width, 4), device="cuda", generator=g)  # noqa: E731
    x, w = rows(M), rows(N)
    c, s, cw, sw = (torch.full(size, 99, dtype=t, device="cuda")
                    for n in (M, N) for size, t in (((n, K), torch.int8), ((n,), torch.float32)))
    for a, b, d in ((x, c, s), (w, cw, sw)):
        R.quantize_rows(ptr(a), "f32", a.shape[1], len(a), width, ptr(b), K, ptr(d), stream(torch))
    y, space = torch.zeros(M, N, device="cuda"), torch.zeros(R.linear_i8_workspace(M, N, K), dtype=torch.uint8, device="cuda")
    R.linear_i8(ptr(cw), K, ptr(sw), ptr(c), K, ptr(s), None, ptr(y), N, M, N, K, ptr(space), space.numel(), stream(torch))
    want = ((c[:, :width].double() @ cw[:, :width].double().t().contiguous()).float() * s[:, None]) * sw
    assert torch.equal(y, want)
    # (each value is off by half a step of its row's scale at most, the products by what that makes of a sum)
    v, vw, h, hw = x[:, :width].double(), w[:, :width].double(), s.double()[:, None] / 2, sw.double()[:, None] / 2
    off = h * vw.abs().sum(-1)[None] + v.abs().sum(-1, keepdim=True) * hw.t() + width * h * hw.t()
    assert ((y.double() - v @ vw.t().contiguous()).abs() <= off * (1 + 1e-4) + 1e-30).all()


def test_linear_i8_captured(torch):
    """Products of every kind of kernel in one graph and one workspace, replayed with eager calls in between."""
    sizes = [(1, 300, 640), (20, 896, 896), (311, 401, 6768), (70, 130, 1040), (300, 1152, 896), (687, 875, 14512)]
    space = torch.zeros(max(R.linear_i8_workspace(*s) for s in sizes), dtype=torch.uint8, device="cuda")
    products = [Product(torch, *s, bias=True, space=space, seed=i) for i, s in enumerate(sizes)]
    other = Product(torch, 311, 401, 6768, seed=11)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for p in products:
            p.run()
    for i in range(4):
        for p in products:
            p.X.copy_(p.X.roll(i, 0))
            p.Y.fill_(55.0)
        space.fill_(i)
        graph.replay()
        other.run()
        torch.cuda.synchronize()
        for p in products + [other]:
            p.check()


def test_linear_i8_offsets_past_32_bits(torch):
    """W, X and Y of more than 2^32 bytes."""
    N, K, ld = 5000, 64, 1 << 20
    W = torch.zeros(N, ld, dtype=torch.int8, device="cuda")
    for M in (3, 40, 300):
        p = Product(torch, M, N, K)
        W[:, :K] = p.W
        p.W, p.strides = W, (ld, K, N)
        p.run()
        p.check()
    X = W
    for n in (20, 300):
        p = Product(torch, N, n, K, seed=2)
        X[:, :K] = p.X
        p.X, p.strides = X, (K, ld, n)
        p.run()
        p.check()
    del W, X, p
    p = Product(torch, 5000, 300, 128, pady=(1 << 18))
    p.run()
    assert torch.equal(p.Y[:5000, :300], p.want())
    assert (p.Y[:5000, 300:310] == 55).all() and (p.Y[5000] == 55).all()


# ---------------------------------------------------------------------------
# Together, as a program uses them
# ---------------------------------------------------------------------------
class Block:
    """One transformer block with 8-bit products over a paged cache, on `most` rows."""

    def __init__(self, torch, most, hidden=256, heads=4, kv=2, inter=672, seed=0):
        self.torch, self.most, self.hidden, self.heads, self.kv, self.inter = torch, most, hidden, heads, kv, inter
        self.hd = hd = hidden // heads
        g = gen(torch, seed)
        self.qkv_n = (heads + 2 * kv) * hd
        self.weights = {}
        self.plain = {}
        for name, (n, k) in dict(qkv=(self.qkv_n, hidden), o=(hidden, hidden), gu=(2 * inter, hidden), down=(hidden, inter)).items():
            w = (torch.randn(n, k, device="cuda", generator=g) * 0.05).bfloat16()
            codes, scales = torch.zeros(n, k, dtype=torch.int8, device="cuda"), torch.zeros(n, device="cuda")
            R.quantize_rows(ptr(w), "bf16", k, n, k, ptr(codes), k, ptr(scales), stream(torch))
            self.weights[name] = (codes, scales)
        self.bias = torch.randn(self.qkv_n, device="cuda", generator=g).bfloat16()
        self.norms = [(1 + 0.1 * torch.randn(hidden, device="cuda", generator=g)).bfloat16() for _ in range(3)]
        self.inv = (1e4 ** -(torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)).float()
        self.pages, self.ps, self.R = 64, 16, 3
        self.k, self.v = (torch.zeros(self.pages * self.ps, kv, hd, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        self.cache = R.PagedCache(ptr(self.k), ptr(self.v), "bf16", kv, hd, self.ps, self.pages)
        self.table = torch.arange(self.pages, device="cuda", dtype=torch.int32).view(4, 16)[:3].contiguous()
        f = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
        b = lambda *s: torch.zeros(*s, dtype=torch.int8, device="cuda")  # noqa: E731
        i = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
        self.x, self.qkv, self.att, self.o, self.gu, self.d, self.y = (f(most, n) for n in (
            hidden, self.qkv_n, hidden, hidden, 2 * inter, hidden, hidden))
        self.c1, self.c2, self.c3, self.c4 = b(most, hidden), b(most, hidden), b(most, hidden), b(most, inter)
        self.s1, self.s2, self.s3, self.s4 = (f(most) for _ in range(4))
        self.row_start, self.start, self.pos = i(4), i(3), i(most)
        self.slots = torch.full((most,), -1, dtype=torch.int64, device="cuda")
        wa = R.paged_attention_workspace(most, 3, heads, kv, hd)
        self.wa = torch.zeros(wa, dtype=torch.uint8, device="cuda")
        self.wl = torch.zeros(max(R.linear_i8_workspace(most, n, k) for n, k in ((self.qkv_n, hidden), (2 * inter, hidden), (hidden, inter))),
                              dtype=torch.uint8, device="cuda")

    def batch(self, past, add, seed):
        torch = self.torch
        rows = sum(add)
        pos = np.concatenate([p + np.arange(a) for p, a in zip(past, add)] or [[]])
        req = np.concatenate([np.full(a, r) for r, a in enumerate(add)] or [[]]).astype(int)
        slots = np.full(self.most, -1, np.int64)
        table = self.table.cpu().numpy()
        slots[:rows] = table[req, pos.astype(int) // self.ps] * self.ps + pos.astype(int) % self.ps
        full = np.zeros(self.most, np.int32)
        full[:rows] = pos
        self.row_start.copy_(torch.from_numpy(np.cumsum([0, *add]).astype(np.int32)))
        self.start.copy_(torch.tensor(past, dtype=torch.int32))
        self.pos.copy_(torch.from_numpy(full))
        self.slots.copy_(torch.from_numpy(slots))
        self.x.copy_(torch.randn(self.most, self.hidden, device="cuda", generator=gen(torch, seed)))
        self.d.copy_(torch.randn(self.most, self.hidden, device="cuda", generator=gen(torch, seed + 1)))

    def product(self, name, codes, scales, bias, out, s):
        w, ws = self.weights[name]
        n, k = w.shape
        R.linear_i8(ptr(w), k, ptr(ws), ptr(codes), k, ptr(scales), ptr(bias), ptr(out), n, self.most, n, k, ptr(self.wl), self.wl.numel(), s)

    def step(self):
        s, T, h, H, K, hd = stream(self.torch), self.most, self.hidden, self.heads, self.kv, self.hd
        # (x is the residual, d what the block before this adds to it)
        R.add_norm(ptr(self.x), h, ptr(self.d), h, T, h, ptr(self.norms[0]), "bf16", EPS, ptr(self.x), h, None, 0, ptr(self.c1), h, ptr(self.s1), s)
        self.product("qkv", self.c1, self.s1, self.bias, self.qkv, s)
        ld, base = self.qkv_n, ptr(self.qkv)
        R.norm_rope_append(self.cache, base, ld, base + 4 * H * hd, ld, base + 4 * (H + K) * hd, ld, T, H, base, ld, ptr(self.inv),
                           ptr(self.pos), ptr(self.slots), "split_half", None, None, EPS, s)
        R.paged_attention(self.cache, ptr(self.table), 16, ptr(self.row_start), ptr(self.start), 3, base, ld, ptr(self.att), h, T, H,
                          hd ** -0.5, 0, ptr(self.wa), self.wa.numel(), s)
        R.quantize_rows(ptr(self.att), "f32", h, T, h, ptr(self.c2), h, ptr(self.s2), s)
        self.product("o", self.c2, self.s2, None, self.o, s)
        R.add_norm(ptr(self.x), h, ptr(self.o), h, T, h, ptr(self.norms[1]), "bf16", EPS, ptr(self.x), h, None, 0, ptr(self.c3), h, ptr(self.s3), s)
        self.product("gu", self.c3, self.s3, None, self.gu, s)
        R.silu_mul(ptr(self.gu), 2 * self.inter, ptr(self.gu) + 4 * self.inter, 2 * self.inter, T, self.inter, ptr(self.c4), self.inter,
                   ptr(self.s4), s)
        self.product("down", self.c4, self.s4, None, self.d, s)
        # the last norm, in f32 for the vocabulary's product in bf16
        R.add_norm(ptr(self.x), h, ptr(self.d), h, T, h, ptr(self.norms[2]), "bf16", EPS, None, 0, ptr(self.y), h, None, 0, None, s)

    def state(self):
        return [t.clone() for t in (self.x, self.qkv, self.att, self.o, self.gu, self.d, self.y, self.c1, self.c2, self.c3, self.c4, self.s1,
                                    self.s2, self.s3, self.s4, self.k, self.v)]

    def check(self, x0, d0, rows):
        """Every stage against 64 bits on what the stage before it left."""
        n = lambda t: t.double().cpu().numpy()  # noqa: E731
        h1 = n(x0 + d0)
        check_codes(n(self.c1), n(self.s1), norm_value(h1, n(self.norms[0])))
        check_codes(n(self.c2), n(self.s2), n(self.att))
        assert self.torch.equal(self.x, (x0 + d0) + self.o)
        check_codes(n(self.c3), n(self.s3), norm_value(n(self.x), n(self.norms[1])))
        gu = self.gu.cpu().numpy()
        check_codes(n(self.c4), n(self.s4), gate_value(gu[:, : self.inter], gu[:, self.inter:].astype(np.float64)))
        for name, c, s, out in (("o", self.c2, self.s2, self.o), ("gu", self.c3, self.s3, self.gu), ("down", self.c4, self.s4, self.d)):
            w, ws = self.weights[name]
            want = ((c.double() @ w.double().t()).float() * s[:, None]) * ws
            assert self.torch.equal(out, want), name
        w, ws = self.weights["qkv"]
        qkv = ((self.c1.double() @ w.double().t()).float() * self.s1[:, None]) * ws + self.bias.float()
        kd = self.heads * self.hd
        assert self.torch.equal(self.qkv[:, kd:], qkv[:, kd:])  # (q is turned in place)
        v = qkv[:, kd + self.kv * self.hd:].view(self.most, self.kv, self.hd).bfloat16()
        live = self.slots[:rows]
        assert self.torch.equal(self.v[live], v[:rows])
        check_y(n(self.y), norm_value((self.x + self.d).cpu().numpy(), n(self.norms[2])))


BATCHES = [((0, 0, 0), (20, 7, 1)), ((20, 7, 1), (1, 1, 1)), ((21, 8, 2), (5, 0, 3)), ((26, 8, 5), (1, 30, 1))]


def test_a_block_of_products(torch):
    block = Block(torch, 40)
    for i, (past, add) in enumerate(BATCHES):
        block.batch(past, add, 10 * i)
        x0, d0 = block.x.clone(), block.d.clone()
        block.step()
        block.check(x0, d0, sum(add))


def test_a_captured_block_equals_an_eager_one(torch):
    eager, captured = Block(torch, 40), Block(torch, 40)
    for b in (eager, captured):  # what a first call sets up is set up outside of the capture
        b.batch(*BATCHES[0], 0)
        b.step()
        b.k.zero_(), b.v.zero_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step()
    for i, (past, add) in enumerate(BATCHES + BATCHES[:1]):
        for b in (eager, captured):
            b.batch(past, add, 10 * i)
        eager.step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager.state(), captured.state()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 5, 40, 300])
def test_calls_repeat_to_the_bit(torch, rows):
    block = Block(torch, rows, hidden=896, heads=14, kv=2, inter=4864)
    add = (rows, 0, 0)
    first = None
    for _ in range(3):
        block.batch((0, 0, 0), add if rows <= 256 else (256, 44, 0), 1)
        block.step()
        state = block.state()
        first = first or state
        for a, b in zip(first, state):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------
# The ends of each kernel's widths, up to the widest rows that registers hold
# ---------------------------------------------------------------------------
EDGES = [2048, 2049, 4097, 8193, 16385, 24571, 24576, 24577, 24592, 28001, 32765, 32768, 32769, 32784]


def far_rows(torch, width, ld, seed):
    """Rows whose largest value is one of the last, another one of each (so that a value that is dropped shows in all)."""
    x = torch.randn(5, ld, device="cuda", generator=gen(torch, seed))
    x[:, width:] = float("nan")
    for r in range(5):
        x[r, max(0, width - 1 - 3 * r)] = 20.0 + r
    return x


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("width", EDGES)
def test_quantize_rows_at_the_ends_of_widths(torch, width, kind):
    ld = up(width, 8) + 8
    x = far_rows(torch, width, ld, width)
    x = x if kind == "f32" else x.bfloat16()
    out = Codes(torch, 5, width, 1)
    R.quantize_rows(ptr(x), kind, ld, 5, width, *out.args, stream(torch))
    equal_codes(*out.get(), x[:, :width].double().cpu().numpy())


@pytest.mark.parametrize("place", ["apart", "sum is x", "y is x", "y is delta, sum is x", "y is x, no sum", "y is delta, no sum"])
@pytest.mark.parametrize("width", EDGES)
def test_add_norm_at_the_ends_of_widths(torch, width, place):
    ld = up(width, 4) + 4
    g = gen(torch, width + 3)
    x, d = far_rows(torch, width, ld, width + 1), torch.randn(5, ld, device="cuda", generator=g)
    w = (1 + 0.3 * torch.randn(width, device="cuda", generator=g)).to(torch.bfloat16 if width % 2 else torch.float32)
    h = (x + d)[:, :width].cpu().numpy()
    other, more = torch.full((5, ld), 77.0, device="cuda"), torch.full((5, ld), 77.0, device="cuda")
    total, y = {"apart": (other, more), "sum is x": (x, None), "y is x": (other, x), "y is delta, sum is x": (x, d),
                "y is x, no sum": (None, x), "y is delta, no sum": (None, d)}[place]
    behind = [None if t is None else t[:, width:].cpu().numpy() for t in (total, y)]
    out = Codes(torch, 5, width, 1)
    R.add_norm(ptr(x), ld, ptr(d), ld, 5, width, ptr(w), "bf16" if width % 2 else "f32", EPS, ptr(total), ld, ptr(y), ld, *out.args,
               stream(torch))
    v = norm_value(h, w.double().cpu().numpy())
    check_codes(*out.get(), v)
    if total is not None:
        assert np.array_equal(total[:, :width].cpu().numpy(), h)
    if y is not None:
        check_y(y[:, :width].double().cpu().numpy(), v)
    for t, b in zip((total, y), behind):
        assert t is None or np.array_equal(t[:, width:].cpu().numpy(), b, equal_nan=True)


@pytest.mark.parametrize("width", EDGES)
def test_silu_mul_at_the_ends_of_widths(torch, width):
    ld = up(width, 4) + 4
    gate, u = far_rows(torch, width, ld, width + 4), far_rows(torch, width, ld, width + 5)
    gate[4, :width] *= 60  # gates of -150 and less
    out = Codes(torch, 5, width, 1)
    R.silu_mul(ptr(gate), ld, ptr(u), ld, 5, width, *out.args, stream(torch))
    check_codes(*out.get(), gate_value(gate[:, :width].cpu().numpy(), u[:, :width].double().cpu().numpy()))


# ---------------------------------------------------------------------------
# Workspaces that calls leave parts of K in
# ---------------------------------------------------------------------------
class Space:
    """A workspace of what calls of these sizes ask for, with marks behind it."""

    def __init__(self, torch, sizes):
        self.bytes = max(R.linear_i8_workspace(*s) for s in sizes)
        self.all = torch.full((self.bytes + 4096,), 7, dtype=torch.uint8, device="cuda")
        self.part = self.all[: self.bytes]

    def fill(self, torch, seed):
        self.part.random_(0, 256, generator=gen(torch, seed))

    def check(self):
        assert (self.all[self.bytes:] == 7).all(), "written behind the workspace"


@pytest.mark.parametrize("size", SPLIT)
def test_linear_i8_writes_no_more_than_its_workspace(torch, size):
    space = Space(torch, [size])
    p = Product(torch, *size, bias=True, space=space.part, seed=7)
    for i in range(2):
        space.fill(torch, i)
        p.run()
        p.check()
    space.check()


def test_linear_i8_one_workspace_for_parts_of_all_sizes(torch):
    """A workspace made for the largest call serves calls with parts and without, in any order, whatever is in it."""
    sizes = [s for pair in zip(SPLIT, [(1, 2048, 2048), (5, 40, 131056), (48, 1152, 8192), (129, 300, 4096)] * 3) for s in pair]
    space = Space(torch, sizes)
    products = [Product(torch, *s, bias=i % 3 == 0, pady=i % 2, space=space.part, seed=i) for i, s in enumerate(sizes)]
    for turn in range(3):
        space.fill(torch, turn)
        for p in products:
            p.run()
        torch.cuda.synchronize()
        for p in products:
            p.check()
        products = products[::-1] if turn else products[7:] + products[:7]
    space.check()


@pytest.mark.parametrize("first,second", [(0, 1), (2, 4), (3, 5), (6, 0), (7, 8)])
def test_linear_i8_parts_on_two_streams(torch, first, second):
    """Calls with parts that overlap, a workspace each."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    products = [Product(torch, *SPLIT[i], seed=8) for i in (first, second)]
    torch.cuda.synchronize()
    for _ in range(10):
        for p, s in zip(products, streams):
            p.run(s.cuda_stream)
    torch.cuda.synchronize()
    for p in products:
        p.check()


def test_linear_i8_two_graphs_with_one_workspace(torch):
    """Graphs that are replayed one after the other may share it, with eager calls on it in between."""
    sizes = [SPLIT[0], SPLIT[1], SPLIT[4], SPLIT[5]]
    space = Space(torch, sizes)
    products = [Product(torch, *s, bias=True, space=space.part, seed=20 + i) for i, s in enumerate(sizes)]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, part in zip(graphs, (products[:2], products[2:])):
        with torch.cuda.graph(graph):
            for p in part:
                p.run()
    eager = Product(torch, *SPLIT[6], space=space.part, seed=30)
    for i in range(4):
        for p in products:
            p.X.copy_(p.X.roll(i, 0))
        for graph in graphs[:: 1 if i % 2 else -1]:
            graph.replay()
            eager.run()
        torch.cuda.synchronize()
        for p in products + [eager]:
            p.check()
    space.check()


# ---------------------------------------------------------------------------
# Rows far apart, and more of them than a launch takes
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("which", ["W", "X", "Y"])
@pytest.mark.parametrize("M,N,K", FAR)
def test_linear_i8_strides_over_4_MiB(torch, M, N, K, which):
    p = Product(torch, M, N, K, bias=True, pady=FAR_STRIDE // 4 - N if which == "Y" else 0, seed=9)
    if which != "Y":
        tight = getattr(p, which)
        far = torch.zeros(len(tight), FAR_STRIDE, dtype=torch.int8, device="cuda")
        far[:, :K] = tight
        far[:, K:K + 64] = 99
        setattr(p, which, far)
        p.strides = tuple(FAR_STRIDE if n == which else s for n, s in zip("WXY", p.strides))
    want = p.want()
    for _ in range(2):
        p.run()
        assert torch.equal(p.Y[:M, :N], want)
        assert (p.Y[:M, N:] == 55).all() and (p.Y[M:] == 55).all()
        p.Y.fill_(55.0)


@pytest.mark.parametrize("M,N,K", HUGE)
def test_linear_i8_more_blocks_than_a_launch_takes(torch, M, N, K):
    p = Product(torch, M, N, K, bias=True, seed=10)
    p.run()
    part = 1 << 24
    for m in range(0, M, part):
        for n in range(0, N, part):
            rows, cols = slice(m, min(m + part, M)), slice(n, min(n + part, N))
            # (whole numbers below 2^24; one side has one row)
            y = (p.X[rows].float() * p.W[cols].float()).sum(-1).view(rows.stop - m, cols.stop - n)
            want = (y * p.xs[rows, None]) * p.ws[cols] + p.bias[cols].float()
            assert torch.equal(p.Y[rows, cols], want), (m, n)
    assert (p.Y[M:] == 55).all()


# ---------------------------------------------------------------------------
# Calls that share inputs, rows by the million, rows far apart, the least scales
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("width", [5, 401, 2050, 18944, 33000])
@pytest.mark.parametrize("place", ["apart", "sum is both", "y is both"])
def test_add_norm_of_rows_and_themselves(torch, width, place):
    ld = up(width, 4)
    x, w = torch.randn(4, ld, device="cuda", generator=gen(torch, 13)), torch.randn(width, device="cuda", generator=gen(torch, 14))
    h = (x + x)[:, :width].cpu().numpy()
    total, y = {"apart": (torch.zeros_like(x), torch.zeros_like(x)), "sum is both": (x, torch.zeros_like(x)), "y is both": (None, x)}[place]
    out = Codes(torch, 4, width)
    R.add_norm(ptr(x), ld, ptr(x), ld, 4, width, ptr(w), "f32", EPS, ptr(total), ld, ptr(y), ld, *out.args, stream(torch))
    v = norm_value(h, w.double().cpu().numpy())
    check_codes(*out.get(), v)
    check_y(y[:, :width].double().cpu().numpy(), v)
    assert total is None or np.array_equal(total[:, :width].cpu().numpy(), h)


@pytest.mark.parametrize("width", [5, 401, 2050, 18944, 33000])
def test_silu_mul_of_rows_and_themselves(torch, width):
    ld = up(width, 4)
    x, out = torch.randn(4, ld, device="cuda", generator=gen(torch, 15)), Codes(torch, 4, width)
    R.silu_mul(ptr(x), ld, ptr(x), ld, 4, width, *out.args, stream(torch))
    v = x[:, :width].cpu().numpy()
    check_codes(*out.get(), gate_value(v, v.astype(np.float64)))


@pytest.mark.parametrize("n,K", [(1, 64), (20, 640), (300, 1040), (311, 6768)])
def test_linear_i8_of_rows_and_themselves(torch, n, K):
    p = Product(torch, n, n, K)
    p.W, p.ws = p.X, p.xs
    p.run()
    p.check()


@pytest.mark.parametrize("rows,width", [((1 << 22) + 5, 20), ((1 << 20) + 3, 1028)])
def test_norm_and_gate_of_more_rows_than_a_launch_has_blocks(torch, rows, width):
    g = gen(torch, 16)
    x, d = (torch.empty(rows, width, device="cuda").uniform_(-2, 2, generator=g) for _ in range(2))
    w = torch.randn(width, device="cuda", generator=g)
    some = torch.cat([torch.arange(200), torch.randint(0, rows, (200,)), torch.arange(rows - 200, rows)]).cuda()
    n = lambda t: t.double().cpu().numpy()  # noqa: E731

    def outputs():
        codes = torch.full((rows + 1, up(width, 16)), 99, dtype=torch.int8, device="cuda")
        return codes, torch.full((rows + 1,), -5.0, device="cuda")

    def check(codes, scales, v):
        assert (codes[rows] == 99).all() and scales[rows] == -5 and (codes[:rows, width:] == 0).all()
        assert (scales[:rows] > 0).all() and (codes[:rows].abs().amax(-1) == 127).all()  # (every row was formed)
        check_codes(n(codes[some, :width]), n(scales[some]), v)

    codes, scales = outputs()
    R.silu_mul(ptr(x), width, ptr(d), width, rows, width, ptr(codes), codes.shape[1], ptr(scales), stream(torch))
    check(codes, scales, gate_value(x[some].cpu().numpy(), n(d[some])))
    h = x + d
    codes, scales = outputs()
    R.add_norm(ptr(x), width, ptr(d), width, rows, width, ptr(w), "f32", EPS, ptr(x), width, ptr(d), width, ptr(codes), codes.shape[1],
               ptr(scales), stream(torch))
    v = norm_value(h[some].cpu().numpy(), n(w))
    check(codes, scales, v)
    check_y(n(d[some]), v)
    assert torch.equal(x, h)


def test_norm_and_gate_offsets_past_32_bits(torch):
    """Strides that put the last rows' values and codes behind 2^32 bytes."""
    ld, rows, width = 1 << 28, 6, 1000
    g = gen(torch, 17)
    x, d = (torch.zeros(rows, ld, device="cuda") for _ in range(2))
    for t in (x, d):
        t[:, :width] = torch.randn(rows, width, device="cuda", generator=g)
    w = torch.randn(width, device="cuda", generator=g)
    codes, scales = torch.zeros(rows, 1 << 30, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    n = lambda t: t.double().cpu().numpy()  # noqa: E731
    v = gate_value(x[:, :width].cpu().numpy(), n(d[:, :width]))
    R.silu_mul(ptr(x), ld, ptr(d), ld, rows, width, ptr(codes), 1 << 30, ptr(scales), stream(torch))
    check_codes(n(codes[:, :width]), n(scales), v)
    h = (x[:, :width] + d[:, :width]).cpu().numpy()
    R.add_norm(ptr(x), ld, ptr(d), ld, rows, width, ptr(w), "f32", EPS, ptr(x), ld, ptr(d), ld, ptr(codes), 1 << 30, ptr(scales), stream(torch))
    v = norm_value(h, n(w))
    check_codes(n(codes[:, :width]), n(scales), v)
    check_y(n(d[:, :width]), v)
    assert np.array_equal(x[:, :width].cpu().numpy(), h) and not x[:, width:width + 64].any() and not d[:, width:width + 64].any()


@pytest.mark.parametrize("width", [33, 2000, 33000])
def test_least_scales(torch, width):
    """Scales of few bits: the codes of values that 127 of them do not reach are 127 and -127."""
    rows, ld, least = 12, up(width, 8), 2.0 ** -149
    rng = np.random.RandomState(width)
    tops = np.array([63, 64, 127, 190, 191, 254, 300, 1000, 5000, 100000, 1 << 20, 1 << 24])  # (in steps of the denormals)
    m = rng.randint(-tops[:, None], tops[:, None] + 1, (rows, width)).astype(np.float64)
    m[:, width // 2] = tops
    x = torch.zeros(rows, ld, device="cuda")
    x[:, :width] = torch.from_numpy((m * least).astype(np.float32)).cuda()
    assert np.array_equal(x[:, :width].double().cpu().numpy(), m * least)
    out = Codes(torch, rows, width)
    R.quantize_rows(ptr(x), "f32", ld, rows, width, *out.args, stream(torch))
    codes, scales = out.get()
    equal_codes(codes, scales, m * least)
    assert scales[0] == 0 and scales[3] == least and codes[3, width // 2] == 127 and abs(m[3, width // 2] - 127) > 60
    half = (x * 2.0 ** 16).bfloat16()  # (whole steps of bf16's denormals, or its 8 bits)
    out = Codes(torch, rows, width)
    R.quantize_rows(ptr(half), "bf16", ld, rows, width, *out.args, stream(torch))
    equal_codes(*out.get(), half[:, :width].double().cpu().numpy())
    gate = torch.randn(rows, ld, device="cuda", generator=gen(torch, 18))
    out = Codes(torch, rows, width)
    R.silu_mul(ptr(gate), ld, ptr(x), ld, rows, width, *out.args, stream(torch))
    check_codes(*out.get(), gate_value(gate[:, :width].cpu().numpy(), m * least))
    for t in x[[3, 6, 8]]:
        y, out = torch.zeros(rows, ld, device="cuda"), Codes(torch, rows, width)
        R.add_norm(ptr(gate), ld, None, 0, rows, width, ptr(t), "f32", EPS, None, 0, ptr(y), ld, *out.args, stream(torch))
        v = norm_value(gate[:, :width].cpu().numpy(), t[:width].double().cpu().numpy())
        check_codes(*out.get(), v)
        check_y(y[:, :width].double().cpu().numpy(), v)


def test_products_from_two_threads(torch):
    """Calls at once from two threads of the host, a stream and a workspace each."""
    import threading

    products = [Product(torch, *SPLIT[i], bias=True, seed=40 + i) for i in (0, 1)] + [Product(torch, *s, seed=43) for s in ((5, 413, 2672), (300, 896, 896))]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    failed = []

    def work(k):
        try:
            for _ in range(10):
                for p in products[k::2]:
                    p.run(streams[k].cuda_stream)
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed
    for p in products:
        p.check()
