"""The kernels of 8-bit products as the compiler writes them, without a GPU. Two things that no result shows reliably:

* A product's result is not read before the product has written it (see test_kernel_listing.py).
* The tile kernels read the next half's fragments while this half's products run: those loads stand in the source without
  a wait of their own, so the compiler takes their registers as written. Nothing may touch such a register, and nothing
  may spill, between the load and the wait that stands in front of its use.
"""
import re
import shlex
import shutil
import subprocess

import pytest
import test_kernel_listing as listings
from test_kernel_listing import CSRC, early_reads, instructions, kernels, registers

# Passes (4 cycles each) of the products, and 4 more wait states.
PRODUCTS = {"v_mfma_i32_16x16x64_i8": 4 + 4, "v_mfma_i32_32x32x32_i8": 8 + 4}


@pytest.fixture(scope="module")
def listing(tmp_path_factory):
    plan = subprocess.run(["make", "-n", "-B", "-C", str(CSRC)], check=True, capture_output=True, text=True).stdout
    command = shlex.split(next(line for line in plan.split("\n") if "-c " in line and "linear_i8.hip" in line))
    if not shutil.which(command[0]):
        pytest.skip("no device compiler")
    out = tmp_path_factory.mktemp("listing") / "linear_i8.s"
    command[command.index("-o") + 1] = str(out)
    command[command.index("-c")] = "-S"
    subprocess.run(command + ["--cuda-device-only"], check=True, capture_output=True)
    return out.read_text()


def touched_in_flight(lines):
    """Instructions that touch a register which an LDS read is still to write, on any way through the function."""
    ins, labels = instructions(lines)
    found = []
    for i, (op, operands) in enumerate(ins):
        if not op.startswith("ds_read"):
            continue
        result = registers(operands.split(",")[0])
        ways, seen = [i + 1], set()
        while ways:
            k = ways.pop()
            if k >= len(ins) or k in seen:
                continue
            seen.add(k)
            o, a = ins[k]
            if o == "s_endpgm" or (o == "s_waitcnt" and "lgkmcnt(0)" in a):
                continue
            if registers(a) & result:
                found.append(f"{op} {operands} -> {o} {a}")
                continue
            if o == "s_branch":
                ways.append(labels[a])
                continue
            if o.startswith("s_cbranch"):
                ways.append(labels[a])
            ways.append(k + 1)
    return found


def test_listing_holds_the_kernels(listing):
    names = [name for name, lines in kernels(listing) if any("v_mfma" in line for line in lines)]
    assert any("linear_i8_stream_kernel" in n for n in names) and any("linear_i8_tile_kernel" in n for n in names)


def test_results_of_products_are_not_read_early(listing, monkeypatch):
    monkeypatch.setattr(listings, "PRODUCTS", PRODUCTS)
    bad = {name: found for name, lines in kernels(listing) if (found := early_reads(lines))}
    assert not bad, bad


def test_fragments_in_flight_are_left_alone(listing):
    """(The stream kernels' reads have their wait in the same block of assembly, and the compiler counts its own.)"""
    tiles = [(name, lines) for name, lines in kernels(listing) if "linear_i8_tile_kernel" in name]
    bad = {name: found for name, lines in tiles if (found := touched_in_flight(lines))}
    assert tiles and not bad, bad


def test_loops_hold_no_spills(listing):
    """(In front of the loop and behind it they cost nothing that a measurement shows.)"""
    for name, lines in kernels(listing):
        text = "\n".join(lines)
        for block in re.split(r"\n\.LBB\w+:", text):
            if block.count("v_mfma") >= 4 and "s_cbranch" in block:
                assert "scratch_" not in block, name


@pytest.mark.parametrize("tail,bad", [
    ("\ts_waitcnt lgkmcnt(0)\n\tv_add_u32_e32 v9, v1, v2", False),
    ("\tv_add_u32_e32 v9, v1, v20\n\ts_waitcnt lgkmcnt(0)", True),
    ("\tv_add_u32_e32 v9, v5, v20\n\ts_waitcnt lgkmcnt(0)", False),
    ("\ts_waitcnt vmcnt(0)\n\tv_mov_b32_e32 v2, v20", True),
    ("\ts_cbranch_scc0 .LBB0_1\n; %bb.1:\n\ts_waitcnt lgkmcnt(0)", True),  # round the loop to the use at its start
])
def test_touches_in_flight_are_found(tail, bad):
    lines = (".LBB0_1:\n\tv_mul_f32_e32 v30, v1, v31\n\tds_read_b128 v[0:3], v31\n" + tail + "\n\ts_endpgm").split("\n")
    assert bool(touched_in_flight(lines)) == bad
