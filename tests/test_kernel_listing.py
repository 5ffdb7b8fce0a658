"""The attention kernels over a paged cache as the compiler writes them, without a GPU: two faults of the compiler were found
in them, which leave wrong results and no error, so every build of them is looked over for both.

* A matrix product's result is read by another instruction before the product has written it. Nothing in the hardware
  waits there: the compiler has to spend the wait states, and it has counted them along one of two ways to the read.
* A spilled vector register is stored (or loaded) at a block's start ahead of the instruction that gives the lanes of a
  divergent region back, so that those lanes keep what was in memory (or in the register).
"""
import re
import shlex
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "vvli_amd" / "csrc"

# Passes (4 cycles each) of the products that the kernels use, and wait states between a product and another instruction
# that touches its result: passes + 4 for 16-bit operands, passes + 2 for f32 ones.
PRODUCTS = {"v_mfma_f32_16x16x32_bf16": 4 + 4, "v_mfma_f32_16x16x32_f16": 4 + 4, "v_mfma_f32_32x32x16_bf16": 8 + 4,
            "v_mfma_f32_32x32x16_f16": 8 + 4, "v_mfma_f32_16x16x4_f32": 8 + 2, "v_mfma_f32_32x32x2_f32": 16 + 2}
REG = re.compile(r"\b([va])(?:\[(\d+):(\d+)\]|(\d+)\b)")
LOADS = ("ds_read", "global_load", "scratch_load", "buffer_load", "flat_load")


def registers(text):
    out = set()
    for kind, lo, hi, one in REG.findall(text):
        out |= {(kind, int(one))} if one else {(kind, i) for i in range(int(lo), int(hi) + 1)}
    return out


def kernels(listing):
    """(name, lines) of every function."""
    for m in re.finditer(r"^(_Z\w+):[^\n]*\n(.*?)^\.Lfunc_end", listing, re.S | re.M):
        yield m.group(1), m.group(2).split("\n")


def instructions(lines):
    """[(operation, operands)] and the place of every label among them."""
    ins, labels = [], {}
    for line in lines:
        label = re.match(r"(\.LBB\w+):", line)
        if label:
            labels[label.group(1)] = len(ins)
        text = line.split(";")[0].strip()
        if line.startswith("\t") and text and not text.startswith("."):
            op, _, operands = text.partition(" ")
            ins.append((op, operands.strip()))
    return ins, labels


def early_reads(lines):
    """Instructions that touch a product's result too early, on any way through the function."""
    ins, labels = instructions(lines)
    found = []
    for i, (op, operands) in enumerate(ins):
        if not op.startswith("v_mfma"):
            continue
        need, parts = PRODUCTS[op], [p.strip() for p in operands.split(",")]
        result = registers(parts[0])
        ways, seen = [(i + 1, 0)], {}
        while ways:
            k, waited = ways.pop()
            if k >= len(ins) or waited >= need or seen.get(k, need) <= waited:
                continue
            seen[k] = waited
            o, a = ins[k]
            if o == "s_nop":
                ways.append((k + 1, waited + int(a, 0) + 1))
                continue
            if o == "s_endpgm":
                continue
            args = [p.strip() for p in a.split(",")]
            if o.startswith("v_mfma"):
                if registers(args[1] + " " + args[2]) & result:
                    found.append(f"{op} {operands} -> {o} {a}: {waited} of {need}")
                if registers(args[0]) & result:  # (the next one of the same sum: products wait for each other's sums)
                    continue
            elif o.startswith(("v_", "ds_", "global_", "scratch_", "buffer_", "flat_")):
                touched = ",".join(args[1:]) if o.startswith(LOADS) else a  # (a load's own result comes far later)
                if registers(touched) & result:
                    found.append(f"{op} {operands} -> {o} {a}: {waited} of {need}")
                    continue
            if o == "s_branch":
                ways.append((labels[a], waited + 1))
                continue
            if o.startswith("s_cbranch"):
                ways.append((labels[a], waited + 1))
            ways.append((k + 1, waited + 1))
    return found


def spills_ahead_of_exec(lines):
    """Spills and reloads of vector registers between a block's start and the s_or_b64 exec that stands in it."""
    found, block = [], []
    for line in lines:
        if re.match(r"\.LBB|; %bb", line):
            block = []
        text = line.strip()
        if not line.startswith("\t") or text.startswith((";", ".")):
            continue
        if re.match(r"s_or_b64\s+exec, exec", text):
            found += [t for t in block if re.search(r"Folded (Spill|Reload)|Reload Reuse", t) and re.match(r"scratch_|v_accvgpr", t)]
            block = []
        block.append(text)
        if re.match(r"s_c?branch|s_endpgm", text):
            block = []
    return found


@pytest.fixture(scope="module")
def listing(tmp_path_factory):
    plan = subprocess.run(["make", "-n", "-B", "-C", str(CSRC)], check=True, capture_output=True, text=True).stdout
    command = shlex.split(next(line for line in plan.split("\n") if "-c " in line and "paged_attention.hip" in line))
    if not shutil.which(command[0]):
        pytest.skip("no device compiler")
    out = tmp_path_factory.mktemp("listing") / "paged_attention.s"
    command[command.index("-o") + 1] = str(out)
    command[command.index("-c")] = "-S"
    subprocess.run(command + ["--cuda-device-only"], check=True, capture_output=True)
    return out.read_text()


def test_listing_holds_the_kernels(listing):
    names = [name for name, lines in kernels(listing) if any("v_mfma" in line for line in lines)]
    assert len([n for n in names if "paged_attn_kernel" in n]) == 9 and len([n for n in names if "paged_wide_kernel" in n]) == 9


def test_results_of_products_are_not_read_early(listing):
    bad = {name: found for name, lines in kernels(listing) if (found := early_reads(lines))}
    assert not bad, bad


def test_spills_stand_behind_the_lanes_return(listing):
    bad = {name: found for name, lines in kernels(listing) if (found := spills_ahead_of_exec(lines))}
    assert not bad, bad


# ---------------------------------------------------------------------------
# What the two looks find, on listings written by hand
# ---------------------------------------------------------------------------
PRODUCT = "\tv_mfma_f32_32x32x2_f32 v[0:15], v20, v21, v[0:15]"


@pytest.mark.parametrize("tail,early", [
    ("\ts_nop 15\n\ts_nop 1\n\tv_add_f32_e32 v30, v15, v31", False),
    ("\ts_nop 15\n\ts_nop 0\n\tv_add_f32_e32 v30, v15, v31", True),
    ("\tv_add_f32_e32 v30, v16, v31", False),
    ("\tds_read_b128 v[0:3], v31", False),
    ("\tds_read_b128 v[40:43], v3", True),
    ("\tglobal_store_dwordx4 v30, v[12:15], s[0:1]", True),
    ("\tv_mfma_f32_32x32x2_f32 v[0:15], v20, v21, v[0:15]\n\ts_nop 15\n\ts_nop 1\n\tv_mov_b32_e32 v30, v3", False),
    ("\tv_mfma_f32_32x32x2_f32 v[32:47], v3, v21, v[32:47]", True),
    # one of two ways to the read is long enough
    ("\ts_cbranch_vccz .LBB0_2\n; %bb.1:\n\ts_nop 15\n\ts_nop 1\n.LBB0_2:\n\tv_add_f32_e32 v30, v15, v31", True),
    ("\ts_cbranch_vccz .LBB0_2\n; %bb.1:\n\ts_nop 3\n.LBB0_2:\n\ts_nop 15\n\ts_nop 0\n\tv_add_f32_e32 v30, v15, v31", False),
    # round a loop
    ("\ts_branch .LBB0_1", True),
])
def test_early_reads_are_found(tail, early):
    lines = (".LBB0_1:\n\tv_mul_f32_e32 v30, v1, v31\n" + PRODUCT + "\n" + tail + "\n\ts_endpgm").split("\n")
    assert bool(early_reads(lines)) == early


@pytest.mark.parametrize("block,found", [
    (".LBB0_4:\n\tscratch_store_dword off, v33, off offset:72 ; 4-byte Folded Spill\n\ts_or_b64 exec, exec, s[4:5]", True),
    (".LBB0_4:\n\tscratch_load_dword v33, off, off offset:72 ; 4-byte Folded Reload\n\ts_or_b64 exec, exec, s[4:5]", True),
    (".LBB0_4:\n\ts_or_b64 exec, exec, s[4:5]\n\tscratch_store_dword off, v33, off offset:72 ; 4-byte Folded Spill", False),
    ("; %bb.3:\n\tscratch_store_dword off, v33, off offset:72 ; 4-byte Folded Spill\n.LBB0_4:\n\ts_or_b64 exec, exec, s[4:5]", False),
    (".LBB0_4:\n\tv_mov_b32_e32 v1, v2\n\ts_or_b64 exec, exec, s[4:5]", False),
])
def test_spills_ahead_of_the_lanes_return_are_found(block, found):
    assert bool(spills_ahead_of_exec(block.split("\n"))) == found
