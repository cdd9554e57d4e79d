"""What the compiler cannot see to in loads to LDS that are written as instructions, looked for in the library's own device code, without a GPU."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJ = os.path.join(ROOT, "aws_ofi_nccl_amd", "lib", "obj")
LLVM = "/opt/rocm/llvm/bin"
STATES = 5  # between a vector instruction's write of a scalar register and a memory instruction that reads it
SOURCES = ["expert_product", "expert_grad", "expert_weight_grad", "expert_few"]


def device_code(name, tmp):
    """Instructions, one a line, labels among them."""
    obj = os.path.join(OBJ, name + ".hip.o")
    if not os.path.exists(obj):
        from aws_ofi_nccl_amd import build
        build.build_library()
    bundle, code = os.path.join(tmp, name + ".bundle"), os.path.join(tmp, name + ".o")
    subprocess.run([LLVM + "/llvm-objcopy", "--dump-section", ".hip_fatbin=" + bundle, obj, os.path.join(tmp, "rest.o")], check=True)
    subprocess.run([LLVM + "/clang-offload-bundler", "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
                    "--input=" + bundle, "--output=" + code], check=True)
    text = subprocess.run([LLVM + "/llvm-objdump", "-d", "--no-show-raw-insn", "--no-leading-addr", code], stdout=subprocess.PIPE, check=True,
                          text=True).stdout
    return [line.split("//")[0].strip() for line in text.splitlines() if line.startswith("\t")]


def scalars(operand):
    """The scalar registers of an operand: s7, s[4:7]."""
    one, run = re.fullmatch(r"s(\d+)", operand), re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    return {int(one[1])} if one else set(range(int(run[1]), int(run[2]) + 1)) if run else set()


def too_early(code):
    """Buffer loads to LDS whose descriptor a vector instruction wrote fewer than STATES wait states before, as (write, load)."""
    found, loads = [], 0
    for k, line in enumerate(code):
        if not (line.startswith("buffer_load") and line.endswith(" lds")):
            continue
        loads += 1
        reads, states = scalars(line.split(",")[1].strip()), 0
        for before in reversed(code[max(0, k - STATES):k]):
            if states >= STATES:
                break
            name, _, operands = before.partition(" ")
            if name.startswith("v_") and scalars(operands.split(",")[0].strip()) & reads:
                found.append((before, line))
                break
            states += 1 + (int(operands) if name == "s_nop" else 0)
    return found, loads


def test_the_search_finds_an_early_load():
    load = "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    for write in ("v_readfirstlane_b32 s6, v8", "v_readlane_b32 s5, v197, 7", "v_cmp_eq_u32_e64 s[6:7], v0, v1"):
        assert too_early([write, "s_mov_b32 m0, s9", "s_nop 0", load]) == ([(write, load)], 1)
        assert too_early([write, "s_mov_b32 m0, s9", "s_nop 2", load]) == ([(write, load)], 1)
        assert too_early([write, "s_mov_b32 m0, s9", "s_nop 3", load]) == ([], 1)
    assert too_early(["v_readfirstlane_b32 s8, v8", load]) == ([], 1)


@pytest.mark.parametrize("name", SOURCES)
def test_descriptors_are_there_when_a_load_to_lds_reads_them(name, tmp_path):
    if not os.path.exists(LLVM + "/llvm-objdump"):
        pytest.skip("no disassembler")
    found, loads = too_early(device_code(name, str(tmp_path)))
    assert not found, "%d of %d, the first: %s / %s" % (len(found), loads, *found[0])
    assert loads > 0 or name == "expert_few"


def test_the_place_in_lds_is_set_for_each_load(tmp_path):
    """M0, which has it, is the compiler's too: behind a load that sets it, the compiler's next one sets it anew."""
    from aws_ofi_nccl_amd import build
    if not os.path.exists(build.HIPCC):
        pytest.skip("no compiler")
    out = os.path.join(str(tmp_path), "places.s")
    subprocess.run([build.HIPCC] + build.COMMON + ["-w", "--cuda-device-only", "-S", "-x", "hip",
                                                   os.path.join(ROOT, "tests", "host", "lds_places_kernel.hip"), "-o", out], check=True)
    with open(out) as f:
        code = [line.split(";")[0].strip() for line in f]
    set_since, loads = False, 0
    for line in code:
        set_since = set_since or bool(re.match(r"s_\w+ m0,", line))
        if line.startswith("buffer_load") and line.endswith(" lds"):
            assert set_since, line
            set_since, loads = False, loads + 1
    assert loads == 5
