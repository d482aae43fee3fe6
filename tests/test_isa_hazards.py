"""Wait states that the compiler does not see to because the instruction stands in inline assembly, looked for in the library
as it was built: CPU only, with the disassembler of the ROCm installation."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
REGISTER = re.compile(r"s\[(\d+):(\d+)\]|s(\d+)$")


def scalars(operand):
    m = REGISTER.match(operand.strip())
    if not m:
        return set()
    return {int(m[3])} if m[3] else set(range(int(m[1]), int(m[2]) + 1))


def states(name, rest):
    return int(rest.strip(), 0) + 1 if name == "s_nop" else 1


def too_near(lines):
    """(loads into LDS with a scalar address, those of them that follow a vector instruction's write of that address within five
    wait states)."""
    code = []
    for line in lines:
        line = line.split("//")[0].strip()
        if line and not line.endswith(":"):
            name, _, rest = line.partition(" ")
            code.append((name, rest))
    found, bad = 0, []
    for n, (name, rest) in enumerate(code):
        if not name.startswith("global_load_lds"):
            continue
        address = scalars(rest.split(",")[1].split()[0])
        if not address:
            continue
        found += 1
        passed, at = 0, n - 1
        while at >= 0 and passed < 5:
            before, args = code[at]
            if before in ("s_branch", "s_endpgm", "s_setpc_b64"):
                break
            if before.startswith("v_") and scalars(args.split(",")[0]) & address:
                bad.append([" ".join(c) for c in code[at:n + 1]])
                break
            passed += states(before, args)
            at -= 1
    return found, bad


def test_the_check_sees_a_short_wait():
    pair = ["v_readfirstlane_b32 s7, v5", "v_readfirstlane_b32 s6, v4"]
    load = ["s_mov_b32 m0, s35", "s_nop %d", "global_load_lds_dwordx4 v6, s[6:7]"]
    for nop, short in ((0, True), (2, True), (3, False), (4, False)):
        found, bad = too_near(pair + [x.replace("%d", str(nop)) for x in load])
        assert found == 1 and bool(bad) == short, nop


def test_loads_into_lds_wait_for_their_address(tmp_path):
    lib = os.path.join(ROOT, "vit_amd", "libvtcnn_hip.so")
    if not os.path.exists(lib) or not os.path.exists(OBJDUMP):
        pytest.skip("no built library or no disassembler")
    shutil.copy(lib, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    found = 0
    for part in sorted(tmp_path.glob("lib.so.*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(part)], check=True, stdout=subprocess.PIPE, text=True).stdout
        n, bad = too_near(text.splitlines())
        found += n
        assert not bad, (part.name, len(bad), bad[0])
    assert found > 100  # the attention's kernels are in the library
