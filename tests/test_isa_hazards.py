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


def strangers(lines):
    """Instructions that touch m0 and are neither the write directly before a load into LDS (a wait between) nor such a load."""
    code = [x for x in (line.split("//")[0].strip() for line in lines) if re.match(r"[a-z]\w+( |$)", x)]
    return [x for n, x in enumerate(code) if re.search(r"\bm0\b|movrel|gws|ordered_count|_lds_|sendmsg", x) and not x.startswith("global_load_lds_dwordx4")
            and not (x.startswith("s_mov_b32 m0,") and code[n + 1].startswith("s_nop") and code[n + 2].startswith("global_load_lds_dwordx4"))]


def test_the_check_sees_other_users_of_m0():
    load = ["s_mov_b32 m0, s35", "s_nop 4", "global_load_lds_dwordx4 v6, s[6:7]"]
    assert not strangers(load * 2)
    for x in ("s_movrels_b32 s0, s1", "v_mov_b32_e32 v0, m0", "s_mov_b32 m0, -1", "s_sendmsg sendmsg(MSG_INTERRUPT)"):
        assert len(strangers(load + [x, "s_nop 0", "s_nop 0"])) == 1


def test_loads_into_lds_wait_for_their_address(tmp_path):
    lib = os.path.join(ROOT, "vit_amd", "libvtcnn_hip.so")
    if not os.path.exists(lib) or not os.path.exists(OBJDUMP):
        pytest.skip("no built library or no disassembler")
    shutil.copy(lib, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, stdout=subprocess.DEVNULL)
    found = 0
    for part in sorted(tmp_path.glob("lib.so.*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(part)], check=True, stdout=subprocess.PIPE, text=True).stdout.partition("section .text")[2]
        n, bad = too_near(text.splitlines())
        found += n
        assert not n or not strangers(text.splitlines()), (part.name, strangers(text.splitlines())[0])
        assert not bad, (part.name, len(bad), bad[0])
    assert found > 100  # the attention's kernels are in the library
