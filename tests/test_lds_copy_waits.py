"""The wait states of the copies from memory straight into LDS, read from the
built library (no GPU needed).

Such a copy takes its LDS address from m0 and part of its memory address from
scalar registers.  On gfx9 the hardware does not wait for either: one wait state
has to stand between a scalar instruction that writes m0 and the copy, five
between a vector instruction that writes a scalar register and a memory
instruction that reads it.  The compiler puts them in for its own instructions
and does not look into inline assembly, which the kernels issue these copies
from."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from tcfp_amd import _hip

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
COPY = re.compile(r"^(global_load_lds_\w+ .*|buffer_load_\w+ .* lds)$")


def _code_objects(where: Path):
    """The disassembly of every source's GPU code in the library."""
    if not OBJDUMP.exists():
        pytest.skip(f"{OBJDUMP} is not there")
    lib = where / "lib.so"
    shutil.copy(_hip.LIB_PATH, lib)  # (the tool writes beside its input)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True, cwd=where)
    for obj in sorted(where.glob("lib.so.*gfx950")):
        yield subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", obj], check=True,
                             capture_output=True, text=True).stdout


def _written(ins: str) -> set:
    """Scalar registers (numbers, or "m0") that an instruction writes, by its
    first operand."""
    op, _, rest = ins.partition(" ")
    if not op.startswith(("s_", "v_")) or op.startswith(("s_cmp", "s_waitcnt", "s_barrier")):
        return set()
    return _registers(rest.split(",")[0])


def _registers(text: str) -> set:
    found = {"m0"} if re.search(r"\bm0\b", text) else set()
    found |= {int(n) for n in re.findall(r"\bs(\d+)\b", text)}
    for lo, hi in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        found |= set(range(int(lo), int(hi) + 1))
    return found


def short_waits(text: str) -> tuple[int, list]:
    """How many copies a disassembly holds, and those whose waits are short."""
    copies, short, kernel, seen = 0, [], "?", []
    for line in text.splitlines():
        if m := re.match(r"^[0-9a-f]+ <(\S+)>:", line):
            kernel, seen = m[1], []
            continue
        ins = line.split("//")[0].strip()
        if not line.startswith("\t") or not ins:
            continue
        if COPY.match(ins):
            copies += 1
            reads, states = _registers(ins), 0
            for past in reversed(seen):
                if past.startswith(("s_branch", "s_endpgm", "s_setpc")) or states >= 5:
                    break
                wrote = _written(past)
                if "m0" in wrote and states < 1:
                    short.append((kernel, past, ins))
                if past.startswith("v_") and wrote & (reads | {"m0"}):
                    short.append((kernel, past, ins))
                states += int(past.split()[1], 0) + 1 if past.startswith("s_nop") else 1
        seen.append(ins)
        del seen[:-8]
    return copies, short


def test_the_check_itself():
    def dis(*ins):
        return "0000 <k>:\n" + "".join(f"\t{i} // 0: 0\n" for i in ins)

    copy = "global_load_lds_dwordx4 v1, s[2:3]"
    assert short_waits(dis("s_mov_b32 m0, s0", copy))[1]
    assert not short_waits(dis("s_mov_b32 m0, s0", "s_nop 0", copy))[1]
    assert not short_waits(dis("s_mov_b32 m0, s0", "v_add_u32_e32 v0, v1, v2", copy))[1]
    assert short_waits(dis("v_readfirstlane_b32 s3, v0", "s_nop 3", copy))[1]
    assert not short_waits(dis("v_readfirstlane_b32 s3, v0", "s_nop 4", copy))[1]
    assert not short_waits(dis("s_add_u32 s3, s4, s5", copy))[1]
    assert short_waits(dis("s_add_i32 m0, s1, s2", "buffer_load_ubyte v1, s[4:7], 0 offen lds"))[1]
    assert short_waits(dis(copy, "buffer_load_dword v1, s[4:7], 0 offen")) == (1, [])


@pytest.mark.parametrize("kernel", ["attend_wide_kernel", "gemm_nt_dma_kernel"])
def test_copies_into_lds_keep_their_wait_states(kernel, tmp_path):
    text = next(t for t in _code_objects(tmp_path) if kernel in t)
    copies, short = short_waits(text)
    assert copies > 0
    assert not short, (len(short), copies, short[:3])
