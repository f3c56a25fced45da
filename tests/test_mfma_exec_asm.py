"""Matrix instructions run whatever EXEC says.  A wavefront that should not run one has to branch around it: behind an EXEC narrowed by a condition
that the compiler took for a lane's, without a branch, it would multiply what its registers happen to hold.  The engine's own gfx950 code is
disassembled (no GPU needed) and every matrix instruction looked at."""
import os
import re
import shutil
import subprocess

import pytest

from phc_gnn_amd import build

OBJDUMP = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")


def unguarded(lines):
    """(matrix instructions, {function: how many stand behind a narrowed EXEC that no branch has looked at})."""
    total, bad, fn, narrowed = 0, {}, None, False
    for line in lines:
        head = re.match(r"^(?:[0-9a-f]+ )?<?(\w+)>?:", line)
        if head and not line.startswith("."):
            fn, narrowed = head.group(1), False
            continue
        text = line.split("//")[0].split(";")[0].strip()
        op = text.split(" ")[0]
        if op in ("s_cbranch_execz", "s_branch", "s_endpgm", "s_setpc_b64"):
            narrowed = False                                      # (behind execz some lane is active; behind the others nothing falls through)
        elif "saveexec" in op or re.match(r"s_(and|andn2|xor)\w*_b64 exec,", text):
            narrowed = True
        elif re.match(r"s_(or|mov)_b64 exec,", text):
            narrowed = False
        elif op.startswith("v_mfma"):
            total += 1
            if narrowed:
                bad[fn] = bad.get(fn, 0) + 1
    return total, bad


def test_the_reader_sees_what_it_looks_for():
    guarded = ["f:", "s_and_saveexec_b64 s[0:1], vcc", "s_cbranch_execz .LBB0_1", "v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]",
               ".LBB0_1:", "s_or_b64 exec, exec, s[0:1]", "v_mfma_f32_16x16x32_bf16 a[0:3], v[0:3], v[4:7], a[0:3]"]
    assert unguarded(guarded) == (2, {})
    assert unguarded(guarded[:2] + guarded[3:]) == (2, {"f": 1})
    assert unguarded(guarded[:2] + [".LBB0_7:"] + guarded[3:]) == (2, {"f": 1})


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")
def test_no_matrix_instruction_behind_a_narrowed_exec(tmp_path):
    if not os.path.exists(build.LIB_PATH):
        build.build()
    lib = shutil.copy(build.LIB_PATH, tmp_path / "engine.so")
    subprocess.run([OBJDUMP, "--offloading", str(lib)], check=True, cwd=tmp_path, stdout=subprocess.DEVNULL)
    objects = sorted(p for p in tmp_path.iterdir() if build.ARCH in p.name)
    assert objects
    total = 0
    for obj in objects:
        with subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", str(obj)], stdout=subprocess.PIPE, text=True) as p:
            n, bad = unguarded(p.stdout)
        assert p.returncode == 0
        total += n
        assert not bad, bad
    assert total > 10000                                          # (the engine's products)
