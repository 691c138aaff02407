"""Static checks of the product HIP kernels' ISA (CPU; hipcc cross-compiles gfx950 here).

The bf16 noise-MLP kernel (csrc/noise_mlp.hip solo::) reads its weight fragments and biases with
inline-asm ds_reads and counted lgkmcnt waits.  The compiler sees an asm read's output as written
at once, so if it ever reused, copied or spilled such a register before the wait that covers it,
data landing later would corrupt the register (a round-5 development build clobbered a 64-bit
address that way and faulted the GPU).  tools/asm_hazard.py scans the built ISA for any use of a
register with an LDS read in flight."""
import os
import shutil
import subprocess
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("/opt/rocm/bin/hipcc") is None, reason="hipcc not installed")
@pytest.mark.parametrize("kernel", ["noise_mlp_solo_kernel"])
def test_no_register_use_while_an_lds_read_is_in_flight(kernel):
    r = subprocess.run([sys.executable, os.path.join(REPO, "tools", "asm_hazard.py"), kernel],
                       capture_output=True, text=True, timeout=600)
    print(r.stdout)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "0 hazard(s)" in r.stdout


@pytest.mark.skipif(shutil.which("/opt/rocm/bin/hipcc") is None, reason="hipcc not installed")
def test_noise_mlp_as_the_makefile_builds_it(tmp_path):
    """The same with the library's own flags, and no scratch memory: a launch that needs it waits for its queue's share,
    so that a kernel that polls a flag could keep the launch in front of that flag from starting."""
    csrc = os.path.join(REPO, "pointcloud_style_transfer_amd", "csrc")
    line = subprocess.run(["make", "-n", "-B", "-C", csrc, "build/noise_mlp.o"], capture_output=True, text=True, check=True).stdout
    cmd = next(ln for ln in line.splitlines() if " -c noise_mlp.hip " in ln).split()
    assert "-packed-fp32-ops" in cmd
    asm = tmp_path / "noise_mlp.s"
    cmd = cmd[:cmd.index("-c")] + ["--cuda-device-only", "-S", "noise_mlp.hip", "-o", str(asm)]
    subprocess.run(cmd, check=True, capture_output=True, cwd=csrc)
    text = asm.read_text()
    for part in text.split("; ScratchSize: ")[1:]:
        name = text[:text.index(part)].rsplit(".globl", 1)[-1].split()[0]
        assert "solo_kernel" not in name or part.split()[0] == "0", name
    assert "noise_mlp_solo_kernel" in text
    flags = cmd[1:cmd.index("--cuda-device-only")]
    r = subprocess.run([sys.executable, os.path.join(REPO, "tools", "asm_hazard.py"), "noise_mlp_solo_kernel",
                        *[f for f in flags if not f.startswith(("-I", "-O", "-W", "--offload", "-std"))]],
                       capture_output=True, text=True, timeout=600)
    assert r.returncode == 0 and "0 hazard(s)" in r.stdout, r.stdout + r.stderr
