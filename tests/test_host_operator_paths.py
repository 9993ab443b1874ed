"""The host side of the operators between a layer's projections, run without a GPU against the HIP stand-in of tests/hipstub/: the
forms, grids, workspaces and argument checks of sptmm_adapters_*, sptmm_heads_norm_rotate and sptmm_attention over their whole range."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG, STUB = os.path.join(ROOT, "sptmm_amd"), os.path.join(ROOT, "tests", "hipstub")


def test_every_form_is_a_launch_that_the_device_takes(tmp_path):
    import sptmm_amd

    sptmm_amd.lib()  # the built library (raises if missing)
    exe, stub = str(tmp_path / "operator_stress"), str(tmp_path / "hipstub.o")
    cc = ["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-pthread"]
    for cmd in ([*cc, "-DhipLaunchKernel=hipstub_launch", "-c", "-o", stub, os.path.join(STUB, "hipstub.cpp")],
                [*cc, "-rdynamic", "-o", exe, os.path.join(STUB, "operator_stress.cpp"), stub, "-L" + PKG, "-lsptmm", "-Wl,-rpath," + PKG]):
        r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-3000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, (r.stdout + r.stderr)[-3000:]
    one, four = re.search(r"one thread: (\d+) launches", r.stdout), re.search(r"four threads: (\d+) launches in all", r.stdout)
    assert one and four, r.stdout
    assert int(one.group(1)) > 10000 and int(four.group(1)) == 5 * int(one.group(1))
