"""The compiled kernels of pcl_paged_tree_attention: their registers."""
import os
import re
import subprocess

import pytest


def resources(source):
    """{kernel: (scratch bytes a lane, vector registers spilled)} of a source."""
    import importlib.util
    import tempfile
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "power-cpu-llm_amd")
    spec = importlib.util.spec_from_file_location("hip_build", os.path.join(root, "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    with tempfile.TemporaryDirectory() as tmp:
        res = subprocess.run(
            [build.HIPCC] + [f for f in build.FLAGS if f != "-shared"] +
            ["--cuda-device-only", "-c", "-Rpass-analysis=kernel-resource-usage",
             os.path.join(root, "csrc", source), "-o", os.path.join(tmp, "k.o")],
            capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-2000:]
    found = {}
    for line in res.stderr.splitlines():
        m = re.search(r"Function Name: (\S+)", line)
        if m:
            words = found.setdefault(m.group(1), {})
        m = re.search(r"(ScratchSize \[bytes/lane\]|VGPRs Spill): (\d+)", line)
        if m:
            words[m.group(1)[0]] = int(m.group(2))
    return {name: (w["S"], w["V"]) for name, w in found.items()}


def test_no_kernel_of_few_rows_keeps_its_words_in_memory():
    from concurrent.futures import ThreadPoolExecutor
    if not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("hipcc absent")
    with ThreadPoolExecutor(4) as pool:
        found = dict(x for r in pool.map(resources, ["paged_tree_d%d.hip" % dk for dk in
                                                     (512, 64, 128, 256)]) for x in r.items())
    kernels = {n: w for n, w in found.items() if "paged_tree_kernel" in n}
    assert len(kernels) == 48
    assert {n: w for n, w in kernels.items() if w != (0, 0)} == {}
