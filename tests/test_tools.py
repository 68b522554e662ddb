"""The build scripts under tools/, with a stand-in for the compiler."""
import glob
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STAND_IN = """#!/bin/bash
echo "$*" >> "$CALLS"
for ((i = 1; i <= $#; i++)); do [ "${!i}" = -o ] && j=$((i + 1)) && out="${!j}"; done
case " $* " in *" -shared "*) gcc -shared -o "$out" -x c /dev/null;; *) : > "$out";; esac
"""


@pytest.mark.skipif(not os.path.isdir(os.path.join(ROOT, ".git")), reason="needs the history")
def test_a_build_of_another_commit_compiles_all_its_sources(tmp_path):
    cc, calls = tmp_path / "cc", tmp_path / "calls"
    cc.write_text(STAND_IN)
    cc.chmod(0o755)
    name = "of_test_%d" % os.getpid()
    try:
        subprocess.run(["bash", "tools/build_ref_variant.sh", name, "HEAD", "-DSOME=1"], cwd=ROOT, check=True,
                       stdout=subprocess.DEVNULL, env=dict(os.environ, HIPCC=str(cc), CALLS=str(calls)))
        assert os.path.exists(os.path.join(ROOT, "build", "ab", name, "libpss.so"))
    finally:
        shutil.rmtree(os.path.join(ROOT, "build", "ab", name), ignore_errors=True)
    lines = calls.read_text().splitlines()
    compiled = {line.split()[-1] for line in lines if " -c " in line}
    tracked = subprocess.run(["git", "ls-tree", "--name-only", "HEAD", "partiallyshuffledistributedsampler_amd/csrc/"],
                             cwd=ROOT, check=True, capture_output=True, text=True).stdout.split()
    sources = {os.path.basename(f) for f in tracked if f.endswith((".hip", ".cpp"))} - {"pss_torch.cpp"}
    assert compiled == sources
    assert all("-DSOME=1" in line and "-packed-fp32-ops" in line for line in lines if " -c " in line)


def test_every_list_of_sources_is_whole():
    csrc = os.path.join(ROOT, "partiallyshuffledistributedsampler_amd", "csrc")
    sources = {os.path.basename(f) for e in ("hip", "cpp") for f in glob.glob(os.path.join(csrc, "*." + e))}
    for path in ("tools/build_variant.sh", "tools/sanitize/Makefile"):
        text = open(os.path.join(ROOT, path)).read().split()
        assert sources - {"pss_torch.cpp"} <= {w.rstrip(";") for w in text}, path
