"""The developer build (sod100k_amd/csrc/dev_build.sh) compiles what the product build compiles."""
import os
import shutil
import subprocess

import pytest

from sod100k_amd import _native as N


def test_dev_build_names_every_source(tmp_path):
    """Run on a copy of the folder with a compiler that writes down what it is asked for: every source, every flag of the product build
    and a refusal of undefined symbols; the copy gets the library only where the compiler made one."""
    if N.hipcc_path() is None:
        pytest.skip("hipcc not found")
    pkg = tmp_path / "sod100k_amd"
    os.makedirs(pkg / "csrc")
    for f in ("__init__.py", "_native.py"):
        shutil.copy(os.path.join(N.HERE, f), pkg / f)
    for f in os.listdir(N.CSRC):
        if f.endswith((".hip", ".h", ".inl", ".sh")):
            shutil.copy(os.path.join(N.CSRC, f), pkg / "csrc" / f)
    shutil.copytree(os.path.join(os.path.dirname(N.HERE), "include"), tmp_path / "include")
    (tmp_path / "bin").mkdir()
    fake = tmp_path / "bin" / "hipcc"
    fake.write_text('#!/bin/bash\necho "$@" >> "$ASKED"\n[ -n "$BROKEN" ] && { echo "error: undefined"; exit 1; }\n'
                    'while [ $# -gt 0 ]; do [ "$1" = -o ] && echo made > "$2"; shift; done\n')
    fake.chmod(0o755)
    asked, lib = tmp_path / "asked", pkg / "csrc" / "libcsnet_hip.so"
    env = dict(os.environ, PATH=f"{tmp_path}/bin:{os.environ['PATH']}", OUT=str(tmp_path / "out"), ASKED=str(asked))
    lib.write_text("before")
    r = subprocess.run(["bash", str(pkg / "csrc" / "dev_build.sh")], env=dict(env, BROKEN="1"), stdout=subprocess.DEVNULL)
    assert r.returncode != 0 and lib.read_text() == "before"
    asked.write_text("")
    subprocess.run(["bash", str(pkg / "csrc" / "dev_build.sh")], env=env, check=True, stdout=subprocess.DEVNULL)
    calls = [line.split() for line in asked.read_text().splitlines()]
    compiled = [c for c in calls if "-c" in c and any(w.endswith(".hip") for w in c)]
    assert sorted(os.path.basename(w) for c in compiled for w in c if w.endswith(".hip")) == sorted(N.SOURCES)
    assert all(set(N.HIPCC_FLAGS) <= set(c) for c in compiled)
    link, = [c for c in calls if "-shared" in c]
    assert "-Wl,--no-undefined" in link
    assert sorted(os.path.basename(w) for w in link if w.endswith(".o")) == sorted([s[:-4] + ".o" for s in N.SOURCES] + ["csn_build_id.o"])
    assert lib.read_text() == "made\n"
