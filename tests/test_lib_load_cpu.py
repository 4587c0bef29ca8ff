"""CPU: libraries that were built before an entry point was added, or for another ABI version."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OLD = 'extern "C" int spn_abi_version() { return VERSION; }\nextern "C" int spn_tuning_count() { return 0; }\n' \
      'extern "C" const char* spn_last_error() { return "nothing"; }\nextern "C" int spn_known(int x) { return x; }\n'


def _run(tmp_path, version, program):
    src, so = tmp_path / "old.cpp", tmp_path / "old.so"
    src.write_text(OLD.replace("VERSION", str(version)))
    subprocess.run([shutil.which("g++") or "c++", "-shared", "-fPIC", "-o", str(so), str(src)], check=True)
    r = subprocess.run([sys.executable, "-c", "from scoreperformer_amd import lib\nfrom scoreperformer_amd.lib import SpnError\n" + program], cwd=ROOT,
                       env={**os.environ, "SPN_LIB": str(so)}, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return r.stdout


def test_a_library_without_the_newer_entry_points_loads_and_says_what_is_missing(tmp_path):
    out = _run(tmp_path, 10, """
h = lib.load()
assert h.spn_known(0) == 0 and lib.load() is h
lib.call("spn_known", 0)
for use in (lambda: lib.call("spn_paged_plan"), lambda: h.spn_paged_attn_workspace_bytes(1, 1, 1, 1, 16, 1)):
    try:
        use()
    except SpnError as e:
        print(e)
assert not hasattr(h, "spn_paged_attn")
""")
    lines = out.splitlines()
    assert len(lines) == 2 and "spn_paged_plan" in lines[0] and "spn_paged_attn_workspace_bytes" in lines[1] and all("rebuild it" in x for x in lines)


@pytest.mark.parametrize("version", [9, 11])
def test_a_library_of_another_abi_version_is_refused_by_its_version(tmp_path, version):
    out = _run(tmp_path, version, """
for _ in range(2):
    try:
        lib.load()
    except SpnError as e:
        print(e)
""")
    assert out.count(f"has ABI version {version}") == 2 and out.count("rebuild it") == 2
