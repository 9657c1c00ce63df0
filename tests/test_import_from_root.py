"""`import ra_spmm` in a program whose only own entry on the path is the repository's root."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
PACKAGE = ROOT / "ra-spmm_amd" / "ra_spmm"


def run(code):
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)


@pytest.mark.parametrize("first", ["import ra_spmm", "from ra_spmm import diff_attention", "import ra_spmm.capi",
                                   "import ra_spmm.transformer as T", "from ra_spmm import _C"])
def test_the_package_itself_is_imported(first):
    r = run(f"""
import sys
sys.path[:] = [p for p in sys.path if 'ra-spmm_amd' not in p]
{first}
import importlib
import ra_spmm
assert ra_spmm is sys.modules['ra_spmm'] and ra_spmm.__name__ == 'ra_spmm'
before = ra_spmm._C
ra_spmm = importlib.reload(ra_spmm)
assert ra_spmm._C is before and callable(ra_spmm.make_attention_plan)
print(ra_spmm.__file__)
""")
    assert r.returncode == 0, r.stderr[-2000:]
    assert Path(r.stdout.strip().splitlines()[-1]) == PACKAGE / "__init__.py"


def test_a_measured_program_finds_the_operators():
    r = run("import perf.operators as o, ra_spmm; assert callable(ra_spmm.diff_attention) and len(o.listed()) >= 4")
    assert r.returncode == 0, r.stderr[-2000:]
