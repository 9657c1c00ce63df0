"""`import ra_spmm` from the repository's root: the package lies in ra-spmm_amd/, which goes to the front of the path
(a search that still met this file first would run it again on a reload), and takes this module's place."""
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent / "ra-spmm_amd"))
del sys.modules[__name__]

import ra_spmm  # noqa: E402,F401
