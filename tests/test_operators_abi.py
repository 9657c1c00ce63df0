"""The C entries of the attention, head-norm and 8-bit operators on a host without a GPU: structures as the header lays
them out, arguments refused before any launch, the names and keywords of the torch surface."""
import ctypes
import inspect
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import ra_spmm
from ra_spmm import capi

HEADER = Path(__file__).resolve().parents[1] / "include" / "ra_spmm.h"
OK, INVALID, UNSUPPORTED, INACTIVE = 0, 1, 4, 5


def test_structures_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not found")
    pairs = [(capi.AttnShape, "ra_attn_shape"), (capi.AttnInfo, "ra_attn_info"), (capi.NormShape, "ra_norm_shape")]
    lines = []
    for cls, name in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "ra_spmm.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-std=c99", "-I", str(HEADER.parent), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls, _ in pairs:
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def attn(**kw):
    s = capi.AttnShape(q_heads=4, kv_heads=2, head_dim=16, value_dim=32, dtype=0, scale=0.25, ldq=128, ldk=64, ldv=64)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("change,status", [
    (dict(dtype=7), INVALID), (dict(q_heads=3), INVALID), (dict(kv_heads=0), INVALID), (dict(head_dim=0), INVALID),
    (dict(head_dim=129), UNSUPPORTED), (dict(value_dim=257), UNSUPPORTED), (dict(ldq=1 << 30), UNSUPPORTED),
    (dict(ldk=63), INVALID), (dict(ldv=10), INVALID), (dict(ldq=100), INVALID)], ids=str)
def test_attention_shapes_are_refused(change, status):
    lib = capi.load()
    fake = ctypes.c_void_p(4096)  # never read: the shape is refused first
    got = lib.ra_attn_csr(fake, fake, 3, 5, 10, ctypes.byref(attn(**change)), fake, fake, fake, fake, None, fake, fake, 1 << 30, None)
    assert got == status and b"attention" in lib.ra_last_error()


def test_attention_arguments_are_refused():
    lib = capi.load()
    fake, odd, n = ctypes.c_void_p(4096), ctypes.c_void_p(4098), ctypes.c_int64()
    assert lib.ra_attn_csr_workspace(None, 1, 1, ctypes.byref(n)) == INVALID
    assert lib.ra_attn_csr_workspace(ctypes.byref(attn()), 4, 4 * 6000, ctypes.byref(n)) == OK and n.value > 0
    call = lambda **k: lib.ra_attn_csr(*[k.get(x, d) for x, d in (  # noqa: E731
        ("rowptr", fake), ("colind", fake), ("M", 4), ("K", 5), ("nnz", 24000), ("shape", ctypes.byref(attn())), ("q", fake),
        ("k", fake), ("v", fake), ("lam", fake), ("bias", None), ("out", fake), ("work", fake), ("bytes", n.value), ("st", None))])
    assert call(bytes=n.value - 1) == INVALID and b"workspace" in lib.ra_last_error()
    assert call(work=odd) == INVALID
    assert call(q=None) == INVALID and call(lam=None) == INVALID and call(M=-1) == INVALID and call(nnz=1 << 40) == INVALID
    assert call(out=odd) == INVALID and b"aligned" in lib.ra_last_error()
    assert call(M=0, nnz=0) == OK  # nothing to do
    # a wave for every row at least: a launch holds fewer than 2^32 threads
    assert call(M=1 << 26, nnz=0) == UNSUPPORTED and b"too many" in lib.ra_last_error()
    p = ctypes.c_void_p()
    assert lib.ra_attn_plan_create(None, None, 3, 3, 5, 1, None, ctypes.byref(p)) == INVALID
    assert lib.ra_attn_plan_create(fake, fake, 3, 3, 1 << 32, 1, None, ctypes.byref(p)) == UNSUPPORTED
    assert lib.ra_attn_plan_run(None, ctypes.byref(attn()), *[None] * 8) == INVALID
    assert lib.ra_attn_plan_get_info(None, None) == INVALID
    lib.ra_attn_plan_destroy(None)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=9), INVALID), (dict(layout=2), INVALID), (dict(rot_dim=3), INVALID), (dict(rot_dim=18), INVALID),
    (dict(head_dim=257), UNSUPPORTED), (dict(q_heads=0, k_heads=0), INVALID), (dict(ldq=10), INVALID), (dict(rows=-1), INVALID),
    (dict(rows=1 << 30, ldq=64), UNSUPPORTED)], ids=str)
def test_norm_shapes_are_refused(change, status):
    s = capi.NormShape(rows=3, q_heads=4, k_heads=2, head_dim=16, rot_dim=8, positions=10, layout=0, dtype=0, eps=1e-6,
                       ldq=64, ldk=32)
    for k, v in change.items():
        setattr(s, k, v)
    n = ctypes.c_int64()
    assert capi.load().ra_head_norm_workspace(ctypes.byref(s), ctypes.byref(n)) == status


def test_pack_arguments_are_refused():
    lib = capi.load()
    fake, odd, n = ctypes.c_void_p(4096), ctypes.c_void_p(4097), ctypes.c_int64()
    assert lib.ra_pack8(fake, 4, 0, 8, 0, fake, fake, None) == INVALID
    assert lib.ra_pack8(fake, 4, 8, 7, 0, fake, fake, None) == INVALID
    assert lib.ra_pack8(fake, 4, 8, 8, 3, fake, fake, None) == INVALID
    assert lib.ra_pack8(fake, 4, 8, 8, 0, odd, fake, None) == INVALID
    assert lib.ra_pack8(None, 4, 8, 8, 0, fake, fake, None) == INVALID
    assert lib.ra_relu_pack8(fake, 4, 8, 8, 0, None, fake, fake, None) == INVALID
    assert lib.ra_unpack8(fake, fake, -1, 8, 1, 0, fake, None) == INVALID
    assert lib.ra_weight_grad8_workspace(-1, 8, 8, ctypes.byref(n)) == INVALID
    assert lib.ra_weight_grad8_workspace(1 << 20, 47, 256, ctypes.byref(n)) == OK and n.value > 0
    assert lib.ra_weight_grad8(fake, fake, fake, 1 << 20, 47, 256, 47, 0, 0, fake, fake, n.value - 1, None) == INVALID
    assert lib.ra_weight_grad8(fake, fake, fake, 1 << 20, 47, 256, 46, 0, 0, fake, fake, n.value, None) == INVALID
    assert lib.ra_pack8(None, 0, 8, 8, 0, None, None, None) == OK  # no rows


SURFACE = {
    "make_attention_plan": ["rowptr", "colind", "M", "K", "backward"],
    "run_attention_plan": ["plan", "q", "k", "v", "lam", "scale", "bias"],
    "run_attention_plan_train": ["plan", "q", "k", "v", "lam", "scale", "bias"],
    "run_attention_plan_backward": ["plan", "q", "k", "v", "lam", "stats", "grad_out", "scale", "bias"],
    "diff_attention_csr": ["rowptr", "colind", "q", "k", "v", "lam", "scale", "bias"],
    "diff_attention": ["plan", "q", "k", "v", "lam", "scale", "bias"],
    "head_norm_rotate": ["q", "k", "wq", "wk", "table", "positions", "eps", "layout"],
    "rotation_table": ["positions", "rot_dim", "base", "scaling", "device"],
    "pack8": ["x"], "relu_pack8": ["x"], "unpack8": ["p", "dtype"], "relu_grad8": ["grad", "p"], "weight_grad8": ["grad", "p"],
    "relu8": ["x"], "linear8": ["x", "weight", "packed"],
}


def test_surface():
    for name, want in SURFACE.items():
        fn = getattr(ra_spmm, name)
        try:
            got = list(inspect.signature(fn).parameters)
        except (TypeError, ValueError):
            first = fn.__doc__.splitlines()[0]
            got = [a.split(":")[0].strip() for a in first[first.index("(") + 1:first.rindex(")")].split(",") if ":" in a]
        assert got == want, (name, got)


def test_host_tensors_are_refused():
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ra_spmm.pack8(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        ra_spmm.head_norm_rotate(x.view(4, 1, 8), None, torch.ones(8), None)
