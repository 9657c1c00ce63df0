"""The C entries of embedding lookup, layer norm and distillation on a host without a GPU: structures as the header lays them
out, arguments refused before any launch, the names and keywords of the torch surface."""
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
OK, INVALID, UNSUPPORTED = 0, 1, 4
FAKE, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(4098)  # never read: refused first


def test_structures_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not found")
    pairs = [(capi.EmbedShape, "ra_embed_shape"), (capi.LayerNormShape, "ra_layer_norm_shape"), (capi.DistillShape, "ra_distill_shape")]
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


def embed(**kw):
    s = capi.EmbedShape(count=10, rows=20, dim=16, dtype=0, ids64=1, has_padding=0, padding=0, ld_table=16, ld_grad=16, scale=1.0)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("change,status", [
    (dict(dtype=3), INVALID), (dict(count=-1), INVALID), (dict(rows=-1), INVALID), (dict(dim=0), INVALID), (dict(dim=(1 << 20) + 1), UNSUPPORTED),
    (dict(count=(1 << 31) - (1 << 24)), UNSUPPORTED), (dict(rows=(1 << 31) - 2), UNSUPPORTED)], ids=str)
def test_embed_shapes_are_refused(change, status):
    lib, n, s = capi.load(), ctypes.c_int64(), ctypes.byref(embed(**change))
    assert lib.ra_embed(s, FAKE, FAKE, FAKE, None) == status and b"embed" in lib.ra_last_error()
    assert lib.ra_embed_workspace(s, ctypes.byref(n)) == status
    assert lib.ra_embed_backward(s, FAKE, FAKE, FAKE, FAKE, 1 << 40, None) == status


def test_embed_arguments_are_refused():
    lib, n, s = capi.load(), ctypes.c_int64(), ctypes.byref(embed())
    assert lib.ra_embed(None, FAKE, FAKE, FAKE, None) == INVALID and lib.ra_embed_workspace(s, None) == INVALID
    assert lib.ra_embed(s, None, FAKE, FAKE, None) == INVALID and lib.ra_embed(s, FAKE, None, FAKE, None) == INVALID
    assert lib.ra_embed(s, FAKE, FAKE, None, None) == INVALID
    assert lib.ra_embed(ctypes.byref(embed(ld_table=15)), FAKE, FAKE, FAKE, None) == INVALID and b"overlap" in lib.ra_last_error()
    assert lib.ra_embed_workspace(s, ctypes.byref(n)) == OK and n.value > 0
    call = lambda shape=s, ids=FAKE, grad=FAKE, to=FAKE, work=FAKE, size=n.value: lib.ra_embed_backward(  # noqa: E731
        shape, ids, grad, to, work, size, None)
    assert call(ids=None) == call(grad=None) == call(to=None) == call(work=None) == INVALID
    assert call(size=n.value - 1) == INVALID and b"workspace" in lib.ra_last_error()
    assert call(work=ODD) == INVALID and b"aligned" in lib.ra_last_error()
    assert call(shape=ctypes.byref(embed(ld_grad=15))) == INVALID
    # Nothing to do: no positions, or no table rows to write.
    assert lib.ra_embed(ctypes.byref(embed(count=0)), None, None, None, None) == OK
    assert lib.ra_embed_backward(ctypes.byref(embed(count=0, rows=0)), None, None, None, None, 0, None) == OK
    for count in (1, 100, 1 << 20, (1 << 31) - (1 << 24) - 1):  # the workspace grows with the positions, not past reason
        assert lib.ra_embed_workspace(ctypes.byref(embed(count=count)), ctypes.byref(n)) == OK
        assert 0 < n.value < 17 * count + (64 << 20)


def norm(**kw):
    s = capi.LayerNormShape(rows=10, dim=16, dtype=0, eps=1e-5, ldx=16, ldr=16)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("change,status", [
    (dict(dtype=3), INVALID), (dict(rows=-1), INVALID), (dict(dim=0), INVALID), (dict(dim=16385, ldx=16385), UNSUPPORTED),
    (dict(rows=1 << 31), UNSUPPORTED), (dict(ldx=15), INVALID)], ids=str)
def test_layer_norm_shapes_are_refused(change, status):
    lib, n, s = capi.load(), ctypes.c_int64(), ctypes.byref(norm(**change))
    assert lib.ra_layer_norm(s, FAKE, None, FAKE, FAKE, FAKE, None, FAKE, None) == status and b"layer norm" in lib.ra_last_error()
    assert lib.ra_layer_norm_workspace(s, ctypes.byref(n)) == status
    assert lib.ra_layer_norm_backward(s, *[FAKE] * 9, 1 << 40, None) == status


def test_layer_norm_arguments_are_refused():
    lib, n, s = capi.load(), ctypes.c_int64(), ctypes.byref(norm())
    call = lambda shape=s, x=FAKE, r=FAKE, y=FAKE, h=FAKE: lib.ra_layer_norm(shape, x, r, FAKE, FAKE, y, h, None, None)  # noqa: E731
    assert call(shape=None) == call(x=None) == call(y=None) == INVALID
    assert call(r=None) == call(h=None) == INVALID and b"residual" in lib.ra_last_error()
    assert call(shape=ctypes.byref(norm(ldr=15))) == INVALID and b"ldr" in lib.ra_last_error()
    assert lib.ra_layer_norm_workspace(s, None) == INVALID
    assert lib.ra_layer_norm_workspace(s, ctypes.byref(n)) == OK and n.value > 0
    back = lambda h=FAKE, stats=FAKE, g=FAKE, dx=FAKE, work=FAKE, size=n.value: lib.ra_layer_norm_backward(  # noqa: E731
        s, h, FAKE, stats, g, None, dx, FAKE, FAKE, work, size, None)
    assert back(h=None) == back(stats=None) == back(g=None) == back(dx=None) == back(work=None) == INVALID
    assert back(size=n.value - 1) == INVALID and b"workspace" in lib.ra_last_error()
    assert back(work=ODD) == INVALID and b"aligned" in lib.ra_last_error()
    assert lib.ra_layer_norm(ctypes.byref(norm(rows=0)), None, None, None, None, None, None, None, None) == OK
    assert lib.ra_layer_norm_backward(ctypes.byref(norm(rows=0)), *[None] * 9, 0, None) == OK


def distill(**kw):
    s = capi.DistillShape(rows=10, classes=50, kept=5, dtype=0, teacher_dtype=0, ids64=1, labels64=1, reduction=1, temperature=2.0, hard=0.0,
                          ld_logits=50, ld_teacher=5, ld_ids=5)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("change,status", [
    (dict(dtype=3), INVALID), (dict(teacher_dtype=-1), INVALID), (dict(rows=-1), INVALID), (dict(classes=0), INVALID), (dict(kept=-1), INVALID),
    (dict(kept=1025, ld_teacher=1025, ld_ids=1025), UNSUPPORTED), (dict(rows=1 << 31), UNSUPPORTED),
    (dict(classes=(1 << 30) + 1, ld_logits=1 << 31), UNSUPPORTED), (dict(reduction=3), INVALID), (dict(temperature=0.0), INVALID),
    (dict(temperature=float("nan")), INVALID), (dict(temperature=1001.0), INVALID), (dict(hard=-0.1), INVALID), (dict(hard=1.1), INVALID),
    (dict(hard=float("nan")), INVALID), (dict(ld_logits=49), INVALID), (dict(ld_teacher=4), INVALID), (dict(ld_ids=4), INVALID)], ids=str)
def test_distill_shapes_are_refused(change, status):
    lib, n, s = capi.load(), ctypes.c_int64(), ctypes.byref(distill(**change))
    assert lib.ra_distill_workspace(s, ctypes.byref(n)) == status and b"distill" in lib.ra_last_error()
    assert lib.ra_distill_loss(s, *[FAKE] * 9, 1 << 40, None) == status
    assert lib.ra_distill_backward(s, *[FAKE] * 7, None) == status


def test_distill_arguments_are_refused():
    lib, n, s = capi.load(), ctypes.c_int64(), ctypes.byref(distill())
    assert lib.ra_distill_workspace(s, None) == INVALID
    assert lib.ra_distill_workspace(s, ctypes.byref(n)) == OK and n.value > 0
    call = lambda shape=s, x=FAKE, t=FAKE, ids=FAKE, labels=None, loss=FAKE, work=FAKE, size=n.value: lib.ra_distill_loss(  # noqa: E731
        shape, x, t, ids, labels, None, loss, None, None, work, size, None)
    assert call(x=None) == call(t=None) == call(ids=None) == call(loss=None) == call(work=None) == INVALID
    assert call(shape=ctypes.byref(distill(hard=0.5))) == INVALID and b"labels" in lib.ra_last_error()
    assert call(size=n.value - 1) == INVALID and b"workspace" in lib.ra_last_error()
    assert call(work=ODD) == INVALID and b"aligned" in lib.ra_last_error()
    back = lambda x=FAKE, stats=FAKE, up=FAKE, grad=FAKE: lib.ra_distill_backward(  # noqa: E731
        s, x, FAKE, FAKE, None, stats, up, grad, None)
    assert back(x=None) == back(stats=None) == back(up=None) == back(grad=None) == INVALID
    rows0 = ctypes.byref(distill(rows=0, reduction=0))
    assert lib.ra_distill_loss(rows0, *[None] * 9, 0, None) == OK and lib.ra_distill_backward(rows0, *[None] * 7, None) == OK


SURFACE = {
    "embed": ["ids", "table", "scale", "padding"],
    "layer_norm": ["x", "weight", "bias", "eps", "residual"],
    "distill_loss": ["logits", "teacher", "ids", "temperature", "labels", "hard", "reduction"],
    "distill_loss_grad": ["logits", "teacher", "ids", "temperature", "labels", "hard", "reduction", "factor"],
}


def test_surface():
    for name, want in SURFACE.items():
        assert list(inspect.signature(getattr(ra_spmm, name)).parameters) == want, name


def test_host_tensors_are_refused():
    x, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64)
    for call in (lambda: ra_spmm.embed(ids, x), lambda: ra_spmm.layer_norm(x), lambda: ra_spmm.layer_norm(x, residual=x),
                 lambda: ra_spmm.distill_loss(x, x[:, :2], ids), lambda: ra_spmm.distill_loss_grad(x, x[:, :2], ids)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_arguments_that_do_not_fit_are_refused():
    x, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="shape"):
        ra_spmm.layer_norm(x, residual=x[:3])
    with pytest.raises(RuntimeError, match="axis"):
        ra_spmm.layer_norm(torch.tensor(1.0))
    with pytest.raises(RuntimeError, match="gradient"):
        ra_spmm.distill_loss(x, torch.zeros(4, 2, requires_grad=True), ids)
