"""The C entries of embedding lookup, layer norm and distillation refuse outputs and workspaces that share memory with an input
or with each other, before any launch: a host without a GPU sees it.  Nothing here is read, every call is refused."""
import ctypes

import pytest

from ra_spmm import capi
from test_model_operators_abi import INVALID, distill, embed, norm

MB = 1 << 20


def refused(call, places, moved, onto, by, names):
    """The call with the tensor `moved` set `by` bytes from `onto`, all others 1 MB apart."""
    at = {name: (i + 1) * MB for i, name in enumerate(places)}
    at[moved] = at[onto] + by
    assert call(*[ctypes.c_void_p(at[name]) for name in places]) == INVALID
    error = capi.load().ra_last_error().decode()
    assert "overlaps" in error and all(n in error for n in names), error


@pytest.mark.parametrize("onto,name,last", [("ids", "ids", 79), ("table", "the table", 1279)])
def test_embed(onto, name, last):
    places, lib, s = ("ids", "table", "out"), capi.load(), ctypes.byref(embed())
    for by in (0, last, -639):  # out: 10 x 16 floats
        refused(lambda *t: lib.ra_embed(s, *t, None), places, "out", onto, by, ("out", name))


@pytest.mark.parametrize("moved,onto,names", [
    ("dtable", "grad", ("gradient", "grad")), ("dtable", "ids", ("gradient", "ids")), ("work", "grad", ("workspace", "grad")),
    ("work", "ids", ("workspace", "ids")), ("work", "dtable", ("workspace", "gradient"))], ids=str)
def test_embed_backward(moved, onto, names):
    places, lib, s = ("ids", "grad", "dtable", "work"), capi.load(), ctypes.byref(embed())
    for by in (0, 64, -64):
        refused(lambda i, g, t, w: lib.ra_embed_backward(s, i, g, t, w, MB // 2, None), places, moved, onto, by, names)


NORM = ("x", "residual", "weight", "bias", "y", "sum", "stats")


@pytest.mark.parametrize("moved,onto,by", [
    ("y", "weight", 0), ("sum", "bias", 60), ("y", "x", 4), ("y", "x", -636), ("sum", "x", 64), ("sum", "residual", -64), ("y", "residual", 639),
    ("y", "sum", 0), ("stats", "x", 0), ("stats", "residual", 0), ("stats", "weight", -72), ("stats", "y", 632), ("stats", "sum", 0)], ids=str)
def test_layer_norm(moved, onto, by):
    lib, s = capi.load(), ctypes.byref(norm())
    refused(lambda *t: lib.ra_layer_norm(s, *t, None), NORM, moved, onto, by, (moved, onto))


@pytest.mark.parametrize("moved,onto,change", [("y", "x", dict(ldx=17)), ("sum", "x", dict(ldx=17)), ("y", "residual", dict(ldr=18)),
                                               ("sum", "residual", dict(ldr=18))], ids=str)
def test_layer_norm_in_place_of_strided_rows(moved, onto, change):
    lib, s = capi.load(), ctypes.byref(norm(**change))
    refused(lambda *t: lib.ra_layer_norm(s, *t, None), NORM, moved, onto, 0, (moved, onto))


BACK = ("h", "weight", "stats", "grad_y", "grad_sum", "dx", "dweight", "dbias", "workspace")


@pytest.mark.parametrize("moved,onto,by,change", [
    ("dx", "weight", 0, {}), ("dx", "stats", 72, {}), ("dx", "h", 4, {}), ("dx", "h", 0, dict(ldx=17)), ("dx", "grad_y", -4, {}),
    ("dx", "grad_sum", 636, {}), ("dweight", "h", 0, {}), ("dweight", "weight", 0, {}), ("dbias", "dweight", 32, {}), ("dbias", "dx", 0, {}),
    ("dbias", "grad_y", 0, {}), ("workspace", "h", 0, {}), ("workspace", "grad_sum", 0, {}), ("workspace", "dx", 0, {}),
    ("workspace", "dbias", -64, {}), ("workspace", "stats", 64, {})], ids=str)
def test_layer_norm_backward(moved, onto, by, change):
    lib, s = capi.load(), ctypes.byref(norm(**change))
    refused(lambda *t: lib.ra_layer_norm_backward(s, *t, MB // 2, None), BACK, moved, onto, by, (moved, onto))


@pytest.mark.parametrize("rows,classes", [(10, 50), (40_000, 40), (10, 3000), (10, 100_000)])
@pytest.mark.parametrize("moved,onto,names", [
    ("grad", "logits", ("gradient", "logits")), ("grad", "teacher", ("gradient", "teacher")), ("grad", "ids", ("gradient", "ids")),
    ("grad", "labels", ("gradient", "labels")), ("grad", "factor", ("gradient", "factor")), ("loss", "logits", ("loss", "logits")),
    ("stats", "logits", ("stats", "logits")), ("work", "logits", ("workspace", "logits")), ("work", "grad", ("workspace", "gradient")),
    ("stats", "grad", ("gradient", "stats")), ("loss", "grad", ("gradient", "loss"))], ids=str)
def test_distill(rows, classes, moved, onto, names):
    lib, n = capi.load(), ctypes.c_int64()
    s = ctypes.byref(distill(rows=rows, classes=classes, ld_logits=classes, hard=0.5))
    assert lib.ra_distill_workspace(s, ctypes.byref(n)) == 0
    places = {p: (i + 1) << 30 for i, p in enumerate(("logits", "teacher", "ids", "labels", "factor", "loss", "stats", "grad", "work"))}
    for by in (0, 16):
        if by and onto == "factor":
            continue  # one float
        at = dict(places)
        at[moved] = at[onto] + by
        assert lib.ra_distill_loss(s, *[ctypes.c_void_p(a) for a in at.values()], n.value, None) == INVALID
        error = lib.ra_last_error().decode()
        assert "overlaps" in error and all(w in error for w in names), error


@pytest.mark.parametrize("onto", ["logits", "teacher", "ids", "labels", "stats", "grad_loss"])
def test_distill_backward(onto):
    lib, s = capi.load(), ctypes.byref(distill(hard=0.5))
    refused(lambda *t: lib.ra_distill_backward(s, *t, None), ("logits", "teacher", "ids", "labels", "stats", "grad_loss", "grad"), "grad", onto, 0,
            ("gradient", onto))
