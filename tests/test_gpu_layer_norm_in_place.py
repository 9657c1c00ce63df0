"""Layer norm through the C entries with outputs in the place of inputs: the same bits as elsewhere, at rows of a part of a
wave, of a wave and of a workgroup, with whole packets and without."""
import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

from ra_spmm import capi  # noqa: E402

CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
DIMS = [3, 16, 47, 256, 1000, 1030, 1100, 4099, 8191, 8192, 16383]


def p(t):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def forward(dtype, x, r, w, b, y, total, stats):
    s = capi.LayerNormShape(rows=x.size(0), dim=x.size(1), dtype=CODES[dtype], eps=1e-5, ldx=x.size(1), ldr=x.size(1))
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert capi.load().ra_layer_norm(ctypes.byref(s), p(x), p(r), p(w), p(b), p(y), p(total), p(stats), stream) == 0


def backward(dtype, h, w, stats, gy, gs, dx, dw, db):
    s = capi.LayerNormShape(rows=h.size(0), dim=h.size(1), dtype=CODES[dtype], eps=1e-5, ldx=h.size(1), ldr=0)
    n = ctypes.c_int64()
    assert capi.load().ra_layer_norm_workspace(ctypes.byref(s), ctypes.byref(n)) == 0
    work = torch.empty(n.value, dtype=torch.uint8, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert capi.load().ra_layer_norm_backward(ctypes.byref(s), p(h), p(w), p(stats), p(gy), p(gs), p(dx), p(dw), p(db), p(work), n, stream) == 0


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("dtype", list(CODES), ids=str)
def test_in_place(D, dtype):
    M = 700
    gen = torch.Generator("cuda").manual_seed(D)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, res, w, b = r(M, D).to(dtype), r(M, D).to(dtype), r(D), r(D)
    new = lambda t: torch.full_like(t, float("nan"))  # noqa: E731
    stats = r(M, 2)
    y, total = new(x), new(x)
    forward(dtype, x, res, w, b, y, total, stats)
    assert torch.equal(total, (x.float() + res.float()).to(dtype))
    for a, c in (("y", "x"), ("y", "res"), ("sum", "x"), ("sum", "res"), ("both", "x"), ("both", "res")):
        xi, ri, yi, si, st = x.clone(), res.clone(), new(x), new(x), new(stats)
        at, other = (xi, ri) if c == "x" else (ri, xi)
        if a == "y":
            yi = at
        elif a == "sum":
            si = at
        else:
            yi, si = at, other
        forward(dtype, xi, ri, w, b, yi, si, st)
        assert torch.equal(yi, y) and torch.equal(si, total) and torch.equal(st, stats), (a, c)
    alone, xi = new(x), x.clone()
    forward(dtype, x, None, w, b, alone, None, None)
    forward(dtype, xi, None, w, b, xi, None, None)
    assert torch.equal(xi, alone)

    gy, gs = r(M, D).to(dtype), r(M, D).to(dtype)
    dx, dw, db = new(x), new(w), new(w)
    backward(dtype, total, w, stats, gy, gs, dx, dw, db)
    for at in ("h", "gy", "gs"):
        t = {"h": total.clone(), "gy": gy.clone(), "gs": gs.clone()}
        dwi, dbi = new(w), new(w)
        backward(dtype, t["h"], w, stats, t["gy"], t["gs"], t[at], dwi, dbi)
        assert torch.equal(t[at], dx) and torch.equal(dwi, dw) and torch.equal(dbi, db), at
