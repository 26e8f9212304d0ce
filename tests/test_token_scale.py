"""Scales that fp32 does not hold: elements are multiplied by one fp32 factor, scale / (1 - p)."""

import ctypes

import pytest
import torch

from flashoptim_jax_b200 import _lib

TOO_MUCH = [(1e39, 0.0), (-4e38, 0.0), (3e38, 0.5), (1e308, 0.999), (float("inf"), 0.0), (float("nan"), 0.5), (float("inf"), 1.0)]
TOO_LITTLE = [(1e-46, 0.0), (-1e-39, 0.0), (2.0**-127, 0.25), (5e-324, 0.0)]
# the factor is 0 where everything is dropped
FINE = [(3.4e38, 0.0), (-3.4e38, 0.0), (2.0**-126, 0.0), (-(2.0**-127), 0.5), (0.0, 0.0), (-0.0, 0.5), (1e30, 1.0), (1e-300, 1.0)]


def _drop(p):
    return _lib.FoDropout(p=p, seed=1, offset=2)


def _status(scale, p, empty):
    """Of both calls; the ones that are not refused have nothing to do."""
    lib = _lib.lib()
    n = 0 if empty else 1
    e = _lib.FoEmbed(struct_size=ctypes.sizeof(_lib.FoEmbed), table_dtype=1, out_dtype=1, ids_bits=64, table=64, ids=64, out=64, n_tokens=n, rows=8, dim=8, row_stride=8,
                     scale=scale, dropout=_drop(p))
    g = _lib.FoEmbedGrad(struct_size=ctypes.sizeof(_lib.FoEmbedGrad), dy_dtype=1, out_dtype=1, ids_bits=64, accumulate=1, dy=64, ids=64, out=64, n_tokens=n, rows=8, dim=8,
                         dy_stride=8, scale=scale, dropout=_drop(p))
    out = []
    for call, d in ((lib.fo_embed, e), (lib.fo_embed_grad, g)):
        out.append((call(ctypes.byref(d), None), lib.fo_last_error()))
    return out


@pytest.mark.parametrize("scale,p", TOO_MUCH + TOO_LITTLE)
@pytest.mark.parametrize("empty", [True, False])
def test_scales_that_are_no_fp32_factor_are_refused(scale, p, empty):
    for status, text in _status(scale, p, empty):
        assert status == 1 and b"scale" in text


@pytest.mark.parametrize("scale,p", FINE)
def test_scales_that_are(scale, p):
    assert [status for status, _ in _status(scale, p, True)] == [0, 0]


@pytest.mark.gpu
def test_from_python():
    import flashoptim_jax_b200 as fo

    table, ids, dy = torch.ones((5, 8), device="cuda"), torch.arange(5, device="cuda"), torch.ones((5, 8), device="cuda")
    for scale, p in TOO_MUCH + TOO_LITTLE:
        for dtype in (None, torch.float32):  # through the host extension, and past it
            with pytest.raises(ValueError, match="scale"):
                fo.embed(table, ids, scale=scale, p=p, dtype=dtype)
            with pytest.raises(ValueError, match="scale"):
                fo.embed_grad(dy, ids, 5, scale=scale, p=p, dtype=dtype)
    for scale in (3.4e38, 2.0**-126, -(2.0**-126)):
        want = torch.full((5, 8), scale, dtype=torch.float32, device="cuda")
        assert torch.equal(fo.embed(table, ids, scale=scale), want)
        assert torch.equal(fo.embed_grad(dy, ids, 5, scale=scale), want)
        assert torch.equal(fo.embed_grad(dy.repeat(20, 1)[:96] * 0.0 + 1.0, torch.arange(96, device="cuda"), 96, scale=scale)[:5], want)
