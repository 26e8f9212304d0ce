"""Embedding and dropout without a GPU: the oracle's generator against published vectors, refusals of the library and of the package."""

import ctypes

import numpy as np
import pytest
import torch

import flashoptim_jax_b200 as fo
from flashoptim_jax_b200 import _lib, embedding
from tests import token_oracle as T


@pytest.mark.parametrize("counter,key,want", [
    ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_the_oracles_generator_gives_the_published_answers(counter, key, want):
    assert tuple(int(x) for x in T.philox4x32(counter, key)) == want


def test_the_share_of_dropped_elements_is_p():
    for p in (0.1, 0.5, 0.9):
        n = 1 << 18
        dropped = n - int(T.keep(n, p, 3, 4).sum())
        assert abs(dropped - n * p) < 6 * np.sqrt(n * p * (1 - p))  # six standard deviations of a binomial
    assert T.keep(1000, 0.0, 1, 2).all() and not T.keep(1000, 1.0, 1, 2).any()
    assert not np.array_equal(T.keep(1000, 0.5, 1, 2), T.keep(1000, 0.5, 1, 3))
    assert not np.array_equal(T.keep(1000, 0.5, 1, 2), T.keep(1000, 0.5, 2, 2))


def test_struct_sizes_match_the_header_layout():
    assert ctypes.sizeof(_lib.FoDropout) == 40
    assert ctypes.sizeof(_lib.FoEmbed) == 144
    assert ctypes.sizeof(_lib.FoEmbedGrad) == 144


def _embed_desc(**more):
    d = _lib.FoEmbed(struct_size=ctypes.sizeof(_lib.FoEmbed), table_dtype=1, out_dtype=1, ids_bits=64, table=64, ids=64, out=64, n_tokens=1, rows=8, dim=8,
                     row_stride=8, ecc_stride=8, scale=1.0)
    for k, v in more.items():
        setattr(d, k, v)
    return d


def _grad_desc(**more):
    d = _lib.FoEmbedGrad(struct_size=ctypes.sizeof(_lib.FoEmbedGrad), dy_dtype=1, out_dtype=1, ids_bits=64, dy=64, ids=64, out=64, n_tokens=1, rows=8, dim=8,
                         dy_stride=8, scale=1.0, workspace=64, workspace_bytes=1 << 30)
    for k, v in more.items():
        setattr(d, k, v)
    return d


def _drop(p, bits=0, at=0):
    return _lib.FoDropout(p=p, seed=1, offset=2, dev_offset=at, dev_offset_bits=bits)


# (every one of these is refused before anything is launched: no pointer here is one)
@pytest.mark.parametrize("more,status,text", [
    (dict(struct_size=3), 1, b"ABI mismatch"), (dict(table_dtype=3), 1, b"table_dtype"), (dict(out_dtype=2), 1, b"out_dtype"), (dict(ecc_bits=4), 1, b"ecc_bits"),
    (dict(table_dtype=0, out_dtype=0, ecc_bits=8), 1, b"carries no ECC"), (dict(ids_bits=16), 1, b"ids_bits"), (dict(dropout=_drop(1.5)), 1, b"p = 1.5"),
    (dict(dropout=_drop(float("nan"))), 1, b"p = "), (dict(dropout=_drop(0.5, 8, 64)), 1, b"dev_offset_bits"), (dict(ids=0), 1, b"null"), (dict(table=0), 1, b"null"),
    (dict(ecc_bits=8, ecc=0), 1, b"null"), (dict(row_stride=7), 1, b"elements apart"), (dict(ecc_bits=8, ecc=64, ecc_stride=7), 1, b"elements apart"),
    (dict(n_tokens=1 << 32), 4, b"tokens"), (dict(dim=1 << 28, row_stride=1 << 28), 4, b"tokens"),
])
def test_fo_embed_refuses(more, status, text):
    lib = _lib.lib()
    assert lib.fo_embed(ctypes.byref(_embed_desc(**more)), None) == status
    assert text in lib.fo_last_error()


@pytest.mark.parametrize("more,status,text", [
    (dict(struct_size=3), 1, b"ABI mismatch"), (dict(dy_dtype=3), 1, b"dy_dtype"), (dict(out_dtype=-1), 1, b"out_dtype"), (dict(ids_bits=0), 1, b"ids_bits"),
    (dict(dropout=_drop(-0.1)), 1, b"p = -0.1"), (dict(out=0), 1, b"null"), (dict(dy=0), 1, b"null"), (dict(dy_stride=7), 1, b"elements apart"),
    (dict(n_tokens=(1 << 31) - 1), 4, b"tokens"), (dict(rows=(1 << 31) - 1), 4, b"rows"), (dict(dim=1 << 24, dy_stride=1 << 24), 4, b"elements"),
    (dict(n_tokens=65, workspace_bytes=16), 1, b"workspace"), (dict(n_tokens=65, workspace=0), 1, b"workspace"), (dict(n_tokens=65, workspace=72), 1, b"workspace"),
])
def test_fo_embed_grad_refuses(more, status, text):
    lib = _lib.lib()
    assert lib.fo_embed_grad(ctypes.byref(_grad_desc(**more)), None) == status
    assert text in lib.fo_last_error()


def test_fo_dropout_refuses():
    lib = _lib.lib()
    assert lib.fo_dropout(64, 0, 64, 5, 1, ctypes.byref(_drop(0.1)), None) == 1 and b"dtype" in lib.fo_last_error()
    assert lib.fo_dropout(64, 0, 64, 1, 1, None, None) == 1 and b"null" in lib.fo_last_error()
    assert lib.fo_dropout(0, 0, 64, 1, 1, ctypes.byref(_drop(0.1)), None) == 1 and b"null" in lib.fo_last_error()
    assert lib.fo_dropout(64, 0, 64, 1, 1, ctypes.byref(_drop(2.0)), None) == 1 and b"p = 2" in lib.fo_last_error()
    assert lib.fo_dropout(64, 0, 64, 1, 1 << 61, ctypes.byref(_drop(0.1)), None) == 4


def test_nothing_to_do_needs_no_gpu():
    lib = _lib.lib()
    assert lib.fo_embed(None, None) == 1 and lib.fo_embed_grad(None, None) == 1
    assert lib.fo_embed(ctypes.byref(_embed_desc(n_tokens=0, ids=0, out=0)), None) == 0
    assert lib.fo_embed(ctypes.byref(_embed_desc(dim=0, row_stride=0, ids=0, out=0)), None) == 0
    assert lib.fo_embed_grad(ctypes.byref(_grad_desc(rows=0, out=0)), None) == 0
    assert lib.fo_embed_grad(ctypes.byref(_grad_desc(n_tokens=0, accumulate=1)), None) == 0
    assert lib.fo_dropout(0, 0, 0, 1, 0, ctypes.byref(_drop(0.1)), None) == 0


def test_workspace_sizes():
    lib = _lib.lib()

    def need(rows, dim, n):
        out = ctypes.c_uint64(99)
        assert lib.fo_embed_grad_workspace(rows, dim, n, ctypes.byref(out)) == 0
        return out.value

    assert need(0, 8, 5) == 0 and need(5, 0, 5) == 0
    assert need(50257, 768, 1) == 0 and need(50257, 768, 64) == 0  # a handful of tokens needs none
    # keys and positions, and where each row's tokens begin; partial sums of one row at either end of a chunk stay a few megabytes whatever the sizes
    for rows, dim, n in ((1, 1, 65), (100, 7, 333), (50257, 768, 16384), (128256, 4096, 1 << 20), (2**31 - 2, 8, 2**31 - 2), (8, 2**24 - 1, 65)):
        assert 8 * n <= need(rows, dim, n) <= 17 * n + 4 * rows + 8 * dim + (64 << 20), (rows, dim, n)
    assert lib.fo_embed_grad_workspace(2**31, 8, 1, ctypes.byref(ctypes.c_uint64())) == 4
    assert lib.fo_embed_grad_workspace(8, 8, 1, None) == 1


def test_tensors_on_the_host_are_refused():
    table, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        fo.embed(table, ids)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        fo.embed_grad(torch.zeros(3, 8), ids, 4)
    with pytest.raises(RuntimeError, match="CUDA devices only"):
        fo.dropout(table, 0.5, 1)
    with pytest.raises(TypeError, match="torch.Tensor"):
        fo.dropout([1.0], 0.5, 1)


def test_gradient_trees_without_tokens_are_handed_on_as_they_are():
    grads = {"a": torch.zeros(2), "b": [torch.zeros(3)]}
    assert embedding.dense_gradients(grads, grads) is grads
    # other trees than the parameters' are left to the step, which refuses them
    odd = {"a": fo.TokenGradient(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))}
    assert embedding.dense_gradients(grads, odd) is odd


def test_a_token_gradient_belongs_to_a_matrix():
    g = fo.TokenGradient(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="does not belong"):
        g.dense(torch.zeros(5))
    with pytest.raises(ValueError, match="does not belong"):
        g.dense(torch.zeros(5, 4))
