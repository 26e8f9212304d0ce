"""Calls behind one another on one stream that share a workspace, through the C ABI, with nothing to wait for between them."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu


def whole(shape, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-8, 9, shape, generator=g).to(dtype).cuda()


def exact(dy, ids, rows):
    good = (ids >= 0) & (ids < rows)
    total = torch.zeros((rows, dy.shape[1]), dtype=torch.int64, device="cuda")
    return total.index_add_(0, ids[good], dy[good].long())


@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("n,rows,dim", [(65, 400, 8), (3000, 9000, 64), (8192, 50_000, 72), (20_000, 3000, 33), (30_000, 40_000, 256), (70_000, 5000, 24)])
def test_calls_that_share_a_workspace(n, rows, dim, p):
    """Whole numbers, so that every sum is exact: a row that was cleared, or left as it was, by the ids of an earlier call shows."""
    from flashoptim_jax_b200 import _lib

    lib, stream = _lib.lib(), torch.cuda.current_stream().cuda_stream
    need = ctypes.c_uint64()
    _lib.check(lib.fo_embed_grad_workspace(rows, dim, n, ctypes.byref(need)))
    workspace = torch.empty(need.value, dtype=torch.uint8, device="cuda")
    dy = whole((n, dim), n, torch.float32)
    g = torch.Generator().manual_seed(n)
    low, high = torch.randint(0, rows // 2, (n,), generator=g), torch.randint(rows // 2, rows, (n,), generator=g)
    calls = [low, high, torch.full((n,), rows - 1), low.flip(0), torch.full((n,), -1), torch.arange(n) % rows, torch.zeros(n, dtype=torch.int64), high]
    calls = [c.cuda() for c in calls]
    out = torch.full((4, len(calls), rows, dim), float("nan"), device="cuda")
    torch.cuda.synchronize()
    for k in range(4):
        for c, ids in enumerate(calls):
            f = _lib.FoEmbedGrad(struct_size=ctypes.sizeof(_lib.FoEmbedGrad), dy_dtype=_lib.FO_F32, out_dtype=_lib.FO_F32, ids_bits=64, dy=dy.data_ptr(), ids=ids.data_ptr(),
                                 out=out[k, c].data_ptr(), n_tokens=n, rows=rows, dim=dim, dy_stride=dim, scale=1.0, workspace=workspace.data_ptr(),
                                 workspace_bytes=need.value, dropout=_lib.FoDropout(p=p, seed=3, offset=4))
            _lib.check(lib.fo_embed_grad(ctypes.byref(f), stream))
    if p:
        import flashoptim_jax_b200 as fo

        dy = fo.dropout(dy, p, 3, 4)  # times 2: exact
    for c, ids in enumerate(calls):
        want = exact(dy, ids, rows).float()
        for k in range(4):
            assert torch.equal(out[k, c], want), (k, c)
