"""What autograd may and may not ask of the lookup, its gradient and dropout."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

pytestmark = pytest.mark.gpu


def _calls():
    import flashoptim_jax_b200 as fo

    x, r = torch.ones(6, 8, device="cuda"), torch.full((6, 8), 2.0, device="cuda")
    ids = torch.arange(6, device="cuda")
    return {
        "embed": (lambda t: fo.embed(t, ids, p=0.1), x),
        "embed to another type": (lambda t: fo.embed(t, ids, dtype=torch.float32), x.bfloat16()),
        "embed of master weights": (lambda t: fo.embed(t, ids, ecc=torch.zeros((6, 8), dtype=torch.int8, device="cuda")), x.bfloat16()),
        "embed of a parameter": (lambda t: fo.embed(t, ids), x.clone().requires_grad_()),
        "dropout": (lambda t: fo.dropout(t, 0.5, 1), x),
        "dropout of a view": (lambda t: fo.dropout(t, 0.5, 1), x.t()),
        "residual": (lambda t: fo.dropout(x, 0.5, 1, residual=t), r),
        "embed_grad": (lambda t: fo.embed_grad(t, ids, 9), x),
        "embed_grad to another type": (lambda t: fo.embed_grad(t, ids, 9, dtype=torch.float32), x.half()),
        "out": (lambda t: fo.embed_grad(x, ids, 6, out=t, accumulate=True), r),
    }


NAMES = ["embed", "embed to another type", "embed of master weights", "embed of a parameter", "dropout", "dropout of a view", "residual", "embed_grad", "embed_grad to another type", "out"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name):
    """None of the calls knows forward-mode derivatives: a result without a tangent would be a derivative of zero."""
    call, x = _calls()[name]
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(forward_ad.make_dual(x, torch.ones_like(x)))
        call(x)  # beside dual numbers, ordinary ones are as ever
    call(x)
