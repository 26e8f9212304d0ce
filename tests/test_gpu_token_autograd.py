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


@pytest.mark.parametrize("accumulate", [False, True])
def test_a_gradient_is_not_written_into_a_graph(accumulate):
    """The sums know nothing of the graph that `out` belongs to: its gradient would be that of what `out` held before."""
    import flashoptim_jax_b200 as fo

    dy, ids = torch.ones(6, 8, device="cuda"), torch.arange(6, device="cuda")
    leaf = torch.ones(9, 8, device="cuda", requires_grad=True)
    for out in (leaf, leaf * 2):
        before = out.detach().clone()
        with pytest.raises(RuntimeError, match="out"):
            fo.embed_grad(dy, ids, 9, out=out, accumulate=accumulate)
        assert torch.equal(out.detach(), before)
    with torch.no_grad():  # as torch's own operators with out=
        got = fo.embed_grad(dy, ids, 9, out=leaf, accumulate=accumulate)
    assert got is leaf and torch.equal(leaf.detach()[:6], dy + (1.0 if accumulate else 0.0))
