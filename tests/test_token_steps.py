"""Steps whose gradients hold no tokens pay for none: what the optimizers ask of a tree of gradients, on the CPU with the device calls replaced."""

import contextlib

import pytest
import torch

import flashoptim_jax_b200 as fo
from flashoptim_jax_b200 import _engine, _lib, clipping, embedding


class _Stop(Exception):
    pass


def _stop(*args, **more):
    raise _Stop


def _tree():
    return {"a": torch.zeros(4, 3), "b": [torch.zeros(3), torch.zeros(2, 2)]}


def _tokens():
    return fo.TokenGradient(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int64))


def _count_walks(monkeypatch):
    walks, real = [], embedding.pytree.tree_leaves

    def counted(tree, *args, **more):
        walks.append(tree)
        return real(tree, *args, **more)

    monkeypatch.setattr(embedding.pytree, "tree_leaves", counted)
    return walks


@pytest.mark.parametrize("name,state", [("flash_adamw", fo.FlashAdamState), ("flash_lion", fo.FlashLionState), ("flash_sgdw", fo.FlashSGDState)])
@pytest.mark.parametrize("capturable", [True, False])
def test_a_step_without_tokens_looks_for_none_in_a_walk_of_its_own(monkeypatch, name, state, capturable):
    tx = getattr(fo, name)(learning_rate=1e-3, capturable=capturable)
    walks = _count_walks(monkeypatch)
    monkeypatch.setattr(_engine, "device_step_scalars", _stop)
    monkeypatch.setattr(_engine, "make_work", _stop)
    params, grads = _tree(), _tree()
    fields = {f: _tree() for f in state._fields if f != "count"}
    with pytest.raises(_Stop):
        tx.step(params, state(count=torch.zeros((), dtype=torch.int32), **fields), grads)
    assert not any(w is grads for w in walks)
    # and finds the tokens where there are some
    asked = []
    monkeypatch.setattr(fo.TokenGradient, "dense", lambda self, param, out=None: asked.append(tuple(param.shape)) or torch.zeros_like(param))
    with pytest.raises(_Stop):
        tx.step(params, state(count=torch.zeros((), dtype=torch.int32), **fields), {**grads, "a": _tokens()})
    assert asked == [(4, 3)]


class _Host:
    def __init__(self, answer):
        self.answer, self.asked = answer, []

    def sq_norm(self, grads):
        self.asked.append(grads)
        return self.answer(grads)


def test_clipping_asks_for_the_norm_once(monkeypatch):
    """A tree that the host extension leaves to the general path is not handed to it again."""
    host, of, walks = _Host(lambda grads: None), [], _count_walks(monkeypatch)
    monkeypatch.setattr(_lib, "host", lambda: host)
    monkeypatch.setattr(_engine, "grad_clip", lambda sq, most: contextlib.nullcontext())
    monkeypatch.setattr(_engine, "sq_norm_of", lambda leaves: of.append(len(leaves)) or torch.zeros(1, dtype=torch.float64))
    tx = clipping.clip_by_global_norm(fo.FlashOptimizer(init=None, step=lambda params, state, grads: (params, state)), 1.0)
    grads = _tree()
    tx.step(_tree(), {"clip": (), "opt": ()}, grads)
    assert len(host.asked) == 1 and of == [3] and sum(w is grads for w in walks) == 1


def test_clipping_makes_the_gradient_of_tokens_first(monkeypatch):
    host = _Host(lambda grads: None if any(type(g) is fo.TokenGradient for g in embedding.pytree.tree_leaves(grads)) else torch.zeros(1, dtype=torch.float64))
    monkeypatch.setattr(_lib, "host", lambda: host)
    monkeypatch.setattr(_engine, "grad_clip", lambda sq, most: contextlib.nullcontext())
    monkeypatch.setattr(fo.TokenGradient, "dense", lambda self, param, out=None: torch.ones_like(param))
    seen = []
    tx = clipping.clip_by_global_norm(fo.FlashOptimizer(init=None, step=lambda params, state, grads: seen.append(grads) or (params, state)), 1.0)
    tx.step(_tree(), {"clip": (), "opt": ()}, {**_tree(), "a": _tokens()})
    assert len(host.asked) == 2 and torch.equal(seen[0]["a"], torch.ones(4, 3))
    with pytest.raises(ValueError, match="must match"):
        tx.step(_tree(), {"clip": (), "opt": ()}, {"a": _tokens()})
