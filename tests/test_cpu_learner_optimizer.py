"""CPU: the optimizer's options, copies and checkpoints (a step itself needs a GPU)."""

from __future__ import annotations

import copy
import io
import pickle

import pytest
import torch


@pytest.fixture(scope="module")
def ext():
    from cugo_amd import _cugo_torch50_hip

    return _cugo_torch50_hip


def _optimizer(ext, dtype=torch.bfloat16, **over):
    from cugo_amd import learner

    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(37, 20), torch.nn.Linear(20, 3)).to(dtype)
    opt = learner.AdamW(ext, [dict(params=net[0].parameters(), weight_decay=0.2),
                              dict(params=net[1].parameters(), lr=1e-2)],
                        **{**dict(lr=1e-3, betas=(0.8, 0.95), eps=1e-6, max_norm=0.5,
                                  state_bits=8, seed=9), **over})
    opt.prepare()
    for i, s in enumerate(opt.state.values()):
        s["step"].fill_(i + 5)
        for t in s.values():
            if t.dtype == torch.float32:
                t.normal_()
    return net, opt


def _same(a, b):
    for p, q in zip(a._all(), b._all()):
        assert torch.equal(p, q)
        assert a.state[p].keys() == b.state[q].keys()
        for k, t in a.state[p].items():
            assert t.dtype == b.state[q][k].dtype and torch.equal(t.float(), b.state[q][k].float()), k
    for name in ("betas", "eps", "max_norm", "seed", "state_bits"):
        assert getattr(a, name) == getattr(b, name), name
    for g, h in zip(a.param_groups, b.param_groups):
        assert g["lr"] == h["lr"] and g["weight_decay"] == h["weight_decay"]


@pytest.mark.parametrize("bits", [8, 32])
def test_copied_and_pickled(ext, bits):
    """A copy has every option and state, a step count of its own, and the extension."""
    net, opt = _optimizer(ext, state_bits=bits)
    net2, two = copy.deepcopy((net, opt))
    buffer = io.BytesIO()
    torch.save(opt, buffer)
    buffer.seek(0)
    others = [two, torch.load(buffer, weights_only=False)]
    if bits == 32:  # (pickle by itself does not take torch's float8 tensors)
        others.append(pickle.loads(pickle.dumps(opt)))
    assert two._all()[0] is net2[0].weight
    for other in others:
        _same(opt, other)
        assert other.ext is ext
        other.prepare()
        assert other._steps.tolist() == [5, 6, 7, 8]
        other._steps += 1
        assert [int(other.state[p]["step"]) for p in other._all()] == [6, 7, 8, 9]
    assert opt._steps.tolist() == [5, 6, 7, 8]
