"""CPU: the optimizer's options, copies and checkpoints (a step itself needs a GPU)."""

from __future__ import annotations

import copy
import io
import pickle
import warnings

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


def test_a_checkpoint_carries_the_options(ext):
    """Into an optimizer made with others; one written before the options were in the groups leaves
    them as they are."""
    _, opt = _optimizer(ext)
    _, other = _optimizer(ext, betas=(0.7, 0.9), eps=1e-3, max_norm=None, seed=1, lr=1.0)
    saved = opt.state_dict()
    other.load_state_dict(saved)
    assert (other.betas, other.eps, other.max_norm, other.seed) == ((0.8, 0.95), 1e-6, 0.5, 9)
    assert [g["lr"] for g in other.param_groups] == [1e-3, 1e-2]
    for g in saved["param_groups"]:
        for k in ("betas", "eps", "max_norm", "seed"):
            del g[k]
    _, old = _optimizer(ext, betas=(0.7, 0.9), eps=1e-3, max_norm=None, seed=1)
    old.load_state_dict(saved)
    assert (old.betas, old.eps, old.max_norm, old.seed) == ((0.7, 0.9), 1e-3, None, 1)


def test_options_of_the_whole_step(ext):
    """Schedulers may move the betas, together; groups that differ in them are refused."""
    from cugo_amd import learner

    _, opt = _optimizer(ext)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")  # no step before the scheduler's
        schedule = torch.optim.lr_scheduler.OneCycleLR(opt, max_lr=0.1, total_steps=10)
        assert opt.betas[0] == 0.95 and opt.betas[1] == 0.95
        for _ in range(3):
            schedule.step()
    assert 0.85 <= opt.betas[0] < 0.95
    opt.betas, opt.seed = (0.5, 0.6), 3
    assert all(g["betas"] == (0.5, 0.6) and g["seed"] == 3 for g in opt.param_groups)
    opt.param_groups[1]["betas"] = [0.5, 0.6]
    assert opt.betas == (0.5, 0.6)
    for name, value in (("betas", (0.5, 0.7)), ("eps", 0.1), ("max_norm", 7.0), ("seed", 4)):
        _, opt = _optimizer(ext)
        opt.param_groups[1][name] = value
        with pytest.raises(ValueError, match=name):
            opt.step()
    with pytest.raises(ValueError, match="betas"):
        learner.AdamW(ext, [dict(params=[torch.nn.Parameter(torch.zeros(2))], betas=(0.1, 0.1)),
                            dict(params=[torch.nn.Parameter(torch.zeros(2))])]).step()


def test_options_that_make_no_sense_are_refused(ext):
    """As torch's own optimizer does, for the defaults and for a group's."""
    from cugo_amd import learner

    p = lambda: torch.nn.Parameter(torch.zeros(2))  # noqa: E731
    nan = float("nan")
    for bad in (dict(lr=-1e-3), dict(lr=nan), dict(weight_decay=-0.1), dict(weight_decay=nan),
                dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8),
                dict(max_norm=0.0), dict(max_norm=-1.0)):
        with pytest.raises(ValueError, match=next(iter(bad))):
            learner.AdamW(ext, [p()], **bad)
        opt = learner.AdamW(ext, [p()])
        with pytest.raises(ValueError, match=next(iter(bad))):
            opt.add_param_group(dict(params=[p()], **bad))
        assert len(opt.param_groups) == 1
    learner.AdamW(ext, [p()], lr=torch.tensor([0.1]), weight_decay=0.0, max_norm=None)
    learner.AdamW(ext, [p()], lr=0.0, eps=0.0, betas=(0.0, 0.0))


def test_a_checkpoint_that_does_not_fit_changes_nothing(ext):
    _, opt = _optimizer(ext)
    keep = copy.deepcopy(opt)
    saved = copy.deepcopy(opt.state_dict())
    saved["param_groups"][0]["lr"] = 7.0
    del saved["state"][0]
    short = copy.deepcopy(saved)
    short["state"][3]["exp_avg"] = short["state"][3]["exp_avg"][:1]
    other = copy.deepcopy(saved)
    other["state"][3]["exp_avg_sq"] = other["state"][3]["exp_avg_sq"].float()
    lacking = copy.deepcopy(saved)
    del lacking["state"][3]["step"]
    fewer = copy.deepcopy(saved)
    fewer["param_groups"].pop()
    fewer["param_groups"][0]["params"] = [0, 1, 2, 3]
    for bad in (short, other, lacking, fewer):
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
        _same(opt, keep)


def test_a_checkpoint_of_torchs_own(ext):
    """Float32 parameters: the same moments, and steps, which torch counts in float32 on the host."""
    from cugo_amd import learner

    net, _ = _optimizer(ext, torch.float32)
    theirs = torch.optim.AdamW(net.parameters(), lr=3e-3, betas=(0.8, 0.9))
    for p in net.parameters():
        p.grad = torch.randn_like(p)
    theirs.step()
    saved = theirs.state_dict()
    ours = learner.AdamW(ext, net.parameters(), max_norm=2.0)
    ours.load_state_dict(saved)
    assert ours.betas == (0.8, 0.9) and ours.max_norm == 2.0
    ours.prepare()
    assert ours._steps.tolist() == [1, 1, 1, 1]
    for p in net.parameters():
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(ours.state[p][k], theirs.state[p][k])
    for s in saved["state"].values():
        s["step"] = 3  # as older ones counted
    ours.load_state_dict(saved)
    ours.prepare()
    assert ours._steps.tolist() == [3, 3, 3, 3]


def test_a_later_group_takes_the_options_as_they_are_now(ext):
    """Set, moved by a scheduler or loaded since the optimizer was made."""
    _, opt = _optimizer(ext)
    opt.betas, opt.max_norm, opt.seed = (0.5, 0.6), None, 3
    for g in opt.param_groups:
        g["eps"] = 0.25
    two = copy.deepcopy(opt)
    _, three = _optimizer(ext, betas=(0.7, 0.9))
    three.load_state_dict(opt.state_dict())
    for o in (opt, two, three):
        o.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2).bfloat16())]))
        assert (o.betas, o.max_norm, o.seed, o.eps) == ((0.5, 0.6), None, 3, 0.25)
        assert o.param_groups[2]["lr"] == 1e-3  # a group's own, as the optimizer was made with
    opt.add_param_group(dict(params=[torch.nn.Parameter(torch.zeros(2).bfloat16())], seed=4))
    with pytest.raises(ValueError, match="seed"):
        opt.seed
