"""CPU: what the learner's C entry points and operations refuse before anything is launched."""

from __future__ import annotations

import ctypes

import pytest
import torch

from tests.conftest import REPO

F32, F16, BF16 = 0, 1, 2
P, I64, I32, F64 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_double


class Loss(ctypes.Structure):
    _fields_ = [("n", I64), ("actions", I64), ("logits_dtype", I32), ("value_dtype", I32),
                ("logits", P), ("ref_logits", P), ("legal", P), ("logits_stride", I64),
                ("ref_stride", I64), ("legal_stride", I64), ("action", P), ("old_logp", P),
                ("advantage", P), ("weight", P), ("value", P), ("returns", P), ("scale", P),
                ("clip_low", F64), ("clip_high", F64), ("kl_coef", F64), ("entropy_coef", F64),
                ("value_coef", F64), ("d_logits", P), ("d_logits_stride", I64), ("d_value", P),
                ("logp", P), ("loss", P), ("stats", P), ("partials", P)]


class Tensor(ctypes.Structure):
    _fields_ = [("param", P), ("grad", P), ("master", P), ("exp_avg", P), ("exp_avg_sq", P),
                ("exp_avg_scale", P), ("exp_avg_sq_scale", P), ("step", P), ("numel", I64),
                ("lr", F64), ("weight_decay", F64), ("place", ctypes.c_int32),
                ("param_dtype", ctypes.c_int16), ("grad_dtype", ctypes.c_int16)]


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(REPO / "cugo_amd" / "libcugo_hip.so"))
    lib.cugo_policy_loss.argtypes = [P, P]
    lib.cugo_scale_gradients.argtypes = [I32, P, I64, I32, P, I64, P, P]
    lib.cugo_advantages.argtypes = [I32, P, P, P, P, P, P, I64, I64, F64, F64, P, P, P, I64, P]
    lib.cugo_advantages_workspace.argtypes = [I64, I64]
    lib.cugo_advantages_workspace.restype = I64
    lib.cugo_adamw_workspace.argtypes = [I64]
    lib.cugo_adamw_workspace.restype = I64
    lib.cugo_adamw.argtypes = [P, I64, I32, F64, F64, F64, P, F64, ctypes.c_uint64, P, P, I64, P]
    return lib


BUF = ctypes.create_string_buffer(64)
AT = ctypes.addressof(BUF)


def _loss(**over):
    x = dict(n=4, actions=179, logits_dtype=BF16, value_dtype=F32, logits=AT, logits_stride=179,
             action=AT, old_logp=AT, advantage=AT, logp=AT, loss=AT, stats=AT, partials=AT)
    return Loss(**{**x, **over})


def test_policy_loss(lib):
    assert lib.cugo_policy_loss(None, None) == -1
    for over, code in ((dict(n=-1), -1), (dict(actions=0), -1), (dict(actions=(1 << 30) + 1), -1),
                       (dict(logits=None), -1), (dict(action=None), -1), (dict(old_logp=None), -1),
                       (dict(advantage=None), -1), (dict(logp=None), -1), (dict(loss=None), -1),
                       (dict(stats=None), -1), (dict(partials=None), -1), (dict(value=AT), -1),
                       (dict(returns=AT), -1), (dict(d_value=AT), -1), (dict(logits_dtype=3), -2),
                       (dict(value=AT, returns=AT, value_dtype=7), -2),
                       (dict(logits_stride=1 << 24), -4), (dict(legal_stride=1 << 24), -4),
                       (dict(ref_stride=1 << 30), -4)):
        x = _loss(**over)
        assert lib.cugo_policy_loss(ctypes.byref(x), None) == code, over


def test_policy_loss_strides(lib):
    """Rows that run backwards, and gradients whose rows overlap."""
    for over in (dict(logits_stride=-179), dict(legal_stride=-1), dict(ref_stride=-179),
                 dict(actions=2000, logits_stride=-2000), dict(d_logits=AT, d_logits_stride=178),
                 dict(d_logits=AT, d_logits_stride=0)):
        x = _loss(**over)
        assert lib.cugo_policy_loss(ctypes.byref(x), None) == -4, over


def test_scale_gradients(lib):
    assert lib.cugo_scale_gradients(F32, AT, -1, F32, None, 0, AT, None) == -1
    assert lib.cugo_scale_gradients(F32, None, 4, F32, None, 0, AT, None) == -1
    assert lib.cugo_scale_gradients(F32, AT, 4, F32, None, 2, AT, None) == -1
    assert lib.cugo_scale_gradients(F32, AT, 4, F32, None, 0, None, None) == -1
    assert lib.cugo_scale_gradients(5, AT, 4, F32, None, 0, AT, None) == -2
    assert lib.cugo_scale_gradients(F32, None, 0, F32, None, 0, AT, None) == 0


def test_advantages(lib):
    def go(dtype=F32, reward=AT, value=AT, done=AT, player=None, bootstrap=AT, last=None, steps=8,
           batch=4, advantage=AT, returns=AT, scratch=None, size=0):
        return lib.cugo_advantages(dtype, reward, value, done, player, bootstrap, last, steps, batch,
                                   0.9, 0.9, advantage, returns, scratch, size, None)

    assert go(steps=0) == go(batch=0) == 0
    for over in (dict(steps=-1), dict(batch=-1), dict(batch=1 << 37), dict(reward=None),
                 dict(value=None), dict(done=None), dict(bootstrap=None), dict(advantage=None),
                 dict(returns=None), dict(player=AT), dict(last=AT)):
        assert go(**over) == -1, over
    assert go(dtype=3) == -2
    need = lib.cugo_advantages_workspace(100_000, 3)
    assert need > 0 and need % 24 == 0
    assert go(steps=100_000, batch=3) == -3
    assert go(steps=100_000, batch=3, scratch=AT, size=need - 1) == -3
    assert lib.cugo_advantages_workspace(0, 5) == lib.cugo_advantages_workspace(8, 4) == 0


def test_adamw(lib):
    ok = dict(param=AT, grad=AT, exp_avg=AT, exp_avg_sq=AT, step=AT, numel=8, param_dtype=F32,
              grad_dtype=F32)

    def go(bits=32, count=1, tensors=True, scratch=AT, size=1 << 20, **over):
        t = Tensor(**{**ok, **over})
        return lib.cugo_adamw(ctypes.byref(t) if tensors else None, count, bits, 0.9, 0.999, 1e-8,
                              None, 0.0, 0, None, scratch, size, None)

    assert lib.cugo_adamw(None, 0, 32, 0.9, 0.999, 1e-8, None, 0.0, 0, None, None, 0, None) == 0
    assert go(count=-1) == go(tensors=False) == go(scratch=None) == -1
    assert go(bits=16) == -2
    assert go(size=lib.cugo_adamw_workspace(1) - 1) == -3
    for over in (dict(numel=-1), dict(numel=(1 << 36) + 1), dict(param=None), dict(grad=None),
                 dict(exp_avg=None), dict(exp_avg_sq=None), dict(step=None), dict(master=AT),
                 dict(param_dtype=BF16)):
        assert go(**over) == -1, over
    assert go(param_dtype=9) == go(grad_dtype=-1) == -2
    assert go(bits=8) == go(bits=8, exp_avg_scale=AT) == -1
    assert lib.cugo_adamw_workspace(0) == 0
    assert lib.cugo_adamw_workspace(33) == 2 * lib.cugo_adamw_workspace(32)


def test_operations_refuse_cpu_tensors():
    from cugo_amd import _cugo_torch50_hip as m
    from cugo_amd import learner

    n, a = 3, 5
    z, act, v = torch.zeros(n, a), torch.zeros(n, dtype=torch.long), torch.zeros(n)
    with pytest.raises(RuntimeError, match="CUDA"):
        learner.policy_loss(m, z, act, v, v)
    with pytest.raises(RuntimeError, match="CUDA"):
        learner.advantages(m, torch.zeros(2, 3), torch.zeros(2, 3), torch.zeros(2, 3).bool(),
                           torch.zeros(3), 0.9, 0.9)
    with pytest.raises(RuntimeError, match="CUDA"):
        learner.adamw_step(m, [v], [v], [v], [v], torch.zeros(1, dtype=torch.long), lr=0.1)
    with pytest.raises((RuntimeError, TypeError), match="list"):
        m.adamw_step([1], [v], [v], [v], torch.zeros(1, dtype=torch.long), [0.1], [0.1], 0.9, 0.99,
                     1e-8)
    with pytest.raises(RuntimeError, match="no parameters"):
        learner.adamw_step(m, [], [], [], [], torch.zeros(0, dtype=torch.long), lr=0.1)
    with pytest.raises(ValueError, match="state_bits"):
        learner.AdamW(m, [torch.nn.Parameter(v)], state_bits=4)
