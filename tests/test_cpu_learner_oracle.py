"""CPU: the learner's oracle (oracle/learner_ref.py) pinned by closed forms, by differences and by
torch's own operations."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import learner_ref as ref


def _inputs(n, a, seed, share=0.4):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(n, a, generator=g, dtype=torch.float64) * 2
    legal = torch.rand(n, a, generator=g) < share
    legal[torch.arange(n), torch.randint(0, a, (n,), generator=g)] = True
    action = (torch.rand(n, a, generator=g) * legal).argmax(1)
    old = logits.masked_fill(~legal, -math.inf).log_softmax(1)
    old = old.gather(1, action[:, None])[:, 0] + 0.3 * torch.randn(n, generator=g)
    return dict(logits=logits, action=action, old_logp=old,
                advantage=torch.randn(n, generator=g, dtype=torch.float64), legal=legal,
                ref=logits + torch.randn(n, a, generator=g, dtype=torch.float64),
                value=torch.randn(n, generator=g, dtype=torch.float64),
                returns=torch.randn(n, generator=g, dtype=torch.float64),
                weight=torch.rand(n, generator=g, dtype=torch.float64),
                clip=(0.2, 0.3), kl_coef=0.3, entropy_coef=0.2, value_coef=0.7)


def test_policy_loss_gradient_is_the_loss_differences():
    x = _inputs(7, 9, 1)
    got = ref.policy_loss(**x)
    h = 1e-6
    for name in ("logits", "value"):
        for i in torch.cartesian_prod(torch.arange(7), torch.arange(9)) if name == "logits" else torch.arange(7)[:, None]:
            at = tuple(i.tolist())
            up, down = x[name].clone(), x[name].clone()
            up[at] += h
            down[at] -= h
            slope = (ref.policy_loss(**{**x, name: up})["loss"]
                     - ref.policy_loss(**{**x, name: down})["loss"]) / (2 * h)
            assert abs(slope - got["d_" + name][at]) < 1e-8, (name, at)


def test_policy_loss_closed_forms():
    one = torch.zeros(1, dtype=torch.float64)
    # k equal legal logits: entropy log k, log-probability -log k, ratio 1
    z = torch.full((1, 6), 3.0, dtype=torch.float64)
    legal = torch.tensor([[True, True, False, True, True, False]])
    got = ref.policy_loss(z, torch.tensor([1]), one - math.log(4), one + 2, legal)
    assert got["stats"].tolist() == pytest.approx([-2, 0, 0, math.log(4), 0, 0], abs=1e-12)
    assert got["d_logits"][0].tolist() == pytest.approx([0.5, -1.5, 0, 0.5, 0.5, 0], abs=1e-12)
    # a ratio past the clip: the bound times the advantage, no gradient
    got = ref.policy_loss(z, torch.tensor([1]), one - math.log(8), one + 2, legal)
    assert got["stats"][0] == pytest.approx(-2.4) and got["stats"][4] == 1
    assert got["d_logits"].abs().max() == 0
    # the same ratio with a negative advantage is not cut
    got = ref.policy_loss(z, torch.tensor([1]), one - math.log(8), one - 2, legal)
    assert got["stats"][0] == pytest.approx(4.0) and got["stats"][4] == 0
    # an illegal action: ratio 0; an empty row: the value term alone
    got = ref.policy_loss(z, torch.tensor([2]), one, one - 2, legal)
    assert got["logp"][0] == -math.inf and got["stats"][0] == pytest.approx(1.6)
    got = ref.policy_loss(z, torch.tensor([2]), one, one, legal & False, value=one + 3,
                          returns=one + 1)
    assert got["loss"] == 1.0 and got["d_value"][0] == 1.0 and got["logp"][0] == 0
    # KL to itself is 0, and to another policy the sum by hand
    got = ref.policy_loss(z, torch.tensor([0]), one, one, ref=z + 5, kl_coef=1.0)
    assert got["stats"][2] == pytest.approx(0, abs=1e-14)
    q = torch.tensor([[0.0, math.log(3.0)]], dtype=torch.float64)
    got = ref.policy_loss(q * 0, torch.tensor([0]), one, one, ref=q)
    assert got["stats"][2] == pytest.approx(0.5 * math.log(0.5 / 0.25) + 0.5 * math.log(0.5 / 0.75))


def test_advantages_closed_forms():
    t, b = 6, 3
    g = torch.Generator().manual_seed(2)
    r = torch.randn(t, b, generator=g, dtype=torch.float64)
    v = torch.randn(t, b, generator=g, dtype=torch.float64)
    last = torch.randn(b, generator=g, dtype=torch.float64)
    none = torch.zeros(t, b, dtype=torch.bool)
    # lam = 1, gamma = 1, nothing done: the rewards to come and the bootstrap, less the value
    adv, ret = ref.advantages(r, v, none, last, 1.0, 1.0)
    assert torch.allclose(ret, r.flip(0).cumsum(0).flip(0) + last)
    assert torch.allclose(adv, ret - v)
    # lam = 0: one step's difference; all done: the reward alone
    adv, _ = ref.advantages(r, v, none, last, 0.9, 0.0)
    assert torch.allclose(adv, r + 0.9 * torch.cat([v[1:], last[None]]) - v)
    adv, ret = ref.advantages(r, v, ~none, last, 0.9, 0.9)
    assert torch.allclose(ret, r)
    # the other player's side: all signs turn, rewards being player 0's
    who = torch.ones(t, b, dtype=torch.uint8)
    other, _ = ref.advantages(-r, v, none, last, 0.9, 0.8, who, who[0])
    mine, _ = ref.advantages(r, v, none, last, 0.9, 0.8)
    assert torch.allclose(other, mine)


def test_adamw_is_torchs():
    g = torch.Generator().manual_seed(3)
    w = torch.randn(50, generator=g, dtype=torch.float64)
    p = torch.nn.Parameter(w.clone())
    opt = torch.optim.AdamW([p], lr=0.01, betas=(0.8, 0.95), eps=1e-5, weight_decay=0.1)
    m = v = torch.zeros_like(w)
    for t in range(1, 6):
        grad = torch.randn(50, generator=g, dtype=torch.float64)
        p.grad = grad
        opt.step()
        w, m, v = ref.adamw(w, grad, m, v, t, 0.01, (0.8, 0.95), 1e-5, 0.1)
        assert torch.allclose(w, p.detach(), rtol=0, atol=1e-14)


@pytest.mark.parametrize("mantissa,least,dtype", [(3, -6, torch.float8_e4m3fn),
                                                  (2, -14, torch.float8_e5m2)])
def test_codes_are_the_types(mantissa, least, dtype):
    """The codes' values are torch's float8 values; a representable value keeps its code under any
    bits; a value between two codes becomes each with the share of the bits that its place says."""
    count = 127 if mantissa == 3 else 124
    values = torch.arange(count, dtype=torch.uint8).view(dtype).double()
    for c in range(count):
        y = ref.value_of(c, mantissa, least)
        assert y == values[c]
        assert ref.code(y, 0, mantissa, least) == ref.code(y, ref.MASK, mantissa, least) == c
    for c in (0, 1, 2**mantissa - 1, 2**mantissa, 40, 77):
        low, high = ref.value_of(c, mantissa, least), ref.value_of(c + 1, mantissa, least)
        y = low + 0.25 * (high - low)
        got = [ref.code(y, b << 24, mantissa, least) for b in range(256)]
        assert sorted(set(got)) == [c, c + 1] and got.count(c + 1) == 64


def test_rounding_words():
    """word() and words() agree; every input bit turns each output bit about half the time, and
    the words of neighbouring values, steps, tensors and seeds look unrelated."""
    w = ref.words(123456789012, 5, 17, 4096)
    assert [ref.word(123456789012, 5, 17, i) for i in (0, 1, 77, 4095)] == w[[0, 1, 77, 4095]].tolist()
    assert len(set(w.tolist())) == 4096  # mix is one to one
    n = 1 << 15
    base = ref.words(1, 0, 1, n).double() / 2**32
    others = [ref.words(1, 0, 2, n), ref.words(1, 1, 1, n), ref.words(2, 0, 1, n),
              ref.words(1, 0, 1, n).roll(1), ref.words(1 << 32, 0, 1, n)]
    for x in [base] + [o.double() / 2**32 for o in others]:
        assert abs(x.mean() - 0.5) < 5 * (1 / 12 / n) ** 0.5
        assert abs(x.var() - 1 / 12) < 5 * (1 / 180 / n) ** 0.5
    for o in others:
        corr = torch.corrcoef(torch.stack([base, o.double() / 2**32]))[0, 1]
        assert abs(corr) < 5 / n**0.5
    # the low 16 bits, which round the second moment, likewise
    low = (ref.words(1, 0, 1, n) & 0xFFFF).double() / 65536
    assert abs(low.mean() - 0.5) < 5 * (1 / 12 / n) ** 0.5
    assert abs(torch.corrcoef(torch.stack([base, low]))[0, 1]) < 5 / n**0.5
