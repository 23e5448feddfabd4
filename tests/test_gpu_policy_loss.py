"""policy_loss and its gradients against the oracle in 64 bits.

Tolerances, counted before any run, with u = 2^-24 (half a float32 step).  A log-probability l
carries E = u (4 |l| + adds + 16): |l| for the rounded product in the exponent's argument and for
the logarithm's multiplication, the adds of a chain of sums (a lane's elements, then a tree of at
most 16), and 16 for the exponential's and the logarithm's own last places (v_exp_f32 and v_log_f32
are good to one) and the differences around them.  A probability and a ratio then carry E
relative to themselves; a gradient w p (pull + c_k (d - K) + c_e (l + H)) carries 4 E of w p times
the sum of its parts' sizes, the taken action's w pull once more; stored, half a step of its type
(or half of float16's smallest value)."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import learner_ref as ref
from tests.conftest import announce

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
LEAST = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24}
ARGS = dict(clip=(0.2, 0.3), kl_coef=0.3, entropy_coef=0.05, value_coef=0.7)


def make(n, a, dtype, seed, legal=True, with_ref=True, value=torch.float32, weight=True,
         share=0.3):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(n, a, generator=g) * 2).to(dtype)
    on = torch.rand(n, a, generator=g) < share if legal else torch.ones(n, a, dtype=torch.bool)
    if legal and n > 1:
        on[n // 2] = False  # a row without a legal action
    noise = torch.rand(n, a, generator=g)
    action = torch.where(on, noise, -1.0).argmax(1)
    old = logits.float().masked_fill(~on, -1e30).log_softmax(1).gather(1, action[:, None])[:, 0]
    x = dict(logits=logits, action=action, old_logp=old + 0.3 * torch.randn(n, generator=g),
             advantage=torch.randn(n, generator=g), legal=on if legal else None,
             ref=(logits.float() + torch.randn(n, a, generator=g)).to(dtype) if with_ref else None,
             value=torch.randn(n, generator=g).to(value) if value is not None else None,
             returns=torch.randn(n, generator=g) if value is not None else None,
             weight=None)
    if weight:
        x["weight"] = torch.rand(n, generator=g) * (torch.rand(n, generator=g) < 0.8)
    return x


def call(ext, x, grad=True, **over):
    from cugo_amd import learner

    on = lambda t: t.to(DEV) if isinstance(t, torch.Tensor) else t  # noqa: E731
    logits, value = on(x["logits"]), on(x["value"])
    if grad:
        logits = logits.detach().requires_grad_()
        value = None if value is None else value.detach().requires_grad_()
    out = learner.policy_loss(
        ext, logits, on(x["action"]), on(x["old_logp"]), on(x["advantage"]), legal=on(x["legal"]),
        ref_logits=on(x["ref"]), value=value, returns=on(x["returns"]), weight=on(x["weight"]),
        **{**ARGS, **over})
    got = {"loss": out.loss.detach(), "stats": out.stats, "logp": out.logp}
    if grad:
        leaves = [logits] + ([value] if value is not None else [])
        grads = torch.autograd.grad(out.loss, leaves)
        got["d_logits"], got["d_value"] = grads[0], grads[1] if value is not None else None
    return got


def check(x, got, scale=1.0):
    want = ref.policy_loss(**x, **ARGS, scale=scale)
    n, a = x["logits"].shape
    w = (x["weight"].double() if x["weight"] is not None else torch.full((n,), 1.0 / n)).abs()
    adds = (a / 64 if a <= 256 else a / 256) + 16
    on = x["legal"] if x["legal"] is not None else torch.ones(n, a, dtype=torch.bool)
    z = x["logits"].double().masked_fill(~on, -math.inf)
    ell = ref.log_softmax(z).nan_to_num(nan=0, neginf=0, posinf=0)
    p = torch.where(on, ell.exp(), 0.0)
    size = torch.where(p > 1e-46, ell.abs(), 0.0)
    d = torch.zeros_like(ell)
    if x["ref"] is not None:
        q = x["ref"].double().masked_fill(~on, -math.inf)
        lq = ref.log_softmax(q).nan_to_num(nan=0, neginf=0, posinf=0)
        d = torch.where(p > 1e-46, (ell - lq).abs(), 0.0)
        size = torch.maximum(size, torch.where(p > 1e-46, lq.abs(), 0.0))
    err = U * (4 * size + adds + 16)          # E of each entry
    row = (p * err).sum(1) + U * 16           # and of a row's mean
    logp = want["logp"]
    fine = logp > -math.inf
    assert torch.equal(got["logp"].cpu() == -math.inf, ~fine)
    e_act = U * (4 * logp.abs() + adds + 16)
    assert ((got["logp"].cpu().double() - logp).abs()[fine] <= e_act[fine]).all()
    ratio = torch.where(fine, (logp - x["old_logp"].double()).exp(), 0.0)
    drift = torch.where(fine, (logp - x["old_logp"].double()).abs(), 0.0)
    e_act = torch.where(fine, e_act, 0.0) + U * drift * 2
    pull = (ratio * x["advantage"].double()).abs()
    most = lambda t: t.max(1).values  # noqa: E731
    tol = torch.stack([
        (w * pull * (e_act + 8 * U)).sum(),
        w.sum() * 0, (w * 4 * (row * (1 + most(d)) + (p * err * d).sum(1))).sum(),
        (w * 4 * (row * (1 + most(size)))).sum(), w.sum() * 4 * U,
        (w * ((ratio + 1 + drift) * 4 * U + (ratio + 1) * e_act)).sum()])
    if x["value"] is not None:
        tol[1] = (w * 4 * U * (x["value"].double() - x["returns"].double()) ** 2).sum()
    tol = tol + U * want["stats"].abs() + 1e-37
    bad = torch.isinf(want["stats"])
    assert torch.equal(got["stats"].cpu().double()[bad], want["stats"][bad])
    diff = (got["stats"].cpu().double() - want["stats"]).abs()
    assert (diff[~bad] <= tol[~bad]).all(), (diff, tol)
    t_loss = abs(scale) * (tol[0] + 0.7 * tol[1] + 0.3 * tol[2] + 0.05 * tol[3]) + U * want["loss"].abs()
    assert (got["loss"].cpu().double() - want["loss"]).abs() <= t_loss * 2
    if "d_logits" not in got:
        return
    for name in ("d_logits", "d_value"):
        if got[name] is None:
            continue
        dt = got[name].dtype
        goal = want[name]
        if name == "d_logits":
            parts = pull[:, None] + 0.3 * (d + (p * d).sum(1, keepdim=True)) + \
                0.05 * (size + (p * size).sum(1, keepdim=True))
            t = 4 * p * parts * (err + row[:, None] + e_act[:, None])
            t.scatter_add_(1, x["action"].clamp(0, a - 1)[:, None],
                           (4 * pull * (e_act + 4 * U))[:, None])
            t = t * w[:, None] * abs(scale)
        else:
            t = goal.abs() * 4 * U
        t = t + goal.abs() * HALF[dt] * 1.01 + LEAST[dt] / 2 + 2.0**-140
        diff = (got[name].cpu().double() - goal).abs()
        assert (diff <= t).all(), (name, diff.max(), (diff / t).max())
        off = on if name == "d_logits" else None
        if off is not None:
            assert (got[name].cpu()[~off] == 0).all()


SIZES = [(5, 1), (9, 2), (6, 3), (7, 4), (3, 5), (17, 16), (5, 17), (4, 63), (4, 64), (4, 65),
         (3, 128), (3, 129), (40, 179), (3, 191), (3, 192), (3, 193), (3, 255), (3, 256), (3, 257),
         (3, 383), (3, 385), (2, 512), (5, 513), (2, 767), (2, 769), (3, 1024), (3, 1025), (2, 2047), (2, 2048), (3, 2049), (2, 4096), (2, 4097),
         (2, 4099), (1, 179), (1, 33001), (2, 8192), (2, 8193), (1, 16384), (2, 16385), (1, 32768),
         (1, 32769)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,a", SIZES)
def test_against_the_oracle(ext, n, a, dtype):
    for k, (legal, with_ref, weight, value) in enumerate([
            (True, True, True, torch.float32), (False, True, False, None),
            (True, False, False, torch.bfloat16), (False, False, True, torch.float16)]):
        announce(f"policy_loss {n}x{a} {dtype} variant {k}")
        x = make(n, a, dtype, 100 * a + k, legal, with_ref, value, weight)
        check(x, call(ext, x))
        check(x, call(ext, x, grad=False))


@pytest.mark.parametrize("a", [2, 7, 20, 40, 60, 179, 300, 1500, 9000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_special_entries(ext, a, dtype):
    """-inf, the type's lowest value, NaN and infinities in illegal places, rows whose legal
    logits are all -inf, actions that are illegal or outside, weights of zero over NaN rows."""
    announce(f"special {a} {dtype}")
    n = 12
    x = make(n, a, dtype, a, share=0.5)
    x["legal"][:, 0] = True
    x["legal"][5] = False
    x["weight"] = torch.rand(n) + 0.1
    low = torch.finfo(dtype).min
    for i, junk in enumerate((math.nan, math.inf, -math.inf, low)):
        x["logits"][i] = torch.where(x["legal"][i], x["logits"][i], junk)
        x["ref"][i] = torch.where(x["legal"][i], x["ref"][i], junk)
    x["logits"][4, 1:] = low           # legal, beside one ordinary logit
    x["ref"][4, 1:] = low
    x["action"][4] = 0
    x["old_logp"][4] = -0.1
    x["logits"][6, 1:] = -math.inf     # legal, without probability
    x["action"][6] = 0
    x["old_logp"][6] = 0.1
    x["logits"][7] = -math.inf         # all of them: as without a legal action
    x["ref"][7] = 0
    x["logits"][3], x["ref"][2] = low, low  # a whole row of it: as equal logits
    x["action"][8], x["action"][9], x["action"][10] = -1, a, 2**40
    x["logits"][11] = math.nan         # of weight zero
    x["ref"][11] = math.nan
    x["advantage"][11], x["old_logp"][11] = math.nan, math.nan
    x["value"][11], x["returns"][11] = math.nan, math.inf
    x["weight"][11] = 0
    x["action"][:4] = torch.where(x["legal"][:4], 1.0, 0.0).argmax(1)
    got = call(ext, x)
    assert got["stats"][5] == math.inf  # the actions without probability
    y = {k: v[:11] if isinstance(v, torch.Tensor) else v for k, v in x.items()}
    want11 = {k: v[:11] if k in ("logp", "d_logits", "d_value") else v for k, v in got.items()}
    check(y, want11)
    assert (got["d_logits"][11] == 0).all() and got["d_value"][11] == 0
    assert (got["d_logits"][7] == 0).all() and got["logp"][7] == 0


def test_nan_in_a_legal_logit_shows(ext):
    for a in (3, 179, 600, 2000, 33000):
        for bad in (math.nan, math.inf):
            x = make(3, a, torch.float32, a, share=0.9, weight=False)
            x["legal"][0, 0] = True
            x["logits"][0, 0] = bad
            got = call(ext, x)
            assert torch.isnan(got["loss"]) and torch.isnan(got["logp"][0])
            assert not torch.isnan(got["d_logits"][2]).any()


def test_the_only_legal_action_is_certain(ext):
    """Log-probability, entropy and KL term 0 exactly, whatever the logit; and no gradient but the
    pull's rounding."""
    for dtype in (torch.float32, torch.bfloat16):
        for a in (1, 2, 64, 179, 300, 1024, 2000, 40000):
            x = make(4, a, dtype, a, weight=False)
            x["logits"] = (x["logits"].float() * 7.3).to(dtype)
            x["legal"][:] = False
            x["action"] = torch.tensor([0, a // 3, a // 2, a - 1])
            x["legal"][torch.arange(4), x["action"]] = True
            got = call(ext, x)
            assert (got["logp"] == 0).all() and (got["stats"][2:4] == 0).all(), (a, dtype)
            assert (got["d_logits"][~x["legal"].to(DEV)] == 0).all()


def test_a_reference_without_the_action_is_infinitely_far(ext):
    """A legal action that the other policy never takes: the KL term is infinite, the rest is not."""
    for a in (2, 40, 179, 300, 1000, 2000, 9000, 40000):
        for dtype in (torch.float32, torch.bfloat16):
            x = make(3, a, dtype, a, weight=False, share=0.9)
            x["legal"][0, :2] = True
            x["ref"][0, 0] = -math.inf
            got = call(ext, x)
            assert got["stats"][2] == math.inf and got["loss"] == math.inf, a
            assert torch.isfinite(got["stats"][[0, 1, 3, 4, 5]]).all()
            x["legal"][0, 0] = False  # illegal: of no account
            x["action"][0] = 1
            assert torch.isfinite(call(ext, x)["loss"]), a


def test_nan_in_the_only_legal_logit_shows(ext):
    """No other logit is there to be the largest: the row must not pass for one without any."""
    for a in (1, 3, 40, 179, 300, 1024, 2000, 9000, 40000):
        for only_it in (True, False):
            x = make(3, a, torch.bfloat16, a, weight=False)
            x["legal"][0] = False
            x["legal"][0, a // 2] = only_it
            x["logits"][0] = math.nan if not only_it else x["logits"][0]
            x["logits"][0, a // 2] = math.nan
            x["action"][0] = a // 2
            got = call(ext, x)
            if only_it:
                assert torch.isnan(got["loss"]) and torch.isnan(got["logp"][0]), a
                assert torch.isnan(got["d_logits"][0, a // 2]), a
            else:  # all of the row illegal
                assert not torch.isnan(got["loss"]) and (got["d_logits"][0] == 0).all(), a


def test_loss_divided_in_place(ext):
    from cugo_amd import learner

    x = make(5, 30, torch.float32, 3, weight=False)
    on = {k: v.to(DEV) for k, v in x.items() if isinstance(v, torch.Tensor)}
    want = call(ext, x)
    logits = on["logits"].requires_grad_()
    out = learner.policy_loss(ext, logits, on["action"], on["old_logp"], on["advantage"],
                              legal=on["legal"], ref_logits=on["ref"], value=on["value"],
                              returns=on["returns"], **ARGS)
    loss = out.loss
    loss /= 4
    out.stats.mul_(2)
    loss.backward()
    assert torch.equal(logits.grad, want["d_logits"] * 0.25)
    assert torch.equal(loss.detach(), want["loss"] / 4)


def test_rows_far_apart(ext):
    """Rows more than 2^24 elements apart, of few and of many actions: the contiguous results."""
    for a in (2, 179, 2000):
        x = make(3, a, torch.bfloat16, a, weight=False)
        room = torch.zeros(3, (1 << 24) + 3, dtype=torch.bfloat16, device=DEV)
        room[:, 1:1 + a] = x["logits"].to(DEV)
        p, q = call(ext, dict(x, logits=room[:, 1:1 + a])), call(ext, x)
        for k in p:
            assert torch.equal(p[k], q[k]), k


FEW = [(1, 1), (65, 1), (63, 3), (64, 4), (130, 7), (66, 15), (67, 18), (65, 31), (64, 32), (3, 33),
       (65, 47), (129, 48), (33, 49), (31, 50), (70, 61), (300, 5)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,a", FEW)
def test_few_actions(ext, n, a, dtype):
    """Rows of 4 and of 8 lanes, on both sides of each line, and workgroups that end inside."""
    for k, (legal, with_ref, weight, value) in enumerate([
            (True, True, True, torch.float32), (False, True, False, None),
            (True, False, False, torch.bfloat16), (False, False, True, torch.float16)]):
        announce(f"policy_loss {n}x{a} {dtype} variant {k}")
        x = make(n, a, dtype, 100 * a + k, legal, with_ref, value, weight)
        check(x, call(ext, x))
        check(x, call(ext, x, grad=False))


@pytest.mark.parametrize("a", [1, 3, 4, 30, 48, 64])
def test_few_actions_as_far_apart_as_rows_are_addressed(ext, a):
    """float32 rows 2^24 - 1 elements apart: the last of a workgroup's 64 begins 4,227,858,180 bytes
    behind the first."""
    n, stride = 65, (1 << 24) - 1
    announce(f"far apart {n}x{a}")
    x = make(n, a, torch.float32, a, weight=False)
    room = torch.empty((n - 1) * stride + a, dtype=torch.float32, device=DEV)
    logits = room.as_strided((n, a), (stride, 1))
    logits.copy_(x["logits"])
    p, q = call(ext, dict(x, logits=logits)), call(ext, x)
    for k in p:
        assert torch.equal(p[k], q[k]), k


def test_strides_and_offsets(ext):
    """Logits that are the columns of a wider head, from an odd column on; reference logits of
    one row for all; a mask cut out of a wider one: the results of contiguous copies, bit by bit."""
    n, a = 37, 179
    for dtype in (torch.bfloat16, torch.float32, torch.float16):
        for shift in (0, 1, 3):
            announce(f"strides {dtype} {shift}")
            x = make(n, a, dtype, 5 + shift)
            head = torch.zeros(n, a + 5, dtype=dtype, device=DEV)
            head[:, shift:shift + a] = x["logits"].to(DEV)
            mask = torch.zeros(n, a + 7, dtype=torch.bool, device=DEV)
            mask[:, shift + 2:shift + 2 + a] = x["legal"].to(DEV)
            one = x["ref"][:1].to(DEV)
            y = dict(x, logits=head[:, shift:shift + a], legal=mask[:, shift + 2:shift + 2 + a],
                     ref=one.expand(n, a))
            z = dict(x, ref=one.expand(n, a).contiguous())
            p, q = call(ext, y), call(ext, z)
            for k in p:
                assert torch.equal(p[k], q[k]), k


def test_gradient_is_the_loss_differences(ext):
    """Central differences of the float32 loss along random directions, step h = 2^-6: the cubic
    term is below h^2 / 6 max |L'''| (|L'''| of these losses is below 8 along a unit direction)
    and the losses carry about 2^-21 each."""
    x = make(6, 20, torch.float32, 9, weight=False)
    got = call(ext, x)
    g = torch.Generator().manual_seed(1)
    h = 2.0**-6
    for _ in range(8):
        v = torch.randn(6, 20, generator=g)
        v /= v.norm()
        up = call(ext, dict(x, logits=x["logits"] + h * v), grad=False)["loss"].double()
        down = call(ext, dict(x, logits=x["logits"] - h * v), grad=False)["loss"].double()
        slope = ((up - down) / (2 * h)).cpu()
        along = (got["d_logits"].cpu().double() * v).sum()
        assert abs(slope - along) <= h * h * 8 / 6 + 2.0**-21 / h, (slope, along)


def test_large_batches_and_repeats(ext):
    """More rows than one round of workgroups: against torch's float64 operations and autograd;
    a second call gives the same bits."""
    n, a = 200_003, 179
    g = torch.Generator(device=DEV).manual_seed(3)
    logits = (torch.randn(n, a, generator=g, device=DEV) * 2).bfloat16()
    legal = torch.rand(n, a, generator=g, device=DEV) < 0.1
    legal[:, 7] = True
    action = (torch.rand(n, a, generator=g, device=DEV) * legal).argmax(1)
    adv = torch.randn(n, generator=g, device=DEV)
    x64 = logits.double().requires_grad_()
    ell = x64.masked_fill(~legal, -math.inf).log_softmax(1)
    lp = ell.gather(1, action[:, None])[:, 0]
    old = (lp.detach() + 0.3 * torch.randn(n, generator=g, device=DEV)).float()
    r = (lp - old.double()).exp()
    safe = ell.masked_fill(~legal, 0)
    loss = -(torch.minimum(r * adv, r.clamp(0.8, 1.3) * adv)
             - 0.05 * (ell.exp() * safe).sum(1)).mean()
    loss.backward()
    x = dict(logits=logits, action=action, old_logp=old, advantage=adv, legal=legal, ref=None,
             value=None, returns=None, weight=None)
    got, again = call(ext, x), call(ext, x)
    for k in ("loss", "stats", "logp", "d_logits"):
        assert torch.equal(got[k], again[k])
    # a row's parts are below 8 in size, their errors below 64 u of them
    assert abs(got["loss"].double() - loss.detach()) < 8 * 64 * U
    assert (got["logp"].double() - lp.detach()).abs().max() < 128 * U
    diff = (got["d_logits"].double() - x64.grad).abs()
    # half a bf16 step, and 64 u of the pull's size where p - 1 or the sum cancels
    assert (diff <= x64.grad.abs() * 2.0**-8 + 64 * U * 16 / n).all()


def test_scaled_losses(ext):
    """loss_scale is in the gradients before they are rounded; a gradient of the loss other than
    1 multiplies them after; one backward pass hands them out."""
    from cugo_amd import learner

    x = make(33, 179, torch.float16, 4, weight=False)
    s = torch.tensor(4096.0, device=DEV)
    got = call(ext, x, loss_scale=s)
    check(x, got, scale=4096.0)
    plain = call(ext, x)
    logits = x["logits"].to(DEV).requires_grad_()
    value = x["value"].to(DEV).requires_grad_()
    on = {k: v.to(DEV) for k, v in x.items() if isinstance(v, torch.Tensor)}
    out = learner.policy_loss(ext, logits, on["action"], on["old_logp"], on["advantage"],
                              legal=on["legal"], ref_logits=on["ref"], value=value,
                              returns=on["returns"], **ARGS)
    (out.loss * 0.5 + out.loss.detach()).backward(retain_graph=True)
    assert torch.equal(logits.grad, (plain["d_logits"].float() * 0.5).half())
    assert torch.equal(value.grad, plain["d_value"] * 0.5)
    with pytest.raises(RuntimeError, match="once"):
        out.loss.backward()
    again = learner.policy_loss(ext, logits, on["action"], on["old_logp"], on["advantage"])
    with pytest.raises(RuntimeError, match="differentiated once"):
        torch.autograd.grad(again.loss, logits, create_graph=True)
    assert not out.stats.requires_grad and not out.logp.requires_grad
    with torch.no_grad():
        quiet = learner.policy_loss(ext, logits, on["action"], on["old_logp"], on["advantage"])
    assert not quiet.loss.requires_grad


def test_only_one_side_wants_gradients(ext):
    from cugo_amd import learner

    x = make(9, 30, torch.float32, 8, weight=False)
    on = {k: v.to(DEV) for k, v in x.items() if isinstance(v, torch.Tensor)}
    both = call(ext, x)
    for which in ("logits", "value"):
        a = on["logits"].clone().requires_grad_(which == "logits")
        v = on["value"].clone().requires_grad_(which == "value")
        out = learner.policy_loss(ext, a, on["action"], on["old_logp"], on["advantage"],
                                  legal=on["legal"], ref_logits=on["ref"], value=v,
                                  returns=on["returns"], **ARGS)
        out.loss.backward()
        assert torch.equal(a.grad if which == "logits" else v.grad, both["d_" + which])
        assert (v.grad if which == "logits" else a.grad) is None


def test_no_rows(ext):
    x = make(4, 179, torch.bfloat16, 2, weight=False)
    x = {k: v[:0] if isinstance(v, torch.Tensor) else v for k, v in x.items()}
    got = call(ext, x)
    assert got["loss"] == 0 and (got["stats"] == 0).all()
    assert got["d_logits"].shape == (0, 179) and got["d_value"].shape == (0,)


def test_in_a_graph_and_on_another_stream(ext):
    """A captured loss and backward, replayed on new inputs with eager work in between, equals the
    eager results; so does a call on a side stream."""
    from cugo_amd import learner

    xs = [make(500, 179, torch.bfloat16, 50 + k, weight=False) for k in range(4)]
    keys = ("logits", "action", "old_logp", "advantage", "legal", "ref", "value", "returns")
    at = {k: xs[0][k].to(DEV).clone() for k in keys}
    logits, value = at["logits"].requires_grad_(), at["value"].requires_grad_()

    def once():
        out = learner.policy_loss(ext, logits, at["action"], at["old_logp"], at["advantage"],
                                  legal=at["legal"], ref_logits=at["ref"], value=value,
                                  returns=at["returns"], **ARGS)
        return (out.loss.detach(), out.stats, out.logp,
                *torch.autograd.grad(out.loss, [logits, value]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = once()
    torch.cuda.current_stream().wait_stream(side)
    want = call(ext, xs[0])
    names = ("loss", "stats", "logp", "d_logits", "d_value")
    for name, t in zip(names, first):
        assert torch.equal(t, want[name])
    del first
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for x in xs[1:] + xs[:1]:
        with torch.no_grad():
            for k in keys:
                at[k].copy_(x[k])
        graph.replay()
        want = call(ext, x)  # eager work between the replays
        torch.cuda.synchronize()
        for name, t in zip(names, held):
            assert torch.equal(t, want[name]), name


def test_refusals(ext):
    from cugo_amd import learner

    x = make(4, 10, torch.float32, 1, weight=False)
    on = {k: v.to(DEV) for k, v in x.items() if isinstance(v, torch.Tensor)}

    def go(**over):
        y = {**on, **over}
        return learner.policy_loss(ext, y["logits"], y["action"], y["old_logp"], y["advantage"],
                                   legal=y["legal"], ref_logits=y["ref"], value=y["value"],
                                   returns=y["returns"], weight=y.get("weight"),
                                   clip=y.get("clip", (0.2, 0.2)), kl_coef=y.get("kl_coef", 0.0),
                                   loss_scale=y.get("loss_scale"))

    go()
    for over in (dict(logits=on["logits"].cpu()), dict(logits=on["logits"].double()),
                 dict(logits=on["logits"][:, :0], legal=None, ref=None),
                 dict(logits=on["logits"].t()), dict(legal=on["legal"][:, :9]),
                 dict(legal=on["legal"].byte()), dict(ref=on["ref"].bfloat16()),
                 dict(logits=on["logits"].t().contiguous().t()),
                 dict(action=on["action"].int()), dict(action=on["action"][:3]),
                 dict(old_logp=on["old_logp"].double()), dict(advantage=on["advantage"][None]),
                 dict(returns=None), dict(value=None), dict(value=on["value"].double()),
                 dict(weight=on["value"].bfloat16()), dict(clip=(-0.1, 0.2)),
                 dict(kl_coef=math.inf), dict(loss_scale=torch.ones(2, device=DEV)),
                 dict(loss_scale=torch.ones(1))):
        with pytest.raises(RuntimeError):
            go(**over)


def _bits_of(t):
    return t.view(torch.int16) if t.element_size() == 2 else t.view(torch.int32)


@pytest.mark.parametrize("n,a", [(12_100_000, 179), (66_000, 33_000)])
def test_offsets_past_32_bits(ext, n, a):
    """More than 2^31 logits: the first, a middle and the last rows are those of calls on them alone,
    with the weights of the whole."""
    announce(f"policy_loss {n}x{a}")
    g = torch.Generator(device=DEV).manual_seed(8)
    logits = torch.empty(n, a, dtype=torch.bfloat16, device=DEV).normal_(generator=g).requires_grad_()
    action = torch.randint(0, a, (n,), generator=g, device=DEV)
    old = torch.full((n,), -math.log(a), device=DEV)
    adv = torch.randn(n, generator=g, device=DEV)
    weight = torch.full((n,), 0.01, device=DEV)
    loss, stats, logp = ext.policy_loss(logits, action, old, adv, weight=weight, entropy_coef=0.1)
    grad, = torch.autograd.grad(loss, [logits])
    for first in (0, n // 2 + 1, n - 40):
        rows = slice(first, first + 40)
        part = logits.detach()[rows].clone().requires_grad_()
        p_loss, _, p_logp = ext.policy_loss(part, action[rows].clone(), old[rows].clone(),
                                            adv[rows].clone(), weight=weight[rows].clone(),
                                            entropy_coef=0.1)
        p_grad, = torch.autograd.grad(p_loss, [part])
        assert torch.equal(logp[rows], p_logp)
        assert torch.equal(_bits_of(grad[rows].contiguous()), _bits_of(p_grad))
    assert torch.isfinite(loss)


def test_two_streams_at_once(ext):
    """Calls of two streams side by side keep to their own scratch memory."""
    xs = [make(3000, 179, torch.bfloat16, 70 + k, weight=False) for k in range(2)]
    want = [call(ext, x) for x in xs]
    on = [{k: v.to(DEV) for k, v in x.items() if isinstance(v, torch.Tensor)} for x in xs]
    from cugo_amd import learner

    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                out = learner.policy_loss(
                    ext, on[k]["logits"].requires_grad_(), on[k]["action"], on[k]["old_logp"],
                    on[k]["advantage"], legal=on[k]["legal"], ref_logits=on[k]["ref"],
                    value=on[k]["value"], returns=on[k]["returns"], **ARGS)
                got[k].append((out.loss.detach(), out.stats,
                               *torch.autograd.grad(out.loss, [on[k]["logits"]])))
    torch.cuda.synchronize()
    for k in range(2):
        for loss, stats, grad in got[k]:
            assert torch.equal(loss, want[k]["loss"]) and torch.equal(stats, want[k]["stats"])
            assert torch.equal(grad, want[k]["d_logits"])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("a,few", [(7, False), (20, False), (40, False), (64, False), (100, False),
                                   (179, False), (179, True), (300, False), (600, False),
                                   (1000, False), (1000, True), (2000, False), (2000, True),
                                   (9000, False), (40000, False), (40000, True)])
def test_a_taken_action_far_below_the_others(ext, a, few, dtype):
    """100 below the row's largest logit a probability is 0 in float32; the log-probability and the
    ratio are not, and the gradient has the action's pull."""
    for with_ref in (True, False):
        announce(f"far action {a} {few} {dtype} {with_ref}")
        x = make(6, a, dtype, a, legal=few, with_ref=with_ref, weight=False, value=None,
                 share=8 / a)
        on = x["legal"] if few else torch.ones(6, a, dtype=torch.bool)
        on[:, :2] = True
        x["action"] = torch.tensor([a - 1, 0, a // 2, 1, a - 1, 0])
        on[torch.arange(6), x["action"]] = True
        for i in (0, 2, 4, 5):
            others = on[i].clone()
            others[x["action"][i]] = False
            x["logits"][i, x["action"][i]] = x["logits"][i][others].float().max() - 100
        z = x["logits"].double().masked_fill(~on, -math.inf)
        logp = ref.log_softmax(z).gather(1, x["action"][:, None])[:, 0]
        assert (logp[[0, 2, 4, 5]] < -99).all()
        x["old_logp"] = (logp + 0.1).float()  # inside the clip
        x["advantage"] = torch.tensor([1.0, -1.0, -2.0, 0.5, 0.7, 3.0])
        got = call(ext, x)
        check(x, got)
        taken = got["d_logits"].cpu().gather(1, x["action"][:, None])[:, 0].float()
        assert (taken[[0, 2, 4, 5]].abs() > 0.05).all(), taken


def test_a_rows_gradient_is_its_own(ext):
    """Whatever the masks of the rows beside it: few legal actions are listed, many are not."""
    a = 179
    x = make(4, a, torch.float32, 1, weight=False, value=None, share=0.05)
    x["legal"][:, :2] = True
    x["action"][:] = 1
    x["logits"][0, 1] = -100.0
    x["old_logp"][0] = -100.0
    few = call(ext, x)
    many = call(ext, dict(x, legal=x["legal"] | (torch.arange(4) > 0)[:, None]))
    assert few["d_logits"][0].abs().max() > 0.01
    # both carry the errors counted above, below 64 u (4 |l| = 400 in the exponent) of the pull
    assert (few["d_logits"][0] - many["d_logits"][0]).abs().max() <= 2 * (400 + 64) * U


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("a", [3, 20, 40, 64, 100, 179, 300, 600, 1000, 2000, 9000, 40000])
def test_illegal_actions_have_no_gradient_in_rows_that_are_not_finite(ext, a, dtype):
    """NaN or infinite advantages, logits and KL terms, and an illegal action with an infinite
    advantage: the loss shows them, the illegal entries' gradients are 0 all the same, whether few
    of the actions are legal or most."""
    for share in (0.04, 0.9):
        announce(f"not finite {a} {dtype} {share}")
        x = make(5, a, dtype, a, weight=False, share=share)
        x["legal"][:, 0] = True
        x["legal"][:, a // 2] = False
        x["action"][:] = 0
        x["old_logp"][:] = -1.0
        x["advantage"][0] = math.nan
        x["ref"][1, 0] = -math.inf
        x["logits"][2, 0] = math.nan
        x["logits"][3, 0] = math.inf
        x["advantage"][4], x["action"][4] = math.inf, a // 2
        for rows in (range(5), *([i] for i in range(5))):
            keep = list(rows)
            y = {k: v[keep] if isinstance(v, torch.Tensor) else v for k, v in x.items()}
            got = call(ext, y)
            assert not torch.isfinite(got["loss"]), keep
            assert (got["d_logits"].cpu()[~y["legal"]] == 0).all(), keep
            if keep == [0]:
                # so has a legal one without probability, listed or not
                y["logits"], y["legal"] = y["logits"].clone(), y["legal"].clone()
                y["legal"][0, a - 1], y["logits"][0, a - 1] = True, -math.inf
                assert call(ext, y)["d_logits"][0, a - 1] == 0


@pytest.mark.parametrize("a", [1, 3, 40, 64, 179, 300, 1024, 2000])
@pytest.mark.parametrize("n", [0, 1])
def test_one_row_of_a_far_stride(ext, n, a):
    """A single row, or none, has no next one: its stride is of no account, 2^24 elements and more
    included."""
    stride = (1 << 24) + 3
    x = make(1, a, torch.bfloat16, a, weight=False, share=0.9)
    x = {k: v[:n] if isinstance(v, torch.Tensor) else v for k, v in x.items()}
    room = {k: torch.zeros(a, dtype=x[k].dtype, device=DEV) for k in ("logits", "legal", "ref")}
    apart = {}
    for k, t in room.items():
        apart[k] = t.as_strided((n, a), (stride, 1))
        apart[k].copy_(x[k])
    assert n == 0 or apart["logits"].stride(0) == stride
    p, q = call(ext, {**x, **apart}), call(ext, x)
    for k in p:
        assert torch.equal(p[k], q[k]), k
