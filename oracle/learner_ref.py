"""The learner's operators from their definitions, in 64 bits (torch, any device).

`policy_loss` and its gradient formula, `advantages` step by step, `adamw` value by value with
the 8-bit moments' rounding (codes, scales and words) spelled out in integers."""

from __future__ import annotations

import math

import torch

MASK = 0xFFFFFFFF
BLOCK = 256


def log_softmax(z):
    """Shifted first: beside logits of float32's lowest value a logarithm is lost even here."""
    z = z - z.max(-1, keepdim=True).values
    return z - z.logsumexp(-1, keepdim=True)


def policy_loss(logits, action, old_logp, advantage, legal=None, ref=None, value=None,
                returns=None, weight=None, clip=(0.2, 0.2), kl_coef=0.0, entropy_coef=0.0,
                value_coef=0.5, scale=1.0):
    """A dict of loss, stats [6], logp [n], d_logits [n, A] and d_value [n], all float64, row by
    row over the legal entries alone."""
    n, a = logits.shape
    z = logits.double().cpu()
    on = torch.ones(n, a, dtype=torch.bool) if legal is None else legal.cpu()
    q = None if ref is None else ref.double().cpu()
    w = torch.full((n,), 1.0 / n, dtype=torch.float64) if weight is None else weight.double().cpu()
    act, old, adv = action.cpu(), old_logp.double().cpu(), advantage.double().cpu()
    stats = torch.zeros(6, dtype=torch.float64)
    logp = torch.zeros(n, dtype=torch.float64)
    d_logits = torch.zeros(n, a, dtype=torch.float64)
    d_value = torch.zeros(n, dtype=torch.float64)
    for i in range(n):
        idx = on[i].nonzero()[:, 0]
        zi = z[i, idx]
        if value is not None and w[i] != 0:
            err = value[i].double().cpu() - returns[i].double().cpu()
            stats[1] += w[i] * 0.5 * err**2
            d_value[i] = scale * w[i] * value_coef * err
        if len(idx) == 0 or bool((zi == -math.inf).all()):
            continue
        ell = log_softmax(zi)
        p = ell.exp()
        has = p > 1e-46  # what float32 holds beside the row's largest
        where = (idx == act[i]).nonzero()[:, 0]
        lp = ell[where[0]] if len(where) else torch.tensor(-math.inf, dtype=torch.float64)
        logp[i] = lp
        if w[i] == 0:
            continue
        entropy = -torch.where(has, p * ell, 0.0).sum()
        kl = torch.zeros((), dtype=torch.float64)
        d = torch.zeros_like(p)
        if q is not None:
            qi = q[i, idx]
            d = torch.where(has, ell - log_softmax(qi), 0.0)
            kl = torch.where(has, p * d, 0.0).sum()
        drift = lp - old[i]
        r = torch.zeros(()).double() if lp == -math.inf else drift.exp()
        bound = r.clamp(1 - clip[0], 1 + clip[1])
        cut = bool(r * adv[i] > bound * adv[i])
        gain = bound * adv[i] if cut else r * adv[i]
        stats[0] += w[i] * -gain
        stats[2] += w[i] * kl
        stats[3] += w[i] * entropy
        stats[4] += w[i] * cut
        stats[5] += w[i] * (r - 1 - drift)
        pull = 0.0 if cut else float(r * adv[i])
        g = pull * p + kl_coef * torch.where(has, p * (d - kl), 0.0)
        g = g + entropy_coef * torch.where(has, p * (ell + entropy), 0.0)
        if len(where):
            g[where[0]] -= pull
        d_logits[i, idx] = scale * w[i] * g
    loss = stats[0] + value_coef * stats[1] + kl_coef * stats[2] - entropy_coef * stats[3]
    return {"loss": scale * loss, "stats": stats, "logp": logp, "d_logits": d_logits,
            "d_value": d_value}


def advantages(reward, value, done, bootstrap, gamma, lam, player=None, last_player=None):
    """(advantage, returns), float64, from the last step back."""
    steps, batch = reward.shape
    reward, done = reward.double().cpu(), done.cpu()
    v = torch.cat([value.double().cpu(), bootstrap.double().cpu()[None]])
    who = (torch.zeros(steps + 1, batch) if player is None
           else torch.cat([player.cpu(), last_player.cpu()[None]]))
    s = 1.0 - 2.0 * (who != 0).double()
    a = torch.zeros(batch, dtype=torch.float64)
    out = torch.zeros(steps, batch, dtype=torch.float64)
    for t in reversed(range(steps)):
        follow = torch.where(done[t], 0.0, s[t + 1] * v[t + 1])
        a = reward[t] + gamma * follow - s[t] * v[t] + torch.where(done[t], 0.0, gamma * lam * a)
        out[t] = s[t] * a
    return out, out + v[:-1]


def mix(x: int) -> int:
    x &= MASK
    x = ((x ^ (x >> 17)) * 0x9E3779B9) & MASK
    x = ((x ^ (x >> 14)) * 0xBB67AE85) & MASK
    return x ^ (x >> 15)


def word(seed: int, place: int, step: int, index: int) -> int:
    """The 32 bits that round value `index` of the tensor at `place` at `step`."""
    k = mix((seed & MASK) ^ mix(((seed >> 32) & MASK) + 1))
    k = mix(mix(k + place) + (step & MASK))
    return mix((index & MASK) ^ mix(k + (index >> 32) * 0x9E3779B9))


def words(seed: int, place: int, step: int, count: int) -> torch.Tensor:
    """word() of indices 0 .. count - 1, int64."""
    k = mix((seed & MASK) ^ mix(((seed >> 32) & MASK) + 1))
    k = mix(mix(mix(k + place) + (step & MASK)))
    x = torch.arange(count) ^ k
    x = ((x ^ (x >> 17)) * 0x9E3779B9) & MASK
    x = ((x ^ (x >> 14)) * 0xBB67AE85) & MASK
    return x ^ (x >> 15)


def code(y: float, bits: int, mantissa: int, least: int) -> int:
    """y >= 0 as a code with `mantissa` bits and smallest normal value 2^least, rounded up with
    the chance of what is cut off: bits / 2^32 of the last place is added, then cut."""
    if y == 0:
        return 0
    e = max(math.frexp(y)[1] - 1, least)  # y in [2^e, 2^(e + 1)), or below the normal values
    drop = 23 - mantissa
    units = int(y * 2.0 ** (23 - e))      # in steps of 2^(e - 23), as float32 holds it
    kept = (units + (bits >> (32 - drop))) >> drop
    return kept + (e - least) * 2**mantissa


def value_of(c: int, mantissa: int, least: int) -> float:
    exponent, fraction = c >> mantissa, c & (2**mantissa - 1)
    if exponent == 0:
        return fraction * 2.0 ** (least - mantissa)
    return (1 + fraction / 2**mantissa) * 2.0 ** (least + exponent - 1)


def adamw(w, g, m, v, t, lr, betas, eps, weight_decay, clip=1.0):
    """(w, m, v) after step t (1 for the first), float64."""
    w, g, m, v = (x.double().cpu() for x in (w, g, m, v))
    g = g * clip
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    hat_m, hat_v = m / (1 - betas[0] ** t), v / (1 - betas[1] ** t)
    return w - lr * (weight_decay * w + hat_m / (hat_v.sqrt() + eps)), m, v
