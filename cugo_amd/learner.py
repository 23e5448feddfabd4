"""What learns from a rollout: advantages, the policy loss with its gradients, AdamW.

The reference's PPO update (python/cugo_ppo50.py:514-739) runs these in torch operations; here
each is HIP kernels behind one call:

  * `advantages`: generalised advantage estimation over a horizon of two-player games, each
    decision seen from its mover's side; the rollout buffer's columns are read once, or twice
    where few games over many steps are split over the device;
  * `policy_loss`: the clipped policy loss over each row's legal actions with a KL term to
    another policy, an entropy bonus and the value loss.  The loss and the gradients of the
    logits and the value come from one reading of the logits (two of rows of over 32,768
    actions, 16,384 in float32); `backward()` hands the gradients on (multiplied by the loss's
    own gradient where that is not 1);
  * `adamw_step`: one AdamW step over many tensors at once, the gradients' norm clipped, the
    moments in float32 or in 8 bits; `AdamW` is the torch optimizer over it.

`PpoLearner` is the update of a `MlpRollout`'s actor from its buffer.  Everything runs on the
current stream without synchronising and can be captured in a HIP graph.
"""

from __future__ import annotations

import copy
import importlib
from typing import NamedTuple, Sequence

import torch

from .rollout import MlpRollout, fused_forward, mlp_forward

STATS = ("policy", "value", "kl", "entropy", "cut", "drift")


# ------------------------------------------------------------------------------- the loss


class PolicyLoss(NamedTuple):
    """`loss`: float32 scalar, differentiable in the logits and the value.  `stats`: float32
    [6], the weighted sums named in STATS (cut: the weight of rows whose ratio the clip cut
    off; drift: of r - 1 - log r, an estimate of the KL from the collecting policy).  `logp`:
    float32 [n], the actions' log-probabilities now."""

    loss: torch.Tensor
    stats: torch.Tensor
    logp: torch.Tensor


def policy_loss(ext, logits: torch.Tensor, action: torch.Tensor, old_logp: torch.Tensor,
                advantage: torch.Tensor, *, legal: torch.Tensor | None = None,
                ref_logits: torch.Tensor | None = None, value: torch.Tensor | None = None,
                returns: torch.Tensor | None = None, weight: torch.Tensor | None = None,
                clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0,
                entropy_coef: float = 0.0, value_coef: float = 0.5,
                loss_scale: torch.Tensor | None = None) -> PolicyLoss:
    """The loss of n decisions over A actions:

        sum_i w_i [ -min(r A, clip(r, 1 - clip[0], 1 + clip[1]) A) + value_coef (V - R)^2 / 2
                    + kl_coef KL(p || p_ref) - entropy_coef H(p) ],  r = exp(log p_a - old_logp)

    logits [n, A] float32, float16 or bfloat16 (any distance between rows); action int64 [n];
    old_logp and advantage float32 [n]; legal bool [n, A] (None: every action is); ref_logits
    like logits (None: no KL term); value [n] (any of the three types) with returns float32
    [n]; weight float32 [n] (None: 1 / n each).  Gradients reach logits and value, rounded once
    to their types (and once more where the loss's own gradient is not 1).

    A row of weight 0 counts nowhere and gets zero gradients, whatever it holds.  A row
    without a legal action has only the value term (its logp is 0).  An illegal action has
    log-probability -inf, ratio 0 and no gradient.  NaN in a legal logit shows in the loss; what
    illegal entries hold is never used.

    loss_scale (a one-element float32 tensor on the device) multiplies the loss and its
    gradients before they are rounded, as float16 gradients need: call `backward()` on the
    scaled loss directly.  The gradients are handed out by one backward pass; a second pass
    through the same loss raises."""
    return PolicyLoss(*ext.policy_loss(logits, action, old_logp, advantage, legal, ref_logits,
                                       value, returns, weight, clip[0], clip[1], kl_coef,
                                       entropy_coef, value_coef, loss_scale))


# ------------------------------------------------------------------------------- advantages


def advantages(ext, reward: torch.Tensor, value: torch.Tensor, done: torch.Tensor,
               bootstrap: torch.Tensor, gamma: float, lam: float, *,
               player: torch.Tensor | None = None, last_player: torch.Tensor | None = None,
               advantage: torch.Tensor | None = None, returns: torch.Tensor | None = None
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """Generalised advantage estimation over [steps, batch] decisions of two-player games:
    (advantage, returns), float32, returns = advantage + value.

    reward float32 is player 0's (the rollout buffer's column); value (float32, float16 or
    bfloat16) is the mover's estimate before the step; player uint8 says who moves (None: one
    player); done bool ends a game with the step, and nothing after it is read into it.
    bootstrap [batch] (value's type) and last_player [batch] belong to the state behind the last
    step.  Advantages and returns are the mover's.  `advantage` and `returns`, if given,
    receive the results; they must not overlap the inputs."""
    return tuple(ext.advantages(reward, value.detach(), done, bootstrap.detach(), gamma, lam,
                                player, last_player, advantage, returns))


# ------------------------------------------------------------------------------- AdamW


def _each(x: float | Sequence[float], n: int) -> list[float]:
    return [float(x)] * n if isinstance(x, (int, float)) else [float(v) for v in x]


@torch.no_grad()
def adamw_step(ext, params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor | None],
               exp_avg: Sequence[torch.Tensor], exp_avg_sq: Sequence[torch.Tensor],
               steps: torch.Tensor, *, lr: float | Sequence[float],
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
               weight_decay: float | Sequence[float] = 0.01, max_norm: float | None = None,
               master: Sequence[torch.Tensor | None] | None = None,
               exp_avg_scale: Sequence[torch.Tensor] | None = None,
               exp_avg_sq_scale: Sequence[torch.Tensor] | None = None,
               lr_scale: torch.Tensor | None = None, seed: int = 0) -> torch.Tensor | None:
    """One AdamW step of all parameters, in place; with max_norm, the gradients are scaled
    down to that norm (over all of them together) and their norm is returned (a float32 scalar
    on the device).

    params and grads are contiguous float32, float16 or bfloat16 (a grad of None leaves its
    parameter and state as they are); a 16-bit parameter has a float32 `master`, which the step
    updates and the parameter is rounded from.  steps int64 [n] counts each parameter's steps on
    the device.  lr and weight_decay are numbers or one for each parameter; lr_scale, a
    one-element float32 tensor on the device, multiplies every lr (a schedule inside a captured
    graph).  exp_avg and exp_avg_sq are float32, or with exp_avg_scale and exp_avg_sq_scale
    float8_e4m3fn and float8_e5m2 codes of the moment over its block's scale (float32, one for
    each ADAMW_BLOCK = 256 values); the codes are rounded stochastically, by bits that follow
    from `seed`, the parameter's place in the list, its step and the value's index."""
    n = len(params)
    return ext.adamw_step(list(params), list(grads), list(exp_avg), list(exp_avg_sq), steps,
                          _each(lr, n), _each(weight_decay, n), betas[0], betas[1], eps, max_norm,
                          None if master is None else list(master),
                          None if exp_avg_scale is None else list(exp_avg_scale),
                          None if exp_avg_sq_scale is None else list(exp_avg_sq_scale),
                          lr_scale, seed)


def _of_all_groups(name: str) -> property:
    """An option that one step has once: a group's entry, the same in every group."""

    def get(self):
        first, *others = (g[name] for g in self.param_groups)
        plain = tuple(first) if isinstance(first, (list, tuple)) else first
        for x in others:
            if x is not first and (tuple(x) if isinstance(x, (list, tuple)) else x) != plain:
                raise ValueError(f"{name} must be the same for every group")
        return plain

    def put(self, value) -> None:
        for g in self.param_groups:
            g[name] = value

    return property(get, put)


class AdamW(torch.optim.Optimizer):
    """AdamW over `adamw_step`: one call for all parameters of all groups.

    Groups may set lr and weight_decay.  betas, eps, max_norm and seed are in the groups too
    (for schedulers and checkpoints), the same in every one, as an lr that is a one-element
    float32 tensor on the device is.  state_bits 32 keeps the moments in float32, 8 in 8 bits
    (about 2 bytes a value instead of 8).  16-bit parameters get a float32 master in the state.
    `grad_norm` is the last step's norm when max_norm is set."""

    def __init__(self, ext, params, lr: float | torch.Tensor = 3e-4,
                 betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, max_norm: float | None = None,
                 state_bits: int = 32, seed: int = 0) -> None:
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        self.ext, self.state_bits = ext, state_bits
        self.grad_norm: torch.Tensor | None = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay,
                                      max_norm=max_norm, seed=seed))
        self._steps: torch.Tensor | None = None

    betas, eps = _of_all_groups("betas"), _of_all_groups("eps")
    max_norm, seed = _of_all_groups("max_norm"), _of_all_groups("seed")

    def _options(self) -> dict:
        return {k: getattr(self, k) for k in ("betas", "eps", "max_norm", "seed")}

    def add_param_group(self, param_group: dict) -> None:
        if hasattr(self, "_steps"):  # made already: the options as they are now
            param_group = {**self._options(), **param_group}
        o = {**self.defaults, **param_group}
        for name in ("lr", "weight_decay", "eps"):
            if not isinstance(o[name], torch.Tensor) and not o[name] >= 0:
                raise ValueError(f"{name} must not be negative: {o[name]}")
        if not all(0 <= b < 1 for b in o["betas"]):
            raise ValueError(f"betas must lie in [0, 1): {o['betas']}")
        if o["max_norm"] is not None and not o["max_norm"] > 0:
            raise ValueError(f"max_norm must be positive: {o['max_norm']}")
        super().add_param_group(param_group)

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), "state_bits": self.state_bits,
                "grad_norm": self.grad_norm, "extension": self.ext.__name__}

    def __setstate__(self, state: dict) -> None:
        """Of a copy (the extension is found again by its name), or of the base class's
        load_state_dict, which passes state and groups alone."""
        state = dict(state)
        if "extension" in state:
            self.ext = importlib.import_module(state.pop("extension"))
        super().__setstate__(state)
        self._steps = None  # gathered again from the parameters' own counts

    def _all(self) -> list[torch.Tensor]:
        return [p for g in self.param_groups for p in g["params"]]

    def _new_state(self, p: torch.Tensor) -> dict:
        s = {}
        if self.state_bits == 8:
            blocks = -(-p.numel() // self.ext.ADAMW_BLOCK)
            s["exp_avg"] = torch.zeros(p.shape, dtype=torch.float8_e4m3fn, device=p.device)
            s["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float8_e5m2, device=p.device)
            s["exp_avg_scale"] = torch.zeros(blocks, device=p.device)
            s["exp_avg_sq_scale"] = torch.zeros(blocks, device=p.device)
        else:
            s["exp_avg"] = torch.zeros(p.shape, device=p.device)
            s["exp_avg_sq"] = torch.zeros(p.shape, device=p.device)
        if p.dtype != torch.float32:
            s["master"] = p.detach().float()
        return s

    @torch.no_grad()
    def prepare(self) -> None:
        """Creates the state of parameters that have none (the first `step` does; call it before
        capturing one)."""
        params = self._all()
        if (self._steps is not None and self._steps.numel() == len(params)
                and all(p in self.state for p in params)):
            return
        steps = torch.zeros(len(params), dtype=torch.int64, device=params[0].device)
        for i, p in enumerate(params):
            s = self.state[p]
            if not s:
                s.update(self._new_state(p))
            if "step" in s:
                steps[i] = s["step"]
            s["step"] = steps[i]
        self._steps = steps

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self.prepare()
        params = self._all()
        states = [self.state[p] for p in params]
        lrs = [g["lr"] for g in self.param_groups for _ in g["params"]]
        scale = None
        if any(isinstance(x, torch.Tensor) for x in lrs):
            scale = lrs[0]
            if any(x is not scale for x in lrs):
                raise ValueError("an lr tensor must be the same for every group")
            lrs = [1.0] * len(params)
        grads = []
        for p in params:
            if p.grad is not None and p.grad.is_sparse:
                raise RuntimeError("AdamW does not take sparse gradients")
            grads.append(None if p.grad is None else p.grad.contiguous())
        eight = self.state_bits == 8
        self.grad_norm = adamw_step(
            self.ext, params, grads, [s["exp_avg"] for s in states],
            [s["exp_avg_sq"] for s in states], self._steps, lr=lrs, betas=self.betas,
            eps=self.eps,
            weight_decay=[g["weight_decay"] for g in self.param_groups for _ in g["params"]],
            max_norm=self.max_norm, master=[s.get("master") for s in states],
            exp_avg_scale=[s["exp_avg_scale"] for s in states] if eight else None,
            exp_avg_sq_scale=[s["exp_avg_sq_scale"] for s in states] if eight else None,
            lr_scale=scale, seed=self.seed)
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        """The base class would convert the state to the parameters' types; here every entry
        keeps its own.  A state that does not fit is refused before anything is changed."""
        saved = state_dict["state"]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        states = []
        for i, p in zip(ids, self._all()):
            if i not in saved:
                continue
            fresh = self._new_state(p)
            for name, t in fresh.items():
                got = saved[i].get(name)
                if got is None or got.shape != t.shape or got.dtype != t.dtype:
                    raise ValueError(f"the saved state's {name} does not fit the parameter")
                t.copy_(got)
            if "step" not in saved[i]:
                raise ValueError("the saved state has no step")
            fresh["step"] = torch.as_tensor(saved[i]["step"], dtype=torch.int64).clone()
            states.append((p, fresh))
        # an option that the saved groups do not have stays as it is
        groups = [{**self._options(), **g} for g in state_dict["param_groups"]]
        super().load_state_dict({"state": {}, "param_groups": groups})
        self.state.clear()
        for p, fresh in states:
            self.state[p].update(fresh)


# ------------------------------------------------------------------------------- the update


class PpoLearner:
    """PPO updates of a rollout's actor from its buffer (the reference's update,
    python/cugo_ppo50.py:514-739, over `MlpRollout`'s columns).

    `update()` estimates the advantages of the buffer's horizon, runs `epochs` passes over its
    decisions in shuffled minibatches (the actor's forward and backward pass through torch,
    `policy_loss`, one AdamW step each) and packs the new weights for the next rollout.  With
    kl_coef, the KL term holds the policy to the one that the last `set_reference()` kept."""

    def __init__(self, ro: MlpRollout, lr: float | torch.Tensor = 3e-4, minibatch: int = 16384,
                 epochs: int = 1, gamma: float = 1.0, lam: float = 0.95,
                 clip: tuple[float, float] = (0.2, 0.2), kl_coef: float = 0.0,
                 entropy_coef: float = 0.01, value_coef: float = 0.5,
                 weight_decay: float = 0.01, max_norm: float | None = 1.0,
                 state_bits: int = 32, seed: int = 0) -> None:
        self.ro, self.ext = ro, ro.ext
        self.minibatch, self.epochs = minibatch, epochs
        self.gamma, self.lam = gamma, lam
        self.loss_args = dict(clip=clip, kl_coef=kl_coef, entropy_coef=entropy_coef,
                              value_coef=value_coef)
        self.optimizer = AdamW(ro.ext, ro.actor.parameters(), lr=lr, weight_decay=weight_decay,
                               max_norm=max_norm, state_bits=state_bits, seed=seed)
        self.reference = None
        if kl_coef:
            self.set_reference()
        batch = ro.batch
        dev = ro.buffer.features.device
        self._features = torch.empty((batch, ro.buffer.features.shape[2]), dtype=torch.bfloat16,
                                     device=dev)

    def set_reference(self) -> None:
        """Keeps a copy of the actor as it is now for the KL term."""
        self.reference = copy.deepcopy(self.ro.actor).requires_grad_(False)

    @torch.no_grad()
    def _value(self, x: torch.Tensor) -> torch.Tensor:
        if self.ro.fused_kernel:
            return mlp_forward(self.ext, self.ro.packed, x)[1]
        return fused_forward(self.ext, self.ro.actor, x)[1].float()

    @torch.no_grad()
    def estimate(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(advantage, returns) [horizon, batch] of the buffer, the games' states now being
        those behind its last step."""
        buf = self.ro.buffer
        now = self.ext.observe_bf16(self.ro.states, self._features)
        return advantages(self.ext, buf.reward, buf.value, buf.done, self._value(self._features),
                          self.gamma, self.lam, player=buf.player, last_player=now[2])

    def update(self, generator: torch.Generator | None = None) -> torch.Tensor:
        """One update; the minibatches' mean loss and stats, float32 [7] on the device."""
        buf, actor = self.ro.buffer, self.ro.actor
        advantage, returns = (x.flatten() for x in self.estimate())
        mean, std = advantage.mean(), advantage.std(correction=0)
        advantage = (advantage - mean) / (std + 1e-8)
        features, legal = buf.features.flatten(0, 1), buf.legal.flatten(0, 1)
        action, old_logp = buf.action.flatten(), buf.logp.flatten()
        n = action.numel()
        total, count = torch.zeros(7, device=action.device), 0
        for _ in range(self.epochs):
            order = torch.randperm(n, generator=generator, device=action.device)
            for part in order.split(self.minibatch):
                x = features[part]
                logits, value = actor(x)
                ref = None
                if self.reference is not None:
                    with torch.no_grad():
                        ref, _ = self.reference(x)
                out = policy_loss(self.ext, logits, action[part], old_logp[part],
                                  advantage[part], legal=legal[part], ref_logits=ref, value=value,
                                  returns=returns[part], **self.loss_args)
                self.optimizer.zero_grad()
                out.loss.backward()
                self.optimizer.step()
                total[0] += out.loss.detach()
                total[1:] += out.stats
                count += 1
        self.ro.repack()
        return total / max(count, 1)
