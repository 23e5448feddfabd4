"""The learner's operators together, as PpoLearner runs them on a rollout."""

from __future__ import annotations

import copy

import pytest
import torch

from oracle import learner_ref as ref
from tests.conftest import announce

pytestmark = pytest.mark.gpu

DEV = "cuda"
SEED_BASE = 0x243F6A8885A308D3


def _rollout(ext, width=512, batch=64, horizon=8):
    from cugo_amd.rollout import MlpRollout, ResidualMlpActor

    torch.manual_seed(1)
    actor = ResidualMlpActor(width, 2).to(DEV, torch.bfloat16)
    g = torch.Generator(device=DEV).manual_seed(2)
    return MlpRollout(ext, actor, batch, horizon, SEED_BASE, g)


@pytest.mark.parametrize("width", [512, 256])
def test_rollout_records_the_player(ext, width):
    """The buffer's player column is observe's player of each step's state."""
    ro = _rollout(ext, width)
    seen = []
    act = ro.act

    def watch(t):
        seen.append(ext.observe(ro.states)[2].clone())
        return act(t)

    ro.act = watch
    buf = ro.collect()
    assert torch.equal(buf.player, torch.stack(seen))
    assert set(buf.player.unique().tolist()) == {0, 1}


@pytest.mark.parametrize("width", [512, 256])
def test_one_update_step_by_step(ext, width):
    """update() over one minibatch of everything: the estimate, the loss, its gradients through
    the actor and the step, each against the oracle on what the one before it gave."""
    from cugo_amd import learner

    announce(f"one update {width}")
    ro = _rollout(ext, width)
    buf = ro.collect()
    lrn = learner.PpoLearner(ro, lr=1e-3, minibatch=1 << 20, kl_coef=0.2, gamma=0.99)
    adv, ret = lrn.estimate()
    features, legal, player, _, _ = ext.observe(ro.states)
    with torch.no_grad():
        value = lrn._value(features.bfloat16())
    want = ref.advantages(buf.reward, buf.value, buf.done, value, 0.99, 0.95, buf.player, player)
    assert (adv.cpu() - want[0]).abs().max() < 1e-4 * (1 + want[0].abs().max())
    assert (ret.cpu() - want[1]).abs().max() < 1e-4 * (1 + want[1].abs().max())
    before = copy.deepcopy(ro.actor)
    stats = lrn.update(torch.Generator(device=DEV).manual_seed(3))
    # the same update by hand: torch's backward of the oracle's gradients, the oracle's AdamW
    n = adv.numel()
    flat = (adv - adv.mean()) / (adv.std(correction=0) + 1e-8)
    order = torch.randperm(n, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    pick = lambda t: t.flatten(0, 1)[order]  # noqa: E731
    x = pick(buf.features)
    logits, v = before(x)
    with torch.no_grad():
        ref_logits = before(x)[0]
    got = ref.policy_loss(logits.detach(), pick(buf.action), pick(buf.logp), pick(flat),
                          pick(buf.legal), ref_logits, v.detach(), pick(ret), None, (0.2, 0.2),
                          0.2, 0.01, 0.5)
    assert abs(stats[0].cpu() - got["loss"]) < 1e-4 * (1 + abs(got["loss"]))
    assert (stats[1:].cpu() - got["stats"]).abs().max() < 1e-4 * (1 + got["stats"].abs().max())
    torch.autograd.backward([logits, v], [got["d_logits"].to(DEV, torch.bfloat16),
                                          got["d_value"].to(DEV, torch.bfloat16)])
    grads = [p.grad for p in before.parameters()]
    norm = torch.cat([g.double().flatten() for g in grads]).norm().cpu()
    # the two backward passes differ where a gradient of the logits is a bf16 step away, which
    # the norm shows at a step's size at most
    assert abs(lrn.optimizer.grad_norm.cpu() - norm) < 2.0**-7 * norm
    clip = min(1.0, 1.0 / (float(lrn.optimizer.grad_norm) + 1e-6))
    for p, q in zip(ro.actor.parameters(), before.parameters()):
        zero = torch.zeros(p.shape)
        w, _, _ = ref.adamw(q.detach(), p.grad, zero, zero, 1, 1e-3, (0.9, 0.999), 1e-8, 0.01, clip)
        master = lrn.optimizer.state[p]["master"]
        assert (master.cpu() - w).abs().max() < 1e-6
        assert torch.equal(p, master.bfloat16())


def test_the_next_rollout_plays_the_new_weights(ext):
    """Updates between captured horizons: the packed weights are the actor's, the replay's records
    come from them, and nothing in the games goes wrong."""
    from cugo_amd import learner
    from cugo_amd.rollout import mlp_forward, pack_actor

    announce("updates between replays")
    ro = _rollout(ext, 512, 256, 16)
    ro.capture()
    lrn = learner.PpoLearner(ro, lr=1e-3, minibatch=1000, epochs=2, state_bits=8, gamma=0.99)
    for k in range(3):
        buf = ro.replay()
        fresh = pack_actor(ext, ro.actor)
        logits, value = mlp_forward(ext, fresh, buf.features[3])
        assert torch.equal(buf.value[3], value)
        ell = logits.float().masked_fill(~buf.legal[3], -1e30).log_softmax(1)
        want = ell.gather(1, buf.action[3][:, None])[:, 0]
        assert (buf.logp[3] - want).abs().max() < 1e-4
        was = [p.detach().clone() for p in ro.actor.parameters()]
        stats = lrn.update()
        assert torch.isfinite(stats).all()
        moved = [not torch.equal(p, q) for p, q in zip(ro.actor.parameters(), was)]
        assert all(moved)
    steps = {int(lrn.optimizer.state[p]["step"]) for p in ro.actor.parameters()}
    assert steps == {3 * 2 * -(-256 * 16 // 1000)}


def test_loss_and_step_captured_together(ext):
    """Logits that are parameters themselves, learnt by replays of one captured loss, backward pass
    and AdamW step, with eager work in between: bit for bit the eager steps on copies."""
    from cugo_amd import learner

    announce("loss and step captured")
    n, a = 300, 179
    g = torch.Generator(device=DEV).manual_seed(4)
    legal = torch.rand(n, a, generator=g, device=DEV) < 0.2
    legal[:, 3] = True
    action = (torch.rand(n, a, generator=g, device=DEV) * legal).argmax(1)
    old = torch.full((n,), -3.0, device=DEV)
    advantage = torch.randn(n, generator=g, device=DEV)
    start = torch.randn(n, a, generator=g, device=DEV)

    def fresh():
        return dict(w=start.bfloat16().requires_grad_(), master=start.clone(),
                    m=torch.zeros(n, a, dtype=torch.float8_e4m3fn, device=DEV),
                    v=torch.zeros(n, a, dtype=torch.float8_e5m2, device=DEV),
                    ms=torch.zeros(-(-n * a // 256), device=DEV),
                    vs=torch.zeros(-(-n * a // 256), device=DEV),
                    steps=torch.zeros(1, dtype=torch.int64, device=DEV))

    def once(s):
        out = learner.policy_loss(ext, s["w"], action, old, advantage, legal=legal,
                                  entropy_coef=0.01)
        grad, = torch.autograd.grad(out.loss, [s["w"]])
        norm = learner.adamw_step(ext, [s["w"]], [grad], [s["m"]], [s["v"]], s["steps"], lr=0.01,
                                  max_norm=0.1, master=[s["master"]], exp_avg_scale=[s["ms"]],
                                  exp_avg_sq_scale=[s["vs"]], seed=3)
        return out.loss.detach(), norm

    eager, played = fresh(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once(played)
    torch.cuda.current_stream().wait_stream(side)
    once(eager)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, norm = once(played)
    for _ in range(6):
        graph.replay()
        want_loss, want_norm = once(eager)
        assert torch.equal(loss, want_loss) and torch.equal(norm, want_norm)
    torch.cuda.synchronize()
    for k in eager:
        assert torch.equal(eager[k].detach().float(), played[k].detach().float()), k
    assert int(played["steps"]) == 7


@pytest.mark.parametrize("width", [512, 256])
def test_a_buffer_without_the_player(ext, width):
    """A RolloutBuffer of the seven columns that it had before `player` still takes a rollout, the
    same one; an update from it is refused, as it cannot tell whose the values are."""
    from cugo_amd import learner
    from cugo_amd.rollout import RolloutBuffer

    announce(f"seven columns {width}")
    one, two = _rollout(ext, width), _rollout(ext, width)
    names = ("features", "legal", "action", "logp", "value", "reward", "done")
    two.buffer = RolloutBuffer(*(torch.empty_like(getattr(one.buffer, k)) for k in names))
    a, b = one.collect(), two.collect()
    for k in names:
        assert torch.equal(getattr(a, k), getattr(b, k)), k
    assert b.player is None
    with pytest.raises(RuntimeError, match="player"):
        learner.PpoLearner(two).update()
