"""advantages against the oracle in 64 bits.

Tolerance, counted before any run: an advantage is a sum of terms d_k (gamma lam)^(k - t), each a
few roundings of its parts; a term passes one multiply-add for each step inside a lane (4 or 8),
each doubling of the scan (6), each wavefront (8 or 16), each pass and each chunk behind it, so u (32 + T / 64)
of the sum of the parts' sizes bounds it, u = 2^-24; returns add one rounding."""

from __future__ import annotations

import pytest
import torch

from oracle import learner_ref as ref
from tests.conftest import announce

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24


def make(t, b, dtype, seed, share=0.05, players=True):
    g = torch.Generator().manual_seed(seed)
    x = dict(reward=torch.randn(t, b, generator=g), value=torch.randn(t, b, generator=g).to(dtype),
             done=torch.rand(t, b, generator=g) < share,
             bootstrap=torch.randn(b, generator=g).to(dtype), player=None, last_player=None)
    if players:
        x["player"] = torch.randint(0, 2, (t, b), generator=g, dtype=torch.uint8)
        x["last_player"] = torch.randint(0, 2, (b,), generator=g, dtype=torch.uint8)
    return x


def call(ext, x, gamma, lam, **out):
    from cugo_amd import learner

    y = {k: v.to(DEV) if v is not None else None for k, v in x.items()}
    return learner.advantages(ext, y["reward"], y["value"], y["done"], y["bootstrap"], gamma, lam,
                              player=y["player"], last_player=y["last_player"], **out)


def check(x, gamma, lam, got):
    adv, ret = ref.advantages(**x, gamma=gamma, lam=lam)
    t = x["reward"].shape[0]
    sizes = {**x, "reward": x["reward"].abs(), "value": -x["value"].abs(),
             "bootstrap": x["bootstrap"].abs(), "player": None, "last_player": None}
    # |r| + |V| + gamma |V'| a step: the value's sign above makes d their sum, the next value's
    # part is put in by hand
    follow = torch.cat([x["value"].double().abs(), x["bootstrap"].double().abs()[None]])[1:]
    sizes["reward"] = (x["reward"].double().abs() + 2 * gamma * follow * ~x["done"])
    part, _ = ref.advantages(**sizes, gamma=gamma, lam=lam)
    tol = U * (32 + t / 64) * part.abs() + 1e-37
    diff = (got[0].cpu().double() - adv).abs()
    assert (diff <= tol).all(), ((diff / tol).max(), diff.max())
    diff = (got[1].cpu().double() - ret).abs()
    assert (diff <= tol + U * ret.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,b", [(1, 1), (1, 70), (2, 5), (7, 3), (8, 64), (9, 65), (63, 33),
                                 (64, 1), (65, 2), (128, 300), (513, 1), (512, 17), (4097, 2),
                                 (1000, 33), (4096, 64), (5000, 3), (20001, 45), (70001, 1),
                                 (129, 40000), (3, 70001), (5, 9), (16, 130), (17, 64), (61, 100),
                                 (65, 700), (127, 65), (130, 64), (200, 31), (600, 500), (257, 9000)])
def test_against_the_oracle(ext, t, b, dtype):
    announce(f"advantages {t}x{b} {dtype}")
    for k, (gamma, lam, share, players) in enumerate([(0.997, 0.95, 0.05, True),
                                                      (1.0, 1.0, 0.002, False),
                                                      (0.9, 0.0, 0.5, True)]):
        if t * b > 100_000 and (k > 0 or dtype == torch.float16):
            continue
        x = make(t, b, dtype, t + b + k, share, players)
        check(x, gamma, lam, call(ext, x, gamma, lam))


def test_nothing_passes_a_done_step(ext):
    """NaN and infinities in the next game's rewards and values, and in the bootstrap, stay there."""
    for t, b in ((40, 7), (600, 3), (3000, 1)):
        x = make(t, b, torch.float32, t, share=0.0)
        half = t // 2
        x["done"][half] = True
        x["reward"][half + 1:] = float("nan")
        x["value"][half + 1:] = float("inf")
        x["bootstrap"][:] = float("nan")
        got = call(ext, x, 0.99, 0.95)
        front = {k: v[:half + 1] if v is not None and v.dim() == 2 else v for k, v in x.items()}
        front["bootstrap"] = torch.zeros(b)
        check(front, 0.99, 0.95, [g[:half + 1] for g in got])
        x["done"][-1] = True
        x["reward"][half + 1:] = 1.0
        x["value"][half + 1:] = 1.0
        got = call(ext, x, 0.99, 0.95)
        assert torch.isfinite(got[0]).all() and torch.isfinite(got[1]).all()


def test_nothing_passes_a_factor_of_zero(ext):
    """With lam = 0 a step reads the next one's value alone, not what becomes of it."""
    for t, b in ((40, 70), (700, 3), (3000, 100)):
        x = make(t, b, torch.float32, t, share=0.0)
        x["reward"][5::9] = float("nan")
        adv, _ = call(ext, x, 0.99, 0.0)
        bad = torch.isnan(x["reward"])
        assert torch.equal(torch.isnan(adv).cpu(), bad)
        y = dict(x, reward=x["reward"].nan_to_num(nan=0.0))
        check({k: v[:5] if v.dim() == 2 else v for k, v in y.items()} | {
            "bootstrap": y["value"][5], "last_player": y["player"][5]}, 0.99, 0.0,
            [z[:5] for z in call(ext, x, 0.99, 0.0)])


def test_what_is_not_finite_shows_however_far_ahead(ext):
    """gamma lam to the power of the steps between is far below the least float32: a NaN or an
    infinity is still in every step before it, as in the recurrence, up to the game's beginning."""
    for t, b, decay in ((400, 70, 0.5), (3000, 1, 0.9), (2000, 3, 1e-3), (5000, 45, 0.25),
                        (1200, 2, 1e-30)):
        x = make(t, b, torch.float32, t, share=0.0)
        x["done"][t // 3] = True
        x["reward"][t - 7, 0] = float("nan")
        if b > 1:
            x["reward"][t - 3, 1] = float("inf")
            x["value"][t - 9, b - 1] = float("nan")
        adv, _ = call(ext, x, 1.0, decay)
        want, _ = ref.advantages(**x, gamma=1.0, lam=decay)
        assert torch.equal(torch.isfinite(adv).cpu(), torch.isfinite(want)), (t, b, decay)
        assert torch.equal(torch.isnan(adv).cpu(), torch.isnan(want)), (t, b, decay)


def test_outputs_streams_graphs(ext):
    """Results in given tensors; a side stream; captured and replayed on new inputs."""
    xs = [make(700, 5, torch.float32, 20 + k) for k in range(3)]
    want = [call(ext, x, 0.99, 0.9) for x in xs]
    at = {k: v.to(DEV) for k, v in xs[0].items()}
    adv, ret = torch.full((700, 5), 7.0, device=DEV), torch.full((700, 5), 7.0, device=DEV)

    def once():
        return ext.advantages(at["reward"], at["value"], at["done"], at["bootstrap"], 0.99, 0.9,
                              at["player"], at["last_player"], adv, ret)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    torch.cuda.current_stream().wait_stream(side)
    assert got[0].data_ptr() == adv.data_ptr() and got[1].data_ptr() == ret.data_ptr()
    assert torch.equal(adv, want[0][0]) and torch.equal(ret, want[0][1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        once()
    for k in (1, 2, 0, 1):
        for name, t in at.items():
            t.copy_(xs[k][name])
        graph.replay()
        again = call(ext, xs[k], 0.99, 0.9)
        assert torch.equal(adv, again[0]) and torch.equal(ret, again[1])
        assert torch.equal(again[0], want[k][0])


def test_offsets_past_32_bits(ext):
    """More than 2^31 steps: the last games are those of a call on them alone."""
    t, b = 70, 31_000_001
    announce(f"advantages {t}x{b}")
    g = torch.Generator(device=DEV).manual_seed(3)
    reward = torch.empty(t, b, device=DEV).normal_(generator=g)
    value = torch.empty(t, b, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    done = torch.zeros(t, b, dtype=torch.bool, device=DEV)
    done[30] = True
    bootstrap = torch.ones(b, dtype=torch.bfloat16, device=DEV)
    adv, ret = ext.advantages(reward, value, done, bootstrap, 0.99, 0.95)
    for cols in (slice(0, 100), slice(b // 2, b // 2 + 100), slice(b - 100, b)):
        part = [x[..., cols].contiguous() for x in (reward, value, done, bootstrap)]
        a, r = ext.advantages(*part, 0.99, 0.95)
        diff = torch.maximum((adv[:, cols] - a).abs().max(), (ret[:, cols] - r).abs().max())
        assert diff < 1e-4, diff  # another split of the steps: other roundings of sums below 100


def test_empty(ext):
    for t, b in ((0, 5), (5, 0), (0, 0)):
        x = make(t, b, torch.float32, 1)
        adv, ret = call(ext, x, 0.9, 0.9)
        assert adv.shape == (t, b) and ret.shape == (t, b)


def test_refusals(ext):
    from cugo_amd import learner

    x = {k: v.to(DEV) for k, v in make(6, 4, torch.float32, 1).items()}

    def go(gamma=0.9, lam=0.9, **over):
        y = {**x, **over}
        return learner.advantages(ext, y["reward"], y["value"], y["done"], y["bootstrap"], gamma,
                                  lam, player=y["player"], last_player=y["last_player"],
                                  advantage=y.get("advantage"))

    go()
    for over in (dict(reward=x["reward"].cpu()), dict(reward=x["reward"].double()),
                 dict(reward=x["reward"].t()), dict(value=x["value"][:5]),
                 dict(value=x["value"].double()), dict(done=x["done"].byte()),
                 dict(done=x["done"].t().contiguous().t()), dict(bootstrap=x["bootstrap"].half()),
                 dict(bootstrap=x["bootstrap"][:3]), dict(player=None), dict(last_player=None),
                 dict(player=x["player"].long()), dict(gamma=1.5), dict(lam=-0.1),
                 dict(advantage=x["reward"]), dict(advantage=x["value"]),
                 dict(advantage=torch.empty(4, 6, device=DEV)),
                 dict(advantage=torch.empty(6, 4, device=DEV, dtype=torch.float64))):
        with pytest.raises(RuntimeError):
            go(**over)
