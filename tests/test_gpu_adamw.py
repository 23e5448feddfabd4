"""adamw_step and AdamW against the oracle in 64 bits.

Tolerances, counted before any run, u = 2^-24: a moment is three rounded float32 operations on
values of the sizes |b m| and |(1 - b) g| (and g's scaling by the clip, two more): 6 u of their
sum.  The step has the moment's error, a square root, two products, a sum and a quotient, 16 u of
its size, and 3 u of the weight.  8-bit codes are compared exactly: the float32 values before the
rounding follow from IEEE operations in the documented order, which torch's CPU operations
repeat."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import learner_ref as ref
from tests.conftest import announce

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0**-24
BETAS, EPS = (0.9, 0.999), 1e-8
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def make(sizes, param, grad, seed, bits=32, scale=1e-2):
    """Tensors on the device and float32 copies of what they hold on the CPU."""
    g = torch.Generator().manual_seed(seed)
    x = dict(params=[], grads=[], exp_avg=[], exp_avg_sq=[], master=[], exp_avg_scale=[],
             exp_avg_sq_scale=[])
    for n in sizes:
        w = torch.randn(n, generator=g)
        size = torch.exp(2 * torch.randn(n, generator=g)) * scale
        x["params"].append(w.to(param))
        x["grads"].append((torch.randn(n, generator=g) * size).to(grad))
        x["master"].append(None if param == torch.float32 else w)
        m, v = torch.randn(n, generator=g) * size, (torch.randn(n, generator=g) * size) ** 2
        if bits == 8:
            for name, y, top, dt in (("exp_avg", m, 256.0, torch.float8_e4m3fn),
                                     ("exp_avg_sq", v, 32768.0, torch.float8_e5m2)):
                pad = torch.nn.functional.pad(y, (0, -n % ref.BLOCK)).view(-1, ref.BLOCK)
                s = pad.abs().amax(1).clamp_min(2.0**-100) / top
                x[name].append((pad / s[:, None]).view(-1)[:n].to(dt))
                x[name + "_scale"].append(s)
        else:
            x["exp_avg"].append(m)
            x["exp_avg_sq"].append(v)
    x["steps"] = torch.arange(len(sizes)) * 7
    return x


def to_device(x):
    move = lambda v: v if v is None else v.to(DEV)  # noqa: E731
    y = {k: move(v) if not isinstance(v, list) else [move(t) for t in v] for k, v in x.items()}
    if all(t is None for t in y["master"]):
        y["master"] = None
    if not y["exp_avg_scale"]:
        y["exp_avg_scale"] = y["exp_avg_sq_scale"] = None
    return y


def step(ext, y, **over):
    from cugo_amd import learner

    args = dict(lr=3e-3, betas=BETAS, eps=EPS, weight_decay=0.1, master=y["master"],
                exp_avg_scale=y["exp_avg_scale"], exp_avg_sq_scale=y["exp_avg_sq_scale"], seed=77)
    return learner.adamw_step(ext, y["params"], y["grads"], y["exp_avg"], y["exp_avg_sq"],
                              y["steps"], **{**args, **over})


def moments(x, i):
    """Tensor i's moments as the float32 values they stand for."""
    m, v = x["exp_avg"][i], x["exp_avg_sq"][i]
    if not x["exp_avg_scale"]:
        return m, v
    n = m.numel()
    wide = lambda s: s.repeat_interleave(ref.BLOCK)[:n]  # noqa: E731
    return m.float() * wide(x["exp_avg_scale"][i]), v.float() * wide(x["exp_avg_sq_scale"][i])


def check(x, y, norm, max_norm=None, lr=3e-3, weight_decay=0.1, seed=77):
    grads64 = torch.cat([g.double().flatten() for g in x["grads"] if g is not None])
    clip, clip32 = 1.0, None
    if max_norm is not None:
        want = grads64.norm()
        assert abs(norm.cpu().double() - want) <= 4 * U * want
        clip = min(1.0, max_norm / (float(want) + 1e-6))
        clip32 = (max_norm / (norm.cpu() + 1e-6)).clamp_max(1.0)
    else:
        assert norm is None
    for i, g in enumerate(x["grads"]):
        n = x["params"][i].numel()
        if g is None:
            for k in ("params", "exp_avg", "exp_avg_sq", "steps", "master"):
                if y[k] is not None and y[k][i] is not None:
                    assert torch.equal(y[k][i].cpu(), x[k][i])
            continue
        t = int(x["steps"][i]) + 1
        assert int(y["steps"][i]) == t
        m0, v0 = moments(x, i)
        w0 = x["master"][i] if x["master"][i] is not None else x["params"][i]
        each = lambda z: z[i] if isinstance(z, list) else z  # noqa: E731
        w, m, v = ref.adamw(w0, g, m0, v0, t, each(lr), BETAS, EPS, each(weight_decay), clip)
        g64 = g.double().abs() * clip
        tol_m = 6 * U * (0.9 * m0.double().abs() + 0.1 * g64) + 1e-45
        tol_v = 8 * U * (0.999 * v0.double() + 0.001 * g64**2) + 1e-44
        root = (v / (1 - 0.999**t)).sqrt() + EPS
        move = each(lr) * (m.abs() + tol_m) / (1 - 0.9**t) / root
        tol_w = 3 * U * w.abs() + 16 * U * move + each(lr) * tol_m / (1 - 0.9**t) / root * 2 + 1e-45
        got = (y["master"][i] if y["master"] is not None and y["master"][i] is not None
               else y["params"][i]).cpu()
        diff = (got.double() - w).abs()
        assert (diff <= tol_w).all(), (i, n, (diff / tol_w).max())
        if x["master"][i] is not None:
            assert torch.equal(y["params"][i].cpu(), got.to(y["params"][i].dtype))
        if not x["exp_avg_scale"]:
            assert ((y["exp_avg"][i].cpu().double() - m).abs() <= tol_m).all()
            assert ((y["exp_avg_sq"][i].cpu().double() - v).abs() <= tol_v).all()
            continue
        # the float32 values in the documented order, and their codes in integers
        g32 = g.float() if clip32 is None else g.float() * clip32
        m32 = m0 * 0.9 + g32 * (1 - 0.9)
        v32 = v0 * 0.999 + (g32 * g32) * (1 - 0.999)
        word = ref.words(seed, i, t, n)
        for name, z, top, mant, least in (("exp_avg", m32, 256.0, 3, -6),
                                          ("exp_avg_sq", v32, 32768.0, 2, -14)):
            blocks = torch.nn.functional.pad(z, (0, -n % ref.BLOCK)).view(-1, ref.BLOCK)
            most = blocks.abs().amax(1).clamp_min(2.0**-100)
            assert torch.equal(y[name + "_scale"][i].cpu(), most * (1 / top))
            up = (z.abs() * (top / most).repeat_interleave(ref.BLOCK)[:n]).tolist()
            bits = word if name == "exp_avg" else (word << 16) & ref.MASK
            codes = [ref.code(a, b, mant, least) for a, b in zip(up, bits.tolist())]
            codes = torch.tensor(codes)
            if name == "exp_avg_sq":
                codes = torch.where(z > 0, codes.clamp_min(1), codes)
            got = y[name][i].cpu().view(torch.uint8).long()
            sign = got >> 7
            assert torch.equal(got & 127, codes), name
            assert torch.equal((sign == 1) & (codes > 0), (z < 0) & (codes > 0))


SIZES = [1, 2, 3, 4, 5, 63, 255, 256, 257, 511, 1023, 4095, 4096, 4097, 10001, 0, 40000]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad", [(torch.float32, torch.float32),
                                        (torch.bfloat16, torch.bfloat16),
                                        (torch.float16, torch.float32),
                                        (torch.float32, torch.bfloat16),
                                        (torch.bfloat16, torch.float16)])
def test_against_the_oracle(ext, bits, param, grad):
    for max_norm in (None, 0.5, 1e6):
        announce(f"adamw {bits} {param} {grad} {max_norm}")
        x = make(SIZES, param, grad, 3, bits)
        y = to_device(x)
        norm = step(ext, y, max_norm=max_norm)
        check(x, y, norm, max_norm)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_some_without_a_gradient(ext, bits):
    """More tensors than one launch takes; a decay and a rate for each; gradients of None."""
    announce(f"adamw many {bits}")
    sizes = [(37 * k) % 901 + 1 for k in range(101)]
    x = make(sizes, torch.bfloat16, torch.bfloat16, 4, bits)
    for k in (0, 31, 32, 64, 100):
        x["grads"][k] = None
    lr = [1e-3 * (1 + k % 5) for k in range(101)]
    decay = [0.01 * (k % 3) for k in range(101)]
    y = to_device(x)
    norm = step(ext, y, max_norm=1.0, lr=lr, weight_decay=decay)
    check(x, y, norm, 1.0, lr, decay)
    none = dict(x, grads=[None] * 101)
    z = to_device(none)
    assert float(step(ext, z, max_norm=1.0)) == 0.0
    assert all(torch.equal(a.cpu(), b) for a, b in zip(z["params"], none["params"]))
    assert torch.equal(z["steps"].cpu(), x["steps"])


def test_unaligned_tensors(ext):
    """Tensors that start at odd elements of a buffer (no wide access fits): the same bits."""
    for bits in (32, 8):
        announce(f"adamw unaligned {bits}")
        x = make([1000, 517], torch.bfloat16, torch.bfloat16, 5, bits)
        y = to_device(x)

        def shifted(t, by):
            if t is None:
                return None
            room = torch.zeros(t.numel() + 8, dtype=torch.uint8 if t.element_size() == 1 else t.dtype,
                               device=DEV)
            at = room[by:by + t.numel()]
            at.copy_(t.view(torch.uint8) if t.element_size() == 1 else t)
            return at.view(t.dtype)

        z = {k: [shifted(t, 1 + j % 3) for j, t in enumerate(v)] if isinstance(v, list) else v
             for k, v in y.items()}
        z["steps"] = y["steps"].clone()
        a, b = step(ext, y, max_norm=1.0), step(ext, z, max_norm=1.0)
        assert torch.equal(a, b)
        for k in ("params", "master", "exp_avg", "exp_avg_sq", "exp_avg_scale"):
            for p, q in zip(y[k] or [], z[k] or []):
                same = (lambda t: t.view(torch.uint8) if t.element_size() == 1 else t)
                assert torch.equal(same(p), same(q)), k


def test_extreme_moments_in_8_bits(ext):
    """All zeros stay zeros; tiny values keep a second moment above 0; a block with a NaN or an
    infinity reads NaN throughout, its neighbours do not."""
    n = 4 * ref.BLOCK
    x = make([n], torch.float32, torch.float32, 6, 8)
    for k in ("exp_avg", "exp_avg_sq"):
        x[k] = [torch.zeros(n).to(x[k][0].dtype)]
        x[k + "_scale"] = [torch.zeros(4)]
    g = torch.zeros(n)
    g[256:512] = 1e-12
    g[256] = 1.0                 # 24 orders of magnitude of v in one block
    g[512:768] = 1e-25           # squares below float32
    g[800] = math.nan
    x["grads"] = [g]
    y = to_device(x)
    step(ext, y)
    now = {**{k: [t.cpu() for t in v] for k, v in y.items() if isinstance(v, list)}}
    m, v = moments(now, 0)
    assert (m[:256] == 0).all() and (v[:256] == 0).all()
    assert (v[256:512] > 0).all() and torch.isfinite(v[256:512]).all()
    assert torch.isfinite(m[256:768]).all() and torch.isfinite(y["params"][0][:768]).all()
    assert torch.isnan(m[768:]).all() and torch.isnan(v[768:]).all()
    # the smallest second moment a block can hold keeps its steps within the first moment's over
    # its root: nothing is divided by eps alone
    move = (y["params"][0].cpu() - x["params"][0] * (1 - 3e-4)).abs()[256:512]
    assert move.max() <= 3e-3 * 1.01
    x["grads"] = [torch.full((n,), math.inf)]
    y = to_device(x)
    step(ext, y)
    assert torch.isnan(moments({k: [t.cpu() for t in v] for k, v in y.items() if isinstance(v, list)},
                               0)[1]).all()


def test_rounding_is_unbiased(ext):
    """With no gradient, 300 steps take v to 0.999^300 and m to 0.9^20 in the mean.  Each step's
    rounding moves a value by at most a code step (a quarter for v, an eighth for m) with mean 0, so
    after T steps the mean over N values deviates by at most 5 sqrt(T) / 4 / sqrt(N) of the start
    (variance of a step at most (step / 2)^2, five sigma)."""
    n = 1 << 18
    x = make([n], torch.float32, torch.float32, 7, 8)
    g = torch.Generator().manual_seed(1)
    for k, dt, top in (("exp_avg", torch.float8_e4m3fn, 256.0),
                       ("exp_avg_sq", torch.float8_e5m2, 32768.0)):
        u = torch.rand(n, generator=g) * 0.9 + 0.1
        x[k] = [(u * top).to(dt)]
        x[k + "_scale"] = [torch.full((n // 256,), 1 / top)]
    x["grads"] = [torch.zeros(n)]
    m0, v0 = (t.double().mean() for t in moments(x, 0))
    y = to_device(x)
    for t in range(1, 301):
        step(ext, y)
        if t in (20, 300):
            now = {k: [z.cpu() for z in v] for k, v in y.items() if isinstance(v, list)}
            m, v = (z.double().mean() for z in moments(now, 0))
            if t == 20:
                assert abs(m - m0 * 0.9**20) < 5 * math.sqrt(20) / 16 / math.sqrt(n)
    assert abs(v - v0 * 0.999**300) < 5 * math.sqrt(300) / 8 / math.sqrt(n)


def test_streams_graphs_and_schedules(ext):
    """A captured step with a device rate, replayed with eager work between, equals eager steps."""
    for bits in (32, 8):
        announce(f"adamw graph {bits}")
        x = make([5000, 33, 1], torch.bfloat16, torch.bfloat16, 8, bits)
        a, b = to_device(x), to_device(x)
        rate = torch.ones(1, device=DEV)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(ext, a, max_norm=1.0, lr_scale=rate)
        torch.cuda.current_stream().wait_stream(side)
        step(ext, b, max_norm=1.0, lr_scale=rate)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step(ext, a, max_norm=1.0, lr_scale=rate)
        for k in range(4):
            rate.fill_(0.5 ** k)
            for p, q in zip(a["grads"], b["grads"]):
                p.copy_(torch.randn_like(p) * 0.01)
                q.copy_(p)
            graph.replay()
            norm = step(ext, b, max_norm=1.0, lr=3e-3 * 0.5**k)
            assert torch.equal(held, norm)
            torch.cuda.synchronize()
            for name in ("params", "master", "exp_avg", "exp_avg_sq"):
                for p, q in zip(a[name], b[name]):
                    assert torch.equal(p.float(), q.float()), (name, k)
        assert a["steps"].tolist() == b["steps"].tolist() == [5, 12, 19]


def test_refusals(ext):
    x = make([300, 20], torch.bfloat16, torch.bfloat16, 9, 8)
    y = to_device(x)
    wide = to_device(make([300, 20], torch.float32, torch.float32, 9))

    def bad(state, exc=RuntimeError, args=None, **over):
        with pytest.raises(exc):
            step(ext, {**state, **over}, **(args or {}))

    p, m = y["params"], y["master"]
    bad(y, params=[p[0].cpu(), p[1]])
    bad(y, params=[p[0], p[1].double()])
    bad(y, params=[p[0].view(10, 30).t(), p[1]])
    bad(y, master=None)
    bad(y, master=[m[0], None])
    bad(y, master=[m[0], m[1][:19]])
    bad(wide, master=wide["params"])
    bad(y, params=[p[0], p[0]], grads=[y["grads"][0]] * 2, master=[m[0], m[0]],
        exp_avg=[y["exp_avg"][0]] * 2, exp_avg_sq=[y["exp_avg_sq"][0]] * 2,
        exp_avg_scale=[y["exp_avg_scale"][0]] * 2, exp_avg_sq_scale=[y["exp_avg_sq_scale"][0]] * 2)
    bad(wide, exp_avg_sq=wide["exp_avg"])
    bad(wide, params=[wide["params"][0], wide["params"][0][10:30]])
    bad(wide, grads=[wide["params"][0], wide["grads"][1]])
    bad(wide, grads=[wide["exp_avg"][0], wide["grads"][1]])
    bad(y, grads=y["grads"][:1])
    bad(y, grads=[y["grads"][0], y["grads"][1].long()])
    bad(y, grads=[y["grads"][0], y["grads"][0]])
    bad(y, exp_avg_scale=None)
    bad(y, exp_avg_scale=[y["exp_avg_scale"][0]] * 2)
    bad(y, exp_avg=wide["exp_avg"])
    bad(y, steps=y["steps"].int())
    bad(y, steps=y["steps"][:1])
    bad(y, args=dict(betas=(1.0, 0.9)))
    bad(y, args=dict(eps=-1.0))
    bad(y, args=dict(max_norm=0.0))
    bad(y, args=dict(lr_scale=torch.ones(1)))
    bad(y, args=dict(lr=[0.1]))
    bad(y, params=[], grads=[], exp_avg=[], exp_avg_sq=[], master=[], exp_avg_scale=[],
        exp_avg_sq_scale=[], steps=y["steps"][:0])


# --------------------------------------------------------------------------- the optimizer


def _net(dtype):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(37, 64), torch.nn.Tanh(),
                               torch.nn.Linear(64, 11)).to(DEV, dtype)


def test_optimizer_matches_torchs(ext):
    """Float32, two groups: every step within the step's tolerance of torch's AdamW on the same
    gradients (each at most 40 u of the weight and of the step)."""
    from cugo_amd import learner

    a, b = _net(torch.float32), _net(torch.float32)
    groups = lambda n: [dict(params=[n[0].weight, n[2].weight], weight_decay=0.1),  # noqa: E731
                        dict(params=[n[0].bias, n[2].bias], weight_decay=0.0, lr=1e-2)]
    ours = learner.AdamW(ext, groups(a), lr=3e-3)
    torchs = torch.optim.AdamW(groups(b), lr=3e-3)
    for k in range(20):
        for p, q in zip(a.parameters(), b.parameters()):
            p.grad = torch.randn_like(p)
            q.grad = p.grad.clone()
        before = p.grad._version, a[0].weight._version
        ours.step()
        torchs.step()
        assert a[0].weight._version > before[1]
        for p, q in zip(a.parameters(), b.parameters()):
            # k steps of at most lr sqrt(k) each way, 40 u of the weight and the moves so far
            assert (p - q).abs().max() <= 40 * U * (k + 1) * (q.abs().max() + 1e-2 * (k + 1))


@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_state_is_saved_and_loaded(ext, bits):
    from cugo_amd import learner

    a, b = _net(torch.bfloat16), _net(torch.bfloat16)
    x = torch.randn(50, 37, device=DEV).bfloat16()

    def train(net, opt, k):
        for _ in range(k):
            opt.zero_grad()
            net(x).float().square().mean().backward()
            opt.step()

    one = learner.AdamW(ext, a.parameters(), max_norm=0.5, state_bits=bits, seed=5)
    train(a, one, 3)
    assert one.grad_norm.shape == () and one.grad_norm > 0
    saved = one.state_dict()
    b.load_state_dict(a.state_dict())
    two = learner.AdamW(ext, b.parameters(), max_norm=0.5, state_bits=bits, seed=5)
    two.load_state_dict(saved)
    train(a, one, 3)
    train(b, two, 3)
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)
        assert torch.equal(one.state[p]["master"], two.state[q]["master"])
        assert int(two.state[q]["step"]) == 6
    wrong = learner.AdamW(ext, b.parameters(), state_bits=40 - bits)
    with pytest.raises(ValueError, match="fit"):
        wrong.load_state_dict(saved)


def test_offsets_past_32_bits(ext):
    """A tensor of more than 2^32 values with 8-bit moments: its last blocks' values, scales and
    codes, whose rounding words take the index's upper bits."""
    from cugo_amd import learner

    n = (1 << 32) + 3 * ref.BLOCK + 77
    tail = 2 * ref.BLOCK + 77
    announce(f"adamw {n}")
    blocks = -(-n // ref.BLOCK)
    w = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    grad = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    master = torch.zeros(n, device=DEV)
    g = torch.randn(tail, generator=torch.Generator().manual_seed(1)).bfloat16()
    grad[-tail:] = g.to(DEV)
    m = torch.zeros(n, dtype=torch.float8_e4m3fn, device=DEV)
    v = torch.zeros(n, dtype=torch.float8_e5m2, device=DEV)
    ms, vs = torch.zeros(blocks, device=DEV), torch.zeros(blocks, device=DEV)
    steps = torch.zeros(1, dtype=torch.int64, device=DEV)
    norm = learner.adamw_step(ext, [w], [grad], [m], [v], steps, lr=0.1, weight_decay=0.0,
                              max_norm=1e9, master=[master], exp_avg_scale=[ms],
                              exp_avg_sq_scale=[vs], seed=77)
    assert abs(float(norm) - float(g.double().norm())) < 1e-5 * float(norm)
    assert (master[:-tail][::9973] == 0).all()
    # from moments of zero the first step is lr g / (|g| + eps), within 16 u and the moments' 14
    goal = -0.1 * g.double() / (g.double().abs() + EPS)
    off = float((master[-tail:].cpu().double() - goal).abs().max())
    assert off <= 0.1 * 30 * U
    g32 = g.float()
    for got, scale, z, top, mant, least in (
            (m, ms, g32 * (1 - 0.9), 256.0, 3, -6),
            (v, vs, (g32 * g32) * (1 - 0.999), 32768.0, 2, -14)):
        most = torch.stack([x.abs().max() for x in z.split(ref.BLOCK)])
        assert torch.equal(scale[-3:].cpu(), most * (1 / top))
        up = (z.abs() * (top / most).repeat_interleave(ref.BLOCK)[:tail]).tolist()
        for i in range(0, tail, 7):
            word = ref.word(77, 0, 1, n - tail + i)
            bits = word if mant == 3 else (word << 16) & ref.MASK
            want = ref.code(up[i], bits, mant, least)
            if mant == 2 and z[i] > 0:
                want = max(want, 1)
            assert int(got[n - tail + i].view(torch.uint8)) & 127 == want, i


def test_one_gradient_for_two_parameters(ext):
    """Gradients are read only: two parameters may share one."""
    x = make([700, 700], torch.float32, torch.float32, 11)
    x["grads"][1] = x["grads"][0]
    y = to_device(x)
    y["grads"][1] = y["grads"][0]
    norm = step(ext, y, max_norm=1.0)
    check(x, y, norm, 1.0)


def test_optimizer_groups_rates_and_gradients_of_none(ext):
    from cugo_amd import learner

    net = _net(torch.float32)
    opt = learner.AdamW(ext, [net[0].weight], lr=torch.tensor([1e-2], device=DEV))
    net[0].weight.grad = torch.ones_like(net[0].weight)
    was = net[0].weight.detach().clone()
    opt.step()
    assert torch.allclose(net[0].weight, was * (1 - 1e-4) - 1e-2, atol=1e-6)
    opt.add_param_group(dict(params=[net[2].weight, net[2].bias], lr=opt.param_groups[0]["lr"]))
    net[2].bias.grad = torch.ones(11, device=DEV, dtype=torch.float32)
    kept = net[2].weight.detach().clone()
    opt.step()
    steps = [int(opt.state[p]["step"]) for p in (net[0].weight, net[2].weight, net[2].bias)]
    assert steps == [2, 0, 1]
    assert torch.equal(net[2].weight, kept)
    opt.param_groups[1]["lr"] = 0.1
    with pytest.raises(ValueError, match="same"):
        opt.step()
    with pytest.raises(ValueError):
        learner.AdamW(ext, net.parameters(), state_bits=16)


def _moved(t, by):
    """t's values `by` elements behind an aligned address."""
    bits = (lambda x: x.view(torch.uint8) if x.element_size() == 1 else x)
    room = torch.zeros(t.numel() + 8, dtype=bits(t).dtype, device=DEV)
    room[by:by + t.numel()].copy_(bits(t))
    return room[by:by + t.numel()].view(t.dtype)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param,grad", [(torch.float32, torch.float32),
                                        (torch.bfloat16, torch.bfloat16),
                                        (torch.float16, torch.float32)])
def test_whole_chunks_at_any_address(ext, bits, param, grad):
    """Tensors of several whole chunks of 4,096 values, one stream at a time (and all of them) away
    from a wide access's alignment: the bits of aligned tensors."""
    sizes = [4096, 8192 + 5, 12288]
    x = make(sizes, param, grad, 12, bits)
    y = to_device(x)
    norm = step(ext, y, max_norm=1.0)
    check(x, y, norm, 1.0)
    streams = ["params", "grads", "exp_avg", "exp_avg_sq"]
    streams += ["master"] if param != torch.float32 else []
    for which in [[s] for s in streams] + [streams]:
        for by in (1, 2, 3):
            announce(f"adamw {bits} {param} {grad} {which} {by}")
            z = to_device(x)
            for s in which:
                z[s] = [_moved(t, by) for t in z[s]]
            assert torch.equal(step(ext, z, max_norm=1.0), norm)
            for k in ("params", "master", "exp_avg", "exp_avg_sq", "exp_avg_scale",
                      "exp_avg_sq_scale"):
                for p, q in zip(y[k] or [], z[k] or []):
                    same = (lambda t: t.view(torch.uint8) if t.element_size() == 1 else t)
                    assert torch.equal(same(p), same(q)), (which, by, k)


@pytest.mark.parametrize("bits", [32, 8])
def test_copied_optimizers_step_alike(ext, bits):
    """A deep copy, and one loaded from a checkpoint into other options, take the same steps, moved
    betas among them."""
    import copy

    from cugo_amd import learner

    net = _net(torch.bfloat16)
    opt = learner.AdamW(ext, net.parameters(), lr=1e-3, betas=(0.8, 0.95), max_norm=0.3,
                        state_bits=bits, seed=4)

    def steps(nets, opts, count, seed):
        for k in range(count):
            g = torch.Generator(device=DEV).manual_seed(seed + k)
            grads = [torch.randn(p.shape, generator=g, device=DEV).bfloat16()
                     for p in nets[0].parameters()]
            for n, o in zip(nets, opts):
                for p, x in zip(n.parameters(), grads):
                    p.grad = x.clone()
                o.betas = (0.8 + 0.01 * k, 0.95)
                o.step()

    steps([net], [opt], 3, 1)
    net2, two = copy.deepcopy((net, opt))
    net3 = copy.deepcopy(net)
    three = learner.AdamW(ext, net3.parameters(), lr=1.0, state_bits=bits)
    three.load_state_dict(opt.state_dict())
    assert three.seed == 4 and three.max_norm == 0.3
    steps([net, net2, net3], [opt, two, three], 3, 10)
    for other, o in ((net2, two), (net3, three)):
        assert torch.equal(o.grad_norm, opt.grad_norm)
        for p, q in zip(net.parameters(), other.parameters()):
            assert torch.equal(p, q) and int(o.state[q]["step"]) == 6
            for k in ("master", "exp_avg", "exp_avg_sq"):
                assert torch.equal(opt.state[p][k].float(), o.state[q][k].float()), k
