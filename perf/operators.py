"""The learner's operators as cases that can be timed and compared.

Between the rollout that records decisions and the next one with better weights stand three
operators, each reached through `cugo_amd.learner`:

  loss   `policy_loss`: the clipped policy loss with a KL term to another policy, an entropy
         bonus and the value loss, over the legal actions of each row, and its gradients
  gae    `advantages`: generalised advantage estimation over a horizon of games between two
         players, from each mover's side
  adamw  `adamw_step`: one AdamW step over many tensors at once, with the norm of all
         gradients clipped, the moments in 32 bits or in 8

The plain forms below are the definitions in elementary torch operations.
"""

import torch

own = False

ACTIONS, FEATURES = 179, 720
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CLIP_LOW, CLIP_HIGH = 0.2, 0.3
KL_COEF, ENTROPY_COEF, VALUE_COEF = 0.1, 0.01, 0.5
GAMMA, LAM = 0.997, 0.95
LR, BETAS, EPS, DECAY, MAX_NORM = 3e-4, (0.9, 0.999), 1e-8, 0.01, 1.0
BLOCK = 256  # values that share a scale of the 8-bit moments
SEED = 0x5EED1234ABCD  # of the moments' stochastic rounding
MOST_LOGITS = 1048576 * ACTIONS
MOST_STEPS = 128 * 65536
MOST_PARAMS = 36_000_000


def listed():
    return [
        # A minibatch of a small debugging run: the call's own latency.
        {"name": "loss_256", "kind": "loss", "rows": 256, "actions": ACTIONS, "dtype": "bf16",
         "legal": True, "ref": False, "value": True, "weight": False, "grad": True},
        # The usual minibatch of a policy update.
        {"name": "loss_16384", "kind": "loss", "rows": 16384, "actions": ACTIONS, "dtype": "bf16",
         "legal": True, "ref": True, "value": True, "weight": False, "grad": True},
        # Float32 logits of sequences padded to a common length: an odd number of rows, some of
        # weight zero.
        {"name": "loss_padded_65539", "kind": "loss", "rows": 65539, "actions": ACTIONS,
         "dtype": "f32", "legal": True, "ref": True, "value": True, "weight": True, "grad": True},
        # 32 steps of 32,768 games at once, with the KL term.
        {"name": "loss_1m", "kind": "loss", "rows": 1048576, "actions": ACTIONS, "dtype": "bf16",
         "legal": True, "ref": True, "value": True, "weight": False, "grad": True},
        # The loss alone (no gradient) of an evaluation batch in half precision.
        {"name": "loss_eval_100003", "kind": "loss", "rows": 100003, "actions": ACTIONS,
         "dtype": "f16", "legal": True, "ref": False, "value": True, "weight": False,
         "grad": False},
        # A vocabulary instead of a game's actions: long rows, every entry legal.
        {"name": "loss_vocab_32000", "kind": "loss", "rows": 4096, "actions": 32000,
         "dtype": "bf16", "legal": False, "ref": True, "value": False, "weight": False,
         "grad": True},
        # The rollout's horizon: 128 steps of 32,768 games.
        {"name": "gae_128x32768", "kind": "gae", "steps": 128, "batch": 32768, "value": "f32"},
        # Few games over a long horizon, odd sizes, bf16 values.
        {"name": "gae_20001x45", "kind": "gae", "steps": 20001, "batch": 45, "value": "bf16"},
        # The rollout's actor: bf16 parameters with float32 masters, gradients clipped.
        {"name": "adamw_actor", "kind": "adamw", "width": 512, "blocks": 3, "param": "bf16",
         "grad": "bf16", "bits": 32, "clip": True},
        # The same actor with 8-bit moments.
        {"name": "adamw_actor_8bit", "kind": "adamw", "width": 512, "blocks": 3, "param": "bf16",
         "grad": "bf16", "bits": 8, "clip": True},
        # A wide actor (2,048, four blocks) in float32.
        {"name": "adamw_wide", "kind": "adamw", "width": 2048, "blocks": 4, "param": "f32",
         "grad": "f32", "bits": 32, "clip": True},
        # The wide actor with bf16 parameters, float32 masters and 8-bit moments, not clipped.
        {"name": "adamw_wide_8bit", "kind": "adamw", "width": 2048, "blocks": 4, "param": "bf16",
         "grad": "bf16", "bits": 8, "clip": False},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(["loss", "loss", "gae", "adamw"])
    if kind == "loss":
        # half of the draws over the game's actions, the rest from a handful to a vocabulary
        actions = ACTIONS if rng.random() < 0.5 else _log_int(rng, 2, 50000)
        rows = _log_int(rng, 1, max(1, min(1048576, MOST_LOGITS // actions)))
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        if dtype == "f32":
            rows = max(1, rows // 2)
        return {"kind": kind, "rows": rows, "actions": actions, "dtype": dtype,
                "legal": actions <= 1024 and rng.random() < 0.8, "ref": rng.random() < 0.5,
                "value": rng.random() < 0.7, "weight": rng.random() < 0.4,
                "grad": rng.random() < 0.8}
    if kind == "gae":
        steps = _log_int(rng, 1, 20001)
        return {"kind": kind, "steps": steps, "batch": _log_int(rng, 1, min(65536, MOST_STEPS // steps)),
                "value": rng.choice(["f32", "bf16", "f16"])}
    while True:
        case = {"kind": kind, "width": _log_int(rng, 16, 2048), "blocks": rng.randint(1, 4),
                "param": rng.choice(["f32", "bf16", "f16"]), "grad": rng.choice(["f32", "bf16"]),
                "bits": rng.choice([8, 32]), "clip": rng.random() < 0.7}
        if sum(_sizes(case)) <= MOST_PARAMS:
            return case


def _sizes(case):
    """The tensors of a residual MLP actor: input layer, blocks (norm, two layers), norm, heads."""
    d = case["width"]
    return ([d * FEATURES, d] + [d, d, d * d, d, d * d, d] * case["blocks"]
            + [d, d, d * ACTIONS, ACTIONS, d, 1])


# ------------------------------------------------------------------------------ inputs


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "loss":
        return {"case": case, **_prepare_loss(case, gen)}
    if case["kind"] == "gae":
        return {"case": case, **_prepare_gae(case, gen)}
    return {"case": case, **_prepare_adamw(case, gen)}


def _prepare_loss(case, gen):
    n, a, dt = case["rows"], case["actions"], DTYPES[case["dtype"]]
    dev = "cuda"

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    logits = (randn(n, a) * 1.5).to(dt)
    legal = None
    if case["legal"]:
        # 1 to about 20 legal actions of 179 (as many in proportion of other counts); about one
        # row in 500 has none (a game that is over)
        share = torch.rand(n, 1, generator=gen, device=dev) * 0.11 + 1.0 / a
        legal = torch.rand(n, a, generator=gen, device=dev) < share
        legal &= (torch.rand(n, 1, generator=gen, device=dev) > 0.002)
    # the action: a draw from the policy that collected, whose logits differ a little
    old = logits.float() + 0.2 * randn(n, a)
    if legal is not None:
        old.masked_fill_(~legal, -1e30)
    noise = torch.rand(n, a, generator=gen, device=dev).clamp_(1e-20, 1 - 1e-7).log_().neg_().log_().neg_()
    action = noise.add_(old).argmax(1)
    del noise
    old_logp = old.log_softmax(1).gather(1, action[:, None])[:, 0].contiguous()
    del old
    state = {"logits": logits.requires_grad_(case["grad"]), "legal": legal, "action": action,
             "old_logp": old_logp, "advantage": randn(n), "ref": None, "value": None,
             "returns": None, "weight": None}
    if case["ref"]:
        state["ref"] = (logits.detach().float() + 0.5 * randn(n, a)).to(dt)
    if case["value"]:
        state["value"] = randn(n).to(dt).requires_grad_(case["grad"])
        state["returns"] = randn(n)
    if case["weight"]:
        keep = torch.rand(n, generator=gen, device=dev) < 0.85
        state["weight"] = keep.float() / n
    return state


def _prepare_gae(case, gen):
    t, b, dt = case["steps"], case["batch"], DTYPES[case["value"]]

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    done = rand(t, b) < 0.035  # games of about 28 decisions
    reward = torch.where(done, torch.randn(t, b, generator=gen, device="cuda") * 3, 0.0)
    return {"reward": reward, "done": done,
            "value": torch.randn(t, b, generator=gen, device="cuda").to(dt),
            "player": (rand(t, b) < 0.5).to(torch.uint8),
            "bootstrap": torch.randn(b, generator=gen, device="cuda").to(dt),
            "last_player": (rand(b) < 0.5).to(torch.uint8)}


def _prepare_adamw(case, gen):
    """The tensors lie in flat buffers, each from a multiple of 256 values on (a plain form over
    whole buffers then costs no launches for each tensor); gaps hold zeros, which stay zeros."""
    sizes = _sizes(case)
    starts, total = [], 0
    for s in sizes:
        starts.append(total)
        total += -(-s // BLOCK) * BLOCK
    inside = torch.zeros(total, dtype=torch.bool, device="cuda")
    for s, n in zip(starts, sizes):
        inside[s:s + n] = True

    def filled(values):
        return torch.where(inside, values, 0.0)

    def randn():
        return torch.randn(total, generator=gen, device="cuda")

    def parts(flat, unit=1):
        return [flat[s // unit:(s + n + unit - 1) // unit] for s, n in zip(starts, sizes)]

    param, grad_dt = DTYPES[case["param"]], DTYPES[case["grad"]]
    w = filled(randn() * 0.02)
    # gradients and moments of a run that has gone on for a while: a spread of magnitudes
    size = torch.exp(randn()) * 1e-4
    state = {"sizes": sizes, "param": w.to(param), "grad": filled(randn() * size).to(grad_dt),
             "master": None if case["param"] == "f32" else w.clone(),
             "steps": torch.full((len(sizes),), 100, dtype=torch.int64, device="cuda"),
             "m_scale": None, "v_scale": None}
    m, v = filled(randn() * size * 0.3), filled((randn() * size).square() * 0.5)
    if case["bits"] == 8:
        for name, x, dt, top in (("m", m, torch.float8_e4m3fn, 256.0), ("v", v, torch.float8_e5m2, 32768.0)):
            scale = x.view(-1, BLOCK).abs().amax(1).clamp_min(2.0**-100) / top
            state[name + "_scale"] = scale
            state[name] = (x.view(-1, BLOCK) / scale[:, None]).view(-1).to(dt)
    else:
        state["m"], state["v"] = m, v
    state["lists"] = {k: parts(state[k]) if state[k] is not None else None
                      for k in ("param", "grad", "master", "m", "v")}
    for k in ("m_scale", "v_scale"):
        state["lists"][k] = parts(state[k], BLOCK) if state[k] is not None else None
    return state


# ------------------------------------------------------------------------------ one pass


def run(state):
    case = state["case"]
    if case["kind"] == "loss":
        return _own_loss(state) if own else _plain_loss(state)
    if case["kind"] == "gae":
        return _own_gae(state) if own else _plain_gae(state)
    return _own_adamw(state) if own else _plain_adamw(state)


def _ext():
    from cugo_amd import load_extension

    return load_extension()


def _own_loss(s):
    from cugo_amd import learner

    out = learner.policy_loss(
        _ext(), s["logits"], s["action"], s["old_logp"], s["advantage"], legal=s["legal"],
        ref_logits=s["ref"], value=s["value"], returns=s["returns"], weight=s["weight"],
        clip=(CLIP_LOW, CLIP_HIGH), kl_coef=KL_COEF, entropy_coef=ENTROPY_COEF,
        value_coef=VALUE_COEF)
    result = {"loss": out.loss.detach(), "stats": out.stats, "logp": out.logp}
    if s["case"]["grad"]:
        leaves = [s["logits"]] + ([s["value"]] if s["value"] is not None else [])
        grads = torch.autograd.grad(out.loss, leaves)
        result["d_logits"] = grads[0]
        if s["value"] is not None:
            result["d_value"] = grads[1]
    return result


@torch.no_grad()
def _plain_loss(s):
    case = s["case"]
    n = case["rows"]
    z = s["logits"].float()
    if s["legal"] is not None:
        z = torch.where(s["legal"], z, -torch.inf)
    top = z.amax(1, keepdim=True)
    some = top > -torch.inf  # rows with a legal action
    e = torch.exp(z - torch.where(some, top, 0.0))
    total = e.sum(1, keepdim=True)
    p = e / torch.where(some, total, 1.0)
    ell = z - torch.where(some, top + torch.log(total), 0.0)  # log-probabilities
    has = p > 0
    entropy = -torch.where(has, p * ell, 0.0).sum(1)
    w = s["weight"] if s["weight"] is not None else torch.full_like(s["old_logp"], 1.0 / n)
    logp = torch.where(some[:, 0], ell.gather(1, s["action"][:, None])[:, 0], 0.0)
    # an action without probability: ratio 0; a row without legal actions has no policy terms
    log_ratio = logp - s["old_logp"]
    ratio = torch.where(logp > -torch.inf, torch.exp(log_ratio), 0.0)
    adv = s["advantage"]
    clipped = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    surrogate = torch.minimum(ratio * adv, clipped * adv)
    cut = ratio * adv > clipped * adv
    row = some[:, 0] & (w != 0)
    wp = torch.where(row, w, 0.0)
    kl = torch.zeros_like(w)
    d = None
    if s["ref"] is not None:
        zr = s["ref"].float()
        if s["legal"] is not None:
            zr = torch.where(s["legal"], zr, -torch.inf)
        topr = torch.where(some, zr.amax(1, keepdim=True), 0.0)
        lser = topr + torch.log(torch.exp(zr - topr).sum(1, keepdim=True))
        d = torch.where(has, ell - (zr - lser), 0.0)
        kl = (p * d).sum(1)

    def mean(x):
        return torch.where(row, wp * x, 0.0).double().sum().float()

    value_sum = torch.zeros((), device=w.device)
    if s["value"] is not None:
        err = s["value"].float() - s["returns"]
        value_sum = torch.where(w != 0, w * 0.5 * err * err, 0.0).double().sum().float()
    stats = torch.stack([mean(-surrogate), value_sum, mean(kl), mean(entropy),
                         mean(cut.float()), mean((ratio - 1) - log_ratio)])
    loss = stats[0] + VALUE_COEF * stats[1] + KL_COEF * stats[2] - ENTROPY_COEF * stats[3]
    result = {"loss": loss, "stats": stats, "logp": logp}
    if case["grad"]:
        pull = torch.where(cut, 0.0, ratio * adv)[:, None]
        hot = torch.zeros_like(p).scatter_(1, s["action"][:, None], 1.0)
        g = pull * (p - hot) + ENTROPY_COEF * torch.where(has, p * (ell + entropy[:, None]), 0.0)
        if d is not None:
            g = g + KL_COEF * p * (d - kl[:, None])
        result["d_logits"] = torch.where(row[:, None], wp[:, None] * g, 0.0).to(s["logits"].dtype)
        if s["value"] is not None:
            result["d_value"] = torch.where(w != 0, w * VALUE_COEF * err, 0.0).to(s["value"].dtype)
    return result


def _own_gae(s):
    from cugo_amd import learner

    advantage, returns = learner.advantages(
        _ext(), s["reward"], s["value"], s["done"], s["bootstrap"], GAMMA, LAM,
        player=s["player"], last_player=s["last_player"])
    return {"advantage": advantage, "returns": returns}


def _plain_gae(s):
    """A scan over the steps in doubling strides: after stride k, the sums run over 2 k steps."""
    sign = 1.0 - 2.0 * s["player"].float()
    v = sign * s["value"].float()  # from player 0's side, as the rewards are
    last = (1.0 - 2.0 * s["last_player"].float()) * s["bootstrap"].float()
    following = torch.cat([v[1:], last[None]])
    total = s["reward"] + torch.where(s["done"], 0.0, GAMMA * following) - v
    keep = torch.where(s["done"], 0.0, GAMMA * LAM)
    stride, steps = 1, s["case"]["steps"]
    while stride < steps:
        total = torch.cat([total[:-stride] + keep[:-stride] * total[stride:], total[-stride:]])
        keep = torch.cat([keep[:-stride] * keep[stride:], torch.zeros_like(keep[-stride:])])
        stride *= 2
    advantage = sign * total
    return {"advantage": advantage, "returns": advantage + s["value"].float()}


def _own_adamw(s):
    from cugo_amd import learner

    x = s["lists"]
    scales = {} if s["m_scale"] is None else {"exp_avg_scale": x["m_scale"], "exp_avg_sq_scale": x["v_scale"]}
    norm = learner.adamw_step(
        _ext(), x["param"], x["grad"], x["m"], x["v"], s["steps"], lr=LR, betas=BETAS, eps=EPS,
        weight_decay=DECAY, max_norm=MAX_NORM if s["case"]["clip"] else None, master=x["master"],
        seed=SEED, **scales)
    return _adamw_result(s, norm)


def _adamw_result(s, norm):
    names = ("param", "master", "m", "v", "m_scale", "v_scale", "steps")
    return {"norm": norm, **{k: s[k] for k in names}}


MASK = 0xFFFFFFFF


def _mix(x):
    """32 bits mixed by two multiplications with odd constants (the fractions of the golden
    ratio and of the square root of 3) between shifted exclusive ors; int64 tensors."""
    x = x & MASK
    x = ((x ^ (x >> 17)) * 0x9E3779B9) & MASK
    x = ((x ^ (x >> 14)) * 0xBB67AE85) & MASK
    return x ^ (x >> 15)


def _words(s):
    """The 32 bits that round each value: of the seed, the tensor's place in the list, the step
    and the value's place in its tensor (all places are below 2^32 here)."""
    dev = s["steps"].device
    padded = torch.tensor([-(-n // BLOCK) * BLOCK for n in s["sizes"]], device=dev)
    tensor = torch.arange(len(s["sizes"]), device=dev)
    seed = torch.tensor([SEED & MASK, SEED >> 32], dtype=torch.int64, device=dev)
    key = _mix(seed[0] ^ _mix(seed[1] + 1))
    key = _mix(_mix(_mix(key + tensor) + s["steps"]))
    place = torch.arange(s["m"].numel(), device=dev)
    first = padded.cumsum(0) - padded
    key, first = (torch.repeat_interleave(x, padded, output_size=s["m"].numel()) for x in (key, first))
    return _mix((place - first) ^ key)


def _codes(y, word, drop, least):
    """y >= 0 rounded to a code of 23 - drop mantissa bits (`least`: the binary exponent of the
    smallest normal value), up with the probability of what is cut off: word's upper bits, 32
    bits, are added below the last kept bit before the cut."""
    normal = y >= 2.0**least
    bits = torch.where(normal, y.view(torch.int32).long(), (y * 2.0**(23 - least)).long())
    code = (bits + (word >> (32 - drop))) >> drop
    return code - torch.where(normal, (126 + least) * 2**(23 - drop), 0)


def _quantized(x, word, top, drop, least):
    x = x.view(-1, BLOCK)
    most = x.abs().amax(1, keepdim=True).clamp_min(2.0**-100)
    code = _codes((x.abs() * (top / most)).view(-1), word, drop, least)
    return code, (most * (1.0 / top)).view(-1)


@torch.no_grad()
def _plain_adamw(s):
    beta1, beta2 = BETAS
    g = s["grad"].float()
    norm = None
    if s["case"]["clip"]:
        norm = g.double().square().sum().sqrt().float()
        g = g * (MAX_NORM / (norm + 1e-6)).clamp_max(1.0)
    s["steps"] += 1
    t = s["steps"][0].double()
    step_size = (LR / (1 - beta1**t)).float()
    root = (1 / (1 - beta2**t).sqrt()).float()
    m, v = s["m"], s["v"]
    if s["m_scale"] is not None:
        m = (m.float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (v.float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1)
    m = m * beta1 + g * (1 - beta1)
    v = v * beta2 + (g * g) * (1 - beta2)
    w = s["master"] if s["master"] is not None else s["param"]
    w.copy_(w * (1 - LR * DECAY) - step_size * (m / (v.sqrt() * root + EPS)))
    if s["master"] is not None:
        s["param"].copy_(w)
    if s["m_scale"] is None:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return _adamw_result(s, norm)
    word = _words(s)
    # the first moment: sign, 4 bits of exponent, 3 of mantissa; the second 5 and 2, where a
    # value above zero stays above zero
    code, scale = _quantized(m, word, 256.0, 20, -6)
    s["m"].view(torch.uint8).copy_(torch.where(torch.signbit(m), code + 128, code))
    s["m_scale"].copy_(scale)
    code, scale = _quantized(v, (word << 16) & MASK, 32768.0, 21, -14)
    s["v"].view(torch.uint8).copy_(torch.where(v > 0, code.clamp_min(1), code))
    s["v_scale"].copy_(scale)
    return _adamw_result(s, norm)


# ------------------------------------------------------------------------------ the work


def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if case["kind"] == "loss":
        n, a, e = case["rows"], case["actions"], size[case["dtype"]]
        row = a * (e * (1 + case["ref"] + case["grad"]) + case["legal"])
        # action, old log-probability, advantage in, log-probability out
        row += 8 + 4 + 4 + 4 + 4 * case["weight"]
        if case["value"]:
            row += e + 4 + e * case["grad"]
        # an exponential, its sum and the entropy's product; the gradient's products
        return {"bytes": n * row, "flops": n * a * (6 + 6 * case["ref"] + 6 * case["grad"])}
    if case["kind"] == "gae":
        t, b, e = case["steps"], case["batch"], size[case["value"]]
        return {"bytes": t * b * (4 + e + 1 + 1 + 4 + 4) + b * (e + 1), "flops": t * b * 8}
    n, e = sum(_sizes(case)), size[case["param"]]
    value = size[case["grad"]] + (8 if case["param"] == "f32" else 8 + e)
    value += 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * value, "flops": n * 20}


# ------------------------------------------------------------------------------ 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "loss":
        return _exact_loss(state)
    if case["kind"] == "gae":
        return _exact_gae(state)
    return _exact_adamw(state)


def _exact_loss(s):
    """The definition in 64 bits; the gradients by differentiating it."""
    case = s["case"]
    n = case["rows"]
    legal = s["legal"] if s["legal"] is not None else torch.ones_like(s["logits"], dtype=torch.bool)
    some = legal.any(1)
    shown = legal | ~some[:, None]  # an empty row stands in with every action, at weight zero

    def log_probabilities(logits):
        return logits.masked_fill(~shown, -torch.inf).log_softmax(1)

    logits = s["logits"].detach().double().requires_grad_(case["grad"])
    w = s["weight"].double() if s["weight"] is not None else torch.full((n,), 1.0 / n, device="cuda", dtype=torch.float64)
    wp = w * some
    ell = log_probabilities(logits)
    safe = ell.masked_fill(~shown, 0.0)
    p = ell.exp()
    logp = ell.gather(1, s["action"][:, None])[:, 0]
    old, adv = s["old_logp"].double(), s["advantage"].double()
    ratio = (logp - old).exp()
    clipped = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
    policy = (wp * -torch.minimum(ratio * adv, clipped * adv)).sum()
    entropy = (wp * -(p * safe).sum(1)).sum()
    kl = torch.zeros((), dtype=torch.float64, device="cuda")
    if s["ref"] is not None:
        q = log_probabilities(s["ref"].double()).masked_fill(~shown, 0.0)
        kl = (wp * (p * (safe - q)).sum(1)).sum()
        del q
    loss = policy + KL_COEF * kl - ENTROPY_COEF * entropy
    value_loss = torch.zeros_like(kl)
    if s["value"] is not None:
        value = s["value"].detach().double().requires_grad_(case["grad"])
        value_loss = (w * 0.5 * (value - s["returns"].double()) ** 2).sum()
        loss = loss + VALUE_COEF * value_loss
    cut = (wp * (ratio * adv > clipped * adv)).sum()
    drift = (wp * (ratio - 1 - (logp - old))).sum()
    result = {"loss": loss.detach(), "stats": torch.stack([policy, value_loss, kl, entropy, cut, drift]).detach(),
              "logp": torch.where(some, logp, 0.0).detach()}
    del p, ell, safe
    if case["grad"]:
        loss.backward()
        result["d_logits"] = logits.grad
        if s["value"] is not None:
            result["d_value"] = value.grad
    return result


def _exact_gae(s):
    """Step by step from the last one back."""
    sign = torch.cat([1 - 2 * s["player"].double(), 1 - 2 * s["last_player"].double()[None]])
    v = torch.cat([s["value"], s["bootstrap"][None]]).double()
    advantage = torch.zeros_like(v)
    live = (~s["done"]).double()
    turn = sign[:-1] * sign[1:] * live  # the next mover's side seen from this one's
    own_reward = sign[:-1] * s["reward"].double()
    for t in reversed(range(s["case"]["steps"])):
        advantage[t] = own_reward[t] - v[t] + GAMMA * turn[t] * (v[t + 1] + LAM * advantage[t + 1])
    return {"advantage": advantage[:-1], "returns": advantage[:-1] + v[:-1]}


def _exact_adamw(s):
    """Tensor by tensor in 64 bits; the 8-bit codes, whose rounding is drawn, have no value here."""
    beta1, beta2 = BETAS
    x, eight = s["lists"], s["m_scale"] is not None
    norm = torch.cat([g.double() for g in x["grad"]]).norm()
    coef = min(1.0, MAX_NORM / (float(norm) + 1e-6)) if s["case"]["clip"] else 1.0
    out = {k: None if s[k] is None else torch.zeros(s[k].shape, dtype=torch.float64, device="cuda")
           for k in ("param", "master", "m", "v", "m_scale", "v_scale")}
    at = 0
    for i, n in enumerate(s["sizes"]):
        blocks = -(-n // BLOCK)
        t = int(s["steps"][i]) + 1
        g = x["grad"][i].double() * coef
        m, v = x["m"][i].double(), x["v"][i].double()
        if eight:
            m = m * x["m_scale"][i].double().repeat_interleave(BLOCK)[:n]
            v = v * x["v_scale"][i].double().repeat_interleave(BLOCK)[:n]
        m = beta1 * m + (1 - beta1) * g
        v = beta2 * v + (1 - beta2) * g * g
        w = (x["master"] if x["master"] is not None else x["param"])[i].double()
        w = w - LR * (DECAY * w + m / (1 - beta1**t) / ((v / (1 - beta2**t)).sqrt() + EPS))
        for k in ("param", "master"):
            if out[k] is not None:
                out[k][at:at + n] = w
        if eight:
            for k, y, top in (("m_scale", m, 256.0), ("v_scale", v, 32768.0)):
                y = torch.nn.functional.pad(y.abs(), (0, blocks * BLOCK - n)).view(-1, BLOCK)
                out[k][at // BLOCK:at // BLOCK + blocks] = y.amax(1).clamp_min(2.0**-100) / top
        else:
            out["m"][at:at + n], out["v"][at:at + n] = m, v
        at += blocks * BLOCK
    if eight:
        out["m"] = out["v"] = None
    return {"norm": norm if s["case"]["clip"] else None, **out, "steps": s["steps"] + 1}
