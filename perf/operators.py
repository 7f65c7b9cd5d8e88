"""What the update-side operators cost: the clipped policy loss and the clipped value loss with their gradients, the global gradient
norm with clipping, and the products grouped by network.

A case names an operator and its sizes.  `run` computes it either in plain torch operations (`own = False`) or through this package's
public functions (`own = True`); `exact` gives the same outputs from the definition in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
CLIP, ENTROPY_COEF, KL_COEF = 0.2, 0.01, 0.05          # clip of the ratio, weight of the entropy, weight of the KL term
VALUE_CLIP, HUBER_DELTA = 0.2, 10.0
GRAD_SCALE = {"f32": 1.0, "bf16": 1.0, "f16": 1024.0}  # loss scaling: the mean over many rows leaves gradients below the range of f16
# the reference-architecture network on the 5 x 4 grid: conv 20 -> 32, 192 -> 64, 64 -> 64, head of 6
NETWORK = [(32, 20, 3, 3), (32,), (64, 192), (64,), (64, 64), (64,), (6, 64), (6,)]


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one kitchen's episode, both agents: the smallest update, where the latency of the call counts
        dict(name="policy_episode", op="policy_loss", how="grad", rows=400, actions=6, dtype="f32", available="rows", weights=True,
             kl=False, pad=0),
        # one of four minibatches of 200 steps x 65 536 kitchens x 2 agents, float actions as the minibatch generators yield them
        dict(name="policy_minibatch", op="policy_loss", how="grad", rows=6553600, actions=6, dtype="f32", available="one", weights=True,
             kl=True, pad=0),
        # a batch of tokens over a large vocabulary, KL to a reference policy, padded positions without weight
        dict(name="policy_tokens", op="policy_loss", how="grad", rows=4096, actions=32768, dtype="bf16", available="none", weights=True,
             kl=True, pad=0),
        # an odd vocabulary inside a padded row, through autograd
        dict(name="policy_tokens_odd", op="policy_loss", how="autograd", rows=1023, actions=50021, dtype="f16", available="none",
             weights=False, kl=True, pad=27),
        # the critic of that smallest update
        dict(name="value_episode", op="value_loss", how="grad", rows=400, dtype="f32", weights=True, normalizer=True, huber=True),
        # a whole batch of 200 steps x 65 536 kitchens x 2 agents, through autograd
        dict(name="value_batch", op="value_loss", how="autograd", rows=26214400, dtype="f32", weights=True, normalizer=True, huber=True),
        # one actor's gradients (8 tensors, 20 k elements)
        dict(name="clip_actor", op="clip_grad_norm", kind="networks", count=1, dtype="f32", clipped=True, align=64, sizes_seed=0),
        # 32 conventions' networks, 256 small tensors
        dict(name="clip_population", op="clip_grad_norm", kind="networks", count=32, dtype="f32", clipped=True, align=64, sizes_seed=0),
        # a large model's gradients: 290 tensors from vectors to matrices, bf16 among f32
        dict(name="clip_large", op="clip_grad_norm", kind="blocks", count=290, dtype="mixed", smallest=1000, largest=16000000,
             clipped=True, align=64, sizes_seed=3),
        # the first dense layer of 15 segments' critics over 61 k rows, forward and backward
        dict(name="grouped_critics", op="grouped_linear", how="train", groups=15, rows=61440, k=192, n=64, dtype="f32", spread=0.0, tail=0,
             sizes_seed=1),
        # single rows dealt to many networks: the weights are all there is to read
        dict(name="grouped_decode", op="grouped_linear", how="forward", groups=32, rows=61, k=2048, n=2048, dtype="bf16", spread=1.0, tail=0,
             sizes_seed=2),
        # a large training batch, ragged groups and rows behind the last one
        dict(name="grouped_large", op="grouped_linear", how="train", groups=16, rows=16411, k=2048, n=4096, dtype="bf16", spread=1.0, tail=27,
             sizes_seed=5),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["policy_loss", "policy_loss", "value_loss", "clip_grad_norm", "grouped_linear", "grouped_linear"])
    if op == "policy_loss":
        actions = _log_int(rng, 2, 131072)
        rows = _log_int(rng, 1, max(1, min(6000000, 100000000 // actions)))
        return dict(op=op, how=rng.choice(["grad", "autograd", "forward"]), rows=rows, actions=actions,
                    dtype=rng.choice(["f32", "bf16", "f16"]), available=rng.choice(["none", "one", "rows"]) if rows * actions < 50000000 else "none",
                    weights=rng.random() < 0.7, kl=rng.random() < 0.5, pad=rng.choice([0, 0, 1, 27, 64]))
    if op == "value_loss":
        return dict(op=op, how=rng.choice(["grad", "autograd", "forward"]), rows=_log_int(rng, 1, 26000000),
                    dtype=rng.choice(["f32", "f32", "bf16", "f16"]), weights=rng.random() < 0.7, normalizer=rng.random() < 0.5,
                    huber=rng.random() < 0.7)
    if op == "clip_grad_norm":
        if rng.random() < 0.3:
            return dict(op=op, kind="networks", count=_log_int(rng, 1, 64), dtype=rng.choice(["f32", "bf16"]), clipped=rng.random() < 0.7,
                        align=rng.choice([1, 64]), sizes_seed=rng.randrange(1000))
        count = _log_int(rng, 1, 600)
        largest = _log_int(rng, 1, max(1, min(16000000, 500000000 // count)))
        return dict(op=op, kind="blocks", count=count, dtype=rng.choice(["f32", "bf16", "f16", "mixed"]), smallest=1, largest=largest,
                    clipped=rng.random() < 0.7, align=rng.choice([1, 64]), sizes_seed=rng.randrange(1000))
    groups = _log_int(rng, 1, 64)
    k, n = _log_int(rng, 8, 4096), _log_int(rng, 8, 4096)
    if rng.random() < 0.6:
        k, n = max(8, k // 8 * 8), max(8, n // 8 * 8)
    dtype = rng.choice(["f32", "bf16", "f16"])
    most = (8e9 if dtype == "f32" else 1.2e11) / (k * n)
    rows = _log_int(rng, 1, max(1, min(60000, int(most))))
    return dict(op=op, how=rng.choice(["train", "forward"]), groups=groups, rows=rows, k=k, n=n, dtype=dtype, spread=rng.choice([0.0, 1.0]),
                tail=rng.choice([0, 0, 3]) if rows > 3 else 0, sizes_seed=rng.randrange(1000))


def _group_sizes(case):
    """Rows per group: even, or ragged (a few groups hold most, some none)."""
    rows, groups = case["rows"] - case["tail"], case["groups"]
    r = random.Random(case["sizes_seed"])
    share = [math.exp(case["spread"] * r.gauss(0.0, 0.8)) for _ in range(groups)]
    cuts, total, acc = [0], sum(share), 0.0
    for s in share:
        acc += s
        cuts.append(int(round(rows * acc / total)))
    cuts[-1] = rows
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _clip_shapes(case):
    """[(number of elements, dtype name)] of the gradients."""
    r = random.Random(case["sizes_seed"])
    if case["kind"] == "networks":
        return [(math.prod(s), case["dtype"]) for _ in range(case["count"]) for s in NETWORK]
    low, high = math.log(case["smallest"]), math.log(case["largest"])
    sizes = [int(round(math.exp(r.uniform(low, high)))) for _ in range(case["count"])]
    return [(s, ("bf16" if r.random() < 0.75 else "f32") if case["dtype"] == "mixed" else case["dtype"]) for s in sizes]


# --------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _policy_inputs(case, seed):
    g, rows, acts = _generator(seed), case["rows"], case["actions"]
    randn = lambda *s: torch.randn(s, device="cuda", generator=g)
    rand = lambda *s: torch.rand(s, device="cuda", generator=g)
    actions = torch.randint(0, acts, (rows,), device="cuda", generator=g)
    buf = (randn(rows, acts + case["pad"]) * 1.5).to(DTYPES[case["dtype"]])
    logits = buf[:, :acts]
    # the taken action is mostly a likely one, as it is when the policy that took it is nearly this one
    lift = torch.where(rand(rows) < 0.8, 0.7 * math.log(acts), 0.0)
    at = actions.unsqueeze(1)
    logits.scatter_(1, at, (logits.gather(1, at).float() + lift.unsqueeze(1)).to(logits.dtype))
    avail = None
    if case["available"] == "one":                     # every action of every row: the broadcast view that the generators yield
        avail = torch.ones((1, acts), device="cuda").expand(rows, -1)
    elif case["available"] == "rows":
        avail = (rand(rows, acts) < 0.85).float()
        avail.scatter_(1, at, 1.0)
        avail[rand(rows) < 0.01] = 0.0                 # rows that may do nothing
    z = logits.float() if avail is None else torch.where(avail != 0, logits.float(), -1e30)
    lp = (z.gather(1, at) - torch.logsumexp(z, 1, keepdim=True)).squeeze(1)
    del z
    change = randn(rows) * 0.15                        # log of the ratio
    # not within 1e-3 of the clip's border, where the gradient jumps and 32 and 64 bits fall on different sides
    for border in (math.log(1 - CLIP), math.log(1 + CLIP)):
        change = torch.where((change - border).abs() < 1e-3, torch.full_like(change, 0.01), change)
    old, ref = lp - change, lp - randn(rows) * 0.2
    adv = randn(rows)
    weights = (rand(rows) < 0.93).float() if case["weights"] else None
    if weights is not None and acts > 64:              # padded positions carry no action
        actions = torch.where((weights == 0) & (rand(rows) < 0.5), torch.full_like(actions, -1), actions)
    elif acts <= 64:
        actions = actions.float().unsqueeze(1)         # the reference's buffers hold actions as floats [n, 1]
    return dict(logits=logits, actions=actions, old=old, adv=adv, ref=ref if case["kl"] else None, weights=weights, avail=avail)


def _value_inputs(case, seed):
    g, rows = _generator(seed), case["rows"]
    randn = lambda: torch.randn((rows, 1), device="cuda", generator=g)
    mean, std = (3.0, 2.5) if case["normalizer"] else (0.0, 1.0)
    preds = randn()
    values = (preds + 0.25 * randn()).to(DTYPES[case["dtype"]])
    target = preds + randn() * 1.5 + 15.0 * (torch.rand((rows, 1), device="cuda", generator=g) < 0.02)
    returns = target * std + mean
    # off the borders where the gradient jumps: the clip's edge, and both errors equally large behind it
    v, t = values.double(), (returns.double() - mean) / std
    clipped = preds.double() + (v - preds.double()).clamp(-VALUE_CLIP, VALUE_CLIP)
    near = ((v - preds.double()).abs() - VALUE_CLIP).abs() < 1e-4
    near |= ((v - preds.double()).abs() > VALUE_CLIP) & (((t - v).abs() - (t - clipped).abs()).abs() < 1e-4)
    preds = torch.where(near, values.float() + 0.01, preds)
    weights = (torch.rand((rows, 1), device="cuda", generator=g) < 0.93).float() if case["weights"] else None
    return dict(values=values, preds=preds, returns=returns, weights=weights, norm=(mean, std) if case["normalizer"] else None)


def _clip_inputs(case, seed):
    g = _generator(seed)
    grads = [(torch.randn(n, device="cuda", generator=g) * 0.02).to(DTYPES[d]) for n, d in _clip_shapes(case)]
    total = math.sqrt(sum(n for n, _ in _clip_shapes(case))) * 0.02            # about the norm of such gradients
    # the clipped gradients go to flat buckets, one per type, each tensor at its place in them
    out, flat = [], []
    for name in sorted({d for _, d in _clip_shapes(case)}):
        places, end = [], 0
        for i, (n, d) in enumerate(_clip_shapes(case)):
            if d == name:
                places.append((i, end, n))
                end += -(-n // case["align"]) * case["align"]
        flat.append(torch.zeros(end, dtype=DTYPES[name], device="cuda"))
        out += [(i, flat[-1][a:a + n]) for i, a, n in places]
    return dict(grads=grads, max_norm=total * (0.3 if case["clipped"] else 10.0), out=[t for _, t in sorted(out, key=lambda p: p[0])], flat=flat)


def _grouped_inputs(case, seed):
    g, dt = _generator(seed), DTYPES[case["dtype"]]
    sizes = _group_sizes(case)
    cuts = [0]
    for s in sizes:
        cuts.append(cuts[-1] + s)
    rows, k, n, groups = case["rows"], case["k"], case["n"], case["groups"]
    randn = lambda *s: torch.randn(s, device="cuda", generator=g)
    return dict(x=randn(rows, k).relu_().to(dt), weight=(randn(groups, n, k) / math.sqrt(k)).to(dt), bias=(randn(groups, n) * 0.1).to(dt),
                dy=(randn(rows, n) / math.sqrt(rows)).to(dt), cuts=cuts, offsets=torch.tensor(cuts, dtype=torch.int32, device="cuda"))


_INPUTS = {"policy_loss": _policy_inputs, "value_loss": _value_inputs, "clip_grad_norm": _clip_inputs, "grouped_linear": _grouped_inputs}


def prepare(case, seed):
    state = _INPUTS[case["op"]](case, seed)
    state["case"] = case
    if case.get("how") == "autograd":
        state["logits" if case["op"] == "policy_loss" else "values"].requires_grad_()
        state["scale"] = torch.tensor(GRAD_SCALE[case["dtype"]], device="cuda")
    if case.get("how") == "train":
        for leaf in ("x", "weight", "bias"):
            state[leaf].requires_grad_()
    return state


# ------------------------------------------------------------------------------------------------------- the plain forms
def _plain_policy(s):
    case, acts = s["case"], s["case"]["actions"]
    z = s["logits"].float()
    action = s["actions"].reshape(-1).long()
    in_range = (action >= 0) & (action < acts)
    at = action.clamp(0, acts - 1).unsqueeze(1)
    possible = z != -math.inf
    if s["avail"] is not None:
        possible &= s["avail"] != 0
    top = torch.where(possible, z, -math.inf).amax(1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.where(possible, torch.exp(z - top), 0.0)
    total = e.sum(1, keepdim=True)
    logp = torch.where(possible, z - top - torch.log(total), 0.0)
    p = torch.where(total > 0, e / total, 0.0)
    entropy = -(p * logp).sum(1)
    weight = torch.ones_like(s["old"]) if s["weights"] is None else s["weights"]
    weight = torch.where(in_range, weight, 0.0)
    norm = weight.sum()
    counts = (weight != 0) & possible.gather(1, at).squeeze(1)
    w = torch.where(counts, weight / norm, 0.0)
    lp = torch.where(counts, logp.gather(1, at).squeeze(1), 0.0)
    old = torch.where(counts, s["old"], 0.0)
    adv = torch.where(counts, s["adv"], 0.0)
    ratio = torch.exp(lp - old)
    kept = torch.clamp(ratio, 1 - CLIP, 1 + CLIP)
    pol = -torch.minimum(ratio * adv, kept * adv)
    slope = -torch.where(((adv > 0) & (ratio > 1 + CLIP)) | ((adv < 0) & (ratio < 1 - CLIP)), 0.0, adv * ratio)
    kl = torch.zeros_like(lp)
    if s["ref"] is not None:
        d = torch.where(counts, s["ref"], 0.0) - lp
        kl = torch.exp(d) - d - 1
        slope = slope + KL_COEF * (1 - torch.exp(d))
    clipped = ((ratio < 1 - CLIP) | (ratio > 1 + CLIP)).float()
    means = [(w * t).sum() for t in (pol, torch.where(counts, entropy, 0.0), kl, clipped, ratio)]
    loss = means[0] - ENTROPY_COEF * means[1] + (KL_COEF * means[2] if s["ref"] is not None else 0.0)
    out = [loss, torch.stack(means)]
    if case["how"] == "forward":
        return out
    w = w * GRAD_SCALE[case["dtype"]]
    grad = (w * slope).unsqueeze(1) * (torch.zeros_like(p).scatter_(1, at, 1.0) - p)
    grad += (w * ENTROPY_COEF).unsqueeze(1) * p * (logp + entropy.unsqueeze(1))
    return out + [torch.where(counts.unsqueeze(1) & possible, grad, 0.0).to(s["logits"].dtype)]


def _plain_value(s):
    v, v0 = s["values"].float(), s["preds"]
    target = s["returns"] if s["norm"] is None else (s["returns"] - s["norm"][0]) / s["norm"][1]
    w = torch.ones_like(v0) if s["weights"] is None else s["weights"]
    w = torch.where(w != 0, w / w.sum(), 0.0)
    e0, e1 = target - v, target - (v0 + torch.clamp(v - v0, -VALUE_CLIP, VALUE_CLIP))
    if s["case"]["huber"]:
        h = lambda e: torch.where(e.abs() <= HUBER_DELTA, e * e / 2, HUBER_DELTA * (e.abs() - HUBER_DELTA / 2))
        slope = torch.clamp(e0, -HUBER_DELTA, HUBER_DELTA)
    else:
        h = lambda e: e * e / 2
        slope = e0
    h0, h1 = h(e0), h(e1)
    out = [(w * torch.maximum(h0, h1)).sum()]
    if s["case"]["how"] == "forward":
        return out
    return out + [torch.where(((v - v0).abs() <= VALUE_CLIP) | (h0 >= h1), -w * slope * GRAD_SCALE[s["case"]["dtype"]], 0.0).to(s["values"].dtype)]


def _plain_clip(s):
    norm = torch.sqrt(torch.stack([(t.float() ** 2).sum() for t in s["grads"]]).sum())
    scale = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    for t, place in zip(s["grads"], s["out"]):
        place.copy_(t.float() * scale)
    return [norm] + s["flat"]


def _plain_grouped(s):
    case, cuts = s["case"], s["cuts"]
    x, weight, bias = s["x"].float(), s["weight"].float(), s["bias"].float()
    y = torch.zeros((case["rows"], case["n"]), device=x.device)
    for g in range(case["groups"]):
        a, b = cuts[g], cuts[g + 1]
        y[a:b] = x[a:b] @ weight[g].t() + bias[g]
    out = [y.to(s["x"].dtype)]
    if case["how"] == "forward":
        return out
    dy = s["dy"].float()
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(weight), torch.zeros_like(bias)
    for g in range(case["groups"]):
        a, b = cuts[g], cuts[g + 1]
        dx[a:b] = dy[a:b] @ weight[g]
        dw[g] = dy[a:b].t() @ x[a:b]
        db[g] = dy[a:b].sum(0)
    return out + [t.to(s["x"].dtype) for t in (dx, dw, db)]


# ------------------------------------------------------------------------------------------------ the package's operators
def _own_policy(s):
    import diverse_conventions_amd as dc
    how = s["case"]["how"]
    args = (s["logits"], s["actions"], s["old"], s["adv"])
    kw = dict(clip_param=CLIP, entropy_coef=ENTROPY_COEF, kl_coef=KL_COEF, ref_log_probs=s["ref"], active_masks=s["weights"],
              available_actions=s["avail"])
    if how == "grad":
        return list(dc.policy_loss_grad(*args, grad_scale=GRAD_SCALE[s["case"]["dtype"]], **kw))
    loss, stats = dc.policy_loss(*args, **kw)
    return [loss, stats] if how == "forward" else [loss.detach(), stats, torch.autograd.grad(loss, s["logits"], s["scale"])[0]]


def _own_value(s):
    import diverse_conventions_amd as dc
    how = s["case"]["how"]
    args = (s["values"], s["preds"], s["returns"])
    kw = dict(clip_param=VALUE_CLIP, huber_delta=HUBER_DELTA if s["case"]["huber"] else None, active_masks=s["weights"],
              value_normalizer=s["norm"])
    if how == "grad":
        return list(dc.value_loss_grad(*args, grad_scale=GRAD_SCALE[s["case"]["dtype"]], **kw))
    loss = dc.value_loss(*args, **kw)
    return [loss] if how == "forward" else [loss.detach(), torch.autograd.grad(loss, s["values"], s["scale"])[0]]


def _own_clip(s):
    import diverse_conventions_amd as dc
    return [dc.clip_grad_norm(s["grads"], s["max_norm"], out=s["out"])] + s["flat"]


def _own_grouped(s):
    import diverse_conventions_amd as dc
    y = dc.grouped_linear(s["x"], s["weight"], s["offsets"], s["bias"])
    if s["case"]["how"] == "forward":
        return [y]
    return [y.detach(), *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])]


_PLAIN = {"policy_loss": _plain_policy, "value_loss": _plain_value, "clip_grad_norm": _plain_clip, "grouped_linear": _plain_grouped}
_OWN = {"policy_loss": _own_policy, "value_loss": _own_value, "clip_grad_norm": _own_clip, "grouped_linear": _own_grouped}


def run(state):
    if own:
        return _OWN[state["case"]["op"]](state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


# --------------------------------------------------------------------------------------------------- the work of one pass
def work(case):
    op = case["op"]
    grad = case.get("how") in ("grad", "autograd", "train")
    if op == "policy_loss":
        rows, acts, size = case["rows"], case["actions"], BYTES[case["dtype"]]
        per_row = 8 + (8 if acts > 64 else 4) + (4 if case["weights"] else 0) + (4 if case["kl"] else 0)
        moved = rows * (acts * size * (2 if grad else 1) + per_row)
        moved += {"none": 0, "one": 4 * acts, "rows": 4 * rows * acts}[case["available"]]
        return {"bytes": moved, "flops": rows * acts * (12 if grad else 6)}
    if op == "value_loss":
        size = BYTES[case["dtype"]]
        return {"bytes": case["rows"] * (8 + size + (4 if case["weights"] else 0) + (size if grad else 0)), "flops": case["rows"] * 16}
    if op == "clip_grad_norm":
        shapes = _clip_shapes(case)
        return {"bytes": 2 * sum(n * BYTES[d] for n, d in shapes), "flops": 3 * sum(n for n, _ in shapes)}
    size, groups, k, n, rows = BYTES[case["dtype"]], case["groups"], case["k"], case["n"], case["rows"]
    used = [r for r in _group_sizes(case) if r]
    m = sum(used)
    x, y, w = m * k, rows * n, len(used) * n * k
    if not grad:
        return {"bytes": size * (x + y + w + len(used) * n), "flops": 2 * m * n * k}
    # read x, weight, bias, dy; write y, dx, dw, db
    return {"bytes": size * (x + w + len(used) * n + m * n + y + rows * k + groups * n * k + groups * n), "flops": 6 * m * n * k}


# ------------------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_policy(case, s):
    acts = case["actions"]
    z = s["logits"].double()
    keep = torch.isfinite(z) if s["avail"] is None else torch.isfinite(z) & (s["avail"] != 0)
    z = torch.where(keep, z, torch.full_like(z, -1e300)).requires_grad_(case["how"] != "forward")
    action = s["actions"].reshape(-1).long()
    valid = (action >= 0) & (action < acts)
    action = torch.where(valid, action, torch.zeros_like(action))
    weight = valid.double() * (1.0 if s["weights"] is None else s["weights"].double())
    norm = weight.sum()
    used = weight.ne(0) & keep[torch.arange(len(action), device=z.device), action]
    share = (weight / norm)[used]
    logp = torch.log_softmax(z, 1)
    lp = logp[torch.arange(len(action), device=z.device), action][used]
    entropy = -(logp.exp() * logp).sum(1)[used]
    ratio = torch.exp(lp - s["old"].double()[used])
    adv = s["adv"].double()[used]
    pol = -torch.minimum(ratio * adv, ratio.clamp(1 - CLIP, 1 + CLIP) * adv)
    kl = torch.zeros_like(lp)
    if s["ref"] is not None:
        d = s["ref"].double()[used] - lp
        kl = d.exp() - 1 - d
    outside = ((ratio - 1).abs() > CLIP).double()
    means = torch.stack([(share * t).sum() for t in (pol, entropy, kl, outside, ratio)])
    loss = means[0] - ENTROPY_COEF * means[1] + KL_COEF * means[2]
    out = [loss.detach(), means.detach()]
    return out if case["how"] == "forward" else out + [torch.autograd.grad(loss * GRAD_SCALE[case["dtype"]], z)[0]]


def _exact_value(case, s):
    v = s["values"].double().requires_grad_(case["how"] != "forward")
    v0, mean_std = s["preds"].double(), s["norm"] or (0.0, 1.0)
    target = (s["returns"].double() - mean_std[0]) / mean_std[1]
    w = torch.ones_like(v0) if s["weights"] is None else s["weights"].double()

    def h(e):
        if not case["huber"]:
            return 0.5 * e ** 2
        inner = e.abs().clamp(max=HUBER_DELTA)
        return inner * (e.abs() - 0.5 * inner)

    worst = torch.max(h(target - v), h(target - v0 - (v - v0).clamp(-VALUE_CLIP, VALUE_CLIP)))
    loss = (w * worst).sum() / w.sum().clamp(min=1e-300)
    return [loss.detach()] if case["how"] == "forward" else [loss.detach(), torch.autograd.grad(loss * GRAD_SCALE[case["dtype"]], v)[0]]


def _exact_clip(case, s):
    squares = 0.0
    for t in s["grads"]:
        squares = squares + t.double().pow(2).sum()
    norm = squares ** 0.5
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    out = [norm]
    for bucket in s["flat"]:
        whole = torch.zeros(len(bucket), dtype=torch.float64, device=bucket.device)
        for t, place in zip(s["grads"], s["out"]):
            if place.dtype == bucket.dtype:
                first = place.storage_offset()
                whole[first:first + len(t)] = t.double() * factor
        out.append(whole)
    return out


def _exact_grouped(case, s):
    dev = s["x"].device
    y = torch.zeros(case["rows"], case["n"], dtype=torch.float64, device=dev)
    dx = torch.zeros(case["rows"], case["k"], dtype=torch.float64, device=dev)
    dw = torch.zeros(case["groups"], case["n"], case["k"], dtype=torch.float64, device=dev)
    db = torch.zeros(case["groups"], case["n"], dtype=torch.float64, device=dev)
    for g, (first, last) in enumerate(zip(s["cuts"], s["cuts"][1:])):
        if last == first:
            continue
        rows, w, d = s["x"][first:last].double(), s["weight"][g].double(), s["dy"][first:last].double()
        y[first:last] = torch.addmm(s["bias"][g].double(), rows, w.t().contiguous())
        if case["how"] == "train":
            dx[first:last] = torch.mm(d, w)
            dw[g] = torch.mm(d.t().contiguous(), rows)
            db[g] = d.sum(0)
    return [y] if case["how"] == "forward" else [y, dx, dw, db]


def exact(case, seed):
    s = _INPUTS[case["op"]](case, seed)
    fn = {"policy_loss": _exact_policy, "value_loss": _exact_value, "clip_grad_norm": _exact_clip, "grouped_linear": _exact_grouped}
    return fn[case["op"]](case, s)
