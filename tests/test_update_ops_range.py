"""The update-side operators at the edges of their inputs' range: logits far from 0, policies next to their reference, values that are not
numbers, calls that are refused.  Definitions in float64 as in test_update_ops.py, whose tolerance (ROW, derived there) is used per element:

A logit's gradient is c1 ([j taken] - p_j) + ce p_j (log p_j + H) times the row's share of the weight.  p_j carries a relative error of at
most 2^-24 (3 |log p_j| + 2) from its exponential and 7e-6 from the sum, log p_j + H an absolute one of 2^-22 (|log p_j| + H), c1 that of the
row's terms: together less than ROW (1 + |log p_j|) p_j of the row's terms, and ROW of them where j is taken.  Below 1e-37 f32 leaves its
normal range.  Where an action is not possible the gradient is 0 and nothing else.
"""
import math

import numpy as np
import pytest
import torch

from test_update_ops import DTYPES, POLICY_SIZES, ROW, check_policy, f64, half_step, oracle_policy, policy_inputs, value_inputs


def masked_log_softmax(s):
    z = torch.from_numpy(f64(s["logits"]))
    if s["avail"] is not None:
        z = torch.where(s["avail"].cpu() != 0, z, -math.inf)
    return torch.log_softmax(z, 1).numpy()


def gradient_excess(s, grad, scale, clip=0.2, entropy_coef=0.01, kl_coef=0.05):
    """-> [rows, actions]: by how much the error of each element is above its bound (positive: wrong)"""
    _, _, want, size = oracle_policy(s, clip=clip, entropy_coef=entropy_coef, kl_coef=kl_coef)
    want = want * scale
    logp = masked_log_softmax(s)
    impossible = ~(logp > -np.inf)                         # and rows that nothing is possible in (NaN)
    logp = np.where(impossible, 0.0, logp)
    share = np.where(impossible, 0.0, np.exp(logp) * (1 + np.abs(logp)))
    a = f64(s["actions"]).reshape(-1)
    for r in np.flatnonzero((a >= 0) & (a < want.shape[1])):
        share[r, int(a[r])] += 1.0
    bound = ROW * scale * size[:, None] * share + half_step(want, s["logits"].dtype) + 1e-37 * scale * size[:, None]
    return np.abs(grad - want) - np.where(impossible, 0.0, bound)


def check_gradient(s, grad, scale, **kw):
    excess = gradient_excess(s, f64(grad), scale, **kw)
    assert np.all(excess <= 0), (float(np.nanmax(excess)), np.argwhere(~(excess <= 0))[:5])


def around_the_logits(s, seed):
    """old and reference log-probabilities near those of the logits as they are stored, away from the clip's borders"""
    g = torch.Generator().manual_seed(seed)
    rows = len(s["actions"])
    lp = torch.from_numpy(masked_log_softmax(s))[torch.arange(rows), s["actions"].cpu()]
    change = torch.randn(rows, generator=g, dtype=torch.float64) * 0.2
    for border in (math.log(0.8), math.log(1.2)):
        change = torch.where((change - border).abs() < 1e-3, torch.full_like(change, 0.01), change)
    s["old"] = (lp - change).float().to(s["logits"].device)
    s["ref"] = (lp + 0.2 * torch.randn(rows, generator=g, dtype=torch.float64)).float().to(s["logits"].device)
    return lp


def fused_autograd_and_value(s, scale=1.0, **coefs):
    """The operator's three ways, checked against the definition."""
    from diverse_conventions_amd import policy_loss, policy_loss_grad
    kw = dict(kl_coef=0.05, ref_log_probs=s["ref"], active_masks=s["weights"], available_actions=s["avail"]) | coefs
    fused = policy_loss_grad(s["logits"], s["actions"], s["old"], s["adv"], grad_scale=scale, **kw)
    leaf = s["logits"].clone().requires_grad_()
    loss, stats = policy_loss(leaf, s["actions"], s["old"], s["adv"], **kw)
    (grad,) = torch.autograd.grad(loss, leaf, torch.tensor(scale, device="cuda"))
    with torch.no_grad():
        value = policy_loss(leaf, s["actions"], s["old"], s["adv"], **kw)
    return fused, (loss.detach(), stats, grad), value


# ------------------------------------------------------------------------------------------------- logits far from 0, finite masks
RANGES = [("all", f) for f in (1e9, -1e9, 1e10, -1e10, -1e20, 1e30, -1e30, -6e4)] + [("few", f) for f in (-1e9, -1e10, -1e30, -6e4)] + \
         [("shift", f) for f in (30.0, -30.0, 1e3, 1e4, 1e6)]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [6, 13, 40, 300, 5000, 40000, 140000])
@pytest.mark.parametrize("kind,value,dtype", [(k, v, d) for k, v in RANGES for d, t in DTYPES.items() if abs(v) <= torch.finfo(t).max],
                         ids=lambda v: v if isinstance(v, str) else f"{v:g}")
def test_policy_loss_of_logits_far_from_zero(kind, value, n, dtype):
    """Rows of one large value (uniform), a few ordinary logits among a finite fill (whole wavefronts and lanes see only the fill), all
    logits shifted: the loss is that of the differences, whatever they are relative to."""
    dt = DTYPES[dtype]
    rows, scale = 3, 1024.0 if dtype == "f16" else 1.0
    s = policy_inputs(n + 1, rows, n, torch.float32, "none", False, True, "cuda")
    z = s["logits"]
    if kind == "all":
        z.fill_(value)
    elif kind == "shift":
        z += value
    else:
        keep = torch.tensor(sorted({1, n // 3, n // 2, n - 2}), device="cuda")
        few = torch.full_like(z, value)
        few[:, keep] = z[:, keep]
        z.copy_(few)
        s["actions"] = keep[torch.arange(rows, device="cuda") % len(keep)]
    s["logits"] = z.to(dt)
    around_the_logits(s, n)
    fused, auto, plain = fused_autograd_and_value(s, scale)
    for r in (fused, auto):
        check_policy(s, r, scale)
        check_gradient(s, r[2], scale)
    assert torch.equal(plain[0], auto[0]) and torch.equal(plain[1], auto[1])


# ------------------------------------------------------------------------------------------------ policies next to their reference
@pytest.mark.gpu
@pytest.mark.parametrize("n,rows", [(6, 4000), (13, 1000), (40, 1000), (5000, 200)])
@pytest.mark.parametrize("spread", [0.0, 1e-4, 1e-3, 3e-2, 0.3, 2.0])
def test_policy_loss_kl_next_to_the_reference_policy(spread, n, rows):
    """kl = exp(d) - d - 1 with d = ref - lp is about d^2 / 2 and never negative.  lp carries at most
    t = 2^-24 (3 (log n + 1) + 2 + min(n, 64) + 4 |lp| + 4): the sum's error (as above, with at most 64 roundings of a partial sum), the
    logarithm's and the two products'; kl therefore |exp(d) - 1| t + exp(d) t^2, the rounding of a few operations (2^-21 of it) and, where
    d is large enough to subtract, that of exp(d)."""
    s = policy_inputs(n, rows, n, available="none", weights=False, device="cuda")
    lp = around_the_logits(s, n).numpy()
    g = torch.Generator().manual_seed(rows)
    s["ref"] = torch.from_numpy(lp + spread * torch.randn(rows, generator=g, dtype=torch.float64).numpy()).float().cuda()
    s["adv"].zero_()
    fused, auto, _ = fused_autograd_and_value(s, kl_coef=1.0, entropy_coef=0.0)
    d = f64(s["ref"]) - lp
    kl = np.where(np.abs(d) < 1e-3, d * d / 2 * (1 + d / 3 + d * d / 12), np.expm1(d) - d)
    t = 2.0 ** -24 * (3 * (math.log(n) + 1) + 6 + min(n, 64) + 4 * np.abs(lp))
    bound = np.abs(np.expm1(d)) * t + np.exp(d) * t * t + 2.0 ** -21 * kl + np.where(np.abs(d) > 0.2, 2.0 ** -22 * (np.exp(d) + np.abs(d)), 0.0)
    taken = np.arange(rows), f64(s["actions"]).astype(int)
    want = -np.expm1(d) * -np.expm1(lp) / rows             # (1 - exp(d)) (1 - p) of the taken action
    for loss, stats, grad in (fused, auto):
        got = float(stats[2].double())
        assert got >= 0 and abs(got - kl.mean()) <= bound.mean() + 2.0 ** -23 * kl.mean(), (got, kl.mean(), bound.mean())
        assert abs(float(loss.double()) - kl.mean()) <= bound.mean() + 2.0 ** -23 * kl.mean()
        assert np.all(np.abs(f64(grad)[taken] - want) <= (np.exp(d) * t + 4 * t * np.abs(np.expm1(d))) / rows)


# ----------------------------------------------------------------------------------------------------- what is not a number beside masks
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [6, 40, 300, 5000, 70001, 140000])
def test_policy_loss_impossible_actions_get_zero_in_every_row(n, dtype):
    """Rows whose terms are not finite though their logits are: an advantage or a log-probability that is NaN, a ratio or a KL term that
    overflows.  Their impossible actions still get 0, the other rows are as ever."""
    s = policy_inputs(n, 7, n, DTYPES[dtype], "rows", False, True, "cuda")
    lp = around_the_logits(s, n)
    clean = s["logits"].clone()
    free = torch.where(torch.arange(n) == (s["actions"][6].item() + 1) % n, -math.inf, 0.0)      # -inf as a mask of its own
    s["logits"][6] = clean[6] + free.to(clean)
    s["adv"][1] = math.nan
    s["old"][2], s["adv"][2] = float(lp[2]) - 200.0, -1.0                   # ratio exp(200)
    s["old"][3] = math.nan
    s["ref"][4] = math.nan
    s["ref"][5] = 300.0
    s["ref"][6] = 300.0
    impossible = (s["avail"] == 0) | (s["logits"] == -math.inf)
    assert impossible.any()
    fused, auto, _ = fused_autograd_and_value(s)
    for _, _, grad in (fused, auto):
        assert not grad[impossible].isnan().any() and not grad[impossible].any()
        assert torch.isfinite(grad[0]).all()
        assert all(not torch.isfinite(grad[r]).all() for r in range(1, 7))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [6, 13, 40, 5000, 70001])
def test_policy_loss_gradient_of_a_large_scale(n):
    """A gradient scaled by 1e12: actions whose probability is 0 in f32 get 0, masked ones too."""
    s = policy_inputs(n, 5, n, available="rows", weights=False, device="cuda")
    a = s["actions"]
    far = (torch.rand((5, n), device="cuda", generator=torch.Generator("cuda").manual_seed(n)) < 0.5) & (torch.arange(n, device="cuda") != a[:, None])
    s["logits"][far] = -1e30
    s["logits"][0, (a[0] + 1) % n] = -1e30
    around_the_logits(s, n)
    fused, auto, _ = fused_autograd_and_value(s, 1e12)
    for r in (fused, auto):
        check_gradient(s, r[2], 1e12)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [6, 40, 5000, 70001])
def test_policy_loss_kl_of_an_action_of_no_probability_is_infinite(n):
    """The taken action at the type's lowest value: its log-probability is beyond f32 in units of log 2, exp(ref - lp) - (ref - lp) - 1 is
    infinite and not NaN; without the KL term the row is an ordinary one of ratio 0."""
    for value in (torch.finfo(torch.float32).min, -3e38):
        s = policy_inputs(n, 4, n, available="none", weights=False, device="cuda")
        s["logits"][1, s["actions"][1]] = value
        fused, auto, plain = fused_autograd_and_value(s)
        for loss, stats, *_ in (fused, auto, plain):
            assert float(loss) == math.inf and float(stats[2]) == math.inf and torch.isfinite(stats[[0, 1, 3, 4]]).all()
        s["ref"] = None
        fused, auto, plain = fused_autograd_and_value(s)
        for r in (fused, auto):
            check_policy(s, r)
            check_gradient(s, r[2], 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [6, 40, 5000])
def test_policy_loss_of_a_zero_advantage_and_a_ratio_beyond_f32(n):
    """An advantage of 0 contributes 0 however large the ratio: old log-probabilities 100 below, with and without a clip."""
    s = policy_inputs(n, 4, n, available="none", weights=False, ref=False, device="cuda")
    lp = around_the_logits(s, n)
    s["old"][1], s["adv"][1], s["ref"] = float(lp[1]) - 100.0, 0.0, None
    s["old"][2], s["adv"][2] = float(lp[2]) - 100.0, 1.5                    # clipped: no gradient through the ratio
    for clip in (0.2, math.inf):
        if clip == math.inf:
            s["adv"][2] = 0.0
        fused, auto, plain = fused_autograd_and_value(s, clip_param=clip)
        want, means, _, size = oracle_policy(s, clip=clip, kl_coef=0.05)
        size[1:3] = 1.0                                    # the ratio's size times 0 is no measure; the terms are below 1
        for r in (fused, auto, plain):
            assert abs(float(r[0]) - want) <= ROW * (abs(want) + size.sum()), (float(r[0]), want)
            assert abs(float(r[1][0]) - means[0]) <= ROW * (abs(means[0]) + size.sum()) and float(r[1][4]) == math.inf
        for r in (fused, auto):
            check_gradient(s, r[2], 1.0, clip=clip)
            entropy_only = f64(r[2])[1:3]
            assert np.all(np.abs(entropy_only) <= 0.01 * (1 + math.log(n)))


@pytest.mark.gpu
@pytest.mark.parametrize("n,at", [(40, 5), (41, 40), (5003, 5002), (70000, 333)])
def test_value_loss_shows_old_values_that_are_not_numbers(n, at):
    """max(h(e0), h(e1)) is not a number where the rollout's value is none; without the clipped branch that value is not looked at."""
    from diverse_conventions_amd import value_loss, value_loss_grad
    v, v0, ret, w = value_inputs(n, n, torch.float32, True, None)
    v0[at], w[at] = math.nan, 1.0
    others = torch.arange(n, device="cuda") != at
    for delta in (10.0, None):
        leaf = v.clone().requires_grad_()
        one = value_loss(leaf, v0, ret, huber_delta=delta, active_masks=w)
        for loss, grad in (value_loss_grad(v, v0, ret, huber_delta=delta, active_masks=w), (one, torch.autograd.grad(one, leaf)[0])):
            assert torch.isnan(loss) and torch.isnan(grad[at]) and torch.isfinite(grad[others]).all()
        loss, grad = value_loss_grad(v, v0, ret, clip_param=None, huber_delta=delta, active_masks=w)
        assert torch.isfinite(loss) and torch.isfinite(grad).all()
        skipped = torch.where(others, w, 0.0)
        loss, grad = value_loss_grad(v, v0, ret, huber_delta=delta, active_masks=skipped)
        assert torch.isfinite(loss) and torch.isfinite(grad).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [6, 40, 5000])
def test_policy_loss_actions_stored_as_floats(n):
    """Outside [0, actions) is padding, also between -1 and 0; -0.0 is action 0."""
    s = policy_inputs(n, 8, n, available="none", device="cuda")
    s["weights"][:] = 1.0
    s["actions"] = torch.tensor([-0.5, -0.0, n - 1.0, float(n), math.nan, math.inf, -1e-30, -1.0], device="cuda")
    floats, _, _ = fused_autograd_and_value(s)
    s["actions"] = torch.tensor([-1, 0, n - 1, n, -1, -1, -1, -1], device="cuda")
    whole, _, _ = fused_autograd_and_value(s)
    assert all(torch.equal(a, b) for a, b in zip(floats, whole))
    check_policy(s, floats)
    # 1024 rows and more: the weights are added up by a launch of their own
    big = policy_inputs(n, 1500 + n % 7, min(n, 40), available="none", weights=False, device="cuda")
    a = torch.where(torch.arange(len(big["actions"]), device="cuda") % 3 == 0, -0.5, big["actions"].float())
    big["actions"] = a
    floats, _, _ = fused_autograd_and_value(big)
    big["actions"] = torch.where(a < 0, -1, a.long())
    whole, _, _ = fused_autograd_and_value(big)
    assert all(torch.equal(x, y) for x, y in zip(floats, whole))


@pytest.mark.gpu
def test_policy_loss_actions_stored_as_floats_beyond_their_whole_numbers():
    """2^24 + 1 actions: the number of actions is no float of its own, its last action is."""
    from diverse_conventions_amd import policy_loss_grad
    n = 2 ** 24 + 1
    z, one = torch.zeros((1, n), dtype=torch.bfloat16, device="cuda"), torch.ones(1, device="cuda")
    last = torch.tensor([n - 1], device="cuda")
    assert int(last.float()) == n - 1
    want = policy_loss_grad(z, last, -math.log(n) * one, one)
    got = policy_loss_grad(z, last.float(), -math.log(n) * one, one)
    assert float(want[1][4]) > 0.9 and all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------------------------------------------------------------ refusals
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_forward_mode_is_refused(device):
    """The operators have no forward-mode derivative: a dual tensor is refused, not stripped of its tangent.  Inside a dual level calls
    without tangents work."""
    import torch.autograd.forward_ad as forward_ad
    from diverse_conventions_amd import clip_grad_norm, grouped_linear, policy_loss, policy_loss_grad, value_loss, value_loss_grad
    z, a, r = torch.zeros((4, 6), device=device), torch.zeros(4, dtype=torch.int64, device=device), torch.zeros(4, device=device)
    x, w, o, b = torch.ones((4, 8), device=device), torch.ones((1, 3, 8), device=device), torch.tensor([0, 4], device=device), torch.ones((1, 3), device=device)
    calls = []
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for fn in (policy_loss, policy_loss_grad):
            calls += [lambda fn=fn: fn(dual(z), a, r, r), lambda fn=fn: fn(z, a, dual(r), r), lambda fn=fn: fn(z, a, r, dual(r)),
                      lambda fn=fn: fn(z, a, r, r, ref_log_probs=dual(r)), lambda fn=fn: fn(z, a, r, r, active_masks=dual(r))]
        for fn in (value_loss, value_loss_grad):
            calls += [lambda fn=fn: fn(dual(r), r, r), lambda fn=fn: fn(r, dual(r), r), lambda fn=fn: fn(r, r, dual(r)),
                      lambda fn=fn: fn(r, r, r, active_masks=dual(r))]
        calls += [lambda: grouped_linear(dual(x), w, o, b), lambda: grouped_linear(x, dual(w), o, b), lambda: grouped_linear(x, w, o, dual(b)),
                  lambda: grouped_linear(dual(x), w.clone().requires_grad_(), o), lambda: clip_grad_norm([r, dual(x)], 1.0)]
        for call in calls:
            with pytest.raises(RuntimeError, match="forward mode"):
                call()
        if device == "cuda":
            policy_loss(z, a, r, r), value_loss(r, r, r), grouped_linear(x, w, o, b), clip_grad_norm([x], 1.0)


@pytest.mark.gpu
def test_value_loss_with_a_normalizer_object():
    """An object with running_mean_var() is read back at the call and gives what its (mean, standard deviation) pair gives."""
    from diverse_conventions_amd import value_loss, value_loss_grad

    class Normalizer:
        def running_mean_var(self):
            return torch.tensor([1.5], device="cuda"), torch.tensor([6.25], device="cuda")

    v, v0, ret, w = value_inputs(3, 5000, torch.float32, True, (1.5, 2.5))
    for a, b in zip(value_loss_grad(v, v0, ret, active_masks=w, value_normalizer=Normalizer()), value_loss_grad(v, v0, ret, active_masks=w, value_normalizer=(1.5, 2.5))):
        assert torch.equal(a, b)
    leaf = v.clone().requires_grad_()
    (x,) = torch.autograd.grad(value_loss(leaf, v0, ret, active_masks=w, value_normalizer=Normalizer()), leaf)
    (y,) = torch.autograd.grad(value_loss(leaf, v0, ret, active_masks=w, value_normalizer=(1.5, 2.5)), leaf)
    assert torch.equal(x, y)


# ------------------------------------------------------------------------------------------------- every element of the gradient
def gradient_case(rows, n, k, dtype, device):
    """The inputs of the sizes' test in test_update_ops.py; float16 gradients are scaled so that those of long rows stay above its subnormals."""
    available, weights, ref = [("none", False, False), ("rows", True, True), ("one", True, False)][k]
    s = policy_inputs(rows * 7 + n + k, rows, n, DTYPES[dtype], available, weights, ref, device)
    return s, 4096.0 if dtype == "f16" and n > 100 else 64.0 if dtype == "f16" else 1.0


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,n", [(400, 6), (40, 255), (5, 1000), (2, 16385), (1, 50021), (2, 70001), (1, 131072)])
def test_the_gradient_check_notices_what_is_left_out(rows, n, dtype):
    """On the definition itself: rounded to the type it passes; without the actions that were not taken, or without a row's last piece, it
    does not."""
    for k in range(3):
        s, scale = gradient_case(rows, n, k, dtype, "cpu")
        if s["weights"] is not None:
            s["weights"][0] = 0.7
        grad = oracle_policy(s, kl_coef=0.05)[2] * scale
        rounded = f64(torch.from_numpy(grad).to(DTYPES[dtype]))
        assert np.all(gradient_excess(s, rounded, scale) <= 0)
        taken = np.zeros(grad.shape, bool)
        taken[np.arange(rows), f64(s["actions"]).astype(int)] = True
        only = gradient_excess(s, np.where(taken, rounded, 0.0), scale)
        wanted = (grad != 0) & ~taken
        assert np.mean(only[wanted] > 0) > 0.75, np.mean(only[wanted] > 0)
        tail = rounded.copy()
        tail[:, -8:] = np.where(taken, rounded, 0.0)[:, -8:]
        assert np.any(gradient_excess(s, tail, scale) > 0)
        assert np.any(gradient_excess(s, rounded * (1 + 1e-2), scale) > 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,n", POLICY_SIZES)
def test_policy_loss_every_element_of_the_gradient(rows, n, dtype):
    for k in range(3):
        s, scale = gradient_case(rows, n, k, dtype, "cuda")
        fused, auto, _ = fused_autograd_and_value(s, scale)
        for r in (fused, auto):
            check_gradient(s, r[2], scale)


@pytest.mark.gpu
def test_policy_loss_every_element_of_rows_read_twice():
    """Rows longer than the registers hold, with a mask, in a padded buffer, and the rows that the test of offsets beyond 32 bits compares with."""
    s = policy_inputs(3, 4, 70001, torch.bfloat16, "none", False, False, "cuda")
    from diverse_conventions_amd import policy_loss_grad
    check_gradient(s, policy_loss_grad(s["logits"], s["actions"], s["old"], s["adv"])[2], 1.0, kl_coef=0.0)
    s = policy_inputs(5, 3, 70003, torch.float32, "rows", True, True, "cuda")
    s["weights"][:] = 1.0
    wide = torch.full((3, 70010), math.nan, device="cuda")
    wide[:, 3:70006] = s["logits"]
    s["logits"] = wide[:, 3:70006]
    fused, auto, _ = fused_autograd_and_value(s)
    for r in (fused, auto):
        check_gradient(s, r[2], 1.0)


# ------------------------------------------------------------------------------------------------- the autograd forms in a graph
@pytest.mark.gpu
def test_losses_through_autograd_in_a_captured_graph():
    """Forward and backward captured once and replayed on new inputs, eager calls and synchronisations between the replays."""
    from diverse_conventions_amd import policy_loss, value_loss
    small = policy_inputs(31, 9001, 6, device="cuda")
    long = policy_inputs(32, 5, 5000, torch.bfloat16, device="cuda", available="none")
    v, v0, ret, w = value_inputs(33, 9001, torch.float32, True, (1.0, 2.0))
    leaves = [t.requires_grad_() for t in (small["logits"], long["logits"], v)]

    def step():
        out = []
        for s in (small, long):
            loss, stats = policy_loss(s["logits"], s["actions"], s["old"], s["adv"], kl_coef=0.05, ref_log_probs=s["ref"], active_masks=s["weights"],
                                      available_actions=s["avail"])
            out += [loss.detach(), stats, *torch.autograd.grad(loss * 3.0, s["logits"])]
        loss = value_loss(v, v0, ret, active_masks=w, value_normalizer=(1.0, 2.0))
        return out + [loss.detach(), *torch.autograd.grad(loss, v)]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        with torch.no_grad():
            for t in leaves:
                t.normal_()
            small["weights"].uniform_()
        graph.replay()
        torch.cuda.synchronize()
        seen = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(seen, want)), k
