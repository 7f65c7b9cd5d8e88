"""The update-side operators (policy_loss, value_loss, clip_grad_norm) against their definitions in float64 (oracle/update_oracle.py).

Tolerances.  A row's softmax sums carry a relative error of at most 2^-24 (3 |u| + 2) per term exp(u) (rounding of z - m, of the product
with log2 e, of exp2) plus the rounding of the sum, and sum p |u| <= log A + 1: at most 2^-24 (3 (log A + 1) + 2 + 64) < 7e-6 for A up to
2^18.  lp, the ratio and every term of the gradient inherit that once or twice: 3e-5 of the row's terms.  A result of type T is
rounded once more: half a step, eps(T) / 2 of its value, and half the smallest subnormal for float16.
"""
import math

import numpy as np
import pytest
import torch

from oracle import update_oracle

ROW = 3e-5
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(x, dtype):
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return np.abs(x) * torch.finfo(dtype).eps / 2 + tiny


def f64(t):
    return t.detach().double().cpu().numpy()


# ---------------------------------------------------------------------------------------------------------- definitions (CPU)
def policy_inputs(seed, rows, n, dtype=torch.float32, available="rows", weights=True, ref=True, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((rows, n), generator=g) * 2).to(dtype)
    actions = torch.randint(0, n, (rows,), generator=g)
    avail = None
    if available == "rows":
        avail = (torch.rand((rows, n), generator=g) < 0.8).float()
        avail[torch.arange(rows), actions] = 1.0
    elif available == "one":
        avail = torch.ones((1, n)).expand(rows, n)
    z = logits.double() if avail is None else torch.where(avail != 0, logits.double(), -math.inf)
    lp = (torch.log_softmax(z, 1).gather(1, actions[:, None]).squeeze(1))
    change = torch.randn(rows, generator=g, dtype=torch.float64) * 0.2
    for border in (math.log(0.8), math.log(1.2)):          # the gradient jumps there: 32 and 64 bits may not fall on different sides
        change = torch.where((change - border).abs() < 1e-3, torch.full_like(change, 0.01), change)
    out = dict(logits=logits, actions=actions, old=(lp - change).float(), adv=torch.randn(rows, generator=g),
               ref=(lp + 0.2 * torch.randn(rows, generator=g, dtype=torch.float64)).float() if ref else None,
               weights=(torch.rand(rows, generator=g) < 0.8).float() * torch.rand(rows, generator=g) if weights else None, avail=avail)
    return {k: v.to(device) if v is not None and k != "avail" else v for k, v in out.items()} | {
        "avail": None if avail is None else avail.to(device) if available == "rows" else torch.ones((1, n), device=device).expand(rows, n)}


def oracle_policy(s, **kw):
    with np.errstate(all="ignore"):
        return update_oracle.policy_loss(f64(s["logits"]), f64(s["actions"]), f64(s["old"]), f64(s["adv"]), ref=None if s["ref"] is None else f64(s["ref"]),
                                         weights=None if s["weights"] is None else f64(s["weights"]), available=None if s["avail"] is None else f64(s["avail"]), **kw)


def test_oracle_policy_gradient_equals_differences():
    s = policy_inputs(3, 7, 5)
    kw = dict(entropy_coef=0.05, kl_coef=0.3)
    s["logits"] = s["logits"].double()
    _, _, grad, _ = oracle_policy(s, **kw)
    h, z = 1e-6, s["logits"]
    for r in range(7):
        for j in range(5):
            d = torch.zeros_like(z)
            d[r, j] = h
            diff = (oracle_policy(dict(s, logits=z + d), **kw)[0] - oracle_policy(dict(s, logits=z - d), **kw)[0]) / (2 * h)
            assert abs(diff - grad[r, j]) < 1e-8, (r, j)


@pytest.mark.parametrize("delta", [None, 0.7])
def test_oracle_value_gradient_equals_differences(delta):
    rng = np.random.default_rng(0)
    v, v0, ret, w = rng.normal(size=40), rng.normal(size=40), rng.normal(size=40) * 2, rng.random(40)
    v0 = np.where(np.abs(np.abs(v - v0) - 0.2) < 1e-3, v, v0)
    kw = dict(delta=delta, weights=w, mean=0.4, std=1.7)
    _, grad = update_oracle.value_loss(v, v0, ret, **kw)
    for i in range(40):
        d = np.zeros(40)
        d[i] = 1e-6
        diff = (update_oracle.value_loss(v + d, v0, ret, **kw)[0] - update_oracle.value_loss(v - d, v0, ret, **kw)[0]) / 2e-6
        assert abs(diff - grad[i]) < 1e-8, i


# ------------------------------------------------------------------------------------------------------------- refusals (CPU)
def test_refusals_on_the_host():
    from diverse_conventions_amd import clip_grad_norm, policy_loss, value_loss
    z, n = torch.zeros((4, 6)), torch.zeros(4)
    with pytest.raises(ValueError):
        policy_loss(z, torch.zeros(4, dtype=torch.int64), n, n)          # not on a GPU
    with pytest.raises(ValueError):
        value_loss(n, n, n)
    with pytest.raises(ValueError):
        clip_grad_norm([n], 1.0)
    with pytest.raises(ValueError):
        clip_grad_norm([n], 1.0, norm_type=3)
    with pytest.raises(ValueError):
        clip_grad_norm([n], -1.0)
    assert float(clip_grad_norm([], 1.0)) == 0.0


def test_c_entries_refuse_with_a_code_and_a_text():
    import ctypes
    from diverse_conventions_amd import native
    L = native.lib()
    a = native.OcPolicyLossArgs()
    assert L.oc_policy_loss(None, 0, None, None) == -1
    assert L.oc_policy_loss(ctypes.byref(a), 7, None, None) == -1
    assert L.oc_policy_loss(ctypes.byref(a), 0, None, None) == -1 and "n_actions 0" in L.oc_last_error().decode()
    a.n_actions, a.row_stride, a.rows = 6, 5, 4
    assert L.oc_policy_loss(ctypes.byref(a), 0, None, None) == -1 and "row_stride 5" in L.oc_last_error().decode()
    a.row_stride = 6
    assert L.oc_policy_loss(ctypes.byref(a), 0, None, None) == -1 and "NULL" in L.oc_last_error().decode()
    a.logits_type = 3
    assert L.oc_policy_loss(ctypes.byref(a), 0, None, None) == -1 and "logits_type 3" in L.oc_last_error().decode()
    v = native.OcValueLossArgs()
    assert L.oc_value_loss(None, 0, None, None) == -1
    v.n = -1
    assert L.oc_value_loss(ctypes.byref(v), 0, None, None) == -1 and "n -1" in L.oc_last_error().decode()
    v.n = 1
    assert L.oc_value_loss(ctypes.byref(v), 1, None, None) == -1 and "NULL" in L.oc_last_error().decode()
    assert L.oc_grad_norm_clip(-1, None, None, None, None, 1.0, 0, None, None, None) == -1
    assert L.oc_grad_norm_workspace_bytes(-1) == -1 and L.oc_grad_norm_workspace_bytes(10) > 80


# ------------------------------------------------------------------------------------------------------------- policy loss (GPU)
def check_policy(s, result, scale=1.0, clip=0.2, entropy_coef=0.01, kl_coef=0.05):
    loss, means, grad, size = oracle_policy(s, clip=clip, entropy_coef=entropy_coef, kl_coef=kl_coef)
    span = ROW * (size.sum() + abs(loss)) + 1e-9
    assert abs(float(result[0]) - loss) <= span, (float(result[0]), loss)
    assert np.all(np.abs(f64(result[1]) - means) <= ROW * (np.abs(means) + size.sum() + 1)), (f64(result[1]), means)
    if len(result) > 2 and result[2] is not None:
        got, want = f64(result[2]), grad * scale
        assert result[2].dtype == s["logits"].dtype and result[2].is_contiguous()
        bound = ROW * scale * size[:, None] + half_step(want, s["logits"].dtype)
        assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) - bound))


POLICY_SIZES = [(1, 1), (3, 1), (1, 2), (255, 3), (256, 4), (257, 5), (400, 6), (1000, 6), (513, 7), (300, 8), (300, 9), (70, 16), (33, 17), (17, 63),
                (16, 64), (15, 65), (5, 127), (9, 129), (40, 255), (7, 257), (6, 513), (5, 1000), (4, 1025), (3, 2049), (3, 4100), (2, 8193), (2, 16385),
                (2, 32771), (1, 50021), (2, 70001), (1, 131072)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,n", POLICY_SIZES)
def test_policy_loss_and_gradient(rows, n, dtype):
    from diverse_conventions_amd import policy_loss, policy_loss_grad
    for k, (available, weights, ref) in enumerate([("none", False, False), ("rows", True, True), ("one", True, False)]):
        s = policy_inputs(rows * 7 + n + k, rows, n, DTYPES[dtype], available, weights, ref, "cuda")
        kw = dict(kl_coef=0.05, ref_log_probs=s["ref"], active_masks=s["weights"], available_actions=s["avail"])
        scale = 64.0 if dtype == "f16" else 1.0
        fused = policy_loss_grad(s["logits"], s["actions"], s["old"], s["adv"], grad_scale=scale, **kw)
        check_policy(s, fused, scale)
        leaf = s["logits"].clone().requires_grad_()
        loss, stats = policy_loss(leaf, s["actions"].float().unsqueeze(1), s["old"], s["adv"], **kw)
        (grad,) = torch.autograd.grad(loss, leaf, torch.tensor(scale, device="cuda"))
        check_policy(s, (loss, stats, grad), scale)
        with torch.no_grad():
            plain = policy_loss(leaf, s["actions"].int(), s["old"], s["adv"], **kw)
        assert torch.equal(plain[0], loss) and torch.equal(plain[1], stats)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [6, 13, 40, 300, 5000, 40000])
def test_policy_loss_masks_that_leave_little(n, dtype):
    """Rows without any available action, with the taken one unavailable, of weight 0 with NaN inside, padded actions; NaN, infinities
    and the type's lowest value in masked places; -inf as a mask of its own, a whole row of it; f32 / bool / uint8 masks."""
    from diverse_conventions_amd import policy_loss_grad
    rows, dt = 24, DTYPES[dtype]
    s = policy_inputs(n, rows, n, dt, "rows", True, True, "cuda")
    z, av, a, w = s["logits"], s["avail"], s["actions"], s["weights"]
    w[:] = 1.0
    fill = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dt).min], device="cuda").to(dt)
    z.copy_(torch.where(av != 0, z, fill[torch.arange(rows * n, device="cuda").view(rows, n) % 4]))
    av[0] = 0                                              # nothing is available
    av[1, a[1]] = 0                                        # the taken action is not
    w[2] = 0
    z[2] = math.nan
    s["old"][2] = s["adv"][2] = s["ref"][2] = math.nan     # not read
    a[3], a[4] = -1, n                                     # padding
    z[5] = -math.inf                                       # nothing is possible
    z[6] = torch.finfo(dt).min                             # a uniform row at the bottom of the range
    av[6] = 1
    s["old"][6], s["ref"][6] = -math.log(n) - 0.1, -math.log(n)
    z[7, a[7]] = -math.inf
    z[8] = -math.inf
    z[8, a[8]] = 0.5                                       # one possible action
    s["old"][8], s["ref"][8] = 0.01, -0.02
    if n > 6:                                              # -inf beside ordinary logits
        z[9, (a[9] + 1) % n] = -math.inf
    kw = dict(kl_coef=0.05, ref_log_probs=s["ref"], active_masks=w)
    results = [policy_loss_grad(z, a, s["old"], s["adv"], available_actions=m, **kw) for m in (av, av != 0, (av != 0).to(torch.uint8) * 255)]
    for r in results:
        assert torch.isfinite(r[0]) and torch.isfinite(r[1]).all() and torch.isfinite(r[2]).all()
        check_policy(s, r)
        assert not r[2][[0, 1, 2, 3, 4, 5, 7]].any()
    # everything masked, or no weight at all
    for m, wt in ((torch.zeros_like(av), w), (av, torch.zeros_like(w))):
        r = policy_loss_grad(z, a, s["old"], s["adv"], available_actions=m, kl_coef=0.05, ref_log_probs=s["ref"], active_masks=wt)
        assert float(r[0]) == 0 and not r[1].any() and not r[2].any()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [6, 40, 5000, 40000])
def test_policy_loss_shows_what_is_not_a_number(n):
    from diverse_conventions_amd import policy_loss_grad
    for value in (math.nan, math.inf):
        s = policy_inputs(1, 5, n, available="none", device="cuda", weights=False)
        s["logits"][2, (int(s["actions"][2]) + 1) % n] = value
        loss, _, grad = policy_loss_grad(s["logits"], s["actions"], s["old"], s["adv"])
        assert torch.isnan(loss) and torch.isnan(grad[2]).any() and torch.isfinite(grad[[0, 1, 3, 4]]).all()
    s["logits"][2] = math.nan
    loss, _, grad = policy_loss_grad(s["logits"], s["actions"], s["old"], s["adv"])
    assert torch.isnan(loss) and torch.isnan(grad[2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n,pad,off", [(6, 2, 1), (6, 1, 0), (50, 3, 3), (700, 5, 1), (9001, 7, 5)])
def test_policy_loss_rows_of_a_padded_buffer(n, pad, off, dtype):
    from diverse_conventions_amd import policy_loss, policy_loss_grad
    s = policy_inputs(5, 37, n, DTYPES[dtype], "rows", True, True, "cuda")
    buf = torch.full((37, n + pad + off), math.nan, device="cuda", dtype=DTYPES[dtype])
    buf[:, off:off + n] = s["logits"]
    masks = torch.full((37, n + pad + off), math.nan, device="cuda")
    masks[:, off:off + n] = s["avail"]
    kw = dict(kl_coef=0.05, ref_log_probs=s["ref"], active_masks=s["weights"], available_actions=masks[:, off:off + n])
    check_policy(s, policy_loss_grad(buf[:, off:off + n], s["actions"], s["old"], s["adv"], **kw))
    leaf = buf[:, off:off + n].detach().requires_grad_()
    loss, stats = policy_loss(leaf, s["actions"], s["old"], s["adv"], **kw)
    loss.backward()
    check_policy(s, (loss, stats, leaf.grad.contiguous()))


@pytest.mark.gpu
def test_policy_loss_many_rows_and_leading_dimensions():
    """Over the row counts where the weight is added up by a launch of its own, [T, N, A, actions] as buffers hold it."""
    from diverse_conventions_amd import policy_loss_grad
    s = policy_inputs(11, 30 * 200 * 2, 6, device="cuda")
    shaped = lambda t, *last: t.view(30, 200, 2, *last)
    r = policy_loss_grad(shaped(s["logits"], 6), shaped(s["actions"], 1), shaped(s["old"], 1), shaped(s["adv"], 1), kl_coef=0.05,
                         ref_log_probs=shaped(s["ref"], 1), active_masks=shaped(s["weights"], 1), available_actions=shaped(s["avail"], 6))
    assert r[2].shape == (30, 200, 2, 6)
    check_policy(s, (r[0], r[1], r[2].view(-1, 6)))
    again = policy_loss_grad(s["logits"], s["actions"], s["old"], s["adv"], kl_coef=0.05, ref_log_probs=s["ref"], active_masks=s["weights"], available_actions=s["avail"])
    assert torch.equal(r[0], again[0]) and torch.equal(r[1], again[1]) and torch.equal(r[2].view(-1, 6), again[2])
    empty = policy_loss_grad(s["logits"][:0], s["actions"][:0], s["old"][:0], s["adv"][:0])
    assert float(empty[0]) == 0 and empty[2].shape == (0, 6)


@pytest.mark.gpu
def test_policy_loss_gradient_follows_differences():
    """The f32 kernel's own loss, along the gradient's direction: a step of 1e-2 along a unit direction changes the loss by the slope
    times the step up to the curvature's third order (central difference), and the loss carries ROW of its terms."""
    from diverse_conventions_amd import policy_loss, policy_loss_grad
    s = policy_inputs(2, 64, 6, available="none", weights=False, device="cuda")
    kw = dict(clip_param=1e6, entropy_coef=0.05, kl_coef=0.3, ref_log_probs=s["ref"])
    loss, _, grad = policy_loss_grad(s["logits"], s["actions"], s["old"], s["adv"], **kw)
    d = grad / grad.norm()
    h = 1e-2
    up = policy_loss(s["logits"] + h * d, s["actions"], s["old"], s["adv"], **kw)[0]
    down = policy_loss(s["logits"] - h * d, s["actions"], s["old"], s["adv"], **kw)[0]
    slope = float((up.double() - down.double()) / (2 * h))
    size = oracle_policy(s, clip=1e6, entropy_coef=0.05, kl_coef=0.3)[3].sum()
    assert abs(slope - float(grad.norm())) <= ROW * size / h + h * h * 10 * size


@pytest.mark.gpu
def test_policy_loss_refusals():
    from diverse_conventions_amd import policy_loss, policy_loss_grad
    s = policy_inputs(0, 8, 6, device="cuda")
    good = dict(logits=s["logits"], actions=s["actions"], old_log_probs=s["old"], advantages=s["adv"])
    for bad in (dict(logits=s["logits"].double()), dict(logits=s["logits"].t().contiguous().t()), dict(logits=s["logits"][:1].expand(8, 6)),
                dict(logits=s["logits"].cpu()), dict(actions=s["actions"][:4]), dict(actions=s["actions"].to(torch.int8)), dict(actions=s["actions"].cpu()),
                dict(old_log_probs=s["old"].double()), dict(advantages=s["adv"][:5]), dict(active_masks=torch.ones(7, device="cuda")),
                dict(available_actions=torch.ones((8, 5), device="cuda")), dict(available_actions=torch.ones((8, 6), device="cuda").double()),
                dict(ref_log_probs=s["old"].half()), dict(clip_param=-0.1), dict(clip_param=math.nan), dict(old_log_probs=torch.zeros((8, 2), device="cuda")[:, 0])):
        for fn in (policy_loss, policy_loss_grad):
            with pytest.raises(ValueError):
                fn(**{**good, **bad})


# -------------------------------------------------------------------------------------------------------------- value loss (GPU)
def value_inputs(seed, n, dtype, weights, norm, clip=0.2):
    g = torch.Generator().manual_seed(seed)
    v0 = torch.randn(n, generator=g)
    v = (v0 + 0.3 * torch.randn(n, generator=g)).to(dtype)
    mean, std = norm or (0.0, 1.0)
    y = v0 + 2 * torch.randn(n, generator=g) + 20 * (torch.rand(n, generator=g) < 0.05)
    ret = y * std + mean
    d, t = v.double() - v0.double(), (ret.double() - mean) / std
    e0, e1 = t - v.double(), t - (v0.double() + d.clamp(-clip, clip))
    near = ((d.abs() - clip).abs() < 1e-4) | ((d.abs() > clip) & ((e0.abs() - e1.abs()).abs() < 1e-4))      # the gradient jumps there
    v0 = torch.where(near, v.float(), v0)
    w = (torch.rand(n, generator=g) < 0.8).float() * torch.rand(n, generator=g) if weights else None
    return [t.cuda() if t is not None else None for t in (v, v0, ret, w)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 255, 400, 1023, 1024, 1025, 4099, 8192, 8193, 100003])
def test_value_loss_and_gradient(n, dtype):
    """A sample's value carries at most 2^-24 * 6 of (|y| + |v| + |v0|)^2-sized terms: e = y - v has rounding 2^-24 (|y| + |e|) twice, squared."""
    from diverse_conventions_amd import value_loss, value_loss_grad
    for weights, norm, delta, clip in ((False, None, 10.0, 0.2), (True, (0.7, 2.5), 10.0, 0.2), (True, None, None, 0.2), (True, (-3.0, 0.1), 0.5, None)):
        v, v0, ret, w = value_inputs(n, n, DTYPES[dtype], weights, norm, clip or 1e9)
        mean, std = norm or (0.0, 1.0)
        loss, grad = update_oracle.value_loss(f64(v), f64(v0), f64(ret), clip, delta, None if w is None else f64(w), mean, std)
        scale = 256.0 if dtype == "f16" else 1.0
        kw = dict(clip_param=clip, huber_delta=delta, active_masks=w, value_normalizer=norm)
        y = np.abs(f64(ret)) / std + abs(mean) / std + np.abs(f64(v)) + np.abs(f64(v0))
        wt = np.ones(n) if w is None else f64(w)
        share = wt / wt.sum() if wt.sum() else wt
        span_loss = 2.0 ** -24 * 12 * (share * y * y).sum() + 2.0 ** -24 * abs(loss)
        bound = scale * 2.0 ** -24 * 12 * share * y + half_step(grad * scale, DTYPES[dtype])
        fused = value_loss_grad(v, v0, ret, grad_scale=scale, **kw)
        leaf = v.clone().requires_grad_()
        one = value_loss(leaf, v0, ret, **kw)
        (g,) = torch.autograd.grad(one, leaf, torch.tensor(scale, device="cuda"))
        for got_loss, got in (fused, (one, g)):
            assert abs(float(got_loss) - loss) <= span_loss, (float(got_loss), loss)
            assert got.dtype == v.dtype and np.all(np.abs(f64(got) - grad * scale) <= bound)
        assert torch.equal(value_loss(v, v0, ret, **kw), one.detach())


@pytest.mark.gpu
def test_value_loss_special_samples_and_refusals():
    from diverse_conventions_amd import value_loss, value_loss_grad
    v, v0, ret, w = value_inputs(0, 40, torch.float32, True, None)
    w[3] = w[11] = 0
    v[3], v0[3], ret[11] = math.nan, math.inf, math.nan     # of weight 0: not looked at
    loss, grad = value_loss_grad(v, v0, ret, active_masks=w)
    assert torch.isfinite(loss) and torch.isfinite(grad).all() and float(grad[3]) == 0 and float(grad[11]) == 0
    want, _ = update_oracle.value_loss(*(np.nan_to_num(f64(t), posinf=0) for t in (v, v0, ret)), weights=f64(w))
    assert abs(float(loss) - want) < 1e-5 * abs(want)
    zero = value_loss_grad(v, v0, ret, active_masks=torch.zeros_like(w))
    assert float(zero[0]) == 0 and not zero[1].any()
    assert float(value_loss(v[:0], v0[:0], ret[:0])) == 0
    ret[5] = math.nan
    w[5] = 1
    loss, grad = value_loss_grad(v, v0, ret, active_masks=w)
    assert torch.isnan(loss) and torch.isnan(grad[5]) and torch.isfinite(grad[4])
    for bad in (dict(values=v.double()), dict(values=v.cpu()), dict(values=torch.zeros((40, 2), device="cuda")[:, 0]), dict(value_preds=v0[:5]),
                dict(returns=ret.half()), dict(active_masks=w[:7]), dict(clip_param=-1.0), dict(huber_delta=-1.0), dict(value_normalizer=(0.0, 0.0))):
        with pytest.raises(ValueError):
            value_loss(**{**dict(values=v, value_preds=v0, returns=ret), **bad})


# ---------------------------------------------------------------------------------------------------------- gradient norm (GPU)
def make_grads(sizes, seed, dtypes=(torch.float32,), scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(dtypes[i % len(dtypes)]).cuda() for i, n in enumerate(sizes)]


def check_clip(norm, got, grads, max_norm, inf_norm=False):
    """The norm is the f64 sum rounded once (2^-24), the factor has three more roundings, the product one: 5 * 2^-24, then the type's."""
    want_norm, want = update_oracle.clip_grads([f64(g) for g in grads], max_norm, inf_norm)
    assert abs(float(norm) - want_norm) <= 2.0 ** -23 * want_norm
    for o, x, t in zip(got, want, grads):
        assert o.dtype == t.dtype and np.all(np.abs(f64(o).reshape(x.shape) - x) <= 5 * 2.0 ** -24 * np.abs(x) + half_step(x, t.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1], [0, 3], [7, 1, 0, 4096, 4097, 5], [5760, 32, 12288, 64, 4096, 64, 384, 6], [100003, 1, 70001], list(range(1, 300)), [9000000, 3]],
                         ids=lambda s: f"{len(s)}x{sum(s)}")
@pytest.mark.parametrize("dtypes", [("f32",), ("bf16",), ("f16",), ("f32", "bf16", "f16")], ids="-".join)
def test_clip_grad_norm(sizes, dtypes):
    from diverse_conventions_amd import clip_grad_norm
    grads = make_grads(sizes, sum(sizes), [DTYPES[d] for d in dtypes])
    raw = [g.clone() for g in grads]
    for max_norm in (0.5, 1e9):
        for norm_type in (2.0, math.inf):
            inf_norm = norm_type == math.inf
            alone = clip_grad_norm(grads, norm_type=norm_type)
            out = [torch.full_like(g, math.nan) for g in grads]
            norm = clip_grad_norm(grads, max_norm, norm_type, out=out)
            assert torch.equal(alone, norm) and all(torch.equal(g, r) for g, r in zip(grads, raw))
            check_clip(norm, out, raw, max_norm, inf_norm)
            again = clip_grad_norm(grads, max_norm, norm_type)
            assert torch.equal(norm, again) and all(torch.equal(g, o) for g, o in zip(grads, out))
            for g, r in zip(grads, raw):
                g.copy_(r)


@pytest.mark.gpu
def test_clip_grad_norm_parameters_layouts_and_odd_places():
    from diverse_conventions_amd import clip_grad_norm
    net = torch.nn.Sequential(torch.nn.Conv2d(20, 32, 3), torch.nn.Linear(64, 6)).cuda()
    net[0].weight.grad = torch.randn((32, 20, 3, 3), device="cuda").to(memory_format=torch.channels_last)
    net[1].weight.grad = torch.randn((64, 6), device="cuda").t()
    net[1].bias.grad = torch.randn(6, device="cuda")                     # net[0].bias has none
    mine = [p.grad.clone(memory_format=torch.preserve_format) for p in net.parameters() if p.grad is not None]
    norm = clip_grad_norm(net.parameters(), 1.0)
    check_clip(norm, [p.grad for p in net.parameters() if p.grad is not None], mine, 1.0)
    # pieces of one buffer at odd places, the elements between them untouched
    for dt in (torch.float32, torch.bfloat16):
        buf = torch.randn(10000, device="cuda").to(dt)
        raw = buf.clone()
        views = [buf[1:4098], buf[4100:4103], buf[5001:9999]]
        check_clip(clip_grad_norm(views, 0.1), views, [raw[1:4098], raw[4100:4103], raw[5001:9999]], 0.1)
        keep = torch.ones(10000, dtype=torch.bool, device="cuda")
        for a, b in ((1, 4098), (4100, 4103), (5001, 9999)):
            keep[a:b] = False
        assert torch.equal(buf[keep], raw[keep])


@pytest.mark.gpu
def test_clip_grad_norm_at_the_ends_of_the_range():
    from diverse_conventions_amd import clip_grad_norm
    tiny, huge = torch.full((1000,), 1e-30, device="cuda"), torch.full((1000,), 1e30, device="cuda")
    assert abs(float(clip_grad_norm([tiny])) / (math.sqrt(1000) * float(tiny[0].double())) - 1) < 1e-6
    assert abs(float(clip_grad_norm([huge])) / (math.sqrt(1000) * float(huge[0].double())) - 1) < 1e-6
    zero = torch.zeros(100, device="cuda")
    assert float(clip_grad_norm([zero], 1.0)) == 0 and not zero.any()
    for value in (math.nan, math.inf):
        g = torch.ones(5000, device="cuda")
        g[4321] = value
        for norm_type in (2.0, math.inf):
            h = g.clone()
            norm = clip_grad_norm([h], 1.0, norm_type)
            want = torch.clamp(1.0 / (norm + 1e-6), max=1.0) * g
            assert not torch.isfinite(norm) and torch.equal(torch.isnan(h), torch.isnan(want)) and torch.equal(torch.nan_to_num(h), torch.nan_to_num(want))
    g = torch.ones(10, device="cuda")
    for bad in (dict(grads=[g.double()]), dict(grads=[g, g.cpu()]), dict(grads=[g[::2]]), dict(grads=[g[:1].expand(4)]), dict(grads=[g, g]),
                dict(grads=[g], out=[g[:5]]), dict(grads=[g], out=[g.half()]), dict(grads=[g], out=[]), dict(grads=[g], norm_type=1)):
        with pytest.raises(ValueError):
            clip_grad_norm(**{**dict(max_norm=1.0), **bad})


# ------------------------------------------------------------------------------------------------- streams, graphs, the run of them
@pytest.mark.gpu
def test_update_operators_on_another_stream_and_two_at_once():
    from diverse_conventions_amd import clip_grad_norm, policy_loss_grad, value_loss_grad
    s = policy_inputs(4, 20000, 6, device="cuda")
    v, v0, ret, w = value_inputs(4, 20000, torch.float32, True, None)
    grads = make_grads([300000, 77, 4096], 1)

    def all_three():
        p = policy_loss_grad(s["logits"], s["actions"], s["old"], s["adv"], active_masks=s["weights"], available_actions=s["avail"])
        q = value_loss_grad(v, v0, ret, active_masks=w)
        out = [torch.empty_like(g) for g in grads]
        return [*p, *q, clip_grad_norm(grads, 1.0, out=out), *out]

    want = all_three()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(all_three())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


@pytest.mark.gpu
def test_update_operators_in_a_captured_graph():
    from diverse_conventions_amd import clip_grad_norm, policy_loss_grad, value_loss_grad
    s = policy_inputs(6, 9001, 6, device="cuda")
    big = policy_inputs(7, 5, 5000, torch.bfloat16, device="cuda", available="none")
    v, v0, ret, w = value_inputs(6, 9001, torch.float32, True, (1.0, 2.0))
    grads = make_grads([30000, 77, 4096], 2)
    out = [torch.empty_like(g) for g in grads]

    def step():
        p = policy_loss_grad(s["logits"], s["actions"], s["old"], s["adv"], active_masks=s["weights"], available_actions=s["avail"])
        b = policy_loss_grad(big["logits"], big["actions"], big["old"], big["adv"], active_masks=big["weights"])
        q = value_loss_grad(v, v0, ret, active_masks=w, value_normalizer=(1.0, 2.0))
        return [*p, *b, *q, clip_grad_norm(grads, 1.0, out=out)]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        s["logits"].normal_()
        big["logits"].normal_()
        v.normal_()
        grads[0].normal_()
        graph.replay()
        torch.cuda.synchronize()
        seen = [t.clone() for t in held] + [o.clone() for o in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(seen, want + out)), k


@pytest.mark.gpu
def test_one_update_of_an_actor_and_a_critic():
    """The operators as an update uses them, against torch's own operations: losses, gradients of the networks' weights, clipping."""
    from diverse_conventions_amd import clip_grad_norm, policy_loss, value_loss
    torch.manual_seed(0)
    actor, critic = torch.nn.Linear(32, 6).cuda(), torch.nn.Linear(32, 1).cuda()
    x = torch.randn((500, 32), device="cuda")
    s = policy_inputs(9, 500, 6, available="rows", device="cuda", ref=False)
    with torch.no_grad():
        masked = torch.where(s["avail"] != 0, actor(x), torch.full((), -1e10, device="cuda"))
        s["old"] = torch.log_softmax(masked, -1).gather(1, s["actions"][:, None]).squeeze(1) + 0.01 * torch.randn(500, device="cuda")
    v0, ret = torch.randn((500, 1), device="cuda"), torch.randn((500, 1), device="cuda")

    def own():
        loss, _ = policy_loss(actor(x), s["actions"], s["old"], s["adv"], active_masks=s["weights"], available_actions=s["avail"])
        return loss, value_loss(critic(x), v0, ret, active_masks=s["weights"].unsqueeze(1))

    def plain():
        logp = torch.log_softmax(torch.where(s["avail"] != 0, actor(x), torch.full((), -1e10, device="cuda")), -1)
        ratio = torch.exp(logp.gather(1, s["actions"][:, None]).squeeze(1) - s["old"])
        surr = torch.min(ratio * s["adv"], torch.clamp(ratio, 0.8, 1.2) * s["adv"])
        w = s["weights"]
        p_loss = -(surr * w).sum() / w.sum() - 0.01 * (-(logp.exp() * logp).sum(-1) * w).sum() / w.sum()
        v = critic(x)
        huber = lambda e: torch.where(e.abs() <= 10, e * e / 2, 10 * (e.abs() - 5))
        worst = torch.max(huber(ret - v), huber(ret - (v0 + (v - v0).clamp(-0.2, 0.2))))
        return p_loss, (worst * w.unsqueeze(1)).sum() / w.sum()

    results = []
    for losses in (own, plain):
        for net in (actor, critic):
            net.zero_grad(set_to_none=True)
        p, v = losses()
        total = p + v
        total.backward()
        if losses is own:
            norms = [clip_grad_norm(net.parameters(), 0.05) for net in (actor, critic)]
        else:
            norms = [torch.nn.utils.clip_grad_norm_(net.parameters(), 0.05) for net in (actor, critic)]
        results.append([p.detach(), v.detach(), *norms, *(q.grad.clone() for net in (actor, critic) for q in net.parameters())])
    for a, b in zip(*results):
        # f32 on both sides: 1e-4 of the largest element (sums of 500 terms of which each side rounds every one)
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4 * float(b.abs().max())), (a, b)


@pytest.mark.gpu
def test_losses_under_hooks_on_saved_tensors_and_in_place_changes():
    """Tensors that a hook keeps on the host come back as others, elsewhere; one changed in place is noticed."""
    from diverse_conventions_amd import policy_loss, value_loss
    s = policy_inputs(8, 300, 6, device="cuda")
    v, v0, ret, w = value_inputs(8, 300, torch.float32, True, None)
    kw = dict(kl_coef=0.05, ref_log_probs=s["ref"], active_masks=s["weights"], available_actions=s["avail"])

    def both(hooked):
        z, y = torch.zeros((300, 9), device="cuda"), v.clone().requires_grad_()
        z[:, 1:7] = s["logits"]
        leaf = z.requires_grad_()
        with torch.autograd.graph.save_on_cpu() if hooked else torch.enable_grad():
            one, _ = policy_loss((leaf * 1.0)[:, 1:7], s["actions"], s["old"], s["adv"], **kw)
            two = value_loss(y * 1.0, v0, ret, active_masks=w)
        junk = [torch.full((300, 9), math.nan, device="cuda") for _ in range(20)]       # what was freed is overwritten
        grads = torch.autograd.grad(one + two, (leaf, y))
        del junk
        return grads

    for a, b in zip(both(True), both(False)):
        assert torch.equal(a, b)
    mid = s["logits"].clone().requires_grad_() * 1.0
    loss, _ = policy_loss(mid, s["actions"], s["old"], s["adv"])
    mid.mul_(2.0)
    with pytest.raises(RuntimeError):
        loss.backward()
    loss, stats = policy_loss(s["logits"].clone().requires_grad_(), s["actions"], s["old"], s["adv"])
    loss += 1.0                                            # the results are the caller's
    stats.mul_(0.0)
    loss.backward()


@pytest.mark.gpu
def test_policy_loss_beyond_32_bit_offsets():
    """Rows whose first element lies behind 2^31 elements, and 2^32 bytes of gradient: the last rows against the same rows alone."""
    from diverse_conventions_amd import policy_loss_grad
    n, rows = 70001, 30700                                 # 2.149e9 elements, 4.3 GB each of logits and gradient in bfloat16
    assert n * rows > 2 ** 31
    logits = torch.zeros((rows, n), dtype=torch.bfloat16, device="cuda")
    s = policy_inputs(3, 4, n, torch.bfloat16, "none", False, False, "cuda")
    logits[-4:] = s["logits"]
    actions = torch.full((rows,), -1, device="cuda")       # padding, but for the last rows
    actions[-4:] = s["actions"]
    old, adv = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    old[-4:], adv[-4:] = s["old"], s["adv"]
    loss, _, grad = policy_loss_grad(logits, actions, old, adv)
    want, _, alone = policy_loss_grad(s["logits"], s["actions"], s["old"], s["adv"])
    assert torch.equal(grad[-4:], alone) and not grad[:-4:997].any() and not grad[-5].any()
    assert abs(float(loss) - float(want)) <= 1e-6 * abs(float(want))      # f64 sums in another order, rounded once
    del logits, grad
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_losses_of_unusual_but_allowed_calls():
    """One row without a leading dimension, no rows, coefficients of zero, a clip of zero, a broadcast byte mask over many actions, a KL
    statistic without its term, backward twice."""
    from diverse_conventions_amd import policy_loss, policy_loss_grad, value_loss
    s = policy_inputs(21, 1, 6, available="none", weights=False, device="cuda")
    leaf = s["logits"][0].clone().requires_grad_()
    loss, stats = policy_loss(leaf, s["actions"].squeeze(), s["old"].squeeze(), s["adv"].squeeze(), kl_coef=0.05, ref_log_probs=s["ref"])
    first, second = (torch.autograd.grad(loss, leaf, retain_graph=True)[0] for _ in range(2))
    assert first.shape == (6,) and torch.equal(first, second)
    check_policy(s, (loss.detach(), stats, first.unsqueeze(0)))
    for n in (6, 40):
        none = torch.zeros((0, n), device="cuda", requires_grad=True)
        e = torch.zeros(0, device="cuda")
        loss, _ = policy_loss(none, e, e, e)
        assert float(loss.detach()) == 0 and torch.autograd.grad(loss, none)[0].shape == (0, n)
    for n in (6, 40, 3000):
        s = policy_inputs(22, 50, n, available="none", device="cuda")
        mask = torch.ones((1, n), dtype=torch.uint8, device="cuda")
        mask[0, 1] = 0
        s["actions"] = torch.where(s["actions"] == 1, 0, s["actions"])
        s["avail"] = mask.expand(50, n)
        for clip, ce, ck in ((0.0, 0.0, 0.0), (0.2, 0.3, 0.0), (0.2, 0.0, 0.7)):
            # exp(lp - old) is not within 1e-3 of the clip's borders: old is drawn anew around the masked distribution
            z = torch.where(s["avail"] != 0, s["logits"].double(), -math.inf)
            lp = torch.log_softmax(z, 1).gather(1, s["actions"][:, None]).squeeze(1)
            s["old"] = (lp - torch.where(torch.arange(50, device="cuda") % 2 == 0, 0.1, -0.3)).float()
            r = policy_loss_grad(s["logits"], s["actions"], s["old"], s["adv"], clip_param=clip, entropy_coef=ce, kl_coef=ck, ref_log_probs=s["ref"],
                                 active_masks=s["weights"], available_actions=s["avail"])
            check_policy(s, r, clip=clip, entropy_coef=ce, kl_coef=ck)
    v = torch.tensor(0.5, device="cuda", requires_grad=True)
    loss = value_loss(v, torch.tensor(0.4, device="cuda"), torch.tensor(2.0, device="cuda"))
    (g,) = torch.autograd.grad(loss, v)
    assert g.shape == () and abs(float(loss.detach()) - 1.125) < 1e-6 and abs(float(g) + 1.5) < 1e-6
    empty = torch.zeros((0, 1), device="cuda", requires_grad=True)
    assert torch.autograd.grad(value_loss(empty, empty.detach(), empty.detach()), empty)[0].shape == (0, 1)


@pytest.mark.gpu
def test_clip_grad_norm_of_nothing_and_onto_itself():
    from diverse_conventions_amd import clip_grad_norm
    empty = [torch.zeros(0, device="cuda"), torch.zeros((0, 3), device="cuda")]
    assert float(clip_grad_norm(empty)) == 0 and float(clip_grad_norm(empty, 1.0)) == 0
    grads = make_grads([5000, 33], 4)
    raw = [g.clone() for g in grads]
    norm = clip_grad_norm((g for g in grads), 0.25, out=grads)          # a generator; the results onto the gradients themselves
    check_clip(norm, grads, raw, 0.25)
    untouched = [g.clone() for g in raw]
    clip_grad_norm(untouched, 0.0)
    assert not any(g.any() for g in untouched)
