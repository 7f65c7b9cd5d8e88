"""float64 restatement of the update-side operators: the clipped policy loss, the clipped value loss (the arithmetic of the reference's
train/MAPPO/r_mappo.py, ppo_update and cal_value_loss), gradient clipping (torch.nn.utils.clip_grad_norm_) and the products grouped by
network.  TEST INFRASTRUCTURE ONLY.  No fixture of the reference covers the losses (parity unpinned): the formulas are checked against
finite differences."""
import numpy as np


def policy_loss(logits, actions, old, adv, clip=0.2, entropy_coef=0.01, kl_coef=0.0, ref=None, weights=None, available=None):
    """-> loss, means [5], d loss / d logits, size of the row's terms [rows] (what a rounding error is relative to)"""
    z = np.asarray(logits, np.float64)
    rows, n = z.shape
    possible = z != -np.inf
    if available is not None:
        possible &= np.broadcast_to(np.asarray(available), z.shape) != 0
    a = np.asarray(actions, np.float64).reshape(-1)
    w = np.ones(rows) if weights is None else np.asarray(weights, np.float64).reshape(-1)
    grad, size, sums, total = np.zeros_like(z), np.zeros(rows), np.zeros(5), 0.0
    old, adv = (np.asarray(t, np.float64).reshape(-1) for t in (old, adv))
    ref = None if ref is None else np.asarray(ref, np.float64).reshape(-1)
    valid = [r for r in range(rows) if 0 <= a[r] < n]
    total = sum(w[r] for r in valid)
    for r in valid:
        j = int(a[r])
        if w[r] == 0 or not possible[r, j]:
            continue
        at = np.flatnonzero(possible[r])
        zr = z[r, at]
        top = zr.max()
        lp = zr - top - np.log(np.exp(zr - top).sum())
        p = np.exp(lp)
        mine = lp[np.flatnonzero(at == j)[0]]
        entropy = -(p * lp).sum()
        ratio = np.exp(mine - old[r])
        clipped = min(max(ratio, 1 - clip), 1 + clip)
        sums[:2] += w[r] * np.array([-min(ratio * adv[r], clipped * adv[r]), entropy])
        c1 = 0.0 if (adv[r] > 0 and ratio > 1 + clip) or (adv[r] < 0 and ratio < 1 - clip) else -adv[r] * ratio
        if ref is not None:
            d = ref[r] - mine
            sums[2] += w[r] * (np.expm1(d) - d)
            c1 -= kl_coef * np.expm1(d)
            size[r] += abs(kl_coef) * (np.exp(d) + 1 + abs(d))
        sums[3] += w[r] * (not 1 - clip <= ratio <= 1 + clip)
        sums[4] += w[r] * ratio
        g = c1 * ((at == j) - p) + entropy_coef * p * (lp + entropy)
        grad[r, at] = g * w[r] / total
        size[r] = (size[r] + abs(ratio * adv[r]) + abs(entropy_coef) * (1 + entropy)) * abs(w[r] / total)
    if total == 0:
        return 0.0, np.zeros(5), np.zeros_like(z), size
    means = sums / total
    return means[0] - entropy_coef * means[1] + (kl_coef * means[2] if ref is not None else 0.0), means, grad, size


def value_loss(values, preds, returns, clip=0.2, delta=10.0, weights=None, mean=0.0, std=1.0):
    """-> loss, d loss / d values"""
    v, v0, ret = (np.asarray(t, np.float64).reshape(-1) for t in (values, preds, returns))
    w = np.ones_like(v) if weights is None else np.asarray(weights, np.float64).reshape(-1)
    on = w != 0
    v, v0, ret = (np.where(on, t, 0.0) for t in (v, v0, ret))
    y = (ret - mean) / std

    def h(e):
        return e * e / 2 if delta is None else np.where(np.abs(e) <= delta, e * e / 2, delta * (np.abs(e) - delta / 2))

    e0 = y - v
    slope = e0 if delta is None else np.clip(e0, -delta, delta)
    worst, free = h(e0), np.ones_like(on)
    if clip is not None:
        h1 = h(y - (v0 + np.clip(v - v0, -clip, clip)))
        free = (np.abs(v - v0) <= clip) | (h(e0) >= h1)
        worst = np.where(free, h(e0), h1)
    total = w.sum()
    if total == 0:
        return 0.0, np.zeros_like(v)
    return (w * worst).sum() / total, np.where(on & free, -w * slope / total, 0.0)


def clip_grads(grads, max_norm=None, inf_norm=False):
    """-> norm, clipped gradients"""
    flat = [np.asarray(g, np.float64) for g in grads]
    norm = max((np.abs(g).max() for g in flat if g.size), default=0.0) if inf_norm else np.sqrt(sum((g * g).sum() for g in flat))
    f = 1.0 if max_norm is None else min(1.0, max_norm / (norm + 1e-6))
    return norm, [g * f for g in flat]


def grouped_linear(x, weight, offsets, bias=None, dy=None):
    """-> y, and with dy: dx, dweight, dbias"""
    x, weight = np.asarray(x, np.float64), np.asarray(weight, np.float64)
    y = np.zeros((x.shape[0], weight.shape[1]))
    dx, dw, db = np.zeros_like(x), np.zeros_like(weight), np.zeros(weight.shape[:2])
    for g in range(weight.shape[0]):
        a, b = int(offsets[g]), int(offsets[g + 1])
        y[a:b] = x[a:b] @ weight[g].T + (0 if bias is None else np.asarray(bias, np.float64)[g])
        if dy is not None:
            d = np.asarray(dy, np.float64)[a:b]
            dx[a:b], dw[g], db[g] = d @ weight[g], d.T @ x[a:b], d.sum(0)
    return (y,) if dy is None else (y, dx, dw, db)
