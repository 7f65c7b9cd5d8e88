"""grouped_linear: products of rows sorted by network with each network's weights, forward and backward, against oracle/update_oracle.py.

Two kinds of inputs.  Small whole numbers: every product and every partial sum is a whole number below 2^24 and so exact in f32 in any
order, and the results must be the exact sums rounded once to the type -- equal, bit for bit.  Real numbers: a sum of R products in f32
carries at most (R + 2) 2^-24 of the sum of the products' magnitudes, then half a step of the type."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import update_oracle

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def f64(t):
    return t.detach().double().cpu().numpy()


def inputs(sizes, k, n, dtype, seed, whole, head=0, tail=0):
    g = torch.Generator().manual_seed(seed)
    rows = head + sum(sizes) + tail
    if whole:                                              # at most 4 * 2 * R < 2^24; f16 results below 65504 are checked by the caller's sizes
        draw = lambda *s, top: torch.randint(-top, top + 1, s, generator=g).float()
        x, w, b, dy = draw(rows, k, top=2), draw(len(sizes), n, k, top=2), draw(len(sizes), n, top=2), draw(rows, n, top=2)
    else:
        x, w, b, dy = (torch.randn(s, generator=g) for s in ((rows, k), (len(sizes), n, k), (len(sizes), n), (rows, n)))
    cuts = np.concatenate([[head], head + np.cumsum(sizes)])
    return [t.to(DTYPES[dtype]).cuda() for t in (x, w, b, dy)] + [cuts]


def check(got, want, bound, dtype, whole, what):
    assert got.dtype == DTYPES[dtype], what
    if whole:
        exact = torch.from_numpy(want).to(DTYPES[dtype]).double().numpy()
        assert np.array_equal(f64(got), exact), (what, np.argwhere(f64(got) != exact)[:5])
    else:
        limit = bound + np.abs(want) * torch.finfo(DTYPES[dtype]).eps / 2 + (2.0 ** -25 if dtype == "f16" else 0)
        assert np.all(np.abs(f64(got) - want) <= limit), (what, float(np.max(np.abs(f64(got) - want) - limit)))


def run_and_check(sizes, k, n, dtype, seed, whole, head=0, tail=0, offsets_type=torch.int32, bias=True):
    from diverse_conventions_amd import grouped_linear
    x, w, b, dy, cuts = inputs(sizes, k, n, dtype, seed, whole, head, tail)
    offsets = torch.tensor(cuts, dtype=offsets_type, device="cuda")
    leaves = [t.requires_grad_() for t in ((x, w, b) if bias else (x, w))]
    y = grouped_linear(x, w, offsets, b if bias else None)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(grouped_linear(x, w, offsets, b if bias else None), y)
    want = update_oracle.grouped_linear(f64(x), f64(w), cuts, f64(b) if bias else None, f64(dy))
    sums = update_oracle.grouped_linear(np.abs(f64(x)), np.abs(f64(w)), cuts, np.abs(f64(b)) if bias else None, np.abs(f64(dy)))
    longest = max(sizes)
    for name, got, exact, size, r in zip(("y", "dx", "dw", "db"), (y, *grads), want, sums, (k + 1, n, longest, longest)):
        check(got, exact, (r + 2) * 2.0 ** -24 * size, dtype, whole, name)


SHAPES = [
    ([1], 1, 1), ([5], 3, 7), ([0, 1, 0], 8, 16), ([1, 2, 0, 3], 33, 65), ([16] * 5, 64, 64), ([17, 0, 31, 40], 72, 40), ([64, 65, 63], 192, 64),
    ([100, 3, 130], 64, 6), ([200, 0, 57], 64, 1), ([128, 129], 128, 128), ([300, 1, 0, 77], 136, 264), ([1] * 70, 40, 24), ([0] * 65 + [9, 200] + [0] * 3, 16, 16),
    ([257, 255], 100, 260), ([90, 11], 130, 132), ([1000], 192, 64), ([4, 4, 4], 520, 1032), ([700, 2, 701], 255, 129),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("sizes,k,n", SHAPES, ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)}g{sum(v)}")
def test_grouped_linear_small_numbers_are_exact(sizes, k, n, dtype):
    run_and_check(sizes, k, n, dtype, 1, True)
    run_and_check(sizes, k, n, dtype, 2, True, head=3, tail=70, offsets_type=torch.int64, bias=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("sizes,k,n", SHAPES, ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)}g{sum(v)}")
def test_grouped_linear_real_numbers(sizes, k, n, dtype):
    run_and_check(sizes, k, n, dtype, 3, False, tail=2)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,k,n", [([600, 0, 1700, 255, 1541], 512, 1536), ([4096], 1024, 1024), ([511, 513] * 4, 264, 3080), ([300] * 60, 257, 513)],
                         ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)}g{sum(v)}")
def test_grouped_linear_large_tiles(sizes, k, n, dtype):
    run_and_check(sizes, k, n, dtype, 4, True, head=1, tail=5)


@pytest.mark.gpu
def test_grouped_linear_long_groups_are_summed_in_pieces():
    for dtype in DTYPES:
        run_and_check([20000, 3, 9000], 24, 16, dtype, 5, True)
        run_and_check([30000], 192, 64, dtype, 6, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_grouped_linear_strides_single_gradients_and_nonfinite_neighbours(dtype):
    """Rows out of a wider buffer with NaN beside them, NaN in other groups' rows and in rows of no group: nothing leaks into a group."""
    from diverse_conventions_amd import grouped_linear
    sizes, k, n = [40, 0, 25], 24, 40
    x, w, b, dy, cuts = inputs(sizes, k, n, dtype, 7, True, head=2, tail=3)
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    want = update_oracle.grouped_linear(f64(x), f64(w), cuts, f64(b), f64(dy))
    for pad, off in ((8, 0), (5, 3)):
        buf = torch.full((x.shape[0], k + pad), float("nan"), dtype=x.dtype, device="cuda")
        buf[:, off:off + k] = x
        buf[:2], buf[-3:] = float("nan"), float("inf")
        d = dy.clone()
        d[:2], d[-3:] = float("inf"), float("nan")
        leaf, weight, bias = buf[:, off:off + k].detach().requires_grad_(), w.clone().requires_grad_(), b.clone().requires_grad_()
        y = grouped_linear(leaf, weight, offsets, bias)
        for got, exact, name in zip((y, *torch.autograd.grad(y, (leaf, weight, bias), d, retain_graph=True)), want, ("y", "dx", "dw", "db")):
            check(got, exact, None, dtype, True, name)
        for only, exact in zip((leaf, weight, bias), want[1:]):
            check(torch.autograd.grad(y, only, d, retain_graph=True)[0], exact, None, dtype, True, "one")
        poisoned = buf[:, off:off + k].clone()
        poisoned[2:42] = float("nan")                      # group 0
        y2 = grouped_linear(poisoned, w, offsets, b)
        assert torch.isnan(y2[2:42]).all() and torch.equal(y2[42:], y[42:])
    (g,) = torch.autograd.grad(grouped_linear(leaf, w, offsets).sum(), leaf)         # an expanded upstream gradient
    ones = update_oracle.grouped_linear(f64(x), f64(w), cuts, None, np.ones((x.shape[0], n)))[1]
    check(g, ones, None, dtype, True, "expanded")


@pytest.mark.gpu
def test_grouped_linear_no_rows_and_offsets_out_of_range():
    from diverse_conventions_amd import grouped_linear
    w, b = torch.randn((3, 8, 4), device="cuda").requires_grad_(), torch.randn((3, 8), device="cuda").requires_grad_()
    x = torch.randn((0, 4), device="cuda").requires_grad_()
    y = grouped_linear(x, w, torch.zeros(4, dtype=torch.int32, device="cuda"), b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.zeros((0, 8), device="cuda"))
    assert y.shape == (0, 8) and dx.shape == (0, 4) and not dw.any() and not db.any()
    x = torch.randn((10, 4), device="cuda")
    with torch.no_grad():
        clamped = grouped_linear(x, w, torch.tensor([-5, 3, 7, 99], device="cuda"), b)
        assert torch.equal(clamped, grouped_linear(x, w, torch.tensor([0, 3, 7, 10], device="cuda"), b))


@pytest.mark.gpu
def test_grouped_linear_refusals():
    from diverse_conventions_amd import grouped_linear
    x, w, b, o = torch.randn((10, 4), device="cuda"), torch.randn((3, 8, 4), device="cuda"), torch.randn((3, 8), device="cuda"), torch.tensor([0, 3, 7, 10], device="cuda")
    for bad in (dict(x=x.double()), dict(x=x.cpu()), dict(x=x[0]), dict(x=x.t().contiguous().t()), dict(x=x[:1].expand(10, 4)), dict(weight=w.half()),
                dict(weight=w[:, :, :3]), dict(weight=w.transpose(1, 2).contiguous().transpose(1, 2)), dict(weight=w[:0]), dict(bias=b[:2]), dict(bias=b.half()),
                dict(offsets=o[:3]), dict(offsets=o.float()), dict(offsets=o.cpu())):
        with pytest.raises(ValueError):
            grouped_linear(**{**dict(x=x, weight=w, offsets=o, bias=b), **bad})


def test_grouped_linear_refuses_on_the_host():
    from diverse_conventions_amd import grouped_linear, native
    with pytest.raises(ValueError):
        grouped_linear(torch.zeros((4, 4)), torch.zeros((1, 4, 4)), torch.tensor([0, 4]))
    L, a = native.lib(), native.OcGroupedLinearArgs()
    assert L.oc_grouped_linear(None, None, None) == -1 and L.oc_grouped_linear_workspace_bytes(None, 0) == -1
    assert L.oc_grouped_linear(ctypes.byref(a), None, None) == -1 and "groups 0" in L.oc_last_error().decode()
    a.groups, a.in_features, a.out_features, a.rows, a.x_stride = 2, 8, 8, 4, 7
    assert L.oc_grouped_linear(ctypes.byref(a), None, None) == -1 and "x_stride 7" in L.oc_last_error().decode()
    a.x_stride = 8
    assert L.oc_grouped_linear(ctypes.byref(a), None, None) == -1 and "NULL" in L.oc_last_error().decode()
    assert L.oc_grouped_linear_backward(ctypes.byref(a), None, None) == -1


def test_oracle_grouped_gradients_equal_differences():
    rng = np.random.default_rng(0)
    x, w, b, dy, cuts = rng.normal(size=(6, 3)), rng.normal(size=(2, 4, 3)), rng.normal(size=(2, 4)), rng.normal(size=(6, 4)), [1, 3, 5]
    _, dx, dw, db = update_oracle.grouped_linear(x, w, cuts, b, dy)
    value = lambda: (update_oracle.grouped_linear(x, w, cuts, b)[0] * dy).sum()
    for t, g in ((x, dx), (w, dw), (b, db)):
        for at in np.ndindex(t.shape):
            keep = t[at]
            t[at] = keep + 0.5
            up = value()
            t[at] = keep - 0.5
            assert abs(up - value() - g[at]) < 1e-12           # linear in each argument
            t[at] = keep


@pytest.mark.gpu
def test_grouped_linear_streams_and_graph():
    from diverse_conventions_amd import grouped_linear
    cases = []
    for sizes, k, n, dtype in (([40, 0, 2000], 24, 16, "f32"), ([300, 700, 1100], 512, 768, "bf16"), ([3, 1, 2], 64, 128, "f16")):
        x, w, b, dy, cuts = inputs(sizes, k, n, dtype, 8, False, tail=4)
        cases.append((x.requires_grad_(), w.requires_grad_(), b.requires_grad_(), dy, torch.tensor(cuts, dtype=torch.int32, device="cuda")))

    def step():
        out = []
        for x, w, b, dy, o in cases:
            y = grouped_linear(x, w, o, b)
            out += [y.detach(), *torch.autograd.grad(y, (x, w, b), dy)]
        return out

    want = step()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(2):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for r in range(4):
        for x, w, b, dy, o in cases:
            with torch.no_grad():
                x.normal_()
                dy.normal_()
        graph.replay()
        torch.cuda.synchronize()
        seen = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(seen, step())), r
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_a_population_of_critics_learns_in_one_pass():
    """Pairing segments as groups: two grouped layers, the value loss, gradients and clipping, against one network after the other."""
    from diverse_conventions_amd import clip_grad_norm, grouped_linear, pairing_segments, value_loss
    segments = pairing_segments(40, 3)
    cuts = [0]
    for s in segments:
        cuts.append(cuts[-1] + s.stop - s.start)
    groups, rows = len(segments), cuts[-1]
    g = torch.Generator(device="cuda").manual_seed(0)
    randn = lambda *s: torch.randn(s, device="cuda", generator=g)
    x, v0, ret = randn(rows, 192).relu(), randn(rows, 1), randn(rows, 1)
    params = [randn(groups, 64, 192) * 0.1, randn(groups, 64) * 0.1, randn(groups, 1, 64) * 0.1, randn(groups, 1)]
    offsets = torch.tensor(cuts, device="cuda")
    one = [p.clone().requires_grad_() for p in params]
    h = grouped_linear(x, one[0], offsets, one[1]).relu()
    value_loss(grouped_linear(h, one[2], offsets, one[3]), v0, ret).backward()
    norm = clip_grad_norm([p.grad for p in one], 0.01)
    two = [p.clone().double().requires_grad_() for p in params]
    out = []
    for i in range(groups):
        rows_i = x[cuts[i]:cuts[i + 1]].double()
        out.append((rows_i @ two[0][i].t().contiguous() + two[1][i]).relu() @ two[2][i].t().contiguous() + two[3][i])
    v = torch.cat(out)
    huber = lambda e: torch.where(e.abs() <= 10, e * e / 2, 10 * (e.abs() - 5))
    torch.max(huber(ret - v), huber(ret - (v0 + (v - v0).clamp(-0.2, 0.2)))).mean().backward()
    want = torch.nn.utils.clip_grad_norm_(two, 0.01)
    # f32 against f64: sums of up to 280 * 64 * 192 rounded terms; a hidden unit or a clip decided the other way would move a gradient by
    # one sample's share, 1 / 280 of it
    assert abs(float(norm) - float(want)) < 1e-3 * float(want)
    for a, b in zip(one, two):
        assert float((a.grad.double() - b.grad).norm()) < 1e-2 * float(b.grad.norm())


@pytest.mark.gpu
def test_grouped_linear_under_hooks_on_saved_tensors():
    from diverse_conventions_amd import grouped_linear
    x, w, b, dy, cuts = inputs([30, 20], 24, 40, "f32", 9, True)
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    got = []
    for hooked in (True, False):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        wide = torch.cat([leaves[0], leaves[0]], 1)
        with torch.autograd.graph.save_on_cpu() if hooked else torch.enable_grad():
            y = grouped_linear(wide[:, :24], leaves[1] * 1.0, offsets, leaves[2])
        del wide
        junk = [torch.full((50, 48), float("nan"), device="cuda") for _ in range(20)]
        got.append(torch.autograd.grad(y, leaves, dy))
        del junk
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.gpu
def test_grouped_linear_beyond_32_bit_offsets():
    """Weights of more than 2^31 elements, rows and results behind 2^31 elements: the last group against the same group alone."""
    from diverse_conventions_amd import grouped_linear
    k, n, groups = 1024, 2048, 1030                        # 2.16e9 weights
    w = torch.zeros((groups, n, k), dtype=torch.bfloat16, device="cuda")
    x, last, _, dy, _ = inputs([40], k, n, "bf16", 10, True)
    w[-1] = last[0]
    cuts = torch.zeros(groups + 1, dtype=torch.int64, device="cuda")
    cuts[-1] = 40
    y = grouped_linear(x, w, cuts)
    one = torch.tensor([0, 40], device="cuda")
    assert torch.equal(y, grouped_linear(x, last, one))
    del w
    rows = 1_100_000                                       # 2.25e9 results, 1.1e9 inputs
    big = torch.zeros((rows, k), dtype=torch.bfloat16, device="cuda")
    big[-40:] = x
    leaf, weight = big.requires_grad_(), last.clone().requires_grad_()
    y = grouped_linear(leaf, weight, torch.tensor([rows - 40, rows], device="cuda"))
    alone = [x.clone().requires_grad_(), last.clone().requires_grad_()]
    z = grouped_linear(alone[0], alone[1], one)
    assert torch.equal(y[-40:], z) and not y[:-40:9973].any() and not y[-41].any()
    d = torch.zeros_like(y)
    d[-40:] = dy
    dx, dw = torch.autograd.grad(y, (leaf, weight), d)
    zx, zw = torch.autograd.grad(z, alone, dy)
    assert torch.equal(dx[-40:], zx) and torch.equal(dw, zw) and not dx[:-40:9973].any() and not dx[-41].any()
    torch.cuda.empty_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("sizes,k,n", [([20000, 19111, 1], 16, 256), ([20000, 19111, 1], 72, 256), ([39000], 104, 264), ([39000], 160, 256),
                                       ([0, 1, 5, 40, 64, 65, 130, 200] * 2, 1024, 1024), ([9000, 0, 10001], 1024, 24), ([9000, 3, 10001], 1024, 136)],
                         ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)}g{sum(v)}")
def test_grouped_linear_large_tiles_of_few_steps(sizes, k, n, dtype):
    """Reductions of none to a few steps through the tiles whose pipeline is deeper than that: short rows, narrow results, groups of few rows."""
    run_and_check(sizes, k, n, dtype, 11, True, tail=1)


@pytest.mark.gpu
def test_grouped_linear_large_tiles_in_a_graph():
    from diverse_conventions_amd import grouped_linear
    x, w, b, dy, cuts = inputs([1000, 2048, 1500], 768, 2560, "bf16", 12, False, tail=4)
    o, leaves = torch.tensor(cuts, dtype=torch.int32, device="cuda"), [t.requires_grad_() for t in (x, w, b)]

    def step():
        y = grouped_linear(x, w, o, b)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for r in range(4):
        with torch.no_grad():
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        seen = [t.clone() for t in held]
        assert all(torch.equal(a, c) for a, c in zip(seen, step())), r
        torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("sizes,k,n", [([1], 4096, 64), ([3], 2000, 520), ([33, 0, 5], 1032, 1000), ([120], 4100, 200), ([50], 999, 2001), ([200, 90], 600, 70),
                                       ([7], 64, 4096), ([100], 130, 2056)], ids=lambda v: str(v) if isinstance(v, int) else f"{len(v)}g{sum(v)}")
def test_grouped_linear_few_rows_of_many_features(sizes, k, n, dtype):
    """Products whose reduction is cut and joined: forward over in_features, dx over out_features; rows of no group, without and with a bias."""
    run_and_check(sizes, k, n, dtype, 13, True, head=2, tail=3)
    run_and_check(sizes, k, n, dtype, 14, True, bias=False)
    run_and_check(sizes, k, n, dtype, 15, False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_grouped_linear_one_gradient_at_a_time(dtype):
    """Only x, only the weights or only the bias wants a gradient: the others are not computed, the workspace holds what is."""
    from diverse_conventions_amd import grouped_linear
    for sizes, k, n in (([3000, 0, 40], 24, 72), ([5], 2048, 600)):
        x, w, b, dy, cuts = inputs(sizes, k, n, dtype, 16, True)
        offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda")
        want = update_oracle.grouped_linear(f64(x), f64(w), cuts, f64(b), f64(dy))[1:]
        for only in range(3):
            args = [t.clone().requires_grad_() if i == only else t for i, t in enumerate((x, w, b))]
            y = grouped_linear(args[0], args[1], offsets, args[2])
            check(torch.autograd.grad(y, args[only], dy)[0], want[only], None, dtype, True, only)
