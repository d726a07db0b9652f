"""Rows of one batch that go through different weights, against plain forms in 64 bits: the gate's choice (bz_route_topk), entries and
rows in their groups' order (bz_group_rows), results back at their rows and the gradient of that (bz_merge_rows, bz_merge_rows_grad),
every group's layer (bz_grouped_fc), a shared layer with an adapter a row (bz_fc_adapters).

Bars.  Choices, orders, positions and moved rows are exact.  Sums: an output of type t is rounded once, half a step of t relative to it
(2^-8 bf16, 2^-11 fp16, 2^-24 fp32), and an fp32 sum of K products is off by at most (K + 4) * 2^-24 of the sum of their absolute
values, K counting every addition in any order.  Activations have slopes of at most 1 (SwiGLU's are written where they are used), and
exp, reciprocal and division by at most 16 * 2^-24.  The low-rank factor of 2-byte layers is two bf16s, 2^-17 of it.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_STEP = {"bf16": 2.0**-8, "f16": 2.0**-11, "f32": 2.0**-24}
EPS = 2.0**-24


@pytest.fixture(scope="module")
def bz():
    import torch
    import blaze_hip
    assert torch.cuda.is_available(), "no GPU visible"
    blaze_hip.device_check()
    return blaze_hip


def _t(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _normal(seed, shape, std=1.0, dtype="f32"):
    x = np.random.default_rng(seed).standard_normal(shape).astype(np.float32) * np.float32(std)
    import torch
    return torch.from_numpy(x).cuda().to(_t(dtype))


def _pitched(x, pad, fill):
    """the same matrix (or stack) with `pad` more elements a row, which hold `fill`"""
    import torch
    if pad == 0:
        return x
    wide = torch.full((*x.shape[:-1], x.shape[-1] + pad), fill, dtype=x.dtype, device=x.device)
    wide[..., :x.shape[-1]] = x
    return wide[..., :x.shape[-1]]


def _close(got, want, bar, what):
    import torch
    off = (got.double() - want).abs()
    same = (got.double() == want) | (torch.isnan(got.double()) & torch.isnan(want))
    bad = ~((off <= bar) | same)
    assert not bool(bad.any()), "%s: %d of %d off, the worst by %.3g where %.3g is allowed" % (
        what, int(bad.sum()), bad.numel(), float(off[bad].max()), float(bar.expand_as(off)[bad][off[bad].argmax()]))


# ---------------------------------------------------------------------------------------------- the gate's choice
def _route_want(l, k, score, renorm, scale):
    """by Python's own sort of (logit, index)"""
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    ids, ws = [], []
    for row in l:
        best = sorted((i for i in range(len(row)) if row[i] > -np.inf), key=lambda i: (-row[i], i))[:k]
        if score == "softmax":
            m = max(row)
            e = [1.0 if row[i] == m else np.exp(row[i] - m) if row[i] > -np.inf else 0.0 for i in range(len(row))]
            w = [e[i] / sum(e) for i in best]
        else:
            w = [1.0 / (1.0 + np.exp(-row[i])) for i in best]
        if renorm:
            w = [x / sum(w) if sum(w) > 0 else 0.0 for x in w]
        ids.append(best + [-1] * (k - len(best)))
        ws.append([x * scale for x in w] + [0.0] * (k - len(best)))
    return np.array(ids, np.int32).reshape(-1, k), np.array(ws, np.float64).reshape(-1, k)


@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 8, 2), (3, 16, 16), (65, 17, 3), (300, 60, 4), (257, 64, 1), (33, 100, 8), (50, 128, 16), (19, 160, 6),
                                      (9, 256, 8), (7, 257, 5), (5, 1000, 16), (2, 1024, 8)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_route_topk(bz, rows, n, k, dtype):
    print("case", rows, n, k, dtype, flush=True)
    logits = _normal(rows * n + k, (rows, n), 1.5, dtype)
    if dtype != "f32":
        logits = (logits * 4).round() / 4  # ties in most rows
    logits = _pitched(logits, (rows + k) % 3, 100.0)
    for score in ("softmax", "sigmoid"):
        for renorm in (False, True):
            ids, w = bz.route_topk(logits, k, score={"softmax": bz.ROUTE_SOFTMAX, "sigmoid": bz.ROUTE_SIGMOID}[score], renormalize=renorm, scale=1.5)
            want_ids, want = _route_want(logits.float().cpu().numpy(), k, score, renorm, 1.5)
            assert np.array_equal(ids.cpu().numpy(), want_ids)
            # exp, a sum of n terms, two divisions
            np.testing.assert_allclose(w.cpu().numpy(), want, rtol=(n + 32) * EPS, atol=0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [6, 40, 128, 200, 600])
def test_route_topk_of_what_is_no_number(bz, dtype, n):
    import torch
    inf, nan = float("inf"), float("nan")
    logits = _normal(n, (12, n), 1.0, dtype)
    logits[0] = -inf
    logits[1] = nan
    logits[2, 1:] = -inf
    logits[3, ::2] = nan
    logits[4] = torch.finfo(logits.dtype).min
    logits[5, 3] = inf
    logits[6, 1] = logits[6, 4] = inf
    logits[7] = 0.0
    logits[8, : n - 2] = -inf
    logits[9] = torch.finfo(logits.dtype).max
    for score in ("softmax", "sigmoid"):
        for renorm in (False, True):
            ids, w = bz.route_topk(logits, 5, score={"softmax": bz.ROUTE_SOFTMAX, "sigmoid": bz.ROUTE_SIGMOID}[score], renormalize=renorm)
            with np.errstate(all="ignore"):
                want_ids, want = _route_want(logits.float().cpu().numpy(), 5, score, renorm, 1.0)
            assert np.array_equal(ids.cpu().numpy(), want_ids)
            np.testing.assert_allclose(w.cpu().numpy(), want, rtol=(n + 32) * EPS, atol=2.0**-126)  # (e^-88 and below may be flushed)


def test_route_topk_of_no_rows(bz):
    import torch
    ids, w = bz.route_topk(torch.empty((0, 8), device="cuda"), 2)
    assert ids.shape == (0, 2) and w.shape == (0, 2)


# ---------------------------------------------------------------------------------------------- entries in their groups' order
def _group_want(ids, groups):
    order = [i for g in range(groups) for i in np.nonzero(ids == g)[0]]
    position = np.full(ids.size, -1, np.int32)
    position[order] = np.arange(len(order))
    return np.concatenate([[0], np.cumsum([(ids == g).sum() for g in range(groups)])]).astype(np.int32), np.array(order, np.int32), position


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 255, 256, 257, 1000, 4096, 8191, 8192, 8193, 10000, 65537, 600001])
@pytest.mark.parametrize("groups", [1, 2, 7, 64, 128, 1000, 1024])
def test_group_rows_orders_entries(bz, n, groups):
    import torch
    print("case", n, groups, flush=True)
    rng = np.random.default_rng(n + groups)
    ids = rng.integers(0, groups, n).astype(np.int32)
    if groups > 2:
        ids[rng.random(n) < 0.5] = groups // 2  # one crowded group
        ids[ids == 1] = 0                       # one empty one
    out = rng.random(n) < 0.1
    ids[out] = rng.choice([-1, groups, groups + 5, -2**31, 2**31 - 1], out.sum())
    dev = torch.from_numpy(ids).cuda()
    order = torch.full((n, ), 77, dtype=torch.int32, device="cuda")
    offsets, order, position = bz.group_rows(dev, groups, order=order)
    want_offsets, want_order, want_position = _group_want(ids, groups)
    assert np.array_equal(offsets.cpu().numpy(), want_offsets)
    assert np.array_equal(position.cpu().numpy(), want_position)
    kept = len(want_order)
    assert np.array_equal(order.cpu().numpy()[:kept], want_order) and (order[kept:] == 77).all()
    again = bz.group_rows(dev, groups)
    assert torch.equal(again[0], offsets) and torch.equal(again[1][:kept], order[:kept]) and torch.equal(again[2], position)


def test_group_rows_of_one_group_and_of_none(bz):
    import torch
    ids = torch.full((9000, ), 3, dtype=torch.int32, device="cuda")
    offsets, order, position = bz.group_rows(ids, 8)
    assert offsets.tolist() == [0, 0, 0, 0] + [9000] * 5 and order.tolist() == list(range(9000)) == position.tolist()
    offsets, _, position = bz.group_rows(torch.full((9000, ), -1, dtype=torch.int32, device="cuda"), 8)
    assert offsets.tolist() == [0] * 9 and (position == -1).all()
    offsets, order, position = bz.group_rows(torch.empty(0, dtype=torch.int32, device="cuda"), 5)
    assert offsets.tolist() == [0] * 6 and order.numel() == 0 == position.numel()


@pytest.mark.parametrize("rows,k,groups,dim", [(1, 1, 1, 1), (1, 4, 8, 2048), (5, 2, 3, 7), (100, 3, 8, 445), (64, 8, 60, 13), (300, 16, 32, 96), (2048, 2, 8, 896),
                                               (3000, 6, 64, 33), (1500, 8, 128, 256)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_group_rows_moves_rows(bz, rows, k, groups, dim, dtype):
    import torch
    print("case", rows, k, groups, dim, dtype, flush=True)
    rng = np.random.default_rng(rows + dim)
    ids = rng.integers(0, groups, (rows, k)).astype(np.int32)
    ids[rng.random(rows) < 0.2] = -1
    x = _pitched(_normal(dim, (rows, dim), 1.0, dtype), rows % 2 * 3, 9.0)
    x[0, 0] = float("nan")
    out = _pitched(torch.full((rows * k, dim), 5.0, dtype=x.dtype, device="cuda"), rows % 3, 6.0)
    offsets, order, position, xs = bz.group_rows(torch.from_numpy(ids).cuda(), groups, x=x, out=out)
    _, want_order, _ = _group_want(ids.reshape(-1), groups)
    kept = len(want_order)
    want = x.cpu()[torch.from_numpy(want_order // k).long()]
    assert torch.equal(xs[:kept].cpu().view(torch.int32 if dtype == "f32" else torch.int16), want.view(torch.int32 if dtype == "f32" else torch.int16))
    assert (xs[kept:] == 5.0).all()
    if rows % 3:
        assert (out.as_strided((rows * k - 1, rows % 3), (out.stride(0), 1), out.storage_offset() + dim) == 6.0).all()


@pytest.mark.parametrize("rows,k,groups,dim", [(8192, 2, 1000, 20), (8192, 1, 3, 40), (8193, 1, 5, 16), (1024, 16, 30, 50), (1025, 16, 30, 9), (4000, 4, 512, 24)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_group_rows_moves_rows_of_some_thousand_entries(bz, rows, k, groups, dim, dtype):
    test_group_rows_moves_rows(bz, rows, k, groups, dim, dtype)


@pytest.mark.parametrize("dim", [901, 904, 1024])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_group_rows_moves_more_than_the_caches_keep(bz, dim, dtype):
    import torch
    rows, k, groups = 40000, 2, 50
    ids = torch.from_numpy(np.random.default_rng(dim).integers(-1, groups, (rows, k)).astype(np.int32)).cuda()
    x = _normal(dim, (rows, dim), 1.0, dtype)
    out = torch.full((rows * k + 2, dim + 1), 5.0, dtype=x.dtype, device="cuda")
    offsets, order, position, xs = bz.group_rows(ids, groups, x=x, out=out[1:-1, :dim])
    kept = int(offsets[-1])
    assert kept == int((ids >= 0).sum()) and torch.equal(xs[:kept], x[order[:kept].long() // k])
    assert bool((xs[kept:] == 5.0).all()) and bool((out[:, dim] == 5.0).all()) and bool((out[0] == 5.0).all()) and bool((out[-1] == 5.0).all())


# ---------------------------------------------------------------------------------------------- results back at their rows
def _positions(seed, rows, k, spare):
    """every entry a position of its own among rows * k + spare, some none"""
    rng = np.random.default_rng(seed)
    p = rng.permutation(rows * k + spare)[:rows * k].astype(np.int32).reshape(rows, k)
    p[rng.random((rows, k)) < 0.2] = -1
    p[rng.random(rows) < 0.1] = -1
    if rows > 3:
        p[2, 0], p[3, 0] = rows * k + spare, 2**31 - 1  # outside
    import torch
    return torch.from_numpy(p).cuda()


MERGES = [(1, 1, 1), (1, 8, 2048), (4, 2, 7), (33, 3, 3), (300, 4, 445), (129, 16, 130), (64, 5, 1000), (700, 8, 96), (2048, 2, 513)]


@pytest.mark.parametrize("rows,k,dim", MERGES)
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("weighted", [True, False])
def test_merge_rows(bz, rows, k, dim, dtype, out, weighted):
    import torch
    print("case", rows, k, dim, dtype, out, weighted, flush=True)
    position = _positions(rows + dim, rows, k, 3)
    n = rows * k + 3
    xs = _pitched(_normal(dim, (n, dim), 1.0, dtype), dim % 3, 9.0)
    there = (position >= 0) & (position < n)
    named = torch.zeros(n, dtype=torch.bool, device="cuda")
    named[position[there].long()] = True
    xs[~named] = float("nan")  # no row that nobody names is looked at
    w = _normal(k, (rows, k)) if weighted else None
    y = _pitched(torch.full((rows, dim), 3.0, dtype=_t(out), device="cuda"), rows % 3, 7.0)
    bz.merge_rows(xs, position, w, out=y)
    terms = torch.where(there[:, :, None], xs[position.clamp(0, n - 1).long()].double() * (w.double()[:, :, None] if weighted else 1.0), 0.0)
    want = terms.sum(1)
    _close(y, want, HALF_STEP[out] * want.abs() * (1 + 2.0**-8) + (k + 4) * EPS * terms.abs().sum(1) + 2.0**-25 * (out == "f16"), "y")
    assert bool((y[~there.any(1)] == 0).all())
    assert torch.equal(y, bz.merge_rows(xs, position, w, out_dtype={"f32": bz.F32, "f16": bz.F16, "bf16": bz.BF16}[out]))


@pytest.mark.parametrize("rows,k,dim", MERGES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("weighted", [True, False])
def test_merge_rows_gradient(bz, rows, k, dim, dtype, weighted):
    import torch
    print("case", rows, k, dim, dtype, weighted, flush=True)
    position = _positions(rows + dim, rows, k, 3)
    n = rows * k + 3
    xs = _pitched(_normal(dim, (n, dim), 1.0, dtype), dim % 2, 9.0)
    dy = _pitched(_normal(dim + 1, (rows, dim), 1.0, dtype), rows % 2, 9.0)
    w = _normal(k, (rows, k)) if weighted else None
    there = (position >= 0) & (position < n)
    named = torch.zeros(n, dtype=torch.bool, device="cuda")
    named[position[there].long()] = True
    xs[~named] = float("nan")
    dxs = _pitched(torch.full((n, dim), 4.0, dtype=xs.dtype, device="cuda"), rows % 3, 7.0)
    dxs, dw = bz.merge_rows_grad(dy, xs, position, w, dxs=dxs)
    t, j = torch.nonzero(there, as_tuple=True)
    want = torch.full((n, dim), 4.0, dtype=torch.float64, device="cuda")
    want[position[t, j].long()] = dy[t].double() * (w[t, j, None].double() if weighted else 1.0)
    _close(dxs, want, (HALF_STEP[dtype] + EPS) * want.abs() * (1 + 2.0**-8) + 2.0**-25 * (dtype == "f16"), "dxs")
    assert bool((dxs[~named] == 4.0).all())
    products = torch.where(there[:, :, None], xs[position.clamp(0, n - 1).long()].double() * dy.double()[:, None, :], 0.0)
    _close(dw, products.sum(2), (dim + 4) * EPS * products.abs().sum(2), "dweights")
    assert bool((dw[~there] == 0).all())


@pytest.mark.parametrize("rows,k,dim,dtype", [(20000, 2, 901, "f32"), (40000, 2, 905, "bf16"), (9000, 8, 1024, "f16"), (16000, 16, 264, "bf16")])
def test_merge_rows_gradient_of_more_than_the_caches_keep(bz, rows, k, dim, dtype):
    test_merge_rows_gradient(bz, rows, k, dim, dtype, True)


def test_merge_gradient_is_what_differences_give(bz):
    """merge_rows is linear in the rows and in the weights: the difference over a step of 1 is the derivative, up to rounding."""
    import torch
    rows, k, dim = 40, 3, 50
    ids = torch.from_numpy(np.random.default_rng(0).integers(-1, 6, (rows, k)).astype(np.int32)).cuda()
    x = _normal(1, (rows, dim))
    offsets, order, position, xs = bz.group_rows(ids, 6, x=x, out=torch.zeros((rows * k, dim), device="cuda"))
    w, dy = _normal(2, (rows, k)), _normal(3, (rows, dim))
    dxs, dw = bz.merge_rows_grad(dy, xs, position, w)
    loss = lambda r, v: (bz.merge_rows(r, position, v).double() * dy.double()).sum()  # noqa: E731
    step_xs, step_w = _normal(4, xs.shape), _normal(5, w.shape)
    # 64 bits from y on: each y is off by (k + 5) steps of at most the terms' sizes, and there are rows * dim of them
    bar = 2 * (k + 5) * EPS * 4 * float((dy.abs().double().sum() * k * 16))
    assert abs(float(loss(xs + step_xs, w) - loss(xs, w)) - float((dxs.double() * step_xs.double()).sum())) < bar
    assert abs(float(loss(xs, w + step_w) - loss(xs, w)) - float((dw.double() * step_w.double()).sum())) < bar
    # and the move's own gradient is the merge without weights
    dx = bz.merge_rows(dxs, position)
    moved = lambda v: (bz.group_rows(ids, 6, x=v, out=torch.zeros_like(dxs))[3].double() * dxs.double()).sum()  # noqa: E731
    step = _normal(6, x.shape)
    assert abs(float(moved(x + step) - moved(x)) - float((dx.double() * step.double()).sum())) < bar


# ---------------------------------------------------------------------------------------------- layers
def _act(bz, name, n, groups, seed):
    """(arguments of the call, f(v [rows, n], group) in 64 bits, slope bound)"""
    import torch
    if name == "prelu":
        s = _normal(seed, (groups, n)).abs().clamp(max=1.0).contiguous()
        return dict(act=bz.ACT_PRELU, act_params=(s, )), lambda v, g: torch.where(v > 0, v, v * s[g].double())
    if name == "relu":
        return dict(act=bz.ACT_LEAKY_RELU, act_alpha=0.0), lambda v, g: v.clamp(min=0)
    if name == "leaky":
        return dict(act=bz.ACT_LEAKY_RELU, act_alpha=0.25), lambda v, g: torch.where(v >= 0, v, 0.25 * v)
    if name == "sigmoid":
        return dict(act=bz.ACT_SIGMOID), lambda v, g: torch.sigmoid(v)
    if name == "dice":
        gamma, mean = _normal(seed, (groups, n), 0.1), _normal(seed + 1, (groups, n), 0.1)
        var = _normal(seed + 2, (groups, n)).abs() + 1.0

        def dice(v, g):
            p = torch.sigmoid((v - mean[g].double()) / torch.sqrt(var[g].double() + 1e-8))
            return ((1 - p) * gamma[g].double() + p) * v
        return dict(act=bz.ACT_DICE, act_params=(gamma, mean, var)), dice
    return dict(act=bz.ACT_NONE), lambda v, g: v


def _cuts(seed, m, groups, spare):
    """offsets of groups of all lengths, none among them, over m - spare rows"""
    rng = np.random.default_rng(seed)
    share = rng.random(groups)**3 * (rng.random(groups) > 0.25)
    share = share / max(share.sum(), 1e-9)
    cuts = np.concatenate([[0], np.round(np.cumsum(share) * (m - spare))]).astype(np.int32)
    cuts[-1] = m - spare if share.sum() > 0 else 0
    return cuts


def _grouped_case(bz, m, n, k, groups, dtype, out, act, gather, pads=(0, 0, 0), seed=0, spare=0, bias=True):
    import torch
    gated = act == "swiglu"
    cols = 2 * n if gated else n
    per = 3
    source = (m + per - 1) // per if gather else m
    cuts = _cuts(seed, m, groups, spare)
    a = _pitched(_normal(seed + 1, (max(source, 1), k), 1.0, dtype), pads[0], float("nan"))
    w = _pitched(_normal(seed + 2, (groups, cols, k), 1.0 / np.sqrt(k), dtype), pads[1], float("nan"))
    b = _normal(seed + 3, (groups, cols), 0.1) if bias else None
    rows = None
    if gather:
        r = np.random.default_rng(seed + 4).integers(0, source * per, m).astype(np.int32)
        if m > 4:
            r[1], r[3] = -per, source * per + 2  # rows of zeros
        rows = torch.from_numpy(r).cuda()
    args, f = (dict(act=bz.ACT_SWIGLU), None) if gated else _act(bz, act, n, groups, seed + 5)
    y = _pitched(torch.full((m, n), 3.0, dtype=_t(out), device="cuda"), pads[2], 7.0)
    got = bz.grouped_fc(a, w, torch.from_numpy(cuts).cuda(), k, rows=rows, rows_per=per if gather else 1, bias=b, out=y, **args)
    assert got is y
    if gather:
        at = torch.div(rows, per, rounding_mode="trunc").long()
        there = (at >= 0) & (at < source)
        x = torch.where(there[:, None], a[at.clamp(0, source - 1)].double(), 0.0)
    else:
        x = a.double()
    steps = (k + 8) * EPS
    for g in range(groups):
        lo, hi = int(cuts[g]), int(cuts[g + 1])
        if lo == hi:
            continue
        wg = w[g].double().contiguous()
        v = x[lo:hi] @ wg.t() + (b[g].double() if bias else 0.0)
        size = x[lo:hi].abs() @ wg.abs().t() + (b[g].abs().double() if bias else 0.0)
        if gated:
            gate, up = v[:, :n], v[:, n:]
            want = gate * torch.sigmoid(gate) * up
            # |silu'| <= 1.1, and both factors as wrong as they may be
            bar = 1.1 * steps * size[:, :n] * (up.abs() + steps * size[:, n:]) + gate.abs() * steps * size[:, n:] + 16 * EPS * want.abs()
        else:
            want = f(v, g)
            bar = (2.0 if act == "dice" else 1.0) * steps * size + 16 * EPS * (want.abs() + (v.abs() if act == "dice" else 0.0))
        _close(y[lo:hi], want, HALF_STEP[out] * (want.abs() + bar) + bar + (2.0**-25 if out == "f16" else 2.0**-120), "group %d, rows %d..%d" % (g, lo, hi))
    assert bool((y[int(cuts[-1]):] == 3.0).all()), "rows behind the last group"
    if pads[2] and m > 1:
        assert bool((y.as_strided((m - 1, pads[2]), (y.stride(0), 1), y.storage_offset() + n) == 7.0).all()), "between rows"
    return y


GROUPED = [(1, 1, 1, 1), (1, 16, 8, 4), (2, 8, 3, 2), (7, 33, 5, 3), (16, 64, 64, 4), (33, 40, 100, 8), (64, 256, 512, 16), (65, 130, 130, 5), (100, 200, 80, 6),
           (200, 512, 896, 8), (513, 96, 1000, 60), (600, 264, 200, 3), (1500, 128, 72, 1000), (2000, 320, 256, 2)]


@pytest.mark.parametrize("m,n,k,groups", GROUPED)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped_fc(bz, m, n, k, groups, dtype, gather):
    for i, act in enumerate(["none", "swiglu"]):
        print("case", m, n, k, groups, dtype, gather, act, flush=True)
        _grouped_case(bz, m, n, k, groups, dtype, dtype, act, gather, seed=m + n + k, spare=min(m // 4, 5) * i)


@pytest.mark.parametrize("m,n,k,groups", [(2600, 5000, 136, 3), (5000, 2560, 520, 7), (1100, 13000, 8, 2), (6000, 2100, 64, 70)])
@pytest.mark.parametrize("dtype,out,act", [("f16", "f16", "none"), ("bf16", "bf16", "swiglu"), ("bf16", "f32", "prelu"), ("f16", "f32", "swiglu"), ("f16", "f16", "dice")])
def test_grouped_fc_of_many_rows(bz, m, n, k, groups, dtype, out, act):
    print("case", m, n, k, groups, dtype, out, act, flush=True)
    _grouped_case(bz, m, n, k, groups, dtype, out, act, True, (8, 16, 0), seed=m, spare=3)
    _grouped_case(bz, m, n, k, groups, dtype, out, act, False, (0, 0, 1), seed=m + 1, bias=False)


@pytest.mark.parametrize("act", ["none", "prelu", "relu", "leaky", "sigmoid", "dice", "swiglu"])
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16")])
def test_grouped_fc_activations_and_pitches(bz, act, dtype, out):
    for m, n, k, groups, pads in ((70, 72, 96, 5, (0, 0, 0)), (300, 100, 130, 7, (1, 3, 5)), (12, 64, 256, 3, (8, 8, 8))):
        for bias in (True, False):
            print("case", act, dtype, out, m, n, k, groups, pads, bias, flush=True)
            _grouped_case(bz, m, n, k, groups, dtype, out, act, True, pads, seed=m, spare=2, bias=bias)


def test_grouped_fc_of_one_slope_a_group(bz):
    import torch
    a, w = _normal(0, (9, 16)), _normal(1, (3, 8, 16))
    slope = torch.tensor([0.5, 0.25, 0.125], device="cuda")
    y = bz.grouped_fc(a, w, torch.tensor([0, 2, 5, 9], dtype=torch.int32, device="cuda"), 16, act=bz.ACT_PRELU, act_params=(slope, ))
    g = torch.tensor([0, 0, 1, 1, 1, 2, 2, 2, 2], device="cuda")
    v = torch.matmul(w.double()[g], a.double()[:, :, None])[:, :, 0]
    _close(y, torch.where(v > 0, v, v * slope.double()[g, None]), 24 * EPS * 16 * torch.ones_like(v), "y")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_grouped_fc_offsets_that_make_no_sense_touch_nothing_outside(bz, dtype):
    import torch
    m, n, k = 40, 24, 32
    a, w = _normal(0, (m, k), 1.0, dtype), _normal(1, (4, n, k), 1.0, dtype)
    whole = torch.full((m + 20, n), 3.0, dtype=a.dtype, device="cuda")
    for cuts in ([0, 30, 10, 20, 90], [-5, 3, 3, 3, 3], [50, 60, 70, 80, 90], [2**31 - 1, 0, -2**31, 8, 8]):
        whole.fill_(3.0)
        bz.grouped_fc(a, w, torch.tensor(cuts, dtype=torch.int32, device="cuda"), k, out=whole[10:10 + m])
        assert bool((whole[:10] == 3.0).all()) and bool((whole[10 + m:] == 3.0).all())


def test_grouped_fc_rows_do_not_reach_into_each_other(bz):
    """what is no number in one row or one group's weight stays there"""
    import torch
    for dtype in ("f32", "f16", "bf16"):
        m, n, k = 90, 48, 72
        cuts = torch.tensor([0, 20, 50, 90], dtype=torch.int32, device="cuda")
        a, w = _normal(0, (m, k), 1.0, dtype), _normal(1, (3, n, k), 1.0, dtype)
        want = bz.grouped_fc(a, w, cuts, k)
        a2, w2 = a.clone(), w.clone()
        a2[25, 3], a2[70, k - 1], w2[0] = float("nan"), float("inf"), float("nan")
        got = bz.grouped_fc(a2, w2, cuts, k)
        keep = [r for r in range(20, m) if r not in (25, 70)]
        assert torch.equal(got[keep], want[keep])
        assert bool(torch.isnan(got[:20]).all()) and bool(torch.isnan(got[25]).all())


@pytest.mark.parametrize("m,n,k,groups", [(600, 160, 200, 2), (3000, 600, 72, 3)])
def test_grouped_fc_fp32_of_what_is_no_number_or_close_to_it(bz, m, n, k, groups):
    """infinities, NaNs, the largest and the smallest floats, where operands are multiplied in pieces"""
    import torch
    inf, nan, big = float("inf"), float("nan"), torch.finfo(torch.float32).max
    cuts = torch.tensor([m * g // groups for g in range(groups + 1)], dtype=torch.int32, device="cuda")
    a, w = _normal(0, (m, k)), _normal(1, (groups, n, k), 1.0 / np.sqrt(k))
    a[3, 5], a[4, 0], a[5], a[70, 7] = inf, -inf, inf, nan
    w[0, 9, 2], w[0, 33] = nan, 1e-30
    a[100] = 0.0
    a[101, 1:], a[101, 0] = 0.0, big      # finite products of the largest float
    a[102] = 1e-37
    a[103:110] *= 1e30
    last = int(cuts[-2])
    a[last + 1], a[last + 2] = big, -1e38  # sums that overflow, or not
    w[-1, :20] = w[-1, :20].abs()
    got = bz.grouped_fc(a, w, cuts, k).double()
    for g in range(groups):
        lo, hi = int(cuts[g]), int(cuts[g + 1])
        x, v = a[lo:hi].double(), w[g].double()
        want = torch.zeros((hi - lo, n), dtype=torch.float64, device="cuda")
        size = torch.zeros_like(want)
        for j in range(k):  # column by column: infinite terms as IEEE has them
            want += x[:, j, None] * v[None, :, j]
            size += (x[:, j, None] * v[None, :, j]).abs()
        fine = torch.isfinite(want) & (size < 3e38)
        # an operand below 2^-110 is off by up to 2^-126, times the largest of the other row (where the sum is finite, all of both are)
        bar = (k + 8) * EPS * size + k * 2.0**-126 * (1.0 + x.abs().amax(1, keepdim=True).clamp(max=1e38) + v.abs().amax(1)[None, :])
        _close(torch.where(fine, got[lo:hi], 0.0), torch.where(fine, want, 0.0), torch.where(fine, bar, 0.0), "finite sums of group %d" % g)
        bad = ~torch.isfinite(want)
        assert torch.equal(torch.isnan(got[lo:hi][bad]), torch.isnan(want[bad])) and torch.equal(torch.isinf(got[lo:hi][bad]), torch.isinf(want[bad]))
        assert bool((got[lo:hi][torch.isinf(want)] == want[torch.isinf(want)]).all())


@pytest.mark.parametrize("m,n,k,groups", [(2000, 640, 520, 3), (9000, 1100, 136, 9), (300, 96, 2048, 2)])
@pytest.mark.parametrize("act", ["none", "swiglu", "dice"])
def test_grouped_fc_fp32_of_many_rows(bz, m, n, k, groups, act):
    _grouped_case(bz, m, n, k, groups, "f32", "f32", act, True, (4, 8, 0), seed=m, spare=3)
    _grouped_case(bz, m, n, k, groups, "f32", "f32", act, False, (0, 0, 1), seed=m + 1, bias=False)


# lengths and widths at which layers are cut into tiles of every size, with and without alignment
LONGER = [(2000, 300, 77, 3), (1500, 1200, 45, 4), (2900, 520, 200, 5), (2100, 1100, 264, 1), (2100, 2000, 72, 9), (4300, 1030, 136, 6), (3900, 1000, 72, 1)]


@pytest.mark.parametrize("m,n,k,groups", LONGER)
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
def test_grouped_fc_of_some_thousand_rows(bz, m, n, k, groups, dtype, out):
    for i, act in enumerate(["none", "swiglu", "prelu"]):
        print("case", m, n, k, groups, dtype, out, act, flush=True)
        _grouped_case(bz, m, n, k, groups, dtype, out, act, i != 1, (8 * i, 8, i), seed=m + i, spare=7 * i, bias=i != 2)


def _adapters_case(bz, m, n, k, adapters, rank, dtype, out, act, pads=(0, 0, 0, 0), seed=0, segments=0, alpha=1.0, beta=1.0, bias=True, scale=True):
    import torch
    rng = np.random.default_rng(seed)
    a = _pitched(_normal(seed + 1, (m, k), 1.0, dtype), pads[0], float("nan"))
    w = _pitched(_normal(seed + 2, (n, k), 1.0 / np.sqrt(k), dtype), pads[1], float("nan"))
    down = _pitched(_normal(seed + 3, (adapters, rank, k), 1.0 / np.sqrt(k), dtype), pads[2], float("nan"))
    up = _pitched(_normal(seed + 4, (adapters, n, rank), 1.0 / np.sqrt(rank), dtype), pads[3], float("nan"))
    s = (_normal(seed + 5, (adapters, )).abs() + 0.25) if scale else None
    b = _normal(seed + 6, (n, ), 0.1) if bias else None
    if segments:
        ids = np.sort(rng.integers(0, segments, m)) * 7 % (adapters + 1) - 1
    else:
        ids = rng.integers(-1, adapters, m)
    ids = ids.astype(np.int32)
    if m > 2:
        ids[m // 2] = adapters + 3  # none
    used = set(ids.tolist())
    for g in range(adapters):  # nobody's: looked at by nobody
        if g not in used:
            down[g], up[g] = float("nan"), float("nan")
    args, f = _act(bz, act, n, 1, seed + 7)
    y = bz.fc_adapters(a, w, k, down, up, torch.from_numpy(ids).cuda(), rank=rank, scale=s, bias=b, alpha=alpha, beta=beta,
                       out_dtype={"f32": bz.F32, "f16": bz.F16, "bf16": bz.BF16}[out], **args)
    x, wd = a.double(), w.double()
    v = alpha * (x @ wd.t()) + (beta * b.double() if bias else 0.0)
    bar = (k + 8) * EPS * (abs(alpha) * (x.abs() @ wd.abs().t()) + (abs(beta) * b.abs().double() if bias else 0.0))
    size = v.abs()
    low_eps = EPS if dtype == "f32" else 2.0**-16
    for g in sorted(used):
        if 0 <= g < adapters:
            r = torch.from_numpy(np.nonzero(ids == g)[0]).cuda()
            dg, ug, sg = down[g].double().contiguous(), up[g].double().contiguous(), float(s[g]) if scale else 1.0
            low, low_size = sg * (x[r] @ dg.t()), sg * (x[r].abs() @ dg.abs().t())
            add = low @ ug.t()
            v[r] += add
            bar[r] += ((k + 8) * EPS * low_size + low_eps * low.abs()) @ ug.abs().t() + (3 * rank + 8) * EPS * (low.abs() @ ug.abs().t())
            size[r] += add.abs()
    want = f(v, 0)
    bar = (2.0 if act == "dice" else 1.0) * (bar + 4 * EPS * size) + 16 * EPS * (want.abs() + v.abs())
    _close(y, want, HALF_STEP[out] * (want.abs() + bar) + bar + (2.0**-25 if out == "f16" else 2.0**-120), "y")


ADAPTERS = [(1, 1, 1, 1, 1), (1, 64, 64, 3, 16), (2, 40, 100, 2, 8), (5, 33, 7, 4, 3), (31, 96, 130, 40, 5), (32, 256, 512, 64, 16), (33, 72, 200, 1, 4),
            (64, 130, 65, 9, 33), (100, 64, 64, 100, 8), (200, 200, 96, 12, 64), (300, 64, 896, 5, 17), (129, 48, 32, 2, 256), (700, 320, 256, 8, 32)]


@pytest.mark.parametrize("m,n,k,adapters,rank", ADAPTERS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("segments", [0, 6])
def test_fc_adapters(bz, m, n, k, adapters, rank, dtype, segments):
    print("case", m, n, k, adapters, rank, dtype, segments, flush=True)
    _adapters_case(bz, m, n, k, adapters, rank, dtype, dtype, "none", seed=m + n + k, segments=segments)


@pytest.mark.parametrize("act", ["none", "prelu", "relu", "sigmoid", "dice"])
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32"), ("bf16", "bf16")])
def test_fc_adapters_activations_and_pitches(bz, act, dtype, out):
    for m, n, k, adapters, rank, pads in ((70, 72, 96, 5, 8, (0, 0, 0, 0)), (90, 100, 130, 7, 12, (1, 3, 5, 1)), (40, 64, 256, 3, 16, (8, 8, 8, 8))):
        print("case", act, dtype, out, m, n, k, pads, flush=True)
        _adapters_case(bz, m, n, k, adapters, rank, dtype, out, act, pads, seed=m, segments=4, alpha=0.5, beta=2.0)
        _adapters_case(bz, m, n, k, adapters, rank, dtype, out, act, pads, seed=m + 1, bias=False, scale=False)


@pytest.mark.parametrize("m,n,k,adapters,rank", [(1300, 10000, 136, 5, 20), (3000, 4100, 72, 30, 64), (5100, 2600, 520, 3, 8)])
@pytest.mark.parametrize("dtype,out,act", [("f16", "f16", "none"), ("bf16", "bf16", "prelu"), ("bf16", "f32", "none"), ("f16", "f16", "sigmoid")])
def test_fc_adapters_of_many_rows(bz, m, n, k, adapters, rank, dtype, out, act):
    print("case", m, n, k, adapters, rank, dtype, out, act, flush=True)
    _adapters_case(bz, m, n, k, adapters, rank, dtype, out, act, (8, 16, 0, 8), seed=m, segments=9, alpha=0.5, beta=2.0)
    _adapters_case(bz, m, n, k, adapters, rank, dtype, out, act, (0, 0, 0, 0), seed=m + 1)


@pytest.mark.parametrize("m,n,k,adapters", LONGER)
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("rank", [7, 16, 96])
def test_fc_adapters_of_some_thousand_rows(bz, m, n, k, adapters, dtype, out, rank):
    print("case", m, n, k, adapters, dtype, out, rank, flush=True)
    _adapters_case(bz, m, n, k, adapters, rank, dtype, out, "none", (0, 8, 0, 0), seed=m, segments=9, alpha=0.5)
    _adapters_case(bz, m, n, k, adapters, rank, dtype, out, "prelu", (8, 0, 8, 8), seed=m + 1, bias=False, scale=False)


def test_fc_adapters_without_any_is_the_layer(bz):
    import torch
    a, w = _normal(0, (50, 64), 1.0, "f16"), _normal(1, (40, 64), 0.1, "f16")
    b = _normal(2, (40, ))
    none = torch.full((50, ), -1, dtype=torch.int32, device="cuda")
    y = bz.fc_adapters(a, w, 64, torch.empty((0, 8, 64), dtype=a.dtype, device="cuda"), torch.empty((0, 40, 8), dtype=a.dtype, device="cuda"), none, bias=b)
    z = bz.fc_adapters(a, w, 64, _normal(3, (2, 8, 64), 1.0, "f16"), _normal(4, (2, 40, 8), 1.0, "f16"), none, bias=b)
    want = a.double() @ w.double().t() + b.double()
    bar = 72 * EPS * (a.double().abs() @ w.double().abs().t() + b.double().abs()) + 2.0**-11 * want.abs() * 1.001 + 2.0**-25
    _close(y, want, bar, "no adapters")
    _close(z, want, bar, "adapters that nobody has")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_fc_adapters_reach_no_other_row(bz, dtype):
    """an adapter of infinities and NaNs, and a row of them, among 32 rows that share a block: every other row is bit for bit what it was"""
    import torch
    m, n, k, r = 64, 64, 64, 8
    a, w = _normal(0, (m, k), 1.0, dtype), _normal(1, (n, k), 1.0, dtype)
    down, up = _normal(2, (6, r, k), 1.0, dtype), _normal(3, (6, n, r), 1.0, dtype)
    ids = torch.arange(m, device="cuda", dtype=torch.int32) % 7 - 1
    want = bz.fc_adapters(a, w, k, down, up, ids)
    down2, up2, a2 = down.clone(), up.clone(), a.clone()
    down2[2], up2[4], a2[9] = float("inf"), float("nan"), float("nan")
    got = bz.fc_adapters(a2, w, k, down2, up2, ids)
    keep = (ids != 2) & (ids != 4)
    keep[9] = False
    assert torch.equal(got[keep], want[keep]) and bool(torch.isfinite(want[keep]).all())
    assert not bool(torch.isfinite(got[ids == 4]).any()) and not bool(torch.isfinite(got[ids == 2]).any())


def test_fc_adapters_factor_beyond_fp16(bz):
    """a low-rank factor of 10^5, which fp16 cannot hold, whose product with small weights it can"""
    import torch
    k = 256
    a, down = torch.full((8, k), 20.0, dtype=torch.float16, device="cuda"), torch.full((1, 4, k), 20.0, dtype=torch.float16, device="cuda")
    w, up = torch.zeros((16, k), dtype=torch.float16, device="cuda"), torch.full((1, 16, 4), 1e-3, dtype=torch.float16, device="cuda")
    y = bz.fc_adapters(a, w, k, down, up, torch.zeros(8, dtype=torch.int32, device="cuda"))
    want = 20.0 * 20.0 * k * 4 * float(up[0, 0, 0])
    assert bool(((y.double() - want).abs() <= want * (2.0**-11 + 2.0**-15)).all())


# ---------------------------------------------------------------------------------------------- together
def _mixture(bz, x, gate, w1, b1, w2, b2, experts, k, stream=None):
    logits = bz.fc_fused(x, gate, x.shape[1], out_dtype=bz.F32, stream=stream)
    ids, weights = bz.route_topk(logits, k, renormalize=True, stream=stream)
    offsets, order, position = bz.group_rows(ids, experts, stream=stream)
    h = bz.grouped_fc(x, w1, offsets, x.shape[1], rows=order, rows_per=k, bias=b1, act=bz.ACT_SWIGLU, stream=stream)
    y = bz.grouped_fc(h, w2, offsets, h.shape[1], bias=b2, stream=stream)
    return logits, bz.merge_rows(y, position, weights, out_dtype=bz.F32, stream=stream)


def _mixture_inputs(bz, T, dim, hidden, experts, dtype, seed=0):
    code = {"f32": bz.F32, "f16": bz.F16, "bf16": bz.BF16}[dtype]
    gate = bz.pack_weight(_normal(seed, (dim, experts), 1.0 / np.sqrt(dim)), False, code)
    w1, w2 = _normal(seed + 1, (experts, 2 * hidden, dim), dim**-0.5, dtype), _normal(seed + 2, (experts, dim, hidden), hidden**-0.5, dtype)
    return gate, w1, _normal(seed + 3, (experts, 2 * hidden), 0.1), w2, _normal(seed + 4, (experts, dim), 0.1), _normal(seed + 5, (T, dim), 1.0, dtype)


@pytest.mark.parametrize("T,dim,hidden,experts,k", [(1, 64, 32, 4, 2), (50, 72, 40, 8, 3), (333, 128, 96, 16, 4)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_mixture_of_experts(bz, T, dim, hidden, experts, k, dtype):
    import torch
    gate, w1, b1, w2, b2, x = _mixture_inputs(bz, T, dim, hidden, experts, dtype)
    logits, y = _mixture(bz, x, gate, w1, b1, w2, b2, experts, k)
    p = torch.softmax(logits.double(), 1)
    best = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :k]
    weights = p.gather(1, best) / p.gather(1, best).sum(1, keepdim=True)
    want, size = torch.zeros((T, dim), dtype=torch.float64, device="cuda"), torch.zeros((T, dim), dtype=torch.float64, device="cuda")
    for j in range(k):
        for e in range(experts):
            r = torch.nonzero(best[:, j] == e)[:, 0]
            if r.numel():
                v = x[r].double() @ w1[e].double().t() + b1[e].double()
                h = torch.nn.functional.silu(v[:, :hidden]) * v[:, hidden:]
                want[r] += weights[r, j, None] * (h @ w2[e].double().t() + b2[e].double())
                size[r] += weights[r, j, None] * (h.abs() @ w2[e].double().abs().t() + b2[e].double().abs())
    # h and an expert's result are rounded to the type, each half a step of it; what fp32 sums add is far below 2^-12
    _close(y, want, (2.1 * HALF_STEP[dtype] + (dim + hidden + 64) * 4 * EPS) * size, "y")


def test_mixture_captured_replayed_and_on_another_stream(bz):
    import torch
    T, dim, hidden, experts, k = 70, 64, 48, 8, 2
    gate, w1, b1, w2, b2, x = _mixture_inputs(bz, T, dim, hidden, experts, "bf16")
    wants = []
    for seed in range(3):
        x.copy_(_normal(100 + seed, (T, dim), 1.0, "bf16"))
        wants.append(_mixture(bz, x, gate, w1, b1, w2, b2, experts, k)[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    y = _mixture(bz, x, gate, w1, b1, w2, b2, experts, k, stream=side)[1]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, wants[2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _mixture(bz, x, gate, w1, b1, w2, b2, experts, k)[1]
    for turn in range(4):
        x.copy_(_normal(100 + turn % 3, (T, dim), 1.0, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, wants[turn % 3]), "replay %d" % turn
        assert torch.equal(_mixture(bz, x, gate, w1, b1, w2, b2, experts, k)[1], wants[turn % 3])


def test_sort_of_many_entries_and_adapters_captured_and_replayed(bz):
    import torch
    ids = torch.from_numpy(np.random.default_rng(0).integers(-1, 50, 30000).astype(np.int32)).cuda()
    m, n, k = 40, 64, 96
    a, w = _normal(0, (m, k), 1.0, "f16"), _normal(1, (n, k), 0.1, "f16")
    down, up = _normal(2, (5, 8, k), 0.1, "f16"), _normal(3, (5, n, 8), 0.3, "f16")
    own = torch.arange(m, device="cuda", dtype=torch.int32) % 6 - 1
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        offsets, order, position = bz.group_rows(ids, 50)
        y = bz.fc_adapters(a, w, k, down, up, own)
    for turn in range(3):
        ids.copy_(torch.from_numpy(np.random.default_rng(turn).integers(-1, 50, 30000).astype(np.int32)))
        own.copy_(torch.roll(own, 1))
        graph.replay()
        torch.cuda.synchronize()
        want = bz.group_rows(ids, 50)
        kept = int(want[0][-1])
        assert torch.equal(offsets, want[0]) and torch.equal(order[:kept], want[1][:kept]) and torch.equal(position, want[2])
        assert torch.equal(y, bz.fc_adapters(a, w, k, down, up, own))


def _far(rows, cols, pitch, dtype, fill):
    """a matrix whose rows are so far apart that offsets pass 32 bits"""
    import torch
    whole = torch.empty((rows - 1) * pitch + cols, dtype=_t(dtype), device="cuda")
    far = whole.as_strided((rows, cols), (pitch, 1))
    far.copy_(fill)
    return far


@pytest.mark.parametrize("k", [64, 65])
@pytest.mark.parametrize("m", [60, 2100])
def test_layers_of_operands_beyond_4_gb(bz, m, k):
    """a layer is the same with all of its operands spread over more than 2^32 bytes, up to the order of its sums"""
    import torch
    n, groups, rank = 320, 3, 8
    a, w, b = _normal(0, (m, k), 1.0, "bf16"), _normal(1, (n, k), 0.1, "bf16"), _normal(2, (n, ), 0.1)
    far_a = _far(m, k, 2**31 // (m - 1) // 8 * 8 + 4096, "bf16", a)
    far_w = _far(n, k, 2**31 // (n - 1) // 8 * 8 + 4096, "bf16", w)
    far_y = _far(m, n, 2**31 // (m - 1) + 4097, "bf16", torch.zeros((m, n), dtype=torch.bfloat16, device="cuda"))
    v = a.double() @ w.double().t() + b.double()
    bar = (k + 8) * EPS * (a.double().abs() @ w.double().abs().t() + b.double().abs())
    rows = torch.arange(m - 1, -1, -1, dtype=torch.int32, device="cuda")
    bz.grouped_fc(far_a, far_w[None], torch.tensor([0, m], dtype=torch.int32, device="cuda"), k, rows=rows, bias=b[None].contiguous(), out=far_y)
    _close(far_y, v.flip(0), HALF_STEP["bf16"] * (v.flip(0).abs() + bar.flip(0)) + bar.flip(0), "one group")
    del far_w
    stack = torch.empty((groups - 1) * 2**30 + n * k, dtype=torch.bfloat16, device="cuda").as_strided((groups, n, k), (2**30, k, 1))
    stack.copy_(w[None] * torch.tensor([1.0, 2.0, 0.5], dtype=torch.bfloat16, device="cuda")[:, None, None])
    cuts = [0, m // 4, m // 2, m]
    y = bz.grouped_fc(far_a, stack, torch.tensor(cuts, dtype=torch.int32, device="cuda"), k)
    for g, times in enumerate((1.0, 2.0, 0.5)):
        part = slice(cuts[g], cuts[g + 1])
        want, off = (v[part] - b.double()) * times, bar[part] * times
        _close(y[part], want, HALF_STEP["bf16"] * (want.abs() + off) + off, "group %d" % g)
    del stack
    down = torch.empty(2 * 2**30 + rank * k, dtype=torch.bfloat16, device="cuda").as_strided((3, rank, k), (2**30, k, 1))
    up = torch.empty(2 * 2**30 + n * rank, dtype=torch.bfloat16, device="cuda").as_strided((3, n, rank), (2**30, rank, 1))
    down.copy_(_normal(3, (3, rank, k), 0.1, "bf16"))
    up.copy_(_normal(4, (3, n, rank), 0.3, "bf16"))
    ids = torch.arange(m, dtype=torch.int32, device="cuda") % 4
    near = bz.fc_adapters(a, w, k, down.contiguous(), up.contiguous(), ids, bias=b, out_dtype=bz.F32)
    far = bz.fc_adapters(far_a, w, k, down, up, ids, bias=b, out_dtype=bz.F32)
    size = torch.zeros_like(v)
    for g in range(3):
        size[ids == g] = (a[ids == g].double().abs() @ down[g].double().abs().t()) @ up[g].double().abs().t()
    # sums in another order, and a factor's lowest bits with them
    _close(far, near.double(), 2 * bar + 2 * (2.0**-16 + (k + 3 * rank + 16) * EPS) * size, "adapters")


def test_rows_beyond_2_to_the_31_elements_move_and_come_back(bz):
    import torch
    rows, k, groups, dim = 300, 2, 5, 100
    pitch = 2**31 // (rows * k - 1) + 4099
    ids = torch.from_numpy(np.random.default_rng(0).integers(-1, groups, (rows, k)).astype(np.int32)).cuda()
    x, w = _normal(1, (rows, dim), 1.0, "f16"), _normal(2, (rows, k))
    zeros = torch.zeros((rows * k, dim), dtype=torch.float16, device="cuda")
    far = _far(rows * k, dim, pitch, "f16", zeros)
    far_x = _far(rows, dim, 2 * pitch, "f16", x)
    offsets, order, position, xs = bz.group_rows(ids, groups, x=x, out=zeros)
    assert torch.equal(bz.group_rows(ids, groups, x=far_x, out=far)[3], xs)
    assert torch.equal(bz.merge_rows(far, position, w, out=far_x), bz.merge_rows(xs, position, w))
    dxs, dw = bz.merge_rows_grad(x, xs, position, w)
    far_dxs, far_dw = bz.merge_rows_grad(far_x.copy_(x), far, position, w, dxs=far)
    assert torch.equal(dw, far_dw)
    there = torch.zeros(rows * k, dtype=torch.bool, device="cuda")
    there[position[position >= 0].long()] = True
    assert torch.equal(far_dxs[there], dxs[there])


def test_two_graphs_and_two_streams_at_once(bz):
    """calls keep nothing: replays of two graphs and eager calls run beside each other"""
    import torch
    T, dim, hidden, experts, k = 600, 64, 48, 8, 2
    graphs, outs, wants, xs = [], [], [], []
    for seed in range(2):
        gate, w1, b1, w2, b2, x = _mixture_inputs(bz, T, dim, hidden, experts, "f16")
        x.copy_(_normal(200 + seed, (T, dim), 1.0, "f16"))
        wants.append(_mixture(bz, x, gate, w1, b1, w2, b2, experts, k)[1])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = _mixture(bz, x, gate, w1, b1, w2, b2, experts, k)[1]
        graphs.append(graph), outs.append(y), xs.append((gate, w1, b1, w2, b2, x))
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for y in outs:
            y.zero_()
        torch.cuda.synchronize()
        for graph, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                graph.replay()
        gate, w1, b1, w2, b2, x = xs[turn % 2]
        eager = _mixture(bz, x, gate, w1, b1, w2, b2, experts, k)[1]
        torch.cuda.synchronize()
        assert torch.equal(outs[0], wants[0]) and torch.equal(outs[1], wants[1]) and torch.equal(eager, wants[turn % 2])


def test_tensors_that_do_not_fit_are_refused(bz):
    import torch
    with pytest.raises(bz.BlazeHipError, match="not on a GPU"):
        bz.route_topk(torch.zeros((2, 4)), 1)
    with pytest.raises(bz.BlazeHipError, match="not on a GPU"):
        bz.group_rows(torch.zeros(4, dtype=torch.int32, device="cuda"), 2, x=torch.zeros((4, 2)))
    with pytest.raises(bz.BlazeHipError, match="int32"):
        bz.group_rows(torch.zeros(4, dtype=torch.int64, device="cuda"), 2)
    with pytest.raises(bz.BlazeHipError, match="contiguous rows"):
        bz.route_topk(_normal(0, (8, 8)).t(), 2)
    with pytest.raises(bz.BlazeHipError, match=r"\(16, 4\)"):
        bz.group_rows(torch.zeros(16, dtype=torch.int32, device="cuda"), 2, x=_normal(0, (8, 4)), out=_normal(0, (8, 4)))
    with pytest.raises(bz.BlazeHipError, match="act_params"):
        bz.grouped_fc(_normal(0, (4, 8)), _normal(1, (2, 6, 8)), torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"), 8, act=bz.ACT_PRELU,
                      act_params=(_normal(2, (2, 5)), ))


# ---------------------------------------------------------------------------------------------- rows of zeros
# (rows, columns, K, groups, elements between rows of w beyond K): the kernel for few rows, both kinds of the one for rows that begin anywhere, the one for
# many rows
ZERO_ROWS = [(40, 24, 64, 3, 0), (4096, 1024, 64, 8, 0), (3000, 700, 72, 3, 1), (2500, 1000, 45, 2, 0)]


@pytest.mark.parametrize("m,n,k,groups,pad", ZERO_ROWS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "sigmoid", "swiglu"])
@pytest.mark.parametrize("bias", [True, False])
def test_grouped_fc_of_no_rows_at_all(bz, m, n, k, groups, pad, dtype, act, bias):
    """an `a` of no rows: every row number is outside, and every row is one of zeros"""
    import torch
    print("case", m, n, k, groups, pad, dtype, act, bias, flush=True)
    cols = 2 * n if act == "swiglu" else n
    w = _pitched(_normal(1, (groups, cols, k), 1.0, dtype), pad, float("nan"))
    b = _normal(2, (groups, cols)) if bias else None
    cuts = torch.tensor([m * g // groups for g in range(groups + 1)], dtype=torch.int32, device="cuda")
    rows = torch.arange(m, dtype=torch.int32, device="cuda")
    code = {"none": bz.ACT_NONE, "sigmoid": bz.ACT_SIGMOID, "swiglu": bz.ACT_SWIGLU}[act]
    y = bz.grouped_fc(torch.empty((0, k), dtype=w.dtype, device="cuda"), w, cuts, k, rows=rows, rows_per=2, bias=b, act=code)
    v = b.double() if bias else torch.zeros((groups, cols), dtype=torch.float64, device="cuda")
    f = {"none": lambda v: v, "sigmoid": torch.sigmoid, "swiglu": lambda v: v[:, :n] * torch.sigmoid(v[:, :n]) * v[:, n:]}[act]
    want = f(v).repeat_interleave(cuts[1:].long() - cuts[:-1].long(), 0)
    _close(y, want, (HALF_STEP[dtype] + 32 * EPS) * want.abs() + (2.0**-25 if dtype == "f16" else 0.0), "y")


def test_dice_of_one_parameter_a_group_is_refused(bz):
    """where a parameter a column is read"""
    import torch
    a, w, cuts = _normal(0, (4, 8)), _normal(1, (2, 6, 8)), torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    one, full = torch.ones((2, 1), device="cuda"), torch.ones((2, 6), device="cuda")
    with pytest.raises(bz.BlazeHipError, match="act_params"):
        bz.grouped_fc(a, w, cuts, 8, act=bz.ACT_DICE, act_params=(one, full, full))
    with pytest.raises(bz.BlazeHipError, match="act_params"):
        bz.fc_adapters(a, w[0], 8, _normal(2, (1, 3, 8)), _normal(3, (1, 6, 3)), torch.zeros(4, dtype=torch.int32, device="cuda"), act=bz.ACT_DICE,
                       act_params=(one[0], full[0], full[0]))


@pytest.mark.parametrize("m,n,k,groups,pad", ZERO_ROWS)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("per", [1, 2, 3])
def test_grouped_fc_row_numbers_outside_are_rows_of_zeros(bz, m, n, k, groups, pad, dtype, act, per):
    """-1, as a list is padded, and every other number below 0 or behind the last: as if `a` had a row of zeros there"""
    import torch
    print("case", m, n, k, groups, pad, dtype, act, per, flush=True)
    source = 50
    cols = 2 * n if act == "swiglu" else n
    a, w, b = _normal(1, (source, k), 1.0, dtype), _pitched(_normal(2, (groups, cols, k), k**-0.5, dtype), pad, 0.0), _normal(3, (groups, cols), 0.1)
    cuts = torch.tensor([m * g // groups for g in range(groups + 1)], dtype=torch.int32, device="cuda")
    rng = np.random.default_rng(m + per)
    rows = rng.integers(0, source * per, m).astype(np.int32)
    outside = np.arange(m) % 3 == 1
    rows[outside] = rng.choice([-1, 1 - per, -per, -per - 1, -1000, -2**31, source * per, source * per + per - 1, 2**31 - 1], outside.sum())
    rows[outside & (rows == 0)] = -1  # (1 - per of one entry a row)
    spare = torch.cat([a, torch.zeros((1, k), dtype=a.dtype, device="cuda")])
    inside = torch.from_numpy(np.where(outside, source * per, rows).astype(np.int32)).cuda()
    code = bz.ACT_SWIGLU if act == "swiglu" else bz.ACT_NONE
    got = bz.grouped_fc(a, w, cuts, k, rows=torch.from_numpy(rows).cuda(), rows_per=per, bias=b, act=code)
    want = bz.grouped_fc(spare, w, cuts, k, rows=inside, rows_per=per, bias=b, act=code)
    assert torch.equal(got, want)
    v = b.double().repeat_interleave(cuts[1:].long() - cuts[:-1].long(), 0)[torch.from_numpy(outside).cuda()]
    zero = v[:, :n] * torch.sigmoid(v[:, :n]) * v[:, n:] if act == "swiglu" else v
    _close(got[torch.from_numpy(outside).cuda()], zero, (HALF_STEP[dtype] + 32 * EPS) * zero.abs() + (2.0**-25 if dtype == "f16" else 0.0), "rows of zeros")


# ---------------------------------------------------------------------------------------------- activations over all of their range
def _values(dtype):
    """pre-activations over the range that any type has: small, large, either sign"""
    v = [0.0, 1.0, -1.0, 0.25, 8.0, -8.0, 20.0, -20.0, 60.0, -60.0, 88.0, -88.0, 88.75, -88.75, 89.0, 100.0, -100.0, 104.0, 300.0, -300.0, 5e3, -5e3, 6e4, -6e4]
    return v + ([1e30, -1e30, 3e38, -3e38] if dtype != "f16" else []) + [float("inf"), float("-inf"), float("nan")]


# (rows, elements between rows of w beyond K) at N 1100, K 64: the kernel for few rows, the one for rows that begin anywhere, the one for many rows
BY_KERNEL = [(20, 0), (3000, 1), (3000, 0)]


def _spread(bz, m, pad, dtype, groups, n=1100, k=64):
    """an `a` and a `w` whose products are exactly the values of _values, one a row: (a, w, cuts, v [m, n] in 64 bits)"""
    import torch
    values = torch.tensor(_values(dtype), dtype=torch.float64, device="cuda").to(_t(dtype))
    a = torch.zeros((m, k), dtype=_t(dtype), device="cuda")
    at = torch.arange(m, device="cuda") % values.numel()
    a[:, 5] = values[at]
    w = torch.zeros((groups, n, k), dtype=_t(dtype), device="cuda")
    w[:, :, 5] = 1.0
    cuts = torch.tensor([m * g // groups for g in range(groups + 1)], dtype=torch.int32, device="cuda")
    return a, _pitched(w, pad, 0.0), cuts, values[at].double()[:, None].expand(m, n)


@pytest.mark.parametrize("m,pad", BY_KERNEL)
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
def test_sigmoid_layers_over_their_range(bz, m, pad, dtype, out):
    """every pre-activation has its sigmoid, infinities among them"""
    import torch
    code = {"f32": bz.F32, "f16": bz.F16, "bf16": bz.BF16}[out]
    a, w, cuts, v = _spread(bz, m, pad, dtype, 3)
    some = torch.isfinite(v)
    want = torch.sigmoid(v)
    # exp of an exact argument, a sum and a division, rounded once; what is below 2^-126 may be flushed
    bar = (HALF_STEP[out] + 16 * EPS) * want.nan_to_num(0.0) + (2.0**-25 if out == "f16" else 2.0**-126)
    y = bz.grouped_fc(a, w, cuts, 64, act=bz.ACT_SIGMOID, out_dtype=code)
    _close(y, want, bar, "grouped")
    z = bz.fc_adapters(a, w[0], 64, torch.zeros((2, 8, 64), dtype=a.dtype, device="cuda"), torch.zeros((2, 1100, 8), dtype=a.dtype, device="cuda"),
                       (torch.arange(m, device="cuda") % 3 - 1).to(torch.int32), act=bz.ACT_SIGMOID, out_dtype=code)
    _close(z[some], want[some], bar[some], "adapters")  # (an infinity times down's zeros is none of them)


@pytest.mark.parametrize("m,pad", BY_KERNEL)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_sigmoid_layers_of_infinite_sums(bz, m, pad, dtype):
    """a bias of either infinity is an infinite pre-activation, whose sigmoid is 1 or 0"""
    import torch
    a, w, cuts, _ = _spread(bz, m, pad, dtype, 2)
    a.fill_(0.5)
    bias = torch.zeros((2, 1100), device="cuda")
    bias[0, ::2], bias[1, ::3] = float("inf"), float("-inf")
    y = bz.grouped_fc(a, w, cuts, 64, bias=bias, act=bz.ACT_SIGMOID)
    half = torch.sigmoid(torch.tensor(0.5, dtype=torch.float64)).item()
    cut = int(cuts[1])
    want = torch.full((m, 1100), half, dtype=torch.float64, device="cuda")
    want[:cut, ::2], want[cut:, ::3] = 1.0, 0.0
    _close(y, want, (HALF_STEP[dtype] + 16 * EPS) * want, "y")


@pytest.mark.parametrize("m,pad", BY_KERNEL)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("slope", [0.0, 0.25])
def test_relu_layers_over_their_range(bz, m, pad, dtype, slope):
    """-infinity is 0 with a slope of 0, and a NaN stays one"""
    import torch
    a, w, cuts, v = _spread(bz, m, pad, dtype, 3)
    y = bz.grouped_fc(a, w, cuts, 64, act=bz.ACT_LEAKY_RELU, act_alpha=slope)
    want = torch.where(v >= 0, v, torch.nan_to_num(slope * v, nan=0.0, neginf=-float("inf")))
    want = torch.where(torch.isnan(v), v, want)
    _close(y, want, (HALF_STEP[dtype] + EPS) * want.nan_to_num(0.0, 0.0, 0.0).abs(), "y")
    bias = torch.zeros((3, 1100), device="cuda")
    bias[:, ::2] = -float("inf")
    a.fill_(0.5)
    z = bz.grouped_fc(a, w, cuts, 64, bias=bias, act=bz.ACT_LEAKY_RELU, act_alpha=slope)
    assert bool((z[:, ::2] == (0.0 if slope == 0 else -float("inf"))).all()) and bool((z[:, 1::2] == 0.5).all())
    ids = (torch.arange(m, device="cuda") % 3 - 1).to(torch.int32)
    z = bz.fc_adapters(a, w[0], 64, torch.zeros((2, 8, 64), dtype=a.dtype, device="cuda"), torch.zeros((2, 1100, 8), dtype=a.dtype, device="cuda"), ids,
                       bias=bias[0].contiguous(), act=bz.ACT_LEAKY_RELU, act_alpha=slope)
    assert bool((z[:, ::2] == (0.0 if slope == 0 else -float("inf"))).all()) and bool((z[:, 1::2] == 0.5).all())


@pytest.mark.parametrize("m,pad", BY_KERNEL)
@pytest.mark.parametrize("nosqrt", [True, False])
def test_fp32_dice_far_from_its_mean(bz, m, pad, nosqrt):
    """Far below the mean Dice is e^(v - mean) v and little else: pre-activations that are exact, a deviation of 1, so that what is off
    is the activation's own arithmetic.  Rounded: v - mean and its quotient not at all (small whole numbers and quarters over 1), exp by 2 steps,
    1 + t, 1 / that, two products and a sum by one each; 16 steps in all."""
    import torch
    n, k, groups = 1100, 64, 2
    a = torch.zeros((m, k), device="cuda")
    a[:, 9] = -(torch.arange(m, device="cuda") % 280) / 4.0
    w = torch.zeros((groups, n, k), device="cuda")
    w[:, :, 9] = 1.0
    cuts = torch.tensor([0, m // 3, m], dtype=torch.int32, device="cuda")
    gamma, mean, var = torch.zeros((groups, n), device="cuda"), torch.full((groups, n), 2.0, device="cuda"), torch.ones((groups, n), device="cuda")
    y = bz.grouped_fc(a, _pitched(w, pad, 0.0), cuts, k, act=bz.ACT_DICE, act_params=(gamma, mean, var), dice_nosqrt=nosqrt)
    v = a[:, 9].double()[:, None].expand(m, n)
    want = torch.sigmoid(v - 2.0) * v  # (sqrt(1 + 1e-8) is 1 in fp32)
    _close(y, want, 16 * EPS * want.abs(), "grouped")
    z = bz.fc_adapters(a, _pitched(w, pad, 0.0)[0], k, torch.zeros((1, 4, k), device="cuda"), torch.zeros((1, n, 4), device="cuda"),
                       torch.zeros(m, dtype=torch.int32, device="cuda"), act=bz.ACT_DICE, act_params=(gamma[0], mean[0], var[0]), dice_nosqrt=nosqrt)
    _close(z, want, 16 * EPS * want.abs(), "adapters")


@pytest.mark.parametrize("m,pad", BY_KERNEL)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_dice_of_infinite_sums(bz, m, pad, dtype):
    """v above, gamma * v below: infinities where those are"""
    import torch
    n, k, groups = 1100, 64, 2
    a, w = torch.full((m, k), 0.5, dtype=_t(dtype), device="cuda"), torch.zeros((groups, n, k), dtype=_t(dtype), device="cuda")
    bias = torch.zeros((groups, n), device="cuda")
    bias[:, ::3], bias[:, 1::3] = float("inf"), -float("inf")
    params = torch.full((groups, n), 0.5, device="cuda"), torch.zeros((groups, n), device="cuda"), torch.ones((groups, n), device="cuda")
    cuts = torch.tensor([0, m // 3, m], dtype=torch.int32, device="cuda")
    y = bz.grouped_fc(a, _pitched(w, pad, 0.0), cuts, k, bias=bias, act=bz.ACT_DICE, act_params=params)
    assert bool((y[:, ::3] == float("inf")).all()) and bool((y[:, 1::3] == -float("inf")).all()) and bool((y[:, 2::3] == 0).all())


@pytest.mark.parametrize("scale_a,scale_w", [(2.0**-124, 1.0), (2.0**-124, 2.0**20), (2.0**-124, 2.0**60), (2.0**-118, 2.0**60), (2.0**-124, 2.0**110), (2.0**60, 2.0**-124),
                                             (2.0**20, 2.0**-124), (2.0**-60, 2.0**-50), (1.0, 2.0**-120)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k,groups", [(2500, 700, 200, 3), (30, 700, 200, 3)])
def test_grouped_fc_fp32_of_very_small_operands(bz, scale_a, scale_w, gated, m, n, k, groups):
    """Some rows so small that a split in pieces drops bits of them, beside ordinary ones, in long batches and short ones: fp32 sums like any
    other, (K + 8) * 2^-24 of their terms, and 2^-126 for what may be flushed of each product."""
    import torch
    cols = 2 * n if gated else n
    small = torch.arange(m, device="cuda") % 5 == 2
    a, w = _normal(0, (m, k)), _normal(1, (groups, cols, k), 1.0 / np.sqrt(k))
    small_cols = torch.arange(cols, device="cuda") % 7 == 3
    # (1 and more, so that no operand is below 2^-126 itself)
    a[small] = torch.sign(a[small]) * (1.0 + a[small].abs()) * scale_a
    w[:, small_cols] = torch.sign(w[:, small_cols]) * (1.0 + w[:, small_cols].abs()) * scale_w
    cuts = torch.tensor([m * g // groups for g in range(groups + 1)], dtype=torch.int32, device="cuda")
    if gated:  # up: the gate is one half of a row's first input, so that silu(gate) * up is linear in up
        a[:, 0] = 2.0
        w[:, :n] = 0.0
        w[:, :n, 0] = 0.5  # gate 1 in every row
        w[:, n:, 0] = 0.0
        y = bz.grouped_fc(a, w, cuts, k, act=bz.ACT_SWIGLU).double()
        factor = float(torch.sigmoid(torch.tensor(1.0, dtype=torch.float64)))
        w = w[:, n:]
    else:
        y, factor = bz.grouped_fc(a, w, cuts, k).double(), 1.0
    for g in range(groups):
        lo, hi = int(cuts[g]), int(cuts[g + 1])
        x, v = a[lo:hi].double(), w[g].double()
        want, size = x @ v.t(), x.abs() @ v.abs().t()
        _close(y[lo:hi], factor * want, factor * ((k + 8) * EPS * size + k * 2.0**-126) + 32 * EPS * want.abs(), "group %d" % g)


def test_fc_adapters_fp32_of_very_small_operands(bz):
    import torch
    m, n, k, rank = 2500, 1000, 200, 8
    a, w = _normal(0, (m, k)), _normal(1, (n, k), 2.0**20 / np.sqrt(k))
    a[::5] = torch.sign(a[::5]) * (1.0 + a[::5].abs()) * 2.0**-124
    down, up = _normal(2, (2, rank, k), 2.0**20 / np.sqrt(k)), _normal(3, (2, n, rank))
    ids = (torch.arange(m, device="cuda") % 3 - 1).to(torch.int32)
    y = bz.fc_adapters(a, w, k, down, up, ids)
    x = a.double()
    want, size = x @ w.double().t(), x.abs() @ w.double().abs().t()
    for g in range(2):
        r = ids == g
        want[r] += (x[r] @ down[g].double().t()) @ up[g].double().t()
        size[r] += (x[r].abs() @ down[g].double().abs().t()) @ up[g].double().abs().t()
    _close(y, want, (k + 3 * rank + 24) * EPS * size + (k + rank) * 2.0**-126 * 2.0**4, "y")


def test_grouped_fc_fp32_results_do_not_depend_on_a_row_of_zeros_or_large_ones(bz):
    """rows beside rows of zeros, of very large numbers and of infinities are bit for bit what they are without them"""
    import torch
    m, n, k = 2500, 700, 200
    a, w = _normal(0, (m, k)), _normal(1, (2, n, k), 1.0 / np.sqrt(k))
    cuts = torch.tensor([0, 1000, m], dtype=torch.int32, device="cuda")
    a[::3] *= 2.0**-60
    want = bz.grouped_fc(a, w, cuts, k)
    other = torch.arange(m, device="cuda") % 64 == 17
    for value in (0.0, 1e30, float("inf")):
        b = a.clone()
        b[other] = value
        assert torch.equal(bz.grouped_fc(b, w, cuts, k)[~other], want[~other])


# ---------------------------------------------------------------------------------------------- adapters of infinities
def _bounds_case(bz, m, pad, dtype, rank, adapters, n=700, k=64):
    """positive operands of an adapter layer, so that no infinity meets another one's opposite; w at another pitch by `pad`"""
    import torch
    a, w = _normal(0, (m, k), 1.0, dtype).abs() + 0.25, _normal(1, (n, k), k**-0.5, dtype).abs()
    down, up = _normal(2, (adapters, rank, k), k**-0.5, dtype).abs() + 2.0**-6, _normal(3, (adapters, n, rank), rank**-0.5, dtype).abs() + 2.0**-6
    return a, _pitched(w, pad, 0.0), down, up


def _adapters_want(a, w, down, up, ids):
    """in 64 bits, a product and a sum at a time, so that what is no number comes as it does by IEEE"""
    import torch
    y = (a.double()[:, None, :] * w.double()[None]).sum(2)
    for g in range(down.shape[0]):
        r = torch.nonzero(ids == g)[:, 0]
        if r.numel():
            low = (a[r].double()[:, None, :] * down[g].double()[None]).sum(2)
            y[r] += (low[:, None, :] * up[g].double()[None]).sum(2)
    return y


@pytest.mark.parametrize("m,pad", [(20, 0), (900, 1), (900, 0)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rank", [16, 32, 48])
def test_fc_adapters_of_infinite_weights(bz, m, pad, dtype, rank):
    """an infinity of either sign in `up` is one in the rows of its adapter, and one in a row's factor is one there: no NaNs"""
    import torch
    print("case", m, pad, dtype, rank, flush=True)
    inf = float("inf")
    a, w, down, up = _bounds_case(bz, m, pad, dtype, rank, 3)
    ids = (torch.arange(m, device="cuda") // 7 % 4 - 1).to(torch.int32)
    up[0, 5, 3], up[1, 6, rank - 1], up[2, 650, 0], up[2, 651, 9] = inf, -inf, inf, float("nan")
    want = _adapters_want(a, w, down, up, ids)
    got = bz.fc_adapters(a, w, 64, down, up, ids).double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and int(torch.isnan(want).sum()) == int((ids == 2).sum())
    far = torch.isinf(want)
    assert int(far.sum()) == int((ids >= 0).sum()) and bool((got[far] == want[far]).all())
    near = torch.isfinite(want)
    _close(got[near], want[near], (HALF_STEP[dtype] + 2.0**-15) * want[near].abs(), "finite")  # (all terms are positive)
    # and of rows whose factors are infinite, by the row or by the adapter
    a, w, down, up = _bounds_case(bz, m, pad, dtype, rank, 3)
    a[::11, 7] = inf
    down[1, 4, 9] = inf
    want = _adapters_want(a, w, down, up, ids)
    assert not bool(torch.isnan(want).any()) and bool(torch.isinf(want).any())
    got = bz.fc_adapters(a, w, 64, down, up, ids).double()
    far = torch.isinf(want)
    assert bool((got[far] == want[far]).all())
    _close(got[~far], want[~far], (HALF_STEP[dtype] + 2.0**-15) * want[~far].abs(), "finite")


@pytest.mark.parametrize("m,pad", [(32, 0), (900, 1), (900, 0)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rank", [1, 5, 8, 20, 40])
def test_fc_adapters_of_an_infinite_row_at_any_rank(bz, m, pad, dtype, rank):
    """a row of an infinity, and one of an adapter whose scale is infinite, alone with the adapter in its block or among many rows of it, at ranks
    that are filled up with zeros: infinite, not NaN"""
    import torch
    print("case", m, pad, dtype, rank, flush=True)
    inf = float("inf")
    a, w, down, up = _bounds_case(bz, m, pad, dtype, rank, 3)
    a[3, 7], a[20, 0] = inf, inf
    alone = torch.zeros(m, dtype=torch.int32, device="cuda")  # (adapter 0, and in the first block one row each of 1 and 2)
    alone[3], alone[20] = 1, 2
    among = torch.ones(m, dtype=torch.int32, device="cuda")
    scale = torch.tensor([1.0, 0.5, inf], device="cuda")
    for ids in (alone, among):
        y = bz.fc_adapters(a, w, 64, down, up, ids, scale=scale)
        assert bool((y[3] == inf).all()) and bool((y[20] == inf).all())
        rest = torch.arange(m, device="cuda") % 32
        rest = (rest != 3) & (rest != 20)
        assert bool(torch.isfinite(y[rest]).all())
    many = torch.full((m, ), 2, dtype=torch.int32, device="cuda")
    y = bz.fc_adapters(a, w, 64, down, up, many, scale=scale)
    assert bool((y == inf).all())


@pytest.mark.parametrize("m", [20, 900])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("together", [False, True])
def test_fc_adapters_of_the_largest_finite_factor(bz, m, dtype, together):
    """a factor next to the largest float, which a bf16 rounds to infinity: its product with a small weight is finite"""
    import torch
    n, k, rank = 700, 64, 16
    a, down, up = (torch.zeros(s, dtype=_t(dtype), device="cuda") for s in ((m, k), (m, rank, k), (m, n, rank)))
    a[:, 0], down[:, 0, 0], up[:, :, 0] = 1.0, 1.0, 2.0**-14
    w = torch.zeros((n, k), dtype=a.dtype, device="cuda")
    ids = torch.zeros(m, dtype=torch.int32, device="cuda") if together else torch.arange(m, dtype=torch.int32, device="cuda")
    for value in (3.4e38, -3.4e38, 3.3961775292304957e38, float(torch.finfo(torch.float32).max)):
        y = bz.fc_adapters(a, w, k, down, up, ids, scale=torch.full((m, ), value, device="cuda"), out_dtype=bz.F32)
        want = torch.full((m, n), value, dtype=torch.float32, device="cuda").double() * 2.0**-14
        _close(y, want, 2.0**-16 * want.abs(), "%g" % value)


# ---------------------------------------------------------------------------------------------- more than 2^32 threads' worth of rows
@pytest.mark.parametrize("rows,n", [(2**28 + 77, 2), (2**26 + 5, 129)])
def test_route_topk_of_more_rows_than_a_launch_has_threads_for(bz, rows, n):
    import torch
    logits = torch.empty((rows, n), dtype=torch.float16, device="cuda").normal_()
    ids, w = bz.route_topk(logits, 1, renormalize=True)
    assert bool((w == 1).all())
    for at in (0, rows // 2 - 500, 2**25 - 500, 2**27 - 500, rows - 1000):
        part = logits[at:at + 1000].float()
        if part.shape[0]:
            first = (part == part.amax(1, keepdim=True)).int().argmax(1)
            assert torch.equal(ids[at:at + part.shape[0], 0].long(), first), at
    del logits, ids, w
    torch.cuda.empty_cache()


def test_merge_gradient_of_more_rows_than_a_launch_has_threads_for(bz):
    import torch
    rows, dim = 2**26 + 3, 8
    dy, xs = (torch.empty((rows, dim), dtype=torch.float16, device="cuda").normal_() for _ in range(2))
    position = torch.arange(rows - 1, -1, -1, dtype=torch.int32, device="cuda")[:, None].contiguous()
    w = torch.empty((rows, 1), device="cuda").normal_()
    dxs, dw = bz.merge_rows_grad(dy, xs, position, w, dxs=torch.empty_like(xs))
    for at in (0, 2**25 - 500, rows - 1000):
        t = slice(at, at + 1000)
        to = position[t, 0].long()
        want = (w[t].double() * dy[t].double())
        _close(dxs[to], want, (HALF_STEP["f16"] + EPS) * want.abs() * (1 + 2.0**-8) + 2.0**-25, "dxs from %d" % at)
        products = dy[t].double() * xs[to].double()
        _close(dw[t, 0], products.sum(1), (dim + 4) * EPS * products.abs().sum(1), "dweights from %d" % at)
    del dy, xs, dxs, dw, w, position
    torch.cuda.empty_cache()


def test_rows_of_more_chunks_than_a_launch_has_threads_move_and_merge(bz):
    import torch
    rows, dim = 2**22 + 1, 8 * 1025
    few = _normal(0, (100, dim), 1.0, "f16")
    position = torch.randint(100, (rows, 1), device="cuda", dtype=torch.int32)
    x = bz.merge_rows(few, position)
    ats = [slice(0, 300), slice(2**31 // 1025 - 100, 2**31 // 1025 + 100), slice(rows - 300, rows)]
    for t in ats:
        assert torch.equal(x[t], few[position[t, 0].long()])
    ids = (torch.arange(rows, device="cuda") % 2).to(torch.int32)[:, None].contiguous()
    offsets, order, to, xs = bz.group_rows(ids, 2, x=x)
    assert offsets.tolist() == [0, rows // 2 + 1, rows]
    for t in ats:
        assert torch.equal(xs[to[t, 0].long()], x[t])
    del x, xs
    torch.cuda.empty_cache()


def test_calls_on_a_stream_of_this_device(bz):
    import torch
    side = torch.cuda.Stream()
    logits = _normal(0, (40, 8))
    want = bz.route_topk(logits, 2)
    side.wait_stream(torch.cuda.current_stream())
    got = bz.route_topk(logits, 2, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = bz.route_topk(logits, 2, stream=torch.cuda.default_stream())
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0])


@pytest.mark.parametrize("m", [20, 900])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rank", [1, 16])
def test_fc_adapters_lose_no_more_than_a_factors_rounding(bz, m, dtype, rank):
    """A factor is two bf16s; its product with `up`, whose numbers two bf16s hold, loses nothing but what fp32 sums lose: four products a
    term and the sums, (4 + 4) * rank steps of the terms."""
    import torch
    n = 700
    a, down = _normal(0, (m, 1), 1.0, dtype), _normal(1, (1, rank, 1), 1.0, dtype)
    up, w = _normal(2, (1, n, rank), 1.0, dtype), torch.zeros((n, 1), dtype=_t(dtype), device="cuda")
    y = bz.fc_adapters(a, w, 1, down, up, torch.zeros(m, dtype=torch.int32, device="cuda"), out_dtype=bz.F32)
    v = a.float() * down[0, :, 0].float()  # (exact: the product of two numbers of 11 bits or fewer)
    hi = v.bfloat16()
    factor = hi.double() + (v - hi.float()).bfloat16().double()
    want, size = factor @ up[0].double().t(), factor.abs() @ up[0].double().abs().t()
    _close(y, want, 8 * rank * EPS * size, "y")
