"""The operators for batches whose rows go through different weights: what is measured of them, and their plain forms.

Five kinds of work, each over the range of sizes that it is used at:

  route     a gate's logits to the k experts of every row and their weights
  sort      the entries (row, expert) in the experts' order, and the rows copied there
  merge     the experts' rows back where they came from, weighted and added up
  merge_grad  that sum's gradient
  experts   every expert's layer on its rows (bias and activation in it), the rows sorted already or picked up where they are
  adapters  a layer shared by all rows, plus the low-rank product that each row's request names
"""
import math
import os
import sys

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # the gate of one request's one row: latency alone
        dict(name="route_f32_one_row", kind="route", dtype="f32", rows=1, experts=8, k=2, score="softmax", renorm=True, masked=0.0, padded=0.0),
        # the gate of a long batch over many experts, some of them out of service, some rows padding
        dict(name="route_bf16_16384", kind="route", dtype="bf16", rows=16384, experts=128, k=8, score="softmax", renorm=True, masked=0.05, padded=0.02),
        # the headline batch and input width, two experts of eight a sample
        dict(name="sort_f16_2048", kind="sort", dtype="f16", rows=2048, experts=8, k=2, dim=896, padded=0.0),
        # a long batch over many experts, some rows padding
        dict(name="sort_bf16_16384", kind="sort", dtype="bf16", rows=16384, experts=128, k=8, dim=2048, padded=0.02),
        # the results of a few hundred candidates, rows of an odd width
        dict(name="merge_f32_300", kind="merge", dtype="f32", rows=300, experts=16, k=4, dim=445, padded=0.0),
        # the gradient of a long batch's results
        dict(name="merge_grad_bf16_8192", kind="merge_grad", dtype="bf16", rows=8192, experts=64, k=8, dim=2048, padded=0.02),
        # the headline batch through eight experts in fp32, the engine's default type
        dict(name="experts_f32_2048", kind="experts", dtype="f32", rows=2048, experts=8, k=2, dim=896, n=512, act="prelu", gather=True),
        # few rows and much weight: a serving step of 64 rows through sixteen gated experts
        dict(name="experts_bf16_64", kind="experts", dtype="bf16", rows=64, experts=16, k=4, dim=2048, n=1024, act="swiglu", gather=True),
        # the largest: a long batch through thirty-two gated experts
        dict(name="experts_bf16_8192", kind="experts", dtype="bf16", rows=8192, experts=32, k=4, dim=2048, n=1024, act="swiglu", gather=True),
        # thirty-two requests of one row each, every one with an adapter of its own
        dict(name="adapters_bf16_32", kind="adapters", dtype="bf16", rows=32, requests=32, adapters=64, rank=16, dim=2048, n=2048, act="none", none=0.0),
        # the headline batch and first layer, a few requests' candidates with their customers' adapters
        dict(name="adapters_f16_2048", kind="adapters", dtype="f16", rows=2048, requests=12, adapters=40, rank=8, dim=896, n=512, act="prelu", none=0.2),
        # a long batch of long requests through a wide layer
        dict(name="adapters_bf16_8192", kind="adapters", dtype="bf16", rows=8192, requests=24, adapters=32, rank=32, dim=4096, n=4096, act="none", none=0.1),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "sort", "merge", "merge_grad", "experts", "experts", "adapters", "adapters"])
    dtype = rng.choice(["f16", "bf16", "f32"])
    es = SIZE[dtype]
    experts = rng.choice([4, 6, 8, 16, 16, 32, 60, 64, 128])
    k = rng.randint(1, min(8, experts))
    padded = rng.choice([0.0, 0.0, 0.03])
    if kind == "route":
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, 16384), experts=experts, k=k, score=rng.choice(["softmax", "softmax", "sigmoid"]),
                    renorm=rng.random() < 0.6, masked=rng.choice([0.0, 0.05]), padded=padded)
    if kind in ("sort", "merge", "merge_grad"):
        dim = _log(rng, 32, 4096)
        if rng.random() < 0.7:
            dim = (dim + 7) // 8 * 8
        most = (5e8 if kind == "sort" else 2.5e8) / (k * dim * es)
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, max(2, min(16384, int(most)))), experts=experts, k=k, dim=dim, padded=padded)
    dim, n = _log(rng, 64, 4096), _log(rng, 40, 4096)
    if rng.random() < 0.8:
        dim, n = (dim + 7) // 8 * 8, (n + 7) // 8 * 8
    flops = 2e11 if dtype != "f32" else 2e10
    if kind == "experts":
        experts = rng.choice([4, 6, 8, 16, 32, 60])
        k = rng.randint(1, min(6, experts))
        act = rng.choice(["none", "relu", "prelu", "sigmoid", "swiglu", "swiglu"])
        n = min(n, int(2.5e8 / (experts * dim)))
        most = flops / (2.0 * k * dim * n * (2 if act == "swiglu" else 1))
        return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, max(2, min(8192, int(most)))), experts=experts, k=k, dim=dim, n=n, act=act,
                    gather=rng.random() < 0.6)
    rows = _log(rng, 1, max(2, min(8192, int(flops / (2.0 * dim * n)))))
    return dict(kind=kind, dtype=dtype, rows=rows, requests=_log(rng, 1, min(rows, 128)), adapters=rng.randint(1, 48), rank=rng.choice([4, 8, 8, 16, 16, 32, 48, 64]),
                dim=dim, n=n, act=rng.choice(["none", "none", "relu", "prelu", "sigmoid"]), none=rng.choice([0.0, 0.1, 0.5]))


# ---------------------------------------------------------------------------------------------- inputs
def _up8(v):
    return (v + 7) // 8 * 8


def _normal(gen, shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=gen).to(dtype)


def _picks(gen, rows, experts, k):
    """k different experts a row, some chosen more often than others, as a trained gate's are"""
    popular = -0.3 * torch.log(1.0 + torch.randperm(experts, generator=gen, device="cuda").float())
    noise = torch.rand((rows, experts), generator=gen, device="cuda").clamp_(1e-7, 1.0 - 1e-7)
    return torch.sort(popular - torch.log(-torch.log(noise)), dim=1, descending=True, stable=True)[1][:, :k].to(torch.int32).contiguous()


def _pad(gen, ids, share):
    """some rows are padding, which no expert takes"""
    if share:
        ids[torch.rand(ids.shape[0], generator=gen, device="cuda") < share] = -1
    return ids


def _sorted(ids, groups):
    """(offsets, order, position) of the entries in their groups' order; entries of no group come last"""
    flat = ids.reshape(-1).long()
    n = flat.numel()
    key = torch.where((flat >= 0) & (flat < groups), flat, groups)
    key, order = torch.sort(key, stable=True)
    offsets = torch.searchsorted(key, torch.arange(groups + 1, device=key.device))
    at = torch.arange(n, device=key.device)
    position = torch.empty_like(at)
    position[order] = at
    position = torch.where((flat >= 0) & (flat < groups), position, -1).reshape(ids.shape)
    order = torch.where(at < offsets[groups], order, 0)
    return offsets.to(torch.int32), order.to(torch.int32), position.to(torch.int32)


def _packed(gen, shape, k, dtype):
    """weights [..., k] of standard deviation 1 / sqrt(k), rows at a pitch of whole 8 elements, zeros between"""
    w = torch.zeros((*shape, _up8(k)), dtype=dtype, device="cuda")
    for i in range(shape[0]):
        w[i, ..., :k] = _normal(gen, (*shape[1:], k), 1.0 / math.sqrt(k), dtype)
    return w


def prepare(case, seed):
    torch.cuda.set_device(0)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    kind, dt, T = case["kind"], TORCH[case["dtype"]], case["rows"]
    if kind == "route":
        logits = _normal(gen, (T, case["experts"]), 1.5, dt)
        if case["masked"]:
            logits[:, torch.rand(case["experts"], generator=gen, device="cuda") < case["masked"]] = -math.inf
        if case["padded"]:
            logits[torch.rand(T, generator=gen, device="cuda") < case["padded"]] = -math.inf
        st.update(logits=logits, ids=torch.zeros((T, case["k"]), dtype=torch.int32, device="cuda"), weights=torch.zeros((T, case["k"]), device="cuda"))
        return st
    if kind in ("sort", "merge", "merge_grad"):
        k, dim, n = case["k"], case["dim"], T * case["k"]
        ids = _pad(gen, _picks(gen, T, case["experts"], k), case["padded"])
        if kind == "sort":
            st.update(ids=ids, x=_normal(gen, (T, dim), 1.0, dt), offsets=torch.zeros(case["experts"] + 1, dtype=torch.int32, device="cuda"),
                      order=torch.zeros(n, dtype=torch.int32, device="cuda"), position=torch.zeros((T, k), dtype=torch.int32, device="cuda"),
                      xs=torch.zeros((n, dim), dtype=dt, device="cuda"))
            return st
        weights = torch.softmax(_normal(gen, (T, k)), 1)
        st.update(position=_sorted(ids, case["experts"])[2], weights=weights, xs=_normal(gen, (n, dim), 1.0, dt))
        if kind == "merge":
            st.update(y=torch.zeros((T, dim), dtype=dt, device="cuda"))
        else:
            st.update(dy=_normal(gen, (T, dim), 1.0, dt), dxs=torch.zeros((n, dim), dtype=dt, device="cuda"), dw=torch.zeros((T, k), device="cuda"))
        return st
    dim, n = case["dim"], case["n"]
    x = _normal(gen, (T, dim), 1.0, dt)
    if kind == "experts":
        experts, k = case["experts"], case["k"]
        offsets, order, _ = _sorted(_picks(gen, T, experts, k), experts)
        cols = 2 * n if case["act"] == "swiglu" else n
        st.update(x=x if case["gather"] else x[(order // k).long()], offsets=offsets, order=order, w=_packed(gen, (experts, cols), dim, dt),
                  bias=_normal(gen, (experts, cols), 0.1), y=torch.zeros((T * k, n), dtype=dt, device="cuda"))
        if case["act"] == "prelu":
            st.update(slope=torch.empty((experts, n), device="cuda").uniform_(0.1, 0.4, generator=gen))
        return st
    # the rows of a request stand together; requests of one length or another, some without an adapter
    A, R = case["adapters"], case["rank"]
    cuts = torch.sort(torch.randperm(T - 1, generator=gen, device="cuda")[:case["requests"] - 1] + 1)[0] if T > 1 else torch.zeros(0, device="cuda").long()
    request = torch.searchsorted(cuts, torch.arange(T, device="cuda"), right=True)
    adapter = torch.randint(A, (case["requests"], ), generator=gen, device="cuda", dtype=torch.int32)
    if case["requests"] <= A:
        adapter = torch.randperm(A, generator=gen, device="cuda")[:case["requests"]].to(torch.int32)
    adapter[torch.rand(case["requests"], generator=gen, device="cuda") < case["none"]] = -1
    st.update(x=x, w=_packed(gen, (1, n), dim, dt)[0], bias=_normal(gen, (n, ), 0.1), down=_packed(gen, (A, R), dim, dt), up=_packed(gen, (A, n), R, dt),
              scale=torch.empty(A, device="cuda").uniform_(0.25, 2.0, generator=gen), ids=adapter[request].contiguous(),
              y=torch.zeros((T, n), dtype=dt, device="cuda"))
    if case["act"] == "prelu":
        st.update(slope=torch.empty(n, device="cuda").uniform_(0.1, 0.4, generator=gen))
    return st


# ---------------------------------------------------------------------------------------------- the plain forms
def _activated(v, act, slope=None):
    if act == "relu":
        return torch.where(v >= 0, v, torch.zeros_like(v))
    if act == "prelu":
        return torch.where(v > 0, v, v * slope)
    if act == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-v))
    return v


def _plain_route(st):
    l, k = st["logits"].float(), st["k"]
    l = torch.where(torch.isnan(l), -math.inf, l)
    if st["score"] == "softmax":
        m = torch.amax(l, 1, keepdim=True)
        p = torch.where(l == -math.inf, 0.0, torch.exp(l - m))
        total = torch.sum(p, 1, keepdim=True)
        p = torch.where(total > 0, p / total, 0.0)
    else:
        p = 1.0 / (1.0 + torch.exp(-l))
    top, ids = torch.sort(l, dim=1, descending=True, stable=True)
    none = top[:, :k] == -math.inf
    ids = ids[:, :k]
    w = torch.where(none, 0.0, torch.gather(p, 1, ids))
    if st["renorm"]:
        total = torch.sum(w, 1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return torch.where(none, -1, ids).to(torch.int32), w


def _plain_sort(st):
    offsets, order, position = _sorted(st["ids"], st["experts"])
    kept = torch.arange(order.numel(), device=order.device) < offsets[-1]
    xs = torch.where(kept[:, None], st["x"][(order // st["k"]).long()], 0.0)
    return offsets, order, position, xs


def _plain_merge(st):
    position = st["position"]
    rows = st["xs"][position.clamp(min=0).long()].float() * st["weights"][:, :, None]
    return torch.sum(torch.where((position >= 0)[:, :, None], rows, 0.0), 1).to(st["xs"].dtype)


def _plain_merge_grad(st):
    position, dy, xs = st["position"], st["dy"].float(), st["xs"]
    n, dim = xs.shape
    there = position >= 0
    dxs = torch.zeros((n + 1, dim), dtype=xs.dtype, device=xs.device)
    dxs[torch.where(there, position, n).long()] = (st["weights"][:, :, None] * dy[:, None, :]).to(xs.dtype)
    dw = torch.sum(xs[position.clamp(min=0).long()].float() * dy[:, None, :], 2)
    return dxs[:n], torch.where(there, dw, 0.0)


def _plain_experts(st):
    """one product over all experts, each one's rows filled up to the most that any has"""
    dim, n, offsets, order, act = st["dim"], st["n"], st["offsets"].long(), st["order"].long(), st["act"]
    R, experts = order.numel(), offsets.numel() - 1
    at = torch.arange(R, device=order.device)
    expert = torch.searchsorted(offsets, at, right=True) - 1
    slot = at - offsets[expert]
    a = st["x"].float()
    a = a[order // st["k"]] if st["gather"] else a
    filled = torch.zeros((experts, int((offsets[1:] - offsets[:-1]).max()), dim), device=a.device)
    filled[expert, slot] = a
    v = torch.matmul(filled, st["w"][:, :, :dim].float().transpose(1, 2)) + st["bias"][:, None, :]
    if act == "swiglu":
        v = v[:, :, :n] / (1.0 + torch.exp(-v[:, :, :n])) * v[:, :, n:]
    else:
        v = _activated(v, act, st["slope"][:, None, :] if act == "prelu" else None)
    return v[expert, slot].to(st["x"].dtype)


def _plain_adapters(st):
    """both products of every adapter for every row, those of other rows' adapters taken as zero between"""
    dim, R, A, ids = st["dim"], st["rank"], st["adapters"], st["ids"]
    x = st["x"].float()
    low = torch.matmul(x, st["down"][:, :, :dim].float().reshape(A * R, dim).t()).reshape(-1, A, R)
    mine = torch.arange(A, device=ids.device)[None, :] == ids[:, None]
    low = torch.where(mine[:, :, None], low * st["scale"][None, :, None], 0.0).reshape(-1, A * R)
    up = st["up"][:, :, :R].float().permute(0, 2, 1).reshape(A * R, st["n"])
    v = torch.matmul(x, st["w"][:, :dim].float().t()) + torch.matmul(low, up) + st["bias"]
    return _activated(v, st["act"], st.get("slope")).to(st["x"].dtype)


_PLAIN = dict(route=_plain_route, sort=_plain_sort, merge=_plain_merge, merge_grad=_plain_merge_grad, experts=_plain_experts, adapters=_plain_adapters)


# ---------------------------------------------------------------------------------------------- one pass
def _bz():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "x-deeplearning_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import blaze_hip
    return blaze_hip


def _own_route(bz, st):
    score = bz.ROUTE_SOFTMAX if st["score"] == "softmax" else bz.ROUTE_SIGMOID
    return bz.route_topk(st["logits"], st["k"], score=score, renormalize=st["renorm"], ids=st["ids"], weights=st["weights"])


def _own_sort(bz, st):
    return bz.group_rows(st["ids"], st["experts"], x=st["x"], offsets=st["offsets"], order=st["order"], position=st["position"], out=st["xs"])


def _own_merge(bz, st):
    return bz.merge_rows(st["xs"], st["position"], st["weights"], out=st["y"])


def _own_merge_grad(bz, st):
    return bz.merge_rows_grad(st["dy"], st["xs"], st["position"], st["weights"], dxs=st["dxs"], dweights=st["dw"])


def _own_act(bz, st):
    if st["act"] == "prelu":
        return dict(act=bz.ACT_PRELU, act_params=(st["slope"], ))
    if st["act"] == "relu":
        return dict(act=bz.ACT_LEAKY_RELU, act_alpha=0.0)
    return dict(act={"none": bz.ACT_NONE, "sigmoid": bz.ACT_SIGMOID, "swiglu": bz.ACT_SWIGLU}[st["act"]])


def _own_experts(bz, st):
    picked = dict(rows=st["order"], rows_per=st["k"]) if st["gather"] else {}
    return bz.grouped_fc(st["x"], st["w"], st["offsets"], st["dim"], bias=st["bias"], out=st["y"], **picked, **_own_act(bz, st))


def _own_adapters(bz, st):
    return bz.fc_adapters(st["x"], st["w"], st["dim"], st["down"], st["up"], st["ids"], rank=st["rank"], scale=st["scale"], bias=st["bias"], out=st["y"],
                          **_own_act(bz, st))


_OWN = dict(route=_own_route, sort=_own_sort, merge=_own_merge, merge_grad=_own_merge_grad, experts=_own_experts, adapters=_own_adapters)


def run(state):
    if own:
        return _OWN[state["kind"]](_bz(), state)
    return _PLAIN[state["kind"]](state)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, T, es = case["kind"], case["rows"], SIZE[case["dtype"]]
    if kind == "route":
        return {"bytes": T * (case["experts"] * es + 8.0 * case["k"]), "flops": 4.0 * T * case["experts"]}
    if kind in ("sort", "merge", "merge_grad"):
        k, dim, taken = case["k"], case["dim"], T * (1.0 - case["padded"])
        if kind == "sort":
            return {"bytes": 12.0 * T * k + 4.0 * (case["experts"] + 1) + taken * dim * es * (1 + k), "flops": 0.0}
        if kind == "merge":
            return {"bytes": 8.0 * T * k + taken * k * dim * es + T * dim * es, "flops": 2.0 * taken * k * dim}
        return {"bytes": 12.0 * T * k + taken * dim * es * (1 + 2 * k), "flops": 3.0 * taken * k * dim}
    dim, n = case["dim"], case["n"]
    if kind == "experts":
        R, cols = T * case["k"], n * (2 if case["act"] == "swiglu" else 1)
        used = case["experts"] * -math.expm1(-R / case["experts"])
        return {"bytes": used * cols * (dim * es + 4.0) + (T if case["gather"] else R) * dim * es + 4.0 * R + R * n * es, "flops": 2.0 * R * dim * cols}
    R, used = case["rank"], min(case["requests"], case["adapters"]) * (1.0 - case["none"])
    return {"bytes": n * dim * es + 4.0 * n + used * R * (dim + n) * es + T * ((dim + n) * es + 4.0),
            "flops": 2.0 * T * dim * n + 2.0 * T * (1.0 - case["none"]) * R * (dim + n)}


# ---------------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        l = st["logits"].double()
        l = torch.nan_to_num(l, nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        p = torch.nan_to_num(torch.softmax(l, 1), nan=0.0) if case["score"] == "softmax" else torch.sigmoid(l)
        best = torch.sort(l, dim=1, descending=True, stable=True)[1][:, :case["k"]]
        w = p.gather(1, best) * (l.gather(1, best) > -math.inf)
        if case["renorm"]:
            w = torch.nan_to_num(w / w.sum(1, keepdim=True), nan=0.0)
        return None, w
    if kind == "sort":
        flat = st["ids"].reshape(-1)
        xs = torch.zeros(st["xs"].shape, dtype=torch.float64, device="cuda")
        entries = torch.cat([torch.nonzero(flat == e)[:, 0] for e in range(case["experts"])])
        xs[:entries.numel()] = st["x"][entries // case["k"]].double()
        return None, None, None, xs
    if kind in ("merge", "merge_grad"):
        xs, k = st["xs"].double(), case["k"]
        if kind == "merge":
            y = torch.zeros(st["y"].shape, dtype=torch.float64, device="cuda")
            for j in range(k):
                p = st["position"][:, j].long()
                t = torch.nonzero(p >= 0)[:, 0]
                y[t] += st["weights"][t, j, None].double() * xs[p[t]]
            return y
        dxs, dw = torch.zeros_like(xs), torch.zeros((case["rows"], k), dtype=torch.float64, device="cuda")
        for j in range(k):
            p = st["position"][:, j].long()
            t = torch.nonzero(p >= 0)[:, 0]
            dxs[p[t]] = st["weights"][t, j, None].double() * st["dy"][t].double()
            dw[t, j] = (st["dy"][t].double() * xs[p[t]]).sum(1)
        return dxs, dw
    n, dim, act = case["n"], case["dim"], case["act"]

    def finish(v, slope):
        if act == "swiglu":
            return v[:, :n] * torch.sigmoid(v[:, :n]) * v[:, n:]
        if act == "relu":
            return v.clamp(min=0.0)
        if act == "prelu":
            return v.clamp(min=0.0) + slope.double() * v.clamp(max=0.0)
        return torch.sigmoid(v) if act == "sigmoid" else v

    y = torch.zeros(st["y"].shape, dtype=torch.float64, device="cuda")
    if kind == "experts":
        cut = st["offsets"].tolist()
        for e in range(case["experts"]):
            if cut[e + 1] > cut[e]:
                rows = st["order"][cut[e]:cut[e + 1]].long() // case["k"] if case["gather"] else slice(cut[e], cut[e + 1])
                v = st["x"][rows].double() @ st["w"][e, :, :dim].double().t() + st["bias"][e].double()
                y[cut[e]:cut[e + 1]] = finish(v, st["slope"][e] if act == "prelu" else None)
        return y
    x = st["x"].double()
    y = x @ st["w"][:, :dim].double().t() + st["bias"].double()
    for g in range(case["adapters"]):
        rows = torch.nonzero(st["ids"] == g)[:, 0]
        if rows.numel():
            y[rows] += st["scale"][g].double() * (x[rows] @ st["down"][g, :, :dim].double().t()) @ st["up"][g, :, :case["rank"]].double().t()
    return finish(y, st.get("slope"))
