"""Operators of nets whose rows go through different weights (TopKGate, ExpertDispatch, GroupedGemm, ExpertCombine, AdapterGemm), run
through a Predictor, against plain forms in 64 bits.

Bars: choices are exact.  A layer's output of type t is rounded once (half a step: 2^-24 fp32, 2^-11 fp16) and an fp32 sum of K products is
off by at most (K + 8) * 2^-24 of its absolute terms' sum; a tensor between two operators is rounded to its type.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
EPS = 2.0**-24


@pytest.fixture(scope="module")
def pb():
    import torch
    import blaze_hip
    import pyblaze_hip
    assert torch.cuda.is_available(), "no GPU visible"
    blaze_hip.device_check()
    return pyblaze_hip


def _half(dtype):
    return 2.0**-24 if dtype == np.float32 else 2.0**-11


def _round(x, dtype):
    return x.astype(np.float32).astype(dtype).astype(np.float64)


def _mixture(pb, dtype, dim, hidden, experts, k, gather, transb=False, weighted=True):
    """x -> Gemm -> TopKGate -> ExpertDispatch -> GroupedGemm(swiglu) -> GroupedGemm -> ExpertCombine; (manager, weights in 64 bits)"""
    code = pb.K_FLOAT16 if dtype == np.float16 else pb.K_FLOAT
    rng = np.random.default_rng(dim + hidden)
    w = dict(gate=rng.standard_normal((dim, experts)) / np.sqrt(dim), w1=rng.standard_normal((experts, dim, 2 * hidden)) / np.sqrt(dim),
             b1=rng.standard_normal((experts, 2 * hidden)) * 0.1, w2=rng.standard_normal((experts, hidden, dim)) / np.sqrt(hidden),
             b2=rng.standard_normal((experts, dim)) * 0.1, zero=np.zeros(experts))
    w = {n: _round(v, dtype) for n, v in w.items()}
    nb = pb.NetBuilder("mixture", device_type=1)
    nb.external_input("x", code)
    for name, t in (("y", code), ("ids", pb.K_INT32), ("weights", pb.K_FLOAT), ("logits", code)):
        nb.external_output(name, t)
    for name, v in w.items():
        v = np.swapaxes(v, 1, 2) if transb and name in ("w1", "w2") else v
        nb.constant(name, v.astype(np.float32), dtype=code)
    nb.op("Gemm", ["x", "gate", "zero"], ["logits"])
    nb.op("TopKGate", ["logits"], ["ids", "weights"], k=k, renormalize=True)
    nb.op("ExpertDispatch", ["x", "ids"], ["xs", "offsets", "position", "order"], experts=experts)
    if gather:
        nb.op("GroupedGemm", ["x", "w1", "offsets", "b1", "order"], ["h"], activation="swiglu", transB=transb)
    else:
        nb.op("GroupedGemm", ["xs", "w1", "offsets", "b1"], ["h"], activation="swiglu", transB=transb)
    nb.op("GroupedGemm", ["h", "w2", "offsets", "b2"], ["ys"], transB=transb)
    nb.op("ExpertCombine", ["ys", "position", "weights"] if weighted else ["ys", "position"], ["y"])
    pm = pb.PredictorManager()
    pm.load_model_from_string(nb.text(), True)
    return pm, w


def _mixture_want(w, x, ids, weights, dtype, hidden):
    want, size = np.zeros(x.shape), np.zeros(x.shape)
    for t in range(x.shape[0]):
        for j, e in enumerate(ids[t]):
            v = x[t] @ w["w1"][e] + w["b1"][e]
            h = v[:hidden] / (1.0 + np.exp(-v[:hidden])) * v[hidden:]
            want[t] += weights[t, j] * (h @ w["w2"][e] + w["b2"][e])
            size[t] += weights[t, j] * (np.abs(h) @ np.abs(w["w2"][e]) + np.abs(w["b2"][e]))
    return want, size


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("gather,transb", [(False, False), (True, True), (True, False)])
@pytest.mark.parametrize("dim,hidden,experts,k", [(64, 48, 8, 2), (50, 37, 5, 3)])
def test_mixture_of_experts_net(pb, dtype, gather, transb, dim, hidden, experts, k):
    pm, w = _mixture(pb, dtype, dim, hidden, experts, k, gather, transb)
    p = pm.create_predictor(1, 0)
    for rows in (1, 33, 700, 33, 6000):  # shapes change from pass to pass; the last one's entries are counted in a launch of their own
        print("case", dtype.__name__, gather, transb, dim, rows, flush=True)
        x = _round(np.random.default_rng(rows).standard_normal((rows, dim)), dtype)
        p.feed("x", x.astype(dtype))
        p.forward()
        logits, ids, weights = (p.output_asnumpy(n) for n in ("logits", "ids", "weights"))
        assert ids.dtype == np.int32 and weights.dtype == np.float32
        best = np.argsort(-logits.astype(np.float64), axis=1, kind="stable")[:, :k]
        assert np.array_equal(ids, best)
        e = np.exp(np.take_along_axis(logits.astype(np.float64), best, 1))
        np.testing.assert_allclose(weights, e / e.sum(1, keepdims=True), rtol=40 * EPS)
        some = np.unique(np.linspace(0, rows - 1, 60).astype(int))
        want, size = _mixture_want(w, x[some], ids[some], weights[some].astype(np.float64), dtype, hidden)
        bar = (3.2 * _half(dtype) + (dim + hidden + 64) * 4 * EPS) * size + _half(dtype) * np.abs(want)
        assert (np.abs(p.output_asnumpy("y")[some].astype(np.float64) - want) <= bar).all()


def test_rows_without_an_expert_come_back_as_zeros(pb):
    """ids fed as they are, some of none, and no weights"""
    rng = np.random.default_rng(0)
    rows, dim, experts, k = 90, 40, 6, 2
    wt, x = rng.standard_normal((experts, dim, dim)).astype(np.float32), rng.standard_normal((rows, dim)).astype(np.float32)
    ids = rng.integers(0, experts, (rows, k)).astype(np.int32)
    ids[5], ids[60:], ids[7, 1], ids[8, 0] = -1, experts, -1, 1000
    nb = pb.NetBuilder("n", device_type=1)
    nb.external_input("x", pb.K_FLOAT)
    nb.external_input("ids", pb.K_INT32)
    nb.external_output("y", pb.K_FLOAT)
    nb.constant("w", wt)
    nb.op("ExpertDispatch", ["x", "ids"], ["xs", "offsets", "position"], experts=experts)
    nb.op("GroupedGemm", ["xs", "w", "offsets"], ["h"], activation="leaky_relu", alpha=0.25)
    nb.op("ExpertCombine", ["h", "position"], ["y"])
    pm = pb.PredictorManager()
    pm.load_model_from_string(nb.text(), True)
    p = pm.create_predictor(1, 0)
    p.feed("x", x)
    p.feed("ids", ids)
    p.forward()
    y = p.output_asnumpy("y")
    want, size = np.zeros((rows, dim)), np.zeros((rows, dim))
    for t in range(rows):
        for e in ids[t]:
            if 0 <= e < experts:
                v = x[t].astype(np.float64) @ wt[e]
                want[t] += np.where(v >= 0, v, 0.25 * v)
                size[t] += np.abs(x[t]).astype(np.float64) @ np.abs(wt[e])
    assert (np.abs(y - want) <= (dim + 16) * EPS * size).all()
    assert (y[60:] == 0).all() and (y[5] == 0).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("transb", [False, True])
@pytest.mark.parametrize("k,n,adapters,rank", [(64, 48, 5, 8), (50, 33, 3, 5)])
def test_adapter_gemm_net(pb, dtype, transb, k, n, adapters, rank):
    code = pb.K_FLOAT16 if dtype == np.float16 else pb.K_FLOAT
    rng = np.random.default_rng(k)
    w = {name: _round(v, dtype) for name, v in dict(
        w=rng.standard_normal((k, n)) / np.sqrt(k), b=rng.standard_normal(n), down=rng.standard_normal((adapters, rank, k)) / np.sqrt(k),
        up=rng.standard_normal((adapters, n, rank)) / np.sqrt(rank), scale=rng.uniform(0.5, 2.0, adapters)).items()}
    nb = pb.NetBuilder("adapters", device_type=1)
    nb.external_input("x", code)
    nb.external_input("ids", pb.K_INT32)
    nb.external_output("y", code)
    nb.external_output("plain", code)
    for name, v in w.items():
        nb.constant(name, (v.T if transb and name == "w" else v).astype(np.float32), dtype=code)
    nb.op("AdapterGemm", ["x", "w", "b", "down", "up", "ids", "scale"], ["y"], transB=transb, alpha=0.5, beta=2.0)
    nb.op("AdapterGemm", ["x", "w", "b", "down", "up", "ids"], ["plain"], transB=transb)
    pm = pb.PredictorManager()
    pm.load_model_from_string(nb.text(), True)
    p = pm.create_predictor(1, 0)
    for rows in (1, 40, 700, 3):
        print("case", dtype.__name__, transb, k, rows, flush=True)
        x = _round(rng.standard_normal((rows, k)), dtype)
        ids = rng.integers(-1, adapters + 1, rows).astype(np.int32)
        p.feed("x", x.astype(dtype))
        p.feed("ids", ids)
        p.forward()
        for out, scale, alpha, beta in (("y", w["scale"], 0.5, 2.0), ("plain", np.ones(adapters), 1.0, 1.0)):
            want = alpha * (x @ w["w"]) + beta * w["b"]
            size = alpha * (np.abs(x) @ np.abs(w["w"])) + beta * np.abs(w["b"])
            slack = np.zeros_like(want)
            for g in range(adapters):
                r = ids == g
                low, lows = scale[g] * (x[r] @ w["down"][g].T), scale[g] * (np.abs(x[r]) @ np.abs(w["down"][g].T))
                want[r] += low @ w["up"][g].T
                size[r] += lows @ np.abs(w["up"][g].T)
                slack[r] = 2.0**-16 * (np.abs(low) @ np.abs(w["up"][g].T)) if dtype == np.float16 else 0.0
            bar = (k + 3 * rank + 24) * EPS * size + slack
            bar = bar + _half(dtype) * (np.abs(want) + bar) + (2.0**-25 if dtype == np.float16 else 0.0)
            assert (np.abs(p.output_asnumpy(out).astype(np.float64) - want) <= bar).all(), (out, rows)


@pytest.mark.parametrize("op,inputs,outputs,args,text", [
    ("TopKGate", ["x"], ["a", "b"], dict(k=17), "k=17"),
    ("TopKGate", ["x"], ["a", "b"], dict(k=2, score="tanh"), "score=tanh"),
    ("ExpertDispatch", ["x", "ids"], ["a", "b", "c"], dict(), "experts=0"),
    ("ExpertDispatch", ["x", "ids"], ["a", "b", "c"], dict(experts=2000), "experts=2000"),
    ("GroupedGemm", ["x", "w", "offsets"], ["a"], dict(activation="gelu"), "activation=gelu"),
])
def test_arguments_that_are_refused(pb, op, inputs, outputs, args, text):
    nb = pb.NetBuilder("n", device_type=1)
    nb.external_input("x", pb.K_FLOAT)
    nb.external_input("ids", pb.K_INT32)
    nb.external_input("offsets", pb.K_INT32)
    nb.external_output(outputs[0], pb.K_FLOAT)
    nb.constant("w", np.zeros((2, 4, 4), np.float32))
    nb.op(op, inputs, outputs, **args)
    pm = pb.PredictorManager()
    with pytest.raises(pb.BlazeError, match=text):
        pm.load_model_from_string(nb.text(), True)
        pm.create_predictor(1, 0)


@pytest.mark.parametrize("op,outputs,args,shapes,text", [
    ("TopKGate", ["a", "b"], dict(k=5), dict(x=(3, 4)), "k=5 of n=4"),
    ("ExpertDispatch", ["a", "b", "c"], dict(experts=3), dict(x=(3, 4), i=(2, 2)), "rows of x and ids differ"),
    ("GroupedGemm", ["a"], dict(), dict(x=(3, 5), w=(2, 4, 4), i=(3, )), "K=5 of A, 4 of W"),
    ("GroupedGemm", ["a"], dict(), dict(x=(3, 4), w=(2, 4, 4), i=(2, )), "groups=2"),
    ("GroupedGemm", ["a"], dict(activation="swiglu"), dict(x=(3, 4), w=(2, 4, 5), i=(3, )), "swiglu of 5"),
    ("ExpertCombine", ["a"], dict(), dict(x=(3, 4), i=(3, )), "not 2-D"),
])
def test_shapes_that_are_refused(pb, op, outputs, args, shapes, text):
    nb = pb.NetBuilder("n", device_type=1)
    for name in shapes:
        nb.external_input(name, pb.K_INT32 if name == "i" else pb.K_FLOAT)
    nb.external_output(outputs[0], pb.K_FLOAT)
    nb.op(op, list(shapes), outputs, **args)
    pm = pb.PredictorManager()
    pm.load_model_from_string(nb.text(), True)
    p = pm.create_predictor(1, 0)
    for name, shape in shapes.items():
        p.feed(name, np.zeros(shape, np.int32 if name == "i" else np.float32))
    with pytest.raises(pb.BlazeError, match=text):
        p.forward()


def test_steady_state_allocates_nothing(pb):
    pm, _ = _mixture(pb, np.float16, 64, 48, 8, 2, True)
    p = pm.create_predictor(1, 0)
    x = np.random.default_rng(0).standard_normal((500, 64)).astype(np.float16)
    p.feed("x", x)
    p.forward()
    want, before = p.output_asnumpy("y"), pb.allocation_count()
    for _ in range(5):
        p.feed("x", x)
        p.forward()
        assert np.array_equal(p.output_asnumpy("y"), want)
    assert pb.allocation_count() == before


def test_predictors_on_threads_of_their_own(pb):
    import threading
    pm, _ = _mixture(pb, np.float32, 64, 48, 8, 2, False)
    p = pm.create_predictor(1, 0)
    xs = [np.random.default_rng(i).standard_normal((200 + 50 * i, 64)).astype(np.float32) for i in range(3)]
    wants = []
    for x in xs:
        p.feed("x", x)
        p.forward()
        wants.append(p.output_asnumpy("y"))
    bad = []

    def serve(i):
        q = pm.create_predictor(1, 0)
        for turn in range(10):
            x = (i + turn) % 3
            q.feed("x", xs[x])
            q.forward()
            if not np.array_equal(q.output_asnumpy("y"), wants[x]):
                bad.append((i, turn))

    threads = [threading.Thread(target=serve, args=(i, )) for i in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_grouped_gemm_sigmoid_over_its_range(pb, dtype):
    code = pb.K_FLOAT16 if dtype == np.float16 else pb.K_FLOAT
    v = np.array([0.0, 1.0, -1.0, 20.0, -20.0, 88.0, 88.75, 89.0, -89.0, 120.0, 3e3, -3e3, 6e4, -6e4])
    x, w = np.zeros((v.size, 8)), np.zeros((2, 8, 40))
    x[:, 3], w[:, 3] = v, 1.0
    nb = pb.NetBuilder("n", device_type=1)
    nb.external_input("x", code)
    nb.external_input("offsets", pb.K_INT32)
    nb.external_output("y", code)
    nb.constant("w", w.astype(np.float32), dtype=code)
    nb.op("GroupedGemm", ["x", "w", "offsets"], ["y"], activation="sigmoid")
    pm = pb.PredictorManager()
    pm.load_model_from_string(nb.text(), True)
    p = pm.create_predictor(1, 0)
    p.feed("x", x.astype(dtype))
    p.feed("offsets", np.array([0, 5, v.size], np.int32))
    p.forward()
    with np.errstate(over="ignore"):
        want = np.broadcast_to((1.0 / (1.0 + np.exp(-v.astype(dtype).astype(np.float64))))[:, None], (v.size, 40))
    bar = (_half(dtype) + 16 * EPS) * want + (2.0**-25 if dtype == np.float16 else 2.0**-126)
    assert (np.abs(p.output_asnumpy("y").astype(np.float64) - want) <= bar).all()
