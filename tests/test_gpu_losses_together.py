"""The losses of a language model's training step as a program uses them together: a vocabulary head whose
hidden states also feed a router, a student's logits under distillation, gradients accumulated into the same
tensors, Adam over all of them, several steps; against the same program in 64 bits. And the losses beside the
library's other state: captured graphs, growing scratch, shut down and started again, calls that wait."""
import ctypes

import numpy as np
import pytest

import test_gpu_distill
import test_gpu_head
import test_gpu_router
from util import TEST_ASYNC, GpuEngine

pytestmark = pytest.mark.gpu

ROWS, DIM, CLASSES, EXPERTS, K, TOP = 70, 24, 301, 24, 3, 5
LR, B1, B2, EPS = 1e-2, 0.9, 0.999, 1e-8


def data(seed=0):
    r = np.random.RandomState(seed)
    labels = r.randint(0, CLASSES, ROWS).astype(np.int32)
    labels[::9] = -100
    ids = np.stack([r.choice(CLASSES, TOP, replace=False) for _ in range(ROWS)]).astype(np.int32)
    ids[::7, 3:] = -1
    return {"x": r.standard_normal((ROWS, DIM)).astype(np.float32), "w": (0.5 * r.standard_normal((CLASSES, DIM))).astype(np.float32),
            "s": r.standard_normal((ROWS, CLASSES)).astype(np.float32), "labels": labels, "ids": ids,
            "teacher": -np.sort(-r.standard_normal((ROWS, TOP)), 1).astype(np.float32),
            "keep": (labels >= 0).astype(np.int32), "gw": (0.1 * r.standard_normal((ROWS, K))).astype(np.float32)}


def exact_step(p, d):
    """The gradients and losses of one step in 64 bits, p the parameters, and the router's choice."""
    head, _ = test_gpu_head.reference(p["x"], p["w"], d["labels"])
    dis, _ = test_gpu_distill.reference(p["s"], d["ids"], d["teacher"], T=2.0)
    rout, _, whole = test_gpu_router.reference(p["x"], K, d["keep"], True, d["gw"], 0.1)
    return ({"x": head["grad_x"] + rout["grad_x"], "w": head["grad_w"], "s": dis["grad_x"]},
            [head["loss"], dis["loss"], rout["loss"]], whole["chosen"])


def step(m, t, g, out):
    for k in "xws":
        g[k].zero()
    m.linear_cross_entropy_step(out["head"], g["x"], g["w"], t["x"], t["w"], t["labels"], out["one"])
    m.distill_step(out["dis"], g["s"], t["s"], t["ids"], t["teacher"], out["one"], temperature=2.0)
    m.router_forward(out["weights"], out["chosen"], out["counts"], out["bal"], t["x"], keep=t["keep"], normalise=True)
    m.router_backward(g["x"], t["x"], out["chosen"], out["counts"], t["gw"], out["tenth"], keep=t["keep"], normalise=True)


def program(m, d):
    t = {k: (m.IndexTensor if v.dtype == np.int32 else m.Tensor).from_numpy(v) for k, v in d.items()}
    g = {k: m.Tensor(t[k].shape()) for k in "xws"}
    out = {"head": m.Tensor(1), "dis": m.Tensor(1), "bal": m.Tensor(1), "weights": m.Tensor(ROWS, K),
           "chosen": m.IndexTensor(ROWS, K), "counts": m.IndexTensor(EXPERTS), "one": m.Tensor.from_numpy(np.float32([1])),
           "tenth": m.Tensor.from_numpy(np.float32([0.1]))}
    return t, g, out


def test_training_steps():
    m = GpuEngine().m
    d = data()
    t, g, out = program(m, d)
    opt = m.Adam([(t[k], g[k]) for k in "xws"], lr=LR, beta1=B1, beta2=B2, epsilon=EPS)
    first = None
    for it in range(4):
        p = {k: t[k].to_numpy() for k in "xws"}  # the library's own parameters: rounding does not build up
        grads, losses, order = exact_step(p, d)
        step(m, t, g, out)
        got = [out["head"][0], out["dis"][0], out["bal"][0]]
        assert np.allclose(got, losses, rtol=2e-6), it
        assert np.array_equal(out["chosen"].to_numpy(), order)
        for k in "xws":
            off = np.abs(g[k].to_numpy() - grads[k])
            assert off.max() <= 4e-6 * np.abs(grads[k]).max(), (it, k, off.max())
        opt.step()
        first = first or got
    assert np.isfinite(got).all()


def test_beside_captured_graphs():
    """A captured model replays with its own results while the losses grow the library's scratch around it."""
    m = GpuEngine().m
    d = data(1)
    t, g, out = program(m, d)
    r = np.random.RandomState(3)
    gr = m.Graph()
    x = gr.input((32, 1000), trainable=True)
    gr.loss(gr.op(m.OP.MEAN, gr.op(m.OP.SUM, gr.op(m.OP.EXP, x), attributes={"axis": 0})))
    model = m.Model(gr)
    xin = m.Tensor.from_numpy(r.standard_normal((32, 1000)).astype(np.float32))
    model.forward(xin)
    model.parameters.grads.set_zero()
    model.backward()
    want = model.parameters.grads[x].to_numpy()
    step(m, t, g, out)
    ref = {k: g[k].to_numpy() for k in "xws"}
    model.capture("step")
    big = r.standard_normal((700, 96)).astype(np.float32), r.standard_normal((9000, 96)).astype(np.float32)
    tb = [m.Tensor.from_numpy(a) for a in big]
    lb, gw, loss = m.IndexTensor.from_numpy(r.randint(0, 9000, 700)), m.Tensor(9000, 96), m.Tensor(1)
    for _ in range(3):
        step(m, t, g, out)
        for k in "xws":
            assert np.array_equal(g[k].to_numpy(), ref[k])
        m.linear_cross_entropy_step(loss, None, gw, tb[0], tb[1], lb, out["one"], accumulate=False)
        model.replay("step")
        m.sync()
        assert np.array_equal(model.parameters.grads[x].to_numpy(), want)


def test_after_shutdown_and_without_async():
    m = GpuEngine().m
    d = data(2)
    t, g, out = program(m, d)
    step(m, t, g, out)
    ref = {k: g[k].to_numpy() for k in "xws"}
    try:
        m._lib.call("mh_shutdown")
        m.init(0, asynchronous=False)  # every call waits for its own end
        step(m, t, g, out)
        for k in "xws":
            assert np.array_equal(g[k].to_numpy(), ref[k])
    finally:
        m._lib.call("mh_shutdown")
        m.init(0, asynchronous=TEST_ASYNC)


def test_many_sizes_in_turn_share_the_scratch():
    """Calls of falling and rising sizes, queued without waiting: each finds its own workspace whole."""
    m = GpuEngine().m
    r = np.random.RandomState(4)
    runs = []
    for rows, dim, classes in ((300, 40, 4000), (5, 3, 7), (64, 500, 900), (1, 1, 1), (600, 40, 2000), (33, 64, 12000)):
        x, w = m.Tensor.from_numpy(r.standard_normal((rows, dim))), m.Tensor.from_numpy(r.standard_normal((classes, dim)))
        lb = m.IndexTensor.from_numpy(r.randint(0, classes, rows))
        k = min(classes, 6)
        ids, te = m.IndexTensor.from_numpy(r.randint(0, classes, (rows, k))), m.Tensor.from_numpy(r.standard_normal((rows, k)))
        lg, one = m.Tensor.from_numpy(r.standard_normal((rows, classes))), m.Tensor.from_numpy(np.float32([1]))
        runs.append((x, w, lb, ids, te, lg, one))

    def go(i, wait):
        x, w, lb, ids, te, lg, one = runs[i]
        o = [m.Tensor(1), m.Tensor(x.shape()), m.Tensor(w.shape()), m.Tensor(1), m.Tensor(lg.shape())]
        m.linear_cross_entropy_step(o[0], o[1], o[2], x, w, lb, one, accumulate=False)
        m.distill_step(o[3], o[4], lg, ids, te, one, accumulate=False)
        if wait:
            m.sync()
        return o

    alone = [[a.to_numpy() for a in go(i, True)] for i in range(len(runs))]
    queued = [go(i, False) for i in range(len(runs))]
    for a, q in zip(alone, queued):
        for u, v in zip(a, q):
            assert np.array_equal(u, v.to_numpy())


def test_a_refused_allocation_does_not_fail_the_next_call():
    """An allocation that the device cannot hold returns an error, and the calls behind it go on."""
    m = GpuEngine().m
    d = data(3)
    t, g, out = program(m, d)
    step(m, t, g, out)
    ref = {k: g[k].to_numpy() for k in "xws"}
    with pytest.raises(m.MantleHipError) as e:
        m._lib.call("mh_malloc", ctypes.byref(ctypes.c_void_p()), 1 << 46)
    assert e.value.code == m._lib.ERR_HIP
    step(m, t, g, out)
    for k in "xws":
        assert np.array_equal(g[k].to_numpy(), ref[k])
