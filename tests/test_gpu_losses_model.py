"""The losses behind a model of the library's own: a graph makes the hidden states, the vocabulary head and the router read
them where they lie in the model's memory, their gradients go back into Model.backward as its upper gradient, and Adam
steps the graph's parameters and the head's. Every step against the same in 64 bits."""
import numpy as np
import pytest

import test_gpu_head
import test_gpu_router
from util import GpuEngine

pytestmark = pytest.mark.gpu

ROWS, DIM, CLASSES, K = 90, 24, 301, 3


def build(m, r):
    g = m.Graph()
    x = g.input((ROWS, DIM))
    gamma = g.param((1, DIM), init=(1 + 0.1 * r.standard_normal((1, DIM))).astype(np.float32))
    beta = g.param((1, DIM), init=(0.1 * r.standard_normal((1, DIM))).astype(np.float32))
    h = g.op(m.OP.TANH, g.op(m.OP.ADD, g.op(m.OP.MUL, x, gamma), beta))
    g.out(h)
    return g, gamma, beta, h


def exact(x, gamma, beta, h, w, labels, gw):
    """The gradients from the hidden states that the model computed."""
    head, _ = test_gpu_head.reference(h, w, labels)
    rout, _, _ = test_gpu_router.reference(h, K, (labels >= 0).astype(np.int32), True, gw, 0.1)
    gh = head["grad_x"] + rout["grad_x"]
    gu = gh * (1 - h.astype(np.float64) ** 2)
    return gh, {"w": head["grad_w"], "gamma": (gu * x).sum(0, keepdims=True), "beta": gu.sum(0, keepdims=True)}, \
        [head["loss"], rout["loss"]]


@pytest.mark.parametrize("captured", [False, True])
def test_training_steps(captured):
    m = GpuEngine().m
    r = np.random.RandomState(91)
    x = r.standard_normal((ROWS, DIM)).astype(np.float32)
    labels = r.randint(0, CLASSES, ROWS).astype(np.int32)
    labels[::9] = -100
    gwts = (0.1 * r.standard_normal((ROWS, K))).astype(np.float32)
    g, gamma, beta, h = build(m, r)
    model = m.Model(g)
    w, grad_w = m.Tensor.from_numpy((0.5 * r.standard_normal((CLASSES, DIM))).astype(np.float32)), m.Tensor(CLASSES, DIM)
    tx, tl, keep = m.Tensor.from_numpy(x), m.IndexTensor.from_numpy(labels), m.IndexTensor.from_numpy((labels >= 0).astype(np.int32))
    one, tenth, tgw = m.Tensor.from_numpy(np.float32([1])), m.Tensor.from_numpy(np.float32([0.1])), m.Tensor.from_numpy(gwts)
    loss, bal, weights, chosen, counts = m.Tensor(1), m.Tensor(1), m.Tensor(ROWS, K), m.IndexTensor(ROWS, K), m.IndexTensor(DIM)
    gh = m.Tensor(ROWS, DIM)
    opts = [m.Adam(model.parameters, lr=1e-2), m.Adam([(w, grad_w)], lr=1e-2)]
    hidden = model.parameters.tensors[h]  # where the model keeps them
    model.inference(tx)
    if captured:
        model.capture("forward")
    before = None
    for step in range(4):
        for o in opts:
            o.zero_grad()
        gh.zero()
        if captured:
            model.replay("forward")
        else:
            model.inference(tx)
        m.linear_cross_entropy_step(loss, gh, grad_w, hidden, w, tl, one)
        m.router_forward(weights, chosen, counts, bal, hidden, keep=keep, normalise=True)
        m.router_backward(gh, hidden, chosen, counts, tgw, tenth, keep=keep, normalise=True)
        model.backward(gh)
        par = {"gamma": model.parameters.tensors[gamma].to_numpy(), "beta": model.parameters.tensors[beta].to_numpy()}
        h_now, w_now = hidden.to_numpy(), w.to_numpy()
        assert np.allclose(h_now, np.tanh(x * par["gamma"] + par["beta"]), atol=1e-6)
        want_h, want, losses = exact(x, par["gamma"], par["beta"], h_now, w_now, labels, gwts)
        assert np.allclose([loss[0], bal[0]], losses, rtol=2e-6), step
        got = {"w": grad_w.to_numpy(), "gamma": model.parameters.grads[gamma].to_numpy(), "beta": model.parameters.grads[beta].to_numpy()}
        assert np.abs(gh.to_numpy() - want_h).max() <= 4e-6 * np.abs(want_h).max()
        for name in want:
            # gamma and beta: ROWS fp32 terms more, and tanh's derivative from an h rounded to 2^-24
            off, scale = np.abs(got[name] - want[name]).max(), np.abs(want[name]).max()
            assert off <= 2e-5 * max(scale, np.abs(want_h).max()), (step, name, off, scale)
        for o in opts:
            o.step()
        assert before is None or not np.array_equal(before, par["gamma"])
        before = par["gamma"]
