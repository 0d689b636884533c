"""What stands around the losses of a language model, as a program uses it together: the residual stream normalised before a
vocabulary head, a grouped router with its bias, a student's logits under distillation from which the next labels are drawn,
and Adam over all of it with the gradients' norm clipped; several steps, against the same program in 64 bits. And these
calls beside the library's other state: captured graphs, growing scratch, shut down and started again; tensors of more than 2^31
elements."""
import numpy as np
import pytest

import test_gpu_distill
import test_gpu_group_router
import test_gpu_head
import test_gpu_norm
import test_gpu_sample
from util import TEST_ASYNC, GpuEngine, assert_bitexact

pytestmark = pytest.mark.gpu

ROWS, DIM, CLASSES, EXPERTS, K, GROUPS, OPEN, TOP = 70, 24, 301, 24, 3, 6, 3, 5
LR, B1, B2, EPS, TINY, TOP_NORM, RATE = 1e-2, 0.9, 0.999, 1e-8, 1e-5, 0.05, 0.01
NAMES = ("x", "nw", "w", "s", "z")


def data(seed=0):
    r = np.random.RandomState(seed)
    f = lambda *a: r.standard_normal(a).astype(np.float32)  # noqa: E731
    ids = np.stack([r.choice(CLASSES, TOP, replace=False) for _ in range(ROWS)]).astype(np.int32)
    ids[::7, 3:] = -1
    labels = r.randint(0, CLASSES, ROWS).astype(np.int32)
    return {"x": f(ROWS, DIM), "res": f(ROWS, DIM), "nw": 1 + 0.1 * f(DIM), "w": 0.5 * f(CLASSES, DIM), "s": f(ROWS, CLASSES),
            "z": f(ROWS, EXPERTS), "labels": labels, "ids": ids, "teacher": -np.sort(-f(ROWS, TOP), 1), "gsum": 0.01 * f(ROWS, DIM),
            "keep": (r.uniform(size=ROWS) > 0.1).astype(np.int32), "gw": 0.1 * f(ROWS, K), "u": r.uniform(size=ROWS).astype(np.float32),
            "temperature": r.choice([0.0, 0.7, 1.0], ROWS).astype(np.float32), "top_k": r.choice([0, 40], ROWS).astype(np.int32),
            "top_p": np.full(ROWS, 0.9, np.float32)}


def program(m, d):
    t = {k: (m.IndexTensor if v.dtype == np.int32 else m.Tensor).from_numpy(v) for k, v in d.items()}
    o = {k: m.Tensor(1) for k in ("head", "dis")}
    o.update(out=m.Tensor(ROWS, DIM), h=m.Tensor(ROWS, DIM), gout=m.Tensor(ROWS, DIM), weights=m.Tensor(ROWS, K),
             chosen=m.IndexTensor(ROWS, K), counts=m.IndexTensor(EXPERTS), bias=m.Tensor(EXPERTS), logprob=m.Tensor(ROWS),
             one=m.Tensor.from_numpy(np.float32([1])))
    g = {k: m.Tensor(t[k].shape()) for k in NAMES}
    return t, g, o, m.Adam([(t[k], g[k]) for k in NAMES], lr=LR, beta1=B1, beta2=B2, epsilon=EPS, max_norm=TOP_NORM)


def step(m, t, g, o, opt=None):
    m.rms_norm_forward(o["out"], t["x"], t["nw"], residual=t["res"], sum=o["h"], eps=TINY)
    m.linear_cross_entropy_step(o["head"], o["gout"], g["w"], o["out"], t["w"], t["labels"], o["one"], accumulate=False)
    m.rms_norm_backward(g["x"], g["nw"], o["gout"], o["h"], t["nw"], grad_sum=t["gsum"], eps=TINY, accumulate=False)
    m.distill_step(o["dis"], g["s"], t["s"], t["ids"], t["teacher"], o["one"], accumulate=False)
    m.group_router_forward(o["weights"], o["chosen"], o["counts"], t["z"], bias=o["bias"], keep=t["keep"], groups=GROUPS, keep_groups=OPEN)
    m.group_router_backward(g["z"], t["z"], o["chosen"], t["gw"], keep=t["keep"], accumulate=False)
    m.router_bias_update(o["bias"], o["counts"], RATE)
    if opt is not None:
        opt.step()
    m.sample_tokens(t["labels"], t["s"], t["u"], temperature=t["temperature"], top_k=t["top_k"], top_p=t["top_p"], logprob=o["logprob"])


def exact_step(p, d):
    """One step in 64 bits from the library's parameters p: gradients, the router's choice, the losses."""
    h = p["x"] + d["res"]
    out, _ = test_gpu_norm.reference(h, p["nw"], TINY)
    head, _ = test_gpu_head.reference(out["out"].astype(np.float32), p["w"], p["labels"])
    norm, _ = test_gpu_norm.reference(h, p["nw"], TINY, head["grad_x"].astype(np.float32), d["gsum"])
    dis, _ = test_gpu_distill.reference(p["s"], d["ids"], d["teacher"])
    rout, _, whole = test_gpu_group_router.reference(p["z"], K, p["bias"], d["keep"], GROUPS, OPEN, gw=d["gw"])
    return ({"x": norm["grad_x"], "nw": norm["grad_w"], "w": head["grad_w"], "s": dis["grad_x"], "z": rout["grad_x"]},
            whole, [head["loss"], dis["loss"]])


def test_training_steps():
    m = GpuEngine().m
    d = data()
    t, g, o, opt = program(m, d)
    for it in range(1, 5):
        p = {k: t[k].to_numpy() for k in (*NAMES, "labels")}
        p["bias"] = o["bias"].to_numpy()
        was_m, was_v = ([a.to_numpy() for a in s] for s in (opt.momentum_grads, opt.rms_grads))
        grads, whole, losses = exact_step(p, d)
        step(m, t, g, o, opt)
        assert np.allclose([o["head"][0], o["dis"][0]], losses, rtol=4e-6), it
        assert np.array_equal(o["chosen"].to_numpy(), whole["chosen"]) and np.array_equal(o["counts"].to_numpy(), whole["counts"])
        c = whole["counts"].astype(np.int64) * EXPERTS
        assert_bitexact(o["bias"].to_numpy(), np.where(c < c.sum() // EXPERTS, p["bias"] + np.float32(RATE),
                                                       np.where(c > c.sum() // EXPERTS, p["bias"] - np.float32(RATE), p["bias"])), "bias")
        norm = np.sqrt(sum((v ** 2).sum() for v in grads.values()))
        assert norm > TOP_NORM and abs(opt.grad_norm[0] - norm) <= 1e-5 * norm
        for i, k in enumerate(NAMES):
            mine = g[k].to_numpy()
            assert np.abs(mine - grads[k]).max() <= 1e-5 * np.abs(grads[k]).max(), (it, k)
            mk, vk = (a[i].to_numpy() for a in (opt.momentum_grads, opt.rms_grads))
            gc = mine.astype(np.float64) * TOP_NORM / float(opt.grad_norm[0])
            em, ev = B1 * was_m[i].astype(np.float64) + (1 - B1) * gc, B2 * was_v[i].astype(np.float64) + (1 - B2) * gc * gc
            # 1 - beta in fp32: 2^-24 of 0.999 is 6e-5 of 0.001
            assert np.abs(mk - em).max() <= 2e-6 * np.abs(em).max() and np.abs(vk - ev).max() <= 1e-4 * np.abs(ev).max()
            # the update from the library's own moments; 1 - 0.999^it in fp32 is off by 6e-5 of itself at most
            ep = p[k] - LR * (mk / (1 - B1 ** it)) / (np.sqrt(vk / (1 - B2 ** it)) + EPS)
            assert np.abs(t[k].to_numpy() - ep).max() <= 1e-4 * LR * np.abs(mk / (1 - B1 ** it) / (np.sqrt(vk / (1 - B2 ** it)) + EPS)).max() + 1e-6
        # the labels of the next step, drawn from the student as it is now
        s, tokens, lp = t["s"].to_numpy(), t["labels"].to_numpy(), o["logprob"].to_numpy()
        for r in range(ROWS):
            may, _ = test_gpu_sample.reference(s[r], d["u"][r], d["temperature"][r], int(d["top_k"][r]), 0.9)
            assert tokens[r] in may and any(abs(lp[r] - v) <= off for v, off in may[tokens[r]]), r


def results(t, g, o):
    return {**{k: v.to_numpy() for k, v in g.items()}, **{k: v.to_numpy() for k, v in o.items()}, "tokens": t["labels"].to_numpy()}


def same(a, b):
    for k in a:
        assert np.array_equal(a[k], b[k]), k


def again(m, t, g, o, d):
    """The step from the beginning, without an update."""
    for k, v in d.items():
        m._lib.call("mh_memcpy_h2d", t[k].ptr, v.ctypes.data, 4 * v.size)
    o["bias"].zero()
    step(m, t, g, o)
    m.grad_norm(o["head"], list(g.values()))
    return results(t, g, o)


def test_beside_captured_graphs():
    """A captured model replays with its own results while these calls grow the library's scratch around it."""
    m = GpuEngine().m
    d = data(1)
    t, g, o, _ = program(m, d)
    r = np.random.RandomState(3)
    gr = m.Graph()
    x = gr.input((32, 1000), trainable=True)
    gr.loss(gr.op(m.OP.MEAN, gr.op(m.OP.SUM, gr.op(m.OP.EXP, x), attributes={"axis": 0})))
    model = m.Model(gr)
    model.forward(m.Tensor.from_numpy(r.standard_normal((32, 1000)).astype(np.float32)))
    model.parameters.grads.set_zero()
    model.backward()
    want = model.parameters.grads[x].to_numpy()
    ref = again(m, t, g, o, d)
    model.capture("step")
    big = m.Tensor.from_numpy(r.standard_normal((30000, 60)).astype(np.float32))
    wide = m.Tensor.from_numpy(r.standard_normal((600, 3000)).astype(np.float32))
    gx, gw, w = m.Tensor(600, 3000), m.Tensor(3000), m.Tensor.from_numpy(np.ones(3000))
    bw, bc, bn = m.Tensor(30000, 4), m.IndexTensor(30000, 4), m.IndexTensor(60)
    seen = None
    for _ in range(3):
        same(again(m, t, g, o, d), ref)
        m.group_router_forward(bw, bc, bn, big, groups=6, keep_groups=3)
        m.rms_norm_backward(gx, gw, wide, wide, w, accumulate=False)
        model.replay("step")
        m.sync()
        assert np.array_equal(model.parameters.grads[x].to_numpy(), want)
        now = (bw.to_numpy(), bc.to_numpy(), bn.to_numpy(), gx.to_numpy(), gw.to_numpy())
        seen = seen or now
        assert all(np.array_equal(a, b) for a, b in zip(seen, now)) and now[2].sum() == 120000


def test_after_shutdown_and_without_async():
    m = GpuEngine().m
    d = data(2)
    t, g, o, _ = program(m, d)
    ref = again(m, t, g, o, d)
    try:
        m._lib.call("mh_shutdown")
        m.init(0, asynchronous=False)  # every call waits for its own end
        same(again(m, t, g, o, d), ref)
    finally:
        m._lib.call("mh_shutdown")
        m.init(0, asynchronous=TEST_ASYNC)


def test_queued_calls_share_the_scratch():
    """Calls of falling and rising sizes, queued without waiting: each finds its own workspace whole."""
    m = GpuEngine().m
    r = np.random.RandomState(4)
    T = m.Tensor.from_numpy
    sets = []
    for rows, dim, experts in ((5000, 64, 32), (3, 5, 7), (700, 2000, 128), (1, 1, 1), (2500, 17000, 60), (4000, 300, 256)):
        sets.append((T(r.standard_normal((rows, dim))), T(r.standard_normal(dim)), T(r.standard_normal((rows, experts))), min(4, experts)))

    def go(x, w, z, k, wait):
        rows, experts = z.shape().dims
        o = [m.Tensor(x.shape()), m.Tensor(w.shape()), m.Tensor(rows, k), m.IndexTensor(rows, k), m.IndexTensor(experts), m.Tensor(1)]
        m.rms_norm_backward(o[0], o[1], x, x, w, accumulate=False)
        m.group_router_forward(o[2], o[3], o[4], z)
        m.grad_norm(o[5], [x, w, z] * 70)
        if wait:
            m.sync()
        return o

    alone = [[a.to_numpy() for a in go(*s, True)] for s in sets]
    queued = [go(*s, False) for s in sets]
    for a, q in zip(alone, queued):
        for u, v in zip(a, q):
            assert np.array_equal(u, v.to_numpy())


def far(m, rows, width, seed):
    """A tensor of random numbers made on the device, and its last three rows on the host."""
    x = m.Tensor(rows, width)
    m._lib.call("mh_rand_normal", x.ptr, rows * width, seed, 0.0, 2.0)
    last = m.Tensor(3, width)
    m._lib.call("mh_memcpy_d2d", last.ptr, x.ptr + 4 * (rows - 3) * width, 12 * width)
    return x, last


def test_more_than_2_to_31_elements():
    """The last rows of long tensors have the results of a call over them alone."""
    m = GpuEngine().m
    for rows, dim in ((66000, 32768), (550000, 4000)):
        print(f"\n[around] norm {rows} {dim}", flush=True)
        x, last = far(m, rows, dim, 5)
        w, gx = m.Tensor.from_numpy(np.linspace(0.5, 1.5, dim)), m.Tensor(rows, dim)
        small = m.Tensor(3, dim)
        for call in (lambda a, b: m.rms_norm_forward(a, b, w), lambda a, b: m.rms_norm_backward(a, None, b, b, w, accumulate=False)):
            call(gx, x)
            call(small, last)
            end = m.Tensor.over(gx.ptr + 4 * (rows - 3) * dim, (3, dim), gx)
            assert_bitexact(end.to_numpy(), small.to_numpy(), "last rows")
        del gx, x, end
    rows, experts, k = 8500000, 256, 4
    print(f"\n[around] router {rows} {experts}", flush=True)
    z, last = far(m, rows, experts, 6)
    res = [m.Tensor(rows, k), m.IndexTensor(rows, k), m.IndexTensor(experts)]
    m.group_router_forward(*res, z, groups=8, keep_groups=4)
    small = [m.Tensor(3, k), m.IndexTensor(3, k), m.IndexTensor(experts)]
    m.group_router_forward(*small, last, groups=8, keep_groups=4)
    off = 4 * (rows - 3) * k
    assert_bitexact(m.Tensor.over(res[0].ptr + off, (3, k), res[0]).to_numpy(), small[0].to_numpy(), "weights")
    assert np.array_equal(m.IndexTensor.over(res[1].ptr + off, (3, k), res[1]).to_numpy(), small[1].to_numpy())
    assert res[2].to_numpy().astype(np.int64).sum() == rows * k
    gx, gw, sgw = m.Tensor(rows, experts), m.Tensor(rows, k), m.Tensor(3, k)
    m._lib.call("mh_fill", gw.ptr, 0.5, rows * k)
    m._lib.call("mh_fill", sgw.ptr, 0.5, 3 * k)
    sg = m.Tensor(3, experts)
    m.group_router_backward(gx, z, res[1], gw, normalise=False, accumulate=False)
    m.group_router_backward(sg, last, small[1], sgw, normalise=False, accumulate=False)
    assert_bitexact(m.Tensor.over(gx.ptr + 4 * (rows - 3) * experts, (3, experts), gx).to_numpy(), sg.to_numpy(), "gradient")
    del gx, z, res
    rows, classes = 17000, 131072
    print(f"\n[around] sample {rows} {classes}", flush=True)
    x, last = far(m, rows, classes, 7)
    u, p = m.Tensor(rows), m.Tensor(rows)
    m._lib.call("mh_rand_uniform", u.ptr, rows, 8, 0.0, 1.0)
    m._lib.call("mh_fill", p.ptr, 0.8, rows)
    tok, stok = m.IndexTensor(rows), m.IndexTensor(3)
    m.sample_tokens(tok, x, u, top_p=p)
    m.sample_tokens(stok, last, m.Tensor.over(u.ptr + 4 * (rows - 3), (3,), u), top_p=m.Tensor.over(p.ptr, (3,), p))
    assert np.array_equal(tok.to_numpy()[-3:], stok.to_numpy())
    # the whole tensor's norm from its sixteenths', which are of fewer than 2^31
    norm, squares = m.Tensor(1), 0.0
    for i in range(16):
        part = rows * classes // 16
        m.grad_norm(norm, [m.Tensor.over(x.ptr + 4 * part * i, (part,), x)])
        squares += norm[0] ** 2
    m.grad_norm(norm, [x])
    assert abs(norm[0] - np.sqrt(squares)) <= 3 * 2.0 ** -24 * norm[0]
    m.clip_grad_norm(None, [x], 1.0)
    m.grad_norm(norm, [x])
    assert abs(norm[0] - 1.0) <= 1e-6


def test_a_row_as_long_as_a_tensor():
    m = GpuEngine().m
    dim = (1 << 28) + 5  # more parts of 4096 than a grid's second dimension holds
    x, out = m.Tensor(1, dim), m.Tensor(1, dim)
    m._lib.call("mh_fill", x.ptr, 3.0, dim)
    w, gw = m.Tensor(dim), m.Tensor(dim)
    m._lib.call("mh_fill", w.ptr, 2.0, dim)
    m.rms_norm_forward(out, x, w, eps=0.0)
    end = m.Tensor.over(out.ptr + 4 * (dim - 9), (9,), out)
    assert (end.to_numpy() == 2.0).all()
    m.rms_norm_backward(out, gw, x, x, w, eps=0.0, accumulate=False)
    # w g is constant along the row: its part along u is all of it
    assert np.abs(end.to_numpy()).max() <= 4 * 2.0 ** -24 * 2
    assert (m.Tensor.over(gw.ptr + 4 * (dim - 9), (9,), gw).to_numpy() == 3.0).all()
