"""The norm of many gradients, their clipping, and Adam with it (grad_norm, clip_grad_norm, Adam(max_norm=)) against
64 bits.

Tolerances, U = 2^-24. The squares are added in 64 bits (n 2^-53 of the sum, which is nothing here): the norm is one rounding,
1.01 U of itself. A clipped gradient is c = max_norm / norm rounded (U), times g (U): 2.01 U. Adam with clipping has the bits of
clipping and Adam."""
import ctypes

import numpy as np
import pytest

from util import GpuEngine, assert_bitexact

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def m_():
    return GpuEngine().m


def norm_of(arrays):
    return np.sqrt(sum((a.astype(np.float64) ** 2).sum() for a in arrays))


def tensors(m, arrays):
    return [m.Tensor.from_numpy(a) for a in arrays]


def some(sizes, seed, std=1.0):
    r = np.random.RandomState(seed)
    return [(std * r.standard_normal(n)).astype(np.float32) for n in sizes]


SIZES = [[1], [3], [4], [4095], [4096], [4097], [8192, 1, 4100], [100003], [5, 0, 7], list(range(1, 40)), [33] * 161, [1] * 500,
         [3000000], [1 << 20, 3, 1 << 18, 77]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
def test_norm_and_clip(sizes):
    print(f"\n[clip] {len(sizes)} {sizes[:4]}", flush=True)
    m, g = m_(), some(sizes, seed=len(sizes))
    t, norm = tensors(m, g), m.Tensor(1)
    want = norm_of(g)
    m.grad_norm(norm, t)
    assert abs(norm[0] - want) <= 1.01 * U * want
    for part in (0.3, 1.0, 1.5):
        t = tensors(m, g)
        top = float(np.float32(part * want))
        m.clip_grad_norm(norm, t, top)
        assert abs(norm[0] - want) <= 1.01 * U * want
        for a, b in zip(t, g):
            if part > 1:
                assert_bitexact(a.to_numpy(), b, "unclipped")
            else:
                c = min(1.0, top / want)
                assert (np.abs(a.to_numpy() - c * b.astype(np.float64)) <= 2.01 * U * np.abs(b) * c + 1e-45).all()


def test_none_and_empty():
    m, norm = m_(), m_().Tensor.from_numpy(np.float32([5]))
    m.grad_norm(norm, [])
    assert norm[0] == 0
    e = m.Tensor((0,))
    m.clip_grad_norm(norm, [e, e], 1.0)
    assert norm[0] == 0
    m.clip_grad_norm(None, [], 1.0)
    opt = m.Adam([], max_norm=1.0)
    opt.step()
    assert opt.grad_norm[0] == 0


@pytest.mark.parametrize("std", [1e-30, 1e30, 3e-44])
def test_sizes_of_elements(std):
    """Squares that fp32 does not hold; a norm past fp32's largest is infinite, and clips all the same."""
    m, g = m_(), some([1000, 77], seed=1, std=std)
    t, norm = tensors(m, g), m.Tensor(1)
    m.clip_grad_norm(norm, t, 1.0)
    want = norm_of(g)
    assert abs(norm[0] - want) <= 1.01 * U * want + 1e-45
    c = min(1.0, 1.0 / want)
    for a, b in zip(t, g):
        assert (np.abs(a.to_numpy() - c * b.astype(np.float64)) <= 2.01 * U * np.abs(b) * c + 1e-45).all()
    big = [np.full(1000, 3e38, np.float32)]
    t = tensors(m, big)
    m.clip_grad_norm(norm, t, 2.0)
    assert norm[0] == np.inf
    c = 2.0 / norm_of(big)  # a subnormal in fp32: half of the least, relative to it
    assert (np.abs(t[0].to_numpy() - c * big[0].astype(np.float64)) <= 3e38 * 2.0 ** -150 * 1.01 + 2 * U * 3e38 * c).all()


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_no_number_scales_nothing(bad):
    m, g = m_(), some([5000, 300], seed=2)
    g[1][7] = bad
    t, norm = tensors(m, g), m.Tensor(1)
    m.clip_grad_norm(norm, t, 0.5)
    assert np.isnan(norm[0]) if np.isnan(bad) else norm[0] == np.inf
    for a, b in zip(t, g):
        assert_bitexact(a.to_numpy(), b, "unscaled")


def test_limits():
    m, g = m_(), some([100], seed=3)
    for top, want in ((float("inf"), g[0]), (0.0, 0 * g[0])):
        t = tensors(m, g)
        m.clip_grad_norm(None, t, top)
        assert np.array_equal(t[0].to_numpy(), want)
    z, norm = m.Tensor(50), m.Tensor(1)
    m.clip_grad_norm(norm, [z], 0.0)
    assert norm[0] == 0 and (z.to_numpy() == 0).all()


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_any_alignment(offset):
    m = m_()
    for n in (1, 2, 5, 4096, 9001):
        a = some([n], seed=n)[0]
        buf = m.Tensor.from_numpy(np.concatenate([np.full(offset, 9.0), a, np.full(8, 9.0)]))
        t, norm = m.Tensor.over(buf.ptr + 4 * offset, (n,), buf), m.Tensor(1)
        m.clip_grad_norm(norm, [t], 0.25)
        want = norm_of([a])
        assert abs(norm[0] - want) <= 1.01 * U * want
        whole = buf.to_numpy()
        assert (whole[:offset] == 9).all() and (whole[offset + n:] == 9).all()
        assert (np.abs(whole[offset:offset + n] - min(1, 0.25 / want) * a) <= 2.01 * U * np.abs(a)).all()


def test_tensors_in_any_order_and_neighbours():
    """Neighbours in an arena share no elements, in whatever order they are given."""
    m = m_()
    a = some([1000], seed=4)[0]
    arena, norm = m.Tensor.from_numpy(a), m.Tensor(1)
    cuts = [0, 10, 11, 300, 999, 1000]
    parts = [m.Tensor.over(arena.ptr + 4 * p, (q - p,), arena) for p, q in zip(cuts, cuts[1:])]
    m.clip_grad_norm(norm, [parts[i] for i in (3, 0, 4, 1, 2)], 1.0)
    want = norm_of([a])
    assert (np.abs(arena.to_numpy() - a / want) <= 2.01 * U * np.abs(a / want)).all()
    # the norm alone may count one twice
    t = m.Tensor.from_numpy(a)
    m.grad_norm(norm, [t, t])
    assert abs(norm[0] - np.sqrt(2) * want) <= 2 * U * want


SETS = [[50], [4096], [1 << 20], [1000, 7, 0, 333], [64] * 90, [100001, 3]]


@pytest.mark.parametrize("clipped", [True, False])
@pytest.mark.parametrize("sizes", SETS, ids=lambda s: f"{len(s)}x{s[0]}")
def test_adam_has_the_bits_of_the_two_calls(sizes, clipped):
    m = m_()
    p, g = some(sizes, seed=5), some(sizes, seed=6)
    top = float(np.float32(norm_of(g) * (0.2 if clipped else 3.0)))
    one = m.Adam(list(zip(tensors(m, p), tensors(m, g))), lr=0.01, max_norm=top)
    two = m.Adam(list(zip(tensors(m, p), tensors(m, g))), lr=0.01)
    norm = m.Tensor(1)
    for _ in range(3):
        one.step()
        for (_, a), b in zip(two.params, g):  # as the first call found them
            m._lib.call("mh_memcpy_h2d", a.ptr, b.ctypes.data, 4 * b.size)
        m.clip_grad_norm(norm, [a for _, a in two.params], top)
        two.step()
    assert one.grad_norm[0] == norm[0]
    for (a, ga), (b, _), gn in zip(one.params, two.params, g):
        assert_bitexact(a.to_numpy(), b.to_numpy(), "parameters")
        assert_bitexact(ga.to_numpy(), gn, "the gradients stay")
    for a, b in zip((*one.momentum_grads, *one.rms_grads), (*two.momentum_grads, *two.rms_grads)):
        assert_bitexact(a.to_numpy(), b.to_numpy(), "state")


def test_adam_of_a_model():
    m = m_()
    r = np.random.RandomState(7)
    x = r.standard_normal((20, 30)).astype(np.float32)

    def model():
        g = m.Graph()
        i = g.input((20, 30))
        w, b = g.param((1, 30), init=np.linspace(-1, 1, 30).reshape(1, 30)), g.param((20, 1), init=np.ones((20, 1)))
        g.loss(g.op(m.OP.SUM, g.op(m.OP.MUL, g.op(m.OP.ADD, i, b), w)))
        mod = m.Model(g)
        mod.forward(x)
        mod.parameters.grads.set_zero()
        mod.backward()
        return mod, (w, b)

    (one, syms), (two, _) = model(), model()
    grads = [two.parameters.grads[s] for s in syms]
    want = norm_of([g.to_numpy() for g in grads])
    a, b = m.Adam(one.parameters, max_norm=0.5), m.Adam(two.parameters)
    a.step()
    m.clip_grad_norm(None, grads, 0.5)
    b.step()
    assert abs(a.grad_norm[0] - want) <= 1.01 * U * want
    for s in syms:
        assert_bitexact(one.parameters.tensors[s].to_numpy(), two.parameters.tensors[s].to_numpy(), "parameters")
    a.grad_norm = None  # goes without
    a.step()


def test_misaligned_memory_is_refused():
    m = m_()
    t = m.Tensor(100)
    ptrs, sizes = (ctypes.c_void_p * 1)(t.ptr + 2), (ctypes.c_int64 * 1)(10)
    with pytest.raises(m.MantleHipError) as e:
        m._lib.call("mh_grad_norm", 1, ptrs, sizes, t.ptr)
    assert e.value.code == m._lib.ERR_INVALID


def test_the_same_bits_on_every_call():
    m, g = m_(), some([1 << 22, 12345], seed=8)
    t, norm = tensors(m, g), m.Tensor(1)
    seen = set()
    for _ in range(3):
        m.grad_norm(norm, t)
        seen.add(norm[0])
    assert len(seen) == 1
