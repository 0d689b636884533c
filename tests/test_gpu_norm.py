"""Root-mean-square norm with the residual's addition (rms_norm_*) against the formulas in 64 bits.

Tolerances, U = 2^-24. The sum x + residual is one rounding: equal bits. The scale is a 64-bit value rounded to fp32
(U), u = h scale and out = u w a rounding each: 3 U of out. In the backward w g is a rounding (U), so mean(w g u) is off by
U mean |w g u| and its own rounding; u by 2 U, u mean and the difference by a rounding each, the scale and its product by
two, the sums with grad_sum and what was there by one each. A sum over rows makes `depth` additions: rows / 1024 a lane
(at most 1024 workgroups), 7 over the lanes of a workgroup, 128 + 8 over the workgroups; its terms are off by 3 U."""
import numpy as np
import pytest

from util import GpuEngine, assert_bitexact

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TINY = 1e-44  # a subnormal result's rounding


def m_():
    return GpuEngine().m


def reference(h, w, eps, g=None, gsum=None):
    hd, wd = h.astype(np.float64), w.astype(np.float64)
    s = 1.0 / np.sqrt((hd * hd).mean(-1, keepdims=True) + float(np.float32(eps)))
    u = hd * s
    out = {"out": u * wd}
    bound = {"out": 3.1 * U * np.abs(out["out"]) + TINY}
    if g is None:
        return out, bound
    gd = g.astype(np.float64)
    wg = gd * wd
    mean = (wg * u).mean(-1, keepdims=True)
    gx = s * (wg - u * mean)
    off = s * (4 * np.abs(wg) + 7 * np.abs(u * mean) + np.abs(u) * np.abs(wg * u).mean(-1, keepdims=True)) * 1.01 * U
    if gsum is not None:
        gx = gx + gsum
    out["grad_x"], bound["grad_x"] = gx, off + 1.1 * U * np.abs(gx) + TINY
    rows = h.reshape(-1, h.shape[-1]).shape[0]
    depth = min(rows, rows // 1024 + 150) + 3
    axes = tuple(range(h.ndim - 1))
    out["grad_w"], bound["grad_w"] = (gd * u).sum(axes), (depth + 1) * U * np.abs(gd * u).sum(axes) + TINY
    return out, bound


def check(got, want, bound, what=""):
    for k, v in want.items():
        off = np.abs(got[k].astype(np.float64) - v)
        assert np.isfinite(got[k]).all(), f"{what} {k}: not finite"
        over = off > bound[k]
        assert not over.any(), f"{what} {k}: {over.sum()} of {over.size} beyond the bound, worst {off.max():.3g}"


def inputs(shape, seed, std=1.0):
    r = np.random.RandomState(seed)
    f = lambda *s: r.standard_normal(s).astype(np.float32)  # noqa: E731
    return {"x": (std * f(*shape)).astype(np.float32), "res": (std * f(*shape)).astype(np.float32),
            "w": (1 + 0.2 * f(shape[-1])).astype(np.float32), "g": f(*shape), "gsum": f(*shape)}


def run(m, d, eps=1e-5, residual=True, gsum=True, accumulate=None):
    T = m.Tensor.from_numpy
    t = {k: T(v) for k, v in d.items()}
    shape = d["x"].shape
    out, total = m.Tensor(shape), m.Tensor(shape)
    m.rms_norm_forward(out, t["x"], t["w"], residual=t["res"] if residual else None, sum=total, eps=eps)
    gx, gw = (T(np.full(shape, 7.0)), T(np.full(shape[-1], 7.0))) if accumulate is None else (T(accumulate[0]), T(accumulate[1]))
    m.rms_norm_backward(gx, gw, t["g"], total, t["w"], grad_sum=t["gsum"] if gsum else None, eps=eps,
                        accumulate=accumulate is not None)
    return {"out": out.to_numpy(), "sum": total.to_numpy(), "grad_x": gx.to_numpy(), "grad_w": gw.to_numpy()}


SIZES = [(1, 1), (3, 2), (5, 3), (1, 4), (70, 5), (300, 16), (257, 17), (100, 32), (1000, 33), (65, 64), (129, 65), (66, 128),
         (77, 130), (9, 255), (200, 257), (64, 512), (1023, 513), (33, 768), (7, 1000), (40, 1024), (3, 1025), (1100, 1500),
         (5, 2047), (1030, 2048), (6, 2051), (1, 4096), (19, 4097), (3, 8192), (4, 8200), (2, 16384), (3, 16385), (70, 20001), (1, 40000),
         (70000, 8)]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size):
    print(f"\n[norm] {size}", flush=True)
    d = inputs(size, seed=sum(size))
    got = run(m_(), d)
    h = d["x"] + d["res"]
    assert_bitexact(got["sum"], h, "sum")
    check(got, *reference(h, d["w"], 1e-5, d["g"], d["gsum"]), what=str(size))


@pytest.mark.parametrize("shape", [(2, 3, 40), (4, 1, 2, 600), (5,)], ids=str)
def test_ranks(shape):
    d = inputs(shape, seed=7)
    got = run(m_(), d, residual=False, gsum=False)
    assert_bitexact(got["sum"], d["x"], "sum")
    check(got, *reference(d["x"], d["w"], 1e-5, d["g"]), what=str(shape))


@pytest.mark.parametrize("size", [(40, 100), (9, 1000), (5, 3000), (4, 20000)], ids=str)
def test_gradients_are_added(size):
    d = inputs(size, seed=3)
    r = np.random.RandomState(4)
    was = r.standard_normal(size).astype(np.float32), r.standard_normal(size[1]).astype(np.float32)
    got = run(m_(), d, accumulate=was)
    want, bound = reference(d["x"] + d["res"], d["w"], 1e-5, d["g"], d["gsum"])
    for k, a in (("grad_x", was[0]), ("grad_w", was[1])):
        bound[k] = bound[k] + 1.1 * U * np.abs(want[k] + a)
        want[k] = want[k] + a
    check(got, want, bound, "added")


@pytest.mark.parametrize("size", [(40, 100), (5, 3000), (3, 10000), (4, 20000)], ids=str)
def test_one_gradient_alone(size):
    m, d = m_(), inputs(size, seed=5)
    want, bound = reference(d["x"], d["w"], 1e-5, d["g"])
    T = m.Tensor.from_numpy
    x, w, g = T(d["x"]), T(d["w"]), T(d["g"])
    gx, gw = m.Tensor(size), m.Tensor(size[1])
    m.rms_norm_backward(gx, None, g, x, w, eps=1e-5, accumulate=False)
    m.rms_norm_backward(None, gw, g, x, w, eps=1e-5, accumulate=False)
    check({"grad_x": gx.to_numpy(), "grad_w": gw.to_numpy()}, {k: want[k] for k in ("grad_x", "grad_w")}, bound)
    m.rms_norm_backward(None, None, g, x, w)


@pytest.mark.parametrize("size", [(40, 100), (6, 1000), (5, 3000), (4, 20000)], ids=str)
def test_in_place(size):
    """The sum over the residual or x, the output over x, the gradient over those of the sum or the output."""
    m, d = m_(), inputs(size, seed=6)
    T = m.Tensor.from_numpy
    ref = run(m, d)
    for total_at in ("res", "x", None):
        for out_at in ("x", None):
            if out_at == total_at == "x":
                continue
            t = {k: T(v) for k, v in d.items()}
            out = t["x"] if out_at else m.Tensor(size)
            total = m.Tensor(size) if total_at is None else t[total_at]
            m.rms_norm_forward(out, t["x"], t["w"], residual=t["res"], sum=total, eps=1e-5)
            assert_bitexact(out.to_numpy(), ref["out"], f"{out_at} {total_at}")
            assert_bitexact(total.to_numpy(), ref["sum"], f"{out_at} {total_at}")
    for at in ("gsum", "g"):
        t = {k: T(v) for k, v in d.items()}
        gw = m.Tensor(size[1])
        m.rms_norm_backward(t[at], gw, t["g"], T(ref["sum"]), t["w"], grad_sum=t["gsum"], eps=1e-5, accumulate=False)
        assert_bitexact(t[at].to_numpy(), ref["grad_x"], at)
        assert_bitexact(gw.to_numpy(), ref["grad_w"], at)


@pytest.mark.parametrize("std", [1e-20, 1e19, 1e37])
@pytest.mark.parametrize("size", [(20, 40), (5, 3000), (3, 20000)], ids=str)
def test_sizes_of_elements(size, std):
    """Squares that fp32 does not hold."""
    d = inputs(size, seed=8, std=std)
    d["gsum"][:] = 0
    got = run(m_(), d, eps=0.0)
    want, bound = reference(d["x"] + d["res"], d["w"], 0.0, d["g"], d["gsum"])
    check(got, want, bound, str(std))


@pytest.mark.parametrize("size", [(20, 40), (5, 3000), (2, 9000), (3, 20000)], ids=str)
def test_scales_past_the_range(size):
    """1 / sqrt(mean h^2) above the largest float, and below the least normal one."""
    r = np.random.RandomState(18)
    d = inputs(size, seed=18, std=1e-41)
    d["g"] = (1e-12 * d["g"]).astype(np.float32)
    d["gsum"][:] = 0
    large = dict(d, x=np.where(r.uniform(size=size) < 0.5, -3.3e38, 3.3e38).astype(np.float32), g=inputs(size, seed=19)["g"])
    large["res"] = np.zeros(size, np.float32)
    for what, e in (("small", d), ("large", large)):
        got = run(m_(), e, eps=0.0)
        want, bound = reference(e["x"] + e["res"], e["w"], 0.0, e["g"], e["gsum"])
        check(got, want, bound, what)


def test_rows_of_zeros_and_of_no_numbers():
    m = m_()
    for size in ((6, 50), (6, 1000), (6, 3000), (6, 20000)):
        d = inputs(size, seed=9)
        d["x"][1] = d["res"][1] = 0.0
        d["x"][3, -1] = np.nan
        d["x"][4, 0] = np.inf
        got = run(m, d)
        h = d["x"] + d["res"]
        fine = [0, 1, 2, 5]
        want, bound = reference(h[fine], d["w"], 1e-5, d["g"][fine], d["gsum"][fine])
        check({k: got[k][fine] for k in ("out", "grad_x")}, {k: want[k] for k in ("out", "grad_x")}, bound, str(size))
        assert (got["out"][1] == 0).all()
        assert np.isnan(got["out"][3]).all() and np.isnan(got["grad_x"][3]).all()
        assert np.isnan(got["out"][4, 0]) and (got["out"][4, 1:] == 0).all()
        assert np.isnan(got["grad_w"]).any()
        # eps 0: a row of zeros has no direction
        assert np.isnan(run(m, d, eps=0.0)["out"][1]).all()


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_any_alignment(offset):
    """Tensors that begin 4, 8 and 12 bytes past a 16-byte boundary."""
    m = m_()
    for size in ((30, 64), (7, 1024), (4, 2049), (3, 17000)):
        d = inputs(size, seed=10)
        n = size[0] * size[1]

        def at(a):
            buf = m.Tensor.from_numpy(np.concatenate([np.full(offset, 9.0), a.reshape(-1), np.full(8, 9.0)]))
            return buf, m.Tensor.over(buf.ptr + 4 * offset, a.shape, buf)

        t = {k: at(v) for k, v in d.items()}
        o = {k: at(np.zeros(size, np.float32)) for k in ("out", "sum", "grad_x")}
        gw = at(np.zeros(size[1], np.float32))
        m.rms_norm_forward(o["out"][1], t["x"][1], t["w"][1], residual=t["res"][1], sum=o["sum"][1], eps=1e-5)
        m.rms_norm_backward(o["grad_x"][1], gw[1], t["g"][1], o["sum"][1], t["w"][1], grad_sum=t["gsum"][1], eps=1e-5, accumulate=False)
        ref = run(m, d)
        for k in o:
            whole = o[k][0].to_numpy()
            assert_bitexact(whole[offset:offset + n].reshape(size), ref[k], k)
            assert (whole[:offset] == 9).all() and (whole[offset + n:] == 9).all()
        assert_bitexact(gw[0].to_numpy()[offset:offset + size[1]], ref["grad_w"], "grad_w")


def test_gradients_against_differences():
    """The derivative along a direction, from differences of the formula in 64 bits."""
    size, eps = (11, 37), 1e-3
    d = inputs(size, seed=11)
    got = run(m_(), d, eps=eps)
    r = np.random.RandomState(12)
    dx, dw = r.standard_normal(size), r.standard_normal(size[1])

    def value(k):
        h = d["x"].astype(np.float64) + d["res"] + k * dx
        out = h / np.sqrt((h * h).mean(1, keepdims=True) + float(np.float32(eps))) * (d["w"] + k * dw)
        return (out * d["g"]).sum() + (h * d["gsum"]).sum()

    k = 1e-4
    slope = (8 * (value(k) - value(-k)) - (value(2 * k) - value(-2 * k))) / (12 * k)
    mine = (got["grad_x"] * dx).sum() + (got["grad_w"] * dw).sum()
    scale = np.abs(got["grad_x"] * dx).sum() + np.abs(got["grad_w"] * dw).sum()
    assert abs(slope - mine) < 40 * U * scale, (slope, mine)


def test_no_rows():
    m = m_()
    gw, w = m.Tensor.from_numpy(np.full(5, 3.0)), m.Tensor.from_numpy(np.ones(5))
    a, b = m.Tensor((0, 5)), m.Tensor((0, 5))
    m.rms_norm_forward(a, b, w)
    m.rms_norm_backward(a, gw, b, b, w)
    assert (gw.to_numpy() == 3).all()
    m.rms_norm_backward(a, gw, b, b, w, accumulate=False)
    assert (gw.to_numpy() == 0).all()


def test_the_same_bits_on_every_call():
    m, d = m_(), inputs((5000, 300), seed=13)
    a, b = run(m, d), run(m, d)
    for k in a:
        assert_bitexact(a[k], b[k], k)
