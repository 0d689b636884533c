"""The vocabulary head's cross entropy at sizes that are cut into several rounds: rows of a forward, elements a thread,
summation lengths."""
import numpy as np
import pytest

from test_gpu_head import check, inputs, m_, reference, run

pytestmark = pytest.mark.gpu


def forward(m, x, w, labels):
    rows = x.shape[0]
    loss, lse, rl = m.Tensor(1), m.Tensor(rows), m.Tensor(rows)
    m.linear_cross_entropy_forward(loss, lse, m.Tensor.from_numpy(x), m.Tensor.from_numpy(w), m.IndexTensor.from_numpy(labels), row_loss=rl)
    return {"loss": loss.to_numpy()[0], "row_lse": lse.to_numpy(), "row_loss": rl.to_numpy()}


def test_forward_cut_by_its_statistics():
    """2^24 classes: 2048 rows at once. Rows of eight kinds, whose results are those of one row of each, bit for bit; those
    against 64 bits."""
    m = m_()
    rows, classes = 2100, (1 << 24) - 5
    r = np.random.RandomState(61)
    kinds = r.standard_normal((8, 2)).astype(np.float32)
    w = r.standard_normal((classes, 2)).astype(np.float32)
    some = r.randint(0, classes, 8).astype(np.int32)
    which = r.randint(0, 8, rows)
    labels = some[which]
    labels[::11] = -1
    print("\n[head] forward in two cuts", flush=True)
    got = forward(m, kinds[which], w, labels)
    keep = labels >= 0
    one, bound = [], []
    for k in range(8):
        want, b = reference(kinds[k:k + 1], w, some[k:k + 1])
        one.append(want)
        bound.append(b)
    for name in ("row_lse", "row_loss"):
        want = np.array([o[name][0] for o in one])[which] * keep
        tol = np.array([b[name][0] for b in bound])[which] * keep
        assert (np.abs(got[name] - want) <= tol).all(), name
        assert not got[name][~keep].any()
        for k in range(8):
            same = got[name][keep & (which == k)]
            assert (same == same[0]).all(), (name, k)
    loss = (np.array([o["row_loss"][0] for o in one])[which] * keep).sum() / keep.sum()
    assert abs(got["loss"] - loss) <= max(b["row_loss"][0] for b in bound)
