"""Gradients of the row softmax and of LayerNorm against their formulas in 64 bits, at bounds derived in
training_reference.py."""
import numpy as np
import pytest

import training_reference as ref
from kernel_optimization_amd import inputs

pytestmark = pytest.mark.gpu

KINDS = ["f32", "f16", "bf16"]
GUARD = 64  # bytes behind every output and workspace that have to stay as they were


class Out:
    """A device output with guard bytes behind it; starts full of NaN bit patterns."""

    def __init__(self, ko, nbytes, skew=0):
        self.buf = ko.DeviceBuffer.from_numpy(np.full(skew + nbytes + GUARD, 0xFF, np.uint8))
        self.nbytes, self.skew = nbytes, skew
        self.ptr = self.buf.ptr + skew

    def get(self, dtype, shape):
        raw = self.buf.download(np.uint8, (self.skew + self.nbytes + GUARD,))
        assert (raw[:self.skew] == 0xFF).all() and (raw[self.skew + self.nbytes:] == 0xFF).all(), "written outside"
        return raw[self.skew:self.skew + self.nbytes].view(dtype).reshape(shape)


def skewed(ko, a, skew):
    """Device copy of `a` that starts `skew` bytes behind an aligned address: (buffer to keep, address)."""
    raw = np.concatenate([np.zeros(skew, np.uint8), np.ascontiguousarray(a).view(np.uint8).reshape(-1)])
    buf = ko.DeviceBuffer.from_numpy(raw)
    return buf, buf.ptr + skew


def dtype_of(kind):
    return np.float32 if kind == "f32" else np.uint16


def _softmax(x):
    e = np.exp(x - x.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


def run_softmax_backward(ko, y, dy, kind, valid_len=None, rps=0, workspace=True, in_place=None, skew=0):
    rows, cols = y.shape
    keep_y, py = skewed(ko, y, skew)
    keep_dy, pdy = skewed(ko, dy, skew)
    out = Out(ko, y.nbytes, skew)
    target = {None: out.ptr, "y": py, "dy": pdy}[in_place]
    dv = None if valid_len is None else ko.DeviceBuffer.from_numpy(np.asarray(valid_len, np.int32))
    n = ko.softmax_backward_workspace_bytes(rows, cols) if workspace else 0
    ws = Out(ko, n) if n else None
    kw = dict(valid_len=dv, rows_per_seq=rps, workspace=ws.ptr if ws else None, workspace_bytes=n)
    if kind == "f32":
        ko.softmax_backward(py, pdy, target, rows, cols, **kw)
    else:
        ko.softmax_backward16(py, pdy, target, rows, cols, dtype=ko.F16 if kind == "f16" else ko.BF16, **kw)
    ko.synchronize()
    if ws:
        ws.get(np.uint8, (n,))
    if in_place:
        return (keep_y if in_place == "y" else keep_dy).download(dtype_of(kind), y.shape, skew)
    return out.get(dtype_of(kind), y.shape)


def check_softmax_backward(ko, y, dy, kind, valid_len=None, rps=0, **kw):
    got = run_softmax_backward(ko, y, dy, kind, valid_len, rps, **kw)
    want, off = ref.softmax_backward(ref.to_float(y, kind), ref.to_float(dy, kind), valid_len, rps)
    ref.assert_within(ref.to_float(got, kind), want, off + ref.rounded(kind, want) * (1 + 1e-6), "dx")
    return got


# one column to rows that are cut into pieces; both sides of every mapping's border, whole vectors and not
SOFTMAX_SHAPES = [(1, 1), (3, 7), (70, 8), (5, 64), (64, 128), (9, 129), (33, 200), (7, 513), (5, 1000), (4, 1024), (3, 1025),
                  (3, 2048), (2, 4100), (3, 8192), (2, 16384), (2, 16385), (2, 33000), (3, 40000), (1, 70001), (70, 66000)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", SOFTMAX_SHAPES)
def test_softmax_backward(ko, rows, cols, kind):
    y, _ = ref.to_storage(_softmax(inputs.normal_f32((rows, cols), 900 + cols, 0.0, 4.0).astype(np.float64)), kind)
    dy, _ = ref.to_storage(inputs.normal_f32((rows, cols), 901 + cols), kind)
    got = check_softmax_backward(ko, y, dy, kind)
    np.testing.assert_array_equal(run_softmax_backward(ko, y, dy, kind), got)  # the same bits from call to call
    np.testing.assert_array_equal(run_softmax_backward(ko, y, dy, kind, in_place="dy"), got)
    np.testing.assert_array_equal(run_softmax_backward(ko, y, dy, kind, in_place="y"), got)
    check_softmax_backward(ko, y, dy, kind, workspace=False)
    check_softmax_backward(ko, y, dy, kind, skew=4)  # off 16-byte boundaries


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,rps", [(40, 8, 1), (40, 37, 3), (33, 200, 4), (24, 512, 5), (20, 1000, 3), (12, 4100, 2),
                                           (12, 8192, 1), (9, 20000, 1), (6, 70000, 1)])
def test_softmax_backward_masked(ko, rows, cols, rps, kind):
    """Lengths of nothing, one column, whole rows and the columns around vectors; beyond the valid columns dy is NaN and
    must not be looked at."""
    nseq = (rows + rps - 1) // rps
    lens = np.array([[0, 1, cols, cols - 1, 8, 9, 7, -3, cols + 5, cols // 2, 64][i % 11] for i in range(nseq)], np.int32)
    x = inputs.normal_f32((rows, cols), 910 + cols, 0.0, 4.0).astype(np.float64)
    keep = ref.keep_columns(rows, cols, lens, rps)
    y = np.where(keep, x, -10000.0)
    y, y64 = ref.to_storage(_softmax(y), kind)
    dy = inputs.normal_f32((rows, cols), 911 + cols)
    dy[~keep & (y64 == 0)] = np.nan
    dy, _ = ref.to_storage(dy, kind)
    got = check_softmax_backward(ko, y, dy, kind, lens, rps)
    assert not ref.to_float(got, kind)[~keep].any()
    np.testing.assert_array_equal(run_softmax_backward(ko, y, dy, kind, lens, rps, in_place="dy"), got)
    np.testing.assert_array_equal(run_softmax_backward(ko, y, dy, kind, lens, rps, in_place="y"), got)
    check_softmax_backward(ko, y, dy, kind, lens, rps, workspace=False)
    check_softmax_backward(ko, y, dy, kind, lens, rps, skew=4)


@pytest.mark.parametrize("cols", [40, 600, 5000, 20000, 70000])
def test_softmax_backward_where_the_padding_has_weight(ko, cols):
    """Valid scores around -9998: exp(x - max) of the padding (-10000) is not 0, and its dy counts."""
    rows = 6
    lens = np.array([cols // 2, 1, cols - 1, cols, 0, cols // 3], np.int32)
    x = inputs.normal_f32((rows, cols), 920, -9998.0, 1.0).astype(np.float64)
    keep = ref.keep_columns(rows, cols, lens, 1)
    y, y64 = ref.to_storage(_softmax(np.where(keep, x, -10000.0)), "f32")
    assert (y64[~keep] > 0).all()
    dy, _ = ref.to_storage(inputs.normal_f32((rows, cols), 921), "f32")
    for workspace in (True, False):
        check_softmax_backward(ko, y, dy, "f32", lens, 1, workspace=workspace)


def test_softmax_backward_special_values(ko):
    """A NaN in one row's dy stays in that row."""
    for cols in (100, 128, 3000, 70000):
        y, _ = ref.to_storage(_softmax(inputs.normal_f32((4, cols), 930, 0.0, 2.0).astype(np.float64)), "f32")
        dy = inputs.normal_f32((4, cols), 931)
        dy[2, cols // 2] = np.nan
        got = run_softmax_backward(ko, y, dy, "f32")
        assert np.isnan(got[2]).all() and np.isfinite(got[[0, 1, 3]]).all()


# ---- LayerNorm

def run_layernorm_backward(ko, dy, x, mean, rstd, kind, gamma=None, dres=None, unbiased=False, workspace=True, in_place=None,
                           skew=0, want_gamma=True, want_beta=True):
    rows, cols = x.shape
    keep = [skewed(ko, a, skew) if a is not None else (None, None) for a in (dy, x, dres, gamma)]
    out = Out(ko, x.nbytes, skew)
    target = {None: out.ptr, "dy": keep[0][1], "x": keep[1][1], "dres": keep[2][1]}[in_place]
    dm, dr = ko.DeviceBuffer.from_numpy(mean.astype(np.float32)), ko.DeviceBuffer.from_numpy(rstd.astype(np.float32))
    dg, db = Out(ko, cols * 4), Out(ko, cols * 4)
    n = ko.layernorm_backward_workspace_bytes(rows, cols) if workspace else 0
    ws = Out(ko, n) if n else None
    kw = dict(gamma=keep[3][1], dres=keep[2][1], dgamma=dg.ptr if want_gamma else None, dbeta=db.ptr if want_beta else None,
              unbiased=unbiased, workspace=ws.ptr if ws else None, workspace_bytes=n)
    args = (keep[0][1], keep[1][1], dm, dr, target, rows, cols)
    if kind == "f32":
        ko.layernorm_backward(*args, **kw)
    else:
        ko.layernorm_backward16(*args, dtype=ko.F16 if kind == "f16" else ko.BF16, **kw)
    ko.synchronize()
    if ws:
        ws.get(np.uint8, (n,))
    sums = [o.get(np.uint32, (cols,)).view(np.float32) if w else None for o, w in ((dg, want_gamma), (db, want_beta))]
    if not want_gamma:
        assert (dg.get(np.uint8, (cols * 4,)) == 0xFF).all()
    if not want_beta:
        assert (db.get(np.uint8, (cols * 4,)) == 0xFF).all()
    if in_place:
        dx = keep[{"dy": 0, "x": 1, "dres": 2}[in_place]][0].download(dtype_of(kind), x.shape, skew)
    else:
        dx = out.get(dtype_of(kind), x.shape)
    return dx, sums[0], sums[1]


def layernorm_case(rows, cols, kind, seed, affine=True, residual=True, unbiased=False):
    x, x64 = ref.to_storage(inputs.normal_f32((rows, cols), seed, 0.5, 2.0), kind)
    dy, _ = ref.to_storage(inputs.normal_f32((rows, cols), seed + 1), kind)
    gamma = ref.to_storage(inputs.normal_f32((cols,), seed + 2, 1.0, 0.1), kind)[0] if affine else None
    dres = ref.to_storage(inputs.normal_f32((rows, cols), seed + 3), kind)[0] if residual else None
    mean = x64.mean(1).astype(np.float32)
    d = max(1, cols - 1) if unbiased else cols
    rstd = (1 / np.sqrt(((x64 - x64.mean(1, keepdims=True)) ** 2).sum(1) / d + 1e-5)).astype(np.float32)
    return dict(dy=dy, x=x, mean=mean, rstd=rstd, gamma=gamma, dres=dres, unbiased=unbiased)


def check_layernorm_backward(ko, case, kind, **kw):
    got = run_layernorm_backward(ko, kind=kind, **case, **kw)
    f = lambda a: None if a is None else ref.to_float(a, kind)
    want, off = ref.layernorm_backward(f(case["dy"]), f(case["x"]), case["mean"].astype(np.float64),
                                       case["rstd"].astype(np.float64), f(case["gamma"]), f(case["dres"]), case["unbiased"])
    ref.assert_within(f(got[0]), want[0], off[0] + ref.rounded(kind, want[0]) * (1 + 1e-6), "dx")
    for g, w, o, name in zip(got[1:], want[1:], off[1:], ("dgamma", "dbeta")):
        if g is not None:
            ref.assert_within(g, w, o, name)
    return got


LAYERNORM_SHAPES = [(1, 1), (2, 2), (3, 7), (130, 8), (5, 64), (64, 128), (9, 129), (33, 200), (100, 768), (7, 513), (5, 1000),
                    (3001, 72), (900, 1001), (4, 1024), (3, 1025), (2, 2048), (2, 2049), (1500, 2304), (2, 4104), (3, 8192),
                    (2, 8193), (2, 16384), (600, 4096), (2, 16392), (3, 40000), (1, 70001), (1, 300)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", LAYERNORM_SHAPES)
def test_layernorm_backward(ko, rows, cols, kind):
    unbiased = cols % 3 == 2
    case = layernorm_case(rows, cols, kind, 1000 + cols, unbiased=unbiased)
    got = check_layernorm_backward(ko, case, kind)
    for a, b in zip(run_layernorm_backward(ko, kind=kind, **case), got):
        np.testing.assert_array_equal(a, b)                    # the same bits from call to call
    for place in ("dy", "x", "dres"):
        for a, b in zip(run_layernorm_backward(ko, kind=kind, **case, in_place=place), got):
            np.testing.assert_array_equal(a, b, err_msg=place)
    check_layernorm_backward(ko, case, kind, workspace=False)
    check_layernorm_backward(ko, case, kind, workspace=False, in_place="dy")
    check_layernorm_backward(ko, case, kind, skew=4)           # off 16-byte boundaries
    check_layernorm_backward(ko, layernorm_case(rows, cols, kind, 1500 + cols, False, False), kind)


@pytest.mark.parametrize("cols", [64, 768, 4096, 20000])
def test_layernorm_backward_optional_results(ko, cols):
    case = layernorm_case(37, cols, "f32", 1100)
    full = check_layernorm_backward(ko, case, "f32")
    for g, b in ((True, False), (False, True), (False, False)):
        for workspace in (True, False):
            got = check_layernorm_backward(ko, case, "f32", want_gamma=g, want_beta=b, workspace=workspace)
            np.testing.assert_array_equal(got[0], full[0])


def test_layernorm_backward_no_rows(ko):
    """The sum over no rows is 0."""
    dg, db = Out(ko, 400), Out(ko, 400)
    ko.layernorm_backward(None, None, None, None, None, 0, 100, dgamma=dg.ptr, dbeta=db.ptr)
    ko.synchronize()
    assert not dg.get(np.float32, (100,)).any() and not db.get(np.float32, (100,)).any()


@pytest.mark.parametrize("cols", [64, 768, 1001, 4096, 20000])
def test_layernorm_backward_special_values(ko, cols):
    """A NaN row (its mean and rstd are NaN then) poisons its dx and the sums over the rows, no other row's dx."""
    case = layernorm_case(9, cols, "f32", 1200)
    case["mean"][4] = case["rstd"][4] = np.nan
    dx, dgamma, dbeta = run_layernorm_backward(ko, kind="f32", **case)
    others = np.arange(9) != 4
    assert np.isnan(dx[4]).all() and np.isfinite(dx[others]).all()
    assert np.isnan(dgamma).all() and np.isfinite(dbeta).all()


def test_layernorm_backward_follows_the_forward_call(ko):
    """mean and rstd as the library's forward pass leaves them, against differences of the forward formula."""
    rows, cols = 6, 40
    x = inputs.normal_f32((rows, cols), 1300, 0.5, 2.0)
    gamma, beta = inputs.normal_f32((cols,), 1301, 1.0, 0.1), inputs.normal_f32((cols,), 1302)
    dy = inputs.normal_f32((rows, cols), 1303)
    _, mean, rstd = ko.layernorm_host(x, gamma, beta, eps=1e-5, unbiased=True)
    dx, dgamma, dbeta = run_layernorm_backward(ko, dy, x, mean, rstd, "f32", gamma=gamma, unbiased=True)

    def loss(v, g, b):
        d = v - v.mean(1, keepdims=True)
        return ((d / np.sqrt((d * d).sum(1, keepdims=True) / (cols - 1) + 1e-5) * g + b) * dy).sum()

    x64, g64, b64 = x.astype(np.float64), gamma.astype(np.float64), beta.astype(np.float64)
    step = 1e-5
    for got, at in ((dx, 0), (dgamma, 1), (dbeta, 2)):
        args = [x64, g64, b64]
        for i in np.ndindex(*args[at].shape):
            hi, lo = [a.copy() for a in args], [a.copy() for a in args]
            hi[at][i] += step
            lo[at][i] -= step
            num = (loss(*hi) - loss(*lo)) / (2 * step)
            # the forward gate on mean and rstd (1e-5 of their scale) times sums of six to forty terms of size 1 to 3
            assert abs(num - got[i]) <= 1e-4 * max(1.0, abs(num)), (at, i, num, got[i])


# both sides of the forms for few rows (up to 256 of them: one launch), rows of three and four vectors per thread of the largest
# workgroup, and rows shorter than a vector
@pytest.mark.parametrize("rows,cols,kind", [(256, 136, "bf16"), (257, 136, "bf16"), (256, 2056, "f32"), (257, 2056, "f32"),
                                            (40, 9000, "f32"), (300, 12288, "f32"), (40, 12300, "f32"), (3, 16384, "f32"),
                                            (3, 16400, "f32"), (1025, 5, "f16"), (700, 3, "f32"), (20000, 24, "f32"),
                                            (3000, 768, "bf16"), (2049, 1536, "f16"), (520, 4096, "bf16")])
def test_layernorm_backward_borders(ko, rows, cols, kind):
    case = layernorm_case(rows, cols, kind, 1700 + cols)
    got = check_layernorm_backward(ko, case, kind)
    for place in ("dy", "x"):
        for a, b in zip(run_layernorm_backward(ko, kind=kind, **case, in_place=place), got):
            np.testing.assert_array_equal(a, b, err_msg=place)
    check_layernorm_backward(ko, case, kind, workspace=False)
    check_layernorm_backward(ko, case, kind, skew=4)


def test_backward_workspaces_stay_small():
    """Sizes that a caller can always allocate: 64 MB at most, whatever the shape."""
    import kernel_optimization_amd as ko
    for rows in (1, 2, 300, 100000, 1 << 30):
        for cols in (1, 7, 768, 16384, 16385, 100000, 1 << 30):
            assert ko.layernorm_backward_workspace_bytes(rows, cols) <= 64 << 20
            assert ko.softmax_backward_workspace_bytes(rows, cols) <= 64 << 20
            assert ko.token_logprob_workspace_bytes(rows, cols) <= 64 << 20
