"""How far the training-side operators' sums may be off by their real depth: long sums of terms of one sign, whose roundings add
up where they are all made in one 32-bit accumulator."""
import numpy as np
import pytest

import training_reference as ref
from test_gpu_backward_rows import KINDS, run_layernorm_backward

pytestmark = pytest.mark.gpu

U = ref.U


# (rows, columns): through the column kernel alone where there is no workspace, where rows are shorter than a vector and where they
# are longer than the registers; else through the row kernel
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(786432, 24), (200000, 40), (300001, 3), (70000, 130), (6000, 17000)])
def test_column_sums_over_many_rows(ko, rows, cols, kind):
    rng = np.random.default_rng(rows + cols)
    dy, dy64 = ref.to_storage(rng.uniform(0.5, 1.0, (rows, cols)).astype(np.float32), kind)
    x, x64 = ref.to_storage(rng.uniform(1.0, 2.0, (rows, cols)).astype(np.float32), kind)
    mean, rstd = np.full(rows, 0.25, np.float32), np.full(rows, 1.5, np.float32)
    want_g, want_b = (dy64 * ((x64 - 0.25) * 1.5)).sum(0), dy64.sum(0)
    for workspace in (True, False):
        _, dgamma, dbeta = run_layernorm_backward(ko, dy, x, mean, rstd, kind, workspace=workspace)
        # without a workspace: eight terms in 32 bits, then 64, and one rounding.  With one: eight terms likewise, or a lane group's
        # rows one after the other (512 workgroups of 4 wavefronts with 8 lane groups of 8 lanes: rows / 16384; rows of 130 columns
        # 16 to 64 lanes, rows / 2048 at least), 32 lane groups, and the partial rows, eight of them in turn and a tree of 64 lanes
        depth = 8 + 1 if not workspace else max(8, rows / (16384 if cols <= 64 else 2048)) + 32 + 8 + 6
        # xh carries two roundings, its product with dy one
        ref.assert_within(dgamma, want_g, (depth + 3) * U * want_g, "dgamma, workspace %s" % workspace)
        ref.assert_within(dbeta, want_b, depth * U * want_b, "dbeta, workspace %s" % workspace)


# scale log2(e) as one 32-bit number is off by 1e-9 of itself for scale 1; for these by at least 0.9 of half a step
def _awkward_scale(near):
    log2e = 1.4426950408889634
    for scale in np.float32(near) + np.arange(2000, dtype=np.float32) * np.spacing(np.float32(near)):
        c = float(scale) * log2e
        step = float(np.spacing(np.float32(c)))
        if 0.45 * step <= abs(float(np.float32(c)) - c) and c < 1.1 * 2.0 ** np.floor(np.log2(c)):
            return float(scale)
    raise AssertionError("no such scale")


@pytest.mark.parametrize("level", [0.0, 20.0, -60.0])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [30522, 128256])
def test_log_probabilities_are_differences_of_more_than_32_bits(ko, cols, kind, level):
    """A KL term sees the log-probability before it is rounded: kl(d) with d = reference - logp near 0.4 moves by 0.49 of logp's
    error.  At labels of logp about -24 a logarithm in 32 bits is off by up to half a step of numbers from 16 to 32, 9.5e-7, 5.5e-7 in
    root mean square, and scale log2(e) in one 32-bit number by 5.7e-8 of the distance from the label to where the other columns'
    weight lies, some 14, or of the logits' level where that is not taken off first, the same way in every row: 2.7e-7 and 4e-7 of kl.
    What the kernels may be off by, of kl: d's own rounding 1.5e-8 at most, three roundings of kl around 0.09 2e-8 at most, a bias of half
    a step in the exponentials 1.5e-8; the sums (32 bits in a few hundred threads) below 1e-8: root mean square below 4e-8.  Their
    arguments' rounding is 5.5e-7 in root mean square for arguments from 16 to 32 (3.8e-7 of a column's weight), and as
    many of them are independent as there are different logits: in fp32 thousands (below 1e-8 of kl); in bf16 numbers from 16 to 32 are
    1/8 apart, and a normal distribution's weight of standard deviation 1.2 lies on 1.2 2 sqrt(pi) 8 = 34 of them: 3.2e-8 of kl, and
    as it is the same draw for all rows, twice that is allowed for.  (Numbers beyond 32, 1/4 apart: 17 of them, 4.5e-8.)"""
    rows = 48
    rng = np.random.default_rng(cols)
    scale = _awkward_scale(0.7)
    x = rng.normal(level, 1.2, (rows, cols)).astype(np.float32)
    labels = rng.integers(0, cols, rows).astype(np.int32)
    at = np.arange(rows)
    x[at, labels] = level + rng.uniform(-20.0, -18.0, rows)
    stored, values = ref.to_storage(x, kind)
    z = values * scale
    top = z.max(1)
    logp = z[at, labels] - top - np.log(np.exp(z - top[:, None]).sum(1))
    assert -30 < logp.min() and logp.max() < -16
    reference = (logp + 0.4).astype(np.float32)
    d = reference.astype(np.float64) - logp
    want = np.expm1(d) - d
    bufs = [ko.DeviceBuffer.from_numpy(a) for a in (stored, labels, reference, np.zeros(rows, np.float32))]
    loss, kl, grad = ko.DeviceBuffer(4 * rows), ko.DeviceBuffer(4 * rows), ko.DeviceBuffer(stored.nbytes)
    n = ko.token_logprob_workspace_bytes(rows, cols)
    ws = ko.DeviceBuffer(max(n, 16))
    typed = {} if kind == "f32" else dict(dtype=ko.BF16)
    op = ko.policy_loss if kind == "f32" else ko.policy_loss16
    for gradient, work in ((True, False), (False, False), (True, True)):
        op(bufs[0], bufs[1], bufs[3], loss, rows, cols, ref_logp=bufs[2], scale=scale, kl=kl, dlogits=grad if gradient else None,
           workspace=ws if work and n else None, workspace_bytes=n if work else 0, **typed)
        ko.synchronize()
        off = kl.download(np.float32, (rows,)) - want
        rms = np.sqrt((off ** 2).mean())
        assert rms < 4e-8 + (0.0 if kind == "f32" or level == 0.0 else 2 * (3.2e-8 if level == 20.0 else 4.5e-8)), (gradient, work, rms)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1001, 9001, 70001])
def test_all_but_certain_labels(ko, cols, kind):
    """A label 20 to 30 above the others: logp is minus their sum, relative to the label.  From the sum relative to the largest of the
    others that is one factor of exp(-16 to -26), whose argument in 32 bits would put 3.8e-7 in root mean square on all of logp (half
    a step of numbers from 16 to 64 in base 2, 9.5e-7 or more).  What may be off: logp's own rounding and that of its series 3e-8
    each in root mean square, a hardware exponential 3e-8, the sum 2e-8 (bf16: the arguments of some hundred different logits, 0 to 8
    below the maximum, 1.4e-7 by the square root of fifty): below 7e-8 together."""
    rows = 60
    rng = np.random.default_rng(cols + 7)
    x = rng.normal(0.0, 1.0, (rows, cols)).astype(np.float32)
    labels = rng.integers(0, cols, rows).astype(np.int32)
    at = np.arange(rows)
    x[at, labels] = rng.uniform(20.0, 30.0, rows)
    stored, values = ref.to_storage(x, kind)
    others = np.exp(values - values[at, labels][:, None])
    others[at, labels] = 0.0
    want = -np.log1p(others.sum(1))
    bufs = [ko.DeviceBuffer.from_numpy(a) for a in (stored, labels, np.zeros(rows, np.float32))]
    logp, loss, grad = ko.DeviceBuffer(4 * rows), ko.DeviceBuffer(4 * rows), ko.DeviceBuffer(rows * (cols + 1) * 4)
    n = ko.token_logprob_workspace_bytes(rows, cols)
    ws = ko.DeviceBuffer(max(n, 16))
    typed = {} if kind == "f32" else dict(dtype=ko.BF16)
    score, policy = (ko.token_logprob, ko.policy_loss) if kind == "f32" else (ko.token_logprob16, ko.policy_loss16)
    forms = dict(score=lambda w: score(bufs[0], bufs[1], logp, rows, cols, **w, **typed),
                 policy=lambda w: policy(bufs[0], bufs[1], bufs[2], loss, rows, cols, logp=logp, dlogits=grad, **w, **typed),
                 alone=lambda w: policy(bufs[0], bufs[1], bufs[2], loss, rows, cols, logp=logp, **w, **typed),
                 apart=lambda w: policy(bufs[0], bufs[1], bufs[2], loss, rows, cols, logp=logp, dlogits=grad, ldd=cols + 1, **w, **typed))
    for name, run in forms.items():
        for w in ({}, dict(workspace=ws, workspace_bytes=n)):
            run(w)
            ko.synchronize()
            off = logp.download(np.float32, (rows,)) / want - 1.0
            rms = np.sqrt((off ** 2).mean())
            assert rms < 1e-7, (name, bool(w), rms)
