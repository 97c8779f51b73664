"""Rows of logits far from 0 and rows with values that are no numbers, in every form of the token losses: each form is named by
the sizes and arguments that lead to it."""
import numpy as np
import pytest

import training_reference as ref
from test_gpu_backward_rows import KINDS, Out
from test_gpu_token_loss import Call, check_policy, policy_case, run_policy

pytestmark = pytest.mark.gpu


class FarScores(ref.Scores):
    """Scores whose log-probabilities stay finite where the label's probability is below the smallest 64-bit number."""

    def __init__(self, logits, labels, scale=1.0, alive=None):
        with np.errstate(over="ignore"):
            super().__init__(logits, labels, scale, alive)
        z = self.z[self.rows, self.at]
        with np.errstate(invalid="ignore"):
            far = z - np.log(np.exp(self.z).sum(1))
        self.logp = np.where(self.alive & (z < -30.0), far, self.logp)


def far_call(ko, rows, cols, kind, scale, magnitudes, seed, pad=0, workspace=True):
    """Every row around one of +-magnitudes: all columns the same, some steps of the type apart, or one column above the rest;
    the label among the largest or not."""
    call = Call(ko, rows, cols, kind, seed, pad, 0, workspace, scale)
    rng = np.random.default_rng(seed + 1)
    at = np.arange(rows)
    level = (np.array(magnitudes, np.float64)[at % len(magnitudes)] * np.where(at // len(magnitudes) % 2, -1.0, 1.0))[:, None]
    bits = {"f32": 24, "f16": 11, "bf16": 8}[kind]
    step = 2.0 ** (np.floor(np.log2(np.abs(level))) + 1 - bits)       # the type's distance of numbers there
    way = (at // (2 * len(magnitudes)) % 3)[:, None]
    x = np.zeros((rows, call.ld))
    x[:, :cols] = level + np.where(way == 1, step * rng.integers(0, 4, (rows, cols)), 0.0)
    label = np.maximum(call.labels, 0)
    one = (label + (at % 2)) % cols                                   # the label's column or the next one
    x[at, one] += np.where(way[:, 0] == 2, 8 * step[:, 0], 0.0)
    x[call.labels < 0] = np.nan
    x[:, cols:] = np.nan
    call.stored, values = ref.to_storage(x, kind)
    call.values = values[:, :cols]
    assert np.isfinite(call.values[call.labels >= 0]).all()
    call.keep.upload(call.stored)
    call.scores = FarScores(call.values, call.labels, scale)
    return call


# rows of one wavefront and of workgroups, whole and cut into pieces, eight to a wavefront, longer than the registers
FAR_SHAPES = [(47, 19), (95, 1001), (53, 9001), (47, 33000), (47, 70001), (70, 70001), (16391, 40), (32779, 37)]


@pytest.mark.parametrize("kind,scale,magnitudes", [("f32", 1 / 0.7, [3e5, 1e6, 3e6, 1e7, 1e8, 1e9, 1e10]),
                                                   ("f32", 10.0, [1e5, 1e7, 4e7, 1e12]), ("f32", 0.8, [1e9, 1e20]),
                                                   ("bf16", 1 / 0.7, [1e6, 1e9, 1e12, 1e20]), ("f16", 1e5, [5.0, 70.0, 3000.0, 6e4])])
@pytest.mark.parametrize("rows,cols", FAR_SHAPES)
def test_logprob_of_rows_far_from_zero(ko, rows, cols, kind, scale, magnitudes):
    """The label's logit times scale log2(e) is rounded before it is taken off the others': far from 0 by more than their
    differences."""
    call = far_call(ko, rows, cols, kind, scale, magnitudes, 4000 + cols)
    s = call.scores
    # each column's exponential may be flushed to 0 below 2^-126; where the label is all but certain logp is minus their sum
    off = s.logp_off + cols * 2.0 ** -126
    logp, stats = call.logprob()
    ref.assert_within(logp, s.logp, off, "logp")
    np.testing.assert_array_equal(stats[:, 0], s.top.astype(np.float32))
    ref.assert_within(stats[:, 1], s.logsum, s.logsum_off + cols * 2.0 ** -126, "log sum")
    case = policy_case(call, cols, False, False)
    for pad, gradient in ((0, True), (1, True), (0, False)):
        got = run_policy(call, case, pad, gradient=gradient, kl_coef=0.0)
        ref.assert_within(got["logp"], s.logp, off, "logp of the policy loss")


# (beyond 1e30 the differences from the row's maximum were taken first, below nothing is lost)
@pytest.mark.parametrize("kind,scale,magnitudes", [("f32", 1.0, [1e6, 1e7, 1e8, 1e9, 4e9, 1e10, 1e12, 1e20, 1e32]),
                                                   ("f32", 1 / 0.7, [4e9, 1e10, 3e29, 1e30]), ("f32", 1e-10, [1e17, 1e20, 1e24]),
                                                   ("bf16", 1.0, [1e8, 1e10, 1e20, 1e35]), ("bf16", 1 / 0.7, [4e9, 1e12]),
                                                   ("f16", 1e6, [100.0, 4e3, 6e4]), ("f16", 1e20, [1.0, 6e4])])
@pytest.mark.parametrize("rows,cols", FAR_SHAPES)
def test_policy_gradient_of_rows_far_from_zero(ko, rows, cols, kind, scale, magnitudes):
    """With ratio 1 and no KL term the gradient is -advantage scale (onehot - softmax): with a large scale beyond binary16's
    numbers, then it is infinite."""
    call = far_call(ko, rows, cols, kind, scale, magnitudes, 4100 + cols)
    case = policy_case(call, cols, False, False, False)
    first = {}
    for pad in (1, 0):
        got = run_policy(call, case, pad, kl_coef=0.0)
        first["dlogits"] = got["dlogits"]
        d = ref.to_float(np.ascontiguousarray(got.pop("dlogits")), kind)
        check_policy(call, got, case, 0.0)
        alive = call.labels >= 0
        want, off = call.scores.gradient(np.where(alive, -case["advantage"].astype(np.float64), 0.0), 0.0, call.scores.s_off)
        off = off + ref.rounded(kind, want) * (1 + 1e-6)
        # (65520 rounds to infinity)
        large, beyond = (np.abs(want) - off >= 65520, np.abs(want) + off >= 65520) if kind == "f16" else (want != want, want != want)
        assert (d[large] == np.copysign(np.inf, want[large])).all()
        either = beyond & ~large & np.isinf(d)
        assert (np.sign(d[either]) == np.sign(want[either])).all()
        ref.assert_within(d[~large & ~either], want[~large & ~either], off[~large & ~either], "dlogits")
        assert not d[~alive].any()
    got = run_policy(call, case, 0, in_place=True, kl_coef=0.0)
    np.testing.assert_array_equal(got["dlogits"], first["dlogits"])


def test_a_masked_row_with_a_label(ko):
    """All columns at -1e10, by every length that a workgroup's registers are cut for: the gradient is that of a uniform row."""
    for cols in (33, 300, 700, 2000, 4100, 8200, 16500, 33000, 65536, 66000):
        x = np.full((70, cols), -1e10, np.float32)
        labels = (np.arange(70) * 37 % cols).astype(np.int32)
        bufs = [ko.DeviceBuffer.from_numpy(a) for a in (x, labels, np.ones(70, np.float32))]
        loss, d = ko.DeviceBuffer(4 * 70), ko.DeviceBuffer(x.nbytes)
        ko.policy_loss(bufs[0], bufs[1], bufs[2], loss, 70, cols, dlogits=d)
        ko.synchronize()
        want = np.full((70, cols), 1.0 / cols)
        want[np.arange(70), labels] -= 1.0
        # the sum of ones is exact to the last step (whole numbers below 2^24), then a division and a product
        np.testing.assert_allclose(d.download(np.float32, x.shape), want, rtol=8 * ref.U)


# the policy loss's forms: (rows, columns, padding of the gradient's rows, with a gradient, with a workspace)
POLICY_FORMS = [(41, 1001, 0, True, True), (41, 9001, 0, True, True), (41, 1001, 1, True, True), (41, 9001, 0, False, True),
                (7, 70001, 0, True, True), (7, 70001, 0, False, True), (7, 70001, 0, True, False), (70, 70001, 0, True, True),
                (32779, 37, 0, True, True), (5, 3, 0, True, True)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,pad,gradient,workspace", POLICY_FORMS)
def test_an_impossible_label_of_the_policy_that_trains(ko, rows, cols, pad, gradient, workspace, kind):
    """Without old log-probabilities the ratio is 1, also for a label at -inf: the loss is -advantage, and the gradient takes
    weight from the other columns."""
    call = Call(ko, rows, cols, kind, 4300 + cols, 0, 0, workspace)
    live = np.flatnonzero(call.labels >= 0)
    lost = live[::3]
    x = np.where((call.labels >= 0)[:, None], call.values, np.nan).astype(np.float32)
    x[lost, call.labels[lost]] = -np.inf
    call.stored, call.values = ref.to_storage(x, kind)
    call.keep.upload(call.stored)
    with np.errstate(divide="ignore"):
        call.scores = ref.Scores(call.values, call.labels)
    case = policy_case(call, 14, False, False)
    got = run_policy(call, case, pad, gradient=gradient, kl_coef=0.0)
    assert (got["logp"][lost] == -np.inf).all()
    call.scores.logp[lost] = 0.0        # (the ratio does not depend on it)
    rest = np.setdiff1d(np.arange(rows), lost)
    want = ref.policy(call.scores, np.where(call.labels >= 0, case["advantage"], 1.0), None, None,
                      np.where(call.labels >= 0, case["weight"], 1.0), 0.2, 0.28, 0.0)
    for name in ("loss", "loss_sum"):
        ref.assert_within(got[name], *want[name], name)
    ref.assert_within(got["logp"][rest], want["logp"][0][rest], want["logp"][1][rest], "logp")
    if gradient:
        call.check_gradient(got["dlogits"], want["dlogits"])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,pad,gradient,workspace", POLICY_FORMS)
def test_no_advantage_hides_no_broken_row(ko, rows, cols, pad, gradient, workspace, kind):
    """A NaN or +inf logit, or a label beyond the vocabulary, makes a row's outputs and gradient NaN also where its advantage is 0
    and no KL term counts; a sound row without advantage has loss and gradient 0."""
    call = Call(ko, rows, cols, kind, 4200 + cols, 0, 0, workspace)
    alive = call.labels >= 0
    case = policy_case(call, 13)
    case["advantage"][alive] = 0.0
    x = np.where(alive[:, None], call.values, np.nan).astype(np.float32)
    bad = np.flatnonzero(alive)[:4]
    assert len(bad) >= 3
    call.labels[bad[0]] = cols
    x[bad[1], cols // 2] = np.nan
    x[bad[2], (call.labels[bad[2]] + 1) % cols] = np.inf
    if len(bad) > 3:
        x[bad[3], call.labels[bad[3]]] = np.inf
    for name in ("old", "ref"):
        case[name][bad] = -1.0
    call.keep.upload(ref.to_storage(x, kind)[0])
    call.d_labels.upload(call.labels)
    sound = np.setdiff1d(np.arange(rows), bad)
    for old, reference in ((True, True), (True, False), (False, False)):
        given = dict(case, old=case["old"] if old else None, ref=case["ref"] if reference else None)
        got = run_policy(call, given, pad, gradient=gradient, kl_coef=0.0)
        assert np.isnan(got["logp"][bad]).all() and np.isnan(got["loss"][bad]).all() and np.isnan(got["loss_sum"]).all()
        assert not got["loss"][sound].any() and np.isfinite(got["logp"][sound]).all()
        if reference:
            assert np.isnan(got["kl"][bad]).all()
        if gradient:
            d = ref.to_float(np.ascontiguousarray(got["dlogits"]), kind)
            assert np.isnan(d[bad]).all() and not d[sound].any()


@pytest.mark.parametrize("pairs", [1, 4, 7, 40])
def test_preference_loss_of_certain_pairs(ko, pairs):
    """A chosen or rejected token of probability 0 puts the rewards infinitely far apart: a side whose share of the loss is 0
    adds nothing."""
    tokens = 2 * pairs
    offsets = np.arange(tokens + 1, dtype=np.int32)
    rf = np.full(tokens, -1.0, np.float32)
    bufs = [ko.DeviceBuffer.from_numpy(a) for a in (rf, offsets)]
    for side, sign in ((0, -1.0), (1, 1.0)):        # the chosen or the rejected token is the impossible one: margin -inf or inf
        logp = np.full(tokens, -1.0, np.float32)
        logp[side::2] = -np.inf
        d_logp = ko.DeviceBuffer.from_numpy(logp)
        for eps, want in ((0.0, 0.0 if sign > 0 else np.inf), (1.0, np.inf if sign > 0 else 0.0), (0.5, np.inf)):
            loss, dlogp, total = Out(ko, 4 * pairs), Out(ko, 4 * tokens), Out(ko, 4)
            ko.preference_loss(d_logp, bufs[0], bufs[1], pairs, tokens, loss.ptr, beta=0.5, label_smoothing=eps, pair_weight=1.0,
                               dlogp=dlogp.ptr, loss_sum=total.ptr)
            ko.synchronize()
            assert (loss.get(np.float32, (pairs,)) == want).all(), (sign, eps)
            assert total.get(np.float32, (1,))[0] == want * pairs if want else total.get(np.float32, (1,))[0] == 0.0
            slope = 0.5 * (eps - (1.0 if sign < 0 else 0.0))       # d loss / d margin, times beta
            np.testing.assert_array_equal(dlogp.get(np.float32, (tokens,)), np.tile([slope, -slope], pairs))


def _random_offsets(pairs, back, seed):
    """Offsets that run forwards on the whole and backwards by up to `back` at every turn, some of them far out."""
    rng = np.random.default_rng(seed)
    offsets = 7 * np.arange(2 * pairs + 1) + rng.integers(-back, back + 1, 2 * pairs + 1)
    wild = rng.random(2 * pairs + 1) < 0.5 / (pairs + 1)
    offsets[wild] = rng.choice([-2 ** 31, -5, 2 ** 31 - 1], int(wild.sum()))
    if pairs > 2:
        offsets[[2, 4]] = offsets[[4, 2]]
    return offsets.astype(np.int32)


@pytest.mark.parametrize("labelled", [True, False])
@pytest.mark.parametrize("pairs,back", [(1, 40), (2, 9), (3, 30), (7, 0), (16, 12), (17, 12), (300, 25), (1024, 9), (1025, 9), (9001, 100),
                                        (30000, 0)])
def test_pairs_that_share_tokens(ko, pairs, back, labelled):
    """Offsets that go backwards between pairs: rewards and losses are those of a pair's own offsets; a pair writes the gradient
    from the largest offset before it on, so that no token is written twice, and the same bits come from call to call."""
    tokens = 14 * pairs - 3
    offsets = _random_offsets(pairs, back, pairs)
    rng = np.random.default_rng(pairs + 1)
    logp, rf = rng.normal(-2, 1, tokens).astype(np.float32), rng.normal(-2, 1, tokens).astype(np.float32)
    labels = np.where(rng.random(tokens) < 0.2, -1, 7).astype(np.int32) if labelled else None
    want = ref.preference(logp, rf, offsets, labels, 0.3, 0.1)
    slope, touched = np.zeros(tokens), np.zeros(tokens, bool)
    most = np.clip(np.maximum.accumulate(offsets.astype(np.int64)), 0, tokens)
    share = float(np.float32(0.3)) * float(np.float32(1.0 / pairs))
    for p in range(pairs):
        at = np.clip(np.maximum.accumulate(np.maximum(offsets[2 * p:2 * p + 3].astype(np.int64), 0)), 0, tokens)
        margin = want["rewards"][0][2 * p] - want["rewards"][0][2 * p + 1]
        up = (float(np.float32(0.1)) - 1.0 / (1.0 + np.exp(margin))) * share
        begin = most[2 * p]
        slope[begin:max(begin, at[1])], slope[max(begin, at[1]):max(begin, at[2])] = up, -up
        touched[begin:max(begin, at[2])] = True
    if labels is not None:
        slope[labels < 0] = 0.0
    d = [ko.DeviceBuffer.from_numpy(a) for a in (logp, rf, offsets)]
    d_labels = None if labels is None else ko.DeviceBuffer.from_numpy(labels)
    before = None
    for _ in range(3):
        outs = dict(pair_loss=Out(ko, 4 * pairs), rewards=Out(ko, 8 * pairs), dlogp=Out(ko, 4 * tokens), loss_sum=Out(ko, 4))
        ko.preference_loss(d[0], d[1], d[2], pairs, tokens, outs["pair_loss"].ptr, labels=d_labels, beta=0.3, label_smoothing=0.1,
                           rewards=outs["rewards"].ptr, dlogp=outs["dlogp"].ptr, loss_sum=outs["loss_sum"].ptr)
        ko.synchronize()
        for name, n in (("pair_loss", pairs), ("rewards", 2 * pairs), ("loss_sum", 1)):
            ref.assert_within(outs[name].get(np.float32, (n,)), *want[name], name)
        raw = outs["dlogp"].get(np.uint32, (tokens,))
        assert (raw[~touched] == 0xFFFFFFFF).all()
        ref.assert_within(raw.view(np.float32)[touched], slope[touched], (2 * ref.U * np.abs(slope) + 1e-13)[touched], "dlogp")
        if before is not None:
            np.testing.assert_array_equal(raw, before)
        before = raw


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,pad", [(41, 90, 0), (41, 1001, 0), (41, 1001, 1), (30, 9001, 0), (7, 70001, 0), (16391, 40, 0),
                                           (16391, 600, 0)])
def test_broken_rows_of_every_type(ko, rows, cols, pad, kind):
    """NaN and infinite logits and labels beyond the vocabulary stay in their own rows, in log-probabilities, statistics and
    gradients; the gradient takes the statistics that the forward call left."""
    call = Call(ko, rows, cols, kind, 4400 + cols, 0, 4)
    live = np.flatnonzero(call.labels >= 0)
    bad = live[:4]
    x = np.where((call.labels >= 0)[:, None], call.values, np.nan).astype(np.float32)
    x[bad[0], cols // 2] = np.nan
    x[bad[1], (call.labels[bad[1]] + 1) % cols] = np.inf
    x[bad[2], call.labels[bad[2]]] = np.nan
    call.labels[bad[3]] = 2 ** 31 - 1
    call.keep.upload(np.concatenate([np.zeros(4, np.uint8), ref.to_storage(x, kind)[0].reshape(-1).view(np.uint8)]))
    call.d_labels.upload(call.labels)
    sound = np.setdiff1d(np.arange(rows), bad)
    logp, stats = call.logprob()
    s = call.scores
    assert np.isnan(logp[bad]).all() and np.isnan(stats[bad, 1]).all()
    ref.assert_within(logp[sound], s.logp[sound], s.logp_off[sound], "logp")
    dlogp = np.linspace(-1.0, 1.0, rows).astype(np.float32) + np.float32(0.01)
    s.top, s.logsum = stats[:, 0].astype(np.float64), stats[:, 1].astype(np.float64)
    got = ref.to_float(np.ascontiguousarray(call.backward(dlogp, pad)), kind)
    assert np.isnan(got[bad]).all()
    value, off = s.gradient(dlogp.astype(np.float64), 0.0, s.logsum_off + 3 * ref.U * np.abs(s.logsum) + 2 * ref.U)
    off = off + ref.rounded(kind, value) * (1 + 1e-6)
    ref.assert_within(got[sound], value[sound], off[sound], "dlogits")
