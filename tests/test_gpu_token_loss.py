"""Token log-probabilities, the clipped policy loss and the preference loss against their formulas in 64 bits, at bounds
derived in training_reference.py."""
import numpy as np
import pytest

import training_reference as ref
from kernel_optimization_amd import inputs
from test_gpu_backward_rows import KINDS, Out, dtype_of, skewed

pytestmark = pytest.mark.gpu

# one column to a whole vocabulary; few rows (cut into pieces) and more rows than compute units
SHAPES = [(1, 1), (2, 2), (5, 7), (3, 100), (300, 33), (4, 1001), (300, 1024), (33, 5003), (150, 4096), (200, 8200), (6, 30522),
          (130, 16390), (5, 50257), (2, 128256), (140, 66000), (1, 200001)]


def make_rows(rows, cols, ld, kind, seed):
    """Stored logits [rows, ld], their values [rows, cols], labels: some rows without one (NaN logits there), likely and
    unlikely labels, -inf and lowest-value masks.  What lies between the rows is NaN."""
    x = inputs.normal_f32((rows, ld), seed, 0.0, 2.0)
    rng = np.random.default_rng(seed)
    labels = rng.integers(0, cols, rows).astype(np.int32)
    r = np.arange(rows)
    x[r, labels] += rng.choice([0.0, 8.0, 25.0], rows).astype(np.float32)
    lowest = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3895314e38}[kind]
    for row in range(rows):
        if row % 5 == 1 and cols > 2:  # half of the vocabulary masked, the label's column among the rest
            cut = rng.random(cols) < 0.5
            cut[labels[row]] = False
            x[row, :cols][cut] = -np.inf if row % 2 else lowest
    dead = (rng.random(rows) < 0.2) & (r > 0)
    labels[dead] = -1 - rng.integers(0, 100, int(dead.sum())).astype(np.int32)
    x[dead] = np.nan
    x[:, cols:] = np.nan
    stored, values = ref.to_storage(x, kind)
    return stored, values[:, :cols], labels


class Call:
    """Device copies of one call's inputs."""

    def __init__(self, ko, rows, cols, kind, seed, pad=0, skew=0, workspace=True, scale=1.0):
        self.ko, self.rows, self.cols, self.kind, self.skew, self.scale = ko, rows, cols, kind, skew, scale
        self.ld = cols + pad
        self.stored, self.values, self.labels = make_rows(rows, cols, self.ld, kind, seed)
        self.keep, self.logits = skewed(ko, self.stored, skew)
        self.d_labels = ko.DeviceBuffer.from_numpy(self.labels)
        self.bytes = ko.token_logprob_workspace_bytes(rows, cols) if workspace else 0
        self.ws = Out(ko, self.bytes) if self.bytes else None
        self.kw = dict(ld=self.ld, scale=scale)
        self.typed = {} if kind == "f32" else dict(dtype=ko.F16 if kind == "f16" else ko.BF16)
        self.work = dict(workspace=self.ws.ptr if self.ws else None, workspace_bytes=self.bytes)
        self.scores = ref.Scores(self.values, self.labels, scale)

    def op(self, name):
        return getattr(self.ko, name + ("" if self.kind == "f32" else "16"))

    def logprob(self):
        logp, stats = Out(self.ko, 4 * self.rows), Out(self.ko, 8 * self.rows)
        self.op("token_logprob")(self.logits, self.d_labels, logp.ptr, self.rows, self.cols, row_stats=stats.ptr, **self.kw,
                                 **self.typed, **self.work)
        self.ko.synchronize()
        if self.ws:
            self.ws.get(np.uint8, (self.bytes,))
        return logp.get(np.float32, (self.rows,)), stats.get(np.float32, (self.rows, 2))

    def check_logprob(self):
        logp, stats = self.logprob()
        s = self.scores
        ref.assert_within(logp, s.logp, s.logp_off, "logp")
        np.testing.assert_array_equal(stats[:, 0], s.top.astype(np.float32))
        ref.assert_within(stats[:, 1], s.logsum, s.logsum_off, "log sum")
        return logp, stats

    def gradient_out(self, pad, in_place):
        """(address, function that fetches [rows, cols] and checks that nothing between the rows changed)"""
        size = self.stored.itemsize
        ldd = self.cols + pad
        if in_place:
            before = self.stored

            def fetch():
                got = self.keep.download(dtype_of(self.kind), before.shape, self.skew)
                np.testing.assert_array_equal(got[:, self.cols:], before[:, self.cols:])
                return got[:, :self.cols]
            return self.logits, self.ld, fetch
        out = Out(self.ko, self.rows * ldd * size, self.skew)

        def fetch():
            got = out.get(dtype_of(self.kind), (self.rows, ldd))
            assert (np.ascontiguousarray(got[:, self.cols:]).view(np.uint8) == 0xFF).all()
            return got[:, :self.cols]
        return out.ptr, ldd, fetch

    def backward(self, dlogp, pad, in_place=False):
        s = self.scores
        stats = np.stack([s.top, s.logsum], 1).astype(np.float32)
        d_stats, d_dlogp = self.ko.DeviceBuffer.from_numpy(stats), self.ko.DeviceBuffer.from_numpy(dlogp)
        ptr, ldd, fetch = self.gradient_out(pad, in_place)
        self.op("token_logprob_backward")(self.logits, self.d_labels, d_stats, d_dlogp, ptr, self.rows, self.cols, ldd=ldd,
                                          **self.kw, **self.typed)
        self.ko.synchronize()
        return fetch()

    def check_gradient(self, got, want):
        value, off = want
        ref.assert_within(ref.to_float(np.ascontiguousarray(got), self.kind), value,
                          off + ref.rounded(self.kind, value) * (1 + 1e-6), "dlogits")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_token_logprob_and_its_gradient(ko, rows, cols, kind):
    for pad, skew, scale, workspace in ((0, 0, 1.0, True), (3, 4, 0.625, True), (8, 0, 1.5, False)):
        call = Call(ko, rows, cols, kind, 2000 + cols, pad, skew, workspace, scale)
        logp, stats = call.check_logprob()
        again = call.logprob()
        np.testing.assert_array_equal(again[0], logp)          # the same bits from call to call
        np.testing.assert_array_equal(again[1], stats)
        dlogp = inputs.normal_f32((rows,), 2001 + cols)
        dlogp[rows // 2] = 0.0
        # the log sum handed over is rounded to fp32 and multiplied once
        want = call.scores.gradient(dlogp.astype(np.float64), 0.0, 3 * ref.U * np.abs(call.scores.logsum) + 2 * ref.U)
        got = call.backward(dlogp, pad)
        call.check_gradient(got, want)
        assert not ref.to_float(np.ascontiguousarray(got), kind)[(call.labels < 0) | (dlogp == 0)].any()
        call.check_gradient(call.backward(dlogp, pad + 1), want)   # rows that lie differently: element by element
        np.testing.assert_array_equal(call.backward(dlogp, pad, in_place=True), got)


def policy_case(call, seed, old=True, reference=True, weight=True):
    rows, s = call.rows, call.scores
    rng = np.random.default_rng(seed)
    shift = rng.choice([-0.6, -0.3, -0.1, -0.01, 0.0, 0.02, 0.1, 0.2, 0.35, 0.9], rows) + rng.uniform(0, 1e-3, rows)
    case = dict(advantage=rng.normal(0, 1, rows).astype(np.float32))
    case["advantage"][rows // 3] = 0.0
    case["old"] = (s.logp - shift).astype(np.float32) if old else None
    case["ref"] = (s.logp + rng.choice([0.0, 1e-4, 0.05, -0.4, 0.8, -2.0], rows)).astype(np.float32) if reference else None
    case["weight"] = rng.uniform(0.5, 1.5, rows).astype(np.float32) if weight else None
    for name in ("advantage", "old", "ref", "weight"):     # rows without a label: nothing of theirs is looked at
        if case[name] is not None:
            case[name][call.labels < 0] = np.nan
    return case


def run_policy(call, case, pad, in_place=False, gradient=True, kl_coef=0.05, low=0.2, high=0.28):
    ko, rows = call.ko, call.rows
    d = {k: None if v is None else ko.DeviceBuffer.from_numpy(v) for k, v in case.items()}
    outs = {k: Out(ko, 4 * rows) for k in ("logp", "kl", "loss")}
    total = Out(ko, 4)
    ptr, ldd, fetch = call.gradient_out(pad, in_place)
    call.op("policy_loss")(call.logits, call.d_labels, d["advantage"], outs["loss"].ptr, rows, call.cols, old_logp=d["old"],
                           ref_logp=d["ref"], weight=d["weight"], clip_low=low, clip_high=high, kl_coef=kl_coef,
                           logp=outs["logp"].ptr, kl=outs["kl"].ptr, loss_sum=total.ptr, dlogits=ptr if gradient else None,
                           ldd=ldd, **call.kw, **call.typed, **call.work)
    ko.synchronize()
    got = {k: o.get(np.float32, (rows,)) for k, o in outs.items()}
    got["loss_sum"] = total.get(np.float32, (1,))
    if gradient:
        got["dlogits"] = fetch()
    return got


def check_policy(call, got, case, kl_coef=0.05, low=0.2, high=0.28):
    alive = call.labels >= 0
    clean = {k: None if v is None else np.where(alive, v, 1.0).astype(np.float64) for k, v in case.items()}
    scores = call.scores
    if clean["weight"] is not None:
        scores = ref.Scores(call.values, call.labels, call.scale, clean["weight"] != 0)
    want = ref.policy(scores, clean["advantage"], clean["old"], clean["ref"], clean["weight"], low, high, kl_coef)
    for name in ("logp", "kl", "loss", "loss_sum"):
        ref.assert_within(got[name], *want[name], name)
    if "dlogits" in got:
        call.check_gradient(got["dlogits"], want["dlogits"])
        dead = np.where(alive, clean["weight"] if clean["weight"] is not None else 1.0, 0.0) == 0
        assert not ref.to_float(np.ascontiguousarray(got["dlogits"]), call.kind)[dead].any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_policy_loss(ko, rows, cols, kind):
    for pad, skew, scale, workspace in ((0, 0, 1.0, True), (3, 4, 0.625, False), (8, 0, 1.5, False)):
        call = Call(ko, rows, cols, kind, 3000 + cols, pad, skew, workspace, scale)
        case = policy_case(call, cols)
        got = run_policy(call, case, pad)
        check_policy(call, got, case)
        again = run_policy(call, case, pad)
        for name in got:
            np.testing.assert_array_equal(again[name], got[name], err_msg=name)
        check_policy(call, run_policy(call, case, pad + 1), case)              # element by element
        check_policy(call, run_policy(call, case, pad, gradient=False), case)
        got_in_place = run_policy(call, case, pad, in_place=True)
        for name in got:
            np.testing.assert_array_equal(got_in_place[name], got[name], err_msg=name)


@pytest.mark.parametrize("rows,cols", [(5, 1001), (40, 33000), (300, 2000)])
def test_policy_loss_options(ko, rows, cols):
    for old, reference, weight in ((False, True, True), (True, False, True), (True, True, False), (False, False, False)):
        call = Call(ko, rows, cols, "bf16", 3100, 8)
        case = policy_case(call, 7, old, reference, weight)
        check_policy(call, run_policy(call, case, 8), case)
        check_policy(call, run_policy(call, case, 8, kl_coef=0.0, low=0.0, high=0.0), case, 0.0, 0.0, 0.0)


@pytest.mark.parametrize("rows,cols", [(5, 1001), (40, 33000), (300, 2000), (300, 40001)])
def test_policy_loss_weight_zero_rows_are_not_read(ko, rows, cols):
    call = Call(ko, rows, cols, "f32", 3200)
    case = policy_case(call, 8)
    off = np.arange(rows) % 3 == 1
    case["weight"][off] = 0.0
    x = call.stored.copy()
    x[off] = np.nan
    call.keep.upload(x)
    call.values = np.where(off[:, None], 0.0, call.values)
    check_policy(call, run_policy(call, case, 0), case)


@pytest.mark.parametrize("rows,cols", [(4, 1001), (40, 33000), (300, 2000), (300, 40001)])
def test_labels_beyond_the_vocabulary_and_nan_logits(ko, rows, cols):
    """A label that is no column gives NaN for its row, a NaN or +inf logit too; other rows are as they would be."""
    call = Call(ko, rows, cols, "f32", 3300)
    case = policy_case(call, 9)
    base = run_policy(call, case, 0)
    logp0, _ = call.logprob()
    grad0 = call.backward(np.ones(rows, np.float32), 0)
    bad = np.array([0, 2, 3])
    call.labels[bad] = [cols, 2 ** 31 - 1, 1]
    for name in ("advantage", "old", "ref", "weight"):
        case[name][bad] = 0.5
    x = call.stored.copy()
    x[3] = 1.0
    x[3, cols - 1] = np.inf
    call.keep.upload(x)
    call.d_labels.upload(call.labels)
    other = np.setdiff1d(np.arange(rows), bad)
    got = run_policy(call, case, 0)
    for name in ("logp", "kl", "loss", "dlogits"):
        assert np.isnan(got[name][bad]).all(), name
        np.testing.assert_array_equal(got[name][other], base[name][other], err_msg=name)
    assert np.isnan(got["loss_sum"]).all()
    logp, stats = call.logprob()
    assert np.isnan(logp[bad]).all() and np.isnan(stats[bad, 1]).all()
    np.testing.assert_array_equal(logp[other], logp0[other])
    grad = call.backward(np.ones(rows, np.float32), 0)   # (the statistics of row 3 here are the old row's: finite)
    assert np.isnan(grad[[0, 2]]).all()
    np.testing.assert_array_equal(grad[other], grad0[other])


def test_a_row_of_minus_infinity_and_an_impossible_label(ko):
    for rows, cols in ((3, 1000), (300, 1000)):
        x = inputs.normal_f32((rows, cols), 3400)
        x[0] = -np.inf
        x[1, 5] = -np.inf
        labels = np.full(rows, 5, np.int32)
        d_x, d_l, d_lp = ko.DeviceBuffer.from_numpy(x), ko.DeviceBuffer.from_numpy(labels), ko.DeviceBuffer(4 * rows)
        ko.token_logprob(d_x, d_l, d_lp, rows, cols)
        ko.synchronize()
        lp = d_lp.download(np.float32, (rows,))
        assert np.isnan(lp[0]) and lp[1] == -np.inf and np.isfinite(lp[2:]).all()


def test_policy_loss_extremes(ko):
    """No advantage: no surrogate, however large the ratio; a large ratio with a positive advantage is clipped."""
    cols = 64
    x = np.zeros((4, cols), np.float32)
    labels = np.full(4, 3, np.int32)
    lp = -np.log(64.0)
    old = np.array([lp - 200.0, lp - 200.0, lp - 200.0, lp + 200.0], np.float32)
    adv = np.array([0.0, 2.0, -1.0, -1.0], np.float32)
    bufs = [ko.DeviceBuffer.from_numpy(a) for a in (x, labels, old, adv)]
    loss, d = ko.DeviceBuffer(16), ko.DeviceBuffer(x.nbytes)
    ko.policy_loss(bufs[0], bufs[1], bufs[3], loss, 4, cols, old_logp=bufs[2], clip_low=0.25, clip_high=0.5, dlogits=d)
    ko.synchronize()
    loss, d = loss.download(np.float32, (4,)), d.download(np.float32, x.shape)
    assert loss[0] == 0 and loss[1] == -3.0 and loss[2] == np.inf and loss[3] == 0.75
    assert not d[[0, 1, 3]].any() and not np.isfinite(d[2]).all()


def test_policy_loss_no_rows(ko):
    total = Out(ko, 4)
    ko.policy_loss(None, None, None, None, 0, 8, loss_sum=total.ptr)
    ko.synchronize()
    assert total.get(np.float32, (1,))[0] == 0.0


# ---- preference loss

@pytest.mark.parametrize("eps", [0.0, 0.1])
@pytest.mark.parametrize("lens", [[1, 1], [0, 3], [5, 0], [0, 0], [40, 17, 3, 200, 1, 1], [5000, 2600, 1, 4097], [1] * 600])
def test_preference_loss(ko, lens, eps):
    lens = np.array(lens)
    pairs = len(lens) // 2
    before, behind = 3, 5  # tokens of no sequence
    offsets = np.concatenate([[before], before + np.cumsum(lens)]).astype(np.int32)
    tokens = int(offsets[-1]) + behind
    rng = np.random.default_rng(int(lens.sum()))
    logp = rng.normal(-2, 1, tokens).astype(np.float32)
    rf = (logp + rng.normal(0, 0.3, tokens)).astype(np.float32)
    labels = np.where(rng.random(tokens) < 0.2, -1, 7).astype(np.int32)
    logp[labels < 0] = np.nan
    rf[labels < 0] = np.inf
    for with_labels in (True, False):
        if not with_labels:
            logp, rf = np.where(labels < 0, -1.0, logp).astype(np.float32), np.where(labels < 0, -1.5, rf).astype(np.float32)
        want = ref.preference(logp, rf, offsets, labels if with_labels else None, 0.1, eps)
        d = [ko.DeviceBuffer.from_numpy(a) for a in (logp, rf, offsets, labels)]
        outs = dict(pair_loss=Out(ko, 4 * pairs), rewards=Out(ko, 8 * pairs), dlogp=Out(ko, 4 * tokens), loss_sum=Out(ko, 4))
        ko.preference_loss(d[0], d[1], d[2], pairs, tokens, outs["pair_loss"].ptr, labels=d[3] if with_labels else None,
                           beta=0.1, label_smoothing=eps, rewards=outs["rewards"].ptr, dlogp=outs["dlogp"].ptr,
                           loss_sum=outs["loss_sum"].ptr)
        ko.synchronize()
        for name, n in (("pair_loss", pairs), ("rewards", 2 * pairs), ("loss_sum", 1)):
            ref.assert_within(outs[name].get(np.float32, (n,)), *want[name], name)
        raw = outs["dlogp"].get(np.uint32, (tokens,))
        touched = want["touched"]
        assert (raw[~touched] == 0xFFFFFFFF).all()
        ref.assert_within(raw.view(np.float32)[touched], want["dlogp"][0][touched], want["dlogp"][1][touched], "dlogp")
        ko.preference_loss(d[0], d[1], d[2], pairs, tokens, outs["pair_loss"].ptr, labels=d[3] if with_labels else None)
        ko.synchronize()
        ref.assert_within(outs["pair_loss"].get(np.float32, (pairs,)),
                          *ref.preference(logp, rf, offsets, labels if with_labels else None)["pair_loss"], "loss alone")


def test_preference_loss_offsets_lead_nowhere(ko):
    """Offsets before the first token, behind the last one or going backwards never lead outside the arrays."""
    tokens = 100
    rng = np.random.default_rng(5)
    logp, rf = rng.normal(-2, 1, tokens).astype(np.float32), rng.normal(-2, 1, tokens).astype(np.float32)
    offsets = np.array([-50, 10, 5, 2 ** 31 - 1, 60, -2 ** 31, 1000], np.int32)
    want = ref.preference(logp, rf, offsets)
    d = [ko.DeviceBuffer.from_numpy(a) for a in (logp, rf, offsets)]
    loss, rewards, dlogp = Out(ko, 12), Out(ko, 24), Out(ko, 4 * tokens)
    ko.preference_loss(d[0], d[1], d[2], 3, tokens, loss.ptr, rewards=rewards.ptr, dlogp=dlogp.ptr)
    ko.synchronize()
    ref.assert_within(loss.get(np.float32, (3,)), *want["pair_loss"], "pair_loss")
    ref.assert_within(rewards.get(np.float32, (6,)), *want["rewards"], "rewards")
    dlogp.get(np.float32, (tokens,))


def test_preference_loss_extremes(ko):
    """Rewards far apart: the loss is the gap, its slope 0 or -beta; no overflow."""
    logp, rf = np.array([0.0, -5e4, -5e4, 0.0], np.float32), np.zeros(4, np.float32)
    offsets = np.arange(5, dtype=np.int32)
    d = [ko.DeviceBuffer.from_numpy(a) for a in (logp, rf, offsets)]
    loss, dlogp, total = Out(ko, 8), Out(ko, 16), Out(ko, 4)
    ko.preference_loss(d[0], d[1], d[2], 2, 4, loss.ptr, beta=1.0, pair_weight=1.0, dlogp=dlogp.ptr, loss_sum=total.ptr)
    ko.synchronize()
    np.testing.assert_array_equal(loss.get(np.float32, (2,)), [0.0, 5e4])
    np.testing.assert_array_equal(dlogp.get(np.float32, (4,)), [0.0, 0.0, -1.0, 1.0])
    assert total.get(np.float32, (1,))[0] == 5e4


def test_preference_loss_no_pairs(ko):
    total = Out(ko, 4)
    ko.preference_loss(None, None, None, 0, 0, None, loss_sum=total.ptr)
    ko.synchronize()
    assert total.get(np.float32, (1,))[0] == 0.0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(5, 40), (300, 333), (300, 9001)])
def test_policy_loss_unlikely_labels_and_lowest_values(ko, rows, cols, kind):
    """Labels far below the row's maximum, rows of nothing but the type's lowest value, and a label that is -inf."""
    call = Call(ko, rows, cols, kind, 3600)
    lowest = {"f32": np.finfo(np.float32).min, "f16": -65504.0, "bf16": -3.3895314e38}[kind]
    x = call.values.copy()
    live = np.flatnonzero(call.labels >= 0)
    r = np.arange(rows)
    x[live, call.labels[live]] -= np.array([0.0, 20.0, 28.0, 60.0])[live % 4]
    x[live[0]] = lowest                                       # a uniform distribution
    x[live[1], :] = lowest                                    # all but two columns masked
    x[live[1], [call.labels[live[1]], (call.labels[live[1]] + 1) % cols]] = [1.0, 2.0]
    stored, values = ref.to_storage(x, kind)
    call.keep.upload(stored)
    call.values = values
    call.stored = stored
    call.scores = ref.Scores(values, call.labels)
    case = policy_case(call, 11)
    check_policy(call, run_policy(call, case, 0), case)
    # the label's own logit is -inf: logp is, too, and with no pull from its reference the gradient is finite
    x = stored.copy()
    x[live[2], call.labels[live[2]]] = {"f32": -np.inf, "f16": 0xFC00, "bf16": 0xFF80}[kind]
    call.keep.upload(x)
    case["ref"] = None
    got = run_policy(call, case, 0, kl_coef=0.0)
    assert got["logp"][live[2]] == -np.inf
    assert np.isfinite(ref.to_float(np.ascontiguousarray(got["dlogits"]), kind)[live]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(7, 19), (300, 333), (300, 2050), (270, 9001), (260, 33000)])
def test_labels_in_the_first_and_last_columns(ko, rows, cols, kind):
    """Where rows start off a vector the first and last columns are taken one by one, and where a workgroup has more threads
    than the row has vectors the last vector is written by several."""
    call = Call(ko, rows, cols, kind, 3700)
    at = np.arange(rows) % 18
    alive = call.labels >= 0
    call.labels[alive] = np.where(at < 9, at, cols - 1 - (at - 9))[alive]
    x = np.nan_to_num(call.values, nan=0.0, neginf=-5.0)
    x = np.where(x < -100.0, -5.0, x)
    x[np.arange(rows), np.maximum(call.labels, 0)] += 3.0
    call.stored, call.values = ref.to_storage(x, kind)
    call.keep.upload(call.stored)
    call.d_labels.upload(call.labels)
    call.scores = ref.Scores(call.values, call.labels)
    case = policy_case(call, 12)
    check_policy(call, run_policy(call, case, 0), case)
    call.check_logprob()
    dlogp = inputs.normal_f32((rows,), 3701)
    want = call.scores.gradient(dlogp.astype(np.float64), 0.0, 3 * ref.U * np.abs(call.scores.logsum) + 2 * ref.U)
    call.check_gradient(call.backward(dlogp, 0), want)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vectors", [1, 2, 63, 64, 65, 128, 129, 257, 260, 319, 513, 1025, 1537, 2049, 3 * 1024 + 1, 4097, 5121, 6145,
                                     8193, 10241, 12289, 14337, 16384, 16385])
def test_policy_loss_where_one_way_ends_and_the_next_begins(ko, vectors, kind):
    """Rows of one 16-byte vector more than the last shape of a workgroup takes, whole and with single elements around them."""
    per = 4 if kind == "f32" else 8
    for pad, skew, more in ((0, 0, 0), (3, 4, per - 1), (0, 0, -1)):
        call = Call(ko, 4, vectors * per + more, kind, 3800 + vectors, pad, skew, False)
        case = policy_case(call, vectors)
        got = run_policy(call, case, pad)
        check_policy(call, got, case)


@pytest.mark.parametrize("lens", [[3, 2] * 2 + [0, 9], [70, 300] * 4, [0, 1] + [200, 150] * 4, [33, 64] * 16, [31, 1] * 17, [4000, 4184],
                                  [4000, 4185], [513, 511] * 8, [8000, 1, 0, 0, 1, 0]])
def test_preference_loss_of_few_and_more_pairs(ko, lens):
    """Both sides of the border between one workgroup for every pair and one for each."""
    test_preference_loss(ko, lens, 0.1)


# rows longer than the registers of a workgroup (16384 vectors): in pieces, and one workgroup each
@pytest.mark.parametrize("rows", [5, 65])
@pytest.mark.parametrize("kind,cols", [("f32", 70001), ("bf16", 140001)])
def test_rows_longer_than_the_registers(ko, rows, kind, cols):
    test_policy_loss_unlikely_labels_and_lowest_values(ko, rows, cols, kind)
    test_labels_in_the_first_and_last_columns(ko, rows, cols, kind)


@pytest.mark.parametrize("rows,cols", [(5, 70001), (65, 70001)])
def test_special_rows_longer_than_the_registers(ko, rows, cols):
    test_policy_loss_weight_zero_rows_are_not_read(ko, rows, cols)
    test_labels_beyond_the_vocabulary_and_nan_logits(ko, rows, cols)
    test_policy_loss_options(ko, rows, cols)


# several short rows per wavefront: every number of them at the end, every kind of row among the others
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(1, 40), (7, 256), (8, 257), (9, 512), (17, 100), (1003, 500), (23, 1000), (64, 1030), (5000, 90)])
def test_short_rows(ko, rows, cols, kind):
    test_token_logprob_and_its_gradient(ko, rows, cols, kind)
    test_policy_loss(ko, rows, cols, kind)
    if rows > 20:
        test_policy_loss_unlikely_labels_and_lowest_values(ko, rows, cols, kind)
        test_labels_in_the_first_and_last_columns(ko, rows, cols, kind)


@pytest.mark.parametrize("rows,cols", [(30, 90), (30, 250), (30, 509)])
def test_special_short_rows(ko, rows, cols):
    test_policy_loss_weight_zero_rows_are_not_read(ko, rows, cols)
    test_labels_beyond_the_vocabulary_and_nan_logits(ko, rows, cols)
    test_policy_loss_options(ko, rows, cols)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(16384, 130), (16391, 40), (32768, 64), (33003, 65), (33001, 250)])
def test_many_short_rows(ko, rows, cols, kind):
    """Eight rows per wavefront, the log-probabilities' from 16384 rows on, the policy loss's from 32768."""
    test_token_logprob_and_its_gradient(ko, rows, cols, kind)
    test_policy_loss(ko, rows, cols, kind)
    test_policy_loss_unlikely_labels_and_lowest_values(ko, rows, cols, kind)
    test_labels_in_the_first_and_last_columns(ko, rows, cols, kind)


@pytest.mark.parametrize("rows,cols", [(33001, 90), (16400, 509)])
def test_special_ones_among_many_short_rows(ko, rows, cols):
    test_policy_loss_weight_zero_rows_are_not_read(ko, rows, cols)
    test_labels_beyond_the_vocabulary_and_nan_logits(ko, rows, cols)
    test_policy_loss_options(ko, rows, cols)
