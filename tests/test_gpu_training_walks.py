"""Forms of the training-side operators that only many rows reach: workgroups that walk over rows, here on grids cut to three of
them, and eight rows of two vectors per lane to a wavefront."""
import ctypes

import numpy as np
import pytest

import test_gpu_token_loss as token_loss
import training_reference as ref
from kernel_optimization_amd import inputs
from test_gpu_backward_rows import KINDS, _softmax, check_layernorm_backward, check_softmax_backward, layernorm_case
from test_gpu_streams_and_graphs import _hip_runtime
from test_gpu_token_loss import Call, policy_case, run_policy

pytestmark = pytest.mark.gpu


@pytest.fixture
def three_workgroups(ko):
    ko.set_tuning("rows.most_workgroups", 3)
    yield
    ko.set_tuning("rows.most_workgroups", 0)


# every number of threads per row of the log-probabilities and of the policy loss without a gradient, one row at a time and eight
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(61, 257), (61, 1001), (50, 2049), (50, 4100), (40, 8200), (50, 12000), (40, 33001), (40, 70001),
                                       (16400, 130), (16391, 300)])
def test_walks_of_the_token_losses(ko, three_workgroups, rows, cols, kind):
    """Rows without a label, with one beyond the vocabulary and with one far below the others, which is summed twice, between
    ordinary ones, so that what one row left in LDS is there when another comes."""
    call = Call(ko, rows, cols, kind, 5000 + cols, 3, 0, False)
    live = np.flatnonzero(call.labels >= 0)
    x = np.where((call.labels >= 0)[:, None], call.values, np.nan).astype(np.float32)
    far = live[::3]
    x[far, call.labels[far]] -= 70.0
    stored = np.full((rows, call.ld), np.nan, np.float32)
    stored[:, :cols] = x
    call.stored, values = ref.to_storage(stored, kind)
    call.values = values[:, :cols]
    call.keep.upload(call.stored)
    alive = call.labels >= 0
    beyond = np.zeros(rows, bool)
    beyond[live[1::4]] = True
    call.scores = ref.Scores(call.values, call.labels, 1.0, ~beyond)
    call.labels[beyond] = cols + np.arange(beyond.sum())
    call.d_labels.upload(call.labels)
    sound, dead = alive & ~beyond, ~alive
    logp, stats = call.logprob()
    s = call.scores
    assert np.isnan(logp[beyond]).all() and np.isnan(stats[beyond]).all() and not logp[dead].any()
    ref.assert_within(logp[sound], s.logp[sound], s.logp_off[sound], "logp")
    np.testing.assert_array_equal(stats[sound, 0], s.top[sound].astype(np.float32))
    ref.assert_within(stats[sound, 1], s.logsum[sound], s.logsum_off[sound], "log sum")
    case = policy_case(call, cols)
    for name in ("old", "ref", "weight"):
        case[name][beyond] = 0.5
    clean = {k: np.where(sound, v, 1.0).astype(np.float64) for k, v in case.items()}
    want = ref.policy(s, clean["advantage"], clean["old"], clean["ref"], clean["weight"], 0.2, 0.28, 0.05)
    for gradient, pad in ((False, 3), (True, 4)):       # (with rows that lie differently: a second read, by elements)
        got = run_policy(call, case, pad, gradient=gradient)
        assert np.isnan(got["loss_sum"]).all()
        for name in ("logp", "kl", "loss"):
            assert np.isnan(got[name][beyond]).all() and not got[name][dead].any()
            ref.assert_within(got[name][sound], want[name][0][sound], want[name][1][sound], name)
        if gradient:
            d = ref.to_float(np.ascontiguousarray(got["dlogits"]), kind)
            assert np.isnan(d[beyond]).all() and not d[dead].any()
            value, off = want["dlogits"]
            ref.assert_within(d[sound], value[sound], (off + ref.rounded(kind, value) * (1 + 1e-6))[sound], "dlogits")


@pytest.mark.parametrize("lens", [[1] * 600, [40, 17, 3, 200, 1, 1] * 20, [5000, 2600, 1, 4097], [3, 1] * 1500])
def test_walks_of_the_preference_loss(ko, three_workgroups, lens):
    token_loss.test_preference_loss(ko, lens, 0.1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,rps", [(301, 37, 3), (301, 512, 4), (70, 1001, 1), (31, 3000, 2), (25, 8200, 3), (17, 20000, 1),
                                           (11, 70001, 1), (70, 66000, 1)])
def test_walks_of_the_softmax_gradient(ko, three_workgroups, rows, cols, rps, kind):
    x = inputs.normal_f32((rows, cols), 5100 + cols, 0.0, 4.0).astype(np.float64)
    dy, _ = ref.to_storage(inputs.normal_f32((rows, cols), 5101 + cols), kind)
    y, _ = ref.to_storage(_softmax(x), kind)
    check_softmax_backward(ko, y, dy, kind, workspace=False)
    lens = (np.arange((rows + rps - 1) // rps) * 977 % (cols + 3) - 1).astype(np.int32)
    keep = ref.keep_columns(rows, cols, lens, rps)
    y, _ = ref.to_storage(_softmax(np.where(keep, x, -10000.0)), kind)
    check_softmax_backward(ko, y, dy, kind, lens, rps, workspace=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(300, 3), (20, 17000), (15, 40001)])
def test_walks_of_the_layernorm_gradient(ko, three_workgroups, rows, cols, kind):
    check_layernorm_backward(ko, layernorm_case(rows, cols, kind, 5200 + cols), kind)


@pytest.mark.parametrize("kind,cols", [("f16", 520), ("f16", 703), ("bf16", 777), ("bf16", 1024), ("f16", 1031), ("f32", 300), ("f32", 404),
                                       ("f32", 511)])
def test_many_rows_of_two_vectors_per_lane(ko, kind, cols):
    token_loss.test_token_logprob_and_its_gradient(ko, 16391, cols, kind)


def test_rows_behind_32_bit_offsets_against_64_bits(ko):
    """66000 rows of 33000 bf16 columns: rows next to where 32-bit offsets in elements (65075.2 rows) and in bytes (32537.6) end, and the
    last ones, against the formulas."""
    rows, cols = 66000, 33000
    size = rows * cols * 2
    a, b, d = ko.DeviceBuffer(size), ko.DeviceBuffer(size), ko.DeviceBuffer(size)
    ko.fill_uniform_16(a, rows * cols, 84, dtype=ko.BF16)
    ko.fill_uniform_16(b, rows * cols, 85, dtype=ko.BF16)
    rng = np.random.default_rng(86)
    some = np.array([0, 32537, 32538, 65074, 65075, 65076, 65999])
    labels = rng.integers(0, cols, rows).astype(np.int32)
    f = {k: rng.uniform(*v, rows).astype(np.float32) for k, v in dict(mean=(-.1, .1), rstd=(.5, 2), dlogp=(.5, 1), adv=(-1, 1)).items()}
    dev = {k: ko.DeviceBuffer.from_numpy(v) for k, v in f.items()}
    dl, logp, stats, loss = ko.DeviceBuffer.from_numpy(labels), *(ko.DeviceBuffer(n * rows) for n in (4, 8, 4))

    def fetch(buf):
        return np.stack([ref.to_float(buf.download(np.uint16, (cols,), int(r) * cols * 2), "bf16") for r in some])

    def check(value, off, name):
        ref.assert_within(fetch(d), value, off + ref.rounded("bf16", value) * (1 + 1e-6), name)

    x, y = fetch(a), fetch(b)
    typed = dict(dtype=ko.BF16)
    ko.layernorm_backward16(a, b, dev["mean"], dev["rstd"], d, rows, cols, **typed)
    (value, _, _), (off, _, _) = ref.layernorm_backward(x, y, f["mean"][some].astype(np.float64), f["rstd"][some].astype(np.float64))
    check(value, off, "LayerNorm")
    ko.softmax_backward16(a, b, d, rows, cols, **typed)
    check(*ref.softmax_backward(x, y), "softmax")
    ko.token_logprob16(a, dl, logp, rows, cols, row_stats=stats, **typed)
    ko.token_logprob_backward16(a, dl, stats, dev["dlogp"], d, rows, cols, **typed)
    s = ref.Scores(x, labels[some])
    ref.assert_within(logp.download(np.float32, (rows,))[some], s.logp, s.logp_off, "logp")
    check(*s.gradient(f["dlogp"][some].astype(np.float64), 0.0, s.logsum_off + 3 * ref.U * np.abs(s.logsum) + 2 * ref.U), "logp gradient")
    ko.policy_loss16(a, dl, dev["adv"], loss, rows, cols, dlogits=d, **typed)
    want = ref.policy(s, f["adv"][some].astype(np.float64))
    ref.assert_within(loss.download(np.float32, (rows,))[some], *want["loss"], "loss")
    check(*want["dlogits"], "policy gradient")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("per_row", [9, 64, 65, 127, 128, 129])
def test_the_number_of_rows_does_not_matter(ko, per_row, kind):
    """Many rows go eight to a wavefront up to 128 vectors, in the policy loss up to 64: log-probabilities have the bits of a few rows'
    call, the policy loss beyond 64 vectors, too."""
    many, few, cols = 33003, 200, per_row * (4 if kind == "f32" else 8) + 1
    call = Call(ko, few, cols, kind, 5300 + cols, 7 if kind == "f32" else 15)     # (rows of whole vectors, started anywhere)
    case = policy_case(call, 5)
    alone, scored = call.logprob(), run_policy(call, case, 7)
    rows = np.concatenate([np.arange(few), np.random.default_rng(5).integers(0, few, many - few)])
    call.rows, call.stored, call.labels = many, call.stored[rows], call.labels[rows]
    call.keep, call.logits = ko.DeviceBuffer.from_numpy(call.stored), None
    call.logits = call.keep.ptr
    call.d_labels = ko.DeviceBuffer.from_numpy(call.labels)
    case = {k: None if v is None else v[rows] for k, v in case.items()}
    for got, want in zip(call.logprob(), alone):
        np.testing.assert_array_equal(got[:few], want)
    if cols // (4 if kind == "f32" else 8) > 64:
        got = run_policy(call, case, 7)
        for name in ("logp", "kl", "loss", "dlogits"):
            np.testing.assert_array_equal(got[name][:few], scored[name], err_msg=name)


def test_many_pairs_in_a_graph(ko):
    """More pairs than one workgroup each looks through: the launch that prepares them passes its results through pair_loss, in every
    replay anew, with eager calls of other sizes in between."""
    hip = _hip_runtime()
    rng = np.random.default_rng(54)
    steps = []
    for pairs in (1025, 1024, 5000):
        offsets = np.concatenate([[0], np.cumsum(rng.integers(0, 9, 2 * pairs))])
        offsets[rng.integers(1, 2 * pairs, pairs // 50)] -= 30                    # some lead into earlier pairs
        tokens = int(offsets.max()) + 3
        bufs = [ko.DeviceBuffer.from_numpy(v) for v in (rng.normal(-2, 1, tokens).astype(np.float32),
                                                        rng.normal(-2, 1, tokens).astype(np.float32), offsets.astype(np.int32))]
        outs = {k: (ko.DeviceBuffer(4 * n), n) for k, n in dict(pair_loss=pairs, dlogp=tokens, loss_sum=1).items()}
        steps.append((pairs, tokens, bufs, outs))

    def run(step, stream):
        pairs, tokens, (logp, rf, offsets), outs = step
        ko.preference_loss(logp, rf, offsets, pairs, tokens, outs["pair_loss"][0], dlogp=outs["dlogp"][0],
                           loss_sum=outs["loss_sum"][0], stream=stream)

    def clear():
        for step in steps:
            for buf, n in step[3].values():
                buf.upload(np.full(n, np.nan, np.float32))

    def results():
        return [buf.download(np.uint32, (n,)) for step in steps for buf, n in step[3].values()]

    clear()
    for step in steps:
        run(step, None)
    ko.synchronize()
    want = results()
    stream, graph, graph_exec = ko.Stream(), ctypes.c_void_p(), ctypes.c_void_p()
    assert hip.hipStreamBeginCapture(stream.handle, 0) == 0
    try:
        for step in steps[::2]:
            run(step, stream)
    finally:
        rc = hip.hipStreamEndCapture(stream.handle, ctypes.byref(graph))
    assert rc == 0 and graph.value
    try:
        assert hip.hipGraphInstantiate(ctypes.byref(graph_exec), graph, None, None, 0) == 0
        for _ in range(4):
            clear()
            ko.synchronize()
            assert hip.hipGraphLaunch(graph_exec, stream.handle) == 0
            run(steps[1], None)
            stream.synchronize()
            ko.synchronize()
            for got, expected in zip(results(), want):
                np.testing.assert_array_equal(got, expected)
    finally:
        if graph_exec.value:
            hip.hipGraphExecDestroy(graph_exec)
        hip.hipGraphDestroy(graph)
