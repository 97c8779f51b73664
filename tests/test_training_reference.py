"""The 64-bit formulas that the backward and loss kernels are held to, against central differences of the forward
formulas, and what the entry points refuse (both need no GPU)."""
import numpy as np
import pytest

import kernel_optimization_amd as ko
import training_reference as ref


def _numeric(f, x, step=1e-5):
    g = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        hi, lo = x.copy(), x.copy()
        hi[i] += step
        lo[i] -= step
        g[i] = (f(hi) - f(lo)) / (2 * step)
    return g


def _softmax(x):
    e = np.exp(x - x.max(1, keepdims=True))
    return e / e.sum(1, keepdims=True)


@pytest.mark.parametrize("low", [0.0, -9998.0])
def test_softmax_gradient_matches_differences(low):
    """Also where the valid scores are so low (-9998) that the padding, at -10000, has weight."""
    rng = np.random.default_rng(1)
    x, dy = rng.normal(0, 1, (4, 7)) + low, rng.normal(0, 1, (4, 7))
    lens = np.array([7, 3, 1, 0])

    def forward(v):
        return _softmax(np.where(ref.keep_columns(4, 7, lens, 1), v, -10000.0))

    dx, _ = ref.softmax_backward(forward(x), dy, lens, 1)
    np.testing.assert_allclose(dx, _numeric(lambda v: (forward(v) * dy).sum(), x), atol=2e-7)


@pytest.mark.parametrize("unbiased", [False, True])
@pytest.mark.parametrize("residual", [False, True])
def test_layernorm_gradient_matches_differences(unbiased, residual):
    rng = np.random.default_rng(2)
    x, dy = rng.normal(0.5, 2, (3, 9)), rng.normal(0, 1, (3, 9))
    gamma, beta = rng.normal(1, 0.1, 9), rng.normal(0, 0.1, 9)
    dres = rng.normal(0, 1, (3, 9)) if residual else None

    def stats(v):
        mean = v.mean(1)
        return mean, 1 / np.sqrt(((v - mean[:, None]) ** 2).sum(1) / (8 if unbiased else 9) + 1e-5)

    def loss(v, g, b):
        mean, rstd = stats(v)
        y = (v - mean[:, None]) * rstd[:, None] * g + b
        return (y * dy).sum() + (0.0 if dres is None else (v * dres).sum())

    (dx, dgamma, dbeta), _ = ref.layernorm_backward(dy, x, *stats(x), gamma, dres, unbiased)
    np.testing.assert_allclose(dx, _numeric(lambda v: loss(v, gamma, beta), x), atol=1e-8)
    np.testing.assert_allclose(dgamma, _numeric(lambda v: loss(x, v, beta), gamma), atol=1e-8)
    np.testing.assert_allclose(dbeta, _numeric(lambda v: loss(x, gamma, v), beta), atol=1e-8)


@pytest.mark.parametrize("scale", [1.0, 0.625])
def test_logprob_and_policy_gradients_match_differences(scale):
    rng = np.random.default_rng(3)
    x = rng.normal(0, 2, (6, 5))
    labels = np.array([0, 4, 2, -1, 3, 1])
    coeff = rng.normal(0, 1, 6)
    d, _ = ref.Scores(x, labels, scale).gradient(coeff)
    np.testing.assert_allclose(d, _numeric(lambda v: (coeff * ref.Scores(v, labels, scale).logp).sum(), x), atol=1e-8)

    lp = ref.Scores(x, labels, scale).logp
    adv = np.array([1.0, -1.0, 0.5, 2.0, -0.7, 0.0])
    old = lp - np.array([0.4, 0.5, 0.05, 0.0, -0.5, 0.1])  # clipped, not clipped, not, dead, clipped, no advantage
    kw = dict(old=old, ref=lp + rng.normal(0, 0.3, 6), weight=rng.uniform(0.5, 1.5, 6), kl_coef=0.25)
    total = lambda v: ref.policy(ref.Scores(v, labels, scale), adv, **kw)["loss_sum"][0][0]
    d = ref.policy(ref.Scores(x, labels, scale), adv, **kw)["dlogits"][0]
    assert not d[3].any()
    np.testing.assert_allclose(d, _numeric(total, x), atol=1e-8)


@pytest.mark.parametrize("eps", [0.0, 0.1])
def test_preference_gradient_matches_differences(eps):
    rng = np.random.default_rng(4)
    lp, rf = rng.normal(-2, 1, 20), rng.normal(-2, 1, 20)
    offsets = np.array([1, 6, 6, 13, 19])   # an empty rejected sequence; tokens 0 and 19 belong to none
    labels = np.where(np.arange(20) % 5 == 2, -1, 1)
    kw = dict(labels=labels, beta=0.5, eps=eps)
    got = ref.preference(lp, rf, offsets, **kw)
    num = _numeric(lambda v: ref.preference(v, rf, offsets, **kw)["loss_sum"][0][0], lp)
    np.testing.assert_allclose(got["dlogp"][0], num, atol=1e-8)


# ---- refusals: checked on the host before anything touches a device

BAD = 0x1000  # a pointer that is never followed


def _refused(status, code, word):
    assert status == code, (status, ko.last_error())
    assert word in ko.last_error()


def test_softmax_backward_refusals():
    f, h = ko.lib().ko_softmax_backward_f32, ko.lib().ko_softmax_backward_16
    inv = ko.KO_ERR_INVALID_ARGUMENT
    _refused(f(None, BAD, BAD, 4, 8, None, 0, None, 0, None), inv, "null")
    _refused(f(BAD, BAD, BAD, -1, 8, None, 0, None, 0, None), inv, "rows")
    _refused(f(BAD, BAD, BAD, 4, 0, None, 0, None, 0, None), inv, "cols")
    _refused(f(BAD, BAD, BAD, 4, (1 << 30) + 1, None, 0, None, 0, None), ko.KO_ERR_UNSUPPORTED_SHAPE, "too large")
    _refused(f(BAD + 2, BAD, BAD, 4, 8, None, 0, None, 0, None), inv, "aligned")
    _refused(f(BAD, BAD, BAD, 4, 8, BAD, 0, None, 0, None), inv, "rows_per_seq")
    need = ko.softmax_backward_workspace_bytes(2, 200000)
    assert need > 0 and ko.softmax_backward_workspace_bytes(1000, 128) == 0
    _refused(f(BAD, BAD, BAD, 2, 200000, None, 0, BAD, need - 1, None), inv, "workspace")
    _refused(f(BAD, BAD, BAD, 2, 200000, None, 0, BAD + 4, need, None), inv, "16-byte")
    _refused(h(BAD, BAD, BAD, 4, 8, None, 0, 2, None, 0, None), inv, "dtype")
    assert f(None, None, None, 0, 8, None, 0, None, 0, None) == ko.KO_OK


def test_layernorm_backward_refusals():
    f, h = ko.lib().ko_layernorm_backward_f32, ko.lib().ko_layernorm_backward_16
    inv = ko.KO_ERR_INVALID_ARGUMENT
    for missing in (0, 1, 2, 3, 6):  # dy, in, mean, rstd, dx
        p = [BAD] * 9
        p[missing] = None
        _refused(f(*p, 4, 8, 0, None, 0, None), inv, "null")
    _refused(f(*[BAD] * 9, -1, 8, 0, None, 0, None), inv, "rows")
    _refused(f(*[BAD] * 9, 4, 0, 0, None, 0, None), inv, "cols")
    _refused(f(*[BAD] * 9, 4, (1 << 30) + 1, 0, None, 0, None), ko.KO_ERR_UNSUPPORTED_SHAPE, "too large")
    _refused(f(BAD + 1, *[BAD] * 8, 4, 8, 0, None, 0, None), inv, "aligned")
    _refused(f(*[BAD] * 7, BAD + 2, BAD, 4, 8, 0, None, 0, None), inv, "4-byte")
    need = ko.layernorm_backward_workspace_bytes(100, 768)
    assert need >= 2 * 768 * 4
    _refused(f(*[BAD] * 9, 100, 768, 0, BAD, need - 1, None), inv, "workspace")
    _refused(h(*[BAD] * 9, 4, 8, 0, 7, None, 0, None), inv, "dtype")
    assert f(*[None] * 9, 0, 8, 0, None, 0, None) == ko.KO_OK


def test_token_logprob_refusals():
    lib, inv = ko.lib(), ko.KO_ERR_INVALID_ARGUMENT
    f, h, b = lib.ko_token_logprob_f32, lib.ko_token_logprob_16, lib.ko_token_logprob_backward_f32
    _refused(f(None, 8, BAD, 1.0, BAD, None, 4, 8, None, 0, None), inv, "null")
    _refused(f(BAD, 8, BAD, 1.0, None, None, 4, 8, None, 0, None), inv, "logp")
    _refused(f(BAD, 7, BAD, 1.0, BAD, None, 4, 8, None, 0, None), inv, "ld")
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        _refused(f(BAD, 8, BAD, scale, BAD, None, 4, 8, None, 0, None), inv, "scale")
    _refused(f(BAD, 8, BAD, 1.0, BAD, None, 4, 0, None, 0, None), inv, "cols")
    _refused(f(BAD, 1 << 31, BAD, 1.0, BAD, None, 4, (1 << 30) + 1, None, 0, None), ko.KO_ERR_UNSUPPORTED_SHAPE, "too large")
    _refused(f(BAD + 2, 8, BAD, 1.0, BAD, None, 4, 8, None, 0, None), inv, "aligned")
    need = ko.token_logprob_workspace_bytes(4, 100000)
    assert need > 0 and ko.token_logprob_workspace_bytes(4096, 50257) == 0
    _refused(f(BAD, 100000, BAD, 1.0, BAD, None, 4, 100000, BAD, need - 1, None), inv, "workspace")
    _refused(h(BAD, 8, BAD, 1.0, BAD, None, 4, 8, 5, None, 0, None), inv, "dtype")
    _refused(b(BAD, 8, BAD, 1.0, None, BAD, BAD, 8, 4, 8, None), inv, "row_stats")
    _refused(b(BAD, 8, BAD, 1.0, BAD, BAD, BAD, 7, 4, 8, None), inv, "ldd")
    _refused(b(BAD, 8, BAD, 1.0, BAD, BAD, None, 8, 4, 8, None), inv, "dlogits")
    assert f(None, 8, None, 1.0, None, None, 0, 8, None, 0, None) == ko.KO_OK


def test_policy_and_preference_refusals():
    lib, inv = ko.lib(), ko.KO_ERR_INVALID_ARGUMENT

    def policy(logits=BAD, labels=BAD, adv=BAD, loss=BAD, ld=8, ldd=8, low=0.2, high=0.2, kl=0.0, scale=1.0):
        return lib.ko_policy_loss_f32(logits, ld, labels, None, None, adv, None, scale, low, high, kl, None, None, loss, None,
                                      BAD, ldd, 4, 8, None, 0, None)

    _refused(policy(logits=None), inv, "null")
    _refused(policy(labels=None), inv, "null")
    _refused(policy(adv=None), inv, "null")
    _refused(policy(loss=None), inv, "null")
    _refused(policy(ldd=3), inv, "ldd")
    _refused(policy(low=1.5), inv, "clip")
    _refused(policy(high=-0.1), inv, "clip")
    _refused(policy(high=float("nan")), inv, "clip")
    _refused(policy(kl=float("inf")), inv, "kl_coef")
    _refused(policy(scale=0.0), inv, "scale")

    def preference(logp=BAD, ref_logp=BAD, offsets=BAD, pairs=2, tokens=9, beta=0.1, eps=0.0, loss=BAD):
        return lib.ko_preference_loss_f32(logp, ref_logp, None, offsets, pairs, tokens, beta, eps, 0.5, loss, None, None, None,
                                          None)

    _refused(preference(logp=None), inv, "null")
    _refused(preference(offsets=None), inv, "null")
    _refused(preference(loss=None), inv, "null")
    _refused(preference(pairs=-1), inv, "pairs")
    _refused(preference(tokens=1 << 31), inv, "tokens")
    _refused(preference(beta=float("nan")), inv, "beta")
    _refused(preference(eps=1.5), inv, "label_smoothing")
    assert preference(pairs=0) == ko.KO_OK


def test_gradients_over_logits_of_another_row_stride_are_refused():
    """In place the rows have to lie alike: with another stride a row's gradient falls on logits that are still to be read."""
    backward, policy = ko.lib().ko_token_logprob_backward_f32, ko.lib().ko_policy_loss_f32
    _refused(backward(BAD, 12, BAD, 1.0, BAD, BAD, BAD, 8, 4, 8, None), ko.KO_ERR_INVALID_ARGUMENT, "ldd")
    _refused(policy(BAD, 8, BAD, None, None, BAD, None, 1.0, 0.2, 0.2, 0.0, None, None, BAD, None, BAD, 12, 4, 8, None, 0, None),
             ko.KO_ERR_INVALID_ARGUMENT, "ldd")
