"""The backward passes and losses in 64 bits (numpy, straight from their formulas), each with a bound on what fp32
arithmetic and one rounding to the storage type can do to it.

u = 2^-24 is half a step of fp32.  A sum of n terms taken in any order of depth d is off by at most d u sum|terms|; the
kernels' sums have a serial part of at most DEPTH terms per thread (longer rows: cols / 256) and a tree of at most 20
steps.  Storage rounding: half a step, eps / 2 of the value (binary16 2^-11, bfloat16 2^-8, fp32 2^-24), in binary16's
subnormal range 2^-25 absolute; fp32 results below 2^-126 may be flushed to zero."""
import numpy as np

U = 2.0 ** -24
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}


def depth(n):
    return max(100, n / 256) + 30


def rounded(kind, value):
    """Half a storage step of `value`."""
    return HALF_STEP[kind] * np.abs(value) + TINY[kind]


def assert_within(got, want, bound, what):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert np.all(np.isfinite(got)), "%s: %d values are not finite" % (what, np.sum(~np.isfinite(got)))
    over = np.abs(got - want) / bound
    worst = np.unravel_index(np.argmax(over), over.shape) if over.size else None
    assert over.size == 0 or over[worst] <= 1.0, "%s at %s: %r, want %r +- %r" % (what, worst, got[worst], want[worst],
                                                                                  np.broadcast_to(bound, over.shape)[worst])


# ---- storage types

def to_storage(x, kind):
    """float array -> (array of the storage type's bits or floats, its values in float64)"""
    from kernel_optimization_amd import inputs
    x = np.asarray(x, np.float32)
    if kind == "f32":
        return x, x.astype(np.float64)
    with np.errstate(over="ignore"):
        bits = inputs.f32_to_bf16_bits(x).reshape(x.shape) if kind == "bf16" else x.astype(np.float16).view(np.uint16)
    return bits, to_float(bits, kind)


def to_float(stored, kind):
    from kernel_optimization_amd import inputs
    if kind == "f32":
        return stored.astype(np.float64)
    if kind == "bf16":
        return inputs.bf16_bits_to_f32(stored).astype(np.float64).reshape(stored.shape)
    return stored.view(np.float16).astype(np.float64)


# ---- softmax

def keep_columns(rows, cols, valid_len, rows_per_seq):
    if valid_len is None:
        return np.ones((rows, cols), bool)
    lens = np.clip(np.asarray(valid_len), 0, cols)[np.arange(rows) // rows_per_seq]
    return np.arange(cols)[None, :] < lens[:, None]


def softmax_backward(y, dy, valid_len=None, rows_per_seq=0):
    """dx, and the bound on its fp32 arithmetic."""
    rows, cols = y.shape
    keep = keep_columns(rows, cols, valid_len, rows_per_seq)
    counts = keep | (y != 0)
    dy = np.where(counts, dy, 0.0)
    y = np.where(counts, y, 0.0)
    t = (y * dy).sum(1, keepdims=True)
    t_off = depth(cols) * U * np.abs(y * dy).sum(1, keepdims=True)
    dx = np.where(keep, y * (dy - t), 0.0)
    off = np.where(keep, np.abs(y) * (t_off + 2 * U * (np.abs(dy) + np.abs(t))), 0.0)
    return dx, off


# ---- LayerNorm

def layernorm_backward(dy, x, mean, rstd, gamma=None, dres=None, unbiased=False):
    """((dx, dgamma, dbeta), (their bounds on fp32 arithmetic))"""
    rows, cols = x.shape
    d = cols - 1 if unbiased else cols
    rstd = rstd[:, None]
    xh = (x - mean[:, None]) * rstd
    g = dy if gamma is None else dy * gamma
    c1 = g.sum(1, keepdims=True) / cols
    c2 = (g * xh).sum(1, keepdims=True) / d
    dx = rstd * (g - c1 - xh * c2)
    # x - mean, times rstd, times dy gamma: 3 roundings of each term of the sums beside the sums' own
    c1_off = (depth(cols) + 4) * U * np.abs(g).sum(1, keepdims=True) / cols
    c2_off = (depth(cols) + 6) * U * np.abs(g * xh).sum(1, keepdims=True) / d
    off = rstd * (c1_off + np.abs(xh) * c2_off + U * (4 * np.abs(g) + 4 * np.abs(c1) + 6 * np.abs(xh * c2)))
    if dres is not None:
        dx = dx + dres
        off = off + 2 * U * np.abs(dres)
    n = rows / 4 + 40  # rows in a row in one thread at most (the column kernel), and the trees above it
    dgamma, dbeta = (dy * xh).sum(0), dy.sum(0)
    return (dx, dgamma, dbeta), (off, (n + 3) * U * np.abs(dy * xh).sum(0) + 2.0 ** -126,
                                 n * U * np.abs(dy).sum(0) + 2.0 ** -126)


# ---- rows of logits

class Scores:
    """Everything about rows of logits (float64 [rows, cols]) and their labels; rows whose label is negative are dead."""

    def __init__(self, logits, labels, scale=1.0, alive=None):
        rows, cols = logits.shape
        labels = np.asarray(labels)
        self.scale = scale = float(np.float32(scale))
        self.alive = (labels >= 0) if alive is None else (labels >= 0) & alive
        at = np.maximum(labels, 0)
        r = np.arange(rows)
        x = np.where(self.alive[:, None], logits, 0.0)
        self.top = x.max(1)
        self.z = (x - self.top[:, None]) * scale
        e = np.exp(self.z)
        e_label = e[r, at]
        others = e.copy()
        others[r, at] = 0.0
        s = others.sum(1)
        self.p = e / (s + e_label)[:, None]
        self.rest = s / (s + e_label)                    # 1 - p(label)
        with np.errstate(divide="ignore"):
            self.logp = np.where(self.alive, -np.log1p(s / e_label), 0.0)
        self.logsum = np.where(self.alive, np.log1p(s + np.expm1(self.z[r, at])), 0.0)
        self.at, self.rows = at, r
        # relative error of S: each exponential's argument carries 4 roundings, the exponential 2, the sum its depth
        with np.errstate(invalid="ignore"):
            weighted = np.where(others > 0, others * np.abs(self.z), 0.0).sum(1)
        self.s_off = U * (4 * weighted / np.maximum(s, 1e-300) + depth(cols) + 4)
        self.top = np.where(self.alive, self.top, 0.0)

    @property
    def logp_off(self):
        """log p = -log1p(S / e): its derivative by log S is -(1 - p), so that a likely label's is known relative to its size;
        3e-8: the logarithm put together from parts."""
        return self.rest * (self.s_off + 12 * U) + 2 * U * np.abs(self.logp) + np.where(self.rest > 0.5, 4e-8, 0.0) + 1e-37

    @property
    def logsum_off(self):
        likely = self.z[self.rows, self.at] == 0
        small = np.where(likely & (self.rest <= 0.5), 0.0, 4e-8 + self.s_off + 12 * U)
        return self.rest * (self.s_off + 12 * U) + small + 2 * U * np.abs(self.logsum) + 1e-37

    def gradient(self, coeff, coeff_off=0.0, logsum_error=0.0):
        """d sum(coeff logp) / d logits and its bound; coeff_off: error of coeff, logsum_error: of the log sum that the
        exponentials are divided by."""
        coeff = np.where(self.alive, coeff, 0.0)[:, None]
        c_off = np.where(self.alive, coeff_off, 0.0)[:, None]
        l_off = np.broadcast_to(np.asarray(logsum_error, np.float64), self.alive.shape)[:, None]
        d = -coeff * self.scale * self.p
        with np.errstate(invalid="ignore"):
            off = np.where(self.p > 0, np.abs(coeff) * self.scale * self.p * (4 * U * np.abs(self.z) + 20 * U + l_off), 0.0)
        off = off + self.scale * self.p * c_off
        r, at = self.rows, self.at
        d[r, at] = coeff[:, 0] * self.scale * self.rest
        z_at = np.where(self.p[r, at] > 0, np.abs(self.z[r, at]), 0.0)
        off[r, at] = self.scale * (np.abs(coeff[:, 0]) * (self.p[r, at] * (4 * U * z_at + l_off[:, 0]) + 20 * U * self.rest)
                                   + c_off[:, 0] * self.rest)
        return d, off + 1e-37


def policy(scores, advantage, old=None, ref=None, weight=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0):
    """dict of (value, bound) for logp, kl, loss, loss_sum and dlogits"""
    clip_low, clip_high, kl_coef = (float(np.float32(v)) for v in (clip_low, clip_high, kl_coef))
    lp, lp_off, alive = scores.logp, scores.logp_off, scores.alive
    a = np.asarray(advantage, np.float64)
    w = np.ones_like(a) if weight is None else np.asarray(weight, np.float64)
    ratio = np.ones_like(lp) if old is None else np.exp(lp - np.asarray(old, np.float64))
    # the exponent is rounded to fp32
    ratio_off = 0.0 * lp if old is None else ratio * (lp_off + U * np.abs(lp - old) + 4 * U)
    with np.errstate(invalid="ignore"):
        clipped = np.where(a > 0, ratio > 1 + clip_high, ratio < 1 - clip_low) & (a != 0)
        surrogate = np.where(a == 0, 0.0, np.minimum(ratio * a, np.clip(ratio, 1 - clip_low, 1 + clip_high) * a))
        slope = np.where(clipped | (a == 0), 0.0, -a * ratio)
        slope_off = np.where(clipped | (a == 0), 0.0, np.abs(a) * ratio_off)
    loss, loss_off = -surrogate, slope_off
    kl, kl_off = np.zeros_like(lp), np.zeros_like(lp)
    if ref is not None:
        d = np.asarray(ref, np.float64) - lp
        d_off = lp_off + U * np.abs(d)
        up = np.expm1(d)
        kl = np.where(np.abs(d) < 1e-3, d * d * (0.5 + d / 6 + d * d / 24), up - d)
        # kl(d + o) - kl(d) = up(d) o + exp(xi) o^2 / 2 with xi between d and d + o: where d is of the size of its own error
        # o, up(d) is, too, and the square is as large as the first term
        kl_off = np.abs(up) * d_off + np.exp(np.abs(d)) * d_off ** 2 + np.where(np.abs(d) < 0.5, 12 * U * kl, 3 * U * (np.abs(up) + np.abs(d))) + 1e-37
        loss, loss_off = loss + kl_coef * kl, loss_off + abs(kl_coef) * kl_off
        slope = slope - kl_coef * up
        slope_off = slope_off + abs(kl_coef) * (np.exp(d) * d_off + 4 * U * np.abs(up))
    z = np.zeros_like(lp)
    loss, loss_off = np.where(alive, w * loss, z), np.where(alive, np.abs(w) * loss_off + 2 * U * np.abs(w * loss), z)
    coeff, coeff_off = w * slope, np.abs(w) * slope_off + 4 * U * np.abs(w * slope)
    return dict(logp=(lp, lp_off), kl=(np.where(alive, kl, z), np.where(alive, kl_off, z) + 1e-37),
                loss=(loss, loss_off + 1e-37),
                loss_sum=(loss.sum(keepdims=True), loss_off.sum(keepdims=True) + 2 * U * np.abs(loss).sum() + 1e-37),
                dlogits=scores.gradient(coeff, coeff_off, scores.s_off), coeff=coeff)


def preference(logp, ref, offsets, labels=None, beta=0.1, eps=0.0, pair_weight=None):
    """dict of (value, bound); offsets as the operator takes them"""
    tokens = len(logp)
    pairs = (len(offsets) - 1) // 2
    beta, eps = float(np.float32(beta)), float(np.float32(eps))
    pair_weight = float(np.float32(1.0 / pairs if pair_weight is None else pair_weight))
    counts = np.ones(tokens, bool) if labels is None else np.asarray(labels) >= 0
    diff = np.where(counts, np.where(counts, logp, 0.0).astype(np.float64) - np.where(counts, ref, 0.0), 0.0)
    rewards, losses = np.zeros(2 * pairs), np.zeros(pairs)
    dlogp, touched = np.zeros(tokens), np.zeros(tokens, bool)
    for p in range(pairs):
        at = []
        for i in range(3):
            v = max(int(offsets[2 * p + i]), at[-1] if at else 0)
            at.append(min(v, tokens))
        r = [beta * diff[at[i]:at[i + 1]].sum() for i in range(2)]
        rewards[2 * p:2 * p + 2] = r
        h = r[0] - r[1]
        soft = lambda v: np.logaddexp(0.0, v)
        losses[p] = (1 - eps) * soft(-h) + eps * soft(h)
        up = (eps - 1.0 / (1.0 + np.exp(h))) * beta * pair_weight
        dlogp[at[0]:at[1]], dlogp[at[1]:at[2]] = up, -up
        touched[at[0]:at[2]] = True
    dlogp = np.where(counts, dlogp, 0.0)
    total = np.array([pair_weight * losses.sum()])
    return dict(rewards=(rewards, 2 * U * np.abs(rewards) + 1e-12), pair_loss=(losses, 2 * U * np.abs(losses) + 1e-12),
                dlogp=(dlogp, 2 * U * np.abs(dlogp) + 1e-13), loss_sum=(total, 4 * U * np.abs(total) + 1e-12), touched=touched)
