"""The operators that train through the framework's row operators, as measurable cases: the backward passes of
LayerNorm and of the padding-masked softmax, the log-probabilities of labels under rows of logits, the preference loss
on paired sequences and the clipped policy loss with a KL term, each forward and backward from and to the logits.

`run` computes a case with elementary torch operations (own = False) or with the calls a user makes of
kernel_optimization_amd (own = True)."""
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # -- LayerNorm backward
        # one sequence of 128 tokens through BERT-base's LayerNorm: the smallest call, where latency counts
        dict(name="layernorm_backward_f32_128x768", op="layernorm_backward", dtype="f32", rows=128, cols=768,
             unbiased=False, dres=False, affine=True),
        # BERT-base's hidden states, batch 128 x sequence 128, in training precision
        dict(name="layernorm_backward_bf16_16384x768", op="layernorm_backward", dtype="bf16", rows=16384, cols=768,
             unbiased=False, dres=False, affine=True),
        # an odd width and a ragged token count: rows off 16-byte boundaries; the variance divides by cols - 1
        dict(name="layernorm_backward_f16_5003x1001", op="layernorm_backward", dtype="f16", rows=5003, cols=1001,
             unbiased=True, dres=True, affine=True),
        # a pre-norm block of a large model: the residual branch's gradient is added on the way
        dict(name="layernorm_backward_bf16_65536x4096", op="layernorm_backward", dtype="bf16", rows=65536, cols=4096,
             unbiased=False, dres=True, affine=True),
        # -- softmax backward
        # attention scores of BERT-base, batch 128 x 12 heads x sequence 128
        dict(name="softmax_backward_f32_196608x128", op="softmax_backward", dtype="f32", rows=196608, cols=128,
             rows_per_seq=0),
        # the padding-masked scores at sequence 512: 12 heads x 512 query rows share a sequence's length
        dict(name="softmax_backward_f16_786432x512_masked", op="softmax_backward", dtype="f16", rows=786432, cols=512,
             rows_per_seq=6144),
        # -- token log-probabilities
        # cross entropy on a short answer over a 50257-token vocabulary whose logits come from padded weights, and back
        dict(name="token_logprob_f16_32x50257", op="token_logprob", dtype="f16", rows=32, cols=50257, ld=50304,
             scale=1.0, backward=True),
        # scoring 4096 tokens with the reference model: no gradient
        dict(name="token_logprob_bf16_4096x128256", op="token_logprob", dtype="bf16", rows=4096, cols=128256,
             ld=128256, scale=1.0, backward=False),
        # -- preference loss: a training step's part from the logits to their gradient
        # two pairs of short answers over an odd vocabulary, fp32
        dict(name="preference_f32_2pairs_x1001", op="preference", dtype="f32", pairs=2, max_len=40, cols=1001, ld=1001,
             label_smoothing=0.0),
        # eight pairs of answers of up to 512 tokens; contiguous rows of 50257 columns start off 16-byte boundaries
        dict(name="preference_bf16_8pairs_x50257", op="preference", dtype="bf16", pairs=8, max_len=512, cols=50257,
             ld=50257, label_smoothing=0.1),
        # -- clipped policy loss with KL
        # a short rollout over BERT's vocabulary in fp32
        dict(name="policy_f32_16x30522", op="policy", dtype="f32", rows=16, cols=30522, ld=30522, scale=1.0,
             reference=True),
        # a micro-batch of 4096 tokens, temperature 0.7
        dict(name="policy_bf16_4096x128256", op="policy", dtype="bf16", rows=4096, cols=128256, ld=128256,
             scale=1.0 / 0.7, reference=True),
    ]


def _loss_scale(case):
    """Training in binary16 multiplies the loss so that small gradients stay above that type's smallest numbers."""
    return 4096.0 if case["dtype"] == "f16" else 1.0


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Half of the widths are whole 16-byte vectors, the others are whatever comes."""
    c = _log_uniform(rng, lo, hi)
    return max(8, c // 8 * 8) if rng.random() < 0.5 else c


def draw(rng: random.Random):
    op = rng.choice(["layernorm_backward", "softmax_backward", "token_logprob", "preference", "policy"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "layernorm_backward":
        cols = _width(rng, 16, 16384)
        rows = _log_uniform(rng, 1, min(65536, (1 << 27) // cols))
        return dict(op=op, dtype=dtype, rows=rows, cols=cols, unbiased=rng.random() < 0.5, dres=rng.random() < 0.5,
                    affine=rng.random() < 0.8)
    if op == "softmax_backward":
        cols = _width(rng, 4, 8192)
        rows = _log_uniform(rng, 1, min(786432, (1 << 27) // cols))
        return dict(op=op, dtype=dtype, rows=rows, cols=cols,
                    rows_per_seq=_log_uniform(rng, 1, rows) if rng.random() < 0.5 else 0)
    if op == "preference":
        cols = _width(rng, 100, 131072)
        max_len = _log_uniform(rng, 2, 512)
        pairs = rng.randint(1, max(1, min(16, (1 << 27) // (2 * max_len * cols))))
        ld = cols if rng.random() < 0.5 else (cols + 63) // 64 * 64
        return dict(op=op, dtype=dtype, pairs=pairs, max_len=max_len, cols=cols, ld=ld,
                    label_smoothing=rng.choice([0.0, 0.1]))
    cols = _width(rng, 100, 262144)
    rows = _log_uniform(rng, 1, min(8192, (1 << 27) // cols))
    ld = cols if rng.random() < 0.5 else (cols + 63) // 64 * 64
    case = dict(op=op, dtype=dtype, rows=rows, cols=cols, ld=ld, scale=rng.choice([1.0, 1.0 / 0.7, 0.8]))
    if op == "policy":
        case["reference"] = rng.random() < 0.7
    else:
        case["backward"] = rng.random() < 0.5
    return case


# ---- inputs --------------------------------------------------------------------------------------------------------

def _normal(g, shape, mean, std, dtype):
    return (torch.randn(shape, device="cuda", generator=g) * std + mean).to(dtype)


def _uniform(g, shape, lo, hi):
    return torch.rand(shape, device="cuda", generator=g) * (hi - lo) + lo


def _logits(g, rows, cols, ld, dtype):
    """Logits of a language model and the labels drawn from it: noise of standard deviation 2, the label's raised so that
    most labels are likely; one row in eight is a prompt's, without a label."""
    logits = _normal(g, (rows, ld), 0.0, 2.0, dtype)
    labels = torch.randint(0, cols, (rows,), device="cuda", generator=g)
    at = torch.arange(rows, device="cuda")
    logits[at, labels] = (logits[at, labels].float() + _uniform(g, (rows,), 4.0, 14.0)).to(dtype)
    prompt = _uniform(g, (rows,), 0.0, 1.0) < 0.125
    return logits, torch.where(prompt, -1, labels).to(torch.int32)


def _label_logprob(logits, labels, cols, scale):
    """Log-probability of each row's label in 64 bits, 0 for rows without one."""
    out = torch.zeros(labels.numel(), dtype=torch.float64, device="cuda")
    step = max(1, (1 << 26) // cols)
    for r in range(0, labels.numel(), step):
        z = logits[r:r + step, :cols].double() * scale
        lab = labels[r:r + step].long()
        lp = z.gather(1, lab.clamp(min=0)[:, None])[:, 0] - torch.logsumexp(z, 1)
        out[r:r + step] = torch.where(lab < 0, 0.0, lp)
    return out


def _sequence_lengths(case, seed):
    """Lengths of the case's answers: the same ones for every seed, in an order of the seed's own."""
    fixed = random.Random(case["pairs"] * 1000 + case["max_len"])
    lens = [fixed.randint(max(1, case["max_len"] // 4), case["max_len"]) for _ in range(2 * case["pairs"])]
    random.Random(seed).shuffle(lens)
    return lens


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    op, cols = case["op"], case["cols"]
    s = dict(case=case)
    if op == "layernorm_backward":
        rows = case["rows"]
        s["x"] = _normal(g, (rows, cols), 0.5, 2.0, dt)
        s["dy"] = _normal(g, (rows, cols), 0.0, 1.0, dt)
        s["gamma"] = _normal(g, (cols,), 1.0, 0.1, dt) if case["affine"] else None
        s["dres"] = _normal(g, (rows, cols), 0.0, 1.0, dt) if case["dres"] else None
        # what the forward pass left: fp32 mean and rstd of every row
        x = s["x"].float()
        mean = x.mean(1, dtype=torch.float32)
        denominator = max(1, cols - 1) if case["unbiased"] else cols
        var = (x - mean[:, None]).square().sum(1) / denominator
        s["mean"], s["rstd"] = mean, torch.rsqrt(var + 1e-5)
        s["dx"] = torch.empty_like(s["x"])
        s["dgamma"] = torch.empty(cols, device="cuda")
        s["dbeta"] = torch.empty(cols, device="cuda")
    elif op == "softmax_backward":
        rows, rps = case["rows"], case["rows_per_seq"]
        x = _normal(g, (rows, cols), 0.0, 4.0, torch.float32)
        s["lens"] = None
        if rps:
            nseq = (rows + rps - 1) // rps
            s["lens"] = torch.randint(max(1, cols // 8), cols + 1, (nseq,), device="cuda", generator=g, dtype=torch.int32)
            per_row = s["lens"].repeat_interleave(rps)[:rows]
            x.masked_fill_(torch.arange(cols, device="cuda") >= per_row[:, None], -10000.0)
        s["y"] = torch.softmax(x, 1).to(dt)
        del x
        s["dy"] = _normal(g, (rows, cols), 0.0, 1.0, dt)
        s["dx"] = torch.empty_like(s["y"])
    else:
        if op == "preference":
            lens = _sequence_lengths(case, seed)
            s["offsets"] = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")
            rows = sum(lens)
        else:
            rows = case["rows"]
        s["rows"] = rows
        s["logits"], s["labels"] = _logits(g, rows, cols, case["ld"], dt)
        scale = case.get("scale", 1.0)
        s["logp"] = torch.empty(rows, device="cuda")
        if op != "policy":
            s["row_stats"] = torch.empty((rows, 2), device="cuda")
        if op == "token_logprob" and case["backward"]:
            s["dlogp"] = _normal(g, (rows,), -1.0, 0.2, torch.float32) * (_loss_scale(case) / rows)
            s["dlogits"] = torch.empty_like(s["logits"])
        if op != "token_logprob":
            lp = _label_logprob(s["logits"], s["labels"], cols, scale)
            drift = torch.randn(rows, device="cuda", generator=g).double()
            if op == "preference":
                # training has moved whole answers: a drift per token and one in common, as rewards of size 1 come from
                drift += torch.randn(2 * case["pairs"], device="cuda", generator=g).double().repeat_interleave(
                    torch.tensor(lens, device="cuda"))
            s["ref_logp"] = torch.where(s["labels"] < 0, 0.0, lp + 0.1 * drift).float()
            s["dlogits"] = torch.empty_like(s["logits"])
            s["loss_sum"] = torch.empty(1, device="cuda")
        if op == "preference":
            s["dlogp"] = torch.empty(rows, device="cuda")
            s["pair_loss"] = torch.empty(case["pairs"], device="cuda")
            s["rewards"] = torch.empty(2 * case["pairs"], device="cuda")
        if op == "policy":
            # the policy has moved since the rollout: ratios mostly near 1, a tail beyond the clip range.  Which side of the
            # clip border a ratio lies on is a yes or no, so no ratio is put within 1e-3 of one.
            shift = 0.15 * torch.randn(rows, device="cuda", generator=g).double()
            for border in (math.log(1.0 - 0.2), math.log(1.0 + 0.28)):
                near = (shift - border).abs() < 1e-3
                shift = torch.where(near, shift + 3e-3, shift)
            s["old_logp"] = torch.where(s["labels"] < 0, 0.0, lp - shift).float()
            if not case["reference"]:
                s["ref_logp"] = None
            s["advantage"] = _normal(g, (rows,), 0.0, 1.0, torch.float32)
            s["weight"] = (_uniform(g, (rows,), 0.5, 1.5) * (_loss_scale(case) / rows)).float()
            s["loss"] = torch.empty(rows, device="cuda")
            s["kl"] = torch.empty(rows, device="cuda")
    if own:
        import kernel_optimization_amd as ko
        if op == "layernorm_backward":
            n = ko.layernorm_backward_workspace_bytes(case["rows"], cols)
        elif op == "softmax_backward":
            n = ko.softmax_backward_workspace_bytes(case["rows"], cols)
        else:
            n = ko.token_logprob_workspace_bytes(s["rows"], cols)
        s["workspace"] = torch.empty(n, dtype=torch.uint8, device="cuda") if n else None
        s["workspace_bytes"] = n
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    return _PLAIN[op](state)


def _plain_layernorm_backward(s):
    case, dt = s["case"], s["x"].dtype
    cols = case["cols"]
    dy = s["dy"].float()
    rstd = s["rstd"][:, None]
    xhat = (s["x"].float() - s["mean"][:, None]) * rstd
    g = dy if s["gamma"] is None else dy * s["gamma"].float()
    c1 = g.sum(1, keepdim=True) / cols
    c2 = (g * xhat).sum(1, keepdim=True) / (max(1, cols - 1) if case["unbiased"] else cols)
    dx = rstd * (g - c1 - xhat * c2)
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return dx.to(dt), (dy * xhat).sum(0), dy.sum(0)


def _plain_softmax_backward(s):
    case = s["case"]
    y, dy = s["y"].float(), s["dy"].float()
    dot = torch.where(y != 0, y * dy, 0.0).sum(1, keepdim=True)
    dx = y * (dy - dot)
    if s["lens"] is not None:
        per_row = s["lens"].repeat_interleave(case["rows_per_seq"])[:case["rows"]]
        dx = torch.where(torch.arange(case["cols"], device="cuda") < per_row[:, None], dx, 0.0)
    return dx.to(s["y"].dtype)


def _plain_logprob(logits, labels, cols, scale):
    """logp in 64 bits, (max, log sum), and what the gradient is made of: the other columns' exp(scale (x - max)) and their
    sum next to the whole one.  The label's own column stays out of the sum: of a likely label, whose logp is close to
    zero, the others' sum is what matters, and 1 + it would round it away."""
    x = logits[:, :cols].float()
    m = x.max(1, keepdim=True).values
    lab = labels.long()
    at = lab.clamp(min=0)[:, None]
    z = ((x.gather(1, at) - m) * scale).double()
    e = torch.exp((x - m) * scale)
    e.scatter_(1, at, 0.0)
    others = e.sum(1, keepdim=True, dtype=torch.float64)
    logsum = torch.log1p(others + torch.expm1(z))
    some = lab >= 0
    logp = torch.where(some, (z - logsum)[:, 0], 0.0)
    stats = torch.where(some[:, None], torch.cat([m, logsum.float()], 1), 0.0)
    return logp, stats, e, others, others + torch.exp(z)


def _plain_dlogits(e, others, total, labels, dlogp, scale, dtype):
    coeff = torch.where(labels >= 0, dlogp.double() * scale, 0.0)[:, None]
    d = e * (-coeff / total).float()
    d.scatter_(1, labels.long().clamp(min=0)[:, None], (coeff * (others / total)).float())
    return d.to(dtype)


def _plain_token_logprob(s):
    case = s["case"]
    logp, stats, *parts = _plain_logprob(s["logits"], s["labels"], case["cols"], case["scale"])
    if not case["backward"]:
        return logp.float(), stats
    return logp.float(), stats, _plain_dlogits(*parts, s["labels"], s["dlogp"], case["scale"], s["logits"].dtype)


def _plain_preference(s):
    case = s["case"]
    pairs, eps = case["pairs"], case["label_smoothing"]
    logp, _, *parts = _plain_logprob(s["logits"], s["labels"], case["cols"], 1.0)
    ratio = torch.where(s["labels"] >= 0, logp - s["ref_logp"].double(), 0.0)
    seq = torch.bucketize(torch.arange(s["rows"], device="cuda", dtype=torch.int32), s["offsets"][1:], right=True)
    sums = torch.zeros(2 * pairs, dtype=torch.float64, device="cuda").index_add_(0, seq, ratio)
    rewards = _PREFERENCE_BETA * sums
    h = rewards[0::2] - rewards[1::2]
    softplus = torch.log1p(torch.exp(-h.abs()))
    pair_loss = (1.0 - eps) * (softplus + (-h).clamp(min=0)) + eps * (softplus + h.clamp(min=0))
    pair_weight = _loss_scale(case) / pairs
    dh = (eps - (1.0 / (1.0 + torch.exp(h)))) * (_PREFERENCE_BETA * pair_weight)
    dlogp = torch.stack([dh, -dh], 1).reshape(-1)[seq]
    dlogits = _plain_dlogits(*parts, s["labels"], dlogp, 1.0, s["logits"].dtype)
    return pair_loss.float(), rewards.float(), (pair_loss.sum() * pair_weight).float().reshape(1), dlogits


def _plain_policy(s):
    case = s["case"]
    lp, _, *parts = _plain_logprob(s["logits"], s["labels"], case["cols"], case["scale"])
    some = s["labels"] >= 0
    adv, w = s["advantage"].double(), s["weight"].double()
    ratio = torch.exp(lp - s["old_logp"].double())
    surrogate = torch.minimum(ratio * adv, ratio.clamp(1.0 - _CLIP_LOW, 1.0 + _CLIP_HIGH) * adv)
    free = torch.where(adv > 0, ratio <= 1.0 + _CLIP_HIGH, ratio >= 1.0 - _CLIP_LOW)
    dlogp = -torch.where(free, ratio * adv, 0.0)
    kl = torch.zeros_like(lp)
    if s["ref_logp"] is not None:
        d = s["ref_logp"].double() - lp
        kl = torch.exp(d) - 1.0 - d
        dlogp = dlogp + _KL_COEF * (1.0 - torch.exp(d))
    kl = torch.where(some, kl, 0.0)
    loss = torch.where(some, w * (_KL_COEF * kl - surrogate), 0.0)
    dlogits = _plain_dlogits(*parts, s["labels"], w * dlogp, case["scale"], s["logits"].dtype)
    return lp.float(), kl.float(), loss.float(), loss.sum().float().reshape(1), dlogits


_PREFERENCE_BETA = 0.1
_CLIP_LOW, _CLIP_HIGH, _KL_COEF = 0.2, 0.28, 0.05

_PLAIN = dict(layernorm_backward=_plain_layernorm_backward, softmax_backward=_plain_softmax_backward,
              token_logprob=_plain_token_logprob, preference=_plain_preference, policy=_plain_policy)


# ---- the framework's calls -------------------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _kind(ko, case):
    return {"f16": ko.F16, "bf16": ko.BF16}[case["dtype"]]


def _own_layernorm_backward(s):
    import kernel_optimization_amd as ko
    case = s["case"]
    args = (_ptr(s["dy"]), _ptr(s["x"]), _ptr(s["mean"]), _ptr(s["rstd"]), _ptr(s["dx"]), case["rows"], case["cols"])
    kw = dict(gamma=_ptr(s["gamma"]), dres=_ptr(s["dres"]), dgamma=_ptr(s["dgamma"]), dbeta=_ptr(s["dbeta"]),
              unbiased=case["unbiased"], workspace=_ptr(s["workspace"]), workspace_bytes=s["workspace_bytes"],
              stream=_stream())
    if case["dtype"] == "f32":
        ko.layernorm_backward(*args, **kw)
    else:
        ko.layernorm_backward16(*args, dtype=_kind(ko, case), **kw)
    return s["dx"], s["dgamma"], s["dbeta"]


def _own_softmax_backward(s):
    import kernel_optimization_amd as ko
    case = s["case"]
    args = (_ptr(s["y"]), _ptr(s["dy"]), _ptr(s["dx"]), case["rows"], case["cols"])
    kw = dict(valid_len=_ptr(s["lens"]), rows_per_seq=case["rows_per_seq"], workspace=_ptr(s["workspace"]),
              workspace_bytes=s["workspace_bytes"], stream=_stream())
    if case["dtype"] == "f32":
        ko.softmax_backward(*args, **kw)
    else:
        ko.softmax_backward16(*args, dtype=_kind(ko, case), **kw)
    return s["dx"]


def _own_logprob(ko, s, scale):
    case = s["case"]
    args = (_ptr(s["logits"]), _ptr(s["labels"]), _ptr(s["logp"]), s["rows"], case["cols"])
    kw = dict(ld=case["ld"], scale=scale, row_stats=_ptr(s["row_stats"]), workspace=_ptr(s["workspace"]),
              workspace_bytes=s["workspace_bytes"], stream=_stream())
    if case["dtype"] == "f32":
        ko.token_logprob(*args, **kw)
    else:
        ko.token_logprob16(*args, dtype=_kind(ko, case), **kw)


def _own_token_logprob(s):
    import kernel_optimization_amd as ko
    case = s["case"]
    _own_logprob(ko, s, case["scale"])
    if not case["backward"]:
        return s["logp"], s["row_stats"]
    return s["logp"], s["row_stats"], _own_dlogits(ko, s, case["scale"])


def _own_dlogits(ko, s, scale):
    case = s["case"]
    args = (_ptr(s["logits"]), _ptr(s["labels"]), _ptr(s["row_stats"]), _ptr(s["dlogp"]), _ptr(s["dlogits"]),
            s["rows"], case["cols"])
    kw = dict(ld=case["ld"], ldd=case["ld"], scale=scale, stream=_stream())
    if case["dtype"] == "f32":
        ko.token_logprob_backward(*args, **kw)
    else:
        ko.token_logprob_backward16(*args, dtype=_kind(ko, case), **kw)
    return s["dlogits"][:, :case["cols"]]


def _own_preference(s):
    import kernel_optimization_amd as ko
    case = s["case"]
    _own_logprob(ko, s, 1.0)
    ko.preference_loss(_ptr(s["logp"]), _ptr(s["ref_logp"]), _ptr(s["offsets"]), case["pairs"], s["rows"],
                       _ptr(s["pair_loss"]), labels=_ptr(s["labels"]), beta=_PREFERENCE_BETA,
                       label_smoothing=case["label_smoothing"], pair_weight=_loss_scale(case) / case["pairs"],
                       rewards=_ptr(s["rewards"]), dlogp=_ptr(s["dlogp"]), loss_sum=_ptr(s["loss_sum"]),
                       stream=_stream())
    return s["pair_loss"], s["rewards"], s["loss_sum"], _own_dlogits(ko, s, 1.0)


def _own_policy(s):
    import kernel_optimization_amd as ko
    case = s["case"]
    args = (_ptr(s["logits"]), _ptr(s["labels"]), _ptr(s["advantage"]), _ptr(s["loss"]), s["rows"], case["cols"])
    kw = dict(ld=case["ld"], old_logp=_ptr(s["old_logp"]), ref_logp=_ptr(s["ref_logp"]), weight=_ptr(s["weight"]),
              scale=case["scale"], clip_low=_CLIP_LOW, clip_high=_CLIP_HIGH, kl_coef=_KL_COEF, logp=_ptr(s["logp"]),
              kl=_ptr(s["kl"]), loss_sum=_ptr(s["loss_sum"]), dlogits=_ptr(s["dlogits"]), ldd=case["ld"],
              workspace=_ptr(s["workspace"]), workspace_bytes=s["workspace_bytes"], stream=_stream())
    if case["dtype"] == "f32":
        ko.policy_loss(*args, **kw)
    else:
        ko.policy_loss16(*args, dtype=_kind(ko, case), **kw)
    return s["logp"], s["kl"], s["loss"], s["loss_sum"], s["dlogits"][:, :case["cols"]]


_OWN = dict(layernorm_backward=_own_layernorm_backward, softmax_backward=_own_softmax_backward,
            token_logprob=_own_token_logprob, preference=_own_preference, policy=_own_policy)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    size, cols, op = _SIZE[case["dtype"]], case["cols"], case["op"]
    if op == "layernorm_backward":
        n = case["rows"] * cols
        streams = 3 + (1 if case["dres"] else 0)
        return dict(bytes=streams * n * size + 8 * case["rows"] + (size if case["affine"] else 0) * cols + 8 * cols,
                    flops=14 * n)
    if op == "softmax_backward":
        n = case["rows"] * cols
        # with a mask the mean valid length is 9/16 of the columns; the rest is written only
        read = 2 * n * 9 // 16 if case["rows_per_seq"] else 2 * n
        return dict(bytes=(read + n) * size, flops=4 * n)
    if op == "preference":
        rows = sum(_sequence_lengths(case, 0))
        # the loss of a pair stands between reading its logits and writing their gradient: two reads, one write; rows without
        # a label (one in eight) are only written
        n = rows * cols
        return dict(bytes=(2 * n * 7 // 8 + n) * size + 24 * rows, flops=9 * n * 7 // 8)
    n = case["rows"] * cols
    if op == "token_logprob":
        # the gradient waits for what comes of the log-probabilities: a second read, and a write of all rows
        passes = 7 * n // 8 + (7 * n // 8 + n if case["backward"] else 0)
        return dict(bytes=passes * size + 20 * case["rows"], flops=(9 if case["backward"] else 4) * n * 7 // 8)
    return dict(bytes=(n * 7 // 8 + n) * size + 36 * case["rows"], flops=9 * n * 7 // 8)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op, cols = case["op"], case["cols"]
    if op == "layernorm_backward":
        denominator = max(1, cols - 1) if case["unbiased"] else cols
        dx = torch.empty((case["rows"], cols), dtype=torch.float64, device="cuda")
        dgamma = torch.zeros(cols, dtype=torch.float64, device="cuda")
        dbeta = torch.zeros(cols, dtype=torch.float64, device="cuda")
        step = max(1, (1 << 25) // cols)
        for r in range(0, case["rows"], step):
            rows = slice(r, r + step)
            dy, x = s["dy"][rows].double(), s["x"][rows].double()
            mean, rstd = s["mean"][rows].double()[:, None], s["rstd"][rows].double()[:, None]
            dev = x - mean
            up = dy if s["gamma"] is None else dy * s["gamma"].double()
            # through the shift, the mean and the variance
            dvar = -0.5 * rstd ** 3 * torch.sum(up * dev, 1, keepdim=True)
            dx[rows] = up * rstd - torch.mean(up, 1, keepdim=True) * rstd + dvar * 2.0 * dev / denominator
            if s["dres"] is not None:
                dx[rows] += s["dres"][rows].double()
            dgamma += torch.sum(dy * dev * rstd, 0)
            dbeta += torch.sum(dy, 0)
        return dx, dgamma, dbeta
    if op == "softmax_backward":
        dx = torch.zeros((case["rows"], cols), dtype=torch.float64, device="cuda")
        step = max(1, (1 << 25) // cols)
        for r in range(0, case["rows"], step):
            y, dy = s["y"][r:r + step].double(), s["dy"][r:r + step].double()
            weighted = y * dy
            d = weighted - y * torch.sum(weighted, 1, keepdim=True)
            if s["lens"] is not None:
                seq = torch.arange(r, min(r + step, case["rows"]), device="cuda") // case["rows_per_seq"]
                d.masked_fill_(torch.arange(cols, device="cuda")[None] >= s["lens"][seq][:, None], 0.0)
            dx[r:r + step] = d
        return dx
    rows = s["rows"]
    scale = case.get("scale", 1.0)
    labels = s["labels"].long()
    live = labels >= 0
    logp = _label_logprob(s["logits"], s["labels"], cols, scale)
    if op == "token_logprob":
        top = torch.where(live, s["logits"][:, :cols].amax(1).double(), 0.0)
        at = s["logits"].gather(1, labels.clamp(min=0)[:, None])[:, 0].double()
        head = [logp, torch.stack([top, torch.where(live, (at - top) * scale - logp, 0.0)], 1)]
        if not case["backward"]:
            return tuple(head)
        dlogp = s["dlogp"].double()
    elif op == "preference":
        eps, pairs = case["label_smoothing"], case["pairs"]
        bounds = s["offsets"].tolist()
        rewards, dlogp = [], torch.zeros(rows, dtype=torch.float64, device="cuda")
        for q in range(2 * pairs):
            cut = slice(bounds[q], bounds[q + 1])
            rewards.append(_PREFERENCE_BETA * float(((logp[cut] - s["ref_logp"][cut].double()) * live[cut]).sum()))
        losses = []
        for p in range(pairs):
            h = rewards[2 * p] - rewards[2 * p + 1]
            log_sig = lambda v: -math.log1p(math.exp(-v)) if v >= 0 else v - math.log1p(math.exp(v))
            losses.append(-(1.0 - eps) * log_sig(h) - eps * log_sig(-h))
            slope = (eps * math.exp(log_sig(h)) - (1.0 - eps) * math.exp(log_sig(-h))) * _PREFERENCE_BETA
            slope *= _loss_scale(case) / pairs
            dlogp[bounds[2 * p]:bounds[2 * p + 1]] = slope
            dlogp[bounds[2 * p + 1]:bounds[2 * p + 2]] = -slope
        head = [torch.tensor(v, dtype=torch.float64, device="cuda") for v in (losses, rewards, [sum(losses) * _loss_scale(case) / pairs])]
    else:
        ratio = torch.exp(logp - s["old_logp"].double())
        adv, w = s["advantage"].double(), s["weight"].double()
        clipped = torch.clamp(ratio, 1.0 - _CLIP_LOW, 1.0 + _CLIP_HIGH)
        surrogate = torch.minimum(ratio * adv, clipped * adv)
        slope = torch.where(ratio * adv <= clipped * adv, -ratio * adv, 0.0)
        kl = torch.zeros_like(logp)
        if s["ref_logp"] is not None:
            d = s["ref_logp"].double() - logp
            kl = torch.expm1(d) - d
            slope = slope - _KL_COEF * torch.expm1(d)
        dlogp = w * slope
        kl = kl * live
        loss = w * (_KL_COEF * kl - surrogate) * live
        head = [logp, kl, loss, loss.sum().reshape(1)]
    dlogits = torch.empty((rows, cols), dtype=torch.float64, device="cuda")
    step = max(1, (1 << 25) // cols)
    for r in range(0, rows, step):
        coeff = (dlogp * live * scale)[r:r + step, None]
        d = -coeff * torch.softmax(s["logits"][r:r + step, :cols].double() * scale, 1)
        hit = torch.arange(d.shape[0], device="cuda")
        d[hit, labels[r:r + step].clamp(min=0)] += coeff[:, 0]
        dlogits[r:r + step] = d
    return (*head, dlogits)
