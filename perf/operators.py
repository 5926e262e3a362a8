"""The two ends of a network on tokens, timed: the embedding of token ids with its gradient, and the losses on choices
(label log-probabilities, clipped policy loss with a KL term, preference loss) with theirs.

A network's outputs are spike values z, its logits are -z, and an output that does not spike is 1e5. A row whose label is
outside the classes does not count, a token outside the table never spikes.

With `own` the calls are the framework's entry points; without it the same formulas in elementary torch operations.
"""
import math
import random

import torch

own = False

NO_SPIKE = 1e5
BETA, SMOOTHING = 0.1, 0.05                  # preference loss
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.05   # policy loss
MOST_LOGITS = 8192 * 50021                   # of a drawn case, as of the largest listed one
MOST_TABLE = 131072 * 512


# ------------------------------------------------------------------------------------------------- the cases
def _embed(N, V, D, mode, spikes, scale, pad):
    """mode "lookup": evaluation, nothing asks for a gradient; "train": lookup and the table's gradient."""
    return dict(op="embed", N=N, V=V, D=D, mode=mode, spikes=spikes, scale=scale, pad=pad)


def _logp(R, J, mode):
    return dict(op="logp", R=R, J=J, mode=mode)


def _policy(R, J):
    return dict(op="policy", R=R, J=J)


def _prefer(P, R, J):
    return dict(op="prefer", P=P, R=R, J=J)


def listed():
    return [
        # the next token of one request, into a 784-input network: latency
        dict(_embed(1, 10007, 784, "lookup", True, 1.0, False), name="embed one token"),
        # a batch of 64 texts of 1024 tokens, evaluation
        dict(_embed(64 * 1024, 131072, 512, "lookup", False, 8.0, False), name="embed lookup 65536x512"),
        # a step on a small vocabulary and a small batch, padded texts
        dict(_embed(300, 1000, 100, "train", True, 1.0, True), name="embed train 300x100"),
        # odd sizes: rows of the table that start anywhere, a prime vocabulary
        dict(_embed(7 * 1001, 50021, 129, "train", True, 0.5, True), name="embed train 7007x129"),
        # a large step: every second token is one of a few hundred, many rows of the table are not touched
        dict(_embed(128 * 1024, 131072, 512, "train", False, 8.0, False), name="embed train 131072x512"),
        # fine-tuning on the ten classes of the benchmark networks, log-probabilities differentiated
        dict(_logp(256, 10, "grad"), name="logp grad 256x10"),
        # scoring texts by a frozen network: what the losses below take as old and reference log-probabilities
        dict(_logp(4096, 32768, "score"), name="logp score 4096x32768"),
        # ten actions, one decision a sample
        dict(_policy(1024, 10), name="policy 1024x10"),
        # a thousand classes, the outputs of the ImageNet-shaped network
        dict(_policy(16384, 1000), name="policy 16384x1000"),
        # tokens of a vocabulary with an odd size: rows that start anywhere
        dict(_policy(8192, 50021), name="policy 8192x50021"),
        # a few short pairs
        dict(_prefer(8, 517, 1000), name="prefer 8 pairs 517x1000"),
        # pairs of texts over a vocabulary
        dict(_prefer(16, 8192, 32768), name="prefer 16 pairs 8192x32768"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("embed", "embed", "logp", "policy", "policy", "prefer"))
    if op == "embed":
        N, V, D = _log_int(rng, 1, 131072), _log_int(rng, 2, 131072), _log_int(rng, 8, 1024)
        most = MOST_TABLE // max(N, V)
        D = min(D, most)
        if rng.random() < 0.5 and D > 4:
            D -= D % 4
        return _embed(N, V, D, rng.choice(("lookup", "train", "train")), rng.random() < 0.5, rng.choice((0.5, 1.0, 8.0)),
                      rng.random() < 0.5)
    J = _log_int(rng, 2, 65536)
    if rng.random() < 0.5 and J > 4:
        J -= J % 4
    R = min(_log_int(rng, 1, 65536), MOST_LOGITS // J)
    if op == "logp":
        return _logp(R, J, rng.choice(("score", "grad")))
    if op == "policy":
        return _policy(R, J)
    P = _log_int(rng, 1, 64)
    return _prefer(P, max(R, 2 * P), J)


# ------------------------------------------------------------------------------------------------- inputs
def _tokens(N, V, gen):
    """Ids in order of frequency, as vocabularies are: the chance of an id falls with its place (log-uniform)."""
    u = torch.rand(N, device="cuda", dtype=torch.float64, generator=gen)
    return ((u * math.log(V + 1)).exp().floor().long() - 1).clamp_(0, V - 1)


def _spikes_and_labels(R, J, gen):
    """Spike values as a network's last layer gives them (three in ten do not spike, now and then a whole row) and labels
    drawn from softmax(-z), one row in sixteen without one; and the labels' log-probabilities."""
    z = torch.randn(R, J, device="cuda", generator=gen).abs_().mul_(3.0).add_(1.0)
    label = torch.empty(R, dtype=torch.int64, device="cuda")
    logp = torch.empty(R, device="cuda")
    step = max(1, (1 << 27) // J)
    starts = range(0, R, step)
    for r in starts:
        part = z[r:r + step]
        part.masked_fill_(torch.rand(part.shape, device="cuda", generator=gen) < 0.3, NO_SPIKE)
        part.masked_fill_(torch.rand(part.shape[0], 1, device="cuda", generator=gen) < 1 / 512, NO_SPIKE)
        gumbel = torch.rand(part.shape, device="cuda", generator=gen).clamp_(1e-12, 1 - 1e-7).log_().neg_().log_()
        label[r:r + step] = (part + gumbel).argmin(1)
        logp[r:r + step] = torch.log_softmax(-part, 1).gather(1, label[r:r + step, None])[:, 0]
    label.masked_fill_(torch.rand(R, device="cuda", generator=gen) < 1 / 16, -1)
    return z, label, logp


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)
    s = dict(case=c)
    noise = lambda n: torch.randn(n, device="cuda", generator=gen)  # noqa: E731
    if c["op"] == "embed":
        N, V, D = c["N"], c["V"], c["D"]
        s["ids"] = _tokens(N, V, gen)
        if c["pad"]:
            s["ids"][N - N // 8:] = -1               # the ends of texts that are shorter than the batch's longest
        # spike times in [0, 1) where they are encoded, spike values otherwise
        table = torch.rand(V, D, device="cuda", generator=gen)
        s["table"] = table if c["spikes"] else table.add_(1.0)
        if c["mode"] == "train":
            s["table"].requires_grad_(True)
            s["g"] = torch.randn(N, D, device="cuda", generator=gen)
        return s
    R, J = c["R"], c["J"]
    z, label, logp = _spikes_and_labels(R, J, gen)
    s.update(z=z, label=label)
    if c["op"] == "logp":
        if c["mode"] == "grad":
            z.requires_grad_(True)
            s["g"] = noise(R)
        return s
    z.requires_grad_(True)
    if c["op"] == "policy":
        s.update(old=logp + 0.2 * noise(R), ref=logp + 0.3 * noise(R), advantage=noise(R))
        return s
    P = c["P"]
    host = random.Random(seed)
    used = R - R // 64                               # the last rows belong to no text
    cuts = sorted(host.randrange(used + 1) for _ in range(2 * P - 1))
    s["starts"] = torch.tensor([0] + cuts + [used], dtype=torch.int64, device="cuda")
    label.masked_fill_(torch.rand(R, device="cuda", generator=gen) < 0.2, -1)      # the prompts' rows
    total = torch.cat((logp.new_zeros(1, dtype=torch.float64), (logp.double() * (label >= 0)).cumsum(0)))[s["starts"]]
    s["ref"] = (total[1:] - total[:-1] + 8.0 * noise(2 * P)).float()
    return s


# ------------------------------------------------------------------------------------------------- the plain form
def _row_sums(z):
    """max(-z), exp(-z - max) and its sum, of every row."""
    top = (-z).amax(1)
    e = torch.exp(-z - top[:, None])
    return top, e, e.sum(1, dtype=torch.float64)


def _label_logp(z, label, top, total):
    counts = (label >= 0) & (label < z.shape[1])
    at = label.clamp(0, z.shape[1] - 1)
    logp = (-z.gather(1, at[:, None])[:, 0].double() - top.double()) - total.log()
    return torch.where(counts, logp, 0.0), counts, at


def _logits_gradient(e, total, factor, counts, at):
    """factor * (softmax(-z) - onehot), factor a number per row in 64 bits."""
    factor = torch.where(counts, factor, 0.0)
    g = e * (factor / total).float()[:, None]
    rows = torch.arange(len(at), device=at.device)
    g[rows, at] -= factor.float()
    return g


def _plain_embed(s):
    c, ids, table = s["case"], s["ids"], s["table"].detach()
    there = (ids >= 0) & (ids < c["V"])
    at = ids.clamp(0, c["V"] - 1)
    y = table[at] * c["scale"]
    if c["spikes"]:
        y = y.exp()
    y[~there] = NO_SPIKE
    if c["mode"] == "lookup":
        return [y]
    grad = torch.zeros(c["V"], c["D"], dtype=torch.float64, device="cuda")       # long sums: the frequent tokens
    grad.index_add_(0, at[there], s["g"][there].double())
    if c["spikes"]:
        grad *= (table * c["scale"]).exp()
    return [y, (grad * c["scale"]).float()]


def _plain_logp(s):
    z, label = s["z"].detach(), s["label"]
    top, e, total = _row_sums(z)
    logp, counts, at = _label_logp(z, label, top, total)
    if s["case"]["mode"] == "score":
        return [logp.float()]
    return [logp.float(), _logits_gradient(e, total, s["g"].double(), counts, at)]


def _plain_policy(s):
    z = s["z"].detach()
    top, e, total = _row_sums(z)
    logp, counts, at = _label_logp(z, s["label"], top, total)
    n = counts.sum().clamp(min=1)
    adv = s["advantage"].double()
    ratio = torch.exp(logp - s["old"].double())
    lower, upper = 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH
    clipped = ((adv > 0) & (ratio > upper)) | ((adv < 0) & (ratio < lower))
    away = s["ref"].double() - logp
    kl = away.expm1() - away
    gain = torch.where(clipped, ratio.clamp(lower, upper), ratio) * adv
    loss = torch.where(counts, KL_COEF * kl - gain, 0.0).sum() / n
    factor = (-KL_COEF * away.expm1() - torch.where(clipped, 0.0, ratio * adv)) / n
    stats = torch.stack((torch.where(counts, kl, 0.0).sum() / n, (clipped & counts).sum() / n))
    return [loss.float(), stats.float(), _logits_gradient(e, total, factor, counts, at)]


def _plain_prefer(s):
    z, starts, P = s["z"].detach(), s["starts"], s["case"]["P"]
    top, e, total = _row_sums(z)
    logp, counts, at = _label_logp(z, s["label"], top, total)
    upto = torch.cat((logp.new_zeros(1), logp.cumsum(0)))[starts]
    ratio = upto[1:] - upto[:-1] - s["ref"].double()
    margin = BETA * (ratio[:P] - ratio[P:])
    right, wrong = torch.log1p(torch.exp(-margin.abs())) + (-margin).clamp(min=0), torch.log1p(torch.exp(-margin.abs())) + margin.clamp(min=0)
    loss = ((1 - SMOOTHING) * right + SMOOTHING * wrong).mean()
    per_pair = BETA / P * (1 / (1 + torch.exp(-margin)) - (1 - SMOOTHING))
    row = torch.arange(len(at), device=at.device)
    text = torch.searchsorted(starts, row, right=True) - 1
    inside = text < 2 * P
    factor = torch.where(inside, torch.cat((per_pair, -per_pair))[text.clamp(max=2 * P - 1)], 0.0)
    return [loss.float(), margin.float(), _logits_gradient(e, total, factor, counts, at)]


_PLAIN = dict(embed=_plain_embed, logp=_plain_logp, policy=_plain_policy, prefer=_plain_prefer)


# ------------------------------------------------------------------------------------------------- the framework's calls
def _own_embed(s):
    from snntc_2023_b200 import ops
    c = s["case"]
    y = ops.snn_embedding(s["ids"], s["table"], scale=c["scale"], spikes=c["spikes"])
    if c["mode"] == "lookup":
        return [y]
    return [y, *torch.autograd.grad(y, s["table"], s["g"])]


def _own_logp(s):
    from snntc_2023_b200 import train
    logp = train.label_log_probs(s["z"], s["label"])
    if s["case"]["mode"] == "score":
        return [logp]
    return [logp, *torch.autograd.grad(logp, s["z"], s["g"])]


def _own_policy(s):
    from snntc_2023_b200 import train
    loss, stats = train.policy_loss(s["z"], s["label"], s["old"], s["advantage"], ref_logp=s["ref"], clip_low=CLIP_LOW,
                                    clip_high=CLIP_HIGH, kl_coef=KL_COEF, with_stats=True)
    return [loss, stats, *torch.autograd.grad(loss, s["z"])]


def _own_prefer(s):
    from snntc_2023_b200 import train
    loss, margins = train.preference_loss(s["z"], s["label"], s["starts"], ref_logp=s["ref"], beta=BETA,
                                          label_smoothing=SMOOTHING, with_margins=True)
    return [loss, margins, *torch.autograd.grad(loss, s["z"])]


_OWN = dict(embed=_own_embed, logp=_own_logp, policy=_own_policy, prefer=_own_prefer)


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------- bytes and flops
def _distinct(N, V):
    """Expected number of different ids among N of them."""
    v = torch.arange(V, dtype=torch.float64)
    p = ((v + 2).log() - (v + 1).log()) / math.log(V + 1)
    return float((1 - (1 - p) ** N).sum())


def work(case):
    c = case
    if c["op"] == "embed":
        N, V, D = c["N"], c["V"], c["D"]
        tokens = N - N // 8 if c["pad"] else N
        nbytes = 8 * N + 4 * D * (_distinct(tokens, V) + N)
        flops = N * D * (2 if c["spikes"] else 1)
        if c["mode"] == "train":
            nbytes += 4 * D * (tokens + V)
            flops += D * (tokens + 2 * V)
        return dict(bytes=nbytes, flops=flops)
    R, J = c["R"], c["J"]
    per_row = {"logp": 8 + 4 + 4, "policy": 8 + 12, "prefer": 8}[c["op"]]
    grad = c["op"] != "logp" or c["mode"] == "grad"
    return dict(bytes=4 * R * J * (2 if grad else 1) + per_row * R + (32 * c["P"] if c["op"] == "prefer" else 0),
                flops=R * J * (7 if grad else 4))


# ------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definitions in 64 bits, gradients by differentiating them."""
    s = prepare(case, seed)
    c = case
    if c["op"] == "embed":
        table = s["table"].detach().double()
        known = s["ids"] >= 0
        values = table * c["scale"]
        slope = torch.full_like(table, c["scale"])
        if c["spikes"]:
            values = torch.exp(values)
            slope = c["scale"] * values
        y = torch.full((c["N"], c["D"]), NO_SPIKE, dtype=torch.float64, device="cuda")
        y[known] = values[s["ids"][known]]
        if c["mode"] == "lookup":
            return [y]
        sums = torch.zeros_like(table).index_put_((s["ids"][known],), s["g"][known].double(), accumulate=True)
        return [y, sums * slope]
    z = s["z"].detach().double().requires_grad_(c["op"] != "logp" or c["mode"] == "grad")
    known = s["label"] >= 0
    logp = torch.where(known, torch.log_softmax(-z, 1).gather(1, s["label"].clamp(min=0)[:, None])[:, 0], 0.0)
    if c["op"] == "logp":
        if c["mode"] == "score":
            return [logp]
        return [logp.detach(), *torch.autograd.grad(logp, z, s["g"].double())]
    if c["op"] == "policy":
        old, ref, adv = (s[k].double()[known] for k in ("old", "ref", "advantage"))
        lp = logp[known]
        n = max(1, len(lp))
        ratio = torch.exp(lp - old)
        held = ratio.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH)
        kl = torch.exp(ref - lp) - (ref - lp) - 1
        loss = (KL_COEF * kl - torch.minimum(ratio * adv, held * adv)).sum() / n
        stats = torch.stack((kl.sum() / n, (held * adv < ratio * adv).sum() / n))
        return [loss.detach(), stats.detach(), *torch.autograd.grad(loss, z)]
    P = c["P"]
    bounds = s["starts"].tolist()
    texts = torch.stack([logp[a:b].sum() for a, b in zip(bounds[:-1], bounds[1:])])
    ratio = texts - s["ref"].double()
    margin = BETA * (ratio[:P] - ratio[P:])
    up, down = torch.nn.functional.logsigmoid(margin), torch.nn.functional.logsigmoid(-margin)
    loss = -((1 - SMOOTHING) * up + SMOOTHING * down).mean()
    return [loss.detach(), margin.detach(), *torch.autograd.grad(loss, z)]
