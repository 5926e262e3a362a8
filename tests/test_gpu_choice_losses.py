"""GPU tests of the losses on choices -- label log-probabilities, clipped policy loss, preference loss -- against float64
evaluations of their formulas.

Tolerances, with u = 2^-24 (half a step of float32), d_j = -z_j - max(-z): a term exp(d_j) of a row's sum is off by the rounding of
d_j, of log2(e) and of their product, 2.5 |d_j| u, and by the exponential's own 2^-22 = 4 u at most; the sum of a row by its longest chain of
additions, 64 u for the row lengths here (a lane adds eight terms at a time, a long row's lanes some forty times, and the tree over
lanes and warps has 10 levels), which weights the terms' errors by p_j. So total is off by REL = (4 + 64 + 2.5 sum_j p_j |d_j|) u relative, lp by REL + |lp| u (its own rounding),
p_j by REL + (2.5 |d_j| + 4 + 3) u relative, and a gradient factor * (p - onehot) by |factor| (p_j * that + 2 u) where factor is exact."""
import math

import pytest

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _logits(R, J, seed, ignore=0.1):
    """Spike values, three in ten without a spike, the first row without any; labels among the likelier half."""
    import torch
    g = torch.Generator("cuda").manual_seed(seed)
    z = torch.rand(R, J, device="cuda", generator=g) * 6 + 1
    z[torch.rand(R, J, device="cuda", generator=g) < 0.3] = 1e5
    z[0] = 1e5
    lab = (z + torch.rand(R, J, device="cuda", generator=g)).argmin(1)
    lab[torch.rand(R, device="cuda", generator=g) < ignore] = -1
    return z, lab


class Ref:
    """Softmax of the rows in float64 and the bounds of the module's docstring."""

    def __init__(self, z, lab):
        import torch
        R, J = z.shape
        self.counts = (lab >= 0) & (lab < J)
        at = lab.clamp(0, J - 1)
        x = -z.double()
        x = torch.where(self.counts[:, None], x, torch.zeros_like(x))
        self.lp = torch.where(self.counts, torch.log_softmax(x, 1).gather(1, at[:, None])[:, 0], 0.0)
        self.p = torch.softmax(x, 1)
        d = (x.amax(1, keepdim=True) - x).clamp(max=200.0)          # (beyond that p is 0 on both sides)
        self.rel = (68 + 2.5 * (self.p * d).sum(1)) * U
        self.p_rel = self.rel[:, None] + (2.5 * d + 7) * U
        self.hot = torch.zeros_like(self.p)
        self.hot[torch.arange(R, device=z.device), at] = 1.0

    def check_lp(self, lp):
        assert ((lp.double() - self.lp).abs() <= self.counts * (self.rel + self.lp.abs() * U) * 1.001).all()

    def check_grad(self, grad, factor, factor_tol, times=1):
        """factor: float64 per row; factor_tol: how far the kernel's may be off; times: grad is a sum with so many gradients' errors"""
        import torch
        factor, factor_tol = torch.where(self.counts, factor, 0.0)[:, None], torch.where(self.counts, factor_tol, 0.0)[:, None]
        want = factor * (self.p - self.hot)
        tol = factor.abs() * (self.p * self.p_rel + 2 * U * (self.p + self.hot)) + factor_tol * (self.p + self.hot) * 1.01 + 1e-38
        err = (grad.double() - want).abs()
        assert (err <= times * tol * 1.001).all(), float((err / tol).max())
        assert (grad[~self.counts] == 0).all()


SHAPES = [(1, 1), (1, 2), (3, 1), (2, 3), (37, 10), (257, 10), (5, 13), (6, 14), (7, 29), (4, 31), (5, 61), (65, 64), (9, 125), (3, 128), (8, 253),
          (33, 257), (3, 509), (4, 1000), (130, 1000), (3, 1021), (2, 1024), (3, 2049), (5, 4093), (2, 8191), (3, 8192), (1, 8193), (2, 16381),
          (2, 16385), (3, 32768), (2, 50021), (1, 65536), (2, 131070), (1, 131073), (1, 262147), (5000, 17), (40000, 2)]


@pytest.mark.parametrize("R,J", SHAPES)
def test_label_log_probs_and_their_gradient(R, J):
    import torch
    from snntc_2023_b200 import train
    z, lab = _logits(R, J, R * 7 + J)
    ref = Ref(z, lab)
    z1 = z.clone().requires_grad_(True)
    lp = train.label_log_probs(z1, lab)
    assert lp.shape == (R,) and lp.dtype == torch.float32
    ref.check_lp(lp.detach())
    up = torch.randn(R, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    lp.backward(up)
    ref.check_grad(z1.grad, up.double(), torch.zeros(R, dtype=torch.float64, device="cuda"))
    with torch.no_grad():
        assert torch.equal(train.label_log_probs(z1, lab), lp)
    assert torch.equal(train.label_log_probs(z, lab.int()), lp.detach())


def _policy_ref(ref, old, adv, refp, lo, hi, kl_coef):
    """loss, stats and factors in float64; and how far an error of lp, ref.rel + u |lp| at most (the kernel keeps lp in 64 bits), moves
    them. Rows whose ratio is nearer to the border than that are reported."""
    import torch
    n = max(1, int(ref.counts.sum()))
    dlp = ref.rel
    ratio = torch.exp(ref.lp - old.double())
    a = adv.double()
    near = torch.minimum((ratio - (1 + hi)).abs(), (ratio - (1 - lo)).abs()) <= ratio * dlp * 1.01 + 1e-12
    clipped = ((a > 0) & (ratio > 1 + hi)) | ((a < 0) & (ratio < 1 - lo))
    gain = torch.where(clipped, ratio.clamp(1 - lo, 1 + hi), ratio) * a
    slope = torch.where(clipped, 0.0, -ratio * a)
    slack = torch.where(clipped, 0.0, (ratio * a).abs() * dlp)
    loss, kl = -gain, torch.zeros_like(a)
    loss_slack, kl_slack = slack.clone(), torch.zeros_like(a)
    if refp is not None:
        away = refp.double() - ref.lp
        kl = torch.expm1(away) - away
        loss = loss + kl_coef * kl
        slope = slope - kl_coef * torch.expm1(away)
        slack = slack + abs(kl_coef) * torch.exp(away) * dlp
        kl_slack = torch.expm1(away).abs() * dlp + torch.exp(away) * dlp ** 2
        loss_slack = loss_slack + abs(kl_coef) * kl_slack
    c = ref.counts
    mean = lambda v: float(torch.where(c, v.double(), 0.0).sum()) / n  # noqa: E731
    tiny = 1e-9        # the 64-bit arithmetic of a row, relative to its terms
    sizes = gain.abs() + kl.abs() * abs(kl_coef)
    return dict(loss=mean(loss), loss_tol=mean(loss_slack) * 1.01 + tiny * mean(sizes), kl=mean(kl), kl_tol=mean(kl_slack) * 1.01 + tiny * mean(kl.abs()),
                clipped=mean(clipped), factor=slope / n, factor_tol=(slack * 1.01 + slope.abs() * (U + tiny)) / n, near=bool((near & c).any()))


@pytest.mark.parametrize("R,J", SHAPES)
@pytest.mark.parametrize("with_ref", [True, False])
def test_policy_loss_and_its_gradient(R, J, with_ref):
    import torch
    from snntc_2023_b200 import train
    z, lab = _logits(R, J, R + 3 * J)
    ref = Ref(z, lab)
    g = torch.Generator("cuda").manual_seed(4)
    noise = lambda s: s * torch.randn(R, device="cuda", generator=g)  # noqa: E731
    old, refp, adv = (ref.lp + noise(0.3)).float(), (ref.lp + noise(0.5)).float(), noise(1.0)
    for t in (old, refp, adv):
        t[~ref.counts] = float("nan")                 # what stands beside a row that does not count is not read
    refp = refp if with_ref else None
    kl_coef = 0.3 if with_ref else 0.0
    want = _policy_ref(ref, old, adv, refp, 0.2, 0.25, kl_coef)
    assert not want["near"], "a ratio lies on the border of the clip: another seed"
    z1 = z.clone().requires_grad_(True)
    loss, stats = train.policy_loss(z1, lab, old, adv, ref_logp=refp, clip_low=0.2, clip_high=0.25, kl_coef=kl_coef, with_stats=True)
    assert loss.dim() == 0 and stats.shape == (2,) and not stats.requires_grad
    close = lambda got, w, tol: abs(float(got) - w) <= tol + abs(w) * U + 1e-30  # noqa: E731
    assert close(loss, want["loss"], want["loss_tol"]) and close(stats[0], want["kl"], want["kl_tol"]) and close(stats[1], want["clipped"], 1e-12)
    loss.backward()
    ref.check_grad(z1.grad, want["factor"], want["factor_tol"])
    first = z1.grad.clone()
    # an upstream factor other than one, twice over the same graph (the second time on top of the first)
    z1.grad = None
    again = train.policy_loss(z1, lab, old, adv, ref_logp=refp, clip_low=0.2, clip_high=0.25, kl_coef=kl_coef)
    assert torch.equal(again, loss)
    (again * -2.0).backward(retain_graph=True)
    assert torch.equal(z1.grad, -2.0 * first)         # (a power of two moves no rounding)
    again.backward()
    ref.check_grad(-z1.grad, want["factor"], want["factor_tol"], times=4)      # -2 of the first, one of its own; the last is the sum's rounding
    with torch.no_grad():
        alone = train.policy_loss(z1, lab, old, adv, ref_logp=refp, clip_low=0.2, clip_high=0.25, kl_coef=kl_coef, with_stats=True)
    assert torch.equal(alone[0], loss) and torch.equal(alone[1], stats)


def _texts(R, P, seed, tail):
    """2P+1 ascending offsets, an empty text among them where there are several, `tail` rows behind the last."""
    import random

    import torch
    rng = random.Random(seed)
    cuts = sorted(rng.randrange(R - tail + 1) for _ in range(2 * P - 1))
    if P > 1:
        cuts[1] = cuts[0]
    return torch.tensor([0] + cuts + [R - tail], device="cuda")


def _preference_ref(ref, starts, refp, beta, eps):
    import torch
    b = starts.tolist()
    P = (len(b) - 1) // 2
    text = lambda v: torch.stack([v[x:y].sum() for x, y in zip(b[:-1], b[1:])])  # noqa: E731
    s = text(ref.lp)
    slack = text(torch.where(ref.counts, ref.rel, 0.0))
    if refp is not None:
        s = s - refp.double()
    m = beta * (s[:P] - s[P:])
    dm = abs(beta) * (slack[:P] + slack[P:]) * 1.01 + 1e-12 * (1 + s[:P].abs() + s[P:].abs())
    sig = torch.sigmoid(m)
    loss = -((1 - eps) * torch.nn.functional.logsigmoid(m) + eps * torch.nn.functional.logsigmoid(-m))
    per = beta / P * (sig - (1 - eps))
    per_tol = abs(beta) / P * dm / 4 + per.abs() * U * 1.01 + abs(beta) / P * 1e-15
    factor, tol = torch.zeros_like(ref.lp), torch.zeros_like(ref.lp)
    for k in range(P):
        for t, sign in ((k, 1.0), (P + k, -1.0)):
            factor[b[t]:b[t + 1]], tol[b[t]:b[t + 1]] = sign * per[k], per_tol[k]
    return dict(loss=float(loss.mean()), loss_tol=float(dm.mean()), m=m, dm=dm, factor=factor, factor_tol=tol)


@pytest.mark.parametrize("R,J,P,tail", [(2, 3, 1, 0), (7, 10, 1, 2), (37, 10, 5, 3), (64, 1000, 8, 0), (517, 333, 8, 20), (40, 8192, 3, 1), (24, 16390, 2, 4),
                                        (12, 50021, 2, 1), (6, 131073, 1, 1), (3000, 5, 700, 100), (20000, 7, 1, 0), (10, 4, 30, 0)])
@pytest.mark.parametrize("with_ref", [True, False])
def test_preference_loss_and_its_gradient(R, J, P, tail, with_ref):
    import torch
    from snntc_2023_b200 import train
    z, lab = _logits(R, J, R + J + P, ignore=0.2)
    z[R - tail:] = float("nan")                       # rows behind the last text: no part in anything
    lab[R - tail:] = -1
    starts = _texts(R, P, R + P, tail)
    ref = Ref(z, lab)
    g = torch.Generator("cuda").manual_seed(6)
    b = starts.tolist()
    sums = torch.stack([ref.lp[x:y].sum() for x, y in zip(b[:-1], b[1:])])
    refp = (sums + 4 * torch.randn(2 * P, device="cuda", generator=g)).float() if with_ref else None
    beta, eps = (0.3, 0.1) if with_ref else (0.01, 0.0)
    want = _preference_ref(ref, starts, refp, beta, eps)
    z1 = z.clone().requires_grad_(True)
    loss, m = train.preference_loss(z1, lab, starts, ref_logp=refp, beta=beta, label_smoothing=eps, with_margins=True)
    assert m.shape == (P,) and not m.requires_grad
    assert ((m.double() - want["m"]).abs() <= want["dm"] + want["m"].abs() * U).all()
    assert abs(float(loss) - want["loss"]) <= want["loss_tol"] + abs(want["loss"]) * U
    loss.backward()
    ref.check_grad(z1.grad, want["factor"], want["factor_tol"])
    first = z1.grad.clone()
    z1.grad = None
    again = train.preference_loss(z1, lab, starts.int(), ref_logp=refp, beta=beta, label_smoothing=eps)
    (again * 4.0).backward()
    assert torch.equal(again, loss) and torch.equal(z1.grad, 4.0 * first)
    with torch.no_grad():
        assert torch.equal(train.preference_loss(z1, lab, starts, ref_logp=refp, beta=beta, label_smoothing=eps), loss)


def test_rows_of_a_text_that_a_label_leaves_out_but_no_text_owns():
    """Rows behind the last text whose labels are classes: no gradient, whatever their logits."""
    import torch
    from snntc_2023_b200 import train
    z, lab = _logits(20, 9, 2, ignore=0.0)
    starts = torch.tensor([0, 6, 14], device="cuda")
    z1 = z.clone().requires_grad_(True)
    loss = train.preference_loss(z1, lab, starts, beta=0.01)
    loss.backward()
    assert (z1.grad[14:] == 0).all() and z1.grad[:14].abs().sum(1).gt(0).all()
    short = train.preference_loss(z[:14], lab[:14], starts, beta=0.01)
    assert torch.equal(short, loss.detach())


def test_padded_texts_are_the_packed_ones():
    import torch
    from snntc_2023_b200 import train
    z, lab = _logits(6 * 11, 50, 9, ignore=0.3)
    zp, labp = z.view(6, 11, 50).clone().requires_grad_(True), lab.view(6, 11)
    refp = torch.randn(6, device="cuda")
    loss, m = train.preference_loss(zp, labp, ref_logp=refp, beta=0.2, with_margins=True)
    loss.backward()
    zq = z.clone().requires_grad_(True)
    packed, mq = train.preference_loss(zq, lab, torch.arange(0, 67, 11, device="cuda"), ref_logp=refp, beta=0.2, with_margins=True)
    packed.backward()
    assert torch.equal(loss, packed) and torch.equal(m, mq) and torch.equal(zp.grad.view(66, 50), zq.grad)
    lp = train.label_log_probs(zp, labp)
    assert lp.shape == (6, 11) and torch.equal(lp.view(-1), train.label_log_probs(zq, lab))


def test_offsets_that_are_no_offsets_stay_inside():
    """Offsets that descend or leave the rows are held to them: numbers without meaning, but no access outside."""
    import torch
    from snntc_2023_b200 import train
    z, lab = _logits(30, 12, 3)
    for bad in ([5, 2, 28], [-7, 12, 10 ** 12], [0, 50, 40, 31, 60], [2 ** 62, -2 ** 62, 3]):
        z1 = z.clone().requires_grad_(True)
        loss = train.preference_loss(z1, lab, torch.tensor(bad, device="cuda"), beta=0.01)
        loss.backward()
        assert math.isfinite(float(loss.detach())) and z1.grad.isfinite().all()


def test_no_row_counts():
    import torch
    from snntc_2023_b200 import train
    for R, J in ((1, 5), (70, 10), (9, 2000), (3, 40000)):
        z = torch.full((R, J), float("nan"), device="cuda", requires_grad=True)
        lab = torch.full((R,), -1, device="cuda")
        lab[0] = J
        nan = torch.full((R,), float("nan"), device="cuda")
        loss, stats = train.policy_loss(z, lab, nan, nan, ref_logp=nan, kl_coef=1.0, with_stats=True)
        loss.backward()
        assert float(loss) == 0 and (stats == 0).all() and (z.grad == 0).all()
        z.grad = None
        lp = train.label_log_probs(z, lab)
        lp.sum().backward()
        assert (lp == 0).all() and (z.grad == 0).all()
        z.grad = None
        loss = train.preference_loss(z, lab, torch.tensor([0, R, R], device="cuda"))
        loss.backward()
        assert abs(float(loss) - math.log(2)) < 1e-6 and (z.grad == 0).all()


def test_infinite_and_nan_outputs():
    """Outputs at +inf have no part in a softmax; a row with a NaN is NaN and touches no other row."""
    import torch
    from snntc_2023_b200 import train
    for J in (7, 100, 700, 5000, 20000):
        z, lab = _logits(6, J, J, ignore=0.0)
        z[1:, 0] = float("inf")
        lab[lab == 0] = 1
        z[3, 2] = float("nan")
        z1 = z.clone().requires_grad_(True)
        lp = train.label_log_probs(z1, lab)
        lp.sum().backward()
        keep = [0, 1, 2, 4, 5]
        zf = z[keep].clone()
        zf[zf == float("inf")] = 1e30
        ref = Ref(zf, lab[keep])
        ref.check_lp(lp.detach()[keep])
        ref.check_grad(z1.grad[keep], torch.ones(5, dtype=torch.float64, device="cuda"), torch.zeros(5, dtype=torch.float64, device="cuda"))
        assert lp[3].isnan() and z1.grad[3, 1].isnan()


@pytest.mark.parametrize("J", [9, 120, 900, 3500, 30000])
def test_outputs_masked_by_the_largest_value(J):
    """Classes switched off by the largest float: no part in a softmax, the row that has nothing else is uniform; and the lowest value,
    beside which everything else is nothing."""
    import torch
    from snntc_2023_b200 import train
    most = torch.finfo(torch.float32).max
    z, lab = _logits(5, J, J + 1, ignore=0.0)
    z[1:, J // 2:] = most
    lab[1:] = 0
    z[3] = most
    z[4, 0] = -most
    z1 = z.clone().requires_grad_(True)
    lp = train.label_log_probs(z1, lab)
    lp.sum().backward()
    assert abs(float(lp[3].detach()) + math.log(J)) < 1e-5 * math.log(J) and float(lp[4].detach()) == 0.0
    assert not z1.grad[1:3, J // 2:].any() and not z1.grad[4].any()
    keep = [0, 1, 2]
    ref = Ref(z[keep].clamp(max=1e30), lab[keep])
    ref.check_lp(lp.detach()[keep])
    ref.check_grad(z1.grad[keep], torch.ones(3, dtype=torch.float64, device="cuda"), torch.zeros(3, dtype=torch.float64, device="cuda"))
    old = lp.detach() - 0.01
    loss = train.policy_loss(z1, lab, old, torch.ones(5, device="cuda"), ref_logp=old, kl_coef=0.1)
    (grad,) = torch.autograd.grad(loss, z1)
    assert loss.isfinite() and grad.isfinite().all()


def test_gradients_against_differences():
    """Central differences of the losses in float64 (their formulas' own, at the kernels' inputs) along random directions: with steps of
    1e-6 they are good to 1e-7 of the slope's size."""
    import torch
    from snntc_2023_b200 import train
    g = torch.Generator("cuda").manual_seed(0)
    R, J = 24, 40
    z = torch.rand(R, J, device="cuda", generator=g) * 4 + 1
    lab = torch.randint(0, J, (R,), device="cuda", generator=g)
    lab[5] = -1
    c = lab >= 0
    lp_of = lambda y: torch.where(c, torch.log_softmax(-y, 1).gather(1, lab.clamp(min=0)[:, None])[:, 0], 0.0)  # noqa: E731
    lp0 = lp_of(z.double())
    old, refp, adv = (lp0 + 0.3 * torch.randn(R, device="cuda", generator=g)).float(), (lp0 - 0.2).float(), torch.randn(R, device="cuda", generator=g)
    starts = torch.tensor([0, 6, 9, 9, 22], device="cuda")

    def policy(y):
        lp = lp_of(y)[c]
        r, a, w = torch.exp(lp - old.double()[c]), adv.double()[c], refp.double()[c] - lp
        return (0.4 * (torch.exp(w) - w - 1) - torch.minimum(r * a, r.clamp(0.8, 1.2) * a)).mean()

    def preference(y):
        s = torch.stack([lp_of(y)[i:j].sum() for i, j in ((0, 6), (6, 9), (9, 9), (9, 22))])
        m = 0.2 * (s[:2] - s[2:])
        return -(0.9 * torch.nn.functional.logsigmoid(m) + 0.1 * torch.nn.functional.logsigmoid(-m)).mean()

    calls = ((policy, lambda y: train.policy_loss(y, lab, old, adv, ref_logp=refp, kl_coef=0.4)),
             (preference, lambda y: train.preference_loss(y, lab, starts, beta=0.2, label_smoothing=0.1)),
             (lambda y: lp_of(y).sum(), lambda y: train.label_log_probs(y, lab).sum()))
    for plain, call in calls:
        z1 = z.clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(call(z1), z1)
        for _ in range(8):
            v = torch.randn(R, J, device="cuda", dtype=torch.float64, generator=g)
            slope = float((plain(z.double() + 1e-6 * v) - plain(z.double() - 1e-6 * v)) / 2e-6)
            size = float((grad.double() * v).abs().sum())
            assert abs(float((grad.double() * v).sum()) - slope) <= 2e-6 * size      # 1e-7 of the difference, the rest float32's p and factors


def test_strides_offsets_and_leading_dimensions():
    import torch
    from snntc_2023_b200 import train
    z, lab = _logits(60, 33, 11)
    wide = torch.rand(60, 80, device="cuda")
    wide[:, 7:40] = z
    base = wide.clone().requires_grad_(True)
    lp = train.label_log_probs(base[:, 7:40], lab)
    lp.sum().backward()
    z1 = z.clone().requires_grad_(True)
    plain = train.label_log_probs(z1, lab)
    plain.sum().backward()
    assert torch.equal(lp, plain) and torch.equal(base.grad[:, 7:40], z1.grad) and not base.grad[:, :7].any() and not base.grad[:, 40:].any()
    for off in (1, 2, 3):                             # contiguous rows that start off 16 bytes
        for J in (33, 1028, 9000):
            zz, ll = _logits(7, J, off + J)
            buf = torch.empty(off + zz.numel(), device="cuda")
            moved = buf[off:].view(7, J).copy_(zz).detach().requires_grad_(True)
            zz.requires_grad_(True)
            adv = torch.randn(7, device="cuda")
            old = train.label_log_probs(zz, ll).detach() - 0.1
            a, b = (train.policy_loss(t, ll, old, adv) for t in (moved, zz))
            a.backward()
            b.backward()
            assert torch.allclose(a, b, rtol=1e-5) and torch.allclose(moved.grad, zz.grad, rtol=1e-5, atol=1e-9)
    zl, ll = z.view(3, 4, 5, 33), lab.view(3, 4, 5)
    moved = train.label_log_probs(zl.transpose(0, 1), ll.transpose(0, 1))     # (a row's bits may go with where it starts to 16 bytes)
    Ref(z, lab).check_lp(moved.transpose(0, 1).reshape(60))


def test_more_than_32_bits_of_logits():
    import torch
    from snntc_2023_b200 import train
    R, J = 66000, 32800                               # 2.16e9 logits
    z = torch.full((R, J), 4.0, device="cuda")
    z[:, 5] = 1.0
    z[-1, J - 1] = 0.5
    lab = torch.full((R,), -1, device="cuda")
    lab[0], lab[R // 2], lab[R - 1] = 5, 5, J - 1
    z.requires_grad_(True)
    lp = train.label_log_probs(z, lab)
    rows = torch.tensor([0, R // 2, R - 1], device="cuda")
    ref = Ref(z.detach()[rows], lab[rows])
    ref.check_lp(lp.detach()[rows])
    old = lp.detach() - 0.05
    del lp
    loss = train.policy_loss(z, lab, old, torch.ones(R, device="cuda"))
    (grad,) = torch.autograd.grad(loss, z)
    f = -torch.exp(ref.lp - old[rows].double()) / 3
    ref.check_grad(grad[rows], f, f.abs() * (ref.rel * 1.1 + 2 * U))
    grad[rows] = 0
    assert not grad.any()


def test_refusals():
    import torch
    from snntc_2023_b200 import _lib, train
    z, lab = _logits(8, 5, 1)
    v = torch.zeros(8, device="cuda")
    for bad in (z.double(), z.half(), z[0], z[:0], z[:, :0], z.view(2, 4, 5)):
        with pytest.raises(ValueError):
            train.label_log_probs(bad, lab[:bad.shape[0]] if bad.dim() == 2 and bad.shape[0] == 0 else lab)
    for bad in (lab.float(), lab.bool(), lab[:7], lab.view(2, 4)):
        with pytest.raises(ValueError):
            train.label_log_probs(z, bad)
    with pytest.raises(ValueError):
        train.policy_loss(z, lab, v[:7], v)
    with pytest.raises(ValueError):
        train.policy_loss(z, lab, v, v.double())
    for bad in (v.view(4, 2), v[:1], v[0]):                               # as many values in another shape, or to be broadcast
        with pytest.raises(ValueError):
            train.policy_loss(z, lab, v, bad)
    with pytest.raises(ValueError):
        train.policy_loss(z.view(2, 4, 5), lab.view(2, 4), v.view(4, 2), v.view(2, 4))
    with pytest.raises(_lib.SnntcError):
        train.policy_loss(z, lab, v.cpu(), v)
    with pytest.raises(ValueError, match="detach"):
        train.policy_loss(z, lab, v, v.clone().requires_grad_(True))
    with pytest.raises(ValueError, match="ref_logp"):
        train.policy_loss(z, lab, v, v, kl_coef=0.1)
    for kw in (dict(clip_low=-0.1), dict(clip_low=1.5), dict(clip_high=-1.0), dict(clip_high=float("nan")), dict(kl_coef=float("inf"), ref_logp=v)):
        with pytest.raises(ValueError):
            train.policy_loss(z, lab, v, v, **kw)
    starts = torch.tensor([0, 4, 8], device="cuda")
    for bad in (None, starts[:2], starts[:1], starts.float(), starts.view(1, 3), starts.cpu()):
        with pytest.raises(ValueError):
            train.preference_loss(z, lab, bad)
    for kw in (dict(beta=float("nan")), dict(label_smoothing=-0.1), dict(label_smoothing=2.0), dict(ref_logp=v)):
        with pytest.raises(ValueError):
            train.preference_loss(z, lab, starts, **kw)
    with pytest.raises(ValueError):
        train.preference_loss(z.view(1, 8, 5), lab.view(1, 8))            # an odd number of padded texts
    z1 = z.clone().requires_grad_(True)
    for loss in (train.label_log_probs(z1, lab).sum(), train.policy_loss(z1, lab, v, v), train.preference_loss(z1, lab, starts)):
        with pytest.raises(RuntimeError, match="create_graph"):
            torch.autograd.grad(loss, z1, create_graph=True)
    loss = train.policy_loss(z1, lab, v, v)
    with torch.no_grad():
        z1 += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_a_loss_used_twice_and_beside_others():
    """One node, one backward: the factors of a loss that enters an objective twice add up before its kernel runs; beside another loss of
    the same logits the gradients are added."""
    import torch
    from snntc_2023_b200 import train
    z, lab = _logits(40, 30, 8)
    adv = torch.randn(40, device="cuda")
    old = train.label_log_probs(z, lab) - 0.1
    z1 = z.clone().requires_grad_(True)
    loss = train.policy_loss(z1, lab, old, adv)
    other = train.loss_func(z1, lab.clamp(min=0))
    (alone,) = torch.autograd.grad(loss, z1, retain_graph=True)           # hands the kept gradient out
    mine = alone.clone()
    (ce,) = torch.autograd.grad(other, z1, retain_graph=True)
    alone.zero_()                                                         # (the caller's: nothing of it is read again)
    (both,) = torch.autograd.grad(loss * 3.0 + loss + other, z1)
    assert torch.allclose(both, 4.0 * mine + ce, rtol=1e-5, atol=1e-9)


def test_two_threads_at_once():
    """Both directions of every loss from two host threads on streams of their own: the results of calls one after the other."""
    import threading

    import torch
    cases = []
    for k, (R, J) in enumerate(((300, 40), (64, 9000))):
        z, lab = _logits(R, J, 70 + k)
        cases.append((z, lab, -2 - torch.rand(R, device="cuda"), torch.randn(R, device="cuda"), -2 - torch.rand(R, device="cuda"),
                      torch.tensor([0, R // 4, R // 2, R // 2, R], device="cuda")))
    plain = [_all_losses(c[0].clone().requires_grad_(True), *c[1:]) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = _all_losses(cases[k][0].clone().requires_grad_(True), *cases[k][1:])
                torch.cuda.current_stream().synchronize()
                bad.extend(1 for a, b in zip(got, plain[k]) if not torch.equal(a, b))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def _all_losses(z, lab, old, adv, refp, starts):
    import torch
    from snntc_2023_b200 import train
    out = []
    for loss in (train.policy_loss(z, lab, old, adv, ref_logp=refp, kl_coef=0.1), train.preference_loss(z, lab, starts, beta=0.05),
                 (train.label_log_probs(z, lab) * adv).sum()):
        out += [loss.detach(), torch.autograd.grad(loss, z)[0]]
    return out


@pytest.mark.parametrize("R,J", [(64, 10), (300, 500), (40, 20011)])
def test_captured_replayed_and_on_other_streams(R, J):
    """Forward and gradient captured once and replayed on other inputs; two captured graphs and plain calls on two streams at once."""
    import torch
    sets = []
    for k in range(2):
        z, lab = _logits(R, J, 50 + k)
        sets.append((z, lab, -2 - torch.rand(R, device="cuda"), torch.randn(R, device="cuda"), -2 - torch.rand(R, device="cuda"),
                     torch.tensor([0, R // 4 + k, R // 2, R // 2, R - k], device="cuda")))
    plain = [_all_losses(s[0].clone().requires_grad_(True), *s[1:]) for s in sets]
    graphs = []
    for k in range(2):
        own = [t.clone() for t in sets[k]]
        own[0].requires_grad_(True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _all_losses(*own)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _all_losses(*own)
        graphs.append((graph, own, out))
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))  # noqa: E731
    graph, own, out = graphs[0]
    for k in (1, 0):
        with torch.no_grad():
            for dst, src in zip(own, sets[k]):
                dst.copy_(src)
        graph.replay()
        assert same(out, plain[k])
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                graphs[k][0].replay()
            with torch.cuda.stream(streams[2 + k]):
                got[k].append(_all_losses(sets[k][0].clone().requires_grad_(True), *sets[k][1:]))
    torch.cuda.synchronize()
    assert all(same(g, plain[k]) for k in range(2) for g in got[k])
    assert same(graphs[0][2], plain[0]) and same(graphs[1][2], plain[1])


def test_a_capture_beside_a_live_eager_graph_is_refused():
    import torch
    from snntc_2023_b200 import train
    z, lab = _logits(16, 9, 1)
    z.requires_grad_(True)
    alive = train.label_log_probs(z, lab)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            train.label_log_probs(z, lab).sum().backward()
    torch.cuda.synchronize()
    alive.sum().backward()
    assert z.grad.isfinite().all()


def _beside_a_silent_label(R, J, seed):
    """Every row counts, ratios lie at exp(+-0.1), inside the clip. In row R // 2 the label's output does not spike while others do: its
    log-probability is near -1e5, the reference's is -3."""
    import torch
    z, lab = _logits(R, J, seed, ignore=0.0)
    at = R // 2
    z[at] = 2.0
    z[at, lab[at]] = 1e5
    g = torch.Generator("cuda").manual_seed(seed)
    lp = Ref(z, lab).lp
    old = (lp + 0.1 * torch.randn(R, device="cuda", generator=g).sign()).float()
    adv, refp = torch.randn(R, device="cuda", generator=g), (lp + 0.1).float()
    old[at] = lp[at].float()
    refp[at] = -3.0
    return z, lab, old, adv, refp, at


SILENT = [(6, 10), (400, 60), (90, 1000), (40, 1500), (6, 5000), (4, 40000)]


@pytest.mark.parametrize("R,J", SILENT)
def test_a_reference_without_weight_has_no_part_in_the_loss(R, J):
    """A KL coefficient of 0 beside a reference, for the statistics: the call without it, also where the KL term overflows."""
    import torch
    from snntc_2023_b200 import train
    z, lab, old, adv, refp, at = _beside_a_silent_label(R, J, R + J)
    results = []
    for r in (refp, None):
        z1 = z.clone().requires_grad_(True)
        loss, stats = train.policy_loss(z1, lab, old, adv, ref_logp=r, with_stats=True)
        (grad,) = torch.autograd.grad(loss, z1)
        results.append((loss.detach(), grad, stats))
    (loss, grad, stats), (plain, want, _) = results
    assert loss.isfinite() and grad.isfinite().all() and torch.equal(loss, plain) and torch.equal(grad, want)
    assert float(stats[0]) == math.inf and torch.equal(stats[1], results[1][2][1])


@pytest.mark.parametrize("R,J", SILENT)
def test_a_kl_term_that_overflows_stays_in_its_row(R, J):
    """With a weight the infinite term is the formula's own: the loss is infinite, the rows beside it are as ever."""
    import torch
    from snntc_2023_b200 import train
    z, lab, old, adv, refp, at = _beside_a_silent_label(R, J, R + J)
    z1 = z.clone().requires_grad_(True)
    loss = train.policy_loss(z1, lab, old, adv, ref_logp=refp, kl_coef=0.1)
    (grad,) = torch.autograd.grad(loss, z1)
    assert float(loss.detach()) == math.inf and not grad[at].isfinite().all()
    ref = Ref(z, lab)
    want = _policy_ref(ref, old, adv, refp, 0.2, 0.2, 0.1)
    ref.counts[at] = False                            # (left out of what follows)
    grad[at] = 0
    ref.check_grad(grad, want["factor"], want["factor_tol"])


@pytest.mark.parametrize("R,J", SILENT)
def test_an_advantage_of_nothing_beside_a_ratio_that_overflows(R, J):
    """A label that the old network gave next to nothing: its ratio overflows, and with an advantage of 0 the row has no part in the
    loss, as with any other ratio."""
    import torch
    from snntc_2023_b200 import train
    z, lab, old, adv, _, at = _beside_a_silent_label(R, J, R + J + 1)
    z[at, lab[at]] = 1.0
    adv[at] = 0.0
    results = []
    for o in (-1e5, -0.5):
        old[at] = o
        z1 = z.clone().requires_grad_(True)
        loss = train.policy_loss(z1, lab, old, adv)
        (grad,) = torch.autograd.grad(loss, z1)
        results.append((loss.detach(), grad))
    assert results[0][0].isfinite() and not results[0][1][at].any()
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
    z[at, 0] = float("nan")                           # what is no number stays so
    assert train.policy_loss(z, lab, old, adv).isnan()


@pytest.mark.parametrize("P", [2, 20])
@pytest.mark.parametrize("smoothing", [0.0, 1.0])
def test_a_margin_without_bounds_beside_a_smoothing_of_nothing(P, smoothing):
    """A text with a label that its network rules out (an output at +inf) has an infinite margin. Where that is the side which the
    loss wants, the pair's loss is 0, as its limit is: -log sigma(inf), and nothing of the other side's."""
    import torch
    from snntc_2023_b200 import train
    z, lab = _logits(6 * P, 12, P, ignore=0.0)
    starts = torch.arange(0, 6 * P + 1, 3, device="cuda")
    refp = train.label_log_probs(z, lab).view(2 * P, 3).sum(1)            # margins near 0 elsewhere
    row = 3 * P + 1 if smoothing == 0 else 1                              # of the rejected text of pair 0, or of the preferred one
    z[row, lab[row]] = float("inf")
    z1 = z.clone().requires_grad_(True)
    loss, m = train.preference_loss(z1, lab, starts, ref_logp=refp, label_smoothing=smoothing, with_margins=True)
    (grad,) = torch.autograd.grad(loss, z1)
    assert float(m[0]) == (math.inf if smoothing == 0 else -math.inf) and m[1:].isfinite().all()
    # the other pairs: m is 0 but for lp's 32 bits in refp, below 1e-3 beside rows of 1e5 (u |lp| of three rows, times 0.1)
    assert abs(float(loss) - math.log(2) * (P - 1) / P) < 1e-3 * math.log(2)
    pair = torch.zeros(6 * P, dtype=torch.bool, device="cuda")
    pair[0:3] = pair[3 * P:3 * P + 3] = True
    assert grad.isfinite().all() and not grad[pair].any() and grad[~pair].any()


def _one_loss(kind, z, lab, old, adv, refp, starts):
    from snntc_2023_b200 import train
    if kind == "policy":
        return train.policy_loss(z, lab, old, adv, ref_logp=refp, kl_coef=0.1)
    return train.preference_loss(z, lab, starts, beta=0.01) if kind == "preference" else train.label_log_probs(z, lab).sum()


def _check_one_loss(kind, grad, z, lab, old, adv, refp, starts):
    import torch
    ref = Ref(z.detach(), lab)
    if kind == "policy":
        want = _policy_ref(ref, old, adv, refp, 0.2, 0.2, 0.1)
    elif kind == "preference":
        want = _preference_ref(ref, starts, None, 0.01, 0.0)
    else:
        want = dict(factor=torch.ones_like(ref.lp), factor_tol=torch.zeros_like(ref.lp))
    ref.check_grad(grad, want["factor"], want["factor_tol"])


def _one_loss_inputs(R, J, seed):
    """Ratios at exp(+-0.1), inside the clip."""
    import torch
    z, lab = _logits(R, J, seed)
    g = torch.Generator("cuda").manual_seed(seed)
    lp = Ref(z, lab).lp
    old = (lp + 0.1 * torch.randn(R, device="cuda", generator=g).sign()).float()
    starts = torch.tensor([0, R // 4 + seed % 2, R // 2, R // 2 + 1, R - 1], device="cuda")
    return [z, lab, old, torch.randn(R, device="cuda", generator=g), (lp + 0.1).float(), starts]


@pytest.mark.parametrize("R,J", [(64, 10), (300, 500), (40, 20011)])
@pytest.mark.parametrize("kind", ["policy", "preference", "logp"])
def test_forward_and_backward_captured_apart(R, J, kind):
    """Two graphs, the backward's replayed again and again behind one replay of the forward's, with other upstream gradients: each
    replay the gradient at the inputs of the last forward."""
    import torch
    sets = [_one_loss_inputs(R, J, 80 + k) for k in range(2)]
    up = torch.ones((), device="cuda")
    own = [t.clone() for t in sets[0]]
    own[0].requires_grad_(True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(_one_loss(kind, *own), own[0], up)
    torch.cuda.synchronize()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, stream=side):
        loss = _one_loss(kind, *own)
    with torch.cuda.graph(backward, stream=side, pool=forward.pool()):
        (grad,) = torch.autograd.grad(loss, own[0], up, retain_graph=True)

    def replay(k):
        for dst, src in zip(own, sets[k]):
            dst.data.copy_(src)                       # (not autograd's to notice: the forward's replay follows)
        forward.replay()

    for k in (1, 0):
        replay(k)
        for u in (-2.0, 0.0, 1.0, 4.0, 4.0):          # (powers of two move no rounding)
            up.fill_(u)
            backward.replay()
            if u == 0:
                assert not grad.any()
            else:
                _check_one_loss(kind, grad / u, *sets[k])
    torch.cuda.synchronize()
    # and an eager backward of the captured forward: a tensor of its own, which later replays leave alone
    with torch.cuda.stream(side):
        (mine,) = torch.autograd.grad(loss, own[0], up, retain_graph=True)
    torch.cuda.synchronize()
    replay(1)
    backward.replay()
    _check_one_loss(kind, mine / 4.0, *sets[0])
    _check_one_loss(kind, grad / 4.0, *sets[1])


def test_a_captured_backward_of_an_eager_loss():
    """The forward ran eagerly, on the stream that the backward is captured on."""
    import torch
    own = _one_loss_inputs(50, 30, 5)
    z = own[0].clone().requires_grad_(True)
    up = torch.full((), -2.0, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = _one_loss("policy", z, *own[1:])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        (grad,) = torch.autograd.grad(loss, z, up, retain_graph=True)
    for u in (-2.0, 4.0, 4.0, 0.0, 1.0):
        up.fill_(u)
        graph.replay()
        if u == 0:
            assert not grad.any()
        else:
            _check_one_loss("policy", grad / u, *own)


# Row lengths and counts that the shapes above leave out: rows streamed by a warp (1025 to 1800 outputs), parts of a warp to a row with more
# rows than one cluster takes, and two turns of the one cluster (9 to 16 CTAs' worth of rows).
MORE_SHAPES = [(40, 1500), (3000, 1501), (7, 1800), (300, 1025), (2000, 60), (2000, 120), (600, 250), (200, 500), (100, 500), (3000, 10), (700, 50),
               (20000, 30)]


@pytest.mark.parametrize("R,J", MORE_SHAPES)
def test_label_log_probs_of_more_shapes(R, J):
    test_label_log_probs_and_their_gradient(R, J)


@pytest.mark.parametrize("R,J", MORE_SHAPES)
def test_policy_loss_of_more_shapes(R, J):
    """Ratios at exp(+-0.1) and, beyond the clip, at exp(+-0.5)."""
    import torch
    from snntc_2023_b200 import train
    z, lab = _logits(R, J, R + 5 * J)
    ref = Ref(z, lab)
    g = torch.Generator("cuda").manual_seed(9)
    off = torch.tensor([-0.5, -0.1, 0.1, 0.5], device="cuda")[torch.randint(0, 4, (R,), device="cuda", generator=g)]
    old, adv, refp = (ref.lp + off).float(), torch.randn(R, device="cuda", generator=g), (ref.lp + 0.5 * torch.randn(R, device="cuda", generator=g)).float()
    want = _policy_ref(ref, old, adv, refp, 0.2, 0.25, 0.3)
    assert not want["near"]
    z1 = z.clone().requires_grad_(True)
    loss, stats = train.policy_loss(z1, lab, old, adv, ref_logp=refp, clip_low=0.2, clip_high=0.25, kl_coef=0.3, with_stats=True)
    for got, name in ((loss.detach(), "loss"), (stats[0], "kl")):
        assert abs(float(got) - want[name]) <= want[name + "_tol"] + abs(want[name]) * U
    assert abs(float(stats[1]) - want["clipped"]) <= U
    for _ in range(2):                                # the gradient that was formed with the loss, and one formed from what it keeps
        (grad,) = torch.autograd.grad(loss, z1, retain_graph=True)
        ref.check_grad(grad, want["factor"], want["factor_tol"])


@pytest.mark.parametrize("R,J", MORE_SHAPES)
def test_preference_loss_of_more_shapes(R, J):
    for with_ref in (True, False):
        test_preference_loss_and_its_gradient(R, J, 3, 2, with_ref)


def test_two_threads_and_their_errors():
    """As test_two_threads_at_once, with an error in a thread as an error of the test, and every round counted."""
    from concurrent.futures import ThreadPoolExecutor

    import torch
    cases = []
    for k, (R, J) in enumerate(((300, 40), (64, 9000))):
        z, lab = _logits(R, J, 70 + k)
        cases.append((z, lab, -2 - torch.rand(R, device="cuda"), torch.randn(R, device="cuda"), -2 - torch.rand(R, device="cuda"),
                      torch.tensor([0, R // 4, R // 2, R // 2, R], device="cuda")))
    plain = [_all_losses(c[0].clone().requires_grad_(True), *c[1:]) for c in cases]
    torch.cuda.synchronize()

    def work(k):
        equal = 0
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = _all_losses(cases[k][0].clone().requires_grad_(True), *cases[k][1:])
                torch.cuda.current_stream().synchronize()
                equal += len(got) == len(plain[k]) and all(torch.equal(a, b) for a, b in zip(got, plain[k]))
        return equal

    with ThreadPoolExecutor(2) as pool:
        assert list(pool.map(work, range(2))) == [20, 20]


@pytest.mark.parametrize("R,J", SILENT)
def test_a_label_that_its_network_rules_out(R, J):
    """The label's output at +inf: its ratio is 0, its KL term infinite, which is the mean's; the loss without a weight for it is finite,
    and with one infinite, no NaN."""
    import torch
    from snntc_2023_b200 import train
    z, lab, old, adv, refp, at = _beside_a_silent_label(R, J, R + J + 2)
    z[at, lab[at]] = math.inf
    old[at], adv[at] = -2.0, 1.0
    z1 = z.clone().requires_grad_(True)
    loss, stats = train.policy_loss(z1, lab, old, adv, ref_logp=refp, with_stats=True)
    (grad,) = torch.autograd.grad(loss, z1)
    assert loss.isfinite() and float(stats[0]) == math.inf and grad.isfinite().all() and not grad[at].any()
    assert float(train.policy_loss(z, lab, old, adv, ref_logp=refp, kl_coef=0.1)) == math.inf
