"""The policy operators from their formulas, one position at a time in 64 bits
(numpy), with a bound on the rounding of the 32-bit kernels beside each result.

u = 2^-24 is half a step of fp32. The bounds count roundings of the formulas,
not of a particular order: for a listed move with s = (z - top) / T,
* s: the subtraction, 1/T and the product: 3 u |s|;
* exp(s): 4 u (two steps of the function) + 3 u |s|; the sum of at most 256 of
  them over 8 + 5 additions: 13 u more; weighted by p the |s| average at most
  log 256 < 6, so log(sum) is off by at most u (4 + 13 + 3 * 6) + 4 u of its own;
* logp = s - log(sum): at most u (40 + 4 |s| + 4 log(sum)); ``slack`` below doubles it.
p = exp(s) / sum has that relative error. A result that is a sum of products of
p, logp and given numbers is off by at most slack * u * (the sum of the
products' magnitudes, with 1 added to each logp), plus half a step of its type.
"""
import numpy as np

U = 2.0 ** -24


class Row:
    """Softmax of one position's list; ``cols`` None for a malformed list."""

    def __init__(self, logits, cols, temp):
        self.cols = np.asarray(cols[:256], np.int64)
        z = np.zeros(len(self.cols))
        ok = (self.cols >= 0) & (self.cols < len(logits))
        z[ok] = np.asarray(logits, np.float64)[self.cols[ok]]
        self.ok, self.z, self.temp = ok, z, temp
        self.live = len(z) > 0 and not np.all(z == -np.inf)
        with np.errstate(all="ignore"):
            if self.live:
                top = z.max() if not np.isnan(z).any() else np.nan
                s = (z - top) / temp
                e = np.exp(s)
                self.log_s = np.log(e.sum())
                self.logp, self.p = s - self.log_s, e / e.sum()
                self.h = -np.sum(np.where(self.p > 0, self.p * self.logp, self.p))
                far = np.abs(s[np.isfinite(s)])
                far = far[far < 1e4]
                self.slack = 80 + 8 * (far.max() if len(far) else 0) + 8 * np.nan_to_num(self.log_s)
            else:
                self.logp, self.p = np.full(len(z), -np.inf), np.zeros(len(z))
                self.h, self.log_s, self.slack = 0.0, 0.0, 80.0

    def dense(self, g, size):
        """Values per listed move -> the row; repeated columns get the sum."""
        row = np.zeros(size)
        np.add.at(row, self.cols[self.ok], np.asarray(g)[self.ok])
        return row

    def backward(self, gm, ga, played, gh):
        """(gradient, magnitudes) of each listed move's logit."""
        with np.errstate(all="ignore"):
            one = np.zeros(len(self.p))
            if played >= 0:
                one[played] = 1
            lp = np.where(self.p > 0, self.logp, 0)
            g = gm - self.p * (gm.sum() + ga) + one * ga - gh * self.p * (lp + self.h)
            m = np.abs(gm) + self.p * (np.abs(gm).sum() + abs(ga)) + one * abs(ga) + abs(gh) * self.p * (np.abs(lp) + self.h + 1)
        return g / self.temp, m / self.temp


def step(dtype):
    """Half a step of the type, relative, and below its normal range absolute."""
    return {"f32": (2.0 ** -24, 2.0 ** -149), "bf16": (2.0 ** -8, 2.0 ** -133), "f16": (2.0 ** -11, 2.0 ** -25)}[dtype]


def grad_bound(g, m, slack, dtype):
    rel, tiny = step(dtype)
    off = slack * U * m + 1e-37
    return off + rel * (np.abs(g) + off) + tiny


def clip_row(row, played, old, adv, weight, ref, low, high, beta, eta, scale):
    """Loss, KL and gradient of one position, with their bounds: a dict."""
    with np.errstate(all="ignore"):
        lp = row.logp[played]
        r = np.exp(lp - old)
        border = 1 + high if adv > 0 else 1 - low
        active = not (r > border) if adv > 0 else not (r < border)
        kl = klm = 0.0
        delta = np.zeros(len(row.p))
        if ref is not None:
            both = row.p > 0
            delta = np.where(both, row.logp - ref.logp, 0)
            kl = np.sum(np.where(both, row.p * delta, 0))
            klm = np.sum((row.p + ref.p) * (1 + np.abs(delta)))
        w = scale * weight
        loss = w * (-adv * (r if active else border) + beta * kl - eta * row.h)
        one = np.zeros(len(row.p))
        one[played] = 1
        slope = -adv * r if active else 0.0
        lpg = np.where(row.p > 0, row.logp, 0)
        g = w / row.temp * (slope * (one - row.p) + beta * row.p * (delta - kl) + eta * row.p * (lpg + row.h))
        more = 1 + abs(lp) + abs(old)  # the ratio's own error: that of logp - old, relative
        m = abs(w) / row.temp * (abs(slope) * more * (one + row.p) + abs(beta) * row.p * (np.abs(delta) + kl + klm + 1) + abs(eta) * row.p * (np.abs(lpg) + row.h + 1))
        lossm = abs(w) * (abs(adv) * max(r, border) * more + abs(beta) * klm + abs(eta) * (row.h + 1))
    slack = max(row.slack, ref.slack) if ref is not None else row.slack
    return dict(loss=loss, kl=kl, g=g, loss_off=slack * U * lossm, kl_off=slack * U * klm, m=m, slack=slack, r=r, active=active)


def preference(gains_w, gains_l, beta, eps, w):
    m = beta * (gains_w - gains_l)
    less, more = np.logaddexp(0, -m), np.logaddexp(0, m)
    loss = w * ((1 - eps) * less + eps * more)
    up, down = np.exp(-np.logaddexp(0, -m)), np.exp(-np.logaddexp(0, m))
    return m, loss, w * beta * (eps * up - (1 - eps) * down)
