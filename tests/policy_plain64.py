"""The policy operators' formulas over a whole batch at once, in 64-bit torch
operations on the tensors' device, with the bounds that policy_reference.py
derives. For batches too large to go through row by row: finite logits, lists
of at most 256 moves."""
import torch

from tests.policy_reference import U, step


class Rows64:
    def __init__(self, logits, off, index, played, temp):
        self.n, self.classes = logits.shape
        self.temp, dev = temp, logits.device
        off = off.long() - off[0].long()
        self.count = off[1:] - off[:-1]
        self.row = torch.repeat_interleave(torch.arange(self.n, device=dev), self.count)
        self.cols = index.long()
        z = logits[self.row, self.cols].double()
        low = torch.full((self.n,), -torch.inf, dtype=torch.float64, device=dev)
        self.s = (z - low.scatter_reduce(0, self.row, z, "amax")[self.row]) / temp
        e = torch.exp(self.s)
        total = self.sum(e)
        self.live = self.count > 0
        self.log_s = torch.log(torch.where(self.live, total, 1.0))
        self.logp, self.p = self.s - self.log_s[self.row], e / total[self.row]
        self.h = -self.sum(self.p * self.logp)
        far = torch.zeros_like(self.log_s).scatter_reduce(0, self.row, self.s.abs(), "amax")
        self.slack = 80 + 8 * far + 8 * self.log_s
        self.takes = self.live & (played >= 0)
        self.at = (off[:-1] + played.long())[self.takes]  # entry of each played move
        self.one = torch.zeros_like(self.p)
        self.one[self.at] = 1.0
        self.played_logp = torch.zeros_like(self.log_s)
        self.played_logp[self.takes] = self.logp[self.at]

    def sum(self, v):
        return torch.zeros(self.n, dtype=torch.float64, device=v.device).index_add_(0, self.row, v)

    def backward(self, gm, ga, gh):
        """Gradient of each listed move's logit from those of logp, played
        log-probability and entropy (per move, per row, per row), and its magnitudes."""
        ga, gh = torch.where(self.takes, ga.double(), 0.0), gh.double()
        gm, r = gm.double(), self.row
        g = gm - self.p * (self.sum(gm) + ga)[r] + self.one * ga[r] - gh[r] * self.p * (self.logp + self.h[r])
        m = (gm.abs() + self.p * (self.sum(gm.abs()) + ga.abs())[r] + self.one * ga.abs()[r]
             + gh.abs()[r] * self.p * (self.logp.abs() + self.h[r] + 1))
        return g / self.temp, m / self.temp

    def dense(self, g):
        out = torch.zeros(self.n, self.classes, dtype=torch.float64, device=g.device)
        return out.index_put_((self.row, self.cols), g, accumulate=True)

    def check_dense(self, got, g, m, slack, dtype):
        """got against the rows of g, off by the roundings that m and slack (per move) count."""
        rel, tiny = step(dtype)
        want = self.dense(g)
        off = self.dense(slack * U * m + 1e-37)
        off += rel * (want.abs() + off) + tiny * self.dense(torch.ones_like(g))
        return near(got, want, off)


def clip64(r, old, adv, weight, ref, low, high, beta, eta, scale):
    """Loss, KL, gradient and their bounds (policy_reference.clip_row over a batch)."""
    old, adv, w = old.double(), adv.double(), weight.double() * scale
    lp = r.played_logp
    ratio = torch.exp(lp - old)
    border = torch.full_like(adv, 1 - low).masked_fill_(adv > 0, 1 + high)  # (where() of two numbers is 32-bit)
    active = torch.where(adv > 0, ratio <= border, ratio >= border)
    kl = klm = torch.zeros_like(lp)
    delta, slack = torch.zeros_like(r.p), r.slack
    if ref is not None:
        delta = r.logp - ref.logp
        kl = r.sum(r.p * delta)
        klm = r.sum((r.p + ref.p) * (1 + delta.abs()))
        slack = torch.maximum(slack, ref.slack)
    loss = w * (-adv * torch.where(active, ratio, border) + beta * kl - eta * r.h)
    slope = torch.where(active, -adv * ratio, 0.0)
    more = 1 + lp.abs() + old.abs()
    k = r.row
    g = (w / r.temp)[k] * (slope[k] * (r.one - r.p) + beta * r.p * (delta - kl[k]) + eta * r.p * (r.logp + r.h[k]))
    m = (w.abs() / r.temp)[k] * ((slope.abs() * more)[k] * (r.one + r.p) + beta * r.p * (delta.abs() + (kl + klm)[k] + 1)
                                 + eta * r.p * (r.logp.abs() + r.h[k] + 1))
    lossm = w.abs() * (adv.abs() * torch.maximum(ratio, border) * more + beta * klm + eta * (r.h + 1))
    takes = r.takes
    return dict(loss=torch.where(takes, loss, 0.0), loss_off=torch.where(takes, slack * U * lossm + U * loss.abs(), 0.0),
                kl=kl, kl_off=slack * U * klm, g=torch.where(takes[k], g, 0.0), m=torch.where(takes[k], m, 0.0), slack=slack[k])


def near(got, want, off):
    bad = ~((got.double() - want).abs() <= off)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), want[bad][:4].tolist(), int(bad.sum()))
