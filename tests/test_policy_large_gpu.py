"""The policy operators where warps take many positions one after another:
lists loaded ahead, turns from the shared counter, long lists first (and too
many of them for that), row images that are used again, totals by a cluster."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from metalfish_b200 import policy  # noqa: E402
from tests.policy_plain64 import Rows64, clip64, near  # noqa: E402
from tests.policy_reference import U  # noqa: E402

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MARK = 12345.0  # what no result is: an entry that was not written shows


class Big:
    """n positions of `shortest` to 60 moves, a share of them 65 to 218 (or 256,
    the last that counts); columns 3 apart from a random start, none twice."""

    def __init__(self, dtype, n, classes=1858, long_share=0.04, shortest=0, pad=0, temp=1.0, seed=0):
        rng = np.random.default_rng(seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        count = rng.integers(shortest, 61, n)
        long = rng.random(n) < long_share
        count[long] = rng.integers(65, min(219, classes), int(long.sum()))
        if classes > 256 and long.any():
            count[np.flatnonzero(long)[0]] = 256
        off = np.concatenate([[0], np.cumsum(count)])
        row = np.repeat(np.arange(n), count)
        start = rng.integers(0, classes, n)
        assert math.gcd(3, classes) == 1
        self.index = torch.from_numpy(((start[row] + 3 * (np.arange(off[-1]) - off[row])) % classes).astype(np.int16)).cuda()
        self.off = torch.from_numpy((off + 11).astype(np.int32)).cuda()  # lists that do not start at 0
        played = np.where(rng.random(n) < 0.1, -1, (rng.random(n) * np.minimum(count, 256)).astype(np.int64))
        self.played = torch.from_numpy(np.where(count > 0, played, -1).astype(np.int32)).cuda()
        self.logits = (2 * torch.randn(n, classes + pad, generator=g, device="cuda")).to(TYPES[dtype])[:, :classes]
        self.dtype, self.n, self.classes, self.temp, self.gen = dtype, n, classes, temp, g
        self.long = int((count > 64).sum())

    def rows64(self, logits=None):
        return Rows64(self.logits if logits is None else logits, self.off, self.index, self.played, self.temp)

    def noise(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda")

    def struct(self):
        return policy._rows(self.logits, self.off, self.index, self.played, self.temp)[0]

    def full(self, n=None):
        return torch.full((self.n if n is None else n,), MARK, device="cuda")

    def grad(self, kind=None, pad=0):
        wide = torch.full((self.n, self.classes + pad), MARK, device="cuda").to(TYPES[kind or self.dtype])
        return wide, wide[:, :self.classes]


# positions for more than three turns of 5920 (scores, lines) or 3552 (row images) warps;
# with 60000, every list long, a CTA has more than the 64 that it can keep
SIZES = [dict(n=20011), dict(n=20011, pad=6, temp=1.3), dict(n=13001, classes=4288), dict(n=60000, classes=301, long_share=1.0),
         dict(n=700, classes=32767), dict(n=12001, long_share=0.0, shortest=1)]
IDS = ["20011", "20011 padded", "13001 wide", "60000 long", "700 widest", "12001 short"]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("size", SIZES, ids=IDS)
def test_scores(dtype, size):
    x = Big(dtype, seed=1, **size)
    moves, at, h = x.full(len(x.index)), x.full(), x.full()
    policy._call(policy._lib().mfb200_move_logprobs, 0, x.struct(), moves.data_ptr(), at.data_ptr(), h.data_ptr())
    r = x.rows64()
    near(moves, r.logp, (r.slack * U)[r.row] * (1 + r.logp.abs()))
    near(at, r.played_logp, r.slack * U * (1 + r.played_logp.abs()))
    near(h, r.h, r.slack * U * (1 + 2 * r.h))


@pytest.mark.parametrize("dtype,kind", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f32", "f16")])
@pytest.mark.parametrize("size", SIZES, ids=IDS)
def test_backward(dtype, kind, size):
    x = Big(dtype, seed=2, **size)
    gm, ga, gh = x.noise(len(x.index)), x.noise(x.n), x.noise(x.n)
    wide, grad = x.grad(kind, 5)
    policy.move_logprobs_backward(x.logits, x.off, x.index, x.played, grad_moves=gm, grad_played=ga, grad_entropy=gh,
                                  softmax_temp=x.temp, grad_logits=grad)
    r = x.rows64()
    g, m = r.backward(gm, ga, gh)
    r.check_dense(grad, g, m, r.slack[r.row], kind)
    assert (wide[:, x.classes:] == wide[0, -1]).all() and wide[0, -1] == torch.tensor(MARK).to(TYPES[kind])


@pytest.mark.parametrize("with_grad", [True, False], ids=["gradient", "no gradient"])
@pytest.mark.parametrize("dtype,ref_dtype", [("f32", "f32"), ("bf16", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", None), ("f32", None)])
@pytest.mark.parametrize("size", SIZES, ids=IDS)
def test_clipped_loss(dtype, ref_dtype, size, with_grad):
    x = Big(dtype, seed=3, **size)
    r = x.rows64()
    other = None if ref_dtype is None else (x.logits.float() + 0.3 * x.noise(x.n, x.classes)).to(TYPES[ref_dtype])
    old, adv, w = (r.played_logp + 0.3 * x.noise(x.n)).float(), x.noise(x.n), x.noise(x.n).abs()
    beta, eta, scale = 0.1 if other is not None else 0.0, 0.02, 64.0 / x.n
    out = [x.full() for _ in range(4)]
    total = x.full(1)
    wide, grad = x.grad()
    cfg = policy._ClipConfig(0.2, 0.3, beta, eta, scale)
    p = [None if t is None else t.data_ptr() for t in (out[0], out[1], None if other is None else out[2], out[3])]
    policy._call(policy._lib().mfb200_clipped_policy_loss, 0, x.struct(), cfg, old.data_ptr(), adv.data_ptr(), w.data_ptr(),
                 None if other is None else other.data_ptr(), x.classes, policy.TYPES[other.dtype] if other is not None else 0,
                 *p, total.data_ptr(), grad.data_ptr() if with_grad else None, x.classes, policy.TYPES[grad.dtype])
    loss, logp, kl, h = out
    d = clip64(r, old, adv, w, None if other is None else x.rows64(other), 0.2, 0.3, beta, eta, float(np.float32(scale)))
    near(loss, d["loss"], d["loss_off"])
    near(logp, r.played_logp, r.slack * U * (1 + r.played_logp.abs()))
    near(h, r.h, r.slack * U * (1 + 2 * r.h))
    if other is not None:
        near(kl, d["kl"], d["kl_off"])
    check_total(total, loss)
    if with_grad:
        r.check_dense(grad, d["g"], d["m"], d["slack"], dtype)


def check_total(total, loss):
    """Losses summed in 64 bits, in some order, and rounded once."""
    v = loss.double().cpu().numpy()
    want = math.fsum(v)
    assert abs(total.item() - want) <= U * abs(want) + len(v) * 2.0 ** -53 * np.abs(v).sum()


@pytest.mark.parametrize("n", [1, 31, 15360, 15361, 16384, 16385, 50001, 131073])
def test_totals(n):
    """By one CTA up to 16384 losses, by a cluster of eight above; 16 loads at once from 15361."""
    x = Big("f32", n, classes=64, long_share=0.0, shortest=1, seed=4)
    one = torch.ones(n, device="cuda")
    out = policy.clipped_policy_loss(x.logits, x.off, x.index, x.played, -one, x.noise(n), entropy_coef=0.1, grad=False)
    assert out.grad_logits is None
    check_total(out.total, out.loss)


def line_cuts(n, lines, rng):
    """2 * pairs lines over the n positions, some of none; positions before and behind them in none."""
    cuts = np.sort(rng.integers(5, n - 4, lines + 1))
    cuts[3] = cuts[4]
    return cuts


@pytest.mark.parametrize("with_grad", [True, False], ids=["gradient", "no gradient"])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("size,pairs", [(dict(n=20011), 90), (dict(n=20011, pad=6, temp=1.3), 4000), (dict(n=13001, classes=4288), 6),
                                        (dict(n=60000, classes=301, long_share=1.0), 20000), (dict(n=700, classes=32767), 30)],
                         ids=["20011", "20011 padded", "13001 wide", "60000 long", "700 widest"])
def test_preference(dtype, size, pairs, with_grad):
    x = Big(dtype, seed=5, **size)
    rng = np.random.default_rng(6)
    cuts = line_cuts(x.n, 2 * pairs, rng)
    lines = torch.from_numpy(cuts.astype(np.int32)).cuda()
    r = x.rows64()
    frozen = (r.played_logp + 0.3 * x.noise(x.n)).float()
    w = x.noise(pairs).abs() + 0.5
    beta, eps, scale = 0.25, 0.125, 8.0
    logp, rest, row_grad, line_logp, margin, loss, total = (x.full(k) for k in (x.n, x.n, x.n, 2 * pairs, pairs, pairs, 1))
    wide, grad = x.grad()
    policy._call(policy._lib().mfb200_preference_loss, 0, x.struct(), policy._PreferenceConfig(beta, eps, scale), lines.data_ptr(), pairs,
                 frozen.data_ptr(), w.data_ptr(), logp.data_ptr(), rest.data_ptr(), row_grad.data_ptr(), line_logp.data_ptr(),
                 margin.data_ptr(), loss.data_ptr(), total.data_ptr(), grad.data_ptr() if with_grad else None, x.classes,
                 policy.TYPES[grad.dtype])
    # a log-probability is made in 64 bits (policy_reference: 100 steps of 2^-52 for kernel and oracle,
    # per unit of |s| and log S) and rounded once; its rest once more
    tiny = 100 * 2.0 ** -52 * (1 + r.slack / 8)
    near(logp, r.played_logp, U * r.played_logp.abs() + tiny)
    near(logp.double() + rest.double(), r.played_logp, U ** 2 * r.played_logp.abs() + tiny)
    line = torch.bucketize(torch.arange(x.n, device="cuda"), lines.long(), right=True) - 1  # -1 and 2 pairs: in none
    inside = (line >= 0) & (line < 2 * pairs)

    def per_line(v):
        return torch.zeros(2 * pairs, dtype=torch.float64, device="cuda").index_add_(0, line[inside], v[inside])

    gain = torch.where(r.takes, r.played_logp - frozen.double(), 0.0)
    gains, sums = per_line(gain), per_line(r.played_logp)
    deep = per_line(torch.ones_like(gain)) + 8  # additions of a line
    off = per_line(U ** 2 * r.played_logp.abs() + tiny) + deep * 2.0 ** -52 * per_line(gain.abs() + r.played_logp.abs())
    near(line_logp, sums, off + U * sums.abs())
    m = beta * (gains[::2] - gains[1::2])
    m_off = beta * (off[::2] + off[1::2]) + 2 * U * m.abs()
    near(margin, m, m_off)
    less, more = torch.nn.functional.softplus(-m, threshold=1e9), torch.nn.functional.softplus(m, threshold=1e9)
    c = w.double() * scale
    want = c * ((1 - eps) * less + eps * more)
    near(loss, want, c * (m_off + 16 * U * (1 + m.abs())))
    check_total(total, loss)
    slope = c * beta * (eps * torch.sigmoid(m) - (1 - eps) * torch.sigmoid(-m))
    slope_off = c * beta * (m_off + 16 * U)
    pair = (line // 2).clamp(0, pairs - 1)
    ga = torch.where(inside & r.takes, torch.where(line % 2 == 0, slope[pair], -slope[pair]), 0.0)
    near(row_grad, ga, torch.where(ga != 0, slope_off[pair] + U * ga.abs(), 0.0))
    if with_grad:
        none = torch.zeros_like(r.p)
        g, mag = r.backward(none, ga, torch.zeros_like(ga))
        more = slope_off[pair] / ga.abs().clamp(min=1e-30) / U  # the slope's own error, relative to it
        r.check_dense(grad, g, mag, (r.slack + more)[r.row], dtype)


def test_visit_counts_over_a_training_batch():
    """The scores and their backward pass, one after the other as a step takes them, in 16 bits."""
    x = Big("bf16", 16384, seed=7)
    r = x.rows64()
    visits = torch.rand(len(x.index), generator=x.gen, device="cuda")
    visits = (visits / r.sum(visits.double())[r.row]).float() / x.n
    out = policy.move_logprobs(x.logits, x.off, x.index)
    grad = policy.move_logprobs_backward(x.logits, x.off, x.index, grad_moves=-visits)
    near(out.moves, r.logp, (r.slack * U)[r.row] * (1 + r.logp.abs()))
    zero = torch.zeros(x.n, device="cuda")
    g, m = r.backward(-visits, zero, zero)
    r.check_dense(grad, g, m, r.slack[r.row], "bf16")
