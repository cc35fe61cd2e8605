"""Infinities, switched-off terms, far offsets and rows that take no part, in
the policy operators: against their formulas in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from metalfish_b200 import policy  # noqa: E402
from tests import policy_reference as ref  # noqa: E402
from tests.test_policy_ops_gpu import Batch, check_clip, clip_case, line_case, near  # noqa: E402

pytestmark = pytest.mark.gpu
INF = np.inf


def play(x, at):
    x.played_host[:] = at
    x.played.copy_(torch.from_numpy(x.played_host))


def terms(m, eps):
    """-(1 - eps) log sigma(m) - eps log sigma(-m), without the term whose
    coefficient is 0: the definition at an infinite margin."""
    return ((1 - eps) * np.logaddexp(0, -m) if eps < 1 else 0.0) + (eps * np.logaddexp(0, m) if eps > 0 else 0.0)


@pytest.mark.parametrize("eps", [0.0, 0.25, 1.0])
def test_preference_with_infinite_margins(eps):
    """A played move of logit -inf (log-probability -inf) in the rejected or
    the preferred line, and a reference value of -inf in either: the margin is
    infinite, the loss is 0 where only the term that is left has a coefficient."""
    x = Batch("f32", 1858, [20] * 12, 40)
    play(x, 3)
    for b in (3, 4):  # rejected move of pair 1, preferred one of pair 2
        x.logits[b, int(x.lists[b][3])] = -INF
    rows, logp, frozen, lines = line_case(x, np.arange(13))
    frozen[[3, 4]] = -3.0  # (from line_case they are -inf too, and the difference undefined)
    frozen[[3, 4]] = -3.0  # (from line_case they are -inf too, and the difference undefined)
    frozen[[3, 4]] = -3.0  # (from line_case they are -inf too, and the difference undefined)
    frozen[[3, 4]] = -3.0  # (from line_case they are -inf too, and the difference undefined)
    frozen[[3, 4]] = -3.0  # (from line_case they are -inf too, and the difference undefined)
    frozen[6] = frozen[9] = -INF  # preferred of pair 3, rejected of pair 4
    want = [None, INF, -INF, INF, -INF, None]
    scale = 3.0
    out = policy.preference_loss(*x.args(), lines, x.f32(frozen), beta=0.4, label_smoothing=eps, scale=scale)
    for i, m in enumerate(want):
        got, loss = out.margin[i].item(), out.loss[i].item()
        if m is None:
            assert np.isfinite(got) and np.isfinite(loss)
            continue
        assert got == m
        assert loss == scale * terms(m, eps), (i, loss)
        # sigma(m) and sigma(-m) are 0 and 1: U covers the one product's rounding
        slope = scale * 0.4 * (eps * (m > 0) - (1 - eps) * (m < 0))
        near(out.row_grad[2 * i:2 * i + 2].cpu().numpy(), [slope, -slope], 4 * ref.U * abs(slope), "row_grad")
    assert torch.isfinite(out.grad_logits).all()
    finite = torch.isfinite(out.loss)
    total = out.loss.double().sum().item()
    assert (out.total.item() == INF) if not finite.all() else abs(out.total.item() - total) <= 2 * ref.U * abs(total)


def test_preference_without_a_margin():
    """beta 0 takes the margin out, an infinite one too."""
    x = Batch("f32", 1858, [20] * 2, 41)
    play(x, 3)
    x.logits[1, int(x.lists[1][3])] = -INF
    lines = torch.arange(3, dtype=torch.int32, device="cuda")
    out = policy.preference_loss(*x.args(), lines, torch.zeros(2, device="cuda"), beta=0.0)
    assert out.margin.item() == 0 and (out.grad_logits == 0).all()
    near(out.loss.item(), np.log(2), 4 * ref.U)


@pytest.mark.parametrize("value", [-INF, INF, np.nan])
@pytest.mark.parametrize("dtype,ref_dtype", [("f32", "f32"), ("bf16", "f32")])
def test_kl_is_watched_without_taking_part(value, dtype, ref_dtype):
    """With kl_coef 0 the KL is given and is no part of the loss, whatever it is."""
    x = Batch(dtype, 1858, [40, 70, 0, 20], 42)
    play(x, [3, 66, -1, 5])
    rows, other, old, adv, w = clip_case(x, True, ref_dtype)
    for b in (0, 1, 3):
        other[b, int(x.lists[b][9])] = value
    args = x.f32(old), x.f32(adv)
    out = policy.clipped_policy_loss(*x.args(), *args, ref_logits=other, weight=x.f32(w), entropy_coef=0.02)
    kl = out.kl.cpu().numpy()
    assert kl[2] == 0
    assert np.all(kl[[0, 1, 3]] == INF) if value == -INF else np.isnan(kl[[0, 1, 3]]).all()
    check_clip(x, out, rows, None, old, adv, w, 0.2, 0.2, 0.0, 0.02, 0.25)


def test_advantage_of_zero_with_a_ratio_out_of_range():
    """-min(r A, clip(r) A) is 0 for A = 0, also where r overflows 32 bits or is infinite."""
    x = Batch("f32", 1858, [20] * 4, 43)
    play(x, 3)
    old = np.array([-200.0, -INF, -90.0, -3.0], np.float32)
    zero = torch.zeros(4, device="cuda")
    out = policy.clipped_policy_loss(*x.args(), x.f32(old), zero, entropy_coef=0.5, scale=1.0)
    rows = x.rows()
    for b, row in enumerate(rows):
        near(out.loss[b].item(), -0.5 * row.h, row.slack * ref.U * (1 + 2 * row.h), f"loss {b}")
    g = np.zeros((4, 1858))
    off = np.zeros((4, 1858))
    for b, row in enumerate(rows):
        v, m = row.backward(np.zeros(20), 0.0, 3, -0.5)
        g[b] = row.dense(v, 1858)
        off[b] = row.dense(row.slack * ref.U * m, 1858)
    near(out.grad_logits.cpu().numpy(), g, off + ref.U * np.abs(g), "grad")


@pytest.mark.parametrize("shift", [65536.0, -1e6, 3e7])
@pytest.mark.parametrize("which", ["policy", "reference"])
def test_kl_of_logits_with_an_offset_of_their_own(shift, which):
    """A softmax does not see a number that is added to a whole row. The given
    32-bit logits are the oracle's too, so its bounds hold unchanged: each
    logit minus its row's largest is exact or off by U of itself."""
    x = Batch("f32", 1858, [40, 64, 90, 2] * 8, 44)
    rows, other, old, adv, w = clip_case(x)
    if which == "policy":
        x.logits = x.logits + shift
    else:
        other = other + shift
    rows = x.rows()
    old = np.array([r.logp[a] if a >= 0 else 0.0 for r, a in zip(rows, x.played_host)], np.float32) - np.float32(0.1)
    out = policy.clipped_policy_loss(*x.args(), x.f32(old), x.f32(adv), ref_logits=other, weight=x.f32(w), kl_coef=0.3,
                                     entropy_coef=0.01)
    check_clip(x, out, rows, x.rows(other), old, adv, w, 0.2, 0.2, 0.3, 0.01, 1.0 / x.n)


@pytest.mark.parametrize("which", ["policy", "reference", "both"])
def test_kl_where_every_listed_logit_is_the_lowest(which):
    """A mask of the type's lowest value over a whole list makes it uniform."""
    x = Batch("f32", 1858, [40] * 4, 45)
    play(x, 3)
    rows, other, old, adv, w = clip_case(x)
    low = torch.finfo(torch.float32).min
    for b in (1, 2):
        at = torch.from_numpy(np.asarray(x.lists[b], np.int64)).cuda()
        if which != "reference":
            x.logits[b, at] = low
        if which != "policy":
            other[b, at] = low
    rows = x.rows()
    old = np.array([r.logp[3] for r in rows], np.float32)
    out = policy.clipped_policy_loss(*x.args(), x.f32(old), x.f32(adv), ref_logits=other, weight=x.f32(w), kl_coef=0.3)
    check_clip(x, out, rows, x.rows(other), old, adv, w, 0.2, 0.2, 0.3, 0.0, 0.25)


@pytest.mark.parametrize("value", [np.nan, INF])
def test_positions_that_take_no_part_have_no_gradient(value):
    """Padding of any content, in a line without a played move or in no line:
    its gradient is 0 and the pairs do not see it."""
    x = Batch("f32", 1858, [20, 70, 20, 20, 20, 90, 20], 46)
    play(x, [3, -1, -1, 2, 5, 6, 7])
    lines = torch.tensor([0, 3, 5], dtype=torch.int32, device="cuda")  # 5 and 6 are in no line
    frozen = torch.full((7,), -3.0, device="cuda")
    want = policy.preference_loss(*x.args(), lines, frozen)
    for b in (1, 2, 5, 6):
        x.logits[b, int(x.lists[b][7])] = value
    out = policy.preference_loss(*x.args(), lines, frozen)
    for a, b in ((out.total, want.total), (out.loss, want.loss), (out.margin, want.margin), (out.line_logp, want.line_logp),
                 (out.row_grad, want.row_grad)):
        assert torch.equal(a, b)
    assert (out.grad_logits[[1, 2, 5, 6]] == 0).all()
    assert torch.equal(out.grad_logits[[0, 3, 4]], want.grad_logits[[0, 3, 4]])
    # the clipped loss of a position without a played move likewise
    one = torch.ones(7, device="cuda")
    clip = policy.clipped_policy_loss(*x.args(), frozen, one, entropy_coef=0.1)
    assert (clip.grad_logits[[1, 2]] == 0).all() and (clip.loss[[1, 2]] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("gap", [0, 1, 5])
def test_gradient_in_the_logits_own_buffer(dtype, gap):
    """Logits and gradient in columns of one wide buffer, the gradient's rows at any
    alignment: as in buffers of their own, and nothing else is written."""
    x = Batch(dtype, 301, [20, 70, 0, 33, 300] * 60, 47)
    wide = torch.full((x.n, 2 * 301 + gap + 3), 7.0, dtype=x.logits.dtype, device="cuda")
    wide[:, 1:302] = x.logits
    before = wide.clone()
    logits, grad = wide[:, 1:302], wide[:, 302 + gap:603 + gap]
    rest = x.args()[1:]
    one = torch.ones(x.n, device="cuda")
    lines = torch.arange(0, x.n + 1, 10, dtype=torch.int32, device="cuda")
    want = [policy.move_logprobs_backward(*x.args(), grad_played=one),
            policy.clipped_policy_loss(*x.args(), one - 4, one, entropy_coef=0.1).grad_logits,
            policy.preference_loss(*x.args(), lines[:31], one - 4).grad_logits]
    calls = [lambda: policy.move_logprobs_backward(logits, *rest, grad_played=one, grad_logits=grad),
             lambda: policy.clipped_policy_loss(logits, *rest, one - 4, one, entropy_coef=0.1, grad_logits=grad),
             lambda: policy.preference_loss(logits, *rest, lines[:31], one - 4, grad_logits=grad)]
    for call, g in zip(calls, want):
        grad.fill_(7.0)
        call()
        assert torch.equal(grad, g)
        wide[:, 302 + gap:603 + gap] = 7.0
        assert torch.equal(wide, before)


def test_log_probabilities_of_lines_are_rounded_once():
    """Made in 64 bits (100 steps of 2^-52 between kernel and oracle, per unit of
    |s|, as where lines cancel) and rounded once: U |logp|. From 32-bit
    exponentials they would be off by some U whatever |logp| is. One rounding to nearest leans
    to neither side: errors of at most U |logp|, in the mean below a third of that
    rms, leave U rms(logp) / sqrt(3 n); five times that is allowed."""
    temp, n = 1.93, 1200
    x = Batch("f32", 1858, [int(k) for k in np.random.default_rng(5).integers(2, 60, n)], 29, temp)
    x.logits[:, :] *= 0.25  # log-probabilities of -0.2 to -5
    rows, logp, frozen, lines = line_case(x, [0, 800, n])
    out = policy.preference_loss(*x.args(), lines, x.f32(frozen), beta=0.1, softmax_temp=temp)
    off = out.logp.double().cpu().numpy() - logp
    tiny = 100 * 2.0 ** -52 * (1 + np.array([r.slack for r in rows]) / 8)
    assert np.all(np.abs(off) <= ref.U * np.abs(logp) + tiny)
    assert abs(off.mean()) <= 5 * ref.U * np.sqrt(np.mean(logp ** 2) / (3 * n))


@pytest.mark.parametrize("shift", [0.0, 3.0, 100.0, -65536.0])
@pytest.mark.parametrize("near_by", [1e-3, 0.3])
def test_kl_keeps_its_digits_at_any_offset(near_by, shift):
    """Each d = log p - log q is good to a few U of itself and of the two
    normalisations' difference, whose error is common to all d and cancels in sum p
    (e^-d - 1 + d) to first order; the terms are positive, so the KL's relative
    error is that of p, below slack U (policy_reference doubles it)."""
    x = Batch("f32", 1858, [40, 64, 90, 2] * 16, 48)
    _, other, old, adv, _ = clip_case(x, near_by=near_by)
    x.logits = x.logits + shift
    out = policy.clipped_policy_loss(*x.args(), x.f32(old), x.f32(adv), ref_logits=other, kl_coef=1.0)
    for b, (p, q) in enumerate(zip(x.rows(), x.rows(other))):
        # (from 64-bit differences of the logits: log p - log q loses half of the oracle's digits)
        d = (p.z - q.z) - (p.z.max() - q.z.max()) + (q.log_s - p.log_s)
        kl = np.sum(p.p * (np.expm1(-d) + d))
        near(out.kl[b].item(), kl, p.slack * ref.U * kl, f"kl {b}")
