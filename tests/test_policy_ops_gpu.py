"""The policy operators on the GPU against their formulas in 64 bits
(tests/policy_reference.py, which derives the tolerances)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from metalfish_b200 import policy  # noqa: E402
from tests import policy_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# lengths at the edges of a warp's groups of 32, of the 256 that count, and beyond
LENGTHS = [0, 1, 2, 31, 32, 33, 64, 65, 255, 256, 257, 300]


class Batch:
    """Rows, lists and played moves; `lists` fixed by the caller or random."""

    def __init__(self, dtype, classes, lengths, seed, temp=1.0, start=0, shift=0, pad=0, lists=None, spread=2.0):
        rng = np.random.default_rng(seed)
        self.rng, self.dtype, self.classes, self.temp = rng, dtype, classes, temp
        self.lists = lists if lists is not None else [
            rng.choice(classes, n, replace=n > classes) for n in lengths]
        n = len(self.lists)
        self.n = n
        # rows start `shift` elements into a row and are `pad` elements longer: any alignment
        wide = torch.from_numpy(rng.standard_normal((n, classes + shift + pad)).astype(np.float32) * spread)
        self.wide = wide.to(TYPES[dtype]).cuda()
        self.logits = self.wide[:, shift:shift + classes]
        off = np.concatenate([[0], np.cumsum([len(x) for x in self.lists])]) + start
        self.off = torch.from_numpy(off.astype(np.int32)).cuda()
        flat = np.concatenate([np.asarray(x, np.int64) for x in self.lists]) if n else np.zeros(0)
        self.flat = flat.astype(np.int16)
        self.index = torch.from_numpy(self.flat).cuda()
        play = [int(rng.integers(-1, min(256, len(x)))) if len(x) else -1 for x in self.lists]
        self.played_host = np.asarray(play, np.int32)
        self.played = torch.from_numpy(self.played_host).cuda()

    def f32(self, a):
        return torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda()

    def rows(self, logits=None):
        host = (self.logits if logits is None else logits).float().cpu().numpy()
        return [ref.Row(host[b], self.lists[b], self.temp) for b in range(self.n)]

    def args(self):
        return self.logits, self.off, self.index, self.played


def near(got, want, off, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        bad = ~(same | (np.abs(got - want) <= off))
    assert not bad.any(), (what, got[bad][:4], want[bad][:4], np.broadcast_to(off, got.shape)[bad][:4])


def check_scores(x, out):
    moves = out.moves.cpu().numpy()
    at = 0
    for b, row in enumerate(x.rows()):
        n = len(x.lists[b])
        got = moves[at:at + n]
        lp = row.logp
        near(got[:256], lp, row.slack * ref.U * (1 + np.abs(np.where(np.isfinite(lp), lp, 0))), f"moves {b}")
        assert np.all(got[256:] == -np.inf)
        at += n
        a = int(x.played_host[b])
        takes = row.live and a >= 0
        want = row.logp[a] if takes else 0.0
        near(out.played[b].item(), want, row.slack * ref.U * (1 + abs(want)), f"played {b}")
        near(out.entropy[b].item(), row.h, row.slack * ref.U * (1 + 2 * row.h), f"entropy {b}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("classes,shift,pad,start,temp", [
    (1858, 0, 0, 0, 1.0), (1858, 1, 0, 17, 0.61), (1858, 3, 4, 0, 2.2), (4288, 0, 0, 0, 1.0),
    (32767, 5, 2, 3, 1.0), (301, 0, 3, 0, 1.3)])
def test_move_logprobs(dtype, classes, shift, pad, start, temp):
    x = Batch(dtype, classes, LENGTHS, 1, temp, start, shift, pad)
    check_scores(x, policy.move_logprobs(*x.args(), softmax_temp=temp))


@pytest.mark.parametrize("n", [1, 7, 148, 149, 1200, 5000])
def test_move_logprobs_batches(n):
    rng = np.random.default_rng(n)
    x = Batch("f32", 1858, rng.integers(0, 60, n), n)
    check_scores(x, policy.move_logprobs(*x.args()))
    out = policy.move_logprobs(x.logits, x.off, x.index)
    assert out.played is None


def dense(x, rows, per_row):
    """Expected gradient and its bound from per-row (g, m, slack)."""
    g, off = np.zeros((x.n, x.classes)), np.zeros((x.n, x.classes))
    for b, row in enumerate(rows):
        if per_row[b] is None:
            continue
        v, m, slack = per_row[b]
        g[b] = row.dense(v, x.classes)
        on = row.dense(np.ones(len(v)), x.classes) > 0
        off[b] = np.where(on, ref.grad_bound(g[b], row.dense(m, x.classes), slack, x.dtype), 0)
    return g, off


def check_backward(x, gm, ga, gh, grad):
    rows, per, at = x.rows(), [], 0
    for b, row in enumerate(rows):
        n = len(row.p)
        v = None
        if row.live:
            m = gm[at:at + n].astype(np.float64) if gm is not None else np.zeros(n)
            a = int(x.played_host[b])
            g, mag = row.backward(m, float(ga[b]) if ga is not None and a >= 0 else 0.0, a,
                                  float(gh[b]) if gh is not None else 0.0)
            v = g, mag, row.slack
        per.append(v)
        at += len(x.lists[b])
    want, off = dense(x, rows, per)
    near(grad.float().cpu().numpy(), want, off, "grad")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("classes,shift,pad,temp,parts", [
    (1858, 0, 0, 1.0, "mph"), (1858, 1, 0, 0.61, "m"), (1858, 3, 4, 2.2, "p"), (4288, 0, 0, 1.0, "h"),
    (32767, 5, 2, 1.0, "mph"), (301, 0, 3, 1.3, "mp"), (1858, 0, 0, 1.0, "")])
def test_move_logprobs_backward(dtype, classes, shift, pad, temp, parts):
    x = Batch(dtype, classes, LENGTHS, 2, temp, 5, shift, pad)
    gm = x.rng.standard_normal(len(x.flat)).astype(np.float32) if "m" in parts else None
    ga = x.rng.standard_normal(x.n).astype(np.float32) if "p" in parts else None
    gh = x.rng.standard_normal(x.n).astype(np.float32) if "h" in parts else None
    wide = torch.full((x.n, classes + shift + pad), 7.0, dtype=TYPES[dtype], device="cuda")
    grad = policy.move_logprobs_backward(
        *x.args(), grad_moves=None if gm is None else x.f32(gm), grad_played=None if ga is None else x.f32(ga),
        grad_entropy=None if gh is None else x.f32(gh), softmax_temp=temp,
        grad_logits=wide[:, shift:shift + classes])
    check_backward(x, gm, ga, gh, grad)
    # the elements between the rows are as they were
    assert (wide[:, :shift] == 7).all() and (wide[:, shift + classes:] == 7).all()


@pytest.mark.parametrize("kind", list(TYPES))
def test_gradient_in_another_type(kind):
    x = Batch("bf16", 1858, LENGTHS, 3)
    ga = x.rng.standard_normal(x.n).astype(np.float32)
    out = torch.empty(x.n, 1858, dtype=TYPES[kind], device="cuda")
    grad = policy.move_logprobs_backward(*x.args(), grad_played=x.f32(ga), grad_logits=out)
    x.dtype = kind
    check_backward(x, None, ga, None, grad)


def clip_case(x, with_ref=True, ref_dtype="f32", near_by=0.3):
    rows = x.rows()
    other = None
    if with_ref:
        other = (x.logits.float() + near_by * torch.from_numpy(
            x.rng.standard_normal((x.n, x.classes)).astype(np.float32)).cuda()).to(TYPES[ref_dtype])
    old = np.array([(r.logp[a] if a >= 0 and r.live and np.isfinite(r.logp[a]) else 0.0) + 0.2 * x.rng.standard_normal()
                    for r, a in zip(rows, x.played_host)], np.float32)
    adv = x.rng.standard_normal(x.n).astype(np.float32)
    w = x.rng.random(x.n).astype(np.float32)
    return rows, other, old, adv, w


def check_clip(x, out, rows, refs, old, adv, w, low, high, beta, eta, scale):
    per, total, total_off = [], 0.0, 0.0
    for b, row in enumerate(rows):
        a = int(x.played_host[b])
        near(out.entropy[b].item(), row.h, row.slack * ref.U * (1 + 2 * row.h), "entropy")
        if not row.live or a < 0:
            assert out.loss[b].item() == 0 and out.logp[b].item() == 0
            per.append(None)
            continue
        d = ref.clip_row(row, a, float(old[b]), float(adv[b]), float(w[b]), refs[b] if refs else None,
                         low, high, beta, eta, scale)
        near(out.loss[b].item(), d["loss"], d["loss_off"] + ref.U * abs(d["loss"]), f"loss {b}")
        near(out.logp[b].item(), row.logp[a], row.slack * ref.U * (1 + abs(row.logp[a])), "logp")
        if refs:
            near(out.kl[b].item(), d["kl"], d["kl_off"], "kl")
        total += d["loss"]
        total_off += d["loss_off"] + ref.U * abs(d["loss"])
        per.append((d["g"], d["m"], d["slack"]))
    near(out.total.item(), total, total_off + ref.U * abs(total), "total")
    want, off = dense(x, rows, per)
    near(out.grad_logits.float().cpu().numpy(), want, off, "grad")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("classes,shift,pad,temp,with_ref,ref_dtype,beta,eta", [
    (1858, 0, 0, 1.0, True, "f32", 0.05, 0.0), (1858, 1, 0, 0.61, True, "bf16", 0.3, 0.01),
    (1858, 3, 4, 2.2, False, "f32", 0.0, 0.02), (4288, 0, 0, 1.0, True, "f16", 0.05, 0.01),
    (32767, 5, 2, 1.0, True, "f32", 1.0, 0.0), (301, 0, 3, 1.3, False, "f32", 0.0, 0.0)])
def test_clipped_policy_loss(dtype, classes, shift, pad, temp, with_ref, ref_dtype, beta, eta):
    x = Batch(dtype, classes, LENGTHS * 3, 4, temp, 9, shift, pad)
    rows, other, old, adv, w = clip_case(x, with_ref, ref_dtype)
    scale = 64.0 / x.n
    out = policy.clipped_policy_loss(*x.args(), x.f32(old), x.f32(adv), ref_logits=other, weight=x.f32(w),
                                     clip_low=0.2, clip_high=0.3, kl_coef=beta, entropy_coef=eta, scale=scale,
                                     softmax_temp=temp)
    refs = x.rows(other) if with_ref else None
    check_clip(x, out, rows, refs, old, adv, w, 0.2, 0.3, beta, eta, scale)


@pytest.mark.parametrize("n", [1, 7, 148, 149, 1200, 5000])
def test_clipped_policy_loss_batches(n):
    rng = np.random.default_rng(n + 1)
    x = Batch("f32", 1858, rng.integers(0, 60, n), n + 1)
    rows, other, old, adv, w = clip_case(x)
    out = policy.clipped_policy_loss(*x.args(), x.f32(old), x.f32(adv), ref_logits=other, kl_coef=0.1)
    check_clip(x, out, rows, x.rows(other), old, adv, np.ones(n), 0.2, 0.2, 0.1, 0.0, 1.0 / n)


def test_near_policies_keep_their_kl():
    """KL of two policies 1e-3 apart is about 5e-7: 7 digits below its terms.
    Each difference d of the logits is exact to u |z| ~ 4 u, and enters as
    p d err(d), so the KL is good to about 8 u / 1e-3 relative; 2e-3 covers the rounding."""
    x = Batch("f32", 1858, [40] * 64, 5)
    x.played.clamp_(min=0)
    x.played_host = np.maximum(x.played_host, 0)
    _, other, old, adv, _ = clip_case(x, near_by=1e-3)
    out = policy.clipped_policy_loss(*x.args(), x.f32(old), x.f32(adv), ref_logits=other, kl_coef=1.0)
    for b, (row, q) in enumerate(zip(x.rows(), x.rows(other))):
        kl = np.sum(row.p * (row.logp - q.logp))
        assert abs(out.kl[b].item() - kl) <= 2e-3 * kl


def test_clip_border_is_decided_in_64_bits():
    """Ratios at and around the border: the gradient's jump follows the
    64-bit ratio of the given 32-bit numbers for every one of them."""
    n = 4000
    x = Batch("f32", 1858, [35] * n, 6)
    x.played.clamp_(min=0)
    x.played_host = np.maximum(x.played_host, 0)
    rows = x.rows()
    adv = np.where(np.arange(n) % 2 == 0, 1.0, -1.0).astype(np.float32)
    border = np.where(adv > 0, np.log1p(0.25), np.log1p(-0.25))
    old = np.array([r.logp[a] for r, a in zip(rows, x.played_host)]) - border
    old = old.astype(np.float32)  # within half a step of the border, on either side of it
    out = policy.clipped_policy_loss(*x.args(), x.f32(old), x.f32(adv), clip_low=0.25, clip_high=0.25, scale=1.0)
    got = out.grad_logits.abs().amax(1).cpu().numpy() > 0
    want = np.empty(n, bool)
    for b, r in enumerate(rows):
        ratio = np.exp(r.logp[x.played_host[b]] - float(old[b]))
        want[b] = not ratio > 1.25 if adv[b] > 0 else not ratio < 0.75
    assert 0.2 < want.mean() < 0.8
    np.testing.assert_array_equal(got, want)


def line_case(x, cuts):
    rows = x.rows()
    logp = np.array([r.logp[a] if a >= 0 and r.live else 0.0 for r, a in zip(rows, x.played_host)])
    frozen = (logp + 0.3 * x.rng.standard_normal(x.n)).astype(np.float32)
    return rows, logp, frozen, torch.from_numpy(np.asarray(cuts, np.int32)).cuda()


def check_preference(x, out, rows, logp, frozen, cuts, beta, eps, w, scale):
    takes = np.array([r.live and a >= 0 for r, a in zip(rows, x.played_host)])
    row_off = np.array([r.slack * ref.U for r in rows]) * (1 + np.abs(logp) + np.abs(frozen))
    per = [None] * x.n
    total = total_off = 0.0
    slopes = np.zeros(x.n)
    for i in range(len(cuts) // 2):
        gain, off, sums = [], 0.0, []
        for side in range(2):
            at = np.arange(cuts[2 * i + side], cuts[2 * i + side + 1])
            at = at[takes[at]]
            gain.append(np.sum(logp[at] - frozen[at].astype(np.float64)))
            sums.append(np.sum(logp[at]))
            off += beta * row_off[at].sum()
            near(out.line_logp[2 * i + side].item(), sums[-1], row_off[at].sum() + ref.U * abs(sums[-1]), "line")
        m, loss, slope = ref.preference(gain[0], gain[1], beta, eps, scale * w[i])
        off += 2 * ref.U * abs(m)
        near(out.margin[i].item(), m, off, "margin")
        loss_off = abs(scale * w[i]) * (off + 16 * ref.U * (1 + abs(m)))
        near(out.loss[i].item(), loss, loss_off, "loss")
        total += loss
        total_off += loss_off
        slope_off = abs(scale * w[i]) * beta * (off + 16 * ref.U)
        for side in range(2):
            for b in range(cuts[2 * i + side], cuts[2 * i + side + 1]):
                if not takes[b]:
                    continue
                ga = -slope if side else slope
                slopes[b] = ga
                g, mag = rows[b].backward(np.zeros(len(rows[b].p)), ga, int(x.played_host[b]), 0.0)
                # the slope's own error, relative to it, on top of the row's
                more = slope_off / max(abs(ga), 1e-30) / ref.U
                per[b] = g, mag, rows[b].slack + more
                near(out.row_grad[b].item(), ga, slope_off + ref.U * abs(ga), "row_grad")
    out_of = np.setdiff1d(np.arange(x.n), [b for b in range(x.n) if per[b] is not None])
    assert (out.row_grad[torch.from_numpy(out_of).cuda()] == 0).all()
    near(out.total.item(), total, total_off + ref.U * abs(total), "total")
    near(out.logp.cpu().numpy(), logp, row_off, "logp")
    want, off = dense(x, rows, per)
    near(out.grad_logits.float().cpu().numpy(), want, off, "grad")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("beta,eps,temp,shift,pad", [(0.1, 0.0, 1.0, 0, 0), (0.5, 0.1, 1.4, 1, 0), (2.0, 0.0, 1.0, 3, 4)])
def test_preference_loss(dtype, beta, eps, temp, shift, pad):
    """Lines of 0, 1, 32, 33 and 70 positions; positions before and behind the lines."""
    cuts = [3, 4, 4, 36, 69, 139, 140, 140, 140]
    x = Batch(dtype, 1858, [int(v) for v in np.random.default_rng(8).integers(0, 70, 150)], 8, temp, 2, shift, pad)
    rows, logp, frozen, lines = line_case(x, cuts)
    w = x.rng.random(4).astype(np.float32) + 0.5
    out = policy.preference_loss(*x.args(), lines, x.f32(frozen), beta=beta, label_smoothing=eps, weight=x.f32(w),
                                 scale=8.0, softmax_temp=temp)
    check_preference(x, out, rows, logp, frozen, cuts, beta, eps, w, 8.0)


def test_preference_margins_of_long_lines():
    """What leans to one side in a log-probability adds up over the 400 positions
    that one line is longer than the other. Each value: the exponentials 4 u
    and their arguments u |s|, weighted by p at most 4 u + 6 u, seven additions
    7 u, one rounding u |logp|. Their mean: errors of either sign, of 2 u (rms)
    at most, leave 2 u / sqrt(1200) = 0.06 u; 0.3 u is five times that."""
    temp = 1.93  # neither it nor its reciprocal is an fp32 number
    x = Batch("f32", 1858, [int(n) for n in np.random.default_rng(5).integers(2, 60, 1200)], 29, temp)
    rows, logp, frozen, lines = line_case(x, [0, 800, 1200])
    out = policy.preference_loss(*x.args(), lines, x.f32(frozen), beta=0.1, softmax_temp=temp)
    off = (out.logp.double().cpu().numpy() - logp) / ref.U
    assert np.all(np.abs(off) <= 17 + np.abs(logp))
    assert abs(off.mean()) <= 0.3
    check_preference(x, out, rows, logp, frozen, [0, 800, 1200], 0.1, 0.0, [1.0], 1.0)


@pytest.mark.parametrize("temp", [1.0, 1.93])
def test_preference_margins_of_lines_that_cancel(temp):
    """References that are the rounded log-probabilities themselves leave some
    1e-7 of each line. A row's log-probability is made in 64 bits (exponentials,
    logarithm, arguments below 20 and eight additions: 50 steps of 2^-52, and as
    many in the oracle) and its rest is rounded once, U |rest| <= U^2 |logp|."""
    x = Batch("f32", 1858, [31, 2, 64, 218, 1, 33, 20, 40, 7, 0, 65, 30], 31, temp)
    rows, logp, _, lines = line_case(x, [0, 6, 12])
    frozen = logp.astype(np.float32)
    out = policy.preference_loss(*x.args(), lines, x.f32(frozen), beta=1.0, softmax_temp=temp)
    gain = logp - frozen.astype(np.float64)
    margin = gain[:6].sum() - gain[6:].sum()
    off = np.sum(ref.U ** 2 * np.abs(logp) + 100 * 2.0 ** -52)
    assert abs(out.margin.item() - margin) <= off + ref.U * abs(margin)


@pytest.mark.parametrize("pairs,plies", [(1, 1), (300, 4), (2, 700), (1300, 1)])
def test_preference_loss_sizes(pairs, plies):
    rng = np.random.default_rng(pairs)
    lens = rng.integers(max(1, plies - 2), plies + 1, 2 * pairs)
    cuts = np.concatenate([[0], np.cumsum(lens)])
    x = Batch("f32", 1858, rng.integers(0, 50, cuts[-1]), pairs)
    rows, logp, frozen, lines = line_case(x, cuts)
    out = policy.preference_loss(*x.args(), lines, x.f32(frozen), beta=0.2)
    check_preference(x, out, rows, logp, frozen, cuts, 0.2, 0.0, np.ones(pairs), 1.0 / pairs)


# ---------------------------------------------------------------- where it can go wrong

def test_repeated_and_foreign_indices():
    """The same index twice and five times, across groups of 32, and indices
    outside the row (logit 0, no gradient)."""
    rng = np.random.default_rng(11)
    base = rng.choice(1858, 90, replace=False)
    lists = [[5, 5], [9, 7, 9, 9, 9, 9], list(base) + [base[0], base[40], base[0]], [-1, 3, 1858, 32767, 9],
             [-1, -1], list(base[:32]) + list(base[:32]), [1857, 0, 1857]]
    x = Batch("f32", 1858, None, 11, 1.0, 0, lists=lists)
    x.played_host = np.array([1, 3, 92, 0, 1, 40, 2], np.int32)
    x.played.copy_(torch.from_numpy(x.played_host))
    check_scores(x, policy.move_logprobs(*x.args()))
    gm, ga = x.rng.standard_normal(len(x.flat)).astype(np.float32), x.rng.standard_normal(7).astype(np.float32)
    grad = policy.move_logprobs_backward(*x.args(), grad_moves=x.f32(gm), grad_played=x.f32(ga))
    check_backward(x, gm, ga, None, grad)
    rows, other, old, adv, w = clip_case(x)
    out = policy.clipped_policy_loss(*x.args(), x.f32(old), x.f32(adv), ref_logits=other, weight=x.f32(w), kl_coef=0.1, entropy_coef=0.01)
    check_clip(x, out, rows, x.rows(other), old, adv, w, 0.2, 0.2, 0.1, 0.01, 1.0 / 7)


def test_lowest_values_infinities_and_masked_columns():
    """Listed logits of -inf and of the type's lowest value, all of them and
    some; NaN and infinities in columns that are not listed."""
    x = Batch("f32", 1858, [40] * 6, 12)
    x.played_host[:] = [0, 0, 0, 0, 0, 39]
    x.played.copy_(torch.from_numpy(x.played_host))
    low = torch.finfo(torch.float32).min
    host = torch.full((6, 1858), float("nan"), device="cuda")
    host[:, ::2] = float("inf")
    for b in range(6):
        at = torch.from_numpy(np.asarray(x.lists[b], np.int64)).cuda()
        v = x.logits[b, at].clone()
        if b == 0:
            v[:] = -np.inf
        if b == 1:
            v[:] = low
        if b == 2:
            v[1::2] = -np.inf
        if b == 3:
            v[1::2] = low
        if b == 4:
            v[0] = -np.inf  # the played move
        host[b, at] = v
    x.logits = host
    out = policy.move_logprobs(*x.args())
    check = x.rows()
    assert not check[0].live and check[1].live
    assert (out.moves[:40] == -np.inf).all() and out.played[0] == 0 and out.entropy[0] == 0
    moves = out.moves.cpu().numpy().reshape(6, 40)
    for b in (1, 2, 5):
        near(moves[b], check[b].logp, 200 * ref.U * 12, f"row {b}")
    near(moves[3][0::2], check[3].logp[0::2], 200 * ref.U * 12, "kept")
    assert (moves[3][1::2] < -1e38).all()
    assert out.played[4].item() == -np.inf
    assert np.isfinite(out.entropy.cpu().numpy()).all()
    ones = torch.ones(6, device="cuda")
    grad = policy.move_logprobs_backward(*x.args(), grad_played=ones, grad_entropy=ones)
    assert torch.isfinite(grad).all() and (grad[0] == 0).all()
    loss = policy.clipped_policy_loss(*x.args(), torch.zeros(6, device="cuda"), ones, entropy_coef=0.1)
    assert torch.isfinite(loss.grad_logits).all() and (loss.grad_logits[0] == 0).all()
    assert loss.loss[0] == 0 and torch.isfinite(loss.loss).all()


def test_nan_and_infinity_among_listed_logits_stay_in_their_row():
    x = Batch("f32", 1858, [40] * 4, 13)
    x.played_host[:] = 3
    x.played.fill_(3)
    x.logits[1, int(x.lists[1][7])] = float("nan")
    x.logits[2, int(x.lists[2][7])] = float("inf")
    out = policy.move_logprobs(*x.args())
    bad = torch.isnan(out.moves.reshape(4, 40)).any(1).cpu().tolist()
    assert bad == [False, True, True, False]
    assert torch.isnan(out.played).cpu().tolist() == bad
    zero, one = torch.zeros(4, device="cuda"), torch.ones(4, device="cuda")
    got = policy.clipped_policy_loss(*x.args(), zero - 3, one, entropy_coef=0.1)
    assert torch.isnan(got.loss).cpu().tolist() == bad
    assert torch.isnan(got.grad_logits).any(1).cpu().tolist() == bad
    lines = torch.arange(9, dtype=torch.int32, device="cuda").clamp(max=4)
    pref = policy.preference_loss(*x.args(), lines, zero - 3)
    assert torch.isnan(pref.logp).cpu().tolist() == bad
    assert torch.isnan(pref.margin).cpu().tolist() == [True, True, False, False]
    off = torch.ones(1858, dtype=torch.bool)
    off[torch.from_numpy(np.asarray(x.lists[1], np.int64))] = False
    assert (got.grad_logits[1].cpu()[off] == 0).all()


def test_reference_without_a_move_makes_the_kl_infinite():
    x = Batch("f32", 1858, [40] * 4, 27)
    x.played_host[:] = 3
    x.played.fill_(3)
    other = x.logits.clone()
    other[1, int(x.lists[1][9])] = -np.inf
    x.logits[2, int(x.lists[2][9])] = -np.inf  # the policy does not play it either: no term
    other[2, int(x.lists[2][9])] = -np.inf
    other[3, int(x.lists[3][9])] = float("nan")
    zero, one = torch.zeros(4, device="cuda"), torch.ones(4, device="cuda")
    out = policy.clipped_policy_loss(*x.args(), zero - 3, one, ref_logits=other, kl_coef=0.1)
    kl = out.kl.cpu().numpy()
    assert kl[0] == 0 and kl[1] == np.inf and abs(kl[2]) < 1e-6 and np.isnan(kl[3])
    assert np.isinf(out.loss[1].item())
    for b in (0, 2):
        assert torch.isfinite(out.grad_logits[b]).all() and torch.isfinite(out.loss[b])


@pytest.mark.parametrize("case", ["decreasing", "beyond", "before", "played high", "played low"])
def test_malformed_positions_are_nan_and_alone(case):
    """Lists that decrease or reach outside the indices, played moves that are
    not in the list: NaN for that position, nothing read past the list."""
    x = Batch("f32", 1858, [20, 20, 20, 20], 14)
    off, played = x.off.cpu().numpy().copy(), np.array([1, 2, 3, 4], np.int32)
    hit = [1]
    if case == "decreasing":
        off[2] = off[1] - 5
        hit = [1]
    elif case == "beyond":
        off[4] = 10 ** 9
        hit = [3]
    elif case == "before":
        off[2] = -7
        hit = [1, 2]
    else:
        played[1] = 20 if case == "played high" else -2
    x.off.copy_(torch.from_numpy(off))
    x.played.copy_(torch.from_numpy(played))
    zero, one = torch.zeros(4, device="cuda"), torch.ones(4, device="cuda")
    got = policy.clipped_policy_loss(*x.args(), zero - 3, one, ref_logits=x.logits.clone(), kl_coef=0.1)
    want = [b in hit for b in range(4)]
    for t in (got.loss, got.logp, got.kl, got.entropy):
        assert torch.isnan(t).cpu().tolist() == want
    assert torch.isnan(got.grad_logits).all(1).cpu().tolist() == want
    assert torch.isnan(got.grad_logits).any(1).cpu().tolist() == want
    score = policy.move_logprobs(*x.args())
    assert torch.isnan(score.played).cpu().tolist() == want
    grad = policy.move_logprobs_backward(*x.args(), grad_played=one)
    assert torch.isnan(grad).all(1).cpu().tolist() == want
    lines = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device="cuda")
    pref = policy.preference_loss(*x.args(), lines, zero - 3)
    assert torch.isnan(pref.loss).cpu().tolist() == [any(want[:2]), any(want[2:])]


@pytest.mark.parametrize("cuts", [[0, 2, 1, 3, 4], [-1, 2, 2, 3, 4], [0, 1, 2, 3, 5]])
def test_malformed_lines_are_nan(cuts):
    x = Batch("f32", 1858, [20] * 4, 15)
    lines = torch.tensor(cuts, dtype=torch.int32, device="cuda")
    out = policy.preference_loss(*x.args(), lines, torch.zeros(4, device="cuda"))
    bad = [cuts[0] < 0 or cuts[1] < cuts[0] or cuts[2] < cuts[1], cuts[3] < cuts[2] or cuts[4] > 4]
    assert torch.isnan(out.margin).cpu().tolist() == bad
    assert torch.isnan(out.loss).cpu().tolist() == bad
    assert torch.isfinite(out.grad_logits).all()


def test_lines_that_two_pairs_share():
    """Offsets that decrease between two pairs put positions into both: each
    pair's results are those of its own lines, whichever is worked on first."""
    x = Batch("f32", 1858, [20, 25, 0, 30], 18)
    frozen = torch.tensor([-3.0, -2.0, -5.0, -1.0], device="cuda")
    cuts = [0, 1, 4, 2, 1, 2, 4]  # (0, 1, 4) and (1, 2, 4) are in order, (4, 2, 1) is not
    out = policy.preference_loss(*x.args(), torch.tensor(cuts, dtype=torch.int32, device="cuda"), frozen)
    assert torch.isnan(out.loss).cpu().tolist() == [False, True, False]
    for i in (0, 2):
        own = torch.tensor(cuts[2 * i:2 * i + 3], dtype=torch.int32, device="cuda")
        one = policy.preference_loss(*x.args(), own, frozen)
        assert torch.equal(one.margin[0], out.margin[i])
        assert torch.equal(one.line_logp, out.line_logp[2 * i:2 * i + 2])
    assert torch.isfinite(out.grad_logits).all() and out.row_grad[2].item() == 0


def test_nothing_at_all():
    off = torch.zeros(1, dtype=torch.int32, device="cuda")
    idx, none = torch.zeros(0, dtype=torch.int16, device="cuda"), torch.zeros(0, device="cuda")
    logits, played = torch.zeros(0, 1858, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    assert policy.move_logprobs(logits, off, idx, played).moves.numel() == 0
    out = policy.clipped_policy_loss(logits, off, idx, played, none, none)
    assert out.total.item() == 0 and out.grad_logits.shape == (0, 1858)
    out = policy.preference_loss(logits, off, idx, played, off, none)
    assert out.total.item() == 0
    # positions without pairs, and pairs without positions (a margin of 0 each)
    x = Batch("f32", 1858, [20] * 3, 16)
    out = policy.preference_loss(*x.args(), off, torch.zeros(3, device="cuda"))
    assert out.total.item() == 0 and (out.grad_logits == 0).all() and (out.row_grad == 0).all()
    lines = torch.zeros(5, dtype=torch.int32, device="cuda")
    out = policy.preference_loss(logits, off, idx, played, lines, none)
    np.testing.assert_allclose(out.loss.cpu().numpy(), np.log(2) / 2, rtol=4 * ref.U)
    # only empty lists
    empty = torch.zeros(4, dtype=torch.int32, device="cuda")
    out = policy.clipped_policy_loss(x.logits, empty, idx, x.played, torch.zeros(3, device="cuda"), torch.ones(3, device="cuda"))
    assert out.total.item() == 0 and (out.grad_logits == 0).all()


def test_one_class():
    x = Batch("f16", 1, None, 17, lists=[[0], [], [0, 0], [0]])
    x.played_host[:] = [0, -1, 1, -1]
    x.played.copy_(torch.from_numpy(x.played_host))
    check_scores(x, policy.move_logprobs(*x.args()))
    ga = np.ones(4, np.float32)
    check_backward(x, None, ga, None, policy.move_logprobs_backward(*x.args(), grad_played=x.f32(ga)))


def test_rows_beyond_2_to_the_31_elements():
    """Three rows 1.2e9 elements apart: the last starts past 2^31."""
    stride = 1_200_000_007
    x = Batch("bf16", 1858, [30, 41, 50], 18)
    store = torch.empty(2 * stride + 1858, dtype=torch.bfloat16, device="cuda")
    far = store.as_strided((3, 1858), (stride, 1))
    far.copy_(x.logits)
    x.logits = far
    check_scores(x, policy.move_logprobs(*x.args()))
    out = torch.empty(2 * stride + 1858, dtype=torch.bfloat16, device="cuda").as_strided((3, 1858), (stride, 1))
    ga = np.ones(3, np.float32)
    check_backward(x, None, ga, None, policy.move_logprobs_backward(*x.args(), grad_played=x.f32(ga), grad_logits=out))


def test_python_checks():
    x = Batch("f32", 1858, [20] * 4, 19)
    z = torch.zeros(4, device="cuda")
    with pytest.raises(ValueError, match="move_offsets"):
        policy.move_logprobs(x.logits, x.off[:-1], x.index)
    with pytest.raises(ValueError, match="move_offsets"):
        policy.move_logprobs(x.logits, x.off.long(), x.index)
    with pytest.raises(ValueError, match="move_index"):
        policy.move_logprobs(x.logits, x.off, x.index.int())
    with pytest.raises(ValueError, match="move_index is on cpu"):
        policy.move_logprobs(x.logits, x.off, x.index.cpu())
    with pytest.raises(ValueError, match="contiguous"):
        policy.move_logprobs(x.logits, x.off, x.index[::2])
    with pytest.raises(ValueError, match="unit stride"):
        policy.move_logprobs(x.logits.t().contiguous().t(), x.off, x.index)
    with pytest.raises(ValueError, match="float32"):
        policy.move_logprobs(x.logits.double(), x.off, x.index)
    with pytest.raises(ValueError, match="played"):
        policy.clipped_policy_loss(x.logits, x.off, x.index, None, z, z)
    with pytest.raises(ValueError, match="played"):
        policy.move_logprobs_backward(x.logits, x.off, x.index, grad_played=z)
    with pytest.raises(ValueError, match="ref_logits"):
        policy.clipped_policy_loss(*x.args(), z, z, ref_logits=x.logits[:3])
    with pytest.raises(ValueError, match="grad_logits"):
        policy.clipped_policy_loss(*x.args(), z, z, grad_logits=x.logits[:3])
    with pytest.raises(ValueError, match="line_offsets"):
        policy.preference_loss(*x.args(), x.off[:4], z)
    with pytest.raises(RuntimeError, match="overlaps"):
        policy.clipped_policy_loss(*x.args(), z, z, grad_logits=x.logits)
    with pytest.raises(RuntimeError, match="softmax_temp"):
        policy.move_logprobs(*x.args(), softmax_temp=0.0)
    with pytest.raises(RuntimeError, match="stride"):
        policy.move_logprobs(x.logits[:1].expand(4, 1858), x.off, x.index)


def test_host_pointers_are_refused():
    L = policy._lib()
    host = np.zeros((2, 1858), np.float32)
    off = np.zeros(3, np.int32)
    rows = policy._Rows(host.ctypes.data, 1858, 0, 2, 1858, off.ctypes.data, None, 0, None, 1.0)
    torch.zeros(1, device="cuda")
    assert L.mfb200_move_logprobs(rows, None, None, host.ctypes.data, None) != 0
    assert b"device" in L.mfb200_policy_last_error()


def same(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b) if p is not None)


def test_results_do_not_depend_on_timing():
    rng = np.random.default_rng(20)
    x = Batch("f32", 1858, rng.integers(0, 60, 3000), 20)
    rows, other, old, adv, w = clip_case(x)
    lines = torch.arange(0, 3001, 100, dtype=torch.int32, device="cuda")
    lines = lines[:31]
    first = None
    for _ in range(5):
        a = policy.clipped_policy_loss(*x.args(), x.f32(old), x.f32(adv), ref_logits=other, kl_coef=0.1)
        b = policy.preference_loss(*x.args(), lines, x.f32(old))
        if first is None:
            first = a, b
        assert same(a, first[0]) and same(b, first[1])


def test_two_streams_at_once():
    """Two losses on two streams share nothing."""
    x, y = Batch("f32", 1858, [33] * 4000, 21), Batch("f32", 1858, [33] * 4000, 22)
    z = torch.zeros(4000, device="cuda") - 3
    one = torch.ones(4000, device="cuda")
    want = [policy.clipped_policy_loss(*b.args(), z, one, entropy_coef=0.1) for b in (x, y)]
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for k, b in enumerate((x, y)):
            with torch.cuda.stream(s[k]):
                got.append((k, policy.clipped_policy_loss(*b.args(), z, one, entropy_coef=0.1)))
    torch.cuda.synchronize()
    assert all(same(g, want[k]) for k, g in got)


def test_captured_and_replayed_with_new_inputs():
    """Two graphs, replayed in turn with inputs that change between replays."""
    a, b = Batch("bf16", 1858, [33] * 300, 23), Batch("bf16", 1858, [20] * 300, 24)
    lines = torch.arange(0, 301, 10, dtype=torch.int32, device="cuda")
    lines = lines[:31]
    z, one = torch.zeros(300, device="cuda") - 3, torch.ones(300, device="cuda")

    def step(x):
        return (policy.move_logprobs(*x.args()),
                policy.clipped_policy_loss(*x.args(), z, one, ref_logits=x.logits * 0.5, kl_coef=0.1),
                policy.preference_loss(*x.args(), lines, z))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a), step(b)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for x in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(x))
        graphs.append(g)
    for k in range(3):
        for x in (a, b):
            x.wide.copy_(torch.randn(x.wide.shape, device="cuda"))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, out in zip((a, b), outs):
            for got, want in zip(out, step(x)):
                assert same(got, want)


def test_the_calls_allocate_nothing():
    """Free device memory is the same after many calls into given buffers."""
    x = Batch("f32", 1858, [33] * 500, 28)
    z, one = torch.zeros(500, device="cuda") - 3, torch.ones(500, device="cuda")
    lines = torch.arange(0, 501, 10, dtype=torch.int32, device="cuda")
    grad = torch.empty(500, 1858, device="cuda")
    out = [torch.empty(500, device="cuda") for _ in range(6)]
    total, moves = torch.empty((), device="cuda"), torch.empty(len(x.flat), device="cuda")
    L = policy._lib()
    rows = policy._rows(*x.args(), 1.0)[0]
    p = [t.data_ptr() for t in out]

    def calls():
        assert L.mfb200_move_logprobs(rows, moves.data_ptr(), p[0], p[1], None) == 0
        assert L.mfb200_clipped_policy_loss(
            rows, policy._ClipConfig(0.2, 0.2, 0.0, 0.1, 1.0), z.data_ptr(), one.data_ptr(), None, None, 0, 0,
            p[0], p[1], None, p[2], total.data_ptr(), grad.data_ptr(), 1858, 0, None) == 0
        assert L.mfb200_preference_loss(
            rows, policy._PreferenceConfig(0.1, 0.0, 1.0), lines.data_ptr(), 25, z.data_ptr(), None, p[0], p[1],
            p[2], p[3], p[4], p[5], total.data_ptr(), grad.data_ptr(), 1858, 0, None) == 0

    calls()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(50):
        calls()
    torch.cuda.synchronize()
    assert torch.cuda.mem_get_info()[0] == free


# ---------------------------------------------------------------- gradients against differences

def test_gradients_against_differences():
    """Central differences of the 64-bit losses, step 1e-5 (their error: 1e-10
    of the loss's curvature, 1e-11 of its rounding / step), against the kernels'
    fp32 gradients: 2e-5 of the largest entry covers both."""
    x = Batch("f32", 40, [12, 12, 12, 12], 25, 1.3)
    x.played_host[:] = [3, 5, 0, 11]
    x.played.copy_(torch.from_numpy(x.played_host))
    rows, other, old, adv, w = clip_case(x)
    refs = x.rows(other)
    host = x.logits.cpu().numpy().astype(np.float64)
    cuts = [0, 1, 2, 3, 4]
    _, _, frozen, lines = line_case(x, cuts)

    def clip_loss(h):
        total = 0.0
        for b in range(4):
            r = ref.Row(h[b], x.lists[b], x.temp)
            total += ref.clip_row(r, int(x.played_host[b]), float(old[b]), float(adv[b]), float(w[b]), refs[b], 0.2, 0.2, 0.3, 0.05, 0.25)["loss"]
        return total

    def line_loss(h):
        lp = [ref.Row(h[b], x.lists[b], x.temp).logp[x.played_host[b]] - float(frozen[b]) for b in range(4)]
        return ref.preference(lp[0], lp[1], 0.7, 0.1, 0.5)[1] + ref.preference(lp[2], lp[3], 0.7, 0.1, 0.5)[1]

    got = [policy.clipped_policy_loss(*x.args(), x.f32(old), x.f32(adv), ref_logits=other, weight=x.f32(w), kl_coef=0.3, entropy_coef=0.05,
                                      softmax_temp=1.3).grad_logits,
           policy.preference_loss(*x.args(), lines, x.f32(frozen), beta=0.7, label_smoothing=0.1, softmax_temp=1.3).grad_logits]
    for loss, grad in zip((clip_loss, line_loss), got):
        diff = np.zeros((4, 40))
        for b in range(4):
            for c in range(40):
                up, down = host.copy(), host.copy()
                up[b, c] += 1e-5
                down[b, c] -= 1e-5
                diff[b, c] = (loss(up) - loss(down)) / 2e-5
        assert np.abs(grad.cpu().numpy() - diff).max() <= 2e-5 * np.abs(diff).max()
