"""The two 64-bit forms of the policy operators that the GPU tests use, row by
row (policy_reference) and over a batch (policy_plain64), against one another."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests import policy_reference as ref  # noqa: E402
from tests.policy_plain64 import Rows64, clip64, near  # noqa: E402


@pytest.mark.parametrize("temp", [1.0, 0.61])
@pytest.mark.parametrize("with_ref", [True, False])
def test_both_forms_agree(temp, with_ref):
    rng = np.random.default_rng(1)
    n, classes = 40, 50
    lists = [rng.choice(classes, k, replace=False) for k in rng.integers(0, 40, n)]
    logits, other = rng.standard_normal((2, n, classes)) * 2
    off = np.concatenate([[0], np.cumsum([len(c) for c in lists])]) + 7
    played = np.array([rng.integers(-1, len(c)) if len(c) else -1 for c in lists])
    t = torch.from_numpy
    index = t(np.concatenate(lists).astype(np.int16))
    big = Rows64(t(logits), t(off.astype(np.int32)), index, t(played.astype(np.int32)), temp)
    frozen = Rows64(t(other), t(off.astype(np.int32)), index, t(played.astype(np.int32)), temp)
    gm, ga, gh, old, adv, w = rng.standard_normal((6, max(n, len(index))))
    ga, gh, old, adv, w = ga[:n], gh[:n], old[:n] - 3, adv[:n], np.abs(w[:n])
    gm = gm[:len(index)]
    g, m = big.backward(t(gm), t(ga), t(gh))
    d = clip64(big, t(old), t(adv), t(w), frozen if with_ref else None, 0.2, 0.3, 0.1 * with_ref, 0.02, 0.5)
    for b in range(n):
        row, at = ref.Row(logits[b], lists[b], temp), slice(off[b] - 7, off[b + 1] - 7)
        a, k = int(played[b]), len(lists[b])
        if k == 0:
            assert big.h[b] == 0 and big.played_logp[b] == 0 and d["loss"][b] == 0
            continue
        np.testing.assert_allclose(big.logp[at], row.logp, rtol=1e-12, atol=1e-12)
        np.testing.assert_allclose([big.h[b], big.slack[b]], [row.h, row.slack], rtol=1e-12, atol=1e-12)
        want = row.backward(gm[at], ga[b] if a >= 0 else 0.0, a, gh[b])
        np.testing.assert_allclose(torch.stack([g, m])[:, at], np.stack(want), rtol=1e-10, atol=1e-12)
        if a < 0:
            assert d["loss"][b] == 0 and (d["g"][at] == 0).all()
            continue
        q = ref.Row(other[b], lists[b], temp)
        c = ref.clip_row(row, a, old[b], adv[b], w[b], q if with_ref else None, 0.2, 0.3, 0.1 * with_ref, 0.02, 0.5)
        for name in ("loss", "kl", "kl_off"):
            np.testing.assert_allclose(d[name][b], c[name], rtol=1e-9, atol=1e-14)
        np.testing.assert_allclose(d["loss_off"][b], c["loss_off"] + ref.U * abs(c["loss"]), rtol=1e-9, atol=1e-14)
        np.testing.assert_allclose(d["g"][at], c["g"], rtol=1e-9, atol=1e-12)
        np.testing.assert_allclose(d["m"][at], c["m"], rtol=1e-9, atol=1e-12)
        np.testing.assert_allclose(big.dense(g)[b], row.dense(want[0], classes), rtol=1e-10, atol=1e-12)


def test_near_finds_an_entry_that_was_not_written():
    v = torch.zeros(5, dtype=torch.float64)
    near(v, v, v)
    for bad in (12345.0, float("nan")):
        got = v.clone()
        got[3] = bad
        with pytest.raises(AssertionError):
            near(got, v, v + 1)
