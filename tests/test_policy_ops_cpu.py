"""Refusals of the policy operators: every check that needs no device memory
(no GPU; the pointers below are never followed)."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from metalfish_b200 import policy  # noqa: E402

A = 1 << 20  # an aligned address that nothing reads


def rows(**kw):
    d = dict(logits=A, logits_stride=1858, logits_type=0, batch=4, classes=1858, move_offsets=2 * A,
             move_index=3 * A, num_moves=100, played=4 * A, softmax_temp=1.0)
    d.update(kw)
    return policy._Rows(*[d[n] for n, _ in policy._Rows._fields_])


def refused(rc, text):
    got = policy._lib().mfb200_policy_last_error().decode()
    assert rc != 0 and text in got, got


G = 64 * A


def backward(r, gm=None, ga=5 * A, gh=None, grad=G, stride=1858, kind=0):
    return policy._lib().mfb200_move_logprobs_backward(r, gm, ga, gh, grad, stride, kind, None)


def clip(r, cfg=(0.2, 0.2, 0.0, 0.0, 1.0), old=5 * A, adv=6 * A, w=None, ref=None, ref_stride=1858,
         ref_kind=0, loss=7 * A, logp=None, kl=None, h=None, total=None, grad=G, stride=1858, kind=0):
    return policy._lib().mfb200_clipped_policy_loss(
        r, policy._ClipConfig(*cfg), old, adv, w, ref, ref_stride, ref_kind, loss, logp, kl, h, total,
        grad, stride, kind, None)


def prefer(r, cfg=(0.1, 0.0, 1.0), lines=5 * A, pairs=2, ref=6 * A, w=None, logp=7 * A, row_grad=8 * A,
           line_logp=9 * A, margin=10 * A, loss=11 * A, total=12 * A, rest=13 * A, grad=G, stride=1858,
           kind=0):
    return policy._lib().mfb200_preference_loss(
        r, policy._PreferenceConfig(*cfg), lines, pairs, ref, w, logp, rest, row_grad, line_logp,
        margin, loss, total, grad, stride, kind, None)


ROWS = [(dict(classes=0), "classes"), (dict(classes=32768, logits_stride=40000), "classes"),
        (dict(logits=None), "null logits"), (dict(logits_stride=1857), "stride"),
        (dict(logits_stride=1 << 60), "stride"), (dict(logits_type=3), "type"),
        (dict(logits_type=-1), "type"), (dict(logits=A + 2), "aligned"),
        (dict(logits=A + 1, logits_type=1), "aligned"), (dict(batch=-1), "negative"),
        (dict(move_offsets=None), "move_offsets"), (dict(move_offsets=A + 2), "aligned"),
        (dict(move_index=None), "move_index"), (dict(num_moves=-1), "num_moves"),
        (dict(num_moves=1 << 31), "num_moves"), (dict(played=4 * A + 1), "aligned"),
        (dict(softmax_temp=0.0), "softmax_temp"), (dict(softmax_temp=-1.0), "softmax_temp"),
        (dict(softmax_temp=float("nan")), "softmax_temp"),
        (dict(softmax_temp=float("inf")), "softmax_temp"), (dict(softmax_temp=1e-31), "softmax_temp")]


@pytest.mark.parametrize("bad,text", ROWS)
def test_rows_refused_by_every_call(bad, text):
    score = policy._lib().mfb200_move_logprobs(rows(**bad), A, A, A, None)
    refused(score, text)
    for call in (backward, clip, prefer):
        refused(call(rows(**bad)), text)


def test_null_structs():
    L = policy._lib()
    refused(L.mfb200_move_logprobs(None, A, A, A, None), "null rows")
    refused(L.mfb200_move_logprobs_backward(None, A, A, A, G, 1858, 0, None), "null rows")
    refused(L.mfb200_clipped_policy_loss(None, None, *[None] * 4, 0, 0, *[None] * 6, 0, 0, None), "null rows")
    refused(L.mfb200_preference_loss(None, None, None, 0, *[None] * 10, 0, 0, None), "null rows")


def test_move_logprobs_refusals():
    f = policy._lib().mfb200_move_logprobs
    refused(f(rows(), None, None, None, None), "no output")
    refused(f(rows(played=None), A, A, A, None), "played")
    refused(f(rows(), A + 1, None, None, None), "aligned")


OVERLAPS = [A, A + 4 * 1858 * 3, 2 * A, 3 * A, 4 * A]


@pytest.mark.parametrize("at", OVERLAPS)
def test_gradient_may_not_overlap_the_rows(at):
    for call in (backward, clip, prefer):
        refused(call(rows(), grad=at), "overlaps")


def test_gradient_matrix_refusals():
    for call in (backward, clip, prefer):
        refused(call(rows(), stride=1857), "stride")
        refused(call(rows(), kind=7), "type")
        refused(call(rows(), grad=G + 2), "aligned")
    refused(backward(rows(), grad=None), "null")
    refused(backward(rows(), gm=G), "overlaps")
    refused(backward(rows(), ga=G), "overlaps")
    refused(backward(rows(), gh=G + 1858 * 16 - 4), "overlaps")
    refused(backward(rows(), ga=A + 1), "aligned")
    refused(backward(rows(played=None)), "played")


def test_clipped_loss_refusals():
    refused(clip(rows(played=None)), "played")
    refused(clip(rows(), old=None), "old_logp")
    refused(clip(rows(), adv=None), "advantage")
    refused(clip(rows(), adv=A + 2), "aligned")
    for low, high in ((-0.1, 0.2), (1.1, 0.2), (0.2, -0.1), (float("nan"), 0.2), (0.2, float("nan")),
                      (0.2, float("inf"))):
        refused(clip(rows(), cfg=(low, high, 0.0, 0.0, 1.0)), "clip_low")
    for k in range(2, 5):
        cfg = [0.2, 0.2, 0.0, 0.0, 1.0]
        cfg[k] = float("inf")
        refused(clip(rows(), cfg=cfg, ref=20 * A), "finite")
    refused(clip(rows(), cfg=(0.2, 0.2, 0.1, 0.0, 1.0)), "reference")
    refused(clip(rows(), kl=13 * A), "reference")
    refused(clip(rows(), ref=20 * A, ref_stride=1), "stride")
    refused(clip(rows(), ref=20 * A, ref_kind=9), "type")
    refused(clip(rows(), ref=G), "overlaps")
    refused(clip(rows(), loss=None, total=13 * A), "total")
    refused(clip(rows(), loss=None, grad=None), "no output")
    refused(clip(rows(), loss=G + 8), "overlaps")


def test_preference_refusals():
    refused(prefer(rows(played=None)), "played")
    refused(prefer(rows(), pairs=-1), "negative")
    refused(prefer(rows(), pairs=1 << 30), "too many")
    for name in ("lines", "line_logp", "margin", "loss", "ref", "logp", "rest", "row_grad"):
        refused(prefer(rows(), **{name: None}), "null")
        refused(prefer(rows(), **{name: A + 2}), "aligned")
        refused(prefer(rows(), **{name: G}), "overlaps")
    for cfg in ((float("nan"), 0.0, 1.0), (0.1, 0.0, float("inf"))):
        refused(prefer(rows(), cfg=cfg), "finite")
    for eps in (-0.1, 1.1, float("nan")):
        refused(prefer(rows(), cfg=(0.1, eps, 1.0)), "label_smoothing")


def test_empty_batch_does_nothing():
    r = rows(batch=0, logits=None, move_offsets=None)
    assert policy._lib().mfb200_move_logprobs(r, None, None, None, None) == 0
    assert backward(r, grad=None) == 0
    assert clip(r, total=None) == 0
    assert prefer(r, pairs=0, total=None) == 0


def test_python_mirror_refuses_cpu_tensors():
    t = torch.zeros(2, 1858)
    off, idx = torch.zeros(3, dtype=torch.int32), torch.zeros(0, dtype=torch.int16)
    with pytest.raises(ValueError, match="CUDA"):
        policy.move_logprobs(t, off, idx)
    with pytest.raises(ValueError, match="2-D"):
        policy.move_logprobs(t[0], off, idx)


def test_without_a_device_the_call_fails_loudly():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    rc = policy._lib().mfb200_move_logprobs(rows(), A, A, A, None)
    refused(rc, "device")
    assert ctypes.sizeof(policy._Rows) == 72
