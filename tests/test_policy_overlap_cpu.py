"""Which gradients overlap another matrix of their call (no GPU; the pointers
are never followed: a call that is not refused for them fails for its device)."""
import pytest

pytest.importorskip("torch")

from tests.test_policy_ops_cpu import A, backward, clip, prefer, refused, rows  # noqa: E402

WIDE = 4000  # elements between rows


def wide(**kw):
    return rows(logits_stride=WIDE, **kw)


@pytest.mark.parametrize("at", [1858, 1859, 2142, WIDE + 1858, 1858 - WIDE, 1858 - 3 * WIDE])
def test_gradient_in_other_columns_of_the_logits_buffer(at):
    for call in (backward, clip, prefer):
        refused(call(wide(), grad=A + 4 * at, stride=WIDE), "device")


@pytest.mark.parametrize("at", [0, 1, 1857, 2143, WIDE - 1, WIDE, WIDE + 1857, WIDE + 2143, -1, -WIDE, 1 - 1858,
                                3 * WIDE + 1857])
def test_gradient_in_columns_of_the_logits(at):
    for call in (backward, clip, prefer):
        refused(call(wide(), grad=A + 4 * at, stride=WIDE), "overlaps")


def test_other_pitches_and_one_row():
    for call in (backward, clip, prefer):
        refused(call(wide(), grad=A + 4 * 1858, stride=WIDE + 1), "overlaps")
        # 16-bit rows of the same pitch in bytes, and of the same stride in elements
        refused(call(wide(), grad=A + 4 * 1858, stride=2 * WIDE, kind=1), "device")
        refused(call(wide(), grad=A + 4 * 1858, stride=WIDE, kind=1), "overlaps")
        # a single row: what lies behind it is free whatever its stride
        refused(call(wide(batch=1), grad=A + 4 * 1858, stride=1858), "device")
        refused(call(wide(batch=1), grad=A + 4 * 1857, stride=1858), "overlaps")
        refused(call(wide(batch=1), grad=A + 4 * 1857, stride=WIDE), "overlaps")


def test_gradient_beside_the_reference():
    refused(clip(rows(), ref=40 * A, ref_stride=WIDE, grad=40 * A + 4 * 1858, stride=WIDE), "device")
    refused(clip(rows(), ref=40 * A, ref_stride=WIDE, grad=40 * A + 4 * 1857, stride=WIDE), "overlaps")
    # arrays between the gradient's rows are refused
    refused(clip(rows(), grad=64 * A, stride=WIDE, loss=64 * A + 4 * 1858), "overlaps")
