"""mfb200_evaluate_logprobs and the device operator keep one rule for what
they are given, and the call leaves the caller's thread as it found it."""
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from metalfish_b200 import policy, synthetic  # noqa: E402
from metalfish_b200.netfile import PackedInputs  # noqa: E402
from metalfish_b200.network import create_network  # noqa: E402
from tests.conftest import GOLDEN  # noqa: E402

pytestmark = pytest.mark.gpu
B = 8


@pytest.fixture(scope="module")
def setup():
    p = np.load(os.path.join(GOLDEN, "positions.npz"))
    inp = PackedInputs(p["masks"][:B], p["values"][:B])
    net = create_network(synthetic.TINY, synthetic.generate(synthetic.TINY, 11, perturb_norms=True), max_batch=B)
    off = np.array([0, 20, 20, 50, 50, 120, 140, 141, 160], np.int32)  # positions 1 and 3 have no legal move
    idx = np.random.default_rng(1).integers(0, 1858, 160).astype(np.int16)
    yield net, inp, off, idx
    net.close()


def test_played_move_of_a_position_without_moves(setup):
    """It has none, whatever place from -1 up is given; below that the call is
    refused by the handle and the position NaN from the operator, empty or not."""
    net, inp, off, idx = setup
    played = np.array([3, 0, 29, 17, 5, -1, 0, 2], np.int32)
    none = played.copy()
    none[[1, 3]] = -1
    got, want = net.evaluate_logprobs(inp, off, idx, played), net.evaluate_logprobs(inp, off, idx, none)
    assert got[1][1] == 0 and got[1][3] == 0 and got[1][5] == 0
    for a, b in zip(got, want):
        np.testing.assert_array_equal(a, b)
    logits = torch.from_numpy(net.evaluate_packed(inp).policy).cuda()
    lists = torch.from_numpy(off).cuda(), torch.from_numpy(idx).cuda()
    out = policy.move_logprobs(logits, *lists, torch.from_numpy(played).cuda())
    np.testing.assert_array_equal(out.played.cpu().numpy(), got[1])
    for b in (0, 1):
        bad = played.copy()
        bad[b] = -2
        with pytest.raises(RuntimeError, match="played"):
            net.evaluate_logprobs(inp, off, idx, bad)
        out = policy.move_logprobs(logits, *lists, torch.from_numpy(bad).cuda())
        assert torch.isnan(out.played).nonzero().flatten().cpu().tolist() == [b]


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_the_callers_device_stays_current(setup):
    """A handle on two devices: each shard runs on a thread of its own."""
    _, inp, off, idx = setup
    pair = create_network(synthetic.TINY, synthetic.generate(synthetic.TINY, 11, perturb_norms=True), max_batch=B, num_devices=2)
    try:
        for device in (0, 1):
            torch.cuda.set_device(device)
            pair.evaluate_logprobs(inp, off, idx)
            assert torch.cuda.current_device() == device
    finally:
        torch.cuda.set_device(0)
        pair.close()
