"""The policy operators as they are used together: a network of this library
gives reference and behaviour log-probabilities and logits on the device, a
trainer's parameters give the policy's, and the losses' gradients train them."""
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from metalfish_b200 import policy, synthetic  # noqa: E402
from metalfish_b200.netfile import PackedInputs  # noqa: E402
from metalfish_b200.network import create_network  # noqa: E402
from tests import policy_reference as ref  # noqa: E402
from tests.conftest import GOLDEN  # noqa: E402

pytestmark = pytest.mark.gpu
B = 96


@pytest.fixture(scope="module")
def setup():
    p = np.load(os.path.join(GOLDEN, "positions.npz"))
    z = np.load(os.path.join(GOLDEN, "legal_moves.npz"))
    off = z["offsets"][40:40 + B + 1]  # does not start at 0
    idx = z["index"][off[0]:off[-1]]
    inp = PackedInputs(p["masks"][40:40 + B], p["values"][40:40 + B])
    net = create_network(synthetic.TINY, synthetic.generate(synthetic.TINY, 11, perturb_norms=True), max_batch=B)
    count = np.diff(off)
    rng = np.random.default_rng(3)
    played = np.array([rng.integers(0, min(n, 256)) if n else -1 for n in count], np.int32)
    played[5] = -1
    yield net, inp, off.astype(np.int32), idx, played
    net.close()


def device_logits(net, inp):
    """The frozen network's logits on the device, on torch's stream."""
    m = torch.from_numpy(inp.masks.view(np.int64)).cuda()
    v = torch.from_numpy(np.ascontiguousarray(inp.values, np.float32)).cuda()
    pol = torch.empty(B, 1858, device="cuda")
    wdl, mlh = torch.empty(B, 3, device="cuda"), torch.empty(B, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    net.evaluate_device(m.data_ptr(), v.data_ptr(), B, pol.data_ptr(), wdl.data_ptr(), mlh.data_ptr(), side.cuda_stream)
    torch.cuda.current_stream().wait_stream(side)
    return pol


@pytest.mark.parametrize("temp", [1.0, 0.61])
def test_evaluate_logprobs_is_the_softmax_of_the_logits(setup, temp):
    net, inp, off, idx, played = setup
    logp, at, ent, wdl, mlh = net.evaluate_logprobs(inp, off, idx, played, temp)
    out = net.evaluate_packed(inp)
    np.testing.assert_array_equal(wdl, out.wdl)
    np.testing.assert_array_equal(mlh, out.moves_left)
    for b in range(B):
        cols = idx[off[b] - off[0]:off[b + 1] - off[0]]
        row = ref.Row(out.policy[b], cols, float(np.float32(temp)))
        got = logp[off[b] - off[0]:off[b + 1] - off[0]]
        assert np.all(np.abs(got - row.logp) <= row.slack * ref.U * (1 + np.abs(row.logp)))
        want = row.logp[played[b]] if played[b] >= 0 else 0.0
        assert abs(at[b] - want) <= row.slack * ref.U * (1 + abs(want))
        assert abs(ent[b] - row.h) <= row.slack * ref.U * (1 + 2 * row.h)
    # the same bits through the device operator
    dev = policy.move_logprobs(device_logits(net, inp), torch.from_numpy(off).cuda(), torch.from_numpy(idx).cuda(),
                               torch.from_numpy(played).cuda(), softmax_temp=float(np.float32(temp)))
    np.testing.assert_array_equal(dev.moves.cpu().numpy(), logp)
    np.testing.assert_array_equal(dev.played.cpu().numpy(), at)
    np.testing.assert_array_equal(dev.entropy.cpu().numpy(), ent)


def test_evaluate_logprobs_without_played_and_its_refusals(setup):
    net, inp, off, idx, played = setup
    logp, at, ent, _, _ = net.evaluate_logprobs(inp, off, idx)
    assert at is None and np.isfinite(logp).all() and np.isfinite(ent).all()
    with pytest.raises(RuntimeError, match="softmax_temp"):
        net.evaluate_logprobs(inp, off, idx, played, 0.0)
    bad = played.copy()
    bad[3] = off[4] - off[3]
    with pytest.raises(RuntimeError, match="played"):
        net.evaluate_logprobs(inp, off, idx, bad)
    wrong = off.copy()
    wrong[3] = wrong[4] + 1
    with pytest.raises(RuntimeError, match="non-decreasing"):
        net.evaluate_logprobs(inp, wrong, idx, None)
    with pytest.raises(ValueError, match="move_offsets"):
        net.evaluate_logprobs(inp, off[:-1], idx)
    with pytest.raises(ValueError, match="move_index"):
        net.evaluate_logprobs(inp, off, idx[:-1])
    with pytest.raises(ValueError, match="played"):
        net.evaluate_logprobs(inp, off, idx, played[:-1])


def test_priors_are_unchanged_by_it(setup):
    """evaluate_priors shares buffers with evaluate_logprobs."""
    net, inp, off, idx, played = setup
    first = net.evaluate_priors(inp, off, idx, 1.0)
    net.evaluate_logprobs(inp, off, idx, played)
    again = net.evaluate_priors(inp, off, idx, 1.0)
    for a, b in zip(first, again):
        np.testing.assert_array_equal(a, b)


def test_a_tuning_step(setup):
    """A head on frozen features is tuned by each loss against the frozen
    network; the step through autograd equals the one by the formulas."""
    net, inp, off_h, idx_h, played_h = setup
    off, idx = torch.from_numpy(off_h).cuda(), torch.from_numpy(idx_h).cuda()
    played = torch.from_numpy(played_h).cuda()
    frozen = device_logits(net, inp)
    old = policy.move_logprobs(frozen, off, idx, played).played
    g = torch.Generator(device="cuda").manual_seed(4)
    feats = torch.randn(B, 32, generator=g, device="cuda")
    w = (0.05 * torch.randn(32, 1858, generator=g, device="cuda")).requires_grad_()
    adv = torch.randn(B, generator=g, device="cuda")
    lines = torch.arange(0, B + 1, 8, dtype=torch.int32, device="cuda")[:13]

    def steps(logits):
        clip = policy.clipped_policy_loss(logits, off, idx, played, old, adv, ref_logits=frozen, kl_coef=0.1, entropy_coef=0.01)
        pref = policy.preference_loss(logits, off, idx, played, lines, old, beta=0.3)
        visits = torch.full((len(idx_h),), -1.0 / B, device="cuda")
        return clip.grad_logits, pref.grad_logits, policy.move_logprobs_backward(logits, off, idx, grad_moves=visits)

    logits = frozen + feats @ w
    grads = steps(logits.detach())
    logits.backward(sum(grads))
    # the formulas, row by row in 64 bits
    host, frozen_h = logits.detach().cpu().numpy(), frozen.cpu().numpy()
    old_h, adv_h = old.cpu().numpy().astype(np.float64), adv.cpu().numpy()
    rows = [ref.Row(host[b], idx_h[off_h[b] - off_h[0]:off_h[b + 1] - off_h[0]], 1.0) for b in range(B)]
    want, off_by = np.zeros((B, 1858)), np.zeros((B, 1858))
    takes = [r.live and a >= 0 for r, a in zip(rows, played_h)]
    gain = np.array([r.logp[a] - o if t else 0.0 for r, a, o, t in zip(rows, played_h, old_h, takes)])
    sums = np.add.reduceat(gain, np.arange(0, B, 8))
    slope = np.repeat([s * v for i in range(6) for v in (1, -1)
                       for s in [ref.preference(sums[2 * i], sums[2 * i + 1], 0.3, 0.0, 1 / 6)[2]]], 8)
    for b, r in enumerate(rows):
        if not r.live:
            continue
        gm, mm = r.backward(np.full(len(r.p), -1.0 / B), 0.0, -1, 0.0)
        g_row, m_row = gm, mm
        if takes[b]:
            frozen_row = ref.Row(frozen_h[b], r.cols, 1.0)
            d = ref.clip_row(r, played_h[b], old_h[b], float(adv_h[b]), 1.0, frozen_row, 0.2, 0.2, 0.1, 0.01, 1.0 / B)
            gp, mp = r.backward(np.zeros(len(r.p)), slope[b], played_h[b], 0.0)
            # the margin's own error: 8 + 8 rows, each off by slack u (1 + |logp| + |old|) <= slack u 20
            g_row, m_row = gm + d["g"] + gp, mm + d["m"] + mp * (1 + 0.3 * 16 * 20)
        want[b] = r.dense(g_row, 1858)
        off_by[b] = r.dense(2 * r.slack * ref.U * m_row + 4 * ref.U * np.abs(g_row), 1858)
    got = sum(x.double() for x in grads).cpu().numpy()
    assert (np.abs(got - want) <= off_by).all()
    # autograd carries it to the parameters: feats^T grad, a product of B terms in fp32
    lhs = w.grad.double().cpu().numpy()
    f64 = feats.double().cpu().numpy()
    bound = np.abs(f64).T @ (off_by + B * 2 * ref.U * np.abs(want)) + 1e-12
    assert (np.abs(lhs - f64.T @ want) <= bound).all()


def test_a_step_captured_while_an_eager_graph_lives(setup):
    """The losses are captured and replayed while an eager autograd graph of
    the same parameters is alive."""
    net, inp, off_h, idx_h, played_h = setup
    off, idx, played = (torch.from_numpy(a).cuda() for a in (off_h, idx_h, played_h))
    frozen = device_logits(net, inp)
    old = policy.move_logprobs(frozen, off, idx, played).played
    adv = torch.ones(B, device="cuda")
    w = torch.zeros(B, 1858, device="cuda", requires_grad=True)
    eager = frozen + w  # an eager graph of the leaf, kept alive
    step = torch.cuda.Stream()
    step.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(step):
        policy.clipped_policy_loss(eager.detach(), off, idx, played, old, adv)
    torch.cuda.current_stream().wait_stream(step)
    logits = eager.detach().clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = policy.clipped_policy_loss(logits, off, idx, played, old, adv)
    graph.replay()
    eager.backward(out.grad_logits)
    torch.cuda.synchronize()
    want = policy.clipped_policy_loss(logits, off, idx, played, old, adv).grad_logits
    assert torch.equal(w.grad, want)


two = pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")


@two
def test_two_devices_shard_the_log_probabilities(setup):
    _, inp, off, idx, played = setup
    t = synthetic.generate(synthetic.TINY, 11, perturb_norms=True)
    pair = create_network(synthetic.TINY, t, max_batch=B, num_devices=2)
    one = create_network(synthetic.TINY, t, max_batch=B)
    try:
        got = pair.evaluate_logprobs(inp, off, idx, played)
        half = B // 2
        for lo, hi in ((0, half), (half, B)):
            want = one.evaluate_logprobs(PackedInputs(inp.masks[lo:hi], inp.values[lo:hi]), off[lo:hi + 1],
                                         idx[off[lo] - off[0]:off[hi] - off[0]], played[lo:hi])
            np.testing.assert_array_equal(got[0][off[lo] - off[0]:off[hi] - off[0]], want[0])
            for a, b in zip(got[1:], want[1:]):
                np.testing.assert_array_equal(a[lo:hi], b)
    finally:
        pair.close()
        one.close()


@two
def test_tensors_on_another_device_than_the_current_one(setup):
    _, _, off, idx, played = setup
    logits = torch.randn(B, 1858)
    args = [torch.from_numpy(a) for a in (off, idx, played)]
    want = policy.move_logprobs(logits.to("cuda:0"), *[a.to("cuda:0") for a in args])
    assert torch.cuda.current_device() == 0
    got = policy.move_logprobs(logits.to("cuda:1"), *[a.to("cuda:1") for a in args])
    assert torch.cuda.current_device() == 0 and got.moves.device.index == 1
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b.cpu())
    with pytest.raises(ValueError, match="cuda:0"):
        policy.move_logprobs(logits.to("cuda:1"), *[a.to("cuda:0") for a in args])
