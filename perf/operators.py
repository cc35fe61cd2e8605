"""Cases of the policy operators: log-probabilities over the legal moves, the clipped policy loss
with its KL term, and the preference loss over lines of moves, with their gradients.

Every operator reads what ``evaluate_priors`` reads: a row of policy logits for each position and
the legal moves of each position as a CSR list of policy indices. Here each is written a second
time in elementary torch operations (``own = False``) and a third time from its definition in 64
bits (``exact``), so that the kernels of ``metalfish_b200.policy`` can be timed against the first
and checked against both.

Inputs are shaped as the engine's are: 31 +- 10 legal moves a position (the average of the 4096
playout positions of the test fixtures), a few queen endings with up to 218, about one position
in 110 with no legal move (mate, stalemate), and the indices of a position spread over the row in
small groups (a piece's moves lie next to each other in the 1858-move list).
"""
import math

import numpy as np
import torch

own = False

MOVES = 1858          # the engine's policy outputs
RAW = 64 * 64 + 8 * 24  # its raw attention logits, before the gather onto the 1858 moves
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LOSS_SCALE = {"f32": 1.0, "bf16": 1.0, "f16": 1024.0}  # half-precision gradients of a mean would vanish


def listed():
    return [
        # one position scored at the root of a search: latency
        dict(name="score 1", op="score", batch=1, classes=MOVES, dtype="f32", pad=0, temp=1.0),
        # a network batch of 1024 positions scored by the frozen network (fp32 logits)
        dict(name="score 1024", op="score", batch=1024, classes=MOVES, dtype="f32", pad=0, temp=1.0),
        # a shard of self-play games re-scored by a trainer under autocast, rows padded to a multiple of 64
        dict(name="score 50021 bf16", op="score", batch=50021, classes=MOVES, dtype="bf16", pad=62, temp=1.3),
        # cross-entropy to the search's visit counts on one search minibatch, raw attention logits
        dict(name="visits 37 raw", op="visits", batch=37, classes=RAW, dtype="f32", pad=0, temp=1.0),
        # the same on a training batch under autocast
        dict(name="visits 16384 bf16", op="visits", batch=16384, classes=MOVES, dtype="bf16", pad=0, temp=1.0),
        # a reinforcement step on one search minibatch: latency
        dict(name="clip 32", op="clip", batch=32, classes=MOVES, dtype="f32", pad=0, temp=1.0, ref=True, entropy=0.0),
        # a reinforcement step on the batch that the forward is quoted at
        dict(name="clip 1024", op="clip", batch=1024, classes=MOVES, dtype="f32", pad=0, temp=1.0, ref=True, entropy=0.01),
        # an odd batch in half precision with padded rows and no reference network
        dict(name="clip 9001 f16", op="clip", batch=9001, classes=MOVES, dtype="f16", pad=6, temp=1.0, ref=False, entropy=0.01),
        # the largest: a whole replay shard in fp32 against the frozen network
        dict(name="clip 65536", op="clip", batch=65536, classes=MOVES, dtype="f32", pad=0, temp=1.0, ref=True, entropy=0.0),
        # two candidate lines of a few plies: latency
        dict(name="prefer 1 pair", op="prefer", pairs=1, plies=6, classes=MOVES, dtype="f32", pad=0, temp=1.0, smoothing=0.0),
        # a batch of pairs of lines, 1 to 23 plies each
        dict(name="prefer 256 pairs", op="prefer", pairs=256, plies=12, classes=MOVES, dtype="f32", pad=0, temp=1.0, smoothing=0.0),
        # few pairs of whole games, 1 to 239 plies each, under autocast
        dict(name="prefer 96 games bf16", op="prefer", pairs=96, plies=120, classes=MOVES, dtype="bf16", pad=0, temp=1.2, smoothing=0.1),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    c = dict(op=rng.choice(["score", "visits", "clip", "prefer"]), classes=rng.choice([MOVES, MOVES, RAW]),
             dtype=rng.choice(["f32", "bf16", "f16"]), pad=rng.choice([0, 0, 2, 6, 62]), temp=round(rng.uniform(0.7, 2.0), 2))
    most = 60000 if c["classes"] == MOVES else 25000
    if c["op"] == "prefer":
        c["plies"] = spread(1, 150)
        c["pairs"] = spread(1, max(1, most // (2 * c["plies"] + 2)))
        c["smoothing"] = rng.choice([0.0, 0.05])
    else:
        c["batch"] = spread(1, most)
    if c["op"] == "clip":
        c["ref"] = rng.random() < 0.7
        c["entropy"] = rng.choice([0.0, 0.01])
    return c


# ---------------------------------------------------------------- inputs

def line_lengths(case):
    """Lengths of the 2 * pairs lines: 1 .. 2 * plies - 1 in equal shares."""
    k = np.arange(2 * case["pairs"])
    return 1 + (k * (2 * case["plies"] - 1)) // (2 * case["pairs"]) if case["pairs"] > 1 else np.array([case["plies"], max(1, case["plies"] - 1)])


def rows(case):
    return int(line_lengths(case).sum()) if case["op"] == "prefer" else case["batch"]


def move_counts(n):
    """Legal moves of n positions: the same for every seed, so that work() can count them."""
    b = torch.arange(n, dtype=torch.float64)
    c = torch.round(31 + 10 * math.sqrt(2) * torch.erfinv(2 * (b + 0.5) / n - 1)).long().clamp(1, 100)
    k = torch.arange(n)
    c[k % 200 == 150] = (60 + (k * 37) % 159)[k % 200 == 150]
    c[k % 110 == 109] = 0
    return c


def prepare(case, seed):
    dev = torch.device("cuda" if torch.cuda.is_available() else "cpu")
    g = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    n, w, t = rows(case), case["classes"], TYPES[case["dtype"]]
    counts = move_counts(n)[torch.randperm(n, generator=host)]
    offsets = torch.zeros(n + 1, dtype=torch.int32)
    offsets[1:] = counts.cumsum(0)
    total, widest = int(offsets[-1]), int(counts.max())
    counts, offsets = counts.to(dev), offsets.to(dev)

    # edge j of a position: groups of two, 5 columns apart, evenly over the row from a random start
    row = torch.repeat_interleave(torch.arange(n, device=dev), counts, output_size=total)
    j = torch.arange(total, device=dev) - offsets[:-1].long()[row]
    step = w // ((counts + 1) // 2).clamp(min=1)
    start = torch.randint(0, w, (n,), generator=g, device=dev)
    index = ((start[row] + (j // 2) * step[row] + 5 * (j % 2)) % w).to(torch.int16)

    wide = torch.empty(n, w + case["pad"], dtype=t, device=dev)
    wide.copy_(torch.randn(wide.shape, generator=g, device=dev) * 2)
    logits = wide[:, :w]
    s = dict(case=case, logits=logits, offsets=offsets, index=index, widest=max(1, widest))

    # what the frozen networks said: their logits are the policy's, some noise away
    live = counts > 0
    spot = padded(s)
    z = torch.where(spot["mask"], logits.gather(1, spot["cols"]).double(), -math.inf) / case["temp"]
    noise = torch.randn(z.shape, generator=g, device=dev)
    old = z + 0.15 * noise
    pick = (old - torch.log(-torch.log(torch.rand(z.shape, generator=g, device=dev, dtype=torch.float64)))).argmax(1)
    played = torch.where(live, pick, torch.zeros_like(pick))
    said = (old - old.logsumexp(1, keepdim=True)).gather(1, played[:, None])[:, 0]
    s["frozen"] = torch.where(live, said, torch.zeros_like(said)).float()
    # about one position in 50 is padding or the other side's move, one without legal moves has none
    idle = (torch.rand(n, generator=g, device=dev) < 0.02) | ~live
    if n == 1:
        idle &= ~live
    s["played"] = torch.where(idle, torch.full_like(played, -1), played).to(torch.int32)

    if case["op"] == "visits":
        share = torch.exp(z - z.logsumexp(1, keepdim=True)).nan_to_num(0.0)
        share = torch.where(spot["mask"], share + torch.rand(z.shape, generator=g, device=dev), 0.0)
        share = share / share.sum(1, keepdim=True).clamp(min=1e-9)
        by = LOSS_SCALE[case["dtype"]] / n
        s["grad_moves"] = (-share * by).float()[spot["mask"]].contiguous()
        s["grad_entropy"] = torch.full((n,), -0.01 * by, device=dev)
    if case["op"] == "clip":
        s["advantage"] = torch.randn(n, generator=g, device=dev)
        s["weight"] = torch.rand(n, generator=g, device=dev) * (torch.rand(n, generator=g, device=dev) > 0.05)
        if case["ref"]:
            s["ref"] = logits.float() + 0.3 * torch.randn(n, w, generator=g, device=dev)
    if case["op"] == "prefer":
        lens = torch.from_numpy(line_lengths(case))
        lens = lens[torch.randperm(len(lens), generator=host)] if case["pairs"] > 1 else lens
        lines = torch.zeros(2 * case["pairs"] + 1, dtype=torch.int32)
        lines[1:] = lens.cumsum(0)
        s["lines"] = lines.to(dev)
        s["weight"] = torch.rand(case["pairs"], generator=g, device=dev) + 0.5
    return s


# ---------------------------------------------------------------- the plain form

def padded(s):
    """The CSR lists as a [positions, widest] table of columns and its mask."""
    off = s["offsets"].long() - s["offsets"][:1].long()
    j = torch.arange(s["widest"], device=off.device)
    mask = j < (off[1:] - off[:-1])[:, None]
    at = torch.where(mask, off[:-1, None] + j, 0)
    cols = s["index"].long()[at] if s["index"].numel() else torch.zeros_like(at)
    return {"mask": mask, "at": at, "cols": torch.where(mask, cols, 0), "live": mask.any(1)}


def listed_again(s, table):
    """A [positions, widest] table's masked entries in the order of the CSR lists."""
    off = s["offsets"].long() - s["offsets"][:1].long()
    e = s["index"].numel()
    row = torch.repeat_interleave(torch.arange(len(off) - 1, device=off.device), off[1:] - off[:-1], output_size=e)
    return table[row, torch.arange(e, device=off.device) - off[row]]


def log_softmax(x, mask, live):
    """Over the masked entries of each row; 0 elsewhere and in rows that have none."""
    top = torch.where(live, torch.where(mask, x, -math.inf).amax(1), 0)[:, None]
    e = torch.where(mask, torch.exp(x - top), 0)
    lse = torch.log(torch.where(live, e.sum(1), 1))[:, None]
    return torch.where(mask, x - top - lse, 0)


def pick(table, played):
    return torch.where(played >= 0, table.gather(1, played.clamp(min=0).long()[:, None])[:, 0], 0)


def spread(s, spot, g):
    """The gradient of every edge in its place of an otherwise zero row."""
    grad = torch.zeros(s["logits"].shape, dtype=torch.float32, device=g.device)
    grad.scatter_add_(1, spot["cols"], torch.where(spot["mask"], g, 0))
    return grad.to(s["logits"].dtype)


def run(s):
    if own:
        return run_own(s)
    case, played = s["case"], s["played"]
    spot = padded(s)
    mask, live, t = spot["mask"], spot["live"], case["temp"]
    z = s["logits"].gather(1, spot["cols"])
    logp = log_softmax(z.float() / t, mask, live)
    p = torch.where(mask, torch.exp(logp), 0)
    entropy = -(p * logp).sum(1)
    at_played = (torch.arange(s["widest"], device=z.device) == played[:, None]).float()

    if case["op"] == "score":
        return {"moves": listed_again(s, logp), "played": pick(logp, played), "entropy": entropy}
    if case["op"] == "visits":
        gm = torch.where(mask, s["grad_moves"][spot["at"]], 0)
        gh = s["grad_entropy"][:, None]
        g = (gm - p * gm.sum(1, keepdim=True) - gh * p * (logp + entropy[:, None])) / t
        return {"moves": listed_again(s, logp), "entropy": entropy, "grad_logits": spread(s, spot, g)}
    if case["op"] == "clip":
        n = len(played)
        takes = (played >= 0) & live
        lp = pick(logp, played)
        exact_lp = pick(log_softmax(z.double() / t, mask, live), played)  # the clip's borders
        ratio, r64 = torch.exp(lp - s["frozen"]), torch.exp(exact_lp - s["frozen"].double())
        a = s["advantage"]
        active = torch.where(a > 0, r64 <= 1.2, r64 >= 0.8)
        loss = -torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a)
        g = torch.where(active, -a * ratio, 0)[:, None] * (at_played - p)
        kl = torch.zeros_like(loss)
        if "ref" in s:
            # near networks: the difference of two logarithms of nearly the same size
            far = log_softmax(s["ref"].gather(1, spot["cols"]).double() / t, mask, live)
            near = log_softmax(z.double() / t, mask, live)
            kl = torch.where(mask, torch.exp(near) * (near - far), 0).sum(1).float()
            delta = (near - far).float()
            loss = loss + 0.05 * kl
            g = g + 0.05 * p * (delta - kl[:, None])
        loss = loss - case["entropy"] * entropy
        g = g + case["entropy"] * p * (logp + entropy[:, None])
        scale = torch.where(takes, s["weight"] * (LOSS_SCALE[case["dtype"]] / n), 0)
        loss = torch.where(takes, scale * loss, 0)
        g = torch.where(takes[:, None], scale[:, None] * g / t, 0)
        out = {"total": loss.double().sum().float(), "loss": loss, "logp": lp, "entropy": entropy, "grad_logits": spread(s, spot, g)}
        return {**out, "kl": kl} if "ref" in s else out

    # prefer: beta 0.1, the scaled mean over the pairs
    pairs, beta, eps = case["pairs"], 0.1, case["smoothing"]
    takes = (played >= 0) & live
    lp = pick(logp, played)
    lines = s["lines"].long()
    line = torch.repeat_interleave(torch.arange(2 * pairs, device=lp.device), lines[1:] - lines[:-1], output_size=len(lp))
    line_logp = torch.zeros(2 * pairs, dtype=torch.float64, device=lp.device).index_add_(0, line, lp.double())
    gain = torch.zeros_like(line_logp).index_add_(0, line, torch.where(takes, lp.double() - s["frozen"].double(), 0))
    margin = (beta * (gain[0::2] - gain[1::2])).float()
    rest = torch.log1p(torch.exp(-margin.abs()))
    less, more = rest + (-margin).clamp(min=0), rest + margin.clamp(min=0)  # -log sigma(m), -log sigma(-m)
    scale = s["weight"] * (LOSS_SCALE[case["dtype"]] / pairs)
    loss = scale * ((1 - eps) * less + eps * more)
    slope = scale * beta * (eps * torch.sigmoid(margin) - (1 - eps) * torch.sigmoid(-margin))
    row_grad = torch.where(takes, torch.stack([slope, -slope], 1).reshape(-1)[line], 0)
    g = row_grad[:, None] * (at_played - p) / t
    return {"total": loss.double().sum().float(), "loss": loss, "margin": margin, "line_logp": line_logp.float(), "logp": lp,
            "grad_logits": spread(s, spot, g)}


def run_own(s):
    from metalfish_b200 import policy
    case = s["case"]
    lists = (s["logits"], s["offsets"], s["index"])
    if case["op"] == "score":
        out = policy.move_logprobs(*lists, s["played"], softmax_temp=case["temp"])
        return {"moves": out.moves, "played": out.played, "entropy": out.entropy}
    if case["op"] == "visits":
        out = policy.move_logprobs(*lists, softmax_temp=case["temp"])
        grad = policy.move_logprobs_backward(*lists, grad_moves=s["grad_moves"], grad_entropy=s["grad_entropy"], softmax_temp=case["temp"])
        return {"moves": out.moves, "entropy": out.entropy, "grad_logits": grad}
    if case["op"] == "clip":
        out = policy.clipped_policy_loss(*lists, s["played"], s["frozen"], s["advantage"], ref_logits=s.get("ref"), weight=s["weight"],
                                         clip_low=0.2, clip_high=0.2, kl_coef=0.05 if case["ref"] else 0.0, entropy_coef=case["entropy"],
                                         scale=LOSS_SCALE[case["dtype"]] / len(s["played"]), softmax_temp=case["temp"])
        got = {"total": out.total, "loss": out.loss, "logp": out.logp, "entropy": out.entropy, "grad_logits": out.grad_logits}
        return {**got, "kl": out.kl} if case["ref"] else got
    out = policy.preference_loss(*lists, s["played"], s["lines"], s["frozen"], beta=0.1, label_smoothing=case["smoothing"], weight=s["weight"],
                                 scale=LOSS_SCALE[case["dtype"]] / case["pairs"], softmax_temp=case["temp"])
    return {"total": out.total, "loss": out.loss, "margin": out.margin, "line_logp": out.line_logp, "logp": out.logp, "grad_logits": out.grad_logits}


# ---------------------------------------------------------------- work

def work(case):
    """Each legal move's logit (and the reference's), index and results once; the gradient rows whole."""
    n, w = rows(case), case["classes"]
    e = int(move_counts(n).sum())
    size = 4 if case["dtype"] == "f32" else 2
    lists = e * (size + 2) + 4 * (n + 1)
    grad = n * w * size
    if case["op"] == "score":
        return {"bytes": lists + 4 * n + 4 * e + 8 * n, "flops": 12 * e}
    if case["op"] == "visits":
        return {"bytes": lists + 4 * e + 4 * n + 4 * e + 4 * n + grad, "flops": 24 * e}
    if case["op"] == "clip":
        return {"bytes": lists + (4 * e if case["ref"] else 0) + 16 * n + 12 * n + (4 * n if case["ref"] else 0) + grad,
                "flops": (40 if case["ref"] else 24) * e}
    return {"bytes": lists + 8 * n + 4 * n + 32 * case["pairs"] + grad, "flops": 24 * e}


# ---------------------------------------------------------------- from the definition, in 64 bits

def exact(case, seed):
    """Flat over the CSR entries in 64 bits; the gradients by differentiating the definition."""
    s = prepare(case, seed)
    off = s["offsets"].long()
    n, k = len(off) - 1, off[1:] - off[:-1]
    row = torch.repeat_interleave(torch.arange(n, device=off.device), k)
    cols = s["index"].long()
    leaf = s["logits"].double()
    differentiate = case["op"] != "score"
    leaf.requires_grad_(differentiate)

    def over_rows(v):
        return torch.zeros(n, dtype=torch.float64, device=v.device).index_add(0, row, v)

    def normalised(table):
        u = table[row, cols] / case["temp"]
        return u - torch.log(over_rows(torch.exp(u)))[row]  # |u| stays below 30

    lp = normalised(leaf)
    entropy = -over_rows(torch.exp(lp) * lp)
    has = (s["played"] >= 0) & (k > 0)
    spot = (off[:-1] + s["played"].long())[has]
    of_played = torch.zeros(n, dtype=torch.float64, device=off.device).index_put((has.nonzero()[:, 0],), lp[spot])

    def slope(value):
        return torch.autograd.grad(value, leaf)[0]

    if case["op"] == "score":
        return {"moves": lp, "played": of_played, "entropy": entropy}
    if case["op"] == "visits":
        value = (s["grad_moves"].double() * lp).sum() + (s["grad_entropy"].double() * entropy).sum()
        return {"moves": lp.detach(), "entropy": entropy.detach(), "grad_logits": slope(value)}
    if case["op"] == "clip":
        r, a = torch.exp(of_played - s["frozen"].double()), s["advantage"].double()
        one = -torch.min(r * a, torch.clamp(r, 1 - 0.2, 1 + 0.2) * a) - case["entropy"] * entropy
        kl = None
        if case["ref"]:
            kl = over_rows(torch.exp(lp) * (lp - normalised(s["ref"].double())))
            one = one + 0.05 * kl
        loss = torch.where(has, one, torch.zeros_like(one)) * s["weight"].double() * LOSS_SCALE[case["dtype"]] / n
        got = {"total": loss.sum().detach(), "loss": loss.detach(), "logp": of_played.detach(), "entropy": entropy.detach(), "grad_logits": slope(loss.sum())}
        return {**got, "kl": kl.detach()} if case["ref"] else got
    lines = s["lines"].long()
    line = torch.bucketize(torch.arange(n, device=off.device), lines[1:], right=True)
    gain = torch.where(has, of_played - s["frozen"].double(), torch.zeros_like(of_played))
    sums = torch.zeros(2 * case["pairs"], dtype=torch.float64, device=off.device)
    line_logp, gains = sums.index_add(0, line, of_played), sums.index_add(0, line, gain)
    m = 0.1 * (gains[::2] - gains[1::2])
    eps = case["smoothing"]
    loss = -(1 - eps) * torch.nn.functional.logsigmoid(m) - eps * torch.nn.functional.logsigmoid(-m)
    loss = loss * s["weight"].double() * LOSS_SCALE[case["dtype"]] / case["pairs"]
    return {"total": loss.sum().detach(), "loss": loss.detach(), "margin": m.detach(), "line_logp": line_logp.detach(), "logp": of_played.detach(),
            "grad_logits": slope(loss.sum())}
