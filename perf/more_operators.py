"""Cases and plain forms of the operators around the training of adapters:

* ``logprobs``   -- log-probabilities of given tokens, and their gradient (``losses.token_logprobs``,
  ``losses.token_logprobs_backward``);
* ``policy``     -- the clipped policy loss with a KL term, and its gradient (``losses.policy_loss``);
* ``preference`` -- the preference loss of pairs of sequences, and its gradient (``losses.preference_loss``);
* ``clip``       -- norms of the adapters' gradients over many tensors, and their clipping
  (``adapters.clip_gradients``).

The vocabulary of 151936 and the widths 1536, 256 and 8960 are those of the decode step's model; 28 layers, ranks
16, 30 and 32 and the three experts are the adapters' own.
"""
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CLIP, KL, BETA = (0.2, 0.2), 0.04, 0.1
# (d_in, d_out) of the projections that have adapters
PROJECTIONS = {"attention": [(1536, 1536), (1536, 256)],
               "all": [(1536, 1536), (1536, 256), (1536, 256), (1536, 1536), (1536, 8960), (1536, 8960), (8960, 1536)]}


def listed():
    lp, po, pr, c = "logprobs", "policy", "preference", "clip"
    v = 151936
    return [
        # the next token of one request scored: latency is all there is
        dict(name="score_1", op=lp, sequences=1, tokens=1, vocab=v, dtype="bf16", packed=False, backward=False),
        # a batch scored under the reference model, prompts and padding left out
        dict(name="score_8x509", op=lp, sequences=8, tokens=509, vocab=v, dtype="bf16", packed=False, backward=False),
        # a supervised step on ragged sequences, an odd vocabulary, logits in 32 bits
        dict(name="sft_odd", op=lp, sequences=9, tokens=101, vocab=50257, dtype="fp32", packed=False, backward=True),
        # a step on the answers to one question, a few tokens each
        dict(name="policy_4x19", op=po, sequences=4, tokens=19, vocab=v, dtype="bf16", packed=False, reduction="token"),
        # a step on 16 answers of up to 384 tokens
        dict(name="policy_16x384", op=po, sequences=16, tokens=384, vocab=v, dtype="bf16", packed=False, reduction="token"),
        # the same in 32 bits on packed sequences, each with the same weight
        dict(name="policy_packed", op=po, sequences=13, tokens=77, vocab=v, dtype="fp32", packed=True, reduction="sequence"),
        # one pair of short answers
        dict(name="pair_1x23", op=pr, sequences=2, tokens=23, vocab=v, dtype="bf16", packed=False, kind="sigmoid", average=False),
        # eight pairs of up to 320 tokens
        dict(name="pairs_8x320", op=pr, sequences=16, tokens=320, vocab=v, dtype="bf16", packed=False, kind="sigmoid", average=False),
        # packed pairs over an odd vocabulary, averaged over their tokens
        dict(name="pairs_packed", op=pr, sequences=10, tokens=119, vocab=50257, dtype="fp16", packed=True, kind="squared", average=True),
        # the gradients of one layer, three adapters of an odd rank
        dict(name="clip_layer", op=c, layers=1, adapters=3, rank=30, projections="attention", dtype="fp16", each=True),
        # all layers of the decoder's adapters, each expert clipped by itself
        dict(name="clip_experts", op=c, layers=28, adapters=3, rank=16, projections="attention", dtype="bf16", each=True),
        # adapters on every projection in 32 bits under one norm
        dict(name="clip_all", op=c, layers=28, adapters=8, rank=32, projections="all", dtype="fp32", each=False),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["logprobs", "policy", "preference", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    size = 4 if dtype == "fp32" else 2
    if op == "clip":
        case = dict(op=op, layers=rng.randint(1, 28), adapters=_log(rng, 1, 32), rank=rng.choice([16, 30, 32, _log(rng, 1, 64)]),
                    projections=rng.choice(["attention", "all"]), dtype=dtype, each=rng.random() < 0.7)
        while _elements(case) * size > 10 ** 9:
            case["adapters"] = (case["adapters"] + 1) // 2
            case["layers"] = (case["layers"] + 1) // 2
        return case
    vocab = rng.choice([151936, 50257, _log(rng, 1000, 151936)])
    most = min(4096, 10 ** 9 // (vocab * size))
    sequences = _log(rng, 1, 32) if op != "preference" else 2 * _log(rng, 1, 16)
    case = dict(op=op, sequences=sequences, tokens=_log(rng, 1, max(1, most // sequences)), vocab=vocab, dtype=dtype, packed=rng.random() < 0.4)
    if op == "logprobs":
        case.update(packed=False, backward=rng.random() < 0.5)
    elif op == "policy":
        case.update(reduction=rng.choice(["token", "sequence", "sum"]))
    else:
        case.update(kind=rng.choice(["sigmoid", "sigmoid", "squared"]), average=rng.random() < 0.5)
    return case


# ---------------------------------------------------------------- inputs


def _lengths(case):
    """(length, prompt) of each sequence; the first one fills its row.  They belong to the case, whatever the seed."""
    s, t = case["sequences"], case["tokens"]
    rng = random.Random(s * 1000003 + t)
    lengths = [t] + [rng.randint((t + 2) // 3, t) for _ in range(s - 1)]
    return [(n, rng.randint(0, n // 2)) for n in lengths]


def _rows(case):
    """(rows of logits, rows that count); packed batches end with five rows that belong to no sequence."""
    lengths = _lengths(case)
    rows = sum(n for n, _ in lengths) + 5 if case["packed"] else case["sequences"] * case["tokens"]
    return rows, sum(n - p for n, p in lengths)


def _shapes(case):
    e, r = case["adapters"], case["rank"]
    return [shape for i, o in PROJECTIONS[case["projections"]] for shape in ((e, r, i), (e, o, r))]


def _elements(case):
    return case["layers"] * sum(math.prod(shape) for shape in _shapes(case))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    t = TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=dev) * std

    if case["op"] == "clip":
        e = case["adapters"]
        # norms from half to twice of what is allowed
        size = 2.0 ** (2 * torch.rand((e,), generator=g, device=dev) - 1)
        std = size * (_elements(case) / (e if case["each"] else 1)) ** -0.5
        if not case["each"]:
            std = std * 1.5
        buffers = [(normal(case["layers"], *shape) * std[:, None, None]).to(t) for shape in _shapes(case)]
        outs = [torch.empty_like(b) for b in buffers]
        per_layer = lambda many: [b[k] for k in range(case["layers"]) for b in many]  # noqa: E731
        return dict(case=case, buffers=buffers, outs=outs, grads=per_layer(buffers), into=per_layer(outs))

    s, v = case["sequences"], case["vocab"]
    lengths = _lengths(case)
    rows, _ = _rows(case)
    logits = torch.empty((rows, v), dtype=t, device=dev)
    logp = torch.empty((rows,), dtype=torch.float64, device=dev)
    targets = torch.randint(0, v, (rows,), generator=g, device=dev)
    top = math.log(v) + 3.0
    for k in range(0, rows, 1024):
        z = normal(min(1024, rows - k), v, std=2.5)
        y = targets[k:k + 1024, None]
        # a model's own tokens are likely ones
        z.scatter_(1, y, top + normal(z.shape[0], 1, std=2.0))
        logits[k:k + 1024] = z.to(t)
        z = logits[k:k + 1024].float()
        m = z.amax(1, keepdim=True)
        logp[k:k + 1024] = (z.gather(1, y) - m)[:, 0].double() - (z - m).exp_().sum(1).double().log()
    counts = torch.zeros((rows,), dtype=torch.bool, device=dev)
    at = 0
    for n, p in lengths:
        counts[at + p:at + n] = True
        at += n if case["packed"] else case["tokens"]
    targets[~counts] = -100
    if case["packed"]:
        starts = [0]
        for n, _ in lengths:
            starts.append(starts[-1] + n)
        shape = (rows,)
    else:
        starts, shape = None, (s, case["tokens"])
    state = dict(case=case, logits=logits.view(*shape, v), targets=targets.view(shape),
                 starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device=dev))
    if case["op"] == "logprobs":
        if case["backward"]:
            state["grad"] = normal(*shape, std=1.0 if t is torch.float16 else 1e-2)
    elif case["op"] == "policy":
        # the model has moved a little since the answers were sampled; no ratio lies on a border of the clipping
        moved = 0.15 * torch.randn((rows,), generator=g, device=dev, dtype=torch.float64)
        for border in (math.log(1 - CLIP[0]), math.log(1 + CLIP[1])):
            moved = torch.where((moved - border).abs() < 2e-3, border + 4e-3, moved)
        state["old"] = (logp - moved).float().view(shape)
        state["ref"] = (logp + 0.2 * normal(rows)).float().view(shape)
        state["advantages"] = normal(s)
        state["grad_scale"] = torch.full((), 64.0 if t is torch.float16 else 1.0, device=dev)
    else:
        # the model already leans to the chosen answers, the first half of the sequences
        chosen = torch.zeros((rows,), dtype=torch.float64, device=dev)
        chosen[:starts[s // 2] if case["packed"] else rows // 2] = 1.0
        state["ref"] = (logp + 0.03 - 0.1 * chosen + 0.05 * normal(rows)).float().view(shape)
        state["grad_scale"] = torch.full((), 64.0 if t is torch.float16 else 1.0, device=dev)
    return state


# ---------------------------------------------------------------- the operators


def _stats(s):
    """z - max, exp of it, the sum of that, the target or 0, whether it counts, the log-probability: of all rows."""
    z = s["logits"].reshape(-1, s["case"]["vocab"]).float()
    y = s["targets"].reshape(-1)
    counts = y >= 0
    y = y.clamp_min(0)
    z = z - z.amax(1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(1, keepdim=True)
    logp = z.gather(1, y[:, None])[:, 0].double() - total[:, 0].double().log()
    return e, total, y, counts, torch.where(counts, logp, 0.0)


def _gradient(s, g, e, total, y):
    """g_t ([v = y] - p_tv) in the logits' type and shape."""
    dz = e * (-g[:, None] / total)
    dz[torch.arange(y.numel(), device=y.device), y] += g
    return dz.to(s["logits"].dtype).view(s["logits"].shape)


def _member(s, counts):
    """[sequences, rows]: 1 where the row counts and belongs to the sequence."""
    n, c = counts.numel(), s["case"]
    at = torch.arange(n, device=counts.device)
    k = torch.arange(c["sequences"], device=counts.device)[:, None]
    if s["starts"] is None:
        inside = at // c["tokens"] == k
    else:
        inside = (at >= s["starts"][:-1, None]) & (at < s["starts"][1:, None])
    return (inside & counts).double()


def _logprobs(s):
    e, total, y, counts, logp = _stats(s)
    out = dict(logprobs=logp.float().view(s["targets"].shape))
    if "grad" in s:
        out["grad"] = _gradient(s, torch.where(counts, s["grad"].reshape(-1), 0.0), e, total, y)
    return out


def _policy(s):
    e, total, y, counts, logp = _stats(s)
    member = _member(s, counts)
    per = member.sum(1)
    if s["case"]["reduction"] == "token":
        w = member.sum(0) / per.sum().clamp_min(1)
    elif s["case"]["reduction"] == "sequence":
        w = (1 / (per.clamp_min(1) * per.numel())) @ member
    else:
        w = member.sum(0)
    a = s["advantages"].double() @ member
    ratio = torch.where(counts, torch.exp(logp - s["old"].reshape(-1).double()), 1.0)
    clipped = ratio.clamp(1 - CLIP[0], 1 + CLIP[1])
    d = torch.where(counts, s["ref"].reshape(-1).double() - logp, 0.0)
    # exp(d) - 1 - d by its series where that cancels
    k = torch.where(d.abs() < 1e-2, d * d * (0.5 + d * (1 / 6 + d * (1 / 24 + d / 120))), torch.exp(d) - 1 - d)
    loss = (w * (KL * k - torch.minimum(ratio * a, clipped * a))).sum()
    g = w * (KL * (1 - torch.exp(d)) - torch.where(ratio * a <= clipped * a, ratio * a, 0.0)) * s["grad_scale"].double()
    return dict(loss=loss.float(), logprobs=logp.float().view(s["targets"].shape), grad=_gradient(s, g.float(), e, total, y))


def _preference(s):
    e, total, y, counts, logp = _stats(s)
    member = _member(s, counts)
    if s["case"]["average"]:
        member = member / member.sum(1, keepdim=True).clamp_min(1)
    lead = member @ torch.where(counts, logp - s["ref"].reshape(-1).double(), 0.0)
    pairs = lead.numel() // 2
    d = lead[:pairs] - lead[pairs:]
    if s["case"]["kind"] == "sigmoid":
        loss = torch.log(1 + torch.exp(-BETA * d)).mean()
        slope = -BETA / (1 + torch.exp(BETA * d))
    else:
        loss = (d - 0.5 / BETA).square().mean()
        slope = 2 * (d - 0.5 / BETA)
    g = torch.cat([slope, -slope]) @ member / pairs * s["grad_scale"].double()
    return dict(loss=loss.float(), margins=(BETA * d).float(), logprobs=logp.float().view(s["targets"].shape),
                grad=_gradient(s, g.float(), e, total, y))


def _clip(s):
    each = s["case"]["each"]
    squares = [b.float().square().sum((0, 2, 3)).double() for b in s["buffers"]]
    squares = torch.stack(squares).sum(0)
    norms = (squares if each else squares.sum()).sqrt()
    factor = torch.where(norms > 1, 1 / norms, 1.0).float().expand(s["case"]["adapters"])
    return dict(norms=norms.float(), outs=[(b.float() * factor[:, None, None]).to(b.dtype) for b in s["buffers"]])


def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        from provenloop_b200 import adapters, losses
        if op == "logprobs":
            out = dict(logprobs=losses.token_logprobs(s["logits"], s["targets"]))
            if "grad" in s:
                out["grad"] = losses.token_logprobs_backward(s["grad"], s["logits"], s["targets"])
            return out
        if op == "policy":
            loss, logp, grad = losses.policy_loss(s["logits"], s["targets"], s["old"], s["advantages"], ref_logprobs=s["ref"],
                                                  starts=s["starts"], clip=CLIP, kl=KL, reduction=case["reduction"],
                                                  grad_scale=s["grad_scale"])
            return dict(loss=loss, logprobs=logp, grad=grad)
        if op == "preference":
            loss, margins, logp, grad = losses.preference_loss(s["logits"], s["targets"], s["ref"], starts=s["starts"], beta=BETA,
                                                               kind=case["kind"], average=case["average"], grad_scale=s["grad_scale"])
            return dict(loss=loss, margins=margins, logprobs=logp, grad=grad)
        norms = adapters.clip_gradients(s["grads"], 1.0, adapters=case["adapters"] if case["each"] else None, out=s["into"])
        return dict(norms=norms, outs=s["outs"])
    return {"logprobs": _logprobs, "policy": _policy, "preference": _preference, "clip": _clip}[op](s)


# ---------------------------------------------------------------- what is needed, and 64-bit values


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "clip":
        n = _elements(case)
        return {"bytes": 2 * n * size, "flops": 3 * n}
    rows, counted = _rows(case)
    v = case["vocab"]
    written = rows * v * size if case["op"] != "logprobs" or case["backward"] else 0
    small = {"logprobs": 16 if case.get("backward") else 12, "policy": 20, "preference": 16}[case["op"]]
    return {"bytes": counted * v * size + written + rows * small, "flops": counted * v * (7 if written else 4)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        wide = [b.double() for b in s["buffers"]]
        norms = torch.zeros((case["adapters"],), dtype=torch.float64, device=wide[0].device)
        for e in range(case["adapters"]):
            for b in wide:
                norms[e] += torch.linalg.vector_norm(b[:, e]) ** 2
        norms = norms.sqrt() if case["each"] else torch.linalg.vector_norm(norms.sqrt())
        for e in range(case["adapters"]):
            n = float(norms[e] if case["each"] else norms)
            for b in wide:
                b[:, e] /= max(n, 1.0)
        return dict(norms=norms, outs=wide)

    # log-probabilities and p, row block by row block
    v = case["vocab"]
    z = s["logits"].reshape(-1, v)
    y = s["targets"].reshape(-1)
    n = y.numel()
    used = (y >= 0).nonzero()[:, 0]
    logp = torch.zeros((n,), dtype=torch.float64, device=z.device)
    for part in used.split(256):
        logp[part] = torch.log_softmax(z[part].double(), 1).gather(1, y[part, None])[:, 0]

    def gradient(g):
        dz = torch.zeros((n, v), dtype=torch.float64, device=z.device)
        for part in used.split(256):
            p = torch.softmax(z[part].double(), 1)
            p.mul_(-g[part, None])
            p.scatter_add_(1, y[part, None], g[part, None])
            dz[part] = p
        return dz.view(s["logits"].shape)

    shaped = logp.view(s["targets"].shape)
    if case["op"] == "logprobs":
        out = dict(logprobs=shaped)
        if case["backward"]:
            out["grad"] = gradient(s["grad"].reshape(-1).double())
        return out

    # the rows of each sequence that count
    groups, at = [], 0
    for length, prompt in _lengths(case):
        groups.append(torch.arange(at + prompt, at + length, device=z.device))
        at += length if case["packed"] else case["tokens"]
    ref, g = s["ref"].reshape(-1).double(), torch.zeros_like(logp)
    scale = float(s["grad_scale"])
    loss = 0.0
    if case["op"] == "policy":
        old = s["old"].reshape(-1).double()
        for k, rows in enumerate(groups):
            if not len(rows):
                continue
            weight = {"token": 1 / len(used) if len(used) else 0.0, "sequence": 1 / (len(groups) * len(rows)), "sum": 1.0}[case["reduction"]]
            a = float(s["advantages"][k])
            l = logp[rows].clone().requires_grad_()
            rho = torch.exp(l - old[rows])
            gain = torch.minimum(rho * a, rho.clamp(1 - CLIP[0], 1 + CLIP[1]) * a)
            lead = ref[rows] - l
            part = (weight * (KL * (torch.expm1(lead) - lead) - gain)).sum()
            g[rows] = torch.autograd.grad(part, l)[0] * scale
            loss += float(part)
        return dict(loss=torch.tensor(loss, dtype=torch.float64), logprobs=shaped, grad=gradient(g))
    pairs, margins = len(groups) // 2, []
    for k in range(pairs):
        chosen, rejected = groups[k], groups[pairs + k]
        l = [logp[rows].clone().requires_grad_() for rows in (chosen, rejected)]
        sums = [(x - ref[rows]).sum() / (max(1, len(rows)) if case["average"] else 1) for x, rows in zip(l, (chosen, rejected))]
        d = sums[0] - sums[1]
        part = (torch.nn.functional.softplus(-BETA * d) if case["kind"] == "sigmoid" else (d - 1 / (2 * BETA)) ** 2) / pairs
        for rows, x in zip((chosen, rejected), torch.autograd.grad(part, l)):
            g[rows] = x * scale
        loss += float(part)
        margins.append(float(BETA * d))
    return dict(loss=torch.tensor(loss, dtype=torch.float64), margins=torch.tensor(margins, dtype=torch.float64), logprobs=shaped, grad=gradient(g))
