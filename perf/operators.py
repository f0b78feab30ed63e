"""Cases and plain forms of the decode-step operators beside the encrypted LoRA delta:

* ``project``  -- low-rank adapters of many requests beside a shared projection (``adapters.adapter_project``);
* ``backward`` -- its gradients for the input and the adapters (``adapters.adapter_project_backward``);
* ``rules``    -- penalties, biases and grammar masks on next-token logits, with the greedy pick
  (``logits.apply_rules``).

The widths 1536, 256 and 8960 and the vocabulary of 151936 are those of the decode step's model
(hidden, key/value, feed-forward); ranks 16, 30 and 32 and the three experts are the adapters' own.
"""
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    p, b, r = "project", "backward", "rules"
    return [
        # one request's next token through the query projection: latency is all there is
        dict(name="decode_1", op=p, n=1, d_in=1536, d_out=1536, rank=16, adapters=3, dtype="bf16", form="weight", runs=1),
        # 48 requests' next tokens, nearly every one with an adapter of its own, through the down projection
        dict(name="decode_48", op=p, n=48, d_in=8960, d_out=1536, rank=30, adapters=64, dtype="fp16", form="weight", runs=48),
        # a prefill batch of 23 prompts of ragged lengths through the gate projection
        dict(name="prefill_4099", op=p, n=4099, d_in=1536, d_out=8960, rank=32, adapters=8, dtype="bf16", form="weight", runs=23),
        # the adapters alone, added to a value projection that the model has already computed
        dict(name="added_2048", op=p, n=2048, d_in=1536, d_out=256, rank=16, adapters=3, dtype="bf16", form="base", runs=9),
        # adapters as they are loaded, in 32 bits, odd widths
        dict(name="single_precision", op=p, n=201, d_in=1001, d_out=771, rank=5, adapters=4, dtype="fp32", form="weight", runs=6),
        # a training step's micro-batch of the three experts on the query projection
        dict(name="train_8192", op=b, n=8192, d_in=1536, d_out=1536, rank=16, adapters=3, dtype="bf16", form="weight", runs=16),
        # a short ragged batch on the value projection, with a loss scale
        dict(name="train_517", op=b, n=517, d_in=1536, d_out=256, rank=30, adapters=5, dtype="fp16", form="weight", runs=11),
        # adapters trained beside a projection that is differentiated elsewhere
        dict(name="train_added", op=b, n=2048, d_in=8960, d_out=1536, rank=32, adapters=4, dtype="bf16", form="base", runs=7),
        # one request's next token after a long chat
        dict(name="rules_1", op=r, n=1, vocab=151936, history=4096, biases=16, dtype="bf16", mask=True, written=True),
        # a serving batch in which every rule is used, the logits in 32 bits
        dict(name="rules_64", op=r, n=64, vocab=151936, history=2048, biases=300, dtype="fp32", mask=True, written=True),
        # a large batch decoded greedily: only the picks are wanted
        dict(name="rules_256_pick", op=r, n=256, vocab=151936, history=1024, biases=8, dtype="bf16", mask=True, written=False),
        # an odd vocabulary, without a grammar
        dict(name="rules_odd", op=r, n=19, vocab=50257, history=777, biases=0, dtype="fp16", mask=False, written=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["project", "project", "backward", "rules"])
    if op == "rules":
        n, vocab = _log(rng, 1, 256), rng.choice([151936, _log(rng, 1000, 151936)])
        return dict(op=op, n=n, vocab=vocab, history=rng.choice([0, _log(rng, 1, 4096)]), biases=rng.choice([0, _log(rng, 1, 300)]),
                    dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), mask=rng.random() < 0.5, written=rng.random() < 0.75)
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    most = 1024 if dtype == "fp32" else 4096
    n = _log(rng, 1, most) if op == "project" else _log(rng, 64, most)
    d_in, d_out = rng.choice([(1536, 1536), (1536, 256), (1536, 8960), (8960, 1536), (_log(rng, 64, 4000), _log(rng, 64, 4000))])
    if dtype == "fp32":
        d_in, d_out = min(d_in, 1537), min(d_out, 1537)
    runs = rng.choice([n, max(1, n // 150)])
    return dict(op=op, n=n, d_in=d_in, d_out=d_out, rank=rng.choice([16, 16, 8, 30, 32, 64, _log(rng, 1, 64)]),
                adapters=_log(rng, 1, 64), dtype=dtype, form=rng.choice(["weight", "weight", "base"]), runs=runs)


# ---------------------------------------------------------------- inputs


def _ids(case, g, dev):
    """One adapter index per token: `runs` stretches of tokens (requests), each with an adapter or none (-1)."""
    n, runs = case["n"], case["runs"]
    which = torch.randint(0, case["adapters"] + 1, (runs,), generator=g, device=dev) - (1 if runs > 4 else 0)
    which = which.clamp_max(case["adapters"] - 1)
    if runs >= n:
        return which[:n].to(torch.int32)
    cuts = torch.randint(0, n, (runs - 1,), generator=g, device=dev).sort().values
    return which[torch.searchsorted(cuts, torch.arange(n, device=dev), right=True)].to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    t = TYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=dev) * std

    if case["op"] == "rules":
        n, v, h, b = case["n"], case["vocab"], case["history"], case["biases"]
        s = dict(case=case, logits=normal(n, v, std=3.0).to(t))
        if h:
            # token frequencies fall off as in text: a few ids make up most of a history
            u = torch.rand((n, h), generator=g, device=dev, dtype=torch.float64)
            s["tokens"] = (v ** u - 1).long().clamp_(0, v - 1) * 7919 % v
            s["lengths"] = torch.randint(0, h + 1, (n,), generator=g, device=dev, dtype=torch.int32) if n > 1 else \
                torch.full((n,), h, device=dev, dtype=torch.int32)
            s["prompt_lengths"] = (s["lengths"] * torch.rand((n,), generator=g, device=dev)).int()
            s["repetition"] = 1.0 + 0.3 * torch.rand((n,), generator=g, device=dev)
            s["frequency"] = 0.5 * torch.rand((n,), generator=g, device=dev)
            s["presence"] = 0.5 * torch.rand((n,), generator=g, device=dev)
        if b:
            s["bias_ids"] = torch.randint(-1, v, (n, b), generator=g, device=dev)
            s["bias_values"] = normal(n, b, std=4.0)
        if case["mask"]:
            # about one token in sixteen is allowed; in a batch the last row's grammar allows none
            w = [torch.randint(-2 ** 31, 2 ** 31, (n, (v + 31) // 32), generator=g, device=dev) for _ in range(4)]
            s["mask"] = (w[0] & w[1] & w[2] & w[3]).int()
            if n > 1:
                s["mask"][-1] = 0
        return s

    n, i, o, r, e = case["n"], case["d_in"], case["d_out"], case["rank"], case["adapters"]
    s = dict(case=case, x=normal(n, i).to(t), a=normal(e, r, i, std=i ** -0.5).to(t), b=normal(e, o, r, std=0.5 * r ** -0.5).to(t),
             ids=_ids(case, g, dev), scale=0.5 + torch.rand((e,), generator=g, device=dev))
    if case["form"] == "weight":
        s["w"] = normal(o, i, std=i ** -0.5).to(t)
    if case["op"] == "backward":
        s["dy"] = normal(n, o, std=1.0 if t is torch.float16 else 1e-2).to(t)
    elif case["form"] == "weight":
        s["bias"] = normal(o, std=0.1).to(t)
    else:
        s["base"] = normal(n, o).to(t)
    return s


# ---------------------------------------------------------------- the operators


def _low(x, a, s):
    """[n, adapters, rank]: scale_e x a_e^T at each token's own adapter, zero at the others."""
    e, r, _ = a.shape
    mine = torch.arange(e, device=x.device) == s["ids"][:, None]
    z = (x @ a.reshape(e * r, -1).T).view(-1, e, r)
    return torch.where(mine[:, :, None], z, 0.0) * s["scale"].to(z.dtype)[:, None]


def _project(s):
    x, a, b = s["x"].float(), s["a"].float(), s["b"].float()
    e, r, o = a.shape[0], a.shape[1], b.shape[1]
    y = _low(x, a, s).view(-1, e * r) @ b.transpose(1, 2).reshape(e * r, o)
    if "w" in s:
        y = y + x @ s["w"].float().T + s["bias"].float()
    else:
        y = y + s["base"].float()
    return y.to(s["x"].dtype)


def _backward(s):
    x, a, b, dy = s["x"].float(), s["a"].float(), s["b"].float(), s["dy"].float()
    e, r, i = a.shape
    o = b.shape[1]
    u = _low(dy, b.transpose(1, 2), s).view(-1, e * r)
    dx = u @ a.view(e * r, i)
    if "w" in s:
        dx = dx + dy @ s["w"].float()
    da = (u.T @ x).view(e, r, i)
    db = (_low(x, a, s).view(-1, e * r).T @ dy).view(e, r, o).transpose(1, 2)
    t = s["x"].dtype
    return [dx.to(t), da.to(t), db.contiguous().to(t)]


def _rules(s, dtype=torch.float32):
    z = s["logits"].to(dtype)
    n, v = z.shape
    at = torch.arange(v, device=z.device)
    if "tokens" in s:
        where = torch.arange(s["tokens"].shape[1], device=z.device)
        used = where < s["lengths"][:, None]
        said = used & (where >= s["prompt_lengths"][:, None])
        seen = torch.zeros((n, v), device=z.device, dtype=torch.int32).scatter_add_(1, s["tokens"], used.int()) > 0
        count = torch.zeros((n, v), device=z.device, dtype=torch.int32).scatter_add_(1, s["tokens"], said.int())
        rho, f, p = (s[k].to(dtype)[:, None] for k in ("repetition", "frequency", "presence"))
        z = torch.where(seen, torch.where(z > 0, z / rho, z * rho), z)
        z = torch.where(count > 0, z - f * count - p, z)
    if "bias_ids" in s:
        ids, k = s["bias_ids"], s["bias_ids"].shape[1]
        order = torch.arange(k, device=z.device).expand(n, k)
        last = torch.full((n, v + 1), -1, device=z.device)
        last.scatter_reduce_(1, torch.where(ids >= 0, ids, v), order, "amax")
        last = last[:, :v]
        z = torch.where(last >= 0, z + s["bias_values"].to(dtype).gather(1, last.clamp_min(0)), z)
    if "mask" in s:
        open_ = s["mask"][:, at // 32] >> (at % 32) & 1
        z = torch.where(open_ != 0, z, -torch.inf)
    top = z.amax(1, keepdim=True)
    pick = torch.where(z == top, at, v).amin(1)
    pick = torch.where(top[:, 0] == -torch.inf, -1, pick)
    return z, pick


def run(s):
    op = s["case"]["op"]
    if own:
        from provenloop_b200 import adapters, logits
        if op == "project":
            return adapters.adapter_project(s["x"], s["a"], s["b"], s["ids"], weight=s.get("w"), bias=s.get("bias"),
                                            base=s.get("base"), scale=s["scale"])
        if op == "backward":
            return adapters.adapter_project_backward(s["dy"], s["x"], s["a"], s["b"], s["ids"], weight=s.get("w"), scale=s["scale"])
        z, pick = logits.apply_rules(s["logits"], tokens=s.get("tokens"), lengths=s.get("lengths"),
                                     prompt_lengths=s.get("prompt_lengths"), repetition=s.get("repetition"),
                                     frequency=s.get("frequency"), presence=s.get("presence"), bias_ids=s.get("bias_ids"),
                                     bias_values=s.get("bias_values"), mask=s.get("mask"), write=s["case"]["written"])
        return dict(pick=pick, logits=z) if s["case"]["written"] else dict(pick=pick)
    if op == "project":
        return _project(s)
    if op == "backward":
        return _backward(s)
    z, pick = _rules(s)
    return dict(pick=pick, logits=z.to(s["logits"].dtype)) if s["case"]["written"] else dict(pick=pick)


# ---------------------------------------------------------------- what is needed, and 64-bit values


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    n = case["n"]
    if case["op"] == "rules":
        v = case["vocab"]
        per_row = v * size * (2 if case["written"] else 1) + case["history"] * 8 + case["biases"] * 12 + 28
        return {"bytes": n * (per_row + (v / 8 if case["mask"] else 0)), "flops": n * v}
    i, o, r = case["d_in"], case["d_out"], case["rank"]
    low = min(case["adapters"], n) * r * (i + o)
    w = i * o if case["form"] == "weight" else 0
    if case["op"] == "project":
        return {"bytes": size * (n * (i + o) + low + w + (0 if w else n * o)) + 4 * n, "flops": 2 * n * (w + r * (i + o))}
    return {"bytes": size * (n * (2 * i + o) + low + case["adapters"] * r * (i + o) + w) + 4 * n,
            "flops": 2 * n * (w + r * (3 * i + 2 * o))}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rules":
        z = s["logits"].double()
        n, v = z.shape
        for k in range(n):
            if "tokens" in s:
                m, p = int(s["lengths"][k]), int(s["prompt_lengths"][k])
                rho, f, pres = (s[q][k].double() for q in ("repetition", "frequency", "presence"))
                ids = s["tokens"][k, :m].unique()
                z[k, ids] = torch.where(z[k, ids] > 0, z[k, ids] / rho, z[k, ids] * rho)
                ids, times = s["tokens"][k, p:m].unique(return_counts=True)
                z[k, ids] -= f * times + pres
            if "bias_ids" in s:
                kept = {}
                for q, c in zip(s["bias_ids"][k].tolist(), s["bias_values"][k].tolist()):
                    kept[q] = c
                kept.pop(-1, None)
                if kept:
                    z[k, torch.tensor(list(kept), device=z.device)] += torch.tensor(list(kept.values()), device=z.device, dtype=z.dtype)
        if "mask" in s:
            bits = torch.stack([(s["mask"] >> q) & 1 for q in range(32)], -1).view(n, -1)[:, :v]
            z.masked_fill_(bits == 0, -torch.inf)
        return dict(pick=None, logits=z) if case["written"] else None
    x, a, b = s["x"].double(), s["a"].double(), s["b"].double()
    back = case["op"] == "backward"
    if back:
        dy = s["dy"].double()
        y = dy @ s["w"].double() if "w" in s else torch.zeros_like(x)
        da, db = torch.zeros_like(a), torch.zeros_like(b)
    else:
        y = x @ s["w"].double().T + s["bias"].double() if "w" in s else s["base"].double()
    for k in range(case["adapters"]):
        rows = (s["ids"] == k).nonzero()[:, 0]
        c = s["scale"][k].double()
        if back:
            u = c * (dy[rows] @ b[k])
            y[rows] += u @ a[k]
            da[k] = u.T @ x[rows]
            db[k] = c * (dy[rows].T @ (x[rows] @ a[k].T))
        else:
            y[rows] += c * ((x[rows] @ a[k].T) @ b[k].T)
    return [y, da, db] if back else y
