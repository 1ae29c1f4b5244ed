"""The operators of token policies, each as a case that can be timed: the embedding of tokens, the
gated linear recurrence over an episode, and the log probabilities of the actions taken.

``run`` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at
the end) or, where ``own`` is true, through pearl_amd's operators.  ``exact`` is the definition in
64 bits."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
LARGEST = 2 ** 27  # elements of the largest listed case


def listed():
    return [
        # the last actions of 64 environments, one row each
        {"name": "embed act", "op": "embed", "dtype": "fp32", "tokens": 64, "vocab": 16, "dim": 128, "train": False},
        # one training batch of token observations
        {"name": "embed train", "op": "embed", "dtype": "bf16", "tokens": 16384, "vocab": 32768, "dim": 1024, "train": True},
        # an odd table with few rows, each of them drawn many times
        {"name": "embed odd", "op": "embed", "dtype": "fp32", "tokens": 5003, "vocab": 1003, "dim": 333, "train": True},
        # one step of 256 episodes that are being acted in
        {"name": "recurrence step", "op": "step", "dtype": "bf16", "batch": 256, "dim": 1024, "gate": "logit"},
        # a training batch of histories that hold several episodes each
        {"name": "recurrence train", "op": "recurrence", "dtype": "bf16", "batch": 16, "time": 2048, "dim": 1024, "gate": "logit",
         "reverse": False, "resets": True, "lengths": False, "train": True},
        # one long history, read once to continue from its state
        {"name": "recurrence long", "op": "recurrence", "dtype": "bf16", "batch": 1, "time": 65536, "dim": 512, "gate": "logit",
         "reverse": False, "resets": False, "lengths": False, "train": False},
        # advantages of 4096 environments over 128 steps, backwards in time
        {"name": "recurrence advantages", "op": "recurrence", "dtype": "fp32", "batch": 1, "time": 128, "dim": 4096, "gate": "decay",
         "reverse": True, "resets": True, "lengths": False, "train": False},
        # a padded batch of odd sizes
        {"name": "recurrence padded", "op": "recurrence", "dtype": "fp16", "batch": 7, "time": 1001, "dim": 257, "gate": "logit",
         "reverse": False, "resets": False, "lengths": True, "train": True},
        # the policy heads of 64 environments, with the best alternatives to each action
        {"name": "log probs act", "op": "log_probs", "dtype": "fp32", "rows": 64, "actions": 16, "mask": True, "temperature": 1.0, "top": 4, "train": False},
        # a rollout of 65536 transitions with 16 actions
        {"name": "log probs rollout", "op": "log_probs", "dtype": "fp32", "rows": 65536, "actions": 16, "mask": True, "temperature": 1.0, "top": 0, "train": True},
        # a training batch of tokens over a large vocabulary
        {"name": "log probs train", "op": "log_probs", "dtype": "bf16", "rows": 4096, "actions": 32768, "mask": False, "temperature": 1.0, "top": 0, "train": True},
        # a few rows over a very large vocabulary, with 20 alternatives
        {"name": "log probs serve", "op": "log_probs", "dtype": "bf16", "rows": 16, "actions": 131072, "mask": False, "temperature": 0.7, "top": 20, "train": False},
    ]


def _size(rng, low, high):
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["embed", "step", "recurrence", "recurrence", "log_probs", "log_probs"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op == "embed":
        dim = _size(rng, 16, 2048)
        vocab = _size(rng, 16, min(131072, LARGEST // 2 // dim))
        return {"op": op, "dtype": dtype, "tokens": _size(rng, 1, min(65536, LARGEST // 2 // dim)), "vocab": vocab, "dim": dim,
                "train": rng.random() < 0.6}
    if op == "step":
        return {"op": op, "dtype": dtype, "batch": _size(rng, 1, 1024), "dim": _size(rng, 16, 4096), "gate": rng.choice(["logit", "decay"])}
    if op == "recurrence":
        dim = _size(rng, 16, 4096)
        time = _size(rng, 2, 65536)
        batch = _size(rng, 1, max(1, min(64, LARGEST // 4 // dim // time))) if dim * time <= LARGEST // 4 else 1
        if batch * dim * time > LARGEST // 4:
            time = LARGEST // 4 // dim
        return {"op": op, "dtype": dtype, "batch": batch, "time": time, "dim": dim, "gate": rng.choice(["logit", "logit", "decay"]),
                "reverse": rng.random() < 0.3, "resets": rng.random() < 0.5, "lengths": rng.random() < 0.3, "train": rng.random() < 0.6}
    actions = _size(rng, 2, 200000)
    train = rng.random() < 0.6
    return {"op": op, "dtype": dtype, "rows": _size(rng, 1, max(1, min(65536, LARGEST // 2 // actions))), "actions": actions,
            "mask": rng.random() < 0.5, "temperature": rng.choice([1.0, 1.0, 0.7, 1.3]),
            "top": 0 if train else rng.choice([0, 1, 5, 20, 50]), "train": train}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, kind=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(kind)

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    s = dict(case)
    if case["op"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        s["weight"] = normal(v, d, scale=0.02)
        # the k-th token of a vocabulary is drawn about 1/k as often as the first
        s["ids"] = (torch.exp(uniform(n) * math.log(v + 1)).long() - 1).clamp(0, v - 1)
        s["scale"] = math.sqrt(d)
        if case["train"]:
            s["d_out"] = normal(n, d)
        return s
    if case["op"] == "log_probs":
        r, a = case["rows"], case["actions"]
        s["logits"] = normal(r, a, scale=2.0)
        s["taken"] = (uniform(r) * a).long().clamp(0, a - 1)
        s["unavailable"] = None
        if case["mask"]:
            s["unavailable"] = uniform(r, a) < 0.25
            s["unavailable"].scatter_(1, s["taken"][:, None], False)
        if case["train"]:
            s["d_log_prob"], s["d_entropy"] = normal(r, kind=torch.float32), normal(r, kind=torch.float32, scale=0.01)
        return s
    b, t, d = case["batch"], case.get("time", 1), case["dim"]
    s["x"] = normal(b, t, d)
    if case["gate"] == "logit":
        s["g"] = (torch.randn(b, t, d, generator=gen, device="cuda") + 3.0).to(dtype)  # memories of about twenty steps
    else:
        s["g"] = (0.9 + 0.0999 * uniform(b, t, d)).to(dtype)
    s["h0"] = normal(b, d, kind=torch.float32)
    if case["op"] == "step":
        s["x"], s["g"] = s["x"][:, 0], s["g"][:, 0]
        return s
    s["starts"] = uniform(b, t) < 1.0 / 128 if case["resets"] else None
    s["ends"] = (uniform(b) * (t + 1)).int() if case["lengths"] else None
    if case["train"]:
        s["d_h"], s["d_last"] = normal(b, t, d), normal(b, d, kind=torch.float32)
    return s


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"embed": _plain_embed, "step": _plain_step, "recurrence": _plain_recurrence, "log_probs": _plain_log_probs}[state["op"]](state)


def _own(s):
    """The calls of a learner, which runs its backward pass explicitly as the framework's own learners do."""
    import pearl_amd
    if s["op"] == "embed":
        out = pearl_amd.embed_tokens(s["weight"], s["ids"], scale=s["scale"])
        if not s["train"]:
            return {"out": out}
        return {"out": out, "d_weight": pearl_amd.embed_tokens_grad(s["d_out"], s["ids"], s["vocab"], scale=s["scale"])}
    logit = s.get("gate") == "logit"
    if s["op"] == "step":
        h, last = pearl_amd.gated_recurrence_step(s["x"], s["g"], s["h0"], gate_logits=logit)
        return {"h": h, "last": last}
    if s["op"] == "recurrence":
        how = {"resets": s["starts"], "lengths": s["ends"], "gate_logits": logit, "reverse": s["reverse"]}
        if not s["train"]:
            h, last = pearl_amd.gated_recurrence(s["x"], s["g"], s["h0"], **how)
            return {"h": h, "last": last}
        h, last, kept = pearl_amd.gated_recurrence(s["x"], s["g"], s["h0"], keep=True, **how)
        dx, dg, d0 = pearl_amd.gated_recurrence_grad(s["x"], s["g"], kept, s["d_h"], s["d_last"], **how)
        return {"h": h, "last": last, "d_x": dx, "d_g": dg, "d_h0": d0}
    o = pearl_amd.action_log_probs(s["logits"], s["taken"], s["unavailable"], temperature=s["temperature"], top=s["top"])
    out = {"log_prob": o.log_prob, "entropy": o.entropy}
    if s["train"]:
        out["d_logits"] = pearl_amd.action_log_probs_grad(o, s["logits"], s["taken"], s["d_log_prob"], s["d_entropy"],
                                                          s["unavailable"], temperature=s["temperature"])
    if s["top"]:
        out.update({"top": o.top_actions, "top_log_prob": o.top_log_probs})
    return out


def _plain_embed(s):
    w, ids, scale = s["weight"], s["ids"], s["scale"]
    out = (w[ids].float() * scale).to(w.dtype)
    if not s["train"]:
        return {"out": out}
    d_weight = torch.zeros(w.shape, dtype=torch.float32, device=w.device).index_add_(0, ids, s["d_out"].float())
    return {"out": out, "d_weight": (d_weight * scale).to(w.dtype)}


def _plain_gate(s):
    """The factor of the state before, that of the input, in 32 bits."""
    g = s["g"].float()
    if s["gate"] == "logit":
        return 1.0 / (1.0 + torch.exp(-g)), 1.0 / (1.0 + torch.exp(g))
    return g, torch.ones_like(g)


def _plain_step(s):
    a, keep = _plain_gate(s)
    h = a * s["h0"] + keep * s["x"].float()
    return {"h": h.to(s["x"].dtype), "last": h}


def _scan(a, b):
    """h[t] = a[t] h[t - 1] + b[t] along dimension 1, by doubling the steps that a pair spans."""
    n = 1
    while n < a.shape[1]:
        b = torch.cat((b[:, :n], b[:, n:] + a[:, n:] * b[:, :-n]), 1)
        a = torch.cat((a[:, :n], a[:, n:] * a[:, :-n]), 1)
        n *= 2
    return b


def _turned(v, order):
    return v if order is None else torch.gather(v, 1, order.view(order.shape + (1,) * (v.dim() - 2)).expand(v.shape))


def _plain_recurrence(s):
    x, (a, keep), h0 = s["x"].float(), _plain_gate(s), s["h0"]
    b, t, d = x.shape
    step = torch.arange(t, device=x.device).expand(b, t)
    ends = torch.full((b, 1), t, device=x.device) if s["ends"] is None else s["ends"].long()[:, None]
    valid = step < ends
    # a reversed history is read from its last step; steps behind the end stay where they are
    order = torch.where(valid, ends - 1 - step, step) if s["reverse"] else None
    x, a, keep = _turned(x, order), _turned(a, order), _turned(keep, order)
    forget = torch.zeros_like(valid) if s["starts"] is None else _turned(s["starts"], order)
    behind = ~valid[:, :, None]
    decay = torch.where(behind, 1.0, torch.where(forget[:, :, None], 0.0, a))
    into = torch.where(behind, 0.0, keep * x)
    into = torch.cat((into[:, :1] + decay[:, :1] * h0[:, None], into[:, 1:]), 1)
    h = _scan(decay, into)
    out = {"h": _turned(torch.where(behind, 0.0, h), order).to(s["x"].dtype), "last": h[:, -1]}
    if not s["train"]:
        return out
    d_h = torch.where(behind, 0.0, _turned(s["d_h"].float(), order))
    d_h = torch.cat((d_h[:, :-1], d_h[:, -1:] + s["d_last"][:, None]), 1)
    after = torch.cat((decay[:, 1:], torch.zeros_like(decay[:, :1])), 1)
    grad = _scan(after.flip(1), d_h.flip(1)).flip(1)
    before = torch.where(forget[:, :, None], 0.0, torch.cat((h0[:, None], h[:, :-1]), 1))
    if s["gate"] == "logit":
        d_x, d_g = grad * keep, grad * a * keep * (before - x)
    else:
        d_x, d_g = grad, grad * before
    out["d_x"] = _turned(torch.where(behind, 0.0, d_x), order).to(s["x"].dtype)
    out["d_g"] = _turned(torch.where(behind, 0.0, d_g), order).to(s["g"].dtype)
    out["d_h0"] = decay[:, 0] * grad[:, 0]
    return out


def _plain_log_probs(s):
    logits = s["logits"].float()
    if s["unavailable"] is not None:
        logits = logits.masked_fill(s["unavailable"], -math.inf)
    z = logits / s["temperature"]
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    log_p = z - top - torch.log(e.sum(1, keepdim=True))
    p = torch.exp(log_p)
    weighted = torch.where(p > 0, p * log_p, 0.0)
    out = {"log_prob": log_p.gather(1, s["taken"][:, None])[:, 0], "entropy": -weighted.sum(1)}
    if s["train"]:
        d = -s["d_log_prob"][:, None] * p - s["d_entropy"][:, None] * (weighted + p * out["entropy"][:, None])
        d.scatter_add_(1, s["taken"][:, None], s["d_log_prob"][:, None])
        out["d_logits"] = (d / s["temperature"]).to(s["logits"].dtype)
    if s["top"]:
        # by the logits themselves: log probabilities of different logits may round to the same number
        best, ids = torch.sort(logits, dim=1, descending=True, stable=True)
        k = min(s["top"], s["actions"])
        best, ids = best[:, :k], ids[:, :k]
        log_best = log_p.gather(1, ids)
        out["top"] = torch.nn.functional.pad(torch.where(best > -math.inf, ids, -1), (0, s["top"] - k), value=-1)
        out["top_log_prob"] = torch.nn.functional.pad(log_best, (0, s["top"] - k), value=-math.inf)
    return out


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "embed":
        n, v, d = case["tokens"], case["vocab"], case["dim"]
        # rows that n draws reach: the token k is drawn with a chance of about 1 / (k ln v)
        seen = sum(1.0 - (1.0 - math.log(1.0 + 1.0 / k) / math.log(v + 1)) ** n for k in range(1, v + 1))
        back = n * d * e + v * d * e + 8 * n if case["train"] else 0
        return {"bytes": 8 * n + seen * d * e + n * d * e + back, "flops": n * d * (3 if case["train"] else 1)}
    if case["op"] == "step":
        n = case["batch"] * case["dim"]
        return {"bytes": n * (3 * e + 8), "flops": 8 * n}
    if case["op"] == "recurrence":
        b, t, d = case["batch"], case["time"], case["dim"]
        n = b * t * d
        extra = (b * t if case["resets"] else 0) + 8 * b * d
        if case["train"]:
            return {"bytes": 8 * n * e + 2 * extra, "flops": 20 * n}
        return {"bytes": 3 * n * e + extra, "flops": 7 * n}
    r, a = case["rows"], case["actions"]
    once = r * a * (e + (1 if case["mask"] else 0)) + 16 * r
    if case["train"]:
        return {"bytes": 2 * once + r * a * e + 8 * r, "flops": 14 * r * a}
    return {"bytes": once + 12 * r * case["top"], "flops": 6 * r * a}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"embed": _exact_embed, "step": _exact_step, "recurrence": _exact_recurrence, "log_probs": _exact_log_probs}[case["op"]](s)


def _exact_embed(s):
    w, ids, scale = s["weight"].double(), s["ids"], s["scale"]
    out = {"out": scale * torch.index_select(w, 0, ids)}
    if s["train"]:
        # the sums of runs of equal tokens, as differences of one running sum for some columns at a time
        order = torch.argsort(ids)
        counts = torch.bincount(ids, minlength=s["vocab"])
        ends = torch.cumsum(counts, 0)
        parts = []
        for piece in torch.split(s["d_out"], 64, 1):
            run_sum = torch.nn.functional.pad(torch.cumsum(piece.double()[order], 0), (0, 0, 1, 0))
            parts.append(run_sum[ends] - run_sum[ends - counts])
        out["d_weight"] = scale * torch.cat(parts, 1)
    return out


def _exact_step(s):
    g, x, h0 = s["g"].double(), s["x"].double(), s["h0"].double()
    h = torch.lerp(x, h0, torch.sigmoid(g)) if s["gate"] == "logit" else g * h0 + x
    return {"h": h, "last": h}


def _exact_recurrence(s):
    if s["train"] and s["time"] > 40000:
        return None
    logit = s["gate"] == "logit"
    g, x = s["g"].double(), s["x"].double()
    a = torch.sigmoid(g) if logit else g
    b, t, d = x.shape
    # every step of every history in its own order: step k of history i is at[i, k], or -1 behind its end
    ends = [t] * b if s["ends"] is None else s["ends"].tolist()
    at = torch.full((b, t), -1)
    for i, n in enumerate(ends):
        at[i, :n] = torch.arange(n).flip(0) if s["reverse"] else torch.arange(n)
    at = at.to(x.device)
    row = torch.arange(b, device=x.device)
    forget = torch.zeros(b, t, dtype=torch.bool, device=x.device) if s["starts"] is None else s["starts"]
    h, state, before = torch.zeros_like(x), s["h0"].double(), torch.zeros_like(x)
    for k in range(t):
        now = at[:, k]
        on = (now >= 0)[:, None]
        p = now.clamp(min=0)
        old = torch.where(forget[row, p][:, None], 0.0, state)
        f = a[row, p]
        new = f * old + ((1 - f) * x[row, p] if logit else x[row, p])
        h[row, p] = torch.where(on, new, h[row, p])
        before[row, p] = torch.where(on, old, before[row, p])
        state = torch.where(on, new, state)
    out = {"h": h, "last": state}
    if s["train"]:
        grad, d_h = s["d_last"].double(), s["d_h"].double()
        d_x, d_g = torch.zeros_like(x), torch.zeros_like(x)
        for k in reversed(range(t)):
            now = at[:, k]
            on = (now >= 0)[:, None]
            p = now.clamp(min=0)
            f = a[row, p]
            here = grad + d_h[row, p]
            gx, gf = (here * (1 - f), here * f * (1 - f) * (before[row, p] - x[row, p])) if logit else (here, here * before[row, p])
            d_x[row, p] = torch.where(on, gx, d_x[row, p])
            d_g[row, p] = torch.where(on, gf, d_g[row, p])
            back = torch.where(forget[row, p][:, None], 0.0, f * here)
            grad = torch.where(on, back, grad)
        out.update(d_x=d_x, d_g=d_g, d_h0=grad)
    return out


def _exact_log_probs(s):
    keys = ["log_prob", "entropy"] + (["d_logits"] if s["train"] else []) + (["top", "top_log_prob"] if s["top"] else [])
    parts = {k: [] for k in keys}
    rows = max(1, 2 ** 26 // s["actions"])
    for r in range(0, s["rows"], rows):
        z = s["logits"][r:r + rows].double() / s["temperature"]
        if s["unavailable"] is not None:
            z = torch.where(s["unavailable"][r:r + rows], -math.inf, z)
        taken = s["taken"][r:r + rows]
        lse = torch.logsumexp(z, 1)
        p = torch.exp(z - lse[:, None])
        finite = torch.where(z == -math.inf, 0.0, z)
        entropy = lse - (p * finite).sum(1)
        parts["log_prob"].append(z[torch.arange(len(z), device=z.device), taken] - lse)
        parts["entropy"].append(entropy)
        if s["train"]:
            g, k = s["d_log_prob"][r:r + rows].double()[:, None], s["d_entropy"][r:r + rows].double()[:, None]
            one = torch.zeros_like(p).scatter_(1, taken[:, None], 1.0)
            d = g * (one - p) - k * p * (finite - lse[:, None] + entropy[:, None])
            parts["d_logits"].append(d / s["temperature"])
        if s["top"]:
            left = z.clone()
            ids, values = [], []
            for _ in range(s["top"]):
                best = left.amax(1)
                first = (left == best[:, None]).int().argmax(1)
                none = best == -math.inf
                ids.append(torch.where(none, -1, first))
                values.append(torch.where(none, -math.inf, best - lse))
                left.scatter_(1, first[:, None], -math.inf)
            parts["top"].append(torch.stack(ids, 1))
            parts["top_log_prob"].append(torch.stack(values, 1))
    return {k: torch.cat(v) for k, v in parts.items()}
