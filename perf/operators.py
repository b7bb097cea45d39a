"""The operators between an observation and an action, as they are measured: a gated linear recurrence (over segments with its
gradients, and one step at a time) and the action head on its logits (adjusted logits, sampling, re-evaluation with gradients).

`own = False`: elementary torch operations in 32 bits (64 where an action is picked next to a border of the distribution);
`own = True`: the framework's entry points.  Sizes: 24 agents per environment, 4096 environments, 8192 segments of 256 steps and a
hidden width of 128 are the framework's own; wide vocabularies are generic.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # the trainer's whole batch: 8192 segments of 256 steps through the recurrent core, forward and backward
        {"name": "segments", "op": "recurrence", "rows": 8192, "steps": 256, "width": 128, "type": "bf16", "packed": True, "resets": 0.004},
        # one agent's record over many episodes, kept as one row: all the work lies along time
        {"name": "one_record", "op": "recurrence", "rows": 1, "steps": 65536, "width": 128, "type": "f32", "packed": False, "resets": 0.0005},
        # an ordinary minibatch, odd in every direction
        {"name": "minibatch", "op": "recurrence", "rows": 250, "steps": 129, "width": 100, "type": "f16", "packed": False, "resets": 0.01},
        # one environment's 24 agents, one step: latency
        {"name": "step_one_env", "op": "step", "rows": 24, "width": 128, "type": "f32", "resets": 0.01},
        # every agent of 4096 environments, one step
        {"name": "step_all_envs", "op": "step", "rows": 98304, "width": 128, "type": "bf16", "resets": 0.001},
        # a batch of sequences over a wide vocabulary, all controls on
        {"name": "adjust_vocabulary", "op": "adjust", "rows": 64, "width": 50001, "type": "bf16", "train": False, "mask": "packed", "bias": "shared", "history": 512, "temperature": 0.8},
        # a large action table with vibes, masks and recent actions, with the gradient
        {"name": "adjust_actions", "op": "adjust", "rows": 24576, "width": 157, "type": "f32", "train": True, "mask": "bool", "bias": "none", "history": 32, "temperature": 1.0},
        # one environment's 24 agents pick among the arena's five actions: latency
        {"name": "sample_one_env", "op": "sample", "rows": 24, "width": 5, "type": "f32", "mask": "none", "bias": "none", "history": 0, "temperature": 1.0},
        # every agent of 4096 environments, some actions masked, the last 16 penalised
        {"name": "sample_all_envs", "op": "sample", "rows": 98304, "width": 5, "type": "bf16", "mask": "bool", "bias": "none", "history": 16, "temperature": 1.0},
        # few rows, a wide vocabulary, all controls on
        {"name": "sample_vocabulary", "op": "sample", "rows": 16, "width": 131072, "type": "f16", "mask": "packed", "bias": "rows", "history": 2048, "temperature": 0.7},
        # the trainer's whole batch of stored actions: log-probability and entropy, forward and backward
        {"name": "evaluate_segments", "op": "evaluate", "rows": 8192 * 256, "width": 5, "type": "bf16", "mask": "none", "bias": "none", "history": 0, "temperature": 1.0},
        # the same over a wide vocabulary
        {"name": "evaluate_vocabulary", "op": "evaluate", "rows": 2048, "width": 32003, "type": "bf16", "mask": "packed", "bias": "none", "history": 0, "temperature": 1.25},
    ]


def _log_between(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "step", "adjust", "sample", "evaluate"])
    case = {"op": op, "type": rng.choice(["f32", "bf16", "f16"])}
    if op == "recurrence":
        case["steps"] = _log_between(rng, 1, 65536)
        case["width"] = _log_between(rng, 1, 1024)
        case["rows"] = _log_between(rng, 1, max(1, min(16384, (1 << 25) // (case["steps"] * case["width"]))))
        while case["rows"] * case["steps"] * case["width"] > 1 << 26:
            case["width"] = max(1, case["width"] // 2)
        case["packed"] = rng.random() < 0.5
        case["resets"] = rng.choice([0.0, 0.002, 0.05])
    elif op == "step":
        case["rows"] = _log_between(rng, 1, 131072)
        case["width"] = _log_between(rng, 1, min(2048, (1 << 25) // case["rows"]))
        case["resets"] = rng.choice([0.0, 0.002, 0.05])
    else:
        case["width"] = _log_between(rng, 2, 131072)
        case["rows"] = _log_between(rng, 1, max(1, min(1 << 20, (1 << 24) // case["width"])))
        case["mask"] = rng.choice(["none", "bool", "packed"])
        case["bias"] = rng.choice(["none", "shared", "rows"])
        case["history"] = rng.choice([0, 0, _log_between(rng, 1, max(1, min(4096, (1 << 24) // case["rows"])))])
        case["temperature"] = rng.choice([1.0, round(rng.uniform(0.5, 2.0), 3)])
        if op == "adjust":
            case["train"] = rng.random() < 0.5
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _pack(allowed):
    """bit v % 32 of word v // 32: token v is allowed."""
    n, v = allowed.shape
    words = (v + 31) // 32
    bits = torch.zeros(n, words * 32, dtype=torch.bool, device=allowed.device)
    bits[:, :v] = allowed
    w = bits.view(n, words, 32).long() << torch.arange(32, device=allowed.device)
    w = w.sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, v, t = case["rows"], case["width"], TYPES[case["type"]]
    normal = lambda *s, dtype=torch.float32: torch.randn(*s, generator=g, device="cuda", dtype=dtype)  # noqa: E731
    uniform = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    if case["op"] == "recurrence":
        steps = case["steps"]
        # candidates around zero, gates that keep most of the state (as a trained core's do)
        if case["packed"]:
            x = normal(n, steps, 2 * v, dtype=t)
            x[..., v:].mul_(1.5).add_(2.0)
            gate = None
        else:
            x, gate = normal(n, steps, v, dtype=t), normal(n, steps, v, dtype=t).mul_(1.5).add_(2.0).requires_grad_()
        return {"case": case, "x": x.requires_grad_(), "gate": gate, "state": normal(n, v).requires_grad_(), "resets": uniform(n, steps) < case["resets"],
                "dh": normal(n, steps, v, dtype=t), "dlast": normal(n, v)}  # fmt: skip
    if case["op"] == "step":
        return {"case": case, "x": normal(n, v, dtype=t), "gate": normal(n, v, dtype=t).mul_(1.5).add_(2.0), "state": normal(n, v), "resets": uniform(n) < case["resets"]}
    logits = (normal(n, v) * 2.0).to(t)
    s = {"case": case, "controls": {"temperature": case["temperature"]}}
    allowed = None
    if case["mask"] != "none":  # about three fifths are allowed; in one row of a hundred nothing is
        allowed = (uniform(n, v) < 0.6) & (uniform(n, 1) >= 0.01)
        s["controls"]["allowed"] = allowed if case["mask"] == "bool" else _pack(allowed)
    if case["bias"] != "none":
        s["controls"]["bias"] = normal(v) if case["bias"] == "shared" else normal(n, v)
    if case["history"]:  # recent tokens, low numbers more often, the unused end of a row filled with -1
        h = (uniform(n, case["history"]).pow(3) * v).to(torch.int32).clamp_(max=v - 1)
        used = (uniform(n, 1) * (case["history"] + 1)).to(torch.int32)
        h[torch.arange(case["history"], device="cuda")[None, :] >= used] = -1
        s["controls"] |= {"history": h, "repetition": 1.25, "presence": 0.5, "frequency": 0.125}
    if case["op"] == "sample":
        s["uniforms"] = uniform(n)
    if case["op"] == "evaluate":
        noise = uniform(n, v).clamp_(min=1e-30).log_().neg_().log_().neg_()
        noise += logits
        if allowed is not None:
            noise[~allowed] = -math.inf
        s["actions"] = noise.argmax(1).to(torch.int32)
        if allowed is not None:
            s["actions"][~allowed.any(1)] = -1
        s["dlogp"], s["dentropy"] = normal(n), normal(n) * 0.1
    if case["op"] == "adjust" and case["train"]:
        s["dout"] = normal(n, v, dtype=t)
    s["logits"] = logits.requires_grad_(case["op"] == "evaluate" or bool(case.get("train")))
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------


def _scan(a, b):
    """h[t] = a[t] * h[t-1] + b[t] along dim 1 from h[-1] = 0: pairs, then pairs of pairs, ..."""
    k, steps = 1, a.shape[1]
    while k < steps:
        b = torch.cat([b[:, :k], b[:, k:] + a[:, k:] * b[:, :-k]], 1)
        a = torch.cat([a[:, :k], a[:, k:] * a[:, :-k]], 1)
        k *= 2
    return b


def _recurrence(s):
    v = s["case"]["width"]
    x = s["x"].detach()
    x, g = (x[..., :v], x[..., v:]) if s["gate"] is None else (x, s["gate"].detach())
    t, x, g = x.dtype, x.float(), g.float()
    a, keep = torch.sigmoid(g), ~s["resets"][..., None]
    ak = a * keep
    b = torch.sigmoid(-g) * x
    state = s["state"].detach()
    b[:, 0] += ak[:, 0] * state
    h = _scan(ak, b)
    del b
    before = torch.cat([state[:, None], h[:, :-1]], 1) * keep
    d = s["dh"].float()
    d[:, -1] += s["dlast"]
    # the same scan against time: d[t] += a[t+1] * d[t+1]
    d = _scan(torch.cat([ak[:, 1:], ak[:, :1]], 1).flip(1), d.flip(1)).flip(1)
    dx = torch.sigmoid(-g) * d
    dg = d * (before - x) * a * torch.sigmoid(-g)
    out = {"h": h.to(t), "last": h[:, -1].clone(), "dstate": ak[:, 0] * d[:, 0]}
    return out | ({"dx": torch.cat([dx, dg], -1).to(t)} if s["gate"] is None else {"dx": dx.to(t), "dgate": dg.to(t)})


def _step(s):
    x, g = s["x"].float(), s["gate"].float()
    before = torch.where(s["resets"][:, None], 0.0, s["state"])
    h = torch.sigmoid(g) * before + torch.sigmoid(-g) * x
    return {"h": h.to(s["x"].dtype), "state": h}


def _unpack(words, v):
    bits = (words[..., None] >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1
    return bits.flatten(-2)[..., :v].bool()


def _adjusted(s, dtype):
    """The adjusted logits, and what their gradient is multiplied by."""
    c, v = s["controls"], s["case"]["width"]
    l = s["logits"].detach().to(dtype)
    slope = torch.full_like(l, 1.0 / c["temperature"])
    if "history" in c:
        h = c["history"].long()
        counts = torch.zeros(l.shape[0], v + 1, dtype=dtype, device=l.device)
        counts.scatter_add_(1, torch.where((h >= 0) & (h < v), h, v), torch.ones_like(h, dtype=dtype))
        counts = counts[:, :v]
        seen = counts > 0
        slope = torch.where(seen, torch.where(l > 0, slope / c["repetition"], slope * c["repetition"]), slope)
        l = torch.where(seen, torch.where(l > 0, l / c["repetition"], l * c["repetition"]), l)
        l = l - c["frequency"] * counts - c["presence"] * seen
    if "bias" in c:
        l = l + c["bias"]
    l = l / c["temperature"]
    if "allowed" in c:
        ok = c["allowed"] if c["allowed"].dtype == torch.bool else _unpack(c["allowed"], v)
        l = torch.where(ok, l, -math.inf)
        slope = slope * ok
    return l, slope


def _adjust(s):
    t = s["logits"].dtype
    l, slope = _adjusted(s, torch.float32)
    return {"adjusted": l.to(t)} | ({"dlogits": (s["dout"].float() * slope).to(t)} if s["case"]["train"] else {})


def _distribution(l):
    m = l.max(1, keepdim=True).values
    empty = m == -math.inf
    e = torch.exp(l - torch.where(empty, 0.0, m))
    z = e.sum(1, keepdim=True)
    z = torch.where(empty, 1.0, z)
    logq = l - torch.where(empty, 0.0, m) - torch.log(z)
    q = e / z
    entropy = -torch.where(q > 0, q * logq, 0.0).sum(1)
    return q, logq, entropy, empty[:, 0], e, z


def _sample(s):
    l, _ = _adjusted(s, torch.float64)  # an action next to a border is the one that 64 bits give
    q, logq, entropy, empty, e, z = _distribution(l)
    above = torch.cumsum(e, 1) > s["uniforms"][:, None].double() * z
    last = l.shape[1] - 1 - (e.flip(1) > 0).to(torch.int8).argmax(1)
    action = torch.where(above.any(1), above.to(torch.int8).argmax(1), last)
    logp = logq.gather(1, action[:, None])[:, 0]
    return {"actions": torch.where(empty, -1, action).to(torch.int32), "logp": torch.where(empty, 0.0, logp).float(), "entropy": entropy.float()}


def _evaluate(s):
    l, slope = _adjusted(s, torch.float32)
    q, logq, entropy, empty, _, _ = _distribution(l)
    a = s["actions"].long()
    at = a.clamp(min=0)[:, None]
    logp = torch.where(empty, 0.0, logq.gather(1, at)[:, 0])
    d = -s["dlogp"][:, None] * q
    d.scatter_add_(1, at, s["dlogp"][:, None])
    d -= s["dentropy"][:, None] * torch.where(q > 0, q * (logq + entropy[:, None]), 0.0)
    d = torch.where(empty[:, None] | (slope == 0), 0.0, d * slope)
    return {"logp": logp, "entropy": entropy, "dlogits": d.to(s["logits"].dtype)}


# ---- one pass ---------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _own(s)
    return {"recurrence": _recurrence, "step": _step, "adjust": _adjust, "sample": _sample, "evaluate": _evaluate}[s["case"]["op"]](s)


def _own(s):
    from metta_amd import action_head, recurrence

    op = s["case"]["op"]
    if op == "step":
        h, state = recurrence.gated_recurrence_step(s["x"], s["gate"], s["state"], s["resets"])
        return {"h": h, "state": state}
    if op == "recurrence":
        h, last = recurrence.gated_recurrence(s["x"], s["gate"], s["state"], s["resets"])
        leaves = [s["x"], s["state"]] + ([] if s["gate"] is None else [s["gate"]])
        grads = torch.autograd.grad([h, last], leaves, [s["dh"], s["dlast"]])
        if s["dh"].dtype == torch.float32:  # the plain form adds dlast to a 32-bit dh where it lies: a state called again is
            s["dh"][:, -1] += s["dlast"]  # the same on both sides only if this one does so too, after its own pass
        out = {"h": h.detach(), "last": last.detach(), "dstate": grads[1], "dx": grads[0]}
        return out if s["gate"] is None else out | {"dgate": grads[2]}
    if op == "adjust":
        l = action_head.adjust_logits(s["logits"], **s["controls"])
        if not s["case"]["train"]:
            return {"adjusted": l}
        return {"adjusted": l.detach(), "dlogits": torch.autograd.grad(l, s["logits"], s["dout"])[0]}
    if op == "sample":
        actions, logp, entropy = action_head.sample_actions(s["logits"], s["uniforms"], **s["controls"])
        return {"actions": actions, "logp": logp, "entropy": entropy}
    logp, entropy = action_head.evaluate_actions(s["logits"], s["actions"], **s["controls"])
    (d,) = torch.autograd.grad([logp, entropy], [s["logits"]], [s["dlogp"], s["dentropy"]])
    return {"logp": logp.detach(), "entropy": entropy.detach(), "dlogits": d}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------


def work(case):
    n, v, s = case["rows"], case["width"], SIZE[case["type"]]
    if case["op"] == "step":
        # candidate, gate and state in; state and (where it is of another type) output out; one reset per row
        return {"bytes": n * v * (2 * s + 8 + (s if s < 4 else 0)) + n, "flops": 9 * n * v}
    if case["op"] == "recurrence":
        e = n * case["steps"]
        # candidate, gate and output's gradient in; output and two gradients out; resets; state, last and their gradients
        return {"bytes": e * v * 6 * s + e + n * v * 16, "flops": 26 * e * v}
    e = n * v
    controls = {"none": 0, "bool": e, "packed": 4 * n * ((v + 31) // 32)}[case["mask"]]
    controls += {"none": 0, "shared": 4 * v, "rows": 4 * e}[case["bias"]] + 4 * n * case["history"]
    if case["op"] == "adjust":
        # logits in, adjusted logits out; with the gradient also dout in, dlogits out
        return {"bytes": e * s * (4 if case["train"] else 2) + controls, "flops": 6 * e}
    if case["op"] == "sample":
        return {"bytes": e * s + controls + 16 * n, "flops": 12 * e}
    return {"bytes": 2 * e * s + controls + 20 * n, "flops": 24 * e}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------


def _exact_logits(s):
    """Adjusted logits and slopes, built from the end of the definition: masks, scale, bias, penalties."""
    c, l = s["controls"], s["logits"].detach().double()
    n, v = l.shape
    counts = torch.zeros(n, v, dtype=torch.float64, device=l.device)
    if "history" in c:
        rows = torch.arange(n, device=l.device)[:, None].expand_as(c["history"])
        real = (c["history"] >= 0) & (c["history"] < v)
        one = torch.ones((), dtype=torch.float64, device=l.device)
        counts.index_put_((rows[real], c["history"][real].long()), one, accumulate=True)
    r, f, p = (c.get(k, d) for k, d in (("repetition", 1.0), ("frequency", 0.0), ("presence", 0.0)))
    factor = torch.ones_like(l)
    factor[(counts > 0) & (l > 0)] = 1.0 / r
    factor[(counts > 0) & (l <= 0)] = r
    out = (l * factor - f * counts - p * counts.clamp(max=1.0) + c.get("bias", 0.0)) / c["temperature"]
    factor /= c["temperature"]
    if "allowed" in c:
        m = c["allowed"]
        if m.dtype != torch.bool:
            at = torch.arange(v, device=l.device)
            m = (m[:, at // 32].long() >> (at % 32)) & 1 == 1
        out[~m], factor[~m] = -math.inf, 0.0
    return out, factor


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("recurrence", "step"):
        v = case["width"]
        x = s["x"].detach()
        x, g = (x[..., :v].double(), x[..., v:].double()) if s["gate"] is None else (x.double(), s["gate"].detach().double())
        a = 1.0 / (1.0 + torch.exp(-g))
        w = 1.0 / (1.0 + torch.exp(g))
        state = s["state"].detach().double()
        if case["op"] == "step":
            h = a * (state * ~s["resets"][:, None]) + w * x
            return {"h": h, "state": h}
        ak = (a * ~s["resets"][..., None]).transpose(0, 1).contiguous()
        h = (w * x).transpose(0, 1).contiguous()
        before = state
        for t in range(case["steps"]):
            h[t].addcmul_(ak[t], before)
            before = h[t]
        d = s["dh"].double().transpose(0, 1).contiguous()
        d[-1] += s["dlast"]
        for t in range(case["steps"] - 2, -1, -1):
            d[t].addcmul_(ak[t + 1], d[t + 1])
        out = {"last": h[-1].clone(), "dstate": ak[0] * d[0]}
        h, d = h.transpose(0, 1), d.transpose(0, 1)
        out["h"] = h
        keep = torch.cat([state[:, None], h[:, :-1]], 1) * ~s["resets"][..., None]
        dx, dg = d * w, d * (keep - x) * (a * w)
        return out | ({"dx": torch.cat([dx, dg], -1)} if s["gate"] is None else {"dx": dx, "dgate": dg})
    l, factor = _exact_logits(s)
    if case["op"] == "adjust":
        return {"adjusted": l} | ({"dlogits": s["dout"].double() * factor} if case["train"] else {})
    lse = torch.logsumexp(l, 1)
    empty = lse == -math.inf
    logq = torch.where(empty[:, None], -math.inf, l - torch.where(empty, 0.0, lse)[:, None])
    q = torch.exp(logq)
    entropy = torch.special.entr(q).sum(1)
    if case["op"] == "sample":
        shifted = torch.exp(l - torch.where(empty, 0.0, l.amax(1))[:, None])
        total = shifted.cumsum(1)
        u = s["uniforms"].double()[:, None] * shifted.sum(1, keepdim=True)
        picked = torch.searchsorted(total, u, right=True)[:, 0]  # the first whose running sum is above u
        order = torch.arange(l.shape[1], device=l.device)
        picked = torch.minimum(picked, torch.where(shifted > 0, order, 0).amax(1))
        logp = torch.where(empty, 0.0, logq.gather(1, picked[:, None])[:, 0])
        return {"actions": torch.where(empty, -1, picked).to(torch.int32), "logp": logp, "entropy": entropy}
    at = s["actions"].long().clamp(min=0)[:, None]
    logp = torch.where(empty, 0.0, logq.gather(1, at)[:, 0])
    hit = torch.zeros_like(q).scatter_(1, at, 1.0)
    d = s["dlogp"].double()[:, None] * (hit - q) - s["dentropy"].double()[:, None] * torch.nan_to_num(q * (logq + entropy[:, None]), nan=0.0)
    return {"logp": logp, "entropy": entropy, "dlogits": torch.where(empty[:, None], 0.0, d * factor)}
