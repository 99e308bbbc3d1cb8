"""The policy-side operators of ``isaaclab_amd.rl``, case by case, in their plain form and as a user calls them:
sampling an action from logits, evaluating stored actions with the gradient by the logits, and the global norm of many
gradients with clipping.  ``own`` chooses between the two."""
import math
import random

import torch

own = False

_DT = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_BYTES = {"float32": 4, "bfloat16": 2, "float16": 2}


# -- cases ------------------------------------------------------------------------------------------------------------
def _sample(name, dtype, rows, vocab, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, masked=False, per_row=False, scale=2.0):
    c = {"op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k,
         "top_p": top_p, "min_p": min_p, "masked": masked, "per_row": per_row, "scale": scale}
    return dict(c, name=name) if name else c


def _evaluate(name, dtype, rows, vocab, temperature=1.0, masked=False, scale=2.0):
    c = {"op": "evaluate", "dtype": dtype, "rows": rows, "vocab": vocab, "temperature": temperature, "masked": masked,
         "scale": scale}
    return dict(c, name=name) if name else c


def _clip(name, dtype, count, total, in_place, clipped):
    c = {"op": "clip", "dtype": dtype, "count": count, "total": total, "in_place": in_place, "clipped": clipped}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one environment being watched while a policy with 32 discrete actions plays: latency
        _sample("sample-one-env", "float32", 1, 32),
        # a rollout step of 4096 environments x 12 joints, each joint's target out of 256 bins
        _sample("sample-joint-bins", "float32", 4096 * 12, 256, temperature=0.8, top_p=0.95),
        # an odd number of environments with forbidden actions and settings of their own (exploration schedules)
        _sample("sample-masked-rows", "bfloat16", 4099, 1000, masked=True, per_row=True),
        # a single answer of a policy over action tokens, long odd vocabulary
        _sample("sample-long-one", "bfloat16", 1, 100003, temperature=0.9, top_k=50, top_p=0.9, scale=3.0),
        # a batch of environments on a vocabulary of action tokens
        _sample("sample-long-batch", "bfloat16", 1024, 131072, temperature=0.7, top_p=0.95, min_p=0.02, scale=3.0),
        # a handful of stored decisions, masked, odd width: latency of the evaluation and its gradient
        _evaluate("evaluate-small", "float32", 64, 19, masked=True),
        # a PPO minibatch: 4096 environments x 24 steps / 4 minibatches, 12 joints of 64 bins each
        _evaluate("evaluate-minibatch", "float32", 4096 * 24 // 4 * 12, 64),
        # rows of odd length: no row but the first starts on a vector boundary
        _evaluate("evaluate-odd-rows", "bfloat16", 2047, 50001, temperature=0.7, scale=3.0),
        # the largest update: action tokens of a whole rollout
        _evaluate("evaluate-large", "bfloat16", 8192, 32768, scale=3.0),
        # actor and critic (235 observations, hidden 512 / 256 / 128, 12 actions), below the bound as most updates are
        _clip("clip-policy", "float32", 17, 0, True, False),
        # many ragged 16-bit gradients clipped into the 32-bit ones that an optimiser reads
        _clip("clip-ragged", "bfloat16", 57, 2_300_017, False, True),
        # a large policy, gradients of both kinds, clipped
        _clip("clip-large", "mixed", 48, 160_000_000, False, True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "evaluate", "clip"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "clip":
        count = rng.randint(1, 60)
        return _clip(None, rng.choice([dtype, "mixed"]), count, _log_int(rng, max(1000, 2 * count), 120_000_000),
                     False, rng.random() < 0.7)
    vocab = _log_int(rng, 2, 131072)
    rows = _log_int(rng, 1, max(1, min(200_000, 60_000_000 // vocab)))
    temperature = round(rng.uniform(0.5, 1.5), 3)
    scale = round(rng.uniform(0.5, 4.0), 2)
    if op == "evaluate":
        return _evaluate(None, dtype, rows, vocab, temperature, rng.random() < 0.4, scale)
    return _sample(None, dtype, rows, vocab, temperature, rng.choice([0, 0, rng.randint(1, 200)]),
                   rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]), rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 4)]),
                   rng.random() < 0.3, rng.random() < 0.3, scale)


def _sizes(case):
    """Shapes of the gradients of a case: an actor-critic for total = 0, else ``count`` ragged ones that sum to total."""
    if case["total"] == 0:
        dims = [235, 512, 256, 128]
        shapes = [(12,)]                                   # the action noise
        for last in (12, 1):
            for a, b in zip(dims, dims[1:] + [last]):
                shapes += [(b, a), (b,)]
        return shapes
    r = random.Random(case["count"] * 7919 + case["total"])
    weights = [math.exp(r.uniform(-4.0, 2.0)) for _ in range(case["count"])]
    sizes = [max(1, int(case["total"] * w / sum(weights))) for w in weights]
    return [(s,) for s in sizes]


def _dtypes(case, n):
    if case["dtype"] == "mixed":
        return [torch.bfloat16 if i % 2 else torch.float32 for i in range(n)]
    return [_DT[case["dtype"]]] * n


# -- inputs -----------------------------------------------------------------------------------------------------------
def _logits(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1_000_003 + case["rows"] * 31 + case["vocab"])
    x = torch.randn(case["rows"], case["vocab"], generator=g, device="cuda")
    x = x.mul_(case["scale"]).to(_DT[case["dtype"]])
    mask = None
    if case["masked"]:
        mask = torch.rand(case["rows"], case["vocab"], generator=g, device="cuda") < 0.7
        mask[:, 0] = True
    return g, x, mask


def prepare(case, seed):
    if case["op"] == "clip":
        g = torch.Generator(device="cuda").manual_seed(seed * 1_000_003 + case["count"])
        shapes = _sizes(case)
        grads = [(torch.randn(s, generator=g, device="cuda") * 0.02).to(d) for s, d in zip(shapes, _dtypes(case, len(shapes)))]
        # expected norm 0.02 sqrt(N)
        expected = 0.02 * math.sqrt(sum(t.numel() for t in grads))
        state = {"case": case, "max_norm": expected * (0.25 if case["clipped"] else 4.0)}
        if case["in_place"]:
            state["parameters"] = []
            for t in grads:
                p = torch.nn.Parameter(torch.empty_like(t))
                p.grad = t
                state["parameters"].append(p)
        else:
            state["grads"] = grads
            state["out"] = [torch.empty(t.shape, dtype=torch.float32, device="cuda") for t in grads]
        return state
    g, x, mask = _logits(case, seed)
    rows = case["rows"]
    state = {"case": case, "logits": x, "mask": mask}
    if case["op"] == "evaluate":
        x.requires_grad_()
        a = torch.randint(0, case["vocab"], (rows,), generator=g, device="cuda")
        state["actions"] = a if mask is None else torch.where(mask.gather(1, a[:, None])[:, 0], a, torch.zeros_like(a))
        state["grad_log_prob"] = torch.randn(rows, generator=g, device="cuda")
        state["grad_entropy"] = torch.randn(rows, generator=g, device="cuda") * 0.1
        return state
    state["u"] = torch.rand(rows, generator=g, device="cuda")
    for k in ("temperature", "top_k", "top_p", "min_p"):
        state[k] = case[k]
    if case["per_row"]:
        def rnd(lo, hi):
            return torch.rand(rows, generator=g, device="cuda") * (hi - lo) + lo
        state["temperature"] = rnd(0.5, 1.5)
        state["top_k"] = torch.randint(0, 200, (rows,), generator=g, device="cuda", dtype=torch.int32)
        state["top_p"] = rnd(0.5, 1.05).clamp(max=1.0)
        state["min_p"] = rnd(-0.05, 0.1).clamp(min=0.0)
    return state


# -- plain forms ------------------------------------------------------------------------------------------------------
def _col(v, rows):
    """A setting as a column in 64 bits, holding the value that 32 bits hold."""
    if isinstance(v, torch.Tensor):
        return v.double()[:, None]
    return torch.full((rows, 1), float(torch.tensor(float(v), dtype=torch.float32)), dtype=torch.float64, device="cuda")


def _plain_sample(s):
    x, mask = s["logits"], s["mask"]
    rows, vocab = x.shape
    z = x.double() + 0.0
    if mask is not None:
        z = z.masked_fill(~mask, -math.inf)
    m = z.amax(1, keepdim=True)
    w = torch.exp((z - m) / _col(s["temperature"], rows))
    truncated = s["case"]["per_row"] or s["top_k"] > 0 or s["top_p"] < 1.0 or s["min_p"] > 0.0
    if truncated:
        _, order = torch.sort(z, dim=1, descending=True, stable=True)
        ws = w.gather(1, order)
        k = _col(s["top_k"], rows)
        k = torch.where(k > 0, k, vocab)
        keep = torch.arange(vocab, device="cuda")[None, :] < k
        p = _col(s["top_p"], rows)
        wk = torch.where(keep, ws, 0.0)
        upto = wk.cumsum(1)
        before = torch.cat([torch.zeros_like(upto[:, :1]), upto[:, :-1]], 1)
        keep &= (before < p * upto[:, -1:]) | (p >= 1.0)
        keep &= ws >= _col(s["min_p"], rows)
        keep[:, 0] = True
        w = torch.where(torch.zeros_like(keep).scatter_(1, order, keep), w, 0.0)
    c = w.cumsum(1)
    actions = (c > s["u"].double()[:, None] * c[:, -1:]).to(torch.uint8).argmax(1)
    log_prob = torch.log(w.gather(1, actions[:, None]) / c[:, -1:])[:, 0]
    return actions, log_prob.float()


def _plain_evaluate(s):
    x, mask, a = s["logits"].detach(), s["mask"], s["actions"][:, None]
    inv_t = 1.0 / s["case"]["temperature"]
    z = x.float() * inv_t
    if mask is not None:
        z = z.masked_fill(~mask, -math.inf)
    d = z - z.amax(1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_total = torch.log(total)
    log_prob = d.gather(1, a) - log_total
    p = e / total
    log_p = d - log_total
    if mask is not None:
        log_p = log_p.masked_fill(~mask, 0.0)
    entropy = -(p * log_p).sum(1, keepdim=True)
    gl, ge = s["grad_log_prob"][:, None], s["grad_entropy"][:, None]
    grad = -p * (gl + ge * (log_p + entropy))
    grad = grad.scatter_add(1, a, gl) * inv_t
    return log_prob[:, 0], entropy[:, 0], grad.to(x.dtype)


def _plain_clip(s):
    grads = [p.grad for p in s["parameters"]] if "parameters" in s else s["grads"]
    norm = torch.stack([(t.double() * t.double()).sum() for t in grads]).sum().sqrt()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    out = grads if "parameters" in s else s["out"]
    for t, o in zip(grads, out):
        o.copy_(t.float() * factor)
    return [norm.float()] + out


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"sample": _plain_sample, "evaluate": _plain_evaluate, "clip": _plain_clip}[op](state)
    from isaaclab_amd import rl

    if op == "sample":
        return rl.sample_categorical(state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                                     top_p=state["top_p"], min_p=state["min_p"], mask=state["mask"])
    if op == "evaluate":
        log_prob, entropy = rl.evaluate_categorical(state["logits"], state["actions"],
                                                    temperature=state["case"]["temperature"], mask=state["mask"])
        grad, = torch.autograd.grad((log_prob, entropy), state["logits"], (state["grad_log_prob"], state["grad_entropy"]))
        return log_prob.detach(), entropy.detach(), grad
    if "parameters" in state:
        norm = rl.clip_grad_norm_(state["parameters"], state["max_norm"])
        return [norm] + [p.grad for p in state["parameters"]]
    out, norm = rl.clip_grads(state["grads"], state["max_norm"], out=state["out"])
    return [norm] + out


def work(case):
    if case["op"] == "clip":
        shapes = _sizes(case)
        n = [math.prod(s) for s in shapes]
        read = sum(k * d.itemsize for k, d in zip(n, _dtypes(case, len(n))))
        # gradients below the bound stay as they are
        return {"bytes": read + (0 if case["in_place"] and not case["clipped"] else 4 * sum(n)), "flops": 3 * sum(n)}
    n, e = case["rows"] * case["vocab"], _BYTES[case["dtype"]]
    mask = n if case["masked"] else 0
    if case["op"] == "sample":
        return {"bytes": n * e + mask + case["rows"] * 16, "flops": 4 * n}
    # logits and mask in, gradient out; action, two results and their two gradients a row
    return {"bytes": 2 * n * e + mask + case["rows"] * 24, "flops": 12 * n}


# -- the definition in 64 bits ----------------------------------------------------------------------------------------
def _exact_sample(s):
    rows, vocab = s["logits"].shape
    actions, log_prob = [], []
    step = max(1, 40_000_000 // vocab)

    def part(v, at):
        return v[at].to(torch.float64).unsqueeze(1) if isinstance(v, torch.Tensor) else torch.tensor(v, dtype=torch.float32, device="cuda").to(torch.float64).view(1, 1)

    for first in range(0, rows, step):
        at = slice(first, first + step)
        x = s["logits"][at].to(torch.float64)
        x = torch.where(x == 0.0, torch.zeros_like(x), x)
        if s["mask"] is not None:
            x = torch.where(s["mask"][at], x, torch.full_like(x, -math.inf))
        n = x.shape[0]
        falling = torch.sort(x, dim=1, descending=True).values
        weight = torch.exp((falling - falling[:, :1]) / part(s["temperature"], at))
        place = torch.arange(vocab, device="cuda").expand(n, vocab)
        k = part(s["top_k"], at).expand(n, 1)
        kept = torch.where(k > 0, torch.minimum(k, torch.full_like(k, vocab)), torch.full_like(k, vocab)).long()
        weight_k = weight * (place < kept)
        reached = torch.cumsum(weight_k, 1)
        p = part(s["top_p"], at).expand(n, 1)
        # members of the shortest prefix that holds a share p: one more than those whose prefix falls short of it
        short = (reached < p * reached[:, -1:]).sum(1, keepdim=True) + 1
        kept = torch.where(p < 1.0, torch.minimum(kept, short), kept)
        heavy = (weight >= part(s["min_p"], at)).sum(1, keepdim=True)
        kept = torch.clamp(torch.minimum(kept, heavy), min=1)
        border = falling.gather(1, kept - 1)
        above, level = x > border, x == border
        room = kept - above.sum(1, keepdim=True)
        chosen = above | (level & (torch.cumsum(level.long(), 1) <= room))
        mass = torch.where(chosen, torch.exp((x - falling[:, :1]) / part(s["temperature"], at)), torch.zeros_like(x))
        line = torch.cumsum(mass, 1)
        aim = s["u"][at].to(torch.float64).unsqueeze(1) * line[:, -1:]
        a = (line <= aim).sum(1)
        actions.append(a)
        log_prob.append((x.gather(1, a[:, None]) - falling[:, :1])[:, 0] / part(s["temperature"], at)[:, 0] - torch.log(line[:, -1]))
    return torch.cat(actions), torch.cat(log_prob)


def _exact_evaluate(s):
    t = float(s["case"]["temperature"])
    x, a = s["logits"].detach(), s["actions"]
    rows, vocab = x.shape
    parts = []
    step = max(1, 40_000_000 // vocab)
    for first in range(0, rows, step):
        at = slice(first, first + step)
        z = x[at].to(torch.float64) / t
        allowed = torch.ones_like(z, dtype=torch.bool) if s["mask"] is None else s["mask"][at]
        top = torch.where(allowed, z, torch.full_like(z, -math.inf)).max(1, keepdim=True).values
        e = torch.where(allowed, torch.exp(z - top), torch.zeros_like(z))
        lse = top + torch.log(e.sum(1, keepdim=True))
        p = torch.where(allowed, torch.exp(z - lse), torch.zeros_like(z))
        hot = torch.zeros_like(z)
        hot[torch.arange(z.shape[0], device="cuda"), a[at]] = 1.0
        surprise = torch.where(allowed, lse - z, torch.zeros_like(z))
        entropy = (p * surprise).sum(1, keepdim=True)
        gl, ge = s["grad_log_prob"][at].double()[:, None], s["grad_entropy"][at].double()[:, None]
        grad = (gl * (hot - p) + ge * p * (surprise - entropy)) / t
        log_prob = -(surprise * hot).sum(1)
        # the gradient in 32 bits: rounded far below what any of its types holds, at half the memory
        parts.append((log_prob, entropy[:, 0], grad if x.dtype == torch.float32 else grad.float()))
    return tuple(torch.cat([q[i] for q in parts]) for i in range(3))


def _exact_clip(s):
    grads = [p.grad.detach() for p in s["parameters"]] if "parameters" in s else s["grads"]
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(t.flatten().to(torch.float64))) ** 2 for t in grads))
    factor = min(1.0, s["max_norm"] / (norm + 1e-6))
    return [torch.tensor(norm, dtype=torch.float64)] + [t.to(torch.float64) * factor for t in grads]


def exact(case, seed):
    state = prepare(case, seed)
    return {"sample": _exact_sample, "evaluate": _exact_evaluate, "clip": _exact_clip}[case["op"]](state)
