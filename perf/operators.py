"""Measured cases of the per-token loss operators over a vocabulary.

Two operators of ``koochak_b200.ops.functional``:

* ``token_logprobs``: log probability of a given token per row of logits, the
  entropy of the row's distribution and its most likely alternatives, with
  the gradient of the first two;
* ``topk_distillation``: KL divergence from a teacher known by its top logits
  to the student's distribution, with its gradient.

``run`` computes them in plain torch (fp32, rounded once at the end) or, with
``own`` set, through the framework's entry points. ``exact`` computes the
definitions in 64 bits, with autograd for the gradients.
"""

import math

import torch

own = False

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _logprobs(name, path, dtype, rows, vocab, pad, top_k=0, temperature=1.0, ignored=0, banned=0):
    return {"name": name, "op": "logprobs", "path": path, "dtype": dtype, "rows": rows, "vocab": vocab, "pad": pad,
            "top_k": top_k, "temperature": temperature, "ignored": ignored, "banned": banned}


def _distill(name, path, dtype, rows, vocab, pad, slots, tail, reduction, temperature=1.0, empty=0, scale=1.0):
    return {"name": name, "op": "distill", "path": path, "dtype": dtype, "rows": rows, "vocab": vocab, "pad": pad,
            "slots": slots, "tail": tail, "reduction": reduction, "temperature": temperature, "empty": empty,
            "scale": scale}


def listed():
    return [
        # One sampled token and its alternatives, as an interactive session shows them: latency.
        _logprobs("one_token_alternatives", "forward", "bf16", 1, 50257, True, top_k=5, temperature=0.8),
        # A few answers scored with the alternatives at each position; some tokens may never be produced.
        _logprobs("answers_scored", "forward", "bf16", 257, 32000, True, top_k=20, ignored=31, banned=100),
        # Perplexity and entropy of an evaluation batch at the GPT-2 benchmark's 16 x 1024 tokens.
        _logprobs("evaluation_batch", "forward", "bf16", 16384, 50257, True),
        # A teacher with a wide vocabulary writes its top 64 per position, from fp32 logits.
        _logprobs("teacher_alternatives", "forward", "fp32", 4096, 131072, True, top_k=64),
        # Policy-gradient step with an entropy bonus on the Llama-style micro-batch (4 x 2048), padded tail.
        _logprobs("policy_update", "train", "bf16", 8192, 32000, True, temperature=0.7, ignored=1024),
        # The same on a small vocabulary with unpadded odd rows.
        _logprobs("policy_small_vocabulary", "train", "fp16", 333, 1001, False, top_k=4),
        # A short fp32 batch with a top-8 teacher, rows weighted after the loss is known.
        _distill("distill_short_batch", "train", "fp32", 48, 4099, False, 8, False, "none", temperature=2.0, empty=5),
        # GPT-2 sized student, top-64 teacher with the rest of its mass in one bucket: the training step's loss.
        _distill("distill_full_batch", "train", "bf16", 16384, 50257, True, 64, True, "sum"),
        # Llama-style micro-batch, top-32 teacher renormalised at temperature 2, padded tail.
        _distill("distill_micro_batch", "train", "bf16", 8192, 32000, True, 32, False, "sum", temperature=2.0,
                 empty=1024),
        # Validation of a distilled student on unpadded fp16 logits: the loss alone.
        _distill("distill_validation", "forward", "fp16", 4096, 50257, False, 100, True, "none"),
        # Wide vocabulary, top-128 teacher, fp32 logits, per-row weights from autograd.
        _distill("distill_wide_vocabulary", "train", "fp32", 1024, 131072, True, 128, True, "none"),
        # fp16 training under a gradient scaler: the upstream factor arrives with the backward pass.
        _distill("distill_scaled_fp16", "train", "fp16", 2048, 50257, True, 16, False, "sum", scale=1024.0),
    ]


def _between(rng, low, high):
    """A whole number, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    path = rng.choice(["forward", "train"])
    vocab = _between(rng, 1000, 131072)
    most = (2 if dtype == "fp32" else 4) * 10 ** 8 // vocab
    rows = _between(rng, 1, min(16384, most))
    pad = rng.random() < 0.6
    temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
    left_out = rng.choice([0, 0, rows // 8])
    if rng.random() < 0.5:
        top_k = 0 if rng.random() < 0.4 else _between(rng, 1, 128)
        banned = rng.choice([0, vocab // 50])
        return _logprobs("", path, dtype, rows, vocab, pad, top_k, temperature, left_out, banned)
    reduction = "none" if path == "forward" else rng.choice(["none", "sum"])
    scale = 1024.0 if dtype == "fp16" and reduction == "sum" else 1.0
    return _distill("", path, dtype, rows, vocab, pad, _between(rng, 1, 128), rng.random() < 0.5, reduction,
                    temperature, left_out, scale)


def prepare(case, seed):
    rows, vocab = case["rows"], case["vocab"]
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=gen)

    # Logits as a trained model gives them: a broad bulk and some tokens well above it.
    ld = (vocab + 63) // 64 * 64 if case["pad"] else vocab
    logits = normal(rows, ld, dtype=DTYPES[case["dtype"]]).mul_(2.0)[:, :vocab]
    slots = case["slots"] if case["op"] == "distill" else 8
    first = torch.randint(0, vocab, (rows, 1), device="cuda", generator=gen)
    step = 7919 if vocab % 7919 else 7907
    ids = (first + step * torch.arange(slots, device="cuda")) % vocab
    likely = normal(rows, slots).sort(dim=1, descending=True).values * 2.0 + 8.0
    logits.scatter_(1, ids, (likely + 0.7 * normal(rows, slots)).to(logits.dtype))
    state = {"case": case, "logits": logits}

    if case["op"] == "logprobs":
        tokens = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
        usual = torch.rand(rows, device="cuda", generator=gen) < 0.75
        tokens = torch.where(usual, ids[:, 0], tokens)
        if case["banned"]:
            logits[:, :case["banned"]] = -math.inf
            tokens = tokens.clamp_min(case["banned"])
        if case["ignored"]:
            tokens[rows - case["ignored"]:] = IGNORE
        state["tokens"] = tokens
        if case["path"] == "train":
            state["dlogprobs"] = normal(rows) / rows
            state["dentropy"] = normal(rows) * 0.1 / rows
    else:
        teacher = likely
        if case["tail"]:  # log probabilities, with about e^8 of the mass elsewhere
            rest = normal(rows, 1) * 0.5 + 8.0
            teacher = torch.log_softmax(torch.cat([likely, rest], dim=1), dim=1)[:, :slots]
        ragged = torch.rand(rows, slots, device="cuda", generator=gen) < 0.05
        ragged[:, 0] = False
        if case["empty"]:
            ragged[rows - case["empty"]:] = True
        state["ids"] = ids.masked_fill(ragged, -1)
        state["teacher"] = teacher.contiguous()
        weight = torch.rand(rows, device="cuda", generator=gen) + 0.5
        if case["empty"]:
            weight[rows - case["empty"]:] = 0.0
        state["weight"] = weight / max(1, rows - case["empty"])
        state["scale"] = torch.full((), case["scale"], device="cuda")
    state["logits"] = logits.requires_grad_(case["path"] == "train")
    return state


# ------------------------------------------------------------- plain form


def _plain_top(logits, top_k):
    """The ``top_k`` largest per row, ties to the lowest index: keys of the value's order above the index."""
    bits = (logits.float() + 0.0).view(torch.int32)
    order = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    index = torch.arange(logits.shape[1], device=logits.device)
    keys = order.long() * 2 ** 32 + (2 ** 32 - 1 - index)
    return 2 ** 32 - 1 - (keys.topk(top_k, dim=1).values & (2 ** 32 - 1))


def _plain_logprobs(state):
    case = state["case"]
    logits, tokens = state["logits"].detach(), state["tokens"]
    counted = tokens != IGNORE
    z = logits.float() / case["temperature"]
    high = z.max(dim=1, keepdim=True).values
    logp = z - high - (z - high).exp().sum(dim=1, keepdim=True).log()
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    entropy = -plogp.sum(dim=1)
    given = tokens.clamp_min(0)[:, None]
    out = {"logprobs": torch.where(counted, logp.gather(1, given)[:, 0], 0.0),
           "entropy": torch.where(counted, entropy, 0.0)}
    if case["top_k"]:
        top = _plain_top(logits, case["top_k"])
        out["top_logprobs"] = torch.where(counted[:, None], logp.gather(1, top), 0.0)
        out["top_ids"] = torch.where(counted[:, None], top, -1)
    if case["path"] == "train":
        dlogp, dent = state["dlogprobs"][:, None], state["dentropy"][:, None]
        grad = -p * dlogp - dent * (plogp + p * entropy[:, None])
        grad.scatter_add_(1, given, dlogp)
        grad = torch.where(counted[:, None], grad / case["temperature"], 0.0)
        out["dlogits"] = grad.to(logits.dtype)
    return out


def _plain_distill(state):
    case = state["case"]
    logits, ids = state["logits"].detach(), state["ids"]
    temperature = case["temperature"]
    valid = (ids >= 0) & (ids < case["vocab"])
    some = valid.any(dim=1)
    at = torch.where(valid, ids, 0)
    t = torch.where(valid, state["teacher"].float(), -math.inf)
    if case["tail"]:
        q = t.exp()
    else:
        e = ((t - t.max(dim=1, keepdim=True).values.clamp_min(-3e38)) / temperature).exp()
        q = e / e.sum(dim=1, keepdim=True).clamp_min(1e-30)
    z = logits.float() / temperature
    high = z.max(dim=1, keepdim=True).values
    e = (z - high).exp()
    total = e.sum(dim=1, keepdim=True)
    logp = z.gather(1, at) - high - total.log()
    terms = torch.where(q > 0, q * (q.clamp_min(1e-38).log() - logp), 0.0)
    loss = terms.sum(dim=1)
    mass = q.sum(dim=1)
    inside = torch.zeros_like(e)
    if case["tail"]:
        inside.scatter_add_(1, at, valid.float())
        outside = torch.where(inside > 0, 0.0, e)
        rest = outside.sum(dim=1)
        q_rest = (1.0 - mass).clamp_min(0.0)
        p_rest = rest / total[:, 0]
        loss = loss + torch.where(q_rest > 0, q_rest * (q_rest.clamp_min(1e-38).log() - p_rest.log()), 0.0)
    loss = torch.where(some, loss, 0.0)
    if case["reduction"] == "sum":
        out = {"loss": torch.where(state["weight"] != 0, state["weight"] * loss, 0.0).sum()}
    else:
        out = {"loss": loss}
    if case["path"] == "train":
        if case["tail"]:
            grad = e * ((mass + q_rest) / total[:, 0])[:, None]
            grad = grad - outside * (q_rest / rest)[:, None]
        else:
            grad = e * (mass / total[:, 0])[:, None]
        grad = grad.scatter_add_(1, at, -q)
        factor = state["weight"] / temperature
        if case["reduction"] == "sum":
            factor = factor * state["scale"]
        grad = torch.where((some & (factor != 0))[:, None], grad * factor[:, None], 0.0)
        out["dlogits"] = grad.to(logits.dtype)
    return out


# ------------------------------------------------------- framework's calls


def _own_logprobs(state):
    from koochak_b200.ops import functional as kf

    case = state["case"]
    res = kf.token_logprobs(state["logits"], state["tokens"], top_k=case["top_k"], temperature=case["temperature"],
                            ignore_index=IGNORE)
    out = {"logprobs": res.logprobs.detach(), "entropy": res.entropy.detach()}
    if case["top_k"]:
        out["top_logprobs"] = res.top_logprobs
        out["top_ids"] = res.top_ids
    if case["path"] == "train":
        (out["dlogits"],) = torch.autograd.grad((res.logprobs, res.entropy), state["logits"],
                                                (state["dlogprobs"], state["dentropy"]))
    return out


def _own_distill(state):
    from koochak_b200.ops import functional as kf

    case = state["case"]
    summed = case["reduction"] == "sum"
    loss = kf.topk_distillation(state["logits"], state["ids"], state["teacher"], temperature=case["temperature"],
                                tail=case["tail"], weight=state["weight"] if summed else None,
                                reduction=case["reduction"])
    out = {"loss": loss.detach()}
    if case["path"] == "train":
        upstream = state["scale"] if summed else state["weight"]
        (out["dlogits"],) = torch.autograd.grad(loss, state["logits"], upstream)
    return out


def run(state):
    if state["case"]["op"] == "logprobs":
        return _own_logprobs(state) if own else _plain_logprobs(state)
    return _own_distill(state) if own else _plain_distill(state)


def work(case):
    rows, vocab = case["rows"], case["vocab"]
    item = 4 if case["dtype"] == "fp32" else 2
    logprobs = case["op"] == "logprobs"
    read = rows - (case["ignored"] if logprobs else case["empty"])  # rows left out are not looked at
    size = read * vocab * item
    flops = read * vocab * (6 if logprobs else 4)
    if logprobs:
        size += rows * (8 + 4 + 4 + 12 * case["top_k"])
    else:
        size += rows * (12 * case["slots"] + 4 + (4 if case["reduction"] == "sum" else 0))
    if case["path"] == "train":
        size += rows * vocab * item + rows * 8
        flops += read * vocab * 4
    return {"bytes": size, "flops": flops}


# ----------------------------------------------------------- 64-bit values


def _exact_logprobs(case, logits, state, part):
    tokens = state["tokens"][part]
    counted = tokens != IGNORE
    z = logits / case["temperature"]
    logp = torch.log_softmax(z, dim=1)
    entropy = torch.special.entr(logp.exp()).sum(dim=1)
    given = logp[torch.arange(len(tokens), device=logits.device), tokens.clamp_min(0)]
    out = {"logprobs": given.masked_fill(~counted, 0.0), "entropy": entropy.masked_fill(~counted, 0.0)}
    if case["top_k"]:
        order = logits.detach().sort(dim=1, descending=True, stable=True).indices[:, :case["top_k"]]
        out["top_logprobs"] = logp.gather(1, order).masked_fill(~counted[:, None], 0.0)
        out["top_ids"] = order.masked_fill(~counted[:, None], -1)
    if case["path"] == "train":
        with torch.no_grad():  # the derivatives of log p[t] and of -sum p log p, column by column
            p = logp.exp()
            hot = torch.zeros_like(p).scatter_(1, tokens.clamp_min(0)[:, None], 1.0)
            slope = torch.special.xlogy(p, p) + p * entropy[:, None]
            grad = state["dlogprobs"][part].double()[:, None] * (hot - p)
            grad -= state["dentropy"][part].double()[:, None] * slope
            out["dlogits"] = (grad / case["temperature"]).masked_fill(~counted[:, None], 0.0)
    return out


def _exact_distill(case, logits, state, part):
    ids, teacher = state["ids"][part], state["teacher"][part].double()
    weight = state["weight"][part].double()
    valid = (ids >= 0) & (ids < case["vocab"])
    with torch.enable_grad():
        z = logits.requires_grad_()
        logp = torch.log_softmax(z / case["temperature"], dim=1)
        at = logp.gather(1, ids.clamp_min(0))
        if case["tail"]:
            q = teacher.masked_fill(~valid, -math.inf).exp()
        else:
            masked = (teacher / case["temperature"]).masked_fill(~valid, -math.inf)
            q = torch.softmax(masked, dim=1).nan_to_num(0.0)
        loss = (torch.special.xlogy(q, q) - torch.where(valid, q * at, 0.0)).sum(dim=1)
        if case["tail"]:
            known = torch.zeros_like(logp).scatter_add_(1, ids.clamp_min(0), valid.double()) > 0
            rest = logp.masked_fill(known, -math.inf).logsumexp(dim=1)
            q_rest = (1.0 - q.sum(dim=1)).clamp_min(0.0)
            loss = loss + torch.special.xlogy(q_rest, q_rest) - q_rest * rest
        loss = torch.where(valid.any(dim=1), loss, 0.0)
        out = {"loss": loss.detach()}
        if case["reduction"] == "sum":
            loss = weight * loss
            out["loss"] = loss.detach()
            upstream = torch.full_like(loss, case["scale"])
        else:
            upstream = weight
        if case["path"] == "train":
            (out["dlogits"],) = torch.autograd.grad(loss, z, upstream)
    return out


def exact(case, seed):
    state = prepare(case, seed)
    logits = state["logits"].detach()
    kind = _exact_logprobs if case["op"] == "logprobs" else _exact_distill
    at_once = max(1, 2 ** 26 // case["vocab"])
    parts = []
    for low in range(0, case["rows"], at_once):
        part = slice(low, min(case["rows"], low + at_once))
        parts.append(kind(case, logits[part].double(), state, part))
    out = {key: torch.cat([p[key] for p in parts]) for key in parts[0]}
    if case["op"] == "distill" and case["reduction"] == "sum":
        out["loss"] = out["loss"].sum()
    return out
