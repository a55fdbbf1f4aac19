"""Cases of the operators on the output head's logits, and their plain forms.

  token_logprobs          log probabilities of given tokens, the entropy of every row and its top
                          alternatives; with gradients for training on them
  topk_distillation_loss  distillation from a teacher's top logits, forward and backward

`own` selects the package's operators; otherwise `run` computes the plain form: elementary torch
operations in 32 bits on whatever type the logits have, rounded once at the end.

A case: `op` ("score": forward of token_logprobs, "policy": its forward and backward, "distill":
the distillation loss, with its backward where `grad`), `b` sequences of `n` positions over `v`
columns, `dtype` of the logits, `k` alternatives or teacher entries, `temperature`, and
  view    "plain": contiguous logits; "shift": logits[:, :-1] of n + 1 positions (the next-token
          shift); "pad": rows of a wider, padded buffer
  masked  share of the positions that the mask leaves out
  banned  some columns hold -inf (tokens that a sampler excluded)
  ragged  teacher rows of different lengths, the rest filled up with id -1
"""
import math

import torch

own = False


def _case(name, op, b, n, v, dtype="bf16", k=0, temperature=1.0, view="plain", masked=0.0, banned=False,
          ragged=False, grad=False):
    c = {"op": op, "b": b, "n": n, "v": v, "dtype": dtype, "k": k, "temperature": temperature, "view": view,
         "masked": masked, "banned": banned, "ragged": ragged, "grad": grad}
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # one sampled token's record: its log probability and eight alternatives (latency)
        _case("score_one_token", "score", 1, 1, 128256, k=8),
        # the tokens of one step of a batch in generation, sampled at a temperature with banned tokens
        _case("score_decode_batch", "score", 48, 1, 128256, k=20, temperature=0.8, banned=True),
        # prompts scored for evaluation: the shifted view of the logits, no alternatives
        _case("score_prompt", "score", 2, 1024, 128256, view="shift"),
        # a teacher's targets for distillation: its top logits at every position
        _case("teacher_targets", "score", 4, 1024, 128256, k=64),
        # an odd vocabulary in f32: rows start at every alignment
        _case("score_odd_f32", "score", 3, 259, 50257, dtype="f32", k=5, temperature=0.7, masked=0.2),
        # policy training on a short rollout (small call, f32)
        _case("policy_small", "policy", 4, 16, 32000, dtype="f32", masked=0.25, grad=True),
        # policy training with an entropy bonus on a batch of rollouts, prompts masked out
        _case("policy_step", "policy", 8, 512, 128256, masked=0.25, grad=True),
        # distillation on a few positions (small call)
        _case("distill_few", "distill", 1, 7, 32000, k=16, grad=True),
        # odd vocabulary, f32, softened targets, teacher rows of different lengths
        _case("distill_odd_f32", "distill", 5, 211, 50257, dtype="f32", k=33, temperature=2.0, ragged=True, grad=True),
        # the loss alone, on held-out data, from a padded lm_head
        _case("distill_eval", "distill", 2, 1000, 128255, k=20, view="pad"),
        # a distillation step with padded positions masked out
        _case("distill_step", "distill", 4, 1024, 128256, k=64, masked=0.1, grad=True),
        # the largest distillation step
        _case("distill_large", "distill", 2, 4096, 128256, k=32, grad=True),
    ]


def draw(rng):
    op = rng.choice(["score", "score", "policy", "distill", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    v = int(round(math.exp(rng.uniform(math.log(1000), math.log(131072)))))
    rows = math.exp(rng.uniform(0.0, math.log(min(8192, 2 ** 29 / v))))
    b = rng.choice([1, 2, 3, 4])
    n = max(1, int(rows / b))
    k = int(round(math.exp(rng.uniform(0.0, math.log(128)))))
    if op == "policy" or (op == "score" and rng.random() < 0.25):
        k = 0
    return _case(None, op, b, n, v, dtype=dtype, k=k, temperature=rng.choice([1.0, 0.6, 0.9, 1.5, 2.0]),
                 view=rng.choice(["plain", "plain", "shift", "pad"]), masked=rng.choice([0.0, 0.0, 0.1, 0.4]),
                 banned=op == "score" and rng.random() < 0.3, ragged=op == "distill" and rng.random() < 0.5,
                 grad=op == "policy" or (op == "distill" and rng.random() < 0.7))


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    b, n, v, k, dt = case["b"], case["n"], case["v"], case["k"], _dtype(case)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=dev)

    buf = torch.randn((b, n + (case["view"] == "shift"), (v // 16 + 1) * 16 if case["view"] == "pad" else v),
                      generator=g, device=dev, dtype=dt)
    buf.mul_(2.5)
    logits = buf[:, :n, :v]
    # peaks: columns start, start + step, ... (distinct), the first ones far above the rest
    peaks = max(k, 8)
    start = (uniform(b, n, 1) * v).long().clamp_(max=v - 1)
    step = 1 + (uniform(b, n, 1) * (v // peaks - 1)).long()
    cols = (start + step * torch.arange(peaks, device=dev)) % v
    height = 9.0 - 0.25 * torch.arange(peaks, device=dev) + torch.randn((b, n, peaks), generator=g, device=dev)
    logits.scatter_(2, cols, height.to(dt))
    state = {"case": case, "temperature": case["temperature"], "k": k}
    if case["banned"]:
        bans = (uniform(b, n, 200) * v).long().clamp_(max=v - 1)
        logits.scatter_(2, bans, float("-inf"))
    state["mask"] = uniform(b, n) >= case["masked"] if case["masked"] else None
    if case["op"] == "distill":
        state["ids"] = cols[..., :k].contiguous()
        teacher = 10.0 - 0.3 * torch.arange(k, device=dev) + 1.5 * torch.randn((b, n, k), generator=g, device=dev)
        state["teacher"] = teacher.sort(dim=-1, descending=True).values
        if case["ragged"]:
            length = (uniform(b, n, 1) * (k + 1)).long()  # 0 to k entries
            state["ids"].masked_fill_(torch.arange(k, device=dev) >= length, -1)
    else:
        pick = (uniform(b, n, 1) ** 3 * peaks).long().clamp_(max=peaks - 1)
        state["tokens"] = cols.gather(2, pick)[..., 0]
        if case["banned"]:  # a sampled token is never a banned one
            logits.scatter_(2, state["tokens"][..., None], 8.0)
    if case["grad"]:
        state["dloss"] = torch.randn((b, n), generator=g, device=dev) * 0.5
        state["dentropy"] = torch.full((b, n), 0.01, device=dev)
    # the logits are a value of the user's program: a leaf that asks for its gradient
    state["logits"] = logits.requires_grad_(True) if case["grad"] else logits
    return state


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    op, logits, mask, temp = state["case"]["op"], state["logits"], state["mask"], state["temperature"]
    if op == "distill":
        from macrogpt_jax_b200.distill import topk_distillation_loss
        loss = topk_distillation_loss(logits, state["ids"], state["teacher"], temperature=temp, mask=mask)
        if not state["case"]["grad"]:
            return {"loss": loss}
        (dlogits,) = torch.autograd.grad(loss, logits, state["dloss"])
        return {"loss": loss.detach(), "dlogits": dlogits}
    from macrogpt_jax_b200.logprobs import token_logprobs
    out = token_logprobs(logits, state["tokens"], top_k=state["k"], temperature=temp, mask=mask)
    if op == "policy":
        (dlogits,) = torch.autograd.grad((out.logprob, out.entropy), logits, (state["dloss"], state["dentropy"]))
        return {"logprob": out.logprob.detach(), "entropy": out.entropy.detach(), "dlogits": dlogits}
    res = {"logprob": out.logprob, "entropy": out.entropy}
    if state["k"]:
        res["top_logprobs"], res["top_ids"] = out.top_logprobs, out.top_ids
    return res


def _top_columns(x, k):
    """The k largest of every row, ties to the lowest column: one whole number per element orders
    by value first, then by column."""
    bits = (x + 0.0).view(torch.int32).to(torch.int64)  # + 0.0: one zero
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    order = order * 2 ** 32 + (2 ** 32 - 1 - torch.arange(x.shape[-1], device=x.device))
    best = order.topk(k, dim=-1).values
    return 2 ** 32 - 1 - (best & 0xFFFFFFFF)


def _run_plain(state):
    case, mask = state["case"], state["mask"]
    logits = state["logits"].detach()
    x = logits.to(torch.float32)
    y = x / state["temperature"]
    m = y.max(dim=-1, keepdim=True).values
    e = torch.exp(y - m)
    s = e.sum(dim=-1, keepdim=True)
    lse = m + torch.log(s)
    keep = None if mask is None else mask.to(torch.float32)
    if case["op"] == "distill":
        ids, t = state["ids"], state["teacher"] / state["temperature"]
        valid = ids >= 0
        t = torch.where(valid, t, float("-inf"))
        tm = t.max(dim=-1, keepdim=True).values
        tm = torch.where(torch.isinf(tm), 0.0, tm)
        te = torch.exp(t - tm)
        ts = te.sum(dim=-1, keepdim=True).clamp_(min=1e-30)
        q = te / ts
        logq = torch.where(valid, t - tm - torch.log(ts), 0.0)
        logp = y.gather(2, ids.clamp(min=0)) - lse
        loss = torch.where(valid, q * (logq - logp), 0.0).sum(dim=-1)
        if keep is not None:
            loss = loss * keep
        if not case["grad"]:
            return {"loss": loss}
        g = state["dloss"] if keep is None else state["dloss"] * keep
        g = (g / state["temperature"])[..., None]
        any_entry = valid.any(dim=-1, keepdim=True).to(torch.float32)
        d = e.div_(s).mul_(g * any_entry)
        d.scatter_add_(2, ids.clamp(min=0), -g * q)
        return {"loss": loss, "dlogits": d.to(logits.dtype)}
    tokens = state["tokens"][..., None]
    logprob = (y.gather(2, tokens) - lse)[..., 0]
    z = (y - m).clamp_(min=-200.0)  # exp is 0 there, and 0 times the clamped value is 0
    entropy = (torch.log(s) - (e * z).sum(dim=-1, keepdim=True) / s)[..., 0]
    res = {"logprob": logprob, "entropy": entropy}
    if case["op"] == "policy":
        g, h = state["dloss"], state["dentropy"]
        if keep is not None:
            g, h = g * keep, h * keep
        g, h = (g / state["temperature"])[..., None], (h / state["temperature"])[..., None]
        p = e.div_(s)
        logp = z.sub_(torch.log(s))
        d = logp.add_(entropy[..., None]).mul_(h).add_(g).mul_(p).neg_()
        d.scatter_add_(2, tokens, g.expand(tokens.shape))
        res["dlogits"] = d.to(logits.dtype)
    elif case["k"]:
        top = _top_columns(x, case["k"])
        res["top_logprobs"], res["top_ids"] = y.gather(2, top) - lse, top
    if keep is not None:
        res["logprob"], res["entropy"] = logprob * keep, entropy * keep
        if case["op"] == "score" and case["k"]:
            res["top_logprobs"] = torch.where(mask[..., None], res["top_logprobs"], float("-inf"))
            res["top_ids"] = torch.where(mask[..., None], res["top_ids"], -1)
    return res


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    rows, v, k = case["b"] * case["n"], case["v"], case["k"]
    kept = rows * (1.0 - case["masked"])
    nbytes = kept * v * es  # the logits of the rows that count, once
    flops = kept * v * (3 if case["op"] == "distill" else 5)  # scale, exp, sum (and its product with y)
    if case["op"] == "distill":
        nbytes += rows * (k * 12 + 4)  # teacher ids and logits, the loss
    else:
        nbytes += rows * (8 + 8 + 12 * k)  # token, log probability, entropy, alternatives
    if case["grad"]:
        nbytes += rows * v * es + rows * 4  # the gradient, zero rows included
        flops += kept * v * (4 if case["op"] == "policy" else 2)
    return {"bytes": nbytes, "flops": flops}


def exact(case, seed):
    """The definitions in 64 bits, a block of positions at a time."""
    st = prepare(case, seed)
    t = st["temperature"]
    b, n, v, k = case["b"], case["n"], case["v"], case["k"]
    logits = st["logits"].detach()
    block = max(1, 2 ** 26 // v)
    out = {}

    def put(name, i, sl, value):
        if name not in out:
            out[name] = torch.empty((b, n) + tuple(value.shape[1:]), dtype=value.dtype, device=value.device)
        out[name][i, sl] = value

    for i in range(b):
        for p0 in range(0, n, block):
            sl = slice(p0, min(p0 + block, n))
            rows = logits[i, sl].to(torch.float64)
            keep = torch.ones(rows.shape[0], dtype=torch.bool, device=rows.device)
            if st["mask"] is not None:
                keep = st["mask"][i, sl]
            logp = torch.log_softmax(rows / t, dim=-1)
            prob = logp.exp()
            if case["op"] == "distill":
                ids = st["ids"][i, sl]
                dense = torch.zeros_like(prob)
                has = ids >= 0
                teacher = st["teacher"][i, sl].to(torch.float64) / t
                teacher = teacher.masked_fill(~has, float("-inf"))
                q = torch.nan_to_num(torch.softmax(teacher, dim=-1), nan=0.0)
                picked = logp.gather(1, ids.clamp(min=0))
                put("loss", i, sl, torch.where(keep, (torch.special.xlogy(q, q) - q * picked).sum(dim=-1), 0.0))
                if case["grad"]:
                    dense.scatter_add_(1, ids.clamp(min=0), q)
                    w = (st["dloss"][i, sl].to(torch.float64) * keep / t)[:, None]
                    put("dlogits", i, sl, w * (prob * has.any(dim=-1, keepdim=True) - dense))
                continue
            tok = st["tokens"][i, sl][:, None]
            ent = -torch.where(prob > 0, prob * logp, 0.0).sum(dim=-1)
            put("logprob", i, sl, torch.where(keep, logp.gather(1, tok)[:, 0], 0.0))
            put("entropy", i, sl, torch.where(keep, ent, 0.0))
            if case["op"] == "policy":
                wl = (st["dloss"][i, sl].to(torch.float64) * keep / t)[:, None]
                we = (st["dentropy"][i, sl].to(torch.float64) * keep / t)[:, None]
                d = -prob * (wl + we * (torch.where(prob > 0, logp, 0.0) + ent[:, None]))
                d.scatter_add_(1, tok, wl)
                put("dlogits", i, sl, d)
            elif k:
                top = torch.sort(rows, dim=-1, descending=True, stable=True).indices[:, :k]
                put("top_logprobs", i, sl, torch.where(keep[:, None], logp.gather(1, top), float("-inf")))
                put("top_ids", i, sl, torch.where(keep[:, None], top, -1))
    return out
