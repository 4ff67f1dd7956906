"""The language-model operators next to the draft head's losses, over the sizes that a program meets.

  logprobs   log-probabilities of given tokens, entropy and the K best alternatives of each row of
             logits (`aspec_amd.token_logprobs.token_logprobs`), alone or with the backward to the
             logits
  distill    cross-entropy and the KL divergence from a teacher of which the K best tokens'
             log-probabilities were kept (`aspec_amd.topk_distill`): forward, forward + backward
             ("autograd"), or losses and gradient in one pass ("fused")

`listed()` gives the standing cases and `draw()` more of the same ranges. `prepare()` makes what a
program holds before the call, `run()` is one pass (the plain form in torch, or, with `own`, the
framework's call), `work()` what the pass cannot do without, `exact()` the same results in 64 bits.
"""

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
IGNORE = -100
NO_TAIL = 2.0 ** -20   # a teacher's remaining mass up to this is the rounding of its log-probabilities
MOST = 8192 * 32000    # logits in the largest case


# ---- the cases -----------------------------------------------------------------------------------
def _logprobs(name, rows, vocab, dtype, top_k, *, temperature=1.0, backward=False, pad=0, masked=0):
    """`pad` unused columns behind each row (a row stride of vocab + pad), `masked` columns at the
    vocabulary's end whose logits are -inf (an output layer rounded up in size)."""
    return {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "top_k": top_k,
            "temperature": temperature, "backward": backward, "pad": pad, "masked": masked}


def _distill(name, rows, vocab, dtype, kept, path, *, teacher_rows=0, tail="bucket", temperature=1.0, pad=0):
    """`kept` teacher tokens per row; `teacher_rows` > 0: a table of that many teacher rows, addressed
    per draft row."""
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "kept": kept,
            "path": path, "teacher_rows": teacher_rows, "tail": tail, "temperature": temperature, "pad": pad}


def listed():
    return [
        # Serving, one token: the row of the full target vocabulary with the 20 alternatives that an
        # API returns. Latency.
        _logprobs("logprobs_one_row", 1, 151936, "bf16", 20),
        # Verifying one block of 16 draft tokens over the draft vocabulary at a temperature. Latency.
        _logprobs("logprobs_draft_block", 16, 32000, "f16", 5, temperature=0.7),
        # The teacher's pass over a 4096-token document: the 64 best tokens of each position are what
        # a distillation cache keeps.
        _logprobs("logprobs_teacher_cache", 4096, 32000, "bf16", 64, masked=24),
        # Scoring a batch from fp32 logits of the full vocabulary.
        _logprobs("logprobs_score_f32", 1536, 151936, "f32", 8),
        # Policy-gradient training on all draft positions of a 4096-token row: log-probability and
        # entropy with their gradient.
        _logprobs("logprobs_train", 8192, 32000, "bf16", 0, backward=True),
        # An odd vocabulary in rows padded to a multiple of 64, gradients through the alternatives too.
        _logprobs("logprobs_odd_f16", 509, 50021, "f16", 37, backward=True, pad=27),
        # One draft block's loss and gradient. Latency.
        _distill("distill_draft_block", 16, 32000, "bf16", 16, "autograd"),
        # The head's objective on all draft positions of a 4096-token row, teacher rows by position.
        _distill("distill_head_fused", 8192, 32000, "bf16", 64, "fused", teacher_rows=4096),
        # The same through autograd at a temperature, from the kept tokens alone.
        _distill("distill_head_autograd", 8192, 32000, "bf16", 64, "autograd", teacher_rows=4096,
                 tail="renormalize", temperature=2.0),
        # The full target vocabulary, a chunk of rows, a wide teacher.
        _distill("distill_full_vocab", 1536, 151936, "bf16", 128, "fused"),
        # Odd sizes everywhere in fp16, rows padded.
        _distill("distill_odd_f16", 1021, 30011, "f16", 7, "autograd", teacher_rows=333, pad=5),
        # Evaluation from fp32 logits: losses and acceptance without a gradient.
        _distill("distill_eval_f32", 1024, 65536, "f32", 32, "forward"),
    ]


def _log_uniform(rng, low, high):
    return int(round(low * (high / low) ** rng.random()))


def draw(rng):
    vocab = min(_log_uniform(rng, 257, 152064), 152064)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    most = MOST // (2 if dtype == "f32" else 1)
    rows = min(_log_uniform(rng, 1, 8192), most // (vocab + 64))
    temperature = rng.choice([1.0, 1.0, 0.6, 2.0])
    pad = rng.choice([0, 0, rng.randrange(1, 64)])
    if rng.random() < 0.5:
        case = _logprobs("", rows, vocab, dtype, rng.choice([0, 1, rng.randrange(2, 129)]), temperature=temperature,
                         backward=rng.random() < 0.5, pad=pad, masked=rng.choice([0, rng.randrange(1, 100)]))
    else:
        path = rng.choice(["autograd", "fused", "forward"])
        case = _distill("", rows, vocab, dtype, _log_uniform(rng, 1, 128), path,
                        teacher_rows=rng.choice([0, max(1, rows // 2)]), tail=rng.choice(["bucket", "renormalize"]),
                        temperature=temperature, pad=pad)
    del case["name"]
    return case


# ---- what a program holds before the call --------------------------------------------------------
def _padded(x, pad):
    """x [rows, vocab] as a view of rows that are `pad` columns longer."""
    if not pad:
        return x
    buffer = torch.zeros(x.shape[0], x.shape[1] + pad, dtype=x.dtype, device=x.device)
    buffer[:, :x.shape[1]] = x
    return buffer[:, :x.shape[1]]


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    def whole(high, *shape):
        return torch.randint(0, high, shape, device=DEV, generator=g)

    state = {"case": case}
    if case["op"] == "logprobs":
        # rows from flat to confident: a spread of scales, and one token well ahead in most rows
        x = normal(rows, vocab).mul_(1.0 + 2.0 * torch.rand(rows, 1, device=DEV, generator=g))
        ids = whole(vocab - case["masked"], rows)
        x.scatter_add_(1, ids[:, None], 12.0 * torch.rand(rows, 1, device=DEV, generator=g))
        if case["masked"]:
            x[:, vocab - case["masked"]:] = -float("inf")
        ids = torch.where(torch.rand(rows, device=DEV, generator=g) < 0.25, whole(vocab - case["masked"], rows), ids)
        state["x"], state["ids"] = _padded(x.to(dtype), case["pad"]), ids
        state["grads"] = [normal(rows), 0.1 * normal(rows)]
        if case["top_k"]:
            state["grads"].append(normal(rows, case["top_k"]))
        state["x"].requires_grad_(case["backward"])
        return state
    trows, kept = case["teacher_rows"] or rows, case["kept"]
    z = normal(trows, vocab).mul_(2.0)
    best = whole(vocab, trows, 8)
    z.scatter_add_(1, best, 10.0 * torch.rand(trows, 8, device=DEV, generator=g))
    state["teacher_rows"] = whole(trows, rows) if case["teacher_rows"] else None
    # what a cache keeps: the best tokens of the teacher's row at the temperature, in some rows fewer
    # than there is room for (the others are -1)
    scaled = z / case["temperature"]
    top = torch.topk(scaled, kept, dim=-1)
    logprobs = top.values - torch.logsumexp(scaled, dim=-1, keepdim=True)
    del scaled
    fewer = torch.arange(kept, device=DEV)[None] >= 1 + (kept * 2.0 * torch.rand(trows, 1, device=DEV, generator=g)).long()
    state["teacher_indices"] = torch.where(fewer, -1, top.indices)
    state["teacher_logprobs"] = torch.where(fewer, -float("inf"), logprobs)
    x = z[state["teacher_rows"]] if case["teacher_rows"] else z
    x = x.add_(normal(rows, vocab))
    state["x"] = _padded(x.to(dtype), case["pad"]).requires_grad_(case["path"] == "autograd")
    targets = whole(vocab, rows)
    state["targets"] = torch.where(torch.rand(rows, device=DEV, generator=g) < 0.1, IGNORE, targets)
    # the objective's per-row weights: 0 for a row that is masked out
    live = torch.rand(rows, device=DEV, generator=g) > 0.1
    state["ce_weights"] = 0.1 * torch.rand(rows, device=DEV, generator=g) * live
    state["kl_weights"] = 0.9 * torch.rand(rows, device=DEV, generator=g) * live
    return state


# ---- the plain forms -----------------------------------------------------------------------------
def _softmax(x):
    """(p, log p, e, sum e) of rows in 32 bits."""
    m = x.max(dim=-1, keepdim=True).values
    e = torch.exp(x - m)
    total = e.sum(dim=-1, keepdim=True)
    return e / total, x - m - torch.log(total), e, total


def _top(x, k):
    """Indices of each row's k largest values, ties to the lowest index: the value's bits as an
    ordered whole number, the index below them."""
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = order * 2 ** 24 + (2 ** 24 - 1 - torch.arange(x.shape[-1], device=x.device))
    return (2 ** 24 - 1) - (torch.topk(key, k, dim=-1).values & (2 ** 24 - 1))


def _plain_logprobs(s):
    case, x = s["case"], s["x"].detach().float()
    temperature, k = case["temperature"], case["top_k"]
    p, logp, _, _ = _softmax(x / temperature)
    plogp = torch.where(p > 0, p * logp, 0.0)
    chosen = logp.gather(1, s["ids"][:, None]).squeeze(1)
    entropy = -plogp.sum(dim=-1)
    out = {"logprobs": chosen, "entropy": entropy}
    if k:
        indices = _top(x, k)
        out["top_logprobs"], out["top_indices"] = logp.gather(1, indices), indices
    if case["backward"]:
        g_chosen, g_entropy = s["grads"][0], s["grads"][1]
        lost = g_chosen + (s["grads"][2].sum(dim=-1) if k else 0.0)
        grad = -lost[:, None] * p - g_entropy[:, None] * (plogp + entropy[:, None] * p)
        grad.scatter_add_(1, s["ids"][:, None], g_chosen[:, None])
        if k:
            grad.scatter_add_(1, indices, s["grads"][2])
        out["grad"] = (grad / temperature).to(s["x"].dtype)
    return out


def _plain_distill(s):
    case, x = s["case"], s["x"].detach().float()
    rows, vocab, temperature = case["rows"], case["vocab"], case["temperature"]
    index, teacher = s["teacher_indices"], s["teacher_logprobs"]
    if s["teacher_rows"] is not None:
        index, teacher = index[s["teacher_rows"]], teacher[s["teacher_rows"]]
    used = index >= 0
    q = torch.where(used, torch.exp(teacher.double()), 0.0)  # 64 bits: 1 - sum q is small
    mass = q.sum(dim=-1, keepdim=True)
    if case["tail"] == "renormalize":
        q, rest = q / mass, torch.zeros_like(mass)
    else:
        rest = (1.0 - mass).clamp(min=0.0)
        rest = torch.where(rest <= NO_TAIL, 0.0, rest)
    q, rest = q.float(), rest.float()
    mass = q.sum(dim=-1, keepdim=True)
    p, logp, e, total = _softmax(x / temperature)
    # column `vocab` takes the unused slots
    slot = torch.where(used, index, vocab)
    kept = torch.zeros(rows, vocab + 1, dtype=torch.bool, device=x.device).scatter_(1, slot, True)[:, :vocab]
    tail = torch.where(kept, 0.0, e).sum(dim=-1, keepdim=True) / total
    at = slot.clamp(max=vocab - 1)
    p_at, logp_at = p.gather(1, at), logp.gather(1, at)
    some = rest > 0
    kl = torch.where(q > 0, q * (torch.log(torch.where(q > 0, q, 1.0)) - logp_at), 0.0).sum(dim=-1)
    kl = kl + torch.where(some, rest * (torch.log(torch.where(some, rest, 1.0)) - torch.log(tail)), 0.0).squeeze(1)
    accept = torch.where(used, torch.minimum(p_at, q), 0.0).sum(dim=-1) + torch.minimum(rest, tail).squeeze(1)
    hard = s["targets"] != IGNORE
    label = s["targets"].clamp(min=0)[:, None]
    p_one, logp_one = (p, logp) if temperature == 1.0 else _softmax(x)[:2]
    ce = torch.where(hard, -logp_one.gather(1, label).squeeze(1), 0.0)
    out = {"ce": ce, "kl": kl, "accept_rate": accept}
    if case["path"] != "forward":
        g_kl = s["kl_weights"][:, None] / temperature
        g_ce = torch.where(hard, s["ce_weights"], 0.0)[:, None]
        outside = torch.where(some, 1.0 - rest / (mass + rest) / tail, 1.0) * (mass + rest)
        grad = torch.empty(rows, vocab + 1, dtype=torch.float32, device=x.device)
        grad[:, :vocab] = g_kl * p * torch.where(kept, mass + rest, outside) + g_ce * p_one
        grad.scatter_add_(1, slot, -g_kl * q)
        grad.scatter_add_(1, label, -g_ce)
        out["grad"] = grad[:, :vocab].to(s["x"].dtype)
    return out


# ---- the framework's calls -----------------------------------------------------------------------
def _own_logprobs(s):
    from aspec_amd.token_logprobs import token_logprobs

    case = s["case"]
    # scoring alone: the ids come from the program's own sampling, so nothing waits for their check
    got = token_logprobs(s["x"], s["ids"], top_k=case["top_k"], temperature=case["temperature"],
                         check_ids=case["backward"])
    out = {"logprobs": got.logprobs, "entropy": got.entropy}
    if case["top_k"]:
        out["top_logprobs"], out["top_indices"] = got.top_logprobs, got.top_indices
    if case["backward"]:
        losses = [got.logprobs, got.entropy] + ([got.top_logprobs] if case["top_k"] else [])
        out["grad"] = torch.autograd.grad(losses, s["x"], s["grads"])[0]
        out = {k: v.detach() for k, v in out.items()}
    return out


def _own_distill(s):
    from aspec_amd.topk_distill import topk_distill_from_logits, topk_distill_fused_grad

    case = s["case"]
    args = (s["x"], s["targets"], s["teacher_indices"], s["teacher_logprobs"])
    more = {"teacher_rows": s["teacher_rows"], "tail": case["tail"], "temperature": case["temperature"]}
    if case["path"] == "fused":
        ce, kl, accept, grad = topk_distill_fused_grad(*args, ce_weights=s["ce_weights"], kl_weights=s["kl_weights"],
                                                       **more)
        return {"ce": ce, "kl": kl, "accept_rate": accept, "grad": grad}
    ce, kl, accept = topk_distill_from_logits(*args, **more)
    out = {"ce": ce.detach(), "kl": kl.detach(), "accept_rate": accept}
    if case["path"] == "autograd":
        out["grad"] = torch.autograd.grad([ce, kl], s["x"], [s["ce_weights"], s["kl_weights"]])[0]
    return out


def run(state):
    if state["case"]["op"] == "logprobs":
        return _own_logprobs(state) if own else _plain_logprobs(state)
    return _own_distill(state) if own else _plain_distill(state)


# ---- the work ------------------------------------------------------------------------------------
def work(case):
    rows, vocab, size = case["rows"], case["vocab"], DTYPES[case["dtype"]].itemsize
    logits = rows * vocab
    if case["op"] == "logprobs":
        k, grad = case["top_k"], case["backward"]
        small = rows * (8 + 8 + 12 * k) + (rows * (8 + 4 * k) if grad else 0)
        # maximum, difference, exponential, sum, entropy's product and sum; the gradient's as many
        return {"bytes": logits * size * (2 if grad else 1) + small, "flops": logits * (12 if grad else 6)}
    grad = case["path"] != "forward"
    pairs = (case["teacher_rows"] or rows) * case["kept"]
    small = 12 * pairs + rows * (8 + 12 + (8 if case["teacher_rows"] else 0) + (8 if grad else 0))
    return {"bytes": logits * size * (2 if grad else 1) + small, "flops": logits * (8 if grad else 4)}


# ---- the definition in 64 bits -------------------------------------------------------------------
def _exact_logprobs(s, a, b):
    case, k = s["case"], s["case"]["top_k"]
    x = s["x"].detach()[a:b].double().requires_grad_(True)
    logp = torch.log_softmax(x / case["temperature"], dim=-1)
    finite = torch.where(torch.isinf(logp), 0.0, logp)
    out = {"logprobs": logp[torch.arange(b - a, device=x.device), s["ids"][a:b]],
           "entropy": -(torch.exp(logp) * finite).sum(dim=-1)}
    if k:
        out["top_indices"] = torch.sort(x.detach(), dim=-1, descending=True, stable=True).indices[:, :k].contiguous()
        out["top_logprobs"] = torch.take_along_dim(logp, out["top_indices"], dim=-1)
    if case["backward"]:
        total = (out["logprobs"] * s["grads"][0][a:b]).sum() + (out["entropy"] * s["grads"][1][a:b]).sum()
        if k:
            total = total + (out["top_logprobs"] * s["grads"][2][a:b]).sum()
        out["grad"] = torch.autograd.grad(total, x)[0]
    return out


def _exact_distill(s, a, b):
    case = s["case"]
    x = s["x"].detach()[a:b].double().requires_grad_(True)
    at = s["teacher_rows"][a:b] if s["teacher_rows"] is not None else torch.arange(a, b, device=x.device)
    index, logq = s["teacher_indices"][at], s["teacher_logprobs"][at].double()
    used = (index >= 0) & (logq > -float("inf"))
    if case["tail"] == "renormalize":
        logq = logq - torch.logsumexp(logq.masked_fill(~used, -float("inf")), dim=-1, keepdim=True)
    logq = logq.masked_fill(~used, 0.0)
    q = torch.exp(logq) * used
    logp = torch.log_softmax(x / case["temperature"], dim=-1)
    where = index.clamp(min=0)
    logp_at = torch.take_along_dim(logp, where, dim=-1)
    kl = (q * (logq - logp_at)).sum(dim=-1)
    # every teacher token's probability, for the tokens outside and the overlap
    drop = torch.zeros_like(logp, dtype=torch.bool)
    rows, slots = (index >= 0).nonzero(as_tuple=True)
    drop[rows, index[rows, slots]] = True
    log_tail = torch.logsumexp(logp.masked_fill(drop, -float("inf")), dim=-1)
    accept = (torch.minimum(q, torch.exp(logp_at)) * used).sum(dim=-1)
    if case["tail"] == "bucket":
        rest = 1.0 - q.sum(dim=-1)
        rest = rest * (rest > NO_TAIL)
        kl = kl + rest * (torch.log(rest.clamp(min=NO_TAIL)) - torch.where(rest > 0, log_tail, 0.0))
        accept = accept + torch.minimum(rest, torch.exp(log_tail))
    ce = torch.nn.functional.cross_entropy(x, s["targets"][a:b], reduction="none", ignore_index=IGNORE)
    out = {"ce": ce, "kl": kl, "accept_rate": accept}
    if case["path"] != "forward":
        total = (ce * s["ce_weights"][a:b]).sum() + (kl * s["kl_weights"][a:b]).sum()
        out["grad"] = torch.autograd.grad(total, x)[0]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    part = _exact_logprobs if case["op"] == "logprobs" else _exact_distill
    step = max(1, 2 ** 24 // case["vocab"])
    parts = [part(state, a, min(a + step, case["rows"])) for a in range(0, case["rows"], step)]
    # in the order of `run`'s outputs
    names = [n for n in ("logprobs", "entropy", "top_logprobs", "top_indices", "ce", "kl", "accept_rate", "grad")
             if n in parts[0]]
    return {n: torch.cat([p[n].detach() for p in parts]) for n in names}
