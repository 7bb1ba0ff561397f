"""What is measured of the token objectives: scoring label tokens against a model's logits, and distilling from a teacher's top logits.

Both work on what the collator hands out: ``labels`` (batch, positions), ragged, padded with -100, beside logits
(batch, positions, vocabulary).  A case is a dict of plain values:

  op      "score"          logprobs of the labels, entropy, top alternatives (top = 0: none)
          "score_train"    logprobs and entropy, and the gradient of the logits from upstream gradients of both
          "distill"        mean distillation loss and the gradient of the logits
          "distill_each"   one loss per position, and the gradient from upstream weights per position
  batch, positions, vocab  logits are (batch, positions, vocab)
  dtype                    of the logits and of their gradient
  ragged                   clips have between a quarter and all of the positions; the rest of the labels is -100
  shifted                  logits are the first ``positions`` of ``positions + 1`` (a view whose batch stride is larger)
  suppressed               share of the vocabulary whose logits are -inf (tokens that decoding rules out)
  top                      alternatives returned / teacher entries kept
  temperature, alpha       of the softmax / the weight of the teacher's term
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(name, op, batch, positions, vocab, dtype, ragged=True, shifted=False, suppressed=0.0, top=0, temperature=1.0, alpha=0.5):
    return {"name": name, "op": op, "batch": batch, "positions": positions, "vocab": vocab, "dtype": dtype, "ragged": ragged,
            "shifted": shifted, "suppressed": suppressed, "top": top, "temperature": temperature, "alpha": alpha}


def listed():
    return [
        # one decoding step of one clip: a single row, its confidence and best continuations, some tokens ruled out
        _case("step of one clip", "score", 1, 1, 50021, "bf16", ragged=False, suppressed=0.002, top=8),
        # one decoding step of a batch of clips
        _case("step of 64 clips", "score", 64, 1, 50021, "fp16", ragged=False, suppressed=0.002, top=16, temperature=0.7),
        # an evaluation batch: how sure the model was of the reference transcripts (no alternatives)
        _case("evaluation batch", "score", 48, 64, 50021, "bf16"),
        # the teacher's pass over a batch of 256 clips whose alternatives go to the feature cache
        _case("teacher pass", "score", 256, 64, 50021, "bf16", top=16),
        # the same for long transcripts, in 32 bits, many alternatives kept
        _case("teacher pass, long", "score", 16, 1024, 32000, "fp32", top=64),
        # training on scores (logprobs and entropy have gradients), small and ordinary
        _case("score training, small", "score_train", 8, 48, 10000, "fp32"),
        _case("score training", "score_train", 32, 128, 32000, "bf16", shifted=True),
        # distillation on one clip's transcript, small vocabulary
        _case("distill one clip", "distill", 1, 40, 10000, "fp32", ragged=False, top=8),
        # an ordinary fine-tuning batch
        _case("distill batch", "distill", 48, 64, 50021, "bf16", top=16, temperature=2.0),
        # long transcripts: the largest step
        _case("distill long", "distill", 16, 1024, 50021, "bf16", top=32, temperature=2.0, alpha=0.8),
        # a wide multilingual vocabulary, half precision, the most teacher entries
        _case("distill wide", "distill", 8, 128, 200019, "fp16", top=64, temperature=3.0),
        # per-position losses that the training loop weights itself
        _case("distill, weighted positions", "distill_each", 32, 100, 32000, "bf16", shifted=True, top=20, temperature=1.5, alpha=0.9),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["score", "score", "score_train", "distill", "distill", "distill_each"])
    vocab = log(1000, 210000)
    positions = 1 if op == "score" and rng.random() < 0.3 else log(2, 1024)
    # no more logits than the largest listed case of the same kind, and no more than 512 clips
    batch = log(1, max(1, min(512, (800_000_000 if op != "score" else 500_000_000) // (vocab * positions))))
    top = 0 if op == "score_train" or (op == "score" and rng.random() < 0.2) else log(1, 64)
    case = _case("", op, batch, positions, vocab, rng.choice(list(DTYPES)), ragged=positions > 1 and rng.random() < 0.8,
                 shifted=positions > 1 and rng.random() < 0.3, suppressed=rng.choice([0.0, 0.002]) if op == "score" else 0.0, top=top,
                 temperature=rng.choice([1.0, 1.0, 2.0, 0.7, 1.5, 3.0, 4.0]), alpha=rng.choice([0.5, 0.8, 1.0, 0.3]))
    del case["name"]
    return case


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    B, P, V, K = case["batch"], case["positions"], case["vocab"], case["top"]
    dtype = DTYPES[case["dtype"]]
    full = torch.empty((B, P + 1 if case["shifted"] else P, V), dtype=dtype, device=dev)
    full.normal_(0.0, 2.5, generator=g)
    logits = full[:, :P]
    labels = torch.randint(0, V, (B, P), device=dev, generator=g)
    if case["ragged"]:
        n = torch.randint(max(1, P // 4), P + 1, (B, 1), device=dev, generator=g)
        labels = torch.where(torch.arange(P, device=dev)[None] < n, labels, -100)
    # a model that has learnt something: the label stands out from the rest, by more or less
    at = labels.clamp_min(0)[..., None]
    boost = 4.0 + 5.0 * torch.rand((B, P, 1), device=dev, generator=g)
    logits.scatter_(2, at, (logits.gather(2, at).float() + boost).to(dtype))
    state = {"case": dict(case), "labels": labels}
    if case["suppressed"]:
        off = torch.randperm(V, device=dev, generator=g)[: max(1, int(V * case["suppressed"]))]
        full[..., off] = -math.inf
    if case["op"].startswith("distill"):
        # what a teacher's pass left in the cache: K distinct entries in falling order, the label mostly among them
        first = torch.randint(0, V, (B, P, 1), device=dev, generator=g)
        first = torch.where((torch.rand((B, P, 1), device=dev, generator=g) < 0.8) & (labels[..., None] >= 0), labels[..., None], first)
        step = 1 + torch.randint(0, max(1, V // max(K, 1) - 1), (B, P, K), device=dev, generator=g)
        step[..., :1] = 0
        state["teacher_ids"] = (first + step.cumsum(-1)) % V
        drop = 4.0 * torch.rand((B, P, K), device=dev, generator=g)
        drop[..., :1] = 0
        state["teacher_logits"] = -drop.cumsum(-1)
        # padding positions hold no teacher entries
        state["teacher_ids"].masked_fill_((labels < 0)[..., None], -1)
        state["teacher_logits"].masked_fill_((labels < 0)[..., None], -math.inf)
    if case["op"] in ("score_train", "distill_each"):
        state["weights"] = torch.rand((B, P), device=dev, generator=g) / (B * P)
    if case["op"] == "score_train":
        state["entropy_weights"] = torch.full((B, P), 0.01 / (B * P), device=dev)
    state["logits"] = logits.detach().requires_grad_(case["op"] != "score")
    return state


# ---------------------------------------------------------------------------------------- plain forms, in 32 bits
def _log_softmax(x, temperature):
    y = x if temperature == 1.0 else x / temperature
    y = y - y.amax(-1, keepdim=True)
    return y - y.exp().sum(-1, keepdim=True).log()


def _top(x, lp, k):
    """The k largest of x, ties to the lowest index: one whole number orders value and index."""
    bits = (x + 0.0).view(torch.int32).to(torch.int64)
    key = bits ^ ((bits >> 31) & 0x7FFFFFFF)
    key = key * 2 ** 31 + torch.arange(x.shape[-1] - 1, -1, -1, device=x.device)
    ids = x.shape[-1] - 1 - key.topk(k, -1).values % 2 ** 31
    return ids, lp.gather(-1, ids)


def _score(case, x, labels):
    valid = labels >= 0
    lp = _log_softmax(x, case["temperature"])
    p = lp.exp()
    logprob = torch.where(valid, lp.gather(-1, labels.clamp_min(0)[..., None])[..., 0], 0.0)
    entropy = torch.where(valid, -torch.where(p > 0, p * lp, 0.0).sum(-1), 0.0)
    return valid, lp, p, logprob, entropy


def _score_plain(s):
    case, labels = s["case"], s["labels"]
    x = s["logits"].float()
    valid, lp, p, logprob, entropy = _score(case, x, labels)
    out = {"logprobs": logprob, "entropy": entropy}
    if case["top"]:
        ids, top = _top(x, lp, case["top"])
        out["top_ids"] = torch.where(valid[..., None], ids, -1)
        out["top_logprobs"] = torch.where(valid[..., None], top, -math.inf)
    return out


def _score_train_plain(s):
    case, labels = s["case"], s["labels"]
    valid, lp, p, logprob, entropy = _score(case, s["logits"].float(), labels)
    gl = torch.where(valid, s["weights"], 0.0)[..., None]
    ge = torch.where(valid, s["entropy_weights"], 0.0)[..., None]
    grad = -p * (gl + ge * (lp + entropy[..., None]))
    grad.scatter_add_(-1, labels.clamp_min(0)[..., None], gl)
    return {"logprobs": logprob, "entropy": entropy, "grad": (grad / case["temperature"]).to(s["logits"].dtype)}


def _distill_plain(s, each):
    case, labels, tau, alpha = s["case"], s["labels"], s["case"]["temperature"], s["case"]["alpha"]
    x = s["logits"].float()
    valid = labels >= 0
    kept = s["teacher_ids"] >= 0
    ids, at = s["teacher_ids"].clamp_min(0), labels.clamp_min(0)[..., None]
    lq = torch.where(kept, _log_softmax(torch.where(kept, s["teacher_logits"].float(), -1e30), tau), 0.0)
    q = torch.where(kept, lq.exp(), 0.0)
    lp = _log_softmax(x, 1.0)
    lpt = lp if tau == 1.0 else _log_softmax(x, tau)
    kl = (q * (lq - lpt.gather(-1, ids))).sum(-1)
    loss = alpha * tau * tau * kl - (1.0 - alpha) * lp.gather(-1, at)[..., 0]
    loss = torch.where(valid, loss, 0.0)
    w = s["weights"] if each else 1.0 / valid.sum().clamp_min(1)
    w = torch.where(valid, w, 0.0)[..., None]
    grad = w * (alpha * tau * q.sum(-1, keepdim=True) * lpt.exp() + (1.0 - alpha) * lp.exp())
    grad.scatter_add_(-1, ids, -w * alpha * tau * q)
    grad.scatter_add_(-1, at, -w * (1.0 - alpha))
    return {"loss": loss if each else loss.sum() / valid.sum().clamp_min(1), "grad": grad.to(s["logits"].dtype)}


# ---------------------------------------------------------------------------------------- the framework's calls
def _score_own(s):
    from speech_to_text_amd import token_logprobs
    case = s["case"]
    r = token_logprobs(s["logits"], s["labels"], top_k=case["top"], entropy=True, temperature=case["temperature"])
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if case["top"]:
        out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
    return out


def _score_train_own(s):
    from speech_to_text_amd import token_logprobs
    r = token_logprobs(s["logits"], s["labels"], entropy=True, temperature=s["case"]["temperature"])
    grad, = torch.autograd.grad((r.logprobs, r.entropy), s["logits"], (s["weights"], s["entropy_weights"]))
    return {"logprobs": r.logprobs.detach(), "entropy": r.entropy.detach(), "grad": grad}


def _distill_own(s, each):
    from speech_to_text_amd import distillation_loss
    case = s["case"]
    loss = distillation_loss(s["logits"], s["labels"], s["teacher_ids"], s["teacher_logits"], temperature=case["temperature"],
                             alpha=case["alpha"], reduction="none" if each else "mean")
    grad, = torch.autograd.grad(loss, s["logits"], s["weights"] if each else None)
    return {"loss": loss.detach(), "grad": grad}


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "score":
            return _score_own(state)
        if op == "score_train":
            return _score_train_own(state)
        return _distill_own(state, op == "distill_each")
    with torch.no_grad():
        if op == "score":
            return _score_plain(state)
        if op == "score_train":
            return _score_train_plain(state)
        return _distill_plain(state, op == "distill_each")


def work(case):
    rows, V, K = case["batch"] * case["positions"], case["vocab"], case["top"]
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    share = 0.625 if case["ragged"] else 1.0          # rows that are read: the mean length of a ragged clip
    read = rows * share * V * size
    if case["op"] == "score":
        return {"bytes": read + rows * (8 + 8 + 12 * K), "flops": rows * share * V * 5}
    if case["op"] == "score_train":
        return {"bytes": read + rows * (V * size + 8 + 16), "flops": rows * share * V * 9}
    return {"bytes": read + rows * (V * size + 8 + 12 * K + 8), "flops": rows * share * V * 10}


# ---------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    B, P, V, K = case["batch"], case["positions"], case["vocab"], case["top"]
    op, T, alpha = case["op"], case["temperature"], case["alpha"]
    logits, labels = s["logits"].detach(), s["labels"]
    rows = [(b, t) for b in range(B) for t in range(P)]
    size = max(1, 200_000_000 // V)
    count = max(1, int((labels != -100).sum()))
    parts = {}

    def put(name, value):
        parts.setdefault(name, []).append(value)

    flat = torch.arange(B * P, device=logits.device)
    for c0 in range(0, len(rows), size):
        r = flat[c0:c0 + size]
        b, t = r // P, r % P
        z = logits[b, t].double()
        y, live = labels[b, t], labels[b, t] != -100
        y0 = y.clamp(min=0)
        n = torch.arange(len(r), device=z.device)
        logp = z / T - torch.logsumexp(z / T, 1)[:, None]
        if op in ("score", "score_train"):
            p = logp.exp()
            h = -torch.xlogy(p, p).sum(1)
            put("logprobs", torch.where(live, logp[n, y0], 0.0))
            put("entropy", torch.where(live, h, 0.0))
            if op == "score" and K:
                order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :K]
                put("top_ids", torch.where(live[:, None], order, -1))
                put("top_logprobs", torch.where(live[:, None], logp.gather(1, order), -math.inf))
            if op == "score_train":
                gl, gh = s["weights"][b, t].double() * live, s["entropy_weights"][b, t].double() * live
                d = -gl[:, None] * p - gh[:, None] * p * (logp + h[:, None])
                d[n, y0] += gl
                put("grad", d / T)
            continue
        ids, have = s["teacher_ids"][b, t], s["teacher_ids"][b, t] >= 0
        q = torch.softmax(s["teacher_logits"][b, t].double() / T, 1)
        q = torch.where(have, q, 0.0)
        kl = (torch.xlogy(q, q) - q * logp.gather(1, ids.clamp(min=0))).sum(1)
        log1 = z - torch.logsumexp(z, 1)[:, None]
        loss = torch.where(live, alpha * T ** 2 * kl - (1 - alpha) * log1[n, y0], 0.0)
        put("loss", loss)
        w = s["weights"][b, t].double() * live if op == "distill_each" else live.double() / count
        d = logp.exp() * (alpha * T * q.sum(1))[:, None] + (1 - alpha) * log1.exp()
        for k in range(K):
            d[n, ids[:, k].clamp(min=0)] -= alpha * T * q[:, k]
        d[n, y0] -= 1 - alpha
        put("grad", torch.where(live[:, None], d, 0.0) * w[:, None])
    out = {}
    for name, v in parts.items():
        v = torch.cat(v)
        out[name] = v.reshape(labels.shape + v.shape[1:])
    if op == "distill":
        out["loss"] = out["loss"].sum() / count
    return out
