"""Measured cases of the decoder's two ends: ``token_embedding`` and ``linear_token_logprobs``.

``run`` computes a case either in its plain form (elementary torch operations in 32 bits,
rounded once at the end) or, where ``own`` is true, through this package's operators;
``exact`` gives the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
IGNORE = -100
PAD = 0


# ------------------------------------------------------------------------------------------ cases
def _embedding(name, batch, seq, d, vocab, positions, pad, dtype, train):
    """positions: "none"; "arange": 0.. along each sequence; "packed": documents one after the other, each from 0.
    pad: the sequences end in padding, whose row takes no gradient."""
    return {"name": name, "op": "token_embedding", "batch": batch, "seq": seq, "d": d, "vocab": vocab,
            "positions": positions, "pad": pad, "dtype": dtype, "train": train}


def _logprobs(name, rows, d, vocab, bias, banned, dtype, train):
    return {"name": name, "op": "linear_token_logprobs", "rows": rows, "d": d, "vocab": vocab, "bias": bias,
            "banned": banned, "dtype": dtype, "train": train}


def listed():
    return [
        # one new position of the decoder in 8 sequences: latency
        _embedding("embedding token", 8, 1, 256, 128, "arange", False, "bf16", False),
        # a prefill of a wide model: the rows' bytes
        _embedding("embedding prefill wide", 16, 4096, 2048, 50001, "none", False, "f16", False),
        # the decoder's training step over 8 sequences of 4096 tokens: few rows, each with many tokens
        _embedding("embedding train", 8, 4096, 256, 128, "arange", False, "bf16", True),
        # a training step over a large odd vocabulary, packed documents: most rows get nothing
        _embedding("embedding train large", 8, 4096, 1024, 50001, "packed", False, "bf16", True),
        # odd sizes in full precision, sequences that end in padding
        _embedding("embedding train odd", 3, 683, 1001, 10007, "arange", True, "f32", True),
        # scoring one token of the decoder's vocabulary: latency
        _logprobs("head token", 1, 256, 128, False, False, "bf16", False),
        # scoring a small serving batch over a large vocabulary, a quarter of it banned: the weight's bytes
        _logprobs("head serving", 16, 4096, 131072, True, True, "f16", False),
        # scoring 8 sequences of 4096 tokens over a large odd vocabulary
        _logprobs("head score", 32768, 256, 50001, False, False, "bf16", False),
        # the decoder's training loss over 8 sequences of 4096 tokens
        _logprobs("head train", 32768, 256, 128, False, False, "bf16", True),
        # a training loss over a large odd vocabulary
        _logprobs("head train large", 8192, 1024, 50001, False, False, "bf16", True),
        # a wide model's training loss over a larger one
        _logprobs("head train wide", 4096, 4096, 131072, False, False, "bf16", True),
        # odd sizes in full precision, with a bias
        _logprobs("head train odd", 1531, 509, 10007, True, False, "f32", True),
    ]


def _log_uniform(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.6
    step = rng.choice([1, 64])  # widths are multiples of 64 or anything
    embedding = rng.random() < 0.4
    while True:
        d = step * _log_uniform(rng, max(1, 16 // step), 4096 // step)
        vocab = _log_uniform(rng, 2, 131072)
        if embedding:
            batch, seq = _log_uniform(rng, 1, 64), _log_uniform(rng, 1, 16384)
            if batch * seq * d <= 16 * 4096 * 2048 and vocab * d <= 131072 * 1024:
                c = _embedding("", batch, seq, d, vocab, rng.choice(["none", "arange", "packed"]),
                               rng.random() < 0.3, dtype, train)
                break
        else:
            rows = _log_uniform(rng, 1, 32768)
            if rows * d * vocab <= 2**41 // (8 if dtype == "f32" else 1) and rows * vocab <= 32768 * 50001:
                c = _logprobs("", rows, d, vocab, rng.random() < 0.5, False, dtype, train)
                c["banned"] = c["bias"] and not train and vocab >= 128 and rng.random() < 0.5
                break
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    train, vocab, d = case["train"], case["vocab"], case["d"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * scale).to(dt)

    def zipf(*shape):
        # text: the k-th most frequent token about 1 / k as frequent as the first
        u = torch.rand(*shape, device=dev, generator=g, dtype=torch.float64)
        return (torch.exp(u * math.log(vocab + 1)).long() - 1).clamp_(0, vocab - 1)

    s = {"case": case}
    if case["op"] == "token_embedding":
        b, t = case["batch"], case["seq"]
        s["tokens"] = zipf(b, t) if vocab > 128 else torch.randint(0, vocab, (b, t), device=dev, generator=g)
        s["scale"] = math.sqrt(d) if vocab > 128 else 1.0
        s["weight"] = normal(vocab, d, scale=d ** -0.5)
        s["position_weight"] = s["positions"] = None
        if case["positions"] != "none":
            s["position_weight"] = normal(t + 3, d, scale=0.1)
        if case["positions"] == "packed":
            # a document starts with each sequence and about every 200 tokens
            at = torch.arange(t, device=dev)
            starts = torch.where(torch.rand(b, t, device=dev, generator=g) < 1 / 200, at, 0)
            s["positions"] = at - torch.cummax(starts, 1).values
        if case["pad"]:
            kept = torch.randint(1, t + 1, (b, 1), device=dev, generator=g)
            s["tokens"][torch.arange(t, device=dev) >= kept] = PAD
        if train:
            s["dy"] = normal(b, t, d, scale=0.1)
            for n in ("weight", "position_weight"):
                if s[n] is not None:
                    s[n].requires_grad_()
    else:
        rows = case["rows"]
        # rows as a LayerNorm leaves them, weights that give logits of a spread of 2.5
        s["x"] = normal(rows, d)
        s["weight"] = normal(vocab, d, scale=2.5 * d ** -0.5)
        s["bias"] = normal(vocab, scale=0.5) if case["bias"] else None
        s["tokens"] = torch.randint(0, vocab, (rows,), device=dev, generator=g)
        if case["banned"]:
            s["bias"].masked_fill_(torch.rand(vocab, device=dev, generator=g) < 0.25, -math.inf)
        if train:
            s["tokens"][torch.rand(rows, device=dev, generator=g) < 0.05] = IGNORE  # prompt tokens carry no loss
            s["dlogprob"] = torch.randn(rows, device=dev, generator=g) * 0.2 - 1
            s["dentropy"] = torch.randn(rows, device=dev, generator=g) * 0.01
            for n in ("x", "weight", "bias"):
                if s[n] is not None:
                    s[n].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return (_OWN if own else _PLAIN)[s["case"]["op"]](s)


def _own_embedding(s):
    from wayfinder_attention_b200 import token_embedding

    case = s["case"]
    y = token_embedding(s["tokens"], s["weight"], scale=s["scale"], position_weight=s["position_weight"],
                        positions=s["positions"], padding_index=PAD if case["pad"] else None)
    if not case["train"]:
        return {"y": y}
    names = [n for n in ("weight", "position_weight") if s[n] is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
    return {"y": y, **{"d" + n: v for n, v in zip(names, grads)}}


def _own_logprobs(s):
    from wayfinder_attention_b200 import linear_token_logprobs

    r = linear_token_logprobs(s["x"], s["weight"], s["tokens"], bias=s["bias"], ignore_index=IGNORE)
    out = {"logprob": r.logprob, "entropy": r.entropy}
    if s["case"]["train"]:
        names = [n for n in ("x", "weight", "bias") if s[n] is not None]
        grads = torch.autograd.grad([r.logprob, r.entropy], [s[n] for n in names], [s["dlogprob"], s["dentropy"]])
        out.update({"d" + n: v for n, v in zip(names, grads)})
    return out


@torch.no_grad()
def _plain_embedding(s):
    case, dt = s["case"], s["weight"].dtype
    tokens, w, pw = s["tokens"], s["weight"], s["position_weight"]
    y = w[tokens].float() * s["scale"]
    at = None
    if pw is not None:
        at = s["positions"]
        if at is None:
            at = torch.arange(case["seq"], device=tokens.device).expand_as(tokens)
        y += pw[at].float()
    out = {"y": y.to(dt)}
    if case["train"]:
        dy = s["dy"].float().flatten(0, 1)
        dw = torch.zeros(w.shape, device=w.device).index_add_(0, tokens.flatten(), dy * s["scale"])
        if case["pad"]:
            dw[PAD] = 0
        out["dweight"] = dw.to(dt)
        if pw is not None:
            out["dposition_weight"] = torch.zeros(pw.shape, device=w.device).index_add_(0, at.flatten(), dy).to(dt)
    return out


@torch.no_grad()
def _plain_logprobs(s):
    dt, tokens = s["x"].dtype, s["tokens"]
    x, w = s["x"].float(), s["weight"].float()
    z = torch.matmul(x, w.t())
    if s["bias"] is not None:
        z += s["bias"].float()
    lp = z - z.max(-1, keepdim=True).values
    p = torch.exp(lp)
    total = p.sum(-1, keepdim=True)
    p /= total
    lp -= torch.log(total)
    plp = torch.where(p > 0, p * lp, 0.0)
    entropy = -plp.sum(-1)
    kept = tokens != IGNORE
    at = torch.where(kept, tokens, 0).unsqueeze(-1)
    out = {"logprob": torch.where(kept, torch.gather(lp, 1, at).squeeze(-1), 0.0), "entropy": entropy}
    if s["case"]["train"]:
        gl = torch.where(kept, s["dlogprob"], 0.0).unsqueeze(-1)
        dz = -gl * p - s["dentropy"].unsqueeze(-1) * (plp + p * entropy.unsqueeze(-1))
        dz.scatter_add_(1, at, gl)
        out["dx"] = torch.matmul(dz, w).to(dt)
        out["dweight"] = torch.matmul(dz.t(), x).to(dt)
        if s["bias"] is not None:
            out["dbias"] = dz.sum(0).to(dt)
    return out


_OWN = {"token_embedding": _own_embedding, "linear_token_logprobs": _own_logprobs}
_PLAIN = {"token_embedding": _plain_embedding, "linear_token_logprobs": _plain_logprobs}


# ------------------------------------------------------------------------------------------ floors
def work(case):
    sz, d, v = SIZES[case["dtype"]], case["d"], case["vocab"]
    if case["op"] == "token_embedding":
        n = case["batch"] * case["seq"]
        at = 0 if case["positions"] == "none" else case["seq"] + 3
        # rows of the table that are read at all
        rank = torch.arange(v, dtype=torch.float64)
        freq = torch.log1p(1 / (rank + 1)) / math.log(v + 1) if v > 128 else torch.full((v,), 1 / v, dtype=torch.float64)
        distinct = min(n, int((1 - (1 - freq) ** n).sum()) + 1)
        read = distinct * d + min(at, case["seq"]) * d
        ids = 8 * n * (2 if case["positions"] == "packed" else 1)
        if not case["train"]:
            return {"bytes": sz * (read + n * d) + ids, "flops": 2 * n * d}
        return {"bytes": sz * (read + 2 * n * d + v * d + at * d) + ids, "flops": 4 * n * d}
    rows = case["rows"]
    small = 16 * rows  # token; logprob and entropy
    weights = v * d + (v if case["bias"] else 0)
    if not case["train"]:
        return {"bytes": sz * (rows * d + weights) + small, "flops": 2 * rows * d * v}
    return {"bytes": 2 * sz * (rows * d + weights) + small + 8 * rows, "flops": 6 * rows * d * v}


# ------------------------------------------------------------------------------------------ 64 bits
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    d64 = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "token_embedding":
        b, t, d = case["batch"], case["seq"], case["d"]
        ids = s["tokens"].reshape(-1)
        place = None
        if case["positions"] == "arange":
            place = torch.arange(t, device=ids.device).repeat(b)
        elif case["positions"] == "packed":
            place = s["positions"].reshape(-1)
        y = torch.index_select(d64["weight"], 0, ids).mul_(s["scale"])
        if place is not None:
            y += torch.index_select(d64["position_weight"], 0, place)
        out = {"y": y.reshape(b, t, d)}
        if case["train"]:
            def sums(at, rows):  # of the gradients at each index: differences of running sums would lose bits
                order = torch.argsort(at, stable=True)
                lengths = torch.bincount(at, minlength=rows)
                g = d64["dy"].reshape(-1, d)[order]
                return torch.segment_reduce(g, "sum", lengths=lengths, axis=0, initial=0.0)

            out["dweight"] = sums(ids, case["vocab"]) * s["scale"]
            if case["pad"]:
                out["dweight"][PAD].zero_()
            if place is not None:
                out["dposition_weight"] = sums(place, t + 3)
        return out
    x, w, tokens = d64["x"], d64["weight"], s["tokens"]
    names = ["logprob", "entropy"] + (["dx"] if case["train"] else [])
    parts = {n: [] for n in names}
    dw, db = torch.zeros_like(w) if case["train"] else None, 0.0
    for lo in range(0, case["rows"], 2048):
        xs, ts = x[lo:lo + 2048], tokens[lo:lo + 2048]
        logits = xs @ w.T if s["bias"] is None else torch.addmm(d64["bias"], xs, w.T)
        logp = torch.log_softmax(logits, dim=-1)
        del logits
        prob = logp.exp()
        entropy = torch.special.entr(prob).sum(-1)
        each, valid, at = torch.arange(len(ts), device=ts.device), ts >= 0, ts.clamp_min(0)
        parts["logprob"].append(logp[each, at].masked_fill(~valid, 0.0))
        parts["entropy"].append(entropy)
        if case["train"]:
            gl = d64["dlogprob"][lo:lo + 2048].masked_fill(~valid, 0.0)
            gh = d64["dentropy"][lo:lo + 2048]
            dz = prob.mul_(logp.add_(entropy[:, None]).mul_(gh[:, None]).add_(gl[:, None])).neg_()
            dz[each, at] += gl
            parts["dx"].append(dz @ w)
            dw.addmm_(dz.T, xs)
            db = db + dz.sum(0)
    out = {n: torch.cat(v) for n, v in parts.items()}
    if case["train"]:
        out["dweight"] = dw
        if s["bias"] is not None:
            out["dbias"] = db
    return out
