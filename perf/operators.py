"""Measured cases of the decoder's dense operators: ``fused_linear``, ``layer_norm`` and ``token_logprobs``.

``run`` computes a case either in its plain form (elementary torch operations in 32 bits,
rounded once at the end) or, where ``own`` is true, through this package's operators;
``exact`` gives the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-5
IGNORE = -100


# ------------------------------------------------------------------------------------------ cases
def _linear(name, rows, d_in, d_out, act, residual, dtype, train):
    return {"name": name, "op": "fused_linear", "rows": rows, "d_in": d_in, "d_out": d_out, "act": act,
            "residual": residual, "dtype": dtype, "train": train}


def _norm(name, rows, d, dtype, train):
    return {"name": name, "op": "layer_norm", "rows": rows, "d": d, "dtype": dtype, "train": train}


def _logprobs(name, rows, vocab, top, banned, dtype, train):
    return {"name": name, "op": "token_logprobs", "rows": rows, "vocab": vocab, "top": top, "banned": banned,
            "dtype": dtype, "train": train}


def listed():
    return [
        # the decoder's FFN expansion for one new token: latency
        _linear("linear token", 1, 256, 1024, "gelu", False, "bf16", False),
        # a wide model's output projection + residual for a small batch of new tokens: the weights' bytes
        _linear("linear few tokens", 7, 4096, 4096, "none", True, "f16", False),
        # the decoder's FFN expansion over a prefill of 8 sequences of 4096 tokens
        _linear("linear prefill", 32768, 256, 1024, "gelu", False, "bf16", False),
        # a wider FFN expansion in a training step
        _linear("linear train", 8192, 1024, 4096, "gelu", False, "bf16", True),
        # odd widths in full precision, training
        _linear("linear train odd", 1531, 509, 1021, "silu", True, "f32", True),
        # the decoder's norms over the same prefill
        _norm("norm prefill", 32768, 256, "bf16", False),
        # a wide model's norm in a training step
        _norm("norm train wide", 8192, 4096, "bf16", True),
        # an odd width in full precision, training
        _norm("norm train odd", 2049, 1001, "f32", True),
        # scoring one token of the decoder's vocabulary with alternatives: latency
        _logprobs("logprobs token", 1, 128, 5, False, "bf16", False),
        # the decoder's training loss over 8 sequences of 4096 tokens
        _logprobs("logprobs train", 32768, 128, 0, False, "bf16", True),
        # a serving batch over a large vocabulary, constrained decoding, 20 alternatives
        _logprobs("logprobs serving", 16, 131072, 20, True, "f32", False),
        # a training loss over a large odd vocabulary
        _logprobs("logprobs train large", 4096, 50001, 0, False, "bf16", True),
    ]


def _log_uniform(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    op = rng.choice(["fused_linear", "fused_linear", "layer_norm", "token_logprobs"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    train = rng.random() < 0.5
    while True:
        rows = _log_uniform(rng, 1, 32768)
        if op == "fused_linear":
            # widths are multiples of 64 or anything
            step = rng.choice([1, 64])
            d_in, d_out = (step * _log_uniform(rng, max(1, 16 // step), 4096 // step) for _ in range(2))
            if rows * d_in * d_out <= 8192 * 1024 * 4096 // (4 if dtype == "f32" else 1):
                c = _linear("", rows, d_in, d_out, rng.choice(["none", "gelu", "relu", "silu"]), rng.random() < 0.5,
                            dtype, train)
                break
        elif op == "layer_norm":
            d = _log_uniform(rng, 2, 16384)
            if rows * d <= 8192 * 4096:
                c = _norm("", rows, d, dtype, train)
                break
        else:
            vocab = _log_uniform(rng, 2, 131072)
            top = 0 if train else min(vocab, rng.randrange(0, 33))
            if rows * vocab <= 4096 * 50001 // (4 if top else 1):
                c = _logprobs("", rows, vocab, top, top > 0 and vocab >= 128 and rng.random() < 0.3, dtype, train)
                break
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    train = case["train"]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, device=dev, generator=g) * scale + shift).to(dt)

    s = {"case": case}
    rows = case["rows"]
    if case["op"] == "fused_linear":
        # rows as a LayerNorm leaves them, weights that keep the variance
        d_in, d_out = case["d_in"], case["d_out"]
        s["x"] = normal(rows, d_in)
        s["weight"] = normal(d_out, d_in, scale=d_in ** -0.5)
        s["bias"] = normal(d_out, scale=0.1)
        s["residual"] = normal(rows, d_out) if case["residual"] else None
        if train:
            s["dy"] = normal(rows, d_out, scale=0.1)
            for n in ("x", "weight", "bias", "residual"):
                if s[n] is not None:
                    s[n].requires_grad_()
    elif case["op"] == "layer_norm":
        # a residual stream: rows with a mean of their own
        d = case["d"]
        s["x"] = (torch.randn(rows, d, device=dev, generator=g) * 2
                  + torch.randn(rows, 1, device=dev, generator=g)).to(dt)
        s["weight"] = normal(d, scale=0.1, shift=1.0)
        s["bias"] = normal(d, scale=0.1)
        if train:
            s["dy"] = normal(rows, d, scale=0.1)
            for n in ("x", "weight", "bias"):
                s[n].requires_grad_()
    else:
        vocab = case["vocab"]
        s["logits"] = normal(rows, vocab, scale=2.5)
        s["tokens"] = torch.randint(0, vocab, (rows,), device=dev, generator=g)
        if case["banned"]:
            # constrained decoding: a quarter of the vocabulary may not be said
            s["logits"].masked_fill_(torch.rand(rows, vocab, device=dev, generator=g) < 0.25, -math.inf)
        if train:
            s["tokens"][torch.rand(rows, device=dev, generator=g) < 0.05] = IGNORE  # prompt tokens carry no loss
            s["dlogprob"] = torch.randn(rows, device=dev, generator=g) * 0.2 - 1
            s["dentropy"] = torch.randn(rows, device=dev, generator=g) * 0.01
            s["logits"].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    return (_OWN if own else _PLAIN)[s["case"]["op"]](s)


def _own_linear(s):
    from wayfinder_attention_b200 import fused_linear

    y = fused_linear(s["x"], s["weight"], s["bias"], activation=s["case"]["act"], residual=s["residual"])
    if not s["case"]["train"]:
        return {"y": y}
    names = [n for n in ("x", "weight", "bias", "residual") if s[n] is not None]
    grads = torch.autograd.grad(y, [s[n] for n in names], s["dy"])
    return {"y": y, **{"d" + n: v for n, v in zip(names, grads)}}


def _own_norm(s):
    from wayfinder_attention_b200 import layer_norm

    y = layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
    if not s["case"]["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [s["x"], s["weight"], s["bias"]], s["dy"])
    return {"y": y, "dx": grads[0], "dweight": grads[1], "dbias": grads[2]}


def _own_logprobs(s):
    from wayfinder_attention_b200 import token_logprobs

    case = s["case"]
    r = token_logprobs(s["logits"], s["tokens"], top_n=case["top"], ignore_index=IGNORE)
    out = {"logprob": r.logprob, "entropy": r.entropy}
    if case["top"]:
        out["top_logprobs"], out["top_tokens"] = r.top_logprobs, r.top_tokens
    if case["train"]:
        out["dlogits"], = torch.autograd.grad([r.logprob, r.entropy], [s["logits"]], [s["dlogprob"], s["dentropy"]])
    return out


@torch.no_grad()
def _plain_linear(s):
    case, dt = s["case"], s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    z = torch.matmul(x, w.t()) + b
    if case["act"] == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        h = z * cdf
    elif case["act"] == "silu":
        sig = 1 / (1 + torch.exp(-z))
        h = z * sig
    elif case["act"] == "relu":
        h = torch.where(z > 0, z, 0.0)
    else:
        h = z
    y = h if s["residual"] is None else h + s["residual"].float()
    out = {"y": y.to(dt)}
    if case["train"]:
        dy = s["dy"].float()
        if case["act"] == "gelu":
            dz = dy * (cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
        elif case["act"] == "silu":
            dz = dy * (sig * (1 + z * (1 - sig)))
        elif case["act"] == "relu":
            dz = torch.where(z > 0, dy, 0.0)
        else:
            dz = dy
        out["dx"] = torch.matmul(dz, w).to(dt)
        out["dweight"] = torch.matmul(dz.t(), x).to(dt)
        out["dbias"] = dz.sum(0).to(dt)
        if s["residual"] is not None:
            out["dresidual"] = s["dy"]
    return out


@torch.no_grad()
def _plain_norm(s):
    dt = s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    c = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    xhat = c * rstd
    out = {"y": (xhat * w + b).to(dt)}
    if s["case"]["train"]:
        dy = s["dy"].float()
        g = dy * w
        out["dx"] = (rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))).to(dt)
        out["dweight"] = (dy * xhat).sum(0).to(dt)
        out["dbias"] = dy.sum(0).to(dt)
    return out


@torch.no_grad()
def _plain_logprobs(s):
    case = s["case"]
    x = s["logits"].float()
    tokens = s["tokens"]
    top = x.max(-1, keepdim=True).values
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    p = e / total
    lp = x - lse
    plp = torch.where(p > 0, p * lp, 0.0)
    entropy = -plp.sum(-1)
    kept = tokens != IGNORE
    at = torch.where(kept, tokens, 0).unsqueeze(-1)
    logprob = torch.where(kept, torch.gather(lp, 1, at).squeeze(-1), 0.0)
    out = {"logprob": logprob, "entropy": entropy}
    if case["top"]:
        values, index = torch.sort(x, dim=-1, descending=True, stable=True)
        out["top_logprobs"] = values[:, :case["top"]] - lse
        out["top_tokens"] = index[:, :case["top"]].contiguous()
    if case["train"]:
        gl = torch.where(kept, s["dlogprob"], 0.0).unsqueeze(-1)
        d = -gl * p - s["dentropy"].unsqueeze(-1) * (plp + p * entropy.unsqueeze(-1))
        d.scatter_add_(1, at, gl)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


_OWN = {"fused_linear": _own_linear, "layer_norm": _own_norm, "token_logprobs": _own_logprobs}
_PLAIN = {"fused_linear": _plain_linear, "layer_norm": _plain_norm, "token_logprobs": _plain_logprobs}


# ------------------------------------------------------------------------------------------ floors
def work(case):
    sz, rows = SIZES[case["dtype"]], case["rows"]
    if case["op"] == "fused_linear":
        k, n = case["d_in"], case["d_out"]
        act_rows = rows * n * (2 if case["residual"] else 1)  # y and the residual
        if not case["train"]:
            return {"bytes": sz * (rows * k + n * k + n + act_rows), "flops": 2 * rows * k * n}
        return {"bytes": sz * (2 * rows * k + 2 * n * k + 2 * n + act_rows + rows * n), "flops": 6 * rows * k * n}
    if case["op"] == "layer_norm":
        d = case["d"]
        if not case["train"]:
            return {"bytes": sz * (2 * rows * d + 2 * d), "flops": 8 * rows * d}
        return {"bytes": sz * (4 * rows * d + 4 * d), "flops": 20 * rows * d}
    v = case["vocab"]
    small = rows * (8 + 8 + case["top"] * 12)  # tokens; logprob and entropy; alternatives
    if not case["train"]:
        return {"bytes": sz * rows * v + small, "flops": 6 * rows * v}
    return {"bytes": 2 * sz * rows * v + small + 8 * rows, "flops": 12 * rows * v}


# ------------------------------------------------------------------------------------------ 64 bits
@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    d64 = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "fused_linear":
        z = torch.addmm(d64["bias"], d64["x"], d64["weight"].T)
        if case["act"] == "gelu":
            phi = torch.special.ndtr(z)
            y, slope = z * phi, phi + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi)
        elif case["act"] == "silu":
            sg = torch.special.expit(z)
            y, slope = z * sg, sg + z * sg * torch.special.expit(-z)
        elif case["act"] == "relu":
            y, slope = z.clamp_min(0), (z > 0).double()
        else:
            y, slope = z, None
        if case["residual"]:
            y = y + d64["residual"]
        out = {"y": y}
        if case["train"]:
            dz = d64["dy"] if slope is None else d64["dy"] * slope
            out["dx"], out["dweight"], out["dbias"] = dz @ d64["weight"], dz.T @ d64["x"], dz.sum(0)
            if case["residual"]:
                out["dresidual"] = d64["dy"]
        return out
    if case["op"] == "layer_norm":
        x, w = d64["x"], d64["weight"]
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        sd = (var + EPS).sqrt()
        n = (x - mean) / sd
        out = {"y": n * w + d64["bias"]}
        if case["train"]:
            g = d64["dy"] * w
            out["dx"] = (g - g.mean(1, keepdim=True) - n * (n * g).mean(1, keepdim=True)) / sd
            out["dweight"], out["dbias"] = (d64["dy"] * n).sum(0), d64["dy"].sum(0)
        return out
    x, rows = d64["logits"], case["rows"]
    logp = torch.log_softmax(x, dim=-1)
    prob = logp.exp()
    entropy = torch.special.entr(prob).sum(-1)
    valid = s["tokens"] >= 0
    at = s["tokens"].clamp_min(0)
    each = torch.arange(rows, device=x.device)
    out = {"logprob": logp[each, at].masked_fill(~valid, 0.0), "entropy": entropy}
    if case["top"]:
        order = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :case["top"]].contiguous()
        out["top_logprobs"], out["top_tokens"] = logp.gather(1, order), order
    if case["train"]:
        gl = d64["dlogprob"].masked_fill(~valid, 0.0)
        d = -prob * (gl[:, None] + d64["dentropy"][:, None] * (logp + entropy[:, None]))
        d[each, at] += gl
        out["dlogits"] = d
    return out
