"""Operators between a block's output and its scored tokens, as cases with a plain and a 64-bit form.

Around the log-probabilities that this package computes and the decoding step that makes tokens,
a post-training program also runs
  log-probabilities with the K most likely alternatives of every position (rollouts, evaluation,
  a teacher's lists), with their gradient,
  log-probabilities of K given tokens per position (a student on a teacher's lists), with their
  gradient,
  the norm after a block and the one before the next, with the block's gate and scales between
  them (in training with its gradient, in serving with an output in 8 bits),
  and the 8-bit matrix product with bias, activation and residual.

`run` computes the plain form with elementary torch operations; with `own` set it calls
`kernel_opt`.  `exact` computes the same in 64 bits, written apart from the plain form.
Vocabulary and hidden sizes are those of this repository's benchmark and tests (V = 32000,
50257, 128256, 151936, 152064; H = 3584, 2051), with odd and ragged ones between.
"""
import math
import os
import sys

import torch

own = False

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
BLOCK = 128          # columns (and weight rows) that share a scale
AMAX_FLOOR = 1e-30   # a block of zeros gets a scale that is not zero
EPS = 1e-6
IGNORED = -100       # pads a list of tokens that is shorter than the others
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one decoding sequence whose alternatives the client asked for: latency counts
        {"name": "top one row", "op": "top", "rows": 1, "vocab": 151936, "dtype": "bf16", "spread": 3.0, "k": 20,
         "temperature": 1.0, "grad": False},
        # rollouts scored with their alternatives at the sampling temperature
        {"name": "top rollouts", "op": "top", "rows": 512, "vocab": 152064, "dtype": "bf16", "spread": 3.0, "k": 20,
         "temperature": 0.8, "grad": False},
        # a teacher's lists over a vocabulary whose rows start at odd addresses
        {"name": "top teacher odd", "op": "top", "rows": 1023, "vocab": 50257, "dtype": "fp16", "spread": 2.0, "k": 64,
         "temperature": 1.0, "grad": False},
        # a training step that uses the target, the entropy and the alternatives
        {"name": "top train", "op": "top", "rows": 1024, "vocab": 128256, "dtype": "bf16", "spread": 3.0, "k": 8,
         "temperature": 1.0, "grad": True},
        # a student's step on a teacher's lists of 32 tokens
        {"name": "tokens train", "op": "tokens", "rows": 2048, "vocab": 151936, "dtype": "bf16", "spread": 3.0, "k": 32,
         "temperature": 1.0, "grad": True},
        # the same, small, in fp32, with short lists and a temperature
        {"name": "tokens train odd fp32", "op": "tokens", "rows": 333, "vocab": 50257, "dtype": "fp32", "spread": 2.5,
         "k": 7, "temperature": 2.0, "grad": True},
        # a block's end in a training step: 8 x 1024 tokens, a learned gate per column
        {"name": "norms train 8192x3584", "op": "norm_train", "rows": 8192, "hidden": 3584, "dtype": "bf16",
         "gate": "column", "branch_scale": 1.0, "residual_scale": 1.0},
        # a small fp32 model with an odd width and a gate per element
        {"name": "norms train odd fp32", "op": "norm_train", "rows": 777, "hidden": 2051, "dtype": "fp32",
         "gate": "full", "branch_scale": 0.5, "residual_scale": 1.0},
        # one sequence decoding: the norms in front of an 8-bit layer, where latency counts
        {"name": "norms 8-bit one token", "op": "norm_fp8", "rows": 1, "hidden": 3584, "dtype": "bf16",
         "gate": "none", "branch_scale": 1.0, "residual_scale": 1.0},
        # a prompt's rows on their way into an 8-bit layer
        {"name": "norms 8-bit prompt", "op": "norm_fp8", "rows": 8192, "hidden": 3584, "dtype": "bf16",
         "gate": "token", "branch_scale": 0.7, "residual_scale": 1.0},
        # a decoding batch through a layer's first product, with bias and activation
        {"name": "linear act batch of 16", "op": "linear", "tokens": 16, "inner": 3584, "outer": 14336, "out": "bf16",
         "bias": True, "activation": "gelu_tanh", "residual": False},
        # a prompt through the second product, added to the residual stream
        {"name": "linear residual prompt", "op": "linear", "tokens": 2048, "inner": 14336, "outer": 3584, "out": "bf16",
         "bias": False, "activation": None, "residual": True},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["top", "top", "tokens", "tokens", "norm_train", "norm_fp8", "linear", "linear"])
    if op in ("top", "tokens"):
        vocab = rng.choice([32000, 50257, 128256, 151936, 152064, _log(rng, 200, 152064)])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        grad = op == "tokens" or rng.random() < 0.4
        most = 2048 * 151936 // (2 if dtype == "fp32" else 1) // (1 if op == "tokens" else 2)
        return {"op": op, "rows": min(_log(rng, 1, 4096), max(1, most // vocab)), "vocab": vocab, "dtype": dtype,
                "spread": round(rng.uniform(1.5, 5.0), 2), "k": _log(rng, 1, 100),
                "temperature": rng.choice([1.0, round(rng.uniform(0.5, 2.0), 2)]), "grad": grad}
    if op in ("norm_train", "norm_fp8"):
        hidden = _log(rng, 128, 8192)
        if rng.random() < 0.7:
            hidden = max(128, hidden // 64 * 64)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        most = 8192 * 3584 // (2 if dtype == "fp32" else 1)
        return {"op": op, "rows": min(_log(rng, 1, 16384), max(1, most // hidden)), "hidden": hidden, "dtype": dtype,
                "gate": rng.choice(["none", "column", "token", "full"]),
                "branch_scale": rng.choice([1.0, round(rng.uniform(0.1, 2.0), 2)]),
                "residual_scale": rng.choice([1.0, round(rng.uniform(0.5, 1.0), 2)])}
    inner = 16 * _log(rng, 16, 896)
    outer = min(_log(rng, 500, 32768), 32768 * 3584 // inner)
    tokens = min(_log(rng, 1, 4096), max(1, 2048 * 14336 * 3584 // (inner * outer)), max(1, 2048 * 32768 // outer))
    return {"op": op, "tokens": tokens, "inner": inner, "outer": outer, "out": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "bias": rng.random() < 0.6, "activation": rng.choice([None, "relu", "silu", "gelu", "gelu_tanh"]),
            "residual": rng.random() < 0.5}


def _blocks(n):
    return -(-n // BLOCK)


def _quantise_rows(x):
    """(e4m3 values, fp32 scales) of x [n, k], one scale per row and 128 columns."""
    n, k = x.shape
    p = torch.nn.functional.pad(x, (0, _blocks(k) * BLOCK - k)).view(n, -1, BLOCK)
    scale = p.abs().amax(2).clamp(min=AMAX_FLOOR) / FP8_MAX
    return (p / scale[:, :, None]).to(FP8).view(n, -1)[:, :k].contiguous(), scale


def _quantise_blocks(w):
    """(e4m3 values, fp32 scales) of w [n, k], one scale per block of 128 x 128."""
    n, k = w.shape
    nb, kb = _blocks(n), _blocks(k)
    p = torch.nn.functional.pad(w, (0, kb * BLOCK - k, 0, nb * BLOCK - n)).view(nb, BLOCK, kb, BLOCK)
    scale = p.abs().amax((1, 3)).clamp(min=AMAX_FLOOR) / FP8_MAX
    q = (p / scale[:, None, :, None]).to(FP8).view(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous()
    return q, scale


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = dict(case)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(shape, generator=g, device="cuda")

    if c["op"] in ("top", "tokens"):
        n, v, t = c["rows"], c["vocab"], TYPES[c["dtype"]]
        z = normal(n, v).mul_(c["spread"])
        # half of the rows as a trained model leaves them: a few tokens stand out
        raised = torch.randint(0, v, (n, 24), generator=g, device="cuda")
        z[::2].scatter_add_(1, raised[::2], 4.0 * c["spread"] * uniform(n, 24)[::2])
        k = c["k"] = min(c["k"], v)
        s = {"case": c, "logits": z.to(t)}
        if c["op"] == "top":
            s["targets"] = torch.where(uniform(n) < 0.7, z.argmax(1), raised[:, 0])
        else:
            # a teacher that mostly agrees: the largest of the logits with noise on them; every
            # eighth list is shorter
            s["tokens"] = z.add_(0.5 * c["spread"] * normal(n, v)).topk(k, 1).indices
            if k > 1:
                s["tokens"][::8, k // 2:] = IGNORED
        if c["grad"]:
            s["logits"].requires_grad_(True)
            s["g_entropy"] = 0.01 * normal(n)
            if c["op"] == "top":
                s["g_logprob"], s["g_top"] = normal(n), 0.1 * normal(n, k)
            else:
                # a cross entropy's: the teacher's probabilities, none on the padding
                s["g_logprobs"] = -torch.softmax(2.0 * normal(n, k), 1) * (s["tokens"] != IGNORED)
        return s
    if c["op"] in ("norm_train", "norm_fp8"):
        t = TYPES[c["dtype"]]
        n, h = c["rows"], c["hidden"]
        # a block's output and the stream it is added to, with the few large columns that streams have
        wide = torch.where(uniform(h) < 0.01, 8.0, 1.0)
        s = {"case": c, "x": (3.0 * normal(n, h)).to(t), "residual": (2.0 * normal(n, h) * wide).to(t),
             "post_weight": (1.0 + 0.1 * normal(h)).to(t), "weight": (1.0 + 0.1 * normal(h)).to(t), "gate": None}
        if c["gate"] != "none":
            shape = {"column": (h,), "token": (n, 1), "full": (n, h)}[c["gate"]]
            s["gate"] = (0.5 + 0.2 * normal(*shape)).to(t)
        if c["op"] == "norm_train":
            s["g_y"], s["g_stream"] = normal(n, h).to(t), normal(n, h).to(t)
            for k in ("x", "residual", "post_weight", "weight", "gate"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
        return s
    m, k, n = c["tokens"], c["inner"], c["outer"]
    t = TYPES[c["out"]]
    xq, xs = _quantise_rows(normal(m, k))
    wq, ws = _quantise_blocks(normal(n, k).mul_(k ** -0.5))
    return {"case": c, "xq": xq, "xs": xs, "wq": wq, "ws": ws, "bias": (0.5 * normal(n)).to(t) if c["bias"] else None,
            "residual": normal(m, n).to(t) if c["residual"] else None}


# ------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------
def _scale(c):
    """The factor of the logits: 1 / temperature as an fp32 number."""
    return torch.tensor(1.0 / c["temperature"], dtype=torch.float64).float().item()


def _plain_logprobs(s):
    # values in 32 bits; the long sums of weights in 64
    c, scale = s["case"], _scale(s["case"])
    with torch.no_grad():
        x = s["logits"].float()
        n, v = x.shape
        y = x * scale
        top = y.amax(1, keepdim=True)
        d = y - top
        w = torch.exp(d)
        total = w.sum(1, keepdim=True, dtype=torch.float64)
        log_total = total.log()
        lse = top.double() + log_total
        entropy = (log_total - (w * d).sum(1, keepdim=True, dtype=torch.float64) / total)[:, 0]

        def of(ids):  # an id outside the vocabulary reads a logit of 0
            there = (ids >= 0) & (ids < v)
            return (torch.where(there, y.gather(1, ids.clamp(0, v - 1)), 0.0).double() - lse).float(), there

        if c["op"] == "top":
            ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :c["k"]]
            listed_ids = torch.cat([s["targets"][:, None], ids], 1)
        else:
            listed_ids = s["tokens"]
        lp, there = of(listed_ids)
        out = {"entropy": entropy.float(), "lse": lse[:, 0].float()}
        if c["op"] == "top":
            out.update({"logprob": lp[:, 0], "ids": ids, "top": lp[:, 1:]})
        else:
            out["logprobs"] = lp
        if c["grad"]:
            g = torch.cat([s["g_logprob"][:, None], s["g_top"]], 1) if c["op"] == "top" else s["g_logprobs"]
            logp = y - lse.float()
            g_entropy = s["g_entropy"][:, None]
            dy = logp.exp() * (-g.sum(1, keepdim=True) - g_entropy * (logp + entropy.float()[:, None]))
            dy.scatter_add_(1, listed_ids.clamp(0, v - 1), g * there)
            out["dlogits"] = (dy * scale).to(s["logits"].dtype)
        return out


def _plain_norms(s):
    # the stream is a stored tensor of the inputs' type; the second norm reads what is stored
    c, t = s["case"], s["x"].dtype
    x, post, w = s["x"].float(), s["post_weight"].float(), s["weight"].float()
    gate = 1.0 if s["gate"] is None else s["gate"].float()
    r1 = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    n1 = x * r1
    stream = (c["residual_scale"] * s["residual"].float() + c["branch_scale"] * (gate * (n1 * post))).to(t)
    f = stream.float()
    r2 = torch.rsqrt((f * f).mean(1, keepdim=True) + EPS)
    n2 = f * r2
    return x, post, w, gate, r1, n1, stream, r2, n2


def _plain_norm_train(s):
    c, t = s["case"], s["x"].dtype
    with torch.no_grad():
        x, post, w, gate, r1, n1, stream, r2, n2 = _plain_norms(s)
        g = s["g_y"].float()
        gw = g * w
        ds = r2 * (gw - n2 * (gw * n2).mean(1, keepdim=True)) + s["g_stream"].float()
        db = ds * c["branch_scale"]
        dn = db * gate
        gp = dn * post
        out = {"y": (n2 * w).to(t), "stream": stream,
               "dx": (r1 * (gp - n1 * (gp * n1).mean(1, keepdim=True))).to(t),
               "dresidual": (c["residual_scale"] * ds).to(t), "dpost": (dn * n1).sum(0).to(t), "dweight": (g * n2).sum(0).to(t)}
        if s["gate"] is not None:
            dg = db * (n1 * post)
            if c["gate"] != "full":
                dg = dg.sum(0) if c["gate"] == "column" else dg.sum(1, keepdim=True)
            out["dgate"] = dg.to(t)
        return out


def _plain_norm_fp8(s):
    w, stream, n2 = (_plain_norms(s)[i] for i in (2, 6, 8))
    q, scale = _quantise_rows(n2 * w)
    return {"q": q, "scales": scale, "stream": stream}


def _plain_linear(s):
    c = s["case"]
    k, n = s["xq"].shape[1], s["wq"].shape[0]
    x = s["xq"].float() * s["xs"].repeat_interleave(BLOCK, 1)[:, :k]
    w = s["wq"].float() * s["ws"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if c["activation"] == "relu":
        z = z.clamp(min=0)
    elif c["activation"] == "silu":
        z = z / (1 + torch.exp(-z))
    elif c["activation"] == "gelu":
        z = 0.5 * z * torch.erfc(-z * math.sqrt(0.5))
    elif c["activation"] == "gelu_tanh":
        z = z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if s["residual"] is not None:
        z = z + s["residual"].float()
    return {"y": z.to(TYPES[c["out"]])}


def _plain(s):
    return {"top": _plain_logprobs, "tokens": _plain_logprobs, "norm_train": _plain_norm_train,
            "norm_fp8": _plain_norm_fp8, "linear": _plain_linear}[s["case"]["op"]](s)


# ------------------------------------------------------------------------------------------
# The framework's calls
# ------------------------------------------------------------------------------------------
def _kernel_opt():
    if "kernel_opt" not in sys.modules:
        at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                          "fused-logprob-entropy-cuda-kernel-for-llm-post-training_b200")
        if not os.path.isdir(at):
            at = os.path.join(os.getcwd(), "fused-logprob-entropy-cuda-kernel-for-llm-post-training_b200")
        if at not in sys.path:
            sys.path.insert(0, at)
    import kernel_opt
    return kernel_opt


def _own(s):
    ko = _kernel_opt()
    c = s["case"]
    op = c["op"]
    if op == "top":
        logprob, entropy, lse, ids, top = ko.fused_top_logprobs(s["logits"], s["targets"], c["k"], c["temperature"])
        out = {"entropy": entropy, "lse": lse, "logprob": logprob, "ids": ids, "top": top}
        if c["grad"]:
            out["dlogits"], = torch.autograd.grad((logprob, entropy, top), s["logits"],
                                                  (s["g_logprob"], s["g_entropy"], s["g_top"]))
        return out
    if op == "tokens":
        logprobs, entropy, lse = ko.fused_token_logprobs(s["logits"], s["tokens"], c["temperature"])
        out = {"entropy": entropy, "lse": lse, "logprobs": logprobs}
        if c["grad"]:
            out["dlogits"], = torch.autograd.grad((logprobs, entropy), s["logits"], (s["g_logprobs"], s["g_entropy"]))
        return out
    if op in ("norm_train", "norm_fp8"):
        call = ko.fused_sandwich_rmsnorm if op == "norm_train" else ko.fused_sandwich_rmsnorm_fp8
        got = call(s["x"], s["residual"], s["post_weight"], s["weight"], s["gate"], c["branch_scale"],
                   c["residual_scale"], EPS)
        if op == "norm_fp8":
            return dict(zip(("q", "scales", "stream"), got))
        wrt = {"dx": s["x"], "dresidual": s["residual"], "dpost": s["post_weight"], "dweight": s["weight"], "dgate": s["gate"]}
        wrt = {k: v for k, v in wrt.items() if v is not None}
        grads = torch.autograd.grad(got, list(wrt.values()), (s["g_y"], s["g_stream"]))
        return {"y": got[0], "stream": got[1], **dict(zip(wrt, grads))}
    return {"y": ko.fp8_linear(s["xq"], s["xs"], s["wq"], s["ws"], TYPES[c["out"]], bias=s["bias"],
                               activation=c["activation"], residual=s["residual"])}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    if case["op"] in ("top", "tokens"):
        n, v, k = case["rows"], case["vocab"], min(case["k"], case["vocab"])
        b = 4 if case["dtype"] == "fp32" else 2
        # ids and log-probabilities of the list, entropy, lse (and the target's); the backward
        # reads the logits again, since a step's own work lies between, and writes their gradient
        small = n * (12 * k + 8 + (12 if case["op"] == "top" else 0))
        return {"bytes": n * v * b * (3 if case["grad"] else 1) + small * (2 if case["grad"] else 1),
                "flops": n * v * (14 if case["grad"] else 6)}
    if case["op"] in ("norm_train", "norm_fp8"):
        n, h = case["rows"], case["hidden"]
        b = 4 if case["dtype"] == "fp32" else 2
        full = case["gate"] == "full"
        if case["op"] == "norm_train":
            # forward: x, residual in, y, stream out; backward: two gradients, x and the stream
            # (again, as above) in, two out; a gate per element twice in, its gradient out
            return {"bytes": ((13 if full else 10) * n * h + 4 * h) * b, "flops": 40 * n * h}
        return {"bytes": ((4 if full else 3) * n * h + 2 * h) * b + n * h + 4 * n * _blocks(h), "flops": 14 * n * h}
    m, k, n = case["tokens"], case["inner"], case["outer"]
    b = 4 if case["out"] == "fp32" else 2
    scales = 4 * _blocks(k) * (m + _blocks(n))
    return {"bytes": m * k + n * k + scales + m * n * b * (2 if case["residual"] else 1) + (n * b if case["bias"] else 0),
            "flops": 2 * m * k * n}


# ------------------------------------------------------------------------------------------
# The same in 64 bits
# ------------------------------------------------------------------------------------------
def _exact_logprobs(s):
    c, scale = s["case"], _scale(s["case"])
    n, v = s["logits"].shape
    parts = []
    step = max(1, (1 << 26) // v)
    for r in range(0, n, step):
        at = slice(r, r + step)
        x = s["logits"].detach()[at].double().requires_grad_(c["grad"])
        logp = torch.log_softmax(x * scale, 1)
        lse = torch.logsumexp(x.detach() * scale, 1)
        p = logp.exp()
        entropy = -(p * logp).sum(1)
        part = {"entropy": entropy.detach(), "lse": lse}

        def of(ids):
            inside = (ids >= 0) & (ids < v)
            outside = (logp.logsumexp(1) - torch.logsumexp(x * scale, 1))[:, None]  # 0 - lse
            return torch.where(inside, logp.gather(1, torch.where(inside, ids, 0)), outside)

        if c["op"] == "top":
            part["ids"] = torch.argsort(x.detach(), dim=1, descending=True, stable=True)[:, :c["k"]]
            lp = of(torch.cat([s["targets"][at, None], part["ids"]], 1))
            part["logprob"], part["top"] = lp.detach()[:, 0], lp.detach()[:, 1:]
        else:
            lp = of(s["tokens"][at])
            part["logprobs"] = lp.detach()
        if c["grad"]:
            g = torch.cat([s["g_logprob"][at, None], s["g_top"][at]], 1) if c["op"] == "top" else s["g_logprobs"][at]
            loss = (lp * g.double()).sum() + (entropy * s["g_entropy"][at].double()).sum()
            part["dlogits"], = torch.autograd.grad(loss, x)
        parts.append(part)
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_norm(s, train):
    c = s["case"]
    leaf = {k: s[k].detach().double().requires_grad_(train)
            for k in ("x", "residual", "post_weight", "weight", "gate") if s[k] is not None}
    h = leaf["x"].shape[1]

    def normed(a, weight):
        return a * weight / (a.square().sum(1, keepdim=True) / h + EPS).sqrt()

    branch = normed(leaf["x"], leaf["post_weight"]) * c["branch_scale"]
    if s["gate"] is not None:
        branch = branch * leaf["gate"]
    total = leaf["residual"] * c["residual_scale"] + branch
    # the stream as it is stored, its rounding passed over by the gradient
    stored = total + (total.detach().to(s["x"].dtype).double() - total.detach())
    y = normed(stored, leaf["weight"])
    if train:
        grads = torch.autograd.grad((y, stored), list(leaf.values()), (s["g_y"].double(), s["g_stream"].double()))
        names = {"x": "dx", "residual": "dresidual", "post_weight": "dpost", "weight": "dweight", "gate": "dgate"}
        return {"y": y.detach(), "stream": total.detach(), **{names[k]: g for k, g in zip(leaf, grads)}}
    n = y.shape[0]
    scale = torch.empty(n, _blocks(h), dtype=torch.float64, device=y.device)
    q = torch.empty_like(y)
    for b, part in enumerate(y.split(BLOCK, 1)):
        scale[:, b] = part.abs().amax(1).clamp(min=AMAX_FLOOR) / FP8_MAX
        q[:, b * BLOCK:b * BLOCK + part.shape[1]] = (part / scale[:, b:b + 1]).to(FP8).double()
    return {"q": q, "scales": scale, "stream": total}


def _exact_linear(s):
    c = s["case"]
    m, k = s["xq"].shape
    n = s["wq"].shape[0]
    z = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    of_row = torch.arange(n, device="cuda") // BLOCK
    for b in range(_blocks(k)):
        at = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
        z += (s["xq"][:, at].double() @ s["wq"][:, at].double().t()) * s["xs"][:, b:b + 1].double() * s["ws"][:, b].double()[of_row]
    if s["bias"] is not None:
        z += s["bias"].double()
    act = {None: lambda a: a, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
           "gelu_tanh": lambda a: torch.nn.functional.gelu(a, approximate="tanh")}
    z = act[c["activation"]](z)
    return {"y": z + s["residual"].double() if s["residual"] is not None else z}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        return _exact_linear(s)
    if op in ("top", "tokens"):
        return _exact_logprobs(s)
    return _exact_norm(s, op == "norm_train")
