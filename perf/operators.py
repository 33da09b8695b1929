"""The operators of a decoding step's tail, as cases with a plain form and a 64-bit form.

From the residual stream to the next token a language model runs
  the residual's addition and the root-mean-square norm (in training with its gradient;
  in serving with an output in 8 bits, one scale per row and 128 columns),
  the matrix product in 8 bits (the LM head of a decoding step, or any other layer),
  and the choice of a token with temperature, top-k, top-p and min-p from a given uniform
  random number, with the token's log-probability.

`run` computes the plain form with elementary torch operations; with `own` set it calls
`kernel_opt`.  `exact` computes the same in 64 bits, written apart from the plain form.
Vocabulary and hidden sizes are those of this repository's benchmark and tests (V = 32000,
50257, 128256, 151936, 152064; H = 3584), with odd and ragged ones between.
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
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one training step's final norm at GRPO's 16 x 1024 tokens: forward and backward
        {"name": "norm train 16384x3584", "op": "norm_train", "rows": 16384, "hidden": 3584, "dtype": "bf16"},
        # a small fp32 model with an odd width: rows that no vector load fits
        {"name": "norm train odd fp32", "op": "norm_train", "rows": 777, "hidden": 2051, "dtype": "fp32"},
        # one sequence decoding: the norm in front of the 8-bit head, where latency counts
        {"name": "norm 8-bit one token", "op": "norm_fp8", "rows": 1, "hidden": 3584, "dtype": "bf16"},
        # a prompt's rows on their way into an 8-bit layer
        {"name": "norm 8-bit prompt", "op": "norm_fp8", "rows": 8192, "hidden": 3584, "dtype": "bf16"},
        # the LM head of one decoding sequence: the weight's bytes are the work
        {"name": "head one token", "op": "linear", "tokens": 1, "inner": 3584, "outer": 152064, "out": "bf16"},
        # the LM head of a decoding batch
        {"name": "head batch of 64", "op": "linear", "tokens": 64, "inner": 3584, "outer": 128256, "out": "bf16"},
        # a small ragged layer: no dimension is a multiple of a tile
        {"name": "linear ragged", "op": "linear", "tokens": 37, "inner": 1040, "outer": 4100, "out": "fp32"},
        # a prompt through a wide layer: the tensor cores are the work
        {"name": "linear prompt", "op": "linear", "tokens": 2048, "inner": 3584, "outer": 32768, "out": "bf16"},
        # one sequence decoding at temperature 1
        {"name": "sample one row", "op": "sample", "rows": 1, "vocab": 151936, "dtype": "bf16", "spread": 3.0,
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mixed": False},
        # GRPO rollouts: many sequences, the whole distribution
        {"name": "sample rollouts", "op": "sample", "rows": 512, "vocab": 152064, "dtype": "bf16", "spread": 3.0,
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mixed": False},
        # a serving batch in which every request brings its own settings
        {"name": "sample mixed requests", "op": "sample", "rows": 64, "vocab": 128256, "dtype": "fp32", "spread": 2.5,
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mixed": True},
        # a flat nucleus over a vocabulary whose rows start at odd addresses
        {"name": "sample nucleus odd", "op": "sample", "rows": 128, "vocab": 50257, "dtype": "fp16", "spread": 2.0,
         "temperature": 0.8, "top_k": 0, "top_p": 0.95, "min_p": 0.0, "mixed": False},
    ]


def _log(rng, low, high):
    """A whole number between low and high, spread evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm_train", "norm_fp8", "linear", "sample"])
    if op in ("norm_train", "norm_fp8"):
        hidden = _log(rng, 128, 8192)
        if rng.random() < 0.7:
            hidden = max(128, hidden // 64 * 64)
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        most = 16384 * 3584 // (2 if dtype == "fp32" else 1)
        return {"op": op, "rows": min(_log(rng, 1, 16384), max(1, most // hidden)), "hidden": hidden, "dtype": dtype}
    if op == "linear":
        inner = 16 * _log(rng, 16, 512)
        outer = min(_log(rng, 500, 152064), 152064 * 3584 // inner)
        tokens = min(_log(rng, 1, 4096), max(1, 2048 * 3584 * 32768 // (inner * outer)), max(1, 2048 * 32768 // outer))
        return {"op": op, "tokens": tokens, "inner": inner, "outer": outer, "out": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    vocab = rng.choice([32000, 50257, 128256, 151936, 152064, _log(rng, 1000, 152064)])
    rows = min(_log(rng, 1, 1024), max(1, 512 * 152064 // vocab))
    kind = rng.choice(["whole", "top_k", "top_p", "both", "min_p", "mixed"])
    return {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "spread": round(rng.uniform(1.5, 5.0), 2), "temperature": round(rng.uniform(0.5, 1.3), 2),
            "top_k": _log(rng, 1, 1000) if kind in ("top_k", "both") else 0,
            "top_p": round(rng.uniform(0.5, 0.99), 3) if kind in ("top_p", "both") else 1.0,
            "min_p": round(rng.uniform(0.01, 0.2), 3) if kind == "min_p" else 0.0, "mixed": kind == "mixed"}


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

    if c["op"] in ("norm_train", "norm_fp8"):
        t = TYPES[c["dtype"]]
        n, h = c["rows"], c["hidden"]
        grad = c["op"] == "norm_train"
        # a layer's output and the stream it is added to, with the few large columns that streams have
        wide = torch.where(torch.rand(h, generator=g, device="cuda") < 0.01, 8.0, 1.0)
        s = {"case": c, "x": normal(n, h).to(t), "residual": (2.0 * normal(n, h) * wide).to(t),
             "weight": (1.0 + 0.1 * normal(h)).to(t)}
        if grad:
            s["g_y"], s["g_stream"] = normal(n, h).to(t), normal(n, h).to(t)
            for k in ("x", "residual", "weight"):
                s[k].requires_grad_(True)
        return s
    if c["op"] == "linear":
        m, k, n = c["tokens"], c["inner"], c["outer"]
        xq, xs = _quantise_rows(normal(m, k))
        wq, ws = _quantise_blocks(normal(n, k).mul_(k ** -0.5))
        return {"case": c, "xq": xq, "xs": xs, "wq": wq, "ws": ws}
    n, v = c["rows"], c["vocab"]
    z = normal(n, v).mul_(c["spread"])
    # half of the rows as a trained model leaves them: a few tokens stand out
    raised = torch.randint(0, v, (n, 24), generator=g, device="cuda")
    z[::2].scatter_add_(1, raised[::2], 4.0 * c["spread"] * torch.rand((n, 24), generator=g, device="cuda")[::2])
    s = {"case": c, "logits": z.to(TYPES[c["dtype"]]), "u": torch.rand(n, generator=g, device="cuda")}
    if c["mixed"]:
        def pick(values, dtype):
            at = torch.randint(0, len(values), (n,), generator=g, device="cuda")
            return torch.tensor(values, dtype=dtype, device="cuda")[at]
        s["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.2], torch.float32)
        s["top_k"] = pick([0, 0, 20, 50, 1000], torch.int32)
        s["top_p"] = pick([1.0, 1.0, 0.8, 0.9, 0.95], torch.float32)
        s["min_p"] = pick([0.0, 0.0, 0.0, 0.05, 0.1], torch.float32)
    else:
        s.update({k: c[k] for k in ("temperature", "top_k", "top_p", "min_p")})
    return s


# ------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------
def _plain_norm_train(s):
    # the stream is a stored tensor of the inputs' type; the norm reads what is stored
    t = s["x"].dtype
    with torch.no_grad():
        w = s["weight"].float()
        stream = (s["x"].float() + s["residual"].float()).to(t)
        f = stream.float()
        rstd = torch.rsqrt((f * f).mean(1, keepdim=True) + EPS)
        n = f * rstd
        y = (n * w).to(t)
        g = s["g_y"].float()
        gw = g * w
        d = (rstd * (gw - n * (gw * n).mean(1, keepdim=True)) + s["g_stream"].float()).to(t)
        dw = (g * n).sum(0).to(s["weight"].dtype)
        return {"y": y, "stream": stream, "dx": d, "dresidual": d, "dweight": dw}


def _plain_norm_fp8(s):
    t = s["x"].dtype
    stream = (s["x"].float() + s["residual"].float()).to(t)
    f = stream.float()
    q, scale = _quantise_rows(f * torch.rsqrt((f * f).mean(1, keepdim=True) + EPS) * s["weight"].float())
    return {"q": q, "scales": scale, "stream": stream}


def _plain_linear(s):
    k, n = s["xq"].shape[1], s["wq"].shape[0]
    x = s["xq"].float() * s["xs"].repeat_interleave(BLOCK, 1)[:, :k]
    w = s["wq"].float() * s["ws"].repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return {"y": (x @ w.t()).to(TYPES[s["case"]["out"]])}


def _setting(v, n, dtype):
    return v.to(dtype) if isinstance(v, torch.Tensor) else torch.full((n,), v, dtype=dtype, device="cuda")


def _plain_sample(s):
    # values and weights in 32 bits; the sums of weights in 64, because a token is a whole
    # number and must not hang on the order in which a row's weights were added
    n, v = s["logits"].shape
    t = _setting(s["temperature"], n, torch.float64)
    greedy = t == 0
    scale = (1.0 / torch.where(greedy, 1.0, t)).float()
    y = s["logits"].float() * scale[:, None]
    w = torch.exp(y - y.amax(1, keepdim=True))
    total = w.sum(1, dtype=torch.float64)
    # rank: the value downwards, the lowest index first among equals
    ws, order = torch.sort(w, dim=1, descending=True, stable=True)
    rank = torch.arange(v, device="cuda")
    k = _setting(s["top_k"], n, torch.int64)
    k = torch.where((k <= 0) | (k > v), v, k)
    keep = rank < k[:, None]
    wd = ws.double() * keep
    before = wd.cumsum(1) - wd
    p = _setting(s["top_p"], n, torch.float32).double()
    keep &= (before < p[:, None] * wd.sum(1, keepdim=True)) | (p[:, None] >= 1)
    keep &= ws >= _setting(s["min_p"], n, torch.float32)[:, None]
    keep[:, 0] = True
    keep &= (rank == 0) | ~greedy[:, None]
    kept = torch.zeros_like(wd).scatter_(1, order, ws.double() * keep)
    upto = kept.cumsum(1)
    mass = upto[:, -1]
    token = (upto <= (s["u"].double() * mass)[:, None]).sum(1)
    wt = w.gather(1, token[:, None])[:, 0].double().log()
    return {"token": token, "logprob": (wt - total.log()).float(), "kept_logprob": (wt - mass.log()).float()}


def _plain(s):
    return {"norm_train": _plain_norm_train, "norm_fp8": _plain_norm_fp8, "linear": _plain_linear,
            "sample": _plain_sample}[s["case"]["op"]](s)


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
    op = s["case"]["op"]
    if op == "norm_train":
        y, stream = ko.fused_residual_rmsnorm(s["x"], s["residual"], s["weight"], EPS)
        dx, dr, dw = torch.autograd.grad((y, stream), (s["x"], s["residual"], s["weight"]), (s["g_y"], s["g_stream"]))
        return {"y": y, "stream": stream, "dx": dx, "dresidual": dr, "dweight": dw}
    if op == "norm_fp8":
        q, scale, stream = ko.fused_residual_rmsnorm_fp8(s["x"], s["residual"], s["weight"], EPS)
        return {"q": q, "scales": scale, "stream": stream}
    if op == "linear":
        return {"y": ko.fp8_linear(s["xq"], s["xs"], s["wq"], s["ws"], TYPES[s["case"]["out"]])}
    token, logprob, kept = ko.sample_tokens(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return {"token": token, "logprob": logprob, "kept_logprob": kept}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    if case["op"] in ("norm_train", "norm_fp8"):
        n, h = case["rows"], case["hidden"]
        b = 4 if case["dtype"] == "fp32" else 2
        if case["op"] == "norm_train":
            # forward: x, residual in, y, stream out; backward: two gradients in, one out (the
            # stream again, since a step's own work lies between); the weight and its gradient
            return {"bytes": (8 * n * h + 2 * h) * b, "flops": 16 * n * h}
        return {"bytes": (3 * n * h + h) * b + n * h + 4 * n * _blocks(h), "flops": 8 * n * h}
    if case["op"] == "linear":
        m, k, n = case["tokens"], case["inner"], case["outer"]
        scales = 4 * _blocks(k) * (m + _blocks(n))
        return {"bytes": m * k + n * k + scales + m * n * (4 if case["out"] == "fp32" else 2), "flops": 2 * m * k * n}
    n, v = case["rows"], case["vocab"]
    return {"bytes": n * v * (4 if case["dtype"] == "fp32" else 2) + 20 * n, "flops": 6 * n * v}


# ------------------------------------------------------------------------------------------
# The same in 64 bits
# ------------------------------------------------------------------------------------------
def _exact_norm(s, train):
    x, r, w = (s[k].detach().double() for k in ("x", "residual", "weight"))
    n, h = x.shape
    total = x + r
    f = total.to(s["x"].dtype).double()  # the stream as it is stored
    norm = f / (f.square().sum(1, keepdim=True) / h + EPS).sqrt()
    if train:
        inv = norm.norm(dim=1, keepdim=True) / f.norm(dim=1, keepdim=True)
        gy = s["g_y"].double()
        along = (gy * w * norm).sum(1, keepdim=True) / h
        d = inv * gy * w - inv * along * norm + s["g_stream"].double()
        return {"y": norm * w, "stream": total, "dx": d, "dresidual": d, "dweight": torch.einsum("nh,nh->h", gy, norm)}
    y = norm * w
    scale = torch.empty(n, _blocks(h), dtype=torch.float64, device=y.device)
    q = torch.empty_like(y)
    for b, part in enumerate(y.split(BLOCK, 1)):
        scale[:, b] = part.abs().amax(1).clamp(min=AMAX_FLOOR) / FP8_MAX
        q[:, b * BLOCK:b * BLOCK + part.shape[1]] = (part / scale[:, b:b + 1]).to(FP8).double()
    return {"q": q, "scales": scale, "stream": total}


def _exact_linear(s):
    m, k = s["xq"].shape
    n = s["wq"].shape[0]
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    of_row = torch.arange(n, device="cuda") // BLOCK
    for b in range(_blocks(k)):
        at = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
        y += (s["xq"][:, at].double() @ s["wq"][:, at].double().t()) * s["xs"][:, b:b + 1].double() * s["ws"][:, b].double()[of_row]
    return {"y": y}


def _exact_sample(s):
    n, v = s["logits"].shape
    per_row = {k: s[k].tolist() if isinstance(s[k], torch.Tensor) else [s[k]] * n
               for k in ("temperature", "top_k", "top_p", "min_p")}
    logprob, kept_logprob = [], []
    for i in range(n):
        t = per_row["temperature"][i]
        y = s["logits"][i].double() * torch.tensor(1.0 / t if t else 1.0).float().item()
        logp = torch.log_softmax(y, 0)
        down, order = torch.sort(logp, descending=True, stable=True)
        k = per_row["top_k"][i]
        down = down[:k if 0 < k < v else v]
        prob = down.exp()
        if per_row["top_p"][i] < 1:
            cum = prob.cumsum(0) / prob.sum()
            down = down[:1 + int((cum[:-1] < per_row["top_p"][i]).sum())]
        if per_row["min_p"][i] > 0:
            down = down[:max(1, int((down - down[0] >= math.log(per_row["min_p"][i])).sum()))]
        if not t:
            down = down[:1]
        index, back = torch.sort(order[:down.numel()])
        inner = down[back] - torch.logsumexp(down, 0)
        cum = inner.exp().cumsum(0)
        at = min(int(torch.searchsorted(cum, s["u"][i].double(), right=True)), index.numel() - 1)
        logprob.append(logp[index[at]])
        kept_logprob.append(inner[at])
    return {"token": None, "logprob": torch.stack(logprob), "kept_logprob": torch.stack(kept_logprob)}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "linear":
        return _exact_linear(s)
    if op == "sample":
        return _exact_sample(s)
    return _exact_norm(s, op == "norm_train")
