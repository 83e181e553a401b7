"""The training operators of llm_hgemm as they are measured: the cases, their inputs, a plain
form of each operator in elementary torch operations, and the calls a user makes.

Three operators, in the order of a training step: the gated feed-forward block and its
backward pass, the softmax cross entropy of a language-model head (taken from the hidden
states and the head's weight, with its gradient), and the orthogonalised update of a weight
(Newton-Schulz products, as the Muon optimiser takes it).
"""

import os
import sys

import torch

own = False   # the calls of the framework's operators instead of the plain forms

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
IGNORE = -100
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # Gated feed-forward block. "forward" is the block alone (evaluation, or one
        # token while a model under training is sampled from), "step" forward and backward.
        {"name": "ffn 1 token", "op": "ffn", "pass": "forward", "tokens": 1, "hidden": 2560,
         "inter": 9728, "dtype": "fp16"},        # one token of the 4B model's block: streams the weights
        {"name": "ffn small step", "op": "ffn", "pass": "step", "tokens": 24, "hidden": 256,
         "inter": 688, "dtype": "bf16"},         # a test-sized model: launches and latency
        {"name": "ffn odd step", "op": "ffn", "pass": "step", "tokens": 509, "hidden": 1024,
         "inter": 2816, "dtype": "bf16"},        # a short ragged batch of a small model
        {"name": "ffn 4B step", "op": "ffn", "pass": "step", "tokens": 4096, "hidden": 2560,
         "inter": 9728, "dtype": "fp16"},        # the 4B model's block on a full micro-batch
        # Cross entropy from the hidden states. "forward" scores a text (perplexity).
        {"name": "loss small step", "op": "loss", "pass": "step", "tokens": 24, "hidden": 256,
         "vocab": 4001, "reduction": "mean", "dtype": "fp16"},      # test-sized, odd vocabulary
        {"name": "loss odd step", "op": "loss", "pass": "step", "tokens": 777, "hidden": 1024,
         "vocab": 50257, "reduction": "none", "dtype": "bf16"},     # weighted tokens, a prime-ish vocabulary
        {"name": "loss 4B scoring", "op": "loss", "pass": "forward", "tokens": 2048, "hidden": 2560,
         "vocab": 151936, "reduction": "none", "dtype": "fp16"},    # a prompt's log-likelihoods
        {"name": "loss 4B step", "op": "loss", "pass": "step", "tokens": 4096, "hidden": 2560,
         "vocab": 151936, "reduction": "mean", "dtype": "bf16"},    # the head of a full micro-batch
        # Orthogonalised updates, of matrices as the models above have them.
        {"name": "orth small", "op": "orth", "batch": 1, "rows": 256, "cols": 96, "dtype": "bf16"},
        {"name": "orth stacked odd", "op": "orth", "batch": 4, "rows": 333, "cols": 1001, "dtype": "fp16"},
        {"name": "orth key projection", "op": "orth", "batch": 1, "rows": 1024, "cols": 2560, "dtype": "bf16"},
        {"name": "orth 4B gate", "op": "orth", "batch": 1, "rows": 9728, "cols": 2560, "dtype": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    largest = {op: max(work(c)["flops"] for c in listed() if c["op"] == op) for op in ("ffn", "loss", "orth")}
    while True:
        op = rng.choice(("ffn", "loss", "orth"))
        case = {"op": op, "dtype": rng.choice(("fp16", "bf16"))}
        if op == "ffn":
            case["pass"] = rng.choice(("forward", "step", "step"))
            case["tokens"] = _spread(rng, 1, 4096)
            case["hidden"] = 8 * _spread(rng, 8, 320)
            case["inter"] = 8 * _spread(rng, 16, 1216)
        elif op == "loss":
            case["pass"] = rng.choice(("forward", "step", "step"))
            case["reduction"] = rng.choice(("mean", "sum", "none"))
            case["tokens"] = _spread(rng, 1, 4096)
            case["hidden"] = 8 * _spread(rng, 8, 320)
            case["vocab"] = _spread(rng, 500, 151936)
        else:
            case["batch"] = rng.choice((1, 1, 1, 2, 3, 4))
            case["rows"] = _spread(rng, 16, 9728)
            case["cols"] = _spread(rng, 16, 9728)
        if work(case)["flops"] <= largest[op]:
            return case


# ----------------------------------------------------------------- inputs ----

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    step = case.get("pass") == "step"
    state = {"case": dict(case)}
    if case["op"] == "ffn":
        t, h, i = case["tokens"], case["hidden"], case["inter"]
        state["x"] = normal(t, h).requires_grad_(step)                 # a norm's output: about 1
        for name, shape in (("gate", (i, h)), ("up", (i, h)), ("down", (h, i))):
            state[name] = normal(*shape, scale=shape[1] ** -0.5).requires_grad_(step)
        state["dy"] = normal(t, h)                                     # with the loss scale on it
    elif case["op"] == "loss":
        t, h, v = case["tokens"], case["hidden"], case["vocab"]
        weight = normal(v, h, scale=h ** -0.5)
        target = torch.randint(0, v, (t,), generator=gen, device="cuda")
        # A model that has learnt something: the target's logit lies 0 to 8 above the others'.
        known = torch.rand((t, 1), generator=gen, device="cuda") * 8
        x = (torch.randn((t, h), generator=gen, device="cuda") + known * weight[target].float()).to(dtype)
        skip = torch.rand((t,), generator=gen, device="cuda") < 0.1    # prompt or padding tokens
        skip[0] = False
        state["target"] = torch.where(skip, torch.full_like(target, IGNORE), target)
        state["x"], state["weight"] = x.requires_grad_(step), weight.requires_grad_(step)
        scale = 1024.0 if dtype == torch.float16 else 1.0              # a loss scale, as fp16 training has
        if case["reduction"] == "none":
            state["dloss"] = torch.rand((t,), generator=gen, device="cuda") * scale / t
        else:
            state["dloss"] = torch.full((), scale / (t if case["reduction"] == "sum" else 1), device="cuda")
    else:
        # A gradient's spectrum: a few strong directions over noise, and its small values.
        b, m, n = case["batch"], case["rows"], case["cols"]
        k = min(m, n, 16)
        strong = torch.randn((b, m, k), generator=gen, device="cuda") @ torch.randn((b, k, n), generator=gen, device="cuda")
        g = torch.randn((b, m, n), generator=gen, device="cuda") + strong * (0.5 * k ** -0.5)
        g = (g * 1e-3).to(dtype)
        state["g"] = g[0] if b == 1 else g
    return state


# -------------------------------------------------------------- plain form ----

def _plain_ffn(s):
    x, gate, up, down = (s[k].detach().float() for k in ("x", "gate", "up", "down"))
    dtype = s["x"].dtype
    g, u = x @ gate.t(), x @ up.t()
    sig = 1 / (1 + torch.exp(-g))
    h = g * sig * u
    y = (h @ down.t()).to(dtype)
    if s["case"]["pass"] == "forward":
        return y
    dy = s["dy"].float()
    dh = dy @ down
    du = dh * (g * sig)
    dg = dh * u * (sig * (1 + g * (1 - sig)))
    dx = dg @ gate + du @ up
    return [y] + [t.to(dtype) for t in (dx, dg.t() @ x, du.t() @ x, dy.t() @ h)]


def _plain_loss(s):
    x, weight, target = s["x"].detach().float(), s["weight"].detach().float(), s["target"]
    dtype, reduction = s["x"].dtype, s["case"]["reduction"]
    logits = x @ weight.t()
    top = logits.max(dim=1, keepdim=True).values
    p = torch.exp(logits - top)
    total = p.sum(dim=1, keepdim=True)
    keep = target != IGNORE
    at = torch.where(keep, target, torch.zeros_like(target)).unsqueeze(1)
    loss = (torch.log(total) + top - logits.gather(1, at)).squeeze(1) * keep
    count = keep.sum()
    out = loss if reduction == "none" else loss.double().sum() / (count if reduction == "mean" else 1)
    out = out.float()
    if s["case"]["pass"] == "forward":
        return out
    del logits
    row = s["dloss"] * keep / (count if reduction == "mean" else 1)
    p /= total
    p.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    p *= row.unsqueeze(1)
    return [out, (p @ weight).to(dtype), (p.t() @ x).to(dtype)]


def _plain_orth(s):
    g = s["g"].float()
    tall = g.shape[-2] > g.shape[-1]
    x = g.mT if tall else g
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        p = x @ x.mT
        x = a * x + (b * p + c * (p @ p)) @ x
    return (x.mT if tall else x).to(s["g"].dtype).contiguous()


# --------------------------------------------------------------------- run ----

def _package():
    """The package lies in a folder of its own below the repository's root."""
    try:
        import llm_hgemm
    except ImportError:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(root, "llm-tensorcore-hgemm_b200"))
        import llm_hgemm
    return llm_hgemm


def run(state):
    case = state["case"]
    if not own:
        return {"ffn": _plain_ffn, "loss": _plain_loss, "orth": _plain_orth}[case["op"]](state)
    lib = _package()
    if case["op"] == "ffn":
        leaves = [state[k] for k in ("x", "gate", "up", "down")]
        y = lib.gated_ffn(*leaves)
        if case["pass"] == "forward":
            return y
        return [y.detach(), *torch.autograd.grad(y, leaves, state["dy"])]
    if case["op"] == "loss":
        leaves = [state["x"], state["weight"]]
        loss = lib.linear_cross_entropy(*leaves, state["target"], reduction=case["reduction"], ignore_index=IGNORE)
        if case["pass"] == "forward":
            return loss
        return [loss.detach(), *torch.autograd.grad(loss, leaves, state["dloss"])]
    return lib.orthogonalize(state["g"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)


# -------------------------------------------------------------------- work ----

def work(case):
    if case["op"] == "ffn":
        t, h, i = case["tokens"], case["hidden"], case["inter"]
        products = 3 if case["pass"] == "forward" else 9
        elements = (2 * t * h + 3 * h * i) if case["pass"] == "forward" else (4 * t * h + 6 * h * i)
        return {"bytes": 2 * elements, "flops": 2 * products * t * h * i}
    if case["op"] == "loss":
        t, h, v = case["tokens"], case["hidden"], case["vocab"]
        loss = 4 * (t if case["reduction"] == "none" else 1)
        if case["pass"] == "forward":
            return {"bytes": 2 * h * (t + v) + 8 * t + loss, "flops": 2 * t * h * v}
        # The logits, and the two products of their gradient.
        return {"bytes": 4 * h * (t + v) + 8 * t + 2 * loss, "flops": 6 * t * h * v}
    b, m, n = case["batch"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # A step: X X^T and its square, symmetric (half of each to compute), and the product with X.
    return {"bytes": 4 * b * m * n, "flops": STEPS * b * (m * m * n + m ** 3 + 2 * m * m * n)}


# ------------------------------------------------------------- in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "ffn":
        names = ("x", "gate", "up", "down")
        leaves = [wide[k].requires_grad_(case["pass"] == "step") for k in names]
        x, gate, up, down = leaves
        pre = torch.matmul(x, gate.T)
        y = torch.matmul(pre * torch.sigmoid(pre) * torch.matmul(x, up.T), down.T)
        if case["pass"] == "forward":
            return y
        return [y.detach(), *torch.autograd.grad(y, leaves, wide["dy"])]
    if case["op"] == "loss":
        x, weight, target = wide["x"], wide["weight"], s["target"]
        rows = torch.nonzero(target != IGNORE).squeeze(1)
        loss = torch.zeros(len(target), dtype=torch.float64, device=x.device)
        scale = wide["dloss"].expand(len(target))
        if case["reduction"] == "mean":
            scale = scale / len(rows)
        dx, dw = torch.zeros_like(x), torch.zeros_like(weight)
        for part in rows.split(1024):   # the kept tokens, some at a time
            logp = torch.log_softmax(torch.matmul(x[part], weight.T), dim=-1)
            each = torch.arange(len(part), device=x.device)
            loss[part] = -logp[each, target[part]]
            if case["pass"] == "step":
                d = logp.exp_()
                d[each, target[part]] -= 1
                d *= scale[part, None]
                dx[part] = torch.matmul(d, weight)
                dw += torch.matmul(d.T, x[part])
        out = {"none": loss, "sum": loss.sum(), "mean": loss.sum() / len(rows)}[case["reduction"]]
        return out if case["pass"] == "forward" else [out, dx, dw]
    # The same polynomial on the other side's Gram matrix where that is the smaller one, by Horner's rule.
    g = wide["g"]
    a, b, c = COEFFICIENTS
    x = g / (torch.linalg.vector_norm(g, dim=(-2, -1), keepdim=True) + EPS)
    left = g.shape[-2] <= g.shape[-1]
    eye = torch.eye(min(g.shape[-2:]), dtype=torch.float64, device=g.device)
    for _ in range(STEPS):
        gram = torch.matmul(x, x.mT) if left else torch.matmul(x.mT, x)
        poly = a * eye + torch.matmul(gram, b * eye + c * gram)
        x = torch.matmul(poly, x) if left else torch.matmul(x, poly)
    return x
