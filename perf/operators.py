"""Operators at the output end of a language model, as timed cases: in their plain form, elementary torch operations, and as
this framework's calls.

    logprobs   what a model says about given tokens: the log probability of each row's token, the entropy of the row and its
               most probable tokens: `Context.token_logprobs`
    policy     the same without the list, and the gradient of the logits from gradients of log probabilities and entropies (a
               policy's training step): `Context.token_logprobs`, `Context.token_logprobs_backward`
    distill    the loss of a student against a teacher's most probable tokens, and its gradient: `Context.distillation_loss`,
               in one call or, as autograd asks for it, with `Context.distillation_loss_backward`
    norm       layer norm: `Context.layernorm`, and with "step" its backward pass, the reduction of the weight's and the
               bias's gradients in it: `Context.layernorm_backward`
"""
import math

import torch

own = False


def listed():
    return [
        # one token being generated, with the alternatives that a client asks for
        {"name": "logprobs_1", "kind": "logprobs", "rows": 1, "vocab": 32000, "pad": 0, "top": 20, "masked": 0.0, "rounded": False, "temperature": 1.0},
        # sixteen sequences being generated, a vocabulary of odd size, logits that a 16-bit classifier rounded (equal values)
        {"name": "logprobs_16", "kind": "logprobs", "rows": 16, "vocab": 64001, "pad": 0, "top": 5, "masked": 0.0, "rounded": True, "temperature": 0.7},
        # the trainer's batch of 16 x 256 tokens scored by a teacher
        {"name": "logprobs_4096", "kind": "logprobs", "rows": 4096, "vocab": 32000, "pad": 0, "top": 20, "masked": 0.0, "rounded": False, "temperature": 1.0},
        # a ragged batch whose rows end in padding, with most of the vocabulary ruled out
        {"name": "logprobs_777", "kind": "logprobs", "rows": 777, "vocab": 12345, "pad": 7, "top": 64, "masked": 0.9, "rounded": False, "temperature": 1.3},
        # a policy's step on the trainer's batch
        {"name": "policy_4096", "kind": "policy", "rows": 4096, "vocab": 32000, "pad": 0, "masked": 0.0, "rounded": False, "temperature": 1.0},
        # a short one over a vocabulary of odd size
        {"name": "policy_300", "kind": "policy", "rows": 300, "vocab": 10007, "pad": 0, "masked": 0.0, "rounded": True, "temperature": 0.7},
        # the trainer's batch against the 64 tokens that a teacher kept of each row
        {"name": "distill_4096", "kind": "distill", "rows": 4096, "vocab": 32000, "pad": 0, "top": 64, "split": False, "temperature": 2.0},
        # a ragged batch, forward and backward pass called one after the other, rows padded to whole tiles
        {"name": "distill_500", "kind": "distill", "rows": 500, "vocab": 32000, "pad": 64, "top": 20, "split": True, "temperature": 1.0},
        # a micro-batch
        {"name": "distill_32", "kind": "distill", "rows": 32, "vocab": 8001, "pad": 0, "top": 10, "split": False, "temperature": 1.5},
        # one token being generated
        {"name": "norm_1x4096", "kind": "norm", "rows": 1, "cols": 4096, "step": False},
        # the trainer's rows
        {"name": "norm_4096x288", "kind": "norm", "rows": 4096, "cols": 288, "step": True},
        # the 1B-scale configuration at its full token count
        {"name": "norm_16384x2048", "kind": "norm", "rows": 16384, "cols": 2048, "step": True},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(["logprobs", "logprobs", "policy", "policy", "distill", "distill", "norm", "norm"])
    if kind == "norm":
        cols = rng.choice([_spread(rng, 64, 8192), 4 * _spread(rng, 16, 2048)])
        return {"kind": kind, "rows": _spread(rng, 1, 16384 * 2048 // cols), "cols": cols, "step": rng.random() < 0.7}
    vocab = rng.choice([_spread(rng, 500, 64000), 32000])
    case = {"kind": kind, "rows": _spread(rng, 1, 4096 * 32000 // (vocab + 64)), "vocab": vocab, "pad": rng.choice([0, 0, 3, 64]),
            "temperature": rng.choice([0.5, 0.7, 1.0, 1.0, 1.3, 2.0])}
    if kind != "policy":
        case["top"] = _spread(rng, 1, 64)
    if kind == "distill":
        case["split"] = rng.random() < 0.5
    else:
        case["masked"], case["rounded"] = rng.choice([0.0, 0.0, 0.5, 0.95]), rng.random() < 0.4
    return case


# -- inputs ----------------------------------------------------------------------------------------------------------

def _logits(g, rows, vocab, pad, rounded=False, masked=0.0):
    """Rows as a classifier writes them: a bell with a few tokens far above it, [rows, vocab + pad] of which `vocab` columns are read."""
    x = torch.randn(rows, vocab + pad, device="cuda", generator=g).mul_(1.5)
    at = (torch.randint(0, vocab, (rows, 1), device="cuda", generator=g) + torch.arange(24, device="cuda") * (vocab // 24)).remainder_(vocab)
    x.scatter_(1, at, torch.rand(rows, 24, device="cuda", generator=g).mul_(9.0).add_(3.0))
    if rounded:
        x = x.bfloat16().float()
    if masked:
        x.masked_fill_(torch.rand(rows, vocab + pad, device="cuda", generator=g) < masked, -math.inf)
        x[:, rows % vocab] = 1.0                       # at least one token is left
    return x


def _context():
    """A program has one context for its stream, whatever inputs it meets."""
    if not hasattr(_context, "kept"):
        from motifcl_b200 import Context
        _context.kept = Context.on_torch_stream(torch.cuda.current_device())
    return _context.kept


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["kind"] == "norm":
        R, C = case["rows"], case["cols"]
        s["x"] = torch.randn(R, C, device="cuda", generator=g).mul_(1.7).add_(torch.randn(R, 1, device="cuda", generator=g))
        s["weight"] = torch.rand(C, device="cuda", generator=g) + 0.5
        s["bias"] = torch.randn(C, device="cuda", generator=g).mul_(0.1)
        s["dy"] = torch.randn(R, C, device="cuda", generator=g).mul_(0.02)
        if own:
            s["ctx"] = _context()
        return s
    R, V = case["rows"], case["vocab"]
    s["logits"] = x = _logits(g, R, V, case["pad"], case.get("rounded", False), case.get("masked", 0.0))
    if case["kind"] == "distill":
        # a teacher that agrees with the student here and there
        start = torch.randint(0, V, (R, 1), device="cuda", generator=g)
        s["ids"] = (start + torch.arange(case["top"], device="cuda") * (V // case["top"])).remainder_(V).int()
        s["ids"][:, :1] = x[:, :V].argmax(dim=1, keepdim=True).int()
        s["ids"][:, 1:].masked_fill_(s["ids"][:, 1:] == s["ids"][:, :1], -1)      # a teacher names a token once; shorter lists end in -1
        s["teacher"] = torch.randn(R, case["top"], device="cuda", generator=g).mul_(2.0).sort(dim=1, descending=True).values
        s["one"] = torch.ones(1, device="cuda")
        if R > 8:
            s["ids"][R // 2:R // 2 + R // 16 + 1] = -1                              # padding between sequences
    else:
        gumbel = torch.rand(R, V, device="cuda", generator=g).clamp_(min=1e-20).log_().neg_().log_().neg_()
        s["tokens"] = gumbel.add_(x[:, :V], alpha=1.0 / case["temperature"]).argmax(dim=1).int()       # sampled from the row
        if R > 8:
            s["tokens"][R // 2:R // 2 + R // 16 + 1] = -1
        if case["kind"] == "policy":
            s["dlogp"] = torch.randn(R, device="cuda", generator=g).div_(R)
            s["dent"] = torch.full((R,), -0.01 / R, device="cuda")
    if own:
        s["ctx"] = _context()
    return s


# -- the plain forms -------------------------------------------------------------------------------------------------

def _softmax_parts(x, temperature):
    """z - max z, its exponentials and their sum, for z = x / temperature."""
    d = (x - x.amax(dim=1, keepdim=True)) / temperature
    e = d.exp()
    return d, e, e.sum(dim=1, keepdim=True)


def _plain_logprobs(s):
    x, tokens = s["logits"][:, :s["vocab"]], s["tokens"].long()
    d, e, total = _softmax_parts(x, s["temperature"])
    valid = tokens >= 0
    log_total = total.log()
    picked = d.gather(1, tokens.clamp(min=0)[:, None]) - log_total
    logp = torch.where(valid, picked[:, 0], torch.zeros_like(picked[:, 0]))
    p = e / total
    weighted = torch.where(p > 0, p * d, torch.zeros_like(p))
    return logp, log_total[:, 0] - weighted.sum(dim=1), d, p, log_total


def _plain_top(x, k):
    """The k largest of each row, largest first, equal ones by their place: one whole number that orders both."""
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    key = key * (1 << 32) + (x.shape[1] - torch.arange(x.shape[1], device=x.device))
    return x.shape[1] - (key.topk(k, dim=1).values & 0xFFFFFFFF)


def _run_plain(s):
    kind = s["kind"]
    if kind == "logprobs":
        logp, entropy, d, p, log_total = _plain_logprobs(s)
        ids = _plain_top(s["logits"][:, :s["vocab"]], s["top"])
        return [logp, entropy, ids.int(), d.gather(1, ids) - log_total]
    if kind == "policy":
        logp, entropy, d, p, log_total = _plain_logprobs(s)
        tokens = s["tokens"].long()
        up = torch.where(tokens >= 0, s["dlogp"], torch.zeros_like(s["dlogp"]))[:, None]
        log_p = torch.where(p > 0, d - log_total, torch.zeros_like(d))
        grad = -up * p - s["dent"][:, None] * p * (log_p + entropy[:, None])
        grad.scatter_add_(1, tokens.clamp(min=0)[:, None], up)
        return [logp, entropy, grad / s["temperature"]]
    if kind == "distill":
        x, ids, T = s["logits"][:, :s["vocab"]], s["ids"].long(), s["temperature"]
        d, e, total = _softmax_parts(x, T)
        valid = ids >= 0
        any_valid = valid.any(dim=1, keepdim=True)
        at = ids.clamp(min=0)
        a = torch.where(valid, s["teacher"], torch.full_like(s["teacher"], -math.inf))
        a = torch.where(any_valid, a, torch.zeros_like(a))
        b, w, sum_w = _softmax_parts(a, T)
        t = torch.where(valid, w / sum_w, torch.zeros_like(w))
        log_ratio = torch.where(t > 0, b - sum_w.log() - (d.gather(1, at) - total.log()), torch.zeros_like(t))
        losses = (t * log_ratio).sum(dim=1)
        grad = (e / total) * any_valid
        grad.scatter_add_(1, at, -t)
        return [losses, losses.mean().reshape(1), grad / (T * x.shape[0])]
    x, w = s["x"], s["weight"]
    centred = x - x.mean(dim=1, keepdim=True)
    inv = 1.0 / ((centred * centred).mean(dim=1, keepdim=True) + 1e-5).sqrt()
    normed = centred * inv
    y = normed * w + s["bias"]
    if not s["step"]:
        return [y]
    dy = s["dy"]
    gw = dy * w
    dx = inv * (gw - gw.mean(dim=1, keepdim=True) - normed * (gw * normed).mean(dim=1, keepdim=True))
    return [y, dx, (dy * normed).sum(dim=0), dy.sum(dim=0)]


# -- the framework's calls ---------------------------------------------------------------------------------------------

def _run_own(s):
    ctx, kind = s["ctx"], s["kind"]
    if kind == "norm":
        x, R, C = s["x"], s["rows"], s["cols"]
        y = torch.empty_like(x)
        if not s["step"]:
            ctx.layernorm(x, s["weight"], s["bias"], y, None, R, C, 1e-5)
            return [y]
        stats, dx, dw, db = torch.empty(R, 2, device="cuda"), torch.empty_like(x), torch.empty_like(s["weight"]), torch.empty_like(s["bias"])
        ctx.layernorm(x, s["weight"], s["bias"], y, stats, R, C, 1e-5)
        ctx.layernorm_backward(x, s["weight"], s["dy"], stats, dx, dw, db, R, C)
        return [y, dx, dw, db]
    x, R, V, T = s["logits"], s["rows"], s["vocab"], s["temperature"]
    stride = V + s["pad"]
    if kind == "distill":
        losses, loss, grad = torch.empty(R, device="cuda"), torch.empty(1, device="cuda"), torch.empty_like(x)
        if s["split"]:
            stats = torch.empty(R, 2, device="cuda")
            ctx.distillation_loss(x, s["ids"], s["teacher"], losses, loss, stats, None, None, R, V, s["top"], T, stride)
            ctx.distillation_loss_backward(x, s["ids"], s["teacher"], stats, s["one"], grad, R, V, s["top"], T, stride)
        else:
            ctx.distillation_loss(x, s["ids"], s["teacher"], losses, loss, None, s["one"], grad, R, V, s["top"], T, stride)
        return [losses, loss, grad[:, :V]]
    logp, entropy = torch.empty(R, device="cuda"), torch.empty(R, device="cuda")
    if kind == "logprobs":
        ids, top = torch.empty(R, s["top"], dtype=torch.int32, device="cuda"), torch.empty(R, s["top"], device="cuda")
        ctx.token_logprobs(x, s["tokens"], logp, entropy, ids, top, None, R, V, s["top"], T, stride)
        return [logp, entropy, ids, top]
    stats, grad = torch.empty(R, 2, device="cuda"), torch.empty_like(x)
    ctx.token_logprobs(x, s["tokens"], logp, entropy, None, None, stats, R, V, 0, T, stride)
    ctx.token_logprobs_backward(x, s["tokens"], stats, entropy, s["dlogp"], s["dent"], grad, R, V, T, stride)
    return [logp, entropy, grad[:, :V]]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# -- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    if case["kind"] == "norm":
        R, C = case["rows"], case["cols"]
        if not case["step"]:
            return {"bytes": 8.0 * R * C + 8.0 * C, "flops": 8.0 * R * C}
        return {"bytes": 16.0 * R * C + 16.0 * C, "flops": 20.0 * R * C}          # x and dy in, y and dx out
    n, R = float(case["rows"]) * case["vocab"], case["rows"]
    if case["kind"] == "logprobs":
        return {"bytes": 4.0 * n + R * (12.0 + 8.0 * case["top"]), "flops": 6.0 * n}
    if case["kind"] == "policy":
        return {"bytes": 8.0 * n + 20.0 * R, "flops": 14.0 * n}
    return {"bytes": 8.0 * n + R * (4.0 + 8.0 * case["top"]), "flops": 8.0 * n}


# -- the definitions in 64 bits --------------------------------------------------------------------------------------

def _exact_rows(s, r0, r1):
    """Results of rows r0 to r1 of one of the kinds over a vocabulary; gradients by differentiation."""
    V, T = s["vocab"], s["temperature"]
    z = (s["logits"][r0:r1, :V].double() / T).requires_grad_(s["kind"] != "logprobs")
    lse = torch.logsumexp(z, dim=1)
    rows = torch.arange(r1 - r0, device=z.device)
    if s["kind"] == "distill":
        ids = s["ids"][r0:r1].long()
        t = torch.softmax((s["teacher"][r0:r1].double() / T).masked_fill(ids < 0, -math.inf), dim=1).nan_to_num(nan=0.0)
        log_q = z[rows[:, None], ids.clamp(min=0)] - lse[:, None]
        losses = torch.special.xlogy(t, t).sum(dim=1) - torch.where(t > 0, t * log_q, 0.0).sum(dim=1)
        grad, = torch.autograd.grad(losses.sum() / s["rows"], z)
        return [losses.detach(), grad / T]
    tokens = s["tokens"][r0:r1].long()
    logp = torch.where(tokens >= 0, z[rows, tokens.clamp(min=0)] - lse, 0.0)
    q = torch.exp(z - lse[:, None])
    entropy = lse - (q * z.masked_fill(z == -math.inf, 0.0)).sum(dim=1)
    if s["kind"] == "policy":
        grad, = torch.autograd.grad((logp * s["dlogp"][r0:r1]).sum() + (entropy * s["dent"][r0:r1]).sum(), z)
        return [logp.detach(), entropy.detach(), grad / T]
    order = torch.sort(s["logits"][r0:r1, :V], dim=1, descending=True, stable=True).indices[:, :s["top"]]
    return [logp, entropy, order.int(), z.gather(1, order) - lse[:, None]]


def exact(case, seed):
    global own
    asked, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = asked
    if case["kind"] != "norm":
        step = max(1, (1 << 25) // case["vocab"])
        parts = [_exact_rows(s, r, min(case["rows"], r + step)) for r in range(0, case["rows"], step)]
        out = [torch.cat(p) for p in zip(*parts)]
        if case["kind"] == "distill":
            out.insert(1, out[0].mean().reshape(1))
        return out
    x, w, b = (s[k].double().requires_grad_(case["step"]) for k in ("x", "weight", "bias"))
    var, mean = torch.var_mean(x, dim=1, keepdim=True, correction=0)
    y = (x - mean) / torch.sqrt(var + 1e-5) * w + b
    if not case["step"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, (x, w, b), s["dy"].double())]
