"""Rows of logits: log probabilities of given tokens with entropies and most probable tokens, their gradient, and the loss against a
teacher's kept tokens with its gradient, against the definitions in float64.

Tolerances come from the roundings of the fp32 arithmetic, with u = 2^-24 (half a last bit), d = (x - m) / T <= 0, m the row's largest:
    d            x - m, 1 / T and their product round: |d| (1 + u)^3, so 3 u |d|
    e = exp(d)   its argument d log2(e) has 4 roundings (4 u |d|), the exponential 2 last bits (4 u): relative 4 u |d| + 4 u
    s = sum e    an fp32 sum is off by at most u per addition that a term goes through: those of a thread (n / 512, or n / (512 CTAs)),
                 then 4 + 16 + 8 across warps and CTAs, and one rescaling (5 u): S(n) = n / 512 + 40, besides the terms' own 4 u (|d| + 1)
                 weighted with p: 4 u (E|d| + 1)
    ln s         2 last bits of the result (4 u |ln s|) and s's relative error
    ln p         the sum of both, and one more rounding (u |ln p|)
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NEG = -math.inf
LOWEST = float(np.finfo(np.float32).min)


class Row64:
    """The definition in float64 of fp32 logits, and the tolerances above.  x [R, V] fp32 on any device."""

    def __init__(self, x, T):
        x = x.detach().cpu().double()
        self.x, self.T = x, float(np.float32(T))
        self.V = x.shape[1]
        m = x.amax(dim=1, keepdim=True)
        self.dead = (m == NEG)                                    # nothing is left
        self.d = torch.where(self.dead, torch.full_like(x, NEG), (x - m) / self.T)
        e = torch.exp(self.d)
        self.s = e.sum(dim=1, keepdim=True)
        self.p = torch.where(self.dead, torch.zeros_like(e), e / self.s)
        self.logp = self.d - torch.log(self.s)
        self.logp = torch.where(self.dead, torch.full_like(x, NEG), self.logp)
        fin = torch.where(self.p > 0, self.d, torch.zeros_like(x))
        mean_d = (self.p * fin.abs()).sum(dim=1, keepdim=True)
        self.H = torch.where(self.dead, torch.zeros_like(m), torch.log(self.s) + mean_d)
        sums = self.V / 512 + 40
        self.tol_s = U * (4 * (mean_d + 1) + sums)                  # relative
        ls = torch.log(self.s).abs().nan_to_num(posinf=0.0)
        fin_all = self.d.nan_to_num(neginf=0.0)
        self.tol_logp = 3 * U * fin_all.abs() + 4 * U * ls + self.tol_s + U * self.logp.nan_to_num(neginf=0.0).abs()
        # a = sum e d: terms have d's error twice (in e and as a factor): p (4 d^2 + 8 |d|) u, its additions, then a / s
        sq = (self.p * fin * fin).sum(dim=1, keepdim=True)
        self.tol_H = 4 * U * ls + self.tol_s * (1 + mean_d) + U * (4 * sq + 8 * mean_d + sums * mean_d) + 4 * U * (self.H + mean_d)
        self.tol_p = self.p * (4 * U * (fin_all.abs() + 2) + self.tol_s)


def near(got, want, tol, what=""):
    got, want = got.detach().cpu().double(), want.double()
    want = torch.where(want.abs() > -LOWEST, torch.sign(want) * math.inf, want)      # beyond fp32
    tol = torch.broadcast_to(torch.as_tensor(tol, dtype=torch.float64), want.shape)
    assert got.shape == want.shape, what
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), what
    err = (got - want)[fin].abs()
    # 1e-35: exponentials below 2^-126 are 0, times what they are multiplied with (a few hundred at most)
    assert bool((err <= tol[fin] + 1e-35).all()), (what, float((err / (tol[fin] + 1e-35)).max()), float(err.max()))


def make_logits(R, V, pad=0, offset=0, seed=0, spread=3.0, rounded=False):
    """[R, V] view of a buffer with `pad` columns behind each row and `offset` floats in front, all of them NaN."""
    g = torch.Generator().manual_seed(seed * 7919 + R * 31 + V)
    stride = V + pad
    flat = torch.full((offset + R * stride,), math.nan)
    x = flat[offset:].view(R, stride)[:, :V]
    x.copy_(torch.randn(R, V, generator=g) * spread)
    if rounded:
        x.copy_(x.bfloat16().float())
    flat = flat.to("cuda")
    return flat[offset:].view(R, stride)[:, :V], stride


def special_rows(x):
    """Puts rows that a softmax can go wrong at into x [R >= 8, V] and returns what they are."""
    V = x.shape[1]
    x[0] = NEG                                    # nothing is left
    x[1] = LOWEST                                 # the lowest float everywhere: a uniform row
    x[2, : V - 1] = LOWEST                        # ... as a mask
    x[3, 1:] = NEG                                # one token is left
    x[4] = 7.25                                   # all equal
    x[5] = torch.arange(V, device=x.device) * (20.0 / V)          # ascending: values above any early bound
    x[6] = 1e30                                   # far from zero
    x[6, V // 2] = 1.00001e30
    x[7, : V // 2] = NEG


def top_of(x, k):
    return torch.sort(x.detach().cpu(), dim=1, descending=True, stable=True).indices[:, :k]


def run_logprobs(ctx, x, stride, tokens, k, T, entropy=True, stats=True):
    R, V = x.shape
    out = {"logp": torch.full((R,), 9.0, device="cuda"), "H": torch.full((R,), 9.0, device="cuda") if entropy else None,
           "ids": torch.full((R, k), -7, dtype=torch.int32, device="cuda") if k else None, "top": torch.full((R, k), 9.0, device="cuda") if k else None,
           "stats": torch.full((R, 2), 9.0, device="cuda") if stats else None}
    ctx.token_logprobs(x, tokens, out["logp"], out["H"], out["ids"], out["top"], out["stats"], R, V, k, T, stride)
    torch.cuda.synchronize()
    return out


def check_logprobs(ctx, x, stride, k, T, tokens):
    R, V = x.shape
    got = run_logprobs(ctx, x, stride, tokens.to("cuda", torch.int32), k, T)
    want = Row64(x, T)
    rows = torch.arange(R)
    tok = tokens.long()
    valid = (tok >= 0) & (tok < V)
    at = tok.clamp(0, V - 1)
    near(got["logp"], torch.where(valid, want.logp[rows, at], torch.zeros(R, dtype=torch.float64)), want.tol_logp[rows, at], "log probabilities")
    near(got["H"], want.H[:, 0], want.tol_H[:, 0], "entropy")
    if k:
        ids = top_of(x, k)
        assert torch.equal(got["ids"].cpu().long(), ids)
        near(got["top"], want.logp.gather(1, ids), want.tol_logp.gather(1, ids), "top log probabilities")
    live = ~want.dead[:, 0]
    assert torch.equal(got["stats"][:, 0].cpu()[live], x.detach().cpu().amax(dim=1)[live])
    near(got["stats"][:, 1], torch.where(live, want.s[:, 0], torch.zeros(R, dtype=torch.float64)), want.tol_s[:, 0] * want.s[:, 0].nan_to_num(), "sums")
    return got, want


@pytest.mark.parametrize("R,V,pad,offset,k,T", [
    (1, 1, 0, 0, 1, 1.0),
    (3, 2, 1, 1, 2, 0.5),
    (9, 5, 0, 0, 5, 1.0),
    (17, 127, 1, 0, 127, 2.0),
    (5, 128, 0, 3, 128, 1.0),
    (40, 1000, 0, 0, 20, 0.7),
    (33, 1001, 0, 2, 7, 1.0),             # every row starts at another alignment
    (8, 2049, 3, 1, 128, 1.3),
    (700, 3001, 0, 0, 3, 1.0),            # more rows than SMs
    (2500, 515, 1, 0, 17, 1.0),           # more rows than CTAs
    (1, 32000, 0, 0, 20, 1.0),            # a row over several CTAs
    (1, 32003, 5, 1, 128, 1.0),
    (40, 32000, 64, 0, 64, 0.3),
    (2, 150001, 0, 0, 50, 1.0),
    (300, 32000, 0, 0, 1, 1.0),
    (500, 500, 0, 0, 0, 1.0),             # a warp a row
    (3001, 513, 1, 2, 0, 0.5),
    (1200, 1025, 0, 1, 0, 1.0),
    (600, 2048, 3, 3, 0, 2.0),
    (700, 3, 0, 0, 0, 1.0),
    (500, 2049, 1, 1, 0, 1.0),            # two warps
    (450, 4096, 0, 0, 0, 0.7),
    (450, 8189, 1, 3, 0, 1.0),            # four
    (190, 60003, 1, 0, 20, 1.0),          # two CTAs a row, three on an SM
    (110, 128256, 0, 0, 128, 1.0),
])
def test_token_logprobs(ctx, R, V, pad, offset, k, T):
    x, stride = make_logits(R, V, pad, offset, seed=1)
    g = torch.Generator().manual_seed(R + V)
    tokens = torch.randint(0, V, (R,), generator=g)
    if R > 2:
        tokens[1], tokens[2] = -1, V
    check_logprobs(ctx, x, stride, k, T, tokens)


@pytest.mark.parametrize("R,V,k,T", [(12, 600, 128, 1.0), (9, 5000, 20, 0.5), (8, 32001, 64, 1.0), (8, 32000, 128, 2.0), (8, 70000, 5, 1.0), (200, 9000, 33, 1.0), (150, 4097, 50, 1.0),
                                     (20, 16384, 128, 0.7), (21, 16385, 128, 1.0), (900, 9000, 20, 1.0), (500, 3001, 64, 1.0)])
@pytest.mark.parametrize("rounded", [False, True])
def test_token_logprobs_of_masked_and_extreme_rows(ctx, R, V, k, T, rounded):
    x, stride = make_logits(R, V, 1, 1, seed=2, rounded=rounded)
    special_rows(x)
    tokens = torch.full((R,), 0)
    tokens[5], tokens[6], tokens[7] = V - 1, V // 2, 1
    check_logprobs(ctx, x, stride, k, T, tokens)


@pytest.mark.parametrize("R,V,k,rounded", [(160, 90001, 20, False), (155, 50000, 128, False), (160, 70003, 64, True), (150, 150000, 1, False), (300, 24001, 100, True)])
def test_top_tokens_of_rows_of_many_steps(ctx, R, V, k, rounded):
    """More rows than clusters take, each long enough for several bounds on the way."""
    x, stride = make_logits(R, V, 1, 0, seed=6, rounded=rounded)
    special_rows(x)
    x[8] = torch.arange(V, 0, -1, device=x.device) * (20.0 / V)      # descending: the first bound is the last
    x[9, V // 2:] += 30.0                                           # everything that counts behind the middle
    x[10].copy_(torch.where(torch.arange(V, device=x.device) % 4096 < 1024, x[10] + 9.0, x[10]))
    tokens = torch.full((R,), 0)
    tokens[5], tokens[6], tokens[7] = V - 1, V // 2, 1
    check_logprobs(ctx, x, stride, k, 1.0, tokens)


@pytest.mark.parametrize("R,V", [(460, 5), (450, 511), (500, 1500), (447, 3999), (447, 8001)])
def test_short_rows_that_go_wrong(ctx, R, V):
    x, stride = make_logits(R, V, 1, 1, seed=7)
    special_rows(x)
    tokens = torch.full((R,), 0)
    tokens[5], tokens[6], tokens[7], tokens[8], tokens[9] = V - 1, V // 2, 1, -1, V
    check_logprobs(ctx, x, stride, 0, 1.0, tokens)
    x[10, V // 3] = math.nan
    x[11, V - 1] = math.inf
    x[12] = math.nan
    got = run_logprobs(ctx, x, stride, tokens.to("cuda", torch.int32), 0, 1.0)
    bad = torch.zeros(R, dtype=torch.bool)
    bad[10:13] = True
    for n in ("logp", "H"):
        assert torch.equal(torch.isnan(got[n]).cpu(), bad), n


@pytest.mark.parametrize("R,V,k,pad,offset", [(460, 5, 5, 0, 0), (447, 100, 100, 1, 1), (450, 511, 20, 1, 0), (500, 512, 128, 0, 0), (450, 700, 64, 3, 2), (890, 1024, 1, 0, 0),
                                              (900, 1025, 127, 0, 3), (1000, 2047, 2, 1, 1), (900, 2048, 128, 0, 0), (888, 2045, 20, 0, 1),
                                              (30, 900, 50, 0, 1), (21, 1023, 128, 1, 0)])
@pytest.mark.parametrize("rounded", [False, True])
def test_top_tokens_of_short_rows(ctx, R, V, k, pad, offset, rounded):
    x, stride = make_logits(R, V, pad, offset, seed=8, rounded=rounded)
    special_rows(x)
    g = torch.Generator().manual_seed(V + k)
    x[8] = (torch.arange(V) % 3 == 0).float().to(x.device)               # two values: more equal ones than are collected
    x[9] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0).to(x.device)  # zeros of both signs are equal
    x[10] = torch.randint(0, 7, (V,), generator=g).float().to(x.device)
    x[11] = torch.where(torch.rand(V, generator=g) < 0.97, NEG, 1.0).to(x.device)
    x[12] = torch.where(torch.rand(V, generator=g) < 0.5, -1e-45, 1e-45).to(x.device)
    x[13] = torch.arange(V, 0, -1, device=x.device) * 1e-3
    x[14, ::32] += 40.0
    x[15, : V // 2] += 40.0
    x[16, 0], x[17, V - 1] = 99.0, 99.0
    tokens = torch.randint(0, V, (R,), generator=g)
    check_logprobs(ctx, x, stride, k, 1.0, tokens)
    x[18, V // 3], x[19, V // 2], x[20] = math.nan, math.inf, math.nan
    got = run_logprobs(ctx, x, stride, tokens.to("cuda", torch.int32), k, 1.0)
    assert bool((got["ids"][18:21] == -1).all()) and bool(torch.isnan(got["top"][18:21]).all())
    ids = top_of(x, k)
    ok = torch.ones(R, dtype=torch.bool)
    ok[18:21] = False
    assert torch.equal(got["ids"].cpu().long()[ok], ids[ok])


def test_top_tokens_where_one_thread_has_all_large_values(ctx):
    """More values above a bound from the threads' largest than are collected at once."""
    V, k = 32000, 128
    for period in (2048, 512, 4096, 16384):
        x = torch.randn(4, V)
        at = torch.arange(V)
        for lanes in range(4):
            hot = (at % period) < 4 * (lanes + 1) * 7
            x[lanes][hot] = 50.0 + at[hot] * 1e-3
        x[3] = torch.arange(V) * 1e-3 - 5.0
        x = x.to("cuda")
        check_logprobs(ctx, x, V, k, 1.0, torch.zeros(4, dtype=torch.long))


def test_top_tokens_of_many_equal_values(ctx):
    g = torch.Generator().manual_seed(5)
    for V, levels in ((32000, 2), (32000, 5), (5000, 3), (100, 1), (32000, 300)):
        x = torch.randint(0, levels, (40, V), generator=g).float().to("cuda")
        x[3] = torch.where(x[3] > 0, 0.0, -0.0)                     # zeros of both signs are equal
        check_logprobs(ctx, x, V, min(V, 100), 1.0, torch.zeros(40, dtype=torch.long))


@pytest.mark.parametrize("R,V", [(6, 300), (6, 32000), (6, 5000), (6, 16000)])
def test_rows_with_nan_or_infinity(ctx, R, V):
    x, stride = make_logits(R, V, seed=3)
    x[1, V // 3] = math.nan
    x[2, V // 3] = math.inf
    x[3] = math.nan
    tokens = torch.tensor([0, 0, V // 3, 0, 5, -1], dtype=torch.int32)
    x[5, 0] = math.nan                                              # a padded row: its log probability is 0 all the same
    got = run_logprobs(ctx, x, stride, tokens.to("cuda"), 9, 1.0)
    bad = torch.tensor([False, True, True, True, False, False])
    assert torch.equal(torch.isnan(got["logp"]).cpu(), bad) and float(got["logp"][5]) == 0.0
    bad[5] = True
    assert torch.equal(torch.isnan(got["H"]).cpu(), bad)
    assert torch.equal(torch.isnan(got["top"]).all(dim=1).cpu(), bad) and torch.equal(torch.isnan(got["top"]).any(dim=1).cpu(), bad)
    assert bool((got["ids"].cpu()[bad] == -1).all()) and torch.equal(got["ids"].cpu()[~bad].long(), top_of(x, 9)[~bad])


def test_outputs_that_are_not_asked_for(ctx):
    R, V = 70, 999
    x, stride = make_logits(R, V, seed=4)
    tokens = torch.randint(0, V, (R,), dtype=torch.int32).to("cuda")
    full = run_logprobs(ctx, x, stride, tokens, 11, 1.5)
    bits = lambda a, b: torch.equal(a.view(torch.int32), b.view(torch.int32))
    logp, H, ids, top, stats = (torch.empty_like(full[n]) for n in ("logp", "H", "ids", "top", "stats"))
    ctx.token_logprobs(x, tokens, logp, None, None, None, None, R, V, 0, 1.5)
    ctx.token_logprobs(x, None, None, H, None, None, None, R, V, 0, 1.5)
    ctx.token_logprobs(x, None, None, None, ids, None, None, R, V, 11, 1.5)
    ctx.token_logprobs(x, None, None, None, None, top, None, R, V, 11, 1.5)
    ctx.token_logprobs(x, None, None, None, None, None, stats, R, V, 0, 1.5)
    torch.cuda.synchronize()
    for a, n in ((logp, "logp"), (H, "H"), (ids, "ids"), (top, "top"), (stats, "stats")):
        assert bits(a, full[n]), n


# ---- gradient of log probabilities and entropies ------------------------------------------------------------------------

def policy_grad(want, tokens, dlogp, dent):
    """Formula and tolerance: dx = (up (1[token] - p) - h p (ln p + H)) / T."""
    R, V = want.x.shape
    tok = tokens.long()
    valid = (tok >= 0) & (tok < V)
    up = torch.where(valid, dlogp.double(), torch.zeros(R, dtype=torch.float64)) if dlogp is not None else torch.zeros(R, dtype=torch.float64)
    h = dent.double() if dent is not None else torch.zeros(R, dtype=torch.float64)
    hot = torch.zeros(R, V, dtype=torch.float64)
    hot[torch.arange(R)[valid], tok[valid]] = 1.0
    logp = torch.where(want.p > 0, want.logp, torch.zeros_like(want.p))
    up, h = up[:, None], h[:, None]
    core = -up * want.p - h * want.p * (logp + want.H)
    live = ~want.dead
    grad = torch.where(live, (core + hot * up) / want.T, torch.zeros_like(core))
    size = up.abs() + h.abs() * (logp.abs() + want.H)
    # p's own error; that of ln p + H, in which ln s cancels between terms of its size; a few roundings of the terms
    tol = (want.tol_p * size + want.p * h.abs() * (want.tol_logp + want.tol_H + 8 * U * torch.log(want.s).abs().nan_to_num(posinf=0.0))
           + 16 * U * want.p * size + 8 * U * hot * up.abs()) / want.T
    return grad, tol


@pytest.mark.parametrize("R,V,pad,offset,T", [(1, 1, 0, 0, 1.0), (9, 130, 1, 1, 0.5), (70, 1001, 0, 2, 1.0), (8, 32000, 0, 0, 2.0), (1, 50003, 2, 1, 1.0),
                                             (700, 2048, 0, 0, 1.0), (2600, 515, 0, 0, 0.7), (460, 4001, 1, 1, 1.0), (450, 8192, 0, 0, 2.0)])
@pytest.mark.parametrize("which", ["both", "logp", "entropy"])
@pytest.mark.parametrize("in_place", [False, True])
def test_token_logprobs_backward(ctx, R, V, pad, offset, T, which, in_place):
    x, stride = make_logits(R, V, pad, offset, seed=6)
    if R >= 8:
        special_rows(x)
    g = torch.Generator().manual_seed(R * 3 + V)
    tokens = torch.randint(0, V, (R,), generator=g)
    if R > 2:
        tokens[R // 2] = -1
        tokens[R - 1] = V
    dlogp = torch.randn(R, generator=g) if which != "entropy" else None
    dent = torch.randn(R, generator=g) if which != "logp" else None
    fwd = run_logprobs(ctx, x, stride, tokens.int().to("cuda"), 0, T)
    want, tol = policy_grad(Row64(x, T), tokens, dlogp, dent)
    if in_place:
        grad, before = x, None
    else:
        before = torch.full((offset + R * stride,), 5.0, device="cuda")
        grad = before[offset:].view(R, stride)[:, :V]
    dev = lambda a: None if a is None else a.to("cuda")
    ctx.token_logprobs_backward(x, tokens.int().to("cuda") if dlogp is not None else None, fwd["stats"], fwd["H"] if dent is not None else None, dev(dlogp),
                                dev(dent), grad, R, V, T, stride)
    torch.cuda.synchronize()
    near(grad, want, tol)
    if before is not None and (pad or offset):                      # nothing beside the rows is written
        rest = before.clone()
        rest[offset:].view(R, stride)[:, :V] = 5.0
        assert bool((rest == 5.0).all())


def test_gradient_is_exactly_zero_where_nothing_is_asked(ctx):
    R, V = 6, 777
    x, stride = make_logits(R, V, seed=7)
    x[0] = math.nan
    x[1] = math.inf
    x[2] = NEG
    tokens = torch.tensor([-1, V + 5, 3, 0, 4, 4], dtype=torch.int32, device="cuda")
    dlogp = torch.tensor([1.0, 1.0, 1.0, 0.0, 2.0, 2.0], device="cuda")
    fwd = run_logprobs(ctx, x, stride, tokens, 0, 1.0)
    grad = torch.full_like(x, 3.0)
    ctx.token_logprobs_backward(x, tokens, fwd["stats"], None, dlogp, None, grad, R, V)
    torch.cuda.synchronize()
    assert bool((grad[:4] == 0.0).all()) and bool((grad[4:] != 0.0).any())


@pytest.mark.parametrize("R,V", [(460, 777), (450, 3001), (20, 20001)])
def test_gradient_is_exactly_zero_where_nothing_is_asked_of_other_rows(ctx, R, V):
    """Warps a row, and tiles of a row."""
    x, stride = make_logits(R, V, 1, 0, seed=46)
    x[0], x[1], x[2], x[3, V // 2] = math.nan, math.inf, NEG, math.nan
    tokens = torch.full((R,), 4, dtype=torch.int32, device="cuda")
    tokens[0], tokens[1] = -1, V + 5
    dlogp, dent = torch.ones(R, device="cuda"), torch.zeros(R, device="cuda")
    dlogp[3] = 0.0
    fwd = run_logprobs(ctx, x, stride, tokens, 0, 1.0)
    for second in (None, dent):
        grad = torch.full((R * stride,), 3.0, device="cuda").view(R, stride)[:, :V]
        ctx.token_logprobs_backward(x, tokens, fwd["stats"], fwd["H"] if second is not None else None, dlogp, second, grad, R, V, 1.0, stride)
        torch.cuda.synchronize()
        assert bool((grad[:4] == 0.0).all()) and bool((grad[4:] != 0.0).any(dim=1).all())


@pytest.mark.parametrize("which", ["both", "logp"])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pad", [0, 1])
def test_token_gradients_of_more_rows_than_ctas(ctx, which, in_place, pad):
    """Three rows a CTA of the gradient's kernel."""
    V, per = 4101, 16 * ctx.sm_count
    R = 2 * per + 200
    x, stride = make_logits(R, V, pad, 0, seed=47)
    special_rows(x)
    special_rows(x[per:])
    special_rows(x[2 * per + 100:])
    g = torch.Generator().manual_seed(48)
    tokens = torch.randint(0, V, (R,), generator=g)
    tokens[20:40], tokens[per + 30:per + 50], tokens[2 * per + 40:2 * per + 60] = -1, V, -1
    dlogp, dent = torch.randn(R, generator=g), torch.randn(R, generator=g) if which == "both" else None
    rows = torch.cat([torch.arange(200), torch.arange(per, per + 200), torch.arange(2 * per, R)])
    want, tol = policy_grad(Row64(x[rows.to(x.device)], 1.0), tokens[rows], dlogp[rows], dent[rows] if dent is not None else None)
    tokens = tokens.int().to("cuda")
    fwd = run_logprobs(ctx, x, stride, tokens, 0, 1.0)
    grad = x if in_place else torch.empty(R * stride, device="cuda").view(R, stride)[:, :V]
    ctx.token_logprobs_backward(x, tokens, fwd["stats"], fwd["H"] if dent is not None else None, dlogp.to("cuda"), dent.to("cuda") if dent is not None else None, grad, R,
                                V, 1.0, stride)
    torch.cuda.synchronize()
    near(grad[rows.to(grad.device)], want, tol)


def test_gradients_against_differences(ctx):
    """Directional derivatives of the definitions in float64: differences of step h are off by h^2 / 6 of a third derivative (of order
    the value) and by 2^-52 / h: 1e-10 at h = 1e-5; the gradient itself by what policy_grad allows, below 1e-5 of its size here."""
    R, V, T, h = 5, 400, 0.8, 1e-5
    x, stride = make_logits(R, V, seed=8)
    g = torch.Generator().manual_seed(9)
    tokens = torch.randint(0, V, (R,), generator=g)
    dlogp, dent = torch.randn(R, generator=g), torch.randn(R, generator=g)
    ids = torch.stack([torch.randperm(V, generator=g)[:12] for _ in range(R)]).int()
    teacher = torch.randn(R, 12, generator=g) * 2
    fwd = run_logprobs(ctx, x, stride, tokens.int().to("cuda"), 0, T)
    grad, grad2 = torch.empty_like(x), torch.empty_like(x)
    ctx.token_logprobs_backward(x, tokens.int().to("cuda"), fwd["stats"], fwd["H"], dlogp.to("cuda"), dent.to("cuda"), grad, R, V, T)
    part, out = torch.empty(R, device="cuda"), torch.empty(1, device="cuda")
    ctx.distillation_loss(x, ids.to("cuda"), teacher.to("cuda"), part, out, None, torch.tensor([2.5], device="cuda"), grad2, R, V, 12, T)
    torch.cuda.synchronize()
    t = torch.softmax(teacher.double() / float(np.float32(T)), dim=1)

    def policy(z):
        lp = torch.log_softmax(z / float(np.float32(T)), dim=1)
        return (lp[torch.arange(R), tokens] * dlogp.double()).sum() - (dent.double() * (lp.exp() * lp).sum(dim=1)).sum()

    def distill(z):
        lp = torch.log_softmax(z / float(np.float32(T)), dim=1)
        return 2.5 * (t * (t.log() - lp.gather(1, ids.long()))).sum(dim=1).mean()

    z = x.cpu().double()
    for seed in range(6):
        v = torch.randn(R, V, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
        for f, gr in ((policy, grad), (distill, grad2)):
            diff = float((f(z + h * v) - f(z - h * v)) / (2 * h))
            got = float((gr.cpu().double() * v).sum())
            size = float(gr.cpu().double().norm() * v.norm())
            assert abs(got - diff) <= 1e-5 * size, (f.__name__, got, diff)


# ---- distillation ----------------------------------------------------------------------------------------------------------

def make_teacher(R, V, K, seed):
    g = torch.Generator().manual_seed(seed + R + V + K)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] if V < 100000 else torch.randint(0, V, (K,), generator=g) for _ in range(R)]).int()
    return ids, torch.randn(R, K, generator=g) * 2.5


def distill_ref(x, ids, a, T, up=1.0):
    """Losses, gradient of up times their mean, and tolerances for both."""
    want = Row64(x, T)
    R, V = want.x.shape
    ids, T64 = ids.long(), want.T
    valid = (ids >= 0) & (ids < V)
    at = ids.clamp(0, V - 1)
    z = torch.where(valid, a.double(), torch.full_like(a.double(), NEG)) / T64
    top = z.amax(dim=1, keepdim=True)
    empty = top == NEG
    d = torch.where(empty, torch.full_like(z, NEG), z - top)
    w = torch.exp(d)
    S = w.sum(dim=1, keepdim=True)
    t = torch.where(empty, torch.zeros_like(w), w / S)
    log_t = torch.where(t > 0, d - torch.log(S), torch.zeros_like(d))
    logq = want.logp.gather(1, at)
    ratio = torch.where(t > 0, log_t - logq, torch.zeros_like(t))
    losses = torch.where(t > 0, t * ratio, torch.zeros_like(t)).sum(dim=1)
    K = ids.shape[1]
    dd = d.nan_to_num(neginf=0.0).abs()
    mean_dd = (t * dd).sum(dim=1, keepdim=True)
    tol_S = U * (4 * (mean_dd + 1) + 16)                             # four additions a lane, five across
    tol_t = t * (4 * U * (dd + 3) + tol_S)
    tol_lt = 3 * U * dd + tol_S + 5 * U * torch.log(S).abs().nan_to_num()
    fr = ratio.abs().nan_to_num(posinf=0.0)
    tol_loss = (tol_t * fr + t * (tol_lt + want.tol_logp.gather(1, at) + 2 * U * fr) + 12 * U * t * fr).sum(dim=1)
    named = torch.zeros(R, V, dtype=torch.float64).scatter_add_(1, at, t)
    tol_named = torch.zeros(R, V, dtype=torch.float64).scatter_add_(1, at, tol_t + K * U * t)
    live = ~empty & ~want.dead
    f = up / (T64 * R)
    grad = torch.where(live, (want.p - named) * f, torch.zeros_like(want.p))
    tol_grad = (want.tol_p + tol_named + 8 * U * (want.p + named)) * abs(f)
    return losses, tol_loss, grad, tol_grad


def run_distill(ctx, x, stride, ids, a, T, up, form):
    R, V = x.shape
    K = ids.shape[1]
    ids, a = ids.to("cuda"), a.to("cuda")
    part, out, stats, go = torch.full((R,), 9.0, device="cuda"), torch.full((1,), 9.0, device="cuda"), torch.empty(R, 2, device="cuda"), torch.tensor([up], device="cuda")
    store = torch.full((R * stride,), 5.0, device="cuda")
    grad = store.view(R, stride)[:, :V]
    if form == "in place":
        grad = x
    if form == "split":
        ctx.distillation_loss(x, ids, a, part, out, stats, None, None, R, V, K, T, stride)
        ctx.distillation_loss_backward(x, ids, a, stats, go, grad, R, V, K, T, stride)
    elif form == "split in place":
        grad = x
        ctx.distillation_loss(x, ids, a, part, out, stats, None, None, R, V, K, T, stride)
        ctx.distillation_loss_backward(x, ids, a, stats, go, grad, R, V, K, T, stride)
    else:
        ctx.distillation_loss(x, ids, a, part, out, stats, go, grad, R, V, K, T, stride)
    torch.cuda.synchronize()
    if not form.endswith("in place"):
        rest = store.clone()
        rest.view(R, stride)[:, :V] = 5.0
        assert bool((rest == 5.0).all())                            # nothing beside the rows is written
    return part, out, grad


FORMS = ["one call", "split", "in place", "split in place"]


@pytest.mark.parametrize("R,V,K,pad,offset,T", [(1, 1, 1, 0, 0, 1.0), (3, 5, 5, 1, 1, 2.0), (20, 128, 128, 0, 0, 1.0), (33, 1001, 7, 0, 2, 0.5), (600, 2500, 64, 0, 0, 2.0),
                                              (2500, 300, 3, 1, 0, 1.0), (1, 32000, 20, 0, 0, 1.0), (12, 33001, 128, 3, 1, 1.5), (40, 32000, 64, 0, 0, 4.0),
                                              (900, 1000, 128, 0, 1, 1.0), (455, 2047, 33, 2, 3, 0.5), (1000, 4001, 64, 1, 0, 2.0), (600, 8190, 20, 0, 0, 1.0),
                                              (450, 9001, 64, 1, 0, 1.0), (446, 16384, 8, 0, 0, 1.0),
                                              (300, 24581, 5, 0, 0, 1.0), (450, 32000, 64, 0, 0, 2.0), (310, 33001, 33, 3, 1, 0.7), (297, 45056, 128, 4, 3, 1.0)])
@pytest.mark.parametrize("form", FORMS)
def test_distillation(ctx, R, V, K, pad, offset, T, form):
    x, stride = make_logits(R, V, pad, offset, seed=10)
    ids, a = make_teacher(R, V, K, 1)
    if R > 2:
        ids[1, K // 2:] = -1                                        # a shorter list
        ids[2] = V                                                  # none at all
    losses, tol_l, grad, tol_g = distill_ref(x, ids, a, T, 1.75)
    part, out, got = run_distill(ctx, x, stride, ids, a, T, 1.75, form)
    near(part, losses, tol_l, "losses")
    # the mean: a sum of R terms in 1024 lanes and a tree
    near(out, losses.mean().reshape(1), float(tol_l.mean()) + U * (R / 1024 + 20) * float(losses.abs().mean()), "mean")
    near(got, grad, tol_g, "gradient")


# rows in the ring of chunks: three whole ones, in two to seven chunks, as long as there is room for, and in parts over two, four and eight CTAs;
# every row at another alignment where the pad is odd
@pytest.mark.parametrize("R,V,K,pad,offset,T", [(700, 11264, 20, 0, 0, 1.0), (301, 13001, 128, 1, 0, 2.0), (500, 17749, 9, 0, 2, 1.0), (450, 20003, 64, 2, 1, 0.8),
                                              (310, 22001, 33, 0, 0, 1.0), (300, 28004, 5, 1, 3, 1.0), (299, 36000, 64, 0, 0, 1.5), (298, 40001, 7, 0, 1, 1.0),
                                              (297, 49152, 16, 0, 0, 1.0), (310, 49157, 64, 0, 1, 1.0), (170, 70001, 100, 1, 0, 2.0), (160, 128256, 64, 0, 0, 1.0),
                                              (76, 150003, 11, 2, 3, 1.0), (45, 262144, 8, 0, 0, 1.0), (200, 24001, 20, 3, 0, 1.0), (110, 50003, 64, 0, 0, 1.0),
                                              (100, 24001, 20, 3, 0, 1.0)])
@pytest.mark.parametrize("form", ["one call", "in place"])
def test_distillation_of_long_rows(ctx, R, V, K, pad, offset, T, form):
    x, stride = make_logits(R, V, pad, offset, seed=17)
    ids, a = make_teacher(R, V, K, 6)
    ids[1, K // 2:] = -1
    ids[2] = V
    ids[3, 1:] = ids[3, 0]                                          # one token K times
    ids[4, :4] = torch.tensor([0, V - 1, 1, V - 2])                 # at the ends, outside whole quads
    x[5] = NEG
    x[6, V // 4:] = NEG                                             # CTAs of which nothing is left
    x[7] = LOWEST
    losses, tol_l, grad, tol_g = distill_ref(x, ids, a, T, 0.5)
    part, out, got = run_distill(ctx, x, stride, ids, a, T, 0.5, form)
    near(part, losses, tol_l, "losses")
    near(got, grad, tol_g, "gradient")


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("R,V", [(16, 500), (16, 40000), (320, 26000), (460, 500), (460, 1500), (460, 3001), (450, 7777)])
def test_distillation_lists_and_rows_that_go_wrong(ctx, R, V, form):
    K = 10
    x, stride = make_logits(R, V, 1, 0, seed=11)
    special_rows(x)
    ids, a = make_teacher(R, V, K, 2)
    ids[3, 0], ids[3, 1:] = 0, -1                                   # the one token that is left
    ids[7] = torch.arange(K)                                        # tokens that are masked: an infinite loss
    ids[8] = 5                                                      # the same token ten times
    ids[9, 4], ids[9, 9] = ids[9, 0], ids[9, 0]
    a[10, 1:] = NEG                                                 # entries without probability
    a[11] = NEG                                                     # no entries
    a[12] = LOWEST
    a[13, 0] = 1e4
    ids[14] = torch.arange(K) + V // 2
    x[15, ids[15, 3].long()] = NEG
    a[15, 3] = NEG                                                  # no probability either side: nothing to the loss
    losses, tol_l, grad, tol_g = distill_ref(x, ids, a, 1.0)
    part, out, got = run_distill(ctx, x, stride, ids, a, 1.0, 1.0, form)
    near(part, losses, tol_l, "losses")
    near(got, grad, tol_g, "gradient")
    assert float(part[0]) == math.inf and float(part[11]) == 0.0


# (rows a wave, rows, columns, entries, pad, offset): rings of one CTA a row and of two, eight rows and more for each; the same rows with gradients that
# start elsewhere between 16-byte boundaries, which go by a second time, three of them for each CTA
@pytest.mark.parametrize("wave,R,V,K,pad,offset", [(148, 1300, 17000, 20, 0, 0), (148, 1250, 17003, 128, 1, 0), (74, 700, 50003, 7, 0, 0), (592, 1400, 17001, 20, 0, 1), (592, 1300, 17000, 64, 0, 2)])
@pytest.mark.parametrize("form", ["one call", "in place"])
def test_distillation_of_many_long_rows(ctx, wave, R, V, K, pad, offset, form):
    x, stride = make_logits(R, V, pad, offset, seed=49)
    ids, a = make_teacher(R, V, K, 13)
    for first in range(0, R - wave, wave):                          # other rows than their neighbours' in every wave
        turn = first // wave
        special = torch.arange(first + 8 * turn, min(R, first + 8 * turn + 7))
        if len(special) < 7:
            continue
        r = [int(i) for i in special]
        ids[r[0]] = -1
        ids[r[1], 1:] = -1
        ids[r[2], 1:] = ids[r[2], 0]
        ids[r[3], 0], ids[r[3], K - 1] = V - 1, 0
        x[r[4]] = NEG
        x[r[5], V // 3:] = NEG
        a[r[6], 1:] = NEG
    rows = torch.cat([torch.arange(min(100, wave)) + first for first in range(0, R, wave)] + [torch.arange(R - 20, R)])
    rows = rows[rows < R].unique()
    losses, tol_l, grad, tol_g = distill_ref(x[rows.to(x.device)], ids[rows], a[rows], 1.5, 0.75 * len(rows) / R)
    part, out, got = run_distill(ctx, x, stride, ids, a, 1.5, 0.75, form)
    near(part[rows.to(part.device)], losses, tol_l, "losses")
    near(got[rows.to(got.device)], grad, tol_g, "gradient")


@pytest.mark.parametrize("form", ["split", "split in place"])
def test_lists_of_a_ctas_next_rows(ctx, form):
    """Three rows a CTA of the gradient's kernel, whose lists come to the same place: behind rows of which nothing is asked, behind rows with a list of
    their own, and none behind a list."""
    V, K, per = 8300, 20, 16 * ctx.sm_count
    R = 2 * per + 300
    x, stride = make_logits(R, V, 0, 0, seed=41)
    ids, a = make_teacher(R, V, K, 9)
    ids[:400] = -1
    ids[300:400, 7] = V
    x[600:700] = NEG
    ids[per + 200:per + 400] = -1
    ids[per + 700:per + 800, 1:] = -1
    ids[2 * per + 100:2 * per + 150] = -1
    rows = torch.cat([torch.arange(900), torch.arange(per, per + 900), torch.arange(2 * per, R)])
    losses, tol_l, grad, tol_g = distill_ref(x[rows.to(x.device)], ids[rows], a[rows], 2.0, 1.5 * len(rows) / R)
    part, out, got = run_distill(ctx, x, stride, ids, a, 2.0, 1.5, form)
    near(part[rows], losses, tol_l, "losses")
    near(got[rows], grad, tol_g, "gradient")


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("K", [33, 64, 128])
def test_distillation_lists_longer_than_a_warp(ctx, K, form):
    """Entries without a token and tokens named twice, in every group of 32 entries and across them."""
    R, V = 12, 3000
    x, stride = make_logits(R, V, 1, 0, seed=16)
    ids, a = make_teacher(R, V, K, 5)
    ids[0] = -1
    ids[1, 0] = -1
    ids[2, ::2] = -1
    ids[3, 31], ids[3, 32] = -1, -32                                # any number outside the vocabulary
    ids[4, K - 1] = ids[4, 0]
    ids[5, 32] = ids[5, 1]
    ids[6] = torch.arange(K) % 7
    ids[7, 1] = ids[7, 0]
    ids[8, K - 1] = ids[8, K - 2]
    ids[9] = V + torch.arange(K)
    ids[9, K - 1] = 3
    ids[10, :32] = -1
    losses, tol_l, grad, tol_g = distill_ref(x, ids, a, 1.25)
    part, out, got = run_distill(ctx, x, stride, ids, a, 1.25, 1.0, form)
    near(part, losses, tol_l, "losses")
    near(got, grad, tol_g, "gradient")


@pytest.mark.parametrize("form", ["one call", "split"])
@pytest.mark.parametrize("R,V", [(7, 3000), (300, 25001), (160, 60001), (460, 900), (460, 2500), (450, 8000)])
def test_distillation_of_rows_with_nan(ctx, R, V, form):
    K = 5
    x, stride = make_logits(R, V, seed=12)
    ids, a = make_teacher(R, V, K, 3)
    x[0, 7] = math.nan
    x[1, 7] = math.inf
    x[2] = math.nan
    ids[2] = -1                                                     # a padded row may hold anything
    a[3, 2] = math.nan
    a[4, 2] = math.inf
    part, out, got = run_distill(ctx, x, stride, ids, a, 1.0, 1.0, form)
    bad = torch.tensor([True, True, False, True, True] + [False] * (R - 5))
    assert torch.equal(torch.isnan(part).cpu(), bad) and torch.equal(torch.isnan(got).any(dim=1).cpu(), bad)
    assert torch.equal(torch.isnan(got).all(dim=1).cpu(), bad)
    assert float(part[2]) == 0.0 and bool((got[2] == 0.0).all())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("R,V,pad", [(7, 3000, 0), (300, 25001, 1), (160, 60001, 0), (460, 900, 0), (460, 2500, 1), (450, 8000, 0), (450, 12001, 0), (460, 18000, 0)])
def test_gradient_is_exactly_zero_where_the_losss_gradient_is(ctx, R, V, pad, form):
    x, stride = make_logits(R, V, pad, 0, seed=43)
    ids, a = make_teacher(R, V, 5, 10)
    x[0, 7], x[1, V - 1], x[2], x[3] = math.nan, math.inf, math.nan, NEG
    a[4, 2], a[5, 2] = math.nan, math.inf
    part, out, got = run_distill(ctx, x, stride, ids, a, 1.0, 0.0, form)
    assert bool((got == 0.0).all())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("R,V,pad", [(8, 3000, 0), (512, 900, 0), (512, 17000, 0), (512, 6001, 1), (256, 30000, 0)])
def test_gradients_of_listed_tokens_beside_probabilities_that_underflow(ctx, R, V, pad, form):
    up = 2.0 ** -147
    x, stride = make_logits(R, V, pad, 0, seed=42)
    x.zero_()
    ids = torch.arange(R, dtype=torch.int32)[:, None] * 3 % V
    part, out, got = run_distill(ctx, x, stride, ids, torch.zeros(R, 1), 1.0, R * up, form)
    want = torch.zeros(R, V).scatter_(1, ids.long(), -up)
    assert torch.equal(got.cpu(), want)


def test_a_teachers_list_and_its_log_probabilities_teach_the_same(ctx):
    """What token_logprobs keeps of a teacher, put into distillation_loss: the same loss as from its logits, and 0 for a student that
    gives these tokens alone its probability."""
    R, V, K, T = 50, 4000, 16, 2.0
    x, stride = make_logits(R, V, seed=13)
    y, _ = make_logits(R, V, seed=14)
    got = run_logprobs(ctx, x, stride, torch.zeros(R, dtype=torch.int32, device="cuda"), K, 1.0)
    logits = x.gather(1, got["ids"].long())
    one = run_distill(ctx, y, stride, got["ids"], got["top"], T, 1.0, "one call")
    two = run_distill(ctx, y, stride, got["ids"], logits, T, 1.0, "one call")
    losses, tol_l, grad, tol_g = distill_ref(y, got["ids"].cpu(), logits.cpu(), T)
    near(two[0], losses, tol_l)
    # the log probabilities are the logits less a constant, each rounded to half a last bit of itself (below 16: 2^-21) after tol_logp (below 2e-5)
    shift = 2 * (2e-5 + 2.0 ** -21) / T
    near(one[0], losses, tol_l + shift * (losses.abs() + 12.0))
    student = torch.full((R, V), NEG, device="cuda").scatter_(1, got["ids"].long(), logits)
    same = run_distill(ctx, student, V, got["ids"], logits, T, 1.0, "one call")
    losses, tol_l, grad, tol_g = distill_ref(student, got["ids"].cpu(), logits.cpu(), T)
    near(same[0], losses, tol_l)
    assert float(losses.abs().max()) < 1e-12
    near(same[2], grad, tol_g)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("R,V,pad", [(8, 3000, 0), (512, 900, 0), (512, 17000, 0), (512, 6001, 1)])
def test_gradient_of_the_smallest_temperature(ctx, R, V, pad, form):
    x, stride = make_logits(R, V, pad, 0, seed=45)
    ids, a = make_teacher(R, V, 3, 12)
    losses, tol_l, grad, tol_g = distill_ref(x, ids, a, 1e-30, 1e9)
    part, out, got = run_distill(ctx, x, stride, ids, a, 1e-30, 1e9, form)
    near(got, grad, tol_g)


@pytest.mark.parametrize("R,V", [(1, 300), (7, 3000), (300, 25000), (460, 901), (460, 9000)])
@pytest.mark.parametrize("first", [False, True])
def test_logits_and_gradients_side_by_side(ctx, R, V, first):
    stride = 2 * V + 8
    x0, _ = make_logits(R, V, seed=44)
    ids, a = make_teacher(R, V, 5, 11)
    losses, tol_l, grad, tol_g = distill_ref(x0, ids, a, 1.0, 1.0)
    for form in range(2):
        both = torch.full((R, stride), 5.0, device="cuda")
        x, got = (both[:, V + 4:2 * V + 4], both[:, :V]) if first else (both[:, :V], both[:, V + 4:2 * V + 4])
        x.copy_(x0)
        one, part, out, stats = torch.ones(1, device="cuda"), torch.empty(R, device="cuda"), torch.empty(1, device="cuda"), torch.empty(R, 2, device="cuda")
        if form == 0:
            ctx.distillation_loss(x, ids.cuda(), a.cuda(), part, out, stats, one, got, R, V, 5, 1.0, stride)
        else:
            ctx.distillation_loss(x, ids.cuda(), a.cuda(), part, out, stats, None, None, R, V, 5, 1.0, stride)
            ctx.distillation_loss_backward(x, ids.cuda(), a.cuda(), stats, one, got, R, V, 5, 1.0, stride)
        torch.cuda.synchronize()
        near(got, grad, tol_g)
        assert torch.equal(x, x0) and bool((both[:, V:V + 4] == 5.0).all()) and bool((both[:, 2 * V + 4:] == 5.0).all())


# ---- streams, recordings, repetition --------------------------------------------------------------------------------------

def test_recorded_and_replayed_with_new_inputs(ctx):
    R, V, K = 37, 32000, 20
    x, stride = make_logits(R, V, seed=15)
    tokens = torch.randint(0, V, (R,), dtype=torch.int32).to("cuda")
    logp, H, ids, top, stats = (torch.empty(R, device="cuda"), torch.empty(R, device="cuda"), torch.empty(R, K, dtype=torch.int32, device="cuda"),
                                torch.empty(R, K, device="cuda"), torch.empty(R, 2, device="cuda"))
    one, up = torch.ones(1, device="cuda"), torch.randn(R, device="cuda")
    part, out, g1, g2 = torch.empty(R, device="cuda"), torch.empty(1, device="cuda"), torch.empty_like(x), torch.empty_like(x)

    def step():
        ctx.token_logprobs(x, tokens, logp, H, ids, top, stats, R, V, K)
        ctx.token_logprobs_backward(x, tokens, stats, H, up, up, g1, R, V)
        ctx.distillation_loss(x, ids, top, part, out, None, one, g2, R, V, K)

    outs = (logp, H, ids, top, stats, g1, part, out, g2)
    torch.cuda.synchronize()
    ctx.batch_begin()
    step()
    batch = ctx.batch_end()
    for seed in range(3):
        y, _ = make_logits(R, V, seed=20 + seed)
        x.copy_(y)
        batch.launch()
        ctx.finish()
        first = [t.clone() for t in outs]
        for t in outs:
            t.zero_()
        step()
        ctx.finish()
        for a, b in zip(first, outs):
            assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    batch.close()


def test_two_contexts_at_once(ctx):
    from motifcl_b200 import Context
    R, V, K = 60, 20000, 33
    x, stride = make_logits(R, V, seed=30)
    y, _ = make_logits(R, V, seed=31)
    torch.cuda.synchronize()
    tokens = torch.zeros(R, dtype=torch.int32, device="cuda")
    want = [run_logprobs(ctx, t, stride, tokens, K, 1.0) for t in (x, y)]
    other = Context(0)
    outs = [[torch.empty_like(w[n]) for n in ("logp", "H", "ids", "top", "stats")] for w in want]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, t, o in ((ctx, x, outs[0]), (other, y, outs[1])):
            c.token_logprobs(t, tokens, *o, R, V, K)
    ctx.finish()
    other.finish()
    for w, o in zip(want, outs):
        for n, t in zip(("logp", "H", "ids", "top", "stats"), o):
            assert torch.equal(w[n].view(torch.int32), t.view(torch.int32)), n
    other.close()


@pytest.mark.parametrize("R,V", [(300, 30000), (160, 60001), (460, 700), (460, 9001)])
def test_distillation_recorded_and_on_two_contexts_at_once(ctx, R, V):
    """Rings of chunks, clusters of them, and warps a row: the same bits alone, replayed with new inputs, and while another context runs the same."""
    from motifcl_b200 import Context
    K = 12
    x, y = make_logits(R, V, seed=32)[0], make_logits(R, V, seed=33)[0]
    ids, a = (t.to("cuda") for t in make_teacher(R, V, K, 8))
    one = torch.ones(1, device="cuda")
    outs = lambda: (torch.empty(R, device="cuda"), torch.empty(1, device="cuda"), torch.empty(R, 2, device="cuda"), torch.empty(R, V, device="cuda"))

    def step(c, t, o):
        c.distillation_loss(t, ids, a, o[0], o[1], o[2], one, o[3], R, V, K)

    same = lambda p, q: all(torch.equal(u.view(torch.int32), v.view(torch.int32)) for u, v in zip(p, q))
    want, got = [outs(), outs()], [outs(), outs()]
    other = Context(0)
    torch.cuda.synchronize()
    step(ctx, x, want[0])
    step(ctx, y, want[1])
    ctx.finish()
    for _ in range(4):
        step(ctx, x, got[0])
        step(other, y, got[1])
    ctx.finish()
    other.finish()
    assert same(want[0], got[0]) and same(want[1], got[1])
    ctx.batch_begin()
    step(ctx, x, got[0])
    batch = ctx.batch_end()
    x.copy_(y)
    torch.cuda.synchronize()
    for _ in range(3):
        for t in got[0]:
            t.zero_()
        torch.cuda.synchronize()
        batch.launch()
        ctx.finish()
        assert same(want[1], got[0])
    batch.close()
    other.close()


def test_a_row_beyond_32_bits_of_offset(ctx):
    """2.2e9 floats from the first row to the last: 8.9 GB, of which three rows are looked at."""
    V, stride = 1000, 50_000_000
    R = 45
    store = torch.empty(R * stride, device="cuda")
    x = store.view(R, stride)[:, :V]
    g = torch.Generator().manual_seed(40)
    x.copy_((torch.randn(R, V, generator=g) * 3).to("cuda"))
    check_logprobs(ctx, x, stride, 10, 1.0, torch.arange(R))
    fwd = run_logprobs(ctx, x, stride, torch.arange(R, dtype=torch.int32, device="cuda"), 0, 1.0)
    want, tol = policy_grad(Row64(x, 1.0), torch.arange(R), torch.ones(R), None)
    ctx.token_logprobs_backward(x, torch.arange(R, dtype=torch.int32, device="cuda"), fwd["stats"], None, torch.ones(R, device="cuda"), None, x, R, V, 1.0, stride)
    torch.cuda.synchronize()
    near(x, want, tol)


# ---- refusals ---------------------------------------------------------------------------------------------------------------

def test_refusals(ctx):
    from motifcl_b200 import MotifclCudaError
    R, V, K = 4, 100, 5
    x = torch.randn(R, V, device="cuda")
    tok = torch.zeros(R, dtype=torch.int32, device="cuda")
    f = lambda *s: torch.empty(*s, device="cuda")
    ids, a, one = torch.zeros(R, K, dtype=torch.int32, device="cuda"), f(R, K), torch.ones(1, device="cuda")
    big = torch.zeros(R, 200, dtype=torch.int32, device="cuda")

    def refused(text, call, *args, **kw):
        with pytest.raises(MotifclCudaError) as e:
            call(*args, **kw)
        assert e.value.code == 1 and text in e.value.message, e.value.message

    lp = ctx.token_logprobs
    refused("non-zero", lp, x, tok, f(R), None, None, None, None, 0, V)
    refused("non-zero", lp, x, tok, f(R), None, None, None, None, R, 0)
    refused("row_stride", lp, x, tok, f(R), None, None, None, None, R, V, row_stride=V - 1)
    refused("too large", lp, x, tok, f(R), None, None, None, None, R, V, row_stride=1 << 62)
    refused("too large", lp, x, tok, f(R), None, None, None, None, R, 1 << 31)
    refused("too large", lp, x, tok, f(R), None, None, None, None, R, (1 << 30) + 1)
    for T in (0.0, -1.0, math.nan, math.inf, 1e-35, 1e35):
        refused("temperature", lp, x, tok, f(R), None, None, None, None, R, V, 0, T)
    refused("n_top", lp, x, tok, f(R), None, big, f(R, 200), None, R, V, 129)
    refused("n_top", lp, x[:, :3].contiguous(), tok, f(R), None, ids, f(R, K), None, R, 3, 4)
    refused("go together", lp, x, tok, None, None, None, None, None, R, V)
    refused("go together", lp, x, None, f(R), None, None, None, None, R, V)
    refused("go together", lp, x, tok, f(R), None, None, None, None, R, V, 3)
    refused("go together", lp, x, tok, f(R), None, ids, None, None, R, V, 0)
    refused("no output", lp, x, None, None, None, None, None, None, R, V)
    refused("logits is NULL", lp, None, tok, f(R), None, None, None, None, R, V)
    refused("aligned", lp, x.data_ptr() + 2, tok, f(R), None, None, None, None, R, V)
    bw = ctx.token_logprobs_backward
    refused("no gradient", bw, x, tok, f(R, 2), f(R), None, None, f(R, V), R, V)
    refused("tokens is NULL", bw, x, None, f(R, 2), f(R), f(R), None, f(R, V), R, V)
    refused("entropy is NULL", bw, x, tok, f(R, 2), None, None, f(R), f(R, V), R, V)
    refused("row_stats is NULL", bw, x, tok, None, None, f(R), None, f(R, V), R, V)
    refused("grad_logits is NULL", bw, x, tok, f(R, 2), None, f(R), None, None, R, V)
    refused("overlaps", bw, x, tok, f(R, 2), None, f(R), None, x.data_ptr() + 16, R, V)
    dl = ctx.distillation_loss
    refused("teacher tokens", dl, x, ids, a, f(R), f(1), None, None, None, R, V, 0)
    refused("teacher tokens", dl, x, big, f(R, 200), f(R), f(1), None, None, None, R, V, 129)
    refused("teacher_ids is NULL", dl, x, None, a, f(R), f(1), None, None, None, R, V, K)
    refused("partial is NULL", dl, x, ids, a, None, f(1), None, None, None, R, V, K)
    refused("out is NULL", dl, x, ids, a, f(R), None, None, None, None, R, V, K)
    refused("go together", dl, x, ids, a, f(R), f(1), None, one, None, R, V, K)
    refused("go together", dl, x, ids, a, f(R), f(1), None, None, f(R, V), R, V, K)
    refused("overlaps", dl, x, ids, a, f(R), f(1), None, one, x.data_ptr() + 4, R, V, K)
    db = ctx.distillation_loss_backward
    refused("row_stats is NULL", db, x, ids, a, None, one, f(R, V), R, V, K)
    refused("grad_out is NULL", db, x, ids, a, f(R, 2), None, f(R, V), R, V, K)
    refused("temperature", db, x, ids, a, f(R, 2), one, f(R, V), R, V, K, -2.0)
    ctx.finish()
