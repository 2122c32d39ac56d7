"""Layer norm forward and backward against the definition in float64, and the output end of a model as one run: layer norm, classifier,
a teacher's most probable tokens, the student's loss and its gradient back to the norm's weights.

Tolerances, u = 2^-24 (half a last bit), n = (x - mean) / deviation, N columns, A = N / 1024 + 20 additions a term goes through at most
(four columns at a time by 256 threads, or a warp's part, then a tree):
    mean          (A + 1) u mean|x|
    x - mean      u |x - mean| + the mean's error
    variance      twice the relative error of x - mean in the mean of squares (first order of the mean's error drops out: x - mean sums to
                  0), (A + 3) u; 1 / sqrt: half of it, 3 u more
    n             relative (A / 2 + 8) u, plus the mean's error over the deviation
    y             |n w| times that, 2 u (|n w| + |b|)
    dx            every term has n's or a sum's error: see dx_tol
    dw, db        sums over R rows: (R / (rows added by one thread at a time) ... at most R) additions bounded by R' = R / 8 + 40, of terms
                  with n's error
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Norm64:
    def __init__(self, x, w, b, dy, eps):
        x, w, dy = x.double(), w.double(), dy.double()
        R, N = x.shape
        self.mean = x.mean(dim=1, keepdim=True)
        var = ((x - self.mean) ** 2).mean(dim=1, keepdim=True)
        self.inv = 1.0 / torch.sqrt(var + eps)
        n = (x - self.mean) * self.inv
        self.y = n * w + (b.double() if b is not None else 0.0)
        g = dy * w
        sg, sgn = g.mean(dim=1, keepdim=True), (g * n).mean(dim=1, keepdim=True)
        self.dx = self.inv * (g - sg - n * sgn)
        self.dw, self.db = (dy * n).sum(dim=0), dy.sum(dim=0)
        A = N / 1024 + 20
        self.tol_mean = (A + 1) * U * x.abs().mean(dim=1, keepdim=True)
        shift = self.tol_mean * self.inv                           # of n, from the mean
        self.tol_inv = self.inv * ((A / 2 + 8) * U + shift ** 2)
        tol_n = n.abs() * ((A / 2 + 8) * U + shift ** 2) + shift + U * n.abs()
        self.tol_y = tol_n * w.abs() + 2 * U * ((n * w).abs() + (b.double().abs() if b is not None else 0.0))
        mg, mgn = g.abs().mean(dim=1, keepdim=True), (g * n).abs().mean(dim=1, keepdim=True)
        tol_sgn = (A + 3) * U * mgn + (g.abs() * tol_n).mean(dim=1, keepdim=True)
        self.tol_dx = self.inv * (4 * U * (g.abs() + mg + (n * sgn).abs()) + (A + 2) * U * mg + n.abs() * tol_sgn + tol_n * sgn.abs()) + \
            self.dx.abs() * ((A / 2 + 8) * U + shift ** 2)
        adds = R / 8 + 40
        self.tol_dw = (dy.abs() * tol_n).sum(dim=0) + (adds + 3) * U * (dy * n).abs().sum(dim=0)
        self.tol_db = (adds + 1) * U * dy.abs().sum(dim=0)


def near(got, want, tol, what):
    err = (got.detach().cpu().double().reshape(want.shape) - want).abs()
    assert bool((err <= tol + 1e-37).all()), (what, float((err / (tol + 1e-37)).max()))


def inputs(R, N, seed=0, offset=0.0, spread=1.7):
    g = torch.Generator().manual_seed(seed * 7919 + R * 31 + N)
    x = torch.randn(R, N, generator=g) * spread + torch.randn(R, 1, generator=g) + offset
    return x, torch.rand(N, generator=g) + 0.5, torch.randn(N, generator=g) * 0.3, torch.randn(R, N, generator=g)


def place(t, shift=0):
    """On the device, `shift` floats behind a 16-byte boundary."""
    flat = torch.full((t.numel() + shift,), math.nan, device="cuda")
    v = flat[shift:].view(t.shape)
    v.copy_(t)
    return v


SHAPES = [(1, 1), (7, 1), (3, 2), (5, 31), (9, 64), (33, 100), (257, 288), (64, 300), (1000, 384), (3, 511), (20, 1000), (40, 1024), (17, 1025), (300, 2048),
          (1, 4096), (150, 4100), (10, 8192), (5, 8196), (6, 20001), (5000, 96), (700, 1536)]


@pytest.mark.parametrize("R,N", SHAPES)
@pytest.mark.parametrize("shift,bias", [(0, True), (1, False)])
def test_layernorm_forward_and_backward(ctx, R, N, shift, bias):
    x, w, b, dy = inputs(R, N)
    eps = 1e-5
    want = Norm64(x, w, b if bias else None, dy, eps)
    xd, wd, bd, dyd = place(x, shift), place(w, shift), place(b, shift) if bias else None, place(dy, shift)
    y, stats, dx = place(torch.zeros(R, N), shift), torch.empty(R, 2, device="cuda"), place(torch.zeros(R, N), shift)
    dw, db = torch.full((N,), 123.0, device="cuda"), torch.full((N,), 123.0, device="cuda")
    ctx.layernorm(xd, wd, bd, y, stats, R, N, eps)
    ctx.layernorm_backward(xd, wd, dyd, stats, dx, dw, db, R, N)
    torch.cuda.synchronize()
    near(y, want.y, want.tol_y, "y")
    near(stats[:, :1], want.mean, want.tol_mean, "mean")
    near(stats[:, 1:], want.inv, want.tol_inv, "inverse deviation")
    near(dx, want.dx, want.tol_dx, "dx")
    near(dw, want.dw, want.tol_dw, "dw")
    near(db, want.db, want.tol_db, "db")
    y2 = torch.empty(R, N, device="cuda")
    ctx.layernorm(xd, wd, bd, y2, None, R, N, eps)                  # statistics not kept
    torch.cuda.synchronize()
    near(y2, want.y, want.tol_y, "y without statistics")


@pytest.mark.parametrize("N", [96, 288, 2048, 9000])
@pytest.mark.parametrize("offset,spread", [(300.0, 1.0), (-5e4, 3.0), (0.0, 1e-6), (0.0, 1e15)])
def test_rows_far_from_zero_small_and_large(ctx, N, offset, spread):
    x, w, b, dy = inputs(12, N, 3, offset, spread)
    want = Norm64(x, w, b, dy, 1e-12)
    xd, wd, bd, dyd = (t.to("cuda") for t in (x, w, b, dy))
    y, stats, dx, dw, db = torch.empty_like(xd), torch.empty(12, 2, device="cuda"), torch.empty_like(xd), torch.empty_like(wd), torch.empty_like(wd)
    ctx.layernorm(xd, wd, bd, y, stats, 12, N, 1e-12)
    ctx.layernorm_backward(xd, wd, dyd, stats, dx, dw, db, 12, N)
    torch.cuda.synchronize()
    near(y, want.y, want.tol_y, "y")
    near(dx, want.dx, want.tol_dx, "dx")
    near(dw, want.dw, want.tol_dw, "dw")


@pytest.mark.parametrize("R,N", [(50, 288), (50, 2048), (9, 9001)])
def test_constant_rows_and_rows_with_nan(ctx, R, N):
    x, w, b, dy = inputs(R, N, 4)
    x[1] = 0.0
    x[2] = 3.0                                                      # exactly representable sums: n = 0
    x[3, N // 2] = math.nan
    x[4, 0] = math.inf
    xd, wd, bd, dyd = (t.to("cuda") for t in (x, w, b, dy))
    y, stats, dx = torch.empty_like(xd), torch.empty(R, 2, device="cuda"), torch.empty_like(xd)
    ctx.layernorm(xd, wd, bd, y, stats, R, N, 1e-5)
    ctx.layernorm_backward(xd, wd, dyd, stats, dx, None, None, R, N)
    torch.cuda.synchronize()
    assert torch.equal(y[1:3].cpu(), b.expand(2, N)) and bool(torch.isfinite(dx[1:3]).all())
    bad = torch.zeros(R, dtype=torch.bool)
    bad[3:5] = True
    assert torch.equal(torch.isnan(y).any(dim=1).cpu(), bad) and torch.equal(torch.isnan(dx).any(dim=1).cpu(), bad)


@pytest.mark.parametrize("R,N", [(200, 288), (100, 2048), (30, 4096), (12, 9000), (40, 333)])
def test_outputs_not_asked_for_in_place_and_the_same_bits_again(ctx, R, N):
    x, w, b, dy = (t.to("cuda") for t in inputs(R, N, 5))
    stats, dx, dw, db = torch.empty(R, 2, device="cuda"), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    y = torch.empty_like(x)
    ctx.layernorm(x, w, b, y, stats, R, N, 1e-5)
    ctx.layernorm_backward(x, w, dy, stats, dx, dw, db, R, N)
    outs = [torch.zeros_like(t) for t in (dx, dw, db)]
    ctx.layernorm_backward(x, w, dy, stats, outs[0], None, None, R, N)
    ctx.layernorm_backward(x, w, dy, stats, None, outs[1], None, R, N)
    ctx.layernorm_backward(x, w, dy, stats, None, None, outs[2], R, N)
    torch.cuda.synchronize()
    for a, c in zip((dx, dw, db), outs):
        assert torch.equal(a, c)
    for at in ("x", "dy"):
        x2, dy2, w2, b2 = x.clone(), dy.clone(), torch.empty_like(w), torch.empty_like(w)
        ctx.layernorm_backward(x2, w, dy2, stats, x2 if at == "x" else dy2, w2, b2, R, N)
        torch.cuda.synchronize()
        assert torch.equal(x2 if at == "x" else dy2, dx) and torch.equal(w2, dw) and torch.equal(b2, db)
    x2 = x.clone()
    ctx.layernorm(x2, w, b, x2, None, R, N, 1e-5)
    torch.cuda.synchronize()
    assert torch.equal(x2, y)


def test_gradients_against_differences(ctx):
    """Directional derivatives of the definition in float64, step 1e-5: off by 1e-9 of the third derivative's size."""
    R, N, eps, h = 6, 70, 1e-5, 1e-5
    x, w, b, dy = inputs(R, N, 6)
    stats, dx, dw, db = torch.empty(R, 2, device="cuda"), torch.empty(R, N, device="cuda"), torch.empty(N, device="cuda"), torch.empty(N, device="cuda")
    xd, wd, bd, dyd = (t.to("cuda") for t in (x, w, b, dy))
    ctx.layernorm(xd, wd, bd, torch.empty_like(xd), stats, R, N, eps)
    ctx.layernorm_backward(xd, wd, dyd, stats, dx, dw, db, R, N)
    torch.cuda.synchronize()

    def loss(x, w, b):
        c = x - x.mean(dim=1, keepdim=True)
        return ((c / torch.sqrt((c * c).mean(dim=1, keepdim=True) + eps) * w + b) * dy.double()).sum()

    p = [t.double() for t in (x, w, b)]
    for i, got in enumerate((dx, dw, db)):
        v = torch.randn(p[i].shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        up = loss(*[t + h * v if j == i else t for j, t in enumerate(p)])
        down = loss(*[t - h * v if j == i else t for j, t in enumerate(p)])
        got = got.cpu().double()
        assert abs(float((got * v).sum()) - float(up - down) / (2 * h)) <= 1e-5 * float(got.norm() * v.norm())


def test_recorded_and_replayed(ctx):
    R, N = 90, 2048
    x, w, b, dy = (t.to("cuda") for t in inputs(R, N, 7))
    y, stats, dx, dw, db = torch.empty_like(x), torch.empty(R, 2, device="cuda"), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)

    def step():
        ctx.layernorm(x, w, b, y, stats, R, N, 1e-5)
        ctx.layernorm_backward(x, w, dy, stats, dx, dw, db, R, N)

    step()                                                          # the workspace has its size
    torch.cuda.synchronize()
    ctx.batch_begin()
    step()
    batch = ctx.batch_end()
    for seed in range(3):
        x.copy_(inputs(R, N, 8 + seed)[0])
        batch.launch()
        ctx.finish()
        first = [t.clone() for t in (y, stats, dx, dw, db)]
        step()
        ctx.finish()
        for a, c in zip(first, (y, stats, dx, dw, db)):
            assert torch.equal(a, c)
    batch.close()


def test_refusals(ctx):
    from motifcl_b200 import MotifclCudaError
    f = lambda *s: torch.ones(*s, device="cuda")
    R, N = 3, 8

    def refused(text, call, *args):
        with pytest.raises(MotifclCudaError) as e:
            call(*args)
        assert e.value.code == 1 and text in e.value.message, e.value.message

    ln, bw = ctx.layernorm, ctx.layernorm_backward
    refused("non-zero", ln, f(R, N), f(N), f(N), f(R, N), None, 0, N, 1e-5)
    refused("non-zero", ln, f(R, N), f(N), f(N), f(R, N), None, R, 0, 1e-5)
    refused("too large", ln, f(R, N), f(N), f(N), f(R, N), None, R, 1 << 31, 1e-5)
    refused("too large", ln, f(R, N), f(N), f(N), f(R, N), None, R, (1 << 30) + 1, 1e-5)
    refused("too large", bw, f(R, N), f(N), f(R, N), f(R, 2), f(R, N), None, None, R, (1 << 30) + 1)
    for eps in (-1e-6, math.nan, math.inf):
        refused("eps", ln, f(R, N), f(N), f(N), f(R, N), None, R, N, eps)
    refused("x is NULL", ln, None, f(N), f(N), f(R, N), None, R, N, 1e-5)
    refused("weight is NULL", ln, f(R, N), None, f(N), f(R, N), None, R, N, 1e-5)
    refused("out is NULL", ln, f(R, N), f(N), f(N), None, None, R, N, 1e-5)
    refused("aligned", ln, f(R, N).data_ptr() + 1, f(N), f(N), f(R, N), None, R, N, 1e-5)
    refused("no output", bw, f(R, N), f(N), f(R, N), f(R, 2), None, None, None, R, N)
    refused("row_stats is NULL", bw, f(R, N), f(N), f(R, N), None, f(R, N), None, None, R, N)
    refused("grad_out is NULL", bw, f(R, N), f(N), None, f(R, 2), f(R, N), None, None, R, N)
    refused("non-zero", bw, f(R, N), f(N), f(R, N), f(R, 2), f(R, N), None, None, R, 0)
    ctx.finish()


@pytest.mark.parametrize("R,D,V,K,T", [(70, 288, 3000, 20, 2.0), (5, 64, 40000, 8, 1.0)])
def test_the_output_end_of_a_model(ctx, R, D, V, K, T):
    """Student and teacher: layer norm, classifier; the teacher's most probable tokens; the student's loss, its gradient through the classifier
    and the norm.  float64 end to end, relative L2 of each result: the classifier's products are held to 1e-5 by the header, and every
    other step to less, so 4e-5 for what went through two of them."""
    x, w, b, _ = inputs(R, D, 9)
    g = torch.Generator().manual_seed(R)
    xt = x + 0.3 * torch.randn(R, D, generator=g)
    head = torch.randn(V, D, generator=g) * (3.0 / math.sqrt(D))
    xd, xtd, wd, bd, hd = (t.to("cuda") for t in (x, xt, w, b, head))
    h, ht, stats = torch.empty_like(xd), torch.empty_like(xd), torch.empty(R, 2, device="cuda")
    zs, zt = torch.empty(R, V, device="cuda"), torch.empty(R, V, device="cuda")
    ids, top = torch.empty(R, K, dtype=torch.int32, device="cuda"), torch.empty(R, K, device="cuda")
    part, out, one = torch.empty(R, device="cuda"), torch.empty(1, device="cuda"), torch.ones(1, device="cuda")
    dh, dhead, dx, dw, db = torch.empty_like(xd), torch.empty_like(hd), torch.empty_like(xd), torch.empty_like(wd), torch.empty_like(wd)
    ctx.layernorm(xtd, wd, bd, ht, None, R, D, 1e-5)
    ctx.matmul_f32(ht, hd, zt, R, D, V, trans_b=True)
    ctx.token_logprobs(zt, None, None, None, ids, top, None, R, V, K)
    ctx.layernorm(xd, wd, bd, h, stats, R, D, 1e-5)
    ctx.matmul_f32(h, hd, zs, R, D, V, trans_b=True)
    ctx.distillation_loss(zs, ids, top, part, out, None, one, zs, R, V, K, T)       # the gradient in the logits' place
    ctx.matmul_f32(zs, hd, dh, R, V, D)
    ctx.matmul_f32(zs, h, dhead, V, R, D, trans_a=True)
    ctx.layernorm_backward(xd, wd, dh, stats, dx, dw, db, R, D)
    torch.cuda.synchronize()

    norm = lambda x, w, b: torch.nn.functional.layer_norm(x, (D,), w, b, 1e-5)
    p = [t.double().requires_grad_(True) for t in (x, w, b, head)]
    with torch.no_grad():
        at = torch.log_softmax(norm(xt.double(), p[1], p[2]) @ p[3].T, dim=1).gather(1, ids.cpu().long())
    t = torch.softmax(at / T, dim=1)
    q = torch.log_softmax(norm(p[0], p[1], p[2]) @ p[3].T / T, dim=1).gather(1, ids.cpu().long())
    losses = (t * (t.log() - q)).sum(dim=1)
    grads = torch.autograd.grad(losses.mean(), p)
    rel = lambda a, r: float((a.cpu().double() - r).norm() / r.norm())
    assert rel(top, at) <= 2e-5 and rel(part, losses.detach()) <= 4e-5
    for got, want in zip((dx, dw, db, dhead), grads):
        assert rel(got, want) <= 4e-5
