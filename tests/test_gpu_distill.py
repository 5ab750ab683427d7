"""Distillation from a teacher's top logits against its formula in float64.

Tolerances.  Scaled logits s = (z - max) / T carry a few roundings: the exponentials are off by about 4 (1 + |s|) 2^-24 of
themselves, the sum l of V of them by no more than its worst term's and a few roundings of partial sums; log q by 8 (1 + |s|) 2^-24.
The loss is a sum of p (log p - log q) with p within 8 (1 + |t|) 2^-24 of itself.  A gradient element w T (q - p) inherits the
errors of q and p and is rounded to the logits' type once (u = finfo.eps / 2 of itself).  16 units instead of 8 are allowed.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS32 = 2.0 ** -24


def dev():
    return torch.device("cuda", 0)


def reference(z, t, idx, w, temp):
    """(loss, grad, error scales of both) in float64 on the CPU, row by row from the definition."""
    z, t, idx, w = z.double().cpu(), t.double().cpu(), idx.long().cpu(), w.double().cpu()
    m, v = z.shape
    there = (idx >= 0) & (t > -math.inf)
    some = there.any(1)
    s = z / temp
    top = s.max(1, keepdim=True).values
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(s - top)
    total = e.sum(1, keepdim=True)
    q = torch.where(total > 0, e / total, torch.zeros_like(e))
    tt = torch.where(there, t / temp, torch.full_like(t, -math.inf))
    tm = torch.where(some[:, None], tt.max(1, keepdim=True).values, torch.zeros((m, 1), dtype=torch.float64))
    pe = torch.where(there, torch.exp(tt - tm), torch.zeros_like(tt))
    p = pe / pe.sum(1, keepdim=True).clamp_min(1e-300)
    sj = (s - top).gather(1, idx.clamp(0, v - 1))
    log_q = torch.where(sj == -math.inf, sj, sj - torch.log(total))
    log_p = tt - tm - torch.log(pe.sum(1, keepdim=True).clamp_min(1e-300))
    terms = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p))
    loss = temp ** 2 * terms.sum(1)
    size = lambda x: torch.where(x.isfinite(), x.abs(), torch.zeros_like(x))  # noqa: E731
    loss_scale = temp ** 2 * (p * (1 + size(tt - tm)) * (2 + size(log_p) + size(log_q) + size(sj))).sum(1)
    grad = q * some[:, None]
    scale = q * (1 + size(s - top))
    grad.scatter_add_(1, idx.clamp(0, v - 1), -p)
    scale.scatter_add_(1, idx.clamp(0, v - 1), p * (1 + size(tt - tm)))
    f = temp * w[:, None]
    return loss, grad * f, loss_scale, scale * f.abs()


def case(m, v, k, dtype, seed, teacher_dtype=None, index_dtype=torch.int32, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    z = (torch.randn((m, v), generator=gen) * spread).to(dtype)
    t = (torch.randn((m, k), generator=gen) * 2.0).to(dtype if teacher_dtype is None else teacher_dtype)
    idx = torch.stack([torch.randperm(v, generator=gen)[:k] for _ in range(m)]) if k <= v else torch.randint(0, v, (m, k), generator=gen)
    w = torch.rand((m,), generator=gen) + 0.5
    drop = torch.rand((m, k), generator=gen) < 0.15
    idx = torch.where(drop, torch.full_like(idx, -1), idx)
    if m > 2:
        idx[m // 2] = -1                 # a row of nothing
    if k > 2 and m > 1:
        idx[0, 2] = idx[0, 0] = v - 1    # a class named twice
    return [x.to(dev()) for x in (z, t, idx.to(index_dtype), w)]


def run_all(z, t, idx, w, temp):
    from volterra_vae_amd.dense_ops import topk_distillation, topk_distillation_step
    plain = topk_distillation(z, t, idx, temperature=temp)
    leaf = z.detach().requires_grad_(True)
    loss = topk_distillation(leaf, t, idx, temperature=temp)
    (grad,) = torch.autograd.grad(loss, leaf, w)
    step_loss, step_grad = topk_distillation_step(z, t, idx, w, temperature=temp)
    return (plain, loss.detach(), step_loss), (grad, step_grad)


def check(z, t, idx, w, temp):
    ref, ref_grad, scale, grad_scale = reference(z, t, idx, w, temp)
    losses, grads = run_all(z, t, idx, w, temp)
    for loss in losses:
        err = (loss.double().cpu() - ref).abs()
        assert loss.dtype == torch.float32 and bool((err <= 16 * EPS32 * scale + 1e-30).all()), float((err / (scale + 1e-30)).max())
    for grad in grads:
        assert grad.dtype == z.dtype and grad.shape == z.shape
        err = (grad.double().cpu() - ref_grad).abs()
        tiny = torch.finfo(z.dtype).tiny * torch.finfo(z.dtype).eps   # below the smallest subnormal of the type
        bound = torch.finfo(z.dtype).eps / 2 * ref_grad.abs() + 16 * EPS32 * grad_scale + tiny
        assert bool((err <= bound).all()), float((err - bound).max())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("v", [1, 2, 3, 8, 17, 31, 64, 65, 127, 128, 255, 256, 500, 511, 1000, 1025, 4095, 4097, 16400, 32000, 33001, 65521, 70001])
def test_matches_the_formula(v, dtype):
    m = 37 if v < 3000 else 5
    for i, k in enumerate(sorted({1, min(v, 5), min(v, 33)})):
        check(*case(m, v, k, dtype, v + i), temp=[1.0, 2.0, 0.7][i])


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_teacher_types_index_types_and_strides(dtype):
    for v in (60, 3001, 40000):
        for td in DTYPES:
            for it in (torch.int32, torch.int64):
                z, t, idx, w = case(6, v, 9, dtype, v + 1, td, it)
                check(z, t, idx, w, 1.5)
        zb = torch.full((6, v + 5), float("nan"), dtype=dtype, device=dev())
        zs = zb[:, 3:3 + v]
        zs.copy_(z)
        tb, ib = torch.zeros((6, 14), dtype=t.dtype, device=dev()), torch.zeros((6, 11), dtype=idx.dtype, device=dev())
        tb[:, 2:11], ib[:, 1:10] = t, idx
        for a, b in zip(run_all(zs, tb[:, 2:11], ib[:, 1:10], w, 1.5)[0], run_all(z, t, idx, w, 1.5)[0]):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
        check(zs, tb[:, 2:11], ib[:, 1:10], w, 1.5)


def test_many_entries_and_repeated_classes():
    for dtype in DTYPES:
        for v, k in ((7, 100), (300, 1024), (5000, 1024), (5000, 200)):
            z, t, idx, w = case(9, v, k, dtype, v + k)
            idx[3] = 2 % v               # every entry of a row the same class
            check(z, t, idx, w, 1.0)
            a, b = run_all(z, t, idx, w, 1.0), run_all(z, t, idx, w, 1.0)
            assert all(torch.equal(p, q) for x, y in zip(a, b) for p, q in zip(x, y))


def test_masked_logits_and_rows_of_nothing():
    """-inf among the student's logits (masked classes), lowest finite values, rows of nothing but -inf, teachers at -inf."""
    for dtype in DTYPES:
        for v in (9, 200, 2000, 40000):
            z, t, idx, w = case(8, v, 4, dtype, 3)
            idx = torch.arange(4, device=dev(), dtype=torch.int32).repeat(8, 1)
            z[0, 5:] = -math.inf                  # masked classes that the teacher does not name
            z[1] = torch.finfo(dtype).min         # the type's lowest value everywhere: uniform
            z[1, 0] = 0.0
            t[2] = -math.inf                      # teacher without a present entry
            z[3, 4:] = torch.finfo(dtype).min
            idx[5] = -1
            z[5, 2] = math.nan                    # a row without entries is 0 whatever its logits
            losses, grads = run_all(z, t, idx, w, 1.0)
            ok = torch.tensor([0, 1, 2, 3, 4, 6, 7])
            ref, ref_grad, scale, grad_scale = reference(z[ok], t[ok], idx[ok], w[ok], 1.0)
            for loss in losses:
                assert bool(((loss.cpu().double()[ok] - ref).abs() <= 16 * EPS32 * scale + 1e-30).all())
                assert float(loss[2]) == 0.0 and float(loss[5]) == 0.0
            for grad in grads:
                g = grad.cpu().double()
                assert float(g[2].abs().sum()) == 0.0 and float(g[5].abs().sum()) == 0.0
                bound = torch.finfo(dtype).eps / 2 * ref_grad.abs() + 16 * EPS32 * grad_scale + torch.finfo(dtype).tiny
                assert bool(((g[ok] - ref_grad).abs() <= bound).all())
            # a class that the teacher names is masked: infinite loss, gradient w T (q - p) still finite
            z, t, idx, w = case(3, v, 2, dtype, 4)
            idx = torch.tensor([[0, 1]] * 3, dtype=torch.int32, device=dev())
            z[0, 0] = -math.inf
            z[1] = -math.inf
            losses, grads = run_all(z, t, idx, w, 1.0)
            for loss in losses:
                assert float(loss[0]) == math.inf and float(loss[1]) == math.inf and math.isfinite(float(loss[2]))
            _, ref_grad, _, grad_scale = reference(z, t, idx, w, 1.0)
            for grad in grads:
                bound = torch.finfo(dtype).eps / 2 * ref_grad.abs() + 16 * EPS32 * grad_scale + torch.finfo(dtype).tiny
                assert bool(((grad.cpu().double() - ref_grad).abs() <= bound).all())


def test_what_cannot_be_answered_is_nan_in_its_row_alone():
    for dtype in DTYPES:
        for v in (12, 300, 6000, 70000):
            z, t, idx, w = case(7, v, 3, dtype, 6)
            idx[:] = torch.tensor([0, 1, 2], device=dev())
            good = run_all(z, t, idx, w, 1.0)
            z[0, v - 1], z[1, 3], t[2, 1], idx[4, 2], t[5, 0] = math.nan, math.inf, math.nan, v, math.inf
            losses, grads = run_all(z, t, idx, w, 1.0)
            for a, b in zip(losses, good[0]):
                assert all(math.isnan(float(a[r])) for r in (0, 1, 2, 4, 5)) and torch.equal(a[[3, 6]], b[[3, 6]])
            for a, b in zip(grads, good[1]):
                assert all(bool(torch.isnan(a[r]).any()) for r in (0, 1, 2, 4, 5)) and torch.equal(a[[3, 6]], b[[3, 6]])


def test_no_rows_one_weight_for_all_and_a_side_stream():
    from volterra_vae_amd.dense_ops import topk_distillation, topk_distillation_step
    z, t, idx, w = case(40, 333, 6, torch.float32, 1)
    assert topk_distillation(z[:0], t[:0], idx[:0]).shape == (0,)
    assert topk_distillation_step(z[:0], t[:0], idx[:0], w[:0])[1].shape == (0, 333)
    leaf = z.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(topk_distillation(leaf, t, idx).mean(), leaf)   # upstream weights with stride 0
    want = topk_distillation_step(z, t, idx, torch.full_like(w, 1 / 40))[1]
    assert torch.allclose(g, want, rtol=1e-5, atol=1e-9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = topk_distillation(z, t, idx)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(loss, topk_distillation(z, t, idx))


def test_offsets_beyond_32_bits():
    """Logits and gradient of more than 2^32 elements, rows held in registers and rows read twice: the last rows
    against the formula (a row that starts elsewhere in a 16-byte piece adds up in another order)."""
    from volterra_vae_amd.dense_ops import topk_distillation_step
    for m, v in (((1 << 16) + 9, 65600), ((1 << 15) + 3, 131200), ((1 << 27) + 5, 33)):
        z = torch.zeros((m, v), dtype=torch.bfloat16, device=dev())
        zs, ts, idxs, ws = case(64, v, 4, torch.bfloat16, 2)
        z[-64:] = zs
        t, idx, w = ts[:1].repeat(m, 1), torch.zeros((m, 4), dtype=torch.int32, device=dev()), torch.ones(m, device=dev())
        t[-64:], idx[-64:], w[-64:] = ts, idxs, ws
        loss, grad = topk_distillation_step(z, t, idx, w)
        ref, ref_grad, scale, grad_scale = reference(zs, ts, idxs, ws, 1.0)
        assert bool(((loss[-64:].double().cpu() - ref).abs() <= 16 * EPS32 * scale + 1e-30).all())
        assert bool(((grad[-64:].double().cpu() - ref_grad).abs() <= 2.0 ** -8 * ref_grad.abs() + 16 * EPS32 * grad_scale + 1e-37).all())
        assert grad.numel() > 1 << 32 and bool(torch.isfinite(loss).all())
        del z, grad


def test_the_gradient_agrees_with_differences():
    """h = 2^-5 along a unit direction: truncation h^2 / 6 of a third derivative below 1 / T, rounding 2^-22 / h: 1e-3 of the scale."""
    from volterra_vae_amd.dense_ops import topk_distillation, topk_distillation_step
    z, t, idx, w = case(20, 50, 5, torch.float32, 2, spread=1.0)
    g = topk_distillation_step(z, t, idx, w, temperature=1.3)[1].double()
    gen = torch.Generator().manual_seed(0)
    v = torch.randn(z.shape, generator=gen).to(dev())
    v /= v.norm()
    h = 2.0 ** -5
    f = lambda a: (topk_distillation(a, t, idx, temperature=1.3).double() * w.double()).sum()  # noqa: E731
    fd = float((f(z + h * v) - f(z - h * v)) / (2 * h))
    assert abs(fd - float((g * v.double()).sum())) <= 1e-3 * float(g.norm())


def test_a_captured_step_replays():
    from volterra_vae_amd.dense_ops import topk_distillation_step
    for v in (40, 900, 50000):
        z, t, idx, w = case(30, v, 7, torch.bfloat16, v)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            topk_distillation_step(z, t, idx, w)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = topk_distillation_step(z, t, idx, w)
        for _ in range(3):
            z.copy_(z.roll(1, 0))
            eager = [x.clone() for x in topk_distillation_step(z, t, idx, w)]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(captured, eager))


def test_refusals():
    from volterra_vae_amd._lib import V2VAEError
    from volterra_vae_amd.dense_ops import topk_distillation, topk_distillation_step
    z, t = torch.zeros(6, 9, device=dev()), torch.zeros(6, 3, device=dev())
    i, w = torch.zeros(6, 3, dtype=torch.int64, device=dev()), torch.ones(6, device=dev())
    for error, match, args, kw in (
            (NotImplementedError, "float32, bfloat16 or float16", (z.double(), t, i), {}),
            (NotImplementedError, "teacher_logits", (z, t.double(), i), {}),
            (ValueError, "int32 or int64", (z, t, i.short()), {}),
            (ValueError, "expected", (z, t[:5], i), {}),
            (ValueError, "expected", (z, t, i[:, :2]), {}),
            (ValueError, "entries a row", (z, t[:, :0], i[:, :0]), {}),
            (ValueError, "entries a row", (z, torch.zeros(6, 1025, device=dev()), torch.zeros(6, 1025, dtype=torch.int32, device=dev())), {}),
            (ValueError, "no classes", (z[:, :0], t, i), {}),
            (ValueError, "unit stride", (torch.zeros(9, 6, device=dev()).t(), t, i), {}),
            (ValueError, "not differentiable in the teacher", (z, t.clone().requires_grad_(), i), {}),
            (RuntimeError, "no CPU implementation", (z, t.cpu(), i), {}),
            (V2VAEError, "v2vae_distill_fwd", (z[:1].expand(6, 9), t, i), {}),
            *((ValueError, "temperature", (z, t, i), dict(temperature=x)) for x in (0.0, -1.0, 9e-5, 2e4, float("nan"), float("inf")))):
        with pytest.raises(error, match=match):
            topk_distillation(*args, **kw)
    for bad in (w[:5], w.double(), torch.ones(1, device=dev()).expand(6)):
        with pytest.raises(ValueError, match="row_weight"):
            topk_distillation_step(z, t, i, bad)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_every_number_of_entries_beside_every_length_of_rows(dtype):
    """More entries than a short row's lanes, as many, fewer; classes named twice."""
    for v in (9, 33, 70, 130, 260, 600, 1500, 5000):
        for k in (1, 8, 9, 16, 17, 32, 33, 64, 65, 200):
            z, t, idx, w = case(7, v, min(k, v), dtype, v + k)
            if k > 3:
                idx[::2, 2] = idx[::2, 0]
            check(z, t, idx, w, 1.3)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_many_long_rows(dtype):
    """Rows that are streamed for the loss: aligned and not, with masked parts and rows of nothing, more entries than a wave has lanes."""
    for v, k in ((17029, 16), (8200, 100)):
        z, t, idx, w = case(520, v, k, dtype, v)
        z[:, 100:5000] = -math.inf
        z[7] = -math.inf
        idx[7] = -1
        idx[8, :2] = 3 * v // 4
        idx[idx >= 100] = idx[idx >= 100].clamp_min(5000)
        check(z, t, idx, w, 0.8)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_padded_rows_that_are_kept_on_the_host_between_the_passes(dtype):
    """save_on_cpu gives strided rows back contiguous; the gradient is that of the same rows without the hooks, to the rounding of sums
    whose rows start elsewhere in a 16-byte piece, and within the formula's bound."""
    from volterra_vae_amd.dense_ops import topk_distillation
    for v in (60, 3001, 40000):
        z, t, idx, w = case(6, v, 9, dtype, v + 2)
        zb, tb, ib = (torch.zeros((6, x.shape[1] + 7), dtype=x.dtype, device=dev()) for x in (z, t, idx))
        zb[:, 3:3 + v], tb[:, 2:11], ib[:, 1:10] = z, t, idx
        leaf = zb[:, 3:3 + v].requires_grad_(True)
        with torch.autograd.graph.save_on_cpu():
            loss = topk_distillation(leaf, tb[:, 2:11], ib[:, 1:10], temperature=1.5)
        (grad,) = torch.autograd.grad(loss, leaf, w)
        _, ref_grad, _, grad_scale = reference(z, t, idx, w, 1.5)
        tiny = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        bound = torch.finfo(dtype).eps / 2 * ref_grad.abs() + 16 * EPS32 * grad_scale + tiny
        assert bool(((grad.double().cpu() - ref_grad).abs() <= bound).all())
