"""Dense layers (linear, gated block) against their formulas in float64: sizes, strides, alignment, activations, gradients.

Tolerances.  With S2 = sqrt(sum_k x_k^2 w_k^2), a float32 sum of n rounded steps over such terms is off by about sqrt(n) 2^-24 S2
(independent roundings of partial sums no larger than a few S2); 8 of these are allowed.  A float32 product in three bf16 pieces
takes 6 accumulations per 16 terms and drops less than 2^-24 of a term, which the same bound covers.  A value rounded to the
tensors' type is off by at most u = finfo.eps / 2 of itself: once for a result, and once per term (at random, 6 sigma of u S2) for
dz, which is rounded before the two gradient products.  Activations have slopes up to 1.13 and second derivatives up to 1 and
are computed to a few units of 2^-24; the factor 4 on the float32 part of the gradients covers them.
Below finfo.tiny the step of a type is fixed at tiny * eps (2^-24 in float16), so a rounding is off by up to tiny * eps / 2 there
(2^-25), however small the value: once for a result, and for dz times sqrt(sum of squares) of what it is multiplied with.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS32 = 2.0 ** -24


def dev():
    return torch.device("cuda", 0)


def u(dtype):
    return torch.finfo(dtype).eps / 2


def normal(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * scale).to(dtype).to(dev())


def act64(kind, z):
    return {"none": lambda v: v, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
            "tanh": torch.tanh}[kind](z)


def s2(a, b):
    """sqrt(a^2 b^2) over the contraction of a [M, K] with b [N, K]."""
    return ((a * a) @ (b * b).t()).sqrt()


def floor_of(dtype):
    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2


def near(got, ref, bound, what):
    assert got.shape == ref.shape, what
    bound = bound + floor_of(got.dtype)
    err = (got.double() - ref).abs()
    worst = float((err - bound).max()) if err.numel() else -1.0
    assert torch.isfinite(got).all() and worst <= 0, f"{what}: error {float(err.max()):.3g} beyond its bound by {worst:.3g}"


def steps(k, dtype):
    return (6 * k / 16 if dtype == torch.float32 else k / 16) + 16


def laid_out(t, how):
    """The same values with another row stride / start: rows `pad` elements apart further, starting `lead` elements in."""
    lead, pad = {"plain": (0, 0), "odd": (1, 3), "wide": (8, 8)}[how]
    if how == "plain" or t.dim() != 2:
        return t
    buf = torch.full((lead + t.shape[0] * (t.shape[1] + pad) + 8,), 7.0, dtype=t.dtype, device=t.device)
    v = torch.as_strided(buf, t.shape, (t.shape[1] + pad, 1), lead)
    v.copy_(t)
    return v


SHAPES = [(1, 1, 1), (1, 4096, 72), (2, 129, 5), (5, 64, 130), (11, 50, 64), (16, 1000, 33), (17, 50, 64), (64, 64, 64), (65, 8, 1),
          (129, 130, 67), (200, 257, 300), (1000, 96, 33), (40, 3000, 24), (257, 512, 384), (2500, 48, 40), (3, 8200, 9), (30, 1000, 40), (4, 1301, 35), (7, 2049, 2050)]


def linear_case(m, k, n, dtype, act, bias, residual, how, seed):
    gen = torch.Generator().manual_seed(seed)
    x = laid_out(normal(gen, m, k, dtype=dtype), how)
    w = laid_out(normal(gen, n, k, scale=k ** -0.5, dtype=dtype), how)
    b = normal(gen, n, scale=0.5, dtype=dtype) if bias else None
    r = laid_out(normal(gen, m, n, dtype=dtype), how) if residual else None
    dy = laid_out(normal(gen, m, n, dtype=dtype), how)
    return x, w, b, r, dy


def check_linear(x, w, b, r, dy, act, got_y, grads, dtype):
    X, W, D = x.detach().double(), w.detach().double(), dy.double()
    leaves = [X.requires_grad_(True), W.requires_grad_(True)]
    B = b.detach().double().requires_grad_(True) if b is not None else None
    z = X @ W.t() + (B if B is not None else 0.0)
    y = act64(act, z)
    y = y + r.detach().double() if r is not None else y
    ref = torch.autograd.grad(y, leaves + ([B] if B is not None else []), D)
    X, W, y, z = X.detach(), W.detach(), y.detach(), z.detach()
    k, (m, n) = X.shape[1], y.shape
    f32 = 8 * EPS32 * steps(k, dtype) ** 0.5
    extra = (B.detach().abs() if B is not None else 0.0) + (r.detach().double().abs() if r is not None else 0.0)
    near(got_y, y, u(dtype) * y.abs() + 1.13 * f32 * s2(X, W) + 16 * EPS32 * (extra + y.abs()) + 1e-30, "y")
    if grads is None:
        return
    rounded, low = (0.0, 0.0) if act == "none" else (6 * u(dtype), 6 * floor_of(dtype))
    dx, dw, db = grads
    zerr = (1 + s2(X, W).max())   # an error of z of f32 * S2 enters act' with a second derivative up to 1
    near(dx, ref[0], u(dtype) * ref[0].abs() + (rounded + 32 * EPS32 * (steps(n, dtype) ** 0.5 + steps(k, dtype) ** 0.5) * zerr)
         * s2(D, W.t()) + low * s2(torch.ones_like(D), W.t()) + 1e-30, "dx")
    near(dw, ref[1], u(dtype) * ref[1].abs() + (rounded + 32 * EPS32 * (steps(m, dtype) ** 0.5 + steps(k, dtype) ** 0.5) * zerr)
         * s2(D.t(), X.t()) + low * s2(torch.ones_like(D).t(), X.t()) + 1e-30, "dw")
    if db is not None:
        near(db, ref[2], u(dtype) * ref[2].abs() + 32 * EPS32 * (m ** 0.5 + steps(k, dtype) ** 0.5) * zerr
             * (D * D).sum(0).sqrt() + 1e-30, "db")


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_linear_matches_its_formula(shape, dtype):
    from volterra_vae_amd.dense_ops import linear_backward, linear_forward
    m, k, n = shape
    seed = m * 7 + k * 3 + n
    kinds = ["none", "silu", "gelu", "tanh", "silu"]
    for i, how in enumerate(["plain", "odd", "wide"]):
        act = kinds[(seed + i) % 5]
        x, w, b, r, dy = linear_case(m, k, n, dtype, act, (seed + i) % 2 == 0, i > 0, how, seed + i)
        y, z = linear_forward(x, w, b, residual=r, activation=act, keep=True)
        y2, _ = linear_forward(x, w, b, residual=r, activation=act)
        assert torch.equal(y, y2)
        grads = linear_backward(dy, x, w, z, activation=act, need=(True, True, b is not None))
        check_linear(x, w, b, r, dy, act, y, grads, dtype)
        again = linear_backward(dy, x, w, z, activation=act, need=(True, True, b is not None))
        assert all(p is None or torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "tanh"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_linear_through_autograd_and_leading_dimensions(dtype, act):
    from volterra_vae_amd.dense_ops import linear
    x, w, b, r, dy = linear_case(6 * 35, 72, 56, dtype, act, True, True, "plain", 3)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    y = linear(leaves[0].view(6, 35, 72), leaves[1], leaves[2], residual=leaves[3].view(6, 35, 56), activation=act)
    assert y.shape == (6, 35, 56)
    y.backward(dy.view(6, 35, 56))
    check_linear(x, w, b, r, dy, act, y.detach().view(-1, 56), [t.grad for t in leaves[:3]], dtype)
    assert torch.equal(leaves[3].grad, dy)
    # the registered op is the same call; a gradient that is one number for all (stride 0) is accepted
    op = torch.ops.v2vae.linear(leaves[0], leaves[1], leaves[2], residual=leaves[3], activation=act)
    assert torch.equal(op, y.view(-1, 56))
    (g,) = torch.autograd.grad(op.sum(), leaves[2])
    check_linear(x, w, b, r, torch.ones_like(dy), act, op.detach(),
                 torch.autograd.grad(linear(leaves[0], leaves[1], leaves[2], residual=leaves[3], activation=act),
                                     leaves[:3], torch.ones_like(dy)), dtype)
    assert g.shape == b.shape


def check_gated(x, wg, wu, bg, bu, dh, act, h, grads, dtype):
    t = [v.detach().double().requires_grad_(True) if v is not None else None for v in (x, wg, wu, bg, bu)]
    X, G, U = t[:3]
    g = X @ G.t() + (t[3] if bg is not None else 0.0)
    up = X @ U.t() + (t[4] if bu is not None else 0.0)
    ref_h = act64(act, g) * up
    D = dh.double()
    ref = torch.autograd.grad(ref_h, [v for v in t if v is not None], D)
    X, G, U, g, up, ref_h = (v.detach() for v in (X, G, U, g, up, ref_h))
    k, (m, n) = X.shape[1], ref_h.shape
    a = act64(act, g).abs()
    bias = (0.0 if bg is None else bg.double().abs()), (0.0 if bu is None else bu.double().abs())
    f32 = 8 * EPS32 * steps(k, dtype) ** 0.5
    zg, zu = f32 * s2(X, G) + 16 * EPS32 * bias[0], f32 * s2(X, U) + 16 * EPS32 * bias[1]
    near(h, ref_h, u(dtype) * ref_h.abs() + 1.13 * zg * up.abs() + zu * a + 16 * EPS32 * ref_h.abs() + 1e-30, "h")
    if grads is None:
        return
    # |dg| <= 1.13 |dh u|, |du| <= |dh act(g)|; both rounded once
    dg, du = 1.13 * D.abs() * up.abs(), D.abs() * a
    slack = 32 * EPS32 * (1 + max(float(s2(X, G).max()), float(s2(X, U).max())))
    e_g, e_u = D.abs() * (1 + up.abs()), D.abs() * (1 + a)       # what errors of g and u are multiplied with

    def product(i, p, q, axis_steps, names):
        terms = sum(6 * u(dtype) * s2(v, o) + 6 * floor_of(dtype) * s2(torch.ones_like(v), o) + slack * (axis_steps ** 0.5 + steps(k, dtype) ** 0.5) * s2(e, o) for v, e, o in zip(p, q, names))
        near(grads[i], ref[i], u(dtype) * ref[i].abs() + terms + 1e-30, f"gradient {i}")

    product(0, (dg, du), (e_g, e_u), steps(2 * n, dtype), (G.t(), U.t()))
    product(1, (dg.t(),), (e_g.t(),), steps(m, dtype), (X.t(),))
    product(2, (du.t(),), (e_u.t(),), steps(m, dtype), (X.t(),))
    if bg is not None:
        for i, e in ((3, e_g), (4, e_u)):
            near(grads[i], ref[i], u(dtype) * ref[i].abs() + slack * (m ** 0.5 + steps(k, dtype) ** 0.5) * (e * e).sum(0).sqrt() + 1e-30,
                 f"gradient {i}")


def gated_case(m, k, n, dtype, bias, how, seed):
    gen = torch.Generator().manual_seed(seed)
    x = laid_out(normal(gen, m, k, dtype=dtype), how)
    wg, wu = (laid_out(normal(gen, n, k, scale=k ** -0.5, dtype=dtype), h) for h in (how, "wide" if how == "odd" else how))
    bg, bu = (normal(gen, n, scale=0.5, dtype=dtype) if bias else None for _ in range(2))
    return x, wg, wu, bg, bu, laid_out(normal(gen, m, n, dtype=dtype), how)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_gated_block_matches_its_formula(shape, dtype):
    from volterra_vae_amd.dense_ops import gated_backward, gated_forward
    m, k, n = shape
    for i, how in enumerate(["plain", "odd", "wide"]):
        act = ["silu", "gelu", "tanh"][(m + i) % 3]
        x, wg, wu, bg, bu, dh = gated_case(m, k, n, dtype, i != 1, how, m + k + n + i)
        h, gu = gated_forward(x, wg, wu, bg, bu, activation=act, keep=True)
        assert torch.equal(h, gated_forward(x, wg, wu, bg, bu, activation=act)[0])
        need = (True, True, True, bg is not None, bu is not None)
        grads = gated_backward(dh, x, wg, wu, gu, activation=act, need=need)
        check_gated(x, wg, wu, bg, bu, dh, act, h, grads, dtype)
        again = gated_backward(dh, x, wg, wu, gu, activation=act, need=need)
        assert all(p is None or torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_gated_block_through_autograd(dtype):
    from volterra_vae_amd.dense_ops import gated_linear
    x, wg, wu, bg, bu, dh = gated_case(150, 88, 104, dtype, True, "plain", 5)
    leaves = [t.clone().requires_grad_(True) for t in (x, wg, wu, bg, bu)]
    h = gated_linear(leaves[0].view(3, 50, 88), *leaves[1:], activation="gelu")
    h.backward(dh.view(3, 50, 104))
    check_gated(x, wg, wu, bg, bu, dh, "gelu", h.detach().view(150, 104), [t.grad for t in leaves], dtype)
    assert torch.equal(torch.ops.v2vae.gated_linear(*leaves, activation="gelu").view(-1), h.view(-1))
    # only one of the gradients wanted: the others are not formed and the one is the same
    only = [t.detach().clone() for t in leaves]
    only[2].requires_grad_(True)
    (g,) = torch.autograd.grad(gated_linear(*only, activation="gelu"), only[2], dh)
    assert torch.equal(g, leaves[2].grad)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_shapes_of_many_tiles(dtype):
    """Several tiles in both directions, ends that fill no tile, long contractions that are split, weights with different strides."""
    from volterra_vae_amd.dense_ops import gated_backward, gated_forward, linear_backward, linear_forward
    for m, k, n, act in ((4100, 1032, 520, "silu"), (300, 2056, 4104, "gelu"), (9000, 72, 136, "tanh"), (2304, 512, 2304, "none"), (70, 8192, 64, "none")):
        x, w, b, r, dy = linear_case(m, k, n, dtype, act, True, True, "wide", m)
        y, z = linear_forward(x, w, b, residual=r, activation=act, keep=True)
        check_linear(x, w, b, r, dy, act, y, linear_backward(dy, x, w, z, activation=act), dtype)
    for m, k, n in ((4100, 520, 1032), (600, 2048, 520), (5000, 64, 136)):
        x, wg, wu, bg, bu, dh = gated_case(m, k, n, dtype, True, "plain", m)
        for up in (wu, laid_out(wu, "wide"), laid_out(wu, "odd")):
            h, gu = gated_forward(x, wg, up, bg, bu, keep=True)
            check_gated(x, wg, up, bg, bu, dh, "silu", h, gated_backward(dh, x, wg, up, gu), dtype)


def test_gradients_agree_with_differences():
    """Central differences of float64-accumulated losses through the float32 kernels: step h = 2^-6, truncation h^2 / 6 times the third
    derivative along the direction (of order 1) and rounding 2^-24 / h of the values: 2e-3 of the directional derivative's scale."""
    from volterra_vae_amd.dense_ops import gated_linear, linear
    gen = torch.Generator().manual_seed(11)
    x, w, b = normal(gen, 90, 40), normal(gen, 30, 40, scale=0.15), normal(gen, 30, scale=0.3)
    wu, c = normal(gen, 30, 40, scale=0.15), normal(gen, 90, 30)
    for f, args in ((lambda *a: linear(*a, activation="gelu"), (x, w, b)), (lambda *a: gated_linear(a[0], a[1], a[2]), (x, w, wu))):
        for i in range(len(args)):
            leaves = [t.clone().requires_grad_(j == i) for j, t in enumerate(args)]
            (g,) = torch.autograd.grad(f(*leaves), leaves[i], c)
            v = normal(gen, *args[i].shape, scale=args[i].numel() ** -0.5)
            h = 2.0 ** -6
            hi, lo = ([t + s * h * v if j == i else t for j, t in enumerate(args)] for s in (1, -1))
            fd = ((f(*hi).double() - f(*lo).double()) * c.double()).sum() / (2 * h)
            scale = float(g.double().norm() * v.double().norm())
            assert abs(float(fd) - float((g.double() * v.double()).sum())) <= 2e-3 * scale


def test_rows_of_an_input_may_overlap():
    """Sliding windows of one sequence as a strided matrix, in both layouts of a product (x and its weight gradient)."""
    from volterra_vae_amd.dense_ops import linear_backward, linear_forward
    gen = torch.Generator().manual_seed(2)
    for dtype in DTYPES:
        y = normal(gen, 8 * 600 + 70, dtype=dtype)
        for window, hop in ((50, 2), (64, 8), (25, 1)):
            x = torch.as_strided(y, (600, window), (hop, 1), 3)
            w, dy = normal(gen, 20, window, scale=0.2, dtype=dtype), normal(gen, 600, 20, dtype=dtype)
            same = x.contiguous()
            assert torch.equal(linear_forward(x, w)[0], linear_forward(same, w)[0])
            for p, q in zip(linear_backward(dy, x, w), linear_backward(dy, same, w)):
                assert torch.equal(p, q)


@pytest.mark.parametrize("act", ["none", "relu"])
def test_gated_block_with_the_other_activations(act):
    from volterra_vae_amd.dense_ops import gated_backward, gated_forward
    for dtype in DTYPES:
        x, wg, wu, bg, bu, dh = gated_case(90, 56, 48, dtype, True, "plain", 21)
        h, gu = gated_forward(x, wg, wu, bg, bu, activation=act, keep=True)
        check_gated(x, wg, wu, bg, bu, dh, act, h, gated_backward(dh, x, wg, wu, gu, activation=act), dtype)


def test_one_row_repeated_and_one_tensor_in_two_places():
    """Rows with stride 0, the input as its own residual, one weight as gate and up: values and summed gradients."""
    from volterra_vae_amd.dense_ops import gated_linear, linear
    gen = torch.Generator().manual_seed(6)
    for dtype in DTYPES:
        row, w = normal(gen, 1, 64, dtype=dtype), normal(gen, 64, 64, scale=0.1, dtype=dtype)
        for m in (5, 40, 1500):
            assert torch.equal(linear(row.expand(m, 64), w), linear(row.repeat(m, 1), w))
            assert torch.equal(gated_linear(row.expand(m, 64), w, w), gated_linear(row.repeat(m, 1), w, w))
        x = normal(gen, 33, 64, dtype=dtype).requires_grad_(True)
        w.requires_grad_(True)
        x2, w2 = x.detach().clone().requires_grad_(True), w.detach().clone().requires_grad_(True)
        dy = normal(gen, 33, 64, dtype=dtype)
        got = torch.autograd.grad(linear(x, w, residual=x, activation="tanh"), (x, w), dy)
        r2 = x.detach().clone().requires_grad_(True)
        dx, dw, dr = torch.autograd.grad(linear(x2, w2, residual=r2, activation="tanh"), (x2, w2, r2), dy)
        assert torch.equal(got[0], dx + dr) and torch.equal(got[1], dw)
        got = torch.autograd.grad(gated_linear(x, w, w), w, dy)[0]
        wa, wb = (w.detach().clone().requires_grad_(True) for _ in range(2))
        assert torch.equal(got, sum(torch.autograd.grad(gated_linear(x, wa, wb), (wa, wb), dy)))


def test_offsets_beyond_32_bits():
    """Activations and outputs of more than 2^32 elements: everything is zero but the last rows, whose results are those of these rows
    alone (cut along the contraction in another way: to rounding, not to the bit)."""
    from volterra_vae_amd.dense_ops import linear_backward, linear_forward
    gen = torch.Generator().manual_seed(1)
    for dtype, m, k in ((torch.bfloat16, (1 << 21) + 77, 2056), (torch.float32, (1 << 20) + 99, 4104), (torch.float16, (1 << 21) + 5, 2051)):
        w = normal(gen, 24, k, scale=k ** -0.5, dtype=dtype)
        x = torch.zeros((m, k), dtype=dtype, device=dev())
        tail = normal(gen, 300, k, dtype=dtype)
        x[-300:] = tail
        y = linear_forward(x, w)[0]
        ref = tail.double() @ w.double().t()
        near(y[-300:], ref, u(dtype) * ref.abs() + 8 * EPS32 * steps(k, dtype) ** 0.5 * s2(tail.double(), w.double()) + 1e-30, "y")
        assert float(y[:-300].abs().max()) == 0.0
        dy = torch.zeros_like(y)
        dy[-300:] = normal(gen, 300, 24, dtype=dtype)
        dx, dw, db = linear_backward(dy, x, w)
        ref = dy[-300:].double().t() @ tail.double()
        near(dw, ref, u(dtype) * ref.abs() + 32 * EPS32 * steps(300, dtype) ** 0.5 * s2(dy[-300:].double().t(), tail.double().t()) + 1e-30, "dw")
        ref = dy[-300:].double() @ w.double()
        near(dx[-300:], ref, u(dtype) * ref.abs() + 32 * EPS32 * steps(24, dtype) ** 0.5 * s2(dy[-300:].double(), w.double().t()) + 1e-30, "dx")
        assert float(dx[:-300].abs().max()) == 0.0
        del x, y, dy, dx
    # an output beyond 2^32 elements
    x, w = normal(gen, (1 << 20) + 33, 8, dtype=torch.bfloat16), normal(gen, 4104, 8, dtype=torch.bfloat16)
    y = linear_forward(x, w)[0]
    ref = x[-2000:].double() @ w.double().t()
    assert y.numel() > 1 << 32
    near(y[-2000:], ref, u(y.dtype) * ref.abs() + 8 * EPS32 * steps(8, y.dtype) ** 0.5 * s2(x[-2000:].double(), w.double()), "y")


def test_no_rows_give_empty_outputs_and_zero_parameter_gradients():
    from volterra_vae_amd.dense_ops import gated_linear, linear
    for dtype in DTYPES:
        x = torch.empty((0, 12), dtype=dtype, device=dev(), requires_grad=True)
        w, wu = (torch.randn(7, 12, device=dev()).to(dtype).requires_grad_(True) for _ in range(2))
        b = torch.randn(7, device=dev()).to(dtype).requires_grad_(True)
        for y, leaves in ((linear(x, w, b, activation="silu"), (x, w, b)), (linear(x, w, b), (x, w, b)),
                          (gated_linear(x, w, wu, b, None), (x, w, wu, b))):
            assert y.shape == (0, 7)
            for g, leaf in zip(torch.autograd.grad(y, leaves, torch.empty_like(y)), leaves):
                assert g.shape == leaf.shape and float(g.abs().sum()) == 0.0


def test_what_lies_beside_the_outputs_rows_and_the_inputs_is_left_alone():
    """NaN around strided inputs never reaches an output, and a result of few rows writes nothing behind them."""
    from volterra_vae_amd import _lib
    from volterra_vae_amd.dense_ops import _dense, linear_backward, linear_forward
    gen = torch.Generator().manual_seed(4)
    for dtype in DTYPES:
        for m, k, n in ((3, 50, 40), (70, 50, 40), (130, 64, 72)):
            buf = torch.full((m + 4, k + 24), float("nan"), dtype=dtype, device=dev())
            x = buf[2:2 + m, 8:8 + k]
            x.copy_(normal(gen, m, k, dtype=dtype))
            wbuf = torch.full((n + 2, k + 8), float("nan"), dtype=dtype, device=dev())
            w = wbuf[1:1 + n, :k]
            w.copy_(normal(gen, n, k, scale=0.1, dtype=dtype))
            y, _ = linear_forward(x, w)
            assert torch.isfinite(y).all()
            assert all(torch.isfinite(t).all() for t in linear_backward(y, x, w))
            out = torch.full((m + 3, n), 5.0, dtype=dtype, device=dev())
            d = _dense(x, w, 0)
            ws = torch.empty(max(256, _lib.lib.v2vae_linear_workspace_bytes(d, 0)), dtype=torch.uint8, device=dev())
            _lib.check(_lib.lib.v2vae_linear_fwd(d, x.data_ptr(), w.data_ptr(), None, None, out.data_ptr(), None, ws.data_ptr(),
                                                 torch.cuda.current_stream().cuda_stream))
            assert torch.equal(out[:m], y) and bool((out[m:] == 5.0).all())


def test_extreme_pre_activations_have_finite_gradients():
    from volterra_vae_amd.dense_ops import gated_linear, linear
    for dtype in DTYPES:
        x = torch.tensor([[-300.0], [-90.0], [-20.0], [0.0], [20.0], [90.0], [300.0]] * 5, device=dev()).to(dtype).requires_grad_(True)
        w = torch.ones((3, 1), dtype=dtype, device=dev(), requires_grad=True)
        for act in ("silu", "gelu", "tanh", "relu"):
            y = linear(x, w, activation=act)
            ref = act64(act, x.detach().double() @ w.detach().double().t())
            assert torch.allclose(y.double(), ref, rtol=2 * u(dtype) + 1e-6, atol=1e-6)
            for g in torch.autograd.grad(y, (x, w), torch.ones_like(y)):
                assert torch.isfinite(g).all()
            h = gated_linear(x, w, w, activation=act)
            X, W = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
            H = act64(act, X @ W.t()) * (X @ W.t())
            for g, r in zip(torch.autograd.grad(h, (x, w), torch.ones_like(h)), torch.autograd.grad(H, (X, W), torch.ones_like(H))):
                # dw sums 300 * 300 over five rows: beyond float16's 65504, inf there and only there
                assert not torch.isnan(g).any() and bool((torch.isfinite(g) | (r.abs() > torch.finfo(dtype).max)).all())


def test_calls_on_another_stream():
    from volterra_vae_amd.dense_ops import gated_linear, linear
    x, wg, wu, bg, bu, dh = gated_case(300, 128, 160, torch.bfloat16, True, "plain", 8)
    want = linear(gated_linear(x, wg, wu, bg, bu), wg.t().contiguous())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear(gated_linear(x, wg, wu, bg, bu), wg.t().contiguous())
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_a_captured_block_replays_with_new_inputs():
    """Forward and explicit backward of linear(gated_linear(x)) in one HIP graph, replayed on changing inputs with eager calls of the
    same operators in between; every replay against the eager result."""
    from volterra_vae_amd.dense_ops import gated_backward, gated_forward, linear_backward, linear_forward
    for dtype, m in ((torch.float32, 200), (torch.bfloat16, 2000), (torch.float16, 4)):
        x, wg, wu, bg, bu, _ = gated_case(m, 96, 64, dtype, True, "plain", 9)
        wd, dy = wg.t().contiguous(), torch.ones((m, 96), dtype=dtype, device=dev())

        def block():
            h, gu = gated_forward(x, wg, wu, bg, bu, keep=True)
            y, z = linear_forward(h, wd, residual=x, activation="tanh", keep=True)
            dh, dwd, _ = linear_backward(dy, h, wd, z, activation="tanh", need=(True, True, False))
            return [y, dwd, *gated_backward(dh, x, wg, wu, gu)]

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = block()
        for r in range(4):
            x.copy_(x.roll(1, 0) * 0.9 + 0.01 * r)
            eager = [t.clone() for t in block()]
            graph.replay()
            torch.cuda.synchronize()
            for p, q in zip(captured, eager):
                assert torch.equal(p, q)


def test_every_tile_width_of_the_float32_product():
    """Column counts for which tiles of 64, 96, 128 and 160 columns are chosen, in both directions of a layer."""
    from volterra_vae_amd.dense_ops import linear_backward, linear_forward
    for k, n in ((40, 20), (96, 70), (130, 128), (150, 300), (161, 95), (300, 33)):
        x, w, b, r, dy = linear_case(66000, k, n, torch.float32, "silu", True, True, "odd" if k % 2 else "plain", k)
        y, z = linear_forward(x, w, b, residual=r, activation="silu", keep=True)
        check_linear(x, w, b, r, dy, "silu", y, linear_backward(dy, x, w, z, activation="silu"), torch.float32)


def test_refusals():
    from volterra_vae_amd._lib import V2VAEError
    from volterra_vae_amd.dense_ops import gated_backward, gated_forward, gated_linear, linear, linear_backward, linear_forward
    x, w, b = (torch.zeros(*s, device=dev()) for s in ((6, 5), (4, 5), (4,)))
    neg = torch.zeros(6, 1, dtype=torch.complex64, device=dev()).conj().imag
    assert neg.is_neg()
    for match, args, kw in (
            ("weight is torch.bfloat16", (x, w.bfloat16()), {}),
            ("weight: 4 columns", (x, w[:, :4]), {}),
            ("weight must have 2 dim", (x, w[0]), {}),
            ("weight must have unit stride", (x, torch.zeros(4, 10, device=dev())[:, ::2]), {}),
            ("x must have unit stride", (torch.zeros(5, 6, device=dev()).t(), w), {}),
            ("weight: empty", (x, w[:0]), {}),
            ("bias: 3 values", (x, w, b[:3]), {}),
            ("bias is torch.float16", (x, w, b.half()), {}),
            ("bias must have unit stride", (x, w, torch.zeros(1, device=dev()).expand(4)), {}),
            ("residual: expected", (x, w, b), dict(residual=torch.zeros(6, 5, device=dev()))),
            ("negation that is not carried out", (neg, w[:, :1]), {}),
            ("negation that is not carried out", (x[:, :1], neg[:4]), {}),
            ("weight must be|weight is on|weight must live", (x, w.cpu()), {})):
        with pytest.raises((ValueError, RuntimeError), match=match):
            linear(*args, **kw)
    with pytest.raises(NotImplementedError, match="float32, bfloat16 or float16"):
        linear(x.double(), w.double())
    with pytest.raises(ValueError, match="weight_up: expected"):
        gated_linear(x, w, w[:3])
    with pytest.raises(ValueError, match="bias_up: 3 values"):
        gated_linear(x, w, w, b, b[:3])
    wide = torch.empty_strided((2, 5), ((1 << 22) + 1, 1), device=dev())
    with pytest.raises(V2VAEError):
        linear(wide, w)
    with pytest.raises(V2VAEError):
        linear_backward(torch.zeros(2, 4, device=dev()), wide, w)
    y, z = linear_forward(x, w, b, activation="silu", keep=True)
    for match, args in (("z: the pre-activations", (y, x, w)), ("kept pre-activations is", (y, x, w, z.half())),
                        ("expected a contiguous", (y, x, w, z[:5])), ("expected a contiguous", (y, x, w, torch.zeros(6, 8, device=dev())[:, ::2][:, :4])),
                        ("dy: expected", (y[:5], x, w, z)), ("dy is", (y.half(), x, w, z))):
        with pytest.raises(ValueError, match=match + "|unit stride"):
            linear_backward(*args, activation="silu")
    h, gu = gated_forward(x, w, w, keep=True)
    with pytest.raises(ValueError, match="expected a contiguous"):
        gated_backward(h, x, w, w, gu[:, :5])
    with pytest.raises(ValueError, match="dh: expected"):
        gated_backward(h[:, :3], x, w, w, gu)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_every_choice_of_gradients_gives_the_same_ones(dtype):
    from volterra_vae_amd.dense_ops import gated_backward, gated_forward, linear_backward, linear_forward
    x, w, b, r, dy = linear_case(70, 33, 45, dtype, "silu", True, True, "odd", 3)
    _, z = linear_forward(x, w, b, activation="silu", keep=True)
    full = linear_backward(dy, x, w, z, activation="silu")
    plain = linear_backward(dy, x, w)
    for i in range(8):
        need = [bool(i >> q & 1) for q in range(3)]
        for every, some in ((full, linear_backward(dy, x, w, z, activation="silu", need=need)), (plain, linear_backward(dy, x, w, need=need))):
            for n, p, q in zip(need, every, some):
                assert torch.equal(p, q) if n else q is None
    x, wg, wu, bg, bu, dh = gated_case(70, 33, 45, dtype, True, "odd", 3)
    _, gu = gated_forward(x, wg, wu, bg, bu, keep=True)
    full = gated_backward(dh, x, wg, wu, gu)
    for i in range(32):
        need = [bool(i >> q & 1) for q in range(5)]
        for n, p, q in zip(need, full, gated_backward(dh, x, wg, wu, gu, need=need)):
            assert torch.equal(p, q) if n else q is None


def test_few_float32_rows_of_long_and_few_weights():
    """The contraction in parts: every number of parts that the rule gives, with and without a rest."""
    from volterra_vae_amd.dense_ops import gated_forward, linear_forward
    for m, k, n in ((1, 3200, 16), (9, 8165, 504), (13, 6696, 876), (32, 4096, 33), (17, 20500, 5), (3, 40000, 100), (5, 22401, 9), (2, 3199, 700)):
        x, w, b, r, dy = linear_case(m, k, n, torch.float32, "silu", True, True, "odd", m + k)
        y, z = linear_forward(x, w, b, residual=r, activation="silu", keep=True)
        check_linear(x, w, b, r, dy, "silu", y, None, torch.float32)
        near(z, x.double() @ w.double().t() + b.double(), 8 * EPS32 * steps(k, torch.float32) ** 0.5 * s2(x.double(), w.double())
             + 16 * EPS32 * b.double().abs() + 1e-30, "z")
        x, wg, wu, bg, bu, dh = gated_case(m, k, n, torch.float32, True, "odd", m + k)
        h, gu = gated_forward(x, wg, wu, bg, bu, keep=True)
        check_gated(x, wg, wu, bg, bu, dh, "silu", h, None, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_narrow_layers_of_many_rows(dtype):
    """Few inputs, few outputs or both, at aligned and at odd widths, each with its gradients."""
    from volterra_vae_amd.dense_ops import gated_backward, gated_forward, linear_backward, linear_forward
    for m, k, n in ((5000, 40, 24), (3001, 64, 64), (20001, 25, 603), (20001, 603, 25), (9001, 9, 33), (4097, 200, 8), (2500, 8, 1000)):
        x, w, b, r, dy = linear_case(m, k, n, dtype, "silu", True, True, "odd" if k % 2 else "plain", k + n)
        y, z = linear_forward(x, w, b, residual=r, activation="silu", keep=True)
        check_linear(x, w, b, r, dy, "silu", y, linear_backward(dy, x, w, z, activation="silu"), dtype)
        x, wg, wu, bg, bu, dh = gated_case(m, k, n, dtype, True, "odd" if k % 2 else "plain", k + n)
        h, gu = gated_forward(x, wg, wu, bg, bu, keep=True)
        check_gated(x, wg, wu, bg, bu, dh, "silu", h, gated_backward(dh, x, wg, wu, gu), dtype)


@pytest.mark.parametrize("m,k,n", [(300, 1024, 96), (500, 1024, 256), (1024, 2048, 512), (4096, 2048, 1000)], ids=lambda v: str(v))
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_one_weight_of_a_gated_block(dtype, m, k, n):
    """The other weight frozen, at sizes where one gradient alone has fewer tiles than the chip has room for: the same bits as of both
    gradients, and nothing written behind the workspace that was asked for."""
    from volterra_vae_amd import _lib
    from volterra_vae_amd.dense_ops import _dense, gated_backward, gated_forward, gated_linear
    x, wg, wu, bg, bu, dh = gated_case(m, k, n, dtype, True, "plain", m)
    h, gu = gated_forward(x, wg, wu, bg, bu, keep=True)
    full = gated_backward(dh, x, wg, wu, gu)
    check_gated(x, wg, wu, bg, bu, dh, "silu", h, full, dtype)
    for i in (1, 2):
        leaves = [t.clone().requires_grad_(j in (0, i)) for j, t in enumerate((x, wg, wu, bg, bu))]
        gx, gw = torch.autograd.grad(gated_linear(*leaves), (leaves[0], leaves[i]), dh)
        assert torch.equal(gx, full[0]) and torch.equal(gw, full[i])
        d = _dense(x, wg, 2, w2=wu, dy=dh)
        size = _lib.lib.v2vae_gated_workspace_bytes(d, 1)
        behind = 2 * n * k * 4 * 4   # more than four parts of two gradients would take
        ws = torch.full((size + behind,), 0x5A, dtype=torch.uint8, device=dev())
        out = torch.empty_like(wg)
        _lib.check(_lib.lib.v2vae_gated_bwd(d, x.data_ptr(), wg.data_ptr(), wu.data_ptr(), gu.data_ptr(), dh.data_ptr(), None,
                                            out.data_ptr() if i == 1 else None, out.data_ptr() if i == 2 else None, None, None, ws.data_ptr(),
                                            torch.cuda.current_stream().cuda_stream))
        assert torch.equal(out, full[i]) and bool((ws[size:] == 0x5A).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16", "f16"])
def test_layers_whose_tensors_are_kept_on_the_host_between_the_passes(dtype):
    """save_on_cpu gives strided rows back contiguous: gradients within the same bounds."""
    from volterra_vae_amd.dense_ops import gated_linear, linear
    x, w, b, r, dy = linear_case(70, 72, 56, dtype, "silu", True, True, "odd", 4)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    with torch.autograd.graph.save_on_cpu():
        y = linear(*leaves, residual=r, activation="silu")
    check_linear(x, w, b, r, dy, "silu", y.detach(), torch.autograd.grad(y, leaves, dy), dtype)
    x, wg, wu, bg, bu, dh = gated_case(70, 72, 56, dtype, True, "odd", 4)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, bg, bu)]
    with torch.autograd.graph.save_on_cpu():
        h = gated_linear(*leaves)
    check_gated(x, wg, wu, bg, bu, dh, "silu", h.detach(), torch.autograd.grad(h, leaves, dh), dtype)


@pytest.mark.parametrize("act", ["tanh", "silu", "gelu"])
def test_slopes_keep_their_relative_accuracy_in_the_tails(act):
    """The bias gradient of a layer of one row is act'(z) itself, z = the kept pre-activation.  In units of 2^-24 of the value: tanh' is
    1 - t^2 up to 0.55 (t^2 <= 0.25: below 2), then 4 e / (1 + e)^2 with e within 3, the reciprocal within 2 and there twice, three products:
    10.  silu' = s + z e s^2 and gelu' = Phi + z phi are sums of two terms, each of an exponential within 3 and some five factors and
    products (Phi: a polynomial whose terms add up to 2.5 times its value, ten steps of half a unit: 13): 16 of both terms'
    magnitudes.  16 are allowed to all; tanh up to where e = exp(-2 |z|) is the smallest normal number."""
    from volterra_vae_amd.dense_ops import linear_backward

    def slopes(z):
        z = z[None].to(dev())
        x, w, dy = torch.zeros(1, 1, device=dev()), torch.zeros(z.shape[1], 1, device=dev()), torch.ones_like(z)
        return linear_backward(dy, x, w, z, activation=act, need=(False, False, True))[2].double()

    z = torch.cat((torch.linspace(0.0, 3.0, 3001), torch.linspace(3.0, 12.0, 9001), torch.linspace(12.0, 43.0, 3101)))
    z = torch.cat((z, -z))
    z = z[z.abs() <= {"tanh": 43.0, "silu": 40.0, "gelu": 12.0}[act]]
    Z = z.double().to(dev())
    if act == "tanh":
        terms = [torch.cosh(Z) ** -2]
    elif act == "silu":
        s = torch.sigmoid(Z)
        terms = [s, Z * s * torch.sigmoid(-Z)]
    else:
        terms = [0.5 * torch.erfc(-Z / 2 ** 0.5), Z * torch.exp(-0.5 * Z * Z) / (2 * torch.pi) ** 0.5]
    err, size = (slopes(z) - sum(terms)).abs(), sum(t.abs() for t in terms)
    assert bool((err <= 16 * EPS32 * size).all()), float((err / size).max() / EPS32)
    # far out: 0 on the left, 0 (tanh) or 1 on the right, and a NaN stays one.  silu' is held at its value at -80, which is
    # s (1 - 80 e s) = -79 exp(-80) = -79 * 1.8049e-35 = -1.426e-33.
    far = slopes(torch.tensor([-90.0, -1e30, -3e38, -float("inf"), 90.0, 1e30, 3e38, float("inf"), float("nan")])).cpu()
    assert far[:4].abs().max() < 1.43e-33 and bool((far[4:8] == (0.0 if act == "tanh" else 1.0)).all()) and bool(torch.isnan(far[8]))


def test_a_layer_beside_a_very_wide_one():
    """The gradient of a piece of a concatenation more than 2^22 wide arrives with that row stride."""
    from volterra_vae_amd.dense_ops import gated_linear, linear
    for dtype in DTYPES:
        x, w, b, r, dy = linear_case(40, 50, 24, dtype, "silu", True, False, "plain", 6)
        wide = torch.ones((40, (1 << 22) + 8), dtype=dtype, device=dev())
        for f in (lambda *a: linear(*a, activation="silu"), lambda x, w, b: gated_linear(x, w, w, b, b)):
            leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
            beside = torch.cat((f(*leaves), wide), 1)
            factor = torch.zeros_like(beside)
            factor[:, :24] = dy
            got = torch.autograd.grad(beside, leaves, factor)
            assert all(torch.equal(p, q) for p, q in zip(got, torch.autograd.grad(f(*leaves), leaves, dy)))
