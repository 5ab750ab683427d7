"""The dense layers and the distillation loss where a dispatch mode is at work: what a trace records is the operators, not the empty
outputs that their kernels would fill.  Every comparison is with the eager call, to the bit: the same kernels run."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def inputs(dtype, seed, m=70, k=48, n=33):
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen).to(dtype).cuda()  # noqa: E731
    x, w, u, b, d = normal(m, k), normal(n, k) * 0.2, normal(n, k) * 0.2, normal(n), normal(k, n) * 0.2
    t, i = normal(m, 5), torch.argsort(torch.rand((m, k), generator=gen), 1)[:, :5].cuda()
    return x, w, u, b, d, t, i, torch.rand(m, generator=gen).cuda()


def training_pass(x, w, u, b, d, t, i, v):
    from volterra_vae_amd.dense_ops import gated_linear, linear, topk_distillation
    leaves = [a.detach().requires_grad_(True) for a in (x, w, u, b, d)]
    y = linear(gated_linear(*leaves[:4]), leaves[4], residual=leaves[0], activation="tanh")
    loss = topk_distillation(y, t, i, temperature=2.0)
    return (loss.detach(), *torch.autograd.grad(loss, leaves, v))


def registered_pass(x, w, u, b, d, t, i, v):
    leaves = [a.detach().requires_grad_(True) for a in (x, w, u, b, d)]
    y = torch.ops.v2vae.linear(torch.ops.v2vae.gated_linear(*leaves[:4]), leaves[4], residual=leaves[0], activation="tanh")
    loss = torch.ops.v2vae.topk_distillation(y, t, i, temperature=2.0)
    return (loss.detach(), *torch.autograd.grad(loss, leaves, v))


@pytest.mark.parametrize("mode", ["real", "fake"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_a_traced_training_pass_computes_for_new_inputs(dtype, mode):
    from torch.fx.experimental.proxy_tensor import make_fx
    for f in (training_pass, registered_pass):
        graph = make_fx(f, tracing_mode=mode)(*inputs(dtype, 1))
        assert all(f"v2vae.{name}" in graph.code for name in ("linear_forward", "linear_backward", "gated_forward", "gated_backward",
                                                              "distillation_forward", "distillation_backward")), graph.code
        for seed in (2, 3):
            new = inputs(dtype, seed)
            for got, want in zip(graph(*new), f(*new), strict=True):
                assert torch.equal(got, want)


def test_schema_shapes_and_registration_of_the_passes():
    from volterra_vae_amd.dense_ops import gated_forward, linear_forward
    for dtype in (torch.float32, torch.bfloat16):
        x, w, u, b, d, t, i, v = inputs(dtype, 4)
        ops = torch.ops.v2vae
        tests = ("test_schema", "test_faketensor")
        y, z = linear_forward(x, w, b, activation="silu", keep=True)
        h, gu = gated_forward(x, w, u, keep=True)
        loss, stats = ops.distillation_forward(x, t, i, 1.5, True)
        for op, args in ((ops.linear_forward, (x, w, b, None, "silu", True)), (ops.linear_forward, (x, w, None, y, "none", False)),
                         (ops.linear_backward, (y, x, w, z, "silu", [True, True, True])), (ops.linear_backward, (y, x, w, None, "none", [False, True, False])),
                         (ops.gated_forward, (x, w, u, b, b, "gelu", True)), (ops.gated_forward, (x, w, u, None, None, "silu", False)),
                         (ops.gated_backward, (h, x, w, u, gu, "silu", [True, True, False, False, True])),
                         (ops.distillation_forward, (x, t, i, 1.5, True)), (ops.distillation_forward, (x, t, i, 1.5, False)),
                         (ops.distillation_backward, (v, x, t, i, stats, 1.5)), (ops.distillation_step, (x, t, i, v, 1.5)),
                         (ops.linear, (x, w, b)), (ops.gated_linear, (x, w, u)), (ops.topk_distillation, (x, t, i))):
            torch.library.opcheck(op.default, args, test_utils=tests)


def test_modes_that_only_watch_change_nothing():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    args = inputs(torch.float32, 5)
    want = training_pass(*args)
    with Watch() as outer, Watch() as inner:
        got = training_pass(*args)
    assert all(torch.equal(p, q) for p, q in zip(got, want, strict=True))
    for mode in (outer, inner):
        assert sum("v2vae" in name for name in mode.seen) == 6
