"""Refusals of the dense layers and the distillation loss, on the host: nothing is launched."""
import ctypes as C

import pytest
import torch

from volterra_vae_amd import _lib, dense_ops

P = 0x1000  # an aligned address that no call may reach


def dense(**over):
    d = dict(dtype=0, activation=0, rows=64, in_=50, out=30, ld_x=50, ld_w=50, ld_w2=50, ld_res=30, ld_dy=30)
    d.update(over)
    return _lib.Dense(*[d[f] for f, _ in _lib.Dense._fields_])


def distill(**over):
    d = dict(dtype=0, teacher_dtype=0, index_bits=32, k=4, rows=8, vocab=100, ld_logits=100, ld_teacher=4, ld_index=4, temperature=1.0, reserved=0)
    d.update(over)
    return _lib.Distill(*[d[f] for f, _ in _lib.Distill._fields_])


BAD = [dict(dtype=3), dict(dtype=-1), dict(activation=5), dict(activation=-1), dict(rows=-1), dict(in_=0), dict(out=0), dict(ld_x=-1),
       dict(ld_w=-4)]


@pytest.mark.parametrize("over", BAD, ids=str)
def test_bad_descriptions_are_refused(over):
    d = dense(**over)
    assert _lib.lib.v2vae_linear_fwd(d, P, P, None, None, P, None, P, None) == _lib.EINVAL
    assert _lib.lib.v2vae_linear_bwd(d, P, P, P, P, P, P, P, P, None) == _lib.EINVAL
    assert _lib.lib.v2vae_gated_fwd(d, P, P, P, None, None, P, None, P, None) == _lib.EINVAL
    assert _lib.lib.v2vae_gated_bwd(d, P, P, P, P, P, P, P, P, P, P, P, None) == _lib.EINVAL
    for back in (0, 1):
        assert _lib.lib.v2vae_linear_workspace_bytes(d, back) == 0 and _lib.lib.v2vae_gated_workspace_bytes(d, back) == 0


def test_sizes_beyond_the_limits_are_refused():
    for over in (dict(rows=(1 << 30) + 1), dict(in_=(1 << 22) + 1), dict(out=1 << 31), dict(rows=1 << 30, out=1 << 22), dict(rows=1 << 30), dict(rows=1 << 26, out=1024, ld_res=1024),
                 dict(ld_x=(1 << 22) + 1), dict(ld_w=(1 << 22) + 1)):
        assert _lib.lib.v2vae_linear_fwd(dense(**over), P, P, None, None, P, None, P, None) == _lib.ESIZE
        assert _lib.lib.v2vae_linear_workspace_bytes(dense(**over), 1) == 0
    assert _lib.lib.v2vae_distill_fwd(distill(k=1025, ld_teacher=1025, ld_index=1025), P, P, P, P, None, None) == _lib.ESIZE
    assert _lib.lib.v2vae_distill_fwd(distill(rows=(1 << 30) + 1), P, P, P, P, None, None) == _lib.ESIZE
    # more rows than a launch has threads for
    assert _lib.lib.v2vae_distill_fwd(distill(rows=1 << 30), P, P, P, P, None, None) == _lib.ESIZE
    assert _lib.lib.v2vae_distill_fwd(distill(rows=1 << 23, vocab=20000, ld_logits=20000), P, P, P, P, None, None) == _lib.ESIZE


def test_missing_and_misaligned_pointers_are_refused():
    f = _lib.lib.v2vae_linear_fwd
    d = dense()
    for bad in ((None, P, None, None, P, None), (P, None, None, None, P, None), (P, P, None, None, None, None), (P + 2, P, None, None, P, None),
                (P, P, P + 1, None, P, None), (P, P, None, P + 2, P, None), (P, P, None, None, P, P + 2)):
        assert f(d, *bad, P, None) == _lib.EINVAL
    assert f(d, P, P, None, None, P, None, P + 8, None) == _lib.EINVAL          # the workspace is 256-byte aligned
    assert f(dense(ld_res=-1), P, P, None, P, P, None, P, None) == _lib.EINVAL
    b = _lib.lib.v2vae_linear_bwd
    assert b(d, P, P, None, None, P, P, P, P, None) == _lib.EINVAL               # no dy
    assert b(d, P, P, None, P, P, P, P, None, None) == _lib.EINVAL               # no workspace
    assert b(dense(activation=2), P, P, None, P, P, P, P, P, None) == _lib.EINVAL  # an activation without its pre-activations
    assert b(d, None, P, None, P, P, P, P, P, None) == _lib.EINVAL               # dw without x
    assert b(dense(ld_dy=-1), P, P, None, P, P, P, P, P, None) == _lib.EINVAL
    g = _lib.lib.v2vae_gated_bwd
    assert g(d, P, P, P, None, P, P, P, P, P, P, P, None) == _lib.EINVAL
    assert g(d, P, P, None, P, P, P, P, P, P, P, P, None) == _lib.EINVAL
    assert _lib.lib.v2vae_gated_fwd(d, P, P, None, None, None, P, None, P, None) == _lib.EINVAL
    assert f(None, P, P, None, None, P, None, P, None) == _lib.EINVAL


@pytest.mark.parametrize("over", [dict(dtype=3), dict(teacher_dtype=-1), dict(index_bits=16), dict(k=0), dict(rows=-1), dict(vocab=0),
                                  dict(ld_logits=99), dict(ld_teacher=3), dict(ld_index=3), dict(temperature=0.0),
                                  dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
                                  dict(temperature=9e-5), dict(temperature=2e4), dict(reserved=1)], ids=str)
def test_bad_distillations_are_refused(over):
    d = distill(**over)
    assert _lib.lib.v2vae_distill_fwd(d, P, P, P, P, None, None) == _lib.EINVAL
    assert _lib.lib.v2vae_distill_bwd(d, P, P, P, P, P, P, None) == _lib.EINVAL
    assert _lib.lib.v2vae_distill_step(d, P, P, P, P, P, P, None) == _lib.EINVAL


def test_distillation_pointers():
    d = distill()
    assert _lib.lib.v2vae_distill_fwd(d, P, P, P, None, None, None) == _lib.EINVAL
    assert _lib.lib.v2vae_distill_bwd(d, P, P, P, None, P, P, None) == _lib.EINVAL   # statistics of the forward pass
    assert _lib.lib.v2vae_distill_step(d, P, P, P, None, P, P, None) == _lib.EINVAL
    assert _lib.lib.v2vae_distill_fwd(d, P + 2, P, P, P, None, None) == _lib.EINVAL
    assert _lib.lib.v2vae_distill_fwd(distill(index_bits=64), P, P, P + 4, P, None, None) == _lib.EINVAL


def test_no_rows_launch_nothing():
    assert _lib.lib.v2vae_linear_fwd(dense(rows=0), None, None, None, None, None, None, None, None) == _lib.OK
    assert _lib.lib.v2vae_gated_fwd(dense(rows=0), None, None, None, None, None, None, None, None, None) == _lib.OK
    assert _lib.lib.v2vae_distill_step(distill(rows=0), None, None, None, None, None, None, None) == _lib.OK


def test_the_python_layer_refuses_what_is_not_on_a_gpu_or_not_a_tensor():
    x, w = torch.zeros(4, 3), torch.zeros(5, 3)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        dense_ops.linear(x, w)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        dense_ops.gated_linear(x, w, w)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        dense_ops.topk_distillation(x, torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="none of none, relu, silu, gelu, tanh"):
        dense_ops.linear(x, w, activation="selu")
    with pytest.raises(ValueError, match="x must be a tensor"):
        dense_ops.linear([[1.0]], w)
    with pytest.raises(ValueError, match="rows"):
        dense_ops.linear(x, w, residual=torch.zeros(3, 5))


def test_structures_match_the_header():
    """Field names and order of the two argument blocks, and their sizes under the C rules."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "v2vae_hip.h")).read()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    for name, struct in (("v2vae_dense", _lib.Dense), ("v2vae_distill", _lib.Distill)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
        declared = re.findall(r"(\w+)\s+(\w+);", body)
        kinds = {"int32_t": C.c_int32, "int64_t": C.c_int64, "float": C.c_float}
        assert [(n.rstrip("_"), t) for n, t in struct._fields_] == [(n, kinds[k]) for k, n in declared]


def without_launches(monkeypatch):
    """CPU tensors pass the checks and what would be launched is listed: (entry point, its arguments)."""
    calls = []
    monkeypatch.setattr(dense_ops, "_enqueue", lambda fn, name, t, *args: calls.append((name, args)))
    monkeypatch.setattr(dense_ops, "_check_tensor", lambda *args, **kw: None)
    monkeypatch.setattr(dense_ops, "_workspace", lambda gated, backward, d, x: torch.empty(256, dtype=torch.uint8))
    return calls


def test_the_backward_passes_describe_the_tensors_that_saved_tensor_hooks_give_back(monkeypatch):
    """Hooks that move saved tensors elsewhere give strided ones back contiguous: the row strides of the backward call are theirs, not
    those of the forward call."""
    calls = without_launches(monkeypatch)
    z = torch.zeros(6, 20)[:, 3:12].requires_grad_(True)
    t, i = torch.zeros(6, 8)[:, 2:5], torch.zeros(6, 7, dtype=torch.int32)[:, 1:4]
    x, w = torch.zeros(40, 20)[:, 3:12].requires_grad_(True), torch.zeros(5, 16)[:, :9].requires_grad_(True)
    held = []   # what the hooks give back lives on: an address then names one tensor

    def unpack(t):
        held.append(t.contiguous())
        return held[-1]

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        outs = [dense_ops.topk_distillation(z, t, i), dense_ops.linear(x, w, activation="silu"), dense_ops.gated_linear(x, w, w)]
    for out, leaf in zip(outs, (z, x, x)):
        torch.autograd.grad(out, leaf, torch.ones_like(out))
    by_name = {name: args for name, args in calls}
    d = by_name["v2vae_distill_fwd"][0]
    assert (d.ld_logits, d.ld_teacher, d.ld_index) == (20, 8, 7)
    d, *pointers = by_name["v2vae_distill_bwd"]
    addresses = {a.data_ptr() for a in held}
    assert pointers[0] in addresses and (d.ld_logits, d.ld_teacher, d.ld_index) == (9, 3, 3)
    for name in ("v2vae_linear", "v2vae_gated"):
        d = by_name[name + "_fwd"][0]
        assert (d.ld_x, d.ld_w) == (20, 16)
        d, *pointers = by_name[name + "_bwd"]
        assert pointers[0] in addresses and (d.ld_x, d.ld_w) == (9, 9)


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A dual tensor in any place raises, with and without a graph, in the differentiable and in the explicit passes; without tangents
    the same calls pass inside a dual level."""
    from torch.autograd import forward_ad as fw
    calls = without_launches(monkeypatch)
    x, w, b, r = torch.zeros(6, 5), torch.zeros(4, 5), torch.zeros(4), torch.zeros(6, 4)
    z, t, i = torch.zeros(6, 9), torch.zeros(6, 3), torch.zeros(6, 3, dtype=torch.int32)
    gu, v = torch.zeros(2, 6, 4), torch.zeros(6)
    passes = [(lambda x, w, b, r: dense_ops.linear(x, w, b, residual=r), (x, w, b, r)),
              (lambda x, w, u, b, c: dense_ops.gated_linear(x, w, u, b, c), (x, w, w, b, b)),
              (lambda z, t: dense_ops.topk_distillation(z, t, i), (z, t)),
              (lambda z, t, v: dense_ops.topk_distillation_step(z, t, i, v), (z, t, v)),
              (lambda x, w, b, r: dense_ops.linear_forward(x, w, b, residual=r), (x, w, b, r)),
              (lambda x, w, u: dense_ops.gated_forward(x, w, u), (x, w, w)),
              (lambda d, x, w, z: dense_ops.linear_backward(d, x, w, z, activation="silu"), (r, x, w, r)),
              (lambda d, x, w, u, g: dense_ops.gated_backward(d, x, w, u, g), (r, x, w, w, gu))]
    with fw.dual_level():
        for f, args in passes:
            f(*args)
            for place in range(len(args)):
                dual = [fw.make_dual(a.clone(), torch.ones_like(a)) if n == place else a for n, a in enumerate(args)]
                before = len(calls)
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*dual)
                assert len(calls) == before
        with pytest.raises(NotImplementedError):
            dense_ops.linear(fw.make_dual(x.clone().requires_grad_(), torch.ones_like(x)), w)
        for out, leaf in ((lambda a: dense_ops.linear(a, w), x), (lambda a: dense_ops.gated_linear(a, w, w), x),
                          (lambda a: dense_ops.topk_distillation(a, t, i), z)):
            leaf = leaf.clone().requires_grad_()
            y = out(leaf)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, leaf, fw.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_every_pass_enters_a_traced_graph_as_an_op():
    """Fake tensors through every pass: shapes and types of the results, and a graph whose nodes are the passes."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx

    def passes(x, w, u, b, t, i, v):
        h, gu = dense_ops.gated_forward(x, w, u, b, keep=True)
        y, z = dense_ops.linear_forward(h, w.t().contiguous(), residual=x, activation="tanh", keep=True)
        loss, dy = dense_ops.topk_distillation_step(y, t, i, v, temperature=2.0)
        dh, dw, db = dense_ops.linear_backward(dy, h, w.t().contiguous(), z, activation="tanh", need=(True, False, True))
        assert dw is None
        grads = dense_ops.gated_backward(dh, x, w, u, gu, need=(True, True, False, True, False))
        assert grads[2] is None and grads[4] is None
        plain = torch.ops.v2vae.linear(x, w, b), torch.ops.v2vae.gated_linear(x, w, u), torch.ops.v2vae.topk_distillation(x, t, i)
        return (y, z, gu, loss, dy, dh, db, grads[0], grads[1], grads[3], *plain)

    for dtype in (torch.float32, torch.bfloat16):
        with FakeTensorMode():
            new = lambda *shape, dt=dtype: torch.empty(shape, dtype=dt, device="cuda")  # noqa: E731
            args = (new(6, 8), new(4, 8), new(4, 8), new(4), new(6, 3), new(6, 3, dt=torch.int64), new(6, dt=torch.float32))
            out = passes(*args)
            f32 = torch.float32
            assert [(tuple(o.shape), o.dtype) for o in out] == [
                ((6, 8), dtype), ((6, 8), f32), ((2, 6, 4), f32), ((6,), f32), ((6, 8), dtype), ((6, 4), dtype), ((8,), dtype), ((6, 8), dtype),
                ((4, 8), dtype), ((4,), dtype), ((6, 4), dtype), ((6, 4), dtype), ((6,), f32)]
            code = make_fx(passes)(*args).code
        for name in ("gated_forward", "linear_forward", "distillation_step", "linear_backward", "gated_backward", "distillation_forward"):
            assert f"v2vae.{name}" in code, code


def test_a_gradient_whose_rows_lie_far_apart_is_taken_as_a_copy(monkeypatch):
    """Row strides beyond 2^22 are refused in what a caller lays out; the stride of an incoming gradient is not the caller's doing (the
    piece of a wide concatenation's gradient, say)."""
    calls = without_launches(monkeypatch)
    far = (1 << 22) + 8
    x, w = torch.zeros(2, 5).requires_grad_(True), torch.zeros(4, 5)
    for out, name in ((dense_ops.linear(x, w), "v2vae_linear_bwd"), (dense_ops.gated_linear(x, w, w), "v2vae_gated_bwd")):
        for stride, taken in ((far, 4), (1 << 22, 1 << 22)):
            dy = torch.zeros(2 * far)[:].as_strided((2, 4), (stride, 1))
            torch.autograd.grad(out, x, dy, retain_graph=True)
            assert calls[-1][0] == name and calls[-1][1][0].ld_dy == taken
