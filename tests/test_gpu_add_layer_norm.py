"""add_layer_norm against float64 on the CPU, at the widths, row counts, types and layouts where its kernels can go wrong.

Tolerances: the sum of two numbers and all that follows is fp32, rounded once to the result's type (half a step, `unit`).  With z of
size Z in a row, the mean is off by no more than (log2 of the lanes and eight more) 2^-24 Z, so xhat by some 32 roundings of
Z / deviation; the factors below are Z rstd (the largest of a row) times 2^-19.  A gradient's row sums add the same relative to
the sizes of what is added, column sums add rows one after the other: 2^-24 times the rows of a slab, below 2^-24 rows."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
IDS = {F32: "fp32", F16: "fp16", BF16: "bf16"}
UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 0.0, F16: 2.0 ** -25, BF16: 0.0}
CALC = 2.0 ** -19


def make(shape, x=F32, residual=F32, params=F32, affine=True, eps=1e-5, seed=0, mean=2.0):
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=gen)
    t = dict(x=normal(*shape).to(x), residual=None if residual is None else (normal(*shape) + mean).to(residual))
    wide = F32 if residual is None and x == F32 or F32 in (x, residual) else x
    t["norm"] = torch.nn.LayerNorm(shape[-1], eps=eps, elementwise_affine=affine)
    if affine:
        with torch.no_grad():
            t["norm"].weight.copy_(1 + 0.3 * normal(shape[-1]))
            t["norm"].bias.copy_(0.3 * normal(shape[-1]))
    t["norm"].to(params)
    t["grad"], t["grad_sum"] = normal(*shape).to(wide), normal(*shape).to(wide)
    return t


def reference(t, stream, out_type):
    """{name: (value, tolerance)}"""
    x, r = t["x"].double(), None if t["residual"] is None else t["residual"].double()
    wide = t["grad_sum"].dtype
    norm = t["norm"]
    width = x.shape[-1]
    rows = x.numel() // width
    one = torch.ones(width, dtype=torch.float64)
    w = one if norm.weight is None else norm.weight.detach().double()
    b = 0 * one if norm.bias is None else norm.bias.detach().double()
    z = x if r is None else x + r
    centred = z - z.mean(-1, keepdim=True)
    rstd = (centred.pow(2).mean(-1, keepdim=True) + norm.eps).rsqrt()
    xhat = centred * rstd
    off = CALC * z.abs().amax(-1, keepdim=True) * rstd              # of xhat
    round_to = lambda v, dtype: UNIT[dtype] * v.abs() + TINY[dtype]
    out = xhat * w + b
    found = {"out": (out, round_to(out, out_type) + off * w.abs() * (1 + xhat.abs()))}
    found["sum"] = (z, round_to(z, wide))
    g = t["grad"].double()
    around = t["grad_sum"].double() if stream else 0 * g
    a = g * w
    mean = lambda v: v.mean(-1, keepdim=True)
    dz = rstd * (a - mean(a) - xhat * mean(a * xhat))
    size = rstd * (a.abs() + mean(a.abs()) + xhat.abs() * mean((a * xhat).abs()))
    dz_off = CALC * (size + around.abs()) + off * rstd * (mean((a * xhat).abs()) + xhat.abs() * mean(a.abs())) + off * size
    dz = dz + around
    for name, tensor in (("grad_x", t["x"]), ("grad_residual", t["residual"])):
        if tensor is not None:
            found[name] = (dz, round_to(dz, tensor.dtype) + dz_off)
    if norm.weight is not None:
        flat = lambda v: v.reshape(-1, width).sum(0)
        dtype = norm.weight.dtype
        dw, db = flat(g * xhat), flat(g)
        found["grad_weight"] = (dw, round_to(dw, dtype) + flat(g.abs() * off) + 2.0 ** -24 * (rows + 64) * flat((g * xhat).abs()))
        found["grad_bias"] = (db, round_to(db, dtype) + 2.0 ** -24 * (rows + 64) * flat(g.abs()))
    return found


def close(got, want, what):
    value, tolerance = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape
    assert torch.isfinite(got).all(), f"{what}: not finite"
    beyond = (got - value).abs() - tolerance
    assert beyond.numel() == 0 or beyond.max() <= 0, f"{what}: {beyond.max():.3e} beyond tolerance, error {(got - value).abs().max():.3e}"


def check(t, stream=False, change=lambda v: v, autocast=None):
    from dcnv4_amd.functions import add_layer_norm
    norm = t["norm"].cuda()
    t = dict(t, norm=t["norm"])
    x = change(t["x"].cuda()).detach().requires_grad_()
    residual = None if t["residual"] is None else change(t["residual"].cuda()).detach().requires_grad_()
    with torch.autocast("cuda", dtype=autocast or F16, enabled=autocast is not None):
        got = add_layer_norm(x, residual, norm, return_sum=stream)
    outs = list(got) if stream else [got]
    wide = t["grad_sum"].dtype
    out_type = F32 if autocast is not None else wide
    assert outs[0].dtype == out_type and (not stream or outs[1].dtype == wide)
    sent = [change(t["grad"].cuda().to(out_type))] + ([change(t["grad_sum"].cuda())] if stream else [])
    wanted = {"grad_x": x, "grad_residual": residual, "grad_weight": norm.weight, "grad_bias": norm.bias}
    wanted = {name: leaf for name, leaf in wanted.items() if leaf is not None}
    grads = torch.autograd.grad(outs, list(wanted.values()), sent)
    t["norm"] = norm.cpu()
    want = reference(t, stream, out_type)
    close(outs[0], want["out"], "out")
    if stream:
        close(outs[1], want["sum"], "sum")
    for name, grad in zip(wanted, grads):
        assert grad.dtype == wanted[name].dtype
        close(grad, want[name], name)


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("width", (1, 2, 7, 8, 9, 31, 64, 100, 112, 256, 257, 511, 520, 1001, 2048, 2050, 4099, 8191, 8192))
def test_widths(width, dtype):
    check(make((2, 13, width), dtype, dtype, dtype, seed=width))


@pytest.mark.parametrize("dtype", (F32, F16), ids=IDS.get)
@pytest.mark.parametrize("rows,width", [(1, 256), (2, 64), (3, 8192), (777, 600), (20001, 24), (9000, 112), (4097, 257)])
def test_rows(rows, width, dtype):
    check(make((rows, width), dtype, dtype, dtype, seed=rows))


@pytest.mark.parametrize("dtype", (F32, F16), ids=IDS.get)
@pytest.mark.parametrize("rows,width", [(16384, 513), (16385, 515), (16385, 520), (16390, 1024), (16390, 1032)])
def test_many_rows_of_some_hundred_channels(rows, width, dtype):
    check(make((rows, width), dtype, dtype, dtype, seed=rows))


@pytest.mark.parametrize("stream", (False, True), ids=("post", "stream"))
@pytest.mark.parametrize("width", (96, 333))
@pytest.mark.parametrize("x,residual,params", [(F16, F32, F32), (F32, F16, F32), (BF16, F32, F32), (F32, BF16, BF16), (F16, F16, F32), (BF16, BF16, F32),
                                               (F16, None, F16), (F32, None, F32), (BF16, None, F32), (F16, F32, F16)],
                         ids=lambda t: IDS.get(t, "none"))
def test_mixed_types(x, residual, params, width, stream):
    check(make((37, width), x, residual, params, seed=5), stream=stream)


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("width", (64, 1001))
def test_the_sum_as_a_result(width, dtype):
    check(make((5, 60, width), dtype, dtype, dtype, seed=6), stream=True)


def test_no_parameters_and_one_of_two():
    check(make((40, 72), affine=False))
    t = make((40, 72), seed=3)
    t["norm"] = torch.nn.LayerNorm(72, bias=False)
    t["norm"].weight.data.uniform_(0.5, 1.5)
    check(t)


@pytest.mark.parametrize("dtype", (F32, F16), ids=IDS.get)
@pytest.mark.parametrize("width", (64, 75))
def test_layouts(width, dtype):
    shape = (3, 21, width)
    t = make(shape, dtype, dtype, dtype, seed=7)
    layouts = {
        "rows apart": lambda v: torch.cat((v, v[..., :5]), -1)[..., :width],
        "odd offset": lambda v: torch.cat((v.new_zeros(1), v.reshape(-1)))[1:].view(v.shape),
        "axes swapped": lambda v: v.transpose(0, 1).contiguous().transpose(0, 1),
        "channels not dense": lambda v: torch.stack((v, v), -1)[..., 0],
    }
    for change in layouts.values():
        check(t, change=change)
        check(t, change=change, stream=True)


def test_an_expanded_residual_gets_its_summed_gradient():
    from dcnv4_amd.functions import add_layer_norm
    t = make((4, 30, 64), seed=8)
    norm = t["norm"].cuda()
    one = t["residual"][:1].cuda().requires_grad_()
    x = t["x"].cuda().requires_grad_()
    out = add_layer_norm(x, one.expand(4, 30, 64), norm)
    gx, gr = torch.autograd.grad(out, (x, one), t["grad"].cuda())
    t["residual"] = t["residual"][:1].expand(4, 30, 64)
    t["norm"] = norm.cpu()
    want = reference(t, False, F32)
    close(out, want["out"], "out")
    close(gx, want["grad_x"], "grad_x")
    value, tolerance = want["grad_residual"]
    close(gr, (value.sum(0, keepdim=True), tolerance.sum(0, keepdim=True) + 2.0 ** -22 * value.abs().sum(0, keepdim=True)), "grad_residual")
    # and a residual that broadcasts by itself, which torch's operators add
    gx2, gr2 = torch.autograd.grad(add_layer_norm(x, one, norm.cuda()), (x, one), t["grad"].cuda())
    assert (gx2 - gx).abs().max() < 1e-4 and (gr2 - gr).abs().max() < 1e-4


def test_rows_far_from_zero_and_constant_rows():
    t = make((50, 384), mean=300.0, seed=9)
    check(t)
    t = make((8, 384), seed=9)
    t["x"][:] = 0.25
    t["residual"][:] = 0.5              # no deviation at all: eps alone
    check(t)


@pytest.mark.parametrize("amp", (F16, BF16), ids=IDS.get)
def test_under_autocast_the_result_is_fp32(amp):
    check(make((64, 256), amp, F32, F32, seed=10), autocast=amp)
    check(make((64, 256), amp, amp, F32, seed=10), autocast=amp)
    check(make((64, 255), amp, amp, F32, seed=10), autocast=amp, stream=True)


def test_empty():
    from dcnv4_amd.functions import add_layer_norm
    norm = torch.nn.LayerNorm(32).cuda()
    x = torch.zeros(0, 5, 32, device="cuda", requires_grad=True)
    out, total = add_layer_norm(x, x.detach(), norm, return_sum=True)
    assert out.shape == total.shape == x.shape
    gx, gw, gb = torch.autograd.grad((out, total), (x, norm.weight, norm.bias), (torch.zeros_like(out), torch.zeros_like(out)))
    assert gx.shape == x.shape and not gw.any() and not gb.any()


def test_only_the_gradients_that_are_asked_for_and_only_one_result_used():
    from dcnv4_amd.functions import add_layer_norm
    t = make((70, 130), F16, F32, F32, seed=11)
    norm, x, r = t["norm"].cuda(), t["x"].cuda().requires_grad_(), t["residual"].cuda().requires_grad_()
    g, gs = t["grad"].cuda(), t["grad_sum"].cuda()
    wanted = (x, r, norm.weight, norm.bias)
    whole = torch.autograd.grad(add_layer_norm(x, r, norm, return_sum=True), wanted, (g, gs))
    for i, leaf in enumerate(wanted):
        one, = torch.autograd.grad(add_layer_norm(x, r, norm, return_sum=True), leaf, (g, gs))
        assert torch.equal(one, whole[i])
    # the sum alone is an addition
    gx, gr, gw = torch.autograd.grad(add_layer_norm(x, r, norm, return_sum=True)[1], (x, r, norm.weight), gs, allow_unused=True)
    assert torch.equal(gx, gs.half()) and torch.equal(gr, gs) and (gw is None or not gw.any())
    # the result alone
    out, total = add_layer_norm(x, r, norm, return_sum=True)
    first = torch.autograd.grad(out, wanted, g)
    zero = torch.autograd.grad(add_layer_norm(x, r, norm, return_sum=True), wanted, (g, torch.zeros_like(gs)))
    assert all(torch.equal(a, b) for a, b in zip(first, zero))


def test_results_repeat_and_replay():
    from dcnv4_amd.functions import add_layer_norm
    t = make((3000, 112), F16, F16, F16, seed=12)
    norm, x, r, g = t["norm"].cuda(), t["x"].cuda().requires_grad_(), t["residual"].cuda().requires_grad_(), t["grad"].cuda()
    wanted = (x, r, norm.weight, norm.bias)
    step = lambda: (lambda o: (o.detach(), *torch.autograd.grad(o, wanted, g)))(add_layer_norm(x, r, norm))
    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (13, 14, 15):
        other = make((3000, 112), F16, F16, F16, seed=seed)
        with torch.no_grad():
            x.copy_(other["x"])
            r.copy_(other["residual"])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_the_functions_own_python_agrees():
    from dcnv4_amd.functions import add_layer_norm
    t = make((33, 48), F16, F32, F32, seed=16)
    norm, x, r = t["norm"].cuda(), t["x"].cuda().requires_grad_(), t["residual"].cuda().requires_grad_()
    g, gs = t["grad"].cuda(), t["grad_sum"].cuda()
    wanted = (x, r, norm.weight, norm.bias)

    class Watch(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Watch():
        watched = add_layer_norm(x, r, norm)
    plain = add_layer_norm(x, r, norm)
    assert torch.equal(watched, plain)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(watched, wanted, g), torch.autograd.grad(plain, wanted, g)))
    with Watch():
        watched = add_layer_norm(x, r, norm, return_sum=True)
    assert all(a.shape == b.shape and a.dtype == b.dtype for a, b in zip(torch.autograd.grad(watched, wanted, (g, gs)), wanted))


def test_calls_that_are_left_to_torch():
    from dcnv4_amd.functions import add_layer_norm
    norm = torch.nn.LayerNorm((4, 6)).cuda()
    x, r = torch.randn(3, 4, 6, device="cuda"), torch.randn(3, 4, 6, device="cuda")
    assert torch.equal(add_layer_norm(x, r, norm), norm(x + r))
    norm = torch.nn.LayerNorm(6).cuda().double()
    out, total = add_layer_norm(x.double(), r.double(), norm, return_sum=True)
    assert torch.equal(out, norm(x.double() + r.double())) and torch.equal(total, x.double() + r.double())
    norm = torch.nn.LayerNorm(9000).cuda()
    x = torch.randn(3, 9000, device="cuda")
    assert torch.equal(add_layer_norm(x, None, norm), norm(x))


def test_refusals_of_the_raw_function():
    from dcnv4_amd import ext
    x = torch.zeros(4, 32, device="cuda")
    for match, args in (("shape", (x, x[:2], None, None, 1e-5)), ("CUDA tensor", (x.cpu(), None, None, None, 1e-5)),
                        ("different 16-bit", (x.half(), x.bfloat16(), None, None, 1e-5)), ("expected", (x, None, x[0, :8], None, 1e-5)),
                        ("channels", (torch.zeros(1, 8200, device="cuda"), None, None, None, 1e-5)), ("dtype", (x.double(), None, None, None, 1e-5)),
                        ("different types", (x, None, x[0], x[0].half(), 1e-5))):
        with pytest.raises(RuntimeError, match=match):
            ext.add_layer_norm_forward(*args)
