"""What query_attention and add_layer_norm make of calls at the ends of what they take, and of what a program has put around them."""
import pytest
import torch

from oracle import query_attention as oracle_attention
from tests.test_gpu_query_attention import BF16, F16, F32, IDS, TINY, UNIT, close

pytestmark = pytest.mark.gpu


def test_heads_whose_rows_lie_too_far_apart_are_refused():
    from dcnv4_amd.functions import query_attention

    def refused(match, lq, lk, m, mk, d, dtype=F16, n=1):
        one = torch.zeros(1, 1, 1, d, dtype=dtype, device="cuda")      # expanded: refused before anything is allocated
        q, k = one.expand(n, lq, m, d), one.expand(n, lk, mk, d)
        with pytest.raises(RuntimeError, match=match):
            query_attention(q, k, k)

    refused("heads of the query.* 128 tokens .*31 - 1 bytes", 128, 1, 1 << 18, 1 << 18, 32)
    refused("heads of the query.* 256 tokens .*31 - 1 bytes", 5000, 1, 1 << 17, 1, 32)
    refused("heads of the key.* 128 tokens .*31 - 1 bytes", 1, 128, 1 << 18, 1 << 18, 32)
    refused("heads of the query.* 64 tokens .*31 - 1 bytes", 64, 1, 1 << 17, 1, 121)      # copied to 128 channels
    refused("heads of the query.* 256 tokens .*31 - 1 bytes", 256, 1, 1 << 16, 1, 32, F32)
    # workgroups of 64 columns, backward if not forward
    refused("24 - 1 pieces of 64", 65, 1, 8, 1, 128, n=1 << 20)


def test_the_most_heads_that_are_taken():
    from dcnv4_amd.functions import query_attention
    n, m, d = 128, (1 << 18) - 1, 32
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, grad = (torch.empty(1, n, m, d, dtype=F16, device="cuda").normal_(generator=gen) for _ in range(4))
    wanted = [t.requires_grad_() for t in (q, k, v)]
    out = query_attention(q, k, v)
    grads = torch.autograd.grad(out, wanted, grad)
    ends = torch.tensor([0, 1, m // 2, m - 2, m - 1], device="cuda")
    few = lambda t: t.detach()[:, :, ends].cpu()
    want = oracle_attention.attention(few(q), few(k), few(v), few(grad), unit=UNIT[F16], tiny=TINY[F16])
    for name, got in zip(("out", "grad_query", "grad_key", "grad_value"), (out, *grads)):
        close(few(got), want[name], name)


@pytest.mark.parametrize("dtype", (F16, F32), ids=IDS.get)
def test_single_tokens_of_very_many_heads(dtype):
    # one row: nothing lies behind it
    from dcnv4_amd.functions import query_attention
    m, d = (1 << 20) + 3, 32
    gen = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.empty(1, 1, m, d, dtype=dtype, device="cuda").normal_(generator=gen) for _ in range(3))
    # v w (1 / w) for the only weight w: three roundings of fp32, which fp16 does not show
    off = (query_attention(q, k, v).double() - v.double()).abs() / v.double().abs().clamp_min(1e-30)
    assert off.max() <= (0 if dtype == F16 else 3 * 2.0 ** -24)


class Doubled(torch.nn.LayerNorm):
    def forward(self, x):
        return 2 * super().forward(x)


class Named(torch.nn.LayerNorm):
    """A subclass that leaves the forward as it is."""


def norm_inputs(width=64):
    gen = torch.Generator().manual_seed(3)
    return [torch.randn(5, 7, width, generator=gen).cuda() for _ in range(3)]


def seen_by(norm, register):
    """What a hook that `register` puts on the norm sees of a call and its backward."""
    from dcnv4_amd.functions import add_layer_norm
    x, r, grad = norm_inputs()
    seen = []
    handle = register(lambda *args: seen.append(args))
    try:
        out = add_layer_norm(x.requires_grad_(), r, norm)
        out.backward(grad)
    finally:
        handle.remove()
    assert (out - torch.nn.functional.layer_norm(x + r, (64,), norm.weight, norm.bias, norm.eps)).abs().max() < 1e-5
    return seen


def test_hooks_of_a_norm_run():
    norm = torch.nn.LayerNorm(64).cuda()
    module = torch.nn.modules.module
    for register in (norm.register_forward_hook, norm.register_forward_pre_hook, norm.register_full_backward_hook, norm.register_full_backward_pre_hook,
                     module.register_module_forward_hook, module.register_module_forward_pre_hook):
        assert len(seen_by(norm, register)) == 1, register


def test_a_norms_own_forward_runs():
    from dcnv4_amd.functions import add_layer_norm
    x, r, _ = norm_inputs()
    norm = Doubled(64).cuda()
    out, total = add_layer_norm(x, r, norm, return_sum=True)
    assert torch.equal(out, norm(x + r)) and torch.equal(total, x + r)
    norm = torch.nn.LayerNorm(64).cuda()
    norm.forward = lambda x: x + 1
    assert torch.equal(add_layer_norm(x, r, norm), x + r + 1)
    assert torch.equal(add_layer_norm(x, r, torch.nn.Identity()), x + r)
    rms = torch.nn.RMSNorm(64).cuda()
    assert torch.equal(add_layer_norm(x, r, rms), rms(x + r))


def test_a_subclass_that_leaves_the_forward_as_it_is_takes_the_kernels():
    from dcnv4_amd.functions import add_layer_norm
    x, r, _ = norm_inputs()
    out = add_layer_norm(x.requires_grad_(), r, Named(64).cuda())
    assert out.grad_fn.name() == "AddLayerNormFunctionBackward"


def test_a_block_tails_norm_runs_its_hooks_and_its_own_forward():
    from dcnv4_amd.functions import layer_norm_residual
    x, r, _ = norm_inputs()
    gamma = torch.rand(64, device="cuda")
    norm, seen = torch.nn.LayerNorm(64).cuda(), []
    plain = layer_norm_residual(x, norm, gamma, r)
    handle = norm.register_forward_hook(lambda *args: seen.append(args))
    hooked = layer_norm_residual(x, norm, gamma, r)
    handle.remove()
    assert len(seen) == 1 and (hooked - plain).abs().max() < 1e-5
    doubled = Doubled(64).cuda()
    assert torch.equal(layer_norm_residual(x, doubled, gamma, r), r + gamma * doubled(x))
    assert torch.equal(layer_norm_residual(x, torch.nn.Identity()), x)
    assert layer_norm_residual(x.requires_grad_(), Named(64).cuda()).grad_fn.name() == "LayerNormResidualFunctionBackward"


def test_hooks_inside_a_layer_run():
    from dcnv4_amd.models.flash_intern_image import InternImageLayer
    layer = InternImageLayer(channels=64, groups=4, layer_scale=1.0).cuda().eval()
    norms = [m for m in layer.modules() if isinstance(m, torch.nn.LayerNorm)]
    x, seen = torch.randn(1, 64, 64, device="cuda"), []
    with torch.no_grad():
        plain = layer(x, (8, 8))
        handles = [m.register_forward_hook(lambda *args: seen.append(args)) for m in norms]
        hooked = layer(x, (8, 8))
    for h in handles:
        h.remove()
    assert norms and len(seen) == len(norms) and (hooked - plain).abs().max() < 1e-4


def attention_inputs(dtype):
    from tests.test_gpu_query_attention import inputs, leaves, on_gpu
    t = on_gpu(inputs(2, 500, 500, 4, 4, 32, dtype, mask="documents", distance=True, seed=51))
    return t, leaves(t)


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
def test_all_that_attention_keeps_passes_through_hooks_for_saved_tensors(dtype):
    from tests.test_gpu_query_attention import call
    t, wanted = attention_inputs(dtype)
    plain = call(t)
    plain_grads = torch.autograd.grad(plain, wanted, t["grad"])
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        out = call(t)
    # what stays on the GPU is the result
    assert torch.cuda.memory_allocated() - before <= out.numel() * out.element_size() + 512
    assert torch.equal(out, plain)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, wanted, t["grad"]), plain_grads))


@pytest.mark.parametrize("dtype", (F32, F16), ids=IDS.get)
def test_all_that_a_normalised_sum_keeps_passes_through_hooks_for_saved_tensors(dtype):
    from dcnv4_amd.functions import add_layer_norm
    gen = torch.Generator().manual_seed(4)
    x, r, grad = (torch.randn(20000, 16, generator=gen).to(dtype).cuda() for _ in range(3))
    norm = torch.nn.LayerNorm(16).cuda().to(dtype)
    wanted = [x.requires_grad_(), r.requires_grad_(), norm.weight, norm.bias]
    plain = add_layer_norm(x, r, norm)
    plain_grads = torch.autograd.grad(plain, wanted, grad)
    before = torch.cuda.memory_allocated()
    with torch.autograd.graph.save_on_cpu():
        out = add_layer_norm(x, r, norm)
    assert torch.cuda.memory_allocated() - before <= out.numel() * out.element_size() + 512
    assert torch.equal(out, plain)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, wanted, grad), plain_grads))


def test_operators_under_checkpointing():
    from torch.utils.checkpoint import checkpoint
    from dcnv4_amd.functions import add_layer_norm
    from tests.test_gpu_query_attention import call
    t, wanted = attention_inputs(F16)
    norm = torch.nn.LayerNorm(32).cuda()
    wanted.append(norm.weight)

    def step(query):
        return add_layer_norm(call(dict(t, q=query)), query, norm)

    plain = step(t["q"])
    out = checkpoint(step, t["q"], use_reentrant=False)
    assert torch.equal(out, plain)
    for a, b in zip(torch.autograd.grad(out, wanted, t["grad"].to(out.dtype)), torch.autograd.grad(plain, wanted, t["grad"].to(out.dtype))):
        assert torch.equal(a, b)


def test_a_second_backward_of_what_is_kept_and_of_what_is_freed():
    from tests.test_gpu_query_attention import call
    t, wanted = attention_inputs(F16)
    out = call(t)
    first = torch.autograd.grad(out, wanted, t["grad"], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(out, wanted, t["grad"])))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, wanted, t["grad"])


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
def test_rows_without_deviation_do_not_show_in_the_weights_gradient(dtype):
    # 64 equal numbers have an exact mean: xhat is zero, forward and backward, whatever their size beside the deviation
    from dcnv4_amd.functions import add_layer_norm
    gen = torch.Generator().manual_seed(5)
    norm = torch.nn.LayerNorm(64).cuda()
    x = (torch.randint(1, 200, (300, 1), generator=gen) * 3.0).expand(300, 64).to(dtype).cuda().requires_grad_()
    r = torch.ones(300, 64, dtype=dtype, device="cuda")
    out = add_layer_norm(x, r, norm)
    grad = torch.randn(300, 64, generator=gen).to(out.dtype).cuda()
    assert torch.equal(out, norm.bias.to(out.dtype).expand(300, 64))
    grad_weight, grad_x = torch.autograd.grad(out, (norm.weight, x), grad)
    assert not grad_weight.any()
    # and the summands' are rstd (g - mean(g)): a rounding of the type, and a few of fp32 of sums of 64
    g = grad.double()
    want = (g - g.mean(-1, keepdim=True)) * norm.eps ** -0.5
    off = UNIT[dtype] * want.abs() + 2.0 ** -20 * norm.eps ** -0.5 * (g.abs() + g.abs().mean(-1, keepdim=True))
    assert ((grad_x.double() - want).abs() <= off).all()
