"""How add_layer_norm and layer_norm_residual judge a norm, and what they make of it without a GPU."""
import pytest
import torch


class Named(torch.nn.LayerNorm):
    """The forward as it is."""


class Doubled(torch.nn.LayerNorm):
    def forward(self, x):
        return 2 * super().forward(x)


def test_which_norms_are_their_parameters_and_nothing_else():
    from dcnv4_amd import ext
    plain = ext._native.plain_layer_norm
    norm = torch.nn.LayerNorm(8)
    assert plain(norm, 8) and plain(Named(8), 8) and plain(torch.nn.LayerNorm(8, elementwise_affine=False), 8)
    assert not plain(norm, 7) and not plain(norm, 1 << 40) and not plain(torch.nn.LayerNorm((2, 8)), 8)
    assert not plain(Doubled(8), 8) and not plain(torch.nn.RMSNorm(8), 8) and not plain(torch.nn.Identity(), 8) and not plain(None, 8)
    for register in (norm.register_forward_hook, norm.register_forward_pre_hook, norm.register_full_backward_hook, norm.register_full_backward_pre_hook,
                     torch.nn.modules.module.register_module_forward_hook, torch.nn.modules.module.register_module_full_backward_hook):
        handle = register(lambda *args: None)
        assert not plain(norm, 8), register
        handle.remove()
        assert plain(norm, 8)
    norm.forward = lambda x: x
    assert not plain(norm, 8)
    with pytest.raises(TypeError):
        plain(norm, "8")
    with pytest.raises(TypeError):
        plain(norm)


def test_any_norm_of_cpu_tensors_runs():
    from dcnv4_amd.functions import add_layer_norm, layer_norm_residual
    x, r = torch.randn(4, 8), torch.randn(4, 8)
    for norm in (torch.nn.LayerNorm(8), Doubled(8), torch.nn.RMSNorm(8), torch.nn.Identity()):
        out, total = add_layer_norm(x, r, norm, return_sum=True)
        assert torch.equal(total, x + r) and torch.equal(out, norm(total))
        assert torch.equal(add_layer_norm(x, None, norm), norm(x))
        assert torch.equal(layer_norm_residual(x, norm, None, r), r + norm(x))
