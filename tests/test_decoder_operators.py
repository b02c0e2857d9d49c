"""What query_attention and add_layer_norm refuse or leave to torch without a GPU, and the oracle of the first."""
import pytest
import torch

from oracle import query_attention as oracle_attention


def test_attention_refuses_cpu_tensors():
    from dcnv4_amd.functions import query_attention
    t = torch.zeros(1, 3, 2, 8)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        query_attention(t, t, t)
    with pytest.raises(RuntimeError, match="no gradient for positions"):
        query_attention(t, t, t, positions=torch.zeros(1, 3, 2, requires_grad=True), slopes=torch.zeros(2))


def test_normalised_sum_of_cpu_tensors_is_torchs():
    from dcnv4_amd.functions import add_layer_norm
    norm = torch.nn.LayerNorm(6)
    x, r = torch.randn(4, 6), torch.randn(4, 6)
    out, total = add_layer_norm(x, r, norm, return_sum=True)
    assert torch.equal(out, norm(x + r)) and torch.equal(total, x + r)
    assert torch.equal(add_layer_norm(x, None, norm), norm(x))
    assert torch.equal(add_layer_norm(x, r[:1], norm), norm(x + r[:1]))


def test_oracle_agrees_with_torch_and_with_differences():
    gen = torch.Generator().manual_seed(0)
    normal = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)
    q, k, v, g = normal(2, 5, 4, 6), normal(2, 7, 2, 6), normal(2, 7, 2, 6), normal(2, 5, 4, 6)
    plain = oracle_attention.attention(q, k, v)["out"][0]
    spread = lambda t: t.transpose(1, 2).repeat_interleave(2, 1)
    want = torch.nn.functional.scaled_dot_product_attention(q.transpose(1, 2), spread(k), spread(v)).transpose(1, 2)
    assert torch.allclose(plain, want, rtol=1e-12, atol=1e-12)

    slopes = torch.rand(4, generator=gen, dtype=torch.float64)
    kw = dict(cap=2.0, q_segments=torch.tensor([[0, 1, 1, 2, -1], [1, 1, 2, 2, 3]]), q_points=torch.rand(2, 5, 2, generator=gen),
              k_segments=torch.tensor([[0, 0, 1, 1, 2, -1, -1], [1, 1, 1, 2, 2, 2, 2]]), k_points=torch.rand(2, 7, 2, generator=gen))
    found = oracle_attention.attention(q, k, v, g, slopes=slopes, **kw)
    assert not found["out"][0][0, 4].any() and not found["out"][0][1, 4].any()          # rows that see nothing
    for i, name in enumerate(("grad_query", "grad_key", "grad_value", "grad_slopes")):
        args = [q, k, v, slopes]
        way = normal(*args[i].shape)

        def along(step):
            moved = [a + step * way if n == i else a for n, a in enumerate(args)]
            return (oracle_attention.attention(*moved[:3], slopes=moved[3], **kw)["out"][0] * g).sum()

        slope = (along(1e-5) - along(-1e-5)) / 2e-5
        assert abs(slope - (found[name][0] * way).sum()) < 1e-7


def test_oracle_gives_no_weight_to_what_is_not_seen():
    q, k, v = torch.ones(1, 2, 1, 4), torch.ones(1, 3, 1, 4), torch.ones(1, 3, 1, 4)
    k[0, 2], v[0, 2] = float("nan"), float("inf")
    found = oracle_attention.attention(q, k, v, q, k_segments=torch.tensor([[0, 0, -1]]))
    assert torch.equal(found["out"][0], torch.ones(1, 2, 1, 4, dtype=torch.float64))
    assert all(torch.isfinite(value).all() and torch.isfinite(tolerance).all() for value, tolerance in found.values())
