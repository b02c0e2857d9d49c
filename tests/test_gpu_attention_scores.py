"""query_attention's scores at the ends of their range: caps from a few units to the largest that is taken, positions far from zero, slopes of
any size."""
import pytest
import torch

from tests.test_gpu_query_attention import BF16, F16, F32, IDS, call, check, inputs, leaves, on_gpu

pytestmark = pytest.mark.gpu


# A cap far above the scores leaves them as they are.
@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("mask,distance", [("none", False), ("random", False), ("documents", True)])
@pytest.mark.parametrize("cap", (1e-3, 200.0, 256.0, 257.0, 1e4, 1e6, 1e9, 1e30))
def test_caps_of_any_size(cap, mask, distance, dtype):
    check(inputs(1, 150, 150, 2, 1, 32, dtype, mask=mask, distance=distance, seed=41), cap=cap)


# Scores of up to some hundred, on both sides of where a cap of 300 or 1000 bends them.
@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("cap", (300.0, 1000.0))
def test_scores_that_a_large_cap_bends(cap, dtype):
    t = inputs(1, 150, 150, 2, 2, 16, dtype, seed=42)
    check(t, scale=20.0, cap=cap)
    check(t, scale=-1.0, cap=cap)


def placed(t, gen, offset, step=1 / 16, extent=800):
    """Points on a grid that fp32 holds exactly, so that two of them are as far apart wherever the grid begins."""
    n, lq, lk = t["q"].shape[0], t["q"].shape[1], t["k"].shape[1]
    offset = torch.tensor(offset, dtype=F32)
    for name, length in (("q_points", lq), ("k_points", lk)):
        t[name] = torch.randint(0, extent, (n, length, 2), generator=gen) * step + offset
    return t


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("cap", (0.0, 30.0))
@pytest.mark.parametrize("slope", (0.3, 1.0, 16.0, 1e-7, -0.7))
def test_distances_do_not_depend_on_where_the_points_lie(slope, cap, dtype):
    found = []
    for offset in ((0, 0), (1300, 700), (-20000, 100)):
        t = on_gpu(placed(inputs(2, 130, 150, 2, 2, 32, dtype, distance=True, seed=43), torch.Generator().manual_seed(5), offset))
        t["slopes"] = torch.full((2,), slope, device="cuda")
        wanted = leaves(t)
        out = call(t, cap=cap)
        found.append((out, *torch.autograd.grad(out, wanted, t["grad"])))
    for other in found[1:]:
        assert all(torch.equal(a, b) for a, b in zip(found[0], other))


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("mask", ("none", "random"))
def test_distances_in_pixels(mask, dtype):
    t = inputs(2, 130, 150, 6, 3, 32, dtype, mask=mask, distance=True, seed=44)
    placed(t, torch.Generator().manual_seed(6), (1000, 1000))
    t["slopes"] = torch.tensor([1e-3, 0.05, 1.0, 1.3, 16.0, 300.0])
    check(t)


# Slopes about where scores change their units: 2^20 times the product's factor and 2^-20 of it; and far beyond.
@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("scale", (0.17, -0.17, 0.0))
def test_slopes_of_any_size(scale, dtype):
    t = inputs(1, 90, 110, 12, 12, 32, dtype, distance=True, seed=45)
    t["slopes"] = torch.tensor([0.0, 1e-40, 1e-30, 1.5e-7, 1.7e-7, 2e-7, 1.7e5, 1.8e5, 2e5, 1e10, 1e25, -1e-30])
    t["k_points"][:, :45] = t["q_points"][:, 45:]          # some of the points meet
    t["q_points"][:, :45] = t["k_points"][:, :45]
    check(t, scale=scale)


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
def test_scales_to_the_end_of_their_range(dtype):
    from dcnv4_amd.functions import query_attention
    q, k = torch.zeros(1, 5, 2, 16, dtype=dtype, device="cuda"), torch.ones(1, 8, 2, 16, dtype=dtype, device="cuda")
    v = torch.ones(1, 8, 2, 16, dtype=dtype, device="cuda")
    # products of zero: all keys weigh the same, and the eight of them add up to one
    for scale, cap in ((1e30, 0.0), (-1e30, 0.0), (1.0, 1e-30), (1e30, 1.0), (-1e30, 1e30)):
        assert torch.equal(query_attention(q, k, v, scale=scale, cap=cap), torch.ones_like(q)), (scale, cap)
    for scale, cap, match in ((3e38, 0.0, "scale must be between"), (-1.1e30, 0.0, "scale must be between"), (2.0, 1e-30, "times cap"), (1e30, 0.5, "times cap")):
        with pytest.raises(RuntimeError, match=match):
            query_attention(q, k, v, scale=scale, cap=cap)


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("bad", (float("inf"), float("nan")))
@pytest.mark.parametrize("lq,lk,where", [(40, 300, 3), (40, 300, 299), (700, 130, 129), (1, 20, 19), (2, 5001, 5000)])
def test_an_infinite_value_that_all_see_stays_in_its_head(lq, lk, where, bad, dtype):
    t = on_gpu(inputs(1, lq, lk, 2, 2, 32, dtype, seed=46, spread=0.3))
    for train in (False, True):
        wanted = leaves(t) if train else []
        clean = call(t).detach()
        v = t["v"].detach().clone()
        v[0, where, 1, 5] = bad
        out = call(dict(t, v=v.requires_grad_(train))).detach()
        assert not torch.isfinite(out[:, :, 1, 5]).any()
        assert torch.equal(out[:, :, 0], clean[:, :, 0])


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("lq,lk", [(3, 1), (40, 300), (2, 5001)])
@pytest.mark.parametrize("cap", (0.0, 50.0))
def test_gradients_of_rows_that_are_far_from_all_keys(cap, lq, lk, dtype):
    t = inputs(2, lq, lk, 2, 2, 32, dtype, distance=True, seed=47)
    t["q_points"][:], t["k_points"][:] = 0.0, 1.0
    t["q_points"][:, 0] = 1.0          # where all keys are
    t["slopes"] = torch.tensor([30.0, 1e4])
    check(t, cap=cap)
    # the second head's queries, but for the first, are a million and a half away
    t["slopes"] = torch.tensor([30.0, 1.1e6])
    gpu = on_gpu(t)
    wanted = leaves(gpu)
    out = call(gpu, cap=cap)
    near = call(dict(gpu, slopes=torch.tensor([30.0, 0.0], device="cuda")), cap=cap)
    # distances that are all alike do not weigh, but for the last bits that scores of their size leave of the products
    assert torch.isfinite(out).all() and torch.equal(out[:, 0, 1], near[:, 0, 1])
    grad_query, grad_key, grad_value, grad_slopes = torch.autograd.grad(out, wanted, gpu["grad"])
    assert torch.isnan(grad_query[:, 1:, 1]).all() and torch.isnan(grad_key[:, :, 1]).all() and torch.isnan(grad_value[:, :, 1]).all()
    assert all(torch.isfinite(g).all() for g in (grad_query[:, :, 0], grad_query[:, 0], grad_key[:, :, 0], grad_value[:, :, 0], grad_slopes[0]))
    assert torch.isnan(grad_slopes[1])


# heads and queries for every number of columns a workgroup takes
@pytest.mark.parametrize("dtype", (F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("n,m,lq,mask,distance", [(1, 2, 200, "none", True), (1, 8, 1030, "random", False), (1, 16, 1030, "none", False), (2, 16, 1030, "none", True),
                                                  (3, 16, 1030, "none", False), (2, 16, 600, "documents", True)])
@pytest.mark.parametrize("width", (32, 64, 128))
def test_large_caps_in_every_shape_of_workgroup(width, n, m, lq, mask, distance, dtype):
    check(inputs(n, lq, lq, m, m, width, dtype, mask=mask, distance=distance, seed=width + m), device="cuda", cap=1000.0)
