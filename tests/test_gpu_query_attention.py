"""query_attention against float64 (oracle/query_attention.py, which also says how far roundings can take a result), at the
lengths, widths, masks and layouts where a tiled kernel can go wrong."""
import pytest
import torch

from oracle import query_attention as oracle_attention

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
IDS = {F32: "fp32", F16: "fp16", BF16: "bf16"}
# half a step relative to a value, and of the subnormals
UNIT = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 0.0, F16: 2.0 ** -25, BF16: 0.0}


def normal(gen, *shape):
    return torch.randn(shape, generator=gen)


def inputs(n, lq, lk, m, mk, d, dtype, mask="none", distance=False, seed=0, spread=1.5):
    gen = torch.Generator().manual_seed(seed)
    t = dict(q=(normal(gen, n, lq, m, d) * spread).to(dtype), k=normal(gen, n, lk, mk, d).to(dtype), v=normal(gen, n, lk, mk, d).to(dtype),
             grad=normal(gen, n, lq, m, d).to(dtype), q_segments=None, k_segments=None, q_points=None, k_points=None, slopes=None)
    if mask == "random":           # any order of any numbers, rows that see nothing among them
        t["q_segments"] = torch.randint(-1, 5, (n, lq), generator=gen, dtype=torch.int32)
        t["k_segments"] = torch.randint(-2, 4, (n, lk), generator=gen, dtype=torch.int32)
        t["k_segments"][0][t["k_segments"][0] == 0] = 7          # nothing shared in the first sequence
    elif mask == "padding":
        t["k_segments"] = torch.zeros(n, lk, dtype=torch.int32)
        for b in range(n):
            t["k_segments"][b, lk - lk * b // n - b:] = -1
    elif mask == "documents":      # lq == lk: packed sequences, each longer than the one before, padding behind
        ids = torch.zeros(n, lq, dtype=torch.int32)
        at, i = 0, 1
        while at < lq:
            ids[:, at:at + 3 * i] = i
            at, i = at + 3 * i, i + 1
        ids[:, lq - lq // 7:] = -1
        t["q_segments"] = t["k_segments"] = ids
    elif mask == "prefix":
        ids = torch.ones(n, lq, dtype=torch.int32)
        ids[:, :lq // 3] = 0
        ids[:, 2 * lq // 3:] = 1 << 30
        t["q_segments"] = t["k_segments"] = ids
    elif mask == "nothing":
        t["q_segments"] = torch.full((n, lq), 3, dtype=torch.int32)
        t["k_segments"] = torch.full((n, lk), 4, dtype=torch.int32)
    if distance:
        t["q_points"], t["k_points"] = torch.rand(n, lq, 2, generator=gen), torch.rand(n, lk, 2, generator=gen)
        t["slopes"] = torch.linspace(-0.5, 6.0, m)
    return t


def on_gpu(t):
    return {name: None if v is None else v.cuda() for name, v in t.items()}


def call(t, **kw):
    from dcnv4_amd.functions import query_attention
    return query_attention(t["q"], t["k"], t["v"], segments=t["q_segments"], key_segments=t["k_segments"], positions=t["q_points"],
                           key_positions=t["k_points"], slopes=t["slopes"], **kw)


def leaves(t):
    for name in ("q", "k", "v", "slopes"):
        if t[name] is not None:
            t[name] = t[name].detach().requires_grad_()
    return [t[name] for name in ("q", "k", "v", "slopes") if t[name] is not None]


def close(got, want, what):
    value, tolerance = want
    got = got.detach().to(value.device).double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    beyond = (got - value).abs() - tolerance
    assert beyond.numel() == 0 or beyond.max() <= 0, f"{what}: {beyond.max():.3e} beyond tolerance, error {(got - value).abs().max():.3e}"


def check(t, train=True, device="cpu", **kw):
    dtype = t["q"].dtype
    gpu = on_gpu(t)
    wanted = leaves(gpu) if train else []
    out = call(gpu, **kw)
    assert out.dtype == dtype and out.is_contiguous()
    want = oracle_attention.attention(t["q"], t["k"], t["v"], t["grad"] if train else None, q_segments=t["q_segments"],
                                      k_segments=t["k_segments"], q_points=t["q_points"], k_points=t["k_points"], slopes=t["slopes"],
                                      unit=UNIT[dtype], tiny=TINY[dtype], device=device, **kw)
    close(out, want["out"], "out")
    if train:
        for name, got in zip(("grad_query", "grad_key", "grad_value", "grad_slopes"), torch.autograd.grad(out, wanted, gpu["grad"])):
            close(got, want[name], name)
    return out


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("lq,lk", [(1, 1), (1, 300), (300, 1), (15, 17), (16, 64), (64, 128), (65, 63), (129, 200), (300, 300)])
def test_lengths(lq, lk, dtype):
    check(inputs(2, lq, lk, 3, 3, 32, dtype, seed=lq + lk))


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("width", (1, 5, 8, 16, 24, 25, 40, 48, 64, 72, 96, 104, 127, 128))
def test_widths(width, dtype):
    check(inputs(1, 70, 83, 2, 2, width, dtype, mask="random", seed=width))


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("m,mk", [(4, 1), (6, 2), (12, 4), (5, 5), (1, 1)])
def test_heads_that_share_a_key_head(m, mk, dtype):
    check(inputs(2, 50, 77, m, mk, 32, dtype, mask="padding", seed=m))


@pytest.mark.parametrize("mask", ("none", "random"))
@pytest.mark.parametrize("m,lk", [(8, 17000), (6, 9000)])
def test_heads_that_share_a_key_head_of_a_long_memory(m, lk, mask):
    # the heads in two parts of four, and in six of one
    check(inputs(4, 40, lk, m, 1, 32, F16, mask=mask, seed=m), device="cuda")


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("cap,distance", [(0.0, True), (3.0, False), (50.0, False), (8.0, True)])
@pytest.mark.parametrize("mask", ("none", "random", "documents", "prefix", "nothing"))
def test_masks_caps_and_distances(mask, cap, distance, dtype):
    check(inputs(2, 150, 150, 2, 1, 32, dtype, mask=mask, distance=distance, seed=11), cap=cap)


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
def test_a_few_queries_over_a_long_memory(dtype):
    for lq in (1, 3, 17):
        check(inputs(2, lq, 5001, 2, 2, 32, dtype, mask="padding", distance=lq == 3, seed=lq))


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
def test_many_queries_of_few_keys(dtype):
    check(inputs(1, 3001, 7, 2, 2, 64, dtype, mask="padding", seed=4))


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
def test_long_rows_with_peaks(dtype):
    # weights from 1 down to nothing, the largest scores anywhere in the row
    check(inputs(1, 600, 1100, 1, 1, 64, dtype, seed=5, spread=6.0))


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
def test_scores_that_grow_along_the_row(dtype):
    t = inputs(1, 40, 700, 1, 1, 32, dtype, seed=6)
    t["k"] = (t["k"].float() * 0.05 + torch.linspace(-1, 1, 700).view(1, -1, 1, 1)).to(dtype)
    t["q"] = (t["q"].float() * 0.05 + torch.linspace(-6, 6, 40).view(1, -1, 1, 1)).to(dtype)
    check(t)


# heads and queries for every number of columns a workgroup takes, forward and backward, with and without masks
@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("n,m,lq,mask", [(1, 2, 200, "none"), (1, 8, 1030, "random"), (1, 16, 1030, "none"), (2, 16, 1030, "none"), (2, 16, 600, "documents")])
@pytest.mark.parametrize("width", (32, 64, 128))
def test_every_shape_of_workgroup(width, n, m, lq, mask, dtype):
    check(inputs(n, lq, lq, m, m, width, dtype, mask=mask, seed=width + m), device="cuda")


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("distance", (False, True))
@pytest.mark.parametrize("width", (32, 64, 128))
def test_workgroups_of_128_columns(width, distance, dtype):
    check(inputs(3, 1030, 1030, 16, 16, width, dtype, distance=distance, seed=width), device="cuda")


@pytest.mark.parametrize("width", (32, 64))
def test_many_heads_with_masks(width):
    check(inputs(8, 1030, 1030, 16, 16, width, F16, mask="prefix", seed=width), device="cuda")


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("scale", (-0.4, 0.0, 1e-12, 3.0))
def test_scales(scale, dtype):
    t = inputs(1, 90, 130, 2, 2, 16, dtype, mask="random", seed=31, spread=0.7)
    check(t, scale=scale)
    check(t, scale=scale, cap=5.0)


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
def test_distances_of_any_size_and_slope(dtype):
    t = inputs(1, 70, 90, 6, 3, 16, dtype, mask="padding", distance=True, seed=32)
    t["slopes"] = torch.tensor([0.0, 1e-30, -3.0, 40.0, 1e-4, -1e-20])
    check(t)
    t["q_points"], t["k_points"] = t["q_points"] * 1000, t["k_points"] * 1000      # pixels
    t["slopes"] = t["slopes"] * 1e-3
    check(t, cap=6.0)


def test_a_memory_whose_offsets_pass_32_bits():
    # 4.3e9 elements; of 17 million keys the last hundred are seen, and some in between
    n = (1 << 24) + 77
    gen = torch.Generator(device="cuda").manual_seed(2)
    k = torch.empty(1, n, 8, 32, dtype=F16, device="cuda").normal_(generator=gen)
    v = torch.empty_like(k).normal_(generator=gen)
    q = torch.randn(1, 3, 8, 32, generator=gen, device="cuda").to(F16)
    ids = torch.full((1, n), -1, dtype=torch.int32, device="cuda")
    seen = torch.cat((torch.arange(n // 2, n // 2 + 50, device="cuda"), torch.arange(n - 100, n, device="cuda")))
    ids[:, seen] = 0
    from dcnv4_amd.functions import query_attention
    few = [x[:, seen].contiguous().requires_grad_() for x in (k, v)]
    out = query_attention(q, few[0], few[1])
    whole = query_attention(q, k, v, key_segments=ids)
    # the same weights, added up in another order and from another maximum: a rounding of each weight and of the result
    assert (whole.float() - out.float()).abs().max() <= 4 * UNIT[F16] * v[:, seen].float().abs().max()
    grad = torch.randn(1, 3, 8, 32, generator=gen, device="cuda").to(F16)
    want = torch.autograd.grad(out, few, grad)
    k.requires_grad_()
    v.requires_grad_()
    got = torch.autograd.grad(query_attention(q, k, v, key_segments=ids), (k, v), grad)
    for a, b in zip(got, want):
        assert (a[:, seen].float() - b.float()).abs().max() <= 8 * UNIT[F16] * b.float().abs().max()
        assert torch.count_nonzero(a) == torch.count_nonzero(a[:, seen])


@pytest.mark.parametrize("pitch", (5 << 10, (1 << 23) - 16, (1 << 23) + 16, 3 << 22))
def test_tokens_that_lie_megabytes_apart(pitch):
    # a tile of 128 or 256 rows reaches over 2 GB from its first one
    n, l, m, d = 2, 600, 8, 32
    t = on_gpu(inputs(n, l, l, m, m, d, F16, seed=24))
    plain_leaves = leaves(t)
    plain = call(t)
    plain_grads = torch.autograd.grad(plain, plain_leaves, t["grad"])
    memory = torch.empty(n * l * pitch // 2, dtype=F16, device="cuda")
    far = dict(t)
    for i, name in enumerate(("q", "k", "v", "grad")):
        far[name] = memory.as_strided((n, l, m, d), (l * pitch // 2, pitch // 2, d, 1), i * m * d).copy_(t[name].detach())
    far_leaves = [far[name].requires_grad_() for name in ("q", "k", "v")]
    out = call(far)
    assert torch.equal(out, plain)
    for got, want in zip(torch.autograd.grad(out, far_leaves, far["grad"]), plain_grads):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", (F16, BF16), ids=IDS.get)
def test_gradients_of_tiny_and_of_large_size(dtype):
    for factor in (1e-4, 300.0):
        t = inputs(1, 200, 200, 2, 2, 32, dtype, mask="documents", seed=7)
        t["grad"] = (t["grad"].float() * factor).to(dtype)
        check(t)


@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
def test_views_of_a_fused_projection_and_other_layouts(dtype):
    n, lq, m, d = 2, 90, 4, 32
    t = inputs(n, lq, lq, m, m, d, dtype, mask="random", distance=True, seed=8)
    layouts = {
        "fused": lambda x: torch.stack((x, x + 1, x - 1), 2)[:, :, 0],
        "heads first": lambda x: x.transpose(1, 2).contiguous().transpose(1, 2),
        "tokens first": lambda x: x.transpose(0, 1).contiguous().transpose(0, 1),
        "width not dense": lambda x: torch.stack((x, x), -1)[..., 0],
        "odd offset": lambda x: torch.cat((x.new_zeros(1), x.reshape(-1)))[1:].view(x.shape),
        "odd row": lambda x: torch.cat((x.flatten(2), x.new_zeros(n, lq, 3)), 2)[..., :m * d].unflatten(2, (m, d)),
    }
    base = on_gpu(t)
    plain = torch.autograd.grad(call(dict(base, q=(q := base["q"].requires_grad_()), k=(k := base["k"].requires_grad_()),
                                          v=(v := base["v"].requires_grad_()))), (q, k, v), base["grad"])
    for name, change in layouts.items():
        moved = {x: change(base[x].detach()) for x in ("q", "k", "v", "grad")}
        assert all(torch.equal(moved[x], base[x]) for x in moved)
        other = dict(base, **moved)
        with_grad = [other[x].requires_grad_() for x in ("q", "k", "v")]
        other["q_segments"] = torch.stack((base["q_segments"],) * 2, -1)[..., 0]
        other["q_points"] = torch.stack((base["q_points"],) * 2, -1)[..., 0]
        got = torch.autograd.grad(call(other), with_grad, moved["grad"])
        for a, b in zip(got, plain):
            assert torch.equal(a, b), name
    check(t)


@pytest.mark.parametrize("dtype", (F32, F16), ids=IDS.get)
def test_expanded_inputs_get_their_summed_gradients(dtype):
    t = inputs(3, 40, 55, 4, 4, 16, dtype, seed=9)
    t["k"], t["v"] = t["k"][:1, :, :1].expand(3, 55, 4, 16), t["v"][:, :, :1].expand(3, 55, 4, 16)
    gpu = on_gpu(t)
    k, v = gpu["k"][:1, :, :1].contiguous().requires_grad_(), gpu["v"][:, :, :1].contiguous().requires_grad_()
    q = gpu["q"].requires_grad_()
    out = call(dict(gpu, k=k.expand(3, 55, 4, 16), v=v.expand(3, 55, 4, 16)))
    grads = torch.autograd.grad(out, (q, k, v), gpu["grad"])
    want = oracle_attention.attention(t["q"], t["k"], t["v"], t["grad"], unit=UNIT[dtype], tiny=TINY[dtype])
    close(out, want["out"], "out")
    close(grads[0], want["grad_query"], "grad_query")
    summed = lambda name, dims, terms: tuple(x.sum(dims, keepdim=True) for x in want[name][:1]) + (
        want[name][1].sum(dims, keepdim=True) + terms * UNIT[dtype] * want[name][0].abs().sum(dims, keepdim=True),)
    close(grads[1], summed("grad_key", (0, 2), 12), "grad_key")
    close(grads[2], summed("grad_value", (2,), 4), "grad_value")


@pytest.mark.parametrize("bad", (float("nan"), float("inf"), -float("inf")))
@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
def test_what_is_not_seen_may_hold_anything(dtype, bad):
    n, lq, lk = 2, 140, 140
    t = inputs(n, lq, lk, 2, 2, 32, dtype, seed=10, distance=True)
    ids = torch.ones(n, lq, dtype=torch.int32)
    ids[:, 60:] = 2
    ids[:, 120:] = -1
    t["q_segments"] = t["k_segments"] = ids
    hidden = ids < 0
    for name in ("q", "k", "v", "grad"):
        t[name][hidden] = bad
    t["q_points"][hidden] = bad
    t["k_points"][hidden] = bad
    check(t)
    # and the rows of a group that nobody else sees: the other group's results and gradients are those without it
    t = inputs(n, lq, lk, 2, 2, 32, dtype, seed=10)
    t["q_segments"] = t["k_segments"] = ids
    clean = on_gpu(t)
    first = slice(0, 60)
    wanted = leaves(clean)
    reference = call(clean)
    reference_grads = torch.autograd.grad(reference, wanted, clean["grad"])
    for name in ("q", "k", "v", "grad"):
        t[name][:, 60:] = bad
    dirty = on_gpu(t)
    wanted = leaves(dirty)
    out = call(dirty)
    grads = torch.autograd.grad(out, wanted, dirty["grad"])
    seen = lambda x: x[:, first]
    tolerance = {F32: 1e-4, F16: 2e-2, BF16: 1e-1}[dtype]          # two ways to add up; the size of results is one
    for a, b in zip((out, *grads), (reference, *reference_grads)):
        assert torch.isfinite(seen(a)).all()
        assert (seen(a).float() - seen(b).float()).abs().max() <= tolerance * seen(b).float().abs().max()


@pytest.mark.parametrize("dtype", (F32, F16), ids=IDS.get)
@pytest.mark.parametrize("n,lq,lk", [(0, 4, 4), (2, 0, 5), (2, 5, 0)])
def test_empty_batches_and_lengths(n, lq, lk, dtype):
    t = inputs(n, lq, lk, 2, 2, 16, dtype, seed=1)
    t["slopes"], t["q_points"], t["k_points"] = torch.ones(2), torch.rand(n, lq, 2), torch.rand(n, lk, 2)
    gpu = on_gpu(t)
    wanted = leaves(gpu)
    out = call(gpu)
    assert out.shape == (n, lq, 2, 16) and not out.any()
    for leaf, g in zip(wanted, torch.autograd.grad(out, wanted, gpu["grad"])):
        assert g.shape == leaf.shape and not g.any()


def test_gradients_agree_with_differences():
    t = inputs(1, 9, 12, 2, 1, 8, F32, mask="random", distance=True, seed=12)
    gpu = on_gpu(t)
    wanted = leaves(gpu)
    out = call(gpu, cap=4.0)
    grads = torch.autograd.grad(out, wanted, gpu["grad"])
    gen = torch.Generator().manual_seed(3)
    for name, leaf, grad in zip(("q", "k", "v", "slopes"), wanted, grads):
        way = normal(gen, *leaf.shape).cuda()
        step = 2.0 ** -7
        with torch.no_grad():
            ahead, behind = (call(dict(gpu, **{name: leaf + s * way}), cap=4.0) for s in (step, -step))
        slope = ((ahead - behind).double() * gpu["grad"].double()).sum() / (2 * step)
        want = (grad.double() * way.double()).sum()
        # step^2 times third derivatives of a few units, and the differences' rounding over the step
        assert abs(slope - want) <= 2e-2 * (1 + abs(want)), (name, slope, want)


def test_only_the_gradients_that_are_asked_for():
    t = on_gpu(inputs(1, 40, 50, 2, 1, 32, F16, seed=13, distance=True))
    full = dict(t)
    names = ("q", "k", "v", "slopes")
    all_leaves = leaves(full)
    all_grads = torch.autograd.grad(call(full), all_leaves, t["grad"])
    for i, name in enumerate(names):
        one = dict(t)
        one[name] = t[name].detach().clone().requires_grad_()
        for other in names:
            if other != name:
                one[other] = t[other].detach()
        got, = torch.autograd.grad(call(one), one[name], t["grad"])
        assert torch.equal(got, all_grads[i]), name


def test_results_repeat_bit_for_bit():
    t = on_gpu(inputs(2, 333, 777, 4, 2, 64, BF16, mask="random", distance=True, seed=14))
    wanted = leaves(t)
    first = call(t, cap=20.0)
    first_grads = torch.autograd.grad(first, wanted, t["grad"])
    for _ in range(3):
        out = call(t, cap=20.0)
        assert torch.equal(out, first)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, wanted, t["grad"]), first_grads))


def test_a_captured_pass_replays_on_new_inputs():
    t = inputs(2, 200, 200, 2, 2, 32, F16, mask="documents", distance=True, seed=15)
    gpu = on_gpu(t)
    wanted = leaves(gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(call(gpu, cap=9.0), wanted, gpu["grad"])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(gpu, cap=9.0)
        grads = torch.autograd.grad(out, wanted, gpu["grad"])
    for seed in (16, 17, 18):
        fresh = on_gpu(inputs(2, 200, 200, 2, 2, 32, F16, mask="documents", distance=True, seed=seed))
        with torch.no_grad():
            for name in ("q", "k", "v", "grad", "q_points", "k_points"):
                gpu[name].copy_(fresh[name])
        graph.replay()
        torch.cuda.synchronize()
        eager_leaves = leaves(fresh)
        eager = call(fresh, cap=9.0)
        eager_grads = torch.autograd.grad(eager, eager_leaves, fresh["grad"])
        assert torch.equal(out, eager)
        assert all(torch.equal(a, b) for a, b in zip(grads, eager_grads))


def test_two_calls_on_two_streams():
    a, b = (on_gpu(inputs(2, 300, 4000, 4, 4, 32, F16, seed=s)) for s in (19, 20))
    alone = [call(x) for x in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        for s, x in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(call(x))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert torch.equal(out, alone[i % 2])


def test_autocast_casts_and_gradients_come_back_in_the_inputs_type():
    t = on_gpu(inputs(1, 60, 60, 2, 2, 32, F32, seed=21))
    wanted = leaves(t)
    with torch.autocast("cuda", dtype=BF16):
        out = call(t)
    assert out.dtype == BF16
    grads = torch.autograd.grad(out, wanted, t["grad"].to(BF16))
    halves = {name: None if v is None else v.detach().to(BF16) for name, v in t.items()}
    half_leaves = leaves(halves)
    ref = call(halves)
    assert torch.equal(ref, out)
    for got, want in zip(grads, torch.autograd.grad(ref, half_leaves, halves["grad"])):
        assert got.dtype == F32 and torch.equal(got, want.float())


def test_a_changed_input_is_noticed_and_second_derivatives_are_refused():
    t = on_gpu(inputs(1, 20, 20, 1, 1, 16, F32, seed=22))
    q, k, v = leaves(t)
    out = call(t)
    with torch.no_grad():
        k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(t["grad"])
    t = on_gpu(inputs(1, 20, 20, 1, 1, 16, F32, seed=22))
    wanted = leaves(t)
    g, = torch.autograd.grad(call(t), wanted[:1], t["grad"], create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_a_traced_call_computes_its_result():
    t = on_gpu(inputs(1, 33, 33, 2, 2, 16, F32, seed=23))
    from dcnv4_amd.functions import query_attention
    want = call(t)
    # the Function's own Python, which runs where torch records operators
    class Watch(torch.utils._python_dispatch.TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))
    wanted = leaves(t)
    with Watch():
        out = query_attention(t["q"], t["k"], t["v"])
    assert torch.equal(out, want)
    plain = torch.autograd.grad(call(t), wanted, t["grad"])
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, wanted, t["grad"]), plain))


def test_refusals():
    from dcnv4_amd.functions import query_attention
    z = lambda *s, dtype=F16: torch.zeros(*s, dtype=dtype, device="cuda")
    q, k, v = z(2, 5, 4, 32), z(2, 7, 2, 32), z(2, 7, 2, 32)
    ok = dict(query=q, key=k, value=v)

    def refused(match, error=RuntimeError, **kw):
        with pytest.raises(error, match=match):
            query_attention(**{**ok, **kw})

    refused("dtype Float, expected Half", key=k.float())
    refused("dtype", query=q.double(), key=k.double(), value=v.double())
    refused("4-d", query=q[0])
    refused("expected", value=v[:, :6])
    refused("expected", key=k[:1])
    refused("share", key=z(2, 7, 3, 32), value=z(2, 7, 3, 32))
    refused("channels are not supported", query=z(1, 2, 1, 136), key=z(1, 2, 1, 136), value=z(1, 2, 1, 136))
    refused("CUDA tensor", value=v.cpu())
    refused("expected Int", segments=z(2, 5, dtype=torch.int64), key_segments=z(2, 7, dtype=torch.int32))
    refused("expected", segments=z(2, 5, dtype=torch.int32))           # seven keys
    refused("go together", positions=z(2, 5, 2, dtype=F32), key_positions=z(2, 7, 2, dtype=F32))
    refused("expected Float", positions=z(2, 5, 2), key_positions=z(2, 7, 2), slopes=z(4, dtype=F32))
    refused("slopes", positions=z(2, 5, 2, dtype=F32), key_positions=z(2, 7, 2, dtype=F32), slopes=z(2, dtype=F32))
    refused("no gradient for positions", positions=z(2, 5, 2, dtype=F32).requires_grad_(), key_positions=z(2, 7, 2, dtype=F32), slopes=z(4, dtype=F32))
    refused("cap", cap=-1.0)
    refused("cap", cap=1e-60)
    refused("scale", scale=float("inf"))
    refused("scale", scale=float("nan"))
    refused("cap", cap=float("inf"))
    refused("cap", cap=float("nan"))


def test_batches_beyond_a_launch_are_refused():
    from dcnv4_amd.functions import query_attention
    one = torch.zeros(1, 1, 1, 8, dtype=F16, device="cuda")
    for shape, match in (((1 << 21, 1, 8, 8), "24 - 1 pieces"), ((1 << 20, 129, 8, 8), "24 - 1 pieces"), ((1 << 20, 300, 8, 8), "31 - 1 rows")):
        many = one.expand(shape)      # refused before anything is allocated
        with pytest.raises(RuntimeError, match=match):
            query_attention(many, many, many)
