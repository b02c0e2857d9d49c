"""The operators between the sampling layers of a deformable decoder, as its users run them: attention among queries
(with groups of queries that do not see each other, padding, a bias by the distance of reference points, capped scores)
and the layer normalisation of a sum, with their gradients.

A case is a dict of plain values; ``prepare`` makes what a program has in hand before the call, ``run`` is one pass, in
elementary torch operations or, with ``own`` set, through the framework.  The kinds:

  attention   query_attention: (B, Nq, heads, width) queries over (B, Nk, kv_heads, width) keys and values
  norm        add_layer_norm: LayerNorm(x + residual) over rows

The masks of an attention case, by what a token's segment number says (0: everybody sees it, -1: padding):

  none        all see all
  padding     pictures of a batch differ in size: keys behind a picture's own are padding
  denoising   ``groups`` groups of ``group_size`` denoising queries in front of the matching queries, which all see
  documents   sequences of ragged lengths one behind the other, padding at the end
  prefix      the same behind a part that all sequences see
"""
import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_RAGGED = (1.0, 0.35, 1.6, 0.8, 0.05, 1.2)          # lengths of consecutive sequences, in units of group_size


def listed():
    def attention(name, batch, queries, keys, heads, width, dtype, train, kv_heads=0, mask="none", groups=0, group_size=0,
                  cap=0.0, distance=False):
        return dict(name=name, kind="attention", batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads or heads,
                    width=width, dtype=dtype, train=train, mask=mask, groups=groups, group_size=group_size, cap=cap,
                    distance=distance)

    def norm(name, rows, width, x, residual, params, train, stream):
        return dict(name=name, kind="norm", rows=rows, width=width, x=x, residual=residual, params=params, train=train,
                    stream=stream)

    return [
        # self-attention of a decoder's 300 queries, one picture: the smallest call, latency counts
        attention("attention fwd 1x300 fp16", 1, 300, 0, 8, 32, "float16", False),
        # one pooling query a picture over the pixels of a padded four-level pyramid: a single token, a long odd axis
        attention("attention fwd 2x1 over 22223 fp16", 2, 1, 22223, 8, 32, "float16", False, mask="padding"),
        # proposals of four pictures, scores lowered by the distance of their reference points
        attention("attention fwd 4x2500 distance bf16", 4, 2500, 0, 8, 32, "bfloat16", False, distance=True),
        # a decoder in mixed-precision training: 900 matching queries behind five groups of 40 denoising ones
        attention("attention train 2x1100 denoising fp16", 2, 1100, 0, 8, 32, "float16", True, mask="denoising", groups=5, group_size=40),
        # the same without denoising, single precision
        attention("attention train 4x900 fp32", 4, 900, 0, 8, 32, "float32", True),
        # shared key heads of 128, sequences of ragged lengths behind a common prefix
        attention("attention train 1x5003 prefix fp16", 1, 5003, 0, 16, 128, "float16", True, kv_heads=4, mask="prefix", group_size=700),
        # every pixel of an 88 x 88 feature map a query, capped scores, learnt slopes: the largest
        attention("attention train 2x7744 cap distance bf16", 2, 7744, 0, 8, 64, "bfloat16", True, cap=20.0, distance=True),
        # post-norm of a decoder's 300 queries
        norm("norm fwd 300x256 fp16", 300, 256, "float16", "float16", "float16", False, False),
        # the same in mixed-precision training, two pictures of 1100 queries: 16-bit branch, fp32 stream and parameters
        norm("norm train 2200x256 amp", 2200, 256, "float16", "float32", "float32", True, False),
        # encoder layer of a detector, two pictures, single precision
        norm("norm train 44446x256 fp32", 44446, 256, "float32", "float32", "float32", True, False),
        # a width that is no whole number of vectors
        norm("norm train 5003x1001 bf16", 5003, 1001, "bfloat16", "bfloat16", "bfloat16", True, False),
        # first stage of FlashInternImage-B at batch 128 in pre-norm form: the sum is the stream, and comes back with a gradient
        norm("norm train 401408x112 stream fp16", 401408, 112, "float16", "float16", "float16", True, True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_one(rng):
    if rng.random() < 0.6:
        dtype = rng.choice(tuple(_DTYPES))
        mask = rng.choice(("none", "none", "padding", "denoising", "documents", "prefix"))
        queries = _log_int(rng, 1, 10000)
        cross = mask in ("none", "padding") and rng.random() < 0.4
        kv_heads = _log_int(rng, 1, 16)
        case = dict(kind="attention", batch=_log_int(rng, 1, 32), queries=queries, keys=_log_int(rng, 1, 30000) if cross else 0,
                    heads=kv_heads * rng.choice((1, 1, 1, 2, 4)), kv_heads=kv_heads,
                    width=rng.choice((16, 32, 32, 32, 64, 64, 96, 128, 8 * rng.randint(1, 16), rng.randint(4, 128))),
                    dtype=dtype, train=rng.random() < 0.5, mask=mask,
                    groups=rng.randint(1, 12) if mask == "denoising" else 0,
                    group_size=max(1, queries // rng.randint(2, 40)) if mask not in ("none", "padding") else 0,
                    cap=rng.choice((0.0, 0.0, 10.0, 30.0, 50.0)), distance=rng.random() < 0.35)
        pairs = case["batch"] * case["heads"] * queries * (case["keys"] or queries)
        # an fp32 pair costs an order of magnitude more than a 16-bit one
        limit = 2 * 8 * 7744 ** 2 * 64 // (8 if dtype == "float32" else 1)
        size = case["batch"] * max(queries, case["keys"]) * case["heads"] * case["width"]
        return case if pairs * case["width"] <= limit and pairs <= 2 * 8 * 7744 ** 2 and size <= 50_000_000 else None
    x = rng.choice(tuple(_DTYPES))
    mixed = x != "float32" and rng.random() < 0.4
    case = dict(kind="norm", rows=_log_int(rng, 1, 401408), width=_log_int(rng, 8, 8192), x=x, residual="float32" if mixed else x,
                params="float32" if mixed else x, train=rng.random() < 0.6, stream=rng.random() < 0.4)
    return case if case["rows"] * case["width"] * (2 if x == "float32" or mixed else 1) <= 401408 * 112 else None


def draw(rng):
    while True:
        case = _draw_one(rng)
        if case is not None:
            return case


def _segments(case, b):
    """[(segment, tokens)] of the b-th sequence of a batch, in order: the keys' for the padding mask, else the tokens'."""
    n, mask, size = case["keys"] or case["queries"], case["mask"], case["group_size"]
    padded = b * n // (4 * case["batch"])             # none in the first of a batch, up to a quarter of the last
    if mask == "padding":
        return [(0, n - padded), (-1, padded)]
    runs, at = [], 0

    def add(segment, tokens, end):
        nonlocal at
        tokens = max(0, min(tokens, end - at))
        runs.append((segment, tokens))
        at += tokens

    if mask == "denoising":
        for g in range(case["groups"]):
            add(g + 1, size, n)
        add(0, n, n)
        return runs
    if mask == "prefix":
        add(0, max(1, size // 2), n)
    i = 0
    while at < n - padded:
        add(i + 1, max(1, int(size * _RAGGED[i % len(_RAGGED)])), n - padded)
        i += 1
    add(-1, n, n)
    return runs


def _visible_pairs(case):
    nq, nk = case["queries"], case["keys"] or case["queries"]
    if case["mask"] == "none":
        return case["batch"] * nq * nk
    pairs = 0
    for b in range(case["batch"]):
        runs = _segments(case, b)
        if case["mask"] == "padding":
            pairs += nq * runs[0][1]
            continue
        shared = sum(tokens for segment, tokens in runs if segment == 0)
        pairs += sum(tokens * (shared + (tokens if segment > 0 else 0)) for segment, tokens in runs if segment >= 0)
    return pairs


def _segment_tensor(case):
    rows = [torch.cat([torch.full((tokens,), segment, dtype=torch.int32) for segment, tokens in _segments(case, b)])
            for b in range(case["batch"])]
    return torch.stack(rows).cuda()


def _prepare_attention(case, normal, gen):
    dtype = _DTYPES[case["dtype"]]
    b, nq, nk, h, hk, d = (case[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "width"))
    state = dict(kind="attention", train=case["train"], cap=case["cap"], segments=None, key_segments=None, positions=None,
                 key_positions=None, slopes=None)
    # queries as long as trained ones, so that a row's weights differ by orders of magnitude
    if nk == 0 and hk == h:          # one projection's output in three views, as a layer's in_proj leaves it
        packed = normal(b, nq, 3, h, d)
        packed[:, :, 0] *= 1.5
        q, k, v = packed.to(dtype).unbind(2)
    else:
        q = (normal(b, nq, h, d) * 1.5).to(dtype)
        k, v = normal(b, nk or nq, hk, d).to(dtype), normal(b, nk or nq, hk, d).to(dtype)
    if case["mask"] == "padding":
        state["key_segments"] = _segment_tensor(case)
        state["segments"] = torch.zeros(b, nq, dtype=torch.int32, device="cuda")
        if nk == 0:                  # self-attention: padded tokens are padding as queries too
            state["segments"], state["key_segments"] = state["key_segments"], None
    elif case["mask"] != "none":
        state["segments"] = _segment_tensor(case)
    if case["distance"]:             # reference points in the unit square; heads from far- to short-sighted
        state["positions"] = torch.rand(b, nq, 2, generator=gen, device="cuda")
        if nk:
            state["key_positions"] = torch.rand(b, nk, 2, generator=gen, device="cuda")
        state["slopes"] = torch.logspace(-1, 4, h, base=2.0, device="cuda") * (1 + 0.1 * normal(h))
    leaves = [t.detach() for t in (q, k, v)]
    if case["train"]:
        if case["distance"]:
            state["slopes"].requires_grad_()
        leaves = [t.requires_grad_() for t in leaves]
        state["grad"] = normal(b, nq, h, d).to(dtype)
    return dict(state, query=leaves[0], key=leaves[1], value=leaves[2])


def _prepare_norm(case, normal):
    rows, width = case["rows"], case["width"]
    # a residual stream: channels with means of their own, a few of them large
    centre = normal(width) * 0.5
    centre[:: max(1, width // 4)] += 6.0
    x = normal(rows, width).to(_DTYPES[case["x"]])
    residual = (normal(rows, width) + centre).to(_DTYPES[case["residual"]])
    norm = torch.nn.LayerNorm(width, eps=1e-6, device="cuda")
    with torch.no_grad():
        norm.weight.add_(0.2 * normal(width))
        norm.bias.add_(0.2 * normal(width))
    norm.to(_DTYPES[case["params"]])
    state = dict(kind="norm", train=case["train"], stream=case["stream"], x=x, residual=residual, norm=norm)
    if case["train"]:
        x.requires_grad_()
        residual.requires_grad_()
        state["grad"] = normal(rows, width).to(residual.dtype)
        if case["stream"]:
            state["grad_stream"] = normal(rows, width).to(residual.dtype)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    return _prepare_attention(case, normal, gen) if case["kind"] == "attention" else _prepare_norm(case, normal)


def _plain_attention(state):
    """Sequence by sequence, all heads at once: the scores of a whole batch would not be worth their memory."""
    query, key, value, train = state["query"], state["key"], state["value"], state["train"]
    b, nq, h, d = query.shape
    spread = torch.arange(h, device="cuda") // (h // key.shape[2])         # head -> key head
    slopes = state["slopes"]
    segments, positions = state["segments"], state["positions"]
    key_segments = segments if state["key_segments"] is None else state["key_segments"]
    key_positions = positions if state["key_positions"] is None else state["key_positions"]
    outs, grads = [], []
    slope_grad = 0.0
    for i in range(b):
        q, k, v = (t[i].detach().float().requires_grad_(train) for t in (query, key, value))
        slope = slopes.detach().requires_grad_(train) if slopes is not None else None
        with torch.set_grad_enabled(train):
            kh, vh = k.transpose(0, 1)[spread].contiguous(), v.transpose(0, 1)[spread].contiguous()
            s = torch.matmul(q.transpose(0, 1).contiguous(), kh.transpose(1, 2).contiguous()) * d ** -0.5
            if state["cap"]:
                s = state["cap"] * torch.tanh(s / state["cap"])
            if slope is not None:
                diff = positions[i][:, None] - key_positions[i][None]
                s = s - slope[:, None, None] * (diff * diff).sum(-1).sqrt()
            if segments is not None:
                a, c = segments[i][:, None], key_segments[i][None]
                s = torch.where((a >= 0) & ((a == c) | (c == 0)), s, float("-inf"))
            top = s.detach().amax(-1, keepdim=True)
            p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
            total = p.sum(-1, keepdim=True)
            out = (torch.matmul(p, vh) / torch.where(total > 0, total, 1.0)).transpose(0, 1)
        outs.append(out.detach().to(query.dtype))
        if train:
            got = torch.autograd.grad(out, [q, k, v] + ([slope] if slope is not None else []), state["grad"][i].float())
            grads.append([g.to(query.dtype) for g in got[:3]])
            if slope is not None:
                slope_grad = slope_grad + got[3]
    out = torch.stack(outs)
    if not train:
        return out
    found = [out] + [torch.stack(g) for g in zip(*grads)]
    return (*found, slope_grad) if slopes is not None else tuple(found)


def _plain_norm(state):
    x, residual, norm = state["x"].detach(), state["residual"].detach(), state["norm"]
    weight, bias = norm.weight.detach().float(), norm.bias.detach().float()
    z = x.float() + residual.float()
    centred = z - z.mean(-1, keepdim=True)
    rstd = ((centred * centred).mean(-1, keepdim=True) + norm.eps).rsqrt()
    normed = centred * rstd
    outs = [(normed * weight + bias).to(residual.dtype)]
    if state["stream"]:
        outs.append(z.to(residual.dtype))
    if state["train"]:
        g = state["grad"].float()
        a = g * weight
        dz = rstd * (a - a.mean(-1, keepdim=True) - normed * (a * normed).mean(-1, keepdim=True))
        if state["stream"]:
            dz = dz + state["grad_stream"].float()
        outs += [dz.to(x.dtype), dz.to(residual.dtype), (g * normed).sum(0).to(norm.weight.dtype), g.sum(0).to(norm.bias.dtype)]
    return tuple(outs)


def _own_attention(state):
    from dcnv4_amd.functions import query_attention
    inputs = [state["query"], state["key"], state["value"]]
    out = query_attention(*inputs, cap=state["cap"], segments=state["segments"], key_segments=state["key_segments"],
                          positions=state["positions"], key_positions=state["key_positions"], slopes=state["slopes"])
    if not state["train"]:
        return out
    if state["slopes"] is not None:
        inputs.append(state["slopes"])
    return (out.detach(), *torch.autograd.grad(out, inputs, state["grad"]))


def _own_norm(state):
    from dcnv4_amd.functions import add_layer_norm
    x, residual, norm = state["x"], state["residual"], state["norm"]
    with torch.set_grad_enabled(state["train"]):
        outs = add_layer_norm(x, residual, norm, return_sum=state["stream"])
    outs = outs if state["stream"] else (outs,)
    if not state["train"]:
        return outs
    grads = [state["grad"]] + ([state["grad_stream"]] if state["stream"] else [])
    return (*(o.detach() for o in outs), *torch.autograd.grad(outs, [x, residual, norm.weight, norm.bias], grads))


def run(state):
    if state["kind"] == "attention":
        return _own_attention(state) if own else _plain_attention(state)
    return _own_norm(state) if own else _plain_norm(state)


def work(case):
    """Bytes: every tensor that goes in or comes out, once. Operations: the products of visible pairs, two forward and four
    more backward; of a normalised element 8 forward and 12 backward."""
    if case["kind"] == "attention":
        size = 4 if case["dtype"] == "float32" else 2
        nq, nk = case["queries"], case["keys"] or case["queries"]
        rows_q = case["batch"] * nq * case["heads"] * case["width"]
        rows_k = case["batch"] * nk * case["kv_heads"] * case["width"]
        moved = size * (2 * rows_q + 2 * rows_k) * (2 if case["train"] else 1)
        extra = (4 if case["mask"] != "none" else 0) + (8 if case["distance"] else 0)
        products = 6 if case["train"] else 2
        return {"bytes": moved + extra * case["batch"] * (nq + nk),
                "flops": products * 2 * case["width"] * case["heads"] * _visible_pairs(case)}
    elements = case["rows"] * case["width"]
    x, r = (4 if case[k] == "float32" else 2 for k in ("x", "residual"))
    moved = x + 2 * r + (r if case["stream"] else 0)                # in, in, out and the sum
    if case["train"]:                                               # gradients in, gradients out
        moved += r + (r if case["stream"] else 0) + (x if x != r else 0) + r
    return {"bytes": elements * moved, "flops": elements * (20 if case["train"] else 8)}


def _exact_attention(case, state):
    train, cap, scale = case["train"], case["cap"], case["width"] ** -0.5
    q, k, v = (state[n].detach().double() for n in ("query", "key", "value"))
    b, nq, h, d = q.shape
    nk, share = k.shape[1], h // k.shape[2]
    ids, points = state["segments"], state["positions"]
    key_ids = ids if state["key_segments"] is None else state["key_segments"]
    key_points = points if state["key_positions"] is None else state["key_positions"]
    out, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    dslope = torch.zeros(h, dtype=torch.float64, device="cuda")
    step = max(1, (1 << 26) // max(nk, 1))             # rows at a time
    for i in range(b):
        for head in range(h):
            key, value = k[i, :, head // share].contiguous(), v[i, :, head // share].contiguous()
            for at in range(0, nq, step):
                rows = slice(at, min(nq, at + step))
                query = q[i, rows, head].contiguous()
                s = scale * (query @ key.t())
                if cap:
                    th = torch.tanh(s / cap)
                    s = cap * th
                if points is not None:
                    apart = torch.hypot(points[i, rows, 0, None].double() - key_points[i, None, :, 0].double(),
                                        points[i, rows, 1, None].double() - key_points[i, None, :, 1].double())
                    s = s - state["slopes"][head].detach().double() * apart
                if ids is not None:
                    mine, theirs = ids[i, rows, None], key_ids[i, None]
                    s = s.masked_fill((mine < 0) | ((theirs != mine) & (theirs != 0)), -math.inf)
                p = torch.softmax(s, -1).nan_to_num(0.0)           # a row that sees nothing: zeros
                out[i, rows, head] = p @ value
                if train:
                    go = state["grad"][i, rows, head].double()
                    dv[i, :, head // share] += p.t() @ go
                    dp = go @ value.t()
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
                    if points is not None:
                        dslope[head] -= (ds * apart).sum()
                    if cap:
                        ds = ds * (1 - th * th)
                    dq[i, rows, head] = scale * (ds @ key)
                    dk[i, :, head // share] += scale * (ds.t() @ query)
    if not train:
        return out
    return (out, dq, dk, dv, dslope) if points is not None else (out, dq, dk, dv)


def _exact_norm(case, state):
    norm, train = state["norm"], case["train"]
    x, residual, weight, bias = (t.detach().double().requires_grad_(train) for t in (state["x"], state["residual"], norm.weight, norm.bias))
    z = x + residual
    var, mean = torch.var_mean(z, -1, correction=0, keepdim=True)
    outs = [(z - mean) / torch.sqrt(var + norm.eps) * weight + bias] + ([z] if case["stream"] else [])
    if not train:
        return tuple(outs)
    sent = [state["grad"].double()] + ([state["grad_stream"].double()] if case["stream"] else [])
    return (*(o.detach() for o in outs), *torch.autograd.grad(outs, [x, residual, weight, bias], sent))


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_attention(case, state) if case["kind"] == "attention" else _exact_norm(case, state)
