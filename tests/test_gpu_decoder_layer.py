"""A deformable decoder's layer as a program would build it: attention among queries, normalised sums, sampling attention and an MLP, trained.
The same layer with plain torch operators in the places of query_attention and add_layer_norm says what it should compute."""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

LEVELS = [(20, 24), (10, 12), (5, 6), (3, 3)]


def plain_attention(q, k, v, segments, points, slopes, cap):
    s = torch.einsum("nqmd,nkmd->nmqk", q, k) * q.shape[-1] ** -0.5
    s = cap * torch.tanh(s / cap) - slopes.view(1, -1, 1, 1) * (points[:, :, None] - points[:, None]).norm(dim=-1)[:, None]
    mine, theirs = segments[:, :, None], segments[:, None]
    see = ((mine >= 0) & ((mine == theirs) | (theirs == 0)))[:, None]
    p = torch.softmax(s.masked_fill(~see, -torch.inf), -1).nan_to_num(0.0)
    return torch.einsum("nmqk,nkmd->nqmd", p, v)


class Layer(nn.Module):
    def __init__(self, width=256, heads=8, hidden=512, plain=False):
        super().__init__()
        from dcnv4_amd import FlashDeformAttn
        self.heads, self.plain = heads, plain
        self.in_proj, self.out_proj = nn.Linear(width, 3 * width), nn.Linear(width, width)
        self.slopes = nn.Parameter(torch.linspace(0.2, 4.0, heads))
        self.cross = FlashDeformAttn(width, len(LEVELS), heads, 4)
        self.fc1, self.fc2 = nn.Linear(width, hidden), nn.Linear(hidden, width)
        self.norm1, self.norm2, self.norm3 = (nn.LayerNorm(width) for _ in range(3))

    def add(self, x, residual, norm):
        from dcnv4_amd.functions import add_layer_norm
        return norm(x + residual) if self.plain else add_layer_norm(x, residual, norm)

    def forward(self, x, segments, points, memory, shapes, starts):
        from dcnv4_amd.functions import query_attention
        q, k, v = self.in_proj(x).unflatten(-1, (3, self.heads, -1)).unbind(2)
        if self.plain:
            mixed = plain_attention(q, k, v, segments, points, self.slopes, 20.0)
        else:
            mixed = query_attention(q, k, v, segments=segments, positions=points, slopes=self.slopes, cap=20.0)
        x = self.add(self.out_proj(mixed.flatten(2)), x, self.norm1)
        reference = points[:, :, None].expand(-1, -1, len(LEVELS), -1)
        x = self.add(self.cross(x, reference, memory, shapes, starts), x, self.norm2)
        return self.add(self.fc2(torch.relu(self.fc1(x))), x, self.norm3)


def setting(seed=0, n=2, queries=130):
    gen = torch.Generator().manual_seed(seed)
    pixels = sum(h * w for h, w in LEVELS)
    segments = torch.zeros(n, queries, dtype=torch.int32)
    segments[:, :20], segments[:, 20:40] = 1, 2          # two groups of denoising queries before the matching ones
    segments[1, 120:] = -1                               # fewer queries in the second picture
    shapes = torch.tensor(LEVELS)
    starts = torch.cat((shapes.new_zeros(1), shapes.prod(1).cumsum(0)[:-1]))
    t = dict(x=torch.randn(n, queries, 256, generator=gen), segments=segments, points=torch.rand(n, queries, 2, generator=gen),
             memory=torch.randn(n, pixels, 256, generator=gen), shapes=shapes, starts=starts)
    return {name: v.cuda() for name, v in t.items()}, torch.randn(n, queries, 256, generator=gen).cuda()


def run(layer, t, grad, amp=None):
    t = dict(t, x=t["x"].clone().requires_grad_(), memory=t["memory"].clone().requires_grad_())
    with torch.autocast("cuda", dtype=amp or torch.float16, enabled=amp is not None):
        out = layer(**t)
    names = ["x", "memory"] + [n for n, _ in layer.named_parameters()]
    return out.detach(), dict(zip(names, torch.autograd.grad(out, [t["x"], t["memory"], *layer.parameters()], grad.to(out.dtype))))


def test_the_layer_and_its_gradients():
    torch.manual_seed(1)
    own = Layer().cuda()
    plain = Layer(plain=True).cuda()
    plain.load_state_dict(own.state_dict())
    t, grad = setting()
    out, grads = run(own, t, grad)
    want, want_grads = run(plain, t, grad)
    # fp32 throughout, products of depth 512 at most: some hundred roundings of 2^-24 of sums that may cancel by a factor of ten
    far = lambda a, b: ((a - b).norm() / b.norm()).item()
    assert far(out, want) < 1e-4
    for name in grads:
        assert far(grads[name], want_grads[name]) < 1e-3, name


@pytest.mark.parametrize("amp", (torch.float16, torch.bfloat16), ids=("fp16", "bf16"))
def test_the_layer_in_mixed_precision(amp):
    torch.manual_seed(1)
    own = Layer().cuda()
    t, grad = setting(seed=3)
    out, grads = run(own, t, grad, amp)
    want, want_grads = run(own, t, grad)
    assert out.dtype == torch.float32          # torch's layer norm under autocast
    # five products and two attentions in a row, each a rounding or two of 16 bits of what goes in and comes out; the bf16 roundings of a
    # sampling point's logits show most, and of the loss's gradient through three norms
    limit = 20 * {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[amp]
    far = lambda a, b: ((a.float() - b).norm() / b.norm()).item()
    assert far(out, want) < limit
    for name in grads:
        assert torch.isfinite(grads[name]).all() and grads[name].dtype == want_grads[name].dtype
        assert far(grads[name], want_grads[name]) < 4 * limit, name


def test_steps_of_training_run():
    torch.manual_seed(2)
    layer = Layer().cuda()
    start = {n: p.detach().clone() for n, p in layer.named_parameters()}
    t, grad = setting(seed=5)
    optimiser = torch.optim.SGD(layer.parameters(), lr=1e-3)
    # the forward pass adds in one order; the sampling attention's backward, in fp32 with few queries, in any, so the steps' ends are not compared
    assert torch.equal(run(layer, t, grad)[0], run(layer, t, grad)[0])
    for _ in range(3):
        out, grads = run(layer, t, grad)
        for name, p in layer.named_parameters():
            p.grad = grads[name]
        optimiser.step()
    assert torch.isfinite(out).all()
    for name, p in layer.named_parameters():
        assert torch.isfinite(p).all() and (not grads[name].any() or not torch.equal(p, start[name])), name
