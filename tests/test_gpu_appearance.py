"""The decoder of rendered images that puts embedding, group norm and cross attention together: its
gradients against differences, and training on photographs of different exposure, on rendered images."""
import pytest
import torch

from tdgs_amd import appearance, decoder, host, synthetic

pytestmark = pytest.mark.gpu


def test_differentiable_functions_against_torch(gpu):
    """The three functions under torch's differentiation against the same formulas in 64 bits: relative errors of
    float32 chains of a few hundred additions, far below 1e-4."""
    gen = torch.Generator().manual_seed(0)

    def leaf(*shape):
        return torch.randn(shape, generator=gen).cuda().requires_grad_(True)

    table, wk, x = leaf(10, 32), leaf(32, 32), leaf(1, 50, 32)
    tokens = torch.tensor([1, 3, 3, 9, 0, 3], device="cuda")
    weight, bias = leaf(32), leaf(32)
    coef = torch.randn((1, 50, 4, 8), generator=gen).cuda()
    known = decoder.embedding(table, tokens, scale=2.0) @ wk * 0.2
    q = decoder.group_norm(x, 4, weight, bias, activation="gelu").reshape(1, 50, 4, 8)
    kv = known.reshape(1, 6, 4, 8)
    out = decoder.cross_attention(q, kv, kv)
    grads = torch.autograd.grad((out * coef).sum(), (table, wk, x, weight, bias))
    leaves = [t.detach().double().requires_grad_(True) for t in (table, wk, x, weight, bias)]
    t2, wk2, x2, w2, b2 = leaves
    kv2 = (t2[tokens] * 2.0 @ wk2 * 0.2).reshape(6, 4, 8)
    g = x2.reshape(50, 4, 8)
    g = (g - g.mean(dim=(0, 2), keepdim=True)) / torch.sqrt(g.var(dim=(0, 2), unbiased=False, keepdim=True) + 1e-5)
    q2 = torch.nn.functional.gelu(g.reshape(50, 32) * w2 + b2).reshape(50, 4, 8)
    p = torch.softmax(torch.einsum("ihd,jhd->hij", q2, kv2) * 8 ** -0.5, dim=2)
    want_out = torch.einsum("hij,jhd->ihd", p, kv2)
    assert (out[0].double() - want_out).norm() <= 1e-4 * want_out.norm()
    for a, b in zip(grads, torch.autograd.grad((want_out * coef[0].double()).sum(), leaves)):
        assert (a.double() - b).norm() <= 1e-4 * b.norm()


@pytest.mark.parametrize("states", [False, True], ids=["tokens", "states"])
def test_gradients_against_differences(gpu, states):
    """Central differences of step 2^-6 along unit directions: their error is the third derivative's share, below
    1e-2 of the gradient's norm."""
    gen = torch.Generator().manual_seed(1)
    dec = appearance.AppearanceDecoder(3, channels=32, groups=4, states_dim=20 if states else 0)
    dec.parameters["colour_out"].data.mul_(10)
    rgb = torch.rand((33, 22, 3), generator=gen).cuda()
    known = torch.randn((7, 20), generator=gen).cuda() if states else None
    coef = torch.randn((33, 22, 3), generator=gen).cuda()
    x = rgb.clone().requires_grad_(True)
    (dec(x, 1, known) * coef).sum().backward()
    leaves = dict(dec.parameters, rgb=x)
    with torch.no_grad():
        for name, leaf in leaves.items():
            value = leaf.data.clone()
            d = torch.randn(leaf.shape, generator=gen).cuda()
            d /= d.norm()
            f = []
            for sign in (1, -1):
                leaf.data.copy_(value + sign * 2.0 ** -6 * d)
                f.append((dec(x, 1, known).double() * coef).sum())
            leaf.data.copy_(value)
            want = (f[0] - f[1]) * 2.0 ** 5
            assert abs((leaf.grad.double() * d.double()).sum() - want) <= 1e-2 * leaf.grad.double().norm(), name
    table = dec.parameters["table"].grad.reshape(3, 4, 32)
    assert not table[0].any() and table[1].any() and not table[2].any()   # only the photograph's own tokens


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_learns_the_photographs_exposure(gpu, dtype):
    """Photographs are renders of another exposure and tint each: the decoder learns them, to a fifth of the loss at
    the start, and the gradient that reaches the rendered image is finite and not zero."""
    w = synthetic.config(3, n=20000, cameras=3)
    g = gpu.TrainableGaussiansVector.from_host(w.gaussians, 0)
    gen = torch.Generator().manual_seed(2)
    renders, photographs = [], []
    for cam in w.cameras[:3]:
        t = host.Tiling.for_camera(cam, 16, 16)
        out = gpu.RenderOutputs.for_camera(cam, 0)
        options = host.RenderOptions.for_camera(cam, w.gaussians.sh_degree, background_color=(0.3, 0.3, 0.3))
        gpu.render_(out, g, cam, t, options, gpu.RenderBuffers(len(g), t, 0))
        renders.append(out.rgb)
        photographs.append(out.rgb * (0.6 + torch.rand(3, generator=gen)).cuda() + 0.1 * torch.rand(3, generator=gen).cuda())
    dec = appearance.AppearanceDecoder(3, dtype=dtype)
    optimizer = dec.optimizer(3e-3)
    loss = appearance.AppearanceLoss(renders[0].shape[0], renders[0].shape[1])
    first = last = 0.0
    for it in range(150):
        grad = loss.step_(dec, optimizer, renders[it % 3], it % 3, photographs[it % 3])
        if it < 3:
            first += loss.value() / 3
        if it >= 147:
            last += loss.value() / 3
    assert torch.isfinite(grad).all() and grad.any()
    assert last < first / 5, (first, last)
