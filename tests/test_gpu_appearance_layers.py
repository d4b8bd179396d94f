"""The decoder of rendered images with its options, which run linear layers, head norms with rotation and dropout together
with attention, group norm and embedding: against the same formulas in 64 bits, gradients against differences, and training."""
import pytest
import torch

from tdgs_amd import appearance, decoder

pytestmark = pytest.mark.gpu


def make(dtype=torch.float32, dropout=0.0, states_dim=12):
    dec = appearance.AppearanceDecoder(3, channels=32, heads=2, groups=4, states_dim=states_dim, dtype=dtype, rotary=True,
                                       feed_forward=48, dropout=dropout, seed=5)
    gen = torch.Generator().manual_seed(9)
    for name, p in dec.parameters.items():   # nothing at its starting ones and zeros
        p.data.add_(0.2 * torch.randn(p.shape, generator=gen).cuda())
    return dec


def inputs():
    gen = torch.Generator().manual_seed(1)
    rgb = torch.rand((33, 22, 3), generator=gen).cuda()
    states = torch.randn((7, 12), generator=gen).cuda()
    return rgb, states, torch.randint(0, 9, (7, 2), generator=gen).cuda().float() + 0.25, \
        torch.randn((33, 22, 3), generator=gen).cuda()


def in_64_bits(dec, rgb, image, states, places):
    p = {k: v.detach().double().requires_grad_(True) for k, v in dec.parameters.items()}
    rgb = rgb.double().requires_grad_(True)
    s, c, h = dec.patch, dec.channels, dec.heads
    w, ht, _ = rgb.shape
    pw, ph = -(-w // s), -(-ht // s)
    x = torch.nn.functional.pad(rgb, (0, 0, 0, ph * s - ht, 0, pw * s - w))
    x = x.reshape(pw, s, ph, s, 3).permute(0, 2, 1, 3, 4).reshape(pw * ph, -1) @ p["patch_in"]

    def norm(y, i, act):
        y = y.reshape(pw * ph, dec.groups, -1)
        y = (y - y.mean((0, 2), keepdim=True)) / torch.sqrt(y.var((0, 2), unbiased=False, keepdim=True) + 1e-5)
        y = y.reshape(pw * ph, c) * p[f"norm{i}_weight"] + p[f"norm{i}_bias"]
        return y * torch.sigmoid(y) if act else y

    def turn(y, weight, at):
        y = y.reshape(-1, h, c // h)
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight
        n = dec.rotary.pairs
        f = torch.tensor([100.0 ** (-j / (n // 2)) for j in range(n // 2)], dtype=torch.float64, device="cuda")
        angle = torch.cat([at[:, :1].double() * f, at[:, 1:].double() * f], 1)[:, None]
        a, b = y[..., :n], y[..., n:2 * n]
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), y[..., 2 * n:]], -1)

    known = p["table"][image * dec.tokens:(image + 1) * dec.tokens] * c ** 0.5
    known = torch.cat([known, states.double() @ p["states_in"]])
    at = torch.cartesian_prod(torch.arange(pw), torch.arange(ph)).cuda()
    q = turn(norm(x, 1, True) @ p["query"], p["query_norm"], at)
    k = turn(known @ p["key"], p["key_norm"], torch.cat([torch.zeros(dec.tokens, 2).cuda(), places]))
    v = (known @ p["value"]).reshape(-1, h, c // h)
    a = torch.stack([torch.softmax(q[:, i] @ k[:, i].T * (c // h) ** -0.5, 1) @ v[:, i] for i in range(h)], 1)
    x = x + a.reshape(pw * ph, c) @ p["attention_out"]
    y = norm(x, 3, False) @ p["forward_in"] + p["forward_in_bias"]
    x = x + 0.5 * y * torch.erfc(-y * 0.5 ** 0.5) @ p["forward_out"] + p["forward_out_bias"]
    gain, offset = (norm(x, 2, True) @ p["colour_out"]).reshape(pw, ph, 6).split(3, dim=2)
    gain, offset = (t.repeat_interleave(s, 0).repeat_interleave(s, 1)[:w, :ht] for t in (gain, offset))
    return rgb * (1 + gain) + offset, dict(p, rgb=rgb)


def test_against_64_bits(gpu):
    """Chains of some hundred operations in float32, each to 2^-23 or so of what it adds up: far below 1e-4."""
    dec = make()
    rgb, states, places, coef = inputs()
    x = rgb.clone().requires_grad_(True)
    out = dec(x, 1, states, states_positions=places)
    want, leaves = in_64_bits(dec, rgb, 1, states, places)
    assert (out - want).norm() <= 1e-4 * want.norm()
    (out * coef).sum().backward()
    grads = torch.autograd.grad((want * coef).sum(), list(leaves.values()))
    for (name, _), g in zip(leaves.items(), grads):
        got = x.grad if name == "rgb" else dec.parameters[name].grad
        assert (got - g).norm() <= 1e-4 * g.norm(), name


@pytest.mark.parametrize("dropout", [0.0, 0.3])
def test_gradients_against_differences(gpu, dropout):
    """Central differences of step 2^-7 along unit directions, with the masks of one pass."""
    dec = make(dropout=dropout)
    rgb, states, places, coef = inputs()

    def value():
        dec.passes.fill_(4)
        return (dec(x, 2, states, states_positions=places, train=True).double() * coef).sum()

    x = rgb.clone().requires_grad_(True)
    value().backward()
    gen = torch.Generator().manual_seed(3)
    with torch.no_grad():
        for name, leaf in dict(dec.parameters, rgb=x).items():
            before = leaf.data.clone()
            d = torch.randn(leaf.shape, generator=gen).cuda()
            d /= d.norm()
            f = []
            for sign in (1, -1):
                leaf.data.copy_(before + sign * 2.0 ** -7 * d)
                f.append(value())
            leaf.data.copy_(before)
            want = (f[0] - f[1]) * 2.0 ** 6
            assert abs((leaf.grad.double() * d.double()).sum() - want) <= 1e-2 * leaf.grad.double().norm(), name


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_trains(gpu, dtype):
    dec = make(dtype, dropout=0.2, states_dim=0)
    rgb = inputs()[0]
    optimizer, loss = dec.optimizer(1e-3), appearance.AppearanceLoss(33, 22)
    before = {k: v.detach().clone() for k, v in dec.parameters.items()}
    for i in range(3):
        grad = loss.step_(dec, optimizer, rgb, i, rgb * 0.5)
        assert torch.isfinite(grad).all() and grad.any()
    assert int(dec.passes) == 3
    for k, v in dec.parameters.items():
        assert torch.isfinite(v).all() and not torch.equal(v, before[k]), k
    with torch.no_grad():
        a, b = dec(rgb, 0), dec(rgb, 0)
        c, d = dec(rgb, 0, train=True), dec(rgb, 0, train=True)
    assert torch.equal(a, b) and not torch.equal(c, d)


def test_options_leave_the_others_parameters(gpu):
    plain = appearance.AppearanceDecoder(3, seed=2).parameters
    more = appearance.AppearanceDecoder(3, seed=2, rotary=True, feed_forward=64, dropout=0.1).parameters
    for k, v in plain.items():
        assert torch.equal(v, more[k]), k


def test_block_in_a_graph(gpu):
    """Norms, attention, linear layers and dropout of a decoder's block captured together: each replay, with eager work and
    another call's mask between, is the eager block's result."""
    gen = torch.Generator().manual_seed(4)
    c, h, n = 64, 4, 300
    t = torch.bfloat16

    def rand(*shape):
        return torch.randn(shape, generator=gen).to(t).cuda()

    x, qkv, w_out, w_in, w_back = rand(1, n, c), rand(c, 3 * c) * 0.1, rand(c, c) * 0.1, rand(c, 256) * 0.1, rand(256, c) * 0.1
    bias, wq, wk = rand(256), 1 + 0.1 * rand(c // h).float(), 1 + 0.1 * rand(c // h).float()
    rotary, call = decoder.Rotary((4, 4)), torch.zeros(1, dtype=torch.int64, device="cuda")
    places = torch.randint(0, 40, (n, 2), generator=gen).cuda()
    fused, hidden, out = rand(1, n, 3 * c), rand(1, n, 256), rand(1, n, c)
    q, k, v = fused.reshape(1, n, 3, h, c // h).unbind(2)
    a = torch.empty((1, n, h, c // h), dtype=t, device="cuda")
    temps = (decoder.linear_temp(x, qkv), decoder.cross_attention_temp(q, k), decoder.linear_temp(x, w_out),
             decoder.linear_temp(x, w_in), decoder.linear_temp(hidden, w_back))

    def block():
        decoder.linear_(fused, x, qkv, temp=temps[0])
        decoder.head_norm_(q, k, q, k, wq, wk, rotary=rotary, positions=places)
        decoder.cross_attention_(a, q, k, v, temp=temps[1])
        decoder.linear_(out, a.reshape(1, n, c), w_out, residual=x, temp=temps[2])
        decoder.linear_(hidden, out, w_in, bias, activation="gelu", temp=temps[3])
        decoder.dropout_(hidden, hidden, 0.1, 3, call=call)
        decoder.linear_(out, hidden, w_back, residual=out, temp=temps[4])

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        block()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block()
        call.add_(1)
    for i in range(3):
        x.copy_(rand(1, n, c))
        call.fill_(i)
        block()
        want = out.clone()
        torch.cuda.synchronize()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
