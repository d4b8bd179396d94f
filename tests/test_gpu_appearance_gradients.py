"""Gradients through the appearance decoder with all its options, dropout among them: against the same formulas in 64 bits
under the same masks, and against differences along the gradient itself."""
import numpy as np
import pytest
import torch

from test_dropout_words import philox
from tdgs_amd import appearance

pytestmark = pytest.mark.gpu

P, SEED, PASS = 0.3, 5, 4


def make():
    dec = appearance.AppearanceDecoder(3, channels=32, heads=2, groups=4, states_dim=12, rotary=True, feed_forward=48, dropout=P, seed=SEED)
    gen = torch.Generator().manual_seed(9)
    for p in dec.parameters.values():   # nothing at its starting ones and zeros
        p.data.add_(0.2 * torch.randn(p.shape, generator=gen).cuda())
    return dec


def inputs():
    gen = torch.Generator().manual_seed(1)
    rgb, states = torch.rand((33, 22, 3), generator=gen).cuda(), torch.randn((7, 12), generator=gen).cuda()
    return rgb, states, torch.randint(0, 9, (7, 2), generator=gen).cuda().float() + 0.25, torch.randn((33, 22, 3), generator=gen).cuda()


def drop(y, layer):
    """In 64 bits, with the mask of the training pass."""
    low, by, seed = np.uint64(2 ** 32 - 1), np.uint64(32), 2 * SEED + layer
    i = np.arange((y.numel() + 3) // 4, dtype=np.uint64)
    words = philox((i & low, i >> by, np.full_like(i, PASS), np.zeros_like(i)), (seed, 0))
    keep = np.stack(words, 1).reshape(-1)[:y.numel()] >= np.uint64(int(P * 2.0 ** 32))
    return torch.where(torch.from_numpy(keep).cuda().reshape(y.shape), y / (1 - P), 0.0)


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
        n = c // h // 4
        f = torch.tensor([100.0 ** (-j / n) for j in range(n)], dtype=torch.float64, device="cuda")
        angle = torch.cat([at[:, :1].double() * f, at[:, 1:].double() * f], 1)[:, None]
        a, b = y[..., :2 * n], y[..., 2 * n:4 * n]
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), y[..., 4 * n:]], -1)

    known = p["table"][image * dec.tokens:(image + 1) * dec.tokens] * c ** 0.5
    known = torch.cat([known, states.double() @ p["states_in"]])
    at = torch.cartesian_prod(torch.arange(pw), torch.arange(ph)).cuda()
    q = turn(norm(x, 1, True) @ p["query"], p["query_norm"], at)
    k = turn(known @ p["key"], p["key_norm"], torch.cat([torch.zeros(dec.tokens, 2).cuda(), places]))
    v = (known @ p["value"]).reshape(-1, h, c // h)
    a = torch.stack([torch.softmax(q[:, i] @ k[:, i].T * (c // h) ** -0.5, 1) @ v[:, i] for i in range(h)], 1)
    x = x + drop(a.reshape(pw * ph, c) @ p["attention_out"], 0)
    y = norm(x, 3, False) @ p["forward_in"] + p["forward_in_bias"]
    x = x + drop(0.5 * y * torch.erfc(-y * 0.5 ** 0.5) @ p["forward_out"] + p["forward_out_bias"], 1)
    gain, offset = (norm(x, 2, True) @ p["colour_out"]).reshape(pw, ph, 6).split(3, dim=2)
    gain, offset = (t.repeat_interleave(s, 0).repeat_interleave(s, 1)[:w, :ht] for t in (gain, offset))
    return rgb * (1 + gain) + offset, dict(p, rgb=rgb)


def test_against_64_bits_under_the_same_masks(gpu):
    """Chains of some hundred operations in float32, each to 2^-23 or so of what it adds up: far below 1e-4."""
    dec = make()
    rgb, states, places, coef = inputs()
    dec.passes.fill_(PASS)
    x = rgb.clone().requires_grad_(True)
    out = dec(x, 1, states, states_positions=places, train=True)
    want, leaves = in_64_bits(dec, rgb, 1, states, places)
    assert (out - want).norm() <= 1e-4 * want.norm()
    (out * coef).sum().backward()
    for (name, _), g in zip(leaves.items(), torch.autograd.grad((want * coef).sum(), list(leaves.values()))):
        got = x.grad if name == "rgb" else dec.parameters[name].grad
        assert (got - g).norm() <= 1e-4 * g.norm(), name


def test_differences_along_the_gradient(gpu):
    """Central differences along each leaf's own gradient, where they are as large as they can be: the gradient's norm. Steps of
    2^-7: terms of the third order are 2^-14 of a leaf's curvature, and float32's noise below 1e-3 of values of about 100."""
    dec = make()
    rgb, states, places, coef = inputs()

    def value():
        dec.passes.fill_(PASS)
        return (dec(x, 2, states, states_positions=places, train=True).double() * coef).sum()

    x = rgb.clone().requires_grad_(True)
    value().backward()
    with torch.no_grad():
        for name, leaf in dict(dec.parameters, rgb=x).items():
            before, norm = leaf.data.clone(), leaf.grad.double().norm()
            d = leaf.grad / leaf.grad.norm()
            f = []
            for sign in (1, -1):
                leaf.data.copy_(before + sign * 2.0 ** -7 * d)
                f.append(value())
            leaf.data.copy_(before)
            assert abs(norm - (f[0] - f[1]) * 2.0 ** 6) <= 1e-2 * norm, name
