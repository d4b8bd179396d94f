"""A learned decoder of rendered images: the appearance of each photograph of a collection.

Photographs of one scene differ in exposure, white balance and weather; a model trained on them directly
bakes the differences into its Gaussians. AppearanceDecoder stands between the rendered image and the
loss: it looks up the photograph's embedding tokens, lets the image's patches attend them (and, where
given, an encoder's states of a reference photograph) and corrects each patch's colours by a gain
and an offset. It puts the operators of decoder.py together: embedding, group norm with SiLU (channels
last, the layout images are rendered in) and cross attention; the linear layers between them are plain
matrix products. The reference has no counterpart.
"""
from __future__ import annotations

import torch

from . import decoder
from .core import _dev, lib
from .training import loss_grad_


class AppearanceDecoder:
    """Colour correction of rendered images by photograph.

    channels is split into `heads` heads and `groups` groups; every photograph has `tokens` embedding
    tokens; patch is the side of the square of pixels that shares a correction. dtype is the type of the
    features between float32 parameters. states_dim, where not 0, is the width of an encoder's states."""

    def __init__(self, nb_images, channels=64, heads=4, groups=8, tokens=4, patch=4, states_dim=0,
                 dtype=torch.float32, seed=0, device=0):
        if channels % heads or channels % groups:
            raise ValueError(f"{channels} channels do not divide into {heads} heads and {groups} groups")
        d = self.device = _dev(device)
        self.nb_images, self.channels, self.heads, self.groups = nb_images, channels, heads, groups
        self.tokens, self.patch, self.dtype = tokens, patch, dtype
        gen = torch.Generator(device=d)
        gen.manual_seed(seed)

        def weight(rows, cols, gain=1.0):
            return gain * rows ** -0.5 * torch.randn((rows, cols), generator=gen, device=d)

        c = channels
        self.parameters = {
            "table": torch.randn((nb_images * tokens, c), generator=gen, device=d) * c ** -0.5,
            "patch_in": weight(3 * patch * patch, c),
            "norm1_weight": torch.ones(c, device=d), "norm1_bias": torch.zeros(c, device=d),
            "query": weight(c, c), "key": weight(c, c), "value": weight(c, c), "attention_out": weight(c, c),
            "norm2_weight": torch.ones(c, device=d), "norm2_bias": torch.zeros(c, device=d),
            "colour_out": weight(c, 6, 0.1),
        }
        if states_dim:
            self.parameters["states_in"] = weight(states_dim, c)
        for p in self.parameters.values():
            p.requires_grad_(True)

    def __call__(self, rgb, image, states=None):
        """The corrected (w, h, 3) float32 image of the rendered one, as photograph `image` of the collection
        shows it; states (length, states_dim) are an encoder's. Differentiable for rgb and the parameters."""
        if not isinstance(image, torch.Tensor) and not 0 <= image < self.nb_images:
            raise ValueError(f"photograph {image} of a collection of {self.nb_images}")
        p, s, c = self.parameters, self.patch, self.channels
        w, h, _ = rgb.shape
        pw, ph = -(-w // s), -(-h // s)
        padded = torch.nn.functional.pad(rgb, (0, 0, 0, ph * s - h, 0, pw * s - w))
        patches = padded.reshape(pw, s, ph, s, 3).permute(0, 2, 1, 3, 4).reshape(pw * ph, 3 * s * s)
        x = torch.mm(patches, p["patch_in"]).to(self.dtype)[None]
        q = decoder.group_norm(x, self.groups, p["norm1_weight"], p["norm1_bias"])

        ids = image * self.tokens + torch.arange(self.tokens, device=rgb.device)
        known = decoder.embedding(p["table"], ids, scale=c ** 0.5)
        if states is not None:
            known = torch.cat([known, torch.mm(states, p["states_in"])])

        def heads(t, weight):
            return torch.mm(t, weight.to(t.dtype)).reshape(1, t.shape[0], self.heads, c // self.heads)

        known = known.to(self.dtype)
        a = decoder.cross_attention(heads(q[0], p["query"]), heads(known, p["key"]), heads(known, p["value"]))
        x = x + torch.mm(a.reshape(pw * ph, c), p["attention_out"].to(self.dtype))
        x = decoder.group_norm(x, self.groups, p["norm2_weight"], p["norm2_bias"])
        gain, offset = torch.mm(x[0].float(), p["colour_out"]).reshape(pw, ph, 6).split(3, dim=2)

        def pixels(t):
            return t.repeat_interleave(s, dim=0).repeat_interleave(s, dim=1)[:w, :h]

        return rgb * (1 + pixels(gain)) + pixels(offset)

    def optimizer(self, lr=1e-3):
        return torch.optim.Adam(self.parameters.values(), lr=lr)


class AppearanceLoss:
    """The training loss (L1 and D-SSIM, as the trainer's) of corrected images against photographs."""

    def __init__(self, width, height, dssim_weight=0.2, device=0):
        d = _dev(device)
        self.dssim_weight, self.pixels = dssim_weight, 3 * width * height
        self.sums = torch.zeros(2, dtype=torch.float64, device=d)
        self.temp = torch.empty(int(lib().tdgs_loss_temp_bytes(width, height)), dtype=torch.uint8, device=d)

    def step_(self, decoder_, optimizer, rgb, image, photograph, states=None):
        """One step of the decoder's parameters on a rendered image; returns the loss's gradient for that
        image, from which the render's backward pass goes on. The loss's sums stay on the device (value())."""
        rgb = rgb.detach().requires_grad_(True)
        optimizer.zero_grad(set_to_none=True)
        corrected = decoder_(rgb, image, states).contiguous()
        grad = torch.empty_like(corrected)
        self.sums.zero_()
        loss_grad_(corrected.detach(), photograph, grad, self.dssim_weight, self.sums, self.temp)
        corrected.backward(grad)
        optimizer.step()
        return rgb.grad

    def value(self):
        """The loss of the last step (synchronises)."""
        l1, ssim = self.sums.cpu().tolist()
        w = self.dssim_weight
        return (1 - w) * l1 / self.pixels + w * (1 - ssim / self.pixels)
