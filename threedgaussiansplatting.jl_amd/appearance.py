"""A learned decoder of rendered images: the appearance of each photograph of a collection.

Photographs of one scene differ in exposure, white balance and weather; a model trained on them directly
bakes the differences into its Gaussians. AppearanceDecoder stands between the rendered image and the
loss: it looks up the photograph's embedding tokens, lets the image's patches attend them (and, where
given, an encoder's states of a reference photograph) and corrects each patch's colours by a gain
and an offset. It puts the operators of decoder.py together: embedding, group norm with SiLU (channels
last, the layout images are rendered in) and cross attention; by option also norms of queries and keys with a
rotation by position, a feed-forward layer and dropout, whose linear layers are decoder.py's too. The other linear
layers are plain matrix products. The reference has no counterpart.
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
    features between float32 parameters. states_dim, where not 0, is the width of an encoder's states.

    rotary norms each head's queries and keys and rotates them by position: patches by their column and row in half
    of a head's pairs each, an encoder's states by what a call gives, tokens not at all, so that a photograph's
    correction can depend on the place in the image (vignetting). feed_forward, where not 0, is the width of a layer with GELU
    behind the attention. dropout is the probability with which training passes drop what attention and that layer add."""

    def __init__(self, nb_images, channels=64, heads=4, groups=8, tokens=4, patch=4, states_dim=0,
                 dtype=torch.float32, seed=0, device=0, rotary=False, feed_forward=0, dropout=0.0):
        if channels % heads or channels % groups:
            raise ValueError(f"{channels} channels do not divide into {heads} heads and {groups} groups")
        if rotary and channels // heads < 4:
            raise ValueError(f"heads of {channels // heads} channels cannot be rotated on two axes")
        if not 0 <= dropout < 1:
            raise ValueError(f"dropout of {dropout}")
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
        self.rotary = decoder.Rotary((c // heads // 4,) * 2, base=100.0, device=device) if rotary else None
        if rotary:
            self.parameters.update(query_norm=torch.ones(c // heads, device=d), key_norm=torch.ones(c // heads, device=d))
        if feed_forward:
            self.parameters.update(
                norm3_weight=torch.ones(c, device=d), norm3_bias=torch.zeros(c, device=d),
                forward_in=weight(c, feed_forward), forward_in_bias=torch.zeros(feed_forward, device=d),
                forward_out=weight(feed_forward, c), forward_out_bias=torch.zeros(c, device=d))
        for p in self.parameters.values():
            p.requires_grad_(True)
        self.dropout, self.seed = dropout, seed
        self.passes = torch.zeros(1, dtype=torch.int64, device=d)   # training passes, whose masks differ

    def _patch_places(self, pw, ph):
        """Column and row of each of pw x ph patches, made on the call's own stream or in its own graph."""
        at = (torch.arange(n, dtype=torch.int32, device=self.device) for n in (pw, ph))
        return torch.stack(torch.meshgrid(*at, indexing="ij"), dim=2).reshape(pw * ph, 2)

    def _add(self, x, y, weight, bias, layer, train):
        """x + y weight + bias, the sum's second part dropped in training."""
        p = self.parameters
        bias = None if bias is None else p[bias].to(y.dtype)
        if not (train and self.dropout):
            return decoder.linear(y, p[weight].to(y.dtype), bias, residual=x)
        return decoder.dropout(decoder.linear(y, p[weight].to(y.dtype), bias), self.dropout, 2 * self.seed + layer,
                               call=self.passes, residual=x)

    def __call__(self, rgb, image, states=None, *, states_positions=None, train=False):
        """The corrected (w, h, 3) float32 image of the rendered one, as photograph `image` of the collection
        shows it; states (length, states_dim) are an encoder's, states_positions (length, 2; with rotary) their
        columns and rows, in patches (without them all at 0, as the tokens). train: with dropout. Differentiable for rgb and
        the parameters."""
        if not isinstance(image, torch.Tensor) and not 0 <= image < self.nb_images:
            raise ValueError(f"photograph {image} of a collection of {self.nb_images}")
        if states_positions is not None:
            if self.rotary is None or states is None:
                raise ValueError(f"states_positions without {'rotary' if self.rotary is None else 'states'}")
            if states_positions.shape != (states.shape[0], 2):
                raise ValueError(f"states_positions have shape {tuple(states_positions.shape)}, not ({states.shape[0]}, 2)")
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
        q, k = heads(q[0], p["query"]), heads(known, p["key"])
        if self.rotary is not None:
            places = torch.zeros((known.shape[0], 2), device=rgb.device)   # (whole columns and rows, or between them)
            if states_positions is not None:
                places[self.tokens:] = states_positions
            q = decoder.head_norm(q, None, p["query_norm"], rotary=self.rotary, positions=self._patch_places(pw, ph))
            k = decoder.head_norm(k, None, p["key_norm"], rotary=self.rotary, positions=places)
        a = decoder.cross_attention(q, k, heads(known, p["value"])).reshape(1, pw * ph, c)
        if self.dropout or self.rotary is not None or "forward_in" in p:
            x = self._add(x, a, "attention_out", None, 0, train)
        else:
            x = x + torch.mm(a[0], p["attention_out"].to(self.dtype))
        if "forward_in" in p:
            y = decoder.group_norm(x, self.groups, p["norm3_weight"], p["norm3_bias"], activation="identity")
            y = decoder.linear(y, p["forward_in"].to(self.dtype), p["forward_in_bias"].to(self.dtype), activation="gelu")
            x = self._add(x, y, "forward_out", "forward_out_bias", 1, train)
        if train and self.dropout:
            self.passes.add_(1)
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

    def step_(self, decoder_, optimizer, rgb, image, photograph, states=None, states_positions=None):
        """One step of the decoder's parameters on a rendered image, with states and their positions as the decoder takes
        them; returns the loss's gradient for that image, from which the render's backward pass goes on. The loss's sums
        stay on the device (value())."""
        rgb = rgb.detach().requires_grad_(True)
        optimizer.zero_grad(set_to_none=True)
        options = {"train": True} if getattr(decoder_, "dropout", 0.0) else {}
        if states_positions is not None:
            options["states_positions"] = states_positions
        corrected = decoder_(rgb, image, states, **options).contiguous()
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
