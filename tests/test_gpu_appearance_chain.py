"""From the Gaussians through render, decoder and loss and back: the gradient that AppearanceLoss.step_ returns goes on into
backward_."""
import pytest
import torch

from tdgs_amd import appearance, host, synthetic

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("states", [False, True], ids=["tokens", "states"])
def test_colours_against_differences(gpu, states):
    """The loss's derivative for every Gaussian's colour in a channel (the constant harmonic, whose sum over the Gaussians
    backward_ gives) against central differences of the whole chain, step 2^-6: the colour moves by 0.28 of that, the
    L1 loss's kinks and the third derivatives leave less than 2% of the gradient's norm."""
    w = synthetic.config(0, n=3000)
    cam, degree = w.cameras[0], w.gaussians.sh_degree
    g = gpu.TrainableGaussiansVector.from_host(w.gaussians, 0)
    t = host.Tiling.for_camera(cam, 16, 16)
    options = host.RenderOptions.for_camera(cam, degree, background_color=(0.4, 0.4, 0.4))
    out, buf = gpu.RenderOutputs.for_camera(cam, 0), gpu.RenderBuffers(len(g), t, 0)
    dec = appearance.AppearanceDecoder(2, channels=32, groups=4, states_dim=12 if states else 0)
    dec.parameters["colour_out"].data.mul_(5)
    known = torch.randn((9, 12), generator=torch.Generator().manual_seed(1)).cuda() if states else None
    loss = appearance.AppearanceLoss(*out.rgb.shape[:2])
    frozen = torch.optim.SGD(dec.parameters.values(), lr=0.0)

    def step():
        gpu.render_(out, g, cam, t, options, buf)
        return loss.step_(dec, frozen, out.rgb, 1, photograph, known)

    gpu.render_(out, g, cam, t, options, buf)
    photograph = (0.5 * out.rgb + 0.1 * torch.rand(out.rgb.shape, generator=torch.Generator().manual_seed(2)).cuda()).contiguous()
    rgb_grad = step()
    fg = gpu.FilteredGaussiansGradientsVector(buf.capacity, degree, 0)
    gpu.backward_(fg, rgb_grad, out, g, cam, t, options, buf)
    got = fg.sh[:buf.nb_fgaussians, :, 0].double().sum(dim=0).cpu()
    want = []
    for c in range(3):
        values, sh = [], g.sh.clone()
        for sign in (1, -1):
            g.sh[:, c, 0] = sh[:, c, 0] + sign * 2.0 ** -6
            step()
            values.append(loss.value())
        g.sh.copy_(sh)
        want.append((values[0] - values[1]) * 2.0 ** 5)
    want = torch.tensor(want, dtype=torch.float64)
    assert got.norm() > 1e-3
    assert (got - want).abs().max() <= 2e-2 * got.norm(), (got, want)
