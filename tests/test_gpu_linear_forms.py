"""Linear layers at sizes whose products take the large forms (ln_plan's model of them, in csrc/linear.hip): tiles that go to LDS
directly of 128x128, 128x256 and 256x256, and float's of 128x128; both layouts of the weight and of its gradient, depths of several
steps that end inside one, operands between NaN, results between values that stay."""
import pytest
import torch

from tdgs_amd import decoder

pytestmark = pytest.mark.gpu

# rows, in, out: the forms of the forward product, dx and dweight
HALF = {
    "128x128 128x128 64x64": (20008, 264, 264),        # depths of 264: four steps of 64 and 8 more
    "128x256 64x64 64x64": (3000, 264, 2056),          # eight steps of 32 and 8 more
    "256x256 128x64 128x128": (6000, 1544, 2056),      # 24 steps and 8 more; 6000 rows: 93 steps and 48 in two splits
    "128x64 256x256 128x128": (6000, 2056, 1544),
    "128x64 128x64 256x256": (4100, 2056, 2056),       # 64 steps and 4 more, in three splits
    "64x64 64x64 128x256": (140, 1032, 4104),          # four steps of 32 and 12 more
}
FLOAT = {
    "128x128 64x64 64x64": (5001, 133, 2052),          # eight steps of 16 and 5 more
    "64x64 128x128 64x64": (5001, 2052, 133),
    "64x64 64x64 128x128": (4100, 1028, 2052),         # 256 steps and 4 more, in five splits
}
NAN, MARK = float("nan"), 77.0


def around(rows, cols, value, t, seed=None):
    """A matrix whose rows start on 16 bytes, inside a buffer of `value`, and the buffer."""
    big = torch.full((rows + 4, -(-cols // 8) * 8 + 16), value, dtype=t, device="cuda")
    view = big[2:rows + 2, 8:cols + 8]
    if seed is not None:
        view.copy_(torch.randn((rows, cols), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))
    return view, big


def close(got, want, t, steps, extra):
    """Relative error over the tensor: `steps` roundings to the type, each half a step at most, and `extra`."""
    error, norm = (got.double() - want).norm(), want.norm()
    assert error <= (steps * torch.finfo(t).eps / 2 + extra) * norm, (error / norm).item()


def check(t, size, layout, act):
    m, k, n = size
    x, dout, res = around(m, k, NAN, t, 1)[0], around(m, n, NAN, t, 3)[0], around(m, n, NAN, t, 4)[0]
    w = around(k, n, NAN, t, 2)[0] if layout == "in_out" else around(n, k, NAN, t, 2)[0].T
    w.mul_(k ** -0.5)
    bias = torch.randn(n, generator=torch.Generator().manual_seed(5)).to(t).cuda()
    outs = {"out": (m, n), "pre": (m, n), "dx": (m, k), "dw": (k, n), "dwt": (n, k)}
    outs = {name: around(*shape, MARK, t) for name, shape in outs.items()}
    out, pre, dx, dw, dwt = (view for view, _ in outs.values())
    db = torch.empty_like(bias)
    kw = {"activation": act, "pre": pre if act != "identity" else None}
    decoder.linear_(out, x, w, bias, residual=res, **kw)
    decoder.linear_grad_(dx, dw, db, dout, x, w, **kw)
    decoder.linear_grad_(None, dwt.T, None, dout, x, w, **kw)
    for name, (view, big) in outs.items():
        copy = view.clone()
        view.fill_(MARK)
        assert (big == MARK).all(), name
        view.copy_(copy)
    z = x.double() @ w.double() + bias.double()
    sg = torch.sigmoid(z)
    y, dz = (z, dout.double()) if act == "identity" else (z * sg, dout.double() * sg * (1 + z * (1 - sg)))
    # out: rounded once, sums of 32 bits (up to sqrt(depth) half steps of 2^-24 on average, taken four times over). Gradients
    # with a slope: pre rounded (act'' is below 1, z on average below 2), dz and the result rounded
    steps = 1 if act == "identity" else 4

    def sums(depth):
        return 4 * depth ** 0.5 * 2.0 ** -24
    close(out, y + res.double(), t, 1, sums(k))
    close(dx, dz @ w.double().T, t, steps, sums(n) + sums(k))
    want = x.double().T @ dz
    close(dw, want, t, steps, sums(m) + sums(k))
    close(dwt.T, want, t, steps, sums(m) + sums(k))
    close(db, dz.sum(0), t, steps, 4 * sums(m) + sums(k))


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("layout", ["in_out", "out_in"])
@pytest.mark.parametrize("size", HALF, ids=str)
def test_half(gpu, t, layout, size):
    check(t, HALF[size], layout, "identity")
    check(t, HALF[size], layout, "silu")


@pytest.mark.parametrize("layout", ["in_out", "out_in"])
@pytest.mark.parametrize("size", FLOAT, ids=str)
def test_float(gpu, layout, size):
    check(torch.float32, FLOAT[size], layout, "silu")


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [*HALF.values(), (5001, 133, 2052), (4, 96, 40), (1, 520, 64), (3, 40, 37), (700, 512, 33), (64, 4096, 48)], ids=str)
def test_residual_in_place(gpu, t, size):
    """residual = out in every epilogue (few rows, joined splits, tiles through registers and directly, outputs that divide by
    eight or not): the bits of the call with a result of its own."""
    m, k, n = size
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, w, r = (torch.randn(s, generator=gen, device="cuda").to(t) for s in ((m, k), (k, n), (m, n)))
    for act in ("identity", "gelu"):
        want = torch.empty_like(r)
        decoder.linear_(want, x, w / k ** 0.5, residual=r, activation=act)
        y = x.double() @ (w / k ** 0.5).double()
        y = y if act == "identity" else 0.5 * y * torch.erfc(-y * 0.5 ** 0.5)
        close(want, y + r.double(), t, 1, 4 * k ** 0.5 * 2.0 ** -24 + 2.0 ** -20)
        got = r.clone()
        decoder.linear_(got, x, w / k ** 0.5, residual=got, activation=act)
        assert torch.equal(got, want)


@pytest.mark.parametrize("size", [(6000, 2056, 1544), (20008, 264, 264)], ids=str)
def test_the_same_bits_every_time(gpu, size):
    t = torch.bfloat16
    m, k, n = size
    gen = torch.Generator(device="cuda").manual_seed(7)
    x, w, dout = (torch.randn(s, generator=gen, device="cuda").to(t) for s in ((m, k), (k, n), (m, n)))
    results = []
    for _ in range(3):
        out, dx, dw = torch.empty_like(dout), torch.empty_like(x), torch.empty_like(w)
        decoder.linear_(out, x, w)
        decoder.linear_grad_(dx, dw, None, dout, x, w)
        results.append((out, dx, dw))
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))
