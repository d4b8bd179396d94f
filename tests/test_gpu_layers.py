"""Linear layers, head norms, rotations and dropout as a program uses them: under torch's differentiation, on streams and in
graphs, without elements, past 32-bit offsets, next to values that must not be read or written."""
import numpy as np
import pytest
import torch

from tdgs_amd import decoder

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0, t=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(t).cuda()


def near(a, b, error, step=0.0):
    """Within `error` relative to the tensor, and `step` for every element."""
    off = (a.double() - b.double()).norm()
    assert off <= error * b.double().norm() + step * a.numel() ** 0.5, (off / b.double().norm()).item()


def test_differentiable_functions_against_torch(gpu):
    """Chains of float32 operations whose sums are of a few hundred terms: far below 1e-5 each."""
    x, b, r = rand(4, 30, 24), rand(40, seed=2), rand(4, 40, 30, seed=3).transpose(1, 2)
    w = rand(33, 40, seed=1)[:24] * 0.2
    wq = 1 + 0.2 * rand(10, seed=4)
    coef = rand(4, 30, 4, 10, seed=5)
    rotary, places = decoder.Rotary((2, 3), pairs="interleaved"), torch.randint(0, 50, (30, 2), device="cuda")
    leaves = [v.detach().requires_grad_(True) for v in (x, w, b, r, wq)]
    y = decoder.linear(leaves[0].transpose(0, 1).transpose(0, 1), leaves[1], leaves[2], residual=leaves[3], activation="gelu")
    q = y.reshape(4, 30, 4, 10)
    q, k = decoder.head_norm(q, q[:, :, 1:3], leaves[4], None, rotary=rotary, positions=places)
    z = decoder.rotate(q, None, rotary, places, inverse=True)
    got = torch.autograd.grad((z * coef).sum() + (k * coef[:, :, :2]).sum(), leaves)

    same = [v.detach().double().requires_grad_(True) for v in leaves]
    a = same[0] @ same[1] + same[2]
    y2 = (same[3] + 0.5 * a * torch.erfc(-a * 0.5 ** 0.5)).reshape(4, 30, 4, 10)
    n = y2 / torch.sqrt((y2 * y2).mean(-1, keepdim=True) + 1e-6)
    f = torch.cat([10000.0 ** (-torch.arange(m, dtype=torch.float64, device="cuda") / m) for m in (2, 3)])
    angle = (places.double()[:, [0, 0, 1, 1, 1]] * f)[None, :, None]
    kk = n[:, :, 1:3]
    e, o = kk[..., 0::2], kk[..., 1::2]
    kk = torch.stack([e * angle.cos() - o * angle.sin(), e * angle.sin() + o * angle.cos()], -1).flatten(-2)
    near(z, n * same[4], 1e-5)
    near(k, kk, 1e-5)
    for g, h in zip(got, torch.autograd.grad((n * same[4] * coef).sum() + (kk * coef[:, :, :2]).sum(), same)):
        near(g, h, 1e-5)


def test_what_is_not_wanted_is_not_computed(gpu):
    """Frozen tensors, results that nothing depends on, single results."""
    x, w, b = rand(7, 8), rand(8, 16, seed=1), rand(16, seed=2)
    for frozen in range(3):
        leaves = [v.detach().requires_grad_(i != frozen) for i, v in enumerate((x, w, b))]
        out = decoder.linear(*leaves, activation="silu")
        out.backward(torch.ones_like(out))
        z = (x @ w + b).double()
        dz = torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z)))
        for i, want in enumerate((dz @ w.double().T, x.double().T @ dz, dz.sum(0))):
            assert (leaves[i].grad is None) == (i == frozen)
            if i != frozen:
                near(leaves[i].grad, want, 1e-5)
    r = rand(7, 16, seed=3).requires_grad_(True)
    out = decoder.linear(x, w, b, residual=r, activation="silu")
    out.backward(torch.ones_like(out))
    assert torch.equal(r.grad, torch.ones_like(r))
    q, k = rand(2, 3, 4, 8).requires_grad_(True), rand(2, 3, 4, 8, seed=1).requires_grad_(True)
    decoder.head_norm(q, k)[0].sum().backward()   # k's result is not used
    assert not k.grad.any() and torch.isfinite(q.grad).all()
    assert decoder.head_norm(q[0, 0, 0].reshape(1, 1, 1, 8)).shape == (1, 1, 1, 8)


@pytest.mark.parametrize("name", ["linear", "head_norm", "rotate", "dropout"])
@pytest.mark.parametrize("constant", [False, True])
def test_second_derivatives_raise(gpu, name, constant):
    x = rand(1, 3, 2, 8).requires_grad_(True)
    rotary, places = decoder.Rotary((4,)), torch.arange(3, device="cuda")[:, None]
    y = {"linear": lambda: decoder.linear(x, rand(8, 8), activation="silu"), "head_norm": lambda: decoder.head_norm(x),
         "rotate": lambda: decoder.rotate(x, None, rotary, places), "dropout": lambda: decoder.dropout(x, 0.5, 1)}[name]()
    g, = torch.autograd.grad((y * (1.0 if constant else y)).sum(), x, create_graph=True)
    if g.requires_grad:   # (a linear operator's gradient does not depend on x where dout is constant)
        with pytest.raises(RuntimeError, match="differentiated again"):
            torch.autograd.grad(g.sum(), x)
    assert g.requires_grad or (constant and name in ("rotate", "dropout"))


def test_nothing_to_do(gpu):
    for t in (torch.float32, torch.bfloat16):
        x, w, out = rand(0, 8, t=t), rand(8, 16, t=t), rand(0, 16, t=t)
        decoder.linear_(out, x, w, activation="gelu", pre=out.clone())
        for dw in (torch.full((8, 20), 5.0, dtype=t, device="cuda")[:, :16], torch.full((16, 8), 5.0, dtype=t, device="cuda").T):
            db = torch.full((16,), 5.0, dtype=t, device="cuda")
            decoder.linear_grad_(x.clone(), dw, db, out, x, w, activation="gelu", pre=out)
            assert not dw.any() and not db.any()
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        q = rand(*shape)
        dw = torch.full((8,), 5.0, device="cuda")
        decoder.head_norm_(q, None, q.clone())
        decoder.head_norm_grad_(q, None, dw, None, q, None, q.clone())
        assert not dw.any()
    q, k = rand(2, 3, 0, 8), rand(2, 3, 2, 8)   # no queries, but keys
    near(decoder.head_norm(q, k)[1], k / torch.sqrt((k * k).mean(-1, keepdim=True) + 1e-6), 1e-6)
    for shape in ((0,), (0, 5), (5, 0)):
        assert decoder.dropout(rand(*shape), 0.5, 1).shape == shape


@pytest.mark.parametrize("scale", [2.0 ** -20, 1.0, 2.0 ** 14])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_half_gradients_over_its_range(gpu, scale, act):
    """float16 gradients of upstream gradients at both ends of its range: errors of the type's rounding, once for dz and once
    for the result (2^-11 each; pre is given). Results below 2^-14 are rounded to multiples of 2^-24, so that each of
    them may be off by half of that, 2^-25, however large the others are: dx of the smallest scale is about 1e-5, of
    which that is 0.003."""
    x, w, pre = rand(600, 64, t=torch.float16) / 64, rand(64, 96, seed=1, t=torch.float16) / 8, rand(600, 96, seed=2, t=torch.float16)
    dout = (scale * rand(600, 96, seed=3)).clamp(-60000, 60000).half()
    x = x / max(scale, 1.0) ** 0.5 * min(scale, 1.0) ** -0.5   # (so that dweight is in the range)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(96, dtype=torch.float16, device="cuda")
    decoder.linear_grad_(dx, dw, db, dout / 64, x, w * min(scale, 1.0) ** -0.5, activation=act, pre=pre)
    z = pre.double().requires_grad_(True)
    y = z * torch.sigmoid(z) if act == "silu" else 0.5 * z * torch.erfc(-z * 0.5 ** 0.5)
    dz, = torch.autograd.grad(y, z, (dout / 64).double())
    near(dx, dz @ (w * min(scale, 1.0) ** -0.5).double().T, 2.0 ** -10, 2.0 ** -25)
    near(dw, x.double().T @ dz, 2.0 ** -10, 2.0 ** -25)


@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["in_out", "out_in"])
@pytest.mark.parametrize("size", [(1, 200, 3000), (4, 130, 700), (60, 72, 1000), (700, 515, 90)], ids=str)
def test_few_slopes_keep_their_bits(gpu, t, layout, size):
    """Up to 65536 elements of dz are operands with twice the type's bits: gradients are as exact as their own rounding, whose
    relative error, spread evenly up to half a step, is 0.43 of that half step over a tensor (with dz rounded too, 0.61)."""
    m, k, n = size
    x, pre, dout = rand(m, k, t=t), rand(m, n, seed=1, t=t), rand(m, n, seed=2, t=t)
    w = rand(k, n, seed=3, t=t) if layout == "in_out" else rand(n, k, seed=3, t=t).T
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(n, dtype=t, device="cuda")
    decoder.linear_grad_(dx, dw, db, dout, x, w, activation="silu", pre=pre)
    z = pre.double()
    dz = dout.double() * torch.sigmoid(z) * (1 + z * (1 - torch.sigmoid(z)))
    for got, want in ((dx, dz @ w.double().T), (dw, x.double().T @ dz), (db, dz.sum(0))):
        near(got, want, 0.5 * torch.finfo(t).eps / 2 + 2.0 ** -18)


def test_infinite_upstream_gradients_stay_in_their_rows(gpu):
    x, w, pre = rand(40, 16, t=torch.float16), rand(16, 24, seed=1, t=torch.float16), rand(40, 24, seed=2, t=torch.float16)
    dout = rand(40, 24, seed=3, t=torch.float16)
    want = torch.empty_like(x)
    decoder.linear_grad_(want, None, None, dout, x, w, activation="silu", pre=pre)
    dout[7, 3] = float("inf")
    dx = torch.empty_like(x)
    decoder.linear_grad_(dx, None, None, dout, x, w, activation="silu", pre=pre)
    rows = torch.arange(40, device="cuda") != 7
    assert not torch.isfinite(dx[7]).all()
    near(dx[rows], want[rows], 2.0 ** -9)


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [(70, 40, 24), (200, 136, 72), (700, 515, 130), (1, 40, 24), (3, 100, 50), (300, 6, 5), (3000, 72, 200), (9000, 200, 520)], ids=str)
@pytest.mark.parametrize("shift", [3, 8], ids=["unaligned", "aligned"])
def test_only_its_rows_are_read_and_written(gpu, t, size, shift):
    """NaN all around the operands is not read into a result, and what lies around the results stays as it was."""
    m, k, n = size

    def around(rows, cols, seed, value):
        big = torch.full((rows + 4, -(-cols // 8) * 8 + 16), value, dtype=t, device="cuda")
        big[2:rows + 2, shift:cols + shift] = rand(rows, cols, seed=seed, t=t)
        return big, big[2:rows + 2, shift:cols + shift]

    nan = float("nan")
    x, w, dout, res = (around(a, b, i, nan)[1] for i, (a, b) in enumerate(((m, k), (k, n), (m, n), (m, n))))
    wt = around(n, k, 9, nan)[1].T
    outs = {name: around(a, b, 5, 77.0) for name, (a, b) in dict(out=(m, n), pre=(m, n), dx=(m, k), dw=(k, n), dwt=(n, k)).items()}
    for weight in (w, wt):
        decoder.linear_(outs["out"][1], x, weight, residual=res, activation="silu", pre=outs["pre"][1])
        decoder.linear_grad_(outs["dx"][1], outs["dw"][1], None, dout, x, weight, activation="silu", pre=outs["pre"][1])
        decoder.linear_grad_(None, outs["dwt"][1].T, None, dout, x, weight, activation="silu", pre=outs["pre"][1])
        z = x.double() @ weight.double()
        near(outs["out"][1], res.double() + z * torch.sigmoid(z), 2 * torch.finfo(t).eps + 1e-5)
        for big, view in outs.values():
            assert torch.isfinite(big).all()
            mark = view.clone()
            view.fill_(77.0)
            assert (big == 77).all()
            view.copy_(mark)
        near(outs["dwt"][1].T, outs["dw"][1], 2 * torch.finfo(t).eps + 1e-5)


def test_nan_stays_in_its_row(gpu):
    x, w = rand(300, 64, t=torch.bfloat16), rand(64, 72, seed=1, t=torch.bfloat16)
    x[17, 5], x[18, 6] = float("nan"), float("inf")
    for act in ("identity", "gelu", "silu", "relu"):
        out = decoder.linear(x, w, activation=act)
        assert torch.isnan(out[17]).all() and torch.isfinite(torch.cat([out[:17], out[19:]])).all()
    q = rand(2, 5, 3, 16)
    q[1, 2, 1, 4] = float("nan")
    out = decoder.head_norm(q, rotary=decoder.Rotary((8,)), positions=torch.arange(5, device="cuda")[:, None])
    bad = torch.isnan(out).any(-1)
    assert bad[1, 2, 1] and bad.sum() == 1


def test_streams_and_graphs(gpu):
    """The gradient of a layer and of head norms on a stream of its own and captured, replayed with new inputs between eager
    calls: the eager results' bits each time."""
    for t in (torch.float16, torch.bfloat16, torch.float32):
        x, w, b = rand(3000, 64, t=t), rand(64, 96, seed=1, t=t) / 8, rand(96, seed=2, t=t)
        pre, out, dout = rand(3000, 96, t=t), rand(3000, 96, t=t), rand(3000, 96, seed=3, t=t)
        dx, dw, db, wq = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b), 1 + 0.1 * rand(16, seed=4)
        q, dq, dwq = out.reshape(3, 1000, 6, 16), torch.empty((3, 1000, 6, 16), dtype=t, device="cuda"), torch.empty(16, device="cuda")
        temp, qtemp = decoder.linear_temp(x, w, grad=True), decoder.head_norm_temp(q)

        def step():
            decoder.linear_(out, x, w, b, activation="gelu", pre=pre, temp=temp)
            decoder.linear_grad_(dx, dw, db, dout, x, w, activation="gelu", pre=pre, temp=temp)
            decoder.head_norm_grad_(dq, None, dwq, None, q, None, q, q_weight=wq, temp=qtemp)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for i in range(3):
            x.copy_(rand(3000, 64, seed=10 + i, t=t))
            dout.copy_(rand(3000, 96, seed=20 + i, t=t) * 10.0 ** (i - 1))
            results = (out, dx, dw, db, dq, dwq)
            step()
            want = [v.clone() for v in results]
            temp.fill_(255)
            for v in results:
                v.zero_()
            graph.replay()
            torch.cuda.synchronize()
            for a, c in zip(results, want):
                assert torch.equal(a, c)


def test_two_calls_at_once(gpu):
    """Layers of different sizes on two streams, each with its scratch, in flight together: the bits of one after the other."""
    def layer(seed, m, k, n, t, act):
        x, w, dout = rand(m, k, seed=seed, t=t), rand(k, n, seed=seed + 1, t=t) / k ** 0.5, rand(m, n, seed=seed + 2, t=t)
        out, pre, dx, dw, db = torch.empty_like(dout), torch.empty_like(dout), torch.empty_like(x), torch.empty_like(w), dout[0].clone()
        q, dq, temp = out.reshape(1, m, -1, 8), torch.empty_like(out).reshape(1, m, -1, 8), decoder.linear_temp(x, w, grad=True)

        def run():
            decoder.linear_(out, x, w, activation=act, pre=pre, temp=temp)
            decoder.linear_grad_(dx, dw, db, dout, x, w, activation=act, pre=pre, temp=temp)
            decoder.rotate_(dq, None, q, None, rotary, places[:m])
            decoder.dropout_(out, out, 0.3, seed)
        return run, (out, dx, dw, db, dq)

    rotary, places = decoder.Rotary((4,)), torch.arange(20000, device="cuda")[:, None]
    layers = [layer(0, 9000, 256, 512, torch.bfloat16, "gelu"), layer(5, 20000, 64, 40, torch.float32, "silu")]
    wants = []
    for run, results in layers:
        run()
        wants.append([r.clone() for r in results])
    streams = [torch.cuda.Stream() for _ in layers]
    torch.cuda.synchronize()
    for _ in range(4):
        for stream, (run, _) in zip(streams, layers):
            with torch.cuda.stream(stream):
                run()
    torch.cuda.synchronize()
    for (_, results), want in zip(layers, wants):
        for a, b in zip(results, want):
            assert torch.equal(a, b)


def test_offsets_past_32_bits(gpu):
    """Tensors of more than 2^31 elements: the last rows are those of a small call."""
    t = torch.bfloat16
    rows = 2 ** 31 // 2048 + 1000
    x = torch.empty((rows, 2048), dtype=t, device="cuda")
    tail = rand(300, 2048, t=t)
    x.zero_()
    x[-300:] = tail
    w = rand(2048, 16, seed=1, t=t) / 45
    out = decoder.linear(x, w)
    near(out[-300:], tail.double() @ w.double(), 2.0 ** -8)
    assert not out[:-300].any()
    dout = rand(rows, 16, seed=2, t=t)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    decoder.linear_grad_(dx, dw, None, dout, x, w)
    near(dx[-300:], dout[-300:].double() @ w.double().T, 2.0 ** -8)
    near(dw, tail.double().T @ dout[-300:].double(), 2.0 ** -8)
    y = decoder.dropout(x, 0.25, 6)
    n = x.numel()
    c = np.arange(n // 4 - 4096, n // 4, dtype=np.uint64)
    low, by = np.uint64(2 ** 32 - 1), np.uint64(32)
    c = [c & low, c >> by, np.zeros_like(c), np.zeros_like(c)]
    for r in range(10):
        k0, k1 = np.uint64((6 + 0x9E3779B9 * r) & 0xFFFFFFFF), np.uint64((0xBB67AE85 * r) & 0xFFFFFFFF)
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> by) ^ c[1] ^ k0, b & low, (a >> by) ^ c[3] ^ k1, a & low]
    keep = torch.from_numpy(np.stack(c, 1).reshape(-1) >= np.uint64(2 ** 30)).cuda()
    want = torch.where(keep, x.reshape(-1)[-16384:].float() * (1 / 0.75), 0).to(t)
    assert torch.equal(y.reshape(-1)[-16384:], want)
    del y, dx, out
    q = x[:rows // 8 * 8].reshape(1, rows // 8, 128, 128)
    places = torch.arange(rows // 8, device="cuda")[:, None]
    rotary = decoder.Rotary((64,))
    z = decoder.head_norm(q, rotary=rotary, positions=places)
    assert torch.equal(z[:, -30:], decoder.head_norm(q[:, -30:].clone(), rotary=rotary, positions=places[-30:].contiguous()))


def test_the_same_bits_every_time(gpu):
    x, w, dout = rand(5000, 96, t=torch.bfloat16), rand(96, 136, seed=1, t=torch.bfloat16), rand(5000, 136, seed=2, t=torch.bfloat16)
    results = []
    for _ in range(3):
        leaves = [v.detach().requires_grad_(True) for v in (x, w)]
        decoder.linear(*leaves, activation="silu").backward(dout)
        results.append([v.grad for v in leaves])
    for r in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, results[0]))


def test_single_rows_of_distant_buffers(gpu):
    """The stride of a single row means nothing: one row, feature or output of buffers whose rows are 64 MB apart."""
    big = torch.zeros((2, 2 ** 24), device="cuda")
    x, w = big[1:, :40], rand(40, 24, seed=1)
    x.copy_(rand(1, 40))
    near(decoder.linear(x, w), x.double() @ w.double(), 1e-6)
    column = rand(40, 1, seed=2)
    near(decoder.linear(rand(9, 1, seed=3), big[:1, 100:124].copy_(rand(1, 24, seed=4))),
         rand(9, 1, seed=3).double() @ rand(1, 24, seed=4).double(), 1e-6)
    near(decoder.linear(rand(9, 40, seed=3), column), rand(9, 40, seed=3).double() @ column.double(), 1e-6)
    with pytest.raises(Exception, match="too far apart"):
        decoder.linear_(torch.empty((2, 24), device="cuda"), big[:, :40], w)
