"""8-bit floating point with a scale for each block of 128, against 64-bit restatements of the formulas.

u is half a step of the result's type relative to the value (one rounding). A block's scale is one
division in 32 bits; its codes are those of the exact quotient, so they are compared for equality. A
product's 32-bit sums are off by at most a step, 2^-23, of the sum of magnitudes for each addition.
"""

import pytest
import torch

import qr_v2_b200_kernel_b200 as qr

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn


def _randn(*shape, seed=0, dtype=SF, size=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (size * torch.randn(*shape, generator=gen, device="cuda")).to(dtype)


def _tops(x, tile):
    """The largest magnitude of each block, in 64 bits, and the same for each entry."""
    rows, cols = x.shape
    pad = torch.zeros(-(-rows // tile) * tile, -(-cols // 128) * 128, dtype=torch.float64, device=x.device)
    pad[:rows, :cols] = x.double().abs()
    a = pad.reshape(-1, tile, pad.shape[1] // 128, 128).amax((1, 3))
    return a, a.repeat_interleave(tile, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _nearest(q):
    """64-bit numbers to those of four significant bits, not finer than 2^-9, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0**-6))) - 3)
    return (q / step).round() * step


def _check(x, tile):
    codes, scale = qr.quantize_fp8(x, tile_rows=tile)
    a, each = _tops(x.reshape(-1, x.shape[-1]), tile)
    assert codes.dtype == E4M3 and codes.shape == x.shape
    assert torch.all((scale.reshape(a.shape).double() - a / 448).abs() <= 2.0**-24 * a / 448)
    flat = x.reshape(-1, x.shape[-1]).double()
    want = torch.where(each > 0, _nearest(flat * 448 / each.clamp_min(1e-300)), 0.0)
    assert torch.equal(codes.double().reshape(want.shape), want)
    return codes, scale


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("tile", [1, 128])
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (2, 128), (130, 129), (1, 4096), (127, 255), (128, 256), (257, 1000), (3, 2047),
                                        (1000, 392), (1, 40000)])
def test_quantize_fp8(rows, cols, tile, dtype):
    x = _randn(rows, cols, seed=rows + cols, dtype=dtype) * torch.exp(_randn(cols, seed=5)).to(dtype)
    codes, scale = _check(x, tile)
    _, each = _tops(x, tile)
    spread = scale.repeat_interleave(tile, 0)[:rows].repeat_interleave(128, 1)[:, :cols].double()
    for out in (BF, HF, SF):
        v = qr.dequantize_fp8(codes, scale, out, tile_rows=tile)
        exact = codes.double() * spread
        # one product in 32 bits, one rounding; the smallest numbers of 16 bits are 2^-24 apart
        assert v.dtype == out and torch.all((v.double() - exact).abs() <= (U[out] + 2.0**-24) * exact.abs() + (2.0**-25 if out == HF else 1e-44))


def test_many_rows_go_four_blocks_to_a_thread():
    for dtype in (BF, SF):
        _check(_randn(5003, 1152, seed=1, dtype=dtype), 1)
        _check(_randn(5003, 1151, seed=2, dtype=dtype), 1)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
def test_entries_midway_between_codes(dtype):
    # With 448 in the block codes are the entries' own rounding, and all midpoints occur; with 7 2^k they do at another size.
    codes = torch.arange(0, 0x7F, device="cuda").to(torch.uint8).view(E4M3).float()
    mid = ((codes[1:] + codes[:-1]) / 2)[:125]
    for top in (448.0, 7.0, 1.75, 3.0):
        row = torch.cat([torch.tensor([448.0], device="cuda"), mid, -mid[:1]]) * (top / 448)
        _check(row.to(dtype)[None].contiguous(), 1)
    if dtype == SF:  # next to them, too
        row = torch.cat([torch.tensor([448.0], device="cuda"), mid])
        for to in (0.0, 1e9):
            _check(torch.cat([row[:1], torch.nextafter(row[1:], torch.full_like(mid, to))])[None].contiguous(), 1)
        a = 3.3333333  # midpoints of a block whose quotients 32 bits do not hold
        near = (row.double() * a / 448).float()
        _check(torch.cat([near, near, torch.nextafter(near, torch.zeros_like(near))])[None].contiguous()[:, :126], 1)


@pytest.mark.parametrize("tile", [1, 128])
def test_ends_of_the_range(tile):
    for dtype, sizes in ((BF, (2.0**-90, 2.0**-60, 2.0**100, 1.5 * 2.0**127)), (SF, (2.0**-90, 2.0**127)), (HF, (2.0**-14, 6e4))):
        for size in sizes:
            x = _randn(3, 300, seed=4, dtype=SF)
            _check((x / x.abs().max() * size).to(dtype), tile)
    x = _randn(130, 384, seed=6)
    x[:, 130] = float("nan")
    x[3, 260] = float("inf")
    x[:, :128] *= 2.0**-126
    codes, scale = qr.quantize_fp8(x, tile_rows=tile)
    assert torch.all(scale[:, 0] == 0) and torch.all(codes[:, :128].float() == 0)
    assert torch.all(scale[:, 1].isnan()) and torch.all(codes[:, 128:256].float() == 0)
    bad = torch.zeros(scale.shape[0], dtype=torch.bool, device="cuda")
    bad[3 // tile] = True
    assert torch.equal(scale[:, 2].isnan(), bad)
    v = qr.dequantize_fp8(codes, scale, SF, tile_rows=tile)
    assert torch.all(v[:, 128:256].isnan()) and torch.all(v[:, :128] == 0)
    assert qr.quantize_fp8(torch.zeros(2, 5, device="cuda"))[1].eq(0).all()


def test_shapes_strides_and_alignment():
    x = _randn(3, 4, 5, 200, seed=3, dtype=BF)
    codes, scale = qr.quantize_fp8(x)
    assert codes.shape == x.shape and scale.shape == (3, 4, 5, 2)
    flat, flat_scale = qr.quantize_fp8(x.reshape(60, 200))
    assert torch.equal(codes.reshape(60, 200).view(torch.uint8), flat.view(torch.uint8)) and torch.equal(scale.reshape(60, 2), flat_scale)
    for view in (x.transpose(0, 2), x[..., 1:130], x[:, 1:, ::2], x[..., ::3]):
        a, s = qr.quantize_fp8(view)
        b, t = qr.quantize_fp8(view.contiguous())
        assert torch.equal(a.float(), b.float()) and torch.equal(s, t)
        assert torch.equal(qr.dequantize_fp8(a, s), qr.dequantize_fp8(b.contiguous(), t))
    wide = _randn(300, 600, seed=8, dtype=HF)
    for view in (wide[1:, 3:], wide.T, wide[::2, ::2]):
        a, s = qr.quantize_fp8(view, tile_rows=128)
        b, t = qr.quantize_fp8(view.contiguous(), tile_rows=128)
        assert torch.equal(a.float(), b.float()) and torch.equal(s, t)
    one, s1 = qr.quantize_fp8(x[0, 0, 0])
    assert one.shape == (200,) and s1.shape == (2,)
    for shape in ((0, 128), (4, 0), (2, 0, 7)):
        codes, scale = qr.quantize_fp8(torch.zeros(shape, device="cuda"))
        assert codes.shape == shape and qr.dequantize_fp8(codes, scale).shape == shape


# ---- the product ----------------------------------------------------------------------------


def _operands(rows, outs, depth, seed=0):
    x = _randn(rows, depth, seed=seed, dtype=SF) * torch.exp(0.5 * _randn(depth, seed=seed + 1))
    w = _randn(outs, depth, seed=seed + 2, dtype=SF, size=depth**-0.5)
    return qr.quantize_fp8(x), qr.quantize_fp8(w, tile_rows=128)


def _values64(codes, scale, tile):
    rows, cols = codes.shape
    return codes.double() * scale.double().repeat_interleave(tile, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _check_linear(x, w, bias, dtype):
    (xc, xs), (wc, ws) = x, w
    y = qr.fp8_linear(xc, xs, wc, ws, bias, dtype=dtype)
    a, b = _values64(xc, xs, 1), _values64(wc, ws, 128)
    want = a @ b.T + (bias.double() if bias is not None else 0)
    size = a.abs() @ b.abs().T + (bias.double().abs() if bias is not None else 0)
    # 128 additions in a block, as many as there are blocks, two factors and the bias
    adds = 128 + xs.shape[1] + 4
    assert y.dtype == dtype and y.shape == want.shape
    err = (y.double() - want).abs()
    bound = U[dtype] * want.abs() + adds * 2.0**-23 * size * (1 + U[dtype]) + (2.0**-25 if dtype == HF else 1e-44)
    assert torch.all(err <= bound), ((err / bound).max().item())
    # and not a systematic loss: sums of many roundings stay near their square root
    rest = (err - U[dtype] * want.abs()).clamp_min(0) / size.clamp_min(1e-300)
    assert rest.max() <= 64 * 2.0**-24
    return y


@pytest.mark.parametrize("rows, outs, depth", [
    (1, 1, 1), (1, 5, 127), (1, 128, 128), (2, 100, 129), (1, 4096, 4096), (3, 130, 1000), (4, 257, 520), (5, 1000, 2000), (8, 512, 1024),
    (9, 40, 300), (16, 4096, 1024), (17, 300, 384), (33, 129, 640), (64, 1000, 2048), (100, 256, 100), (128, 128, 4096), (129, 127, 257),
    (333, 1000, 2000), (256, 512, 512), (513, 300, 1111), (1000, 1537, 130), (2048, 2048, 256), (1111, 2222, 3333)])
def test_fp8_linear(rows, outs, depth):
    x, w = _operands(rows, outs, depth, seed=rows)
    bias = _randn(outs, seed=9)
    for dtype in (BF, HF, SF):
        _check_linear(x, w, None, dtype)
        _check_linear(x, w, bias.to(dtype), dtype)


def test_every_row_count_of_the_small_kernels():
    _, w = _operands(1, 515, 1300)
    for rows in list(range(1, 40)) + [63, 65, 96, 127, 160, 255, 257]:
        x, _ = _operands(rows, 1, 1300, seed=rows)
        _check_linear(x, w, None, SF)


@pytest.mark.parametrize("rows", [1, 3, 20, 300])
def test_linear_layouts(rows):
    x, w = _operands(rows, 259, 389)
    want = qr.fp8_linear(*x, *w)
    pad = torch.empty(rows + 1, 391, dtype=torch.uint8, device="cuda").view(E4M3)[1:, 2:]
    pad.view(torch.uint8).copy_(x[0].view(torch.uint8))
    wpad = torch.empty(259, 397, dtype=torch.uint8, device="cuda").view(E4M3)[:, 3:392]
    wpad.view(torch.uint8).copy_(w[0].view(torch.uint8))
    xs = x[1].T.contiguous().T  # scales with other strides
    for a, b in ((pad, w[0]), (x[0], wpad), (pad, wpad), (x[0].contiguous(), w[0].contiguous())):
        assert torch.equal(qr.fp8_linear(a, xs, b, w[1]), want)
    a = x[0].view(torch.uint8).unflatten(0, (1, rows)).view(E4M3)
    assert torch.equal(qr.fp8_linear(a, x[1][None], *w), want[None])
    single = qr.fp8_linear(x[0][0], x[1][0], *w)
    assert single.shape == (259,) and torch.allclose(single.float(), want[0].float(), rtol=2.0**-7, atol=1e-6)
    assert qr.fp8_linear(x[0][:0], x[1][:0], *w).shape == (0, 259)
    assert qr.fp8_linear(*x, w[0][:0], w[1][:0]).shape == (rows, 0)


@pytest.mark.parametrize("rows", [1, 6, 40, 300])
def test_linear_scales_and_odd_codes(rows):
    x, w = _operands(rows, 300, 640)
    big = torch.exp2(torch.randint(-40, 40, x[1].shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").float())
    _check_linear((x[0], x[1] * big), w, None, SF)
    s = x[1].clone()
    s[rows // 2, 2] = float("nan")
    y = qr.fp8_linear(x[0], s, *w)
    assert y[rows // 2].isnan().all() and y.isnan().sum() == 300
    t = w[1].clone()
    t[1, 1] = float("nan")
    y = qr.fp8_linear(*x, w[0], t)
    assert y[:, 128:256].isnan().all() and y.isnan().sum() == rows * 128
    c = x[0].clone()
    c.view(torch.uint8)[rows - 1, 5] = 0x7F  # the format's NaN
    y = qr.fp8_linear(c, x[1], *w)
    assert y[rows - 1].isnan().all() and y.isnan().sum() == 300
    top = torch.full((rows, 640), 448.0, device="cuda").to(E4M3)  # the largest sums
    one = torch.ones(rows, 5, device="cuda")
    y = qr.fp8_linear(top, one, torch.full((300, 640), 448.0, device="cuda").to(E4M3), torch.ones(3, 5, device="cuda"), dtype=SF)
    assert torch.all(y == 640 * 448.0**2)


def test_a_row_does_not_depend_on_its_neighbours():
    x, w = _operands(300, 256, 512)
    y = qr.fp8_linear(*x, *w, dtype=SF)
    c = x[0].clone()
    c.view(torch.uint8)[:150] = 0x7F
    assert torch.equal(qr.fp8_linear(c, x[1], *w, dtype=SF)[150:], y[150:])
    assert torch.equal(qr.fp8_linear(*x, *w, dtype=SF), y)


def test_fp8_refusals():
    (xc, xs), (wc, ws) = _operands(4, 8, 256)
    b = torch.zeros(8, device="cuda", dtype=BF)
    for call, error in (
            (lambda: qr.quantize_fp8(xs.double()), TypeError), (lambda: qr.quantize_fp8(xs, tile_rows=2), ValueError),
            (lambda: qr.quantize_fp8(xs[None], tile_rows=128), ValueError), (lambda: qr.quantize_fp8(xs.cpu()), RuntimeError),
            (lambda: qr.quantize_fp8(xs.clone().requires_grad_()), RuntimeError),
            (lambda: qr.dequantize_fp8(xc, xs[:, :1]), ValueError), (lambda: qr.dequantize_fp8(xc.float(), xs), TypeError),
            (lambda: qr.dequantize_fp8(xc, xs, torch.float64), TypeError),
            (lambda: qr.fp8_linear(xc, xs, wc[:, :128], ws), ValueError), (lambda: qr.fp8_linear(xc, xs[:, :1], wc, ws), ValueError),
            (lambda: qr.fp8_linear(xc, xs, wc, ws[:, :1]), ValueError), (lambda: qr.fp8_linear(xc.float(), xs, wc, ws), TypeError),
            (lambda: qr.fp8_linear(xc, xs, wc, ws, b[:4]), ValueError), (lambda: qr.fp8_linear(xc, xs, wc, ws, b.float()), TypeError),
            (lambda: qr.fp8_linear(xc, xs.double(), wc, ws), TypeError), (lambda: qr.fp8_linear(xc[:, :0], xs[:, :0], wc[:, :0], ws[:, :0]), ValueError)):
        with pytest.raises(error):
            call()


def test_fp8_in_a_graph_and_on_another_stream():
    x = [_randn(20, 1000, seed=s, dtype=BF) for s in (1, 2)]
    w = qr.quantize_fp8(_randn(300, 1000, seed=3, dtype=BF, size=0.03), tile_rows=128)

    def chain(x):
        codes, scale = qr.quantize_fp8(x)
        return qr.fp8_linear(codes, scale, *w), qr.dequantize_fp8(codes, scale)

    want = [chain(v) for v in x]
    hold = x[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = chain(hold)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(hold)
    for v, expect in zip(x, want):
        hold.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, expect))
