"""4-bit matrices against a float64 restatement: the same codes and scales, products within float32 rounding."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([i * 2.0 ** -9 for i in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:119])


def microscale():
    from bsipytorch_b200 import microscale as m
    return m


def nearest(v, table):
    up = np.clip(np.searchsorted(table, v), 1, len(table) - 1)
    low = up - 1
    to_low, to_up = v - table[low], table[up] - v
    return np.where((to_low < to_up) | ((to_low == to_up) & (low % 2 == 0)), low, up)


def packed(x, fmt):
    """(values, block scales, row scales) of x (float64)."""
    rows, K = x.shape
    block = 32 if fmt == "mxfp4" else 16
    b = np.pad(x, ((0, 0), (0, -K % block))).reshape(rows, -1, block)
    amax = np.abs(b).max(-1)
    if fmt == "mxfp4":
        _, e = np.frexp(amax)
        scale = np.where(amax > 0, np.ldexp(1.0, np.maximum(e - 3, -127)), 2.0 ** -127)
        g = np.ones(rows)
    else:
        m, e = np.frexp(amax.max(-1) / 2688.0)
        g = np.where(amax.max(-1) > 0, np.ldexp(1.0, np.maximum(np.where(m == 0.5, e - 1, e), -100)), 1.0)
        scale = E4M3[nearest(amax / (6.0 * g[:, None]), E4M3)]
    full = (scale * g[:, None])[..., None]
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(full > 0, GRID[nearest(np.abs(b) / full, GRID)] * np.sign(b) * full, 0.0)
    return q.reshape(rows, -1)[:, :K], scale, g


def inputs(rows, K, dtype, seed, kind="plain"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, K, generator=g)
    x *= 1.0 + 19.0 * (torch.rand(K, generator=g) < 0.02)
    if kind == "borders":          # quotients on and beside every border between two codes
        x = (torch.randint(-24, 25, (rows, K), generator=g) / 4.0) * 2.0 ** torch.randint(-3, 4, (rows, 1), generator=g)
    elif kind == "wide":           # magnitudes over many powers of two, whole blocks far below the row's largest, zeros
        x *= 2.0 ** torch.randint(-40, 10, (rows, K), generator=g)
        x[:, : K // 3] = 0.0
        x[0] = 0.0
    return x.to(dtype)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype,kind", [(d, k) for d in DT for k in ("plain", "borders", "wide") if (d, k) != ("fp16", "wide")])
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 17), (130, 64), (5, 1000), (2, 4096), (1, 40000), (261, 515)])
def test_codes_and_scales(fmt, dtype, kind, rows, K):
    x = inputs(rows, K, DT[dtype], rows + K, kind)
    q = microscale().quantize_fp4(x.cuda(), fmt)
    values, scale, g = packed(x.double().numpy(), fmt)
    assert np.array_equal(q.block_scales().double().cpu().numpy(), scale)
    if fmt == "nvfp4":
        assert np.array_equal(q.row_scale.double().cpu().numpy(), g)
    assert np.array_equal(q.dequantize(torch.float32).double().cpu().numpy(), values.astype(np.float32).astype(np.float64))
    assert torch.equal(q.dequantize().cpu(), torch.from_numpy(values).to(torch.float32).to(DT[dtype]))
    assert q.shape == (rows, K) and q.dtype == DT[dtype]


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("dtype", list(DT))
def test_every_byte_of_codes_in_every_place(fmt, dtype):
    """Unpacked values of all 256 bytes at each of 16 neighbouring places, with block scales of 1; a width that ends inside a piece."""
    m = microscale()
    grid = np.concatenate([GRID, -GRID])
    first = m.quantize_fp4(torch.full((256, 32 * 8 - 3), 6.0 if fmt == "nvfp4" else 4.0, device="cuda"), fmt)
    assert first.block_scales().mul(1.0 if first.row_scale is None else first.row_scale[:, None]).eq(1.0).all()
    codes = ((torch.arange(256)[:, None] + 37 * torch.arange(128)[None]) % 256).to(torch.uint8)
    values = np.stack([grid[codes.numpy() & 15], grid[codes.numpy() >> 4]], -1).reshape(256, 256)[:, :253]
    got = first._replace(codes=codes.cuda()).dequantize(DT[dtype])
    assert np.array_equal(got.double().cpu().numpy(), values)


def test_every_quotient_of_sixteen_bits_beside_the_borders():
    """nvfp4, bfloat16: every value in a block whose largest makes each of the scale's significands."""
    out = []
    for m in range(8, 16):
        top = 6.0 * m / 8.0 * 64            # block scale m / 8 times a power of two, when the row's own power fits
        v = torch.arange(0, 0x7F80).to(torch.int16).view(torch.bfloat16).double()
        v = v[(v <= top) & (v > top * 2 ** -12)]
        v = torch.nn.functional.pad(v, (0, -len(v) % 15)).view(-1, 15)
        out.append(torch.cat([torch.full((len(v), 1), top, dtype=torch.float64), v], 1).reshape(1, -1))
    for row in out:
        x = row.to(torch.bfloat16)
        q = microscale().quantize_fp4(x.cuda(), "nvfp4").dequantize(torch.float32)
        assert np.array_equal(q.double().cpu().numpy(), packed(x.double().numpy(), "nvfp4")[0])


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_strided_and_misaligned_rows(fmt):
    m = microscale()
    whole = inputs(40, 700, torch.bfloat16, 3).cuda()
    for x in (whole[:, 8:520], whole[:, 3:500], whole[::3, 1:], whole.t(), whole[:1, 5:6], whole[0].expand(4, 700)):
        want = m.quantize_fp4(x.contiguous(), fmt)
        got = m.quantize_fp4(x, fmt)
        assert torch.equal(want.codes, got.codes) and torch.equal(want.block_scales(), got.block_scales())
    cube = whole.view(4, 10, 700)
    assert torch.equal(m.quantize_fp4(cube, fmt).codes, m.quantize_fp4(whole, fmt).codes)


# A sum of K products in float32: each addition is off by at most half a step of a partial sum, which is no larger than the sum of
# the magnitudes; the tensor cores add 64 products at a time and may cut instead of rounding, 2^-23 of the largest term each. With
# n = K / 64 + 8 additions behind one another that is at most n * 2^-22 of the sum of magnitudes; rms far less.
def product_tolerance(magnitudes, want, K, dtype):
    eps = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return (K / 64 + 8) * 2.0 ** -22 * magnitudes + 1.01 * eps * np.abs(want) + tiny


def check_product(x, w, bias, fmt, relu, y):
    xq, wq = packed(x.double().numpy(), fmt)[0], packed(w.double().numpy(), fmt)[0]
    want = xq @ wq.T + (0.0 if bias is None else bias.double().numpy())
    size = np.abs(xq) @ np.abs(wq).T + (0.0 if bias is None else np.abs(bias.double().numpy()))
    if relu:
        want = np.maximum(want, 0.0)
    far = np.abs(y.double().cpu().numpy() - want) - product_tolerance(size, want, x.shape[1], y.dtype)
    assert far.max() <= 0, (np.unravel_index(far.argmax(), far.shape), far.max())


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M,K,N", [(1, 32, 8), (1, 64, 128), (1, 4096, 300), (3, 1000, 129), (16, 2048, 512), (17, 256, 127), (32, 8192, 256),
                                   (33, 515, 1024), (64, 1024, 1000), (65, 300, 64), (128, 512, 256), (129, 768, 384), (256, 4096, 128), (300, 1025, 257),
                                   (513, 640, 2048), (1025, 2048, 1300)])
def test_products(fmt, M, K, N):
    for dtype in (torch.bfloat16, torch.float32) if M % 2 else (torch.float16,):
        x, w = inputs(M, K, dtype, M + K), inputs(N, K, torch.float32, N) * 0.05
        bias = torch.randn(N, generator=torch.Generator().manual_seed(1)) if N % 2 == 0 else None
        m = microscale()
        wq = m.quantize_fp4(w.cuda(), fmt)
        y = m.fp4_linear(x.cuda(), wq, None if bias is None else bias.cuda(), relu=N % 3 == 0)
        assert y.dtype == dtype and y.shape == (M, N)
        check_product(x, w, bias, fmt, N % 3 == 0, y)
        from bsipytorch_b200 import bsi_ops
        assert bsi_ops.device_status() == 0


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_products_again_packed_once_and_in_a_graph(fmt):
    m = microscale()
    x, w = inputs(48, 2000, torch.bfloat16, 1).cuda(), m.quantize_fp4(inputs(640, 2000, torch.float32, 2).cuda(), fmt)
    y = m.fp4_linear(x, w)
    assert torch.equal(y, m.fp4_linear(x, w)) and torch.equal(y, m.fp4_linear(m.quantize_fp4(x, fmt), w))
    assert torch.equal(y[:5], m.fp4_linear(x, w)[:5]) and torch.equal(m.fp4_linear(x.view(4, 12, 2000), w), y.view(4, 12, 640))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = m.fp4_linear(x, w)
    x.copy_(inputs(48, 2000, torch.bfloat16, 9))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, m.fp4_linear(x, w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = m.fp4_linear(x, w)
    side.synchronize()
    assert torch.equal(other, held)


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_a_row_that_is_not_finite(fmt):
    m = microscale()
    x = inputs(5, 512, torch.bfloat16, 1)
    w = inputs(200, 512, torch.float32, 2)
    clean = m.fp4_linear(x.cuda(), m.quantize_fp4(w.cuda(), fmt))
    x[2, 100], x[4, 300] = float("nan"), -float("inf")
    w[7, 5] = float("inf")
    y = m.fp4_linear(x.cuda(), m.quantize_fp4(w.cuda(), fmt))
    bad = torch.zeros(5, 200, dtype=torch.bool, device="cuda")
    bad[[2, 4]] = True
    bad[:, 7] = True
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], clean[~bad])
    assert torch.isnan(m.quantize_fp4(x.cuda(), fmt).dequantize()[2, 100])


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M,N", [(2, 130), (60, 300), (130, 257), (1030, 3500)])
def test_rows_at_both_ends_of_float32(fmt, M, N):
    """The factors of a token and of a weight's row are infinite together, or 0, where the sum times both is in range; the narrow kernel
    and both widths of the paired one."""
    K = 64
    x, w = inputs(M, K, torch.float32, M).clamp(-4, 4), (inputs(N, K, torch.float32, N) * 0.05).clamp(-0.2, 0.2)
    x[0, 0], w[0, :32], w[0, 40] = 3e38, 0.0, 1e8         # 2^117 * 2^16, a sum of 0
    if fmt == "nvfp4":                                    # 2^-75 * 2^-75, a sum of 64 * 2688^2
        for r in (1, -1):
            x[r], w[r] = 2688.0 * 2.0 ** -75, 2688.0 * 2.0 ** -75
    m = microscale()
    for bias in (None, torch.linspace(-1, 1, N)):
        y = m.fp4_linear(x.cuda(), m.quantize_fp4(w.cuda(), fmt), None if bias is None else bias.cuda())
        assert bool(torch.isfinite(y).all())
        check_product(x, w, bias, fmt, False, y)
    # nvfp4: nothing but the bias, as what the token has beside 3e38 is below its row's scales (an mxfp4 block has a scale of its own)
    assert fmt == "mxfp4" or y[0, 0] == -1.0


def test_one_row_without_a_batch_dimension():
    m = microscale()
    w = m.quantize_fp4(torch.randn(70, 96, device="cuda"))
    x = torch.randn(3, 96, device="cuda").half()
    bias = torch.randn(70, device="cuda").half()
    y = m.fp4_linear(x, w, bias, out_dtype=torch.float32)
    assert y.dtype == torch.float32 and torch.equal(m.fp4_linear(x[1], w, bias, out_dtype=torch.float32), y[1])
    assert torch.equal(m.fp4_linear(x[1:2], w, bias), y[1:2].half()) and torch.equal(y, m.fp4_linear(x, w, bias.float(), out_dtype=torch.float32))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_a_row_does_not_depend_on_its_batch(fmt):
    """Tiles, parts along K and kernels change with the number of tokens; what a token gets changes by the order of float32 sums only."""
    m = microscale()
    w = m.quantize_fp4(inputs(384, 3000, torch.float32, 2).cuda(), fmt)
    x = inputs(300, 3000, torch.bfloat16, 1).cuda()
    packed_rows = m.quantize_fp4(x, fmt)
    for rows in (1, 16, 17, 33, 65, 128, 129, 300):
        q = m.quantize_fp4(x[:rows], fmt)
        assert torch.equal(q.codes, packed_rows.codes[:rows]) and torch.equal(q.block_scales(), packed_rows.block_scales()[:rows])
        check_product(x[:rows].cpu(), inputs(384, 3000, torch.float32, 2), None, fmt, False, m.fp4_linear(x[:rows], w, out_dtype=torch.float32))


def test_no_rows():
    m = microscale()
    assert m.fp4_linear(torch.ones(3, 32, device="cuda"), m.quantize_fp4(torch.empty(0, 32, device="cuda"))).shape == (3, 0)
    w = m.quantize_fp4(torch.randn(64, 96, device="cuda"))
    assert m.fp4_linear(torch.empty(0, 96, device="cuda"), w).shape == (0, 64)
    assert m.quantize_fp4(torch.empty(0, 96, device="cuda")).dequantize().shape == (0, 96)


def test_layer_and_model_walk():
    m = microscale()
    torch.manual_seed(0)
    lin = torch.nn.Linear(512, 384).cuda().half()
    layer = m.FP4Linear(lin, "mxfp4")
    x = torch.randn(2, 9, 512, device="cuda").half()
    check_product(x.reshape(18, 512).cpu(), lin.weight.detach().cpu(), lin.bias.detach().float().cpu(), "mxfp4", False, layer(x).reshape(18, 384))
    again = m.FP4Linear(torch.nn.Linear(512, 384).cuda(), "mxfp4")
    again.load_state_dict(layer.state_dict())
    assert torch.equal(again(x), layer(x))
    halved = m.FP4Linear(torch.nn.Linear(512, 384).cuda(), "nvfp4").half()
    assert halved.bias.dtype == torch.float32 and halved.row_scale.dtype == torch.float32 and halved.codes.dtype == torch.uint8


def test_refusals():
    m = microscale()
    w = m.quantize_fp4(torch.randn(64, 96, device="cuda"))
    x = torch.randn(4, 96, device="cuda")
    with pytest.raises(ValueError):
        m.quantize_fp4(x, "fp4")
    for call in (lambda: m.quantize_fp4(x.cpu()), lambda: m.quantize_fp4(x.double()), lambda: m.quantize_fp4(x[:, :0]),
                 lambda: m.fp4_linear(x[:, :64], w), lambda: m.fp4_linear(x, w, torch.zeros(63, device="cuda")), lambda: m.fp4_linear(x, w, torch.zeros(64)),
                 lambda: m.fp4_linear(m.quantize_fp4(x, "mxfp4"), w), lambda: m.fp4_linear(x, w, out_dtype=torch.float64),
                 lambda: m.fp4_linear(x, w._replace(codes=w.codes[:, :32])), lambda: m.fp4_linear(x, w._replace(scales=w.scales[:-1])),
                 lambda: m.fp4_linear(x, w._replace(row_scale=None)), lambda: m.fp4_linear(x, w._replace(features=200))):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_packed_activations_of_another_width_are_refused(fmt):
    """Also where both widths round up to the same bytes."""
    m = microscale()
    w = m.quantize_fp4(torch.randn(64, 50, device="cuda"), fmt)
    for features in (40, 49, 51, 64, 96):
        with pytest.raises(RuntimeError, match="features"):
            m.fp4_linear(m.quantize_fp4(torch.randn(4, features, device="cuda"), fmt), w)
    x = torch.randn(4, 50, device="cuda")
    assert torch.equal(m.fp4_linear(m.quantize_fp4(x, fmt), w), m.fp4_linear(x, w))


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("outputs", [1, 100, 128, 300])
def test_a_layer_s_buffers(fmt, outputs):
    """Each on an allocation of its own, with nothing in it that depends on what the memory held before."""
    m = microscale()
    lin = torch.nn.Linear(515, outputs, device="cuda")
    states = []
    for fill in (0x5A, 0xA5):
        used = [torch.full((n,), fill, dtype=torch.uint8, device="cuda") for n in [4096] * 64 + [1 << 16] * 64 + [1 << 19] * 16 + [1 << 22]]
        del used
        layer = m.FP4Linear(lin, fmt)
        for b in layer.buffers():
            assert b.untyped_storage().nbytes() == b.nbytes
        states.append(layer.state_dict())
    assert states[0].keys() == states[1].keys() and all(torch.equal(states[0][k], states[1][k]) for k in states[0])
    x = torch.randn(3, 515, device="cuda")
    assert torch.equal(layer(x), m.fp4_linear(x, m.quantize_fp4(lin.weight.detach(), fmt), lin.bias.detach()))


# 74 pairs of CTAs walk over tiles of 256 outputs. In order: 70 tiles of 256 tokens, 180 of them (three rounds), 120 tiles of 128 tokens
# (two rounds, as many as 80 wide ones), the same in one block, 120 tiles of 256 tokens and nine blocks. The ring goes on from one tile
# to the next out of step with it.
@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("M,K,N", [(1030, 515, 3500), (2100, 300, 5003), (384, 1100, 10240), (371, 96, 10235), (1500, 2090, 4999)])
def test_products_of_more_tiles_than_pairs(fmt, M, K, N):
    x, w = inputs(M, K, torch.bfloat16, M + K), inputs(N, K, torch.float32, N) * 0.05
    bias = torch.randn(N, generator=torch.Generator().manual_seed(1)) if N % 2 == 0 else None
    m = microscale()
    wq = m.quantize_fp4(w.cuda(), fmt)
    y = m.fp4_linear(x.cuda(), wq, None if bias is None else bias.cuda(), relu=N % 3 == 0, out_dtype=torch.float32 if K % 2 else None)
    check_product(x, w, bias, fmt, N % 3 == 0, y)
    from bsipytorch_b200 import bsi_ops
    assert bsi_ops.device_status() == 0


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
def test_more_elements_than_32_bits_count(fmt):
    m = microscale()
    x = torch.empty(131073, 16400, dtype=torch.bfloat16, device="cuda").normal_(0.0, 1.0, generator=torch.Generator(device="cuda").manual_seed(2))
    q = m.quantize_fp4(x, fmt)
    back = q.dequantize()
    last = m.quantize_fp4(x[-200:], fmt)
    assert torch.equal(q.codes[-200:], last.codes) and torch.equal(back[-200:], last.dequantize())
    w = m.quantize_fp4(inputs(140, 16400, torch.float32, 3).cuda(), fmt)
    y = m.fp4_linear(q, w)
    assert torch.equal(y[-200:].isfinite().all(), torch.tensor(True, device="cuda"))
    check_product(x[-3:].cpu(), inputs(140, 16400, torch.float32, 3), None, fmt, False, y[-3:])
