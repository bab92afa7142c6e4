"""8-bit blocks (``ops/fp8.py``): rows and weights in E4M3 with scales for blocks of 128, the products on them, the layers and the
checkpoint store. Expected values come from the definitions in 64 bits.

Tolerances. Codes and what they stand for are compared exactly: a power-of-two scale leaves one nearest E4M3 number. A product of M x K
by K x N is rounded to bf16 once (2^-8 relative) after sums in fp32: each of the K products of a row enters one addition in the tensor
core and each of the K / 128 blocks one scaled addition, every one off by at most 2^-23 of the sum of magnitudes (the tensor core may
drop bits instead of rounding), so |y - exact| <= 2^-8 |exact| + (K + 2 K / 128 + 4) 2^-23 sum |x8| |w8| (1 + 2^-8)."""
import math

import pytest
import torch

from axolotl_b200.ops.fp8 import (dequantize_fp8_rows, dequantize_fp8_weight, fp8_adapter_grad, fp8_gemm, fp8_linear, fp8_lora_linear,
                                  quantize_fp8_rows, quantize_fp8_weight)

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF16, EPS32 = 2.0 ** -8, 2.0 ** -23


def _table():
    """The finite numbers of E4M3 by their definition: sign, four exponent bits with bias 7, three of mantissa."""
    vals = {}
    for c in range(127):
        e, m = c >> 3, c & 7
        vals[c] = (m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
    return torch.tensor([vals[c] for c in range(127)], dtype=torch.float64)


def _codes_by_search(x):
    """(values q s, scales) of rows, by search in the table in 64 bits; x finite."""
    T, K = x.shape
    table = _table()
    nb = -(-K // 128)
    out, scales = torch.zeros(T, K, dtype=torch.float64), torch.ones(nb, T, dtype=torch.float64)
    for b in range(nb):
        v = x[:, b * 128:(b + 1) * 128].double()
        for t in range(T):
            top = v[t].abs().max().item()
            s = 1.0
            if top > 0:
                e = math.frexp(top / 448)[1]              # 64 bits: exact to far below a bf16 or fp32 step
                s = 2.0 ** (e - 1) if top == 448 * 2.0 ** (e - 1) else 2.0 ** e
                s = max(s, 2.0 ** -126)
            u = v[t].abs() / s
            i = torch.searchsorted(table, u).clamp(max=126)
            lo = (i - 1).clamp(min=0)
            dl, dh = u - table[lo], table[i] - u
            pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, i)
            pick = torch.where(table[pick] * s < 2.0 ** 128, pick, lo)      # a finite value stays finite
            out[t, b * 128:(b + 1) * 128] = table[pick] * s * v[t].sign()
            scales[b, t] = s
    return out, scales


def _weight8(codes, scale):
    n, k = codes.shape
    return codes.cpu().double() * scale.cpu().double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _make(shape, seed, dtype=torch.bfloat16, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[0], 1, generator=g))).to(dtype)


def _assert_product(y, a, b, extra=None, terms=0):
    """y [M, N] bf16 against a [M, K] b [K, N] (+ a2 b2) in 64 bits."""
    want, size = a @ b, a.abs() @ b.abs()
    K = a.shape[1]
    if extra is not None:
        want, size = want + extra[0] @ extra[1], size + extra[0].abs() @ extra[1].abs()
        K += extra[0].shape[1]
    tol = BF16 * want.abs() + (K + 2 * (K // 128 + 1) + 4 + terms) * EPS32 * size * (1 + BF16) + 1e-38
    diff = (y.cpu().double() - want).abs()
    assert y.dtype == torch.bfloat16 and (diff <= tol).all(), f"worst excess {(diff - tol).max().item()}"


# ------------------------------------------------------------------ rows
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 128), (3, 127), (2, 129), (9, 200), (5, 1032), (17, 2056)])
def test_rows_are_the_nearest_codes(T, K, dtype, dev):
    x = _make((T, K), T * 1000 + K, dtype)
    x[0, : min(K, 3)] = 0
    codes, scale = quantize_fp8_rows(x.to(dev))
    want, scales = _codes_by_search(x)
    assert codes.shape == (T, K) and codes.dtype == torch.float8_e4m3fn and codes.stride(0) % 16 == 0
    assert torch.equal(scale.cpu().double(), scales)
    # in fp32 every value of the codes is exact; bf16 holds them too
    assert torch.equal(dequantize_fp8_rows(codes, scale, torch.float32).cpu().double(), want)
    assert torch.equal(dequantize_fp8_rows(codes, scale).cpu().double(), want)


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_ties_borders_and_extremes(dev):
    """Ties to even, a maximum of exactly 448 2^j and just above, zeros, the smallest and largest numbers, subnormal ones."""
    x = torch.zeros(8, 256)
    x[0, :6] = torch.tensor([448.0, 1.0625, 1.1875, 17.0, 19.0, -17.0])           # scale 1, ties between codes
    x[1, :2] = torch.tensor([450.0, 3.0])                                         # just above 448: scale 2
    x[2, 0] = torch.finfo(torch.bfloat16).max
    x[3, :2] = torch.tensor([2.0 ** -133, -(2.0 ** -130)])                        # bf16 subnormals: scale 2^-126
    x[4, 130] = 3.5
    x[5, :3] = torch.tensor([448.0 * 2 ** -20, 2.0 ** -30, 2.0 ** -31])
    x[6, :3] = torch.tensor([256.0, 2.0 ** -9, 2.0 ** -10])                       # smallest code, half of it (a tie with zero)
    x = x.bfloat16()
    codes, scale = quantize_fp8_rows(x.to(dev))
    want, scales = _codes_by_search(x)
    assert torch.equal(scale.cpu().double(), scales) and scale[0, 7] == 1 and scale[0, 0] == 1 and scale[0, 1] == 2
    assert torch.equal(dequantize_fp8_rows(codes, scale, torch.float32).cpu().double(), want)


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_nan_and_infinity_leave_their_neighbours_alone(dev):
    x = _make((4, 300), 3)
    y = x.clone()
    y[0, 5], y[1, 130], y[2, 299], y[3, :128] = float("nan"), float("inf"), float("-inf"), float("nan")
    x[0, 5] = x[1, 130] = x[2, 299] = 0                   # what the others' maximum is taken over
    x[3, :128] = 0
    want, got = (dequantize_fp8_rows(*quantize_fp8_rows(t.to(dev))).cpu() for t in (x, y))
    odd = ~torch.isfinite(y)
    assert torch.equal(torch.isnan(got), odd) and torch.equal(got[~odd], want[~odd])


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_of_other_strides(dev):
    base = _make((12, 700), 5).to(dev)
    for x in (base[:, 1:650], base[::2, 8:520], base.t()[:300], base[3:4].expand(5, 700), base[:, :1].expand(12, 256)):
        codes, scale = quantize_fp8_rows(x)
        want, scales = quantize_fp8_rows(x.clone().contiguous())
        assert torch.equal(scale, scales) and torch.equal(codes.view(torch.uint8), want.view(torch.uint8))
        # codes and scales of other strides back
        odd = torch.empty(codes.shape[0], codes.shape[1] + 3, dtype=torch.uint8, device=dev)[:, 3:].view(torch.float8_e4m3fn)
        odd.view(torch.uint8).copy_(codes.view(torch.uint8))
        assert torch.equal(dequantize_fp8_rows(odd, scale.t().contiguous().t()), dequantize_fp8_rows(codes, scale))


@pytest.mark.parametrize("dev", DEVICES)
def test_rows_none(dev):
    codes, scale = quantize_fp8_rows(torch.empty(0, 256, dtype=torch.bfloat16, device=dev))
    assert codes.shape == (0, 256) and scale.shape == (2, 0) and dequantize_fp8_rows(codes, scale).shape == (0, 256)


def test_refusals():
    x = torch.randn(4, 256).bfloat16()
    codes, scale = quantize_fp8_rows(x)
    w, ws = quantize_fp8_weight(torch.randn(130, 256))
    for bad, kind in ((x[0], ValueError), (torch.zeros(3, 0), ValueError), (x.double(), TypeError), (x.int(), TypeError)):
        with pytest.raises(kind):
            quantize_fp8_rows(bad)
    for args, kind in (((codes.view(torch.uint8), scale), TypeError), ((codes, scale.t()), ValueError), ((codes, scale.double()), ValueError),
                       ((codes, scale[:1]), ValueError), ((codes[0], scale), ValueError), ((codes, scale, torch.float64), TypeError)):
        with pytest.raises(kind):
            dequantize_fp8_rows(*args)
    for bad in (torch.zeros(0, 5), torch.zeros(3)):
        with pytest.raises(ValueError):
            quantize_fp8_weight(bad)
    for args, kind in (((codes[:, :128], scale[:1], w, ws), ValueError), ((codes, scale, w, ws[:1]), ValueError),
                       ((codes, scale, w.view(torch.uint8), ws), TypeError), ((codes, scale[:, :3], w, ws), ValueError)):
        with pytest.raises(kind):
            fp8_gemm(*args)
    with pytest.raises(ValueError):
        fp8_gemm(codes, scale, w, ws, a2=torch.zeros(4, 8).bfloat16(), b2=torch.zeros(8, 130).bfloat16())
    for args in ((x[:, :200], w, ws), (x, w, ws[:, :1]), (x.to("meta"), w, ws)):
        with pytest.raises(ValueError):
            fp8_linear(*args)
    for args, kw in (((torch.zeros(5, 8).bfloat16(), codes, scale), {}), ((torch.zeros(4).bfloat16(), codes, scale), {}),
                     ((torch.zeros(4, 8).bfloat16(), codes, scale), dict(out=torch.zeros(8, 255))),
                     ((torch.zeros(4, 8).bfloat16(), codes, scale), dict(out=torch.zeros(8, 256).bfloat16()))):
        with pytest.raises(ValueError):
            fp8_adapter_grad(*args, **kw)


# ------------------------------------------------------------------ weights and products
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (130, 200), (300, 129)])
def test_weight_codes_are_half_a_step_off(N, K, dev):
    w = _make((N, K), N + K, torch.float32, 1.0)
    w[0, : K // 2] = 0
    codes, scale = quantize_fp8_weight(w.to(dev))
    assert codes.shape == (N, K) and codes.stride(0) % 16 == 0 and scale.shape == (-(-N // 128), -(-K // 128))
    back = _weight8(codes, scale)
    s = scale.cpu().double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    # half a step of E4M3, 2^-4 relative or 2^-10 of the scale below its normal range, and the fp32 division's rounding
    assert ((back - w.double()).abs() <= torch.maximum(w.double().abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -20)).all()
    got = dequantize_fp8_weight(codes, scale).cpu().double()
    assert ((got - back).abs() <= BF16 * back.abs()).all()


PRODUCTS = [(1, 1, 1), (1, 16, 128), (5, 130, 300), (33, 128, 256), (128, 128, 128), (129, 257, 384), (200, 520, 1032), (300, 1000, 136)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("M,N,K", PRODUCTS)
def test_product(M, N, K, trans, dev):
    x = _make((M, K), M + N + K, spread=1.0)
    codes, scale = quantize_fp8_rows(x.to(dev))
    w, ws = quantize_fp8_weight(_make((K, N) if trans else (N, K), 7 * M + K, torch.float32, 1.0).to(dev))
    y = fp8_gemm(codes, scale, w, ws, trans_w=trans)
    x8, w8 = dequantize_fp8_rows(codes, scale, torch.float32).cpu().double(), _weight8(w, ws)
    _assert_product(y, x8, w8 if trans else w8.t())


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [128, 192, 256])
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("rank", [0, 8, 16, 72])
def test_product_tiles_and_extension(tile, trans, rank, monkeypatch):
    """Every tile size whatever the rule picks, with and without the bf16 K-extension, more tiles than workers."""
    from axolotl_b200.ops import fp8

    monkeypatch.setattr(fp8, "_tile", lambda *a: tile)
    for M, N, K in ((130, 264, 200), (2100, 2600, 256)):
        x = _make((M, K), M, spread=1.0).cuda()
        codes, scale = quantize_fp8_rows(x)
        w, ws = quantize_fp8_weight(_make((K, N) if trans else (N, K), K, torch.float32, 1.0).cuda())
        a2 = _make((M, rank), 3, spread=0.0).cuda() if rank else None
        b2 = _make((rank, N) if trans else (N, rank), 4, spread=0.0).cuda() if rank else None
        y = fp8_gemm(codes, scale, w, ws, trans_w=trans, a2=a2, b2=b2)
        x8, w8 = dequantize_fp8_rows(codes, scale, torch.float32).cpu().double(), _weight8(w, ws)
        ext = (a2.cpu().double(), (b2 if trans else b2.t()).cpu().double()) if rank else None
        _assert_product(y, x8, w8 if trans else w8.t(), ext)


@pytest.mark.parametrize("dev", DEVICES)
def test_product_of_nan_rows(dev):
    """A NaN in one row of the input is that row's alone; a NaN code of the weight is its output column's."""
    x = _make((140, 256), 1, spread=0.0)
    w, ws = quantize_fp8_weight(_make((136, 256), 2, torch.float32, 0.0).to(dev))
    clean = fp8_linear(x.to(dev), w, ws)
    x[3, 17], x[139, 200] = float("nan"), float("inf")
    got = fp8_linear(x.to(dev), w, ws)
    rows = torch.tensor([i not in (3, 139) for i in range(140)])
    assert torch.isnan(got[~rows]).all() and torch.equal(got[rows], clean[rows])
    wn = w.clone()
    wn[100, 9] = float("nan")
    col = fp8_linear(_make((140, 256), 1, spread=0.0).to(dev), wn, ws)
    cols = torch.arange(136) != 100
    assert torch.isnan(col[:, 100]).all() and torch.equal(col[:, cols], clean[:, cols])


# ------------------------------------------------------------------ layers
def _rows8(x):
    return dequantize_fp8_rows(*quantize_fp8_rows(x.cpu()), dtype=torch.float32).double()


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("shape,N", [((3, 7, 200), 136), ((1, 128), 16), ((260, 264), 520)])
def test_linear_and_its_input_gradient(shape, N, dev):
    K = shape[-1]
    x = _make((math.prod(shape[:-1]), K), K, spread=0.5).view(shape)
    dy = _make((math.prod(shape[:-1]), N), N, spread=0.5).view(*shape[:-1], N) * 1e-3
    dy[..., :1, :] = 0
    w, ws = quantize_fp8_weight(_make((N, K), 5, torch.float32, 0.0).to(dev))
    xl = x.to(dev).requires_grad_(True)
    y = fp8_linear(xl, w, ws)
    (dx,) = torch.autograd.grad(y, [xl], dy.to(dev))
    w8 = _weight8(w, ws)
    assert y.shape == (*shape[:-1], N) and dx.shape == shape
    _assert_product(y.reshape(-1, N), _rows8(x.reshape(-1, K)), w8.t())
    _assert_product(dx.reshape(-1, K), _rows8(dy.reshape(-1, N)), w8)


@pytest.mark.parametrize("dev", DEVICES)
def test_linear_bias_and_its_gradient(dev):
    x, w32 = _make((40, 256), 1, spread=0.0), _make((64, 256), 2, torch.float32, 0.0)
    w, ws = quantize_fp8_weight(w32.to(dev))
    bias = _make((1, 64), 3, spread=0.0)[0].to(dev).requires_grad_(True)
    y = fp8_linear(x.to(dev), w, ws, bias)
    assert torch.equal(y, fp8_linear(x.to(dev), w, ws) + bias)
    dy = _make((40, 64), 4, spread=0.0)
    (db,) = torch.autograd.grad(y, [bias], dy.to(dev))
    want = dy.double().sum(0)
    assert ((db.cpu().double() - want).abs() <= BF16 * want.abs() + 40 * EPS32 * dy.double().abs().sum(0)).all()


@pytest.mark.parametrize("dev", DEVICES)
def test_linear_gradient_by_differences(dev):
    """Where every value is its own code (small integers; weights that are powers of two) the layer is linear without rounding: the
    gradient is what differences give, exactly."""
    g = torch.Generator().manual_seed(0)
    x = torch.randint(-2, 3, (6, 128), generator=g).bfloat16()
    x[:, 0] = 2                                            # the block's maximum stays where it is
    w = torch.where(torch.rand(16, 128, generator=g) < 0.1, 0.5, 0.0)
    w[0, 0] = 0.5
    codes, scale = quantize_fp8_weight(w.to(dev))
    dy = torch.randint(-2, 3, (6, 16), generator=g).bfloat16()
    xl = x.to(dev).requires_grad_(True)
    (dx,) = torch.autograd.grad(fp8_linear(xl, codes, scale), [xl], dy.to(dev))
    for t, k in ((0, 1), (3, 77), (5, 127)):
        step = torch.zeros(6, 128).bfloat16()
        step[t, k] = 1
        up, down = (fp8_linear((x + d * step).to(dev), codes, scale).cpu().double() for d in (1, -1))
        assert ((up - down) * dy.double()).sum() / 2 == dx[t, k].cpu().double()


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,N,blocks", [(1, 256, 128, ((0, 128, 0, 8),)), (70, 520, 264, ((0, 200, 0, 8), (200, 64, 8, 8))),
                                          (600, 1024, 640, ((0, 640, 0, 16),)), (700, 264, 1032, ((128, 904, 0, 32),)),
                                          (90, 131, 77, ((0, 77, 0, 8),)), (20, 256, 128, ((0, 128, 0, 72),))])
@pytest.mark.parametrize("masters", [torch.float32, torch.bfloat16])
def test_lora_linear_and_its_gradients(T, K, N, blocks, masters):
    R = sum(b[3] for b in blocks)
    x, dy = _make((T, K), 1, spread=0.5), _make((T, N), 2, spread=0.5) * 1e-2
    dy[: T // 3] = 0
    w, ws = quantize_fp8_weight(_make((N, K), 3, torch.float32, 0.0).cuda())
    A = _make((R, K), 4, torch.float32, 0.0) * K ** -0.5
    B = torch.zeros(N, R)
    for r0, rows, c0, r in blocks:
        B[r0:r0 + rows, c0:c0 + r] = _make((rows, r), 5, torch.float32, 0.0) * 0.1
    A16, B16 = A.bfloat16(), B.bfloat16()
    xl, Al, Bl = x.cuda().requires_grad_(True), A.to(masters).cuda().requires_grad_(True), B.to(masters).cuda().requires_grad_(True)
    y = fp8_lora_linear(xl, w, ws, Al, Bl, A16.cuda(), B16.cuda(), 2.0, blocks)
    dx, dA, dB = torch.autograd.grad(y, [xl, Al, Bl], dy.cuda())
    a, b, w8, x64, dy64 = A16.double(), B16.double(), _weight8(w, ws), x.double(), dy.double()
    x8 = _rows8(x)
    low, tall = 2 * x64 @ a.t(), 2 * dy64 @ b
    # the two low-rank products are rounded to bf16 after sums of K or N terms: each is off by 2^-8 of itself and that
    low_e = BF16 * low.abs() + (K + 2) * EPS32 * 2 * x64.abs() @ a.abs().t()
    tall_e = BF16 * tall.abs() + (N + 2) * EPS32 * 2 * dy64.abs() @ b.abs()

    def near(got, want, off, terms):
        tol = off + terms * EPS32 * (want.abs() + off)
        assert ((got.cpu().double() - want).abs() <= tol + 1e-30).all()

    want = x8 @ w8.t() + low @ b.t()
    size = x8.abs() @ w8.abs().t() + low.abs() @ b.abs().t()
    near(y, want, BF16 * want.abs() + (low_e @ b.abs().t() + (K + R + 40) * EPS32 * size) * (1 + BF16), 4)
    dy8 = _rows8(dy)
    want = dy8 @ w8 + tall @ a
    size = dy8.abs() @ w8.abs() + tall.abs() @ a.abs()
    near(dx, want, BF16 * want.abs() + (tall_e @ a.abs() + (N + R + 40) * EPS32 * size) * (1 + BF16), 4)
    assert dA.dtype == dB.dtype == masters
    half = BF16 if masters == torch.bfloat16 else 0.0       # and the gradients' own rounding
    want, size = tall.t() @ x8, tall.abs().t() @ x8.abs()
    near(dA, want, half * (1 + BF16) * want.abs() + (1 + half) * tall_e.t() @ x8.abs() + (T + 8) * EPS32 * size, 4)
    wantB, size = dy64.t() @ low, dy64.abs().t() @ low.abs()
    offB = half * (1 + BF16) * wantB.abs() + (1 + half) * dy64.abs().t() @ low_e + (T + 8) * EPS32 * size
    for r0, rows, c0, r in blocks:
        near(dB[r0:r0 + rows, c0:c0 + r], wantB[r0:r0 + rows, c0:c0 + r], offB[r0:r0 + rows, c0:c0 + r], 4)
    assert (dB.cpu()[B == 0] == 0).all() or len(blocks) == 1


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("T,K,R", [(1, 128, 8), (77, 200, 16), (300, 1000, 40), (1030, 264, 64), (2100, 136, 5), (129, 4360, 1), (700, 520, 200)])
def test_adapter_gradient_from_saved_rows(T, K, R, dev):
    x, t = _make((T, K), T + K, spread=0.5), _make((T, R), R, spread=0.5)
    codes, scale = quantize_fp8_rows(x.to(dev))
    want, size = t.double().t() @ _rows8(x), t.double().abs().t() @ _rows8(x).abs()
    tol = (T + 16) * EPS32 * size + 1e-30                   # T products in fp32 sums
    got = fp8_adapter_grad(t.to(dev), codes, scale)
    assert got.dtype == torch.float32 and ((got.cpu().double() - want).abs() <= tol).all()
    base = _make((R, K), 9, torch.float32, 0.0)
    into = base.clone().to(dev)
    assert fp8_adapter_grad(t.to(dev), codes, scale, out=into) is into
    assert ((into.cpu().double() - base.double() - want).abs() <= tol + (T + 16) * EPS32 * base.double().abs()).all()
    # a result and codes of other strides, the same sums
    wide = torch.zeros(K, R, device=dev).t()
    assert torch.equal(fp8_adapter_grad(t.to(dev), codes, scale, out=wide), got)
    turned = scale.t().contiguous().t()
    assert torch.equal(fp8_adapter_grad(t.t().contiguous().t().to(dev), codes, turned), got)


# ------------------------------------------------------------------ checkpoints
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_store_gives_back_the_coded_values(dtype, dev):
    from axolotl_b200.train.activation_memory import make_store

    store = make_store("fp8", dev)
    for shape in ((5, 300), (2, 3, 128), (7,), (0, 64), ()):
        x = torch.randn(shape).to(dtype).to(dev)
        got = store.get(store.put(x))
        assert got.shape == x.shape and got.dtype == dtype and got.device == x.device
        if x.dim() and x.numel():
            want = _codes_by_search(x.cpu().reshape(-1, shape[-1]))[0].to(dtype).view(shape)
            assert torch.equal(got.cpu(), want)
        else:
            assert torch.equal(got, x)
    ids = torch.arange(6, device=dev)
    h = store.put(ids)
    assert torch.equal(store.get(h), ids)
    with pytest.raises(RuntimeError):
        store.get(h)


@pytest.mark.parametrize("dev", DEVICES)
def test_checkpoint_recomputes_from_the_coded_input(dev):
    """The forward pass sees the exact layer input, the recomputation the coded one: gradients are those of the layer at ``x8``."""
    from axolotl_b200.train.activation_memory import make_store, offloaded_checkpoint

    g = torch.Generator().manual_seed(2)
    W = torch.randn(128, 128, generator=g).to(dev).requires_grad_(True)
    x = torch.randn(64, 128, generator=g).to(dev).requires_grad_(True)
    dy = torch.randn(64, 128, generator=g).to(dev)
    layer = lambda h, r: (torch.tanh(h @ W), h if r is None else r)
    y, _ = offloaded_checkpoint(layer, make_store("fp8", dev), (x, None))
    assert torch.equal(y, torch.tanh(x @ W))
    y.backward(dy)
    x8 = dequantize_fp8_rows(*quantize_fp8_rows(x.detach()), dtype=torch.float32).requires_grad_(True)
    W2 = W.detach().clone().requires_grad_(True)
    torch.tanh(x8 @ W2).backward(dy)
    assert torch.equal(x.grad, x8.grad) and torch.equal(W.grad, W2.grad)


# ------------------------------------------------------------------ in the framework
@pytest.mark.parametrize("dev", DEVICES)
def test_fused_linear_in_8_bits(dev):
    """The module with its adapter: the forward pass is the layer's definition, a change of dtype leaves the codes alone, dequantising and
    merging use the coded weight."""
    from axolotl_b200.models.layers import FusedLinear

    dtype = torch.bfloat16 if dev == "cuda" else torch.float32
    lin = FusedLinear(200, [136, 64], ["a", "b"], dtype=dtype, device=dev)
    with torch.no_grad():
        lin.weight.copy_(_make((200, 200), 1, spread=0.0))
    lin.quantize_fp8_()
    before = lin.weight.data.clone()
    lin.quantize_fp8_()
    lin.add_lora(8, 16, targets=["b"])
    with torch.no_grad():
        lin.lora_B[136:].normal_(0, 0.05)
    lin.refresh_shadows()
    lin.to(torch.bfloat16)
    assert lin.weight.dtype == torch.uint8 and torch.equal(lin.weight.data, before) and not lin.weight.requires_grad
    lin.to(dtype)
    w8 = _weight8(lin.weight.data.view(torch.float8_e4m3fn), lin.weight._axb_quant.scale)
    x = _make((70, 200), 2, dtype, 0.3)
    y = lin(x.to(dev)).detach().cpu().double()
    A, B = (t.detach().cpu().bfloat16().double() if dev == "cuda" else t.detach().double() for t in (lin.lora_A, lin.lora_B))
    low = lin.scaling * x.double() @ A.t()
    base = _rows8(x) @ w8.t()
    size = _rows8(x).abs() @ w8.abs().t() + lin.scaling * (x.double().abs() @ A.abs().t()) @ B.abs().t()
    # the product and, on the device, the low-rank one are rounded to bf16; sums in fp32 (the adapter's masters stay fp32 on the CPU)
    tol = BF16 * (base.abs() + 2 * (low @ B.t()).abs() + low.abs() @ B.abs().t()) + 300 * EPS32 * size
    assert ((y - base - low @ B.t()).abs() <= tol).all()
    dense = lin._dense_weight().cpu().double()
    assert ((dense - w8).abs() <= BF16 * w8.abs()).all()
    lin.merge_lora_()
    assert lin.weight.dtype == torch.bfloat16 and getattr(lin.weight, "_axb_quant", None) is None and lin.merged


@pytest.mark.parametrize("dev", DEVICES)
def test_dropout_and_dora_on_8_bit_weights_run(dev):
    from axolotl_b200.models.layers import FusedLinear

    dtype = torch.bfloat16 if dev == "cuda" else torch.float32
    for kw in (dict(dropout=0.5), dict(use_dora=True)):
        lin = FusedLinear(128, [64], ["a"], dtype=dtype, device=dev)
        with torch.no_grad():
            lin.weight.copy_(_make((64, 128), 1, spread=0.0))
        lin.quantize_fp8_()
        lin.add_lora(8, 16, **kw)
        x = _make((16, 128), 2, dtype, 0.0).to(dev).requires_grad_(True)
        base = fp8_linear(x.detach(), lin.weight.data.view(torch.float8_e4m3fn), lin.weight._axb_quant.scale)
        y = lin.train()(x)                                 # B is zero: the adapter adds nothing yet
        assert ((y - base).abs() <= 2 * BF16 * base.abs()).all()
        y.sum().backward()
        assert torch.isfinite(x.grad).all() and lin.lora_B.grad.abs().sum() > 0


def test_base_weights_fp8_is_checked():
    from axolotl_b200.config.load import load_cfg

    base = {"model_preset": "tiny-llama", "lora_r": 8, "lora_alpha": 16, "lora_target_linear": True, "sequence_len": 64,
            "micro_batch_size": 1, "gradient_accumulation_steps": 1, "max_steps": 1, "learning_rate": 1e-3, "output_dir": "unused",
            "device": "cpu", "datasets": [{"path": "synthetic", "type": "_synthetic"}], "base_weights_fp8": True}
    for bad in (dict(adapter="qlora", load_in_4bit=True), dict(adapter=None), dict(adapter="mora"), dict(adapter="lora", tensor_parallel_size=2)):
        with pytest.raises(ValueError):
            load_cfg({**base, **bad})
    with pytest.raises(ValueError):
        load_cfg({**base, "adapter": "lora", "activation_offloading": "fp8"})                       # without checkpointing
    with pytest.raises(ValueError):
        load_cfg({**base, "adapter": "lora", "gradient_checkpointing": True, "activation_offloading": "int8"})
    cfg = load_cfg({**base, "adapter": "lora", "gradient_checkpointing": True, "activation_offloading": "fp8"})
    assert cfg["base_weights_fp8"] is True and cfg["activation_offloading"] == "fp8"


@pytest.mark.parametrize("dev", DEVICES)
def test_training_run_with_8_bit_weights_and_checkpoints(dev, tmp_path):
    """The training entry point with both: every projection of the layers is in 8 bits, an adapter is written, the frozen codes are what
    they were."""
    from axolotl_b200.config.load import load_cfg
    from axolotl_b200.train.activation_memory import Fp8Store
    from axolotl_b200.train.run import train

    cfg = load_cfg({"model_preset": "tiny-llama", "adapter": "lora", "base_weights_fp8": True, "lora_r": 8, "lora_alpha": 16,
                    "lora_target_linear": True, "sequence_len": 128, "micro_batch_size": 2, "gradient_accumulation_steps": 1, "max_steps": 3,
                    "learning_rate": 1e-3, "optimizer": "adamw_torch", "lr_scheduler": "constant", "output_dir": str(tmp_path / "o"),
                    "device": dev, "logging_steps": 1, "sample_packing": True, "gradient_checkpointing": True, "activation_offloading": "fp8",
                    "datasets": [{"path": "synthetic", "type": "_synthetic", "length": 16, "min_length": 32, "max_length": 64,
                                  "max_input_id": 400}]})
    model, _, trainer = train(cfg)
    assert all(m.weight.dtype == torch.uint8 for n, m in model.fused_linears() if n.startswith("layers."))
    assert isinstance(model.ckpt_store, Fp8Store) and model.ckpt_store.bytes_out > 0
    assert all(math.isfinite(l["loss"]) for l in trainer.log_history if "loss" in l)
    assert (tmp_path / "o" / "adapter_model.safetensors").exists()


@pytest.mark.gpu
def test_model_gradients_beside_the_dense_model():
    """A two-layer model with 8-bit projections, adapters and 8-bit checkpoints beside the same model with the coded weights in bf16:
    adapter gradients and logits. Every product of a layer quantises its operands with a relative rms error of 2^-4 / sqrt(3) / 1.4 = 2.6 %;
    a gradient passes about 7 products a layer and direction and the checkpoint, 2 x 2 x 8 = 32 of them: sqrt(32) 2.6 % = 15 %, tested at
    25 %."""
    from axolotl_b200.models.config import preset
    from axolotl_b200.models.lora import LoraSpec, inject_lora, quantize_base_fp8_
    from axolotl_b200.models.transformer import CausalLM
    from axolotl_b200.ops import _lib

    cfg = preset("tiny-llama", num_hidden_layers=2, vocab_size=512)
    grads, logits = [], []
    for coded in (True, False):
        model = CausalLM(cfg, dtype=torch.bfloat16, device="cuda").init_weights(0)
        saved = quantize_base_fp8_(model)
        assert saved > 0
        if not coded:
            for n, m in model.fused_linears():
                if n.startswith("layers."):
                    m.dequantize_()
        torch.manual_seed(1)
        inject_lora(model, LoraSpec(r=8, lora_alpha=16, target_modules=["q_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj"]))
        with torch.no_grad():
            for _, m in model.fused_linears():
                if m.lora_B is not None:
                    for _, B in m.peft_tensors().values():
                        B.normal_(0, 0.05)
        model.refresh_lora_shadows()
        model.enable_gradient_checkpointing(True, offload="fp8" if coded else None)
        model.train()
        ids = torch.randint(0, 512, (2, 160), generator=torch.Generator().manual_seed(3)).cuda()
        out = model(ids, labels=ids)
        out.loss.backward()
        grads.append({n: p.grad.float() for n, p in model.named_parameters() if p.grad is not None})
        with torch.no_grad():
            logits.append(model.eval()(ids, return_logits=True).logits.float())
    _lib.check_status()
    assert grads[0].keys() == grads[1].keys() and len(grads[0]) >= 8
    rel = lambda a, b: ((a - b).norm() / b.norm()).item()
    assert rel(logits[0], logits[1]) < 0.25
    for n, g in grads[1].items():
        assert rel(grads[0][n], g) < 0.25, n


@pytest.mark.gpu
def test_generation_with_8_bit_weights():
    """Prefill and cached steps run the 8-bit products; the same prompts give the same tokens."""
    from axolotl_b200.models.config import preset
    from axolotl_b200.models.kv_cache import generate_cached
    from axolotl_b200.models.lora import quantize_base_fp8_
    from axolotl_b200.models.transformer import CausalLM

    model = CausalLM(preset("tiny-llama", num_hidden_layers=2, vocab_size=512), dtype=torch.bfloat16, device="cuda").init_weights(0).eval()
    quantize_base_fp8_(model)
    prompts = [[5, 9, 200, 31], [7] * 19, [1]]
    out = generate_cached(model, prompts, 5)
    assert [len(o) for o in out] == [5, 5, 5] and all(0 <= t < 512 for o in out for t in o)
    assert generate_cached(model, prompts, 5) == out


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 16, 17, 32, 40, 64])
@pytest.mark.parametrize("N,K,rank", [(1, 128, 0), (128, 2048, 0), (130, 1000, 8), (1000, 4096, 16), (4200, 4104, 72), (20000, 264, 0)])
def test_few_tokens(T, N, K, rank, monkeypatch):
    """A few tokens: every split of K over a cluster, K and N that end inside a block, the bf16 extension, rows of x that do
    not start on 16 bytes."""
    from axolotl_b200.ops import _lib, fp8

    x = _make((T, K + 1), T + K, spread=1.0).cuda()[:, : K]
    x[0, 0] = 0
    w, ws = quantize_fp8_weight(_make((N, K), N, torch.float32, 1.0).cuda())
    a2 = _make((T, rank), 3, spread=0.0).cuda() if rank else None
    b2 = _make((N, rank), 4, spread=0.0).cuda() if rank else None
    for rows in (x, x.contiguous()):
        for few in (2, 1, 0):                              # quantised inside, before, and by tiles
            monkeypatch.setattr(fp8, "_few", lambda *a: few)
            y, q = fp8._product(rows, w, ws, a2=a2, b2=b2)
            _lib.check_status()
            assert (q is None) == (few == 2)
            ext = (a2.cpu().double(), b2.t().cpu().double()) if rank else None
            _assert_product(y, _rows8(x), _weight8(w, ws).t(), ext, terms=16)


@pytest.mark.gpu
def test_few_tokens_with_nan_and_infinity():
    from axolotl_b200.ops import fp8

    x = _make((20, 512), 1, spread=0.0).cuda()
    w, ws = quantize_fp8_weight(_make((256, 512), 2, torch.float32, 0.0).cuda())
    clean = fp8._product(x, w, ws)[0]
    x[3, 17], x[19, 500] = float("nan"), float("-inf")
    got = fp8._product(x, w, ws)[0]
    rows = torch.tensor([i not in (3, 19) for i in range(20)])
    assert torch.isnan(got[~rows]).all() and torch.equal(got[rows], clean[rows])
    x = torch.zeros(2, 256, dtype=torch.bfloat16, device="cuda")
    x[0, 3], x[1, 5] = torch.finfo(torch.bfloat16).max, 2.0 ** -133
    w, ws = quantize_fp8_weight((torch.eye(256) * 2.0 ** -6).cuda())
    _assert_product(fp8._product(x, w, ws)[0], _rows8(x), _weight8(w, ws).t())


def test_adapter_gradient_of_no_rows():
    codes, scale = quantize_fp8_rows(torch.empty(0, 256, dtype=torch.bfloat16))
    assert torch.equal(fp8_adapter_grad(torch.empty(0, 8).bfloat16(), codes, scale), torch.zeros(8, 256))


@pytest.mark.gpu
def test_adapter_gradient_with_nan():
    """NaN codes reach the columns they stand in and no others."""
    x = _make((300, 384), 1, spread=0.0)
    t = _make((300, 16), 2, spread=0.0).cuda()
    clean = fp8_adapter_grad(t, *quantize_fp8_rows(x.cuda()))
    x[299, 5], x[0, 130] = float("inf"), float("nan")
    got = fp8_adapter_grad(t, *quantize_fp8_rows(x.cuda()))
    nan = torch.isnan(got).all(0).cpu()
    assert nan.nonzero().flatten().tolist() == [5, 130] and torch.isfinite(got[:, ~nan]).all()
    same = torch.ones(384, dtype=torch.bool)
    same[:256] = False                                     # blocks whose maximum may have been the value that is gone
    assert torch.equal(got[:, same], clean[:, same])


@pytest.mark.gpu
@pytest.mark.parametrize("T,R", [(70, 8), (600, 16), (600, 72)])
def test_lora_gradients_into_flat_buffers(T, R):
    """Parameters whose gradient has a place of its own get the same gradients there, added to what it holds."""
    K, N = 520, 264
    x, dy = _make((T, K), 1, spread=0.5).cuda(), (_make((T, N), 2, spread=0.5) * 1e-2).cuda()
    w, ws = quantize_fp8_weight(_make((N, K), 3, torch.float32, 0.0).cuda())
    A, B = (_make((R, K), 4, torch.float32, 0.0) * K ** -0.5).cuda(), (_make((N, R), 5, torch.float32, 0.0) * 0.1).cuda()
    grads = []
    for flat in (False, True):
        Al, Bl, xl = A.clone().requires_grad_(True), B.clone().requires_grad_(True), x.clone().requires_grad_(True)
        if flat:
            Al._axb_grad, Bl._axb_grad = torch.ones_like(A), torch.full_like(B, 2.0)
        y = fp8_lora_linear(xl, w, ws, Al, Bl, A.bfloat16(), B.bfloat16(), 0.5, ((0, N, 0, R),))
        y.backward(dy)
        assert (Al.grad is None) == flat and (Bl.grad is None) == flat
        grads.append((y, xl.grad, Al._axb_grad - 1 if flat else Al.grad, Bl._axb_grad - 2 if flat else Bl.grad))
    assert torch.equal(grads[0][0], grads[1][0])
    # t and dB are sums of fp32 atomics in any order: dB is off by (T + 8) 2^-23 of the sum of magnitudes, t may round to the bf16 number
    # next to it (2^-7), dx and dA with it, dx to the next bf16 number; adding to 1 or 2 rounds to 2^-23 of the sum
    t = (0.5 * dy.double() @ B.bfloat16().double()).abs() + (N + 8) * EPS32 * 0.5 * dy.double().abs() @ B.double().abs()
    low = (0.5 * x.double().abs() @ A.double().abs().t()) * (1 + 2 * BF16)
    offs = (2 * BF16 * (t @ A.double().abs() + grads[0][1].double().abs()), 2 * BF16 * t.t() @ (x.double().abs() * 1.1),
            (T + 8) * EPS32 * dy.double().abs().t() @ low)
    for a, b, off in zip(grads[0][1:], grads[1][1:], offs):
        assert ((a.double() - b.double()).abs() <= off + 4 * EPS32 * (2 + a.double().abs())).all()


@pytest.mark.gpu
def test_lora_without_gradients_keeps_nothing():
    """Under no_grad, or with a frozen adapter, the layer gives the same result; without an adapter gradient no codes are kept."""
    x = _make((40, 256), 1, spread=0.5).cuda()
    w, ws = quantize_fp8_weight(_make((128, 256), 3, torch.float32, 0.0).cuda())
    A, B = _make((8, 256), 4, spread=0.0).cuda() * 0.06, _make((128, 8), 5, spread=0.0).cuda() * 0.1
    args = (w, ws, A, B, A, B, 2.0, ((0, 128, 0, 8),))
    with torch.no_grad():
        want = fp8_lora_linear(x, *args)
    xl = x.clone().requires_grad_(True)
    y = fp8_lora_linear(xl, *args)
    assert torch.equal(y, want) and y.grad_fn.saved_tensors[0] is None
    (dx,) = torch.autograd.grad(y, [xl], torch.ones_like(y))
    assert torch.isfinite(dx).all()


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1, 8, 40, 100])
@pytest.mark.parametrize("lora", [False, True])
def test_generation_step_in_one_call_per_layer(batch, lora, monkeypatch):
    """A step of layers whose projections are in 8 bits (all of them, or some beside dense ones): the one-call form against the layers' own
    forward, the same kernels on the same operands. What differs is the norm before a dependent launch and the rotary embedding inside the
    attention launch: a few bf16 roundings (2^-8 each; 0.012 allows three), which the quantiser of the next product keeps or doubles on
    the few values that then round to the next code."""
    from axolotl_b200.models import decode_step
    from axolotl_b200.models.config import preset
    from axolotl_b200.models.kv_cache import KVCache, _DecodeMeta
    from axolotl_b200.models.lora import ALL_LINEAR, LoraSpec, inject_lora, quantize_base_fp8_
    from axolotl_b200.models.transformer import CausalLM
    from axolotl_b200.ops import _lib

    torch.manual_seed(5)
    m = CausalLM(preset("tiny-llama", vocab_size=512, num_hidden_layers=3), dtype=torch.bfloat16, device="cuda").init_weights(0).eval()
    m.layers[1].mlp.down_proj.quantize_fp8_()              # one alone in its layer
    for n, f in list(m.fused_linears()):
        if n.startswith(("layers.0.", "layers.2.")):
            f.quantize_fp8_()
    if lora:
        inject_lora(m, LoraSpec(r=8, lora_alpha=16, target_modules=list(ALL_LINEAR)))
        with torch.no_grad():
            for _, f in m.fused_linears():
                if f.lora_B is not None:
                    for _, B in f.peft_tensors().values():
                        B.normal_(0, 0.05)
        m.refresh_lora_shadows()
    pos = torch.randint(0, 60, (batch,), device="cuda")
    tok = torch.randint(0, 512, (batch,), device="cuda")
    at = m.layers[0].self_attn
    k, v = torch.randn(2, 3, batch, 64, at.Hk * at.D, device="cuda").bfloat16()
    done, outs = [], []
    real = decode_step.DecodeStep.layer
    monkeypatch.setattr(decode_step.DecodeStep, "layer", lambda self, *a: done.append(real(self, *a) if not force else None) or done[-1])
    for force in (False, True):
        cache = KVCache(m, batch, 64)
        cache.k.copy_(k)
        cache.v.copy_(v)
        with torch.no_grad():
            o = m(tok[None], pos.int()[None], attn_meta=_DecodeMeta(cache, torch.arange(batch, device="cuda"), pos, True), return_logits=True)
        outs.append((o.logits.float(), cache.k.float(), cache.v.float()))
    _lib.check_status()
    assert [d is not None for d in done] == [True] * 3 + [False] * 3
    for a, b in zip(*outs):
        assert torch.isfinite(a).all() and ((a - b).norm() <= 0.012 * b.norm()).item()


# ------------------------------------------------------------------ calls that ordinary use makes rarely
@pytest.mark.parametrize("dev", DEVICES)
def test_no_rows(dev):
    w, ws = quantize_fp8_weight(torch.randn(64, 128).to(dev))
    A, B = torch.randn(8, 128).bfloat16().to(dev), torch.randn(64, 8).bfloat16().to(dev)
    for call in (lambda x: fp8_linear(x, w, ws), lambda x: fp8_lora_linear(x, w, ws, A, B, A, B, 1.0, ((0, 64, 0, 8),))):
        x = torch.empty(2, 0, 128, dtype=torch.bfloat16, device=dev, requires_grad=True)
        y = call(x)
        assert y.shape == (2, 0, 64) and y.dtype == torch.bfloat16
        y.sum().backward()
        assert x.grad.shape == x.shape


@pytest.mark.parametrize("dev", DEVICES)
def test_weight_with_nan_and_infinity(dev):
    w = torch.randn(140, 260)
    w[3, 5], w[139, 259] = float("nan"), float("-inf")
    codes, scale = quantize_fp8_weight(w.to(dev))
    back = _weight8(codes, scale)
    odd = ~torch.isfinite(w)
    assert torch.isfinite(scale).all() and torch.equal(torch.isnan(back), odd)
    s = scale.cpu().double().repeat_interleave(128, 0)[:140].repeat_interleave(128, 1)[:, :260]
    ok = (back - w.double()).abs() <= torch.maximum(w.double().abs() * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -20)
    assert ok[~odd].all()


def test_lora_refusals():
    w, ws = quantize_fp8_weight(torch.randn(64, 128))
    x, A, B = torch.randn(4, 128).bfloat16(), torch.randn(8, 128).bfloat16(), torch.randn(64, 8).bfloat16()
    from axolotl_b200.ops.fp8 import _flat_blocks

    for blocks in ((), ((0, 65, 0, 8),), ((0, 64, 4, 8),), ((-1, 8, 0, 8),), ((0, 64, 0),)):
        with pytest.raises(ValueError):
            _flat_blocks(blocks, 64, 8)
    codes, scale = quantize_fp8_rows(x)
    for a2, b2 in ((A[:4, :8], None), (A[:3, :8], B), (A[:4, :8].to("meta"), B)):
        with pytest.raises(ValueError):
            fp8_gemm(codes, scale, w, ws, a2=a2, b2=b2)


@pytest.mark.gpu
def test_lora_refusals_on_the_device():
    w, ws = quantize_fp8_weight(torch.randn(64, 128).cuda())
    x, A, B = torch.randn(4, 128).bfloat16().cuda(), torch.randn(8, 128).bfloat16().cuda(), torch.randn(64, 8).bfloat16().cuda()
    blk = ((0, 64, 0, 8),)
    for args in ((A[:, :64], B, A[:, :64], B), (A, B[:32], A, B[:32]), (A, B, A.float(), B), (A, B, A[:4], B), (A, B, A.cpu(), B),
                 (A, B, A, B.cpu())):
        with pytest.raises(ValueError):
            fp8_lora_linear(x, w, ws, *args, 1.0, blk)
    with pytest.raises(ValueError):
        fp8_lora_linear(x, w, ws, A, B, A, B, 1.0, ((0, 64, 0, 16),))
    with pytest.raises(TypeError):
        fp8_linear(x.float(), w, ws)
    with pytest.raises(ValueError):
        fp8_linear(x, w.cpu(), ws.cpu())
    with pytest.raises(TypeError):
        fp8_gemm(*quantize_fp8_rows(x), w, ws, a2=A[:4, :8].float(), b2=B)
    with pytest.raises(TypeError):
        fp8_adapter_grad(torch.zeros(4, 8, device="cuda"), *quantize_fp8_rows(x))


@pytest.mark.gpu
def test_operands_off_a_16_byte_boundary():
    """Inputs, gradients, adapters and extensions that start in the middle of a 16-byte vector give what aligned ones give."""
    T, K, N, R = 300, 264, 136, 8

    def off(t):                                            # the same values one element further on
        wide = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        wide[1:].copy_(t.reshape(-1))
        return wide[1:].view(t.shape)

    x, dy = _make((T, K), 1, spread=0.3).cuda(), _make((T, N), 2, spread=0.3).cuda()
    w, ws = quantize_fp8_weight(_make((N, K), 3, torch.float32, 0.0).cuda())
    A, B = _make((R, K), 4, spread=0.0).cuda() * 0.06, _make((N, R), 5, spread=0.0).cuda() * 0.1
    assert off(x).data_ptr() % 16 and off(x).is_contiguous()
    res = []
    for f in (lambda t: t, off):
        xl = f(x).requires_grad_(True)
        y = fp8_linear(xl, w, ws)
        Al, Bl = f(A).requires_grad_(True), f(B).requires_grad_(True)
        z = fp8_lora_linear(f(x), w, ws, Al, Bl, f(A), f(B), 1.0, ((0, N, 0, R),))
        codes, scale = quantize_fp8_rows(f(x))
        res.append([y, torch.autograd.grad(y, [xl], f(dy))[0], z, *torch.autograd.grad(z, [Al, Bl], f(dy)),
                    fp8_gemm(codes, scale, w, ws, a2=f(dy)[:, :5], b2=f(B)[:, :5]), fp8_adapter_grad(f(dy)[:, :7], codes, scale)])
    for i, (a, b) in enumerate(zip(*res)):
        if i in (3, 4):                                    # sums of atomics in any order, of t that may round to its neighbour (2^-7)
            assert ((a.double() - b.double()).abs().max() <= 2.0 ** -6 * a.double().abs().max()).item()
        else:
            assert torch.equal(a, b), i


@pytest.mark.gpu
def test_captured_and_replayed_on_another_stream():
    """Graphs of the products (every form), the adapter's layer with its backward pass and the checkpoint store, replayed on new inputs beside
    one another: each gives what the eager call gives."""
    from axolotl_b200.train.activation_memory import make_store

    N, K, R = 264, 1032, 8
    w, ws = quantize_fp8_weight(_make((N, K), 3, torch.float32, 0.0).cuda())
    A, B = _make((R, K), 4, spread=0.0).cuda() * 0.06, _make((N, R), 5, spread=0.0).cuda() * 0.1
    calls = []
    for T in (1, 40, 64, 300):
        calls.append((T, lambda x: fp8_linear(x, w, ws)))
    calls.append((600, lambda x: fp8_lora_linear(x, w, ws, A, B, A, B, 1.0, ((0, N, 0, R),))))

    def stored(x):
        store = make_store("fp8", x.device)
        return store.get(store.put(x))

    def trained(x):
        xl = x.detach().requires_grad_(True)
        y = fp8_linear(xl, w, ws)
        return torch.autograd.grad(y, [xl], torch.ones_like(y))[0]

    calls += [(77, stored), (130, trained)]
    stream = torch.cuda.Stream()
    graphs = []
    for i, (T, f) in enumerate(calls):
        x = _make((T, K), i, spread=0.3).cuda()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            with torch.no_grad() if f is not trained else torch.enable_grad():
                f(x)
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            with torch.no_grad() if f is not trained else torch.enable_grad():
                out = f(x)
        graphs.append((g, x, out, f))
    for i, (g, x, _, _) in enumerate(graphs):
        x.copy_(_make(tuple(x.shape), 100 + i, spread=0.3))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        for _ in range(2):
            for g, _, _, _ in graphs:
                g.replay()
    torch.cuda.synchronize()
    for i, (g, x, out, f) in enumerate(graphs):
        with torch.no_grad() if f is not trained else torch.enable_grad():
            assert torch.equal(out, f(x)), i


@pytest.mark.gpu
def test_results_repeat_bit_for_bit():
    """Nothing but t and dB of an adapter is summed in an order that may change."""
    x = _make((700, 1032), 1, spread=0.3).cuda()
    w, ws = quantize_fp8_weight(_make((520, 1032), 2, torch.float32, 0.0).cuda())
    codes, scale = quantize_fp8_rows(x)
    t = _make((700, 16), 3, spread=0.0).cuda()
    for f in (lambda: fp8_gemm(codes, scale, w, ws), lambda: fp8_linear(x[:5], w, ws), lambda: fp8_linear(x[:60], w, ws),
              lambda: fp8_adapter_grad(t, codes, scale)):
        first = f()
        assert all(torch.equal(first, f()) for _ in range(5))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_bias_in_another_type(dtype, dev):
    """The result and the gradient that comes back stay bf16: the sum is rounded once, and dx is what it is without a bias."""
    T, K, N, R = 40, 256, 64, 8
    x, dy = _make((T, K), 1, spread=0.0).to(dev), _make((T, N), 2, spread=0.0).to(dev)
    w, ws = quantize_fp8_weight(_make((N, K), 3, torch.float32, 0.0).to(dev))
    A, B = (_make((R, K), 4, spread=0.0) * 0.06).to(dev), (_make((N, R), 5, spread=0.0) * 0.1).to(dev)
    bias = _make((1, N), 6, torch.float32, 0.0)[0].to(dtype).to(dev)
    for f in (lambda x, b: fp8_linear(x, w, ws, b), lambda x, b: fp8_lora_linear(x, w, ws, A, B, A, B, 1.0, ((0, N, 0, R),), b)):
        x0, xb, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True), bias.clone().requires_grad_(True)
        y0, yb = f(x0, None), f(xb, b)
        assert yb.dtype == torch.bfloat16
        (d0,) = torch.autograd.grad(y0, [x0], dy)
        db, d1 = torch.autograd.grad(yb, [b, xb], dy)
        assert db.dtype == dtype       # the adapter's t is summed in any order and may round to its neighbour (2^-7)
        assert ((d0.double() - d1.double()).abs().max() <= 2.0 ** -6 * d0.double().abs().max()).item()
        want = dy.double().sum(0)
        half = torch.finfo(dtype).eps / 2
        assert ((db.double() - want).abs() <= half * want.abs() + T * EPS32 * dy.double().abs().sum(0) * (1 + half)).all()
        with torch.no_grad():
            assert torch.equal(f(x, bias), yb)
    assert torch.equal(fp8_linear(x, w, ws, bias), (fp8_linear(x, w, ws).float() + bias.float()).bfloat16())
    for wrong in (bias[:1], bias[None], bias.repeat(2)):
        with pytest.raises(ValueError):
            fp8_linear(x, w, ws, wrong)
        with pytest.raises(ValueError):
            fp8_lora_linear(x, w, ws, A, B, A, B, 1.0, ((0, N, 0, R),), wrong)


@pytest.mark.gpu
@pytest.mark.parametrize("coded", [True, False])
def test_store_taken_back_on_another_stream(coded):
    """What one stream stores, another takes back: it waits for the codes, and their memory is not given out again while it reads them."""
    from axolotl_b200.train.activation_memory import make_store

    x = _make((512, 1024), 1, spread=0.3).cuda()
    x = x if coded else x.double()
    want = dequantize_fp8_rows(*quantize_fp8_rows(x)) if coded else x.clone()
    store, side = make_store("fp8", x.device), torch.cuda.Stream()
    torch.cuda.synchronize()
    late = torch.zeros_like(x)
    torch.cuda._sleep(20_000_000)                          # some 10 ms
    late.copy_(x)
    h = store.put(late)
    kept = h.gpu.data_ptr()
    del late
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        got = store.get(h)
        got = got if coded else got.clone()
    fresh = [torch.full((want.numel() * (1 if coded else 8) + 16384 * coded,), 0x55, dtype=torch.uint8, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and kept and fresh


@pytest.mark.parametrize("dev", DEVICES)
def test_frozen_parameter_moves_between_the_passes(dev):
    """Autograd saves the frozen parameter itself: data that leave after the forward pass are let go, and come back for the backward pass."""
    from axolotl_b200.models.layers import FusedLinear

    m = FusedLinear(256, [128], ["a"], dtype=torch.bfloat16, device=dev)
    with torch.no_grad():
        m.weight.copy_(_make((128, 256), 1, spread=0.0))
    m.quantize_fp8_()
    x, dy = _make((30, 256), 2, spread=0.0).to(dev), _make((30, 128), 3, spread=0.0).to(dev)
    x0 = x.clone().requires_grad_(True)
    (want,) = torch.autograd.grad(m(x0), [x0], dy)
    x1 = x.clone().requires_grad_(True)
    y = m(x1)
    kept = m.weight.data.clone()
    m.weight.data = torch.empty(0, dtype=torch.uint8, device=dev)
    m.weight.data = kept
    assert any(t is m.weight for t in y.grad_fn.saved_tensors)
    (got,) = torch.autograd.grad(y, [x1], dy)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dev", DEVICES)
def test_second_derivatives_are_refused(dev):
    w, ws = quantize_fp8_weight(_make((64, 128), 3, torch.float32, 0.0).to(dev))
    x = _make((4, 128), 1, spread=0.0).to(dev).requires_grad_(True)
    (dx,) = torch.autograd.grad(fp8_linear(x, w, ws).float().pow(2).sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError):
        dx.float().sum().backward()


@pytest.mark.parametrize("dev", DEVICES)
def test_layer_offloading_of_8_bit_layers(dev):
    """Frozen layers that live in host memory give the loss and the gradients of resident ones. On the device the sums of t are atomic: t may
    round to its neighbour (2^-8). A value that is off by d of itself takes another code with a probability of d / step, and is off by a
    step (at most 2^-3) then: sqrt(2^-8 2^-3) = 2.2 % rms at each quantisation of a gradient. It passes four of them a layer, 12 in all:
    sqrt(12) 2.2 % = 8 %."""
    from axolotl_b200.models.config import preset
    from axolotl_b200.models.lora import LoraSpec, inject_lora, quantize_base_fp8_
    from axolotl_b200.models.transformer import CausalLM
    from axolotl_b200.train.activation_memory import LayerOffloader

    cfg = preset("tiny-llama", num_hidden_layers=3, vocab_size=512)
    grads, losses = [], []
    for offload in (False, True):
        m = CausalLM(cfg, dtype=torch.bfloat16 if dev == "cuda" else torch.float32, device=dev).init_weights(0)
        quantize_base_fp8_(m)
        torch.manual_seed(1)
        inject_lora(m, LoraSpec(r=8, lora_alpha=16, target_modules=["q_proj", "o_proj", "gate_proj", "up_proj", "down_proj"]))
        with torch.no_grad():
            for _, f in m.fused_linears():
                if f.lora_B is not None:
                    for _, B in f.peft_tensors().values():
                        B.normal_(0, 0.05)
        m.refresh_lora_shadows()
        m.train()
        if offload:
            LayerOffloader(m, dev)
        ids = torch.randint(0, 512, (1, 96), generator=torch.Generator().manual_seed(2)).to(dev)
        loss = m(ids, labels=ids).loss
        loss.backward()
        losses.append(loss.item())
        grads.append({n: p.grad.float() for n, p in m.named_parameters() if p.grad is not None})
    assert losses[0] == losses[1] and grads[0].keys() == grads[1].keys() and grads[0]
    for n, g in grads[0].items():
        assert ((g - grads[1][n]).norm() <= 0.08 * g.norm()).item(), n


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows behind 2^31 values are those of a short call: codes, values, products, both gradients and the checkpoint."""
    from axolotl_b200.train.activation_memory import make_store

    T, K, N, R, n = (1 << 18) + 5, 8200, 72, 8, 9
    assert (T - n) * K > 1 << 31
    x = torch.empty(T, K, dtype=torch.bfloat16, device="cuda").normal_()
    tail = x[T - n:].clone()
    codes, scale = quantize_fp8_rows(x)
    c, s = quantize_fp8_rows(tail)
    assert torch.equal(codes[T - n:].view(torch.uint8), c.view(torch.uint8)) and torch.equal(scale[:, T - n:], s)
    want = dequantize_fp8_rows(c, s)
    assert torch.equal(dequantize_fp8_rows(codes, scale)[T - n:], want)
    store = make_store("fp8", "cuda")
    assert torch.equal(store.get(store.put(x))[T - n:], want)
    t = torch.zeros(T, R, dtype=torch.bfloat16, device="cuda")
    t[T - n:] = _make((n, R), 1, spread=0.0).cuda()
    t64 = t[T - n:].cpu().double()
    exact, size = t64.t() @ want.cpu().double(), t64.abs().t() @ want.cpu().double().abs()
    assert ((fp8_adapter_grad(t, codes, scale).cpu().double() - exact).abs() <= (n + 8) * EPS32 * size).all()
    del codes, scale
    w, ws = quantize_fp8_weight(_make((N, K), 3, torch.float32, 0.0).cuda())
    dy = torch.zeros(T, N, dtype=torch.bfloat16, device="cuda")
    dy[T - n:] = _make((n, N), 4, spread=0.0).cuda()
    xl = x.requires_grad_(True)
    y = fp8_linear(xl, w, ws)
    (dx,) = torch.autograd.grad(y, [xl], dy)
    w8 = _weight8(w, ws)
    _assert_product(y[T - n:], want.cpu().double(), w8.t())
    _assert_product(dx[T - n:], _rows8(dy[T - n:].cpu()), w8)
    assert not dx[:T - n].any().item()


@pytest.mark.gpu
@pytest.mark.parametrize("T,K,R", [(1, 264, 8), (65, 8, 16), (129, 200, 24), (300, 904, 40), (960, 4096, 16), (2053, 2056, 32), (4100, 4104, 16),
                                   (4100, 4104, 64), (9000, 1288, 16)])
def test_codes_and_low_rank_product_in_one_pass(T, K, R):
    """What the forward pass keeps: the codes are those of the quantiser, bit for bit and every time, and s x A^T is that of the values
    before they were coded; rows with NaN and infinities stay to themselves."""
    x = _make((T, K), T + K, spread=0.5)
    if T > 64:
        x[7, 3], x[64, 5], x[T - 1, K - 1] = float("nan"), float("inf"), float("-inf")
    A, N = _make((R, K), 4, spread=0.0) * K ** -0.5, 40
    B = torch.zeros(N, R, dtype=torch.bfloat16, device="cuda")
    w, ws = quantize_fp8_weight(_make((N, K), 3, torch.float32, 0.0).cuda())
    xd, Al, Ad = x.cuda(), A.cuda().requires_grad_(True), A.cuda()
    codes, scale = quantize_fp8_rows(xd)
    from axolotl_b200.ops.fp8 import _unpacked

    for i in range(8):
        y = fp8_lora_linear(xd, w, ws, Al, B, Ad, B, 0.5, ((0, N, 0, R),))
        q, xa = y.grad_fn.saved_tensors[0], y.grad_fn.saved_tensors[7]
        c, s = _unpacked(q, T, K)
        assert torch.equal(c.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(s, scale), i
        first = xa if i == 0 else first
        assert torch.equal(xa.view(torch.int16), first.view(torch.int16)), i
    want, size = 0.5 * xd.double() @ Ad.double().t(), 0.5 * xd.double().abs() @ Ad.double().abs().t()
    ok = torch.isfinite(xd).all(1)
    diff = (xa.double() - want).abs()
    assert (diff <= BF16 * want.abs() + (K + 8) * EPS32 * size * (1 + BF16) + 1e-38)[ok].all()
    assert not torch.isfinite(xa[~ok]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", [(5, 4616, 1544), (20, 6280, 1288), (33, 9224, 776), (64, 4616, 4104), (64, 6280, 3336), (50, 9224, 2056)])
def test_few_tokens_over_clusters_of_three_five_and_six(T, N, K):
    x = _make((T, K), T + K, spread=0.5)
    w, ws = quantize_fp8_weight(_make((N, K), 3, torch.float32, 0.0).cuda())
    _assert_product(fp8_linear(x.cuda(), w, ws), _rows8(x), _weight8(w, ws).t())


@pytest.mark.gpu
@pytest.mark.parametrize("T,K", [(800, 4616), (1300, 5512), (700, 6280), (400, 9224), (390, 11656)])
def test_adapter_gradient_over_clusters_of_three_five_and_six(T, K):
    x, t = _make((T, K), T + K, spread=0.5), _make((T, 16), 2, spread=0.5)
    codes, scale = quantize_fp8_rows(x.cuda())
    want, size = t.double().t() @ _rows8(x), t.double().abs().t() @ _rows8(x).abs()
    got = fp8_adapter_grad(t.cuda(), codes, scale)
    assert ((got.cpu().double() - want).abs() <= (T + 8) * EPS32 * size * (1 + 2.0 ** -20)).all()
    assert torch.equal(got, fp8_adapter_grad(t.cuda(), codes, scale))


@pytest.mark.parametrize("dev", DEVICES)
def test_no_rows_reach_all_that_learns(dev):
    """Frozen inputs without rows: the adapter and the bias receive zeros."""
    w, ws = quantize_fp8_weight(torch.randn(64, 128).to(dev))
    A, B = (torch.randn(s).to(dev).requires_grad_(True) for s in ((8, 128), (64, 8)))
    bias = torch.randn(64, device=dev, requires_grad=True)
    x = torch.empty(0, 128, dtype=torch.bfloat16, device=dev)
    y = fp8_lora_linear(x, w, ws, A, B, A.detach().bfloat16(), B.detach().bfloat16(), 1.0, ((0, 64, 0, 8),), bias)
    assert y.shape == (0, 64) and y.dtype == torch.bfloat16
    for g in (*torch.autograd.grad(y.sum(), [A, B, bias]), *torch.autograd.grad(fp8_linear(x, w, ws, bias).sum(), [bias])):
        assert not g.any()


@pytest.mark.gpu
def test_adapter_layer_captured_forward_and_backward():
    """A graph of the adapter's layer both ways, replayed on other inputs, beside the eager call."""
    T, K, N, R = 1000, 1160, 328, 16
    w, ws = quantize_fp8_weight(_make((N, K), 3, torch.float32, 0.0).cuda())
    A, B = _make((R, K), 4, spread=0.0).cuda() * 0.06, _make((N, R), 5, spread=0.0).cuda() * 0.1
    x, dy = _make((T, K), 1, spread=0.3).cuda(), _make((T, N), 2, spread=0.3).cuda()

    def both():
        xl, a, b = x.detach().requires_grad_(True), A.detach().requires_grad_(True), B.detach().requires_grad_(True)
        y = fp8_lora_linear(xl, w, ws, a, b, A, B, 0.5, ((0, N, 0, R),))
        return [y, *torch.autograd.grad(y, [xl, a, b], dy)]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        both()
    stream.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        outs = both()
    for seed in (11, 12):
        x.copy_(_make((T, K), seed, spread=0.3))
        dy.copy_(_make((T, N), seed + 1, spread=0.3))
        g.replay()
        torch.cuda.synchronize()
        got = [o.detach().clone() for o in outs]
        want = both()
        assert torch.equal(got[0], want[0])
        for a, b in zip(got[1:], want[1:]):                # t and dB are summed in any order and may round to their neighbours (2^-7)
            assert ((a.double() - b.detach().double()).abs().max() <= 2.0 ** -6 * b.detach().double().abs().max()).item()


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls of every form in flight on two streams give what they give alone."""
    N, K, R = 1160, 2056, 16
    w, ws = quantize_fp8_weight(_make((N, K), 3, torch.float32, 0.0).cuda())
    A, B = _make((R, K), 4, spread=0.0).cuda() * 0.06, _make((N, R), 5, spread=0.0).cuda() * 0.1
    xs = [_make((T, K), T, spread=0.3).cuda() for T in (1, 40, 64, 200, 1200)]
    t = _make((1200, R), 6, spread=0.0).cuda()
    codes, scale = quantize_fp8_rows(xs[-1])
    Al = A.clone().requires_grad_(True)
    calls = [lambda x=x: fp8_linear(x, w, ws) for x in xs]
    calls += [lambda x=x: fp8_lora_linear(x, w, ws, Al, B, A, B, 1.0, ((0, N, 0, R),)) for x in xs]
    calls += [lambda: fp8_adapter_grad(t, codes, scale), lambda: quantize_fp8_rows(xs[-1])[0].view(torch.uint8)]
    alone = [f() for f in calls]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(4):
        for s, o, order in zip(streams, outs, (calls, calls[::-1])):
            with torch.cuda.stream(s):
                o.append([f() for f in order])
    torch.cuda.synchronize()
    for o, order in zip(outs, (alone, alone[::-1])):
        for run in o:
            assert all(torch.equal(a, b) for a, b in zip(run, order))
