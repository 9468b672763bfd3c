"""Microscaled 4-bit matrices on the GPU against numpy in 64 bits: codes and
scales bit for bit, products within the bound of an f32 sum."""
import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import gpu as G
from tests import ref_mx4 as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24  # unit roundoff of f32


@pytest.fixture(scope="module")
def gpu():
    g = rgpu_b200.Gpu(0)
    yield g
    g.close()


def _bf16(x):
    return rgpu_b200.bf16_to_f32(rgpu_b200.f32_to_bf16(np.ascontiguousarray(x, np.float32))).reshape(x.shape)


def _upload(gpu, x, dtype, ld=None, offset=0):
    """x on the device with row stride ld and its first element `offset` elements into an allocation filled with NaN."""
    ld = ld or x.shape[1]
    t = torch.bfloat16 if dtype == "bf16" else torch.float32
    buf = torch.full((offset + x.shape[0] * ld + 8,), float("nan"), dtype=t, device="cuda")
    view = buf[offset:offset + x.shape[0] * ld].view(x.shape[0], ld)[:, :x.shape[1]]
    view.copy_(torch.from_numpy(np.ascontiguousarray(x, np.float32)))
    torch.cuda.synchronize()
    return gpu.wrap(buf.data_ptr() + offset * buf.element_size(), x.shape, dtype, ld), buf, view


class Held:
    """A matrix in caller memory, every byte that the format does not fix set to `junk`."""

    def __init__(self, gpu, rows, k, junk=0xA5):
        cb, sb = rgpu_b200.Mx4Tensor.nbytes(rows, k)
        self.codes = torch.full((max(cb, 16),), junk, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((max(sb, 16),), junk, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        self.rows, self.k, self.cb, self.sb = rows, k, cb, sb
        self.q = gpu.mx4_wrap(self.codes.data_ptr(), self.scales.data_ptr(), rows, k)

    def set(self, codes, scales):
        self.codes[:self.cb] = torch.from_numpy(R.pack(codes).ravel()).cuda()
        self.scales[:self.sb] = torch.from_numpy(R.tile_scales(scales, fill=255).ravel()).cuda()
        torch.cuda.synchronize()
        return self

    def get(self, gpu):
        gpu.sync()
        two = self.codes[:self.cb].cpu().numpy().reshape(self.rows, -1)
        codes = np.stack([two & 15, two >> 4], 2).reshape(self.rows, -1)
        blocks = -(-self.k // 32)
        groups = -(-blocks // 4)
        every = R.untile_scales(self.scales[:self.sb].cpu().numpy(), self.rows, groups * 4)
        return codes, every[:, :blocks], every[:, blocks:]


def _inputs(rows, k, seed):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, k)) * np.exp(rng.standard_normal((rows, 1)) * 3)).astype(np.float32)
    flat = x.ravel()
    if flat.size >= 64:
        # every boundary between two codes, in a block whose scale is 1
        flat[:14] = [4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -0.75, -5.0, 7.99, -0.0, 0.0]
        flat[14:32] = 0.1
    if rows > 2:
        x[1] = 0.0                       # a block of zeros
        x[2] = np.float32(1e-42)         # subnormal
    if rows > 4:
        x[3] = np.float32(3e38)          # the largest exponent
        x[4, 0] = np.nan
        x[4, -1] = np.inf
    return x


SHAPES = [(1, 1), (1, 32), (1, 33), (3, 31), (5, 64), (7, 100), (31, 127), (33, 128), (65, 129), (128, 160), (129, 257),
          (130, 1000), (300, 513)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("rows,k", SHAPES)
def test_quantize_is_exact(gpu, rows, k, axis, dtype):
    x = _inputs(rows, k, rows * 1000 + k)
    x = _bf16(x) if dtype == "bf16" else x
    codes, scales = R.quantize(x)
    for pad, offset in ((0, 0), (3, 0), (8, 1)):  # packed, odd row stride, unaligned start
        src, _keep, _ = _upload(gpu, x if axis == 1 else x.T, dtype, (k if axis == 1 else rows) + pad, offset)
        held = Held(gpu, rows, k)
        gpu.mx4_quantize(src, held.q, axis=axis)
        got, got_scales, padding = held.get(gpu)
        assert np.array_equal(got_scales, scales)
        assert np.array_equal(got[:, :k], np.where(np.repeat(scales == 255, 32, 1)[:, :k], got[:, :k], codes[:, :k]))
        assert not np.any(got[:, k:] & 7), "elements past k must be zero"
        assert not np.any(padding == 255), "scales past the last block must not be NaN"


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k", SHAPES)
def test_dequantize_is_exact(gpu, rows, k, dtype):
    rng = np.random.default_rng(rows + 7 * k)
    blocks = -(-k // 32)
    codes = rng.integers(0, 16, (rows, blocks * 32)).astype(np.uint8)
    codes[:, k:] = 0
    scales = rng.integers(0, 252, (rows, blocks)).astype(np.uint8)
    scales.ravel()[::7] = 0
    if scales.size > 3:
        scales.ravel()[3] = 255
    want = R.values(codes, scales, k).astype(np.float32)
    held = Held(gpu, rows, k).set(codes, scales)
    for pad, offset in ((0, 0), (5, 0), (8, 1)):
        dst, _keep, view = _upload(gpu, np.zeros((rows, k)), dtype, k + pad, offset)
        gpu.mx4_dequantize(held.q, dst)
        gpu.sync()
        assert np.array_equal(view.float().cpu().numpy(), want, equal_nan=True)


def _operand(gpu, rows, k, seed, wide=False):
    rng = np.random.default_rng(seed)
    blocks = -(-k // 32)
    codes = rng.integers(0, 16, (rows, blocks * 32)).astype(np.uint8)
    codes[:, k:] = 0
    lo, hi = (100, 150) if wide else (124, 131)
    scales = rng.integers(lo, hi, (rows, blocks)).astype(np.uint8)
    return Held(gpu, rows, k).set(codes, scales), R.values(codes, scales, k)


def _product_check(got, a, b, bias, relu, dtype):
    """An f32 sum of k products in any order, each addition off by at most 2U of the sum of magnitudes (the tensor
    cores cut, not round), then the bias, then for bf16 the unit roundoff of 8 bits, 2^-8."""
    k = a.shape[1]
    want = a @ b.T + (bias if bias is not None else 0.0)
    size = np.abs(a) @ np.abs(b).T + (np.abs(bias) if bias is not None else 0.0)
    if relu:
        want = np.maximum(want, 0.0)
    tol = 2 * U * (k + 2) * size + 1e-37
    if dtype == "bf16":
        tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside, worst {np.abs(got - want)[bad].max():.3e}"


PRODUCTS = [(1, 1, 1), (1, 1, 32), (1, 17, 33), (2, 130, 64), (3, 128, 65), (16, 200, 100), (31, 129, 224), (32, 1000, 256),
            (33, 64, 288), (63, 500, 96), (64, 256, 512), (65, 257, 1000), (100, 1, 513), (127, 127, 127), (128, 128, 128),
            (129, 384, 320), (255, 130, 2048), (256, 256, 256), (257, 513, 640), (300, 1000, 1024), (513, 777, 1056),
            (1024, 512, 96), (1, 4096, 4096), (7, 1000, 8192), (48, 3000, 1500), (640, 1280, 2560),
            (2000, 2001, 1100), (1601, 2304, 800), (2305, 1537, 64), (4100, 3001, 33)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(gpu, m, n, k, dtype):
    a, av = _operand(gpu, m, k, m * 7 + k)
    b, bv = _operand(gpu, n, k, n * 13 + k + 1)
    bias = np.random.default_rng(n).standard_normal((1, n)).astype(np.float32) * 10
    tb = gpu.upload(bias)
    for pad, offset, epi in ((0, 0, "none"), (-n % 32, 0, "bias"), (-n % 16 + 8, 8, "bias"), (3, 1, "bias_relu")):
        c, buf, view = _upload(gpu, np.zeros((m, n)), dtype, n + pad, offset)
        before = buf.clone()
        gpu.mx4_matmul(a.q, b.q, c, bias=None if epi == "none" else tb, relu=epi == "bias_relu")
        gpu.sync()
        _product_check(view.double().cpu().numpy(), av, bv, None if epi == "none" else bias.astype(np.float64),
                       epi == "bias_relu", dtype)
        # nothing outside C is written
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask[offset:offset + m * (n + pad)].view(m, n + pad)[:, :n] = False
        assert torch.equal(buf[mask].isnan(), before[mask].isnan())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(2047, 1000, 2500), (500, 4096, 2081), (1500, 1400, 3200), (255, 8200, 2304), (129, 9401, 4097)])
def test_product_over_a_long_axis(gpu, m, n, k, dtype):
    test_product(gpu, m, n, k, dtype)


def test_product_with_scales_far_apart(gpu):
    a, av = _operand(gpu, 70, 512, 1, wide=True)
    b, bv = _operand(gpu, 200, 512, 2, wide=True)
    c = gpu.zeros((70, 200))
    gpu.mx4_matmul(a.q, b.q, c)
    _product_check(gpu.download(c).astype(np.float64), av, bv, None, False, "f32")


def test_each_scale_reaches_its_block(gpu):
    # one row of ones against rows that differ in one block's scale only: a scale taken from another
    # row, block or half of a tile shows as a wrong whole number
    n, k = 300, 32 * 21
    codes = np.full((n, k), 2, np.uint8)  # 1.0
    scales = np.full((n, k // 32), 127, np.uint8)
    for r in range(n):
        scales[r, r % 21] = 127 + 1 + r % 5
    b = Held(gpu, n, k).set(codes, scales)
    for m in (1, 40, 100, 130, 300):
        ca, sa = np.full((m, k), 2, np.uint8), np.full((m, k // 32), 127, np.uint8)
        for r in range(m):
            sa[r, (r * 5) % 21] = 127 + 3 + r % 4
        a = Held(gpu, m, k).set(ca, sa)
        c = gpu.zeros((m, n))
        gpu.mx4_matmul(a.q, b.q, c)
        assert np.array_equal(gpu.download(c), R.values(ca, sa, k) @ R.values(codes, scales, k).T)


def test_nan_scale_stays_in_its_row(gpu):
    a, av = _operand(gpu, 40, 96, 3)
    b, bv = _operand(gpu, 150, 96, 4)
    codes, scales = np.full((40, 96), 2, np.uint8), np.full((40, 3), 127, np.uint8)
    scales[5, 1] = 255
    a.set(codes, scales)
    c = gpu.zeros((40, 150))
    gpu.mx4_matmul(a.q, b.q, c, relu=True)
    got = gpu.download(c)
    assert np.isnan(got[5]).all()
    assert np.isfinite(np.delete(got, 5, 0)).all()


def test_empty_extents(gpu):
    bias = gpu.upload(np.array([[1.0, -2.0, 3.0]], np.float32))
    c = gpu.upload(np.full((2, 3), 9.0, np.float32))
    gpu.mx4_matmul(gpu.mx4_zeros(2, 0), gpu.mx4_zeros(3, 0), c, bias=bias, relu=True)  # k = 0: the bias alone
    assert np.array_equal(gpu.download(c), [[1, 0, 3]] * 2)
    gpu.mx4_matmul(gpu.mx4_zeros(0, 64), gpu.mx4_zeros(3, 64), gpu.zeros((0, 3)))
    gpu.mx4_matmul(gpu.mx4_zeros(2, 64), gpu.mx4_zeros(0, 64), gpu.zeros((2, 0)))
    gpu.mx4_quantize(gpu.zeros((0, 64)), gpu.mx4_zeros(0, 64))
    gpu.mx4_dequantize(gpu.mx4_zeros(5, 0), gpu.zeros((5, 0)))
    gpu.sync()


def test_dense_layer_products(gpu):
    # Y = X W, dX = dY W^T and dW = X^T dY of one layer, each from operands quantised along the summed axis
    rng = np.random.default_rng(0)
    m, d, u = 96, 160, 224
    x, w, dy = (rng.standard_normal(s).astype(np.float32) for s in ((m, d), (d, u), (m, u)))
    tx, tw, tdy = gpu.upload(x), gpu.upload(w), gpu.upload(dy)

    def val(t):
        return R.values(*R.quantize(t), t.shape[1])

    for a, b, shape, want in (
            (gpu.mx4_quantize(tx), gpu.mx4_quantize(tw, axis=0), (m, u), (val(x), val(w.T))),
            (gpu.mx4_quantize(tdy), gpu.mx4_quantize(tw), (m, d), (val(dy), val(w))),
            (gpu.mx4_quantize(tx, axis=0), gpu.mx4_quantize(tdy, axis=0), (d, u), (val(x.T), val(dy.T)))):
        c = gpu.zeros(shape)
        gpu.mx4_matmul(a, b, c)
        _product_check(gpu.download(c).astype(np.float64), *want, None, False, "f32")


def test_same_bits_every_time_and_on_another_stream(gpu):
    a, _ = _operand(gpu, 33, 4096, 5)
    b, _ = _operand(gpu, 500, 4096, 6)
    out = []
    side = torch.cuda.Stream()
    for stream in (None, side.cuda_stream, None):
        gpu.set_stream(stream)
        c = gpu.zeros((33, 500))
        gpu.mx4_matmul(a.q, b.q, c)
        out.append(gpu.download(c))
        c.free()
    gpu.set_stream(None)
    assert np.array_equal(out[0], out[1]) and np.array_equal(out[0], out[2])


def test_refusals(gpu):
    q = gpu.mx4_zeros(4, 64)
    f = gpu.zeros((4, 64))

    def refused(call, word):
        with pytest.raises(rgpu_b200.RtError) as e:
            call()
        assert e.value.code == G.RT_ERR_INVALID and word in str(e.value), str(e.value)

    refused(lambda: gpu.mx4_quantize(f, gpu.mx4_zeros(64, 4)), "dst 64x4")
    refused(lambda: gpu.mx4_quantize(f, gpu.mx4_zeros(4, 64), axis=0), "64x4 along the blocks")
    refused(lambda: gpu.mx4_quantize(f, q, axis=2), "axis")
    refused(lambda: gpu.mx4_quantize(gpu.zeros((4, 64), "u32"), q), "f32 or bf16")
    refused(lambda: gpu.mx4_dequantize(q, gpu.zeros((4, 65))), "dst 4x65")
    refused(lambda: gpu.mx4_dequantize(q, gpu.zeros((4, 64), "u32")), "f32 or bf16")
    refused(lambda: gpu.mx4_matmul(q, gpu.mx4_zeros(4, 32), gpu.zeros((4, 4))), "second extents differ")
    refused(lambda: gpu.mx4_matmul(q, gpu.mx4_zeros(5, 64), gpu.zeros((4, 4))), "not 4x5")
    refused(lambda: gpu.mx4_matmul(q, q, gpu.zeros((4, 4), "u32")), "f32 or bf16")
    refused(lambda: gpu.mx4_matmul(q, q, gpu.zeros((4, 4)), bias=gpu.zeros((1, 5))), "bias")
    refused(lambda: gpu.mx4_matmul(q, q, gpu.zeros((4, 4)), bias=gpu.zeros((1, 4), "bf16")), "bias must be f32")
    refused(lambda: gpu.mx4_zeros(-1, 4), "negative")
    refused(lambda: gpu.mx4_zeros(1 << 31, 4), "2^31")
    refused(lambda: gpu.mx4_wrap(q.codes_ptr + 8, q.scales_ptr, 4, 64), "16-byte aligned")
    refused(lambda: gpu.mx4_wrap(0, q.scales_ptr, 4, 64), "NULL")
    other = rgpu_b200.Gpu(0)
    refused(lambda: gpu.mx4_quantize(f, other.mx4_zeros(4, 64)), "another context")
    refused(lambda: gpu.mx4_dequantize(q, other.zeros((4, 64))), "another context")
    refused(lambda: gpu.mx4_matmul(q, q, gpu.zeros((4, 4)), bias=other.zeros((1, 4))), "another context")
    f.free()
    refused(lambda: gpu.block_forward(f, h=gpu.zeros((4, 64))), "")
