"""8-bit block-scaled matrices on the GPU against numpy in 64 bits: codes and scales bit
for bit, products within the bound of an f32 sum."""
import numpy as np
import pytest

import rgpu_b200
from rgpu_b200 import gpu as G
from tests import ref_tokens as R

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24  # half a step of f32


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
    """A matrix in caller memory; every byte that the format leaves open is 0x7F, a NaN, or for scales 255."""

    def __init__(self, gpu, rows, k):
        cb, sb = rgpu_b200.Fp8Tensor.nbytes(rows, k)
        self.codes = torch.full((max(cb, 16) + 64,), 0x7F, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((max(sb, 16) + 64,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        self.rows, self.k, self.cb, self.sb = rows, k, cb, sb
        self.q = gpu.fp8_wrap(self.codes.data_ptr(), self.scales.data_ptr(), rows, k)

    def set(self, codes, scales):
        stride = -(-self.k // 16) * 16
        whole = np.full((self.rows, stride), 0x7F, np.uint8)
        whole[:, :self.k] = codes[:, :self.k]
        self.codes[:self.cb] = torch.from_numpy(whole.ravel()).cuda()
        groups = -(-scales.shape[1] // 4) * 4
        every = np.full((self.rows, groups), 255, np.uint8)
        every[:, :scales.shape[1]] = scales
        self.scales[:self.sb] = torch.from_numpy(R.tile_scales(every, fill=255).ravel()).cuda()
        torch.cuda.synchronize()
        return self

    def get(self, gpu):
        gpu.sync()
        assert (self.codes[self.cb:] == 0x7F).all() and (self.scales[self.sb:] == 255).all(), "bytes behind the matrix"
        codes = self.codes[:self.cb].cpu().numpy().reshape(self.rows, -1)[:, :self.k]
        return codes, R.untile_scales(self.scales[:self.sb].cpu().numpy(), self.rows, -(-self.k // 128))


def _inputs(rows, k, seed):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, k)) * np.exp(rng.standard_normal((rows, 1)) * 3)).astype(np.float32)
    if k >= 128:
        # values half way between two codes, in a block whose scale is 1
        x[0, :14] = [448.0, 17.0, 19.0, 1.0625, -1.1875, 2.0 ** -10, 3 * 2.0 ** -10, 432.0, -0.0, 0.0, 2.0 ** -11, 21.0, 23.0, 27.0]
        x[0, 14:128] = 0.1
    if rows > 2:
        x[1] = 0.0
        x[2] = np.float32(1e-42)         # subnormal
    if rows > 6:
        x[3] = np.float32(3e38)          # the largest exponent
        x[4, 0] = np.nan
        x[4, -1] = np.inf
        x[5, k // 2] = 449.0             # just over 448: the next scale
        x[6] *= np.float32(1e-36)
    return x


SHAPES = [(1, 1), (1, 16), (1, 17), (3, 31), (5, 128), (7, 129), (31, 255), (33, 256), (65, 257), (128, 384), (129, 500),
          (130, 1000), (300, 513), (40, 1535)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("axis", [0, 1])
@pytest.mark.parametrize("rows,k", SHAPES)
def test_quantize_is_exact(gpu, rows, k, axis, dtype):
    x = _inputs(rows, k, rows * 1000 + k)
    x = _bf16(x) if dtype == "bf16" else x
    codes, scales = R.quantize(x)
    for pad, offset in ((0, 0), (3, 0), (8, 1), (-(k if axis else rows) % 16, 8)):  # packed, odd stride, odd start, 16 bytes
        src, _keep, _ = _upload(gpu, x if axis == 1 else x.T, dtype, (k if axis == 1 else rows) + pad, offset)
        held = Held(gpu, rows, k)
        gpu.fp8_quantize(src, held.q, axis=axis)
        got, got_scales = held.get(gpu)
        assert np.array_equal(got_scales, scales)
        nan = np.repeat(scales == 255, 128, 1)[:, :k]
        assert np.array_equal(got[~nan], codes[~nan])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,k", SHAPES)
def test_dequantize_is_exact(gpu, rows, k, dtype):
    rng = np.random.default_rng(rows + 7 * k)
    codes = rng.integers(0, 256, (rows, k)).astype(np.uint8)
    scales = rng.integers(1, 246, (rows, -(-k // 128))).astype(np.uint8)
    scales.ravel()[::7] = 0 if dtype == "f32" else 1
    if scales.size > 3:
        scales.ravel()[3] = 255
    want = R.values(codes, scales, k)
    want = want.astype(np.float32)
    if dtype == "bf16":  # four significant bits fit, but for the smallest exponents
        want = np.where(np.isnan(want), np.nan, _bf16(np.nan_to_num(want, posinf=0, neginf=0))).astype(np.float32)
    held = Held(gpu, rows, k).set(codes, scales)
    for pad, offset in ((0, 0), (5, 0), (8, 1), (-k % 16, 8)):
        dst, buf, view = _upload(gpu, np.zeros((rows, k)), dtype, k + pad, offset)
        before = buf.clone()
        gpu.fp8_dequantize(held.q, dst)
        gpu.sync()
        assert np.array_equal(view.float().cpu().numpy(), want, equal_nan=True)
        view.copy_(before[offset:offset + rows * (k + pad)].view(rows, k + pad)[:, :k])
        assert torch.equal(buf.isnan(), before.isnan()), "elements beside dst were written"


def _operand(gpu, rows, k, seed, wide=False):
    rng = np.random.default_rng(seed)
    codes = rng.integers(0, 255, (rows, k)).astype(np.uint8)
    codes[codes == 127] = 126
    lo, hi = (100, 150) if wide else (120, 125)
    scales = rng.integers(lo, hi, (rows, -(-k // 128))).astype(np.uint8)
    return Held(gpu, rows, k).set(codes, scales), R.values(codes, scales, k)


def _product_check(got, a, b, bias, relu, dtype):
    """An f32 sum of k exact products (4 + 4 significant bits) in any order, each addition off by at most 2U of the sum of
    magnitudes (the tensor cores cut, not round), then the bias, then for bf16 half a step of 8 bits, 2^-8."""
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


PRODUCTS = [(1, 1, 1), (1, 1, 16), (1, 17, 33), (2, 130, 64), (3, 128, 129), (16, 200, 100), (31, 129, 224), (32, 1000, 256),
            (33, 64, 288), (63, 500, 96), (64, 256, 512), (65, 257, 1000), (100, 1, 513), (127, 127, 127), (128, 128, 128),
            (129, 384, 320), (255, 130, 2048), (256, 256, 256), (257, 513, 640), (300, 1000, 1024), (513, 777, 1056),
            (1024, 512, 96), (1, 4096, 4096), (7, 1000, 8192), (48, 2900, 1500), (640, 1280, 2560),
            (2000, 2001, 1100), (1601, 2304, 800), (2305, 1537, 64), (4100, 3001, 33),
            # rings that turn over, unequal shares of k
            (2600, 2050, 1050), (1600, 2304, 1697), (7, 1000, 2176), (3, 520, 4100), (33, 300, 4608), (1, 128, 32801),
            (2047, 1000, 1250), (500, 4096, 1041), (129, 9401, 2049),
            # pairs that split k, evenly and not; 128 tokens with k split in two and four
            (300, 4300, 6209), (2047, 1000, 6400), (513, 2300, 8193), (200, 2100, 4200), (1024, 1000, 4353)]


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
        for _ in range(2):  # the second call meets what the first one left in shared memory and TMEM
            gpu.fp8_matmul(a.q, b.q, c, bias=None if epi == "none" else tb, relu=epi == "bias_relu")
        gpu.sync()
        _product_check(view.double().cpu().numpy(), av, bv, None if epi == "none" else bias.astype(np.float64),
                       epi == "bias_relu", dtype)
        # nothing outside C is written
        mask = torch.ones_like(buf, dtype=torch.bool)
        mask[offset:offset + m * (n + pad)].view(m, n + pad)[:, :n] = False
        assert torch.equal(buf[mask].isnan(), before[mask].isnan())


def test_product_with_scales_far_apart(gpu):
    a, av = _operand(gpu, 70, 1100, 1, wide=True)
    b, bv = _operand(gpu, 200, 1100, 2, wide=True)
    c = gpu.zeros((70, 200))
    gpu.fp8_matmul(a.q, b.q, c)
    _product_check(gpu.download(c).astype(np.float64), av, bv, None, False, "f32")


def test_each_scale_reaches_its_block(gpu):
    # one row of ones against rows that differ in one block's scale only: a scale taken from another
    # row or block shows as a wrong whole number
    n, blocks = 300, 21
    k = 128 * blocks
    one = int(np.flatnonzero(R.VALUES == 1.0)[0])
    codes = np.full((n, k), one, np.uint8)
    scales = np.full((n, blocks), 127, np.uint8)
    for r in range(n):
        scales[r, r % blocks] = 127 + 1 + r % 5
    b = Held(gpu, n, k).set(codes, scales)
    for m in (1, 40, 100, 130, 300, 2500):
        ca, sa = np.full((m, k), one, np.uint8), np.full((m, blocks), 127, np.uint8)
        for r in range(m):
            sa[r, (r * 5) % blocks] = 127 + 3 + r % 4
        a = Held(gpu, m, k).set(ca, sa)
        c = gpu.zeros((m, n))
        gpu.fp8_matmul(a.q, b.q, c)
        assert np.array_equal(gpu.download(c), R.values(ca, sa, k) @ R.values(codes, scales, k).T)


def test_nan_stays_in_its_row(gpu):
    a, av = _operand(gpu, 40, 300, 3)
    b, bv = _operand(gpu, 150, 300, 4)
    one = int(np.flatnonzero(R.VALUES == 1.0)[0])
    codes, scales = np.full((40, 300), one, np.uint8), np.full((40, 3), 127, np.uint8)
    scales[5, 1] = 255
    codes[9, 299] = 0x7F
    a.set(codes, scales)
    c = gpu.zeros((40, 150))
    gpu.fp8_matmul(a.q, b.q, c, relu=True)
    got = gpu.download(c)
    assert np.isnan(got[[5, 9]]).all()
    assert np.isfinite(np.delete(got, [5, 9], 0)).all()


def test_empty_extents(gpu):
    bias = gpu.upload(np.array([[1.0, -2.0, 3.0]], np.float32))
    c = gpu.upload(np.full((2, 3), 9.0, np.float32))
    gpu.fp8_matmul(gpu.fp8_zeros(2, 0), gpu.fp8_zeros(3, 0), c, bias=bias, relu=True)  # k = 0: the bias alone
    assert np.array_equal(gpu.download(c), [[1, 0, 3]] * 2)
    gpu.fp8_matmul(gpu.fp8_zeros(0, 64), gpu.fp8_zeros(3, 64), gpu.zeros((0, 3)))
    gpu.fp8_matmul(gpu.fp8_zeros(2, 64), gpu.fp8_zeros(0, 64), gpu.zeros((2, 0)))
    gpu.fp8_quantize(gpu.zeros((0, 64)), gpu.fp8_zeros(0, 64))
    gpu.fp8_dequantize(gpu.fp8_zeros(5, 0), gpu.zeros((5, 0)))
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
            (gpu.fp8_quantize(tx), gpu.fp8_quantize(tw, axis=0), (m, u), (val(x), val(w.T))),
            (gpu.fp8_quantize(tdy), gpu.fp8_quantize(tw), (m, d), (val(dy), val(w))),
            (gpu.fp8_quantize(tx, axis=0), gpu.fp8_quantize(tdy, axis=0), (d, u), (val(x.T), val(dy.T)))):
        c = gpu.zeros(shape)
        gpu.fp8_matmul(a, b, c)
        _product_check(gpu.download(c).astype(np.float64), *want, None, False, "f32")


def test_same_bits_every_time_and_on_another_stream(gpu):
    a, _ = _operand(gpu, 33, 4096, 5)
    b, _ = _operand(gpu, 500, 4096, 6)
    out = []
    side = torch.cuda.Stream()
    for stream in (None, side.cuda_stream, None):
        gpu.set_stream(stream)
        c = gpu.zeros((33, 500))
        gpu.fp8_matmul(a.q, b.q, c)
        out.append(gpu.download(c))
        c.free()
    gpu.set_stream(None)
    assert np.array_equal(out[0], out[1]) and np.array_equal(out[0], out[2])


@pytest.mark.parametrize("m,n,k", [(20, 300, 700), (300, 4300, 6209)])
def test_captured(gpu, m, n, k):
    x = torch.zeros(m, k, device="cuda")
    w = torch.randn(k, n, device="cuda")
    c = torch.zeros(m, n, device="cuda")
    tx, tw, tc = (gpu.wrap(t.data_ptr(), t.shape) for t in (x, w, c))
    qx, qw = gpu.fp8_zeros(m, k), gpu.fp8_zeros(n, k)
    gpu.sync()
    torch.cuda.synchronize()
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    gpu.set_stream(stream.cuda_stream)
    try:
        with torch.cuda.graph(graph, stream=stream):
            gpu.fp8_quantize(tx, qx)
            gpu.fp8_quantize(tw, qw, axis=0)
            gpu.fp8_matmul(qx, qw, tc)
    finally:
        gpu.set_stream(None)
    for seed in (1, 2):
        torch.manual_seed(seed)
        x.copy_(torch.randn(m, k, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = c.clone()
        gpu.fp8_matmul(gpu.fp8_quantize(tx), gpu.fp8_quantize(tw, axis=0), tc)
        gpu.sync()
        assert torch.equal(got, c) and got.any()


def test_refusals(gpu):
    q = gpu.fp8_zeros(4, 64)
    f = gpu.zeros((4, 64))

    def refused(call, word):
        with pytest.raises(rgpu_b200.RtError) as e:
            call()
        assert e.value.code == G.RT_ERR_INVALID and word in str(e.value), str(e.value)

    refused(lambda: gpu.fp8_quantize(f, gpu.fp8_zeros(64, 4)), "dst 64x4")
    refused(lambda: gpu.fp8_quantize(f, gpu.fp8_zeros(4, 64), axis=0), "64x4 along the blocks")
    refused(lambda: gpu.fp8_quantize(f, q, axis=2), "axis")
    refused(lambda: gpu.fp8_quantize(gpu.zeros((4, 64), "u32"), q), "f32 or bf16")
    refused(lambda: gpu.fp8_dequantize(q, gpu.zeros((4, 65))), "dst 4x65")
    refused(lambda: gpu.fp8_dequantize(q, gpu.zeros((4, 64), "u32")), "f32 or bf16")
    refused(lambda: gpu.fp8_matmul(q, gpu.fp8_zeros(4, 32), gpu.zeros((4, 4))), "second extents differ")
    refused(lambda: gpu.fp8_matmul(q, gpu.fp8_zeros(5, 64), gpu.zeros((4, 4))), "not 4x5")
    refused(lambda: gpu.fp8_matmul(q, q, gpu.zeros((4, 4), "u32")), "f32 or bf16")
    refused(lambda: gpu.fp8_matmul(q, q, gpu.zeros((4, 4)), bias=gpu.zeros((1, 5))), "bias")
    refused(lambda: gpu.fp8_matmul(q, q, gpu.zeros((4, 4)), bias=gpu.zeros((1, 4), "bf16")), "bias must be f32")
    refused(lambda: gpu.fp8_zeros(-1, 4), "negative")
    refused(lambda: gpu.fp8_zeros(1 << 31, 4), "2^31")
    refused(lambda: gpu.fp8_wrap(q.codes_ptr + 8, q.scales_ptr, 4, 64), "16-byte aligned")
    refused(lambda: gpu.fp8_wrap(0, q.scales_ptr, 4, 64), "NULL")
    other = rgpu_b200.Gpu(0)
    refused(lambda: gpu.fp8_quantize(f, other.fp8_zeros(4, 64)), "another context")
    refused(lambda: gpu.fp8_dequantize(q, other.zeros((4, 64))), "another context")
    refused(lambda: gpu.fp8_matmul(q, q, gpu.zeros((4, 4)), bias=other.zeros((1, 4))), "another context")
