"""MXFP4 quantisation, the way back and the encoder product on it, against plain forms in 64 bits; their refusals.

Quantisation has one right answer (the scale is a power of two, so scaling is exact and only the rounding to e2m1 is left):
codes and scales are compared bit for bit.  The product of two e2m1 values and two powers of two is exact, so a sum of K of
them in fp32 is off by at most K roundings of partial sums no larger than S = sum |x w|; a matrix instruction may cut
instead of round, 2^-23 each: |error| <= K 2^-23 S, plus the bias' addition (2^-24 of the result) and the rounding to the
output's type (half a step of it)."""
import pytest
import torch

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)


def quantise_ref(x):
    """[R, K] -> (code per column [R, Kp], scale byte [R, Kp / 32]): the nearest of the eight magnitudes, the one with an even
    code in a tie."""
    x = x.detach().double().cpu()
    R, K = x.shape
    x = torch.cat([x, torch.zeros(R, -K % 128, dtype=torch.float64)], 1).view(R, -1, 32)
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad.unsqueeze(-1), 0.0, x)
    e = torch.frexp(torch.where(bad, 1.0, top)).exponent - 3
    e = torch.where(top == 0, -127, e).clamp(-127, 127)
    y = torch.ldexp(x.abs(), -e.unsqueeze(-1)).clamp(max=6.0)
    dist = (y.unsqueeze(-1) - GRID).abs() + torch.tensor([0, 1e-14] * 4, dtype=torch.float64)  # (odd codes lose ties)
    code = dist.argmin(-1) + 8 * torch.signbit(x)
    code = torch.where(bad.unsqueeze(-1), 0, code)
    return code.view(R, -1), torch.where(bad, 255, e + 127)


def values_ref(code, scale, K):
    v = torch.where(code >= 8, -1.0, 1.0).double() * GRID[code % 8]
    v = v.view(code.shape[0], -1, 32) * torch.where(scale == 255, torch.nan, torch.ldexp(torch.ones(()).double(), scale - 127)).unsqueeze(-1)
    return v.view(code.shape[0], -1)[:, :K]


def unpacked(q):
    c = q.codes.cpu()
    return torch.stack((c & 15, c >> 4), -1).view(c.shape[0], -1).long(), q.scales.cpu().long()


# ---------------------------------------------------------------------------------------------------------------- CPU
def test_reference_ties_and_ends():
    """The oracle itself, on values worked out by hand."""
    row = torch.tensor([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, -0.25, -5.0, 0.26, 4.0] + [0.0] * 20])
    code, scale = quantise_ref(row)
    assert scale.tolist()[0][0] == 127  # 4 <= 7 < 8: e = 2 - 2
    assert code[0, :12].tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 8, 14, 1, 6]


def test_refusals_without_a_gpu():
    from clt_training_amd import _lib, hip_ops as ops

    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)  # noqa: E731
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.mxfp4_quantize(torch.zeros(2, 32))
    with pytest.raises(ValueError, match="matrix"):
        ops.mxfp4_quantize(torch.zeros(32))
    with pytest.raises(TypeError, match="float32 / bfloat16"):
        ops.mxfp4_quantize(torch.zeros(2, 32, dtype=torch.float16))
    with pytest.raises(ValueError, match="100 columns"):
        ops.MXFP4Tensor(u8(4, 50), u8(4, 4), 100)
    with pytest.raises(ValueError, match="scales"):
        ops.MXFP4Tensor(u8(4, 64), u8(4, 2), 100)
    with pytest.raises(TypeError, match="uint8"):
        ops.MXFP4Tensor(torch.zeros(4, 64), u8(4, 4), 100)
    W = ops.MXFP4Tensor(u8(4, 64), u8(4, 4), 100)
    assert W.shape == (4, 100)
    with pytest.raises(TypeError, match="MXFP4Tensor"):
        ops.mxfp4_linear(torch.zeros(2, 100), torch.zeros(4, 100))
    with pytest.raises(ValueError, match="does not fit"):
        ops.mxfp4_linear(torch.zeros(2, 99), W)
    with pytest.raises(ValueError, match="bias"):
        ops.mxfp4_linear(torch.zeros(2, 100), W, torch.zeros(5))
    with pytest.raises(TypeError, match="float32 / bfloat16"):
        ops.mxfp4_linear(torch.zeros(2, 100), W, out_dtype=torch.float16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.mxfp4_linear(torch.zeros(2, 100), W)
    with pytest.raises(TypeError, match="float32 / bfloat16"):
        W.dequantize(torch.float64)
    with pytest.raises(NotImplementedError, match="activation"):
        ops.encode_topk_mxfp4(torch.zeros(2, 100), W, None, 2, activation="batchtopk")
    # the C entries check before they launch
    lib = _lib.load()
    p, q = 4096, 4097  # (never dereferenced on the host)
    assert lib.clt_mxfp4_quantize(None, 0, 32, 1, 32, p, p, None) == -1
    assert lib.clt_mxfp4_quantize(p, 7, 32, 1, 32, p, p, None) == -1
    assert lib.clt_mxfp4_quantize(p, 0, 32, 0, 32, p, p, None) == -1
    assert lib.clt_mxfp4_quantize(p, 0, 32, 1, 32, p + 8, p, None) == -1 and b"misaligned" in lib.clt_last_error()
    assert lib.clt_mxfp4_dequantize(p, p, 1, 32, q, 1, None) == -1
    assert lib.clt_mxfp4_dequantize(p, p, 1, 0, p, 1, None) == -1
    assert lib.clt_mxfp4_linear(p, p, p, p, None, 0, 1, 8, 32, 0, p, 0, 7, None) == -1  # ldo < M
    assert lib.clt_mxfp4_linear(p, p, p, p, p, 9, 1, 8, 32, 0, p, 0, 8, None) == -1
    assert lib.clt_mxfp4_linear(p, p, p, p, None, 0, 1 << 40, 8, 32, 0, p, 0, 8, None) == -2
    assert lib.clt_mxfp4_linear(p, p + 1, p, p, None, 0, 1, 8, 32, 0, p, 0, 8, None) == -1


def test_c_refusals_of_sizes_and_workspace():
    from clt_training_amd import _lib

    lib = _lib.load()
    p = 4096
    assert lib.clt_mxfp4_quantize(p, 0, 32, 2**28, 128, p, p, None) == -1  # (more than a launch's threads can count)
    assert lib.clt_mxfp4_dequantize(p, p, 2**28, 128, p, 0, None) == -1
    x = lambda N, M, K, ws, size, a=p: lib.clt_mxfp4_linear_x(a, 0, K, p, p, None, 0, N, M, K, 0, p, 0, M, ws, size, None)  # noqa: E731
    need = lib.clt_mxfp4_linear_x_workspace_bytes(70, 300)
    assert need == 70 * 192 + 70 * 12
    assert x(70, 8, 300, None, 0) == -4 and x(70, 8, 300, p, need - 1) == -4 and b"workspace" in lib.clt_last_error()
    assert x(70, 8, 300, p + 4, need) == -1 and b"misaligned" in lib.clt_last_error()
    assert x(70, 8, 300, p, need, None) == -1 and x(70, 8, 300, p, need, p + 2) == -1
    assert x(70, 2**31, 300, p, need) == -2 and x(2**31, 8, 300, p, need) == -2 and x(2, 8, 2**24, p, need) == -2
    assert lib.clt_mxfp4_linear_x_workspace_bytes(1, 768) == 0


def test_large_product_keeps_its_registers(tmp_path):
    """The waits of the 256 x 256 kernel count its stores and LDS transfers: a spilled register would be one more access
    to memory than they know of.  The compiler's resource report must show no scratch for any of the product's kernels."""
    import subprocess

    from clt_training_amd.build import CSRC, FLAGS, HIPCC

    out = subprocess.run([HIPCC, *FLAGS, "-Rpass-analysis=kernel-resource-usage", "-c", str(CSRC / "mxfp4.hip"), "-o", str(tmp_path / "o")],
                         capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[-2000:]
    seen, name = {}, None
    for line in out.stderr.splitlines():
        if "Function Name:" in line:
            name = line.split("Function Name:")[1].split()[0]
        elif "ScratchSize" in line and name:
            seen[name] = int(line.split("ScratchSize [bytes/lane]:")[1].split()[0])
    for kernel, forms in (("mxfp4_big_kernel", 4), ("mxfp4_tile_kernel", 4), ("mxfp4_split_kernel", 2)):
        found = {k: v for k, v in seen.items() if kernel in k}
        assert len(found) == forms and not any(found.values()), found


def test_fused_encoder_refuses_a_stray_quantised_weight():
    from clt_training_amd import hip_ops as ops
    from clt_training_amd.fused_encoder import fused_encoder

    W = ops.MXFP4Tensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 128)
    x, w, b = torch.zeros(2, 128), torch.zeros(4, 128), torch.zeros(4)
    with pytest.raises(ValueError, match="weight_mxfp4"):
        fused_encoder(x, w, b, 2, weight_mxfp4=W)
    with pytest.raises(ValueError, match="weight_mxfp4"):
        fused_encoder(x, torch.zeros(5, 128), b, 2, use_mxfp4=True, weight_mxfp4=W)


def test_output_that_shares_memory_is_refused_whatever_its_strides():
    """Random layouts of x, bias and an output with gaps in one buffer: refused exactly when a byte is common.  (On the CPU: a call
    that passes the check is refused for that.)"""
    import random

    from clt_training_amd import hip_ops as ops

    rng = random.Random(0)
    seen = {True: 0, False: 0}
    for _ in range(400):
        N, M, K = rng.randint(1, 5), rng.randint(1, 6), rng.randint(1, 6)
        buf = torch.zeros(150)
        place = torch.arange(150)
        view = lambda t, r, c, pitch, at: t.as_strided((r, c), (pitch, 1), at)  # noqa: E731
        ox = (N, M, rng.randint(M, 12), rng.randint(0, 60))
        xx = (N, K, rng.choice((0, K, ox[2], rng.randint(1, 12))), rng.randint(0, 60))
        bx = (1, M, M, rng.randint(0, 100))
        spot = [set(view(place, *a).flatten().tolist()) for a in (ox, xx, bx)]
        common = bool(spot[0] & (spot[1] | spot[2]))
        seen[common] += 1
        W = ops.MXFP4Tensor(torch.zeros(M, 64, dtype=torch.uint8), torch.zeros(M, 4, dtype=torch.uint8), K)
        with pytest.raises(RuntimeError, match="memory" if common else "no CPU fallback"):
            ops.mxfp4_linear(view(buf, *xx), W, view(buf, *bx)[0], out=view(buf, *ox))
    assert min(seen.values()) > 50
    # the weight's codes and scales, and what is packed
    room = torch.zeros(4096, dtype=torch.uint8)
    codes, scales = room[1024:1024 + 8 * 64].view(8, 64), room[512:512 + 32].view(8, 4)
    W, x = ops.MXFP4Tensor(codes, scales, 40), torch.zeros(3, 40)
    other = ops.MXFP4Tensor(torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 4, dtype=torch.uint8), 40)
    out = lambda at: room.view(torch.float32).as_strided((3, 8), (50, 1), at // 4)  # noqa: E731 (32 bytes every 200)
    for given in ((x, W), (ops.MXFP4Tensor(codes[:3], scales[:3], 40), other)):
        for at in (1024 - 32 - 400, 2048):
            with pytest.raises(RuntimeError, match="no CPU fallback"):
                ops.mxfp4_linear(*given, out=out(at))
        for at in (1024 - 4, 1024 - 200 + 160, 1024 - 400, 512 + 8 - 200):
            with pytest.raises(RuntimeError, match="memory"):
                ops.mxfp4_linear(*given, out=out(at))


def route(N, M, K, dtype=torch.bfloat16, ldo=None):
    from clt_training_amd import _lib

    return _lib.load().clt_mxfp4_linear_route(N, M, K, 0 if dtype == torch.float32 else 1, M if ldo is None else ldo).decode()


def test_routes_that_the_cases_below_are_meant_for():
    """Every kernel has its cases; what the large kernel's cases need to reach its whole-line stores holds for them."""
    every = {"few", "split", "64 x 64", "128 x 128", "256 x 256"}
    for K, cases in ((300, ROUTES), (1100, LONG_ROUTES[:-1]), (1900, LONG_ROUTES[-1:])):
        found = {route(N, M, K) for N, M in cases}
        assert found == {300: every - {"split"}, 1100: every, 1900: {"split"}}[K], (K, found)
    for N, M in WHOLE_LINES:
        for K in (64, 300, 512, 700):
            for dtype, size in ((torch.float32, 4), (torch.bfloat16, 2)):
                assert route(N, M, K, dtype) == "256 x 256" and M * size % 128 == 0
                assert -(-N // 256) * -(-M // 256) > 3 * 256  # (several tiles for every workgroup)
    from clt_training_amd import _lib

    for sizes in ((0, 8, 32), (1, 0, 32), (1, 8, 0), (1, 8, 32, torch.float32, 7), (2**31, 8, 32), (8, 8, 2**24), (2**20, 2**20, 32)):
        assert route(*sizes) == ""
    assert _lib.load().clt_mxfp4_linear_route(1, 8, 32, 9, 8) == b""


# ---------------------------------------------------------------------------------------------------------------- GPU
def matrix(R, K, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, K, generator=g) * torch.exp(spread * torch.randn(R, K, generator=g))
    return x.to(dtype).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,K", [(1, 1), (1, 32), (3, 31), (5, 33), (2, 127), (7, 128), (4, 129), (33, 768), (9, 1001), (130, 2048)])
def test_quantise_bit_for_bit(R, K, dtype):
    from clt_training_amd import hip_ops as ops

    x = matrix(R, K, dtype, R * 1000 + K)
    q = ops.mxfp4_quantize(x)
    code, scale = quantise_ref(x)
    got_c, got_s = unpacked(q)
    assert torch.equal(got_s, scale)
    assert torch.equal(got_c, code)
    for out in (torch.float32, torch.bfloat16):
        v = q.dequantize(out)
        assert v.shape == (R, K) and v.dtype == out
        assert torch.equal(v.double().cpu(), values_ref(code, scale, K))


@pytest.mark.gpu
def test_quantise_every_bfloat16():
    """All 65536 bit patterns: ties, the smallest and the largest numbers, infinities and NaN, each as the head of a block."""
    from clt_training_amd import hip_ops as ops

    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.zeros(65536 // 4, 128, dtype=torch.bfloat16)
    for j in range(4):  # the value, a half, a third (rounded) and the negative of it in a block of their own
        b = v[j::4]
        x[:, 32 * j], x[:, 32 * j + 1], x[:, 32 * j + 7], x[:, 32 * j + 31] = b, b * 0.5, (b.float() / 3).bfloat16(), -b * 0.75
    q = ops.mxfp4_quantize(x.cuda())
    code, scale = quantise_ref(x)
    got_c, got_s = unpacked(q)
    assert torch.equal(got_s, scale) and torch.equal(got_c, code)
    assert torch.equal(torch.nan_to_num(q.dequantize().double().cpu(), nan=7e77), torch.nan_to_num(values_ref(code, scale, 128), nan=7e77))


@pytest.mark.gpu
def test_quantise_views_and_another_stream():
    from clt_training_amd import hip_ops as ops

    big = matrix(40, 300, torch.bfloat16, 3)
    for x in (big[:, 100:228], big[3:4, 1:130], big[::2, 5:105], big.t(), big[:, ::2], big[:1].expand(6, 300)):
        a, b = ops.mxfp4_quantize(x), ops.mxfp4_quantize(x.contiguous())
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    assert ops.mxfp4_quantize(big[:0]).dequantize().shape == (0, 300)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ops.mxfp4_linear(big, ops.mxfp4_quantize(big))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, ops.mxfp4_linear(big, ops.mxfp4_quantize(big)))


def check_linear(N, M, K, xdt, odt, bias, relu, seed, spread=1.0, out=None):
    from clt_training_amd import hip_ops as ops

    x, W = matrix(N, K, xdt, seed, spread), matrix(M, K, torch.float32, seed + 1, spread)
    b = None if bias is None else matrix(1, M, bias, seed + 2)[0]
    Wq = ops.mxfp4_quantize(W)
    y = ops.mxfp4_linear(x, Wq, b, relu=relu, out_dtype=odt, out=out)
    assert y.shape == (N, M) and y.dtype == odt
    xv, wv = ops.mxfp4_quantize(x).dequantize().double(), Wq.dequantize().double()
    ref = xv @ wv.t()
    room = K * 2.0**-23 * (xv.abs() @ wv.abs().t())
    if b is not None:
        ref = ref + b.double()
        room = room + 2.0**-24 * ref.abs()
    room = room + (torch.finfo(odt).eps / 2 if odt != torch.float32 else 0) * (ref.abs() + room)
    if relu:
        ref = ref.clamp(min=0)
    bad = ((y.double() - ref).abs() > room).nonzero()
    assert len(bad) == 0, (N, M, K, len(bad), bad[:4].tolist())
    return x, Wq, b, y


SHAPES = [(1, 1, 1), (1, 70, 32), (2, 33, 129), (1, 4096, 768), (3, 1000, 768), (15, 129, 100), (16, 256, 64), (17, 255, 384), (31, 97, 33),
          (32, 64, 1000), (33, 513, 768), (64, 300, 256), (65, 777, 2048), (127, 128, 128), (128, 257, 640), (129, 1023, 768), (200, 512, 4096),
          (256, 256, 512), (257, 300, 769), (300, 2049, 96)]


@pytest.mark.gpu
@pytest.mark.parametrize("N,M,K", SHAPES)
def test_linear_shapes(N, M, K):
    check_linear(N, M, K, torch.bfloat16, torch.bfloat16, torch.float32, True, N + M)
    check_linear(N, M, K, torch.float32, torch.float32, None, False, N + K)
    check_linear(N, M, K, torch.bfloat16, torch.float32, torch.bfloat16, False, M + K, spread=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [32, 100, 200, 300, 500, 512, 600, 770, 1100])
def test_linear_many_tiles(K):
    """Problems of several hundred tiles, with rows and columns left over, and every way a row's columns can end."""
    check_linear(2100, 9000, K, torch.bfloat16, torch.bfloat16, torch.float32, True, K)
    check_linear(4096 + 17, 4096 + 40, K, torch.bfloat16, torch.float32, torch.bfloat16, False, K + 1)
    check_linear(300, 40001, K, torch.float32, torch.bfloat16, None, True, K + 2, spread=3.0)


@pytest.mark.gpu
def test_linear_special_values():
    """NaN blocks reach every output of their row and no other; ReLU keeps NaN; the scales' ends meet in the product."""
    from clt_training_amd import hip_ops as ops

    for N in (5, 40, 300):  # (a different route for few rows)
        x, W = matrix(N, 256, torch.float32, 1), matrix(70, 256, torch.float32, 2)
        x[1, 3], W[9, 200], x[3], W[4] = float("nan"), float("-inf"), 0, 0
        x[2] *= 2.0**100
        W[7] *= 2.0**-110
        xq, Wq = ops.mxfp4_quantize(x), ops.mxfp4_quantize(W)
        for relu in (False, True):
            y = ops.mxfp4_linear(xq, Wq, relu=relu)
            ref = xq.dequantize().double() @ Wq.dequantize().double().t()
            ref = torch.where(ref < 0, 0, ref) if relu else ref
            assert torch.equal(torch.isnan(y), torch.isnan(ref))
            assert torch.isnan(y[1]).all() and torch.isnan(y[:, 9]).all() and int(torch.isnan(y).sum()) == 70 + N - 1
            ok = torch.isfinite(ref)
            room = 256 * 2.0**-23 * (torch.nan_to_num(xq.dequantize().double()).abs() @ torch.nan_to_num(Wq.dequantize().double()).abs().t())
            assert ((y.double() - ref).abs() <= room)[ok].all()
            assert (y[3][:9] == 0).all() and (y[4:, 4] == 0).all()


# Every way through the product: few tokens, tiles of 32 x 32 (long rows), 64 x 64, 128 x 128 and 256 x 256.
ROUTES = [(40, 300), (100, 5100), (20, 66001), (3, 70001), (3, 90001), (50, 41003), (200, 8101), (500, 23001), (100, 100001), (520, 40001),
          (2100, 30001)]


@pytest.mark.gpu
@pytest.mark.parametrize("K", [31, 128, 300, 512, 700, 1100])
@pytest.mark.parametrize("N,M", ROUTES)
def test_linear_every_route(N, M, K):
    check_linear(N, M, K, torch.bfloat16, torch.bfloat16, torch.float32, True, N + K)
    check_linear(N, M, K, torch.float32, torch.float32, torch.bfloat16, False, M + K, spread=3.0)


@pytest.mark.gpu
@pytest.mark.parametrize("N,M,K", [(2, 300, 20000), (20, 66001, 7000), (50, 41003, 2900), (300, 1000, 12000), (260, 50000, 2600)])
def test_linear_long_rows(N, M, K):
    check_linear(N, M, K, torch.bfloat16, torch.float32, torch.float32, False, N + K)


@pytest.mark.gpu
@pytest.mark.parametrize("N,M", ROUTES)
def test_linear_special_values_every_route(N, M):
    """As test_linear_special_values, with rows whose last 128 columns are followed by a row of NaN, and biases that are not
    finite."""
    from clt_training_amd import hip_ops as ops

    x, W = matrix(N, 300, torch.float32, 1), matrix(M, 300, torch.float32, 2)
    b = matrix(1, M, torch.float32, 3)[0]
    x[1, 299], W[9, 3], W[M - 1, 200] = float("nan"), float("-inf"), float("nan")
    b[0], b[1], b[2] = float("nan"), float("inf"), float("-inf")
    xq, Wq = ops.mxfp4_quantize(x), ops.mxfp4_quantize(W)
    xv, wv = xq.dequantize().double(), Wq.dequantize().double()
    ref = xv @ wv.t() + b.double()
    room = 300 * 2.0**-23 * (torch.nan_to_num(xv).abs() @ torch.nan_to_num(wv).abs().t()) + 2.0**-24 * ref.abs()
    for relu in (False, True):
        want = torch.where(ref < 0, 0, ref) if relu else ref
        for given in (x, xq):
            y = ops.mxfp4_linear(given, Wq, b, relu=relu)
            assert torch.equal(torch.isnan(y), torch.isnan(want)) and int(torch.isnan(y).sum()) == M + 3 * (N - 1)
            sure = torch.isfinite(want)
            assert ((y.double() - want).abs() <= room)[sure].all() and torch.equal(y.double()[torch.isinf(want)], want[torch.isinf(want)])


@pytest.mark.gpu
@pytest.mark.parametrize("N,M", ROUTES)
def test_linear_any_alignment_every_route(N, M):
    """Rows of ``out`` at odd addresses and with gaps, bias and x at odd addresses: the same bits, and nothing beside them written."""
    from clt_training_amd import hip_ops as ops

    for dt in (torch.bfloat16, torch.float32):
        xs = matrix(N, 303, torch.float32, 4)
        b = matrix(1, M + 1, torch.bfloat16, 5)[0][1:]
        Wq = ops.mxfp4_quantize(matrix(M, 300, torch.float32, 6))
        want = ops.mxfp4_linear(xs[:, 1:301].contiguous(), Wq, b.clone(), relu=True, out_dtype=dt)
        big = torch.full((N + 2, M + 9), 7.0, dtype=dt, device="cuda")
        y = ops.mxfp4_linear(xs[:, 1:301], Wq, b, relu=True, out=big[1:N + 1, 3:3 + M])
        assert torch.equal(y, want)
        y.fill_(7)
        assert (big == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N,M", ROUTES)
def test_linear_two_graphs_and_two_streams(N, M):
    """Two graphs of the same sizes, captured one after the other and replayed in turn with eager work between, and two streams at
    once: no call shares anything with another."""
    from clt_training_amd import hip_ops as ops

    W = [ops.mxfp4_quantize(matrix(M, 300, torch.float32, 7 + i)) for i in range(2)]
    x = [matrix(N, 300, torch.bfloat16, 9 + i) for i in range(2)]
    eager = lambda i: ops.mxfp4_linear(x[i], W[i], relu=True)  # noqa: E731
    eager(0), eager(1)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(eager(i))
        graphs.append(g)
    for seed in range(3):
        for i in range(2):
            x[i].copy_(matrix(N, 300, torch.bfloat16, 20 + 2 * seed + i))
        want = [eager(0), eager(1)]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = eager(i)
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.gpu
def test_linear_refuses_an_output_over_an_input():
    from clt_training_amd import hip_ops as ops

    x = matrix(64, 64, torch.float32, 1)
    W = ops.mxfp4_quantize(matrix(64, 64, torch.float32, 2))
    with pytest.raises(RuntimeError, match="memory"):
        ops.mxfp4_linear(x, W, out=x)
    with pytest.raises(RuntimeError, match="memory"):
        ops.mxfp4_linear(x[:1], W, x[0], out=x[:1])
    with pytest.raises(ValueError, match="overlap"):
        ops.mxfp4_linear(x, W, out=x[:1].expand(64, 64))
    assert ops.mxfp4_linear(x[:0], W).shape == (0, 64) and ops.mxfp4_linear(x, ops.mxfp4_quantize(x[:0])).shape == (64, 0)


@pytest.mark.gpu
def test_linear_out_rows_keep_their_neighbours():
    """``out`` with gaps between the rows: only its own columns are written; rows behind the last token stay as they were."""
    for N, M in ((3, 70), (40, 129), (300, 257), (130, 512)):
        for dt in (torch.bfloat16, torch.float32):
            big = torch.full((N + 2, M + 37), 7.0, dtype=dt, device="cuda")
            check_linear(N, M, 200, torch.bfloat16, dt, torch.float32, True, 5, out=big[1:N + 1, 8:8 + M])
            inner = big.clone()
            inner[1:N + 1, 8:8 + M] = 7
            assert (inner == 7).all()
            check_linear(N, M, 200, torch.bfloat16, dt, torch.float32, True, 5, out=big[1:N + 1, 3:3 + M])  # (unaligned rows)


@pytest.mark.gpu
def test_linear_large_offsets():
    """An output of more than 2^31 elements (its last rows against the same rows on their own) and the same bits on a second run."""
    from clt_training_amd import hip_ops as ops

    N, M, K = 8200, 270000, 64
    x, W, b = matrix(N, K, torch.bfloat16, 1), matrix(M, K, torch.bfloat16, 2), matrix(1, M, torch.float32, 3)[0]
    Wq = ops.mxfp4_quantize(W)
    y = ops.mxfp4_linear(x, Wq, b, relu=True)
    assert y.numel() > 2**31
    assert torch.equal(y[-300:], ops.mxfp4_linear(x[-300:], Wq, b, relu=True))
    assert torch.equal(y[:300], ops.mxfp4_linear(x[:300], Wq, b, relu=True))
    ref = (ops.mxfp4_quantize(x[-2:]).dequantize().double() @ Wq.dequantize().double().t() + b.double()).clamp(min=0)
    torch.testing.assert_close(y[-2:].double(), ref, rtol=2.0**-8 + 2.0**-16, atol=64 * 2.0**-23 * 64 * 40)


@pytest.mark.gpu
def test_graph_replays():
    """Quantise, product and top-k captured; replays on new inputs with eager work in between."""
    from clt_training_amd import hip_ops as ops

    W, b = ops.mxfp4_quantize(matrix(2000, 256, torch.float32, 1)), matrix(1, 2000, torch.float32, 2)[0]
    x = matrix(50, 256, torch.bfloat16, 3)
    eager = lambda: ops.topk_rows(ops.mxfp4_linear(x, W, b, relu=True), 8)  # noqa: E731
    eager()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        v, i = eager()
    for seed in range(4):
        x.copy_(matrix(50, 256, torch.bfloat16, 10 + seed))
        ev, ei = eager()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(v, ev) and torch.equal(i, ei)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["topk", "groupmax", "batchtopk"])
def test_fused_encoder_values_and_gradients(activation):
    """Values and indices: those of the product; gradients: v_nk = x_n . W_i + b_i for the selected positive latents."""
    from clt_training_amd import hip_ops as ops
    from clt_training_amd.fused_encoder import fused_encoder

    N, M, K, k = 60, 512, 96, 8
    x = matrix(N, K, torch.float32, 1, 0.3).requires_grad_()
    W = torch.nn.Parameter(matrix(M, K, torch.float32, 2, 0.3))
    b = torch.nn.Parameter(matrix(1, M, torch.float32, 3)[0].detach().clone())
    v, i = fused_encoder(x, W, b, k, activation, use_mxfp4=True)
    pre = ops.mxfp4_linear(x.detach(), ops.mxfp4_quantize(W.detach()), b.detach(), relu=True)
    if activation == "topk":
        ev, ei = ops.topk_rows(pre, k)
        assert torch.equal(v, ev) and torch.equal(i, ei)
    else:
        assert torch.equal(pre.gather(1, i)[v > 0], v[v > 0])
    gv = matrix(N, v.shape[1], torch.float32, 4)
    v.backward(gv)
    on = (gv * (v > 0)).double()
    gW = torch.zeros(M, K, dtype=torch.float64, device="cuda").index_add_(0, i.flatten(), (on.unsqueeze(-1) * x.detach().double().unsqueeze(1)).flatten(0, 1))
    gb = torch.zeros(M, dtype=torch.float64, device="cuda").index_add_(0, i.flatten(), on.flatten())
    gx = (on.unsqueeze(-1) * W.detach().double()[i]).sum(1)
    for got, ref in ((W.grad, gW), (b.grad, gb), (x.grad, gx)):
        assert float((got.double() - ref).norm() / ref.norm()) < 1e-5
    # the same with the weight quantised beforehand
    v2, i2 = fused_encoder(x.detach(), W.detach(), b.detach(), k, activation, use_mxfp4=True, weight_mxfp4=ops.mxfp4_quantize(W.detach()))
    assert torch.equal(v2, v) and torch.equal(i2, i)


@pytest.mark.gpu
def test_gradients_against_differences():
    """Inputs that 4 bits hold exactly, moved to neighbours that they hold too: the selected values change by grad . delta."""
    from clt_training_amd.fused_encoder import fused_encoder

    g = torch.Generator().manual_seed(0)
    grid = torch.tensor([-3.0, -2, -1, 0, 1, 2, 3])
    N, M, K, k = 6, 64, 128, 3
    x, W = grid[torch.randint(7, (N, K), generator=g)], grid[torch.randint(7, (M, K), generator=g)]
    x[:, ::32], W[:, ::32] = 6.0, 6.0  # every block's scale is 1
    x, W, b = x.cuda().requires_grad_(), torch.nn.Parameter(W.cuda()), torch.nn.Parameter(torch.zeros(M, device="cuda"))
    v, i = fused_encoder(x, W, b, k, use_mxfp4=True)
    v.sum().backward()
    total = lambda x, W: fused_encoder(x, W, b, k, use_mxfp4=True)  # noqa: E731
    tried = 0
    for n, c in ((0, 1), (3, 40), (5, 127)):
        moved = x.detach().clone()
        moved[n, c] += 1 if moved[n, c] < 3 else -1
        v2, i2 = total(moved, W.detach())
        if all(set(p.tolist()) == set(q.tolist()) for p, q in zip(i, i2)):
            tried += 1
            assert float(v2.sum() - v.sum()) == float((x.grad * (moved - x.detach())).sum())
    for c in (1, 50, 126):
        r = int(i[2, 0])
        moved = W.detach().clone()
        moved[r, c] += 1 if moved[r, c] < 3 else -1
        v2, i2 = total(x.detach(), moved)
        if all(set(p.tolist()) == set(q.tolist()) for p, q in zip(i, i2)):
            tried += 1
            assert float(v2.sum() - v.sum()) == float((W.grad * (moved - W.detach())).sum())
    assert tried >= 2


@pytest.mark.gpu
def test_sparse_coder_serving_snapshot():
    """quantize_encoder: what encode gives follows the weight at that moment, with and without gradients, until it is taken off."""
    from clt_training_amd import SparseCoder, SparseCoderConfig

    torch.manual_seed(0)
    sc = SparseCoder(64, SparseCoderConfig(k=4, expansion_factor=8, transcode=True), "cuda", dtype=torch.float32)
    x = torch.randn(9, 64, device="cuda")
    plain = sc.encode(x)
    a = sc.quantize_encoder().encode(x)
    with torch.no_grad():
        sc.encoder.weight.mul_(-1)
        b = sc.encode(x)
        assert torch.equal(a.top_acts, b.top_acts) and torch.equal(a.top_indices, b.top_indices)
        c = sc.quantize_encoder().encode(x)
        assert not torch.equal(a.top_indices, c.top_indices)
        sc.encoder.weight.mul_(-1)
        d = sc.quantize_encoder(False).encode(x)
    assert torch.equal(d.top_indices, plain.top_indices) and torch.equal(d.top_acts, plain.top_acts)
    assert "encoder_mxfp4" not in sc.state_dict()


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", ["adam", "adamw", "adamw8"])
def test_trainer_runs_with_4_bit_encoder(optimizer):
    """The operators together, as a training run uses them: quantise -> product -> top-k -> decode -> backward -> step, twice
    with the same seeds: the same bits; the selected latents are the product's."""
    from clt_training_amd import SparseCoderConfig, TrainConfig, Trainer, hip_ops as ops

    hooks = ["a", "b"]

    def batches():
        g = torch.Generator().manual_seed(1)
        return [{h: (torch.randn(96, 64, generator=g).bfloat16().cuda(), torch.randn(96, 64, generator=g).bfloat16().cuda()) for h in hooks} for _ in range(4)]

    def train():
        cfg = TrainConfig(sae=SparseCoderConfig(dtype="bfloat16", k=8, expansion_factor=8, transcode=True, skip_connection=True, use_mxfp4=True),
                          hookpoints=list(hooks), cross_layer=2, optimizer=optimizer, lr=1e-3, lr_warmup_steps=1)
        tr = Trainer(cfg, batches())
        for b in tr.dataset:
            fvus = tr.step(b)
            assert all(bool(torch.isfinite(f)) for f in fvus.values())
        return tr

    a, b = train(), train()
    for p, q in zip((p for s in a.saes.values() for p in s.parameters()), (p for s in b.saes.values() for p in s.parameters())):
        assert torch.equal(p, q)
    sae, x = a.saes["a"], batches()[0]["a"][0]
    enc = sae.encode(x)
    pre = ops.mxfp4_linear(x, ops.mxfp4_quantize(sae.encoder.weight.detach()), sae.encoder.bias.detach(), relu=True)
    assert torch.equal(enc.top_indices, ops.topk_rows(pre, 8)[1])


@pytest.mark.gpu
def test_linear_output_beside_its_inputs():
    """An output with gaps between its rows: x or the bias in the gaps is fine, over them is refused."""
    from clt_training_amd import hip_ops as ops

    W = ops.mxfp4_quantize(matrix(64, 64, torch.float32, 2))
    buf = torch.zeros(40, 160, device="cuda")
    x = buf[:, :64]
    x.copy_(matrix(40, 64, torch.float32, 1))
    want = ops.mxfp4_linear(x.contiguous(), W)
    with pytest.raises(RuntimeError, match="memory"):
        ops.mxfp4_linear(x, W, out=buf[:, 32:96])
    with pytest.raises(RuntimeError, match="memory"):
        ops.mxfp4_linear(want, W, buf[7, 70:134], out=buf[:, 96:])
    assert torch.equal(ops.mxfp4_linear(x, W, out=buf[:, 64:128]), want)
    half = buf[:, 0:128:2].clone()
    assert torch.equal(ops.mxfp4_linear(buf[:, 0:128:2], W, out=buf[:, 64:128]), ops.mxfp4_linear(half, W))  # (a copy is read)


@pytest.mark.gpu
def test_autograd_sees_that_an_output_was_written():
    from clt_training_amd import hip_ops as ops

    W = ops.mxfp4_quantize(matrix(64, 64, torch.float32, 2))
    a = matrix(40, 64, torch.float32, 1)
    for given in (a, ops.mxfp4_quantize(a)):
        buf = torch.zeros(40, 64, device="cuda")
        y = (torch.ones(40, 64, device="cuda", requires_grad=True) * buf).sum()
        ops.mxfp4_linear(given, W, out=buf)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        buf = torch.zeros(40, 64, device="cuda")
    assert torch.equal(ops.mxfp4_linear(a, W, out=buf), ops.mxfp4_linear(a, W))


# The forms that the cases above leave out.  Tiles of 256 x 256 whose rows are whole lines of 128 bytes, several for every
# workgroup; rows of at least four stages that end in half a stage, whatever the kernel.
WHOLE_LINES = [(2048, 30208), (2100, 30208), (2048, 30016), (2100, 30016)]  # (rows and columns that fill their tiles, or do not)
LONG_ROUTES = [(40, 300), (100, 5100), (3, 90001), (50, 41003), (500, 23001), (520, 40001), (40, 300)]


def long_cases():
    return [(N, M, 1100) for N, M in LONG_ROUTES[:-1]] + [(N, M, 1900) for N, M in LONG_ROUTES[-1:]]


def drawn(R, K, seed, dtype=torch.float32):
    """As ``matrix``, made on the GPU (large ones)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(R, K, generator=g, device="cuda")
    return (x * torch.exp(torch.randn(R, K, generator=g, device="cuda"))).to(dtype)


def exact_product(xq, Wq, b=None):
    """In 64 bits, and how far fp32 accumulation may be off (the module's bound); NaN wherever a NaN goes in."""
    xv, wv = xq.dequantize().double(), Wq.dequantize().double()
    ref = xv @ wv.t()
    room = xv.shape[1] * 2.0**-23 * (torch.nan_to_num(xv).abs() @ torch.nan_to_num(wv).abs().t())
    if b is not None:
        ref = ref + b.double()
        room = room + 2.0**-24 * ref.abs()
    return ref, room


@pytest.mark.gpu
@pytest.mark.parametrize("K", [64, 300, 512, 700])
@pytest.mark.parametrize("N,M", WHOLE_LINES)
def test_linear_whole_lines(N, M, K):
    """Every form of the large kernel: both types, with and without ReLU, no bias or one of either type."""
    from clt_training_amd import hip_ops as ops

    xq, Wq = ops.mxfp4_quantize(drawn(N, K, 1)), ops.mxfp4_quantize(drawn(M, K, 2))
    for b in (None, drawn(1, M, 3)[0], drawn(1, M, 4, torch.bfloat16)[0]):
        ref, room = exact_product(xq, Wq, b)
        for relu in (False, True):
            want = ref.clamp(min=0) if relu else ref
            for dt in (torch.bfloat16, torch.float32):
                assert route(N, M, K, dt) == "256 x 256"
                y = ops.mxfp4_linear(xq, Wq, b, relu=relu, out_dtype=dt)
                assert y.data_ptr() % 128 == 0
                allowed = room + (torch.finfo(dt).eps / 2 if dt != torch.float32 else 0) * (ref.abs() + room)
                bad = ((y.double() - want).abs() > allowed).nonzero()
                assert len(bad) == 0, (b is not None and b.dtype, relu, dt, len(bad), bad[:4].tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("N,M,K", long_cases())
def test_linear_special_values_in_long_rows(N, M, K):
    """NaN in every quarter of the columns and in the last, half-empty stage, rows of NaN behind rows that end there, and biases
    that are not finite."""
    from clt_training_amd import hip_ops as ops

    x, W, b = drawn(N, K, 1), drawn(M, K, 2), drawn(1, M, 3)[0]
    x[1] = float("nan")
    bad_rows = [9, 21, 33, 40, 47, M - 1]
    for r, c in zip(bad_rows, (3, K // 4 + 40, K // 2 + 40, K - 150, K - 1, K - 60)):
        W[r, c] = float("-inf")
    W[21], W[M - 1] = float("nan"), float("nan")
    b[0], b[1], b[2] = float("nan"), float("inf"), float("-inf")
    xq, Wq = ops.mxfp4_quantize(x), ops.mxfp4_quantize(W)
    ref, room = exact_product(xq, Wq, b)
    for relu in (False, True):
        want = torch.where(ref < 0, 0, ref) if relu else ref
        for given in (x, xq):
            y = ops.mxfp4_linear(given, Wq, b, relu=relu)
            assert torch.equal(torch.isnan(y), torch.isnan(want)) and int(torch.isnan(y).sum()) == M + (1 + len(bad_rows)) * (N - 1)
            sure = torch.isfinite(want)
            assert ((y.double() - want).abs() <= room)[sure].all() and torch.equal(y.double()[torch.isinf(want)], want[torch.isinf(want)])


@pytest.mark.gpu
@pytest.mark.parametrize("N,M,K", long_cases())
def test_linear_any_alignment_in_long_rows(N, M, K):
    """As test_linear_any_alignment_every_route."""
    from clt_training_amd import hip_ops as ops

    xs, b, Wq = drawn(N, K + 3, 4), drawn(1, M + 1, 5, torch.bfloat16)[0][1:], ops.mxfp4_quantize(drawn(M, K, 6))
    for dt in (torch.bfloat16, torch.float32):
        want = ops.mxfp4_linear(xs[:, 1:K + 1].contiguous(), Wq, b.clone(), relu=True, out_dtype=dt)
        big = torch.full((N + 2, M + 9), 7.0, dtype=dt, device="cuda")
        y = ops.mxfp4_linear(xs[:, 1:K + 1], Wq, b, relu=True, out=big[1:N + 1, 3:3 + M])
        assert torch.equal(y, want)
        y.fill_(7)
        assert (big == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("N,M,K", long_cases())
def test_linear_two_graphs_in_long_rows(N, M, K):
    """Two captured graphs replayed in turn, three times, with eager work between."""
    from clt_training_amd import hip_ops as ops

    W = [ops.mxfp4_quantize(drawn(M, K, 7 + i)) for i in range(2)]
    x = [drawn(N, K, 9 + i, torch.bfloat16) for i in range(2)]
    eager = lambda i: ops.mxfp4_linear(x[i], W[i], relu=True)  # noqa: E731
    eager(0), eager(1)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(eager(i))
        graphs.append(g)
    for seed in range(3):
        for i in range(2):
            x[i].copy_(drawn(N, K, 20 + 2 * seed + i, torch.bfloat16))
        want = [eager(0), eager(1)]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
