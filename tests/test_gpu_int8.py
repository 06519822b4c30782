"""The operators on rows of 8-bit integers against their formulas in 64 bits: rows made 8-bit, the norm that makes them, products."""
import math

import pytest
import torch

import int8_oracle as oracle
from int8_oracle import U

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from jllm_serve_amd.kernels import ops
    ops.library()
    return ops


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def seeded(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def strided(x, pad, at=0):
    """The same rows further apart, beginning ``at`` entries into their memory."""
    big = torch.full((x.shape[0] * (x.shape[1] + pad) + at + 1,), 77, dtype=x.dtype, device=x.device)
    view = big[at:at + x.shape[0] * (x.shape[1] + pad)].view(x.shape[0], x.shape[1] + pad)[:, :x.shape[1]]
    view.copy_(x)
    return view, big


WIDTHS = [1, 3, 7, 8, 9, 15, 16, 64, 100, 505, 512, 520, 1000, 1024, 1031, 2048, 2055, 4096, 5120, 5123, 6151, 8192, 8200, 12288, 17408, 25600, 32768, 32771, 40000]


# fp32 roundings of a norm's scale: the inverse root (its sum is in 64 bits), two products, the quotient; and of an entry against the row's
# largest, where the inverse root cancels: two products each, the quotient 127 / largest, the last product
NORM_SCALE, NORM_ENTRY = 5, 6


# ------------------------------------------------------------------------------------------------ rows made 8-bit


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_rows(ops, width, dtype):
    gen = seeded(width)
    x = (normal(gen, 5, width) * torch.tensor([1.0, 1e-3, 4e4, 1e-20, 1.0], device=DEV)[:, None]).to(dtype)
    x[4] = 0
    got = ops.quantize_rows(x)
    assert got.q.dtype == torch.int8 and got.scale.dtype == torch.float32
    oracle.check_rows(got.q, got.scale, x, 2, 1)
    assert float(got.scale[4]) == 0 and not got.q[4].any()
    for pad, at in ((1, 0), (8, 3), (0, 1), (24, 8)):
        again = ops.quantize_rows(strided(x, pad, at)[0])
        assert torch.equal(again.q, got.q) and torch.equal(again.scale, got.scale)
    for t in (torch.float32, torch.bfloat16):
        back = got.tensor(t)
        want = (got.q.float() * got.scale[:, None]).to(t)
        assert back.dtype == t and torch.equal(back, want)
    q, _ = strided(got.q, 5, 3)
    assert torch.equal(ops.Int8Rows(q, got.scale).tensor(torch.float32), got.tensor(torch.float32))


def test_quantize_rounds_halves_to_even(ops):
    """A largest value of 127 makes the scale one: what lies between whole numbers goes to the even one."""
    x = torch.arange(-127, 127.5, 0.5, device=DEV)[None, :].contiguous()
    got = ops.quantize_rows(x)
    assert float(got.scale[0]) == 1
    assert torch.equal(got.q.float(), torch.round(x))
    oracle.check_rows(got.q, got.scale, x, 0, 0)


@pytest.mark.parametrize("width", [5, 9, 700, 4096, 9000, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_quantize_rows_of_all_magnitudes(ops, width, dtype):
    gen = seeded(3)
    x = normal(gen, 6, width).clamp(-3, 3)
    scale = torch.tensor([2.0 ** e for e in (125, -90, -105, -120, -135, -149)], dtype=torch.float64)
    x = (x.double().cpu() * scale[:, None]).to(dtype).to(DEV)
    got = ops.quantize_rows(x)
    # (below 2^-100 the rows are scaled up first, exactly)
    oracle.check_rows(got.q, got.scale, x, 2, 1)


@pytest.mark.parametrize("width", [4, 40, 1500, 8192, 33000])
def test_rows_with_nan_or_infinity(ops, width):
    gen = seeded(5)
    x = normal(gen, 5, width)
    x[1, width // 2] = float("nan")
    x[2, 0] = float("inf")
    x[3, width - 1] = -float("inf")
    got = ops.quantize_rows(x)
    assert torch.isnan(got.scale).tolist() == [False, True, True, True, False]
    assert not got.q[1:4].any()
    clean = ops.quantize_rows(x[[0, 4]].contiguous())
    assert torch.equal(got.q[[0, 4]], clean.q) and torch.equal(got.scale[[0, 4]], clean.scale)
    g = torch.ones(width, device=DEV)
    got = ops.rmsnorm_int8(x, g, 1e-6)
    assert torch.isnan(got.scale).tolist() == [False, True, True, True, False] and not got.q[1:4].any()
    w = ops.quantize_rows(normal(gen, 7, width))
    y = ops.gemm_int8(got, w, out_dtype=torch.float32)
    assert torch.isnan(y[1:4]).all() and not torch.isnan(y[[0, 4]]).any()


@pytest.mark.parametrize("rows", [0, 1, 2, 300, 5000])
def test_numbers_of_rows(ops, rows):
    gen = seeded(rows)
    x = normal(gen, rows, 264)
    got = ops.quantize_rows(x)
    assert got.q.shape == (rows, 264) and got.scale.shape == (rows,)
    normed = ops.rmsnorm_int8(x, torch.ones(264, device=DEV), 1e-6)
    assert normed.tensor(torch.bfloat16).shape == (rows, 264)
    if rows:
        oracle.check_rows(got.q, got.scale, x, 2, 1)
        oracle.check_rows(normed.q, normed.scale, oracle.norm(x, torch.ones(264), 1e-6)[1], NORM_ENTRY, NORM_SCALE)


# ------------------------------------------------------------------------------------------------ the norm


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("adt,gdt", [(None, torch.bfloat16), (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_rmsnorm_int8(ops, width, adt, gdt):
    gen = seeded(width)
    x = normal(gen, 5, width) * 3
    x[2] = 0
    gain = (1 + 0.2 * normal(gen, width)).to(gdt)
    add = None
    if adt is not None:
        add = normal(gen, 5, width).to(adt)
        add[2] = 0
    h, y = oracle.norm(x, gain, 1e-5, add)
    before = x.clone()
    place = torch.empty_like(x) if add is not None else None
    got = ops.rmsnorm_int8(x, gain, 1e-5, add=add, out=place)
    assert torch.equal(x, before)
    oracle.check_rows(got.q, got.scale, y, NORM_ENTRY, NORM_SCALE)
    assert float(got.scale[2]) == 0 and not got.q[2].any()
    if add is not None:
        assert torch.equal(place.cpu(), h)
    # rows, sums and gains that begin anywhere, the sum in place: the same bits
    for pad, at in ((1, 1), (8, 0), (3, 2)):
        xs, xbig = strided(x, pad, at)
        gs = strided(gain[None, :], 0, at)[0][0]
        kept = xbig.clone()
        as_ = None if add is None else strided(add, pad + 2, at)[0]
        again = ops.rmsnorm_int8(xs, gs, 1e-5, add=as_)
        assert torch.equal(again.q, got.q) and torch.equal(again.scale, got.scale)
        if add is not None:
            assert torch.equal(xs, place)
            xs.copy_(x)
        assert torch.equal(xbig, kept)  # nothing between the rows or behind them was written


@pytest.mark.parametrize("width", [5, 40, 100, 1031, 5120, 20000, 33000])
def test_norm_of_a_sum_of_shared_rows(ops, width):
    """The rows to add may be x itself, and the sum may go into them."""
    gen = seeded(width)
    x, add, g = normal(gen, 6, width), normal(gen, 6, width), normal(gen, width)
    want, place = ops.rmsnorm_int8(x, g, 1e-6, add=add, out=torch.empty_like(x)), x + add
    into = add.clone()
    got = ops.rmsnorm_int8(x, g, 1e-6, add=into, out=into)
    assert torch.equal(got.q, want.q) and torch.equal(got.scale, want.scale) and torch.equal(into, place)
    twice = x.clone()
    got = ops.rmsnorm_int8(twice, g, 1e-6, add=twice)
    want = ops.rmsnorm_int8(2 * x, g, 1e-6)
    assert torch.equal(got.q, want.q) and torch.equal(got.scale, want.scale) and torch.equal(twice, 2 * x)


@pytest.mark.parametrize("width", [40, 5120, 33000])
def test_norm_of_large_and_small_rows(ops, width):
    """Rows whose squares fp32 does not hold: beyond 1e38, and below 1e-45 with an eps as small."""
    gen = seeded(width)
    x = normal(gen, 4, width).clamp(-4, 4) * torch.tensor([1e30, 1e-30, 3e37, 1.0], device=DEV)[:, None]
    g = 1 + 0.1 * normal(gen, width)
    got = ops.rmsnorm_int8(x, g, 1e-38)
    oracle.check_rows(got.q, got.scale, oracle.norm(x, g, float(torch.tensor(1e-38)))[1], NORM_ENTRY, NORM_SCALE)


def test_norm_of_rows_beside_others(ops):
    """A row's bits do not depend on the rows beside it."""
    gen = seeded(2)
    x, g = normal(gen, 400, 2560), normal(gen, 2560)
    whole = ops.rmsnorm_int8(x, g, 1e-6)
    for r in (0, 17, 399):
        one = ops.rmsnorm_int8(x[r:r + 1], g, 1e-6)
        assert torch.equal(one.q[0], whole.q[r]) and torch.equal(one.scale[0], whole.scale[r])


# ------------------------------------------------------------------------------------------------ products

SHAPES = [(1, 1, 1), (1, 16, 128), (2, 3, 15), (3, 50, 70), (5, 48, 384), (7, 129, 16), (8, 6144, 256), (1, 4096, 1152), (16, 4112, 512), (16, 80, 4096),
          (17, 80, 256), (20, 4112, 512), (31, 100, 1037), (33, 16, 1024), (64, 304, 640), (50, 144, 2176), (64, 1000, 1040), (48, 512, 8192),
          (65, 96, 128), (77, 205, 1037), (90, 136, 320), (100, 256, 64), (128, 256, 512), (130, 272, 2064), (200, 130, 96), (255, 1000, 272),
          (256, 256, 1024), (257, 513, 144), (300, 384, 4096), (631, 640, 2176), (1000, 192, 136), (1100, 530, 1040), (513, 4100, 528)]


def operands(ops, gen, M, N, K):
    a = ops.quantize_rows(normal(gen, M, K))
    w = ops.quantize_rows(normal(gen, N, K) / math.sqrt(K))
    w2 = ops.quantize_rows(normal(gen, N, K) / math.sqrt(K))
    return a, w, w2


def close(got, want, tol):
    got = got.double().cpu()
    assert not torch.isnan(got).any()
    off = (got - want).abs() - tol
    assert (off <= 0).all(), (float(off.max()), int((off > 0).sum()), want.numel())


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm_int8(ops, M, N, K):
    gen = seeded(M * 7 + N + K)
    a, w, w2 = operands(ops, gen, M, N, K)
    b32, b16 = normal(gen, N), normal(gen, N).bfloat16()
    for bias in (None, b32, b16):
        y, tol = oracle.product(a, w, bias)
        for dtype in (torch.float32, torch.bfloat16):
            out = ops.gemm_int8(a, w, bias=bias, out_dtype=dtype)
            assert out.dtype == dtype
            close(out, y, oracle.stored(tol, y, dtype))
    # added into the residual
    res = normal(gen, M, N)
    y, tol = oracle.product(a, w, b32, res)
    assert ops.gemm_int8(a, w, bias=b32, out=res, epilogue=ops.EPI_ADD) is res
    close(res, y, tol)
    # gated: z with its roundings, exp2 and the reciprocal to one unit each, their argument's six roundings, the last products
    z, u = oracle.sums(a, w), oracle.sums(a, w2)
    y = oracle.gate("silu", z, u)
    tol = y.abs() * (13 + 6 * z.abs()) * U * 1.01 + 1e-30
    for dtype in (torch.float32, torch.bfloat16):
        out = ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED, out_dtype=dtype)
        close(out, y, oracle.stored(tol, y, dtype))


@pytest.mark.parametrize("M,N,K", [(1, 50, 70), (5, 48, 384), (20, 208, 512), (64, 304, 640), (77, 205, 1037), (300, 384, 1024), (257, 513, 144)])
def test_gemm_int8_rows_anywhere(ops, M, N, K):
    """Operands and outputs whose rows lie apart and begin at any byte: the same bits, and nothing beside the outputs is written."""
    gen = seeded(N)
    a, w, w2 = operands(ops, gen, M, N, K)
    bias = normal(gen, N)
    want = ops.gemm_int8(a, w, bias=bias, out_dtype=torch.float32)
    gated = ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED)
    added = normal(gen, M, N)
    base = added.clone()
    ops.gemm_int8(a, w, out=added, epilogue=ops.EPI_ADD)
    for pad, at in ((16, 0), (128, 16), (1, 0), (5, 3), (0, 1)):
        a_, w_, w2_ = (ops.Int8Rows(strided(t.q, pad, at)[0], t.scale) for t in (a, w, w2))
        out, big = strided(torch.zeros_like(want), pad, at)
        kept = big.clone()
        assert torch.equal(ops.gemm_int8(a_, w_, bias=bias, out=out), want)
        out.zero_()
        assert torch.equal(big, kept)
        out, big = strided(torch.zeros_like(gated), pad, at)
        kept = big.clone()
        assert torch.equal(ops.gemm_int8(a_, w_, w2=w2_, epilogue=ops.EPI_GATED, out=out), gated)
        out.zero_()
        assert torch.equal(big, kept)
        out, big = strided(base, pad, at)
        kept = big.clone()
        assert torch.equal(ops.gemm_int8(a_, w_, out=out, epilogue=ops.EPI_ADD), added)
        out.copy_(base)
        assert torch.equal(big, kept)


@pytest.mark.parametrize("M,N", [(1, 40), (9, 64), (40, 64), (70, 144), (300, 272)])
def test_largest_sums(ops, M, N):
    """131,071 products of -128 and -128 are the largest sum that 32 bits hold; every sum is exact."""
    K = 131071
    a = torch.full((M, K), -128, dtype=torch.int8, device=DEV)
    w = torch.full((N, K), -128, dtype=torch.int8, device=DEV)
    w[1::2] = 127
    a[:, 0], w[:, 0] = 1, 1
    a_, w_ = ops.Int8Rows(a, torch.ones(M, device=DEV)), ops.Int8Rows(w, torch.ones(N, device=DEV))
    want = torch.tensor([(K - 1) * 128 * 128 + 1, -(K - 1) * 128 * 127 + 1], dtype=torch.float64).to(torch.float32).repeat(N // 2)
    assert torch.equal(ops.gemm_int8(a_, w_, out_dtype=torch.float32).cpu(), want.expand(M, N))


@pytest.mark.parametrize("M,N,K,pad,at,kernel", [
    (1, 300, 4096, 0, 0, "jllm_gemm_int8_stream"), (64, 300, 4096, 16, 16, "jllm_gemm_int8_stream"), (40, 300, 4096, "a", 3, "jllm_gemm_int8_stream"),
    (65, 300, 1040, 0, 0, "jllm_gemm_int8_tiled"), (100, 300, 1040, "a", 1, "jllm_gemm_int8_tiled"), (2100, 4096, 2064, 0, 0, "jllm_gemm_int8_large"),
    (2100, 4096, 2061, 0, 0, "jllm_gemm_int8_large"), (2100, 4096, 2064, 1, 0, "jllm_gemm_int8_large"), (2100, 4096, 2064, 0, 5, "jllm_gemm_int8_large"),
    (3, 300, 8191, 0, 0, None), (70, 300, 8191, 0, 0, None), (3, 300, 131071, 0, 0, None), (1100, 300, 131071, 0, 0, None), (200, 130, 144, 1, 0, None)])
@pytest.mark.parametrize("gated", [False, True])
def test_each_kernel_takes_its_products(ops, M, N, K, pad, at, kernel, gated):
    """Which kernel a product goes through (None: the general one), with K cut or whole, operands as they lie or laid out anew."""
    gen = seeded(M + K)
    a, w, w2 = operands(ops, gen, M, N, K)
    if pad == "a":  # the activations alone begin anywhere
        a = ops.Int8Rows(strided(a.q, 0, at)[0], a.scale)
    elif pad or at:
        a, w, w2 = (ops.Int8Rows(strided(t.q, pad, at)[0], t.scale) for t in (a, w, w2))
    ops.reset_stats()
    if gated:
        got = ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED, out_dtype=torch.float32)
    else:
        got = ops.gemm_int8(a, w, out_dtype=torch.float32)
    ran = ops.stats()
    assert list(ran["ran"]) == ([kernel] if kernel else []) and list(ran["general"]) == ([] if kernel else ["jllm_gemm_int8"]), ran
    if gated:
        z, u = oracle.sums(a, w), oracle.sums(a, w2)
        y = oracle.gate("silu", z, u)
        tol = y.abs() * (13 + 6 * z.abs()) * U * 1.01 + 1e-30
    else:
        y, tol = oracle.product(a, w)
    close(got, y, tol)


TILES = [("jllm_gemm_int8_tiled", t) for t in (64064, 64128, 128128)] + [("jllm_gemm_int8_large", t) for t in (128256, 256128, 192256, 256256)]


@pytest.mark.parametrize("kernel,tile", TILES)
@pytest.mark.parametrize("K", [144, 256, 400, 640, 656, 1040, 2176, 2192])
def test_every_tile(ops, monkeypatch, kernel, tile, K):
    """Each tile by name, at numbers of whole and cut stages around its ring's depth, K whole and in parts, with rows and columns that end inside a
    tile: the bits of the general kernel."""
    gen = seeded(tile + K)
    for M, N in ((1, 5), (70, 300), (300, 130), (513, 520)):
        a, w, w2 = operands(ops, gen, M, N, K)
        bias, base = normal(gen, N), normal(gen, M, N)
        monkeypatch.setattr(ops, "_int8_plans", lambda *args: ())
        want = ops.gemm_int8(a, w, bias=bias, out_dtype=torch.float32)
        narrow = ops.gemm_int8(a, w)
        gated = ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED, out_dtype=torch.float32)
        added = ops.gemm_int8(a, w, out=base.clone(), epilogue=ops.EPI_ADD)
        for parts in (1, 2, 3, 5):
            stages = -(-K // 128)
            if parts > 1 and stages <= -(-stages // parts) * (parts - 1):
                continue  # a part without any
            monkeypatch.setattr(ops, "_int8_plans", lambda *args: ((0.0, kernel, tile, parts),))
            ops.reset_stats()
            assert torch.equal(ops.gemm_int8(a, w, bias=bias, out_dtype=torch.float32), want)
            assert torch.equal(ops.gemm_int8(a, w), narrow)
            assert torch.equal(ops.gemm_int8(a, w, out=base.clone(), epilogue=ops.EPI_ADD), added)
            assert ops.stats()["ran"] == {kernel: 3}
            if parts == 1:
                assert torch.equal(ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED, out_dtype=torch.float32), gated)


@pytest.mark.parametrize("kernel,tile", TILES)
@pytest.mark.parametrize("K", [144, 256, 656, 1040, 2192])
def test_every_tile_gated_in_parts(ops, monkeypatch, kernel, tile, K):
    """Both weights' sums of every part, rows and columns ending inside a tile: the bits of the general kernel."""
    gen = seeded(tile + K + 1)
    for M, N in ((1, 5), (70, 300), (300, 130), (513, 523)):
        a, w, w2 = operands(ops, gen, M, N, K)
        bias = normal(gen, N)
        call = lambda dtype: ops.gemm_int8(a, w, w2=w2, bias=bias, epilogue=ops.EPI_GATED, out_dtype=dtype)
        monkeypatch.setattr(ops, "_int8_plans", lambda *args: ())
        want, narrow = call(torch.float32), call(torch.bfloat16)
        for parts in (2, 3, 5):
            stages = -(-K // 128)
            if stages <= -(-stages // parts) * (parts - 1):
                continue
            monkeypatch.setattr(ops, "_int8_plans", lambda *args: ((0.0, kernel, tile, parts),))
            ops.reset_stats()
            assert torch.equal(call(torch.float32), want) and torch.equal(call(torch.bfloat16), narrow)
            assert ops.stats()["ran"] == {kernel: 2}


PLACES = [("", 0, 1)] + [(kernel, tile, parts) for kernel, tile in TILES + [("jllm_gemm_int8_stream", 24)] for parts in (1, 2)]


@pytest.mark.parametrize("kernel,size,parts", PLACES)
def test_outputs_at_any_element(ops, monkeypatch, kernel, size, parts):
    """Rows of outputs that begin at any element and lie any distance apart, whole runs of columns and cut ones: the values, and nothing beside them."""
    gen = seeded(size + parts)
    M, K = 64 if kernel.endswith("stream") else 150, 656
    for N, pad, at in ((261, 0, 1), (256, 1, 0), (256, 3, 5), (262, 2, 2), (512, 5, 3)):
        a, w, w2 = operands(ops, gen, M, N, K)
        for dtype in (torch.float32, torch.bfloat16):
            for kw in (dict(), dict(w2=w2, epilogue=ops.EPI_GATED)) + ((dict(epilogue=ops.EPI_ADD),) if dtype == torch.float32 else ()):
                adds = kw.get("epilogue") == ops.EPI_ADD
                monkeypatch.setattr(ops, "_int8_plans", lambda *args: ())
                want = ops.gemm_int8(a, w, out=torch.ones(M, N, device="cuda"), **kw) if adds else ops.gemm_int8(a, w, out_dtype=dtype, **kw)
                monkeypatch.setattr(ops, "_int8_plans", lambda *args: ((0.0, kernel, size, parts),) if kernel else ())
                memory = torch.ones(at + M * (N + pad) + 8, dtype=dtype, device="cuda")
                out = memory[at:at + M * (N + pad)].view(M, N + pad)[:, :N]
                ops.gemm_int8(a, w, out=out, **kw)
                assert torch.equal(out, want)
                out.fill_(1)
                assert (memory == 1).all()


@pytest.mark.parametrize("M", [1, 8, 9, 30, 48, 64])
@pytest.mark.parametrize("K", [16, 128, 144, 1040, 2176, 8208])
def test_every_number_of_weight_rows(ops, monkeypatch, M, K):
    """The weight-streaming kernel at every number of weight rows per workgroup, K whole and in parts: the bits of the general kernel."""
    gen = seeded(M + K)
    N = 203
    a, w, w2 = operands(ops, gen, M, N, K)
    base = normal(gen, M, N)
    monkeypatch.setattr(ops, "_int8_plans", lambda *args: ())
    want = ops.gemm_int8(a, w)
    gated = ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED)
    added = ops.gemm_int8(a, w, out=base.clone(), epilogue=ops.EPI_ADD)
    for rows in (1, 3, 8, 12, 16, 20, 24, 28, 32, 40, 48, 56, 64, 72, 80, 96):
        for parts in (1, 2, 4, 7):
            monkeypatch.setattr(ops, "_int8_plans", lambda *args: ((0.0, "jllm_gemm_int8_stream", rows, parts),))
            ops.reset_stats()
            assert torch.equal(ops.gemm_int8(a, w), want)
            assert torch.equal(ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED), gated)
            assert torch.equal(ops.gemm_int8(a, w, out=base.clone(), epilogue=ops.EPI_ADD), added)
            assert ops.stats()["ran"] == {"jllm_gemm_int8_stream": 3}


@pytest.mark.parametrize("gate,limit", [("gelu_tanh", 0.0), ("swish_clamped", 1.5)])
@pytest.mark.parametrize("M,N,K", [(3, 50, 70), (4, 256, 512), (40, 256, 512), (300, 272, 528)])
def test_gate_functions(ops, gate, limit, M, N, K):
    gen = seeded(K)
    a, w, w2 = operands(ops, gen, M, N, K)
    z, u = oracle.sums(a, w), oracle.sums(a, w2)
    y = oracle.gate(gate, z, u, limit)
    got = ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED, gate=ops.GATE_FUNCTIONS[gate], gate_limit=limit, out_dtype=torch.float32)
    if gate == "gelu_tanh":  # the exponent 2 inner log2(e) with some 17 roundings of its terms
        inner = 0.7978845608028654 * (z.abs() + 0.044715 * z.abs() ** 3)
        tol = y.abs() * (13 + 34 * inner) * U * 1.01 + 1e-30
    else:  # 1.702 g; u + 1 may cancel
        g = torch.clamp(z, max=limit)
        s = (g * torch.sigmoid(1.702 * g)).abs()
        tol = y.abs() * (13 + 12 * g.abs()) * U + s * 4 * U * (u.abs() + 1) + 1e-30
    close(got, y, tol)


@pytest.mark.parametrize("gate,limit", [("silu", 0.0), ("gelu_tanh", 0.0), ("swish_clamped", 1.5)])
def test_gate_functions_alike_in_every_kernel(ops, monkeypatch, gate, limit):
    gen = seeded(31)
    for kernel, size in TILES + [("jllm_gemm_int8_stream", 24)]:
        M, N, K = 64 if kernel.endswith("stream") else 300, 264, 1040
        a, w, w2 = operands(ops, gen, M, N, K)
        call = lambda: ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED, gate=ops.GATE_FUNCTIONS[gate], gate_limit=limit, out_dtype=torch.float32)
        monkeypatch.setattr(ops, "_int8_plans", lambda *args: ())
        want = call()
        for parts in (1, 3):
            monkeypatch.setattr(ops, "_int8_plans", lambda *args: ((0.0, kernel, size, parts),))
            assert torch.equal(call(), want), (kernel, size, parts)


@pytest.mark.parametrize("gate,limit", [("silu", 0.0), ("gelu_tanh", 0.0), ("swish_clamped", 1.5)])
@pytest.mark.parametrize("M", [3, 40, 90, 300])
def test_rows_and_channels_without_numbers(ops, gate, limit, M):
    """A row of activations with a NaN is a row of NaN behind every gate, a weight's channel a column; nothing else is."""
    gen = seeded(M)
    N, K = 300, 512
    x, y, z = normal(gen, M, K), normal(gen, N, K), normal(gen, N, K)
    x[1, 7], y[5, 0], z[290, K - 1] = float("nan"), float("inf"), float("nan")
    a, w, w2 = (ops.quantize_rows(t) for t in (x, y, z))
    got = ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED, gate=ops.GATE_FUNCTIONS[gate], gate_limit=limit, out_dtype=torch.float32)
    want = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    want[1], want[:, 5], want[:, 290] = True, True, True
    assert torch.equal(torch.isnan(got), want)
    want[:, 290] = False
    want[1] = True
    assert torch.equal(torch.isnan(ops.gemm_int8(a, w)), want)


def test_offsets_beyond_32_bits(ops):
    """Rows, weights and outputs of more than 2^31 entries: the ends of them against the same rows alone."""
    n, width = 70000, 32768
    x = torch.empty((n, width), dtype=torch.bfloat16, device=DEV)
    gen = seeded(1)
    some = normal(gen, 500, width).bfloat16()
    for r in range(0, n, 500):
        x[r:r + 500] = some
        x[r:r + 500] *= 1 + r % 3
    ends = slice(n - 300, n)
    rows = ops.quantize_rows(x)
    want = ops.quantize_rows(x[ends])
    assert torch.equal(rows.q[ends], want.q) and torch.equal(rows.scale[ends], want.scale)
    assert torch.equal(rows.tensor(torch.bfloat16)[ends], want.tensor(torch.bfloat16))
    # activations of 2.3 GB, and outputs as many
    w = ops.quantize_rows(normal(gen, 200, width))
    assert torch.equal(ops.gemm_int8(rows, w)[ends], ops.gemm_int8(want, w))
    narrow = ops.Int8Rows(rows.q[:, :64], rows.scale)
    wide = ops.quantize_rows(normal(gen, width, 64))
    out = ops.gemm_int8(narrow, wide)
    assert out.numel() > 1 << 31
    assert torch.equal(out[ends], ops.gemm_int8(ops.Int8Rows(narrow.q[ends], narrow.scale[ends]), wide))
    del out
    # weights of 4.6 GB: both ends of two copies, for every kernel
    q = torch.cat([rows.q, rows.q])
    scale = torch.cat([rows.scale, rows.scale])
    big = ops.Int8Rows(q, scale)
    last = ops.Int8Rows(q[2 * n - 300:], scale[2 * n - 300:])
    for m in (1, 40, 100, 700):
        a = ops.quantize_rows(normal(gen, m, width))
        got = ops.gemm_int8(a, big, out_dtype=torch.float32)
        assert torch.equal(got[:, 2 * n - 300:], ops.gemm_int8(a, last, out_dtype=torch.float32))
        got = ops.gemm_int8(a, big, w2=big, epilogue=ops.EPI_GATED)
        assert torch.equal(got[:, 2 * n - 300:], ops.gemm_int8(a, last, w2=last, epilogue=ops.EPI_GATED))
    # and as activations
    got = ops.gemm_int8(big, w)
    assert torch.equal(got[2 * n - 300:], ops.gemm_int8(last, w))
    del q, big, last, rows
    # the norm of a stream of 9 GB, the sum in place
    h = x.float()
    g = 1 + 0.1 * normal(gen, width)
    before = h[ends].clone()
    rows = ops.rmsnorm_int8(h, g, 1e-6, add=x)
    want = ops.rmsnorm_int8(before, g, 1e-6, add=x[ends])
    assert torch.equal(rows.q[ends], want.q) and torch.equal(rows.scale[ends], want.scale) and torch.equal(h[ends], before)


def test_a_row_has_the_same_bits_in_any_batch(ops):
    """Whatever kernel, tile and cut the number of rows leads to, with every epilogue."""
    gen = seeded(11)
    a, w, w2 = operands(ops, gen, 1200, 640, 1152)
    bias, base = normal(gen, 640), normal(gen, 1200, 640)
    calls = [lambda part, rows: ops.gemm_int8(part, w, bias=bias, out_dtype=torch.float32), lambda part, rows: ops.gemm_int8(part, w),
             lambda part, rows: ops.gemm_int8(part, w, w2=w2, epilogue=ops.EPI_GATED, out_dtype=torch.float32),
             lambda part, rows: ops.gemm_int8(part, w, bias=bias, out=base[rows].clone(), epilogue=ops.EPI_ADD)]
    whole = [call(a, slice(0, 1200)) for call in calls]
    for n in (1, 5, 16, 17, 33, 64, 65, 128, 200, 257, 513, 1100):
        rows = slice(3, 3 + n)
        for call, want in zip(calls, whole):
            assert torch.equal(call(ops.Int8Rows(a.q[rows], a.scale[rows]), rows), want[rows]), n


def test_no_rows_and_no_outputs(ops):
    gen = seeded(1)
    a, w, _ = operands(ops, gen, 4, 32, 64)
    none = ops.Int8Rows(a.q[:0], a.scale[:0])
    assert ops.gemm_int8(none, w).shape == (0, 32)
    assert ops.gemm_int8(a, ops.Int8Rows(w.q[:0], w.scale[:0])).shape == (4, 0)


# ------------------------------------------------------------------------------------------------ together


def feed_forward(ops, x, attended, gain, gate, up, down):
    """A layer's second half on 8-bit weights: x += what the attention left; x += down(silu(gate n) * (up n)) with n the norm of x."""
    n = ops.rmsnorm_int8(x, gain, 1e-6, add=attended)
    hidden = ops.gemm_int8(n, gate, w2=up, epilogue=ops.EPI_GATED)
    return n, hidden, ops.gemm_int8(ops.quantize_rows(hidden), down, out=x, epilogue=ops.EPI_ADD)


@pytest.mark.parametrize("rows,width,inner", [(1, 256, 768), (8, 512, 1536), (37, 320, 1000), (64, 1024, 2048), (130, 256, 768), (600, 512, 1024)])
def test_a_feed_forward_of_8_bit_rows(ops, rows, width, inner):
    gen = seeded(rows)
    x0, attended = normal(gen, rows, width), normal(gen, rows, width).bfloat16()
    gain = 1 + 0.1 * normal(gen, width)
    full = [normal(gen, inner, width) / math.sqrt(width), normal(gen, inner, width) / math.sqrt(width), normal(gen, width, inner) / math.sqrt(inner)]
    gate, up, down = (ops.quantize_rows(t) for t in full)
    x = x0.clone()
    n, hidden, out = feed_forward(ops, x, attended, gain, gate, up, down)
    # every step against the formula on the step's own inputs
    h, y = oracle.norm(x0, gain, 1e-6, attended)
    oracle.check_rows(n.q, n.scale, y, NORM_ENTRY, NORM_SCALE)
    z, u = oracle.sums(n, gate), oracle.sums(n, up)
    want = oracle.gate("silu", z, u)
    close(hidden, want, oracle.stored(want.abs() * (13 + 6 * z.abs()) * U * 1.01 + 1e-30, want, torch.bfloat16))
    rows8 = ops.quantize_rows(hidden)
    want, tol = oracle.product(rows8, down, None, h)
    close(out, want, tol)
    # and the whole against the same without 8-bit rows: a rounding to whole steps of max / 127 is off by a step / sqrt(12) on
    # average; five such roundings of rows whose largest value is up to 4.5 times their root mean square (8 for the hidden
    # rows, whose values are products), independent of each other, and twice that for good measure
    full_y = oracle.gate("silu", y @ full[0].double().cpu().t(), y @ full[1].double().cpu().t()) @ full[2].double().cpu().t()
    step = math.sqrt(5 * 4.5 ** 2 + 10 ** 2) / 127 / math.sqrt(12)
    delta = out.double().cpu() - h.double()
    assert float((delta - full_y).norm() / full_y.norm()) < 2 * step


@pytest.mark.parametrize("rows", [1, 8, 40, 200])
def test_captured_and_replayed(ops, rows):
    """The four launches as a graph, replayed on new inputs, with eager work between the replays."""
    gen = seeded(rows)
    width, inner = 512, 1536
    weights = [ops.quantize_rows(normal(gen, *s) / 20) for s in ((inner, width), (inner, width), (width, inner))]
    gain = 1 + 0.1 * normal(gen, width)
    x, add = normal(gen, rows, width), normal(gen, rows, width).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        feed_forward(ops, x.clone(), add, gain, *weights)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n, hidden, out = feed_forward(ops, x, add, gain, *weights)
    for turn in range(4):
        fresh, fresh_add = normal(gen, rows, width), normal(gen, rows, width).bfloat16()
        x.copy_(fresh)
        add.copy_(fresh_add)
        graph.replay()
        want = feed_forward(ops, fresh, fresh_add, gain, *weights)
        torch.cuda.synchronize()
        assert torch.equal(n.q, want[0].q) and torch.equal(hidden, want[1]) and torch.equal(out, want[2])


def test_two_graphs_and_two_streams_share_nothing(ops):
    """Products that cut K, in two graphs replayed at once on two streams beside an eager one on a third."""
    gen = seeded(4)
    a, w, _ = operands(ops, gen, 40, 256, 8192)
    b, v, _ = operands(ops, gen, 300, 320, 8192)
    want_a, want_b = ops.gemm_int8(a, w, out_dtype=torch.float32).clone(), ops.gemm_int8(b, v, out_dtype=torch.float32).clone()
    streams = [torch.cuda.Stream() for _ in range(3)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for s, (p, q) in zip(streams, ((a, w), (b, v))):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(ops.gemm_int8(p, q, out_dtype=torch.float32))
        graphs.append(g)
    for turn in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = [ops.gemm_int8(a, w, out_dtype=torch.float32), ops.gemm_int8(b, v, out_dtype=torch.float32)]
        torch.cuda.synchronize()
        for got, want in zip(outs + eager, (want_a, want_b) * 2):
            assert torch.equal(got, want)
