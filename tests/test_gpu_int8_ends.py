"""The operators on rows of 8-bit integers at the ends of what they take."""
import math

import pytest
import torch

import int8_oracle as oracle
from int8_oracle import U

pytestmark = pytest.mark.gpu

DEV = "cuda"
NORM_SCALE, NORM_ENTRY = 5, 6  # fp32 roundings of a norm's scale and of an entry against its row's largest


@pytest.fixture(scope="module")
def ops():
    from jllm_serve_amd.kernels import ops
    ops.library()
    return ops


@pytest.fixture(autouse=True)
def memory():
    yield
    torch.cuda.empty_cache()


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEV)


def seeded(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def repeated(rows, n):
    """``n`` rows, these ones again and again (copied: an index of 2^26 rows and more is beyond torch's own launches)."""
    out = torch.empty((n, *rows.shape[1:]), dtype=rows.dtype, device=DEV)
    whole = n - n % rows.shape[0]
    out[:whole].view(-1, *rows.shape)[:] = rows
    out[whole:] = rows[:n - whole]
    return out


def same(got, rows):
    """Whether ``got`` is these rows again and again."""
    period, step = rows.shape[0], rows.shape[0] * max(1, (1 << 24) // rows.shape[0])
    want = rows.repeat(step // period, *(1,) * (rows.dim() - 1))
    return all(torch.equal(got[at:at + step], want[:min(step, got.shape[0] - at)]) for at in range(0, got.shape[0], step))


# ------------------------------------------------------------------------------------------------ more than one launch takes: 2^32 threads


@pytest.mark.parametrize("rows,width", [((1 << 24) + 300, 3), ((1 << 26) + 300, 8)])
def test_rows_beyond_one_launch(ops, rows, width):
    """A row is a workgroup of 256 threads (of a width below 8) or of 64."""
    gen = seeded(width)
    few, add, gain = normal(gen, 1000, width), normal(gen, 1000, width).bfloat16(), normal(gen, width)
    want = ops.quantize_rows(few.bfloat16())
    got = ops.quantize_rows(repeated(few.bfloat16(), rows))
    assert same(got.q, want.q) and same(got.scale, want.scale)
    del got
    total = few.clone()
    want = ops.rmsnorm_int8(total, gain, 1e-6, add=add)
    x = repeated(few, rows)
    got = ops.rmsnorm_int8(x, gain, 1e-6, add=repeated(add, rows))
    assert same(got.q, want.q) and same(got.scale, want.scale) and same(x, total)


def test_values_beyond_one_launch(ops):
    """More than 2^32 entries read back one a thread: rows of fewer than eight."""
    rows, width = 620_000_000, 7
    few = ops.quantize_rows(normal(seeded(7), 1000, width))
    got = ops.Int8Rows(repeated(few.q, rows), repeated(few.scale, rows)).tensor(torch.bfloat16)
    assert same(got, few.tensor(torch.bfloat16))


@pytest.mark.parametrize("K", [64, 128, 50, 200])
def test_products_of_more_rows_than_a_grid_has(ops, K):
    """Tiles of 64 rows, of which a grid takes 65,535 above each other; K for the fast kernels and for the general one."""
    gen = seeded(K)
    M, N = 5_000_000, 16
    a = ops.quantize_rows(normal(gen, 1000, K))
    many = ops.Int8Rows(repeated(a.q, M), repeated(a.scale, M))
    w, w2 = (ops.quantize_rows(normal(gen, N, K) / math.sqrt(K)) for _ in range(2))
    bias, base = normal(gen, N), normal(gen, 1000, N)
    assert same(ops.gemm_int8(many, w, bias=bias), ops.gemm_int8(a, w, bias=bias))
    assert same(ops.gemm_int8(many, w, w2=w2, epilogue=ops.EPI_GATED), ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED))
    out = repeated(base, M)
    assert ops.gemm_int8(many, w, out=out, epilogue=ops.EPI_ADD) is out
    assert same(out, ops.gemm_int8(a, w, out=base.clone(), epilogue=ops.EPI_ADD))


@pytest.mark.parametrize("N,K", [((1 << 27) + 700, 16), ((1 << 30) + 64, 1)])
def test_products_of_more_outputs_than_a_grid_has(ops, N, K):
    gen = seeded(K)
    w = ops.quantize_rows(normal(gen, 1000, K))
    many = ops.Int8Rows(repeated(w.q, N), repeated(w.scale, N))
    a, bias = ops.quantize_rows(normal(gen, 1, K)), normal(gen, 1000)
    got = ops.gemm_int8(a, many, bias=repeated(bias, N))
    assert same(got[0], ops.gemm_int8(a, w, bias=bias)[0])


# ------------------------------------------------------------------------------------------------ values at the ends of fp32


@pytest.mark.parametrize("width", [5, 40, 1031, 5120, 33000])
@pytest.mark.parametrize("added", [False, True])
def test_norm_at_the_ends_of_fp32(ops, width, added):
    """Rows near fp32's largest, whose inverse root mean square lies below its normal numbers; with an eps of zero rows below them, whose
    inverse is beyond its largest, and rows of zeros."""
    gen = seeded(width)
    tens = torch.tensor([3e38, 1e38, 1e30, 1.0, 1e-30, 1e-38, 1e-42, 0.0], dtype=torch.float64)
    x = (torch.rand(8, width, generator=gen, device=DEV).double().cpu() * 1.8 - 0.9).clamp(-0.9, 0.9)
    x[:, width // 2] = 0.95
    x = (x * tens[:, None]).float().to(DEV)
    gain = 1 + 0.1 * normal(gen, width)
    add = x * 0.0625 if added else None
    h, _ = oracle.norm(x[:7], gain, 0.0, None if add is None else add[:7])
    y = oracle.norm(h, gain, 0.0)[1]
    got = ops.rmsnorm_int8(x, gain, 0.0, add=add, out=torch.empty_like(x) if added else None)
    oracle.check_rows(got.q[:7], got.scale[:7], y, NORM_ENTRY, NORM_SCALE)
    assert float(got.scale[7]) == 0 and not got.q[7].any()


KERNELS = [("", 0, 1)] + [(kernel, size, parts) for kernel, size in (("jllm_gemm_int8_stream", 24), ("jllm_gemm_int8_tiled", 64064), ("jllm_gemm_int8_tiled", 128128),
                                                                     ("jllm_gemm_int8_large", 256256)) for parts in (1, 3)]


@pytest.mark.parametrize("kernel,size,parts", KERNELS)
@pytest.mark.parametrize("N", [256, 203])
def test_products_of_rows_near_the_largest(ops, monkeypatch, kernel, size, parts, N):
    """Rows whose scale times the sum is beyond fp32, which the channel's scale brings back; the rows beside them keep their bits."""
    gen = seeded(N)
    M, K = 64 if kernel.endswith("stream") else 150, 1040
    x = normal(gen, M, K).clamp(-4, 4)
    far = torch.arange(M, device=DEV) % 3 == 1
    x[far] *= torch.tensor([8e37, 1e35, 1e30], device=DEV).repeat(M)[:int(far.sum()), None]
    a = ops.quantize_rows(x)
    w = ops.quantize_rows(normal(gen, N, K) * 1e-12)
    tiny, fine = ops.quantize_rows(normal(gen, N, K) * 1e-40), ops.quantize_rows(normal(gen, N, K))
    bias, base = normal(gen, N), normal(gen, M, N)
    monkeypatch.setattr(ops, "_int8_plans", lambda *args: ((0.0, kernel, size, parts),) if kernel else ())
    for weight in (w, tiny):
        y, tol = oracle.product(a, weight, bias)
        got = ops.gemm_int8(a, weight, bias=bias, out_dtype=torch.float32).double().cpu()
        assert torch.isfinite(got).all() and ((got - y).abs() <= tol).all()
        y, tol = oracle.product(a, weight, None, base)
        got = ops.gemm_int8(a, weight, out=base.clone(), epilogue=ops.EPI_ADD).double().cpu()
        assert torch.isfinite(got).all() and ((got - y).abs() <= tol).all()
    # gated: the row that is brought back into range, times a value that keeps it there (|z| to 1e30: the gate is 0 or z)
    z, u = oracle.sums(a, w), oracle.sums(a, tiny)
    y = oracle.gate("silu", z, u)
    some = (z.abs() > 1e3) & (y.abs() < 1e38)
    assert int(some.sum()) > N
    got = ops.gemm_int8(a, w, w2=tiny, epilogue=ops.EPI_GATED, out_dtype=torch.float32).double().cpu()
    assert ((got - y).abs() <= y.abs() * 16 * U + 1e-30)[some].all()
    # and the others
    near = ~far
    alone = ops.Int8Rows(a.q[near], a.scale[near])
    whole = ops.gemm_int8(a, fine, bias=bias)
    assert torch.equal(whole[near], ops.gemm_int8(alone, fine, bias=bias))


@pytest.mark.parametrize("kernel,size,parts", KERNELS)
def test_scales_below_zero(ops, monkeypatch, kernel, size, parts):
    """Rows at hand may have any scale: -s stands for the row of s with its sign turned, near fp32's largest too."""
    gen = seeded(3)
    M, N, K = 64 if kernel.endswith("stream") else 150, 203, 1040
    a, w = ops.quantize_rows(normal(gen, M, K).clamp(-4, 4) * 8e37), ops.quantize_rows(normal(gen, N, K) * 1e-12)
    monkeypatch.setattr(ops, "_int8_plans", lambda *args: ((0.0, kernel, size, parts),) if kernel else ())
    want = ops.gemm_int8(a, w, out_dtype=torch.float32)
    assert torch.isfinite(want).all()
    assert torch.equal(ops.gemm_int8(ops.Int8Rows(a.q, -a.scale), w, out_dtype=torch.float32), -want)


# ------------------------------------------------------------------------------------------------ gates in fp32


@pytest.mark.parametrize("gate,limit", [("silu", 0.0), ("swish_clamped", 60.0), ("gelu_tanh", 0.0)])
@pytest.mark.parametrize("M,N,K", [(3, 50, 70), (40, 256, 512), (64, 203, 640), (100, 256, 512), (130, 272, 2064), (300, 272, 528)])
def test_gates_in_fp32(ops, gate, limit, M, N, K):
    """A gated output in fp32 is as good as its two sums in fp32 allow: against the gate in 64 bits of those sums as they are rounded, whatever
    their size.

    2^x one unit (two halves), what its argument's rounding left one product with one rounding of its factor (3), 1 + that (1), the
    reciprocal one unit (2), two products (2), (u + 1) (1): 11 halves of a step, where an argument rounded by itself costs |z| of them. gelu's argument
    has 7 roundings of its own, times 2 |inner|. The reciprocal of more than 2^126 may be zero: what is lost lies below 128 * 2^-126 times |u|."""
    gen = seeded(M + N)
    a = ops.quantize_rows(normal(gen, M, K))
    w, w2 = (ops.quantize_rows(normal(gen, N, K) * (25 if gate != "gelu_tanh" else 3) / math.sqrt(K)) for _ in range(2))

    def sums(weight):  # as the kernels round them
        s = (a.q.cpu().double() @ weight.q.cpu().double().t()).float()
        return ((s * a.scale.cpu()[:, None]) * weight.scale.cpu()[None, :]).double()

    z, u = sums(w), sums(w2)
    assert float(z.abs().max()) > (60 if gate != "gelu_tanh" else 5)
    y = oracle.gate(gate, z, u, limit)
    tol = 11 * U * y.abs()
    if gate == "gelu_tanh":  # 0.5 (1 + tanh x) as the sigmoid of 2x: where it is small, the sum has no digits left in 64 bits either
        inner = 0.7978845608028654 * (z + 0.044715 * z ** 3)
        y = z * torch.sigmoid(2 * inner) * u
        tol = (11 + 14 * inner.abs()) * U * y.abs()
    tol = tol * 1.01 + 128 * 2.0 ** -126 * (u.abs() + 1)
    got = ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED, gate=ops.GATE_FUNCTIONS[gate], gate_limit=limit, out_dtype=torch.float32).double().cpu()
    off = (got - y).abs() - tol
    assert (off <= 0).all(), (float((got - y).abs().div(y.abs().clamp_min(1e-30)).max() / U), int((off > 0).sum()))
