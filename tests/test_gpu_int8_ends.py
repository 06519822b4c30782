"""The operators on rows of 8-bit integers at the ends of what they take."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


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
