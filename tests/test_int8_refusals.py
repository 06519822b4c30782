"""What the operators on rows of 8-bit integers refuse, and with which words, before anything is launched (no GPU)."""
import pytest
import torch

from jllm_serve_amd.kernels import ops


def rows(n=4, width=32):
    return ops.Int8Rows(torch.zeros((n, width), dtype=torch.int8), torch.ones(n))


def refused(words, call, *args, **kw):
    with pytest.raises(ops.KernelError) as e:
        call(*args, **kw)
    assert words in str(e.value), str(e.value)


def test_no_cpu_path():
    refused("GPU only", ops.quantize_rows, torch.zeros(3, 8))
    refused("GPU only", ops.rmsnorm_int8, torch.zeros(3, 8), torch.zeros(8), 1e-6)
    refused("GPU only", ops.gemm_int8, rows(), rows(6))
    refused("GPU only", rows().tensor, torch.float32)


def test_quantize_rows():
    refused("contiguous rows", ops.quantize_rows, torch.zeros(8))
    refused("contiguous rows", ops.quantize_rows, torch.zeros(8, 4).t())
    refused("float32 or bfloat16", ops.quantize_rows, torch.zeros(3, 8, dtype=torch.float16))
    refused("without entries", ops.quantize_rows, torch.zeros(3, 0))


def test_int8_rows():
    """What does not make 8-bit rows is refused where they are made."""
    q = torch.zeros((4, 8), dtype=torch.int8)
    refused("must be int8", ops.Int8Rows, q.view(torch.uint8), torch.ones(4))
    refused("one entry per row", ops.Int8Rows, q, torch.ones(3))
    refused("one entry per row", ops.Int8Rows, q, torch.ones(4, dtype=torch.float64))
    refused("one entry per row", ops.Int8Rows, q, torch.ones(4, 1))
    refused("contiguous fp32", ops.Int8Rows, q, torch.ones(8)[::2])
    refused("contiguous rows", ops.Int8Rows, torch.zeros((8, 4), dtype=torch.int8).t(), torch.ones(4))
    refused("contiguous rows", ops.Int8Rows, q[0], torch.ones(1))
    refused("float32 or bfloat16", rows().tensor, torch.float16)
    with pytest.raises(AttributeError):
        rows().q = q
    with pytest.raises(AttributeError):
        rows().scale = torch.ones(4)


def test_rmsnorm_int8():
    x, g = torch.zeros(3, 8), torch.ones(8)
    refused("fp32 rows", ops.rmsnorm_int8, x.bfloat16(), g, 1e-6)
    refused("contiguous rows", ops.rmsnorm_int8, torch.zeros(8, 3).t(), g, 1e-6)
    refused("no norm", ops.rmsnorm_int8, torch.zeros(3, 0), torch.ones(0), 1e-6)
    refused("gain has 7", ops.rmsnorm_int8, x, torch.ones(7), 1e-6)
    refused("float32 or bfloat16", ops.rmsnorm_int8, x, g.half(), 1e-6)
    refused("without rows to add", ops.rmsnorm_int8, x, g, 1e-6, out=torch.zeros(3, 8))
    refused("rows to add", ops.rmsnorm_int8, x, g, 1e-6, add=torch.zeros(2, 8))
    refused("float32 or bfloat16", ops.rmsnorm_int8, x, g, 1e-6, add=x.half())
    refused("fp32 tensor of x's shape", ops.rmsnorm_int8, x, g, 1e-6, add=x, out=x.bfloat16())
    refused("fp32 tensor of x's shape", ops.rmsnorm_int8, x, g, 1e-6, add=x, out=torch.zeros(3, 9))
    refused("rows of their own", ops.rmsnorm_int8, x, g, 1e-6, add=x, out=torch.zeros(1, 8).expand(3, 8))
    refused("rows of their own", ops.rmsnorm_int8, torch.zeros(1, 8).expand(3, 8), g, 1e-6, add=x)
    refused("rows of their own", ops.rmsnorm_int8, x, g, 1e-6, add=x, out=torch.zeros(30).as_strided((3, 8), (7, 1)))


def test_gemm_int8():
    a, w = rows(4), rows(6)
    refused("must be Int8Rows", ops.gemm_int8, a.q, w)
    refused("must be Int8Rows", ops.gemm_int8, a, w.q)
    refused("must be Int8Rows", ops.gemm_int8, a, w, w2=w.q, epilogue=ops.EPI_GATED)
    refused("input rows have 32", ops.gemm_int8, a, rows(6, 31))
    refused("rows of 0", ops.gemm_int8, rows(4, 0), rows(6, 0))
    refused("leave 32 bits", ops.gemm_int8, rows(1, 131072), rows(1, 131072))
    refused("exactly two weights", ops.gemm_int8, a, w, w2=w)
    refused("exactly two weights", ops.gemm_int8, a, w, epilogue=ops.EPI_GATED)
    refused("exactly two weights", ops.gemm_int8, a, w, epilogue=3)
    refused("agree in shape", ops.gemm_int8, a, w, w2=rows(5), epilogue=ops.EPI_GATED)
    refused("without the gated", ops.gemm_int8, a, w, gate=1)
    refused("without the gated", ops.gemm_int8, a, w, w2=w, epilogue=ops.EPI_GATED, gate=1 << 20)
    refused("bias has 5", ops.gemm_int8, a, w, bias=torch.zeros(5))
    refused("bias has 6", ops.gemm_int8, a, w, bias=torch.zeros(12)[::2])
    refused("float32 or bfloat16", ops.gemm_int8, a, w, bias=torch.zeros(6, dtype=torch.float16))
    refused("fp32 output", ops.gemm_int8, a, w, epilogue=ops.EPI_ADD)
    refused("fp32 output", ops.gemm_int8, a, w, out=torch.zeros(4, 6).bfloat16(), epilogue=ops.EPI_ADD)
    refused("expected (4, 6)", ops.gemm_int8, a, w, out=torch.zeros(4, 7))
    refused("asked for", ops.gemm_int8, a, w, out=torch.zeros(4, 6), out_dtype=torch.bfloat16)
    refused("rows of their own", ops.gemm_int8, a, w, out=torch.zeros(1, 6).expand(4, 6))
    refused("contiguous rows", ops.gemm_int8, a, w, out=torch.zeros(6, 4).t())
    refused("float32 or bfloat16", ops.gemm_int8, a, w, out_dtype=torch.float16)
    refused("float32 or bfloat16", ops.gemm_int8, a, w, out=torch.zeros(4, 6).half())


def test_a_single_row_may_have_any_stride():
    """A row alone has no distance to the next: it is not refused for the stride it happens to have."""
    assert ops._own_rows_of(torch.zeros(8, 1).t(), "row") == (1, 8, 8)
    refused("2^31", ops._rows_of, torch.empty_strided((2, 1), (1 << 31, 1), dtype=torch.int8, device="meta"), "rows")


@pytest.mark.parametrize("n, width", [(0, 5), (1, 1), (1, 16), (3, 7), (4, 8), (5, 13), (64, 129)])
def test_rows_and_scales_of_one_allocation(n, width):
    """What the kernels make: the scales and the rows, each on 16 bytes, neither over the other, both inside the allocation."""
    rows = ops.Int8Rows._new(n, width, torch.empty(0))
    assert rows.q.dtype is torch.int8 and rows.q.shape == (n, width) == rows.shape and rows.q.is_contiguous()
    assert rows.scale.dtype is torch.float32 and rows.scale.shape == (n,) and rows.scale.is_contiguous()
    if n:
        assert (rows.q.data_ptr(), rows.scale.data_ptr()) == rows._addresses()
        assert (rows.q.data_ptr() - rows.scale.data_ptr()) % 16 == 0
        rows.q.fill_(-7)
        rows.scale.copy_(torch.arange(n))
        assert (rows.q == -7).all() and (rows.scale == torch.arange(n)).all()
        storage = rows.scale.untyped_storage()
        assert rows.q.data_ptr() + n * width <= storage.data_ptr() + storage.nbytes()
