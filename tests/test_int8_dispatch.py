"""How products of 8-bit rows are launched: pieces and grids that a launch can have (no GPU)."""
import pytest
import torch

import recorded
from jllm_serve_amd.kernels import ops

MOST_THREADS, MOST_UP = 1 << 32, 65535  # of a grid: threads (fewer), workgroups above each other


def grid(kernel, size, M, N, gated, parts):
    """(workgroups beside each other, above each other, behind each other, threads of one) as the entry point launches them."""
    if kernel == "jllm_gemm_int8_stream":
        return -(-N // size), parts, 1, 256
    rows, columns = divmod(64064 if kernel == "jllm_gemm_int8" else size, 1000)
    return -(-N // (columns // (2 if gated else 1))), -(-M // rows), parts, 512 if rows >= 128 else 256


def fits(*launch):
    x, y, z, threads = grid(*launch)
    return y <= MOST_UP and z <= MOST_UP and x * y * z * threads < MOST_THREADS


@pytest.mark.parametrize("M", [1, 8, 64, 65, 4096, 70000, 1 << 20, 1 << 21])
@pytest.mark.parametrize("N", [1, 16, 200, 4096, 25600, 200000, 1 << 22, 1 << 26])
def test_every_plan_fits_its_launch(M, N):
    if M * N > ops.INT8_MOST_SUMS:
        M = ops.INT8_MOST_SUMS // N
    for K in (1, 16, 128, 144, 1024, 4096, 131071):
        for gated in (False, True):
            assert fits("jllm_gemm_int8", 0, M, N, gated, ops._int8_general(-(-M // 64), N, K, gated)[1]), (K, gated)
            for _, kernel, size, parts in ops._int8_plans(M, N, -(-K // 16) * 16 if K < 131071 else 131056, gated):
                assert fits(kernel, size, M, N, gated, parts), (K, gated, kernel, size, parts)


@pytest.mark.parametrize("M,N,K", [(5, 20, 64), (2_097_152, 16, 64), (2_097_153, 16, 64), (5_000_000, 16, 50), (9_000_000, 3, 128), (1, (1 << 26) + 1, 16),
                                   (3, 1 << 30, 1), (70, (1 << 27) + 5, 4), (1 << 20, 1 << 17, 32), (2_500_000, 70_000, 16)])
@pytest.mark.parametrize("kind", ["store", "add", "gated"])
def test_a_product_of_any_size_is_made_of_pieces_that_fit(monkeypatch, M, N, K, kind):
    """Every output once, with its row, its channels and its bias, in launches that a grid can have."""
    seen = recorded.record(monkeypatch)
    monkeypatch.setattr(ops, "_here", lambda *tensors: None)
    # (a tensor without memory lies at 0; here its place is where its part of the whole begins)
    monkeypatch.setattr(ops.Int8Rows, "_addresses", lambda rows: (16 * rows.q.storage_offset(), rows.scale.storage_offset()))
    rows = lambda n: ops.Int8Rows(recorded.tensor(n, K, dtype=torch.int8), recorded.tensor(n, dtype=torch.float32))
    a, w = rows(M), rows(N)
    out = recorded.tensor(M, N, dtype=torch.float32)
    kw = dict(store=dict(), add=dict(epilogue=ops.EPI_ADD), gated=dict(epilogue=ops.EPI_GATED, w2=rows(N), gate=1))[kind]
    assert ops.gemm_int8(a, w, bias=recorded.tensor(N), out=out, **kw) is out
    done = []
    for name, args in seen:
        if name == "jllm_int8_lay_out":
            continue
        m, n, k, epilogue = args[14:18]
        assert k in (K, -(-K // 16) * 16) and (args[13] == N or m == 1)
        assert epilogue == dict(store=0, add=1, gated=2 | 1 << 8)[kind]
        size, parts = (0, args[19]) if name == "jllm_gemm_int8" else args[19:21]
        assert fits(name, size, m, n, kind == "gated", parts)
        if not kind == "gated":
            assert args[8] is None
        else:
            assert args[8] == args[5]
        done.append((args[2], args[5], m, n))
    columns = sorted({(c, n) for _, c, _, n in done})
    assert [c for c, _ in columns] == [sum(n for _, n in columns[:i]) for i in range(len(columns))] and sum(n for _, n in columns) == N
    for c, n in columns:
        pieces = sorted((r, m) for r, at, m, _ in done if at == c)
        assert [r for r, _ in pieces] == [sum(m for _, m in pieces[:i]) for i in range(len(pieces))] and sum(m for _, m in pieces) == M
    assert len(done) == 1 or M > ops.INT8_MOST_ROWS or N > ops.INT8_MOST_OUTPUTS or M * N > ops.INT8_MOST_SUMS


@pytest.mark.parametrize("M,N,K,at", [(1, 64, 128, 0), (40, 96, 8192, 0), (40, 96, 8191, 0), (70, 64, 8192, 0), (70, 64, 128, 3), (600, 640, 2061, 0)])
def test_kept_launches_keep_their_operands(monkeypatch, M, N, K, at):
    """Every address that a kept launch was given lies in a tensor that is kept with it: operands, results, sums of a cut K, rows laid out anew."""
    recorded.record(monkeypatch)
    calls = []
    monkeypatch.setattr(ops, "_try", lambda name, *args: calls.append((name, args)) or True)
    monkeypatch.setattr(ops, "_call", lambda name, *args: calls.append((name, args)))
    monkeypatch.setattr(ops, "_here", lambda *tensors: None)
    with ops.kept_launches() as kept:
        x = torch.empty(M * K + at, dtype=torch.float32)[at:].view(M, K)
        a = ops.rmsnorm_int8(x, torch.empty(K), 1e-6, add=torch.empty((M, K)), out=torch.empty((M, K)))
        ops.rmsnorm_int8(x, torch.empty(K), 1e-6)
        w, w2 = (ops.Int8Rows(torch.empty(N * K + at, dtype=torch.int8)[at:].view(N, K), torch.empty(N)) for _ in range(2))
        ops.gemm_int8(a, w, bias=torch.empty(N))
        ops.gemm_int8(a, w, out=torch.empty((M, N)), epilogue=ops.EPI_ADD)
        ops.quantize_rows(ops.gemm_int8(a, w, w2=w2, epilogue=ops.EPI_GATED)).tensor(torch.float32)
    memory = [(t.untyped_storage().data_ptr(), t.untyped_storage().nbytes()) for t in kept.tensors]
    assert len(calls) >= 7
    for name, args in calls:
        types = ops._SIGS.get(name) or ops._OPTIONAL_SIGS[name]
        assert len(types) == len(args)
        for i, (kind, value) in enumerate(zip(types[:-1], args)):  # (the last is the stream)
            if kind is ops._P and value:
                assert any(start <= value < start + size for start, size in memory), (name, i)
