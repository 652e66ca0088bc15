"""FP32 products wide enough for the CTA-pair kernel (at least 296 tiles of 256 x 256 on 148 SMs), against 64 bits, and
products with a matrix that the call before wrote."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from tempo_compiler_b200 import lib
    lib.load()
    yield
    from tempo_compiler_b200 import ops
    torch.cuda.synchronize()
    assert ops.watchdog() == 0


@pytest.mark.parametrize("m,n,k", [(300, 38001, 200), (257, 40003, 8), (2047, 9473, 768), (1, 75777, 72), (513, 25603, 72),
                                   (1024, 18945, 136), (384, 37889, 1024)])
def test_wide_products_match_64_bits(m: int, n: int, k: int) -> None:
    """Within the FP32 accumulation of k exact products, k 2^-23 sum |a| |w|; remainders of rows, columns and depth; a
    buffer's padding columns and the rows behind the last stay."""
    from tempo_compiler_b200 import ops
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert -(-m // 256) * -(-n // 256) >= 4 * (sms // 2), "the shape no longer reaches the pair kernel"
    rng = np.random.default_rng(m + n)
    a = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).cuda().to(torch.bfloat16)
    w = torch.from_numpy((0.1 * rng.standard_normal((n, k))).astype(np.float32)).cuda().to(torch.bfloat16)
    buffer = torch.full((m + 3, (n + 7) // 8 * 8 + 8), 5.0, device="cuda")
    got = ops.gemm_f32(a, w, out=buffer[:m, :n])
    want = a.double() @ w.double().T
    bound = k * 2.0 ** -23 * (a.double().abs() @ w.double().abs().T)
    assert ((got.double() - want).abs() <= bound).all()
    assert (buffer[:m, n:] == 5.0).all() and (buffer[m:] == 5.0).all()
    assert torch.equal(ops.gemm_f32(a, w), got)


@pytest.mark.parametrize("m,n,k", [(5, 1000, 768), (64, 4096, 512), (200, 2000, 64), (300, 38001, 200)])
def test_both_operands_of_the_call_before(m: int, n: int, k: int) -> None:
    """Operands that the library's own calls write right before, as attention scores take them, eagerly and in a graph."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(k)

    def matrix(rows: int, columns: int) -> "torch.Tensor":
        return torch.from_numpy((0.1 * rng.standard_normal((rows, columns))).astype(np.float32)).cuda().to(torch.bfloat16)

    x, y, weights = matrix(m, 256), matrix(n, 256), matrix(k, 256)
    a, w = ops.gemm(x, weights), ops.gemm(y, weights)
    torch.cuda.synchronize()
    want = ops.gemm_f32(a, w)
    torch.cuda.synchronize()
    outs = []

    def chain() -> None:
        for swap in range(6):
            for t in (a, w):
                t.fill_(3.0)
            first, second = ((x, a), (y, w)) if swap % 2 else ((y, w), (x, a))
            ops.gemm(first[0], weights, out=first[1])
            ops.gemm(second[0], weights, out=second[1])
            outs.append(ops.gemm_f32(a, w))

    chain()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    graph.replay()
    torch.cuda.synchronize()
    assert len(outs) == 12 and all(torch.equal(out, want) for out in outs)
