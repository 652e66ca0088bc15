"""Decode attention over the 4-bit cache where scores, keys and values differ by many powers of two within one sequence,
against the softmax average in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

from tests import _q4

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


def _i32(values) -> "torch.Tensor":
    return torch.as_tensor(np.asarray(values, np.int32), device="cuda")


def _bf16(x: np.ndarray) -> "torch.Tensor":
    return torch.from_numpy(np.asarray(x, np.float32)).cuda().to(torch.bfloat16)


def _cached(keys: np.ndarray, values: np.ndarray):
    """A cache of one sequence and key head with these rows [positions, head], and what it holds, in 64 bits: keys,
    values, and the scale and low of each row's key and value groups [positions, groups]."""
    from tempo_compiler_b200 import ops
    n, head = keys.shape
    rows = torch.cat([_bf16(keys), _bf16(values)], 1)
    cache = ops.kv_cache_q4(1, 1, n, head)
    ops.kv_store_q4(rows, cache, _i32(np.zeros(n)), _i32(np.arange(n)))
    held = []
    for part in (rows[:, :head], rows[:, head:]):
        codes, scale, low = _q4.quantise(part.double().cpu().numpy().reshape(n, -1, 64))
        held.append(((codes * scale + low).reshape(n, head), scale[..., 0], low[..., 0]))
    return cache, held


def _check(q: "torch.Tensor", held, got: "torch.Tensor") -> None:
    """The bound of an output of 64 dimensions with the values' widest range R = 15 scale and greatest |low| L in those 64
    dimensions. The output's own rounding is 2^-8 of it. Rounding each weight to FP16 moves the average by at most 2^-11
    of R. A score is a sum over the groups of 64, each of scale x code and low against the query, in FP32 and with the
    query's dimensions rounded at 2^-25 of the greatest of its group: it is off by at most (66 2^-23) sum |q| (15 scale +
    |low|) over the groups, and twice that, times R, moves the average. The sums over the positions are off by n 2^-23,
    and the exponentials and powers of two by 2^-20, of R + L."""
    (keys, k_scale, k_low), (values, v_scale, v_low) = held
    n, head = keys.shape
    q = q.double().cpu().numpy().reshape(-1, head)
    got = got.double().cpu().numpy().reshape(q.shape)
    assert np.isfinite(got).all()
    score = q @ keys.T
    p = np.exp(score - score.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    want = p @ values
    spread = (np.abs(q).reshape(len(q), -1, 64).sum(2) @ (15 * k_scale + np.abs(k_low)).T).max(1)[:, None]
    wide = np.repeat(15 * v_scale.max(0), 64)
    size = wide + np.repeat(np.abs(v_low).max(0), 64)
    bound = (2.0 ** -8 * np.abs(want) + wide * (2.0 ** -11 + 2 * 66 * 2.0 ** -23 * spread) +
             size * (n * 2.0 ** -23 + 2.0 ** -20) + 1e-37)
    worst = np.max(np.abs(got - want) / bound)
    assert worst <= 1.0, f"{worst:.3f} of the bound"


def _attend(q: "torch.Tensor", cache, n: int, heads: int, copies: int) -> "torch.Tensor":
    """The attention of `heads` equal rows of queries over `copies` copies of a sequence (few: clusters or the workspace,
    many: a CTA each), which all give the same."""
    from tempo_compiler_b200 import ops
    out = ops.decode_attention_q4(q.reshape(1, -1).repeat(copies, 1), cache.repeat(copies, 1, 1, 1), _i32([n] * copies),
                                  heads=heads)
    if copies > 1:
        assert torch.equal(out, out[:1].expand_as(out))
    return out[0]


SPLITS = [(40, 1), (70, 500), (300, 1), (300, 40), (300, 200), (3000, 1), (3000, 3), (9000, 1)]


@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("n,copies", SPLITS)
@pytest.mark.parametrize("small", [0.0, 1e-20])
@pytest.mark.parametrize("large", [1e12, 1e20, 1e29])
@pytest.mark.parametrize("small_first", [True, False])
def test_runs_of_zero_values_beside_large_ones(head: int, n: int, copies: int, small: float, large: float,
                                               small_first: bool) -> None:
    """Whole runs of positions, of a warp, of a CTA, with value rows of zeros or next to nothing: they keep their share of
    the softmax however large the values of the others are."""
    rng = np.random.default_rng(n + copies)
    keys, values = rng.standard_normal((2, n, head))
    near = np.arange(n) < 3 * n // 4
    values *= np.where(near if small_first else ~near, small, large)[:, None]
    cache, held = _cached(keys, values)
    q = _bf16(rng.standard_normal((4, head)) * 0.5 / head ** 0.5)
    q[0] = 0.0
    for heads in (1, 4):
        _check(q[:heads], held, _attend(q[:heads], cache, n, heads, copies))


@pytest.mark.parametrize("n,copies", SPLITS)
@pytest.mark.parametrize("ratio", [1e-3, 1e-5, 1e-7, 1e-10, 1e-20, 0.0])
@pytest.mark.parametrize("smaller", [0, 1])
def test_halves_of_a_value_row_of_different_size(n: int, copies: int, ratio: float, smaller: int) -> None:
    """Each 64 of a head's 128 dimensions are as exact as they would be alone."""
    rng = np.random.default_rng(n + copies)
    keys, values = rng.standard_normal((2, n, 128))
    values[:, 64 * smaller:64 * smaller + 64] *= ratio
    cache, held = _cached(keys, values)
    q = _bf16(rng.standard_normal((4, 128)) * 0.1)
    for heads in (1, 4):
        _check(q[:heads], held, _attend(q[:heads], cache, n, heads, copies))


@pytest.mark.parametrize("n,copies", SPLITS)
@pytest.mark.parametrize("ratio", [1e-3, 1e-6, 1e-8, 1e-12, 1e-25])
@pytest.mark.parametrize("smaller", [0, 1])
def test_halves_of_a_query_of_different_size(n: int, copies: int, ratio: float, smaller: int) -> None:
    """A half of the query that is far smaller than the other decides the scores all the same where its keys are as much
    larger than the others'."""
    rng = np.random.default_rng(n + copies)
    keys, values = rng.standard_normal((2, n, 128))
    small, large = slice(64 * smaller, 64 * smaller + 64), slice(64 - 64 * smaller, 128 - 64 * smaller)
    keys[:, small] /= ratio
    q = rng.standard_normal((4, 128)) * 0.2
    q[:, small] *= ratio
    keys[:, large] *= 0.25
    cache, held = _cached(keys, values)
    q = _bf16(q)
    for heads in (1, 4):
        _check(q[:heads], held, _attend(q[:heads], cache, n, heads, copies))


def test_a_long_tail_of_small_weights_counts() -> None:
    """A million positions of weight 2^-25.5 beside a few of weight 1: together they are 0.5 % of the average."""
    from tempo_compiler_b200 import ops
    n, heads, run = 1 << 20, 4096, 1 << 18   # so many queries that each four warps read all of it, a run to a warp
    first, other = np.zeros((2, 128), np.float32)
    even = np.arange(64) % 2 == 0
    first[64:], other[64:] = np.where(even, 0, 15), np.where(even, 15, 0)
    other[:64] = -0.55078125                 # (BF16 holds it)
    rows = _bf16(np.stack([first, other]))[(torch.arange(n, device="cuda") % run != 0).long()]
    cache = ops.kv_cache_q4(1, 1, n)
    ops.kv_store_q4(rows, cache, _i32(np.zeros(n)), torch.arange(n, dtype=torch.int32, device="cuda"))
    q = torch.full((1, heads * 64), 0.5, dtype=torch.bfloat16, device="cuda")
    got = ops.decode_attention_q4(q, cache, _i32([n]), heads=heads).double().cpu().numpy().reshape(heads, 64)
    ones = n // run
    tail = (n - ones) * np.exp(-0.55078125 * 32)
    want = np.where(even, 15 * tail, 15 * ones) / (ones + tail)
    # as above, with exact products: the output's rounding, 2^-11 of the tail's share and of the others' for the weights'
    # (they move the average by what they move apart), a running sum of run / 32 weights a lane, of 2^-24 each
    share = tail / (ones + tail)
    bound = 2.0 ** -8 * want + 15 * (2 * 2.0 ** -11 * share + share * (run / 32 * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -20)
    assert (np.abs(got - want) <= bound).all(), np.max(np.abs(got - want) / bound)
