"""Log probabilities, entropies and alternatives of logits against the definition in 64 bits; the FP32 LM head before
them.

The bound on a log probability x - m - ln l: every term e^(x - m) of l carries 2^-21 of itself (the exponential and the
rounding of its argument, whose size the terms that matter keep below 2^5), a sum over `vocab` terms split over at
least 128 threads at most (vocab / 128 + 64) 2^-24, and the final differences 2^-22 of the result. The entropy's second
sum weighs the same errors with |x - m|, at most 2 + ln(vocab) times the first on average."""

from __future__ import annotations

import math

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


def _i32(values) -> "torch.Tensor":
    return torch.as_tensor(np.asarray(values, np.int32), device="cuda")


def _reference(logits: np.ndarray, ids: np.ndarray, top: int):
    """(logprob, entropy, top_logprob, top_ids) in 64 bits; rows without NaN or +infinity."""
    x = logits.astype(np.float64)
    rows, vocab = x.shape
    with np.errstate(divide="ignore", invalid="ignore"):
        m = x.max(1, keepdims=True)
        d = np.where(np.isneginf(m), -np.inf, x - np.where(np.isneginf(m), 0.0, m))
        e = np.exp(d)
        logs = d - np.log(e.sum(1, keepdims=True))
        logs[np.isneginf(m[:, 0])] = -np.inf
        p = np.where(np.isneginf(logs), 0.0, np.exp(logs))
        entropy = -(p * np.where(p > 0, logs, 0.0)).sum(1)
    inside = (ids >= 0) & (ids < vocab)
    logprob = np.where(inside, logs[np.arange(rows), np.where(inside, ids, 0)], 0.0)
    order = np.argsort(-x, axis=1, kind="stable")[:, :top]
    return logprob, entropy, np.take_along_axis(logs, order, 1), order


def _close(got, want: np.ndarray, vocab: int, weight: float = 1.0) -> None:
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    fine = np.isfinite(want)
    error = np.abs(got[fine] - want[fine])
    bound = weight * (2.0 ** -21 + (vocab / 128 + 64) * 2.0 ** -24) + 2.0 ** -22 * np.abs(want[fine])
    assert (error <= bound).all(), f"{np.max(error / bound):.3f} of the bound"


def _check(logits: "torch.Tensor", ids: np.ndarray, top: int, scores) -> None:
    vocab = logits.shape[1]
    logprob, entropy, best, order = _reference(logits.float().cpu().numpy(), ids, top)
    _close(scores.logprob, logprob, vocab)
    _close(scores.entropy, entropy, vocab, 2 + math.log(vocab))
    if top:
        np.testing.assert_array_equal(scores.top_ids.cpu().numpy(), order)
        _close(scores.top_logprob, best, vocab)


def _logits(rng, rows: int, vocab: int, dtype) -> "torch.Tensor":
    x = rng.standard_normal((rows, vocab)) * (1 + 4 * rng.random((rows, 1))) - 35
    return torch.from_numpy(x.astype(np.float32)).cuda().to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (2, 31, 31), (5, 33, 32), (1, 600, 20), (4, 1023, 5),
                                            (2, 4097, 32), (1, 50257, 20), (7, 50257, 5), (300, 50257, 1),
                                            (3, 152064, 32), (1, 1000003, 8), (17, 8192, 0)])
def test_scores_match_the_definition(dtype, rows: int, vocab: int, top: int) -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(rows * 7 + vocab)
    logits = _logits(rng, rows, vocab, dtype)
    ids = rng.integers(0, vocab, rows)
    ids[rows // 2] = int(logits[rows // 2].argmax())
    scores = ops.token_logprobs(logits, _i32(ids), top=top)
    _check(logits, ids, top, scores)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("stride,offset", [(50257, 1), (50260, 0), (50300, 3), (50264, 5)])
def test_rows_at_any_stride_and_alignment(dtype, stride: int, offset: int) -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(stride)
    rows, vocab = 6, 50251
    flat = torch.full((rows * stride + offset + 64,), 1e30, dtype=dtype, device="cuda")  # nothing of it may count
    logits = flat[offset:offset + rows * stride].view(rows, stride)[:, :vocab]
    logits.copy_(_logits(rng, rows, vocab, dtype))
    ids = rng.integers(0, vocab, rows)
    _check(logits, ids, 7, ops.token_logprobs(logits, _i32(ids), top=7))


def test_ties_go_to_the_lower_index() -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(3)
    vocab = 30011
    x = np.round(rng.standard_normal((6, vocab)) * 2).astype(np.float32)   # a handful of distinct values
    x[1] = 0.25                                                            # all equal
    x[2] = np.where(np.arange(vocab) % 2, 0.0, -0.0)                       # zeros of both signs are equal
    x[3] = np.arange(vocab) // 100                                         # rising steps: the last hundred tie
    x[4] = -(np.arange(vocab) // 100)                                      # falling steps
    logits = torch.from_numpy(x).cuda()
    ids = rng.integers(0, vocab, 6)
    for top in (1, 20, 32):
        _check(logits, ids, top, ops.token_logprobs(logits, _i32(ids), top=top))


@pytest.mark.parametrize("vocab", [50257, 200003])
def test_rows_in_order_and_against_it(vocab: int) -> None:
    """Rising logits, where every later one beats all before it, falling ones, and the best in the last places."""
    from tempo_compiler_b200 import ops
    x = np.zeros((4, vocab), np.float32)
    x[0] = np.arange(vocab) * 1e-3
    x[1] = x[0][::-1]
    x[2, -40:] = 5 + np.arange(40) % 7
    x[3, ::997] = 3
    ids = np.array([vocab - 1, 0, vocab - 1, 1])
    for rows in (slice(0, 4), slice(0, 1)):
        logits = torch.from_numpy(x[rows].copy()).cuda()
        _check(logits, ids[rows], 32, ops.token_logprobs(logits, _i32(ids[rows]), top=32))
    many = torch.from_numpy(x).cuda().repeat(80, 1)
    _check(many, np.tile(ids, 80), 20, ops.token_logprobs(many, _i32(np.tile(ids, 80)), top=20))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_logits(dtype) -> None:
    """Masks of -infinity and of the type's lowest value, rows with one token left, and a row with none."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(4)
    vocab, low = 20001, torch.finfo(dtype).min
    logits = _logits(rng, 8, vocab, dtype)
    keep = torch.from_numpy(rng.random((8, vocab)) < 1e-3).cuda()
    logits[0].masked_fill_(~keep[0], -math.inf)
    logits[1].masked_fill_(~keep[1], low)
    logits[2] = -math.inf
    logits[2, 77] = -3.0                      # one token left
    logits[3] = -math.inf                     # none
    logits[4] = low                           # every token at the lowest value: uniform
    logits[5, :vocab - 3] = -math.inf         # only the last three
    logits[6, 1:] = -math.inf                 # only the first
    logits[7, ::2] = -math.inf
    logits[7, 1::2] = low
    ids = np.array([int(keep[0].nonzero()[0]), 5, 77, 9, 100, vocab - 1, 1, 3])
    for top in (0, 5, 32):
        _check(logits, ids, top, ops.token_logprobs(logits, _i32(ids), top=top))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [3001, 50257])
@pytest.mark.parametrize("size", [1e6, 1e9, 1e10, 1e12, 1e20, 1e29, 1.5e38])
def test_logits_of_any_size(dtype, vocab: int, size: float) -> None:
    """Masks of any large negative value among ordinary logits, rows of nothing else, and rows of large positive logits."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(int(math.log2(size)))
    logits = _logits(rng, 8, vocab, dtype)
    logits[0, torch.from_numpy(rng.random(vocab) < 0.97).cuda()] = -size
    logits[1, :vocab // 2] = -size            # before the others
    logits[2, vocab // 2:] = -size            # behind them
    logits[3] = -size                         # uniform
    logits[4] = -size
    logits[4, 500] = -size * 0.75             # one token takes all
    logits[5, 77] = size
    logits[6] = size
    logits[6, ::2] = -size
    logits[7, ::3] = size
    logits[7, 1::3] = -math.inf
    ids = np.array([vocab - 1, 0, vocab - 1, 9, 500, 78, 1, 3])
    for top in (0, 5, 32):
        _check(logits, ids, top, ops.token_logprobs(logits, _i32(ids), top=top))
    many = logits.repeat(40, 1)               # a CTA to a row
    _check(many, np.tile(ids, 40), 5, ops.token_logprobs(many, _i32(np.tile(ids, 40)), top=5))


def test_nan_and_infinity() -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(5)
    logits = _logits(rng, 4, 9001, torch.float32)
    clean = ops.token_logprobs(logits, _i32([1, 2, 3, 4]), top=3)
    logits[1, 8000] = math.nan
    logits[2, 10] = math.inf
    scores = ops.token_logprobs(logits, _i32([1, 2, 3, 4]), top=3)
    for r in (1, 2):
        assert math.isnan(scores.logprob[r]) and math.isnan(scores.entropy[r]) and scores.top_logprob[r].isnan().all()
    assert scores.top_ids[1, 0] == 8000 and scores.top_ids[2, 0] == 10
    assert torch.equal(scores.top_ids[1, 1:], clean.top_ids[1, :2])
    for r in (0, 3):
        assert all(torch.equal(a[r], b[r]) for a, b in zip(scores, clean))


def test_rows_without_a_token_score_zero() -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(6)
    logits = _logits(rng, 5, 777, torch.float32)
    ids = np.array([-1, 776, 777, -2 ** 31, 2 ** 31 - 1])
    scores = ops.token_logprobs(logits, _i32(ids), top=2)
    _check(logits, ids, 2, scores)
    assert scores.logprob[[0, 2, 3, 4]].eq(0).all() and scores.logprob[1] < 0


def test_outputs_of_the_caller_and_a_replayed_graph() -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(7)
    rows, vocab, top = 9, 50257, 4
    logits = _logits(rng, rows, vocab, torch.float32)
    ids = _i32(rng.integers(0, vocab, rows))
    buffers = [torch.full((rows + 2,), 9.0, device="cuda") for _ in range(2)]
    out = ops.TokenScores(buffers[0][1:-1], buffers[1][1:-1],
                          torch.empty((rows, top), device="cuda"),
                          torch.empty((rows, top), dtype=torch.int32, device="cuda"))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert ops.token_logprobs(logits, ids, top=top, out=out) is out
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.token_logprobs(logits, ids, top=top, out=out)
    for _ in range(2):
        logits.copy_(_logits(rng, rows, vocab, torch.float32))
        ids.copy_(_i32(rng.integers(0, vocab, rows)))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        stream.synchronize()
        _check(logits, ids.cpu().numpy(), top, out)
        eager = ops.token_logprobs(logits, ids, top=top)
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
    for b in buffers:
        assert b[0] == 9.0 and b[-1] == 9.0


def test_slots_take_the_results() -> None:
    """Each row's results in the block its slot names, and nothing elsewhere, over one row to many."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(10)
    for rows in (1, 5, 200):
        vocab, top, blocks = 9001, 3, 4
        logits = _logits(rng, rows, vocab, torch.float32)
        ids = _i32(rng.integers(0, vocab, rows))
        want = ops.token_logprobs(logits, ids, top=top)
        out = ops.TokenScores(torch.full((blocks, rows), 7.0, device="cuda"), torch.full((blocks, rows), 7.0, device="cuda"),
                              torch.full((blocks, rows, top), 7.0, device="cuda"),
                              torch.full((blocks, rows, top), 7, dtype=torch.int32, device="cuda"))
        slots = rng.integers(8, 14, rows)  # less 10: blocks -2 .. 3
        ops.token_logprobs(logits, ids, top=top, out=out, slots=_i32(slots), slot_offset=-10)
        for r, slot in enumerate(slots - 10):
            for got, value in zip(out, want):
                for b in range(blocks):
                    assert torch.equal(got[b, r], value[r]) if b == slot else (got[b, r] == 7).all()


def test_offsets_past_32_bits() -> None:
    """Rows 2^31 elements into a matrix, and a row stride that makes byte offsets pass 2^32."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(8)
    flat = torch.zeros((3 << 30) + 4096, dtype=torch.bfloat16, device="cuda")
    logits = torch.as_strided(flat, (3, 4000), (3 << 29, 1))
    logits.copy_(_logits(rng, 3, 4000, torch.bfloat16))
    ids = rng.integers(0, 4000, 3)
    _check(logits, ids, 5, ops.token_logprobs(logits, _i32(ids), top=5))


# ---- the FP32 LM head -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("m,n,k", [(1, 50257, 768), (3, 257, 64), (8, 1000, 768), (9, 50257, 768), (64, 513, 200),
                                   (129, 255, 8), (300, 2049, 768), (700, 8191, 1024)])
def test_gemm_f32_matches_64_bits(m: int, n: int, k: int) -> None:
    """Within the FP32 accumulation of k exact products, k 2^-23 sum |a| |w|; a buffer's padding columns stay."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(m + n)
    a = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).cuda().to(torch.bfloat16)
    w = torch.from_numpy((0.1 * rng.standard_normal((n, k))).astype(np.float32)).cuda().to(torch.bfloat16)
    stride = (n + 7) // 8 * 8 + 8
    buffer = torch.full((m, stride), 5.0, device="cuda")
    got = ops.gemm_f32(a, w, out=buffer[:, :n])
    want = a.double() @ w.double().T
    bound = k * 2.0 ** -23 * (a.double().abs() @ w.double().abs().T)
    assert ((got.double() - want).abs() <= bound).all()
    assert (buffer[:, n:] == 5.0).all()
    assert torch.equal(ops.gemm_f32(a, w), got)


def test_head_and_scores_together() -> None:
    """Hidden rows to log probabilities: the alternatives are the FP32 logits' own order, the greedy pick the argmax."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(9)
    rows, vocab, width = 70, 50257, 768
    hidden = torch.from_numpy(rng.standard_normal((rows, width)).astype(np.float32)).cuda().to(torch.bfloat16)
    table = torch.from_numpy((0.1 * rng.standard_normal((vocab, width))).astype(np.float32)).cuda().to(torch.bfloat16)
    logits = ops.gemm_f32(hidden, table)
    ids = rng.integers(0, vocab, rows)
    scores = ops.token_logprobs(logits, _i32(ids), top=5)
    _check(logits, ids, 5, scores)
    tiles = (vocab + 255) // 256
    part_val = torch.empty((rows, tiles), device="cuda")
    part_idx = torch.empty((rows, tiles), dtype=torch.int32, device="cuda")
    picked = torch.empty(rows, dtype=torch.int32, device="cuda")
    ops.gemm_argmax(hidden, table, part_val, part_idx)
    ops.argmax_finish(part_val, part_idx, picked)
    assert torch.equal(picked, scores.top_ids[:, 0])


def test_the_wrappers_refuse_what_does_not_fit() -> None:
    from tempo_compiler_b200 import ops
    logits, ids = torch.zeros((3, 40), device="cuda"), _i32([0, 1, 2])
    good = ops.token_logprobs(logits, ids, top=2)
    wide = ops.TokenScores(*(t[None].repeat(2, *[1] * t.dim()) for t in good))
    a, w = (torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cases = [
        (lambda: ops.token_logprobs(logits.half(), ids), "float32"),
        (lambda: ops.token_logprobs(logits, ids[:2]), "as many ids"),
        (lambda: ops.token_logprobs(logits, ids.long()), "int32"),
        (lambda: ops.token_logprobs(logits, ids, top=33), "top"),
        (lambda: ops.token_logprobs(logits, ids, top=-1), "top"),
        (lambda: ops.token_logprobs(logits[:, :5], ids, top=6), "top"),
        (lambda: ops.token_logprobs(logits.T, ids), "contiguous rows|as many"),
        (lambda: ops.token_logprobs(logits[:1].expand(3, -1), ids), "overlap"),
        (lambda: ops.token_logprobs(logits[:0], ids[:0]), "rows 0"),
        (lambda: ops.token_logprobs(logits, ids, top=3, out=good), "must be"),
        (lambda: ops.token_logprobs(logits, ids, top=2, out=good._replace(top_ids=None)), "needed"),
        (lambda: ops.token_logprobs(logits, ids, top=2, out=good._replace(entropy=good.entropy.double())), "float32"),
        (lambda: ops.token_logprobs(logits, ids, slots=ids), "outputs"),
        (lambda: ops.token_logprobs(logits, ids, top=2, out=good, slots=ids), "must be"),
        (lambda: ops.token_logprobs(logits, ids, top=2, out=wide, slots=ids[:2]), "as many slots"),
        (lambda: ops.gemm_f32(a, w.float()), "bfloat16"),
        (lambda: ops.gemm_f32(a, w[:, :32].contiguous()), "inner"),
        (lambda: ops.gemm_f32(a, w, out=torch.zeros((4, 5), device="cuda")), "out must be"),
        (lambda: ops.gemm_f32(a, w, out=torch.zeros((4, 5), device="cuda")[:, :4]), "row stride"),
        (lambda: ops.gemm_f32(a, w, out=torch.zeros((4, 12), device="cuda")[:, 1:5]), "aligned"),
    ]
    for call, words in cases:
        with pytest.raises(ValueError, match=words):
            call()
