"""The 4-bit key/value cache on a B200: stored rows read back as the definition says, bit for bit; decode attention over
the cache against the softmax average in 64 bits (tests/_q4.py derives its bound); the entry points' refusals are in
tests/test_q4_refusals_cpu.py."""

from __future__ import annotations

import math

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


def _rows(rng, *shape) -> "torch.Tensor":
    x = rng.standard_normal(shape) * np.exp(0.5 * rng.standard_normal((*shape[:-1], 1)))
    return torch.from_numpy(x.astype(np.float32)).cuda().to(torch.bfloat16)


def _expected(qkv: "torch.Tensor", kv_heads: int, head: int) -> np.ndarray:
    """The BF16 rows a store and a load of qkv's key and value columns give, as float32."""
    kv = qkv[:, qkv.shape[1] - 2 * kv_heads * head:].float().cpu().numpy()
    value = _q4.dequantise(kv.reshape(kv.shape[0], -1, 64)).reshape(kv.shape)
    return torch.from_numpy(value).to(torch.float32).to(torch.bfloat16).float().numpy()


def _fill(cache, rng, heads: int = 0):
    """Random rows at every place of a cache."""
    from tempo_compiler_b200 import ops
    seqs, kv_heads, tiles, size = cache.shape
    head, capacity = size // 1152 * 64, tiles * 16
    rows = _rows(rng, seqs * capacity, 2 * kv_heads, head).reshape(seqs * capacity, -1)
    seq = _i32(np.repeat(np.arange(seqs), capacity))
    ops.kv_store_q4(rows, cache, seq, _i32(np.tile(np.arange(capacity), seqs)))
    return rows


def _check_attention(qkv, cache, lengths, heads, got) -> None:
    head = cache.shape[3] // 1152 * 64
    q = qkv[:, :heads * head].double().cpu().numpy().reshape(cache.shape[0], heads, head)
    want, bound = _q4.attend(q, cache.cpu().numpy(), lengths, heads)
    error = np.abs(got.double().cpu().numpy().reshape(want.shape) - want)
    assert np.isfinite(error).all()
    worst = np.max(error / np.maximum(bound, 1e-30) * (error > 0))
    assert worst <= 1.0, f"{worst:.3f} of the bound"


# ---- storing and reading back -----------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads,head", [(12, 12, 64), (0, 1, 64), (5, 5, 128), (8, 2, 128), (3, 3, 64)])
@pytest.mark.parametrize("seqs,tokens", [(1, 1), (3, 17), (2, 130)])
def test_stored_rows_read_back(heads: int, kv_heads: int, head: int, seqs: int, tokens: int) -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(heads * 131 + head + tokens)
    qkv = _rows(rng, seqs * tokens, heads + 2 * kv_heads, head).reshape(seqs * tokens, -1)
    cache = ops.kv_cache_q4(seqs, kv_heads, tokens + 9, head)
    seq, pos = np.repeat(np.arange(seqs), tokens), np.tile(np.arange(tokens) + 9, seqs)
    order = rng.permutation(seqs * tokens)
    ops.kv_store_q4(qkv[torch.from_numpy(order).cuda()].contiguous(), cache, _i32(seq[order]), _i32(pos[order]))
    got = ops.kv_load_q4(cache, _i32(seq), _i32(pos)).float().cpu().numpy()
    np.testing.assert_array_equal(got, _expected(qkv, kv_heads, head))


def test_rows_with_little_or_nothing_to_tell_apart() -> None:
    """All-equal rows (scale 0), zeros, rows of two neighbouring values, wide ranges, signed zeros and subnormals."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(5)
    base = rng.standard_normal((8, 128)).astype(np.float32)
    base[0] = 0.0
    base[1] = -3.25
    base[2] = np.where(np.arange(128) % 2, 1.0, 1.0078125)
    base[3] *= 1e30
    base[4] *= 1e-30
    base[5, ::2] = -0.0
    base[6] = np.arange(128) % 16          # every quotient an integer
    base[7] = (np.arange(128) % 31) * 0.5  # ties to even
    qkv = torch.from_numpy(base).cuda().to(torch.bfloat16)
    cache = ops.kv_cache_q4(1, 1, 16)
    seq, pos = _i32(np.zeros(8)), _i32(np.arange(8))
    ops.kv_store_q4(qkv, cache, seq, pos)
    got = ops.kv_load_q4(cache, seq, pos).float().cpu().numpy()
    np.testing.assert_array_equal(got, _expected(qkv, 1, 64))


def test_rows_that_are_not_finite_read_as_nan_and_leave_the_others() -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(6)
    qkv = _rows(rng, 4, 2, 64).reshape(4, 128)
    qkv[1, 5], qkv[2, 70], qkv[3, 0], qkv[3, 1] = float("nan"), float("inf"), 3.0e38, -3.0e38
    cache = ops.kv_cache_q4(1, 1, 16)
    seq, pos = _i32(np.zeros(4)), _i32(np.arange(4))
    ops.kv_store_q4(qkv, cache, seq, pos)
    got = ops.kv_load_q4(cache, seq, pos)
    assert torch.isnan(got[1, :64]).all() and torch.isnan(got[2, 64:]).all() and torch.isnan(got[3, :64]).all()
    clean = torch.ones(4, 128, dtype=torch.bool)
    clean[1, :64] = clean[2, 64:] = clean[3, :64] = False
    want = _expected(torch.where(clean.cuda(), qkv, torch.zeros_like(qkv)), 1, 64)
    np.testing.assert_array_equal(got.float().cpu().numpy()[clean.numpy()], want[clean.numpy()])


def test_places_outside_the_cache_are_skipped_and_read_as_zeros() -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(7)
    cache = ops.kv_cache_q4(2, 3, 32)
    _fill(cache, rng)
    before = cache.clone()
    qkv = _rows(rng, 6, 9, 64).reshape(6, -1)
    seq, pos = _i32([0, -1, 2, 1, 1, 1 << 30]), _i32([-1, 3, 3, 32, 1 << 30, 0])
    ops.kv_store_q4(qkv, cache, seq, pos)
    assert torch.equal(cache, before)
    assert not ops.kv_load_q4(cache, seq, pos).any()
    # one row inside: only its own place changes
    ops.kv_store_q4(qkv, cache, _i32([1, -1, -1, -1, -1, -1]), _i32([17, 0, 0, 0, 0, 0]))
    changed = (cache != before).nonzero()
    assert set(changed[:, 0].tolist()) == {1} and set(changed[:, 2].tolist()) == {1}
    inside = changed[:, 3]
    slot = torch.where(inside < 1024, inside % 512 // 32, (inside - 1024) // 8)
    assert set(slot.tolist()) == {1}


def test_rows_at_a_stride_and_offset() -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(8)
    wide = _rows(rng, 21, 9, 64).reshape(21, -1)
    qkv = wide[:, 64:7 * 64]  # two query heads, two key and two value heads at a row stride of nine heads
    cache = ops.kv_cache_q4(1, 2, 32)
    seq, pos = _i32(np.zeros(21)), _i32(np.arange(21))
    ops.kv_store_q4(qkv, cache, seq, pos)
    out = torch.full((21, 2 * 2 * 64 + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.kv_load_q4(cache, seq, pos, out=out[:, :256])
    np.testing.assert_array_equal(out[:, :256].float().cpu().numpy(), _expected(qkv, 2, 64))
    assert (out[:, 256:] == 7.0).all()
    lengths = [21]
    got = ops.decode_attention_q4(wide[:1, 64:7 * 64], cache, _i32(lengths))
    _check_attention(wide[:1, 64:7 * 64], cache, lengths, 2, got)


@pytest.mark.parametrize("head", [64, 128])
@pytest.mark.parametrize("offset,pad", [(0, 0), (8, 0), (0, 8), (8, 8), (16, 16)])
def test_rows_on_16_and_on_32_bytes(head: int, offset: int, pad: int) -> None:
    """Rows that begin on 32 bytes go by wider accesses than others; both store and read back alike, and nothing between
    the rows is written."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(21)
    rows, width = 71, 2 * 3 * head
    stride = width + pad
    flat = torch.zeros(rows * stride + 32, dtype=torch.bfloat16, device="cuda")
    qkv = flat[offset:offset + rows * stride].view(rows, stride)[:, :width]
    qkv.copy_(_rows(rng, rows, 6, head).reshape(rows, -1))
    cache = ops.kv_cache_q4(2, 3, 64, head)
    seq, pos = _i32(np.arange(rows) % 2), _i32(np.arange(rows) // 2)
    ops.kv_store_q4(qkv, cache, seq, pos)
    back = torch.full_like(flat, 7.0)
    out = back[offset:offset + rows * stride].view(rows, stride)[:, :width]
    ops.kv_load_q4(cache, seq, pos, out=out)
    np.testing.assert_array_equal(out.float().cpu().numpy(), _expected(qkv, 3, head))
    assert int((back == 7.0).sum()) >= back.numel() - rows * width and (back[:offset] == 7.0).all()
    assert (back[offset + rows * stride - pad:] == 7.0).all()


# ---- attention --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,kv_heads,head", [(12, 12, 64), (1, 1, 64), (8, 2, 64), (9, 1, 64), (40, 2, 64),
                                                 (4, 4, 128), (14, 2, 128), (17, 1, 128)])
@pytest.mark.parametrize("lengths", [[1], [15, 16, 17], [0, 1, 2, 63, 64, 65, 127, 400], [513, 0, 512, 300]])
def test_attention_matches_the_average(heads: int, kv_heads: int, head: int, lengths: list[int]) -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(heads + head + len(lengths))
    seqs = len(lengths)
    cache = ops.kv_cache_q4(seqs, kv_heads, max(lengths), head)
    _fill(cache, rng)
    qkv = (_rows(rng, seqs, heads + 2 * kv_heads, head) * (1.5 / head ** 0.5)).reshape(seqs, -1)
    got = ops.decode_attention_q4(qkv, cache, _i32(lengths))
    _check_attention(qkv, cache, lengths, heads, got)
    for s, n in enumerate(lengths):
        if n == 0:
            assert not got[s].any()
    # the offset counts the step's own token, and lengths past the capacity are clamped to it
    capacity = cache.shape[2] * 16
    shifted = [n - 1 for n in lengths]
    assert torch.equal(ops.decode_attention_q4(qkv, cache, _i32(shifted), length_offset=1), got)
    far = ops.decode_attention_q4(qkv, cache, _i32([2 ** 31 - 1] * seqs), length_offset=2 ** 31 - 1)
    assert torch.equal(far, ops.decode_attention_q4(qkv, cache, _i32([capacity] * seqs)))
    none = ops.decode_attention_q4(qkv, cache, _i32([-2 ** 31] * seqs), length_offset=-2 ** 31)
    assert not none.any()


@pytest.mark.parametrize("seqs,heads,kv_heads,head,length", [(1, 12, 12, 64, 5000), (1, 4, 1, 128, 20011),
                                                             (40, 12, 12, 64, 333), (150, 2, 1, 64, 97)])
def test_attention_over_grids_of_every_shape(seqs: int, heads: int, kv_heads: int, head: int, length: int) -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(length)
    cache = ops.kv_cache_q4(seqs, kv_heads, length, head)
    _fill(cache, rng)
    lengths = rng.integers(length // 2, length + 1, seqs)
    lengths[0] = length
    qkv = (_rows(rng, seqs, heads, head) * (1.5 / head ** 0.5)).reshape(seqs, -1)
    got = ops.decode_attention_q4(qkv, cache, _i32(lengths), heads=heads)
    _check_attention(qkv, cache, lengths, heads, got)


@pytest.mark.parametrize("heads,kv_heads,head", [(12, 12, 64), (24, 12, 64), (48, 12, 64), (64, 8, 64), (12, 12, 128),
                                                 (32, 8, 128), (64, 8, 128)])
@pytest.mark.parametrize("seqs,length", [(3, 300), (20, 420), (30, 400), (45, 260), (260, 33), (2, 2000), (1, 6000)])
def test_attention_over_every_split(seqs: int, length: int, heads: int, kv_heads: int, head: int) -> None:
    """CTAs of two, four and eight warps, clusters and the workspace, for one to eight queries a key head."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(seqs)
    cache = ops.kv_cache_q4(seqs, kv_heads, length, head)
    _fill(cache, rng)
    lengths = rng.integers(1, length + 1, seqs)
    qkv = (_rows(rng, seqs, heads, head) * (1.5 / head ** 0.5)).reshape(seqs, -1)
    got = ops.decode_attention_q4(qkv, cache, _i32(lengths), heads=heads)
    some = np.unique(np.concatenate([[0, seqs - 1], rng.integers(0, seqs, 3)]))
    index = torch.from_numpy(some).cuda()
    _check_attention(qkv[index], cache[index], lengths[some], heads, got[index])


def test_attention_reads_nothing_past_the_length() -> None:
    """NaN rows and a later, far greater key behind the last position change nothing."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(11)
    lengths = [1, 16, 29, 70]
    cache = ops.kv_cache_q4(4, 2, 96)
    _fill(cache, rng)
    qkv = (_rows(rng, 4, 4, 64) * 0.2).reshape(4, -1)
    want = ops.decode_attention_q4(qkv, cache, _i32(lengths), heads=4)
    bad = _rows(rng, 4, 4, 64).reshape(4, -1) * 1e4
    bad[2] = float("nan")
    bad[3, 100] = float("inf")
    for ahead in (0, 1, 2, 16, 25):
        ops.kv_store_q4(bad, cache, _i32(np.arange(4)), _i32(np.asarray(lengths) + ahead))
    assert torch.equal(ops.decode_attention_q4(qkv, cache, _i32(lengths), heads=4), want)


@pytest.mark.parametrize("k_size,v_size,q_size", [(1.0, 1e-6, 1.0), (1.0, 1e20, 1.0), (1e-20, 1.0, 1.0),
                                                  (30.0, 1.0, 3.0), (1e-4, 1e-30, 1e4), (1e4, 1.0, 1e-4)])
def test_attention_over_keys_and_values_of_any_size(k_size: float, v_size: float, q_size: float) -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(12)
    cache = ops.kv_cache_q4(2, 2, 200)
    rows = _rows(rng, 400, 4, 64).float()
    rows[:, :2] *= k_size
    rows[:, 2:] *= v_size
    rows[7::13, 2:] = 0.0   # value rows without any range
    rows = rows.to(torch.bfloat16).reshape(400, -1)
    ops.kv_store_q4(rows, cache, _i32(np.repeat([0, 1], 200)), _i32(np.tile(np.arange(200), 2)))
    qkv = (_rows(rng, 2, 2, 64).float() * 0.2 * q_size).to(torch.bfloat16).reshape(2, -1)
    got = ops.decode_attention_q4(qkv, cache, _i32([200, 131]), heads=2)
    _check_attention(qkv, cache, [200, 131], 2, got)


def test_scores_that_rise_and_fall_along_the_keys() -> None:
    """The running maximum moves at every tile, or only at the first: a weight of all but one key vanishes."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(13)
    n = 300
    cache = ops.kv_cache_q4(2, 1, n)
    rows = _rows(rng, 2 * n, 2, 64).float()
    slope = np.concatenate([np.arange(n), np.arange(n)[::-1]]).astype(np.float32)
    rows[:, 0] = rows[:, 0] * 0.1 + torch.from_numpy(slope).cuda()[:, None] * 0.05
    rows = rows.to(torch.bfloat16).reshape(2 * n, -1)
    ops.kv_store_q4(rows, cache, _i32(np.repeat([0, 1], n)), _i32(np.tile(np.arange(n), 2)))
    qkv = torch.full((2, 64), 0.5, dtype=torch.bfloat16, device="cuda")
    got = ops.decode_attention_q4(qkv, cache, _i32([n, n]), heads=1)
    _check_attention(qkv, cache, [n, n], 1, got)


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("n", [1, 16, 300, 9000])
def test_scores_far_below_zero(n: int, rising: bool) -> None:
    """Scores from -6e35 down: the least negative position takes all of the weight, and its value row is the output but
    for the FP16 rounding of its weight, a few FP32 roundings of 64 + 15 steps, and the output's own."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(n)
    cache = ops.kv_cache_q4(1, 1, n)
    rows = _rows(rng, n, 2, 64).float()
    factor = 1 + np.minimum(np.arange(n), 100).astype(np.float32) / 8
    rows[:, 0] = -1e17 * torch.from_numpy(factor[::-1].copy() if rising else factor).cuda()[:, None]
    rows = rows.to(torch.bfloat16).reshape(n, -1)
    ops.kv_store_q4(rows, cache, _i32(np.zeros(n)), _i32(np.arange(n)))
    qkv = torch.full((1, 64), 1e17, dtype=torch.bfloat16, device="cuda")
    got = ops.decode_attention_q4(qkv, cache, _i32([n]), heads=1).double().cpu().numpy()[0]
    codes, scale, low = _q4.quantise(rows[n - 1 if rising else 0, 64:].float().cpu().numpy())
    want, wide = codes * scale + low, 15 * scale
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -11 + 2.0 ** -16) * wide).all()


@pytest.mark.parametrize("head,n", [(64, 40), (64, 1152), (128, 9000)])
@pytest.mark.parametrize("score", [1e8, -1e8, 1e11, -1e11, 1e30, -1e30])
@pytest.mark.parametrize("v_size", [1e-25, 1.0, 1e6, 1e25])
def test_scores_and_values_of_any_size(head: int, n: int, score: float, v_size: float) -> None:
    """Beside scores of 2^27 and more the values' size counts for nothing in FP32: the position with the greatest score still
    gives its value row, as above."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(n)
    cache = ops.kv_cache_q4(1, 1, n, head)
    rows = _rows(rng, n, 2, head).float()
    factor = 1 + np.minimum(np.arange(n), 100).astype(np.float32) / 8
    size = math.sqrt(abs(score) / head)
    rows[:, 0] = math.copysign(size, score) * torch.from_numpy(factor[::-1].copy() if score > 0 else factor).cuda()[:, None]
    rows[:, 1] *= v_size
    rows = rows.to(torch.bfloat16).reshape(n, -1)
    ops.kv_store_q4(rows, cache, _i32(np.zeros(n)), _i32(np.arange(n)))
    # the greatest score is position 0's, shared by as many as the factor's clamp gives it to
    best = int((rows[:, 0] == rows[0, 0]).sum())
    qkv = torch.full((1, 3 * head), size, dtype=torch.bfloat16, device="cuda")
    got = ops.decode_attention_q4(qkv, cache, _i32([n]), heads=3).double().cpu().numpy().reshape(3, -1, 64)
    codes, scale, low = _q4.quantise(rows[:best, head:].float().cpu().numpy().reshape(best, -1, 64))
    want, wide = (codes * scale + low).mean(0), 15 * scale.max(0)
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + (2.0 ** -11 + 2.0 ** -16 + best * 2.0 ** -23) * wide).all()


def test_a_nan_key_or_value_within_the_length_shows_in_its_own_head() -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(14)
    cache = ops.kv_cache_q4(1, 3, 64)
    _fill(cache, rng)
    qkv = (_rows(rng, 1, 3, 64) * 0.2).reshape(1, -1)
    want = ops.decode_attention_q4(qkv, cache, _i32([64]), heads=3)
    row = _rows(rng, 1, 6, 64).reshape(1, -1)
    ops.kv_store_q4(row, cache, _i32([0]), _i32([40]))
    want = ops.decode_attention_q4(qkv, cache, _i32([64]), heads=3)
    row[0, 3] = float("nan")            # key head 0
    row[0, 5 * 64 + 1] = float("inf")   # value head 2
    ops.kv_store_q4(row, cache, _i32([0]), _i32([40]))
    got = ops.decode_attention_q4(qkv, cache, _i32([64]), heads=3)
    assert torch.isnan(got[:, :64]).all() and torch.isnan(got[:, 128:]).all()
    assert torch.equal(got[:, 64:128], want[:, 64:128])


def test_a_slice_of_sequences_is_a_cache_and_its_neighbours_stay() -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(15)
    cache = ops.kv_cache_q4(5, 2, 48)
    _fill(cache, rng)
    before = cache.clone()
    qkv = _rows(rng, 2, 6, 64).reshape(2, -1)
    part = cache[2:4]
    ops.kv_store_q4(qkv, part, _i32([0, 1]), _i32([5, 47]))
    assert torch.equal(cache[:2], before[:2]) and torch.equal(cache[4:], before[4:])
    out = torch.full((4, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.decode_attention_q4(qkv, part, _i32([6, 48]), out=out[1:3])
    _check_attention(qkv, part, [6, 48], 2, out[1:3])
    assert (out[0] == 3.0).all() and (out[3] == 3.0).all()


def test_offsets_past_32_bits() -> None:
    """The last sequence of a cache of more than 4 GiB."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(16)
    seqs, capacity = 5, 1 << 20  # 5 x 12 x 65536 tiles x 1152 bytes = 4.5 GB
    cache = ops.kv_cache_q4(seqs, 12, capacity)
    assert cache.numel() > 1 << 32
    qkv = _rows(rng, 3, 36, 64).reshape(3, -1)
    seq, pos = _i32([4, 4, 4]), _i32([0, 1, capacity - 1])
    ops.kv_store_q4(qkv, cache, seq, pos)
    np.testing.assert_array_equal(ops.kv_load_q4(cache, seq, pos).float().cpu().numpy(), _expected(qkv, 12, 64))
    q = (_rows(rng, seqs, 12, 64) * 0.2).reshape(seqs, -1)
    got = ops.decode_attention_q4(q, cache, _i32([0, 0, 0, 0, 2]), heads=12)
    assert not got[:4].any()
    _check_attention(q[4:], cache[4:, :, :1], [2], 12, got[4:])


def test_store_and_attention_in_one_graph_on_another_stream() -> None:
    """A decode step's append and attention, captured once and replayed with other rows, against the eager calls."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(17)
    seqs = 7
    cache = ops.kv_cache_q4(seqs, 4, 80)
    _fill(cache, rng)
    qkv = (_rows(rng, seqs, 12, 64) * 0.3).reshape(seqs, -1)
    seq, pos = _i32(np.arange(seqs)), _i32(rng.integers(0, 79, seqs))
    out = torch.zeros((seqs, 256), dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.kv_store_q4(qkv, cache, seq, pos)
        ops.decode_attention_q4(qkv, cache, pos, length_offset=1, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.kv_store_q4(qkv, cache, seq, pos)
            ops.decode_attention_q4(qkv, cache, pos, length_offset=1, out=out)
            pos += 1
    stream.synchronize()
    eager_cache, eager_pos = cache.clone(), pos.clone()
    for step in range(3):
        qkv.copy_((_rows(rng, seqs, 12, 64) * 0.3).reshape(seqs, -1))
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        stream.synchronize()
        ops.kv_store_q4(qkv, eager_cache, seq, eager_pos)
        want = ops.decode_attention_q4(qkv, eager_cache, eager_pos, length_offset=1)
        eager_pos += 1
        assert torch.equal(out, want) and torch.equal(cache, eager_cache)


def test_two_graphs_of_split_calls_at_once() -> None:
    """Two captured calls that go through a workspace each, replayed on two streams at the same time."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(19)
    states = []
    for k in range(2):
        cache = ops.kv_cache_q4(1, 2, 9000)
        _fill(cache, rng)
        qkv = (_rows(rng, 1, 6, 64) * 0.2).reshape(1, -1)
        lengths = _i32([8000 + k])
        assert ops.decode_attention_q4_workspace_bytes(1, 6, 2, 64, cache.shape[2] * 16) > 0
        want = ops.decode_attention_q4(qkv, cache, lengths, heads=6)
        stream, out = torch.cuda.Stream(), torch.zeros_like(want)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            ops.decode_attention_q4(qkv, cache, lengths, heads=6, out=out)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                for _ in range(4):
                    ops.decode_attention_q4(qkv, cache, lengths, heads=6, out=out)
        states.append((stream, graph, out, want, (qkv, cache, lengths)))
    torch.cuda.synchronize()
    for _, _, out, _, _ in states:
        out.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, graph, _, _, _ in states:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, want, _ in states:
        assert torch.equal(out, want)


def test_one_graph_of_every_split() -> None:
    """Calls of one CTA a pair, of clusters and of the workspace in one captured graph beside an eager stream of others."""
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(23)
    calls = []
    for seqs, heads, kv_heads, head, n in ((3, 12, 12, 64, 384), (1, 12, 12, 64, 1152), (2, 8, 2, 128, 2100),
                                           (1, 4, 1, 64, 9000), (300, 12, 12, 64, 40)):
        cache = ops.kv_cache_q4(seqs, kv_heads, n, head)
        _fill(cache, rng)
        qkv = (_rows(rng, seqs, heads, head) * (1.5 / head ** 0.5)).reshape(seqs, -1)
        lengths = rng.integers(0, n + 1, seqs)
        want = ops.decode_attention_q4(qkv, cache, _i32(lengths), heads=heads)
        _check_attention(qkv, cache, lengths, heads, want)
        calls.append((qkv, cache, _i32(lengths), heads, torch.zeros_like(want), want))
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for qkv, cache, lengths, heads, out, _ in calls:
            ops.decode_attention_q4(qkv, cache, lengths, heads=heads, out=out)
    for _ in range(4):
        for call in calls:
            call[4].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        eager = [ops.decode_attention_q4(qkv, cache, lengths, heads=heads) for qkv, cache, lengths, heads, _, _ in calls]
        torch.cuda.synchronize()
        for (_, _, _, _, out, want), other in zip(calls, eager):
            assert torch.equal(out, want) and torch.equal(other, want)


def test_the_same_inputs_give_the_same_bits() -> None:
    from tempo_compiler_b200 import ops
    rng = np.random.default_rng(18)
    cache = ops.kv_cache_q4(3, 4, 3000)
    _fill(cache, rng)
    qkv = (_rows(rng, 3, 8, 64) * 0.2).reshape(3, -1)
    lengths = _i32([3000, 1777, 5])
    first = ops.decode_attention_q4(qkv, cache, lengths, heads=8)
    for _ in range(5):
        assert torch.equal(ops.decode_attention_q4(qkv, cache, lengths, heads=8), first)


def test_the_wrappers_refuse_what_does_not_fit() -> None:
    from tempo_compiler_b200 import ops
    cache = ops.kv_cache_q4(2, 3, 32)
    qkv = torch.zeros((2, 9 * 64), dtype=torch.bfloat16, device="cuda")
    two, three = _i32([0, 1]), _i32([0, 1, 2])
    out = torch.zeros((2, 192), dtype=torch.bfloat16, device="cuda")
    cases = [
        (lambda: ops.kv_store_q4(qkv.float(), cache, two, two), "bfloat16"),
        (lambda: ops.kv_store_q4(qkv[:, :500], cache, two, two), "heads of 64"),
        (lambda: ops.kv_store_q4(qkv[:, :320], cache, two, two), "heads of 64"),
        (lambda: ops.kv_store_q4(qkv, cache, three, two), "as many"),
        (lambda: ops.kv_store_q4(qkv, cache, two.long(), two), "int32"),
        (lambda: ops.kv_store_q4(qkv, cache.view(2, 3, 1, 2304)[..., :1000], two, two), "contiguous"),
        (lambda: ops.kv_store_q4(qkv, cache.view(2, 3, -1), two, two), "kv_cache_q4"),
        (lambda: ops.kv_store_q4(qkv.T.contiguous().T, cache, two, two), "contiguous rows"),
        (lambda: ops.kv_store_q4(qkv[:1].expand(2, -1), cache, two, two), "overlap"),
        (lambda: ops.kv_store_q4(qkv[:0], cache, two[:0], two[:0]), "rows 0"),
        (lambda: ops.kv_store_q4(qkv.view(-1)[4:4 + 2 * 512].view(2, 512)[:, :384], cache, two, two), "aligned"),
        (lambda: ops.kv_load_q4(cache, two, three), "as many"),
        (lambda: ops.kv_load_q4(cache, two, two, out=out), "out must be"),
        (lambda: ops.decode_attention_q4(qkv, cache, three), "a length each"),
        (lambda: ops.decode_attention_q4(qkv[:1], cache, two), "a length each"),
        (lambda: ops.decode_attention_q4(qkv, cache, two, heads=4), "multiple of"),
        (lambda: ops.decode_attention_q4(qkv, cache, two, heads=12), "query heads"),
        (lambda: ops.decode_attention_q4(qkv[:, :384], cache, two), "query heads"),
        (lambda: ops.decode_attention_q4(qkv, cache, two, out=out[:, :128]), "contiguous"),
        (lambda: ops.decode_attention_q4(qkv, cache, two, out=out[:1]), "out must be"),
        (lambda: ops.decode_attention_q4(qkv, cache, two.cpu()), "CUDA"),
        (lambda: ops.decode_attention_q4(qkv, cache.cpu(), two), "CUDA"),
    ]
    for call, words in cases:
        with pytest.raises(ValueError, match=words):
            call()
