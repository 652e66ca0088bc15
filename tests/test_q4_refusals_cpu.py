"""What the 4-bit cache's and the scores' entry points refuse, before any device work (no GPU)."""

from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")


def _buffer() -> int:
    """A 16-byte aligned host address: refusals never look behind it."""
    _buffer.keep = ctypes.create_string_buffer(256)
    return (ctypes.addressof(_buffer.keep) + 63) // 64 * 64


def _status(name: str, *args) -> int:
    from tempo_compiler_b200 import lib
    return getattr(lib.load(), name)(*args)


GOOD_STORE = dict(ldq=2304, rows=4, seqs=2, heads=12, kv_heads=12, head=64, capacity=32)


@pytest.mark.parametrize("change", [dict(ldq=2296), dict(ldq=2308), dict(rows=0), dict(seqs=0), dict(kv_heads=0),
                                    dict(head=96), dict(head=32), dict(capacity=0), dict(capacity=40),
                                    dict(heads=0xFFFFFFFF), dict(rows=0xFFFFFFFF), dict(kv_heads=0x80000000)])
def test_store_and_load_refuse(change: dict) -> None:
    from tempo_compiler_b200 import lib
    a = {**GOOD_STORE, **change}
    p = _buffer()
    assert _status("tempo_kv_store_q4", p, a["ldq"], p, p, p, a["rows"], a["seqs"], a["heads"], a["kv_heads"], a["head"],
                   a["capacity"], None) == lib.ERR_VALUE
    if "heads" in change:
        return
    ldo = {2296: 1528, 2308: 1540}.get(a["ldq"], 1536)
    assert _status("tempo_kv_load_q4", p, p, ldo, p, p, a["rows"], a["seqs"], a["kv_heads"], a["head"], a["capacity"],
                   None) == lib.ERR_VALUE


@pytest.mark.parametrize("which", range(4))
def test_store_and_load_refuse_missing_or_misaligned_pointers(which: int) -> None:
    from tempo_compiler_b200 import lib
    for bad in (None, _buffer() + 8):
        if which >= 2 and bad is not None:
            continue  # the index arrays only need to be there
        p = [_buffer()] * 4
        p[which] = bad
        assert _status("tempo_kv_store_q4", p[0], 2304, p[1], p[2], p[3], 4, 2, 12, 12, 64, 32, None) == lib.ERR_VALUE
        assert _status("tempo_kv_load_q4", p[1], p[0], 1536, p[2], p[3], 4, 2, 12, 64, 32, None) == lib.ERR_VALUE


@pytest.mark.parametrize("change", [dict(ldq=760), dict(ldq=772), dict(seqs=0), dict(seqs=65536), dict(heads=0),
                                    dict(heads=13), dict(kv_heads=0), dict(kv_heads=5), dict(kv_heads=65536, heads=65536),
                                    dict(head=80), dict(capacity=0), dict(capacity=31)])
def test_attention_refuses(change: dict) -> None:
    from tempo_compiler_b200 import lib
    a = {**dict(ldq=768, seqs=2, heads=12, kv_heads=12, head=64, capacity=32), **change}
    p = _buffer()
    assert _status("tempo_decode_attention_q4", p, a["ldq"], p, p, 0, p, a["seqs"], a["heads"], a["kv_heads"], a["head"],
                   a["capacity"], None, 0, None) == lib.ERR_VALUE
    if "ldq" not in change:
        assert _status("tempo_decode_attention_q4_workspace", a["seqs"], a["heads"], a["kv_heads"], a["head"],
                       a["capacity"], ctypes.byref(ctypes.c_uint64())) == lib.ERR_VALUE


@pytest.mark.parametrize("which,bad", [(0, None), (0, 8), (1, None), (1, 8), (2, None), (3, None), (3, 8)])
def test_attention_refuses_pointers(which: int, bad) -> None:
    from tempo_compiler_b200 import lib
    p = [_buffer()] * 4
    p[which] = None if bad is None else p[which] + bad
    assert _status("tempo_decode_attention_q4", p[0], 768, p[1], p[2], 0, p[3], 2, 12, 12, 64, 32, None, 0,
                   None) == lib.ERR_VALUE


def test_attention_refuses_a_workspace_that_is_missing_small_or_misaligned() -> None:
    """One sequence of one key head and a long capacity needs one; short or many sequences do not."""
    from tempo_compiler_b200 import lib
    size, p = ctypes.c_uint64(), _buffer()
    assert _status("tempo_decode_attention_q4_workspace", 1, 4, 1, 128, 65536, ctypes.byref(size)) == lib.OK
    assert size.value > 0
    for pointer, given in ((None, size.value), (p, size.value - 1), (p + 8, size.value)):
        assert _status("tempo_decode_attention_q4", p, 512, p, p, 0, p, 1, 4, 1, 128, 65536, pointer, given,
                       None) == lib.ERR_VALUE
    assert _status("tempo_decode_attention_q4_workspace", 1, 4, 1, 128, 65536, None) == lib.ERR_VALUE
    for seqs, capacity in ((1, 256), (512, 65536)):
        assert _status("tempo_decode_attention_q4_workspace", seqs, 12, 12, 64, capacity, ctypes.byref(size)) == lib.OK
        assert size.value == 0


@pytest.mark.parametrize("change", [dict(rows=0), dict(vocab=0), dict(ld=99), dict(top=33), dict(vocab=8, top=9),
                                    dict(bf16=2), dict(rows=0x80000000), dict(vocab=0x80000000, ld=1 << 40)])
def test_scores_refuse(change: dict) -> None:
    from tempo_compiler_b200 import lib
    a = {**dict(ld=100, bf16=0, rows=2, vocab=100, top=5), **change}
    p = _buffer()
    assert _status("tempo_token_logprobs", p, a["ld"], a["bf16"], p, a["rows"], a["vocab"], a["top"], p, p, p, p,
                   None, 0, 0, None) == lib.ERR_VALUE


@pytest.mark.parametrize("which,bad", [(0, None), (0, 2), (1, None), (2, None), (3, None), (4, None), (5, None)])
def test_scores_refuse_pointers(which: int, bad) -> None:
    from tempo_compiler_b200 import lib
    p = [_buffer()] * 6
    p[which] = None if bad is None else p[which] + bad
    assert _status("tempo_token_logprobs", p[0], 100, 0, p[1], 2, 100, 5, p[2], p[3], p[4], p[5], None, 0, 0,
                   None) == lib.ERR_VALUE


def test_scores_refuse_slots_without_any() -> None:
    from tempo_compiler_b200 import lib
    p = _buffer()
    assert _status("tempo_token_logprobs", p, 100, 0, p, 2, 100, 0, p, p, None, None, p, 0, 0, None) == lib.ERR_VALUE


def test_fp32_product_refuses_other_modes() -> None:
    from tempo_compiler_b200 import lib
    p = _buffer()
    good = [p, 64, p, 64, None, None, 0, p, 16, 4, 16, 64]
    for change in ({4: p}, {5: p, 6: 16}):
        args = [change.get(i, v) for i, v in enumerate(good)]
        assert _status("tempo_gemm", *args, lib.GEMM_F32, None, None, None) == lib.ERR_VALUE
    for flags in (lib.GEMM_F32 | lib.GEMM_GELU, lib.GEMM_F32 | lib.GEMM_ARGMAX, lib.GEMM_F32 | lib.GEMM_LN):
        assert _status("tempo_gemm", *good, flags, p, p, None) == lib.ERR_VALUE
    assert _status("tempo_gemm_rowstats", *good, lib.GEMM_F32, p, None) == lib.ERR_VALUE


def test_the_torch_wrappers_refuse_host_tensors_and_bad_shapes() -> None:
    from tempo_compiler_b200 import ops
    cache = torch.zeros((1, 1, 1, 1152), dtype=torch.uint8)
    ids = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_store_q4(torch.zeros((1, 128), dtype=torch.bfloat16), cache, ids, ids)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_load_q4(cache, ids, ids)
    with pytest.raises(ValueError, match="CUDA"):
        ops.decode_attention_q4(torch.zeros((1, 64), dtype=torch.bfloat16), cache, ids, heads=1)
    with pytest.raises(ValueError, match="CUDA"):
        ops.token_logprobs(torch.zeros((1, 8)), ids)
    with pytest.raises(ValueError, match="CUDA"):
        ops.gemm_f32(torch.zeros((1, 8), dtype=torch.bfloat16), torch.zeros((8, 8), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="64 or 128"):
        ops.kv_cache_q4(1, 1, 16, 96, device="cpu")
    with pytest.raises(ValueError, match="needs"):
        ops.kv_cache_q4(1, 1, 0, device="cpu")
    assert ops.kv_cache_q4(2, 3, 17, 128, device="cpu").shape == (2, 3, 2, 2304)
