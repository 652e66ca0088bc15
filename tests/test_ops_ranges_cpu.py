"""The torch wrappers of the 4-bit cache and the scores pass strides and offsets on in 32 bits: what 32 bits do not hold is
refused, not cut off (no GPU: stand-ins have the attributes of tensors on one)."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")


class _OnGpu:
    """A tensor of a given type, shape and strides on cuda:0, without memory."""

    is_cuda, device = True, torch.device("cuda", 0)

    def __init__(self, dtype, shape, strides=None) -> None:
        self.dtype, self.shape = dtype, torch.Size(shape)
        self.strides = strides
        if strides is None:
            self.strides, size = [], 1
            for n in reversed(shape):
                self.strides.insert(0, size)
                size *= n
        self.contiguous = strides is None

    def dim(self) -> int:
        return len(self.shape)

    def stride(self) -> tuple:
        return tuple(self.strides)

    def numel(self) -> int:
        return self.shape.numel()

    def get_device(self) -> int:
        return 0

    def is_contiguous(self) -> bool:
        return self.contiguous

    def data_ptr(self) -> int:
        return 4096

    def new_empty(self, size, dtype=None) -> "_OnGpu":
        return _OnGpu(dtype or self.dtype, (size,) if isinstance(size, int) else size)


@pytest.fixture
def launched(monkeypatch):
    from tempo_compiler_b200 import ops
    calls = []
    monkeypatch.setattr(ops, "_launch_at", lambda device, name, *args: calls.append((name, args)))
    return calls


def _i32(*shape: int) -> _OnGpu:
    return _OnGpu(torch.int32, shape)


@pytest.mark.parametrize("stride", [2 ** 32, 2 ** 32 + 2304, 2 ** 40])
def test_row_strides_of_more_than_32_bits_are_refused(launched, stride: int) -> None:
    from tempo_compiler_b200 import ops
    cache, two = _OnGpu(torch.uint8, (2, 12, 3, 1152)), _i32(2)
    far = _OnGpu(torch.bfloat16, (2, 2304), (stride, 1))
    with pytest.raises(ValueError, match="stride"):
        ops.kv_store_q4(far, cache, two, two)
    with pytest.raises(ValueError, match="stride"):
        ops.decode_attention_q4(far, cache, two)
    with pytest.raises(ValueError, match="stride"):
        ops.kv_load_q4(cache, two, two, out=_OnGpu(torch.bfloat16, (2, 1536), (stride, 1)))
    with pytest.raises(ValueError, match="stride"):
        ops.gemm_f32(_OnGpu(torch.bfloat16, (2, 64)), _OnGpu(torch.bfloat16, (40, 64)),
                     out=_OnGpu(torch.float32, (2, 40), (stride, 1)))
    assert not launched
    # the greatest that 32 bits and the kernels' alignment hold, and logits at any stride
    most = _OnGpu(torch.bfloat16, (2, 2304), (2 ** 32 - 8, 1))
    ops.kv_store_q4(most, cache, two, two)
    assert launched.pop()[1][1] == 2 ** 32 - 8
    ops.token_logprobs(_OnGpu(torch.float32, (2, 40), (stride, 1)), two, out=ops.TokenScores(
        _OnGpu(torch.float32, (2,)), _OnGpu(torch.float32, (2,))))
    assert launched.pop()[1][1] == stride


@pytest.mark.parametrize("offset", [2 ** 31, 2 ** 32 + 5, -2 ** 31 - 1])
def test_offsets_of_more_than_32_bits_are_refused(launched, offset: int) -> None:
    from tempo_compiler_b200 import ops
    cache, two = _OnGpu(torch.uint8, (2, 12, 3, 1152)), _i32(2)
    with pytest.raises(ValueError, match="length_offset"):
        ops.decode_attention_q4(_OnGpu(torch.bfloat16, (2, 2304)), cache, two, length_offset=offset)
    out = ops.TokenScores(_OnGpu(torch.float32, (3, 2)), _OnGpu(torch.float32, (3, 2)))
    with pytest.raises(ValueError, match="slot_offset"):
        ops.token_logprobs(_OnGpu(torch.float32, (2, 40)), two, out=out, slots=two, slot_offset=offset)
    assert not launched
    for held in (2 ** 31 - 1, -2 ** 31):
        ops.decode_attention_q4(_OnGpu(torch.bfloat16, (2, 2304)), cache, two, length_offset=held)
        ops.token_logprobs(_OnGpu(torch.float32, (2, 40)), two, out=out, slots=two, slot_offset=held)
    assert len(launched) == 4
