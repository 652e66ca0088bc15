"""torch-tensor wrappers over the native C-ABI entry points (section 3 of include/tempo_b200.h).

torch supplies device memory and the current CUDA stream; every op passes raw pointers and sizes to
libtempo_b200.so, whose kernels do the work. Nothing here computes on its own, and nothing falls back: a CPU tensor,
a wrong dtype or a missing library raises.
"""

from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from tempo_compiler_b200 import lib as _lib


_LAUNCHES = [0]


def _stream() -> int:
    """The current device's current stream, as the library takes it (a Stream object costs 3 us more to make)."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _launch(name: str, *args) -> None:
    """Calls one kernel-launching entry point of the library (one kernel per call) and counts it."""
    _LAUNCHES[0] += 1
    _lib.call(name, *args)


def reset_launch_count() -> None:
    _LAUNCHES[0] = 0


def launch_count() -> int:
    """Kernel launches issued through this module since the last reset (graph replays are not counted)."""
    return _LAUNCHES[0]


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _check(t: torch.Tensor, dtype: torch.dtype, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor: the B200 kernels have no CPU path")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _operand(t: torch.Tensor, dtype: torch.dtype, name: str, device: int) -> None:
    """A contiguous operand on the call's device (its number, as get_device gives it)."""
    if t.dtype is dtype and t.get_device() == device and t.is_contiguous():
        return
    _check(t, dtype, name)
    raise ValueError(f"{name} is on {t.device}, the call's first operand on cuda:{device}")


def _matrix(t: torch.Tensor, dtype: torch.dtype, name: str, device: int | None = None) -> tuple[int, int, int, int]:
    """(rows, columns, row stride, device) of a matrix whose rows are contiguous, at any row stride; a single row's own
    stride means nothing. Without `device` the matrix is the call's first operand."""
    if t.dtype is not dtype or not t.is_cuda:
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor: the B200 kernels have no CPU path")
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() == 2:
        rows, width = t.shape
        step, unit = t.stride()
        if (unit == 1 or width == 1) and (step >= width or rows == 1):
            on = t.get_device()
            if device is not None and on != device:
                raise ValueError(f"{name} is on {t.device}, the call's first operand on cuda:{device}")
            return rows, width, step if rows != 1 else (width + 7) // 8 * 8, on
    raise ValueError(f"{name} must be a matrix of contiguous rows that do not overlap")


def _stride32(stride: int, name: str) -> int:
    """A row stride that the entry point takes in 32 bits."""
    if stride >> 32:
        raise ValueError(f"{name} has a row stride of {stride} elements: 32 bits hold no more than {2 ** 32 - 1}")
    return stride


def _int32(value: int, name: str) -> int:
    """An offset that the entry point takes in 32 bits."""
    if not -2 ** 31 <= value < 2 ** 31:
        raise ValueError(f"{name} must be in [-2^31, 2^31), got {value}")
    return value


_ENTRIES: dict[str, object] = {}


def _launch_at(device: int, name: str, *args) -> None:
    """_launch on the current stream of `device`, which need not be the current device."""
    entry = _ENTRIES.get(name)
    if entry is None:
        entry = _ENTRIES[name] = getattr(_lib.load(), name)
    if device == torch._C._cuda_getDevice():
        status = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = entry(*args, torch._C._cuda_getCurrentRawStream(device))
    _LAUNCHES[0] += 1
    if status:
        _lib.check(status)


def gemm(a: torch.Tensor, w_t: torch.Tensor, *, bias: torch.Tensor | None = None,
         residual: torch.Tensor | None = None, gelu: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[M, N] = epilogue(a[M, K] @ w_t[N, K]^T): + bias, exact-erf GELU (of the BF16-rounded sum), + residual. The
    kernel reads w_t before earlier calls of this module have finished: w_t must not be what they write."""
    _check(a, torch.bfloat16, "a")
    _check(w_t, torch.bfloat16, "w_t")
    m, k = a.shape
    n = w_t.shape[0]
    if w_t.shape[1] != k:
        raise ValueError(f"inner dimensions differ: a {tuple(a.shape)}, w_t {tuple(w_t.shape)}")
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=a.device)
    _check(out, torch.bfloat16, "out")
    if bias is not None:
        _check(bias, torch.bfloat16, "bias")
    if residual is not None:
        _check(residual, torch.bfloat16, "residual")
    flags = _lib.GEMM_GELU if gelu else 0
    _launch("tempo_gemm", a.data_ptr(), k, w_t.data_ptr(), k, _ptr(bias), _ptr(residual), n, out.data_ptr(), n, m, n,
              k, flags, None, None, _stream())
    return out


def gemm_f32(a: torch.Tensor, w_t: torch.Tensor, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[M, N] = a[M, K] @ w_t[N, K]^T in FP32, the accumulators unrounded (an LM head's logits). `out` may have a
    row stride of its own, a multiple of 8; without it the rows are padded to one and the view of N columns returned.
    Both operands may be what an earlier call writes."""
    _check(a, torch.bfloat16, "a")
    device = a.get_device()
    _operand(w_t, torch.bfloat16, "w_t", device)
    m, k = a.shape
    n = w_t.shape[0]
    if w_t.shape[1] != k:
        raise ValueError(f"inner dimensions differ: a {tuple(a.shape)}, w_t {tuple(w_t.shape)}")
    if out is None:
        out = a.new_empty((m, (n + 7) // 8 * 8), dtype=torch.float32)[:, :n]
    out_rows, out_columns, stride, _ = _matrix(out, torch.float32, "out", device)
    if out_rows != m or out_columns != n:
        raise ValueError(f"out must be {(m, n)}, got {tuple(out.shape)}")
    _launch_at(device, "tempo_gemm", a.data_ptr(), k, w_t.data_ptr(), k, None, None, n, out.data_ptr(),
               _stride32(stride, "out"), m, n, k, _lib.GEMM_F32, None, None)
    return out


def gemm_qkv(a: torch.Tensor, w_t: torch.Tensor, bias: torch.Tensor, out: torch.Tensor, k_cache: torch.Tensor,
             v_cache: torch.Tensor, *, tokens_per_seq: int = 0, positions: torch.Tensor | None = None) -> torch.Tensor:
    """The QKV projection (+ bias) into `out`, its key and value columns also stored into the [seq][head][pos][64]
    caches: row r is sequence r // tokens_per_seq at r % tokens_per_seq, or sequence r at positions[r]."""
    _check(a, torch.bfloat16, "a")
    _check(w_t, torch.bfloat16, "w_t")
    _check(out, torch.bfloat16, "out")
    m, k = a.shape
    seqs, heads, capacity, head = k_cache.shape
    _launch("tempo_gemm_qkv", a.data_ptr(), k, w_t.data_ptr(), k, bias.data_ptr(), out.data_ptr(), out.shape[1], m, k,
            k_cache.data_ptr(), v_cache.data_ptr(), seqs, heads, head, capacity, tokens_per_seq, _ptr(positions),
            _stream())
    return out


def gemm_ln(x: torch.Tensor, w_folded: torch.Tensor, colsum: torch.Tensor, bias_folded: torch.Tensor, *,
            epsilon: float = 1e-5, gelu: bool = False, out: torch.Tensor | None = None,
            k_cache: torch.Tensor | None = None, v_cache: torch.Tensor | None = None,
            positions: torch.Tensor | None = None) -> torch.Tensor:
    """out = epilogue(LayerNorm(x) @ W + b) with the LayerNorm folded into the weights: w_folded[N, K] = (gamma * W)^T
    in BF16, colsum[N] = its FP32 row sums, bias_folded[N] = b + beta @ W in FP32; the row statistics are computed in
    the kernel. With the caches (and positions) the key and value columns are also stored, as in gemm_qkv decode."""
    _check(x, torch.bfloat16, "x")
    _check(w_folded, torch.bfloat16, "w_folded")
    _check(colsum, torch.float32, "colsum")
    _check(bias_folded, torch.float32, "bias_folded")
    m, k = x.shape
    n = w_folded.shape[0]
    if w_folded.shape[1] != k:
        raise ValueError(f"inner dimensions differ: x {tuple(x.shape)}, w_folded {tuple(w_folded.shape)}")
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=x.device)
    _check(out, torch.bfloat16, "out")
    seqs = heads = head = capacity = 0
    if k_cache is not None:
        seqs, heads, capacity, head = k_cache.shape
    _launch("tempo_gemm_ln", x.data_ptr(), k, w_folded.data_ptr(), k, colsum.data_ptr(), bias_folded.data_ptr(),
            float(epsilon), out.data_ptr(), out.shape[1], m, n, k, _lib.GEMM_GELU if gelu else 0, _ptr(k_cache),
            _ptr(v_cache), seqs, heads, head, capacity, _ptr(positions), _stream())
    return out


def gemm_rowstats(a: torch.Tensor, w_t: torch.Tensor, row_stats: torch.Tensor, *, bias: torch.Tensor | None = None,
                  residual: torch.Tensor | None = None, gelu: bool = False,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """gemm that also writes the statistics partials of its BF16 output rows into row_stats [M, N / 16, 2] (FP32
    mean and M2 of each 16-column chunk), for the folded LayerNorm of the projection that reads those rows next."""
    _check(a, torch.bfloat16, "a")
    _check(w_t, torch.bfloat16, "w_t")
    _check(row_stats, torch.float32, "row_stats")
    m, k = a.shape
    n = w_t.shape[0]
    if w_t.shape[1] != k:
        raise ValueError(f"inner dimensions differ: a {tuple(a.shape)}, w_t {tuple(w_t.shape)}")
    if row_stats.numel() < m * n // 8:
        raise ValueError(f"row_stats holds {row_stats.numel()} floats, {m * n // 8} needed")
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=a.device)
    _check(out, torch.bfloat16, "out")
    _launch("tempo_gemm_rowstats", a.data_ptr(), k, w_t.data_ptr(), k, _ptr(bias), _ptr(residual), n, out.data_ptr(),
            n, m, n, k, _lib.GEMM_GELU if gelu else 0, row_stats.data_ptr(), _stream())
    return out


def gemm_ln_rowstats(x: torch.Tensor, w_folded: torch.Tensor, colsum: torch.Tensor, bias_folded: torch.Tensor,
                     row_stats: torch.Tensor, *, epsilon: float = 1e-5, gelu: bool = False,
                     out: torch.Tensor | None = None, k_cache: torch.Tensor | None = None,
                     v_cache: torch.Tensor | None = None, positions: torch.Tensor | None = None) -> torch.Tensor:
    """gemm_ln with the rows' statistics combined from row_stats [M, K / 16, 2] (gemm_rowstats' or row_stats'
    partials of x) instead of computed in the kernel."""
    _check(x, torch.bfloat16, "x")
    _check(w_folded, torch.bfloat16, "w_folded")
    _check(colsum, torch.float32, "colsum")
    _check(bias_folded, torch.float32, "bias_folded")
    _check(row_stats, torch.float32, "row_stats")
    m, k = x.shape
    n = w_folded.shape[0]
    if w_folded.shape[1] != k:
        raise ValueError(f"inner dimensions differ: x {tuple(x.shape)}, w_folded {tuple(w_folded.shape)}")
    if row_stats.numel() < m * k // 8:
        raise ValueError(f"row_stats holds {row_stats.numel()} floats, {m * k // 8} needed")
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=x.device)
    _check(out, torch.bfloat16, "out")
    seqs = heads = head = capacity = 0
    if k_cache is not None:
        seqs, heads, capacity, head = k_cache.shape
    _launch("tempo_gemm_ln_rowstats", x.data_ptr(), k, w_folded.data_ptr(), k, colsum.data_ptr(),
            bias_folded.data_ptr(), float(epsilon), row_stats.data_ptr(), out.data_ptr(), out.shape[1], m, n, k,
            _lib.GEMM_GELU if gelu else 0, _ptr(k_cache), _ptr(v_cache), seqs, heads, head, capacity,
            _ptr(positions), _stream())
    return out


def row_stats(x: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    """The statistics partials of x's rows ([M, K / 16, 2] FP32 into `out`), as gemm_rowstats writes them."""
    _check(x, torch.bfloat16, "x")
    _check(out, torch.float32, "out")
    m, k = x.shape
    if out.numel() < m * k // 8:
        raise ValueError(f"out holds {out.numel()} floats, {m * k // 8} needed")
    _launch("tempo_row_stats", x.data_ptr(), x.stride(0), m, k, out.data_ptr(), _stream())
    return out


def gemm_norm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, w_t: torch.Tensor, *, epsilon: float = 1e-5,
              bias: torch.Tensor | None = None, gelu: bool = False, out: torch.Tensor | None = None,
              k_cache: torch.Tensor | None = None, v_cache: torch.Tensor | None = None,
              positions: torch.Tensor | None = None, part_val: torch.Tensor | None = None,
              part_idx: torch.Tensor | None = None) -> torch.Tensor | None:
    """LayerNorm(x) then the projection, one launch for at most 8 rows: the bits of layernorm() followed by gemm()
    (gemm_qkv with the caches and positions; gemm_argmax with the partial buffers, returning None)."""
    _check(x, torch.bfloat16, "x")
    _check(w_t, torch.bfloat16, "w_t")
    m, k = x.shape
    n = w_t.shape[0]
    if w_t.shape[1] != k:
        raise ValueError(f"inner dimensions differ: x {tuple(x.shape)}, w_t {tuple(w_t.shape)}")
    argmax = part_val is not None
    if not argmax and out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=x.device)
    heads = head = capacity = 0
    if k_cache is not None:
        _, heads, capacity, head = k_cache.shape
    flags = _lib.GEMM_ARGMAX if argmax else (_lib.GEMM_GELU if gelu else 0)
    _launch("tempo_gemm_norm", x.data_ptr(), x.stride(0), gamma.data_ptr(), beta.data_ptr(), float(epsilon),
            w_t.data_ptr(), w_t.stride(0), _ptr(bias), _ptr(out), out.stride(0) if out is not None else n, m, n, k,
            flags, _ptr(part_val), _ptr(part_idx), _ptr(k_cache), _ptr(v_cache), heads, head, capacity,
            _ptr(positions), _stream())
    return None if argmax else out


def gemm_argmax(a: torch.Tensor, w_t: torch.Tensor, part_val: torch.Tensor, part_idx: torch.Tensor) -> None:
    """Per-row (max, first argmax) of a @ w_t^T over each 256-column tile into the partial buffers [M, ceil(N/256)]."""
    _check(a, torch.bfloat16, "a")
    _check(w_t, torch.bfloat16, "w_t")
    m, k = a.shape
    n = w_t.shape[0]
    _launch("tempo_gemm", a.data_ptr(), k, w_t.data_ptr(), k, None, None, n, None, n, m, n, k, _lib.GEMM_ARGMAX,
              part_val.data_ptr(), part_idx.data_ptr(), _stream())


def decode_step_workspace_bytes(rows: int, width: int, heads: int, vocab: int) -> int:
    size = ctypes.c_uint64()
    _lib.call("tempo_decode_step_workspace", rows, width, heads, vocab, ctypes.byref(size))
    return int(size.value)


def decode_step(args: "_lib.DecodeStepArgs") -> None:
    """One persistent decode step (tempo_decode_step) with prepared arguments, on the current stream."""
    _launch("tempo_decode_step", ctypes.byref(args), _stream())


def argmax_finish(part_val: torch.Tensor, part_idx: torch.Tensor, ids: torch.Tensor, *,
                  tokens_out: torch.Tensor | None = None, positions: torch.Tensor | None = None,
                  index_offset: int = 0, advance: int = 0) -> None:
    """ids = per-row argmax; tokens_out[r, positions[r] + index_offset] = ids[r]; positions += advance."""
    rows, tiles = part_val.shape
    stride = tokens_out.shape[1] if tokens_out is not None else 0
    _launch("tempo_argmax_finish", part_val.data_ptr(), part_idx.data_ptr(), rows, tiles, ids.data_ptr(),
              _ptr(tokens_out), stride, _ptr(positions), index_offset, advance, _stream())


def layernorm(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, *, epsilon: float = 1e-5,
              out: torch.Tensor | None = None, rows: int | None = None, row_stride: int | None = None) -> torch.Tensor:
    """LayerNorm of `rows` rows of x read `row_stride` elements apart (default: every row of a contiguous x)."""
    if not x.is_cuda or x.dtype != torch.bfloat16:
        raise ValueError("x must be a CUDA bfloat16 tensor")
    features = x.shape[-1]
    rows = x.numel() // features if rows is None else rows
    row_stride = features if row_stride is None else row_stride
    if out is None:
        out = torch.empty((rows, features), dtype=torch.bfloat16, device=x.device)
    _launch("tempo_layernorm", x.data_ptr(), row_stride, gamma.data_ptr(), beta.data_ptr(), out.data_ptr(), rows,
              features, float(epsilon), _stream())
    return out


def embed(ids: torch.Tensor, positions: torch.Tensor, wte: torch.Tensor, wpe: torch.Tensor, *,
          out: torch.Tensor | None = None) -> torch.Tensor:
    _check(ids, torch.int32, "ids")
    _check(positions, torch.int32, "positions")
    rows, width = ids.numel(), wte.shape[1]
    if out is None:
        out = torch.empty((rows, width), dtype=torch.bfloat16, device=wte.device)
    _launch("tempo_embed", ids.data_ptr(), positions.data_ptr(), wte.data_ptr(), wpe.data_ptr(), out.data_ptr(), rows,
              width, wte.shape[0], wpe.shape[0], _stream())
    return out


def attention_prefill(qkv: torch.Tensor, seqs: int, tokens: int, heads: int, *,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    _check(qkv, torch.bfloat16, "qkv")
    width = qkv.shape[1] // 3
    if out is None:
        out = torch.empty((seqs * tokens, width), dtype=torch.bfloat16, device=qkv.device)
    _launch("tempo_attention_prefill", qkv.data_ptr(), out.data_ptr(), seqs, tokens, heads, width // heads, _stream())
    return out


def kv_store(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, seq_of: torch.Tensor,
             pos_of: torch.Tensor) -> None:
    seqs, heads, capacity, head = k_cache.shape
    _launch("tempo_kv_store", qkv.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), seq_of.data_ptr(),
              pos_of.data_ptr(), seq_of.numel(), seqs, heads, head, capacity, _stream())


def decode_attention(qkv: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, lengths: torch.Tensor, *,
                     length_offset: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    seqs, heads, capacity, head = k_cache.shape
    if out is None:
        out = torch.empty((seqs, heads * head), dtype=torch.bfloat16, device=qkv.device)
    _launch("tempo_decode_attention", qkv.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), lengths.data_ptr(),
              length_offset, out.data_ptr(), seqs, heads, head, capacity, _stream())
    return out


# ---- the 4-bit key / value cache ----

def kv_cache_q4(seqs: int, kv_heads: int, capacity: int, head: int = 64, *,
                device: torch.device | str = "cuda") -> torch.Tensor:
    """An empty 4-bit cache, [seqs, kv_heads, ceil(capacity / 16), 1152 * head / 64] uint8 (include/tempo_b200.h has
    the layout): `capacity` positions, rounded up to whole tiles of 16, at 72 bytes per position, head and 64
    dimensions. A slice of its sequences is a cache too."""
    if head not in (64, 128):
        raise ValueError(f"the 4-bit cache holds heads of 64 or 128 dimensions, got {head}")
    if seqs <= 0 or kv_heads <= 0 or capacity <= 0:
        raise ValueError(f"a cache needs sequences, heads and positions, got {seqs}, {kv_heads}, {capacity}")
    tiles = (capacity + _lib.Q4_TILE - 1) // _lib.Q4_TILE
    return torch.zeros((seqs, kv_heads, tiles, _lib.Q4_BLOCK_BYTES * head // 64), dtype=torch.uint8, device=device)


def _q4_shape(cache: torch.Tensor, device: int) -> tuple[int, int, int, int]:
    """(seqs, kv_heads, head, capacity) of a 4-bit cache."""
    _operand(cache, torch.uint8, "cache", device)
    if device < 0:
        raise ValueError("cache must be a CUDA tensor: the B200 kernels have no CPU path")
    if cache.dim() == 4:
        seqs, kv_heads, tiles, size = cache.shape
        if size == _lib.Q4_BLOCK_BYTES or size == 2 * _lib.Q4_BLOCK_BYTES:
            return seqs, kv_heads, 64 if size == _lib.Q4_BLOCK_BYTES else 128, tiles * _lib.Q4_TILE
    raise ValueError(f"cache must be [seqs, kv_heads, tiles, 1152 or 2304] as kv_cache_q4 makes it, got "
                     f"{tuple(cache.shape)}")


def _places(rows: int, seq_of: torch.Tensor, pos_of: torch.Tensor, device: int) -> None:
    _operand(seq_of, torch.int32, "seq_of", device)
    _operand(pos_of, torch.int32, "pos_of", device)
    if seq_of.numel() != rows or pos_of.numel() != rows:
        raise ValueError(f"{rows} rows need as many sequences and positions, got {seq_of.numel()} and {pos_of.numel()}")


def kv_store_q4(qkv: torch.Tensor, cache: torch.Tensor, seq_of: torch.Tensor, pos_of: torch.Tensor) -> None:
    """kv_store into a 4-bit cache: the key and value columns of row r of qkv ([rows, (heads + 2 kv_heads) * head],
    at any row stride that is a multiple of 8; no query columns are needed) quantised into sequence seq_of[r] at
    position pos_of[r]. Rows outside the cache are skipped; the others must name different places."""
    rows, width, stride, device = _matrix(qkv, torch.bfloat16, "qkv")
    seqs, kv_heads, head, capacity = _q4_shape(cache, device)
    heads = width // head - 2 * kv_heads
    if width % head or heads < 0:
        raise ValueError(f"qkv rows of {width} are not query, key and value heads of {head} ({kv_heads} key heads)")
    _places(rows, seq_of, pos_of, device)
    _launch_at(device, "tempo_kv_store_q4", qkv.data_ptr(), _stride32(stride, "qkv"), cache.data_ptr(),
               seq_of.data_ptr(), pos_of.data_ptr(), rows, seqs, heads, kv_heads, head, capacity)


def kv_load_q4(cache: torch.Tensor, seq_of: torch.Tensor, pos_of: torch.Tensor, *,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """The keys and values a 4-bit cache holds at the given places, [rows, 2 kv_heads * head] BF16 (kv_store_q4 takes
    them back). Places outside the cache give zeros."""
    device = cache.get_device()
    seqs, kv_heads, head, capacity = _q4_shape(cache, device)
    rows, width = pos_of.numel(), 2 * kv_heads * head
    _places(rows, seq_of, pos_of, device)
    stride = width
    if out is None:
        out = cache.new_empty((rows, width), dtype=torch.bfloat16)
    else:
        out_rows, out_width, stride, _ = _matrix(out, torch.bfloat16, "out", device)
        if out_rows != rows or out_width != width:
            raise ValueError(f"out must be {(rows, width)}, got {tuple(out.shape)}")
    _launch_at(device, "tempo_kv_load_q4", cache.data_ptr(), out.data_ptr(), _stride32(stride, "out"),
               seq_of.data_ptr(), pos_of.data_ptr(), rows, seqs, kv_heads, head, capacity)
    return out


@functools.lru_cache(maxsize=1024)
def decode_attention_q4_workspace_bytes(seqs: int, heads: int, kv_heads: int, head: int, capacity: int) -> int:
    """Bytes of workspace a decode_attention_q4 call of these sizes needs (0 for most)."""
    size = ctypes.c_uint64()
    _lib.call("tempo_decode_attention_q4_workspace", seqs, heads, kv_heads, head, capacity, ctypes.byref(size))
    return int(size.value)


def decode_attention_q4(qkv: torch.Tensor, cache: torch.Tensor, lengths: torch.Tensor, *, length_offset: int = 0,
                        heads: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """decode_attention over a 4-bit cache: the query columns of row s of qkv (scaled by 1/sqrt(head)) over the first
    lengths[s] + length_offset positions of sequence s; a sequence without positions gives zeros. The row holds query,
    key and value heads, unless `heads` says how many query heads it begins with."""
    rows, width, stride, device = _matrix(qkv, torch.bfloat16, "qkv")
    seqs, kv_heads, head, capacity = _q4_shape(cache, device)
    _operand(lengths, torch.int32, "lengths", device)
    if heads is None:
        heads = width // head - 2 * kv_heads
    if width % head or heads <= 0 or heads % kv_heads or heads * head > width:
        raise ValueError(f"qkv rows of {width} do not begin with {heads} query heads of {head}, a multiple of "
                         f"{kv_heads} key heads")
    if rows != seqs or lengths.numel() != seqs:
        raise ValueError(f"{seqs} sequences need a query row and a length each, got {rows} and {lengths.numel()}")
    if out is None:
        out = qkv.new_empty((seqs, heads * head))
    else:
        _operand(out, torch.bfloat16, "out", device)
        if out.shape != (seqs, heads * head):
            raise ValueError(f"out must be {(seqs, heads * head)}, got {tuple(out.shape)}")
    size = decode_attention_q4_workspace_bytes(seqs, heads, kv_heads, head, capacity)
    workspace = qkv.new_empty(size, dtype=torch.uint8) if size else None
    _launch_at(device, "tempo_decode_attention_q4", qkv.data_ptr(), _stride32(stride, "qkv"), cache.data_ptr(),
               lengths.data_ptr(), _int32(length_offset, "length_offset"), out.data_ptr(), seqs, heads, kv_heads, head,
               capacity, _ptr(workspace), size)
    return out


# ---- scores of logits ----

class TokenScores(NamedTuple):
    """Per row: the given token's log probability and the entropy [rows]; the alternatives' log probabilities and ids
    [rows, top], likeliest first (absent from the tuple's values when top is 0)."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_logprob: torch.Tensor | None = None
    top_ids: torch.Tensor | None = None


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, *, top: int = 0, out: TokenScores | None = None,
                   slots: torch.Tensor | None = None, slot_offset: int = 0) -> TokenScores:
    """Log probabilities of ids[r] under softmax(logits[r]) (FP32 or BF16 rows at any stride), the rows' entropies in
    nats and their `top` (at most 32) likeliest tokens, ties to the lower id. A row whose id is outside the vocabulary
    (a padded row) scores 0; include/tempo_b200.h says what infinities and NaN give. With `slots` (int32, one a row)
    the tensors of `out` have a leading dimension, and row r's results go to its index slots[r] + slot_offset, or
    nowhere when that is outside: one captured call serves every step."""
    bf16 = logits.dtype is torch.bfloat16
    rows, vocab, stride, device = _matrix(logits, torch.bfloat16 if bf16 else torch.float32, "logits")
    _operand(ids, torch.int32, "ids", device)
    if ids.numel() != rows:
        raise ValueError(f"{rows} rows need as many ids, got {ids.numel()}")
    if top and not 0 < top <= min(32, vocab):
        raise ValueError(f"top must be in [0, {min(32, vocab)}], got {top}")
    blocks = 0
    if out is None:
        if slots is not None:
            raise ValueError("slots need the outputs they index")
        # one allocation, split
        if top:
            words = logits.new_empty(2 * rows * (1 + top), dtype=torch.float32)
            logprob, entropy, best, order = words.split((rows, rows, rows * top, rows * top))
            top_logprob, top_ids = best.view(rows, top), order.view(torch.int32).view(rows, top)
        else:
            logprob, entropy = logits.new_empty((2, rows), dtype=torch.float32).unbind()
            top_logprob = top_ids = None
        out = TokenScores(logprob, entropy, top_logprob, top_ids)
    else:
        lead = ()
        if slots is not None:
            _operand(slots, torch.int32, "slots", device)
            if slots.numel() != rows:
                raise ValueError(f"{rows} rows need as many slots, got {slots.numel()}")
            blocks = out.logprob.shape[0]
            lead = (blocks,)
        for name, t, shape, dtype in (("logprob", out.logprob, (*lead, rows), torch.float32),
                                      ("entropy", out.entropy, (*lead, rows), torch.float32),
                                      ("top_logprob", out.top_logprob, (*lead, rows, top), torch.float32),
                                      ("top_ids", out.top_ids, (*lead, rows, top), torch.int32)):
            if name.startswith("top") and not top:
                continue
            if t is None:
                raise ValueError(f"out.{name} is needed for {top} alternatives")
            _operand(t, dtype, f"out.{name}", device)
            if t.shape != shape:
                raise ValueError(f"out.{name} must be {shape}, got {tuple(t.shape)}")
    _launch_at(device, "tempo_token_logprobs", logits.data_ptr(), stride, int(bf16), ids.data_ptr(), rows, vocab, top,
               out.logprob.data_ptr(), out.entropy.data_ptr(), _ptr(out.top_logprob), _ptr(out.top_ids), _ptr(slots),
               _int32(slot_offset, "slot_offset"), blocks)
    return out


# ---- the packed per-block ops on raw device tensors (uint16 words) ----

def block_gemm(activations: torch.Tensor, weights: torch.Tensor, drain: torch.Tensor, bias: torch.Tensor | None,
               depth: int, columns: int, activate: bool) -> None:
    _launch("tempo_block_gemm", activations.data_ptr(), weights.data_ptr(), drain.data_ptr(), _ptr(bias), depth,
              columns, int(activate), _stream())


def block_add(left: torch.Tensor, right: torch.Tensor, out: torch.Tensor, features: int, broadcast: bool) -> None:
    _launch("tempo_block_add", left.data_ptr(), right.data_ptr(), out.data_ptr(), features, int(broadcast), _stream())


def block_layernorm(rows: torch.Tensor, constants: torch.Tensor, out: torch.Tensor, features: int) -> None:
    _launch("tempo_block_layernorm", rows.data_ptr(), constants.data_ptr(), out.data_ptr(), features, _stream())


def block_attention(constants: torch.Tensor, fused_operand: int, tokens: int, heads: int) -> None:
    _launch("tempo_block_attention", constants.data_ptr(), fused_operand, tokens, heads, 64, _stream())


def block_decode_attention(constants: torch.Tensor, cache_operand: int, fused_operand: int, keys: int, heads: int,
                           stated: int = 0) -> None:
    _launch("tempo_block_decode_attention", constants.data_ptr(), cache_operand, fused_operand, keys, heads, 64,
              stated, _stream())


def block_copy(source: int, destination: int, rows: int, stride: int) -> None:
    _launch("tempo_block_copy", source, destination, rows, stride, _stream())


def watchdog() -> int:
    """Reads and clears the kernels' bounded-wait watchdog (0 = no wait expired)."""
    import ctypes
    code = ctypes.c_int32()
    _lib.call("tempo_watchdog", ctypes.byref(code))
    return int(code.value)


def stream_read(src: torch.Tensor, sink: torch.Tensor | None = None) -> torch.Tensor:
    """Calibration: streams `src` (a contiguous device tensor) once through the HBM read path; returns the sink the
    kernel folds it into. Its rate is the read ceiling of the bandwidth-bound kernels."""
    if not src.is_contiguous():
        raise ValueError("stream_read needs a contiguous source")
    threads = ctypes.c_uint32()
    _lib.call("tempo_stream_read_threads", ctypes.byref(threads))
    if sink is None:
        sink = torch.empty(threads.value * 16, dtype=torch.uint8, device=src.device)
    elif sink.numel() * sink.element_size() < threads.value * 16:
        raise ValueError("stream_read sink too small")
    _launch("tempo_stream_read", src.data_ptr(), src.numel() * src.element_size(), sink.data_ptr(), _stream())
    return sink

