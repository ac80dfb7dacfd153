"""Low-bit serving operators: a paged KV cache held in 4 bits, and projections in 8-bit
integers.  ``include/kvbp.h`` states the formats and the arithmetic.

* ``kv4_pool`` makes a pool of pages; ``kv4_append`` finishes the q/k/v rows (bias, q/k
  RMSNorm, RoPE) and stores K and V in 4 bits; ``kv4_attend`` is one token's attention over
  the pages with the per-slot eviction score; ``kv4_gather`` reads slots back as bf16.
* ``int8_quantize_rows`` rounds rows to 8 bits with a scale each (a token's activations, or a
  weight's output channels); ``int8_linear`` is the projection of bf16 rows by such a weight.

Every call enqueues on the current stream of its tensors' device, allocates what it returns
(and its workspace) from torch's caching allocator, and can be captured in a CUDA graph.
Arguments that do not fit raise ``ValueError``, those that the library itself refuses (outputs that
overlap inputs, a misaligned pool, sizes it does not support) ``capi.KVBPError``; problems found on the device (a slot or page
out of range) set bits of ``dev_err``, an int32 tensor of one element, when one is given.
"""

from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import capi
from .capi import check, lib

BLOCK = 2304  # bytes of 16 slots of one kv head (KVBP_KV4_BLOCK)
HEAD_DIM = 128
_SCALE = 1.0 / math.sqrt(HEAD_DIM)
_INT_MAX = 0x7FFFFFFF  # the library's sizes are 32-bit, and ctypes would drop the bits above
_U8, _I8, _I32, _F32, _BF16 = torch.uint8, torch.int8, torch.int32, torch.float32, torch.bfloat16
# the current stream's handle of a device index (torch.cuda.current_stream makes an object)
_raw_stream = torch._C._cuda_getCurrentRawStream


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, dev: torch.device, shape: tuple) -> None:
    """``t`` is a dense tensor of this type, device and shape."""
    if t.dtype is dtype and t.shape == shape and t.device == dev and t.is_contiguous():
        return
    if t.dtype is not dtype or t.device != dev:
        raise ValueError(f"{name} must be {dtype} on {dev}, got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"{name} must be contiguous")


def _fits(a: int, b: int = 0) -> None:
    if a > _INT_MAX or b > _INT_MAX:
        raise ValueError(f"a size or stride of {max(a, b)} does not fit the library's 32-bit sizes")


def _launch(fn, what: str, dev: torch.device, *args) -> None:
    """``fn(stream, *args)`` on the current stream of ``dev``, with ``dev`` as the current
    device."""
    if dev.type != "cuda":
        raise ValueError("the low-bit operators run on CUDA devices only")
    idx = dev.index
    if torch.cuda.current_device() == idx:
        status = fn(_raw_stream(idx), *args)
    else:
        with torch.cuda.device(idx):
            status = fn(_raw_stream(idx), *args)
    if status:
        check(status, what)


@lru_cache(maxsize=1024)
def _attn_workspace(B: int, hq: int, hkv: int, limit: int, score: bool) -> int:
    return lib().kvbp_kv4_attn_workspace(B, hq, hkv, limit, score)


@lru_cache(maxsize=1024)
def _linear_workspace(M: int, K: int) -> int:
    return lib().kvbp_int8_linear_workspace(M, K)


def kv4_pool(n_pages: int, n_kv_heads: int, page_size: int = 64, device=None) -> torch.Tensor:
    """A pool of ``n_pages`` zeroed pages: uint8 [n_pages, n_kv_heads, page_size / 16, 2304]."""
    if page_size <= 0 or page_size % 16:
        raise ValueError(f"page_size {page_size} is not a multiple of 16")
    if n_pages <= 0 or n_kv_heads <= 0:
        raise ValueError("n_pages and n_kv_heads must be > 0")
    return torch.zeros(n_pages, n_kv_heads, page_size // 16, BLOCK, dtype=_U8,
                       device=torch.device("cuda") if device is None else device)


def _pool(pool: torch.Tensor, table: torch.Tensor) -> tuple:
    """(pages, kv heads, page size, sequences, pages per sequence, device) after the checks."""
    shape, tshape, dev = pool.shape, table.shape, pool.device
    if len(shape) != 4 or len(tshape) != 2:
        raise ValueError("pool must be [pages, kv heads, blocks, 2304] and page_table [sequences, pages]")
    n_pages, hkv, per, _ = shape
    _need(pool, "pool", _U8, dev, (n_pages, hkv, per, BLOCK))
    _need(table, "page_table", _I32, dev, tshape)
    _fits(tshape[0], tshape[1] * (per * 16 or 1) + 64)  # slot numbers (the pool's sizes fit if its bytes do)
    return n_pages, hkv, per * 16, tshape[0], tshape[1], dev


def _rows(rows: int, B: int, seq: Optional[torch.Tensor], dev: torch.device) -> int:
    """Rows per sequence when no ``seq`` names each row's sequence."""
    if seq is not None:
        _need(seq, "seq", _I32, dev, (rows,))
        return 1
    if B == 0 or rows % B:
        raise ValueError(f"{rows} rows do not divide over {B} sequences: pass seq")
    return max(1, rows // B)


def kv4_append(pool: torch.Tensor, page_table: torch.Tensor, qkv: torch.Tensor, slots: torch.Tensor, *, n_heads: int,
               seq: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
               inv_freq: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
               q_out: Optional[torch.Tensor] = None, dev_err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Finish rows of the q/k/v projection and store their K and V in the 4-bit pages.

    ``qkv`` [rows, (n_heads + 2 kv_heads) * 128] bf16 (rows may be strided); row r goes to
    logical slot ``slots[r]`` (negative: not stored) of sequence ``seq[r]`` (default: the
    rows divide evenly over the page table's sequences).  The slots that one call stores for a
    sequence must differ: of two rows for one slot either's bytes may stay.  With ``inv_freq``
    [64] float32, q and k are rotated by ``positions[r]``.  Returns q [rows, n_heads, 128] bf16."""
    n_pages, hkv, page, B, width, dev = _pool(pool, page_table)
    if qkv.dtype is not _BF16 or qkv.device != dev or qkv.dim() != 2:
        raise ValueError("qkv must be a bfloat16 matrix on the pool's device")
    rows, cols = qkv.shape
    nh = n_heads + 2 * hkv
    if n_heads < 0 or cols != nh * HEAD_DIM:
        raise ValueError(f"qkv has {cols} columns, {n_heads} + 2 * {hkv} heads need {nh * HEAD_DIM}")
    ldq, step = qkv.stride()
    if rows <= 1:
        ldq = cols
    if rows and cols and (step != 1 or ldq < cols):
        raise ValueError("qkv's columns must be contiguous and its rows must not overlap")
    _fits(rows, ldq)
    _need(slots, "slots", _I32, dev, (rows,))
    per = _rows(rows, B, seq, dev)
    if (inv_freq is None) != (positions is None):
        raise ValueError("positions and inv_freq go together")
    if inv_freq is not None:
        _need(inv_freq, "inv_freq", _F32, dev, (HEAD_DIM // 2,))
        _need(positions, "positions", _I32, dev, (rows,))
    if bias is not None:
        _need(bias, "bias", _BF16, dev, (nh * HEAD_DIM,))
    if q_norm is not None:
        _need(q_norm, "q_norm", _BF16, dev, (HEAD_DIM,))
    if k_norm is not None:
        _need(k_norm, "k_norm", _BF16, dev, (HEAD_DIM,))
    if q_out is None:
        q_out = qkv.new_empty((rows, n_heads, HEAD_DIM))
    else:
        _need(q_out, "q_out", _BF16, dev, (rows, n_heads, HEAD_DIM))
    if dev_err is not None:
        _need(dev_err, "dev_err", _I32, dev, (1,))
    if rows == 0:
        return q_out
    if n_pages == 0 or width == 0 or hkv == 0 or page == 0:
        raise ValueError("the pool and the page table must not be empty")
    _launch(
        lib().kvbp_kv4_append, "kv4_append", dev, rows, per, _ptr(seq), B, n_heads, hkv, HEAD_DIM, page, n_pages, width,
        qkv.data_ptr(), ldq, _ptr(bias), _ptr(q_norm), _ptr(k_norm), eps,
        _ptr(inv_freq), _ptr(positions), slots.data_ptr(), page_table.data_ptr(), q_out.data_ptr() if n_heads else None,
        pool.data_ptr(), _ptr(dev_err),
    )
    return q_out


def kv4_gather(pool: torch.Tensor, page_table: torch.Tensor, slots: torch.Tensor, *,
               seq: Optional[torch.Tensor] = None, heads_first: bool = False,
               dev_err: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """K and V of the listed slots as the bf16 values their codes stand for: two tensors
    [rows, kv_heads, 128], or [kv_heads, rows, 128] (the prefill attention's layout) with
    ``heads_first``.  Rows of negative or out-of-range slots are zeros."""
    n_pages, hkv, page, B, width, dev = _pool(pool, page_table)
    rows = slots.numel()
    _need(slots, "slots", _I32, dev, (rows,))
    _fits(rows)
    per = _rows(rows, B, seq, dev)
    if dev_err is not None:
        _need(dev_err, "dev_err", _I32, dev, (1,))
    shape = (hkv, rows, HEAD_DIM) if heads_first else (rows, hkv, HEAD_DIM)
    k = torch.empty(shape, dtype=_BF16, device=dev)
    v = torch.empty_like(k)
    if rows == 0:
        return k, v
    if n_pages == 0 or width == 0 or hkv == 0 or page == 0:
        raise ValueError("the pool and the page table must not be empty")
    row_stride, head_stride = (HEAD_DIM, rows * HEAD_DIM) if heads_first else (hkv * HEAD_DIM, HEAD_DIM)
    _launch(
        lib().kvbp_kv4_gather, "kv4_gather", dev, rows, per, _ptr(seq), B, hkv, HEAD_DIM, page, n_pages, width,
        slots.data_ptr(), page_table.data_ptr(), pool.data_ptr(), k.data_ptr(), v.data_ptr(), row_stride, head_stride,
        _ptr(dev_err),
    )
    return k, v


def kv4_attend(pool: torch.Tensor, page_table: torch.Tensor, lens: torch.Tensor, q: torch.Tensor, *,
               slot_pos: Optional[torch.Tensor] = None, step_score: Optional[torch.Tensor] = None,
               scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
               dev_err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One token's attention per sequence: q [B, heads, 128] bf16 over the live slots
    s < lens[b] with slot_pos[b, s] >= 0 (all of them without ``slot_pos`` [B, S]).
    ``step_score`` [B, S] float32 is max-accumulated with every live slot's largest
    probability over the heads.  ``scale`` defaults to 1 / sqrt(128).  Returns out
    [B, heads, 128] bf16; a sequence without a live slot gives zeros."""
    n_pages, hkv, page, B, width, dev = _pool(pool, page_table)
    _need(lens, "lens", _I32, dev, (B,))
    hq = q.shape[1] if q.dim() == 3 else 0
    _need(q, "q", _BF16, dev, (B, hq, HEAD_DIM))
    if hkv == 0 or hq == 0 or hq % hkv or hq // hkv > 8:
        raise ValueError(f"{hq} query heads over {hkv} kv heads: whole groups of at most 8 are supported")
    S = 0
    if slot_pos is not None:
        S = slot_pos.shape[-1] if slot_pos.dim() else 0
        _need(slot_pos, "slot_pos", _I32, dev, (B, S))
    if step_score is not None:
        S = S if slot_pos is not None else step_score.shape[-1] if step_score.dim() else 0
        _need(step_score, "step_score", _F32, dev, (B, S))
    if out is None:
        out = torch.empty_like(q)
    else:
        _need(out, "out", _BF16, dev, (B, hq, HEAD_DIM))
    if dev_err is not None:
        _need(dev_err, "dev_err", _I32, dev, (1,))
    if B == 0:
        return out
    _fits(S, hq)
    if n_pages == 0 or width == 0 or page == 0 or ((slot_pos is not None or step_score is not None) and S == 0):
        raise ValueError("the pool, the page table, slot_pos and step_score must not be empty")
    limit = min(width * page, S) if S else width * page
    ws_bytes = _attn_workspace(B, hq, hkv, limit, step_score is not None)
    ws = pool.new_empty(ws_bytes) if ws_bytes else None  # short sequences need none
    _launch(
        lib().kvbp_kv4_attn, "kv4_attn", dev, B, hq, hkv, HEAD_DIM, page, n_pages, width, q.data_ptr(), pool.data_ptr(),
        page_table.data_ptr(), lens.data_ptr(), _ptr(slot_pos), S, _SCALE if scale is None else scale, out.data_ptr(),
        _ptr(step_score), _ptr(ws), ws_bytes, _ptr(dev_err),
    )
    return out


def _matrix(x: torch.Tensor, name: str, dtype: torch.dtype) -> tuple:
    """(rows, columns, row stride) of a matrix with dense columns and rows apart."""
    if x.dtype is not dtype or x.dim() != 2:
        raise ValueError(f"{name} must be a {dtype} matrix")
    rows, cols = x.shape
    _fits(rows, cols)
    ld, step = x.stride()
    if rows <= 1:
        ld = cols
    if rows and cols and (step != 1 or ld < cols):
        raise ValueError(f"{name}'s columns must be contiguous and its rows must not overlap")
    return rows, cols, ld


def int8_quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of a bf16 matrix in 8 bits: codes int8 [rows, K] (a view of storage whose rows
    start on 16-byte boundaries, as ``int8_linear`` wants its weight) and scales float32
    [rows]; x is about codes * scale."""
    rows, K, ldx = _matrix(x, "x", _BF16)
    dev = x.device
    pitch = (K + 15) // 16 * 16
    q = torch.zeros(rows, pitch, dtype=_I8, device=dev) if pitch != K else torch.empty(
        rows, K, dtype=_I8, device=dev)
    s = torch.empty(rows, dtype=_F32, device=dev)
    if rows and K:
        _launch(lib().kvbp_int8_quant_rows, "int8_quant_rows", dev, rows, K, x.data_ptr(), ldx, q.data_ptr(),
                pitch, s.data_ptr())
    else:
        s.zero_()
    return q[:, :K], s


def int8_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                out_dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None,
                dev_err: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [M, K] bf16 times w [N, K] int8 (rows on 16-byte boundaries, scales w_scale [N]) plus
    bias [N] bf16: each row of x is rounded to 8 bits with its own scale, the sums are exact
    32-bit integers, and y = sum * x_scale * w_scale + bias is rounded once to ``out_dtype``
    (bfloat16 or float32)."""
    M, K, ldx = _matrix(x, "x", _BF16)
    N, Kw, ldw = _matrix(w, "w", _I8)
    dev, pitch = x.device, (K + 15) // 16 * 16
    if w.device != dev or Kw != K:
        raise ValueError(f"w must be [N, {K}] on {dev}, got {tuple(w.shape)} on {w.device}")
    if K == 0 or N == 0:
        raise ValueError("int8_linear needs at least one input and one output feature")
    if N == 1:
        ldw = pitch
    if ldw % 16 or w.data_ptr() % 16:
        raise ValueError("w's rows must start on 16-byte boundaries (int8_quantize_rows makes such weights)")
    _need(w_scale, "w_scale", _F32, dev, (N,))
    if bias is not None:
        _need(bias, "bias", _BF16, dev, (N,))
    if out_dtype is not _BF16 and out_dtype is not _F32:
        raise ValueError("out_dtype must be bfloat16 or float32")
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype, device=dev)
    else:
        _need(out, "out", out_dtype, dev, (M, N))
    if dev_err is not None:
        _need(dev_err, "dev_err", _I32, dev, (1,))
    if M == 0:
        return out
    ws_bytes = _linear_workspace(M, K)  # the codes and scales of x, unless it is one row
    ws = w.new_empty(ws_bytes) if ws_bytes else None
    _launch(lib().kvbp_int8_linear, "int8_linear", dev, out_dtype is _F32, M, N, K, w.data_ptr(), ldw,
            w_scale.data_ptr(), x.data_ptr(), ldx, _ptr(bias), out.data_ptr(), N, _ptr(ws), ws_bytes, _ptr(dev_err))
    return out
