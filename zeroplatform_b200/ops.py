"""Host-side mirror of the reference operators on the quantized-linear + paged-KV path.

Names and argument meaning follow the reference (kzxl/ZeroPlatform):

* ``QuantizedKernels.mat_vec_mul_q8_0 / mat_vec_add_q8_0 / ..._q4_0`` --
  ZeroLlm/src/ZeroLlm.Core/Quantization/QuantizedKernels.cs:190-349 (y = W x, y += W x)
* ``TensorBlas.gemv_q8_0 / gemv_q4_0`` -- ZeroTensor/src/ZeroTensor.Core/TensorBlas.Quantized.cs:447-485
  (host arrays in, host array out; goes through the reference bridge ABI ``zc_gemv_*``)
* ``TensorOps.paged_attention`` -- ZeroTensor/src/ZeroTensor.Core/TensorOps.Neural.cs:2372-2476
* ``reserve_pages``, ``trim_pages``, ``append_kv``, ``sparse_paged_attention``, ``lora_add``, ``process_logits`` --
  one step of a mixed serving batch, its state on the device (no counterpart in the reference, whose page tables,
  histories and sampling rules are per call on the host)
* ``QuantizedWeight`` -- a weight uploaded once and kept in the device layout (the repack of the
  reference's BlockQ8_0 / BlockQ4_0 arrays, BlockQ8_0.cs:10-17, BlockQ4_0.cs:10-17).

Device tensors are torch CUDA tensors (PyTorch provides the memory and the stream); every compute
call goes through libzero_tensor.so.  Errors raise ZcError (the C# bridge instead falls back to its
managed code on a non-zero status).
"""
from __future__ import annotations

import math
from typing import NamedTuple

import numpy as np
import torch

import ctypes as C

from . import _lib
from ._lib import LogitsRules, ZcError, check, lib

QK = 32
Q8_BYTES = 34
Q4_BYTES = 18


def _stream(stream=None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _np_ptr(a: np.ndarray) -> int:
    assert a.flags["C_CONTIGUOUS"]
    return a.ctypes.data


def quantize(qtype: int, w: torch.Tensor, stream=None) -> torch.Tensor:
    """LlmQuantizer.QuantizeToQ8_0 / QuantizeToQ4_0 on the device: fp32 [..., cols] -> packed AoS blocks
    (uint8 [..., cols/32*34] or [..., cols/32*18]), bit-identical to the reference quantizer."""
    w = w.contiguous()
    if w.dtype != torch.float32 or w.shape[-1] % QK:
        raise ZcError("quantize expects fp32 with a last dimension that is a multiple of 32")
    bpb = Q8_BYTES if qtype == 8 else Q4_BYTES
    out = torch.empty(w.shape[:-1] + (w.shape[-1] // QK * bpb,), dtype=torch.uint8, device=w.device)
    fn = lib().zcu_quantize_q8_0 if qtype == 8 else lib().zcu_quantize_q4_0
    check(fn(w.data_ptr(), out.data_ptr(), w.numel(), _stream(stream)), "quantize")
    return out


class QuantizedWeight:
    """A Q8_0 or Q4_0 weight matrix [rows][cols] resident on the GPU in the SoA layout."""

    def __init__(self, qtype: int, qs: torch.Tensor, d: torch.Tensor, rows: int, cols: int):
        self.qtype, self.qs, self.d, self.rows, self.cols = qtype, qs, d, rows, cols

    @staticmethod
    def upload(qtype: int, blocks, rows: int, cols: int, device="cuda", stream=None) -> "QuantizedWeight":
        """Upload the reference's packed blocks (numpy uint8 or a torch uint8 tensor) and repack."""
        if cols % QK:
            raise ZcError("cols must be a multiple of 32")
        bpb = Q8_BYTES if qtype == 8 else Q4_BYTES
        nbytes = rows * (cols // QK) * bpb
        if isinstance(blocks, np.ndarray):
            aos = torch.from_numpy(np.ascontiguousarray(blocks).reshape(-1)[:nbytes]).to(device, non_blocking=False)
        else:
            aos = blocks.reshape(-1)[:nbytes].to(device).contiguous()
        if aos.numel() != nbytes:
            raise ZcError(f"expected {nbytes} bytes of blocks, got {aos.numel()}")
        if qtype == 8:
            qs = torch.empty((rows, cols), dtype=torch.int8, device=device)
            fn = lib().zcu_q8_0_repack
        else:
            qs = torch.empty((rows, cols // 2), dtype=torch.uint8, device=device)
            fn = lib().zcu_q4_0_repack
        d = torch.empty((rows, cols // QK), dtype=torch.int16, device=device)
        check(fn(aos.data_ptr(), qs.data_ptr(), d.data_ptr(), rows, cols, _stream(stream)), "repack")
        return QuantizedWeight(qtype, qs, d, rows, cols)

    @property
    def nbytes(self) -> int:
        return self.qs.numel() * self.qs.element_size() + self.d.numel() * 2

    def gemv(self, x: torch.Tensor, y: torch.Tensor | None = None, accumulate: bool = False, stream=None):
        if y is None:
            y = torch.empty(self.rows, dtype=torch.float32, device=x.device)
        fn = lib().zcu_gemv_q8_0 if self.qtype == 8 else lib().zcu_gemv_q4_0
        check(fn(self.qs.data_ptr(), self.d.data_ptr(), x.data_ptr(), y.data_ptr(), self.rows, self.cols,
                 int(accumulate), _stream(stream)), "gemv")
        return y


class QuantizedKernels:
    """QuantizedKernels (QuantizedKernels.cs) over device-resident weights."""

    @staticmethod
    def mat_vec_mul_q8_0(w: QuantizedWeight, x, y, rows, cols, stream=None):
        assert w.qtype == 8 and (rows, cols) == (w.rows, w.cols)
        return w.gemv(x, y, False, stream)

    @staticmethod
    def mat_vec_add_q8_0(w: QuantizedWeight, x, y, rows, cols, stream=None):
        assert w.qtype == 8 and (rows, cols) == (w.rows, w.cols)
        return w.gemv(x, y, True, stream)

    @staticmethod
    def mat_vec_mul_q4_0(w: QuantizedWeight, x, y, rows, cols, stream=None):
        assert w.qtype == 4 and (rows, cols) == (w.rows, w.cols)
        return w.gemv(x, y, False, stream)

    @staticmethod
    def mat_vec_add_q4_0(w: QuantizedWeight, x, y, rows, cols, stream=None):
        assert w.qtype == 4 and (rows, cols) == (w.rows, w.cols)
        return w.gemv(x, y, True, stream)


class TensorBlas:
    """TensorBlas.GemvQ8_0 / GemvQ4_0 (TensorBlas.Quantized.cs:447-485) through the bridge ABI."""

    @staticmethod
    def gemv_q8_0(activation: np.ndarray, packed_weights: np.ndarray, n_rows: int, k_cols: int) -> np.ndarray:
        x = np.ascontiguousarray(activation, dtype=np.float32)
        w = np.ascontiguousarray(packed_weights, dtype=np.uint8)
        y = np.empty(n_rows, dtype=np.float32)
        check(lib().zc_gemv_q8_0(_np_ptr(w), _np_ptr(x), _np_ptr(y), n_rows, k_cols), "zc_gemv_q8_0")
        return y

    @staticmethod
    def gemv_q4_0(activation: np.ndarray, packed_weights: np.ndarray, n_rows: int, k_cols: int) -> np.ndarray:
        x = np.ascontiguousarray(activation, dtype=np.float32)
        w = np.ascontiguousarray(packed_weights, dtype=np.uint8)
        y = np.empty(n_rows, dtype=np.float32)
        check(lib().zc_gemv_q4_0(_np_ptr(w), _np_ptr(x), _np_ptr(y), n_rows, k_cols), "zc_gemv_q4_0")
        return y


class TensorOps:
    @staticmethod
    def paged_attention(q, k_cache, v_cache, block_table, context_len: int, scale: float | None = None):
        """TensorOps.PagedAttention: q [hq, hd]; caches [num_blocks, block_size, hkv, hd] fp32.

        numpy inputs run through the bridge ABI (zc_paged_attention_f32, host memory); torch CUDA
        tensors run the device entry point on the current stream.
        """
        hq, hd = q.shape
        nb, bs, hkv, _ = k_cache.shape
        if scale is None:
            scale = float(np.float32(1.0) / np.float32(np.sqrt(np.float64(hd))))
        if isinstance(q, np.ndarray):
            qn = np.ascontiguousarray(q, dtype=np.float32)
            kn = np.ascontiguousarray(k_cache, dtype=np.float32)
            vn = np.ascontiguousarray(v_cache, dtype=np.float32)
            bt = np.ascontiguousarray(block_table, dtype=np.int32)
            out = np.empty_like(qn)
            check(lib().zc_paged_attention_f32(hq, hkv, hd, bs, context_len, scale, _np_ptr(qn), _np_ptr(kn),
                                               _np_ptr(vn), _np_ptr(bt) if bt.size else 0, _np_ptr(out)),
                  "zc_paged_attention_f32")
            return out
        dev = q.device
        bt = torch.as_tensor(np.asarray(block_table, dtype=np.int32)).to(dev) if not torch.is_tensor(
            block_table) else block_table.to(dev, torch.int32)
        ctx = torch.tensor([context_len], dtype=torch.int32, device=dev)
        out = torch.empty_like(q)
        kv_dtype = 1 if k_cache.dtype == torch.float16 else 0
        check(lib().zcu_paged_attention(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), kv_dtype,
                                        bt.data_ptr(), ctx.data_ptr(), out.data_ptr(), 1, hq, hkv, hd, bs,
                                        max(1, bt.numel()), nb, bs * hkv * hd, hkv * hd, hd, scale, context_len,
                                        _stream()), "zcu_paged_attention")
        return out


def paged_attention_batched(q, k_pool, v_pool, page_table, ctx_len, hkv: int, page_size: int, num_pages: int,
                            page_stride: int, slot_stride: int, head_stride: int, scale: float, max_ctx: int,
                            out=None, stream=None):
    """Device paged attention for a batch of sequences (GqaAttention.Forward per sequence).

    q [batch, hq, hd] fp32; k_pool/v_pool fp16 or fp32 device buffers addressed with the given element
    strides; page_table [batch, max_pages] int32; ctx_len [batch] int32, both on the device."""
    batch, hq, hd = q.shape
    if out is None:
        out = torch.empty_like(q)
    kv_dtype = 1 if k_pool.dtype == torch.float16 else 0
    check(lib().zcu_paged_attention(q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), kv_dtype,
                                    page_table.data_ptr(), ctx_len.data_ptr(), out.data_ptr(), batch, hq, hkv, hd,
                                    page_size, page_table.shape[1], num_pages, page_stride, slot_stride,
                                    head_stride, scale, max_ctx, _stream(stream)), "zcu_paged_attention")
    return out


class LlmSampler:
    """LlmSampler.Sample (ZeroLlm/src/ZeroLlm.Core/Sampling/LlmSampler.cs:21-172) on device logits."""

    @staticmethod
    def sample(logits: torch.Tensor, past=None, temperature=0.7, top_p=0.9, min_p=0.0, top_k=40,
               repetition_penalty=1.1, u=None, stream=None) -> torch.Tensor:
        """logits [rows][vocab] fp32 on the device (modified in place, as the reference modifies its span); past: a
        list of token sequences, one per row (or None); u [rows]: the draws standing for (float)random.NextDouble()
        (unused on the greedy branch).  Returns the tokens [rows] (int32, device)."""
        from ._lib import SamplingConfig
        lg = logits if logits.dim() == 2 else logits.view(1, -1)
        rows, vocab = lg.shape
        cfg = SamplingConfig(temperature, top_p, min_p, top_k, repetition_penalty)
        past_t = plen_t = None
        pcap = 0
        if past is not None:
            pcap = max(1, max(len(p) for p in past))
            buf = np.zeros((rows, pcap), np.int32)
            lens = np.zeros(rows, np.int32)
            for r, p in enumerate(past):
                buf[r, :len(p)] = p
                lens[r] = len(p)
            past_t, plen_t = torch.from_numpy(buf).to(lg.device), torch.from_numpy(lens).to(lg.device)
        u_t = None if u is None else torch.as_tensor(u, dtype=torch.float32, device=lg.device).reshape(rows)
        out = torch.empty(rows, dtype=torch.int32, device=lg.device)
        check(lib().zcu_sample(lg.data_ptr(), rows, vocab, _ptr(past_t), _ptr(plen_t), pcap, C.byref(cfg), _ptr(u_t),
                               out.data_ptr(), None, None, None, 0, _stream(stream)), "sample")
        return out


# ---- one step of a mixed serving batch (zcu_pages_*, zcu_append_kv, zcu_sparse_paged_attention, zcu_lora_add,
#      zcu_process_logits).  Each function first offers its arguments to _dispatch, which checks and calls in one step
#      (True: enqueued); what that declines goes through the checks and the ctypes call below it. ----

_FLOAT_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _call(fn, what: str, device: int, stream, *args):
    """fn(*args, stream) on CUDA device `device`, whichever is current; the stream defaults to that device's current one."""
    try:
        if device == torch._C._cuda_getDevice():
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device) if stream is None else stream.cuda_stream)
        else:
            with torch.cuda.device(device):
                rc = fn(*args, torch._C._cuda_getCurrentRawStream(device) if stream is None else stream.cuda_stream)
    except C.ArgumentError as e:  # a number of the wrong kind or beyond 32 bits
        raise ZcError(f"{what}: {e}") from None
    if rc:
        check(rc, what)


def _arg(what: str, t, dtype, device: int, shape=None):
    """The address of a contiguous tensor on that CUDA device, of that type and, if given, shape (None: NULL)."""
    if t is None:
        return None
    if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous() or \
            (shape is not None and t.shape != shape):
        raise ZcError(f"{what} must be a contiguous {dtype} tensor on cuda:{device}"
                      f"{'' if shape is None else f' of shape {tuple(shape)}'}, got {t.dtype} {tuple(t.shape)} "
                      f"on {t.device}")
    return t.data_ptr()


def _empty(shape, dtype, device, stream):
    """A new tensor that belongs to the stream the call runs on."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    with torch.cuda.stream(stream):
        return torch.empty(shape, dtype=dtype, device=device)


def _cuda(what: str, t) -> int:
    """The index of the CUDA device that a tensor is on."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise ZcError(f"{what} must be a CUDA tensor")
    return t.get_device()


def _pool_args(page_table, seq_len, free_pages, free_count, page_size):
    dev = _cuda("page_table", page_table)
    if page_table.dim() != 2 or free_pages.dim() != 1:
        raise ZcError("page_table must be [max_rows, max_pages] and free_pages [num_pages]")
    rows, cols = page_table.shape
    i = torch.int32
    return dev, (_arg("page_table", page_table, i, dev), _arg("seq_len", seq_len, i, dev, (rows,)),
                 _arg("free_pages", free_pages, i, dev), _arg("free_count", free_count, i, dev, (1,)), rows, cols,
                 free_pages.shape[0], page_size)


class PagePlan(NamedTuple):
    """What reserve_pages says of a step's tokens: start [batch + 1], slots int64 [tokens], positions, token_rows and
    ctx_len [tokens], granted [batch] (int32)."""

    start: torch.Tensor
    slots: torch.Tensor
    positions: torch.Tensor
    token_rows: torch.Tensor
    ctx_len: torch.Tensor
    granted: torch.Tensor

    @staticmethod
    def empty(batch: int, tokens: int, device="cuda", stream=None) -> "PagePlan":
        e = lambda n, t=torch.int32: _empty(n, t, device, stream)  # noqa: E731
        return PagePlan(e(batch + 1), e(tokens, torch.int64), e(tokens), e(tokens), e(tokens), e(batch))


def reserve_pages(page_table, seq_len, free_pages, free_count, n_new, page_size: int, rows=None, tokens=None, out=None,
                  stream=None) -> PagePlan:
    """Block tables and slot maps from request lengths, on the device (zcu_pages_reserve): request b adds n_new[b]
    tokens to table row rows[b] (None: row b) of the pool (page_table [max_rows, max_pages], seq_len [max_rows], the
    stack free_pages [num_pages] of *free_count ids; int32, updated in place).  The first request that finds too few pages
    and all behind it are refused, so those with the first claim come first.  `tokens` is the length of the step's
    token arrays (room behind the last token is padding), taken from `out` (a PagePlan to write to) when that is
    given."""
    if out is None:
        if tokens is None:
            raise ZcError("reserve_pages needs tokens, the length of the step's token arrays, or out")
        out = PagePlan.empty(n_new.shape[0], tokens, page_table.device, stream)
        tokens = None
    d = _lib.dispatch
    if d and stream is None and tokens is None and d.reserve_pages(page_table, seq_len, free_pages, free_count,
                                                                   page_size, n_new, rows, *out):
        return out if isinstance(out, PagePlan) else PagePlan(*out)
    dev, pool = _pool_args(page_table, seq_len, free_pages, free_count, page_size)
    batch = n_new.shape[0]
    start, slots, positions, token_rows, ctx_len, granted = out
    n = slots.shape[0]
    if tokens is not None and tokens != n:
        raise ZcError(f"out has room for {n} tokens, not {tokens}")
    i, at = torch.int32, (n,)
    _call(lib().zcu_pages_reserve, "reserve_pages", dev, stream, *pool, _arg("rows", rows, i, dev, (batch,)),
          _arg("n_new", n_new, i, dev, (batch,)), batch, n, _arg("start", start, i, dev, (batch + 1,)),
          _arg("slots", slots, torch.int64, dev, at), _arg("positions", positions, i, dev, at),
          _arg("token_rows", token_rows, i, dev, at), _arg("ctx_len", ctx_len, i, dev, at),
          _arg("granted", granted, i, dev, (batch,)))
    return out if isinstance(out, PagePlan) else PagePlan(*out)


def trim_pages(page_table, seq_len, free_pages, free_count, new_len, page_size: int, rows=None, stream=None) -> None:
    """Row rows[b] (None: row b) keeps min(new_len[b], its length) tokens; the pages behind them go back to the stack
    (zcu_pages_trim).  new_len 0 frees a sequence; a shorter one takes rejected drafts back."""
    d = _lib.dispatch
    if d and stream is None and d.trim_pages(page_table, seq_len, free_pages, free_count, page_size, new_len, rows):
        return
    dev, pool = _pool_args(page_table, seq_len, free_pages, free_count, page_size)
    batch = new_len.shape[0]
    _call(lib().zcu_pages_trim, "trim_pages", dev, stream, *pool, _arg("rows", rows, torch.int32, dev, (batch,)),
          _arg("new_len", new_len, torch.int32, dev, (batch,)), batch)


def _kv_pools(k_pool, v_pool, dev):
    """(dtype code, pages, hkv, page size, hd, page / slot / head stride) of pools [pages, hkv, page size, hd], any
    strides with contiguous heads; a [pages, page size, hkv, hd] pool is passed as pool.transpose(1, 2)."""
    shape, strides = k_pool.shape, k_pool.stride()
    if len(shape) != 4 or shape != v_pool.shape or strides != v_pool.stride():
        raise ZcError("k_pool and v_pool must be [pages, kv heads, page size, head size] with the same strides")
    if k_pool.dtype not in (torch.float32, torch.float16) or v_pool.dtype != k_pool.dtype:
        raise ZcError("k_pool and v_pool must be fp32 or fp16")
    if k_pool.get_device() != dev or v_pool.get_device() != dev or strides[3] != 1:
        raise ZcError(f"k_pool and v_pool must be on cuda:{dev} with contiguous heads")
    return _FLOAT_CODE[k_pool.dtype], *shape, strides[0], strides[2], strides[1]


def append_kv(k, v, slots, k_pool, v_pool, bounds=None, scales=None, stream=None) -> None:
    """Keys and values [tokens, hkv, hd] (fp32 or fp16; any token stride) into paged pools [pages, hkv, page size, hd]
    at slots [tokens] (int64; reserve_pages' slots, negative ones skipped; the tokens of one page in ascending slots with
    no other page's tokens between them).  bounds int8 [pages, hkv, 2, hd] and scales fp32 [pages, hkv] receive the 8-bit
    key bounds of the pages written, which sparse_paged_attention scores pages by (zcu_append_kv)."""
    d = _lib.dispatch
    if d and stream is None and d.append_kv(k, v, slots, k_pool, v_pool, bounds, scales):
        return
    dev = _cuda("k", k)
    code, pages, hkv, page, hd, sp, ss, sh = _kv_pools(k_pool, v_pool, dev)
    shape, ks, vs = k.shape, k.stride(), v.stride()
    if len(shape) != 3 or shape != v.shape or shape[1:] != (hkv, hd) or k.dtype != v.dtype or v.get_device() != dev:
        raise ZcError(f"k and v must both be [tokens, {hkv}, {hd}] of one type on one device")
    if k.dtype not in (torch.float32, torch.float16):
        raise ZcError("k and v must be fp32 or fp16")
    if ks[2] != 1 or vs[2] != 1 or (hkv > 1 and (ks[1] != hd or vs[1] != hd)):
        raise ZcError("the heads of k and v must be contiguous")
    tokens = shape[0]
    _call(lib().zcu_append_kv, "append_kv", dev, stream, k.data_ptr(), v.data_ptr(), _FLOAT_CODE[k.dtype], ks[0],
          vs[0], _arg("slots", slots, torch.int64, dev, (tokens,)), tokens, k_pool.data_ptr(),
          v_pool.data_ptr(), code, hkv, hd, page, pages, sp, ss, sh,
          _arg("bounds", bounds, torch.int8, dev, (pages, hkv, 2, hd)),
          _arg("scales", scales, torch.float32, dev, (pages, hkv)))


def sparse_paged_attention(q, k_pool, v_pool, bounds, scales, page_table, ctx_len, budget: int, rows=None, sink: int = 1,
                           recent: int = 1, scale=None, max_ctx=None, out=None, sel=None, stream=None):
    """Decode attention of q [batch, hq, hd] fp32 (any row stride) over the `budget` pages per query and KV head that
    the key bounds score highest, the first `sink` and last `recent` pages always among them
    (zcu_sparse_paged_attention).

    Pools [pages, hkv, page size, hd] and bounds / scales as append_kv keeps them; page_table [rows, max_pages] and
    ctx_len [batch] int32; query b reads table row rows[b] (None: b; reserve_pages' token_rows), so several queries of
    one sequence may share a row.  max_ctx bounds ctx_len (default: what the table holds).  Returns (out [batch, hq,
    hd], sel [batch, hkv, budget]: the chosen pages as indices into the table row, ascending, -1 behind them)."""
    d = _lib.dispatch
    if d and stream is None and out is not None and sel is not None and d.sparse_paged_attention(
            q, k_pool, v_pool, bounds, scales, page_table, ctx_len, budget, rows, sink, recent, scale, max_ctx, out,
            sel):
        return out, sel
    dev = _cuda("q", q)
    code, pages, hkv, page, hd, sp, ss, sh = _kv_pools(k_pool, v_pool, dev)
    shape, qs = q.shape, q.stride()
    if len(shape) != 3 or q.dtype is not torch.float32 or shape[2] != hd or \
            (q.numel() and (qs[2] != 1 or (shape[1] > 1 and qs[1] != hd))):
        raise ZcError(f"q must be [batch, hq, {hd}] fp32 with contiguous heads")
    batch, hq, _ = shape
    if page_table.dim() != 2:
        raise ZcError("page_table must be [rows, max_pages]")
    table_rows, max_pages = page_table.shape
    if scale is None:
        scale = 1.0 / math.sqrt(hd)
    if max_ctx is None:
        max_ctx = min(max_pages * page, (1 << 30) - page)
    i, f = torch.int32, torch.float32
    if out is None:
        out = _empty((batch, hq, hd), f, q.device, stream)
    if sel is None:
        sel = _empty((batch, hkv, budget), i, q.device, stream)
    _call(lib().zcu_sparse_paged_attention, "sparse_paged_attention", dev, stream, q.data_ptr(), qs[0],
          k_pool.data_ptr(), v_pool.data_ptr(), code, _arg("bounds", bounds, torch.int8, dev, (pages, hkv, 2, hd)),
          _arg("scales", scales, f, dev, (pages, hkv)), _arg("page_table", page_table, i, dev), table_rows,
          _arg("rows", rows, i, dev, (batch,)), _arg("ctx_len", ctx_len, i, dev, (batch,)),
          _arg("out", out, f, dev, (batch, hq, hd)), _arg("sel", sel, i, dev, (batch, hkv, budget)), batch, hq, hkv,
          hd, page, max_pages, pages, sp, ss, sh, scale, max_ctx, budget, sink, recent)
    return out, sel


def lora_add(y, x, a, b, adapter, ranks=None, scales=None, out=None, stream=None):
    """out[r] = y[r] + scales[e] * (x[r] a[e].T) b[e].T for e = adapter[r] (rows with an adapter outside the tensor: y[r]):
    each request's low-rank adapter beside a shared projection's output y (zcu_lora_add).

    x [rows, k], y [rows, n] fp32 (any row stride), a [adapters, rank, k], b [adapters, n, rank] fp32, fp16 or bf16,
    adapter [rows] int32; ranks [adapters] int32 for adapters that use fewer than rank, scales [adapters] fp32.  out
    defaults to y, in place."""
    if out is None:
        out = y
    d = _lib.dispatch
    if d and stream is None and d.lora_add(y, x, a, b, adapter, ranks, scales, out):
        return out
    dev = _cuda("y", y)
    if y.dim() != 2 or x.dim() != 2 or a.dim() != 3 or b.dim() != 3:
        raise ZcError("x and y must be matrices, a and b stacks of matrices")
    rows, n = y.shape
    na, rank, k = a.shape
    xs, ys, os = x.stride(), y.stride(), out.stride()
    for name, t, shape, st in (("x", x, (rows, k), xs), ("y", y, (rows, n), ys), ("out", out, (rows, n), os)):
        if t.shape != shape or t.dtype is not torch.float32 or t.get_device() != dev or (st[1] != 1 and t.numel()):
            raise ZcError(f"{name} must be {list(shape)} fp32 on cuda:{dev} with contiguous rows")
    if a.dtype not in _FLOAT_CODE:
        raise ZcError("a and b must be fp32, fp16 or bf16")
    i, f = torch.int32, torch.float32
    _call(lib().zcu_lora_add, "lora_add", dev, stream, x.data_ptr(), xs[0], y.data_ptr(), ys[0],
          out.data_ptr(), os[0], _arg("a", a, a.dtype, dev), _arg("b", b, a.dtype, dev, (na, n, rank)),
          _FLOAT_CODE[a.dtype], _arg("adapter", adapter, i, dev, (rows,)), _arg("ranks", ranks, i, dev, (na,)),
          _arg("scales", scales, f, dev, (na,)), rows, k, n, na, rank)
    return out


def process_logits(logits, out=None, past=None, past_len=None, prompt_len=None, past_rows=None, repetition=None,
                   frequency=None, presence=None, bias_start=None, bias_ids=None, bias=None, mask=None, mask_rows=None,
                   stream=None):
    """Per-request rules on logits [rows, vocab] (fp32, fp16 or bf16; any row stride) before LlmSampler.sample: penalties
    for the tokens of a history, biases, grammar masks (zcu_process_logits).  Writes fp32 to `out`, by default the
    logits themselves when these are fp32 and a new tensor otherwise, and returns it.

    past [n, cap], past_len [n], prompt_len [n]: histories, row past_rows[r] (None: r) for row r; repetition divides
    positive logits (multiplies others) of every token seen, frequency and presence are subtracted for the ones behind
    the prompt, each [rows] fp32.  bias_start [rows + 1], bias_ids, bias: each row's biased tokens.  mask [m, words]
    int32: bit t % 32 of word t / 32 allows token t; row r uses mask_rows[r] (None: r; outside: unmasked)."""
    if out is None and logits.dtype is torch.float32:
        out = logits
    d = _lib.dispatch
    if d and stream is None and out is not None and d.process_logits(
            logits, out, past, past_len, prompt_len, past_rows, repetition, frequency, presence, bias_start, bias_ids,
            bias, mask, mask_rows):
        return out
    dev = _cuda("logits", logits)
    code, xs = _FLOAT_CODE.get(logits.dtype), logits.stride()
    if len(xs) != 2 or code is None or (xs[1] != 1 and logits.numel()):
        raise ZcError("logits must be [rows, vocab] fp32, fp16 or bf16 with contiguous rows")
    rows, vocab = logits.shape
    if out is None:
        out = _empty((rows, vocab), torch.float32, logits.device, stream)
    os = out.stride()
    if out.shape != (rows, vocab) or out.dtype is not torch.float32 or out.get_device() != dev or \
            (os[1] != 1 and out.numel()):
        raise ZcError(f"out must be [{rows}, {vocab}] fp32 on cuda:{dev} with contiguous rows")
    i, f, at = torch.int32, torch.float32, (rows,)
    n, cap = (0, 0) if past is None else past.shape
    masks, words = (0, 0) if mask is None else mask.shape
    n_bias = 0 if bias is None else bias.shape[0]
    if max(n, cap, masks, n_bias) > 0x7fffffff:
        raise ZcError("past, mask and bias must have fewer than 2^31 rows and entries a row")
    if past is not None and past_rows is None and n < rows:
        raise ZcError(f"past has {n} rows for {rows} rows of logits and no past_rows")
    if (bias_start is None) != (bias is None) or (bias_ids is None) != (bias is None):
        raise ZcError("bias_start, bias_ids and bias go together")
    r = LogitsRules(_arg("past", past, i, dev), _arg("past_len", past_len, i, dev, (n,)),
                    _arg("prompt_len", prompt_len, i, dev, (n,)), _arg("past_rows", past_rows, i, dev, at), cap, n,
                    _arg("repetition", repetition, f, dev, at), _arg("frequency", frequency, f, dev, at),
                    _arg("presence", presence, f, dev, at), _arg("bias_start", bias_start, i, dev, (rows + 1,)),
                    _arg("bias_ids", bias_ids, i, dev, (n_bias,)), _arg("bias", bias, f, dev), n_bias, masks,
                    _arg("mask", mask, i, dev), _arg("mask_rows", mask_rows, i, dev, at), words)
    _call(lib().zcu_process_logits, "process_logits", dev, stream, logits.data_ptr(), code,
          xs[0], out.data_ptr(), os[0], rows, vocab, C.byref(r))
    return out
