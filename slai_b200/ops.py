"""Host-side mirror of slai's operator interface for the decode path, on top of the C ABI.

Names, argument order and error behaviour follow the Rust operators (`crates/slai/src/ops/*.rs`) and the
dispatcher `LlmContext` (`crates/slai/src/context.rs`); each class cites the interface it stands for.
Tensors are plain device buffers (`GpuVector`) holding f32; nothing here computes on the host.
"""
from __future__ import annotations

import ctypes as C
import enum

import numpy as np

from . import _lib
from ._lib import (AttnParams, SlaiError, FMT_F32, FMT_Q8_0, FMT_Q4_K, FMT_Q5_K, FMT_Q6_K, KV_F16, KV_F32)

_F32, _I32 = np.dtype(np.float32), np.dtype(np.int32)


class Backend:
    """The `B: Backend` of slang-hal as the decode path uses it: buffers, `write_buffer`, `read_buffer`,
    `synchronize` (call sites: crates/slai-chat/src/chat_llama2.rs:180-230).  One CUDA stream per backend."""

    _recording = False  # between a RecordedPass's enter and exit

    def __init__(self, device: int = 0):
        self.lib = _lib.load()
        h = C.c_void_p()
        rc = self.lib.slai_ctx_create(device, C.byref(h))
        if rc != 0:
            raise SlaiError(rc, (self.lib.slai_last_error_string(None) or b"").decode() or "cannot create a context")
        self.h = h
        self.device = device

    # -- errors ------------------------------------------------------------------------------------
    def check(self, rc: int):
        if rc != 0:
            raise SlaiError(rc, (self.lib.slai_last_error_string(self.h) or b"").decode())

    # -- buffers -----------------------------------------------------------------------------------
    def malloc(self, nbytes: int) -> int:
        p = C.c_void_p()
        self.check(self.lib.slai_malloc(self.h, nbytes, C.byref(p)))
        return p.value

    def free(self, ptr: int):
        if getattr(self, "_recording", False):
            self._deferred.append(ptr)  # a free would invalidate the recording (it synchronises the device)
            return
        self.check(self.lib.slai_free(self.h, C.c_void_p(ptr)))

    def write_buffer(self, dst: int, src: np.ndarray):
        src = np.ascontiguousarray(src)
        self.check(self.lib.slai_write_buffer(self.h, C.c_void_p(dst), src.ctypes.data_as(C.c_void_p), src.nbytes))
        self.synchronize()  # `src` may be a temporary

    def read_buffer(self, src: int, out: np.ndarray):
        assert out.flags["C_CONTIGUOUS"]
        self.check(self.lib.slai_read_buffer(self.h, out.ctypes.data_as(C.c_void_p), C.c_void_p(src), out.nbytes))
        return out

    def synchronize(self):
        self.check(self.lib.slai_ctx_sync(self.h))

    def vector(self, data, dtype=np.float32) -> "GpuVector":
        a = np.ascontiguousarray(data, dtype=dtype)
        v = GpuVector(self, a.size, dtype)
        self.write_buffer(v.ptr, a)
        return v

    def zeros(self, n: int, dtype=np.float32) -> "GpuVector":
        v = GpuVector(self, n, dtype)
        self.check(self.lib.slai_memset(self.h, C.c_void_p(v.ptr), 0, v.nbytes))
        return v

    def device_info(self):
        name = C.create_string_buffer(128)
        sms = C.c_int()
        self.check(self.lib.slai_ctx_device_info(self.h, name, 128, C.byref(sms)))
        return name.value.decode(), sms.value

    def mem_info(self):
        free, total = C.c_size_t(), C.c_size_t()
        self.check(self.lib.slai_ctx_mem_info(self.h, C.byref(free), C.byref(total)))
        return free.value, total.value

    def set_wait_limit(self, rounds: int):
        """Rounds a bounded device-side wait polls before it gives up (SLAI_ERR_TIMEOUT at the next synchronisation)."""
        self.check(self.lib.slai_ctx_set_wait_limit(self.h, rounds))

    def record(self) -> "RecordedPass":
        """Record the operator calls made inside the `with` block instead of running them (the reference's encoder:
        begin_pass ... submit, context.rs:63-96); replay with `.launch(times)`."""
        return RecordedPass(self)

    def timer_start(self):
        self.check(self.lib.slai_timer_start(self.h))

    def timer_stop(self) -> float:
        ms = C.c_float()
        self.check(self.lib.slai_timer_stop(self.h, C.byref(ms)))
        return ms.value

    def close(self):
        if getattr(self, "h", None):
            self.lib.slai_ctx_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class RecordedPass:
    def __init__(self, backend: "Backend"):
        self.backend = backend
        self.h = C.c_void_p()

    def __enter__(self):
        self.backend._deferred = []
        self.backend._deferred_handles = []
        self.backend._recording = True
        self.backend.check(self.backend.lib.slai_pass_begin(self.backend.h))
        return self

    def __exit__(self, et, ev, tb):
        rc = self.backend.lib.slai_pass_end(self.backend.h, C.byref(self.h))
        self.backend._recording = False
        for ptr in self.backend._deferred:  # buffers dropped by the garbage collector while recording
            self.backend.free(ptr)
        self.backend._deferred = []
        for destroy, h in self.backend._deferred_handles:  # ... and handles
            destroy(h)
        self.backend._deferred_handles = []
        if et is None:
            self.backend.check(rc)
        return False

    def launch(self, times: int = 1):
        self.backend.check(self.backend.lib.slai_pass_launch(self.backend.h, self.h, times))

    def close(self):
        if self.h:
            self.backend.lib.slai_pass_destroy(self.backend.h, self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class GpuVector:
    """`GpuVector<f32, B>` / `GpuTensor`: an owned device buffer (stensor, seen at context.rs:10-15)."""

    def __init__(self, backend: Backend, n: int, dtype=np.float32):
        self.backend = backend
        self.n = int(n)
        self.dtype = np.dtype(dtype)
        self.nbytes = self.n * self.dtype.itemsize
        self.ptr = backend.malloc(max(self.nbytes, 16))

    def __len__(self):
        return self.n

    def to_numpy(self) -> np.ndarray:
        out = np.empty(self.n, dtype=self.dtype)
        return self.backend.read_buffer(self.ptr, out)

    def view(self, offset: int, n: int) -> "GpuVectorView":
        assert 0 <= offset and offset + n <= self.n
        return GpuVectorView(self, offset, n)

    def __del__(self):
        try:
            if self.backend.h:
                self.backend.free(self.ptr)
        except Exception:
            pass


class GpuVectorView:
    """A contiguous sub-range of a `GpuVector` (`GpuTensorView`, e.g. `key_cache[l].column(pos)`)."""

    def __init__(self, base: GpuVector, offset: int, n: int):
        self.base, self.n = base, int(n)
        self.backend, self.dtype = base.backend, base.dtype
        self.ptr = base.ptr + offset * base.dtype.itemsize
        self.nbytes = self.n * base.dtype.itemsize

    def __len__(self):
        return self.n

    def to_numpy(self) -> np.ndarray:
        out = np.empty(self.n, dtype=self.dtype)
        return self.backend.read_buffer(self.ptr, out)


def _ptr(x) -> C.c_void_p:
    return C.c_void_p(x.ptr) if x is not None else C.c_void_p(None)


class GpuQuantMatrix:
    """`GpuQuantMatrix<B>` (crates/slai/src/quantized_matrix.rs:11-22) built like
    `GgufTensorData::to_gpu_matrix` (crates/slai/src/gguf.rs:133-194): raw GGUF blocks, row-major rows."""

    def __init__(self, backend: Backend, fmt: int, nrows: int, ncols: int, blocks: np.ndarray | None = None,
                 device_blocks: int | None = None, nbytes: int | None = None):
        self.backend = backend
        h = C.c_void_p()
        if blocks is not None:
            b = np.ascontiguousarray(blocks).view(np.uint8).reshape(-1)
            self._keep = b
            backend.check(backend.lib.slai_qmatrix_create(backend.h, fmt, nrows, ncols, b.ctypes.data_as(C.c_void_p), b.size,
                                                          C.byref(h)))
        else:
            backend.check(backend.lib.slai_qmatrix_create_from_device(backend.h, fmt, nrows, ncols, C.c_void_p(device_blocks),
                                                                      nbytes, C.byref(h)))
        self.h = h
        self.fmt, self.nrows, self.ncols = fmt, nrows, ncols

    @classmethod
    def synthetic(cls, backend: Backend, fmt: int, nrows: int, ncols: int, seed: int, std: float, keep_raw: bool = False):
        """Blocks quantised on the device from seeded N(0, std) values (model-sized benchmark inputs)."""
        from .synth import BLOCK_BYTES, BLOCK_ELEMS
        nbytes = nrows * (ncols // BLOCK_ELEMS[fmt]) * BLOCK_BYTES[fmt]
        raw = GpuVector(backend, nbytes, np.uint8)
        backend.check(backend.lib.slai_synth_blocks(backend.h, fmt, nrows, ncols, seed, std, C.c_void_p(raw.ptr)))
        m = cls(backend, fmt, nrows, ncols, device_blocks=raw.ptr, nbytes=nbytes)
        backend.synchronize()
        if keep_raw:
            m.raw = raw
        return m

    def shape(self):
        return (self.nrows, self.ncols)

    def device_bytes(self) -> int:
        return int(self.backend.lib.slai_qmatrix_device_bytes(self.h))

    def dequantize(self) -> np.ndarray:
        """Bit-exact `Block*::dequantize()` of every block, evaluated on the device."""
        out = GpuVector(self.backend, self.nrows * self.ncols)
        self.backend.check(self.backend.lib.slai_qmatrix_dequantize(self.backend.h, self.h, C.c_void_p(out.ptr)))
        return out.to_numpy().reshape(self.nrows, self.ncols)

    def dequantize_row(self, row: int) -> np.ndarray:
        out = GpuVector(self.backend, self.ncols)
        self.backend.check(self.backend.lib.slai_qmatrix_dequantize_row(self.backend.h, self.h, row, C.c_void_p(out.ptr)))
        return out.to_numpy()

    def __del__(self):
        try:
            if self.backend.h and self.h and not getattr(self.backend, "_recording", False):
                self.backend.lib.slai_qmatrix_destroy(self.h)
                self.h = None
        except Exception:
            pass


class RoPEVariant(enum.IntEnum):
    """crates/slai/src/ops/rope.rs:8-14"""
    Original = 0
    Neox = 1


class UnaryOp(enum.IntEnum):
    """crates/slai/src/ops/unary.rs:11-35 (same order)"""
    Abs = 0
    Sgn = 1
    Neg = 2
    Step = 3
    Elu = 4
    Gelu = 5
    GeluQuick = 6
    Silu = 7
    Tanh = 8
    Sin = 9
    Cos = 10
    Relu = 11
    Sigmoid = 12
    HardSigmoid = 13
    Sqr = 14
    Sqrt = 15
    Log = 16
    LeakyRelu = 17
    Clamp = 18
    Scale = 19
    AddScalar = 20


class BatchedMultiqueryAttentionParams:
    """crates/slai/src/ops/batched_multiquery_attention.rs:17-29"""

    def __init__(self, seq_len, kv_dim, kv_mul, n_heads, head_size, pos):
        self.seq_len, self.kv_dim, self.kv_mul, self.n_heads, self.head_size, self.pos = seq_len, kv_dim, kv_mul, n_heads, head_size, pos

    def to_c(self) -> AttnParams:
        return AttnParams(self.seq_len, self.kv_dim, self.kv_mul, self.n_heads, self.head_size, self.pos)


def _int32(what: str, x) -> np.ndarray:
    """x as int32 numbers, if that is what they are: numpy cuts off what does not fit."""
    a = np.asarray(x)
    if a.dtype == _I32:
        return np.ascontiguousarray(a)
    try:
        with np.errstate(invalid="ignore"):
            b = np.ascontiguousarray(a, dtype=_I32)
        if (b == a).all():
            return b
    except (OverflowError, TypeError, ValueError):
        pass
    raise SlaiError(_lib.ERR_SHAPE, f"paged step: {what} are not int32 numbers")


class PagedLayer:
    """A layer's pages (`slai_paged_layer`): key and value buffers and the strides, in elements, between pages, cache heads and positions."""

    def __init__(self, keys, values, page_stride: int, head_stride: int, pos_stride: int):
        self.keys, self.values = keys, values  # held: the pages outlive the layer
        self.strides = (page_stride, head_stride, pos_stride)
        self.elements = min(len(keys), len(values))
        self.nbytes = min(getattr(keys, "nbytes", None) or 4 * len(keys), getattr(values, "nbytes", None) or 4 * len(values))
        self.c = _lib.PagedLayer(keys.ptr, values.ptr, page_stride, head_stride, pos_stride)
        self.at = C.addressof(self.c)


class PagedKv:
    """Keys and values of many sequences in pages (`slai_paged`): what a model's layers have in common, and the current step.  The reference's cache is
    one dense tensor of one sequence (crates/slai/src/models/llama2/transformer.rs:87-106).

    max_table: table entries of a step, a page that several sequences share counting for each of them.  None: every sequence may use every page, up to 2^20 entries
    in all (4 MB on the device, 8 MB of pinned memory), or each page once where there are more pages than that."""

    def __init__(self, backend: Backend, n_q_heads: int, n_kv_heads: int, head_size: int, page_size: int, n_pages: int, kv_dtype: int = KV_F16,
                 max_seqs: int = 8, max_tokens: int = 512, max_table: int | None = None):
        self.backend = backend
        self.n_q_heads, self.n_kv_heads, self.head_size, self.page_size, self.n_pages = n_q_heads, n_kv_heads, head_size, page_size, n_pages
        self.kv_dtype, self.max_tokens, self.width = kv_dtype, max_tokens, n_q_heads * head_size
        self.kv_bytes = 2 if kv_dtype == KV_F16 else 4
        self.last = (n_pages - 1, n_kv_heads - 1, page_size - 1, head_size)  # the last element's place, by a layer's strides
        self.rows = None  # of the current step
        cfg = _lib.PagedConfig(n_q_heads, n_kv_heads, head_size, page_size, n_pages, kv_dtype, max_seqs, max_tokens, max_table or max(n_pages, min(n_pages * max_seqs, 1 << 20)))
        h = C.c_void_p()
        backend.check(backend.lib.slai_paged_create(backend.h, C.byref(cfg), C.byref(h)))
        self.h = h

    def step(self, pos0, n_new, tables):
        """Sequence b: `pos0[b]` cached positions, `n_new[b]` new tokens behind them, pages `tables[b]` in order of their positions."""
        pos0, n_new, tables = _int32("pos0", pos0), _int32("n_new", n_new), _int32("tables", tables)
        n = pos0.size
        if pos0.ndim != 1 or n_new.shape != pos0.shape or tables.ndim != 2 or tables.shape[0] != n:
            raise SlaiError(_lib.ERR_SHAPE, f"paged step: lengths of {pos0.shape}, {n_new.shape} and tables of {tables.shape}")
        at = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
        self.backend.check(self.backend.lib.slai_paged_step(self.h, n, at(pos0), at(n_new), at(tables), tables.shape[1]))
        self.rows = int(n_new.sum())

    def check_layer(self, layer: PagedLayer):
        pages, heads, positions, size = self.last
        page, head, pos = layer.strides
        need = pages * page + heads * head + positions * pos + size
        if layer.elements < need or layer.nbytes < self.kv_bytes * need:
            raise SlaiError(_lib.ERR_SHAPE, f"paged: pages of {layer.elements} elements in {layer.nbytes} bytes, {need} elements of {self.kv_bytes} needed")

    def rows_in_use(self):
        """Rows that a call's buffers hold: the step's, or, for a call that is recorded and replayed for other steps, the most that a step can have."""
        return self.max_tokens if self.backend._recording else self.rows

    def __del__(self):
        try:
            if self.backend.h and self.h:
                destroy, h, self.h = self.backend.lib.slai_paged_destroy, self.h, None
                if getattr(self.backend, "_recording", False):
                    self.backend._deferred_handles.append((destroy, h))  # (as Backend.free)
                else:
                    destroy(h)
        except Exception:
            pass


class QkNormRope:
    """`slai_qk_params`: RmsNorm of every head of q and k (where weights are given) and their rotation by position (`variant` None: none).  Leading
    dimensions: floats between two tokens' rows, 0 = packed."""

    def __init__(self, head_size: int, n_q_heads: int, n_kv_heads: int, variant: RoPEVariant | None = RoPEVariant.Original, base_freq: float = 10000.0,
                 eps: float = 1e-5, q_norm=None, k_norm=None, q_ld: int = 0, k_ld: int = 0, v_ld: int = 0, q_out_ld: int = 0, k_out_ld: int = 0):
        for w in (q_norm, k_norm):
            if w is not None and (len(w) != head_size or getattr(w, "dtype", _F32) != _F32):
                raise SlaiError(_lib.ERR_SHAPE, f"qk: {len(w)} norm weights of {getattr(w, 'dtype', _F32)} for heads of {head_size} floats")
        self.norms = (q_norm, k_norm)  # held
        self.q_width, self.k_width = n_q_heads * head_size, n_kv_heads * head_size
        self.q_ld, self.k_ld, self.v_ld = q_ld or self.q_width, k_ld or self.k_width, v_ld or self.k_width
        self.q_out_ld, self.k_out_ld = q_out_ld or self.q_width, k_out_ld or self.k_width
        self.c = _lib.QkParams(head_size, n_q_heads, n_kv_heads, -1 if variant is None else int(variant), base_freq, eps, _ptr(q_norm).value,
                               _ptr(k_norm).value, q_ld, k_ld, v_ld, q_out_ld, k_out_ld)
        self.at = C.addressof(self.c)
        self.rows = (self.q_width, self.k_width, self.q_ld, self.k_ld, self.v_ld, self.q_out_ld, self.k_out_ld)


def _refuse_context():
    raise SlaiError(_lib.ERR_INVALID_ARG, "paged: the handle is another context's (its calls would run on that context's stream)")


def _refuse_rows(what: str, x, rows: int, width: int, ld: int):
    if x is not None and len(x) >= (rows - 1) * (ld or width) + width:
        if x.dtype == _F32:  # (a type of its own that says it is f32)
            return
        raise SlaiError(_lib.ERR_SHAPE, f"{what}: rows are floats, not {x.dtype}")
    raise SlaiError(_lib.ERR_SHAPE, f"{what}: {0 if x is None else len(x)} floats for {rows} rows of {width}, {ld or width} apart")


class LlmContext:
    """`LlmContext<'a, B>` (crates/slai/src/context.rs:68-96): one method per operator; work is enqueued on the
    backend's stream (`begin_submission` ... `submit`), nothing blocks until `submit().synchronize()`."""

    def __init__(self, backend: Backend):
        self.backend = backend
        self.lib = backend.lib
        self.h = backend.h

    def begin_submission(self):  # context.rs:79-88 — recording is implicit: calls enqueue on the stream
        return self

    def submit(self):  # context.rs:90-95
        return self

    # GemvQuant::launch (ops/gemv_quant.rs:206-312); LlmContext::matmul_quant_assign (context.rs:355-369)
    def matmul_quant_assign(self, out, a: GpuQuantMatrix, b, n_batch: int = 1):
        if len(b) != a.ncols * n_batch or len(out) != a.nrows * n_batch:
            raise SlaiError(_lib.ERR_SHAPE, f"Gemv: dimension mismatch ({a.nrows}x{a.ncols} * {len(b)} -> {len(out)})")
        self.backend.check(self.lib.slai_gemv_quant(self.h, _ptr(out), a.h, _ptr(b), n_batch))

    def ffn_gate_up(self, out, w_gate: GpuQuantMatrix, w_up: GpuQuantMatrix, x, norm_w=None, eps: float = 1e-5):
        """out = silu(Wgate n(x)) * (Wup n(x)), n = RmsNorm: the operators of transformer.rs:356-361 as one kernel."""
        self.backend.check(self.lib.slai_ffn_gate_up(self.h, _ptr(out), w_gate.h, w_up.h, _ptr(x), _ptr(norm_w) if norm_w is not None else None, eps))

    # Tensor-parallel exchange operators (no counterpart in the reference): a row-parallel product whose partial goes
    # to every rank's exchange region, and a product whose input is the sum over ranks of such an exchange.
    def matmul_quant_partial(self, a: GpuQuantMatrix, b, resid, index: int, per_token: int):
        if len(b) != a.ncols or (resid is not None and len(resid) != a.nrows):
            raise SlaiError(_lib.ERR_SHAPE, "Gemv: dimension mismatch")
        self.backend.check(self.lib.slai_gemv_quant_partial(self.h, a.h, _ptr(b), _ptr(resid), index, per_token))

    def matmul_quant_reduced(self, out, a: GpuQuantMatrix, norm_w, eps: float, index: int, per_token: int, sum_out):
        if len(out) != a.nrows or len(norm_w) != a.ncols or len(sum_out) != a.ncols:
            raise SlaiError(_lib.ERR_SHAPE, "Gemv: dimension mismatch")
        self.backend.check(self.lib.slai_gemv_quant_reduced(self.h, _ptr(out), a.h, _ptr(norm_w), eps, index, per_token, _ptr(sum_out)))

    def token_tick(self):
        self.backend.check(self.lib.slai_tp_token_tick(self.h))

    def peer_loopback(self, ranks: int, rank: int):
        self.backend.check(self.lib.slai_tp_peer_loopback(self.h, ranks, rank))

    # RmsNorm::launch (ops/rms_norm.rs:35-67); LlmContext::rms_norm_assign
    def rms_norm_assign(self, result, value, weight, eps: float = 1e-5):
        if not (len(result) == len(value) == len(weight)):
            raise SlaiError(_lib.ERR_SHAPE, "rms_norm: length mismatch")
        self.backend.check(self.lib.slai_rms_norm(self.h, _ptr(result), _ptr(value), _ptr(weight), len(value), eps))

    # RoPE::launch (ops/rope.rs:45-85)
    def rope(self, variant: RoPEVariant, in_out_q, in_out_k, head_size: int, kv_dim: int, pos: int, base_freq: float = 10000.0):
        self.backend.check(self.lib.slai_rope(self.h, int(variant), _ptr(in_out_q), len(in_out_q), _ptr(in_out_k), head_size,
                                              kv_dim, pos, base_freq))

    # Silu::launch (ops/silu.rs:24-48)
    def silu(self, in_out_h1, in_h2):
        if len(in_out_h1) != len(in_h2):
            raise SlaiError(_lib.ERR_SHAPE, "silu: length mismatch")
        self.backend.check(self.lib.slai_silu_gate(self.h, _ptr(in_out_h1), _ptr(in_h2), len(in_out_h1)))

    # Unary::launch / launch_inplace (ops/unary.rs:171-306)
    def unary(self, op: UnaryOp, dest, src, args=(0.0, 0.0, 0.0, 0.0)):
        a = (C.c_float * 4)(*(list(args) + [0.0] * (4 - len(args))))
        self.backend.check(self.lib.slai_unary(self.h, int(op), _ptr(dest), _ptr(src), len(src), a))

    def gelu_inplace(self, x):
        self.unary(UnaryOp.Gelu, x, x)

    # SoftMax::launch_cols (ops/softmax.rs:22-40)
    def softmax_cols(self, in_out_mat, nrows: int, ncols: int, col_stride: int | None = None):
        self.backend.check(self.lib.slai_softmax_cols(self.h, _ptr(in_out_mat), nrows, ncols, col_stride or nrows))

    # LayerNorm::launch_cols (ops/layernorm.rs:25-60) (+ the caller's gamma/beta, gpt2/cpu.rs:239-240)
    def layernorm(self, output, input, eps: float = 1e-5, gamma=None, beta=None):
        if len(output) != len(input):
            raise SlaiError(_lib.ERR_SHAPE, "layernorm: length mismatch")
        self.backend.check(self.lib.slai_layernorm(self.h, _ptr(output), _ptr(input), len(input), eps, _ptr(gamma), _ptr(beta)))

    # LlmContext::add_assign / mul_assign / copy (context.rs:428-469,660-673)
    def add_assign(self, a, b):
        self.backend.check(self.lib.slai_add_assign(self.h, _ptr(a), _ptr(b), len(a)))

    def mul_assign(self, a, b):
        self.backend.check(self.lib.slai_mul_assign(self.h, _ptr(a), _ptr(b), len(a)))

    def copy(self, dst, src):
        self.backend.check(self.lib.slai_copy(self.h, _ptr(dst), _ptr(src), len(src)))

    # BatchedMultiqueryAttention::launch (ops/batched_multiquery_attention.rs:32-100)
    def attention(self, params: BatchedMultiqueryAttentionParams, q, key_cache, value_cache, xb, kv_dtype: int = KV_F32):
        p = params.to_c()
        self.backend.check(self.lib.slai_attention(self.h, C.byref(p), _ptr(q), _ptr(key_cache), _ptr(value_cache), kv_dtype, _ptr(xb)))

    def kv_append(self, key_cache, value_cache, k, v, kv_dim: int, pos: int, kv_dtype: int = KV_F32):
        self.backend.check(self.lib.slai_kv_append(self.h, _ptr(key_cache), _ptr(value_cache), kv_dtype, _ptr(k), _ptr(v), kv_dim, pos))

    # Paged caches (the operators they stand beside: RmsNorm, RoPE, key_cache.column(pos), BatchedMultiqueryAttention).  A buffer of n rows holds at least the
    # (n - 1) * leading dimension + width floats from its first row to its last.
    def qk_norm_rope(self, how: QkNormRope, positions, q, k, q_out, k_out):
        """Norm and rotation of the rows of q and k, token t at position positions[t] (int32 on the device; negative: left as it is)."""
        n = len(positions)
        if getattr(positions, "dtype", _I32) is not _I32 and np.dtype(positions.dtype).itemsize != 4:
            raise SlaiError(_lib.ERR_SHAPE, f"qk_norm_rope: positions are int32 numbers, not {positions.dtype}")
        if n > 0:
            m, f, (w, k_w, q_ld, k_ld, _, q_out_ld, k_out_ld) = n - 1, _F32, how.rows
            if w:
                if q is None or len(q) < m * q_ld + w or getattr(q, "dtype", f) is not f:
                    _refuse_rows("qk_norm_rope: q", q, n, w, q_ld)
                if q_out is None or len(q_out) < m * q_out_ld + w or getattr(q_out, "dtype", f) is not f:
                    _refuse_rows("qk_norm_rope: q_out", q_out, n, w, q_out_ld)
            if k_w:
                if k is None or len(k) < m * k_ld + k_w or getattr(k, "dtype", f) is not f:
                    _refuse_rows("qk_norm_rope: k", k, n, k_w, k_ld)
                if k_out is None or len(k_out) < m * k_out_ld + k_w or getattr(k_out, "dtype", f) is not f:
                    _refuse_rows("qk_norm_rope: k_out", k_out, n, k_w, k_out_ld)
        rc = self.lib.slai_qk_norm_rope(self.h, how.at, n, positions.ptr, None if q is None else q.ptr, None if k is None else k.ptr,
                                        None if q_out is None else q_out.ptr, None if k_out is None else k_out.ptr)
        if rc:
            self.backend.check(rc)

    def paged_append(self, paged: PagedKv, layer: PagedLayer, how: QkNormRope, q, k, v, q_out):
        """The same for the rows of the current step; keys and values go into their pages, q to q_out."""
        if paged.backend is not self.backend:
            _refuse_context()
        paged.check_layer(layer)
        n = paged.rows_in_use()
        if n:
            m, f, (w, k_w, q_ld, k_ld, v_ld, q_out_ld, _) = n - 1, _F32, how.rows
            if w:
                if q is None or len(q) < m * q_ld + w or getattr(q, "dtype", f) is not f:
                    _refuse_rows("paged_append: q", q, n, w, q_ld)
                if q_out is None or len(q_out) < m * q_out_ld + w or getattr(q_out, "dtype", f) is not f:
                    _refuse_rows("paged_append: q_out", q_out, n, w, q_out_ld)
            if k is None or len(k) < m * k_ld + k_w or getattr(k, "dtype", f) is not f:
                _refuse_rows("paged_append: k", k, n, k_w, k_ld)
            if v is None or len(v) < m * v_ld + k_w or getattr(v, "dtype", f) is not f:
                _refuse_rows("paged_append: v", v, n, k_w, v_ld)
        rc = self.lib.slai_paged_append(paged.h, layer.at, how.at, None if q is None else q.ptr, None if k is None else k.ptr, None if v is None else v.ptr,
                                        None if q_out is None else q_out.ptr)
        if rc:
            self.backend.check(rc)

    def paged_attention(self, paged: PagedKv, layer: PagedLayer, q, out, scale: float = 0.0, q_ld: int = 0, out_ld: int = 0):
        """Causal attention of the step's tokens to what their sequences hold (scale 0: 1 / sqrt(head_size)).  f32 sums; products of operands of 21 to 24 bits, by the
        cache's type and the step: `slai_paged_attention`."""
        if paged.backend is not self.backend:
            _refuse_context()
        paged.check_layer(layer)
        n, width = paged.rows_in_use(), paged.width
        if n:
            if len(q) < (n - 1) * (q_ld or width) + width or getattr(q, "dtype", _F32) is not _F32:
                _refuse_rows("paged_attention: q", q, n, width, q_ld)
            if len(out) < (n - 1) * (out_ld or width) + width or getattr(out, "dtype", _F32) is not _F32:
                _refuse_rows("paged_attention: out", out, n, width, out_ld)
        rc = self.lib.slai_paged_attention(paged.h, layer.at, q.ptr, q_ld, scale, out.ptr, out_ld)
        if rc:
            self.backend.check(rc)

    def sample(self, logits: GpuVector, temperature: float, topp: float, coin: float) -> int:
        """`Sampler::sample` (models/sampler.rs:33-54) on the device, the uniform number `coin` given; `logits` is
        overwritten with the probabilities."""
        out = GpuVector(self.backend, 1, np.int32)
        self.backend.check(self.backend.lib.slai_sample(self.backend.h, C.c_void_p(logits.ptr), logits.n, temperature, topp, coin,
                                                        C.c_void_p(out.ptr)))
        return int(out.to_numpy()[0])

    # Sampler::sample_argmax (models/sampler.rs:55-57)
    def argmax(self, v) -> int:
        out = self.backend.zeros(1, np.int32)
        self.backend.check(self.lib.slai_argmax(self.h, _ptr(v), len(v), _ptr(out)))
        return int(out.to_numpy()[0])
