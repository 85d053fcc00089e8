"""Host-side mirror of the reference's `ModelForward` boundary over the C-ABI
library (`include/cheetah_cuda.h`), plus thin wrappers of the op entries.

`CudaQwen2` behaves like `Qwen2Native` (`src/chat/registrations/qwen2.rs:600-635`)
behind `ModelForward` (`src/chat/registry.rs:57-85`): `forward(tokens, offset)`
returns the final position's logits, `clear_cache()`, `kv_snapshot()`,
`restore_kv_prefix(snapshot, positions)`, `clone()` (shares weights, empty
KV, `registry.rs:95-117`) and `device_name()`. Errors surface as
`CheetahCudaError` carrying the library's last-error string, the way the Rust
side maps `check_native_result` (`src/native.rs:1860-1870`) to `Err(String)`.

There is no CPU fallback: constructing anything here without the built
library or without a CUDA device raises.
"""

from __future__ import annotations

import ctypes as C
import os
from pathlib import Path
from typing import NamedTuple, Optional, Sequence

import numpy as np

from .prepared import PreparedModel, resolve_config

# The in-tree build; CHEETAH_CUDA_LIB selects another build of the same ABI.
LIB_PATH = Path(os.environ.get("CHEETAH_CUDA_LIB") or Path(__file__).resolve().parent / "libcheetah_cuda.so")

KV_BF16, KV_F32 = 0, 1


class CheetahCudaError(RuntimeError):
    pass


class CudaConfig(C.Structure):
    _fields_ = [
        ("hidden_size", C.c_uint32), ("num_layers", C.c_uint32), ("q_heads", C.c_uint32),
        ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("rotary_dim", C.c_uint32),
        ("intermediate_size", C.c_uint32), ("vocab_size", C.c_uint32), ("rms_eps", C.c_float),
        ("rope_theta", C.c_float), ("tie_word_embeddings", C.c_int32),
        ("sliding_window", C.c_uint32), ("max_positions", C.c_uint32),
        ("kv_page_tokens", C.c_uint32), ("kv_pool_tokens", C.c_uint32), ("kv_dtype", C.c_int32),
    ]


class ModelInfo(C.Structure):
    _fields_ = [
        ("weight_bytes", C.c_uint64), ("kv_pool_bytes", C.c_uint64),
        ("kv_pages_total", C.c_uint32), ("kv_pages_free", C.c_uint32),
        ("device", C.c_int32), ("quant", C.c_int32),
        ("persistent_decode", C.c_int32), ("reserved", C.c_int32),
    ]


class Residency(C.Structure):
    _fields_ = [("unit_ids", C.POINTER(C.c_char_p)), ("tiers", C.POINTER(C.c_char_p)), ("count", C.c_size_t)]


class ResidencyInfo(C.Structure):
    _fields_ = [
        ("resident_linear_bytes", C.c_uint64), ("streamed_linear_bytes", C.c_uint64),
        ("staging_bytes", C.c_uint64), ("resident_linears", C.c_uint32), ("streamed_linears", C.c_uint32),
        ("planned", C.c_int32), ("reserved", C.c_int32),
    ]


class DecodeAttentionArgs(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("k_pool", C.c_void_p), ("v_pool", C.c_void_p),
        ("kv_dtype", C.c_int32), ("page_table", C.c_void_p), ("max_pages_per_seq", C.c_uint32),
        ("seq_lens", C.c_void_p), ("max_seq_len", C.c_uint32), ("num_pages", C.c_uint32),
        ("page_tokens", C.c_uint32), ("batch", C.c_uint32), ("q_heads", C.c_uint32),
        ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("sliding_window", C.c_uint32),
        ("out", C.c_void_p),
    ]


class PrefillAttentionArgs(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("k_pool", C.c_void_p), ("v_pool", C.c_void_p),
        ("page_table", C.c_void_p), ("max_pages", C.c_uint32), ("num_pages", C.c_uint32),
        ("page_tokens", C.c_uint32), ("tokens", C.c_uint32), ("offset", C.c_uint32),
        ("q_heads", C.c_uint32), ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32),
        ("sliding_window", C.c_uint32), ("out", C.c_void_p),
    ]


class PageSlotsArgs(C.Structure):
    _fields_ = [
        ("cached", C.c_void_p), ("new_tokens", C.c_void_p), ("free_pages", C.c_void_p),
        ("free_count", C.c_void_p), ("free_capacity", C.c_uint32), ("batch", C.c_uint32),
        ("page_table", C.c_void_p), ("max_pages_per_seq", C.c_uint32), ("num_pages", C.c_uint32),
        ("page_tokens", C.c_uint32), ("max_tokens", C.c_uint32), ("row_starts", C.c_void_p),
        ("seq_lens", C.c_void_p), ("positions", C.c_void_p), ("seq_ids", C.c_void_p),
        ("slots", C.c_void_p), ("counts", C.c_void_p),
    ]


class QkNormRopeArgs(C.Structure):
    _fields_ = [
        ("qkv", C.c_void_p), ("qkv_stride", C.c_size_t), ("dtype", C.c_int32), ("kv_dtype", C.c_int32),
        ("q_norm", C.c_void_p), ("k_norm", C.c_void_p), ("eps", C.c_float), ("rope_cos", C.c_void_p),
        ("rope_sin", C.c_void_p), ("max_positions", C.c_uint32), ("rotary_dim", C.c_uint32),
        ("positions", C.c_void_p), ("slots", C.c_void_p), ("tokens", C.c_uint32), ("q_heads", C.c_uint32),
        ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("q_out", C.c_void_p), ("k_pool", C.c_void_p),
        ("v_pool", C.c_void_p), ("num_pages", C.c_uint32), ("page_tokens", C.c_uint32),
    ]


class TreeAttentionArgs(C.Structure):
    _fields_ = [
        ("q", C.c_void_p), ("q_stride", C.c_size_t), ("rows", C.c_uint32), ("k_pool", C.c_void_p),
        ("v_pool", C.c_void_p), ("page_table", C.c_void_p), ("max_pages_per_seq", C.c_uint32),
        ("num_pages", C.c_uint32), ("page_tokens", C.c_uint32), ("seq_lens", C.c_void_p),
        ("row_starts", C.c_void_p), ("batch", C.c_uint32), ("tree_mask", C.c_void_p),
        ("mask_words", C.c_uint32), ("positions", C.c_void_p), ("sliding_window", C.c_uint32),
        ("q_heads", C.c_uint32), ("kv_heads", C.c_uint32), ("head_dim", C.c_uint32), ("out", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class TokenLogprobsArgs(C.Structure):
    _fields_ = [
        ("logits", C.c_void_p), ("row_stride", C.c_size_t), ("dtype", C.c_int32), ("rows", C.c_uint32),
        ("vocab", C.c_uint32), ("tokens", C.c_void_p), ("top", C.c_uint32), ("logprob", C.c_void_p),
        ("rank", C.c_void_p), ("entropy", C.c_void_p), ("top_ids", C.c_void_p), ("top_logprobs", C.c_void_p),
    ]


# Every symbol include/cheetah_cuda.h declares, with its ctypes signature.
_P, _S, _I = C.c_void_p, C.c_size_t, C.c_int
SIGNATURES = {
    "cheetah_cuda_last_error": (C.c_char_p, []),
    "cheetah_cuda_abi_version": (_I, []),
    "cheetah_cuda_device_count": (_I, [C.POINTER(C.c_int)]),
    "cheetah_cuda_model_open": (_I, [C.c_char_p, C.POINTER(CudaConfig), C.c_char_p, _I, C.POINTER(_P)]),
    "cheetah_cuda_model_free": (_I, [_P]),
    "cheetah_cuda_model_info": (_I, [_P, C.POINTER(ModelInfo)]),
    "cheetah_cuda_model_open_ex": (_I, [C.c_char_p, C.POINTER(CudaConfig), C.c_char_p, _I, C.POINTER(Residency),
                                        C.POINTER(_P)]),
    "cheetah_cuda_model_page_in_unit": (_I, [_P, C.c_char_p, _I, C.POINTER(_I)]),
    "cheetah_cuda_model_evict_unit": (_I, [_P, C.c_char_p, C.POINTER(_I)]),
    "cheetah_cuda_model_residency": (_I, [_P, C.POINTER(ResidencyInfo)]),
    "cheetah_cuda_seq_new": (_I, [_P, C.POINTER(_P)]),
    "cheetah_cuda_seq_free": (_I, [_P]),
    "cheetah_cuda_seq_clear": (_I, [_P]),
    "cheetah_cuda_seq_positions": (_I, [_P, C.POINTER(_S)]),
    "cheetah_cuda_forward": (_I, [_P, _P, _S, _S, _P]),
    "cheetah_cuda_forward_ex": (_I, [_P, _P, _S, _S, _P, _P]),
    "cheetah_cuda_model_coalesce_stats": (_I, [_P, C.POINTER(C.c_uint64), C.POINTER(C.c_uint64),
                                                C.POINTER(C.c_uint64)]),
    "cheetah_cuda_forward_batch": (_I, [_P, _P, _P, _P, _S, _P, _P]),
    "cheetah_cuda_forward_batch_greedy": (_I, [_P, _P, _P, _P, _S, _S, _P]),
    "cheetah_cuda_generate_greedy": (_I, [_P, C.c_uint32, _S, _S, _P]),
    "cheetah_cuda_seq_stream": (_I, [_P, C.POINTER(_P)]),
    "cheetah_cuda_model_batch_stream": (_I, [_P, C.POINTER(_P)]),
    "cheetah_cuda_seq_snapshot": (_I, [_P, C.POINTER(_P)]),
    "cheetah_cuda_snapshot_positions": (_I, [_P, C.POINTER(_S)]),
    "cheetah_cuda_seq_restore_prefix": (_I, [_P, _P, _S]),
    "cheetah_cuda_snapshot_free": (_I, [_P]),
    "cheetah_cuda_seq_export_kv": (_I, [_P, _S, _P, _P]),
    "cheetah_cuda_op_gemv_bf16": (_I, [_P, _S, _S, _P, _S, _P, _P]),
    "cheetah_cuda_op_decode_attention": (_I, [C.POINTER(DecodeAttentionArgs), _P]),
    "cheetah_cuda_op_decode_attention_noalloc": (_I, [C.POINTER(DecodeAttentionArgs), _P]),
    "cheetah_cuda_op_prefill_attention": (_I, [C.POINTER(PrefillAttentionArgs), _P]),
    "cheetah_cuda_quant_buffer_bytes": (_I, [C.c_char_p, _S, _S, C.POINTER(_S)]),
    "cheetah_cuda_op_quantize_q8": (_I, [_P, _S, _S, _P, _P]),
    "cheetah_cuda_op_quantize_q4": (_I, [_P, _S, _S, _P, _P]),
    "cheetah_cuda_op_gemv_q8": (_I, [_P, _S, _S, _P, _S, _P, _P]),
    "cheetah_cuda_op_gemv_q4": (_I, [_P, _S, _S, _P, _S, _P, _P]),
    "cheetah_cuda_op_page_slots": (_I, [C.POINTER(PageSlotsArgs), _P]),
    "cheetah_cuda_op_qk_norm_rope": (_I, [C.POINTER(QkNormRopeArgs), _P]),
    "cheetah_cuda_op_tree_attention_workspace": (_I, [C.POINTER(TreeAttentionArgs), C.POINTER(_S)]),
    "cheetah_cuda_op_tree_attention": (_I, [C.POINTER(TreeAttentionArgs), _P]),
    "cheetah_cuda_op_token_logprobs": (_I, [C.POINTER(TokenLogprobsArgs), _P]),
}

_lib: Optional[C.CDLL] = None


def lib() -> C.CDLL:
    """Load libcheetah_cuda.so (built in-tree by `cheetah_b200.build`)."""
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise CheetahCudaError(
                f"{LIB_PATH} is missing: build it with `python -m cheetah_b200.build` "
                "(there is no CPU fallback).")
        handle = C.CDLL(str(LIB_PATH))
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(handle, name)
            fn.restype = res
            fn.argtypes = args
        _lib = handle
    return _lib


def _check(rc: int) -> None:
    if rc != 0:
        raise CheetahCudaError(lib().cheetah_cuda_last_error().decode(errors="replace"))


def _ptr(a: np.ndarray) -> int:
    return a.ctypes.data


def device_count() -> int:
    n = C.c_int(0)
    _check(lib().cheetah_cuda_device_count(C.byref(n)))
    return n.value


class CudaModel:
    """HBM-resident weights + KV page pool on one device (`model_open`)."""

    def __init__(self, prepared_dir: os.PathLike, quant: str = "bf16", device: int = 0,
                 kv_dtype: str = "bf16", max_positions: Optional[int] = None,
                 kv_pool_tokens: int = 0, kv_page_tokens: int = 0,
                 config: Optional[dict] = None, residency: Optional[dict] = None):
        """`residency`: an Ant plan {unit id: "vram" | "ram" | "disk"}
        (`cheetah_cuda_model_open_ex`); None opens every unit HBM-resident."""
        self.prepared_dir = Path(prepared_dir)
        cfg = dict(config) if config else resolve_config(PreparedModel(self.prepared_dir), max_positions)
        if max_positions:
            cfg["max_positions"] = int(max_positions)
        self.cfg = cfg
        self.quant = quant
        c = CudaConfig(cfg["hidden_size"], cfg["num_layers"], cfg["q_heads"], cfg["kv_heads"],
                       cfg["head_dim"], cfg["rotary_dim"], cfg["intermediate_size"], cfg["vocab_size"],
                       cfg["rms_eps"], cfg["rope_theta"], cfg["tie_word_embeddings"],
                       cfg["sliding_window"], cfg["max_positions"], kv_page_tokens, kv_pool_tokens,
                       KV_F32 if kv_dtype == "f32" else KV_BF16)
        handle = C.c_void_p()
        if residency is None:
            _check(lib().cheetah_cuda_model_open(str(self.prepared_dir).encode(), C.byref(c),
                                                 quant.encode(), device, C.byref(handle)))
        else:
            items = sorted(residency.items())
            ids = (C.c_char_p * max(1, len(items)))(*[k.encode() for k, _ in items])
            tiers = (C.c_char_p * max(1, len(items)))(*[v.encode() for _, v in items])
            plan = Residency(ids, tiers, len(items))
            _check(lib().cheetah_cuda_model_open_ex(str(self.prepared_dir).encode(), C.byref(c), quant.encode(),
                                                    device, C.byref(plan), C.byref(handle)))
        self._h = handle

    @property
    def handle(self) -> C.c_void_p:
        return self._h

    def info(self) -> dict:
        info = ModelInfo()
        _check(lib().cheetah_cuda_model_info(self._h, C.byref(info)))
        return {f: getattr(info, f) for f, _ in ModelInfo._fields_}

    def residency(self) -> dict:
        info = ResidencyInfo()
        _check(lib().cheetah_cuda_model_residency(self._h, C.byref(info)))
        return {f: getattr(info, f) for f, _ in ResidencyInfo._fields_}

    def page_in_unit(self, unit_id: str, tier: int = 0) -> bool:
        """`AntTierControl::page_in_unit`: True when the manifest knows the unit."""
        known = C.c_int(0)
        _check(lib().cheetah_cuda_model_page_in_unit(self._h, unit_id.encode(), tier, C.byref(known)))
        return bool(known.value)

    def evict_unit(self, unit_id: str) -> bool:
        """`AntTierControl::evict_unit`: True when the manifest knows the unit."""
        known = C.c_int(0)
        _check(lib().cheetah_cuda_model_evict_unit(self._h, unit_id.encode(), C.byref(known)))
        return bool(known.value)

    def close(self) -> None:
        if getattr(self, "_h", None):
            lib().cheetah_cuda_model_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def new_sequence(self) -> "CudaQwen2":
        return CudaQwen2(self)

    def forward_batch(self, seqs, tokens, offsets, want_logits: bool = False):
        """One decode token for each sequence (`cheetah_cuda_forward_batch`).
        Returns the greedy ids (and the [B, vocab] logits when asked)."""
        B = len(seqs)
        handles = (C.c_void_p * B)(*[s._h.value for s in seqs])
        t = np.ascontiguousarray(np.asarray(tokens, dtype=np.uint32))
        o = np.ascontiguousarray(np.asarray(offsets, dtype=np.uint64))
        am = np.zeros(B, dtype=np.uint32)
        logits = np.empty((B, self.cfg["vocab_size"]), dtype=np.float32) if want_logits else None
        _check(lib().cheetah_cuda_forward_batch(self._h, handles, _ptr(t), _ptr(o), B,
                                                _ptr(logits) if want_logits else None, _ptr(am)))
        return (am, logits) if want_logits else am

    def coalesce_stats(self) -> dict:
        """Counters of the batcher behind `forward`: single-token calls,
        calls that ran inside batched steps, batched steps."""
        a, b, c = C.c_uint64(0), C.c_uint64(0), C.c_uint64(0)
        _check(lib().cheetah_cuda_model_coalesce_stats(self._h, C.byref(a), C.byref(b), C.byref(c)))
        return {"calls": a.value, "batched_calls": b.value, "batches": c.value}

    def batch_stream_handle(self) -> int:
        """The stream batched calls run on (0 before the first batched call)."""
        s = C.c_void_p()
        _check(lib().cheetah_cuda_model_batch_stream(self._h, C.byref(s)))
        return s.value or 0

    def forward_batch_greedy(self, seqs, tokens, offsets, steps: int) -> np.ndarray:
        """`steps` greedy tokens for each sequence with no host round trip
        between steps (`cheetah_cuda_forward_batch_greedy`): uint32 [B, steps],
        row b holding the ids generated after tokens[b]."""
        B = len(seqs)
        handles = (C.c_void_p * B)(*[s._h.value for s in seqs])
        t = np.ascontiguousarray(np.asarray(tokens, dtype=np.uint32))
        o = np.ascontiguousarray(np.asarray(offsets, dtype=np.uint64))
        out = np.zeros((B, steps), dtype=np.uint32)
        _check(lib().cheetah_cuda_forward_batch_greedy(self._h, handles, _ptr(t), _ptr(o), B, steps, _ptr(out)))
        return out


class CudaSnapshot:
    def __init__(self, handle: C.c_void_p, model: CudaModel):
        self._h = handle
        self._model = model

    @property
    def positions(self) -> int:
        n = C.c_size_t(0)
        _check(lib().cheetah_cuda_snapshot_positions(self._h, C.byref(n)))
        return n.value

    def __del__(self):
        if getattr(self, "_h", None):
            lib().cheetah_cuda_snapshot_free(self._h)
            self._h = None


class CudaQwen2:
    """`ModelForward` over one sequence of a `CudaModel` (`qwen2.rs:600-635`)."""

    def __init__(self, model: CudaModel):
        self.model = model
        self.cfg = model.cfg
        handle = C.c_void_p()
        _check(lib().cheetah_cuda_seq_new(model.handle, C.byref(handle)))
        self._h = handle
        self._logits = np.zeros(self.cfg["vocab_size"], dtype=np.float32)

    @classmethod
    def load(cls, prepared_dir: os.PathLike, **kwargs) -> "CudaQwen2":
        return cls(CudaModel(prepared_dir, **kwargs))

    def device_name(self) -> str:
        return "cuda-b200"

    def clone(self) -> "CudaQwen2":
        """Shares the weights, starts with an empty KV (`registry.rs:95-117`)."""
        return CudaQwen2(self.model)

    def forward(self, tokens: Sequence[int], offset: int, out: Optional[np.ndarray] = None) -> np.ndarray:
        t = np.ascontiguousarray(np.asarray(tokens, dtype=np.uint32))
        logits = out if out is not None else np.empty(self.cfg["vocab_size"], dtype=np.float32)
        _check(lib().cheetah_cuda_forward(self._h, _ptr(t) if t.size else None, t.size, offset,
                                          _ptr(logits)))
        return logits

    def forward_greedy(self, tokens: Sequence[int], offset: int,
                       logits_out: Optional[np.ndarray] = None) -> int:
        """Forward plus on-device greedy argmax (`engine.rs:2247-2253`)."""
        t = np.ascontiguousarray(np.asarray(tokens, dtype=np.uint32))
        am = C.c_uint32(0)
        lp = _ptr(logits_out) if logits_out is not None else None
        _check(lib().cheetah_cuda_forward_ex(self._h, _ptr(t) if t.size else None, t.size, offset,
                                             lp, C.byref(am)))
        return am.value

    def generate_greedy(self, first_token: int, offset: int, steps: int,
                        wait: bool = True) -> Optional[np.ndarray]:
        """Device-resident greedy decode of `steps` tokens (no host round trip
        per token). With wait=False the steps are only enqueued."""
        out = np.zeros(steps, dtype=np.uint32) if wait else None
        _check(lib().cheetah_cuda_generate_greedy(self._h, int(first_token), offset, steps,
                                                  _ptr(out) if wait else None))
        return out

    def stream_handle(self) -> int:
        s = C.c_void_p()
        _check(lib().cheetah_cuda_seq_stream(self._h, C.byref(s)))
        return s.value or 0

    def clear_cache(self) -> None:
        _check(lib().cheetah_cuda_seq_clear(self._h))

    def positions(self) -> int:
        n = C.c_size_t(0)
        _check(lib().cheetah_cuda_seq_positions(self._h, C.byref(n)))
        return n.value

    def kv_snapshot(self) -> CudaSnapshot:
        handle = C.c_void_p()
        _check(lib().cheetah_cuda_seq_snapshot(self._h, C.byref(handle)))
        return CudaSnapshot(handle, self.model)

    def restore_kv_prefix(self, snapshot: CudaSnapshot, positions: int) -> bool:
        _check(lib().cheetah_cuda_seq_restore_prefix(self._h, snapshot._h, positions))
        return True

    def kv_layer(self, layer: int):
        n = self.positions() * self.cfg["kv_heads"] * self.cfg["head_dim"]
        k = np.zeros(n, dtype=np.float32)
        v = np.zeros(n, dtype=np.float32)
        if n:
            _check(lib().cheetah_cuda_seq_export_kv(self._h, layer, _ptr(k), _ptr(v)))
        return k, v

    def close(self) -> None:
        if getattr(self, "_h", None):
            lib().cheetah_cuda_seq_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


# ---- op entries over torch CUDA tensors (caller-owned device memory) ----

def _stream_ptr(stream) -> Optional[int]:
    import torch
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def gemv_bf16(weight, x, stream=None):
    """y = W . x (`ops.rs:246`). weight: bf16 [rows, cols]; x: f32 [batch, cols]."""
    import torch
    assert weight.dtype == torch.bfloat16 and x.dtype == torch.float32 and weight.is_cuda
    rows, cols = weight.shape
    xb = x.reshape(-1, cols).contiguous()
    y = torch.empty(xb.shape[0], rows, dtype=torch.float32, device=x.device)
    _check(lib().cheetah_cuda_op_gemv_bf16(weight.data_ptr(), rows, cols, xb.data_ptr(),
                                           xb.shape[0], y.data_ptr(), _stream_ptr(stream)))
    return y


def quant_buffer_bytes(fmt: str, rows: int, cols: int) -> int:
    n = C.c_size_t(0)
    _check(lib().cheetah_cuda_quant_buffer_bytes(fmt.encode(), rows, cols, C.byref(n)))
    return n.value


def quantize(weight, fmt: str, stream=None):
    """Per-row q8/q4 quantisation (`q8.rs:91`, `q4.rs:126`) of bf16 [rows, cols]
    on the device; returns the uint8 buffer in the reference layout."""
    import torch
    assert weight.dtype == torch.bfloat16 and weight.is_cuda and weight.is_contiguous()
    rows, cols = weight.shape
    out = torch.empty(quant_buffer_bytes(fmt, rows, cols), dtype=torch.uint8, device=weight.device)
    fn = lib().cheetah_cuda_op_quantize_q8 if fmt == "q8" else lib().cheetah_cuda_op_quantize_q4
    _check(fn(weight.data_ptr(), rows, cols, out.data_ptr(), _stream_ptr(stream)))
    return out


def gemv_quant(buffer, fmt: str, rows: int, cols: int, x, stream=None):
    """y = W . x over a q8/q4 reference-layout buffer (`ops.rs:544`, `:586`)."""
    import torch
    xb = x.reshape(-1, cols).contiguous()
    y = torch.empty(xb.shape[0], rows, dtype=torch.float32, device=x.device)
    fn = lib().cheetah_cuda_op_gemv_q8 if fmt == "q8" else lib().cheetah_cuda_op_gemv_q4
    _check(fn(buffer.data_ptr(), rows, cols, xb.data_ptr(), xb.shape[0], y.data_ptr(), _stream_ptr(stream)))
    return y


def decode_attention(q, k_pool, v_pool, page_table, seq_lens, max_seq_len: int,
                     sliding_window: int = 0, out=None, stream=None, noalloc: bool = False):
    """Paged GQA decode attention (`ops.rs:1357-1467`). noalloc=True takes the
    entry point whose scratch is a fixed array inside the library (for callers
    that cannot let the library allocate device memory).

    q [B, q_heads, D] f32; k_pool/v_pool [pages, kv_heads, page_tokens, D]
    bf16 or f32; page_table [B, max_pages] int32; seq_lens [B] int32."""
    import torch
    B, qh, D = q.shape
    pages, kvh, pt, D2 = k_pool.shape
    assert D == D2 and v_pool.shape == k_pool.shape and page_table.dtype == torch.int32
    if out is None:
        out = torch.empty_like(q)
    args = DecodeAttentionArgs(
        q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(),
        KV_F32 if k_pool.dtype == torch.float32 else KV_BF16,
        page_table.data_ptr(), page_table.shape[1], seq_lens.data_ptr(), max_seq_len, pages, pt,
        B, qh, kvh, D, sliding_window, out.data_ptr())
    fn = lib().cheetah_cuda_op_decode_attention_noalloc if noalloc else lib().cheetah_cuda_op_decode_attention
    _check(fn(C.byref(args), _stream_ptr(stream)))
    return out


def prefill_attention(q, k_pool, v_pool, page_table, offset: int, sliding_window: int = 0,
                      out=None, stream=None):
    """Causal attention of a prefill chunk (`ops.rs:1357-1421` per query row).

    q [T, q_heads, D] bf16 (RoPE applied) for positions offset .. offset+T-1;
    k_pool/v_pool [pages, kv_heads, page_tokens, D] bf16 holding positions
    0 .. offset+T-1 of the sequence; page_table [max_pages] int32.
    Returns out [T, q_heads, D] bf16."""
    import torch
    T, qh, D = q.shape
    pages, kvh, pt, D2 = k_pool.shape
    assert D == D2 and v_pool.shape == k_pool.shape and page_table.dtype == torch.int32
    assert q.dtype == torch.bfloat16 and k_pool.dtype == torch.bfloat16 and q.is_contiguous()
    if out is None:
        out = torch.empty_like(q)
    args = PrefillAttentionArgs(q.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), page_table.data_ptr(),
                                page_table.numel(), pages, pt, T, offset, qh, kvh, D, sliding_window,
                                out.data_ptr())
    _check(lib().cheetah_cuda_op_prefill_attention(C.byref(args), _stream_ptr(stream)))
    return out


# ---- one step that verifies drafted tokens -------------------------------
#
# The calls take torch CUDA tensors of one device and run on its current
# stream, or on `stream`; what they allocate belongs to that stream, as if the
# call stood inside `torch.cuda.stream(stream)`. A step runs them once per
# layer or token, so the host's part of a call is kept short: torch's and the
# library's names are looked up once (`_bind`), checks stand inline.

_bound = None


class _Bound:
    """What the calls need of torch and of the library, looked up once."""

    def __init__(self):
        import torch
        self.current_device = torch._C._cuda_getDevice
        self.raw_stream = torch._C._cuda_getCurrentRawStream
        self.empty, self.empty_like = torch.empty, torch.empty_like
        self.i32, self.i64, self.u8 = torch.int32, torch.int64, torch.uint8
        self.bf16, self.f32 = torch.bfloat16, torch.float32
        handle = lib()
        for name in ("page_slots", "qk_norm_rope", "tree_attention", "token_logprobs"):
            setattr(self, name, getattr(handle, "cheetah_cuda_op_" + name))


def _bind() -> _Bound:
    global _bound
    _bound = _Bound()
    return _bound


def _context(device: int, stream):
    """The context in which `device` is current and, given one, `stream`."""
    import torch
    if stream is None:
        return torch.cuda.device(device)
    if stream.device.index != device:
        raise CheetahCudaError("the stream belongs to another device than the tensors")
    return torch.cuda.stream(stream)


def _fits(t, dtype, device: int) -> bool:
    return t.dtype is dtype and t.get_device() == device and t.is_contiguous()


def _refuse(op: str, device: int, **wanted) -> None:
    """Raises for the first of name=(tensor, dtype) that `_fits` refuses."""
    for name, (t, dtype) in wanted.items():
        if t is not None and not _fits(t, dtype, device):
            raise CheetahCudaError(f"{op}: {name} must be a contiguous {dtype} tensor on cuda:{device}")


class PageSlots(NamedTuple):
    row_starts: object  # int32 [batch + 1]
    seq_lens: object    # int32 [batch]
    positions: object   # int32 [max_tokens]
    seq_ids: object     # int32 [max_tokens]
    slots: object       # int32 [max_tokens]
    counts: object      # int32 [3]: rows asked for, pages taken, sequences refused


def page_slots(cached, new_tokens, free_pages, free_count, page_table, num_pages: int, page_tokens: int,
               max_tokens: int, stream=None) -> PageSlots:
    """Block tables and slot maps of a step from request lengths
    (`cheetah_cuda_op_page_slots`). cached, new_tokens int32 [B]; free_pages
    int32 [F], of which the first free_count (int32 [1]) are free; page_table
    int32 [B, max_pages] is extended in place. Sequences that do not fit are
    refused, not raised: see counts."""
    o = _bound or _bind()
    device = page_table.get_device()
    if device < 0 or page_table.dim() != 2:
        raise CheetahCudaError("page_slots: page_table must be a CUDA tensor [batch, max_pages]")
    if stream is not None or device != o.current_device():
        with _context(device, stream):
            return page_slots(cached, new_tokens, free_pages, free_count, page_table, num_pages, page_tokens, max_tokens)
    i32 = o.i32
    if not (_fits(cached, i32, device) and _fits(new_tokens, i32, device) and _fits(free_pages, i32, device)
            and _fits(free_count, i32, device) and _fits(page_table, i32, device)):
        _refuse("page_slots", device, cached=(cached, i32), new_tokens=(new_tokens, i32), free_pages=(free_pages, i32),
                free_count=(free_count, i32), page_table=(page_table, i32))
    B, width = page_table.shape
    if cached.numel() != B or new_tokens.numel() != B or free_count.numel() != 1:
        raise CheetahCudaError("page_slots: cached and new_tokens must hold one length per table row, free_count one number")
    if not (0 < max_tokens < 2 ** 31 and 0 < num_pages < 2 ** 31 and 0 < page_tokens < 2 ** 31):
        raise CheetahCudaError("page_slots: max_tokens, num_pages and page_tokens must be positive and below 2^31")
    # One buffer; the per-row outputs begin at 16-byte boundaries.
    pad = -max_tokens % 4
    row = max_tokens + pad
    buffer = o.empty(3 * row + 2 * B + 4, dtype=i32, device=page_table.device)
    if pad:
        positions, _, ids, _, slots, _, starts, lens, counts = buffer.split_with_sizes(
            (max_tokens, pad, max_tokens, pad, max_tokens, pad, B + 1, B, 3))
    else:
        positions, ids, slots, starts, lens, counts = buffer.split_with_sizes((row, row, row, B + 1, B, 3))
    at = buffer.data_ptr()
    args = PageSlotsArgs(cached.data_ptr(), new_tokens.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(),
                         free_pages.numel(), B, page_table.data_ptr(), width, num_pages, page_tokens, max_tokens,
                         at + 12 * row, at + 12 * row + 4 * (B + 1), at, at + 4 * row, at + 8 * row,
                         at + 12 * row + 8 * B + 4)
    if o.page_slots(args, o.raw_stream(device)):
        _check(-1)
    return PageSlots(starts, lens, positions, ids, slots, counts)


def qk_norm_rope(qkv, q_heads: int, kv_heads: int, positions, slots, rope_cos, rope_sin, k_pool, v_pool,
                 q_norm=None, k_norm=None, eps: float = 1e-6, q_out=None, stream=None):
    """Per-head RMSNorm of q and k, rotation at `positions`, K/V appended at
    `slots` (`cheetah_cuda_op_qk_norm_rope`). qkv [T, q_heads + 2 kv_heads, D]
    (or the same flattened) bf16 or f32, rows may be strided; positions, slots
    int32 [T], -1 skips; rope_cos, rope_sin f32 [max_positions, rotary_dim/2];
    the pools bf16 or f32, written in place. Returns q_out [T, q_heads, D]."""
    o = _bound or _bind()
    device = qkv.get_device()
    i32, f32, bf16 = o.i32, o.f32, o.bf16
    dtype, pool = qkv.dtype, k_pool.dtype
    if device < 0 or (dtype is not bf16 and dtype is not f32):
        raise CheetahCudaError("qk_norm_rope: qkv must be a bf16 or f32 CUDA tensor")
    if stream is not None or device != o.current_device():
        with _context(device, stream):
            return qk_norm_rope(qkv, q_heads, kv_heads, positions, slots, rope_cos, rope_sin, k_pool, v_pool, q_norm,
                                k_norm, eps, q_out)
    shape = k_pool.shape
    if len(shape) != 4 or shape != v_pool.shape or (pool is not bf16 and pool is not f32):
        raise CheetahCudaError("qk_norm_rope: the pools must be bf16 or f32 [pages, kv_heads, page_tokens, head_dim] of one shape")
    pages, kvh, pt, D = shape
    T = qkv.shape[0]
    width = (q_heads + 2 * kv_heads) * D
    strides = qkv.stride()
    if not (T > 0 and kvh == kv_heads and q_heads > 0 and qkv.numel() == T * width
            and (strides[1:] == (D, 1) and qkv.shape[2] == D or len(strides) == 2 and strides[1] == 1)):
        raise CheetahCudaError("qk_norm_rope: qkv must be [tokens, q_heads + 2 kv_heads, head_dim] with contiguous rows")
    if not (_fits(positions, i32, device) and _fits(slots, i32, device) and _fits(rope_cos, f32, device)
            and _fits(rope_sin, f32, device) and _fits(k_pool, pool, device) and _fits(v_pool, pool, device)
            and (q_norm is None or _fits(q_norm, f32, device)) and (k_norm is None or _fits(k_norm, f32, device))
            and (q_out is None or _fits(q_out, dtype, device))):
        _refuse("qk_norm_rope", device, positions=(positions, i32), slots=(slots, i32), rope_cos=(rope_cos, f32),
                rope_sin=(rope_sin, f32), k_pool=(k_pool, pool), v_pool=(v_pool, pool), q_norm=(q_norm, f32),
                k_norm=(k_norm, f32), q_out=(q_out, dtype))
    if positions.numel() != T or slots.numel() != T:
        raise CheetahCudaError("qk_norm_rope: positions and slots must hold one entry per row")
    table = rope_cos.shape
    if len(table) != 2 or table != rope_sin.shape:
        raise CheetahCudaError("qk_norm_rope: rope_cos and rope_sin must be [max_positions, rotary_dim/2]")
    if (q_norm is not None and q_norm.numel() != D) or (k_norm is not None and k_norm.numel() != D):
        raise CheetahCudaError("qk_norm_rope: a norm weight must be [head_dim]")
    if q_out is None:
        q_out = qkv.new_empty((T, q_heads, D))
    elif q_out.numel() != T * q_heads * D:
        raise CheetahCudaError("qk_norm_rope: q_out must be [tokens, q_heads, head_dim]")
    args = QkNormRopeArgs(qkv.data_ptr(), strides[0] if T > 1 else width, KV_F32 if dtype is f32 else KV_BF16,
                          KV_F32 if pool is f32 else KV_BF16, None if q_norm is None else q_norm.data_ptr(),
                          None if k_norm is None else k_norm.data_ptr(), eps, rope_cos.data_ptr(), rope_sin.data_ptr(),
                          table[0], 2 * table[1], positions.data_ptr(), slots.data_ptr(), T, q_heads, kv_heads, D,
                          q_out.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), pages, pt)
    if o.qk_norm_rope(args, o.raw_stream(device)):
        _check(-1)
    return q_out


def tree_attention(q, k_pool, v_pool, page_table, seq_lens, row_starts, tree_mask, positions=None,
                   sliding_window: int = 0, out=None, workspace=None, stream=None):
    """Attention of a batch's drafted nodes over their cached context and the
    nodes their mask rows name (`cheetah_cuda_op_tree_attention`). q [rows,
    q_heads, D] bf16 (rows may be strided); pools bf16; page_table int32 [B,
    max_pages]; seq_lens int32 [B]; row_starts int32 [B + 1]; tree_mask int64
    [rows, words], bit j % 64 of word j / 64 for node j; positions int32 [rows]
    (needed with a window). Rows behind the last sequence stay as `out` holds
    them. workspace: a uint8 tensor of `tree_attention_workspace` bytes that no
    overlapping call uses; None takes one from torch's allocator."""
    o = _bound or _bind()
    device = q.get_device()
    i32, bf16 = o.i32, o.bf16
    if device < 0 or q.dtype is not bf16 or q.dim() != 3:
        raise CheetahCudaError("tree_attention: q must be a bf16 CUDA tensor [rows, q_heads, head_dim]")
    if stream is not None or device != o.current_device():
        with _context(device, stream):
            return tree_attention(q, k_pool, v_pool, page_table, seq_lens, row_starts, tree_mask, positions,
                                  sliding_window, out, workspace)
    rows, qh, D = q.shape
    strides = q.stride()
    if rows < 1 or strides[1:] != (D, 1):
        raise CheetahCudaError("tree_attention: q must have contiguous rows")
    shape = k_pool.shape
    if len(shape) != 4 or shape != v_pool.shape or shape[3] != D:
        raise CheetahCudaError("tree_attention: the pools must be bf16 [pages, kv_heads, page_tokens, head_dim] of q's head_dim")
    if not (_fits(k_pool, bf16, device) and _fits(v_pool, bf16, device) and _fits(page_table, i32, device)
            and _fits(seq_lens, i32, device) and _fits(row_starts, i32, device) and _fits(tree_mask, o.i64, device)
            and (positions is None or _fits(positions, i32, device)) and (out is None or _fits(out, bf16, device))
            and (workspace is None or _fits(workspace, o.u8, device))):
        _refuse("tree_attention", device, k_pool=(k_pool, bf16), v_pool=(v_pool, bf16), page_table=(page_table, i32),
                seq_lens=(seq_lens, i32), row_starts=(row_starts, i32), tree_mask=(tree_mask, o.i64),
                positions=(positions, i32), out=(out, bf16), workspace=(workspace, o.u8))
    B = seq_lens.numel()
    table, mask = page_table.shape, tree_mask.shape
    if len(table) != 2 or table[0] != B or row_starts.numel() != B + 1:
        raise CheetahCudaError("tree_attention: page_table must be [batch, max_pages] and row_starts [batch + 1]")
    if len(mask) != 2 or mask[0] != rows:
        raise CheetahCudaError("tree_attention: tree_mask must be [rows, words]")
    if positions is not None and positions.numel() != rows:
        raise CheetahCudaError("tree_attention: positions must hold one entry per row")
    if not 0 <= sliding_window < 2 ** 31:
        raise CheetahCudaError("tree_attention: sliding_window must be 0 .. 2^31-1")
    if out is None:
        out = o.empty_like(q) if strides[0] == qh * D else q.new_empty((rows, qh, D))
    elif out.shape != q.shape:
        raise CheetahCudaError("tree_attention: out must have q's shape")
    if workspace is None:
        workspace = o.empty(tree_attention_workspace(D, device), dtype=o.u8, device=q.device)
    args = TreeAttentionArgs(q.data_ptr(), strides[0] if rows > 1 else qh * D, rows, k_pool.data_ptr(), v_pool.data_ptr(),
                             page_table.data_ptr(), table[1], shape[0], shape[2], seq_lens.data_ptr(),
                             row_starts.data_ptr(), B, tree_mask.data_ptr(), mask[1],
                             None if positions is None else positions.data_ptr(), sliding_window, qh, shape[1], D,
                             out.data_ptr(), workspace.data_ptr(), workspace.numel())
    if o.tree_attention(args, o.raw_stream(device)):
        _check(-1)
    return out


_tree_workspace_bytes: dict = {}  # (device, head_dim) -> bytes, a property of the GPU


def tree_attention_workspace(head_dim: int, device: Optional[int] = None) -> int:
    """Bytes of a `tree_attention` workspace on `device` (default: the current one)."""
    if device is None:
        device = (_bound or _bind()).current_device()
    size = _tree_workspace_bytes.get((device, head_dim))
    if size is None:
        # Every field but head_dim is the least that passes the checks.
        args = TreeAttentionArgs(rows=1, max_pages_per_seq=1, num_pages=1, page_tokens=16, batch=1, mask_words=1,
                                 q_heads=1, kv_heads=1, head_dim=head_dim)
        n = C.c_size_t(0)
        with _context(device, None):
            _check(lib().cheetah_cuda_op_tree_attention_workspace(C.byref(args), C.byref(n)))
        size = _tree_workspace_bytes[(device, head_dim)] = n.value
    return size


class TokenLogprobs(NamedTuple):
    logprob: object       # f32 [rows]
    entropy: object       # f32 [rows]
    rank: object          # int32 [rows]
    top_ids: object       # int32 [rows, top]
    top_logprobs: object  # f32 [rows, top]


def token_logprobs(logits, tokens, top: int = 0, stream=None) -> TokenLogprobs:
    """Log probability and rank of tokens[r] (int32) in row r of logits [rows,
    vocab] (f32 or bf16, rows may be strided), the row's entropy and its `top`
    likeliest tokens (`cheetah_cuda_op_token_logprobs`)."""
    o = _bound or _bind()
    device = logits.get_device()
    f32, dtype = o.f32, logits.dtype
    if device < 0 or (dtype is not f32 and dtype is not o.bf16) or logits.dim() != 2:
        raise CheetahCudaError("token_logprobs: logits must be a bf16 or f32 CUDA tensor [rows, vocab]")
    if stream is not None or device != o.current_device():
        with _context(device, stream):
            return token_logprobs(logits, tokens, top)
    rows, vocab = logits.shape
    strides = logits.stride()
    if rows < 1 or vocab < 1 or (strides[1] != 1 and vocab > 1):
        raise CheetahCudaError("token_logprobs: logits must have contiguous rows")
    if not _fits(tokens, o.i32, device):
        _refuse("token_logprobs", device, tokens=(tokens, o.i32))
    if tokens.dim() != 1 or tokens.numel() != rows:
        raise CheetahCudaError("token_logprobs: tokens must be [rows]")
    if not 0 <= top <= min(32, vocab):
        raise CheetahCudaError("token_logprobs: top must be at most 32 and at most vocab")
    rank = o.empty_like(tokens)
    logprob = o.empty_like(tokens, dtype=f32)
    entropy = o.empty_like(logprob)
    ids, best = tokens.new_empty((rows, top)), logprob.new_empty((rows, top))
    args = TokenLogprobsArgs(logits.data_ptr(), strides[0] if rows > 1 else vocab, KV_F32 if dtype is f32 else KV_BF16,
                             rows, vocab, tokens.data_ptr(), top, logprob.data_ptr(), rank.data_ptr(),
                             entropy.data_ptr(), ids.data_ptr() if top else None, best.data_ptr() if top else None)
    if o.token_logprobs(args, o.raw_stream(device)):
        _check(-1)
    return TokenLogprobs(logprob, entropy, rank, ids, best)
