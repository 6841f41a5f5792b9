"""ctypes mirror of the gfx950 C ABI (include/fortai_hip_backend.h).

Python counterpart of the reference's iso_c_binding wrapper
(src/backend/cuda/fortai_backend_cuda.f90): opaque handles with create /
destroy, and every nonzero return code raised as ``BackendError`` with the
context's last error message (the wrapper maps them to status_t,
fortai_backend_cuda.f90:418-431).  There is no CPU fallback: if
``libfortai_hip.so`` is missing or no GPU is visible, creating a context raises.
"""

from __future__ import annotations

import ctypes as C
import os
from typing import Optional, Sequence

import numpy as np

# the in-tree build; FORTAI_HIP_LIBRARY names another build of the same library
LIB_PATH = os.environ.get("FORTAI_HIP_LIBRARY") or \
    os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "libfortai_hip.so")

OK, INVALID, RUNTIME_ERROR = 0, 1, 2

_vp, _i, _i64, _sz, _f = C.c_void_p, C.c_int, C.c_int64, C.c_size_t, C.c_float
_d = C.c_double
_fp, _i64p, _u16p = C.POINTER(C.c_float), C.POINTER(C.c_int64), C.POINTER(C.c_uint16)
_vpp = C.POINTER(C.c_void_p)

# name -> argtypes (all return int unless listed in _RESTYPE)
_SIGNATURES = {
    "fortai_hip_q8_context_create": [_i, _vpp],
    "fortai_hip_q8_context_destroy": [_vp],
    "fortai_hip_q8_context_set_position": [_vp, _i],
    "fortai_hip_q8_context_capture_begin": [_vp],
    "fortai_hip_q8_context_capture_end": [_vp],
    "fortai_hip_q8_context_graph_launch": [_vp],
    "fortai_hip_q8_context_synchronize": [_vp],
    "fortai_hip_q8_context_scratch_bytes": [_vp, C.POINTER(C.c_size_t)],
    "fortai_hip_q8_context_timer_start": [_vp],
    "fortai_hip_q8_context_timer_stop": [_vp, _fp],
    "fortai_hip_q8_weights_upload": [_vp, _vp, _sz, _i, _i, _vpp],
    "fortai_hip_q8_weights_destroy": [_vp],
    "fortai_hip_q8_device_buffer_create": [_vp, _sz, _vpp],
    "fortai_hip_q8_device_buffer_destroy": [_vp, _vp],
    "fortai_hip_q8_device_buffer_upload": [_vp, _vp, _vp, _sz],
    "fortai_hip_q8_device_buffer_upload_ptr": [_vp, _vp, _vp, _sz],
    "fortai_hip_q8_device_buffer_download": [_vp, _vp, _vp, _sz],
    "fortai_hip_q8_matvec_resident": [_vp, _vp, _vp, _vp, _fp],
    "fortai_hip_q8_matvec_device_f32": [_vp, _vp, _vp, _sz, _vp, _sz],
    "fortai_hip_qwen35_embedding_device": [_vp, _vp, _i64, _vp, _sz],
    "fortai_hip_qwen35_copy_device": [_vp, _vp, _vp, _sz],
    "fortai_hip_qwen35_add_device": [_vp, _vp, _vp, _vp, _sz],
    "fortai_hip_qwen35_rms_norm_device": [_vp, _vp, _vp, _vp, _sz, _f],
    "fortai_hip_q8_matvec_host": [_vp, _vp, _vp, _sz, _vp, _sz, _fp],
    "fortai_hip_q8_matvec_host_pair": [_vp, _vp, _vp, _vp, _sz, _vp, _sz, _vp, _sz, _fp],
    "fortai_hip_q8_matvec_host_triplet": [_vp, _vp, _vp, _vp, _vp, _sz, _vp, _sz, _vp, _sz, _vp, _sz, _fp],
    "fortai_hip_q8_matvec_host_triplet_contiguous": [_vp, _vp, _vp, _vp, _vp, _sz, _vp, _sz, _fp],
    "fortai_hip_q8_ffn_host": [_vp, _vp, _vp, _vp, _vp, _sz, _vp, _sz, _fp],
    "fortai_hip_q8_ffn_device": [_vp, _vp, _vp, _vp, _vp, _sz, _vp, _sz],
    "fortai_hip_qwen35_recurrent_create": [_vp, _vp, _vp, _vp, _vp, _vp, _vp, _sz, _i, _i, _vp, _sz, _vp, _sz,
                                           _vp, _sz, _i, _i, _i, _i, _i, _f, _vpp],
    "fortai_hip_qwen35_recurrent_destroy": [_vp],
    "fortai_hip_qwen35_recurrent_reset": [_vp],
    "fortai_hip_qwen35_recurrent_run": [_vp, _vp, _sz, _vp, _sz, _fp],
    "fortai_hip_qwen35_recurrent_run_device": [_vp, _vp, _sz, _vp, _sz],
    "fortai_hip_qwen35_attention_create": [_vp, _vp, _vp, _vp, _vp, _vp, _sz, _vp, _sz, _i, _i, _i, _i, _i, _i,
                                           _f, _f, _vpp],
    "fortai_hip_qwen35_attention_destroy": [_vp],
    "fortai_hip_qwen35_attention_reset": [_vp],
    "fortai_hip_qwen35_attention_run_device": [_vp, _vp, _sz, _i, _vp, _sz],
    "fortai_hip_q8_last_error": [_vp],
    "fortai_hip_f16_weights_upload": [_vp, _vp, _sz, _i, _i, _vpp],
    "fortai_hip_f16_weights_destroy": [_vp],
    "fortai_hip_f16_matvec_device": [_vp, _vp, _vp, _sz, _vp, _sz, _vp],
    "fortai_hip_qwen35_embedding_f16_device": [_vp, _vp, _i64, _vp, _sz],
    "fortai_hip_argmax_device": [_vp, _vp, _sz, _vp],
    "fortai_hip_q8_quantize_device": [_vp, _vp, _sz, _vp, _vp],
    "fortai_hip_q8_block_dots_device": [_vp, _vp, _vp, _vp],
    "fortai_hip_q8_batch_matvec_noalloc": [_vp, _vp, _vp, _i, _vp],
    "fortai_hip_q8_batch_matvec_device": [_vp, _vp, _vp, _i, _vp, _fp],
    "fortai_hip_q8_pack_bytes": [_i, _i],
    "fortai_hip_q8_weights_pack": [_vp, _vp, _sz],
    "fortai_hip_q8_weights_upload_packed": [_vp, _vp, _sz, _i, _i, _vpp],
    "fortai_hip_q8_tokens_bytes": [_i, _i],
    "fortai_hip_q8_quantize_tokens_device": [_vp, _vp, _i, _i, _vp],
    "fortai_hip_q8_mmq_device": [_vp, _vp, _vp, _i, _vp, _vp, _fp],
    "fortai_hip_q8_mmq_exact_device": [_vp, _vp, _vp, _i, _vp, _vp, _fp],
    "fortai_hip_q8_mmq_block_dots": [_vp, _vp, _vp, _i, _vp],
    "fortai_hip_q8_mmq_chunks_device": [_vp, _vp, _vp, _i, _i, _vp, _vp],
    "fortai_hip_qwen35_recurrent_core_steps_device": [_vp, _vp, _vp, _vp, _i, _vp],
    "fortai_hip_qwen35_recurrent_core_device": [_vp, _vp, _vp, _vp, _vp],
    "fortai_hip_qwen35_recurrent_state_download": [_vp, _vp, _sz, _vp, _sz],
    "fortai_hip_qwen35_recurrent_state_upload": [_vp, _vp, _sz, _vp, _sz],
    "fortai_hip_qwen35_attention_core_device": [_vp, _vp, _vp, _vp, _vp],
    "fortai_hip_qwen35_attention_prefill_core_device": [_vp, _vp, _vp, _vp, _i, _i, _vp],
    "fortai_hip_qwen35_attention_cache_download": [_vp, _vp, _vp, _i],
    "fortai_hip_qwen35_attention_cache_upload": [_vp, _vp, _vp, _i],
    "fortai_hip_qwen35_decoder_create": [_vp, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _vp,
                                         _i, _f, _vpp],
    "fortai_hip_qwen35_decoder_destroy": [_vp],
    "fortai_hip_qwen35_decoder_reset": [_vp],
    "fortai_hip_qwen35_decoder_forward": [_vp, _i64, _i, _vp, _vp],
    "fortai_hip_qwen35_decoder_generate": [_vp, _i64, _i, _i, _vp],
    "fortai_hip_qwen35_decoder_replay": [_vp, _i],
    "fortai_hip_qwen35_decoder_logits": [_vp, _vpp],
    "fortai_hip_qwen35_decoder_trace": [_vp, _i, _i, _vp],
    "fortai_hip_qwen35_decoder_status": [_vp],
    "fortai_hip_qwen35_decoder_plan": [_vp, _vp, _sz, C.POINTER(C.c_size_t)],
    "fortai_hip_qwen35_batch_plan": [_vp, _i, _vp, _sz, C.POINTER(C.c_size_t)],
    "fortai_hip_qwen35_batch_create": [_vp, _i, _i, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp,
                                       _vp, _i, _f, _vpp],
    "fortai_hip_qwen35_batch_destroy": [_vp],
    "fortai_hip_qwen35_batch_reset": [_vp],
    "fortai_hip_qwen35_batch_forward": [_vp, _vp, _vp, _vp, _vp],
    "fortai_hip_qwen35_batch_generate": [_vp, _vp, _vp, _i, _vp],
    "fortai_hip_qwen35_batch_replay": [_vp, _i],
    "fortai_hip_qwen35_batch_logits": [_vp, _vpp],
    "fortai_hip_qwen35_batch_prefill": [_vp, _vp, _i, _vp, _vp, _fp],
    "fortai_hip_qwen35_attention_set_exact_max": [_vp, _i],
    "fortai_hip_qwen35_attention_set_test_options": [_vp, _i, _i],
    "fortai_hip_qwen35_decoder_set_mode": [_vp, _i],
    "fortai_hip_qwen35_batch_set_mode": [_vp, _i],
    "fortai_hip_qwen35_batch_set_prefill_mode": [_vp, _i],
    "fortai_hip_rope_create": [_vp, _i, _i, _d, _i, _d, _i, _d, _d, _d, _vpp],
    "fortai_hip_rope_destroy": [_vp],
    "fortai_hip_rope_device": [_vp, _i, _vp, _i64, _i64, _i, _i, _i, _vp, _vp, _f, _vp, _i64, _i64],
    "fortai_hip_kv8_bytes": [_i, _i, _i, _i, _i],
    "fortai_hip_kv8_create": [_vp, _i, _i, _i, _i, _i, _vp, _sz, _vpp],
    "fortai_hip_kv8_destroy": [_vp],
    "fortai_hip_kv8_append_device": [_vp, _i, _vp, _i, _vp, _i64, _vp, _i64],
    "fortai_hip_kv8_read_device": [_vp, _i, _vp, _i, _vp, _i64, _vp, _i64],
    "fortai_hip_kv8_attention_device": [_vp, _i, _vp, _i, _vp, _i64, _i64, _vp, _i, _f, _i, _vp, _i64],
    "fortai_hip_kv8_copy_pages": [_vp, _vp, _vp, _i],
    "fortai_hip_verifier_create": [_vp, _i, _i, _i, _vpp],
    "fortai_hip_verifier_destroy": [_vp],
    "fortai_hip_verify_drafts_device": [_vp, _i, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _i, _vp, _i, _vp, _vp, _vp],
    "fortai_hip_kv8_pages_create": [_i, _i, _i, _i, _vpp],
    "fortai_hip_kv8_pages_destroy": [_vp],
    "fortai_hip_kv8_pages_extend": [_vp, _i, _i, _vp, _vp, _vp],
    "fortai_hip_kv8_pages_fork": [_vp, _i, _i, _i64],
    "fortai_hip_kv8_pages_truncate": [_vp, _i, _i64],
    "fortai_hip_kv8_pages_compact": [_vp, _vp, _vp, _i, _vp],
    "fortai_hip_kv8_pages_length": [_vp, _i],
    "fortai_hip_kv8_pages_free_count": [_vp],
    "fortai_hip_kv8_pages_tables": [_vp, _vp, _i, _vp, _i],
    "fortai_hip_kv8_shared_attention_device": [_vp, _i, _vp, _vp, _i, _vp, _i64, _i64, _vp, _i, _f, _i, _i, _vp, _i64],
    "fortai_hip_kv8_pages_groups": [_vp, _vp, _i, _vp, _vp, _vp, _vp],
    "fortai_hip_norm_tokens_device": [_vp, _i, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i, _f, _vp, _i64, _i, _i, _vp, _i64,
                                      _vp],
    "fortai_hip_q8_tokens_read_device": [_vp, _i, _vp, _i, _i, _vp, _i64],
    "fortai_hip_logits_adjust_device": [_vp, _i, _vp, _i64, _i, _i, _i, _vp, _vp, _vp, _i64],
    "fortai_hip_gdn_bytes": [_i, _i, _i, _i, _i, _i, _i],
    "fortai_hip_gdn_create": [_vp, _i, _i, _i, _i, _i, _i, _i, _i, _vp, _sz, _vpp],
    "fortai_hip_gdn_destroy": [_vp],
    "fortai_hip_gdn_run_device": [_vp, _i, _vp, _i, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _vp, _vp, _f, _vp, _i64],
    "fortai_hip_gdn_copy_slots": [_vp, _vp, _vp, _i],
}
_RESTYPE = {"fortai_hip_q8_last_error": C.c_char_p, "fortai_hip_q8_tokens_bytes": C.c_size_t,
            "fortai_hip_q8_pack_bytes": C.c_size_t, "fortai_hip_kv8_bytes": C.c_size_t,
            "fortai_hip_kv8_pages_length": C.c_int64, "fortai_hip_gdn_bytes": C.c_size_t}

_lib: Optional[C.CDLL] = None


# option values of include/fortai_hip_backend.h
DECODER_DIRECT = 1
DECODER_MATVEC_ONLY = 2
DECODER_FAMILIES = {"matvec": 2, "gdn": 4, "attention": 8, "head": 16}
PREFILL_MODES = {"exact": 0, "matvec": 1, "fast": 2}
DTYPES = {"f32": 0, "f16": 1, "bf16": 2}
ROPE_SCALINGS = {"none": 0, "linear": 1, "yarn": 2}


class BackendError(RuntimeError):
    def __init__(self, code: int, what: str, message: str = ""):
        super().__init__(f"{what} failed with code {code}" + (f": {message}" if message else ""))
        self.code = code


def load(path: str = LIB_PATH) -> C.CDLL:
    """Load libfortai_hip.so (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(path):
        raise FileNotFoundError(f"{path} is missing: run fortai_amd.build.build() (no CPU fallback exists)")
    lib = C.CDLL(path)
    for name, args in _SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = _RESTYPE.get(name, C.c_int)
    _lib = lib
    return lib


def exported_symbols() -> Sequence[str]:
    return list(_SIGNATURES)


def _plan(ctx, name: str, *args):
    """Read a recorded plan: [(operation, kernel, batch)] (PlanIR steps)."""
    need = C.c_size_t()
    ctx.call(name, *args, None, 0, C.byref(need))
    buf = C.create_string_buffer(need.value)
    ctx.call(name, *args, buf, need.value, C.byref(need))
    steps = []
    for line in buf.value.decode().splitlines():
        op, kernel, batch = line.split("\t")
        steps.append((op, kernel, int(batch)))
    return steps


def _ptr(a: np.ndarray) -> C.c_void_p:
    return C.c_void_p(a.ctypes.data)


class LogitRules(C.Structure):
    """fortai_hip_logit_rules: what Context.adjust_logits applies."""

    _fields_ = [("window", _i), ("mask_count", _i), ("penalties", _vp), ("tokens", _vp), ("history", _vp),
                ("history_lengths", _vp), ("bias", _vp), ("masks", _vp), ("mask_of", _vp), ("history_pitch", _i64),
                ("bias_pitch", _i64), ("mask_pitch", _i64)]


class Context:
    """A device context: stream, device position/token, scratch (fortai_cuda_q8_context)."""

    def __init__(self, device: int = 0):
        self.lib = load()
        h = C.c_void_p()
        rc = self.lib.fortai_hip_q8_context_create(device, C.byref(h))
        if rc != OK:
            raise BackendError(rc, "fortai_hip_q8_context_create (is a GPU visible?)")
        self.h = h

    def check(self, rc: int, what: str) -> None:
        if rc != OK:
            msg = self.lib.fortai_hip_q8_last_error(self.h)
            raise BackendError(rc, what, msg.decode() if msg else "")

    def call(self, name: str, *args) -> None:
        self.check(getattr(self.lib, name)(*args), name)

    def close(self) -> None:
        if getattr(self, "h", None):
            self.lib.fortai_hip_q8_context_destroy(self.h)
            self.h = None

    def set_position(self, position: int) -> None:
        self.call("fortai_hip_q8_context_set_position", self.h, position)

    def scratch_bytes(self) -> int:
        """Bytes of the scratch buffers this context has allocated on demand."""
        n = C.c_size_t()
        self.call("fortai_hip_q8_context_scratch_bytes", self.h, C.byref(n))
        return n.value

    def synchronize(self) -> None:
        self.call("fortai_hip_q8_context_synchronize", self.h)

    def timer_start(self) -> None:
        self.call("fortai_hip_q8_context_timer_start", self.h)

    def timer_stop(self) -> float:
        ms = C.c_float()
        self.call("fortai_hip_q8_context_timer_stop", self.h, C.byref(ms))
        return float(ms.value)

    def capture_begin(self) -> None:
        self.call("fortai_hip_q8_context_capture_begin", self.h)

    def capture_end(self) -> None:
        self.call("fortai_hip_q8_context_capture_end", self.h)

    def graph_launch(self) -> None:
        self.call("fortai_hip_q8_context_graph_launch", self.h)

    # ---- around a step's products (device arrays as addresses or DeviceBuffers; dense unless pitches are given)
    def norm_tokens(self, x, rows: int, width: int, dtype: str = "f32", residual=None, sum=None, norm=None,
                    group: Optional[int] = None, eps: float = 1e-6, gate=None, output=None, tokens=None,
                    x_pitch: Optional[int] = None, residual_pitch: Optional[int] = None, sum_pitch: Optional[int] = None,
                    gate_pitch: Optional[int] = None, output_pitch: Optional[int] = None) -> None:
        """x [rows][width] (+ residual -> sum), RMS norm over groups, gate -> output and 8-bit tokens
        (fortai_hip_norm_tokens_device)."""
        pitch = lambda p: width if p is None else p
        self.check(self.lib.fortai_hip_norm_tokens_device(
            self.h, DTYPES[dtype], _dev(x), pitch(x_pitch), _dev(residual), pitch(residual_pitch), _dev(sum), pitch(sum_pitch),
            _dev(norm), width if group is None else group, eps, _dev(gate), pitch(gate_pitch), rows, width, _dev(output),
            pitch(output_pitch), _dev(tokens)), "fortai_hip_norm_tokens_device")

    def tokens_read(self, tokens, rows: int, width: int, out, dtype: str = "f32", out_pitch: Optional[int] = None) -> None:
        """The values of a buffer of 8-bit tokens as rows."""
        self.check(self.lib.fortai_hip_q8_tokens_read_device(self.h, DTYPES[dtype], _dev(tokens), rows, width, _dev(out),
                                                             width if out_pitch is None else out_pitch),
                   "fortai_hip_q8_tokens_read_device")

    def adjust_logits(self, logits, vocab: int, out, row_starts, sequences: int, rows: int, dtype: str = "f32", tokens=None,
                      history=None, history_pitch: Optional[int] = None, history_lengths=None, window: int = 0, penalties=None, bias=None,
                      bias_pitch: int = 0, masks=None, mask_count: int = 0, mask_pitch: Optional[int] = None, mask_of=None,
                      pitch: Optional[int] = None, out_pitch: Optional[int] = None) -> None:
        """Penalties for repeated tokens, biases and masks on logits [rows][vocab] (fortai_hip_logits_adjust_device).  A
        history [sequences][history_pitch] comes with its pitch, which is all of a sequence's that can count."""
        if history_pitch is None:
            history_pitch = 0 if history is None else -1  # refused: a pitch of nothing would count nothing
        rules = LogitRules(window, mask_count, _dev(penalties), _dev(tokens), _dev(history), _dev(history_lengths), _dev(bias),
                           _dev(masks), _dev(mask_of), history_pitch, bias_pitch,
                           (vocab + 31) // 32 if mask_pitch is None else mask_pitch)
        self.check(self.lib.fortai_hip_logits_adjust_device(
            self.h, DTYPES[dtype], _dev(logits), vocab if pitch is None else pitch, rows, vocab, sequences, _dev(row_starts),
            C.addressof(rules), _dev(out), vocab if out_pitch is None else out_pitch), "fortai_hip_logits_adjust_device")

    # ---- device buffers
    def alloc(self, nbytes: int) -> "DeviceBuffer":
        return DeviceBuffer(self, nbytes)

    def upload_array(self, a: np.ndarray) -> "DeviceBuffer":
        a = np.ascontiguousarray(a)
        buf = DeviceBuffer(self, max(a.nbytes, 1))
        buf.upload(a)
        return buf


class DeviceBuffer:
    def __init__(self, ctx: Context, nbytes: int):
        self.ctx = ctx
        self.nbytes = int(nbytes)
        h = C.c_void_p()
        ctx.call("fortai_hip_q8_device_buffer_create", ctx.h, self.nbytes, C.byref(h))
        self.h = h

    @property
    def ptr(self) -> C.c_void_p:
        return self.h

    def upload(self, a: np.ndarray) -> None:
        a = np.ascontiguousarray(a)
        if a.nbytes > self.nbytes:
            raise ValueError("upload larger than the buffer")
        self.ctx.call("fortai_hip_q8_device_buffer_upload", self.ctx.h, self.h, _ptr(a), a.nbytes)

    def download(self, dtype, count: Optional[int] = None) -> np.ndarray:
        dtype = np.dtype(dtype)
        count = self.nbytes // dtype.itemsize if count is None else count
        out = np.empty(count, dtype=dtype)
        self.ctx.call("fortai_hip_q8_device_buffer_download", self.ctx.h, _ptr(out), self.h, out.nbytes)
        return out

    def free(self) -> None:
        if self.h:
            self.ctx.lib.fortai_hip_q8_device_buffer_destroy(self.ctx.h, self.h)
            self.h = None


class Q8Weights:
    """Resident Q8_0 matrix (GGUF bytes [rows][width/32][34])."""

    def __init__(self, ctx: Context, gguf_bytes: Optional[np.ndarray], rows: int, width: int,
                 packed: Optional[np.ndarray] = None):
        self.ctx, self.rows, self.width = ctx, rows, width
        h = C.c_void_p()
        if packed is not None:
            planes = np.ascontiguousarray(packed).view(np.uint8)
            ctx.call("fortai_hip_q8_weights_upload_packed", ctx.h, _ptr(planes), planes.nbytes, rows, width,
                     C.byref(h))
        else:
            data = np.ascontiguousarray(gguf_bytes).view(np.uint8)
            ctx.call("fortai_hip_q8_weights_upload", ctx.h, _ptr(data), data.nbytes, rows, width, C.byref(h))
        self.h = h

    @classmethod
    def from_packed(cls, ctx: Context, planes: np.ndarray, rows: int, width: int) -> "Q8Weights":
        """A resident matrix from planes written by pack() (no repack)."""
        return cls(ctx, None, rows, width, packed=planes)

    def pack(self) -> np.ndarray:
        """The resident (repacked) planes, for a weight-pack cache."""
        n = self.ctx.lib.fortai_hip_q8_pack_bytes(self.rows, self.width)
        out = np.empty(n, dtype=np.uint8)
        self.ctx.call("fortai_hip_q8_weights_pack", self.h, _ptr(out), n)
        return out

    def free(self) -> None:
        if self.h:
            self.ctx.lib.fortai_hip_q8_weights_destroy(self.h)
            self.h = None


class F16Weights:
    """Resident fp16 matrix (GGUF F16 row-major [rows][width])."""

    def __init__(self, ctx: Context, bits: np.ndarray, rows: int, width: int):
        self.ctx, self.rows, self.width = ctx, rows, width
        data = np.ascontiguousarray(bits).view(np.uint16)
        h = C.c_void_p()
        ctx.call("fortai_hip_f16_weights_upload", ctx.h, _ptr(data), data.nbytes, rows, width, C.byref(h))
        self.h = h

    def free(self) -> None:
        if self.h:
            self.ctx.lib.fortai_hip_f16_weights_destroy(self.h)
            self.h = None


class Recurrent:
    """Qwen3.5 Gated DeltaNet layer (fortai_cuda_qwen35_recurrent)."""

    def __init__(self, ctx: Context, qkv: Q8Weights, gate: Q8Weights, alpha: Q8Weights, beta: Q8Weights,
                 out: Q8Weights, conv_w: np.ndarray, conv_size: int, conv_kernel: int, ssm_a: np.ndarray,
                 ssm_dt: np.ndarray, ssm_norm: np.ndarray, state_size: int, key_heads: int, value_heads: int,
                 head_size: int, inner_size: int, eps: float):
        self.ctx = ctx
        self.dims = dict(conv_size=conv_size, conv_kernel=conv_kernel, state_size=state_size, key_heads=key_heads,
                         value_heads=value_heads, head_size=head_size, inner_size=inner_size)
        arrays = [np.ascontiguousarray(a, dtype=np.float32) for a in (conv_w, ssm_a, ssm_dt, ssm_norm)]
        h = C.c_void_p()
        ctx.call("fortai_hip_qwen35_recurrent_create", ctx.h, qkv.h, gate.h, alpha.h, beta.h, out.h,
                 _ptr(arrays[0]), arrays[0].nbytes, conv_size, conv_kernel, _ptr(arrays[1]), arrays[1].nbytes,
                 _ptr(arrays[2]), arrays[2].nbytes, _ptr(arrays[3]), arrays[3].nbytes, state_size, key_heads,
                 value_heads, head_size, inner_size, eps, C.byref(h))
        self.h = h

    def reset(self) -> None:
        self.ctx.call("fortai_hip_qwen35_recurrent_reset", self.h)

    def state(self):
        d = self.dims
        gdn = np.empty(d["value_heads"] * d["head_size"] ** 2, dtype=np.float32)
        conv = np.empty((d["conv_kernel"] - 1) * d["conv_size"], dtype=np.float32)
        self.ctx.call("fortai_hip_qwen35_recurrent_state_download", self.h, _ptr(gdn), gdn.nbytes, _ptr(conv),
                      conv.nbytes)
        return gdn, conv

    def set_state(self, gdn: np.ndarray, conv: np.ndarray) -> None:
        gdn = np.ascontiguousarray(gdn, dtype=np.float32)
        conv = np.ascontiguousarray(conv, dtype=np.float32)
        self.ctx.call("fortai_hip_qwen35_recurrent_state_upload", self.h, _ptr(gdn), gdn.nbytes, _ptr(conv),
                      conv.nbytes)

    def free(self) -> None:
        if self.h:
            self.ctx.lib.fortai_hip_qwen35_recurrent_destroy(self.h)
            self.h = None


class Attention:
    """Qwen3.5 gated full-attention layer (fortai_cuda_qwen35_attention)."""

    def __init__(self, ctx: Context, q: Q8Weights, k: Q8Weights, v: Q8Weights, o: Q8Weights, q_norm: np.ndarray,
                 k_norm: np.ndarray, heads: int, kv_heads: int, head_size: int, value_size: int, max_context: int,
                 rope_dim: int, rope_base: float, eps: float):
        self.ctx = ctx
        self.dims = dict(heads=heads, kv_heads=kv_heads, head_size=head_size, value_size=value_size,
                         max_context=max_context)
        qn = np.ascontiguousarray(q_norm, dtype=np.float32)
        kn = np.ascontiguousarray(k_norm, dtype=np.float32)
        h = C.c_void_p()
        ctx.call("fortai_hip_qwen35_attention_create", ctx.h, q.h, k.h, v.h, o.h, _ptr(qn), qn.nbytes, _ptr(kn),
                 kn.nbytes, heads, kv_heads, head_size, value_size, max_context, rope_dim, rope_base, eps,
                 C.byref(h))
        self.h = h

    def reset(self) -> None:
        self.ctx.call("fortai_hip_qwen35_attention_reset", self.h)

    def set_exact_max(self, exact_max: int) -> None:
        """Positions up to which the output keeps the reference's summation
        orders (default 8192); split-K beyond.  Before a decoder is created."""
        self.ctx.call("fortai_hip_qwen35_attention_set_exact_max", self.h, exact_max)

    def set_test_options(self, z_skew: int = 0, force_wide: bool = False) -> None:
        """Test only: shift the Z candidate windows; the wide output kernel for one sequence."""
        self.ctx.call("fortai_hip_qwen35_attention_set_test_options", self.h, z_skew, 1 if force_wide else 0)

    def cache(self, positions: int):
        d = self.dims
        k = np.empty(positions * d["kv_heads"] * d["head_size"], dtype=np.uint16)
        v = np.empty(positions * d["kv_heads"] * d["value_size"], dtype=np.uint16)
        self.ctx.call("fortai_hip_qwen35_attention_cache_download", self.h, _ptr(k), _ptr(v), positions)
        return k, v

    def set_cache(self, k: np.ndarray, v: np.ndarray, positions: int) -> None:
        k = np.ascontiguousarray(k, dtype=np.uint16)
        v = np.ascontiguousarray(v, dtype=np.uint16)
        self.ctx.call("fortai_hip_qwen35_attention_cache_upload", self.h, _ptr(k), _ptr(v), positions)

    def free(self) -> None:
        if self.h:
            self.ctx.lib.fortai_hip_qwen35_attention_destroy(self.h)
            self.h = None


class Decoder:
    """Fused whole-token decoder (one captured HIP graph per step)."""

    def __init__(self, ctx: Context, recurrent: Sequence[Optional[Recurrent]],
                 attention: Sequence[Optional[Attention]], ffn_gate: Sequence[Q8Weights],
                 ffn_up: Sequence[Q8Weights], ffn_down: Sequence[Q8Weights], attn_norm: Sequence[np.ndarray],
                 post_norm: Sequence[np.ndarray], output_norm: np.ndarray, hidden: int,
                 embedding, output, max_context: int, eps: float, vocab: int):
        self.ctx, self.vocab, self.max_context = ctx, vocab, max_context
        n = len(ffn_gate)

        def harr(items):
            return (C.c_void_p * n)(*[(x.h if x is not None else None) for x in items])

        self._norms = [np.ascontiguousarray(a, dtype=np.float32) for a in list(attn_norm) + list(post_norm)]
        an = (C.c_void_p * n)(*[_ptr(a) for a in self._norms[:n]])
        pn = (C.c_void_p * n)(*[_ptr(a) for a in self._norms[n:]])
        self._onorm = np.ascontiguousarray(output_norm, dtype=np.float32)
        e16 = embedding.h if isinstance(embedding, F16Weights) else None
        e8 = embedding.h if isinstance(embedding, Q8Weights) else None
        o16 = output.h if isinstance(output, F16Weights) else None
        o8 = output.h if isinstance(output, Q8Weights) else None
        h = C.c_void_p()
        ctx.call("fortai_hip_qwen35_decoder_create", ctx.h, n, harr(recurrent), harr(attention), harr(ffn_gate),
                 harr(ffn_up), harr(ffn_down), an, pn, _ptr(self._onorm), hidden, e16, e8, o16, o8, max_context,
                 eps, C.byref(h))
        self.h = h
        self.logits = np.zeros(vocab, dtype=np.float32)

    def reset(self) -> None:
        self.ctx.call("fortai_hip_qwen35_decoder_reset", self.h)

    def set_mode(self, direct: bool = False, matvec_only: bool = False, only: Sequence[str] = ()) -> None:
        """direct: enqueue the kernels every step instead of a graph replay
        (kernel tracing); matvec_only / only: timing probes that enqueue only
        those kernel families ("matvec", "gdn", "attention", "head")."""
        flags = (DECODER_DIRECT if direct else 0) | (DECODER_MATVEC_ONLY if matvec_only else 0)
        for f in only:
            flags |= DECODER_FAMILIES[f]
        self.ctx.call("fortai_hip_qwen35_decoder_set_mode", self.h, flags)

    def forward(self, token: int, position: int, want_logits: bool = True) -> int:
        nxt = np.zeros(1, dtype=np.int64)
        self.ctx.call("fortai_hip_qwen35_decoder_forward", self.h, token, position,
                      _ptr(self.logits) if want_logits else None, _ptr(nxt))
        return int(nxt[0])

    def generate(self, token: int, position: int, steps: int) -> np.ndarray:
        trace = np.zeros(steps, dtype=np.int64)
        self.ctx.call("fortai_hip_qwen35_decoder_generate", self.h, token, position, steps, _ptr(trace))
        return trace

    def replay(self, steps: int) -> None:
        self.ctx.call("fortai_hip_qwen35_decoder_replay", self.h, steps)

    def trace(self, first: int, count: int) -> np.ndarray:
        """The greedy ids chosen at positions first .. first+count-1."""
        out = np.zeros(count, dtype=np.int64)
        self.ctx.call("fortai_hip_qwen35_decoder_trace", self.h, first, count, _ptr(out))
        return out

    def check(self) -> None:
        """Wait for the queued steps; raise if one failed."""
        self.ctx.call("fortai_hip_qwen35_decoder_status", self.h)

    def plan(self):
        """The launches of one step: [(operation, kernel, batch)]."""
        return _plan(self.ctx, "fortai_hip_qwen35_decoder_plan", self.h)

    def free(self) -> None:
        if self.h:
            self.ctx.lib.fortai_hip_qwen35_decoder_destroy(self.h)
            self.h = None


class BatchDecoder:
    """``batch`` independent sequences over one set of layers and weights (one
    captured graph per step, every weight read once for all sequences)."""

    def __init__(self, ctx: Context, batch: int, recurrent: Sequence[Optional[Recurrent]],
                 attention: Sequence[Optional[Attention]], ffn_gate: Sequence[Q8Weights],
                 ffn_up: Sequence[Q8Weights], ffn_down: Sequence[Q8Weights], attn_norm: Sequence[np.ndarray],
                 post_norm: Sequence[np.ndarray], output_norm: np.ndarray, hidden: int,
                 embedding, output, max_context: int, eps: float, vocab: int):
        self.ctx, self.batch, self.vocab, self.max_context = ctx, batch, vocab, max_context
        n = len(ffn_gate)

        def harr(items):
            return (C.c_void_p * n)(*[(x.h if x is not None else None) for x in items])

        self._norms = [np.ascontiguousarray(a, dtype=np.float32) for a in list(attn_norm) + list(post_norm)]
        an = (C.c_void_p * n)(*[_ptr(a) for a in self._norms[:n]])
        pn = (C.c_void_p * n)(*[_ptr(a) for a in self._norms[n:]])
        self._onorm = np.ascontiguousarray(output_norm, dtype=np.float32)
        e16 = embedding.h if isinstance(embedding, F16Weights) else None
        e8 = embedding.h if isinstance(embedding, Q8Weights) else None
        o16 = output.h if isinstance(output, F16Weights) else None
        o8 = output.h if isinstance(output, Q8Weights) else None
        h = C.c_void_p()
        ctx.call("fortai_hip_qwen35_batch_create", ctx.h, batch, n, harr(recurrent), harr(attention),
                 harr(ffn_gate), harr(ffn_up), harr(ffn_down), an, pn, _ptr(self._onorm), hidden, e16, e8, o16, o8,
                 max_context, eps, C.byref(h))
        self.h = h
        self.logits = np.zeros((batch, vocab), dtype=np.float32)

    def _inputs(self, tokens, positions):
        t = np.ascontiguousarray(tokens, dtype=np.int64)
        p = np.ascontiguousarray(positions, dtype=np.int32)
        if t.shape != (self.batch,) or p.shape != (self.batch,):
            raise ValueError(f"need {self.batch} tokens and positions")
        return t, p

    def reset(self) -> None:
        self.ctx.call("fortai_hip_qwen35_batch_reset", self.h)

    def set_mode(self, direct: bool = False) -> None:
        self.ctx.call("fortai_hip_qwen35_batch_set_mode", self.h, DECODER_DIRECT if direct else 0)

    def set_prefill_mode(self, mode: str) -> None:
        """'exact' (default), 'matvec' (same bits) or 'fast' (not bit-exact)."""
        self.ctx.call("fortai_hip_qwen35_batch_set_prefill_mode", self.h, PREFILL_MODES[mode])

    def forward(self, tokens, positions, want_logits: bool = True) -> np.ndarray:
        t, p = self._inputs(tokens, positions)
        nxt = np.zeros(self.batch, dtype=np.int64)
        self.ctx.call("fortai_hip_qwen35_batch_forward", self.h, _ptr(t), _ptr(p),
                      _ptr(self.logits) if want_logits else None, _ptr(nxt))
        return nxt

    def generate(self, tokens, positions, steps: int) -> np.ndarray:
        t, p = self._inputs(tokens, positions)
        trace = np.zeros((self.batch, steps), dtype=np.int64)
        self.ctx.call("fortai_hip_qwen35_batch_generate", self.h, _ptr(t), _ptr(p), steps, _ptr(trace))
        return trace

    def replay(self, steps: int) -> None:
        self.ctx.call("fortai_hip_qwen35_batch_replay", self.h, steps)

    def plan(self, prefill: bool = False):
        """The launches of one batched step (or of the last prefill)."""
        return _plan(self.ctx, "fortai_hip_qwen35_batch_plan", self.h, 1 if prefill else 0)

    def prefill(self, tokens, want_logits: bool = True):
        """Prompt tokens [batch][T] from position 0; returns (next tokens,
        prefill milliseconds); logits of the last prompt token in .logits."""
        t = np.ascontiguousarray(tokens, dtype=np.int64)
        if t.ndim != 2 or t.shape[0] != self.batch:
            raise ValueError(f"need tokens [{self.batch}][T]")
        nxt = np.zeros(self.batch, dtype=np.int64)
        ms = C.c_float()
        self.ctx.call("fortai_hip_qwen35_batch_prefill", self.h, _ptr(t), t.shape[1], _ptr(nxt),
                      _ptr(self.logits) if want_logits else None, C.byref(ms))
        return nxt, ms.value

    def free(self) -> None:
        if self.h:
            self.ctx.lib.fortai_hip_qwen35_batch_destroy(self.h)
            self.h = None


def _dev(x):
    """A device address: None, an integer (a tensor's data_ptr()), a c_void_p or a DeviceBuffer."""
    return x.h if isinstance(x, DeviceBuffer) else x


class Rope:
    """Rotary positions of query and key heads, with an optional per-head RMSNorm
    in front.  ``scaling``: 'none', 'linear' (factor) or 'yarn' (factor,
    original_context, beta_fast, beta_slow)."""

    def __init__(self, ctx: Context, rope_dim: int, interleaved: bool = False, base: float = 1.0e4,
                 scaling: str = "none", factor: float = 1.0, original_context: int = 0, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, attention_factor: float = 1.0):
        self.ctx, self.rope_dim = ctx, rope_dim
        h = C.c_void_p()
        ctx.call("fortai_hip_rope_create", ctx.h, rope_dim, 1 if interleaved else 0, base, ROPE_SCALINGS[scaling],
                 factor, original_context, beta_fast, beta_slow, attention_factor, C.byref(h))
        self.h = h

    def apply(self, x, positions, rows: int, heads: int, head_size: int, out, dtype: str = "f32",
              row_pitch: Optional[int] = None, head_pitch: Optional[int] = None, out_row_pitch: Optional[int] = None,
              out_head_pitch: Optional[int] = None, norm=None, eps: float = 1e-6) -> None:
        """x [rows][heads][head_size] (dense unless pitches are given) at
        positions[rows] (int32) -> out; out may be x itself."""
        hp = head_size if head_pitch is None else head_pitch
        rp = heads * hp if row_pitch is None else row_pitch
        ohp = head_size if out_head_pitch is None else out_head_pitch
        orp = heads * ohp if out_row_pitch is None else out_row_pitch
        self.ctx.check(self.ctx.lib.fortai_hip_rope_device(self.h, DTYPES[dtype], _dev(x), rp, hp, rows, heads,
                                                           head_size, _dev(positions), _dev(norm), eps, _dev(out),
                                                           orp, ohp), "fortai_hip_rope_device")

    def free(self) -> None:
        if self.h:
            self.ctx.lib.fortai_hip_rope_destroy(self.h)
            self.h = None


class Kv8Batch(C.Structure):
    """Which rows of a call belong to which sequence of an 8-bit cache, and where
    its tokens lie (fortai_hip_kv8_batch): device int32 row_starts [sequences + 1],
    lengths [sequences] (tokens before the rows) and tables [sequences][table_pitch]."""

    _fields_ = [("sequences", _i), ("rows", _i), ("max_rows", _i), ("table_pitch", _i), ("row_starts", _vp),
                ("lengths", _vp), ("tables", _vp)]

    def __init__(self, sequences: int, rows: int, max_rows: int, row_starts, lengths, tables, table_pitch: int):
        super().__init__(sequences, rows, max_rows, table_pitch, _dev(row_starts), _dev(lengths), _dev(tables))


class Kv8Groups(C.Structure):
    """Which sequences of a batch share their first tokens' pages (fortai_hip_kv8_groups): device int32 starts
    [groups + 1], shared [groups] tokens and group_of [sequences]; max_rows: the most rows of a group."""

    _fields_ = [("groups", _i), ("max_rows", _i), ("starts", _vp), ("shared", _vp), ("group_of", _vp)]

    def __init__(self, groups: int, max_rows: int, starts, shared, group_of):
        super().__init__(groups, max_rows, _dev(starts), _dev(shared), _dev(group_of))


class Kv8Cache:
    """8-bit paged key/value cache (fortai_hip_kv8_cache), over the caller's
    device storage of Kv8Cache.bytes() bytes or over its own."""

    def __init__(self, ctx: Context, layers: int, pages: int, page_tokens: int, kv_heads: int, head_size: int,
                 storage=None, storage_bytes: int = 0):
        self.ctx = ctx
        self.layers, self.pages, self.page_tokens = layers, pages, page_tokens
        self.kv_heads, self.head_size = kv_heads, head_size
        h = C.c_void_p()
        ctx.call("fortai_hip_kv8_create", ctx.h, layers, pages, page_tokens, kv_heads, head_size, _dev(storage),
                 storage_bytes, C.byref(h))
        self.h = h

    @staticmethod
    def bytes(layers: int, pages: int, page_tokens: int, kv_heads: int, head_size: int) -> int:
        """Bytes of the storage (0: no such cache)."""
        return load().fortai_hip_kv8_bytes(layers, pages, page_tokens, kv_heads, head_size)

    def append(self, layer: int, batch: Kv8Batch, keys, values, dtype: str = "f32", key_pitch: Optional[int] = None,
               value_pitch: Optional[int] = None) -> None:
        """Store rows of keys and values [rows][kv_heads][head_size] (dense unless pitches are given)."""
        width = self.kv_heads * self.head_size
        self.ctx.check(self.ctx.lib.fortai_hip_kv8_append_device(
            self.h, layer, C.addressof(batch), DTYPES[dtype], _dev(keys), width if key_pitch is None else key_pitch,
            _dev(values), width if value_pitch is None else value_pitch), "fortai_hip_kv8_append_device")

    def read(self, layer: int, batch: Kv8Batch, keys, values, dtype: str = "f32", key_pitch: Optional[int] = None,
             value_pitch: Optional[int] = None) -> None:
        """The batch's rows as the values that their codes stand for."""
        width = self.kv_heads * self.head_size
        self.ctx.check(self.ctx.lib.fortai_hip_kv8_read_device(
            self.h, layer, C.addressof(batch), DTYPES[dtype], _dev(keys), width if key_pitch is None else key_pitch,
            _dev(values), width if value_pitch is None else value_pitch), "fortai_hip_kv8_read_device")

    def attention(self, layer: int, batch: Kv8Batch, query, heads: int, out, scale: float, max_length: int,
                  dtype: str = "f32", gate=None, query_pitch: Optional[int] = None,
                  query_head_pitch: Optional[int] = None, out_pitch: Optional[int] = None) -> None:
        """Attention of the batch's rows: query [rows][heads][head_size] (dense unless pitches are given; gate,
        where given, at the same pitches) -> out [rows][heads][head_size].  max_length: about the longest
        sequence with its rows, for cutting the work."""
        hp = self.head_size if query_head_pitch is None else query_head_pitch
        self.ctx.check(self.ctx.lib.fortai_hip_kv8_attention_device(
            self.h, layer, C.addressof(batch), DTYPES[dtype], _dev(query), heads * hp if query_pitch is None else query_pitch,
            hp, _dev(gate), heads, scale, max_length, _dev(out), heads * self.head_size if out_pitch is None else out_pitch),
            "fortai_hip_kv8_attention_device")

    def shared_attention(self, layer: int, batch: Kv8Batch, sharing: Kv8Groups, query, heads: int, out, scale: float,
                         max_length: int, max_shared: int, dtype: str = "f32", gate=None, query_pitch: Optional[int] = None,
                         query_head_pitch: Optional[int] = None, out_pitch: Optional[int] = None) -> None:
        """attention() with the tokens that groups of sequences share read once for all their rows; max_shared: about
        the most of them."""
        hp = self.head_size if query_head_pitch is None else query_head_pitch
        self.ctx.check(self.ctx.lib.fortai_hip_kv8_shared_attention_device(
            self.h, layer, C.addressof(batch), C.addressof(sharing), DTYPES[dtype], _dev(query),
            heads * hp if query_pitch is None else query_pitch, hp, _dev(gate), heads, scale, max_length, max_shared, _dev(out),
            heads * self.head_size if out_pitch is None else out_pitch), "fortai_hip_kv8_shared_attention_device")

    def copy_pages(self, source, target) -> None:
        """Page target[i] becomes a copy of page source[i], in every layer (host int32 arrays)."""
        f = np.ascontiguousarray(source, dtype=np.int32)
        t = np.ascontiguousarray(target, dtype=np.int32)
        if f.shape != t.shape or f.ndim != 1:
            raise ValueError("need as many source as target pages")
        self.ctx.check(self.ctx.lib.fortai_hip_kv8_copy_pages(self.h, f.ctypes.data, t.ctypes.data, len(f)),
                       "fortai_hip_kv8_copy_pages")

    def free(self) -> None:
        if self.h:
            self.ctx.lib.fortai_hip_kv8_destroy(self.h)
            self.h = None


class Kv8Pages:
    """Page bookkeeping of a pool (fortai_hip_kv8_pages): host only, no GPU."""

    def __init__(self, pages: int, page_tokens: int, sequences: int, table_pitch: int):
        self.lib, self.pages, self.table_pitch = load(), pages, table_pitch
        h = C.c_void_p()
        self._check(self.lib.fortai_hip_kv8_pages_create(pages, page_tokens, sequences, table_pitch, C.byref(h)),
                    "fortai_hip_kv8_pages_create")
        self.h = h

    @staticmethod
    def _check(rc: int, what: str) -> None:
        if rc != OK:
            raise BackendError(rc, what)

    def extend(self, sequence: int, tokens: int):
        """Room for more tokens; the (from, to) page pairs that have to be copied first (none or one)."""
        f, t, n = C.c_int32(), C.c_int32(), C.c_int()
        self._check(self.lib.fortai_hip_kv8_pages_extend(self.h, sequence, tokens, C.byref(f), C.byref(t), C.byref(n)),
                    "fortai_hip_kv8_pages_extend")
        return [(f.value, t.value)] if n.value else []

    def fork(self, sequence: int, fork: int, length: int) -> None:
        self._check(self.lib.fortai_hip_kv8_pages_fork(self.h, sequence, fork, length), "fortai_hip_kv8_pages_fork")

    def truncate(self, sequence: int, length: int = 0) -> None:
        self._check(self.lib.fortai_hip_kv8_pages_truncate(self.h, sequence, length), "fortai_hip_kv8_pages_truncate")

    def compact(self, capacity: Optional[int] = None):
        """Move live pages to the pool's lower end; the moves as (from, to) arrays."""
        n = C.c_int()
        capacity = self.pages if capacity is None else capacity
        f, t = np.empty(max(capacity, 1), dtype=np.int32), np.empty(max(capacity, 1), dtype=np.int32)
        self._check(self.lib.fortai_hip_kv8_pages_compact(self.h, _ptr(f), _ptr(t), capacity, C.byref(n)),
                    "fortai_hip_kv8_pages_compact")
        return f[:n.value].copy(), t[:n.value].copy()

    def length(self, sequence: int) -> int:
        return self.lib.fortai_hip_kv8_pages_length(self.h, sequence)

    def free_count(self) -> int:
        return self.lib.fortai_hip_kv8_pages_free_count(self.h)

    def tables(self, sequences) -> np.ndarray:
        """The pages of these sequences, int32 [len(sequences)][table_pitch], -1 behind the last."""
        s = np.ascontiguousarray(sequences, dtype=np.int32)
        out = np.empty((len(s), self.table_pitch), dtype=np.int32)
        self._check(self.lib.fortai_hip_kv8_pages_tables(self.h, _ptr(s), len(s), _ptr(out), self.table_pitch),
                    "fortai_hip_kv8_pages_tables")
        return out

    def groups(self, sequences):
        """Which of these sequences share leading pages with the ones before them: int32 arrays starts [groups + 1],
        shared [groups] and group_of [len(sequences)], for Kv8Groups."""
        s = np.ascontiguousarray(sequences, dtype=np.int32)
        starts, shared, group_of = (np.zeros(len(s) + 1, dtype=np.int32) for _ in range(3))
        n = C.c_int()
        self._check(self.lib.fortai_hip_kv8_pages_groups(self.h, _ptr(s), len(s), _ptr(starts), _ptr(shared), _ptr(group_of),
                                                         C.byref(n)), "fortai_hip_kv8_pages_groups")
        return starts[:n.value + 1].copy(), shared[:n.value].copy(), group_of[:len(s)].copy()

    def free(self) -> None:
        if self.h:
            self.lib.fortai_hip_kv8_pages_destroy(self.h)
            self.h = None


class Verifier:
    """Verification of drafted tokens against the target's logits
    (fortai_hip_verify_drafts_device), for up to max_rows rows of max_sequences
    sequences and one vocabulary."""

    def __init__(self, ctx: Context, max_rows: int, max_sequences: int, vocab: int):
        self.ctx, self.vocab = ctx, vocab
        h = C.c_void_p()
        ctx.call("fortai_hip_verifier_create", ctx.h, max_rows, max_sequences, vocab, C.byref(h))
        self.h = h

    def run(self, target_logits, tokens, uniforms, row_starts, sequences: int, rows: int, emitted, accepted,
            dtype: str = "f32", draft_logits=None, temperatures=None, logprobs=None,
            target_pitch: Optional[int] = None, draft_pitch: Optional[int] = None) -> None:
        """Device arrays: target_logits and draft_logits [rows][vocab] (dense unless pitches are given), tokens int64
        [rows], uniforms fp32 [rows], row_starts int32 [sequences + 1], temperatures fp32 [sequences] -> emitted int64
        [rows], accepted int32 [sequences], logprobs fp32 [rows]."""
        self.ctx.check(self.ctx.lib.fortai_hip_verify_drafts_device(
            self.h, DTYPES[dtype], _dev(target_logits), self.vocab if target_pitch is None else target_pitch,
            _dev(draft_logits), self.vocab if draft_pitch is None else draft_pitch, _dev(tokens), _dev(uniforms),
            _dev(temperatures), sequences, _dev(row_starts), rows, _dev(emitted), _dev(accepted), _dev(logprobs)),
            "fortai_hip_verify_drafts_device")

    def free(self) -> None:
        if self.h:
            self.ctx.lib.fortai_hip_verifier_destroy(self.h)
            self.h = None


class GdnBatch(C.Structure):
    """Which rows of a call belong to which sequence, and where its state is (fortai_hip_gdn_batch): device int32
    row_starts [sequences + 1], slots [sequences] and standing [sequences] (None: every pending row stands)."""

    _fields_ = [("sequences", _i), ("rows", _i), ("max_rows", _i), ("row_starts", _vp), ("slots", _vp), ("standing", _vp)]

    def __init__(self, sequences: int, rows: int, max_rows: int, row_starts, slots, standing=None):
        super().__init__(sequences, rows, max_rows, _dev(row_starts), _dev(slots), _dev(standing))


class GdnCache:
    """States of the gated delta rule (fortai_hip_gdn_cache), over the caller's device storage of GdnCache.bytes()
    bytes or over its own, for calls of up to max_rows rows."""

    def __init__(self, ctx: Context, layers: int, slots: int, key_heads: int, value_heads: int, head_size: int,
                 conv_kernel: int, pending: int, max_rows: int, storage=None, storage_bytes: int = 0):
        self.ctx, self.slots = ctx, slots
        self.channels, self.value_heads, self.width = (2 * key_heads + value_heads) * head_size, value_heads, value_heads * head_size
        h = C.c_void_p()
        ctx.call("fortai_hip_gdn_create", ctx.h, layers, slots, key_heads, value_heads, head_size, conv_kernel, pending, max_rows,
                 _dev(storage), storage_bytes, C.byref(h))
        self.h = h

    @staticmethod
    def bytes(layers: int, slots: int, key_heads: int, value_heads: int, head_size: int, conv_kernel: int, pending: int) -> int:
        """Bytes of the storage (0: no such cache)."""
        return load().fortai_hip_gdn_bytes(layers, slots, key_heads, value_heads, head_size, conv_kernel, pending)

    def run(self, layer: int, batch: GdnBatch, qkv, alpha, beta, conv, ssm_a, ssm_dt, out, dtype: str = "f32",
            eps: float = 1e-6, qkv_pitch: Optional[int] = None, alpha_pitch: Optional[int] = None,
            beta_pitch: Optional[int] = None, out_pitch: Optional[int] = None) -> None:
        """The batch's rows: qkv [rows][channels], alpha and beta [rows][value_heads] (dense unless pitches are given),
        fp32 conv [channels][conv_kernel], ssm_a and ssm_dt [value_heads] -> out [rows][value_heads][head_size]."""
        self.ctx.check(self.ctx.lib.fortai_hip_gdn_run_device(
            self.h, layer, C.addressof(batch), DTYPES[dtype], _dev(qkv), self.channels if qkv_pitch is None else qkv_pitch,
            _dev(alpha), self.value_heads if alpha_pitch is None else alpha_pitch, _dev(beta),
            self.value_heads if beta_pitch is None else beta_pitch, _dev(conv), _dev(ssm_a), _dev(ssm_dt), eps, _dev(out),
            self.width if out_pitch is None else out_pitch), "fortai_hip_gdn_run_device")

    def copy_slots(self, source, target) -> None:
        """Slot target[i] becomes a copy of slot source[i], in every layer (host int32 arrays)."""
        f = np.ascontiguousarray(source, dtype=np.int32)
        t = np.ascontiguousarray(target, dtype=np.int32)
        if f.shape != t.shape or f.ndim != 1:
            raise ValueError("need as many source as target slots")
        self.ctx.check(self.ctx.lib.fortai_hip_gdn_copy_slots(self.h, f.ctypes.data, t.ctypes.data, len(f)),
                       "fortai_hip_gdn_copy_slots")

    def free(self) -> None:
        if self.h:
            self.ctx.lib.fortai_hip_gdn_destroy(self.h)
            self.h = None
