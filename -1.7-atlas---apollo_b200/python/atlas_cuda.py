"""ctypes binding of libatlas_cuda's C ABI (include/atlas_cuda.h, include/atlas_runtime.h,
include/gpu_matvec.h, include/atlas_synth.h).

The library is the in-tree ``libatlas_cuda.so`` next to this package's ``csrc/``.
Loading fails loudly when it is missing: there is no Python or CPU fallback.
"""
from __future__ import annotations

import ctypes
import os
import sys
from itertools import accumulate
from operator import mul

PKG_DIR = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB_PATH = os.path.join(PKG_DIR, "libatlas_cuda.so")

ATLAS_OK = 0
ERRORS = {
    -1: "EINVAL", -2: "ENODEV", -3: "ENOMEM", -4: "ECUDA", -5: "ETIMEOUT", -6: "ENCCL", -7: "ERANGE",
}
TYPE_F32, TYPE_F16, TYPE_Q5_0, TYPE_Q5_1, TYPE_Q8_0, TYPE_Q4_K, TYPE_Q5_K, TYPE_Q6_K = 0, 1, 6, 7, 8, 12, 13, 14
BLOCK_BYTES = {TYPE_F16: 2, TYPE_Q5_0: 22, TYPE_Q5_1: 24, TYPE_Q8_0: 34, TYPE_Q4_K: 144, TYPE_Q5_K: 176,
               TYPE_Q6_K: 210}
BLOCK_ELEMS = {TYPE_F16: 1, TYPE_Q5_0: 32, TYPE_Q5_1: 32, TYPE_Q8_0: 32, TYPE_Q4_K: 256, TYPE_Q5_K: 256,
               TYPE_Q6_K: 256}

# Every symbol the public headers declare (checked by the CPU test suite).
EXPORTS = [
    "atlas_cuda_create", "atlas_cuda_destroy", "atlas_cuda_last_error", "atlas_cuda_prefill",
    "atlas_cuda_decode", "atlas_cuda_generate", "atlas_cuda_stats", "atlas_cuda_dequant",
    "atlas_cuda_gemv", "atlas_cuda_gemm", "atlas_cuda_device_info", "atlas_cuda_trace_step",
    "atlas_cuda_device_ms", "atlas_cuda_trace_graph", "atlas_cuda_gemv_noalloc", "atlas_cuda_tp_slice", "atlas_cuda_tp_handle",
    "atlas_cuda_tp_connect", "atlas_cuda_prefill_seq", "atlas_cuda_generate_batch", "atlas_cuda_decode_batch",
    "atlas_cuda_kv8_append", "atlas_cuda_kv8_read", "atlas_cuda_kv8_attn", "atlas_cuda_kv8_attn_sparse",
    "atlas_cuda_kv8_attn_form",
    "atlas_cuda_paged_work", "atlas_cuda_paged_fork", "atlas_cuda_paged_reserve", "atlas_cuda_paged_compact",
    "atlas_cuda_paged_append", "atlas_cuda_paged_attn", "atlas_cuda_paged_attn_form",
    "brain_gpu_init", "brain_gpu_matvec_batch", "brain_gpu_matvec", "brain_gpu_shutdown",
    "atlas_rt_open", "atlas_rt_close", "atlas_rt_error", "atlas_rt_shape", "atlas_rt_data_base",
    "atlas_rt_find_tensor", "atlas_rt_file_bytes", "atlas_rt_device", "atlas_rt_forward_token",
    "atlas_rt_prefill", "atlas_rt_generate",
    "atlas_synth_write_gguf", "atlas_synth_q4k_blocks", "atlas_synth_q6k_blocks", "atlas_synth_file_size",
]


class AtlasError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"{ERRORS.get(code, code)}: {msg}")
        self.code = code


class SynthConfig(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in
                ("hidden", "layers", "q_heads", "kv_heads", "head_dim", "ffn", "vocab", "context_length")] + [
        ("rope_base", ctypes.c_float), ("tied", ctypes.c_int32), ("qkv_bias", ctypes.c_int32),
        ("threads", ctypes.c_int32), ("seed", ctypes.c_uint64), ("qk_norm", ctypes.c_int32),
        ("alt_type", ctypes.c_int32), ("layer_mix", ctypes.c_int32)]


class Shape(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in
                ("hidden_size", "q_dim", "kv_dim", "q_heads", "kv_heads", "head_dim", "ffn_size", "layers",
                 "max_context", "vocab_size")] + [
        ("rope_base", ctypes.c_float), ("has_qk_norm", ctypes.c_int32), ("architecture", ctypes.c_char * 64)]


class TensorInfo(ctypes.Structure):
    _fields_ = [("name", ctypes.c_char * 256), ("n_dims", ctypes.c_uint32), ("dims", ctypes.c_uint64 * 4),
                ("type", ctypes.c_uint32), ("offset", ctypes.c_uint64)]


class RtOptions(ctypes.Structure):
    _fields_ = [("device", ctypes.c_int32), ("max_context", ctypes.c_uint32), ("max_prefill", ctypes.c_uint32),
                ("kv_fp16", ctypes.c_int32), ("no_device", ctypes.c_int32), ("tp_rank", ctypes.c_int32),
                ("tp_size", ctypes.c_int32), ("max_batch", ctypes.c_uint32)]


class ModelDesc(ctypes.Structure):
    """AtlasModelDesc (include/atlas_cuda.h)."""
    _fields_ = [(n, ctypes.c_uint32) for n in
                ("hidden", "q_dim", "kv_dim", "q_heads", "kv_heads", "head_dim", "ffn", "layers", "vocab",
                 "max_context", "max_prefill")] + [
        ("rope_base", ctypes.c_float), ("rms_eps", ctypes.c_float)] + [
        (n, ctypes.c_int32) for n in ("has_qk_norm", "kv_fp16", "device", "tp_rank", "tp_size")] + [
        ("max_batch", ctypes.c_uint32)]


class TpSlice(ctypes.Structure):
    """AtlasTpSlice: one tensor-parallel rank's share of the model."""
    _fields_ = [(n, ctypes.c_uint32) for n in
                ("q_head0", "q_heads", "kv_head0", "kv_heads", "o_block0", "o_blocks", "o_lo", "o_hi",
                 "ffn_row0", "ffn_rows", "vocab_row0", "vocab_rows")]

    def as_dict(self):
        return {n: getattr(self, n) for n, _ in self._fields_}


class Kv8Desc(ctypes.Structure):
    """AtlasKv8 (include/atlas_cuda.h)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale", "k_sum")] + [
        (n, ctypes.c_uint32) for n in ("nseq", "kv_heads", "max_context", "block")]


class PagedDesc(ctypes.Structure):
    """AtlasPaged (include/atlas_cuda.h)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "table", "refs", "work")] + [("work_bytes", ctypes.c_uint64)] + [
        (n, ctypes.c_uint32) for n in ("type", "layers", "pages", "kv_heads", "page", "nseq", "max_pages")]


TP_HANDLE_BYTES = 64


class BrainGpuMatvec(ctypes.Structure):
    _fields_ = [("offset", ctypes.c_uint64), ("rows", ctypes.c_uint64), ("cols", ctypes.c_uint64),
                ("type", ctypes.c_uint32), ("input", ctypes.c_void_p), ("output", ctypes.c_void_p)]


_LIB = None


def lib() -> ctypes.CDLL:
    """Load the in-tree library (raises if it was not built)."""
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise FileNotFoundError(f"{LIB_PATH} is missing: build it with __graft_entry__.build()")
        L = ctypes.CDLL(LIB_PATH, mode=ctypes.RTLD_GLOBAL)
        P, U32, U64, I32 = ctypes.c_void_p, ctypes.c_uint32, ctypes.c_uint64, ctypes.c_int
        L.atlas_cuda_last_error.restype = ctypes.c_char_p
        L.atlas_cuda_last_error.argtypes = [P]
        L.atlas_cuda_dequant.argtypes = [U32, P, U64, P, P]
        L.atlas_cuda_gemv.argtypes = [U32, P, U64, U64, P, P, P]
        L.atlas_cuda_gemv_noalloc.argtypes = [U32, P, U64, U64, P, P, P]
        L.atlas_cuda_gemm.argtypes = [U32, P, U64, U64, P, U64, P, P]
        L.atlas_cuda_device_info.argtypes = [I32, P, P, P]
        L.atlas_cuda_decode.argtypes = [P, U32, U32, P, P]
        L.atlas_cuda_prefill.argtypes = [P, P, U32, U32, P, P]
        L.atlas_cuda_generate.argtypes = [P, U32, U32, U32, P]
        L.atlas_cuda_stats.argtypes = [P, P, P]
        L.atlas_cuda_device_ms.argtypes = [P, P]
        L.atlas_cuda_trace_step.argtypes = [P, U32, U32, P, ctypes.c_size_t, P, P, P]
        L.atlas_cuda_trace_graph.argtypes = [P, U32, U32, P, ctypes.c_size_t, P, P, P]
        L.atlas_cuda_tp_slice.argtypes = [P, I32, I32, P]
        L.atlas_cuda_tp_handle.argtypes = [P, P]
        L.atlas_cuda_tp_connect.argtypes = [P, P]
        L.atlas_rt_open.argtypes = [ctypes.c_char_p, P, P]
        L.atlas_rt_close.argtypes = [P]
        L.atlas_rt_error.restype = ctypes.c_char_p
        L.atlas_rt_error.argtypes = [P]
        L.atlas_rt_shape.argtypes = [P, P]
        L.atlas_rt_data_base.restype = U64
        L.atlas_rt_data_base.argtypes = [P]
        L.atlas_rt_find_tensor.argtypes = [P, ctypes.c_char_p, P]
        L.atlas_rt_file_bytes.restype = P
        L.atlas_rt_file_bytes.argtypes = [P, P]
        L.atlas_rt_device.restype = P
        L.atlas_rt_device.argtypes = [P]
        L.atlas_rt_forward_token.argtypes = [P, U32, U32, P, P]
        L.atlas_rt_prefill.argtypes = [P, P, U32, U32, P, P]
        L.atlas_rt_generate.argtypes = [P, U32, U32, U32, P]
        L.atlas_cuda_prefill_seq.argtypes = [P, U32, P, U32, U32, P, P]
        L.atlas_cuda_generate_batch.argtypes = [P, U32, P, P, U32, P]
        L.atlas_cuda_decode_batch.argtypes = [P, U32, P, P, P, P]
        L.atlas_cuda_kv8_append.argtypes = [P, U32, P, P, P, P, U64, P]
        L.atlas_cuda_kv8_read.argtypes = [P, U32, P, P, P, P, U64, P]
        L.atlas_cuda_kv8_attn.argtypes = [P, U32, U32, P, P, P, U64, P, U64, P]
        L.atlas_cuda_kv8_attn_form.argtypes = [P, U32, U32, P, P]
        L.atlas_cuda_kv8_attn_sparse.argtypes = [P, U32, U32, U32, P, P, P, U64, P, U64, P, P]
        L.atlas_cuda_paged_work.argtypes = [P, P]
        L.atlas_cuda_paged_fork.argtypes = [P, P, P, P, P]
        L.atlas_cuda_paged_reserve.argtypes = [P, U32, P, P, P, P]
        L.atlas_cuda_paged_compact.argtypes = [P, P, P]
        L.atlas_cuda_paged_append.argtypes = [P, U32, U32, P, P, P, P, U64, P]
        L.atlas_cuda_paged_attn_form.argtypes = [P, U32, U32, P]
        L.atlas_cuda_paged_attn.argtypes = [P, U32, U32, U32, P, P, P, U64, P, U64, P]
        L.atlas_synth_write_gguf.argtypes = [P, ctypes.c_char_p]
        L.atlas_synth_q4k_blocks.argtypes = [U64, U64, P, U64]
        L.atlas_synth_q6k_blocks.argtypes = [U64, U64, P, U64]
        L.atlas_synth_file_size.restype = U64
        L.atlas_synth_file_size.argtypes = [P]
        L.brain_gpu_init.argtypes = [P, ctypes.c_size_t]
        L.brain_gpu_matvec_batch.argtypes = [P, ctypes.c_size_t]
        L.brain_gpu_matvec.argtypes = [U64, U32, U64, U64, P, P]
        _LIB = L
    return _LIB


def check(rc: int, where: str = "", handle=None) -> None:
    if rc != ATLAS_OK:
        msg = lib().atlas_cuda_last_error(handle)
        raise AtlasError(rc, f"{where}: {msg.decode() if msg else ''}")


def _ptr(a) -> ctypes.c_void_p:
    """Host numpy array or device torch tensor -> void*."""
    if a is None:
        return ctypes.c_void_p(0)
    if hasattr(a, "data_ptr"):
        return ctypes.c_void_p(a.data_ptr())
    return a.ctypes.data_as(ctypes.c_void_p)


def write_synthetic_gguf(path: str, *, hidden: int, layers: int, q_heads: int, kv_heads: int, ffn: int, vocab: int,
                         head_dim: int = 128, context_length: int = 32768, rope_base: float = 1e6,
                         tied: bool = True, qkv_bias: bool = True, seed: int = 0, threads: int = 0,
                         qk_norm: bool = False, alt_type: int = 0, layer_mix: bool = False) -> int:
    """qk_norm: a qwen3 file (per-head q/k RMSNorm weights). alt_type: another
    block type (F16, Q5_0, Q5_1, Q8_0, Q5_K) for attn_q, ffn_gate, ffn_up,
    ffn_down and the head. layer_mix: odd layers' attn_v and ffn_down are Q4_K."""
    cfg = SynthConfig(hidden, layers, q_heads, kv_heads, head_dim, ffn, vocab, context_length, rope_base,
                      int(tied), int(qkv_bias), threads, seed, int(qk_norm), int(alt_type), int(layer_mix))
    rc = lib().atlas_synth_write_gguf(ctypes.byref(cfg), path.encode())
    if rc != 0:
        raise RuntimeError(f"synthetic GGUF write failed: {path}")
    return lib().atlas_synth_file_size(ctypes.byref(cfg))


def synth_blocks(type_id: int, n: int, seed: int = 0, stream: int = 0):
    import numpy as np
    out = np.zeros(n * BLOCK_BYTES[type_id], np.uint8)
    fn = lib().atlas_synth_q4k_blocks if type_id == TYPE_Q4_K else lib().atlas_synth_q6k_blocks
    fn(seed, stream, _ptr(out), n)
    return out


class Runtime:
    """Reference-shaped model API: open a GGUF, forward tokens, prefill, generate."""

    def __init__(self, path: str, *, device: int = 0, max_context: int = 0, max_prefill: int = 0,
                 kv_fp16: bool = False, no_device: bool = False, tp_rank: int = 0, tp_size: int = 1,
                 max_batch: int = 1):
        self._h = ctypes.c_void_p()
        opt = RtOptions(device, max_context, max_prefill, int(kv_fp16), int(no_device), tp_rank, tp_size, max_batch)
        self.tp_rank, self.tp_size = tp_rank, tp_size
        rc = lib().atlas_rt_open(path.encode(), ctypes.byref(opt), ctypes.byref(self._h))
        if rc != ATLAS_OK:
            msg = lib().atlas_rt_error(self._h).decode()
            lib().atlas_rt_close(self._h)
            self._h = None
            raise AtlasError(rc, f"atlas_rt_open({path}): {msg}")
        s = Shape()
        lib().atlas_rt_shape(self._h, ctypes.byref(s))
        self.shape = s
        self.vocab = s.vocab_size

    def _check(self, rc: int, where: str) -> None:
        if rc != ATLAS_OK:
            raise AtlasError(rc, f"{where}: {lib().atlas_rt_error(self._h).decode()}")

    def tensor(self, name: str) -> TensorInfo | None:
        t = TensorInfo()
        return t if lib().atlas_rt_find_tensor(self._h, name.encode(), ctypes.byref(t)) else None

    @property
    def data_base(self) -> int:
        return lib().atlas_rt_data_base(self._h)

    def forward(self, token: int, pos: int, want_logits: bool = True):
        import numpy as np
        logits = np.zeros(self.vocab, np.float32) if want_logits else None
        am = ctypes.c_uint32()
        self._check(lib().atlas_rt_forward_token(self._h, token, pos, _ptr(logits), ctypes.byref(am)), "forward")
        return logits, am.value

    def prefill(self, ids, pos0: int = 0, want_logits: bool = True):
        import numpy as np
        ids = np.ascontiguousarray(ids, dtype=np.uint32)
        logits = np.zeros(self.vocab, np.float32) if want_logits else None
        am = ctypes.c_uint32()
        self._check(lib().atlas_rt_prefill(self._h, _ptr(ids), len(ids), pos0, _ptr(logits), ctypes.byref(am)),
                    "prefill")
        return logits, am.value

    def generate(self, first: int, pos0: int, steps: int):
        import numpy as np
        out = np.zeros(steps, np.uint32)
        self._check(lib().atlas_rt_generate(self._h, first, pos0, steps, _ptr(out)), "generate")
        return out

    def prefill_seq(self, seq: int, ids, pos0: int = 0, want_logits: bool = True):
        """atlas_cuda_prefill into sequence seq's KV cache (open with max_batch > seq)."""
        import numpy as np
        ids = np.ascontiguousarray(ids, dtype=np.uint32)
        logits = np.zeros(self.vocab, np.float32) if want_logits else None
        am = ctypes.c_uint32()
        dev = lib().atlas_rt_device(self._h)
        check(lib().atlas_cuda_prefill_seq(dev, seq, _ptr(ids), len(ids), pos0, _ptr(logits), ctypes.byref(am)),
              "prefill_seq", dev)
        return logits, am.value

    def generate_batch(self, first, pos0, steps: int):
        """Greedy steps of len(first) sequences at once: array [nseq, steps] of picks."""
        import numpy as np
        first = np.ascontiguousarray(first, dtype=np.uint32)
        pos0 = np.ascontiguousarray(pos0, dtype=np.uint32)
        out = np.zeros((len(first), steps), np.uint32)
        dev = lib().atlas_rt_device(self._h)
        check(lib().atlas_cuda_generate_batch(dev, len(first), _ptr(first), _ptr(pos0), steps, _ptr(out)),
              "generate_batch", dev)
        return out

    def decode_batch(self, ids, pos, want_logits: bool = True):
        """One step of len(ids) sequences: (logits [nseq, vocab] or None, picks [nseq])."""
        import numpy as np
        ids = np.ascontiguousarray(ids, dtype=np.uint32)
        pos = np.ascontiguousarray(pos, dtype=np.uint32)
        logits = np.zeros((len(ids), self.vocab), np.float32) if want_logits else None
        am = np.zeros(len(ids), np.uint32)
        dev = lib().atlas_rt_device(self._h)
        check(lib().atlas_cuda_decode_batch(dev, len(ids), _ptr(ids), _ptr(pos), _ptr(logits), _ptr(am)),
              "decode_batch", dev)
        return logits, am

    def trace_step(self, token: int, pos: int):
        """One traced decode step: (stamps[cta, phase, 4], inner stamps[cta, phase, 8], phase kind codes)."""
        import numpy as np
        dev = lib().atlas_rt_device(self._h)
        nc, nph = ctypes.c_uint32(), ctypes.c_uint32()
        lib().atlas_cuda_trace_step(dev, token, pos, None, 0, ctypes.byref(nc), ctypes.byref(nph), None)
        per = nc.value * nph.value
        buf = np.zeros(per * 12, np.uint64)
        kinds = np.zeros(nph.value, np.uint32)
        check(lib().atlas_cuda_trace_step(dev, token, pos, _ptr(buf), buf.size, ctypes.byref(nc), ctypes.byref(nph),
                                          _ptr(kinds)), "trace_step", dev)
        return buf[:per * 4].reshape(nc.value, nph.value, 4), buf[per * 4:].reshape(nc.value, nph.value, 8), kinds

    def trace_graph(self, token: int, pos: int):
        """One decode step of the graph engine with device timestamps:
        array [launch, cta, word] of globaltimer ns (0 = not recorded); word 0
        start, 1 inputs ready, 2 + w warp w done (atlas_cuda_trace_graph)."""
        import numpy as np
        dev = lib().atlas_rt_device(self._h)
        nl, nc, nw = ctypes.c_uint32(), ctypes.c_uint32(), ctypes.c_uint32()
        check(lib().atlas_cuda_trace_graph(dev, token, pos, None, 0, ctypes.byref(nl), ctypes.byref(nc),
                                           ctypes.byref(nw)), "trace_graph", dev)
        buf = np.zeros(nl.value * nc.value * nw.value, np.uint64)
        check(lib().atlas_cuda_trace_graph(dev, token, pos, _ptr(buf), buf.size, None, None, None), "trace_graph", dev)
        return buf.reshape(nl.value, nc.value, nw.value)

    def tp_slice(self) -> TpSlice:
        """This rank's share of the model (the whole model without tensor parallelism)."""
        s = self.shape
        return tp_slice(dict(hidden=s.hidden_size, q_heads=s.q_heads, kv_heads=s.kv_heads, ffn=s.ffn_size,
                             vocab=s.vocab_size), self.tp_rank, self.tp_size)

    def tp_handle(self) -> bytes:
        """The exchange area of this rank, to hand to every other rank."""
        buf = ctypes.create_string_buffer(TP_HANDLE_BYTES)
        dev = lib().atlas_rt_device(self._h)
        check(lib().atlas_cuda_tp_handle(dev, buf), "atlas_cuda_tp_handle", dev)
        return buf.raw

    def tp_connect(self, handles) -> None:
        """handles: every rank's tp_handle() in rank order; builds the decode step."""
        if len(handles) != self.tp_size or any(len(b) != TP_HANDLE_BYTES for b in handles):
            raise ValueError("tp_connect needs tp_size handles of TP_HANDLE_BYTES bytes")
        buf = ctypes.create_string_buffer(b"".join(handles), TP_HANDLE_BYTES * self.tp_size)
        dev = lib().atlas_rt_device(self._h)
        check(lib().atlas_cuda_tp_connect(dev, buf), "atlas_cuda_tp_connect", dev)

    def stats(self):
        """(kernel launches since creation, device ms of the last call, device ms of all calls)."""
        n = ctypes.c_uint64()
        ms = ctypes.c_double()
        tot = ctypes.c_double()
        dev = lib().atlas_rt_device(self._h)
        lib().atlas_cuda_stats(dev, ctypes.byref(n), ctypes.byref(ms))
        lib().atlas_cuda_device_ms(dev, ctypes.byref(tot))
        return n.value, ms.value, tot.value

    def close(self) -> None:
        if self._h:
            lib().atlas_rt_close(self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def tp_slice(shape: dict, rank: int, size: int) -> TpSlice:
    """atlas_cuda_tp_slice for a shape given as hidden / q_heads / kv_heads / ffn / vocab."""
    d = ModelDesc()
    d.hidden, d.q_heads, d.kv_heads, d.ffn, d.vocab = (shape[k] for k in ("hidden", "q_heads", "kv_heads", "ffn",
                                                                           "vocab"))
    d.head_dim, d.q_dim, d.kv_dim = 128, 128 * d.q_heads, 128 * d.kv_heads
    out = TpSlice()
    check(lib().atlas_cuda_tp_slice(ctypes.byref(d), rank, size, ctypes.byref(out)), "atlas_cuda_tp_slice")
    return out


def connect_tp(rt: "Runtime", group=None) -> None:
    """Exchange the ranks' handles through torch.distributed (any backend:
    the handles are 64 host bytes each) and connect this rank's runtime."""
    import torch.distributed as dist
    handles = [None] * rt.tp_size
    dist.all_gather_object(handles, rt.tp_handle(), group=group)
    rt.tp_connect(handles)


def dequant(type_id: int, d_blocks, nblocks: int, d_out, stream: int = 0) -> None:
    check(lib().atlas_cuda_dequant(type_id, _ptr(d_blocks), nblocks, _ptr(d_out), ctypes.c_void_p(stream)),
          "atlas_cuda_dequant")


def gemv(type_id: int, d_w, rows: int, cols: int, d_x, d_y, stream: int = 0) -> None:
    check(lib().atlas_cuda_gemv(type_id, _ptr(d_w), rows, cols, _ptr(d_x), _ptr(d_y), ctypes.c_void_p(stream)),
          "atlas_cuda_gemv")


def gemv_noalloc(type_id: int, d_w, rows: int, cols: int, d_x, d_y, stream: int = 0) -> None:
    check(lib().atlas_cuda_gemv_noalloc(type_id, _ptr(d_w), rows, cols, _ptr(d_x), _ptr(d_y),
                                        ctypes.c_void_p(stream)), "atlas_cuda_gemv_noalloc")


def gemm(type_id: int, d_w, rows: int, cols: int, d_x, tokens: int, d_y, stream: int = 0) -> None:
    check(lib().atlas_cuda_gemm(type_id, _ptr(d_w), rows, cols, _ptr(d_x), tokens, _ptr(d_y),
                                ctypes.c_void_p(stream)), "atlas_cuda_gemm")


def _kind(t) -> str:
    """The name of a tensor's element type."""
    return str(t.dtype).rpartition(".")[2]


class Kv8Cache:
    """An 8-bit KV cache of one layer in caller-owned device buffers (AtlasKv8, include/atlas_cuda.h).

    k, v: int8 [nseq, kv_heads, max_context, 128]; k_scale, v_scale: float32 [nseq, kv_heads, ceil(max_context / block)];
    k_sum: int16 [nseq, kv_heads, ceil(max_context / block), 128], or None (kv8_attn_sparse then refuses the cache).
    The object keeps references to the buffers; they must be dense, which is checked where they say so."""

    def __init__(self, k, v, k_scale, v_scale, k_sum=None, *, nseq: int, kv_heads: int, max_context: int, block: int):
        blocks = -(-max_context // block) if block > 0 else 0
        for t, n, kind in ((k, max_context * 128, "int8"), (v, max_context * 128, "int8"), (k_scale, blocks, "float32"),
                           (v_scale, blocks, "float32"), (k_sum, blocks * 128, "int16")):
            if hasattr(t, "is_contiguous") and (not t.is_contiguous() or _kind(t) != kind
                                                or t.numel() != nseq * kv_heads * n):
                raise ValueError("Kv8Cache: a buffer of another size or type, or one that is not dense")
        self.buffers = (k, v, k_scale, v_scale, k_sum)
        self.nseq, self.kv_heads, self.max_context, self.block = nseq, kv_heads, max_context, block
        self.desc = Kv8Desc(*(None if t is None else t.data_ptr() for t in self.buffers), nseq, kv_heads, max_context,
                            block)
        self._ref = ctypes.byref(self.desc)
        # the types that the calls look for first, where the buffers are torch's
        self._f32 = getattr(k_scale, "dtype", None)
        self._i32 = sys.modules["torch"].int32 if "torch" in sys.modules else None


def _addr(t):
    return None if t is None else t.data_ptr()


def _kv8_ints(who: str, name: str, t, n: int) -> None:
    """Refuses a tensor that does not begin with n dense 32-bit integers."""
    if t is not None and hasattr(t, "dtype") and (
            _kind(t) not in ("int32", "uint32") or t.numel() < n or not t.is_contiguous()):
        raise AtlasError(-1, f"{who}: {name} must be {n} dense 32-bit integers")


def _kv8_rows(who: str, name: str, t, nseq: int, tokens: int, heads: int, ld: int, kind: str = "float32") -> None:
    """Refuses a tensor that is not token rows [nseq, tokens, heads, 128] of type `kind`, ld values from token to token (0:
    dense). One that is not 4-dimensional must be dense, and long enough. A dense one of just the size passes if its dimensions
    begin and end where those do, so that the same values are in the same places ([nseq, heads, 1, 128] of one token)."""
    if not tokens or not hasattr(t, "dtype"):
        return
    step = ld or heads * 128
    if t.dim() == 4:
        shape, stride = t.shape, t.stride()
        ok = (shape[0] >= nseq and shape[1] >= tokens and shape[2] >= heads and shape[3] == 128 and stride[3] == 1
              and (heads == 1 or stride[2] == 128) and (tokens == 1 or stride[1] == step)
              and (nseq == 1 or stride[0] == tokens * step)
              or t.is_contiguous() and t.numel() == nseq * tokens * step and step == heads * 128
              and {1, 128, step, tokens * step, nseq * tokens * step}.issuperset(accumulate(reversed(shape), mul)))
    else:
        ok = t.is_contiguous() and t.numel() >= (nseq * tokens - 1) * step + heads * 128
    if not ok or _kind(t) != kind:
        raise AtlasError(-1, f"{who}: {name} must be {kind} rows of {nseq} sequences x {tokens} tokens x {heads} heads x 128, "
                             f"{step} values from token to token")


def _kv8_check(who: str, cache: Kv8Cache, tokens: int, heads: int, pos0, n_tok, names, a, lda: int, b, ldb: int) -> None:
    """Refuses tensors of another type, layout or size. a, b: rows of `heads` each. Dense ones of just the shape, as most
    calls have, pass at once."""
    n = cache.nseq
    shape, f32, i32 = (n, tokens, heads, 128), cache._f32, cache._i32
    try:
        if (a.dtype is f32 and b.dtype is f32 and pos0.dtype is i32 and a.shape == shape and b.shape == shape
                and pos0.nbytes == 4 * n and a.is_contiguous() and b.is_contiguous() and pos0.is_contiguous()
                and (n_tok is None or n_tok.dtype is i32 and n_tok.nbytes == 4 * n and n_tok.is_contiguous())
                and not lda and not ldb):
            return
    except AttributeError:   # not a tensor, but an object with an address: what can be seen of it is checked
        pass
    _kv8_rows(who, names[0], a, n, tokens, heads, lda)
    _kv8_rows(who, names[1], b, n, tokens, heads, ldb)
    _kv8_ints(who, "pos0", pos0, n)
    _kv8_ints(who, "n_tok", n_tok, n)


def kv8_append(cache: Kv8Cache, tokens: int, pos0, k, v, n_tok=None, ld: int = 0, stream: int = 0) -> None:
    """Stores up to `tokens` new rows k, v [nseq, tokens, kv_heads, 128] of each sequence s at positions pos0[s], ...
    (pos0, n_tok: 32-bit device integers; n_tok None: all of them). atlas_cuda_kv8_append. Here and below, `stream` is a
    cudaStream_t (0: the legacy default stream), and tensors of another type, layout or size are refused."""
    _kv8_check("kv8_append", cache, tokens, cache.kv_heads, pos0, n_tok, ("k", "v"), k, ld, v, ld)
    check(lib().atlas_cuda_kv8_append(cache._ref, tokens, pos0.data_ptr(), _addr(n_tok), k.data_ptr(), v.data_ptr(), ld,
                                      stream), "kv8_append")


def kv8_read(cache: Kv8Cache, tokens: int, pos0, k, v, n_tok=None, ld: int = 0, stream: int = 0) -> None:
    """The rows at positions pos0[s], ... as the values that they stand for, into k, v [nseq, tokens, kv_heads, 128].
    atlas_cuda_kv8_read."""
    _kv8_check("kv8_read", cache, tokens, cache.kv_heads, pos0, n_tok, ("k", "v"), k, ld, v, ld)
    check(lib().atlas_cuda_kv8_read(cache._ref, tokens, pos0.data_ptr(), _addr(n_tok), k.data_ptr(), v.data_ptr(), ld,
                                    stream), "kv8_read")


def kv8_attn(cache: Kv8Cache, q_heads: int, tokens: int, pos0, q, out, n_tok=None, ldq: int = 0, ldo: int = 0,
             stream: int = 0) -> None:
    """Causal attention of q [nseq, tokens, q_heads, 128] over the cache into out. atlas_cuda_kv8_attn."""
    _kv8_check("kv8_attn", cache, tokens, q_heads, pos0, n_tok, ("q", "out"), q, ldq, out, ldo)
    check(lib().atlas_cuda_kv8_attn(cache._ref, q_heads, tokens, pos0.data_ptr(), _addr(n_tok), q.data_ptr(), ldq,
                                    out.data_ptr(), ldo, stream), "kv8_attn")


def kv8_attn_form(cache: Kv8Cache, q_heads: int, tokens: int) -> tuple:
    """(rows of a KV head that a CTA takes, CTAs that share their positions) of such a kv8_attn on the current device.
    atlas_cuda_kv8_attn_form."""
    rows, ctas = ctypes.c_uint32(), ctypes.c_uint32()
    check(lib().atlas_cuda_kv8_attn_form(cache._ref, q_heads, tokens, ctypes.byref(rows), ctypes.byref(ctas)),
          "kv8_attn_form")
    return rows.value, ctas.value


def kv8_attn_sparse(cache: Kv8Cache, q_heads: int, tokens: int, n_sel: int, pos0, q, out, sel, n_tok=None, ldq: int = 0,
                    ldo: int = 0, stream: int = 0) -> None:
    """Attention over the n_sel blocks that each token and KV head selects; sel [nseq, tokens, kv_heads, n_sel] (int32)
    receives them. atlas_cuda_kv8_attn_sparse."""
    _kv8_check("kv8_attn_sparse", cache, tokens, q_heads, pos0, n_tok, ("q", "out"), q, ldq, out, ldo)
    _kv8_ints("kv8_attn_sparse", "sel", sel, cache.nseq * tokens * cache.kv_heads * n_sel)
    check(lib().atlas_cuda_kv8_attn_sparse(cache._ref, q_heads, tokens, n_sel, pos0.data_ptr(), _addr(n_tok),
                                           q.data_ptr(), ldq, out.data_ptr(), ldo, sel.data_ptr(), stream),
          "kv8_attn_sparse")


_PAGED_TYPES = {"float16": 0, "bfloat16": 1}


class PagedCache:
    """A paged KV cache of all layers in caller-owned device buffers (AtlasPaged, include/atlas_cuda.h).

    k, v: float16 or bfloat16 [layers, pages, kv_heads, page, 128]; table: int32 [nseq, max_pages], -1 where there is no page;
    refs: int32 [pages], how many entries name each page. An empty cache has a table of -1 and refs of 0. `work`: the calls'
    workspace, at least paged_work_bytes(pages) bytes of the same device (None: one is made). The object keeps references to
    the tensors. Calls on one cache are ordered by their streams; caches that share a workspace count as one."""

    def __init__(self, k, v, table, refs, work=None):
        if (k.dim() != 5 or k.shape[4] != 128 or tuple(v.shape) != tuple(k.shape) or _kind(k) not in _PAGED_TYPES
                or _kind(v) != _kind(k) or not k.is_contiguous() or not v.is_contiguous()):
            raise ValueError("PagedCache: k and v must be dense float16 or bfloat16 [layers, pages, kv_heads, page, 128]")
        self.layers, self.pages, self.kv_heads, self.page = (int(x) for x in k.shape[:4])
        if table.dim() != 2 or _kind(table) != "int32" or not table.is_contiguous():
            raise ValueError("PagedCache: the table must be dense int32 [nseq, max_pages]")
        if refs.dim() != 1 or refs.numel() != self.pages or _kind(refs) != "int32" or not refs.is_contiguous():
            raise ValueError("PagedCache: refs must be dense int32 [pages]")
        self.nseq, self.max_pages = (int(x) for x in table.shape)
        self.kind, self.dtype, self._i32 = _kind(k), k.dtype, table.dtype
        self.desc = PagedDesc(k.data_ptr(), v.data_ptr(), table.data_ptr(), refs.data_ptr(), None, 0, _PAGED_TYPES[self.kind],
                              self.layers, self.pages, self.kv_heads, self.page, self.nseq, self.max_pages)
        self._ref = ctypes.byref(self.desc)
        need = ctypes.c_uint64()
        check(lib().atlas_cuda_paged_work(self._ref, ctypes.byref(need)), "paged_work")
        if work is None:
            work = k.new_empty((need.value + 1) // 2)   # of 2-byte values
        if not work.is_contiguous() or work.nbytes < need.value:
            raise ValueError(f"PagedCache: the workspace must be {need.value} dense bytes")
        self.buffers = (k, v, table, refs, work)
        if len({t.device for t in self.buffers}) != 1:
            raise ValueError("PagedCache: the buffers must be of one device")
        self.desc.work, self.desc.work_bytes = work.data_ptr(), work.nbytes


def _paged_ints(who: str, cache: PagedCache, name: str, t, n: int) -> None:
    """_kv8_ints; a tensor of just the size and type, as most calls have, passes at once."""
    if t is not None and not (t.dtype is cache._i32 and t.nbytes == 4 * n and t.is_contiguous()):
        _kv8_ints(who, name, t, n)


def _paged_check(who: str, cache: PagedCache, tokens: int, heads: int, pos0, n_tok, names=(), a=None, lda: int = 0, b=None,
                 ldb: int = 0) -> None:
    """Refuses tensors of another type, layout or size. a, b: rows of `heads` each, or None. Dense ones of just the shape, as
    most calls have, pass at once."""
    n, shape, kind, i32 = cache.nseq, (cache.nseq, tokens, heads, 128), cache.dtype, cache._i32
    if ((a is None or a.dtype is kind and b.dtype is kind and a.shape == shape and b.shape == shape and not lda and not ldb
         and a.is_contiguous() and b.is_contiguous())
            and pos0.dtype is i32 and pos0.nbytes == 4 * n and pos0.is_contiguous()
            and (n_tok is None or n_tok.dtype is i32 and n_tok.nbytes == 4 * n and n_tok.is_contiguous())):
        return
    if a is not None:
        _kv8_rows(who, names[0], a, n, tokens, heads, lda, cache.kind)
        _kv8_rows(who, names[1], b, n, tokens, heads, ldb, cache.kind)
    _kv8_ints(who, "pos0", pos0, n)
    _kv8_ints(who, "n_tok", n_tok, n)


def paged_fork(cache: PagedCache, parent, length, first=None, stream: int = 0) -> None:
    """Sequence s becomes what sequence parent[s] was up to position length[s] (and from first[s] on): int32 [nseq] each.
    atlas_cuda_paged_fork. Here and below, `stream` is a cudaStream_t (0: the legacy default stream), and tensors of another
    type, layout or size are refused."""
    _paged_ints("paged_fork", cache, "parent", parent, cache.nseq)
    _paged_ints("paged_fork", cache, "length", length, cache.nseq)
    _paged_ints("paged_fork", cache, "first", first, cache.nseq)
    check(lib().atlas_cuda_paged_fork(cache._ref, _addr(parent), _addr(length), _addr(first), stream), "paged_fork")


def paged_reserve(cache: PagedCache, tokens: int, pos0, short, n_tok=None, stream: int = 0) -> None:
    """Gives each sequence s pages of its own for positions pos0[s], ... of its next n_tok[s] tokens (None: `tokens`); short
    (int32 [1]) receives how many pages are lacking, and then nothing has changed. atlas_cuda_paged_reserve."""
    _paged_check("paged_reserve", cache, tokens, 0, pos0, n_tok)
    _paged_ints("paged_reserve", cache, "short", short, 1)
    check(lib().atlas_cuda_paged_reserve(cache._ref, tokens, pos0.data_ptr(), _addr(n_tok), _addr(short), stream),
          "paged_reserve")


def paged_compact(cache: PagedCache, used, stream: int = 0) -> None:
    """Moves the pages in use to the pool's start; used (int32 [1]) receives how many there are. atlas_cuda_paged_compact."""
    _paged_ints("paged_compact", cache, "used", used, 1)
    check(lib().atlas_cuda_paged_compact(cache._ref, _addr(used), stream), "paged_compact")


def paged_append(cache: PagedCache, layer: int, tokens: int, pos0, k, v, n_tok=None, ld: int = 0, stream: int = 0) -> None:
    """Stores up to `tokens` new rows k, v [nseq, tokens, kv_heads, 128] of a layer at positions pos0[s], ... (pos0, n_tok:
    int32 [nseq]; n_tok None: all of them). atlas_cuda_paged_append."""
    _paged_check("paged_append", cache, tokens, cache.kv_heads, pos0, n_tok, ("k", "v"), k, ld, v, ld)
    check(lib().atlas_cuda_paged_append(cache._ref, layer, tokens, pos0.data_ptr(), _addr(n_tok), k.data_ptr(), v.data_ptr(),
                                        ld, stream), "paged_append")


def paged_attn(cache: PagedCache, layer: int, q_heads: int, tokens: int, pos0, q, out, n_tok=None, ldq: int = 0, ldo: int = 0,
               stream: int = 0) -> None:
    """Causal attention of q [nseq, tokens, q_heads, 128] over a layer's pages into out. atlas_cuda_paged_attn."""
    _paged_check("paged_attn", cache, tokens, q_heads, pos0, n_tok, ("q", "out"), q, ldq, out, ldo)
    check(lib().atlas_cuda_paged_attn(cache._ref, layer, q_heads, tokens, pos0.data_ptr(), _addr(n_tok), q.data_ptr(), ldq,
                                      out.data_ptr(), ldo, stream), "paged_attn")


def paged_attn_form(cache: PagedCache, q_heads: int, tokens: int) -> int:
    """The rows of a KV head that a CTA takes at a time in such a paged_attn on the current device. atlas_cuda_paged_attn_form."""
    rows = ctypes.c_uint32()
    check(lib().atlas_cuda_paged_attn_form(cache._ref, q_heads, tokens, ctypes.byref(rows)), "paged_attn_form")
    return rows.value
