"""ctypes binding of ``libkata_attn.so`` (the C ABI in ``include/kata_attn.h``) for the tests and the benchmark.

torch is used only to own device memory and streams; every attention computation goes through the C ABI into the
hand-written CUDA kernels. There is no CPU or PyTorch fallback: if the library is missing, loading raises.
"""
from __future__ import annotations

import array
import ctypes as C
import os

import numpy as np
import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libkata_attn.so")

OK = 0
KV_FP16, KV_INT8, KV_INT8V, KV_INT8G = 0, 1, 2, 3
_KV_MODES = {"fp16": KV_FP16, "int8": KV_INT8, "int8v": KV_INT8V, "int8g": KV_INT8G}   # the reference's KATA_KV values (src/engine.cpp:54)
ROUND_RINT, ROUND_HALF_AWAY = 0, 1
ACT_F32, ACT_BF16, ACT_F16 = 0, 1, 2
_ACT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # KATA_ACT_*
QD, KVD, QFULL, MAX_BATCH = 6144, 1024, 12288, 64

EXPORTS = [
    "kata_attn_create", "kata_attn_destroy", "kata_attn_reset", "kata_attn_numerics_tag", "kata_attn_last_error", "kata_attn_check",
    "kata_attn_prep", "kata_attn_prep_axes", "kata_attn_kv_quant", "kata_attn_decode", "kata_attn_decode_scalar", "kata_attn_prefill",
    "kata_attn_decode_partial", "kata_attn_merge_parts", "kata_attn_kv_planes", "kata_attn_kv_plane_row_bytes",
    "kata_attn_kv_plane_read", "kata_attn_kv_plane_write", "kata_attn_kv_plane_ptr", "kata_attn_mark_rows_written", "kata_attn_launch_count", "kata_attn_decode_static", "kata_attn_decode_static_check", "kata_attn_set_position_offset", "kata_attn_set_kv_heads", "kata_attn_out_fwht",
    "kata_attn_layers_step", "kata_attn_layers_decode", "kata_attn_prefill_plan", "kata_attn_decode_plan", "kata_attn_host_step_create", "kata_attn_host_step_destroy", "kata_attn_host_step_run",
    "kata_attn_peer_create", "kata_attn_peer_open", "kata_attn_peer_open_pointers", "kata_attn_peer_buffer", "kata_attn_peer_set_wait_polls", "kata_attn_peer_exchange_merge", "kata_attn_peer_decode", "kata_attn_peer_layers_step",
    "kata_attn_peer_check", "kata_attn_peer_resync", "kata_attn_peer_last_error", "kata_attn_peer_destroy",
    "kata_draft_create", "kata_draft_destroy", "kata_draft_reset", "kata_draft_last_error", "kata_draft_qk", "kata_draft_attn", "kata_draft_ring_ptr",
    "kata_draft_ring_read", "kata_draft_ring_write", "kata_draft_launch_count",
]


class Config(C.Structure):
    _fields_ = [("device", C.c_int32), ("n_layers", C.c_int32), ("n_seqs", C.c_int32), ("max_ctx", C.POINTER(C.c_int32)),
                ("kv_mode", C.c_int32), ("quant_round", C.c_int32), ("dec_chunk", C.c_int32), ("flags", C.c_int32)]


class KataError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"kata_attn error {code}: {msg}")
        self.code = code


_lib = None


def lib() -> C.CDLL:
    """Loads the library; raises if it has not been built (``python -m kata_b200.build``)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `python -m kata_b200.build` (there is no fallback path)")
        L = C.CDLL(LIB_PATH)
        L.kata_attn_numerics_tag.restype = C.c_char_p
        L.kata_attn_last_error.restype = C.c_char_p
        L.kata_attn_kv_plane_row_bytes.restype = C.c_size_t
        L.kata_attn_kv_plane_ptr.restype = C.c_void_p
        L.kata_attn_launch_count.restype = C.c_uint64
        for name in EXPORTS:
            getattr(L, name)
        for name, (res, args) in _PAGED_SIGNATURES.items():
            f = getattr(L, name)
            f.restype, f.argtypes = res, args
        _lib = L
    return _lib


def _i32(xs):
    """ctypes int32 array of a list / numpy vector of small integers (about 1 us; the numpy route costs three times that per call)."""
    if isinstance(xs, np.ndarray):
        xs = xs.reshape(-1).tolist()
    a = (C.c_int32 * len(xs))(*[int(x) for x in xs])
    return a, a


def _dp(t):
    if t is None:
        return C.c_void_p(0)
    assert t.is_cuda and t.is_contiguous()
    return C.c_void_p(t.data_ptr())


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def out_fwht(x, sign, out=None):
    """The engine's attention output transform (sign, 1024-point Walsh-Hadamard per block, 1/32): x [rows][width] fp32 on the GPU."""
    out = torch.empty_like(x) if out is None else out
    assert x.dtype == torch.float32 and sign.dtype == torch.float32 and x.dim() == 2
    rc = lib().kata_attn_out_fwht(_dp(x), _dp(sign), _dp(out), C.c_int64(x.shape[0]), C.c_int32(x.shape[1]), _stream())
    if rc != OK:
        raise KataError(rc, "kata_attn_out_fwht")
    return out


class _Native:
    """A native context. It is destroyed when the last that holds it is gone: the Python object, by close(), or a tensor that aliases its memory."""

    def __init__(self, destroy, h):
        self.destroy, self.h = destroy, h

    def __del__(self):
        try:
            self.destroy(self.h)
        except Exception:
            pass


def _alias(native, ptr, shape, kind, device):
    """A tensor over a native context's memory; torch keeps the interface object, and with it the context, as long as the storage lives."""
    class _Memory:
        __cuda_array_interface__ = {"shape": shape, "typestr": kind, "data": (ptr, False), "version": 3, "strides": None}
    memory = _Memory()
    memory.native = native
    return torch.as_tensor(memory, device=device)


class AttnContext:
    """One context per GPU: the KV caches of ``len(max_ctx)`` sequences x ``n_layers`` layers plus all scratch."""

    def __init__(self, n_layers: int, max_ctx, kv_mode: str = "fp16", quant_round: str = "rint", device: int | None = None, dec_chunk: int = 0, legacy_prefill: bool = False, flags: int = 0):
        self.L = lib()
        self.device = torch.cuda.current_device() if device is None else device
        self.max_ctx, mp = _i32(max_ctx)
        self.n_layers, self.n_seqs = n_layers, len(self.max_ctx)
        if kv_mode not in _KV_MODES:
            raise ValueError(f"kv_mode {kv_mode!r}: one of {sorted(_KV_MODES)}")
        self.int8, self.kv_mode = kv_mode == "int8", kv_mode
        cfg = Config(self.device, n_layers, self.n_seqs, mp, _KV_MODES[kv_mode], ROUND_HALF_AWAY if quant_round == "half_away" else ROUND_RINT, dec_chunk, (1 if legacy_prefill else 0) | int(flags))
        self.h = C.c_void_p()
        rc = self.L.kata_attn_create(C.byref(cfg), C.byref(self.h))
        if rc != OK:
            raise KataError(rc, "kata_attn_create failed")
        self._native = _Native(self.L.kata_attn_destroy, self.h)

    def close(self):
        self.h, self._native = C.c_void_p(), None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _ck(self, rc):
        if rc != OK:
            raise KataError(rc, self.L.kata_attn_last_error(self.h).decode())

    def tag(self) -> str:
        return self.L.kata_attn_numerics_tag(self.h).decode()

    def reset(self):
        self._ck(self.L.kata_attn_reset(self.h, _stream()))

    def check(self):
        self._ck(self.L.kata_attn_check(self.h, _stream()))

    def set_position_offset(self, seq: int, first_position: int):
        self._ck(self.L.kata_attn_set_position_offset(self.h, seq, first_position))

    def set_kv_heads(self, kv_head_lo: int, kv_head_n: int):
        """This context computes KV heads [lo, lo + n) only (a rank of a head-sharded group)."""
        self._ck(self.L.kata_attn_set_kv_heads(self.h, kv_head_lo, kv_head_n))

    def launches(self) -> int:
        return int(self.L.kata_attn_launch_count(self.h))

    def prep(self, layer, seq_ids, pos0, T, qfull, kproj, vproj, qnorm, knorm, h0=0, nh=32, q16=None, q32=None, gate=None, want_q32=False):
        """Returns (q16, q32 or None, gate). qfull [n][T][12288], kproj/vproj [n][T][1024] in fp32 or bf16."""
        sa, sp = _i32(seq_ids)
        pa, pp = _i32(pos0)
        n = len(sa)
        ref = kproj if kproj is not None else qfull
        act = _ACT[ref.dtype]
        dev = ref.device
        if h0 < 24:
            q16 = torch.empty((n, T, QD), dtype=torch.float16, device=dev) if q16 is None else q16
            gate = torch.empty((n, T, QD), dtype=torch.float32, device=dev) if gate is None else gate
            if want_q32 and q32 is None:
                q32 = torch.empty((n, T, QD), dtype=torch.float32, device=dev)
        self._ck(self.L.kata_attn_prep(self.h, layer, n, sp, pp, T, _dp(qfull), _dp(kproj), _dp(vproj), act, _dp(qnorm), _dp(knorm),
                                       _dp(q16), _dp(q32), _dp(gate), h0, nh, _stream()))
        return q16, q32, gate

    def prep_axes(self, layer, seq_ids, pos0, T, axis_pos, sections, qfull, kproj, vproj, qnorm, knorm, interleaved=False, h0=0, nh=32, q16=None, q32=None, gate=None):
        """As prep, with rotary positions of three axes: axis_pos int32 [n][T][3] on the device, sections the frequencies per axis (sum 32) (kata_attn_prep_axes)."""
        sa, sp = _i32(seq_ids)
        pa, pp = _i32(pos0)
        n, ref = len(sa), kproj if kproj is not None else qfull
        if axis_pos.dtype != torch.int32 or axis_pos.numel() != n * T * 3 or not axis_pos.is_contiguous() or axis_pos.device != ref.device or len(sections) != 3:
            raise ValueError(f"axis_pos: a contiguous int32 tensor [{n}][{T}][3] on {ref.device} and three sections are needed")
        if h0 < 24:
            q16 = torch.empty((n, T, QD), dtype=torch.float16, device=ref.device) if q16 is None else q16
            gate = torch.empty((n, T, QD), dtype=torch.float32, device=ref.device) if gate is None else gate
        xa, xp = _i32(sections)
        self._ck(self.L.kata_attn_prep_axes(self.h, layer, n, sp, pp, T, _dp(axis_pos), xp, 1 if interleaved else 0, _dp(qfull), _dp(kproj), _dp(vproj), _ACT[ref.dtype],
                                            _dp(qnorm), _dp(knorm), _dp(q16), _dp(q32), _dp(gate), h0, nh, _stream()))
        return q16, q32, gate

    def layers_step(self, n_layers, seq_ids, pos0, T, qfull, kproj, vproj, qnorm, knorm, q16, gate, out, first_pos=0):
        """prep + decode of layers 0..n_layers-1 in one call; every tensor is [n_layers][...] on the device."""
        sa, sp = _i32(seq_ids); pa, pp = _i32(pos0)
        self._ck(self.L.kata_attn_layers_step(self.h, n_layers, len(sa), sp, pp, T, first_pos, _dp(qfull), _dp(kproj), _dp(vproj), _ACT[qfull.dtype], _dp(qnorm), _dp(knorm),
                                              _dp(q16), _dp(gate), _dp(out), _ACT[out.dtype], _stream()))
        return out

    def layers_decode(self, n_layers, seq_ids, pos_base, T, q16, gate, out, first_pos=0):
        """kata_attn_decode of layers 0..n_layers-1 in one call (the attention kernels by themselves); tensors are [n_layers][...]."""
        sa, sp = _i32(seq_ids); pa, pp = _i32(pos_base)
        self._ck(self.L.kata_attn_layers_decode(self.h, n_layers, len(sa), sp, pp, T, first_pos, _dp(q16), _dp(gate), _dp(out), _ACT[out.dtype], _stream()))
        return out

    def kv_quant(self, layer, seq, ks, vs, pos0):
        self._ck(self.L.kata_attn_kv_quant(self.h, layer, seq, _dp(ks), _dp(vs), vs.shape[0], pos0, _stream()))   # ks may be None on an int8v context

    def decode(self, layer, seq_ids, pos_base, T, q16, gate, first_pos=0, out=None, out_dtype=torch.float32):
        sa, sp = _i32(seq_ids)
        pa, pp = _i32(pos_base)
        n = len(sa)
        out = torch.empty((n, T, QD), dtype=out_dtype, device=q16.device) if out is None else out
        self._ck(self.L.kata_attn_decode(self.h, layer, n, sp, pp, T, first_pos, _dp(q16), _dp(gate), _dp(out), _ACT[out.dtype], _stream()))
        return out

    def decode_scalar(self, layer, seq_ids, pos_base, T, q32, gate, first_pos=0, out=None):
        sa, sp = _i32(seq_ids)
        pa, pp = _i32(pos_base)
        n = len(sa)
        out = torch.empty((n, T, QD), dtype=torch.float32, device=q32.device) if out is None else out
        self._ck(self.L.kata_attn_decode_scalar(self.h, layer, n, sp, pp, T, first_pos, _dp(q32), _dp(gate), _dp(out), _stream()))
        return out

    def prefill(self, layer, seq_ids, pos_base, M, q16, gate, out=None, out_dtype=torch.float32):
        sa, sp = _i32(seq_ids)
        pa, pp = _i32(pos_base)
        n = len(sa)
        out = torch.empty((n, M, QD), dtype=out_dtype, device=q16.device) if out is None else out
        self._ck(self.L.kata_attn_prefill(self.h, layer, n, sp, pp, M, _dp(q16), _dp(gate), _dp(out), _ACT[out.dtype], _stream()))
        return out

    def decode_partial(self, layer, seq, pos_base, T, key_lo, key_hi, q16, part=None):
        part = torch.empty((T * 24, 258), dtype=torch.float32, device=q16.device) if part is None else part
        self._ck(self.L.kata_attn_decode_partial(self.h, layer, seq, pos_base, T, key_lo, key_hi, _dp(q16), _dp(part), _stream()))
        return part

    def merge_parts(self, parts, T, gate, out=None, out_dtype=torch.float32):
        n_parts = parts.shape[0]
        out = torch.empty((T, QD), dtype=out_dtype, device=parts.device) if out is None else out
        self._ck(self.L.kata_attn_merge_parts(self.h, _dp(parts), n_parts, T, _dp(gate), _dp(out), _ACT[out.dtype], _stream()))
        return out

    # ---- KV planes (prefix-cache contract) ----
    def kv_planes(self) -> int:
        return int(self.L.kata_attn_kv_planes(self.h))

    def plane_row_bytes(self, plane: int) -> int:
        return int(self.L.kata_attn_kv_plane_row_bytes(self.h, plane))

    def plane_read(self, layer, seq, plane, row0, nrows) -> np.ndarray:
        buf = np.empty(nrows * self.plane_row_bytes(plane), np.uint8)
        self._ck(self.L.kata_attn_kv_plane_read(self.h, layer, seq, plane, row0, nrows, buf.ctypes.data_as(C.c_void_p)))
        return buf

    def plane_write(self, layer, seq, plane, row0, data: np.ndarray):
        data = np.ascontiguousarray(data).view(np.uint8).reshape(-1)
        rb = self.plane_row_bytes(plane)
        assert rb and data.size % rb == 0
        self._ck(self.L.kata_attn_kv_plane_write(self.h, layer, seq, plane, row0, data.size // rb, data.ctypes.data_as(C.c_void_p)))

    def plane_ptr(self, layer, seq, plane) -> int:
        return int(self.L.kata_attn_kv_plane_ptr(self.h, layer, seq, plane) or 0)

    def mark_rows_written(self, seq: int, pos_lo: int):
        self._ck(self.L.kata_attn_mark_rows_written(self.h, seq, pos_lo))

    def plane_tensor(self, layer, seq, plane, nrows) -> torch.Tensor:
        """A uint8 CUDA tensor [nrows][row bytes] aliasing the plane's rows (through kata_attn_kv_plane_ptr): lets a test write rows with a
        device-side copy, as a device-resident restore would."""
        return _alias(self._native, self.plane_ptr(layer, seq, plane), (nrows, self.plane_row_bytes(plane)), "|u1", torch.device("cuda", self.device))


def decode_static(k_rows, v_rows, seq_row0, pos_base, T, q16, gate, first_pos=0, out=None, out_dtype=torch.float32):
    """kata_attn_decode_static: decode over caller-owned fp16 K/V rows ([rows][1024] tensors) with no context and no
    allocation inside the library. Returns (status code, out)."""
    L = lib()
    n = len(pos_base)
    rows0 = (C.c_int64 * n)(*[int(x) for x in seq_row0])
    pa, pp = _i32(pos_base)
    out = torch.empty((n, T, QD), dtype=out_dtype, device=q16.device) if out is None else out
    rc = L.kata_attn_decode_static(_dp(k_rows), _dp(v_rows), C.c_int64(k_rows.shape[0]), n, rows0, pp, T, first_pos, _dp(q16), _dp(gate), _dp(out),
                                   _ACT[out.dtype], _stream())
    return rc, out


class DraftConfig(C.Structure):
    _fields_ = [("device", C.c_int32), ("n_layers", C.c_int32), ("ring", C.c_int32), ("window", C.c_int32)]


class DraftContext:
    """The block drafter's K/V rings and attention (include/kata_draft.h; Draft::kbuf/vbuf, src/draft.h:36)."""

    def __init__(self, n_layers: int = 5, ring: int = 4096, window: int = 2048, device: int | None = None):
        self.L = lib()
        self.L.kata_draft_last_error.restype = C.c_char_p
        self.L.kata_draft_ring_ptr.restype = C.c_void_p
        self.L.kata_draft_launch_count.restype = C.c_uint64
        self.device = torch.cuda.current_device() if device is None else device
        self.n_layers, self.ring, self.window = n_layers, ring, window
        self.h = C.c_void_p()
        cfg = DraftConfig(self.device, n_layers, ring, window)
        rc = self.L.kata_draft_create(C.byref(cfg), C.byref(self.h))
        if rc != OK:
            raise KataError(rc, "kata_draft_create failed")

    def close(self):
        if self.h:
            self.L.kata_draft_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _ck(self, rc):
        if rc != OK:
            raise KataError(rc, self.L.kata_draft_last_error(self.h).decode())

    def reset(self):
        self._ck(self.L.kata_draft_reset(self.h, _stream()))

    def launches(self) -> int:
        return int(self.L.kata_draft_launch_count(self.h))

    def qk(self, layer, qin, kin, vin, qnorm, knorm, pos0, out=None):
        """k_draft_qk (returns the fp32 query rows) or, with qin None, k_draft_ctx_kv."""
        T = kin.shape[0]
        qout = (torch.empty((T, 4096), dtype=torch.float32, device=kin.device) if out is None else out) if qin is not None else None
        self._ck(self.L.kata_draft_qk(self.h, layer, _dp(qin), _dp(kin), _dp(vin), _dp(qnorm), _dp(knorm), _dp(qout), pos0, T, _stream()))
        return qout

    def attn(self, layer, q, pos0, out=None):
        T = q.shape[0]
        out = torch.empty((T, 4096), dtype=torch.float32, device=q.device) if out is None else out
        self._ck(self.L.kata_draft_attn(self.h, layer, _dp(q), _dp(out), pos0, T, _stream()))
        return out

    def ring_read(self, layer, value: bool, row0: int = 0, nrows: int | None = None) -> np.ndarray:
        nrows = self.ring - row0 if nrows is None else nrows
        buf = np.empty((nrows, 1024), np.uint16)
        self._ck(self.L.kata_draft_ring_read(self.h, layer, int(value), row0, nrows, buf.ctypes.data_as(C.c_void_p)))
        return buf

    def ring_write(self, layer, value: bool, row0: int, data: np.ndarray):
        data = np.ascontiguousarray(data).view(np.uint16).reshape(-1, 1024)
        self._ck(self.L.kata_draft_ring_write(self.h, layer, int(value), row0, data.shape[0], data.ctypes.data_as(C.c_void_p)))


class HostStep:
    """A decode or verify step of all layers with the projections and the output rows in pinned host memory (kata_attn_host_step_*):
    the copies of the neighbouring layers run under the layer that computes."""

    def __init__(self, ctx: "AttnContext", max_n: int, max_T: int = 1, act_dtype=torch.float32):
        self.L = lib(); self.ctx = ctx; self.h = C.c_void_p(); self.act = act_dtype
        rc = self.L.kata_attn_host_step_create(ctx.h, ctx.device, max_n, max_T, _ACT[act_dtype], C.byref(self.h))
        if rc != OK:
            raise KataError(rc, "kata_attn_host_step_create failed")

    def run(self, n_layers, seq_ids, pos0, T, h_qfull, h_kproj, h_vproj, d_qnorm, d_knorm, h_out, first_pos=0):
        """h_*: pinned host tensors [n_layers][n][T][...]; d_qnorm, d_knorm: device [n_layers][256]. Enqueued on the current stream."""
        sa, sp = _i32(seq_ids); pa, pp = _i32(pos0)
        for t in (h_qfull, h_kproj, h_vproj, h_out):
            assert t.device.type == "cpu" and t.is_contiguous()
        rc = self.L.kata_attn_host_step_run(self.h, n_layers, len(sa), sp, pp, T, first_pos, C.c_void_p(h_qfull.data_ptr()), C.c_void_p(h_kproj.data_ptr()), C.c_void_p(h_vproj.data_ptr()),
                                            _dp(d_qnorm), _dp(d_knorm), C.c_void_p(h_out.data_ptr()), _stream())
        if rc != OK:
            raise KataError(rc, self.L.kata_attn_last_error(self.ctx.h).decode() or "kata_attn_host_step_run failed")
        return h_out

    def close(self):
        if self.h:
            self.L.kata_attn_host_step_destroy(self.h); self.h = C.c_void_p()


class PeerExchange:
    """Push-and-merge of the split-KV parts between the GPUs of one box (kata_attn_peer_*): one process per GPU, handles swapped
    through ``torch.distributed`` object collectives (host side, once); the per-layer exchange itself runs no library collective."""

    def __init__(self, rank: int, world: int, device: int | None = None, group=None, buffers=None):
        self.L = lib()
        self.L.kata_attn_peer_last_error.restype = C.c_char_p
        self.L.kata_attn_peer_buffer.restype = C.c_void_p
        self.rank, self.world = rank, world
        self.device = torch.cuda.current_device() if device is None else device
        self.h = C.c_void_p()
        handle = (C.c_ubyte * 64)()
        rc = self.L.kata_attn_peer_create(self.device, rank, world, C.byref(self.h), handle)
        if rc != OK:
            raise KataError(rc, "kata_attn_peer_create failed")
        if buffers is not None:       # same process: device addresses of every rank's buffer (tests)
            self.open_pointers(buffers)
        elif world > 1 and group is not False:
            import torch.distributed as dist
            got = [None] * world
            dist.all_gather_object(got, bytes(handle), group=group)
            blob = (C.c_ubyte * (64 * world)).from_buffer_copy(b"".join(got))
            self._ck(self.L.kata_attn_peer_open(self.h, blob))

    def buffer(self) -> int:
        return int(self.L.kata_attn_peer_buffer(self.h) or 0)

    def open_pointers(self, buffers):
        arr = (C.c_void_p * self.world)(*[C.c_void_p(int(b)) for b in buffers])
        self._ck(self.L.kata_attn_peer_open_pointers(self.h, arr))

    def set_wait_polls(self, polls: int):
        self._ck(self.L.kata_attn_peer_set_wait_polls(self.h, C.c_uint32(polls)))

    def _ck(self, rc):
        if rc != OK:
            raise KataError(rc, self.L.kata_attn_peer_last_error(self.h).decode())

    def exchange_merge(self, part, T, gate, out=None, out_dtype=torch.float32):
        out = torch.empty((T, QD), dtype=out_dtype, device=part.device) if out is None else out
        self._ck(self.L.kata_attn_peer_exchange_merge(self.h, _dp(part), T, _dp(gate), _dp(out), _ACT[out.dtype], _stream()))
        return out

    def decode(self, ctx, layer, seq, pos_base, T, key_lo, key_hi, q16, gate, out=None, out_dtype=torch.float32):
        """This rank's share of a decode whose keys are split across the ranks, exchange and merge included (kata_attn_peer_decode)."""
        out = torch.empty((T, QD), dtype=out_dtype, device=q16.device) if out is None else out
        self._ck(self.L.kata_attn_peer_decode(self.h, ctx.h, layer, seq, pos_base, T, key_lo, key_hi, _dp(q16), _dp(gate), _dp(out), _ACT[out.dtype], _stream()))
        return out

    def layers_step(self, ctx, n_layers, seq, pos, T, key_lo, key_hi, appends, qfull, kproj, vproj, qnorm, knorm, q16, gate, out):
        """prep + split-KV decode of layers 0..n_layers-1 in one call (kata_attn_peer_layers_step); every tensor is [n_layers][T][...] on the device."""
        self._ck(self.L.kata_attn_peer_layers_step(self.h, ctx.h, n_layers, seq, pos, T, key_lo, key_hi, 1 if appends else 0, _dp(qfull), _dp(kproj), _dp(vproj), _ACT[qfull.dtype],
                                                   _dp(qnorm), _dp(knorm), _dp(q16), _dp(gate), _dp(out), _ACT[out.dtype], _stream()))
        return out

    def check(self):
        self._ck(self.L.kata_attn_peer_check(self.h, _stream()))

    def resync(self, call_number: int):
        self._ck(self.L.kata_attn_peer_resync(self.h, C.c_uint32(call_number)))

    def close(self):
        if self.h:
            self.L.kata_attn_peer_destroy(self.h)
            self.h = C.c_void_p()


_P, _I = C.c_void_p, C.c_int32
_PAGED_SIGNATURES = {   # declared, so that addresses and numbers pass as plain integers
    "kata_pages_create": (_I, [_I, _I, _I, _I, _P]), "kata_pages_destroy": (_I, [_P]), "kata_pages_reserve": (_I, [_P, _I, _I]), "kata_pages_trim": (_I, [_P, _I, _I]),
    "kata_pages_fork": (_I, [_P, _I, _I, _I, _P, _P, _P]), "kata_pages_count": (_I, [_P, _I]), "kata_pages_get": (_I, [_P, _I, _P, _I]), "kata_pages_free_count": (_I, [_P]), "kata_pages_owners": (_I, [_P, _I]),
    "kata_paged_create": (_I, [_P, _P]), "kata_paged_destroy": (_I, [_P]), "kata_paged_last_error": (C.c_char_p, [_P]), "kata_paged_launch_count": (C.c_uint64, [_P]), "kata_paged_check": (_I, [_P, _P]),
    "kata_paged_plane_ptr": (_P, [_P, _I, _I]), "kata_paged_reserve": (_I, [_P, _I, _I, _P]), "kata_paged_trim": (_I, [_P, _I, _I]), "kata_paged_fork": (_I, [_P, _I, _I, _I, _P]), "kata_paged_table": (_P, [_P]),
    "kata_paged_prep": (_I, [_P, _I, _I, _P, _P, _I, _P, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P]), "kata_paged_decode": (_I, [_P, _I, _I, _P, _P, _I, _P, _P, _P, _I, _I, _P]),
    "kata_paged_evict": (_I, [_P, _I, _I, _I, _P, _P, _P, _I, _I, _I, _P, _P]), "kata_paged_import": (_I, [_P, _I, _I, _I, _I, _I, _P, _I, _I, _I, _P]),
    "kata_paged_decode_plan": (_I, [_I, _P, _I, _I, _I, _P, _I, _P]),
}
PAGED_EXPORTS = list(_PAGED_SIGNATURES)
_PLANES = ("k", "v", "k_scale", "v_scale", "weight", "age")   # KATA_PAGED_* planes
PAGED_GATED, PAGED_WEIGHTS = 1, 2
_F16, _F32, _I32 = (torch.float16,), (torch.float32,), (torch.int32,)


def _ints(xs):
    """int32 array of a sequence of integers: its buffer is what the C call reads."""
    return array.array("i", xs.reshape(-1).tolist() if isinstance(xs, np.ndarray) else xs)


class PagedConfig(C.Structure):
    _fields_ = [("device", C.c_int32), ("n_layers", C.c_int32), ("n_seqs", C.c_int32), ("n_pages", C.c_int32), ("page_size", C.c_int32), ("max_slots", C.c_int32), ("heads", C.c_int32), ("kv_heads", C.c_int32),
                ("head_dim", C.c_int32), ("kv_mode", C.c_int32), ("rot_dim", C.c_int32), ("section", C.c_int32 * 3), ("interleaved", C.c_int32), ("flags", C.c_int32), ("rope_theta", C.c_double), ("planes", C.c_void_p * 6)]


class PagedContext:
    """A KV cache in pages (include/kata_paged.h): page tables, the prep that appends with positions of up to three axes, attention of
    the newest tokens over the pages, and eviction by accumulated attention weight."""

    def __init__(self, n_layers: int, n_seqs: int, n_pages: int, page_size: int, max_slots: int, heads: int = 24, kv_heads: int = 4, head_dim: int = 256, kv_mode: str = "fp16", rot_dim: int = 64, theta: float = 1e7,
                 sections=None, interleaved: bool = False, gated: bool = True, weights: bool = False, planes=None, device: int | None = None):
        """``sections``: rotary frequencies per axis (time, height, width), all on the first axis by default. ``planes``: the caller's tensors for planes
        ("k", "v", "k_scale", "v_scale", "weight", "age") in the header's layout, [n_layers] of them; the others are allocated, zero-filled."""
        L = self.L = lib()
        self.device = torch.cuda.current_device() if device is None else device
        self.cuda = torch.device("cuda", self.device)
        self.n_layers, self.n_seqs, self.n_pages, self.page_size, self.max_slots = n_layers, n_seqs, n_pages, page_size, max_slots
        self.heads, self.kv_heads, self.head_dim, self.kv_mode, self.gated, self.weights = heads, kv_heads, head_dim, kv_mode, gated, weights
        if kv_mode not in _KV_MODES:
            raise ValueError(f"kv_mode {kv_mode!r}: fp16 or int8")
        self.planes = dict(planes or {})
        for name, t in self.planes.items():
            if name not in _PLANES:
                raise ValueError(f"plane {name!r}: one of {_PLANES}")
            want = {"k": torch.int8 if kv_mode == "int8" else torch.float16, "weight": torch.float32, "age": torch.int32}.get("k" if name == "v" else name, torch.float16)
            n = n_layers * n_pages * page_size * kv_heads * (head_dim if name in ("k", "v") else 1)
            if not t.is_cuda or not t.is_contiguous() or t.dtype != want or t.numel() != n or t.device.index != self.device:
                raise ValueError(f"plane {name!r}: a contiguous {want} tensor of {n} elements on device {self.device}")
        sec = tuple(sections) if sections is not None else (rot_dim // 2, 0, 0)
        cfg = PagedConfig(self.device, n_layers, n_seqs, n_pages, page_size, max_slots, heads, kv_heads, head_dim, _KV_MODES[kv_mode], rot_dim, (C.c_int32 * 3)(*sec), int(interleaved),
                          (PAGED_GATED if gated else 0) | (PAGED_WEIGHTS if weights else 0), theta, (C.c_void_p * 6)(*[self.planes[p].data_ptr() if p in self.planes else None for p in _PLANES]))
        self.h = C.c_void_p()
        rc = L.kata_paged_create(C.byref(cfg), C.byref(self.h))
        if rc != OK:
            raise KataError(rc, "kata_paged_create failed")
        self._native = _Native(L.kata_paged_destroy, self.h)
        self._native.planes = self.planes   # the context works on them as long as it lives

    def close(self):
        self.h, self._native = C.c_void_p(), None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _ck(self, rc):
        if rc != OK:
            raise KataError(rc, self.L.kata_paged_last_error(self.h).decode())

    def _s(self):
        return torch._C._cuda_getCurrentRawStream(self.device)   # torch.cuda.current_stream(device).cuda_stream without the object; the context's device, whichever is current

    def check(self):
        self._ck(self.L.kata_paged_check(self.h, self._s()))

    def launches(self) -> int:
        return int(self.L.kata_paged_launch_count(self.h))

    # ---- pages
    def reserve(self, seq: int, n_slots: int):
        self._ck(self.L.kata_paged_reserve(self.h, seq, n_slots, self._s()))

    def trim(self, seq: int, n_slots: int = 0):
        self._ck(self.L.kata_paged_trim(self.h, seq, n_slots))

    def fork(self, src: int, dst: int, n_slots: int):
        self._ck(self.L.kata_paged_fork(self.h, src, dst, n_slots, self._s()))

    def pages(self, seq: int) -> list:
        t = self.L.kata_paged_table(self.h)
        n = self.L.kata_pages_count(t, seq)
        if n < 0:
            raise KataError(2, f"sequence id {seq}")
        buf = (C.c_int32 * max(1, n))()
        self.L.kata_pages_get(t, seq, buf, n)
        return list(buf)[:n]

    def free_pages(self) -> int:
        return self.L.kata_pages_free_count(self.L.kata_paged_table(self.h))

    def plane(self, layer: int, name: str) -> torch.Tensor:
        """A layer's plane as a tensor that aliases it (and keeps the plane's memory as long as it lives, past close() too): k, v [pages][page_size][kv_heads][head_dim], scales [pages][page_size][kv_heads], weight and age [pages][kv_heads][page_size]."""
        P, S, H, D = self.n_pages, self.page_size, self.kv_heads, self.head_dim
        kv = name in ("k", "v")
        shape = (P, S, H, D) if kv else (P, S, H) if name.endswith("scale") else (P, H, S)
        if name in self.planes:
            return self.planes[name].view(self.n_layers, *shape)[layer]
        ptr = self.L.kata_paged_plane_ptr(self.h, layer, _PLANES.index(name))
        if not ptr:
            raise KataError(3, f"no plane {name!r}")
        kind = ("|i1" if self.kv_mode == "int8" else "<f2") if kv else {"weight": "<f4", "age": "<i4"}.get(name, "<f2")
        return _alias(self._native, ptr, shape, kind, self.cuda)

    # ---- the operators
    def _at(self, what, t, n, kinds):
        """The address of a contiguous tensor of n elements of one of these types on the context's device; raises otherwise."""
        if t.dtype not in kinds or t.numel() != n or t.get_device() != self.device or not t.is_contiguous():
            raise ValueError(f"{what}: a contiguous tensor of {n} elements of {kinds} on device {self.device} is needed, not {list(t.shape)} of {t.dtype} on {t.device}")
        return t.data_ptr()

    def prep(self, layer, seq_ids, slot0, T, q, k, v, qnorm, knorm, axis_pos=None, age0=None, q16=None, gate=None):
        """Norm, rotary positions and append of T tokens per sequence into slots slot0.. (kata_paged_prep). q [n][T][heads][(2) head_dim] or None, k, v [n][T][kv_heads][head_dim], axis_pos int32
        [n][T][3] or None (text: age0 + t on every axis). age0: tokens seen before; slot0 by default, which is right until slots of a sequence are evicted. Returns (q16, None, gate) as AttnContext.prep does."""
        ids, at0, ages, D = _ints(seq_ids), _ints(slot0), None if age0 is None else _ints(age0), self.head_dim
        n = len(ids)
        if len(at0) != n or (ages is not None and len(ages) != n):
            raise ValueError("one slot0 (and age0) per sequence")
        act, nq, nk = (k.dtype,) if k.dtype in _ACT else tuple(_ACT), n * T * self.heads * D, n * T * self.kv_heads * D
        kp, vp = self._at("k", k, nk, act), self._at("v", v, nk, act)
        qp = gp = hp = None
        if q is not None:
            qp = self._at("q", q, nq * (2 if self.gated else 1), act)
            q16 = torch.empty(n, T, self.heads * D, dtype=torch.float16, device=k.device) if q16 is None else q16   # (sizes one by one: a microsecond less than as a tuple)
            gate = torch.empty(n, T, self.heads * D, dtype=torch.float32, device=k.device) if gate is None and self.gated else gate
            hp = self._at("q16", q16, nq, _F16)
        if gate is not None:
            gp = self._at("gate", gate, nq, _F32)
        rc = self.L.kata_paged_prep(self.h, layer, n, ids.buffer_info()[0], at0.buffer_info()[0], T, None if axis_pos is None else self._at("axis_pos", axis_pos, n * T * 3, _I32), None if ages is None else ages.buffer_info()[0],
                                    qp, kp, vp, _ACT[k.dtype], None if qnorm is None else self._at("qnorm", qnorm, D, _F32), self._at("knorm", knorm, D, _F32), hp, gp, self._s())
        if rc:
            self._ck(rc)
        return q16, None, gate

    def decode(self, layer, seq_ids, n_slots, T, q16, gate=None, out=None, out_dtype=torch.float32, accumulate=False):
        """Attention of the T newest tokens of each sequence over its n_slots slots (kata_paged_decode)."""
        ids, held = _ints(seq_ids), _ints(n_slots)
        n = len(ids)
        if len(held) != n:
            raise ValueError("one n_slots per sequence")
        nq = n * T * self.heads * self.head_dim
        qp = self._at("q16", q16, nq, _F16)
        out = torch.empty(n, T, self.heads * self.head_dim, dtype=out_dtype, device=q16.device) if out is None else out
        rc = self.L.kata_paged_decode(self.h, layer, n, ids.buffer_info()[0], held.buffer_info()[0], T, qp, None if gate is None else self._at("gate", gate, nq, _F32), self._at("out", out, nq, _ACT), _ACT[out.dtype], 1 if accumulate else 0, self._s())
        if rc:
            self._ck(rc)
        return out

    def evict(self, layer, seq_ids, n_slots, keep, seen, sink=0, recent=0, n_layers=1, src=None):
        """Cuts the sequences to at most ``keep`` slots per KV head by accumulated weight (kata_paged_evict). ``seen``: tokens each sequence has seen (one number, or one per sequence).
        Returns src [n][kv_heads][keep] ([n_layers] of it for more than one layer): the slot each slot's content came from."""
        ids, held = _ints(seq_ids), _ints(n_slots)
        n = len(ids)
        total = _ints([seen] * n if isinstance(seen, int) else seen)
        if len(held) != n or len(total) != n:
            raise ValueError("one n_slots (and seen) per sequence")
        shape = (n, self.kv_heads, keep) if n_layers == 1 else (n_layers, n, self.kv_heads, keep)
        src = torch.empty(*shape, dtype=torch.int32, device=self.cuda) if src is None else src
        rc = self.L.kata_paged_evict(self.h, layer, n_layers, n, ids.buffer_info()[0], held.buffer_info()[0], total.buffer_info()[0], keep, sink, recent, self._at("src", src, n_layers * n * self.kv_heads * keep, _I32), self._s())
        if rc:
            self._ck(rc)
        return src

    def import_rows(self, layer, seq, slot0, n_rows, src: AttnContext, src_layer, src_seq, src_pos, age0=None):
        """Copies n_rows rows of a contiguous context into slots slot0.. (kata_paged_import). age0: the first row's age; slot0 by default, which is right until slots of the sequence are evicted."""
        self._ck(self.L.kata_paged_import(self.h, layer, seq, slot0, n_rows, slot0 if age0 is None else age0, src.h, src_layer, src_seq, src_pos, self._s()))
