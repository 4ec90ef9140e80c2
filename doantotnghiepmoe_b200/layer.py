"""Device MoE layer: router -> softmax -> top-k -> permutation -> INT8
SwiGLU experts -> slot-ordered combine, behind the C ABI's ``moe_handle``.

It replaces the MoE block of the reference's ``OlmoeModel::step_inner``
(src/olmoe.rs:2583-3158) and ``OlmoeModel::prefill`` (:3417-3714).  Tensors are
passed as CUDA tensors (torch provides device memory and streams only); every
computation happens in libmoe_b200.so.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from functools import cached_property

import numpy as np

from ._lib import (MOE_DT_BF16, MOE_DT_F16, MOE_DT_F32, MOE_ERR_INVALID, MOE_OK, MOE_ROUTER_BF16,
                   MOE_ROUTER_F32, MoeBlockNormDesc, MoeDims, MoeError, MoeGroupedDesc, lib,
                   ptr_array)


@dataclass
class MoeConfig:
    hidden: int
    intermediate: int
    num_experts: int
    top_k: int
    norm_topk_prob: bool
    max_tokens: int = 1
    num_layers: int = 1


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


_DTYPES: dict = {}


def _dt(t) -> int:
    """MOE_DT_* of a floating-point tensor."""
    if not _DTYPES:
        import torch
        _DTYPES.update({torch.float32: MOE_DT_F32, torch.float16: MOE_DT_F16,
                        torch.bfloat16: MOE_DT_BF16})
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise MoeError(MOE_ERR_INVALID, f"tensor type {t.dtype} is none of f32, f16 and bf16")
    return code


def mxfp4_strides(k: int) -> tuple:
    """Bytes of codes and of scales of an MXFP4 row of k values
    (moe_mxfp4_code_stride, moe_mxfp4_scale_stride)."""
    return (k + 31) // 32 * 16, (k + 127) // 128 * 4


def _stream(stream) -> int | None:
    if stream is None:
        return None
    return getattr(stream, "cuda_stream", stream)


def _op_stream(stream) -> int | None:
    """The stream argument of an operator call: None is the handle's stream, a
    torch stream that stream itself -- torch's default stream has the handle 0,
    which the C ABI takes for the handle's stream, so it is named by
    cudaStreamLegacy."""
    if stream is None:
        return None
    return getattr(stream, "cuda_stream", stream) or 1


class MoeLayerEngine:
    def __init__(self, cfg: MoeConfig, device: int = 0):
        self.cfg = cfg
        self.device = device
        dims = MoeDims(cfg.hidden, cfg.intermediate, cfg.num_experts, cfg.top_k,
                       int(cfg.norm_topk_prob), cfg.max_tokens, cfg.num_layers)
        out = ctypes.c_void_p()
        st = lib().moe_create(device, ctypes.byref(dims), ctypes.byref(out))
        if st != MOE_OK:
            raise MoeError(st, "moe_create failed")
        self._h = out.value
        self._keep = {}

    def close(self):
        if getattr(self, "_h", None):
            lib().moe_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def _check(self, st: int):
        if st != MOE_OK:
            msg = lib().moe_last_error(self._h)
            raise MoeError(st, msg.decode() if msg else "")

    # -- configuration ---------------------------------------------------
    def set_stream(self, stream):
        self._check(lib().moe_set_stream(self._h, _stream(stream)))

    def set_route_mode(self, mode: int):
        self._check(lib().moe_set_route_mode(self._h, mode))

    def set_path(self, path: int):
        self._check(lib().moe_set_path(self._h, path))

    def set_layer_packed(self, layer: int, experts, scales, router):
        """experts: CUDA int8 [E, 3*I*H] (or uint8 [E, 3*I*H/2]: INT4 nibble
        pairs); scales: CUDA f32 [E, 2I+H]; router: CUDA f32 [E, H] or
        int16/uint16-viewed bf16 bits [E, H]."""
        import torch
        dtype = MOE_ROUTER_F32 if router.dtype == torch.float32 else MOE_ROUTER_BF16
        quant = 1 if experts.dtype == torch.uint8 else 0
        self._keep[layer] = (experts, scales, router)
        self._check(lib().moe_set_layer_packed_q(self._h, layer, experts.data_ptr(),
                                                 scales.data_ptr(), router.data_ptr(), dtype,
                                                 quant))

    def set_layer(self, layer: int, expert_weights: list, expert_scales: list, router):
        """Per-expert device pointers (pool slots) -- the GpuExpertWeights borrow."""
        import torch
        dtype = MOE_ROUTER_F32 if router.dtype == torch.float32 else MOE_ROUTER_BF16
        self._keep[layer] = (expert_weights, expert_scales, router)
        w = ptr_array([t.data_ptr() for t in expert_weights])
        s = ptr_array([t.data_ptr() for t in expert_scales])
        self._check(lib().moe_set_layer(self._h, layer, w, s, router.data_ptr(), dtype))

    # -- compute -----------------------------------------------------------
    def route(self, layer: int, h, ids, gates, probs=None, stream=None):
        self._check(lib().moe_route(self._h, layer, h.data_ptr(), h.shape[0], ids.data_ptr(),
                                    gates.data_ptr(), _ptr(probs), _stream(stream)))

    def route_permute(self, layer: int, h, ids, gates, seg_off, route_token, route_slot,
                      stream=None):
        self._check(lib().moe_route_permute(self._h, layer, h.data_ptr(), h.shape[0],
                                            ids.data_ptr(), gates.data_ptr(),
                                            seg_off.data_ptr(), route_token.data_ptr(),
                                            route_slot.data_ptr(), _stream(stream)))

    def forward(self, layer: int, h, out, resid=None, ids=None, gates=None, stream=None):
        self._check(lib().moe_layer_forward(self._h, layer, h.data_ptr(), _ptr(resid),
                                            out.data_ptr(), h.shape[0], _ptr(ids), _ptr(gates),
                                            _stream(stream)))

    def stack_forward(self, first_layer: int, n_layers: int, x, eps: float = 1e-5, stream=None):
        self._check(lib().moe_stack_forward(self._h, first_layer, n_layers, x.data_ptr(),
                                            x.shape[0], eps, _stream(stream)))

    def forward_host(self, layer: int, h: np.ndarray, resid: np.ndarray | None = None,
                     out: np.ndarray | None = None, ids: np.ndarray | None = None,
                     gates: np.ndarray | None = None):
        """Host buffers in and out (the library copies them).  Buffers in pinned
        host memory are read and written by DMA directly; pageable ones are
        staged.  `out`, `ids` and `gates` may be passed to reuse buffers."""
        h = np.ascontiguousarray(h, np.float32)
        T = h.shape[0]
        K = self.cfg.top_k
        if out is None:
            out = np.empty_like(h)
        if ids is None:
            ids = np.empty((T, K), np.uint32)
        if gates is None:
            gates = np.empty((T, K), np.float32)
        for a, shape, dt in ((out, h.shape, np.float32), (ids, (T, K), np.uint32),
                             (gates, (T, K), np.float32)):
            if a.shape != shape or a.dtype != dt or not a.flags.c_contiguous:
                raise ValueError(f"output buffer must be C-contiguous {dt.__name__}{shape}")
        r = None if resid is None else np.ascontiguousarray(resid, np.float32)
        self._check(lib().moe_layer_forward_host(self._h, layer, h.ctypes.data,
                                                 None if r is None else r.ctypes.data,
                                                 out.ctypes.data, T, ids.ctypes.data,
                                                 gates.ctypes.data))
        return out, ids, gates

    def set_layer_norm(self, layer: int, norm_w=None):
        """Post-attention RMSNorm gain [H] (device tensor) used by stack_forward;
        None restores the unit gain."""
        self._check(lib().moe_set_layer_norm(self._h, layer, _ptr(norm_w)))

    def load_layer(self, ckpt: "Checkpoint", ckpt_layer: int, layer: int | None = None,
                   keep_bf16: bool = True):
        """moe_load_layer: checkpoint layer -> device copy owned by the engine."""
        self._check(lib().moe_load_layer(self._h, ckpt._c, ckpt_layer,
                                         ckpt_layer if layer is None else layer, int(keep_bf16)))

    def sync_status(self, stream=None):
        self._check(lib().moe_sync_status(self._h, _stream(stream)))

    def last_launch_count(self) -> int:
        return int(lib().moe_last_launch_count(self._h))

    # -- operators on device tensors (rows sorted by expert, norms of a block) --
    @cached_property
    def _dev(self):
        import torch
        return torch.device("cuda", self.device)

    @cached_property
    def _bytes(self):
        import torch
        return torch.empty(0, dtype=torch.uint8, device=self._dev)

    def _bad(self, name, t, want):
        raise MoeError(MOE_ERR_INVALID, f"{name}: {want} on cuda:{self.device} wanted, got "
                       f"{t.dtype} {tuple(t.shape)}, strides {t.stride()}, on {t.device}")

    def _rows(self, name, t, R, width) -> int:
        """Row stride of t [R, width] on this engine's device, the elements of
        a row side by side and its rows apart.  A single row has none: any number
        that torch gives it stands for the same tensor, so it gets one that the
        width alone decides and 16-byte accesses allow."""
        if t.device != self._dev or t.shape != (R, width):
            self._bad(name, t, f"[{R}, {width}]")
        ld, step = t.stride()
        if step != 1 and width > 1:
            self._bad(name, t, "rows of adjacent elements")
        if R <= 1:
            return (width + 7) // 8 * 8
        if ld < width:
            self._bad(name, t, "rows that do not overlap")
        return ld

    def _vec(self, name, t, n, dtype):
        """n contiguous elements of this type on this engine's device; None passes."""
        if t is not None and (t.dtype != dtype or t.device != self._dev or t.numel() != n or
                              not t.is_contiguous()):
            self._bad(name, t, f"{n} contiguous {dtype}")

    def _grouped(self, rows_k, rows_n, w, seg_off, result):
        import torch
        xname, oname = ("x", "out") if result is rows_n else ("dx", "dout")
        if w.dim() != 3 or rows_k.dim() != 2 or w.device != self._dev:
            self._bad("w", w, "[experts, n, k]")
        E, n, k = w.shape
        R = rows_k.shape[0]
        es, ld, step = w.stride()
        if (step != 1 and k > 1) or (ld < k and n > 1):
            self._bad("w", w, "rows of adjacent elements that do not overlap")
        self._vec("seg_off", seg_off, E + 1, torch.int32)
        p, q = (rows_k, rows_n) if result is w else \
            (rows_k, w) if result is rows_n else (rows_n, w)
        if p.dtype != q.dtype:
            raise MoeError(MOE_ERR_INVALID, f"operand types differ: {p.dtype}, {q.dtype}")
        return MoeGroupedDesc(E, R, n, k, _dt(p), _dt(result), self._rows(xname, rows_k, R, k),
                              ld if n > 1 else (k + 7) // 8 * 8, es,
                              self._rows(oname, rows_n, R, n))

    def grouped_mm(self, x, w, seg_off, out, stream=None):
        """out[r] = x[r] @ w[e].T for the rows r of expert e, rows sorted by
        expert.  x [R, k], w [E, n, k], both f16 or both bf16; out [R, n] of that
        type or f32; seg_off int32 [E + 1].  Rows outside every segment stay."""
        d = self._grouped(x, out, w, seg_off, out)
        self._check(lib().moe_grouped_mm(self._h, d, x.data_ptr(), w.data_ptr(),
                                         seg_off.data_ptr(), out.data_ptr(), _op_stream(stream)))

    def grouped_mm_dgrad(self, dout, w, seg_off, dx, stream=None):
        """Gradient of grouped_mm's rows: dx[r] = dout[r] @ w[e]."""
        d = self._grouped(dx, dout, w, seg_off, dx)
        self._check(lib().moe_grouped_mm_dgrad(self._h, d, dout.data_ptr(), w.data_ptr(),
                                               seg_off.data_ptr(), dx.data_ptr(),
                                               _op_stream(stream)))

    def grouped_mm_wgrad(self, dout, x, seg_off, dw, stream=None):
        """Gradient of grouped_mm's experts: dw[e] = dout[rows].T @ x[rows], zeros
        for an expert without rows."""
        d = self._grouped(x, dout, dw, seg_off, dw)
        self._check(lib().moe_grouped_mm_wgrad(self._h, d, dout.data_ptr(), x.data_ptr(),
                                               seg_off.data_ptr(), dw.data_ptr(),
                                               _op_stream(stream)))

    def mxfp4_empty(self, rows: int, k: int):
        """Uninitialised (codes, scales) of `rows` MXFP4 rows of k values."""
        lc, ls = mxfp4_strides(k)
        return self._bytes.new_empty(rows, lc), self._bytes.new_empty(rows, ls)

    def _mxfp4(self, name, codes, scales, rows, k):
        import torch
        for t, ld in zip((codes, scales), mxfp4_strides(k)):
            if (t.dtype != torch.uint8 or t.device != self._dev or t.shape != (rows, ld) or
                    not t.is_contiguous()):
                self._bad(name, t, f"contiguous uint8 [{rows}, {ld}]")

    def mxfp4_quantize(self, x, codes, scales, rows=None, stream=None):
        """x [T, k] (f32, f16 or bf16) to MXFP4 rows (mxfp4_empty); `rows` (int32,
        optional) names the row of x that each output row takes."""
        import torch
        if x.dim() != 2:
            self._bad("x", x, "[T, k]")
        T, k = x.shape
        n = T if rows is None else rows.numel()
        self._vec("rows", rows, n, torch.int32)
        self._mxfp4("MXFP4 rows of x", codes, scales, n, k)
        self._check(lib().moe_mxfp4_quantize(self._h, x.data_ptr(), _dt(x),
                                             self._rows("x", x, T, k), T, _ptr(rows), n, k,
                                             codes.data_ptr(), scales.data_ptr(),
                                             _op_stream(stream)))

    def mxfp4_dequantize(self, codes, scales, out, stream=None):
        """The values of MXFP4 rows, into out [R, k] (f32, f16 or bf16)."""
        if out.dim() != 2:
            self._bad("out", out, "[R, k]")
        R, k = out.shape
        self._mxfp4("MXFP4 rows", codes, scales, R, k)
        self._check(lib().moe_mxfp4_dequantize(self._h, codes.data_ptr(), scales.data_ptr(), R, k,
                                               out.data_ptr(), _dt(out),
                                               self._rows("out", out, R, k), _op_stream(stream)))

    def grouped_mm_mxfp4(self, xcodes, xscales, wcodes, wscales, seg_off, k: int, out,
                         stream=None):
        """grouped_mm of MXFP4 rows: x [R] rows, w [E * n] rows of k values, out
        [R, n] in f32, f16 or bf16."""
        import torch
        if out.dim() != 2:
            self._bad("out", out, "[R, n]")
        (R, n), E = out.shape, seg_off.numel() - 1
        self._vec("seg_off", seg_off, E + 1, torch.int32)
        self._mxfp4("MXFP4 rows of x", xcodes, xscales, R, k)
        self._mxfp4("MXFP4 rows of w", wcodes, wscales, E * n, k)
        self._check(lib().moe_grouped_mm_mxfp4(self._h, E, R, n, k, xcodes.data_ptr(),
                                               xscales.data_ptr(), wcodes.data_ptr(),
                                               wscales.data_ptr(), seg_off.data_ptr(),
                                               out.data_ptr(), _dt(out),
                                               self._rows("out", out, R, n), _op_stream(stream)))

    def _norm_kind(self, T, H, *named):
        """(type, row stride) that the given [T, H] tensors share; None where there
        are none."""
        kind = None
        for name, t in named:
            if t is None:
                continue
            if kind is None:
                kind = t.dtype, self._rows(name, t, T, H)
                code = _dt(t)
            elif t.dtype != kind[0] or self._rows(name, t, T, H) != kind[1]:
                self._bad(name, t, f"{kind[0]} rows {kind[1]} apart")
        return kind and (code, kind[1])

    def block_norm(self, x, x_out, h, w_pre=None, y=None, w_post=None, gate=None,
                   post_norm: bool = True, residual_scale: float = 1.0, eps: float = 1e-5,
                   stream=None):
        """x_out = residual_scale * x + gate * norm(y) * w_post, h = norm(x_out) *
        w_pre (RMS norms; post_norm=False adds gate * y).  x, x_out [T, H] of one
        type; y, h [T, H] of that type, or of any when x is f32; gains f32 [H],
        gate f32 [T]; x_out or h may be None, x_out may be x and h may be y."""
        import torch
        if x.dim() != 2:
            self._bad("x", x, "[T, H]")
        T, H = x.shape
        f32 = torch.float32
        self._vec("w_pre", w_pre, H, f32)
        self._vec("w_post", w_post, H, f32)
        self._vec("gate", gate, T, f32)
        rd, rld = self._norm_kind(T, H, ("x", x), ("x_out", x_out))
        bd, bld = self._norm_kind(T, H, ("y", y), ("h", h)) or (rd, rld)
        d = MoeBlockNormDesc(T, H, rd, bd, rld, bld, post_norm, residual_scale, eps)
        self._check(lib().moe_block_norm(self._h, d, x.data_ptr(), _ptr(y), _ptr(w_post),
                                         _ptr(gate), _ptr(w_pre), _ptr(x_out), _ptr(h),
                                         _op_stream(stream)))

    def block_norm_backward(self, dx_out, dh, x_out, w_pre, dx, dw_pre=None, y=None, w_post=None,
                            gate=None, dy=None, dw_post=None, dgate=None, post_norm: bool = True,
                            residual_scale: float = 1.0, eps: float = 1e-5, stream=None):
        """Backward pass of block_norm from its x_out and y: dx, dy and, where
        given, the gradients of the gains (f32 [H]) and of the gate (f32 [T]).
        dx_out or dh may be None (zeros); dx may be dx_out and dy may be dh."""
        import torch
        if x_out.dim() != 2:
            self._bad("x_out", x_out, "[T, H]")
        T, H = x_out.shape
        for name, t, n in (("w_pre", w_pre, H), ("w_post", w_post, H), ("dw_pre", dw_pre, H),
                           ("dw_post", dw_post, H), ("gate", gate, T), ("dgate", dgate, T)):
            if t is not None:
                self._vec(name, t, n, torch.float32)
        rd, rld = self._norm_kind(T, H, ("x_out", x_out), ("dx_out", dx_out), ("dx", dx))
        bd, bld = self._norm_kind(T, H, ("dh", dh), ("y", y), ("dy", dy)) or (rd, rld)
        d = MoeBlockNormDesc(T, H, rd, bd, rld, bld, post_norm, residual_scale, eps)
        L = lib()
        need = L.moe_block_norm_backward_workspace(self._h, d.rows, d.hidden)
        s = _op_stream(stream) or L.moe_get_stream(self._h)
        if s == _op_stream(torch.cuda.current_stream(self._dev)):
            ws = self._bytes.new_empty(need)
        else:  # from the pool of the stream that uses it: its reuse is ordered there
            with torch.cuda.stream(torch.cuda.default_stream(self._dev) if s == 1 else
                                   torch.cuda.ExternalStream(s, device=self._dev)):
                ws = self._bytes.new_empty(need)
        self._check(L.moe_block_norm_backward(self._h, d, _ptr(dx_out), _ptr(dh), x_out.data_ptr(),
                                              _ptr(y), _ptr(w_post), _ptr(gate), _ptr(w_pre),
                                              dx.data_ptr(), _ptr(dy), _ptr(dw_post), _ptr(dgate),
                                              _ptr(dw_pre), ws.data_ptr(), need, s))

    def set_wait_limit(self, ns: int = 0):
        """Bound of the device-side waits (grid barriers, expert-parallel flag
        waits) in nanoseconds; 0 restores the defaults."""
        self._check(lib().moe_set_wait_limit(self._h, int(ns)))

    def debug_wait_flag(self, stream=None):
        """Failure-path probe: a bounded wait on a device flag that nothing
        sets; the next sync_status() raises MoeError(MOE_ERR_TIMEOUT)."""
        self._check(lib().moe_debug_wait_flag(self._h, _stream(stream)))

    # -- expert parallelism (one process per GPU) -------------------------
    def ep_init(self, rank: int, nranks: int, unique_id: bytes, owner):
        owner = np.ascontiguousarray(owner, np.int32)
        assert owner.size == self.cfg.num_experts
        uid = (ctypes.c_ubyte * 128).from_buffer_copy(unique_id)
        self._check(lib().moe_ep_init(self._h, rank, nranks, uid, owner.ctypes.data))

    def ep_set_layer(self, layer: int, experts_local, scales_local, router):
        """experts_local / scales_local: this rank's experts packed in ascending
        global id order; router: the full [E, H] router."""
        import torch
        dtype = MOE_ROUTER_F32 if router.dtype == torch.float32 else MOE_ROUTER_BF16
        self._keep[("ep", layer)] = (experts_local, scales_local, router)
        self._check(lib().moe_ep_set_layer(self._h, layer, _ptr(experts_local),
                                           _ptr(scales_local), router.data_ptr(), dtype))

    def ep_forward(self, layer: int, h, out, resid=None, stream=None):
        self._check(lib().moe_ep_layer_forward(self._h, layer, h.data_ptr(), _ptr(resid),
                                               out.data_ptr(), h.shape[0], _stream(stream)))

    def ep_finalize(self):
        self._check(lib().moe_ep_finalize(self._h))

    def ep_transport(self) -> str:
        """'p2p' (kernels write into peer memory), 'nccl' or 'none'."""
        return {1: "p2p", 0: "nccl"}.get(lib().moe_ep_transport(self._h), "none")

    def set_graphs(self, enable: bool):
        """Replay each call's launch sequence as a CUDA graph (default on)."""
        self._check(lib().moe_set_graphs(self._h, int(enable)))

    def profile(self, enable: bool):
        self._check(lib().moe_profile_enable(self._h, int(enable)))

    def profile_read(self) -> dict:
        """{kernel name: (launches, total ms)} since the previous read."""
        from ._lib import MoeKernelTime
        buf = (MoeKernelTime * 64)()
        n = ctypes.c_int()
        self._check(lib().moe_profile_read(self._h, buf, 64, ctypes.byref(n)))
        return {buf[i].name.decode(): (int(buf[i].launches), float(buf[i].total_ms))
                for i in range(min(n.value, 64))}


def synth_normal(seed: int, kind: int, layer: int, n: int, std: float) -> np.ndarray:
    out = np.empty(n, np.float32)
    st = lib().moe_synth_normal_host(seed, kind, layer, n, std, out.ctypes.data)
    if st != MOE_OK:
        raise MoeError(st, "moe_synth_normal_host failed")
    return out


KIND_ROUTER, KIND_HIDDEN = 3, 4


_DT = {0: ("U8", np.uint8), 1: ("I8", np.int8), 2: ("F16", np.float16),
       3: ("BF16", np.uint16), 4: ("F32", np.float32)}


class Checkpoint:
    """A directory of merged-INT8 safetensors shards (moe_ckpt_open); BF16
    payloads come back as their uint16 bit patterns."""

    def __init__(self, directory: str):
        c = ctypes.c_void_p()
        err = ctypes.create_string_buffer(512)
        st = lib().moe_ckpt_open(directory.encode(), ctypes.byref(c), err, len(err))
        if st != MOE_OK:
            raise MoeError(st, err.value.decode(errors="replace"))
        self._c = c.value

    def close(self):
        if getattr(self, "_c", None):
            lib().moe_ckpt_close(self._c)
            self._c = None

    def __del__(self):
        self.close()

    def __len__(self) -> int:
        return int(lib().moe_ckpt_num_tensors(self._c))

    def info(self, name: str):
        dt, nd = ctypes.c_int(), ctypes.c_int()
        shape = (ctypes.c_int64 * 8)()
        nbytes = ctypes.c_size_t()
        st = lib().moe_ckpt_tensor_info(self._c, name.encode(), ctypes.byref(dt), ctypes.byref(nd),
                                        shape, ctypes.byref(nbytes))
        if st != MOE_OK:
            raise MoeError(st, f"missing tensor: {name}")
        return _DT[dt.value][0], tuple(shape[i] for i in range(nd.value)), int(nbytes.value)

    def read(self, name: str) -> np.ndarray:
        dname, shape, nbytes = self.info(name)
        out = np.empty(shape, _DT[[k for k, v in _DT.items() if v[0] == dname][0]][1])
        st = lib().moe_ckpt_read(self._c, name.encode(), out.ctypes.data, nbytes)
        if st != MOE_OK:
            raise MoeError(st, f"read failed: {name}")
        return out


class _HostBlock:
    """Owner of one moe_host_alloc() block; freed when the last array view
    referring to it goes away."""

    def __init__(self, nbytes: int):
        p = ctypes.c_void_p()
        st = lib().moe_host_alloc(nbytes, ctypes.byref(p))
        if st != MOE_OK:
            raise MoeError(st, "moe_host_alloc failed")
        self.ptr = p.value

    def __del__(self):
        if getattr(self, "ptr", None):
            lib().moe_host_free(self.ptr)
            self.ptr = None


def host_empty(shape, dtype=np.float32) -> np.ndarray:
    """Pinned host array for MoeLayerEngine.forward_host (moe_host_alloc):
    allocate once and reuse across calls."""
    dtype = np.dtype(dtype)
    n = int(np.prod(shape)) * dtype.itemsize
    blk = _HostBlock(max(n, 1))
    raw = (ctypes.c_ubyte * max(n, 1)).from_address(blk.ptr)
    raw._moe_block = blk  # keeps the block alive while any view exists
    return np.frombuffer(raw, dtype=dtype, count=int(np.prod(shape))).reshape(shape)


def ep_unique_id() -> bytes:
    buf = (ctypes.c_ubyte * 128)()
    st = lib().moe_ep_unique_id(buf)
    if st != MOE_OK:
        raise MoeError(st, "moe_ep_unique_id failed (NCCL unavailable?)")
    return bytes(buf)


def synth_expert(seed: int, layer: int, expert: int, H: int, I: int, w, s, stream=None):
    st = lib().moe_synth_expert(seed, layer, expert, H, I, w.data_ptr(), s.data_ptr(),
                                _stream(stream))
    if st != MOE_OK:
        raise MoeError(st, "moe_synth_expert failed")
