"""Host-side mirror of the reference's Q4 matmul seam, over the C ABI.

The reference exposes no plugin interface for this path: the seam is a set of methods
on its Metal engine state.  The methods below keep those names, argument meaning and
error behaviour so that call sites (and tests) read like the reference's:

* ``dispatch_matmul_q4`` / ``dispatch_gemm_q4`` / ``dispatch_gemm_q4_at``
  (crates/inference/src/forward/metal_qwen35/inner/dispatch.rs:148-229, 1037-1097)
* ``dispatch_lora_if_active`` (crates/inference/src/forward/metal_qwen35/inner/layers/mod.rs:15-51)
* ``load_lora_adapter`` / ``unload_lora_adapter`` / ``LoraLayerData``
  (crates/inference/src/forward/metal_qwen35.rs:1699-1716, 3806-3986, 4063-4075)
* ``Q4WeightBuf`` (crates/inference/src/forward/metal_qwen35.rs:599-702)

Buffers are torch CUDA tensors (device memory only); ``*_offset`` arguments are byte
offsets into them, as the Metal encoder takes them.  All compute is in the CUDA library;
nothing here falls back to PyTorch or to the CPU.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
import threading
from dataclasses import dataclass, field
from typing import Dict, List, Optional, Tuple

import numpy as np
import torch

from . import _lib
from ._lib import GatherDesc, LinearArgs, LoraDesc, Lq4Error, RotDesc, check
from .attention import KvCache, RopeTable


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _raw_stream(device: int) -> int:
    """The current stream of `device`, whichever device is current (the short way where torch has it)."""
    return torch.cuda.current_stream(device).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


class _ArgumentBuffer(threading.local):
    """Where a thread packs the arguments of an attention call (the library reads them after the GIL is released)."""

    def __init__(self):
        self.buf = C.create_string_buffer(64 * (1 + _lib.MAX_ROPE_PARTS))
        self.at = C.addressof(self.buf)


class Q4WeightBuf:
    """Device-resident Q4 payload of one ``[n, k]`` weight in the reference block layout."""

    def __init__(self, handle: int, n: int, k: int):
        self._handle = handle
        self.n, self.k = n, k
        self.payload_ptr = _lib.lib().lq4_weights_payload(handle)
        self.payload_bytes = n * (k // 32) * 20

    @classmethod
    def from_host_payload(cls, payload: np.ndarray, n: int, k: int) -> "Q4WeightBuf":
        """Validates every block's scale/bias on the host, then copies to the device."""
        p = np.ascontiguousarray(payload, dtype=np.uint8).reshape(-1)
        if p.size != n * (k // 32) * 20:
            raise ValueError(f"payload has {p.size} bytes, expected {n * (k // 32) * 20} for [{n}, {k}]")
        h = C.c_void_p()
        check(_lib.lib().lq4_weights_upload(p.ctypes.data_as(C.c_void_p), n, k, C.byref(h)))
        return cls(h.value, n, k)

    @classmethod
    def from_q4_file(cls, path: str, expected_shape: Optional[Tuple[int, int]] = None) -> "Q4WeightBuf":
        h = C.c_void_p()
        if expected_shape is None:
            check(_lib.lib().lq4_weights_load_q4_file(path.encode(), None, 0, C.byref(h)))
        else:
            shp = (C.c_uint64 * len(expected_shape))(*expected_shape)
            check(_lib.lib().lq4_weights_load_q4_file(path.encode(), shp, len(expected_shape), C.byref(h)))
        L = _lib.lib()
        return cls(h.value, int(L.lq4_weights_rows(h)), int(L.lq4_weights_cols(h)))

    @classmethod
    def from_device_payload(cls, payload: torch.Tensor, n: int, k: int) -> "Q4WeightBuf":
        """Wraps bytes that are already on the device (e.g. produced by ``quantize``); not validated."""
        assert payload.is_cuda and payload.dtype == torch.uint8 and payload.numel() >= n * (k // 32) * 20
        self = cls.__new__(cls)
        self._handle = None
        self._keep = payload
        self.n, self.k = n, k
        self.payload_ptr = payload.data_ptr()
        self.payload_bytes = n * (k // 32) * 20
        return self

    def free(self) -> None:
        if getattr(self, "_handle", None):
            _lib.lib().lq4_weights_free(self._handle)
            self._handle = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


@dataclass
class LoraLayerData:
    """Input data for one LoRA projection: A row-major ``(rank, d_in)``, B row-major ``(d_out, rank)``."""
    layer_idx: int
    module: str
    a: np.ndarray
    b: np.ndarray
    rank: int
    d_in: int
    d_out: int


@dataclass
class _LoraProjection:
    handle: int
    rank: int
    d_in: int
    d_out: int


@dataclass
class _LoraAdapter:
    projections: List[Dict[str, _LoraProjection]]
    scale: float
    max_rank: int = 0


class PreparedGroup:
    """Argument block of one ``lq4_linear_group`` call, reusable while its tensors live."""

    def __init__(self, backend: "CudaQ4Backend", arr, count: int, outs: List[torch.Tensor], keep):
        self._be, self._arr, self._count, self.outs, self._keep = backend, arr, count, outs, keep
        self._fn = _lib.lib().lq4_linear_group

    def __call__(self) -> List[torch.Tensor]:
        check(self._fn(self._be._ctx, self._arr, self._count, _stream()))
        return self.outs


class PreparedStep:
    """Argument blocks of one ``lq4_decode_step`` call, reusable while its tensors live."""

    def __init__(self, backend: "CudaQ4Backend", garr, ngroups: int, desc, keep, host: bool = False):
        self._be, self._garr, self._ngroups, self._desc, self._keep = backend, garr, ngroups, desc, keep
        self._fn = _lib.lib().lq4_decode_step_host if host else _lib.lib().lq4_decode_step

    def __call__(self) -> None:
        check(self._fn(self._be._ctx, C.cast(self._garr, C.c_void_p), self._ngroups,
                       C.byref(self._desc) if self._desc is not None else None, _stream()))


class CudaQ4Backend:
    """One instance per device and owning thread, like the reference's GPU state."""

    def __init__(self, device: int = 0, num_hidden_layers: int = 1,
                 projection_shapes: Optional[Dict[str, Tuple[int, int]]] = None):
        if not torch.cuda.is_available():
            raise RuntimeError("CudaQ4Backend needs a CUDA device; there is no CPU path")
        self.device = device
        torch.cuda.set_device(device)
        h = C.c_void_p()
        check(_lib.lib().lq4_ctx_create(device, C.byref(h)))
        self._ctx = h.value
        self._lib = _lib.lib()
        self._args = _ArgumentBuffer()
        self.num_hidden_layers = num_hidden_layers
        # module name -> (d_in, d_out); None disables the model-shape check of load_lora_adapter
        self.projection_shapes = projection_shapes
        self.lora: Optional[_LoraAdapter] = None

    def close(self) -> None:
        if self._ctx:
            self.unload_lora_adapter()
            _lib.lib().lq4_ctx_destroy(self._ctx)
            self._ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    # ---- bookkeeping ------------------------------------------------------
    @property
    def launch_count(self) -> int:
        return int(_lib.lib().lq4_ctx_launch_count(self._ctx))

    def check_device_status(self) -> None:
        """Synchronises the current stream of this backend's device and raises if a kernel gave up on a bounded wait
        or skipped an index out of range."""
        check(_lib.lib().lq4_ctx_check(self._ctx, _raw_stream(self.device)))

    def set_option(self, option: int, value: int) -> None:
        """Per-context switches of the library (``_lib.OPT_*``)."""
        check(_lib.lib().lq4_ctx_set_option(self._ctx, option, int(value)))

    def reserve(self, m: int, n: int, k: int, rank: int = 0) -> None:
        check(_lib.lib().lq4_ctx_reserve(self._ctx, m, n, k, rank))

    # ---- the seam -----------------------------------------------------------
    def _linear(self, x_ptr: int, x_dtype: int, w_ptr: int, y_ptr: int, m: int, n: int, k: int, ldy: int = 0,
                lora: Optional[LoraDesc] = None, rot: Optional[RotDesc] = None, path: int = _lib.PATH_AUTO,
                host: bool = False, gather: Optional[GatherDesc] = None,
                wait_gather: Optional[GatherDesc] = None) -> None:
        args = LinearArgs(x_ptr, x_dtype, m, n, k, w_ptr, y_ptr, ldy,
                          C.pointer(lora) if lora is not None else None,
                          C.pointer(rot) if rot is not None else None, path,
                          C.pointer(gather) if gather is not None else None,
                          C.pointer(wait_gather) if wait_gather is not None else None)
        fn = _lib.lib().lq4_linear_host if host else _lib.lib().lq4_linear
        check(fn(self._ctx, C.byref(args), _stream()))

    @staticmethod
    def _require_k(name: str, k: int) -> None:
        # the reference asserts here: dispatch.rs:185-188
        if k <= 0 or k % 32 != 0:
            raise ValueError(f"{name} requires K to be non-zero and divisible by 32, got {k}")

    @staticmethod
    def _dtype_of(x: torch.Tensor) -> int:
        if x.dtype == torch.float32:
            return _lib.DTYPE_F32
        if x.dtype == torch.bfloat16:
            return _lib.DTYPE_BF16
        raise TypeError(f"activations must be float32 or bfloat16, got {x.dtype}")

    def dispatch_gemm_q4_at(self, x: torch.Tensor, x_offset: int, qw: Q4WeightBuf, qw_extra_offset: int,
                            y: torch.Tensor, y_offset: int, m: int, n: int, k: int, *,
                            lora: Optional[LoraDesc] = None, rot: Optional[RotDesc] = None,
                            ldy: int = 0, path: int = _lib.PATH_AUTO, gather: Optional[GatherDesc] = None,
                            wait_gather: Optional[GatherDesc] = None) -> None:
        """``y[m, n] = x[m, k] . Wq4[n, k]^T`` (overwrites y); ``qw_extra_offset`` bytes into the payload."""
        if m == 0 or n == 0:
            return
        self._require_k("dispatch_gemm_q4_at", k)
        assert x.is_cuda and y.is_cuda and y.dtype == torch.float32
        self._linear(x.data_ptr() + x_offset, self._dtype_of(x), qw.payload_ptr + qw_extra_offset,
                     y.data_ptr() + y_offset, m, n, k, ldy, lora, rot, path, gather=gather, wait_gather=wait_gather)

    def dispatch_gemm_q4(self, x: torch.Tensor, x_offset: int, qw: Q4WeightBuf, y: torch.Tensor, y_offset: int,
                         m: int, n: int, k: int, **kw) -> None:
        if m == 0 or n == 0:
            return
        self._require_k("dispatch_gemm_q4", k)
        self.dispatch_gemm_q4_at(x, x_offset, qw, 0, y, y_offset, m, n, k, **kw)

    def dispatch_matmul_q4(self, x: torch.Tensor, qw: Q4WeightBuf, y: torch.Tensor, m: int, n: int, k: int, **kw) -> None:
        """Decode-step form (m == 1 in the reference)."""
        self.dispatch_gemm_q4(x, 0, qw, y, 0, m, n, k, **kw)

    # ---- LoRA ------------------------------------------------------------------
    # Which side of a projection the residual-stream rotation was absorbed on
    # (crates/inference/src/quant/quarot/plan.rs:935-941, tests at :1483-1514).
    QUAROT_INPUT_SIDE = ("q_proj", "k_proj", "v_proj", "gate_proj", "up_proj", "in_proj_qkv", "in_proj_z",
                         "in_proj_b", "in_proj_a")
    QUAROT_OUTPUT_SIDE = ("o_proj", "down_proj", "out_proj")

    def _rotate_adapter_layer(self, layer: LoraLayerData, seed: int, hidden_dim: int):
        """Rotation correction of one adapter projection for a QuaRot base, on the device
        (crates/inference/src/quant/quarot/lora.rs:32-58,150-216): input side ``A <- A R^T`` (R applied to
        every row of A), output side ``B <- R B`` (R applied to every column of B).  Modules outside the
        plan are refused, as in the reference."""
        a = np.ascontiguousarray(layer.a, dtype=np.float32).reshape(layer.rank, layer.d_in)
        b = np.ascontiguousarray(layer.b, dtype=np.float32).reshape(layer.d_out, layer.rank)
        if layer.module in self.QUAROT_INPUT_SIDE:
            if layer.d_in != hidden_dim:
                raise Lq4Error(_lib.ERR_SHAPE, f"rotate_adapter_for_quarot: layer {layer.layer_idx} module "
                                               f"'{layer.module}' has d_in={layer.d_in} but hidden_dim={hidden_dim}")
            signs = self.rot_signs(seed, hidden_dim)
            a = self.hadamard_rows(torch.from_numpy(a).cuda(), signs).cpu().numpy()
        elif layer.module in self.QUAROT_OUTPUT_SIDE:
            if layer.d_out != hidden_dim:
                raise Lq4Error(_lib.ERR_SHAPE, f"rotate_adapter_for_quarot: layer {layer.layer_idx} module "
                                               f"'{layer.module}' has d_out={layer.d_out} but hidden_dim={hidden_dim}")
            signs = self.rot_signs(seed, hidden_dim)
            bt = torch.from_numpy(np.ascontiguousarray(b.T)).cuda()          # columns of B as rows
            b = np.ascontiguousarray(self.hadamard_rows(bt, signs).cpu().numpy().T)
        else:
            raise Lq4Error(_lib.ERR_LORA, f"rotate_adapter_for_quarot: layer {layer.layer_idx} targets module "
                                          f"'{layer.module}' which is not in the rotation plan")
        return a, b

    def load_lora_adapter(self, layers: List[LoraLayerData], scale: float, quarot_seed: Optional[int] = None,
                          quarot_hidden_dim: Optional[int] = None) -> None:
        """Copies the adapter to the device after the reference's load-time checks.  With ``quarot_seed`` (and
        the hidden dimension the base was rotated in) the factors are first corrected for the rotated base."""
        if self.lora is not None:
            raise Lq4Error(_lib.ERR_LORA, "LoRA adapter already loaded; call unload_lora_adapter first")
        if len(layers) == 0:
            raise Lq4Error(_lib.ERR_LORA, "load_lora_adapter: layers must not be empty")
        if not math.isfinite(scale):
            raise Lq4Error(_lib.ERR_LORA, f"load_lora_adapter: scale must be finite, got {scale}")
        if quarot_seed is not None:
            if quarot_hidden_dim is None or quarot_hidden_dim <= 0 or quarot_hidden_dim & (quarot_hidden_dim - 1):
                raise Lq4Error(_lib.ERR_ROT, "quarot_hidden_dim must be a power of two")
        projections: List[Dict[str, _LoraProjection]] = [dict() for _ in range(self.num_hidden_layers)]
        max_rank = 0
        try:
            for layer in layers:
                if layer.rank == 0:
                    raise Lq4Error(_lib.ERR_LORA, f"load_lora_adapter: layer {layer.layer_idx} module "
                                                  f"'{layer.module}' has rank=0")
                if layer.d_in == 0 or layer.d_out == 0:
                    raise Lq4Error(_lib.ERR_LORA, f"load_lora_adapter: layer {layer.layer_idx} module "
                                                  f"'{layer.module}' has zero dimension")
                if layer.layer_idx >= self.num_hidden_layers:
                    raise Lq4Error(_lib.ERR_SHAPE, f"load_lora_adapter: layer_idx {layer.layer_idx} >= "
                                                   f"num_hidden_layers {self.num_hidden_layers}")
                if self.projection_shapes is not None:
                    if layer.module not in self.projection_shapes:
                        raise Lq4Error(_lib.ERR_LORA, f"unknown LoRA module '{layer.module}'")
                    exp = self.projection_shapes[layer.module]
                    if (layer.d_in, layer.d_out) != exp:
                        raise Lq4Error(_lib.ERR_SHAPE, f"load_lora_adapter: layer {layer.layer_idx} module "
                                                       f"'{layer.module}' has (d_in={layer.d_in}, d_out={layer.d_out}) "
                                                       f"but model expects (d_in={exp[0]}, d_out={exp[1]})")
                if layer.module in projections[layer.layer_idx]:
                    raise Lq4Error(_lib.ERR_LORA, f"load_lora_adapter: duplicate projection for layer "
                                                  f"{layer.layer_idx} module '{layer.module}'")
                if quarot_seed is not None:
                    if np.asarray(layer.a).size != layer.rank * layer.d_in or np.asarray(layer.b).size != layer.d_out * layer.rank:
                        raise Lq4Error(_lib.ERR_SHAPE, f"load_lora_adapter: layer {layer.layer_idx} module "
                                                       f"'{layer.module}' factor sizes do not match its shape")
                    a, b = self._rotate_adapter_layer(layer, quarot_seed, quarot_hidden_dim)
                    a, b = a.reshape(-1), b.reshape(-1)
                else:
                    a = np.ascontiguousarray(layer.a, dtype=np.float32).reshape(-1)
                    b = np.ascontiguousarray(layer.b, dtype=np.float32).reshape(-1)
                h = C.c_void_p()
                # A/B length, overflow and u32 checks happen in the library
                check(_lib.lib().lq4_lora_upload(a.ctypes.data_as(C.c_void_p), a.size, b.ctypes.data_as(C.c_void_p),
                                                 b.size, layer.rank, layer.d_in, layer.d_out, scale, C.byref(h)))
                projections[layer.layer_idx][layer.module] = _LoraProjection(h.value, layer.rank, layer.d_in, layer.d_out)
                max_rank = max(max_rank, layer.rank)
        except Exception:
            for d in projections:
                for pr in d.values():
                    _lib.lib().lq4_lora_free(pr.handle)
            raise
        self.lora = _LoraAdapter(projections, float(scale), max_rank)

    def load_lora_adapter_file(self, path: str, quarot_seed: Optional[int] = None,
                               quarot_hidden_dim: Optional[int] = None) -> "PeftAdapter":   # noqa: F821
        """Reads a PEFT or MLX ``.safetensors`` adapter (bounded read, the reference's key grammar and refusals,
        ``lattice_b200/lora_safetensors.py``) and loads it with scale ``alpha / rank``."""
        from .lora_safetensors import load_peft_safetensors
        adapter = load_peft_safetensors(path)
        self.load_lora_adapter(adapter.layers, adapter.scale, quarot_seed, quarot_hidden_dim)
        return adapter

    def unload_lora_adapter(self) -> None:
        if self.lora is not None:
            for d in self.lora.projections:
                for pr in d.values():
                    _lib.lib().lq4_lora_free(pr.handle)
            self.lora = None

    def has_lora_adapter(self) -> bool:
        return self.lora is not None

    def get_projection(self, layer_idx: int, module: str) -> Optional[_LoraProjection]:
        if self.lora is None or layer_idx >= len(self.lora.projections):
            return None
        return self.lora.projections[layer_idx].get(module)

    def lora_desc(self, layer_idx: int, module: str, n0: int = 0, n1: Optional[int] = None) -> Optional[LoraDesc]:
        """Descriptor to pass as ``lora=`` so the delta is added inside the matmul launch."""
        pr = self.get_projection(layer_idx, module)
        if pr is None:
            return None
        d = LoraDesc()
        check(_lib.lib().lq4_lora_desc_for_rows(pr.handle, n0, pr.d_out if n1 is None else n1, C.byref(d)))
        return d

    def dispatch_lora_if_active(self, x: torch.Tensor, x_byte_offset: int, y: torch.Tensor, y_byte_offset: int,
                                layer_idx: int, module: str, m: int = 1, ldy: int = 0) -> None:
        """``y[0..d_out] += scale * B (A x)``; no-op without an adapter or a projection for this module."""
        pr = self.get_projection(layer_idx, module)
        if pr is None:
            return
        d = self.lora_desc(layer_idx, module)
        check(_lib.lib().lq4_lora_apply(self._ctx, x.data_ptr() + x_byte_offset, self._dtype_of(x), m, pr.d_in,
                                        y.data_ptr() + y_byte_offset, pr.d_out, ldy, C.byref(d), _stream()))

    # ---- helpers on device tensors ------------------------------------------------
    def dequantize(self, payload: torch.Tensor, n_blocks: int) -> torch.Tensor:
        out = torch.empty(n_blocks * 32, dtype=torch.float32, device=payload.device)
        check(_lib.lib().lq4_dequant_f32(payload.data_ptr(), n_blocks, out.data_ptr(), _stream()))
        return out

    def quantize(self, data: torch.Tensor, symmetric: bool = False) -> torch.Tensor:
        """Flat 32-chunk quantizer on the device; raises if a block was not representable."""
        assert data.is_cuda and data.dtype == torch.float32 and data.is_contiguous()
        n = data.numel()
        out = torch.empty(((n + 31) // 32) * 20, dtype=torch.uint8, device=data.device)
        st = torch.zeros(1, dtype=torch.int32, device=data.device)
        check(_lib.lib().lq4_quantize_f32(data.data_ptr(), n, int(symmetric), out.data_ptr(), st.data_ptr(), _stream()))
        if int(st.item()) != 0:
            raise Lq4Error(_lib.ERR_BAD_BLOCK, "a block had a non-finite value or unrepresentable scale/bias")
        return out

    _QUANT_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float64: _lib.DTYPE_F64}

    def quantize_tensor(self, data: torch.Tensor, symmetric: bool = False, per_row: bool = False) -> torch.Tensor:
        """The reference's other quantizer entry points on the device, chosen by ``data``'s dtype: f32 flat
        (``quantize_f32_to_q4``) or per row (``quantize_tensor_q4_0``), bf16 (``quantize_bf16_to_q4``), f64
        (``quantize_f64_to_q4_mode``; ``symmetric=True`` is ``quantize_f64_to_q4``).  ``data`` is 1-D or 2-D."""
        assert data.is_cuda and data.is_contiguous() and data.dtype in self._QUANT_DTYPES
        rows, cols = (1, data.numel()) if data.dim() == 1 else (data.shape[0], data.shape[1])
        nb = rows * ((cols + 31) // 32) if per_row else (rows * cols + 31) // 32
        out = torch.empty(nb * 20, dtype=torch.uint8, device=data.device)
        st = torch.zeros(1, dtype=torch.int32, device=data.device)
        check(_lib.lib().lq4_quantize_tensor(data.data_ptr(), self._QUANT_DTYPES[data.dtype], rows, cols, int(per_row),
                                             int(symmetric), out.data_ptr(), st.data_ptr(), _stream()))
        if int(st.item()) != 0:
            raise Lq4Error(_lib.ERR_BAD_BLOCK, "a block had a non-finite value or unrepresentable scale/bias")
        return out

    def absorb_rotation(self, w: torch.Tensor, signs: torch.Tensor, side: str = "input") -> torch.Tensor:
        """``absorb_input_rotation{,_f64}`` (``W <- W R^T``) or ``absorb_output_rotation{,_f64}`` (``W <- R W``)
        in place on a 2-D f32 / f64 device tensor (crates/inference/src/quant/quarot/rotation.rs:86-195)."""
        assert w.is_cuda and w.is_contiguous() and w.dim() == 2 and w.dtype in (torch.float32, torch.float64)
        rot = self.rot_desc(signs)
        fn = _lib.lib().lq4_absorb_input_rotation if side == "input" else _lib.lib().lq4_absorb_output_rotation
        check(fn(w.data_ptr(), self._QUANT_DTYPES[w.dtype], w.shape[0], w.shape[1], C.byref(rot), _stream()))
        return w

    def save_q4_file(self, path: str, payload: torch.Tensor, shape) -> None:
        """``save_q4_file`` (q4_weights.rs:623-645) for a device payload of ``prod(shape)`` weights."""
        assert payload.is_cuda and payload.dtype == torch.uint8
        shp = (C.c_uint64 * len(shape))(*shape)
        n = int(np.prod(shape)) if len(shape) else 0
        assert payload.numel() >= ((n + 31) // 32) * 20
        check(_lib.lib().lq4_q4_file_write(str(path).encode(), shp, len(shape), n, payload.data_ptr(), _stream()))

    def rot_signs(self, seed: int, dim: int) -> torch.Tensor:
        s = torch.empty(dim, dtype=torch.float32, device=f"cuda:{self.device}")
        check(_lib.lib().lq4_rot_signs_from_seed(seed & (2 ** 64 - 1), dim, s.data_ptr(), _stream()))
        return s

    def block_rot_signs(self, seed: int, n: int, block: int) -> torch.Tensor:
        """The flat sign buffer of ``BlockHadamard::new(seed, n, block)`` (hadamard.rs:358-414)."""
        s = torch.empty(max(n, 1), dtype=torch.float32, device=f"cuda:{self.device}")
        check(_lib.lib().lq4_block_rot_signs_from_seed(seed & (2 ** 64 - 1), n, block, s.data_ptr(), _stream()))
        return s[:n]

    @staticmethod
    def rot_desc(signs: torch.Tensor, block: Optional[int] = None) -> RotDesc:
        """``block=None``: one rotation over ``len(signs)`` entries; else the block-diagonal rotation with that
        block size (``signs`` still holds one entry per activation column)."""
        assert signs.is_cuda and signs.dtype == torch.float32
        return RotDesc(signs.data_ptr(), signs.numel() if block is None else block)

    def block_hadamard_rows(self, x: torch.Tensor, signs: torch.Tensor, block: int) -> torch.Tensor:
        """``BlockHadamard::apply`` on every row of ``x`` (``[rows, n]``, ``n = len(signs)``)."""
        assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
        out = torch.empty_like(x)
        rot = self.rot_desc(signs, block)
        n = signs.numel()
        check(_lib.lib().lq4_block_hadamard_rows(x.data_ptr(), out.data_ptr(), x.numel() // max(n, 1), n, C.byref(rot), _stream()))
        return out

    def hadamard_rows(self, x: torch.Tensor, signs: torch.Tensor) -> torch.Tensor:
        assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
        out = torch.empty_like(x)
        rot = self.rot_desc(signs)
        check(_lib.lib().lq4_hadamard_rows(x.data_ptr(), out.data_ptr(), x.numel() // signs.numel(), C.byref(rot), _stream()))
        return out

    def cross_head_hadamard_rows(self, x: torch.Tensor, signs: torch.Tensor, head_dim: int) -> torch.Tensor:
        """The R3 "Hadamard heads" rotation of every row of ``x`` (``[rows, num_heads * head_dim]``,
        ``num_heads = len(signs)``): mixes across heads at each within-head channel."""
        assert x.is_cuda and x.dtype == torch.float32 and x.is_contiguous()
        nh = signs.numel()
        out = torch.empty_like(x)
        check(_lib.lib().lq4_cross_head_hadamard_rows(x.data_ptr(), out.data_ptr(), x.numel() // max(nh * head_dim, 1),
                                                      nh, head_dim, signs.data_ptr(), _stream()))
        return out

    def linear(self, x: torch.Tensor, qw: Q4WeightBuf, *, lora: Optional[LoraDesc] = None,
               rot: Optional[RotDesc] = None, path: int = _lib.PATH_AUTO, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Convenience wrapper: ``x`` is ``[m, k]`` on the device, returns ``[m, n]`` f32."""
        m, k = x.shape
        y = out if out is not None else torch.empty((m, qw.n), dtype=torch.float32, device=x.device)
        self.dispatch_gemm_q4(x.contiguous(), 0, qw, y, 0, m, qw.n, k, lora=lora, rot=rot, path=path)
        return y

    # ---- dense MLP block ------------------------------------------------------------------
    def mlp_block(self, x: torch.Tensor, w_gate_up: Q4WeightBuf, w_down: Q4WeightBuf, *,
                  lora_gate: Optional[LoraDesc] = None, lora_up: Optional[LoraDesc] = None,
                  lora_down: Optional[LoraDesc] = None, gate_up: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None, rot_down: Optional[RotDesc] = None) -> torch.Tensor:
        """The FFN half of the reference's ``encode_mlp_block`` for dense layers: merged gate||up projection
        (``w_gate_up`` is ``[2 * inter, hidden]``), ``silu(gate) * up``, ``down_proj``; ``x`` is ``[m, hidden]``."""
        from ._lib import MlpArgs
        x = x.contiguous()
        m, hidden = x.shape
        inter = w_gate_up.n // 2
        self._require_k("mlp_block", hidden)
        self._require_k("mlp_block", inter)
        if w_gate_up.k != hidden or w_gate_up.n != 2 * inter or w_down.k != inter or w_down.n != hidden:
            raise ValueError("mlp_block: w_gate_up must be [2 * inter, hidden] and w_down [hidden, inter]")
        y = out if out is not None else torch.empty((m, hidden), dtype=torch.float32, device=x.device)
        args = MlpArgs(x.data_ptr(), self._dtype_of(x), m, hidden, inter, w_gate_up.payload_ptr, w_down.payload_ptr,
                       C.pointer(lora_gate) if lora_gate is not None else None,
                       C.pointer(lora_up) if lora_up is not None else None,
                       C.pointer(lora_down) if lora_down is not None else None,
                       gate_up.data_ptr() if gate_up is not None else None, y.data_ptr(),
                       C.pointer(rot_down) if rot_down is not None else None)
        check(_lib.lib().lq4_mlp_block(self._ctx, C.byref(args), _stream()))
        return y

    # ---- rotary positions and the key/value cache --------------------------------------------
    # One decode step makes these calls once per layer on tiny inputs, so the host side counts: arguments are packed
    # into a buffer of the calling thread (the library reads it before a call returns), checks are single comparisons.
    _ROPE_PART = struct.Struct("@PPiiIiQQQQ")
    _ROPE_ARGS = struct.Struct("@PIIIPP")
    _APPEND_ARGS = struct.Struct("@PPPiIQQQPPPP")
    _TREE_ARGS = struct.Struct("@PPiPPPII9QPPPf")
    _VERIFY_ARGS = struct.Struct("@PPiIII4Q8P")
    _ACT_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}

    def _int32(self, name: str, t: torch.Tensor, shape: tuple) -> int:
        if t.dtype is torch.int32 and t.shape == shape and t.is_contiguous() and t.get_device() == self.device:
            return t.data_ptr()
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {list(shape)} on cuda:{self.device}")

    def rope_rows(self, parts, positions: torch.Tensor, rope: Optional[RopeTable] = None, *,
                  out_dtype: Optional[torch.dtype] = None, outs: Optional[List[torch.Tensor]] = None) -> List[torch.Tensor]:
        """Rotary positions of several tensors in one launch.  ``parts`` is a list of ``(x, turn)`` with ``x``
        ``[rows, heads, head_dim]`` (f32 or bf16, any row and head stride: slices of a fused q|k|v row) and
        ``turn`` 1 (rotate), -1 (the transpose: the backward pass) or 0 (convert only, for v); ``positions``
        is ``[rows]`` int32.  Returns new dense tensors of ``out_dtype`` (default: each input's), or fills
        ``outs`` (which may be the inputs themselves)."""
        n = len(parts)
        if n == 0:
            return []
        if n > _lib.MAX_ROPE_PARTS:
            raise ValueError(f"rope_rows takes at most {_lib.MAX_ROPE_PARTS} tensors, got {n}")
        dev, buf, at, types = self.device, self._args.buf, self._args.at, self._ACT_DTYPES
        rows, _, dim = parts[0][0].shape
        ys = []
        for i, (x, turn) in enumerate(parts):
            if x.dim() != 3 or x.get_device() != dev:
                raise ValueError(f"rope_rows: tensors must be [rows, heads, head_dim] on cuda:{dev}")
            (r, heads, d), (x_row, x_head, x_in) = x.shape, x.stride()
            if r != rows or d != dim:
                raise ValueError("rope_rows: tensors must have equal rows and head_dim")
            if x_in != 1:
                x = x.contiguous()
                x_row, x_head, _ = x.stride()
            if outs is None:
                y = torch.empty_like(x, dtype=out_dtype, memory_format=torch.contiguous_format)
                y_row, y_head = heads * dim, dim
            else:
                y = outs[i]
                if y.shape != x.shape or y.get_device() != dev or y.stride(2) != 1:
                    raise ValueError("rope_rows: an output must have its input's shape and device and unit stride along head_dim")
                y_row, y_head, _ = y.stride()
            ys.append(y)
            if x.dtype not in types or y.dtype not in types:
                raise TypeError(f"rope_rows: types are float32 and bfloat16, got {x.dtype} and {y.dtype}")
            self._ROPE_PART.pack_into(buf, 64 + 64 * i, x.data_ptr(), y.data_ptr(), types[x.dtype], types[y.dtype], heads, turn,
                                      x_row, x_head, y_row, y_head)
        if rope is not None and rope.device != dev:
            raise ValueError(f"rope_rows: the frequencies must lie on cuda:{dev}")
        self._ROPE_ARGS.pack_into(buf, 0, at + 64, n, rows, dim, self._int32("positions", positions, (rows,)),
                                  rope.address if rope is not None else 0)
        status = self._lib.lq4_rope_rows(self._ctx, at, _raw_stream(dev))
        if status:
            check(status)
        return ys

    def _cache_rows(self, what: str, cache: KvCache, k: torch.Tensor, v: torch.Tensor):
        """Checks ``[batch, rows, kv_heads, head_dim]`` rows against a cache; returns (k, v) the kernels can read."""
        dev = self.device
        if cache.device != dev or k.get_device() != dev or v.get_device() != dev:
            raise ValueError(f"{what}: the cache, k and v must lie on cuda:{dev}")
        shape = k.shape
        if len(shape) != 4 or v.shape != shape or (shape[0], shape[2], shape[3]) != cache.rows_shape:
            b, h, d = cache.rows_shape
            raise ValueError(f"{what}: k and v must be [{b}, rows, {h}, {d}], got {list(shape)} and {list(v.shape)}")
        if v.dtype is not k.dtype:
            raise TypeError(f"{what}: k and v must have one type, got {k.dtype} and {v.dtype}")
        stride = k.stride()
        if v.stride() != stride or stride[3] != 1:
            k, v = k.contiguous(), v.contiguous()
        return k, v

    def kv_append(self, cache: KvCache, k: torch.Tensor, v: torch.Tensor, kv_lens: torch.Tensor, *,
                  counts: Optional[torch.Tensor] = None, index: Optional[torch.Tensor] = None,
                  new_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Writes rows of ``k`` and ``v`` (``[batch, rows, kv_heads, head_dim]``, f32 or bf16) behind the
        ``kv_lens[b]`` cached ones: all of them, the first ``counts[b]``, or the rows ``index[b, :counts[b]]``
        (what ``verify_draft`` accepted).  Returns the new lengths (a new int32 tensor, or ``new_lens``)."""
        k, v = self._cache_rows("kv_append", cache, k, v)
        b, rows, _, _ = k.shape
        if k.dtype not in self._ACT_DTYPES:
            raise TypeError(f"kv_append: k and v must be float32 or bfloat16, got {k.dtype}")
        lens_at = self._int32("kv_lens", kv_lens, (b,))
        if new_lens is None:
            new_lens = torch.empty_like(kv_lens)
        s0, s1, s2, _ = k.stride()
        self._APPEND_ARGS.pack_into(self._args.buf, 0, cache.address, k.data_ptr(), v.data_ptr(), self._ACT_DTYPES[k.dtype], rows, s0, s1, s2, lens_at,
                                    0 if counts is None else self._int32("counts", counts, (b,)),
                                    0 if index is None else self._int32("index", index, (b, rows)), self._int32("new_lens", new_lens, (b,)))
        status = self._lib.lq4_kv_append(self._ctx, self._args.at, _raw_stream(self.device))
        if status:
            check(status)
        return new_lens

    def tree_attention(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cache: KvCache, kv_lens: torch.Tensor, *,
                       parents: Optional[torch.Tensor] = None, node_counts: Optional[torch.Tensor] = None,
                       scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of up to 64 drafted tokens per sequence (1: an ordinary decode step) over the ``kv_lens[b]``
        cached rows and the nodes' own rows ``k`` and ``v`` (``[batch, nodes, kv_heads, head_dim]`` bf16, not in
        the cache yet).  ``q`` is ``[batch, nodes, q_heads, head_dim]``, f32 or bf16, and the result has its type;
        ``parents[b, t]`` is the node that ``t`` follows (-1: the cached sequence; None: a chain), ``node_counts``
        how many nodes of a sequence are live (the others' rows of ``out`` are left as they were), ``scale``
        defaults to ``head_dim ** -0.5``."""
        k, v = self._cache_rows("tree_attention", cache, k, v)
        if k.dtype is not torch.bfloat16 or q.dtype not in self._ACT_DTYPES:
            raise TypeError(f"tree_attention: q must be float32 or bfloat16 and the nodes' k and v bfloat16, got {q.dtype} and {k.dtype}")
        b, t, heads, dim = q.shape
        kb, kt, _, kd = k.shape
        if b != kb or t != kt or dim != kd or q.get_device() != self.device:
            raise ValueError(f"tree_attention: q must be [{kb}, {kt}, q_heads, {kd}] on cuda:{self.device}, got {list(q.shape)}")
        q0, q1, q2, q3 = q.stride()
        if q3 != 1:
            q = q.contiguous()
            q0, q1, q2, _ = q.stride()
        if out is None:
            out = torch.empty_like(q)
        elif out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != self.device:
            raise ValueError("tree_attention: out must have q's shape, type and device")
        o0, o1, o2, o3 = out.stride()
        if o3 != 1:
            raise ValueError("tree_attention: out must have unit stride along head_dim")
        k0, k1, k2, _ = k.stride()
        self._TREE_ARGS.pack_into(self._args.buf, 0, q.data_ptr(), out.data_ptr(), self._ACT_DTYPES[q.dtype], k.data_ptr(), v.data_ptr(), cache.address,
                                  t, heads, q0, q1, q2, o0, o1, o2, k0, k1, k2, self._int32("kv_lens", kv_lens, (b,)),
                                  0 if node_counts is None else self._int32("node_counts", node_counts, (b,)),
                                  0 if parents is None else self._int32("parents", parents, (b, t)), dim ** -0.5 if scale is None else scale)
        status = self._lib.lq4_tree_attention(self._ctx, self._args.at, _raw_stream(self.device))
        if status:
            check(status)
        return out

    # ---- lm_head: vocabulary projection + exact top-k --------------------------------------
    @staticmethod
    def _split_candidates(cand: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """``cand`` is ``[top_k, 2]`` int32 holding (logit bits, token id) pairs."""
        return cand[:, 0].view(torch.float32), cand[:, 1]        # strided views: no copy kernels

    def logits_topk(self, logits: torch.Tensor, top_k: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """Top ``top_k`` of a device logit row in the reference's candidate order (higher logit first, ties to
        the lower token id, NaN never ranks).  Returns ``(logits[top_k] f32, token_ids[top_k] int32)``; token
        ids of unused slots are -1 (0xFFFFFFFF) with logit -inf."""
        if logits.dtype != torch.float32 or logits.dim() != 1:
            raise TypeError("logits must be a 1-D float32 device tensor")
        logits = logits.contiguous()
        cand = torch.empty((max(top_k, 1), 2), dtype=torch.int32, device=logits.device)
        check(_lib.lib().lq4_logits_topk(self._ctx, logits.data_ptr(), logits.numel(), top_k, cand.data_ptr(), _stream()))
        return self._split_candidates(cand)

    def lm_head_topk(self, x: torch.Tensor, qw: Q4WeightBuf, top_k: int, *, lora: Optional[LoraDesc] = None,
                     rot: Optional[RotDesc] = None, logits_out: Optional[torch.Tensor] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor]:
        """One token's vocabulary projection followed by the exact top-k (the reference's two-stage lm_head
        path).  ``x`` is ``[1, k]`` or ``[k]``; ``logits_out`` (``[n]`` f32), when given, also receives the
        full logit row, otherwise it stays in the context's workspace."""
        x = x.reshape(1, -1).contiguous()
        k = x.shape[1]
        self._require_k("lm_head_topk", k)
        if k != qw.k:
            raise ValueError(f"x has {k} columns, the weights have {qw.k}")
        cand = torch.empty((max(top_k, 1), 2), dtype=torch.int32, device=x.device)
        args = LinearArgs(x.data_ptr(), self._dtype_of(x), 1, qw.n, k, qw.payload_ptr,
                          logits_out.data_ptr() if logits_out is not None else None, 0,
                          C.pointer(lora) if lora is not None else None,
                          C.pointer(rot) if rot is not None else None, _lib.PATH_AUTO, None, None)
        check(_lib.lib().lq4_lm_head_topk(self._ctx, C.byref(args), top_k, cand.data_ptr(), _stream()))
        return self._split_candidates(cand)

    # ---- verification of drafted tokens -----------------------------------------------------
    def verify_draft(self, target_logits: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor, *,
                     draft_logits: Optional[torch.Tensor] = None, parents: Optional[torch.Tensor] = None,
                     node_counts: Optional[torch.Tensor] = None, temperature: Optional[torch.Tensor] = None
                     ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """Which drafted tokens the target accepts, and the token behind them.  ``target_logits`` (and
        ``draft_logits``; None: certain drafts) are ``[batch, nodes, vocab]``, f32 or bf16: row ``t`` is the
        distribution behind node ``t``, node 0 being the last certain token; ``tokens`` and ``parents`` (None: a
        chain) are ``[batch, nodes]`` int32, ``uniforms`` ``[batch, nodes]`` f32 in [0, 1) (entry 0 draws the last
        token), ``temperature`` ``[batch]`` f32 (0: greedy).  Returns ``(path, path_len, next_token)``: the
        accepted nodes from node 0 on with -1 behind them, their number, the next token; ``path`` and
        ``path_len`` are ``index`` and ``counts`` of ``kv_append``."""
        dev = self.device
        b, t, vocab = target_logits.shape
        if target_logits.dtype not in self._ACT_DTYPES:
            raise TypeError(f"verify_draft: logits must be float32 or bfloat16, got {target_logits.dtype}")
        s0, s1, s2 = target_logits.stride()
        if s2 != 1:
            target_logits = target_logits.contiguous()
            s0, s1, _ = target_logits.stride()
        draft_at, d0, d1, d2 = 0, 0, 0, 1
        if draft_logits is not None:
            if draft_logits.shape != target_logits.shape or draft_logits.dtype is not target_logits.dtype:
                raise ValueError("verify_draft: draft_logits must have target_logits' shape and type")
            d0, d1, d2 = draft_logits.stride()
            if d2 != 1:
                draft_logits = draft_logits.contiguous()
                d0, d1, _ = draft_logits.stride()
            draft_at = draft_logits.data_ptr()
        if target_logits.get_device() != dev or (draft_at and draft_logits.get_device() != dev):
            raise ValueError(f"verify_draft: logits must lie on cuda:{dev}")
        f32 = []
        for name, x, shape in (("uniforms", uniforms, (b, t)), ("temperature", temperature, (b,))):
            if x is None:
                f32.append(0)
            elif x.dtype is torch.float32 and x.shape == shape and x.is_contiguous() and x.get_device() == dev:
                f32.append(x.data_ptr())
            else:
                raise ValueError(f"verify_draft: {name} must be a contiguous float32 tensor of shape {list(shape)} on cuda:{dev}")
        path = torch.empty_like(tokens)
        path_len, token = tokens.new_empty((2, b)).unbind()
        self._VERIFY_ARGS.pack_into(self._args.buf, 0, target_logits.data_ptr(), draft_at, self._ACT_DTYPES[target_logits.dtype], b, t, vocab, s0, s1, d0, d1,
                                    self._int32("tokens", tokens, (b, t)), 0 if parents is None else self._int32("parents", parents, (b, t)),
                                    0 if node_counts is None else self._int32("node_counts", node_counts, (b,)), f32[0], f32[1], path.data_ptr(),
                                    path_len.data_ptr(), token.data_ptr())
        status = self._lib.lq4_verify_draft(self._ctx, self._args.at, _raw_stream(dev))
        if status:
            check(status)
        return path, path_len, token

    def prepare_group(self, problems, outs: Optional[List[torch.Tensor]] = None,
                      gather: Optional[GatherDesc] = None, wait_gather: Optional[GatherDesc] = None) -> "PreparedGroup":
        """Builds the argument block of a grouped call once; calling the result launches it.

        ``problems`` is a list of ``(x, qw)`` or ``(x, qw, lora)`` with ``x`` ``[m, k]`` on the device.  The
        tensors are referenced, not copied: refill ``x`` in place between calls.  No output may alias
        another problem's input."""
        n_prob = len(problems)
        arr = (LinearArgs * max(n_prob, 1))()
        keep, ys = [], []
        for i, pr in enumerate(problems):
            x, qw = pr[0], pr[1]
            lora = pr[2] if len(pr) > 2 else None
            m, k = x.shape
            self._require_k("linear_group", k)
            assert x.is_cuda and x.is_contiguous(), "activations are contiguous [m, k] device tensors"
            y = outs[i] if outs is not None else torch.empty((m, qw.n), dtype=torch.float32, device=x.device)
            assert y.is_cuda and y.dtype == torch.float32
            assert y.shape == (m, qw.n) and y.stride(1) == 1, "outputs are [m, n] with unit column stride"
            keep.append((x, qw, lora))
            ys.append(y)
            ldy = y.stride(0) if m > 1 or y.stride(0) >= qw.n else qw.n      # row pitch of a column slice
            arr[i] = LinearArgs(x.data_ptr(), self._dtype_of(x), m, qw.n, k, qw.payload_ptr, y.data_ptr(), ldy,
                                C.pointer(lora) if lora is not None else None, None, _lib.PATH_AUTO,
                                C.pointer(gather) if gather is not None else None,
                                C.pointer(wait_gather) if wait_gather is not None else None)
        keep += [gather, wait_gather]
        return PreparedGroup(self, arr, n_prob, ys, keep)

    def prepare_step(self, groups, step_buffer=None, gathered=None, host: bool = False) -> "PreparedStep":
        """Builds the argument blocks of one ``lq4_decode_step`` call; calling the result launches it.

        ``groups`` is a list of groups, each a list of ``(x, qw, lora, y)`` with ``x`` ``[1, k]`` or ``[k]`` and
        ``y`` ``[n]`` (or ``[1, n]``) device tensors.  A later group's ``x`` may be a slice of
        ``step_buffer.payload`` where earlier groups' ``y`` slices lie.  ``gathered`` lists the payload slices
        that must be complete on this rank when the launch completes.  ``host=True`` makes the call
        ``lq4_decode_step_host``: inputs and outputs may then be pinned host tensors (``pin_memory=True``); the
        inputs are staged in by a kernel chained in front of the step kernel, the outputs are stored by the step
        kernel itself, and the caller synchronises before it reads them."""
        from ._lib import StepDesc, StepGroup, StepRange
        keep, garr = [], (StepGroup * max(len(groups), 1))()
        for gi, grp in enumerate(groups):
            arr = (LinearArgs * max(len(grp), 1))()
            for i, (x, qw, lora, y) in enumerate(grp):
                k = x.numel()
                self._require_k("decode_step", k)
                assert (x.is_cuda or (host and x.is_pinned())) and (y.is_cuda or (host and y.is_pinned()))
                assert y.dtype == torch.float32 and x.is_contiguous() and y.is_contiguous()
                assert k == qw.k and y.numel() == qw.n
                arr[i] = LinearArgs(x.data_ptr(), self._dtype_of(x), 1, qw.n, k, qw.payload_ptr, y.data_ptr(), 0,
                                    C.pointer(lora) if lora is not None else None, None, _lib.PATH_AUTO, None, None)
                keep.append((x, qw, lora, y))
            keep.append(arr)
            garr[gi] = StepGroup(C.cast(arr, C.c_void_p).value, len(grp))
        desc = None
        if step_buffer is not None:
            rng = (StepRange * max(len(gathered or []), 1))()
            for i, t in enumerate(gathered or []):
                assert t.is_cuda and t.dtype == torch.float32 and t.is_contiguous()
                rng[i] = StepRange(t.data_ptr(), t.numel())
            desc = StepDesc(C.pointer(step_buffer.desc), C.cast(rng, C.c_void_p).value, len(gathered or []))
            keep += [rng, step_buffer, gathered]
        return PreparedStep(self, garr, len(groups), desc, keep, host)

    def gather_wait(self, gather: GatherDesc) -> None:
        """Stream-ordered wait until every peer's results of the gathered launches issued so far are here."""
        check(_lib.lib().lq4_gather_wait(self._ctx, C.byref(gather), _stream()))

    def linear_group(self, problems, outs: Optional[List[torch.Tensor]] = None,
                     gather: Optional[GatherDesc] = None, wait_gather: Optional[GatherDesc] = None) -> List[torch.Tensor]:
        """Several independent projections in one call (one persistent launch for decode shapes);
        returns the list of ``[m, n]`` f32 outputs."""
        if len(problems) == 0:
            return []
        problems = [(pr[0].contiguous(),) + tuple(pr[1:]) for pr in problems]
        return self.prepare_group(problems, outs, gather, wait_gather)()

    def linear_host(self, x: np.ndarray, qw: Q4WeightBuf, y: np.ndarray, *, lora: Optional[LoraDesc] = None,
                    rot: Optional[RotDesc] = None) -> None:
        """End-to-end call with HOST activations and output (copies inside the call, waits for y)."""
        m, k = x.shape
        self._require_k("linear_host", k)
        dt = _lib.DTYPE_F32 if x.dtype == np.float32 else _lib.DTYPE_BF16
        self._linear(x.ctypes.data, dt, qw.payload_ptr, y.ctypes.data, m, qw.n, k, 0, lora, rot, host=True)
