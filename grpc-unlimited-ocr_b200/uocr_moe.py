"""Python binding of the C ABI in include/uocr_moe.h, include/uocr_decoder.h and
include/uocr_int8.h (ctypes over libuocr_moe.so).

This is the host-side mirror tests and bench.py call: torch supplies device
memory and streams; every computation happens in libuocr_moe.so's sm_100a
kernels. There is no fallback: if the library is missing the import of
`lib()` raises.
"""
from __future__ import annotations

import ctypes
import os
import struct
from dataclasses import dataclass

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libuocr_moe.so")

UOCR_OK = 0
STATUS_NAMES = {0: "OK", 1: "INVALID_ARGUMENT", 2: "UNSUPPORTED", 3: "CUDA", 4: "OUT_OF_MEMORY", 5: "DEVICE",
                6: "TIMEOUT", 7: "COMM"}
WEIGHT_BF16, WEIGHT_INT8 = 0, 1
MEMORY_HOST, MEMORY_DEVICE = 0, 1
DTYPE_F32, DTYPE_BF16 = 0, 1
PLAN_NO_GRAPHS = 1
PLAN_EP_STRIDED = 4
PLAN_PRE_NORM = 8
PLAN_INT8_ACTIVATIONS = 16
DECODER_CUDA_CORE_ATTENTION = 1
DECODER_INT8_ACTIVATIONS = 2
EP_HANDLE_BYTES = 256

# Synthetic tensor kinds (one generator stream per tensor per layer).
KIND_ROUTER, KIND_GATE, KIND_UP, KIND_DOWN, KIND_SGATE, KIND_SUP, KIND_SDOWN, KIND_X = 1, 2, 3, 4, 5, 6, 7, 8
# ... and the page decoder's tensors (attention, embedding, head, prompt rows, norm gains).
KIND_WQ, KIND_WK, KIND_WV, KIND_WO, KIND_EMBED, KIND_LM_HEAD, KIND_PROMPT, KIND_NORM = 9, 10, 11, 12, 13, 14, 15, 16

# Every symbol include/uocr_decoder.h declares.
DECODER_EXPORTS = [
    "uocr_decoder_create", "uocr_decoder_destroy", "uocr_decoder_bytes", "uocr_decoder_set_layer",
    "uocr_decoder_set_head", "uocr_decoder_prefill", "uocr_decoder_decode", "uocr_decoder_profile_decode",
    "uocr_decoder_check",
]

# Every symbol include/uocr_int8.h declares.
INT8_EXPORTS = ["uocr_quantize_tokens", "uocr_linear_w8a8", "uocr_grouped_w8a8_workspace", "uocr_grouped_linear_w8a8"]

# Every symbol include/uocr_moe.h declares.
EXPORTS = [
    "uocr_last_error", "uocr_abi_version", "uocr_moe_plan_create", "uocr_moe_plan_destroy", "uocr_moe_plan_bytes",
    "uocr_moe_set_layer", "uocr_moe_set_layer_parts", "uocr_checkpoint_open", "uocr_checkpoint_close",
    "uocr_checkpoint_count", "uocr_checkpoint_tensor", "uocr_moe_load_layer", "uocr_moe_forward", "uocr_moe_router_logits", "uocr_moe_forward_stack", "uocr_moe_check", "uocr_moe_profile_stack",
    "uocr_moe_ep_handle", "uocr_moe_ep_connect", "uocr_moe_ep_connect_local", "uocr_moe_ep_forward_local",
    "uocr_ops_check", "uocr_expert_topk",
    "uocr_expert_ffn_one", "uocr_expert_ffn_one_noalloc", "uocr_expert_ffn_one_q8", "uocr_linear", "uocr_quantize_q8", "uocr_synth_fill", "uocr_synth_stream",
]


class UocrError(RuntimeError):
    def __init__(self, code: int, msg: str):
        super().__init__(f"{STATUS_NAMES.get(code, code)}: {msg}")
        self.code = code


class MoeDesc(ctypes.Structure):
    _fields_ = [("hidden", ctypes.c_int64), ("routed_experts", ctypes.c_int64),
                ("experts_per_token", ctypes.c_int64), ("expert_ffn", ctypes.c_int64),
                ("shared_ffn", ctypes.c_int64), ("layers", ctypes.c_int64), ("max_rows", ctypes.c_int64),
                ("weight_format", ctypes.c_int32), ("renormalize", ctypes.c_int32),
                ("router_bias", ctypes.c_int32), ("device", ctypes.c_int32), ("flags", ctypes.c_int32),
                ("ep_world", ctypes.c_int32), ("ep_rank", ctypes.c_int32), ("rms_norm_eps", ctypes.c_float),
                ("reserved", ctypes.c_int32), ("ep_owner", ctypes.c_void_p)]


class EpHandle(ctypes.Structure):
    _fields_ = [("bytes", ctypes.c_ubyte * EP_HANDLE_BYTES)]


class LayerSrc(ctypes.Structure):
    _fields_ = [("memory", ctypes.c_int32), ("dtype", ctypes.c_int32), ("router", ctypes.c_void_p),
                ("router_bias", ctypes.c_void_p), ("gate", ctypes.c_void_p), ("up", ctypes.c_void_p),
                ("down", ctypes.c_void_p), ("shared_gate", ctypes.c_void_p), ("shared_up", ctypes.c_void_p),
                ("shared_down", ctypes.c_void_p), ("norm", ctypes.c_void_p)]


class LayerParts(ctypes.Structure):
    _fields_ = [("memory", ctypes.c_int32), ("dtype", ctypes.c_int32), ("router", ctypes.c_void_p),
                ("router_bias", ctypes.c_void_p), ("gate", ctypes.POINTER(ctypes.c_void_p)),
                ("up", ctypes.POINTER(ctypes.c_void_p)), ("down", ctypes.POINTER(ctypes.c_void_p)),
                ("shared_gate", ctypes.c_void_p), ("shared_up", ctypes.c_void_p), ("shared_down", ctypes.c_void_p),
                ("norm", ctypes.c_void_p)]


MAX_TENSOR_RANK = 8


class TensorView(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("rank", ctypes.c_int32), ("shape", ctypes.c_int64 * MAX_TENSOR_RANK),
                ("data", ctypes.c_void_p), ("bytes", ctypes.c_int64)]


_lib = None


class DecoderDesc(ctypes.Structure):
    _fields_ = [("hidden", ctypes.c_int64), ("layers", ctypes.c_int64), ("heads", ctypes.c_int64),
                ("kv_heads", ctypes.c_int64), ("head_dim", ctypes.c_int64), ("vocab", ctypes.c_int64),
                ("max_positions", ctypes.c_int64), ("max_prefill", ctypes.c_int64),
                ("routed_experts", ctypes.c_int64), ("experts_per_token", ctypes.c_int64),
                ("expert_ffn", ctypes.c_int64), ("shared_ffn", ctypes.c_int64), ("rope_theta", ctypes.c_float),
                ("rms_norm_eps", ctypes.c_float), ("weight_format", ctypes.c_int32), ("renormalize", ctypes.c_int32),
                ("device", ctypes.c_int32), ("flags", ctypes.c_int32)]


class DecoderLayerSrc(ctypes.Structure):
    _fields_ = [("memory", ctypes.c_int32), ("dtype", ctypes.c_int32)] + [
        (n, ctypes.c_void_p) for n in ("input_norm", "wq", "wk", "wv", "wo", "post_norm", "router", "gate", "up",
                                       "down", "shared_gate", "shared_up", "shared_down")]


class LinearW8A8Args(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "x_scales", "w", "w_scales", "bias", "residual", "y")] + [
        (n, ctypes.c_int64) for n in ("m", "n", "k", "ldx", "ldw", "ldr", "ldy")] + [
        ("y_dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


class GroupedW8A8Args(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("x", "x_scales", "row_index", "offsets", "w", "w_scales", "w_up",
                                               "w_up_scales", "y")] + [
        (n, ctypes.c_int64) for n in ("rows", "x_rows", "groups", "n", "k", "ldx", "ldw", "ldy")] + [
        ("y_dtype", ctypes.c_int32), ("reserved", ctypes.c_int32), ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_int64)]


def _packer(args) -> struct.Struct:
    """The fields of a ctypes structure (pointers, int64, int32) as a struct format; null pointers are 0. A call packs
    its arguments in a third of the time that the structure's constructor takes."""
    code = {ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_int32: "i"}
    packer = struct.Struct("@" + "".join(code[kind] for _, kind in args._fields_))
    assert packer.size == ctypes.sizeof(args)
    return packer


_pack_linear, _pack_grouped = _packer(LinearW8A8Args).pack, _packer(GroupedW8A8Args).pack


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is not built: run grpc-unlimited-ocr_b200/build.py (or __graft_entry__.build())")
        L = ctypes.CDLL(LIB_PATH)
        vp, i64, i32, f32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32, ctypes.c_float
        L.uocr_last_error.restype = ctypes.c_char_p
        L.uocr_moe_plan_create.argtypes = [ctypes.POINTER(MoeDesc), ctypes.POINTER(vp)]
        L.uocr_moe_plan_destroy.argtypes = [vp]
        L.uocr_moe_plan_bytes.argtypes = [vp, ctypes.POINTER(i64), ctypes.POINTER(i64)]
        L.uocr_moe_set_layer.argtypes = [vp, i64, ctypes.POINTER(LayerSrc), vp]
        L.uocr_moe_set_layer_parts.argtypes = [vp, i64, ctypes.POINTER(LayerParts), vp]
        L.uocr_checkpoint_open.argtypes = [ctypes.c_char_p, ctypes.POINTER(vp)]
        L.uocr_checkpoint_close.argtypes = [vp]
        L.uocr_checkpoint_count.argtypes = [vp, ctypes.POINTER(i64)]
        L.uocr_checkpoint_tensor.argtypes = [vp, ctypes.c_char_p, ctypes.POINTER(TensorView)]
        L.uocr_moe_load_layer.argtypes = [vp, vp, i64, i64, vp]
        L.uocr_moe_forward.argtypes = [vp, i64, vp, i64, vp, vp, vp, vp]
        L.uocr_moe_router_logits.argtypes = [vp, i64, vp, i64, vp, vp]
        L.uocr_moe_forward_stack.argtypes = [vp, vp, i64, vp]
        L.uocr_moe_check.argtypes = [vp, vp]
        L.uocr_moe_profile_stack.argtypes = [vp, vp, i64, i32, ctypes.POINTER(f32), vp]
        L.uocr_moe_ep_handle.argtypes = [vp, ctypes.POINTER(EpHandle)]
        L.uocr_moe_ep_connect.argtypes = [vp, ctypes.POINTER(EpHandle)]
        L.uocr_moe_ep_connect_local.argtypes = [ctypes.POINTER(vp), i32]
        L.uocr_moe_ep_forward_local.argtypes = [ctypes.POINTER(vp), i32, i64, ctypes.POINTER(vp), ctypes.POINTER(i64),
                                                ctypes.POINTER(vp), vp]
        L.uocr_ops_check.argtypes = [vp]
        L.uocr_expert_topk.argtypes = [vp, i64, i64, i64, i32, vp, vp, vp]
        L.uocr_expert_ffn_one.argtypes = [vp, i64, i64, vp, vp, vp, vp, vp, i64, vp, vp]
        L.uocr_expert_ffn_one_noalloc.argtypes = [vp, i64, i64, vp, vp, vp, vp, vp, i64, vp, vp]
        L.uocr_expert_ffn_one_q8.argtypes =[vp, i64, i64, vp, vp, vp, vp, vp, vp, vp, vp, i64, vp, vp]
        L.uocr_quantize_q8.argtypes = [vp, i32, i64, i64, i64, vp, vp, vp]
        L.uocr_linear.argtypes = [vp, i64, i64, vp, i64, vp, vp, vp]
        L.uocr_synth_fill.argtypes = [ctypes.c_uint64, ctypes.c_uint64, f32, i64, i64, i32, vp, vp]
        L.uocr_synth_stream.argtypes = [ctypes.c_uint64] * 3
        L.uocr_synth_stream.restype = ctypes.c_uint64
        L.uocr_decoder_create.argtypes = [ctypes.POINTER(DecoderDesc), ctypes.POINTER(vp)]
        L.uocr_decoder_destroy.argtypes = [vp]
        L.uocr_decoder_bytes.argtypes = [vp, ctypes.POINTER(i64), ctypes.POINTER(i64)]
        L.uocr_decoder_set_layer.argtypes = [vp, i64, ctypes.POINTER(DecoderLayerSrc), vp]
        L.uocr_decoder_set_head.argtypes = [vp, i32, i32, vp, vp, vp, vp]
        L.uocr_decoder_prefill.argtypes = [vp, vp, i64, vp, vp, vp]
        L.uocr_decoder_decode.argtypes = [vp, i64, vp, vp, vp]
        L.uocr_decoder_check.argtypes = [vp, vp]
        L.uocr_decoder_profile_decode.argtypes = [vp, i64, ctypes.POINTER(f32), vp]
        L.uocr_quantize_tokens.argtypes = [vp, i32, i64, i64, i64, vp, i64, vp, vp]
        L.uocr_linear_w8a8.argtypes = [vp, vp]  # structures, by reference or packed
        L.uocr_grouped_w8a8_workspace.argtypes = [vp, ctypes.POINTER(i64)]
        L.uocr_grouped_linear_w8a8.argtypes = [vp, vp]
        _lib = L
    return _lib


def _check(rc: int) -> None:
    if rc != UOCR_OK:
        raise UocrError(rc, lib().uocr_last_error().decode())


def _ptr(t) -> int | None:
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


_raw_stream = None


def _stream(stream) -> int | None:
    if stream is None:
        global _raw_stream
        import torch
        if _raw_stream is None:
            # The handle alone, 3 us cheaper than a Stream object, where this torch has it.
            _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
                lambda device: torch.cuda.current_stream(device).cuda_stream)
        return _raw_stream(torch.cuda.current_device())
    return stream if isinstance(stream, int) else stream.cuda_stream


@dataclass
class Dims:
    hidden: int
    experts: int
    top_k: int
    ffn: int
    shared_ffn: int
    layers: int = 1


class Plan:
    """One MoE stack on one device (uocr_moe_plan)."""

    def __init__(self, dims: Dims, max_rows: int, weight_format: int = WEIGHT_BF16, renormalize: bool = True,
                 router_bias: bool = False, device: int = 0, flags: int = 0, ep_world: int = 0, ep_rank: int = 0,
                 rms_norm_eps: float = 1e-6, ep_owner=None):
        """ep_world > 1 makes this plan rank ep_rank of an expert-parallel
        group (one process per GPU); connect it with ep_connect (see ep.py).
        ep_owner (a sequence of experts * ep_world ints, see
        ep.balanced_owner_table) places the experts; None = the built-in map.
        flags | PLAN_PRE_NORM puts the decoder's RMSNorm (epsilon
        rms_norm_eps) in front of every layer."""
        self.dims = dims
        self.max_rows = max_rows
        self.weight_format = weight_format
        self.ep_world, self.ep_rank = ep_world, ep_rank
        self._owner = None if ep_owner is None else (ctypes.c_int32 * len(ep_owner))(*[int(v) for v in ep_owner])
        desc = MoeDesc(dims.hidden, dims.experts, dims.top_k, dims.ffn, dims.shared_ffn, dims.layers, max_rows,
                       weight_format, int(renormalize), int(router_bias), device, flags, ep_world, ep_rank,
                       rms_norm_eps, 0,
                       None if self._owner is None else ctypes.cast(self._owner, ctypes.c_void_p).value)
        self.desc = desc
        h = ctypes.c_void_p()
        _check(lib().uocr_moe_plan_create(ctypes.byref(desc), ctypes.byref(h)))
        self.h = h

    def close(self):
        if getattr(self, "h", None):
            lib().uocr_moe_plan_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def bytes(self):
        w, a = ctypes.c_int64(), ctypes.c_int64()
        _check(lib().uocr_moe_plan_bytes(self.h, ctypes.byref(w), ctypes.byref(a)))
        return w.value, a.value

    def set_layer(self, layer: int, router, gate, up, down, shared_gate=None, shared_up=None, shared_down=None,
                  router_bias=None, memory: int = MEMORY_DEVICE, dtype: int = DTYPE_F32, stream=None, norm=None):
        """Arguments are torch tensors (device memory) or raw addresses;
        norm is the layer's RMSNorm gain (PLAN_PRE_NORM; None = ones)."""
        src = LayerSrc(memory, dtype, _ptr(router), _ptr(router_bias), _ptr(gate), _ptr(up), _ptr(down),
                       _ptr(shared_gate), _ptr(shared_up), _ptr(shared_down), _ptr(norm))
        _check(lib().uocr_moe_set_layer(self.h, layer, ctypes.byref(src), _stream(stream)))

    def set_layer_parts(self, layer: int, router, gate, up, down, shared_gate=None, shared_up=None,
                        shared_down=None, router_bias=None, memory: int = MEMORY_DEVICE, dtype: int = DTYPE_BF16,
                        stream=None, norm=None):
        """One tensor (or raw address) per expert in gate/up/down, as a
        checkpoint holds them; None entries are allowed for experts another
        expert-parallel rank holds."""
        def arr(items):
            return (ctypes.c_void_p * len(items))(*[_ptr(t) for t in items]) if items is not None else None
        g, u, d = arr(gate), arr(up), arr(down)
        src = LayerParts(memory, dtype, _ptr(router), _ptr(router_bias),
                         ctypes.cast(g, ctypes.POINTER(ctypes.c_void_p)) if g is not None else None,
                         ctypes.cast(u, ctypes.POINTER(ctypes.c_void_p)) if u is not None else None,
                         ctypes.cast(d, ctypes.POINTER(ctypes.c_void_p)) if d is not None else None,
                         _ptr(shared_gate), _ptr(shared_up), _ptr(shared_down), _ptr(norm))
        _check(lib().uocr_moe_set_layer_parts(self.h, layer, ctypes.byref(src), _stream(stream)))

    def forward(self, layer: int, x, y, ids=None, weights=None, stream=None, rows: int | None = None):
        rows = x.shape[0] if rows is None else rows
        _check(lib().uocr_moe_forward(self.h, layer, _ptr(x), rows, _ptr(y), _ptr(ids), _ptr(weights),
                                      _stream(stream)))

    def router_logits(self, layer: int, x, logits, stream=None, rows: int | None = None):
        """logits [rows, E] = the layer's router gate on x (+ bias, after the plan's pre-norm)."""
        rows = x.shape[0] if rows is None else rows
        _check(lib().uocr_moe_router_logits(self.h, layer, _ptr(x), rows, _ptr(logits), _stream(stream)))

    def forward_stack(self, h, stream=None, rows: int | None = None):
        rows = h.shape[0] if rows is None else rows
        _check(lib().uocr_moe_forward_stack(self.h, _ptr(h), rows, _stream(stream)))

    DECODE_KERNELS = ("router", "gate_up", "down")
    PREFILL_KERNELS = ("router", "topk", "permute", "gate_up_gemm", "down_gemm", "combine")

    def profile_stack(self, h, iters: int, stream=None, rows: int | None = None):
        """Mean device ms per launch of each kernel of the path, and per stack pass."""
        rows = h.shape[0] if rows is None else rows
        out = (ctypes.c_float * 8)()
        _check(lib().uocr_moe_profile_stack(self.h, _ptr(h), rows, iters, out, _stream(stream)))
        names = self.DECODE_KERNELS if int(out[6]) == 3 else (self.EP_PHASES if self.ep_world > 1
                                                                   else self.PREFILL_KERNELS)
        res = {n: out[i] for i, n in enumerate(names)}
        res["stack"] = out[7]
        return res

    def check(self, stream=None):
        _check(lib().uocr_moe_check(self.h, _stream(stream)))

    # ---- expert parallelism
    EP_PHASES = ("route", "exchange_wait", "pull", "expert_gemms", "shared_and_wait", "combine")

    def ep_handle(self) -> bytes:
        h = EpHandle()
        _check(lib().uocr_moe_ep_handle(self.h, ctypes.byref(h)))
        return bytes(h.bytes)

    def ep_connect(self, handles: list[bytes]):
        arr = (EpHandle * len(handles))()
        for i, b in enumerate(handles):
            if len(b) != EP_HANDLE_BYTES:
                raise ValueError("an EP handle is 256 bytes")
            ctypes.memmove(arr[i].bytes, b, EP_HANDLE_BYTES)
        _check(lib().uocr_moe_ep_connect(self.h, arr))


DTYPE_NAMES = {0: "F32", 1: "BF16", 2: "F16", 3: "I64", 4: "I32", 5: "U8"}


class Checkpoint:
    """A checkpoint opened by the library's own reader (uocr_checkpoint_*):
    a shard index or one .safetensors file, memory-mapped read-only."""

    def __init__(self, path):
        h = ctypes.c_void_p()
        _check(lib().uocr_checkpoint_open(os.fsencode(path), ctypes.byref(h)))
        self.h = h

    def close(self):
        if getattr(self, "h", None):
            lib().uocr_checkpoint_close(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __len__(self):
        n = ctypes.c_int64()
        _check(lib().uocr_checkpoint_count(self.h, ctypes.byref(n)))
        return n.value

    def tensor(self, name: str):
        """(dtype name, shape, address, bytes) of a tensor in the mapping."""
        v = TensorView()
        _check(lib().uocr_checkpoint_tensor(self.h, name.encode(), ctypes.byref(v)))
        return DTYPE_NAMES[v.dtype], tuple(v.shape[:v.rank]), v.data, v.bytes

    def load_layer(self, plan: "Plan", layer: int, plan_layer: int, stream=None):
        _check(lib().uocr_moe_load_layer(plan.h, self.h, layer, plan_layer, _stream(stream)))


def ep_connect_local(plans: list[Plan]):
    """Joins plans on one GPU into a group of virtual expert-parallel ranks."""
    arr = (ctypes.c_void_p * len(plans))(*[p.h for p in plans])
    _check(lib().uocr_moe_ep_connect_local(arr, len(plans)))


def ep_forward_local(plans: list[Plan], layer: int, xs, ys, stream=None, rows=None):
    """One layer over a local group: rank i maps xs[i] [rows_i, H] to ys[i]."""
    n = len(plans)
    rows = [x.shape[0] for x in xs] if rows is None else rows
    parr = (ctypes.c_void_p * n)(*[p.h for p in plans])
    xarr = (ctypes.c_void_p * n)(*[_ptr(x) for x in xs])
    yarr = (ctypes.c_void_p * n)(*[_ptr(y) for y in ys])
    rarr = (ctypes.c_int64 * n)(*rows)
    _check(lib().uocr_moe_ep_forward_local(parr, n, layer, xarr, rarr, yarr, _stream(stream)))


def ops_check(stream=None):
    """Synchronises the stream and raises UocrError (UOCR_ERR_DEVICE) when an
    op-level mirror recorded a bad expert id since the last check."""
    _check(lib().uocr_ops_check(_stream(stream)))


def expert_topk(logits, k: int, renormalize: bool, ids, weights, stream=None):
    rows, experts = logits.shape
    _check(lib().uocr_expert_topk(_ptr(logits), rows, experts, k, int(renormalize), _ptr(ids), _ptr(weights),
                                  _stream(stream)))


def expert_ffn_one(x, hidden, ffn, gate, up, down, ids, weights, k, out, stream=None):
    _check(lib().uocr_expert_ffn_one(_ptr(x), hidden, ffn, _ptr(gate), _ptr(up), _ptr(down), _ptr(ids),
                                     _ptr(weights), k, _ptr(out), _stream(stream)))


def expert_ffn_one_noalloc(x, hidden, ffn, gate, up, down, ids, weights, k, out, stream=None):
    """expert_ffn_one for callers that cannot allocate device memory: its
    scratch is a static device array shared by every call (k <= 8,
    ffn <= 8192); calls that overlap on the GPU race."""
    _check(lib().uocr_expert_ffn_one_noalloc(_ptr(x), hidden, ffn, _ptr(gate), _ptr(up), _ptr(down), _ptr(ids),
                                             _ptr(weights), k, _ptr(out), _stream(stream)))


def expert_ffn_one_q8(x, hidden, ffn, gate_q, gate_s, up_q, up_s, down_q, down_s, ids, weights, k, out,
                      stream=None):
    _check(lib().uocr_expert_ffn_one_q8(_ptr(x), hidden, ffn, _ptr(gate_q), _ptr(gate_s), _ptr(up_q), _ptr(up_s),
                                        _ptr(down_q), _ptr(down_s), _ptr(ids), _ptr(weights), k, _ptr(out),
                                        _stream(stream)))


def quantize_q8(w, q, scales, group: int | None = None, stream=None):
    rows, cols = w.shape
    import torch
    dtype = DTYPE_BF16 if w.dtype == torch.bfloat16 else DTYPE_F32
    _check(lib().uocr_quantize_q8(_ptr(w), dtype, rows, cols, cols if group is None else group, _ptr(q),
                                  _ptr(scales), _stream(stream)))


def synth_stream(layer: int, kind: int, index: int) -> int:
    return lib().uocr_synth_stream(layer, kind, index)


def synth_fill(out, seed: int, layer: int, kind: int, index: int, sigma: float, offset: int = 0, stream=None):
    """Fills a contiguous fp32 or bf16 device tensor from the synthetic stream."""
    import torch
    dtype = DTYPE_BF16 if out.dtype == torch.bfloat16 else DTYPE_F32
    _check(lib().uocr_synth_fill(seed, synth_stream(layer, kind, index), sigma, offset, out.numel(), dtype,
                                 _ptr(out), _stream(stream)))


def linear(x, w_bf16, y, bias=None, stream=None):
    """y[m, n] = bf16(x)[m, k] . w[n, k]^T (+ bias) on the tensor cores (uocr_linear)."""
    m, k = x.shape
    n = w_bf16.shape[0]
    _check(lib().uocr_linear(_ptr(x), m, k, _ptr(w_bf16), n, _ptr(bias), _ptr(y), _stream(stream)))


_FLOAT_DTYPES: dict = {}


def _float_dtype(t, what: str) -> int:
    if not _FLOAT_DTYPES:
        import torch
        _FLOAT_DTYPES.update({torch.float32: DTYPE_F32, torch.bfloat16: DTYPE_BF16})
    dtype = _FLOAT_DTYPES.get(t.dtype)
    if dtype is None:
        raise ValueError(f"{what} must be float32 or bfloat16, not {t.dtype}")
    return dtype


def _pitch(t, what: str, rows: int, cols: int) -> int:
    """The row pitch of a [rows, cols] device tensor whose rows are contiguous."""
    if t.shape != (rows, cols) or not t.is_cuda:
        raise ValueError(f"{what} must be a {(rows, cols)} tensor on the GPU, not {tuple(t.shape)} on {t.device}")
    pitch, step = t.stride()
    if step != 1 and cols > 1:
        raise ValueError(f"{what}'s rows must be contiguous")
    return pitch if rows > 1 else cols


def _pitch_i8(t, what: str, rows: int, cols: int) -> int:
    """The same of int8 rows; a single row's pitch is its width rounded up to 16."""
    import torch
    if t.dtype is not torch.int8:
        raise ValueError(f"{what} must be int8, not {t.dtype}")
    pitch = _pitch(t, what, rows, cols)
    return pitch if rows > 1 else (pitch + 15) // 16 * 16


def _vector(t, what: str, n: int, dtype) -> int:
    if t.dtype is not dtype or t.numel() != n or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{what} must be {n} contiguous {dtype} values on the GPU")
    return t.data_ptr()


def quantize_tokens(x, q, scales, stream=None):
    """q (int8) and scales (fp32) = the rows of x [rows, cols] (fp32 or bf16) quantised with one scale per row
    (uocr_quantize_tokens)."""
    import torch
    rows, cols = x.shape
    _check(lib().uocr_quantize_tokens(x.data_ptr(), _float_dtype(x, "x"), rows, cols, _pitch(x, "x", rows, cols),
                                      q.data_ptr(), _pitch_i8(q, "q", rows, cols),
                                      _vector(scales, "scales", rows, torch.float32), _stream(stream)))


def linear_w8a8(x, x_scales, w, w_scales, y, bias=None, residual=None, stream=None):
    """y[m, n] = x[m, k] . w[n, k]^T in int8 with x_scales per row of x and w_scales per row of w (+ bias[n])
    (+ residual[m, n], of y's dtype; may be y itself) (uocr_linear_w8a8)."""
    import torch
    f32, i8 = torch.float32, torch.int8
    m, k = x.shape
    n = w.shape[0]
    (ldx, sx), (ldw, sw), (ldy, sy) = x.stride(), w.stride(), y.stride()
    # The common case in one expression (this call is microseconds of device time); else what is wrong, or a lone column.
    if not (n > 1 and sx == sw == sy == 1 and w.shape[1] == k and y.shape == (m, n) and x.dtype is i8
            and w.dtype is i8 and x.is_cuda and w.is_cuda and y.is_cuda):
        ldx, ldw, ldy = _pitch_i8(x, "x", m, k), _pitch_i8(w, "w", n, k), _pitch(y, "y", m, n)
    elif m == 1:
        ldx, ldy = (k + 15) // 16 * 16, n
    if not (x_scales.dtype is f32 and w_scales.dtype is f32 and x_scales.numel() == m and w_scales.numel() == n
            and x_scales.is_contiguous() and w_scales.is_contiguous() and x_scales.is_cuda and w_scales.is_cuda):
        _vector(x_scales, "x_scales", m, f32), _vector(w_scales, "w_scales", n, f32)
    ldr = res = 0
    if residual is not None:
        if residual.dtype is not y.dtype:
            raise ValueError("residual must have y's dtype")
        res, ldr = residual.data_ptr(), _pitch(residual, "residual", m, n)
    args = _pack_linear(
        x.data_ptr(), x_scales.data_ptr(), w.data_ptr(), w_scales.data_ptr(),
        0 if bias is None else _vector(bias, "bias", n, f32), res, y.data_ptr(), m, n, k, ldx, ldw, ldr, ldy,
        _float_dtype(y, "y"), 0)
    _check(lib().uocr_linear_w8a8(args, _stream(stream)))


def _stack_pitch(t, what: str, groups: int, n: int, k: int) -> int:
    """The row pitch of int8 matrices [groups, n, k] that follow one another, or of their stack [groups * n, k]."""
    import torch
    if t.dim() != 3:
        return _pitch_i8(t, what, groups * n, k)
    if t.shape != (groups, n, k) or t.dtype is not torch.int8 or not t.is_cuda:
        raise ValueError(f"{what} must be int8 {(groups, n, k)} on the GPU, not {t.dtype} {tuple(t.shape)}")
    of_group, pitch, step = t.stride()
    if step != 1 and k > 1:
        raise ValueError(f"{what}'s rows must be contiguous")
    if n == 1:
        pitch = of_group if groups > 1 else (k + 15) // 16 * 16
    elif groups > 1 and of_group != n * pitch:
        raise ValueError(f"{what}'s groups must follow one another")
    return pitch


def _workspace(size: int, device, stream):
    """`size` bytes from torch's allocator for work on `stream` alone. They come from that stream's own blocks: one that
    the current stream gave back may still be in use by what that stream has queued."""
    import torch
    if stream is None:
        return torch.empty(size, dtype=torch.uint8, device=device)
    with torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device) if isinstance(stream, int) else stream):
        return torch.empty(size, dtype=torch.uint8, device=device)


def grouped_linear_w8a8(x, x_scales, w, w_scales, offsets, y, row_index=None, w_up=None, w_up_scales=None,
                        stream=None):
    """Group g's rows offsets[g] .. offsets[g + 1] - 1 of y [rows, n] = x[row_index[r]] . w[g]^T in int8, or with
    w_up silu(x . w[g]^T) * (x . w_up[g]^T) (uocr_grouped_linear_w8a8). w, w_up: [groups, n, k] or the stack
    [groups * n, k]; w_scales: groups * n values; offsets, row_index: int32. Where the call needs a workspace it
    comes from torch's allocator, from the blocks of the stream that the call runs on."""
    import torch
    f32, i32, i8 = torch.float32, torch.int32, torch.int8
    x_rows, k = x.shape
    rows, n = y.shape
    groups = offsets.numel() - 1
    (ldx, sx), (ldy, sy) = x.stride(), y.stride()
    if not (n > 1 and sx == sy == 1 and x.dtype is i8 and x.is_cuda and y.is_cuda):
        ldx, ldy = _pitch_i8(x, "x", x_rows, k), _pitch(y, "y", rows, n)
    else:
        if x_rows == 1:
            ldx = (k + 15) // 16 * 16
        if rows == 1:
            ldy = n
    ldw = _stack_pitch(w, "w", groups, n, k)
    if not (x_scales.dtype is f32 and w_scales.dtype is f32 and offsets.dtype is i32 and x_scales.numel() == x_rows
            and w_scales.numel() == groups * n and x_scales.is_contiguous() and w_scales.is_contiguous()
            and offsets.is_contiguous() and x_scales.is_cuda and w_scales.is_cuda and offsets.is_cuda):
        _vector(x_scales, "x_scales", x_rows, f32), _vector(w_scales, "w_scales", groups * n, f32)
        _vector(offsets, "offsets", groups + 1, i32)
    up = up_scales = index = 0
    if w_up is not None:
        if _stack_pitch(w_up, "w_up", groups, n, k) != ldw:
            raise ValueError("w_up must have w's pitch")
        up, up_scales = w_up.data_ptr(), _vector(w_up_scales, "w_up_scales", groups * n, f32)
    if row_index is not None:
        index = _vector(row_index, "row_index", rows, i32)
    args = (x.data_ptr(), x_scales.data_ptr(), index, offsets.data_ptr(), w.data_ptr(), w_scales.data_ptr(), up,
            up_scales, y.data_ptr(), rows, x_rows, groups, n, k, ldx, ldw, ldy, _float_dtype(y, "y"), 0)
    space, space_bytes = 0, 0
    if row_index is not None:
        need = ctypes.c_int64()
        _check(lib().uocr_grouped_w8a8_workspace(_pack_grouped(*args, 0, 0), ctypes.byref(need)))
        if need.value > 0:
            workspace = _workspace(need.value, y.device, stream)  # held until the launch is made
            space, space_bytes = workspace.data_ptr(), need.value
    _check(lib().uocr_grouped_linear_w8a8(_pack_grouped(*args, space, space_bytes), _stream(stream)))


class Decoder:
    """The page decoder around the MoE (uocr_decoder): attention layers with a
    bf16 KV cache, the MoE block of every layer, lm_head and greedy tokens."""

    def __init__(self, hidden, layers, heads, kv_heads, vocab, max_positions, max_prefill, experts, top_k, ffn,
                 shared_ffn, weight_format: int = WEIGHT_BF16, renormalize: bool = True, rope_theta: float = 1e4,
                 rms_norm_eps: float = 1e-6, device: int = 0, flags: int = 0):
        self.desc = DecoderDesc(hidden, layers, heads, kv_heads, 128, vocab, max_positions, max_prefill, experts,
                                top_k, ffn, shared_ffn, rope_theta, rms_norm_eps, weight_format, int(renormalize),
                                device, flags)
        h = ctypes.c_void_p()
        _check(lib().uocr_decoder_create(ctypes.byref(self.desc), ctypes.byref(h)))
        self.h = h

    def close(self):
        if getattr(self, "h", None) is not None and self.h.value:
            lib().uocr_decoder_destroy(self.h)
            self.h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def bytes(self):
        w, o = ctypes.c_int64(), ctypes.c_int64()
        _check(lib().uocr_decoder_bytes(self.h, ctypes.byref(w), ctypes.byref(o)))
        return w.value, o.value

    def set_layer(self, layer: int, t: dict, memory: int = MEMORY_DEVICE, dtype: int = DTYPE_BF16, stream=None):
        """t: input_norm, wq, wk, wv, wo, post_norm (fp32 gains), router (fp32)
        and the MoE stacks gate, up, down, shared_gate, shared_up, shared_down."""
        src = DecoderLayerSrc(memory, dtype, *[_ptr(t[n]) for n in (
            "input_norm", "wq", "wk", "wv", "wo", "post_norm", "router", "gate", "up", "down", "shared_gate",
            "shared_up", "shared_down")])
        _check(lib().uocr_decoder_set_layer(self.h, layer, ctypes.byref(src), _stream(stream)))

    def set_head(self, embed, final_norm, lm_head, memory: int = MEMORY_DEVICE, dtype: int = DTYPE_BF16,
                 stream=None):
        _check(lib().uocr_decoder_set_head(self.h, memory, dtype, _ptr(embed), _ptr(final_norm), _ptr(lm_head),
                                           _stream(stream)))

    def prefill(self, embeds, logits=None, token=None, stream=None):
        _check(lib().uocr_decoder_prefill(self.h, _ptr(embeds), embeds.shape[0], _ptr(logits), _ptr(token),
                                          _stream(stream)))

    def decode(self, steps: int, tokens=None, logits=None, stream=None):
        _check(lib().uocr_decoder_decode(self.h, steps, _ptr(tokens), _ptr(logits), _stream(stream)))

    def check(self, stream=None):
        _check(lib().uocr_decoder_check(self.h, _stream(stream)))

    def profile_decode(self, steps: int, stream=None) -> dict:
        """Mean ms per step of each phase (plain launches, events between)."""
        ms = (ctypes.c_float * 5)()
        _check(lib().uocr_decoder_profile_decode(self.h, steps, ms, _stream(stream)))
        return dict(zip(("qkv", "attention", "out_proj", "moe", "lm_head"), [round(v, 5) for v in ms]))
