"""FP8-128 on torch tensors: e4m3 codes with an fp32 scale for each block of 128.

quantize_rows and quantize_weight encode, product multiplies bf16 rows with an
encoded weight, experts and Fp8RoutedMoE run routed experts held in it
(include/k3_moe.h has the definitions). Codes are float8_e4m3fn (or uint8)
tensors. torch is used only for device memory and streams: everything runs in
libk3moe.so, on the tensors' device and its current stream. Each call takes its
scratch from torch's allocator for itself, so calls on different streams, and
captured graphs, share none. Autograd sees none of them: an input that requires a
gradient is refused while gradients are recorded (quantizers give codes, which
have none, and take any).
"""
import ctypes

import torch

from ._lib import K3MoeShape, lib
from .layer import make_shape
from .synth import Config

BLOCK = 128
_CODES = (torch.float8_e4m3fn, torch.uint8)
_BF16, _F32, _I32, _I64, _U8 = (torch.bfloat16,), (torch.float32,), (torch.int32,), (torch.int64,), (torch.uint8,)


def _layout(t, name, dtypes, dim, device=None):
    """The address of a contiguous tensor of one of `dtypes` on GPU `device` (any, if None)."""
    if (isinstance(t, torch.Tensor) and t.dtype in dtypes and t.dim() == dim and t.is_contiguous()
            and t.is_cuda and (device is None or t.get_device() == device)):
        return t.data_ptr()
    raise ValueError(
        f"{name}: a contiguous tensor of {dim} dimensions and {' or '.join(map(str, dtypes))} on GPU "
        f"{'' if device is None else device} is wanted"
        + (f", not {t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else ""))


def _no_gradient(t, name):
    """Refuses a tensor whose gradient autograd would be asked for: it would be missing in silence."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, and autograd gets none through this call: pass "
                         f"{name}.detach(), or call it under torch.no_grad() or in an autograd.Function")


def _dense(t, name, dtypes, dim, device=None):
    """_layout of a call's input that no gradient is wanted for; written out for the usual tensor, as
    a call has up to nine of them."""
    if (isinstance(t, torch.Tensor) and t.dtype in dtypes and t.dim() == dim and t.is_contiguous()
            and t.is_cuda and (device is None or t.get_device() == device) and not t.requires_grad):
        return t.data_ptr()
    at = _layout(t, name, dtypes, dim, device)
    _no_gradient(t, name)
    return at


def _public_stream(device):
    return torch.cuda.current_stream(device).cuda_stream


# a call costs the host several microseconds, so device and stream are asked for directly where torch
# has these names; they are not public, and a build may lack them
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_stream)


def _call(fn, device, *args):
    """fn(*args, stream) on `device`, made current for the call if it is not."""
    if _device() == device:
        ok = fn(*args, _stream(device))
    else:
        with torch.cuda.device(device):
            ok = fn(*args, _stream(device))
    if not ok:
        raise RuntimeError(f"{fn.__name__} rejected its arguments or failed to launch")


def _scratch(like, n):
    """n bytes for one call (None for 0) and their address."""
    if n == 0:
        return None, None
    t = like.new_empty((n,), dtype=torch.uint8)
    return t, t.data_ptr()


def _quantize(fn, x, block_rows):
    at = _layout(x, "x", _BF16, 2)  # codes have no gradient, a weight to encode may require one
    rows, cols = x.shape
    if rows == 0 or cols == 0 or cols % BLOCK != 0:
        raise ValueError(f"x: {tuple(x.shape)}, columns in blocks of {BLOCK} are wanted")
    codes = x.new_empty((rows, cols), dtype=torch.float8_e4m3fn)
    scales = x.new_empty((-(-rows // block_rows), cols // BLOCK), dtype=torch.float32)
    _call(fn, x.get_device(), codes.data_ptr(), scales.data_ptr(), at, rows, cols)
    return codes, scales


def quantize_rows(x):
    """bf16 [rows, cols] -> codes [rows, cols], scales [rows, cols / 128]."""
    return _quantize(lib().k3_moe_fp8_128_quantize_rows_bf16, x, 1)


def quantize_weight(w):
    """bf16 [rows, cols] -> codes [rows, cols], scales [ceil(rows / 128), cols / 128]."""
    return _quantize(lib().k3_moe_fp8_128_quantize_weight_bf16, w, BLOCK)


def product(x, codes, scales, out=None):
    """bf16 [T, cols] times an encoded weight [rows, cols] -> bf16 [T, rows]; out, if given, must
    not overlap x."""
    at = _dense(x, "x", _BF16, 2)
    device = x.get_device()
    w, s = _dense(codes, "codes", _CODES, 2, device), _dense(scales, "scales", _F32, 2, device)
    (T, K), (N, K2) = x.shape, codes.shape
    if K != K2 or scales.shape != (-(-N // BLOCK), K // BLOCK):
        raise ValueError(f"product of {tuple(x.shape)} with {tuple(codes.shape)}, scales {tuple(scales.shape)}")
    if out is None:
        out = x.new_empty((T, N))
        to = out.data_ptr()
    else:
        to = _dense(out, "out", _BF16, 2, device)
        if out.shape != (T, N):
            raise ValueError(f"out: {tuple(out.shape)}, wanted {(T, N)}")
    L = lib()
    n = L.k3_moe_fp8_128_scratch_bytes(T, N, K) if T > 1 else 0
    keep, room = _scratch(x, n)
    _call(L.k3_moe_fp8_128_gemm_bf16, device, to, w, s, at, T, N, K, room, n)
    return out


def shape(hidden, experts, top_k, ffn, scaling_factor, activation, beta=4.0, linear_beta=25.0):
    """The layer's shape as the library takes it (K3MoeShape)."""
    return K3MoeShape(hidden, experts, top_k, ffn, scaling_factor, activation, beta, linear_beta)


def _rows(t, name, shape, device):
    """The address of a bf16 tensor of `shape` (None: none)."""
    if t is None:
        return None
    at = _dense(t, name, _BF16, 2, device)
    if t.shape != shape:
        raise ValueError(f"{name}: {tuple(t.shape)}, wanted {tuple(shape)}")
    return at


def _output(out, hidden, device):
    """The output, a new one if None, and its address."""
    if out is None:
        out = hidden.new_empty(hidden.shape)
        return out, out.data_ptr()
    return out, _rows(out, "out", hidden.shape, device)


def _workspace(shape, T, like):
    n = lib().k3_moe_fp8_workspace_bytes(ctypes.byref(shape), T)
    if n == 0:
        raise ValueError("unsupported shape or token count")
    return (*_scratch(like, n), n)


def experts(hidden, ids, weights, table, shape, residual=None, out=None):
    """The expert stage on given routes: bf16 [T, H] -> bf16 [T, H].

    ids (int32) and weights (float32): [T, top_k]; table: int64 [E, 6] device
    tensor of the experts' addresses (Fp8ExpertStore.table; of a table made elsewhere
    only the layout can be checked: codes at multiples of 16 bytes, scales of 4, on
    hidden's device). out may be hidden or residual itself."""
    x = _dense(hidden, "hidden", _BF16, 2)
    T, H = hidden.shape
    device = hidden.get_device()
    if H != shape.hidden:
        raise ValueError(f"hidden: {H} wide, the shape {shape.hidden}")
    i, w = _dense(ids, "ids", _I32, 2, device), _dense(weights, "weights", _F32, 2, device)
    if ids.shape != (T, shape.top_k) or weights.shape != (T, shape.top_k):
        raise ValueError(f"ids {tuple(ids.shape)}, weights {tuple(weights.shape)}, wanted {(T, shape.top_k)}")
    t = _dense(table, "table", _I64, 2, device)
    if table.shape != (shape.expert_count, 6):
        raise ValueError("table: [experts, 6] is wanted")
    res = _rows(residual, "residual", hidden.shape, device)
    out, to = _output(out, hidden, device)
    keep, room, n = _workspace(shape, T, hidden)
    _call(lib().k3_moe_fp8_experts_bf16, device, to, x, res, i, w, t, ctypes.byref(shape), T, room, n)
    return out


class Fp8ExpertStore:
    """All experts of one layer in FP8-128, and the device table of them.

    gate, up: (codes [E, F, H], scales [E, F / 128, H / 128]); down: (codes
    [E, H, F], scales [E, H / 128, F / 128]). Codes start at multiples of 16 bytes: a
    matrix that lies elsewhere in a checkpoint's buffer is to be copied out first."""

    def __init__(self, gate, down, up):
        E, F, H = gate[0].shape
        for (codes, scales), name, rows, cols in ((gate, "gate", F, H), (down, "down", H, F),
                                                  (up, "up", F, H)):
            at = _layout(codes, name, _CODES, 3, gate[0].get_device())
            scales_at = _layout(scales, name + " scales", _F32, 3, gate[0].get_device())
            # the kernels load 16 codes at once; every expert's start as its matrix does
            if at % 16 != 0 or scales_at % 4 != 0:
                raise ValueError(f"{name}: codes at a multiple of 16 bytes and scales of 4 are wanted")
            if (rows % BLOCK != 0 or cols % BLOCK != 0 or codes.shape != (E, rows, cols)
                    or scales.shape != (E, rows // BLOCK, cols // BLOCK)):
                raise ValueError(f"{name}: codes {tuple(codes.shape)}, scales {tuple(scales.shape)}")
        self.experts, self.ffn, self.hidden = E, F, H
        self.gate, self.down, self.up = gate, down, up
        each = torch.arange(E, dtype=torch.int64)
        at = [t.data_ptr() + t.stride(0) * t.element_size() * each
              for pair in (gate, down, up) for t in pair]
        self.table = torch.stack(at, 1).contiguous().to(gate[0].device)

    @classmethod
    def synthetic(cls, experts, hidden, ffn, seed, device="cuda"):
        """N(0, 0.02) weights from a seeded generator, through quantize_weight."""
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def make(rows, cols):
            codes = torch.empty((experts, rows, cols), dtype=torch.float8_e4m3fn, device=device)
            scales = torch.empty((experts, rows // BLOCK, cols // BLOCK), device=device)
            for e in range(experts):
                w = torch.randn((rows, cols), generator=g, device=device) * 0.02
                codes[e], scales[e] = quantize_weight(w.to(torch.bfloat16))
            return codes, scales

        return cls(make(ffn, hidden), make(hidden, ffn), make(ffn, hidden))


class Fp8RoutedMoE:
    """One routed-MoE layer: bf16 router + resident FP8-128 experts."""

    def __init__(self, cfg: Config, router_weight, router_bias, store: Fp8ExpertStore):
        self.cfg, self.shape, self.store = cfg, make_shape(cfg), store
        if (store.experts, store.hidden, store.ffn) != (cfg.experts, cfg.hidden, cfg.ffn):
            raise ValueError("the store's sizes are not the configuration's")
        if store.table.device != router_weight.device:
            raise ValueError(f"the store is on {store.table.device}, router_weight on {router_weight.device}")
        _layout(router_weight, "router_weight", _BF16, 2)
        _layout(router_bias, "router_bias", _F32, 1, router_weight.get_device())
        if router_weight.shape != (cfg.experts, cfg.hidden) or router_bias.shape != (cfg.experts,):
            raise ValueError(f"router_weight {tuple(router_weight.shape)}, router_bias {tuple(router_bias.shape)}")
        self.router_weight, self.router_bias = router_weight, router_bias

    def forward(self, hidden, residual=None, out=None, ids=None, weights=None):
        """ids, weights: optional [T, top_k] tensors that receive the routes."""
        device = self.router_weight.get_device()
        _no_gradient(self.router_weight, "router_weight")
        _no_gradient(self.router_bias, "router_bias")
        x = _dense(hidden, "hidden", _BF16, 2, device)
        T, H = hidden.shape
        if H != self.shape.hidden:
            raise ValueError(f"hidden: {H} wide, the shape {self.shape.hidden}")
        res = _rows(residual, "residual", hidden.shape, device)
        out, to = _output(out, hidden, device)
        copies = []
        for t, name, dtypes in ((ids, "ids", _I32), (weights, "weights", _F32)):
            copies.append(None if t is None else _dense(t, name, dtypes, 2, device))
            if t is not None and t.shape != (T, self.shape.top_k):
                raise ValueError(f"{name}: [T, top_k] is wanted")
        keep, room, n = _workspace(self.shape, T, hidden)
        _call(lib().k3_moe_fp8_forward_bf16, device, to, x, res, self.router_weight.data_ptr(),
              self.router_bias.data_ptr(), self.store.table.data_ptr(), ctypes.byref(self.shape), T,
              *copies, room, n)
        return out

    def experts_only(self, hidden, ids, weights, residual=None, out=None):
        return experts(hidden, ids, weights, self.store.table, self.shape, residual, out)


__all__ = ["quantize_rows", "quantize_weight", "product", "shape", "experts", "Fp8ExpertStore",
           "Fp8RoutedMoE"]
