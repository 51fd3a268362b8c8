"""FP8-128 on torch tensors: e4m3 codes with an fp32 scale for each block of 128.

quantize_rows and quantize_weight encode, product multiplies bf16 rows with an
encoded weight, experts and Fp8RoutedMoE run routed experts held in it
(include/k3_moe.h has the definitions). Codes are float8_e4m3fn (or uint8)
tensors. torch is used only for device memory and streams: everything runs in
libk3moe.so, on the tensors' device and its current stream. Each call takes its
scratch from torch's allocator for itself, so calls on different streams, and
captured graphs, share none.
"""
import ctypes

import torch

from ._lib import K3MoeShape, lib
from .layer import make_shape
from .synth import Config

BLOCK = 128
_CODES = (torch.float8_e4m3fn, torch.uint8)


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _dense(t, name, dtypes, dim, device=None):
    """A contiguous device tensor of one of `dtypes` (and on `device`)."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda, f"{name}: a tensor on the GPU is wanted")
    _need(t.dtype in dtypes, f"{name}: {t.dtype}, wanted {' or '.join(map(str, dtypes))}")
    _need(t.dim() == dim and t.is_contiguous(), f"{name}: a contiguous tensor of {dim} dimensions is wanted")
    _need(device is None or t.device == device, f"{name}: on {t.device}, not {device}")
    return t


class _On:
    """The tensors' device made current for a launch (nothing if it is)."""

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _scratch(n, device):
    """n bytes for one call (None for 0) and its address."""
    if n == 0:
        return None, None
    t = torch.empty(n, dtype=torch.uint8, device=device)
    return t, t.data_ptr()


def _quantize(fn, name, x, block_rows):
    _dense(x, "x", (torch.bfloat16,), 2)
    rows, cols = x.shape
    _need(rows > 0 and cols > 0 and cols % BLOCK == 0, f"{name}: columns in blocks of {BLOCK} are wanted")
    codes = torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty((-(-rows // block_rows), cols // BLOCK), dtype=torch.float32, device=x.device)
    with _On(x.device) as st:
        if not fn(codes.data_ptr(), scales.data_ptr(), x.data_ptr(), rows, cols, st):
            raise RuntimeError(f"{name} rejected its arguments or failed to launch")
    return codes, scales


def quantize_rows(x):
    """bf16 [rows, cols] -> codes [rows, cols], scales [rows, cols / 128]."""
    return _quantize(lib().k3_moe_fp8_128_quantize_rows_bf16, "k3_moe_fp8_128_quantize_rows_bf16", x, 1)


def quantize_weight(w):
    """bf16 [rows, cols] -> codes [rows, cols], scales [ceil(rows / 128), cols / 128]."""
    return _quantize(lib().k3_moe_fp8_128_quantize_weight_bf16,
                     "k3_moe_fp8_128_quantize_weight_bf16", w, BLOCK)


def product(x, codes, scales, out=None):
    """bf16 [T, cols] times an encoded weight [rows, cols] -> bf16 [T, rows]."""
    _dense(x, "x", (torch.bfloat16,), 2)
    _dense(codes, "codes", _CODES, 2, x.device)
    _dense(scales, "scales", (torch.float32,), 2, x.device)
    (T, K), (N, K2) = x.shape, codes.shape
    _need(K == K2 and scales.shape == (-(-N // BLOCK), K // BLOCK),
          f"product of {tuple(x.shape)} with {tuple(codes.shape)}, scales {tuple(scales.shape)}")
    if out is None:
        out = torch.empty((T, N), dtype=torch.bfloat16, device=x.device)
    else:
        _dense(out, "out", (torch.bfloat16,), 2, x.device)
        _need(out.shape == (T, N), f"out: {tuple(out.shape)}, wanted {(T, N)}")
    L = lib()
    n = L.k3_moe_fp8_128_scratch_bytes(T, N, K)
    keep, at = _scratch(n, x.device)
    with _On(x.device) as st:
        if not L.k3_moe_fp8_128_gemm_bf16(out.data_ptr(), codes.data_ptr(), scales.data_ptr(),
                                          x.data_ptr(), T, N, K, at, n, st):
            raise RuntimeError("k3_moe_fp8_128_gemm_bf16 rejected its arguments or failed to launch")
    return out


def shape(hidden, experts, top_k, ffn, scaling_factor, activation, beta=4.0, linear_beta=25.0):
    """The layer's shape as the library takes it (K3MoeShape)."""
    return K3MoeShape(hidden, experts, top_k, ffn, scaling_factor, activation, beta, linear_beta)


def _rows(t, name, T, H, like):
    if t is not None:
        _dense(t, name, (torch.bfloat16,), 2, like.device)
        _need(t.shape == (T, H), f"{name}: {tuple(t.shape)}, wanted {(T, H)}")
    return None if t is None else t.data_ptr()


def _workspace(shape, T, device):
    n = lib().k3_moe_fp8_workspace_bytes(ctypes.byref(shape), T)
    _need(n != 0, "unsupported shape or token count")
    keep, at = _scratch(n, device)
    return keep, at, n


def experts(hidden, ids, weights, table, shape, residual=None, out=None):
    """The expert stage on given routes: bf16 [T, H] -> bf16 [T, H].

    ids (int32) and weights (float32): [T, top_k]; table: int64 [E, 6] device
    tensor of the experts' addresses (Fp8ExpertStore.table)."""
    _dense(hidden, "hidden", (torch.bfloat16,), 2)
    T, H = hidden.shape
    _need(H == shape.hidden, f"hidden: {H} wide, the shape {shape.hidden}")
    for t, name, dtype in ((ids, "ids", torch.int32), (weights, "weights", torch.float32)):
        _dense(t, name, (dtype,), 2, hidden.device)
        _need(t.shape == (T, shape.top_k), f"{name}: {tuple(t.shape)}, wanted {(T, shape.top_k)}")
    _dense(table, "table", (torch.int64,), 2, hidden.device)
    _need(table.shape == (shape.expert_count, 6), "table: [experts, 6] is wanted")
    res = _rows(residual, "residual", T, H, hidden)
    if out is None:
        out = torch.empty_like(hidden)
    to = _rows(out, "out", T, H, hidden)
    keep, at, n = _workspace(shape, T, hidden.device)
    with _On(hidden.device) as st:
        if not lib().k3_moe_fp8_experts_bf16(to, hidden.data_ptr(), res, ids.data_ptr(),
                                             weights.data_ptr(), table.data_ptr(),
                                             ctypes.byref(shape), T, at, n, st):
            raise RuntimeError("k3_moe_fp8_experts_bf16 rejected its arguments or failed to launch")
    return out


class Fp8ExpertStore:
    """All experts of one layer in FP8-128, and the device table of them.

    gate, up: (codes [E, F, H], scales [E, F / 128, H / 128]); down: (codes
    [E, H, F], scales [E, H / 128, F / 128])."""

    def __init__(self, gate, down, up):
        E, F, H = gate[0].shape
        for (codes, scales), name, rows, cols in ((gate, "gate", F, H), (down, "down", H, F),
                                                  (up, "up", F, H)):
            _dense(codes, name, _CODES, 3, gate[0].device)
            _dense(scales, name + " scales", (torch.float32,), 3, gate[0].device)
            _need(rows % BLOCK == 0 and cols % BLOCK == 0 and codes.shape == (E, rows, cols)
                  and scales.shape == (E, rows // BLOCK, cols // BLOCK),
                  f"{name}: codes {tuple(codes.shape)}, scales {tuple(scales.shape)}")
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
        _need((store.experts, store.hidden, store.ffn) == (cfg.experts, cfg.hidden, cfg.ffn),
              "the store's sizes are not the configuration's")
        self.router_weight = _dense(router_weight, "router_weight", (torch.bfloat16,), 2)
        self.router_bias = _dense(router_bias, "router_bias", (torch.float32,), 1)

    def forward(self, hidden, residual=None, out=None, ids=None, weights=None):
        """ids, weights: optional [T, top_k] tensors that receive the routes."""
        _dense(hidden, "hidden", (torch.bfloat16,), 2, self.router_weight.device)
        T, H = hidden.shape
        _need(H == self.shape.hidden, f"hidden: {H} wide, the shape {self.shape.hidden}")
        res = _rows(residual, "residual", T, H, hidden)
        if out is None:
            out = torch.empty_like(hidden)
        to = _rows(out, "out", T, H, hidden)
        for t in (ids, weights):
            _need(t is None or t.shape == (T, self.shape.top_k) and t.element_size() == 4
                  and t.is_contiguous(), "ids, weights: contiguous [T, top_k] of 32 bits are wanted")
        keep, at, n = _workspace(self.shape, T, hidden.device)
        with _On(hidden.device) as st:
            if not lib().k3_moe_fp8_forward_bf16(
                    to, hidden.data_ptr(), res, self.router_weight.data_ptr(),
                    self.router_bias.data_ptr(), self.store.table.data_ptr(),
                    ctypes.byref(self.shape), T, None if ids is None else ids.data_ptr(),
                    None if weights is None else weights.data_ptr(), at, n, st):
                raise RuntimeError("k3_moe_fp8_forward_bf16 rejected its arguments or failed to launch")
        return out

    def experts_only(self, hidden, ids, weights, residual=None, out=None):
        return experts(hidden, ids, weights, self.store.table, self.shape, residual, out)


__all__ = ["quantize_rows", "quantize_weight", "product", "shape", "experts", "Fp8ExpertStore",
           "Fp8RoutedMoE"]
