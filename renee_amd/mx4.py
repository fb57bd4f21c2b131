"""A label matrix in microscaled 4-bit floating point (MX4): a quarter of fp16's bytes, for scoring and as the frozen side of
training on preferences.  No counterpart in the reference, whose classifier is scored with the weights it is trained with
(dl_base.py:736-756).

    labels = layer.quantize_labels()             # an XFCLayer's weights; or MX4Labels.from_weight(weight)
    logits = labels.xfc_forward(embed)           # as XFCLayer.xfc_forward
    values, best = labels.topk(embed, K=5)       # as XFCLayer.topk

The format, the layout and what is exact stand in include/xfc_mi355x.h.  Scratch memory comes from torch's allocator, call by call:
an MX4Labels holds nothing but its codes and scales, and may be used on several streams at once and in several captured graphs.
"""
from __future__ import annotations

import torch

from ._lib import check, lib
from .xfc import _require, g_row_stride

TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # xfc_type


class _On:
    """The device of a call: made current where it is not, with its current stream's handle.  (torch.cuda.device and current_stream take
    some 6 us of host time, as much as the smallest of these kernels.)"""

    _ready = set()  # devices whose kernels' limits have been raised: nothing is left to do inside a captured graph

    def __init__(self, device: torch.device):
        self.index = device.index

    def __enter__(self) -> int:
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        if self.index not in _On._ready:
            check(lib().xfc_init(), "xfc_init")
            _On._ready.add(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *_):
        if self.before != self.index:
            torch.cuda.set_device(self.before)


def _rows(t: torch.Tensor, device: torch.device, dims: int, what: str) -> torch.Tensor:
    """A (rows, dims) matrix as the kernels read it: one of TYPES, on `device`, rows that begin on 16 bytes."""
    if not (isinstance(t, torch.Tensor) and t.dim() == 2 and t.shape[1] == dims):
        raise RuntimeError(f"{what} must be (rows, {dims})")
    if t.dtype not in TYPES:
        raise TypeError(f"{what} must be float16, bfloat16 or float32")
    if t.device != device:
        t = t.detach().to(device)
    ld, one = t.stride()
    if one == 1 and ld >= dims and ld * t.element_size() % 16 == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.detach().clone(memory_format=torch.contiguous_format)


def _check_dims(dims: int) -> None:
    _require(dims > 0 and dims % 8 == 0, "dims must be a multiple of 8")


def _unit_bytes(dims: int):
    """Bytes of codes and of scales of 64 labels (xfc_mx4_code_bytes, xfc_mx4_scale_bytes)."""
    return 1024 * ((dims + 31) // 32), 256 * ((dims + 127) // 128)


def mx4_quantize(weight: torch.Tensor):
    """(codes, scales) of a (labels, dims) matrix in float16, bfloat16 or float32, as uint8 tensors of a row per 64 labels."""
    _require(isinstance(weight, torch.Tensor) and weight.dim() == 2, "weight must be (labels, dims)")
    _require(weight.is_cuda, "expected a GPU tensor")
    numy, dims = weight.shape
    _check_dims(dims)
    weight = _rows(weight, weight.device, dims, "weight")
    units, (code, scale) = (numy + 63) // 64, _unit_bytes(dims)
    codes = torch.empty(units, code, dtype=torch.uint8, device=weight.device)
    scales = torch.empty(units, scale, dtype=torch.uint8, device=weight.device)
    with _On(weight.device) as stream:
        rc = lib().xfc_mx4_quantize(weight.data_ptr(), TYPES[weight.dtype], weight.stride(0), numy, dims, codes.data_ptr(), scales.data_ptr(),
                                    stream)
    check(rc, "xfc_mx4_quantize")
    return codes, scales


def _check_codes(codes: torch.Tensor, scales: torch.Tensor, numy: int, dims: int) -> None:
    _check_dims(dims)
    _require(numy >= 0, "numy must not be negative")
    units = (numy + 63) // 64
    for t, row, what in zip((codes, scales), _unit_bytes(dims), ("codes", "scales")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8:
            raise TypeError(f"{what} must be a uint8 tensor")
        if not t.is_cuda:
            raise RuntimeError("expected a GPU tensor")
        if t.shape != (units, row) or not t.is_contiguous() or t.data_ptr() % 16:
            raise RuntimeError(f"{what} of {numy} labels x {dims} dims must be a contiguous ({units}, {row}) tensor that begins on 16 bytes")
    _require(codes.device == scales.device, "codes and scales must share a device")


def mx4_dequantize(codes: torch.Tensor, scales: torch.Tensor, numy: int, dims: int, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The (numy, dims) matrix that codes and scales stand for, rounded once to `dtype`."""
    _check_codes(codes, scales, numy, dims)
    _require(dtype in TYPES, "dtype must be float16, bfloat16 or float32", TypeError)
    out = torch.empty(numy, dims, dtype=dtype, device=codes.device)
    with _On(codes.device) as stream:
        rc = lib().xfc_mx4_dequantize(codes.data_ptr(), scales.data_ptr(), numy, dims, out.data_ptr(), TYPES[dtype], dims, stream)
    check(rc, "xfc_mx4_dequantize")
    return out


class MX4Labels:
    """`numy` labels of `dims` dims in MX4, as mx4_quantize leaves them, with the scoring operators of XFCLayer.

    Embeddings (float16, bfloat16 or float32) are quantised within the call, in blocks of 32 dims: `embed_bits` 8 (the default; what is
    lost beside the weights' own rounding is small) or 4 (twice the rate of large batches, and exact sums)."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, numy: int, dims: int):
        _check_codes(codes, scales, int(numy), int(dims))
        self.codes, self.scales, self.numy, self.dims, self.device = codes, scales, int(numy), int(dims), codes.device

    @classmethod
    def from_weight(cls, weight: torch.Tensor) -> "MX4Labels":
        return cls(*mx4_quantize(weight), *weight.shape)

    def dequantize(self, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        return mx4_dequantize(self.codes, self.scales, self.numy, self.dims, dtype)

    def xfc_forward(self, embed: torch.Tensor, out: torch.Tensor | None = None, embed_bits: int = 8) -> torch.Tensor:
        """Logits embed . W^T in float16 (dl_base.py:568-573), into `out` if it is given."""
        x = _rows(embed, self.device, self.dims, "embed")
        _require(embed_bits in (4, 8), "embed_bits must be 4 or 8", ValueError)
        bsz, ld = x.shape[0], g_row_stride(self.numy)
        if out is None:
            out = torch.empty(bsz, ld, dtype=torch.float16, device=self.device)
            if ld != self.numy:
                out = out[:, :self.numy]
        else:
            _require(out.dtype == torch.float16 and out.shape == (bsz, self.numy) and out.device == self.device,
                     "out must be float16 (batch, numy) on the labels' device")
            _require(out.numel() == 0 or (out.stride(1) == 1 or self.numy == 1) and (out.stride(0) % 8 == 0 and out.stride(0) >= self.numy or bsz == 1) and
                     out.data_ptr() % 16 == 0, "out must have a row stride that is a multiple of 8 and begin on 16 bytes")
            if bsz > 1:
                ld = out.stride(0)
        if out.numel() == 0:
            return out
        with _On(self.device) as stream:
            rc = lib().xfc_mx4_logits(x.data_ptr(), TYPES[x.dtype], x.stride(0), self.codes.data_ptr(), self.scales.data_ptr(),
                                      out.data_ptr(), ld, bsz, self.numy, self.dims, embed_bits, stream)
        check(rc, "xfc_mx4_logits")
        return out

    def topk(self, embed: torch.Tensor, K: int = 5, numy: int | None = None, embed_bits: int = 8):
        """The K best labels of every row, as XFCLayer.topk: (values fp32, indices int64), ties to the lower label, K <= 8192.
        Up to 8 by fp32 sums, above by the logits in float16."""
        x = _rows(embed, self.device, self.dims, "embed")
        _require(embed_bits in (4, 8), "embed_bits must be 4 or 8", ValueError)
        _require(1 <= K <= 8192 and K <= self.numy, "K must be in 1..min(8192, numy)")
        bsz = x.shape[0]
        values = torch.empty(bsz, K, device=self.device, dtype=torch.float32)
        indices = torch.empty(bsz, K, device=self.device, dtype=torch.int64)
        if bsz == 0:
            return values, indices
        L = lib()
        need = L.xfc_mx4_topk_workspace_bytes(bsz, self.numy, self.dims, K)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        with _On(self.device) as stream:
            rc = L.xfc_mx4_topk(x.data_ptr(), TYPES[x.dtype], x.stride(0), self.codes.data_ptr(), self.scales.data_ptr(), bsz, self.numy,
                                self.dims, self.numy if numy is None else int(numy), int(K), embed_bits, values.data_ptr(),
                                indices.data_ptr(), ws.data_ptr(), need, stream)
        check(rc, "xfc_mx4_topk")
        return values, indices

    # -- checkpoint payload -----------------------------------------------------------------------------
    def state_dict(self) -> dict:
        return {"codes": self.codes.cpu(), "scales": self.scales.cpu(), "numy": self.numy, "dims": self.dims}

    @classmethod
    def from_state_dict(cls, state: dict, device="cuda:0") -> "MX4Labels":
        return cls(state["codes"].to(device), state["scales"].to(device), state["numy"], state["dims"])
