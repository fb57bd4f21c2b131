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
from .xfc import _require, _round_up, _stream

TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # xfc_type


def _rows(t: torch.Tensor, device: torch.device, dims: int, what: str) -> torch.Tensor:
    """A (rows, dims) matrix as the kernels read it: one of TYPES, on `device`, rows that begin on 16 bytes."""
    _require(isinstance(t, torch.Tensor) and t.dim() == 2 and t.shape[1] == dims, f"{what} must be (rows, {dims})")
    _require(t.dtype in TYPES, f"{what} must be float16, bfloat16 or float32", TypeError)
    t = t.detach().to(device)
    whole = t.stride(1) == 1 and t.stride(0) >= dims and t.stride(0) * t.element_size() % 16 == 0 and t.data_ptr() % 16 == 0
    return t if whole else t.clone(memory_format=torch.contiguous_format)


def _check_dims(dims: int) -> None:
    _require(dims > 0 and dims % 8 == 0, "dims must be a multiple of 8")


def mx4_quantize(weight: torch.Tensor):
    """(codes, scales) of a (labels, dims) matrix in float16, bfloat16 or float32, as uint8 tensors of a row per 64 labels."""
    _require(isinstance(weight, torch.Tensor) and weight.dim() == 2, "weight must be (labels, dims)")
    _require(weight.is_cuda, "expected a GPU tensor")
    numy, dims = weight.shape
    _check_dims(dims)
    weight = _rows(weight, weight.device, dims, "weight")
    L, units = lib(), (numy + 63) // 64
    codes = torch.empty(units, L.xfc_mx4_code_bytes(64, dims), dtype=torch.uint8, device=weight.device)
    scales = torch.empty(units, L.xfc_mx4_scale_bytes(64, dims), dtype=torch.uint8, device=weight.device)
    with torch.cuda.device(weight.device):
        rc = L.xfc_mx4_quantize(weight.data_ptr(), TYPES[weight.dtype], weight.stride(0), numy, dims, codes.data_ptr(),
                                scales.data_ptr(), _stream(weight))
    check(rc, "xfc_mx4_quantize")
    return codes, scales


def _check_codes(codes: torch.Tensor, scales: torch.Tensor, numy: int, dims: int) -> None:
    _check_dims(dims)
    _require(numy >= 0, "numy must not be negative")
    L, units = lib(), (numy + 63) // 64
    for t, row, what in ((codes, L.xfc_mx4_code_bytes(64, dims), "codes"), (scales, L.xfc_mx4_scale_bytes(64, dims), "scales")):
        _require(isinstance(t, torch.Tensor) and t.dtype == torch.uint8, f"{what} must be a uint8 tensor", TypeError)
        _require(t.is_cuda, "expected a GPU tensor")
        _require(tuple(t.shape) == (units, row) and t.is_contiguous() and t.data_ptr() % 16 == 0,
                 f"{what} of {numy} labels x {dims} dims must be a contiguous ({units}, {row}) tensor that begins on 16 bytes")
    _require(codes.device == scales.device, "codes and scales must share a device")


def mx4_dequantize(codes: torch.Tensor, scales: torch.Tensor, numy: int, dims: int, dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The (numy, dims) matrix that codes and scales stand for, rounded once to `dtype`."""
    _check_codes(codes, scales, numy, dims)
    _require(dtype in TYPES, "dtype must be float16, bfloat16 or float32", TypeError)
    out = torch.empty(numy, dims, dtype=dtype, device=codes.device)
    with torch.cuda.device(codes.device):
        rc = lib().xfc_mx4_dequantize(codes.data_ptr(), scales.data_ptr(), numy, dims, out.data_ptr(), TYPES[dtype], dims, _stream(out))
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
        bsz = x.shape[0]
        if out is None:
            out = torch.empty(bsz, _round_up(self.numy, 8), dtype=torch.float16, device=self.device)[:, :self.numy]
        _require(out.dtype == torch.float16 and tuple(out.shape) == (bsz, self.numy) and out.device == self.device,
                 "out must be float16 (batch, numy) on the labels' device")
        if out.numel() == 0:
            return out
        _require((out.stride(1) == 1 or self.numy == 1) and (out.stride(0) % 8 == 0 and out.stride(0) >= self.numy or bsz == 1) and
                 out.data_ptr() % 16 == 0, "out must have a row stride that is a multiple of 8 and begin on 16 bytes")
        ldo = out.stride(0) if bsz > 1 else _round_up(self.numy, 8)
        with torch.cuda.device(self.device):
            rc = lib().xfc_mx4_logits(x.data_ptr(), TYPES[x.dtype], x.stride(0), self.codes.data_ptr(), self.scales.data_ptr(),
                                      out.data_ptr(), ldo, bsz, self.numy, self.dims, embed_bits, _stream(x))
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
        need = L.xfc_mx4_topk_workspace_bytes(bsz, self.numy, K)
        if need > 1 << 32 and K > 8:  # the logits of some rows at a time
            need = max(min(need, 1 << 32), L.xfc_mx4_topk_workspace_bytes(min(bsz, 256), self.numy, K))
        ws = torch.empty(need, dtype=torch.uint8, device=self.device)
        with torch.cuda.device(self.device):
            rc = L.xfc_mx4_topk(x.data_ptr(), TYPES[x.dtype], x.stride(0), self.codes.data_ptr(), self.scales.data_ptr(), bsz, self.numy,
                                self.dims, self.numy if numy is None else int(numy), int(K), embed_bits, values.data_ptr(),
                                indices.data_ptr(), ws.data_ptr(), need, _stream(x))
        check(rc, "xfc_mx4_topk")
        return values, indices

    # -- checkpoint payload -----------------------------------------------------------------------------
    def state_dict(self) -> dict:
        return {"codes": self.codes.cpu(), "scales": self.scales.cpu(), "numy": self.numy, "dims": self.dims}

    @classmethod
    def from_state_dict(cls, state: dict, device="cuda:0") -> "MX4Labels":
        return cls(state["codes"].to(device), state["scales"].to(device), state["numy"], state["dims"])
