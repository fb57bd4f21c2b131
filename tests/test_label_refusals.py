"""What MX4 label matrices and the preference loss refuse, on the CPU: nothing here reaches a device."""
import ctypes

import pytest
import torch

from renee_amd import MX4Labels, mx4_dequantize, mx4_quantize, preference
from renee_amd._lib import lib

ONE = ctypes.c_void_p(16)  # never dereferenced: every call below fails validation first
F16, BF16, F32 = 0, 1, 2


def _quantize(W=ONE, type=F16, ldw=64, L=10, d=64, codes=ONE, scales=ONE):
    return lib().xfc_mx4_quantize(W, type, ldw, L, d, codes, scales, None)


@pytest.mark.parametrize("how,code", [
    (dict(W=None), 1), (dict(codes=None), 1), (dict(scales=None), 1), (dict(type=3), 1), (dict(L=-1), 1), (dict(d=0), 1), (dict(L=1 << 31), 1),
    (dict(d=60), 3), (dict(ldw=68), 3), (dict(type=F32, ldw=66), 3), (dict(W=ctypes.c_void_p(24)), 3), (dict(codes=ctypes.c_void_p(8)), 3),
    (dict(ldw=56), 6), (dict(L=0, W=None, codes=None, scales=None), 0), (dict(d=(1 << 31) - 8, ldw=(1 << 31) - 8), 7)])
def test_quantize(how, code):
    assert _quantize(**how) == code
    if "codes" not in how or how["codes"] is not None:
        a = dict(W=ONE, type=F16, ldw=64, L=10, d=64, codes=ONE, scales=ONE) | how
        assert lib().xfc_mx4_dequantize(a["codes"], a["scales"], a["L"], a["d"], a["W"], a["type"], a["ldw"], None) == code


def _logits(X=ONE, type=F16, ldx=64, codes=ONE, scales=ONE, out=ONE, ldo=64, B=2, L=10, d=64, bits=8):
    return lib().xfc_mx4_logits(X, type, ldx, codes, scales, out, ldo, B, L, d, bits, None)


@pytest.mark.parametrize("how,code", [
    (dict(X=None), 1), (dict(out=None), 1), (dict(bits=6), 1), (dict(B=-1), 1), (dict(d=0), 1), (dict(type=-1), 1), (dict(ldx=60), 3), (dict(ldo=12), 3),
    (dict(out=ctypes.c_void_p(8)), 3), (dict(ldo=8), 6), (dict(ldx=56), 6), (dict(d=9096, ldx=9096), 7), (dict(d=16392, ldx=16392, bits=4), 7),
    (dict(L=(1 << 30) + 1, ldo=1 << 31), 7), (dict(B=0, X=None), 0), (dict(L=0, codes=None), 0)])
def test_logits(how, code):
    assert _logits(**how) == code


def _topk(X=ONE, ldx=64, B=2, L=1000, d=64, numy=1000, K=5, bits=4, values=ONE, indices=ONE, ws=ONE, nbytes=1 << 30):
    return lib().xfc_mx4_topk(X, F16, ldx, ONE, ONE, B, L, d, numy, K, bits, values, indices, ws, nbytes, None)


@pytest.mark.parametrize("how,code", [
    (dict(K=0), 1), (dict(K=8193, L=10000), 1), (dict(K=8, L=7), 1), (dict(numy=0), 1), (dict(values=None), 1), (dict(indices=None), 1), (dict(bits=5), 1),
    (dict(ws=None), 4), (dict(nbytes=64), 4), (dict(K=9, nbytes=2 * 1000 * 2 - 16), 4), (dict(ws=ctypes.c_void_p(24)), 3), (dict(B=0), 0)])
def test_topk(how, code):
    assert _topk(**how) == code


def test_workspaces():
    h = lib()
    assert h.xfc_mx4_code_bytes(65, 96) == 2 * 64 * 48 and h.xfc_mx4_scale_bytes(65, 96) == 2 * 64 * 4
    assert h.xfc_mx4_code_bytes(-1, 64) == 0 and h.xfc_mx4_topk_workspace_bytes(4, 0, 64, 1) == 0 and h.xfc_mx4_topk_workspace_bytes(4, 100, 64, 9000) == 0
    assert h.xfc_mx4_topk_workspace_bytes(300, 2812281, 768, 8) < 300 * 2812281 * 4 // 63
    # by maxima, and by logits where the rows are few or K is large
    assert h.xfc_mx4_topk_workspace_bytes(512, 1310720, 768, 100) == 512 * 20480 * 4
    assert h.xfc_mx4_topk_workspace_bytes(8, 1310720, 768, 100) > 8 * 1310720 * 2
    assert h.xfc_mx4_topk_workspace_bytes(512, 131072, 768, 100) > 512 * 131072 * 2


def _preference(X=ONE, type=F16, ldx=64, W=ONE, ldw=64, scales=None, L=10, d=64, rowptr=ONE, chosen=ONE, rejected=ONE, B=2, P=5, beta=0.1,
                smoothing=0.0, loss=ONE, dX=ONE, dx_type=F32, lddx=64, G=None, ldg=0, ws=ONE, nbytes=1 << 20):
    return lib().xfc_preference(X, type, ldx, W, ldw, scales, L, d, rowptr, chosen, rejected, None, None, B, P, beta, smoothing, 1.0, loss, None, dX,
                                dx_type, lddx, G, ldg, ws, nbytes, None)


@pytest.mark.parametrize("how,code", [
    (dict(X=None), 1), (dict(W=None), 1), (dict(rowptr=None), 1), (dict(chosen=None), 1), (dict(rejected=None), 1), (dict(loss=None), 1), (dict(L=0), 1),
    (dict(d=0), 1), (dict(P=-1), 1), (dict(B=1 << 23), 1), (dict(B=(1 << 22) - 1), 1), (dict(dx_type=7), 1), (dict(smoothing=1.5), 1), (dict(smoothing=float("nan")), 1), (dict(beta=float("nan")), 1), (dict(beta=float("inf")), 1),
    (dict(ldx=60), 3), (dict(ldw=60), 3), (dict(scales=ctypes.c_void_p(8)), 3), (dict(ldx=56), 6), (dict(ldw=56), 6), (dict(lddx=56), 6), (dict(G=ONE, ldg=9), 6),
    (dict(d=4104, ldx=4104, ldw=4104, lddx=4104), 7), (dict(P=(1 << 30) + 1), 7), (dict(dX=ctypes.c_void_p(8)), 3), (dict(lddx=66), 3), (dict(ws=None), 4), (dict(nbytes=16), 4), (dict(ws=ctypes.c_void_p(24)), 3)])
def test_preference(how, code):
    assert _preference(**how) == code


def test_python_refuses_what_is_no_gpu_tensor():
    w = torch.zeros(10, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="GPU"):
        mx4_quantize(w)
    with pytest.raises(RuntimeError, match="labels, dims"):
        mx4_quantize(w[0])
    codes, scales = torch.zeros(1, 64 * 32, dtype=torch.uint8), torch.zeros(1, 256, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="GPU"):
        MX4Labels(codes, scales, 10, 64)
    with pytest.raises(RuntimeError, match="multiple of 8"):
        mx4_dequantize(codes, scales, 10, 60)
    with pytest.raises(TypeError, match="uint8"):
        mx4_dequantize(codes.float(), scales, 10, 64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        preference(torch.zeros(1, 64), w, i, i, i)
    with pytest.raises(TypeError, match="float16"):
        preference(torch.zeros(1, 64), w.float(), i, i, i)
    with pytest.raises(RuntimeError, match="XFCLayer"):
        preference(torch.zeros(1, 64), None, i, i, i)


@pytest.mark.parametrize("which", ["reference", "pair_weight"])
def test_what_gets_no_gradient_may_not_ask_for_one(which):
    from renee_amd import preference_loss

    i, t = torch.zeros(2, dtype=torch.int32), torch.zeros(2, requires_grad=True)
    embed, w = torch.zeros(1, 64, requires_grad=True), torch.zeros(10, 64, dtype=torch.float16)
    for x in (embed, embed.detach()):
        with pytest.raises(RuntimeError, match=f"{which}.detach"):
            preference_loss(x, w, i, i, i, **{which: t})
    for ok in (lambda: preference_loss(embed, w, i, i, i, **{which: t.detach()}), torch.no_grad()(lambda: preference_loss(embed, w, i, i, i, **{which: t}))):
        with pytest.raises(RuntimeError, match="GPU"):  # refused for nothing but its device
            ok()


def test_the_logits_of_any_batch_take_bounded_workspace():
    """What top-K above 8 asks for where it writes logits: all rows up to 512 of them or 2 GiB, no more for more rows, and always what 256 rows take."""
    need = lib().xfc_mx4_topk_workspace_bytes
    per = -(-2812281 // 64) * 64 * 2
    assert need(512, 2812281, 768, 1000) > 512 * per and need(8192, 2812281, 768, 1000) == need(512, 2812281, 768, 1000) < 3 << 30
    assert need(100000, 131072, 768, 300) <= 2 << 30 and need(2000, 131072, 768, 300) > 2000 * 131072 * 2
    for L, K in ((20001, 100), (320001, 1000), (1310720, 300), (1310720, 100)):
        sizes = [need(B, L, 768, K) for B in (1, 31, 32, 127, 128, 256, 257, 511, 512, 513, 2048, 5000, 70000)]
        if K > 256:
            assert sizes == sorted(sizes)
            assert all(s >= need(256, L, 768, K) for s in sizes[5:])
    # more rows than fit go in even turns
    assert need(1024, 1310720, 768, 300) == need(512, 1310720, 768, 300) and need(769, 1310720, 768, 300) == need(512, 1310720, 768, 300)
    assert need(768, 1310720, 768, 300) > 768 * 1310720 * 2
