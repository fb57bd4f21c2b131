"""Label matrices in MX4 against the format's definition in 64 bits (oracle/label_oracle.py): codes and scales to the last bit, logits
and top-K at sizes that do not fill a unit, a step, a block or a row tile, blocks of zeros, NaNs and infinities."""
import math

import pytest
import torch

from oracle import label_oracle as O
from renee_amd import MX4Labels, XFCLayer, mx4_dequantize, mx4_quantize

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


def _matrix(L, d, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(L, d, generator=g) * 0.02 * torch.exp2(spread * torch.randn(L, 1, generator=g))
    return w.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L,d", [(1, 8), (63, 32), (64, 64), (65, 72), (130, 128), (129, 200), (200, 768), (70, 136)])
def test_codes_and_scales_are_those_of_the_definition(dev, L, d, dtype):
    w = _matrix(L, d, dtype, L + d)
    w[0] = 0                                        # a block of zeros
    w[L // 2, :4] = torch.tensor([0.25, -0.75, 1.25, 2.5]).to(dtype)  # ties, under a block's largest of 4
    w[L // 2, 4] = 4.0
    w[L - 1, d - 1] = -7.5                          # beyond 6 after scaling
    codes, scales = mx4_quantize(w.to(dev))
    ec, es = O.pack(w)
    assert torch.equal(scales.cpu(), es)
    assert torch.equal(codes.cpu(), ec)
    for out in DTYPES:
        back = mx4_dequantize(codes, scales, L, d, out)
        assert back.dtype == out and torch.equal(back.cpu(), O.rounded(w, 4).to(out))


def test_codes_of_numbers_that_are_not_finite_and_of_the_smallest(dev):
    w = _matrix(8, 96, torch.float32, 3)
    w[1, 40] = float("inf")
    w[2, 0] = float("nan")
    w[3, 95] = -float("inf")
    w[4, :32] = 2.0 ** -130 * torch.arange(32)      # the scale stops at 2^-127
    w[5, :32] = 2.0 ** -125
    w[6, 32:64] = 3e38
    codes, scales = mx4_quantize(w.to(dev))
    ec, es = O.pack(w)
    assert torch.equal(scales.cpu(), es)
    back = mx4_dequantize(codes, scales, 8, 96, torch.float32).cpu()
    expect = O.rounded(w, 4).float()
    assert torch.equal(torch.isnan(back), torch.isnan(expect))
    assert torch.equal(torch.nan_to_num(back, nan=1.0), torch.nan_to_num(expect, nan=1.0))


def test_strided_and_misaligned_weights(dev):
    w = _matrix(100, 264, torch.float16, 5).to(dev)
    for view in (w[:, :200], w[:, 3:203], w.t()[:100, :96], w[::3, 64:128]):
        codes, scales = mx4_quantize(view)
        ec, es = mx4_quantize(view.contiguous())
        assert torch.equal(codes, ec) and torch.equal(scales, es)


def _problem(B, L, d, bits, dtype, seed):
    g = torch.Generator().manual_seed(seed + 1)
    x = torch.randn(B, d, generator=g)
    x = (x / x.norm(dim=1, keepdim=True)).to(dtype)
    w = _matrix(L, d, torch.float16, seed, 0.3)
    z = O.rounded(x, bits) @ O.rounded(w, 4).t()
    return x, w, z


def _logit_tolerance(x, w, bits):
    """fp16 rounds by half a step, 2^-11 of the value or 2^-25; the sums in fp32 by 2^-24 of the magnitudes summed, once a product; and
    with 8 bits the matrix pipe may drop 2^-14 of the largest of four neighbouring products, less than their sum."""
    mass = O.rounded(x, bits).abs() @ O.rounded(w, 4).abs().t()
    return mass * ((2.0 ** -14 if bits == 8 else 0.0) + 2.0 ** -24 * math.log2(2 * x.shape[1])) + 2.0 ** -25


SIZES = [(1, 1, 8), (1, 65, 64), (3, 63, 32), (16, 200, 200), (17, 130, 136), (32, 64, 128), (33, 129, 768), (64, 257, 72), (65, 1000, 384),
         (128, 640, 256), (129, 700, 96), (200, 300, 1024), (300, 5000, 64)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B,L,d", SIZES)
def test_logits(dev, B, L, d, bits):
    x, w, z = _problem(B, L, d, bits, DTYPES[(B + L) % 3], B + L + d)
    labels = MX4Labels.from_weight(w.to(dev))
    got = labels.xfc_forward(x.to(dev), embed_bits=bits).cpu().double()
    tol = _logit_tolerance(x, w, bits) + z.abs() * 2.0 ** -11
    assert got.shape == z.shape and bool(((got - z).abs() <= tol).all()), float(((got - z).abs() / tol).max())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("d", [2048, 4104, 8192])
def test_logits_of_wide_embeddings(dev, d, bits):
    x, w, z = _problem(40, 150, d, bits, torch.float16, d)
    got = MX4Labels.from_weight(w.to(dev)).xfc_forward(x.to(dev), embed_bits=bits).cpu().double()
    tol = _logit_tolerance(x, w, bits) + z.abs() * 2.0 ** -11
    assert bool(((got - z).abs() <= tol).all())


def test_logits_leave_what_lies_beside_them(dev):
    x, w, z = _problem(37, 203, 72, 4, torch.float16, 9)
    out = torch.full((40, 224), 7.0, dtype=torch.float16, device=dev)
    MX4Labels.from_weight(w.to(dev)).xfc_forward(x.to(dev), out=out[:37, :203], embed_bits=4)
    assert bool((out[37:] == 7).all()) and bool((out[:, 203:] == 7).all())
    assert torch.equal(out[:37, :203].cpu(), z.half())  # 4 x 4 bits: sums are exact


@pytest.mark.parametrize("bits", [4, 8])
def test_a_row_or_label_that_is_no_number_stays_by_itself(dev, bits):
    x, w, z = _problem(20, 100, 200, bits, torch.float16, 11)
    x[3, 150] = float("inf")
    w[70, 10] = float("nan")
    got = MX4Labels.from_weight(w.to(dev)).xfc_forward(x.to(dev), embed_bits=bits).cpu()
    bad = torch.zeros(20, 100, dtype=torch.bool)
    bad[3], bad[:, 70] = True, True
    assert torch.equal(torch.isnan(got), bad)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype,scales", [(torch.float16, (6e-8, 3e-7, 1e-5, 1.0, 3e4)), (torch.bfloat16, (1e-38, 3e-38, 1e-5, 1e30)),
                                          (torch.float32, (1e-43, 1e-40, 2e-38, 1.0, 1e30))])
def test_embeddings_of_any_size(dev, dtype, scales, bits):
    """From the smallest numbers of a type to near its largest, each row against labels of one block each."""
    g = torch.Generator().manual_seed(5)
    x = torch.cat([torch.randn(7, 96, generator=g) * s for s in scales]).to(dtype)
    w = torch.zeros(96, 96, dtype=torch.float32)
    w[torch.arange(96), torch.arange(96)] = 1.0
    want = O.rounded(x, bits)
    want[torch.isnan(want).any(1)] = math.nan  # a sum with a NaN is one
    labels = MX4Labels.from_weight(w.to(dev))
    v, i = labels.topk(x.to(dev), 8, embed_bits=bits)  # fp32 sums of one number each
    best = O.topk(want, 8)
    # A row with an infinity (fp16 at 3e4) has no scores.  Of numbers whose scale times the labels' lies below fp32's normal numbers only
    # that they stay there is asked.
    small = want.abs().nan_to_num(1.0).amax(1) < 2.0 ** -118
    v, i = v.cpu().double(), i.cpu()
    assert torch.equal(v[~small], best[0][~small]) and torch.equal(i[~small], best[1][~small].where(best[1][~small] >= 0, torch.tensor(95)))
    assert bool(((v[small] - best[0][small]).abs() <= 2.0 ** -118).all())


def test_codes_beyond_32_bits(dev):
    """12,000,010 labels x 768: 4.9 GB of codes.  The last labels' logits, rows, best places and pairs are those of a matrix of them alone."""
    from renee_amd import pair_margins

    L, d, tail = 12_000_010, 768, 138
    units = -(-L // 64)
    g = torch.Generator(device=dev).manual_seed(3)
    codes = torch.randint(0, 256, (units, 24 * 1024), generator=g, dtype=torch.uint8, device=dev)
    scales = torch.full((units, 6 * 256), 120, dtype=torch.uint8, device=dev)
    scales[-2] = 124  # the best labels are among the last
    labels = MX4Labels(codes, scales, L, d)
    few = MX4Labels(codes[-3:].clone(), scales[-3:].clone(), tail, d)
    x = torch.randn(40, d, generator=g, device=dev)
    assert (L - tail) % 64 == 0
    for rows in (1, 40):
        assert torch.equal(labels.xfc_forward(x[:rows])[:, -tail:], few.xfc_forward(x[:rows]))
        v, i = labels.topk(x[:rows], 5)
        ev, ei = few.topk(x[:rows], 5)
        assert torch.equal(v, ev) and torch.equal(i, ei + L - tail)
    assert torch.equal(mx4_dequantize(codes[-3:].clone(), scales[-3:].clone(), tail, d), labels.dequantize()[-tail:])
    rowptr = torch.tensor([0, 3], dtype=torch.int32, device=dev)
    c, r = (torch.tensor(t, dtype=torch.int32, device=dev) for t in ((0, 70, 137), (137, 5, 64)))
    assert torch.equal(pair_margins(x[:1], labels, rowptr, c + L - tail, r + L - tail), pair_margins(x[:1], few, rowptr, c, r))


def test_matrices_of_more_than_one_launch(dev):
    """A launch has fewer than 2^24 workgroups of 256 threads: units behind those come out as in a matrix of them alone."""
    units, d, tail = (1 << 24) + 5, 8, 7 * 64 - 30
    L = units * 64 - 30
    w = torch.empty(L, d, dtype=torch.float16, device=dev).fill_(0.5)
    w[-tail:] = _matrix(tail, d, torch.float16, 9).to(dev)
    codes, scales = mx4_quantize(w)
    ec, es = mx4_quantize(w[-tail:].clone())
    assert torch.equal(codes[-7:], ec) and torch.equal(scales[-7:], es)
    assert torch.equal(codes[:-7], codes[:1].expand(units - 7, -1)) and torch.equal(scales[:-7], scales[:1].expand(units - 7, -1))
    assert torch.equal(mx4_dequantize(codes, scales, L, d)[-tail:], mx4_dequantize(ec, es, tail, d))


@pytest.mark.parametrize("K", [3, 12])
def test_topk_of_more_rows_than_a_launch_has(dev, K):
    x, w, _ = _problem(1000, 64, 8, 4, torch.float16, 12)
    labels = MX4Labels.from_weight(w.to(dev))
    B = (1 << 22) + 100
    many = x.to(dev).repeat(B // 1000 + 1, 1)[:B]
    v, i = labels.topk(many, K)
    ev, ei = labels.topk(x.to(dev), K)
    assert torch.equal(v, ev.repeat(B // 1000 + 1, 1)[:B]) and torch.equal(i, ei.repeat(B // 1000 + 1, 1)[:B])


# ---- top-K: with 4 bits sums are exact, so that values and labels are those of a stable sort -----------------------------------

@pytest.mark.parametrize("K", [1, 5, 8, 9, 100])
@pytest.mark.parametrize("B,L,d", [(1, 100, 64), (2, 131, 200), (16, 4097, 768), (33, 1000, 72), (100, 3001, 384), (130, 700, 128), (300, 2222, 96)])
def test_topk_with_4_bits(dev, B, L, d, K):
    x, w, z = _problem(B, L, d, 4, DTYPES[(B + K) % 3], B + L + d + K)
    assert torch.equal(z.float().double(), z)
    v, i = MX4Labels.from_weight(w.to(dev)).topk(x.to(dev), K, embed_bits=4)
    ev, ei = O.topk(z.half().double() if K > 8 else z, K)
    assert torch.equal(v.cpu().double(), ev) and torch.equal(i.cpu(), ei)


# (above 8 by maxima alone from 32 rows and 1000 K or more labels on, here 36, 130, 33 and 300 rows: those that several at a time share a CU)
@pytest.mark.parametrize("B,L,d,K", [(2, 70001, 64, 5), (40, 66000, 128, 100), (5, 140003, 64, 8), (3, 70001, 64, 3000), (36, 18729, 8, 9), (130, 40961, 72, 10),
                                     (33, 70001, 200, 16), (3, 414001, 64, 100), (34, 600003, 8, 256), (130, 270011, 8, 256), (300, 41000, 200, 20)])
def test_topk_of_many_labels(dev, B, L, d, K):
    x, w, z = _problem(B, L, d, 4, torch.float16, L + K)
    v, i = MX4Labels.from_weight(w.to(dev)).topk(x.to(dev), K, embed_bits=4)
    ev, ei = O.topk(z.half().double() if K > 8 else z, K)
    assert torch.equal(v.cpu().double(), ev) and torch.equal(i.cpu(), ei)


# (enough rows and labels for the rows to stay in registers, of one to four row tiles and 2 to 6 steps; of 2,500 rows the last 452 do not)
@pytest.mark.parametrize("B,L,d,K,dtype", [(450, 330001, 200, 5, torch.float16), (512, 340000, 384, 8, torch.float32), (2500, 90017, 512, 3, torch.bfloat16),
                                           (1024, 170001, 640, 20, torch.float16), (512, 327745, 768, 8, torch.float16), (900, 164000, 744, 10, torch.float32)])
def test_topk_of_many_rows_and_labels(dev, B, L, d, K, dtype):
    g = torch.Generator(device=dev).manual_seed(L)
    w = (torch.randn(L, d, generator=g, device=dev) * 0.02).half()
    x = torch.randn(B, d, generator=g, device=dev).to(dtype)
    w[-1] *= 1.5
    w[L // 2, 3], w[7, d - 1], x[B - 1, d - 1] = float("nan"), float("inf"), float("nan")
    labels = MX4Labels.from_weight(w)
    v, i = labels.topk(x, K, embed_bits=4)
    exact = labels.dequantize(torch.float32).double().t().contiguous()
    rows = mx4_dequantize(*mx4_quantize(x), B, d, torch.float32).double()
    for r0 in range(0, B, 128):
        z = rows[r0:r0 + 128] @ exact
        z = torch.where(torch.isnan(z), -math.inf, z.half().double() if K > 8 else z)
        ev, ei = (t[:, :K] for t in torch.sort(z, dim=1, descending=True, stable=True))
        assert torch.equal(v[r0:r0 + 128].double(), ev)
        some = ev > -math.inf  # (up to 8 a row without numbers reports the last label)
        assert torch.equal(i[r0:r0 + 128][some], ei[some])


@pytest.mark.parametrize("B,L,d,K", [(1, 1000, 768, 5), (40, 3001, 200, 8), (140, 2000, 64, 3), (20, 4000, 384, 50)])
def test_topk_with_8_bits(dev, B, L, d, K):
    """The labels' scores are within the product's tolerance of the definition's, none that was left out is above them by more than
    twice that, and they are in order."""
    x, w, z = _problem(B, L, d, 8, torch.float32, B + L + d + K)
    v, i = (t.cpu() for t in MX4Labels.from_weight(w.to(dev)).topk(x.to(dev), K))
    tol = _logit_tolerance(x, w, 8) + (z.abs() * 2.0 ** -11 if K > 8 else 0.0)
    assert bool(((v.double() - z.gather(1, i)).abs() <= tol.gather(1, i)).all())
    assert all(len(set(row.tolist())) == K for row in i)
    order = v[:, :-1] - v[:, 1:]
    assert bool((order >= 0).all()) and bool(((order > 0) | (i[:, :-1] < i[:, 1:])).all())
    left = z.clone().scatter_(1, i, -math.inf)
    assert bool((left <= v[:, -1:].double() + tol).all())


def test_topk_ties_go_to_the_lower_label_and_constant_rows(dev):
    w = torch.ones(300, 64, dtype=torch.float16)
    w[7::50] = 2.0
    x = torch.ones(3, 64, dtype=torch.float16)
    x[1] = 0
    for bits in (4, 8):
        for K in (8, 20):
            v, i = MX4Labels.from_weight(w.to(dev)).topk(x.to(dev), K, embed_bits=bits)
            ev, ei = O.topk((x.double() @ w.double().t()), K)
            assert torch.equal(v.cpu().double(), ev) and torch.equal(i.cpu(), ei)


@pytest.mark.parametrize("K", [9, 12])
@pytest.mark.parametrize("B,L", [(40, 1000), (40, 32003), (300, 16003)])
def test_topk_above_8_counts_nan_as_the_least(dev, B, L, K):
    """Rows of equal scores, of fewer numbers than K, of none, and of infinities."""
    w = torch.zeros(L, 64, dtype=torch.float16)
    w[:, 0] = torch.randint(-2, 3, (L,), generator=torch.Generator().manual_seed(L)).half()
    w[5::3] = float("nan")
    w[:, 40] = torch.where(torch.arange(L) % 1009 == 7, 6.0e4, 0.0).half()
    x = torch.zeros(B, 64, dtype=torch.float32)  # by maxima with 16,003 and 32,003 labels
    x[5:, 2] = 1.0
    x[0, 0], x[1, 1], x[2, 0], x[3, 40], x[4, 40] = 1.0, 1.0, float("nan"), 1e30, -1e30
    some = w.clone()
    some[4:] = float("nan")
    for m in (w, some):
        z = (O.rounded(x, 4) @ O.rounded(m, 4).t()).half().double()
        ev, ei = O.topk(torch.where(torch.isnan(z), -math.inf, z), K)
        v, i = MX4Labels.from_weight(m.to(dev)).topk(x.to(dev), K, numy=L - 1, embed_bits=4)
        assert torch.equal(v.cpu().double(), ev) and torch.equal(i.cpu(), ei.clamp(max=L - 2))


def test_topk_without_scores_and_clamped_labels(dev):
    x, w, _ = _problem(4, 200, 64, 4, torch.float16, 21)
    w[3:] = float("nan")
    x[2] = float("nan")
    z = O.rounded(x, 4) @ O.rounded(w, 4).t()
    v, i = MX4Labels.from_weight(w.to(dev)).topk(x.to(dev), 5, numy=150, embed_bits=4)
    ev, ei = O.topk(z, 5)
    assert torch.equal(v.cpu().double(), ev) and torch.equal(i.cpu(), torch.where(ei < 0, 149, ei))


def test_topk_rows_in_turns(dev):
    """A workspace of 256 rows' logits takes 600 rows in three turns."""
    from renee_amd._lib import check, lib

    x, w, z = _problem(600, 3000, 64, 4, torch.float16, 33)
    labels, xd = MX4Labels.from_weight(w.to(dev)), x.to(dev)
    ev, ei = labels.topk(xd, 20, embed_bits=4)
    need = lib().xfc_mx4_topk_workspace_bytes(256, 3000, 64, 20)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    v, i = torch.empty_like(ev), torch.empty_like(ei)
    check(lib().xfc_mx4_topk(xd.data_ptr(), 0, 64, labels.codes.data_ptr(), labels.scales.data_ptr(), 600, 3000, 64, 3000, 20, 4, v.data_ptr(),
                             i.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream), "xfc_mx4_topk")
    assert torch.equal(v, ev) and torch.equal(i, ei)
    assert torch.equal(ei.cpu(), O.topk(z.half().double(), 20)[1])


def test_replays_with_rows_in_registers(dev):
    """Many rows and labels (both forms of maxima), replayed beside eager calls of other labels and beside each other."""
    L, d, B = 340000, 256, 512
    g = torch.Generator(device=dev).manual_seed(6)
    labels, other = (MX4Labels.from_weight((torch.randn(L, d, generator=g, device=dev) * 0.02).half()) for _ in range(2))
    x = torch.randn(B, d, generator=g, device=dev).half()
    calls = [lambda m, K=K: m.topk(x, K, embed_bits=4) for K in (5, 40)]
    graphs, got = [], []
    for call in calls:
        call(labels)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(call(labels))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        x.copy_(torch.randn(B, d, generator=g, device=dev).half())
        want = [call(labels) for call in calls]
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        beside = calls[0](other)
        torch.cuda.synchronize()
        for out, w in zip(got, want):
            assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])
        assert all(torch.equal(p, q) for p, q in zip(beside, calls[0](other)))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("K", [5, 30])
def test_replays_of_two_graphs_on_two_streams(dev, bits, K):
    """Scratch belongs to a call: two captured calls of the same labels run beside each other, with new inputs between replays."""
    x, w, _ = _problem(50, 3000, 128, bits, torch.float16, 41)
    labels = MX4Labels.from_weight(w.to(dev))
    xs = [x.to(dev), x.flip(0).contiguous().to(dev)]
    eager = [labels.topk(t, K, embed_bits=bits) + (labels.xfc_forward(t, embed_bits=bits),) for t in xs]
    torch.cuda.synchronize()
    graphs, got = [], []
    for t in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(labels.topk(t, K, embed_bits=bits) + (labels.xfc_forward(t, embed_bits=bits),))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for outs in got:
            for o in outs:
                o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for outs, want in zip(got, eager):
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_labels_of_a_layer(dev):
    """quantize_labels follows the layer: the fp16 weights, or the fp32 ones where the layer keeps them; and a checkpoint of them."""
    w = _matrix(500, 128, torch.float32, 51)
    x = torch.randn(20, 128, generator=torch.Generator().manual_seed(1)).half()
    for master in (False, True):
        layer = XFCLayer(500, 128, 32, dev, weight=w.to(dev), master_weights=master)
        labels = layer.quantize_labels()
        assert torch.equal(labels.dequantize(torch.float32).cpu(), O.rounded(w if master else w.half(), 4).float())
        # close to the layer's own logits: rounding weights to 4 bits is some 11 % of their norm
        exact, rough = layer.xfc_forward(x.to(dev)).float(), labels.xfc_forward(x.to(dev)).float()
        assert float((rough - exact).norm() / exact.norm()) < 0.25
        again = MX4Labels.from_state_dict(labels.state_dict(), dev)
        assert torch.equal(again.xfc_forward(x.to(dev)), labels.xfc_forward(x.to(dev)))


def test_empty_calls(dev):
    labels = MX4Labels.from_weight(torch.ones(70, 64, device=dev))
    assert labels.xfc_forward(torch.empty(0, 64, device=dev)).shape == (0, 70)
    assert labels.topk(torch.empty(0, 64, device=dev), 3)[1].shape == (0, 3)
    none = MX4Labels.from_weight(torch.empty(0, 64, device=dev))
    assert none.xfc_forward(torch.ones(3, 64, device=dev)).shape == (3, 0)
    assert none.dequantize().shape == (0, 64)


def test_codes_of_a_label_beyond_32_bits(dev):
    """One label of 2^26 + 136 dims: its last steps' codes, 2 GiB behind its first ones, are those of these dims alone."""
    first, d = 1 << 26, (1 << 26) + 136
    w = torch.full((1, d), 0.5, dtype=torch.float16, device=dev)
    w[:, first:] = _matrix(1, 136, torch.float16, 17).to(dev)
    codes, scales = mx4_quantize(w)
    ec, es = mx4_quantize(w[:, first:].contiguous())
    assert torch.equal(codes[:, first // 128 * 4096:], ec) and torch.equal(scales[:, first // 128 * 256:], es)
    back = mx4_dequantize(codes, scales, 1, d)
    assert torch.equal(back[:, first:], mx4_dequantize(ec, es, 1, 136)) and bool((back[:, :first] == 0.5).all())


def test_topk_of_more_rows_than_the_workspace_has_room_for(dev):
    """1,600 rows x 700,001 labels, whose logits are more than 2 GiB: in turns of what that holds, as in one workspace for all of them."""
    from renee_amd._lib import check, lib

    B, L, d, K = 1600, 700001, 64, 300
    g = torch.Generator(device=dev).manual_seed(8)
    labels = MX4Labels.from_weight((torch.randn(L, d, generator=g, device=dev) * 0.02).half())
    x = torch.randn(B, d, generator=g, device=dev).half()
    need, all_rows = lib().xfc_mx4_topk_workspace_bytes(B, L, d, K), B * (-(-L // 64) * 64 * 2 + (-(-L // 64) * 2 + 7) // 8 * 16)
    assert need < all_rows and need <= 2 << 30
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    v, i = labels.topk(x, K)
    assert torch.cuda.max_memory_allocated() - before < need + (64 << 20)
    ws, ev, ei = torch.empty(all_rows, dtype=torch.uint8, device=dev), torch.empty_like(v), torch.empty_like(i)
    check(lib().xfc_mx4_topk(x.data_ptr(), 0, d, labels.codes.data_ptr(), labels.scales.data_ptr(), B, L, d, L, K, 8, ev.data_ptr(), ei.data_ptr(), ws.data_ptr(),
                             all_rows, torch.cuda.current_stream().cuda_stream), "xfc_mx4_topk")
    assert torch.equal(v, ev) and torch.equal(i, ei)


@pytest.mark.parametrize("B,L,d,K", [(36, 18729, 8, 9), (130, 40961, 72, 10), (300, 41000, 200, 20), (33, 70001, 200, 16), (34, 600003, 8, 256), (260, 100003, 136, 40)])
def test_topk_with_8_bits_by_maxima(dev, B, L, d, K):
    """Above 8 labels of enough rows and labels: no logits are written, and the scores that are formed again are those of xfc_forward to the bit, in the
    order of a stable sort; which holds what test_logits asks of them against 64 bits."""
    from renee_amd._lib import lib

    assert lib().xfc_mx4_topk_workspace_bytes(B, L, d, K) < B * L
    x, w, z = _problem(B, L, d, 8, DTYPES[(B + K) % 3], L + K)
    x[B // 2] = 0
    if B > 35:
        x[3, 0] = float("nan")
    z = O.rounded(x, 8) @ O.rounded(w, 4).t()
    labels, xd = MX4Labels.from_weight(w.to(dev)), x.to(dev)
    v, i = labels.topk(xd, K)
    own = labels.xfc_forward(xd).cpu().double()
    ev, ei = O.topk(torch.where(torch.isnan(own), -math.inf, own), K)
    assert torch.equal(v.cpu().double(), ev) and torch.equal(i.cpu(), ei)
    numbers = ~torch.isnan(x.float()).any(1)
    tol = (_logit_tolerance(x, w, 8) + z.abs() * 2.0 ** -11)[numbers]
    chosen = i.cpu()[numbers]
    assert bool(((v.cpu().double()[numbers] - z[numbers].gather(1, chosen)).abs() <= tol.gather(1, chosen)).all())
    left = z[numbers].scatter(1, chosen, -math.inf)
    assert bool((left <= v.cpu().double()[numbers][:, -1:] + tol).all())


@pytest.mark.parametrize("B,K,bits", [(150, 5, 4), (150, 5, 8), (40, 10, 4), (40, 10, 8), (300, 200, 8)])
def test_topk_by_maxima_of_four_units_together(dev, B, K, bits):
    """A million labels and more whose rows do not stay in registers: a wave writes the maxima of four units at once, here with two left over."""
    L, d = 1_100_100, 64
    assert -(-L // 64) % 4 == 2
    g = torch.Generator(device=dev).manual_seed(B + K)
    w = (torch.randn(L, d, generator=g, device=dev) * 0.02).half()
    x = torch.randn(B, d, generator=g, device=dev).half()
    w[-40:] *= 1.25
    w[L // 3, 3], x[B - 1, d - 1] = float("nan"), float("inf")
    labels = MX4Labels.from_weight(w)
    v, i = labels.topk(x, K, embed_bits=bits)
    z = labels.xfc_forward(x, embed_bits=bits).float()
    if K <= 8:  # by the fp32 sums, which the logits are the roundings of
        assert torch.equal(v[:-1].half().float(), z[:-1].gather(1, i[:-1])) and bool((v[:-1, :-1] >= v[:-1, 1:]).all())
        v = v.half().float()
    z = torch.where(torch.isnan(z), -math.inf, z)
    for r0 in range(0, B, 64):
        ev, ei = (t[:, :K] for t in torch.sort(z[r0:r0 + 64], dim=1, descending=True, stable=True))
        assert torch.equal(v[r0:r0 + 64], ev)
        if K > 8:
            assert torch.equal(i[r0:r0 + 64], ei)
