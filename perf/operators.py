"""What the operators on narrow label matrices and on label preferences are measured on.

A label matrix in microscaled 4-bit floating point ("MX4"): blocks of 32 consecutive dims of a label share a scale 2^(byte - 127),
each weight is a sign, two exponent bits and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6).  It serves scoring, and it stands for
the frozen label matrix while an encoder is trained on preferences.  `kind` says which operator a case calls:

  quantize    mx4_quantize, and mx4_dequantize of what it left: the label matrix once through 4 bits
  logits      MX4Labels.xfc_forward: embeddings in 8 or 4 bits times the label matrix, logits rounded to fp16
  topk        MX4Labels.topk: the K best labels of every row
  preference  preference_loss(...).backward() (`form` "input": the gradient of the embeddings), or preference(..., g=...) (`form`
              "g": the pairs' gradient added to the G of a training step), for labels in fp16 or in MX4

Storage.  Labels go in units of 64, dims in steps of 128.  In a unit, label 32 p + 8 q + 4 t + r is row 4 q + r of tile 2 p + t.
codes: per unit and step, the four tiles one after the other, each sixteen rows of the step's blocks (four, fewer in the last step
of a width that is no multiple of 128), a block being 16 bytes, even dims in the lower halves of bytes.  scales: per unit and step
four blocks x sixteen rows x four tiles bytes.
"""
from __future__ import annotations

import math

import torch

own = False

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # a classifier of a few thousand labels and an odd width: launches count
        dict(name="quantize_4k_d200", kind="quantize", L=4097, d=200, dtype="fp16"),
        # the resident fp16 weights of a 131,072-label classifier
        dict(name="quantize_131k", kind="quantize", L=131072, d=768, dtype="fp16"),
        # fp32 master weights
        dict(name="quantize_master_655k", kind="quantize", L=655363, d=768, dtype="fp32"),
        # serving: a handful of queries, all logits
        dict(name="logits_b16_131k", kind="logits", B=16, L=131072, d=768, bits=8, dtype="fp16"),
        # a partial batch, a 384-wide encoder, an odd label count, embeddings in 4 bits
        dict(name="logits_b199_320k_d384", kind="logits", B=199, L=320001, d=384, bits=4, dtype="fp16"),
        # the headline batch
        dict(name="logits_b512_1310k", kind="logits", B=512, L=1310720, d=768, bits=8, dtype="fp16"),
        # serving: a single query
        dict(name="top5_b1_131k", kind="topk", B=1, L=131073, d=768, K=5, bits=4, dtype="fp16"),
        # final evaluation: the hundred best labels
        dict(name="top100_b512_1310k", kind="topk", B=512, L=1310720, d=768, K=100, bits=4, dtype="fp16"),
        # validation during training on the largest data set
        dict(name="top5_b1024_2812k", kind="topk", B=1024, L=2812281, d=768, K=5, bits=4, dtype="fp16"),
        # an encoder in training against a frozen 4-bit label matrix, the small batch
        dict(name="preference_input_b32_131k", kind="preference", form="input", weights="mx4", B=32, L=131072, d=768, pairs=8, dtype="fp32"),
        # the same for a full batch with long slates, labels in fp16
        dict(name="preference_input_b1024_1310k", kind="preference", form="input", weights="fp16", B=1024, L=1310720, d=768, pairs=64, dtype="fp16"),
        # pairs beside the classifier's own loss in a training step
        dict(name="preference_g_b512_131k", kind="preference", form="g", weights="fp16", B=512, L=131072, d=768, pairs=16, dtype="fp16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: 1 to 1024 rows, 1,000 to 2.8 million labels, widths from a 64-wide bottleneck to 1024, odd ones among them."""
    while True:
        kind = rng.choice(["quantize", "logits", "logits", "topk", "topk", "preference", "preference"])
        d = rng.choice([64, 72, 128, 200, 256, 384, 512, 768, 768, 768, 1024])
        L = _log_int(rng, 1000, 2812281)
        B = _log_int(rng, 1, 1024)
        if rng.random() < 0.3:  # full batches are the common case
            B = rng.choice([32, 64, 128, 256, 512, 1024])
        dtype = rng.choice(["fp16", "fp16", "bf16", "fp32"])
        if kind == "quantize":
            case = dict(kind=kind, L=L, d=d, dtype=dtype)
            if L * d > 655363 * 768:
                continue
        elif kind == "logits":
            case = dict(kind=kind, B=B, L=L, d=d, bits=rng.choice([8, 8, 4]), dtype=dtype)
            if B * L > 512 * 1310720:
                continue
        elif kind == "topk":
            case = dict(kind=kind, B=B, L=L, d=d, K=rng.choice([1, 3, 5, 5, 8, 10, 100, 200]), bits=4, dtype=dtype)
            if B * L * (4 if case["K"] > 8 else 1) > 1024 * 2812281:
                continue
        else:
            case = dict(kind=kind, form=rng.choice(["input", "input", "g"]), weights=rng.choice(["fp16", "mx4"]), B=B, L=L, d=d,
                        pairs=_log_int(rng, 1, 64), dtype=dtype)
            if case["form"] == "g" and (B * L > 512 * 1310720 or case["weights"] == "mx4"):
                continue  # G belongs to a classifier in training, whose weights are fp16
        return case


# ---- MX4 in elementary operations ---------------------------------------------------------------------------------------------

def _block_exponent(x, largest):
    """floor(log2 of a block's largest magnitude) - largest, kept in -127 .. 127; x: (..., blocks, 32) fp32."""
    top = x.abs().amax(-1)
    return torch.where(top > 0, torch.frexp(top).exponent - 1 - largest, -127).clamp(-127, 127)


def _e2m1_code(y):
    """The nearest of GRID, ties to an even mantissa, as 3 bits and the sign."""
    a = y.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() + (a > 2.5).byte() + (a >= 3.5).byte() +
            (a > 5.0).byte())
    return code + 8 * (y < 0).byte()


def _pow2(e):
    return torch.ldexp(torch.ones((), device=e.device), e)


def _as_blocks(x):
    """(rows, d) of any type as (rows, blocks, 32) in fp32, padded with zeros."""
    x = x.float()
    return torch.nn.functional.pad(x, (0, -x.shape[1] % 32)).reshape(x.shape[0], -1, 32)


def _quantize_plain(w):
    """codes and scales of (L, d), as the module's text lays them out."""
    L = w.shape[0]
    x = torch.nn.functional.pad(_as_blocks(w), (0, 0, 0, 0, 0, -L % 64))
    e = _block_exponent(x, 2)
    c = _e2m1_code(x / _pow2(e)[..., None])
    c = c[..., 0::2] + 16 * c[..., 1::2]                                  # (labels, blocks, 16)
    U, nb = c.shape[0] // 64, c.shape[1]
    c = c.reshape(U, 2, 4, 2, 4, nb, 16).permute(0, 1, 3, 2, 4, 5, 6).reshape(U, 4, 16, nb, 16)  # unit, tile, row, block
    whole = nb // 4
    head = c[:, :, :, :4 * whole].reshape(U, 4, 16, whole, 4, 16).permute(0, 3, 1, 2, 4, 5).reshape(U, -1)
    codes = torch.cat([head, c[:, :, :, 4 * whole:].reshape(U, -1)], 1)
    s = torch.nn.functional.pad((e + 127).byte(), (0, -nb % 4)).reshape(U, 2, 4, 2, 4, -1, 4)
    scales = s.permute(0, 5, 6, 2, 4, 1, 3).reshape(U, -1)               # unit, step, block, row (q, r), tile (p, t)
    return codes.contiguous(), scales.contiguous()


def _rows_plain(codes, scales, label):
    """The bytes (n, blocks, 16) and scale bytes (n, blocks) of the given labels."""
    U, nb = codes.shape[0], codes.shape[1] // 1024
    unit, p, q, t, r = label // 64, label // 32 % 2, label // 8 % 4, label // 4 % 2, label % 4
    head = codes[:, :nb // 4 * 4096].view(U, nb // 4, 4, 16, 4, 16)
    rest = codes[:, nb // 4 * 4096:].view(U, 4, 16, nb % 4, 16)
    c = torch.cat([head[unit, :, 2 * p + t, 4 * q + r].flatten(1, 2), rest[unit, 2 * p + t, 4 * q + r]], 1)
    return c, scales.view(U, -1, 4, 16, 4)[unit, :, :, 4 * q + r, 2 * p + t].flatten(1)[:, :nb]


def _values_plain(c, s):
    """(n, 32 blocks) in fp32 of bytes and scale bytes."""
    table = torch.tensor(GRID + tuple(-v for v in GRID), device=c.device)
    v = torch.stack([table[(c & 15).int()], table[(c >> 4).int()]], -1).flatten(2)
    return (v * _pow2(s.int() - 127)[..., None]).flatten(1)


def _dequantize_plain(codes, scales, L, d):
    """The (L, d) values in fp32."""
    return _values_plain(*_rows_plain(codes, scales, torch.arange(L, device=codes.device)))[:, :d]


def _embed_plain(x, bits):
    """Embeddings as they enter the product: blocks of 32 dims in 4 bits, or in 8 (four exponent and three mantissa bits)."""
    b = _as_blocks(x)
    if bits == 4:
        e = _block_exponent(b, 2)
        code = _e2m1_code(b / _pow2(e)[..., None])
        table = torch.tensor(GRID + tuple(-v for v in GRID), device=x.device)
        v = table[code.int()]
    else:
        e = _block_exponent(b, 8)
        y = b / _pow2(e)[..., None]
        step = _pow2(torch.frexp(y.abs()).exponent.clamp(min=-5) - 4)
        v = (torch.round(y / step) * step).clamp(-448.0, 448.0)
    return (v * _pow2(e)[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _topk_plain(z, K):
    """The K largest of each row, the lower label first where they are equal: of more candidates than K, by far more than share
    a value, in the order of their labels."""
    label = z.topk(min(2 * K + 64, z.shape[1]), dim=1, sorted=False).indices.sort(dim=1).values
    values, place = z.gather(1, label).sort(dim=1, descending=True, stable=True)
    return values[:, :K], label.gather(1, place[:, :K])


# ---- cases --------------------------------------------------------------------------------------------------------------------

def _weights(L, d, seed, dtype):
    """Label weights as a classifier's initialisation has them, N(0, 0.02), a length of its own for each label."""
    g = torch.Generator(device="cuda")
    g.manual_seed(2000 + seed)
    w = torch.empty(L, d, device="cuda", dtype=dtype)
    step = 1 << 18
    for r in range(0, L, step):
        n = min(step, L - r)
        w[r:r + n] = torch.randn(n, d, generator=g, device="cuda") * (0.02 * (0.5 + torch.rand(n, 1, generator=g, device="cuda")))
    return w


def _quantized(L, d, seed):
    U, nb = -(-L // 64), -(-d // 32)
    codes = torch.empty(U, 1024 * nb, device="cuda", dtype=torch.uint8)
    scales = torch.empty(U, 256 * -(-nb // 4), device="cuda", dtype=torch.uint8)
    w = _weights(L, d, seed, torch.float16)
    for u in range(0, U, 4096):
        codes[u:u + 4096], scales[u:u + 4096] = _quantize_plain(w[64 * u:64 * (u + 4096)])
    return codes, scales


def prepare(case, seed):
    kind, L, d = case["kind"], case["L"], case["d"]
    if kind == "quantize":
        return dict(case=case, W=_weights(L, d, seed, DTYPES[case["dtype"]]))
    g = torch.Generator(device="cuda")
    g.manual_seed(1000 + seed)
    B = case["B"]
    x = torch.randn(B, d, generator=g, device="cuda")
    state = dict(case=case, X=(x / x.norm(dim=1, keepdim=True)).to(DTYPES[case["dtype"]]))
    if kind != "preference" or case["weights"] == "mx4":
        state["codes"], state["scales"] = _quantized(L, d, seed)
    else:
        state["W"] = _weights(L, d, seed, torch.float16)
    if kind == "preference":
        # slates of unequal lengths, a row's two clicked labels against others, one pair in sixteen masked
        P = B * case["pairs"]
        row = (B * torch.rand(P, generator=g, device="cuda") ** 1.5).long().clamp(max=B - 1).sort().values
        state["rowptr"] = torch.searchsorted(row, torch.arange(B + 1, device="cuda")).int()
        clicked = torch.randint(0, L, (B, 2), generator=g, device="cuda")
        chosen = clicked[row, torch.randint(0, 2, (P,), generator=g, device="cuda")]
        masked = torch.rand(P, generator=g, device="cuda") < 1 / 16
        state["chosen"] = torch.where(masked, -1, chosen).int()
        state["rejected"] = torch.randint(0, L, (P,), generator=g, device="cuda").int()
        state["reference"] = torch.randn(P, generator=g, device="cuda") * 0.02
        state["beta"], state["smoothing"] = 2.0, 0.05
        if case["form"] == "g":
            state["G"] = torch.rand(B, -(-L // 8) * 8, generator=g, device="cuda", dtype=torch.float16) * 0.5
        else:
            state["X"].requires_grad_(True)
    return state


def _preference_plain(state):
    case, X = state["case"], state["X"].detach().float()
    rowptr, c, r = state["rowptr"].long(), state["chosen"].long(), state["rejected"].long()
    of = lambda label: state["W"][label].float() if "W" in state else _values_plain(*_rows_plain(state["codes"], state["scales"], label))[:, :case["d"]]  # noqa: E731
    row = torch.repeat_interleave(torch.arange(case["B"], device="cuda"), rowptr[1:] - rowptr[:-1])
    used = c >= 0
    difference = of(c.clamp(min=0)) - of(r)
    margin = torch.where(used, (X[row] * difference).sum(1) - state["reference"], 0.0)
    m, beta, eps = margin * state["beta"], state["beta"], state["smoothing"]
    softplus = torch.log1p(torch.exp(-m.abs()))
    # -(1 - eps) log sigmoid(m) - eps log sigmoid(-m), and its derivative by the margin
    loss = torch.where(used, softplus + (-m).clamp(min=0) * (1 - eps) + m.clamp(min=0) * eps, 0.0)
    slope = torch.where(used, beta * (1 / (1 + torch.exp(-m)) - (1 - eps)), 0.0)
    loss = loss.sum()
    if case["form"] == "input":
        grad = torch.zeros_like(X).index_add_(0, row, difference * slope[:, None])
        return dict(loss=loss, grad_input=grad.to(state["X"].dtype))
    G = state["G"]
    at = torch.cat([row * G.shape[1] + c, row * G.shape[1] + r])[torch.cat([used, used])]
    add = torch.cat([slope, -slope])[torch.cat([used, used])]
    at, place = at.unique(return_inverse=True)
    flat = G.view(-1)
    flat[at] = (flat[at].float() + torch.zeros(at.shape, device="cuda").index_add_(0, place, add)).half()
    return dict(loss=loss, margin=margin, G=G)


def run(state):
    case = state["case"]
    kind, L, d = case["kind"], case["L"], case["d"]
    if own:
        import renee_amd

        if kind == "quantize":
            codes, scales = renee_amd.mx4_quantize(state["W"])
            return renee_amd.mx4_dequantize(codes, scales, L, d, torch.float16)
        labels = state["W"] if "W" in state else renee_amd.MX4Labels(state["codes"], state["scales"], L, d)
        if kind == "logits":
            return labels.xfc_forward(state["X"], embed_bits=case["bits"])
        if kind == "topk":
            values, best = labels.topk(state["X"], case["K"], embed_bits=case["bits"])
            return dict(values=values, labels=best)
        X = state["X"]
        pairs = (state["rowptr"], state["chosen"], state["rejected"])
        how = dict(reference=state["reference"], beta=state["beta"], label_smoothing=state["smoothing"])
        if case["form"] == "g":
            loss, margin, _ = renee_amd.preference(X, labels, *pairs, g=state["G"], **how)
            return dict(loss=loss, margin=margin, G=state["G"])
        X.grad = None
        loss = renee_amd.preference_loss(X, labels, *pairs, **how)
        loss.backward()
        return dict(loss=loss, grad_input=X.grad)
    if kind == "quantize":
        codes, scales = _quantize_plain(state["W"])
        return _dequantize_plain(codes, scales, L, d).half()
    if kind == "preference":
        return _preference_plain(state)
    z = _embed_plain(state["X"], case["bits"]) @ _dequantize_plain(state["codes"], state["scales"], L, d).t()
    if kind == "logits":
        return z.half()
    if case["K"] > 8:  # above 8 labels are ordered by their scores in fp16
        z = z.half()
    values, best = _topk_plain(z, case["K"])
    return dict(values=values.float(), labels=best)


def work(case):
    kind, L, d = case["kind"], case["L"], case["d"]
    size = 4 if case["dtype"] == "fp32" else 2
    narrow = 0.5 * L * d + L * -(-d // 32)
    if kind == "quantize":  # the weights in, the codes and scales out and in again, the values out
        return dict(bytes=size * L * d + 2 * narrow + 2 * L * d, flops=2 * L * d)
    B = case["B"]
    if kind == "logits":
        return dict(bytes=narrow + size * B * d + 2 * B * L, flops=2 * B * L * d)
    if kind == "topk":
        return dict(bytes=narrow + size * B * d + 12 * B * case["K"], flops=2 * B * L * d)
    pairs = B * case["pairs"]
    row = 2 * d if case["weights"] == "fp16" else 0.5 * d + -(-d // 32)
    rows = pairs + min(2 * B, pairs)  # rejected labels, and two chosen ones of each row
    out = size * B * d if case["form"] == "input" else 4 * rows + 4 * pairs
    return dict(bytes=rows * row + size * B * d + 12 * pairs + out, flops=4 * pairs * d)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------

def _values64(x, largest_exponent, mantissa_bits, lowest_exponent, limit):
    """Blocks of 32 of the last axis, rounded to a shared power of two times short floats, element by element from the definition."""
    n, d = x.shape
    y = torch.zeros(n, -(-d // 32) * 32, dtype=torch.float64, device=x.device)
    y[:, :d] = x.double()
    y = y.view(n, -1, 32)
    top = y.abs().max(-1, keepdim=True).values
    shared = torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - largest_exponent
    shared = torch.where(top > 0, shared, -127.0).clamp(-127.0, 127.0)
    y = y * torch.exp2(-shared)
    of = torch.floor(torch.log2(torch.where(y != 0, y.abs(), 1.0))).clamp(min=float(lowest_exponent))
    unit = torch.exp2(of - mantissa_bits)
    y = torch.minimum(torch.round(y.abs() / unit) * unit, torch.tensor(limit, dtype=torch.float64, device=x.device)) * torch.sign(y)
    return (y * torch.exp2(shared)).view(n, -1)[:, :d]


def _labels64(codes, scales, labels, d):
    """The dims of the given labels, each byte fetched from where the layout puts it."""
    nb = -(-d // 32)
    unit, at = labels // 64, labels % 64
    tile, row = 2 * (at // 32) + at // 4 % 2, 4 * (at // 8 % 4) + at % 4
    block = torch.arange(nb, device=labels.device)
    step, within = block // 4, block % 4
    wide = torch.where(step < nb // 4, 4, nb % 4)  # blocks of the step
    first = unit[:, None] * (1024 * nb) + step * 4096 + ((tile * 16 + row)[:, None] * wide + within) * 16
    byte = codes.view(-1)[first[..., None] + torch.arange(16, device=labels.device)].int()
    nibble = torch.stack([byte % 16, byte // 16], -1).view(labels.shape[0], nb, 32)
    exponent, mantissa = nibble // 2 % 4, nibble % 2
    magnitude = torch.where(exponent > 0, (1 + 0.5 * mantissa.double()) * torch.exp2(exponent.double() - 1), 0.5 * mantissa.double())
    s = scales.view(-1)[unit[:, None] * (256 * -(-nb // 4)) + step * 256 + within * 64 + row[:, None] * 4 + tile[:, None]]
    v = magnitude * (1 - 2 * (nibble // 8)) * torch.exp2(s.double() - 127)[..., None]
    return v.view(labels.shape[0], -1)[:, :d]


def exact(case, seed):
    state = prepare(case, seed)
    kind, L, d = case["kind"], case["L"], case["d"]
    if kind == "quantize":
        out = torch.empty(L, d, dtype=torch.float64, device="cuda")
        for r in range(0, L, 1 << 18):
            out[r:r + (1 << 18)] = _values64(state["W"][r:r + (1 << 18)], 2, 1, 0, 6.0)
        return out
    if kind in ("logits", "topk"):
        x = _values64(state["X"], *((2, 1, 0, 6.0) if case["bits"] == 4 else (8, 3, -6, 448.0)))
        z = torch.empty(case["B"], L, dtype=torch.float64, device="cuda")
        for r in range(0, L, 1 << 16):
            ids = torch.arange(r, min(r + (1 << 16), L), device="cuda")
            z[:, r:r + (1 << 16)] = x @ _labels64(state["codes"], state["scales"], ids, d).t()
        if kind == "logits":
            return z
        # above 8 the scores are by definition those rounded to fp16
        return dict(values=(z.half().double() if case["K"] > 8 else z).topk(case["K"], dim=1).values, labels=None)
    X = state["X"].detach().double()
    rowptr = state["rowptr"].tolist()
    grad, total = torch.zeros_like(X), 0.0
    margins = torch.zeros(rowptr[-1], dtype=torch.float64, device="cuda")
    of = (lambda ids: state["W"][ids].double()) if "W" in state else (lambda ids: _labels64(state["codes"], state["scales"], ids, d))
    G = state["G"].double() if case["form"] == "g" else None
    b, eps = state["beta"], state["smoothing"]
    for i in range(case["B"]):
        s = slice(rowptr[i], rowptr[i + 1])
        c, r = state["chosen"][s].long(), state["rejected"][s].long()
        keep = c >= 0
        c, r = c[keep], r[keep]
        if not len(c):
            continue
        diff = of(c) - of(r)
        m = diff @ X[i] - state["reference"][s][keep].double()
        margins[s][keep] = m
        total = total - (1 - eps) * torch.nn.functional.logsigmoid(b * m).sum() - eps * torch.nn.functional.logsigmoid(-b * m).sum()
        slope = b * (torch.sigmoid(b * m) - (1 - eps))
        grad[i] = slope @ diff
        if G is not None:
            G[i].index_put_((c,), slope, accumulate=True)
            G[i].index_put_((r,), -slope, accumulate=True)
    total = torch.as_tensor(total, dtype=torch.float64, device="cuda")
    return dict(loss=total, margin=margins, G=G) if case["form"] == "g" else dict(loss=total, grad_input=grad)
