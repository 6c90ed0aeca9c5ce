"""What is measured of the microscaled operators: 4-bit quantisation, 4-bit products, and 8-bit activation checkpoints.

A microscaled block is 32 neighbouring elements of a row with one scale that is a power of two (a byte: exponent + 127, 255 for a
block that holds an infinity or NaN). The scale is the smallest one at which no element of the block passes the element type's
largest value; elements are rounded to nearest, ties to even. The operators:

  cast      a matrix into blocks and back (what a checkpoint of an activation, or a weight at load, goes through)
  linear    Y = q4(X) W^T with W in 4-bit blocks: the product of a dense layer, activations quantised on the way in
  experts   the whole mixture-of-experts feed-forward on 4-bit blocks: router, top-k, up, SiLU, down, gated sum
  ln_fwd    LayerNorm that also leaves an 8-bit checkpoint of its input for the backward pass
  ln_bwd    the LayerNorm's backward pass from that checkpoint

`own` = False computes them in elementary torch operations, `own` = True through the library."""
import math

import torch

own = False

MAXV = {"e2m1": (0.75, 3), "e4m3": (0.875, 9), "e5m2": (0.875, 16)}      # largest element = first * 2^second
F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
DT = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5


def _lib():
    import os
    import sys
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "test-model-thing-cuda_b200"))
    import tmt_moe_b200
    return tmt_moe_b200


# ---------------------------------------------------------------- cases

def listed():
    return [
        # a few rows of a float32 activation on their way into a checkpoint; the width is no power of two
        dict(name="cast_rows_e4m3", op="cast", rows=37, cols=320, fmt="e4m3", dtype="f32"),
        # a whole batch of bf16 activations into 4 bits and back: 131072 positions at the widest benchmark configuration
        dict(name="cast_batch_e2m1", op="cast", rows=131072, cols=2048, fmt="e2m1", dtype="bf16"),
        # one byte position of one stream through a dense layer: latency
        dict(name="linear_one_row", op="linear", rows=1, k=1024, n=2048, dtype="bf16"),
        # a prompt of odd length, float32 result for a loss or a residual kept in 32 bits
        dict(name="linear_prompt_f32", op="linear", rows=777, k=1344, n=2504, dtype="f32"),
        # a training-sized window (batch 128 x 128 positions) through a 1024 -> 4096 layer
        dict(name="linear_window", op="linear", rows=16384, k=1024, n=4096, dtype="bf16"),
        # 64 sampler streams, one position each, the sampler configuration's experts
        dict(name="experts_decode", op="experts", rows=64, dim=1024, hidden=2048, experts=16, topk=2, router="bf16"),
        # a ragged window through the smallest configuration's experts
        dict(name="experts_ragged", op="experts", rows=2041, dim=512, hidden=1024, experts=4, topk=2, router="f32"),
        # the largest configuration: 131072 tokens, 64 experts, top-4
        dict(name="experts_batch", op="experts", rows=131072, dim=2048, hidden=2048, experts=64, topk=4, router="f32"),
        # one decode step of 64 streams
        dict(name="ln_fwd_streams", op="ln_fwd", rows=64, dim=1024, fmt="e5m2"),
        # the activations of the largest configuration
        dict(name="ln_fwd_batch", op="ln_fwd", rows=131072, dim=2048, fmt="e4m3"),
        # an odd number of rows at a width that is no power of two
        dict(name="ln_bwd_ragged", op="ln_bwd", rows=2047, dim=1280, fmt="e5m2"),
        dict(name="ln_bwd_batch", op="ln_bwd", rows=131072, dim=2048, fmt="e4m3"),
    ]


def _spread(rng, lo, hi, step=1):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    op = rng.choice(["cast", "linear", "experts", "ln_fwd", "ln_bwd"])
    if op == "cast":
        cols = _spread(rng, 64, 8192, 64)
        return dict(op=op, rows=_spread(rng, 1, 131072 * 2048 // max(cols, 2048)), cols=cols, fmt=rng.choice(["e2m1", "e4m3", "e5m2"]),
                    dtype=rng.choice(["bf16", "f32"]))
    if op == "linear":
        return dict(op=op, rows=_spread(rng, 1, 16384), k=_spread(rng, 64, 4096, 64), n=_spread(rng, 64, 4096, 8), dtype=rng.choice(["bf16", "f32"]))
    if op == "experts":
        experts = _spread(rng, 1, 64)
        return dict(op=op, rows=_spread(rng, 1, 32768), dim=_spread(rng, 128, 2048, 64), hidden=_spread(rng, 128, 2048, 64), experts=experts,
                    topk=rng.randint(1, min(4, experts)), router=rng.choice(["bf16", "f32"]))
    dim = _spread(rng, 32, 8192, 32)
    return dict(op=op, rows=_spread(rng, 1, 131072 * 2048 // max(dim, 2048)), dim=dim, fmt=rng.choice(["e4m3", "e5m2"]))


def work(case):
    """Each input once, each output once. Blocks: 1 byte of scale for 32 elements."""
    c, op = case, case["op"]
    if op == "cast":
        n, size = c["rows"] * c["cols"], 2 if c["dtype"] == "bf16" else 4
        block = (0.5 if c["fmt"] == "e2m1" else 1.0) + 1 / 32
        return {"bytes": n * (size + block + block + 2), "flops": 4 * n}      # values in, blocks out; blocks in, bf16 out
    if op == "linear":
        m, n, k = c["rows"], c["n"], c["k"]
        return {"bytes": 2 * m * k + n * k * 17 / 32 + m * n * (2 if c["dtype"] == "bf16" else 4), "flops": 2 * m * n * k}
    if op == "experts":
        t, d, h, e, k = c["rows"], c["dim"], c["hidden"], c["experts"], c["topk"]
        hit = min(e, t * k)
        return {"bytes": 4 * t * d + hit * 2 * d * h * 17 / 32 + e * d * (4 if c["router"] == "f32" else 2), "flops": 2 * t * d * e + 4 * t * k * d * h}
    n, r, d = c["rows"] * c["dim"], c["rows"], c["dim"]
    if op == "ln_fwd":
        return {"bytes": n * (4 + 33 / 32) + 8 * r + 8 * d, "flops": 10 * n}
    return {"bytes": n * (4 + 33 / 32) + 8 * r + 12 * d, "flops": 14 * n}


# ---------------------------------------------------------------- blocks in torch

def _blocks(x, fmt):
    """(elements in units of the scale, scale exponent per block); x: float32, rows of blocks of 32."""
    t, p = MAXV[fmt]
    b = x.reshape(x.shape[0], -1, 32)
    amax = b.abs().amax(-1)
    m, ex = torch.frexp(amax)
    e = torch.where(amax > 0, ex - p + (m > t).int(), torch.full_like(ex, -127)).clamp_(min=-127)
    v = b * torch.exp2(-e.float()).unsqueeze(-1)
    if fmt == "e2m1":
        a = v.abs()
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        v = torch.copysign(torch.round(a / step) * step, v)      # half to even: the even multiple of a step is the even code
    return v.reshape(x.shape), e


def _q(x, fmt):
    """The values that the blocks of x stand for, in float32."""
    v, e = _blocks(x, fmt)
    if fmt != "e2m1":
        v = v.to(F8[fmt]).float()
    return (v.reshape(x.shape[0], -1, 32) * torch.exp2(e.float()).unsqueeze(-1)).reshape(x.shape)


def _pack4(x):
    """4-bit blocks as the library keeps them: two codes a byte (the even element in the low half); the scale bytes in tiles of
    128 rows x 4 blocks, within a tile by row % 32, then row / 32, then block; rows and blocks padded to whole tiles."""
    v, e = _blocks(x, "e2m1")
    a = v.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    r, kb = e.shape
    full = torch.zeros(-(-r // 128) * 128, -(-kb // 4) * 4, dtype=torch.uint8, device=x.device)
    full[:r, :kb] = (e + 127).to(torch.uint8)
    tiles = full.reshape(-1, 4, 32, full.shape[1] // 4, 4).permute(0, 3, 2, 1, 4)
    return codes.contiguous(), tiles.reshape(-1).contiguous()


def _unpack4(codes, scales, rows, cols):
    """The float32 values of _pack4's bytes."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1).reshape(rows, cols // 32, 32)
    s = scales.reshape(-(-rows // 128), -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-(-rows // 128) * 128, -1)[:rows, :cols // 32]
    return (v * torch.exp2(s.float() - 127).unsqueeze(-1)).reshape(rows, cols)


# ---------------------------------------------------------------- states

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _activations(rows, cols, g):
    """Roughly normal, with a few wide columns (as trained layers have), and a block here and there that is all zero."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= torch.where(torch.rand(cols, device="cuda", generator=g) < 0.01, 8.0, 1.0)
    blocks = x.reshape(rows, cols // 32, 32)
    blocks *= (torch.rand(rows, cols // 32, 1, device="cuda", generator=g) > 0.002).float()
    return x


def _ln_inputs(case, seed):
    rows, dim = case["rows"], case["dim"]
    g = _generator(seed)
    x = (_activations(rows, dim, g) + 0.3).to(torch.bfloat16)
    gamma = 1 + 0.2 * torch.randn(dim, device="cuda", generator=g)
    return x, gamma, g


def _experts_inputs(case, seed):
    """Activations on a grid of 1/16 and router weights on a grid of 1/512: every partial sum of a router logit then fits 24 bits, the
    logits are the same in any order of summation, and the selected experts (ties: the lower index) are too."""
    t, d, h, e = case["rows"], case["dim"], case["hidden"], case["experts"]
    g = _generator(seed)
    x = (torch.randn(t, d, device="cuda", generator=g).clamp_(-4, 4) * 16).round_().div_(16).to(torch.bfloat16)
    wr = (torch.randn(e, d, device="cuda", generator=g) * 0.02 * 512).round_().clamp_(-31, 31).div_(512).to(DT[case["router"]])
    weights = [[_pack4((torch.randn(n, k, device="cuda", generator=g) * 0.02).to(torch.bfloat16).float()) for _ in range(e)]
               for n, k in ((h, d), (d, h))]
    return x, wr, weights


def prepare(case, seed):
    op, g = case["op"], _generator(seed)
    s = {"case": case, "op": op}
    if op == "cast":
        s["x"] = _activations(case["rows"], case["cols"], g).to(DT[case["dtype"]])
        if own:
            s["M"] = M = _lib()
            r, c = s["x"].shape
            s["y"] = torch.empty(r, c, dtype=torch.bfloat16, device="cuda")
            four = case["fmt"] == "e2m1"
            s["codes"] = torch.empty(r, c // 2 if four else c, dtype=torch.uint8, device="cuda")
            s["scales"] = torch.empty(M.mxfp4_scale_bytes(r, c) if four else r * (c // 32), dtype=torch.uint8, device="cuda")
    elif op == "linear":
        s["x"] = _activations(case["rows"], case["k"], g).to(torch.bfloat16)
        s["w"] = _pack4((torch.randn(case["n"], case["k"], device="cuda", generator=g) * 0.02).to(torch.bfloat16).float())
        if own:
            s["M"] = M = _lib()
            s["weight"] = M.Mxfp4Weights([(*s["w"], case["n"], case["k"])])
            s["y"] = torch.empty(case["rows"], case["n"], dtype=DT[case["dtype"]], device="cuda")
            s["work"] = torch.empty(M.linear_mxfp4_work_bytes(case["rows"], case["k"]), dtype=torch.uint8, device="cuda")
    elif op == "experts":
        s["x"], s["wr"], s["w"] = _experts_inputs(case, seed)
        if own:
            s["M"] = M = _lib()
            s["moe"] = M.MoE(case["rows"], case["dim"], case["experts"], case["topk"], hidden=case["hidden"],
                             router_dtype=M.F32 if case["router"] == "f32" else M.BF16, training=False)
            s["wup"] = M.Mxfp4Weights([(c, sc, case["hidden"], case["dim"]) for c, sc in s["w"][0]])
            s["wdown"] = M.Mxfp4Weights([(c, sc, case["dim"], case["hidden"]) for c, sc in s["w"][1]])
            s["y"] = torch.empty_like(s["x"])
    else:
        x, s["gamma"], g = _ln_inputs(case, seed)
        rows, dim = x.shape
        if op == "ln_fwd":
            s["x"], s["beta"] = x, 0.2 * torch.randn(dim, device="cuda", generator=g)
        else:
            f = x.float()
            s["mean"] = f.mean(1)
            s["rstd"] = torch.rsqrt(f.var(1, unbiased=False) + EPS)
            v, e = _blocks(f, case["fmt"])
            s["codes"], s["scales"] = v.to(F8[case["fmt"]]).view(torch.uint8), (e + 127).to(torch.uint8)
            s["dy"] = (0.1 * torch.randn(rows, dim, device="cuda", generator=g)).to(torch.bfloat16)
        if own:
            s["M"] = M = _lib()
            s["fmt"] = M.ACT8_E4M3 if case["fmt"] == "e4m3" else M.ACT8_E5M2
            s["out"] = torch.empty(rows, dim, dtype=torch.bfloat16, device="cuda")
            if op == "ln_fwd":
                s["mean"], s["rstd"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
                s["codes"] = torch.empty(rows, dim, dtype=torch.uint8, device="cuda")
                s["scales"] = torch.empty(rows, dim // 32, dtype=torch.uint8, device="cuda")
            else:
                s["dgamma"], s["dbeta"] = torch.empty(dim, device="cuda"), torch.empty(dim, device="cuda")
                s["scratch"] = torch.empty(M.ln_backward_act8_scratch_bytes(rows, dim), dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    M, op, c = s["M"], s["op"], s["case"]
    if op == "cast":
        if c["fmt"] == "e2m1":
            M.quantize_mxfp4(s["x"], s["codes"], s["scales"])
            M.dequantize_mxfp4(s["codes"], s["scales"], s["y"])
        else:
            fmt = M.ACT8_E4M3 if c["fmt"] == "e4m3" else M.ACT8_E5M2
            M.act8_save(s["x"], s["codes"], s["scales"], fmt)
            M.act8_restore(s["codes"], s["scales"], s["y"], fmt)
        return s["y"]
    if op == "linear":
        M.linear_mxfp4(s["x"], s["weight"], s["y"], s["work"])
        return s["y"]
    if op == "experts":
        s["moe"].forward_mxfp4(s["x"], s["wr"], s["wup"], s["wdown"], s["y"])
        return s["y"]
    if op == "ln_fwd":
        M.ln_forward_act8(s["x"], s["gamma"], s["beta"], s["out"], s["mean"], s["rstd"], s["codes"], s["scales"], s["fmt"])
        return s["out"], s["mean"], s["rstd"], s["codes"].view(F8[c["fmt"]]), s["scales"].view(torch.float8_e8m0fnu)
    M.ln_backward_act8(s["codes"], s["scales"], s["dy"], s["gamma"], s["mean"], s["rstd"], s["out"], s["dgamma"], s["dbeta"], s["scratch"], s["fmt"])
    return s["out"], s["dgamma"], s["dbeta"]


def _ffn(x, up, down, d, h):
    """x: the float32 values of quantised rows."""
    p = x @ _unpack4(*up, h, d).T
    return _q(p * torch.sigmoid(p), "e2m1") @ _unpack4(*down, d, h).T


def _run_plain(s):
    op, c = s["op"], s["case"]
    if op == "cast":
        return _q(s["x"].float(), c["fmt"]).to(torch.bfloat16)
    if op == "linear":
        return (_q(s["x"].float(), "e2m1") @ _unpack4(*s["w"], c["n"], c["k"]).T).to(DT[c["dtype"]])
    if op == "experts":
        t, d, h, e, k = c["rows"], c["dim"], c["hidden"], c["experts"], c["topk"]
        x = s["x"].float()
        top, idx = (x @ s["wr"].float().T).sort(dim=1, descending=True, stable=True)
        gate, idx = torch.softmax(top[:, :k], 1), idx[:, :k]
        order = idx.reshape(-1).argsort(stable=True)
        counts = torch.bincount(idx.reshape(-1), minlength=e).tolist()
        groups = torch.split(_q(x, "e2m1")[order // k], counts)
        rows = torch.cat([_ffn(g, up, down, d, h) for g, up, down in zip(groups, *s["w"]) if len(g)])
        rows *= gate.reshape(-1)[order].unsqueeze(1)
        back = torch.empty_like(order).scatter_(0, order, torch.arange(t * k, device=order.device))
        return rows[back].reshape(t, k, d).sum(1).to(torch.bfloat16)
    if op == "ln_fwd":
        x = s["x"].float()
        mean = x.mean(1)
        rstd = torch.rsqrt(x.var(1, unbiased=False) + EPS)
        y = (x - mean.unsqueeze(1)) * rstd.unsqueeze(1) * s["gamma"] + s["beta"]
        v, e = _blocks(x, c["fmt"])
        return y.to(torch.bfloat16), mean, rstd, v.to(F8[c["fmt"]]), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    rows, dim = s["dy"].shape
    v = s["codes"].view(F8[c["fmt"]]).float().reshape(rows, -1, 32)
    x = (v * torch.exp2(s["scales"].float() - 127).unsqueeze(-1)).reshape(rows, dim)
    xh = (x - s["mean"].unsqueeze(1)) * s["rstd"].unsqueeze(1)
    dy = s["dy"].float()
    g = dy * s["gamma"]
    a, b = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = s["rstd"].unsqueeze(1) * (g - a - xh * b)
    return dx.to(torch.bfloat16), (dy * xh).sum(0), dy.sum(0)


# ---------------------------------------------------------------- the definitions in 64 bits

def _grid(fmt):
    """The non-negative values of an element type in the order of their codes."""
    ebits, mbits = {"e2m1": (2, 1), "e4m3": (4, 3), "e5m2": (5, 2)}[fmt]
    bias = (1 << (ebits - 1)) - 1
    top = {"e2m1": 7, "e4m3": 0x7e, "e5m2": 0x7b}[fmt]
    vals = []
    for code in range(top + 1):
        ex, m = code >> mbits, code & ((1 << mbits) - 1)
        vals.append(m * 2.0 ** (1 - bias - mbits) if ex == 0 else (1 + m / (1 << mbits)) * 2.0 ** (ex - bias))
    return vals


def _exact_blocks(x, fmt):
    """(element values, block scales) of float64 rows, from the definition: the smallest power of two that keeps the block's largest
    magnitude within the type, then the nearest value of the type, of two equally near ones that with the even code."""
    vals = torch.tensor(_grid(fmt), dtype=torch.float64, device=x.device)
    b = x.reshape(x.shape[0], -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    e = torch.floor(torch.log2(amax.clamp(min=2.0 ** -150) / vals[-1])) - 1
    for _ in range(3):
        e = torch.where(amax > vals[-1] * torch.exp2(e), e + 1, e)
    scale = torch.exp2(e.clamp(min=-127))
    a = (b / scale).abs()
    mid = (vals[1:] + vals[:-1]) / 2
    low, high = torch.bucketize(a, mid), torch.bucketize(a, mid, right=True)      # they differ on a midpoint alone
    code = torch.where(low % 2 == 0, low, high)
    return (torch.copysign(vals[code], b)).reshape(x.shape), scale.squeeze(-1)


def _exact_q(x, fmt):
    if x.numel() > 1 << 26:      # in pieces: the codes of one piece take 16 bytes an element
        return torch.cat([_exact_q(p, fmt) for p in x.split(max(1, (1 << 26) // x.shape[1]))])
    v, scale = _exact_blocks(x, fmt)
    return (v.reshape(x.shape[0], -1, 32) * scale.unsqueeze(-1)).reshape(x.shape)


def _exact_unpack4(codes, scales, rows, cols):
    """Byte by byte as the layout is written down."""
    vals = torch.tensor(_grid("e2m1"), dtype=torch.float64, device=codes.device)
    nib = torch.empty(rows, cols, dtype=torch.long, device=codes.device)
    nib[:, 0::2], nib[:, 1::2] = (codes % 16).long(), (codes // 16).long()
    v = vals[nib % 8] * torch.where(nib >= 8, -1.0, 1.0).double()
    r = torch.arange(rows, device=codes.device).unsqueeze(1)
    b = torch.arange(cols // 32, device=codes.device).unsqueeze(0)
    tiles = -(-(cols // 32) // 4)
    at = ((r // 128) * tiles + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4
    return (v.reshape(rows, -1, 32) * torch.exp2(scales[at].double() - 127).unsqueeze(-1)).reshape(rows, cols)


def exact(case, seed):
    op = case["op"]
    if op in ("cast", "linear"):
        s = prepare(case, seed)
        if op == "cast":
            return _exact_q(s["x"].double(), case["fmt"])
        return _exact_q(s["x"].double(), "e2m1") @ _exact_unpack4(*s["w"], case["n"], case["k"]).T
    if op == "experts":
        x, wr, (up, down) = _experts_inputs(case, seed)
        t, d, h, k = case["rows"], case["dim"], case["hidden"], case["topk"]
        x = x.double()
        logits = x @ wr.double().T
        keys = logits - torch.arange(case["experts"], device="cuda") * 2.0 ** -40      # logits lie on a grid of 2^-13
        idx = keys.topk(k, 1).indices
        picked = logits.gather(1, idx)
        gate = torch.exp(picked - picked.amax(1, keepdim=True))
        gate /= gate.sum(1, keepdim=True)
        xq = _exact_q(x, "e2m1")
        del x
        y = torch.zeros(t, d, dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            rows, j = torch.where(idx == e)
            if len(rows):
                p = xq[rows] @ _exact_unpack4(*up[e], h, d).T
                y.index_add_(0, rows, gate[rows, j].unsqueeze(1) * (_exact_q(p / (1 + torch.exp(-p)), "e2m1") @ _exact_unpack4(*down[e], d, h).T))
        return y
    if op == "ln_fwd":
        x, gamma, g = _ln_inputs(case, seed)
        beta = 0.2 * torch.randn(x.shape[1], device="cuda", generator=g)
        x = x.double()
        mean = x.mean(1, keepdim=True)
        rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + EPS)
        y = (x - mean) * rstd * gamma.double() + beta.double()
        pieces = [_exact_blocks(p, case["fmt"]) for p in x.split(max(1, (1 << 26) // x.shape[1]))]
        return y, mean.squeeze(1), rstd.squeeze(1), torch.cat([p[0] for p in pieces]), torch.cat([p[1] for p in pieces])
    s = prepare(case, seed)
    rows, dim = s["dy"].shape
    vals = torch.tensor(_grid(case["fmt"]), dtype=torch.float64, device="cuda")
    c = s["codes"].int()
    x = vals[c % 128] * torch.where(c >= 128, -1.0, 1.0).double()
    x = (x.reshape(rows, -1, 32) * torch.exp2(s["scales"].double() - 127).unsqueeze(-1)).reshape(rows, dim)
    rstd = s["rstd"].double().unsqueeze(1)
    xh = (x - s["mean"].double().unsqueeze(1)) * rstd
    del x
    dy = s["dy"].double()
    dgamma, dbeta = (dy * xh).sum(0), dy.sum(0)
    g = dy * s["gamma"].double()
    dx = rstd * (g - g.sum(1, keepdim=True) / dim - xh * ((g * xh).sum(1, keepdim=True) / dim))
    return dx, dgamma, dbeta
