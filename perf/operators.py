"""The operators around the quantized matmul of a decode step or a prompt chunk, through the public entry points and in plain form.

* ``norm``    ``rms_norm``: the residual's addition, the norm, and its output in the stream's type or as the 8-bit
              activation blocks that the package's products read (Q8_0 for the 32-element formats, Q8_K for the k-quants);
* ``mxquant`` ``MxTensor.quantize``: activations or weights to microscaled 4-bit floats (E2M1, an E8M0 scale per 32);
* ``mx``      ``MxMatMul.forward``: the product of activations, quantized to that format on the way, and such weights;
* ``sample``  ``sample``: one token per row of logits with temperature, top-k, top-p and min-p from given uniform numbers.

``run`` computes them in elementary torch operations where ``own`` is false, and calls the package where it is true.
"""
from __future__ import annotations

import numpy as np
import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# the activation blocks are asked for by the format of the weights that will read them
BLOCK = {"Q8_0": 32, "Q4K": 256}


def _norm(name, m, k, x, out, residual=True):
    return {"name": name, "kind": "norm", "m": m, "k": k, "x": x, "out": out, "residual": residual}


def _mx(name, m, n, k, x):
    return {"name": name, "kind": "mx", "m": m, "n": n, "k": k, "x": x}


def _sample(name, b, v, x, t, top_k, top_p, min_p, rows=False):
    return {"name": name, "kind": "sample", "b": b, "v": v, "x": x, "t": t, "top_k": top_k, "top_p": top_p, "min_p": min_p, "rows": rows}


def listed():
    return [
        # one decode token in front of the attention or feed-forward projections of a k-quant model, the smallest call
        _norm("norm Q8_K m1", 1, 4096, "f32", "Q4K"),
        # an odd batch of sequences, a 2048-wide 8-bit model with f16 hidden states; no residual: a model's first norm
        _norm("norm Q8_0 m37 f16", 37, 2048, "f16", "Q8_0", residual=False),
        # a long prompt chunk, the norm kept in the stream's type
        _norm("norm m2048 bf16", 2048, 4096, "bf16", "plain"),
        # a prompt chunk's hidden states to 4 bits
        {"name": "mx quantize m512 bf16", "kind": "mxquant", "m": 512, "k": 4096, "x": "bf16"},
        # one decode token through a key / value projection
        _mx("mx m1 kv", 1, 1024, 4096, "f32"),
        # eight sequences decoded together, gate / up projection
        _mx("mx m8 gate", 8, 14336, 4096, "bf16"),
        # draft tokens or a short prompt, odd length, a row length that is no multiple of 256
        _mx("mx m77 odd", 77, 5000, 2080, "f16"),
        # a prompt chunk through the down projection
        _mx("mx m512 down", 512, 4096, 14336, "bf16"),
        # the largest: a long prompt chunk through the gate / up projection
        _mx("mx m2048 gate", 2048, 14336, 4096, "f32"),
        # one sequence's next token, the usual filters
        _sample("sample b1", 1, 128256, "f32", 0.8, 40, 0.95, 0.05),
        # a large batch, every sequence with settings of its own
        _sample("sample b64 rows", 64, 128256, "f32", 1.0, 0, 0.9, 0.0, rows=True),
        # an odd batch and an odd vocabulary in half precision, where many logits tie; nucleus alone
        _sample("sample b7 bf16", 7, 50257, "bf16", 1.3, 0, 0.99, 0.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choices(("norm", "mxquant", "mx", "sample"), weights=(4, 1, 5, 4))[0]
    x = rng.choice(tuple(TYPES))
    if kind == "norm":
        out = rng.choice(("plain", "Q8_0", "Q4K"))
        m, k = _log_int(rng, 1, 2048), _log_int(rng, 256, 16384)
        if out != "plain":
            k = k // BLOCK[out] * BLOCK[out]
        return {"kind": kind, "m": min(m, (1 << 23) // k), "k": k, "x": x, "out": out, "residual": rng.random() < 0.7}
    if kind == "mxquant":
        m, k = _log_int(rng, 1, 2048), _log_int(rng, 256, 14336) // 32 * 32
        return {"kind": kind, "m": min(m, (1 << 23) // k), "k": k, "x": x}
    if kind == "mx":
        m = rng.randint(1, 8) if rng.random() < 0.4 else _log_int(rng, 9, 2048)
        n, k = _log_int(rng, 256, 14336), _log_int(rng, 512, 14336) // 32 * 32
        return {"kind": kind, "m": max(1, min(m, (1 << 36) // (n * k))), "n": n, "k": k, "x": x}
    v = _log_int(rng, 1000, 200000)
    return {"kind": kind, "b": min(_log_int(rng, 1, 64), (1 << 23) // v), "v": v, "x": x, "t": round(rng.uniform(0.3, 1.5), 2),
            "top_k": rng.choice((0, 0, 1, 20, 50, 400, 2500)), "top_p": rng.choice((1.0, 0.5, 0.9, 0.95, 0.999)),
            "min_p": rng.choice((0.0, 0.0, 0.02, 0.1)), "rows": rng.random() < 0.3}


# ---- inputs ----

def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, dtype = case["kind"], TYPES[case["x"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    state = {"case": case}
    if kind == "norm":
        m, k = case["m"], case["k"]
        # a hidden state has a few channels far larger than the rest
        channels = 1 + 20 * (torch.rand(k, generator=gen, device=DEVICE) < 0.002)
        state["x"] = (normal(m, k) * 0.3).to(dtype)
        state["residual"] = (normal(m, k) * channels).to(dtype) if case["residual"] else None
        state["weight"] = (1 + 0.1 * normal(k)).to(dtype)
    elif kind == "mxquant":
        state["x"] = normal(case["m"], case["k"]).to(dtype)
    elif kind == "mx":
        n, k = case["n"], case["k"]
        state["x"] = normal(case["m"], k).to(dtype)
        codes, exps = _mx_codes(normal(n, k) * 0.02)
        blocks = _mx_blocks(codes, exps)  # as a file stores them
        if own:
            from lloom_b200 import MxMatMul, MxTensor

            state["mat"] = MxMatMul.from_tensor(MxTensor.from_data(blocks, (n, k), DEVICE))
        else:
            state["w"] = blocks
    else:
        b, v = case["b"], case["v"]
        # logits as an output head gives them: a bulk and a few candidates above it
        logits = normal(b, v) * 2.5
        likely = torch.randint(0, v, (b, 24), generator=gen, device=DEVICE)
        logits.scatter_add_(1, likely, 4 + 3 * normal(b, 24).abs())
        state["logits"] = logits.to(dtype)
        state["u"] = torch.rand(b, generator=gen, device=DEVICE)
        settings = {"temperature": case["t"], "top_k": case["top_k"], "top_p": case["top_p"], "min_p": case["min_p"]}
        if case["rows"]:  # every row its own: device tensors
            spread = torch.rand(4, b, generator=gen, device=DEVICE)
            settings = {"temperature": case["t"] * (0.5 + spread[0]),
                        "top_k": ((spread[1] < 0.5) * (1 + spread[1] * 200)).to(torch.int32),
                        "top_p": case["top_p"] * (0.7 + 0.3 * spread[2]),
                        "min_p": case["min_p"] + 0.1 * (spread[3] - 0.5).clamp_min(0)}
        state["settings"] = settings
    return state


# ---- plain forms ----

def _by(a, b):
    """a / b with one rounding (torch multiplies by a reciprocal where one side is a number)."""
    return torch.as_tensor(a, device=DEVICE, dtype=b.dtype).expand_as(b) / b


def _round_half_away(v):
    d = v.double()
    return (d.sign() * (d.abs() + 0.5).floor()).float()


def _q8_values(y, block):
    """What the 8-bit activation blocks of f32 values y stand for."""
    v = y.reshape(*y.shape[:-1], -1, block)
    mag = v.abs()
    amax = mag.amax(-1, keepdim=True)
    if block == 32:  # Q8_0: scale amax / 127, kept in 16 bits
        d = amax / torch.full_like(amax, 127.0)
        inv = torch.where(d != 0, _by(1.0, d), torch.zeros_like(d))
        q = _round_half_away(v * inv)
        d = d.half().float()
    else:  # Q8_K: scaled by the first element of largest magnitude, which becomes -127
        place = torch.arange(block, device=v.device)
        first = torch.where(mag == amax, place, block).amin(-1, keepdim=True)
        inv = _by(-127.0, v.gather(-1, first))
        q = torch.where(amax > 0, _round_half_away(inv * v).clamp(-128, 127), torch.zeros_like(v))
        d = torch.where(amax > 0, _by(1.0, inv), torch.zeros_like(inv))
    return (q * d).reshape(y.shape)


def _plain_norm(case, x, residual, weight):
    h = x.float() if residual is None else (x.float() + residual.float()).to(x.dtype).float()
    ms = h.double().square().sum(-1, keepdim=True) / case["k"]
    inv = (1 / (ms + 1e-5).sqrt()).float()  # 64 bits: the 8-bit codes sit next to borders
    y = h * inv * weight.float()
    y = y.to(x.dtype) if case["out"] == "plain" else _q8_values(y, BLOCK[case["out"]])
    return y if residual is None else (y, h.to(x.dtype))


def _mx_codes(x):
    """E2M1 codes (0 to 15, the sign in bit 3) and the exponents of the scales, a block per 32 values."""
    v = x.float().reshape(*x.shape[:-1], -1, 32)
    amax = v.abs().amax(-1, keepdim=True)
    exps = torch.where(amax > 0, (torch.frexp(amax).exponent - 3).clamp(-127, 127), -127)
    r = torch.ldexp(v.abs(), -exps)
    # borders between neighbouring values; a tie goes to the even code
    code = ((r > 0.25).int() + (r >= 0.75) + (r > 1.25) + (r >= 1.75) + (r > 2.5) + (r >= 3.5) + (r > 5))
    return code + 8 * (v < 0), exps


def _mx_values(codes, exps):
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    return torch.ldexp(table[codes.long()], exps).flatten(-2)


def _mx_blocks(codes, exps):
    """17-byte blocks: the scale's exponent + 127, then elements 0..15 in the low and 16..31 in the high halves of 16 bytes."""
    low, high = codes[..., :16], codes[..., 16:]
    return torch.cat([exps + 127, low + 16 * high], -1).to(torch.uint8).flatten(-2)


def _mx_from_blocks(blocks):
    blk = blocks.reshape(blocks.shape[0], -1, 17).int()
    return _mx_values(torch.cat([blk[..., 1:] & 15, blk[..., 1:] >> 4], -1), blk[..., :1] - 127)


def _per_row(v, b, dtype):
    return torch.as_tensor(v, dtype=dtype, device=DEVICE).expand(b).unsqueeze(1)


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    b, v = logits.shape
    f64 = torch.float64  # a token's probability may be 1e-6, and the draw falls next to its border
    order, at = logits.float().sort(dim=1, descending=True, stable=True)
    order = order.to(f64)
    w = ((order - order[:, :1]) / _per_row(temperature, b, f64)).exp()
    top_k = _per_row(top_k, b, torch.int64)
    rank = torch.arange(v, device=logits.device)
    w = torch.where((rank < top_k) | (top_k == 0), w, 0)
    before = w.cumsum(1) - w
    keep = (before < _per_row(top_p, b, f64) * w.sum(1, keepdim=True)) & (w >= _per_row(min_p, b, f64))
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, at, torch.where(keep, w, 0))
    run_sum = kept.cumsum(1)
    total = run_sum[:, -1:]
    ids = (run_sum <= u.to(f64).unsqueeze(1) * total).sum(1)
    return ids, (kept.gather(1, ids.unsqueeze(1)) / total).squeeze(1).float()


# ---- one pass ----

def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        import lloom_b200 as lb

        if kind == "norm":
            if case["out"] == "plain":
                return lb.rms_norm(state["x"], state["weight"], 1e-5, state["residual"])
            got = lb.rms_norm(state["x"], state["weight"], 1e-5, state["residual"], act_for=getattr(lb.GgmlDType, case["out"]))
            return got.dequantize() if state["residual"] is None else (got[0].dequantize(), got[1])
        if kind == "mxquant":
            return lb.MxTensor.quantize(state["x"]).dequantize()
        if kind == "mx":
            return state["mat"].forward(state["x"])
        return lb.sample(state["logits"], state["u"], **state["settings"])
    if kind == "norm":
        return _plain_norm(case, state["x"], state["residual"], state["weight"])
    if kind == "mxquant":
        return _mx_values(*_mx_codes(state["x"]))
    if kind == "mx":
        return (_mx_values(*_mx_codes(state["x"])) @ _mx_from_blocks(state["w"]).T).to(state["x"].dtype)
    return _plain_sample(state["logits"], state["u"], **state["settings"])


# ---- what a pass cannot do without ----

def work(case):
    kind, size = case["kind"], TYPES[case["x"]].itemsize
    if kind == "norm":
        m, k = case["m"], case["k"]
        out = {"plain": size * k, "Q8_0": k // 32 * 34, "Q4K": k // 256 * 292}[case["out"]]
        return {"bytes": m * (size * k * (3 if case["residual"] else 1) + out) + size * k, "flops": 6 * m * k}
    if kind == "mxquant":
        m, k = case["m"], case["k"]
        return {"bytes": m * (size * k + k // 32 * 17), "flops": 3 * m * k}
    if kind == "mx":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * (k // 32) * 17 + m * (n + k) * size, "flops": 2 * m * n * k}
    return {"bytes": case["b"] * (case["v"] * size + 12), "flops": 10 * case["b"] * case["v"]}


# ---- the definitions in 64 bits ----

def _exact_e2m1(r):
    """Nearest of the eight magnitudes, a tie to the even code."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=r.device)
    hi = torch.searchsorted(grid, r.clamp(max=6.0)).clamp(1, 7)
    to_lo, to_hi = r - grid[hi - 1], grid[hi] - r
    up = (to_hi < to_lo) | ((to_hi == to_lo) & (hi % 2 == 0))
    return torch.where(up, grid[hi], grid[hi - 1])


def _exact_mx(x):
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    for b in range(0, x.shape[-1], 32):
        v = x[:, b:b + 32].double()
        amax = v.abs().amax(1, keepdim=True)
        scale = torch.exp2(torch.floor(torch.log2(amax.clamp_min(1e-300))).clamp_min(-125) - 2)
        out[:, b:b + 32] = v.sign() * _exact_e2m1(v.abs() / scale) * scale
    return out


def _exact_mx_weights(blocks, n, k):
    sign_and_magnitude = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
    table = torch.from_numpy(np.concatenate([sign_and_magnitude, -sign_and_magnitude])).to(blocks.device)
    blk = blocks.view(n, k // 32, 17)
    scale = torch.exp2(blk[:, :, 0].double() - 127).unsqueeze(2)
    w = torch.empty(n, k // 32, 32, dtype=torch.float64, device=blocks.device)
    w[:, :, :16] = table[(blk[:, :, 1:] % 16).long()]
    w[:, :, 16:] = table[(blk[:, :, 1:] // 16).long()]
    return (w * scale).view(n, k)


def _exact_norm(case, x, residual, weight):
    x, weight = x.float().cpu().numpy(), weight.float().cpu().numpy()
    if residual is not None:
        s = torch.from_numpy(x) + residual.float().cpu()
        x = s.to(TYPES[case["x"]]).float().numpy()  # the stream as it is stored
    inv = 1.0 / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-5)
    if case["out"] == "plain":
        y = x * inv * weight
    else:
        # 8-bit codes are defined on values of 32 bits, step by step
        y = (x * inv.astype(np.float32)) * weight
        y = (_exact_q8_0 if case["out"] == "Q8_0" else _exact_q8k)(y.reshape(-1, BLOCK[case["out"]])).reshape(y.shape)
    return y if residual is None else (y, x.astype(np.float64))


def _away(v):
    return np.trunc(v.astype(np.float64) + np.copysign(0.5, v))


def _exact_q8_0(v):
    one = np.float32(1)
    d = np.abs(v).max(1, keepdims=True) / np.float32(127)
    with np.errstate(divide="ignore"):
        inv = np.where(d != 0, one / d, np.float32(0))
    return _away(v * inv) * d.astype(np.float16).astype(np.float64)


def _exact_q8k(v):
    top = np.take_along_axis(v, np.abs(v).argmax(1)[:, None], 1)
    with np.errstate(divide="ignore", invalid="ignore"):
        inv = np.float32(-127) / top
        d = (np.float32(1) / inv).astype(np.float64)
        return np.where(top != 0, np.clip(_away(inv * v), -128, 127) * d, 0.0)


def _exact_sample(case, state):
    logits = state["logits"].double().cpu().numpy()
    b = logits.shape[0]
    s = {k: np.broadcast_to(v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.float64(v), (b,))
         for k, v in state["settings"].items()}
    u = state["u"].double().cpu().numpy()
    ids, probs = np.empty(b, np.int64), np.empty(b)
    for i in range(b):
        rank = np.argsort(-logits[i], kind="stable")
        if s["top_k"][i] > 0:
            rank = rank[:int(s["top_k"][i])]
        w = np.exp((logits[i, rank] - logits[i, rank[0]]) / s["temperature"][i])
        sums = np.cumsum(w.astype(np.longdouble))
        nucleus = int(np.searchsorted(sums, s["top_p"][i] * sums[-1], side="left")) + 1
        length = max(1, min(nucleus, len(w), int((w >= s["min_p"][i]).sum())))
        at = np.sort(rank[:length])
        kept = np.exp((logits[i, at] - logits[i, rank[0]]) / s["temperature"][i]).astype(np.longdouble)
        sums = np.cumsum(kept)
        j = min(int(np.searchsorted(sums, u[i] * sums[-1], side="right")), length - 1)
        ids[i], probs[i] = at[j], float(kept[j] / sums[-1])
    return ids, probs


def exact(case, seed):
    global own
    kept, own = own, False  # the inputs alone
    state = prepare(case, seed)
    own = kept
    kind = case["kind"]
    if kind == "norm":
        return _exact_norm(case, state["x"], state["residual"], state["weight"])
    if kind == "mxquant":
        return _exact_mx(state["x"])
    if kind == "mx":
        return _exact_mx(state["x"]) @ _exact_mx_weights(state["w"], case["n"], case["k"]).T
    return _exact_sample(case, state)
