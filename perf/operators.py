"""Products whose one operand is held in few bits: the cases that are measured, and the operators' plain forms.

  w4_gemm      y = x W^T with W in 4 bits, a scale (and a zero point) for each group of G inputs of an output
  w4_quantize  16-bit weights into that format, and expanded again
  act8_save    activations into 8 bits with a power-of-two exponent for each 32 channels of a token, and restored
  act8_wgrad   the weight gradient of a linear layer, dW = base + X^T dY, from activations held that way

Formats:
  4-bit weights: scales[groups][n] in the 16-bit type of the activations, zeros[groups][n] bytes or none (then 8);
  W[n][k] = scale * (code - zero).  The plain form keeps two codes to a byte, low nibble = even input; the framework packs
  codes in an order of its own.
  8-bit activations: codes[m][pitch] bytes, bit 7 = sign, bits 0-6 = magnitude, pitch = channels rounded up to 16 bytes;
  exponents[m][blocks rounded up to 4] bytes;  X[m][k] = +-magnitude * 2^(exponent - 127), exponent 255 = NaN.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 32  # channels that share an exponent


def listed():
    return [
        # one token through a small projection: the smallest call, where only latency counts
        {"name": "w4_row_2048", "op": "w4_gemm", "m": 1, "n": 2048, "k": 2048, "group": 128, "symmetric": False, "dtype": "f16"},
        # one token through a large square projection: ordinary decoding, bound by the weights' bytes
        {"name": "w4_row_8192", "op": "w4_gemm", "m": 1, "n": 8192, "k": 8192, "group": 128, "symmetric": True, "dtype": "bf16"},
        # a few sequences decoded together, extents that divide by nothing
        {"name": "w4_rows_13_ragged", "op": "w4_gemm", "m": 13, "n": 4099, "k": 5003, "group": 64, "symmetric": False, "dtype": "bf16"},
        # a full decoding batch through an expanding projection, the smallest groups
        {"name": "w4_rows_64", "op": "w4_gemm", "m": 64, "n": 16384, "k": 4096, "group": 32, "symmetric": False, "dtype": "f16"},
        # a prompt: a product bound by the tensor cores
        {"name": "w4_prompt_4096", "op": "w4_gemm", "m": 4096, "n": 8192, "k": 4096, "group": 128, "symmetric": False, "dtype": "bf16"},
        # one layer's weights converted when a model is loaded
        {"name": "w4_quantize_4096", "op": "w4_quantize", "n": 4096, "k": 4096, "group": 128, "symmetric": False, "dtype": "bf16"},
        # a large layer with odd extents
        {"name": "w4_quantize_ragged", "op": "w4_quantize", "n": 8191, "k": 16381, "group": 64, "symmetric": True, "dtype": "f16"},
        # a micro batch of a narrow layer, ragged
        {"name": "act8_save_ragged", "op": "act8_save", "m": 333, "k": 2049, "dtype": "f16"},
        # the activations of a wide layer
        {"name": "act8_save_8192", "op": "act8_save", "m": 8192, "k": 8192, "dtype": "bf16"},
        # a short sequence through a narrow layer: few output tiles, gradient kept in 32 bits
        {"name": "act8_wgrad_1024", "op": "act8_wgrad", "m": 2048, "n": 1024, "k": 1024, "out": "f32", "base": False, "dtype": "f16"},
        # odd extents, gradient rounded to the activations' type
        {"name": "act8_wgrad_ragged", "op": "act8_wgrad", "m": 4099, "n": 2047, "k": 1543, "out": "bf16", "base": False, "dtype": "bf16"},
        # a large layer, added to the gradient of earlier micro batches in 32 bits
        {"name": "act8_wgrad_8192", "op": "act8_wgrad", "m": 16384, "n": 8192, "k": 4096, "out": "f32", "base": True, "dtype": "bf16"},
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["w4_gemm", "w4_gemm", "w4_quantize", "act8_save", "act8_wgrad", "act8_wgrad"])
    dtype = rng.choice(["f16", "bf16"])
    group, symmetric = rng.choice([32, 64, 128]), rng.choice([True, False])
    if op == "w4_gemm":
        n, k = _between(rng, 256, 16384), _between(rng, 256, 16384)
        m = _between(rng, 1, max(1, min(8192, (1 << 37) // (n * k))))
        return {"op": op, "m": m, "n": n, "k": k, "group": group, "symmetric": symmetric, "dtype": dtype}
    if op == "w4_quantize":
        n, k = _between(rng, 256, 16384), _between(rng, 256, 16384)
        n = min(n, (1 << 27) // k)
        return {"op": op, "n": n, "k": k, "group": group, "symmetric": symmetric, "dtype": dtype}
    if op == "act8_save":
        k = _between(rng, 128, 16384)
        return {"op": op, "m": _between(rng, 1, min(65536, (1 << 26) // k)), "k": k, "dtype": dtype}
    n, k = _between(rng, 256, 8192), _between(rng, 256, 8192)
    m = _between(rng, 64, max(64, min(16384, (1 << 38) // (n * k))))
    return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(["f32", dtype]), "base": rng.choice([True, False]), "dtype": dtype}


def _up(x, to):
    return -(-x // to) * to


# ---- the formats in elementary operations


def _power(e):
    """2^e of whole numbers -126 <= e <= 127 in 32 bits, exactly."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _groups(t, size, value=0.0):
    """[rows, cols] -> [rows, groups, size] in 32 bits, the last group filled up with `value`."""
    t = t.float()
    t = torch.nn.functional.pad(t, (0, _up(t.shape[1], size) - t.shape[1]), value=value)
    return t.view(t.shape[0], -1, size)


def _w4_codes(w, group, symmetric):
    """Codes [n, k], scales [n, groups] (of w's type) and zeros [n, groups] of a weight matrix."""
    g = _groups(w, group)
    if symmetric:
        s = (g.abs().amax(2) / 7).to(w.dtype)
        z = torch.full_like(s, 8, dtype=torch.float32)
    else:
        lo, hi = g.amin(2).clamp(max=0), g.amax(2).clamp(min=0)
        s = ((hi - lo) / 15).to(w.dtype)
        z = torch.where(s > 0, torch.round(-lo / s.float()), torch.zeros_like(lo)).clamp(0, 15)
    s32 = s.float()[:, :, None]
    q = torch.where(s32 > 0, torch.round(g / s32), torch.zeros_like(g)) + z[:, :, None]
    return q.clamp(0, 15).view(w.shape[0], -1)[:, : w.shape[1]], s, z


def _w4_values(q, s, z, group):
    """Weights [n, k] in 32 bits that codes [n, k], scales and zeros [n, groups] stand for."""
    g = _groups(q, group)
    return ((g - z.float()[:, :, None]) * s.float()[:, :, None]).view(q.shape[0], -1)[:, : q.shape[1]]


def _w4_pack(q):
    n, k = q.shape
    q = torch.nn.functional.pad(q.to(torch.uint8), (0, 2 * _up(-(-k // 2), 16) - k))
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous()


def _w4_unpack(codes, k):
    return torch.stack([codes & 15, codes >> 4], 2).view(codes.shape[0], -1)[:, :k]


def _act8_codes(x):
    """Bytes [m, k] and exponents [m, blocks] of activations."""
    g = _groups(x, BLOCK)
    amax = g.abs().amax(2)
    low, top = (-24, 9) if x.dtype == torch.float16 else (-126, 120)
    e = torch.frexp(amax)[1] - 1 - 6
    bad = ~torch.isfinite(amax) | (e > top)
    e = torch.where(amax > 0, e.clamp(low, top), torch.full_like(e, low))
    q = torch.round(g.abs() * _power(-e)[:, :, None]).clamp(max=127)
    q = torch.where(torch.isfinite(q), q, torch.zeros_like(q)).to(torch.uint8) | ((g < 0).to(torch.uint8) << 7)
    E = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return q.view(x.shape[0], -1)[:, : x.shape[1]], E


def _act8_values(codes, exponents, k):
    """Activations [m, k] in 32 bits that bytes and exponents stand for."""
    E = exponents[:, : -(-k // BLOCK)].to(torch.int32)
    scale = torch.where(E == 255, torch.full_like(E, math.nan, dtype=torch.float32), _power(E.clamp(1, 254) - 127))
    c = codes[:, :k].to(torch.int32)
    v = _groups(torch.where(c > 127, 128 - c, c), BLOCK) * scale[:, :, None]
    return v.view(codes.shape[0], -1)[:, :k]


# ---- what a program has in hand


def _activations(m, k, dtype, gen):
    """Normal values, a few channels of which are far larger than the others."""
    loud = 1 + 15 * (torch.rand(k, generator=gen, device="cuda") < 0.01)
    return (torch.randn(m, k, generator=gen, device="cuda") * loud).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, op = TYPES[case["dtype"]], case["op"]
    st = {"case": case}
    if op in ("w4_gemm", "w4_quantize"):
        w = (torch.randn(case["n"], case["k"], generator=gen, device="cuda") * case["k"] ** -0.5).to(dtype)
        if op == "w4_quantize":
            st["w"] = w
        else:
            q, s, z = _w4_codes(w, case["group"], case["symmetric"])
            st["scales"] = s.t().contiguous()
            st["zeros"] = None if case["symmetric"] else z.to(torch.uint8).t().contiguous()
            if own:
                from subcuber_b200 import lowbit

                st["weights"] = lowbit.pack_w4(q.to(torch.uint8), st["scales"], st["zeros"], group=case["group"])
                st["workspace"] = lowbit.WorkspaceW4(case["m"], st["weights"])
            else:
                st["codes"] = _w4_pack(q)
            st["x"] = _activations(case["m"], case["k"], dtype, gen)
    else:
        x = _activations(case["m"], case["k"], dtype, gen)
        if op == "act8_save":
            st["x"] = x
        else:
            q, E = _act8_codes(x)
            st["exponents"] = torch.nn.functional.pad(E, (0, _up(E.shape[1], 4) - E.shape[1]), value=1).contiguous()
            st["codes"] = torch.nn.functional.pad(q, (0, _up(case["k"], 16) - case["k"])).contiguous()
            st["dy"] = (torch.randn(case["m"], case["n"], generator=gen, device="cuda") * 0.125).to(dtype)
            st["base"] = torch.randn(case["k"], case["n"], generator=gen, device="cuda").to(TYPES[case["out"]]) if case["base"] else None
            if own:
                from subcuber_b200 import lowbit

                st["saved"] = lowbit.Checkpoint8(st["codes"], st["exponents"], k=case["k"], dtype=dtype)
                st["workspace"] = lowbit.WorkspaceGrad8(st["saved"], case["n"], TYPES[case["out"]])
    return st


def run(st):
    case = st["case"]
    op = case["op"]
    if own:
        from subcuber_b200 import lowbit

        if op == "w4_gemm":
            return lowbit.gemm_w4(st["x"], st["weights"], workspace=st["workspace"])
        if op == "w4_quantize":
            return lowbit.dequantize_w4(lowbit.quantize_w4(st["w"], group=case["group"], symmetric=case["symmetric"]))
        if op == "act8_save":
            return lowbit.restore8(lowbit.save8(st["x"]))
        return lowbit.weight_grad8(st["saved"], st["dy"], base=st["base"], out_dtype=TYPES[case["out"]], workspace=st["workspace"])
    dtype = TYPES[case["dtype"]]
    if op == "w4_gemm":
        s = st["scales"].t()
        z = torch.full_like(s, 8) if st["zeros"] is None else st["zeros"].t()
        w = _w4_values(_w4_unpack(st["codes"], case["k"]), s, z, case["group"])
        return (st["x"].float() @ w.t()).to(dtype)
    if op == "w4_quantize":
        return _w4_values(*_w4_codes(st["w"], case["group"], case["symmetric"]), case["group"]).to(dtype)
    if op == "act8_save":
        return _act8_values(*_act8_codes(st["x"]), case["k"]).to(dtype)
    dw = _act8_values(st["codes"], st["exponents"], case["k"]).t() @ st["dy"].float()
    if st["base"] is not None:
        dw += st["base"].float()
    return dw.to(TYPES[case["out"]])


def work(case):
    op, k = case["op"], case["k"]
    if op in ("w4_gemm", "w4_quantize"):
        n = case["n"]
        held = n * k / 2 + n * -(-k // case["group"]) * (2 if case["symmetric"] else 3)
        if op == "w4_quantize":  # read the weights, write the format; read it, write the values
            return {"bytes": 2 * (2 * n * k + held), "flops": 4 * n * k}
        m = case["m"]
        return {"bytes": held + 2 * m * k + 2 * m * n, "flops": 2 * m * n * k}
    m = case["m"]
    held = m * k + m * -(-k // BLOCK)
    if op == "act8_save":
        return {"bytes": 2 * (2 * m * k + held), "flops": 3 * m * k}
    n = case["n"]
    width = TYPES[case["out"]].itemsize
    return {"bytes": held + 2 * m * n + width * k * n * (2 if case["base"] else 1), "flops": 2 * m * n * k}


# ---- the definitions in 64 bits, written apart from the forms above


def _rounded(t, dtype):
    """Values of 64 bits rounded once to a 16-bit type, as 64 bits."""
    return t.to(dtype).double()


def _step(e):
    """2^e in 64 bits, from its bits."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def exact(case, seed):
    global own
    kept, own = own, False  # the plain codes, whichever side asks
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    op, k = case["op"], case["k"]
    at = torch.arange(k, device="cuda")
    if op == "w4_gemm":
        byte = st["codes"].index_select(1, at // 2).to(torch.int64)
        q = torch.where(at % 2 == 0, byte % 16, byte // 16).double()
        g = at // case["group"]
        z = 8.0 if st["zeros"] is None else st["zeros"].double().index_select(0, g).t()
        return st["x"].double() @ ((q - z) * st["scales"].double().index_select(0, g).t()).t()
    if op == "w4_quantize":
        w, G, dtype = st["w"].double(), case["group"], st["w"].dtype
        out = torch.empty_like(w)
        for first in range(0, k, G):
            part = w[:, first : first + G]
            if case["symmetric"]:
                s = _rounded(part.abs().max(1, keepdim=True).values / 7, dtype)
                z = torch.full_like(s, 8)
            else:
                low = part.min(1, keepdim=True).values.clamp(max=0)
                s = _rounded((part.max(1, keepdim=True).values.clamp(min=0) - low) / 15, dtype)
                z = torch.nan_to_num(torch.round(-low / s), nan=0.0).clamp(0, 15)
            q = (torch.nan_to_num(torch.round(part / s), nan=0.0, posinf=0.0, neginf=0.0) + z).clamp(0, 15)
            out[:, first : first + G] = s * (q - z)
        return out
    if op == "act8_save":
        x = st["x"].double()
        out = torch.empty_like(x)
        low = -24 if st["x"].dtype == torch.float16 else -126
        for first in range(0, k, BLOCK):
            part = x[:, first : first + BLOCK]
            big = part.abs().max(1, keepdim=True).values
            step = _step((torch.frexp(big.clamp(min=1e-300)).exponent - 7).clamp(min=low))
            out[:, first : first + BLOCK] = torch.round(part / step).clamp(-127, 127) * step
        return out
    c = st["codes"][:, :k].to(torch.int64)
    power = _step(st["exponents"].to(torch.int64) - 127).index_select(1, at // BLOCK)
    dw = ((c % 128) * (1 - 2 * (c // 128))).double().mul_(power).t() @ st["dy"].double()
    return dw if st["base"] is None else dw + st["base"].double()
