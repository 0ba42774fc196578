"""Products with one operand held in few bits, on a B200, against plain implementations in 64 bits.

Tolerances.  An output of 16 bits is off by at most half a step, eps / 2 relative, from the sum that was rounded; a sum in
fp32 of terms t_i is off by at most (additions) * 2^-23 * sum |t_i| (every addition, chopped or rounded, is off by at most
one unit of 2^-23 of a partial sum, which sum |t_i| bounds).  A matrix instruction adds 16 terms to its accumulator and
counts for two additions (its own sum of products, and that to the accumulator); a group adds one more for its scale.  Products
with many rows round the weights to 16 bits first: eps / 2 of every term more.  Codes, exponents and restored
activations are compared bit for bit.
"""
import pytest

pytestmark = pytest.mark.gpu

HALF = ["f16", "bf16"]


def T(name):
    import torch

    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def randn(shape, dtype, device, seed, scale=1.0):
    import torch

    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device=device) * scale).to(dtype)


# ------------------------------------------------------------------------------------------------ plain forms, 64 bits
def plain_quantize(w, group, symmetric):
    """codes [n, k], scales and zeros [n, groups], all 64 bits (scales hold values of w's type)."""
    import torch

    n, k = w.shape
    q = torch.empty(n, k, dtype=torch.float64, device=w.device)
    ss, zz = [], []
    for g0 in range(0, k, group):
        p = w[:, g0:g0 + group].double()
        if symmetric:
            r = p.abs().amax(1) / 7
        else:
            lo, hi = p.amin(1).clamp(max=0), p.amax(1).clamp(min=0)
            r = (hi - lo) / 15
        s = r.to(w.dtype).double()
        ok = (s > 0) & torch.isfinite(s)
        safe = torch.where(ok, s, torch.ones_like(s))
        z = torch.full_like(s, 8) if symmetric else torch.where(ok, torch.round(-lo / safe), torch.zeros_like(s)).clamp(0, 15)
        c = torch.where(ok[:, None], torch.round(p / safe[:, None]), torch.zeros_like(p))
        q[:, g0:g0 + group] = (c + z[:, None]).clamp(0, 15)
        ss.append(s)
        zz.append(z)
    return q, torch.stack(ss, 1), torch.stack(zz, 1)


def unpack(w):
    """Codes [n, k] of a WeightsW4, from the documented order."""
    import torch

    n_t, k_b = -(-w.n // 16), -(-w.k // 128)
    words = w.codes.view(torch.int32).view(n_t, k_b, 2, 8, 4, 4)   # tile, block, h, g, t, j
    out = torch.empty(n_t, k_b, 2, 8, 4, 4, 8, dtype=torch.int32, device=w.codes.device)
    for i in range(8):
        out[..., i] = (words >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15
    out = out.permute(0, 2, 3, 1, 5, 4, 6)                         # tile, h, g, block, j, t, i
    return out.reshape(n_t * 16, k_b * 128)[:w.n, :w.k]


def table(t, w):
    """Entries [n, groups] of a table of a WeightsW4, from the documented order."""
    n_t, k_b, per = -(-w.n // 16), -(-w.k // 128), 128 // w.group
    return t.view(n_t, k_b, 16, per).permute(0, 2, 1, 3).reshape(n_t * 16, k_b * per)[:w.n, :-(-w.k // w.group)]


def values(w):
    """Weights [n, k] in 64 bits that a WeightsW4 stands for."""
    import torch

    at = torch.arange(w.k, device=w.codes.device) // w.group
    s = table(w.scales, w).double()[:, at]
    z = 8.0 if w.zeros is None else table(w.zeros, w).double()[:, at]
    return (unpack(w).double() - z) * s


def check_w4_gemm(y, x, w, exact_weights):
    import torch

    wv, xv = values(w), x.double()
    want, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    half = torch.finfo(w.dtype).eps / 2
    sums = (2 * (w.k / 16 + 1) + w.k / 32 + 16) * 2.0 ** -23
    tol = size * (sums + (0 if exact_weights else half)) * (1 + half) + want.abs() * half + torch.finfo(w.dtype).smallest_normal * half * 2
    off = (y.double() - want).abs()
    assert bool((off <= tol).all()), f"{int((off > tol).sum())} of {off.numel()} off, worst {float((off / tol).max()):.2f} x"


def plain_save(x):
    """(codes, exponents, values in 64 bits) of activations."""
    import torch

    m, k = x.shape
    nb = -(-k // 32)
    p = torch.nn.functional.pad(x.double(), (0, nb * 32 - k)).view(m, nb, 32)
    amax = p.abs().amax(2)
    lo, hi = (-24, 9) if x.dtype == torch.float16 else (-126, 120)
    e = torch.frexp(amax).exponent - 7
    bad = ~torch.isfinite(amax) | (e > hi)
    e = torch.where(amax > 0, e.clamp(lo, 200), torch.full_like(e, lo))
    e = torch.where(bad, torch.zeros_like(e), e)
    step = ((e.long() + 1023) << 52).view(torch.float64)
    mag = torch.round(p.abs() / step[..., None]).clamp(max=127)
    mag = torch.where(bad[..., None], torch.zeros_like(mag), mag)
    code = mag.to(torch.int32) | (torch.signbit(p).int() << 7)
    val = torch.where(torch.signbit(p), -mag, mag) * step[..., None]
    val = torch.where(bad[..., None], torch.full_like(val, float("nan")), val)
    E = torch.where(bad, torch.full_like(e, 255), e + 127)
    return code.view(m, -1)[:, :k], E, val.view(m, -1)[:, :k]


def check_grad(dw, xv, dy, base, additions=None):
    """xv: the saved activations' values in 64 bits."""
    import torch

    d = dy.double()
    want, size = xv.t() @ d, xv.abs().t() @ d.abs()
    if base is not None:
        want, size = want + base.double(), size + base.double().abs()
    half = torch.finfo(dw.dtype).eps / 2 if dw.dtype != torch.float32 else 0.0
    n = (2 * (xv.shape[0] / 16 + 1) + 16) if additions is None else additions
    tol = size * n * 2.0 ** -23 * (1 + half) + want.abs() * half + torch.finfo(dw.dtype).smallest_normal * torch.finfo(dw.dtype).eps
    off = (dw.double() - want).abs()
    assert bool((off <= tol).all()), f"{int((off > tol).sum())} of {off.numel()} off, worst {float((off / tol).max()):.2f} x"


# ------------------------------------------------------------------------------------------------ 4-bit weights
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 129), (33, 500), (5, 31), (64, 1024), (40, 515)])
def test_quantize(cuda_device, dtype, symmetric, group, n, k):
    import torch

    from subcuber_b200 import lowbit

    w = randn((n, k), T(dtype), cuda_device, 1, 0.05)
    w[0] = 0                                      # a row of zeros: scale 0
    if n > 4:
        w[3] = w[3].abs()                         # one sign only
        w[4] = -w[4].abs()
    got = lowbit.quantize_w4(w, group=group, symmetric=symmetric)
    q, s, z = plain_quantize(w, group, symmetric)
    assert torch.equal(unpack(got).double(), q)
    assert torch.equal(table(got.scales, got).double(), s)
    if not symmetric:
        assert torch.equal(table(got.zeros, got).double(), z)
    want = values(got).to(w.dtype)
    assert torch.equal(lowbit.dequantize_w4(got), want)


def test_quantize_rows_of_another_matrix(cuda_device):
    """Rows with a pitch, off every vector alignment; an output with a pitch keeps what lies between its rows."""
    import torch

    from subcuber_b200 import lowbit

    big = randn((40, 300), torch.bfloat16, cuda_device, 2)
    w = big[3:36, 7:270]
    got = lowbit.quantize_w4(w, group=64)
    assert torch.equal(unpack(got).double(), plain_quantize(w, 64, False)[0])
    room = torch.full((33, 301), 7.0, dtype=torch.bfloat16, device=cuda_device)
    lowbit.dequantize_w4(got, out=room[:, 5:268])
    assert torch.equal(room[:, 5:268], values(got).to(torch.bfloat16))
    assert bool((room[:, :5] == 7).all()) and bool((room[:, 268:] == 7).all())


@pytest.mark.parametrize("dtype", HALF)
def test_quantize_extremes(cuda_device, dtype):
    import torch

    from subcuber_b200 import lowbit

    fi = torch.finfo(T(dtype))
    w = randn((8, 256), T(dtype), cuda_device, 3)
    w[0] *= fi.smallest_normal * 4                # steps among the subnormal numbers
    w[1] = fi.smallest_normal * fi.eps            # the smallest number: the scale rounds to 0 or to itself
    w[2] = fi.max
    w[3, ::2] = -fi.max / 2
    for symmetric in (True, False):
        got = lowbit.quantize_w4(w, group=128, symmetric=symmetric)
        q, s, _ = plain_quantize(w, 128, symmetric)
        assert torch.equal(table(got.scales, got).double(), s)
        assert torch.equal(unpack(got).double(), q)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_groups_that_are_not_finite_stand_for_nan(cuda_device, symmetric, bad):
    import torch

    from subcuber_b200 import lowbit

    w = randn((20, 256), torch.bfloat16, cuda_device, 4)
    w[7, 130] = bad
    got = lowbit.quantize_w4(w, group=128, symmetric=symmetric)
    back = lowbit.dequantize_w4(got)
    assert bool(torch.isnan(back[7, 128:]).all())
    back[7, 128:] = 0
    assert bool(torch.isfinite(back).all())
    for m in (1, 5, 40, 200):
        x = randn((m, 256), torch.bfloat16, cuda_device, 5)
        y = lowbit.gemm_w4(x, got)
        assert bool(torch.isnan(y[:, 7]).all())
        y[:, 7] = 0
        assert bool(torch.isfinite(y).all())


def test_pack(cuda_device):
    import torch

    from subcuber_b200 import lowbit

    g = torch.Generator(device=cuda_device)
    g.manual_seed(6)
    for n, k, group in ((1, 1, 32), (19, 333, 64), (48, 256, 128)):
        q = torch.randint(0, 16, (n, k), generator=g, device=cuda_device, dtype=torch.uint8)
        scales = randn((-(-k // group), n), torch.float16, cuda_device, 7)
        zeros = torch.randint(0, 16, scales.shape, generator=g, device=cuda_device, dtype=torch.uint8)
        for zz in (zeros, None):
            w = lowbit.pack_w4(q, scales, zz, group=group)
            assert torch.equal(unpack(w), q.int())
            at = torch.arange(k, device=cuda_device) // group
            want = (q.double() - (8.0 if zz is None else zz.double()[at].t())) * scales.double()[at].t()
            assert torch.equal(lowbit.dequantize_w4(w), want.half())
    # rows of a wider matrix of codes
    wide = torch.randint(0, 16, (10, 64), generator=g, device=cuda_device, dtype=torch.uint8)
    w = lowbit.pack_w4(wide[:, 3:40], randn((2, 10), torch.float16, cuda_device, 7), group=32)
    assert torch.equal(unpack(w), wide[:, 3:40].int())


ROWS = [1, 2, 7, 8, 9, 16, 17, 32, 33, 64, 65, 129, 257]


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k,group,symmetric,dtype", [
    (16, 128, 128, True, "f16"), (128, 256, 32, False, "bf16"), (1, 1, 32, False, "f16"), (17, 33, 64, True, "bf16"),
    (250, 1000, 64, False, "f16"), (515, 2047, 128, False, "bf16"), (384, 4096, 32, False, "f16"),
])
def test_gemm_w4(cuda_device, m, n, k, group, symmetric, dtype):
    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((n, k), T(dtype), cuda_device, 8, k ** -0.5), group=group, symmetric=symmetric)
    x = randn((m, k), T(dtype), cuda_device, 9)
    check_w4_gemm(lowbit.gemm_w4(x, w), x, w, exact_weights=False)


@pytest.mark.parametrize("m,n,k,group,symmetric,dtype", [
    (1280, 256, 256, 32, True, "f16"), (1281, 515, 203, 64, False, "bf16"), (1500, 40, 1000, 128, False, "f16"), (4096, 130, 64, 128, True, "bf16"),
    (1300, 1, 1, 32, False, "bf16"),
])
def test_gemm_w4_many_rows(cuda_device, m, n, k, group, symmetric, dtype):
    """From 1280 rows on the weights are expanded once, before the product: the same values, and the same sums."""
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((n, k), T(dtype), cuda_device, 8, k ** -0.5), group=group, symmetric=symmetric)
    x = randn((m, k), T(dtype), cuda_device, 9)
    ws = lowbit.WorkspaceW4(m, w)
    y = lowbit.gemm_w4(x, w, workspace=ws, check=True)
    check_w4_gemm(y, x, w, exact_weights=False)
    # a workspace serves fewer rows too; rows do not depend on the others
    for fewer in (1100, 100, 50, 3):
        part = lowbit.gemm_w4(x[:fewer], w, workspace=ws)
        check_w4_gemm(part, x[:fewer], w, exact_weights=False)
    room = torch.full((m, n + 3), 7.0, dtype=T(dtype), device=cuda_device)
    wide = randn((m, k + 3), T(dtype), cuda_device, 10)[:, 2:2 + k]     # off the 16-byte grid
    lowbit.gemm_w4(wide, w, out=room[:, 1:1 + n])
    check_w4_gemm(room[:, 1:1 + n], wide, w, exact_weights=False)
    assert bool((room[:, :1] == 7).all()) and bool((room[:, 1 + n:] == 7).all())


@pytest.mark.parametrize("m", [1, 5, 24, 40, 150])
@pytest.mark.parametrize("n,k", [(300, 520), (260, 384)])
def test_gemm_w4_rows_of_other_matrices(cuda_device, m, n, k):
    """Activations and results with a pitch, aligned and not; what lies beside and behind the result stays."""
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((n, k), torch.bfloat16, cuda_device, 10, 0.1), group=64)
    for c0, ldx, d0, ldy in ((0, k + 8, 0, n + 4), (3, k + 5, 1, n + 3), (8, k + 16, 8, n + 20)):
        x = randn((m + 2, ldx), torch.bfloat16, cuda_device, 11)[1:1 + m, c0:c0 + k]
        room = torch.full((m + 3, ldy), 7.0, dtype=torch.bfloat16, device=cuda_device)
        lowbit.gemm_w4(x, w, out=room[1:1 + m, d0:d0 + n])
        check_w4_gemm(room[1:1 + m, d0:d0 + n], x, w, exact_weights=False)
        room[1:1 + m, d0:d0 + n] = 7
        assert bool((room == 7).all())


@pytest.mark.parametrize("m", [1, 3, 20, 70, 140])
def test_gemm_w4_keeps_rows_apart(cuda_device, m):
    """An infinity or a NaN among the activations reaches its own row and no other."""
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((70, 300), torch.float16, cuda_device, 12, 0.1), group=32)
    x = randn((m, 300), torch.float16, cuda_device, 13)
    want = lowbit.gemm_w4(x, w)
    hit = m // 2
    for bad in (float("inf"), float("nan"), float("-inf")):
        y = x.clone()
        y[hit, 299] = bad
        got = lowbit.gemm_w4(y, w)
        assert not bool(torch.isfinite(got[hit]).any()) or bool((values(w)[:, 299] == 0).any())
        got[hit] = want[hit]
        assert torch.equal(got, want)


def test_gemm_w4_empty_batch(cuda_device):
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((70, 300), torch.float16, cuda_device, 12))
    assert lowbit.gemm_w4(torch.empty(0, 300, dtype=torch.float16, device=cuda_device), w).shape == (0, 70)


@pytest.mark.parametrize("m", [1, 16, 64, 300])
def test_gemm_w4_same_result_every_time(cuda_device, m):
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((200, 4096), torch.bfloat16, cuda_device, 14, 0.02), group=128)
    x = randn((m, 4096), torch.bfloat16, cuda_device, 15)
    want = lowbit.gemm_w4(x, w)
    for _ in range(20):
        assert torch.equal(lowbit.gemm_w4(x, w), want)


def test_gemm_w4_offsets_past_32_bits(cuda_device):
    """More than 2^32 weights: 2^31 bytes of codes."""
    import torch

    from subcuber_b200 import lowbit

    n, k = 131072 + 37, 32768
    part = lowbit.quantize_w4(randn((16384, k), torch.bfloat16, cuda_device, 16, 0.02), group=128, symmetric=True)
    reps = -(-n // 16384)
    rows = -(-n // 16) * 16
    codes = part.codes.repeat(reps)[: rows * k // 2].clone()
    scales = part.scales.repeat(reps)[: rows * k // 128].clone()
    w = lowbit.WeightsW4(codes, scales, None, n, k, 128)
    tail = randn((37, k), torch.bfloat16, cuda_device, 17, 0.02)      # the last rows differ from the repeated ones
    last = lowbit.quantize_w4(tail, group=128, symmetric=True)
    codes[131072 * k // 2:] = last.codes
    scales[131072 * k // 128:] = last.scales
    for m in (1, 17, 100):
        x = randn((m, k), torch.bfloat16, cuda_device, 18)
        y = lowbit.gemm_w4(x, w)
        check_w4_gemm(y[:, 131072:], x, last, exact_weights=False)
        assert torch.equal(y[:, 114688:131072], y[:, :16384])
    del codes, scales, w
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------ 8-bit activations
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 32), (3, 33), (5, 15), (7, 16), (2, 31), (9, 100), (33, 512), (4, 2049), (300, 640)])
def test_save_and_restore(cuda_device, dtype, m, k):
    import torch

    from subcuber_b200 import lowbit

    x = randn((m, k), T(dtype), cuda_device, 20, 3.0)
    x[0] *= 0.001
    saved = lowbit.save8(x)
    code, E, val = plain_save(x)
    assert torch.equal(saved.codes[:, :k].int(), code)
    assert torch.equal(saved.exponents[:, :E.shape[1]].int(), E)
    back = lowbit.restore8(saved)
    assert torch.equal(back.double(), val)
    step = ((E.long() - 127 + 1023) << 52).view(torch.float64).repeat_interleave(32, 1)[:, :k]
    assert bool(((back.double() - x.double()).abs() <= step).all())


@pytest.mark.parametrize("dtype", HALF)
def test_save_extremes(cuda_device, dtype):
    import torch

    from subcuber_b200 import lowbit

    fi = torch.finfo(T(dtype))
    x = randn((10, 96), T(dtype), cuda_device, 21)
    x[0] = 0
    x[1] = fi.smallest_normal * fi.eps            # the smallest number
    x[2] *= fi.smallest_normal
    x[3] = fi.max if dtype == "f16" else 2.0 ** 126
    x[4] = -x[3]
    x[5, ::3] = -0.0
    x[6, 40] = float("inf")
    x[7, 64] = float("nan")
    x[8, 0] = float("-inf")
    saved = lowbit.save8(x)
    code, E, val = plain_save(x)
    assert torch.equal(saved.exponents[:, :3].int(), E)
    assert torch.equal(saved.codes.int() & 127, code & 127)
    back = lowbit.restore8(saved)
    assert torch.equal(torch.isnan(back), torch.isnan(val))
    assert torch.equal(torch.nan_to_num(back.double()), torch.nan_to_num(val))
    if dtype == "bf16":                           # 2^127 and more have no step whose largest value is finite
        x[3] = fi.max
        assert bool(torch.isnan(lowbit.restore8(lowbit.save8(x))[3]).all())


def test_save_rows_of_another_matrix_into_a_buffer(cuda_device):
    import torch

    from subcuber_b200 import lowbit

    x = randn((50, 333), torch.float16, cuda_device, 22)[4:37, 9:300]
    room = torch.full((40, 512), 9, dtype=torch.uint8, device=cuda_device)
    ex = torch.full((40, 16), 9, dtype=torch.uint8, device=cuda_device)
    out = lowbit.Checkpoint8(room[2:35, :304], ex[2:35, :12], 291, torch.float16)
    lowbit.save8(x, out=out)
    code, E, val = plain_save(x)
    assert torch.equal(out.codes[:, :291].int(), code) and torch.equal(out.exponents[:, :10].int(), E)
    assert bool((room[:2] == 9).all()) and bool((room[35:] == 9).all()) and bool((room[:, 304:] == 9).all())
    assert bool((ex[:2] == 9).all()) and bool((ex[35:] == 9).all()) and bool((ex[:, 10:] == 9).all())
    to = torch.full((33, 300), 7.0, dtype=torch.float16, device=cuda_device)
    lowbit.restore8(out, out=to[:, 4:295])
    assert torch.equal(to[:, 4:295].double(), val) and bool((to[:, :4] == 7).all()) and bool((to[:, 295:] == 7).all())


def test_save_empty(cuda_device):
    import torch

    from subcuber_b200 import lowbit

    saved = lowbit.save8(torch.empty(0, 64, dtype=torch.float16, device=cuda_device))
    assert lowbit.restore8(saved).shape == (0, 64)


GRAD = [(1, 1, 1), (1, 128, 256), (63, 128, 256), (64, 128, 256), (65, 130, 260), (256, 256, 512), (1000, 100, 72), (333, 257, 129),
        (2048, 384, 200), (5000, 64, 640),
        # from 1280 columns on the activations are expanded once, before the product
        (1, 1, 1280), (100, 70, 1280), (333, 257, 1283), (2048, 300, 1500), (70, 33, 4096)]


@pytest.mark.parametrize("dtype,out", [("f16", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("m,k,n", GRAD)
def test_weight_grad(cuda_device, dtype, out, m, k, n):
    from subcuber_b200 import lowbit

    x = randn((m, k), T(dtype), cuda_device, 23, 2.0)
    dy = randn((m, n), T(dtype), cuda_device, 24, 0.1)
    saved = lowbit.save8(x)
    xv = plain_save(x)[2]
    check_grad(lowbit.weight_grad8(saved, dy, out_dtype=T(out)), xv, dy, None)
    base = randn((k, n), T(out), cuda_device, 25)
    got = base.clone()
    lowbit.weight_grad8(saved, dy, base=got, out=got)      # in place
    check_grad(got, xv, dy, base)


@pytest.mark.parametrize("dtype", HALF)
def test_weight_grad_strides(cuda_device, dtype):
    """dY, base and result as parts of wider matrices, aligned and not; what lies beside the result stays."""
    import torch

    from subcuber_b200 import lowbit

    m, k, n = 200, 150, 136
    x = randn((m, k), T(dtype), cuda_device, 26)
    saved = lowbit.save8(x)
    xv = plain_save(x)[2]
    for c0, ld in ((0, n + 8), (8, n + 24), (3, n + 7), (1, n + 1)):
        dy = randn((m, ld), T(dtype), cuda_device, 27)[:, c0:c0 + n]
        base = randn((k, ld), torch.float32, cuda_device, 28)[:, c0:c0 + n]
        room = torch.full((k + 2, ld), 7.0, device=cuda_device)
        lowbit.weight_grad8(saved, dy, base=base, out=room[1:1 + k, c0:c0 + n])
        check_grad(room[1:1 + k, c0:c0 + n], xv, dy, base)
        room[1:1 + k, c0:c0 + n] = 7
        assert bool((room == 7).all())


def test_weight_grad_no_tokens(cuda_device):
    import torch

    from subcuber_b200 import lowbit

    saved = lowbit.save8(torch.empty(0, 70, dtype=torch.float16, device=cuda_device))
    dy = torch.empty(0, 40, dtype=torch.float16, device=cuda_device)
    base = randn((70, 40), torch.float32, cuda_device, 29)
    assert bool((lowbit.weight_grad8(saved, dy) == 0).all())
    assert torch.equal(lowbit.weight_grad8(saved, dy, base=base), base)


def test_weight_grad_not_finite(cuda_device):
    """A token's block that was not finite reaches the rows of its 32 channels only; an infinity in dY its column only."""
    import torch

    from subcuber_b200 import lowbit

    x = randn((100, 128), torch.bfloat16, cuda_device, 30)
    dy = randn((100, 64), torch.bfloat16, cuda_device, 31)
    clean = lowbit.weight_grad8(lowbit.save8(x), dy)
    x[50, 40] = float("inf")
    got = lowbit.weight_grad8(lowbit.save8(x), dy)
    assert bool(torch.isnan(got[32:64]).all())
    got[32:64] = clean[32:64]
    assert torch.equal(got, clean)
    x[50, 40] = 1.0
    saved = lowbit.save8(x)
    clean = lowbit.weight_grad8(saved, dy)
    dy[3, 9] = float("nan")
    got = lowbit.weight_grad8(saved, dy)
    assert bool(torch.isnan(got[:, 9]).all())
    got[:, 9] = clean[:, 9]
    assert torch.equal(got, clean)


def test_weight_grad_extreme_steps(cuda_device):
    """Blocks whose steps lie at both ends of the range, each type's own."""
    import torch

    from subcuber_b200 import lowbit

    for dtype, scales in (("f16", (2.0 ** -24, 2.0 ** -20, 2.0 ** -14, 1.0, 500.0, 15000.0)), ("bf16", (2.0 ** -120, 2.0 ** -60, 1.0, 2.0 ** 60, 2.0 ** 110))):
        for s in scales:
            x = (randn((96, 64), torch.float32, cuda_device, 32).clamp(-4, 4) * s).to(T(dtype))
            dy = randn((96, 48), T(dtype), cuda_device, 33)
            check_grad(lowbit.weight_grad8(lowbit.save8(x), dy), plain_save(x)[2], dy, None)


def test_weight_grad_offsets_past_32_bits(cuda_device):
    """More than 2^31 bytes of codes, and of dY."""
    import torch

    from subcuber_b200 import lowbit

    m, k, n = 262144 + 70, 8192 + 64, 16
    saved = lowbit.Checkpoint8(torch.zeros(m, k, dtype=torch.uint8, device=cuda_device),
                               torch.full((m, 260), 127, dtype=torch.uint8, device=cuda_device), k, torch.bfloat16)
    x = randn((70, k), torch.bfloat16, cuda_device, 34)
    part = lowbit.save8(x)
    saved.codes[262144:] = part.codes
    saved.exponents[262144:, :258] = part.exponents[:, :258]
    dy = torch.zeros(m, n, dtype=torch.bfloat16, device=cuda_device)
    dy[262144:] = randn((70, n), torch.bfloat16, cuda_device, 35)
    check_grad(lowbit.weight_grad8(saved, dy), plain_save(x)[2], dy[262144:], None)
    assert torch.equal(lowbit.restore8(saved)[262144:].double(), plain_save(x)[2])
    del saved
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------------------------ as a user has them
@pytest.mark.parametrize("dtype", HALF)
def test_linear_layer_forward_and_backward(cuda_device, dtype):
    """A linear layer trained with its input saved in 8 bits, then served with its weights in 4 bits.  The gradient is
    checked against the formula and against differences of the loss L = sum(c * (X W))."""
    import torch

    from subcuber_b200 import lowbit, runner

    m, k, n = 192, 256, 128
    x = randn((m, k), T(dtype), cuda_device, 40)
    w = randn((k, n), T(dtype), cuda_device, 41, k ** -0.5)
    kernel = f"blackwell_{dtype}_cubic_2sm_256x256"
    y = runner.gemm(kernel, x, w)
    c = randn((m, n), T(dtype), cuda_device, 42)        # the loss's gradient with respect to y
    saved = lowbit.save8(x)
    del x
    dx = runner.gemm(kernel, c, w.t().contiguous())
    dw = lowbit.weight_grad8(saved, c)
    xv = values_of(saved)
    check_grad(dw, xv, c, None)
    # differences: L is linear in W, so (L(W + h V) - L(W - h V)) / 2h = <dW, V> at any h
    v = randn((k, n), torch.float64, cuda_device, 43)
    loss = lambda weights: (c.double() * (xv @ weights)).sum()
    diff = (loss(w.double() + 0.5 * v) - loss(w.double() - 0.5 * v))
    assert abs(float(diff - (dw.double() * v).sum())) <= 1e-5 * float((dw.double() * v).abs().sum())
    # a second micro batch on top of the first
    saved2 = lowbit.save8(randn((64, k), T(dtype), cuda_device, 44))
    c2 = randn((64, n), T(dtype), cuda_device, 45)
    both = lowbit.weight_grad8(saved2, c2, base=dw)
    check_grad(both, torch.cat([xv, values_of(saved2)]), torch.cat([c, c2]), None)
    # serving: the same weights in 4 bits, a prompt and then one token
    w4 = lowbit.quantize_w4(w.t().contiguous(), group=32)
    for rows in (m, 1):
        x = randn((rows, k), T(dtype), cuda_device, 46)
        check_w4_gemm(lowbit.gemm_w4(x, w4), x, w4, exact_weights=False)
    assert y.shape == (m, n) and dx.shape == (m, k)


def values_of(saved):
    import torch

    k = saved.k
    step = ((saved.exponents[:, :-(-k // 32)].long() - 127 + 1023) << 52).view(torch.float64).repeat_interleave(32, 1)[:, :k]
    c = saved.codes[:, :k].int()
    return torch.where(c > 127, -(c & 127), c).double() * step


@pytest.mark.parametrize("m", [1, 40, 300])
def test_other_stream_and_graphs(cuda_device, m):
    """Calls on a side stream, and two captured graphs (each with its own workspace) replayed at once on two streams."""
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((500, 1024), torch.float16, cuda_device, 50, 0.03))
    xs = [randn((m, 1024), torch.float16, cuda_device, 51 + i) for i in range(2)]
    want = [lowbit.gemm_w4(x, w) for x in xs]
    saved = [lowbit.save8(x) for x in xs]
    grads = [lowbit.weight_grad8(s, y) for s, y in zip(saved, want)]
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    graphs, outs = [], []
    for x, s in zip(xs, streams):
        s.wait_stream(torch.cuda.current_stream(cuda_device))
        ws, gs = lowbit.WorkspaceW4(m, w), lowbit.WorkspaceGrad8(saved[0], 500)
        y = torch.empty(m, 500, dtype=torch.float16, device=cuda_device)
        dw = torch.empty(1024, 500, device=cuda_device)
        cp = lowbit.Checkpoint8(torch.empty_like(saved[0].codes), torch.empty_like(saved[0].exponents), 1024, torch.float16)
        with torch.cuda.stream(s):
            lowbit.gemm_w4(x, w, out=y, workspace=ws)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            lowbit.gemm_w4(x, w, out=y, workspace=ws)
            lowbit.save8(x, out=cp)
            lowbit.weight_grad8(cp, y, out=dw, workspace=gs)
        graphs.append(g)
        outs.append((y, dw, ws, gs, cp))
    for _ in range(10):
        for o in outs:
            o[0].fill_(float("nan"))
            o[1].fill_(float("nan"))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, y, dw in zip(outs, want, grads):
            assert torch.equal(o[0], y) and torch.equal(o[1], dw)


def test_python_refusals(cuda_device):
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((64, 128), torch.float16, cuda_device, 60))
    x = randn((4, 128), torch.float16, cuda_device, 61)
    saved = lowbit.save8(x)
    dy = randn((4, 64), torch.float16, cuda_device, 62)
    bad = [
        lambda: lowbit.gemm_w4(x.bfloat16(), w),
        lambda: lowbit.gemm_w4(x[:, :100], w),
        lambda: lowbit.gemm_w4(x.t(), w),
        lambda: lowbit.gemm_w4(x[0], w),
        lambda: lowbit.gemm_w4(x.cpu(), w),
        lambda: lowbit.gemm_w4(x[:1].expand(4, 128).as_strided((4, 128), (64, 1)), w),
        lambda: lowbit.gemm_w4(x, w, out=torch.empty(4, 63, dtype=torch.float16, device=cuda_device)),
        lambda: lowbit.gemm_w4(x, w, out=torch.empty(4, 64, device=cuda_device)),
        lambda: lowbit.quantize_w4(x.float()),
        lambda: lowbit.quantize_w4(x, group=100),
        lambda: lowbit.pack_w4(x.to(torch.uint8), torch.ones(2, 4, dtype=torch.float16, device=cuda_device)),
        lambda: lowbit.save8(x.float()),
        lambda: lowbit.save8(x, out=lowbit.save8(x[:3])),
        lambda: lowbit.weight_grad8(saved, dy.bfloat16()),
        lambda: lowbit.weight_grad8(saved, dy[:3]),
        lambda: lowbit.weight_grad8(saved, dy[:, :0]),
        lambda: lowbit.weight_grad8(saved, dy, out_dtype=torch.bfloat16),
        lambda: lowbit.weight_grad8(saved, dy, base=torch.zeros(128, 64, dtype=torch.float16, device=cuda_device)),
        lambda: lowbit.weight_grad8(saved, dy, base=torch.zeros(128, 60, device=cuda_device)),
        lambda: lowbit.Checkpoint8(saved.codes[:, :120], saved.exponents, 120, torch.float16),
        lambda: lowbit.WeightsW4(w.codes, w.scales[:8], None, 64, 128, 128),
        lambda: lowbit.WeightsW4(w.codes[:512], w.scales, None, 64, 128, 128),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    small = lowbit.WorkspaceW4(1, w)
    small.nbytes = 0
    with pytest.raises(lowbit.KernelError):
        lowbit.gemm_w4(x, w, workspace=small)


@pytest.mark.parametrize("m", [1, 3, 20, 64])
@pytest.mark.parametrize("n,k,group,symmetric", [(4737, 300, 64, False), (9000, 200, 128, True), (19000, 130, 32, False)])
def test_gemm_w4_many_outputs(cuda_device, m, n, k, group, symmetric):
    """So many outputs that a warp takes two row tiles, and that fewer CTAs (at last one) divide the inputs of 128 rows."""
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((n, k), torch.bfloat16, cuda_device, 70, k ** -0.5), group=group, symmetric=symmetric)
    x = randn((m, k), torch.bfloat16, cuda_device, 71)
    check_w4_gemm(lowbit.gemm_w4(x, w, check=True), x, w, exact_weights=False)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("k", [1, 7, 131, 257])
def test_single_rows_of_odd_length(cuda_device, dtype, k):
    """A single row is taken where it lies, on 16 bytes or off; values behind its end are never used."""
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((40, k), T(dtype), cuda_device, 72, k ** -0.5), group=32)
    for first in (0, 3):
        room = torch.full((1, k + 16), float("nan"), dtype=T(dtype), device=cuda_device)
        x = room[:, first:first + k]
        x.copy_(randn((1, k), T(dtype), cuda_device, 73))
        check_w4_gemm(lowbit.gemm_w4(x, w), x, w, exact_weights=False)
        saved = lowbit.save8(x)
        codes, exps, _ = plain_save(x)
        assert torch.equal(saved.codes[:, :k].int(), codes) and torch.equal(saved.exponents[:, :-(-k // 32)].long(), exps.long())
        check_grad(lowbit.weight_grad8(saved, x), values_of(saved), x, None)
        back = torch.full((1, k + 9), 7.0, dtype=T(dtype), device=cuda_device)
        lowbit.restore8(saved, out=back[:, 1:1 + k])
        assert torch.equal(back[:, 1:1 + k].double(), values_of(saved))
        assert bool((back[:, :1] == 7).all()) and bool((back[:, 1 + k:] == 7).all())


@pytest.mark.parametrize("m", [3, 24, 200])
def test_two_streams_share_the_weights(cuda_device, m):
    """Calls without workspaces on two streams at once, with the same weights and the same saved activations."""
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((900, 512), torch.float16, cuda_device, 74, 0.05))
    xs = [randn((m, 512), torch.float16, cuda_device, 75 + i) for i in range(2)]
    want = [lowbit.gemm_w4(x, w) for x in xs]
    saved = lowbit.save8(xs[0])
    grads = [lowbit.weight_grad8(saved, y) for y in want]
    streams = [torch.cuda.Stream(cuda_device) for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append((lowbit.gemm_w4(xs[i], w), lowbit.weight_grad8(saved, want[i])))
    torch.cuda.synchronize()
    for i in range(2):
        for y, dw in got[i]:
            assert torch.equal(y, want[i]) and torch.equal(dw, grads[i])


def test_status_and_workspace_sizes(cuda_device):
    """`check` passes after good calls of every size; a workspace that is too small is refused, one that is larger serves."""
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((300, 256), torch.bfloat16, cuda_device, 77, 0.06))
    large = lowbit.WorkspaceW4(2000, w)
    for m in (1, 9, 64, 65, 1300):
        x = randn((m, 256), torch.bfloat16, cuda_device, 78)
        y = lowbit.gemm_w4(x, w, check=True)
        assert torch.equal(lowbit.gemm_w4(x, w, workspace=large, check=True), y)
        large.check()
    with pytest.raises(lowbit.KernelError):
        lowbit.gemm_w4(randn((1300, 256), torch.bfloat16, cuda_device, 78), w, workspace=lowbit.WorkspaceW4(64, w))
    for n in (5, 200, 1300):
        dy = randn((70, n), torch.bfloat16, cuda_device, 79)
        saved = lowbit.save8(randn((70, 100), torch.bfloat16, cuda_device, 80))
        dw = lowbit.weight_grad8(saved, dy, check=True)
        check_grad(dw, values_of(saved), dy, None)
        with pytest.raises(lowbit.KernelError):
            lowbit.weight_grad8(saved, dy, workspace=lowbit.WorkspaceW4(1, w))


@pytest.mark.parametrize("m", [9, 16, 33, 64])
@pytest.mark.parametrize("n,k,group", [(1, 1100, 64), (3, 2048, 128), (125, 1030, 32), (130, 2048, 64), (515, 4096, 128), (4097, 512, 32)])
def test_gemm_w4_last_outputs_of_a_cluster(cuda_device, m, n, k, group):
    """CTAs that divide the inputs of 128 outputs, the last of which are not there: results equal those of the same weights
    with whole 128 outputs, which run in the same clusters, and what lies beside the result stays."""
    import torch

    from subcuber_b200 import lowbit

    full = randn((-(-n // 128) * 128, k), torch.bfloat16, cuda_device, 81, k ** -0.5)
    x = randn((m, k), torch.bfloat16, cuda_device, 82)
    want = lowbit.gemm_w4(x, lowbit.quantize_w4(full, group=group), check=True)
    w = lowbit.quantize_w4(full[:n], group=group)
    room = torch.full((m + 2, n + 3), 7.0, dtype=torch.bfloat16, device=cuda_device)
    for _ in range(5):
        room[1:1 + m, 1:1 + n] = 0
        lowbit.gemm_w4(x, w, out=room[1:1 + m, 1:1 + n], check=True)
        assert torch.equal(room[1:1 + m, 1:1 + n], want[:, :n])
    room[1:1 + m, 1:1 + n] = 7
    assert bool((room == 7).all())


@pytest.mark.parametrize("m,n,k", [(20, 300, 2048), (64, 128, 4096), (16, 19000, 256), (100, 300, 2048), (1300, 300, 512)])
def test_gemm_w4_waits_that_run_out_are_reported(cuda_device, m, n, k):
    """Tiles that are never announced: every role gives up within the (shortened) limit, the call says so, and the next call on
    the same device is right.  One CTA and clusters, the products on the way and in two passes."""
    import torch

    from subcuber_b200 import lowbit, runner

    w = lowbit.quantize_w4(randn((n, k), torch.float16, cuda_device, 83, k ** -0.5))
    x = randn((m, k), torch.float16, cuda_device, 84)
    want = lowbit.gemm_w4(x, w, check=True)
    ws = lowbit.WorkspaceW4(m, w)
    opts = runner.options(wait_limit_us=1000, drop_split_flags=True)
    for kw in (dict(check=True), dict(check=True, workspace=ws)):
        with pytest.raises(lowbit.KernelError) as exc:
            lowbit.gemm_w4(x, w, opts=opts, **kw)
        assert exc.value.code in (101, 102, 103, 104)
    lowbit.gemm_w4(x, w, opts=opts, workspace=ws)
    with pytest.raises(lowbit.KernelError):
        ws.check()
    assert torch.equal(lowbit.gemm_w4(x, w, workspace=ws, check=True, opts=runner.options(wait_limit_us=1000000)), want)
    ws.check()


@pytest.mark.parametrize("m,k,n", [(500, 300, 200), (64, 128, 256), (500, 300, 1300)])
def test_weight_grad_waits_that_run_out_are_reported(cuda_device, m, k, n):
    import torch

    from subcuber_b200 import lowbit, runner

    saved = lowbit.save8(randn((m, k), torch.bfloat16, cuda_device, 85))
    dy = randn((m, n), torch.bfloat16, cuda_device, 86)
    want = lowbit.weight_grad8(saved, dy, check=True)
    opts = runner.options(wait_limit_us=1000, drop_split_flags=True)
    with pytest.raises(lowbit.KernelError) as exc:
        lowbit.weight_grad8(saved, dy, check=True, opts=opts)
    assert exc.value.code in (101, 102, 103, 104)
    assert torch.equal(lowbit.weight_grad8(saved, dy, check=True), want)


def test_rows_without_waits_take_options(cuda_device):
    import torch

    from subcuber_b200 import lowbit, runner

    w = lowbit.quantize_w4(randn((300, 512), torch.float16, cuda_device, 87, 0.05))
    x = randn((3, 512), torch.float16, cuda_device, 88)
    opts = runner.options(wait_limit_us=1000, drop_split_flags=True)
    assert torch.equal(lowbit.gemm_w4(x, w, check=True, opts=opts), lowbit.gemm_w4(x, w))
    with pytest.raises(lowbit.KernelError):
        lowbit.gemm_w4(x, w, opts=runner.options(sm_limit=8))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("k", [5, 40, 131, 200])
def test_inputs_behind_the_last_stand_for_zero(cuda_device, k, group):
    """Codes and scales of another quantiser whose values are finite, but would not be with a code of 8 behind the last input."""
    import torch

    from subcuber_b200 import lowbit

    groups = -(-k // group)
    q = torch.ones(20, k, dtype=torch.uint8, device=cuda_device)
    scales = torch.full((groups, 20), 20000.0, dtype=torch.float16, device=cuda_device)
    for zero in (0, 3, 15):
        q.fill_(min(zero + 1, 15) if zero < 15 else 14)
        zeros = torch.full((groups, 20), zero, dtype=torch.uint8, device=cuda_device)
        w = lowbit.pack_w4(q, scales, zeros, group=group)
        assert bool(torch.isfinite(lowbit.dequantize_w4(w)).all())
        for m in (1, 9, 40, 100, 1300):
            x = randn((m, k), torch.float16, cuda_device, 89, 2.0 ** -10)
            check_w4_gemm(lowbit.gemm_w4(x, w), x, w, exact_weights=False)


def test_gemm_w4_more_inputs_than_half_of_31_bits(cuda_device):
    """More than 2^30 inputs: what copies count in, and where the last inputs of 9 and 65 rows are found."""
    import torch

    from subcuber_b200 import lowbit

    k, n, last = (1 << 30) + 384, 16, 1000
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(cuda_device)[0] < 165 << 30:
        pytest.skip("needs 165 GB of free device memory")
    tail = lowbit.quantize_w4(randn((n, 1024), torch.float16, cuda_device, 90, 0.05), group=128, symmetric=True)
    codes = torch.full((n * k // 2,), 0x88, dtype=torch.uint8, device=cuda_device)          # zeros
    scales = torch.ones(n * k // 128, dtype=torch.float16, device=cuda_device)
    codes[-tail.codes.numel():] = tail.codes
    scales[-tail.scales.numel():] = tail.scales
    w = lowbit.WeightsW4(codes, scales, None, n, k, 128)
    x = torch.zeros(65, k, dtype=torch.float16, device=cuda_device)
    x[:, -last:] = randn((65, last), torch.float16, cuda_device, 91)
    for m in (65, 9, 1):
        y = lowbit.gemm_w4(x[:m], w, check=True)
        check_w4_gemm(y, x[:m, -1024:], tail, exact_weights=False)
    del x, codes, scales, w
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m", [9, 16, 64])
def test_gemm_w4_long_sums_of_many_outputs(cuda_device, m):
    """A large term first, its negative last, small ones between: an accumulator that chops loses about two units in the last place of
    the large term with each addition (eight for 128 inputs).  It takes 16384 inputs, so that 1024 of the 8192 additions meet the
    large term; with all of them the sum was off by 2.25."""
    import torch

    from subcuber_b200 import lowbit

    n, k = 149 * 128, 131072
    q = torch.full((n, k), 9, dtype=torch.uint8, device=cuda_device)
    w = lowbit.pack_w4(q, torch.ones(k // 128, n, dtype=torch.float16, device=cuda_device), group=128)    # ones
    del q
    g = torch.Generator(device=cuda_device)
    g.manual_seed(92)
    x = ((torch.rand(m, k, generator=g, device=cuda_device) + 1) * 2.0 ** -10).half()
    want = x[:, 1:-1].double().sum(1, keepdim=True)
    x[:, 0], x[:, -1] = 1024, -1024
    y = lowbit.gemm_w4(x, w, check=True).double()
    unit = 2.0 ** (10 - 23)                                    # of sums from 1024 to 2048
    assert float(want.max()) < 1024
    tol = 2 * 1024 * unit + 8192 * 2 * 2.0 ** -23 * 256 / 8 + 16 * unit + want * 2.0 ** -11   # large, small terms, join, rounding
    assert bool(((y - want).abs() <= tol).all()), f"worst {float(((y - want).abs() / tol).max()):.2f} x"


def _strict_bound(x, wv, k, dtype):
    """The product with weights wv (64 bits), and how far a sum of exact products may be from it: the additions, and half a step of
    the result.  Nothing for a rounding of the weights."""
    import torch

    xv = x.double()
    want, size = xv @ wv.t(), xv.abs() @ wv.abs().t()
    half = torch.finfo(dtype).eps / 2
    sums = (2 * (k / 16 + 1) + k / 32 + 16) * 2.0 ** -23
    return want, size * sums * (1 + half) + want.abs() * half + torch.finfo(dtype).smallest_normal * half * 2


@pytest.mark.parametrize("m", [1, 2, 5, 8])
@pytest.mark.parametrize("n,k,group,symmetric,dtype", [
    (16, 128, 128, True, "f16"), (128, 256, 32, False, "bf16"), (17, 33, 64, True, "bf16"), (250, 1000, 64, False, "f16"),
    (515, 260, 128, False, "bf16"), (384, 512, 32, True, "f16"), (5000, 200, 64, False, "bf16"),
])
def test_gemm_w4_few_rows_have_exact_weights(cuda_device, m, n, k, group, symmetric, dtype):
    """Up to 8 rows codes are multiplied exactly and scales applied in 32 bits.  A product with weights rounded to 16 bits, in 64
    bits otherwise, would not pass."""
    import torch

    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((n, k), T(dtype), cuda_device, 93, k ** -0.5), group=group, symmetric=symmetric)
    x = randn((m, k), T(dtype), cuda_device, 94)
    want, tol = _strict_bound(x, values(w), k, w.dtype)
    off = (lowbit.gemm_w4(x, w).double() - want).abs()
    assert bool((off <= tol).all()), f"{int((off > tol).sum())} of {off.numel()} off, worst {float((off / tol).max()):.2f} x"
    if m * n >= 500:
        rounded = (x.double() @ lowbit.dequantize_w4(w).double().t()).to(w.dtype).double()
        assert bool(((rounded - want).abs() > tol).any())


@pytest.mark.parametrize("m", [9, 16, 17, 33, 64, 65, 129, 257, 1280])
@pytest.mark.parametrize("n,k,group,symmetric,dtype", [
    (16, 128, 128, True, "f16"), (128, 256, 32, False, "bf16"), (1, 1, 32, False, "f16"), (17, 33, 64, True, "bf16"),
    (250, 1000, 64, False, "f16"), (515, 2047, 128, False, "bf16"), (384, 4096, 32, False, "f16"), (19100, 520, 64, False, "f16"),
])
def test_gemm_w4_more_rows_multiply_what_dequantize_gives(cuda_device, m, n, k, group, symmetric, dtype):
    """From 9 rows on the weights are those that dequantize_w4 gives (checked bit for bit above), and their products are exact."""
    from subcuber_b200 import lowbit

    w = lowbit.quantize_w4(randn((n, k), T(dtype), cuda_device, 95, k ** -0.5), group=group, symmetric=symmetric)
    x = randn((m, k), T(dtype), cuda_device, 96)
    want, tol = _strict_bound(x, lowbit.dequantize_w4(w).double(), k, w.dtype)
    off = (lowbit.gemm_w4(x, w).double() - want).abs()
    assert bool((off <= tol).all()), f"{int((off > tol).sum())} of {off.numel()} off, worst {float((off / tol).max()):.2f} x"


@pytest.mark.parametrize("m", [1, 17, 100])
def test_gemm_w4_every_input_counts(cuda_device, m):
    """One row at a time, a single input of x that is not zero: each result is one weight times 1, exactly."""
    import torch

    from subcuber_b200 import lowbit

    n, k = 300, 32768 - 77
    w = lowbit.quantize_w4(randn((n, k), torch.bfloat16, cuda_device, 97, 0.05), group=128)
    wv = lowbit.dequantize_w4(w) if m > 8 else values(w).bfloat16()
    for first in (0, 127, 16384, k - m):
        x = torch.zeros(m, k, dtype=torch.bfloat16, device=cuda_device)
        at = torch.arange(m, device=cuda_device)
        x[at, first + at] = 1
        assert torch.equal(lowbit.gemm_w4(x, w), wv[:, first:first + m].t())
