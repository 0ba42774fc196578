"""Products with one operand held in few bits, host side: argument checks of the C entry points and of the Python calls.
Nothing here launches a kernel (the checks come before any CUDA call)."""
import pytest

P = 1 << 20  # stands for a device address with every alignment; never dereferenced
WS = 1 << 40  # more workspace than any call asks for


def _w4_gemm(lib, dtype=0, x=P, ldx=256, codes=P, scales=P, zeros=P, y=P, ldy=64, m=1, n=64, k=256, group=128, ws=P, nbytes=WS):
    return lib.sb200_w4_gemm(dtype, x, ldx, codes, scales, zeros, y, ldy, m, n, k, group, ws, nbytes, None)


@pytest.mark.parametrize("change,rc", [
    (dict(m=0), 0),                                   # an empty batch: nothing to do
    (dict(m=0, x=None, y=None, ws=None), 0),
    (dict(m=-1), 4), (dict(n=0), 4), (dict(k=0), 4), (dict(n=-5), 4),
    (dict(x=None), 4), (dict(codes=None), 4), (dict(scales=None), 4), (dict(y=None), 4),
    (dict(ldx=255), 4), (dict(ldy=63), 4),
    (dict(dtype=1), 5), (dict(dtype=2), 5), (dict(dtype=7), 5),
    (dict(group=0), 5), (dict(group=16), 5), (dict(group=96), 5), (dict(group=256), 5),
    (dict(x=P + 1), 1), (dict(y=P + 1), 1), (dict(codes=P + 8), 1), (dict(scales=P + 1), 1),
    (dict(n=(1 << 31) - 1, ldy=1 << 31), 5), (dict(k=(1 << 31) - 1, ldx=1 << 31), 5), (dict(m=(1 << 31) - 1), 5),
    (dict(ws=None), 6), (dict(nbytes=0), 6), (dict(ws=P + 16), 6),
    (dict(m=65, nbytes=256), 6), (dict(m=9, k=255, ldx=255, nbytes=256), 6),    # parts of the sums, a copy of x
])
def test_w4_gemm_refuses(lib, change, rc):
    assert _w4_gemm(lib, **change) == rc


def test_w4_sizes(lib):
    assert lib.sb200_w4_codes_bytes(16, 128) == 1024 and lib.sb200_w4_codes_bytes(17, 129) == 4096
    assert lib.sb200_w4_codes_bytes(1, 1) == 1024 and lib.sb200_w4_codes_bytes(0, 5) == 0
    assert lib.sb200_w4_codes_bytes(1 << 20, 1 << 15) == 1 << 34   # offsets pass 32 bits
    assert lib.sb200_w4_table_entries(1, 1, 128) == 16 and lib.sb200_w4_table_entries(17, 129, 32) == 32 * 8
    assert lib.sb200_w4_table_entries(17, 129, 48) == 0 and lib.sb200_w4_table_entries(0, 1, 32) == 0


@pytest.mark.parametrize("args,rc", [
    ((0, None, 64, 8, 64, 32, P, P, P), 4), ((0, P, 63, 8, 64, 32, P, P, P), 4), ((1, P, 64, 8, 64, 32, P, P, P), 5),
    ((0, P, 64, 8, 64, 48, P, P, P), 5), ((0, P + 1, 64, 8, 64, 32, P, P, P), 1), ((0, P, 64, 0, 64, 32, P, P, P), 4),
    ((3, P, 64, 8, 64, 32, P + 4, P, None), 1), ((3, P, 64, 8, 64, 32, P, None, None), 4),
])
def test_w4_quantize_refuses(lib, args, rc):
    assert lib.sb200_w4_quantize(*args, None) == rc


def test_w4_pack_and_dequantize_refuse(lib):
    pack = lambda dtype=0, q=P, ldq=8, s=P, lds=4, z=P, ldz=4, n=4, k=8, group=32, codes=P, scales=P, zeros=P: lib.sb200_w4_pack(
        dtype, q, ldq, s, lds, z, ldz, n, k, group, codes, scales, zeros, None)
    assert pack(q=None) == 4 and pack(ldq=7) == 4 and pack(s=None) == 4 and pack(lds=3) == 4 and pack(ldz=3) == 4
    assert pack(z=None) == 4 and pack(zeros=None) == 4 and pack(n=0) == 4 and pack(scales=None) == 4
    assert pack(codes=P + 1) == 1 and pack(scales=P + 4) == 1 and pack(zeros=P + 2) == 1 and pack(s=P + 1) == 1
    assert pack(dtype=1) == 5 and pack(group=16) == 5
    assert lib.sb200_w4_dequantize(0, P, P, None, 4, 8, 32, None, 8, None) == 4
    assert lib.sb200_w4_dequantize(0, P, P, None, 4, 8, 32, P, 7, None) == 4
    assert lib.sb200_w4_dequantize(1, P, P, None, 4, 8, 32, P, 8, None) == 5
    assert lib.sb200_w4_dequantize(0, P, P, None, 4, 8, 32, P + 1, 8, None) == 1


def _save(lib, dtype=0, x=P, ldx=100, m=4, k=100, codes=P, pitch=112, exps=P, exp_pitch=4):
    return lib.sb200_act8_save(dtype, x, ldx, m, k, codes, pitch, exps, exp_pitch, None)


def _restore(lib, dtype=0, x=P, ldx=100, m=4, k=100, codes=P, pitch=112, exps=P, exp_pitch=4):
    return lib.sb200_act8_restore(dtype, codes, pitch, exps, exp_pitch, m, k, x, ldx, None)


@pytest.mark.parametrize("call", [_save, _restore])
@pytest.mark.parametrize("change,rc", [
    (dict(m=0), 0), (dict(m=0, x=None, codes=None, exps=None), 0),
    (dict(m=-1), 4), (dict(k=0), 4), (dict(x=None), 4), (dict(codes=None), 4), (dict(exps=None), 4),
    (dict(ldx=99), 4), (dict(pitch=96), 4), (dict(exp_pitch=0), 4), (dict(k=129, ldx=129, pitch=144), 4),
    (dict(dtype=1), 5), (dict(dtype=2), 5),
    (dict(x=P + 1), 1), (dict(codes=P + 8), 1), (dict(pitch=104), 1), (dict(exps=P + 2), 1), (dict(exp_pitch=6), 1),
])
def test_act8_save_and_restore_refuse(lib, call, change, rc):
    assert call(lib, **change) == rc


def _wgrad(lib, dtype=0, codes=P, pitch=112, exps=P, exp_pitch=4, dy=P, lddy=24, out_dtype=1, base=None, ldbase=24, dw=P,
           lddw=24, m=4, n=24, k=100, ws=P, nbytes=WS):
    return lib.sb200_act8_wgrad(dtype, codes, pitch, exps, exp_pitch, dy, lddy, out_dtype, base, ldbase, dw, lddw, m, n, k, ws,
                                nbytes, None)


@pytest.mark.parametrize("change,rc", [
    (dict(m=-1), 4), (dict(n=0), 4), (dict(k=0), 4), (dict(codes=None), 4), (dict(exps=None), 4), (dict(dy=None), 4),
    (dict(dw=None), 4), (dict(lddy=23), 4), (dict(lddw=23), 4), (dict(base=P, ldbase=23), 4), (dict(pitch=96), 4),
    (dict(dtype=1), 5), (dict(out_dtype=3), 5), (dict(dtype=3, out_dtype=0), 5), (dict(out_dtype=2), 5),
    (dict(codes=P + 8), 1), (dict(exps=P + 2), 1), (dict(dy=P + 1), 1), (dict(dw=P + 2), 1), (dict(base=P + 2), 1),
    (dict(exp_pitch=1 << 31), 5), (dict(n=(1 << 31) - 1, lddy=1 << 31, lddw=1 << 31), 5),
    (dict(ws=None), 6), (dict(nbytes=0), 6), (dict(ws=P + 128), 6),
])
def test_act8_wgrad_refuses(lib, change, rc):
    assert _wgrad(lib, **change) == rc


def test_workspaces_grow_with_the_rows(lib):
    """A workspace for m rows serves every smaller m, whatever kernel that takes."""
    for aligned in (0, 1):
        w4 = [lib.sb200_w4_gemm_workspace_bytes(0, m, 1000, 500, 64, aligned) for m in (1, 8, 9, 64, 65, 500, 1279, 1280, 5000)]
        assert w4 == sorted(w4) and w4[0] >= 256 and (aligned or w4[0] > 256)
        g8 = [lib.sb200_act8_wgrad_workspace_bytes(3, 1, m, 1500, 300, aligned) for m in (0, 1, 64, 1000, 100000)]
        assert g8 == sorted(g8) and g8[0] >= 256
    assert lib.sb200_w4_gemm_workspace_bytes(0, 1, 1000, 512, 64, 1) == 256


def test_python_calls_refuse_host_tensors():
    import torch

    from subcuber_b200 import lowbit

    h = torch.zeros(16, 128, dtype=torch.float16)
    for call in (lambda: lowbit.quantize_w4(h), lambda: lowbit.save8(h),
                 lambda: lowbit.pack_w4(h.to(torch.uint8), torch.zeros(1, 16, dtype=torch.float16))):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()


def test_python_handles_refuse_wrong_tables():
    """The handles check shapes, types and devices before anything is launched (with meta tensors in place of device ones)."""
    import torch

    from subcuber_b200 import lowbit

    codes = torch.zeros(1024, dtype=torch.uint8)
    scales = torch.zeros(1, 16, dtype=torch.float16)
    with pytest.raises(ValueError):
        lowbit.WeightsW4(codes, scales, None, 16, 128, 128)     # host tensors
    with pytest.raises(ValueError):
        lowbit.WeightsW4(codes, scales, None, 16, 128, 48)
    with pytest.raises(ValueError):
        lowbit.WeightsW4(codes, scales, None, 0, 128, 128)
    with pytest.raises(ValueError):
        lowbit.Checkpoint8(codes.view(8, 128), codes.view(8, 128), 100, torch.float32)
    with pytest.raises(ValueError):
        lowbit.Checkpoint8(codes.view(8, 128), codes.view(8, 128), 0, torch.float16)


class _OnDevice:
    """What the Python calls ask of a tensor, on a device that need not be there."""
    is_cuda = True

    def __init__(self, index, dtype, *shape):
        import torch

        self.device, self.dtype, self.shape = torch.device("cuda", index), dtype, shape

    def dim(self):
        return 2

    def stride(self, axis=None):
        return (self.shape[1], 1) if axis is None else (self.shape[1], 1)[axis]

    def data_ptr(self):
        return P


def test_python_products_refuse_operands_on_different_devices(monkeypatch):
    """Each operand on another device than the others, with and without an `out`."""
    import torch

    from subcuber_b200 import lowbit

    def launched(*args):
        raise AssertionError("the call reached the library")

    monkeypatch.setattr(lowbit, "_call", launched)
    H, F = torch.float16, torch.float32
    w = lowbit.WeightsW4.__new__(lowbit.WeightsW4)
    w._set(64, 128, 128, H, torch.device("cuda", 0), P, P, None)
    w._status_ptr = P
    saved = lowbit.Checkpoint8.__new__(lowbit.Checkpoint8)
    saved._set(4, 128, H, torch.device("cuda", 0), P, 128, P, 4)

    class Room:
        nbytes = WS
        _for = lowbit._Workspace._for

        def __init__(self, index):
            self.device, self.ptr = torch.device("cuda", index), P

    on = _OnDevice
    for call in (
        lambda: lowbit.gemm_w4(on(1, H, 4, 128), w),
        lambda: lowbit.gemm_w4(on(1, H, 4, 128), w, out=on(0, H, 4, 64)),
        lambda: lowbit.gemm_w4(on(0, H, 4, 128), w, out=on(1, H, 4, 64)),
        lambda: lowbit.gemm_w4(on(0, H, 4, 128), w, out=on(0, H, 4, 64), workspace=Room(1)),
        lambda: lowbit.dequantize_w4(w, out=on(1, H, 64, 128)),
        lambda: lowbit.save8(on(1, H, 4, 128), out=saved),
        lambda: lowbit.restore8(saved, out=on(1, H, 4, 128)),
        lambda: lowbit.weight_grad8(saved, on(1, H, 4, 64), workspace=Room(0)),
        lambda: lowbit.weight_grad8(saved, on(1, H, 4, 64), out=on(0, F, 128, 64), workspace=Room(0)),
        lambda: lowbit.weight_grad8(saved, on(0, H, 4, 64), out=on(1, F, 128, 64), workspace=Room(0)),
        lambda: lowbit.weight_grad8(saved, on(0, H, 4, 64), base=on(1, F, 128, 64), out=on(0, F, 128, 64), workspace=Room(0)),
        lambda: lowbit.weight_grad8(saved, on(0, H, 4, 64), out=on(0, F, 128, 64), workspace=Room(1)),
    ):
        with pytest.raises(ValueError, match="device|workspace is on"):
            call()
    with pytest.raises(AssertionError):
        lowbit.gemm_w4(on(0, H, 4, 128), w, out=on(0, H, 4, 64), workspace=Room(0))
    with pytest.raises(ValueError):
        lowbit.WorkspaceGrad8(saved, 64, torch.bfloat16)


@pytest.mark.parametrize("options,rc", [(dict(sm_limit=4), 5), (dict(no_split=1), 5), (dict(wait_limit_us=1000, drop_split_flags=1), 0), (None, 0)])
def test_products_take_the_options_of_waits_only(lib, options, rc):
    import ctypes as C

    from subcuber_b200 import _lib

    o = None if options is None else C.byref(_lib.GemmOptions(**options))
    assert lib.sb200_w4_gemm_opt(0, P, 256, P, P, P, P, 64, 0, 64, 256, 128, P, WS, None, o) == rc       # no rows: nothing runs
    got = lib.sb200_act8_wgrad_opt(0, P, 112, P, 4, P, 24, 1, None, 24, P, 24, 4, 24, 100, None, WS, None, o)
    assert got == (rc or 6)                                                                              # no workspace


def test_python_calls_refuse_extents_past_32_bits(monkeypatch):
    """Counts that ctypes would cut to 32 bits (2^32 tokens to none, 2^32 + 5 to five) are refused, wherever they come from."""
    import torch

    from subcuber_b200 import lowbit

    def launched(*args):
        raise AssertionError("the call reached the library")

    monkeypatch.setattr(lowbit, "_call", launched)
    monkeypatch.setattr(lowbit.WeightsW4, "_empty", launched)
    monkeypatch.setattr(lowbit.Checkpoint8, "_empty", launched)
    H, U, on = torch.float16, torch.uint8, _OnDevice
    w = lowbit.WeightsW4.__new__(lowbit.WeightsW4)
    w._set(64, 128, 128, H, torch.device("cuda", 0), P, P, None)
    w._status_ptr = P
    for many in (1 << 32, (1 << 32) + 5, (1 << 31) - 1):
        saved = lowbit.Checkpoint8.__new__(lowbit.Checkpoint8)
        saved._set(many, 128, H, torch.device("cuda", 0), P, 128, P, 4)
        for call in (
            lambda: lowbit.gemm_w4(on(0, H, many, 128), w, out=on(0, H, many, 64)),
            lambda: lowbit.quantize_w4(on(0, H, many, 128)),
            lambda: lowbit.quantize_w4(on(0, H, 16, many)),
            lambda: lowbit.pack_w4(on(0, U, many, 128), on(0, H, 1, many)),
            lambda: lowbit.save8(on(0, H, many, 128)),
            lambda: lowbit.save8(on(0, H, 4, many)),
            lambda: lowbit.save8(on(0, H, many, 128), out=saved),
            lambda: lowbit.restore8(saved, out=on(0, H, many, 128)),
            lambda: lowbit.weight_grad8(saved, on(0, H, many, 64)),
            lambda: lowbit.WorkspaceW4(many, w),
            lambda: lowbit.WorkspaceW4(-1, w),
            lambda: lowbit.WorkspaceGrad8(saved, many),
            lambda: lowbit.WeightsW4(on(0, U, 1, 1), on(0, H, 1, 1), None, many, 128, 128),
            lambda: lowbit.WeightsW4(on(0, U, 1, 1), on(0, H, 1, 1), None, 16, many, 128),
        ):
            with pytest.raises(ValueError, match=str(many) + "|-1"):
                call()


def test_checked_products_have_a_status_word_of_their_own(monkeypatch):
    """Two checked calls at once with the same weights: the second must not clear what the first will read."""
    import torch

    from subcuber_b200 import lowbit

    class Reached(Exception):
        pass

    words = []

    def call(what, device, *args):
        words.append(args[-2])
        raise Reached

    class Room:
        nbytes = 256

        def __init__(self, m, w, aligned):
            self.ptr = P + 4096 * (1 + len(words))

    monkeypatch.setattr(lowbit, "_call", call)
    monkeypatch.setattr(lowbit, "WorkspaceW4", Room)
    w = lowbit.WeightsW4.__new__(lowbit.WeightsW4)
    w._set(64, 128, 128, torch.float16, torch.device("cuda", 0), P, P, None)
    w._status_ptr = P
    x, y = _OnDevice(0, torch.float16, 40, 128), _OnDevice(0, torch.float16, 40, 64)
    for check in (True, True, False, False):
        with pytest.raises(Reached):
            lowbit.gemm_w4(x, w, out=y, check=check)
    assert len(set(words[:2])) == 2 and P not in words[:2]
    assert words[2:] == [P, P]       # not read by anyone
