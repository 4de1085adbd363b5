"""The e4m3 entry points refuse bad arguments before any work is queued: on
the CPU, with addresses that are never read."""
import ctypes
import struct

import pytest

import rocknpu_b200 as rk
from rocknpu_b200 import capi

torch = pytest.importorskip("torch")

BAD = rk.STATUS_INVALID_ARGUMENT
F32, F16, BF16 = capi.GGML_F32, capi.GGML_F16, capi.GGML_BF16
P = 1 << 20  # an aligned address that nothing reads


def changed(good, **change):
    return list({**good, **change}.values())


QUANTIZE = dict(type=F32, a=P, m=4, k=300, lda=300, out=P, ld8=304, scales=P, lds=3, status=P, stream=None)


@pytest.mark.parametrize("change", [dict(type=12), dict(type=77), dict(a=None), dict(a=P + 2), dict(type=BF16, a=P + 1),
                                    dict(m=0), dict(k=0), dict(m=1 << 40), dict(lda=299), dict(ld8=299), dict(lds=2),
                                    dict(out=None), dict(scales=None), dict(status=None)])
def test_quantize_rows(change):
    assert rk.lib().rocknpu_b200_quantize_rows_f8(*changed(QUANTIZE, **change)) == BAD


PREPARE = dict(type=F16, w=P, n=200, k=300, ldw=300, count=2, out=P, ld8=304, scales=P, status=P, stream=None)


@pytest.mark.parametrize("change", [dict(type=14), dict(w=None), dict(w=P + 1), dict(n=0), dict(k=0), dict(count=0),
                                    dict(ldw=299), dict(ld8=299), dict(out=None), dict(scales=None), dict(status=None)])
def test_prepare(change):
    assert rk.lib().rocknpu_b200_prepare_f8(*changed(PREPARE, **change)) == BAD


PREPARE_Q = dict(kind=4, blocks=P, k=512, n=10, out=P, ld8=512, scales=P, status=P, stream=None)


@pytest.mark.parametrize("change", [dict(kind=3), dict(kind=7), dict(blocks=None), dict(blocks=P + 2), dict(k=300), dict(k=0),
                                    dict(n=0), dict(ld8=511), dict(ld8=514), dict(out=P + 2), dict(out=None),
                                    dict(scales=None), dict(status=None)])
def test_prepare_q(change):
    assert rk.lib().rocknpu_b200_prepare_f8_q(*changed(PREPARE_Q, **change)) == BAD


GEMM = dict(a=P, lda=304, a_s=P, ld_as=3, w=P, ldw=304, w_s=P, out=P, out_type=F32, ldo=200, m=4, k=300, n=200,
            ws=P, ws_bytes=0, status=P, stream=None)


@pytest.mark.parametrize("change", [dict(a=None), dict(a=P + 8), dict(lda=300), dict(lda=288), dict(ld_as=2), dict(w=None),
                                    dict(w=P + 4), dict(ldw=308), dict(ldw=288), dict(w_s=None), dict(out=None),
                                    dict(out=P + 2), dict(out_type=6), dict(ldo=199), dict(m=0), dict(k=0), dict(n=0),
                                    dict(ws=P + 8), dict(status=None), dict(a_s=None)])
def test_gemm(change):
    assert rk.lib().rocknpu_b200_gemm_f8(*changed(GEMM, **change)) == BAD


def matmul_args(**change):
    need = rk.lib().rocknpu_b200_matmul_f8_workspace_bytes(4, 200, 300)
    good = dict(a=P, type=F32, lda=300, w=P, ldw=304, w_s=P, out=P, out_type=F32, ldo=200, m=4, k=300, n=200,
                ws=P, ws_bytes=need, status=P, stream=None)
    if change.pop("short", False):
        good["ws_bytes"] = need - 1
    return changed(good, **change)


@pytest.mark.parametrize("change", [dict(a=None), dict(a=P + 2), dict(type=13), dict(lda=299), dict(w=P + 8), dict(ldw=300),
                                    dict(out=None), dict(out_type=12), dict(ldo=199), dict(m=0), dict(k=0), dict(n=0),
                                    dict(ws=None), dict(ws=P + 8), dict(short=True), dict(status=None)])
def test_matmul(change):
    assert rk.lib().rocknpu_b200_matmul_f8(*matmul_args(**dict(change))) == BAD


def test_workspace_sizes():
    lib = rk.lib()
    assert lib.rocknpu_b200_gemm_f8_workspace_bytes(0, 1, 1) == 0
    assert lib.rocknpu_b200_matmul_f8_workspace_bytes(1, 1, 0) == 0
    for m, n, k in [(1, 1, 1), (16, 28672, 8192), (4096, 28672, 8192)]:
        gemm = lib.rocknpu_b200_gemm_f8_workspace_bytes(m, n, k)
        whole = lib.rocknpu_b200_matmul_f8_workspace_bytes(m, n, k)
        assert 65536 <= gemm < 64 << 20 and whole >= gemm + m * k


# ---- the mixture-of-experts layer --------------------------------------------

def moe_call(short=0, status=P, **change):
    t, h, f, e, top = 5, 512, 256, 4, 2
    a = capi.MoeF8Args(t, h, f, e, top, F32, P, P, h, h, (P, h, f * h, P, 8), (P, h, f * h, P, 8), (P, f, f * h, P, 8),
                       P, F32, h, 1, P, P)
    for name, value in change.items():
        at = a
        *path, last = name.split("__")
        for x in path:
            at = getattr(at, x)
        setattr(at, last, value)
    need = rk.lib().rocknpu_b200_moe_f8_workspace_bytes(t, h, f, e, top, F32)
    assert need > 65536
    return rk.lib().rocknpu_b200_moe_f8(ctypes.byref(a), P, need - short, status, None)


@pytest.mark.parametrize("change", [dict(tokens=0), dict(tokens=65), dict(hidden=500), dict(hidden=0), dict(ffn=250),
                                    dict(experts=0), dict(experts=257), dict(top_k=0), dict(top_k=5), dict(type=12),
                                    dict(x=None), dict(x=P + 2), dict(out=None), dict(ld_x=511), dict(ld_out=511),
                                    dict(router=P + 1), dict(router_type=9), dict(ld_router=511), dict(ids=None),
                                    dict(weights=None), dict(gate__w_f8=None), dict(gate__w_f8=P + 8), dict(up__ld=504),
                                    dict(up__ld=520), dict(down__stride=512 * 256 - 16), dict(down__stride=512 * 256 + 8),
                                    dict(gate__scales=None), dict(up__scale_stride=7), dict(short=1), dict(status=None)])
def test_moe(change):
    assert moe_call(**change) == BAD


def test_moe_without_arguments_or_workspace():
    lib = rk.lib()
    assert lib.rocknpu_b200_moe_f8(None, P, 1 << 30, P, None) == BAD
    a = capi.MoeF8Args()
    assert lib.rocknpu_b200_moe_f8(ctypes.byref(a), None, 0, P, None) == BAD
    assert lib.rocknpu_b200_moe_f8_workspace_bytes(65, 512, 256, 4, 2, F32) == 0
    assert lib.rocknpu_b200_moe_f8_workspace_bytes(1, 512, 256, 4, 17, F32) == 0


def test_moe_argument_bytes():
    """device.moe_f8 packs the argument struct itself."""
    from rocknpu_b200 import device as dev
    assert dev._MOE_ARGS.size == ctypes.sizeof(capi.MoeF8Args)
    values = list(range(1, 34))
    packed = dev._MOE_ARGS.pack(*values[:dev._MOE_ARGS.unpack(bytes(dev._MOE_ARGS.size)).__len__()])
    a = capi.MoeF8Args.from_buffer_copy(packed)
    flat = []
    for name, _ in a._fields_:
        v = getattr(a, name)
        flat += [getattr(v, f) for f, _ in v._fields_] if isinstance(v, ctypes.Structure) else [v]
    assert flat == values[:len(flat)] and struct.calcsize("P") == 8


@pytest.mark.parametrize("bad", [P + 1, P + 2, P + 3])
def test_unaligned_scales_indices_and_status(bad):
    lib = rk.lib()
    for name in ("scales", "status"):
        assert lib.rocknpu_b200_quantize_rows_f8(*changed(QUANTIZE, **{name: bad})) == BAD
        assert lib.rocknpu_b200_prepare_f8(*changed(PREPARE, **{name: bad})) == BAD
        assert lib.rocknpu_b200_prepare_f8_q(*changed(PREPARE_Q, **{name: bad})) == BAD
    for name in ("a_s", "w_s", "status"):
        assert lib.rocknpu_b200_gemm_f8(*changed(GEMM, **{name: bad})) == BAD
    for name in ("w_s", "status"):
        assert lib.rocknpu_b200_matmul_f8(*matmul_args(**{name: bad})) == BAD
    for name in ("gate__scales", "up__scales", "down__scales", "ids", "weights", "status"):
        assert moe_call(**{name: bad}) == BAD


def test_workspace_sizes_of_the_largest_dimensions():
    """Sizes nothing can hold are answered without overflow."""
    lib, most = rk.lib(), 0x7fffff00
    for m, n, k in [(most, 1, most), (1, most, most), (most, most, most)]:
        assert 65536 <= lib.rocknpu_b200_gemm_f8_workspace_bytes(m, n, k) < 64 << 20
        assert lib.rocknpu_b200_matmul_f8_workspace_bytes(m, n, k) >= m * k
    for m, n, k in [(most + 1, 1, 1), (1, most + 1, 1), (1, 1, most + 1)]:
        assert lib.rocknpu_b200_gemm_f8_workspace_bytes(m, n, k) == 0


def test_host_tensors_are_refused():
    from rocknpu_b200 import device as dev
    a, status = torch.zeros((2, 128)), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        dev.quantize_rows_f8(a, status)
    with pytest.raises(ValueError):
        dev.prepare_f8(a, status)


def test_status_codes():
    code = rk.lib().rocknpu_b200_status_code
    assert code(0) == rk.STATUS_OK and code(1) == BAD and code(9) == BAD
    assert code(8) == rk.STATUS_EXECUTION_ERROR and code(5) == rk.STATUS_EXECUTION_ERROR
