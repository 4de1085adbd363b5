"""The e4m3 wrappers take a workspace's size from the tensor: one whose
elements share memory, or leave gaps, is refused."""
import pytest

torch = pytest.importorskip("torch")


def test_only_contiguous_workspaces():
    from rocknpu_b200 import device as dev
    ws = torch.zeros(1 << 16, dtype=torch.uint8)
    assert dev._workspace(ws) == (ws.data_ptr(), 1 << 16)
    assert dev._workspace(ws.view(torch.int32)) == (ws.data_ptr(), 1 << 16)
    for bad in (ws[:1].expand(1 << 30), ws[::2], ws.view(256, 256).t()):
        with pytest.raises(ValueError):
            dev._workspace(bad)


@pytest.mark.gpu
def test_calls_refuse_them():
    from rocknpu_b200 import device as dev
    status = dev.new_status()
    a = torch.randn((4, 256), device="cuda")
    w8, w_s = dev.prepare_f8(torch.randn((256, 256), device="cuda"), status)
    a8, a_s = dev.quantize_rows_f8(a, status)
    experts = w8[None], w_s[None]
    ids, weights = torch.zeros((4, 1), dtype=torch.int32, device="cuda"), torch.ones((4, 1), device="cuda")
    bad = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")[:16].expand(1 << 20, 16)
    for call in (lambda: dev.matmul_f8(a, w8, w_s, status, bad), lambda: dev.gemm_f8(a8, a_s, w8, w_s, status, workspace=bad),
                 lambda: dev.moe_f8(a, experts, experts, experts, status, bad, ids=ids, weights=weights)):
        with pytest.raises(ValueError):
            call()
    assert status.item() == 0
