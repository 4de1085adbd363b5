"""A token's routing does not depend on the tokens beside it: the same bits of
its weights, and so the same choice between nearly equal experts, whatever the
batch."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("x_type", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("e,h,top,pad", [(8, 2048, 2, 0), (64, 2048, 8, 0), (256, 1040, 8, 0), (64, 4096, 4, 0), (64, 272, 4, 3),
                                         (200, 5632, 6, 1)])
def test_routing_is_that_of_a_token_alone(x_type, e, h, top, pad):
    from rocknpu_b200 import device as dev
    t, f = 64, 16
    g = torch.Generator("cuda").manual_seed(e + h)
    x = torch.randn((t, h + pad), device="cuda", generator=g).to(x_type)[:, :h]
    router = torch.randn((e, h), device="cuda", generator=g) / h ** 0.5
    status = dev.new_status()
    gate, up = (dev.prepare_f8(torch.randn((e, f, h), device="cuda", generator=g), status) for _ in range(2))
    down = dev.prepare_f8(torch.randn((e, h, f), device="cuda", generator=g), status)
    ws = dev.new_workspace(dev.moe_f8_workspace_bytes(t, h, f, e, top, x_type))

    def route(rows):
        _, ids, weights = dev.moe_f8(rows, gate, up, down, status, ws, router=router, top_k=top, renormalize=False)
        return ids, weights

    ids, weights = route(x)
    for first, last in ((0, 1), (5, 6), (63, 64), (3, 6), (10, 18), (20, 53)):
        some_ids, some_weights = route(x[first:last])
        assert torch.equal(some_ids, ids[first:last]) and torch.equal(some_weights, weights[first:last])
    assert status.item() == 0
