"""What a status word keeps: a wait that ran out (2 to 8) replaces an operand's
code (1 non-finite, 9 bad index) and is not replaced by one, so that a
workspace which such a wait may have left in use is never taken for clean."""
import ctypes
import threading

import pytest

import rocknpu_b200 as rk
from rocknpu_b200.capi import lib

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

NAN = float("nan")


def calls():
    """Calls that find a non-finite operand, by name."""
    from rocknpu_b200 import device as dev
    a = torch.randn((4, 256), device="cuda")
    a[1, 5] = NAN
    good = torch.randn((4, 256), device="cuda")
    clean = dev.new_status()
    w8, w_s = dev.prepare_f8(torch.randn((256, 256), device="cuda"), clean)
    stack = tuple(t[None].expand(2, *t.shape).contiguous() for t in (w8.view(torch.uint8), w_s))
    experts = (stack[0].view(torch.float8_e4m3fn), stack[1])
    ws = dev.new_workspace(max(dev.matmul_f8_workspace_bytes(64, 256, 256),
                               dev.moe_f8_workspace_bytes(64, 256, 256, 2, 1, torch.float32)))
    blocks = torch.from_numpy(rk.synth_q_weights(rk.Q4_K, 4, 256, seed=1)).cuda()
    blocks[0:2] = torch.tensor([0, 0x7E], dtype=torch.uint8)  # d: an f16 NaN
    router = torch.randn((2, 256), device="cuda")
    ids = torch.zeros((4, 1), dtype=torch.int32, device="cuda")
    bad_ids = torch.full((4, 1), 2, dtype=torch.int32, device="cuda")
    one = torch.ones((4, 1), device="cuda")
    return {
        "quantize_rows_f8": lambda st: dev.quantize_rows_f8(a, st),
        "prepare_f8": lambda st: dev.prepare_f8(a, st),
        "prepare_f8_q": lambda st: dev.prepare_f8_q(rk.Q4_K, blocks, 256, 4, st),
        "matmul_f8": lambda st: dev.matmul_f8(a, w8, w_s, st, ws),
        "matmul_f8 of many rows": lambda st: dev.matmul_f8(a.repeat(16, 1), w8, w_s, st, ws),
        "moe_f8": lambda st: dev.moe_f8(a, experts, experts, experts, st, ws, ids=ids, weights=one),
        "moe_f8 with a router": lambda st: dev.moe_f8(good, experts, experts, experts, st, ws, router=router * NAN, top_k=1),
        "moe_f8 with a bad index": lambda st: dev.moe_f8(good, experts, experts, experts, st, ws, ids=bad_ids, weights=one),
        "quantize_rows": lambda st: dev.quantize_rows(a, st),
        "prepare_w8": lambda st: dev.prepare_w8(rk.Q4_K, blocks, 256, 4, st),
    }


def test_an_operand_does_not_hide_a_wait():
    for name, call in calls().items():
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        call(status)
        assert status.item() == (9 if "index" in name else 1), name
        status.fill_(4)  # as a wait of an earlier call left it
        call(status)
        assert status.item() == 4, name


@pytest.mark.parametrize("before,after", [(0, 6), (1, 6), (9, 6), (4, 4)])
def test_a_wait_replaces_an_operands_code(before, after):
    """The peer barrier's wait for a rank that never enters, given 20 ms."""
    torch.cuda.init()
    handles, results = [], {}
    for rank in range(2):
        raw, h = (ctypes.c_uint8 * 64)(), ctypes.c_void_p()
        assert lib().rocknpu_b200_peer_buffer_create(1 << 20, rank, 2, raw, ctypes.byref(h)) == 0
        handles.append((h.value, bytes(raw)))
    both = (ctypes.c_uint8 * 128).from_buffer_copy(handles[0][1] + handles[1][1])

    def open_(rank):
        results[rank] = lib().rocknpu_b200_peer_buffer_open(handles[rank][0], both)

    try:
        threads = [threading.Thread(target=open_, args=(r,)) for r in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(timeout=120)
        assert results == {0: 0, 1: 0}
        status = torch.full((1,), before, dtype=torch.int32, device="cuda")
        assert lib().rocknpu_b200_set_peer_wait_limit_ms(20) == 0
        stream = torch.cuda.current_stream().cuda_stream
        assert lib().rocknpu_b200_peer_barrier(handles[0][0], status.data_ptr(), stream) == 0
        torch.cuda.synchronize()
        assert status.item() == after
    finally:
        lib().rocknpu_b200_set_peer_wait_limit_ms(0)
        for h, _ in handles:
            lib().rocknpu_b200_peer_buffer_destroy(h)


@pytest.mark.parametrize("bad", [NAN, float("inf"), -float("inf")])
def test_a_weight_of_a_live_slot_is_an_input(bad):
    """Given routing weights: a non-finite one sets the word, except in an empty slot."""
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 5, 256, 128, 3, 2
    status = dev.new_status()
    x = torch.randn((t, h), device="cuda")
    gate, up = (dev.prepare_f8(torch.randn((e, f, h), device="cuda"), status) for _ in range(2))
    down = dev.prepare_f8(torch.randn((e, h, f), device="cuda"), status)
    ws = dev.new_workspace(dev.moe_f8_workspace_bytes(t, h, f, e, top, x.dtype))
    ids = torch.randint(0, e, (t, top), dtype=torch.int32, device="cuda")
    weights = torch.rand((t, top), device="cuda")
    weights[3, 1] = bad
    ids[3, 1] = -1
    dev.moe_f8(x, gate, up, down, status, ws, ids=ids, weights=weights)
    assert status.item() == 0
    ids[3, 1] = 2
    dev.moe_f8(x, gate, up, down, status, ws, ids=ids, weights=weights)
    assert status.item() == 1
    assert not ws[:65536].any()
