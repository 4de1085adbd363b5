"""e4m3 with a scale per block of 128: the activation quantiser, the weight
preparation and the product, against their definition.

The quantisers are compared bit for bit with the definition in f32 (IEEE
quotients, round to nearest even).  The product's bound: a block's 128
products are exact in f32 (4-bit by 4-bit significands) and are summed in
f32, at most one unit in the last place (2^-23 of the running magnitude) per
sum; each of the kb blocks adds one rounding of the scales' product and one
of the multiply-add (2^-24 each), and a split over K one more per part.  So
|out - exact| <= (128 + 3 kb) 2^-23 sum |a w|, plus half a step of a 16-bit
result type.
"""
import numpy as np
import pytest

import oracle
import rocknpu_b200 as rk
from conftest import random_kquant_blocks

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def blocks_of(n):
    return (n + 127) // 128


def scale_of(amax):
    return torch.where(amax == 0, torch.ones_like(amax), (amax * torch.tensor(1.0 / 448.0)).clamp_min(2.0 ** -126))


def ref_rows(a):
    """The quantiser's definition on the CPU: e4m3 codes and scales."""
    m, k = a.shape
    x = torch.nn.functional.pad(a.float(), (0, blocks_of(k) * 128 - k)).view(m, -1, 128)
    s = scale_of(x.abs().amax(dim=2))
    return (x / s[:, :, None]).to(torch.float8_e4m3fn).view(m, -1)[:, :k], s


def ref_weight(w):
    n, k = w.shape
    x = torch.nn.functional.pad(w.float(), (0, blocks_of(k) * 128 - k, 0, blocks_of(n) * 128 - n))
    x = x.view(blocks_of(n), 128, blocks_of(k), 128)
    s = scale_of(x.abs().amax(dim=(1, 3)))
    q = (x / s[:, None, :, None]).to(torch.float8_e4m3fn).view(blocks_of(n) * 128, -1)
    return q[:n, :k], s


def values(q, s, rows):
    """What codes and block scales stand for, in f64."""
    n, k = q.shape
    s = s.double().repeat_interleave(rows, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return q.float().double() * s


def bits(q):
    return q.contiguous().view(torch.uint8)


def check_product(out, a8, a_s, w8, w_s):
    a, w = values(a8.cpu(), a_s.cpu(), 1).cuda(), values(w8.cpu(), w_s.cpu(), 128).cuda()
    ref, mag = a @ w.t(), a.abs() @ w.abs().t()
    kb = blocks_of(a.shape[1])
    bound = (128 + 3 * kb) * 2.0 ** -23 * mag
    if out.dtype != torch.float32:
        # half a step of the type (f16: at least half its smallest subnormal)
        bound = bound + torch.finfo(out.dtype).eps / 2 * (ref.abs() + bound) + 2.0 ** -25
    err = (out.double() - ref).abs()
    assert torch.isfinite(out).all()
    assert (err <= bound).all(), f"max excess {(err / bound.clamp_min(1e-300)).max()}"


def weight(n, k, seed):
    """Random codes of every finite value and scales over a wide range."""
    g = torch.Generator().manual_seed(seed)
    code = torch.randint(0, 256, (n, (k + 15) // 16 * 16), generator=g, dtype=torch.uint8)
    code = torch.where(code & 0x7F == 0x7F, code - 1, code)  # no NaN
    s = torch.exp2(torch.rand((blocks_of(n), blocks_of(k)), generator=g) * 8 - 14)
    return code.view(torch.float8_e4m3fn).cuda()[:, :k], s.cuda()


# ---- quantiser ---------------------------------------------------------------

@pytest.mark.parametrize("type_", list(TYPES))
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 127), (2, 129), (5, 2048), (17, 1000), (300, 136), (2, 5632)])
def test_quantize_rows_bits(type_, m, k):
    from rocknpu_b200 import device as dev
    g = torch.Generator().manual_seed(m * 1000 + k)
    a = (torch.randn((m, k), generator=g) * torch.exp2(torch.randint(-6, 7, (m, 1), generator=g).float()))
    a[torch.rand((m, k), generator=g) < 0.02] *= 30.0
    a[0, :min(k, 128)] = 0.0  # a block of zeros
    a = a.to(TYPES[type_])
    status = dev.new_status()
    q, s = dev.quantize_rows_f8(a.cuda(), status)
    rq, rs = ref_rows(a)
    assert status.item() == 0
    assert torch.equal(s.cpu(), rs)
    assert torch.equal(bits(q).cpu(), bits(rq))


def test_quantize_rows_smallest_and_largest_values():
    from rocknpu_b200 import device as dev
    a = torch.zeros((6, 256))
    a[0, 0] = 1e-45            # scale at its floor
    a[1, 3] = 2.0 ** -120
    a[2, :128] = 3.4e38
    a[3, 200] = -3.4e38
    a[4, :] = torch.linspace(-1e-38, 1e-38, 256)
    a[5, :] = torch.linspace(-448, 448, 256)
    status = dev.new_status()
    q, s = dev.quantize_rows_f8(a.cuda(), status)
    rq, rs = ref_rows(a)
    assert status.item() == 0 and torch.equal(s.cpu(), rs) and torch.equal(bits(q).cpu(), bits(rq))


def nearly_half_quotients():
    """Rows whose quotients lie as near to the middle of two floats as any, next
    to a middle of two e4m3 values: scales S 2^i with S within 40 of a multiple
    of 2^20 (and others), x one of the three floats at s C 2^e, C = 2^20 M +- 1."""
    rng = np.random.default_rng(7)
    rows = []
    for a in range(8, 17):
        for n in list(range(-40, 41)) + [int(v) for v in rng.integers(-2 ** 19, 2 ** 19, 40)]:
            S = a * 2 ** 20 + n
            if not 2 ** 23 <= S < 2 ** 24:
                continue
            s = np.float32(S) * np.float32(2.0 ** -23)
            near = np.float32(s * np.float32(448.0)).view(np.uint32).astype(np.int64) + np.arange(-4, 5)
            amax = near.astype(np.uint32).view(np.float32)
            amax = amax[amax * np.float32(1.0 / 448.0) == s]
            if not len(amax):
                continue
            M = rng.integers(16, 32, 127).astype(object)
            C = M * 2 ** 20 + rng.choice([-1, 0, 1], 127).astype(object)
            e = rng.integers(-10, 8, 127)
            product = np.array([S * int(c) for c in C], dtype=object)  # up to 49 bits
            x = np.array([float(v) for v in product]) * 2.0 ** (-23.0 - 24) * 2.0 ** e
            x = x.astype(np.float32).view(np.int32) + rng.integers(-1, 2, 127).astype(np.int32)
            x = x.view(np.float32) * rng.choice([-1.0, 1.0], 127).astype(np.float32)
            x = np.where(np.abs(x) <= amax[0], x, np.float32(0.0))
            rows.append(np.concatenate([amax[:1], x]).astype(np.float32))
    return torch.from_numpy(np.stack(rows))


@pytest.mark.parametrize("exponent", [0, -60, -83, -84, -100, -110, 100])
def test_quantize_rows_nearly_half_quotients(exponent):
    from rocknpu_b200 import device as dev
    a = nearly_half_quotients() * 2.0 ** exponent
    assert a.shape[0] > 500
    status = dev.new_status()
    q, s = dev.quantize_rows_f8(a.cuda(), status)
    want_q, want_s = ref_rows(a)
    assert status.item() == 0 and torch.equal(s.cpu(), want_s)
    assert torch.equal(bits(q.cpu()), bits(want_q))
    q, s = dev.prepare_f8(a[:, None, :].cuda(), status)
    assert torch.equal(bits(q.cpu()[:, 0]), bits(want_q)) and torch.equal(s.cpu()[:, 0], want_s)


def test_quantize_rows_strided_in_and_out():
    """A column slice of a wider matrix into a slice of a wider one; what lies
    beside it stays."""
    from rocknpu_b200 import device as dev
    wide = torch.randn((9, 700), device="cuda")
    out = torch.full((9, 800), 7, dtype=torch.uint8, device="cuda")
    scales = torch.full((9, 9), -1.0, device="cuda")
    status = dev.new_status()
    a = wide[:, 13:13 + 300]
    dev.quantize_rows_f8(a, status, out=out.view(torch.float8_e4m3fn)[:, 5:305], scales=scales[:, 2:5])
    rq, rs = ref_rows(a.cpu())
    assert torch.equal(out[:, 5:305].cpu(), bits(rq)) and torch.equal(scales[:, 2:5].cpu(), rs)
    assert (out[:, :5] == 7).all() and (out[:, 305:] == 7).all()
    assert (scales[:, :2] == -1).all() and (scales[:, 5:] == -1).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_input_sets_status(bad):
    from rocknpu_b200 import device as dev
    a = torch.randn((4, 300), device="cuda")
    a[2, 299] = bad
    status = dev.new_status()
    dev.quantize_rows_f8(a, status)
    assert status.item() == 1
    status.zero_()
    dev.prepare_f8(a, status)
    assert status.item() == 1


# ---- weight preparation ------------------------------------------------------

@pytest.mark.parametrize("type_", list(TYPES))
@pytest.mark.parametrize("count,n,k", [(1, 1, 1), (1, 128, 128), (2, 129, 127), (3, 200, 333), (1, 256, 2048),
                                       (4, 96, 264)])
def test_prepare_dense_bits(type_, count, n, k):
    from rocknpu_b200 import device as dev
    g = torch.Generator().manual_seed(n + k)
    w = (torch.randn((count, n, k), generator=g) * 0.02).to(TYPES[type_])
    status = dev.new_status()
    q, s = dev.prepare_f8(w.cuda(), status)
    assert status.item() == 0 and q.shape == w.shape and s.shape == (count, blocks_of(n), blocks_of(k))
    for c in range(count):
        rq, rs = ref_weight(w[c])
        assert torch.equal(s[c].cpu(), rs) and torch.equal(bits(q[c]).cpu(), bits(rq))


@pytest.mark.parametrize("kind", [rk.Q4_K, rk.Q5_K, rk.Q6_K])
@pytest.mark.parametrize("n,k", [(1, 256), (128, 512), (130, 768), (300, 2048)])
def test_prepare_kquant_bits(rng, kind, n, k):
    from rocknpu_b200 import device as dev
    blocks = random_kquant_blocks(kind, n * (k // 256), rng)
    status = dev.new_status()
    q, s = dev.prepare_f8_q(kind, torch.from_numpy(blocks).cuda(), k, n, status)
    rq, rs = ref_weight(torch.from_numpy(oracle.dequant(kind, blocks).reshape(n, k)))
    assert status.item() == 0
    assert torch.equal(s.cpu(), rs) and torch.equal(bits(q).cpu(), bits(rq))


# ---- product -----------------------------------------------------------------

@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 128, 128), (1, 5632, 2048), (2, 130, 144), (7, 200, 333),
                                   (16, 2048, 8192), (17, 300, 1000), (33, 128, 4096), (64, 1000, 2048),
                                   (65, 257, 129), (128, 640, 1536), (333, 520, 640), (1000, 300, 4000),
                                   (2048, 2048, 2048)])
def test_product(m, n, k):
    from rocknpu_b200 import device as dev
    w8, w_s = weight(n, k, m + n + k)
    a = torch.randn((m, k), device="cuda", generator=torch.Generator("cuda").manual_seed(n))
    status = dev.new_status()
    a8, a_s = dev.quantize_rows_f8(a, status)
    ws = dev.new_workspace(dev.gemm_f8_workspace_bytes(m, n, k))
    split = dev.gemm_f8(a8, a_s, w8, w_s, status, workspace=ws)
    again = dev.gemm_f8(a8, a_s, w8, w_s, status, workspace=ws)
    whole = dev.gemm_f8(a8, a_s, w8, w_s, status)
    assert status.item() == 0
    check_product(split, a8, a_s, w8, w_s)
    check_product(whole, a8, a_s, w8, w_s)
    assert torch.equal(split, again)
    assert not ws[:65536].any()


@pytest.mark.parametrize("type_", list(TYPES))
@pytest.mark.parametrize("m,n,k", [(1, 300, 2048), (5, 257, 200), (40, 512, 1111), (200, 384, 640)])
def test_matmul_types(type_, m, n, k):
    """One call does what the quantiser and the product do, bit for bit."""
    from rocknpu_b200 import device as dev
    w8, w_s = weight(n, k, n)
    a = (torch.randn((m, k), device="cuda") * 0.1).to(TYPES[type_])
    status = dev.new_status()
    ws = dev.new_workspace(dev.matmul_f8_workspace_bytes(m, n, k))
    out = dev.matmul_f8(a, w8, w_s, status, ws)
    a8, a_s = dev.quantize_rows_f8(a, status)
    ref = dev.gemm_f8(a8, a_s, w8, w_s, status, out_dtype=TYPES[type_], workspace=ws)
    assert out.dtype == a.dtype and torch.equal(out, ref) and status.item() == 0
    check_product(out, a8, a_s, w8, w_s)
    wide = dev.matmul_f8(a, w8, w_s, status, ws, out_dtype=torch.float32)
    assert wide.dtype == torch.float32
    check_product(wide, a8, a_s, w8, w_s)


@pytest.mark.parametrize("type_", list(TYPES))
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 16, 128), (1, 17, 96), (2, 130, 160), (3, 40, 288), (5, 48, 1600),
                                   (8, 5632, 2048), (9, 300, 4096), (16, 1000, 1024), (1, 333, 16384), (2, 6000, 8192),
                                   (8, 2400, 8192), (16, 129, 64), (4, 20000, 512), (1, 40000, 256), (7, 9999, 2080)])
def test_few_tokens(type_, m, n, k):
    """Rows that the product may quantise itself and rows that it may not; a
    weight that starts at a 16-byte boundary only; wider rows around the result."""
    from rocknpu_b200 import device as dev
    w8, w_s = weight(n, k, m + k)
    a = (torch.randn((m, k + 3), device="cuda", generator=torch.Generator("cuda").manual_seed(n)) * 3).to(TYPES[type_])
    a[:, 40:70] = 0
    status = dev.new_status()
    ws = dev.new_workspace(dev.matmul_f8_workspace_bytes(m, n, k))
    for rows in (a[:, :k], a[:, 3:], a[:, :k].contiguous()):
        a8, a_s = dev.quantize_rows_f8(rows, status)
        wide = torch.full((m, n + 9), -5.0, device="cuda")
        out = dev.matmul_f8(rows, w8, w_s, status, ws, out=wide[:, 4:4 + n])
        check_product(out, a8, a_s, w8, w_s)
        assert (wide[:, :4] == -5).all() and (wide[:, 4 + n:] == -5).all()
        assert torch.equal(out, dev.gemm_f8(a8, a_s, w8, w_s, status, workspace=ws))
        own = dev.matmul_f8(rows, w8, w_s, status, ws)
        assert own.dtype == rows.dtype and torch.equal(own, out.to(rows.dtype))
    odd = torch.zeros(n * k + 16, dtype=torch.uint8, device="cuda")[16:].view(n, k).view(torch.float8_e4m3fn)
    odd.view(torch.uint8).copy_(w8.view(torch.uint8))
    check_product(dev.matmul_f8(rows, odd, w_s, status, ws, out_dtype=torch.float32), a8, a_s, w8, w_s)
    assert status.item() == 0
    rows[m - 1, k - 1] = float("nan")
    dev.matmul_f8(rows, w8, w_s, status, ws)
    assert status.item() == 1


def test_matmul_strided_rows_leave_the_rest():
    from rocknpu_b200 import device as dev
    m, n, k = 19, 200, 320
    w8, w_s = weight(n, k + 160, 3)
    w8 = w8[:, 32:32 + k]  # a slice whose rows start at 16-byte boundaries
    w_s = w_s[:, :blocks_of(k)].contiguous()
    a = torch.randn((m, 500), device="cuda")[:, 7:7 + k]
    out = torch.full((m, n + 50), -5.0, device="cuda")
    status = dev.new_status()
    ws = dev.new_workspace(dev.matmul_f8_workspace_bytes(m, n, k))
    dev.matmul_f8(a, w8, w_s, status, ws, out=out[:, 20:20 + n])
    a8, a_s = dev.quantize_rows_f8(a, status)
    check_product(out[:, 20:20 + n], a8, a_s, w8, w_s)
    assert (out[:, :20] == -5).all() and (out[:, 20 + n:] == -5).all() and status.item() == 0


def test_prepared_kquant_through_matmul(rng):
    """A GGUF weight prepared, then multiplied: the chain a user runs."""
    from rocknpu_b200 import device as dev
    m, n, k = 24, 520, 1024
    blocks = rk.synth_q_weights(rk.Q4_K, n, k, seed=5)
    status = dev.new_status()
    w8, w_s = dev.prepare_f8_q(rk.Q4_K, torch.from_numpy(blocks).cuda(), k, n, status)
    a = torch.from_numpy(rk.synth_normal(6, m * k).reshape(m, k)).cuda()
    ws = dev.new_workspace(dev.matmul_f8_workspace_bytes(m, n, k))
    out = dev.matmul_f8(a, w8, w_s, status, ws)
    a8, a_s = dev.quantize_rows_f8(a, status)
    check_product(out, a8, a_s, w8, w_s)
    # and near the unquantised product: each of the two roundings of a term is
    # off by at most 2^-4 of it, or by 2^-10 of its block's scale
    exact = a.cpu().double() @ torch.from_numpy(oracle.dequant(rk.Q4_K, blocks).reshape(n, k)).double().t()
    assert ((out.cpu().double() - exact).norm() / exact.norm()) < 2.0 ** -4 * 2
    assert status.item() == 0


def test_matmul_graph_and_side_stream():
    """Captured on another stream and replayed with new inputs."""
    from rocknpu_b200 import device as dev
    m, n, k = 4, 1000, 2048
    w8, w_s = weight(n, k, 9)
    a = torch.randn((m, k), device="cuda")
    status = dev.new_status()
    ws = dev.new_workspace(dev.matmul_f8_workspace_bytes(m, n, k))
    out = torch.empty((m, n), device="cuda")
    dev.matmul_f8(a, w8, w_s, status, ws, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dev.matmul_f8(a, w8, w_s, status, ws, out=out)
    for seed in range(3):
        a.copy_(torch.randn((m, k), generator=torch.Generator().manual_seed(seed)))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        a8, a_s = dev.quantize_rows_f8(a, status)
        check_product(out, a8, a_s, w8, w_s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dev.matmul_f8(a, w8, w_s, status, ws)
    side.synchronize()
    assert torch.equal(got, out) and status.item() == 0


def test_weights_written_just_before_the_call():
    """The weight's preparation queued right before the product on one stream."""
    from rocknpu_b200 import device as dev
    m, n, k = 3, 4096, 4096
    status = dev.new_status()
    ws = dev.new_workspace(dev.matmul_f8_workspace_bytes(m, n, k))
    a = torch.randn((m, k), device="cuda")
    a8, a_s = dev.quantize_rows_f8(a, status)
    for seed in range(3):
        w = torch.randn((n, k), device="cuda", generator=torch.Generator("cuda").manual_seed(seed))
        w8, w_s = dev.prepare_f8(w, status)
        one = dev.matmul_f8(a, w8, w_s, status, ws)
        w8, w_s = dev.prepare_f8(w, status)
        two = dev.gemm_f8(a8, a_s, w8, w_s, status, workspace=ws)
        torch.cuda.synchronize()
        check_product(one, a8, a_s, w8, w_s)
        assert torch.equal(one, two)


def test_one_workspace_serves_many_shapes():
    from rocknpu_b200 import device as dev
    shapes = [(1, 5632, 2048), (40, 300, 4096), (1, 64, 8192), (200, 1000, 512), (16, 2048, 2048)]
    ws = dev.new_workspace(max(dev.matmul_f8_workspace_bytes(*s) for s in shapes))
    status = dev.new_status()
    for m, n, k in shapes + shapes[::-1]:
        w8, w_s = weight(n, k, m + n)
        a = torch.randn((m, k), device="cuda")
        out = dev.matmul_f8(a, w8, w_s, status, ws)
        a8, a_s = dev.quantize_rows_f8(a, status)
        check_product(out, a8, a_s, w8, w_s)
    assert status.item() == 0


def test_more_than_2_32_values():
    from rocknpu_b200 import device as dev
    m, k = 40000, 110000
    a = torch.empty((m, k), dtype=torch.bfloat16, device="cuda")
    rows = [0, 19999, 39000, m - 1]
    a.zero_()
    for i in rows:
        a[i] = torch.randn(k, generator=torch.Generator().manual_seed(i)).bfloat16()
    status = dev.new_status()
    q, s = dev.quantize_rows_f8(a, status)
    for i in rows:
        rq, rs = ref_rows(a[i:i + 1].cpu())
        assert torch.equal(bits(q[i:i + 1]).cpu(), bits(rq)) and torch.equal(s[i:i + 1].cpu(), rs)
    assert status.item() == 0


def test_output_past_2_31_values():
    from rocknpu_b200 import device as dev
    m, n, k = 66000, 33000, 48
    w8, w_s = weight(n, k, 1)
    a = torch.randn((m, k), device="cuda")
    status = dev.new_status()
    ws = dev.new_workspace(dev.matmul_f8_workspace_bytes(m, n, k))
    out = dev.matmul_f8(a, w8, w_s, status, ws)
    a8, a_s = dev.quantize_rows_f8(a, status)
    for i in (0, 32768, 65077, m - 100):
        check_product(out[i:i + 100], a8[i:i + 100], a_s[i:i + 100], w8, w_s)
    assert status.item() == 0


def test_refusals():
    """Shapes, types and devices that the wrappers turn away."""
    from rocknpu_b200 import device as dev
    w8, w_s = weight(200, 320, 1)
    a = torch.randn((4, 320), device="cuda")
    status = dev.new_status()
    ws = dev.new_workspace(dev.matmul_f8_workspace_bytes(4, 200, 320))
    a8, a_s = dev.quantize_rows_f8(a, status)
    bad = [lambda: dev.quantize_rows_f8(a.double(), status), lambda: dev.quantize_rows_f8(a[0], status),
           lambda: dev.quantize_rows_f8(a.t(), status), lambda: dev.quantize_rows_f8(a[:0], status),
           lambda: dev.quantize_rows_f8(a, status.float()), lambda: dev.quantize_rows_f8(a, status.cpu()),
           lambda: dev.quantize_rows_f8(a, status, out=a8[:, :319]),
           lambda: dev.quantize_rows_f8(a, status, scales=a_s[:, :2]),
           lambda: dev.prepare_f8(a.long(), status), lambda: dev.prepare_f8(a[None, None], status),
           lambda: dev.prepare_f8(torch.randn((4, 9, 320), device="cuda")[::2], status),
           lambda: dev.prepare_f8_q(4, torch.zeros(100, dtype=torch.uint8, device="cuda"), 256, 1, status),
           lambda: dev.prepare_f8_q(9, torch.zeros(1000, dtype=torch.uint8, device="cuda"), 256, 1, status),
           lambda: dev.matmul_f8(a[:, :319], w8, w_s, status, ws), lambda: dev.matmul_f8(a, w8.float(), w_s, status, ws),
           lambda: dev.matmul_f8(a, w8, w_s[:1], status, ws), lambda: dev.matmul_f8(a, w8, w_s.double(), status, ws),
           lambda: dev.matmul_f8(a, w8, w_s, status, ws, out=torch.empty((4, 199), device="cuda")),
           lambda: dev.matmul_f8(a, w8, w_s, status, ws, out_dtype=torch.float64),
           lambda: dev.gemm_f8(a8, a_s[:, :2], w8, w_s, status), lambda: dev.gemm_f8(a8.float(), a_s, w8, w_s, status),
           lambda: dev.gemm_f8(a8, a_s, w8[:, :304], w_s, status)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    odd = torch.zeros((200, 330), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, 1:321]
    for call in (lambda: dev.matmul_f8(a, odd, w_s, status, ws),  # rows not at 16-byte boundaries
                 lambda: dev.matmul_f8(a, w8, w_s, status, ws[:100])):
        with pytest.raises(RuntimeError):
            call()
    assert status.item() == 0
