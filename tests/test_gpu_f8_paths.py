"""The e4m3 product and quantiser in the kernel forms that larger shapes take:
two-SM 256 x 256 tiles (several per pair, remainders in every direction, each
result type, aligned and unaligned results), and quantiser grids that take
more than one step.  Bounds as in the operators' other tests: a block's sum is
off by 128 units of 2^-23 of the sum over magnitudes at most, a block adds
three roundings of 2^-24.

Which kernel ran is read from a captured graph of the call.
"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
driver = pytest.importorskip("cuda.bindings.driver")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def kernels_of(call):
    """Names of the kernels that a call launches."""
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    raw = driver.CUgraph(graph.raw_cuda_graph())

    def ok(result):
        assert result[0] == driver.CUresult.CUDA_SUCCESS, result[0]
        return result[1:]

    count = ok(driver.cuGraphGetNodes(raw, 0))[1]
    names = []
    for node in ok(driver.cuGraphGetNodes(raw, count))[0]:
        if ok(driver.cuGraphNodeGetType(node))[0] == driver.CUgraphNodeType.CU_GRAPH_NODE_TYPE_KERNEL:
            params = ok(driver.cuGraphKernelNodeGetParams(node))[0]
            names.append(ok(driver.cuFuncGetName(params.func))[0].decode())
    return names


def blocks_of(n):
    return (n + 127) // 128


def values(q, s, rows):
    n, k = q.shape
    return q.float().double() * s.double().repeat_interleave(rows, 0)[:n].repeat_interleave(128, 1)[:, :k]


def weight(n, k, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    code = torch.randint(0, 256, (n, (k + 15) // 16 * 16), generator=g, dtype=torch.uint8, device="cuda")
    code = torch.where(code & 0x7F == 0x7F, code - 1, code)  # no NaN
    s = torch.exp2(torch.rand((blocks_of(n), blocks_of(k)), generator=g, device="cuda") * 8 - 14)
    return code.view(torch.float8_e4m3fn)[:, :k], s


def check(out, ref, mag, kb):
    bound = (128 + 3 * kb) * 2.0 ** -23 * mag
    if out.dtype != torch.float32:
        bound = bound + torch.finfo(out.dtype).eps / 2 * (ref.abs() + bound) + 2.0 ** -25
    assert torch.isfinite(out).all()
    assert ((out.double() - ref).abs() <= bound).all()


# one tile per pair with a CTA wholly past m; several, with remainders in m, n
# and k, an odd and an even number of blocks; a CTA wholly past n
PAIR_SHAPES = [(333, 8960, 1536), (2500, 4200, 2100), (2500, 4200, 2296), (1030, 9000, 4000), (700, 20000, 1664)]


@pytest.mark.parametrize("m,n,k", PAIR_SHAPES)
def test_two_sm_tiles(m, n, k):
    from rocknpu_b200 import device as dev
    w8, w_s = weight(n, k, m)
    a = torch.randn((m, k), device="cuda", generator=torch.Generator("cuda").manual_seed(n))
    status = dev.new_status()
    ws = dev.new_workspace(dev.matmul_f8_workspace_bytes(m, n, k))
    a8, a_s = dev.quantize_rows_f8(a, status)
    av, wv = values(a8, a_s, 1), values(w8, w_s, 128)
    ref, mag = av @ wv.t(), av.abs() @ wv.abs().t()
    plain = dev.gemm_f8(a8, a_s, w8, w_s, status, workspace=ws)
    assert any("gemm_f8_pair" in name for name in kernels_of(lambda: dev.gemm_f8(a8, a_s, w8, w_s, status, workspace=ws)))
    check(plain, ref, mag, blocks_of(k))
    assert torch.equal(plain, dev.matmul_f8(a, w8, w_s, status, ws))
    for dtype in TYPES.values():
        # whole rows, rows of an odd pitch, rows whose first value is not at 16 bytes
        for pitch, at in ((n, 0), (n + 5, 2), (n + 8, 1)):
            wide = torch.full((m + 1, pitch), -5.0, dtype=dtype, device="cuda")
            out = dev.gemm_f8(a8, a_s, w8, w_s, status, out=wide[:m, at:at + n], workspace=ws)
            assert torch.equal(out, plain.to(dtype))
            assert (wide[m:] == -5).all() and (wide[:, :at] == -5).all() and (wide[:, at + n:] == -5).all()
    assert status.item() == 0


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 5, 7), (2, 300, 31), (129, 130, 15), (40, 1, 1000)])
def test_smallest_sizes(m, n, k):
    from rocknpu_b200 import device as dev
    w8, w_s = weight(n, k, m)
    a = torch.randn((m, k), device="cuda")
    status = dev.new_status()
    ws = dev.new_workspace(dev.matmul_f8_workspace_bytes(m, n, k))
    a8, a_s = dev.quantize_rows_f8(a, status)
    av, wv = values(a8, a_s, 1), values(w8, w_s, 128)
    out = dev.matmul_f8(a, w8, w_s, status, ws)
    check(out, av @ wv.t(), av.abs() @ wv.abs().t(), blocks_of(k))
    assert torch.equal(out, dev.gemm_f8(a8, a_s, w8, w_s, status, workspace=ws)) and status.item() == 0


@pytest.mark.parametrize("type_", list(TYPES))
@pytest.mark.parametrize("m,k,pad", [(2048, 2048, 0), (3000, 1024, 0), (2050, 1920, 0), (700, 4999, 0), (2048, 2048, 3)])
def test_quantiser_of_more_than_one_step(type_, m, k, pad):
    """More than 20000 blocks: whole pairs of blocks, whole blocks, odd rows,
    codes that are not aligned."""
    from rocknpu_b200 import device as dev
    assert m * blocks_of(k) > 20000
    a = (torch.randn((m, k), generator=torch.Generator().manual_seed(k)) * 3).to(TYPES[type_])
    status = dev.new_status()
    out = None
    if pad:
        out = torch.zeros((m, k + pad), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, pad:]
    q, s = dev.quantize_rows_f8(a.cuda(), status, out=out)
    x = torch.nn.functional.pad(a.float(), (0, blocks_of(k) * 128 - k)).view(m, -1, 128)
    amax = x.abs().amax(dim=2)
    rs = torch.where(amax == 0, torch.ones_like(amax), (amax * torch.tensor(1.0 / 448.0)).clamp_min(2.0 ** -126))
    rq = (x / rs[:, :, None]).to(torch.float8_e4m3fn).view(m, -1)[:, :k]
    assert status.item() == 0 and torch.equal(s.cpu(), rs)
    assert torch.equal(q.cpu().contiguous().view(torch.uint8), rq.contiguous().view(torch.uint8))
