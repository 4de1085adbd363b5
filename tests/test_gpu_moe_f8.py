"""The mixture-of-experts layer over e4m3 expert weights, against its formula
in f64.

Bound for one output y = sum over slots p * sum_f Wd[f] h[f], derived from the
roundings in turn (u = 2^-24, K = 128 values per block; S(.) is the same sum
over magnitudes):
- an activation of a product is off by at most r of its block's largest
  magnitude: r = 2^-23 (f32: two f16 terms), 2^-24 of it (16-bit input types
  are exact down to there) ;
- a product sum over n values and n / K blocks is off by (K + 3 n / K + 2) 2u
  of the sum over magnitudes (as in the product's tests);
so gate and up are off by dg, du <= r B + c S, with B the sum of |w| times the
blocks' largest |x|.  silu has a slope below 1.1 and |silu(g)| <= |g|; its own
evaluation (expf within 2 units, a sum, a quotient, a product) adds 8u.  A
hidden value is then off by dh <= 1.1 dg |up| + |silu(g)| du + 8u |h| + dg du,
and rounded to q of its block's largest (q = 2^-23 f32, 2^-12 16-bit types).
The down product carries dh + q max|h| through sum |Wd|, adds its own sum's
error, and the result its type's half step.
"""
import pytest

import rocknpu_b200 as rk

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24


def blocks_of(n):
    return (n + 127) // 128


def stack(e, n, k, seed):
    """Random e4m3 codes (every finite value) and block scales of about 1 / (100 sqrt(k))."""
    g = torch.Generator().manual_seed(seed)
    code = torch.randint(0, 256, (e, n, k), generator=g, dtype=torch.uint8)
    code = torch.where(code & 0x7F == 0x7F, code - 1, code)
    s = (torch.rand((e, blocks_of(n), blocks_of(k)), generator=g) + 0.5) / (100.0 * k ** 0.5)
    return code.view(torch.float8_e4m3fn).cuda(), s.cuda()


def values(w, s):
    n, k = w.shape[-2:]
    return w.float().double() * s.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]


def block_max(x):
    """Each value replaced by the largest magnitude of its block of 128."""
    n, k = x.shape
    p = torch.nn.functional.pad(x.abs(), (0, blocks_of(k) * 128 - k)).view(n, -1, 128)
    return p.amax(2, keepdim=True).expand_as(p).reshape(n, -1)[:, :k]


def reference(x, gate, up, down, ids, weights):
    """The formula in f64 and its bound."""
    f32 = x.dtype == torch.float32
    x = x.double()
    r, q = (2.0 ** -23, 2.0 ** -23) if f32 else (2.0 ** -24, 2.0 ** -12)
    y, bound = torch.zeros_like(x), torch.zeros_like(x)
    for ex in range(gate[0].shape[0]):
        for slot in range(ids.shape[1]):
            rows = (ids[:, slot] == ex).nonzero()[:, 0]
            if rows.numel() == 0:
                continue
            xs, xb = x[rows], block_max(x[rows])
            wg, wu, wd = (values(w[ex], s[ex]) for w, s in (gate, up, down))
            n = xs.shape[1]
            c = (128 + 3 * blocks_of(n) + 2) * 2 * U
            g, u = xs @ wg.t(), xs @ wu.t()
            dg = r * (xb @ wg.abs().t()) + c * (xs.abs() @ wg.abs().t())
            du = r * (xb @ wu.abs().t()) + c * (xs.abs() @ wu.abs().t())
            silu = g * torch.sigmoid(g)
            h = silu * u
            dh = 1.1 * dg * u.abs() + silu.abs() * du + 1.1 * dg * du + 8 * U * h.abs()
            dh = dh + q * (block_max(h) + dh.amax(1, keepdim=True))
            c = (128 + 3 * blocks_of(h.shape[1]) + 2) * 2 * U
            p = weights[rows, slot:slot + 1].double()
            d = h @ wd.t()
            dd = dh @ wd.abs().t() + c * ((h.abs() + dh) @ wd.abs().t())
            y[rows] += p * d
            # the slot's weight (exp, sum, quotient) and its multiply-add
            bound[rows] += p * (dd + 16 * U * d.abs())
    return y, bound


def check(out, ids, weights, x, gate, up, down):
    y, bound = reference(x, gate, up, down, ids, weights)
    if x.dtype != torch.float32:
        bound = bound + torch.finfo(x.dtype).eps / 2 * (y.abs() + bound) + 2.0 ** -25
    err = (out.double() - y).abs()
    assert torch.isfinite(out).all()
    assert (err <= bound + 1e-30).all(), f"max excess {(err / (bound + 1e-30)).max()}"


def layer(t, h, f, e, top, type_, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((t, h), generator=g)
    x[:, torch.rand(h, generator=g) < 0.01] *= 20.0
    return (x.to(TYPES[type_]).cuda(), stack(e, f, h, seed + 1), stack(e, f, h, seed + 2), stack(e, h, f, seed + 3),
            (torch.randn((e, h), generator=g) / h ** 0.5).cuda())


def workspace(t, h, f, e, top, dtype):
    from rocknpu_b200 import device as dev
    n = dev.moe_f8_workspace_bytes(t, h, f, e, top, dtype)
    assert n > 0
    return dev.new_workspace(n)


def check_routing(x, router, ids, weights, renorm):
    """Choices and weights against f64 logits: a choice may differ only where
    two logits are as close as an f32 sum can tell."""
    logits = x.double() @ router.double().t()
    near = 2.0 ** -23 * 64 * (x.double().abs() @ router.double().abs().t()).amax()
    got = logits.gather(1, ids.long())
    best = logits.sort(1, descending=True).values[:, :ids.shape[1]]
    assert ((got - best).abs() <= near).all()
    assert all(len(set(row)) == len(row) for row in ids.tolist())
    base = got if renorm else logits
    p = torch.exp(got - torch.logsumexp(base, 1, keepdim=True))
    assert ((weights.double() - p).abs() <= (2 * near + 32 * U) * p).all()


SHAPES = [(1, 256, 128, 1, 1), (1, 2048, 5632, 8, 2), (1, 16, 16, 4, 4), (2, 144, 272, 5, 2), (7, 512, 1024, 64, 8),
          (8, 400, 96, 3, 3), (9, 640, 384, 8, 2), (16, 1024, 640, 16, 4), (17, 256, 2240, 4, 1), (33, 768, 256, 8, 3),
          (64, 512, 512, 8, 2), (64, 272, 144, 256, 16), (64, 1536, 512, 2, 2)]


@pytest.mark.parametrize("type_", list(TYPES))
@pytest.mark.parametrize("t,h,f,e,top", SHAPES)
def test_layer_with_router(type_, t, h, f, e, top):
    from rocknpu_b200 import device as dev
    x, gate, up, down, router = layer(t, h, f, e, top, type_, seed=t + f)
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    for renorm in (True, False):
        out, ids, weights = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top, renormalize=renorm)
        assert status.item() == 0
        check_routing(x, router, ids, weights, renorm)
        check(out, ids, weights, x, gate, up, down)
        again = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top, renormalize=renorm)
        assert torch.equal(out, again[0]) and torch.equal(ids, again[1]) and torch.equal(weights, again[2])
        assert not ws[:65536].any()


@pytest.mark.parametrize("type_", list(TYPES))
@pytest.mark.parametrize("t,h,f,e,top", [(1, 256, 256, 4, 2), (5, 512, 320, 8, 3), (20, 256, 512, 6, 2), (64, 384, 256, 3, 2)])
def test_layer_routed_from_outside(type_, t, h, f, e, top):
    """Empty slots, an empty token, the same expert twice."""
    from rocknpu_b200 import device as dev
    x, gate, up, down, _ = layer(t, h, f, e, top, type_, seed=7)
    g = torch.Generator().manual_seed(t)
    ids = torch.randint(-1, e, (t, top), generator=g, dtype=torch.int32)
    weights = torch.rand((t, top), generator=g)
    if t > 1:
        ids[t // 2] = -1
        ids[0, :2] = 1
    weights[ids < 0] = float("nan")  # says nothing
    ids, weights = ids.cuda(), weights.cuda()
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    out, got_ids, got_w = dev.moe_f8(x, gate, up, down, status, ws, ids=ids, weights=weights)
    assert status.item() == 0 and got_ids is ids and got_w is weights
    check(out, ids, torch.nan_to_num(weights), x, gate, up, down)
    if t > 1:
        assert (out[t // 2] == 0).all()


def test_all_tokens_on_one_expert_twice():
    """64 tokens with both slots on one expert: 128 pairs, two passes over its weights."""
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 64, 256, 384, 4, 2
    x, gate, up, down, _ = layer(t, h, f, e, top, "bf16", seed=3)
    ids = torch.full((t, top), 2, dtype=torch.int32, device="cuda")
    weights = torch.rand((t, top), device="cuda")
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    out, _, _ = dev.moe_f8(x, gate, up, down, status, ws, ids=ids, weights=weights)
    assert status.item() == 0
    check(out, ids, weights, x, gate, up, down)


def test_no_slot_used():
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 3, 256, 256, 4, 2
    x, gate, up, down, _ = layer(t, h, f, e, top, "f32")
    ids = torch.full((t, top), -1, dtype=torch.int32, device="cuda")
    out = torch.full((t, h + 8), 5.0, device="cuda")
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    dev.moe_f8(x, gate, up, down, status, ws, ids=ids, weights=torch.ones((t, top), device="cuda"), out=out[:, :h])
    assert status.item() == 0 and (out[:, :h] == 0).all() and (out[:, h:] == 5).all()


@pytest.mark.parametrize("type_", list(TYPES))
def test_padded_rows_may_hold_anything(type_):
    """Tokens whose slots are all empty: NaN and infinities in their rows of x
    and in their weights change nothing and set no status."""
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 11, 272, 160, 4, 3
    x, gate, up, down, _ = layer(t, h, f, e, top, type_, seed=3)
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, e, (t, top), generator=g, dtype=torch.int32)
    weights = torch.rand((t, top), generator=g)
    pad = [0, 4, 5, 10]
    ids[pad] = -1
    ids[1, 0] = -7
    ids, weights = ids.cuda(), weights.cuda()
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    plain, _, _ = dev.moe_f8(x, gate, up, down, status, ws, ids=ids, weights=weights)
    x[0], x[4, 7], x[5], x[10, ::3] = float("nan"), float("inf"), -float("inf"), float("nan")
    weights[pad], weights[1, 0] = float("nan"), float("inf")
    out, _, _ = dev.moe_f8(x, gate, up, down, status, ws, ids=ids, weights=weights)
    assert status.item() == 0
    assert torch.equal(out, plain) and (out[pad] == 0).all()
    x[1, 3] = float("nan")
    dev.moe_f8(x, gate, up, down, status, ws, ids=ids, weights=weights)
    assert status.item() == 1


def test_logits_of_both_zeros_are_equal():
    """Products that underflow to -0 and to +0 take the lower expert too."""
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 2, 256, 256, 6, 3
    x, gate, up, down, _ = layer(t, h, f, e, top, "f32")
    x = torch.full_like(x, 1e-30)
    router = torch.full((e, h), 1e-30, device="cuda")
    router[::2] *= -1.0
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    _, ids, _ = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top)
    assert status.item() == 0
    assert torch.equal(ids.cpu(), torch.arange(top, dtype=torch.int32).expand(t, top))


@pytest.mark.parametrize("raw", [False, True])
def test_given_stream_owns_the_results(raw):
    """A call with a stream allocates on it: results reuse no block that work
    on the current stream may still read."""
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 3, 512, 256, 4, 2
    x, gate, up, down, router = layer(t, h, f, e, top, "bf16")
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    want = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    busy = torch.randn((4096, 4096), device="cuda")
    for _ in range(20):
        busy = busy @ busy * 1e-2
    held = torch.empty_like(want[0])
    address = held.data_ptr()
    del held  # free for the current stream, whose queue is long
    out, ids, weights = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top,
                                   stream=side.cuda_stream if raw else side)
    side.synchronize()
    assert out.data_ptr() != address
    assert torch.equal(out, want[0]) and torch.equal(ids, want[1]) and torch.equal(weights, want[2])
    a8, a_s = dev.quantize_rows_f8(x, status, stream=side)
    w8, w_s = dev.prepare_f8(router, status, stream=side)
    one = dev.gemm_f8(a8, a_s, w8, w_s, status, stream=side)
    need = dev.matmul_f8_workspace_bytes(t, e, h)
    with torch.cuda.stream(side):
        own = dev.new_workspace(need)
    two = dev.matmul_f8(x, w8, w_s, status, own, out_dtype=torch.float32, stream=0 if raw else side)
    torch.cuda.synchronize()
    assert torch.equal(one, two) and status.item() == 0


def test_out_in_place_of_x():
    """x is read before anything is stored: out may be x."""
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 19, 384, 256, 4, 2
    x, gate, up, down, router = layer(t, h, f, e, top, "f32")
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    want = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top)
    got = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top, out=x)
    assert got[0].data_ptr() == x.data_ptr()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and status.item() == 0


def test_index_out_of_range_sets_status():
    from rocknpu_b200 import device as dev
    from rocknpu_b200 import lib
    t, h, f, e, top = 2, 256, 256, 4, 2
    x, gate, up, down, _ = layer(t, h, f, e, top, "f32")
    ids = torch.tensor([[0, 4], [1, 2]], dtype=torch.int32, device="cuda")
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    dev.moe_f8(x, gate, up, down, status, ws, ids=ids, weights=torch.ones((t, top), device="cuda"))
    assert status.item() == 9 and lib().rocknpu_b200_status_code(9) == rk.STATUS_INVALID_ARGUMENT
    assert not ws[:65536].any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_non_finite_input_sets_status(bad):
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 5, 256, 256, 8, 3
    x, gate, up, down, router = layer(t, h, f, e, top, "f32")
    x[3, 77] = bad
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    _, ids, _ = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top)
    assert status.item() == 1 and ((ids >= 0) & (ids < e)).all()
    assert not ws[:65536].any()


def test_equal_logits_take_the_lower_expert():
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 4, 256, 256, 40, 5
    x, gate, up, down, router = layer(t, h, f, e, top, "f32")
    router = router[:1].expand(e, h).contiguous()
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    _, ids, weights = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top)
    assert status.item() == 0
    assert torch.equal(ids.cpu(), torch.arange(top, dtype=torch.int32).expand(t, top))
    assert ((weights - 1.0 / top).abs() <= 8 * U).all()


@pytest.mark.parametrize("router_type", list(TYPES))
def test_strides_and_router_types(router_type):
    """Experts cut out of wider tensors, x and out in wider rows."""
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 6, 272, 160, 4, 2
    x, _, _, _, router = layer(t, h, f, e, top, "f16")
    x = torch.nn.functional.pad(x, (3, 5))[:, 3:3 + h]
    wide = stack(2 * e, f + 32, h + 48, 11)
    gate = (wide[0][::2, :f, 16:16 + h], stack(e, f, h, 12)[1])
    both = stack(e, 2 * f, h, 13)[0]
    up = (both[:, f:], stack(e, f, h, 14)[1])
    down = stack(e, h, f, 15)
    wide_router = torch.nn.functional.pad(router.to(TYPES[router_type]), (1, 2))
    out = torch.full((t, h + 7), 3.0, dtype=torch.float16, device="cuda")
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    _, ids, weights = dev.moe_f8(x, gate, up, down, status, ws, router=wide_router[:, 1:1 + h], top_k=top,
                                 out=out[:, 2:2 + h])
    assert status.item() == 0
    check_routing(x, wide_router[:, 1:1 + h].float(), ids, weights, True)
    check(out[:, 2:2 + h], ids, weights, x, gate, up, down)
    assert (out[:, :2] == 3).all() and (out[:, 2 + h:] == 3).all()


def test_graph_replay_and_side_stream():
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 3, 512, 768, 8, 2
    x, gate, up, down, router = layer(t, h, f, e, top, "f32", seed=1)
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, ids, weights = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top)
    for seed in range(3):
        x.copy_(torch.randn((t, h), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert status.item() == 0
        check_routing(x, router, ids, weights, True)
        check(out, ids, weights, x, gate, up, down)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top)
    side.synchronize()
    assert torch.equal(got[0], out)


def test_two_layers_in_flight_on_two_streams():
    """Two calls with their own workspaces queued on two streams at once."""
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 4, 512, 512, 8, 2
    calls = []
    for seed in (1, 2):
        x, gate, up, down, router = layer(t, h, f, e, top, "f32", seed=seed)
        calls.append((x, gate, up, down, router, workspace(t, h, f, e, top, x.dtype), dev.new_status(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        for x, gate, up, down, router, ws, status, stream in calls:
            with torch.cuda.stream(stream):
                got.append(dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top))
    torch.cuda.synchronize()
    for i, (x, gate, up, down, _, _, status, _) in enumerate(calls):
        assert status.item() == 0
        for out, ids, weights in got[i::2]:
            check(out, ids, weights, x, gate, up, down)


def test_experts_prepared_from_kquants_and_dense():
    """Gate from Q4_K, up from Q6_K, down dense, then the layer and, on its
    output, a product: the operators in the order of a model's step."""
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 5, 512, 256, 4, 2
    status = dev.new_status()

    def kq(kind, seed):
        ws, ss = [], []
        for ex in range(e):
            blocks = torch.from_numpy(rk.synth_q_weights(kind, f, h, seed=seed + ex)).cuda()
            w, s = dev.prepare_f8_q(kind, blocks, h, f, status)
            ws.append(w)
            ss.append(s)
        return torch.stack(ws), torch.stack(ss)

    gate, up = kq(rk.Q4_K, 10), kq(rk.Q6_K, 20)
    down = dev.prepare_f8((torch.randn((e, h, f), device="cuda") * 0.05).bfloat16(), status)
    head = dev.prepare_f8(torch.randn((1000, h), device="cuda") * 0.05, status)
    x = torch.randn((t, h), device="cuda")
    router = torch.randn((e, h), device="cuda") / h ** 0.5
    ws = dev.new_workspace(max(dev.moe_f8_workspace_bytes(t, h, f, e, top, x.dtype),
                               dev.matmul_f8_workspace_bytes(t, 1000, h)))
    y, ids, weights = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top)
    logits = dev.matmul_f8(y, *head, status, ws)
    y2, _, _ = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top)
    assert status.item() == 0 and torch.equal(y, y2)
    check(y, ids, weights, x, gate, up, down)
    q, s = dev.quantize_rows_f8(y, status)
    ref = (q.float().double() * s.double().repeat_interleave(128, 1)) @ values(*head).t()
    assert ((logits.double() - ref).abs() <= 1e-5 * ref.abs().max()).all()


@pytest.mark.parametrize("type_", list(TYPES))
def test_zero_and_tiny_tokens(type_):
    """A token of zeros, one near the bottom of f16, hidden values of widely
    different sizes in one block (gate rows scaled group by group)."""
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 4, 384, 272, 3, 2
    x, gate, up, down, router = layer(t, h, f, e, top, type_, seed=21)
    x[1] = 0
    x[2] *= 1e-4
    up[0].view(torch.uint8)[:, 16:32] = 0                       # a group of zero hidden values
    up[0].view(torch.uint8)[:, 32:48] &= 0x87                   # a group of small ones
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    out, ids, weights = dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top)
    assert status.item() == 0 and (out[1] == 0).all()
    check(out, ids, weights, x, gate, up, down)


def test_beside_other_work():
    """Layers on one stream while products keep the SMs busy on another."""
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 9, 512, 512, 8, 2
    x, gate, up, down, router = layer(t, h, f, e, top, "f32", seed=4)
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    big = torch.randn((4096, 4096), device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        with torch.cuda.stream(side):
            big @ big
        got.append(dev.moe_f8(x, gate, up, down, status, ws, router=router, top_k=top))
    torch.cuda.synchronize()
    assert status.item() == 0
    for out, ids, weights in got:
        assert torch.equal(out, got[0][0])
    check(*got[0], x, gate, up, down)


def test_refusals():
    from rocknpu_b200 import device as dev
    t, h, f, e, top = 4, 256, 128, 4, 2
    x, gate, up, down, router = layer(t, h, f, e, top, "f32")
    status, ws = dev.new_status(), workspace(t, h, f, e, top, x.dtype)
    ids = torch.zeros((t, top), dtype=torch.int32, device="cuda")
    weights = torch.ones((t, top), device="cuda")

    def call(x=x, gate=gate, up=up, down=down, ws=ws, **kw):
        return dev.moe_f8(x, gate, up, down, status, ws, **kw)

    for kw in (dict(), dict(router=router), dict(router=router, top_k=0), dict(router=router, top_k=2, ids=ids),
               dict(router=router[:3], top_k=2), dict(router=router.double(), top_k=2), dict(ids=ids),
               dict(ids=ids.long(), weights=weights), dict(ids=ids, weights=weights[:, :1]),
               dict(ids=ids, weights=weights, top_k=1), dict(ids=ids[:3], weights=weights[:3]),
               dict(ids=ids, weights=weights, x=x.double()), dict(ids=ids, weights=weights, gate=(gate[0][0], gate[1])),
               dict(ids=ids, weights=weights, up=down), dict(ids=ids, weights=weights, down=(down[0], down[1][:3])),
               dict(ids=ids, weights=weights, out=torch.empty((t, h), device="cuda", dtype=torch.float16)),
               dict(ids=ids.cpu(), weights=weights)):
        with pytest.raises(ValueError):
            call(**kw)
            pytest.fail(f"{list(kw)} was accepted")
    for kw in (dict(router=router, top_k=5), dict(ids=ids, weights=weights, ws=ws[:1000]),
               dict(ids=torch.zeros((65, 2), dtype=torch.int32, device="cuda"), weights=torch.ones((65, 2), device="cuda"),
                    x=torch.randn((65, h), device="cuda"))):
        with pytest.raises(RuntimeError):
            call(**kw)
    assert status.item() == 0
