"""The mixture-of-experts layer's hidden values, held with 22 bits relative to
the largest of their group of 16.

Bound for one output, as in the layer's other tests (u = 2^-24, S(.) the same
sum over magnitudes), with the rounding of a hidden value relative to its own
16 values:
- x is off by at most r of its block of 128's largest (f32: two f16 terms,
  r = 2^-23; 16-bit types: one, r = 2^-39);
- a product sum over n values is off by (128 + 3 n / 128 + 2) 2u of S;
- silu has a slope below 1.1, |silu(g)| <= |g|, and 8u for its evaluation;
- a hidden value is two f16 terms of its group's power of two, which puts the
  group's largest in [2^14, 2^15): the remainder is at most 2^3 and rounded to
  2^-9, 2^-23 of 2^14.  Where the block of 128 has a larger group, both terms
  are multiplied by a power of two of 2^-14 or more, and rounded again where
  that gives less than 2^-14: 2^-25 each, against 2^14 2^-14: 2^-24 together.
  q = 2^-23 + 2^-24.
"""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24
Q = 2.0 ** -23 + 2.0 ** -24


def blocks_of(n):
    return (n + 127) // 128


def largest(x, size):
    """Each value replaced by the largest magnitude of its `size` neighbours."""
    n, k = x.shape
    p = torch.nn.functional.pad(x.abs(), (0, (k + size - 1) // size * size - k)).view(n, -1, size)
    return p.amax(2, keepdim=True).expand_as(p).reshape(n, -1)[:, :k]


def values(w, s):
    n, k = w.shape[-2:]
    return w.float().double() * s.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]


def check(out, x, gate, up, down, ids, weights):
    r = 2.0 ** -23 if x.dtype == torch.float32 else 2.0 ** -39
    x64 = x.double()
    y, bound = torch.zeros_like(x64), torch.zeros_like(x64)
    for ex in range(gate[0].shape[0]):
        wg, wu, wd = (values(w[ex], s[ex]) for w, s in (gate, up, down))
        for slot in range(ids.shape[1]):
            rows = (ids[:, slot] == ex).nonzero()[:, 0]
            if rows.numel() == 0:
                continue
            xs, xb = x64[rows], largest(x64[rows], 128)
            c = (128 + 3 * blocks_of(xs.shape[1]) + 2) * 2 * U
            g, u = xs @ wg.t(), xs @ wu.t()
            dg = r * (xb @ wg.abs().t()) + c * (xs.abs() @ wg.abs().t())
            du = r * (xb @ wu.abs().t()) + c * (xs.abs() @ wu.abs().t())
            silu = g * torch.sigmoid(g)
            h = silu * u
            dh = 1.1 * dg * u.abs() + silu.abs() * du + 1.1 * dg * du + 8 * U * h.abs()
            dh = dh + Q * largest(h.abs() + dh, 16)
            c = (128 + 3 * blocks_of(h.shape[1]) + 2) * 2 * U
            p = weights[rows, slot:slot + 1].double()
            d = h @ wd.t()
            y[rows] += p * d
            bound[rows] += p * (dh @ wd.abs().t() + c * ((h.abs() + dh) @ wd.abs().t()) + 16 * U * d.abs())
    if x.dtype != torch.float32:
        # half a step of the result's type (f16: at least half its smallest subnormal)
        bound = bound + torch.finfo(x.dtype).eps / 2 * (y.abs() + bound) + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    err = (out.double() - y).abs()
    assert torch.isfinite(out).all()
    assert (err <= bound).all(), f"max excess {(err / bound.clamp_min(1e-300)).max()}"


def run(x, gate, up, down, ids, weights):
    from rocknpu_b200 import device as dev
    t, h = x.shape
    e, f, _ = gate[0].shape
    status = dev.new_status()
    ws = dev.new_workspace(dev.moe_f8_workspace_bytes(t, h, f, e, ids.shape[1], x.dtype))
    out, _, _ = dev.moe_f8(x, gate, up, down, status, ws, ids=ids, weights=weights)
    assert status.item() == 0
    return out


def codes(v):
    """e4m3 weights of scale 1 from values that are e4m3 numbers."""
    q = v.to(torch.float8_e4m3fn)
    assert torch.equal(q.float(), v)
    s = torch.ones((*v.shape[:-2], blocks_of(v.shape[-2]), blocks_of(v.shape[-1])))
    return q.cuda(), s.cuda()


def routing(t, e, top, g):
    return (torch.randint(0, e, (t, top), generator=g, dtype=torch.int32).cuda(),
            torch.rand((t, top), generator=g).cuda())


@pytest.mark.parametrize("type_", list(TYPES))
@pytest.mark.parametrize("t,e,top", [(1, 1, 1), (4, 1, 1), (8, 2, 1), (13, 2, 2), (30, 2, 1), (64, 2, 2), (64, 1, 1)])
def test_nearly_equal_hidden_values(type_, t, e, top):
    """Differences of hidden values that agree in their first ten bits: down
    rows take one from another, so their distance is the result."""
    g = torch.Generator().manual_seed(t)
    h, f = 48, 144
    x = torch.zeros((t, h))
    x[:, 0] = 1.0
    x[:, 1] = 2.0 ** -10 * torch.randint(1, 4, (t,), generator=g)
    gate, up, down = torch.zeros((e, f, h)), torch.zeros((e, f, h)), torch.zeros((e, h, f))
    gate[:, :, 0] = 1.0
    up[:, :, 0] = 1.0
    up[:, :, 1] = torch.randint(0, 17, (e, f), generator=g).float()  # u = 1 + j x1
    for ex in range(e):
        for i in range(h):
            a, b = torch.randperm(f, generator=g)[:2].tolist()
            down[ex, i, a], down[ex, i, b] = 1.0, -1.0
    ids, weights = routing(t, e, top, g)
    x = x.to(TYPES[type_]).cuda()
    w = codes(gate), codes(up), codes(down)
    check(run(x, *w, ids, weights), x, *w, ids, weights)


@pytest.mark.parametrize("type_", list(TYPES))
@pytest.mark.parametrize("t,e,top", [(1, 1, 1), (3, 2, 1), (8, 1, 1), (13, 2, 2), (30, 2, 1), (64, 2, 2)])
def test_groups_far_below_their_neighbours(type_, t, e, top):
    """Groups of 16 hidden values down to 2^-70 of the others in their block of
    128 (f16: 2^-24), and groups of zeros; each down row looks at one group only."""
    g = torch.Generator().manual_seed(100 + t)
    far = [0, 3, 13, 14, 15, 20, 24, None] if type_ == "f16" else [0, 13, 14, 16, 27, 45, 70, None]
    h, f = 8 * 128, 272
    x = torch.zeros((t, h))
    for tok in range(t):
        for i in range(8):
            d = far[(i + tok) % 8]  # another order per token
            x[tok, 128 * i + 1] = 0.0 if d is None else 2.0 ** -d
    x[:, 0] = 1.0
    group = torch.arange(f) // 16 % 8
    gate, up = torch.zeros((e, f, h)), torch.zeros((e, f, h))
    gate[:, :, 0] = torch.randint(1, 5, (e, f), generator=g).float()
    up[:, torch.arange(f), 128 * group + 1] = torch.randint(1, 17, (e, f), generator=g).float()
    down = torch.randint(-16, 17, (e, h, f), generator=g).float()
    down *= group[None, None, :] == (torch.arange(h) % 8)[None, :, None]
    ids, weights = routing(t, e, top, g)
    x = x.to(TYPES[type_]).cuda()
    w = codes(gate), codes(up), codes(down)
    check(run(x, *w, ids, weights), x, *w, ids, weights)


@pytest.mark.parametrize("type_", list(TYPES))
@pytest.mark.parametrize("t,h,f,e,top", [(1, 512, 640, 4, 2), (13, 512, 2240, 16, 4), (24, 640, 272, 2, 2), (64, 256, 512, 4, 2)])
def test_random_layers(type_, t, h, f, e, top):
    g = torch.Generator().manual_seed(t + f)

    def stack(n, k):
        code = torch.randint(0, 256, (e, n, k), generator=g, dtype=torch.uint8)
        code = torch.where(code & 0x7F == 0x7F, code - 1, code)
        s = (torch.rand((e, blocks_of(n), blocks_of(k)), generator=g) + 0.5) / (100.0 * k ** 0.5)
        return code.view(torch.float8_e4m3fn).cuda(), s.cuda()

    x = torch.randn((t, h), generator=g).to(TYPES[type_]).cuda()
    w = stack(f, h), stack(f, h), stack(h, f)
    ids, weights = routing(t, e, top, g)
    check(run(x, *w, ids, weights), x, *w, ids, weights)
