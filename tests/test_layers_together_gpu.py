"""Products of e4m3 rows, gradients against differences and of second order, unusual layouts, streams, graphs, and the
operators as they are used together: rows kept in 8 bits, normed, decoded, trained and served."""
import pytest
import torch

import layer_bounds as lb

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def rand(g, *s):
    return torch.randn(*s, generator=g, device=DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(1, 64, 64), (3, 100, 7), (4, 256, 33), (5, 16, 16), (130, 128, 64), (129, 130, 131),
                                   (257, 1040, 264), (64, 3, 5), (1000, 144, 48),
                                   (64, 4096, 40), (65, 5001, 33), (30, 2500, 130)])       # sums split over several SMs
def test_quantised_product(m, k, n, dtype):
    import ash

    g = gen(m + k + n)
    for j, act in enumerate(("none", "relu", "silu", "gelu", "sin")):
        x, w = ash.quantize_rows(rand(g, m, k)), ash.quantize_rows(rand(g, n, k) / k**0.5)
        b = rand(g, n).to(dtype) if j % 2 else None
        r = rand(g, m, n).to(dtype) if j % 3 else None
        got = ash.fused_linear(x, w, b, activation=act, residual=r, omega=2.0, dtype=dtype)
        assert got.dtype == dtype and got.shape == (m, n)
        xd, wd = (q.codes.to(lb.D) * q.scales.to(lb.D)[:, None] for q in (x, w))
        z, mag = xd @ wd.T, xd.abs() @ wd.abs().T
        if b is not None:
            z, mag = z + b.to(lb.D), mag + b.to(lb.D).abs()
        # sums of codes 32 at a time, parts of 512 or more joined, the two scales' product and the bias: rounded operations
        ez = (k / 32 + k / 512 + 8) * lb.STEP * mag + lb.TINY
        omega = 2.0 if act == "sin" else 1.0
        a, _, l1, _ = lb.activation(z, act, omega)
        y = a if r is None else a + r.to(lb.D)
        lb.assert_within(got, y, lb.forward_bound(y, z, a, ez, l1, act, r, omega, dtype), f"{act}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype):
    """Rows with strides, odd offsets, three dimensions, expanded residuals: the same numbers as of plain copies."""
    import ash

    g = gen(3)
    big = rand(g, 70, 400).to(dtype)
    w0 = rand(g, 65, 131).to(dtype)
    for m, k, n in ((50, 128, 64), (50, 63, 33), (2, 63, 33)):
        for xo, wo in ((0, 0), (1, 3), (8, 8)):
            x, w = big[:m, xo:xo + k], w0[:n, :k] if wo == 0 else w0[1:n + 1, wo:wo + k] if wo + k <= 131 else w0[:n, :k]
            r = big[:m, 200:200 + n]
            b = big[0, 1:n + 1]
            got = ash.fused_linear(x, w, b, "silu", r)
            want = ash.fused_linear(x.clone(), w.clone(), b.clone(), "silu", r.clone())
            y, z, a, d, ez, l1, _ = lb.linear(x, w, b, "silu", r, 1.0)
            bound = lb.forward_bound(y, z, a, ez, l1, "silu", r, 1.0, dtype)
            lb.assert_within(got, y, bound, "strided")
            lb.assert_within(want, y, bound, "plain")
    x, w = rand(g, 2, 5, 7, 16).to(dtype), rand(g, 24, 16).to(dtype)
    assert ash.fused_linear(x, w).shape == (2, 5, 7, 24) and ash.fused_linear(x[0, 0, 0], w).shape == (24,)
    assert torch.equal(ash.fused_linear(x.transpose(0, 2), w), ash.fused_linear(x, w).transpose(0, 2))
    one = rand(g, 24).to(dtype).requires_grad_(True)      # a residual shared by all rows, an input shared by two layers
    x2 = rand(g, 40, 16).to(dtype).requires_grad_(True)
    y = ash.fused_linear(x2, w, residual=one.expand(40, 24)) + ash.fused_linear(x2, w.clone())
    gx, go = torch.autograd.grad(y.float().sum(), [x2, one])
    assert torch.equal(go, torch.full_like(go, 40.0))
    want = 2 * w.float().sum(0).to(lb.D)
    lb.assert_within(gx, want.expand(40, 16), (w.abs().to(lb.D).sum(0) * 2 * (40 * lb.STEP + 2 * lb.half(dtype))).expand(40, 16), "x")
    t = ash.fused_linear(x2, w0[:16, :24].t()[:, :].contiguous().t()[:, :16])   # a weight that is a transposed view
    assert t.shape == (40, 16)


def test_empty_and_single():
    import ash

    for dtype in (torch.float32, torch.float16):
        w = torch.randn(5, 8, device=DEV, dtype=dtype, requires_grad=True)
        b = torch.randn(5, device=DEV, dtype=dtype, requires_grad=True)
        x = torch.zeros(0, 8, device=DEV, dtype=dtype, requires_grad=True)
        y = ash.fused_linear(x, w, b, "gelu")
        assert y.shape == (0, 5)
        gx, gw, gb = torch.autograd.grad(y.sum(), [x, w, b])
        assert gx.shape == (0, 8) and not bool(gw.any()) and not bool(gb.any())
        assert ash.fused_linear(torch.zeros(2, 0, 8, device=DEV, dtype=dtype), w).shape == (2, 0, 5)
    q = ash.quantize_rows(torch.zeros(0, 8, device=DEV))
    assert ash.fused_linear(q, ash.quantize_rows(torch.ones(5, 8, device=DEV))).shape == (0, 5)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "sin"])
def test_gradient_against_differences(act):
    """Central differences of float64 values of the formula, at the kernel's inputs: h^2/6 |f'''| with h = 2^-10, |f'''| of
    order omega^3, and the gradient's own float32 error."""
    import ash

    g = gen(4)
    x, w, b, r, dy = rand(g, 6, 10), rand(g, 7, 10) / 3, rand(g, 7), rand(g, 6, 7), rand(g, 6, 7)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    grads = torch.autograd.grad(ash.fused_linear(x, w, b, act, r, omega=2.0), leaves, dy)
    u = [rand(g, *t.shape) for t in leaves]
    h = 2.0**-10
    ends = []
    for sign in (1, -1):
        t = [a.detach().to(lb.D) + sign * h * d.to(lb.D) for a, d in zip(leaves, u)]
        z = t[0] @ t[1].T + t[2]
        ends.append(((lb.activation(z, act, 2.0 if act == "sin" else 1.0)[0] + t[3]) * dy.to(lb.D)).sum())
    numeric = ((ends[0] - ends[1]) / (2 * h)).item()
    found = sum((a.to(lb.D) * d.to(lb.D)).sum() for a, d in zip(grads, u)).item()
    size = sum((a.to(lb.D) * d.to(lb.D)).abs().sum() for a, d in zip(grads, u)).item()
    slack = 5e-3 if act == "relu" else 1e-3        # relu: a value within h of its corner
    assert abs(numeric - found) <= slack * size


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "sin"])
def test_second_order(act):
    """A gradient of a gradient, as an eikonal term takes it, against torch's own in 64 bits."""
    import ash

    g = gen(6)
    x, w, b, v = rand(g, 33, 6), rand(g, 9, 6) / 2, rand(g, 9), rand(g, 9)
    om = 1.5

    def term(fn, x, w, b, v):
        y = fn(x, w, b)
        gx, = torch.autograd.grad((y * v).sum(), x, create_graph=True)
        return ((gx.norm(dim=1) - 1) ** 2).sum()

    def plain(x, w, b):
        z = x @ w.T + b
        return {"none": lambda: z, "relu": lambda: z.relu(), "silu": lambda: torch.nn.functional.silu(z),
                "gelu": lambda: torch.nn.functional.gelu(z), "sin": lambda: torch.sin(om * z)}[act]()

    a = [t.clone().requires_grad_(True) for t in (x, w, b)]
    e = [t.to(lb.D).requires_grad_(True) for t in (x, w, b)]
    # another tensor holds the activation's own place in the chain: the inner gradient passes through both layers
    got = torch.autograd.grad(term(lambda x, w, b: ash.fused_linear(x, w, b, act, omega=om), *a, v), a, allow_unused=True)
    want = torch.autograd.grad(term(plain, *e, v.to(lb.D)), e, allow_unused=True)
    for p, q in zip(got, want):
        if q is None or p is None:
            assert (p is None or not bool(p.any())) and (q is None or not bool(q.any()))
            continue
        # float32 sums of at most a few hundred terms through two layers: 2^-24 x 2^9 of the largest
        assert (p.to(lb.D) - q).abs().max() <= 2.0**-15 * max(1.0, q.abs().max().item())


@pytest.mark.parametrize("act", ["none", "silu"])
def test_second_order_without_rows(act):
    import ash

    x, w, b = torch.empty(0, 6, device=DEV), torch.ones(9, 6, device=DEV), torch.ones(9, device=DEV)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(ash.fused_linear(x, w, b, act).sum(), leaves, create_graph=True)
    assert [tuple(t.shape) for t in grads] == [(0, 6), (9, 6), (9,)]
    assert not grads[1].any() and not grads[2].any()


def test_streams_and_graph():
    """On a stream of its own, two at once, and captured: the same bits."""
    import ash

    g = gen(8)
    x, w, b, dy = rand(g, 3000, 48), rand(g, 80, 48), rand(g, 80), rand(g, 3000, 80)
    nw = torch.ones(48, device=DEV)

    def step(x):
        n = ash.rms_norm(x, nw)
        leaves = [t.detach().requires_grad_(True) for t in (n, w, b)]
        y = ash.fused_linear(*leaves, "gelu")
        return [y.detach(), *torch.autograd.grad(y, leaves, dy), *ash.rms_norm(x, nw, quantize=True)]

    want = step(x)
    x2 = x.flip(0).contiguous()
    want2 = step(x2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            a = step(x)
        with torch.cuda.stream(s2):
            c = step(x2)
    torch.cuda.synchronize()
    same = lambda p, q: torch.equal(p.view(torch.uint8), q.view(torch.uint8))
    assert all(same(p, q) for p, q in zip(a, want)) and all(same(p, q) for p, q in zip(c, want2))
    graph, graph2, held = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        out = step(held)
    with torch.cuda.graph(graph2):
        out2 = step(held)
    for src, expect in ((x2, want2), (x, want)):
        held.copy_(src)
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        assert all(same(p, q) for p, q in zip(out, expect)) and all(same(p, q) for p, q in zip(out2, expect))


def test_map_rows_in_a_graph():
    import ash

    n = 2000
    i = torch.arange(n, device=DEV)
    keys = torch.stack([i % 13, i // 13 % 13, i // 169], 1).int()
    m = ash.HashMap(3, 32, n, DEV, value_formats="e4m3")
    m.insert(keys, rand(gen(1), n, 32))
    want = m.find(keys, return_values=True)
    m.find(keys, return_values=True)
    torch.cuda.synchronize()
    graph, asked = torch.cuda.CUDAGraph(), keys.clone()
    with torch.cuda.graph(graph):
        got = m.find(asked, return_values=True)
    asked.copy_(keys.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q.flip(0)) for p, q in zip(got, want))


def test_huge_offsets():
    """Codes, values and rows whose offsets pass 2^31."""
    import ash

    n, width = 9_000_000, 256              # 2.3e9 codes
    m = ash.HashMap(1, width, n, DEV, value_formats="int8")
    keys = torch.arange(n, device=DEV, dtype=torch.int32)[:, None]
    for at in range(0, n, 1_000_000):
        k = keys[at:at + 1_000_000]
        m.insert(k, (k.float() * 0.25).expand(-1, width).contiguous())
    some = torch.cat([keys[:1000], keys[-1000:], keys[::9973]])
    masks, indices, rows = m.find(some, return_values=True)
    assert bool(masks.all()) and int(indices.max()) * width > 2**31
    want = some.float() * 0.25
    scale = (want * (torch.tensor(1.0, device=DEV) / torch.tensor(127.0, device=DEV))).clamp_min(2.0**-126)
    assert torch.equal(rows, (torch.round(want * (1.0 / scale)) * scale).expand(-1, width))
    del m, keys
    torch.cuda.empty_cache()
    rows, width = 1_100_000, 2048          # 2.25e9 values of 2 bytes
    x = torch.ones(rows, width, device=DEV, dtype=torch.bfloat16)
    x[-1] = 2
    x[:, 0] = 3
    w = torch.ones(width, device=DEV, dtype=torch.bfloat16)
    y = ash.rms_norm(x, w)
    assert torch.equal(y[-1], ash.rms_norm(x[-1:].clone(), w)[0]) and torch.equal(y[-2], y[0])
    wt = torch.zeros(16, width, device=DEV, dtype=torch.bfloat16)
    wt[:, 0] = 1
    wt[3, 5] = 1
    y = ash.fused_linear(x, wt)
    assert y.shape == (rows, 16) and bool((y[:, 0] == 3).all()) and y[-1, 3].item() == 5 and y[0, 3].item() == 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_norm_and_head_together(dtype):
    """Feature rows kept as e4m3 in a hash map, read back by key, decoded by a residual head; served in 8 bits too."""
    import ash

    g = gen(12)
    n = 5000
    i = torch.arange(n, device=DEV)
    keys = torch.stack([i % 20, i // 20 % 20, i // 400], 1).int()
    table = ash.HashMap(3, 32, n, DEV, value_formats="e4m3")
    table.insert(keys, rand(g, n, 32))
    asked = torch.cat([keys[::2], keys[:100] + 1000])
    masks, rows = table.find(asked, return_indices=False, return_values=True, value_dtype=dtype)
    assert bool(masks[:-100].all()) and not bool(masks[-100:].any())
    torch.manual_seed(0)
    head = ash.ResidualMLP(32, 64, 4, 2, expansion=2, device=DEV, dtype=dtype)
    y = head(rows)

    def plain(head, rows):
        lin = lambda layer, x: x @ layer.weight.to(lb.D).T + layer.bias.to(lb.D)
        h = lin(head.first_layer, rows)
        for norm, up, down in zip(head.norms, head.up, head.down):
            u = h / torch.sqrt((h * h).mean(1, keepdim=True) + head.eps) * norm.to(lb.D)
            h = h + lin(down, torch.nn.functional.silu(lin(up, u)))
        return lin(head.last_layer, h / torch.sqrt((h * h).mean(1, keepdim=True) + head.eps) * head.norms[-1].to(lb.D))

    want = plain(head, rows.to(lb.D))
    # seven products in a row, each rounded once (its input's rounding again): in norm 2 x 9 half steps at most
    assert (y.to(lb.D) - want).norm() <= (18 * lb.half(dtype) + 2.0**-20) * want.norm()
    (y.float() ** 2).mean().backward()
    grads = {name: p.grad.to(lb.D) for name, p in head.named_parameters()}
    for p in head.parameters():
        p.grad = None
    params = {name: p.detach().to(lb.D).requires_grad_(True) for name, p in head.named_parameters()}
    copy = ash.ResidualMLP(32, 64, 4, 2, expansion=2, device="cpu", dtype=lb.D).to(DEV)
    copy.load_state_dict({k: v.detach() for k, v in params.items()})
    (plain(copy, rows.to(lb.D)) ** 2).mean().backward()
    for name, p in copy.named_parameters():
        # twice the layers' roundings on the way back, on top of those on the way there
        assert (grads[name] - p.grad).norm() <= (60 * lb.half(dtype) + 2.0**-18) * p.grad.norm(), name
    with torch.no_grad():
        served = head.quantize_()(rows)
        # four products of two operands rounded to e4m3 each: 2^-4 of a value at most, a third of that in norm
        assert (served.to(lb.D) - want).norm() <= 8 * 2.0**-4 / 1.7 * want.norm() and not torch.equal(served, y)
        assert torch.equal(head.quantize_(False)(rows), y)


def test_networks():
    """The modules over grid features and positions: shapes, gradients of positions, and an eikonal step."""
    import ash

    torch.manual_seed(1)
    net = ash.SirenNet(3, 32, 1, 3, device=DEV)
    x = (torch.rand(300, 3, device=DEV) * 2 - 1).requires_grad_(True)
    sdf = net(x)
    gx, = torch.autograd.grad(sdf.sum(), x, create_graph=True)
    (gx.norm(dim=1) - 1).abs().mean().backward()
    # a bias reaches the gradient of positions only through its layer's slope: the last layer's has none
    unused = {name for name, p in net.named_parameters() if p.grad is None or not bool(p.grad.any())}
    assert unused == {"last_layer.bias"}
    mlp = ash.MLP(16, 64, 4, 2, residual=True, device=DEV)
    emb = ash.HashEmbedding(3, 100, 16, DEV)
    keys = torch.arange(60, device=DEV, dtype=torch.int32)[:, None].expand(60, 3).contiguous()
    emb.spatial_init_(keys)
    out = mlp(emb(keys))
    out.sum().backward()
    assert out.shape == (60, 4) and bool(emb.embedding.grad.any()) and all(p.grad is not None for p in mlp.parameters())
    grid = ash.UnBoundedSparseDenseGrid(3, 64, 16, 8, cell_size=0.1, device=DEV)
    pts = torch.rand(500, 3, device=DEV)
    grid.spatial_init_(pts)
    with torch.no_grad():
        grid.embeddings.normal_(0, 0.1)
    p = pts.clone().requires_grad_(True)
    feat, mask = grid(p, interpolation="linear")
    loss = mlp(feat)[mask].pow(2).mean()
    loss.backward()
    assert bool(grid.embeddings.grad.any()) and bool(p.grad.any())


def test_tangents_and_transforms_are_refused():
    import ash
    import torch.autograd.forward_ad as fwd

    x, w = torch.randn(9, 8, device=DEV), torch.randn(5, 8, device=DEV)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: ash.fused_linear(d, w), lambda: ash.rms_norm(d, w[0]), lambda: ash.rms_norm(d, w[0], quantize=True),
                     lambda: ash.fused_linear(d, w.clone().requires_grad_(True))):
            with pytest.raises(RuntimeError):
                call()
        assert torch.equal(ash.fused_linear(x, w), ash.fused_linear(x, w))      # none among the tensors
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: ash.fused_linear(t, w))(x[None])


def test_no_wait_ran_out():
    import __ash

    assert __ash.layer_timeouts(DEV) == 0
