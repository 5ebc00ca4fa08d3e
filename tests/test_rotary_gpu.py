"""Rotary positions: kernels against the definition in 64 bits, gradients against the formula and against differences."""
import pytest
import torch

from decoder_reference import HALF_STEP, close, rotate, rotation_bound

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def heads(E, H, N, D, dtype, layout, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "tokens":
        return torch.randn(E, N, H, D, generator=g, device="cuda").to(dtype).permute(0, 2, 1, 3)
    if layout == "odd":     # rows on odd boundaries
        return torch.randn(E, H, N, D + 3, generator=g, device="cuda").to(dtype)[..., 1:D + 1]
    if layout == "inner":   # features not next to one another
        return torch.randn(E, H, D, N, generator=g, device="cuda").to(dtype).transpose(-1, -2)
    return torch.randn(E, H, N, D, generator=g, device="cuda").to(dtype)


SHAPES = [  # E, H, Hk, N, D, dim
    (1, 1, 1, 1, 2, 2), (1, 12, 12, 33, 64, 64), (2, 3, 1, 17, 72, 72), (3, 5, 5, 16, 80, 40), (2, 8, 2, 15, 128, 64), (1, 2, 2, 100, 72, 36),
    (1, 1, 1, 7, 6, 2), (2, 4, 4, 31, 33, 30), (1, 7, 1, 40, 256, 256), (5, 40, 8, 129, 64, 64), (1, 3, 3, 5, 300, 256)]


@pytest.mark.parametrize("layout", ["heads", "tokens", "odd", "inner"])
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,H,Hk,N,D,dim", SHAPES)
def test_rotation_matches_the_definition(E, H, Hk, N, D, dim, dtype, pairs, layout):
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(dim, pairs=pairs)
    q, k = heads(E, H, N, D, dtype, layout, 1), heads(E, Hk, N, D, dtype, layout, 2)
    before = q.clone(), k.clone()
    out = ma.rotary_b200(q, k, r)
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    for x, y in zip((q, k), out):
        want, size = rotate(x, torch.arange(N), r)
        assert y.shape == x.shape and y.dtype == x.dtype
        close(y, want, rotation_bound(want, size, dtype))
        assert torch.equal(y[..., dim:], x[..., dim:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scaling,factor", [(None, 1.0), ("linear", 8.0), ("ntk", 4.0), ("yarn", 16.0)])
@pytest.mark.parametrize("kind", ["int64", "int32", "row", "one"])
def test_positions_and_scalings(kind, scaling, factor, dtype):
    """Far, negative and unordered positions; the angles stay exact."""
    import monarch_attention_b200 as ma
    E, H, N, D = 3, 4, 37, 64
    r = ma.RotaryPositions(D, scaling=scaling, factor=factor, trained_length=4096)
    g = torch.Generator(device="cuda").manual_seed(3)
    p = torch.randint(-2 ** 30, 2 ** 30, (E, N), generator=g, device="cuda")
    p[0, :5] = torch.tensor([0, 1, -1, 2 ** 30, -2 ** 30])
    p = {"int64": p, "int32": p.to(torch.int32), "row": p[1], "one": p[1:2]}[kind]
    q, k = heads(E, H, N, D, dtype, "tokens", 4), heads(E, 1, N, D, dtype, "heads", 5)
    for x, y in zip((q, k), ma.rotary_b200(q, k, r, p)):
        # the definition's own angle: p * f in 64 bits is off by 2^-53 of up to 2^30 radians, 2^-23
        want, size = rotate(x, (p if p.dim() == 2 else p[None])[:, None], r)
        close(y, want, rotation_bound(want, size, dtype) + 2.0 ** -23 * size)


def test_strided_positions_and_only_a_query():
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(32, pairs="interleaved")
    p = torch.arange(200, device="cuda").view(100, 2)[:, 1][None, 10:50].expand(3, -1)
    q = heads(3, 2, 40, 32, torch.float32, "heads", 1)
    y, none = ma.rotary_b200(q, None, r, p)
    want, size = rotate(q, p[:, None], r)
    assert none is None
    close(y, want, rotation_bound(want, size, torch.float32))


def test_empty_inputs():
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(8)
    for shape in ((0, 2, 3, 8), (1, 2, 0, 8), (1, 0, 3, 8)):
        q, k = ma.rotary_b200(torch.zeros(shape, device="cuda"), None, r)
        assert q.shape == shape and k is None


@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("needs", [(True, True), (True, False), (False, True)])
def test_gradients_match_the_formula(needs, dtype, pairs):
    import monarch_attention_b200 as ma
    E, H, Hk, N, D = 2, 6, 2, 19, 64
    r = ma.RotaryPositions(48, pairs=pairs, scaling="yarn", factor=4.0, trained_length=2048)
    p = torch.randint(0, 100000, (E, N), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    q, k = heads(E, H, N, D, dtype, "tokens", 1).requires_grad_(needs[0]), heads(E, Hk, N, D, dtype, "heads", 2).requires_grad_(needs[1])
    out = ma.rotary_b200(q, k, r, p)
    assert (out[0].requires_grad, out[1].requires_grad) == needs
    grads = [heads(*o.shape, dtype, "tokens", 7 + i) for i, o in enumerate(out)]
    torch.autograd.backward([o for o, n in zip(out, needs) if n], [g for g, n in zip(grads, needs) if n])
    for x, g, n in zip((q, k), grads, needs):
        if not n:
            assert x.grad is None
            continue
        want, size = rotate(g, p[:, None], r, inverse=True)
        close(x.grad, want, rotation_bound(want, size, dtype))


def test_gradients_match_differences():
    """Linear, so a difference over any step is exact but for rounding: <grad, d> = <w, f(x + d) - f(x)>."""
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(64)
    q = heads(1, 2, 9, 64, torch.float32, "heads", 1).requires_grad_(True)
    w, d = heads(1, 2, 9, 64, torch.float32, "heads", 2), heads(1, 2, 9, 64, torch.float32, "heads", 3)
    y, _ = ma.rotary_b200(q, None, r)
    (dq,) = torch.autograd.grad(y, q, w)
    z, _ = ma.rotary_b200(q.detach() + d, None, r)
    moved = float((w.double() * (z.double() - y.detach().double())).sum())
    size = float((w.abs().double() * (z.abs() + y.detach().abs()).double()).sum()) * 2
    assert abs(moved - float((dq.double() * d.double()).sum())) <= 16 * 2.0 ** -24 * size


def test_gradient_of_expanded_and_shared_inputs_and_of_the_gradient():
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(16)
    one = torch.randn(1, 1, 5, 16, device="cuda", requires_grad=True)
    y, z = ma.rotary_b200(one.expand(3, 4, 5, 16), one.expand(3, 2, 5, 16), r)
    (y.sum() + z.sum()).backward()   # (the gradient of a sum has strides of zero)
    want, size = rotate(torch.ones(1, 1, 5, 16), torch.arange(5), r, inverse=True)
    # 12 + 6 gradients of one value each, summed in 32 bits
    close(one.grad, 18 * want, 18 * (rotation_bound(want, size, torch.float32) + 18 * 2.0 ** -24 * want.abs()))
    x = torch.randn(1, 2, 5, 16, device="cuda", requires_grad=True)
    y, _ = ma.rotary_b200(x, None, r)
    (dx,) = torch.autograd.grad(y.pow(2).sum(), x, create_graph=True)   # 2 x
    (ddx,) = torch.autograd.grad(dx.sum(), x)
    assert torch.allclose(ddx, torch.full_like(ddx, 2.0), atol=1e-5)
    # only one of two results used: the other's input has a gradient of its own
    q, k = (torch.randn(1, 2, 5, 16, device="cuda", requires_grad=True) for _ in range(2))
    a, _ = ma.rotary_b200(q, k, r)
    a.sum().backward()
    assert q.grad is not None and k.grad is None


def test_attention_module_rotates_queries_and_keys():
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(64)
    x = [heads(2, 3, 197, 64, torch.bfloat16, "tokens", s).requires_grad_(True) for s in range(3)]
    plain, turned = ma.MonarchAttention(15, 2, "pre"), ma.MonarchAttention(15, 2, "pre")
    turned.rotary = r
    q, k = ma.rotary_b200(x[0], x[1], r)
    want, got = plain(q, k, x[2]), turned(*x)
    assert torch.equal(want, got)
    w = heads(2, 3, 197, 64, torch.bfloat16, "heads", 9)
    for a, b in zip(torch.autograd.grad(want, x, w), torch.autograd.grad(got, x, w)):
        assert torch.equal(a, b)


def test_capture_streams_and_replay():
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(64)
    q, k = heads(2, 4, 50, 64, torch.bfloat16, "tokens", 1), heads(2, 2, 50, 64, torch.bfloat16, "tokens", 2)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        out = ma.rotary_b200(q, k, r)
    for seed in (5, 6):
        q.copy_(heads(2, 4, 50, 64, torch.bfloat16, "tokens", seed))
        graph.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = ma.rotary_b200(q, k, r)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])


def test_refusals():
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(64)
    q = torch.zeros(2, 3, 5, 64, device="cuda")
    for bad, error in [(dict(query=q[0]), ValueError), (dict(query=q.double()), ValueError), (dict(key=q[:1]), ValueError), (dict(key=q.half()), ValueError),
                       (dict(key=q[..., :32]), ValueError), (dict(key=q.cpu()), ValueError), (dict(query=q[..., :32]), ValueError),
                       (dict(positions=torch.zeros(2, 4, device="cuda", dtype=torch.int64)), ValueError),
                       (dict(positions=torch.zeros(5, device="cuda")), ValueError), (dict(positions=torch.zeros(5, dtype=torch.int64)), ValueError),
                       (dict(positions=torch.zeros(3, 5, device="cuda", dtype=torch.int32)), ValueError), (dict(rotary=None), TypeError),
                       (dict(query=q.cpu()), RuntimeError)]:
        with pytest.raises(error):
            ma.rotary_b200(**{**dict(query=q, key=None, rotary=r), **bad})


def test_half_steps_are_the_types_own():
    for t, h in HALF_STEP.items():
        assert torch.finfo(t).eps / 2 == h


def test_training_step_is_captured_and_replayed():
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(64)
    q, k = (heads(2, 4, 50, 64, torch.float32, "tokens", s).requires_grad_(True) for s in (1, 2))
    w = heads(2, 4, 50, 64, torch.float32, "heads", 3)
    eager = torch.autograd.grad(ma.rotary_b200(q, k, r), (q, k), (w, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = torch.autograd.grad(ma.rotary_b200(q, k, r), (q, k), (w, w))
    for t in grads:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, grads))


@pytest.mark.parametrize("expanded", [(3, 4, 5), (3, 1, 5), (1, 4, 5), (1, 1, 5), (3, 4, 1)])
def test_expanded_inputs_of_all_kinds(expanded):
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(8, pairs="interleaved")
    x = torch.randn(*expanded, 16, device="cuda").expand(3, 4, 5, 16)
    y, z = ma.rotary_b200(x, x.transpose(0, 1).contiguous().transpose(0, 1), r)
    want, size = rotate(x, torch.arange(5), r)
    close(y, want, rotation_bound(want, size, torch.float32))
    assert torch.equal(y, z) and y.stride(-1) == 1
