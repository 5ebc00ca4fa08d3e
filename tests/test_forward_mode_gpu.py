"""Forward-mode derivatives: the rotation has them, the attentions and the append refuse what they would lose."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("needs", [(True, True), (True, False), (False, True)])
def test_the_tangent_of_a_rotation_is_the_rotated_tangent(needs, inverse):
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(48, scaling="yarn", factor=4.0, trained_length=512)
    p = torch.randint(0, 5000, (2, 9), device="cuda")
    q, k, dq, dk = (torch.randn(2, h, 9, 64, device="cuda") for h in (4, 2, 4, 2))
    plain, turned = ma.rotary_b200(q, k, r, p, inverse=inverse), ma.rotary_b200(dq, dk, r, p, inverse=inverse)
    with fwAD.dual_level():
        x = [fwAD.make_dual(t, d) if n else t for t, d, n in zip((q, k), (dq, dk), needs)]
        out = [fwAD.unpack_dual(t) for t in ma.rotary_b200(*x, r, p, inverse=inverse)]
    for a, t, d, n in zip(out, plain, turned, needs):
        assert torch.equal(a.primal, t)
        assert torch.equal(a.tangent, d) if n else a.tangent is None


def test_a_tangent_beside_a_gradient():
    """Forward over reverse: both are there, and the tangent of the gradient is the inverse rotation of the tangent."""
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(64)
    q, dq, w = (torch.randn(1, 2, 5, 64, device="cuda") for _ in range(3))
    with fwAD.dual_level():
        x = fwAD.make_dual(q.clone().requires_grad_(True), dq)
        y, _ = ma.rotary_b200(x, None, r)
        assert y.requires_grad and torch.equal(fwAD.unpack_dual(y).tangent, ma.rotary_b200(dq, None, r)[0])
        (g,) = torch.autograd.grad(y, x, w)
        assert torch.equal(fwAD.unpack_dual(g).primal, ma.rotary_b200(w, None, r, inverse=True)[0])


def test_the_gradients_own_tangent():
    """The gradient's operation is a rotation too: a dual gradient comes out with its tangent turned back."""
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(64)
    q = torch.randn(1, 2, 5, 64, device="cuda", requires_grad=True)
    w, dw = (torch.randn(1, 2, 5, 64, device="cuda") for _ in range(2))
    y, _ = ma.rotary_b200(q, None, r)
    with fwAD.dual_level():
        (g,) = torch.autograd.grad(y, q, fwAD.make_dual(w, dw))
        assert torch.equal(fwAD.unpack_dual(g).tangent, ma.rotary_b200(dw, None, r, inverse=True)[0])


def test_no_tangent_outside_a_dual_level_or_without_one():
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(64)
    q, dq = (torch.randn(1, 2, 5, 64, device="cuda") for _ in range(2))
    with fwAD.dual_level():
        plain, _ = ma.rotary_b200(q, None, r)
        assert fwAD.unpack_dual(plain).tangent is None
        kept, _ = ma.rotary_b200(fwAD.make_dual(q, dq), None, r)
    assert torch.equal(kept, ma.rotary_b200(q, None, r)[0])


def test_a_tangent_of_zeros_that_has_no_memory():
    import monarch_attention_b200 as ma
    r = ma.RotaryPositions(64)
    q = torch.randn(1, 2, 5, 64, device="cuda")
    with fwAD.dual_level():
        y, _ = ma.rotary_b200(fwAD.make_dual(q, torch._efficientzerotensor(q.shape, device="cuda")), None, r)
        primal, tangent = fwAD.unpack_dual(y)
        assert torch.equal(primal, ma.rotary_b200(q, None, r)[0]) and tangent.shape == q.shape and not bool(tangent.any())


def test_what_has_no_forward_derivative_is_refused():
    """A tangent that would be lost without a word: the attention of the encoder, the append, the attention over the cache."""
    import monarch_attention_b200 as ma
    module = ma.MonarchAttention(16, 2, ma.PadType.post)
    x = [torch.randn(1, 2, 64, 64, device="cuda") for _ in range(3)]
    cache = ma.PagedKV.allocate(4, 2, 64, 16)
    table, lengths = torch.arange(4, dtype=torch.int32, device="cuda").view(1, 4), torch.full((1,), 5, dtype=torch.int32, device="cuda")
    t = torch.randn(1, 2, 5, 64, device="cuda").to(torch.bfloat16)
    with fwAD.dual_level():
        for i in range(3):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                module(*(fwAD.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(x)))
        d = fwAD.make_dual(t, torch.ones_like(t))
        for call in (lambda: ma.append_kv_b200(cache, d, t, table, lengths), lambda: ma.append_kv_b200(cache, t, d, table, lengths),
                     lambda: ma.append_kv_b200(cache, t, t, table, lengths, query=d), lambda: ma.cached_attention_b200(d, cache, table, lengths)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        assert module(*x).shape == x[0].shape   # (a dual level alone asks for nothing)
        ma.append_kv_b200(cache, t, t, table, lengths)
    with torch.no_grad(), fwAD.dual_level():   # (forward mode goes on without the reverse)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ma.cached_attention_b200(fwAD.make_dual(t, torch.ones_like(t)), cache, table, lengths)
