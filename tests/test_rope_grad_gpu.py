"""Gradients through ``rope``: what autograd gives equals the inverse rotation of the
outputs' gradients, for tensors as a model leaves them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _plain(x, pos, tab, interleaved):
    """fp64 rotation of [tokens, H, D] in torch operations."""
    R = tab.shape[1]
    inside = ((pos >= 0) & (pos < tab.shape[0]))[:, None, None]
    row = tab.double()[pos.clamp(0, tab.shape[0] - 1).long()][:, None]
    c, s = row[..., :R // 2], row[..., R // 2:]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    u, w = a * c - b * s, a * s + b * c
    turned = torch.stack([u, w], -1).flatten(-2) if interleaved else torch.cat([u, w], -1)
    return torch.where(inside, torch.cat([turned, x[..., R:]], -1), x)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("with_k", [True, False])
def test_rope_backward(interleaved, with_k):
    """Gradients of slices of one projection against fp64 autograd of the formula.  fp32: the forward and the backward
    are off by at most 2^-21 of a row's largest each (two products and a sum, 2^-22 (|a| + |b|)); the loss is linear, so
    only the backward's error counts."""
    import blackwell_b200 as bw
    T, Hq, Hkv, D, R = 19, 4, 2, 32, 16
    tab = bw.rope_table(16, R, scaling="yarn", factor=4.0, original_length=8)
    pos = torch.randint(-2, 18, (T,), generator=torch.Generator().manual_seed(1)).int().cuda()
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).cuda().requires_grad_()
    wq, wk = torch.randn(T, Hq, D, generator=g).cuda(), torch.randn(T, Hkv, D, generator=g).cuda()

    def split(x):
        return x[:, :Hq * D].view(T, Hq, D), x[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)

    q, k = split(qkv)
    qo, ko = bw.rope(q, k if with_k else None, tab, positions=pos, interleaved=interleaved)
    loss = (qo * wq).sum() + ((ko * wk).sum() if with_k else 0)
    got, = torch.autograd.grad(loss, qkv)
    x = qkv.detach().double().requires_grad_()
    q, k = split(x)
    want = (_plain(q, pos, tab, interleaved) * wq).sum()
    if with_k:
        want = want + (_plain(k, pos, tab, interleaved) * wk).sum()
    want, = torch.autograd.grad(want, x)
    m = max(1.0, float(tab.abs().max()))
    assert (got.double() - want).abs().max() <= 2.0 ** -20 * m * float(torch.cat([wq.flatten(), wk.flatten()]).abs().max())


def test_rope_backward_of_broadcast_and_unused_outputs():
    """A gradient that arrives expanded (of a sum), one output that the loss does not use, bf16, BSHD."""
    import blackwell_b200 as bw
    B, S, Hq, Hkv, D = 2, 7, 3, 1, 64
    tab = bw.rope_table(7, 64)
    q = torch.randn(B, S, Hq, D, device="cuda").bfloat16().requires_grad_()
    k = torch.randn(B, S, Hkv, D, device="cuda").bfloat16().requires_grad_()
    qo, ko = bw.rope(q.transpose(1, 2), k.transpose(1, 2), tab)
    qo.sum().backward()
    ones = torch.ones(B, Hq, S, D, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(q.grad, bw.rope(ones, None, tab, inverse=True)[0].transpose(1, 2))
    assert k.grad is None
    q.grad = None
    qo, ko = bw.rope(q.transpose(1, 2), k.transpose(1, 2), tab)
    ko.sum().backward()
    assert q.grad is None or not q.grad.any()
    assert torch.equal(k.grad, bw.rope(ones[:, :Hkv], None, tab, inverse=True)[0].transpose(1, 2))


def test_rope_gradient_is_differentiable_and_checked():
    """Twice differentiable (it is linear); differences of the call itself; an input changed between the passes is noticed."""
    import blackwell_b200 as bw
    tab = bw.rope_table(9, 16)
    pos = torch.tensor([0, 3, 8], dtype=torch.int32).cuda()
    x = torch.randn(3, 2, 32, device="cuda").requires_grad_()
    w = torch.randn(3, 2, 32, device="cuda").requires_grad_()
    y = bw.rope(x, None, tab, positions=pos)[0]
    gx, = torch.autograd.grad((y * w).sum(), x, create_graph=True)
    z = torch.randn_like(x)
    gw, = torch.autograd.grad((gx * z).sum(), w)
    assert torch.equal(gw, bw.rope(z, None, tab, positions=pos)[0])
    for e in (0, 7, 8, 15, 16, 31):
        d = torch.zeros_like(x)
        d[..., e] = 1.0
        with torch.no_grad():
            diff = (bw.rope(x + d, None, tab, positions=pos)[0].double() - bw.rope(x - d, None, tab, positions=pos)[0].double()) / 2
        # fp32 rounding of x +- d and of both rotations, 2^-21 (|x| + 1) a value, over at most 2 rotated values of w
        tol = 2.0 ** -19 * (float(x.abs().max()) + 1) * float(w.abs().max())
        assert ((diff * w.double()).sum(-1) - gx[..., e].double()).abs().max() <= tol
    y = bw.rope(x, None, tab, positions=pos)[0]
    pos += 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


def test_rope_backward_in_a_graph():
    """Forward and backward captured and replayed with new inputs."""
    import blackwell_b200 as bw
    tab = bw.rope_table(64, 64)
    pos = torch.arange(33, dtype=torch.int32).cuda()
    w = torch.randn(33, 4, 64, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = torch.randn(33, 4, 64, device="cuda").requires_grad_()
        torch.autograd.grad((bw.rope(x, None, tab, positions=pos)[0] * w).sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g, = torch.autograd.grad((bw.rope(x, None, tab, positions=pos)[0] * w).sum(), x)
    w.copy_(torch.randn_like(w))
    pos += 20
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(g, bw.rope(w, None, tab, positions=pos, inverse=True)[0])


def test_rope_without_gradients_is_as_before():
    """No graph under no_grad or for plain inputs; given outputs and in place work there."""
    import blackwell_b200 as bw
    tab = bw.rope_table(8, 16)
    x = torch.randn(5, 2, 16, device="cuda")
    y = bw.rope(x, None, tab)[0]
    assert not y.requires_grad
    x.requires_grad_()
    with pytest.raises(ValueError, match="gradient"):
        bw.rope(x, None, tab, q_out=torch.empty_like(y))
    with torch.no_grad():
        z = bw.rope(x, None, tab)[0]
        bw.rope(x, None, tab, q_out=x)
    assert not z.requires_grad and torch.equal(z, y) and torch.equal(x, y)
