"""The sequence operators together, as a decoder layer and its loss use them: gradients through the differentiable forms
(simvg_amd/models/sequence.py), against the same layer in 64 bits and against differences of its own loss."""
import pytest
import torch

from simvg_amd.models import sequence as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
Hq, Hkv, D, E, V = 4, 2, 64, 128, 700
SECTIONS = (8, 12, 12)
LENS = [37, 1, 0, 90, 64]


def layer(p, x, pos, inv, target, attend, norm_rope, loss):
    """x [T, E] -> q, k, v -> normalised and rotated -> packed causal attention -> projection, residual -> loss over the words"""
    qkv = x @ p["wqkv"]
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1))
    q, k = norm_rope(q, k, pos, inv, p["gq"], p["gk"])
    y = x + attend(q, k, v).flatten(1) @ p["wo"]
    return loss(y, p["words"], target, p["bias"])


def problem(dt, seed=0, tail=11):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T = sum(LENS) + tail
    r = lambda *s, std: (torch.randn(*s, generator=g, device=DEV) * std)  # noqa: E731
    p = dict(wqkv=r(E, (Hq + 2 * Hkv) * D, std=E ** -0.5).to(dt), wo=r(Hq * D, E, std=(Hq * D) ** -0.5).to(dt), words=r(V, E, std=E ** -0.5).to(dt),
             bias=r(V, std=0.1), gq=1 + r(D, std=0.1), gk=1 + r(D, std=0.1))
    x = r(T, E, std=1.0).to(dt)
    pos = torch.randint(0, 50, (T, 3), generator=g, device=DEV, dtype=torch.int32)
    inv = 10000.0 ** (-torch.arange(32, device=DEV, dtype=torch.float64) / 32)
    target = torch.randint(0, V, (T,), generator=g, device=DEV)
    target[sum(LENS):] = -100
    target[::7] = -100
    cu = torch.tensor([sum(LENS[:i]) for i in range(len(LENS) + 1)], dtype=torch.int32, device=DEV)
    return p, x, pos, inv, target, cu


def own_loss(p, x, pos, inv, target, cu):
    plan = S.packed_plan(cu, x.shape[0])
    return layer(p, x, pos, inv, target, lambda q, k, v: S.packed_attention(q, k, v, plan),
                 lambda q, k, pos, inv, gq, gk: S.qk_norm_rope(q, k, pos, inv, SECTIONS, gq, gk), S.vocab_cross_entropy)


def exact_loss(p, x, pos, inv, target):
    import sequence_ref as R

    def attend(q, k, v):
        out, at = [], 0
        for n in LENS:
            s = torch.matmul(q[at:at + n].transpose(0, 1), k[at:at + n].repeat_interleave(Hq // Hkv, 1).permute(1, 2, 0)) * D ** -0.5
            s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1), float("-inf"))
            out.append(torch.matmul(s.softmax(-1), v[at:at + n].repeat_interleave(Hq // Hkv, 1).transpose(0, 1)).transpose(0, 1))
            at += n
        return torch.cat(out + [torch.zeros_like(q[at:])])

    def norm_rope(q, k, pos, inv, gq, gk):
        return tuple(R.rope(t, g, pos, inv, SECTIONS, 1e-6, False)[0] for t, g in ((q, gq), (k, gk)))
    return layer(p, x, pos, inv, target, attend, norm_rope, lambda y, w, t, b: torch.nn.functional.cross_entropy(y @ w.t() + b, t))


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
def test_layer_and_loss_against_64_bits(dt):
    p, x, pos, inv, target, cu = problem(dt)
    scale = 1024.0                                            # a gradient scale, as 16-bit training carries
    leaves = {n: t.clone().requires_grad_() for n, t in (p | {"x": x}).items()}
    loss = own_loss({n: leaves[n] for n in p}, leaves["x"], pos, inv, target, cu)
    (loss * scale).backward()
    exact = {n: t.double().requires_grad_() for n, t in (p | {"x": x}).items()}
    want = exact_loss({n: exact[n] for n in p}, exact["x"], pos, inv, target)
    (want * scale).backward()
    # y is rounded to the type once, and so are qkv, the rotated heads and the attention: the loss averages a hundred rows of them
    h = torch.finfo(dt).eps / 2
    assert abs(float(loss) - float(want)) <= 8 * h
    for n, t in leaves.items():
        e = exact[n].grad
        # seven roundings in a row lie between a leaf and the loss and as many on the way back, each at most half a step of its value:
        # as independent errors sqrt(14) half steps of the gradient's norm, and twice that for what softmax and norm pass on
        off = float((t.grad.double() - e).norm() / e.norm())
        assert off <= 2 * 14 ** 0.5 * h, (n, off)
        assert t.grad.dtype == t.dtype and t.grad.shape == t.shape
    assert not leaves["x"].grad[sum(LENS):].any()             # rows behind the last sequence, all ignored


def test_gradients_against_differences():
    """the norm weights and the bias are fp32 leaves: a step along the gradient changes the loss by its squared length"""
    p, x, pos, inv, target, cu = problem(torch.float16, seed=1)
    for n in ("gq", "gk", "bias"):
        leaf = p[n].clone().requires_grad_()
        own_loss(p | {n: leaf}, x, pos, inv, target, cu).backward()
        g = leaf.grad
        step = 0.25 / float(g.norm())
        up, down = (float(own_loss(p | {n: p[n] + s * step * g}, x, pos, inv, target, cu)) for s in (1, -1))
        slope = (up - down) / (2 * step)
        # the loss moves through 16-bit activations: half a step of them on a loss of 6.6, over a way of 0.5
        assert abs(slope / float(g.norm()) - float(g.norm())) <= 0.05 * float(g.norm()) + 2 * 2.0 ** -11 / 128 ** 0.5, (n, slope)


def test_only_what_is_asked_for_and_expanded_gradients():
    p, x, pos, inv, target, cu = problem(torch.bfloat16, seed=2)
    T = x.shape[0]
    plan = S.packed_plan(cu, T)
    q = torch.randn(T, Hq, D, device=DEV).bfloat16().requires_grad_()
    k, v = torch.randn(T, Hkv, D, device=DEV).bfloat16(), torch.randn(T, Hkv, D, device=DEV).bfloat16()
    S.packed_attention(q, k, v, plan).float().sum().backward()            # an expanded gradient
    assert q.grad is not None and bool(torch.isfinite(q.grad).all())
    y = S.qk_norm_rope(q, k, pos, inv, SECTIONS, p["gq"], p["gk"])
    y[0].float().sum().backward()                                        # no gradient comes for k
    x = x.requires_grad_()
    rows = S.vocab_cross_entropy(x, p["words"], target, reduction="none")
    assert rows.shape == (T,) and not rows[target == -100].any()
    total = S.vocab_cross_entropy(x, p["words"], target, reduction="sum")
    assert abs(float(total) - float(rows.sum())) <= 1e-4 * float(total)
    total.backward()
    assert x.grad is not None and p["words"].grad is None


def test_a_gradient_that_starts_anywhere():
    """contiguous, but 2 bytes off a multiple of 16: a part of a larger gradient"""
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v = (torch.randn(30, h, D, generator=g, device=DEV).bfloat16().requires_grad_() for h in (Hq, Hkv, Hkv))
    plan = S.packed_plan(torch.tensor([0, 30], dtype=torch.int32, device=DEV), 30)
    do = torch.randn(30 * Hq * D + 1, generator=g, device=DEV).bfloat16()
    want = torch.autograd.grad(S.packed_attention(q, k, v, plan), (q, k, v), do[1:].clone().view(30, Hq, D))
    got = torch.autograd.grad(S.packed_attention(q, k, v, plan), (q, k, v), do[1:].view(30, Hq, D))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    pos, inv = torch.zeros(30, 1, dtype=torch.int32, device=DEV), torch.ones(32, dtype=torch.float64, device=DEV)
    y = S.qk_norm_rope(q, k, pos, inv, (32,))
    got = torch.autograd.grad(y, (q, k), (do[1:].view(30, Hq, D), do[1:30 * Hkv * D + 1].view(30, Hkv, D)))
    assert torch.equal(got[0], do[1:].view(30, Hq, D)) and torch.equal(got[1], do[1:30 * Hkv * D + 1].view(30, Hkv, D))


def test_layer_and_gradients_in_a_captured_graph():
    p, x, pos, inv, target, cu = problem(torch.bfloat16, seed=4)
    leaves = {n: t.clone().requires_grad_() for n, t in p.items()}
    plan = S.packed_plan(cu, x.shape[0])

    def step():
        loss = layer(leaves, x, pos, inv, target, lambda q, k, v: S.packed_attention(q, k, v, plan),
                     lambda q, k, pos, inv, gq, gk: S.qk_norm_rope(q, k, pos, inv, SECTIONS, gq, gk),
                     lambda y, w, t, b: S.vocab_cross_entropy(y, w, t, b, reduction="none"))
        return (loss.detach(), *torch.autograd.grad(loss, list(leaves.values()), torch.ones_like(loss)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        x.mul_(1.25)
        graph.replay()
        torch.cuda.synchronize()
        # each result against the eager one, which is the same kernels on the same values
        assert all(torch.equal(a, b) for a, b in zip(out, step())), i
        torch.cuda.synchronize()
