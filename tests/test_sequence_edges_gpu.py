"""The sequence operators at calls that their documentation allows and that are easily got wrong."""
import ctypes as C

import pytest
import torch

import sequence_ref as R
from simvg_amd import _lib, hip_ops as ops
from simvg_amd.models import sequence as S
from test_sequence_gpu import BF16, DEV, F16, F32, attn_case, ce_case, gen, randn

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------------------ vocabulary loss

@pytest.mark.parametrize("value", [torch.finfo(F32).min, -1e30, -1e10, -1e6])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M,V", [(20, 900), (300, 1500)])
def test_words_masked_by_a_large_finite_bias(M, V, dt, value):
    """whole tiles of words whose bias is the type's lowest value, or any that leaves nothing of them: the loss and the gradients are those
    of the words that are left"""
    x, w, t, b, gl = ce_case(M, V, 64, dt, ignored=0.1)
    left = torch.zeros(V, dtype=torch.bool, device=DEV)
    left[:7] = left[500:600] = True
    words = left.nonzero().squeeze(1)
    t = torch.where(t == -100, t, words[t.clamp(min=0) % len(words)])
    place = torch.full((V,), -1, device=DEV)
    place[words] = torch.arange(len(words), device=DEV)
    b = torch.where(left, b, value)
    loss, lse = ops.vocab_ce_fwd(x, w, t, b)
    dx, dw, db = ops.vocab_ce_bwd(x, w, t, lse, gl, b)
    ref = R.vocab_ce(x, w[words], torch.where(t == -100, t, place[t.clamp(min=0)]), b[words], gl)
    got = dict(loss=loss, lse=lse, dx=dx, dw=dw[words], dbias=db[words])
    worst = {n: R.off(v, ref[n], ref["tol"][n]) for n, v in got.items()}
    assert max(worst.values()) <= 1, worst
    assert not dw[~left].any() and not db[~left].any()


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M", [20, 300])
@pytest.mark.parametrize("value", [1e5, 1e10, 1e30])
def test_a_word_far_above_the_others(M, dt, value):
    """its probability is 1, to the last bit: e is 1 there, -1 at the target and 0 elsewhere, all exact in 16 bits"""
    x, w, t, b, gl = ce_case(M, 900, 64, dt, ignored=0.0)
    word = 333
    b[word] = value
    loss, lse = ops.vocab_ce_fwd(x, w, t, b)
    dx, dw, db = ops.vocab_ce_bwd(x, w, t, lse, gl, b)
    e = torch.zeros(M, 900, device=DEV, dtype=torch.float64)
    e[:, word] = 1
    e[torch.arange(M, device=DEV), t] -= 1
    g, X, W = gl.double()[:, None], x.double(), w.double()
    # lse is the word's logit, rounded after 64 products and sums; a probability is off by that difference's exponential where the logits are
    # held to less than a unit, and is 1 or 0 where they are not (1e10 is a multiple of 1024)
    p = 0.0 if value > 1e9 else 4 * (64 + 8) * R.U * float((X.abs() @ W.abs().t()).max()) + 16 * R.U * value
    want, size = (g * (e @ W), (g * e).t() @ X, (g * e).sum(0)), (g * (e.abs() @ W.abs()), (g * e.abs()).t() @ X.abs(), (g * e.abs()).sum(0))
    assert R.off(dx, want[0], (p + (R.h(dt) if p else 0) + 300 * R.U) * size[0] + p * g * W[word].abs() + R.rounded(want[0], dt)) <= 1
    assert R.off(dw, want[1], (p + (R.h(dt) if p else 0) + 400 * R.U) * size[1] + p * (g * X.abs()).sum(0) + R.rounded(want[1], dt)) <= 1
    assert R.off(db, want[2], (p + 400 * R.U) * size[2] + p * g.sum()) <= 1
    assert bool((lse.double() - value).abs().max() <= 64 + 2 * R.U * value) and bool(torch.isfinite(loss).all())


@pytest.mark.parametrize("M", [20, 300])
def test_a_row_far_off_changes_no_bit_of_the_others(M):
    x, w, t, b, gl = ce_case(M, 900, 64, BF16, ignored=0.0)
    loss, lse = ops.vocab_ce_fwd(x, w, t, b)
    dx, _, _ = ops.vocab_ce_bwd(x, w, t, lse, gl, b)
    x2 = x.clone()
    x2[3] = x[3] * 2.0 ** 12                                               # logits of thousands
    loss2, lse2 = ops.vocab_ce_fwd(x2, w, t, b)
    dx2, _, _ = ops.vocab_ce_bwd(x2, w, t, lse2, gl, b)
    others = torch.arange(M, device=DEV) != 3
    assert float(lse2[3]) > 4096 and bool(torch.isfinite(dx2).all())
    assert torch.equal(loss2[others], loss[others]) and torch.equal(lse2[others], lse[others]) and torch.equal(dx2[others], dx[others])
    ref = R.vocab_ce(x2, w, t, b, gl)
    assert R.off(lse2, ref["lse"], ref["tol"]["lse"]) <= 1 and R.off(loss2, ref["loss"], ref["tol"]["loss"]) <= 1
    assert R.off(dx2, ref["dx"], ref["tol"]["dx"]) <= 1


# ------------------------------------------------------------------------------------------------------------------------ attention

@pytest.mark.parametrize("scale", [None, 1.0])
@pytest.mark.parametrize("dt,value", [(F16, torch.finfo(F16).min), (BF16, -1e10), (BF16, -1e30), (BF16, torch.finfo(BF16).min)])
@pytest.mark.parametrize("lens,Hq,Hkv", [([300], 2, 1), ([2500], 2, 1), ([70, 200, 65], 12, 4)], ids=["tiles", "parts", "batch"])
@pytest.mark.parametrize("causal", [True, False])
def test_tiles_of_large_negative_scores(causal, lens, Hq, Hkv, dt, value, scale):
    """the first keys of a sequence, whole tiles of them, have scores that leave nothing of their probability: every row that sees another
    key gets the bits that it gets where those scores are -inf"""
    q, k, v, do, cu = attn_case(lens, Hq, Hkv, 64, dt)
    q, k = q.clone(), k.clone()
    q[..., 0] = 1
    skip, T = 130 if lens[0] > 130 else 64, sum(lens)
    plan = ops.packed_plan(cu, T)

    def run(masked):
        k[:skip, :, 0] = masked
        o, lse = ops.packed_attn_fwd(q, k, v, plan, causal, scale)
        return (o, lse, *ops.packed_attn_bwd(q, k, v, o, lse, do, plan, causal, scale))
    o, lse, dq, dk, dv = run(value)
    wo, wlse, wdq, wdk, wdv = run(float("-inf"))
    rows = slice(skip if causal else 0, T)                                  # those that see another key
    assert bool(torch.isfinite(wo[rows]).all()) and bool(torch.isfinite(wdk[skip:]).all())
    assert torch.equal(o[rows], wo[rows]) and torch.equal(lse[:, rows], wlse[:, rows])
    assert torch.equal(dk[skip:], wdk[skip:]) and torch.equal(dv[skip:], wdv[skip:])
    assert torch.equal(dq[rows][..., 1:], wdq[rows][..., 1:]) and bool(torch.isfinite(dq[rows]).all())
    # the others: some weighted mean of the rows of v
    assert bool(torch.isfinite(o).all()) and float(o.float().abs().max()) <= float(v.float().abs().max()) * (1 + 2 * R.h(dt))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_a_query_changes_no_bit_of_the_others(causal, D):
    """each row's maximum is followed by itself, not by its neighbours in a wave"""
    q, k, v, do, cu = attn_case([400], 2, 1, D, BF16)
    plan = ops.packed_plan(cu, 400)
    o, lse = ops.packed_attn_fwd(q, k, v, plan, causal)
    q2 = q.clone()
    q2[37] = q[37] * 64                                                    # its maximum moves at many tiles
    o2, lse2 = ops.packed_attn_fwd(q2, k, v, plan, causal)
    others = torch.arange(400, device=DEV) != 37
    assert torch.equal(o2[others], o[others]) and torch.equal(lse2[:, others], lse[:, others])
    assert not torch.equal(lse2[:, 37], lse[:, 37])


@pytest.mark.parametrize("causal", [True, False])
def test_a_list_that_is_none_shows_in_lse_beside_a_result_of_the_callers(causal):
    q, k, v, do, _ = attn_case([100], 2, 1, 32, F16)
    for cu in ([0, 60, 40, 100], [0, 101], [1, 100], [0, -1, 100]):
        plan = ops.packed_plan(torch.tensor(cu, dtype=torch.int32, device=DEV), 100)
        keep = torch.full_like(q, 3.0)
        o, lse = ops.packed_attn_fwd(q, k, v, plan, causal, out=keep)
        assert o is keep and bool((keep == 3).all()) and bool(torch.isnan(lse).all()), cu
    # rows behind the last sequence: the result's stay, lse's are zeros
    plan = ops.packed_plan(torch.tensor([0, 60], dtype=torch.int32, device=DEV), 100)
    _, lse = ops.packed_attn_fwd(q, k, v, plan, causal, out=keep)
    assert bool((keep[60:] == 3).all()) and not lse[:, 60:].any() and bool(torch.isfinite(lse).all()) and bool((lse[:, :60] != 0).any())


@pytest.mark.parametrize("lens,Hq,causal", [([1571], 3, False), ([2501], 1, True), ([1667], 1, True)])
def test_attention_cut_over_keys_with_odd_sizes(lens, Hq, causal):
    """sequences long enough to be cut into parts, an odd number of rows and heads: o, lse and gradients"""
    q, k, v, do, cu = attn_case(lens, Hq, 1, 64, BF16)
    plan = ops.packed_plan(cu, lens[0])
    o, lse = ops.packed_attn_fwd(q, k, v, plan, causal)
    dq, dk, dv = ops.packed_attn_bwd(q, k, v, o, lse, do, plan, causal)
    ref = R.attention(q, k, v, lens, causal, 0.125, do)
    worst = {n: R.off(t, ref[n], ref["tol"][n]) for n, t in dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv).items()}
    assert max(worst.values()) <= 1, worst


# ------------------------------------------------------------------------------------------------------------------ results' memory

def test_rotation_in_one_buffer():
    """q and k of a fused projection rotated where they are; results on anything else are refused"""
    T, H, D, sections = 57, 4, 64, (8, 24)
    qkv = randn(gen(4), T, 3 * H * D, dt=BF16)
    q, k, v = (t.view(T, H, D) for t in qkv.split(H * D, dim=1))
    pos = torch.arange(2 * T, device=DEV, dtype=torch.int32).view(T, 2)
    inv = 100.0 ** (-torch.arange(32, device=DEV, dtype=torch.float64) / 32)
    g = 1 + randn(gen(5), D, std=0.1)
    args = (pos, inv, sections, g, g)
    want, values = ops.qk_norm_rope_fwd(q, k, *args), v.clone()
    for bad in (dict(q_out=k), dict(k_out=q), dict(q_out=qkv[:, 8:8 + H * D].view(T, H, D)), dict(q_out=torch.empty_like(q), k_out=q[1:]),
                dict(q_out=v, k_out=v)):
        with pytest.raises((ValueError, _lib.SimvgHipError)):
            ops.qk_norm_rope_fwd(q, k, *args, **bad)
    for bad in (dict(dq_in=k), dict(dq_in=values), dict(dk_in=q), dict(dq_in=q, dk_in=q)):
        with pytest.raises((ValueError, _lib.SimvgHipError)):
            ops.qk_norm_rope_bwd(want[0], values, q, k, *args, **bad)
    ops.qk_norm_rope_fwd(q, k, *args, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(v, values)


def test_attention_and_its_gradients_in_one_buffer():
    """out beside q, k and v in one buffer, the gradients in another; results on an operand are refused"""
    lens, Hq, Hkv, D = [90, 41], 4, 2, 64
    q0, k0, v0, do, cu = attn_case(lens, Hq, Hkv, D, F16)
    T, cuts = sum(lens), [Hq * D, Hkv * D, Hkv * D, Hq * D]
    plan = ops.packed_plan(cu, T)
    want = ops.packed_attn_fwd(q0, k0, v0, plan)
    grads = ops.packed_attn_bwd(q0, k0, v0, *want, do, plan)
    room, rest = torch.zeros(T, sum(cuts), dtype=F16, device=DEV), torch.zeros(T, sum(cuts[:3]), dtype=F16, device=DEV)
    q, k, v, o = (t.view(T, -1, D) for t in room.split(cuts, dim=1))
    mine = [t.view(T, -1, D) for t in rest.split(cuts[:3], dim=1)]
    for a, b in ((q, q0), (k, k0), (v, v0)):
        a.copy_(b)
    for bad in (q, room[:, 8:8 + Hq * D].view(T, Hq, D), room[:, Hkv * D:(Hkv + Hq) * D].view(T, Hq, D)):
        with pytest.raises((ValueError, _lib.SimvgHipError)):
            ops.packed_attn_fwd(q, k, v, plan, out=bad)
    _, lse = ops.packed_attn_fwd(q, k, v, plan, out=o)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    for bad in (mine[:2] + [v], [q, *mine[1:]], [o, *mine[1:]], [mine[0], mine[1], mine[0][:, :Hkv]], [mine[0], mine[1], mine[0][:, 1:1 + Hkv]],
                [rest[:, 8:8 + Hq * D].view(T, Hq, D), *mine[1:]]):
        with pytest.raises((ValueError, _lib.SimvgHipError)):
            ops.packed_attn_bwd(q, k, v, o, lse, do, plan, dq=bad[0], dk=bad[1], dv=bad[2])
    ops.packed_attn_bwd(q, k, v, o, lse, do, plan, dq=mine[0], dk=mine[1], dv=mine[2])
    assert all(torch.equal(a, b) for a, b in zip(mine, grads))
    assert all(torch.equal(a, b) for a, b in ((q, q0), (k, k0), (v, v0), (o, want[0])))


# -------------------------------------------------------------------------------------------------------------------- captured graphs

def graph_nodes(graph):
    """the types of a captured graph's nodes (0 kernel, 1 copy, 2 memset ..), from the HIP library that torch has loaded"""
    path = next(ln.split()[-1] for ln in open("/proc/self/maps") if "libamdhip64" in ln)
    hip, raw, n = C.CDLL(path), C.c_void_p(graph.raw_cuda_graph()), C.c_size_t(0)
    assert hip.hipGraphGetNodes(raw, None, C.byref(n)) == 0
    nodes, kind = (C.c_void_p * n.value)(), C.c_int(-1)
    assert hip.hipGraphGetNodes(raw, nodes, C.byref(n)) == 0
    kinds = []
    for node in nodes:
        assert hip.hipGraphNodeGetType(C.c_void_p(node), C.byref(kind)) == 0
        kinds.append(kind.value)
    return kinds


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("M", [90, 1 << 20])
def test_reduced_loss_in_a_captured_graph(M, reduction):
    """the sum over many rows is a kernel of the library's: torch's own, from some hundred thousand rows on, clears its counters by a memset,
    which replays wrongly"""
    x, w, t, b, _ = ce_case(M, 60, 16, BF16, ignored=0.3)
    leaves = [z.clone().requires_grad_() for z in (x, w, b)]

    def step():
        loss = S.vocab_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction=reduction)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        out = step()
    kinds = graph_nodes(graph)
    assert kinds and set(kinds) == {0}, kinds
    graph.instantiate()
    for i in range(3):
        with torch.no_grad():
            leaves[0].mul_(0.75)
        graph.replay()
        torch.cuda.synchronize()
        assert bool(torch.isfinite(out[0])) and all(torch.equal(p, r) for p, r in zip(out, step())), i
        torch.cuda.synchronize()


@pytest.mark.parametrize("M", [0, 1, 333, 40000])
def test_reduced_loss_and_its_gradients(M):
    x, w, t, b, _ = ce_case(M, 300, 64, F16, ignored=0.3)
    if M == 1:
        t.fill_(7)
    rows = S.vocab_cross_entropy(x, w, t, b, reduction="none").detach().double()
    n = int((t != -100).sum())
    for reduction in ("sum", "mean"):
        leaves = [z.clone().requires_grad_() for z in (x, w, b)]
        loss = S.vocab_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction=reduction)
        assert loss.shape == () and loss.dtype == F32
        if n == 0 and reduction == "mean":
            assert bool(torch.isnan(loss))
            continue
        want = rows.sum() if reduction == "sum" else rows.sum() / n
        assert abs(float(loss.detach()) - float(want)) <= 4 * R.U * float(want)       # rounded once, and the quotient once more
        got = torch.autograd.grad(loss * 512, leaves)
        _, lse = ops.vocab_ce_fwd(x, w, t, b)
        each = torch.full((M,), 512.0 if reduction == "sum" else 512.0 / n, device=DEV)
        for a, c in zip(got, ops.vocab_ce_bwd(x, w, t, lse, each, b)):
            assert torch.equal(a, c)


@pytest.mark.parametrize("T,Hkv", [(1, 1), (1, 2), (70, 1)])
def test_strides_of_dimensions_of_one_mean_nothing(T, Hkv):
    """a token stride of a single token, a head stride of a single head: whatever they are, the same results"""
    Hq, D = 4 * Hkv, 64
    q, k, v, do, cu = (t if t.dim() == 1 else t.clone() for t in attn_case([T], Hq, Hkv, D, F16))

    def odd(t):
        ts, hs, _ = t.stride()
        room = torch.zeros(t.numel() + 64, dtype=t.dtype, device=DEV)
        room[:t.numel()] = t.flatten()
        return room.as_strided(t.shape, (ts if T > 1 else (1 << 24) + 3, hs if t.shape[1] > 1 else 1, 1))
    plan = ops.packed_plan(cu, T)
    want = ops.packed_attn_fwd(q, k, v, plan)
    want += ops.packed_attn_bwd(q, k, v, *want, do, plan)
    a, b, c, d = (odd(t) for t in (q, k, v, do))
    got = ops.packed_attn_fwd(a, b, c, plan, out=odd(torch.zeros_like(q)))
    got += ops.packed_attn_bwd(a, b, c, odd(got[0]), got[1], d, plan, dq=odd(torch.zeros_like(q)), dk=odd(torch.zeros_like(k)),
                               dv=odd(torch.zeros_like(v)))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


# ------------------------------------------------------------------------------------------------------------- few terms in a result

@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("lens,Hq,Hkv,D", [([2] * 154, 2, 2, 32), ([2] * 9, 1, 1, 128), ([1, 20, 5, 128, 127, 0, 65], 4, 2, 64), ([3, 7] * 11, 3, 1, 128),
                                           ([64] * 7, 6, 2, 80), ([33], 1, 1, 8)], ids=lambda x: "-".join(map(str, x[:3])) if isinstance(x, list) else str(x))
def test_short_sequences_are_as_exact_as_their_last_rounding(lens, Hq, Hkv, D, dt, causal):
    """P and dS, where few of them make a result, are not rounded to 16 bits: what is off is the result's own rounding and what 32 bits lose
    (at most n + 2 D + 64 steps of 2^-24 of the terms' magnitudes: a fourteenth of half a step of fp16 where all of them add up)"""
    q, k, v, do, cu = attn_case(lens, Hq, Hkv, D, dt)
    plan = ops.packed_plan(cu, sum(lens))
    o, lse = ops.packed_attn_fwd(q, k, v, plan, causal)
    dq, dk, dv = ops.packed_attn_bwd(q, k, v, o, lse, do, plan, causal)
    ref = R.attention(q, k, v, lens, causal, D ** -0.5, do)
    for name, got in dict(o=o, dq=dq, dk=dk, dv=dv).items():
        least = (ref[name].to(dt).double() - ref[name]).norm()
        assert float((got.double() - ref[name]).norm()) <= 1.1 * float(least) + 1e-6 * float(ref[name].norm()), name


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("lens,D", [([20, 0, 7, 1, 13], 64), ([65, 63, 129, 127, 1], 64), ([421, 401, 0, 413], 128), ([64, 128, 700], 40)],
                         ids=["few", "tiles", "long", "odd"])
def test_short_sequences_in_a_long_batch(lens, D, dt, causal):
    """many rows behind the last sequence: on average a batch of long ones, whose forward pass has no path of its own for short ones"""
    n, tail = sum(lens), 2100
    q, k, v, do, cu = attn_case(lens, 4, 2, D, dt, tail=tail)
    plan = ops.packed_plan(cu, n + tail)
    o, lse = ops.packed_attn_fwd(q, k, v, plan, causal)
    dq, dk, dv = ops.packed_attn_bwd(q, k, v, o, lse, do, plan, causal)
    ref = R.attention(q[:n], k[:n], v[:n], lens, causal, D ** -0.5, do[:n])
    got = dict(o=o[:n], lse=lse[:, :n], dq=dq[:n], dk=dk[:n], dv=dv[:n])
    worst = {name: R.off(t, ref[name], ref["tol"][name]) for name, t in got.items()}
    assert max(worst.values()) <= 1, worst
    assert not any(t[n:].any() for t in (o, dq, dk, dv)) and not lse[:, n:].any()


@pytest.mark.parametrize("tail", [0, 2100])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("lens,at", [([100], 60), ([70, 190], 160), ([128], 0)])
def test_later_rows_that_are_not_finite(lens, at, value, tail):
    """under `causal`, in the path for few tiles and in the other one, forward and backward"""
    q, k, v, do, cu = attn_case(lens, 4, 2, 64, BF16, tail=tail)
    n = sum(lens)
    plan = ops.packed_plan(cu, n + tail)

    def run(**x):
        a = dict(q=q, k=k, v=v, do=do) | x
        o, lse = ops.packed_attn_fwd(a["q"], a["k"], a["v"], plan)
        return (o, *ops.packed_attn_bwd(a["q"], a["k"], a["v"], o, lse, a["do"], plan))
    want = run()
    for name, t in dict(q=q, k=k, v=v, do=do).items():
        x = t.clone()
        x[at] = value
        got = run(**{name: x})
        if name in "kv":                                                   # earlier queries do not see the key
            assert torch.equal(got[0][:at], want[0][:at]) and torch.equal(got[1][:at], want[1][:at]), name
            if name == "v":
                assert not bool(torch.isfinite(got[0][at:n]).any())
                assert value != value or bool((got[0][at:n] == value).all())
        else:                                                              # later keys are not seen by the query
            assert torch.equal(got[2][at + 1:], want[2][at + 1:]) and torch.equal(got[3][at + 1:], want[3][at + 1:]), name
            assert not bool(torch.isfinite(got[2][at]).all()), name
            rows = torch.arange(n + tail, device=DEV) != at
            assert torch.equal(got[0][rows], want[0][rows]) and torch.equal(got[1][rows], want[1][rows]), name
