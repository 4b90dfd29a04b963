"""The sequence operators on the GPU against their definitions in 64 bits (tests/sequence_ref.py derives every bound)."""
import itertools

import pytest
import torch

import sequence_ref as R
from simvg_amd import _lib, hip_ops as ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dt=F32, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dt)


# ------------------------------------------------------------------------------------------------------------- norm + rotation

def rope_case(T, Hq, Hkv, D, sections, dt, seed=0, span=4096, layout="fused", pos_dt=torch.int32):
    g = gen(seed)
    if layout == "fused":                      # slices of a projection's rows
        qkv = randn(g, T, (Hq + 2 * Hkv) * D, dt=dt)
        q, k = qkv[:, :Hq * D].view(T, Hq, D), qkv[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
    elif layout == "heads":                    # heads outside
        q, k = randn(g, Hq, T, D, dt=dt).transpose(0, 1), randn(g, Hkv, T, D, dt=dt).transpose(0, 1)
    else:                                      # rows that start at odd places
        q, k = randn(g, T, Hq, D + 3, dt=dt)[..., 1:D + 1], randn(g, T, Hkv, D + 1, dt=dt)[..., 1:]
    pos = torch.randint(-span, span, (T, len(sections)), generator=g, device=DEV, dtype=pos_dt)
    P = sum(sections)
    inv = 10000.0 ** (-torch.arange(P, device=DEV, dtype=torch.float64) / P)
    return q, k, pos, inv, 1 + randn(g, D, std=0.2), 1 + randn(g, D, std=0.2), randn(g, T, Hq, D, dt=dt), randn(g, T, Hkv, D, dt=dt)


def check_rope(q, k, pos, inv, sections, gq, gk, dq, dk, interleaved, eps=1e-6):
    dt = q.dtype
    args = (q, k, pos, inv, sections, gq, gk, eps, interleaved)
    outs = ops.qk_norm_rope_fwd(*args)
    grads = ops.qk_norm_rope_bwd(dq, dk, *args)
    T, _, D = q.shape
    for x, g, dy, y, dx, dg in ((q, gq, dq, outs[0], grads[0], grads[2]), (k, gk, dk, outs[1], grads[1], grads[3])):
        X = x.double().requires_grad_()
        Gd = None if g is None else g.double().requires_grad_()
        ref, size = R.rope(X, Gd, pos, inv, sections, eps, interleaved)
        # norm (a sum of D squares, rsqrt, two products), the angle (half a step of half a turn, sincospi), two products and a sum
        assert R.off(y, ref.detach(), (24 + D / 8) * R.U * size.detach() + R.rounded(ref.detach(), dt)) <= 1
        leaves = [X] if Gd is None else [X, Gd]
        want = torch.autograd.grad(ref, leaves, dy.double())
        r = 1.0 if g is None else (x.double().square().mean(-1, keepdim=True) + eps).rsqrt()
        P2 = 2 * sum(sections)
        # |dz| <= |dy_a| + |dy_b| of the pair; dn = g dz; dx = r (dn - n mean(dn n))
        _, mag = R.rope(dy.double(), None, pos, inv, sections, eps, interleaved)
        dn = mag if g is None else mag * g.double().abs()
        n = (x.double() * r).abs()
        tol = dn if g is None else r * (dn + n * (dn * n).mean(-1, keepdim=True))
        assert R.off(dx, want[0], (48 + D / 4) * R.U * tol + R.rounded(want[0], dt)) <= 1
        if g is not None and T:
            # a wave's lanes add the rows of its tokens (at least 768 workgroups of 4 waves share them), then 6 halvings of a wave, 4 waves,
            # 1024 / 64 workgroups in each of 64 strands and 4 + 16 sums of those
            adds = (T / (4 * 768) + 1) * x.shape[1] + 6 + 4 + 16 + 4 + 16
            assert R.off(dg, want[1], (adds + 32 + D / 8) * R.U * (mag * n).sum((0, 1))) <= 1
        elif g is not None:
            assert not dg.any()
        assert P2 <= D


@pytest.mark.parametrize("dt", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv,D,sections", [
    (1, 32, 8, 128, (16, 24, 24)), (421, 12, 12, 64, (16, 16)), (1500, 7, 1, 80, (8, 12, 20)), (5, 3, 3, 256, (128,)),
    (130, 4, 2, 96, (0, 16, 8)), (33, 2, 1, 32, (4, 4, 4, 4)), (2, 1, 1, 2, (1,)), (19, 6, 2, 70, (5, 9))])
def test_rope_against_64_bits(T, Hq, Hkv, D, sections, interleaved, dt):
    q, k, pos, inv, gq, gk, dq, dk = rope_case(T, Hq, Hkv, D, sections, dt)
    check_rope(q, k, pos, inv, sections, gq, gk, dq, dk, interleaved)


@pytest.mark.parametrize("layout", ["heads", "odd"])
@pytest.mark.parametrize("dt", [F16, F32])
def test_rope_strides_and_alignment(layout, dt):
    q, k, pos, inv, gq, gk, dq, dk = rope_case(57, 4, 2, 64, (10, 22), dt, layout=layout, pos_dt=torch.int64)
    check_rope(q, k, pos, inv, (10, 22), gq, gk, dq.transpose(0, 1).contiguous().transpose(0, 1), dk, False)


def test_rope_far_positions_keep_their_angle():
    # positions of 2^30: an angle formed in 32 bits would be off by many turns
    sections = (32,)
    q, k, pos, inv, gq, gk, dq, dk = rope_case(64, 2, 2, 64, sections, F32, span=1 << 30)
    check_rope(q, k, pos, inv, sections, gq, gk, dq, dk, False)
    q, k, pos, inv, gq, gk, dq, dk = rope_case(64, 2, 2, 64, sections, F32, span=1 << 40, pos_dt=torch.int64)
    # the reference's own product is off by half a step of 2^40 turns: 2^-13 of a turn
    y, _ = ops.qk_norm_rope_fwd(q, k, pos, inv, sections, gq, gk)
    ref, size = R.rope(q.double(), gq, pos, inv, sections, 1e-6, False)
    assert R.off(y, ref, 2.0 ** -9 * size) <= 1


@pytest.mark.parametrize("dt", [BF16, F32])
def test_rope_without_norm_and_in_place(dt):
    sections = (8, 24)
    q, k, pos, inv, _, _, dq, dk = rope_case(300, 4, 2, 64, sections, dt)
    check_rope(q, k, pos, inv, sections, None, None, dq, dk, False)
    want = ops.qk_norm_rope_fwd(q, k, pos, inv, sections)
    q2, k2 = q.clone(), k.clone()
    ops.qk_norm_rope_fwd(q2, k2, pos, inv, sections, q_out=q2, k_out=k2)
    assert torch.equal(q2, want[0]) and torch.equal(k2, want[1])


def test_rope_no_tokens_and_many_tokens():
    sections = (16, 16)
    q, k, pos, inv, gq, gk, dq, dk = rope_case(0, 2, 2, 64, sections, F16)
    check_rope(q, k, pos, inv, sections, gq, gk, dq, dk, False)
    q, k, pos, inv, gq, gk, dq, dk = rope_case(9001, 3, 1, 64, sections, BF16)     # several rounds of the backward's workgroups
    check_rope(q, k, pos, inv, sections, gq, gk, dq, dk, False)
    a = ops.qk_norm_rope_bwd(dq, dk, q, k, pos, inv, sections, gq, gk)
    b = ops.qk_norm_rope_bwd(dq, dk, q, k, pos, inv, sections, gq, gk)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_rope_rows_far_apart():
    # token stride 2^21: row offsets pass 2^31 elements
    T, Hq, Hkv, D, sections = 1100, 2, 1, 64, (32,)
    big = torch.zeros(T * (1 << 21), device=DEV, dtype=F16)
    g = gen(3)
    q = big.as_strided((T, Hq, D), (1 << 21, D, 1))
    k = big.as_strided((T, Hkv, D), (1 << 21, D, 1), Hq * D)
    q.copy_(randn(g, T, Hq, D, dt=F16))
    k.copy_(randn(g, T, Hkv, D, dt=F16))
    _, _, pos, inv, gq, gk, dq, dk = rope_case(T, Hq, Hkv, D, sections, F16)
    check_rope(q, k, pos, inv, sections, gq, gk, dq, dk, False)


# -------------------------------------------------------------------------------------------------------------------- attention

def attn_case(lens, Hq, Hkv, D, dt, seed=0, tail=0, std=1.0, gstd=1.0):
    g = gen(seed)
    T = sum(lens) + tail
    qkv = randn(g, T, (Hq + 2 * Hkv) * D, dt=dt, std=std)
    q, k, v = (t.view(T, -1, D) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1))
    cu = torch.tensor(list(itertools.accumulate([0] + list(lens))), dtype=torch.int32, device=DEV)
    return q, k, v, randn(g, T, Hq, D, dt=dt, std=gstd), cu


def check_attn(q, k, v, do, cu, lens, causal, scale=None):
    T, Hq, D = q.shape
    plan = ops.packed_plan(cu, T)
    o, lse = ops.packed_attn_fwd(q, k, v, plan, causal, scale)
    dq, dk, dv = ops.packed_attn_bwd(q, k, v, o, lse, do, plan, causal, scale)
    ref = R.attention(q, k, v, lens, causal, D ** -0.5 if scale is None else scale, do)
    got = dict(o=o, lse=lse, dq=dq, dk=dk, dv=dv)
    worst = {n: R.off(t, ref[n], ref["tol"][n]) for n, t in got.items()}
    assert max(worst.values()) <= 1, worst
    return got


LENS = [[1], [20, 0, 7, 1, 13], [64], [65, 63], [128], [129, 127, 1], [421, 401, 0, 413], [700], [33] * 40, [0, 0, 5, 0]]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("lens", LENS, ids=lambda x: "-".join(map(str, x[:5])))
def test_attention_lengths(lens, dt, causal):
    q, k, v, do, cu = attn_case(lens, 4, 2, 64, dt)
    check_attn(q, k, v, do, cu, lens, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 12, 64), (8, 1, 128), (7, 1, 80), (6, 2, 96), (2, 2, 8), (3, 3, 40), (4, 4, 32), (14, 2, 120)])
def test_attention_heads(Hq, Hkv, D, dt, causal):
    lens = [150, 3, 260, 64]
    q, k, v, do, cu = attn_case(lens, Hq, Hkv, D, dt)
    check_attn(q, k, v, do, cu, lens, causal)


@pytest.mark.parametrize("dt", [F16, BF16])
def test_attention_long_and_large_scores(dt):
    lens = [2500]
    q, k, v, do, cu = attn_case(lens, 2, 1, 128, dt)
    check_attn(q, k, v, do, cu, lens, True)
    q, k, v, do, cu = attn_case([300], 2, 1, 64, dt, std=6.0)            # scores of hundreds: the maximum moves
    check_attn(q, k, v, do, cu, [300], True)
    check_attn(q, k, v, do, cu, [300], False, scale=0.01)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_attention_few_key_heads(dt, causal):
    # one key head, long sequences: the queries of a workgroup's keys are cut into parts, over tiles and heads
    for lens, Hq, D in (([2100], 3, 64), ([3000], 1, 128), ([1500, 2, 1400], 5, 40)):
        q, k, v, do, cu = attn_case(lens, Hq, 1, D, dt, tail=70)
        n = sum(lens)
        plan = ops.packed_plan(cu, n + 70)
        o, lse = ops.packed_attn_fwd(q, k, v, plan, causal)
        dq, dk, dv = ops.packed_attn_bwd(q, k, v, o, lse, do, plan, causal)
        ref = R.attention(q[:n], k[:n], v[:n], lens, causal, D ** -0.5, do[:n])
        worst = {name: R.off(t[:n], ref[name], ref["tol"][name]) for name, t in dict(o=o, dq=dq, dk=dk, dv=dv).items()}
        assert max(worst.values()) <= 1, worst
        assert not any(t[n:].any() for t in (o, dq, dk, dv))


@pytest.mark.parametrize("gstd", [1e-4, 300.0])
def test_attention_small_and_large_gradients_in_fp16(gstd):
    # dS of a long row is far below fp16's normal range unless it is brought up
    lens = [1500, 40]
    q, k, v, do, cu = attn_case(lens, 2, 1, 64, F16, gstd=gstd)
    check_attn(q, k, v, do, cu, lens, True)
    check_attn(q, k, (v.float() * 40).half(), do, cu, lens, False)


def test_attention_layouts():
    lens, dt = [90, 200], F16
    T, D = 290, 64
    g = gen(5)
    q = randn(g, 6, T, D, dt=dt).transpose(0, 1)                            # heads outside
    kv = randn(g, T, 2, 3, D, dt=dt)                                        # k and v interleaved
    do = randn(g, T, 6, 2 * D, dt=dt)[..., D:]
    cu = torch.tensor([0, 90, 290], dtype=torch.int32, device=DEV)
    check_attn(q, kv[:, 0], kv[:, 1], do, cu, lens, True)


def test_attention_rows_far_apart():
    lens, Hq, Hkv, D = [1030, 70], 2, 1, 64
    T = sum(lens)
    big = torch.zeros(T * (1 << 21), device=DEV, dtype=BF16)
    q0, k0, v0, do, cu = attn_case(lens, Hq, Hkv, D, BF16)
    q = big.as_strided((T, Hq, D), (1 << 21, D, 1))
    k = big.as_strided((T, Hkv, D), (1 << 21, D, 1), Hq * D)
    v = big.as_strided((T, Hkv, D), (1 << 21, D, 1), (Hq + Hkv) * D)
    for a, b in ((q, q0), (k, k0), (v, v0)):
        a.copy_(b)
    check_attn(q, k, v, do, cu, lens, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt", [F16, BF16])
def test_attention_rows_behind_the_last_sequence(dt, causal):
    lens, tail = [100, 61, 200], 300
    q, k, v, do, cu = attn_case(lens, 4, 2, 64, dt, tail=tail)
    n = sum(lens)
    clean = check_attn(q[:n], k[:n], v[:n], do[:n], cu, lens, causal)
    for t in (q, k, v, do):
        t[n:] = float("nan")
    plan = ops.packed_plan(cu, n + tail)
    o, lse = ops.packed_attn_fwd(q, k, v, plan, causal)
    grads = ops.packed_attn_bwd(q, k, v, o, lse, do, plan, causal)
    for got, want in zip((o, *grads), (clean["o"], clean["dq"], clean["dk"], clean["dv"])):
        assert torch.equal(got[:n], want) and not got[n:].any()
    assert torch.equal(lse[:, :n], clean["lse"]) and not lse[:, n:].any()
    mine = [torch.full_like(t, 7.0) for t in (o, *grads)]                  # the caller's own: left as they were
    ops.packed_attn_fwd(q, k, v, plan, causal, out=mine[0])
    ops.packed_attn_bwd(q, k, v, o, lse, do, plan, causal, dq=mine[1], dk=mine[2], dv=mine[3])
    for got, want in zip(mine, (o, *grads)):
        assert torch.equal(got[:n], want[:n]) and bool((got[n:] == 7).all())


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_does_not_see_what_is_masked(causal, dt, value):
    """values that are not finite in other sequences, and under `causal` in later rows, change nothing; rows that see them do"""
    lens = [70, 150, 40]
    q, k, v, do, cu = attn_case(lens, 4, 2, 64, dt)
    plan = ops.packed_plan(cu, 260)
    o, lse = ops.packed_attn_fwd(q, k, v, plan, causal)
    grads = ops.packed_attn_bwd(q, k, v, o, lse, do, plan, causal)
    at = 70 + 90                                                            # row 90 of the second sequence
    for which in ("q", "k", "v", "do"):
        x = dict(q=q.clone(), k=k.clone(), v=v.clone(), do=do.clone())
        x[which][at] = value
        o2, lse2 = ops.packed_attn_fwd(x["q"], x["k"], x["v"], plan, causal)
        g2 = ops.packed_attn_bwd(x["q"], x["k"], x["v"], o2, lse2, x["do"], plan, causal)
        others = torch.ones(260, dtype=torch.bool, device=DEV)
        others[70:220] = False
        for a, b in zip((o2, *g2), (o, *grads)):
            assert torch.equal(a[others], b[others]), which
        before = slice(70, at) if causal else slice(0, 0)
        if which in ("k", "v"):                                            # earlier queries do not see the key
            assert torch.equal(o2[before], o[before]) and torch.equal(g2[0][before], grads[0][before]), which
            if which == "v":
                seen = o2[at:220] if causal else o2[70:220]
                assert not bool(torch.isfinite(seen).any())
                if value == value:
                    assert bool((seen == value).all())
            else:
                assert not bool(torch.isfinite(g2[0][at]).any())
        else:                                                              # later keys are not seen by the query
            after = slice(at + 1, 220) if causal else slice(0, 0)
            assert torch.equal(g2[1][after], grads[1][after]) and torch.equal(g2[2][after], grads[2][after]), which
            assert not bool(torch.isfinite(g2[1][at]).all()), which
        if which == "q":
            assert bool(torch.isnan(o2[at]).all()) and torch.equal(o2[at + 1:], o[at + 1:]) and torch.equal(o2[:at], o[:at])


def test_attention_scores_of_minus_infinity():
    # every visible score of a row is -inf: no distribution, NaN, and only there
    lens = [40]
    q, k, v, do, cu = attn_case(lens, 1, 1, 32, BF16)
    q, k = q.abs(), k.abs()
    k[0] = float("-inf")
    plan = ops.packed_plan(cu, 40)
    o, _ = ops.packed_attn_fwd(q, k, v, plan, True)
    assert bool(torch.isnan(o[0]).all()) and bool(torch.isfinite(o[1:]).all())
    o2, _ = ops.packed_attn_fwd(q[1:], k[1:], v[1:], ops.packed_plan(torch.tensor([0, 39], dtype=torch.int32, device=DEV), 39), True)
    assert float((o[1:].float() - o2.float()).abs().max()) <= 4 * R.h(BF16) * float(v.float().abs().max())   # one probability each way


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("lens,Hq,Hkv,D", [([1, 20, 5, 128, 127], 4, 2, 64), ([2300], 2, 1, 128), ([64] * 7, 3, 3, 40)], ids=["short", "parts", "tiles"])
def test_attention_rows_with_one_key_have_no_gradient(lens, Hq, Hkv, D, dt):
    """P is 1 and dP is delta: dQ is nothing but what fp32 leaves of their difference, not the output's rounding to 16 bits"""
    q, k, v, do, cu = attn_case(lens, Hq, Hkv, D, dt)
    plan = ops.packed_plan(cu, sum(lens))
    o, lse = ops.packed_attn_fwd(q, k, v, plan, True)
    dq, _, _ = ops.packed_attn_bwd(q, k, v, o, lse, do, plan, True)
    scale, first = D ** -0.5, 0
    for n in lens:
        for h in range(Hq):
            Q, K, V, dO = (t[first:first + n].double() for t in (q[:, h], k[:, h // (Hq // Hkv)], v[:, h // (Hq // Hkv)], do[:, h]))
            # the score: as in sequence_ref.attention; P is off by its error, dP and delta (a sum of it alone) by D products and sums each
            ds = scale * (Q[0].abs() * K[0].abs()).sum() * (D + 8) * R.U + 8 * R.U * (1 + lse[h, first].double().abs())
            at = (dO[0].abs() * V[0].abs()).sum() * (2 * (D + 8) * R.U + 2 * ds)
            if dt == F16:                                                  # the least that dS is rounded to
                at = at + 4 * 2.0 ** -39 * dO.norm(dim=-1).max() * V.norm(dim=-1).max()
            assert bool((dq[first, h].double().abs() <= scale * at * K[0].abs() * (1 + 2 * R.h(dt)) + R.tiny(dt)).all()), (n, h)
        first += n


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("lens,Hq,Hkv", [([300], 2, 1), ([2500], 2, 1), ([70, 200, 65], 12, 4)], ids=["tiles", "parts", "batch"])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_tiles_of_minus_infinity(causal, lens, Hq, Hkv, dt):
    """the first keys of a sequence, whole tiles of them, have scores of -inf: what comes behind them is not lost"""
    q, k, v, do, cu = attn_case(lens, Hq, Hkv, 64, dt)
    q, k = q.clone(), k.clone()
    q[..., 0] = 1
    skip = 130 if lens[0] > 130 else 64
    k[:skip, :, 0] = float("-inf")
    T = sum(lens)
    plan = ops.packed_plan(cu, T)
    o, lse = ops.packed_attn_fwd(q, k, v, plan, causal)
    dq, dk, dv = ops.packed_attn_bwd(q, k, v, o, lse, do, plan, causal)
    alone = slice(0, skip if causal else 0)                                # rows that see nothing else
    assert bool(torch.isnan(o[alone]).all()) and bool((lse[:, alone] == float("-inf")).all())
    # the same rows without those keys, from the definition: a sequence of the rest (causal: from the first that sees it), whose other
    # rows are those of a sequence that is cut after `skip`
    cut = [skip, lens[0] - skip, *lens[1:]] if causal else lens
    kk, vv = k.clone(), v.clone()
    if causal:
        kk[:skip, :, 0] = 0
        ref = R.attention(q, kk, vv, cut, True, 0.125, do)
        for name, t in dict(o=o, dq=dq, dk=dk, dv=dv).items():
            rows = slice(skip, T)
            if name == "dq":                                               # dS 0 times a key of -inf: NaN in that column, by the formula
                assert R.off(t[rows][..., 1:], ref[name][rows][..., 1:], ref["tol"][name][rows][..., 1:]) <= 1
            else:
                assert R.off(t[rows], ref[name][rows], ref["tol"][name][rows]) <= 1, name
        assert R.off(lse[:, skip:], ref["lse"][:, skip:], ref["tol"]["lse"][:, skip:]) <= 1
    else:
        x = q.double(), k.double(), v.double()
        rows = slice(0, lens[0])
        for h in range(Hq):
            Q, K, V = x[0][rows, h], x[1][rows, h // (Hq // Hkv)], x[2][rows, h // (Hq // Hkv)]
            S = 0.125 * Q @ torch.where(torch.isinf(K), 0.0, K).t()
            S[:, :skip] = float("-inf")
            P = S.softmax(-1)
            # the bound of sequence_ref.attention for o, over the keys that are left
            size = (0.125 * Q.abs() @ K[skip:].abs().t()).amax(-1) * 72 * R.U + 8 * R.U * (1 + S.logsumexp(-1).abs())
            tol = (P @ V.abs()) * (R.h(dt) + 2 * size[:, None] + (lens[0] + 64) * R.U) + R.tiny(dt) * V.abs().sum(0) + R.rounded(P @ V, dt)
            assert R.off(o[rows, h], P @ V, tol) <= 1
        assert not dv[:skip].any() and not dk[:skip].any()                 # probabilities of 0
    assert bool(torch.isfinite(dv[skip:]).all()) and bool(torch.isfinite(dk[skip:]).all())


@pytest.mark.parametrize("causal", [True, False])
def test_attention_a_list_that_is_none_is_loud(causal):
    q, k, v, do, _ = attn_case([100], 2, 1, 32, F16)
    for cu in ([0, 60, 40, 100], [0, 101], [1, 100], [0, -1, 100], [0, 2 ** 31 - 1]):
        plan = ops.packed_plan(torch.tensor(cu, dtype=torch.int32, device=DEV), 100)
        o, lse = ops.packed_attn_fwd(q, k, v, plan, causal)
        assert bool(torch.isnan(o).all()) and bool(torch.isnan(lse).all()), cu
        grads = ops.packed_attn_bwd(q, k, v, o, lse, do, plan, causal)
        assert all(bool(torch.isnan(t).all()) for t in grads), cu
        keep = torch.full_like(q, 3.0)
        ops.packed_attn_fwd(q, k, v, plan, causal, out=keep)
        assert bool((keep == 3).all())


def test_attention_many_sequences_and_none():
    lens = [i % 5 for i in range(3000)]                                    # more sequences than the plan's workgroup has threads
    q, k, v, do, cu = attn_case(lens, 2, 1, 32, F16)
    T = sum(lens)
    plan = ops.packed_plan(cu, T)
    o, lse = ops.packed_attn_fwd(q, k, v, plan)
    dq, dk, dv = ops.packed_attn_bwd(q, k, v, o, lse, do, plan)
    sel = slice(sum(lens[:1000]), sum(lens[:1030]))                         # a window of whole sequences
    ref = R.attention(q[sel], k[sel], v[sel], lens[1000:1030], True, 32 ** -0.5, do[sel])
    for n, t in dict(o=o, dq=dq, dk=dk, dv=dv).items():
        assert R.off(t[sel], ref[n], ref["tol"][n]) <= 1, n
    empty = ops.packed_plan(torch.zeros(1, dtype=torch.int32, device=DEV), 50)
    o, lse = ops.packed_attn_fwd(q[:50], k[:50], v[:50], empty)
    assert not o.any() and not lse.any()
    assert not any(t.any() for t in ops.packed_attn_bwd(q[:50], k[:50], v[:50], o, lse, do[:50], empty))
    none = ops.packed_plan(torch.zeros(3, dtype=torch.int32, device=DEV), 0)
    o, lse = ops.packed_attn_fwd(q[:0], k[:0], v[:0], none)
    assert o.shape == (0, 2, 32) and [t.shape[0] for t in ops.packed_attn_bwd(q[:0], k[:0], v[:0], o, lse, do[:0], none)] == [0, 0, 0]


def test_attention_same_bits_at_every_run():
    lens = [300, 7, 900]
    q, k, v, do, cu = attn_case(lens, 8, 2, 128, BF16)
    runs = []
    for _ in range(3):
        plan = ops.packed_plan(cu, sum(lens))
        o, lse = ops.packed_attn_fwd(q, k, v, plan)
        runs.append([o, lse, *ops.packed_attn_bwd(q, k, v, o, lse, do, plan)])
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


# -------------------------------------------------------------------------------------------------------------------- vocabulary

def ce_case(M, V, K, dt, seed=0, bias=True, ignored=0.2, uniform=True, gscale=1024.0):
    g = gen(seed)
    x, w = randn(g, M, K, dt=dt), randn(g, V, K, dt=dt, std=1.5 * K ** -0.5)
    b = randn(g, V, std=0.5) if bias else None
    t = torch.randint(0, V, (M,), generator=g, device=DEV)
    skip = torch.rand(M, generator=g, device=DEV) < ignored
    t = torch.where(skip, -100, t)
    gl = torch.full((M,), gscale / max(1, M), device=DEV) if uniform else randn(g, M, std=gscale / max(1, M))
    return x, w, t, b, gl


def check_ce(x, w, t, b, gl):
    loss, lse = ops.vocab_ce_fwd(x, w, t, b)
    dx, dw, db = ops.vocab_ce_bwd(x, w, t, lse, gl, b)
    ref = R.vocab_ce(x, w, t, b, gl)
    got = dict(loss=loss, lse=lse, dx=dx, dw=dw)
    if b is not None:
        got["dbias"] = db
    worst = {n: R.off(v, ref[n], ref["tol"][n]) for n, v in got.items()}
    assert max(worst.values()) <= 1, worst
    return got


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M,V,K,bias", [
    (1, 1000, 64, True), (20, 6401, 768, True), (64, 257, 8, False), (65, 256, 72, True), (333, 3203, 520, False), (1, 1, 8, True),
    (130, 5000, 264, True), (700, 2049, 128, True), (3, 40000, 16, False), (257, 255, 1032, True)])
def test_vocab_ce_against_64_bits(M, V, K, bias, dt):
    check_ce(*ce_case(M, V, K, dt, bias=bias))


@pytest.mark.parametrize("dt", [F16, BF16])
def test_vocab_ce_rows_of_unequal_weight(dt):
    check_ce(*ce_case(300, 1500, 256, dt, uniform=False))
    check_ce(*ce_case(40, 1500, 256, dt, uniform=False))


@pytest.mark.parametrize("M", [1023, 1025, 4096, 4097])               # rows to a thread of the list's workgroup; a list in one launch or two
def test_vocab_ce_lists_of_rows(M):
    check_ce(*ce_case(M, 270, 72, F16, ignored=0.5, uniform=False))


@pytest.mark.parametrize("dt", [F16, BF16])
def test_vocab_ce_in_several_pieces(dt):
    # 2^27 / 40000 words to a piece: eight pieces, the last one partly empty
    x, w, t, b, gl = ce_case(40000, 25001, 64, dt, ignored=0.5)
    loss, lse = ops.vocab_ce_fwd(x, w, t, b)
    dx, dw, db = ops.vocab_ce_bwd(x, w, t, lse, gl, b)
    sel = slice(31000, 31200)
    ref = R.vocab_ce(x[sel], w, t[sel], b, gl[sel])
    assert all(R.off(v[sel], ref[n], ref["tol"][n]) <= 1 for n, v in dict(loss=loss, lse=lse, dx=dx).items())
    # dw and db: the sums over all rows, in blocks of rows
    want, tol = {}, {}
    for i in range(0, 40000, 4000):
        r = R.vocab_ce(x[i:i + 4000], w, t[i:i + 4000], b, gl[i:i + 4000])
        for n in ("dw", "dbias"):
            want[n] = want.get(n, 0) + r[n]
            tol[n] = tol.get(n, 0) + r["tol"][n] + 4500 * R.U * r[n].abs()
    assert R.off(dw, want["dw"], tol["dw"] + R.rounded(want["dw"], dt)) <= 1
    assert R.off(db, want["dbias"], tol["dbias"]) <= 1


def test_vocab_ce_strides():
    x, w, t, b, gl = ce_case(90, 700, 128, BF16)
    wide = torch.full((90, 200), float("nan"), device=DEV, dtype=BF16)
    wide[:, 8:136] = x
    words = torch.full((700, 136), float("nan"), device=DEV, dtype=BF16)
    words[:, :128] = w
    a, c = check_ce(x, w, t, b, gl), check_ce(wide[:, 8:136], words[:, :128], t, b, gl)
    assert all(torch.equal(a[n], c[n]) for n in a)


def test_vocab_ce_large_logits_and_confident_rows():
    x, w, t, b, gl = ce_case(64, 900, 64, BF16, ignored=0.0)
    check_ce((x.float() * 40).bfloat16(), w, t, b, gl)
    x, w, t, b, gl = ce_case(100, 900, 64, F16, ignored=0.0)
    t = (x.float() @ w.float().t() * 30 + b).argmax(1)
    check_ce((x.float() * 30).half(), w, t, b, gl)


@pytest.mark.parametrize("dt", [F16, BF16])
@pytest.mark.parametrize("M", [50, 200])
def test_vocab_ce_ignored_rows_have_no_part(M, dt):
    x, w, t, b, gl = ce_case(M, 3000, 96, dt, ignored=0.0)
    keep = torch.arange(M, device=DEV) % 3 != 0
    t = torch.where(keep, t, -100)
    want = check_ce(x, w, t, b, gl)
    x2, gl2 = x.clone(), gl.clone()
    x2[~keep] = float("nan")
    gl2[~keep] = float("inf")
    loss, lse = ops.vocab_ce_fwd(x2, w, t, b)
    dx, dw, db = ops.vocab_ce_bwd(x2, w, t, lse, gl2, b)
    assert torch.equal(loss, want["loss"]) and torch.equal(dw, want["dw"]) and torch.equal(dx, want["dx"]) and torch.equal(db, want["dbias"])
    assert not loss[~keep].any() and not dx[~keep].any()
    t3 = torch.where(keep, t, torch.tensor([3000, -1, 1 << 40], device=DEV)[torch.arange(M, device=DEV) % 3])   # no words: loud
    loss, lse = ops.vocab_ce_fwd(x, w, t3, b)
    dx, dw, db = ops.vocab_ce_bwd(x, w, t3, lse, gl, b)
    assert bool(torch.isnan(loss[~keep]).all()) and torch.equal(loss[keep], want["loss"][keep])
    assert torch.equal(dw, want["dw"]) and torch.equal(dx, want["dx"])
    none = torch.full_like(t, -100)
    loss, lse = ops.vocab_ce_fwd(x, w, none, b)
    assert not loss.any() and not any(v.any() for v in ops.vocab_ce_bwd(x, w, none, lse, gl, b))


def test_vocab_ce_ignore_index_may_be_a_word_and_zero_rows():
    x, w, t, b, gl = ce_case(70, 500, 64, F16, ignored=0.0)
    t[::2] = 3
    loss, lse = ops.vocab_ce_fwd(x, w, t, b, ignore_index=3)
    ref = R.vocab_ce(x, w, t, b, gl, ignore_index=3)
    assert R.off(loss, ref["loss"], ref["tol"]["loss"]) <= 1
    dx, dw, db = ops.vocab_ce_bwd(x, w, t, lse, gl, b, ignore_index=3)
    assert R.off(dw, ref["dw"], ref["tol"]["dw"]) <= 1 and R.off(dx, ref["dx"], ref["tol"]["dx"]) <= 1
    loss, lse = ops.vocab_ce_fwd(x[:0], w, t[:0], b)
    dx, dw, db = ops.vocab_ce_bwd(x[:0], w, t[:0], lse, gl[:0], b)
    assert loss.shape == (0,) and dx.shape == (0, 64) and not dw.any() and not db.any()


def test_vocab_ce_same_bits_at_every_run():
    x, w, t, b, gl = ce_case(600, 9000, 256, BF16, uniform=False)
    runs = []
    for _ in range(3):
        loss, lse = ops.vocab_ce_fwd(x, w, t, b)
        runs.append([loss, lse, *ops.vocab_ce_bwd(x, w, t, lse, gl, b)])
    assert all(torch.equal(p, r) for run in runs[1:] for p, r in zip(runs[0], run))


# ------------------------------------------------------------------------------------------------------- streams, graphs, refusals

def all_operators(seed):
    q, k, pos, inv, gq, gk, dq, dk = rope_case(200, 4, 2, 64, (8, 24), F16, seed=seed)
    qa, ka, va, do, cu = attn_case([120, 0, 80], 4, 2, 64, F16, seed=seed)
    x, w, t, b, gl = ce_case(96, 1100, 64, F16, seed=seed)

    def call():
        y = ops.qk_norm_rope_fwd(q, k, pos, inv, (8, 24), gq, gk)
        z = ops.qk_norm_rope_bwd(dq, dk, q, k, pos, inv, (8, 24), gq, gk)
        plan = ops.packed_plan(cu, 200)
        o, lse = ops.packed_attn_fwd(qa, ka, va, plan)
        g = ops.packed_attn_bwd(qa, ka, va, o, lse, do, plan)
        loss, ls = ops.vocab_ce_fwd(x, w, t, b)
        e = ops.vocab_ce_bwd(x, w, t, ls, gl, b)
        return [*y, *z, o, lse, *g, loss, ls, *e]
    return call, [q, k, dq, dk, qa, ka, va, do, x, w, gl]


def test_operators_on_another_stream():
    call, _ = all_operators(1)
    want = call()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = call()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_operators_in_two_captured_graphs():
    calls = [all_operators(s) for s in (1, 2)]
    graphs, outs = [], []
    for call, _ in calls:
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    for round_ in range(3):
        for _, inputs in calls:
            for t in inputs:
                t.mul_(0.5 + round_ % 2)                                   # 0.5, 1.5, 0.5
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (call, _), out in zip(calls, outs):
            assert all(torch.equal(a, b) for a, b in zip(out, call())), round_
        torch.cuda.synchronize()


def test_refusals():
    q, k, pos, inv, gq, gk, dq, dk = rope_case(10, 4, 2, 64, (8, 24), F16)
    E = (ValueError, TypeError, _lib.SimvgHipError)
    for bad in (dict(q=q.float()), dict(k=k[:9]), dict(pos=pos.float()), dict(pos=pos[:, :1]), dict(inv=inv.float()), dict(inv=inv[:-1]),
                dict(sections=(8,)), dict(sections=(40, 24)), dict(sections=()), dict(gq=None), dict(gq=gq.half()), dict(q=q.cpu()),
                dict(q=q[..., ::2]), dict(sections=(-8, 40))):
        a = dict(q=q, k=k, pos=pos, inv=inv, sections=(8, 24), gq=gq, gk=gk) | bad
        with pytest.raises(E):
            ops.qk_norm_rope_fwd(a["q"], a["k"], a["pos"], a["inv"], a["sections"], a["gq"], a["gk"])
    with pytest.raises(E):
        ops.qk_norm_rope_fwd(q, k, pos, inv, (8, 24), q_out=q[:1].expand(10, 4, 64))
    q, k, v, do, cu = attn_case([10], 4, 2, 64, F16)
    plan = ops.packed_plan(cu, 10)
    for bad in (dict(q=q.float()), dict(k=k.bfloat16()), dict(v=v[:9]), dict(k=k[:, :1]), dict(plan=ops.packed_plan(cu, 11)),
                dict(q=q[:, :3]), dict(q=q.cpu()), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(q=q[..., :60], k=k[..., :60], v=v[..., :60]), dict(q=q[..., 1:41], k=k[..., 1:41], v=v[..., 1:41])):
        a = dict(q=q, k=k, v=v, plan=plan, scale=None) | bad
        with pytest.raises(E):
            ops.packed_attn_fwd(a["q"], a["k"], a["v"], a["plan"], True, a["scale"])
    big = torch.zeros(10, 2, 136, device=DEV, dtype=F16)
    with pytest.raises(E):
        ops.packed_attn_fwd(big, big, big, plan)
    o, lse = ops.packed_attn_fwd(q, k, v, plan)
    for bad in (dict(lse=lse.t()), dict(do=do.float()), dict(dq=torch.empty_like(q))):
        a = dict(lse=lse, do=do, dq=None) | bad
        with pytest.raises(E):
            ops.packed_attn_bwd(q, k, v, o, a["lse"], a["do"], plan, dq=a["dq"])
    for bad in (dict(out=k), dict(out=v)):                                 # results in the operands' memory, and in each other's
        with pytest.raises(E):
            ops.packed_attn_fwd(q[:, :2], k, v, plan, out=bad["out"])
    mine = [torch.empty_like(t) for t in (q, k, v)]
    for a, b, c in ((q, mine[1], mine[2]), (do, mine[1], mine[2]), (o, mine[1], mine[2]), (mine[0], k, mine[2]), (mine[0], mine[1], mine[1])):
        with pytest.raises(E):
            ops.packed_attn_bwd(q, k, v, o, lse, do, plan, dq=a, dk=b, dv=c)
    with pytest.raises(E):
        ops.packed_plan(cu.long(), 10)
    with pytest.raises(E):
        ops.packed_plan(cu[:0], 10)
    x, w, t, b, gl = ce_case(10, 50, 64, F16)
    for bad in (dict(x=x.float()), dict(w=w.bfloat16()), dict(x=x[:, :60], w=w[:, :60]), dict(t=t.int()), dict(t=t[:9]), dict(b=b.half()),
                dict(x=x.cpu()), dict(w=w[:, :56]), dict(x=x[:, 1:57], w=w[:, :56])):
        a = dict(x=x, w=w, t=t, b=b) | bad
        with pytest.raises(E):
            ops.vocab_ce_fwd(a["x"], a["w"], a["t"], a["b"])
    loss, lse = ops.vocab_ce_fwd(x, w, t, b)
    with pytest.raises(E):
        ops.vocab_ce_bwd(x, w, t, lse, gl.half(), b)
