"""CPU: what the sequence operators' C entries answer, or refuse, before anything is launched."""
import ctypes as C
import itertools
import random

import pytest
import torch

from simvg_amd import _lib


def refused(fn, args, words):
    """refused with these words.  (Addresses here are numbers: what is not refused ends at the launch, there is no device)"""
    rc = fn(C.byref(args), None)
    return rc < 0 and words in _lib.load().simvg_last_error().decode()


@pytest.mark.parametrize("T,Hq,causal", [(1571, 3, 0), (8191, 1, 1), (2501, 1, 1), (3000, 1, 1), (2900, 3, 0)])
def test_the_parts_sums_of_a_forward_pass_start_at_multiples_of_16_bytes(T, Hq, causal):
    """the workspace of a sequence that is cut over its keys: statistics, then sums of D values, which are written 16 bytes at a time"""
    size = lambda D: _lib.load().simvg_packed_attn_ws_floats(T, 1, Hq, 1, D, causal, 0)  # noqa: E731
    rows = (size(72) - size(64)) // 8                                       # parts x T x Hq
    assert rows > T * Hq and rows % (T * Hq) == 0 and size(128) - size(64) == 64 * rows
    stats = size(64) - 64 * rows
    assert stats >= 2 * rows and stats % 4 == 0


def rope_args(**over):
    """q, k, results and gradients apart from each other, 64 KiB each"""
    at = {n: (i + 1) << 16 for i, n in enumerate(("q", "k", "q_out", "k_out", "dq", "dk"))}
    strides = {p + s: v for p in ("q", "k", "qo", "ko", "dq", "dk") for s, v in (("_ts", 4 * 64), ("_hs", 64))}
    return _lib.QkNormRopeArgs(**(dict(dtype=1, T=20, Hq=4, Hkv=4, D=64, n_axes=1, sections=(C.c_int * 4)(32), eps=1e-6, pos=1 << 20, pos_ld=1,
                                       inv_freq=1 << 21, gq=1 << 22, gk=1 << 22, dgq=1 << 23, dgk=1 << 24, ws=1 << 25) | at | strides | over))


NO_DEVICE = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="would launch on made-up addresses")


def test_rotation_refuses_results_on_other_operands():
    lib = _lib.load()
    a = 1 << 16
    q, k, qo, ko, dq, dk = (i * a for i in range(1, 7))
    both = (lib.simvg_qk_norm_rope_fwd, lib.simvg_qk_norm_rope_bwd)
    for fns, bad in ((both, dict(q_out=k)), (both, dict(k_out=q)), (both, dict(q_out=ko)), (both, dict(q_out=q + 2)), (both, dict(q_out=q + 128)),
                     (both, dict(q_out=q, qo_ts=4 * 64 + 8)), (both, dict(k_out=k, ko_hs=72)), (both, dict(q_out=ko + 16)),
                     (both[1:], dict(q_out=dk)), (both[1:], dict(k_out=dq)), (both[1:], dict(q_out=dq + 8)), (both[1:], dict(k_out=dk - 64))):
        for fn in fns:
            assert refused(fn, rope_args(**bad), "overlaps"), bad


@NO_DEVICE
def test_rotation_takes_results_in_place_and_slices_of_one_buffer():
    lib = _lib.load()
    a = 1 << 16
    q, k, dq, dk = a, 2 * a, 5 * a, 6 * a
    fused = {p + "_ts": 12 * 64 for p in ("q", "k", "qo", "ko", "dq", "dk")}
    for ok in (dict(q_out=q, k_out=k), dict(q_out=q), dict(k=q + 512, **fused), dict(q_out=q + 512, k_out=q + 1024, **fused),
               dict(k=q + 512, q_out=q, k_out=q + 512, **fused)):
        for fn in (lib.simvg_qk_norm_rope_fwd, lib.simvg_qk_norm_rope_bwd):
            assert not refused(fn, rope_args(**ok), "overlaps"), ok
    for ok in (dict(T=1, q_out=q, qo_ts=8, k_out=k, ko_ts=1 << 24), dict(Hkv=1, k_out=k, ko_hs=8)):       # strides that are never walked
        assert not refused(lib.simvg_qk_norm_rope_fwd, rope_args(**ok), "overlaps"), ok
    for ok in (dict(q_out=dq, k_out=dk), dict(q_out=q, k_out=dk)):
        assert not refused(lib.simvg_qk_norm_rope_bwd, rope_args(**ok), "overlaps"), ok


@NO_DEVICE
def test_overlap_is_told_exactly():
    """the check against the sets of values themselves, over small strides: exact where the token strides are the same, never too lax"""
    rng, lib = random.Random(0), _lib.load()

    def values(p, ts, hs, T, H, D):
        return {p // 2 + t * ts + h * hs + d for t, h, d in itertools.product(range(T), range(H), range(D))}
    seen = [0, 0]
    for _ in range(3000):
        T, Hq, Hkv, D = rng.randint(1, 5), rng.randint(1, 3), rng.randint(1, 3), rng.choice([2, 4])
        base, ts, hs = 1 << 16, rng.choice([0, 2, 5, 8, 13, 24]), rng.choice([0, 2, 4, 7, 30])
        ts2, hs2 = rng.choice([ts, ts, ts, 3, 8, 12]), rng.choice([hs, hs, 3, 9])
        p2 = base + 2 * rng.randint(-120, 120)
        args = rope_args(T=T, Hq=Hq, Hkv=Hkv, D=D, sections=(C.c_int * 4)(1), gq=None, gk=None, q=1 << 30, k=1 << 31, q_out=base, qo_ts=ts, qo_hs=hs,
                         k_out=p2, ko_ts=ts2, ko_hs=hs2)
        common = bool(values(base, ts, hs, T, Hq, D) & values(p2, ts2, hs2, T, Hkv, D))
        no = refused(lib.simvg_qk_norm_rope_fwd, args, "overlaps")
        assert no if common else (T > 1 and ts != ts2) or not no, (T, Hq, Hkv, D, ts, hs, ts2, hs2, p2 - base)
        seen[common] += 1
    assert min(seen) > 500


def attn_args(**over):
    names = ("q", "k", "v", "o", "d_o", "dq", "dk", "dv")
    at = {n: (i + 1) << 16 for i, n in enumerate(names)}
    strides = {p + s: v for p in ("q", "k", "v", "o", "do", "dq", "dk", "dv") for s, v in (("_ts", 4 * 64), ("_hs", 64))}
    return _lib.PackedAttnArgs(**(dict(dtype=2, T=20, nseq=1, Hq=4, Hkv=2, D=64, causal=1, scale=0.125, plan=1 << 20, lse=1 << 21, lse_hs=20,
                                       ws=1 << 22) | at | strides | over))


def test_attention_refuses_results_on_operands():
    lib = _lib.load()
    q, k, v, o, do, dq, dk, dv = (i << 16 for i in range(1, 9))
    for bad in (dict(o=q), dict(o=k), dict(o=v), dict(o=q + 128), dict(o=k + 16), dict(o=v - 64)):
        assert refused(lib.simvg_packed_attn_fwd, attn_args(**bad), "overlaps"), bad
    for bad in (dict(dq=q), dict(dq=do), dict(dq=o + 128), dict(dk=k), dict(dk=v + 128), dict(dv=v), dict(dv=q + 256), dict(dk=dv), dict(dq=dk + 128),
                dict(dv=dq + 16), dict(dk=do + 32)):
        assert refused(lib.simvg_packed_attn_bwd, attn_args(**bad), "overlaps"), bad


@NO_DEVICE
def test_attention_takes_slices_of_one_buffer():
    lib = _lib.load()
    q, dq = 1 << 16, 6 << 16
    fused = {p + "_ts": 16 * 64 for p in ("q", "k", "v", "o", "do", "dq", "dk", "dv")}
    heads = {p + s: v for p in ("q", "k", "v", "o") for s, v in (("_ts", 64), ("_hs", 20 * 64))}       # [heads][tokens][D]
    for ok in (dict(k=q + 512, v=q + 768, o=q + 1024, **fused), dict(k=q + 4 * 2560, v=q + 6 * 2560, o=q + 8 * 2560, **heads)):
        assert not refused(lib.simvg_packed_attn_fwd, attn_args(**ok), "overlaps"), ok
    for ok in (dict(dk=dq + 512, dv=dq + 768, **fused), dict(k=q + 512, v=q + 768, dq=q + 1024, dk=q + 1536, dv=q + 1792, **fused)):
        assert not refused(lib.simvg_packed_attn_bwd, attn_args(**ok), "overlaps"), ok


def test_reduced_loss_refuses_before_launching():
    fn = _lib.load().simvg_vocab_ce_reduce
    for bad in (dict(M=-1), dict(M=(1 << 22) + 1), dict(loss=None), dict(target=None), dict(total=None), dict(count=None)):
        a = dict(loss=256, target=512, ignore_index=-100, M=4, mean=1, total=768, count=1024) | bad
        assert fn(*a.values(), None) < 0 and b"vocab_ce_reduce" in _lib.load().simvg_last_error(), bad


@NO_DEVICE
def test_strides_that_are_never_walked_are_not_looked_at():
    lib, names = _lib.load(), ("q", "k", "v", "o", "do", "dq", "dk", "dv")
    for ok in ({"T": 1} | {n + "_ts": (1 << 30) + 3 for n in names}, {"Hq": 1, "Hkv": 1} | {n + "_hs": 1 for n in names}):
        for fn in (lib.simvg_packed_attn_fwd, lib.simvg_packed_attn_bwd):
            assert not refused(fn, attn_args(**ok), "packed_attn"), ok
    for bad, words in (({n + "_ts": 3 for n in names}, "16 bytes"), ({n + "_hs": 3 for n in names}, "16 bytes"), (dict(q_ts=1 << 24), "2^24")):
        assert refused(lib.simvg_packed_attn_fwd, attn_args(**bad), words), bad
    assert lib.simvg_packed_attn_fwd(None, None) < 0 and lib.simvg_packed_attn_bwd(None, None) < 0
