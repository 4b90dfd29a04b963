"""CPU: argument checks of the sequence operators (they return before any launch) and the layout of their argument blocks."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest
import torch

from simvg_amd import _lib, hip_ops as ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BLOCKS = {"simvg_qk_norm_rope_args": _lib.QkNormRopeArgs, "simvg_packed_attn_args": _lib.PackedAttnArgs,
          "simvg_vocab_ce_args": _lib.VocabCeArgs}


def test_argument_blocks_have_the_headers_layout(tmp_path):
    """every member's offset and the size: the header's struct as a C compiler lays it out, the kernels' own declaration of it, and
    the ctypes mirror"""
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = []
    for name, mirror in BLOCKS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f[0]} %zu\\n", offsetof({name}, {f[0]}));' for f in mirror._fields_]
    hdr = os.path.join(ROOT, "include", "simvg_hip.h")
    (tmp_path / "a.c").write_text('#include <stdio.h>\n#include "%s"\nint main(void) { %s return 0; }\n' % (hdr, "\n".join(lines)))
    subprocess.run([cc, str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    got = dict(ln.split() for ln in subprocess.run([str(tmp_path / "a")], check=True, capture_output=True, text=True).stdout.splitlines())
    header = open(hdr).read()
    for name, mirror in BLOCKS.items():
        assert int(got[name]) == C.sizeof(mirror), name
        for f in mirror._fields_:
            assert int(got[f"{name}.{f[0]}"]) == getattr(mirror, f[0]).offset, (name, f[0])
        declared = []
        for src in (header, *(open(os.path.join(ROOT, "simvg_amd", "csrc", f)).read() for f in ("rope.hip", "packed_attn.hip", "vocab_ce.hip"))):
            m = re.search(r"struct %s \{(.*?)\n\}" % name, src, flags=re.S)
            if m:
                declared.append(re.sub(r"\s+", "", re.sub(r"//[^\n]*", "", m.group(1))))
        assert len(declared) == 2 and declared[0] == declared[1], name


def _refused(fn, args, words):
    assert fn(C.byref(args), None) < 0
    assert words in _lib.load().simvg_last_error().decode(), _lib.load().simvg_last_error()


def test_rope_refuses_before_launching():
    lib = _lib.load()
    ok = dict(dtype=1, T=4, Hq=2, Hkv=1, D=64, n_axes=1, sections=(C.c_int * 4)(32), eps=1e-6)
    for bad, words in ((dict(dtype=3), "dtype"), (dict(T=-1), "T >= 0"), (dict(T=1 << 26), "too many"), (dict(Hkv=0), "head"), (dict(D=63), "even"), (dict(D=512), "256"),
                       (dict(n_axes=0), "axes"), (dict(n_axes=5), "axes"), (dict(sections=(C.c_int * 4)(33)), "sections"),
                       (dict(sections=(C.c_int * 4)(-1)), "negative"), (dict(sections=(C.c_int * 4)(0)), "sections"),
                       (dict(gq=16), "both"), (dict(), "null pointer")):
        for fn in (lib.simvg_qk_norm_rope_fwd, lib.simvg_qk_norm_rope_bwd):
            _refused(fn, _lib.QkNormRopeArgs(**(ok | bad)), words)
    ptr = dict(pos=256, pos_ld=1, inv_freq=256, q=256, k=256, q_out=256, k_out=256, gq=256, gk=256)
    _refused(lib.simvg_qk_norm_rope_fwd, _lib.QkNormRopeArgs(**(ok | ptr | dict(pos_ld=0))), "shorter")
    _refused(lib.simvg_qk_norm_rope_bwd, _lib.QkNormRopeArgs(**(ok | ptr)), "null pointer")
    _refused(lib.simvg_qk_norm_rope_bwd, _lib.QkNormRopeArgs(**(ok | ptr | dict(dq=256, dk=256))), "workspace")
    assert lib.simvg_qk_norm_rope_fwd(None, None) < 0


def test_attention_refuses_before_launching():
    lib = _lib.load()
    ok = dict(dtype=2, T=4, nseq=1, Hq=4, Hkv=2, D=64, scale=0.125)
    for bad, words in ((dict(dtype=0), "fp16 or bf16"), (dict(T=-1), "negative"), (dict(nseq=-1), "negative"), (dict(Hq=3), "multiple"),
                       (dict(Hkv=0), "multiple"), (dict(D=60), "multiple of 8"), (dict(D=136), "128"), (dict(D=0), "multiple of 8"),
                       (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
                       (dict(T=1 << 30, Hq=1 << 20, Hkv=1), "too many"), (dict(T=1 << 20, Hq=1 << 12, Hkv=1), "too many"), (dict(), "null pointer")):
        for fn in (lib.simvg_packed_attn_fwd, lib.simvg_packed_attn_bwd):
            _refused(fn, _lib.PackedAttnArgs(**(ok | bad)), words)
    rows = {n: 256 for n in ("plan", "lse", "q", "k", "v", "o")} | {n + s: 64 for n in "qkvo" for s in ("_ts", "_hs")}
    for bad in (dict(q=264), dict(k_ts=60), dict(v_hs=4)):
        _refused(lib.simvg_packed_attn_fwd, _lib.PackedAttnArgs(**(ok | rows | bad)), "16 bytes")
    _refused(lib.simvg_packed_attn_bwd, _lib.PackedAttnArgs(**(ok | rows)), "gradients")
    grads = {n: 256 for n in ("d_o", "dq", "dk", "dv")}
    _refused(lib.simvg_packed_attn_bwd, _lib.PackedAttnArgs(**(ok | rows | grads)), "workspace")
    assert lib.simvg_packed_plan(None, 1, 4, None, None) < 0 and lib.simvg_packed_plan(256, -1, 4, 256, None) < 0
    assert lib.simvg_packed_plan_ints(-1, 3) == 0 and lib.simvg_packed_plan_ints(1000, 3) > 0
    assert lib.simvg_packed_attn_ws_floats(-1, 1, 1, 1, 64, 1, 1) == 0


def test_vocab_ce_refuses_before_launching():
    lib = _lib.load()
    ok = dict(dtype=1, M=4, V=100, K=64, ldx=64, ldw=64)
    ptr = dict(x=256, w=256, target=256, lse=256, loss=256)
    for bad, words in ((dict(dtype=0), "fp16 or bf16"), (dict(M=-1), "M >= 0"), (dict(V=0), "V >= 1"), (dict(K=60), "multiple of 8"), (dict(K=0), "K >= 8"),
                       (dict(M=1 << 23), "too large"), (dict(M=1 << 22, V=1 << 24), "too many"), (dict(ldx=56), "strides"), (dict(ldw=1 << 21), "strides"), (dict(w=None), "16 bytes"),
                       (dict(x=264), "16 bytes"), (dict(target=None), "null pointer"), (dict(lse=None), "null pointer")):
        for fn in (lib.simvg_vocab_ce_fwd, lib.simvg_vocab_ce_bwd):
            _refused(fn, _lib.VocabCeArgs(**(ok | ptr | bad)), words)
    _refused(lib.simvg_vocab_ce_fwd, _lib.VocabCeArgs(**(ok | ptr | dict(loss=None))), "null pointer")
    _refused(lib.simvg_vocab_ce_fwd, _lib.VocabCeArgs(**(ok | ptr)), "workspace")
    grads = dict(dloss=256, dx=256, dw=256, lddx=64, lddw=64)
    _refused(lib.simvg_vocab_ce_bwd, _lib.VocabCeArgs(**(ok | ptr)), "null pointer")
    _refused(lib.simvg_vocab_ce_bwd, _lib.VocabCeArgs(**(ok | ptr | grads | dict(lddw=56))), "gradients")
    _refused(lib.simvg_vocab_ce_bwd, _lib.VocabCeArgs(**(ok | ptr | grads | dict(dbias=256))), "bias")
    _refused(lib.simvg_vocab_ce_bwd, _lib.VocabCeArgs(**(ok | ptr | grads)), "workspace")
    need = lib.simvg_vocab_ce_ws_bytes(4, 100, 64, 0, 1)
    assert need > 0 and need % 256 == 0
    _refused(lib.simvg_vocab_ce_bwd, _lib.VocabCeArgs(**(ok | ptr | grads | dict(ws=256, ws_bytes=need - 1))), "workspace")
    assert lib.simvg_vocab_ce_ws_bytes(0, 100, 64, 0, 1) == 0


def test_operators_refuse_cpu_tensors():
    q = torch.zeros(3, 2, 64, dtype=torch.float16)
    with pytest.raises(_lib.SimvgHipError):
        ops.qk_norm_rope_fwd(q, q, torch.zeros(3, 1, dtype=torch.int32), torch.zeros(32, dtype=torch.float64), (32,))
    with pytest.raises(_lib.SimvgHipError):
        ops.packed_plan(torch.zeros(2, dtype=torch.int32), 3)
    with pytest.raises(_lib.SimvgHipError):
        ops.packed_attn_fwd(q, q, q, ops.PackedPlan(None, 1, 3, torch.zeros(8, dtype=torch.int32)))
    with pytest.raises(_lib.SimvgHipError):
        ops.vocab_ce_fwd(torch.zeros(3, 64, dtype=torch.float16), torch.zeros(5, 64, dtype=torch.float16), torch.zeros(3, dtype=torch.int64))
    from simvg_amd.models import sequence
    with pytest.raises(ValueError):
        sequence.vocab_cross_entropy(q[:, 0], q[:, 1], None, reduction="max")


def test_the_definitions_in_64_bits_agree_with_torch():
    """tests/sequence_ref.py itself, on the CPU: against torch's own softmax, loss and differentiation"""
    import sequence_ref as R
    torch.manual_seed(0)
    lens, Hq, Hkv, D = [5, 0, 9], 4, 2, 8
    q, k, v, do = (torch.randn(14, h, D).half() for h in (Hq, Hkv, Hkv, Hq))
    for causal in (True, False):
        r = R.attention(q, k, v, lens, causal, 0.3, do)
        Q, K, V = (t.double().requires_grad_() for t in (q, k, v))
        out, at = [], 0
        for n in lens:
            s = torch.einsum("ihd,jhd->hij", Q[at:at + n], K[at:at + n].repeat_interleave(2, 1)) * 0.3
            if causal:
                s = s + torch.full((n, n), float("-inf"), dtype=torch.float64).triu(1)
            out.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), V[at:at + n].repeat_interleave(2, 1)))
            at += n
        want = torch.cat(out)
        grads = torch.autograd.grad(want, (Q, K, V), do.double())
        for a, b in zip((r["o"], r["dq"], r["dk"], r["dv"]), (want, *grads)):
            assert float((a - b).abs().max()) < 1e-12
    x, w, b = torch.randn(6, 16).half(), torch.randn(11, 16).half(), torch.randn(11)
    t, g = torch.tensor([3, -100, 0, 10, 5, 5]), torch.randn(6)
    r = R.vocab_ce(x, w, t, b, g)
    X, W, Bd = x.double().requires_grad_(), w.double().requires_grad_(), b.double().requires_grad_()
    loss = torch.nn.functional.cross_entropy(X @ W.t() + Bd, t, reduction="none")
    grads = torch.autograd.grad(loss, (X, W, Bd), g.double())
    for a, c in zip((r["loss"], r["dx"], r["dw"], r["dbias"]), (loss, *grads)):
        assert float((a - c).abs().max()) < 1e-12
    # a rotation keeps the length of every pair, and position 0 changes nothing
    y = torch.randn(4, 2, 12).double()
    pos, inv = torch.tensor([[0, 0], [3, 5], [7, 0], [0, 9]]), torch.rand(5).double()
    for inter in (False, True):
        z, _ = R.rope(y, None, pos, inv, (2, 3), 0.0, inter)
        assert torch.equal(z[0], y[0]) and torch.allclose(z.square().sum(-1), y.square().sum(-1)) and torch.equal(z[..., 10:], y[..., 10:])
