"""What is measured of the sequence operators: the normalised, rotated queries and keys, the attention over packed prompts
that reads them, and the cross entropy over a vocabulary.

`listed()` / `draw()` name the cases, `prepare()` makes the inputs of one, `run()` makes one pass (the framework's kernels where
`own` is true, elementary torch operations in 32 bits where it is not), `exact()` gives the same outputs in 64 bits.

    rope   y = R(theta) (x / rms(x) * g) for every head of q and k, theta[t, j] = pos[t, axis(j)] * inv_freq[j]
    attn   o[i] = sum_j softmax_j(scale q[i].k[j]) v[j] over the keys j of i's own sequence (j <= i where causal)
    loss   loss[i] = log sum_v exp(z[i, v]) - z[i, target[i]],  z = x w^T + bias
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-6
GRAD_SCALE = 1024.0             # what a 16-bit backward pass of this framework carries by default: gradients in fp16's normal range


# ---------------------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # one new token of a grouped-head decoder: the latency of the launch itself
        dict(name="rope one token bf16", op="rope", train=False, dtype="bf16", T=1, Hq=32, Hkv=8, D=128, sections="16 24 24",
             interleaved=False, span=32768),
        # queries and keys of a ViT-B batch, 64 pairs of 20 x 20 patches + 21 tokens, rows and columns as the two axes
        dict(name="rope image batch fp16", op="rope", train=False, dtype="fp16", T=64 * 421, Hq=12, Hkv=12, D=64,
             sections="16 16", interleaved=False, span=32),
        # a packed training batch of long prompts: three axes, far positions, gradients of the inputs and of the norms' weights
        dict(name="rope train bf16", op="rope", train=True, dtype="bf16", T=16384, Hq=32, Hkv=8, D=128, sections="16 24 24",
             interleaved=False, span=1 << 20),
        # the exact mode's rows, an odd count of them, half of the head rotated, neighbouring pairs, one key head
        dict(name="rope train odd fp32", op="rope", train=True, dtype="fp32", T=4099, Hq=7, Hkv=1, D=80, sections="9 11",
             interleaved=True, span=4096),
        # 64 referring expressions of up to 20 tokens: many short sequences, some of them empty
        dict(name="attn expressions fp16", op="attn", train=False, dtype="fp16", n=64, lo=0, hi=20, tail=0, len_seed=1, Hq=12,
             Hkv=12, D=64, causal=True),
        # image patches and text of 64 pairs, packed without their padding, all keys visible
        dict(name="attn train pairs fp16", op="attn", train=True, dtype="fp16", n=64, lo=401, hi=421, tail=37, len_seed=2, Hq=12,
             Hkv=12, D=64, causal=False),
        # one long prompt
        dict(name="attn prompt bf16", op="attn", train=False, dtype="bf16", n=1, lo=16384, hi=16384, tail=0, len_seed=3, Hq=16,
             Hkv=2, D=128, causal=True),
        # a packed training batch of documents of very different lengths
        dict(name="attn train documents bf16", op="attn", train=True, dtype="bf16", n=9, lo=1, hi=4097, tail=5, len_seed=4, Hq=32,
             Hkv=8, D=128, causal=True),
        # the likelihood of one expression of 20 tokens
        dict(name="loss expression fp16", op="loss", train=False, dtype="fp16", M=20, V=64010, K=768, bias=True, ignored=0.0),
        # masked tokens of a batch of 64 expressions, with the head's bias
        dict(name="loss train masked fp16", op="loss", train=True, dtype="fp16", M=1280, V=64010, K=768, bias=True, ignored=0.6),
        # a vocabulary and a width that divide by nothing convenient
        dict(name="loss train odd bf16", op="loss", train=True, dtype="bf16", M=333, V=32003, K=520, bias=False, ignored=0.1),
        # a packed batch of captions through ViT-L's width
        dict(name="loss train captions bf16", op="loss", train=True, dtype="bf16", M=8191, V=64010, K=1024, bias=False, ignored=0.0),
    ]


def _spread(rng, lo, hi):
    """a whole number of [lo, hi], evenly over the logarithm"""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "attn", "loss"])
    train = rng.random() < 0.6
    if op == "rope":
        D = rng.choice([32, 64, 80, 96, 128, 256])
        Hkv = rng.choice([1, 2, 3, 4, 8, 12])
        Hq = Hkv * rng.choice([1, 2, 4, 7])
        pairs = rng.choice([D // 2, D // 2, D // 4])
        axes = rng.randint(1, 4)
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        most = 16384 * 40 * 128 // (2 * (Hq + Hkv) * D)
        return dict(op="rope", train=train, dtype=rng.choice(["fp16", "bf16", "fp32"]), T=_spread(rng, 1, min(32768, most)), Hq=Hq,
                    Hkv=Hkv, D=D, sections=" ".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs])), interleaved=rng.random() < 0.5,
                    span=_spread(rng, 2, 1 << 20))
    if op == "attn":
        D = rng.choice([32, 64, 64, 80, 96, 128, 128])
        Hkv = rng.choice([1, 2, 4, 8, 12])
        Hq = Hkv * rng.choice([1, 1, 2, 4, 7])
        hi = _spread(rng, 1, 8192)
        # the plain form's scores of all sequences, padded to the longest, stay under four GiB
        n = _spread(rng, 1, max(1, min(512, (1 << 30) // (Hq * hi * hi), 65536 // hi)))
        Hq, Hkv = (Hq, Hkv) if Hq * hi * hi <= 1 << 30 else (12, 12) if 12 * hi * hi <= 1 << 30 else (8, 2)
        return dict(op="attn", train=train, dtype=rng.choice(["fp16", "bf16"]), n=n, lo=rng.randint(0, hi), hi=hi,
                    tail=rng.choice([0, 0, 3, 200]), len_seed=rng.randrange(1 << 20), Hq=Hq, Hkv=Hkv, D=D, causal=rng.random() < 0.7)
    K = rng.choice([256, 264, 520, 768, 1024, 2048])
    V = _spread(rng, 1000, 131072)
    M = _spread(rng, 1, max(1, min(16384, 8191 * 64010 * 1024 // (V * K), (1 << 30) // V)))
    return dict(op="loss", train=train, dtype=rng.choice(["fp16", "bf16"]), M=M, V=V, K=K, bias=rng.random() < 0.5,
                ignored=rng.choice([0.0, 0.1, 0.6]))


def _lengths(case):
    rng = random.Random(case["len_seed"])
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["n"])]
    lens[rng.randrange(len(lens))] = case["hi"]
    return lens


def _sections(case):
    return [int(n) for n in case["sections"].split()]


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rope":
        rows, T = case["T"] * (case["Hq"] + case["Hkv"]), case["T"]
        n = rows * case["D"] * size
        # a training pass is the forward pass (read, write) and the backward pass (inputs and gradients read, gradients written)
        return {"bytes": n * (5 if case["train"] else 2) + T * len(_sections(case)) * 4, "flops": rows * case["D"] * (20 if case["train"] else 7)}
    if case["op"] == "attn":
        lens = _lengths(case)
        T, D, Hq, Hkv = sum(lens), case["D"], case["Hq"], case["Hkv"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        q, kv, lse = T * Hq * D * size, 2 * T * Hkv * D * size, T * Hq * 4
        # forward: q k^T and p v.  Backward: the scores again (they are not kept), dv, dp, dq, dk
        if not case["train"]:
            return {"bytes": 2 * q + kv + lse, "flops": 4 * pairs * Hq * D}
        return {"bytes": 6 * q + 3 * kv + 2 * lse, "flops": 14 * pairs * Hq * D}
    M, V, K = case["M"], case["V"], case["K"]
    n = (M * K + V * K) * size + M * 20
    # forward: the logits.  Backward: the logits again (they are not kept), dx, dw
    return {"bytes": n * (3 if case["train"] else 1), "flops": 2 * M * V * K * (4 if case["train"] else 1)}


# --------------------------------------------------------------------------------------------------------------- the inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)

    s = dict(case=case)
    if case["op"] == "rope":
        T, Hq, Hkv, D = case["T"], case["Hq"], case["Hkv"], case["D"]
        qkv = normal(T, (Hq + 2 * Hkv) * D)                                   # the projection's output: q | k | v of a row
        s["q"] = qkv[:, :Hq * D].view(T, Hq, D)
        s["k"] = qkv[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
        s["gq"] = 1.0 + normal(D, std=0.1, dtype=torch.float32)
        s["gk"] = 1.0 + normal(D, std=0.1, dtype=torch.float32)
        s["sections"] = _sections(case)
        pairs = sum(s["sections"])
        s["inv_freq"] = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float64) / pairs)
        s["pos"] = torch.randint(0, case["span"], (T, len(s["sections"])), generator=g, device="cuda", dtype=torch.int32)
        if case["train"]:
            s["dq"], s["dk"] = normal(T, Hq, D), normal(T, Hkv, D)
    elif case["op"] == "attn":
        lens = _lengths(case)
        Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
        T = sum(lens) + case["tail"]
        qkv = normal(T, (Hq + 2 * Hkv) * D)
        s["q"] = qkv[:, :Hq * D].view(T, Hq, D)
        s["k"] = qkv[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D)
        s["v"] = qkv[:, (Hq + Hkv) * D:].view(T, Hkv, D)
        s["cu"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32).cuda()
        s["longest"] = max(lens)
        if case["train"]:
            s["do"] = normal(T, Hq, D)
    else:
        M, V, K = case["M"], case["V"], case["K"]
        s["x"], s["w"] = normal(M, K), normal(V, K, std=1.5 / math.sqrt(K))
        s["bias"] = normal(V, std=0.5, dtype=torch.float32) if case["bias"] else None
        target = torch.randint(0, V, (M,), generator=g, device="cuda")
        skip = torch.rand(M, generator=g, device="cuda") < case["ignored"]
        s["target"] = torch.where(skip, torch.full_like(target, -100), target)
        if case["train"]:
            s["dloss"] = torch.where(skip, 0.0, GRAD_SCALE / max(1, int((~skip).sum()))).float()
    return s


# ------------------------------------------------------------------------------------------------------------------ one pass

def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"rope": _plain_rope, "attn": _plain_attn, "loss": _plain_loss}[case["op"]](s, case)


def _own(s, case):
    from simvg_amd import hip_ops as ops
    if case["op"] == "rope":
        args = (s["q"], s["k"], s["pos"], s["inv_freq"], s["sections"], s["gq"], s["gk"], EPS, case["interleaved"])
        out = list(ops.qk_norm_rope_fwd(*args))
        return out + list(ops.qk_norm_rope_bwd(s["dq"], s["dk"], *args)) if case["train"] else out
    if case["op"] == "attn":
        plan = ops.packed_plan(s["cu"], s["q"].shape[0])
        o, lse = ops.packed_attn_fwd(s["q"], s["k"], s["v"], plan, causal=case["causal"])
        if not case["train"]:
            return [o, lse]
        return [o, lse] + list(ops.packed_attn_bwd(s["q"], s["k"], s["v"], o, lse, s["do"], plan, causal=case["causal"]))
    loss, lse = ops.vocab_ce_fwd(s["x"], s["w"], s["target"], s["bias"])
    if not case["train"]:
        return [loss, lse]
    return [loss, lse] + [t for t in ops.vocab_ce_bwd(s["x"], s["w"], s["target"], lse, s["dloss"], s["bias"]) if t is not None]


def _pairs(x, pairs, interleaved):
    """the two halves of every rotated pair, and what is not rotated"""
    head, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if interleaved:
        return head[..., 0::2], head[..., 1::2], rest
    return head[..., :pairs], head[..., pairs:], rest


def _joined(a, b, rest, interleaved):
    head = torch.stack([a, b], dim=-1).flatten(-2) if interleaved else torch.cat([a, b], dim=-1)
    return torch.cat([head, rest], dim=-1)


def _plain_rope(s, case):
    pairs, inter = sum(s["sections"]), case["interleaved"]
    # far positions: angles in 64 bits
    theta = torch.cat([s["pos"][:, a:a + 1].expand(-1, c) for a, c in enumerate(s["sections"])], dim=1).double() * s["inv_freq"]
    cos, sin = torch.cos(theta).float()[:, None], torch.sin(theta).float()[:, None]

    def forward(x, g):
        x32 = x.float()
        y = x32 * torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS) * g
        a, b, rest = _pairs(y, pairs, inter)
        return _joined(a * cos - b * sin, a * sin + b * cos, rest, inter).to(x.dtype)

    def backward(dy, x, g):
        x32 = x.float()
        r = torch.rsqrt((x32 * x32).mean(-1, keepdim=True) + EPS)
        a, b, rest = _pairs(dy.float(), pairs, inter)
        dz = _joined(a * cos + b * sin, b * cos - a * sin, rest, inter)
        n = x32 * r
        dn = dz * g
        return (r * (dn - n * (dn * n).mean(-1, keepdim=True))).to(x.dtype), (dz * n).sum((0, 1))

    out = [forward(s["q"], s["gq"]), forward(s["k"], s["gk"])]
    if case["train"]:
        (dq, dgq), (dk, dgk) = backward(s["dq"], s["q"], s["gq"]), backward(s["dk"], s["k"], s["gk"])
        out += [dq, dk, dgq, dgk]
    return out


def _plain_attn(s, case):
    """every sequence padded to the longest one; row T is where what belongs to no sequence comes from and goes to"""
    q, k, v, cu, L = s["q"], s["k"], s["v"], s["cu"].long(), s["longest"]
    T, Hq, D = q.shape
    Hkv, n = k.shape[1], cu.numel() - 1
    G, scale = Hq // Hkv, D ** -0.5
    at = torch.arange(L, device="cuda")
    inside = at < (cu[1:] - cu[:-1])[:, None]                                              # [n, L]
    row = torch.where(inside, cu[:-1, None] + at, T)

    def queries(x):                                                                       # [T, Hq, D] -> [n, Hkv, G L, D]
        x = torch.cat([x.float(), torch.zeros(1, Hq, D, device="cuda")])[row]
        return x.view(n, L, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(n, Hkv, G * L, D)

    def keys(x):
        x = torch.cat([x.float(), torch.zeros(1, Hkv, D, device="cuda")])[row]
        return x.permute(0, 2, 1, 3).contiguous()                                         # [n, Hkv, L, D]

    def back(x, heads):                                                                   # [n, heads, L, D] -> [T, heads, D]
        out = torch.zeros(T + 1, heads, x.shape[-1], device="cuda")
        out[row] = x.permute(0, 2, 1, 3)
        out[T] = 0
        return out[:T]

    def of_queries(x):
        return back(x.view(n, Hkv, G, L, -1).reshape(n, Hq, L, -1), Hq)

    seen = inside[:, None, :] & inside[:, :, None]
    if case["causal"]:
        seen = seen & (at[None, :] <= at[:, None])
    Q, K, V = queries(q), keys(k), keys(v)
    S = (Q @ K.transpose(2, 3)).mul_(scale).view(n, Hkv, G, L, L).masked_fill_(~seen[:, None, None], float("-inf"))
    m = S.amax(-1, keepdim=True).clamp_(min=-1e30)
    P = S.sub_(m).exp_()
    total = P.sum(-1, keepdim=True)
    some = total > 0
    P = P.div_(torch.where(some, total, 1.0)).view(n, Hkv, G * L, L)
    O = P @ V
    lse = torch.where(some, m + total.clamp(min=1e-30).log(), 0.0)
    out = [of_queries(O).to(q.dtype), of_queries(lse).squeeze(-1).t().contiguous()]
    if case["train"]:
        dO = queries(s["do"])
        dV = P.transpose(2, 3) @ dO
        delta = (dO * O).sum(-1, keepdim=True)
        dS = (dO @ V.transpose(2, 3)).sub_(delta).mul_(P).mul_(scale)
        out += [of_queries(dS @ K).to(q.dtype), back(dS.transpose(2, 3) @ Q, Hkv).to(q.dtype), back(dV, Hkv).to(q.dtype)]
    return out


def _plain_loss(s, case):
    x, w, target = s["x"].float(), s["w"].float(), s["target"]
    z = x @ w.t()
    if s["bias"] is not None:
        z = z.add_(s["bias"])
    m = z.amax(-1, keepdim=True)
    kept = target >= 0
    at = target.clamp(min=0)[:, None]
    zt = z.gather(1, at).squeeze(1)
    p = z.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    lse = (m + total.log()).squeeze(1)
    out = [torch.where(kept, lse - zt, 0.0), lse]
    if case["train"]:
        dz = p.div_(total).scatter_add_(1, at, torch.full_like(total, -1.0)).mul_(torch.where(kept, s["dloss"], 0.0)[:, None])
        out += [(dz @ w).to(s["x"].dtype), (dz.t() @ x).to(s["w"].dtype)]
        if s["bias"] is not None:
            out.append(dz.double().sum(0).float())
    return out


# ------------------------------------------------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "loss": _exact_loss}[case["op"]](s, case)


def _exact_rope(s, case):
    """a pair as a complex number, turned by exp(i theta); gradients by differentiation of that"""
    pairs = sum(s["sections"])
    axis = [a for a, count in enumerate(s["sections"]) for _ in range(count)]
    theta = s["pos"].double()[:, axis] * s["inv_freq"]
    turn = torch.polar(torch.ones_like(theta), theta)

    def value(x, g):
        y = g * x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
        z = y[..., :2 * pairs].unflatten(-1, (pairs, 2) if case["interleaved"] else (2, pairs))
        z = z if case["interleaved"] else z.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn[:, None])
        return torch.cat([(z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2), y[..., 2 * pairs:]], dim=-1)

    leaves = [s[n].double().requires_grad_(case["train"]) for n in ("q", "k", "gq", "gk")]
    out = [value(leaves[0], leaves[2]), value(leaves[1], leaves[3])]
    if not case["train"]:
        return out
    return [t.detach() for t in out] + list(torch.autograd.grad(out, leaves, [s["dq"].double(), s["dk"].double()]))


def _exact_attn(s, case):
    """one sequence and one key head after the other, queries in blocks"""
    q, k, v = s["q"], s["k"], s["v"]
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    zeros = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
    o, lse, dq, dk, dv = zeros(T, Hq, D), zeros(Hq, T), zeros(T, Hq, D), zeros(T, Hkv, D), zeros(T, Hkv, D)
    first = 0
    for n in _lengths(case):
        for h in range(Hkv if n else 0):
            heads = slice(h * G, (h + 1) * G)
            kk, vv = (t[first:first + n, h].double().requires_grad_(case["train"]) for t in (k, v))
            step = max(1, (1 << 27) // (n * G))
            for i in range(0, n, step):
                rows = slice(first + i, first + min(n, i + step))
                qq = q[rows, heads].double().requires_grad_(case["train"])
                z = torch.matmul(qq.transpose(0, 1), kk.t()) / math.sqrt(D)
                if case["causal"]:
                    hidden = torch.arange(n, device="cuda") > torch.arange(i, i + qq.shape[0], device="cuda")[:, None]
                    z = z.masked_fill(hidden, float("-inf"))
                oo = torch.matmul(torch.softmax(z, -1), vv).transpose(0, 1)
                o[rows, heads] = oo.detach()
                lse[heads, rows] = torch.logsumexp(z.detach(), -1)
                if case["train"]:
                    a, b, c = torch.autograd.grad(oo, (qq, kk, vv), s["do"][rows, heads].double())
                    dq[rows, heads] = a
                    dk[first:first + n, h] += b
                    dv[first:first + n, h] += c
        first += n
    return [o, lse, dq, dk, dv] if case["train"] else [o, lse]


def _exact_loss(s, case):
    """rows in blocks through torch's own loss"""
    x, w, target = s["x"], s["w"].double().requires_grad_(case["train"]), s["target"]
    bias = None if s["bias"] is None else s["bias"].double().requires_grad_(case["train"])
    step = max(1, (1 << 27) // w.shape[0])
    loss, lse, dx = [], [], []
    dw, db = torch.zeros_like(w), None if bias is None else torch.zeros_like(bias)
    for i in range(0, x.shape[0], step):
        xx = x[i:i + step].double().requires_grad_(case["train"])
        z = torch.nn.functional.linear(xx, w, bias)
        each = torch.nn.functional.cross_entropy(z, target[i:i + step], reduction="none", ignore_index=-100)
        loss.append(each.detach())
        lse.append(torch.logsumexp(z.detach(), -1))
        if case["train"]:
            grads = torch.autograd.grad(each, [xx, w] + ([] if bias is None else [bias]), s["dloss"][i:i + step].double())
            dx.append(grads[0])
            dw += grads[1]
            if bias is not None:
                db += grads[2]
    out = [torch.cat(loss), torch.cat(lse)]
    if case["train"]:
        out += [torch.cat(dx), dw.detach()] + ([] if bias is None else [db.detach()])
    return out
