"""The sequence operators in 64 bits, from their definitions, with what a kernel that accumulates in 32 bits and rounds to the operands'
type may be off: every bound below counts roundings of half a step (`torch.finfo(t).eps / 2` of the value) and additions of 2^-24.

U = 2^-24 is half a step of fp32; `h(dt)` half a step of the operands' type; in fp16 a value below 2^-14 is off by up to 2^-25.
fp32 and bf16 have no bits left below their smallest normal value 2^-126: exp2 returns 0 there (a probability e^-100 of what it is
normalised by), and so do products.  What is lost is at most 2^-126 a term: LEAST."""
import torch

U = 2.0 ** -24
LEAST = 2.0 ** -126


def h(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return 2.0 ** -25 if dt == torch.float16 else LEAST


def rounded(ref, dt):
    """what the last rounding of a result may cost"""
    return h(dt) * ref.abs() + tiny(dt)


# ---------------------------------------------------------------------------------------------------------------- norm + rotation

def rope(x, g, pos, inv_freq, sections, eps, interleaved):
    """(value, sum of the magnitudes that were added for it), x [T, H, D] float64"""
    P = sum(sections)
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    theta = pos.double()[:, axis] * inv_freq
    cos, sin = theta.cos()[:, None], theta.sin()[:, None]
    z = x if g is None else g.double() * x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    rot, rest = z[..., :2 * P], z[..., 2 * P:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :P], rot[..., P:])
    ya, yb, size = a * cos - b * sin, a * sin + b * cos, a.abs() + b.abs()

    def join(u, v):
        return torch.cat([torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1), rest], -1)
    return join(ya, yb), torch.cat([join(size, size)[..., :2 * P], rest.abs()], -1)


# ---------------------------------------------------------------------------------------------------------------------- attention

def attention(q, k, v, lens, causal, scale, dout=None):
    """dict of the results in float64 and, under "tol", their bounds; q [T, Hq, D], k, v [T, Hkv, D] in the kernel's type"""
    dt = q.dtype
    T, Hq, D = q.shape
    Hkv, G = k.shape[1], Hq // k.shape[1]
    z = lambda *s: torch.zeros(*s, dtype=torch.float64, device=q.device)  # noqa: E731
    r = dict(o=z(T, Hq, D), lse=z(Hq, T), dq=z(T, Hq, D), dk=z(T, Hkv, D), dv=z(T, Hkv, D))
    tol = {n: torch.zeros_like(t) for n, t in r.items()}
    first = 0
    for n in lens:
        rows = slice(first, first + n)
        first += n
        if n == 0:
            continue
        for hq in range(Hq):
            hk = hq // G
            Q, K, V = q[rows, hq].double(), k[rows, hk].double(), v[rows, hk].double()
            S = scale * Q @ K.t()
            if causal:
                S = S.masked_fill(torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1), float("-inf"))
            lse = torch.logsumexp(S, -1)
            P = (S - lse[:, None]).exp()
            O = P @ V
            r["o"][rows, hq], r["lse"][hq, rows] = O, lse
            # a score: D products and sums in fp32, then scale, the reference's subtraction and exp2 (a few steps of its argument)
            ds = (scale * Q.abs() @ K.abs().t()).amax(-1) * (D + 8) * U + 8 * U * (1 + lse.abs())
            # a probability is rounded to the operands' type, numerator and denominator are sums of n terms
            dp = h(dt) + 2 * ds[:, None] + (n + 64) * U
            small = tiny(dt) * V.abs().sum(0)
            eo = (P @ V.abs()) * dp + small
            tol["o"][rows, hq] = eo + rounded(O, dt)
            tol["lse"][hq, rows] = ds + (n + 64) * U + 4 * U * lse.abs()
            if dout is None:
                continue
            dO = dout[rows, hq].double()
            dP, delta = dO @ V.t(), (dO * O).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            dV, dQ, dK = P.t() @ dO, scale * dS @ K, scale * dS.t() @ Q
            r["dv"][rows, hk] += dV
            r["dq"][rows, hq] = dQ
            r["dk"][rows, hk] += dK
            # in fp16 probabilities times 2^14 and dS times 2^14 over the largest |dO| |V| (rounded up to a power of two) are rounded
            least = 2.0 ** -25 * 2.0 ** -14 if dt == torch.float16 else LEAST
            pe = P * (h(dt) + 2 * ds[:, None] + 8 * U) + least
            # dS: its own rounding, P's error, dP and delta in fp32, and delta is taken from the ROUNDED output
            de = (dO.abs() * (eo + rounded(O, dt))).sum(-1, keepdim=True) + (D + 8) * U * (dO.abs() * O.abs()).sum(-1, keepdim=True)
            dpe = (D + 8) * U * (dO.abs() @ V.abs().t()) + de
            most = dO.norm(dim=-1).max() * V.norm(dim=-1).max()
            se = dS.abs() * (h(dt) + 2 * ds[:, None] + 8 * U) + P * dpe + 4 * least * most      # |dP|, |delta| <= most
            acc = (n * G + 64) * U
            tol["dv"][rows, hk] += pe.t() @ dO.abs() + acc * (P.t() @ dO.abs())
            tol["dq"][rows, hq] = scale * (se @ K.abs() + acc * (dS.abs() @ K.abs()))
            tol["dk"][rows, hk] += scale * (se.t() @ Q.abs() + acc * (dS.abs().t() @ Q.abs()))
    for n in ("dq", "dk", "dv"):
        tol[n] += rounded(r[n], dt)
    r["tol"] = tol
    return r


# -------------------------------------------------------------------------------------------------------------------- vocabulary

def vocab_ce(x, w, target, bias, dloss=None, ignore_index=-100):
    dt, (M, K), V = x.dtype, x.shape, w.shape[0]
    X, W = x.double(), w.double()
    z = X @ W.t()
    # a logit: K products and sums in fp32, the bias, the maximum's subtraction and exp2
    dz = ((X.abs() @ W.abs().t()).amax(-1) * (K + 8) * U)
    if bias is not None:
        z = z + bias.double()
        dz = dz + 4 * U * bias.abs().max().double()
    lse = torch.logsumexp(z, -1)
    dz = dz + 8 * U * (1 + lse.abs())
    on = target != ignore_index
    zt = z.gather(1, target.clamp(min=0)[:, None]).squeeze(1)
    r = dict(loss=torch.where(on, lse - zt, 0.0), lse=lse)
    sums = (V / 256 + 256) * U                       # words summed by a lane, a strand and their joins, at the least parallel
    tol = dict(lse=dz + sums, loss=2 * dz + sums + 4 * U * (lse.abs() + zt.abs()))
    if dloss is not None:
        g = torch.where(on, dloss.double(), 0.0)[:, None]
        p = (z - lse[:, None]).exp()
        e = p.clone()
        e[torch.arange(M, device=x.device), target.clamp(min=0)] -= 1
        e = torch.where(on[:, None], e, 0.0)
        p = torch.where(on[:, None], p, 0.0)
        r.update(dx=g * (e @ W), dw=(g * e).t() @ X, dbias=(g * e).sum(0))
        least = 2.0 ** -25 * 2.0 ** -14 if dt == torch.float16 else LEAST
        exact = p * (2 * dz[:, None] + 8 * U) + 2 * U * e.abs() + LEAST
        ee = torch.where(on[:, None], h(dt) * e.abs() + exact + least, 0.0)
        gx = (g * X).abs()
        tol["dx"] = g.abs() * (ee @ W.abs() + (V / 8 + 64) * U * (e.abs() @ W.abs())) + rounded(r["dx"], dt)
        # g x / max|g| is rounded too, unless the rows' gradients are all the same
        kept = g[on].abs()
        same = kept.numel() == 0 or bool((kept == kept.max()).all())
        xe = 0.0 if same else h(dt) * gx + tiny(dt) * kept.max()
        tol["dw"] = ee.t() @ gx + (e.abs().t() @ (xe + (M / 8 + 64) * U * gx)) + rounded(r["dw"], dt)
        tol["dbias"] = (g.abs() * (exact + (M / 8 + 64) * U * e.abs())).sum(0)
    r["tol"] = tol
    return r


def off(got, ref, tol):
    """the largest error in units of its bound; inf where the result is not finite and should be"""
    got = got.double()
    if not bool(torch.isfinite(got).all()):
        return float("inf")
    d = (got - ref).abs()
    return float(torch.where(d == 0, 0.0, d / tol.clamp(min=1e-300)).max()) if got.numel() else 0.0
