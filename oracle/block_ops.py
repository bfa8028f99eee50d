"""Oracle of the block operators (include/nbx.h "Block operators"): their formulas in float64 with a running
error bound, on the CPU.

``B`` holds a value and a bound on how far a float32 computation of it may be off, whatever the order of its
sums: every operation adds half a step (EPS = 2^-24 relative) to what its operands' bounds give, a sum of n
terms n half steps of the terms' absolute sum.  ``rounded`` adds the half step of the storage type.  So a
kernel that computes the formula in float32 and rounds each result once is within the bound."""
import numpy as np
import torch

EPS = 2.0 ** -24


class B:
    def __init__(self, val, err=None):
        self.val = val.double()
        self.err = torch.zeros_like(self.val) if err is None else err.expand(self.val.shape)

    def _new(self, val, err):
        return B(val, err + EPS * val.abs())

    def __add__(self, o):
        o = o if isinstance(o, B) else B(torch.as_tensor(o, dtype=torch.float64))
        return self._new(self.val + o.val, self.err + o.err)

    def __neg__(self):
        return B(-self.val, self.err)

    def __sub__(self, o):
        return self + (-o if isinstance(o, B) else -torch.as_tensor(o, dtype=torch.float64))

    def __mul__(self, o):
        o = o if isinstance(o, B) else B(torch.as_tensor(o, dtype=torch.float64))
        return self._new(self.val * o.val, self.val.abs() * o.err + o.val.abs() * self.err + self.err * o.err)

    __radd__, __rmul__ = __add__, __mul__

    def sum(self, dim, keepdim=False):
        dims = dim if isinstance(dim, tuple) else (dim,)
        n = int(np.prod([self.val.shape[d] for d in dims]))
        return B(self.val.sum(dim, keepdim=keepdim),
                 (self.err + n * EPS * self.val.abs()).sum(dim, keepdim=keepdim))

    def mean(self, dim, keepdim=False):
        dims = dim if isinstance(dim, tuple) else (dim,)
        return self.sum(dim, keepdim) * (1.0 / int(np.prod([self.val.shape[d] for d in dims])))

    def rsqrt(self):
        v = self.val.rsqrt()
        rel = self.err / self.val          # |d v| <= v (rel / 2) (1 - rel)^-3/2, plus sqrt and division
        return B(v, v * (rel / 2 * (1 - rel).clamp(min=0.1) ** -1.5 + 4 * EPS))

    def recip(self):
        v = 1.0 / self.val
        return B(v, v.abs() * (self.err / self.val.abs() / (1 - (self.err / self.val.abs()).clamp(max=0.5)) + 2 * EPS))

    def exp(self):
        """The argument is scaled to a power of two's in float32 (its rounding counts |x| EPS), then two units."""
        v = self.val.exp()
        return B(v, v * torch.expm1(self.err + (2 * self.val.abs() + 4) * EPS))

    def __getitem__(self, i):
        return B(self.val[i], self.err[i])

    def view(self, *s):
        return B(self.val.reshape(*s), self.err.reshape(*s))

    def expand(self, *s):
        return B(self.val.expand(*s), self.err.expand(*s))

    def where(self, cond, other=0.0):
        return B(torch.where(cond, self.val, torch.as_tensor(other, dtype=torch.float64)),
                 torch.where(cond, self.err, torch.zeros((), dtype=torch.float64)))

    def rounded(self, dtype):
        """Stored in ``dtype``: half a step of the value (float32 results were rounded already), and half the
        smallest step where the value is below the type's normal numbers."""
        f = torch.finfo(dtype)
        step = 0.0 if dtype == torch.float32 else f.eps / 2
        tiny = f.tiny * f.eps / 2
        return B(self.val, self.err + step * (self.val.abs() + self.err) + tiny)


def within(got, ref, what=""):
    """``got`` (any float tensor) is within the bound of ``ref`` (B); equal where the reference is not finite."""
    g = got.detach().double().cpu()
    assert g.shape == ref.val.shape, (what, g.shape, ref.val.shape)
    fine = torch.isfinite(ref.val)
    assert torch.equal(torch.isfinite(g), fine), f"{what}: other places are not finite"
    off = (g - ref.val).abs()[fine] - ref.err[fine]
    if off.numel():
        assert float(off.max()) <= 0.0, (f"{what}: off the bound by {float(off.max()):.3e}, "
                                         f"largest value {float(ref.val[fine].abs().max()):.3e}")


# ------------------------------------------------------------------------------------------------ draws
def philox(seed, call, step, q):
    """Words [len(q), 4] of the blocks q (Philox4x32-10, Salmon et al. 2011)."""
    M = np.uint64(0xFFFFFFFF)
    q = np.asarray(q, np.uint64)
    ctr = [q & M, q >> np.uint64(32), np.full_like(q, call), np.full_like(q, step % 2 ** 32)]
    k0, k1 = seed % 2 ** 32, (seed >> 32) % 2 ** 32
    return philox_words(ctr, k0, k1)


def philox_words(ctr, k0, k1):
    M = np.uint64(0xFFFFFFFF)
    for i in range(10):
        lo, hi = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(hi >> np.uint64(32)) ^ ctr[1] ^ np.uint64((k0 + i * 0x9E3779B9) % 2 ** 32), hi & M,
               (lo >> np.uint64(32)) ^ ctr[3] ^ np.uint64((k1 + i * 0xBB67AE85) % 2 ** 32), lo & M]
    return np.stack(ctr, 1)


def threshold(p):
    return int(65536 * p + 0.5)


def keep_scale(p):
    return 65536.0 / (65536.0 - threshold(p))


def keep(seed, call, step, draws, p):
    """Boolean keep of the draws (any integer tensor)."""
    d = np.asarray(draws, np.uint64).reshape(-1)
    w = philox(seed % 2 ** 64, call, step, d >> np.uint64(3))
    j = (d % np.uint64(8)).astype(np.int64)
    half = (w[np.arange(len(d)), j // 2] >> (np.uint64(16) * (j % 2).astype(np.uint64))) & np.uint64(0xFFFF)
    return torch.from_numpy(half >= threshold(p)).reshape(np.shape(draws))


def pad8(n):
    return (n + 7) // 8 * 8


def dropout_keep(shape, per, group, seed, call, step, p):
    if per == "element":
        return keep(seed, call, step, np.arange(int(np.prod(shape))).reshape(shape), p)
    n = shape[0]
    if per == "group":
        k = keep(seed, call, step, np.arange(n) // group, p)
    else:
        k = keep(seed, call, step, np.arange(n)[:, None] * pad8(shape[-1]) + np.arange(shape[-1])[None], p)
        return k.view(n, *(1,) * (len(shape) - 2), shape[-1]).expand(shape)
    return k.view(n, *(1,) * (len(shape) - 1)).expand(shape)


def dropout(x, k, p):
    """x [...] (torch), keep mask k -> B; the factor itself is rounded to float32."""
    s = B(torch.tensor(keep_scale(p))) if p else B(torch.tensor(1.0))
    s.err = EPS * s.val
    return (B(torch.where(k, x.double(), 0.0)) * s).rounded(x.dtype)


# ------------------------------------------------------------------------------------------------ norms
def _norm(u, kind, eps):
    if kind == "layer":
        u = u - u.mean(-1, True)
    r = ((u * u).mean(-1, True) + eps).rsqrt()
    return u * r, r


def _norm_back(g, xhat, r, kind):
    t = g - xhat * (g * xhat).mean(-1, True)
    if kind == "layer":
        t = t - g.mean(-1, True)
    return t * r


def residual_norm(x, y, gate, post, pre, kind, eps, scale, k, p, dh=None, dz=None):
    """x, y [R, C]; gate [G, C] or None; post / pre (w, b or None) or None; k [R, C] boolean.  Returns a dict of B
    (h, z, and with dh / dz the gradients dx, dy, dgate, dpost_w, ..)."""
    R, C = x.shape
    f32 = lambda v: torch.tensor(float(v))                                                # noqa: E731
    drop = B(torch.tensor(keep_scale(p) if p else 1.0), torch.tensor(EPS * 2)) * B(f32(scale), torch.tensor(EPS * abs(scale)))
    xb, yb = B(x), B(y)
    u = yb
    if post is not None:
        yhat, ry = _norm(yb, kind, eps)
        u = yhat * B(post[0])
        if post[1] is not None:
            u = u + B(post[1])
    gb = None
    if gate is not None:
        gb = B(gate.double().repeat_interleave(R // gate.shape[0], 0))
    h = xb + ((u if gb is None else u * gb) * drop).where(k)
    out = {"h": h.rounded(x.dtype)}
    if pre is not None:
        hhat, rh = _norm(h, kind, eps)
        z = hhat * B(pre[0])
        if pre[1] is not None:
            z = z + B(pre[1])
        out["z"] = z.rounded(y.dtype)
    if dh is None and dz is None:
        return out
    t = B(dh) if dh is not None else B(torch.zeros(R, C))
    if pre is not None:
        dzb = B(dz) if dz is not None else B(torch.zeros(R, C))
        t = t + _norm_back(dzb * B(pre[0]), hhat, rh, kind)
        out["dpre_w"], out["dpre_b"] = (dzb * hhat).sum(0), dzb.sum(0)
    out["dx"] = t.rounded(x.dtype)
    du = (t * drop).where(k)
    if gate is not None:
        out["dgate"] = (du * u).where(k).view(gate.shape[0], R // gate.shape[0], C).sum(1)
        du = du * gb
    if post is not None:
        out["dpost_w"], out["dpost_b"] = (du * yhat).sum(0), du.sum(0)
        du = _norm_back(du * B(post[0]), yhat, ry, kind)
    out["dy"] = du.rounded(y.dtype)
    params = [t for t in ((gate,) + (post or ()) + (pre or ())) if t is not None]
    for n in ("dgate", "dpost_w", "dpost_b", "dpre_w", "dpre_b"):
        if n in out:
            out[n] = out[n].rounded(params[0].dtype)
    return out


def sh_residual_norm(x, y, w, b, eps, k, factor, dh=None, dz=None):
    """x, y [V, (L+1)^2, C]; k boolean of that shape, factor the product of the scales.  Dict of B."""
    V, S, C = x.shape
    L = round(S ** 0.5) - 1
    deg = torch.tensor([l for l in range(L + 1) for _ in range(2 * l + 1)])
    bal = B((1.0 / ((2 * deg + 1) * (L + 1)).double())[:, None])
    bal.err = EPS * bal.val.abs()
    first = (torch.arange(S) == 0)[:, None]
    f = B(torch.tensor(factor), torch.tensor(3 * EPS * factor))
    wd = B(w.double()[deg])
    h = B(x) + (B(torch.where(k, y.double(), 0.0)) * f)
    m0 = h[:, :1].mean(-1, True)
    hc = h - B(torch.where(first, m0.val, 0.0), torch.where(first, m0.err, 0.0))
    r = ((hc * hc * bal).sum((1, 2), True) * (1.0 / C) + eps).rsqrt()
    z = hc * r * wd + B(torch.where(first, b.double(), 0.0))
    out = {"h": h.rounded(x.dtype), "z": z.rounded(x.dtype)}
    if dh is None and dz is None:
        return out
    dzb = B(dz) if dz is not None else B(torch.zeros(V, S, C))
    g = dzb * wd
    coef = (g * hc).sum((1, 2), True) * r * r * r * (1.0 / C)
    t = g * r - hc * bal * coef
    # the mean of the l = 0 row of t: the centred row's share is 0 up to its rounding
    m = t[:, :1].mean(-1, True)
    t = t - B(torch.where(first, m.val, 0.0), torch.where(first, m.err, 0.0))
    if dh is not None:
        t = t + B(dh)
    out["dx"] = t.rounded(x.dtype)
    out["dy"] = (t * f).where(k).rounded(y.dtype)
    rows = (dzb * hc * r).sum(0)
    out["dw"] = B(torch.zeros(L + 1, C, dtype=torch.float64).index_add_(0, deg, rows.val),
                  torch.zeros(L + 1, C, dtype=torch.float64).index_add_(0, deg, rows.err + 13 * EPS * rows.val.abs())).rounded(w.dtype)
    out["db"] = dzb[:, 0].sum(0).rounded(b.dtype)
    return out


def segment_attention(values, logits, ptr, eid, k, p, dout=None):
    """values [E, K, H, D], logits [E, H], lists eid[ptr[v] : ptr[v + 1]]; k [E, H] boolean.  Dict of B."""
    E, K, H, D = values.shape
    V = len(ptr) - 1
    drop = B(torch.tensor(keep_scale(p) if p else 1.0), torch.tensor(EPS * 2 if p else 0.0))
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)                                   # noqa: E731
    out = B(z(V, K, H, D), z(V, K, H, D))
    dv, dl = B(z(E, K, H, D), z(E, K, H, D)), B(z(E, H), z(E, H))
    l = logits.double()
    for v in range(V):
        es = eid[ptr[v]:ptr[v + 1]].long()
        for h in range(H):
            live = es[l[es, h] > -np.inf]
            if not len(live):
                continue
            top = l[live, h].max()
            e = B(l[live, h] - top, EPS * (l[live, h] - top).abs()).exp()
            # weights below the float32 range flush to 0
            e = B(e.val, e.err + 2.0 ** -126)
            # joined parts scale their sums by two more exponentials of differences up to the spread
            spread = float((top - l[live, h].min()).clamp(max=100.0))
            s = e.sum(0)
            s.err = s.err + s.val * EPS * (4 * spread + 16)
            a = e * s.recip()
            a.err = a.err + a.val * EPS * (4 * spread + 16)
            kk = k[live, h]
            w = (a * drop).where(kk)
            val = B(torch.where(kk[:, None, None], values[live, :, h].double(), 0.0))
            o = (w.view(-1, 1, 1) * val).sum(0)
            out.val[v, :, h], out.err[v, :, h] = o.val, o.err
            if dout is not None:
                d = B(dout[v, :, h].double())
                g = w.view(-1, 1, 1) * d[None]
                dv.val[live, :, h], dv.err[live, :, h] = g.val, g.err
                dp = ((val * d[None]).view(len(live), -1).sum(1) * drop).where(kk)
                delta = (a * dp).sum(0)
                t = a * (dp - delta)
                dl.val[live, h], dl.err[live, h] = t.val, t.err
    got = {"out": out.rounded(values.dtype)}
    if dout is not None:
        got["dvalues"], got["dlogits"] = dv.rounded(values.dtype), dl.rounded(logits.dtype)
    return got
