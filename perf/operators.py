"""What the operators around a training block's products are measured on (block_ops.py): dropout whose mask
is never stored, the residual add with its norms and gate, the same with the spherical-harmonics norm, and
attention over the incoming edges of a node.

``own = False``: the plain form of each, elementary torch operations in 32 bits, rounded once at the end.
``own = True``: the calls a user makes.  Every case with ``train`` is a forward and its backward pass.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


# ------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the attention weights of EquiformerV2's training batch (64 systems of 5 bodies, 4 heads): the smallest
        # dropout a step makes, one of many, where the launch is the cost
        dict(name="dropout_attention_weights", op="dropout", per="element", n=1280, S=1, C=4, group=1, p=0.1,
             dtype="f32", train=True),
        # stochastic depth on the constructor's default widths (lmax 6, 128 channels), one draw a system of 5
        dict(name="dropout_path_lmax6", op="dropout", per="group", n=1280, S=49, C=128, group=5, p=0.05,
             dtype="f32", train=True),
        # channel dropout of the same features with an odd number of channels and nodes
        dict(name="dropout_channel_odd", op="dropout", per="channel", n=2047, S=9, C=61, group=1, p=0.2,
             dtype="f16", train=True),
        # hidden activations of a wide feed-forward layer in 16 bits: the largest dropout
        dict(name="dropout_hidden_bf16", op="dropout", per="element", n=8192, S=1, C=4096, group=1, p=0.1,
             dtype="bf16", train=True),
        # one system's nodes in a rollout step (5 bodies x 20 orientations): latency of a serving call
        dict(name="residual_one_system", op="residual", rows=100, C=128, norm="layer", post=False, pre=True, gate=1,
             p=0.0, group=0, scale=1.0, x="f32", y="f32", param="f32", bias=True, train=False),
        # the tail of PONITA's ConvNext block at its training batch: layer scale and residual, no norm
        dict(name="residual_layer_scale", op="residual", rows=6400, C=128, norm="layer", post=False, pre=False,
             gate=1, p=0.0, group=0, scale=1.0, x="f32", y="f32", param="f32", bias=False, train=True),
        # a 16-bit block over an fp32 residual stream, odd sizes, stochastic depth, a gate of its own for every row
        dict(name="residual_mixed_odd", op="residual", rows=2049, C=999, norm="layer", post=True, pre=True, gate=2049,
             p=0.1, group=3, scale=0.5, x="f32", y="f16", param="f32", bias=True, train=True),
        # a wide 16-bit block: norms before and after, a gate for each system, dropout of every element
        dict(name="residual_block_bf16", op="residual", rows=16384, C=2048, norm="rms", post=True, pre=True, gate=64,
             p=0.1, group=0, scale=0.7, x="bf16", y="bf16", param="bf16", bias=False, train=True),
        # EquiformerV2's training configuration (64 channels, lmax 2, 64 systems of 5)
        dict(name="sh_residual_lmax2", op="sh", nodes=320, lmax=2, C=64, path_p=0.05, path_group=5, channel_p=0.0,
             dtype="f32", train=True),
        # the constructor's default widths on a batch of 512 systems, with both dropouts
        dict(name="sh_residual_lmax6", op="sh", nodes=2560, lmax=6, C=128, path_p=0.05, path_group=5, channel_p=0.1,
             dtype="f32", train=True),
        # the graph attention at the constructor's default widths: 5 bodies, fully connected, 128 systems
        dict(name="attention_lmax6", op="attention", nodes=640, edges=2560, K=49, H=8, D=16, p=0.1, graph="full",
             masked=0.0, dtype="f32", logits="f32", train=True),
        # few destinations with long ragged lists of edges, some empty, some edges masked, in 16 bits
        dict(name="attention_long_ragged", op="attention", nodes=96, edges=60000, K=1, H=8, D=64, p=0.1,
             graph="ragged", masked=0.05, dtype="bf16", logits="f32", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["dropout", "residual", "sh", "attention"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.75
    if op == "dropout":
        per = rng.choice(["element", "group", "channel"])
        S, C = (1 if per == "element" else _log(rng, 1, 49)), _log(rng, 1, 4096)
        n = max(1, min(_log(rng, 1, 20000), (1 << 24) // (S * C)))
        return dict(op=op, per=per, n=n, S=S, C=C, group=_log(rng, 1, 64), p=rng.choice([0.05, 0.1, 0.5]),
                    dtype=dtype, train=train)
    if op == "residual":
        C = _log(rng, 8, 8192)
        rows = max(1, min(_log(rng, 1, 30000), (1 << 24) // C))
        rows, gate = rng.choice([(rows, 0), (rows, 1), (rows, rows), (-(-rows // 7) * 7, -(-rows // 7))])
        x = rng.choice([dtype, "f32"])
        p = rng.choice([0.0, 0.1, 0.3])
        return dict(op=op, rows=rows, C=C, norm=rng.choice(["layer", "rms"]), post=rng.random() < 0.5,
                    pre=rng.random() < 0.8, gate=gate, p=p, group=rng.choice([0, 0, 1, 5]) if p else 0,
                    scale=rng.choice([1.0, 0.5]), x=x, y=dtype, param="f32" if x == "f32" else dtype,
                    bias=rng.random() < 0.5, train=train)
    if op == "sh":
        lmax, C = rng.randint(0, 6), _log(rng, 8, 256)
        nodes = max(1, min(_log(rng, 5, 20000), (1 << 23) // ((lmax + 1) ** 2 * C)))
        return dict(op=op, nodes=nodes, lmax=lmax, C=C, path_p=rng.choice([0.0, 0.05]), path_group=_log(rng, 1, 20),
                    channel_p=rng.choice([0.0, 0.1]), dtype=dtype, train=train)
    graph = rng.choice(["full", "ragged"])
    K, H, D = rng.choice([1, 1, 9, 25]), rng.choice([1, 2, 4, 5, 8]), rng.choice([4, 7, 16, 64])
    if graph == "full":
        N = rng.choice([2, 5, 20, 33])
        B = max(1, min(_log(rng, 1, 2000), (1 << 22) // (N * (N - 1) * K * H * D)))
        nodes, edges = B * N, B * N * (N - 1)
    else:
        nodes = _log(rng, 1, 3000)
        edges = max(1, min(_log(rng, 8, 60000), (1 << 22) // (K * H * D)))
    return dict(op=op, nodes=nodes, edges=edges, K=K, H=H, D=D, p=rng.choice([0.0, 0.1]), graph=graph,
                masked=rng.choice([0.0, 0.05]), dtype=dtype, logits=rng.choice([dtype, "f32"]), train=train)


def work(case):
    c = case
    if c["op"] == "dropout":
        n = c["n"] * c["S"] * c["C"]
        return {"bytes": n * _BYTES[c["dtype"]] * (4 if c["train"] else 2), "flops": n * (2 if c["train"] else 1)}
    if c["op"] == "residual":
        n, bx, by, bp = c["rows"] * c["C"], _BYTES[c["x"]], _BYTES[c["y"]], _BYTES[c["param"]]
        par = (c["gate"] + (int(c["post"]) + int(c["pre"])) * (2 if c["bias"] else 1)) * c["C"] * bp
        fwd = n * (2 * bx + by + (by if c["pre"] else 0)) + par          # x, y, h and z
        bwd = n * (2 * bx + by + (by if c["pre"] else 0)) + par          # dh, dx, dy and dz
        return {"bytes": fwd + (bwd if c["train"] else 0), "flops": n * (40 if c["train"] else 15)}
    if c["op"] == "sh":
        n = c["nodes"] * (c["lmax"] + 1) ** 2 * c["C"]
        return {"bytes": n * _BYTES[c["dtype"]] * (8 if c["train"] else 4), "flops": n * (35 if c["train"] else 12)}
    row, b = c["K"] * c["H"] * c["D"], _BYTES[c["dtype"]]
    lg = c["edges"] * c["H"] * _BYTES[c["logits"]]
    fwd = (c["edges"] + c["nodes"]) * row * b + lg
    return {"bytes": fwd * (2 if c["train"] else 1), "flops": c["edges"] * row * (5 if c["train"] else 2)}


# ------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device=dev, generator=g)                                       # noqa: E731
    leaf = lambda t, dt: t.to(_DTYPES[dt]).requires_grad_(c["train"])                                # noqa: E731
    # the generator's state as a program keeps it: the seed and the number of the step
    st = {"case": c, "rng": torch.tensor([seed * 2654435761 + 12345, seed % 1000], device=dev, dtype=torch.int64),
          "call": 3}
    if c["op"] == "dropout":
        shape = (c["n"], c["C"]) if c["S"] == 1 and c["per"] == "element" else (c["n"], c["S"], c["C"])
        st["x"] = leaf(rand(*shape), c["dtype"])
        st["dy"] = rand(*shape).to(_DTYPES[c["dtype"]])
    elif c["op"] == "residual":
        R, C = c["rows"], c["C"]
        wide = torch.exp(0.5 * rand(C))                       # a residual stream's channels differ in size
        st["x"], st["y"] = leaf(rand(R, C) * wide, c["x"]), leaf(rand(R, C), c["y"])
        st["gate"] = leaf(0.5 + 0.3 * rand(c["gate"], C), c["param"]) if c["gate"] else None
        for k in ("post", "pre"):
            st[k + "_w"] = leaf(1.0 + 0.2 * rand(C), c["param"]) if c[k] else None
            st[k + "_b"] = leaf(0.2 * rand(C), c["param"]) if c[k] and c["bias"] else None
        st["dh"], st["dz"] = rand(R, C).to(_DTYPES[c["x"]]), rand(R, C).to(_DTYPES[c["y"]])
    elif c["op"] == "sh":
        shape = (c["nodes"], (c["lmax"] + 1) ** 2, c["C"])
        st["x"], st["y"] = leaf(rand(*shape), c["dtype"]), leaf(rand(*shape), c["dtype"])
        st["w"], st["b"] = leaf(1.0 + 0.2 * rand(c["lmax"] + 1, c["C"]), c["dtype"]), leaf(0.2 * rand(c["C"]), c["dtype"])
        st["dh"], st["dz"] = rand(*shape).to(_DTYPES[c["dtype"]]), rand(*shape).to(_DTYPES[c["dtype"]])
    else:
        V, E = c["nodes"], c["edges"]
        if c["graph"] == "full":     # the fully connected graph, edges by source as the graph builder lists them
            N = E // V + 1
            i = torch.arange(V, device=dev)
            j = torch.arange(N - 1, device=dev)
            dst = ((i // N * N)[:, None] + j + (j >= (i % N)[:, None])).reshape(-1)
        else:                        # lists of very different lengths, every seventh empty
            u = torch.rand(E, device=dev, generator=g)
            dst = (V * u * u).long().clamp_(max=V - 1)
            dst = torch.where((dst % 7 == 3) & (dst > 0), dst - 1, dst)
        order = torch.argsort(dst, stable=True)
        st["dst"] = dst
        st["ptr"] = torch.searchsorted(dst[order].contiguous(), torch.arange(V + 1, device=dev)).to(torch.int32)
        st["eid"] = order.to(torch.int32)
        st["values"] = leaf(rand(E, c["K"], c["H"], c["D"]), c["dtype"])
        lg = 2.0 * rand(E, c["H"])
        if c["masked"]:
            lg = lg.masked_fill(torch.rand(E, c["H"], device=dev, generator=g) < c["masked"], -math.inf)
        st["logits"] = leaf(lg, c["logits"])
        st["dout"] = rand(V, c["K"], c["H"], c["D"]).to(_DTYPES[c["dtype"]])
    return st


# ------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    import nbody_amd  # noqa: F401  (registers the package)
    from nbody_amd import block_ops as B
    c, rng, call = s["case"], s["rng"], s["call"]
    if c["op"] == "dropout":
        y = B.dropout(s["x"], c["p"], rng, call=call, per=c["per"], group=c["group"])
        outs, ins, grads = {"y": y}, {"dx": s["x"]}, (s.get("dy"),)
    elif c["op"] == "residual":
        post = (s["post_w"], s["post_b"]) if c["post"] else None
        pre = (s["pre_w"], s["pre_b"]) if c["pre"] else None
        h, z = B.residual_norm(s["x"], s["y"], gate=s["gate"], scale=c["scale"], post=post, pre=pre, norm=c["norm"],
                               eps=EPS, p=c["p"], group=c["group"], rng=rng, call=call)
        outs = {"h": h, "z": z} if c["pre"] else {"h": h}
        ins = {"dx": s["x"], "dy": s["y"]}
        ins.update({"d" + k: s[k] for k in ("gate", "post_w", "post_b", "pre_w", "pre_b") if s[k] is not None})
        grads = (s["dh"], s["dz"]) if c["pre"] else (s["dh"],)
    elif c["op"] == "sh":
        h, z = B.sh_residual_norm(s["x"], s["y"], s["w"], s["b"], eps=EPS, path_p=c["path_p"],
                                  path_group=c["path_group"], channel_p=c["channel_p"], rng=rng, call=call)
        outs, ins, grads = {"h": h, "z": z}, {"dx": s["x"], "dy": s["y"], "dw": s["w"], "db": s["b"]}, (s["dh"], s["dz"])
    else:
        out = B.segment_attention(s["values"], s["logits"], s["ptr"], s["eid"], p=c["p"], rng=rng, call=call)
        outs, ins, grads = {"out": out}, {"dvalues": s["values"], "dlogits": s["logits"]}, (s["dout"],)
    if c["train"]:
        got = torch.autograd.grad(tuple(outs.values()), tuple(ins.values()), grads)
        outs = {k: v.detach() for k, v in outs.items()} | dict(zip(ins, got))
    return outs


# ------------------------------------------------------------------------------------------- the plain forms
def _keep(s, call, n, p):
    """[n] float32: 0 or 1 / (1 - p) for each draw (Philox4x32-10, eight 16-bit draws a block)."""
    M = 0xFFFFFFFF
    seed, step = s["rng"][0], s["rng"][1]
    q = torch.arange((n + 7) // 8, device=s["rng"].device)
    a, b, c, d = q & M, q >> 32, torch.full_like(q, call), (step & M).expand_as(q)
    k, m = seed & M, (seed >> 32) & M
    for _ in range(10):
        x, y = a * 0xD2511F53, c * 0xCD9E8D57
        a, b, c, d = ((y >> 32) & M) ^ b ^ k, y & M, ((x >> 32) & M) ^ d ^ m, x & M
        k, m = (k + 0x9E3779B9) & M, (m + 0xBB67AE85) & M
    w = torch.stack([a, b, c, d], 1)
    T = int(math.floor(65536 * p + 0.5))
    return (torch.stack([w & 0xFFFF, w >> 16], 2).reshape(-1)[:n] >= T).float() * (65536 / (65536 - T))


def _drop(k, x):
    """k x with a dropped place 0 whatever x holds there."""
    return torch.where(k > 0, x * k, torch.zeros((), device=x.device))


def _norm(u, kind):
    if kind == "layer":
        u = u - u.mean(-1, keepdim=True)
    r = torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS)
    return u * r, r


def _norm_back(g, xhat, r, kind):
    t = g - xhat * (g * xhat).mean(-1, keepdim=True)
    if kind == "layer":
        t = t - g.mean(-1, keepdim=True)
    return t * r


def _pad8(n):
    return (n + 7) // 8 * 8


def _plain_dropout(s):
    c, x = s["case"], s["x"].float()
    n, C = c["n"], c["C"]
    if c["per"] == "element":
        k = _keep(s, s["call"], x.numel(), c["p"]).view(x.shape)
    elif c["per"] == "group":
        k = _keep(s, s["call"], -(-n // c["group"]), c["p"])[torch.arange(n, device=x.device) // c["group"], None, None]
    else:
        k = _keep(s, s["call"], n * _pad8(C), c["p"]).view(n, 1, _pad8(C))[:, :, :C]
    dt = s["x"].dtype
    out = {"y": _drop(k, x).to(dt)}
    if c["train"]:
        out["dx"] = _drop(k, s["dy"].float()).to(dt)
    return out


def _plain_residual(s):
    c, x, y = s["case"], s["x"].float(), s["y"].float()
    R, C, kind = c["rows"], c["C"], c["norm"]
    f = {k: (s[k].float() if s[k] is not None else None) for k in ("gate", "post_w", "post_b", "pre_w", "pre_b")}
    k = torch.ones((), device=x.device)
    if c["p"]:
        k = (_keep(s, s["call"], -(-R // c["group"]), c["p"])[torch.arange(R, device=x.device) // c["group"], None]
             if c["group"] else _keep(s, s["call"], R * _pad8(C), c["p"]).view(R, _pad8(C))[:, :C])
    u = y
    if c["post"]:
        yhat, ry = _norm(y, kind)
        u = yhat * f["post_w"] + (f["post_b"] if c["bias"] else 0.0)
    G = c["gate"]
    gate = f["gate"].repeat_interleave(R // G, 0) if G else 1.0
    h = x + c["scale"] * _drop(k, gate * u)
    out = {"h": h.to(s["x"].dtype)}
    if c["pre"]:
        hhat, rh = _norm(h, kind)
        out["z"] = (hhat * f["pre_w"] + (f["pre_b"] if c["bias"] else 0.0)).to(s["y"].dtype)
    if not c["train"]:
        return out
    t = s["dh"].float()
    par = {}
    if c["pre"]:
        dz = s["dz"].float()
        t = t + _norm_back(dz * f["pre_w"], hhat, rh, kind)
        par["dpre_w"], par["dpre_b"] = (dz * hhat).sum(0), dz.sum(0)
    du = c["scale"] * _drop(k, t)
    dn = du * gate
    if G:
        par["dgate"] = (du * u).view(G, R // G, C).sum(1)
    dy = dn
    if c["post"]:
        par["dpost_w"], par["dpost_b"] = (dn * yhat).sum(0), dn.sum(0)
        dy = _norm_back(dn * f["post_w"], yhat, ry, kind)
    out["dx"], out["dy"] = t.to(s["x"].dtype), dy.to(s["y"].dtype)
    for name in ("gate", "post_w", "post_b", "pre_w", "pre_b"):
        if s[name] is not None:
            out["d" + name] = par["d" + name].to(s[name].dtype)
    return out


def _plain_sh(s):
    c, x, y, w, b = s["case"], s["x"].float(), s["y"].float(), s["w"].float(), s["b"].float()
    V, L, C, dev, dt = c["nodes"], c["lmax"], c["C"], s["x"].device, s["x"].dtype
    deg = torch.arange(L + 1, device=dev).repeat_interleave(2 * torch.arange(L + 1, device=dev) + 1)
    bal = (1.0 / ((2 * deg + 1) * (L + 1)).float())[:, None]
    first = (torch.arange((L + 1) ** 2, device=dev) == 0).float()[:, None]
    k = torch.ones((), device=dev)
    if c["path_p"]:
        k = k * _keep(s, s["call"], -(-V // c["path_group"]), c["path_p"])[
            torch.arange(V, device=dev) // c["path_group"], None, None]
    if c["channel_p"]:
        k = k * _keep(s, s["call"] + 1, V * _pad8(C), c["channel_p"]).view(V, 1, _pad8(C))[:, :, :C]
    h = x + _drop(k, y)
    hc = h - first * h[:, :1].mean(-1, keepdim=True)
    r = torch.rsqrt((bal * hc * hc).sum((1, 2), keepdim=True) / C + EPS)
    out = {"h": h.to(dt), "z": (hc * r * w[deg] + first * b).to(dt)}
    if c["train"]:
        dz = s["dz"].float()
        g = dz * w[deg]
        t = r * g - bal * hc * (r ** 3 / C * (g * hc).sum((1, 2), keepdim=True))
        t = s["dh"].float() + t - first * t[:, :1].mean(-1, keepdim=True)
        rows = (dz * hc * r).sum(0)
        dw = torch.zeros(L + 1, C, device=dev).index_add_(0, deg, rows)
        out.update(dx=t.to(dt), dy=_drop(k, t).to(dt), dw=dw.to(dt), db=dz[:, 0].sum(0).to(dt))
    return out


def _plain_attention(s):
    c, v, l, dst = s["case"], s["values"].float(), s["logits"].float(), s["dst"]
    V, E, H = c["nodes"], c["edges"], c["H"]
    m = torch.full((V, H), -math.inf, device=v.device).scatter_reduce_(0, dst[:, None].expand(E, H), l, "amax")
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(l - m[dst])
    a = e / (torch.zeros(V, H, device=v.device).index_add_(0, dst, e) + 1e-16)[dst]
    a = torch.where(l == -math.inf, torch.zeros_like(a), a)
    k = _keep(s, s["call"], E * H, c["p"]).view(E, H) if c["p"] else torch.ones_like(a)
    w = (a * k)[:, None, :, None]
    out = torch.zeros(V, *v.shape[1:], device=v.device).index_add_(0, dst, _drop(w, v))
    got = {"out": out.to(s["values"].dtype)}
    if c["train"]:
        d = s["dout"].float()[dst]
        dp = _drop(a * k > 0, (d * v).sum((1, 3))) * k
        delta = torch.zeros(V, H, device=v.device).index_add_(0, dst, a * dp)
        got["dvalues"] = (w * d).to(s["values"].dtype)
        got["dlogits"] = (a * (dp - delta[dst])).to(s["logits"].dtype)
    return got


_PLAIN = {"dropout": _plain_dropout, "residual": _plain_residual, "sh": _plain_sh, "attention": _plain_attention}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------- in 64 bits
def _keep64(s, call, n, p):
    """The draws' factors from the generator's definition in numpy's unsigned integers."""
    seed, step = (int(t) % (1 << 64) for t in s["rng"].cpu())
    M = np.uint64(0xFFFFFFFF)
    ctr = np.zeros((4, (n + 7) // 8), np.uint64)
    q = np.arange(ctr.shape[1], dtype=np.uint64)
    ctr[0], ctr[1], ctr[2], ctr[3] = q & M, q >> np.uint64(32), call, step % (1 << 32)
    for i in range(10):
        k0, k1 = np.uint64((seed + i * 0x9E3779B9) % (1 << 32)), np.uint64(((seed >> 32) + i * 0xBB67AE85) % (1 << 32))
        lo, hi = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = np.stack([(hi >> np.uint64(32)) ^ ctr[1] ^ k0, hi & M, (lo >> np.uint64(32)) ^ ctr[3] ^ k1, lo & M])
    half = np.ascontiguousarray(ctr.T.astype("<u4")).view("<u2").reshape(-1)[:n]
    T = int(65536 * p + 0.5)
    return torch.from_numpy(np.where(half >= T, 65536.0 / (65536 - T), 0.0)).to(s["rng"].device)


def exact(case, seed):
    """The operators' definitions in 64 bits; gradients by differentiating them automatically."""
    c, s = case, prepare(case, seed)
    D = lambda t: None if t is None else t.detach().double().requires_grad_(c["train"])              # noqa: E731
    if c["op"] == "dropout":
        x, n, C = D(s["x"]), c["n"], c["C"]
        x3 = x.reshape(n, -1, C)
        if c["per"] == "element":
            k = _keep64(s, s["call"], x.numel(), c["p"]).view(x3.shape)
        elif c["per"] == "group":
            k = _keep64(s, s["call"], (n - 1) // c["group"] + 1, c["p"]).repeat_interleave(c["group"])[:n].view(n, 1, 1)
        else:
            k = _keep64(s, s["call"], n * _pad8(C), c["p"]).view(n, 1, -1)[..., :C]
        outs, ins, gs = {"y": (x3 * k).view(x.shape)}, {"dx": x}, [s["dy"]]
    elif c["op"] == "residual":
        R, C = c["rows"], c["C"]
        x, y = D(s["x"]), D(s["y"])
        par = {k: D(s[k]) for k in ("gate", "post_w", "post_b", "pre_w", "pre_b")}

        def norm(u, which):
            var, mean = torch.var_mean(u, -1, correction=0, keepdim=True)
            u = (u - mean) / (var + EPS).sqrt() if c["norm"] == "layer" else u / (u.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
            u = u * par[which + "_w"]
            return u if par[which + "_b"] is None else u + par[which + "_b"]

        u = norm(y, "post") if c["post"] else y
        if c["gate"]:
            u = (u.view(c["gate"], -1, C) * par["gate"][:, None]).reshape(R, C)
        if c["p"] and c["group"]:
            u = u * _keep64(s, s["call"], (R - 1) // c["group"] + 1, c["p"]).repeat_interleave(c["group"])[:R, None]
        elif c["p"]:
            u = u * _keep64(s, s["call"], R * _pad8(C), c["p"]).view(R, -1)[:, :C]
        h = x + c["scale"] * u
        outs, gs = {"h": h}, [s["dh"]]
        if c["pre"]:
            outs["z"], gs = norm(h, "pre"), [s["dh"], s["dz"]]
        ins = {"dx": x, "dy": y} | {"d" + k: t for k, t in par.items() if t is not None}
    elif c["op"] == "sh":
        V, L, C = c["nodes"], c["lmax"], c["C"]
        x, y, w, b = D(s["x"]), D(s["y"]), D(s["w"]), D(s["b"])
        u = y
        if c["path_p"]:
            k = _keep64(s, s["call"], (V - 1) // c["path_group"] + 1, c["path_p"])
            u = u * k.repeat_interleave(c["path_group"])[:V, None, None]
        if c["channel_p"]:
            u = u * _keep64(s, s["call"] + 1, V * _pad8(C), c["channel_p"]).view(V, 1, -1)[..., :C]
        h = x + u
        parts = [p - p.mean(-1, keepdim=True) if i == 0 else p
                 for i, p in enumerate(h.split([2 * i + 1 for i in range(L + 1)], 1))]
        n = sum(p.pow(2).mean(1).mean(-1) for p in parts) / (L + 1)
        z = torch.cat([p * w[i] for i, p in enumerate(parts)], 1) / (n + EPS).sqrt()[:, None, None]
        z = torch.cat([z[:, :1] + b, z[:, 1:]], 1)
        outs, ins, gs = {"h": h, "z": z}, {"dx": x, "dy": y, "dw": w, "db": b}, [s["dh"], s["dz"]]
    else:
        v, lg = D(s["values"]), D(s["logits"])
        k = (_keep64(s, s["call"], c["edges"] * c["H"], c["p"]) if c["p"]
             else torch.ones(c["edges"] * c["H"], device=v.device, dtype=torch.float64))
        at = torch.nonzero(torch.isfinite(lg.detach()).reshape(-1))[:, 0]      # the (edge, head) pairs that count
        seg = s["dst"][at // c["H"]] * c["H"] + at % c["H"]
        l1 = lg.reshape(-1)[at]
        top = torch.full((c["nodes"] * c["H"],), -math.inf, device=v.device, dtype=torch.float64)
        top = top.scatter_reduce(0, seg, l1.detach(), "amax")
        e = torch.exp(l1 - top[seg])
        a = e / torch.zeros_like(top).index_add(0, seg, e)[seg]
        vh = v.transpose(1, 2).reshape(c["edges"] * c["H"], c["K"] * c["D"])
        out = torch.zeros(c["nodes"] * c["H"], c["K"] * c["D"], device=v.device, dtype=torch.float64)
        out = out.index_add(0, seg, (a * k[at])[:, None] * vh[at])
        out = out.view(c["nodes"], c["H"], c["K"], c["D"]).transpose(1, 2)
        outs, ins, gs = {"out": out}, {"dvalues": v, "dlogits": lg}, [s["dout"]]
    if c["train"]:
        got = torch.autograd.grad(tuple(outs.values()), tuple(ins.values()), [t.double() for t in gs])
        outs = {k: t.detach() for k, t in outs.items()} | dict(zip(ins, got))
    return outs
