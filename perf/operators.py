"""Workloads of the operators around the experts of a mixture-of-experts block, with their plain forms.

Three operators, each as a user's program calls it (``terrace.ops``):

``sort_back``   tokens to expert order and back: ``expert_sort`` and ``expert_unsort``, forward, or forward and backward
``w4``          the experts' products for a few rows each: ``expert_linear_w4`` on 4-bit weights with group scales
``block_norm``  what stands between two blocks: the norm after a block, its gate and scale, the residual sum, and the
                norm before the next block; forward, or forward and backward

``own`` chooses between the plain form (elementary torch operations in 32 bits) and the framework's kernels.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6


def _ops():
    package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "terracemoe-simulator_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    import terrace.ops
    return terrace.ops


# ---- the cases ----------------------------------------------------------------------------------------------------
def _sort(T, E, k, H, dtype, train, dead, name=None):
    c = {"op": "sort_back", "T": T, "E": E, "k": k, "H": H, "dtype": dtype, "train": train, "dead": dead}
    return dict(c, name=name) if name else c


def _w4(T, E, k, N, K, group, dtype, swiglu, zeros, name=None):
    c = {"op": "w4", "T": T, "E": E, "k": k, "N": N, "K": K, "group": group, "dtype": dtype, "swiglu": swiglu,
         "zeros": zeros}
    return dict(c, name=name) if name else c


def _norm(T, H, dtype, residual, train, post, gate, pre, name=None):
    c = {"op": "block_norm", "T": T, "H": H, "dtype": dtype, "residual": residual, "train": train, "post": post,
         "gate": gate, "pre": pre}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one token of a decoding step: 8 of 256 experts, 14 KB rows
        _sort(1, 256, 8, 7168, "bf16", False, 0.0, "sort_back one token"),
        # a ragged batch of decoding requests on a rank that holds part of the experts (the others' pairs are -1)
        _sort(61, 128, 8, 4096, "bf16", False, 0.25, "sort_back decode batch"),
        # a training step of the small f32 geometry, forward and backward
        _sort(4096, 64, 4, 1024, "f32", True, 0.0, "sort_back train f32"),
        # a training step at 16384 tokens with 14 KB rows, forward and backward
        _sort(16384, 256, 8, 7168, "bf16", True, 0.0, "sort_back train bf16"),
        # one token through the gate and up projections of its 8 experts, with the activation
        _w4(1, 256, 8, 4096, 7168, 128, "bf16", True, False, "w4 one token gate-up"),
        # a ragged batch through small experts, f16, short groups with zero points
        _w4(13, 64, 4, 1408, 1024, 32, "f16", False, True, "w4 small experts"),
        # a decoding batch of 64 requests through the down projection: most of 256 experts hold a few rows
        _w4(64, 256, 8, 7168, 2048, 128, "bf16", False, False, "w4 batch down"),
        # a larger batch: tens of rows an expert
        _w4(256, 64, 8, 4096, 4096, 64, "bf16", True, True, "w4 large batch"),
        # one token between two blocks
        _norm(1, 7168, "bf16", "bf16", False, True, "channel", True, "block_norm one token"),
        # a ragged batch with an odd width and a 32-bit residual stream, a gate per token
        _norm(203, 1001, "f16", "f32", False, True, "token", True, "block_norm odd width"),
        # training steps
        _norm(4096, 1024, "f32", "f32", True, True, "token", True, "block_norm train f32"),
        _norm(16384, 7168, "bf16", "bf16", True, True, "channel", True, "block_norm train bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sort_back", "w4", "block_norm"])
    if op == "sort_back":
        dtype = rng.choice(["f32", "bf16", "f16"])
        train = rng.random() < 0.5
        E = rng.choice([8, 16, 60, 64, 128, 160, 256])
        k = rng.choice([1, 2, 4, 6, 8])
        H = rng.choice([1, 8, 1, 8]) * _log(rng, 64, 896)
        T = _log(rng, 1, 16384)
        while T * k * H * BYTES[dtype] > 16384 * 8 * 7168 * 2:
            T //= 2
        return _sort(T, E, k, H, dtype, train, rng.choice([0.0, 0.0, 0.1, 0.5]))
    if op == "w4":
        group = rng.choice([32, 64, 128])
        swiglu = rng.random() < 0.5
        K = group * max(1, _log(rng, 256, 7168) // group)
        N = 2 * _log(rng, 96, 3584) if swiglu else _log(rng, 96, 7168)
        E = rng.choice([1, 8, 32, 60, 64])
        T = _log(rng, 1, 256)
        k = min(E, rng.choice([1, 2, 4, 8]))
        while T > 1 and T * k * N * K > 256 * 8 * 4096 * 4096:
            T //= 2
        return _w4(T, E, k, N, K, group, rng.choice(["bf16", "f16"]), swiglu, rng.random() < 0.5)
    dtype = rng.choice(["f32", "bf16", "f16"])
    residual = rng.choice([dtype, "f32"])
    H = rng.choice([1, 8, 8]) * _log(rng, 64, 1024)
    T = _log(rng, 1, 16384)
    while T * H * (BYTES[dtype] + BYTES[residual]) > 16384 * 7168 * 4:
        T //= 2
    post, pre = rng.choice([(True, True), (True, True), (False, True), (True, False)])
    return _norm(T, H, dtype, residual, rng.random() < 0.5, post, rng.choice(["none", "channel", "token"]), pre)


# ---- inputs -------------------------------------------------------------------------------------------------------
def _routing(gen, T, E, k, dead):
    """[T, k] distinct experts per token, unevenly loaded; a share ``dead`` of the pairs is -1 (no expert here)."""
    load = torch.randn(E, generator=gen, device="cuda") * 0.5
    idx = (torch.randn(T, E, generator=gen, device="cuda") + load).topk(k, dim=1).indices
    if dead:
        idx = torch.where(torch.rand(T, k, generator=gen, device="cuda") < dead, -1, idx)
    return idx.contiguous()


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale + shift).to(dtype)

    dt = DTYPES[case["dtype"]]
    if case["op"] == "sort_back":
        T, E, k, H = case["T"], case["E"], case["k"], case["H"]
        d = {"expert_idx": _routing(gen, T, E, k, case["dead"]), "x": normal((T, H), dt), "ye": normal((T * k, H), dt)}
        w = torch.rand((T, k), generator=gen, device="cuda") + 0.1
        d["weights"] = (w / w.sum(1, keepdim=True)).to(dt)
        if case["train"]:
            d["d_rows"], d["dy"] = normal((T * k, H), dt), normal((T, H), dt)
        return d
    if case["op"] == "w4":
        T, E, k, N, K, g = (case[n] for n in ("T", "E", "k", "N", "K", "group"))
        d = {"codes": torch.randint(0, 256, (E, N, K // 2), generator=gen, device="cuda", dtype=torch.uint8),
             "scales": ((torch.rand((E, N, K // g), generator=gen, device="cuda") + 0.5) / (5 * math.sqrt(K))).to(dt)}
        if case["zeros"]:
            d["zeros"] = torch.randint(0, 16, (E, N, K // g), generator=gen, device="cuda", dtype=torch.uint8)
        d["rows"] = normal((T * k, K), dt)
        e = _routing(gen, T, E, k, 0.0).reshape(-1)
        d["tokens_per_expert"] = (e[None, :] == torch.arange(E, device="cuda")[:, None]).sum(1)
        return d
    T, H = case["T"], case["H"]
    rt = DTYPES[case["residual"]]
    d = {"y": normal((T, H), dt, 3.0), "residual": normal((T, H), rt)}
    if case["post"]:
        d["post_weight"] = normal((H,), dt, 0.2, 1.0)
    if case["gate"] != "none":
        d["gate"] = normal((H,) if case["gate"] == "channel" else (T, 1), dt, 0.3, 0.5)
    if case["pre"]:
        d["pre_weight"] = normal((H,), dt, 0.2, 1.0)
    if case["train"]:
        d["dh"] = normal((T, H), rt)
        if case["pre"]:
            d["dn"] = normal((T, H), dt)
    return d


_LEAVES = {"sort_back": ("x", "ye", "weights"), "block_norm": ("y", "residual", "post_weight", "gate", "pre_weight")}
_SCALE = 0.75                     # the residual scale of every block_norm case


def prepare(case, seed):
    d = _inputs(case, seed)
    state = {"case": case, **d}
    if case["op"] == "w4":
        if own:                   # the handle that a serving program lays out once and keeps
            state["weights"] = _ops().w4_pack(d["codes"], d["scales"], d.get("zeros"))
            for name in ("codes", "scales", "zeros"):
                state.pop(name, None)
    elif own and case["train"]:
        for name in _LEAVES[case["op"]]:
            if name in state:
                state[name].requires_grad_(True)
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"sort_back": _own_sort_back, "w4": _own_w4, "block_norm": _own_block_norm}[op](state)
    return {"sort_back": _plain_sort_back, "w4": _plain_w4, "block_norm": _plain_block_norm}[op](state)


def _own_sort_back(s):
    ops, c = _ops(), s["case"]
    rows, plan = ops.expert_sort(s["x"], s["expert_idx"], c["E"])
    y = ops.expert_unsort(s["ye"], s["weights"], plan)
    out = {"rows": rows, "tokens_per_expert": plan.tokens_per_expert, "where": plan.where, "y": y}
    if c["train"]:
        out["dx"], out["dye"], out["dw"] = torch.autograd.grad((rows, y), (s["x"], s["ye"], s["weights"]),
                                                               (s["d_rows"], s["dy"]))
    return out


def _own_w4(s):
    return _ops().expert_linear_w4(s["rows"], s["tokens_per_expert"], s["weights"], swiglu=s["case"]["swiglu"])


def _own_block_norm(s):
    ops, c = _ops(), s["case"]
    h, n = ops.block_norm(s["y"], s["residual"], s.get("post_weight"), s.get("gate"), s.get("pre_weight"),
                          scale=_SCALE, eps=EPS)
    out = {"h": h, "n": n} if c["pre"] else {"h": h}
    if c["train"]:
        names = [n for n in _LEAVES["block_norm"] if n in s]
        grads = torch.autograd.grad(tuple(out.values()), [s[n] for n in names],
                                    (s["dh"], s["dn"]) if c["pre"] else (s["dh"],))
        out.update(("d_" + n, g) for n, g in zip(names, grads))
    return out


def _plain_sort_back(s):
    c = s["case"]
    T, E, k = c["T"], c["E"], c["k"]
    dt = DTYPES[c["dtype"]]
    key = s["expert_idx"].reshape(-1)
    live = (key >= 0) & (key < E)
    key = torch.where(live, key, E)
    order = torch.argsort(key, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device=key.device)
    counts = torch.zeros(E + 1, dtype=torch.int64, device=key.device).scatter_add_(0, key, torch.ones_like(key))[:E]
    rows = s["x"].float()[order // k] * live[order].float()[:, None]
    lw = live.reshape(T, k).float()
    picked = s["ye"].float()[place].reshape(T, k, -1)
    w = s["weights"].float()
    y = (picked * (w * lw)[:, :, None]).sum(1)
    out = {"rows": rows.to(dt), "tokens_per_expert": counts, "where": torch.where(live, place, -1).reshape(T, k),
           "y": y.to(dt)}
    if c["train"]:
        dy = s["dy"].float()
        out["dx"] = (s["d_rows"].float()[place].reshape(T, k, -1) * lw[:, :, None]).sum(1).to(dt)
        out["dye"] = ((w * lw).reshape(-1)[order][:, None] * dy[order // k]).to(dt)
        out["dw"] = ((picked * dy[:, None, :]).sum(2) * lw).to(dt)
    return out


def _dequantise(codes, scales, zeros, group, dtype):
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).to(dtype)
    z = 8.0 if zeros is None else zeros.to(dtype).repeat_interleave(group, dim=-1)
    return (q - z) * scales.to(dtype).repeat_interleave(group, dim=-1)


def _activate(a, swiglu):
    if not swiglu:
        return a
    g, u = a.chunk(2, dim=-1)
    return g / (1.0 + torch.exp(-g)) * u


def _plain_w4(s):
    c = s["case"]
    P, E, g = c["T"] * c["k"], c["E"], c["group"]
    x = s["rows"].float()
    ends = torch.cumsum(s["tokens_per_expert"], 0)
    expert = torch.searchsorted(ends, torch.arange(P, device=x.device), right=True)
    zeros = s.get("zeros")
    if P <= E:                    # few rows: each row's own expert
        parts = []
        for i in range(0, P, 8):
            e = expert[i:i + 8]
            w = _dequantise(s["codes"][e], s["scales"][e], None if zeros is None else zeros[e], g, torch.float32)
            parts.append(torch.matmul(w, x[i:i + 8, :, None])[:, :, 0])
        acc = torch.cat(parts)
    else:                         # every expert once, over all rows
        acc = torch.zeros((P, c["N"]), device=x.device)
        for e in range(E):
            w = _dequantise(s["codes"][e], s["scales"][e], None if zeros is None else zeros[e], g, torch.float32)
            acc = torch.where((expert == e)[:, None], torch.matmul(x, w.t()), acc)
    return _activate(acc, c["swiglu"]).to(DTYPES[c["dtype"]])


def _plain_block_norm(s):
    c = s["case"]
    dt, rt = DTYPES[c["dtype"]], DTYPES[c["residual"]]
    y, r = s["y"].float(), s["residual"].float()
    H = c["H"]
    wp = s["post_weight"].float() if c["post"] else None
    g = s["gate"].float() if c["gate"] != "none" else None
    wn = s["pre_weight"].float() if c["pre"] else None
    if c["post"]:
        inv1 = torch.rsqrt((y * y).sum(1, keepdim=True) / H + EPS)
        unit = y * inv1
        p = unit * wp
    else:
        p = y
    h = r + (_SCALE * p if g is None else _SCALE * g * p)
    out = {"h": h.to(rt)}
    if c["pre"]:
        inv2 = torch.rsqrt((h * h).sum(1, keepdim=True) / H + EPS)
        hu = h * inv2
        out["n"] = (hu * wn).to(dt)
    if not c["train"]:
        return out
    dh = s["dh"].float()
    if c["pre"]:
        dn = s["dn"].float()
        t = dn * wn
        dh = dh + inv2 * (t - hu * (t * hu).sum(1, keepdim=True) / H)
    dp = _SCALE * dh if g is None else _SCALE * g * dh
    if c["post"]:
        t = dp * wp
        out["d_y"] = (inv1 * (t - unit * (t * unit).sum(1, keepdim=True) / H)).to(dt)
    else:
        out["d_y"] = dp.to(dt)
    out["d_residual"] = dh.to(rt)
    if c["post"]:
        out["d_post_weight"] = (dp * unit).sum(0).to(dt)
    if c["gate"] != "none":
        dg = _SCALE * p * dh
        out["d_gate"] = (dg.sum(0) if c["gate"] == "channel" else dg.sum(1, keepdim=True)).to(dt)
    if c["pre"]:
        out["d_pre_weight"] = (dn * hu).sum(0).to(dt)
    return out


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------
def exact(case, seed):
    d = _inputs(case, seed)
    return {"sort_back": _exact_sort_back, "w4": _exact_w4, "block_norm": _exact_block_norm}[case["op"]](case, d)


def _exact_sort_back(c, d):
    T, E, k, H = c["T"], c["E"], c["k"], c["H"]
    flat = d["expert_idx"].reshape(-1).cpu()
    where = torch.full((T * k,), -1, dtype=torch.int64)
    counts, at = [], 0
    for e in range(E):            # expert by expert, its pairs in the order of the tokens
        mine = (flat == e).nonzero()[:, 0]
        where[mine] = torch.arange(at, at + len(mine))
        counts.append(len(mine))
        at += len(mine)
    where = where.reshape(T, k).cuda()
    rows = torch.zeros((T * k, H), dtype=torch.float64, device="cuda")
    y = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    w = d["weights"].double()
    train = c["train"]
    if train:
        dx, dye, dw = torch.zeros_like(y), torch.zeros_like(rows), torch.zeros_like(w)
    for j in range(k):            # one column of the routing at a time
        t = (where[:, j] >= 0).nonzero()[:, 0]
        at = where[t, j]
        rows[at] = d["x"][t].double()
        ye = d["ye"][at].double()
        y[t] += w[t, j, None] * ye
        if train:
            dy = d["dy"][t].double()
            dx[t] += d["d_rows"][at].double()
            dye[at] = w[t, j, None] * dy
            dw[t, j] = (dy * ye).sum(1)
    out = {"rows": rows, "tokens_per_expert": torch.tensor(counts, device="cuda"), "where": where, "y": y}
    if train:
        out.update(dx=dx, dye=dye, dw=dw)
    return out


def _exact_w4(c, d):
    g = c["group"]
    x = d["rows"].double()
    out, at = [], 0
    for e, n in enumerate(d["tokens_per_expert"].tolist()):
        if n == 0:
            continue
        codes = d["codes"][e].long()
        w = torch.empty((c["N"], c["K"]), dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = (codes % 16).double(), (codes // 16).double()
        w = w.reshape(c["N"], c["K"] // g, g)
        w = w - (d["zeros"][e].double()[:, :, None] if c["zeros"] else 8.0)
        w = (w * d["scales"][e].double()[:, :, None]).reshape(c["N"], c["K"])
        out.append(x[at:at + n] @ w.T)
        at += n
    a = torch.cat(out)
    if c["swiglu"]:
        half = c["N"] // 2
        a = a[:, :half] * torch.sigmoid(a[:, :half]) * a[:, half:]
    return a


def _exact_block_norm(c, d):
    leaves = {n: d[n].double().requires_grad_(c["train"]) for n in _LEAVES["block_norm"] if n in d}

    def unit(v):
        return v / (v.pow(2).mean(-1, keepdim=True) + EPS).sqrt()

    p = unit(leaves["y"]) * leaves["post_weight"] if c["post"] else leaves["y"]
    if "gate" in leaves:
        p = p * leaves["gate"]
    out = {"h": leaves["residual"] + _SCALE * p}
    if c["pre"]:
        out["n"] = unit(out["h"]) * leaves["pre_weight"]
    if c["train"]:
        ups = [d["dh"].double()] + ([d["dn"].double()] if c["pre"] else [])
        grads = torch.autograd.grad(list(out.values()), list(leaves.values()), ups)
        out = {n: v.detach() for n, v in out.items()}
        out.update(("d_" + n, v) for n, v in zip(leaves, grads))
    return out


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "sort_back":
        T, E, k, H = case["T"], case["E"], case["k"], case["H"]
        P = T * k
        small = P * 8 * 2 + E * 8 + P * b
        moved = (T + P) * H * b * 2                       # to expert order, and back
        if not case["train"]:
            return {"bytes": moved + small, "flops": 2 * P * H}
        # backward: the rows' gradient to the tokens; dy and the rows once each for dye and dw
        return {"bytes": moved + (P + T) * H * b + (T + 2 * P) * H * b + small + P * b, "flops": 6 * P * H}
    if case["op"] == "w4":
        T, E, k, N, K, g = (case[n] for n in ("T", "E", "k", "N", "K", "group"))
        P = T * k
        # experts that hold a row, for an even routing
        busy = E * (1.0 - (1.0 - min(1.0, k / E)) ** T)
        per_expert = N * (K // 2 + K // g * (3 if case["zeros"] else 2))
        out = N // 2 if case["swiglu"] else N
        return {"bytes": int(busy * per_expert) + P * (K + out) * b + E * 8, "flops": 2 * P * N * K}
    T, H = case["T"], case["H"]
    rb = BYTES[case["residual"]]
    vectors = sum((case["post"], case["gate"] == "channel", case["pre"])) * H * b
    pre = b if case["pre"] else 0
    if not case["train"]:
        return {"bytes": T * H * (b + 2 * rb + pre) + vectors, "flops": 8 * T * H}
    # backward: y, the residual and both gradients once, d_y and d_residual once
    return {"bytes": T * H * (b + 2 * rb + pre) + T * H * (b + rb + rb + pre + b + rb) + 3 * vectors,
            "flops": 30 * T * H}
