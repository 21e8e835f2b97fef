"""The operators around the experts against plain 64-bit implementations: tokens to expert order and back with its
gradient, the experts' products on 4-bit weights, the norms between blocks; and a run of them together.

Tolerances.  A kernel computes in fp32 and rounds each output once, so an output v may differ from the 64-bit value by
half a step of its type, eps/2 * |v| (plus half the smallest subnormal), and by what fp32 arithmetic adds: every add,
multiply or fused multiply-add is off by at most 2^-24 of its result, so a chain of n of them over terms of magnitude
m_i by at most n * 2^-24 * sum m_i.  Each test takes n from the longest chain of its kernel and the m_i from the
64-bit values."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = 2.0 ** -24


def announce(*what):
    print("[case]", *what, flush=True)


def near(got, want, magnitude, chain, name):
    """``got`` within the rounding of its type and ``chain`` fp32 steps over ``magnitude`` of the 64-bit ``want``."""
    fi = torch.finfo(got.dtype)
    slack = chain * U * magnitude + fi.smallest_normal * fi.eps
    tol = fi.eps / 2 * (want.abs() + slack) + slack
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), (f"{name}: {int(bad.sum())} of {bad.numel()} off, worst "
                                 f"{float((err / tol).nan_to_num(1e9).max()):.3g} of the tolerance")


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def routing(T, E, k, seed, dead=0.0):
    g = gen(seed)
    idx = torch.randn(T, E, generator=g, device=DEV).topk(k, dim=1).indices if E >= k else \
        torch.randint(0, E, (T, k), generator=g, device=DEV)
    if dead:
        idx = torch.where(torch.rand(T, k, generator=g, device=DEV) < dead, -1, idx)
    return idx.contiguous()


def sort_oracle(idx, E):
    """(where, counts, offsets) by a stable sort on the host."""
    flat = idx.reshape(-1).cpu().numpy()
    live = (flat >= 0) & (flat < E)
    where = np.full(flat.size, -1, dtype=np.int64)
    pairs = np.nonzero(live)[0]
    where[pairs[np.argsort(flat[pairs], kind="stable")]] = np.arange(pairs.size)
    counts = np.bincount(flat[pairs], minlength=E)
    return (torch.from_numpy(where.reshape(tuple(idx.shape))), torch.from_numpy(counts.astype(np.int64)),
            torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)))


def check_sort(x, idx, E):
    import terrace.ops as tops
    rows, plan = tops.expert_sort(x, idx, E)
    where, counts, offsets = sort_oracle(idx, E)
    assert torch.equal(plan.where.cpu(), where) and torch.equal(plan.tokens_per_expert.cpu(), counts)
    assert torch.equal(plan.offsets.cpu(), offsets)
    want = torch.zeros((idx.numel(), x.shape[1]), dtype=x.dtype, device=DEV)
    t, j = (where >= 0).nonzero(as_tuple=True)
    want[where[t, j].to(DEV)] = x[t.to(DEV)]
    assert rows.dtype == x.dtype and torch.equal(rows, want)
    return rows, plan


# ---- tokens to expert order ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,E,k,H,dtype,dead", [
    (0, 8, 2, 16, "bf16", 0.0), (1, 1, 1, 1, "f32", 0.0), (1, 256, 8, 7168, "bf16", 0.0), (1, 8, 2, 5, "f16", 1.0),
    (61, 128, 8, 4096, "bf16", 0.25), (64, 2048, 8, 40, "f32", 0.1), (3, 4, 17, 24, "bf16", 0.3), (2, 5, 40, 9, "f16", 0.3),
    (256, 8, 8, 33, "bf16", 0.0), (257, 8, 8, 33, "bf16", 0.2), (1024, 2048, 4, 24, "bf16", 0.1), (1025, 9, 4, 24, "bf16", 0.1), (2048, 7, 1, 64, "f32", 0.5), (2049, 7, 1, 64, "f32", 0.5),
    (4096, 64, 4, 128, "f32", 0.0), (5003, 60, 6, 72, "bf16", 0.1), (3000, 2048, 8, 16, "f16", 0.2),
    (700, 300, 3, 7, "bf16", 1.0), (9000, 256, 8, 520, "bf16", 0.05),
])
def test_expert_sort_sizes(T, E, k, H, dtype, dead):
    announce("expert_sort", T, E, k, H, dtype, dead)
    x = torch.randn((T, H), generator=gen(T + H), device=DEV).to(DT[dtype])
    _, plan = check_sort(x, routing(T, E, k, T + k, dead), E)
    assert int(plan.status[0]) == 0


@pytest.mark.parametrize("T", [40, 900])
def test_expert_sort_ids_outside_the_range_are_no_expert_and_reported(T):
    from terrace import _hip
    announce("expert_sort ids", T)
    idx = routing(T, 16, 4, 3)
    idx[0, 0], idx[T // 2, 2], idx[T - 1, 3] = 16, 1 << 40, -(1 << 40)
    idx[1] = -1                                              # a token without any expert
    x = torch.randn((T, 24), generator=gen(1), device=DEV)
    rows, plan = check_sort(x, idx, 16)
    assert int(plan.status[0]) == _hip.FAULT_ID_RANGE


@pytest.mark.parametrize("T", [50, 3000])
def test_expert_sort_same_expert_twice_strides_and_other_types(T):
    import terrace.ops as tops
    announce("expert_sort strides", T)
    idx = torch.full((T, 3), 2, dtype=torch.int64, device=DEV)          # the same expert three times
    wide = torch.randn((T, 80), generator=gen(2), device=DEV)
    check_sort(wide[:, 8:48], idx, 4)                                   # rows on a stride that is no kilobyte pitch
    check_sort(wide.t().contiguous().t(), idx, 4)                       # columns first
    check_sort(wide[:, 1:34], idx.flip(1), 4)
    check_sort(torch.randint(0, 255, (T, 37), generator=gen(3), device=DEV, dtype=torch.uint8), routing(T, 9, 3, 4), 9)
    pitched = torch.zeros((T, 1024), dtype=torch.uint8, device=DEV)[:, :992]
    pitched.copy_(torch.randint(0, 255, (T, 992), generator=gen(5), device=DEV, dtype=torch.uint8))
    rows, _ = check_sort(pitched, routing(T, 9, 3, 6, 0.2), 9)          # rows on a kilobyte pitch keep it
    assert rows.stride(0) == 1024
    wide_idx = torch.full((T, 6), -1, dtype=torch.int64, device=DEV)
    wide_idx[:, ::2] = routing(T, 9, 3, 7)
    rows, plan = tops.expert_sort(wide, wide_idx[:, ::2], 9)
    same, _ = tops.expert_sort(wide, wide_idx[:, ::2].contiguous(), 9)
    assert torch.equal(rows, same)


def test_expert_sort_gradient():
    import terrace.ops as tops
    for T, E, k, H, dtype, dead in [(5, 8, 3, 40, "f32", 0.3), (300, 16, 8, 264, "bf16", 0.2), (700, 9, 4, 33, "f16", 0.5)]:
        announce("expert_sort gradient", T, E, k, H, dtype, dead)
        idx = routing(T, E, k, T, dead)
        x = torch.randn((T, H), generator=gen(T), device=DEV).to(DT[dtype]).requires_grad_(True)
        rows, plan = tops.expert_sort(x, idx, E)
        g = torch.randn(rows.shape, generator=gen(T + 1), device=DEV).to(rows.dtype)
        g[int(plan.offsets[-1]):] = float("nan")             # rows of no pair send nothing back
        (dx,) = torch.autograd.grad(rows, x, g)
        live = plan.where >= 0
        terms = torch.where(live[..., None], g.double()[plan.where.clamp(min=0)], 0.0)
        near(dx, terms.sum(1), terms.abs().sum(1), k, "dx")


# ---- and back -----------------------------------------------------------------------------------------------------
def unsort_oracle(rows, weights, plan, dy):
    """(y, |y| terms, d_rows, d_weights, |d_weights| terms) in 64 bits."""
    live = plan.where >= 0
    at = plan.where.clamp(min=0)
    w = torch.ones(at.shape, dtype=torch.float64, device=DEV) if weights is None else weights.double()
    picked = torch.where(live[..., None], rows.double()[at], 0.0)
    terms = picked * w[..., None]
    d_rows = torch.zeros(rows.shape, dtype=torch.float64, device=DEV)
    t, j = live.nonzero(as_tuple=True)
    d_rows[at[t, j]] = w[t, j, None] * dy.double()[t]
    products = picked * dy.double()[:, None, :]
    return terms.sum(1), terms.abs().sum(1), d_rows, products.sum(2), products.abs().sum(2)


@pytest.mark.parametrize("T,E,k,H,dtype,wtype,otype,dead", [
    (1, 4, 2, 8, "f32", "f32", None, 0.0), (1, 256, 8, 7168, "bf16", "bf16", None, 0.0),
    (33, 16, 8, 264, "bf16", "f32", "f32", 0.3), (200, 8, 4, 1001, "f16", "f16", None, 0.2),
    (600, 60, 6, 520, "bf16", "bf16", None, 0.5), (40, 4, 3, 24, "f32", "f32", "bf16", 1.0),
    (64, 8, 17, 136, "f32", "bf16", None, 0.1), (1000, 5, 1, 7, "f16", "f32", None, 0.1), (64, 8, 4, 64, "bf16", None, None, 0.2),
    (300, 40, 9, 1, "f32", "f32", None, 0.2),
])
def test_expert_unsort_and_its_gradient(T, E, k, H, dtype, wtype, otype, dead):
    import terrace.ops as tops
    announce("expert_unsort", T, E, k, H, dtype, wtype, otype, dead)
    idx = routing(T, E, k, T + 1, dead)
    _, plan = tops.expert_sort(torch.zeros((T, 8), device=DEV), idx, E)
    g = gen(T + H)
    rows = torch.randn((T * k, H), generator=g, device=DEV).to(DT[dtype])
    rows[int(plan.offsets[-1]):] = float("nan")              # nothing reads the rows of no pair
    rows.requires_grad_(True)
    weights = None
    if wtype:
        weights = torch.rand((T, k), generator=g, device=DEV).to(DT[wtype])
        weights[plan.where < 0] = float("nan")               # nor the weights of pairs without an expert
        weights.requires_grad_(True)
    out_dtype = DT[otype] if otype else None
    y = tops.expert_unsort(rows, weights, plan, out_dtype)
    assert y.dtype == (out_dtype or DT[dtype]) and y.shape == (T, H)
    dy = torch.randn((T, H), generator=g, device=DEV).to(y.dtype)
    clean = None if weights is None else weights.detach().nan_to_num(0.0)
    want_y, mag_y, want_rows, want_w, mag_w = unsort_oracle(rows.detach().nan_to_num(0.0), clean, plan, dy)
    near(y, want_y, mag_y, 2 * k, "y")                       # a product and an add per term
    leaves = (rows,) if weights is None else (rows, weights)
    grads = torch.autograd.grad(y, leaves, dy)
    near(grads[0], want_rows, want_rows.abs(), 1, "d_rows")
    if weights is not None:                                  # a lane's elements, 6 butterfly steps, 4 waves
        near(grads[1], want_w, mag_w, H / 64 + 8 + 10, "d_weights")
        only_w = torch.autograd.grad(tops.expert_unsort(rows.detach(), weights, plan, out_dtype), weights, dy)[0]
        assert torch.equal(only_w, grads[1])
        only_rows = torch.autograd.grad(tops.expert_unsort(rows, weights.detach(), plan, out_dtype), rows, dy)[0]
        assert torch.equal(only_rows, grads[0])
    again = torch.autograd.grad(tops.expert_unsort(rows, weights, plan, out_dtype), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))         # no sum depends on timing


def test_expert_unsort_gradient_against_differences():
    """y is linear in the rows and in the weights, so a central difference has no truncation error: what is left is the
    rounding of y, eps/2 a term, over the step."""
    import terrace.ops as tops
    announce("expert_unsort differences")
    T, E, k, H = 20, 6, 3, 48
    idx = routing(T, E, k, 5, 0.2)
    _, plan = tops.expert_sort(torch.zeros((T, 8), device=DEV), idx, E)
    g = gen(9)
    rows = torch.randn((T * k, H), generator=g, device=DEV).requires_grad_(True)
    weights = torch.rand((T, k), generator=g, device=DEV).requires_grad_(True)
    dy = torch.randn((T, H), generator=g, device=DEV)
    grads = torch.autograd.grad(tops.expert_unsort(rows, weights, plan), (rows, weights), dy)
    for leaf, grad, other in ((0, grads[0], weights), (1, grads[1], rows)):
        base = (rows, weights)[leaf].detach()
        d = torch.randn(base.shape, generator=g, device=DEV)
        step = 0.5

        def loss(v):
            args = (v, weights.detach()) if leaf == 0 else (rows.detach(), v)
            return float((tops.expert_unsort(*args, plan).double() * dy.double()).sum())

        up, down = loss(base + step * d), loss(base - step * d)
        size = float(dy.double().abs().sum()) * 8 * k        # a bound on the sum of |dy y| for these inputs
        assert abs((up - down) / (2 * step) - float((grad.double() * d.double()).sum())) <= 8 * k * U * size / step


# ---- 4-bit products -----------------------------------------------------------------------------------------------
def w4_case(E, N, K, group, dtype, zeros, seed):
    g = gen(seed)
    codes = torch.randint(0, 256, (E, N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = ((torch.rand((E, N, K // group), generator=g, device=DEV) + 0.5) / math.sqrt(K)).to(DT[dtype])
    z = torch.randint(0, 16, scales.shape, generator=g, device=DEV, dtype=torch.uint8) if zeros else None
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double().view(E, N, K // group, group)
    off = z.double()[..., None] if zeros else 8.0
    weight = ((q - off) * scales.double()[..., None]).view(E, N, K)
    # what the kernel adds up: (16 + code) x and (16 + zero) x, each times the scale
    size = ((q + 16 + off + 16) * scales.double()[..., None]).view(E, N, K)
    return codes, scales, z, weight, size


def check_w4(E, N, K, group, dtype, zeros, swiglu, counts, tail=0, seed=0):
    import terrace.ops as tops
    announce("w4", E, N, K, group, dtype, zeros, swiglu, counts, tail)
    codes, scales, z, weight, size = w4_case(E, N, K, group, dtype, zeros, seed)
    packed = tops.w4_pack(codes, scales, z)
    P = sum(counts) + tail
    x = torch.randn((P, K), generator=gen(seed + 1), device=DEV).to(DT[dtype])
    if tail:
        x[P - tail:] = float("nan")                          # rows of no expert are not read into anything
    out = tops.expert_linear_w4(x, torch.tensor(counts, device=DEV), packed, swiglu=swiglu)
    a, m = torch.zeros((P, N), dtype=torch.float64, device=DEV), torch.zeros((P, N), dtype=torch.float64, device=DEV)
    at = 0
    for e, c in enumerate(counts):
        a[at:at + c] = x[at:at + c].double() @ weight[e].T
        m[at:at + c] = x[at:at + c].double().abs() @ size[e].T
        at += c
    # the chain: a group's steps inside the matrix instructions (two units each, for their own way of rounding), then a
    # multiply-add per group and the waves
    chain = 2 * (group + 2) + K / group + 10
    if not swiglu:
        near(out, a, m, chain, "out")
    else:
        gt, up, mg, mu = a[:, :N // 2], a[:, N // 2:], m[:, :N // 2], m[:, N // 2:]
        silu = gt * torch.sigmoid(gt)
        # |silu'| <= 1.1; the exponential and the division: a few units, and |gate| units for the exponent's argument
        mag = 1.1 * mg * up.abs() + silu.abs() * mu + (16 + gt.abs()) / chain * (silu * up).abs()
        near(out, silu * up, mag + chain * U * 1.1 * mg * mu, chain, "out")
    return x, packed, out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("E,N,K,group,zeros,swiglu,counts", [
    (1, 16, 32, 32, False, False, [1]), (1, 1, 128, 128, True, False, [3]), (3, 33, 96, 32, True, False, [0, 5, 1]),
    (4, 64, 256, 128, False, True, [1, 0, 0, 17]), (2, 50, 192, 64, True, True, [16, 15]), (5, 40, 320, 64, False, False, [0] * 5),
    (4, 48, 512, 128, True, False, [40, 33, 1, 0]), (2, 34, 288, 32, False, True, [70, 129]), (70, 18, 64, 64, False, False, [1, 0] * 35),
    (1, 256, 1024, 128, False, False, [1]), (3, 80, 160, 32, True, False, [64, 65, 63]),
    (2, 11000, 160, 32, True, True, [130, 40]), (3, 20000, 128, 128, False, False, [20, 33, 1]), (1, 16400, 96, 32, False, True, [250]),
    (2, 24010, 448, 64, True, False, [64, 64]), (1, 66000, 32, 32, False, False, [33]),
    (1, 50, 640, 128, True, True, [100]), (1, 40, 1120, 32, False, False, [31]), (2, 66, 2048, 64, True, False, [130, 3]),
    (1, 130, 416, 32, True, False, [64]),
])
def test_w4_products(E, N, K, group, zeros, swiglu, counts, dtype):
    check_w4(E, N, K, group, dtype, zeros, swiglu, counts, 0, E + N)
    if sum(counts):
        check_w4(E, N, K, group, dtype, zeros, swiglu, counts, 7, E + N + 1)


def test_w4_one_matrix_without_counts_and_no_rows():
    import terrace.ops as tops
    x, packed, out = check_w4(1, 48, 128, 64, "bf16", False, False, [9])
    assert torch.equal(tops.expert_linear_w4(x, None, packed), out)
    codes, scales, z, _, _ = w4_case(1, 48, 128, 64, "bf16", True, 3)
    flat = tops.w4_pack(codes[0], scales[0], z[0])
    full = tops.w4_pack(codes, scales, z)
    assert torch.equal(tops.expert_linear_w4(x, None, flat), tops.expert_linear_w4(x, None, full))
    assert tuple(tops.expert_linear_w4(x[:0], None, packed).shape) == (0, 48)
    shifted = torch.empty((9 * 128 + 1,), dtype=x.dtype, device=DEV)[1:].view(9, 128).copy_(x)       # off 16 bytes
    assert torch.equal(tops.expert_linear_w4(shifted, None, packed), out)
    wide = torch.randn((9, 300), generator=gen(1), device=DEV).to(x.dtype)
    wide[:, 5:133] = x
    assert torch.equal(tops.expert_linear_w4(wide[:, 5:133], None, packed), out)


def test_w4_counts_that_do_not_fit_the_rows_stay_inside_them():
    import terrace.ops as tops
    announce("w4 counts")
    codes, scales, z, weight, _ = w4_case(3, 32, 64, 32, "bf16", False, 5)
    packed = tops.w4_pack(codes, scales)
    x = torch.randn((10, 64), generator=gen(6), device=DEV).to(torch.bfloat16)
    fits = tops.expert_linear_w4(x, torch.tensor([4, 0, 6], device=DEV), packed)
    over = tops.expert_linear_w4(x, torch.tensor([4, -7, 1 << 40], device=DEV), packed)
    assert torch.equal(fits, over)
    first = tops.expert_linear_w4(x, torch.tensor([1 << 62, 1 << 62, 1 << 62], device=DEV), packed)
    assert torch.equal(first, tops.expert_linear_w4(x, torch.tensor([10, 0, 0], device=DEV), packed))
    none = tops.expert_linear_w4(x, torch.tensor([-1, 0, -(1 << 60)], device=DEV), packed)
    assert not bool(none.any())


# ---- between blocks -----------------------------------------------------------------------------------------------
def norm_oracle(y, r, wp, g, wn, scale, eps, dh=None, dn=None):
    """64-bit values and, for each, the magnitude that its fp32 steps act on."""
    d = [None if t is None else t.double() for t in (y, r, wp, g, wn, dh, dn)]
    y, r, wp, g, wn, dh, dn = d
    H = r.shape[-1]
    one = torch.ones((), dtype=torch.float64, device=DEV)
    has_y = y is not None
    y = torch.zeros_like(r) if y is None else y
    inv1 = 1 / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt() if wp is not None else one
    u = y * inv1
    p = u * wp if wp is not None else u
    f = scale * (g if g is not None else one)
    h = r + f * p
    mh = r.abs() + (f * p).abs()
    val, mag = {"h": h}, {"h": mh}
    inv2 = 1 / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    # an error in h moves inv2 by a relative mean(|h| mh) * inv2^2 <= max-norm ratio of mh to h
    blow = (h.abs() * mh).mean(-1, keepdim=True) * inv2 ** 2 + 1
    v, mv = h * inv2, mh * inv2 * blow
    if wn is not None:
        val["n"], mag["n"] = v * wn, mv * wn.abs()
    if dh is None and dn is None:
        return val, mag
    dh = torch.zeros_like(r) if dh is None else dh
    t = dn * wn if dn is not None else torch.zeros_like(r)
    mt = t.abs()
    dH = dh + inv2 * (t - v * (t * v).mean(-1, keepdim=True))
    mean_tv = (mt * mv).mean(-1, keepdim=True)
    mdH = dh.abs() + inv2 * blow * (mt + mv * mean_tv)
    val["d_residual"], mag["d_residual"] = dH, mdH
    dp, mdp = f * dH, f.abs() * mdH
    if has_y:
        if wp is not None:
            q = wp * u
            mdot = ((dh.abs() + inv2 * blow * mt) * (f * q).abs()).mean(-1, keepdim=True) + \
                inv2 * blow * mean_tv * (mv * (f * q).abs()).mean(-1, keepdim=True)
            val["d_y"] = inv1 * (dp * wp - u * (dp * wp * u).mean(-1, keepdim=True))
            mag["d_y"] = inv1 * (mdp * wp.abs() + u.abs() * mdot)
            val["d_post"], mag["d_post"] = (dp * u).sum(0), (mdp * u.abs()).sum(0)
        else:
            val["d_y"], mag["d_y"] = dp, mdp
        if g is not None:
            dg, mg = scale * p * dH, (scale * p).abs() * mdH
            if g.shape == (H,):
                val["d_gate"], mag["d_gate"] = dg.sum(0), mg.sum(0)
            else:
                # the token's sum is taken as two sums whose difference it is
                val["d_gate"] = dg.sum(-1, keepdim=True)
                mag["d_gate"] = abs(scale) * H * (((dh.abs() + inv2 * blow * mt) * p.abs()).mean(-1, keepdim=True) +
                                                  inv2 * blow * mean_tv * (mv * p.abs()).mean(-1, keepdim=True))
    if dn is not None:
        val["d_pre"], mag["d_pre"] = (dn * v).sum(0), (dn.abs() * mv).sum(0)
    return val, mag


def norm_inputs(T, H, dtype, residual, has_y, post, gate, pre, seed, lead=None):
    g = gen(seed)
    shape = (lead or (T,)) + (H,)

    def normal(s, dt, a=1.0, b=0.0):
        return (torch.randn(s, generator=g, device=DEV) * a + b).to(dt)

    dt, rt = DT[dtype], DT[residual]
    y = normal(shape, dt, 2.0) if has_y else None
    r = normal(shape, rt)
    wp = normal((H,), dt, 0.2, 1.0) if post else None
    gt = None if gate is None else normal((H,) if gate == "channel" else shape[:-1] + (1,), dt, 0.3, 0.5)
    wn = normal((H,), dt, 0.2, 1.0) if pre else None
    dh, dn = normal(shape, rt), normal(shape, dt) if pre else None
    return y, r, wp, gt, wn, dh, dn


def check_norm(T, H, dtype, residual, has_y=True, post=True, gate=None, pre=True, scale=0.75, eps=1e-6, seed=0, use=(1, 1)):
    import terrace.ops as tops
    announce("block_norm", T, H, dtype, residual, has_y, post, gate, pre, use)
    y, r, wp, gt, wn, dh, dn = norm_inputs(T, H, dtype, residual, has_y, post, gate, pre, seed)
    h, n = tops.block_norm(y, r, wp, gt, wn, scale=scale, eps=eps)
    dh = dh if use[0] and has_y else None
    dn = dn if use[1] and pre else None
    val, mag = norm_oracle(y, r, wp, gt, wn, scale, eps, dh, dn)
    chain = H / 64 + 40                                      # a lane's share of the row, 6 + 16 joining steps, the rest
    if has_y:
        assert h.dtype == r.dtype
        near(h, val["h"], mag["h"], chain, "h")
    else:
        assert h is r
    if pre:
        assert n.dtype == (y if has_y else r).dtype
        near(n, val["n"], mag["n"], chain, "n")
    else:
        assert n is None
    leaves = {"d_y": y, "d_residual": r, "d_post": wp, "d_gate": gt, "d_pre": wn}
    leaves = {k: v.requires_grad_(True) for k, v in leaves.items() if v is not None}
    h2, n2 = tops.block_norm(y, r, wp, gt, wn, scale=scale, eps=eps)
    assert (h2 is r) if not has_y else torch.equal(h2, h)
    assert n2 is None or torch.equal(n2, n)
    outs, ups = zip(*[(o, d) for o, d in ((h2, dh), (n2, dn)) if d is not None])
    grads = torch.autograd.grad(outs, list(leaves.values()), ups, allow_unused=True)
    again = torch.autograd.grad(tops_again(y, r, wp, gt, wn, scale, eps, dh, dn), list(leaves.values()), ups, allow_unused=True)
    for (name, leaf), got, twice in zip(leaves.items(), grads, again):
        if name not in val:                                  # the norm before was not used: its weight has no gradient
            assert got is None or not bool(got.any()), name
            continue
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        assert torch.equal(got, twice), name
        near(got, val[name], mag[name], chain + (T if name in ("d_post", "d_gate", "d_pre") else 0), name)


def tops_again(y, r, wp, gt, wn, scale, eps, dh, dn):
    import terrace.ops as tops
    h, n = tops.block_norm(y, r, wp, gt, wn, scale=scale, eps=eps)
    return tuple(o for o, d in ((h, dh), (n, dn)) if d is not None)


@pytest.mark.parametrize("T,H,dtype,residual,has_y,post,gate,pre", [
    (1, 8, "f32", "f32", True, True, "channel", True), (1, 7168, "bf16", "bf16", True, True, "channel", True),
    (3, 1, "f32", "f32", True, True, None, True), (5, 64, "bf16", "f32", True, True, "token", True),
    (203, 1001, "f16", "f32", True, True, "token", True), (130, 264, "bf16", "bf16", True, False, "channel", True),
    (77, 4096, "f16", "f16", True, True, "channel", False), (300, 512, "f32", "f32", True, False, None, False),
    (33, 8192, "bf16", "bf16", True, True, "token", True), (9, 16384, "bf16", "f32", True, True, "channel", True),
    (300, 9000, "f32", "f32", True, True, "token", True), (270, 8193, "bf16", "bf16", True, True, "channel", True), (5, 16383, "f16", "f32", True, True, "token", True),
    (9, 15, "bf16", "bf16", True, True, "channel", True), (700, 7, "f16", "f16", True, True, "token", True), (12, 8191, "bf16", "bf16", True, True, "channel", True),
    (600, 72, "f16", "f16", True, True, "token", False), (40, 640, "bf16", "bf16", False, False, None, True),
    (21, 333, "f32", "f32", False, False, None, True), (1500, 1024, "f32", "f32", True, True, "channel", True),
])
def test_block_norm_and_its_gradient(T, H, dtype, residual, has_y, post, gate, pre):
    check_norm(T, H, dtype, residual, has_y, post, gate, pre, seed=T + H)


def test_block_norm_with_one_of_its_results_unused():
    check_norm(50, 128, "f32", "f32", True, True, "channel", True, use=(1, 0))
    check_norm(50, 128, "bf16", "bf16", True, True, "token", True, use=(0, 1))


def test_block_norm_shapes_strides_and_extremes():
    import terrace.ops as tops
    announce("block_norm strides")
    y, r, wp, gt, wn, _, _ = norm_inputs(24, 96, "bf16", "bf16", True, True, "token", True, 4)
    h, n = tops.block_norm(y, r, wp, gt, wn)
    h3, n3 = tops.block_norm(y.view(2, 3, 4, 96), r.view(2, 3, 4, 96), wp, gt.view(2, 3, 4, 1), wn)
    assert h3.shape == (2, 3, 4, 96) and torch.equal(h3.view(24, 96), h) and torch.equal(n3.view(24, 96), n)
    wide = torch.zeros((24, 200), dtype=torch.bfloat16, device=DEV)
    wide[:, 3:99] = y
    h2, n2 = tops.block_norm(wide[:, 3:99], r.t().contiguous().t(), wp, gt, wn)
    assert torch.equal(h2, h) and torch.equal(n2, n)
    one = torch.randn((96,), generator=gen(2), device=DEV).bfloat16()
    h1, n1 = tops.block_norm(one, one, wp, None, wn)                    # a single row without a leading axis
    h2, n2 = tops.block_norm(one[None], one[None], wp, None, wn)
    assert torch.equal(h1, h2[0]) and torch.equal(n1, n2[0])
    zero = torch.zeros((2, 64), device=DEV)
    h, n = tops.block_norm(zero, zero, torch.ones(64, device=DEV), None, torch.ones(64, device=DEV))
    assert not bool(h.any()) and not bool(n.any())
    bad = torch.randn((3, 64), generator=gen(3), device=DEV)
    good_h, _ = tops.block_norm(bad, bad, torch.ones(64, device=DEV), None, torch.ones(64, device=DEV))
    poisoned = bad.clone()
    poisoned[1, 5] = float("nan")
    h, n = tops.block_norm(poisoned, bad, torch.ones(64, device=DEV), None, torch.ones(64, device=DEV))
    assert bool(h[1].isnan().all()) and torch.equal(h[0], good_h[0]) and torch.equal(h[2], good_h[2])
    empty = torch.zeros((0, 64), device=DEV, requires_grad=True)
    w = torch.ones(64, device=DEV, requires_grad=True)
    h, n = tops.block_norm(empty, empty, w, None, w)
    (dw,) = torch.autograd.grad((h, n), w, (torch.zeros_like(h), torch.zeros_like(n)))
    assert h.shape == (0, 64) and not bool(dw.any())


def test_block_norm_gradient_against_differences():
    """A central difference of step e along d: the third derivative's e^2 term and the forward's rounding over e.  With
    rows of unit size the map's third directional derivative is a few times |d|^3 a row, e = 2^-6, so a relative
    2^-9 of the sum of magnitudes covers both."""
    import terrace.ops as tops
    announce("block_norm differences")
    y, r, wp, gt, wn, dh, dn = norm_inputs(30, 128, "f32", "f32", True, True, "channel", True, 8)
    leaves = [t.requires_grad_(True) for t in (y, r, wp, gt, wn)]
    grads = torch.autograd.grad(tops.block_norm(*leaves, scale=0.75), leaves, (dh, dn))
    step = 2.0 ** -6

    def loss(args):
        h, n = tops.block_norm(*args, scale=0.75)
        return float((h.double() * dh.double()).sum() + (n.double() * dn.double()).sum())

    for i, grad in enumerate(grads):
        base = [t.detach() for t in leaves]
        d = torch.randn(base[i].shape, generator=gen(i), device=DEV)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + step * d, base[i] - step * d
        terms = grad.double() * d.double()
        assert abs((loss(up) - loss(down)) / (2 * step) - float(terms.sum())) <= 2.0 ** -9 * float(terms.abs().sum())


# ---- refusals -----------------------------------------------------------------------------------------------------
def test_refusals():
    import terrace.ops as tops
    announce("refusals")
    x, idx = torch.zeros((4, 32), device=DEV), torch.zeros((4, 2), dtype=torch.int64, device=DEV)
    for args, what in [((x[0], idx, 4), "must be"), ((x, idx[:3], 4), "must be"), ((x, idx.int(), 4), "int64"),
                       ((x, idx, 0), "experts"), ((x, idx, 2049), "experts"), ((x, idx[:, :0], 4), "column"),
                       ((x.cpu(), idx, 4), "ROCm device")]:
        with pytest.raises(RuntimeError, match=what):
            tops.expert_sort(*args)
    rows, plan = tops.expert_sort(x, idx, 4)
    w = torch.ones((4, 2), device=DEV)
    for args, what in [((rows[:7], w, plan), "one row per pair"), ((rows, w[:, :1], plan), "match"),
                       ((rows.double(), w, plan), "float32"), ((rows, w.int(), plan), "float32"),
                       ((rows, w, plan, torch.float64), "float32")]:
        with pytest.raises(RuntimeError, match=what):
            tops.expert_unsort(*args)
    codes = torch.zeros((2, 8, 32), dtype=torch.uint8, device=DEV)
    scales = torch.ones((2, 8, 2), dtype=torch.bfloat16, device=DEV)
    for args, what in [((codes.int(), scales), "uint8"), ((codes, scales[:, :4]), "uint8"), ((codes, scales.float()), "bfloat16"),
                       ((codes, scales[:, :, :0]), "groups"), ((codes, scales.repeat(1, 1, 2)), "groups"),
                       ((codes, scales, torch.zeros((2, 8, 1), dtype=torch.uint8, device=DEV)), "zeros"),
                       ((codes[:, :, :24], scales[:, :, :1]), "groups"), ((codes, scales, scales), "zeros")]:
        with pytest.raises(RuntimeError, match=what):
            tops.w4_pack(*args)
    packed = tops.w4_pack(codes, scales)
    xs, counts = torch.zeros((3, 64), dtype=torch.bfloat16, device=DEV), torch.tensor([1, 2], device=DEV)
    for args, what in [((xs[:, :32], counts, packed), "rows must be"), ((xs.half(), counts, packed), "rows must be"),
                       ((xs, counts.int(), packed), "int64"), ((xs, counts[:1], packed), "int64"), ((xs, None, packed), "needed"),
                       ((xs.clone().requires_grad_(True), counts, packed), "forward only")]:
        with pytest.raises(RuntimeError, match=what):
            tops.expert_linear_w4(*args)
    with pytest.raises(RuntimeError, match="even"):
        tops.expert_linear_w4(xs, counts, tops.w4_pack(codes[:, :7], scales[:, :7]), swiglu=True)
    with torch.no_grad():
        tops.expert_linear_w4(xs.clone().requires_grad_(True), counts, packed)
    y, v = torch.zeros((4, 32), device=DEV), torch.ones(32, device=DEV)
    for args, what in [((y, y[:3]), "one shape"), ((y, y.double()), "float32"), ((y, y.bfloat16()), "residual"),
                       ((y, y, v[:31]), "post_weight"), ((y, y, v, None, v[:31]), "pre_weight"), ((y, y, v, v[:31]), "gate"),
                       ((y, y, v, torch.ones((4, 32), device=DEV)), "gate"), ((None, y, v), "need a y"),
                       ((y[:, :0], y[:, :0]), "rows of 0")]:
        with pytest.raises(RuntimeError, match=what):
            tops.block_norm(*args)
    for H in (16385, 16392):
        big = torch.zeros((1, H), device=DEV)
        with pytest.raises(RuntimeError, match="rows of"):
            tops.block_norm(big, big)


# ---- together -----------------------------------------------------------------------------------------------------
def moe_block(tops, terrace, x, cfg, logits, bias, w_in, w_out, pre, post, gate, nxt):
    """One serving block: the norm before, the route, tokens to expert order, the experts, and back."""
    from terrace.ta2a_fwd import local_forward, w4_experts
    h0, n0 = tops.block_norm(None, x, pre_weight=pre)
    idx, gates, _ = terrace.t_route(logits, bias, cfg, gates_dtype=x.dtype)
    y, _ = local_forward(n0, idx, gates, w4_experts(w_in, w_out), cfg.n_experts)
    return tops.block_norm(y, h0, post, gate, nxt, scale=0.5)


@pytest.mark.parametrize("T", [1, 7, 300])
def test_a_block_of_them_together_and_as_a_graph(T):
    import terrace
    import terrace.ops as tops
    announce("block", T)
    E, k, H, I = 16, 4, 256, 128
    cfg = terrace.TRouteConfig(E, 4, k, 2)
    g = gen(T)

    def normal(s, a=1.0, b=0.0):
        return (torch.randn(s, generator=g, device=DEV) * a + b).bfloat16()

    x, logits, bias = normal((T, H)), torch.rand((T, E), generator=g, device=DEV), torch.zeros(E, device=DEV)
    ci, si, zi, wi, _ = w4_case(E, 2 * I, H, 64, "bf16", True, 1)
    co, so, _, wo, _ = w4_case(E, H, I, 32, "bf16", False, 2)
    w_in, w_out = tops.w4_pack(ci, si, zi), tops.w4_pack(co, so)
    vec = [normal((H,), 0.1, 1.0) for _ in range(4)]
    args = (tops, terrace, x, cfg, logits, bias, w_in, w_out, *vec)
    h, n = moe_block(*args)

    def plain():
        """The same block in 64 bits, rounded where the operators round."""
        def rnd(v):
            return v.bfloat16().double()

        def unit(v):
            return v / (v.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        xd = x.double()
        n0 = rnd(unit(xd) * vec[0].double())
        idx, gates, _ = terrace.t_route(logits, bias, cfg, gates_dtype=x.dtype)
        y = torch.zeros_like(xd)
        for j in range(k):
            a = torch.matmul(wi[idx[:, j]], n0[:, :, None])[..., 0]
            mid = rnd(a[:, :I] * torch.sigmoid(a[:, :I]) * a[:, I:])
            y += gates.double()[:, j, None] * rnd(torch.matmul(wo[idx[:, j]], mid[:, :, None])[..., 0])
        hd = xd + 0.5 * vec[2].double() * unit(rnd(y)) * vec[1].double()
        return hd, unit(hd) * vec[3].double()

    want_h, want_n = plain()
    # a value may fall to the other side of a rounding at four places (n0, mid, the experts' outputs, y), each one bf16
    # step (2^-8 of the value) on part of the terms; through two products their sum stays below four steps of a row's
    # largest, and the last rounding adds half a step
    for got, want in ((h, want_h), (n, want_n)):
        err = (got.double() - want).abs().max(-1).values
        assert bool((err <= 4.5 * 2.0 ** -8 * want.abs().max(-1).values).all()), float(err.max())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            moe_block(*args)                                 # on a stream of its own
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gh, gn = moe_block(*args)
    for rep in range(3):
        announce("block graph", T, rep)
        x.copy_(normal((T, H)))
        logits.copy_(torch.rand((T, E), generator=g, device=DEV))
        eh, en = moe_block(*args)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(gh, eh) and torch.equal(gn, en)


def test_the_local_path_is_the_loopback_path_without_its_hops():
    import terrace.ops as tops
    from conftest import equal_quota_routing
    from terrace.ta2a_fwd import local_forward, ta2a_loopback_forward, w4_experts
    announce("local against loopback")
    T, E, k, M, H, I = 500, 32, 4, 2, 128, 64
    idx = torch.from_numpy(equal_quota_routing(T, k, E, 4, M, 3, sort_rows=True)).to(DEV)       # 4 nodes of 8 cards
    g = gen(4)
    x = torch.randn((T, H), generator=g, device=DEV).bfloat16()
    gates = torch.rand((T, k), generator=g, device=DEV).bfloat16()
    ci, si, _, _, _ = w4_case(E, 2 * I, H, 64, "bf16", False, 1)
    co, so, _, _, _ = w4_case(E, H, I, 64, "bf16", False, 2)
    # every node of the loop-back holds its own 8 experts' slots: the same 8 matrices on each
    ci, si, co, so = (t[:8].repeat(4, 1, 1) for t in (ci, si, co, so))
    here, _ = local_forward(x, idx, gates, w4_experts(tops.w4_pack(ci, si), tops.w4_pack(co, so)), E)
    slots = w4_experts(tops.w4_pack(ci[:8], si[:8]), tops.w4_pack(co[:8], so[:8]))
    there, _ = ta2a_loopback_forward(x, idx, gates, slots, 32, E, 8, M)
    assert torch.equal(here, there)


def test_the_local_path_trains():
    """Gradients of x, the gates and the experts' weights through sort, experts and the way back, against autograd of the
    same layer in 64 bits: f32 products of 32 and 4 terms and 200 rows, so 2^-24 times a few hundred of the terms."""
    from terrace.ta2a_fwd import local_forward
    announce("local trains")
    T, E, k, H = 200, 6, 3, 32
    idx = routing(T, E, k, 8, 0.2)
    g = gen(12)
    x = torch.randn((T, H), generator=g, device=DEV, requires_grad=True)
    gates = torch.rand((T, k), generator=g, device=DEV, requires_grad=True)
    w = (torch.randn((E, H), generator=g, device=DEV) / 4).requires_grad_(True)
    dy = torch.randn((T, H), generator=g, device=DEV)

    def experts(rows, counts):                               # a scale per expert and channel, from the counts alone
        ends = torch.cumsum(counts, 0)
        e = torch.searchsorted(ends, torch.arange(rows.shape[0], device=DEV), right=True).clamp(max=E - 1)
        return rows * w[e]

    y, plan = local_forward(x, idx, gates, experts, E)
    got = torch.autograd.grad(y, (x, gates, w), dy)
    xd, gd, wd = (t.detach().double().requires_grad_(True) for t in (x, gates, w))
    live = (idx >= 0).double()
    yd = ((gd * live)[..., None] * (xd[:, None, :] * wd[idx.clamp(min=0)])).sum(1)
    want = torch.autograd.grad(yd, (xd, gd, wd), dy.double())
    near(y, yd.detach(), (gd.abs()[..., None] * (xd.abs()[:, None, :] * wd.abs()[idx.clamp(min=0)])).sum(1).detach(), 3 * k, "y")
    size = [((gd.abs() * live)[..., None] * wd.abs()[idx.clamp(min=0)] * dy.double().abs()[:, None]).sum(1).detach(),
            (live[..., None] * (xd.abs()[:, None] * wd.abs()[idx.clamp(min=0)] * dy.double().abs()[:, None])).sum(2).detach()]
    terms = ((gd.abs() * live)[..., None] * xd.abs()[:, None] * dy.double().abs()[:, None]).detach()
    size.append(torch.zeros((E, H), dtype=torch.float64, device=DEV).index_add_(0, idx.clamp(min=0).reshape(-1),
                                                                                terms.reshape(-1, H)))
    for name, a, b, m, chain in zip(("x", "gates", "experts"), got, want, size, (3 * k, 2 * H, 3 * T * k)):
        near(a, b, m, chain, name)


@pytest.mark.parametrize("T", [40, 1200])
def test_a_training_step_as_a_graph(T):
    """Forward and backward of all the differentiable operators recorded once and replayed on new inputs, with eager work
    between the replays: every replay gives the eager step's bits."""
    import terrace.ops as tops
    announce("training graph", T)
    E, k, H = 8, 3, 264
    g = gen(T)

    def normal(s, a=1.0, b=0.0):
        return (torch.randn(s, generator=g, device=DEV) * a + b).bfloat16()

    x, gates, idx = normal((T, H)), normal((T, k), 0.2, 0.5), routing(T, E, k, T, 0.2)
    vec = [normal((H,), 0.1, 1.0) for _ in range(3)]
    up = [normal((T, H)), normal((T, H))]
    for t in (x, gates, *vec):
        t.requires_grad_(True)

    def step():
        h0, n0 = tops.block_norm(None, x, pre_weight=vec[0])
        rows, plan = tops.expert_sort(n0, idx, E)
        y = tops.expert_unsort(rows, gates, plan)
        h, n = tops.block_norm(y, h0, vec[1], None, vec[2], scale=0.5)
        return (h.detach(), n.detach(), *torch.autograd.grad((h, n), (x, gates, *vec), up))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(3):
        announce("training graph", T, rep)
        with torch.no_grad():
            x.copy_(normal((T, H)))
            gates.copy_(normal((T, k), 0.2, 0.5))
            idx.copy_(routing(T, E, k, T + rep + 1, 0.2))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_buffers_beyond_four_gigabytes():
    """Offsets past 2^32 bytes in every operator, rows from all over the buffers against the plain formulas."""
    import terrace.ops as tops
    T, H = 300_000, 8192
    announce("large block_norm", T, H)
    g = gen(1)
    y = torch.randn((T, H), generator=g, device=DEV, dtype=torch.bfloat16)
    r = torch.randn((T, H), generator=g, device=DEV, dtype=torch.bfloat16)
    w = torch.ones((H,), device=DEV, dtype=torch.bfloat16)
    pick = torch.tensor([0, 1, 131_072, 262_143, 262_144, T - 1], device=DEV)
    y.requires_grad_(True)
    h, n = tops.block_norm(y, r, w, None, w)
    (dy,) = torch.autograd.grad((h, n), y, (r, r))
    val, mag = norm_oracle(y.detach()[pick], r[pick], w, None, w, 1.0, 1e-6, r[pick], r[pick])
    for name, got in (("h", h), ("n", n), ("d_y", dy)):
        near(got.detach()[pick], val[name], mag[name], H / 64 + 40, name)
    del h, n, dy, y, r
    announce("large expert_sort")
    T, k, H, E = 40_000, 8, 8192, 64                         # 320000 rows of 16 KB
    x = torch.randn((T, H), generator=g, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
    idx = routing(T, E, k, 5)
    rows, plan = tops.expert_sort(x, idx, E)
    where, counts, offsets = sort_oracle(idx, E)
    assert torch.equal(plan.where.cpu(), where)
    at = plan.where[pick[:2].tolist() + [T - 1]]
    assert torch.equal(rows[at.reshape(-1)], x[pick[:2].tolist() + [T - 1]].repeat_interleave(k, 0))
    gates = torch.rand((T, k), generator=g, device=DEV).bfloat16().requires_grad_(True)
    yy = tops.expert_unsort(rows, gates, plan)
    dx, dg = torch.autograd.grad(yy, (x, gates), x.detach())
    tok = torch.tensor([0, T // 2, T - 1], device=DEV)
    xd, gd = x.detach()[tok].double(), gates.detach()[tok].double()
    near(yy.detach()[tok], xd * gd.sum(1, keepdim=True), xd.abs() * gd.sum(1, keepdim=True), 2 * k, "y")
    # the gradient of the rows is rounded before the sort's gradient adds the k of a token: half a bf16 step of each term
    terms = gd[:, :, None] * xd[:, None, :]
    assert bool(((dx[tok].double() - terms.sum(1)).abs() <= 2.0 ** -8 * 1.01 * (terms.abs().sum(1) + terms.sum(1).abs())).all())
    dots = (xd * xd).sum(1, keepdim=True).expand(-1, k)
    near(dg[tok], dots, dots, H / 256 + 20, "d_gates")
    del rows, yy, dx, dg, x
    announce("large w4")
    E, N, K = 300, 4096, 7168                                # 4.4 GB of codes
    codes = torch.randint(0, 256, (E, N, K // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.full((E, N, K // 128), 0.01, device=DEV, dtype=torch.bfloat16)
    packed = tops.w4_pack(codes, scales)
    counts = torch.zeros((E,), dtype=torch.int64, device=DEV)
    counts[0], counts[E - 2], counts[E - 1] = 1, 1, 2
    x = torch.randn((4, K), generator=g, device=DEV).bfloat16()
    out = tops.expert_linear_w4(x, counts, packed)
    for row, e in enumerate((0, E - 2, E - 1, E - 1)):
        q = torch.stack((codes[e] & 15, codes[e] >> 4), -1).flatten(-2).double()
        s = float(scales[0, 0, 0])
        near(out[row], (q - 8) @ x[row].double() * s, (q + 40) @ x[row].double().abs() * s, 2 * 130 + K / 128 + 10, f"row {row}")


def test_w4_zero_points_count_with_their_low_four_bits():
    import terrace.ops as tops
    announce("w4 zeros")
    codes, scales, z, _, _ = w4_case(2, 40, 128, 32, "bf16", True, 3)
    x = torch.randn((5, 128), generator=gen(1), device=DEV).bfloat16()
    counts = torch.tensor([2, 3], device=DEV)
    assert torch.equal(tops.expert_linear_w4(x, counts, tops.w4_pack(codes, scales, z)),
                       tops.expert_linear_w4(x, counts, tops.w4_pack(codes, scales, z | 0xB0)))


def test_expert_sort_rows_without_width():
    import terrace.ops as tops
    announce("no width")
    idx = routing(30, 8, 2, 1)
    wide = torch.randn((30, 16), generator=gen(1), device=DEV)
    rows, plan = tops.expert_sort(wide[:, :0], idx, 8)
    assert rows.shape == (60, 0) and torch.equal(plan.where.cpu(), sort_oracle(idx, 8)[0])
    with pytest.raises(RuntimeError, match="geometry"):
        tops.ExpertPlan(plan.planes, 31, 2, 8)


def test_two_streams_at_once():
    import terrace.ops as tops
    announce("two streams")
    idx = [routing(900, 16, 4, s, 0.1) for s in range(2)]
    x = [torch.randn((900, 264), generator=gen(s), device=DEV).bfloat16() for s in range(2)]
    want = [tops.expert_sort(x[i], idx[i], 16)[0] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(tops.expert_sort(x[i], idx[i], 16)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(r, want[i]) for i in range(2) for r in got[i])


def off_boundary(t):
    """The values of ``t``, packed, starting one element behind a 16-byte boundary."""
    flat = torch.empty((t.numel() + 8,), dtype=t.dtype, device=DEV)
    view = flat[1:1 + t.numel()].view(t.shape)
    view.copy_(t)
    assert view.is_contiguous() and view.data_ptr() % 16
    return view


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_the_sort_and_back_off_a_16_byte_boundary(dtype):
    import terrace.ops as tops
    announce("off boundary", dtype)
    T, E, k, H = 70, 9, 3, 64
    g = gen(31)
    idx = off_boundary(routing(T, E, k, 32, 0.2))
    check_sort(off_boundary(torch.randn((T, H), generator=g, device=DEV).to(DT[dtype])), idx, E)
    _, plan = tops.expert_sort(torch.zeros((T, 8), device=DEV), idx, E)
    rows = off_boundary(torch.randn((T * k, H), generator=g, device=DEV).to(DT[dtype])).requires_grad_(True)
    weights = off_boundary(torch.rand((T, k), generator=g, device=DEV).to(DT[dtype])).requires_grad_(True)
    dy = off_boundary(torch.randn((T, H), generator=g, device=DEV).to(DT[dtype]))
    want_y, mag_y, want_rows, want_w, mag_w = unsort_oracle(rows.detach(), weights.detach(), plan, dy)
    y = tops.expert_unsort(rows, weights, plan)
    near(y, want_y, mag_y, 2 * k, "y")
    d_rows, d_w = torch.autograd.grad(y, (rows, weights), dy)
    near(d_rows, want_rows, want_rows.abs(), 1, "d_rows")
    near(d_w, want_w, mag_w, H / 64 + 8 + 10, "d_weights")


def test_gradients_that_arrive_expanded():
    import terrace.ops as tops
    announce("expanded gradients")
    T, E, k, H = 40, 6, 2, 72
    g = gen(41)
    idx = routing(T, E, k, 42, 0.3)
    x = torch.randn((T, H), generator=g, device=DEV).requires_grad_(True)
    w = torch.rand((T, k), generator=g, device=DEV).requires_grad_(True)
    gain = torch.rand((H,), generator=g, device=DEV).requires_grad_(True)

    def leaves(expanded):
        rows, plan = tops.expert_sort(x, idx, E)
        h, n = tops.block_norm(tops.expert_unsort(rows, w, plan), x, None, None, gain)
        one = torch.ones((), device=DEV).expand(T, H)
        d = one if expanded else one.contiguous()
        direct = torch.autograd.grad(rows, x, torch.ones((), device=DEV).expand(rows.shape) if expanded
                                     else torch.ones_like(rows), retain_graph=True)
        return (*direct, *torch.autograd.grad((h, n), (x, w, gain), (d, d)))

    assert all(torch.equal(a, b) for a, b in zip(leaves(True), leaves(False)))
    alive = (idx >= 0).sum(1, keepdim=True).float().expand(T, H)
    assert torch.equal(leaves(True)[0], alive)               # small integers: exact


def test_two_graphs_replayed_in_turn():
    """Each graph keeps its own index, workspaces and results while the other is replayed and eager calls run between."""
    import terrace.ops as tops
    announce("two graphs")
    E, H = 16, 264
    sets = []
    for i, T in enumerate((900, 1500)):                      # the sorting path
        x = torch.randn((T, H), generator=gen(50 + i), device=DEV).bfloat16()
        idx = routing(T, E, 4, 60 + i, 0.1)
        w = torch.rand((T, 4), generator=gen(70 + i), device=DEV).bfloat16()
        sets.append((x, idx, w))

    def step(x, idx, w):
        rows, plan = tops.expert_sort(x, idx, E)
        y = tops.expert_unsort(rows, w, plan)
        return (rows, plan.offsets, *tops.block_norm(y, x, None, None, torch.ones((H,), dtype=x.dtype, device=DEV)))

    graphs = []
    for s in sets:
        step(*s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*s)
        graphs.append((graph, out))
    for rep in range(3):
        announce("two graphs", rep)
        for i, (x, idx, _) in enumerate(sets):
            x.copy_(torch.randn(x.shape, generator=gen(80 + 2 * rep + i), device=DEV).bfloat16())
            idx.copy_(routing(x.shape[0], E, 4, 90 + 2 * rep + i, 0.1))
        for graph, _ in graphs:
            graph.replay()
        want = [step(*s) for s in sets]
        torch.cuda.synchronize()
        for (_, out), eager in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(out, eager))
