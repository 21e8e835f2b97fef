"""The operators around the experts at the edges of what they take: values that are not finite or very large, derivatives
they do not have, handles that do not fit, and sizes on both sides of each choice of kernel."""
from __future__ import annotations

import pytest
import torch

from test_gpu_experts import (DEV, DT, announce, check_norm, check_sort, check_w4, gen, near, norm_inputs, off_boundary,
                              routing, sort_oracle, w4_case)

pytestmark = pytest.mark.gpu


def same(a, b):
    """Equal bits, NaN included."""
    return torch.equal(a.detach().view(torch.uint8), b.detach().view(torch.uint8))


# ---- block_norm without a gradient of n ---------------------------------------------------------------------------
@pytest.mark.parametrize("T,H", [(70, 264), (530, 1001), (40, 9000), (300, 8193)])
@pytest.mark.parametrize("dtype,residual", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("post,gate", [(False, None), (False, "channel"), (False, "token"), (True, "channel"), (True, "token")])
@pytest.mark.parametrize("pre", [False, True])
def test_block_norm_gradient_of_h_alone_keeps_what_is_not_finite_in_its_place(T, H, dtype, residual, post, gate, pre):
    """Only h is differentiated: its gradient does not depend on the residual, and without a post norm on y only through
    the gate's own gradient, so an infinity or a NaN there changes no other bit."""
    import terrace.ops as tops
    announce("block_norm not finite", T, H, dtype, residual, post, gate, pre)
    y, r, wp, gt, wn, dh, _ = norm_inputs(T, H, dtype, residual, True, post, gate, pre, T + H)

    def grads(y, r):
        leaves = {n: t.detach().clone().requires_grad_(True) for n, t in
                  (("y", y), ("residual", r), ("post", wp), ("gate", gt), ("pre", wn)) if t is not None}
        h, _ = tops.block_norm(leaves["y"], leaves["residual"], leaves.get("post"), leaves.get("gate"), leaves.get("pre"),
                               scale=0.75)
        return dict(zip(leaves, torch.autograd.grad(h, list(leaves.values()), dh, allow_unused=True)))

    clean = grads(y, r)
    assert torch.equal(clean["residual"], dh)
    bad = r.clone()
    bad[3, 5], bad[7, H - 1], bad[T - 1, 0] = float("inf"), float("nan"), float("-inf")
    for name, g in grads(y, bad).items():
        if name == "pre":
            assert g is None or not bool(g.ne(0).any())
        else:
            assert same(g, clean[name]), name
    if post:
        return
    bad = y.clone()
    bad[11, 13], bad[20, H - 2] = float("inf"), float("nan")
    got = grads(bad, r)
    assert same(got["residual"], clean["residual"]) and same(got["y"], clean["y"])
    if gate == "channel":
        off = ~got["gate"].isfinite()
        assert off.nonzero()[:, 0].tolist() == [13, H - 2]
        assert same(got["gate"][~off], clean["gate"][~off])
    elif gate == "token":
        off = ~got["gate"][:, 0].isfinite()
        assert off.nonzero()[:, 0].tolist() == [11, 20]
        assert same(got["gate"][~off], clean["gate"][~off])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("gate", ["token", "channel"])
def test_block_norm_gradient_of_h_alone_on_very_large_values(dtype, gate):
    """|y| about 2^66 without a norm: the products with the gradients stay in range, the squares would not."""
    import terrace.ops as tops
    announce("block_norm large", dtype, gate)
    T, H = 60, 520
    y, r, _, gt, _, dh, _ = norm_inputs(T, H, dtype, dtype, True, False, gate, False, 5)
    y, r = y * 2.0 ** 65, r * 2.0 ** 66
    leaves = [t.requires_grad_(True) for t in (y, r, gt)]
    h, n = tops.block_norm(y, r, None, gt, None)
    dy, dr, dg = torch.autograd.grad(h, leaves, dh)
    assert n is None and torch.equal(dr, dh)
    gd, dhd, yd = gt.detach().double(), dh.double(), y.detach().double()
    near(dy, gd * dhd, (gd * dhd).abs(), 2, "d_y")
    terms = yd * dhd
    if gate == "token":
        near(dg, terms.sum(1, keepdim=True), terms.abs().sum(1, keepdim=True), H / 64 + 40, "d_gate")
    else:
        near(dg, terms.sum(0), terms.abs().sum(0), T + 40, "d_gate")


# ---- block_norm over more rows than are fetched one ahead ----------------------------------------------------------
@pytest.mark.parametrize("H", [7168, 7167, 8200, 8195])
@pytest.mark.parametrize("dtype,residual", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("T,gate", [(2049, "token"), (2900, "channel")])
def test_block_norm_of_long_walks(T, H, dtype, residual, gate):
    """More than 2048 groups of rows: every type with aligned and unaligned rows, 8 and 16 elements a lane, a gate per
    token riding with the rows, and walks that end after an odd and after an even number of rows."""
    check_norm(T, H, dtype, residual, True, True, gate, True, seed=T + H)


@pytest.mark.parametrize("T,H,dtype,residual,has_y,post,gate,pre", [
    (33000, 264, "f16", "f32", True, True, "token", True), (36900, 33, "bf16", "bf16", True, True, "token", False),
    (4200, 4096, "f32", "f32", True, False, "channel", True), (4100, 4095, "f16", "f16", True, True, "token", False),
    (16500, 1000, "bf16", "f32", True, False, "token", True), (2051, 7168, "bf16", "bf16", True, True, None, False),
    (2600, 8000, "f32", "f32", False, False, None, True), (2300, 16384, "f32", "f32", True, False, None, True),
    (2100, 16383, "bf16", "bf16", False, False, None, True), (2561, 9000, "f16", "f32", True, True, "token", False),
])
def test_block_norm_of_long_walks_with_one_norm_and_several_rows_a_workgroup(T, H, dtype, residual, has_y, post, gate, pre):
    check_norm(T, H, dtype, residual, has_y, post, gate, pre, seed=T + H)


# ---- forward mode -------------------------------------------------------------------------------------------------
def test_no_operator_drops_a_forward_mode_tangent():
    """Neither in the forward call nor in a backward pass whose incoming gradient carries one."""
    import torch.autograd.forward_ad as fwAD
    import terrace.ops as tops
    announce("forward mode")
    T, E, k, H = 20, 4, 2, 64
    x, idx = torch.randn((T, H), generator=gen(1), device=DEV), routing(T, E, k, 2)
    rows, plan = tops.expert_sort(x, idx, E)
    w = torch.rand((T, k), generator=gen(3), device=DEV)
    leaf = x.clone().requires_grad_(True)
    results = [tops.expert_sort(leaf, idx, E)[0], tops.expert_unsort(rows.clone().requires_grad_(True), w, plan),
               tops.block_norm(leaf, x)[0]]
    with fwAD.dual_level():
        dual = lambda t: fwAD.make_dual(t, torch.ones_like(t))
        for f in (lambda: tops.expert_sort(dual(x), idx, E), lambda: tops.expert_unsort(dual(rows), w, plan),
                  lambda: tops.expert_unsort(rows, dual(w), plan), lambda: tops.block_norm(dual(x), x),
                  lambda: tops.block_norm(x, x, None, None, dual(x[0]))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                f()
        for out in results:
            with pytest.raises(RuntimeError, match="forward-mode"):
                out.backward(dual(torch.ones_like(out)))
        again, _ = tops.expert_sort(x, idx, E)               # a level alone changes nothing
    assert torch.equal(again, rows)


# ---- 4-bit products of rows that are not finite or very large ------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("E,N,K,group,zeros,swiglu,counts", [
    (1, 40, 1024, 128, False, False, [1]), (1, 256, 96, 32, True, False, [5]), (2, 50, 192, 64, True, True, [16, 15]),
    (3, 33, 288, 32, False, False, [0, 9, 4]), (4, 64, 2048, 128, False, True, [1, 0, 0, 6]),
    (2, 11000, 160, 32, True, True, [130, 40]), (3, 20000, 128, 128, False, False, [20, 33, 1]),
    (1, 16400, 96, 32, False, True, [250]), (2, 24010, 448, 64, True, False, [64, 64]),
])
def test_w4_products_of_rows_that_are_not_finite_or_very_large(E, N, K, group, zeros, swiglu, counts, dtype):
    """An infinite input gives what the definition gives -- an infinity, or NaN where its weight is 0 -- a NaN gives NaN,
    very large inputs a finite result where there is one, and the other rows keep their bits."""
    import terrace.ops as tops
    announce("w4 not finite", E, N, K, group, dtype, zeros, swiglu, counts)
    codes, scales, z, weight, size = w4_case(E, N, K, group, dtype, zeros, N + K)
    packed = tops.w4_pack(codes, scales, z)
    P = sum(counts)
    tokens = torch.tensor(counts, device=DEV)
    clean = torch.randn((P, K), generator=gen(K), device=DEV).to(DT[dtype])
    expert = [e for e, c in enumerate(counts) for _ in range(c)]
    x = clean.clone()
    bad = {0: [float("inf")], P - 1: [float("-inf"), float("inf")], P // 2: [float("nan")]}
    for n, (row, values) in enumerate(bad.items()):
        for i, v in enumerate(values):
            x[row, (37 * n + 61 * i + K - 1) % K] = v
    large = [r for r in (1, P - 2) if 0 <= r < P and r not in bad] if dtype == "bf16" and not swiglu else []
    for row in large:                                        # products with 16 + code pass 2^128, their sums here do not
        x[row] = (clean[row].float() * 2.0 ** 122).bfloat16()
    out = tops.expert_linear_w4(x, tokens, packed, swiglu=swiglu)
    ref = tops.expert_linear_w4(clean, tokens, packed, swiglu=swiglu)
    rest = torch.tensor([r not in bad and r not in large for r in range(P)], device=DEV)
    assert same(out[rest], ref[rest])
    for row in [*bad, *large]:
        xd = x[row].double()
        want = (xd * weight[expert[row]]).sum(-1)
        if swiglu:
            g, u = want[:N // 2], want[N // 2:]
            want = g * torch.sigmoid(g) * u
        got, inf = out[row].double(), want.isinf()
        assert torch.equal(got.isnan(), want.isnan()), row
        assert torch.equal(got[inf], want[inf]), row
        fin = want.isfinite()
        if row in large:
            assert bool(fin.all())
            near(out[row], want, xd.abs() @ size[expert[row]].T, K + 2 * (group + 2) + K / group + 10, "large")
        else:                                                # one infinity or NaN reaches every result of its row
            assert not bool(fin.any())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("E,N,K,group,zeros,swiglu,counts", [
    (1, 16400, 192, 64, False, False, [200]), (2, 16400, 256, 128, False, True, [140, 130]), (1, 16390, 160, 32, False, False, [129]),
    (2, 24010, 320, 64, False, False, [128, 128]), (2, 24010, 320, 64, False, True, [127, 127]),      # 64 rows a tile, and 32
    (1, 16400, 192, 64, True, False, [200]), (2, 16400, 256, 128, True, True, [140, 130]),            # zero points: 32
    (3, 22000, 96, 32, True, False, [9, 9, 9]), (33, 2048, 64, 64, False, False, [8] * 33), (33, 2048, 64, 64, False, True, [9] * 33),
])
def test_w4_products_on_both_sides_of_each_choice_of_kernel(E, N, K, group, zeros, swiglu, counts, dtype):
    check_w4(E, N, K, group, dtype, zeros, swiglu, counts, 5, E + N)


def test_w4_products_of_a_long_prompt():
    """300000 rows over 256 experts of 7168 columns: more 16 x 16 tiles than one launch has workgroups, in far fewer of the
    tiles that run."""
    import terrace.ops as tops
    E, N, K, P = 256, 7168, 32, 300_000
    announce("w4 long", E, N, K, P)
    codes, scales, _, weight, size = w4_case(E, N, K, 32, "bf16", False, 1)
    packed = tops.w4_pack(codes, scales)
    counts = torch.randint(1000, 1300, (E,), generator=gen(2), device=DEV)
    live = int(counts.sum())
    assert live < P - 100
    x = torch.randn((P, K), generator=gen(3), device=DEV).bfloat16()
    out = tops.expert_linear_w4(x, counts, packed)
    assert out.shape == (P, N) and not bool(out[live:].any())
    ends = torch.cumsum(counts, 0)
    for row in (0, int(ends[0]) - 1, int(ends[0]), 131_071, 131_072, live - 1):
        e = int(torch.searchsorted(ends, torch.tensor([row], device=DEV), right=True))
        xd = x[row].double()
        near(out[row], xd @ weight[e].T, xd.abs() @ size[e].T, 2 * 34 + 1 + 10, f"row {row}")


def test_a_handle_of_4_bit_weights_stored_and_built_again():
    import terrace.ops as tops
    announce("w4 handle")
    codes, scales, z, _, _ = w4_case(3, 40, 160, 32, "f16", True, 9)
    w = tops.w4_pack(codes, scales, z)
    x, counts = torch.randn((7, 160), generator=gen(1), device=DEV).half(), torch.tensor([3, 0, 4], device=DEV)
    want = tops.expert_linear_w4(x, counts, w)
    planes = [t.cpu().to(DEV) for t in (w.codes, w.scales, w.zeros)]
    again = tops.W4Weights(*planes, w.n_experts, w.N, w.K, w.group, w.dtype)
    assert torch.equal(tops.expert_linear_w4(x, counts, again), want)
    for name, value in (("N", 56), ("n_experts", 4), ("codes", planes[0][:-1024]), ("zeros", planes[2][1:])):
        bad = tops.W4Weights(*planes, w.n_experts, w.N, w.K, w.group, w.dtype)
        tops.expert_linear_w4(x, counts, bad)
        setattr(bad, name, value)
        with pytest.raises(RuntimeError, match="W4Weights"):
            tops.expert_linear_w4(x, counts if name != "n_experts" else torch.tensor([3, 0, 4, 0], device=DEV), bad)


# ---- the one-launch sort of rows of many pieces ---------------------------------------------------------------------
@pytest.mark.parametrize("T,k,H,dtype,off", [
    (512, 8, 7167, "bf16", False), (512, 8, 7168, "bf16", True), (1, 8, 40001, "f16", False), (1000, 4, 2049, "f32", False),
    (1000, 4, 5000, "f32", True), (2048, 1, 9001, "bf16", False), (120, 17, 4099, "f16", False), (3, 40, 3001, "f32", True),
    (513, 8, 1001, "bf16", False), (1025, 4, 515, "f16", True), (3000, 3, 1001, "f32", True), (2100, 2, 7167, "bf16", False),
])
def test_expert_sort_rows_of_many_pieces(T, k, H, dtype, off):
    """Odd widths and bases off a boundary, where a row is moved in pieces of few bytes; both the one-launch form, whose
    workgroups then take several pieces each, and the sorting path."""
    announce("expert_sort pieces", T, k, H, dtype, off)
    x = torch.randn((T, H), generator=gen(T + H), device=DEV).to(DT[dtype])
    check_sort(off_boundary(x) if off else x, routing(T, 60, k, T, 0.1), 60)


def test_expert_sort_rows_of_megabytes():
    """2048 rows of a million and one elements of two bytes: 4097 pieces a row."""
    import terrace.ops as tops
    T, H = 2048, 1_048_577
    announce("expert_sort megabytes", T, H)
    x = torch.randint(-30000, 30000, (T, H), generator=gen(1), device=DEV, dtype=torch.int16)
    idx = routing(T, 16, 1, 2, 0.1)
    rows, plan = tops.expert_sort(x, idx, 16)
    where, _, offsets = sort_oracle(idx, 16)
    assert torch.equal(plan.where.cpu(), where)
    live = (where[:, 0] >= 0).nonzero()[:, 0].to(DEV)
    for part in live.split(256):
        assert torch.equal(rows[plan.where[part, 0]], x[part])
    assert not bool(rows[int(offsets[-1]):].any())


# ---- many tokens --------------------------------------------------------------------------------------------------
def test_expert_unsort_gradient_of_nine_million_tokens():
    """As many as the forward call takes: more workgroups than 2^31 threads."""
    import terrace.ops as tops
    T, H = 9_000_000, 8
    announce("expert_unsort tokens", T, H)
    idx = torch.randint(-1, 5, (T, 1), generator=gen(1), device=DEV)
    _, plan = tops.expert_sort(torch.zeros((T, 0), device=DEV), idx, 5)
    rows = torch.randn((T, H), generator=gen(2), device=DEV).bfloat16().requires_grad_(True)
    weights = torch.rand((T, 1), generator=gen(3), device=DEV).bfloat16().requires_grad_(True)
    dy = torch.randn((T, H), generator=gen(4), device=DEV).bfloat16()
    y = tops.expert_unsort(rows, weights, plan)
    d_rows, d_w = torch.autograd.grad(y, (rows, weights), dy)
    live, at = plan.where[:, 0] >= 0, plan.where[:, 0].clamp(min=0)
    want = torch.where(live[:, None], rows.detach().double()[at] * weights.detach().double(), 0.0)
    near(y.detach(), want, want.abs(), 2, "y")
    want = torch.zeros((T, H), device=DEV)
    want[at[live]] = (weights.detach().float() * dy.float())[live]
    near(d_rows, want.double(), want.double().abs(), 1, "d_rows")
    terms = torch.where(live[:, None], rows.detach().double()[at] * dy.double(), 0.0)
    near(d_w, terms.sum(1, keepdim=True), terms.abs().sum(1, keepdim=True), H + 10, "d_weights")


def test_expert_unsort_refuses_a_gradient_it_could_not_compute():
    import terrace.ops as tops
    T = (1 << 24) - 1024
    announce("expert_unsort tokens refused", T)
    plan = tops.ExpertPlan(torch.full((T + 2 * 2 + 3,), -1, dtype=torch.int64, device=DEV), T, 1, 2)
    rows = torch.zeros((T, 1), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    with pytest.raises(RuntimeError, match="gradients for up to"):
        tops.expert_unsort(rows, None, plan)


# ---- layouts ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T", [60, 3000])
def test_rows_on_a_kilobyte_pitch_carry_gradients(T):
    import terrace.ops as tops
    announce("pitched gradient", T)
    H, k, E = 480, 3, 7
    x = torch.randn((T, 512), generator=gen(1), device=DEV).bfloat16()[:, :H].requires_grad_(True)
    idx = routing(T, E, k, 2, 0.2)
    rows, plan = tops.expert_sort(x, idx, E)
    assert rows.stride(0) == 512
    packed, _ = tops.expert_sort(x.detach().contiguous(), idx, E)
    assert torch.equal(rows, packed)
    w = torch.rand((T, k), generator=gen(3), device=DEV).bfloat16()
    dy = torch.randn((T, H), generator=gen(4), device=DEV).bfloat16()
    (dx,) = torch.autograd.grad(tops.expert_unsort(rows * 2, w, plan), x, dy)
    leaf = packed.clone().requires_grad_(True)
    (d_rows,) = torch.autograd.grad(tops.expert_unsort(leaf * 2, w, plan), leaf, dy)
    live = plan.where >= 0
    terms = torch.where(live[..., None], d_rows.double()[plan.where.clamp(min=0)], 0.0)
    near(dx, terms.sum(1), terms.abs().sum(1), k, "dx")


def test_gradients_of_rows_without_width():
    import terrace.ops as tops
    announce("no width gradient")
    idx = routing(30, 8, 2, 1, 0.3)
    x = torch.zeros((30, 0), device=DEV, requires_grad=True)
    w = torch.rand((30, 2), generator=gen(2), device=DEV).requires_grad_(True)
    rows, plan = tops.expert_sort(x, idx, 8)
    y = tops.expert_unsort(rows, w, plan)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros((30, 0), device=DEV))
    assert y.shape == dx.shape == (30, 0) and dw.shape == (30, 2) and not bool(dw.any())


def test_a_copied_handle_of_4_bit_weights():
    import copy
    import pickle
    import terrace.ops as tops
    announce("w4 handle copied")
    codes, scales, _, _, _ = w4_case(1, 32, 64, 32, "bf16", False, 1)
    w = tops.w4_pack(codes, scales)
    x = torch.randn((3, 64), generator=gen(1), device=DEV).bfloat16()
    want = tops.expert_linear_w4(x, None, w)
    for other in (copy.copy(w), copy.deepcopy(w), pickle.loads(pickle.dumps(w))):
        assert torch.equal(tops.expert_linear_w4(x, None, other), want)


def test_function_transforms_are_refused_and_not_ignored():
    """torch.func hands the operators wrapped tensors, whose memory they cannot address."""
    import terrace.ops as tops
    announce("function transforms")
    x, v = torch.randn((6, 32), generator=gen(1), device=DEV), torch.ones(32, device=DEV)
    idx = routing(6, 4, 2, 1)
    for f in (lambda t: tops.block_norm(t, x, v)[0], lambda t: tops.expert_sort(t, idx, 4)[0]):
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (x,), (x,))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(t).sum())(x)
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x[None].expand(2, -1, -1).contiguous())
