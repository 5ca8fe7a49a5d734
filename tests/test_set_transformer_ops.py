"""ops.diff_attention, rms_norm, rms_norm_quant and dropout against their definitions in 64 bits, at the sizes, masks and layouts where
they can go wrong.  Tolerances are worst-case bounds worked out from the kernels' roundings (the functions ``*_bound`` below), not measured."""
import ctypes
import math
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from hit_adv_amd import _lib, ops

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24  # half a step of fp32


def half_step(t):
    return torch.finfo(t).eps / 2


def smallest(t):
    return float(torch.finfo(t).smallest_normal)


def check(got, ref, bound, what):
    """|got - ref| <= bound element by element (no NaN in either)."""
    got, ref = got.detach().double().cpu(), ref.detach().double().cpu()
    assert got.shape == ref.shape, what
    assert bool(torch.isfinite(got).all()), "%s: %d values are not finite" % (what, int((~torch.isfinite(got)).sum()))
    over = (got - ref).abs() - torch.as_tensor(bound).double().cpu().expand_as(ref)
    assert float(over.max()) <= 0 if over.numel() else True, "%s: over its bound by %.3g (|ref| there %.3g)" % (
        what, float(over.max()), float(ref.abs().reshape(-1)[over.reshape(-1).argmax()]))


# ---------------------------------------------------------------------------------------------------------------- differential attention
def attention_reference(q, k, v, lam, causal=False, lengths=None, scale=None, dout=None):
    """Definition in 64 bits, and what the bounds need."""
    q, k, v, lam = (x.detach().double().cpu() for x in (q, k, v, lam))
    B, Nq, H, _, D = q.shape
    Nk, Hkv = k.shape[1], k.shape[2]
    G, scale = H // Hkv, D ** -0.5 if scale is None else scale
    hidden = torch.zeros(B, 1, 1, Nq, Nk, dtype=torch.bool)
    j = torch.arange(Nk)
    if causal:
        hidden = hidden | (j[None, :] > torch.arange(Nq)[:, None] + (Nk - Nq))
    if lengths is not None:
        gone = j[None, :] >= lengths.cpu()[:, None]
        hidden = hidden | gone.view(B, 1, 1, 1, Nk)
        k, v = k.masked_fill(gone.view(B, Nk, 1, 1, 1), 0.), v.masked_fill(gone.view(B, Nk, 1, 1), 0.)
    kk, vv = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
    S = torch.einsum("bihmd,bjhmd->bhmij", q, kk) * scale
    dotabs = torch.einsum("bihmd,bjhmd->bhmij", q.abs(), kk.abs()) * abs(scale)
    empty = hidden.all(-1, keepdim=True)
    P = torch.softmax(S.masked_fill(hidden & ~empty, -math.inf), -1).masked_fill(empty, 0.).masked_fill(hidden, 0.)
    l = (lam if lam.dim() and lam.numel() > 1 else lam.reshape(1).expand(H)).view(1, H, 1, 1)
    A = P[:, :, 0] - l * P[:, :, 1]
    r = SimpleNamespace(out=torch.einsum("bhij,bjhd->bihd", A, vv), P=P, l=l, vv=vv, kk=kk, q=q, scale=scale, D=D, Nk=Nk, G=G,
                        top=float((dotabs.masked_fill(hidden, 0.)).max()) if Nk else 0.)
    if dout is not None:
        g = dout.detach().double().cpu()
        dP = torch.einsum("bihd,bjhd->bhij", g, vv).masked_fill(hidden[:, :, 0], 0.)
        rr = (P * dP[:, :, None]).sum(-1)
        sign = torch.stack([torch.ones_like(l), -l], 2)
        dS = P * (dP[:, :, None] - rr[..., None]) * sign
        r.dP, r.r, r.g, r.sign = dP, rr, g, sign
        r.dq = torch.einsum("bhmij,bjhmd->bihmd", dS, kk) * scale
        r.dk = (torch.einsum("bhmij,bihmd->bjhmd", dS, q) * scale).view(B, Nk, Hkv, G, 2, D).sum(3)
        r.dv = torch.einsum("bhij,bihd->bjhd", A, g).view(B, Nk, Hkv, G, 2 * D).sum(3)
        d = -rr[:, :, 1].sum((0, 2))
        r.dlam = d if lam.numel() > 1 or (lam.dim() == 1 and H == 1) else d.sum().reshape(lam.shape)
    return r


def rounding(t, r, terms):
    """(relative error of an input product's sum of |terms|, of a map's value, of a map's product)."""
    # fp32 inputs: three truncated bf16 pieces, dropped products below 2 2^-7 2^-15 + 2^-30 < 2^-20; 16-bit inputs: exact products.
    # A sum of n terms in fp32: n 2^-23 at worst (the matrix cores truncate)
    e_in = (2.0 ** -20 if t is F32 else 0.) + (2 * r.D + 8) * 2.0 ** -23
    # P = 2^(s - max - log2 sum): the error of s in units of log2 (the products', its scaling, three subtractions at |s| <= 2 top log2 e),
    # exp2 and log2 (2 ulp each), the sum of Nk terms
    top = 1.4427 * r.top
    e_p = math.log(2) * 2 * (top * (e_in + 2 * U) + 8 * top * U + 64 * U) + (r.Nk + 8) * U
    # the map as an operand: two bf16 pieces to nearest (2^-18), or three truncated (2^-20); fp16's second operand drops 2^-8 2^-7
    e_m = 2.0 ** -20 if t is F32 else 2.0 ** -17 if t is BF16 else 2.0 ** -14
    return e_in, e_p, e_m + terms * 2.0 ** -23


def attention_bounds(t, r, grads):
    e_in, e_p, e_m = rounding(t, r, r.Nk + 8)
    e = 2 * (e_p + e_m) + 8 * U
    Pa = r.P[:, :, 0] + r.l.abs() * r.P[:, :, 1]
    b = {"out": half_step(t) * r.out.abs() + e * torch.einsum("bhij,bjhd->bihd", Pa, r.vv.abs()) + smallest(t)}
    if not grads:
        return b
    B, Nk, Hkv, G = r.vv.shape[0], r.Nk, r.vv.shape[2] // r.G, r.G
    rows = r.q.shape[1] * r.G
    e_sum = 2 * (e_p + (rows + 8) * 2.0 ** -23 + (2.0 ** -20 if t is F32 else 2.0 ** -14 if t is F16 else 2.0 ** -17)) + 8 * U
    b["dv"] = half_step(t) * r.dv.abs() + e_sum * torch.einsum("bhij,bihd->bjhd", Pa, r.g.abs()).view(B, Nk, Hkv, G, -1).sum(3) + smallest(t)
    dPa = torch.einsum("bihd,bjhd->bhij", r.g.abs(), r.vv.abs())  # |dO| |V|: what dP's error goes by
    e_r = ((2 * e_p + e_in + (r.Nk + 8) * U) * (r.P * dPa[:, :, None])).sum(-1, keepdim=True)
    # dS = P (dP - r): P's error on the difference, and P times the two errors; then its pieces
    dS = r.P * (r.dP[:, :, None] - r.r[..., None]).abs()
    e_ds = (2 * e_p * dS + 1.001 * r.P * (e_in * dPa[:, :, None] + e_r + 2 * U * (r.dP[:, :, None].abs() + r.r[..., None].abs()))) * r.sign.abs()
    dS = dS * r.sign.abs()
    b["dq"] = half_step(t) * r.dq.abs() + 1.01 * abs(r.scale) * torch.einsum("bhmij,bjhmd->bihmd", e_ds + e_m * dS, r.kk.abs()) + smallest(t)
    b["dk"] = half_step(t) * r.dk.abs() + 1.01 * abs(r.scale) * torch.einsum("bhmij,bihmd->bjhmd", e_ds + e_sum * dS, r.q.abs()).view(
        B, Nk, Hkv, G, 2, r.D).sum(3) + smallest(t)
    d = e_r[:, :, 1, :, 0].sum((0, 2)) + 2 * U * r.dlam.abs().max()
    b["dlam"] = d if r.dlam.numel() > 1 or d.numel() == 1 else d.sum()
    return b


def make(t, B, Nq, Nk, H, Hkv, D, seed=0, lam_n=None, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(t).to(device)  # noqa: E731
    lam = (torch.rand(H if lam_n is None else lam_n, generator=g) * 0.6 + 0.2).to(device)
    return n(B, Nq, H, 2, D), n(B, Nk, Hkv, 2, D), n(B, Nk, Hkv, 2 * D), lam, n(B, Nq, H, 2 * D)


def lengths_of(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


CASES = [  # B, Nq, Nk, H, Hkv, D, causal, lengths, lam_n
    (1, 1, 1, 1, 1, 8, False, None, 1),
    (2, 1, 2, 2, 1, 64, True, None, None),
    (1, 2, 1, 1, 1, 16, True, None, None),              # the first query sees nothing
    (3, 1, 300, 6, 2, 32, True, (300, 1, 0), None),     # single tokens over a cache; one sequence is empty
    (2, 3, 1000, 14, 2, 40, True, (1000, 517), 1),      # a few tokens, 7 heads a group
    (2, 33, 31, 2, 2, 24, False, None, None),
    (1, 32, 32, 4, 4, 32, False, None, None),
    (2, 127, 129, 3, 1, 48, True, (129, 64), None),
    (2, 200, 70, 2, 2, 64, True, None, None),           # 130 empty rows
    (3, 96, 160, 8, 4, 56, False, (160, 33, 5), None),
    (1, 257, 257, 4, 2, 64, True, None, 1),
    (2, 64, 64, 65, 1, 8, False, (64, 7), None),        # more heads in a group than a tile has rows
]


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(str(v) for v in c[:6]))
def test_diff_attention_and_its_gradients(t, case):
    B, Nq, Nk, H, Hkv, D, causal, lens, lam_n = case
    q, k, v, lam, g = make(t, B, Nq, Nk, H, Hkv, D, seed=Nk + D, lam_n=lam_n)
    lengths = lengths_of(*lens) if lens else None
    r = attention_reference(q, k, v, lam, causal, lengths, dout=g)
    b = attention_bounds(t, r, True)
    with torch.no_grad():
        check(ops.diff_attention(q, k, v, lam, causal=causal, key_lengths=lengths), r.out, b["out"], "out (no gradient)")
    leaves = [x.requires_grad_() for x in (q, k, v, lam)]
    out = ops.diff_attention(*leaves, causal=causal, key_lengths=lengths)
    assert out.dtype == t and tuple(out.shape) == (B, Nq, H, 2 * D)
    check(out, r.out, b["out"], "out")
    for name, got in zip(("dq", "dk", "dv", "dlam"), torch.autograd.grad(out, leaves, g)):
        check(got, getattr(r, name), b[name], name)


MANY_ROWS_SPLIT = [  # few parts of the keys, joined for many rows at once
    (1, 70, 1100, 4, 2, 40, True, (1037,), None),
    (2, 300, 1500, 2, 2, 64, False, (1500, 0), 1),
    (1, 33, 600, 3, 3, 8, True, None, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("case", MANY_ROWS_SPLIT, ids=lambda c: "x".join(str(v) for v in c[:6]))
def test_diff_attention_many_rows_over_split_keys(t, case):
    test_diff_attention_and_its_gradients(t, case)


@pytest.mark.gpu
def test_diff_attention_gradients_against_differences():
    """Directional derivatives of sum(out g) by central differences of the 64-bit definition (independent of the backward formulas above)."""
    q, k, v, lam, g = make(F32, 1, 9, 11, 2, 1, 8, seed=5)
    leaves = [x.requires_grad_() for x in (q, k, v, lam)]
    grads = torch.autograd.grad(ops.diff_attention(*leaves, causal=True), leaves, g)
    h = 1e-5
    for i, (x, got) in enumerate(zip(leaves, grads)):
        d = torch.randn(x.shape, generator=torch.Generator().manual_seed(i), dtype=torch.float64)
        f = lambda e: (attention_reference(*[(y.detach().double().cpu() + (e * d if y is x else 0.)) for y in leaves], causal=True).out  # noqa: E731
                       * g.double().cpu()).sum()
        num = float((f(h) - f(-h)) / (2 * h))
        ana = float((got.double().cpu() * d).sum())
        # h^2 times a third derivative of order 100 |num|, and the fp32 gradients' own 2^-18
        assert abs(num - ana) <= (100 * h * h + 2.0 ** -18) * float((got.double().cpu().abs() * d.abs()).sum()) + 1e-8, (i, num, ana)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16])
def test_diff_attention_one_visible_key_has_no_score_gradient(t):
    """Where a row sees one key its two probabilities are 1 and dS vanishes exactly, in either kernel."""
    q, k, v, lam, g = make(t, 2, 40, 50, 4, 2, 32, seed=1)
    lengths = lengths_of(1, 1)
    leaves = [x.requires_grad_() for x in (q, k, v, lam)]
    dq, dk, dv, _ = torch.autograd.grad(ops.diff_attention(*leaves, key_lengths=lengths), leaves, g)
    assert not dq.any() and not dk.any() and bool(dv[:, :1].any()) and not dv[:, 1:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_diff_attention_views_caches_and_what_lies_behind_the_lengths(t):
    """A slice of a larger cache (its strides, another order of axes, q inside a fused projection) gives the bits of its contiguous copy; what
    the cache holds behind the lengths (NaN, infinities) is not seen; misaligned and odd-strided views are copied."""
    B, Nq, Nk, H, Hkv, D = 2, 5, 150, 4, 2, 32
    q, k, v, lam, g = make(t, B, Nq, Nk, H, Hkv, D, seed=3)
    lengths = lengths_of(150, 61)
    want = ops.diff_attention(q, k, v, lam, causal=True, key_lengths=lengths)
    cache = torch.full((B, Hkv, 400, 4 * D), float("nan"), device="cuda", dtype=t)
    kc, vc = cache[:, :, 100:250, :2 * D].unflatten(-1, (2, D)).permute(0, 2, 1, 3, 4), cache[:, :, 100:250, 2 * D:].permute(0, 2, 1, 3)
    kc.copy_(k), vc.copy_(v)
    kc[1, 61:], vc[1, 61:] = float("inf"), float("nan")
    qf = torch.randn(B, Nq, 3, H * 2 * D, device="cuda").to(t)
    qf[:, :, 1] = q.flatten(2)
    qv = qf[:, :, 1].view(B, Nq, H, 2, D)
    assert torch.equal(ops.diff_attention(qv, kc, vc, lam, causal=True, key_lengths=lengths), want)
    assert torch.equal(ops.diff_attention(qv, kc, vc, lam, causal=True, key_lengths=lengths.long()), want)
    off = torch.empty(q.numel() + 1, device="cuda", dtype=t)[1:].view_as(q).copy_(q)                     # not 16-byte aligned
    odd = torch.empty(*q.shape[:-1], D + 1, device="cuda", dtype=t)[..., :D].copy_(q)                     # odd row stride
    swap = q.transpose(3, 4).contiguous().transpose(3, 4)                                                # last axis strided
    for x in (off, odd, swap):
        assert torch.equal(ops.diff_attention(x, kc, vc, lam, causal=True, key_lengths=lengths), want)
    one = k[:, :, :1].expand(B, Nk, 4, 2, D)                                                             # a broadcast head: stride 0
    vone = v[:, :, :1].expand(B, Nk, 4, 2 * D)
    assert torch.equal(ops.diff_attention(q, one, vone, lam), ops.diff_attention(q, one.contiguous(), vone.contiguous(), lam))
    # gradients: of views as of copies, nothing from behind the lengths
    leaves = [x.detach().clone().requires_grad_() for x in (q, k, v, lam)]
    ref = torch.autograd.grad(ops.diff_attention(*leaves, causal=True, key_lengths=lengths), leaves, g)
    views = [x.detach().requires_grad_() for x in (qv, kc, vc, lam)]
    got = torch.autograd.grad(ops.diff_attention(*views, causal=True, key_lengths=lengths), views, g.transpose(0, 1).contiguous().transpose(0, 1))
    for a, b in zip(got, ref):
        assert torch.equal(a, b)
    assert not got[1][1, 61:].any() and not got[2][1, 61:].any()


@pytest.mark.gpu
def test_diff_attention_extreme_scores_and_scales():
    """Scores of +-1e4 and a scale of 0: no overflow, no NaN; lam of 0 and 1; large values stay what they are in bf16."""
    q, k, v, lam, _ = make(F32, 1, 40, 70, 2, 2, 16, seed=7)
    for s, e in ((0., 0.), (300., 300.), (-2., 2.)):
        r = attention_reference(q, k, v, lam, scale=s)
        check(ops.diff_attention(q, k, v, lam, scale=s), r.out, attention_bounds(F32, r, False)["out"], "scale %g" % s)
    big = (v.to(BF16) * 2.0 ** 100)
    qb, kb = q.to(BF16), k.to(BF16)
    r = attention_reference(qb, kb, big, torch.ones(2))
    check(ops.diff_attention(qb, kb, big, torch.ones(2, device="cuda")), r.out, attention_bounds(BF16, r, False)["out"], "large values")
    same = ops.diff_attention(torch.cat([qb[:, :, :, :1]] * 2, 3), torch.cat([kb[:, :, :, :1]] * 2, 3), big, torch.ones(2, device="cuda"))
    assert not same.any()  # equal maps, lam = 1


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("at", [0, 1500, 4095])
def test_diff_attention_many_small_probabilities_beside_a_large_one(t, at):
    """4095 keys with 2^-18 of the largest one's probability carry the whole output (the large one's value is 0), and the large one comes
    first, in the middle or last; few rows (the keys are split) and many (they are not)."""
    q, k, v, lam, _ = make(t, 1, 64, 4096, 2, 1, 8, seed=17)
    q, k = torch.zeros_like(q), torch.zeros_like(k)
    q[..., 0, 0] = 1.  # (the second map is uniform)
    k[..., 0, 0] = -12.5
    k[:, at, :, 0, 0] = 0.
    v = v.abs()
    v[:, at] = 0.
    for Nq in (1, 64):
        r = attention_reference(q[:, :Nq], k, v, lam * 1e-3, scale=1.)
        assert float(r.out.min()) > 2.0 ** -8  # (about 0.012)
        check(ops.diff_attention(q[:, :Nq], k, v, lam * 1e-3, scale=1.), r.out, attention_bounds(t, r, False)["out"] - smallest(t), "%d rows" % Nq)


@pytest.mark.gpu
def test_diff_attention_subnormal_values():
    """A column that holds one subnormal value everywhere comes out as that value: the mean is off by far less than half of fp16's last step."""
    q, k, v, _, _ = make(F16, 1, 40, 300, 2, 1, 24, seed=18)
    v = torch.arange(1, 49, device="cuda").to(F32).mul(2.0 ** -24).to(F16).expand_as(v).contiguous()
    for Nq in (1, 40):
        assert torch.equal(ops.diff_attention(q[:, :Nq], k, v, torch.zeros(1, device="cuda")), v[:, :1].expand(1, Nq, 2, 48))


@pytest.mark.gpu
def test_diff_attention_empty_axes():
    for B, Nq, Nk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v, lam, g = make(F32, B, Nq, Nk, 2, 1, 8)
        leaves = [x.requires_grad_() for x in (q, k, v, lam)]
        out = ops.diff_attention(*leaves)
        assert tuple(out.shape) == (B, Nq, 2, 16) and not out.any()
        for x, d in zip(leaves, torch.autograd.grad(out, leaves, g)):
            assert d.shape == x.shape and not d.any()


@pytest.mark.gpu
def test_diff_attention_offsets_beyond_32_bits():
    """A cache of 2.2e9 elements per tensor (bf16, 4.5 GB): the last keys are the right ones."""
    Nk, H, D = 1_100_000, 16, 64
    k = torch.empty(1, Nk, H, 2, D, device="cuda", dtype=BF16).normal_(generator=torch.Generator("cuda").manual_seed(1))
    v = torch.empty(1, Nk, H, 2 * D, device="cuda", dtype=BF16).normal_(generator=torch.Generator("cuda").manual_seed(2))
    q, _, _, lam, _ = make(BF16, 1, 1, 1, H, H, D)
    q = q * 4  # a few keys carry most of the weight
    out = ops.diff_attention(q, k, v, lam, causal=True)
    for h in (0, 15):
        P = torch.softmax(torch.einsum("md,jmd->mj", q[0, 0, h].double(), k[0, :, h].double()) * D ** -0.5, -1)
        ref = (P[0] - lam[h].double() * P[1]) @ v[0, :, h].double()
        mag = (P[0] + lam[h].double() * P[1]) @ v[0, :, h].double().abs()
        # 64 splits' and tiles' sums of 2^20 positive terms in fp32: their worst case is not met; 2^-12 leaves 256 half steps of a part's sum
        check(out[0, 0, h], ref, half_step(BF16) * ref.abs() + 2.0 ** -12 * mag, "head %d" % h)
    del k, v


@pytest.mark.gpu
def test_diff_attention_needs_only_what_is_asked_for():
    q, k, v, lam, g = make(F32, 2, 40, 40, 2, 2, 32, seed=9)
    full = [x.detach().clone().requires_grad_() for x in (q, k, v, lam)]
    ref = torch.autograd.grad(ops.diff_attention(*full), full, g)
    for i in range(4):
        leaves = [x.detach().clone() for x in (q, k, v, lam)]
        leaves[i].requires_grad_()
        assert torch.equal(torch.autograd.grad(ops.diff_attention(*leaves), leaves[i], g)[0], ref[i])
    scalar = torch.tensor(0.5, device="cuda", requires_grad=True)
    r = attention_reference(q, k, v, scalar, dout=g)
    d, = torch.autograd.grad(ops.diff_attention(q, k, v, scalar), scalar, g)
    check(d, r.dlam.reshape(()), attention_bounds(F32, r, True)["dlam"].sum().reshape(()), "dlam of one value")
    x = q.detach().clone().requires_grad_()
    with pytest.raises(RuntimeError):
        gx, = torch.autograd.grad(ops.diff_attention(x, k, v, lam).sum(), x, create_graph=True)
        gx.sum().backward()


@pytest.mark.gpu
def test_diff_attention_refusals():
    q, k, v, lam, _ = make(F32, 2, 4, 6, 4, 2, 16)
    bad = [
        (ValueError, (q[..., 0, :], k, v, lam), {}),
        (ValueError, (q, k[:1], v, lam), {}),
        (ValueError, (q, k, v[..., :16], lam), {}),
        (ValueError, (q[:, :, :3], k, v, lam[:3]), {}),                                # 3 heads over 2
        (ValueError, (q, k, v, lam[:3]), {}),
        (ValueError, (q, k, v, lam.view(2, 2)), {}),
        (ValueError, (q[..., :12], k[..., :12], v[..., :24], lam), {}),                # D = 12
        (ValueError, make(F32, 1, 2, 2, 1, 1, 72)[:4], {}),
        (ValueError, (q, k, v, lam), {"key_lengths": lengths_of(1)}),
        (TypeError, (q, k, v, lam), {"key_lengths": torch.ones(2, device="cuda")}),
        (TypeError, (q, k.to(BF16), v, lam), {}),
        (TypeError, (q.double(), k.double(), v.double(), lam), {}),
        (TypeError, (q, k, v, lam.to(BF16)), {}),
        (TypeError, (q, k, v, 0.5), {}),
        (RuntimeError, (q, k.cpu(), v, lam), {}),
    ]
    for kind, args, kw in bad:
        with pytest.raises(kind):
            ops.diff_attention(*args, **kw)


# ---------------------------------------------------------------------------------------------------------------- norm
def norm_reference(x, w, eps, residual=None, dy=None, dsum=None):
    s = x.detach().double().cpu()
    if residual is not None:
        s = (x.detach().float() + residual.detach().float()).to(x.dtype).double().cpu()
    w = w.detach().double().cpu()
    rs = 1 / torch.sqrt(s.pow(2).mean(-1, keepdim=True) + eps)
    r = SimpleNamespace(s=s, n=s * rs, y=s * rs * w, rs=rs)
    if dy is not None:
        dy = dy.detach().double().cpu()
        g = dy * w
        r.dx = rs * (g - r.n * (g * r.n).mean(-1, keepdim=True))
        r.mag = rs * (g.abs() + r.n.abs() * (g * r.n).abs().mean(-1, keepdim=True))
        if dsum is not None:
            r.dx, r.mag = r.dx + dsum.double().cpu(), r.mag + dsum.double().cpu().abs()
        r.dw, r.dwmag = (dy * r.n).reshape(-1, w.numel()).sum(0), (dy * r.n).abs().reshape(-1, w.numel()).sum(0)
    return r


# rows of every team width and its edges, odd widths, one column, one row
SHAPES = [(1, 1), (3, 7), (5, 64), (33, 128), (7, 129), (9, 512), (2, 513), (6, 1000), (1, 1025), (3, 2048), (2, 4095), (4, 4097), (1, 8192),
          (2, 8193), (1, 16384), (1500, 96), (4200, 20)]


@pytest.mark.gpu
@pytest.mark.parametrize("t,tw", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_rms_norm_and_its_gradients(t, tw, rows, cols):
    g = torch.Generator().manual_seed(rows + cols)
    n = lambda: torch.randn(rows, cols, generator=g).to(t).cuda()  # noqa: E731
    for res in (False, True):
        x, residual, dy, dsum = n().requires_grad_(), n().requires_grad_() if res else None, n(), n() if res else None
        w = (torch.rand(cols, generator=g) + 0.5).to(tw).cuda().requires_grad_()
        r = norm_reference(x, w, 1e-5, residual, dy, dsum)
        # 1 / sqrt(mean): half the sum's cols 2^-24 and a few operations; a mean over cols in the gradient
        e = (cols / 2 + 8) * U
        out = ops.rms_norm(x, w, eps=1e-5, residual=residual)
        y, s = out if res else (out, None)
        check(y, r.y, half_step(t) * r.y.abs() + e * r.y.abs() + smallest(t), "y")
        if res:
            assert torch.equal(s.double().cpu(), r.s)
            dx, dr, dw = torch.autograd.grad((y, s), (x, residual, w), (dy, dsum))
            assert torch.equal(dx, dr)
        else:
            dx, dw = torch.autograd.grad(y, (x, w), dy)
        check(dx, r.dx, half_step(t) * r.dx.abs() + (2 * cols + 16) * U * r.mag + smallest(t), "dx")
        check(dw, r.dw, half_step(tw) * r.dw.abs() + (rows + cols / 2 + 16) * U * r.dwmag + smallest(tw), "dw")
        q, scale, *rest = ops.rms_norm_quant(x.detach(), w.detach(), eps=1e-5, residual=residual.detach() if res else None)
        top = r.y.abs().amax(-1) / 448
        check(scale, top, (e + 2 * U) * top, "scale")
        step = torch.maximum(r.y.abs() * 2.0 ** -4, scale.double().cpu()[:, None] * 2.0 ** -10)  # half a step of e4m3, normal or not
        check(q.double() * scale.double()[:, None], r.y, step * (1 + 2.0 ** -10) + 2 * e * r.y.abs(), "q scale")
        if res:
            assert torch.equal(rest[0].double().cpu(), r.s)


@pytest.mark.gpu
def test_rms_norm_layouts_and_special_rows():
    x = torch.randn(3, 5, 100, device="cuda")
    w = torch.ones(100, device="cuda")
    want = ops.rms_norm(x, w)
    assert want.shape == x.shape
    assert torch.equal(ops.rms_norm(x.transpose(0, 1).contiguous().transpose(0, 1), w), want)
    off = torch.empty(x.numel() + 1, device="cuda")[1:].view_as(x).copy_(x)
    assert torch.equal(ops.rms_norm(off, w), want)
    zero = torch.zeros(2, 100, device="cuda", dtype=BF16, requires_grad=True)
    y = ops.rms_norm(zero, w)
    assert not y.any()
    d, = torch.autograd.grad(y, zero, torch.ones_like(y))
    assert bool(torch.isfinite(d).all())
    q, s = ops.rms_norm_quant(zero.detach(), w)
    assert not q.float().any() and bool((s == 1).all())
    bad = x.clone()
    bad[1, 2, 3] = float("nan")
    y = ops.rms_norm(bad, w)
    keep = torch.ones(3, 5, dtype=torch.bool)
    keep[1, 2] = False
    assert bool(y[1, 2].isnan().all()) and torch.equal(y[keep], want[keep])  # the row alone
    q, s = ops.rms_norm_quant(bad, w)
    assert bool(q[1, 2].float().isnan().all())
    for shape in ((0, 100), (4, 0, 100)):
        e = torch.empty(*shape, device="cuda", requires_grad=True)
        we = w.clone().requires_grad_()
        y = ops.rms_norm(e, we)
        gx, gw = torch.autograd.grad(y, (e, we), torch.empty_like(y))
        assert y.shape == e.shape == gx.shape and not gw.any()
    # the sum alone carries a gradient
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    _, s = ops.rms_norm(a, w, residual=b)
    ga, gb = torch.autograd.grad(s, (a, b), x)
    assert torch.equal(ga, x) and torch.equal(gb, x)
    # the output alone
    yy, _ = ops.rms_norm(a, w, residual=b)
    ga, = torch.autograd.grad(yy, a, x)
    r = norm_reference(a, w, 1e-6, b, x)
    check(ga, r.dx, half_step(F32) * r.dx.abs() + 216 * U * r.mag, "dx without a gradient of the sum")


@pytest.mark.gpu
def test_rms_norm_and_dropout_refusals():
    x, w = torch.randn(4, 32, device="cuda"), torch.ones(32, device="cuda")
    rng = torch.tensor([1, 2], device="cuda")
    for kind, f in [
        (ValueError, lambda: ops.rms_norm(x, w[:31])),
        (ValueError, lambda: ops.rms_norm(x, w, residual=x[:3])),
        (ValueError, lambda: ops.rms_norm(x, w, residual=x.to(BF16))),
        (ValueError, lambda: ops.rms_norm(torch.empty(1, 16385, device="cuda"), torch.empty(16385, device="cuda"))),
        (ValueError, lambda: ops.rms_norm(torch.empty(3, 0, device="cuda"), w[:0])),
        (TypeError, lambda: ops.rms_norm(x, w.to(BF16))),
        (TypeError, lambda: ops.rms_norm(x.double(), w.double())),
        (RuntimeError, lambda: ops.rms_norm(x, w.cpu())),
        (RuntimeError, lambda: ops.rms_norm_quant(x.clone().requires_grad_(), w)),
        (ValueError, lambda: ops.dropout(x, 1.5, rng)),
        (ValueError, lambda: ops.dropout(x, -0.1, rng)),
        (ValueError, lambda: ops.dropout(x, float("nan"), rng)),
        (ValueError, lambda: ops.dropout(x, 0.5, rng[:1])),
        (TypeError, lambda: ops.dropout(x, 0.5, rng.int())),
        (RuntimeError, lambda: ops.dropout(x, 0.5, rng.cpu())),
        (ValueError, lambda: ops.dropout(x, 0.5, rng, residual=x[:2])),
    ]:
        with pytest.raises(kind):
            f()


# ---------------------------------------------------------------------------------------------------------------- dropout
def philox_words(n, seed, offset):
    """Philox4x32-10 in numpy, from the published description."""
    b = np.arange((n + 3) // 4, dtype=np.uint64)
    low, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [b & low, b >> sh, np.full_like(b, offset & 0xFFFFFFFF), np.full_like(b, (offset >> 32) & 0xFFFFFFFF)]
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> sh) ^ c[1] ^ np.uint64(k0), p1 & low, (p0 >> sh) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.from_numpy(np.stack(c, 1).reshape(-1)[:n].astype(np.int64))


def test_philox_known_answers():
    """The published vectors of Philox4x32-10: all zeros, all ones."""
    assert [hex(v) for v in philox_words(4, 0, 0).tolist()] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (9, 5), (32, 512), (2047,), (3, 2049), (1000, 1001)], ids=str)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999, 1.0])
def test_dropout_and_its_gradient(t, shape, p):
    g = torch.Generator().manual_seed(len(shape) + shape[0])
    x, r, dy = (torch.randn(*shape, generator=g).to(t).cuda() for _ in range(3))
    seed, offset = -3 + (1 << 40), (1 << 33) + 5
    rng = torch.tensor([seed, offset], device="cuda")
    factor = (philox_words(x.numel(), seed, offset) >= round(p * 2 ** 32)).float().view(shape) * (1 / (1 - p) if p < 1 else 0.)
    for res in (None, r):
        a, b = x.clone().requires_grad_(), res.clone().requires_grad_() if res is not None else None
        y = ops.dropout(a, p, rng, residual=b)
        f = factor.cuda()
        want = a.detach().float() * f
        want = want + res.float() if res is not None else want
        assert torch.equal(y, want.to(t))  # one product, one sum, one rounding: the same bits
        grads = torch.autograd.grad(y, (a,) if res is None else (a, b), dy)
        assert torch.equal(grads[0], (dy.float() * f).to(t))
        if res is not None:
            assert torch.equal(grads[1], dy)


@pytest.mark.gpu
def test_dropout_rng_layouts_and_special_values():
    x = torch.randn(6, 100, device="cuda")
    rng = torch.tensor([11, 0], device="cuda")
    want = ops.dropout(x, 0.3, rng)
    assert torch.equal(ops.dropout(x.t().contiguous().t(), 0.3, rng), want)
    off = torch.empty(601, device="cuda")[1:].view(6, 100).copy_(x)
    assert torch.equal(ops.dropout(off, 0.3, rng), want)
    assert torch.equal(ops.dropout(x, 0.3, torch.tensor([[11, 5], [0, 7]], device="cuda")[:, 0]), want)  # a strided view of a table
    assert not torch.equal(ops.dropout(x, 0.3, rng + torch.tensor([0, 1], device="cuda")) == 0, want == 0)
    inf = torch.full((1000,), float("inf"), device="cuda")
    y = ops.dropout(inf, 0.5, rng)
    assert bool(((y == 0) | (y == float("inf"))).all()) and bool((y == 0).any())
    assert ops.dropout(x[:0], 0.5, rng).shape == (0, 100)
    a = x.clone().requires_grad_()
    y = ops.dropout(a, 0.3, rng)
    rng[1] += 1
    with pytest.raises(RuntimeError):  # the mask of the backward pass would be another one
        y.sum().backward()


# ---------------------------------------------------------------------------------------------------------------- the block
def _block(x, p, rng, causal=False, lengths=None):
    """norm -> q, k, v -> attention -> head norm -> projection -> dropout + residual -> norm with the residual."""
    B, N, C = x.shape
    H = C // 64
    h = torch.matmul(ops.rms_norm(x, p["n1"]), p["qkv"]).view(B, N, 3, C)
    q, k, v = h.unbind(2)
    a = ops.diff_attention(q.view(B, N, H, 2, 32), k.view(B, N, H, 2, 32), v.view(B, N, H, 64), p["lam"], causal=causal, key_lengths=lengths)
    y = torch.matmul(ops.rms_norm(a, p["nh"]).reshape(B, N, C), p["o"])
    s = ops.dropout(y, 0.25, rng, residual=x)
    return ops.rms_norm(s, p["n2"], residual=x)


def _block_params(C, t, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return {"n1": torch.ones(C).cuda(), "qkv": (r(C, 3 * C) * C ** -0.5).to(t).cuda(), "lam": torch.full((C // 64,), 0.4).cuda(),
            "nh": torch.full((64,), 0.5).cuda(), "o": (r(C, C) * C ** -0.5).to(t).cuda(), "n2": torch.ones(C).cuda()}


@pytest.mark.gpu
def test_block_against_64_bits():
    """The operators strung together in fp32 against the same block in 64 bits: outputs and every gradient to 2^-14 of the gradient's norm (each
    of the eight steps is off by < 2^-18 of its own output's norm, test by test above; the norms' 1/r does not magnify here: rms ~ 1)."""
    B, N, C = 2, 70, 128
    p = {k: v.requires_grad_() for k, v in _block_params(C, F32).items()}
    x = torch.randn(B, N, C, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    rng = torch.tensor([5, 9], device="cuda")
    lengths = lengths_of(70, 41)
    y, s = _block(x, p, rng, True, lengths)
    gy, gs = torch.randn(2, B, N, C, generator=torch.Generator().manual_seed(2)).cuda().unbind(0)
    names = sorted(p)
    grads = torch.autograd.grad((y, s), [x] + [p[n] for n in names], (gy, gs))
    d = {n: p[n].detach().double().cpu().requires_grad_() for n in names}
    xd = x.detach().double().cpu().requires_grad_()
    norm = lambda u, w: u * torch.rsqrt(u.pow(2).mean(-1, keepdim=True) + 1e-6) * w  # noqa: E731
    h = (norm(xd, d["n1"]) @ d["qkv"]).view(B, N, 3, C)
    q, k, v = h[:, :, 0].view(B, N, 2, 2, 32), h[:, :, 1].view(B, N, 2, 2, 32), h[:, :, 2].view(B, N, 2, 64)
    S = torch.einsum("bihmd,bjhmd->bhmij", q, k) * 32 ** -0.5
    j = torch.arange(N)
    hidden = (j[None] > j[:, None])[None] | (j[None, None] >= lengths.cpu()[:, None, None])
    P = torch.softmax(S.masked_fill(hidden[:, None, None], -math.inf), -1)
    a = torch.einsum("bhij,bjhd->bihd", P[:, :, 0] - d["lam"].view(-1, 1, 1) * P[:, :, 1], v)
    o = norm(a, d["nh"]).reshape(B, N, C) @ d["o"]
    keep = (philox_words(o.numel(), 5, 9) >= round(0.25 * 2 ** 32)).double().view_as(o)
    sd = xd + o * keep / 0.75 + xd
    yd = norm(sd, d["n2"])
    ref = torch.autograd.grad((yd, sd), [xd] + [d[n] for n in names], (gy.double().cpu(), gs.double().cpu()))
    for what, got, want in [("y", y, yd), ("s", s, sd)] + list(zip(["x"] + names, grads, ref)):
        off = float((got.detach().double().cpu() - want).norm() / want.norm())
        assert off <= 2.0 ** -14, (what, off)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16])
def test_block_captured_into_a_graph(t):
    """Forward and backward captured once and replayed on new inputs, lengths and mask offsets, with eager work between the replays: every
    replay gives the eager call's bits."""
    B, N, C = 3, 100, 128
    p = {k: v.requires_grad_() for k, v in _block_params(C, t).items()}
    x, gy = torch.randn(B, N, C, device="cuda").to(t).requires_grad_(), torch.randn(B, N, C, device="cuda").to(t)
    rng, lengths = torch.tensor([5, 0], device="cuda"), lengths_of(100, 60, 1)
    names = sorted(p)

    def step():
        y, s = _block(x, p, rng, True, lengths)
        return (y, s) + torch.autograd.grad((y, s), [x] + [p[n] for n in names], (gy, gy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(B, N, C, device="cuda"))
        rng[1] = 17 * i + 1
        lengths.copy_(lengths_of(100 - i, 7 * i, 50))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(held, eager):
            assert torch.equal(a, b), i


@pytest.mark.gpu
def test_token_calls_in_two_graphs_and_on_two_streams():
    """Split calls (their scratch) captured into two graphs replayed in turn, and eager calls on two streams at once: the eager bits."""
    sets = [make(BF16, 4, 1, 2000, 8, 2, 64, seed=s) for s in range(2)]
    want = [ops.diff_attention(*s[:4], causal=True) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, held = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            held.append(ops.diff_attention(*s[:4], causal=True))
    for _ in range(3):
        for h in held:
            h.fill_(float("nan"))
        for gr in graphs:
            gr.replay()
        other = ops.diff_attention(*sets[0][:4], causal=True)
        torch.cuda.synchronize()
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1]) and torch.equal(other, want[0])
    got = [None, None]
    for _ in range(10):
        with torch.cuda.stream(side):
            got[1] = ops.diff_attention(*sets[1][:4], causal=True)
        got[0] = ops.diff_attention(*sets[0][:4], causal=True)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_same_bits_on_every_run_and_for_every_neighbour():
    """Two runs agree bit for bit; a cloud's results do not depend on the other clouds of its batch."""
    q, k, v, lam, g = make(F32, 3, 90, 90, 2, 2, 32, seed=4)
    lengths = lengths_of(90, 50, 3)

    def run(sel):
        leaves = [x[sel].detach().clone().requires_grad_() for x in (q, k, v)]
        out = ops.diff_attention(*leaves, lam, key_lengths=lengths[sel])
        return (out,) + torch.autograd.grad(out, leaves, g[sel])
    a, b, one = run(slice(0, 3)), run(slice(0, 3)), run(slice(1, 2))
    for x, y, z in zip(a, b, one):
        assert torch.equal(x, y) and torch.equal(x[1:2], z)


# ---------------------------------------------------------------------------------------------------------------- the layer
def _pct_args(attention):
    return SimpleNamespace(dropout=0.2, attention=attention)


def test_pct_takes_either_attention_and_refuses_another():
    from hit_adv_amd.model.pct import DA_Layer, Pct, SA_Layer
    assert isinstance(Pct(SimpleNamespace(dropout=0.2)).pt_last.sa1, SA_Layer)
    m = Pct(_pct_args("differential"))
    assert isinstance(m.pt_last.sa4, DA_Layer)
    seeds = {int(getattr(m.pt_last, "sa%d" % i).rng[0]) for i in range(1, 5)}
    assert len(seeds) == 4  # a mask of its own in every layer
    with pytest.raises(ValueError):
        Pct(_pct_args("none"))
    with pytest.raises(ValueError):
        DA_Layer(96)


@pytest.mark.gpu
def test_da_layer_on_the_gpu_is_its_plain_form():
    """DA_Layer's GPU path against its plain CPU path in 64 bits, eval and training without dropout: output and the input's gradient to 2^-14
    of their norms (as in the block's test), weight gradients in training."""
    from hit_adv_amd.model.pct import DA_Layer
    torch.manual_seed(0)
    plain = DA_Layer(256, dropout=0.).double()
    gpu = DA_Layer(256, dropout=0.).cuda()
    gpu.load_state_dict(plain.float().state_dict())
    plain = plain.double()
    x, g = torch.randn(2, 256, 80), torch.randn(2, 256, 80)
    for mode in (False, True):
        plain.train(mode), gpu.train(mode)
        a, b = x.double().requires_grad_(), x.cuda().requires_grad_()
        ya, yb = plain(a), gpu(b)
        wrt_a, wrt_b = [a] + (list(plain.parameters()) if mode else []), [b] + (list(gpu.parameters()) if mode else [])
        for u, w in zip([ya] + list(torch.autograd.grad(ya, wrt_a, g.double())), [yb] + list(torch.autograd.grad(yb, wrt_b, g.cuda()))):
            assert float((u - w.double().cpu()).norm() / u.norm()) <= 2.0 ** -14


@pytest.mark.gpu
def test_da_layer_draws_new_masks_and_repeats_them_backward():
    from hit_adv_amd.model.pct import DA_Layer
    torch.manual_seed(0)
    m = DA_Layer(64, dropout=0.5).cuda().train()
    x = torch.randn(2, 64, 40, device="cuda", requires_grad=True)
    y1 = m(x)
    y2 = m(x)
    z1, z2 = y1 == x, y2 == x  # a dropped element leaves the residual
    assert 0.4 < float(z1.float().mean()) < 0.6 and not torch.equal(z1, z2)
    (y1.sum() + y2.sum()).backward()  # two forwards before a backward
    m.eval()
    assert torch.equal(m(x), m(x)) and not bool((m(x) == x).float().mean() > 0.1)


@pytest.mark.gpu
def test_pct_with_differential_attention_under_attack():
    """The victim with these layers through the package's own attack: runs, captured iterations included, and gives the same bits twice."""
    from hit_adv_amd.ShapeAttack.HiT_ADV import HiT_ADV
    from hit_adv_amd.Dataset.synthetic import synth_batch
    from hit_adv_amd.model.pct import Pct
    from hit_adv_amd.util.adv_utils import UntargetedLogitsAdvLoss
    torch.manual_seed(0)
    model = Pct(_pct_args("differential")).cuda().eval()
    data, label = synth_batch(2, 1024)
    res = []
    for _ in range(2):
        torch.manual_seed(1)
        att = HiT_ADV(model, adv_func=UntargetedLogitsAdvLoss(kappa=30.), central_num=32, total_central_num=64, binary_step=1, num_iter=6,
                      curv_loss_knn=16, verbose=False)
        adv, _ = att.attack(data, label)
        res.append(np.asarray(adv))
    assert np.isfinite(res[0]).all() and np.array_equal(res[0], res[1])


# ---------------------------------------------------------------------------------------------------------------- without a GPU
def test_operators_refuse_cpu_tensors():
    x, w, rng = torch.randn(2, 16), torch.ones(16), torch.zeros(2, dtype=torch.int64)
    q = torch.randn(1, 2, 1, 2, 8)
    with pytest.raises(RuntimeError):
        ops.diff_attention(q, q, torch.randn(1, 2, 1, 16), torch.ones(1))
    with pytest.raises(RuntimeError):
        ops.rms_norm(x, w)
    with pytest.raises(RuntimeError):
        ops.rms_norm_quant(x, w)
    with pytest.raises(RuntimeError):
        ops.dropout(x, 0.5, rng)
    with pytest.raises(TypeError):
        ops.rms_norm([1.0], w)


def test_c_entry_points_refuse_what_they_do_not_take():
    """Error codes, no launches: null pointers, sizes outside the documented range, misaligned strides and bases."""
    lib = _lib.load()
    assert lib.hitadv_diff_attention_supported(1, 2, 4, 4, 4, 2, 64) == 1
    for args in ((3, 2, 4, 4, 4, 2, 64), (1, 2, 4, 4, 4, 3, 64), (1, 2, 4, 4, 4, 2, 12), (1, 2, 4, 4, 4, 2, 72), (1, 0, 4, 4, 4, 2, 64),
                 (1, 2, 4, 2 ** 31, 4, 2, 64), (1, 70000, 4, 4, 4, 2, 64), (1, 1, 2 ** 21, 4, 1, 1, 64), (1, 1, 40000, 4, 64, 1, 64),
                 (1, 1, 1, 1, 1 << 20, 1, 64)):
        assert lib.hitadv_diff_attention_supported(*args) == 0, args
    null, some = ctypes.c_void_p(0), ctypes.c_void_p(4096)
    good = (ctypes.c_int64 * 11)(*([64] * 11))
    f = lambda q=some, lam_n=1, st=good, out=some, D=16: lib.hitadv_diff_attention_fwd(  # noqa: E731
        0, q, some, some, some, lam_n, null, st, 1, 2, 2, 2, 1, D, 0, 0.25, out, null, null, null)
    assert f(q=null) == -1 and f(out=null) == -1 and f(lam_n=3) == -1 and f(D=20) == -1
    assert f(q=ctypes.c_void_p(4100)) == -1 and f(out=ctypes.c_void_p(4104)) == -1
    assert f(st=(ctypes.c_int64 * 11)(*([64] * 10 + [66]))) == -1 and f(st=(ctypes.c_int64 * 11)(*([64] * 10 + [-64]))) == -1
    # a call that is split needs its scratch
    n = lib.hitadv_diff_attention_scratch_floats(1, 1, 8192, 4, 1, 64)
    assert n > 0
    assert lib.hitadv_diff_attention_fwd(1, some, some, some, some, 1, null, good, 1, 1, 8192, 4, 1, 64, 0, 0.125, some, null, null, null) == -1
    assert lib.hitadv_diff_attention_scratch_floats(1, 1, 8192, 4, 3, 64) == 0
    assert lib.hitadv_diff_attention_bwd(0, some, some, some, some, 1, null, good, some, null, 1, 2, 2, 2, 1, 16, 0, 0.25, some, some, some, some,
                                         null, null) == -1
    assert lib.hitadv_rms_norm_fwd(0, 1, some, null, some, 4, 32, 1e-6, some, null, null, null) == -1   # bf16 weights of fp32 rows
    assert lib.hitadv_rms_norm_fwd(0, 0, some, null, some, 4, 16385, 1e-6, some, null, null, null) == -1
    assert lib.hitadv_rms_norm_fwd(0, 0, some, some, some, 4, 32, 1e-6, some, null, null, null) == -1   # a residual and nowhere for the sum
    assert lib.hitadv_rms_norm_e4m3(0, 0, some, null, some, 4, 32, 1e-6, some, null, null, null) == -1
    assert lib.hitadv_rms_norm_bwd(0, 0, some, some, some, some, null, 4, 32, some, null, some, null) == -1
    assert lib.hitadv_rms_norm_bwd_scratch_floats(0, 32) == 0 and lib.hitadv_rms_norm_bwd_scratch_floats(100, 32) >= 32
    assert lib.hitadv_dropout(0, some, null, some, 0, some, 5, 1.0, null) == -1
    assert lib.hitadv_dropout(0, some, null, some, 8, null, 5, 1.0, null) == -1
    assert lib.hitadv_dropout(0, some, null, some, 8, some, 2 ** 32 + 1, 1.0, null) == -1
