"""diff_attention.hip, rms_norm.hip and dropout.hip as they are, run on the CPU's wave64 emulator through the C ABI against the definitions in
64 bits: the index arithmetic, masks, splits and joins, LDS layouts and barriers (not the hardware's rounding of matrix products)."""
import ctypes
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests", "native"))
sys.path.insert(0, os.path.join(ROOT, "tests"))
import emu_build  # noqa: E402
from test_set_transformer_ops import BF16, F16, F32, U, attention_bounds, attention_reference, check, half_step, make, philox_words, smallest  # noqa: E402

pytestmark = pytest.mark.skipif(not os.path.exists(emu_build.CLANGXX), reason="no host clang++")
CODE = {F32: 0, BF16: 1, F16: 2}
I64, F = ctypes.c_int64, ctypes.c_float


def P(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def nan(*shape, dtype=F32):
    return torch.full(shape, float("nan")).to(dtype)


@pytest.fixture(scope="module")
def emulated(tmp_path_factory):
    d = str(tmp_path_factory.mktemp("emu"))
    libs = {stem: ctypes.CDLL(emu_build.build(stem, d)) for stem in ("diff_attention", "rms_norm", "dropout")}
    libs["diff_attention"].hitadv_diff_attention_scratch_floats.restype = I64
    libs["rms_norm"].hitadv_rms_norm_bwd_scratch_floats.restype = I64
    return libs


@pytest.mark.parametrize("t,case", [
    (F32, (1, 40, 40, 2, 1, 32, False, None, 2)),
    (BF16, (2, 70, 33, 3, 3, 64, True, None, 1)),           # 37 rows see nothing
    (F32, (1, 33, 130, 2, 2, 64, True, None, 2)),
    (F16, (2, 5, 170, 7, 1, 40, True, (170, 3), 7)),
    (BF16, (2, 1, 2700, 4, 2, 24, True, (2700, 0), 4)),     # single tokens, more than eight parts of the keys
    (F16, (1, 40, 700, 4, 2, 48, True, (690,), 1)),         # few parts joined for many rows
], ids=str)
def test_differential_attention(emulated, t, case):
    L = emulated["diff_attention"]
    B, Nq, Nk, H, Hkv, D, causal, lengths, lam_n = case
    q, k, v, lam, g = make(t, B, Nq, Nk, H, Hkv, D, seed=3, lam_n=lam_n, device="cpu")
    lens = torch.tensor(lengths, dtype=torch.int32) if lengths else None
    strides = (I64 * 11)(*q.stride()[:4], *k.stride()[:4], *v.stride()[:3])
    n = L.hitadv_diff_attention_scratch_floats(B, Nq, Nk, H, Hkv, D)
    assert (n > 0) == (Nk > 512)
    out, stats, scratch = nan(B, Nq, H, 2 * D, dtype=t), nan(4, B, H, Nq), nan(max(n, 1))
    head = (CODE[t], P(q), P(k), P(v), P(lam), lam_n, P(lens), strides)
    sizes = (B, Nq, Nk, H, Hkv, D, int(causal), F(D ** -0.5))
    assert L.hitadv_diff_attention_fwd(*head, *sizes, P(out), P(stats), P(scratch), None) == 0
    dq, dk, dv, dlam, r = (nan(*x.shape, dtype=x.dtype) for x in (q, k, v, lam, torch.empty(2, B, H, Nq)))
    assert L.hitadv_diff_attention_bwd(*head, P(g), P(stats), *sizes, P(r), P(dq), P(dk), P(dv), P(dlam), None) == 0
    ref = attention_reference(q, k, v, lam, causal, lens, dout=g)
    bounds = attention_bounds(t, ref, True)
    for name, got in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv), ("dlam", dlam)):
        check(got, getattr(ref, name), bounds[name], name)


@pytest.mark.parametrize("t,tw,rows,cols,res", [(F32, F32, 5, 256, True), (BF16, F32, 37, 100, False), (F16, F16, 3, 128, True), (BF16, BF16, 3, 1, True),
                                                (BF16, F32, 2, 4095, True), (F32, F32, 2, 1025, False), (F16, F32, 1, 9001, False)], ids=str)
def test_rms_norm(emulated, t, tw, rows, cols, res):
    L = emulated["rms_norm"]
    gen = torch.Generator().manual_seed(4)
    x, dy, residual, dsum = (torch.randn(rows, cols, generator=gen).to(t) for _ in range(4))
    w = (torch.rand(cols, generator=gen) + 0.5).to(tw)
    if not res:
        residual = dsum = None
    y, s, dx, rstd, dw = nan(rows, cols, dtype=t), nan(rows, cols, dtype=t), nan(rows, cols, dtype=t), nan(rows), nan(cols, dtype=tw)
    q, scale = torch.zeros(rows, cols, dtype=torch.float8_e4m3fn), nan(rows)
    head = (CODE[t], CODE[tw], P(x), P(residual), P(w), I64(rows), cols, F(1e-6))
    assert L.hitadv_rms_norm_fwd(*head, P(y), P(s) if res else None, P(rstd), None) == 0
    total = (x.float() + residual.float()).to(t) if res else x
    if res:
        assert torch.equal(s, total)
    assert L.hitadv_rms_norm_e4m3(*head, P(q), P(scale), P(s) if res else None, None) == 0
    scratch = nan(L.hitadv_rms_norm_bwd_scratch_floats(I64(rows), cols))
    assert L.hitadv_rms_norm_bwd(CODE[t], CODE[tw], P(total), P(w), P(rstd), P(dy), P(dsum), I64(rows), cols, P(dx), P(scratch), P(dw), None) == 0
    f, wd, gd = total.double(), w.double(), dy.double()
    r = 1 / torch.sqrt(f.pow(2).mean(1, keepdim=True) + 1e-6)
    Y, g = f * r * wd, gd * wd
    e = (cols + 16) * U  # a row's sum of squares in fp32, half of it in r, and the products behind it
    check(y, Y, (half_step(t) + e) * Y.abs() + smallest(t), "y")
    m = (g * f).mean(1, keepdim=True)
    ma = (g * f).abs().mean(1, keepdim=True)
    DX = r * (g - f * r * r * m) + (dsum.double() if res else 0)
    check(dx, DX, half_step(t) * DX.abs() + 4 * e * r * (g.abs() + f.abs() * r * r * ma) + 2 * U * DX.abs() + smallest(t), "dx")
    DW = (gd * f * r).sum(0)
    check(dw, DW, half_step(tw) * DW.abs() + (e + (rows + 16) * U) * (gd * f * r).abs().sum(0) + smallest(tw), "dw")
    top = Y.abs().amax(1)
    check(scale, top / 448, (e + 4 * U) * top / 448, "scale")
    # half a step of e4m3 (2^-4 of the value, 2^-10 below its normal range), of the scaled value with its own error
    z = Y / scale.double()[:, None]
    check(q.float(), z, (2.0 ** -4 + 4 * e) * z.abs() + 2.0 ** -10, "q")


@pytest.mark.parametrize("t,n,p,res", [(F32, 10001, 0.3, True), (BF16, 4099, 0.5, False), (F16, 1, 0.1, True), (BF16, 2050, 0.0, True), (F32, 77, 1.0, False)])
def test_dropout(emulated, t, n, p, res):
    gen = torch.Generator().manual_seed(5)
    x, residual = torch.randn(n, generator=gen).to(t), torch.randn(n, generator=gen).to(t) if res else None
    rng = torch.randint(0, 2 ** 62, (2,), generator=gen)
    y, threshold = nan(n, dtype=t), int(round(p * 2 ** 32))
    scale = F(1 / (1 - p) if p < 1 else 0.)
    assert emulated["dropout"].hitadv_dropout(CODE[t], P(x), P(residual), P(y), I64(n), P(rng), ctypes.c_uint64(threshold), scale, None) == 0
    keep = philox_words(n, int(rng[0]), int(rng[1])) >= threshold
    Y = torch.where(keep, x.float() * scale.value, torch.zeros(()))
    assert torch.equal(y, (Y + residual.float() if res else Y).to(t))
