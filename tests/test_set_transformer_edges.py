"""ops.diff_attention, rms_norm, rms_norm_quant and dropout at calls where a wrapper, rather than a kernel, can go wrong.  The CPU tests run the
package's own functions on the kernels' source on the wave emulator: every launch is checked for what its addresses belong to."""
import ctypes
import os
import sys
import weakref

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tests", "native"))
sys.path.insert(0, os.path.join(ROOT, "tests"))
import emu_build  # noqa: E402
from hit_adv_amd import _lib, ops  # noqa: E402
from test_set_transformer_ops import attention_bounds, attention_reference, check, make  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
emulator = pytest.mark.skipif(not os.path.exists(emu_build.CLANGXX), reason="no host clang++")


@pytest.fixture(scope="module")
def emulated(tmp_path_factory):
    """Functions of the emulated kernel files, built when first asked for."""
    d, built = str(tmp_path_factory.mktemp("emu")), {}

    def function(name):
        stem = "diff_attention" if "attention" in name else "rms_norm" if "rms" in name else "dropout"
        if stem not in built:
            built[stem] = ctypes.CDLL(emu_build.build(stem, d))
        f = getattr(built[stem], name)
        f.argtypes, f.restype = _lib.PROTOTYPES[name], _lib._RESTYPE.get(name, ctypes.c_int)
        return f
    return function


class Launches:
    """In ops' place between the wrappers and the library: CPU tensors are taken, and at each launch the tensors whose addresses it got
    have to be there still (what nobody holds, the allocator may hand out again before the launch)."""

    def __init__(self, emulated, monkeypatch):
        self.taken, self.names, self.run, self.emulated = [], [], True, emulated
        monkeypatch.setattr(ops, "_typed", self.typed)
        monkeypatch.setattr(ops, "_at", self.at)
        monkeypatch.setattr(ops, "_call_on", self.launch)

    def typed(self, t, name, like=None, dtypes=ops._DTYPE_CODE):
        assert torch.is_tensor(t) and t.dtype in dtypes, name
        return t

    def at(self, t):
        if t is None:
            return 0
        self.taken.append((weakref.ref(t), t.dtype, tuple(t.shape)))
        return t.data_ptr()

    def launch(self, t, name, *args):
        gone = [(dtype, shape) for r, dtype, shape in self.taken if r() is None]
        types = {dtype for _, dtype, _ in self.taken}
        held, self.taken = [r() for r, _, _ in self.taken], []
        self.names.append(name)
        assert not gone, "%s: tensors given up before the launch: %s" % (name, gone)
        if "attention" in name:  # q, k, v: the strides that go with the addresses
            want = [(n, st) for x in held[:3] for n, st in zip(x.shape[:-1], x.stride())]
            assert all(got == st or n == 1 for got, (n, st) in zip(args[7], want)), "%s: strides %s of tensors with %s" % (name, list(args[7]), want)
        self.types(t, name, types)
        if self.run:
            assert self.emulated(name)(*args, None) == 0

    def types(self, t, name, types):
        pass


@pytest.fixture
def launches(emulated, monkeypatch):
    return Launches(emulated, monkeypatch)


def strided(t):
    """The same values, last axis not contiguous."""
    return t.transpose(0, 1).contiguous().transpose(0, 1)


# ---------------------------------------------------------------------------------------------------------------- gradients' layouts
def norm_gradients(device, layout_y, layout_s, rows=37, cols=100):
    g = torch.Generator().manual_seed(3)
    n = lambda *s: torch.randn(*s, generator=g).to(device)  # noqa: E731
    x, residual, w = n(rows, cols).requires_grad_(), n(rows, cols).requires_grad_(), n(cols).requires_grad_()
    gy, gs = n(rows, cols), n(rows, cols)
    y, s = ops.rms_norm(x, w, residual=residual)
    return torch.autograd.grad((y, s), (x, residual, w), (layout_y(gy), layout_s(gs)))


def same(t):
    return t


LAYOUTS = [(strided, same), (same, strided), (strided, strided)]


def norm_sums(device, plain, rows=37, cols=100):
    """Gradients of y.sum() + 2 s.sum(): autograd hands both to the norm expanded from one value."""
    g = torch.Generator().manual_seed(4)
    n = lambda *s: torch.randn(*s, generator=g).to(device)  # noqa: E731
    x, residual, w = n(rows, cols).requires_grad_(), n(rows, cols).requires_grad_(), n(cols).requires_grad_()
    y, s = ops.rms_norm(x, w, residual=residual)
    if plain:
        return torch.autograd.grad((y, s), (x, residual, w), (torch.ones_like(y), torch.full_like(s, 2.)))
    return torch.autograd.grad(y.sum() + 2 * s.sum(), (x, residual, w))


@emulator
@pytest.mark.parametrize("layout", LAYOUTS, ids=["y", "sum", "both"])
def test_norm_gradients_of_any_layout(launches, layout):
    for a, b in zip(norm_gradients("cpu", *layout), norm_gradients("cpu", same, same)):
        assert torch.equal(a, b)


@emulator
def test_norm_gradients_of_sums(launches):
    for a, b in zip(norm_sums("cpu", False), norm_sums("cpu", True)):
        assert torch.equal(a, b)


def test_every_launch_holds_the_copies_it_reads(launches):
    """Inputs of every operator in a layout that has to be copied first, forward and backward (nothing is launched)."""
    launches.run = False
    g = torch.Generator().manual_seed(5)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, r, w = strided(n(6, 40)).requires_grad_(), strided(n(6, 40)).requires_grad_(), n(40, 2)[:, 0].requires_grad_()
    y, s = ops.rms_norm(x, w, residual=r)
    torch.autograd.grad((y, s), (x, r, w), (strided(n(6, 40)), n(1).expand(6, 40)))
    y = ops.rms_norm(x, w)
    torch.autograd.grad(y, (x, w), strided(n(6, 40)))
    with torch.no_grad():
        ops.rms_norm_quant(x, w, residual=r)
        ops.rms_norm_quant(x, w)
    rng = torch.tensor([[1, 2], [3, 4]])[:, 0]
    torch.autograd.grad(ops.dropout(x, 0.5, rng, residual=r), (x, r), strided(n(6, 40)))
    q, k, v = (n(2, 5, *tail, 17)[..., :16].requires_grad_() for tail in ((4, 2), (2, 2), (2, 2)))
    v = n(2, 5, 2, 33)[..., :32].requires_grad_()
    lam = n(4, 3)[:, 1].requires_grad_()
    lengths = torch.tensor([[5, 0], [3, 0]])[:, 0]
    for kl in (lengths, lengths.int()[:], torch.tensor([[5, 0], [3, 0]], dtype=torch.int32)[:, 0]):
        out = ops.diff_attention(q, k, v, lam, key_lengths=kl)
        torch.autograd.grad(out, (q, k, v, lam), n(1).expand(out.shape))
    assert len(launches.names) == 2 + 2 + 2 + 2 + 3 * 2


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(37, 100), (300, 1000)])
@pytest.mark.parametrize("layout", LAYOUTS, ids=["y", "sum", "both"])
def test_norm_gradients_of_any_layout_on_the_gpu(layout, rows, cols):
    for a, b in zip(norm_gradients("cuda", *layout, rows, cols), norm_gradients("cuda", same, same, rows, cols)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_norm_gradients_of_sums_on_the_gpu():
    for a, b in zip(norm_sums("cuda", False), norm_sums("cuda", True)):
        assert torch.equal(a, b)


def fused_gradients(device, hooks):
    """Gradients of attention over slices of one projection and a norm, what is saved for them going through ``hooks``."""
    g = torch.Generator().manual_seed(11)
    n = lambda *s: torch.randn(*s, generator=g).to(device)  # noqa: E731
    h, lam, w = n(2, 40, 3, 128).requires_grad_(), torch.tensor([0.25, 0.5], device=device, requires_grad=True), n(64).requires_grad_()
    lengths = torch.tensor([40, 21], dtype=torch.int32, device=device)
    with hooks:
        q, k, v = h.unbind(2)
        out = ops.diff_attention(q.view(2, 40, 2, 2, 32), k.view(2, 40, 2, 2, 32), v.view(2, 40, 2, 64), lam, key_lengths=lengths)
        y, s = ops.rms_norm(out, w, residual=out.detach())
        z = ops.dropout(y, 0.5, torch.tensor([1, 2], device=device))
    return torch.autograd.grad((z, s), (h, lam, w), (n(2, 40, 2, 64), n(2, 40, 2, 64)))


def turned(t):
    return t.t().contiguous().t() if t.dim() == 2 else t.transpose(0, -1).contiguous().transpose(0, -1) if t.dim() > 2 else t


HOOKS = {"contiguous": (lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
         "turned": (turned, lambda t: t),
         "misaligned": (lambda t: t.detach(), lambda t: torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape))}


@emulator
@pytest.mark.parametrize("hooks", sorted(HOOKS))
def test_saved_tensors_may_come_back_in_another_layout(launches, hooks):
    """Saved-tensor hooks (activations moved to the host and back) return the values, not the strides."""
    want = fused_gradients("cpu", torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t))
    for a, b in zip(fused_gradients("cpu", torch.autograd.graph.saved_tensors_hooks(*HOOKS[hooks])), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_saved_tensors_may_come_back_in_another_layout_on_the_gpu():
    want = fused_gradients("cuda", torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t))
    for hooks in [torch.autograd.graph.saved_tensors_hooks(*HOOKS[n]) for n in sorted(HOOKS)] + [torch.autograd.graph.save_on_cpu()]:
        for a, b in zip(fused_gradients("cuda", hooks), want):
            assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------------------- torch's default type
class _DefaultType:
    def __init__(self, t):
        self.t = t

    def __enter__(self):
        self.before = torch.get_default_dtype()
        torch.set_default_dtype(self.t)

    def __exit__(self, *_):
        torch.set_default_dtype(self.before)


def every_operator(device, t):
    """Outputs and gradients of each operator in type t (attention: keys split and not)."""
    g = torch.Generator().manual_seed(6)
    n = lambda *s: torch.randn(*s, generator=g, dtype=F32).to(t).to(device)  # noqa: E731
    x, r, w = n(9, 72).requires_grad_(), n(9, 72).requires_grad_(), n(72).float().requires_grad_()
    y, s = ops.rms_norm(x, w, residual=r)
    res = [y, s, *torch.autograd.grad((y, s), (x, r, w), (n(9, 72), n(9, 72)))]
    with torch.no_grad():
        res += ops.rms_norm_quant(x, w, residual=r)
    y = ops.dropout(x, 0.5, torch.tensor([1, 2], device=device), residual=r)
    res += [y, *torch.autograd.grad(y, (x, r), n(9, 72))]
    for Nq, Nk in ((7, 40), (2, 600)):
        q, k, v = n(2, Nq, 2, 2, 16).requires_grad_(), n(2, Nk, 1, 2, 16).requires_grad_(), n(2, Nk, 1, 32).requires_grad_()
        lam = torch.tensor([0.25, 0.5], dtype=F32, device=device, requires_grad=True)
        out = ops.diff_attention(q, k, v, lam, causal=True)
        res += [out, *torch.autograd.grad(out, (q, k, v, lam), n(2, Nq, 2, 32))]
    return res


@emulator
@pytest.mark.parametrize("t,default", [(F32, torch.float64), (F32, BF16), (BF16, F16), (F16, BF16)])  # (a buffer of t itself could not be told)
def test_buffers_do_not_follow_the_default_type(launches, t, default):
    """A program that works with torch.set_default_dtype(bfloat16) gets the same bits: the kernels' own buffers are fp32 whatever it says (half as
    large, a launch would write behind them: the sizes are checked before it)."""
    want = every_operator("cpu", t)

    def types(tensor, name, seen):
        assert seen <= {t, F32, torch.int32, torch.int64, torch.float8_e4m3fn}, "%s: %s" % (name, seen)
    launches.types = types
    with _DefaultType(default):
        got = every_operator("cpu", t)
    assert launches.names[:len(launches.names) // 2] == launches.names[len(launches.names) // 2:]
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("default", [torch.float64, BF16, F16])
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_buffers_do_not_follow_the_default_type_on_the_gpu(t, default):
    want = every_operator("cuda", t)
    with _DefaultType(default):
        got = every_operator("cuda", t)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# ---------------------------------------------------------------------------------------------------------------- infinite scores
INFINITE = [  # rows x keys: one part of the keys, few parts, more than eight
    (40, 70), (40, 700), (3, 2700)]


def infinite_row(device, t, Nq, Nk):
    """Two heads, causal; in map 1 every score of row 2 of head 1 is -inf (an infinite query against negative keys)."""
    g = torch.Generator().manual_seed(7)
    n = lambda *s: torch.randn(*s, generator=g).to(t).to(device)  # noqa: E731
    q, k, v, go = n(1, Nq, 2, 2, 16), n(1, Nk, 2, 2, 16), n(1, Nk, 2, 32), n(1, Nq, 2, 32)
    q[..., 0, 0], k[..., 0, 0] = 1., -k[..., 0, 0].abs() - 0.5
    lam = torch.tensor([0.25, 0.5], dtype=F32, device=device)

    def run(q):
        leaves = [x.clone().requires_grad_() for x in (q, k, v, lam)]
        out = ops.diff_attention(*leaves, causal=True)
        with torch.no_grad():
            same = ops.diff_attention(*leaves, causal=True)
        return out, same, torch.autograd.grad(out, leaves, go)
    bad = q.clone()
    bad[0, 2, 1, 0, 0] = float("inf")
    return run(q), run(bad)


def check_infinite_row(device, t, Nq, Nk):
    """softmax of a row of -inf is NaN: the row, and what map 1 of its query, its keys and their values get of it; nothing else is touched."""
    (out, same, grads), (bad, bad_same, bad_grads) = infinite_row(device, t, Nq, Nk)
    assert torch.equal(out, same) and bool(out.isfinite().all())
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[0, 2, 1] = False
    for x in (bad, bad_same):
        assert bool(x[0, 2, 1].isnan().all()) and torch.equal(x[keep], out[keep])
    dq, dk, dv, dlam = bad_grads
    seen = Nk - Nq + 3  # row 2's keys; (r = NaN reaches map 1 of the keys behind them)
    assert bool(dq[0, 2, 1, 0].isnan().all()) and bool(dk[0, :seen, 1, 0].isnan().all()) and bool(dv[0, :seen, 1].isnan().all())
    keep = torch.ones_like(dq, dtype=torch.bool)
    keep[0, 2, 1, 0] = False
    assert torch.equal(dq[keep], grads[0][keep]) and torch.equal(dlam, grads[3])
    assert torch.equal(dk[:, :, 0], grads[1][:, :, 0]) and torch.equal(dk[:, :, 1, 1], grads[1][:, :, 1, 1])
    assert torch.equal(dv[:, :, 0], grads[2][:, :, 0]) and torch.equal(dv[:, seen:], grads[2][:, seen:])


@emulator
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_a_row_of_infinite_scores_is_nan(launches, t):
    check_infinite_row("cpu", t, *INFINITE[0])
    with torch.no_grad():  # the joins: forward
        for size in INFINITE[1:]:
            q, k, v = (torch.ones(1, size[i > 0], 1, *((2, 8) if i < 2 else (16,))).to(t) for i in range(3))
            q[0, 1] = float("inf")
            out = ops.diff_attention(q, -k, v, torch.tensor(0.5))
            assert bool(out[0, 1].isnan().all()) and torch.equal(out[0, 0], out[0, 2]) and bool(out[0, 0].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("size", INFINITE, ids=str)
def test_a_row_of_infinite_scores_is_nan_on_the_gpu(t, size):
    check_infinite_row("cuda", t, *size)


def one_infinite_key(device, t, Nq, Nk):
    g = torch.Generator().manual_seed(8)
    n = lambda *s: torch.randn(*s, generator=g).to(t).to(device)  # noqa: E731
    q, k, v = n(1, Nq, 2, 2, 16), n(1, Nk, 2, 2, 16), n(1, Nk, 2, 32)
    q[..., 0, 0] = 1.
    lam = torch.tensor([0.25, 0.5], dtype=F32, device=device)
    outs = []
    for value in (-1e4, -float("inf")):  # (a score of -2500: its probability is 0 in fp32)
        k[0, 5, :, 0, 0] = value
        outs.append(ops.diff_attention(q, k, v, lam))
    return outs


def check_one_infinite_key(device, t, Nq, Nk):
    """A key with a score of -inf has probability 0 in 16-bit types; fp32's pieces of an infinity are NaN, and so is the row."""
    far, infinite = one_infinite_key(device, t, Nq, Nk)
    assert bool(far.isfinite().all())
    assert bool(infinite.isnan().all()) if t is F32 else torch.equal(far, infinite)


@emulator
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_one_infinite_score(launches, t):
    check_one_infinite_key("cpu", t, *INFINITE[0])


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("size", INFINITE, ids=str)
def test_one_infinite_score_on_the_gpu(t, size):
    check_one_infinite_key("cuda", t, *size)


# ---------------------------------------------------------------------------------------------------------------- 8-bit rows
def check_special_quant_rows(device, t, cols):
    """scale = max |y| / 448 also where that is not finite: NaN for a row with a NaN (or an infinity in x: its r is 0), inf for an infinite weight."""
    x = torch.ones(4, cols, dtype=t)
    x[0, cols // 2], x[1, 0], x[2, cols - 1] = float("nan"), float("inf"), -float("inf")
    w = torch.ones(cols)
    q, scale = ops.rms_norm_quant(x.to(device), w.to(device))
    q, scale = q.float().cpu(), scale.cpu()
    assert bool(scale[:3].isnan().all()) and bool(q[:3].isnan().all())
    assert bool(scale[3].isfinite()) and bool((q[3] == 448).all())
    w[3] = -float("inf")
    q, scale = ops.rms_norm_quant(x[3:].to(device), w.to(device))
    q = q[0].float().cpu()
    assert float(scale[0]) == float("inf") and bool(q[3].isnan()) and not q[:3].any() and not q[4:].any()
    w[3] = float("nan")
    q, scale = ops.rms_norm_quant(x[3:].to(device), w.to(device))
    assert bool(scale.isnan().all()) and bool(q.float().isnan().all())


SPECIAL_COLS = [5, 64, 500, 3000, 9000]  # each width of a row's team


@emulator
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_quant_rows_that_are_not_finite(launches, t):
    for cols in SPECIAL_COLS[:4]:
        check_special_quant_rows("cpu", t, cols)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("cols", SPECIAL_COLS)
def test_quant_rows_that_are_not_finite_on_the_gpu(t, cols):
    check_special_quant_rows("cuda", t, cols)


def check_tiny_quant_rows(device, cols):
    """Rows whose max |y| / 448 is below the smallest fp32 number are zeros with the scale 1 (0 / 0 would make them NaN, and what is not 0 would be 448)."""
    x = torch.zeros(2, cols)
    x[0, 1::2] = 1e-44
    x[1] = 1.
    w = torch.full((cols,), 1e-3)
    q, scale = ops.rms_norm_quant(x.to(device), w.to(device))
    q, scale = q.float().cpu(), scale.cpu()
    assert float(scale[0]) == 1. and not q[0].any()
    assert float(scale[1]) < 1e-3 and bool((q[1] == 448).all())


@emulator
def test_quant_rows_below_the_smallest_scale(launches):
    for cols in SPECIAL_COLS[:4]:
        check_tiny_quant_rows("cpu", cols)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", SPECIAL_COLS)
def test_quant_rows_below_the_smallest_scale_on_the_gpu(cols):
    check_tiny_quant_rows("cuda", cols)


# ---------------------------------------------------------------------------------------------------------------- many rows
@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(2 ** 28 + 5, 8), (2 ** 26 + 1, 130), (2 ** 24 + 3, 1026)])
def test_norm_of_more_rows_than_a_grid_dimension_takes(rows, cols):
    """2^32 threads are a dimension's limit: 2^28 rows with 16 lanes each, 2^26 with 64, 2^24 with 256.  The rows are those of smaller calls."""
    x = torch.empty(rows, cols, device="cuda", dtype=BF16).normal_(generator=torch.Generator("cuda").manual_seed(1))
    w = torch.rand(cols, generator=torch.Generator().manual_seed(2)).cuda()
    cuts = [*range(0, rows, rows // 5), rows]
    y = ops.rms_norm(x, w)
    for a, b in zip(cuts, cuts[1:]):
        assert torch.equal(y[a:b], ops.rms_norm(x[a:b], w))
    del y
    q, scale = ops.rms_norm_quant(x, w)
    for a, b in zip(cuts, cuts[1:]):
        qs, ss = ops.rms_norm_quant(x[a:b], w)
        assert torch.equal(q[a:b].view(torch.uint8), qs.view(torch.uint8)) and torch.equal(scale[a:b], ss)
    del q, scale, qs, ss
    if cols == 8:
        dx, = torch.autograd.grad(ops.rms_norm(x.requires_grad_(), w), x, x.detach())
        for a, b in zip(cuts, cuts[1:]):
            part = x.detach()[a:b].requires_grad_()
            assert torch.equal(dx[a:b], torch.autograd.grad(ops.rms_norm(part, w), part, part.detach())[0])
        del dx, part
    del x
    torch.cuda.empty_cache()  # (up to 90 GB)


def test_attention_refuses_more_heads_than_the_weights_gradient_has_workgroups_for():
    """dlam's kernel has 1024 threads a head, and a grid dimension ends below 2^32."""
    supported = _lib.load().hitadv_diff_attention_supported
    assert supported(1, 1, 1, 1, 2 ** 22 - 2 ** 7, 2 ** 15 - 1, 8) == 1
    for heads in (2 ** 22, 2 ** 22 + 2 ** 15, 2 ** 24):
        assert supported(1, 1, 1, 1, heads, 2 ** 15, 8) == 0


# ---------------------------------------------------------------------------------------------------------------- scales
def underflow(r, Hkv):
    """What numbers below u = 2^-126, which the exponential and the matrix instruction drop, take from the sums in front of their factor ``scale``:
    a probability (u times what it is multiplied with), the three pieces of A or dS (3 u times the other operand) and the up to six
    products of a term with their sums (6 u)."""
    u = 2.0 ** -126
    B, Nq, H, _, D = r.q.shape
    e = lambda s, *t: torch.einsum(s, *(x.abs() for x in t))  # noqa: E731
    w = (r.dP[:, :, None] - r.r[..., None]).abs() * r.sign.abs() + 3
    a = (4 + r.l.abs()).expand(B, H, Nq, r.Nk)
    heads = lambda t: t.view(B, r.Nk, Hkv, H // Hkv, *t.shape[3:]).sum(3)  # noqa: E731
    return {"out": u * (e("bhij,bjhd->bihd", a, r.vv) + 6 * r.Nk), "dv": u * heads(e("bhij,bihd->bjhd", a, r.g) + 6 * Nq),
            "dq": abs(r.scale) * u * (e("bhmij,bjhmd->bihmd", w, r.kk) + 6 * r.Nk),
            "dk": abs(r.scale) * u * heads(e("bhmij,bihmd->bjhmd", w, r.q) + 6 * Nq), "dlam": u * (r.dP.abs() + 6).sum((0, 2, 3))}


def check_scaled_gradients(device, t, scale, causal, size=(1, 40, 70, 2, 1, 16)):
    """Output and gradients at scores of 1e4, of 0 and with a negative scale.  The bounds hold a probability's error for the scores' size: at 1e4 the
    fp32 numbers that stand for a score, a row's maximum and its logarithm have steps of 2^-10.  What underflows is added: a probability of 2^-120
    in front of a scale of 300 makes a gradient that is not small beside fp32's smallest numbers."""
    q, k, v, lam, g = make(t, *size, seed=21, device=device)
    r = attention_reference(q, k, v, lam, causal, scale=scale, dout=g)
    b, u = attention_bounds(t, r, True), underflow(r, size[4])
    b = {name: b[name] + u[name] for name in b}
    leaves = [x.requires_grad_() for x in (q, k, v, lam)]
    out = ops.diff_attention(*leaves, scale=scale, causal=causal)
    check(out, r.out, b["out"], "out")
    grads = torch.autograd.grad(out, leaves, g)
    for name, got in zip(("dq", "dk", "dv", "dlam"), grads):
        check(got, getattr(r, name), b[name], name)
    if scale == 0.:
        assert not grads[0].any() and not grads[1].any()
    return out, grads


SCALES = [0., 300., -2., -300., 2. ** -20]


@emulator
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_gradients_at_extreme_scales(launches, t):
    for scale in (0., 300., -2.):
        check_scaled_gradients("cpu", t, scale, True)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("scale", SCALES)
@pytest.mark.parametrize("size", [(1, 40, 70, 2, 1, 16), (2, 33, 700, 4, 2, 64)], ids=str)
def test_gradients_at_extreme_scales_on_the_gpu(t, scale, size):
    for causal in (False, True):
        check_scaled_gradients("cuda", t, scale, causal, size)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_a_negative_scale_is_a_negative_query(t):
    """The sign is taken into the operand: the same bits as the query's own sign, dq turned.  (dK = scale dS^T Q sums products of the other sign, and the
    matrix instruction truncates downwards: its last bits differ, and the test above holds it to its bound.)"""
    q, k, v, lam, g = make(t, 2, 50, 90, 4, 2, 32, seed=22)

    def run(q, scale):
        leaves = [x.detach().clone().requires_grad_() for x in (q, k, v, lam)]
        out = ops.diff_attention(*leaves, scale=scale, causal=True)
        return (out, *torch.autograd.grad(out, leaves, g))
    (o, dq, _, dv, dl), (o2, dq2, _, dv2, dl2) = run(q, -0.25), run(-q, 0.25)
    assert torch.equal(o, o2) and torch.equal(dq, -dq2) and torch.equal(dv, dv2) and torch.equal(dl, dl2)


# ---------------------------------------------------------------------------------------------------------------- rows that see nothing
def check_empty_rows_give_nothing(device, t, B, Nq, Nk, H, Hkv, D, lengths=None):
    """Queries in front of the first key (causal, more queries than keys) and all queries of an empty sequence: whatever they and their incoming
    gradients hold -- NaN, infinities -- stays out of every other row's output and of all gradients."""
    q, k, v, lam, g = make(t, B, Nq, Nk, H, Hkv, D, seed=31, device=device)
    kl = torch.tensor(lengths, dtype=torch.int32, device=device) if lengths else None
    seen = torch.full((B, Nq), Nk) if kl is None else kl.cpu().long()[:, None].expand(B, Nq)
    empty = (torch.minimum(seen, torch.arange(Nq) + Nk - Nq + 1) <= 0).to(device)
    assert bool(empty.any()) and not bool(empty.all())

    def run(fill_q, fill_g):
        leaves = [x.clone().requires_grad_() for x in (q.masked_fill(empty[:, :, None, None, None], fill_q), k, v, lam)]
        out = ops.diff_attention(*leaves, causal=True, key_lengths=kl)
        return (out, *torch.autograd.grad(out, leaves, g.masked_fill(empty[:, :, None, None], fill_g)))
    want = run(0., 0.)
    assert not want[0][empty].any() and not want[1][empty].any()
    for fill_q, fill_g in ((0., float("nan")), (float("nan"), 0.), (float("inf"), -float("inf"))):
        for a, b, name in zip(run(fill_q, fill_g), want, ("out", "dq", "dk", "dv", "dlam")):
            assert torch.equal(a, b), (name, fill_q, fill_g)


EMPTY = [(1, 50, 20, 2, 2, 16), (2, 77, 45, 3, 1, 40), (1, 200, 70, 2, 1, 64), (2, 40, 33, 4, 2, 32, (33, 0))]


@emulator
@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_rows_that_see_nothing_give_nothing(launches, t):
    for case in (EMPTY[0], EMPTY[1]):
        check_empty_rows_give_nothing("cpu", t, *case)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("case", EMPTY, ids=str)
def test_rows_that_see_nothing_give_nothing_on_the_gpu(t, case):
    check_empty_rows_give_nothing("cuda", t, *case)


# ---------------------------------------------------------------------------------------------------------------- the layer
@pytest.mark.gpu
@pytest.mark.parametrize("p", [0., 0.5])
def test_da_layer_under_autocast(p):
    """In training as in evaluation the projections' 16-bit output joins the residual in the residual's type."""
    from hit_adv_amd.model.pct import DA_Layer
    torch.manual_seed(0)
    m = DA_Layer(128, dropout=p).cuda()
    x = torch.randn(2, 128, 40, device="cuda")
    outs = {}
    for mode in (False, True):
        m.train(mode)
        with torch.autocast("cuda", dtype=BF16):
            y = m(x.requires_grad_())
        assert y.dtype == F32 and y.shape == x.shape
        g, = torch.autograd.grad(y, x, torch.ones_like(y))
        assert bool(g.isfinite().all())
        outs[mode] = y.detach()
    if p == 0.:
        assert torch.equal(outs[False], outs[True])
    else:  # an element is dropped, or twice what evaluation adds
        d, e = outs[True] - x.detach(), outs[False] - x.detach()
        # either sum is rounded once: 2^-24 of values below 2^3, twice where doubled
        assert bool(((d == 0) | ((d - 2 * e).abs() <= 3 * 2.0 ** -21)).all()) and 0.4 < float((d == 0).float().mean()) < 0.6


@pytest.mark.gpu
def test_da_layer_captured_draws_new_masks():
    """A captured training step: every replay takes the next offset, and gives the eager layer's bits at that offset."""
    from hit_adv_amd.model.pct import DA_Layer
    torch.manual_seed(0)
    m = DA_Layer(64, dropout=0.5).cuda().train()
    x, g = torch.randn(2, 64, 40, device="cuda"), torch.randn(2, 64, 40, device="cuda")
    leaf = x.clone().requires_grad_()

    def step():
        y = m(leaf)
        return y.detach(), *torch.autograd.grad(y, [leaf, m.out.weight], g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    last = None
    for _ in range(4):
        offset = int(m.rng[1])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert int(m.rng[1]) == offset + 1 and (last is None or not torch.equal(got[0], last))
        last = got[0]
        m.rng[1] = offset
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
