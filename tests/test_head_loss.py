"""Losses of a language model's head (ops.linear_cross_entropy,
ops.linear_distillation) against their definitions in float64.

Bounds on the kernels (u = 2^-24; bfloat16 rounds by 2^-8): a logit
is off by at most about 4·sqrt(d)·u·(|h|·|w|) (a dot product in fp32), in base
2 and around a maximum by 4·u·|t| more; p by that relatively, and with
bfloat16 inputs by the 2^-10·ln 2 of a kept logit's step (half of 2^-9). The slopes S of the
logits are rounded to the inputs' type, and so are the gradients, whose
products' sums run in fp32: elementwise

    |dH - exact| <= (e_S + 4·sqrt(V)·u)·(|S|·|W|) + e_out·|dH|,

e_S the sum of what S is off by relative to |p| and |S|, and the same for dW.
"""

import math

import pytest
import torch

from pytorch_opt import ops
from pytorch_opt.ops import OpsArgumentError
from pytorch_opt.ops import reference as ref

DEV = "cuda"
U = 2.0 ** -24
IGNORE = -100


def _make(rows, d, vocab, dtype, seed=0, scale=2.0, device=DEV):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(rows, d, generator=g, dtype=torch.float64)
    w = torch.randn(vocab, d, generator=g, dtype=torch.float64) * (scale / math.sqrt(d))
    w *= torch.exp(0.3 * torch.randn(vocab, 1, generator=g, dtype=torch.float64))
    return h.to(dtype).to(device), w.to(dtype).to(device), g


def _targets(rows, vocab, g, keep=1.0, device=DEV):
    y = torch.randint(0, vocab, (rows,), generator=g)
    y[torch.rand(rows, generator=g) >= keep] = IGNORE
    return y.to(device)


def _teacher(rows, vocab, k, g, ragged=False, device=DEV):
    index = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)]) if rows else \
        torch.zeros(0, k, dtype=torch.long)
    logits = 4 * torch.randn(rows, k, generator=g)
    if ragged:
        index[torch.rand(rows, k, generator=g) < 0.3] = -1
        logits[torch.rand(rows, k, generator=g) < 0.1] = -float("inf")
        index[torch.rand(rows, generator=g) < 0.2] = -1
    return logits.to(device), index.to(device)


class Exact:
    """Loss, slopes of the logits and gradients in float64. want [rows, vocab]
    holds the targets' shares."""

    def __init__(self, h, w, kept, want, entropy, temp=1.0, zeta=0.0, weights=None, reduction="mean"):
        self.h = torch.where(kept[:, None], h.double(), 0.0)
        self.w, self.kept = w.double(), kept
        self.z = self.h @ self.w.T / temp
        self.lse = torch.logsumexp(self.z, 1)
        self.p = torch.exp(self.z - self.lse[:, None])
        rows = temp ** 2 * (self.lse * want.sum(1) - (want * self.z).sum(1) + entropy) + zeta * self.lse ** 2
        self.rows = torch.where(kept, rows, 0.0)
        count = max(1, int(kept.sum()))
        self.loss = {"none": self.rows, "mean": self.rows.sum() / count, "sum": self.rows.sum()}[reduction]
        g = {"none": weights, "mean": 1.0 / count, "sum": 1.0}[reduction]
        self.a = torch.where(kept, torch.ones_like(rows) * g, 0.0)[:, None] * temp
        f = 1 + 2 * zeta * self.lse[:, None] / temp ** 2
        self.dense = self.a * f * self.p
        self.S = self.dense - self.a * want
        self.dh, self.dw = self.S @ self.w, self.S.T @ self.h
        self.temp = temp

    def bounds(self, dtype):
        """(rows' loss, dH, dW) elementwise bounds."""
        rows, d = self.h.shape
        vocab = self.w.shape[0]
        out = 2.0 ** -8 if dtype == torch.bfloat16 else U
        step = 2.0 ** -10 * math.log(2) if dtype == torch.bfloat16 else 0.0
        logit = 4 * math.sqrt(d) * U * (self.h.abs() @ self.w.abs().T) / self.temp + 8 * U * self.z.abs() + 8 * U
        lse = (logit * self.p).sum(1, keepdim=True) + 4 * U * (1 + self.lse.abs()[:, None])
        eS = (step + logit + lse) * self.dense.abs() * 1.01 + (out + 8 * U) * (self.S.abs() + self.dense.abs() * U * 8)
        target = (logit + lse) * (self.a.abs() > 0)
        loss = self.temp ** 2 * 2 * (target.amax(1) + 4 * U * (1 + self.lse.abs())) + 4 * U * self.rows.abs()
        eh = eS @ self.w.abs() + 4 * math.sqrt(vocab) * U * (self.S.abs() @ self.w.abs()) + out * self.dh.abs()
        ew = eS.T @ self.h.abs() + 4 * math.sqrt(rows) * U * (self.S.abs().T @ self.h.abs()) + out * self.dw.abs()
        return loss, eh + 1e-30, ew + 1e-30


def _exact_ce(h, w, y, smooth=0.0, zeta=0.0, weights=None, reduction="mean"):
    vocab = w.shape[0]
    kept = y != IGNORE
    want = torch.full((len(y), vocab), smooth / vocab, dtype=torch.float64, device=h.device)
    want.scatter_add_(1, y.clamp_min(0)[:, None], torch.full((len(y), 1), 1 - smooth, dtype=torch.float64,
                                                              device=h.device))
    return Exact(h, w, kept, want, 0.0, zeta=zeta, weights=weights, reduction=reduction)


def _exact_kd(h, w, logits, index, temp=1.0, weights=None, reduction="mean"):
    there = (index >= 0) & (logits != -float("inf"))
    kept = there.any(1)
    t = torch.where(there, logits.double() / temp, -float("inf"))
    q = torch.where(kept[:, None], t, 0.0).softmax(1) * there
    want = torch.zeros(len(index), w.shape[0], dtype=torch.float64, device=h.device)
    want.scatter_add_(1, index.clamp_min(0), q)
    return Exact(h, w, kept, want, torch.special.xlogy(q, q).sum(1), temp=temp, weights=weights, reduction=reduction)


def _check(exact, loss, dh, dw, dtype, reduction):
    bl, bh, bw = exact.bounds(dtype)
    if reduction != "none":
        bl = bl[exact.kept].sum() / (max(1, int(exact.kept.sum())) if reduction == "mean" else 1) + 4 * U * abs(exact.loss)
    for name, got, want, bound in (("loss", loss, exact.loss, bl), ("dH", dh, exact.dh, bh), ("dW", dw, exact.dw, bw)):
        if got is None:
            continue
        far = (got.double() - want).abs()
        assert torch.isfinite(got).all(), name
        assert bool((far <= bound).all()), (name, float((far / bound.clamp_min(1e-300)).max()), float(far.max()))


SIZES = [
    (1, 1, 1), (1, 64, 128), (2, 3, 5), (5, 40, 33), (64, 64, 640), (128, 128, 256), (129, 136, 1000),
    (300, 256, 257), (257, 1000, 777), (31, 128, 20001), (700, 384, 2048), (1000, 72, 513),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d,vocab", SIZES)
@pytest.mark.parametrize("keep,smooth,zeta", [(1.0, 0.0, 0.0), (0.6, 0.1, 1e-3)])
def test_cross_entropy_matches_float64(native_backend, dtype, rows, d, vocab, keep, smooth, zeta):
    h, w, g = _make(rows, d, vocab, dtype, seed=rows + d + vocab)
    y = _targets(rows, vocab, g, keep)
    h.requires_grad_(), w.requires_grad_()
    for reduction in ("mean", "sum", "none"):
        weights = torch.randn(rows, generator=g).to(DEV) if reduction == "none" else None
        loss = ops.linear_cross_entropy(h, w, y, ignore_index=IGNORE, label_smoothing=smooth, z_loss=zeta,
                                        reduction=reduction)
        assert loss.dtype == torch.float32 and loss.shape == (y.shape if reduction == "none" else ())
        dh, dw = torch.autograd.grad(loss, (h, w), weights)
        e = _exact_ce(h.detach(), w.detach(), y, smooth, zeta, None if weights is None else weights.double(),
                      reduction)
        _check(e, loss.detach(), dh, dw, dtype, reduction)
        with torch.no_grad():
            again = ops.linear_cross_entropy(h, w, y, ignore_index=IGNORE, label_smoothing=smooth, z_loss=zeta,
                                             reduction=reduction)
        _check(e, again, None, None, dtype, reduction)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,d,vocab,k", [(1, 8, 4, 1), (3, 64, 128, 5), (65, 136, 1000, 33), (130, 256, 4097, 64),
                                            (300, 128, 2048, 1024), (257, 1000, 777, 16)])
@pytest.mark.parametrize("temp,ragged", [(1.0, False), (2.5, True)])
def test_distillation_matches_float64(native_backend, dtype, rows, d, vocab, k, temp, ragged):
    h, w, g = _make(rows, d, vocab, dtype, seed=rows + d + k)
    logits, index = _teacher(rows, vocab, k, g, ragged)
    h.requires_grad_(), w.requires_grad_()
    for reduction in ("mean", "sum", "none"):
        weights = torch.randn(rows, generator=g).to(DEV) if reduction == "none" else None
        loss = ops.linear_distillation(h, w, logits, index, temperature=temp, reduction=reduction)
        dh, dw = torch.autograd.grad(loss, (h, w), weights)
        e = _exact_kd(h.detach(), w.detach(), logits, index, temp, None if weights is None else weights.double(),
                      reduction)
        _check(e, loss.detach(), dh, dw, dtype, reduction)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_ids_in_a_row_add_up(native_backend, dtype):
    h, w, g = _make(40, 64, 50, dtype)
    index = torch.randint(0, 50, (40, 70), generator=g).to(DEV)
    logits = torch.randn(40, 70, generator=g).to(DEV)
    h.requires_grad_(), w.requires_grad_()
    loss = ops.linear_distillation(h, w, logits, index)
    dh, dw = torch.autograd.grad(loss, (h, w))
    _check(_exact_kd(h.detach(), w.detach(), logits, index), loss.detach(), dh, dw, dtype, "mean")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_left_out_rows_hold_anything(native_backend, dtype, reduction):
    """NaN and infinities in rows without a target reach nothing."""
    h, w, g = _make(200, 136, 300, dtype)
    y = _targets(200, 300, g, 0.5)
    clean = torch.where((y != IGNORE)[:, None], h, torch.zeros_like(h))
    h[y == IGNORE] = float("nan")
    h[(y == IGNORE).nonzero()[0]] = float("inf")
    outs = []
    for x in (h, clean):
        x, v = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = ops.linear_cross_entropy(x, v, y, reduction=reduction)
        outs.append((loss.detach(), *torch.autograd.grad(loss.sum(), (x, v))))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and torch.isfinite(a).all()
    assert not outs[0][1][y == IGNORE].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [0, 1, 130])
def test_no_row_counts(native_backend, dtype, rows):
    h, w, _ = _make(rows, 72, 130, dtype)
    h.requires_grad_(), w.requires_grad_()
    y = torch.full((rows,), IGNORE, device=DEV)
    index, logits = torch.full((rows, 3), -1, device=DEV), torch.zeros(rows, 3, device=DEV)
    for reduction in ("mean", "sum", "none"):
        for loss in (ops.linear_cross_entropy(h, w, y, reduction=reduction),
                     ops.linear_distillation(h, w, logits, index, reduction=reduction)):
            dh, dw = torch.autograd.grad(loss.sum(), (h, w))
            assert not loss.any() and not dh.any() and not dw.any()
            assert loss.shape == ((rows,) if reduction == "none" else ())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("keep", [1.0, 0.3])
def test_chunks_of_rows(native_backend, dtype, keep, monkeypatch):
    """The smallest chunks (256 rows): dW sums over them, and left-out rows
    leave the last ones empty."""
    h, w, g = _make(1111, 136, 520, dtype)
    y = _targets(1111, 520, g, keep)
    h.requires_grad_(), w.requires_grad_()
    monkeypatch.setattr(type(native_backend), "LOSS_CHUNK_BYTES", 1)
    for reduction in ("mean", "none"):
        weights = torch.randn(1111, generator=g).to(DEV) if reduction == "none" else None
        loss = ops.linear_cross_entropy(h, w, y, reduction=reduction)
        dh, dw = torch.autograd.grad(loss, (h, w), weights)
        e = _exact_ce(h.detach(), w.detach(), y, 0.0, 0.0, None if weights is None else weights.double(), reduction)
        _check(e, loss.detach(), dh, dw, dtype, reduction)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_rows_than_a_grid_is_high(native_backend, dtype):
    """70001 rows in one chunk, a small vocabulary."""
    h, w, g = _make(70001, 64, 40, dtype)
    y = _targets(70001, 40, g, 0.99)
    h.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(h, w, y, reduction="sum")
    dh, dw = torch.autograd.grad(loss, (h, w))
    _check(_exact_ce(h.detach(), w.detach(), y, reduction="sum"), loss.detach(), dh, dw, dtype, "sum")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 120, 192])
def test_weights_read_past_their_rows(native_backend, dtype, d):
    """Widths that need padding, the weight at the end of its allocation and
    in the middle of one whose neighbours are not numbers."""
    h, w, g = _make(50, d, 131, dtype)
    y = _targets(50, 131, g)
    pool = torch.full((3 * w.numel(),), float("nan"), dtype=dtype, device=DEV)
    inner = pool[w.numel():2 * w.numel()].view_as(w).copy_(w)
    wide = torch.full((131, d + 8), float("nan"), dtype=dtype, device=DEV)
    slim = wide[:, :d].copy_(w)
    want = None
    for v in (w, inner, slim):
        a, b = h.clone().requires_grad_(), v.detach().requires_grad_()
        loss = ops.linear_cross_entropy(a, b, y)
        got = (loss.detach(), *torch.autograd.grad(loss, (a, b)))
        assert all(torch.isfinite(t).all() for t in got)
        want = want or got
        for s, t in zip(got, want):
            assert torch.equal(s, t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(native_backend, dtype):
    """Views: a slice of wider rows, a weight off its alignment, transposed
    storage, leading dimensions, one shared row; the same values give the same
    bits as contiguous copies."""
    base, w, g = _make(96, 200, 384, dtype)
    y = _targets(96, 384, g)
    odd = torch.empty(w.numel() + 1, dtype=dtype, device=DEV)[1:].view_as(w).copy_(w)
    for h in (base[:, :128], base[:, 3:131], base.T.contiguous().T[:, :128], base[:1, :128].expand(96, 128)):
        for v in (w[:, :128], w[:, 5:133], odd[:, :128], w.T.contiguous().T[:, :128]):
            got = []
            for a, b in ((h, v), (h.contiguous(), v.contiguous())):
                a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
                loss = ops.linear_cross_entropy(a.unflatten(0, (8, 12)), b, y.view(8, 12), reduction="none")
                assert loss.shape == (8, 12)
                got.append((loss.detach(), *torch.autograd.grad(loss.sum(), (a, b))))
            for s, t in zip(*got):
                assert torch.equal(s, t)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_gradient_alone_and_repeats(native_backend, dtype):
    """Each gradient by itself, a factor on the loss, a second backward
    through a retained graph, equal calls with equal bits."""
    h, w, g = _make(150, 128, 900, dtype)
    y = _targets(150, 900, g, 0.8)
    both = []
    for need in ((True, True), (True, False), (False, True), (True, True)):
        a, b = h.clone().requires_grad_(need[0]), w.clone().requires_grad_(need[1])
        loss = ops.linear_cross_entropy(a, b, y)
        inputs = [t for t in (a, b) if t.requires_grad]
        first = torch.autograd.grad(loss, inputs, retain_graph=True)
        second = torch.autograd.grad(loss, inputs, retain_graph=True)
        scaled = torch.autograd.grad(-4.0 * loss, inputs)
        for f, s, x in zip(first, second, scaled):
            assert torch.equal(f, s) and torch.equal(x, -4.0 * f)
        it = iter(first)
        both.append([next(it) if n else None for n in need])
    assert torch.equal(both[0][0], both[1][0]) and torch.equal(both[0][1], both[2][1])
    assert torch.equal(both[0][0], both[3][0]) and torch.equal(both[0][1], both[3][1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_logits(native_backend, dtype):
    """Logits of hundreds: maxima far above the target's, exponentials that
    only the maximum keeps finite."""
    h, w, g = _make(100, 256, 1500, dtype, scale=60.0)
    y = _targets(100, 1500, g)
    h.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(h, w, y, reduction="sum")
    dh, dw = torch.autograd.grad(loss, (h, w))
    _check(_exact_ce(h.detach(), w.detach(), y, reduction="sum"), loss.detach(), dh, dw, dtype, "sum")


def _plane_floor(e):
    """What fp16 planes add to the bounds on (dH, dW), whatever a value's own
    size: fp16 holds multiples of 2^-24, so a plane of a column scaled to a
    maximum of at least 2^13 is off by up to 2^-25·2^-13 of that maximum. dW
    sums S/a by columns against a·H by columns, dH S/a against W's rows times
    the maxima of S/a."""
    a = torch.where(e.a == 0, 1.0, e.a)
    s, ah = (e.S / a).abs(), (e.a * e.h).abs()
    top = s.amax(0)
    floor = 2.0 ** -38
    dw = floor * (top[:, None] * ah.sum(0) + s.sum(0)[:, None] * ah.amax(0))
    scaled = top[:, None] * e.w.abs()
    dh = floor * e.a.abs() * (scaled.sum(0) + (s / top.clamp_min(1e-300)).sum(1, keepdim=True) * scaled.amax(0))
    return dh, dw


# fp32 products take another form from 129 rows on
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [16, 65, 128, 129, 180])
@pytest.mark.parametrize("d,vocab", [(72, 515), (610, 1100), (256, 1500)])
def test_few_rows_and_more_in_float32(native_backend, rows, d, vocab):
    """Wide logits, equal ids, left-out rows that hold anything, an unaligned
    weight whose neighbours are not numbers."""
    h, w, g = _make(rows, d, vocab, torch.float32, seed=rows + d, scale=20.0)
    pool = torch.full((w.numel() + 9,), float("nan"), device=DEV)
    w = pool[5:5 + w.numel()].view_as(w).copy_(w).requires_grad_()
    index = torch.randint(0, 40, (rows, 70), generator=g).to(DEV)
    logits = torch.randn(rows, 70, generator=g).to(DEV)
    y = _targets(rows, vocab, g, 0.7)
    gone = y == IGNORE
    index[gone] = -1
    h[gone] = float("nan")
    h.requires_grad_()
    clean = torch.where(gone[:, None], 0.0, h.detach())
    for reduction in ("mean", "none"):
        weights = torch.randn(rows, generator=g).to(DEV) if reduction == "none" else None
        g_rows = None if weights is None else weights.double()
        for loss, e in ((ops.linear_cross_entropy(h, w, y, reduction=reduction),
                         _exact_ce(clean, w.detach(), y, 0.0, 0.0, g_rows, reduction)),
                        (ops.linear_distillation(h, w, logits, index, temperature=1.5, reduction=reduction),
                         _exact_kd(clean, w.detach(), logits, index, 1.5, g_rows, reduction))):
            dh, dw = torch.autograd.grad(loss, (h, w), weights)
            if rows > 128:
                bl, bh, bw = e.bounds(torch.float32)
                fh, fw = _plane_floor(e)
                e.bounds = lambda dtype: (bl, bh + fh, bw + fw)
            _check(e, loss.detach(), dh, dw, torch.float32, reduction)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_target_outside_the_vocabulary_is_nan(native_backend, dtype):
    h, w, g = _make(140, 64, 200, dtype)
    y = _targets(140, 200, g, 0.7)
    y[3], y[70], y[9] = 200, -1, 5
    loss = ops.linear_cross_entropy(h, w, y, reduction="none")
    bad = torch.zeros(140, dtype=torch.bool, device=DEV)
    bad[3] = bad[70] = True
    assert torch.equal(torch.isnan(loss), bad)
    index = torch.randint(0, 200, (140, 4), generator=g).to(DEV)
    index[5, 2] = 1 << 40
    loss = ops.linear_distillation(h, w, torch.zeros(140, 4, device=DEV), index, reduction="none")
    assert torch.isnan(loss[5]) and int(torch.isnan(loss).sum()) == 1
    h.requires_grad_(), w.requires_grad_()
    for r in ("mean", "none"):
        dh, dw = torch.autograd.grad(ops.linear_cross_entropy(h, w, y, reduction=r).sum(), (h, w))
        assert torch.isnan(dh[3]).all() and torch.isfinite(dh[9]).all() and torch.isnan(dw).any()


@pytest.mark.gpu
def test_stream_of_its_own(native_backend):
    h, w, g = _make(256, 128, 1000, torch.bfloat16)
    y = _targets(256, 1000, g, 0.9)
    want = ops.linear_cross_entropy(h, w, y, reduction="none")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.linear_cross_entropy(h, w, y, reduction="none")
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(want, got)


@pytest.mark.gpu
def test_captured_in_a_graph(native_backend):
    """Nothing waits for the device: a training call records into a graph,
    and replays follow what the targets then hold."""
    h, w, g = _make(256, 128, 1000, torch.bfloat16)
    h.requires_grad_(), w.requires_grad_()
    y = _targets(256, 1000, g, 0.9)
    ys = [y.clone(), _targets(256, 1000, g, 0.2), y.clone()]

    def call():
        loss = ops.linear_cross_entropy(h, w, y)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for t in ys:
        y.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        for a, b in zip(got, call()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_autocast_uses_bfloat16(native_backend):
    h, w, g = _make(64, 128, 500, torch.float32)
    y = _targets(64, 500, g)
    h.requires_grad_(), w.requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = ops.linear_cross_entropy(h, w, y)
    dh, dw = torch.autograd.grad(loss, (h, w))
    assert loss.dtype == dh.dtype == dw.dtype == torch.float32
    a, b = h.detach().bfloat16().requires_grad_(), w.detach().bfloat16().requires_grad_()
    want = ops.linear_cross_entropy(a, b, y)
    eh, ew = torch.autograd.grad(want, (a, b))
    assert torch.equal(loss, want) and torch.equal(dh, eh.float()) and torch.equal(dw, ew.float())


@pytest.mark.gpu
def test_gradient_against_differences(native_backend):
    """The derivative along a direction against central differences of the
    float64 loss: off by the third derivative (1e-6 squared times it) and the
    kernels' own float32 error."""
    h, w, g = _make(20, 64, 90, torch.float32)
    y = _targets(20, 90, g, 0.8)
    logits, index = _teacher(20, 90, 7, g, True)
    vh, vw = (torch.randn(t.shape, generator=g).double().to(DEV) for t in (h, w))
    h.requires_grad_(), w.requires_grad_()
    for loss, f in (
            (ops.linear_cross_entropy(h, w, y, label_smoothing=0.1, z_loss=1e-2),
             lambda a, b: ref.linear_cross_entropy(a, b, y, label_smoothing=0.1, z_loss=1e-2)),
            (ops.linear_distillation(h, w, logits, index, 2.0),
             lambda a, b: ref.linear_distillation(a, b, logits, index, 2.0))):
        dh, dw = torch.autograd.grad(loss, (h, w))
        got = float((dh.double() * vh).sum() + (dw.double() * vw).sum())
        a, b, e = h.detach().double(), w.detach().double(), 1e-5
        want = float(f(a + e * vh, b + e * vw) - f(a - e * vh, b - e * vw)) / (2 * e)
        scale = float((dh.double() * vh).abs().sum() + (dw.double() * vw).abs().sum())
        assert abs(got - want) <= 1e-5 * scale, (got, want)


@pytest.mark.gpu
def test_refusals_on_the_gpu(native_backend):
    h, w, g = _make(4, 8, 16, torch.float32)
    y = _targets(4, 16, g)
    with pytest.raises(OpsArgumentError, match="float32 and bfloat16"):
        ops.linear_cross_entropy(h.double(), w.double(), y)
    with pytest.raises(OpsArgumentError, match="must be on"):
        ops.linear_cross_entropy(h, w, y.cpu())
    with pytest.raises(OpsArgumentError, match="1024"):
        ops.linear_distillation(h, w, torch.zeros(4, 1025, device=DEV), torch.zeros(4, 1025, device=DEV, dtype=torch.long))


# ---------------------------------------------------------------- on the CPU


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("smooth", [0.0, 0.2])
def test_reference_cross_entropy_is_torchs(reduction, smooth):
    h, w, g = _make(12, 8, 11, torch.float64, device="cpu")
    y = _targets(12, 11, g, 0.7, device="cpu")
    h.requires_grad_(), w.requires_grad_()
    got = ops.linear_cross_entropy(h.view(3, 4, 8), w, y.view(3, 4), label_smoothing=smooth, reduction=reduction)
    want = torch.nn.functional.cross_entropy(h @ w.T, y, label_smoothing=smooth, reduction=reduction)
    torch.testing.assert_close(got.reshape(want.shape), want, rtol=1e-12, atol=1e-13)
    a, b = (torch.autograd.grad(x.square().sum(), (h, w)) for x in (got, want))
    for x, z in zip(a, b):
        torch.testing.assert_close(x, z, rtol=1e-11, atol=1e-13)


def test_reference_distillation_is_a_divergence():
    """Against kl_div over the whole vocabulary, masks and temperature."""
    h, w, g = _make(9, 8, 15, torch.float64, device="cpu")
    logits, index = _teacher(9, 15, 6, g, True, device="cpu")
    there = (index >= 0) & (logits != -float("inf"))
    kept = there.any(1)
    assert 0 < int(kept.sum()) < 9
    q = torch.where(there, logits.double() / 3, -float("inf")).softmax(1).nan_to_num(0.0)
    full = torch.zeros(9, 15, dtype=torch.float64).scatter_add_(1, index.clamp_min(0), q)
    logp = torch.log_softmax(h @ w.T / 3, 1)
    want = 9 * torch.nn.functional.kl_div(logp, full, reduction="none").sum(1) * kept
    got = ops.linear_distillation(h, w, logits, index, temperature=3.0, reduction="none")
    torch.testing.assert_close(got, want, rtol=1e-6, atol=1e-6)  # the teacher's logits are float32
    mean = ops.linear_distillation(h, w, logits, index, temperature=3.0)
    torch.testing.assert_close(mean, got.sum() / kept.sum())


def test_reference_left_out_rows():
    h, w, g = _make(6, 4, 7, torch.float32, device="cpu")
    y = torch.tensor([1, IGNORE, 3, IGNORE, 7, -5])
    h[1] = float("nan")
    h.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(h, w, y, reduction="none")
    assert torch.equal(torch.isnan(loss), torch.tensor([False] * 4 + [True] * 2)) and loss[1] == loss[3] == 0
    dh, dw = torch.autograd.grad(ops.linear_cross_entropy(h, w, y.clamp_max(3).masked_fill(y == -5, IGNORE)), (h, w))
    assert torch.isfinite(dw).all() and not dh[1].any() and not dh[3].any() and dh[0].any()
    assert ops.linear_cross_entropy(h, w, torch.full((6,), IGNORE)) == 0
    assert ops.linear_cross_entropy(h[:0], w, y[:0]) == 0


def test_refusals():
    h, w = torch.zeros(4, 8), torch.zeros(16, 8)
    y, t, i = torch.zeros(4, dtype=torch.long), torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.long)
    for match, call in [
            ("hidden", lambda: ops.linear_cross_entropy(h, w[:, :7], y)),
            ("share a floating type", lambda: ops.linear_cross_entropy(h, w.bfloat16(), y)),
            ("share a floating type", lambda: ops.linear_cross_entropy(h.long(), w.long(), y)),
            ("targets does not match", lambda: ops.linear_cross_entropy(h, w, y[:3])),
            ("token ids", lambda: ops.linear_cross_entropy(h, w, y.float())),
            ("label_smoothing", lambda: ops.linear_cross_entropy(h, w, y, label_smoothing=1.5)),
            ("z_loss", lambda: ops.linear_cross_entropy(h, w, y, z_loss=float("nan"))),
            ("reduction", lambda: ops.linear_cross_entropy(h, w, y, reduction="batch")),
            ("no token", lambda: ops.linear_cross_entropy(h, w[:0], y)),
            ("share a shape", lambda: ops.linear_distillation(h, w, t, i[:, :2])),
            ("share a shape", lambda: ops.linear_distillation(h, w, t[:, :0], i[:, :0])),
            ("does not match", lambda: ops.linear_distillation(h, w, t[:2], i[:2])),
            ("token ids", lambda: ops.linear_distillation(h, w, t, t)),
            ("temperature", lambda: ops.linear_distillation(h, w, t, i, temperature=0.0)),
            ("reduction", lambda: ops.linear_distillation(h, w, t, i, reduction=None))]:
        with pytest.raises(OpsArgumentError, match=match):
            call()


def test_library_refusals():
    """The C entry points check on the host; the pointers are never read."""
    import ctypes

    from pytorch_opt.ops import _hip, native_build

    L = _hip.HipBackend(native_build.library_path())._lib
    a = ctypes.c_void_p(0x1000)

    def ce(hidden=a, ldh=8, weight=a, ldw=8, y=a, dtype=0, rows=4, d=8, vocab=16, smooth=0.0, z=0.0, red=1, gr=None,
           loss=a, lse=None, zt=None, dh=None, dw=None, ws=a, nbytes=1 << 30):
        rc = L.pto_linear_cross_entropy(hidden, ldh, weight, ldw, y, dtype, rows, d, vocab, -100, smooth, z, red, gr,
                                        loss, lse, zt, dh, dw, 0, ws, nbytes, None)
        return rc, L.pto_last_error()

    for word, kw in [(b"dtype", dict(dtype=1)), (b"negative", dict(rows=-1)), (b"no features", dict(d=0)),
                     (b"null operand", dict(weight=None)), (b"null operand", dict(y=None)), (b"null loss", dict(loss=None)),
                     (b"pitch", dict(ldw=7)), (b"reduction", dict(red=3)), (b"smoothing", dict(smooth=-0.1)),
                     (b"finite", dict(z=float("inf"))), (b"aligned", dict(weight=ctypes.c_void_p(0x1004))),
                     (b"their gradients", dict(red=0, dh=a)), (b"backward call", dict(gr=a, red=0, dh=a)),
                     (b"workspace", dict(nbytes=64)), (b"null workspace", dict(ws=None))]:
        rc, message = ce(**kw)
        assert rc != 0 and word in message, (word, message)
    rc = L.pto_linear_distillation(a, 8, a, 8, a, a, 0, 4, 8, 16, 1025, 1.0, 1, None, a, None, None, None, None, 0, a,
                                   1 << 30, None)
    assert rc != 0 and b"1024" in L.pto_last_error()
    rc = L.pto_linear_distillation(a, 8, a, 8, a, a, 0, 4, 8, 16, 4, 0.0, 1, None, a, None, None, None, None, 0, a,
                                   1 << 30, None)
    assert rc != 0 and b"temperature" in L.pto_last_error()
    assert L.pto_scale_pair(None, 5, None, 0, 0, a, None) != 0 and b"null" in L.pto_last_error()
    assert L.pto_scale_pair(None, 0, None, 0, 0, None, None) == 0
    small = L.pto_linear_loss_workspace_bytes(2, 1, 2048, 32000, 1, 2048, 0.0, 0, 0, 0, 0, 0)
    assert 0 < small < 1 << 20  # scoring one token keeps no logits
    most = L.pto_linear_loss_workspace_bytes(2, 1 << 16, 4096, 128000, 1, 4096, 0.0, 0, 0, 1, 1, 0)
    assert most < (5 << 30) + 4 * 128000 * 4096  # 2 GiB of logits, dW's sums, statistics
