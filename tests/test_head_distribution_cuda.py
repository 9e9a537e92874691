"""Log-probabilities and distillation through the head against the same definitions in 64 bits.

Tolerances count roundings.  A logit is a sum of C exact products of bf16 numbers in fp32, 16 of them and the accumulator in
one step that may drop what lies 2^-23 below its largest term: at most 17 (C / 16 + 1) 2^-23 of sum |h w|.  A row's results
add the roundings of its sum of exponentials (one tile of 256 columns adds 2 x 16 per chunk, then 8 chunks and the tiles).
The gradient of the logits is rounded once to bf16 (2^-8 relative) before the two products, whose results are rounded once.
Logits that are kept for the backward pass are fp16 distances d below the largest of their 64 columns: half a step is 2^-11 |d|,
an error of the exponent and so a relative one of the softmax terms (and 2^-25 absolute below fp16's normal range).
"""

import math

import pytest
import torch

from rwkv7m_b200 import ops
from rwkv7m_b200.ops import reference as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _K():
    from rwkv7m_b200.ops import cuda as K

    return K


@pytest.fixture(params=[(0, 4 << 30), (1, 4 << 30), (1, 0)], ids=["single", "pair", "recompute"], autouse=True)
def _modes(request, monkeypatch):
    """The single-CTA and the CTA-pair product, logits kept for the backward pass and computed again."""
    kk = _K()
    old = kk.GEMM_PAIR
    pair, keep = request.param
    kk.set_gemm_pair(bool(pair))
    monkeypatch.setattr(kk, "HEAD_KEEP_BYTES", keep)
    kk.gemm_error_reset(torch.zeros(1, device="cuda"))
    yield
    kk.set_gemm_pair(old)
    assert kk.gemm_error_code(torch.zeros(1, device="cuda")) == 0


def _operands(M, V, C, seed=0, w_dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    h = torch.randn(M, C, generator=g).to(torch.bfloat16).cuda()
    w = (torch.randn(V, C, generator=g) * (2.0 / math.sqrt(C))).to(torch.bfloat16).to(w_dtype).cuda()
    ids = torch.randint(0, V, (M,), generator=g).cuda()
    return h.requires_grad_(), w.requires_grad_(), ids


def _double(*xs):
    return [x.detach().double().requires_grad_() for x in xs]


def _z_error(h, w):
    C = h.shape[1]
    return 17 * (C / 16 + 1) * 2 * U * float((h.detach().double().abs() @ w.detach().double().abs().T).max())


def _row_tol(h, w, z, tau):
    span = float((z.detach().amax(-1) - z.detach().amin(-1)).max()) / tau
    return 2 * _z_error(h, w) / tau + (8 * span + 100 + 4 * math.log(z.shape[1])) * U


def _kept_error(z, terms, tau):
    """Error of the gradient of the logits from keeping them as distances, where ``terms`` are the magnitudes of its softmax
    terms: (2^-11 |d| + 2^-25) / tau of each, 5 % on top for the second order."""
    if _K().HEAD_KEEP_BYTES == 0:
        return 0.0
    M, V = z.shape
    padded = torch.full((M, (V + 63) // 64 * 64), -math.inf, dtype=z.dtype, device=z.device)
    padded[:, :V] = z.detach()
    top = padded.view(M, -1, 64).amax(-1, keepdim=True).expand(M, -1, 64).reshape(M, -1)[:, :V]
    return terms * ((top - z.detach()) * 2.0 ** -11 + 2.0 ** -25) * (1.05 / tau)


def _check_grads(got, want, dz, row_tol, h, w, kept=0.0):
    """``dz``: the gradient of the logits in 64 bits, ``row_tol``: how far an exponent may be off, ``kept``: absolute errors of
    the elements of dz besides."""
    rel = 2.0 ** -8 + 2 * row_tol
    mag = dz.abs() + 1e-30 + kept / rel
    # absolute part: q (A + B ln q) with a rounded sum of two terms of opposite sign is covered by their magnitudes
    for g, wt, mass in ((got[0], want[0], mag @ w.detach().double().abs()),
                        (got[1], want[1], mag.T @ h.detach().double().abs())):
        if g is None:
            continue
        tol = rel * mass + (2.0 ** -8 if g.dtype == torch.bfloat16 else 4 * U) * wt.abs() + 1e-12
        # accumulation of the products in fp32, as for the logits
        tol = tol + 17 * (dz.shape[1] / 16 + 1) * 2 * U * mass
        bad = (g.double() - wt).abs() > tol
        assert not bad.any(), float(((g.double() - wt).abs() / tol).max())


SHAPES = [(1, 1, 8), (1, 7, 16), (3, 256, 64), (5, 300, 64), (64, 1000, 512), (130, 1003, 136), (257, 513, 576), (300, 4099, 512),
          (1000, 9001, 768), (2, 65536, 1024)]


@pytest.mark.parametrize("M,V,C", SHAPES)
@pytest.mark.parametrize("tau", [1.0, 2.3])
def test_head_token_logprobs(M, V, C, tau):
    h, w, ids = _operands(M, V, C, seed=M)
    if M > 4:
        ids[1], ids[3] = -1, V
    g = torch.Generator().manual_seed(1)
    up = [torch.randn(M, generator=g).cuda() for _ in range(2)]
    lp, ent = ops.head_token_logprobs(h, w, ids, temperature=tau)
    got = torch.autograd.grad((lp, ent), (h, w), up)
    hd, wd = _double(h, w)
    zd = hd @ wd.T
    lp2, ent2, _, _ = R.token_logprobs(zd, ids, 0, tau)
    tol = _row_tol(h, w, zd, tau)
    assert (lp.double() - lp2).abs().max() <= tol
    assert (ent.double() - ent2).abs().max() <= tol * 2 * (math.log(V) + 2)
    loss = (lp2 * up[0].double()).sum() + (ent2 * up[1].double()).sum()
    dz, = torch.autograd.grad(loss, zd, retain_graph=True)
    want = torch.autograd.grad(loss, (hd, wd))
    # terms of an element of dz may cancel: bound by their magnitudes
    q = torch.softmax(zd.detach() / tau, -1)
    mass = q * (up[0].abs()[:, None] + up[1].abs()[:, None] * (2 * math.log(V) + 2 - q.log())) / tau
    kept = _kept_error(zd, mass, tau)
    mass.scatter_add_(1, ids.clamp(0, V - 1)[:, None], up[0].abs()[:, None].double() / tau)
    _check_grads(got, want, torch.maximum(dz.abs(), mass * (2 * tol)), tol, h, w, kept)
    if M > 4:
        assert lp[1] == 0 and lp[3] == 0


@pytest.mark.parametrize("M", [1, 2, 31, 32, 33, 63, 64, 65])
@pytest.mark.parametrize("V,C", [(63, 64), (64, 8), (65, 72), (9473, 128), (9537, 64), (18944, 256), (50021, 64)])
def test_few_rows(M, V, C):
    h, w, ids = _operands(M, V, C, seed=V + M)
    ids[0] = V - 1
    ids[M - 1] = 0 if M > 1 else V - 1
    zd = h.detach().double() @ w.detach().double().T
    lp, ent = ops.head_token_logprobs(h, w, ids, temperature=0.7)
    lp2, ent2, _, _ = R.token_logprobs(zd, ids, 0, 0.7)
    tol = _row_tol(h, w, zd, 0.7)
    assert (lp.double() - lp2).abs().max() <= tol and (ent.double() - ent2).abs().max() <= tol * 2 * (math.log(V) + 2)
    g, = torch.autograd.grad(lp.sum(), h)
    q = torch.softmax(zd / 0.7, -1)
    dz = -q
    dz[torch.arange(M), ids] += 1.0
    dz = dz / 0.7
    want = dz @ w.detach().double()
    _check_grads((g, None), (want, None), torch.maximum(dz.abs(), q * (4 * tol)), tol, h, w, _kept_error(zd, q / 0.7, 0.7))


@pytest.mark.parametrize("M", [1, 7, 40, 100])
def test_few_rows_after_rows_of_nan(M):
    """What an earlier call left in shared memory stays out of the results: bit for bit the same after clean rows and NaN."""
    h, w, ids = _operands(M, 9473, 1024, seed=M)
    up = torch.ones(M, device="cuda")
    out = []
    for fill in (0.0, math.nan):
        with torch.no_grad():
            ops.head_token_logprobs(torch.full((128, 1024), fill, dtype=torch.bfloat16, device="cuda"), w, torch.zeros(128, dtype=torch.int32, device="cuda"))
        lp, ent = ops.head_token_logprobs(h, w, ids)
        out.append((lp, ent) + torch.autograd.grad((lp, ent), (h, w), (up, up)))
    for a, b in zip(*out):
        assert torch.isfinite(a).all() and torch.equal(a, b)


def test_a_short_last_chunk():
    """More rows than one launch of the statistics takes."""
    h, w, ids = _operands(32768 + 3, 300, 64)
    with torch.no_grad():
        lp, ent = ops.head_token_logprobs(h, w, ids)
        tail = ops.head_token_logprobs(h[-3:], w, ids[-3:])
    assert torch.equal(lp[-3:], tail[0]) and torch.equal(ent[-3:], tail[1])
    zd = h.detach().double() @ w.detach().double().T
    assert (lp.double() - R.token_logprobs(zd, ids)[0]).abs().max() <= _row_tol(h, w, zd, 1.0)


def _teacher(M, V, K, seed, ids=None):
    g = torch.Generator().manual_seed(seed)
    t_ids = torch.randint(0, V, (M, K), generator=g).cuda()
    t = (torch.randn(M, K, generator=g) * 3).cuda()
    if M > 6:
        t_ids[0] = -1                                # no teacher
        t_ids[1, 0] = V + 5                          # absent alternative
        t[2, K // 2:] = -math.inf
        t_ids[3] = t_ids[3, 0]                       # one id in every place
        t_ids[4, K - 1] = ids[4] if ids is not None else 0
    return t_ids, t


@pytest.mark.parametrize("M,V,C,K", [(1, 1, 8, 1), (2, 9, 16, 4), (8, 300, 64, 3), (130, 1003, 136, 33), (300, 4099, 512, 16),
                                     (257, 513, 576, 256), (1000, 9001, 768, 128), (64, 65536, 512, 64)])
@pytest.mark.parametrize("tau", [1.0, 2.0])
def test_head_distill_loss(M, V, C, K, tau):
    h, w, tgt = _operands(M, V, C, seed=K)
    t_ids, t = _teacher(M, V, K, seed=M, ids=tgt)
    g = torch.Generator().manual_seed(2)
    mask = torch.rand(M, generator=g).cuda()
    if M > 6:
        mask[5] = 0.0
        tgt[6] = -100
    out = ops.head_distill_loss(h, w, tgt, mask, t_ids, t, temperature=tau)
    coef = (0.6 / M, 1.0 / M, 0.4 / M)
    got = torch.autograd.grad(out[0] * coef[0] + out[2] * coef[1] + out[4] * coef[2], (h, w))
    hd, wd = _double(h, w)
    zd = hd @ wd.T
    ref = R.distill_components(zd, tgt, mask.double(), t_ids, t.double(), tau)
    tol = _row_tol(h, w, zd, 1.0) + _row_tol(h, w, zd, tau)
    t_span = float((t.nan_to_num(neginf=0.0).amax() - t.nan_to_num(neginf=0.0).amin())) / tau
    kd_tol = tau * tau * (tol + (8 * t_span + 600) * U)
    msum = float(mask.sum()) + 1
    for i, bound in ((0, tol * msum), (1, 4 * U * msum), (2, 1e-4 * float(zd.max().abs()) * 2 * _z_error(h, w) * M + 1e-9), (3, 0.0),
                     (4, kd_tol * msum), (5, 4 * U * msum)):
        assert abs(float(out[i].detach()) - float(ref[i].detach())) <= bound + 4 * U * abs(float(ref[i].detach())), i
    loss = ref[0] * coef[0] + ref[2] * coef[1] + ref[4] * coef[2]
    dz, = torch.autograd.grad(loss, zd, retain_graph=True)
    want = torch.autograd.grad(loss, (hd, wd))
    m = mask.double()[:, None]
    ids, p = R.teacher_distribution(t_ids, t.double(), V, tau)
    mass = torch.softmax(zd.detach() / tau, -1) * (coef[2] * tau * m) + torch.softmax(zd.detach(), -1) * (coef[0] * m)
    kept = _kept_error(zd, mass, min(1.0, tau))
    mass = mass.scatter_add(1, ids, p * coef[2] * tau * m).scatter_add(1, tgt.clamp(0, V - 1)[:, None], coef[0] * m)
    _check_grads(got, want, torch.maximum(dz.abs(), mass * (2 * tol + (8 * t_span + 600) * U)), tol, h, w, kept)


def test_losses_of_one_kind_and_large_differences():
    """The gradient of the logits is written in units of the larger upstream gradient: one loss alone, weights far apart, a
    gradient from L2Wrap alone, none at all."""
    M, V, C, K = 40, 700, 128, 6
    h, w, tgt = _operands(M, V, C, seed=3)
    t_ids, t = _teacher(M, V, K, seed=4, ids=tgt)
    hd, wd = _double(h, w)
    for coef in ((1.0, 0.0, 0.0), (0.0, 0.0, 1.0), (0.0, 1.0, 0.0), (1e-12, 0.0, 3e-3), (-2.0, 0.0, 1e-20), (0.0, 0.0, 0.0)):
        out = ops.head_distill_loss(h, w, tgt, None, t_ids, t, temperature=2.0)
        got = torch.autograd.grad(out[0] * coef[0] + out[2] * coef[1] + out[4] * coef[2], (h, w))
        zd = hd @ wd.T
        ref = R.distill_components(zd, tgt, None, t_ids, t.double(), 2.0)
        loss = ref[0] * coef[0] + ref[2] * coef[1] + ref[4] * coef[2]
        dz, = torch.autograd.grad(loss, zd, retain_graph=True)
        want = torch.autograd.grad(loss, (hd, wd))
        tol = _row_tol(h, w, zd, 1.0)
        mass = torch.softmax(zd.detach(), -1) * abs(coef[0]) + (torch.softmax(zd.detach() / 2, -1) + 1e-4) * 2 * abs(coef[2])
        _check_grads(got, want, torch.maximum(dz.abs(), mass * (4 * tol + 3000 * U)), tol, h, w, _kept_error(zd, mass, 1.0))


def test_logits_far_apart():
    """Distances between logits beyond 65504: probabilities of exactly 0 and 1, and gradients without a NaN."""
    h, w, ids = _operands(20, 600, 64, seed=8)
    big = (h.detach() * 65536).requires_grad_()
    lp, ent = ops.head_token_logprobs(big, w, ids)
    g = torch.autograd.grad((lp, ent), (big, w), (torch.ones_like(lp), torch.ones_like(lp)))
    zmax = (big.detach().float() @ w.detach().float().T).abs().max()
    assert float(zmax) > 2 * 65504
    assert torch.isfinite(lp).all() and torch.isfinite(ent).all() and all(torch.isfinite(x).all() for x in g)
    top = (big.detach().double() @ w.detach().double().T).argmax(-1)
    sure = ops.head_token_logprobs(big, w, top)[0]
    # the runner-up is far behind in nearly every row, so S is the maximum's own term: 2^(m c - fl(m c)), whose exponent is off by
    # half a step of m c, 2^-24 |m| in natural units (m here is near 5e5, where fp32 logits themselves are 2^-5 apart)
    assert float((sure >= -2 * U * float(zmax)).float().mean()) > 0.8
    t_ids, t = _teacher(20, 600, 5, 1)
    out = ops.head_distill_loss(big, w, ids, None, t_ids, t, temperature=2.0)
    g = torch.autograd.grad(out[0] + out[4], (big, w))
    assert all(torch.isfinite(x).all() for x in g)


def test_several_chunks_and_main_gradient(monkeypatch):
    kk = _K()
    h, w, ids = _operands(150, 1003, 256)
    up = torch.ones(150, device="cuda") / 150

    def grads(weight):
        lp, ent = ops.head_token_logprobs(h, weight, ids)
        return torch.autograd.grad((lp, ent), (h, weight), (up, up), allow_unused=True)

    h, w, ids = _operands(600, 1003, 256)
    up = torch.ones(600, device="cuda") / 600
    one = grads(w)
    monkeypatch.setattr(kk, "HEAD_GRAD_BYTES", 1)         # 256 rows at a time
    many = grads(w)
    # the same roundings of dz; dW is added up in another order in fp32 and rounded once either way
    assert torch.equal(one[0], many[0])
    assert (one[1].double() - many[1].double()).abs().max() <= 2 * 2.0 ** -8 * float(one[1].abs().max())
    w32 = w.detach().float().requires_grad_()
    g32 = grads(w32)
    assert g32[1].dtype == torch.float32
    assert (g32[1].double() - one[1].double()).abs().max() <= 1.01 * 2.0 ** -8 * float(one[1].abs().max())
    held = w.detach().float().requires_grad_()
    held._main_grad = torch.full((1003, 256), 0.5, device="cuda")
    got = grads(held)
    assert got[1] is None
    # fp32 sums of the same terms on top of 0.5: half a step of numbers near 0.5 per chunk
    assert (held._main_grad - 0.5 - g32[1]).abs().max() <= 3 * 2.0 ** -24 + 4 * U * float(g32[1].abs().max())


def test_frozen_sides():
    h, w, ids = _operands(70, 500, 128)
    both = torch.autograd.grad(ops.head_token_logprobs(h, w, ids)[0].sum(), (h, w))
    only_h, = torch.autograd.grad(ops.head_token_logprobs(h, w.detach(), ids)[0].sum(), (h,))
    only_w, = torch.autograd.grad(ops.head_token_logprobs(h.detach(), w, ids)[0].sum(), (w,))
    assert torch.equal(both[0], only_h) and torch.equal(both[1], only_w)
    with torch.no_grad():
        assert not ops.head_token_logprobs(h, w, ids)[0].requires_grad


def test_gradient_of_one_side_alone():
    """Asking for the gradient of the hidden states leaves a bound main gradient of the head as it was."""
    h, w, ids = _operands(70, 500, 128)
    t_ids, t = _teacher(70, 500, 5, 3)
    calls = (lambda head: ops.head_token_logprobs(h, head, ids)[0].sum(),
             lambda head: ops.head_distill_loss(h, head, ids, None, t_ids, t)[4])
    for call in calls:
        both = torch.autograd.grad(call(w), (h, w))
        assert torch.equal(both[0], torch.autograd.grad(call(w), (h,))[0])
        assert torch.equal(both[1], torch.autograd.grad(call(w), (w,))[0])
        held = w.detach().clone().requires_grad_()
        held._main_grad = torch.full((500, 128), 0.5, device="cuda")
        assert torch.equal(both[0], torch.autograd.grad(call(held), (h,))[0])
        assert (held._main_grad == 0.5).all()


def test_many_rows_of_a_small_vocabulary():
    """More rows than a launch's second grid axis holds."""
    M, V, C = 70001, 24, 16
    h, w, ids = _operands(M, V, C)
    lp, ent = ops.head_token_logprobs(h, w, ids)
    got = torch.autograd.grad((lp[-40:].sum() + lp[:40].sum(),), (h, w))
    hd, wd = _double(h, w)
    zd = hd @ wd.T
    ref = R.token_logprobs(zd, ids)
    tol = _row_tol(h, w, zd, 1.0)
    assert (lp - ref[0]).abs().max() <= tol
    want = torch.autograd.grad((ref[0][-40:].sum() + ref[0][:40].sum(),), (hd, wd, zd))
    q = torch.softmax(zd.detach(), -1)
    terms = torch.zeros_like(q)
    terms[-40:], terms[:40] = q[-40:], q[:40]
    _check_grads(got, want, want[2], tol, h, w, kept=_kept_error(zd, terms, 1.0))


def test_layouts_and_other_types():
    h, w, ids = _operands(48, 300, 64)
    want = ops.head_token_logprobs(h.detach(), w.detach(), ids)
    wide = torch.zeros(48, 130, dtype=torch.bfloat16, device="cuda")
    wide[:, 1:65] = h.detach()
    views = [wide[:, 1:65], h.detach().view(6, 8, 64), h.detach().t().contiguous().t()]
    for v in views:
        lp, ent = ops.head_token_logprobs(v, w.detach(), ids.view(v.shape[:-1]))
        assert lp.shape == v.shape[:-1]
        assert torch.equal(lp.reshape(-1), want[0]) and torch.equal(ent.reshape(-1), want[1])
    pad = torch.zeros(300, 72, dtype=torch.bfloat16, device="cuda")
    pad[:, :64] = w.detach()
    assert torch.equal(ops.head_token_logprobs(h.detach(), pad[:, :64], ids)[0], want[0])
    # widths and types without a head kernel go through fp32 logits
    for hh, ww in ((h.detach().float(), w.detach().float()), (h.detach()[:, :59], w.detach()[:, :59])):
        lp, ent = ops.head_token_logprobs(hh, ww, ids)
        ref = R.token_logprobs(hh.double() @ ww.double().T, ids)
        # an fp32 product of at most 64 terms: 64 roundings of sum |h w|
        tol = 2 * 64 * U * float((hh.double().abs() @ ww.double().abs().T).max()) + 500 * U
        assert (lp - ref[0]).abs().max() <= tol and (ent - ref[1]).abs().max() <= 12 * tol
    t_ids, t = _teacher(48, 300, 5, 1)
    a = ops.head_distill_loss(h, w, ids, None, t_ids, t)
    b = ops.head_distill_loss(h.detach().float(), w.detach().float(), ids, None, t_ids, t)
    for x, y in zip(a, b):
        assert abs(float(x.detach()) - float(y)) <= 48 * 2e-4
    e = ops.head_distill_loss(h[:0], w, ids[:0], None, t_ids[:0], t[:0])
    assert [float(x.detach()) for x in e] == [0.0] * 6
    lp, ent = ops.head_token_logprobs(h[:0], w, ids[:0])
    assert lp.shape == (0,) and ent.shape == (0,)


def test_gradient_against_differences():
    # hidden states on a grid of 1/8 and steps of 1/16 are exact in bf16
    g = torch.Generator().manual_seed(9)
    h = (torch.randint(-8, 9, (6, 64), generator=g) / 8).bfloat16().cuda()
    w = (torch.randn(90, 64, generator=g) * 0.2).bfloat16().cuda()
    d = torch.randint(-1, 2, (6, 64), generator=g).bfloat16().cuda()
    ids = torch.randint(0, 90, (6,), generator=g).cuda()
    t_ids, t = _teacher(6, 90, 4, 3)

    def f(x):
        lp, ent = ops.head_token_logprobs(x, w, ids)
        out = ops.head_distill_loss(x, w, ids, None, t_ids, t, temperature=2.0)
        return lp.sum() + 0.3 * ent.sum() + out[0] + 0.5 * out[4] + out[2]

    leaf = h.clone().requires_grad_()
    grad, = torch.autograd.grad(f(leaf), leaf)
    s = 1 / 16
    diff = (float(f(h + s * d)) - float(f(h - s * d))) / (2 * s)
    want = float((grad.double() * d.double()).sum())
    # along d a logit moves by |w d| <= 0.2 * 64^0.5 * 3 = 4.8 a unit, 0.3 a step: the third-order term is at most
    # 6 rows * 4 terms * 4.8^3 / 6 * s^2 = 1.7; the gradient's own rounding is 2^-8 of its mass
    assert abs(diff - want) <= 1.7 + 2.0 ** -6 * float((grad.double().abs() * d.double().abs()).sum())


def test_captured_together_and_replayed():
    h, w, ids = _operands(40, 3000, 256)
    t_ids, t = _teacher(40, 3000, 9, 2)
    mask = torch.ones(40, device="cuda")

    def step():
        lp, ent = ops.head_token_logprobs(h, w, ids)
        out = ops.head_distill_loss(h, w, ids, mask, t_ids, t, temperature=2.0)
        grads = torch.autograd.grad(lp.sum() + ent.sum() + out[0] + out[4] + out[2], (h, w))
        return [lp.detach(), out[4].detach(), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        h.mul_(-0.5)
        mask[3] = 0.0
    graph.replay()
    for a, b in zip(held, step()):
        assert torch.equal(a, b)


def test_refusals_on_a_gpu():
    h, w, ids = _operands(4, 32, 16)
    with pytest.raises(TypeError):
        ops.head_token_logprobs(h.half(), w, ids)
    with pytest.raises(TypeError):
        ops.head_token_logprobs(h, w.half(), ids)
    with pytest.raises(ValueError):
        ops.head_token_logprobs(h, w.cpu(), ids)
