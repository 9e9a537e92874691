"""Kernels on softmax(logits / temperature) against the same definitions in 64 bits.

Tolerances count roundings.  With u = 2^-24 and span the largest |z - max| / tau of the row that matters (finite ones): the
exponent carries 3 roundings (relative 3 u), the exponential 4 u, a thread adds at most 256 terms of a 65536-wide row and
the tree 14 more, so a sum of exponentials is off by (3 span + 4 + 270) u relative, and its logarithm by as much absolutely.
bf16 results add half a step, 2^-8 relative.
"""

import math

import pytest
import torch

from rwkv7m_b200 import ops
from rwkv7m_b200.ops import reference as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _logits(rows, V, dtype, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, V, generator=g) * scale).to(DT[dtype]).cuda()


def _span(z, tau):
    zf = z.double()
    d = (zf.amax(-1, keepdim=True) - zf) / tau
    d = d[torch.isfinite(d)]
    return float(d.max()) if d.numel() else 0.0


def _sum_tol(z, tau):
    return (3 * min(_span(z, tau), 90.0) + 280) * U


def _check_forward(z, ids, k, tau):
    out = ops.token_logprobs(z, ids, top_k=k, temperature=tau)
    want = R.token_logprobs(z.double(), ids, k, tau)
    span = _span(z, tau)
    tol_lp = _sum_tol(z, tau) + 5 * U * span + 24 * U
    # H = ln S - sum q t: the second sum has the first one's error relative to at most ln V + 1
    tol_h = _sum_tol(z, tau) * (math.log(z.shape[-1]) + 2) * 2
    assert torch.allclose(out.logprob.double(), want[0], atol=tol_lp, rtol=0)
    assert torch.allclose(out.entropy.double(), want[1], atol=tol_h, rtol=0)
    if k:
        assert torch.equal(out.top_ids, want[2])
        assert torch.allclose(out.top_logprobs.double(), want[3], atol=tol_lp, rtol=0)
    return out


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 2), (5, 7), (2, 8), (17, 33), (4, 255), (3, 1000), (9, 2048), (3, 4099),
                                    (130, 8190), (2, 65536), (5, 65529), (1, 200003)])
def test_forward(rows, V, dtype):
    z = _logits(rows, V, dtype, seed=V)
    ids = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(1)).cuda()
    for k, tau in ((0, 1.0), (1, 0.6), (min(V, 5), 1.0), (min(V, 64), 2.5)):
        _check_forward(z, ids, k, tau)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V", [513, 4096, 65536])
def test_forward_difficult_rows(V, dtype):
    g = torch.Generator().manual_seed(3)
    low = torch.finfo(DT[dtype]).min
    ramp = torch.arange(V, dtype=torch.float32)
    rows = [
        torch.full((V,), 1.5),                                   # all equal
        ramp / 64, -ramp / 64,                                   # long runs above any bound
        torch.randint(-2, 3, (V,), generator=g).float(),         # ties everywhere
        torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0),        # equal zeros of either sign
        torch.full((V,), -math.inf).index_fill(0, torch.tensor([5, 300, 77]), 1.0),   # three columns left
        torch.full((V,), -math.inf).index_fill(0, torch.tensor([V - 1]), -3.0),       # one column left
        torch.full((V,), low),                                   # the type's lowest value everywhere
        torch.where(torch.arange(V) < 9, 2.0, low),              # and as a mask
        torch.randn(V, generator=g) + 1000.0,                    # far from zero
        (torch.arange(V) // 256 % 2).float() * 8 + torch.randn(V, generator=g) * 1e-2,
    ]
    z = torch.stack(rows).to(DT[dtype]).cuda()
    ids = torch.randint(0, V, (len(rows),), generator=g)
    ids[5], ids[6], ids[8] = 300, V - 1, 3
    for k in (1, 20, 64):
        _check_forward(z, ids.cuda(), k, 1.0)


def test_rows_in_order_take_the_bisection():
    # block by block falling values: few threads hold everything above the bound
    V = 65536
    z = torch.arange(V, dtype=torch.float32)
    z = (z % 256 < 2).float() * 100 + z * 1e-4
    _check_forward(torch.stack((z, z.flip(0), torch.sort(z).values)).cuda(), torch.tensor([1, 2, 3]).cuda(), 64, 1.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_strides_and_offsets(dtype):
    big = _logits(6, 3001, dtype, seed=9)
    ids = torch.tensor([0, 5, 2999, 17, 2, 8]).cuda()
    views = [big[:, 1:], big[:, 3:2500], big[::2], big[:, :1000], big.view(2, 3, 3001), big[1:2].expand(6, 3001),
             big.t().contiguous().t()]
    for v in views:
        lead = v.shape[:-1]
        i = (ids[: math.prod(lead)] % v.shape[-1]).view(lead)
        x = v.detach().clone(memory_format=torch.preserve_format) if v.stride(-1) == 1 else v
        _check_forward(v, i, 7, 1.3)
        leaf = v.detach().requires_grad_()
        g, = torch.autograd.grad(ops.token_logprobs(leaf, i).logprob.sum(), leaf)
        leaf2 = x.contiguous().requires_grad_()
        g2, = torch.autograd.grad(ops.token_logprobs(leaf2, i).logprob.sum(), leaf2)
        # a row's alignment decides which thread adds which terms, so the two sums S of the same exponentials are each off by
        # at most _sum_tol relative and q = 2^t / S by twice that; (i = id) - q has the same absolute error, q <= 1, and is
        # rounded once (half a step of either result in bf16)
        near = 2 * _sum_tol(v, 1.0) + 2 * U + (2 * 2.0 ** -8 * g.abs() if dtype == "bf16" else 0.0)
        assert ((g.double() - g2.double()).abs() <= near).all()


def test_special_ids_and_nan_rows():
    z = _logits(5, 1000, "fp32")
    z[3, 10] = math.nan
    z[4] = -math.inf
    leaf = z.requires_grad_()
    out = ops.token_logprobs(leaf, torch.tensor([-1, 1000, -100, 4, 4]).cuda(), top_k=3)
    assert out.logprob[:3].tolist() == [0.0, 0.0, 0.0]
    assert torch.isnan(out.logprob[3:]).all() and torch.isnan(out.entropy[3:]).all()
    assert torch.isnan(out.top_logprobs[3:]).all() and ((out.top_ids[3:] >= -1) & (out.top_ids[3:] < 1000)).all()
    assert torch.isfinite(out.entropy[:3]).all()
    # rows that receive no gradient are zero, whatever they hold
    w = torch.tensor([1.0, 1.0, 1.0, 0.0, 0.0]).cuda()
    g, = torch.autograd.grad((out.logprob * w).sum() + (out.entropy[:1]).sum(), leaf)
    assert (g[1:] == 0).all() and (g[0] != 0).any()


def _grad_tol(z, want, mass, tau, dtype):
    """``mass``: sum of the magnitudes that an element of the gradient is added up from."""
    tol = (2 * _sum_tol(z, tau) + 30 * U) * mass + 1e-30
    return tol + (2.0 ** -8 * want.abs() if dtype == "bf16" else 0.0)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,V,k,tau", [(1, 1, 0, 1.0), (4, 9, 2, 0.5), (7, 1000, 0, 1.0), (3, 4099, 20, 2.0), (2, 65536, 5, 1.0),
                                          (33, 8191, 0, 0.8)])
def test_token_logprobs_backward(rows, V, k, tau, dtype):
    z = _logits(rows, V, dtype, seed=rows).requires_grad_()
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, V, (rows,), generator=g).cuda()
    ids[rows // 2] = -1 if rows > 2 else ids[0]
    up = [torch.randn(rows, generator=g).cuda() for _ in range(2)]
    gt = torch.randn(rows, k, generator=g).cuda()
    out = ops.token_logprobs(z, ids, top_k=k, temperature=tau)
    loss = (out.logprob * up[0]).sum() + (out.entropy * up[1]).sum() + ((out.top_logprobs * gt).sum() if k else 0.0)
    got, = torch.autograd.grad(loss, z)
    zd = z.detach().double().requires_grad_()
    lp, h, ti, tl = R.token_logprobs(zd, ids, k, tau)
    ld = (lp * up[0].double()).sum() + (h * up[1].double()).sum() + ((tl * gt.double()).sum() if k else 0.0)
    want, = torch.autograd.grad(ld, zd)
    q = torch.softmax(zd.detach() / tau, -1)
    wsum = up[0].abs() + gt.abs().sum(-1)
    inner = wsum[:, None] + up[1].abs()[:, None] * (2 * math.log(V) + 2 - q.clamp(min=1e-300).log())
    mass = q * inner
    mass.scatter_add_(1, ids.clamp(min=0)[:, None], up[0].abs()[:, None].double())
    if k:
        mass.scatter_add_(1, ti.long(), gt.abs().double())
    assert got.dtype == z.dtype
    assert ((got.double() - want).abs() <= _grad_tol(z.detach(), want, mass / tau, tau, dtype)).all()


def test_entropy_gradient_alone_and_no_gradient():
    z = _logits(4, 777, "fp32").requires_grad_()
    ids = torch.zeros(4, dtype=torch.int32, device="cuda")
    out = ops.token_logprobs(z, ids)
    g, = torch.autograd.grad(out.entropy.sum(), z)
    zd = z.detach().double().requires_grad_()
    want, = torch.autograd.grad(R.token_logprobs(zd, ids)[1].sum(), zd)
    assert torch.allclose(g.double(), want, atol=1000 * U, rtol=0)
    with torch.no_grad():
        assert not ops.token_logprobs(z, ids).logprob.requires_grad


def test_backward_against_differences():
    # central differences of the kernel's own forward along a direction: truncation h^2 f'''/6 and rounding / h
    z = _logits(3, 301, "fp32", scale=1.0)
    ids = torch.tensor([1, 2, 300]).cuda()
    d = torch.randn(z.shape, generator=torch.Generator().manual_seed(5)).cuda()
    t_ids = torch.randint(0, 301, (3, 6), generator=torch.Generator().manual_seed(6)).cuda()
    t = torch.randn(3, 6, generator=torch.Generator().manual_seed(7)).cuda()

    def scores(x):
        o = ops.token_logprobs(x, ids)
        return o.logprob.sum() + 0.5 * o.entropy.sum()

    for f in (scores, lambda x: ops.distill_loss(x, t_ids, t, temperature=1.5)[0]):
        leaf = z.clone().requires_grad_()
        g, = torch.autograd.grad(f(leaf), leaf)
        h = 1e-2
        diff = (float(f(z + h * d)) - float(f(z - h * d))) / (2 * h)
        # values up to 40 carry 40 * 300 u / h = 7e-2 at worst, third derivatives along d are below 10
        assert abs(diff - float((g * d).sum())) < 7e-2


def _teacher(rows, V, K, seed, dtype, absent=True):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (rows, K), generator=g)
    t = (torch.randn(rows, K, generator=g) * 3).to(DT[dtype])
    if absent and rows > 2:
        ids[0] = -1                       # an empty teacher
        ids[1, K // 2:] = V + 3           # and a short one
        t[2, : max(1, K // 3)] = -math.inf
    return ids.cuda(), t.cuda()


@pytest.mark.parametrize("dtype,t_dtype", [("bf16", "bf16"), ("fp32", "fp32"), ("fp32", "bf16")])
@pytest.mark.parametrize("rows,V,K,tau", [(1, 1, 1, 1.0), (5, 9, 3, 2.0), (8, 50, 256, 1.0), (6, 4099, 33, 0.7), (4, 65536, 128, 2.0),
                                          (300, 2048, 8, 1.0)])
def test_distill(rows, V, K, tau, dtype, t_dtype):
    z = _logits(rows, V, dtype, seed=K).requires_grad_()
    t_ids, t = _teacher(rows, V, K, seed=V, dtype=t_dtype)
    g = torch.Generator().manual_seed(4)
    mask = torch.rand(rows, generator=g).cuda()
    mask[-1 if rows > 4 else 0] = 0.0 if rows > 4 else 1.0
    total, count = ops.distill_loss(z, t_ids, t, mask, temperature=tau)
    got, = torch.autograd.grad(total * 0.37, z)
    zd = z.detach().double().requires_grad_()
    w_total, w_count = R.distill_loss(zd, t_ids, t.double(), mask.double(), tau)
    want, = torch.autograd.grad(w_total * 0.37, zd)
    # each row's loss: the student's statistics and the teacher's, a short sum of exponentials over <= 256 alternatives
    t_span = float((t.double().nan_to_num(neginf=0.0).amax() - t.double().nan_to_num(neginf=0.0).amin())) / tau
    row_tol = _sum_tol(z.detach(), tau) + (8 * t_span + 8 * _span(z.detach(), tau) + 300) * U
    tol = float(mask.sum()) * tau * tau * row_tol + U * abs(float(w_total.detach()))
    assert abs(float(total.detach()) - float(w_total.detach())) <= tol
    assert abs(float(count) - float(w_count)) <= 2 * U * float(w_count)
    ids, p = R.teacher_distribution(t_ids, t.double(), V, tau)
    mass = torch.softmax(zd.detach() / tau, -1) * (p.sum(-1, keepdim=True) > 0)
    mass.scatter_add_(1, ids, p)
    mass = mass * (0.37 * tau * mask.double()[:, None])
    tol = _grad_tol(z.detach(), want, mass, tau, dtype) + (8 * t_span + 300) * U * mass
    assert ((got.double() - want).abs() <= tol).all()
    if rows > 4:
        assert (got[0] == 0).all() and (got[-1] == 0).all()


def test_distill_unused_rows_may_hold_anything():
    z = _logits(4, 500, "bf16")
    z[0] = math.nan
    z[2] = math.inf
    z = z.requires_grad_()
    t_ids, t = _teacher(4, 500, 7, 1, "fp32", absent=False)
    t_ids[2] = -1
    mask = torch.tensor([False, True, True, True]).cuda()
    total, count = ops.distill_loss(z, t_ids, t, mask)
    g, = torch.autograd.grad(total, z)
    assert math.isfinite(float(total)) and float(count) == 3.0
    assert torch.isfinite(g).all() and (g[[0, 2]] == 0).all() and (g[[1, 3]] != 0).any()
    n, c = ops.distill_loss(z[:0], t_ids[:0], t[:0])
    assert float(n) == 0.0 and float(c) == 0.0


def test_offsets_past_32_bits():
    rows, V = 33001, 65536
    z = torch.empty(rows, V, dtype=torch.bfloat16, device="cuda")
    z.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    ids = torch.arange(rows, device="cuda") % V
    leaf = z.requires_grad_()
    out = ops.token_logprobs(leaf, ids, top_k=3)
    g, = torch.autograd.grad(out.logprob.sum(), leaf)
    tail = z.detach()[-2:].clone().requires_grad_()
    ref = ops.token_logprobs(tail, ids[-2:], top_k=3)
    g2, = torch.autograd.grad(ref.logprob.sum(), tail)
    assert torch.equal(out.logprob[-2:], ref.logprob) and torch.equal(out.top_ids[-2:], ref.top_ids)
    assert torch.equal(g[-2:], g2)


def test_many_rows_backward():
    # more rows than one launch of the backward covers
    z = _logits(70001, 16, "fp32").requires_grad_()
    ids = torch.arange(70001, device="cuda") % 16
    g, = torch.autograd.grad(ops.token_logprobs(z, ids).logprob.sum(), z)
    zd = z.detach().double().requires_grad_()
    want, = torch.autograd.grad(torch.log_softmax(zd, -1).gather(1, ids[:, None]).sum(), zd)
    assert torch.allclose(g.double(), want, atol=400 * U, rtol=0)


def test_captured_and_replayed():
    z = _logits(6, 5000, "bf16").requires_grad_()
    ids = torch.arange(6, device="cuda")
    t_ids, t = _teacher(6, 5000, 9, 2, "bf16")
    mask = torch.ones(6, device="cuda")

    def step():
        o = ops.token_logprobs(z, ids, top_k=4)
        kd, n = ops.distill_loss(z, t_ids, t, mask, temperature=2.0)
        g, = torch.autograd.grad(o.logprob.sum() + o.entropy.sum() + kd / n, z)
        return o.logprob, o.top_ids, kd, g

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    with torch.no_grad():
        z.copy_(_logits(6, 5000, "bf16", seed=8))
        mask[1] = 0.0
    graph.replay()
    fresh = step()
    for a, b in zip(held, fresh):
        assert torch.equal(a, b)


def test_same_result_on_every_run():
    z = _logits(64, 65536, "bf16")
    ids = torch.arange(64, device="cuda")
    first = ops.token_logprobs(z, ids, top_k=20)
    for _ in range(3):
        again = ops.token_logprobs(z, ids, top_k=20)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_wide_ids_do_not_wrap():
    z = _logits(3, 100, "fp32")
    wide = torch.tensor([2 ** 32 + 7, -2 ** 32 + 7, 2 ** 40], device="cuda")
    assert ops.token_logprobs(z, wide).logprob.tolist() == [0.0, 0.0, 0.0]
    t = torch.zeros(3, 2, device="cuda")
    ids = torch.stack((wide, torch.tensor([3, 4, 5], device="cuda")), dim=1)
    only = ops.distill_loss(z, ids[:, 1:], t[:, 1:])[0]
    assert abs(float(ops.distill_loss(z, ids, t)[0]) - float(only)) <= 4 * U * abs(float(only))


def test_one_row_and_scalars():
    z = _logits(1, 777, "bf16")[0]
    out = ops.token_logprobs(z, torch.tensor(5, device="cuda"), top_k=2)
    want = R.token_logprobs(z.double(), torch.tensor(5, device="cuda"), 2)
    assert out.logprob.shape == () and out.top_ids.shape == (2,) and torch.equal(out.top_ids, want[2])
    assert abs(float(out.logprob) - float(want[0])) <= 2000 * U


def test_positive_and_negative_maxima():
    # exactly k thread maxima are positive: the first bit of the search already separates them
    g = torch.Generator().manual_seed(11)
    z = -torch.rand(4, 65536, generator=g) - 0.1
    for r in range(4):
        z[r, torch.randperm(65536, generator=g)[: 12 + r]] *= -1
    for dtype in (torch.float32, torch.bfloat16):
        x = z.to(dtype).cuda()
        for k in (12, 13, 14, 15, 40):
            _check_forward(x, torch.zeros(4, dtype=torch.long, device="cuda"), k, 1.0)


def test_a_second_derivative_is_refused():
    z = _logits(2, 30, "fp32").requires_grad_()
    g, = torch.autograd.grad(ops.token_logprobs(z, torch.zeros(2, dtype=torch.int32, device="cuda")).logprob.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.square().sum(), z)


def test_two_streams_at_once():
    z = [_logits(300, 20000, "bf16", seed=s).requires_grad_() for s in range(2)]
    ids = torch.arange(300, device="cuda")
    want = [ops.token_logprobs(x, ids, top_k=7) for x in z]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [None, None]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = ops.token_logprobs(z[i], ids, top_k=7)
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_refusals_on_a_gpu():
    z = _logits(2, 10, "fp32")
    ids = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (z.half(), z.double()):
        with pytest.raises(TypeError):
            ops.token_logprobs(bad, ids)
    with pytest.raises(ValueError):
        ops.token_logprobs(z, ids.cpu())
    with pytest.raises(ValueError):
        ops.distill_loss(z, ids[:, None], z[:, :1].cpu())
