"""Operators on softmax(logits / temperature): definitions, gradients and refusals on the CPU."""

import math

import pytest
import torch

from rwkv7m_b200 import ops


def _case(rows=5, V=11, K=4, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, V, generator=g, dtype=torch.float64).mul(2).to(dtype)
    ids = torch.randint(0, V, (rows,), generator=g)
    t_ids = torch.randint(0, V, (rows, K), generator=g)
    t = torch.randn(rows, K, generator=g, dtype=torch.float64).mul(2).to(dtype)
    mask = (torch.rand(rows, generator=g) > 0.3).double()
    return z, ids, t_ids, t, mask


def test_token_logprobs_is_log_softmax():
    z, ids, *_ = _case()
    out = ops.token_logprobs(z, ids, top_k=3, temperature=0.7)
    q = torch.softmax(z / 0.7, -1)
    assert torch.allclose(out.logprob, q.log()[torch.arange(5), ids], atol=1e-12)
    assert torch.allclose(out.entropy, -(q * q.log()).sum(-1), atol=1e-12)
    assert torch.equal(out.top_ids.long(), torch.topk(z, 3).indices)
    assert torch.allclose(out.top_logprobs, torch.topk(q.log(), 3).values, atol=1e-12)


def test_ties_go_to_the_lowest_index():
    z = torch.tensor([[1.0, 3.0, 3.0, 0.0, 3.0], [2.0, 2.0, 2.0, 2.0, 2.0]])
    out = ops.token_logprobs(z, torch.tensor([0, 4]), top_k=4)
    assert out.top_ids.tolist() == [[1, 2, 4, 0], [0, 1, 2, 3]]


def test_ids_outside_the_vocabulary_are_no_token():
    z, *_ = _case()
    z = z.clone().requires_grad_()
    out = ops.token_logprobs(z, torch.tensor([-1, 11, 3, -100, 0]))
    assert out.logprob[[0, 1, 3]].tolist() == [0.0, 0.0, 0.0] and (out.logprob[[2, 4]] < 0).all()
    g, = torch.autograd.grad(out.logprob.sum(), z)
    assert (g[[0, 1, 3]] == 0).all() and (g[[2, 4]] != 0).any()


def test_columns_at_minus_infinity_have_no_part():
    z, ids, *_ = _case()
    masked = z.clone()
    masked[:, 4:] = -math.inf
    masked.requires_grad_()
    cut = z[:, :4].clone().requires_grad_()
    ids = ids % 4
    a, b = ops.token_logprobs(masked, ids), ops.token_logprobs(cut, ids)
    assert torch.allclose(a.logprob, b.logprob) and torch.allclose(a.entropy, b.entropy)
    ga, = torch.autograd.grad((a.logprob + a.entropy).sum(), masked)
    gb, = torch.autograd.grad((b.logprob + b.entropy).sum(), cut)
    assert torch.allclose(ga[:, :4], gb) and (ga[:, 4:] == 0).all()


def test_distill_loss_is_the_divergence():
    z, _, _, t, mask = _case()
    t_ids = torch.stack([torch.randperm(11, generator=torch.Generator().manual_seed(i))[:4] for i in range(5)])
    tau = 2.0
    total, count = ops.distill_loss(z, t_ids, t, mask, temperature=tau)
    p = torch.softmax(t / tau, -1)
    logq = torch.log_softmax(z / tau, -1).gather(1, t_ids)
    want = (tau * tau * (p * (p.log() - logq)).sum(-1) * mask).sum()
    assert torch.allclose(total, want) and float(count) == float(mask.sum())
    # a teacher that gives every column turns the loss into the divergence of two full distributions
    full = torch.arange(11).expand(5, 11)
    kd, _ = ops.distill_loss(z, full, z + 3.0, temperature=tau)
    assert abs(float(kd)) < 1e-12


def test_absent_alternatives_and_empty_rows():
    z, _, t_ids, t, _ = _case()
    t_ids = t_ids.clone()
    t = t.clone()
    t_ids[0] = -1
    t[1] = -math.inf
    t_ids[2, 2:] = torch.tensor([11, -5])
    t[3, 0] = -math.inf
    zr = z.clone()
    zr[0] = math.nan          # nothing of an empty row is used
    zr.requires_grad_()
    mask = torch.ones(5, dtype=torch.float64)
    mask[4] = 0.0
    total, count = ops.distill_loss(zr, t_ids, t, mask)
    want = ops.distill_loss(z[2:3], t_ids[2:3, :2], t[2:3, :2])[0] + ops.distill_loss(z[3:4], t_ids[3:4, 1:], t[3:4, 1:])[0]
    assert torch.allclose(total, want) and float(count) == 4.0
    g, = torch.autograd.grad(total, zr)
    assert (g[[0, 1, 4]] == 0).all() and (g[[2, 3]] != 0).any()


def test_an_id_given_twice_counts_with_both():
    z, _, _, t, _ = _case(rows=1, K=3)
    twice = ops.distill_loss(z, torch.tensor([[2, 7, 2]]), t)[0]
    p = torch.softmax(t, -1)[0]
    logq = torch.log_softmax(z, -1)[0]
    assert torch.allclose(twice, (p * (p.log() - logq[[2, 7, 2]])).sum())


@pytest.mark.parametrize("tau", [1.0, 1.7])
def test_gradients_against_differences(tau):
    z, ids, t_ids, t, mask = _case(rows=3, V=6, K=3)
    z.requires_grad_()
    assert torch.autograd.gradcheck(lambda x: ops.token_logprobs(x, ids % 6, temperature=tau)[:2], (z,))
    assert torch.autograd.gradcheck(lambda x: ops.token_logprobs(x, ids % 6, top_k=2, temperature=tau).top_logprobs, (z,))
    assert torch.autograd.gradcheck(lambda x: ops.distill_loss(x, t_ids % 6, t, mask, temperature=tau)[0], (z,))


def test_shapes_and_empty_inputs():
    z, ids, t_ids, t, _ = _case()
    out = ops.token_logprobs(z[0], ids[0], top_k=2)
    assert out.logprob.shape == () and out.top_ids.shape == (2,)
    out = ops.token_logprobs(z.view(1, 5, 11), ids.view(1, 5), top_k=2)
    assert out.entropy.shape == (1, 5) and out.top_logprobs.shape == (1, 5, 2)
    out = ops.token_logprobs(z[:0], ids[:0])
    assert out.logprob.shape == (0,) and out.top_ids is None
    total, count = ops.distill_loss(z[:0], t_ids[:0], t[:0])
    assert float(total) == 0.0 and float(count) == 0.0


def test_refusals():
    z, ids, t_ids, t, mask = _case()
    bad = [
        (TypeError, lambda: ops.token_logprobs(z.long(), ids)),
        (TypeError, lambda: ops.token_logprobs(z, ids.float())),
        (ValueError, lambda: ops.token_logprobs(z, ids[:4])),
        (ValueError, lambda: ops.token_logprobs(z[:, :0], ids)),
        (ValueError, lambda: ops.token_logprobs(z, ids, top_k=12)),
        (ValueError, lambda: ops.token_logprobs(z, ids, top_k=-1)),
        (ValueError, lambda: ops.token_logprobs(torch.zeros(1, 100), torch.zeros(1, dtype=torch.long), top_k=65)),
        (ValueError, lambda: ops.token_logprobs(z, ids, temperature=0.0)),
        (ValueError, lambda: ops.token_logprobs(z, ids, temperature=math.inf)),
        (ValueError, lambda: ops.distill_loss(z, t_ids, t[:, :0])),
        (ValueError, lambda: ops.distill_loss(z, t_ids[:, :2], t)),
        (ValueError, lambda: ops.distill_loss(z, t_ids[:3], t[:3])),
        (TypeError, lambda: ops.distill_loss(z, t_ids.float(), t)),
        (TypeError, lambda: ops.distill_loss(z, t_ids, t.long())),
        (ValueError, lambda: ops.distill_loss(z, t_ids, t, mask[:2])),
        (ValueError, lambda: ops.distill_loss(z, t_ids, t.clone().requires_grad_())),
        (ValueError, lambda: ops.distill_loss(z, t_ids, t, temperature=-1.0)),
        (ValueError, lambda: ops.distill_loss(z, t_ids.expand(5, 4).repeat(1, 65), t.repeat(1, 65))),
        (ValueError, lambda: ops.token_logprobs(z, ids.to("meta"))),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()


def test_head_operators_are_the_logit_operators_behind_a_product():
    z, ids, t_ids, t, mask = _case()
    g = torch.Generator().manual_seed(3)
    h = torch.randn(5, 6, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(11, 6, generator=g, dtype=torch.float64, requires_grad=True)
    ids = ids.clone()
    ids[2] = -1
    lp, ent = ops.head_token_logprobs(h, w, ids, temperature=1.3)
    ref = ops.token_logprobs(h @ w.T, ids, temperature=1.3)
    assert torch.allclose(lp, ref.logprob) and torch.allclose(ent, ref.entropy)
    out = ops.head_distill_loss(h, w, ids, mask, t_ids, t, temperature=1.3)
    z = h @ w.T
    kd = ops.distill_loss(z, t_ids, t, mask, temperature=1.3)
    logp = torch.log_softmax(z, -1)
    weight = mask * (ids >= 0)
    assert torch.allclose(out[0], -(logp[torch.arange(5), ids.clamp(min=0)] * weight).sum())
    assert torch.allclose(out[1], weight.sum())
    assert torch.allclose(out[2], 0.5e-4 * z.max(-1).values.square().sum()) and float(out[3]) == 5.0
    assert torch.allclose(out[4], kd[0]) and torch.allclose(out[5], mask.sum())
    assert torch.autograd.gradcheck(lambda a, b: ops.head_token_logprobs(a, b, ids), (h, w))
    assert torch.autograd.gradcheck(lambda a, b: ops.head_distill_loss(a, b, ids, mask, t_ids, t, temperature=2.0)[::2], (h, w))


def test_head_distill_agrees_with_the_head_loss():
    g = torch.Generator().manual_seed(5)
    h, w = torch.randn(2, 6, 8, generator=g), torch.randn(30, 8, generator=g)
    tgt = torch.randint(0, 30, (2, 6), generator=g)
    mask = (torch.rand(2, 6, generator=g) > 0.4).float()
    t_ids, t = torch.randint(0, 30, (2, 6, 4), generator=g), torch.randn(2, 6, 4, generator=g)
    ln_w, ln_b = torch.ones(8), torch.zeros(8)
    want = ops.head_loss(h, ln_w, ln_b, w, tgt, mask)
    got = ops.head_distill_loss(ops.layer_norm(h, ln_w, ln_b), w, tgt, mask, t_ids, t)
    for a, b in zip(got[:4], want):
        assert torch.allclose(a, b, rtol=1e-5)


def test_head_refusals():
    z, ids, t_ids, t, mask = _case()
    h, w = torch.randn(5, 6), torch.randn(11, 6)
    bad = [
        (TypeError, lambda: ops.head_token_logprobs(h.long(), w, ids)),
        (TypeError, lambda: ops.head_token_logprobs(h, w.long(), ids)),
        (ValueError, lambda: ops.head_token_logprobs(h, w[:, :5], ids)),
        (ValueError, lambda: ops.head_token_logprobs(h, w[0], ids)),
        (ValueError, lambda: ops.head_token_logprobs(h, w[:0], ids)),
        (ValueError, lambda: ops.head_token_logprobs(h, w, ids[:2])),
        (ValueError, lambda: ops.head_token_logprobs(h, w, ids, temperature=0)),
        (ValueError, lambda: ops.head_token_logprobs(h, w.to("meta"), ids)),
        (ValueError, lambda: ops.head_distill_loss(h, w, ids[:2], mask, t_ids, t)),
        (ValueError, lambda: ops.head_distill_loss(h, w, ids, mask[:1], t_ids, t)),
        (ValueError, lambda: ops.head_distill_loss(h, w, ids, mask, t_ids[:, :0], t[:, :0])),
        (TypeError, lambda: ops.head_distill_loss(h, w, ids.float(), mask, t_ids, t)),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
