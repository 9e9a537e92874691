"""Scores and distillation through the public API: generation, scoring, a teacher's targets, the training step."""

import json
import math

import pytest
import torch

import rwkv7m_b200 as R
from rwkv7m_b200 import ops
from rwkv7m_b200.state import init_rwkv_state, init_screen_state
from rwkv7m_b200.train.train_step import accumulate_gradients, generate_toy_batch, initialize_train_state, model_loss

PHASE = "read_screening_only"


def _cfg(**kw):
    return R.tiny_config(vocab_size=62, d_model=32, n_heads=2, use_screening=False, **kw)


def _runtime(device=None, **kw):
    return R.create_runtime(3, _cfg(**kw), device=device)


def _states(cfg, B, device=None):
    return init_rwkv_state(B, cfg, device=device), init_screen_state(B, cfg.screening, device=device)


def test_generated_tokens_come_with_their_scores():
    rt = _runtime()
    prompt = [[1, 2, 3], [4, 5, 6]]
    plain = R.generate_ids(rt, prompt, max_new_tokens=4, temperature=0.0)
    R.reset_runtime_state(rt)
    ids, scores = R.generate_ids(rt, prompt, max_new_tokens=4, temperature=0.0, top_logprobs=3)
    assert torch.equal(ids, plain)
    assert scores.logprob.shape == (2, 4) and scores.top_ids.shape == (2, 4, 3)
    # greedy: the token is the first alternative
    assert torch.equal(scores.top_ids[..., 0], ids) and torch.equal(scores.top_logprobs[..., 0], scores.logprob)
    whole = torch.cat((torch.tensor(prompt, dtype=torch.int32), ids), dim=1)
    again = R.score_ids(rt, whole, top_k=3)
    assert torch.allclose(again.logprob[:, 2:], scores.logprob, atol=1e-5)
    assert torch.allclose(again.entropy[:, 2:], scores.entropy, atol=1e-5)
    R.reset_runtime_state(rt)
    _, none = R.generate_ids(rt, prompt, max_new_tokens=2, temperature=0.0, top_logprobs=0)
    assert none.top_ids is None and none.logprob.shape == (2, 2)


def test_scores_of_a_text():
    rt = _runtime()
    ids = torch.randint(0, 61, (3, 9), generator=torch.Generator().manual_seed(1))
    held = rt.rwkv_state
    out = R.score_ids(rt, ids, temperature=0.8)
    assert rt.rwkv_state is held
    with torch.no_grad():
        logits = rt.model(ids[:, :-1].int(), *_states(rt.config, 3))[0]
    logq = torch.log_softmax(logits / 0.8, -1)
    assert torch.allclose(out.logprob, logq.gather(-1, ids[:, 1:, None])[..., 0], atol=1e-5)
    assert torch.allclose(out.entropy, -(logq.exp() * logq).sum(-1), atol=1e-5)
    assert R.score_ids(rt, ids[0]).logprob.shape == (1, 8)
    for bad in (ids[:, :1], torch.tensor([4])):
        with pytest.raises(ValueError):
            R.score_ids(rt, bad)


def test_long_texts_are_scored_in_slices():
    rt = _runtime()
    ids = torch.randint(0, 61, (600, 10), generator=torch.Generator().manual_seed(2))   # 4096 // 600 = 6 positions a slice
    out = R.score_ids(rt, ids, top_k=2)
    few = R.score_ids(rt, ids[:5], top_k=2)
    assert out.top_ids.shape == (600, 9, 2) and torch.allclose(out.logprob[:5], few.logprob, atol=1e-5)


def test_a_teachers_targets():
    rt = _runtime()
    ids = torch.randint(0, 61, (2, 7), generator=torch.Generator().manual_seed(1))
    t = R.teacher_targets(rt, ids, top_k=5)
    with torch.no_grad():
        logits = rt.model(ids.int(), *_states(rt.config, 2))[0]
    want = torch.topk(torch.log_softmax(logits, -1), 5)
    assert torch.equal(t["teacher_ids"].long(), want.indices) and torch.allclose(t["teacher_logits"], want.values, atol=1e-5)
    with pytest.raises(ValueError):
        R.teacher_targets(rt, ids, top_k=0)


def _batch(B=4, T=8, K=5, seed=1):
    batch = generate_toy_batch(seed, B, T, 61)
    batch["mask"][0, 2:5] = 0.0
    teacher = _runtime(n_layers=1)
    batch.update(R.teacher_targets(teacher, batch["input_ids"], top_k=K))
    batch["teacher_ids"][1, 3] = -1
    return batch


def _train_state(distill=R.DistillConfig(weight=0.3, temperature=2.0)):
    ts = initialize_train_state(7, _cfg(), total_steps=10)
    R.set_distillation(ts.model, distill)
    return ts


def _grads(ts):
    return {n: p.grad.clone() for n, p in ts.model.named_parameters() if p.grad is not None}


def test_the_loss_is_the_mixture():
    batch, ts = _batch(), _train_state()
    rs, ss = _states(ts.config, 4)
    total, (metrics, _, _) = model_loss(ts.model, batch, rs, ss, phase=PHASE)
    logits = ts.model(batch["input_ids"], rs, ss, phase=PHASE)[0]
    ce, n, l2, ln = ops.reference.cross_entropy_l2wrap(logits, batch["target_ids"], batch["mask"])
    kd, kn = ops.distill_loss(logits, batch["teacher_ids"], batch["teacher_logits"], batch["mask"], temperature=2.0)
    assert torch.allclose(total, 0.7 * ce / n + 0.3 * kd / kn + l2 / ln, atol=1e-5)
    assert torch.allclose(metrics["loss"], (ce / n).detach(), atol=1e-5)
    assert torch.allclose(metrics["distill_loss"], (kd / kn).detach(), atol=1e-5)
    # evaluation batches without a teacher are unaffected by the setting
    del batch["teacher_ids"], batch["teacher_logits"]
    total, (metrics, _, _) = model_loss(ts.model, batch, rs, ss, phase=PHASE)
    assert torch.allclose(total, ce / n + l2 / ln, atol=1e-5) and "distill_loss" not in metrics


def test_micro_batches_give_the_gradients_of_the_whole():
    batch = _batch()
    got = []
    for steps in (1, 2):
        ts = _train_state()
        rs, ss = _states(ts.config, 4)
        ts.model.zero_grad()
        _, _, metrics = accumulate_gradients(ts.model, batch, rs, ss, phase=PHASE, gradient_accumulation_steps=steps)
        got.append((_grads(ts), {k: float(metrics[k]) for k in ("loss", "distill_loss", "total_loss")}))
    # a batch of 4 and two of 2 run through other matrix shapes: every fp32 operation on the way (about 100 in a chain) may
    # round differently, 100 * 2^-24 = 6e-6 of the largest element; embedding rows of 1e-4 have gradients near 60, so an
    # absolute bound would not do
    for name in got[0][0]:
        a, b = got[0][0][name], got[1][0][name]
        assert (a - b).abs().max() <= 1e-5 * a.abs().max() + 2e-6, name
    for k, v in got[0][1].items():
        assert abs(v - got[1][1][k]) < 1e-5


def test_training_on_a_teacher_through_the_api():
    batch = _batch(B=2)
    runtime, state = R.create_train_runtime(0, _cfg(), batch_size=2, total_steps=4)
    with pytest.raises(ValueError, match="set_distillation"):
        R.train_batch(state, batch, runtime)
    R.set_distillation(runtime.model, R.DistillConfig())
    before = {n: p.detach().clone() for n, p in state.model.named_parameters()}
    for _ in range(2):      # the schedule's first rate is zero
        state, metrics = R.train_batch(state, batch, runtime)
    assert math.isfinite(float(metrics["distill_loss"])) and math.isfinite(float(metrics["loss"]))
    assert any(not torch.equal(before[n], p) for n, p in state.model.named_parameters())


def test_settings_are_checked():
    for bad in (dict(weight=-0.1), dict(weight=1.5), dict(temperature=0.0), dict(temperature=math.inf)):
        with pytest.raises(ValueError):
            R.DistillConfig(**bad)


def test_a_time_slice_takes_its_part_of_the_teacher():
    from rwkv7m_b200.parallel.context import ContextParallel

    cp = ContextParallel.__new__(ContextParallel)
    cp.rank, cp.world = 1, 2
    batch = _batch(T=8)
    part = cp.slice_batch(batch)
    for key in ("input_ids", "target_ids", "mask", "teacher_ids", "teacher_logits"):
        assert torch.equal(part[key], batch[key][:, 4:])


def _tensor_parallel_rank(rank, init, out):
    import torch.distributed as dist

    from rwkv7m_b200.parallel.tp import TensorParallel

    dist.init_process_group("gloo", init_method=f"file://{init}", rank=rank, world_size=2)
    torch.set_num_threads(1)
    batch = torch.load(out + ".batch")
    results = {}
    for vocab_parallel in (False, True):
        tp = TensorParallel.from_group(vocab_parallel=vocab_parallel)
        ts = initialize_train_state(7, _cfg(), total_steps=10, tp=tp)
        R.set_distillation(ts.model, R.DistillConfig(weight=0.3, temperature=2.0))
        rs = tp.init_rwkv_state(4, ts.config)
        ss = init_screen_state(4, ts.config.screening)
        if vocab_parallel:
            with pytest.raises(ValueError, match="vocab_parallel"):
                model_loss(ts.model, batch, rs, ss, phase=PHASE)
        else:
            total, (metrics, _, _) = model_loss(ts.model, batch, rs, ss, phase=PHASE)
            total.backward()
            results = {"total": float(total.detach()), "kd": float(metrics["distill_loss"])}
            scores = ts.model.compute_token_logprobs(
                ts.model.compute_recurrent_hidden(batch["input_ids"], rs, ss)[0], batch["target_ids"], top_k=2)
            results["logprob"] = scores.logprob.detach().tolist()
    if rank == 0:
        with open(out, "w") as f:
            json.dump(results, f)
    dist.destroy_process_group()


def test_tensor_parallel_ranks_agree_with_one_process(tmp_path):
    batch, ts = _batch(), _train_state()
    rs, ss = _states(ts.config, 4)
    total, (metrics, _, _) = model_loss(ts.model, batch, rs, ss, phase=PHASE)
    hidden = ts.model.compute_recurrent_hidden(batch["input_ids"], rs, ss)[0]
    want = ts.model.compute_token_logprobs(hidden, batch["target_ids"])
    out = str(tmp_path / "out.json")
    torch.save(batch, out + ".batch")
    torch.multiprocessing.spawn(_tensor_parallel_rank, args=(str(tmp_path / "init"), out), nprocs=2)
    with open(out) as f:
        got = json.load(f)
    assert abs(got["total"] - float(total.detach())) < 1e-4 and abs(got["kd"] - float(metrics["distill_loss"])) < 1e-4
    assert torch.allclose(torch.tensor(got["logprob"]), want.logprob.detach(), atol=1e-4)


def test_the_generation_tool_records_scores(tmp_path):
    from rwkv7m_b200.cli import generate
    from rwkv7m_b200.io import save_model_safetensors

    cfg = R.tiny_config(vocab_size=65536, d_model=32, n_heads=2, use_screening=False)
    rt = R.create_runtime(1, cfg)
    path = tmp_path / "model.safetensors"
    save_model_safetensors(path, rt.variables["params"], cfg)
    base = ["--checkpoint", str(path), "--prompt", "hi", "--max-new-tokens", "3", "--temperature", "0", "--device", "cpu"]
    text = generate.main(base)
    assert generate.main(base + ["--top-logprobs", "2", "--json-out", str(tmp_path / "o.json")]) == text
    tokens = json.loads((tmp_path / "o.json").read_text(encoding="utf-8"))["samples"][0]["tokens"]
    assert len(tokens) == 3
    for t in tokens:
        assert t["logprob"] <= 0 and t["entropy"] >= 0 and len(t["top"]) == 2 and t["top"][0]["id"] == t["id"]
    for bad in (["--top-logprobs", "2"], ["--top-logprobs", "65", "--json-out", "x"]):
        with pytest.raises(SystemExit):
            generate.parse_args(base + bad)


# ---- on a GPU: the same paths through the kernels ----------------------------------------------------------------------------


def _gpu_cfg():
    return R.ModelConfig(d_model=256, d_ffn=512, n_layers=2, n_heads=4, head_size=64, vocab_size=2000, max_seq_len=256,
                         dtype="bfloat16", use_screening=False)


@pytest.mark.gpu
def test_gpu_generation_and_scores():
    rt = R.create_runtime(3, _gpu_cfg(), batch_size=2, device="cuda")
    prompt = torch.randint(0, 2000, (2, 20), generator=torch.Generator().manual_seed(1))
    runs = []
    for n in (4, 12):            # eager decoding and the captured step
        R.reset_runtime_state(rt)
        ids, s = R.generate_ids(rt, prompt, max_new_tokens=n, temperature=0.0, top_logprobs=5)
        assert torch.equal(s.top_ids[..., 0], ids) and s.top_logprobs.shape == (2, n, 5)
        assert torch.equal(s.top_logprobs[..., 0], s.logprob)
        runs.append((ids, s))
    assert torch.equal(runs[0][0], runs[1][0][:, :4])
    whole = torch.cat((prompt.cuda().int(), runs[1][0]), dim=1)
    a = R.score_ids(rt, whole)                # through the head, fp32 logits
    b = R.score_ids(rt, whole, top_k=5)       # from the bf16 logits
    # a bf16 logit is off by 2^-8 relative, a log-probability by the token's and the mean one's
    with torch.no_grad():
        logits = rt.model(whole[:, :-1], *_states(rt.config, 2, "cuda"))[0]
    tol = 2 * 2.0 ** -8 * float(logits.abs().max())
    assert (a.logprob - b.logprob).abs().max() <= tol
    assert (b.top_logprobs[..., 0] >= b.logprob).all()


@pytest.mark.gpu
def test_gpu_training_step_matches_the_statements():
    cfg = _gpu_cfg()
    batch = {k: v.cuda() for k, v in generate_toy_batch(2, 2, 64, 2000).items()}
    teacher = R.create_runtime(5, cfg, batch_size=2, device="cuda")
    batch.update(R.teacher_targets(teacher, batch["input_ids"], top_k=9))
    batch["mask"][0, :7] = 0.0
    batch["teacher_ids"][1, 5] = -1
    res = []
    for plain in (False, True):
        ts = initialize_train_state(7, cfg, total_steps=10, device="cuda")
        R.set_distillation(ts.model, R.DistillConfig(weight=0.4, temperature=2.0))
        rs, ss = _states(cfg, 2, "cuda")
        with ops.reference_mode(plain):
            hidden, *_ = ts.model.compute_recurrent_hidden(batch["input_ids"], rs, ss, phase=PHASE)
            hidden = hidden.detach().requires_grad_()
            p = ts.model.compute_distill_loss(hidden, batch["target_ids"], batch["mask"], batch["teacher_ids"],
                                              batch["teacher_logits"], temperature=2.0)
            loss = 0.6 * p["ce_total"] / p["ce_count"] + 0.4 * p["kd_total"] / p["kd_count"] + p["l2_total"] / p["l2_count"]
            loss.backward()
        res.append((p, hidden.grad.float()))
    # the statements round logits, softmax input and every product to bf16: relative 2^-8 of logits below 8, a few times over
    for k in ("ce_total", "l2_total", "kd_total"):
        x, y = float(res[0][0][k].detach()), float(res[1][0][k].detach())
        assert abs(x - y) <= 0.05 * abs(y) + 1e-3, k
    for k in ("ce_count", "l2_count", "kd_count"):
        assert float(res[0][0][k]) == float(res[1][0][k])
    a, b = res[0][1], res[1][1]
    assert float((a - b).norm() / b.norm()) < 0.1


@pytest.mark.gpu
def test_gpu_training_runs_and_accumulates():
    cfg = _gpu_cfg()
    batch = generate_toy_batch(2, 4, 64, 2000)
    teacher = R.create_runtime(5, cfg, batch_size=4, device="cuda")
    batch = {k: v.cuda() for k, v in batch.items()}
    batch.update(R.teacher_targets(teacher, batch["input_ids"], top_k=9))
    flats = []
    for steps in (1, 2):
        runtime, state = R.create_train_runtime(0, cfg, batch_size=4, total_steps=10, device="cuda")
        R.set_distillation(runtime.model, R.DistillConfig())
        rs, ss = _states(cfg, 4, "cuda")
        state.optimizer.zero_grad()
        _, _, metrics = accumulate_gradients(state.model, batch, rs, ss, phase=PHASE, gradient_accumulation_steps=steps)
        flats.append(state.optimizer.flat.grad.float().clone())
        state, metrics = R.train_batch(state, batch, runtime, gradient_accumulation_steps=steps)
        assert math.isfinite(float(metrics["distill_loss"])) and math.isfinite(float(metrics["grad_norm"]))
    assert float((flats[0] - flats[1]).norm() / flats[0].norm()) < 0.02      # bf16 activations of other batch shapes
