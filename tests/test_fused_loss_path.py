"""The linear cross entropy and 8-bit optimizer states inside the framework: models, tensor-parallel layouts, trainer, checkpoints."""
import pytest
import torch

from helpers import dummy_dataloader, make_config, run_distributed, single_process_env, tiny_llama_config, tiny_qwen_config
from test_distributed_cpu import _losses_for

gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ CPU, gloo ranks
def _check_linear_ce():
    import nanotron_b200.distributed as dist
    from nanotron_b200.parallel import ParallelContext
    from nanotron_b200.parallel.tensor_parallel.distributed_differentiable_primitives import differentiable_all_gather, differentiable_identity
    from nanotron_b200.parallel.tensor_parallel.functional import linear_cross_entropy_with_z_loss

    ctx = ParallelContext(tensor_parallel_size=2, pipeline_parallel_size=1, data_parallel_size=1)
    rank = dist.get_rank(ctx.tp_pg)
    torch.manual_seed(0)
    x, w = torch.randn(6, 8), torch.randn(16, 8)
    tgt = torch.tensor([0, 7, 8, 15, 3, 12])
    fx, fw = x.clone().requires_grad_(), w.clone().requires_grad_()
    lz = torch.logsumexp(fx @ fw.t(), -1)
    want = torch.nn.functional.cross_entropy(fx @ fw.t(), tgt, reduction="none")
    (want + 1e-2 * lz**2).mean().backward()
    for sharded_tokens in (False, True):
        mine = (x.chunk(2)[rank] if sharded_tokens else x).clone().requires_grad_()
        local = w.chunk(2)[rank].clone().requires_grad_()
        full = differentiable_all_gather(mine, ctx.tp_pg) if sharded_tokens else differentiable_identity(mine, ctx.tp_pg)
        ce, z = linear_cross_entropy_with_z_loss(full, local, tgt, group=ctx.tp_pg, z_loss_coef=1e-2)
        (ce + z).mean().backward()
        torch.testing.assert_close(ce, want, atol=1e-5, rtol=1e-5)
        torch.testing.assert_close(z, 1e-2 * lz**2, atol=1e-6, rtol=1e-5)
        torch.testing.assert_close(local.grad, fw.grad.chunk(2)[rank], atol=1e-6, rtol=1e-4)
        torch.testing.assert_close(mine.grad, fx.grad.chunk(2)[rank] if sharded_tokens else fx.grad, atol=1e-6, rtol=1e-4)
    ctx.destroy()


def test_vocabulary_shards():
    run_distributed(_check_linear_ce, 2)


def test_fused_loss_trains_like_logits_in_every_layout(tmp_path, monkeypatch):
    want = {m: _losses_for(tmp_path, 1, f"logits_{m}", model=m, tie=m == "qwen") for m in ("llama", "qwen", "moe")}
    monkeypatch.setenv("NTB_LOSS", "fused")
    cases = [("llama", 2, dict(tp=2)), ("llama", 2, dict(tp=2, tp_mode="REDUCE_SCATTER")), ("llama", 2, dict(pp=2)), ("qwen", 1, dict(tie=True)), ("moe", 1, {})]
    for i, (model, world, layout) in enumerate(cases):
        got = _losses_for(tmp_path, world, f"fused_{i}", model=model, **layout)
        for a, b in zip(got, want[model]):
            assert abs(a - b) < 2e-4 * b, (model, layout, got, want[model])


def test_scoring_runs_the_head_for_the_scored_positions_alone(tmp_path, monkeypatch):
    from test_eval_cpu import _scorer_run

    def run(name, world, **layout):
        f = str(tmp_path / f"{name}.pt")
        run_distributed(_scorer_run, world, out_file=f, **layout)
        return torch.load(f)

    want = run("logits", 1, tp=1, pp=1)
    monkeypatch.setenv("NTB_LOSS", "fused")
    for world, layout in ((1, dict(tp=1, pp=1)), (4, dict(tp=2, pp=2))):
        got = run(f"fused_{world}", world, **layout)
        for (x, nx), (y, ny) in zip(got["ll"], want["ll"]):
            assert nx == ny and abs(x - y) < 1e-3, (layout, got["ll"], want["ll"])
        assert got["res"] == want["res"]


def _trainer(model_config, loss="logits", state_bits=32, **kw):
    import nanotron_b200.config as c
    from nanotron_b200.trainer import DistributedTrainer

    single_process_env()
    cfg = make_config(model_config, **kw)
    cfg.kernels = c.KernelArgs(loss=loss)
    cfg.optimizer.optimizer_factory = c.AdamWOptimizerArgs(adam_eps=1e-8, adam_beta1=0.9, adam_beta2=0.95, torch_adam_is_fused=False, state_bits=state_bits)
    t = DistributedTrainer(cfg)
    t.prepare_training()
    return t


@pytest.fixture
def default_loss():
    from nanotron_b200 import ops

    yield
    ops.set_loss("logits")


def test_configuration_selects_loss_and_states(default_loss):
    import nanotron_b200.config as c
    from nanotron_b200 import ops
    from nanotron_b200.parallel.tensor_parallel.nn import DeferredLogits

    t = _trainer(tiny_llama_config(), loss="fused", state_bits=8, steps=2)
    assert ops.get_loss() == "fused" and t.optimizer.get_base_optimizer().state_bits == 8
    seen = []
    t.unwrapped_model.loss.pp_block.register_forward_pre_hook(lambda m, a, kw: seen.append(kw["sharded_logits"]), with_kwargs=True)
    batch = next(dummy_dataloader(t))
    t.training_step(iter([batch]))
    assert len(seen) == 1 and isinstance(seen[0], DeferredLogits)
    model = t.unwrapped_model
    model.eval()  # outside the model's own forward (generation) it gives logits
    ids = torch.zeros(1, 4, dtype=torch.long)
    assert torch.is_tensor(model.model(input_ids=ids, input_mask=torch.ones_like(ids, dtype=torch.bool)))
    model.train()
    assert torch.is_tensor(model.model(input_ids=ids, input_mask=torch.ones_like(ids, dtype=torch.bool)))
    states = [s for s in t.optimizer.get_base_optimizer().state.values()]
    assert states and all(s["exp_avg"].dtype == torch.uint8 for s in states)
    t.parallel_context.destroy()
    with pytest.raises(ValueError):
        ops.set_loss("none")
    with pytest.raises(ValueError):
        c.AdamWOptimizerArgs(adam_eps=1e-8, adam_beta1=0.9, adam_beta2=0.95, torch_adam_is_fused=False, state_bits=16)


def _state8_run(out_file, ckpt_dir, steps, first_step=0, save=False, resume=None, **topology):
    """test_checkpoint_cpu._run with 8-bit states."""
    import nanotron_b200.config as c
    import helpers
    import test_checkpoint_cpu as base

    plain = helpers.make_config

    def with_state_bits(*a, **kw):
        cfg = plain(*a, **kw)
        cfg.optimizer.optimizer_factory = c.AdamWOptimizerArgs(adam_eps=1e-8, adam_beta1=0.9, adam_beta2=0.95, torch_adam_is_fused=False, state_bits=8)
        return cfg

    base.make_config = with_state_bits
    base._run(out_file, ckpt_dir, steps, first_step=first_step, save=save, resume=resume, **topology)


@pytest.mark.parametrize("world,layout", [(1, {}), (2, dict(dp=2, zero=1))])
def test_8_bit_states_resume_exactly(tmp_path, world, layout):
    def losses(name, **kw):
        f = str(tmp_path / f"{name}.pt")
        run_distributed(_state8_run, world, out_file=f, ckpt_dir=str(tmp_path / "ckpt"), **layout, **kw)
        return torch.load(f)

    whole = losses("whole", steps=4)
    assert losses("first", steps=2, save=True) == whole[:2]
    rest = losses("rest", steps=2, first_step=2, resume=str(tmp_path / "ckpt"))
    for a, b in zip(rest, whole[2:]):
        assert abs(a - b) < 1e-6, (whole, rest)


# ------------------------------------------------------------------------------------------------ GPU
@gpu
def test_a_training_step_on_the_gpu_takes_both(default_loss):
    """Loss, head gradient (straight into the fp32 buffer), clipping, and the 8-bit step, against the logits path with 32-bit states.

    The two paths share everything below the head.  bf16 logits are off by 2^-8 of their size, which is under 2 here (standard deviation
    0.4), so a loss by 2^-7 at most, a probability by 2^-7 of itself, and an entry of the scores' gradient by that and 2^-8 of its own
    rounding on either path: under 2 %.  The head's gradient sums entries of both signs: 5 % of its norm leaves room for that."""
    mc = tiny_llama_config(hidden_size=256, intermediate_size=512, num_attention_heads=2, num_key_value_heads=2, vocab_size=1000)
    got = {}
    for name, loss, bits in (("logits", "logits", 32), ("fused", "fused", 8)):
        torch.manual_seed(0)
        t = _trainer(mc, loss=loss, state_bits=bits, seq=128, mbs=4, steps=3, dtype="bfloat16", lr=1e-3)
        batch = next(dummy_dataloader(t))
        captured = {}
        acc = t.grad_accumulator
        head = next(n for n in acc.fp32_grad_buffers if "lm_head" in n)
        step = t.optimizer.step

        def before_step(*a, **kw):
            captured.setdefault("grad", acc.get_grad_buffer(head).clone())
            return step(*a, **kw)

        t.optimizer.step = before_step
        losses = [float(t.training_step(iter([batch]))[1]) for _ in range(3)]
        got[name] = (losses, captured["grad"], {n: p.detach().float().clone() for n, p in t.unwrapped_model.named_parameters()})
        t.parallel_context.destroy()
    (la, ga, pa), (lb, gb, pb) = got["logits"], got["fused"]
    assert abs(la[0] - lb[0]) < 2.0**-7, (la, lb)
    assert (ga - gb).norm() < 0.05 * ga.norm()
    assert all(v.isfinite().all() for v in pb.values())


@gpu
def test_head_loss_and_8_bit_step_as_one_captured_loop():
    """Loss -> gradient in the head's fp32 buffer -> clipping coefficient -> 8-bit step, eagerly and as a replayed graph: the same bytes."""
    from nanotron_b200 import ops
    from nanotron_b200.parallel.tensor_parallel.functional import linear_cross_entropy

    T, H, V = 300, 128, 1000
    gen = torch.Generator().manual_seed(0)
    x, y = torch.randn(T, H, generator=gen).to("cuda", torch.bfloat16), torch.randint(0, V, (T,), generator=gen).cuda()
    start = torch.randn(V, H, generator=gen) / H**0.5

    def make():
        master = start.cuda()
        head = torch.nn.Parameter(master.to(torch.bfloat16))
        head.main_grad = torch.zeros_like(master)
        states = [torch.zeros(V, H, dtype=torch.uint8, device="cuda") for _ in range(2)] + [torch.zeros(V * H // 128, dtype=torch.uint8, device="cuda") for _ in range(2)]
        return master, head, states

    def step(master, head, states):
        head.main_grad.zero_()
        loss = linear_cross_entropy(x, head, y).mean()
        loss.backward()
        norm = head.main_grad.norm()
        coef = torch.clamp(0.1 / (norm + 1e-6), max=1.0)
        ops.adamw_multi_tensor([master], [head.main_grad], [states[0]], [states[1]], exp_avg_exponents=[states[2]], exp_avg_sq_exponents=[states[3]], halves=[head.detach()],
                               lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1, step=2, grad_scale=coef, seed=3)
        return loss.detach()

    eager = make()
    losses = [step(*eager) for _ in range(4)]
    graphed = make()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step(*graphed)
    got = []
    for _ in range(4):
        graph.replay()
        got.append(out.clone())
    torch.cuda.synchronize()
    assert torch.equal(torch.stack(got), torch.stack(losses))
    assert torch.equal(eager[0], graphed[0]) and torch.equal(eager[1], graphed[1])
    for a, b in zip(eager[2], graphed[2]):
        assert torch.equal(a, b)
