"""The engine over 4-bit caches, and models with normed query and key heads in it: steps as they are run, against a plain forward in 64 bits."""

import pytest
import torch

from colossalai_amd.inference import ContinuousBatchEngine, GenerationConfig, InferenceConfig, KVCacheManager, LLMEngine
from colossalai_amd.inference.spec_decode import BatchedSpeculativeEngine, GlideSpeculativeEngine, SpeculativeEngine
from colossalai_amd.models import LlamaConfig, LlamaForCausalLM

gpu = pytest.mark.gpu
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _model(norm, dim=64, device="cpu", dtype=torch.float32, **kw):
    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=128, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                      head_dim_override=dim, max_position_embeddings=256, qk_norm=norm, **kw)
    model = LlamaForCausalLM(cfg).eval()
    with torch.no_grad():  # heads that say something, and norms that are not 1
        for name, p in model.named_parameters():
            if "norm" in name:
                p.copy_(1 + 0.3 * torch.randn(p.shape))
            elif p.dim() == 2:
                p.mul_(4.0)
    return model.to(device, dtype)


def _nearest(x):
    """Numbers of a 4-bit cache: the smallest power of two that 6 of reach the group's largest, the nearest numbers, ties to the even one."""
    x = x.unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    powers = torch.exp2(torch.arange(-126, 127, dtype=torch.float64))
    unit = powers[(6 * powers >= most).int().argmax(-1)].unsqueeze(-1)
    away = ((x.abs() / unit).unsqueeze(-1) - GRID).abs()
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])  # even mantissas first: argmin takes the first of equals
    return (torch.sign(x) * GRID[order[away[..., order].argmin(-1)]] * unit).flatten(-2)


def _plain_logits(model, tokens, four):
    """Logits of every position of one sequence, in 64 bits, with keys and values as a 4-bit cache holds them if ``four``."""
    p = {k: v.detach().double().cpu() for k, v in model.named_parameters()}
    cfg, n = model.config, len(tokens)
    H, G, D = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
    norm = lambda x, w, eps: x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w  # noqa: E731
    angle = torch.arange(n, dtype=torch.float64)[:, None] / cfg.rope_theta ** (torch.arange(0, D, 2, dtype=torch.float64) / D)
    c, s = (t.float().double()[:, None] for t in (angle.cos(), angle.sin()))  # tables are float32
    turn = lambda x: torch.cat([x[..., : D // 2] * c - x[..., D // 2:] * s, x[..., D // 2:] * c + x[..., : D // 2] * s], -1)  # noqa: E731
    x = p["model.embed_tokens.weight"][torch.tensor(tokens)]
    for i in range(cfg.num_hidden_layers):
        at = f"model.layers.{i}."
        h = norm(x, p[at + "input_layernorm_weight"], cfg.rms_norm_eps)
        q, k, v = (h @ p[at + "self_attn.qkv_proj.weight"].t()).view(n, -1, D).split([H, G, G], 1)
        if cfg.qk_norm:
            q, k = (norm(t, p[at + f"self_attn.{w}_norm_weight"], cfg.rms_norm_eps) for t, w in ((q, "q"), (k, "k")))
        q, k = turn(q), turn(k)
        if four:
            k, v = _nearest(k), _nearest(v)
        k, v = (t.repeat_interleave(H // G, 1).transpose(0, 1) for t in (k, v))
        w = (q.transpose(0, 1) @ k.transpose(1, 2) * D ** -0.5).masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), -torch.inf)
        x = x + (torch.softmax(w, -1) @ v).transpose(0, 1).reshape(n, -1) @ p[at + "self_attn.o_proj.weight"].t()
        h = norm(x, p[at + "post_attention_layernorm_weight"], cfg.rms_norm_eps)
        gate, up = (h @ p[at + "mlp.gate_up_proj.weight"].t()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ p[at + "mlp.down_proj.weight"].t()
    return norm(x, p["model.norm_weight"], cfg.rms_norm_eps) @ p["lm_head.weight"].t()


def _engine(model, bits, **kw):
    return ContinuousBatchEngine(model, InferenceConfig(max_batch_size=3, max_input_len=96, max_output_len=32, kv_cache_bits=bits), **kw)


PROMPTS = [list(range(3, 40)), [5], [7, 9, 11, 13, 15], list(range(100, 10, -1)), [1, 2, 3]]


@pytest.mark.parametrize("norm,bits", [(True, 16), (True, 4), (False, 4)])
def test_generates_what_a_plain_forward_does(norm, bits):
    """More requests than slots; every token is the one that the plain forward over the sequence so far puts first."""
    model = _model(norm)
    engine = _engine(model, bits, block_size=16)
    out = engine.generate(PROMPTS, GenerationConfig(max_new_tokens=6))
    for p, o in zip(PROMPTS, out):
        logits = _plain_logits(model, o[:-1], bits == 4)
        assert o[len(p):] == logits[len(p) - 1:].argmax(-1).tolist() and len(o) == len(p) + 6
    assert engine.kv.free_blocks == engine.kv.num_blocks


def _steps(engine, device):
    """Logits of prompts in one step, then of single tokens, as the engine runs them."""
    for i, p in enumerate(PROMPTS[:3]):
        engine.kv.allocate(i, len(p) + 4)
    got = [engine._forward_packed([(i, p, 0) for i, p in enumerate(PROMPTS[:3])])]
    for step in range(3):
        got.append(engine._forward_packed([(i, [20 + step], len(p) + step) for i, p in enumerate(PROMPTS[:3])]))
    return torch.stack(got).double().cpu()


@pytest.mark.parametrize("bits,device,dtype,bound", [(16, "cpu", torch.float32, 1e-4), (4, "cpu", torch.float32, 1e-4), (4, "cpu", torch.bfloat16, 0.2),
                                                     pytest.param(16, "cuda", torch.bfloat16, 0.06, marks=gpu),
                                                     pytest.param(4, "cuda", torch.bfloat16, 0.2, marks=gpu)])
def test_logits(bits, device, dtype, bound):
    """float32: some 2^-20 a layer. bfloat16: two layers round their stream, projections and attention some ten times each, 2^-9 on average:
    0.01. In 4 bits the numbers are about 0.3 of their size apart: where bfloat16 leaves keys and values off by r = 4 * 2^-9 of their size, r / 0.3
    of the codes fall on a border's other side and are off by 0.3, sqrt(0.3 r) = 0.05 of the keys and as much of the values, in each of two
    layers: 0.1, and twice that as the bound (a bfloat16 model on the CPU, other code, is as far off)."""
    model = _model(True, 128, device, dtype)
    with torch.inference_mode():
        got = _steps(_engine(model, bits), device)
    for i, p in enumerate(PROMPTS[:3]):
        want = _plain_logits(model, p + [20, 21, 22], bits == 4)[len(p) - 1:]
        off = (got[:, i] - want).norm() / want.norm()
        assert off < bound, f"{off:.2e}"


@gpu
def test_generates_on_a_gpu():
    """The whole loop; the pools take 17 bytes for 64 of bfloat16 ones."""
    model = _model(True, 128, "cuda", torch.bfloat16)
    engine = _engine(model, 4)
    assert engine.kv.k_pools[0].numel() * 16 * 2 == engine.kv.num_blocks * 16 * 2 * 128 * 17
    out = engine.generate(PROMPTS, GenerationConfig(max_new_tokens=5))
    assert [len(o) for o in out] == [len(p) + 5 for p in PROMPTS] and engine.kv.free_blocks == engine.kv.num_blocks


@pytest.mark.parametrize("device,dtype,bound", [("cpu", torch.float32, 1e-5), pytest.param("cuda", torch.bfloat16, 0.05, marks=gpu)])
def test_norms_and_rotation_in_one_pass(device, dtype, bound):
    """``fused_qk_norm`` gives the logits and gradients of the separate steps but for the rounding between them."""
    ids = torch.randint(0, 128, (2, 50), generator=torch.Generator().manual_seed(1)).to(device)
    got = []
    for fused in (False, True):
        model = _model(True, 128, device, dtype, fused_qk_norm=fused).train()
        model(ids, labels=ids)["loss"].backward()
        logits = model(ids)["logits"].detach()
        got.append([logits] + [p.grad for _, p in sorted(model.named_parameters())])
    for a, b in zip(*got):
        assert (a.double() - b.double()).norm() <= bound * b.double().norm()


def test_refusals():
    with pytest.raises(ValueError):
        _engine(_model(True, 32), 4)
    with pytest.raises(ValueError):
        _engine(_model(True), 8)
    with pytest.raises(ValueError):
        _engine(_model(True), 4, block_size=8)
    with pytest.raises(ValueError):
        KVCacheManager(2, 2, 64, num_blocks=4, device="cpu", layer_shapes=[(2, 64, 64)] * 2, bits=4)
    with pytest.raises(ValueError):
        LLMEngine(_model(False), InferenceConfig(kv_cache_bits=4))
    with pytest.raises(ValueError):
        _engine(_model(False, partial_interleaved_rotary_factor=0.5), 4)
    with pytest.raises(ValueError):
        _engine(_model(True, dtype=torch.float16), 16)
    kv = KVCacheManager(1, 2, 64, num_blocks=4, device="cpu", bits=4)
    kv.allocate(0, 20)
    for call in (lambda: kv.write_prefill(0, 0, torch.zeros(3, 2, 64), torch.zeros(3, 2, 64)),
                 lambda: kv.write_token(0, 0, 3, torch.zeros(2, 64), torch.zeros(2, 64))):
        with pytest.raises(ValueError):
            call()
    assert [t.shape for t in kv.gather_contiguous(0, 0, 20)] == [(20, 2, 64)] * 2


@pytest.mark.parametrize("engine", [SpeculativeEngine, BatchedSpeculativeEngine, GlideSpeculativeEngine])
def test_engines_with_caches_of_their_own_refuse_4_bits(engine):
    model = _model(False)
    with pytest.raises(ValueError):
        engine(model, model, config=InferenceConfig(kv_cache_bits=4))


@pytest.mark.parametrize("norm,bits", [(True, 16), (True, 4), (False, 4)])
@pytest.mark.parametrize("budget", [1, 7, 64])
def test_steps_keep_to_their_budget(norm, bits, budget, monkeypatch):
    """No step runs more tokens than the budget (but one of every sequence that decodes); portions over what is cached, beside single tokens, give
    what the plain forward does."""
    model = _model(norm)
    engine = _engine(model, bits, block_size=16, max_step_tokens=budget)
    forward, steps = engine._forward_packed, []
    monkeypatch.setattr(engine, "_forward_packed", lambda items: steps.append([(len(t), n) for _, t, n in items]) or forward(items))
    out = engine.generate(PROMPTS, GenerationConfig(max_new_tokens=6))
    for p, o in zip(PROMPTS, out):
        logits = _plain_logits(model, o[:-1], bits == 4)
        assert o[len(p):] == logits[len(p) - 1:].argmax(-1).tolist() and len(o) == len(p) + 6
    assert all(sum(n for n, _ in step) <= max(budget, len(step)) for step in steps)
    assert budget == 1 or any(n > 1 and at > 0 for step in steps for n, at in step)
    assert budget == 1 or any({n > 1 for n, _ in step} == {True, False} for step in steps)
    assert engine.kv.free_blocks == engine.kv.num_blocks


@pytest.mark.parametrize("norm", [True, False])
def test_empty_prompts_are_refused(norm):
    engine = _engine(_model(norm), 16)
    with pytest.raises(ValueError):
        engine.generate([[]])
    assert not engine.rm.has_work and engine.generate([[3]], GenerationConfig(max_new_tokens=2))[0][0] == 3


def test_prompts_come_all_or_none():
    """An empty prompt leaves no other one of its call behind; any iterable of tokens is a prompt."""
    engine = _engine(_model(True), 16)
    with pytest.raises(ValueError):
        engine.generate([[3, 4], []])
    assert not engine.rm.has_work
    engine.add_request(iter([5, 6]), 1)
    while engine.rm.has_work:
        engine.step()
    assert engine.kv.free_blocks == engine.kv.num_blocks
