"""Generation with the 4-bit cache, rotary layouts in a model, and combined
sampling filters: what the serving operators are reached by, on the CPU and on
the GPU."""

import pytest
import torch



@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def device(request):
    if request.param == "cpu" and torch.cuda.is_available():
        pytest.skip("the framework's device is the GPU")
    return request.param


def make_model(device, seed=5, **change):
    from megatron_amd import global_state
    from megatron_amd.config import TrainingConfig, set_config
    from megatron_amd.models import LlamaModel
    from megatron_amd.tokenizer.tokenizers import FakeTokenizer

    settings = dict(
        num_layers=2, hidden_size=256, num_attention_heads=4,
        num_attention_heads_kv=2, kv_channels=64, seq_length=64,
        max_position_embeddings=128, micro_batch_size=2, bf16=True,
        hidden_dropout=0.0, attention_dropout=0.0, use_flash_attn=True,
        use_cpu_initialization=True, use_hip_graph_decode=False,
    )
    cfg = TrainingConfig(**{**settings, **change})
    cfg.finalize()
    cfg.pad_vocab_size(100)
    set_config(cfg)
    global_state.set_tokenizer(FakeTokenizer(100))
    torch.manual_seed(seed)
    model = LlamaModel(cfg, parallel_output=False).to(device).bfloat16()
    return model.eval(), cfg


def steps_of(model, tokens, prompt, total):
    """Logits of the prompt's last token and of each step behind it."""
    from megatron_amd.inference.forward_step import ForwardStep
    from megatron_amd.utils import get_ltor_masks_and_position_ids

    mask, _, ids = get_ltor_masks_and_position_ids(tokens, 0, False, False,
                                                   False)
    forward = ForwardStep(model, tokens.shape[0], total)
    out = []
    with torch.no_grad():
        low = 0
        for high in range(prompt, total):
            logits = forward(tokens[:, low:high], ids[:, low:high],
                             mask[..., low:high, :high])
            out.append(logits[:, -1].float().clone())
            low = high
    return out, forward.inference_params


def test_four_bit_cache_prompt_as_before_and_steps_near(dist_single, device):
    """The prompt attends to its tokens as they were; the steps' logits move by
    what 4 bits lose, which is little of their spread (a value is off by half
    a thirtieth of its group's range at most, in sums over many)."""
    torch.manual_seed(1)
    tokens = torch.randint(1, 99, (2, 40), device=device)
    plain, _ = make_model(device)
    want, _ = steps_of(plain, tokens, 20, 40)
    four, _ = make_model(device, kv_cache_bits=4)
    four.load_state_dict(plain.state_dict())
    got, params = steps_of(four, tokens, 20, 40)
    assert torch.equal(got[0], want[0])
    for x, y in zip(got, want):
        assert (x - y).norm() < 0.1 * y.norm()
    from megatron_amd.ops import QuantKVCache

    assert all(isinstance(c, QuantKVCache)
               for c in params.key_value_memory_dict.values())


def test_four_bit_step_is_attention_over_what_is_held(dist_single, device):
    """One attention layer's step against the sum over what its cache holds,
    in 64 bits."""
    from megatron_amd.inference.forward_step import InferenceParams
    from megatron_amd.ops.functional import rotate_reference

    model, cfg = make_model(device, kv_cache_bits=4, rotary_layout="half",
                            rotary_percent=0.5, rope_scaling_type="ntk",
                            rope_scaling_factor=2.0)
    attn = model.language_model.encoder.layers[0].self_attention
    params = InferenceParams(2, 30)
    torch.manual_seed(2)
    x = torch.randn(13, 2, 256, device=device).bfloat16()
    caught = []
    attn.dense.register_forward_pre_hook(
        lambda m, args: caught.append(args[0].detach()))
    with torch.no_grad():
        attn(x[:12], None, inference_params=params)
        params.sequence_len_offset = 12
        attn(x[12:], None, inference_params=params)
        cache = params.key_value_memory_dict[attn.layer_number]
        key, value = (t.double().cpu() for t in cache.dequantize(0, 13))
        mixed, _ = attn.query_key_value(x[12:])
        q = mixed.view(1, 2, 2, 4 * 64)[..., :128].reshape(1, 2, 4, 64)
        cos, sin = attn._tables(x.device)
        q = rotate_reference(q, cos[12].double().expand(1, 2, -1),
                             sin[12].double().expand(1, 2, -1), False)
    got = caught[-1].view(2, 4, 64).double().cpu()
    for i in range(2):
        for head in range(4):
            p = torch.softmax(key[:, i, head // 2] @ q[0, i, head].double()
                              .cpu() / 8.0, 0)
            want = p @ value[:, i, head // 2]
            # read back in bf16 (2^-8), fp16 operands (2^-10), rounded (2^-8),
            # and scores that the keys' rounding moves
            size = p @ value[:, i, head // 2].abs()
            moved = 2 * 2.0 ** -8 * (key[:, i, head // 2].abs()
                                     @ q[0, i, head].double().cpu().abs()
                                     / 8.0).max()
            off = (got[i, head] - want).abs()
            assert (off <= size * (2 * moved + 2.0 ** -6)).all()


def test_four_bit_generation_and_beams(dist_single, device):
    from megatron_amd.inference.generation import (
        beam_search_and_return_on_first_stage,
        generate_tokens_probs_and_return_on_first_stage,
    )

    model, cfg = make_model(device, kv_cache_bits=4)
    torch.manual_seed(3)
    tokens = torch.zeros(2, 24, dtype=torch.long, device=device)
    tokens[:, :8] = torch.randint(1, 99, (2, 8), device=device)
    lengths = torch.tensor([8, 6], device=device)
    out, _, _ = generate_tokens_probs_and_return_on_first_stage(
        model, tokens.clone(), lengths, top_k=20, top_p=0.9, min_p=0.05,
        use_eod_token_for_early_termination=False)
    assert out.shape == (2, 24) and (out < 100).all() and (out >= 0).all()
    one = torch.zeros(1, 16, dtype=torch.long, device=device)
    one[:, :6] = tokens[:1, :6]
    best, scores = beam_search_and_return_on_first_stage(
        model, one, torch.tensor([6], device=device), beam_size=3,
        stop_token=0, num_return_gen=2, length_penalty=1.0)
    assert best.shape[0] == 2 and torch.isfinite(scores).all()


def test_window_with_sinks_in_generation(dist_single, device):
    """A prompt beyond its window: the first tokens stay visible only with
    sinks, and a window that covers everything changes nothing."""
    torch.manual_seed(4)
    tokens = torch.randint(1, 99, (2, 40), device=device)
    runs, weights = {}, None
    for name, change in (
        ("whole", dict()), ("wide", dict(sliding_window_size=64)),
        ("sinks", dict(sliding_window_size=8, attention_sink_size=2)),
        ("all", dict(sliding_window_size=8, attention_sink_size=40)),
    ):
        model, _ = make_model(device, kv_cache_bits=4, **change)
        if weights is not None:
            model.load_state_dict(weights)
        weights = model.state_dict()
        runs[name], _ = steps_of(model, tokens, 20, 40)
    assert all(torch.equal(x, y) for x, y in zip(runs["whole"], runs["wide"]))
    for x, y, z in zip(runs["sinks"], runs["all"], runs["whole"]):
        assert not torch.equal(x, z)
        assert (y - z).norm() < 0.1 * z.norm()


@pytest.mark.parametrize("train", [False, True])
def test_half_layout_is_interleaved_with_permuted_rows(dist_single, device, train):
    """Moving each head's rows of the q and k projections from pairs (2j,
    2j + 1) to (j, j + h/2) and rotating halves gives the same model. Sums run
    in another order, so values differ by roundings of bf16."""
    torch.manual_seed(6)
    tokens = torch.randint(1, 99, (2, 32), device=device)
    plain, _ = make_model(device)
    half, _ = make_model(device, rotary_layout="half")
    half.load_state_dict(plain.state_dict())
    order = torch.cat([torch.arange(0, 64, 2), torch.arange(1, 64, 2)])
    for layer in half.language_model.encoder.layers:
        weight = layer.self_attention.query_key_value.weight.data
        rows = weight.view(2, 4, 64, 256)  # per key head: q, q, k, v
        rows[:, :3] = rows[:, :3][:, :, order.to(device)].clone()
    ids = torch.arange(32, device=device).expand(2, 32)
    if not train:
        with torch.no_grad():
            a, b = (m(tokens, ids, None).float() for m in (plain, half))
        assert (a - b).norm() < 2.0 ** -6 * a.norm()
        got, _ = steps_of(half, tokens, 20, 32)
        want, _ = steps_of(plain, tokens, 20, 32)
        for x, y in zip(got, want):
            assert (x - y).norm() < 2.0 ** -6 * y.norm()
        return
    grads = []
    for m in (plain, half):
        m(tokens, ids, None, labels=tokens).float().mean().backward()
        grads.append([p.grad for n, p in m.named_parameters()
                      if "query_key_value" in n])
    for a, b in zip(*grads):
        b = b.view(2, 4, 64, 256).clone()
        back = torch.empty_like(b)
        back[:, :3][:, :, order.to(device)] = b[:, :3]
        back[:, 3] = b[:, 3]
        a = a.view(2, 4, 64, 256).float()
        assert (a - back.float()).norm() < 2.0 ** -5 * a.norm()


def test_configuration_refuses():
    from megatron_amd.config import TrainingConfig

    for bad in (dict(kv_cache_bits=8), dict(attention_sink_size=4),
                dict(attention_sink_size=4, kv_cache_bits=4),
                dict(attention_sink_size=-1, kv_cache_bits=4,
                     sliding_window_size=8),
                dict(attention_sink_size=4, kv_cache_bits=4,
                     sliding_window_size=8, use_flash_attn=False),
                dict(rotary_layout="other"), dict(rotary_percent=0.0),
                dict(rope_scaling_type="other"),
                dict(rope_scaling_type="yarn"),
                dict(kv_cache_bits=4, pipeline_model_parallel_size=2,
                     world_size=2)):
        with pytest.raises(AssertionError):
            TrainingConfig(**bad).finalize()


def test_sample_with_min_p_and_uniform(device):
    from megatron_amd.inference.sampling import sample

    logits = torch.tensor([[0.0, 3.0, 2.9, -1.0, 9.0]], device=device)
    u = torch.tensor([0.99], device=device)
    assert sample(logits, uniform=u).item() == 4
    assert sample(logits, uniform=u, vocab_size=4).item() == 2
    assert sample(logits, uniform=u, vocab_size=4, min_p=0.95).item() == 1
    assert sample(logits, top_k=2, top_p=0.3, uniform=u,
                  vocab_size=4).item() == 1
    drawn = {sample(logits, min_p=0.5, vocab_size=4).item()
             for _ in range(30)}
    assert drawn <= {1, 2}
    void = torch.full((1, 5), float("-inf"), device=device)
    assert sample(void, uniform=u).item() == 0


def test_min_p_out_of_range_is_refused():
    """By sample, and by the server before it calls upon the other ranks."""
    import asyncio
    import json

    from megatron_amd.inference.sampling import sample
    from megatron_amd.inference.server import MegatronServer

    for bad in (-0.5, 1.5, float("nan")):
        with pytest.raises(ValueError):
            sample(torch.zeros(1, 4), min_p=bad)

    app = MegatronServer(None)._build_app()
    endpoint = next(r.endpoint for r in app.routes if r.path == "/api")

    class Request:
        def __init__(self, **body):
            self.body = body

        async def json(self):
            return dict(prompts=["a"], **self.body)

    for bad in (dict(min_p=-0.5), dict(min_p=1.5), dict(min_p=float("nan")),
                dict(min_p=0.1, temperature=-1.0),
                dict(min_p=0.1, top_k=-1), dict(min_p=0.1, top_p=2.0)):
        answer = asyncio.run(endpoint(Request(**bad)))
        assert answer.status_code == 400
        assert "min_p" in json.loads(answer.body)["message"]


@pytest.mark.gpu
def test_four_bit_steps_captured_as_eager(dist_single):
    """The captured step against the eager one: the same kernels on the same
    values."""
    torch.manual_seed(7)
    tokens = torch.randint(1, 99, (2, 40), device="cuda")
    model, cfg = make_model("cuda", kv_cache_bits=4,
                            rotary_layout="half", rotary_percent=0.5)
    eager, _ = steps_of(model, tokens, 20, 40)
    cfg.use_hip_graph_decode = True
    graph, _ = steps_of(model, tokens, 20, 40)
    for a, b in zip(eager, graph):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [
    dict(),  # the layout whose step is fused with the rotation
    dict(rotary_layout="half"),
    dict(rotary_layout="half", rotary_percent=0.25),
    dict(rope_scaling_type="ntk", rope_scaling_factor=2.0),
    dict(rope_scaling_type="yarn", rope_scaling_factor=4.0,
         rope_original_max_positions=32),
], ids=["plain", "half", "part", "ntk", "yarn"])
@pytest.mark.parametrize("kv_channels", [64, 128])
def test_captured_steps_keep_the_window(dist_single, rotary, kv_channels):
    """Captured steps past the window against the whole sequence at once, as
    in training, and far from what a model without the window gives. Both sides
    round to bf16 in another order: 2^-8 at each of two layers' few steps."""
    torch.manual_seed(8)
    tokens = torch.randint(1, 99, (2, 48), device="cuda")
    change = dict(sliding_window_size=6, use_hip_graph_decode=True,
                  kv_channels=kv_channels, init_method_std=0.1, **rotary)
    model, _ = make_model("cuda", **change)
    got, params = steps_of(model, tokens, 20, 48)
    assert params.use_graph
    ids = torch.arange(48, device="cuda").expand(2, 48)
    with torch.no_grad():
        want = model(tokens, ids, None).float()
    wide, _ = make_model("cuda", **{**change, "sliding_window_size": None})
    wide.load_state_dict(model.state_dict())
    with torch.no_grad():
        whole = wide(tokens, ids, None).float()
    for i, x in enumerate(got):
        at = 19 + i
        size = want[:, at].norm()
        assert (whole[:, at] - want[:, at]).norm() > 2.0 ** -3 * size
        assert (x - want[:, at]).norm() < 2.0 ** -5 * size, at


@pytest.mark.parametrize("bad", [
    dict(kv_cache_bits=4, bf16=False),               # parameters in fp32
    dict(kv_cache_bits=4, kv_channels=80),
    dict(kv_cache_bits=4, kv_channels=None, hidden_size=96),  # heads of 24
    dict(rotary_percent=0.01),                       # no pair of 64 values
    dict(rotary_percent=0.01, rotary_layout="half"),
    dict(rope_scaling_type="ntk", rope_scaling_factor=0.5),
    dict(rope_scaling_type="yarn", rope_scaling_factor=0.5,
         rope_original_max_positions=32),
    dict(rope_scaling_type="yarn", rope_scaling_factor=2.0,
         rope_original_max_positions=0),
    dict(rotary_layout="half", rope_scaling_factor=0.0),
    dict(rotary_layout="half", rope_theta=1.0),
])
def test_configuration_refuses_what_a_call_would(bad):
    """Before a model is built, not in its first forward."""
    from megatron_amd.config import TrainingConfig

    good = dict(num_layers=2, hidden_size=256, num_attention_heads=4,
                kv_channels=64, seq_length=64, max_position_embeddings=128,
                micro_batch_size=2, bf16=True)
    for more in ({}, dict(kv_cache_bits=4), dict(kv_channels=80),
                 dict(kv_cache_bits=4, bf16=False, fp16=True),
                 dict(rotary_percent=0.04), dict(bf16=False)):
        TrainingConfig(**{**good, **more}).finalize()
    with pytest.raises(AssertionError):
        TrainingConfig(**{**good, **bad}).finalize()


@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_forward_mode(device, interleaved):
    """Tangents are turned as their tensors are (the rotation is linear), with
    and without a gradient beside, and through the backward pass."""
    import torch.autograd.forward_ad as fwd

    from megatron_amd.models.rope import precompute_rotary_tables
    from megatron_amd.ops import rotary_embedding

    torch.manual_seed(9)
    q, k, tq, tk, g, tg = (torch.randn(3, 2, n, 24, device=device)
                           for n in (4, 1, 4, 1, 4, 4))
    cos, sin = precompute_rotary_tables(16, 9, device=device)

    def turned(a, b):
        return rotary_embedding(a, b, cos, sin, interleaved=interleaved)

    want_q, want_k = turned(tq, tk)
    back, = torch.autograd.grad(
        turned(q.requires_grad_(), None)[0], q, tg)
    q = q.detach()
    with fwd.dual_level():
        both = turned(fwd.make_dual(q, tq), fwd.make_dual(k, tk))
        assert torch.equal(fwd.unpack_dual(both[0]).tangent, want_q)
        assert torch.equal(fwd.unpack_dual(both[1]).tangent, want_k)
        one = turned(fwd.make_dual(q, tq), k)
        assert torch.equal(fwd.unpack_dual(one[0]).tangent, want_q)
        none = fwd.unpack_dual(one[1]).tangent
        assert none is None or not none.any()
        alone = turned(fwd.make_dual(q, tq), None)
        assert torch.equal(fwd.unpack_dual(alone[0]).tangent, want_q)
        with torch.no_grad():
            quiet = turned(fwd.make_dual(q, tq), k)
            assert torch.equal(fwd.unpack_dual(quiet[0]).tangent, want_q)
        leaf = q.clone().requires_grad_()
        out, _ = turned(fwd.make_dual(leaf, tq), k)
        assert torch.equal(fwd.unpack_dual(out).tangent, want_q)
        dq, = torch.autograd.grad(out, leaf, fwd.make_dual(g, tg))
        assert torch.equal(fwd.unpack_dual(dq).tangent, back)
    _, out = torch.func.jvp(lambda a, b: turned(a, b), (q, k), (tq, tk))
    assert torch.equal(out[0], want_q) and torch.equal(out[1], want_k)


def test_cache_refuses_forward_mode(device):
    """As it refuses a gradient: no tangent is dropped in silence."""
    import torch.autograd.forward_ad as fwd

    from megatron_amd.ops import QuantKVCache

    cache = QuantKVCache(8, 1, 1, 32, device=device)
    x = torch.randn(1, 1, 1, 32, device=device).bfloat16()
    with fwd.dual_level(), torch.no_grad():
        dual = fwd.make_dual(x, x)
        cache.append(x, x, 0)
        cache.attention(x, 0)
        for call in (lambda: cache.append(dual, x, 0),
                     lambda: cache.append(x, dual, 0),
                     lambda: cache.attention(dual, 0)):
            with pytest.raises(ValueError):
                call()


def test_min_p_beside_beams_is_refused():
    """A beam search draws nothing: min_p beside it would go unheard."""
    import asyncio
    import json

    from megatron_amd.inference import server

    app = server.MegatronServer(None)._build_app()
    endpoint = next(r.endpoint for r in app.routes if r.path == "/api")

    class Request:
        async def json(self):
            return dict(prompts=["a"], min_p=0.1, beam_width=2)

    def never(*args, **kw):
        raise AssertionError("the other ranks were called upon")

    with pytest.MonkeyPatch.context() as patch:
        patch.setattr(server, "send_do_beam_search", never)
        answer = asyncio.run(endpoint(Request()))
    assert answer.status_code == 400
    assert "min_p" in json.loads(answer.body)["message"]


def test_layers_share_rotary_tables(dist_single, device):
    """One pair of tables for all layers alike, and none besides; they serve a
    training step also where a generation under inference_mode came first, and
    go with the models that use them."""
    import gc
    import weakref

    tokens = torch.zeros(2, 8, dtype=torch.long, device=device)
    ids = torch.arange(8, device=device).expand(2, 8)
    model, _ = make_model(device, rotary_layout="half")
    other, _ = make_model(device, rotary_layout="half", rope_theta=5000.0)
    with torch.inference_mode():
        model(tokens, ids, None), other(tokens, ids, None)
    first, second = (layer.self_attention
                     for layer in model.language_model.encoder.layers)
    here = tokens.device
    for a, b in zip(first._tables(here), second._tables(here)):
        assert a.data_ptr() == b.data_ptr() and a.dtype == torch.float32
    strange = other.language_model.encoder.layers[0].self_attention
    assert not torch.equal(first._tables(here)[0], strange._tables(here)[0])
    assert not [n for n, _ in model.named_buffers() if "rope" in n]
    plain, _ = make_model(device)
    assert [n for n, _ in plain.named_buffers() if "rope" in n]
    model(tokens, ids, None, labels=tokens).float().mean().backward()
    gone = weakref.ref(first._tables(here)[0])
    del model, first, second, a, b
    gc.collect()
    assert gone() is None


@pytest.mark.parametrize("rotary", [dict(), dict(rotary_layout="half")],
                         ids=["plain", "half"])
def test_uncaptured_steps_keep_the_window(dist_single, device, rotary):
    """As the captured ones (tensor parallel generation does not capture)."""
    torch.manual_seed(10)
    tokens = torch.randint(1, 99, (2, 32), device=device)
    model, _ = make_model(device, sliding_window_size=6, init_method_std=0.1,
                          **rotary)
    got, _ = steps_of(model, tokens, 20, 32)
    ids = torch.arange(32, device=device).expand(2, 32)
    with torch.no_grad():
        want = model(tokens, ids, None).float()
    for i, x in enumerate(got):
        size = want[:, 19 + i].norm()
        assert (x - want[:, 19 + i]).norm() < 2.0 ** -5 * size, 19 + i
