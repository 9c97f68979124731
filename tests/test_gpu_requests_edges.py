"""Batches of many requests at their edges, on the GPU. Oracles and tolerances are those of test_gpu_requests.py."""
import pytest
import torch

from tests.test_gpu_requests import (HALF, K, adapters_exact, adapters_inputs, attention_exact, check, controls_check, controls_exact, controls_inputs, pages,
                                     rand)

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]


@pytest.mark.parametrize("which", ["adapters", "shared"])
def test_a_plan_that_is_dropped_keeps_its_memory_until_its_calls_end(which):
    """Made on one stream, used on another that is busy, and dropped: what the first stream allocates next lies elsewhere."""
    torch.manual_seed(0)
    busy = torch.cuda.Stream()
    if which == "adapters":
        ids = [0, 1, -1, 1]
        inputs = adapters_inputs(4, 2, 64, 64, 8, torch.bfloat16)
        plan = K().AdapterPlan(ids, 2, device="cuda")
        call = lambda plan: K().adapter_add(*inputs, plan)  # noqa: E731
        want, bound = adapters_exact(*inputs, ids)
    else:
        new, keys, groups = [1, 2], [70, 75], [(0, 2, 64)]
        cache, tables = pages(keys, groups, 2, 64, 32, torch.bfloat16)
        q = rand(3, 256)
        plan = K().SharedPrefixPlan(new, keys, groups, 4, 2, 64, 32, device="cuda")
        call = lambda plan: K().paged_attention_shared(q, torch.empty_like(q), cache, tables, plan, 0.125)  # noqa: E731
        want, bound = attention_exact(q, cache, tables, new, keys, [64, 64], 4, 0.125)
    call(plan)
    torch.cuda.synchronize()
    at, n = plan._dev.data_ptr(), plan._dev.numel()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(200_000_000)
        out = call(plan)
    del plan
    later = [torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(4)]
    assert not busy.query(), "the stream was to be busy still"
    assert at not in [t.data_ptr() for t in later]
    torch.cuda.synchronize()
    check(out, want, bound)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("prefix,bs", [(16, 16), (144, 16), (192, 64), (1088, 64)])
@pytest.mark.parametrize("scale", [0.0, 1e-46, 1e-40])      # (1e-46 is 0 in 32 bits)
def test_weights_are_equal_at_scales_of_nothing(dtype, prefix, bs, scale):
    """Prefixes that end inside a tile: what is behind them has no weight, whatever the scale."""
    torch.manual_seed(1)
    new, keys, groups = [1, 2, 1], [prefix + 1, prefix + 20, prefix + 300], [(0, 3, prefix)]
    for d, H, kvh in ((64, 4, 1), (128, 20, 2)):
        cache, tables = pages(keys, groups, kvh, d, bs, dtype)
        plan = K().SharedPrefixPlan(new, keys, groups, H, kvh, d, bs, device="cuda")
        q = rand(4, H * d, dtype=dtype, std=2.0)
        out = K().paged_attention_shared(q, torch.empty_like(q), cache, tables, plan, scale)
        check(out, *attention_exact(q, cache, tables, new, keys, [prefix] * 3, H, scale))


def test_a_converted_bank_serves():
    from hcache_deepspeed_b200.linear import AdapterBank, MultiAdapterLinear
    torch.manual_seed(2)
    bank = AdapterBank(2, 8, 64, 48, dtype=torch.float32)
    for i in range(2):
        bank.load(i, torch.randn(8, 64) / 8, torch.randn(48, 8), 1 / 3 + i)
    layer = MultiAdapterLinear(torch.randn(48, 64) / 8, bank).to("cuda").to(torch.bfloat16)
    ids, x = [1, -1, 0], rand(3, 64)
    y = layer(x, bank.plan(ids))
    check(y, *adapters_exact(K().gemm(x, layer.weight), x, bank.down, bank.up, bank.scales, ids))


@pytest.mark.parametrize("dtype", HALF + [torch.float32])
@pytest.mark.parametrize("n,V,cap,k", [(2, 1500, 40, 1400), (1, 3000, 5, 5000), (200, 300, 1500, 700)])
def test_more_biases_than_a_chunk_keeps(dtype, n, V, cap, k):
    """More than 512 of them in a chunk, of small and of large ones; of a token given twice the last one counts."""
    logits, c = controls_inputs(n, V, dtype, cap, k, 1)
    want, bound = controls_exact(logits, **c)
    out = K().logit_controls(logits, **c)
    controls_check(out, want, bound)
    assert torch.equal(K().logit_controls(logits, logits, **c), out)


@pytest.mark.parametrize("dtype", HALF)
def test_a_grammar_that_changes_with_every_token(dtype):
    from tests.test_requests_edges_cpu import check_grammar, tiny_engine
    check_grammar(tiny_engine(dtype, "cuda"), "cuda")


def test_sessions_decode_under_controls():
    from tests.test_requests_edges_cpu import check_sessions_under_controls, tiny_engine
    check_sessions_under_controls(tiny_engine(torch.bfloat16, "cuda"), "cuda")


def test_generate_under_controls():
    """On the GPU: a mask, a bias and penalties rule; a refused request leaves nothing; a session's second turn."""
    transformers = pytest.importorskip("transformers")
    import hcache_deepspeed_b200 as ds
    torch.manual_seed(0)
    cfg = transformers.LlamaConfig(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                                   max_position_embeddings=512)
    eng = ds.init_inference(transformers.LlamaForCausalLM(cfg).eval().to(torch.bfloat16).cuda(), dtype=torch.bfloat16, replace_with_kernel_inject=True,
                            hcache={"max_context": 512, "max_batch_tokens": 256, "kv_memory_bytes": 64 << 20})
    state = eng.ragged_engine.state_manager
    free, tracked = int(state.free_blocks[0]), state.n_tracked_sequences
    ids = torch.randint(3, 512, (2, 9)).cuda()
    allowed = torch.zeros(2, 512, dtype=torch.bool)
    allowed[0, 5] = allowed[1, 77] = True
    assert eng.generate(input_ids=ids, max_new_tokens=3, allowed=allowed.cuda())[:, 9:].tolist() == [[5] * 3, [77] * 3]
    odd = torch.ones(2, 512, dtype=torch.bool)
    odd[:, ::2] = False
    drawn = eng.generate(input_ids=ids, max_new_tokens=20, do_sample=True, allowed=odd, presence_penalty=-2.0)
    assert (drawn[:, 9:] % 2 == 1).all()
    every = eng.generate(input_ids=ids, max_new_tokens=30, presence_penalty=1e6)       # no token twice
    assert all(len(set(row.tolist())) == len(row) for row in every[:, 9:])
    with pytest.raises(ValueError):
        eng.generate(input_ids=ids, max_new_tokens=3, logit_bias={512: 1.0})
    assert (int(state.free_blocks[0]), state.n_tracked_sequences) == (free, tracked)
    told = eng.generate(input_ids=ids, max_new_tokens=30, session_ids=[5, 6])
    never = eng.generate(input_ids=told[:, -1:], max_new_tokens=30, session_ids=[5, 6], repetition_penalty=1e30)      # what was said has a logit of 0, or of -1e30
    for a, b in zip(told, never):
        assert not set(a.tolist()) & set(b[1:].tolist())


def test_drawing_far_out():
    from tests.test_requests_edges_cpu import check_drawing_far_out
    check_drawing_far_out("cuda")
