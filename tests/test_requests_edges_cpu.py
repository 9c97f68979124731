"""Batches of many requests at their edges, on the host: what plans keep alive, what the wrappers hand to the library and what they refuse."""
import subprocess
import sys

import pytest
import torch

from hcache_deepspeed_b200.inference.sampling import LogitControls, _drawable, sample_next
from hcache_deepspeed_b200.linear import AdapterBank, MultiAdapterLinear
from hcache_deepspeed_b200.ops import kernels, native, plans
from hcache_deepspeed_b200.ops.backend import CpuOps


# ---- the wrappers against a library that only notes its calls ------------------------------------------------------------
class OnGpu(torch.Tensor):
    """A tensor in host memory that says it is on GPU 0."""
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


def gpu(t):
    return torch.Tensor._make_subclass(OnGpu, t)


class Noted:
    """Every entry point notes its arguments and is content."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if name.startswith("hds_"):
            return lambda *args: self.calls.append((name, args)) or 0
        raise AttributeError(name)


class Memory:
    """Device memory of a plan that notes which streams it was recorded for."""

    def __init__(self):
        self.recorded = []

    def record_stream(self, stream):
        self.recorded.append(stream)


@pytest.fixture
def lib(monkeypatch):
    import contextlib
    noted = Noted()
    monkeypatch.setattr(native, "cuda_lib", lambda: noted)
    monkeypatch.setattr(kernels, "_on", lambda index: contextlib.nullcontext())
    noted.stream = 0
    monkeypatch.setattr(kernels, "_raw_stream", lambda index: noted.stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: noted.stream)
    return noted


def placed(plan):
    """The plan as if its arrays were on GPU 0, made on stream 0."""
    plan.index, plan._dev = 0, Memory()
    for name in ("tiles_ptr", "items_ptr", "workers_ptr", "units_ptr", "rows_ptr"):
        setattr(plan, name, 0)
    return plan


def adapters_call(T=3, n=2, K=16, N=8, R=8):
    bf = lambda *s: gpu(torch.zeros(*s, dtype=torch.bfloat16))  # noqa: E731
    return dict(base=bf(T, N), x=bf(T, K), down=bf(n, R, K), up=bf(n, N, R), scales=gpu(torch.zeros(n)), plan=placed(kernels.AdapterPlan([i % n for i in range(T)], n)))


def shared_call(n=2):
    bf = lambda *s: gpu(torch.zeros(*s, dtype=torch.bfloat16))  # noqa: E731
    return dict(q=bf(n, 128), out=bf(n, 128), kv_cache_layer=bf(9, 2, 2, 16, 64), block_tables=gpu(torch.zeros(n, 3, dtype=torch.int32)), scale=0.125,
                plan=placed(plans.SharedPrefixPlan([1] * n, [40] * n, [(0, n, 32)], 2, 2, 64, 16)))


@pytest.mark.parametrize("call,args", [(kernels.adapter_add, adapters_call), (kernels.paged_attention_shared, shared_call)])
def test_a_plan_outlives_its_calls_on_other_streams(lib, call, args):
    """Its memory belongs to the stream that it was made on: for any other one that reads it, it has to be recorded, or a plan that is dropped gives its
    memory away under a running kernel."""
    kw = args()
    for lib.stream in (0, 7, 7, 0, 9, 7):
        call(**kw)
    assert len([c for c in lib.calls if c[0] in ("hds_adapter_add", "hds_paged_attention_shared")]) == 6
    assert kw["plan"]._dev.recorded == [7, 9]


def controls_call(n=3, V=40):
    return dict(logits=gpu(torch.zeros(n, V)))


WRAPPERS = [(kernels.adapter_add, adapters_call, (3, 8), torch.bfloat16), (kernels.paged_attention_shared, shared_call, (2, 128), torch.bfloat16),
            (kernels.logit_controls, controls_call, (3, 40), torch.float32)]


@pytest.mark.parametrize("call,args,shape,dtype", WRAPPERS)
def test_outputs_whose_rows_share_memory_are_refused(lib, call, args, shape, dtype):
    """Two rows of them would be written to the same place, in any order. (A tensor map of the queries has no room for such rows either.)"""
    memory = torch.zeros(4 * shape[1], dtype=dtype)
    for name in ("out", "q") if call is kernels.paged_attention_shared else ("out", ):
        for stride in (0, 1, shape[1] - 1):
            with pytest.raises(ValueError, match="share memory"):
                call(**{**args(), name: gpu(memory.as_strided(shape, (stride, 1)))})
        assert not lib.calls
        call(**{**args(), name: gpu(memory.as_strided(shape, (shape[1], 1)))})
        assert len(lib.calls) >= 1
        lib.calls.clear()


@pytest.mark.parametrize("call,args,shape,dtype", WRAPPERS)
def test_inputs_may_be_one_row_for_all(lib, call, args, shape, dtype):
    kw = args()
    for name in {"adapter_add": ("base", "x"), "paged_attention_shared": ("block_tables", ), "logit_controls": ("logits", )}[call.__name__]:
        kw[name] = gpu(kw[name][:1].as_subclass(torch.Tensor).expand(kw[name].shape))
    call(**kw)
    assert len(lib.calls) >= 1


def test_sizes_that_the_library_takes_in_32_bits_are_refused_beyond(lib):
    """(Address space alone: nobody touches these tensors.)"""
    space = lambda shape, strides, dtype: gpu(torch.empty_strided(shape, strides, dtype=dtype))  # noqa: E731
    i32, f32, bf = torch.int32, torch.float32, torch.bfloat16
    with pytest.raises(ValueError, match="2.31 apart"):
        kernels.paged_attention_shared(**{**shared_call(), "block_tables": space((2, 3), (1 << 31, 1), i32)})
    lengths = gpu(torch.zeros(1, dtype=i32))
    wide = dict(shape=(1, 1 << 30), strides=(1 << 30, 1))
    for kw in (dict(history=space(**wide, dtype=i32), history_len=lengths), dict(bias_ids=space(**wide, dtype=i32), bias=space(**wide, dtype=f32)),
               dict(mask=space((1 << 30, 2), (0, 1), i32), mask_rows=lengths)):
        with pytest.raises(ValueError, match="fewer than 2.30"):
            kernels.logit_controls(**controls_call(1), **kw)
    for K, N in ((1 << 24, 8), (8, 1 << 24)):
        kw = {**adapters_call(1, 1), "base": space((1, N), (N, 1), bf), "x": space((1, K), (K, 1), bf), "down": space((1, 8, K), (8 * K, K, 1), bf),
              "up": space((1, N, 8), (8 * N, 8, 1), bf)}
        with pytest.raises(ValueError, match="below 2.24"):
            kernels.adapter_add(**kw)
    assert not lib.calls


@pytest.mark.parametrize("scale", [2.0**127, 3e38, 1e300, -1e-300])
def test_scales_that_are_no_number_in_the_kernel_are_refused(lib, scale):
    """Exponents are in powers of 2: 3e38 log2(e) is infinite in 32 bits, and infinity times a score of 0 is NaN."""
    with pytest.raises(ValueError, match="scale"):
        kernels.paged_attention_shared(**{**shared_call(), "scale": scale})
    kw = shared_call()
    with pytest.raises(ValueError, match="scale"):
        CpuOps().attention_shared(*(kw[n].as_subclass(torch.Tensor) for n in ("q", "out", "kv_cache_layer", "block_tables")), kw["plan"], scale)
    assert not lib.calls
    kernels.paged_attention_shared(**{**shared_call(), "scale": 1.5e38})
    assert lib.calls[-1][0] == "hds_paged_attention_shared"


def test_the_package_imports_on_a_torch_without_cuda():
    """A build of torch for the CPU alone has none of the ``_cuda_*`` names."""
    gone = "import torch\nfor name in [n for n in dir(torch._C) if n.startswith('_cuda_')]: delattr(torch._C, name)\n"
    mods = ("hcache_deepspeed_b200", "hcache_deepspeed_b200.ops.kernels", "hcache_deepspeed_b200.models.transformer", "hcache_deepspeed_b200.models.hybrid",
            "hcache_deepspeed_b200.linear", "hcache_deepspeed_b200.inference.sampling")
    code = gone + "".join(f"import {m}\n" for m in mods) + "from hcache_deepspeed_b200.ops.plans import AdapterPlan\nAdapterPlan([0, -1], 1)\n"
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


# ---- plans ---------------------------------------------------------------------------------------------------------------
def test_a_plan_leaves_room_behind_the_last_key():
    """The kernels compare places up to a tile of 128 behind the last key with it, in 32 bits."""
    with pytest.raises(ValueError, match="fewer than 2"):
        plans.SharedPrefixPlan([1], [(1 << 31) - 128], [], 1, 1, 64, 16)
    prefix = ((1 << 31) - 129) // 128 * 128
    plan = plans.SharedPrefixPlan([1], [prefix + 2], [(0, 1, prefix)], 1, 1, 64, 128)
    _, _, _, keys, prefix, _, _, _ = plan.items[0].tolist()
    assert keys + 128 < 1 << 31 and -(-prefix // 128) * 128 < 1 << 31


@pytest.mark.parametrize("sms", [20, 74, 148])
def test_a_plan_deals_out_the_sms_that_its_device_has(monkeypatch, sms):
    monkeypatch.setattr(torch.cuda, "get_device_properties", lambda device: type("P", (), {"multi_processor_count": sms}))
    monkeypatch.setattr(plans._Plan, "_place", lambda self, flat, device: 0)
    plan = plans.SharedPrefixPlan([1] * 20, [4096 + 300] * 20, [(0, 20, 4096)], 32, 8, 128, 64, device="cuda")
    assert (plan.p_splits, -(-plan.n_workers // plans.OWN_WORKERS)) == plans.pick_shares(8, 4096, False, 20 * 8 * (19 + plans.OWN_BEGIN), sms)
    assert plan.n_workers < sms * plans.OWN_WORKERS
    alone = plans.SharedPrefixPlan([1] * 20, [4096 + 300] * 20, [], 32, 8, 128, 64, device="cuda")
    assert alone.n_workers == sms * plans.OWN_WORKERS


@pytest.mark.parametrize("args", [adapters_call, shared_call])
def test_copies_of_a_plan_are_the_plan(args):
    """Its lists do not change, and a copy would have the addresses of memory that it does not hold."""
    import copy
    import pickle
    plan = args()["plan"]
    assert copy.copy(plan) is plan and copy.deepcopy({"plan": plan})["plan"] is plan
    with pytest.raises(TypeError, match="process"):
        pickle.dumps(plan)
    there = pickle.loads(pickle.dumps(plans.SharedPrefixPlan([1, 2], [40, 41], [(0, 2, 32)], 2, 2, 64, 16)))      # in host memory alone
    assert there.index == -1 and there.rows == 3 and there.items.shape == (2, 8)


# ---- banks of adapters ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("convert", [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(), lambda m: m.to("cpu", torch.float16),
                                     lambda m: m.half().bfloat16()])
def test_a_converted_bank_keeps_its_scales(convert):
    """They are fp32 whatever the weights' type: nothing else is served, and 1 / 3 has other bits in 16."""
    torch.manual_seed(0)
    bank = AdapterBank(2, 8, 16, 24, dtype=torch.float32)
    bank.load(1, torch.randn(8, 16), torch.randn(24, 8), 1 / 3)
    layer = torch.nn.Sequential(MultiAdapterLinear(torch.randn(24, 16), bank))
    kept = bank.scales.clone()
    assert convert(layer) is layer and layer[0].bank is bank
    assert bank.scales.dtype == torch.float32 and torch.equal(bank.scales, kept)
    assert bank.down.dtype == bank.up.dtype == layer[0].weight.dtype != torch.float32
    assert dict(bank.named_buffers())["scales"] is bank.scales and torch.equal(bank.state_dict()["scales"], kept)
    bank.load(0, torch.randn(4, 16), torch.randn(24, 4), 0.7)
    assert bank.scales[0] == torch.tensor(0.7)


def test_a_bank_loads_from_its_own_rows():
    torch.manual_seed(1)
    bank = AdapterBank(2, 16, 24, 40, dtype=torch.float32)
    down, up = torch.randn(16, 24), torch.randn(40, 16)
    bank.load(0, down, up, 1.0)
    bank.load(0, bank.down[0], bank.up[0], 0.5)                          # another scale
    assert torch.equal(bank.down[0], down) and torch.equal(bank.up[0], up) and bank.scales[0] == 0.5
    bank.load(1, bank.down[0], bank.up[0], 2.0)                          # a copy
    bank.load(0, bank.down[0, 3:10], bank.up[0, :, 3:10], 1.0)           # fewer ranks
    assert torch.equal(bank.down[0, :7], down[3:10]) and torch.equal(bank.up[0, :, :7], up[:, 3:10])
    assert not bank.down[0, 7:].any() and not bank.up[0, :, 7:].any()
    assert torch.equal(bank.down[1], down) and torch.equal(bank.up[1], up)


# ---- generate under controls ---------------------------------------------------------------------------------------------
def small_engine():
    transformers = pytest.importorskip("transformers")
    import hcache_deepspeed_b200 as ds
    torch.manual_seed(0)
    cfg = transformers.LlamaConfig(vocab_size=128, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                                   max_position_embeddings=256)
    return ds.init_inference(transformers.LlamaForCausalLM(cfg).eval(), dtype=torch.float32, replace_with_kernel_inject=True)


REFUSED = [dict(logit_bias={128: 1.0}), dict(logit_bias=[{}]), dict(repetition_penalty=0.0), dict(presence_penalty=[1.0, 2.0, 3.0]),
           dict(allowed=torch.ones(2, 127, dtype=torch.bool)), dict(frequency_penalty=float("nan"))]


def test_a_refused_request_leaves_nothing_behind():
    eng = small_engine()
    state = eng.ragged_engine.state_manager
    ids = torch.randint(3, 128, (2, 9))
    free, tracked = int(state.free_blocks[0]), state.n_tracked_sequences
    for kw in REFUSED:
        with pytest.raises(ValueError):
            eng.generate(input_ids=ids, max_new_tokens=4, **kw)
        assert (int(state.free_blocks[0]), state.n_tracked_sequences) == (free, tracked)
    want = eng.generate(input_ids=ids, max_new_tokens=4, repetition_penalty=1.5)
    for kw in REFUSED:          # a session is as it was: the same prompt, asked again without the mistake, has the same answer
        with pytest.raises(ValueError):
            eng.generate(input_ids=ids, max_new_tokens=4, session_ids=[5, 6], **kw)
    assert torch.equal(eng.generate(input_ids=ids, max_new_tokens=4, session_ids=[5, 6], repetition_penalty=1.5), want)
    assert state.get_sequence(5).seen_tokens == 9 + 3


def test_a_request_that_fails_on_its_way_leaves_nothing_behind(monkeypatch):
    eng = small_engine()
    state = eng.ragged_engine.state_manager
    free, tracked = int(state.free_blocks[0]), state.n_tracked_sequences
    from hcache_deepspeed_b200.inference import sampling
    calls, plain = [], sampling.sample_next

    def failing(*args):
        calls.append(1)
        if len(calls) == 3:
            raise KeyboardInterrupt
        return plain(*args)
    monkeypatch.setattr(sampling, "sample_next", failing)
    with pytest.raises(KeyboardInterrupt):
        eng.generate(input_ids=torch.randint(3, 128, (2, 9)), max_new_tokens=4, logit_bias={3: 1.0})
    assert (int(state.free_blocks[0]), state.n_tracked_sequences) == (free, tracked)


PENALTIES = dict(repetition_penalty=1.9, presence_penalty=0.3, frequency_penalty=[0.2, 0.0])


def test_a_sessions_earlier_turns_count():
    """Two turns give what one call with all of their tokens gives."""
    eng = small_engine()
    ids = torch.randint(3, 128, (2, 9))
    first = eng.generate(input_ids=ids, max_new_tokens=5, session_ids=[5, 6])
    more = torch.cat([first[:, -1:], torch.randint(3, 128, (2, 4))], 1)       # (the last token of an answer has not been fed yet)
    want = eng.generate(input_ids=torch.cat([first[:, :-1], more], 1), max_new_tokens=12, **PENALTIES)
    plain = eng.generate(input_ids=torch.cat([first[:, :-1], more], 1), max_new_tokens=12)
    got = eng.generate(input_ids=more, max_new_tokens=12, session_ids=[5, 6], **PENALTIES)
    assert torch.equal(got, want[:, first.shape[1] - 1:]) and not torch.equal(want, plain)
    third = torch.cat([got[:, -1:], torch.randint(3, 128, (2, 2))], 1)        # a third turn, with the answer given under penalties behind it
    want = eng.generate(input_ids=torch.cat([first[:, :-1], got[:, :-1], third], 1), max_new_tokens=6, **PENALTIES)
    assert torch.equal(eng.generate(input_ids=third, max_new_tokens=6, session_ids=[5, 6], **PENALTIES)[:, 3:], want[:, -6:])


def test_a_session_that_was_dropped_begins_anew():
    eng = small_engine()
    ids, other = torch.randint(3, 128, (2, 9)), torch.randint(3, 128, (2, 7))
    want = eng.generate(input_ids=other, max_new_tokens=8, **PENALTIES)
    for drop in (eng.flush, eng.ragged_engine.flush):
        eng.generate(input_ids=ids, max_new_tokens=5, session_ids=[5, 6])
        for sid in (5, 6):
            drop(sid)
        assert torch.equal(eng.generate(input_ids=other, max_new_tokens=8, session_ids=[5, 6], **PENALTIES), want)
        for sid in (5, 6):
            eng.flush(sid)
    eng.ragged_engine.put([5, 6], list(ids))       # tokens that this engine has not seen: the call's own count
    eng.generate(input_ids=other, max_new_tokens=2, session_ids=[5, 6], **PENALTIES)
    assert eng._context_of(5) == []
    for sid in (5, 6):
        eng.flush(sid)
    assert not eng._context


def test_a_restored_sessions_earlier_turns_count():
    import hcache_deepspeed_b200 as ds
    transformers = pytest.importorskip("transformers")
    torch.manual_seed(0)
    cfg = transformers.LlamaConfig(vocab_size=128, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                                   max_position_embeddings=256)
    eng = ds.init_inference(transformers.LlamaForCausalLM(cfg).eval(), dtype=torch.float32, replace_with_kernel_inject=True, hcache={"enabled": True})
    more = torch.randint(3, 128, (1, 4))
    ids = eng.generate(input_ids=more, max_new_tokens=40)[:, 4:]       # what this model likes to say
    kw = dict(repetition_penalty=3.0)
    eng.forward(ids, session_ids=[5])
    tokens, latents = eng.session_tokens(5), eng.hidden_states(5)
    eng.flush(5)
    eng.restore_hidden_states(5, tokens, latents)
    got = eng.generate(input_ids=more, max_new_tokens=20, session_ids=[5], **kw)
    want = eng.generate(input_ids=torch.cat([ids, more], 1), max_new_tokens=20, **kw)
    assert torch.equal(got, want[:, ids.shape[1]:])


# ---- controls on logits --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kw", [dict(repetition_penalty=1e39), dict(repetition_penalty=[1.0, 1e-46]), dict(presence_penalty=1e39), dict(frequency_penalty=[-1e39, 0.0]),
                                dict(logit_bias={3: 1e39}), dict(logit_bias=[{}, {8: 4e38}])])
def test_controls_refuse_what_is_no_number_in_32_bits(kw):
    """The kernel has them in 32 bits, where 1e39 is infinite and 1e-46 is 0: logits of 0 times or by these are NaN."""
    with pytest.raises(ValueError, match="32 bits"):
        LogitControls([[1], [2]], 9, 3, "cpu", **kw)


def test_controls_at_the_ends_of_32_bits():
    controls = LogitControls([[1, 2]], 4, 3, "cpu", repetition_penalty=3e38, presence_penalty=-1e-30, logit_bias={3: -1e39})
    assert controls.apply(torch.tensor([[1.0, 0.0, -1.0, 1.0]])).tolist() == [[1.0, 0.0, torch.tensor(-3e38).item(), float("-inf")]]
    assert sample_next(torch.tensor([[1.0, 0.0, -1.0, 1.0]]), controls=controls).tolist() == [0]


@pytest.mark.parametrize("places", [[3], [0, -1], [0, 1, 2, 3]])
def test_requests_that_are_not_there_do_not_go_on(places):
    controls = LogitControls([[1], [2], [3]], 9, 3, "cpu", 1.5)
    with pytest.raises(ValueError, match="of 3 requests"):
        controls.keep(places)
    assert controls.n == 3
    controls.keep([2, 0])
    assert controls._c["history"][:, 0].tolist() == [3, 1]
    with pytest.raises(ValueError, match="of 2 requests"):
        controls.keep([2])


def check_drawing_far_out(device):
    """Rows: a bias at the end of 32 bits; penalties that take everything there; two of them, of which one is larger; one token left that is far below;
    infinities beside the largest number. Divided by a temperature below 1 these are infinite, and a softmax of them NaN, which a GPU's context
    does not outlive."""
    allowed = torch.ones(5, 6, dtype=torch.bool)
    allowed[3] = torch.tensor([False, False, True, False, False, False])
    bias = [{4: 3e38}, {v: -3.2e38 + 1e37 * v for v in range(6)}, {v: -3.4e38 + (v == 5) * 1e38 for v in range(6)}, {2: -3.4e38}, {1: 3.4e38}]
    controls = LogitControls([[1]] * 5, 6, 12, device, logit_bias=bias, allowed=allowed)
    logits = torch.zeros(5, 6, device=device)
    logits[4, 3] = float("inf")
    for kw in (dict(temperature=0.1), dict(temperature=1e-9), dict(temperature=0.5, top_k=2), dict(temperature=0.3, top_p=0.5), dict()):
        assert sample_next(logits, do_sample=True, controls=controls, **kw).tolist() == [4, 5, 5, 2, 3], kw


def test_drawing_far_out():
    check_drawing_far_out("cpu")


def test_drawing_at_any_temperature():
    logits, inf = torch.tensor([[1.0, -float("inf"), 2.0]] * 64), float("inf")
    drawn = sample_next(logits, do_sample=True, temperature=inf).tolist()
    assert set(drawn) == {0, 2}
    controls = LogitControls([[1]] * 64, 3, 4, "cpu", allowed=torch.tensor([[True, True, False]] * 64))
    assert sample_next(logits, do_sample=True, temperature=inf, controls=controls).tolist() == [0] * 64
    assert sample_next(logits, do_sample=True, top_p=0.0).tolist() == [2] * 64
    for kw in (dict(temperature=float("nan")), dict(top_p=-0.1)):
        with pytest.raises(ValueError, match="temperature"):
            sample_next(logits, do_sample=True, **kw)
        sample_next(logits, **kw)       # nothing is drawn


def test_ordinary_logits_are_drawn_as_they_are():
    logits = torch.randn(7, 50) * 20
    logits[2, 10:] = float("-inf")
    assert torch.equal(_drawable(logits), logits)


def grammar_loop(engine, uids, prompts, controls, rule, steps, ends):
    """A grammar that changes with every token: ``rule(token)`` is the set that may follow it. Sessions leave the batch at the token ``ends``."""
    from hcache_deepspeed_b200.inference.sampling import sample_next
    answers, alive = [[] for _ in uids], list(range(len(uids)))
    logits, _ = engine.put(uids, prompts, capture_latents=False)
    controls.set_allowed(torch.stack([rule(int(p[-1])) for p in prompts]))
    for _ in range(steps):
        tokens = sample_next(logits, controls=controls).tolist()
        for i, tok in zip(alive, tokens):
            answers[i].append(tok)
        places = [j for j, tok in enumerate(tokens) if tok != ends]
        if not places:
            break
        controls.keep(places)
        alive, tokens = [alive[j] for j in places], [tokens[j] for j in places]
        controls.set_allowed(torch.stack([rule(t) for t in tokens]))
        logits, _ = engine.put([uids[i] for i in alive], [torch.tensor([t], dtype=torch.int32) for t in tokens], capture_latents=False)
    return answers


def tiny_engine(dtype=torch.float32, device="cpu"):
    from hcache_deepspeed_b200.inference.v2 import RaggedInferenceEngineConfig, build_engine_from_arch
    cfg = RaggedInferenceEngineConfig(state_manager=dict(max_tracked_sequences=16, max_ragged_batch_size=256, max_ragged_sequence_count=8, max_context=512,
                                                         memory_config=dict(mode="allocate", size=32 << 20)), hcache={"enabled": True})
    return build_engine_from_arch("tiny-llama-test", cfg, seed=1, dtype=dtype, device=torch.device(device))


def check_grammar(engine, device):
    """Tokens go up by 1 to 5 each, and 7 of a residue ends: every answer follows the rule, and has the penalties of its own history."""
    V = engine.model().spec.vocab

    def rule(token):
        allowed = torch.zeros(V, dtype=torch.bool)
        allowed[[(token + k) % V for k in range(1, 6)]] = True
        allowed[V - 1] = token % 7 == 0          # the end
        return allowed
    prompts = [torch.tensor(p, dtype=torch.int32) for p in ([3, 9, 1], [4], [10, 20, 30, 7])]
    controls = LogitControls(prompts, V, 12, device, presence_penalty=0.5, logit_bias={V - 1: 50.0})
    answers = grammar_loop(engine, [1, 2, 3], prompts, controls, rule, 12, V - 1)
    for p, answer in zip(prompts, answers):
        before = int(p[-1])
        for tok in answer:
            assert rule(before)[tok]
            before = tok
        assert answer[-1] == V - 1 or len(answer) == 12
        assert all((t == V - 1) == (b % 7 == 0) for b, t in zip([int(p[-1])] + answer, answer))       # (the bias takes the end where it is allowed)
    assert answers[2] == [V - 1]


def test_a_grammar_that_changes_with_every_token():
    check_grammar(tiny_engine(), "cpu")


def check_sessions_under_controls(engine, device):
    """``HCacheSessionManager.decode`` of three sessions, one of which ends early, against drawing by hand."""
    from hcache_deepspeed_b200.hcache import HCacheSessionManager
    manager = HCacheSessionManager(engine, allow_recompute=False)
    V = engine.model().spec.vocab
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, V, (n, ), generator=g).to(torch.int32) for n in (5, 9, 3)]
    make = lambda: LogitControls(prompts, V, 8, device, repetition_penalty=[1.5, 3.0, 1.2], frequency_penalty=0.4, logit_bias=[{3: -9.0}, {}, {5: 2.0}])  # noqa: E731
    uids = [11, 12, 13]
    logits = torch.cat([manager.prefill(u, p).clone() for u, p in zip(uids, prompts)])
    seen = []

    def stop(uid, token):
        seen.append((uid, token))
        return uid == 12 and sum(u == 12 for u, _ in seen) == 3
    answers = manager.decode(uids, 8, logits, stop=stop, controls=make())
    assert [len(a) for a in answers] == [8, 3, 8]
    for u in uids:
        engine.flush(u)
    controls, alive = make(), [0, 1, 2]
    logits = torch.cat([engine.put([u], [p], capture_latents=False)[0].clone() for u, p in zip(uids, prompts)])
    for step in range(8):
        ruled = controls.apply(logits)
        for j, i in enumerate(alive):
            assert answers[i][step] == int(ruled[j].float().argmax())
        tokens = torch.tensor([answers[i][step] for i in alive])
        controls.append(tokens)
        if step == 2:
            alive = [0, 2]
            controls.keep([0, 2])
        if step < 7:
            logits, _ = engine.put([uids[i] for i in alive], [torch.tensor([answers[i][step]], dtype=torch.int32) for i in alive], capture_latents=False)


def test_sessions_decode_under_controls():
    check_sessions_under_controls(tiny_engine(), "cpu")
