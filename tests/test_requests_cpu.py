"""Batches of many requests on the host: plans, adapters beside a projection, attention behind shared prefixes, controls on logits."""
import math

import pytest
import torch

from hcache_deepspeed_b200.inference.sampling import LogitControls, pack_mask, sample_next
from hcache_deepspeed_b200.inference.v2.kernels import SharedPrefixAttn
from hcache_deepspeed_b200.linear import AdapterBank, LoRAConfig, LoRAOptimizedLinear, MultiAdapterLinear
from hcache_deepspeed_b200.ops import kernels, plans
from hcache_deepspeed_b200.ops import reference as ref
from hcache_deepspeed_b200.ops.backend import CpuOps


# ---- adapters --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("ids", [[], [0], [-1], [-1, -1, 3], [2, 0, 2, 0, 2], list(range(5)) * 30, [1] * 33, [1] * 97 + [-1] * 130 + [0] * 3, [4] * 200])
def test_every_row_is_in_one_tile_of_its_adapter(ids):
    plan = kernels.AdapterPlan(ids, 5)
    order = sorted(range(len(ids)), key=lambda i: (max(ids[i], -1), i))
    seen = []
    for i, (name, start, n, _) in enumerate(plan.tiles):
        assert 1 <= n <= 64 and (name < 0) == (i >= plan.n_tiles) and (name < 0 or n <= plan.tile_rows)
        seen += range(start, start + n)
        assert all(max(ids[order[p]], -1) == name for p in range(start, start + n))
    assert sorted(seen) == list(range(len(ids)))


def test_plans_of_adapters_refuse_what_is_not_there():
    with pytest.raises(ValueError, match="row 1 has adapter 4"):
        kernels.AdapterPlan([0, 4], 4)
    with pytest.raises(ValueError, match="whole numbers"):
        kernels.AdapterPlan([0.5], 4)
    with pytest.raises(ValueError, match="whole numbers"):
        kernels.AdapterPlan([[0, 1]], 4)


def test_adapters_of_trained_linears_serve_one_batch():
    torch.manual_seed(0)
    made = [LoRAOptimizedLinear(24, 40, lora_config=LoRAConfig(lora_r=r, lora_alpha=8.0), dtype=torch.float32) for r in (3, 8, 12)]
    for m in made:
        torch.nn.init.normal_(m.lora_weight_2.weight)
        m.weight.data.copy_(made[0].weight)
    bank = AdapterBank(4, 12, 24, 40, dtype=torch.float32)
    for i, m in enumerate(made):
        bank.load_linear(i, m)
    layer = MultiAdapterLinear(made[0].weight.data, bank, bias=torch.randn(40))
    ids = [2, -1, 0, 1, 1, 3, 2]        # 3 was never loaded
    x = torch.randn(7, 24)
    y = layer(x, bank.plan(ids))
    for t, i in enumerate(ids):
        want = (made[i](x[t]) if 0 <= i < 3 else x[t] @ made[0].weight.t()) + layer.bias
        torch.testing.assert_close(y[t], want, atol=1e-4, rtol=1e-4)
    assert layer(x[:0], bank.plan([])).shape == (0, 40)
    assert layer(x.view(7, 1, 24), bank.plan(ids)).shape == (7, 1, 40)
    bank.load(2, torch.ones(2, 24), torch.ones(40, 2), 0.5)      # a smaller one leaves nothing of the larger behind
    torch.testing.assert_close(layer(x[:1], bank.plan([2])) - layer(x[:1], bank.plan([-1])), 0.5 * 2 * x[:1].sum().expand(1, 40), atol=1e-4, rtol=1e-4)


def test_banks_refuse_what_does_not_fit():
    for bad in ((0, 8, 16, 16), (1, 0, 16, 16), (1, 257, 16, 16), (1, 8, 12, 16), (1, 8, 16, 20)):
        with pytest.raises(ValueError):
            AdapterBank(*bad)
    bank = AdapterBank(2, 8, 16, 24, dtype=torch.float32)
    for i, down, up in ((2, torch.ones(8, 16), torch.ones(24, 8)), (0, torch.ones(9, 16), torch.ones(24, 9)), (0, torch.ones(8, 16), torch.ones(24, 4)),
                        (0, torch.ones(8, 8), torch.ones(24, 8))):
        with pytest.raises(ValueError):
            bank.load(i, down, up, 1.0)
    with pytest.raises(ValueError):
        MultiAdapterLinear(torch.ones(16, 24), bank)


# ---- attention behind shared prefixes ----------------------------------------------------------------------------------
def test_prefix_plan_lists_rows_and_lengths():
    plan = plans.SharedPrefixPlan([1, 0, 3, 2], [40, 32, 70, 5], [(0, 3, 32)], 8, 2, 64, 16)
    assert plan.rows == 6 and plan.max_blocks == 5
    assert plan.items[:, :5].tolist() == [[0, 0, 1, 40, 32], [1, 1, 0, 32, 32], [2, 1, 3, 70, 32], [3, 4, 2, 5, 0]]
    assert plan.n_tiles == 1      # four rows of 8 / 2 heads share a tile of 128
    wide = plans.SharedPrefixPlan([40] * 3, [200] * 3, [(0, 3, 128)], 8, 2, 64, 16)
    assert wide.n_tiles == 2      # 120 tokens in two tiles of 32 each


@pytest.mark.parametrize("new,keys,groups,match", [
    ([1], [1, 2], [], "same sequences"), ([2], [1], [], "at least its new tokens"), ([-1], [1], [], "at least its new tokens"),
    ([1], [1 << 31], [], "fewer than 2"), ([1, 1], [40, 40], [(0, 3, 16)], "that are there"), ([1, 1], [40, 40], [(-1, 1, 16)], "that are there"),
    ([1, 1], [40, 40], [(0, 0, 16)], "that are there"), ([1, 1], [40, 40], [(0, 2, 16), (1, 1, 16)], "no other group"),
    ([1, 1], [40, 40], [(0, 2, 15)], "whole pages"), ([1, 1], [40, 32], [(0, 2, 32)], "whole pages"), ([1], [40], [(0, 1, -16)], "whole pages")])
def test_prefix_plans_refuse(new, keys, groups, match):
    with pytest.raises(ValueError, match=match):
        plans.SharedPrefixPlan(new, keys, groups, 4, 2, 64, 16)


def test_prefix_plans_refuse_heads_and_blocks():
    for heads in ((4, 3), (0, 1), (4, 0), (129, 1)):
        with pytest.raises(ValueError, match="share"):
            plans.SharedPrefixPlan([1], [4], [], *heads, 64, 16)
    with pytest.raises(ValueError, match="block_size"):
        plans.SharedPrefixPlan([1], [4], [], 4, 2, 64, 24)


@pytest.mark.parametrize("units,prefix", [(0, 0), (1, 16), (1, 128), (1, 65536), (8, 4096), (32, 4096), (148, 8192), (1000, 100000)])
def test_splits_of_a_prefix_have_tiles(units, prefix):
    for two in (False, True):
        for cost in (1, 300, 12288, 1 << 40):
            splits, ctas = plans.pick_shares(units, prefix, two, cost)
            assert 1 <= splits <= max(1, min(64, -(-prefix // 128))) and 1 <= ctas <= 148


@pytest.mark.parametrize("new,keys,groups,H,kvh", [
    ([1], [1], [], 1, 1), ([1, 0, 3, 2], [40, 32, 70, 5], [(0, 3, 32)], 8, 2), ([0, 0, 5], [0, 9, 5], [], 71, 1), ([0, 0], [3, 3], [], 4, 4), ([], [], [], 4, 4),
    ([1 + i % 3 for i in range(50)], [100 + (37 * i) % 901 for i in range(50)], [(0, 20, 96), (30, 5, 64)], 20, 2), ([1] * 3, [40000, 7, 39000], [], 32, 32),
    ([1] * 300, [1 + (i % 7 == 0) * 900 for i in range(300)], [], 4, 4), ([1] * 40, [4097 + i for i in range(40)], [(0, 40, 4096)], 32, 8)])
def test_own_keys_are_dealt_out_whole(new, keys, groups, H, kvh):
    """Walking every worker's piece as the kernel does: each strip of each unit once, and the units' lists name just the workers that were there."""
    plan = plans.SharedPrefixPlan(new, keys, groups, H, kvh, 64, 16)
    items, seen, shares = plan.items.tolist(), {}, set()
    for w, (item, unit, strip, left) in enumerate(plan.workers.tolist()):
        assert left >= 0
        while left > 0:
            _, _, n, k, prefix, unit0, row_tiles, _ = items[item]
            assert n > 0 and 0 <= unit < row_tiles * kvh
            strips = -(-(k - prefix) // 16)
            for s in range(strip, min(strips, strip + left)):
                assert seen.setdefault((unit0 + unit, s), w) == w
            shares.add((unit0 + unit, w))
            left -= min(strips, strip + left) - strip
            strip, unit = 0, unit + 1
            if unit == row_tiles * kvh and left > 0:
                unit, item = 0, item + 1
                while items[item][6] == 0:
                    item += 1
    want = {(u, s) for _, _, n, k, prefix, unit0, rt, _ in items for u in range(unit0, unit0 + rt * kvh) for s in range(-(-(k - prefix) // 16))}
    assert set(seen) == want
    assert shares == {(u, w) for u, (a, b) in enumerate(plan.units.tolist()) for w in range(a, b + 1)}
    assert len({u + w for u, w in shares}) == len(shares) and max((u + w for u, w in shares), default=-1) < plan.n_units + plan.n_workers


@pytest.mark.parametrize("scale", [-1.0, float("inf"), float("nan")])
def test_attention_refuses_scales_that_are_none(scale):
    plan = plans.SharedPrefixPlan([1, 1], [40, 40], [(0, 2, 32)], 4, 2, 64, 16)
    q = torch.zeros(2, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="scale"):
        CpuOps().attention_shared(q, torch.empty_like(q), torch.zeros(9, 2, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(2, 3, dtype=torch.int32), plan, scale)


def test_attention_of_a_group_on_the_host_is_that_of_its_sequences():
    torch.manual_seed(1)
    plan = plans.SharedPrefixPlan([1, 3, 0, 2], [40, 45, 33, 5], [(0, 3, 32)], 6, 2, 32, 16)
    cache = torch.randn(12, 2, 2, 16, 32)
    tables = torch.tensor([[3, 4, 5, 0], [3, 4, 6, 0], [3, 4, 7, 0], [8, 0, 0, 0]], dtype=torch.int32)
    q = torch.randn(7, 6 * 32)
    out = torch.full_like(q, 7.0)
    SharedPrefixAttn(32, torch.float32)(out, q, cache, tables, plan)
    assert (out[6] == 7.0).all()
    row = 0
    for i, (n, keys) in enumerate(zip([1, 3, 0, 2], [40, 45, 33, 5])):
        k, v = ref.gather_kv(cache, tables[i], keys)
        for t in range(n):
            seen = keys - n + t + 1
            for h in range(6):
                w = torch.softmax(k[:seen, h // 3] @ q[row, h * 32:(h + 1) * 32] / math.sqrt(32), 0)
                torch.testing.assert_close(out[row, h * 32:(h + 1) * 32], w @ v[:seen, h // 3], atol=1e-5, rtol=1e-5)
            row += 1
    with pytest.raises(ValueError, match="heads of 32"):
        SharedPrefixAttn(64, torch.float32)(out, q, cache, tables, plan)


# ---- controls on logits ------------------------------------------------------------------------------------------------
def _naive(logits, history, prompts, rep, pres, freq, bias, allowed):
    """Token by token, in 64 bits."""
    out = logits.double().clone()
    for i in range(out.shape[0]):
        for v in range(out.shape[1]):
            x = out[i, v].item()
            if v in history[i]:
                x = x / rep[i] if x > 0 else x * rep[i]
            c = history[i][prompts[i]:].count(v)
            if c:
                x -= freq[i] * c + pres[i]
            if v in bias[i]:
                x += bias[i][v]
            out[i, v] = x if allowed is None or allowed[i, v] else -math.inf
    return out


def test_controls_follow_the_requests_through_a_batch_that_shrinks():
    torch.manual_seed(2)
    V, prompts = 41, [[3, 3, 7], [], [40, 0, 1, 2]]
    rep, pres, freq = [1.5, 1.0, 0.8], [0.5, 0.25, -0.5], [0.125, 0.5, 0.0]
    bias = [{7: 2.0, 8: -3.0}, {}, {40: -100.0}]
    allowed = torch.rand(3, V) < 0.7
    allowed[1] = False       # a grammar that allows nothing
    controls = LogitControls(prompts, V, 4, "cpu", rep, pres, freq, [bias[0], None, bias[2]], allowed)
    told, alive = [list(p) for p in prompts], [0, 1, 2]
    for step in range(4):
        logits = torch.randn(len(alive), V)
        before = logits.clone()
        want = _naive(logits, [told[i] for i in alive], [len(prompts[i]) for i in alive], [rep[i] for i in alive], [pres[i] for i in alive],
                      [freq[i] for i in alive], [bias[i] for i in alive], allowed[alive])
        torch.testing.assert_close(controls.apply(logits).double(), want, atol=1e-5, rtol=1e-5)
        assert torch.equal(logits, before)
        tokens = sample_next(logits, controls=controls)
        assert tokens.tolist() == want.argmax(-1).tolist()
        for i, tok in zip(alive, tokens.tolist()):
            told[i].append(tok)
        if step == 1:
            alive = [0, 2]
            controls.keep([0, 2])
    with pytest.raises(RuntimeError, match="max_new_tokens"):
        controls.append(torch.zeros(2, dtype=torch.int32))


def test_controls_without_any_leave_logits_alone():
    logits = torch.randn(2, 9)
    controls = LogitControls([[1], [2]], 9, 3, "cpu")
    assert controls.apply(logits) is logits
    assert sample_next(logits, controls=controls).tolist() == logits.argmax(-1).tolist()


def test_drawing_where_controls_leave_no_token():
    """Rows: nothing allowed, nothing left by the bias, one token left, an infinite logit."""
    allowed = torch.ones(4, 5, dtype=torch.bool)
    allowed[0] = False
    allowed[1, 2:] = False
    allowed[2] = torch.tensor([False, False, False, True, False])
    controls = LogitControls([[1]] * 4, 5, 6, "cpu", 1.5, logit_bias=[None, {0: -math.inf, 1: -math.inf}, None, None], allowed=allowed)
    logits = torch.zeros(4, 5)
    logits[3, 4] = math.inf
    for kw in ({}, dict(top_k=2), dict(top_p=0.5), dict(temperature=1e-9), dict(temperature=3.0, top_k=1, top_p=0.9)):
        assert sample_next(logits, do_sample=True, controls=controls, **kw).tolist() == [0, 0, 3, 4]


def test_controls_refuse():
    make = lambda **kw: LogitControls([[1], [2]], 9, 3, "cpu", **kw)  # noqa: E731
    for kw, match in ((dict(repetition_penalty=0.0), "positive"), (dict(repetition_penalty=[1.0]), "there are 2"), (dict(presence_penalty=[0.0] * 3), "there are 2"),
                      (dict(repetition_penalty=math.inf), "finite"), (dict(presence_penalty=math.nan), "finite"), (dict(frequency_penalty=-math.inf), "finite"),
                      (dict(logit_bias={3: math.inf}), "finite"), (dict(logit_bias={3: math.nan}), "finite"),
                      (dict(logit_bias=[{}]), "there are 2"), (dict(logit_bias={9: 1.0}), "vocabulary"), (dict(allowed=torch.ones(2, 8, dtype=torch.bool)), "allowed"),
                      (dict(allowed=torch.ones(2, 9)), "allowed")):
        with pytest.raises(ValueError, match=match):
            make(**kw)
    with pytest.raises(ValueError, match="logits must be"):
        make().apply(torch.zeros(3, 9))
    with pytest.raises(ValueError, match="3 tokens"):
        make().append(torch.zeros(3))


def test_masks_are_packed_by_bit():
    allowed = torch.zeros(2, 70, dtype=torch.bool)
    allowed[0, [0, 31, 32, 69]] = True
    allowed[1] = True
    assert pack_mask(allowed).tolist() == [[1 - (1 << 31), 1, 1 << 5], [-1, -1, 63]]


def test_restated_controls_pass_over_what_is_no_token():
    logits = torch.tensor([[1.0, -2.0, 3.0, 4.0]])
    i32 = lambda *v: torch.tensor([v], dtype=torch.int32)  # noqa: E731
    out = CpuOps().logit_controls(logits, torch.empty_like(logits), history=i32(1, 1, 9, -4, 2), history_len=torch.tensor([4], dtype=torch.int32),
                                  prompt_len=torch.tensor([1], dtype=torch.int32), repetition=torch.tensor([2.0]), presence=torch.tensor([0.5]),
                                  frequency=torch.tensor([0.25]), bias_ids=i32(3, -1, 3, 4), bias=torch.tensor([[1.0, 50.0, 2.0, 60.0]]),
                                  mask=i32(0b1011), mask_rows=torch.tensor([0], dtype=torch.int32))
    assert out.tolist() == [[1.0, -4.75, -math.inf, 6.0]]
    out = CpuOps().logit_controls(logits, torch.empty_like(logits), mask=i32(0), mask_rows=torch.tensor([-1], dtype=torch.int32))
    assert out.tolist() == logits.tolist()


BAD_CONTROLS = [
    (dict(history=torch.zeros(2, 3, dtype=torch.int32)), "lengths"), (dict(history_len=torch.zeros(2, dtype=torch.int32)), "lengths"),
    (dict(repetition=torch.ones(2)), "need a history"), (dict(bias=torch.zeros(2, 3)), "their tokens"), (dict(mask_rows=torch.zeros(2, dtype=torch.int32)), "needs masks"),
    (dict(history=torch.zeros(2, 3, dtype=torch.int64), history_len=torch.zeros(2, dtype=torch.int32)), "history must be"),
    (dict(history=torch.zeros(1, 3, dtype=torch.int32), history_len=torch.zeros(2, dtype=torch.int32)), "history must be"),
    (dict(history=torch.zeros(2, 3, dtype=torch.int32), history_len=torch.zeros(2, dtype=torch.int64)), "history_len must be"),
    (dict(history=torch.zeros(2, 3, dtype=torch.int32), history_len=torch.zeros(2, dtype=torch.int32), presence=torch.zeros(1)), "presence must be"),
    (dict(bias=torch.zeros(2, 3), bias_ids=torch.zeros(2, 2, dtype=torch.int32)), "one shape"), (dict(mask=torch.zeros(2, 1, dtype=torch.int32)), "mask must be"),
    (dict(mask=torch.zeros(3, 2, dtype=torch.int32)), "mask must be")]


@pytest.mark.parametrize("kw,match", BAD_CONTROLS)
def test_controls_of_wrong_shapes_are_refused(kw, match):
    with pytest.raises(ValueError, match=match):
        CpuOps().logit_controls(torch.zeros(2, 40), torch.zeros(2, 40), **kw)


def test_generate_under_a_repetition_penalty_matches_hf():
    transformers = pytest.importorskip("transformers")
    import hcache_deepspeed_b200 as ds
    torch.manual_seed(0)
    cfg = transformers.LlamaConfig(vocab_size=128, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                                   max_position_embeddings=256)
    hf = transformers.LlamaForCausalLM(cfg).eval()
    eng = ds.init_inference(hf, dtype=torch.float32, replace_with_kernel_inject=True)
    ids = torch.randint(3, 128, (2, 9))
    want = hf.generate(input_ids=ids, max_new_tokens=12, do_sample=False, pad_token_id=0, repetition_penalty=1.7)
    got = eng.generate(input_ids=ids, max_new_tokens=12, do_sample=False, repetition_penalty=1.7)
    assert torch.equal(got, want[:, :got.shape[1]])
    banned = eng.generate(input_ids=ids, max_new_tokens=4, logit_bias={int(want[0, 9]): -1e9})
    assert banned[0, 9] != want[0, 9]
    allowed = torch.zeros(2, 128, dtype=torch.bool)
    allowed[0, 5] = allowed[1, 77] = True
    assert eng.generate(input_ids=ids, max_new_tokens=3, allowed=allowed)[:, 9:].tolist() == [[5] * 3, [77] * 3]


# ---- the wrappers' checks, against a library that only notes its calls ---------------------------------------------------
def test_wrappers_want_cuda_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        kernels.logit_controls(torch.zeros(1, 4))
    with pytest.raises(ValueError, match="CUDA"):
        kernels.adapter_add(torch.zeros(1, 8), torch.zeros(1, 8), torch.zeros(1, 8, 8), torch.zeros(1, 8, 8), torch.zeros(1), kernels.AdapterPlan([0], 1))
    with pytest.raises(ValueError, match="CUDA"):
        kernels.paged_attention_shared(torch.zeros(1, 64), torch.zeros(1, 64), torch.zeros(1, 2, 1, 16, 64), torch.zeros(1, 1, dtype=torch.int32),
                                       plans.SharedPrefixPlan([1], [1], [], 1, 1, 64, 16), 1.0)
