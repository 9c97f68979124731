"""Batches of many requests on the GPU: adapters beside a projection, attention behind shared prefixes, controls on logits, and a decode step of all
three. Oracles are in 64 bits; tolerances count roundings: a value of type t is off by at most ``finfo(t).eps / 2`` of itself."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.timeout(300)]

HALF = [torch.bfloat16, torch.float16]
U32 = 2.0**-24


def K():
    from hcache_deepspeed_b200.ops import kernels
    return kernels


def rand(*shape, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(*shape, device="cuda") * std).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, want, bound):
    """No element further from ``want`` (64 bits) than its ``bound``."""
    over = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all() and (over <= 0).all(), f"off by up to {over.max().item():.3e} more than allowed"


# ---- adapters ------------------------------------------------------------------------------------------------------------
def adapters_exact(base, x, down, up, scales, ids):
    """(value, bound). The bound: sums of K and R products in 32 bits, of which a step may lose up to 2^-23 of the sum of magnitudes (the tensor cores
    cut off instead of rounding); h as two 16-bit values, 2^-17 of it and less; the result's rounding."""
    want, bound = base.double(), torch.zeros(base.shape, dtype=torch.float64, device="cuda")
    Kd, R = x.shape[1], down.shape[1]
    for t, i in enumerate(ids):
        if i >= 0:
            a, b, s = down[i].double(), up[i].double(), scales[i].double()
            h, mag = x[t].double() @ a.t(), x[t].double().abs() @ a.t().abs()
            dh = mag * (Kd + 8) * 2 * U32 + h.abs() * 2.0**-17
            want[t] += s * (h @ b.t())
            bound[t] = s.abs() * ((dh @ b.t().abs()) + (h.abs() @ b.t().abs()) * (R + 8) * 4 * U32)
    return want, bound + (want.abs() + bound) * (half_step(x.dtype) + 2 * U32) + 1e-9 + (6e-8 if x.dtype == torch.float16 else 0.0)


def adapters_inputs(T, n, Kd, N, R, dtype):
    return (rand(T, N, dtype=dtype), rand(T, Kd, dtype=dtype), rand(n, R, Kd, dtype=dtype, std=Kd**-0.5), rand(n, N, R, dtype=dtype, std=R**-0.5),
            torch.rand(n, device="cuda") + 0.5)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("ids,n,Kd,N,R", [
    ([0], 1, 8, 8, 8), ([2], 3, 4096, 1024, 16), ([-1, 1, -1, 0, 1], 2, 264, 1096, 24), ([-1] * 70, 2, 64, 264, 8), (list(range(33)), 33, 520, 512, 40),
    ([0] * 17 + [1] * 33 + [-1] * 3 + [0] * 16, 2, 1000, 776, 64), ([i % 3 for i in range(200)], 3, 256, 328, 32), ([0] * 130, 1, 72, 2048, 72),
    ([1] * 40 + [0], 2, 512, 72, 256), ([0, 1] * 60, 2, 2048, 256, 136)])
def test_adapters(dtype, ids, n, Kd, N, R):
    torch.manual_seed(0)
    base, x, down, up, scales = adapters_inputs(len(ids), n, Kd, N, R, dtype)
    plan = K().AdapterPlan(ids, n, device="cuda")
    want, bound = adapters_exact(base, x, down, up, scales, ids)
    kept = base.clone()
    out = K().adapter_add(base, x, down, up, scales, plan)
    assert torch.equal(base, kept)
    check(out, want, bound)
    assert torch.equal(K().adapter_add(base, x, down, up, scales, plan, out=base), out) and torch.equal(base, out)       # in place
    assert torch.equal(out[torch.tensor(ids) < 0], kept[torch.tensor(ids) < 0])


@pytest.mark.parametrize("dtype", HALF)
def test_adapters_of_rows_apart_in_memory(dtype):
    torch.manual_seed(1)
    ids = [0, 1, -1, 1, 0, 0, 1]
    base, x, down, up, scales = adapters_inputs(7, 2, 192, 136, 16, dtype)
    wide_x, wide_base, wide_out = (torch.full((7, c), 9.0, dtype=dtype, device="cuda") for c in (208, 160, 152))
    wide_x[:, 8:200], wide_base[:, 16:152] = x, base
    plan = K().AdapterPlan(ids, 2, device="cuda")
    out = K().adapter_add(wide_base[:, 16:152], wide_x[:, 8:200], down, up, scales, plan, out=wide_out[:, 8:144])
    assert torch.equal(out, K().adapter_add(base, x, down, up, scales, plan))
    assert (wide_out[:, :8] == 9).all() and (wide_out[:, 144:] == 9).all()


@pytest.mark.parametrize("rows", [6, 40])       # one kernel, and two
def test_adapters_of_rows_far_apart_and_in_place_of_x(rows):
    ids, ld = [0] * (rows - 2) + [1, -1], 1 << 27
    base, x, down, up, scales = adapters_inputs(rows, 2, 520, 520, 24, torch.bfloat16)
    plan = K().AdapterPlan(ids, 2, device="cuda")
    want, bound = adapters_exact(base, x, down, up, scales, ids)
    wide = torch.empty(rows, ld, dtype=torch.bfloat16, device="cuda")
    far, x_far = wide[:, ld - 520:], wide[:, :520]
    far.copy_(base)
    x_far.copy_(x)
    K().adapter_add(far, x_far, down, up, scales, plan, out=far)
    check(far, want, bound)
    far.copy_(base)
    K().adapter_add(far, x_far, down, up, scales, plan, out=x_far)
    check(x_far, want, bound)
    assert torch.equal(far, base)


def test_adapters_keep_large_and_small_sums():
    """fp16: h of 10^5 has no place in 16 bits, h of 10^-6 few bits."""
    torch.manual_seed(2)
    base, x, down, up, scales = adapters_inputs(4, 2, 512, 64, 16, torch.float16)
    base.zero_()
    x[:2] *= 4000.0
    down[0] *= 30.0
    up[0] *= 2.0**-9
    x[2:] *= 2.0**-10
    up[1] *= 16.0
    ids = [0, 0, 1, 1]
    want, bound = adapters_exact(base, x, down, up, scales, ids)
    assert ((x[:2].float() @ down[0].float().t()).abs() > 65504).any()
    check(K().adapter_add(base, x, down, up, scales, K().AdapterPlan(ids, 2, device="cuda")), want, bound)


def test_a_row_of_an_adapter_keeps_its_nan_to_itself():
    torch.manual_seed(3)
    ids = [0, 0, 1, -1]
    base, x, down, up, scales = adapters_inputs(4, 2, 64, 64, 8, torch.bfloat16)
    plan = K().AdapterPlan(ids, 2, device="cuda")
    clean = K().adapter_add(base, x, down, up, scales, plan)
    x[1, 5] = math.nan
    x[3] = math.nan
    out = K().adapter_add(base, x, down, up, scales, plan)
    assert torch.equal(out[[0, 2, 3]], clean[[0, 2, 3]]) and out[1].isnan().all()


def test_adapters_refuse():
    k = K()
    base, x, down, up, scales = adapters_inputs(3, 2, 64, 32, 8, torch.bfloat16)
    plan = k.AdapterPlan([0, 1, -1], 2, device="cuda")
    good = dict(base=base, x=x, down=down, up=up, scales=scales, plan=plan)
    for kw, err in ((dict(plan=k.AdapterPlan([0, 1], 2, device="cuda")), ValueError), (dict(plan=k.AdapterPlan([0, 1, -1], 3, device="cuda")), ValueError),
                    (dict(plan=k.AdapterPlan([0, 1, -1], 2)), ValueError), (dict(x=x.half()), TypeError), (dict(x=x.float()), TypeError),
                    (dict(scales=scales.half()), TypeError), (dict(scales=scales[:1]), ValueError), (dict(up=up.transpose(1, 2)), ValueError),
                    (dict(down=down[:, :4].contiguous(), up=up[:, :, :4].contiguous()), ValueError), (dict(x=x.t()), ValueError), (dict(scales=scales.cpu()), ValueError),
                    (dict(x=x[:, :60], down=down[:, :, :60].contiguous()), ValueError), (dict(out=base[:, :24]), ValueError), (dict(out=base.half()), ValueError)):
        with pytest.raises(err):
            k.adapter_add(**{**good, **kw})
    wide = torch.zeros(3, 68, dtype=torch.bfloat16, device="cuda")
    from hcache_deepspeed_b200.ops.native import HdsKernelError
    with pytest.raises(HdsKernelError, match="16-byte"):       # rows that start off a boundary
        k.adapter_add(base, wide[:, :64], down, up, scales, plan)
    with pytest.raises(HdsKernelError, match="16-byte"):
        k.adapter_add(base, wide.view(-1)[4:196].view(3, 64), down, up, scales, plan)
    none = k.AdapterPlan([], 2, device="cuda")
    assert k.adapter_add(base[:0], x[:0], down, up, scales, none).shape == (0, 32)


def test_a_linear_with_many_adapters():
    from hcache_deepspeed_b200.linear import AdapterBank, MultiAdapterLinear
    torch.manual_seed(4)
    bank = AdapterBank(3, 12, 256, 512, device="cuda")
    for i in range(3):
        bank.load(i, rand(12 - i, 256, std=1 / 16), rand(512, 12 - i, std=0.3), 0.5)
    w = rand(512, 256, std=1 / 16)
    layer = MultiAdapterLinear(w, bank)
    ids = [0, -1, 2, 1, 2]
    x = rand(5, 256)
    y = layer(x, bank.plan(ids))
    plain = K().gemm(x, w)
    want, bound = adapters_exact(plain, x, bank.down, bank.up, bank.scales, ids)
    check(y, want, bound)


# ---- attention behind shared prefixes --------------------------------------------------------------------------------------
def pages(lengths, groups, kvh, d, bs, dtype, spare=2):
    """(cache, tables) of sequences with that many keys, whose groups share their prefixes' pages; pages in random order, tails and spare pages NaN."""
    own = {}
    ids = iter(torch.randperm(sum(-(-n // bs) for n in lengths) + spare).tolist())
    width = max(-(-n // bs) for n in lengths) + 1
    tables = torch.zeros(len(lengths), width, dtype=torch.int32)
    for first, n, prefix in groups:
        row = [next(ids) for _ in range(prefix // bs)]
        for i in range(first, first + n):
            own[i] = row
    cache = torch.full((sum(-(-n // bs) for n in lengths) + spare, 2, kvh, bs, d), math.nan, dtype=dtype, device="cuda")
    for i, n in enumerate(lengths):
        row = list(own.get(i, []))
        row += [next(ids) for _ in range(-(-n // bs) - len(row))]
        tables[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
        for b, page in enumerate(row):
            live = min(bs, n - b * bs)
            cache[page, :, :, :live] = torch.where(cache[page, :, :, :live].isnan(), rand(2, kvh, live, d, dtype=dtype), cache[page, :, :, :live])
    return cache, tables.cuda()


def attention_exact(q, cache, tables, new, keys, prefix, H, scale):
    """(value, bound). The bound: scores of d products in 32 bits (cut off, see above) and exponentials to 2^-21 move a weight by a factor; of the
    prefix' keys weights are rounded to the type, of the others to 2^-16; sums of all keys in 32 bits; the result's rounding."""
    kvh, bs, d = cache.shape[2], cache.shape[3], cache.shape[4]
    G = H // kvh
    want = torch.empty(sum(new), H, d, dtype=torch.float64, device="cuda")
    bound = torch.empty_like(want)
    row = 0
    u = half_step(q.dtype)
    for i, n in enumerate(new):
        if not n:
            continue
        kv = cache[tables[i, :-(-keys[i] // bs)].long()].double().permute(1, 2, 0, 3, 4).reshape(2, kvh, -1, d)[:, :, :keys[i]]
        k, v = (t.repeat_interleave(G, 0) for t in kv)
        for t in range(n):
            sees = keys[i] - n + t + 1
            x = q[row].double().view(H, d)
            s = torch.einsum("hd,hkd->hk", x, k[:, :sees]) * scale
            ds = (torch.einsum("hd,hkd->hk", x.abs(), k[:, :sees].abs()) * scale * (d + 8) * 2 * U32).amax(1)
            w = torch.softmax(s, 1)
            want[row] = torch.einsum("hk,hkd->hd", w, v[:, :sees])
            mag = torch.einsum("hk,hkd->hd", w, v[:, :sees].abs())
            rounded = torch.einsum("hk,hkd->hd", w[:, :prefix[i]], v[:, :prefix[i]].abs())
            rel = (2 * ds + 2.0**-20)[:, None]
            bound[row] = mag * (rel + 2.0**-15 + (sees + 64) * 2 * U32) + rounded * u + (want[row].abs() + mag * rel) * u
            row += 1
    return want.view(row, -1), bound.view(row, -1) * 1.01 + (6e-8 if q.dtype == torch.float16 else 0.0)


SHARED = [
    # new tokens, own keys, groups (first, n, prefix), heads, KV heads, dim, block
    ([1], [1], [(0, 1, 16)], 1, 1, 64, 16),
    ([1, 1], [1, 17], [(0, 2, 128)], 2, 2, 128, 128),
    ([1, 1, 1], [5, 64, 130], [(0, 3, 144)], 8, 2, 64, 16),
    ([1] * 5, [3, 40, 1, 700, 9], [(0, 2, 64), (3, 2, 192)], 4, 4, 128, 64),         # a lone sequence between two groups
    ([2, 1, 3, 0, 1], [2, 5, 3, 1, 260], [(0, 4, 96)], 14, 2, 128, 32),              # seven heads share a KV head; a sequence without new tokens
    ([1] * 70, [1 + 7 * i % 50 for i in range(70)], [(0, 70, 160)], 8, 1, 64, 32),   # several tiles of rows
    ([1, 4], [30, 4], [(0, 2, 1024)], 20, 2, 64, 64),                                # ten heads share a KV head: two tiles of eight rows and more
    ([1, 1], [20, 33], [(0, 1, 0), (1, 1, 0)], 8, 8, 128, 16),                        # prefixes of no tokens
    ([1, 2], [600, 3000], [], 16, 4, 128, 64),                                       # nothing is shared
    ([1] * 3, [2, 2, 2], [(0, 3, 4096)], 71, 1, 64, 128),                             # one KV head for 71: a tile of one token
    ([1] * 130, [1] * 130, [(0, 130, 48)], 1, 1, 128, 16),
    ([1] * 4, [16000, 3, 1, 40], [(1, 2, 64)], 1, 1, 64, 16),                         # many parts next to few
    ([1] * 160, [8000] + [1 + 3 * i % 20 for i in range(159)], [], 32, 1, 64, 16),    # the same with more rows than fill the device
]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("new,own,groups,H,kvh,d,bs", SHARED)
def test_attention_behind_a_shared_prefix(dtype, new, own, groups, H, kvh, d, bs):
    torch.manual_seed(5)
    prefix = [0] * len(new)
    for first, n, p in groups:
        prefix[first:first + n] = [p] * n
    keys = [p + o for p, o in zip(prefix, own)]
    cache, tables = pages(keys, groups, kvh, d, bs, dtype)
    plan = K().SharedPrefixPlan(new, keys, groups, H, kvh, d, bs, device="cuda")
    q = rand(sum(new) + 2, H * d, dtype=dtype, std=2.0)
    out = torch.full_like(q, 7.0)
    K().paged_attention_shared(q, out, cache, tables, plan, d**-0.5)
    want, bound = attention_exact(q, cache, tables, new, keys, prefix, H, d**-0.5)
    check(out[:-2], want, bound)
    assert (out[-2:] == 7).all()        # rows behind the last sequence


@pytest.mark.parametrize("splits", [1, 2, 3, 8, 64])
@pytest.mark.parametrize("dtype", HALF)
def test_parts_of_prefix_and_own_keys_join(dtype, splits):
    torch.manual_seed(6)
    new, keys, groups = [1, 2, 1], [1100 + 5, 1100 + 900, 2], [(0, 2, 1088)]
    cache, tables = pages(keys, groups, 2, 128, 64, dtype)
    plan = K().SharedPrefixPlan(new, keys, groups, 8, 2, 128, 64, device="cuda")
    plan.p_splits = splits
    q = rand(4, 1024, dtype=dtype, std=3.0)
    out = K().paged_attention_shared(q, torch.empty_like(q), cache, tables, plan, 128**-0.5)
    check(out, *attention_exact(q, cache, tables, new, keys, [1088, 1088, 0], 8, 128**-0.5))


def test_a_prefix_far_above_or_below_the_own_keys():
    """Weights of one part that vanish beside the other's, and maxima that grow by far more than 2^8 between tiles."""
    torch.manual_seed(7)
    new, keys, groups = [1, 1], [512 + 20, 512 + 20], [(0, 2, 512)]
    cache, tables = pages(keys, groups, 1, 64, 16, torch.bfloat16)
    q = rand(2, 4 * 64, std=2.0)
    plan = K().SharedPrefixPlan(new, keys, groups, 4, 1, 64, 16, device="cuda")
    for scale in (0.0, 0.125, 20.0):
        for page, f in ((int(tables[0, 20]), 30.0), (int(tables[1, 32]), 8.0)):
            cache[page, 0, :, :3] *= f
        out = K().paged_attention_shared(q, torch.empty_like(q), cache, tables, plan, scale)
        check(out, *attention_exact(q, cache, tables, new, keys, [512] * 2, 4, scale))


@pytest.mark.parametrize("dtype", HALF)
def test_attention_takes_rows_apart_in_memory(dtype):
    torch.manual_seed(8)
    new, keys, groups = [1, 2], [70, 75], [(0, 2, 64)]
    cache, tables = pages(keys, groups, 2, 64, 32, dtype)
    plan = K().SharedPrefixPlan(new, keys, groups, 4, 2, 64, 32, device="cuda")
    wide = rand(3, 4 * 64 + 2 * 2 * 64 + 8, dtype=dtype)       # q in its place in q | k | v
    out = torch.full((3, 304), 5.0, dtype=dtype, device="cuda")
    K().paged_attention_shared(wide[:, 8:264], out[:, 16:272], cache, tables, plan, 0.125)
    dense = K().paged_attention_shared(wide[:, 8:264].contiguous(), torch.empty(3, 256, dtype=dtype, device="cuda"), cache, tables, plan, 0.125)
    assert torch.equal(out[:, 16:272], dense) and (out[:, :16] == 5).all() and (out[:, 272:] == 5).all()


def test_attention_in_a_cache_of_more_than_2_to_32_values():
    torch.manual_seed(9)
    new, keys, groups, kvh, d, bs = [1, 2], [256 + 30, 256 + 140], [(0, 2, 256)], 8, 128, 128
    small, tables = pages(keys, groups, kvh, d, bs, torch.bfloat16)
    n, first = small.shape[0], 17000
    cache = torch.empty(first + n, 2, kvh, bs, d, dtype=torch.bfloat16, device="cuda")
    assert cache.numel() > 1 << 32
    cache[first:] = small
    plan = K().SharedPrefixPlan(new, keys, groups, 16, kvh, d, bs, device="cuda")
    q = rand(3, 16 * d, std=2.0)
    out = K().paged_attention_shared(q, torch.empty_like(q), cache, tables + first, plan, d**-0.5)
    assert torch.equal(out, K().paged_attention_shared(q, torch.empty_like(q), small, tables, plan, d**-0.5))
    check(out, *attention_exact(q, small, tables, new, keys, [256, 256], 16, d**-0.5))


def test_attention_may_write_over_its_queries():
    torch.manual_seed(10)
    new, keys, groups = [1, 2], [150, 170], [(0, 2, 128)]
    cache, tables = pages(keys, groups, 2, 64, 32, torch.float16)
    plan = K().SharedPrefixPlan(new, keys, groups, 8, 2, 64, 32, device="cuda")
    q = rand(3, 512, dtype=torch.float16)
    want = K().paged_attention_shared(q, torch.empty_like(q), cache, tables, plan, 0.125)
    assert torch.equal(K().paged_attention_shared(q, q, cache, tables, plan, 0.125), want)


def test_attention_refuses():
    k = K()
    plan = k.SharedPrefixPlan([1, 1], [40, 40], [(0, 2, 32)], 4, 2, 64, 16, device="cuda")
    good = dict(q=rand(2, 256), out=rand(2, 256), kv_cache_layer=torch.zeros(9, 2, 2, 16, 64, dtype=torch.bfloat16, device="cuda"),
                block_tables=torch.zeros(2, 3, dtype=torch.int32, device="cuda"), plan=plan, scale=0.125)
    for kw, err in ((dict(q=rand(1, 256)), ValueError), (dict(q=rand(2, 128)), ValueError), (dict(out=rand(1, 256)), ValueError), (dict(out=rand(2, 256).half()), TypeError),
                    (dict(q=rand(2, 256).float()), TypeError), (dict(kv_cache_layer=good["kv_cache_layer"].half()), TypeError),
                    (dict(kv_cache_layer=good["kv_cache_layer"][:, :, :1]), ValueError), (dict(kv_cache_layer=good["kv_cache_layer"].transpose(3, 4)), ValueError),
                    (dict(block_tables=good["block_tables"][:1]), ValueError), (dict(block_tables=good["block_tables"][:, :2]), ValueError),
                    (dict(block_tables=good["block_tables"].long()), ValueError), (dict(block_tables=good["block_tables"].cpu()), ValueError),
                    (dict(plan=k.SharedPrefixPlan([1, 1], [40, 40], [], 4, 2, 64, 16)), ValueError),
                    (dict(scale=-0.125), ValueError), (dict(scale=math.inf), ValueError), (dict(scale=math.nan), ValueError),
                    (dict(plan=k.SharedPrefixPlan([1, 1], [40, 40], [], 4, 2, 96, 16, device="cuda"), q=rand(2, 384), out=rand(2, 384)), ValueError)):
        with pytest.raises(err):
            k.paged_attention_shared(**{**good, **kw})
    from hcache_deepspeed_b200.ops.native import HdsKernelError
    with pytest.raises(HdsKernelError, match="16-byte"):
        k.paged_attention_shared(**{**good, "q": rand(2, 260)[:, :256]})
    nothing = k.SharedPrefixPlan([0, 0], [40, 40], [(0, 2, 32)], 4, 2, 64, 16, device="cuda")
    out = torch.full_like(good["q"], 3.0)
    assert (k.paged_attention_shared(**{**good, "plan": nothing, "out": out}) == 3).all()


# ---- controls on logits ------------------------------------------------------------------------------------------------
def controls_exact(logits, history=None, history_len=None, prompt_len=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias=None, mask=None,
                   mask_rows=None):
    """(value, bound). Each step in 32 bits rounds once: half a step of what stands before and after it; then the result's rounding."""
    x = logits.double().cpu()
    n, V = x.shape
    mag = x.abs()
    for i in range(n):
        if history is not None:
            told = history[i, :max(0, int(history_len[i]))].tolist()
            prompt = int(prompt_len[i]) if prompt_len is not None else 0
            count, seen = {}, set()
            for j, v in enumerate(told):
                if 0 <= v < V:
                    seen.add(v)
                    if j >= prompt:
                        count[v] = count.get(v, 0) + 1
            for v in seen:
                if repetition is not None:
                    r = float(repetition[i])
                    x[i, v] = x[i, v] / r if x[i, v] > 0 else x[i, v] * r
                    mag[i, v] = torch.maximum(mag[i, v], x[i, v].abs())
                if v in count:
                    f, p = (0.0 if t is None else float(t[i]) for t in (frequency, presence))
                    x[i, v] -= f * count[v] + p
                    mag[i, v] += abs(f) * count[v] + abs(p)
        if bias is not None:
            for v, b in {int(t): float(b) for t, b in zip(bias_ids[i], bias[i])}.items():
                if 0 <= v < V:
                    x[i, v] += b
                    mag[i, v] += abs(b)
        m = None if mask is None else (i if mask_rows is None else int(mask_rows[i]))
        if m is not None and 0 <= m < mask.shape[0]:
            for v in range(V):
                if not int(mask[m, v // 32]) >> (v % 32) & 1:
                    x[i, v] = -math.inf
    return x, mag * 8 * U32 + x.abs().nan_to_num(posinf=0.0) * half_step(logits.dtype) + 1e-30 + (6e-8 if logits.dtype == torch.float16 else 0.0)


def controls_check(got, want, bound):
    got = got.double().cpu()
    assert torch.equal(got == -math.inf, want == -math.inf) and not got.isnan().any()
    live = want > -math.inf
    over = ((got - want).abs() - bound)[live]
    assert (over <= 0).all(), over.max()


def controls_inputs(n, V, dtype, cap, k, words, seed=9):
    torch.manual_seed(seed)
    i32 = dict(dtype=torch.int32, device="cuda")
    c = {"history": torch.randint(-2, V + 2, (n, cap), **i32), "history_len": torch.randint(-1, cap + 3, (n, ), **i32), "repetition": torch.rand(n, device="cuda") + 0.5,
         "presence": torch.randn(n, device="cuda"), "frequency": torch.randn(n, device="cuda") / 4}
    c["prompt_len"] = (c["history_len"] // 3).to(torch.int32)
    if k:
        c["bias_ids"], c["bias"] = torch.randint(-2, V + 2, (n, k), **i32), torch.randn(n, k, device="cuda") * 3
    if words:
        c["mask"] = torch.randint(-(1 << 31), 1 << 31, (3, -(-V // 32) + words - 1), **i32)
        c["mask"][2] = 0                       # allows nothing
        c["mask_rows"] = (torch.arange(n) % 5 - 1).to(**i32)      # 3 is no mask
    return rand(n, V, dtype=dtype, std=4.0), c


@pytest.mark.parametrize("dtype", HALF + [torch.float32])
@pytest.mark.parametrize("n,V,cap,k,words", [(1, 1, 1, 0, 1), (3, 31, 5, 2, 1), (2, 33, 40, 3, 2), (7, 1000, 200, 0, 1), (5, 2051, 17, 9, 3), (2, 8193, 3000, 50, 0),
                                             (31, 4097, 64, 300, 1)])
def test_controls(dtype, n, V, cap, k, words):
    logits, c = controls_inputs(n, V, dtype, cap, k, words)
    want, bound = controls_exact(logits, **c)
    before = logits.clone()
    out = K().logit_controls(logits, **c)
    assert torch.equal(logits, before)
    controls_check(out, want, bound)
    assert torch.equal(K().logit_controls(logits, logits, **c), out) and torch.equal(logits, out)      # in place


@pytest.mark.parametrize("dtype", HALF + [torch.float32])
def test_controls_of_large_batches(dtype):
    """Enough rows for the larger chunks, against the restatement in torch."""
    from hcache_deepspeed_b200.ops import reference as ref
    logits, c = controls_inputs(90, 20001, dtype, 500, 20, 1)
    c["history_len"].clamp_(0, 500)
    want = ref.logit_controls(logits.float(), **c).double()
    out = K().logit_controls(logits, **c).double()
    assert torch.equal(out == -math.inf, want == -math.inf)
    live = want > -math.inf
    # up to eight steps in 32 bits on each side, of values up to |x| * 2 (rep >= 1/2), 500 counts of frequencies below 2, and biases below 30; the result's rounding
    bound = 16 * U32 * (logits.double().abs() * 2 + 2 * 500 + 40) + want.abs() * half_step(dtype)
    assert ((out - want).abs() <= bound)[live].all()


@pytest.mark.parametrize("given", [("history", "history_len", "repetition"), ("history", "history_len", "presence"), ("history", "history_len", "prompt_len", "frequency"),
                                   ("bias_ids", "bias"), ("mask", "mask_rows"), ("history", "history_len"), ()])
def test_controls_one_by_one(given):
    logits, c = controls_inputs(6, 777, torch.float32, 50, 8, 1)
    c = {k: c[k] for k in given}
    out = K().logit_controls(logits, **c)
    controls_check(out, *controls_exact(logits, **c))
    if not given:
        assert torch.equal(out, logits)


@pytest.mark.parametrize("dtype", HALF + [torch.float32])
def test_controls_of_rows_on_any_address(dtype):
    logits, c = controls_inputs(4, 301, dtype, 30, 5, 1)
    want, bound = controls_exact(logits, **c)
    for shift_in, shift_out in ((0, 1), (3, 3), (1, 2), (5, 0)):
        wide, out = torch.full((4, 311), 2.0, dtype=dtype, device="cuda"), torch.full((4, 313), 3.0, dtype=dtype, device="cuda")
        wide[:, shift_in:shift_in + 301] = logits
        K().logit_controls(wide[:, shift_in:shift_in + 301], out[:, shift_out:shift_out + 301], **c)
        controls_check(out[:, shift_out:shift_out + 301], want, bound)
        assert (out[:, :shift_out] == 3).all() and (out[:, shift_out + 301:] == 3).all()


def test_controls_of_rows_far_apart():
    V, ld = 5000, 1 << 28
    logits, c = controls_inputs(10, V, torch.float16, 900, 7, 1)
    want, bound = controls_exact(logits, **c)
    wide = torch.empty(10, ld, dtype=torch.float16, device="cuda")
    wide[:, :V] = logits
    K().logit_controls(wide[:, :V], wide[:, ld - V:], **c)
    controls_check(wide[:, ld - V:], want, bound)


def test_controls_pass_infinities_and_nan_on():
    logits = torch.tensor([[math.inf, -math.inf, math.nan, 1.0, math.nan]], device="cuda")
    i32 = lambda *v: torch.tensor([v], dtype=torch.int32, device="cuda")  # noqa: E731
    out = K().logit_controls(logits, history=i32(0, 1, 2, 3), history_len=i32(4)[0], repetition=torch.tensor([2.0], device="cuda"),
                             bias_ids=i32(3), bias=torch.tensor([[-math.inf]], device="cuda"), mask=i32(0b01111))
    assert out[0, 0] == math.inf and out[0, 1] == -math.inf and out[0, 2].isnan() and out[0, 3] == -math.inf and out[0, 4] == -math.inf


def test_a_token_told_often_is_counted_exactly():
    V, n = 70, 40000
    history = torch.full((1, n), 69, dtype=torch.int32, device="cuda")
    history[0, ::4] = 3
    out = K().logit_controls(torch.zeros(1, V, device="cuda"), history=history, history_len=torch.tensor([n], dtype=torch.int32, device="cuda"),
                             frequency=torch.ones(1, device="cuda"))
    assert out[0, 69] == -30000 and out[0, 3] == -10000 and out[0, 4] == 0


def test_controls_refuse_on_the_gpu():
    from tests.test_requests_cpu import BAD_CONTROLS
    logits = torch.zeros(2, 40, device="cuda")
    for kw, match in BAD_CONTROLS:
        with pytest.raises(ValueError, match=match):
            K().logit_controls(logits, **{k: v.cuda() for k, v in kw.items()})
    with pytest.raises(TypeError):
        K().logit_controls(logits.double())
    with pytest.raises(ValueError, match="the call is on"):
        K().logit_controls(logits, bias=torch.zeros(2, 3), bias_ids=torch.zeros(2, 3, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="like logits"):
        K().logit_controls(logits, logits.half())
    assert K().logit_controls(logits[:0]).shape == (0, 40) and K().logit_controls(logits[:, :0]).shape == (2, 0)


# ---- together ------------------------------------------------------------------------------------------------------------
class Step:
    """A decode step of one layer: queries through a projection with adapters, attention behind a shared prefix, an output projection with adapters, logits
    under controls, the most likely token."""

    def __init__(self, dtype, S=9, H=8, kvh=2, d=64, V=1003, width=256):
        torch.manual_seed(10)
        self.new, self.keys, self.groups = [1] * S, [96 + 1 + 13 * i for i in range(S - 2)] + [1, 50], [(0, S - 2, 96)]
        self.prefix = [96] * (S - 2) + [0, 0]
        self.cache, self.tables = pages(self.keys, self.groups, kvh, d, 32, dtype)
        self.ids = [i % 4 - 1 for i in range(S)]
        self.H, self.d, self.scale = H, d, d**-0.5
        self.x = rand(S, width, dtype=dtype)
        self.wq, self.wv = rand(H * d, width, dtype=dtype, std=2 * width**-0.5), rand(V + 5, H * d, dtype=dtype, std=4 * (H * d)**-0.5)[:V]
        _, _, self.dq, self.uq, self.sq = adapters_inputs(S, 3, width, H * d, 16, dtype)
        _, self.c = controls_inputs(S, V, dtype, 40, 6, 1)
        self.c["mask"] |= 1          # token 0 is always allowed
        self.adapters = K().AdapterPlan(self.ids, 3, device="cuda")
        self.plan = K().SharedPrefixPlan(self.new, self.keys, self.groups, H, kvh, d, 32, device="cuda")
        self.o = torch.empty(S, H * d, dtype=dtype, device="cuda")

    def run(self):
        k = K()
        self.base = k.gemm(self.x, self.wq)
        self.q = k.adapter_add(self.base, self.x, self.dq, self.uq, self.sq, self.adapters)
        k.paged_attention_shared(self.q, self.o, self.cache, self.tables, self.plan, self.scale)
        self.logits = k.gemm(self.o, self.wv)
        self.ruled = k.logit_controls(self.logits, **self.c)
        return k.argmax(self.ruled)

    def check(self, tokens):
        check(self.q, *adapters_exact(self.base, self.x, self.dq, self.uq, self.sq, self.ids))
        check(self.o, *attention_exact(self.q, self.cache, self.tables, self.new, self.keys, self.prefix, self.H, self.scale))
        want, bound = controls_exact(self.logits, **self.c)
        controls_check(self.ruled, want, bound)
        assert tokens.tolist() == self.ruled.float().argmax(-1).tolist()


@pytest.mark.parametrize("dtype", HALF)
def test_a_decode_step(dtype):
    step = Step(dtype)
    step.check(step.run())


def test_a_decode_step_in_a_graph_and_on_other_streams():
    """Captured, replayed with other values, and twice at once: two graphs on two streams share plans and inputs."""
    from hcache_deepspeed_b200.utils.cuda_graph import capture
    step = Step(torch.bfloat16)
    step.run()
    first, t1 = capture(step.run)
    kept = {n: getattr(step, n) for n in ("base", "q", "o", "logits", "ruled")}
    step.o = torch.empty_like(step.o)
    second, t2 = capture(step.run)
    step.x.copy_(rand(*step.x.shape))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip((first, second), streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    step.check(t2)
    for n, t in kept.items():
        assert torch.equal(t, getattr(step, n))
        setattr(step, n, t)
    step.check(t1)


def test_tokens_under_controls_on_the_gpu():
    from hcache_deepspeed_b200.inference.sampling import LogitControls, sample_next
    torch.manual_seed(11)
    V = 517
    args = dict(repetition_penalty=1.3, presence_penalty=[0.5, 0.0, 1.0], frequency_penalty=0.25, logit_bias=[{5: 4.0}, None, {7: 3.0, 9: -1.0}],
                allowed=torch.rand(3, V) < 0.5)
    a, b = (LogitControls([[1, 2], [3], []], V, 8, dev, **args) for dev in ("cuda", "cpu"))
    for step in range(8):
        logits = torch.randn(a.n, V)
        assert sample_next(logits.cuda(), controls=a).tolist() == sample_next(logits, controls=b).tolist()
        if step == 3:
            a.keep([0, 2])
            b.keep([0, 2])


def test_drawing_where_controls_leave_no_token_on_the_gpu():
    """Rows: nothing allowed, nothing left by the bias, one token left, an infinite logit."""
    from hcache_deepspeed_b200.inference.sampling import LogitControls, sample_next
    allowed = torch.ones(4, 5, dtype=torch.bool)
    allowed[0] = False
    allowed[1, 2:] = False
    allowed[2] = torch.tensor([False, False, False, True, False])
    controls = LogitControls([[1]] * 4, 5, 6, "cuda", 1.5, logit_bias=[None, {0: -math.inf, 1: -math.inf}, None, None], allowed=allowed)
    logits = torch.zeros(4, 5, device="cuda")
    logits[3, 4] = math.inf
    for kw in ({}, dict(top_k=2), dict(top_p=0.5), dict(temperature=1e-9), dict(temperature=3.0, top_k=1, top_p=0.9)):
        assert sample_next(logits, do_sample=True, controls=controls, **kw).tolist() == [0, 0, 3, 4]
